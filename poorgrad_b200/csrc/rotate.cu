// rotate.cu -- the root-mean-square norm of every query and key head with the rotation by the
// token's position, and its backward pass.
//
// With n = x / sqrt(mean(x^2) + eps) and z = w n, each turned pair (u, v) of z becomes
// (u c - v s, v c + u s).  Back: dz is dy turned by -s, dw = sum dz n over tokens and heads, and
// dx = (w dz - n mean(w dz n)) / sqrt(mean(x^2) + eps); the norm is worked out again from x, so that
// nothing is kept from the forward pass.  Every row is read once and written once.
//
// Measured on B200 (against a copy's 6.55 TB/s): 8 x 1024 tokens x (32 + 8) heads of 128 in bf16
// forward 31 us, 5.4 TB/s, backward 50 us, 5.0 TB/s; (12 + 12) heads of 64 in f32 backward 29 us,
// 5.2 TB/s.  Memory latency bounds it: a lane holds a head's angles, weights and both rows, so few
// warps fit a SM (24 forwards, 16 backwards).  Heads whose chunks are no power of two leave lanes idle
// (24 heads of 80 in bf16 forward 22 us, 2.9 TB/s), and heads of odd halves go element by element (24
// heads of 34 in f32 29 us, 1.8 TB/s).
#include <algorithm>

#include "operators.h"

namespace tb {
namespace {

// The elements of a head fall into dim / 2 pairs: the turned ones as the style says, then the
// rest, which pass as pairs with cosine 1 and sine 0.
struct Pair {
  int u, v;
};
__device__ __forceinline__ Pair pair_of(int p, int dim, int turned, int style) {
  const int half = turned / 2;
  if (p >= half) return {turned + (p - half), turned + (p - half) + (dim - turned) / 2};
  return style == TB_ROTATE_HALVES ? Pair{p, p + half} : Pair{2 * p, 2 * p + 1};
}
__device__ __forceinline__ float2 turn_of(const tb_rotate_desc& d, int64_t position, int p) {
  const int half = (int)d.turned / 2;
  if (position < 0 || position >= d.table_rows) return {NAN, NAN};
  if (p >= half) return {1.0f, 0.0f};
  const float* row = d.table + position * d.turned;
  return {row[p], row[half + p]};
}

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(~0u, v, o);
  return v;
}

struct Row {
  int64_t b, t, head;
  bool key;
};
// Rows in the order token, then query heads, then key heads.
__device__ __forceinline__ Row row_of(const tb_rotate_desc& d, int64_t i) {
  const int64_t heads = d.q_heads + d.k_heads, token = i / heads, h = i % heads;
  return {token / d.length, token % d.length, h < d.q_heads ? h : h - d.q_heads, h >= d.q_heads};
}
template <typename T>
__device__ __forceinline__ T* at(const void* base, const int64_t s[3], const Row& r) {
  return (T*)base + r.b * s[0] + r.t * s[1] + r.head * s[2];
}
__device__ __forceinline__ int64_t position_of(const tb_rotate_desc& d, const Row& r) {
  return d.positions ? d.positions[r.b * d.length + r.t] : r.t;
}

// A warp per head.
template <typename T>
__global__ void k_rotate(tb_rotate_desc d, int64_t rows) {
  pdl_entry();
  const int lane = threadIdx.x % 32, pairs = (int)d.dim / 2;
  const int64_t i = ((int64_t)blockIdx.x * blockDim.x + threadIdx.x) / 32;
  if (i >= rows) return;
  const Row r = row_of(d, i);
  const T* x = at<T>(r.key ? d.k : d.q, r.key ? d.k_strides : d.q_strides, r);
  T* y = at<T>(r.key ? d.k_out : d.q_out, r.key ? d.k_out_strides : d.q_out_strides, r);
  const float* w = r.key ? d.k_weight : d.q_weight;
  const int64_t position = position_of(d, r);
  float2 z[8];
  float squares = 0;
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const int p = lane + 32 * j;
    if (p >= pairs) break;
    const Pair e = pair_of(p, (int)d.dim, (int)d.turned, (int)d.style);
    z[j] = {to_f32(x[e.u]), to_f32(x[e.v])};
    squares += z[j].x * z[j].x + z[j].y * z[j].y;
  }
  const float scale = rsqrtf(warp_sum(squares) / (float)d.dim + (float)d.epsilon);
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const int p = lane + 32 * j;
    if (p >= pairs) break;
    const Pair e = pair_of(p, (int)d.dim, (int)d.turned, (int)d.style);
    const float2 c = turn_of(d, position, p);
    const float u = z[j].x * scale * (w ? w[e.u] : 1.0f), v = z[j].y * scale * (w ? w[e.v] : 1.0f);
    y[e.u] = from_f32<T>(u * c.x - v * c.y);
    y[e.v] = from_f32<T>(v * c.x + u * c.y);
  }
}

// ---- heads of up to 64 elements, or whose rows, halves and rests are whole 16- or 8-byte vectors
//
// G lanes take a head, each VEC pairs of its elements: a vector of first and a vector of second
// elements (or, turned as adjacent pairs, two vectors in a row).  A warp takes 32 / G heads of one
// token at a time, and UNROLL such sets, with one reading of the token's cosines and sines.
// VEC elements as VEC / 2 pairs of f32, for the packed instructions.
template <typename T, int VEC>
struct Chunk;
template <>
struct Chunk<float, 4> {
  typedef float4 type;
  static __device__ __forceinline__ void read(float4 r, float2 (&v)[2]) {
    v[0] = {r.x, r.y};
    v[1] = {r.z, r.w};
  }
  static __device__ __forceinline__ float4 made(const float2 (&v)[2]) {
    return {v[0].x, v[0].y, v[1].x, v[1].y};
  }
};
template <>
struct Chunk<bf16, 4> {
  typedef uint2 type;
  static __device__ __forceinline__ void read(uint2 r, float2 (&v)[2]) {
    v[0] = unpack_bf16(r.x);
    v[1] = unpack_bf16(r.y);
  }
  static __device__ __forceinline__ uint2 made(const float2 (&v)[2]) {
    return {pack_bf16(v[0]), pack_bf16(v[1])};
  }
};
template <>
struct Chunk<bf16, 8> {
  typedef uint4 type;
  static __device__ __forceinline__ void read(uint4 r, float2 (&v)[4]) {
    v[0] = unpack_bf16(r.x);
    v[1] = unpack_bf16(r.y);
    v[2] = unpack_bf16(r.z);
    v[3] = unpack_bf16(r.w);
  }
  static __device__ __forceinline__ uint4 made(const float2 (&v)[4]) {
    return {pack_bf16(v[0]), pack_bf16(v[1]), pack_bf16(v[2]), pack_bf16(v[3])};
  }
};

// Single elements, for heads whose rows are not aligned: the second of each pair of f32 is unused.
template <typename T>
struct Chunk<T, 1> {
  typedef T type;
  static __device__ __forceinline__ void read(T r, float2 (&v)[1]) { v[0] = {to_f32(r), 0.0f}; }
  static __device__ __forceinline__ T made(const float2 (&v)[1]) { return from_f32<T>(v[0].x); }
};

// A lane's part of a head: where its two vectors lie, and what is common to heads of its side.
template <typename T, int VEC, bool ADJACENT>
struct Part {
  typedef Chunk<T, VEC> C;
  typedef typename C::type Raw;
  static constexpr int N = (VEC + 1) / 2;
  int first, second;  // element offsets
  bool in, turns;
  __device__ Part(const tb_rotate_desc& d, int chunk) {
    const int half = (int)d.turned / 2, p = chunk * VEC;
    in = p < (int)d.dim / 2;
    turns = in && p < half;
    if (ADJACENT) {
      first = 2 * p;
      second = first + VEC;
    } else {
      const Pair e = pair_of(p, (int)d.dim, (int)d.turned, TB_ROTATE_HALVES);
      first = e.u;
      second = e.v;
    }
  }
  // Two vectors as first and second elements of the pairs, and back.
  __device__ __forceinline__ void read(Raw r1, Raw r2, float2 (&u)[N], float2 (&v)[N]) const {
    C::read(r1, u);
    C::read(r2, v);
    if (ADJACENT) apart(u, v);
  }
  __device__ __forceinline__ void made(float2 (&u)[N], float2 (&v)[N], Raw& r1, Raw& r2) const {
    if (ADJACENT) joined(u, v);
    r1 = C::made(u);
    r2 = C::made(v);
  }
  // 0 1 2 3 | 4 5 6 7 -> 0 2 4 6 | 1 3 5 7, and back.
  static __device__ __forceinline__ void apart(float2 (&u)[N], float2 (&v)[N]) {
    if constexpr (VEC > 1) {
      float2 w[2 * N];
#pragma unroll
      for (int j = 0; j < N; ++j) w[j] = u[j], w[N + j] = v[j];
#pragma unroll
      for (int j = 0; j < N; ++j) {
        u[j] = {w[2 * j].x, w[2 * j + 1].x};
        v[j] = {w[2 * j].y, w[2 * j + 1].y};
      }
    }
  }
  static __device__ __forceinline__ void joined(float2 (&u)[N], float2 (&v)[N]) {
    if constexpr (VEC > 1) {
      float2 w[2 * N];
#pragma unroll
      for (int j = 0; j < N; ++j) {
        w[2 * j] = {u[j].x, v[j].x};
        w[2 * j + 1] = {u[j].y, v[j].y};
      }
#pragma unroll
      for (int j = 0; j < N; ++j) u[j] = w[j], v[j] = w[N + j];
    }
  }
  static __device__ __forceinline__ void load(const float* from, float2 (&v)[N]) {
    if constexpr (VEC == 1) {
      v[0] = {from[0], 0.0f};
    } else {
#pragma unroll
      for (int j = 0; j < N; j += 2) {
        [[maybe_unused]] const float4 a = *(const float4*)(from + 2 * j);
        v[j] = {a.x, a.y};
        v[j + 1] = {a.z, a.w};
      }
    }
  }
  __device__ __forceinline__ void angles(const tb_rotate_desc& d, int position, int chunk,
                                         float2 (&cosine)[N], float2 (&sine)[N]) const {
    const bool known = position >= 0 && position < d.table_rows;
#pragma unroll
    for (int j = 0; j < N; ++j) {
      cosine[j] = both(known ? 1.0f : NAN);
      sine[j] = both(known ? 0.0f : NAN);
    }
    if (!turns || !known) return;
    const float* row = d.table + position * d.turned + chunk * VEC;
    load(row, cosine);
    load(row + d.turned / 2, sine);
  }
  __device__ __forceinline__ void weights(const float* w, float2 (&u)[N], float2 (&v)[N]) const {
#pragma unroll
    for (int j = 0; j < N; ++j) u[j] = v[j] = both(1.0f);
    if (!w || !in) return;
    load(w + first, u);
    load(w + second, v);
    if (ADJACENT) apart(u, v);
  }
};
template <int N>
__device__ __forceinline__ float squares_of(const float2 (&u)[N], const float2 (&v)[N]) {
  float2 s = mul2(u[0], u[0]);
#pragma unroll
  for (int j = 1; j < N; ++j) s = fma2(u[j], u[j], s);
#pragma unroll
  for (int j = 0; j < N; ++j) s = fma2(v[j], v[j], s);
  return s.x + s.y;
}
template <int G>
__device__ __forceinline__ float group_sum(float v) {
#pragma unroll
  for (int o = G / 2; o > 0; o >>= 1) v += __shfl_xor_sync(~0u, v, o);
  return v;
}

// One side (queries or keys) of a call.
struct Side {
  const void *in, *grad;
  void* out;
  const float* weight;
  int64_t in_s[3], grad_s[3], out_s[3];
  int heads, blocks;  // blocks: sets of heads that a warp takes of one token
};
struct Sides {
  Side q, k;
  int64_t tokens;
};

// The set of heads that a warp takes in one go: item / blocks is the token, the rest the set.
struct Item {
  unsigned token, b, t;
  int from;  // first head of the set
  __device__ Item(const tb_rotate_desc& d, const Side& side, unsigned item, int heads) {
    token = item / (unsigned)side.blocks;
    from = (int)(item - token * side.blocks) * heads;
    b = token / (unsigned)d.length;
    t = token - b * (unsigned)d.length;
  }
  __device__ __forceinline__ int64_t offset(const int64_t s[3], int head) const {
    return b * s[0] + t * s[1] + head * s[2];
  }
  __device__ __forceinline__ int position(const tb_rotate_desc& d) const {
    return d.positions ? d.positions[token] : (int)t;
  }
};

// Blocks [0, q_blocks) take the query heads, the others the key heads, each warp one item after
// the other: the weights stay in registers, and the next item's position is read an item ahead,
// for the angles wait for it.
template <typename T, int VEC, int G, bool ADJACENT, int UNROLL>
__global__ void __launch_bounds__(256, 3) k_rotate_vectors(tb_rotate_desc d, Sides sides, int q_blocks) {
  pdl_entry();
  typedef Part<T, VEC, ADJACENT> P;
  typedef typename P::Raw Raw;
  constexpr int kRows = 32 / G, kWarps = 8, N = (VEC + 1) / 2;
  const int lane = threadIdx.x % 32, warp = threadIdx.x / 32, chunk = lane % G;
  const bool key = (int)blockIdx.x >= q_blocks;
  const Side& side = key ? sides.k : sides.q;
  const int of = key ? gridDim.x - q_blocks : q_blocks, mine = key ? blockIdx.x - q_blocks : blockIdx.x;
  const P part(d, chunk);
  const float share = 1.0f / (float)d.dim, epsilon = (float)d.epsilon;
  const unsigned items = (unsigned)sides.tokens * side.blocks;
  unsigned i = mine * kWarps + warp;
  if (i >= items) return;
  int position = Item(d, side, i, kRows * UNROLL).position(d);
  float2 wu[N], wv[N];
  part.weights(side.weight, wu, wv);
  for (; i < items; i += of * kWarps) {
    const Item item(d, side, i, kRows * UNROLL);
    const int head0 = item.from + lane / G;
    const T* x = (const T*)side.in + item.offset(side.in_s, head0);
    T* y = (T*)side.out + item.offset(side.out_s, head0);
    Raw r1[UNROLL], r2[UNROLL];
#pragma unroll
    for (int h = 0; h < UNROLL; ++h) {
      r1[h] = r2[h] = Raw{};
      if (part.in && head0 + h * kRows < side.heads) {
        const T* row = x + h * kRows * side.in_s[2];
        r1[h] = *(const Raw*)(row + part.first);
        r2[h] = *(const Raw*)(row + part.second);
      }
    }
    float2 cosine[N], sine[N];
    part.angles(d, position, chunk, cosine, sine);
    if (i + of * kWarps < items) position = Item(d, side, i + of * kWarps, kRows * UNROLL).position(d);
#pragma unroll
    for (int h = 0; h < UNROLL; ++h) {
      if (item.from + h * kRows >= side.heads) break;
      float2 u[N], v[N];
      part.read(r1[h], r2[h], u, v);
      const float scale = rsqrtf(group_sum<G>(squares_of(u, v)) * share + epsilon);
#pragma unroll
      for (int j = 0; j < N; ++j) {
        const float2 p = mul2(mul2(u[j], both(scale)), wu[j]), q = mul2(mul2(v[j], both(scale)), wv[j]);
        u[j] = fma2(p, cosine[j], mul2(mul2(q, both(-1.0f)), sine[j]));
        v[j] = fma2(q, cosine[j], mul2(p, sine[j]));
      }
      if (part.in && head0 + h * kRows < side.heads) {
        Raw o1, o2;
        part.made(u, v, o1, o2);
        T* row = y + h * kRows * side.out_s[2];
        *(Raw*)(row + part.first) = o1;
        *(Raw*)(row + part.second) = o2;
      }
    }
  }
}

constexpr int64_t kBackwardBlocks = 2 * 148;  // of each side, at most: rows of partials

// A lane's copy of one vector into its own place in shared memory.
template <typename Raw>
__device__ __forceinline__ void copy_own(Raw* to, const Raw* from) {
  if constexpr (sizeof(Raw) == 16)
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"((unsigned)__cvta_generic_to_shared(to)), "l"(from)
                 : "memory");
  else if constexpr (sizeof(Raw) >= 4)
    asm volatile("cp.async.ca.shared.global [%0], [%1], %2;" ::"r"((unsigned)__cvta_generic_to_shared(to)),
                 "l"(from), "n"((int)sizeof(Raw))
                 : "memory");
  else
    *to = *from;
}

// The same division of work; a lane holds its part of the weight gradient in registers.  That and the
// two rows of every head leave sixteen warps to a SM, too few to wait for their rows by turns, so
// where a lane holds 8 elements of a vector it copies those of its next items into its own places in
// shared memory (40 heads of 128 in bf16: 56 us without, 49 with; 24 heads of 64 in f32, where four
// sets fit the registers: 31 without, 45 with).
constexpr int kCopies = 3;  // items a lane has under way
template <int VEC>
constexpr bool kCopied = VEC == 8;
// Shared memory of a block: the places, then (or alone) its warps' sums of the weight gradient.
template <typename Raw, int VEC, int G, int UNROLL>
constexpr size_t kBackwardBytes = kCopied<VEC> ? (size_t)kCopies * UNROLL * 4 * 256 * sizeof(Raw)
                                               : (size_t)8 * 2 * ((VEC + 1) / 2) * G * sizeof(float2);
template <typename T, int VEC, int G, bool ADJACENT, int UNROLL>
__global__ void __launch_bounds__(256, 2) k_rotate_vectors_backward(tb_rotate_desc d, Sides sides,
                                                                    int q_blocks) {
  pdl_entry();
  typedef Part<T, VEC, ADJACENT> P;
  typedef typename P::Raw Raw;
  constexpr int kRows = 32 / G, kWarps = 8, N = (VEC + 1) / 2;
  const int lane = threadIdx.x % 32, warp = threadIdx.x / 32, chunk = lane % G;
  const bool key = (int)blockIdx.x >= q_blocks;
  const Side& side = key ? sides.k : sides.q;
  const int of = key ? gridDim.x - q_blocks : q_blocks, mine = key ? blockIdx.x - q_blocks : blockIdx.x;
  const P part(d, chunk);
  const float share = 1.0f / (float)d.dim, epsilon = (float)d.epsilon;
  float2 wu[N], wv[N], du[N], dv[N];
  part.weights(side.weight, wu, wv);
#pragma unroll
  for (int j = 0; j < N; ++j) du[j] = dv[j] = both(0.0f);
  const unsigned items = (unsigned)sides.tokens * side.blocks;
  extern __shared__ uint4 places[];
  [[maybe_unused]] const auto place = [&](int copy, int h, int which) -> Raw& {
    return ((Raw*)places)[((copy * UNROLL + h) * 4 + which) * 256 + threadIdx.x];
  };
  const unsigned step = of * kWarps;
  [[maybe_unused]] const auto fetch = [&](int copy, unsigned at) {
    if (at < items) {
      const Item item(d, side, at, kRows * UNROLL);
      const int head0 = item.from + lane / G;
      const T* x = (const T*)side.in + item.offset(side.in_s, head0);
      const T* dy = (const T*)side.grad + item.offset(side.grad_s, head0);
#pragma unroll
      for (int h = 0; h < UNROLL; ++h)
        if (part.in && head0 + h * kRows < side.heads) {
          const T *row = x + h * kRows * side.in_s[2], *grad = dy + h * kRows * side.grad_s[2];
          copy_own(&place(copy, h, 0), (const Raw*)(row + part.first));
          copy_own(&place(copy, h, 1), (const Raw*)(row + part.second));
          copy_own(&place(copy, h, 2), (const Raw*)(grad + part.first));
          copy_own(&place(copy, h, 3), (const Raw*)(grad + part.second));
        }
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
  unsigned i = mine * kWarps + warp;
  if constexpr (kCopied<VEC>)
#pragma unroll
    for (int copy = 0; copy < kCopies - 1; ++copy) fetch(copy, i + copy * step);
  int position = i < items ? Item(d, side, i, kRows * UNROLL).position(d) : 0;
  int now = 0;
  for (; i < items; i += step) {
    const Item item(d, side, i, kRows * UNROLL);
    const int from = item.from, head0 = from + lane / G;
    Raw held[kCopied<VEC> ? 1 : UNROLL][4];
    if constexpr (kCopied<VEC>) {
      fetch(now == 0 ? kCopies - 1 : now - 1, i + (kCopies - 1) * step);
    } else {
      const T* x = (const T*)side.in + item.offset(side.in_s, head0);
      const T* dy = (const T*)side.grad + item.offset(side.grad_s, head0);
#pragma unroll
      for (int h = 0; h < UNROLL; ++h) {
        held[h][0] = held[h][1] = held[h][2] = held[h][3] = Raw{};
        if (part.in && head0 + h * kRows < side.heads) {
          const T *row = x + h * kRows * side.in_s[2], *grad = dy + h * kRows * side.grad_s[2];
          held[h][0] = *(const Raw*)(row + part.first);
          held[h][1] = *(const Raw*)(row + part.second);
          held[h][2] = *(const Raw*)(grad + part.first);
          held[h][3] = *(const Raw*)(grad + part.second);
        }
      }
    }
    T* dx = (T*)side.out + item.offset(side.out_s, head0);
    float2 cosine[N], sine[N];
    part.angles(d, position, chunk, cosine, sine);
    if (i + step < items) position = Item(d, side, i + step, kRows * UNROLL).position(d);
    if constexpr (kCopied<VEC>) asm volatile("cp.async.wait_group %0;" ::"n"(kCopies - 1) : "memory");
#pragma unroll
    for (int h = 0; h < UNROLL; ++h) {
      if (from + h * kRows >= side.heads) break;
      const bool here = part.in && head0 + h * kRows < side.heads;
      float2 u[N], v[N], gu[N], gv[N];
      Raw raw[4] = {};
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        if constexpr (!kCopied<VEC>) raw[w] = held[h][w];
        else if (here) raw[w] = place(now, h, w);
      }
      part.read(raw[0], raw[1], u, v);
      part.read(raw[2], raw[3], gu, gv);
      const float scale = rsqrtf(group_sum<G>(squares_of(u, v)) * share + epsilon);
      float2 inner = both(0.0f);
#pragma unroll
      for (int j = 0; j < N; ++j) {
        const float2 p = fma2(gu[j], cosine[j], mul2(gv[j], sine[j]));
        const float2 q = fma2(gv[j], cosine[j], mul2(mul2(gu[j], both(-1.0f)), sine[j]));
        u[j] = mul2(u[j], both(scale));
        v[j] = mul2(v[j], both(scale));
        if (here) {
          du[j] = fma2(p, u[j], du[j]);
          dv[j] = fma2(q, v[j], dv[j]);
        }
        gu[j] = mul2(p, wu[j]);
        gv[j] = mul2(q, wv[j]);
        inner = fma2(gu[j], u[j], fma2(gv[j], v[j], inner));
      }
      const float mean = group_sum<G>(part.in ? inner.x + inner.y : 0.0f) * share;
#pragma unroll
      for (int j = 0; j < N; ++j) {
        u[j] = mul2(both(scale), fma2(u[j], both(-mean), gu[j]));
        v[j] = mul2(both(scale), fma2(v[j], both(-mean), gv[j]));
      }
      if (here) {
        Raw o1, o2;
        part.made(u, v, o1, o2);
        T* row = dx + h * kRows * side.out_s[2];
        *(Raw*)(row + part.first) = o1;
        *(Raw*)(row + part.second) = o2;
      }
    }
    now = now + 1 == kCopies ? 0 : now + 1;
  }
  if (!d.workspace) return;
  // lanes of one chunk, then the warps, in a fixed order; the elements in their places
#pragma unroll
  for (int j = 0; j < N; ++j) {
#pragma unroll
    for (int o = 16; o >= G; o >>= 1) {
      du[j] = add2(du[j], {__shfl_xor_sync(~0u, du[j].x, o), __shfl_xor_sync(~0u, du[j].y, o)});
      dv[j] = add2(dv[j], {__shfl_xor_sync(~0u, dv[j].x, o), __shfl_xor_sync(~0u, dv[j].y, o)});
    }
  }
  if (ADJACENT) P::joined(du, dv);
  typedef float2 Sums[2 * N][G];
  Sums* sums = (Sums*)places;  // [warps], where the copies were
  static_assert(kWarps * sizeof(Sums) <= kBackwardBytes<Raw, VEC, G, UNROLL>);
  __syncthreads();
  if (lane < G)
#pragma unroll
    for (int j = 0; j < N; ++j) {
      sums[warp][j][chunk] = du[j];
      sums[warp][N + j][chunk] = dv[j];
    }
  __syncthreads();
  for (int i = threadIdx.x; i < 2 * N * G; i += 256) {
    const int j = i / G, c = i % G;
    const P at(d, c);
    if (!at.in) continue;
    float2 s = sums[0][j][c];
#pragma unroll
    for (int w = 1; w < kWarps; ++w) s = add2(s, sums[w][j][c]);
    float* to = (float*)d.workspace + (int64_t)blockIdx.x * d.dim;
    to += j < N ? at.first + 2 * j : at.second + 2 * (j - N);
    if constexpr (VEC == 1) *to = s.x;
    else *(float2*)to = s;
  }
}

// Weight gradients: the blocks' partials in a fixed order, 32 threads an element.
__global__ void __launch_bounds__(1024) k_rotate_weights(tb_rotate_desc d, int q_blocks, int blocks) {
  pdl_entry();
  __shared__ float sums[32][33];
  const int dim = (int)d.dim, per_side = (dim + 31) / 32, lane = threadIdx.x % 32, row = threadIdx.x / 32;
  const bool key = (int)blockIdx.x >= per_side;
  const int first = (blockIdx.x - (key ? per_side : 0)) * 32, j = first + lane;
  const int from = key ? q_blocks : 0, to = key ? blocks : q_blocks;
  float s = 0;
  if (j < dim)
#pragma unroll 8
    for (int b = from + row; b < to; b += 32) s += ((const float*)d.workspace)[(int64_t)b * dim + j];
  sums[row][lane] = s;
  __syncthreads();
  s = warp_sum(sums[lane][row]);  // element `row` of this block's 32
  float* out = key ? d.dk_weight : d.dq_weight;
  if (lane == 0 && first + row < dim && out) out[first + row] = s;
}

// ---- any other head: a warp each

template <typename T>
__global__ void k_rotate_backward(tb_rotate_desc d, int64_t rows) {
  pdl_entry();
  extern __shared__ float sums[];  // [warps][2][dim]
  const int lane = threadIdx.x % 32, warp = threadIdx.x / 32, warps = blockDim.x / 32;
  const int pairs = (int)d.dim / 2, dim = (int)d.dim;
  float* mine = sums + warp * 2 * dim;
  for (int j = lane; j < 2 * dim; j += 32) mine[j] = 0;
  __syncwarp();
  for (int64_t i = (int64_t)blockIdx.x * warps + warp; i < rows; i += (int64_t)gridDim.x * warps) {
    const Row r = row_of(d, i);
    const T* x = at<T>(r.key ? d.k : d.q, r.key ? d.k_strides : d.q_strides, r);
    const T* dy = at<T>(r.key ? d.dk : d.dq, r.key ? d.dk_strides : d.dq_strides, r);
    T* dx = at<T>(r.key ? d.k_out : d.q_out, r.key ? d.k_out_strides : d.q_out_strides, r);
    const float* w = r.key ? d.k_weight : d.q_weight;
    const int64_t position = position_of(d, r);
    float2 z[8], g[8];
    float squares = 0;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const int p = lane + 32 * j;
      if (p >= pairs) break;
      const Pair e = pair_of(p, dim, (int)d.turned, (int)d.style);
      z[j] = {to_f32(x[e.u]), to_f32(x[e.v])};
      squares += z[j].x * z[j].x + z[j].y * z[j].y;
      const float2 c = turn_of(d, position, p);
      const float u = to_f32(dy[e.u]), v = to_f32(dy[e.v]);
      g[j] = {u * c.x + v * c.y, v * c.x - u * c.y};
    }
    const float scale = rsqrtf(warp_sum(squares) / (float)dim + (float)d.epsilon);
    float inner = 0;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const int p = lane + 32 * j;
      if (p >= pairs) break;
      const Pair e = pair_of(p, dim, (int)d.turned, (int)d.style);
      z[j].x *= scale;
      z[j].y *= scale;
      float* to = mine + (r.key ? dim : 0);
      to[e.u] += g[j].x * z[j].x;
      to[e.v] += g[j].y * z[j].y;
      g[j].x *= w ? w[e.u] : 1.0f;
      g[j].y *= w ? w[e.v] : 1.0f;
      inner += g[j].x * z[j].x + g[j].y * z[j].y;
    }
    inner = warp_sum(inner) / (float)dim;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const int p = lane + 32 * j;
      if (p >= pairs) break;
      const Pair e = pair_of(p, dim, (int)d.turned, (int)d.style);
      dx[e.u] = from_f32<T>(scale * (g[j].x - z[j].x * inner));
      dx[e.v] = from_f32<T>(scale * (g[j].y - z[j].y * inner));
    }
  }
  if (!d.workspace) return;
  __syncthreads();
  for (int j = threadIdx.x; j < 2 * dim; j += blockDim.x) {
    float s = 0;
    for (int w = 0; w < warps; ++w) s += sums[w * 2 * dim + j];
    // all query rows of partials, then all key rows
    const int64_t row = blockIdx.x + (j < dim ? 0 : gridDim.x);
    ((float*)d.workspace)[row * dim + (j < dim ? j : j - dim)] = s;
  }
}

int64_t workspace_bytes(const tb_rotate_desc& d) {
  return d.dq_weight || d.dk_weight ? tb_head_rotate_workspace(d.dim) : 0;
}

bool strides_ok(const tb_rotate_desc& d, const int64_t s[3], int64_t heads, bool written) {
  if (!extents_fit({s[0]}) || !extents_fit({s[1]}) || !extents_fit({s[2]})) return false;
  return !written || rows_apart<3>(d.dim, {d.batch, d.length, heads}, {s[0], s[1], s[2]});
}

const char* check(const tb_rotate_desc& d, bool backward) {
  if (d.element != TB_ELEMENT_F32 && d.element != TB_ELEMENT_BF16) return "unknown element type";
  if (d.style != TB_ROTATE_HALVES && d.style != TB_ROTATE_PAIRS) return "unknown style";
  if (!extents_fit({d.batch, d.length, d.q_heads, d.dim}) || d.length > INT32_MAX ||
      !extents_fit({d.batch, d.length, d.k_heads, d.dim}) || !extents_fit({d.table_rows, d.turned}) ||
      d.batch * d.length * (d.q_heads + d.k_heads) > INT32_MAX)
    return "extents out of range";
  if (d.dim < 2 || d.dim > 512 || d.dim % 2) return "dim is even and at most 512";
  if (d.turned < 0 || d.turned > d.dim || d.turned % 2) return "turned is even and at most dim";
  if (!(d.epsilon >= 0) || d.epsilon > 3e38) return "epsilon is finite and not negative";
  const int64_t tokens = d.batch * d.length, size = d.element == TB_ELEMENT_F32 ? 4 : 2;
  if (tokens > 0 && d.q_heads + d.k_heads > 0 && d.turned > 0 && !d.table) return "no table";
  const struct {
    int64_t heads;
    const void *in, *grad, *out;
    const int64_t *in_strides, *grad_strides, *out_strides;
  } sides[2] = {{d.q_heads, d.q, d.dq, d.q_out, d.q_strides, d.dq_strides, d.q_out_strides},
                {d.k_heads, d.k, d.dk, d.k_out, d.k_strides, d.dk_strides, d.k_out_strides}};
  for (const auto& s : sides) {
    if (tokens * s.heads == 0) continue;
    if (!s.in || !s.out || (backward && !s.grad)) return "a required array is NULL";
    if (!aligned_to(s.in, size) || !aligned_to(s.out, size) || (backward && !aligned_to(s.grad, size)))
      return "an array is not aligned to its elements";
    if (!strides_ok(d, s.in_strides, s.heads, false) || !strides_ok(d, s.out_strides, s.heads, true) ||
        (backward && !strides_ok(d, s.grad_strides, s.heads, false)))
      return "strides are negative, too large, or let written heads overlap";
  }
  for (const void* p : {(const void*)d.table, (const void*)d.positions, (const void*)d.q_weight,
                        (const void*)d.k_weight, (const void*)d.dq_weight, (const void*)d.dk_weight})
    if (!aligned_to(p, 4)) return "an array is not aligned to its elements";
  if (backward && workspace_bytes(d) > 0) {
    if (!d.workspace || d.workspace_bytes < workspace_bytes(d)) return "the workspace is too small";
    if (!aligned_to(d.workspace, 16)) return "the workspace is not 16-byte aligned";
  }
  return nullptr;
}

// Whether a side's heads are made of whole vectors of VEC elements.
template <typename T, int VEC>
bool vectors_fit(const tb_rotate_desc& d, const Side& side, bool backward) {
  const auto fits = [&](const void* p, const int64_t s[3]) {
    return aligned_to(p, VEC * sizeof(T)) && (d.batch <= 1 || s[0] % VEC == 0) &&
           (d.length <= 1 || s[1] % VEC == 0) && (side.heads <= 1 || s[2] % VEC == 0);
  };
  return side.heads == 0 || (fits(side.in, side.in_s) && fits(side.out, side.out_s) &&
                             (!backward || fits(side.grad, side.grad_s)) &&
                              aligned_to(side.weight, VEC == 1 ? 4 : 16));
}
template <typename T, int VEC>
bool vectors_fit(const tb_rotate_desc& d, const Sides& sides, bool backward) {
  return d.turned / 2 % VEC == 0 && (d.dim - d.turned) / 2 % VEC == 0 && d.dim / 2 / VEC <= 32 &&
         aligned_to(d.table, VEC == 1 ? 4 : 16) && vectors_fit<T, VEC>(d, sides.q, backward) &&
         vectors_fit<T, VEC>(d, sides.k, backward);
}

cudaError_t enqueue_weights(const tb_rotate_desc& d, int64_t q_blocks, int64_t blocks, cudaStream_t stream) {
  return launch_pdl(k_rotate_weights, dim3((unsigned)(2 * ((d.dim + 31) / 32))), dim3(1024), 0, stream,
                    d, (int)q_blocks, (int)blocks);
}

template <typename T, int VEC, int G, bool ADJACENT>
cudaError_t enqueue_vectors(const tb_rotate_desc& d, Sides sides, bool backward, cudaStream_t stream) {
  // sets of heads a warp takes in one go: as many loads as its registers or places hold
  constexpr int kUnroll = VEC == 8 ? 2 : 4;
  const int kHeads = 32 / G * kUnroll;
  sides.q.blocks = (sides.q.heads + kHeads - 1) / kHeads;
  sides.k.blocks = (sides.k.heads + kHeads - 1) / kHeads;
  const int64_t q_items = sides.tokens * sides.q.blocks, k_items = sides.tokens * sides.k.blocks;
  // as many blocks as run at once, shared out by the sides' work
  const int64_t most = (backward ? 2 : 3) * 148;
  int64_t q_blocks = q_items ? std::max<int64_t>(1, most * q_items / (q_items + k_items)) : 0;
  int64_t k_blocks = k_items ? std::max<int64_t>(1, most - q_blocks) : 0;
  q_blocks = std::min(q_blocks, (q_items + 7) / 8);
  k_blocks = std::min(k_blocks, (k_items + 7) / 8);
  if (!backward)
    return launch_pdl(k_rotate_vectors<T, VEC, G, ADJACENT, kUnroll>,
                      dim3((unsigned)(q_blocks + k_blocks)), dim3(256), 0, stream, d, sides, (int)q_blocks);
  constexpr size_t kShared = kBackwardBytes<typename Chunk<T, VEC>::type, VEC, G, kUnroll>;
  const auto kernel = k_rotate_vectors_backward<T, VEC, G, ADJACENT, kUnroll>;
  static std::atomic<uint64_t> allowed{0};  // devices on which the kernel may use that much
  cudaError_t e = allow_shared((const void*)kernel, kShared, allowed);
  if (e == cudaSuccess)
    e = launch_pdl(kernel, dim3((unsigned)(q_blocks + k_blocks)), dim3(256), kShared, stream, d, sides,
                   (int)q_blocks);
  return e == cudaSuccess && d.workspace ? enqueue_weights(d, q_blocks, q_blocks + k_blocks, stream) : e;
}

template <typename T, int VEC>
cudaError_t enqueue_vectors(const tb_rotate_desc& d, const Sides& sides, bool backward, cudaStream_t stream) {
  const int64_t chunks = d.dim / 2 / VEC;
  const bool adjacent = d.style == TB_ROTATE_PAIRS;
#define TB_ROTATE_GROUP(G)                                                                   \
  if (chunks <= G)                                                                           \
    return adjacent ? enqueue_vectors<T, VEC, G, true>(d, sides, backward, stream)           \
                    : enqueue_vectors<T, VEC, G, false>(d, sides, backward, stream);
  TB_ROTATE_GROUP(4)
  TB_ROTATE_GROUP(8)
  TB_ROTATE_GROUP(16)
  TB_ROTATE_GROUP(32)
#undef TB_ROTATE_GROUP
  return cudaErrorInvalidValue;
}

template <typename T>
cudaError_t enqueue(tb_rotate_desc d, bool backward, cudaStream_t stream) {
  const int64_t tokens = d.batch * d.length, rows = tokens * (d.q_heads + d.k_heads);
  if (!backward || !workspace_bytes(d)) d.workspace = nullptr;
  if (rows == 0) return d.workspace ? enqueue_weights(d, 0, 0, stream) : cudaSuccess;
  Sides sides = {};
  sides.tokens = tokens;
  const auto side = [](Side& s, const void* in, const void* grad, void* out, const float* weight,
                       const int64_t* in_s, const int64_t* grad_s, const int64_t* out_s, int64_t heads) {
    s.in = in;
    s.grad = grad;
    s.out = out;
    s.weight = weight;
    std::copy(in_s, in_s + 3, s.in_s);
    std::copy(grad_s, grad_s + 3, s.grad_s);
    std::copy(out_s, out_s + 3, s.out_s);
    s.heads = (int)heads;
  };
  side(sides.q, d.q, d.dq, d.q_out, d.q_weight, d.q_strides, d.dq_strides, d.q_out_strides, d.q_heads);
  side(sides.k, d.k, d.dk, d.k_out, d.k_weight, d.k_strides, d.dk_strides, d.k_out_strides, d.k_heads);
  constexpr int kVec = 16 / sizeof(T), kHalf = kVec == 8 ? 4 : kVec;
  // Small bf16 heads spread over twice the lanes, with fewer registers each: 8 x 1024 tokens x 24 heads
  // of 64 backwards 21.8 us in 8-byte lanes and 24.7 in 16-byte ones (of 96: 41.5 and 39.7), x 32
  // heads of 32 forwards 10.5 and 12.2 (24 of 64: 13.5 and 13.4).
  const bool spread = kVec == 8 && d.dim <= (backward ? 64 : 32) && vectors_fit<T, kHalf>(d, sides, backward);
  if (!spread && vectors_fit<T, kVec>(d, sides, backward))
    return enqueue_vectors<T, kVec>(d, sides, backward, stream);
  if constexpr (kVec == 8)
    if (vectors_fit<T, 4>(d, sides, backward)) return enqueue_vectors<T, 4>(d, sides, backward, stream);
  if (vectors_fit<T, 1>(d, sides, backward)) return enqueue_vectors<T, 1>(d, sides, backward, stream);
  if (!backward) {
    const int64_t blocks = (rows + 7) / 8;
    return launch_pdl(k_rotate<T>, dim3((unsigned)blocks), dim3(256), 0, stream, d, rows);
  }
  const cudaError_t e = launch_pdl(k_rotate_backward<T>, dim3(kBackwardBlocks), dim3(256),
                                   (size_t)8 * 2 * d.dim * 4, stream, d, rows);
  return e == cudaSuccess && d.workspace ? enqueue_weights(d, kBackwardBlocks, 2 * kBackwardBlocks, stream) : e;
}

int rotate_call(const char* name, const tb_rotate_desc* desc, void* stream, bool backward) {
  OperatorCall call(name, stream);
  if (!desc) return call.invalid("no request");
  const tb_rotate_desc d = *desc;
  if (const char* why = check(d, backward)) return call.invalid(why);
  if (const int code = call.ready()) return code;
  return call.finish(d.element == TB_ELEMENT_F32 ? enqueue<float>(d, backward, call.stream())
                                                 : enqueue<bf16>(d, backward, call.stream()));
}

}  // namespace
}  // namespace tb

extern "C" int tb_head_rotate(const tb_rotate_desc* desc, void* stream) {
  return tb::guarded([&] { return tb::rotate_call("tb_head_rotate", desc, stream, false); });
}
extern "C" int tb_head_rotate_backward(const tb_rotate_desc* desc, void* stream) {
  return tb::guarded([&] { return tb::rotate_call("tb_head_rotate_backward", desc, stream, true); });
}
extern "C" int64_t tb_head_rotate_workspace(int64_t dim) {
  return dim > 0 && dim <= 512 ? tb::kBackwardBlocks * 2 * dim * 4 : 0;
}
