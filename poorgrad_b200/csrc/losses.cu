// losses.cu -- log probabilities of tokens, the clipped policy loss and the paired log-ratio
// loss over a vocabulary, with their gradients by the logits.
//
// With p = softmax(scale z) and L = scale z_t - lse, every loss reaches the logits through L
// alone: dz_v = c scale (1[v = t] - p_v) with c = d loss / d L of the row.  Maxima are taken of
// the raw logits and scale multiplies differences from them, so masks of the type's lowest
// value do not overflow.  The statistics of a row are a running maximum and sum of exponentials.
//
// Measured on B200 (against a copy's 6.55 TB/s): the policy loss with its gradient over 8192 x 50257
// logits, a quarter of the rows hidden, f32 485 us, 5.9 TB/s, bf16 280 us, 5.1 TB/s; the loss
// alone f32 182 us, bf16 103 us, 6.0 TB/s.  Memory bounds the f32 forms (under load the power cap too:
// up to 540 us in a long run), issue slots and the two exponentials a logit the bf16 ones.  Rows that
// leave a thread two or three vectors are furthest from that (8192 x 4099 bf16 43 us, 3.1 TB/s): sums that
// are carried over exactly cost them most (36 us before; 3000 x 130000 f32 477 and 522), and where a
// group of a thread's vectors is odd its last one goes with one that is not there, at a whole vector's
// exponentials.  The longer bf16 rows that are only read gained (123 -> 103).  The preference loss cannot
// know a row's slope before its pair's last row.  It takes all rows' statistics before any gradient, so the
// logits are read twice: 4099 x 50257 bf16 in 184 us, 988 MB at 5.4 TB/s.
#include <cooperative_groups.h>

#include <algorithm>

#include "operators.h"

namespace tb {
namespace {

namespace cg = cooperative_groups;

constexpr float kLog2e = 1.4426950408889634f;

__device__ __forceinline__ float ex2(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}

// A row's statistics, with k = scale log2(e): top, the largest z, and sum, that of 2^(k (z - top) - f).
// f, from 1 to 2, lifts k top to a whole number m, so that a sum is carried over to another top by a
// factor 2^(m - m'), which is exact: ex2 is low by 5e-8 on average (measured below -1), and a sum that
// went through it once for its terms and two or three times more for its tops made all log
// probabilities of an answer too large, by 7e-8 to 1.6e-7.  The once is undone by the top's own term,
// 2^-f, which is as low: it is what the sum is divided by in the end, and a row of one likely token comes
// out right to the last bit.  Where k top is past 2^21, f is 0 and the factors are rounded.
// A sum of 0: no logit above -inf.
// An exponential's argument is one rounded sum, so a term d below the top has a relative error of about
// 2^-25 d besides the instruction's own (7e-7 at 24 below, where expf would leave 5e-8), and below 2^-126
// it is 0.  Such terms weigh that little in the sums; in the gradient of an f32 row they stand alone, and
// two more instructions a logit would be needed there.
struct RowStats {
  float top, sum;
};
// What differences are taken from: -inf would make NaN of -inf logits, and any finite number does.
__device__ __forceinline__ float base_of(float top) { return top == -INFINITY ? 0.0f : top; }
__device__ __forceinline__ float lift_of(float top, float k) {
  const float at = k * top;
  return fabsf(at) < 2097152.0f ? fmaf(-k, top, ceilf(at) + 1.0f) : 0.0f;
}
// The factor that carries a sum over from a top to one that is `less` below it, with their f's.  m - m' is
// whole but for this line's rounding.
__device__ __forceinline__ float carry(float less, float from, float to, float k) {
  const float power = fmaf(k, less, from - to);
  return ex2(from * to != 0.0f ? rintf(power) : power);
}

// 16 bytes of a row.
template <typename T>
struct Vector;
template <>
struct Vector<float> {
  static constexpr int kPairs = 2;
  static __device__ __forceinline__ uint4 nothing() { return {0xff800000u, 0xff800000u, 0xff800000u, 0xff800000u}; }
  static __device__ __forceinline__ void read(uint4 r, float2 (&v)[2]) {
    v[0] = {__uint_as_float(r.x), __uint_as_float(r.y)};
    v[1] = {__uint_as_float(r.z), __uint_as_float(r.w)};
  }
  static __device__ __forceinline__ float top(uint4 r) {
    return fmaxf(fmaxf(__uint_as_float(r.x), __uint_as_float(r.y)),
                 fmaxf(__uint_as_float(r.z), __uint_as_float(r.w)));
  }
  static __device__ __forceinline__ uint4 made(const float2 (&v)[2]) {
    return {__float_as_uint(v[0].x), __float_as_uint(v[0].y), __float_as_uint(v[1].x),
            __float_as_uint(v[1].y)};
  }
};
template <>
struct Vector<bf16> {
  static constexpr int kPairs = 4;
  static __device__ __forceinline__ uint4 nothing() { return {0xff80ff80u, 0xff80ff80u, 0xff80ff80u, 0xff80ff80u}; }
  static __device__ __forceinline__ void read(uint4 r, float2 (&v)[4]) {
    v[0] = unpack_bf16(r.x);
    v[1] = unpack_bf16(r.y);
    v[2] = unpack_bf16(r.z);
    v[3] = unpack_bf16(r.w);
  }
  static __device__ __forceinline__ unsigned top(unsigned a, unsigned b) {  // of each half; NaN last
    unsigned r;
    asm("max.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    return r;
  }
  static __device__ __forceinline__ float top(uint4 r) {
    const float2 t = unpack_bf16(top(top(r.x, r.y), top(r.z, r.w)));
    return fmaxf(t.x, t.y);
  }
  static __device__ __forceinline__ uint4 made(const float2 (&v)[4]) {
    return {pack_bf16(v[0]), pack_bf16(v[1]), pack_bf16(v[2]), pack_bf16(v[3])};
  }
};

// A thread's statistics, and its top's f.
struct ThreadStats {
  RowStats s{-INFINITY, 0.0f};
  float base = 0.0f, lift = 0.0f;
  __device__ __forceinline__ void raise(float top, float k) {
    if (top > s.top) {
      const float to = lift_of(top, k);
      s.sum *= carry(s.top - top, lift, to, k);
      s.top = base = top;
      lift = to;
    }
  }
};
// Adds COUNT vectors: one rescaling for all of them.
template <typename T, int COUNT>
__device__ __forceinline__ void add(ThreadStats& of, const uint4 (&r)[COUNT], float k) {
  typedef Vector<T> Vec;
  float top = Vec::top(r[0]);
#pragma unroll
  for (int j = 1; j < COUNT; ++j) top = fmaxf(top, Vec::top(r[j]));
  of.raise(top, k);
  const float2 minus = both(-of.base), lift = both(-of.lift);
  float2 sum = both(0.0f);
#pragma unroll
  for (int j = 0; j < COUNT; ++j) {
    float2 v[Vec::kPairs];
    Vec::read(r[j], v);
#pragma unroll
    for (int i = 0; i < Vec::kPairs; ++i) {
      const float2 x = fma2(add2(v[i], minus), both(k), lift);
      sum = add2(sum, {ex2(x.x), ex2(x.y)});
    }
  }
  of.s.sum += sum.x + sum.y;
}
__device__ __forceinline__ void add(ThreadStats& of, float z, float k) {
  of.raise(z, k);
  of.s.sum += ex2(fmaf(z - of.base, k, -of.lift));
}

// A row as single elements up to a 16-byte boundary, vectors, and single elements again; the
// vectors and single elements of one block of `ranks` that share the row.
template <typename T>
struct RowShare {
  static constexpr int kVec = 16 / sizeof(T);
  int64_t first, count;  // this block's vectors, counted from the boundary
  int64_t head;          // elements before the boundary
  int64_t single;        // this thread's single element, or -1
  __device__ RowShare(const T* z, int64_t vocab, int rank, int ranks, int64_t per) {
    head = min((int64_t)((16 - ((uintptr_t)z & 15)) & 15) / (int64_t)sizeof(T), vocab);
    const int64_t vectors = (vocab - head) / kVec, tail = head + vectors * kVec;
    first = min(rank * per, vectors);
    count = min(per, vectors - first);
    // threads 0 .. 7 of the first block take the head's elements, 8 .. 15 of the last the tail's
    single = -1;
    if (rank == 0 && threadIdx.x < 8 && threadIdx.x < head) single = threadIdx.x;
    if (rank == ranks - 1 && threadIdx.x >= 8 && threadIdx.x < 16 && tail + threadIdx.x - 8 < vocab)
      single = tail + threadIdx.x - 8;
  }
  __device__ __forceinline__ int64_t element(int64_t vector) const { return head + (first + vector) * kVec; }
};

// A NaN logit makes the sum NaN (the maximum passes it over, the exponential does not), and so does
// +inf, by inf - inf.
__device__ __forceinline__ RowStats warp_stats(RowStats s, float k, int lanes = 32) {
  float top = s.top;
  for (int o = lanes / 2; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(~0u, top, o));
  const float base = base_of(top);
  s.sum *= carry(s.top - base, lift_of(s.top, k), lift_of(base, k), k);
  s.top = top;
  for (int o = lanes / 2; o > 0; o >>= 1) s.sum += __shfl_xor_sync(~0u, s.sum, o);
  return s;
}
// The statistics of all threads, in a fixed order; the first warp gets them (what follows is one
// thread's work, and on small blocks a good part of all if every thread does it).
template <int THREADS>
__device__ __forceinline__ RowStats block_stats(RowStats s, float k) {
  __shared__ RowStats part[THREADS / 32];
  s = warp_stats(s, k);
  if (threadIdx.x % 32 == 0) part[threadIdx.x / 32] = s;
  __syncthreads();
  return threadIdx.x < 32 ? warp_stats(part[threadIdx.x % (THREADS / 32)], k, THREADS / 32) : s;
}

// Statistics of a row straight from memory, for the first warp.
template <typename T, int THREADS>
__device__ __forceinline__ RowStats row_stats(const T* z, int64_t vocab, float k) {
  constexpr int kAtOnce = 4;
  const RowShare<T> row(z, vocab, 0, 1, INT64_MAX / 2);
  const uint4* from = (const uint4*)(z + row.head);
  ThreadStats s;
  if (row.single >= 0) add(s, to_f32(z[row.single]), k);
  int64_t i = threadIdx.x;
  for (; i + (kAtOnce - 1) * THREADS < row.count; i += kAtOnce * THREADS) {
    uint4 r[kAtOnce];
#pragma unroll
    for (int j = 0; j < kAtOnce; ++j) r[j] = from[i + j * THREADS];
    add<T>(s, r, k);
  }
  for (; i < row.count; i += THREADS) {
    const uint4 r[1] = {from[i]};
    add<T>(s, r, k);
  }
  return block_stats<THREADS>(s.s, k);
}

// A row's gradient c scale (1[v = t] - p_v): where it goes, and what it is made of.
template <typename T>
struct RowGradient {
  typedef Vector<T> Vec;
  T* out;
  RowStats s;
  float k, lift, step, share;
  int64_t target;
  bool whole;  // the output's rows start where the input's do, counted in 16 bytes

  __device__ RowGradient(T* out, const T* z, RowStats s, float scale, float slope, int64_t target)
      : out(out), s(s), k(scale * kLog2e), lift(lift_of(s.top, k)), step(slope * scale), share(slope * scale / s.sum),
        target(target), whole((((uintptr_t)out ^ (uintptr_t)z) & 15) == 0) {}

  __device__ __forceinline__ void single(float z, int64_t at) const {
    out[at] = from_f32<T>((at == target ? step : 0.0f) - share * ex2(fmaf(z - s.top, k, -lift)));
  }
  __device__ __forceinline__ uint4 of(uint4 r) const {
    float2 v[Vec::kPairs];
    Vec::read(r, v);
#pragma unroll
    for (int j = 0; j < Vec::kPairs; ++j) {
      const float2 x = fma2(add2(v[j], both(-s.top)), both(k), both(-lift));
      v[j] = mul2({ex2(x.x), ex2(x.y)}, both(-share));
    }
    return Vec::made(v);
  }
  __device__ __forceinline__ void store(uint4 r, int64_t at) const {
    if (whole) {
      *(uint4*)(out + at) = r;
      return;
    }
    const T* v = (const T*)&r;
#pragma unroll
    for (int j = 0; j < 2 * Vec::kPairs; ++j) out[at + j] = v[j];
  }
  // The target's element, for the thread that wrote its vector without the step: `vector` gives the
  // vectors of the row's share by number.
  template <int THREADS, typename F>
  __device__ __forceinline__ void mend(const RowShare<T>& row, F vector) const {
    const int64_t i = (target - row.element(0)) / (2 * Vec::kPairs);
    if (target < row.element(0) || i >= row.count || i % THREADS != (int)threadIdx.x) return;
    const uint4 r = vector(i);
    single(to_f32(((const T*)&r)[(target - row.element(0)) % (2 * Vec::kPairs)]), target);
  }
};
template <typename T, int THREADS>
__device__ __forceinline__ void zero_row(T* out, const T* z, const RowShare<T>& row) {
  const RowGradient<T> g(out, z, {0.0f, 1.0f}, 1.0f, 0.0f, -1);
  if (row.single >= 0) out[row.single] = from_f32<T>(0.0f);
  for (int64_t i = threadIdx.x; i < row.count; i += THREADS) g.store(uint4{0, 0, 0, 0}, row.element(i));
}
// The gradient of a row straight from memory, which may be written over as it is read.
template <typename T, int THREADS>
__device__ __forceinline__ void stream_gradient(const T* z, const RowShare<T>& row, const RowGradient<T>& g) {
  constexpr int kAtOnce = 4;
  const uint4* from = (const uint4*)(z + row.element(0));
  if (row.single >= 0) g.single(to_f32(z[row.single]), row.single);
  const int64_t mine = (g.target - row.element(0)) / RowShare<T>::kVec;  // the target's vector
  uint4 found{};
  int64_t i = threadIdx.x;
  for (; i + (kAtOnce - 1) * THREADS < row.count; i += kAtOnce * THREADS) {
    uint4 r[kAtOnce];
#pragma unroll
    for (int j = 0; j < kAtOnce; ++j) r[j] = from[i + j * THREADS];
#pragma unroll
    for (int j = 0; j < kAtOnce; ++j) {
      if (i + j * THREADS == mine) found = r[j];
      g.store(g.of(r[j]), row.element(i + j * THREADS));
    }
  }
  for (; i < row.count; i += THREADS) {
    const uint4 r = from[i];
    if (i == mine) found = r;
    g.store(g.of(r), row.element(i));
  }
  g.template mend<THREADS>(row, [&](int64_t) { return found; });
}

// Of the sum's logarithm the power of two is added to the logit's share, and 32 bits hold the rest, up
// to 0.35, to 3e-8.  z goes by the k that the sum's terms went by, and not by scale: what k's rounding
// does to the two then cancels where z is a token as likely as the row says.  Real: 64 bits where many
// rows are added up, as one near -10 has a rounding of 5e-7 in 32; 32 where a block waits for it (in
// 64, 16384 x 27 f32 took 8.5 us for 8.0).
template <typename Real>
__device__ __forceinline__ Real logp_of(float z, RowStats s, float scale) {
  const float k = scale * kLog2e, sum = s.sum / ex2(-lift_of(s.top, k));  // at least 1
  if (!(sum < INFINITY)) return NAN;
  const int power = (__float_as_int(sum) - 0x3f3504f3) >> 23;  // leaves sqrt(1/2) to sqrt(2)
  const float rest = __int_as_float(__float_as_int(sum) - (power << 23));
  return (Real)0.6931471805599453 * ((Real)k * ((Real)z - (Real)s.top) - (Real)power) - (Real)logf(rest);
}

template <typename T, int THREADS>
__global__ void __launch_bounds__(THREADS) k_token_logp(const T* logits, int64_t stride,
                                                        const int32_t* targets, int64_t vocab,
                                                        float scale, float* logp) {
  pdl_entry();
  const int64_t n = blockIdx.x, t = targets[n];
  float out = 0.0f;
  if (t >= 0) {
    const T* z = logits + n * stride;
    const RowStats s = row_stats<T, THREADS>(z, vocab, scale * kLog2e);
    if (threadIdx.x == 0 && s.sum != 0.0f) out = t < vocab ? (float)logp_of<double>(to_f32(z[t]), s, scale) : NAN;
  }
  if (threadIdx.x == 0) logp[n] = out;
}

// The loss term of one row and its derivative by the row's log probability.
struct Term {
  float loss, slope;
};
struct TermInputs {
  float advantage, old_logp, ref_logp, weight;
  __device__ TermInputs(const tb_policy_desc& d, int64_t n)
      : advantage(d.advantages[n]), old_logp(d.old_logp[n]), ref_logp(d.kl > 0 ? d.ref_logp[n] : 0.0f),
        weight(d.weights[n]) {}
};
__device__ __forceinline__ Term policy_term(const tb_policy_desc& d, const TermInputs& in, float logp) {
  const float a = in.advantage, r = expf(logp - in.old_logp);
  const float held = fminf(fmaxf(r, 1.0f - (float)d.clip_low), 1.0f + (float)d.clip_high);
  const float plain = r * a, kept = (r != r ? r : held) * a;
  float loss = -(plain <= kept ? plain : kept), slope = plain <= kept ? -plain : 0.0f;
  if (plain != plain) loss = slope = plain;
  if (d.kl > 0) {
    const float x = in.ref_logp - logp, e = expm1f(x);
    loss += (float)d.kl * (e - x);
    slope -= (float)d.kl * e;
  }
  return {in.weight * loss, in.weight * slope};
}

// The loss alone, a block a row.
template <typename T, int THREADS>
__global__ void __launch_bounds__(THREADS) k_policy_terms(tb_policy_desc d) {
  pdl_entry();
  const int64_t n = blockIdx.x, t = d.targets[n];
  const float scale = (float)d.scale;
  float logp = 0.0f;
  Term term{0.0f, 0.0f};
  const TermInputs in(d, n);
  if (t >= 0 && in.weight != 0.0f) {
    const T* z = (const T*)d.logits + n * d.logits_stride;
    const RowStats s = row_stats<T, THREADS>(z, d.vocab, scale * kLog2e);
    if (threadIdx.x == 0 && s.sum != 0.0f) {
      logp = t < d.vocab ? logp_of<float>(to_f32(z[t]), s, scale) : NAN;
      term = policy_term(d, in, logp);
    }
  }
  if (threadIdx.x == 0) {
    d.logp[n] = logp;
    d.token_loss[n] = term.loss;
  }
}

// The loss and its gradient in one reading of the logits: the blocks of a cluster share a row, each
// keeps its part in shared memory until the row's statistics are known.  A thread copies and reads
// its own vectors only, so that nothing but those statistics is waited for.  kKeep vectors a
// thread let two blocks of 512 threads (four of 256, eight of 128) share a SM, one loading while
// the other stores.
constexpr int kKeep = 13, kGroups = 4;

__device__ __forceinline__ void cluster_arrive() {
  asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");
}
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.aligned;" ::: "memory"); }

template <typename T, int THREADS>
__global__ void __launch_bounds__(THREADS, 1280 / THREADS) k_policy(tb_policy_desc d, int ranks, int64_t per) {
  pdl_entry();
  extern __shared__ uint4 kept[];
  __shared__ RowStats parts[8];
  const int64_t n = blockIdx.x / ranks;
  const int rank = blockIdx.x % ranks, keep = (int)((per + THREADS - 1) / THREADS);
  const int64_t t = d.targets[n];
  const TermInputs in(d, n);
  const float scale = (float)d.scale;
  const float k = scale * kLog2e;
  const T* z = (const T*)d.logits + n * d.logits_stride;
  T* out = (T*)d.gradient + n * d.gradient_stride;
  const RowShare<T> row(z, d.vocab, rank, ranks, per);
  // a block may be written to once all of its cluster have started
  cg::cluster_group cluster = cg::this_cluster();
  if (ranks > 1) cluster_arrive();
  if (t < 0 || in.weight == 0.0f) {  // the same for all blocks of the cluster
    if (ranks > 1) cluster_wait();
    zero_row<T, THREADS>(out, z, row);
    if (rank == 0 && threadIdx.x == 0) d.logp[n] = d.token_loss[n] = 0.0f;
    return;
  }
  const uint4* from = (const uint4*)(z + row.element(0));
  const int each = (keep + kGroups - 1) / kGroups, count = (int)row.count;
#pragma unroll
  for (int g = 0; g < kGroups; ++g) {
    const int last = min(count, min(keep, (g + 1) * each) * THREADS);
    for (int i = g * each * THREADS + threadIdx.x; i < last; i += THREADS)
      asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"((unsigned)__cvta_generic_to_shared(kept + i)),
                   "l"(from + i)
                   : "memory");
    asm volatile("cp.async.commit_group;" ::: "memory");
  }
  const float zt = t < d.vocab ? to_f32(z[t]) : 0.0f;
  const float single = row.single >= 0 ? to_f32(z[row.single]) : 0.0f;
  ThreadStats mine;
  if (row.single >= 0) add(mine, single, k);
#pragma unroll
  for (int g = 0; g < kGroups; ++g) {
    if (g == 0) asm volatile("cp.async.wait_group 3;" ::: "memory");
    if (g == 1) asm volatile("cp.async.wait_group 2;" ::: "memory");
    if (g == 2) asm volatile("cp.async.wait_group 1;" ::: "memory");
    if (g == 3) asm volatile("cp.async.wait_group 0;" ::: "memory");
    // by twos, so that they share a rescaling; one past the end is -inf, whose share is 0
    const int last = min(count, min(keep, (g + 1) * each) * THREADS);
    for (int i = g * each * THREADS + threadIdx.x; i < last; i += 2 * THREADS) {
      const uint4 r[2] = {kept[i], i + THREADS < last ? kept[i + THREADS] : Vector<T>::nothing()};
      add<T>(mine, r, k);
    }
  }
  RowStats s = block_stats<THREADS>(mine.s, k);
  if (ranks > 1) {
    cluster_wait();
    if ((int)threadIdx.x < ranks) *cluster.map_shared_rank(&parts[rank], threadIdx.x) = s;
    cluster.sync();
  }
  __shared__ RowStats whole;
  __shared__ float slope;
  if (threadIdx.x < 32) {
    const RowStats none{-INFINITY, 0.0f};
    if (ranks > 1) s = warp_stats((int)threadIdx.x < ranks ? parts[threadIdx.x] : none, k, 8);
    if (threadIdx.x == 0) {
      float logp = 0.0f;
      Term term{0.0f, 0.0f};
      if (s.sum != 0.0f) {
        logp = t < d.vocab ? logp_of<float>(zt, s, scale) : NAN;
        term = policy_term(d, in, logp);
      }
      if (rank == 0) {
        d.logp[n] = logp;
        d.token_loss[n] = term.loss;
      }
      whole = s;
      slope = term.slope;
    }
  }
  __syncthreads();
  if (whole.sum == 0.0f) {
    zero_row<T, THREADS>(out, z, row);
    return;
  }
  const RowGradient<T> g(out, z, whole, scale, slope, t);
  if (row.single >= 0) g.single(single, row.single);
  if (g.whole) {
    uint4* to = (uint4*)(out + row.element(0));
#pragma unroll 2
    for (int i = threadIdx.x; i < count; i += THREADS) to[i] = g.of(kept[i]);
  } else {
    for (int i = threadIdx.x; i < count; i += THREADS) g.store(g.of(kept[i]), row.element(i));
  }
  g.template mend<THREADS>(row, [&](int64_t i) { return kept[i]; });
}

// The same for rows that no cluster can keep: read twice.
template <typename T, int THREADS>
__global__ void __launch_bounds__(THREADS) k_policy_twice(tb_policy_desc d) {
  pdl_entry();
  const int64_t n = blockIdx.x, t = d.targets[n];
  const TermInputs in(d, n);
  const float scale = (float)d.scale;
  const T* z = (const T*)d.logits + n * d.logits_stride;
  T* out = (T*)d.gradient + n * d.gradient_stride;
  const RowShare<T> row(z, d.vocab, 0, 1, INT64_MAX / 2);
  __shared__ RowStats whole;
  __shared__ float slope;
  RowStats s{0.0f, 0.0f};
  if (t >= 0 && in.weight != 0.0f) s = row_stats<T, THREADS>(z, d.vocab, scale * kLog2e);
  if (threadIdx.x == 0) {
    float logp = 0.0f;
    Term term{0.0f, 0.0f};
    if (s.sum != 0.0f) {
      logp = t < d.vocab ? logp_of<float>(to_f32(z[t]), s, scale) : NAN;
      term = policy_term(d, in, logp);
    }
    d.logp[n] = logp;
    d.token_loss[n] = term.loss;
    whole = s;
    slope = term.slope;
  }
  __syncthreads();  // the gradient may overwrite the logits that others still read
  if (whole.sum == 0.0f) zero_row<T, THREADS>(out, z, row);
  else stream_gradient<T, THREADS>(z, row, RowGradient<T>(out, z, whole, scale, slope, t));
}

// ---- small vocabularies: a warp a row, ITEMS logits a lane in registers
template <typename T, int ITEMS>
struct WarpRow {
  float v[ITEMS];
  RowStats s;
  __device__ WarpRow(const T* z, int vocab, float k) {
    const int lane = threadIdx.x % 32;
    s = {-INFINITY, 0.0f};
#pragma unroll
    for (int j = 0; j < ITEMS; ++j) v[j] = lane + 32 * j < vocab ? to_f32(z[lane + 32 * j]) : -INFINITY;
#pragma unroll
    for (int j = 0; j < ITEMS; ++j) s.top = fmaxf(s.top, v[j]);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) s.top = fmaxf(s.top, __shfl_xor_sync(~0u, s.top, o));
    const float base = base_of(s.top), lift = lift_of(base, k);
#pragma unroll
    for (int j = 0; j < ITEMS; ++j) {
      v[j] = ex2(fmaf(v[j] - base, k, -lift));
      s.sum += v[j];
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) s.sum += __shfl_xor_sync(~0u, s.sum, o);
  }
  __device__ void gradient(T* out, int vocab, float scale, float slope, int64_t target) const {
    const int lane = threadIdx.x % 32;
    const float step = slope * scale, share = s.sum == 0.0f ? 0.0f : step / s.sum;
#pragma unroll
    for (int j = 0; j < ITEMS; ++j)
      if (lane + 32 * j < vocab)
        out[lane + 32 * j] = from_f32<T>(s.sum == 0.0f ? 0.0f : (lane + 32 * j == target ? step : 0.0f) - share * v[j]);
  }
};
template <typename T>
__device__ __forceinline__ void zero_warp_row(T* out, int64_t vocab) {
  for (int v = threadIdx.x % 32; v < vocab; v += 32) out[v] = from_f32<T>(0.0f);
}

template <typename T, int ITEMS>
__global__ void __launch_bounds__(256) k_policy_warps(tb_policy_desc d) {
  pdl_entry();
  const int64_t n = (int64_t)blockIdx.x * 8 + threadIdx.x / 32;
  if (n >= d.rows) return;
  const int64_t t = d.targets[n];
  const TermInputs in(d, n);
  const float scale = (float)d.scale;
  const T* z = (const T*)d.logits + n * d.logits_stride;
  T* out = (T*)d.gradient + n * d.gradient_stride;
  float logp = 0.0f;
  Term term{0.0f, 0.0f};
  if (t >= 0 && in.weight != 0.0f) {
    const float zt = t < d.vocab ? to_f32(z[t]) : 0.0f;
    const WarpRow<T, ITEMS> row(z, (int)d.vocab, scale * kLog2e);
    if (row.s.sum != 0.0f) {
      logp = t < d.vocab ? logp_of<float>(zt, row.s, scale) : NAN;
      term = policy_term(d, in, logp);
    }
    __syncwarp();  // the gradient may overwrite the logits that others still read
    if (d.gradient) row.gradient(out, (int)d.vocab, scale, term.slope, t);
  } else if (d.gradient) {
    zero_warp_row(out, d.vocab);
  }
  if (threadIdx.x % 32 == 0) {
    d.logp[n] = logp;
    d.token_loss[n] = term.loss;
  }
}

template <typename T, int ITEMS>
__global__ void __launch_bounds__(256) k_token_logp_warps(const T* logits, int64_t stride, const int32_t* targets,
                                                          int64_t rows, int64_t vocab, float scale, float* logp) {
  pdl_entry();
  const int64_t n = (int64_t)blockIdx.x * 8 + threadIdx.x / 32;
  if (n >= rows) return;
  const int64_t t = targets[n];
  float out = 0.0f;
  if (t >= 0) {
    const T* z = logits + n * stride;
    const float zt = t < vocab ? to_f32(z[t]) : 0.0f;
    const WarpRow<T, ITEMS> row(z, (int)vocab, scale * kLog2e);
    if (row.s.sum != 0.0f) out = t < vocab ? (float)logp_of<double>(zt, row.s, scale) : NAN;
  }
  if (threadIdx.x % 32 == 0) logp[n] = out;
}

// loss[0] = the sum of the terms, in a fixed order and f64.
__global__ void __launch_bounds__(1024) k_sum_terms(const float* terms, int64_t count, float* loss) {
  pdl_entry();
  __shared__ double part[32];
  double s = 0;
#pragma unroll 8
  for (int64_t i = threadIdx.x; i < count; i += 1024) s += terms[i];
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(~0u, s, o);
  if (threadIdx.x % 32 == 0) part[threadIdx.x / 32] = s;
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int w = 1; w < 32; ++w) s += part[w];
    loss[0] = (float)s;
  }
}

// Workspace of the preference loss.
struct PreferenceScratch {
  double* terms;    // [pairs], the weighted losses
  RowStats* stats;  // [rows]
  float* slopes;    // [rows], logp - ref, then the loss's slope by the row's log probability
  __host__ __device__ explicit PreferenceScratch(const tb_preference_desc& d)
      : terms((double*)d.workspace), stats((RowStats*)(terms + d.pairs)), slopes((float*)(stats + d.rows)) {}
};
__device__ __forceinline__ int64_t clamp_row(int64_t v, int64_t rows) {
  return v < 0 ? 0 : v > rows ? rows : v;
}
__device__ __forceinline__ bool scored(const tb_preference_desc& d, int64_t n) {
  return n >= d.offsets[0] && n < d.offsets[2 * d.pairs];
}

template <typename T, int THREADS>
__global__ void __launch_bounds__(THREADS) k_preference_rows(tb_preference_desc d) {
  pdl_entry();
  const int64_t n = blockIdx.x;
  if (!scored(d, n)) {
    if (threadIdx.x == 0 && d.clear & TB_PREFERENCE_CLEAR_LOGP) d.logp[n] = 0.0f;
    return;
  }
  const int64_t t = d.targets[n];
  const float scale = (float)d.scale;
  RowStats s{0.0f, 0.0f};
  double logp = 0.0;
  if (t >= 0) {
    const T* z = (const T*)d.logits + n * d.logits_stride;
    s = row_stats<T, THREADS>(z, d.vocab, scale * kLog2e);
    if (threadIdx.x == 0 && s.sum != 0.0f) logp = t < d.vocab ? logp_of<double>(to_f32(z[t]), s, scale) : NAN;
  }
  if (threadIdx.x == 0) {
    const PreferenceScratch scratch(d);
    scratch.stats[n] = s;
    if (s.sum != 0.0f) scratch.slopes[n] = (float)(logp - (double)d.ref_logp[n]);
    d.logp[n] = (float)logp;
  }
}
template <typename T, int ITEMS>
__global__ void __launch_bounds__(256) k_preference_rows_warps(tb_preference_desc d) {
  pdl_entry();
  const int64_t n = (int64_t)blockIdx.x * 8 + threadIdx.x / 32;
  if (n >= d.rows) return;
  if (!scored(d, n)) {
    if (threadIdx.x % 32 == 0 && d.clear & TB_PREFERENCE_CLEAR_LOGP) d.logp[n] = 0.0f;
    return;
  }
  const int64_t t = d.targets[n];
  const float scale = (float)d.scale;
  RowStats s{0.0f, 0.0f};
  double logp = 0.0;
  if (t >= 0) {
    const T* z = (const T*)d.logits + n * d.logits_stride;
    const float zt = t < d.vocab ? to_f32(z[t]) : 0.0f;
    s = WarpRow<T, ITEMS>(z, (int)d.vocab, scale * kLog2e).s;
    if (s.sum != 0.0f) logp = t < d.vocab ? logp_of<double>(zt, s, scale) : NAN;
  }
  if (threadIdx.x % 32 == 0) {
    const PreferenceScratch scratch(d);
    scratch.stats[n] = s;
    if (s.sum != 0.0f) scratch.slopes[n] = (float)(logp - (double)d.ref_logp[n]);
    d.logp[n] = (float)logp;
  }
}

// A block a pair: both answers' sums in f64 (the margin is a small difference of long sums), the
// pair's term, and its rows' slopes.
constexpr int kPairThreads = 256;
__global__ void __launch_bounds__(kPairThreads) k_preference_pairs(tb_preference_desc d) {
  pdl_entry();
  __shared__ double part[2][kPairThreads / 32];
  const PreferenceScratch scratch(d);
  const int64_t i = blockIdx.x;
  int64_t lo[2], hi[2];
  double ratio[2];
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    lo[k] = clamp_row(d.offsets[i + k * d.pairs], d.rows);
    hi[k] = clamp_row(d.offsets[i + k * d.pairs + 1], d.rows);
    double r = 0;
#pragma unroll 4
    for (int64_t n = lo[k] + threadIdx.x; n < hi[k]; n += kPairThreads)
      if (scratch.stats[n].sum != 0.0f) r += (double)scratch.slopes[n];
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) r += __shfl_xor_sync(~0u, r, o);
    if (threadIdx.x % 32 == 0) part[k][threadIdx.x / 32] = r;
  }
  __syncthreads();
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    ratio[k] = part[k][0];
    for (int w = 1; w < kPairThreads / 32; ++w) ratio[k] += part[k][w];
  }
  const double w = d.weights ? (double)d.weights[i] : 1.0 / (double)d.pairs;
  const double m = d.beta * (ratio[0] - ratio[1]), e = exp(-fabs(m));
  const double soft = log1p(e);                            // -log sigmoid(|m|)
  const double lose = m >= 0 ? e / (1 + e) : 1 / (1 + e);  // sigmoid(-m)
  const double yes = m >= 0 ? soft : soft - m, no = m >= 0 ? soft + m : soft;
  if (threadIdx.x == 0) {
    d.ratios[i] = (float)ratio[0];
    d.ratios[i + d.pairs] = (float)ratio[1];
    // a share of 0 adds nothing, whatever it would multiply
    scratch.terms[i] = w * ((1 - d.smoothing) * yes + (d.smoothing > 0 ? d.smoothing * no : 0.0));
  }
  const float slope = (float)(w * d.beta * (d.smoothing * (1 - lose) - (1 - d.smoothing) * lose));
#pragma unroll
  for (int k = 0; k < 2; ++k)
    for (int64_t n = lo[k] + threadIdx.x; n < hi[k]; n += kPairThreads) scratch.slopes[n] = k ? -slope : slope;
}

// The pairs' terms in a fixed order, by one warp.
__device__ __forceinline__ void sum_pairs(const tb_preference_desc& d) {
  const double* terms = PreferenceScratch(d).terms;
  double s = 0;
  for (int64_t i = threadIdx.x; i < d.pairs; i += 32) s += terms[i];
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(~0u, s, o);
  if (threadIdx.x == 0) d.loss[0] = (float)s;
}
__global__ void k_preference_sum(tb_preference_desc d) {
  pdl_entry();
  sum_pairs(d);
}

template <typename T, int THREADS>
__global__ void __launch_bounds__(THREADS) k_preference_gradient(tb_preference_desc d) {
  pdl_entry();
  if (blockIdx.x == 0 && threadIdx.x < 32) sum_pairs(d);
  // from the last row back, for the rows that were read last may still be in the L2 cache (32 of 288 MB
  // are: 4099 x 50257 bf16 reads 256 from memory here)
  const int64_t n = d.rows - 1 - blockIdx.x;
  const T* z = (const T*)d.logits + n * d.logits_stride;
  T* out = (T*)d.gradient + n * d.gradient_stride;
  const RowShare<T> row(z, d.vocab, 0, 1, INT64_MAX / 2);
  if (!scored(d, n)) {
    if (d.clear & TB_PREFERENCE_CLEAR_GRADIENT) zero_row<T, THREADS>(out, z, row);
    return;
  }
  const PreferenceScratch scratch(d);
  const RowStats s = scratch.stats[n];
  const int64_t t = d.targets[n];
  const float slope = t < d.vocab ? scratch.slopes[n] : NAN;
  if (s.sum == 0.0f) zero_row<T, THREADS>(out, z, row);
  else stream_gradient<T, THREADS>(z, row, RowGradient<T>(out, z, s, (float)d.scale, slope, t));
}
template <typename T>
__global__ void __launch_bounds__(256) k_preference_gradient_warps(tb_preference_desc d) {
  pdl_entry();
  if (blockIdx.x == 0 && threadIdx.x < 32) sum_pairs(d);
  const int64_t n = (int64_t)blockIdx.x * 8 + threadIdx.x / 32;
  if (n >= d.rows) return;
  const T* z = (const T*)d.logits + n * d.logits_stride;
  T* out = (T*)d.gradient + n * d.gradient_stride;
  if (!scored(d, n)) {
    if (d.clear & TB_PREFERENCE_CLEAR_GRADIENT) zero_warp_row(out, d.vocab);
    return;
  }
  const PreferenceScratch scratch(d);
  const RowStats s = scratch.stats[n];
  const int64_t t = d.targets[n];
  if (s.sum == 0.0f) {
    zero_warp_row(out, d.vocab);
    return;
  }
  const RowGradient<T> g(out, z, s, (float)d.scale, t < d.vocab ? scratch.slopes[n] : NAN, t);
#pragma unroll 4
  for (int64_t v = threadIdx.x % 32; v < d.vocab; v += 32) g.single(to_f32(z[v]), v);
}

const char* check_logits(int64_t element, int64_t rows, int64_t vocab, int64_t stride, double scale,
                         const void* logits) {
  if (element != TB_ELEMENT_F32 && element != TB_ELEMENT_BF16) return "unknown element type";
  if (!extents_fit({rows, vocab}) || !extents_fit({rows, stride}) || rows > INT32_MAX)
    return "extents out of range";
  if (rows > 0 && vocab < 1) return "an empty vocabulary";
  // scale log2(e) has to be finite too
  if (!(scale > 0) || scale > 2e38 || (float)scale == 0.0f)
    return "scale is positive and at most 2e38";
  if (rows > 0 && !logits) return "a required array is NULL";
  if (!aligned_to(logits, element == TB_ELEMENT_F32 ? 4 : 2))
    return "an array is not aligned to its elements";
  return nullptr;
}
const char* check_gradient(int64_t element, int64_t rows, int64_t vocab, int64_t stride,
                           const void* gradient) {
  if (!gradient) return nullptr;
  if (!extents_fit({rows, stride}) || (rows > 1 && stride < vocab))
    return "gradient rows overlap or their stride is out of range";
  if (!aligned_to(gradient, element == TB_ELEMENT_F32 ? 4 : 2))
    return "an array is not aligned to its elements";
  return nullptr;
}
bool words_ok(std::initializer_list<const void*> arrays) {
  for (const void* p : arrays)
    if (!p || !aligned_to(p, 4)) return false;
  return true;
}

// Threads of a block that reads a row, or reads and writes one.  Reading, many small blocks hide one
// another's ends (8192 x 50257 bf16: 102 us with 256 threads, 123 with 512); reading and writing, few
// large ones keep to the rows that lie side by side (4099 x 50257 f32: 512 threads 320 us, 256 332).
template <typename T>
int reading_threads(int64_t vocab) {
  return vocab * (int64_t)sizeof(T) / 16 > 1024 ? 256 : 128;
}
template <typename T>
int writing_threads(int64_t vocab) {
  const int64_t vectors = vocab * (int64_t)sizeof(T) / 16;
  return vectors > 4096 ? 512 : vectors > 1024 ? 256 : 128;
}
#define TB_BY_THREADS(THREADS, KERNEL, ...)                                                         \
  switch (THREADS) {                                                                                \
    case 512: return launch_pdl(KERNEL<T, 512>, dim3((unsigned)rows), dim3(512), 0, stream, __VA_ARGS__); \
    case 256: return launch_pdl(KERNEL<T, 256>, dim3((unsigned)rows), dim3(256), 0, stream, __VA_ARGS__); \
    default: return launch_pdl(KERNEL<T, 128>, dim3((unsigned)rows), dim3(128), 0, stream, __VA_ARGS__);  \
  }
// Rows that fit a warp's registers (8192 x 1100 f32 with the gradient: 29 us in 64 registers a lane, 27
// by blocks; bf16 40 and 28).
constexpr int64_t kWarpVocab = 1024;
#define TB_BY_ITEMS(KERNEL, ...)                                                                   \
  {                                                                                                \
    const dim3 grid((unsigned)((rows + 7) / 8)), block(256);                                       \
    if (vocab <= 32) return launch_pdl(KERNEL<T, 1>, grid, block, 0, stream, __VA_ARGS__);         \
    if (vocab <= 128) return launch_pdl(KERNEL<T, 4>, grid, block, 0, stream, __VA_ARGS__);        \
    if (vocab <= 512) return launch_pdl(KERNEL<T, 16>, grid, block, 0, stream, __VA_ARGS__);       \
    return launch_pdl(KERNEL<T, 32>, grid, block, 0, stream, __VA_ARGS__);                         \
  }

template <typename T>
cudaError_t enqueue_logp(const T* logits, int64_t stride, const int32_t* targets, int64_t rows, int64_t vocab,
                         float scale, float* logp, cudaStream_t stream) {
  if (vocab <= kWarpVocab)
    TB_BY_ITEMS(k_token_logp_warps, logits, stride, targets, rows, vocab, scale, logp)
  TB_BY_THREADS(reading_threads<T>(vocab), k_token_logp, logits, stride, targets, vocab, scale, logp)
}

template <typename T, int THREADS>
cudaError_t enqueue_kept(const tb_policy_desc& d, int ranks, int64_t per, cudaStream_t stream) {
  const size_t bytes = (size_t)per * 16;
  const auto kernel = k_policy<T, THREADS>;
  static std::atomic<uint64_t> allowed{0};  // devices on which the kernel may use the most it needs
  if (const cudaError_t e = allow_shared((const void*)kernel, (size_t)kKeep * THREADS * 16, allowed)) return e;
  if (d.rows * ranks > INT32_MAX) return cudaErrorInvalidConfiguration;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(d.rows * ranks));
  cfg.blockDim = dim3(THREADS);
  cfg.dynamicSmemBytes = bytes;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = ranks;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = pdl_enabled() ? 2 : 1;
  return cudaLaunchKernelEx(&cfg, kernel, d, ranks, per);
}
template <typename T>
cudaError_t enqueue_policy(const tb_policy_desc& d, cudaStream_t stream) {
  const int64_t rows = d.rows, vocab = d.vocab;
  if (vocab <= kWarpVocab) TB_BY_ITEMS(k_policy_warps, d)
  if (!d.gradient) TB_BY_THREADS(reading_threads<T>(vocab), k_policy_terms, d)
  const int64_t vectors = vocab * (int64_t)sizeof(T) / 16;
  // one block a row while it holds one (8192 x 16000 bf16: 256 threads 111 us, two blocks of 128
  // 130), else the smallest blocks whose clusters do (8192 x 50257 f32: 8 blocks of 128 threads
  // 495 us, 4 of 256 501, 2 of 512 516; 4 of 512, half filled, 703)
  if (vectors <= kKeep * 128) return enqueue_kept<T, 128>(d, 1, vectors, stream);
  if (vectors <= kKeep * 256) return enqueue_kept<T, 256>(d, 1, vectors, stream);
  if (vectors <= kKeep * 512) return enqueue_kept<T, 512>(d, 1, vectors, stream);
  const auto ranks = [&](int threads) { return (vectors + kKeep * threads - 1) / (kKeep * threads); };
  const auto per = [&](int threads) { return (vectors + ranks(threads) - 1) / ranks(threads); };
  if (ranks(128) <= 8) return enqueue_kept<T, 128>(d, (int)ranks(128), per(128), stream);
  if (ranks(256) <= 8) return enqueue_kept<T, 256>(d, (int)ranks(256), per(256), stream);
  if (ranks(512) <= 8) return enqueue_kept<T, 512>(d, (int)ranks(512), per(512), stream);
  return launch_pdl(k_policy_twice<T, 512>, dim3((unsigned)rows), dim3(512), 0, stream, d);
}
template <typename T>
cudaError_t enqueue_preference_rows(const tb_preference_desc& d, cudaStream_t stream) {
  const int64_t rows = d.rows, vocab = d.vocab;
  if (vocab <= kWarpVocab) TB_BY_ITEMS(k_preference_rows_warps, d)
  TB_BY_THREADS(reading_threads<T>(vocab), k_preference_rows, d)
}
template <typename T>
cudaError_t enqueue_preference_gradient(const tb_preference_desc& d, cudaStream_t stream) {
  const int64_t rows = d.rows, vocab = d.vocab;
  if (vocab <= kWarpVocab)
    return launch_pdl(k_preference_gradient_warps<T>, dim3((unsigned)((rows + 7) / 8)), dim3(256), 0, stream, d);
  TB_BY_THREADS(writing_threads<T>(vocab), k_preference_gradient, d)
}

int token_logp(int64_t element, const void* logits, int64_t stride, const int32_t* targets,
               int64_t rows, int64_t vocab, double scale, float* logp, void* stream) {
  OperatorCall call("tb_token_logp", stream);
  if (const char* why = check_logits(element, rows, vocab, stride, scale, logits))
    return call.invalid(why);
  if (rows > 0 && !words_ok({targets, logp})) return call.invalid("a row array is NULL or unaligned");
  if (const int code = call.ready()) return code;
  if (rows == 0) return TB_OK;
  return call.finish(
      element == TB_ELEMENT_F32
          ? enqueue_logp((const float*)logits, stride, targets, rows, vocab, (float)scale, logp, call.stream())
          : enqueue_logp((const bf16*)logits, stride, targets, rows, vocab, (float)scale, logp, call.stream()));
}

int policy_loss(const tb_policy_desc* desc, void* stream) {
  OperatorCall call("tb_policy_loss", stream);
  if (!desc) return call.invalid("no request");
  const tb_policy_desc d = *desc;
  if (const char* why = check_logits(d.element, d.rows, d.vocab, d.logits_stride, d.scale, d.logits))
    return call.invalid(why);
  if (const char* why = check_gradient(d.element, d.rows, d.vocab, d.gradient_stride, d.gradient))
    return call.invalid(why);
  if (!(d.clip_low >= 0) || !(d.clip_high >= 0) || !(d.kl >= 0) || d.kl > 3e38)
    return call.invalid("clip_low, clip_high and kl are not negative");
  if (!words_ok({d.loss}) ||
      (d.rows > 0 && (!words_ok({d.targets, d.old_logp, d.advantages, d.weights, d.token_loss, d.logp}) ||
                      (d.kl > 0 && !words_ok({d.ref_logp})))))
    return call.invalid("a row array is NULL or unaligned");
  if (const int code = call.ready()) return code;
  cudaError_t e = cudaSuccess;
  if (d.rows > 0)
    e = d.element == TB_ELEMENT_F32 ? enqueue_policy<float>(d, call.stream()) : enqueue_policy<bf16>(d, call.stream());
  if (e == cudaSuccess)
    e = launch_pdl(k_sum_terms, dim3(1), dim3(1024), 0, call.stream(), (const float*)d.token_loss,
                   d.rows, d.loss);
  return call.finish(e);
}

int preference_loss(const tb_preference_desc* desc, void* stream) {
  OperatorCall call("tb_preference_loss", stream);
  if (!desc) return call.invalid("no request");
  const tb_preference_desc d = *desc;
  if (const char* why = check_logits(d.element, d.rows, d.vocab, d.logits_stride, d.scale, d.logits))
    return call.invalid(why);
  if (const char* why = check_gradient(d.element, d.rows, d.vocab, d.gradient_stride, d.gradient))
    return call.invalid(why);
  if (d.pairs < 1 || d.pairs > INT32_MAX / 2) return call.invalid("pairs out of range");
  if (!(d.beta > 0) || d.beta > 3e38) return call.invalid("beta is positive and finite");
  if (!(d.smoothing >= 0 && d.smoothing < 1)) return call.invalid("smoothing lies in [0, 1)");
  if (d.clear & ~(TB_PREFERENCE_CLEAR_LOGP | TB_PREFERENCE_CLEAR_GRADIENT))
    return call.invalid("unknown array to clear");
  if (!words_ok({d.loss, d.ratios, d.offsets}) || !aligned_to(d.weights, 4) ||
      (d.rows > 0 && !words_ok({d.targets, d.ref_logp, d.logp})))
    return call.invalid("a row array is NULL or unaligned");
  if (!d.workspace || d.workspace_bytes < tb_preference_workspace(d.rows, d.pairs))
    return call.invalid("the workspace is too small");
  if (!aligned_to(d.workspace, 16)) return call.invalid("the workspace is not 16-byte aligned");
  if (const int code = call.ready()) return code;
  const bool f32 = d.element == TB_ELEMENT_F32;
  cudaError_t e = cudaSuccess;
  if (d.rows > 0)
    e = f32 ? enqueue_preference_rows<float>(d, call.stream()) : enqueue_preference_rows<bf16>(d, call.stream());
  if (e == cudaSuccess)
    e = launch_pdl(k_preference_pairs, dim3((unsigned)d.pairs), dim3(kPairThreads), 0, call.stream(), d);
  if (e == cudaSuccess && d.rows > 0 && d.gradient)
    e = f32 ? enqueue_preference_gradient<float>(d, call.stream())
            : enqueue_preference_gradient<bf16>(d, call.stream());
  else if (e == cudaSuccess)
    e = launch_pdl(k_preference_sum, dim3(1), dim3(32), 0, call.stream(), d);
  return call.finish(e);
}

}  // namespace
}  // namespace tb

extern "C" int tb_token_logp(int64_t element, const void* logits, int64_t row_stride,
                             const int32_t* targets, int64_t rows, int64_t vocab, double scale,
                             float* logp, void* stream) {
  return tb::guarded([&] {
    return tb::token_logp(element, logits, row_stride, targets, rows, vocab, scale, logp, stream);
  });
}
extern "C" int tb_policy_loss(const tb_policy_desc* desc, void* stream) {
  return tb::guarded([&] { return tb::policy_loss(desc, stream); });
}
extern "C" int tb_preference_loss(const tb_preference_desc* desc, void* stream) {
  return tb::guarded([&] { return tb::preference_loss(desc, stream); });
}
extern "C" int64_t tb_preference_workspace(int64_t rows, int64_t pairs) {
  return rows >= 0 && pairs > 0 && rows <= INT32_MAX && pairs <= INT32_MAX ? pairs * 8 + rows * 12 : 0;
}
