// rotate.cu -- the root-mean-square norm of every query and key head with the rotation by the
// token's position, and its backward pass.
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

constexpr int64_t kBackwardBlocks = 296;  // rows of weight-gradient partials

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
    ((float*)d.workspace)[(int64_t)blockIdx.x * 2 * dim + j] = s;
  }
}

// Weight gradients: the partials in block order, 32 threads an element.
__global__ void k_rotate_weights(tb_rotate_desc d) {
  pdl_entry();
  const int lane = threadIdx.x % 32, dim = (int)d.dim;
  const int j = (int)((blockIdx.x * blockDim.x + threadIdx.x) / 32);
  if (j >= 2 * dim) return;
  float s = 0;
  for (int b = lane; b < kBackwardBlocks; b += 32) s += ((const float*)d.workspace)[b * 2 * dim + j];
  s = warp_sum(s);
  float* out = j < dim ? d.dq_weight : d.dk_weight;
  if (lane == 0 && out) out[j < dim ? j : j - dim] = s;
}

int64_t workspace_bytes(const tb_rotate_desc& d) {
  return d.dq_weight || d.dk_weight ? tb_head_rotate_workspace(d.dim) : 0;
}

bool strides_ok(const tb_rotate_desc& d, const int64_t s[3], int64_t heads, bool written) {
  if (!extents_fit({s[0]}) || !extents_fit({s[1]}) || !extents_fit({s[2]})) return false;
  if (!written) return true;
  return (heads <= 1 || s[2] >= d.dim) && (d.length <= 1 || s[1] >= d.dim) &&
         (d.batch <= 1 || s[0] >= d.dim);
}

const char* check(const tb_rotate_desc& d, bool backward) {
  if (d.element != TB_ELEMENT_F32 && d.element != TB_ELEMENT_BF16) return "unknown element type";
  if (d.style != TB_ROTATE_HALVES && d.style != TB_ROTATE_PAIRS) return "unknown style";
  if (!extents_fit({d.batch, d.length, d.q_heads, d.dim}) || d.length > INT32_MAX ||
      !extents_fit({d.batch, d.length, d.k_heads, d.dim}) || !extents_fit({d.table_rows, d.turned}) ||
      d.q_heads > INT32_MAX / 2 || d.k_heads > INT32_MAX / 2)
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

template <typename T>
cudaError_t enqueue(tb_rotate_desc d, bool backward, cudaStream_t stream) {
  const int64_t rows = d.batch * d.length * (d.q_heads + d.k_heads);
  if (!backward) {
    const int64_t blocks = (rows + 7) / 8;
    if (blocks > INT32_MAX) return cudaErrorInvalidConfiguration;
    return blocks ? launch_pdl(k_rotate<T>, dim3((unsigned)blocks), dim3(256), 0, stream, d, rows)
                  : cudaSuccess;
  }
  if (!workspace_bytes(d)) d.workspace = nullptr;
  if (!rows && !d.workspace) return cudaSuccess;
  cudaError_t e = launch_pdl(k_rotate_backward<T>, dim3(kBackwardBlocks), dim3(256),
                             (size_t)8 * 2 * d.dim * 4, stream, d, rows);
  if (e == cudaSuccess && d.workspace)
    e = launch_pdl(k_rotate_weights, dim3((unsigned)((2 * d.dim + 7) / 8)), dim3(256), 0, stream, d);
  return e;
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
