// losses.cu -- log probabilities of tokens, the clipped policy loss and the paired log-ratio
// loss over a vocabulary, with their gradients by the logits.
//
// With p = softmax(scale z) and L = scale z_t - lse, every loss reaches the logits through L
// alone: dz_v = c scale (1[v = t] - p_v) with c = d loss / d L of the row.  Maxima are taken of
// the raw logits and scale multiplies differences from them, so masks of the type's lowest
// value do not overflow.
#include "operators.h"

namespace tb {
namespace {

constexpr int kThreads = 512;

struct RowStats {
  float top, sum;  // max z, sum exp(scale (z - top)); sum = 0 where no logit is above -inf
};
// Differences from the top are never taken from -inf, and exp(0) = 1 exactly; a NaN or +inf
// logit makes the sum NaN (fmaxf passes a NaN over, the exponential does not).
__device__ __forceinline__ RowStats merge(RowStats p, RowStats q, float scale) {
  const float top = fmaxf(p.top, q.top);
  if (top == -INFINITY) return {top, p.sum + q.sum};
  return {top, p.sum * __expf(scale * (p.top - top)) + q.sum * __expf(scale * (q.top - top))};
}
__device__ __forceinline__ RowStats add(RowStats s, float z, float scale) {
  const float top = fmaxf(s.top, z);
  if (top == -INFINITY) return {top, z != z ? z : s.sum};
  return {top, s.sum * __expf(scale * (s.top - top)) + __expf(scale * (z - top))};
}

// Block-wide statistics of a row; every thread gets them.
template <typename T>
__device__ RowStats row_stats(const T* z, int64_t vocab, float scale) {
  __shared__ RowStats part[kThreads / 32];
  RowStats s{-INFINITY, 0.0f};
  for (int64_t v = threadIdx.x; v < vocab; v += kThreads) s = add(s, to_f32(z[v]), scale);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1)
    s = merge(s, {__shfl_xor_sync(~0u, s.top, o), __shfl_xor_sync(~0u, s.sum, o)}, scale);
  __syncthreads();
  if (threadIdx.x % 32 == 0) part[threadIdx.x / 32] = s;
  __syncthreads();
  s = part[0];
  for (int w = 1; w < kThreads / 32; ++w) s = merge(s, part[w], scale);
  return s;
}

// Writes c scale (1[v = t] - p_v) over a row; zeros for c = 0 rows marked hidden.
template <typename T>
__device__ void row_gradient(const T* z, T* out, int64_t vocab, float scale, RowStats s, int64_t t,
                             float c, bool hidden) {
  const float step = c * scale, share = step / s.sum;
  for (int64_t v = threadIdx.x; v < vocab; v += kThreads) {
    float d = 0.0f;
    if (!hidden) d = (v == t ? step : 0.0f) - share * __expf(scale * (to_f32(z[v]) - s.top));
    out[v] = from_f32<T>(d);
  }
}

__device__ __forceinline__ float logp_of(float z, RowStats s, float scale) {
  return scale * (z - s.top) - logf(s.sum);
}

template <typename T>
__global__ void __launch_bounds__(kThreads) k_token_logp(const T* logits, int64_t stride, const int32_t* targets,
                                                         int64_t vocab, float scale, float* logp) {
  pdl_entry();
  const int64_t n = blockIdx.x, t = targets[n];
  float out = 0.0f;
  if (t >= 0) {
    const T* z = logits + n * stride;
    const RowStats s = row_stats(z, vocab, scale);
    if (s.sum != 0.0f) out = t < vocab ? logp_of(to_f32(z[t]), s, scale) : NAN;
  }
  if (threadIdx.x == 0) logp[n] = out;
}

// The loss term of one row and its derivative by the row's log probability.
struct Term {
  float loss, slope;
};
__device__ __forceinline__ Term policy_term(const tb_policy_desc& d, int64_t n, float logp, float w) {
  const float a = d.advantages[n], r = expf(logp - d.old_logp[n]);
  const float held = fminf(fmaxf(r, 1.0f - (float)d.clip_low), 1.0f + (float)d.clip_high);
  const float plain = r * a, kept = (r != r ? r : held) * a;
  float loss = -(plain <= kept ? plain : kept), slope = plain <= kept ? -plain : 0.0f;
  if (plain != plain) loss = slope = plain;
  if (d.kl > 0) {
    const float x = d.ref_logp[n] - logp, e = expm1f(x);
    loss += (float)d.kl * (e - x);
    slope -= (float)d.kl * e;
  }
  return {w * loss, w * slope};
}

template <typename T>
__global__ void __launch_bounds__(kThreads) k_policy(tb_policy_desc d) {
  pdl_entry();
  const int64_t n = blockIdx.x, t = d.targets[n];
  const float w = d.weights[n], scale = (float)d.scale;
  const T* z = (const T*)d.logits + n * d.logits_stride;
  bool hidden = t < 0 || w == 0.0f;
  RowStats s{0.0f, 1.0f};
  float logp = 0.0f;
  Term term{0.0f, 0.0f};
  if (!hidden) {
    s = row_stats(z, d.vocab, scale);
    hidden = s.sum == 0.0f;
    if (!hidden) {
      logp = t < d.vocab ? logp_of(to_f32(z[t]), s, scale) : NAN;
      term = policy_term(d, n, logp, w);
    }
  }
  __syncthreads();  // the gradient may overwrite the logits that others still read
  if (threadIdx.x == 0) {
    d.logp[n] = logp;
    d.token_loss[n] = term.loss;
  }
  if (d.gradient)
    row_gradient(z, (T*)d.gradient + n * d.gradient_stride, d.vocab, scale, s, t, term.slope, hidden);
}

// loss[0] = the sum of the terms, in a fixed order and f64.
__global__ void __launch_bounds__(1024) k_sum_terms(const float* terms, int64_t count, float* loss) {
  pdl_entry();
  __shared__ double part[32];
  double s = 0;
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

// Workspace of the preference loss: RowStats[rows], then float slopes[rows].
__device__ __forceinline__ int64_t clamp_row(int64_t v, int64_t rows) {
  return v < 0 ? 0 : v > rows ? rows : v;
}

template <typename T>
__global__ void __launch_bounds__(kThreads) k_preference_rows(tb_preference_desc d) {
  pdl_entry();
  const int64_t n = blockIdx.x;
  if (n < d.offsets[0] || n >= d.offsets[2 * d.pairs]) return;
  const int64_t t = d.targets[n];
  const float scale = (float)d.scale;
  RowStats s{0.0f, 0.0f};
  float logp = 0.0f;
  if (t >= 0) {
    const T* z = (const T*)d.logits + n * d.logits_stride;
    s = row_stats(z, d.vocab, scale);
    if (s.sum != 0.0f) logp = t < d.vocab ? logp_of(to_f32(z[t]), s, scale) : NAN;
  }
  if (threadIdx.x == 0) {
    ((RowStats*)d.workspace)[n] = s;
    d.logp[n] = logp;
  }
}

__global__ void __launch_bounds__(1024) k_preference_pairs(tb_preference_desc d) {
  pdl_entry();
  __shared__ double terms[32];
  const int lane = threadIdx.x % 32, warp = threadIdx.x / 32;
  const RowStats* stats = (const RowStats*)d.workspace;
  float* slopes = (float*)(stats + d.rows);
  double total = 0;
  for (int64_t i = warp; i < d.pairs; i += 32) {
    double ratio[2];
    int64_t lo[2], hi[2];
    for (int k = 0; k < 2; ++k) {
      const int64_t s = i + k * d.pairs;
      lo[k] = clamp_row(d.offsets[s], d.rows);
      hi[k] = clamp_row(d.offsets[s + 1], d.rows);
      double r = 0;
      for (int64_t n = lo[k] + lane; n < hi[k]; n += 32)
        if (stats[n].sum != 0.0f) r += (double)d.logp[n] - (double)d.ref_logp[n];
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) r += __shfl_xor_sync(~0u, r, o);
      ratio[k] = r;
      if (lane == 0) d.ratios[s] = (float)r;
    }
    const double w = d.weights ? (double)d.weights[i] : 1.0 / (double)d.pairs;
    const double m = d.beta * (ratio[0] - ratio[1]), e = exp(-fabs(m));
    const double soft = log1p(e);  // -log sigmoid(|m|)
    const double lose = m >= 0 ? e / (1 + e) : 1 / (1 + e);  // sigmoid(-m)
    const double yes = m >= 0 ? soft : soft - m, no = m >= 0 ? soft + m : soft;
    // a share of 0 adds nothing, whatever it would multiply
    total += w * ((1 - d.smoothing) * yes + (d.smoothing > 0 ? d.smoothing * no : 0.0));
    const float slope = (float)(w * d.beta * (d.smoothing * (1 - lose) - (1 - d.smoothing) * lose));
    for (int k = 0; k < 2; ++k)
      for (int64_t n = lo[k] + lane; n < hi[k]; n += 32) slopes[n] = k ? -slope : slope;
  }
  if (lane == 0) terms[warp] = total;
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int w = 1; w < 32; ++w) total += terms[w];
    d.loss[0] = (float)total;
  }
}

template <typename T>
__global__ void __launch_bounds__(kThreads) k_preference_gradient(tb_preference_desc d) {
  pdl_entry();
  const int64_t n = blockIdx.x;
  if (n < d.offsets[0] || n >= d.offsets[2 * d.pairs]) return;
  const RowStats s = ((const RowStats*)d.workspace)[n];
  const float slope = ((const float*)((const RowStats*)d.workspace + d.rows))[n];
  const int64_t t = d.targets[n];
  row_gradient((const T*)d.logits + n * d.logits_stride, (T*)d.gradient + n * d.gradient_stride,
               d.vocab, (float)d.scale, s, t, t < d.vocab ? slope : NAN, s.sum == 0.0f);
}

const char* check_logits(int64_t element, int64_t rows, int64_t vocab, int64_t stride, double scale,
                         const void* logits) {
  if (element != TB_ELEMENT_F32 && element != TB_ELEMENT_BF16) return "unknown element type";
  if (!extents_fit({rows, vocab}) || !extents_fit({rows, stride}) || rows > INT32_MAX)
    return "extents out of range";
  if (rows > 0 && vocab < 1) return "an empty vocabulary";
  if (!(scale > 0) || scale > 3e38 || (float)scale == 0.0f) return "scale is positive and finite";
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

int token_logp(int64_t element, const void* logits, int64_t stride, const int32_t* targets,
               int64_t rows, int64_t vocab, double scale, float* logp, void* stream) {
  OperatorCall call("tb_token_logp", stream);
  if (const char* why = check_logits(element, rows, vocab, stride, scale, logits))
    return call.invalid(why);
  if (rows > 0 && !words_ok({targets, logp})) return call.invalid("a row array is NULL or unaligned");
  if (const int code = call.ready()) return code;
  if (rows == 0) return TB_OK;
  const dim3 grid((unsigned)rows), block(kThreads);
  return call.finish(
      element == TB_ELEMENT_F32
          ? launch_pdl(k_token_logp<float>, grid, block, 0, call.stream(), (const float*)logits,
                       stride, targets, vocab, (float)scale, logp)
          : launch_pdl(k_token_logp<bf16>, grid, block, 0, call.stream(), (const bf16*)logits,
                       stride, targets, vocab, (float)scale, logp));
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
    e = launch_pdl(d.element == TB_ELEMENT_F32 ? k_policy<float> : k_policy<bf16>,
                   dim3((unsigned)d.rows), dim3(kThreads), 0, call.stream(), d);
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
  if (!words_ok({d.loss, d.ratios, d.offsets}) || !aligned_to(d.weights, 4) ||
      (d.rows > 0 && !words_ok({d.targets, d.ref_logp, d.logp})))
    return call.invalid("a row array is NULL or unaligned");
  if (tb_preference_workspace(d.rows) > 0) {
    if (!d.workspace || d.workspace_bytes < tb_preference_workspace(d.rows))
      return call.invalid("the workspace is too small");
    if (!aligned_to(d.workspace, 16)) return call.invalid("the workspace is not 16-byte aligned");
  }
  if (const int code = call.ready()) return code;
  const bool f32 = d.element == TB_ELEMENT_F32;
  const dim3 grid((unsigned)d.rows), block(kThreads);
  cudaError_t e = cudaSuccess;
  if (d.rows > 0)
    e = launch_pdl(f32 ? k_preference_rows<float> : k_preference_rows<bf16>, grid, block, 0,
                   call.stream(), d);
  if (e == cudaSuccess) e = launch_pdl(k_preference_pairs, dim3(1), dim3(1024), 0, call.stream(), d);
  if (e == cudaSuccess && d.rows > 0 && d.gradient)
    e = launch_pdl(f32 ? k_preference_gradient<float> : k_preference_gradient<bf16>, grid, block, 0,
                   call.stream(), d);
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
extern "C" int64_t tb_preference_workspace(int64_t rows) { return rows > 0 ? rows * 12 : 0; }
