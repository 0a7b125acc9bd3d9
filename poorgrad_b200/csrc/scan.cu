// scan.cu -- the gated linear recurrence h_t = a_t h_{t-1} + b_t over time, per channel and
// sequence, and its backward pass.
#include "operators.h"

namespace tb {
namespace {

struct Gate {
  float a, b;  // sigmoid and 1 - sigmoid
};
// Both from one exponential of -|g|, so neither loses bits where it is small.
__device__ __forceinline__ Gate sigmoid_pair(float g) {
  const float e = __expf(-fabsf(g));
  const float r = __fdividef(1.0f, 1.0f + e);
  const float s = e * r;
  return g >= 0 ? Gate{r, s} : Gate{s, r};
}

struct Span {
  int64_t first, last;  // rows of the sequence: [first, last)
};
// Offsets are data: whatever they hold, the span lies within the rows.
__device__ __forceinline__ Span sequence_span(const int32_t* offsets, int64_t s, int64_t length) {
  if (!offsets) return {0, length};
  const int64_t lo = min(max((int64_t)offsets[s], (int64_t)0), length);
  const int64_t hi = min(max((int64_t)offsets[s + 1], lo), length);
  return {lo, hi};
}

// One thread per sequence and channel walks the sequence.
template <typename T, int FORM>
__global__ void k_scan_serial(tb_scan_desc d) {
  pdl_entry();
  const int64_t tiles = (d.channels + blockDim.x - 1) / blockDim.x;
  const int64_t c = blockIdx.x % tiles * blockDim.x + threadIdx.x, s = blockIdx.x / tiles;
  if (c >= d.channels) return;
  const int64_t row = d.sequences ? 0 : s;
  const T* gate = (const T*)d.gate + row * d.gate_strides[0] + c;
  const T* x = (const T*)d.x + row * d.x_strides[0] + c;
  T* h = (T*)d.h + row * d.h_strides[0] + c;
  const Span span = sequence_span(d.offsets, s, d.length);
  float state = d.state ? d.state[s * d.channels + c] : 0.0f;
  for (int64_t t = span.first; t < span.last; ++t) {
    const float g = to_f32(gate[t * d.gate_strides[1]]), v = to_f32(x[t * d.x_strides[1]]);
    if (FORM == TB_SCAN_SIGMOID) {
      const Gate p = sigmoid_pair(g);
      state = p.a * state + p.b * v;
    } else {
      state = g * state + v;
    }
    h[t * d.h_strides[1]] = from_f32<T>(state);
  }
  if (d.final_state) d.final_state[s * d.channels + c] = state;
}

template <typename T, int FORM>
__global__ void k_scan_serial_backward(tb_scan_desc d) {
  pdl_entry();
  const int64_t tiles = (d.channels + blockDim.x - 1) / blockDim.x;
  const int64_t c = blockIdx.x % tiles * blockDim.x + threadIdx.x, s = blockIdx.x / tiles;
  if (c >= d.channels) return;
  const int64_t row = d.sequences ? 0 : s;
  const T* gate = (const T*)d.gate + row * d.gate_strides[0] + c;
  const T* x = (const T*)d.x + row * d.x_strides[0] + c;
  const T* h = (const T*)d.h + row * d.h_strides[0] + c;
  const T* dh = (const T*)d.dh + row * d.dh_strides[0] + c;
  T* dgate = (T*)d.dgate + row * d.dgate_strides[0] + c;
  T* dx = (T*)d.dx + row * d.dx_strides[0] + c;
  const Span span = sequence_span(d.offsets, s, d.length);
  const float state = d.state ? d.state[s * d.channels + c] : 0.0f;
  float carry = d.dfinal ? d.dfinal[s * d.channels + c] : 0.0f;  // a_{t+1} g_{t+1}
  for (int64_t t = span.last - 1; t >= span.first; --t) {
    const float g = to_f32(dh[t * d.dh_strides[1]]) + carry;
    const float before = t > span.first ? to_f32(h[(t - 1) * d.h_strides[1]]) : state;
    float a = to_f32(gate[t * d.gate_strides[1]]), da, dv;
    if (FORM == TB_SCAN_SIGMOID) {
      const Gate p = sigmoid_pair(a);
      a = p.a;
      da = g * (before - to_f32(x[t * d.x_strides[1]])) * p.a * p.b;
      dv = g * p.b;
    } else {
      da = g * before;
      dv = g;
    }
    carry = a * g;
    dgate[t * d.dgate_strides[1]] = from_f32<T>(da);
    dx[t * d.dx_strides[1]] = from_f32<T>(dv);
  }
  if (d.dstate) d.dstate[s * d.channels + c] = carry;
}

bool strides_ok(const tb_scan_desc& d, const int64_t s[2], bool written) {
  if (!extents_fit({s[0]}) || !extents_fit({s[1]})) return false;
  if (!written) return true;
  return (d.length <= 1 || s[1] >= d.channels) && (d.batch <= 1 || s[0] >= d.channels);
}

const char* check(const tb_scan_desc& d, bool backward) {
  if (d.element != TB_ELEMENT_F32 && d.element != TB_ELEMENT_BF16) return "unknown element type";
  if (d.form != TB_SCAN_DIRECT && d.form != TB_SCAN_SIGMOID) return "unknown form";
  if (!extents_fit({d.batch, d.length, d.channels}) || d.length > INT32_MAX ||
      !extents_fit({d.sequences, d.channels}) || d.sequences > INT32_MAX)
    return "extents out of range";
  if (d.sequences ? !d.offsets || d.batch != 1 : d.offsets != nullptr)
    return "packed sequences come with offsets and a batch of 1";
  const bool reads_x = !backward || d.form == TB_SCAN_SIGMOID;
  if (!strides_ok(d, d.gate_strides, false) || (reads_x && !strides_ok(d, d.x_strides, false)) ||
      !strides_ok(d, d.h_strides, !backward) ||
      (backward && (!strides_ok(d, d.dh_strides, false) || !strides_ok(d, d.dgate_strides, true) ||
                    !strides_ok(d, d.dx_strides, true))))
    return "strides are negative, too large, or let written rows overlap";
  if (d.batch * d.length * d.channels > 0) {
    if (!d.gate || (reads_x && !d.x) || !d.h || (backward && (!d.dh || !d.dgate || !d.dx)))
      return "a required array is NULL";
  }
  const int64_t size = d.element == TB_ELEMENT_F32 ? 4 : 2;
  for (const void* p : {d.gate, d.x, (const void*)d.h, d.dh, (const void*)d.dgate, (const void*)d.dx})
    if (!aligned_to(p, size)) return "an array is not aligned to its elements";
  for (const void* p : {(const void*)d.offsets, (const void*)d.state, (const void*)d.final_state,
                        (const void*)d.dfinal, (const void*)d.dstate})
    if (!aligned_to(p, 4)) return "an array is not aligned to its elements";
  return nullptr;
}

template <typename T, int FORM>
cudaError_t enqueue(const tb_scan_desc& d, bool backward, cudaStream_t stream) {
  const int64_t count = d.sequences ? d.sequences : d.batch;
  const int64_t blocks = (d.channels + 127) / 128 * count;
  if (blocks > INT32_MAX) return cudaErrorInvalidConfiguration;
  const dim3 grid((unsigned)blocks);
  return launch_pdl(backward ? k_scan_serial_backward<T, FORM> : k_scan_serial<T, FORM>, grid,
                    dim3(128), 0, stream, d);
}

int scan_call(const char* name, const tb_scan_desc* desc, void* stream, bool backward) {
  OperatorCall call(name, stream);
  if (!desc) return call.invalid("no request");
  const tb_scan_desc d = *desc;
  if (const char* why = check(d, backward)) return call.invalid(why);
  if (const int code = call.ready()) return code;
  if (d.channels == 0 || (d.sequences ? d.sequences : d.batch) == 0) return TB_OK;
  cudaError_t e;
  if (d.element == TB_ELEMENT_F32)
    e = d.form == TB_SCAN_DIRECT ? enqueue<float, TB_SCAN_DIRECT>(d, backward, call.stream())
                                 : enqueue<float, TB_SCAN_SIGMOID>(d, backward, call.stream());
  else
    e = d.form == TB_SCAN_DIRECT ? enqueue<bf16, TB_SCAN_DIRECT>(d, backward, call.stream())
                                 : enqueue<bf16, TB_SCAN_SIGMOID>(d, backward, call.stream());
  return call.finish(e);
}

}  // namespace
}  // namespace tb

extern "C" int tb_gated_scan(const tb_scan_desc* desc, void* stream) {
  return tb::guarded([&] { return tb::scan_call("tb_gated_scan", desc, stream, false); });
}
extern "C" int tb_gated_scan_backward(const tb_scan_desc* desc, void* stream) {
  return tb::guarded([&] { return tb::scan_call("tb_gated_scan_backward", desc, stream, true); });
}
