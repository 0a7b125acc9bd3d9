// scan.cu -- the gated linear recurrence h_t = a_t h_{t-1} + b_t over time, per channel and
// sequence, and its backward pass.
#include <cooperative_groups.h>

#include "operators.h"

namespace tb {
namespace {

namespace cg = cooperative_groups;

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

// V consecutive channels of one row, as loaded.
template <typename T, int V>
struct alignas(sizeof(T) * V) Lane {
  T v[V];
};

__device__ __forceinline__ int64_t clamped_offset(const tb_scan_desc& d, int64_t s) {
  // offsets are data: whatever they hold, rows stay within the array
  return min(max((int64_t)d.offsets[s], (int64_t)0), d.length);
}

// Which of a warp's L rows, in the order they are walked, begin a walk over a sequence, end one,
// and belong to a sequence at all; and each row's sequence (its state row), held by lane i.
struct Marks {
  unsigned enters, leaves, inside;
  int sequence;
};
template <int L, bool BACK>
__device__ __forceinline__ Marks marks_of(const tb_scan_desc& d, int64_t b, int64_t first) {
  const int lane = threadIdx.x % 32;
  const int64_t step = first + lane, t = BACK ? d.length - 1 - step : step;
  const bool here = lane < L && step < d.length;
  bool starts, ends, inside = here;
  int sequence = (int)b;
  if (d.sequences == 0) {
    starts = t == 0;
    ends = t == d.length - 1;
  } else {
    // the last sequence that starts at or before t
    int64_t lo = 0, hi = d.sequences;
    while (hi - lo > 1) {
      const int64_t mid = (lo + hi) / 2;
      if (here && d.offsets[mid] <= t) lo = mid; else hi = mid;
    }
    const int64_t from = d.offsets[lo], to = d.offsets[lo + 1];
    sequence = (int)lo;
    inside = here && from <= t && t < to;
    starts = t == from || t == 0;
    ends = t == to - 1 || t == d.length - 1;
  }
  Marks m;
  m.sequence = sequence;
  m.inside = __ballot_sync(~0u, inside);
  m.enters = __ballot_sync(~0u, inside && (BACK ? ends : starts));
  m.leaves = __ballot_sync(~0u, inside && (BACK ? starts : ends));
  return m;
}

constexpr int kWarps = 8;

// What a run of steps does to the value v carried into it: v -> A v + H, or H alone where a
// sequence begins inside the run (then v belongs to another sequence and may be anything).
struct Affine {
  float A, H;
};
__device__ __forceinline__ float apply(Affine f, bool begins, float v) {
  return begins ? f.H : fmaf(f.A, v, f.H);
}

// The recurrence, or with BACK the gradients, walked backwards: there the carried value is
// c_t = a_t (dh_t + c_{t+1}), g_t = dh_t + c_{t+1}.
//
// A block takes 32 V channels and kWarps * L steps at a time, one warp L consecutive steps, one
// lane V channels: everything is loaded once, at the start, and stays in registers.  Each warp
// reduces its steps to one affine map per channel; the maps are exchanged through shared memory
// (and between the blocks of a cluster, which take consecutive spans of steps), every warp then
// knows the value carried into its steps and walks them again to write the outputs.
template <typename T, int V, int L, int FORM, bool BACK>
__global__ void __launch_bounds__(kWarps * 32, 2) k_scan(tb_scan_desc d, int ranks, int tiles) {
  pdl_entry();
  __shared__ Affine maps[2][kWarps][V][32];
  __shared__ int begins[2][kWarps];
  __shared__ Affine rank_maps[2][8][V][32];
  __shared__ int rank_begins[2][8];
  const int lane = threadIdx.x % 32, warp = threadIdx.x / 32;
  const int rank = blockIdx.x % ranks, tile = blockIdx.x / ranks % tiles;
  const int64_t b = blockIdx.x / ranks / tiles;
  const int64_t c = (int64_t)(tile * 32 + lane) * V;
  const bool in = c < d.channels;
  typedef Lane<T, V> Row;
  const float* entry_state = BACK ? d.dfinal : d.state;
  float* exit_state = BACK ? d.dstate : d.final_state;

  // sequences without a step hand their entry state on
  if (exit_state && rank == 0 && (d.sequences || d.length == 0)) {
    const int64_t count = d.sequences ? d.sequences : 1;
    for (int64_t i = warp; i < count; i += kWarps) {
      if (d.sequences && clamped_offset(d, i + 1) > clamped_offset(d, i)) continue;
      const int64_t row = d.sequences ? i : b;
      if (in)
        for (int v = 0; v < V; ++v)
          exit_state[row * d.channels + c + v] =
              entry_state ? entry_state[row * d.channels + c + v] : 0.0f;
    }
  }

  const T* gate = (const T*)d.gate + b * d.gate_strides[0] + c;
  const T* x = (const T*)d.x + b * d.x_strides[0] + c;
  const T* hs = (const T*)d.h + b * d.h_strides[0] + c;
  const T* dh = (const T*)d.dh + b * d.dh_strides[0] + c;
  constexpr bool kReadsX = !BACK || FORM == TB_SCAN_SIGMOID;

  float carry[V] = {};
  int parity = 0;
  for (int64_t base = 0; base < d.length; base += (int64_t)ranks * kWarps * L, parity ^= 1) {
    const int64_t first = base + (int64_t)(rank * kWarps + warp) * L;
    Row g[L], u[L], before[L], xs[L];  // u: x, or dh backwards
#pragma unroll
    for (int i = 0; i < L; ++i) {
      const int64_t step = first + i, t = BACK ? d.length - 1 - step : step;
      g[i] = {};
      u[i] = {};
      before[i] = {};
      xs[i] = {};
      if (in && step < d.length) {
        g[i] = *(const Row*)(gate + t * d.gate_strides[1]);
        if (BACK) {
          u[i] = *(const Row*)(dh + t * d.dh_strides[1]);
          if (t > 0) before[i] = *(const Row*)(hs + (t - 1) * d.h_strides[1]);
          if (kReadsX) xs[i] = *(const Row*)(x + t * d.x_strides[1]);
        } else {
          u[i] = *(const Row*)(x + t * d.x_strides[1]);
        }
      }
    }
    const Marks m = marks_of<L, BACK>(d, b, first);

    // The added term of each step, and a where the outputs below do not work it out again (to read
    // it from the loaded gate costs fewer registers).  A step that enters a sequence holds the
    // entry state's part in its term, so that state is read before any other state is written.
    // What rows outside every sequence hold goes nowhere: the next row inside one enters it.
    float a[L][V], add[L][V];
    Affine map[V];
#pragma unroll
    for (int v = 0; v < V; ++v) map[v] = {1.0f, 0.0f};
#pragma unroll
    for (int i = 0; i < L; ++i) {
      const bool enters = m.enters >> i & 1;
#pragma unroll
      for (int v = 0; v < V; ++v) {
        float av = to_f32(g[i].v[v]), bv = to_f32(u[i].v[v]);
        if (FORM == TB_SCAN_SIGMOID) {
          const Gate p = sigmoid_pair(av);
          av = p.a;
          if (!BACK) bv *= p.b;
        }
        if (enters) {
          const int row = __shfl_sync(~0u, m.sequence, i);
          const float e = entry_state && in ? entry_state[(int64_t)row * d.channels + c + v] : 0.0f;
          bv = BACK ? bv + e : fmaf(av, e, bv);
        }
        const float kept = BACK ? map[v].H + bv : fmaf(av, map[v].H, bv);
        map[v].H = BACK ? av * (enters ? bv : kept) : enters ? bv : kept;
        map[v].A *= av;
        if (!BACK) a[i][v] = av;
        add[i][v] = bv;
      }
    }
#pragma unroll
    for (int v = 0; v < V; ++v) maps[parity][warp][v][lane] = map[v];
    if (lane == 0) begins[parity][warp] = m.enters != 0;
    __syncthreads();
    if (ranks > 1) {
      // this block's map, to every block of the cluster
      Affine whole[V];
      bool any = false;
#pragma unroll
      for (int v = 0; v < V; ++v) whole[v] = {1.0f, 0.0f};
#pragma unroll
      for (int w = 0; w < kWarps; ++w) {
        const bool begun = begins[parity][w];
        any |= begun;
#pragma unroll
        for (int v = 0; v < V; ++v) {
          const Affine f = maps[parity][w][v][lane];
          whole[v] = {whole[v].A * f.A, apply(f, begun, whole[v].H)};
        }
      }
      cg::cluster_group cluster = cg::this_cluster();
      if (warp < ranks) {
        Affine* to = cluster.map_shared_rank(&rank_maps[parity][rank][0][0], warp);
#pragma unroll
        for (int v = 0; v < V; ++v) to[v * 32 + lane] = whole[v];
        if (lane == 0) *cluster.map_shared_rank(&rank_begins[parity][rank], warp) = any;
      }
      cluster.sync();
    }
    float value[V];
#pragma unroll
    for (int v = 0; v < V; ++v) value[v] = carry[v];
    // the value carried into this block's steps, and past all blocks' steps
    for (int r = 0; r < ranks && ranks > 1; ++r) {
      const bool begun = rank_begins[parity][r];
#pragma unroll
      for (int v = 0; v < V; ++v) {
        if (r == rank) value[v] = carry[v];
        carry[v] = apply(rank_maps[parity][r][v][lane], begun, carry[v]);
      }
    }
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      const bool begun = begins[parity][w];
#pragma unroll
      for (int v = 0; v < V; ++v) {
        if (ranks == 1) {
          if (w == warp) value[v] = carry[v];
          carry[v] = apply(maps[parity][w][v][lane], begun, carry[v]);
        } else if (w < warp) {
          value[v] = apply(maps[parity][w][v][lane], begun, value[v]);
        }
      }
    }

#pragma unroll
    for (int i = 0; i < L; ++i) {
      const int64_t step = first + i, t = BACK ? d.length - 1 - step : step;
      const bool enters = m.enters >> i & 1, inside = m.inside >> i & 1, leaves = m.leaves >> i & 1;
      const int64_t state = leaves ? (int64_t)__shfl_sync(~0u, m.sequence, i) * d.channels + c : 0;
      Row out, out2;
#pragma unroll
      for (int v = 0; v < V; ++v) {
        if (BACK) {
          const float gt = enters ? add[i][v] : add[i][v] + value[v];
          float prior = to_f32(before[i].v[v]);
          if (leaves) prior = d.state && in ? d.state[state + v] : 0.0f;
          float av = to_f32(g[i].v[v]);
          if (FORM == TB_SCAN_SIGMOID) {
            const Gate p = sigmoid_pair(av);
            av = p.a;
            out.v[v] = from_f32<T>(gt * (prior - to_f32(xs[i].v[v])) * p.a * p.b);
            out2.v[v] = from_f32<T>(gt * p.b);
          } else {
            out.v[v] = from_f32<T>(gt * prior);
            out2.v[v] = from_f32<T>(gt);
          }
          value[v] = av * gt;
        } else {
          value[v] = enters ? add[i][v] : fmaf(a[i][v], value[v], add[i][v]);
          out.v[v] = from_f32<T>(value[v]);
        }
      }
      if (in && inside) {
        if (BACK) {
          *(Row*)((T*)d.dgate + b * d.dgate_strides[0] + c + t * d.dgate_strides[1]) = out;
          *(Row*)((T*)d.dx + b * d.dx_strides[0] + c + t * d.dx_strides[1]) = out2;
        } else {
          *(Row*)((T*)d.h + b * d.h_strides[0] + c + t * d.h_strides[1]) = out;
        }
        if (leaves && exit_state)
#pragma unroll
          for (int v = 0; v < V; ++v) exit_state[state + v] = value[v];
      }
    }
  }
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

// Whether every row of the call's arrays can be read and written `bytes` at a time.
bool lanes_fit(const tb_scan_desc& d, bool backward, int64_t size, int64_t bytes) {
  const struct {
    const void* p;
    const int64_t* s;
    bool used;
  } arrays[] = {{d.gate, d.gate_strides, true}, {d.h, d.h_strides, true},
                {d.x, d.x_strides, !backward || d.form == TB_SCAN_SIGMOID},
                {d.dh, d.dh_strides, backward}, {d.dgate, d.dgate_strides, backward},
                {d.dx, d.dx_strides, backward}};
  if (d.channels * size % bytes) return false;
  for (const auto& a : arrays)
    if (a.used && (!aligned_to(a.p, bytes) || (d.batch > 1 && a.s[0] * size % bytes) ||
                   (d.length > 1 && a.s[1] * size % bytes)))
      return false;
  return true;
}

template <typename T, int V, int L, int FORM, bool BACK>
cudaError_t enqueue(const tb_scan_desc& d, cudaStream_t stream) {
  const int64_t tiles = (d.channels + 32 * V - 1) / (32 * V);
  int ranks = 1;
  while (ranks < 8 && d.batch * tiles * ranks < 2 * 148 && (int64_t)ranks * kWarps * L < d.length)
    ranks *= 2;
  const int64_t blocks = d.batch * tiles * ranks;
  if (blocks > INT32_MAX) return cudaErrorInvalidConfiguration;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)blocks);
  cfg.blockDim = dim3(kWarps * 32);
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = ranks;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = pdl_enabled() ? 2 : 1;
  return cudaLaunchKernelEx(&cfg, k_scan<T, V, L, FORM, BACK>, d, ranks, (int)tiles);
}

template <typename T, int FORM, bool BACK>
cudaError_t enqueue_form(const tb_scan_desc& d, cudaStream_t stream) {
  constexpr int64_t kPair = 4 / sizeof(T);  // channels in 4 bytes
  if (kPair == 1 || lanes_fit(d, BACK, sizeof(T), 4))
    return enqueue<T, kPair, 16, FORM, BACK>(d, stream);
  return enqueue<T, 1, 16, FORM, BACK>(d, stream);
}

template <typename T>
cudaError_t enqueue_type(const tb_scan_desc& d, bool backward, cudaStream_t stream) {
  if (d.form == TB_SCAN_DIRECT)
    return backward ? enqueue_form<T, TB_SCAN_DIRECT, true>(d, stream)
                    : enqueue_form<T, TB_SCAN_DIRECT, false>(d, stream);
  return backward ? enqueue_form<T, TB_SCAN_SIGMOID, true>(d, stream)
                  : enqueue_form<T, TB_SCAN_SIGMOID, false>(d, stream);
}

int scan_call(const char* name, const tb_scan_desc* desc, void* stream, bool backward) {
  OperatorCall call(name, stream);
  if (!desc) return call.invalid("no request");
  const tb_scan_desc d = *desc;
  if (const char* why = check(d, backward)) return call.invalid(why);
  if (const int code = call.ready()) return code;
  if (d.channels == 0 || (d.sequences ? d.sequences : d.batch) == 0) return TB_OK;
  const cudaError_t e = d.element == TB_ELEMENT_F32
                            ? enqueue_type<float>(d, backward, call.stream())
                            : enqueue_type<bf16>(d, backward, call.stream());
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
