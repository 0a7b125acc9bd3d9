// scan.cu -- the gated linear recurrence h_t = a_t h_{t-1} + b_t over time, per channel and
// sequence, and its backward pass.
#include <cooperative_groups.h>

#include <algorithm>

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

// How a call is cut: `ranks` blocks of a cluster take consecutive spans of kWarps * L steps, over
// and over, and `parts` such clusters the consecutive parts of the time axis.  With several parts
// a first launch leaves each part's affine map in the workspace, and the second starts each part
// from the maps before it.
struct Cut {
  int ranks, tiles, parts;
  int64_t part_steps;
  Affine* maps;  // [batch][parts][channels], parts > 1
  int* begins;   // [batch][parts]
};

enum { kWhole = 0, kMaps = 1, kFromMaps = 2 };

// The recurrence, or with BACK the gradients, walked backwards: there the carried value is
// c_t = a_t (dh_t + c_{t+1}), g_t = dh_t + c_{t+1}.
//
// A block takes 32 V channels and kWarps * L steps at a time, one warp L consecutive steps, one
// lane V channels: everything is loaded once, at the start, and stays in registers.  Each warp
// reduces its steps to one affine map per channel; the maps are exchanged through shared memory
// (and between the blocks of a cluster), every warp then knows the value carried into its steps
// and walks them again to write the outputs.
template <typename T, int V, int L, int FORM, bool BACK, int PASS>
struct Scan {
  typedef Lane<T, V> Row;
  static constexpr bool kReadsX = FORM == TB_SCAN_SIGMOID || !BACK;
  const tb_scan_desc& d;
  const int lane, warp;
  const int64_t b, c;
  const bool in;  // this lane's channels exist
  const float* entry_state;
  float* exit_state;
  Row g[L], u[L], before[L], xs[L];  // u: x, or dh backwards
  float a[L][V], add[L][V];

  __device__ Scan(const tb_scan_desc& d, int64_t b, int64_t c)
      : d(d), lane(threadIdx.x % 32), warp(threadIdx.x / 32), b(b), c(c), in(c < d.channels),
        entry_state(BACK ? d.dfinal : d.state), exit_state(BACK ? d.dstate : d.final_state) {}

  // A row pointer walks with the steps.
  template <typename P>
  __device__ __forceinline__ P* at(P* base, const int64_t s[2], int64_t t) const {
    return base + b * s[0] + t * s[1] + c;
  }

  // ALL: every step lies within the array and its channels exist.
  template <bool ALL>
  __device__ __forceinline__ void load(int64_t first) {
    const int64_t t0 = BACK ? d.length - 1 - first : first, way = BACK ? -1 : 1;
    const T* pg = at((const T*)d.gate, d.gate_strides, t0);
    const T* pu = BACK ? at((const T*)d.dh, d.dh_strides, t0) : at((const T*)d.x, d.x_strides, t0);
    const T* ph = at((const T*)d.h, d.h_strides, t0 - 1);
    const T* px = at((const T*)d.x, d.x_strides, t0);
    const int64_t sg = way * d.gate_strides[1], su = way * (BACK ? d.dh_strides : d.x_strides)[1];
    const int64_t sh = -d.h_strides[1], sx = -d.x_strides[1];
    const int64_t left = d.length - first;
#pragma unroll
    for (int i = 0; i < L; ++i) {
      const bool here = ALL || (in && i < left);
      if (!ALL) g[i] = u[i] = before[i] = xs[i] = Row{};
      if (here) {
        g[i] = *(const Row*)(pg + i * sg);
        u[i] = *(const Row*)(pu + i * su);
        if (BACK && PASS != kMaps) {
          // the row before the first is the state's
          if (ALL ? i < L - 1 || t0 >= L : t0 - i > 0) before[i] = *(const Row*)(ph + i * sh);
          else before[i] = Row{};
          if (kReadsX) xs[i] = *(const Row*)(px + i * sx);
        }
      }
    }
  }

  // a and the added term of each step (kept where the outputs do not work them out again), and
  // the steps' map.  A step that enters a sequence holds the entry state's part in its term, so
  // that state is read before any other state is written.  What rows outside every sequence hold
  // goes nowhere: the next row inside one enters it.
  template <bool MARKED>
  __device__ __forceinline__ void reduce(const Marks& m, Affine map[V]) {
#pragma unroll
    for (int v = 0; v < V; ++v) map[v] = {1.0f, 0.0f};
#pragma unroll
    for (int i = 0; i < L; ++i) {
      const bool enters = MARKED && (m.enters >> i & 1);
      const int64_t state = enters ? (int64_t)__shfl_sync(~0u, m.sequence, i) * d.channels + c : 0;
#pragma unroll
      for (int v = 0; v < V; ++v) {
        float av = to_f32(g[i].v[v]), bv = to_f32(u[i].v[v]);
        if (FORM == TB_SCAN_SIGMOID) {
          const Gate p = sigmoid_pair(av);
          av = p.a;
          if (!BACK) bv *= p.b;
        }
        if (enters) {
          const float e = entry_state && in ? entry_state[state + v] : 0.0f;
          bv = BACK ? bv + e : fmaf(av, e, bv);
          map[v].H = BACK ? av * bv : bv;
        } else {
          map[v].H = BACK ? av * (map[v].H + bv) : fmaf(av, map[v].H, bv);
        }
        map[v].A *= av;
        if (!BACK) a[i][v] = av;
        add[i][v] = bv;
      }
    }
  }

  // ALL as in load(); MARKED: some step enters or leaves a sequence or lies outside all of them.
  template <bool ALL, bool MARKED>
  __device__ __forceinline__ void write(const Marks& m, int64_t first, float value[V]) {
    const int64_t t0 = BACK ? d.length - 1 - first : first, way = BACK ? -1 : 1;
    T* p1 = BACK ? at((T*)d.dgate, d.dgate_strides, t0) : at((T*)d.h, d.h_strides, t0);
    T* p2 = at((T*)d.dx, d.dx_strides, t0);
    const int64_t s1 = way * (BACK ? d.dgate_strides : d.h_strides)[1], s2 = -d.dx_strides[1];
#pragma unroll
    for (int i = 0; i < L; ++i) {
      const bool enters = MARKED && (m.enters >> i & 1), leaves = MARKED && (m.leaves >> i & 1);
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
            const float gb = gt * p.b;
            out.v[v] = from_f32<T>(gb * p.a * (prior - to_f32(xs[i].v[v])));
            out2.v[v] = from_f32<T>(gb);
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
      if ((ALL || in) && (!MARKED || (m.inside >> i & 1))) {
        *(Row*)(p1 + i * s1) = out;
        if (BACK) *(Row*)(p2 + i * s2) = out2;
      }
      if (leaves && in && exit_state)
#pragma unroll
        for (int v = 0; v < V; ++v) exit_state[state + v] = value[v];
    }
  }
};

template <typename T, int V, int L, int FORM, bool BACK, int PASS>
__global__ void __launch_bounds__(kWarps * 32, 2) k_scan(tb_scan_desc d, Cut cut) {
  pdl_entry();
  __shared__ Affine maps[2][kWarps][V][32];
  __shared__ int begins[2][kWarps];
  __shared__ Affine rank_maps[2][8][V][32];
  __shared__ int rank_begins[2][8];
  const int lane = threadIdx.x % 32, warp = threadIdx.x / 32, ranks = cut.ranks;
  const int rank = blockIdx.x % ranks, tile = blockIdx.x / ranks % cut.tiles;
  const int64_t part = (int64_t)blockIdx.x / ranks / cut.tiles % cut.parts;
  const int64_t b = (int64_t)blockIdx.x / ranks / cut.tiles / cut.parts;
  Scan<T, V, L, FORM, BACK, PASS> s(d, b, (int64_t)(tile * 32 + lane) * V);

  // sequences without a step hand their entry state on
  if (PASS != kMaps && s.exit_state && rank == 0 && part == 0 && (d.sequences || d.length == 0)) {
    const int64_t count = d.sequences ? d.sequences : 1;
    for (int64_t i = warp; i < count; i += kWarps) {
      if (d.sequences && clamped_offset(d, i + 1) > clamped_offset(d, i)) continue;
      const int64_t at = (d.sequences ? i : b) * d.channels + s.c;
      if (s.in)
        for (int v = 0; v < V; ++v) s.exit_state[at + v] = s.entry_state ? s.entry_state[at + v] : 0.0f;
    }
  }

  float carry[V] = {};
  if (PASS == kFromMaps && s.in)
    for (int64_t p = 0; p < part; ++p) {
      const Affine* f = cut.maps + (b * cut.parts + p) * d.channels + s.c;
      const bool begun = cut.begins[b * cut.parts + p];
#pragma unroll
      for (int v = 0; v < V; ++v) carry[v] = apply(f[v], begun, carry[v]);
    }
  Affine whole[V];  // the part's map so far
#pragma unroll
  for (int v = 0; v < V; ++v) whole[v] = {1.0f, 0.0f};
  bool whole_begins = false;

  int parity = 0;
  const int64_t from = part * cut.part_steps, to = min(from + cut.part_steps, d.length);
  for (int64_t base = from; base < to; base += (int64_t)ranks * kWarps * L, parity ^= 1) {
    const int64_t first = base + (int64_t)(rank * kWarps + warp) * L;
    // a part is a whole number of spans, so that no step belongs to two
    const bool all = s.in && first + L <= d.length;
    const bool uniform = __all_sync(~0u, all);
    if (uniform) s.template load<true>(first); else s.template load<false>(first);
    const Marks m = marks_of<L, BACK>(d, b, first);
    const bool marked = m.enters | m.leaves | (m.inside != (1u << L) - 1);
    Affine map[V];
    if (m.enters) s.template reduce<true>(m, map); else s.template reduce<false>(m, map);
#pragma unroll
    for (int v = 0; v < V; ++v) maps[parity][warp][v][lane] = map[v];
    if (lane == 0) begins[parity][warp] = m.enters != 0;
    __syncthreads();
    if (ranks > 1 || PASS == kMaps) {
      // this block's map
      Affine block[V];
      bool any = false;
#pragma unroll
      for (int v = 0; v < V; ++v) block[v] = {1.0f, 0.0f};
#pragma unroll
      for (int w = 0; w < kWarps; ++w) {
        const bool begun = begins[parity][w];
        any |= begun;
#pragma unroll
        for (int v = 0; v < V; ++v) {
          const Affine f = maps[parity][w][v][lane];
          block[v] = {block[v].A * f.A, apply(f, begun, block[v].H)};
        }
      }
      if (PASS == kMaps) {
#pragma unroll
        for (int v = 0; v < V; ++v)
          whole[v] = {whole[v].A * block[v].A, apply(block[v], any, whole[v].H)};
        whole_begins |= any;
        continue;
      }
      cg::cluster_group cluster = cg::this_cluster();
      if (warp < ranks) {  // to every block of the cluster
        Affine* there = cluster.map_shared_rank(&rank_maps[parity][rank][0][0], warp);
#pragma unroll
        for (int v = 0; v < V; ++v) there[v * 32 + lane] = block[v];
        if (lane == 0) *cluster.map_shared_rank(&rank_begins[parity][rank], warp) = any;
      }
      cluster.sync();
    }
    // the value carried into this warp's steps, and past all blocks' steps
    float value[V];
#pragma unroll
    for (int v = 0; v < V; ++v) value[v] = carry[v];
    if (ranks > 1)
      for (int r = 0; r < ranks; ++r) {
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
    if (uniform && !marked) s.template write<true, false>(m, first, value);
    else s.template write<false, true>(m, first, value);
  }
  if (PASS == kMaps && warp == 0) {
    if (s.in)
#pragma unroll
      for (int v = 0; v < V; ++v)
        cut.maps[(b * cut.parts + part) * d.channels + s.c + v] = whole[v];
    if (lane == 0 && tile == 0) cut.begins[b * cut.parts + part] = whole_begins;
  }
}

// Into how many parts the time axis of a call is cut, each part two launches' work: one map of it,
// then its outputs.  1 where the columns alone, or a cluster over each, fill the GPU.
constexpr int64_t kMaxParts = 64;
int parts_of(int64_t columns, int64_t spans) {
  if (columns >= 2 * 148 || (columns * 8 >= 2 * 148 && spans <= 16)) return 1;
  return (int)std::max<int64_t>(1, std::min({kMaxParts, (spans + 1) / 2, 8 * 148 / columns}));
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
  if (d.workspace) {
    if (d.workspace_bytes < tb_gated_scan_workspace(d.batch, d.length, d.channels))
      return "the workspace is too small";
    if (!aligned_to(d.workspace, 16)) return "the workspace is not 16-byte aligned";
  }
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

template <typename T, int V, int L, int FORM, bool BACK, int PASS>
cudaError_t launch(const tb_scan_desc& d, const Cut& cut, cudaStream_t stream) {
  const int64_t blocks = d.batch * cut.parts * cut.tiles * cut.ranks;
  if (blocks > INT32_MAX) return cudaErrorInvalidConfiguration;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)blocks);
  cfg.blockDim = dim3(kWarps * 32);
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = cut.ranks;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = pdl_enabled() ? 2 : 1;
  return cudaLaunchKernelEx(&cfg, k_scan<T, V, L, FORM, BACK, PASS>, d, cut);
}

template <typename T, int V, int L, int FORM, bool BACK>
cudaError_t enqueue(const tb_scan_desc& d, cudaStream_t stream) {
  const int64_t span = kWarps * L;
  Cut cut = {};
  cut.tiles = (int)((d.channels + 32 * V - 1) / (32 * V));
  cut.ranks = cut.parts = 1;
  cut.part_steps = std::max<int64_t>(d.length, 1);
  const int64_t columns = d.batch * cut.tiles, spans = (d.length + span - 1) / span;
  // a state that is read and written in one call is read before it is written only within a launch
  const bool carries = BACK ? d.dstate && d.dstate == d.dfinal : d.final_state && d.final_state == d.state;
  if (d.workspace && columns * spans > 0 && !carries) cut.parts = parts_of(columns, spans);
  if (cut.parts > 1) {
    cut.part_steps = (spans + cut.parts - 1) / cut.parts * span;
    cut.parts = (int)((d.length + cut.part_steps - 1) / cut.part_steps);
    cut.maps = (Affine*)d.workspace;
    cut.begins = (int*)(cut.maps + d.batch * cut.parts * d.channels);
    const cudaError_t e = launch<T, V, L, FORM, BACK, kMaps>(d, cut, stream);
    return e != cudaSuccess ? e : launch<T, V, L, FORM, BACK, kFromMaps>(d, cut, stream);
  }
  while (cut.ranks < 8 && columns * cut.ranks < 2 * 148 && cut.ranks < spans) cut.ranks *= 2;
  return launch<T, V, L, FORM, BACK, kWhole>(d, cut, stream);
}

template <typename T, int FORM, bool BACK>
cudaError_t enqueue_form(const tb_scan_desc& d, cudaStream_t stream) {
  constexpr int64_t kPair = 4 / sizeof(T);  // channels in 4 bytes
  if (kPair == 1 || lanes_fit(d, BACK, sizeof(T), 4))
    // the backward pass of the sigmoid form holds four arrays: 16 pairs of each would spill
    return enqueue<T, kPair, BACK && FORM == TB_SCAN_SIGMOID && kPair == 2 ? 8 : 16, FORM, BACK>(d, stream);
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

int64_t scan_workspace(int64_t batch, int64_t length, int64_t channels) {
  if (!extents_fit({batch, length, channels}) || batch * length * channels == 0) return 0;
  // the widest blocks make the fewest columns, the shortest spans the most parts
  const int64_t parts = parts_of(batch * ((channels + 63) / 64), (length + kWarps * 8 - 1) / (kWarps * 8));
  return parts > 1 ? (batch * parts * (channels * (int64_t)sizeof(Affine) + 4) + 15) / 16 * 16 : 0;
}
}  // namespace tb

extern "C" int tb_gated_scan(const tb_scan_desc* desc, void* stream) {
  return tb::guarded([&] { return tb::scan_call("tb_gated_scan", desc, stream, false); });
}
extern "C" int tb_gated_scan_backward(const tb_scan_desc* desc, void* stream) {
  return tb::guarded([&] { return tb::scan_call("tb_gated_scan_backward", desc, stream, true); });
}
extern "C" int64_t tb_gated_scan_workspace(int64_t batch, int64_t length, int64_t channels) {
  return tb::scan_workspace(batch, length, channels);
}
