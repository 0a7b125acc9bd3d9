// scan.cu -- the gated linear recurrence h_t = a_t h_{t-1} + b_t over time, per channel and
// sequence, and its backward pass g_t = dh_t + a_{t+1} g_{t+1}.
//
// A run of steps maps the value v carried into it to A v + H, and two such maps compose into one, so
// the time axis is cut: a warp takes a few steps of 32 or 64 channels into registers, reduces them to
// their map, learns the value carried into them from the maps before, and walks them again to write.
// Each element is read once and written once, but for calls of few channels and many steps, whose
// parts are reduced by a launch of their own first.
//
// Measured on B200 (bytes moved over time, against a copy's 6.55 TB/s): 16 x 512 x 4096 bf16 direct
// forward 36 us, 5.6 TB/s; 32 x 4096 x 512 bf16 direct forward 74 us, 5.4 TB/s, sigmoid forward 82 us,
// 4.9 TB/s, backward 157 us, 5.1 TB/s; a packed 131072 x 768 bf16 direct forward in two launches 170 us,
// which read 403 MB and read and write 604 MB, both inputs from memory each time.  What bounds it: 31
// (direct forward) to 94 (sigmoid backward) instructions a pair of elements, issued by the sixteen warps a
// SM that 128 registers each leave (issue slots half busy, the rest waiting for rows and for the exchange
// of maps).  Copies through shared memory several runs ahead were slower (16 x 512 x 4096: 44 us), and so
// were lanes of four bf16 (8 x 1024 x 768: 25 us for 15).
#include <cooperative_groups.h>

#include <algorithm>
#include <type_traits>

#include "operators.h"

namespace tb {
namespace {

namespace cg = cooperative_groups;

// One lane's V channels of a row as f32, V = 1 or 2.  Pairs use the packed f32x2 instructions: the
// scan issues some 15 to 25 instructions an element, and that, not memory, bounds it otherwise.
template <int V>
struct Vec;
template <>
struct Vec<1> {
  float x;
  __device__ __forceinline__ float get(int) const { return x; }
  __device__ __forceinline__ void set(int, float v) { x = v; }
};
template <>
struct Vec<2> {
  float2 x;
  __device__ __forceinline__ float get(int i) const { return i ? x.y : x.x; }
  __device__ __forceinline__ void set(int i, float v) { (i ? x.y : x.x) = v; }
};
template <int V>
__device__ __forceinline__ Vec<V> splat(float v) {
  Vec<V> r;
#pragma unroll
  for (int i = 0; i < V; ++i) r.set(i, v);
  return r;
}
__device__ __forceinline__ Vec<1> operator*(Vec<1> a, Vec<1> b) { return {a.x * b.x}; }
__device__ __forceinline__ Vec<1> operator+(Vec<1> a, Vec<1> b) { return {a.x + b.x}; }
__device__ __forceinline__ Vec<1> fma(Vec<1> a, Vec<1> b, Vec<1> c) { return {fmaf(a.x, b.x, c.x)}; }
__device__ __forceinline__ Vec<2> operator*(Vec<2> a, Vec<2> b) { return {mul2(a.x, b.x)}; }
__device__ __forceinline__ Vec<2> operator+(Vec<2> a, Vec<2> b) { return {add2(a.x, b.x)}; }
__device__ __forceinline__ Vec<2> fma(Vec<2> a, Vec<2> b, Vec<2> c) { return {fma2(a.x, b.x, c.x)}; }
template <int V>
__device__ __forceinline__ Vec<V> select(bool p, Vec<V> a, Vec<V> b) {
  Vec<V> r;
#pragma unroll
  for (int i = 0; i < V; ++i) r.set(i, p ? a.get(i) : b.get(i));
  return r;
}

// V channels of one row as stored.
template <typename T, int V>
struct Raw;
template <>
struct Raw<float, 1> {
  typedef float type;
  static __device__ __forceinline__ Vec<1> read(float r) { return {r}; }
  static __device__ __forceinline__ float made(Vec<1> v) { return v.x; }
};
template <>
struct Raw<float, 2> {
  typedef float2 type;
  static __device__ __forceinline__ Vec<2> read(float2 r) { return {r}; }
  static __device__ __forceinline__ float2 made(Vec<2> v) { return v.x; }
};
template <>
struct Raw<bf16, 1> {
  typedef unsigned short type;
  static __device__ __forceinline__ Vec<1> read(unsigned short r) {
    return {__uint_as_float((unsigned)r << 16)};
  }
  static __device__ __forceinline__ unsigned short made(Vec<1> v) {
    return __bfloat16_as_ushort(__float2bfloat16_rn(v.x));
  }
};
template <>
struct Raw<bf16, 2> {
  typedef unsigned type;
  static __device__ __forceinline__ Vec<2> read(unsigned r) { return {unpack_bf16(r)}; }
  static __device__ __forceinline__ unsigned made(Vec<2> v) { return pack_bf16(v.x); }
};

// The bare instructions: the intrinsics around them also serve denormals, which do not matter here
// and cost half of the instructions of a sigmoid.  The argument of the power of two is one rounded
// product, so that 1 - a, where it is small, has a relative error of up to 2^-24 |g| besides the
// instructions' own, as of a gate that is off by one rounding (6e-7 at gates of 10, where expf would leave
// 1e-7).
__device__ __forceinline__ float ex2_approx(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
__device__ __forceinline__ float rcp_approx(float x) {
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}

template <int V>
struct Gate {
  Vec<V> a, b;  // sigmoid and 1 - sigmoid
};
// With e = exp(-g): 1 / (1 + e) and e / (1 + e), so that neither loses bits where it is small.  g is
// held above -87, where e still has a reciprocal (and sigmoid(g) < 2^-125); a NaN stays one.
template <int V>
__device__ __forceinline__ Gate<V> sigmoid_pair(Vec<V> g) {
  Vec<V> e, r;
#pragma unroll
  for (int i = 0; i < V; ++i) {
    float h;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(h) : "f"(g.get(i)), "f"(-87.0f));
    e.set(i, h);
  }
  e = e * splat<V>(-1.4426950408889634f);  // exp(-g) = 2^(-g log2(e))
#pragma unroll
  for (int i = 0; i < V; ++i) e.set(i, ex2_approx(e.get(i)));
  const Vec<V> sum = e + splat<V>(1.0f);
#pragma unroll
  for (int i = 0; i < V; ++i) r.set(i, rcp_approx(sum.get(i)));
  return {r, e * r};
}

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
// How many of the first `sequences` offsets are at or below t (32 are looked at a time).
__device__ __forceinline__ int begun_by(const tb_scan_desc& d, int t) {
  const int lane = threadIdx.x % 32;
  int lo = 0, n = (int)d.sequences;  // the answer lies in [lo, lo + n]
  while (n > 0) {
    const int stride = (n + 31) / 32, i = lo + (lane + 1) * stride - 1;
    const bool below = i < lo + n && d.offsets[i] <= t;
    const int k = __popc(__ballot_sync(~0u, below));
    lo += k * stride;
    n = min(n - k * stride, stride - 1);
  }
  return lo;
}
// The sequence that a warp's last run lay in: most runs lie in the same one and need no search.
struct Known {
  int sequence = 0, from = 0, to = 0;
  // Whether rows [low, high] lie strictly inside it.
  __device__ __forceinline__ bool holds(int low, int high) const { return from < low && high < to - 1; }
};
template <int L, bool BACK>
__device__ __forceinline__ Marks marks_of(const tb_scan_desc& d, int b, int first, Known& known) {
  const int lane = threadIdx.x % 32, length = (int)d.length;
  constexpr unsigned kAll = (1u << L) - 1;
  const int left = length - first;
  const unsigned here = left >= L ? kAll : left <= 0 ? 0u : (1u << left) - 1;
  Marks m;
  if (d.sequences == 0) {
    m.sequence = b;
    m.inside = here;
    m.enters = first == 0 ? here & 1 : 0u;
    m.leaves = left > 0 && left <= L ? 1u << (left - 1) : 0u;
    return m;
  }
  m.inside = kAll;
  m.enters = m.leaves = 0;
  const int low = BACK ? length - first - L : first, high = low + L - 1;  // rows
  if (here == kAll && known.holds(low, high)) {
    m.sequence = known.sequence;
    return m;
  }
  const int begun = begun_by(d, low), s = max(begun - 1, 0);
  // offsets are data: whatever they hold, the first and last rows of the array are borders
  known = {s, max(d.offsets[s], 0), min(d.offsets[s + 1], length)};
  if (here == kAll && begun > 0 && known.holds(low, high)) {
    m.sequence = s;
    return m;
  }
  const int t = BACK ? length - 1 - first - lane : first + lane;
  const bool mine = here >> lane & 1;
  // the last sequence that starts at or before t
  int lo = s, hi = (int)d.sequences;
  while (hi - lo > 1) {
    const int mid = (lo + hi) / 2;
    if (mine && d.offsets[mid] <= t) lo = mid; else hi = mid;
  }
  const int from = d.offsets[lo], to = d.offsets[lo + 1];
  const bool inside = mine && from <= t && t < to;
  const bool starts = t == from || t == 0, ends = t == to - 1 || t == length - 1;
  m.sequence = lo;
  m.inside = __ballot_sync(~0u, inside);
  m.enters = __ballot_sync(~0u, inside && (BACK ? ends : starts));
  m.leaves = __ballot_sync(~0u, inside && (BACK ? starts : ends));
  return m;
}

constexpr int kWarps = 4;
constexpr int kMaxRanks = 8;

// What a run of steps does to the value v carried into it: v -> A v + H, or H alone where a
// sequence begins inside the run (then v belongs to another sequence and may be anything).
template <int V>
struct Affine {
  Vec<V> A, H;
};
template <int V>
__device__ __forceinline__ Vec<V> apply(Affine<V> f, bool begins, Vec<V> v) {
  return select(begins, f.H, fma(f.A, v, f.H));
}
template <int V>
__device__ __forceinline__ bool finite(Vec<V> a) {
  bool r = true;
#pragma unroll
  for (int i = 0; i < V; ++i) r &= fabsf(a.get(i)) < INFINITY;
  return r;
}

// Gates of the direct form may be larger than 1, and their product A may pass the range of 32 bits
// although every step of the recurrence stays within it: an infinite A would make NaN of a carried 0, and
// infinity of a small carried value.  A warp that meets one works its maps out again with A multiplied out
// in 64 bits.  Such a map is marked kWide, and A's place holds the high word, rounded: 21 bits of precision,
// which is what the roundings of sixteen gates in 32 bits leave too.  An A past the range of 64 bits takes
// every value but 0 out of the range of 32 on its way, and of a 0 nothing is left but H.  Products too small
// for 32 bits vanish: a run that shrinks what it is handed by more than 2^126 may hand on nothing of it.
// None of this is inlined: it hardly ever runs, and the kernels have no registers for it.
enum { kBegins = 1, kWide = 2 };  // what is said of a map; one that begins a sequence is never wide
template <int V>
struct Product {
  double x[V];
};
template <int V>
__device__ __forceinline__ Product<V> product_of(Vec<V> a, int said) {
  Product<V> r;
#pragma unroll
  for (int i = 0; i < V; ++i)
    r.x[i] = said & kWide ? __hiloint2double(__float_as_int(a.get(i)), 0) : (double)a.get(i);
  return r;
}
template <int V>
__device__ __forceinline__ Product<V> operator*(Product<V> a, Product<V> b) {
#pragma unroll
  for (int i = 0; i < V; ++i) a.x[i] *= b.x[i];
  return a;
}
template <int V>
__device__ __forceinline__ Vec<V> wide(Product<V> p) {
  Vec<V> r;
#pragma unroll
  for (int i = 0; i < V; ++i) {
    const long long bits = __double_as_longlong(p.x[i]);
    // an infinity or NaN is not rounded, for it might become another value
    r.set(i, __int_as_float((int)((fabs(p.x[i]) < INFINITY ? bits + 0x80000000ll : bits) >> 32)));
  }
  return r;
}
template <int V>
__device__ __forceinline__ Vec<V> apply_any(Affine<V> f, int said, Vec<V> v) {
  if (!(said & kWide)) return apply(f, said & kBegins, v);
  const Product<V> p = product_of(f.A, said);
#pragma unroll
  for (int i = 0; i < V; ++i)
    v.set(i, v.get(i) == 0.0f ? f.H.get(i) : (float)::fma(p.x[i], (double)v.get(i), (double)f.H.get(i)));
  return v;
}
template <int V>
__device__ __noinline__ Vec<V> applied(Affine<V> f, int said, Vec<V> v) {
  return apply_any(f, said, v);
}
template <int V>
struct Said {
  Affine<V> map;
  int said;
};
// The map of one run and another behind it.
template <int V>
__device__ __noinline__ Said<V> joined(Said<V> a, Said<V> b) {
  if (b.said & kBegins) return b;
  const Vec<V> H = apply_any(b.map, b.said, a.map.H);
  if (a.said & kBegins) return {{splat<V>(1.0f), H}, kBegins};
  return {{wide(product_of(a.map.A, a.said) * product_of(b.map.A, b.said)), H}, kWide};
}
// A lane's product of `count` gates, `bytes` apart.
template <typename T, int V>
__device__ __noinline__ Vec<V> wide_run(const char* gate, int64_t bytes, int count) {
  typedef Raw<T, V> R;
  Product<V> p = product_of(splat<V>(1.0f), 0);
  for (int i = 0; i < count; ++i)
    p = p * product_of(R::read(*(const typename R::type*)(gate + bytes * i)), 0);
  return wide(p);
}
// A lane's value carried through `count` maps, and what it is before number `at`.
template <int V>
struct Carried {
  Vec<V> after, before;
  bool arrived = true;
};
template <int V>
__device__ __forceinline__ Carried<V> wide_walk(const Affine<V> (*maps)[32], const int* said, int count, int at,
                                                Vec<V> v) {
  Carried<V> r{v, v};
  for (int i = 0; i < count; ++i) {
    if (i == at) r.before = r.after;
    r.after = apply_any(maps[i][threadIdx.x % 32], said[i], r.after);
  }
  return r;
}
// The maps of a block's warps behind one another.
template <int V>
__device__ __noinline__ Carried<V> wide_round(Affine<V> (*maps)[32], int* said, Affine<V> map, int of, Vec<V> carry) {
  const int lane = threadIdx.x % 32, warp = threadIdx.x / 32;
  maps[warp][lane] = map;
  if (lane == 0) said[warp] = of;
  __syncthreads();
  return wide_walk(maps, said, kWarps, warp, carry);
}
template <int V>
__device__ __noinline__ Said<V> wide_block(Affine<V> (*maps)[32], int* said, Affine<V> map, int of) {
  const int lane = threadIdx.x % 32, warp = threadIdx.x / 32;
  maps[warp][lane] = map;
  if (lane == 0) said[warp] = of;
  __syncthreads();
  Said<V> r{maps[0][lane], said[0]};
  for (int w = 1; w < kWarps; ++w) r = joined(r, {maps[w][lane], said[w]});
  return r;
}

// How a call is cut: `ranks` blocks of a cluster take consecutive spans of kWarps * L steps, over
// and over, and `parts` such clusters the consecutive parts of the time axis.  With several parts
// a first launch leaves each part's affine map in the workspace, and the second starts each part
// from the maps before it.
struct Cut {
  int ranks, tiles, parts;
  int64_t part_steps;
  float2* maps;  // (A, H), [batch][parts][channels], parts > 1
  int* said;     // [batch][parts][tiles]
  unsigned wait_ns;  // what a wait between blocks may take; 0 lets each run out at once
};

// A launch's part: a block walks its columns alone, or the blocks of a cluster together; or one of
// the two launches over parts.
enum { kWhole = 0, kMaps = 1, kFromMaps = 2, kCluster = 3 };

// The exchange of maps between the blocks of a cluster: a lane sends its words straight into every
// block's shared memory, and those count them in at a barrier of their own.  A cluster-wide barrier
// would first wait for the outputs written so far to reach memory, a quarter of the time.
__device__ __forceinline__ unsigned shared_address(const void* p) {
  return (unsigned)__cvta_generic_to_shared(p);
}
__device__ __forceinline__ unsigned of_rank(unsigned address, int rank) {
  unsigned r;
  asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(address), "r"(rank));
  return r;
}
__device__ __forceinline__ void send(unsigned to, unsigned barrier, Affine<2> f) {
  asm volatile("st.async.shared::cluster.mbarrier::complete_tx::bytes.v4.b32 [%0], {%1, %2, %3, %4}, [%5];"
               ::"r"(to), "r"(__float_as_uint(f.A.x.x)), "r"(__float_as_uint(f.A.x.y)),
               "r"(__float_as_uint(f.H.x.x)), "r"(__float_as_uint(f.H.x.y)), "r"(barrier)
               : "memory");
}
__device__ __forceinline__ void send(unsigned to, unsigned barrier, Affine<1> f) {
  asm volatile("st.async.shared::cluster.mbarrier::complete_tx::bytes.v2.b32 [%0], {%1, %2}, [%3];"
               ::"r"(to), "r"(__float_as_uint(f.A.x)), "r"(__float_as_uint(f.H.x)), "r"(barrier)
               : "memory");
}
__device__ __forceinline__ void send(unsigned to, unsigned barrier, int v) {
  asm volatile("st.async.shared::cluster.mbarrier::complete_tx::bytes.b32 [%0], %1, [%2];"
               ::"r"(to), "r"(v), "r"(barrier)
               : "memory");
}
// Set where a wait of the exchange ran out.
__device__ int g_wait_expired;

// Whether all that was expected has arrived; false after `limit` (4 seconds), which nothing but a fault
// explains.  The value carried into the block is NaN for the lane from there on, and it neither waits nor
// sends again, so that the waits for its maps run out too, and none takes a later round's for them.
__device__ __forceinline__ bool arrived(unsigned barrier, int phase, unsigned limit) {
  unsigned long long since = 0;
  while (limit != 0) {
    int done;
    asm volatile(
        "{\n .reg .pred p;\n mbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2;\n"
        " selp.s32 %0, 1, 0, p;\n}"
        : "=r"(done)
        : "r"(barrier), "r"(phase)
        : "memory");
    if (done) return true;
    unsigned long long now;
    asm volatile("mov.u64 %0, %%globaltimer;" : "=l"(now));
    if (since == 0) since = now;
    if (now - since > limit) break;
  }
  g_wait_expired = 1;
  return false;
}
// The end of a block of which a wait ran out: its shared memory stays until nothing can be on its way to it.
// The barrier waits for no block that has left, and the others come to it or leave within their own limits;
// what they sent before has landed long before a millisecond is over.
__device__ __noinline__ void leave_late() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n barrier.cluster.wait.acquire.aligned;" ::: "memory");
  unsigned long long now, since;
  asm volatile("mov.u64 %0, %%globaltimer;" : "=l"(since));
  do {
    asm volatile("mov.u64 %0, %%globaltimer;" : "=l"(now));
  } while (now - since < 1000000);
}

// As wide_round, by the warps of a cluster's blocks.  Each warp sends its map to all blocks by itself, so that
// none waits for another but at the barrier, where waits are bounded.
template <int V>
__device__ __noinline__ Carried<V> wide_exchange(Affine<V> (*maps)[32], int* said, uint64_t* counted, Affine<V> map,
                                                 int of, int ranks, int rank, int phase, unsigned limit, Vec<V> carry) {
  const int lane = threadIdx.x % 32, warp = threadIdx.x / 32, mine = rank * kWarps + warp;
  const unsigned barrier = shared_address(counted);
  if (threadIdx.x == 0)
    asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(barrier),
                 "r"(ranks * kWarps * (32 * (int)sizeof(Affine<V>) + 4))
                 : "memory");
  for (int r = 0; r < ranks; ++r) {
    const unsigned there = of_rank(barrier, r);
    send(of_rank(shared_address(&maps[mine][lane]), r), there, map);
    if (lane == 0) send(of_rank(shared_address(&said[mine]), r), there, of);
  }
  if (__any_sync(~0u, !arrived(barrier, phase, limit))) return {carry, carry, false};
  return wide_walk(maps, said, ranks * kWarps, mine, carry);
}

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
  typedef Raw<T, V> R;
  typedef typename R::type Row;
  static constexpr bool kReadsX = FORM == TB_SCAN_SIGMOID;
  static constexpr bool kGrows = FORM == TB_SCAN_DIRECT;  // products of gates may leave the range
  const tb_scan_desc& d;
  const int64_t b, c;
  const bool in;  // this lane's channels exist
  const float* entry_state;
  float* exit_state;
  struct Rows {
    Row g[L], u[L], before[L], xs[L];  // u: x, or dh backwards
  };
  Vec<V> a[L], add[L];

  __device__ Scan(const tb_scan_desc& d, int64_t b, int64_t c)
      : d(d), b(b), c(c), in(c < d.channels), entry_state(BACK ? d.dfinal : d.state),
        exit_state(BACK ? d.dstate : d.final_state) {}

  // A row of one array, and the bytes from a step's row to the next step's.  Steps lie less than 2^31
  // bytes apart (the host sees to it), so that an address is one 32 x 32-bit multiplication and
  // addition, off the integer pipe that the conversions fill; the direct form forwards is as quick with
  // pointers that walk, and needs fewer registers (packed 131072 x 768 bf16: 168 us, by products 178;
  // 32 x 4096 x 512 bf16 sigmoid: backward 160 by products, 172 walking).
  static constexpr bool kProducts = BACK || FORM == TB_SCAN_SIGMOID;
  typedef std::conditional_t<kProducts, int, int64_t> Step;
  __device__ __forceinline__ const char* at(const void* base, const int64_t s[2], int64_t t) const {
    return (const char*)((const T*)base + b * s[0] + t * s[1] + c);
  }
  __device__ __forceinline__ static Step step(const int64_t s[2]) {
    return (BACK ? -1 : 1) * (Step)s[1] * (Step)sizeof(T);
  }
  __device__ __forceinline__ static Row* row(const char*& p, Step bytes, int i) {
    if (kProducts) return (Row*)(p + (int64_t)bytes * i);
    Row* r = (Row*)p;
    p += bytes;
    return r;
  }

  // ALL: every step lies within the array and its channels exist.
  template <bool ALL>
  __device__ __forceinline__ void load(Rows& r, int first) const {
    const int length = (int)d.length, t0 = BACK ? length - 1 - first : first, left = length - first;
    const char* pg = at(d.gate, d.gate_strides, t0);
    const char* pu = BACK ? at(d.dh, d.dh_strides, t0) : at(d.x, d.x_strides, t0);
    const char* ph = at(d.h, d.h_strides, t0 - 1);
    const char* px = at(d.x, d.x_strides, t0);
    const Step sg = step(d.gate_strides), su = step(BACK ? d.dh_strides : d.x_strides),
              sh = step(d.h_strides), sx = step(d.x_strides);
#pragma unroll
    for (int i = 0; i < L; ++i) {
      if (!ALL) r.g[i] = r.u[i] = r.before[i] = r.xs[i] = Row{};
      const Row *g = row(pg, sg, i), *u = row(pu, su, i);
      if (ALL || (in && i < left)) {
        r.g[i] = *g;
        r.u[i] = *u;
        if (BACK && PASS != kMaps) {
          // the row before the first is the state's
          if (ALL && i < L - 1) r.before[i] = *row(ph, sh, i);
          else r.before[i] = t0 - i > 0 ? *row(ph, sh, i) : Row{};
          if (kReadsX) r.xs[i] = *row(px, sx, i);
        }
      }
    }
  }

  __device__ __forceinline__ Vec<V> state_at(const float* states, int64_t at) const {
    Vec<V> r = splat<V>(0.0f);
    if (states && in)
#pragma unroll
      for (int v = 0; v < V; ++v) r.set(v, states[at + v]);
    return r;
  }

  // The added term of each step (and a, where the outputs do not work it out again), and the
  // steps' map.  A step that enters a sequence holds the entry state's part in its term, so that
  // state is read before any other state is written.  What rows outside every sequence hold goes
  // nowhere: the next row inside one enters it.
  template <bool MARKED>
  __device__ __forceinline__ Affine<V> reduce(const Rows& r, const Marks& m) {
    Affine<V> map{splat<V>(1.0f), splat<V>(0.0f)};
#pragma unroll
    for (int i = 0; i < L; ++i) {
      Vec<V> av = R::read(r.g[i]), bv = R::read(r.u[i]);
      if (FORM == TB_SCAN_SIGMOID) {
        const Gate<V> p = sigmoid_pair(av);
        av = p.a;
        if (!BACK) bv = bv * p.b;
      }
      if (MARKED && (m.enters >> i & 1)) {
        const Vec<V> e =
            state_at(entry_state, (int64_t)__shfl_sync(~0u, m.sequence, i) * d.channels + c);
        bv = BACK ? bv + e : fma(av, e, bv);
        map.H = BACK ? av * bv : bv;
      } else {
        map.H = BACK ? av * (map.H + bv) : fma(av, map.H, bv);
      }
      map.A = map.A * av;
      if (!BACK) a[i] = av;
      add[i] = bv;
    }
    return map;
  }

  // The map of a run of which no row is written yet, with A in 64 bits where 32 do not hold it.
  __device__ __forceinline__ Said<V> said_of(Affine<V> map, const Marks& m, int first) const {
    if (m.enters) return {map, kBegins};
    if (!__any_sync(~0u, !finite(map.A))) return {map, 0};
    const int t0 = BACK ? (int)d.length - 1 - first : first;
    // steps and channels that do not exist have a gate of 0
    map.A = in && first + L <= d.length ? wide_run<T, V>(at(d.gate, d.gate_strides, t0), step(d.gate_strides), L)
                                        : splat<V>(0.0f);
    return {map, kWide};
  }

  // Zeros to the rows before the first and behind the last sequence, for worker `mine` of `all`.
  __device__ __forceinline__ void clear_outside(int mine, int all) const {
    const int length = (int)d.length, begin = (int)clamped_offset(d, 0), end = (int)clamped_offset(d, d.sequences);
    for (int t = mine; t < length; t += all) {
      if (t >= begin && t < end) {
        t += (end - 1 - t) / all * all;  // to the last of these rows that is this worker's
        continue;
      }
      if (!BACK && d.clear & TB_SCAN_CLEAR_H) *(Row*)at(d.h, d.h_strides, t) = Row{};
      if (BACK && d.clear & TB_SCAN_CLEAR_DGATE) *(Row*)at(d.dgate, d.dgate_strides, t) = Row{};
      if (BACK && d.clear & TB_SCAN_CLEAR_DX) *(Row*)at(d.dx, d.dx_strides, t) = Row{};
    }
  }

  // Sequences without a step hand their entry state on, for worker `mine` of `all`, whose lanes look at one
  // sequence each.
  __device__ __forceinline__ void hand_on(int mine, int all) const {
    for (int64_t base = (int64_t)mine * 32; base < d.sequences; base += (int64_t)all * 32) {
      const int64_t i = base + threadIdx.x % 32;
      unsigned empty = __ballot_sync(~0u, i < d.sequences && clamped_offset(d, i + 1) <= clamped_offset(d, i));
      for (; empty; empty &= empty - 1) {
        const int64_t at = (base + __ffs(empty) - 1) * d.channels + c;
        const Vec<V> e = state_at(entry_state, at);
        if (in)
#pragma unroll
          for (int v = 0; v < V; ++v) exit_state[at + v] = e.get(v);
      }
    }
  }

  // ALL as in load(); MARKED: some step enters or leaves a sequence or lies outside all of them.
  template <bool ALL, bool MARKED>
  __device__ __forceinline__ void write(const Rows& r, const Marks& m, int first, Vec<V> value) {
    const int t0 = BACK ? (int)d.length - 1 - first : first;
    const int64_t* strides = BACK ? d.dgate_strides : d.h_strides;
    const char* p1 = at(BACK ? d.dgate : d.h, strides, t0);
    const char* p2 = at(d.dx, d.dx_strides, t0);
    const Step s1 = step(strides), s2 = step(d.dx_strides);
#pragma unroll
    for (int i = 0; i < L; ++i) {
      const bool enters = MARKED && (m.enters >> i & 1), leaves = MARKED && (m.leaves >> i & 1);
      const int64_t state = leaves ? (int64_t)__shfl_sync(~0u, m.sequence, i) * d.channels + c : 0;
      Vec<V> out, out2;
      if (BACK) {
        const Vec<V> gt = MARKED ? select(enters, add[i], add[i] + value) : add[i] + value;
        Vec<V> prior = R::read(r.before[i]), av = R::read(r.g[i]);
        if (leaves) prior = state_at(d.state, state);
        if (FORM == TB_SCAN_SIGMOID) {
          const Gate<V> p = sigmoid_pair(av);
          av = p.a;
          out2 = gt * p.b;
          out = out2 * p.a * fma(R::read(r.xs[i]), splat<V>(-1.0f), prior);
        } else {
          out2 = gt;
          out = gt * prior;
        }
        value = av * gt;
      } else {
        value = MARKED ? select(enters, add[i], fma(a[i], value, add[i])) : fma(a[i], value, add[i]);
        out = value;
      }
      Row* to = row(p1, s1, i);
      if ((ALL || in) && (!MARKED || (m.inside >> i & 1))) {
        *to = R::made(out);
        if (BACK) *row(p2, s2, i) = R::made(out2);
      }
      if (leaves && in && exit_state)
#pragma unroll
        for (int v = 0; v < V; ++v) exit_state[state + v] = value.get(v);
    }
  }
};

template <typename T, int V, int L, int FORM, bool BACK, int PASS>
__global__ void __launch_bounds__(kWarps * 32, 4) k_scan(tb_scan_desc d, Cut cut) {
  pdl_entry();
  __shared__ alignas(16) Affine<V> maps[2][kWarps][32];
  __shared__ int said[2][kWarps];
  constexpr int kHeld = PASS == kCluster ? kMaxRanks : 1;
  __shared__ alignas(16) Affine<V> rank_maps[2][kHeld][32];
  __shared__ int rank_said[2][kHeld];
  __shared__ alignas(8) uint64_t counted[3];  // barriers of the exchange, one a parity, and of wide maps
  constexpr bool kGrows = Scan<T, V, L, FORM, BACK, PASS>::kGrows;
  __shared__ alignas(16) Affine<V> wide_maps[kGrows ? kHeld * kWarps : 1][32];
  __shared__ alignas(8) Vec<V> carries[2][32];  // what a round began with
  __shared__ int wide_said[kGrows ? kHeld * kWarps : 1];
  const int lane = threadIdx.x % 32, warp = __shfl_sync(~0u, threadIdx.x / 32, 0);
  const int ranks = PASS == kCluster ? cut.ranks : 1;
  const int rank = blockIdx.x % ranks, tile = blockIdx.x / ranks % cut.tiles;
  const int part = blockIdx.x / ranks / cut.tiles % cut.parts;
  const int64_t b = blockIdx.x / ranks / cut.tiles / cut.parts;
  Scan<T, V, L, FORM, BACK, PASS> s(d, b, (int64_t)(tile * 32 + lane) * V);

  if constexpr (PASS == kCluster) {
    if (threadIdx.x == 0)
#pragma unroll
      for (int i = 0; i < 3; ++i)
        asm volatile("mbarrier.init.shared::cta.b64 [%0], 1;" ::"r"(shared_address(&counted[i])) : "memory");
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    cg::this_cluster().sync();
  }

  Vec<V> carry = splat<V>(0.0f);
  if (PASS == kFromMaps && s.in) {
    const float2* from = cut.maps + b * cut.parts * d.channels + s.c;
    const int* of = cut.said + b * cut.parts * cut.tiles + tile;
    const auto map = [&](int p) {
      Affine<V> f;
#pragma unroll
      for (int v = 0; v < V; ++v) {
        f.A.set(v, from[p * d.channels + v].x);
        f.H.set(v, from[p * d.channels + v].y);
      }
      return f;
    };
    int seen = 0;
#pragma unroll 8
    for (int p = 0; p < part; ++p) {
      seen |= of[p * cut.tiles];
      carry = apply(map(p), of[p * cut.tiles] & kBegins, carry);
    }
    if (kGrows && seen & kWide) {
      carry = splat<V>(0.0f);
      for (int p = 0; p < part; ++p) carry = applied(map(p), of[p * cut.tiles], carry);
    }
  }
  Affine<V> whole{splat<V>(1.0f), splat<V>(0.0f)};  // the part's map so far
  int whole_said = 0;

  int parity = 0, phase = 0;  // of the exchange's buffers, and of their barriers
  [[maybe_unused]] int wide_phase = 0;
  [[maybe_unused]] int reached = ranks;  // blocks that this one exchanges maps with: 0 once a wait has run out
  [[maybe_unused]] unsigned wait_ns = cut.wait_ns;
  const int from = (int)(part * cut.part_steps), to = (int)min(from + cut.part_steps, d.length);
  const int span = ranks * kWarps * L;
  // a part is a whole number of spans, so that no step belongs to two
  const bool whole_warp = __all_sync(~0u, s.in);
  typename Scan<T, V, L, FORM, BACK, PASS>::Rows rows, next;
  int first = from + (rank * kWarps + warp) * L;
  bool all = whole_warp && first + L <= d.length;
  if (all) s.template load<true>(rows, first); else s.template load<false>(rows, first);
  Known known;
  Marks m = marks_of<L, BACK>(d, (int)b, first, known), next_m = m;
  int base = from;
  const auto run = [&](auto& rows, auto& next) {
    const bool marked = m.enters | m.leaves | (m.inside != (1u << L) - 1);
    const Affine<V> map = m.enters ? s.template reduce<true>(rows, m) : s.template reduce<false>(rows, m);
    // the next steps are on their way while these are finished
    const int next_first = first + span;
    const bool next_all = whole_warp && next_first + L <= d.length;
    if (base + span < to) {
      if (next_all) s.template load<true>(next, next_first);
      else s.template load<false>(next, next_first);
      next_m = marks_of<L, BACK>(d, (int)b, next_first, known);
    }
    maps[parity][warp][lane] = map;
    // whether a product is not finite is said of the run's map (16 x 512 x 4096 bf16 35.8 us, 37.9 by the
    // product of all), or seen in the product of all maps that are walked: an infinity or NaN stays one
    constexpr bool kMarked = kGrows && PASS == kWhole;
    int mark = m.enters ? kBegins : 0;
    if (kMarked && !mark && __any_sync(~0u, !finite(map.A))) mark = kWide;
    if (lane == 0) said[parity][warp] = mark;
    if (kGrows && PASS != kMaps && warp == 0) carries[parity][lane] = carry;
    __syncthreads();
    if constexpr (PASS == kCluster || PASS == kMaps) {
      // this block's map
      Affine<V> block{splat<V>(1.0f), splat<V>(0.0f)};
      int any = 0;
#pragma unroll
      for (int w = 0; w < kWarps; ++w) {
        const int of = said[parity][w];
        const Affine<V> f = maps[parity][w][lane];
        any |= of;
        block = {block.A * f.A, apply(f, of & kBegins, block.H)};
      }
      if constexpr (PASS == kMaps) {
        const Vec<V> A = whole.A * block.A;
        if (kGrows && (whole_said & kWide ||
                       __any_sync(~0u, !finite(block.A) || (!whole_said && !any && !finite(A))))) {
          const Said<V> mine = s.said_of(maps[parity][warp][lane], m, first);
          const Said<V> both = joined({whole, whole_said}, wide_block(wide_maps, wide_said, mine.map, mine.said));
          whole = both.map;
          whole_said = both.said;
        } else {
          whole = {A, apply(block, any & kBegins, whole.H)};
          if (any) whole_said = kBegins;
        }
        m = next_m, first = next_first, all = next_all, base += span, parity ^= 1;
        return;
      }
      const unsigned barrier = shared_address(&counted[parity]);
      if (threadIdx.x == 0 && reached)
        asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(barrier),
                     "r"(ranks * (32 * (int)sizeof(Affine<V>) + 4))
                     : "memory");
      for (int r = warp; r < reached; r += kWarps) {  // to every block of the cluster
        const unsigned there = of_rank(barrier, r);
        send(of_rank(shared_address(&rank_maps[parity][rank][lane]), r), there, block);
        if (lane == 0) send(of_rank(shared_address(&rank_said[parity][rank]), r), there, any & kBegins);
      }
      if (!arrived(barrier, phase, wait_ns)) {
        carry = splat<V>(NAN);
        reached = wait_ns = 0;
      }
      phase ^= parity;
    }
    // the value carried into this warp's steps, and past all blocks' steps
    Vec<V> value = carry;
    [[maybe_unused]] Vec<V> A = splat<V>(1.0f);  // finite where all are
    [[maybe_unused]] int seen = 0;
    if constexpr (PASS == kCluster) {
      for (int r = 0; r < reached; ++r) {
        const Affine<V> f = rank_maps[parity][r][lane];
        if (r == rank) value = carry;
        carry = apply(f, rank_said[parity][r] & kBegins, carry);
        if (kGrows) A = A * f.A;
      }
#pragma unroll
      for (int w = 0; w < kWarps - 1; ++w)
        if (w < warp) value = apply(maps[parity][w][lane], said[parity][w] & kBegins, value);
    } else {
#pragma unroll
      for (int w = 0; w < kWarps; ++w) {
        if (w == warp) value = carry;
        const Affine<V> f = maps[parity][w][lane];
        const int of = said[parity][w];
        if (kMarked) seen |= of;
        else if (kGrows) A = A * f.A;
        carry = apply(f, of & kBegins, carry);
      }
    }
    // the same for all warps of the block, or the cluster; never for what a lane found whose wait ran out, as
    // the other blocks may have left
    if (kMarked ? (seen & kWide) != 0 : kGrows && __any_sync(~0u, !finite(A))) {
      // Where two rows of registers for each step are all there are, what the calls would have to keep is
      // read and reduced again (32 x 4096 x 512 bf16 73 us, 102 with it kept) -- but for entry states, for
      // another warp may be about to write them.
      constexpr bool kAgain = L * V >= 32;
      [[maybe_unused]] volatile float kept[kAgain ? L * V : 1];
      if (kAgain && m.enters)
#pragma unroll
        for (int i = 0; i < L * V; ++i) kept[i] = s.add[i / V].get(i % V);
      const Said<V> mine = s.said_of(maps[parity][warp][lane], m, first);
      Carried<V> c;
      if constexpr (PASS == kCluster) {
        c = wide_exchange(wide_maps, wide_said, &counted[2], mine.map, mine.said, ranks, rank, wide_phase,
                          wait_ns, carries[parity][lane]);
        wide_phase ^= 1;
        if (!c.arrived) {
          c = {splat<V>(NAN), splat<V>(NAN)};
          reached = wait_ns = 0;
        }
      } else {
        c = wide_round(wide_maps, wide_said, mine.map, mine.said, carries[parity][lane]);
      }
      carry = c.after, value = c.before;
      if constexpr (kAgain) {
        s.template load<false>(rows, first);
        s.template reduce<false>(rows, m);
#pragma unroll
        for (int i = 0; i < L; ++i)
          if (m.enters >> i & 1)
#pragma unroll
            for (int v = 0; v < V; ++v) s.add[i].set(v, kept[i * V + v]);
        if (base + span < to) s.template load<false>(next, next_first);
      }
    }
    if (all && !marked) s.template write<true, false>(rows, m, first, value);
    else s.template write<false, true>(rows, m, first, value);
    m = next_m, first = next_first, all = next_all, base += span, parity ^= 1;
  };
  // Forwards, rows are done with once they are reduced, and the next take their place; backwards the
  // two sets take turns.
  while (base < to) {
    if constexpr (BACK && PASS != kMaps) {
      run(rows, next);
      if (base >= to) break;
      run(next, rows);
    } else {
      run(rows, rows);
    }
  }
  // at the end, where no register is held (zeros among the outputs took a tenth of a backward pass) and no
  // block waits for this one
  if (PASS != kMaps && d.sequences) {
    const int worker = (part * ranks + rank) * kWarps + warp, workers = cut.parts * ranks * kWarps;
    if (s.exit_state) s.hand_on(worker, workers);
    if (d.clear && s.in) s.clear_outside(worker, workers);
  }
  if (PASS == kCluster && __syncthreads_or(reached == 0)) leave_late();
  if (PASS == kMaps && warp == 0) {
    if (s.in)
#pragma unroll
      for (int v = 0; v < V; ++v)
        cut.maps[(b * cut.parts + part) * d.channels + s.c + v] = {whole.A.get(v), whole.H.get(v)};
    if (lane == 0) cut.said[(b * cut.parts + part) * cut.tiles + tile] = whole_said;
  }
}

// Short sequences, a decode step's single one among them: a thread takes V channels of one sequence
// and walks it, kAtOnce rows loaded at a time.
template <typename T, int V, int FORM, bool BACK>
__global__ void __launch_bounds__(128) k_scan_short(tb_scan_desc d, int64_t lanes) {
  pdl_entry();
  typedef Raw<T, V> R;
  typedef typename R::type Row;
  constexpr int kAtOnce = 4;
  const int64_t i = (int64_t)blockIdx.x * 128 + threadIdx.x, b = i / lanes, c = (i - b * lanes) * V;
  if (b >= d.batch) return;
  const int length = (int)d.length;
  const auto row = [&](const void* base, const int64_t s[2], int t) {
    return (const Row*)((const T*)base + b * s[0] + t * s[1] + c);
  };
  const auto to = [&](void* base, const int64_t s[2], int t) {
    return (Row*)((T*)base + b * s[0] + t * s[1] + c);
  };
  const auto state_of = [&](const float* from) {
    Vec<V> r = splat<V>(0.0f);
    if (from)
#pragma unroll
      for (int v = 0; v < V; ++v) r.set(v, from[b * d.channels + c + v]);
    return r;
  };
  const Vec<V> initial = BACK ? state_of(d.state) : splat<V>(0.0f);
  Vec<V> value = state_of(BACK ? d.dfinal : d.state);
  for (int first = 0; first < length; first += kAtOnce) {
    Row g[kAtOnce], u[kAtOnce], before[kAtOnce], xs[kAtOnce];
#pragma unroll
    for (int j = 0; j < kAtOnce; ++j) {
      g[j] = u[j] = before[j] = xs[j] = Row{};
      if (first + j < length) {
        const int t = BACK ? length - 1 - first - j : first + j;
        g[j] = *row(d.gate, d.gate_strides, t);
        u[j] = BACK ? *row(d.dh, d.dh_strides, t) : *row(d.x, d.x_strides, t);
        if (BACK && t > 0) before[j] = *row(d.h, d.h_strides, t - 1);
        if (BACK && FORM == TB_SCAN_SIGMOID) xs[j] = *row(d.x, d.x_strides, t);
      }
    }
#pragma unroll
    for (int j = 0; j < kAtOnce; ++j) {
      if (first + j >= length) break;
      const int t = BACK ? length - 1 - first - j : first + j;
      Vec<V> a = R::read(g[j]), w = splat<V>(1.0f);  // w: the form's 1 - a
      const Vec<V> in = R::read(u[j]);
      if (FORM == TB_SCAN_SIGMOID) {
        const Gate<V> p = sigmoid_pair(a);
        a = p.a;
        w = p.b;
      }
      if (BACK) {
        const Vec<V> gt = in + value;
        const Vec<V> prior = t > 0 ? R::read(before[j]) : initial;
        Vec<V> da = gt * prior, dv = gt;
        if (FORM == TB_SCAN_SIGMOID) {
          dv = gt * w;
          da = dv * a * fma(R::read(xs[j]), splat<V>(-1.0f), prior);
        }
        value = a * gt;
        *to(d.dgate, d.dgate_strides, t) = R::made(da);
        *to(d.dx, d.dx_strides, t) = R::made(dv);
      } else {
        value = fma(a, value, FORM == TB_SCAN_SIGMOID ? in * w : in);
        *to(d.h, d.h_strides, t) = R::made(value);
      }
    }
  }
  float* last = BACK ? d.dstate : d.final_state;
  if (last)
#pragma unroll
    for (int v = 0; v < V; ++v) last[b * d.channels + c + v] = value.get(v);
}

// Blocks a cluster: as many as bring two blocks to every SM.
int ranks_of(int64_t columns, int64_t spans) {
  int ranks = 1;
  while (ranks < kMaxRanks && columns * ranks < 2 * 148 && ranks < spans) ranks *= 2;
  return ranks;
}
// Into how many parts the time axis is cut, each part two launches' work: its map, then its
// outputs.  1 where clusters bring two blocks to every SM, however long they walk, for a cut call
// reads its inputs twice (256 columns of 64 spans: 80 us in one launch, 133 cut; 128 of 128 spans
// 93 and 111; 48 of 65 spans 31 and 33), or where there is little to walk (16 columns of 16 spans: 8
// and 8).  But 16 columns of 125 spans take 21 us in one launch and 16 cut, 32 of 128 spans 41 and 31,
// 12 of 2048 spans 728 and 172.  Four blocks run on a SM: parts that fill them once, or twice where
// that leaves long ones (12 columns: 49 parts 176 us, 64 parts 217; 96 columns: 12 parts 39.8, 6 parts
// 43), and at least four spans each, for every part reads the maps of those before it (one column of
// 256 spans: 64 parts 14.2 us, 256 parts 21; of 2048 spans: 296 parts 37, 592 parts 47).
constexpr int64_t kMaxParts = 296;
int parts_of(int64_t columns, int64_t spans) {
  const int ranks = ranks_of(columns, spans);
  if (columns * ranks >= 2 * 148 || spans <= 2 * ranks || (columns * ranks >= 148 && spans <= 8 * ranks)) return 1;
  const int64_t wave = 4 * 148 / columns, fill = wave >= 16 ? wave : 8 * 148 / columns;
  return (int)std::max<int64_t>(1, std::min({kMaxParts, (spans + 3) / 4, fill}));
}

bool strides_ok(const tb_scan_desc& d, const int64_t s[2], bool written) {
  if (!extents_fit({s[0]}) || !extents_fit({s[1]}) || (d.length > 1 && s[1] > INT32_MAX / 4)) return false;
  return !written || rows_apart<2>(d.channels, {d.batch, d.length}, {s[0], s[1]});
}

constexpr int64_t kMaxLength = INT32_MAX - (1 << 16);  // steps are counted in 32 bits, a span past the end

const char* check(const tb_scan_desc& d, bool backward) {
  if (d.element != TB_ELEMENT_F32 && d.element != TB_ELEMENT_BF16) return "unknown element type";
  if (d.form != TB_SCAN_DIRECT && d.form != TB_SCAN_SIGMOID) return "unknown form";
  if (!extents_fit({d.batch, d.length, d.channels}) || d.length > kMaxLength || d.batch > INT32_MAX ||
      d.channels > INT32_MAX ||
      !extents_fit({d.sequences, d.channels}) || d.sequences > INT32_MAX)
    return "extents out of range";
  if (d.sequences ? !d.offsets || d.batch != 1 : d.offsets != nullptr)
    return "packed sequences come with offsets and a batch of 1";
  if (d.clear & ~(TB_SCAN_CLEAR_H | TB_SCAN_CLEAR_DGATE | TB_SCAN_CLEAR_DX)) return "unknown array to clear";
  const bool reads_x = !backward || d.form == TB_SCAN_SIGMOID;
  if (!strides_ok(d, d.gate_strides, false) || (reads_x && !strides_ok(d, d.x_strides, false)) ||
      !strides_ok(d, d.h_strides, !backward) ||
      (backward && (!strides_ok(d, d.dh_strides, false) || !strides_ok(d, d.dgate_strides, true) ||
                    !strides_ok(d, d.dx_strides, true))))
    return "strides are negative, too large (2^29 elements or more from step to step), or let written "
           "rows overlap";
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

std::atomic<unsigned> g_wait_ns{4000000000u};

template <typename T, int V, int L, int FORM, bool BACK, int PASS>
cudaError_t launch(const tb_scan_desc& d, const Cut& cut, cudaStream_t stream) {
  const int64_t blocks = d.batch * cut.parts * cut.tiles * cut.ranks;
  if (blocks > INT32_MAX) return cudaErrorInvalidConfiguration;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)blocks);
  cfg.blockDim = dim3(kWarps * 32);
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  unsigned attrs = 0;
  if (PASS == kCluster) {
    attr[attrs].id = cudaLaunchAttributeClusterDimension;
    attr[attrs].val.clusterDim.x = cut.ranks;
    attr[attrs].val.clusterDim.y = attr[attrs].val.clusterDim.z = 1;
    ++attrs;
  }
  if (pdl_enabled()) {
    attr[attrs].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[attrs].val.programmaticStreamSerializationAllowed = 1;
    ++attrs;
  }
  cfg.attrs = attr;
  cfg.numAttrs = attrs;
  return cudaLaunchKernelEx(&cfg, k_scan<T, V, L, FORM, BACK, PASS>, d, cut);
}

template <typename T, int V, int L, int FORM, bool BACK>
cudaError_t enqueue(const tb_scan_desc& d, cudaStream_t stream) {
  const int64_t span = kWarps * L;
  Cut cut = {};
  cut.wait_ns = g_wait_ns.load(std::memory_order_relaxed);
  cut.tiles = (int)((d.channels + 32 * V - 1) / (32 * V));
  cut.ranks = cut.parts = 1;
  cut.part_steps = std::max<int64_t>(d.length, 1);
  const int64_t columns = d.batch * cut.tiles, spans = (d.length + span - 1) / span;
  // a state that is read and written in one call is read before it is written only within a launch
  // (12 columns of 2048 spans take 728 us so, and 172 with a final state of its own)
  const bool carries = BACK ? d.dstate && d.dstate == d.dfinal : d.final_state && d.final_state == d.state;
  if (d.workspace && columns * spans > 0 && !carries) cut.parts = parts_of(columns, spans);
  if (cut.parts > 1) {
    cut.part_steps = (spans + cut.parts - 1) / cut.parts * span;
    cut.parts = (int)((d.length + cut.part_steps - 1) / cut.part_steps);
    cut.maps = (float2*)d.workspace;
    cut.said = (int*)(cut.maps + d.batch * cut.parts * d.channels);
    const cudaError_t e = launch<T, V, L, FORM, BACK, kMaps>(d, cut, stream);
    return e != cudaSuccess ? e : launch<T, V, L, FORM, BACK, kFromMaps>(d, cut, stream);
  }
  cut.ranks = ranks_of(columns, spans);
  return cut.ranks > 1 ? launch<T, V, L, FORM, BACK, kCluster>(d, cut, stream)
                       : launch<T, V, L, FORM, BACK, kWhole>(d, cut, stream);
}

// Measured, 64 sequences of 2048 f32 channels: 8 steps 2.9 us short and 9.6 tiled, 16 steps 5.8 and
// 10.5, 32 steps 15.0 and 14.8; 4 sequences of 32 steps x 333 channels 3.2 and 2.7.
constexpr int64_t kShort = 16;

template <typename T, int FORM, bool BACK>
cudaError_t enqueue_form(const tb_scan_desc& d, cudaStream_t stream) {
  const bool pairs = lanes_fit(d, BACK, sizeof(T), 2 * sizeof(T));
  if (d.sequences == 0 && d.length <= kShort) {
    const int64_t lanes = pairs ? d.channels / 2 : d.channels, blocks = (d.batch * lanes + 127) / 128;
    if (blocks > INT32_MAX) return cudaErrorInvalidConfiguration;
    return launch_pdl(pairs ? k_scan_short<T, 2, FORM, BACK> : k_scan_short<T, 1, FORM, BACK>,
                      dim3((unsigned)blocks), dim3(128), 0, stream, d, lanes);
  }
  // as many steps a warp as 128 registers hold, with the next ones on their way
  constexpr int kPairs = sizeof(T) == 2 ? (BACK ? 8 : 16) : !BACK || FORM == TB_SCAN_DIRECT ? 8 : 4;
  return pairs ? enqueue<T, 2, kPairs, FORM, BACK>(d, stream)
               : enqueue<T, 1, BACK ? 8 : 16, FORM, BACK>(d, stream);
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
  // whichever block the call takes: columns of 32 or 64 channels, spans of 4, 8 or 16 steps a warp
  int64_t parts = 1;
  for (int64_t width : {32, 64})
    for (int64_t steps : {4, 8, 16})
      parts = std::max<int64_t>(parts, parts_of(batch * ((channels + width - 1) / width),
                                                (length + kWarps * steps - 1) / (kWarps * steps)));
  const int64_t tiles = (channels + 31) / 32, words = 2 * channels + tiles;  // of a part: its maps, what is said
  return parts > 1 ? (batch * parts * words * 4 + 15) / 16 * 16 : 0;
}

int operators_synchronize(void* stream) {
  OperatorCall call("tb_operators_synchronize", stream);
  if (const int code = call.ready()) return code;
  int expired = 0;
  cudaError_t e = cudaStreamSynchronize(call.stream());
  if (e == cudaSuccess) e = cudaMemcpyFromSymbol(&expired, g_wait_expired, sizeof expired);
  if (e == cudaSuccess && expired) e = cudaErrorLaunchTimeout;
  return call.finish(e);
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

extern "C" int tb_operators_synchronize(void* stream) {
  return tb::guarded([&] { return tb::operators_synchronize(stream); });
}

// ---- internal hooks for tests (not part of the public ABI): the limit of a scan's waits, and whether a wait between the blocks of a
// cluster ever ran out on the current device (1), or the flag cannot be read (-1).
extern "C" void tbx_scan_wait_limit(int64_t ns) { tb::g_wait_ns = (unsigned)ns; }
extern "C" int tbx_scan_error(void) {
  int expired = 0;
  return cudaMemcpyFromSymbol(&expired, tb::g_wait_expired, sizeof expired) == cudaSuccess ? expired : -1;
}
