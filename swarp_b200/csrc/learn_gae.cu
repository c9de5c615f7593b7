// Generalised advantage estimates (swarp_gae; contract in include/swarp_b200.h):
//   A_t = d_t + c_t A_{t+1},  d_t = r_t + gamma V'_t - V_t,  c_t = gamma lambda or 0
// a linear recurrence backwards over the steps, one per column.
#include "learn.cuh"

namespace swarp {
namespace learn {
namespace {

template <typename T> struct Args {
  const T *r, *v, *next, *last;
  const uint8_t *term, *trunc;
  T *adv, *ret;
  long long steps, columns, flags;  // flags per step
  int per_flag;
  T gamma, decay;  // gamma lambda
};

template <typename T> struct Step {
  T r = 0, v = 0, next = 0;  // next: V' where next_values are given
  bool term = false, stop = false;
};
template <typename T>
__device__ __forceinline__ Step<T> load_step(const Args<T>& a, long long t, long long j,
                                             long long f) {
  const long long k = t * a.columns + j, g = t * a.flags + f;
  Step<T> s;
  s.r = a.r[k];
  s.v = a.v[k];
  s.next = a.next ? a.next[k] : T(0);
  // both flags are asked for at once; with no decay at all the next step's advantage is out,
  // whatever it is
  const unsigned term = a.term ? a.term[g] : 0, trunc = a.trunc ? a.trunc[g] : 0;
  s.term = term != 0;
  s.stop = (term | trunc | (a.decay == T(0))) != 0;
  return s;
}

// A stretch of steps takes the advantage x after it to b + p x before it, with p the product of
// its decays; such maps compose.
template <typename T> struct Map {
  T p, b;  // x -> b + p x
};
// p is 0 for an end of an episode alone, which keeps whatever is after it out, NaN included. A
// product of decays that underflows stays at the least number above, which still hands a NaN or
// an infinity on and adds nothing else.
template <typename T> __device__ __forceinline__ T least();
template <> __device__ __forceinline__ float least<float>() { return __int_as_float(1); }
template <> __device__ __forceinline__ double least<double>() { return __longlong_as_double(1); }
// maps one after the other, the earliest stretch of time first: x -> first(then(x))
template <typename T> struct Chain {
  T p = 1, b = 0;
  bool ended = false;
  __device__ __forceinline__ void then(Map<T> m) {
    const T q = p * m.p, longer = b + p * m.b;
    b = ended ? b : longer;
    p = q == T(0) ? least<T>() : q;
    ended |= m.p == T(0);
  }
  __device__ __forceinline__ Map<T> map() const { return Map<T>{ended ? T(0) : p, b}; }
};
template <typename T> __device__ __forceinline__ T apply(Map<T> m, T x) {
  return m.p == T(0) ? m.b : m.b + m.p * x;
}

// ------------------------------------------------------------------ many columns
// One thread per W columns (one 16-byte access, or one element) walks the steps backwards.
// The walk is a chain of loads' latencies, so the next stretch of steps is always on its way:
// 64 steps of 256,000 float columns take 49 us, 83% of the copy rate, against 78 without that
// and 178 with one column per thread. A flag byte is kept as loaded and the two flags are
// asked for together; testing the first before asking for the second cost a latency a step.
// Where that is too few threads to keep the memory busy the steps are cut into segments: a
// first launch leaves each segment's map, a second composes the maps of the segments after
// its own and walks its own again.
template <typename T, int W> struct alignas(W * sizeof(T)) Pack {
  T x[W];
};
constexpr int kColumnThreads = 64;

// kAhead steps of a thread's columns, the latest first
template <typename T, int W, int N, bool NEXT> struct Stretch {
  Pack<T, W> r[N], v[N], next[NEXT ? N : 1];
  // one byte for all columns or, where each has its own, a byte per column; as they were
  // loaded: an operation here would wait for each
  uint32_t term[N], trunc[N];
  static __device__ __forceinline__ uint32_t flags_at(const uint8_t* p, long long at, bool own) {
    if (!p) return 0;
    if (W == 1 || !own) return p[at];
    return W == 2 ? *reinterpret_cast<const uint16_t*>(p + at)
                  : *reinterpret_cast<const uint32_t*>(p + at);
  }
  // the steps below t, down to `low`
  __device__ __forceinline__ void load(const Args<T>& a, long long t, long long low, long long j,
                                       long long f) {
    using P = Pack<T, W>;
#pragma unroll
    for (int k = 0; k < N; ++k) {
      const long long step = t - 1 - k;
      if (step < low) return;
      const long long at = step * a.columns + j, g = step * a.flags + f;
      r[k] = *reinterpret_cast<const P*>(a.r + at);
      v[k] = *reinterpret_cast<const P*>(a.v + at);
      if (NEXT) next[NEXT ? k : 0] = *reinterpret_cast<const P*>(a.next + at);
      term[k] = flags_at(a.term, g, a.per_flag == 1);
      trunc[k] = flags_at(a.trunc, g, a.per_flag == 1);
    }
  }
  // A: the advantages after these steps, then before them; p: the product of the decays
  template <bool WRITE>
  __device__ __forceinline__ void walk(const Args<T>& a, long long t, long long low, long long j,
                                       Pack<T, W>& A, Pack<T, W>& after, Pack<T, W>& p) const {
    using P = Pack<T, W>;
    const int apart = a.per_flag == 1 ? 8 : 0;
#pragma unroll
    for (int k = 0; k < N; ++k) {
      const long long step = t - 1 - k;
      if (step < low) return;
      P ret;
#pragma unroll
      for (int c = 0; c < W; ++c) {
        const bool ended = term[k] >> (apart * c) & 255u;
        const bool stop = ended || (trunc[k] >> (apart * c) & 255u) || a.decay == T(0);
        const T follow = NEXT ? next[NEXT ? k : 0].x[c] : after.x[c];
        const T d = r[k].x[c] + (ended ? T(0) : a.gamma * follow) - v[k].x[c];
        A.x[c] = stop ? d : d + a.decay * A.x[c];
        ret.x[c] = A.x[c] + v[k].x[c];
        // an end is -0, and stays -0, which tells it from an underflow
        if (!WRITE) p.x[c] = stop ? -T(0) : p.x[c] * a.decay;
      }
      if (WRITE) {
        *reinterpret_cast<P*>(a.adv + step * a.columns + j) = A;
        *reinterpret_cast<P*>(a.ret + step * a.columns + j) = ret;
      }
      after = v[k];
    }
  }
};

// What the launch is of: all steps at once, the segments' maps, or the segments' steps.
enum Part { kAllSteps, kMaps, kSteps };

template <typename T, int W, bool NEXT, int PART>
__global__ void __launch_bounds__(kColumnThreads)
    gae_columns_kernel(Args<T> a, long long length, T* products, T* offsets) {
  constexpr int kAhead = W == 1 && PART != kAllSteps ? 8 : 4;
  using P = Pack<T, W>;
  const long long thread = blockIdx.x * static_cast<long long>(kColumnThreads) + threadIdx.x;
  const long long j = thread * W;
  if (j >= a.columns) return;
  const long long f = j / a.per_flag;  // the thread's first flag
  const long long seg = PART == kAllSteps ? 0 : blockIdx.y;
  const long long low = seg * length, high = min(a.steps, low + length);
  P A{}, after{}, p;
#pragma unroll
  for (int c = 0; c < W; ++c) p.x[c] = T(1);
  if (!NEXT)
    after = *reinterpret_cast<const P*>(high < a.steps ? a.v + high * a.columns + j : a.last + j);
  // one stretch is on its way while the other is walked
  Stretch<T, W, kAhead, NEXT> s0, s1;
  s0.load(a, high, low, j, f);
  if (PART == kSteps) {
    for (long long s = gridDim.y - 1; s > seg; --s) {
      const P q = *reinterpret_cast<const P*>(products + s * a.columns + j);
      const P b = *reinterpret_cast<const P*>(offsets + s * a.columns + j);
#pragma unroll
      for (int c = 0; c < W; ++c) A.x[c] = apply(Map<T>{q.x[c], b.x[c]}, A.x[c]);
    }
  }
  for (long long t = high; t > low; t -= 2 * kAhead) {
    s1.load(a, t - kAhead, low, j, f);
    s0.template walk<PART != kMaps>(a, t, low, j, A, after, p);
    s0.load(a, t - 2 * kAhead, low, j, f);
    s1.template walk<PART != kMaps>(a, t - kAhead, low, j, A, after, p);
  }
  if (PART == kMaps) {
#pragma unroll
    for (int c = 0; c < W; ++c)
      if (p.x[c] == T(0) && !signbit(p.x[c]) && a.decay > T(0)) p.x[c] = least<T>();
    *reinterpret_cast<P*>(products + seg * a.columns + j) = p;
    *reinterpret_cast<P*>(offsets + seg * a.columns + j) = A;
  }
}

// ------------------------------------------------------------------- few columns
// (32,768 steps of six columns: 4 + 6 us, most of it maps composed one after another: a thread of
// the second kernel goes through its part of the later segments' and then through the n parts and
// the runs after its own, n the CTA's runs of a column, 32 here and up to 256; the first kernel's
// last step is such a chain too. Threads of their own took 6.3 ms, one for each column.) The steps are cut into segments, one per CTA, and a segment into runs of kRun steps, one
// per thread. A thread forms its run's map from its own steps, the CTA composes the runs', and
// the first kernel leaves the segment's map. The second kernel
// composes the maps of the segments after its own, which is the advantage that follows it,
// and walks its runs again with that.
constexpr int kRun = 8;
constexpr int kCtaThreads = 256;

// Columns per CTA: a power of two up to 32, the least that holds them all.
inline int tile_columns(long long columns) {
  int c = 1;
  while (c < 32 && c < columns) c *= 2;
  return c;
}

template <typename T, bool FINAL>
__global__ void __launch_bounds__(kCtaThreads)
    gae_segments_kernel(Args<T> a, int tile, long long segments, Map<T>* maps) {
  __shared__ Map<T> runs[kCtaThreads];
  const int c = threadIdx.x % tile, q = threadIdx.x / tile, n = kCtaThreads / tile;
  const long long seg = blockIdx.x, j = blockIdx.y * static_cast<long long>(tile) + c;
  const bool in = j < a.columns;
  const long long f = in ? j / a.per_flag : 0;
  const long long t0 = (seg * n + q) * kRun;  // the run's first step
  Step<T> s[kRun];
  T after_v = 0;
#pragma unroll
  for (int k = 0; k < kRun; ++k)
    if (in && t0 + k < a.steps) s[k] = load_step(a, t0 + k, j, f);
  if (in && !a.next && t0 < a.steps)
    after_v = t0 + kRun < a.steps ? a.v[(t0 + kRun) * a.columns + j] : a.last[j];
  T x = 0;  // the advantage after the CTA's segment
  if (FINAL) {
    // the later segments in n parts, then the parts in order
    const long long later = segments - 1 - seg, each = (later + n - 1) / n;
    Chain<T> m;
    for (long long k = seg + 1 + q * each; in && k < seg + 1 + min((q + 1) * each, later); ++k)
      m.then(maps[k * a.columns + j]);
    runs[threadIdx.x] = m.map();
    __syncthreads();
    for (int k = n - 1; k >= 0; --k) x = apply(runs[k * tile + c], x);
    __syncthreads();
  }
  T d[kRun];
  Map<T> m{T(1), T(0)};
  bool ended = false;
#pragma unroll
  for (int k = kRun - 1; k >= 0; --k) {
    d[k] = 0;
    if (in && t0 + k < a.steps) {
      d[k] = s[k].r + (s[k].term ? T(0) : a.gamma * (a.next ? s[k].next : after_v)) - s[k].v;
      after_v = s[k].v;
      m.b = s[k].stop ? d[k] : d[k] + a.decay * m.b;
      m.p *= a.decay;
      ended |= s[k].stop;
    }
  }
  m.p = ended ? T(0) : m.p == T(0) ? least<T>() : m.p;
  runs[threadIdx.x] = m;
  __syncthreads();
  if constexpr (FINAL) {
    for (int k = n - 1; k > q; --k) x = apply(runs[k * tile + c], x);
#pragma unroll
    for (int k = kRun - 1; k >= 0; --k) {
      if (in && t0 + k < a.steps) {
        x = s[k].stop ? d[k] : d[k] + a.decay * x;
        const long long at = (t0 + k) * a.columns + j;
        a.adv[at] = x;
        a.ret[at] = x + s[k].v;
      }
    }
  } else if (q == 0 && in) {
    Chain<T> all;
    for (int k = 0; k < n; ++k) all.then(runs[k * tile + c]);
    maps[seg * a.columns + j] = all.map();
  }
}

// Below this many columns a row of them is too short to be read by threads of their own
// (32,768 steps of 257 columns: 112 us by threads; of 255 by runs in CTAs: 146 us).
constexpr long long kFewColumns = 128;
// Threads that keep the memory busy, and the fewest steps worth a segment of their own.
constexpr long long kEnough = 148 * 64 * 3;
constexpr long long kShortest = 32;

struct Plan {
  bool few;
  int tile;                       // few: columns per CTA
  long long segments, length;     // length: steps of a segment, where not few
  int width;                      // columns per thread, where not few
  size_t offsets_at, bytes;
};
Plan plan_of(const swarp_gae_t* g) {
  Plan q{};
  const size_t one = g->dtype == SWARP_F32 ? sizeof(float) : sizeof(double);
  q.few = g->columns < kFewColumns && g->steps > kRun;
  if (q.few) {
    q.tile = tile_columns(g->columns);
    const long long per = static_cast<long long>(kCtaThreads / q.tile) * kRun;
    q.segments = (g->steps + per - 1) / per;
    if (q.segments > 1) q.bytes = 2 * one * q.segments * g->columns;
    return q;
  }
  // whole packs that share a flag or have one each, all of them aligned
  q.width = static_cast<int>(16 / one);
  const bool flags = g->terminated || g->truncated, own = g->columns_per_flag == 1;
  if (g->columns % q.width != 0 || (flags && !own && g->columns_per_flag % q.width != 0))
    q.width = 1;
  if (own)  // a pack's flags are one access
    for (const uint8_t* p : {g->terminated, g->truncated})
      if (reinterpret_cast<uintptr_t>(p) % 4 != 0) q.width = 1;
  for (const void* p : {g->rewards, g->values, g->next_values, g->last_values,
                        static_cast<const void*>(g->advantages),
                        static_cast<const void*>(g->returns)})
    if (reinterpret_cast<uintptr_t>(p) % 16 != 0) q.width = 1;
  const long long threads = g->columns / q.width;
  long long n = threads > 0 ? (kEnough + threads - 1) / threads : 1;
  const long long most = (g->steps + kShortest - 1) / kShortest;
  // with more than half of them there, reading everything twice costs more than it gives
  n = n <= 2 ? 1 : n < most ? n : most;
  if (n < 1) n = 1;
  q.length = (g->steps + n - 1) / n;
  q.segments = q.length > 0 ? (g->steps + q.length - 1) / q.length : 1;
  if (q.segments > 1) {
    q.offsets_at = align256(one * q.segments * g->columns);
    q.bytes = q.offsets_at + one * q.segments * g->columns;
  }
  return q;
}

int check(const swarp_gae_t* g) {
  if (!g || g->steps < 0 || g->columns < 0 || g->columns_per_flag < 1) return SWARP_ERR_INVALID_ARG;
  if (g->columns % g->columns_per_flag != 0) return SWARP_ERR_INVALID_ARG;
  if (g->dtype != SWARP_F32 && g->dtype != SWARP_F64) return SWARP_ERR_INVALID_ARG;
  return SWARP_OK;
}

template <typename T, int W, bool NEXT>
int columns(const Args<T>& a, const Plan& q, void* ws, cudaStream_t st) {
  const long long threads = a.columns / W;
  const dim3 grid(static_cast<unsigned>((threads + kColumnThreads - 1) / kColumnThreads),
                  static_cast<unsigned>(q.segments));
  if (q.segments == 1) {
    gae_columns_kernel<T, W, NEXT, kAllSteps>
        <<<grid, kColumnThreads, 0, st>>>(a, a.steps, nullptr, nullptr);
    return launch_status();
  }
  T* products = static_cast<T*>(ws);
  T* offsets = reinterpret_cast<T*>(static_cast<char*>(ws) + q.offsets_at);
  gae_columns_kernel<T, W, NEXT, kMaps>
      <<<grid, kColumnThreads, 0, st>>>(a, q.length, products, offsets);
  if (const int rc = launch_status()) return rc;
  gae_columns_kernel<T, W, NEXT, kSteps>
      <<<grid, kColumnThreads, 0, st>>>(a, q.length, products, offsets);
  return launch_status();
}

template <typename T> int run(const swarp_gae_t* g, const Plan& q, void* ws, cudaStream_t st) {
  Args<T> a{static_cast<const T*>(g->rewards), static_cast<const T*>(g->values),
            static_cast<const T*>(g->next_values), static_cast<const T*>(g->last_values),
            g->terminated, g->truncated, static_cast<T*>(g->advantages),
            static_cast<T*>(g->returns), g->steps, g->columns, g->columns / g->columns_per_flag,
            g->columns_per_flag, static_cast<T>(g->gamma), static_cast<T>(g->gamma * g->lambda)};
  if (q.few) {
    Map<T>* maps = static_cast<Map<T>*>(ws);
    const long long tiles = (g->columns + q.tile - 1) / q.tile;
    const dim3 grid(static_cast<unsigned>(q.segments), static_cast<unsigned>(tiles));
    if (q.segments > 1) {
      gae_segments_kernel<T, false><<<grid, kCtaThreads, 0, st>>>(a, q.tile, q.segments, maps);
      if (const int rc = launch_status()) return rc;
    }
    gae_segments_kernel<T, true><<<grid, kCtaThreads, 0, st>>>(a, q.tile, q.segments, maps);
    return launch_status();
  }
  return q.width == 1 ? (a.next ? columns<T, 1, true>(a, q, ws, st)
                                : columns<T, 1, false>(a, q, ws, st))
                      : (a.next ? columns<T, 16 / sizeof(T), true>(a, q, ws, st)
                                : columns<T, 16 / sizeof(T), false>(a, q, ws, st));
}

}  // namespace
}  // namespace learn
}  // namespace swarp

using namespace swarp::learn;

extern "C" {

size_t swarp_gae_workspace_bytes(const swarp_gae_t* g) {
  return check(g) == SWARP_OK ? plan_of(g).bytes : 0;
}

int swarp_gae(const swarp_gae_t* g, void* workspace, size_t workspace_bytes, void* stream) {
  if (const int rc = check(g)) return rc;
  if (g->steps == 0 || g->columns == 0) return SWARP_OK;
  if (!g->rewards || !g->values || !g->advantages || !g->returns ||
      (!g->next_values && !g->last_values))
    return SWARP_ERR_INVALID_ARG;
  const Plan q = plan_of(g);
  if (q.bytes > 0 && (!workspace || workspace_bytes < q.bytes)) return SWARP_ERR_WORKSPACE;
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  return g->dtype == SWARP_F32 ? run<float>(g, q, workspace, st)
                               : run<double>(g, q, workspace, st);
}

}  // extern "C"
