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

// ------------------------------------------------------------------ many columns
// One thread per W columns (one 16-byte access, or one element) walks the steps backwards.
template <typename T, int W> struct alignas(W * sizeof(T)) Pack {
  T x[W];
};
constexpr int kColumnThreads = 64;

// kAhead steps of a thread's columns, the latest first
template <typename T, int W, int N, bool NEXT> struct Stretch {
  Pack<T, W> r[N], v[N], next[NEXT ? N : 1];
  uint8_t term[N], trunc[N];
  __device__ __forceinline__ void load(const Args<T>& a, long long t, long long j, long long f) {
    using P = Pack<T, W>;
#pragma unroll
    for (int k = 0; k < N; ++k) {
      const long long step = t - 1 - k;
      if (step < 0) return;
      const long long at = step * a.columns + j, g = step * a.flags + f;
      r[k] = *reinterpret_cast<const P*>(a.r + at);
      v[k] = *reinterpret_cast<const P*>(a.v + at);
      if (NEXT) next[NEXT ? k : 0] = *reinterpret_cast<const P*>(a.next + at);
      term[k] = a.term ? a.term[g] : 0;
      trunc[k] = a.trunc ? a.trunc[g] : 0;
    }
  }
  __device__ __forceinline__ void walk(const Args<T>& a, long long t, long long j,
                                       Pack<T, W>& A, Pack<T, W>& after) const {
    using P = Pack<T, W>;
#pragma unroll
    for (int k = 0; k < N; ++k) {
      const long long step = t - 1 - k;
      if (step < 0) return;
      const bool ended = term[k], stop = term[k] | trunc[k] | (a.decay == T(0));
      P ret;
#pragma unroll
      for (int c = 0; c < W; ++c) {
        const T follow = NEXT ? next[NEXT ? k : 0].x[c] : after.x[c];
        const T d = r[k].x[c] + (ended ? T(0) : a.gamma * follow) - v[k].x[c];
        A.x[c] = stop ? d : d + a.decay * A.x[c];
        ret.x[c] = A.x[c] + v[k].x[c];
      }
      *reinterpret_cast<P*>(a.adv + step * a.columns + j) = A;
      *reinterpret_cast<P*>(a.ret + step * a.columns + j) = ret;
      after = v[k];
    }
  }
};

template <typename T, int W, bool NEXT>
__global__ void __launch_bounds__(kColumnThreads) gae_columns_kernel(Args<T> a) {
  constexpr int kAhead = 4;
  using P = Pack<T, W>;
  const long long j = (blockIdx.x * static_cast<long long>(kColumnThreads) + threadIdx.x) * W;
  if (j >= a.columns) return;
  const long long f = j / a.per_flag;  // W columns share their flags
  P A{}, after{};
  if (!NEXT) after = *reinterpret_cast<const P*>(a.last + j);
  // one stretch is on its way while the other is walked
  Stretch<T, W, kAhead, NEXT> s0, s1;
  s0.load(a, a.steps, j, f);
  for (long long t = a.steps; t > 0; t -= 2 * kAhead) {
    s1.load(a, t - kAhead, j, f);
    s0.walk(a, t, j, A, after);
    s0.load(a, t - 2 * kAhead, j, f);
    s1.walk(a, t - kAhead, j, A, after);
  }
}

// ------------------------------------------------------------------- few columns
// The steps are cut into segments, one per CTA, and a segment into runs of kRun steps, one
// per thread. A run takes the advantage x after it to b + p x before it, with p the product
// of its decays; such maps compose, so a thread forms its run's map from its own steps, the
// CTA composes the runs', and the first kernel leaves the segment's map. The second kernel
// composes the maps of the segments after its own, which is the advantage that follows it,
// and walks its runs again with that.
constexpr int kRun = 8;
constexpr int kCtaThreads = 256;

template <typename T> struct Map {
  T p, b;  // x -> b + p x
};
// an end of an episode (p = 0) keeps whatever is after it out, NaN included
template <typename T> __device__ __forceinline__ Map<T> after(Map<T> first, Map<T> then) {
  // `first` is the earlier stretch of time: x -> first(then(x))
  return Map<T>{first.p * then.p, first.p == T(0) ? first.b : first.b + first.p * then.b};
}
template <typename T> __device__ __forceinline__ T apply(Map<T> m, T x) {
  return m.p == T(0) ? m.b : m.b + m.p * x;
}

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
    Map<T> m{T(1), T(0)};
    for (long long k = seg + 1 + q * each; in && k < seg + 1 + min((q + 1) * each, later); ++k)
      m = after(m, maps[k * a.columns + j]);
    runs[threadIdx.x] = m;
    __syncthreads();
    for (int k = n - 1; k >= 0; --k) x = apply(runs[k * tile + c], x);
    __syncthreads();
  }
  T d[kRun];
  Map<T> m{T(1), T(0)};
#pragma unroll
  for (int k = kRun - 1; k >= 0; --k) {
    d[k] = 0;
    if (in && t0 + k < a.steps) {
      d[k] = s[k].r + (s[k].term ? T(0) : a.gamma * (a.next ? s[k].next : after_v)) - s[k].v;
      after_v = s[k].v;
      m = after(Map<T>{s[k].stop ? T(0) : a.decay, d[k]}, m);
    }
  }
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
    for (int k = 1; k < n; ++k) m = after(m, runs[k * tile + c]);
    maps[seg * a.columns + j] = m;
  }
}

// Threads of their own for all columns keep the memory busy from about this many on.
constexpr long long kManyColumns = 32768;

struct Plan {
  bool split;
  int tile;
  long long segments;
  size_t bytes;
};
Plan plan_of(const swarp_gae_t* g) {
  Plan q{};
  q.tile = tile_columns(g->columns);
  q.split = g->columns < kManyColumns && g->steps > kRun;
  if (q.split) {
    const long long per = static_cast<long long>(kCtaThreads / q.tile) * kRun;
    q.segments = (g->steps + per - 1) / per;
    const size_t one = g->dtype == SWARP_F32 ? sizeof(Map<float>) : sizeof(Map<double>);
    if (q.segments > 1) q.bytes = one * q.segments * g->columns;
  }
  return q;
}

int check(const swarp_gae_t* g) {
  if (!g || g->steps < 0 || g->columns < 0 || g->columns_per_flag < 1) return SWARP_ERR_INVALID_ARG;
  if (g->columns % g->columns_per_flag != 0) return SWARP_ERR_INVALID_ARG;
  if (g->dtype != SWARP_F32 && g->dtype != SWARP_F64) return SWARP_ERR_INVALID_ARG;
  return SWARP_OK;
}

template <typename T> int run(const swarp_gae_t* g, const Plan& q, void* ws, cudaStream_t st) {
  Args<T> a{static_cast<const T*>(g->rewards), static_cast<const T*>(g->values),
            static_cast<const T*>(g->next_values), static_cast<const T*>(g->last_values),
            g->terminated, g->truncated, static_cast<T*>(g->advantages),
            static_cast<T*>(g->returns), g->steps, g->columns, g->columns / g->columns_per_flag,
            g->columns_per_flag, static_cast<T>(g->gamma), static_cast<T>(g->gamma * g->lambda)};
  if (q.split) {
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
  constexpr int W = 16 / sizeof(T);
  // whole packs that share a flag, all of them aligned
  const bool flagged = a.term || a.trunc;
  bool packs = a.columns % W == 0 && (!flagged || a.per_flag % W == 0);
  for (const void* p : {static_cast<const void*>(a.r), static_cast<const void*>(a.v),
                        static_cast<const void*>(a.next), static_cast<const void*>(a.last),
                        static_cast<const void*>(a.adv), static_cast<const void*>(a.ret)})
    packs = packs && reinterpret_cast<uintptr_t>(p) % 16 == 0;
  const long long threads = packs ? a.columns / W : a.columns;
  const unsigned blocks = static_cast<unsigned>((threads + kColumnThreads - 1) / kColumnThreads);
  auto* kernel = packs ? (a.next ? gae_columns_kernel<T, W, true> : gae_columns_kernel<T, W, false>)
                       : (a.next ? gae_columns_kernel<T, 1, true> : gae_columns_kernel<T, 1, false>);
  kernel<<<blocks, kColumnThreads, 0, st>>>(a);
  return launch_status();
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
