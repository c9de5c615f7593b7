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

// One thread per column walks the steps backwards.
template <typename T> __global__ void __launch_bounds__(256) gae_columns_kernel(Args<T> a) {
  const long long j = blockIdx.x * 256ll + threadIdx.x;
  if (j >= a.columns) return;
  const long long f = j / a.per_flag;
  T A = 0, after = a.next ? T(0) : a.last[j];
  for (long long t = a.steps - 1; t >= 0; --t) {
    const long long k = t * a.columns + j;
    const bool term = a.term && a.term[t * a.flags + f];
    const bool stop = term || (a.trunc && a.trunc[t * a.flags + f]);
    const T v = a.v[k], follow = a.next ? a.next[k] : after;
    const T d = a.r[k] + (term ? T(0) : a.gamma * follow) - v;
    A = stop ? d : d + a.decay * A;
    a.adv[k] = A;
    a.ret[k] = A + v;
    after = v;
  }
}

int check(const swarp_gae_t* g) {
  if (!g || g->steps < 0 || g->columns < 0 || g->columns_per_flag < 1) return SWARP_ERR_INVALID_ARG;
  if (g->columns % g->columns_per_flag != 0) return SWARP_ERR_INVALID_ARG;
  if (g->dtype != SWARP_F32 && g->dtype != SWARP_F64) return SWARP_ERR_INVALID_ARG;
  return SWARP_OK;
}

template <typename T> int run(const swarp_gae_t* g, cudaStream_t st) {
  Args<T> a{static_cast<const T*>(g->rewards), static_cast<const T*>(g->values),
            static_cast<const T*>(g->next_values), static_cast<const T*>(g->last_values),
            g->terminated, g->truncated, static_cast<T*>(g->advantages),
            static_cast<T*>(g->returns), g->steps, g->columns, g->columns / g->columns_per_flag,
            g->columns_per_flag, static_cast<T>(g->gamma), static_cast<T>(g->gamma * g->lambda)};
  gae_columns_kernel<T><<<(unsigned)((g->columns + 255) / 256), 256, 0, st>>>(a);
  return launch_status();
}

}  // namespace
}  // namespace learn
}  // namespace swarp

using namespace swarp::learn;

extern "C" {

size_t swarp_gae_workspace_bytes(const swarp_gae_t* g) {
  (void)g;
  return 0;
}

int swarp_gae(const swarp_gae_t* g, void* workspace, size_t workspace_bytes, void* stream) {
  if (const int rc = check(g)) return rc;
  if (g->steps == 0 || g->columns == 0) return SWARP_OK;
  if (!g->rewards || !g->values || !g->advantages || !g->returns ||
      (!g->next_values && !g->last_values))
    return SWARP_ERR_INVALID_ARG;
  const size_t need = swarp_gae_workspace_bytes(g);
  if (need > 0 && (!workspace || workspace_bytes < need)) return SWARP_ERR_WORKSPACE;
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  return g->dtype == SWARP_F32 ? run<float>(g, st) : run<double>(g, st);
}

}  // extern "C"
