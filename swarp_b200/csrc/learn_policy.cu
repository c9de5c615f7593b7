// The clipped policy loss over rows of token logits, and its gradient (swarp_policy_loss,
// swarp_policy_grad, swarp_token_logp; contracts in include/swarp_b200.h).
//
// With m = max z, S = sum e^(z - m) and a the row's token,
//   lp = z_a - m - ln S,   H = ln S - sum e^(z - m) (z - m) / S,   r = e^(lp - old)
//   dloss/dlp = c = -r A where the clip does not cut, + kl (1 - e^(ref - lp))
//   dloss/dz_j = c (1{j = a} - p_j) + ent p_j (ln p_j + H),        p_j = e^(z_j - m) / S
// so one row needs its maximum, two sums, and then one more look at its logits.
#include "learn.cuh"

namespace swarp {
namespace learn {
namespace {

constexpr int kCountBlocks = 64;
constexpr int kLoopThreads = 256;
constexpr int kLoopMaxBlocks = 148 * 8;
constexpr float kLog2e = 1.4426950408889634f;

struct Args {
  const void* logits;
  const void* tokens;
  const float *old_logp, *advantages, *ref_logp;
  const uint8_t* mask;
  const float* cotangent;  // gradient call: scales grad
  const long long* counts; // [kCountBlocks] admitted rows, where mask and mean
  float *logp, *entropy;
  double* partials;        // [blocks][4]
  void* grad;
  long long rows, vocab, inner, stride_outer, stride_inner;
  float lo, hi, kl, ent, grad_scale;
  int tokens_64, mean, skip_unit, with_loss;
};

__device__ __forceinline__ long long row_offset(const Args& a, long long i) {
  return a.inner == a.rows ? i * a.stride_inner
                           : (i / a.inner) * a.stride_outer + (i % a.inner) * a.stride_inner;
}
__device__ __forceinline__ long long token_of(const Args& a, long long i) {
  return a.tokens_64 ? static_cast<const long long*>(a.tokens)[i]
                     : static_cast<const int*>(a.tokens)[i];
}

// 1 / the number of admitted rows (or 1 for a sum); every lane of the warp gets it
__device__ __forceinline__ float row_weight(const Args& a) {
  if (!a.mean) return 1.f;
  long long n = a.rows;
  if (a.mask) {
    n = 0;
    for (int k = threadIdx.x & 31; k < kCountBlocks; k += 32) n += a.counts[k];
    n = warp_sum(n);
  }
  return n > 0 ? 1.f / static_cast<float>(n) : 0.f;
}

struct Row {
  float lp, H, pg, k3, cut;
  float c;  // d(row loss) / d(lp)
};

// The scalar part of a row from its log probability and entropy.
__device__ __forceinline__ Row row_terms(const Args& a, long long i, float lp, float H,
                                         bool empty) {
  Row r{lp, H, 0.f, 0.f, 0.f, 0.f};
  if (empty || !a.with_loss) return r;
  const float A = a.advantages[i];
  const float ratio = expf(lp - a.old_logp[i]);
  const float bounded = fminf(fmaxf(ratio, 1.f - a.lo), 1.f + a.hi);
  const float s1 = ratio * A, s2 = (ratio != ratio ? ratio : bounded) * A;
  r.pg = s1 != s1 ? -s1 : -fminf(s1, s2);
  const bool cut = (A > 0.f && ratio > 1.f + a.hi) || (A < 0.f && ratio < 1.f - a.lo);
  r.cut = cut ? 1.f : 0.f;
  r.c = cut ? 0.f : -s1;
  if (a.ref_logp) {
    const float d = a.ref_logp[i] - lp;
    r.k3 = expm1f(d) - d;
    if (a.kl != 0.f) r.c -= a.kl * expm1f(d);
  }
  return r;
}

// ------------------------------------------------------------------ admitted rows
__global__ void count_kernel(const uint8_t* mask, long long n, long long* counts) {
  __shared__ long long part[8];
  long long c = 0;
  for (long long i = blockIdx.x * 256ll + threadIdx.x; i < n; i += 256ll * kCountBlocks)
    c += mask[i] != 0;
  c = warp_sum(c);
  if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = c;
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int w = 1; w < 8; ++w) c += part[w];
    counts[blockIdx.x] = c;
  }
}

// ------------------------------------------------------------- any row, any length
// One CTA per row at a time, the row read three times (maximum, sums, gradient), the later
// reads from L1 or L2.
struct Block {
  float f[kLoopThreads / 32];
  float g[kLoopThreads / 32];
};
__device__ __forceinline__ float block_max(float v, Block& b) {
  v = warp_max(v);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) b.f[threadIdx.x >> 5] = v;
  __syncthreads();
  v = b.f[0];
  for (int w = 1; w < kLoopThreads / 32; ++w) v = max_nan(v, b.f[w]);
  return v;
}
__device__ __forceinline__ void block_sum2(float& s, float& t, Block& b) {
  s = warp_sum(s);
  t = warp_sum(t);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) b.f[threadIdx.x >> 5] = s, b.g[threadIdx.x >> 5] = t;
  __syncthreads();
  s = t = 0.f;
  for (int w = 0; w < kLoopThreads / 32; ++w) s += b.f[w], t += b.g[w];
}

template <typename T, bool GRAD>
__global__ void __launch_bounds__(kLoopThreads) policy_loop_kernel(Args a) {
  __shared__ Block sh;
  const float cot = a.cotangent ? *a.cotangent : 1.f;
  if (a.skip_unit && cot == 1.f) return;
  const float w = row_weight(a);
  const float wg = w * a.grad_scale * cot;
  double sums[4] = {0, 0, 0, 0};
  for (long long i = blockIdx.x; i < a.rows; i += gridDim.x) {
    T* g = GRAD ? static_cast<T*>(a.grad) + i * a.vocab : nullptr;
    if (a.mask && !a.mask[i]) {
      if (GRAD)
        for (long long j = threadIdx.x; j < a.vocab; j += kLoopThreads) g[j] = from_f<T>(0.f);
      if (threadIdx.x == 0 && a.logp) a.logp[i] = 0.f, a.entropy[i] = 0.f;
      continue;
    }
    const T* z = static_cast<const T*>(a.logits) + row_offset(a, i);
    float m = -INFINITY;
    for (long long j = threadIdx.x; j < a.vocab; j += kLoopThreads) m = max_nan(m, to_f(z[j]));
    m = block_max(m, sh);
    const bool empty = m == -INFINITY;
    if (empty) m = 0.f;
    float s = 0.f, t = 0.f;
    for (long long j = threadIdx.x; j < a.vocab; j += kLoopThreads) {
      const float x = to_f(z[j]) - m, e = exp2f(x * kLog2e);
      s += e;
      t = fmaf(e, max_nan(x, -1e4f), t);
    }
    block_sum2(s, t, sh);
    const float ln = logf(s);
    const long long tok = token_of(a, i);
    const float za = tok >= 0 && tok < a.vocab ? to_f(z[tok]) : NAN;
    const Row r = row_terms(a, i, empty ? (za != za ? za : -INFINITY) : (za - m) - ln,
                            empty ? 0.f : ln - t / s, empty && za == za);
    if (GRAD) {
      // a token outside the vocabulary leaves c = NaN, and with it the row's gradient
      const float c = wg * r.c, inv = empty ? 0.f : 1.f / s, eta = wg * a.ent;
      for (long long j = threadIdx.x; j < a.vocab; j += kLoopThreads) {
        const float x = to_f(z[j]) - m, p = exp2f(x * kLog2e) * inv;
        float d = -c * p;
        if (a.ent != 0.f) d = fmaf(eta * p, max_nan(x, -1e4f) - (empty ? 0.f : ln) + r.H, d);
        if (j == tok) d += c;
        g[j] = from_f<T>(d);
      }
    }
    if (threadIdx.x == 0) {
      if (a.logp) a.logp[i] = r.lp, a.entropy[i] = r.H;
      sums[0] += r.pg, sums[1] += r.k3, sums[2] += r.H, sums[3] += r.cut;
    }
  }
  if (threadIdx.x == 0 && a.partials)
    for (int k = 0; k < 4; ++k) a.partials[blockIdx.x * 4ll + k] = sums[k] * w;
}

// ---------------------------------------------------------------------- the scalars
__global__ void scalars_kernel(const double* partials, long long n, float kl, float ent,
                               float* loss, float* stats) {
  __shared__ double part[8][4];
  double s[4] = {0, 0, 0, 0};
  for (long long i = threadIdx.x; i < n; i += 256)
    for (int k = 0; k < 4; ++k) s[k] += partials[i * 4 + k];
  for (int k = 0; k < 4; ++k) {
    s[k] = warp_sum(s[k]);
    if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5][k] = s[k];
  }
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int w = 1; w < 8; ++w)
      for (int k = 0; k < 4; ++k) s[k] += part[w][k];
    double l = s[0];  // a coefficient of 0 takes its term out, whatever its value
    if (kl != 0.f) l += static_cast<double>(kl) * s[1];
    if (ent != 0.f) l -= static_cast<double>(ent) * s[2];
    *loss = static_cast<float>(l);
    for (int k = 0; k < 4; ++k) stats[k] = static_cast<float>(s[k]);
  }
}

// -------------------------------------------------------------------------- the host
struct Plan {
  long long blocks;
  size_t partials_at, bytes;
};

int check(const swarp_policy_t* p) {
  if (!p || p->rows < 0 || p->vocab < 1 || p->vocab > 0x7fffffffll) return SWARP_ERR_INVALID_ARG;
  if (p->dtype != SWARP_F32 && p->dtype != SWARP_BF16 && p->dtype != SWARP_F16)
    return SWARP_ERR_INVALID_ARG;
  if (p->rows > 0 && (p->inner < 1 || p->rows % p->inner != 0)) return SWARP_ERR_INVALID_ARG;
  return SWARP_OK;
}
Plan plan_of(const swarp_policy_t* p) {
  Plan q;
  q.blocks = p->rows < kLoopMaxBlocks ? p->rows : kLoopMaxBlocks;
  q.partials_at = align256(kCountBlocks * sizeof(long long));
  q.bytes = q.partials_at + align256(sizeof(double) * 4 * (q.blocks > 0 ? q.blocks : 1));
  return q;
}

template <typename T> int run_typed(const Args& a, const Plan& q, cudaStream_t st) {
  if (a.grad)
    policy_loop_kernel<T, true><<<(unsigned)q.blocks, kLoopThreads, 0, st>>>(a);
  else
    policy_loop_kernel<T, false><<<(unsigned)q.blocks, kLoopThreads, 0, st>>>(a);
  return launch_status();
}

enum Call { kLoss, kGrad, kLogp };

int run(const swarp_policy_t* p, Call call, const float* cotangent, int skip_unit,
        void* workspace, size_t workspace_bytes, cudaStream_t st) {
  if (const int rc = check(p)) return rc;
  const bool loss = call == kLoss, some = p->rows > 0;
  if (some && (!p->logits || !p->tokens)) return SWARP_ERR_INVALID_ARG;
  if (call != kLogp && some && (!p->old_logp || !p->advantages)) return SWARP_ERR_INVALID_ARG;
  if (call != kGrad && some && (!p->logp || !p->entropy)) return SWARP_ERR_INVALID_ARG;
  if (loss && (!p->loss || !p->stats)) return SWARP_ERR_INVALID_ARG;
  if (call == kGrad && (!cotangent || (some && !p->grad))) return SWARP_ERR_INVALID_ARG;
  const Plan q = plan_of(p);
  if (!workspace || workspace_bytes < q.bytes) return SWARP_ERR_WORKSPACE;
  char* ws = static_cast<char*>(workspace);
  Args a{};
  a.logits = p->logits;
  a.tokens = p->tokens;
  a.old_logp = p->old_logp;
  a.advantages = p->advantages;
  a.ref_logp = p->ref_logp;
  a.mask = call == kLogp ? nullptr : p->mask;
  a.cotangent = cotangent;
  a.counts = reinterpret_cast<const long long*>(ws);
  a.logp = call == kGrad ? nullptr : p->logp;
  a.entropy = p->entropy;
  a.partials = loss ? reinterpret_cast<double*>(ws + q.partials_at) : nullptr;
  a.grad = call == kLogp ? nullptr : p->grad;
  a.rows = p->rows;
  a.vocab = p->vocab;
  a.inner = p->inner;
  a.stride_outer = p->stride_outer;
  a.stride_inner = p->stride_inner;
  a.lo = p->clip_low;
  a.hi = p->clip_high;
  a.kl = p->kl_coef;
  a.ent = p->entropy_coef;
  a.grad_scale = p->grad_scale;
  a.tokens_64 = p->tokens_64;
  a.mean = p->mean;
  a.skip_unit = skip_unit;
  a.with_loss = call != kLogp;
  if (some) {
    if (a.mask && a.mean) {
      count_kernel<<<kCountBlocks, 256, 0, st>>>(a.mask, a.rows, reinterpret_cast<long long*>(ws));
      if (const int rc = launch_status()) return rc;
    }
    const int rc = p->dtype == SWARP_F32    ? run_typed<float>(a, q, st)
                   : p->dtype == SWARP_BF16 ? run_typed<__nv_bfloat16>(a, q, st)
                                            : run_typed<__half>(a, q, st);
    if (rc) return rc;
  }
  if (loss) {
    scalars_kernel<<<1, 256, 0, st>>>(a.partials, some ? q.blocks : 0, a.kl, a.ent, p->loss,
                                   p->stats);
    return launch_status();
  }
  return SWARP_OK;
}

}  // namespace
}  // namespace learn
}  // namespace swarp

using namespace swarp::learn;

extern "C" {

size_t swarp_policy_workspace_bytes(const swarp_policy_t* p) {
  return check(p) == SWARP_OK ? plan_of(p).bytes : 0;
}
int swarp_policy_loss(const swarp_policy_t* p, void* workspace, size_t workspace_bytes,
                      void* stream) {
  return run(p, kLoss, nullptr, 0, workspace, workspace_bytes, static_cast<cudaStream_t>(stream));
}
int swarp_policy_grad(const swarp_policy_t* p, const float* cotangent, int32_t skip_unit,
                      void* workspace, size_t workspace_bytes, void* stream) {
  return run(p, kGrad, cotangent, skip_unit, workspace, workspace_bytes,
             static_cast<cudaStream_t>(stream));
}
int swarp_token_logp(const swarp_policy_t* p, void* workspace, size_t workspace_bytes,
                     void* stream) {
  return run(p, kLogp, nullptr, 0, workspace, workspace_bytes, static_cast<cudaStream_t>(stream));
}

}  // extern "C"
