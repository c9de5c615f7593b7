// The clipped policy loss over rows of token logits, and its gradient (swarp_policy_loss,
// swarp_policy_grad, swarp_token_logp; contracts in include/swarp_b200.h).
//
// With m = max z, S = sum e^(z - m) and a the row's token,
//   lp = z_a - m - ln S,   H = ln S - sum e^(z - m) (z - m) / S,   r = e^(lp - old)
//   dloss/dlp = c = -r A where the clip does not cut, + kl (1 - e^(ref - lp))
//   dloss/dz_j = c (1{j = a} - p_j) + ent p_j (ln p_j + H),        p_j = e^(z_j - m) / S
// so one row needs its maximum, two sums, and then one more look at its logits.
#include <atomic>
#include <cstdlib>
#include <type_traits>

#include "learn.cuh"

namespace swarp {
namespace learn {
namespace {

constexpr int kCountBlocks = 64;
constexpr int kLoopThreads = 256;
constexpr int kLoopMaxBlocks = 148 * 8;
constexpr long long kWaitClocks = 1ll << 31;  // about a second
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;

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
  long long wait_clocks;   // limit of a wait for a part of a row
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

// What a row's scalar part reads; the kernels load it ahead of the row.
struct Inputs {
  float old, adv, ref;
};
__device__ __forceinline__ Inputs inputs_of(const Args& a, long long i) {
  Inputs x{0.f, 0.f, 0.f};
  if (a.with_loss) {
    x.old = a.old_logp[i];
    x.adv = a.advantages[i];
    if (a.ref_logp) x.ref = a.ref_logp[i];
  }
  return x;
}

// The scalar part of a row from its log probability and entropy. The exponentials are good to
// a few ulp at the arguments that a ratio or a divergence has.
__device__ __forceinline__ Row row_terms(const Args& a, const Inputs& x, float lp, float H,
                                         bool empty) {
  Row r{lp, H, 0.f, 0.f, 0.f, 0.f};
  if (empty || !a.with_loss) return r;
  const float A = x.adv;
  const float ratio = exp2_fast((lp - x.old) * kLog2e);
  const float bounded = fminf(fmaxf(ratio, 1.f - a.lo), 1.f + a.hi);
  const float s1 = ratio * A, s2 = bounded * A;
  r.pg = s1 != s1 ? -s1 : -fminf(s1, s2);
  const bool cut = (A > 0.f && ratio > 1.f + a.hi) || (A < 0.f && ratio < 1.f - a.lo);
  r.cut = cut ? 1.f : 0.f;
  r.c = cut ? 0.f : -s1;
  if (a.ref_logp) {
    const float d = x.ref - lp;
    // e^d - d - 1 and e^d - 1 without the cancellation: d^2 (1/2 + d/6 + ... + d^7/9!), what is
    // left out is below 2^-28 of it for |d| < 1/2. The policy is near its reference as a rule.
    float k3 = 1.f / 362880.f;
    k3 = fmaf(k3, d, 1.f / 40320.f);
    k3 = fmaf(k3, d, 1.f / 5040.f);
    k3 = fmaf(k3, d, 1.f / 720.f);
    k3 = fmaf(k3, d, 1.f / 120.f);
    k3 = fmaf(k3, d, 1.f / 24.f);
    k3 = fmaf(k3, d, 1.f / 6.f);
    k3 = fmaf(k3, d, 0.5f) * d * d;
    float e1 = k3 + d;
    if (!(fabsf(d) < 0.5f)) {
      e1 = exp2_fast(d * kLog2e) - 1.f;
      k3 = e1 - d;
    }
    r.k3 = k3;
    if (a.kl != 0.f) r.c -= a.kl * e1;
  }
  return r;
}

// ------------------------------------------------------------------ admitted rows
__global__ void __launch_bounds__(256) count_kernel(const uint8_t* mask, long long n,
                                                    long long* counts) {
  __shared__ long long part[8];
  const long long at = blockIdx.x * 256ll + threadIdx.x, all = 256ll * kCountBlocks;
  long long c = 0, done = 0;
  if (reinterpret_cast<uintptr_t>(mask) % 16 == 0) {
    const uint4* v = reinterpret_cast<const uint4*>(mask);
    done = n / 16 * 16;
    for (long long i = at; i < n / 16; i += all) {
      const uint4 q = v[i];
      c += __popc(__vcmpne4(q.x, 0)) + __popc(__vcmpne4(q.y, 0)) + __popc(__vcmpne4(q.z, 0)) +
           __popc(__vcmpne4(q.w, 0));
    }
    c /= 8;
  }
  for (long long i = done + at; i < n; i += all) c += mask[i] != 0;
  c = warp_sum(c);
  if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = c;
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int w = 1; w < 8; ++w) c += part[w];
    counts[blockIdx.x] = c;
  }
}

// ------------------------------------------------------------------- short rows
// A group of L lanes takes R rows at a time, lane l of it the elements l, l + L, ... of each
// (E of them, in registers). The R sums over the L lanes are reduced by halving: in each of
// the first log2 R steps a lane hands half of its sums to its partner and keeps the other
// half, so R sums cost R - 1 + log2(L / R) shuffles instead of R log2 L, and leave row
// l / (L / R) with lane l. That lane then does the scalar part of its row, which would
// otherwise cost every lane more than the row's own elements. 200,000 rows of 128 floats take
// 46 us, 71% of the copy rate, bound by 42 instructions an element (61% of the issue slots); of
// 100 bf16 69 us, 20%, waiting for loads of two bytes.
template <int L, int R, typename Op>
__device__ __forceinline__ float reduce_rows(float (&v)[R], int lane, Op op) {
  int n = R;
#pragma unroll
  for (int d = L / 2; d; d >>= 1) {
    if (n > 1) {
      n >>= 1;
      const bool up = lane & d;
#pragma unroll
      for (int k = 0; k < R / 2; ++k) {
        if (k >= n) break;
        const float keep = up ? v[k + n] : v[k], give = up ? v[k] : v[k + n];
        v[k] = op(keep, __shfl_xor_sync(kAll, give, d));
      }
    } else {
      v[0] = op(v[0], __shfl_xor_sync(kAll, v[0], d));
    }
  }
  return v[0];
}

constexpr int kGroupThreads = 256;

template <typename T, int L, int E, int R, bool GRAD>
__global__ void __launch_bounds__(kGroupThreads) policy_group_kernel(Args a) {
  static_assert(R <= L || L == 1, "a lane owns one row");
  constexpr int kPerRow = L / R > 0 ? L / R : 1;  // lanes that share the ownership of a row
  const float cot = a.cotangent ? *a.cotangent : 1.f;
  if (a.skip_unit && cot == 1.f) return;
  const float w = row_weight(a), wg = w * a.grad_scale * cot;
  const int lane = threadIdx.x & 31, l = lane & (L - 1), base = lane - l;
  const int mine = l / kPerRow;
  const int V = static_cast<int>(a.vocab);
  auto most = [](float x, float y) { return max_nan(x, y); };
  auto plus = [](float x, float y) { return x + y; };
  double sums[4] = {0, 0, 0, 0};
  // the whole warp runs as long as one of its groups has rows
  const long long step = static_cast<long long>(gridDim.x) * (kGroupThreads / L) * R;
  long long i0 = (static_cast<long long>(blockIdx.x) * kGroupThreads + threadIdx.x) / L * R;
  for (long long w0 = i0 - base / L * R; w0 < a.rows; w0 += step, i0 += step) {
    const long long i = i0 + mine;
    const bool live = i < a.rows && (!a.mask || a.mask[i]);
    const unsigned lives = __ballot_sync(kAll, live) >> base;
    long long tok = -1;
    float za = 0.f;
    Inputs in0{0.f, 0.f, 0.f};
    if (live) {
      in0 = inputs_of(a, i);
      tok = token_of(a, i);
      za = NAN;
      if (tok >= 0 && tok < V) za = to_f((static_cast<const T*>(a.logits) + row_offset(a, i))[tok]);
    }
    float z[R][E];
    const bool flat = a.inner == a.rows;
    const T* p0 = static_cast<const T*>(a.logits) + i0 * a.stride_inner;
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const T* p = flat ? p0 + r * a.stride_inner
                        : static_cast<const T*>(a.logits) + row_offset(a, i0 + r);
      const bool in = lives >> (r * kPerRow) & 1u;
#pragma unroll
      for (int k = 0; k < E; ++k) {
        const int j = l + L * k;
        z[r][k] = in && j < V ? to_f(p[j]) : -INFINITY;
      }
    }
    float v[R];
#pragma unroll
    for (int r = 0; r < R; ++r) {
      v[r] = z[r][0];
#pragma unroll
      for (int k = 1; k < E; ++k) v[r] = max_nan(v[r], z[r][k]);
    }
    const float top = reduce_rows<L, R>(v, l, most);  // of the lane's own row
    const bool empty = top == -INFINITY;
    const float m = empty ? 0.f : top;
    float u[R], e[R][E];
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const float mr = __shfl_sync(kAll, m, base + r * kPerRow);
      v[r] = u[r] = 0.f;
#pragma unroll
      for (int k = 0; k < E; ++k) {
        // bounded below so that a barred token's e x is 0
        z[r][k] = max_nan(z[r][k] - mr, -1e4f);
        e[r][k] = exp2_fast(z[r][k] * kLog2e);
        v[r] += e[r][k];
        u[r] = fmaf(e[r][k], z[r][k], u[r]);
      }
    }
    const float s = reduce_rows<L, R>(v, l, plus), t = reduce_rows<L, R>(u, l, plus);
    const float ln = empty ? 0.f : __logf(s), inv = empty ? 0.f : __fdividef(1.f, s);
    const Row row = row_terms(a, in0, empty ? (za != za ? za : -INFINITY) : (za - m) - ln,
                              ln - t * inv, !live || (empty && za == za));
    if (l % kPerRow == 0 && live) {
      sums[0] += row.pg, sums[1] += row.k3, sums[2] += row.H, sums[3] += row.cut;
    }
    if (a.logp && l % kPerRow == 0 && i < a.rows) {
      a.logp[i] = live ? row.lp : 0.f;
      a.entropy[i] = live ? row.H : 0.f;
    }
    if (GRAD) {
      // d = e (k0 + k1 x), and c more at the token
      const float c = live ? wg * row.c : 0.f, eta = live ? wg * a.ent : 0.f;
      const float k0 = inv * (eta * (row.H - ln) - c), k1 = inv * eta;
#pragma unroll
      for (int r = 0; r < R; ++r) {
        const int from = base + r * kPerRow;
        const float k0r = __shfl_sync(kAll, k0, from), k1r = __shfl_sync(kAll, k1, from);
        const float cr = __shfl_sync(kAll, c, from);
        const int tr = __shfl_sync(kAll, static_cast<int>(tok), from);
        T* g = static_cast<T*>(a.grad) + (i0 + r) * V;
#pragma unroll
        for (int k = 0; k < E; ++k) {
          const int j = l + L * k;
          float d = e[r][k] * fmaf(k1r, z[r][k], k0r);
          if (j == tr) d += cr;
          // a masked row's places hold e = 0 with k0 = k1 = 0
          if (j < V && i0 + r < a.rows) g[j] = from_f<T>(d);
        }
      }
    }
  }
  if (a.partials) {
    __shared__ double part[kGroupThreads / 32][4];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      sums[k] = warp_sum(sums[k]);
      if (lane == 0) part[threadIdx.x >> 5][k] = sums[k];
    }
    __syncthreads();
    if (threadIdx.x < 4) {
      double x = 0;
      for (int q = 0; q < kGroupThreads / 32; ++q) x += part[q][threadIdx.x];
      a.partials[blockIdx.x * 4ll + threadIdx.x] = x * w;
    }
  }
}

// -------------------------------------------------------------------- longer rows
// A row is spread over a warp, a CTA or a cluster of CTAs, each thread holding NV vectors of
// 16 bytes of it in registers, so the row is read once and its gradient written from the
// same registers. Every thread sums against its own maximum; the sums are put on the row's
// maximum as they are combined.

// 16 bytes of T and their unpacking into pairs of floats
template <typename T> struct Vec;
template <> struct Vec<float> {
  static constexpr int N = 4;
  static __device__ __forceinline__ uint4 all(float x) {
    const uint32_t b = __float_as_uint(x);
    return make_uint4(b, b, b, b);
  }
  static __device__ __forceinline__ float2 pair(const uint4& q, int k) {
    return k == 0 ? make_float2(__uint_as_float(q.x), __uint_as_float(q.y))
                  : make_float2(__uint_as_float(q.z), __uint_as_float(q.w));
  }
  static __device__ __forceinline__ float most(const uint4& q, float m) {
    const float2 a = pair(q, 0), b = pair(q, 1);
    return max_nan(m, max_nan(max_nan(a.x, a.y), max_nan(b.x, b.y)));
  }
  static __device__ __forceinline__ void set(uint4& q, int k, float2 v) {
    if (k == 0) q.x = __float_as_uint(v.x), q.y = __float_as_uint(v.y);
    else q.z = __float_as_uint(v.x), q.w = __float_as_uint(v.y);
  }
};
__device__ __forceinline__ uint32_t word(const uint4& q, int k) {
  return k == 0 ? q.x : k == 1 ? q.y : k == 2 ? q.z : q.w;
}
__device__ __forceinline__ void set_word(uint4& q, int k, uint32_t v) {
  if (k == 0) q.x = v;
  else if (k == 1) q.y = v;
  else if (k == 2) q.z = v;
  else q.w = v;
}
template <> struct Vec<__nv_bfloat16> {
  static constexpr int N = 8;
  static __device__ __forceinline__ uint4 all(float x) {
    const __nv_bfloat162 h = __float2bfloat162_rn(x);
    const uint32_t b = *reinterpret_cast<const uint32_t*>(&h);
    return make_uint4(b, b, b, b);
  }
  static __device__ __forceinline__ float2 pair(const uint4& q, int k) {
    const uint32_t w = word(q, k);
    return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
  }
  static __device__ __forceinline__ float most(const uint4& q, float m) {
    auto h = [&](int k) {
      const uint32_t w = word(q, k);
      return *reinterpret_cast<const __nv_bfloat162*>(&w);
    };
    const __nv_bfloat162 x = __hmax2_nan(__hmax2_nan(h(0), h(1)), __hmax2_nan(h(2), h(3)));
    return max_nan(m, max_nan(__low2float(x), __high2float(x)));
  }
  static __device__ __forceinline__ void set(uint4& q, int k, float2 v) {
    const __nv_bfloat162 h = __float22bfloat162_rn(v);
    set_word(q, k, *reinterpret_cast<const uint32_t*>(&h));
  }
};
template <> struct Vec<__half> {
  static constexpr int N = 8;
  static __device__ __forceinline__ uint4 all(float x) {
    const __half2 h = __float2half2_rn(x);
    const uint32_t b = *reinterpret_cast<const uint32_t*>(&h);
    return make_uint4(b, b, b, b);
  }
  static __device__ __forceinline__ float2 pair(const uint4& q, int k) {
    const uint32_t w = word(q, k);
    return __half22float2(*reinterpret_cast<const __half2*>(&w));
  }
  static __device__ __forceinline__ float most(const uint4& q, float m) {
    auto h = [&](int k) {
      const uint32_t w = word(q, k);
      return *reinterpret_cast<const __half2*>(&w);
    };
    const __half2 x = __hmax2_nan(__hmax2_nan(h(0), h(1)), __hmax2_nan(h(2), h(3)));
    return max_nan(m, max_nan(__low2float(x), __high2float(x)));
  }
  static __device__ __forceinline__ void set(uint4& q, int k, float2 v) {
    const __half2 h = __float22half2_rn(v);
    set_word(q, k, *reinterpret_cast<const uint32_t*>(&h));
  }
};

// A part of a row: the maximum m of its logits, and its sums of 2^x2 and 2^x2 x2. Where m is
// ordinary, x2 is one fused operation, z log2 e - m2 with m2 = log2 e m rounded once: all x2 of
// the part are then (z - m) log2 e plus the same rest, log2 e m - m2, and sums on one m2 stay
// consistent to the last bit (p = 2^x2 / S). The rest is at most half an ulp of m2, so below
// 2^-6 while |m| < 1e5; beyond, it would grow until 2^rest leaves the range, and x2 is formed
// from z - m, without a rest. Masks that fill with a large finite number are of that kind.
struct Part {
  float m, s, t;
};
__device__ __forceinline__ bool ordinary(float m) { return fabsf(m) < 1e5f; }
__device__ __forceinline__ float origin(float m) { return m == -INFINITY ? 0.f : m; }
// m2, rounded as such (not contracted into what it is added to)
__device__ __forceinline__ float scaled(float m) { return __fmul_rn(m, kLog2e); }
// what x2 is too large by (exactly)
__device__ __forceinline__ float rest(float m) {
  return ordinary(m) ? __fmaf_rn(m, kLog2e, -scaled(m)) : 0.f;
}
// x2 of z, for a part that is not ordinary or that holds -inf (2^x2 x2 is to be 0 there)
__device__ __forceinline__ float careful(float z, float m) {
  const float x = ordinary(m) ? fmaf(z, kLog2e, -scaled(m)) : (z - origin(m)) * kLog2e;
  return max_nan(x, -1e4f);
}
// the same for an ordinary m, m2 = scaled(m)
__device__ __forceinline__ float bounded(float z, float m2) {
  return max_nan(fmaf(z, kLog2e, -m2), -1e4f);
}
// The log probability of logit z in a row with maximum m and log2 of its sum; however far below.
__device__ __forceinline__ float logp_of(float z, float m, float log2s) {
  if (m == -INFINITY) return z != z ? z : -INFINITY;  // nothing can be chosen
  return (z - m) - (log2s - rest(m)) * kLn2;
}
// p with its sums on the maximum `top`, in place of its own; a rest is exchanged with the
// maximum that it belongs to
__device__ __forceinline__ void onto(Part& p, float top) {
  float d = __fsub_rn(scaled(p.m), scaled(top));
  // far enough below an ordinary maximum (an empty part among them) nothing remains either way
  if (!(ordinary(top) && (ordinary(p.m) || p.m < -1e6f))) {
    asm volatile("");  // a branch, seldom taken, and no selection
    d = (p.m - origin(top)) * kLog2e + (rest(top) - rest(p.m));
  }
  d = max_nan(d, -1e4f);
  const float f = exp2_fast(d);
  p.t = fmaf(p.s, d, p.t) * f;
  p.s *= f;
  p.m = top;
}
// the parts of G adjacent lanes; `lanes` are the group's
template <int G> __device__ __forceinline__ Part join(Part p, unsigned lanes) {
  float top = p.m;
#pragma unroll
  for (int d = G / 2; d; d >>= 1) top = max_nan(top, __shfl_xor_sync(lanes, top, d));
  onto(p, top);
#pragma unroll
  for (int d = G / 2; d; d >>= 1) {
    p.s += __shfl_xor_sync(lanes, p.s, d);
    p.t += __shfl_xor_sync(lanes, p.t, d);
  }
  return p;
}

__device__ __forceinline__ uint4 load_once(const uint4* p) {
  uint4 q;
  asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];"
               : "=r"(q.x), "=r"(q.y), "=r"(q.z), "=r"(q.w)
               : "l"(p));
  return q;
}

__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
  asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ uint32_t shared_at(const void* p) {
  return static_cast<uint32_t>(__cvta_generic_to_shared(p));
}
__device__ __forceinline__ void mbar_init(uint64_t* b) {
  asm volatile("mbarrier.init.shared::cta.b64 [%0], 1;" ::"r"(shared_at(b)) : "memory");
}
__device__ __forceinline__ void mbar_expect(uint64_t* b, uint32_t bytes) {
  asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(shared_at(b)),
               "r"(bytes)
               : "memory");
}
// Whether the phase comes to its end within some 64 tries and then `clocks` clocks of the SM; a
// limit below zero gives it up without a look.
__device__ __forceinline__ bool mbar_wait(uint64_t* b, uint32_t parity, long long clocks) {
  const uint32_t at = shared_at(b);
  auto ended = [&] {
    uint32_t done;
    asm volatile(
        "{ .reg .pred p;\n"
        "mbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2;\n"
        "selp.u32 %0, 1, 0, p; }"
        : "=r"(done)
        : "r"(at), "r"(parity)
        : "memory");
    return done != 0;
  };
  if (clocks < 0) return false;
  if (ended()) return true;
  const long long from = clock64();
  for (int k = 0; k < 64 || clock64() - from < clocks; ++k)
    if (ended()) return true;
  return false;
}
// p to the same place in the shared memory of CTA `to` of the cluster, counted by its barrier
__device__ __forceinline__ void send(float4* place, uint64_t* bar, int to, Part p) {
  uint32_t d, b;
  asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(d) : "r"(shared_at(place)), "r"(to));
  asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(b) : "r"(shared_at(bar)), "r"(to));
  asm volatile(
      "st.async.weak.shared::cluster.mbarrier::complete_tx::bytes.v4.f32 [%0], {%1, %2, %3, "
      "%4}, [%5];" ::"r"(d),
      "f"(p.m), "f"(p.s), "f"(p.t), "f"(0.f), "r"(b)
      : "memory");
}

// sets a flag at the same place in the shared memory of the cluster's first CTA
__device__ __forceinline__ void tell_first(int* flag) {
  uint32_t d;
  asm("mapa.shared::cluster.u32 %0, %1, 0;" : "=r"(d) : "r"(shared_at(flag)));
  asm volatile("st.shared::cluster.u32 [%0], 1;" ::"r"(d) : "memory");
}

// A row as a thread of its group sees it: whole vectors, and up to N - 1 elements before them
// and after them, one of each with the threads from the first on.
template <typename T> struct Cut {
  const uint4* vec;
  int vecs, head, before, behind;  // places of the thread's single elements, -1 = none
  __device__ __forceinline__ Cut(const T* z, int V, int at) {
    head = min(V, static_cast<int>((16 - (reinterpret_cast<uintptr_t>(z) & 15)) & 15) /
                      static_cast<int>(sizeof(T)));
    vecs = (V - head) / Vec<T>::N;
    vec = reinterpret_cast<const uint4*>(z + head);
    const int tail = head + vecs * Vec<T>::N;
    before = at < head ? at : -1;
    behind = at < V - tail ? tail + at : -1;
  }
};

constexpr int split_block(int threads) { return threads <= 32 ? 256 : threads; }
// Vectors that a thread holds: half of its registers, and as much of a row as makes up for
// the row's sums and scalars, which every warp does for itself (8192 rows of 131072 bf16: 16
// vectors 981 us, 8 with half as many threads again 1176 us).
constexpr int NV = 16;
// CTAs per SM that the registers have to allow: 16 warps of 128
constexpr int split_resident(int threads) { return 512 / split_block(threads); }

// THREADS of 8 to 32: a row per group of so many lanes, C = 1. Otherwise one row per cluster of
// C CTAs of THREADS. Few lanes with many vectors each do a row's scalar part for several rows
// at once. The CTAs are resident ones that walk the rows. With a gradient, a vector's
// registers take the next row's vector as soon as its gradient is out, so the next row is on
// its way while this one is written. The parts of a row go to all CTAs of the cluster by
// asynchronous stores that a barrier in the receiver's shared memory counts: a cluster
// barrier would first wait for the gradient's stores. Each wait for parts has a limit. A warp that
// comes to it sends no more, so all others come to theirs at the next row at the latest; what
// they write from then on is NaN, and so is the loss.
// 8192 rows of 131072 bf16 take 0.98 ms, 68% of the copy rate, 4096 of 32768 124 us, 67%;
// about 18 instructions and two exponentials an element, which fill 55% of the issue slots and
// 45% of the exponential unit, with 16 warps an SM to hide the rest.
template <typename T, int THREADS, int C, bool GRAD>
__global__ void __launch_bounds__(split_block(THREADS), split_resident(THREADS))
    policy_split_kernel(Args a) {
  constexpr bool kLanes = THREADS <= 32;
  constexpr int G = kLanes ? THREADS : 32;  // lanes that join by shuffles
  constexpr int kWarps = kLanes ? 1 : THREADS / 32;
  constexpr int N = Vec<T>::N;
  constexpr int kAllThreads = THREADS * C;
  constexpr int kParts = C * kWarps;
  __shared__ float4 parts[2][kLanes ? 1 : kParts];
  __shared__ uint64_t bars[2];
  __shared__ int any_lost;  // the first CTA's is used
  const float cot = a.cotangent ? *a.cotangent : 1.f;
  if (a.skip_unit && cot == 1.f) return;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int rank = C > 1 ? static_cast<int>(blockIdx.x % C) : 0;  // clusters are runs of C CTAs
  const int at = kLanes ? lane & (G - 1) : rank * THREADS + static_cast<int>(threadIdx.x);
  const unsigned lanes = G == 32 ? kAll : ((1u << G) - 1) << (lane & ~(G - 1));
  const int V = static_cast<int>(a.vocab);
  if (C > 1) {
    if (threadIdx.x == 0) {
      mbar_init(&bars[0]), mbar_init(&bars[1]);
      any_lost = 0;
      asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    cluster_sync();
  }
  const float w = row_weight(a), wg = w * a.grad_scale * cot;
  constexpr int kRowsPerCta = 256 / THREADS;  // kLanes
  const long long first = kLanes ? blockIdx.x * static_cast<long long>(kRowsPerCta) +
                                       threadIdx.x / THREADS
                                 : blockIdx.x / C;
  const long long step = kLanes ? gridDim.x * static_cast<long long>(kRowsPerCta) : gridDim.x / C;
  double sums[4] = {0, 0, 0, 0};
  int turn = 0;
  int lost = -1;  // the turn in which a part did not come to this warp: all that follows is NaN

  // the first row from i on that the mask admits; those before it get their zeros
  auto admitted = [&](long long i) {
    for (; i < a.rows && a.mask && !a.mask[i]; i += step) {
      if (GRAD) {
        T* g = static_cast<T*>(a.grad) + i * V;
        const Cut<T> cut(g, V, at);
        uint4* gv = reinterpret_cast<uint4*>(g + cut.head);
        for (int k = at; k < cut.vecs; k += kAllThreads) gv[k] = make_uint4(0, 0, 0, 0);
        if (cut.before >= 0) g[cut.before] = from_f<T>(0.f);
        if (cut.behind >= 0) g[cut.behind] = from_f<T>(0.f);
      }
      if (at == 0 && a.logp) a.logp[i] = 0.f, a.entropy[i] = 0.f;
    }
    return i;
  };
  auto start_of = [&](long long i) { return static_cast<const T*>(a.logits) + row_offset(a, i); };
  auto at_token = [&](const T* z, long long tok) {
    return tok >= 0 && tok < V ? to_f(z[tok]) : NAN;
  };
  // How many vectors a warp works on in any row, the same for all its lanes. Of the last, lanes
  // may be beyond their row's end (nowhere else: a row has V / N vectors, or one less). In a
  // group of lanes each counts its own.
  const int asks = kLanes ? 0 : __shfl_sync(kAll, at, 0);
  const int of_warp = V / N > asks ? (V / N - asks + kAllThreads - 1) / kAllThreads : 0;
  auto fetch = [&](const Cut<T>& cut, int k, uint4& q) {
    const int j = k * kAllThreads + at;
    if (j < cut.vecs) q = load_once(cut.vec + j);
  };

  long long i = admitted(first);
  if (i < a.rows) {
    uint4 q[NV];
    const T* z = start_of(i);
    Cut<T> cut(z, V, at);
#pragma unroll
    for (int k = 0; k < NV; ++k) fetch(cut, k, q[k]);
    auto single = [&](const T* z, int place) { return place >= 0 ? to_f(z[place]) : -INFINITY; };
    float z0 = single(z, cut.before), z1 = single(z, cut.behind);
    long long tok = token_of(a, i);
    Inputs in = inputs_of(a, i);
    float za = at_token(z, tok);
    bool low = false;  // the thread has met a logit of -inf: its products need care
    while (true) {
      const int count = !kLanes            ? of_warp
                        : cut.vecs > at ? (cut.vecs - at + kAllThreads - 1) / kAllThreads
                                        : 0;
      Part p{max_nan(z0, z1), 0.f, 0.f};
#pragma unroll
      for (int k = 0; k < NV; ++k)
        if (kLanes ? k < count
                   : k < count - 1 || (k == count - 1 && k * kAllThreads + at < cut.vecs))
          p.m = Vec<T>::most(q[k], p.m);
      // lanes beyond the row's end take a logit that adds nothing to the sums, and no NaN
      if (!kLanes && (count - 1) * kAllThreads + at >= cut.vecs) {
#pragma unroll
        for (int k = 0; k < NV; ++k)
          if (k == count - 1) q[k] = Vec<T>::all(p.m - 200.f - 0.25f * fabsf(p.m));
      }
      {
        const float m = p.m, m2 = scaled(m);
        // care 0: none; 1: x2 bounded below; 2: m out of the ordinary
        auto sum = [&](auto care) {
          constexpr int kCare = decltype(care)::value;
          float s[2] = {0.f, 0.f}, t[2] = {0.f, 0.f};
#pragma unroll
          for (int k = 0; k < NV; ++k)
            if (k < count) {
#pragma unroll
              for (int h = 0; h < N / 2; ++h) {
                float2 x = Vec<T>::pair(q[k], h);
                if (kCare == 2) x.x = careful(x.x, m), x.y = careful(x.y, m);
                else if (kCare == 1) x.x = bounded(x.x, m2), x.y = bounded(x.y, m2);
                else x.x = fmaf(x.x, kLog2e, -m2), x.y = fmaf(x.y, kLog2e, -m2);
                const float e0 = exp2_fast(x.x), e1 = exp2_fast(x.y);
                s[0] += e0, s[1] += e1;
                t[0] = fmaf(e0, x.x, t[0]), t[1] = fmaf(e1, x.y, t[1]);
              }
            }
          const float x0 = careful(z0, m), e0 = exp2_fast(x0);
          const float x1 = careful(z1, m), e1 = exp2_fast(x1);
          p.s = s[0] + s[1] + (e0 + e1);
          p.t = fmaf(e0, x0, t[0]) + fmaf(e1, x1, t[1]);
        };
        if (!ordinary(m)) low = true, sum(std::integral_constant<int, 2>{});
        else if (!low) sum(std::integral_constant<int, 0>{});
        // 0 times -inf: again with x2 bounded, and so from now on
        if (ordinary(m) && (low || p.t != p.t)) low = true, sum(std::integral_constant<int, 1>{});
      }
      // the next row, and what can be asked of it already
      const long long i2 = admitted(i + step);
      const bool more = i2 < a.rows;
      const T* z2 = more ? start_of(i2) : z;
      const Cut<T> cut2(z2, more ? V : 0, at);
      const long long tok2 = more ? token_of(a, i2) : -1;
      const Inputs in2 = more ? inputs_of(a, i2) : in;
      if (!GRAD) {
#pragma unroll
        for (int k = 0; k < NV; ++k) fetch(cut2, k, q[k]);
      }
      p = join<G>(p, lanes);
      if (!kLanes) {
        float4* box = parts[turn & 1];
        if (C == 1) {
          if (lane == 0) box[warp] = make_float4(p.m, p.s, p.t, 0.f);
          __syncthreads();
        } else if (lost < 0) {
          uint64_t* bar = &bars[turn & 1];
          if (threadIdx.x == 0) mbar_expect(bar, kParts * sizeof(float4));
          if (lane < C) send(&box[rank * kWarps + warp], bar, lane, p);
          if (!__all_sync(kAll, mbar_wait(bar, (turn >> 1) & 1, a.wait_clocks))) lost = turn;
        }
        constexpr int kEach = (kParts + 31) / 32;
        Part mine[kEach];
        float top = lost < 0 ? -INFINITY : NAN;
#pragma unroll
        for (int k = 0; k < kEach; ++k) {
          const int j = lane + 32 * k;
          mine[k] = Part{-INFINITY, 0.f, 0.f};
          if (j < kParts) {
            const float4 f = box[j];
            mine[k] = Part{f.x, f.y, f.z};
          }
          top = max_nan(top, mine[k].m);
        }
        top = warp_max(top);
        p = Part{top, 0.f, 0.f};
#pragma unroll
        for (int k = 0; k < kEach; ++k) {
          onto(mine[k], top);
          p.s += mine[k].s;
          p.t += mine[k].t;
        }
        p.s = warp_sum(p.s);
        p.t = warp_sum(p.t);
        // The next row's parts go to the other box. The one after that comes to this box only
        // when its sender holds all of the next row's parts, and every warp sends its own of
        // those after it has read this box.
        ++turn;
      }
      const bool empty = p.m == -INFINITY;
      const float m = p.m, log2s = empty ? 0.f : __log2f(p.s);
      const float inv = empty ? 0.f : __fdividef(1.f, p.s);
      const Row r = row_terms(a, in, logp_of(za, m, log2s), (log2s - p.t * inv) * kLn2,
                              empty && za == za);
      if (at == 0) {
        if (a.logp) a.logp[i] = r.lp, a.entropy[i] = r.H;
        sums[0] += r.pg, sums[1] += r.k3, sums[2] += r.H, sums[3] += r.cut;
      }
      if (GRAD) {
        const float c = wg * r.c, eta = wg * a.ent;
        const float k0 = inv * (eta * (r.H - log2s * kLn2) - c), k1 = inv * eta * kLn2;
        const float m2 = scaled(m);
        T* g = static_cast<T*>(a.grad) + i * V;
        uint4* gv = reinterpret_cast<uint4*>(g + cut.head);
        const bool same_phase = (reinterpret_cast<uintptr_t>(gv) & 15) == 0;
        // kind 0: no entropy term; 1: with it; 2: with it, x2 bounded; 3: m out of the ordinary
        auto write = [&](auto kind) {
          constexpr int kKind = decltype(kind)::value;
#pragma unroll
          for (int k = 0; k < NV; ++k) {
            if (k < count) {
              const int j = k * kAllThreads + at;
              uint4 out;
#pragma unroll
              for (int h = 0; h < N / 2; ++h) {
                float2 x = Vec<T>::pair(q[k], h);
                if (kKind == 3) x.x = careful(x.x, m), x.y = careful(x.y, m);
                else if (kKind == 2) x.x = bounded(x.x, m2), x.y = bounded(x.y, m2);
                else x.x = fmaf(x.x, kLog2e, -m2), x.y = fmaf(x.y, kLog2e, -m2);
                const float e0 = exp2_fast(x.x), e1 = exp2_fast(x.y);
                Vec<T>::set(out, h, kKind == 0 ? make_float2(e0 * k0, e1 * k0)
                                               : make_float2(e0 * fmaf(k1, x.x, k0),
                                                             e1 * fmaf(k1, x.y, k0)));
              }
              if (kLanes || j < cut.vecs) {
                if (same_phase) {
                  gv[j] = out;
                } else {
                  const T* o8 = reinterpret_cast<const T*>(&out);
#pragma unroll
                  for (int h = 0; h < N; ++h) g[cut.head + j * N + h] = o8[h];
                }
              }
            }
            fetch(cut2, k, q[k]);
          }
        };
        // without the entropy term a logit of -inf needs no care; with it, a finite one far
        // below must not leave the range when it is multiplied by k1
        if (!ordinary(m)) write(std::integral_constant<int, 3>{});
        else if (a.ent == 0.f) write(std::integral_constant<int, 0>{});
        else if (!low && fabsf(k1) < 0.5f) write(std::integral_constant<int, 1>{});
        else write(std::integral_constant<int, 2>{});
        auto alone = [&](float zj) {
          const float x = careful(zj, m);
          return exp2_fast(x) * fmaf(k1, x, k0);
        };
        if (cut.before >= 0) g[cut.before] = from_f<T>(alone(z0));
        if (cut.behind >= 0) g[cut.behind] = from_f<T>(alone(z1));
        // the token's own place again, by the thread that has just written it
        if (tok >= 0 && tok < V) {
          const int j = static_cast<int>(tok) - cut.head;
          const int tk = static_cast<int>(tok);
          const bool mine = j >= 0 && j < cut.vecs * N ? j / N % kAllThreads == at
                                                       : cut.before == tk || cut.behind == tk;
          if (mine) g[tok] = from_f<T>(alone(za) + c);
        }
      }
      if (!more) break;
      i = i2, z = z2, cut = cut2, tok = tok2, in = in2;
      z0 = single(z, cut.before), z1 = single(z, cut.behind);
      za = at_token(z, tok);
    }
  }
  if (C > 1) {
    if (lost >= 0 && lane == 0) tell_first(&any_lost);
    __syncwarp();
    // Every warp comes here, since its waits end. After it nobody sends; parts that were waited
    // for have come, and those that a warp gave up are given their time again, so that nobody
    // leaves while a part may still be on its way to it.
    cluster_sync();
    if (lost >= 0) mbar_wait(&bars[lost & 1], (lost >> 1) & 1, kWaitClocks);
    if (at == 0 && any_lost) sums[0] = NAN;
  }
  if (!a.partials) return;
  if (kLanes) {
    __shared__ double part[8][4];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const double x = warp_sum(sums[k]);  // of the groups' first lanes
      if (lane == 0) part[warp][k] = x;
    }
    __syncthreads();
    if (threadIdx.x < 4) {
      double x = 0;
      for (int k = 0; k < 8; ++k) x += part[k][threadIdx.x];
      a.partials[blockIdx.x * 4ll + threadIdx.x] = x * w;
    }
  } else if (at == 0) {
    for (int k = 0; k < 4; ++k) a.partials[first * 4 + k] = sums[k] * w;
  }
}

// ------------------------------------------------------- short rows, one after the other
// Many short rows that lie together: a CTA brings 128 of them into shared memory in whole
// vectors, a thread takes one row from there, and the gradients go back the same way. No lane
// waits for another's sums, and nothing is computed twice. E - 4 < V <= E. ROT: rows of an
// even number of words would put many threads on one bank; they then start at different
// places of their rows. 512,000 rows of 21 floats take 23 us, 70% of the copy rate (28
// with a mask): 40 instructions an element fill 71% of the issue slots, and a CTA that waits for
// its copies, one tile at a time, has nothing else to do (six CTAs an SM).
constexpr int kTileRows = 128;

template <typename T, int E, bool ROT, bool GRAD>
__global__ void __launch_bounds__(kTileRows, 6) policy_tile_kernel(Args a) {
  constexpr int N = 16 / sizeof(T), kCopies = (E + N - 1) / N;
  __shared__ __align__(16) T tile[kTileRows * E];
  __shared__ double part[kTileRows / 32][4];
  const float cot = a.cotangent ? *a.cotangent : 1.f;
  if (a.skip_unit && cot == 1.f) return;
  const int V = static_cast<int>(a.vocab), tid = threadIdx.x;
  const int turn = ROT ? (sizeof(T) == 4 ? tid : 2 * tid) % V : 0;
  T* mine = tile + tid * V;
  auto place = [&](int k) -> T& {
    int j = k;
    if (ROT) j += turn, j = j >= V ? j - V : j;
    return mine[j];
  };
  float w = 0.f, wg = 0.f;
  float sums[4] = {0.f, 0.f, 0.f, 0.f};
  for (long long base = static_cast<long long>(blockIdx.x) * kTileRows; base < a.rows;
       base += static_cast<long long>(gridDim.x) * kTileRows) {
    const int n = static_cast<int>(min(a.rows - base, static_cast<long long>(kTileRows)));
    const int cells = n * V, vecs = cells / N;
    const long long i = base + tid;
    {
      const T* z = static_cast<const T*>(a.logits) + base * V;
      const uint4* from = reinterpret_cast<const uint4*>(z);
#pragma unroll
      for (int k = 0; k < kCopies; ++k)
        if (k * kTileRows + tid < vecs)
          asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(
                           shared_at(reinterpret_cast<uint4*>(tile) + k * kTileRows + tid)),
                       "l"(from + k * kTileRows + tid)
                       : "memory");
      if (vecs * N + tid < cells) tile[vecs * N + tid] = z[vecs * N + tid];
    }
    const bool in = tid < n, live = in && (!a.mask || a.mask[i]);
    const long long tok = live ? token_of(a, i) : 0;
    const Inputs in0 = live ? inputs_of(a, i) : Inputs{0.f, 0.f, 0.f};
    if (w == 0.f) w = row_weight(a), wg = w * a.grad_scale * cot;
    asm volatile("cp.async.wait_all;" ::: "memory");
    __syncthreads();
    if (live) {
      float x[E];
      float m = -INFINITY;
#pragma unroll
      for (int k = 0; k < E; ++k) {
        x[k] = k < E - 3 || k < V ? to_f(place(k)) : -INFINITY;
        m = max_nan(m, x[k]);
      }
      const bool there = tok >= 0 && tok < V;
      const float za = there ? to_f(mine[static_cast<int>(tok)]) : NAN;
      const bool empty = m == -INFINITY;
      // x becomes 2^x2, the term of the sum
      float s = 0.f, t = 0.f;
      const float m2 = -scaled(m);
      const bool plain = ordinary(m);
      auto x2_of = [&](float z) {
        return plain ? max_nan(fmaf(z, kLog2e, m2), -1e4f) : careful(z, m);
      };
#pragma unroll
      for (int k = 0; k < E; ++k) {
        const float y = x2_of(x[k]);
        x[k] = exp2_fast(y);
        s += x[k];
        t = fmaf(x[k], y, t);
      }
      const float log2s = empty ? 0.f : __log2f(s), inv = empty ? 0.f : __fdividef(1.f, s);
      const Row r = row_terms(a, in0, logp_of(za, m, log2s), (log2s - t * inv) * kLn2,
                              empty && za == za);
      sums[0] += r.pg, sums[1] += r.k3, sums[2] += r.H, sums[3] += r.cut;
      if (a.logp) a.logp[i] = r.lp, a.entropy[i] = r.H;
      if (GRAD) {
        const float c = wg * r.c, eta = wg * a.ent;
        const float k0 = inv * (eta * (r.H - log2s * kLn2) - c), k1 = inv * eta * kLn2;
        float token_grad = 0.f;
        if (there) {
          const float y = careful(za, m);
          token_grad = exp2_fast(y) * fmaf(k1, y, k0) + c;
        }
        if (a.ent == 0.f) {
#pragma unroll
          for (int k = 0; k < E; ++k)
            if (k < E - 3 || k < V) place(k) = from_f<T>(x[k] * k0);
        } else {
#pragma unroll
          for (int k = 0; k < E; ++k)
            if (k < E - 3 || k < V) {
              T& at = place(k);
              at = from_f<T>(x[k] * fmaf(k1, x2_of(to_f(at)), k0));
            }
        }
        if (there) mine[static_cast<int>(tok)] = from_f<T>(token_grad);
      }
    } else if (in) {
      if (a.logp) a.logp[i] = 0.f, a.entropy[i] = 0.f;
      if (GRAD)
        for (int k = 0; k < V; ++k) mine[k] = from_f<T>(0.f);
    }
    __syncthreads();
    if (GRAD) {
      T* g = static_cast<T*>(a.grad) + base * V;
#pragma unroll
      for (int k = 0; k < kCopies; ++k)
        if (k * kTileRows + tid < vecs)
          reinterpret_cast<uint4*>(g)[k * kTileRows + tid] =
              reinterpret_cast<const uint4*>(tile)[k * kTileRows + tid];
      if (vecs * N + tid < cells) g[vecs * N + tid] = tile[vecs * N + tid];
      __syncthreads();
    }
  }
  if (!a.partials) return;
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const double q = warp_sum(static_cast<double>(sums[k]));
    if ((tid & 31) == 0) part[tid >> 5][k] = q;
  }
  __syncthreads();
  if (tid < 4) {
    double q = 0;
    for (int k = 0; k < kTileRows / 32; ++k) q += part[k][tid];
    a.partials[blockIdx.x * 4ll + tid] = q * w;
  }
}

// ------------------------------------------------------------- any row, any length
// One CTA per row at a time, the row read three times (maximum, sums, gradient), the later
// reads from L1 or L2, element by element. 2048 rows of 151936 floats take 1.9 ms, 20% of the
// copy rate (one read and one write), bound by the loads' latency.
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
    const Row r = row_terms(a, inputs_of(a, i),
                            empty ? (za != za ? za : -INFINITY) : (za - m) - ln,
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
constexpr int kScalarThreads = 512;

__global__ void __launch_bounds__(kScalarThreads)
    scalars_kernel(const double* partials, long long n, float kl, float ent, float* loss,
                   float* stats) {
  __shared__ double part[kScalarThreads / 32][4];
  double s[4] = {0, 0, 0, 0};
#pragma unroll 4
  for (long long i = threadIdx.x; i < n; i += kScalarThreads) {
    const double2 x = reinterpret_cast<const double2*>(partials)[2 * i];
    const double2 y = reinterpret_cast<const double2*>(partials)[2 * i + 1];
    s[0] += x.x, s[1] += x.y, s[2] += y.x, s[3] += y.y;
  }
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    s[k] = warp_sum(s[k]);
    if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5][k] = s[k];
  }
  __syncthreads();
  if (threadIdx.x >= 32) return;
  for (int k = 0; k < 4; ++k)
    s[k] = warp_sum(threadIdx.x < kScalarThreads / 32 ? part[threadIdx.x][k] : 0.0);
  if (threadIdx.x == 0) {
    double l = s[0];  // a coefficient of 0 takes its term out, whatever its value
    if (kl != 0.f) l += static_cast<double>(kl) * s[1];
    if (ent != 0.f) l -= static_cast<double>(ent) * s[2];
    *loss = static_cast<float>(l);
    for (int k = 0; k < 4; ++k) stats[k] = static_cast<float>(s[k]);
  }
}

// -------------------------------------------------------------------------- the host
// How a batch is run, by its vocabulary and type alone: short rows by groups of lanes,
// longer ones by a warp, a CTA or a cluster each, whatever is longer by the loop.
enum Kind { kTile, kGroup, kLaneRows, kSplit, kLoop };
struct Plan {
  Kind kind;
  int lanes, per_lane, rows_each;  // kGroup: L, E, R; kTile: per_lane = E
  int threads, cluster;            // kLaneRows, kSplit
  long long blocks, n_partials;
  size_t partials_at, bytes;
};

// Above, a group of 8 lanes with whole vectors is faster than 32 lanes with single elements:
// 100000 rows of 200 bf16 52 us against 105, of 257 f32 60 against 69; 200000 rows of 100 bf16
// 94 against 69, of 128 f32 77 against 46.
constexpr int kShort = 128;
constexpr int kTileMaxBlocks = 148 * 32;
// Faster than groups of lanes at any number of rows: 512 rows of 25 floats 3.2 us against 4.3,
// 65536 of 21 4.6 against 5.3, 512000 of 21 22.7 against 28.9 (no mask).
constexpr int kTileVocab = 32;

int check(const swarp_policy_t* p) {
  if (!p || p->rows < 0 || p->vocab < 1 || p->vocab > 0x7fffffffll) return SWARP_ERR_INVALID_ARG;
  if (p->dtype != SWARP_F32 && p->dtype != SWARP_BF16 && p->dtype != SWARP_F16)
    return SWARP_ERR_INVALID_ARG;
  if (p->rows > 0 && (p->inner < 1 || p->rows % p->inner != 0)) return SWARP_ERR_INVALID_ARG;
  return SWARP_OK;
}
Plan plan_of(const swarp_policy_t* p) {
  Plan q{};
  const long long V = p->vocab, rows = p->rows;
  const long long vecs = V / (p->dtype == SWARP_F32 ? 4 : 8);
  auto at_most = [&](long long n, long long cap) { return n < 1 ? 1 : n < cap ? n : cap; };
  const bool adjacent = p->inner == rows && p->stride_inner == V &&
                        reinterpret_cast<uintptr_t>(p->logits) % 16 == 0 &&
                        reinterpret_cast<uintptr_t>(p->grad) % 16 == 0;
  if (V <= kTileVocab && adjacent) {
    q.kind = kTile;
    q.per_lane = static_cast<int>((V + 3) / 4 * 4);
    q.blocks = q.n_partials = at_most((rows + kTileRows - 1) / kTileRows, kTileMaxBlocks);
  } else if (V <= kShort) {
    q.kind = kGroup;
    q.lanes = V <= 4 ? 1 : V <= 8 ? 2 : V <= 16 ? 4 : V <= 32 ? 8 : V <= 64 ? 16 : 32;
    q.per_lane = static_cast<int>((V + q.lanes - 1) / q.lanes);
    q.per_lane = q.per_lane <= 3 ? 3 : 4;
    if (q.lanes < 8) q.per_lane = 4;
    q.rows_each = q.lanes <= 8 ? q.lanes : 8;
    const long long rows_per_block = kGroupThreads / q.lanes * q.rows_each;
    q.blocks = at_most((rows + rows_per_block - 1) / rows_per_block, 148 * 8);
    q.n_partials = q.blocks;
  } else if (vecs <= 32 * NV) {
    q.kind = kLaneRows;
    q.threads = vecs <= 8 * NV ? 8 : vecs <= 16 * NV ? 16 : 32;
    q.cluster = 1;
    const int per = 256 / q.threads;
    q.blocks = at_most((rows + per - 1) / per, 148 * split_resident(q.threads));
    q.n_partials = q.blocks;
  } else if (vecs <= 8ll * 256 * NV) {
    // no more threads than the row fills: a CTA's rows come one after the other, and smaller
    // CTAs are more rows at once (16384 rows of 4200 bf16: 64 threads 87 us, 128 133 us)
    q.kind = kSplit;
    q.threads = vecs <= 64 * NV ? 64 : vecs <= 128 * NV ? 128 : 256;
    q.cluster = 1;
    while (vecs > static_cast<long long>(q.cluster) * q.threads * NV) q.cluster *= 2;
    // clusters; a launch may have fewer, as many as the device holds at once
    q.n_partials = at_most(rows, 148ll * split_resident(q.threads) / q.cluster);
    q.blocks = q.n_partials * q.cluster;
  } else {
    q.kind = kLoop;
    q.blocks = q.n_partials = at_most(rows, kLoopMaxBlocks);
  }
  q.partials_at = align256(kCountBlocks * sizeof(long long));
  // the same for every kind, so that it does not depend on the addresses
  q.bytes = q.partials_at + align256(sizeof(double) * 4 * at_most(rows, kTileMaxBlocks));
  return q;
}

template <typename T, int L, int E, int R> int launch_group(const Args& a, const Plan& q,
                                                            cudaStream_t st) {
  const unsigned n = static_cast<unsigned>(q.blocks);
  if (a.grad) policy_group_kernel<T, L, E, R, true><<<n, kGroupThreads, 0, st>>>(a);
  else policy_group_kernel<T, L, E, R, false><<<n, kGroupThreads, 0, st>>>(a);
  return launch_status();
}

template <typename T, int E> int launch_tile(const Args& a, const Plan& q, cudaStream_t st) {
  const unsigned n = static_cast<unsigned>(q.blocks);
  const bool rot = a.vocab % (sizeof(T) == 4 ? 2 : 4) == 0;
  auto* f = a.grad ? (rot ? policy_tile_kernel<T, E, true, true> : policy_tile_kernel<T, E, false, true>)
                   : (rot ? policy_tile_kernel<T, E, true, false> : policy_tile_kernel<T, E, false, false>);
  f<<<n, kTileRows, 0, st>>>(a);
  return launch_status();
}

template <typename T, int THREADS, int C> int launch_split(const Args& a, Plan& q,
                                                                   cudaStream_t st) {
  auto* f = a.grad ? policy_split_kernel<T, THREADS, C, true>
                   : policy_split_kernel<T, THREADS, C, false>;
  cudaLaunchConfig_t cfg{};
  cfg.blockDim = dim3(split_block(THREADS));
  cfg.stream = st;
  cudaLaunchAttribute attr{};
  attr.id = cudaLaunchAttributeClusterDimension;
  attr.val.clusterDim.x = C;
  attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = C > 1 ? 1 : 0;
  cfg.gridDim = dim3(static_cast<unsigned>(q.blocks));
  if (C > 1) {
    // clusters that wait for others to end would double the time: rows are dealt out evenly
    static std::atomic<int> resident[2];
    int n = resident[a.grad != nullptr].load(std::memory_order_relaxed);
    if (n == 0) {
      if (cudaOccupancyMaxActiveClusters(&n, f, &cfg) != cudaSuccess || n < 1)
        return SWARP_ERR_CUDA;
      resident[a.grad != nullptr].store(n, std::memory_order_relaxed);
    }
    if (q.n_partials > n) {
      q.n_partials = n;
      cfg.gridDim.x = static_cast<unsigned>(n * C);
    }
  }
  return cudaLaunchKernelEx(&cfg, f, a) == cudaSuccess ? launch_status() : SWARP_ERR_CUDA;
}

template <typename T> int run_typed(const Args& a, Plan& q, cudaStream_t st) {
  if (q.kind == kTile) {
    switch (q.per_lane) {
      case 4: return launch_tile<T, 4>(a, q, st);
      case 8: return launch_tile<T, 8>(a, q, st);
      case 12: return launch_tile<T, 12>(a, q, st);
      case 16: return launch_tile<T, 16>(a, q, st);
      case 20: return launch_tile<T, 20>(a, q, st);
      case 24: return launch_tile<T, 24>(a, q, st);
      case 28: return launch_tile<T, 28>(a, q, st);
      default: return launch_tile<T, 32>(a, q, st);
    }
  }
  if (q.kind == kGroup) {
    switch (q.lanes) {
      case 1: return launch_group<T, 1, 4, 1>(a, q, st);
      case 2: return launch_group<T, 2, 4, 2>(a, q, st);
      case 4: return launch_group<T, 4, 4, 4>(a, q, st);
      case 8:
        return q.per_lane == 3 ? launch_group<T, 8, 3, 8>(a, q, st)
                               : launch_group<T, 8, 4, 8>(a, q, st);
      case 16:
        return q.per_lane == 3 ? launch_group<T, 16, 3, 8>(a, q, st)
                               : launch_group<T, 16, 4, 8>(a, q, st);
      default:
        return q.per_lane == 3 ? launch_group<T, 32, 3, 8>(a, q, st)
                               : launch_group<T, 32, 4, 8>(a, q, st);
    }
  }
  if (q.kind == kLaneRows)
    return q.threads == 8    ? launch_split<T, 8, 1>(a, q, st)
           : q.threads == 16 ? launch_split<T, 16, 1>(a, q, st)
                             : launch_split<T, 32, 1>(a, q, st);
  if (q.kind == kSplit)
    return q.threads == 64    ? launch_split<T, 64, 1>(a, q, st)
           : q.threads == 128 ? launch_split<T, 128, 1>(a, q, st)
           : q.cluster == 1   ? launch_split<T, 256, 1>(a, q, st)
           : q.cluster == 2   ? launch_split<T, 256, 2>(a, q, st)
           : q.cluster == 4   ? launch_split<T, 256, 4>(a, q, st)
                              : launch_split<T, 256, 8>(a, q, st);
  const unsigned n = static_cast<unsigned>(q.blocks);
  if (a.grad) policy_loop_kernel<T, true><<<n, kLoopThreads, 0, st>>>(a);
  else policy_loop_kernel<T, false><<<n, kLoopThreads, 0, st>>>(a);
  return launch_status();
}

// SWARP_POLICY_WAIT_CLOCKS (read on every call that has clusters) replaces the limit of their
// waits; -1 lets each run out at once, for tests.
long long wait_clocks() {
  const char* s = std::getenv("SWARP_POLICY_WAIT_CLOCKS");
  return s && *s ? std::atoll(s) : kWaitClocks;
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
  Plan q = plan_of(p);
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
  if (q.cluster > 1) a.wait_clocks = wait_clocks();
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
    scalars_kernel<<<1, kScalarThreads, 0, st>>>(a.partials, some ? q.n_partials : 0, a.kl, a.ent, p->loss,
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
