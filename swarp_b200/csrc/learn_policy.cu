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

// ------------------------------------------------------------------- short rows
// A group of L lanes takes R rows at a time, lane l of it the elements l, l + L, ... of each
// (E of them, in registers). The R sums over the L lanes are reduced by halving: in each of
// the first log2 R steps a lane hands half of its sums to its partner and keeps the other
// half, so R sums cost R - 1 + log2(L / R) shuffles instead of R log2 L, and leave row
// l / (L / R) with lane l. That lane then does the scalar part of its row, which would
// otherwise cost every lane more than the row's own elements.
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
    if (live) {
      tok = token_of(a, i);
      za = NAN;
      if (tok >= 0 && tok < V) za = to_f((static_cast<const T*>(a.logits) + row_offset(a, i))[tok]);
    }
    float z[R][E];
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const T* p = static_cast<const T*>(a.logits) + row_offset(a, i0 + r);
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
    const float ln = empty ? 0.f : logf(s), inv = empty ? 0.f : 1.f / s;
    const Row row = row_terms(a, i, empty ? (za != za ? za : -INFINITY) : (za - m) - ln,
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
  static constexpr uint32_t kNegInf = 0xff800000u;
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
  static constexpr uint32_t kNegInf = 0xff80ff80u;
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
  static constexpr uint32_t kNegInf = 0xfc00fc00u;
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

// two floats as one operand of the packed instructions
struct F2 {
  unsigned long long v;
  __device__ __forceinline__ F2(float2 f) {
    asm("mov.b64 %0, {%1, %2};" : "=l"(v) : "f"(f.x), "f"(f.y));
  }
  __device__ __forceinline__ F2(float x) : F2(make_float2(x, x)) {}
  __device__ __forceinline__ float2 f() const {
    float2 r;
    asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(v));
    return r;
  }
};
__device__ __forceinline__ F2 add2(F2 a, F2 b) {
  asm("add.rn.f32x2 %0, %0, %1;" : "+l"(a.v) : "l"(b.v));
  return a;
}
__device__ __forceinline__ F2 mul2(F2 a, F2 b) {
  asm("mul.rn.f32x2 %0, %0, %1;" : "+l"(a.v) : "l"(b.v));
  return a;
}
__device__ __forceinline__ F2 fma2(F2 a, F2 b, F2 c) {
  asm("fma.rn.f32x2 %0, %1, %2, %0;" : "+l"(c.v) : "l"(a.v), "l"(b.v));
  return c;
}

// A part of a row: the maximum of its logits, and its sums of e^x and e^x x with x counted
// from that maximum (from 0 where all are -inf).
struct Part {
  float m, s, t;
};
__device__ __forceinline__ float origin(float m) { return m == -INFINITY ? 0.f : m; }
// p with its sums on the maximum `top`, in place of its own
__device__ __forceinline__ void onto(Part& p, float top) {
  const float d = max_nan(p.m - origin(top), -1e4f);  // a part of nothing: its sums are 0
  const float f = exp2_fast(d * kLog2e);
  p.t = fmaf(p.s, d, p.t) * f;
  p.s *= f;
  p.m = top;
}
__device__ __forceinline__ Part warp_join(Part p) {
  onto(p, warp_max(p.m));
  p.s = warp_sum(p.s);
  p.t = warp_sum(p.t);
  return p;
}

__device__ __forceinline__ uint4 load_once(const uint4* p) {
  uint4 q;
  asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];"
               : "=r"(q.x), "=r"(q.y), "=r"(q.z), "=r"(q.w)
               : "l"(p));
  return q;
}

__device__ __forceinline__ void cluster_arrive() {
  asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
}
__device__ __forceinline__ void cluster_wait() {
  asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}

// THREADS = 32: one row per warp, 8 warps per CTA, C = 1. Otherwise one row per cluster of C
// CTAs of THREADS.
template <typename T, int NV, int THREADS, int C, bool GRAD>
__global__ void __launch_bounds__(THREADS == 32 ? 256 : THREADS) policy_split_kernel(Args a) {
  constexpr bool kWarp = THREADS == 32;
  constexpr int kWarps = kWarp ? 1 : THREADS / 32;
  constexpr int N = Vec<T>::N;
  constexpr int kAllThreads = THREADS * C;
  __shared__ float4 parts[2][kWarp ? 1 : C * kWarps];
  const float cot = a.cotangent ? *a.cotangent : 1.f;
  if (a.skip_unit && cot == 1.f) return;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int rank = C > 1 ? static_cast<int>(blockIdx.x % C) : 0;  // clusters are runs of C CTAs
  const int at = kWarp ? lane : rank * THREADS + static_cast<int>(threadIdx.x);
  if (C > 1) cluster_arrive(), cluster_wait();  // every CTA's shared memory is there
  const float w = row_weight(a), wg = w * a.grad_scale * cot;
  const long long first = kWarp ? blockIdx.x * 8ll + warp : blockIdx.x / C;
  const long long step = kWarp ? gridDim.x * 8ll : gridDim.x / C;
  double sums[4] = {0, 0, 0, 0};
  int turn = 0;
  for (long long i = first; i < a.rows; i += step) {
    T* g = GRAD ? static_cast<T*>(a.grad) + i * a.vocab : nullptr;
    const int V = static_cast<int>(a.vocab);
    if (a.mask && !a.mask[i]) {  // the same for all threads of the row
      if (GRAD) {
        const int head = min(V, static_cast<int>((16 - (reinterpret_cast<uintptr_t>(g) & 15)) & 15) /
                                    static_cast<int>(sizeof(T)));
        const int vecs = (V - head) / N;
        uint4* q = reinterpret_cast<uint4*>(g + head);
        for (int k = at; k < vecs; k += kAllThreads) q[k] = make_uint4(0, 0, 0, 0);
        if (at < head) g[at] = from_f<T>(0.f);
        const int tail = head + vecs * N;
        if (at < V - tail) g[tail + at] = from_f<T>(0.f);
      }
      if (at == 0 && a.logp) a.logp[i] = 0.f, a.entropy[i] = 0.f;
      continue;
    }
    const T* z = static_cast<const T*>(a.logits) + row_offset(a, i);
    const long long tok = token_of(a, i);
    // whole vectors, and up to N - 1 elements before and after them with one thread each
    const int head = min(V, static_cast<int>((16 - (reinterpret_cast<uintptr_t>(z) & 15)) & 15) /
                                static_cast<int>(sizeof(T)));
    const int vecs = (V - head) / N, tail = head + vecs * N;
    const uint4* zv = reinterpret_cast<const uint4*>(z + head);
    uint4 q[NV];
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      const int j = k * kAllThreads + at;
      q[k] = make_uint4(Vec<T>::kNegInf, Vec<T>::kNegInf, Vec<T>::kNegInf, Vec<T>::kNegInf);
      if (j < vecs) q[k] = load_once(zv + j);
    }
    const int edge = at < head ? at : at >= 16 && at - 16 < V - tail ? tail + at - 16 : -1;
    const float ze = edge >= 0 ? to_f(z[edge]) : -INFINITY;
    const float za = tok >= 0 && tok < V ? to_f(z[tok]) : NAN;

    Part p{ze, 0.f, 0.f};
#pragma unroll
    for (int k = 0; k < NV; ++k) p.m = Vec<T>::most(q[k], p.m);
    {
      const F2 o(-origin(p.m)), scale(kLog2e);
      F2 s(0.f), t(0.f);
#pragma unroll
      for (int k = 0; k < NV; ++k) {
#pragma unroll
        for (int h = 0; h < N / 2; ++h) {
          float2 x = add2(F2(Vec<T>::pair(q[k], h)), o).f();
          x.x = max_nan(x.x, -1e4f), x.y = max_nan(x.y, -1e4f);  // so that 0 x stays 0
          float2 e = mul2(F2(x), scale).f();
          e.x = exp2_fast(e.x), e.y = exp2_fast(e.y);
          s = add2(s, F2(e));
          t = fma2(F2(e), F2(x), t);
        }
      }
      const float x = max_nan(ze - origin(p.m), -1e4f), e = exp2_fast(x * kLog2e);
      p.s = s.f().x + s.f().y + e;
      p.t = fmaf(e, x, t.f().x + t.f().y);
    }
    p = warp_join(p);
    if (!kWarp) {
      if (C == 1) {
        if (lane == 0) parts[turn][warp] = make_float4(p.m, p.s, p.t, 0.f);
        __syncthreads();
      } else {
        // every warp's part goes to all CTAs of the cluster
        if (lane < C) {
          uint32_t to, from = static_cast<uint32_t>(
                           __cvta_generic_to_shared(&parts[turn][rank * kWarps + warp]));
          asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(to) : "r"(from), "r"(lane));
          asm volatile("st.shared::cluster.v4.f32 [%0], {%1, %2, %3, %4};" ::"r"(to), "f"(p.m),
                       "f"(p.s), "f"(p.t), "f"(0.f)
                       : "memory");
        }
        cluster_arrive();
        cluster_wait();
      }
      constexpr int kParts = C * kWarps, kEach = (kParts + 31) / 32;
      Part mine[kEach];
      float top = -INFINITY;
#pragma unroll
      for (int k = 0; k < kEach; ++k) {
        const int j = lane + 32 * k;
        mine[k] = Part{-INFINITY, 0.f, 0.f};
        if (j < kParts) {
          const float4 f = parts[turn][j];
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
      // the next row's parts go to the other buffer; the one after that comes past another
      // barrier, which nobody passes before all have read these
      turn ^= 1;
    }
    const bool empty = p.m == -INFINITY;
    const float m = origin(p.m), ln = empty ? 0.f : logf(p.s), inv = empty ? 0.f : 1.f / p.s;
    const Row r = row_terms(a, i, empty ? (za != za ? za : -INFINITY) : (za - m) - ln,
                            ln - p.t * inv, empty && za == za);
    if (at == 0) {
      if (a.logp) a.logp[i] = r.lp, a.entropy[i] = r.H;
      sums[0] += r.pg, sums[1] += r.k3, sums[2] += r.H, sums[3] += r.cut;
    }
    if (GRAD) {
      const float c = wg * r.c, eta = wg * a.ent;
      const float k0 = inv * (eta * (r.H - ln) - c), k1 = inv * eta;
      uint4* gv = reinterpret_cast<uint4*>(g + head);
      const bool same_phase = ((reinterpret_cast<uintptr_t>(gv)) & 15) == 0;
      const F2 o(-m), scale(kLog2e), f0(k0), f1(k1);
      // the vector and the place in it of the token, if this thread holds it
      const int tk = tok >= 0 && tok < V ? static_cast<int>(tok) : -1, tv = tk - head;
      const int tvec = tv >= 0 && tv < vecs * N ? tv / N : -1;
#pragma unroll
      for (int k = 0; k < NV; ++k) {
        const int j = k * kAllThreads + at;
        if (j >= vecs) break;
        uint4 out;
#pragma unroll
        for (int h = 0; h < N / 2; ++h) {
          float2 x = add2(F2(Vec<T>::pair(q[k], h)), o).f();
          if (a.ent != 0.f) x.x = max_nan(x.x, -1e4f), x.y = max_nan(x.y, -1e4f);
          float2 e = mul2(F2(x), scale).f();
          e.x = exp2_fast(e.x), e.y = exp2_fast(e.y);
          float2 d = mul2(F2(e), a.ent != 0.f ? fma2(f1, F2(x), f0) : f0).f();
          if (j == tvec) {
            if (tv % N == 2 * h) d.x += c;
            if (tv % N == 2 * h + 1) d.y += c;
          }
          Vec<T>::set(out, h, d);
        }
        if (same_phase) {
          gv[j] = out;
        } else {
          const T* o8 = reinterpret_cast<const T*>(&out);
#pragma unroll
          for (int h = 0; h < N; ++h) g[head + j * N + h] = o8[h];
        }
      }
      if (edge >= 0) {
        const float x = max_nan(ze - m, -1e4f);
        float d = exp2_fast(x * kLog2e) * fmaf(k1, x, k0);
        if (edge == tk) d += c;
        g[edge] = from_f<T>(d);
      }
    }
  }
  if (!a.partials) return;
  if (kWarp) {
    __shared__ double part[8][4];
    if (lane == 0)
      for (int k = 0; k < 4; ++k) part[warp][k] = sums[k];
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
// How a batch is run, by its vocabulary and type alone: short rows by groups of lanes,
// longer ones by a warp, a CTA or a cluster each, whatever is longer by the loop.
enum Kind { kGroup, kWarpRows, kSplit, kLoop };
struct Plan {
  Kind kind;
  int lanes, per_lane, rows_each;  // kGroup: L, E, R
  int nv, threads, cluster;        // kWarpRows, kSplit
  long long blocks, n_partials;
  size_t partials_at, bytes;
};

constexpr int kShort = 512;

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
  if (V <= kShort) {
    q.kind = kGroup;
    q.lanes = V <= 4 ? 1 : V <= 8 ? 2 : V <= 16 ? 4 : V <= 32 ? 8 : V <= 64 ? 16 : 32;
    q.per_lane = static_cast<int>((V + q.lanes - 1) / q.lanes);
    q.per_lane = q.per_lane <= 3 ? 3 : q.per_lane <= 4 ? 4 : q.per_lane <= 8 ? 8 : 16;
    if (q.lanes < 8) q.per_lane = 4;
    q.rows_each = q.lanes <= 8 ? q.lanes : q.per_lane <= 4 ? 8 : q.per_lane <= 8 ? 4 : 2;
    const long long rows_per_block = kGroupThreads / q.lanes * q.rows_each;
    q.blocks = at_most((rows + rows_per_block - 1) / rows_per_block, 148 * 8);
    q.n_partials = q.blocks;
  } else if (vecs <= 32 * 16) {
    q.kind = kWarpRows;
    q.threads = 32, q.cluster = 1;
    q.nv = vecs <= 32 * 4 ? 4 : vecs <= 32 * 8 ? 8 : 16;
    q.blocks = at_most((rows + 7) / 8, 148 * 8);
    q.n_partials = q.blocks;
  } else if (vecs <= 512ll * 8 * 8) {
    q.kind = kSplit;
    q.nv = vecs <= 256 * 4 ? 4 : 8;
    q.threads = vecs <= 256ll * 8 * 8 ? 256 : 512;
    q.cluster = 1;
    while (vecs > static_cast<long long>(q.cluster) * q.threads * q.nv) q.cluster *= 2;
    const long long clusters = at_most(rows, 148ll * 4 * 256 / q.threads / q.cluster);
    q.blocks = clusters * q.cluster;
    q.n_partials = clusters;
  } else {
    q.kind = kLoop;
    q.blocks = q.n_partials = at_most(rows, kLoopMaxBlocks);
  }
  q.partials_at = align256(kCountBlocks * sizeof(long long));
  q.bytes = q.partials_at + align256(sizeof(double) * 4 * q.n_partials);
  return q;
}

template <typename T, int L, int E, int R> int launch_group(const Args& a, const Plan& q,
                                                            cudaStream_t st) {
  const unsigned n = static_cast<unsigned>(q.blocks);
  if (a.grad) policy_group_kernel<T, L, E, R, true><<<n, kGroupThreads, 0, st>>>(a);
  else policy_group_kernel<T, L, E, R, false><<<n, kGroupThreads, 0, st>>>(a);
  return launch_status();
}

template <typename T, int NV, int THREADS, int C> int launch_split(const Args& a, const Plan& q,
                                                                   cudaStream_t st) {
  auto* f = a.grad ? policy_split_kernel<T, NV, THREADS, C, true>
                   : policy_split_kernel<T, NV, THREADS, C, false>;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(static_cast<unsigned>(q.blocks));
  cfg.blockDim = dim3(THREADS == 32 ? 256 : THREADS);
  cfg.stream = st;
  cudaLaunchAttribute attr{};
  attr.id = cudaLaunchAttributeClusterDimension;
  attr.val.clusterDim.x = C;
  attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = C > 1 ? 1 : 0;
  return cudaLaunchKernelEx(&cfg, f, a) == cudaSuccess ? launch_status() : SWARP_ERR_CUDA;
}

template <typename T> int run_typed(const Args& a, const Plan& q, cudaStream_t st) {
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
        return q.per_lane == 3   ? launch_group<T, 32, 3, 8>(a, q, st)
               : q.per_lane == 4 ? launch_group<T, 32, 4, 8>(a, q, st)
               : q.per_lane == 8 ? launch_group<T, 32, 8, 4>(a, q, st)
                                 : launch_group<T, 32, 16, 2>(a, q, st);
    }
  }
  if (q.kind == kWarpRows)
    return q.nv == 4   ? launch_split<T, 4, 32, 1>(a, q, st)
           : q.nv == 8 ? launch_split<T, 8, 32, 1>(a, q, st)
                       : launch_split<T, 16, 32, 1>(a, q, st);
  if (q.kind == kSplit) {
    if (q.threads == 512) return launch_split<T, 8, 512, 8>(a, q, st);
    if (q.nv == 4) return launch_split<T, 4, 256, 1>(a, q, st);
    return q.cluster == 1   ? launch_split<T, 8, 256, 1>(a, q, st)
           : q.cluster == 2 ? launch_split<T, 8, 256, 2>(a, q, st)
           : q.cluster == 4 ? launch_split<T, 8, 256, 4>(a, q, st)
                            : launch_split<T, 8, 256, 8>(a, q, st);
  }
  const unsigned n = static_cast<unsigned>(q.blocks);
  if (a.grad) policy_loop_kernel<T, true><<<n, kLoopThreads, 0, st>>>(a);
  else policy_loop_kernel<T, false><<<n, kLoopThreads, 0, st>>>(a);
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
    scalars_kernel<<<1, 256, 0, st>>>(a.partials, some ? q.n_partials : 0, a.kl, a.ent, p->loss,
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
