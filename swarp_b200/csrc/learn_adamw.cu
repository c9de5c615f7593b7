// AdamW over many tensors in one launch, moments in 32 or 8 bits (swarp_adamw_step,
// swarp_grad_norm_partials, swarp_moment8_values; contracts in include/swarp_b200.h).
//
// The tensors' pointers and sizes travel in the launch's own parameters, so a step uploads
// nothing and can be captured in a CUDA graph. A CTA finds its tensor and its chunk of it
// by bisection over the running number of chunks.
//
// 8-bit moments round up or down at random, without bias: to the nearest, an average that
// moves by 1 - b2 = 0.1% a step would never leave a code 12.5% wide. Their new values are
// formed with every rounding written out, so the codes depend on the inputs alone.
#include <cuda_fp8.h>

#include <type_traits>

#include "learn.cuh"

namespace swarp {
namespace learn {
namespace {

constexpr int kBlock = SWARP_MOMENT_BLOCK;
constexpr int kThreads = 256;
constexpr int kMaxTensors = 384;  // of one launch
constexpr int kFewTensors = 24;   // launches of so few take a smaller table
constexpr int kChunk = 2048;      // elements per CTA and turn: a block of 256 per warp
constexpr int kNormBlocks = 592;  // partial sums of one launch

// Whole chunks of the tensors whose addresses allow 16- and 32-byte accesses are numbered
// through all tensors, and what is left of them, with the chunks of the other tensors, apart:
// the code for the former asks nothing element by element.
template <int CAP> struct Table {
  int n;
  int first_full[CAP + 1], first_part[CAP + 1];  // number of each tensor's first
  uint32_t key[CAP];
  uint8_t vectors[CAP];
  swarp_adamw_tensor_t t[CAP];
};
static_assert(sizeof(Table<kMaxTensors>) < 32000, "a launch takes 32764 bytes of parameters");

struct Opt {
  float b1, a1, b2, a2;        // a = 1 - b
  float keep, rate, root2, eps;  // 1 - lr wd; lr / (1 - b1^t); 1 / sqrt(1 - b2^t)
  const float* norm;  // of the gradients; null without clipping
  float max_norm;
};

__host__ __device__ __forceinline__ uint32_t mix(uint32_t x) {
  x ^= x >> 16;
  x *= 0xE80B5AE5u;
  x ^= x >> 15;
  x *= 0xCB276749u;
  return x ^ (x >> 16);
}

// the rest of mix(), after its first step
__device__ __forceinline__ uint32_t mix_on(uint32_t x) {
  x *= 0xE80B5AE5u;
  x ^= x >> 15;
  x *= 0xCB276749u;
  return x ^ (x >> 16);
}

// the tensor of chunk b: the last whose first chunk is not beyond it
__device__ __forceinline__ int tensor_of(const int* first, int n, int b) {
  int lo = 0, hi = n - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (first[mid] <= b) lo = mid;
    else hi = mid - 1;
  }
  return lo;
}

// the gradients' scale
__device__ __forceinline__ float clip_scale(const Opt& o) {
  if (!o.norm) return 1.f;
  const float c = o.max_norm / (*o.norm + 1e-6f);
  return c < 1.f || c != c ? c : 1.f;
}

struct Elem {
  float p, m, v;
};
// sqrt(x) and 1 / x to 1 ulp where they are not subnormal: the step's own size is good to 4 ulp
// then, of which the parameter keeps a few parts in a thousand
__device__ __forceinline__ float sqrt_fast(float x) {
  float r;
  asm("sqrt.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
__device__ __forceinline__ float rcp_fast(float x) {
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
// The step of one element; m and v with every rounding written out.
__device__ __forceinline__ Elem adam(const Opt& o, float p, float g, float m, float v) {
  Elem e;
  e.m = __fadd_rn(__fmul_rn(m, o.b1), __fmul_rn(g, o.a1));
  e.v = __fadd_rn(__fmul_rn(v, o.b2), __fmul_rn(__fmul_rn(g, o.a2), g));
  e.p = p * o.keep - o.rate * (e.m * rcp_fast(sqrt_fast(e.v) * o.root2 + o.eps));
  return e;
}

// A code as the float that it stands for; byte k of w.
__device__ __forceinline__ uint32_t byte_of(uint32_t w, int k) {
  return __byte_perm(w, 0, 0x4440 | k);  // the byte alone
}
__device__ __forceinline__ float decode_m(uint32_t code, int exp) {
  const uint32_t f = code & 127u;
  const uint32_t bits = ((f + 8u * exp - 112u) << 20) | ((code & 128u) << 24);
  return f ? __uint_as_float(bits) : 0.f;
}
// the same for a pair of codes of a block with an ordinary exponent: f is then a float of four
// exponent and three mantissa bits, which the hardware knows, times 2^(exp - 134)
__device__ __forceinline__ bool ordinary_exp(int exp) { return exp >= 14 && exp < 255; }
__device__ __forceinline__ float2 decode_m2(uint32_t codes, float scale) {
  const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2(static_cast<__nv_fp8x2_storage_t>(codes),
                                                   __NV_E4M3);
  const float2 f = __half22float2(__half2(h));
  return make_float2(f.x * scale, f.y * scale);
}
__device__ __forceinline__ float decode_v(uint32_t code, int exp) {
  return code ? __uint_as_float((code << 20) + ((8u * exp - 247u) << 20)) : 0.f;
}
// The code, less its offset, of a number with the given bits (no sign): (bits + (r16 << 4)) >> 20
// less base. Two's complement carries the difference through the shift. NANS: a NaN's carry
// must not leave it.
template <bool NANS> __device__ __forceinline__ int encode(uint32_t bits, uint32_t r, int base) {
  if (NANS) return static_cast<int>(min((bits + r) >> 20, 2047u)) - base;
  return static_cast<int>(bits + r - (static_cast<uint32_t>(base) << 20)) >> 20;
}
// four numbers as bytes, what is outside 0..255 at the nearer end
__device__ __forceinline__ uint32_t bytes_of(int a, int b, int c, int d) {
  uint32_t hi, lo;
  asm("cvt.pack.sat.u8.s32.b32 %0, %1, %2, 0;" : "=r"(hi) : "r"(d), "r"(c));
  asm("cvt.pack.sat.u8.s32.b32 %0, %1, %2, %3;" : "=r"(lo) : "r"(b), "r"(a), "r"(hi));
  return lo;
}
// The codes of four first moments: f where it is 8 or more, under the signs.
template <bool NANS>
__device__ __forceinline__ uint32_t encode_m4(const float* m, const uint32_t* r, int base) {
  uint32_t b[4];
  int f[4];
#pragma unroll
  for (int h = 0; h < 4; ++h) {
    b[h] = __float_as_uint(m[h]);
    f[h] = encode<NANS>(b[h] & 0x7fffffffu, (r[h] << 4) & 0xffff0u, base);
  }
  uint32_t w = bytes_of(f[0], f[1], f[2], f[3]);  // none is above 127
  w &= (((w + 0x78787878u) & 0x80808080u) >> 7) * 255u;
  const uint32_t signs = __byte_perm(__byte_perm(b[0], b[1], 0x0073),
                                     __byte_perm(b[2], b[3], 0x0073), 0x5410);
  return w | (signs & 0x80808080u);
}
// The codes of four second moments (never negative): at least 1 where they are not zero.
template <bool NANS>
__device__ __forceinline__ uint32_t encode_v4(const float* v, const uint32_t* r, int base) {
  uint32_t b[4];
  int f[4];
#pragma unroll
  for (int h = 0; h < 4; ++h) {
    b[h] = __float_as_uint(v[h]);
    f[h] = encode<NANS>(b[h], (r[h] >> 12) & 0xffff0u, base);
  }
  if (min(min(f[0], f[1]), min(f[2], f[3])) < 1) {  // seldom
#pragma unroll
    for (int h = 0; h < 4; ++h) f[h] = max(f[h], b[h] ? 1 : 0);
  }
  return bytes_of(f[0], f[1], f[2], f[3]);
}
// the largest of three magnitudes; a NaN is larger than all
__device__ __forceinline__ float most_of(float a, float b, float c) {
  float r;
  asm("max.NaN.abs.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}

// Eight elements per lane, as 32 bytes of float or 16 of a 16-bit type: a warp's 256 are one
// block, and its accesses whole sectors.
__device__ __forceinline__ void load8(const float* p, float (&x)[8]) {
  asm volatile("ld.global.v8.f32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
               : "=f"(x[0]), "=f"(x[1]), "=f"(x[2]), "=f"(x[3]), "=f"(x[4]), "=f"(x[5]),
                 "=f"(x[6]), "=f"(x[7])
               : "l"(p));
}
__device__ __forceinline__ void store8(float* p, const float (&x)[8]) {
  asm volatile("st.global.v8.f32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(p), "f"(x[0]),
               "f"(x[1]), "f"(x[2]), "f"(x[3]), "f"(x[4]), "f"(x[5]), "f"(x[6]), "f"(x[7])
               : "memory");
}
template <typename T> __device__ __forceinline__ void load8(const T* p, float (&x)[8]) {
  const uint4 q = *reinterpret_cast<const uint4*>(p);
  const T* h = reinterpret_cast<const T*>(&q);
#pragma unroll
  for (int k = 0; k < 8; ++k) x[k] = to_f(h[k]);
}
template <typename T> __device__ __forceinline__ void store8(T* p, const float (&x)[8]) {
  uint4 q;
  T* h = reinterpret_cast<T*>(&q);
#pragma unroll
  for (int k = 0; k < 8; ++k) h[k] = from_f<T>(x[k]);
  *reinterpret_cast<uint4*>(p) = q;
}
// n of the eight elements at p, one by one
template <typename T>
__device__ __forceinline__ void load8(const T* p, float (&x)[8], bool vec, int n) {
  if (vec) return load8(p, x);
#pragma unroll
  for (int k = 0; k < 8; ++k) x[k] = k < n ? to_f(p[k]) : 0.f;
}
template <typename T>
__device__ __forceinline__ void store8(T* p, const float (&x)[8], bool vec, int n) {
  if (vec) return store8(p, x);
#pragma unroll
  for (int k = 0; k < 8; ++k)
    if (k < n) p[k] = from_f<T>(x[k]);
}
__device__ __forceinline__ uint2 load_codes(const uint8_t* p, bool vec, int n) {
  if (vec) return *reinterpret_cast<const uint2*>(p);
  uint32_t w[2] = {0, 0};
#pragma unroll
  for (int k = 0; k < 8; ++k)
    if (k < n) w[k / 4] |= static_cast<uint32_t>(p[k]) << (8 * (k % 4));
  return make_uint2(w[0], w[1]);
}
__device__ __forceinline__ void store_codes(uint8_t* p, uint2 q, bool vec, int n) {
  if (vec) {
    *reinterpret_cast<uint2*>(p) = q;
    return;
  }
#pragma unroll
  for (int k = 0; k < 8; ++k)
    if (k < n) p[k] = static_cast<uint8_t>((k < 4 ? q.x : q.y) >> (8 * (k % 4)));
}
// A chunk of a tensor, the same for the whole CTA, and a lane's eight elements of it: element
// `at` of the chunk on, with the tensor's elements from `off` on. The chunk's part of an
// address stays in uniform registers.
struct Place {
  long long off;
  int room;  // the tensor's elements in the chunk
  __device__ __forceinline__ Place(long long off, int room) : off(off), room(room) {}
  // chunk q of those that are not whole
  template <int CAP> __device__ __forceinline__ Place(const Table<CAP>& tab, int k, int q) {
    const int before = tab.first_full[k + 1] - tab.first_full[k];
    off = static_cast<long long>(q - tab.first_part[k] + before) * kChunk;
    const long long left = tab.t[k].n - off;
    room = left < kChunk ? static_cast<int>(left) : kChunk;
  }
};
// whole chunk b
template <int CAP>
__device__ __forceinline__ Place whole_place(const Table<CAP>& tab, int k, int b) {
  return Place(static_cast<long long>(b - tab.first_full[k]) * kChunk, kChunk);
}
struct Lane {
  int at, n;  // the first of the lane's elements in the chunk, and how many are there
  bool any;   // the warp has some
  bool vec;
  __device__ __forceinline__ Lane(const Place& p, bool vectors) {
    at = static_cast<int>(threadIdx.x) * 8;
    const int left = p.room - at;
    n = left >= 8 ? 8 : left > 0 ? left : 0;
    any = (at & ~255) < p.room;
    vec = vectors && n == 8;
  }
};

// ------------------------------------------------------------------- sums of squares
// Eight squares in float, then on in double; where a float does not hold the squares (elements
// above 1e18 or below 1e-15 alone) they too are formed in double, so the norm is good to float
// rounding whatever the gradients' size.
// A CTA takes a run of whole chunks, several in flight, and its share of the others. Bound by
// memory: 300 MB of bf16 in 62 us, 75% of the copy rate (131 with one chunk in flight).
template <typename T, int CAP>
__global__ void __launch_bounds__(kThreads, kNormBlocks / 148)
    norm_kernel(const __grid_constant__ Table<CAP> tab, double* partials) {
  constexpr int kAtOnce = sizeof(T) == 4 ? 4 : 8;
  __shared__ double part[kThreads / 32];
  double s = 0;
  const int grid = static_cast<int>(gridDim.x), cta = static_cast<int>(blockIdx.x);
  auto square = [](const float (&g)[8]) {
    float q = 0.f;
#pragma unroll
    for (int h = 0; h < 8; ++h) q = fmaf(g[h], g[h], q);
    double d = q;
    // (float16 has no such elements; zeros come here too)
    if (!std::is_same<T, __half>::value && !(q > 1e-30f && q < 1e37f)) {
      d = 0;
#pragma unroll
      for (int h = 0; h < 8; ++h) d = fma(static_cast<double>(g[h]), static_cast<double>(g[h]), d);
    }
    return d;
  };
  const int full = tab.first_full[tab.n], each = (full + grid - 1) / grid;
  const int end = min((cta + 1) * each, full);
  int b = cta * each;
  for (int k = b < end ? tensor_of(tab.first_full, tab.n, b) : 0; b < end; ++k) {
    const int first = tab.first_full[k], stop = min(end, tab.first_full[k + 1]);
    const T* p = static_cast<const T*>(tab.t[k].grad) + threadIdx.x * 8;
    for (; b + kAtOnce <= stop; b += kAtOnce) {
      float g[kAtOnce][8];
#pragma unroll
      for (int c = 0; c < kAtOnce; ++c) load8(p + static_cast<long long>(b - first + c) * kChunk, g[c]);
#pragma unroll
      for (int c = 0; c < kAtOnce; ++c) s += square(g[c]);
    }
    for (; b < stop; ++b) {
      float g[8];
      load8(p + static_cast<long long>(b - first) * kChunk, g);
      s += square(g);
    }
  }
  for (int q = cta; q < tab.first_part[tab.n]; q += grid) {
    const int k = tensor_of(tab.first_part, tab.n, q);
    const Place c(tab, k, q);
    const Lane l(c, tab.vectors[k]);
    float g[8];
    load8(static_cast<const T*>(tab.t[k].grad) + c.off + l.at, g, l.vec, l.n);
    s += square(g);
  }
  s = warp_sum(s);
  if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = s;
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int w = 1; w < kThreads / 32; ++w) s += part[w];
    partials[blockIdx.x] = s;
  }
}

// The partial sums in a fixed order, and the norm.
__global__ void norm_finish_kernel(const double* partials, long long n, float* norm) {
  __shared__ double part[kThreads / 32];
  double s = 0;
  for (long long k = threadIdx.x; k < n; k += kThreads) s += partials[k];
  s = warp_sum(s);
  if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = s;
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int w = 1; w < kThreads / 32; ++w) s += part[w];
    *norm = static_cast<float>(sqrt(s));
  }
}

// -------------------------------------------------------------------------- the step
// The new codes of a lane's eight elements from i on (a multiple of 8). NANS: the block has a
// NaN or an infinity.
template <bool NANS>
__device__ __forceinline__ void encode8(const float (&m)[8], const float (&v)[8], uint32_t i,
                                        uint32_t key, int em, int ev, uint2& cm, uint2& cv) {
  // mix((i + h) ^ key): h is in the three lowest bits, which its first step only copies
  const uint32_t x = i ^ key, first = x ^ (x >> 16);
  uint32_t r[8];
#pragma unroll
  for (int h = 0; h < 8; ++h) r[h] = mix_on(first ^ h);
  cm = make_uint2(encode_m4<NANS>(m, r, 8 * em - 112), encode_m4<NANS>(m + 4, r + 4, 8 * em - 112));
  cv = make_uint2(encode_v4<NANS>(v, r, 8 * ev - 247), encode_v4<NANS>(v + 4, r + 4, 8 * ev - 247));
}

__device__ __forceinline__ float* param_of(const swarp_adamw_tensor_t& t) {
  return t.master ? t.master : static_cast<float*>(t.param);
}

// Moments of 32 bits: one chunk per CTA. 28 bytes an element and little arithmetic; the many
// short CTAs keep the memory busiest (150 million elements: 624 us, 104% of the copy rate,
// against 685 with resident CTAs that walk the chunks).
template <bool FULL, typename T>
__device__ __forceinline__ void step32(const swarp_adamw_tensor_t& t, const Place& c,
                                       const Lane& l, const Opt& o, float scale) {
  float *pp = param_of(t) + c.off, *pm = static_cast<float*>(t.exp_avg) + c.off,
        *pv = static_cast<float*>(t.exp_avg_sq) + c.off;
  const bool vec = FULL || l.vec;
  float p[8], g[8], m[8], v[8];
  load8(pp + l.at, p, vec, l.n);
  load8(static_cast<const T*>(t.grad) + c.off + l.at, g, vec, l.n);
  load8(pm + l.at, m, vec, l.n);
  load8(pv + l.at, v, vec, l.n);
#pragma unroll
  for (int h = 0; h < 8; ++h) {
    const Elem e = adam(o, p[h], g[h] * scale, m[h], v[h]);
    p[h] = e.p, m[h] = e.m, v[h] = e.v;
  }
  store8(pm + l.at, m, vec, l.n);
  store8(pv + l.at, v, vec, l.n);
  store8(pp + l.at, p, vec, l.n);
  if (t.master) store8(static_cast<T*>(t.param) + c.off + l.at, p, vec, l.n);
}

template <typename T, int CAP>
__global__ void __launch_bounds__(kThreads, 4)
    adamw32_kernel(const __grid_constant__ Table<CAP> tab, const __grid_constant__ Opt o) {
  const float scale = clip_scale(o);
  const int b = static_cast<int>(blockIdx.x), full = tab.first_full[tab.n];
  if (b < full) {
    const int k = tensor_of(tab.first_full, tab.n, b);
    const Place c = whole_place(tab, k, b);
    step32<true, T>(tab.t[k], c, Lane(c, true), o, scale);
  } else {
    const int k = tensor_of(tab.first_part, tab.n, b - full);
    const Place c(tab, k, b - full);
    step32<false, T>(tab.t[k], c, Lane(c, tab.vectors[k]), o, scale);
  }
}

// Moments of 8 bits: some 65 instructions an element against 16 bytes, so arithmetic and
// memory take about as long. One chunk per CTA here too (250 million elements of bf16: 696 us,
// 89% of the copy rate, against 909 with resident CTAs that ask for the next chunk before they
// work on this one).
constexpr int kResident8 = 4;

// FULL: the chunk is whole, so no access asks.
template <typename T> struct Eight {
  float p[8], g[8];
  uint2 cm, cv;
  int em, ev;

  template <bool FULL>
  __device__ __forceinline__ void load(const swarp_adamw_tensor_t& t, const Place& c,
                                       const Lane& l) {
    const long long block = c.off / kBlock;
    em = (t.exp_avg_exp + block)[threadIdx.x >> 5];
    ev = (t.exp_avg_sq_exp + block)[threadIdx.x >> 5];
    cm = load_codes(static_cast<const uint8_t*>(t.exp_avg) + c.off + l.at, FULL || l.vec, l.n);
    cv = load_codes(static_cast<const uint8_t*>(t.exp_avg_sq) + c.off + l.at, FULL || l.vec, l.n);
    load8(param_of(t) + c.off + l.at, p, FULL || l.vec, l.n);
    load8(static_cast<const T*>(t.grad) + c.off + l.at, g, FULL || l.vec, l.n);
  }

  template <bool FULL>
  __device__ __forceinline__ void step(const swarp_adamw_tensor_t& t, const Place& c,
                                       const Lane& l, const Opt& o, float scale, uint32_t key) {
    float m[8], v[8];
    if (ordinary_exp(em)) {
      const float to = __uint_as_float(static_cast<uint32_t>(em - 7) << 23);
#pragma unroll
      for (int h = 0; h < 4; ++h) {
        const uint32_t w = h < 2 ? cm.x : cm.y;
        const float2 f = decode_m2(h % 2 ? w >> 16 : w & 0xffffu, to);
        m[2 * h] = f.x, m[2 * h + 1] = f.y;
      }
    } else {
#pragma unroll
      for (int h = 0; h < 8; ++h) m[h] = decode_m(byte_of(h < 4 ? cm.x : cm.y, h % 4), em);
    }
    const uint32_t base = (8u * ev - 247u) << 20;
#pragma unroll
    for (int h = 0; h < 8; ++h)
      v[h] = __uint_as_float((byte_of(h < 4 ? cv.x : cv.y, h % 4) << 20) + base);
    if (__vcmpeq4(cv.x, 0) | __vcmpeq4(cv.y, 0)) {  // seldom: a code of zero
#pragma unroll
      for (int h = 0; h < 8; ++h)
        if (byte_of(h < 4 ? cv.x : cv.y, h % 4) == 0) v[h] = 0.f;
    }
    // elements beyond the tensor's end are zeros, and stay zeros
    float tm = 0.f, tv = 0.f;
#pragma unroll
    for (int h = 0; h < 8; ++h) {
      const Elem e = adam(o, p[h], g[h] * scale, m[h], v[h]);
      p[h] = e.p, m[h] = e.m, v[h] = e.v;
      if (h % 2) tm = most_of(tm, m[h - 1], m[h]), tv = most_of(tv, v[h - 1], v[h]);
    }
    store8(param_of(t) + c.off + l.at, p, FULL || l.vec, l.n);
    if (t.master) store8(static_cast<T*>(t.param) + c.off + l.at, p, FULL || l.vec, l.n);
    const int em1 = __reduce_max_sync(kAll, __float_as_uint(tm)) >> 23;
    const int ev1 = __reduce_max_sync(kAll, __float_as_uint(tv)) >> 23;
    const uint32_t i = static_cast<uint32_t>(c.off) + l.at;
    key += static_cast<uint32_t>(c.off >> 32);
    uint2 dm, dv;
    if (max(em1, ev1) < 255) encode8<false>(m, v, i, key, em1, ev1, dm, dv);
    else encode8<true>(m, v, i, key, em1, ev1, dm, dv);
    store_codes(static_cast<uint8_t*>(t.exp_avg) + c.off + l.at, dm, FULL || l.vec, l.n);
    store_codes(static_cast<uint8_t*>(t.exp_avg_sq) + c.off + l.at, dv, FULL || l.vec, l.n);
    if ((threadIdx.x & 31) == 0) {
      const long long block = c.off / kBlock;
      (t.exp_avg_exp + block)[threadIdx.x >> 5] = static_cast<uint8_t>(em1);
      (t.exp_avg_sq_exp + block)[threadIdx.x >> 5] = static_cast<uint8_t>(ev1);
    }
  }
};

template <typename T, int CAP>
__global__ void __launch_bounds__(kThreads, kResident8)
    adamw8_kernel(const __grid_constant__ Table<CAP> tab, const __grid_constant__ Opt o) {
  const float scale = clip_scale(o);
  const int b = static_cast<int>(blockIdx.x), full = tab.first_full[tab.n];
  Eight<T> z;
  if (b < full) {
    const int k = tensor_of(tab.first_full, tab.n, b);
    const Place c = whole_place(tab, k, b);
    const Lane l(c, true);
    z.template load<true>(tab.t[k], c, l);
    z.template step<true>(tab.t[k], c, l, o, scale, tab.key[k]);
  } else {
    const int k = tensor_of(tab.first_part, tab.n, b - full);
    const Place c(tab, k, b - full);
    const Lane l(c, tab.vectors[k]);
    if (!l.any) return;  // the whole warp
    z.template load<false>(tab.t[k], c, l);
    z.template step<false>(tab.t[k], c, l, o, scale, tab.key[k]);
  }
}

template <typename O>
__global__ void __launch_bounds__(kThreads)
    values_kernel(const uint8_t* codes, const uint8_t* exps, long long n, int is_signed,
                  int vectors, O* out) {
  // 16 elements per thread, in two halves; 3 bytes an element at 80% of the copy rate
  const long long i0 = (blockIdx.x * static_cast<long long>(kThreads) + threadIdx.x) * 16;
  if (i0 >= n) return;
  const int e = exps[i0 / kBlock];
  uint2 c[2];
  int left[2];
  bool vec[2];
#pragma unroll
  for (int q = 0; q < 2; ++q) {
    left[q] = static_cast<int>(max(0ll, min(n - i0 - 8 * q, 8ll)));
    vec[q] = vectors && left[q] == 8;
    c[q] = load_codes(codes + i0 + 8 * q, vec[q], left[q]);
  }
#pragma unroll
  for (int q = 0; q < 2; ++q) {
    float x[8];
#pragma unroll
    for (int h = 0; h < 8; ++h) {
      const uint32_t code = byte_of(h < 4 ? c[q].x : c[q].y, h % 4);
      x[h] = is_signed ? decode_m(code, e) : decode_v(code, e);
    }
    store8(out + i0 + 8 * q, x, vec[q], left[q]);
  }
}

// --------------------------------------------------------------------------- the host
bool dtype_ok(int32_t d) { return d == SWARP_F32 || d == SWARP_BF16 || d == SWARP_F16; }

bool aligned(const void* p, uintptr_t n) { return reinterpret_cast<uintptr_t>(p) % n == 0; }
bool vectors_ok(const swarp_adamw_tensor_t& t, int32_t dtype, int bits) {
  const uintptr_t own = dtype == SWARP_F32 ? 32 : 16, moment = bits == 8 ? 8 : 32;
  return aligned(t.param, own) && aligned(t.grad, own) && aligned(t.master, 32) &&
         aligned(t.exp_avg, moment) && aligned(t.exp_avg_sq, moment);
}

// Calls f(table, chunks) for each group of CAP tensors (empty ones take no entry), once at
// least.
template <int CAP, typename F>
int for_each_table(const swarp_adamw_tensor_t* tensors, int64_t n, int32_t dtype, int bits,
                   uint32_t key0, uint32_t first, F f) {
  Table<CAP> tab;
  int64_t i = 0;
  do {
    tab.n = 0;
    long long full = 0, part = 0;
    for (const int64_t end = i + CAP; i < n && i < end; ++i) {
      if (tensors[i].n == 0) continue;
      const bool vec = vectors_ok(tensors[i], dtype, bits);
      tab.t[tab.n] = tensors[i];
      tab.vectors[tab.n] = vec;
      tab.key[tab.n] = mix(key0 + first + static_cast<uint32_t>(i));
      tab.first_full[tab.n] = static_cast<int>(full);
      tab.first_part[tab.n++] = static_cast<int>(part);
      const long long whole = vec ? tensors[i].n / kChunk : 0;
      full += whole;
      part += (tensors[i].n + kChunk - 1) / kChunk - whole;
      if (full + part > 0x3fffffffll) return SWARP_ERR_UNSUPPORTED;
    }
    tab.first_full[tab.n] = static_cast<int>(full);
    tab.first_part[tab.n] = static_cast<int>(part);
    if (const int rc = f(tab, static_cast<int>(full + part))) return rc;
  } while (i < n);
  return SWARP_OK;
}

template <typename T, int CAP>
int step_typed(const swarp_adamw_t* s, const Opt& o, const swarp_adamw_tensor_t* tensors,
               int64_t n, cudaStream_t st) {
  const uint32_t key0 = mix(s->seed + static_cast<uint32_t>(s->step));
  return for_each_table<CAP>(tensors, n, s->dtype, s->moment_bits, key0, s->first_tensor,
                             [&](const Table<CAP>& tab, int chunks) {
                               if (chunks == 0) return static_cast<int>(SWARP_OK);
                               if (s->moment_bits == 8)
                                 adamw8_kernel<T, CAP><<<chunks, kThreads, 0, st>>>(tab, o);
                               else
                                 adamw32_kernel<T, CAP><<<chunks, kThreads, 0, st>>>(tab, o);
                               return launch_status();
                             });
}

template <typename T, int CAP>
int norm_typed(int32_t dtype, const swarp_adamw_tensor_t* tensors, int64_t n, double* partials,
               cudaStream_t st) {
  return for_each_table<CAP>(tensors, n, dtype, 32, 0, 0, [&](const Table<CAP>& tab, int) {
    norm_kernel<T, CAP><<<kNormBlocks, kThreads, 0, st>>>(tab, partials);
    partials += kNormBlocks;
    return launch_status();
  });
}
template <typename T>
int norm(int32_t dtype, const swarp_adamw_tensor_t* tensors, int64_t n, double* partials,
         cudaStream_t st) {
  return n <= kFewTensors ? norm_typed<T, kFewTensors>(dtype, tensors, n, partials, st)
                          : norm_typed<T, kMaxTensors>(dtype, tensors, n, partials, st);
}
template <typename T>
int step(const swarp_adamw_t* s, const Opt& o, const swarp_adamw_tensor_t* tensors, int64_t n,
         cudaStream_t st) {
  return n <= kFewTensors ? step_typed<T, kFewTensors>(s, o, tensors, n, st)
                          : step_typed<T, kMaxTensors>(s, o, tensors, n, st);
}

}  // namespace
}  // namespace learn
}  // namespace swarp

using namespace swarp::learn;

extern "C" {

int64_t swarp_grad_norm_partials_count(int64_t n_tensors) {
  const int64_t launches = (n_tensors + kMaxTensors - 1) / kMaxTensors;
  return n_tensors < 0 ? 0 : kNormBlocks * (launches > 0 ? launches : 1);
}

int swarp_grad_norm_partials(int32_t dtype, const swarp_adamw_tensor_t* tensors,
                             int64_t n_tensors, double* partials, void* stream) {
  if (!dtype_ok(dtype) || n_tensors < 0 || (n_tensors > 0 && !tensors) || !partials)
    return SWARP_ERR_INVALID_ARG;
  for (int64_t i = 0; i < n_tensors; ++i)
    if (tensors[i].n < 0 || (tensors[i].n > 0 && !tensors[i].grad)) return SWARP_ERR_INVALID_ARG;
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  return dtype == SWARP_F32    ? norm<float>(dtype, tensors, n_tensors, partials, st)
         : dtype == SWARP_BF16 ? norm<__nv_bfloat16>(dtype, tensors, n_tensors, partials, st)
                               : norm<__half>(dtype, tensors, n_tensors, partials, st);
}

int swarp_adamw_step(const swarp_adamw_t* s, const swarp_adamw_tensor_t* tensors,
                     int64_t n_tensors, void* stream) {
  if (!s || !dtype_ok(s->dtype) || (s->moment_bits != 32 && s->moment_bits != 8) || s->step < 1)
    return SWARP_ERR_INVALID_ARG;
  if (!(s->beta1 >= 0.0 && s->beta1 < 1.0 && s->beta2 >= 0.0 && s->beta2 < 1.0))
    return SWARP_ERR_INVALID_ARG;
  if (n_tensors < 0 || (n_tensors > 0 && !tensors)) return SWARP_ERR_INVALID_ARG;
  if (s->norm_partials && (s->n_norm_partials < 1 || !(s->max_norm > 0.0) || !s->grad_norm))
    return SWARP_ERR_INVALID_ARG;
  for (int64_t i = 0; i < n_tensors; ++i) {
    const swarp_adamw_tensor_t& t = tensors[i];
    if (t.n < 0) return SWARP_ERR_INVALID_ARG;
    if (t.n == 0) continue;
    if (!t.param || !t.grad || !t.exp_avg || !t.exp_avg_sq) return SWARP_ERR_INVALID_ARG;
    if ((s->dtype == SWARP_F32) != (t.master == nullptr)) return SWARP_ERR_INVALID_ARG;
    if (s->moment_bits == 8 && (!t.exp_avg_exp || !t.exp_avg_sq_exp)) return SWARP_ERR_INVALID_ARG;
  }
  Opt o;
  o.b1 = static_cast<float>(s->beta1);
  o.a1 = static_cast<float>(1.0 - s->beta1);
  o.b2 = static_cast<float>(s->beta2);
  o.a2 = static_cast<float>(1.0 - s->beta2);
  o.keep = static_cast<float>(1.0 - s->lr * s->weight_decay);
  const double t = static_cast<double>(s->step);
  o.rate = static_cast<float>(s->lr / (1.0 - pow(s->beta1, t)));
  o.root2 = static_cast<float>(1.0 / sqrt(1.0 - pow(s->beta2, t)));
  // the kernels take the root of a subnormal v (below 2^-126, whose root is 1e-19) as 0
  o.eps = static_cast<float>(s->eps > 1e-19 ? s->eps : 1e-19);
  o.norm = s->norm_partials ? s->grad_norm : nullptr;
  o.max_norm = static_cast<float>(s->max_norm);
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (s->norm_partials) {
    norm_finish_kernel<<<1, kThreads, 0, st>>>(s->norm_partials, s->n_norm_partials, s->grad_norm);
    if (const int rc = launch_status()) return rc;
  }
  return s->dtype == SWARP_F32    ? step<float>(s, o, tensors, n_tensors, st)
         : s->dtype == SWARP_BF16 ? step<__nv_bfloat16>(s, o, tensors, n_tensors, st)
                                  : step<__half>(s, o, tensors, n_tensors, st);
}

int swarp_moment8_values(const uint8_t* codes, const uint8_t* exponents, int64_t n,
                         int32_t is_signed, int32_t dtype, void* out, void* stream) {
  if (n < 0 || (dtype != SWARP_F32 && dtype != SWARP_BF16)) return SWARP_ERR_INVALID_ARG;
  if (n == 0) return SWARP_OK;
  const int64_t blocks = (n + 16 * kThreads - 1) / (16 * kThreads);
  if (!codes || !exponents || !out || blocks > 0x7fffffffll) return SWARP_ERR_INVALID_ARG;
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  const unsigned grid = static_cast<unsigned>(blocks);
  const int vec = aligned(codes, 8) && aligned(out, dtype == SWARP_F32 ? 32 : 16);
  if (dtype == SWARP_F32)
    values_kernel<<<grid, kThreads, 0, st>>>(codes, exponents, n, is_signed, vec,
                                             static_cast<float*>(out));
  else
    values_kernel<<<grid, kThreads, 0, st>>>(codes, exponents, n, is_signed, vec,
                                             static_cast<__nv_bfloat16*>(out));
  return launch_status();
}

}  // extern "C"
