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

template <int CAP> struct Table {
  int n;
  int first_chunk[CAP + 1];
  uint32_t key[CAP];
  uint8_t vectors[CAP];  // the tensor's addresses allow 16- and 32-byte accesses
  swarp_adamw_tensor_t t[CAP];
};
static_assert(sizeof(Table<kMaxTensors>) < 32000, "a launch takes 32764 bytes of parameters");

struct Opt {
  float b1, a1, b2, a2;        // a = 1 - b
  float keep, rate, root2, eps;  // 1 - lr wd; lr / (1 - b1^t); 1 / sqrt(1 - b2^t)
  const double* partials;
  long long n_partials;
  float max_norm;
  float* norm_out;
};

__host__ __device__ __forceinline__ uint32_t mix(uint32_t x) {
  x ^= x >> 16;
  x *= 0xE80B5AE5u;
  x ^= x >> 15;
  x *= 0xCB276749u;
  return x ^ (x >> 16);
}

// the tensor of chunk b: the last whose first chunk is not beyond it
template <int CAP> __device__ __forceinline__ int tensor_of(const Table<CAP>& tab, int b) {
  int lo = 0, hi = tab.n - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (tab.first_chunk[mid] <= b) lo = mid;
    else hi = mid - 1;
  }
  return lo;
}

// The gradients' scale, the same in every CTA: the partial sums added in a fixed order.
__device__ __forceinline__ float clip_scale(const Opt& o) {
  if (!o.partials) return 1.f;
  __shared__ double part[kThreads / 32];
  __shared__ float scale;
  double s = 0;
  for (long long k = threadIdx.x; k < o.n_partials; k += kThreads) s += o.partials[k];
  s = warp_sum(s);
  if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = s;
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int w = 1; w < kThreads / 32; ++w) s += part[w];
    const float norm = static_cast<float>(sqrt(s));
    const float c = o.max_norm / (norm + 1e-6f);
    scale = c < 1.f || c != c ? c : 1.f;
    if (o.norm_out && blockIdx.x == 0) *o.norm_out = norm;
  }
  __syncthreads();
  return scale;
}

struct Elem {
  float p, m, v;
};
// to 1 ulp, subnormals included; the step's own size is good to 4 ulp then, of which the
// parameter keeps a few parts in a thousand
__device__ __forceinline__ float sqrt_fast(float x) {
  float r;
  asm("sqrt.approx.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
// The step of one element; m and v with every rounding written out.
__device__ __forceinline__ Elem adam(const Opt& o, float p, float g, float m, float v) {
  Elem e;
  e.m = __fadd_rn(__fmul_rn(m, o.b1), __fmul_rn(g, o.a1));
  e.v = __fadd_rn(__fmul_rn(v, o.b2), __fmul_rn(__fmul_rn(g, o.a2), g));
  e.p = p * o.keep - o.rate * __fdividef(e.m, sqrt_fast(e.v) * o.root2 + o.eps);
  return e;
}

__device__ __forceinline__ float decode_m(uint32_t code, int exp) {
  const uint32_t f = code & 127u;
  const uint32_t bits = ((f + 8u * exp - 112u) << 20) | ((code & 128u) << 24);
  return f ? __uint_as_float(bits) : 0.f;
}
__device__ __forceinline__ float decode_v(uint32_t code, int exp) {
  return code ? __uint_as_float((code + 8u * exp - 247u) << 20) : 0.f;
}
// bits: those of the value without its sign; top: the block's exponent
__device__ __forceinline__ uint32_t encode(uint32_t bits, uint32_t r16) {
  return min((bits + (r16 << 4)) >> 20, 2047u);  // 2047: a NaN stays one
}
__device__ __forceinline__ uint32_t encode_m(float m, uint32_t r16, int top) {
  const uint32_t b = __float_as_uint(m);
  const int f = static_cast<int>(encode(b & 0x7fffffffu, r16)) - (8 * top - 112);
  return f < 8 ? 0u : static_cast<uint32_t>(f) | ((b >> 24) & 128u);
}
__device__ __forceinline__ uint32_t encode_v(float v, uint32_t r16, int top) {
  const uint32_t b = __float_as_uint(v) & 0x7fffffffu;
  const int f = static_cast<int>(encode(b, r16)) - (8 * top - 247);
  return static_cast<uint32_t>(max(f, b ? 1 : 0));
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
__device__ __forceinline__ uint32_t code_of(uint2 q, int k) {
  return ((k < 4 ? q.x : q.y) >> (8 * (k % 4))) & 255u;
}

// ------------------------------------------------------------------- sums of squares
// Eight squares in float, then on in double: the norm is good to float rounding at any size.
// Four chunks at a time, so that enough loads are in flight.
template <typename T, int CAP>
__global__ void __launch_bounds__(kThreads)
    norm_kernel(const __grid_constant__ Table<CAP> tab, double* partials) {
  constexpr int kAtOnce = 4;
  __shared__ double part[kThreads / 32];
  double s = 0;
  const int chunks = tab.first_chunk[tab.n];
  for (int b0 = blockIdx.x * kAtOnce; b0 < chunks; b0 += gridDim.x * kAtOnce) {
    float g[kAtOnce][8];
    int k = tensor_of(tab, b0);
#pragma unroll
    for (int c = 0; c < kAtOnce; ++c) {
      const int b = b0 + c;
#pragma unroll
      for (int h = 0; h < 8; ++h) g[c][h] = 0.f;
      if (b >= chunks) continue;
      while (tab.first_chunk[k + 1] <= b) ++k;
      const long long i =
          static_cast<long long>(b - tab.first_chunk[k]) * kChunk + threadIdx.x * 8ll;
      const long long left = static_cast<long long>(tab.t[k].n) - i;
      if (left > 0)
        load8(static_cast<const T*>(tab.t[k].grad) + i, g[c], tab.vectors[k] && left >= 8,
              static_cast<int>(min(left, 8ll)));
    }
#pragma unroll
    for (int c = 0; c < kAtOnce; ++c) {
      float q = 0.f;
#pragma unroll
      for (int h = 0; h < 8; ++h) q = fmaf(g[c][h], g[c][h], q);
      s += q;
    }
  }
  s = warp_sum(s);
  if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = s;
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int w = 1; w < kThreads / 32; ++w) s += part[w];
    partials[blockIdx.x] = s;
  }
}

// -------------------------------------------------------------------------- the step
template <typename T, int BITS, int CAP>
__global__ void __launch_bounds__(kThreads)
    adamw_kernel(const __grid_constant__ Table<CAP> tab, const __grid_constant__ Opt o) {
  const float scale = clip_scale(o);
  const int lane = threadIdx.x & 31;
  for (int b = blockIdx.x; b < tab.first_chunk[tab.n]; b += gridDim.x) {
    const int k = tensor_of(tab, b);
    const swarp_adamw_tensor_t& t = tab.t[k];
    // the warp's block, and the lane's eight elements of it
    const long long block = static_cast<long long>(b - tab.first_chunk[k]) * (kChunk / kBlock) +
                            (threadIdx.x >> 5);
    if (block * kBlock >= t.n) continue;  // the whole warp
    const long long i = block * kBlock + lane * 8;
    const int n = static_cast<int>(max(0ll, min(static_cast<long long>(t.n) - i, 8ll)));
    const bool vec = tab.vectors[k] && n == 8;
    float* pp = t.master ? t.master : static_cast<float*>(t.param);
    float p[8], g[8];
    load8(pp + i, p, vec, n);
    load8(static_cast<const T*>(t.grad) + i, g, vec, n);
    if constexpr (BITS == 32) {
      float m[8], v[8];
      float *pm = static_cast<float*>(t.exp_avg), *pv = static_cast<float*>(t.exp_avg_sq);
      load8(pm + i, m, vec, n);
      load8(pv + i, v, vec, n);
#pragma unroll
      for (int h = 0; h < 8; ++h) {
        const Elem e = adam(o, p[h], g[h] * scale, m[h], v[h]);
        p[h] = e.p, m[h] = e.m, v[h] = e.v;
      }
      store8(pm + i, m, vec, n);
      store8(pv + i, v, vec, n);
    } else {
      uint8_t *pm = static_cast<uint8_t*>(t.exp_avg), *pv = static_cast<uint8_t*>(t.exp_avg_sq);
      const uint2 cm = load_codes(pm + i, vec, n), cv = load_codes(pv + i, vec, n);
      const int em0 = t.exp_avg_exp[block], ev0 = t.exp_avg_sq_exp[block];
      float m[8], v[8];
      uint32_t tm = 0, tv = 0;
#pragma unroll
      for (int h = 0; h < 8; ++h) {
        const Elem e = adam(o, p[h], g[h] * scale, decode_m(code_of(cm, h), em0),
                            decode_v(code_of(cv, h), ev0));
        p[h] = e.p, m[h] = e.m, v[h] = e.v;
        if (h < n) {
          tm = max(tm, __float_as_uint(e.m) & 0x7fffffffu);
          tv = max(tv, __float_as_uint(e.v) & 0x7fffffffu);
        }
      }
      const int em = __reduce_max_sync(kAll, tm) >> 23, ev = __reduce_max_sync(kAll, tv) >> 23;
      uint32_t wm[2] = {0, 0}, wv[2] = {0, 0};
      const uint32_t key = tab.key[k] + static_cast<uint32_t>(i >> 32);
#pragma unroll
      for (int h = 0; h < 8; ++h) {
        const uint32_t r = mix((static_cast<uint32_t>(i) + h) ^ key);
        wm[h / 4] |= encode_m(m[h], r & 0xffffu, em) << (8 * (h % 4));
        wv[h / 4] |= encode_v(v[h], r >> 16, ev) << (8 * (h % 4));
      }
      store_codes(pm + i, make_uint2(wm[0], wm[1]), vec, n);
      store_codes(pv + i, make_uint2(wv[0], wv[1]), vec, n);
      if (lane == 0) t.exp_avg_exp[block] = em, t.exp_avg_sq_exp[block] = ev;
    }
    store8(pp + i, p, vec, n);
    if (t.master) store8(static_cast<T*>(t.param) + i, p, vec, n);
  }
}

template <typename O>
__global__ void __launch_bounds__(kThreads)
    values_kernel(const uint8_t* codes, const uint8_t* exps, long long n, int is_signed,
                  int vectors, O* out) {
  const long long i = (blockIdx.x * static_cast<long long>(kThreads) + threadIdx.x) * 8;
  if (i >= n) return;
  const int left = static_cast<int>(min(n - i, 8ll)), e = exps[i / kBlock];
  const bool vec = vectors && left == 8;
  const uint2 c = load_codes(codes + i, vec, left);
  float x[8];
#pragma unroll
  for (int h = 0; h < 8; ++h)
    x[h] = is_signed ? decode_m(code_of(c, h), e) : decode_v(code_of(c, h), e);
  store8(out + i, x, vec, left);
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
    long long chunks = 0;
    for (const int64_t end = i + CAP; i < n && i < end; ++i) {
      if (tensors[i].n == 0) continue;
      const long long more = (tensors[i].n + kChunk - 1) / kChunk;
      if (chunks + more > 0x3fffffffll) return SWARP_ERR_UNSUPPORTED;
      tab.t[tab.n] = tensors[i];
      tab.vectors[tab.n] = vectors_ok(tensors[i], dtype, bits);
      tab.key[tab.n] = mix(key0 + first + static_cast<uint32_t>(i));
      tab.first_chunk[tab.n++] = static_cast<int>(chunks);
      chunks += more;
    }
    tab.first_chunk[tab.n] = static_cast<int>(chunks);
    if (const int rc = f(tab, static_cast<int>(chunks))) return rc;
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
                               const int blocks = chunks < 148 * 8 ? chunks : 148 * 8;
                               if (s->moment_bits == 8)
                                 adamw_kernel<T, 8, CAP><<<blocks, kThreads, 0, st>>>(tab, o);
                               else
                                 adamw_kernel<T, 32, CAP><<<blocks, kThreads, 0, st>>>(tab, o);
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
  if (s->norm_partials && (s->n_norm_partials < 1 || !(s->max_norm > 0.0)))
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
  o.eps = static_cast<float>(s->eps);
  o.partials = s->norm_partials;
  o.n_partials = s->n_norm_partials;
  o.max_norm = static_cast<float>(s->max_norm);
  o.norm_out = s->grad_norm;
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  return s->dtype == SWARP_F32    ? step<float>(s, o, tensors, n_tensors, st)
         : s->dtype == SWARP_BF16 ? step<__nv_bfloat16>(s, o, tensors, n_tensors, st)
                                  : step<__half>(s, o, tensors, n_tensors, st);
}

int swarp_moment8_values(const uint8_t* codes, const uint8_t* exponents, int64_t n,
                         int32_t is_signed, int32_t dtype, void* out, void* stream) {
  if (n < 0 || (dtype != SWARP_F32 && dtype != SWARP_BF16)) return SWARP_ERR_INVALID_ARG;
  if (n == 0) return SWARP_OK;
  const int64_t blocks = (n + 8 * kThreads - 1) / (8 * kThreads);
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
