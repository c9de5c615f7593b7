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
constexpr int kMaxTensors = 384;  // of one launch: 384 x 76 bytes of its parameters
constexpr int kNormBlocks = 592;  // partial sums of one launch

struct Table {
  int n;
  int first_chunk[kMaxTensors + 1];
  uint32_t key[kMaxTensors];
  swarp_adamw_tensor_t t[kMaxTensors];
};
static_assert(sizeof(Table) < 32000, "a launch takes 32764 bytes of parameters");

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
__device__ __forceinline__ int tensor_of(const Table& tab, int b) {
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
// The step of one element; m and v with every rounding written out.
__device__ __forceinline__ Elem adam(const Opt& o, float p, float g, float m, float v) {
  Elem e;
  e.m = __fadd_rn(__fmul_rn(m, o.b1), __fmul_rn(g, o.a1));
  e.v = __fadd_rn(__fmul_rn(v, o.b2), __fmul_rn(__fmul_rn(g, o.a2), g));
  e.p = p * o.keep - o.rate * (e.m / (sqrtf(e.v) * o.root2 + o.eps));
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

// ------------------------------------------------------------------- sums of squares
constexpr int kChunk = 4096;

template <typename T>
__global__ void __launch_bounds__(kThreads)
    norm_kernel(const __grid_constant__ Table tab, double* partials) {
  __shared__ double part[kThreads / 32];
  double s = 0;
  for (int b = blockIdx.x; b < tab.first_chunk[tab.n]; b += gridDim.x) {
    const int k = tensor_of(tab, b);
    const long long at = static_cast<long long>(b - tab.first_chunk[k]) * kChunk;
    const long long end = min(at + kChunk, static_cast<long long>(tab.t[k].n));
    const T* g = static_cast<const T*>(tab.t[k].grad);
    float q = 0.f;
    for (long long i = at + threadIdx.x; i < end; i += kThreads) {
      const float x = to_f(g[i]);
      q = fmaf(x, x, q);
    }
    s += q;
  }
  s = warp_sum(s);
  if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = s;
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int w = 1; w < kThreads / 32; ++w) s += part[w];
    partials[blockIdx.x] = s;
  }
}

// ------------------------------------------------------------------------- the steps
template <typename T>
__global__ void __launch_bounds__(kThreads)
    adamw32_kernel(const __grid_constant__ Table tab, const __grid_constant__ Opt o) {
  const float scale = clip_scale(o);
  const int k = tensor_of(tab, blockIdx.x);
  const swarp_adamw_tensor_t& t = tab.t[k];
  const long long at = static_cast<long long>(blockIdx.x - tab.first_chunk[k]) * kChunk;
  const long long end = min(at + kChunk, static_cast<long long>(t.n));
  float* m = static_cast<float*>(t.exp_avg);
  float* v = static_cast<float*>(t.exp_avg_sq);
  float* p = t.master ? t.master : static_cast<float*>(t.param);
  for (long long i = at + threadIdx.x; i < end; i += kThreads) {
    const float g = to_f(static_cast<const T*>(t.grad)[i]) * scale;
    const Elem e = adam(o, p[i], g, m[i], v[i]);
    m[i] = e.m;
    v[i] = e.v;
    p[i] = e.p;
    if (t.master) static_cast<T*>(t.param)[i] = from_f<T>(e.p);
  }
}

// One CTA per block of 256 elements.
template <typename T>
__global__ void __launch_bounds__(kThreads)
    adamw8_kernel(const __grid_constant__ Table tab, const __grid_constant__ Opt o) {
  __shared__ uint32_t tops[2][kThreads / 32];
  const float scale = clip_scale(o);
  const int k = tensor_of(tab, blockIdx.x);
  const swarp_adamw_tensor_t& t = tab.t[k];
  const long long block = blockIdx.x - tab.first_chunk[k];
  const long long i = block * kBlock + threadIdx.x;
  const bool in = i < t.n;
  uint8_t* m8 = static_cast<uint8_t*>(t.exp_avg);
  uint8_t* v8 = static_cast<uint8_t*>(t.exp_avg_sq);
  float* p = t.master ? t.master : static_cast<float*>(t.param);
  Elem e{0.f, 0.f, 0.f};
  if (in) {
    const float g = to_f(static_cast<const T*>(t.grad)[i]) * scale;
    e = adam(o, p[i], g, decode_m(m8[i], t.exp_avg_exp[block]),
             decode_v(v8[i], t.exp_avg_sq_exp[block]));
  }
  uint32_t tm = __reduce_max_sync(kAll, __float_as_uint(e.m) & 0x7fffffffu);
  uint32_t tv = __reduce_max_sync(kAll, __float_as_uint(e.v) & 0x7fffffffu);
  if ((threadIdx.x & 31) == 0) tops[0][threadIdx.x >> 5] = tm, tops[1][threadIdx.x >> 5] = tv;
  __syncthreads();
  for (int w = 0; w < kThreads / 32; ++w) tm = max(tm, tops[0][w]), tv = max(tv, tops[1][w]);
  const int em = tm >> 23, ev = tv >> 23;
  if (threadIdx.x == 0) t.exp_avg_exp[block] = em, t.exp_avg_sq_exp[block] = ev;
  if (!in) return;
  const uint32_t h = mix(static_cast<uint32_t>(i) ^ (tab.key[k] + static_cast<uint32_t>(i >> 32)));
  m8[i] = static_cast<uint8_t>(encode_m(e.m, h & 0xffffu, em));
  v8[i] = static_cast<uint8_t>(encode_v(e.v, h >> 16, ev));
  p[i] = e.p;
  if (t.master) static_cast<T*>(t.param)[i] = from_f<T>(e.p);
}

template <typename O>
__global__ void __launch_bounds__(kThreads)
    values_kernel(const uint8_t* codes, const uint8_t* exps, long long n, int is_signed, O* out) {
  const long long i = blockIdx.x * static_cast<long long>(kThreads) + threadIdx.x;
  if (i >= n) return;
  const int e = exps[i / kBlock];
  out[i] = from_f<O>(is_signed ? decode_m(codes[i], e) : decode_v(codes[i], e));
}

// --------------------------------------------------------------------------- the host
bool dtype_ok(int32_t d) { return d == SWARP_F32 || d == SWARP_BF16 || d == SWARP_F16; }

// Calls f(table, chunks) for each group of kMaxTensors tensors (empty ones take no entry), once
// at least.
template <typename F>
int for_each_table(const swarp_adamw_tensor_t* tensors, int64_t n, int chunk, uint32_t key0,
                   uint32_t first, F f) {
  Table tab;
  int64_t i = 0;
  do {
    tab.n = 0;
    long long chunks = 0;
    for (const int64_t end = i + kMaxTensors; i < n && i < end; ++i) {
      if (tensors[i].n == 0) continue;
      const long long more = (tensors[i].n + chunk - 1) / chunk;
      if (chunks + more > 0x7fffffffll) return SWARP_ERR_UNSUPPORTED;
      tab.t[tab.n] = tensors[i];
      tab.key[tab.n] = mix(key0 + first + static_cast<uint32_t>(i));
      tab.first_chunk[tab.n++] = static_cast<int>(chunks);
      chunks += more;
    }
    tab.first_chunk[tab.n] = static_cast<int>(chunks);
    if (const int rc = f(tab, static_cast<int>(chunks))) return rc;
  } while (i < n);
  return SWARP_OK;
}

template <typename T>
int step_typed(const swarp_adamw_t* s, const Opt& o, const swarp_adamw_tensor_t* tensors,
               int64_t n, cudaStream_t st) {
  const uint32_t key0 = mix(s->seed + static_cast<uint32_t>(s->step));
  const bool eight = s->moment_bits == 8;
  return for_each_table(tensors, n, eight ? kBlock : kChunk, key0, s->first_tensor,
                        [&](const Table& tab, int chunks) {
                          if (chunks == 0) return static_cast<int>(SWARP_OK);
                          if (eight) adamw8_kernel<T><<<chunks, kThreads, 0, st>>>(tab, o);
                          else adamw32_kernel<T><<<chunks, kThreads, 0, st>>>(tab, o);
                          return launch_status();
                        });
}

template <typename T>
int norm_typed(const swarp_adamw_tensor_t* tensors, int64_t n, double* partials, cudaStream_t st) {
  return for_each_table(tensors, n, kChunk, 0, 0, [&](const Table& tab, int) {
    norm_kernel<T><<<kNormBlocks, kThreads, 0, st>>>(tab, partials);
    partials += kNormBlocks;
    return launch_status();
  });
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
  return dtype == SWARP_F32    ? norm_typed<float>(tensors, n_tensors, partials, st)
         : dtype == SWARP_BF16 ? norm_typed<__nv_bfloat16>(tensors, n_tensors, partials, st)
                               : norm_typed<__half>(tensors, n_tensors, partials, st);
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
  return s->dtype == SWARP_F32    ? step_typed<float>(s, o, tensors, n_tensors, st)
         : s->dtype == SWARP_BF16 ? step_typed<__nv_bfloat16>(s, o, tensors, n_tensors, st)
                                  : step_typed<__half>(s, o, tensors, n_tensors, st);
}

int swarp_moment8_values(const uint8_t* codes, const uint8_t* exponents, int64_t n,
                         int32_t is_signed, int32_t dtype, void* out, void* stream) {
  if (n < 0 || (dtype != SWARP_F32 && dtype != SWARP_BF16)) return SWARP_ERR_INVALID_ARG;
  if (n == 0) return SWARP_OK;
  if (!codes || !exponents || !out || (n + kThreads - 1) / kThreads > 0x7fffffffll)
    return SWARP_ERR_INVALID_ARG;
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  const unsigned blocks = static_cast<unsigned>((n + kThreads - 1) / kThreads);
  if (dtype == SWARP_F32)
    values_kernel<<<blocks, kThreads, 0, st>>>(codes, exponents, n, is_signed,
                                               static_cast<float*>(out));
  else
    values_kernel<<<blocks, kThreads, 0, st>>>(codes, exponents, n, is_signed,
                                               static_cast<__nv_bfloat16*>(out));
  return launch_status();
}

}  // extern "C"
