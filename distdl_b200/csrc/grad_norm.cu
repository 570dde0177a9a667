// The norm of many tensors together, and their scaling to a largest norm.
//
//   norm = sqrt(sum over tensors and elements of g^2);   g <- g * min(1, max_norm / (norm + 1e-6))
//
// Bandwidth: every element is read for the norm and, where the norm is too large, read and written once more.  The tensors'
// addresses travel as arguments of the kernels (no table in device memory, nothing to keep or to capture), kTensors at a time;
// their elements are dealt to the CTAs in pieces of kPiece.  Squares and their sums are formed in 64 bits: no finite
// gradient overflows or vanishes, and the sum does not depend on the order of many roundings; every CTA writes its own sum,
// and whoever needs the norm adds them in the same order.  The scaling walks the pieces from the last to the first: what the
// norm read last is still in L2.
#include <algorithm>
#include <new>

#include "common.cuh"
#include "runtime.cuh"

#include <cuda_fp16.h>

using namespace dd;

namespace {

constexpr int kThreads = 512;
constexpr int kTensors = 160;                                 // of one launch: its arguments stay below 4 KB
constexpr int kPiece = 65536;                                 // elements: where a piece ends a CTA has less in flight (norm of
                                                              // 2.9e8 bf16 values: 16384 177 us, 32768 96, 65536 91, 131072 92)
constexpr int kCtasPerSm = 2;

struct Tensors {
  void* p[kTensors];
  long long n[kTensors];
  int first[kTensors + 1];                                    // pieces before the tensor
  unsigned char type[kTensors];                               // 0 bf16, 1 fp16, 2 fp32
  int count;
};
static_assert(sizeof(Tensors) < 3800, "arguments of a kernel");

// The tensor of a piece, by bisection.
__device__ __forceinline__ int tensor_of(const Tensors& t, int piece) {
  int lo = 0, hi = t.count - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (t.first[mid] <= piece) lo = mid;
    else hi = mid - 1;
  }
  return lo;
}

__device__ __forceinline__ float to_f(float v) { return v; }
__device__ __forceinline__ float to_f(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_f(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ void set(float* p, float v) { *p = v; }
__device__ __forceinline__ void set(__half* p, float v) { *p = __float2half_rn(v); }
__device__ __forceinline__ void set(__nv_bfloat16* p, float v) { *p = __float2bfloat16_rn(v); }

// A 32-bit word of memory as its one or two elements, and back.
template <typename T> struct Word;
template <> struct Word<float> {
  static constexpr int kElements = 1;
  static __device__ __forceinline__ float2 get(uint32_t u) { return make_float2(__uint_as_float(u), 0.f); }
  static __device__ __forceinline__ uint32_t put(float2 f) { return __float_as_uint(f.x); }
};
template <> struct Word<__half> {
  static constexpr int kElements = 2;
  static __device__ __forceinline__ float2 get(uint32_t u) { return __half22float2(*reinterpret_cast<const __half2*>(&u)); }
  static __device__ __forceinline__ uint32_t put(float2 f) {
    const __half2 h = __floats2half2_rn(f.x, f.y);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
};
template <> struct Word<__nv_bfloat16> {
  static constexpr int kElements = 2;
  static __device__ __forceinline__ float2 get(uint32_t u) { return unpack_bf16x2(u); }
  static __device__ __forceinline__ uint32_t put(float2 f) { return pack_bf16x2(f.x, f.y); }
};

// 16-byte loads of a thread in flight.  Measured (1.5e9 fp32, 2.9e8 bf16 values): norm with 4 829 and 100 us, with 8 823 and
// 96; scaling with 1 1 989 and 230 us, with 2 1 896 and 188, with 4 1 983 and 188 (reads and writes that alternate less often
// would hold more open pages of DRAM).
constexpr int kNormVectors = 8, kScaleVectors = 2;

// Calls one(element) for what is not on 16-byte vectors and many(vectors, i, n) for what is (vectors i, i + kThreads, ... of n:
// V of them), of elements [lo, hi) of p.
template <int V, typename T, typename One, typename Many>
__device__ __forceinline__ void walk(T* p, long long lo, long long hi, One one, Many many) {
  constexpr int VE = 16 / sizeof(T);
  const int off = (int)((16 - reinterpret_cast<uintptr_t>(p + lo) % 16) % 16 / sizeof(T));
  const long long a = min(hi, lo + off), b = a + (hi - a) / VE * VE;
  if (lo + threadIdx.x < a) one(p + lo + threadIdx.x);
  if (b + threadIdx.x < hi) one(p + b + threadIdx.x);
  uint4* v = reinterpret_cast<uint4*>(p + a);
  const int n = (int)((b - a) / VE);
  for (int i = threadIdx.x; i < n; i += V * kThreads) many(v, i, n);
}

template <typename T>
__device__ __forceinline__ double squares(T* p, long long lo, long long hi) {
  double sum = 0.0;
  auto add = [&](uint32_t u) {
    const float2 f = Word<T>::get(u);
    sum = fma((double)f.x, (double)f.x, sum);
    if constexpr (Word<T>::kElements == 2) sum = fma((double)f.y, (double)f.y, sum);
  };
  walk<kNormVectors>(p, lo, hi, [&](T* x) { const double d = to_f(*x); sum = fma(d, d, sum); },
       [&](uint4* v, int i, int n) {
         uint4 r[kNormVectors];
#pragma unroll
         for (int u = 0; u < kNormVectors; ++u) r[u] = i + u * kThreads < n ? v[i + u * kThreads] : make_uint4(0u, 0u, 0u, 0u);
#pragma unroll
         for (int u = 0; u < kNormVectors; ++u) { add(r[u].x); add(r[u].y); add(r[u].z); add(r[u].w); }
       });
  return sum;
}

template <typename T>
__device__ __forceinline__ void scale(T* p, long long lo, long long hi, float c) {
  auto times = [&](uint32_t u) {
    const float2 f = Word<T>::get(u);
    return Word<T>::put(make_float2(f.x * c, f.y * c));
  };
  walk<kScaleVectors>(p, lo, hi, [&](T* x) { set(x, to_f(*x) * c); },
       [&](uint4* v, int i, int n) {
         uint4 r[kScaleVectors];
#pragma unroll
         for (int u = 0; u < kScaleVectors; ++u)
           if (i + u * kThreads < n) r[u] = v[i + u * kThreads];
#pragma unroll
         for (int u = 0; u < kScaleVectors; ++u)
           if (i + u * kThreads < n)
             v[i + u * kThreads] = make_uint4(times(r[u].x), times(r[u].y), times(r[u].z), times(r[u].w));
       });
}

__device__ __forceinline__ double block_sum_d(double v, double* red) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
  __syncthreads();
  double s = 0.0;
  for (int k = 0; k < kThreads / 32; ++k) s += red[k];        // (every thread, in the same order)
  __syncthreads();
  return s;
}

// partial[CTA] = the CTA's sum of squares.
__global__ void __launch_bounds__(kThreads, kCtasPerSm) sumsq_kernel(const __grid_constant__ Tensors t, double* __restrict__ partial) {
  __shared__ double red[kThreads / 32];
  grid_dependency_launch();
  double sum = 0.0;
  for (int piece = blockIdx.x; piece < t.first[t.count]; piece += gridDim.x) {
    const int i = tensor_of(t, piece);
    const long long lo = (long long)(piece - t.first[i]) * kPiece, hi = min(t.n[i], lo + kPiece);
    if (t.type[i] == 0) sum += squares(reinterpret_cast<__nv_bfloat16*>(t.p[i]), lo, hi);
    else if (t.type[i] == 1) sum += squares(reinterpret_cast<__half*>(t.p[i]), lo, hi);
    else sum += squares(reinterpret_cast<float*>(t.p[i]), lo, hi);
  }
  sum = block_sum_d(sum, red);
  if (threadIdx.x == 0) partial[blockIdx.x] = sum;
}

// The sum of squares of all `parts` CTAs (of every launch), in order.
__device__ __forceinline__ double total_of(const double* partial, int parts, double* red) {
  double v = 0.0;
  for (int i = threadIdx.x; i < parts; i += kThreads) v += partial[i];
  return block_sum_d(v, red);
}

__global__ void __launch_bounds__(kThreads) norm_kernel(const double* __restrict__ partial, int parts, float* __restrict__ norm,
                                                        double* __restrict__ squared) {
  __shared__ double red[kThreads / 32];
  const double sum = total_of(partial, parts, red);
  if (threadIdx.x == 0) {
    if (norm != nullptr) *norm = (float)sqrt(sum);
    if (squared != nullptr) *squared = sum;
  }
}

// g *= min(1, max_norm / (norm + 1e-6)); nothing is touched where that is 1.  parts > 0: the norm is that of the partial sums,
// which every CTA adds for itself, and is written to *norm; else it is read there.
__global__ void __launch_bounds__(kThreads, kCtasPerSm)
clip_kernel(const __grid_constant__ Tensors t, const double* __restrict__ partial, int parts, float* __restrict__ norm,
            double max_norm) {
  __shared__ double red[kThreads / 32];
  grid_dependency_launch();
  double size;
  if (parts > 0) {
    size = sqrt(total_of(partial, parts, red));
    if (blockIdx.x == 0 && threadIdx.x == 0) *norm = (float)size;
  } else {
    size = *norm;
  }
  const float c = (float)(max_norm / (size + 1e-6));
  if (c >= 1.f) return;                                       // (a NaN goes on: it is to show)
  const int pieces = t.first[t.count];
  for (int k = blockIdx.x; k < pieces; k += gridDim.x) {
    const int piece = pieces - 1 - k, i = tensor_of(t, piece);
    const long long lo = (long long)(piece - t.first[i]) * kPiece, hi = min(t.n[i], lo + kPiece);
    if (t.type[i] == 0) scale(reinterpret_cast<__nv_bfloat16*>(t.p[i]), lo, hi, c);
    else if (t.type[i] == 1) scale(reinterpret_cast<__half*>(t.p[i]), lo, hi, c);
    else scale(reinterpret_cast<float*>(t.p[i]), lo, hi, c);
  }
}

struct Span { uintptr_t lo, hi; };

// Whether the tensors can be worked on: known types, addresses of whole elements; with `apart`, none of them overlaps another.
int check_tensors(void* const* p, const long long* n, const unsigned char* type, int count, bool apart) {
  if (count < 0 || (count > 0 && (p == nullptr || n == nullptr || type == nullptr))) return DD_ERR_BAD_ARG;
  for (int i = 0; i < count; ++i) {
    if (n[i] < 0 || type[i] > 2 || (n[i] > 0 && p[i] == nullptr)) return DD_ERR_BAD_ARG;
    if (n[i] > 0 && reinterpret_cast<uintptr_t>(p[i]) % (type[i] == 2 ? 4 : 2) != 0) return DD_ERR_ALIGN;
    if (n[i] / kPiece > 0x7ffffff0LL / (count + 1)) return DD_ERR_TOO_LARGE;
  }
  if (!apart || count < 2) return DD_OK;
  Span* s = new (std::nothrow) Span[count];
  if (s == nullptr) return DD_ERR_TOO_LARGE;
  int m = 0;
  for (int i = 0; i < count; ++i)
    if (n[i] > 0) {
      const uintptr_t a = reinterpret_cast<uintptr_t>(p[i]);
      s[m++] = {a, a + (uintptr_t)n[i] * (type[i] == 2 ? 4 : 2)};
    }
  std::sort(s, s + m, [](const Span& a, const Span& b) { return a.lo < b.lo; });
  bool ok = true;
  for (int i = 1; i < m; ++i) ok = ok && s[i - 1].hi <= s[i].lo;
  delete[] s;
  return ok ? DD_OK : DD_ERR_BAD_ARG;
}

// Tensors [from, ...) of as many as one launch takes; returns the number after the last.
int gather(Tensors& t, void* const* p, const long long* n, const unsigned char* type, int count, int from) {
  t.count = 0;
  t.first[0] = 0;
  for (; from < count && t.count < kTensors; ++from) {
    if (n[from] == 0) continue;
    const int i = t.count++;
    t.p[i] = p[from];
    t.n[i] = n[from];
    t.type[i] = type[from];
    t.first[i + 1] = t.first[i] + (int)((n[from] + kPiece - 1) / kPiece);
  }
  return from;
}

inline int ctas_for(const Tensors& t) {
  const int pieces = t.first[t.count], most = current_sm_count() * kCtasPerSm;
  return pieces < most ? pieces : most;
}

}  // namespace

// Rows (of 8 bytes) of scratch for `count` tensors.
DD_API int dd_grad_norm_parts(int count) {
  const long long parts = (long long)current_sm_count() * kCtasPerSm * ((count + kTensors - 1) / kTensors);
  return parts > 0x7fffffffLL ? 0x7fffffff : (int)parts;
}

// Norm of `count` tensors given by address, number of elements and type (0 bf16, 1 fp16, 2 fp32; host arrays), and their
// scaling to max_norm.  scratch: dd_grad_norm_parts(count) words of 8 bytes (not read where the norm is given).
//   given == 0, clip == 0: *norm (fp32) and *squared (fp64, the sum of squares), where they are not null
//   given == 0, clip == 1: *norm, and the tensors clipped
//   given == 1, clip == 1: the tensors clipped by the norm that is in *norm
DD_API int dd_grad_norm(void* const* p, const long long* n, const unsigned char* type, int count, double* scratch, int parts,
                        float* norm, double* squared, double max_norm, int given, int clip, void* stream) {
  int e = check_tensors(p, n, type, count, clip != 0);
  if (e) return e;
  if ((clip && norm == nullptr) || (given && !clip) || (!given && scratch == nullptr)) return DD_ERR_BAD_ARG;
  if (!given && parts < dd_grad_norm_parts(count)) return DD_ERR_BAD_ARG;
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  Tensors t;
  int used = 0, launches = 0;
  if (!given) {
    for (int at = 0; at < count;) {
      at = gather(t, p, n, type, count, at);
      if (t.count == 0) break;
      const int ctas = ctas_for(t);
      sumsq_kernel<<<ctas, kThreads, 0, s>>>(t, scratch + used);
      used += ctas;
      ++launches;
    }
    // (one launch of tensors: the scaling adds the sums up for itself)
    if (!clip || launches != 1) norm_kernel<<<1, kThreads, 0, s>>>(scratch, used, norm, squared);
  }
  if (clip) {
    const bool fold = !given && launches == 1;
    for (int at = 0; at < count;) {
      at = gather(t, p, n, type, count, at);
      if (t.count == 0) break;
      clip_kernel<<<ctas_for(t), kThreads, 0, s>>>(t, scratch, fold ? used : 0, norm, max_norm);
    }
  }
  return (int)cudaGetLastError();
}
