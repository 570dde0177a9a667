// Queries and keys between their projection and attention: rotary positions (either pairing, of a part of the head, at any
// positions) and the RMS norm of every head with the rotation in the same pass, forward and backward.
//
//   rotation   (a, b) -> (a c - b s, b c + a s), c + i s = magnitude e^(i position f), for the pairs of the leading `rd`
//              components of a head: (i, i + rd / 2), or neighbours (2 i, 2 i + 1); the components behind stay
//   norm       u = x r, r = (mean x^2 + eps)^(-1/2);  y = R(u w), w shared by the query heads, another by the key heads
//   backward   g = R^T dy;  dw = sum over tokens and heads of g u;  dx = r (g w - u mean(g w u))
//
// Bandwidth bounds them: a head is read and written once, with 16 bytes per access.  So nothing else travels:
//  * a group of lanes (8 for 128 bf16 components) holds a head in registers, two vectors per lane, and a lane that holds one
//    component of a pair also holds the other (the vectors lie half the rotated part apart, or the pairs lie inside a vector);
//  * the angles are computed, not read: position times frequency in turns in 64 bits, reduced to half a turn (exact for
//    every position below 2^31, where 32 bits are off by radians), then sin and cos in 32 bits, once per lane for all heads of
//    a chunk.  The frequencies travel as arguments of the kernel: no table, no copy, nothing to capture or to keep;
//  * the backward pass recomputes r from x, which it needs anyway.
// A unit of work is a token's chunk of up to kChunkHeads heads of one kind (query / key / rest); units are dealt to the
// groups of a grid of two CTAs per SM, kind by kind, so that the lanes of a warp nearly always do the same.
#include "common.cuh"
#include "runtime.cuh"

#include <cuda_fp16.h>

using namespace dd;

namespace {

constexpr int kThreads = 256;
constexpr int kMaxPairs = 256;        // heads of up to 512 components
constexpr int kCtasPerSm = 2;

enum Kind { kRope = 0, kNormFwd = 1, kNormBwd = 2 };
// How a lane finds the other component of a pair.
enum Pairing {
  kApart = 0,     // halves, rd / 2 whole vectors: in the lane's other vector
  kInside = 1,    // neighbours: in the same vector
  kShared = 2,    // halves at any distance, and single components: through shared memory
};

struct HeadArgs {
  const void* x;              // [tokens, heads, hd] by token and head stride (elements), unit stride inside a head
  long long x_row, x_head;
  const void* dy;             // backward
  long long dy_row, dy_head;
  void* out;                  // y, or dx; may be x
  long long out_row, out_head;
  const void* wq;             // [hd] or null (ones)
  const void* wk;
  const void* positions;      // [seq] of 4 or 8 bytes, of token % seq, or null: offset + token % seq
  float* partial;             // backward: [gridDim.x][2][hd], or null
  long long offset;
  unsigned tokens, seq;
  int heads[3];               // query, key and other heads (those are copied; none in place)
  int chunk[3], chunks[3];    // heads per unit, units per token
  int hd, rd, group;          // group: lanes per head (a power of two)
  int wide_positions, wide_weights, neighbours;
  float magnitude, sign, eps;
  double turns[kMaxPairs];    // frequency of each pair in turns per position
};

template <typename T> __device__ __forceinline__ float to_f(T v);
template <> __device__ __forceinline__ float to_f(float v) { return v; }
template <> __device__ __forceinline__ float to_f(__half v) { return __half2float(v); }
template <> __device__ __forceinline__ float to_f(__nv_bfloat16 v) { return __bfloat162float(v); }
template <typename T> __device__ __forceinline__ T from_f(float v);
template <> __device__ __forceinline__ float from_f(float v) { return v; }
template <> __device__ __forceinline__ __half from_f(float v) { return __float2half_rn(v); }
template <> __device__ __forceinline__ __nv_bfloat16 from_f(float v) { return __float2bfloat16_rn(v); }

// VE components as they lie in memory: 16 bytes, or one component.  (Held as words: arrays of 16-bit values would take a
// register each.)
template <typename T, int VE> struct Pack { uint4 v; };
template <typename T> struct Pack<T, 1> { T v; };

template <typename T, int VE>
__device__ __forceinline__ Pack<T, VE> load_pack(const T* p) {
  Pack<T, VE> r;
  if constexpr (VE == 1) r.v = *p;
  else r.v = *reinterpret_cast<const uint4*>(p);
  return r;
}
template <typename T, int VE>
__device__ __forceinline__ void clear(Pack<T, VE>& r) {
  if constexpr (VE == 1) r.v = from_f<T>(0.f);
  else r.v = make_uint4(0u, 0u, 0u, 0u);
}
__device__ __forceinline__ float2 two(uint32_t u, __nv_bfloat16) {
  return make_float2(__uint_as_float(u << 16), __uint_as_float(u & 0xffff0000u));
}
__device__ __forceinline__ float2 two(uint32_t u, __half) { return __half22float2(*reinterpret_cast<const __half2*>(&u)); }
__device__ __forceinline__ uint32_t word(float a, float b, __nv_bfloat16) { return pack_bf16x2(a, b); }
__device__ __forceinline__ uint32_t word(float a, float b, __half) {
  const __half2 v = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&v);
}
template <typename T, int VE>
__device__ __forceinline__ void unpack(const Pack<T, VE>& r, float* f) {
  if constexpr (VE == 1) {
    f[0] = to_f(r.v);
  } else if constexpr (VE == 4) {
    f[0] = __uint_as_float(r.v.x); f[1] = __uint_as_float(r.v.y); f[2] = __uint_as_float(r.v.z); f[3] = __uint_as_float(r.v.w);
  } else {
    const float2 a = two(r.v.x, T()), b = two(r.v.y, T()), c = two(r.v.z, T()), d = two(r.v.w, T());
    f[0] = a.x; f[1] = a.y; f[2] = b.x; f[3] = b.y; f[4] = c.x; f[5] = c.y; f[6] = d.x; f[7] = d.y;
  }
}
template <typename T, int VE>
__device__ __forceinline__ void store_pack(T* p, const float* f) {
  if constexpr (VE == 1) *p = from_f<T>(f[0]);
  else if constexpr (VE == 4) *reinterpret_cast<float4*>(p) = make_float4(f[0], f[1], f[2], f[3]);
  else *reinterpret_cast<uint4*>(p) = make_uint4(word(f[0], f[1], T()), word(f[2], f[3], T()), word(f[4], f[5], T()),
                                                 word(f[6], f[7], T()));
}

__device__ __forceinline__ float group_sum(float v, int group) {
  for (int o = group >> 1; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// NV vectors of VE components per lane and head.
template <typename T, int VE, int NV, int PAIRING, int KIND>
__global__ void __launch_bounds__(kThreads, kCtasPerSm) heads_kernel(const __grid_constant__ HeadArgs a) {
  constexpr int N = NV * VE;                                  // components per lane
  constexpr int ANGLES = PAIRING == kShared ? N : N / 2;      // pairs per lane (kShared: of every component its pair's)
  constexpr int U = VE == 1 ? 1 : KIND == kNormBwd ? 2 : 4;   // heads whose loads are in flight together
  extern __shared__ float smem[];                             // kShared: a head per group; later dw sums
  grid_dependency_launch();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int g = lane & (a.group - 1), per_warp = 32 / a.group, in_warp = lane / a.group;
  const int vectors = a.hd / VE, half = a.rd >> 1;
  float* exchange = smem + (size_t)(warp * per_warp + in_warp) * a.hd;

  // this lane's vectors of a head, and the pair of each of its components (-1: stays)
  int at[NV];
#pragma unroll
  for (int s = 0; s < NV; ++s) {
    if constexpr (PAIRING == kApart) {
      const int paired = half / VE;                           // lanes that hold a vector of each half
      at[s] = (g < paired ? g + s * paired : 2 * paired + 2 * (g - paired) + s) * VE;
    } else {
      at[s] = (s * a.group + g) * VE;
    }
    if (at[s] >= vectors * VE) at[s] = -1;
  }
  auto pair_of = [&](int i) -> int {                          // i-th angle of this lane
    if constexpr (PAIRING == kApart) {
      return g < half / VE ? at[0] + i : -1;
    } else if constexpr (PAIRING == kInside) {
      const int c = at[2 * i / VE];
      return c < 0 || c + 2 * i % VE >= a.rd ? -1 : (c + 2 * i % VE) >> 1;
    } else {
      const int c = at[i / VE] < 0 ? a.rd : at[i / VE] + i % VE;
      return c >= a.rd ? -1 : a.neighbours ? c >> 1 : c < half ? c : c - half;
    }
  };

  const unsigned stride = gridDim.x * (kThreads / 32) * per_warp;
  unsigned unit0 = (blockIdx.x * (kThreads / 32) + warp) * per_warp;      // of the kind at hand
  // Kind by kind, so that a warp's heads are all of one kind and what belongs to the kind (weights, sums) is held once.
#pragma unroll 1
  for (int kind = 0; kind < 3; ++kind) {
  const bool turns = kind < 2;
  const unsigned units = a.tokens * (unsigned)a.chunks[kind];
  float w[KIND == kRope ? 1 : N];
  if constexpr (KIND != kRope) {
    const void* ws = kind == 0 ? a.wq : kind == 1 ? a.wk : nullptr;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int c = at[i / VE] < 0 ? -1 : at[i / VE] + i % VE;
      w[i] = 1.f;
      if (ws != nullptr && c >= 0)
        w[i] = a.wide_weights ? reinterpret_cast<const float*>(ws)[c] : to_f(reinterpret_cast<const T*>(ws)[c]);
    }
  }
  float sums[KIND == kNormBwd ? N : 1] = {};
  for (; unit0 < units; unit0 += stride) {
    // (every lane of the warp takes part in every step: a group without a unit works on none of its heads)
    const unsigned unit = unit0 + in_warp;
    const bool live = unit < units;
    const unsigned token = live ? unit / (unsigned)a.chunks[kind] : 0u;
    const int first = live ? (int)(unit - token * (unsigned)a.chunks[kind]) * a.chunk[kind] : 0;
    const int count = live ? min(a.chunk[kind], a.heads[kind] - first) : 0;
    const int head0 = first + (kind > 0 ? a.heads[0] : 0) + (kind > 1 ? a.heads[1] : 0);
    const int most = __reduce_max_sync(0xffffffffu, count);

    const T* x = reinterpret_cast<const T*>(a.x) + (long long)token * a.x_row + head0 * a.x_head;
    const T* dy = KIND == kNormBwd ? reinterpret_cast<const T*>(a.dy) + (long long)token * a.dy_row + head0 * a.dy_head
                                   : nullptr;
    T* out = reinterpret_cast<T*>(a.out) + (long long)token * a.out_row + head0 * a.out_head;

    // the first heads' data, before the angles are worked out
    Pack<T, VE> rx[U][NV], rd_[KIND == kNormBwd ? U : 1][NV];
    auto fetch = [&](int h) {
#pragma unroll
      for (int u = 0; u < U; ++u)
#pragma unroll
        for (int s = 0; s < NV; ++s) {
          if (h + u < count && at[s] >= 0) {
            if (KIND != kNormBwd || turns) rx[u][s] = load_pack<T, VE>(x + (h + u) * a.x_head + at[s]);
            if constexpr (KIND == kNormBwd) rd_[u][s] = load_pack<T, VE>(dy + (h + u) * a.dy_head + at[s]);
          } else {
            clear(rx[u][s]);
            if constexpr (KIND == kNormBwd) clear(rd_[u][s]);
          }
        }
    };
    fetch(0);

    float co[ANGLES], si[ANGLES];
    if (turns) {
      long long pos;
      if (a.positions == nullptr) pos = a.offset + token % a.seq;
      else if (a.wide_positions) pos = reinterpret_cast<const long long*>(a.positions)[token % a.seq];
      else pos = reinterpret_cast<const int*>(a.positions)[token % a.seq];
      const double place = (double)pos;
#pragma unroll
      for (int i = 0; i < ANGLES; ++i) {
        const int pair = pair_of(i);
        if (pair >= 0) {
          double t = place * a.turns[pair];
          t -= rint(t);
          sincospif(2.f * (float)t, &si[i], &co[i]);
          co[i] *= a.magnitude;
          si[i] *= a.magnitude * a.sign;
        }
      }
    }
    // the rotation of this lane's components of a head
    auto rotate = [&](float (&v)[N]) {
      if constexpr (PAIRING == kApart) {
        if (turns && g < half / VE) {
#pragma unroll
          for (int e = 0; e < VE; ++e) {
            const float p = v[e], q = v[VE + e];
            v[e] = p * co[e] - q * si[e];
            v[VE + e] = q * co[e] + p * si[e];
          }
        }
      } else if constexpr (PAIRING == kInside) {
#pragma unroll
        for (int i = 0; i < ANGLES; ++i) {
          if (turns && pair_of(i) >= 0) {
            const float p = v[2 * i], q = v[2 * i + 1];
            v[2 * i] = p * co[i] - q * si[i];
            v[2 * i + 1] = q * co[i] + p * si[i];
          }
        }
      } else {
        __syncwarp();
#pragma unroll
        for (int i = 0; i < N; ++i)
          if (at[i / VE] >= 0) exchange[at[i / VE] + i % VE] = v[i];
        __syncwarp();
#pragma unroll
        for (int i = 0; i < N; ++i) {
          const int c = at[i / VE] < 0 ? a.rd : at[i / VE] + i % VE;
          if (turns && c < a.rd) {
            const bool second = a.neighbours ? c & 1 : c >= half;
            const int other = a.neighbours ? c ^ 1 : second ? c - half : c + half;
            const float q = exchange[other];
            v[i] = second ? v[i] * co[i] + q * si[i] : v[i] * co[i] - q * si[i];
          }
        }
      }
    };

    for (int h = 0; h < most; h += U) {
      if (h > 0) fetch(h);
#pragma unroll
      for (int u = 0; u < U; ++u) {
        float v[N];
#pragma unroll
        for (int s = 0; s < NV; ++s) unpack(rx[u][s], v + s * VE);
        if constexpr (KIND == kRope) {
          rotate(v);
        } else if constexpr (KIND == kNormFwd) {
          float q = 0.f;
#pragma unroll
          for (int i = 0; i < N; ++i) q += v[i] * v[i];
          const float r = rsqrtf(group_sum(q, a.group) / (float)a.hd + a.eps);
          if (turns) {
#pragma unroll
            for (int i = 0; i < N; ++i) v[i] *= r * w[i];
          }
          rotate(v);
        } else {
          float d[N];
#pragma unroll
          for (int s = 0; s < NV; ++s) unpack(rd_[u][s], d + s * VE);
          rotate(d);                                          // (a.sign: backwards)
          float q = 0.f, dot = 0.f;
#pragma unroll
          for (int i = 0; i < N; ++i) { q += v[i] * v[i]; dot += d[i] * w[i] * v[i]; }
          q = group_sum(q, a.group);
          dot = group_sum(dot, a.group);
          const float r = rsqrtf(q / (float)a.hd + a.eps);
          const float mean = dot * r / (float)a.hd;           // of g w u
          if (turns) {
#pragma unroll
            for (int i = 0; i < N; ++i) {
              const float unit_x = v[i] * r;
              if (h + u < count) sums[i] += d[i] * unit_x;
              v[i] = r * (d[i] * w[i] - unit_x * mean);
            }
          } else {
#pragma unroll
            for (int i = 0; i < N; ++i) v[i] = d[i];
          }
        }
        if (h + u < count) {
#pragma unroll
          for (int s = 0; s < NV; ++s) {
            if (at[s] >= 0) store_pack<T, VE>(out + (h + u) * a.out_head + at[s], v + s * VE);
          }
        }
      }
    }
  }
  // the deal goes on where the last kind's ended (its units padded to whole warps, so that every group keeps its place)
  unit0 -= (units + per_warp - 1) / per_warp * per_warp;
  if constexpr (KIND == kNormBwd) {
    if (a.partial == nullptr || !turns) continue;
    // the lanes that hold the same components: over the warp by shuffles, over the warps in their order
    __syncthreads();
#pragma unroll
    for (int i = 0; i < N; ++i) {
      float v = sums[i];
      for (int o = a.group; o < 32; o <<= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
      if (in_warp == 0 && at[i / VE] >= 0) smem[warp * a.hd + at[i / VE] + i % VE] = v;
    }
    __syncthreads();
    for (int c = threadIdx.x; c < a.hd; c += kThreads) {
      float v = 0.f;
      for (int k = 0; k < kThreads / 32; ++k) v += smem[k * a.hd + c];
      a.partial[((size_t)blockIdx.x * 2 + kind) * a.hd + c] = v;
    }
    __syncthreads();
  }
  }
}

// dw[c] = sum over the CTAs of partial[cta][which][c], always in the same order: a warp per 32 columns of CTAs' rows, the
// eight warps of a block take every eighth row.
template <typename W>
__global__ void __launch_bounds__(256) heads_dw_kernel(const float* __restrict__ partial, int parts, int hd, W* __restrict__ dwq,
                                                       W* __restrict__ dwk, int accumulate) {
  __shared__ float red[8][33];
  const int lane = threadIdx.x & 31, row = threadIdx.x >> 5;
  const int c = blockIdx.x * 32 + lane;                       // of the two weights' 2 * hd
  float v = 0.f;
  if (c < 2 * hd) {
#pragma unroll 8
    for (int p = row; p < parts; p += 8) v += partial[(size_t)p * 2 * hd + c];
  }
  red[row][lane] = v;
  __syncthreads();
  if (row == 0 && c < 2 * hd) {
    v = 0.f;
    for (int k = 0; k < 8; ++k) v += red[k][lane];
    W* dst = c < hd ? dwq : dwk;
    if (dst != nullptr) {
      dst += c < hd ? c : c - hd;
      *dst = from_f<W>(accumulate ? to_f(*dst) + v : v);
    }
  }
}

// Heads per unit.  More of them share a lane's angles (some 40 instructions each, as many as a head's rotation of the same
// components), fewer give more units: as many as let every group of the grid have a few.
constexpr int kChunkHeads = 8;

template <typename T, int VE, int NV, int PAIRING, int KIND>
int launch(HeadArgs& a, int ctas, cudaStream_t stream) {
  const int groups = kThreads / a.group;
  size_t smem = PAIRING == kShared ? (size_t)groups * a.hd * sizeof(float) : 0;
  if (KIND == kNormBwd && a.partial != nullptr && smem < kThreads / 32 * a.hd * sizeof(float))
    smem = kThreads / 32 * a.hd * sizeof(float);
  heads_kernel<T, VE, NV, PAIRING, KIND><<<ctas, kThreads, smem, stream>>>(a);
  return (int)cudaGetLastError();
}

inline bool aligned(const void* p, long long row, long long head, int size) {
  return p == nullptr || (reinterpret_cast<uintptr_t>(p) % 16 == 0 && row * size % 16 == 0 && head * size % 16 == 0);
}

template <typename T, int KIND>
int dispatch(HeadArgs& a, int* parts, cudaStream_t stream) {
  constexpr int VE = 16 / sizeof(T);
  const int size = sizeof(T);
  // whole vectors need heads of whole vectors at 16-byte addresses and two vectors per lane of a warp; else one component
  // per access, in a warp per head
  const bool vectors = a.hd % VE == 0 && a.hd <= 64 * VE && aligned(a.x, a.x_row, a.x_head, size) &&
                       aligned(a.dy, a.dy_row, a.dy_head, size) && aligned(a.out, a.out_row, a.out_head, size);
  a.group = 32;
  if (vectors)
    for (a.group = 1; a.group * 2 * VE < a.hd; a.group *= 2) {}
  const long long groups = (long long)current_sm_count() * kCtasPerSm * (kThreads / a.group);
  int chunk = kChunkHeads;
  long long units;
  for (;; chunk /= 2) {
    units = 0;
    for (int k = 0; k < 3; ++k) {
      a.chunk[k] = a.heads[k] < chunk ? (a.heads[k] > 0 ? a.heads[k] : 1) : chunk;
      a.chunks[k] = (a.heads[k] + a.chunk[k] - 1) / a.chunk[k];
      units += (long long)a.tokens * a.chunks[k];
    }
    if (chunk == 1 || units >= 2 * groups) break;
  }
  if (units > 0x3fffffffLL) return DD_ERR_TOO_LARGE;
  const long long want = (units + kThreads / a.group - 1) / (kThreads / a.group);
  const int most = current_sm_count() * kCtasPerSm;
  const int ctas = (int)(want < most ? want : most);
  *parts = ctas;
  if (!vectors) return launch<T, 1, 16, kShared, KIND>(a, ctas, stream);
  if (a.neighbours) return launch<T, VE, 2, kInside, KIND>(a, ctas, stream);
  if (a.rd % (2 * VE) == 0) return launch<T, VE, 2, kApart, KIND>(a, ctas, stream);
  return launch<T, VE, 2, kShared, KIND>(a, ctas, stream);
}

template <int KIND>
int dispatch_type(HeadArgs& a, int dtype, int* parts, cudaStream_t stream) {
  if (dtype == 0) return dispatch<__nv_bfloat16, KIND>(a, parts, stream);
  if (dtype == 1) return dispatch<__half, KIND>(a, parts, stream);
  if (dtype == 2) return dispatch<float, KIND>(a, parts, stream);
  return DD_ERR_BAD_ARG;
}

int fill(HeadArgs& a, long long tokens, int hq, int hk, int rest, int hd, int rd, int neighbours, const double* turns,
         float magnitude, const void* positions, int wide_positions, long long offset, long long seq) {
  if (tokens < 0 || hq < 0 || hk < 0 || rest < 0 || hd < 1 || rd < 0 || rd > hd || rd % 2 != 0) return DD_ERR_BAD_ARG;
  if (rd > 0 && turns == nullptr) return DD_ERR_BAD_ARG;
  if (rd > 0 && seq < 1) return DD_ERR_BAD_ARG;
  if (hd > 2 * kMaxPairs || tokens > 0x3fffffffLL) return DD_ERR_TOO_LARGE;
  a.tokens = (unsigned)tokens;
  a.seq = seq < 1 ? 1u : seq > 0x3fffffffLL ? 0x3fffffffu : (unsigned)seq;
  a.heads[0] = hq; a.heads[1] = hk; a.heads[2] = rest;
  a.hd = hd; a.rd = rd; a.neighbours = neighbours;
  a.positions = positions; a.wide_positions = wide_positions; a.offset = offset;
  a.magnitude = magnitude;
  for (int i = 0; i < rd / 2; ++i) a.turns[i] = turns[i];
  return DD_OK;
}

}  // namespace

// CTAs (and rows of the backward pass's scratch) at most.
DD_API int dd_heads_parts() { return current_sm_count() * kCtasPerSm; }

// out = x with the leading `nheads` of `heads` heads rotated (sign -1: backwards); with out == x the other heads are left
// alone, else they are copied.  Tensors [tokens, heads, hd] by token and head stride in elements; dtype 0 bf16, 1 fp16,
// 2 fp32; turns[rd / 2]: frequencies in turns per position (host memory); positions [seq] on the device (4 or 8 bytes
// each) of token % seq, or null for offset + token % seq.
DD_API int dd_rotate_heads(const void* x, long long x_row, long long x_head, void* out, long long out_row, long long out_head,
                           long long tokens, int heads, int nheads, int hd, int rd, int neighbours, const double* turns,
                           float magnitude, float sign, const void* positions, int wide_positions, long long offset,
                           long long seq, int dtype, void* stream) {
  HeadArgs a = {};
  if (nheads > heads) return DD_ERR_BAD_ARG;
  const int r = fill(a, tokens, nheads, 0, x == out ? 0 : heads - nheads, hd, rd, neighbours, turns, magnitude, positions,
                     wide_positions, offset, seq);
  if (r) return r;
  if (tokens == 0 || a.heads[0] + a.heads[2] == 0) return DD_OK;
  if (x == nullptr || out == nullptr) return DD_ERR_BAD_ARG;
  a.x = x; a.x_row = x_row; a.x_head = x_head;
  a.out = out; a.out_row = out_row; a.out_head = out_head;
  a.sign = sign;
  int parts = 0;
  return dispatch_type<kRope>(a, dtype, &parts, reinterpret_cast<cudaStream_t>(stream));
}

// out = the first hq heads of x normed with weight wq and rotated, the next hk with wk, the `rest` behind them copied (left
// alone with out == x).  Weights [hd] of x's type, or fp32 with wide_weights, or null.
DD_API int dd_norm_heads_fwd(const void* x, long long x_row, long long x_head, void* out, long long out_row, long long out_head,
                             const void* wq, const void* wk, int wide_weights, float eps, long long tokens, int hq, int hk,
                             int rest, int hd, int rd, int neighbours, const double* turns, float magnitude,
                             const void* positions, int wide_positions, long long offset, long long seq, int dtype,
                             void* stream) {
  HeadArgs a = {};
  const int r = fill(a, tokens, hq, hk, x == out ? 0 : rest, hd, rd, neighbours, turns, magnitude, positions, wide_positions,
                     offset, seq);
  if (r) return r;
  if (tokens == 0 || a.heads[0] + a.heads[1] + a.heads[2] == 0) return DD_OK;
  if (x == nullptr || out == nullptr) return DD_ERR_BAD_ARG;
  a.x = x; a.x_row = x_row; a.x_head = x_head;
  a.out = out; a.out_row = out_row; a.out_head = out_head;
  a.wq = wq; a.wk = wk; a.wide_weights = wide_weights; a.eps = eps;
  a.sign = 1.f;
  int parts = 0;
  return dispatch_type<kNormFwd>(a, dtype, &parts, reinterpret_cast<cudaStream_t>(stream));
}

// Its gradients: dx [tokens, hq + hk + rest, hd] by strides, dwq / dwk [hd] (null: not wanted) of the weights' type, or with
// accumulate added to what is there, fp32.  partial: dd_heads_parts() * 2 * hd floats of scratch, null if neither is wanted.
DD_API int dd_norm_heads_bwd(const void* x, long long x_row, long long x_head, const void* dy, long long dy_row,
                             long long dy_head, void* dx, long long dx_row, long long dx_head, const void* wq, const void* wk,
                             int wide_weights, float eps, void* dwq, void* dwk, int accumulate, float* partial,
                             long long tokens, int hq, int hk, int rest, int hd, int rd, int neighbours, const double* turns,
                             float magnitude, const void* positions, int wide_positions, long long offset, long long seq,
                             int dtype, void* stream) {
  HeadArgs a = {};
  const int r = fill(a, tokens, hq, hk, rest, hd, rd, neighbours, turns, magnitude, positions, wide_positions, offset, seq);
  if (r) return r;
  if ((dwq != nullptr || dwk != nullptr) && partial == nullptr) return DD_ERR_BAD_ARG;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  int parts = 0;
  if (tokens > 0 && hq + hk + rest > 0) {
    if (x == nullptr || dy == nullptr || dx == nullptr) return DD_ERR_BAD_ARG;
    a.x = x; a.x_row = x_row; a.x_head = x_head;
    a.dy = dy; a.dy_row = dy_row; a.dy_head = dy_head;
    a.out = dx; a.out_row = dx_row; a.out_head = dx_head;
    a.wq = wq; a.wk = wk; a.wide_weights = wide_weights; a.eps = eps;
    a.partial = dwq != nullptr || dwk != nullptr ? partial : nullptr;
    a.sign = -1.f;
    const int e = dispatch_type<kNormBwd>(a, dtype, &parts, st);
    if (e) return e;
  }
  if (dwq == nullptr && dwk == nullptr) return DD_OK;
  const int grid = (2 * hd + 31) / 32;                        // (no tokens: parts = 0, zeros)
  if (accumulate || wide_weights || dtype == 2)
    heads_dw_kernel<float><<<grid, 256, 0, st>>>(partial, parts, hd, (float*)dwq, (float*)dwk, accumulate);
  else if (dtype == 1)
    heads_dw_kernel<__half><<<grid, 256, 0, st>>>(partial, parts, hd, (__half*)dwq, (__half*)dwk, 0);
  else
    heads_dw_kernel<__nv_bfloat16><<<grid, 256, 0, st>>>(partial, parts, hd, (__nv_bfloat16*)dwq, (__nv_bfloat16*)dwk, 0);
  return (int)cudaGetLastError();
}
