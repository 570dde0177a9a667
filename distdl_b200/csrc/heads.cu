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
//    component of a pair also holds the other (the vectors lie half the rotated part apart, or the pairs lie inside a vector; where
//    that half is not whole vectors, the others come from their lanes through shared memory);
//  * the angles are computed, not read: position times frequency in turns in 64 bits, reduced to half a turn (within 10^-6
//    radians for every position below 2^31, where 32 bits are off by whole turns), then sin and cos in 32 bits, once per lane for
//    all heads of a chunk.  The frequencies travel as arguments of the kernel: no table, no copy, nothing to capture or to keep;
//  * the backward pass recomputes r from x, which it needs anyway.
// A unit of work is a token's chunk of heads of one kind (query / key / rest).  Units are dealt to the warps of a grid of two
// CTAs per SM, kind by kind, so that what belongs to a kind is held once; the heads of a unit to the groups of the warp in turn,
// so that a warp reads and writes them as they lie in memory (a group with 16 heads for itself, its neighbours with the next
// token's, 16384 tokens, 48 heads of 128 bf16: rotation 68.4 us, backward 107.9; with four heads 64.6 and 102.5).
#include "common.cuh"
#include "runtime.cuh"

#include <cuda_fp16.h>

#include <cstring>
#include <type_traits>

using namespace dd;

namespace {

constexpr int kThreads = 256;
constexpr int kMaxPairs = 256;        // heads of up to 512 components
constexpr int kCtasPerSm = 2;         // (128 registers a thread: heads side by side count for more than further warps)

enum Kind { kRope = 0, kNorm = 1 };
// Where a lane finds the two components of a pair.
enum Pairing {
  kApart = 0,     // halves that are whole vectors: at the same place of its two vectors
  kInside = 1,    // next to one another in a vector; with single components, any pair of components that it holds
  kCrossed = 2,   // halves that are not whole vectors: one in its vectors, the other in another lane's, by way of shared memory
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
  const void* positions;      // [seq] of 4 or 8 bytes, of token % seq, or null: offset + token % seq, from the place
                              // `split` on offset_behind + token % seq (a sequence of two ranges of positions)
  float* partial;             // backward: [gridDim.x][2][hd], or null
  long long offset;
  unsigned tokens, seq;
  int heads[3];               // query, key and other heads (those are copied; none in place)
  int chunk[3], chunks[3];    // heads per unit (whole rounds of a warp's groups), units per token
  int hd, rd, group;          // group: lanes per head (a power of two)
  int queries;                // forward: of the heads of the first kind, those that take wq
  int wide_positions, wide_weights, neighbours;
  float magnitude, sign, eps, inv_hd;
  unsigned split;             // (behind the others: between them kCrossed spills more in the backward pass:
                              // 16384 tokens, 48 heads, 50 of 128 turned, forward and backward 271 -> 284 us)
  long long offset_behind;
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
__device__ __forceinline__ uint64_t two(uint32_t u, __nv_bfloat16) { return pack_u32x2(u << 16, u & 0xffff0000u); }
__device__ __forceinline__ uint64_t two(uint32_t u, __half) {
  const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&u));
  return pack_f32x2(f.x, f.y);
}
__device__ __forceinline__ uint32_t word(uint64_t v, __nv_bfloat16) {
  const float2 f = unpack_f32x2(v);
  return pack_bf16x2(f.x, f.y);
}
__device__ __forceinline__ uint32_t word(uint64_t v, __half) {
  const float2 f = unpack_f32x2(v);
  const __half2 h = __floats2half2_rn(f.x, f.y);
  return *reinterpret_cast<const uint32_t*>(&h);
}
// NV packs as pairs of fp32 values, one instruction for both (single components pair up as they come).
template <typename T, int VE, int NV>
__device__ __forceinline__ void unpack(const Pack<T, VE> (&r)[NV], uint64_t (&f)[NV * VE / 2]) {
  if constexpr (VE == 1) {
#pragma unroll
    for (int i = 0; i < NV / 2; ++i) f[i] = pack_f32x2(to_f(r[2 * i].v), to_f(r[2 * i + 1].v));
  } else {
#pragma unroll
    for (int s = 0; s < NV; ++s) {
      uint64_t* g = f + s * VE / 2;
      if constexpr (VE == 4) {
        g[0] = pack_u32x2(r[s].v.x, r[s].v.y); g[1] = pack_u32x2(r[s].v.z, r[s].v.w);
      } else {
        g[0] = two(r[s].v.x, T()); g[1] = two(r[s].v.y, T()); g[2] = two(r[s].v.z, T()); g[3] = two(r[s].v.w, T());
      }
    }
  }
}
template <typename T, int VE, int NV>
__device__ __forceinline__ void pack(const uint64_t (&f)[NV * VE / 2], Pack<T, VE> (&r)[NV]) {
  if constexpr (VE == 1) {
#pragma unroll
    for (int i = 0; i < NV / 2; ++i) {
      const float2 g = unpack_f32x2(f[i]);
      r[2 * i].v = from_f<T>(g.x); r[2 * i + 1].v = from_f<T>(g.y);
    }
  } else {
#pragma unroll
    for (int s = 0; s < NV; ++s) {
      const uint64_t* g = f + s * VE / 2;
      if constexpr (VE == 4) {
        const float2 a = unpack_f32x2(g[0]), b = unpack_f32x2(g[1]);
        r[s].v = make_uint4(__float_as_uint(a.x), __float_as_uint(a.y), __float_as_uint(b.x), __float_as_uint(b.y));
      } else {
        r[s].v = make_uint4(word(g[0], T()), word(g[1], T()), word(g[2], T()), word(g[3], T()));
      }
    }
  }
}
template <typename T, int VE>
__device__ __forceinline__ void store_pack(T* p, const Pack<T, VE>& r) {
  if constexpr (VE == 1) *p = r.v;
  else *reinterpret_cast<uint4*>(p) = r.v;
}

// Sine and cosine of 2 pi t, |t| <= 1/2.  For 16-bit heads the fast functions: 2^-21 off at most, a hundredth of a rounding
// step of the result, and the accurate ones are a fifth of the instructions of a pass.
template <typename T>
__device__ __forceinline__ void sin_cos_turns(float t, float* s, float* c) {
  if constexpr (sizeof(T) == 2) {
    *s = __sinf(6.283185307179586f * t);
    *c = __cosf(6.283185307179586f * t);
  } else {
    sincospif(2.f * t, s, c);
  }
}

// Sums over the lanes of a group, two side by side.  GROUP: lanes of a group, 0: `group` of them (a power of two).
template <int GROUP>
__device__ __forceinline__ void group_sums(float& v, float& u, int group) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1)
    if ((GROUP > 0 ? GROUP : group) > o) {
      v += __shfl_xor_sync(0xffffffffu, v, o);
      u += __shfl_xor_sync(0xffffffffu, u, o);
    }
}
template <int GROUP>
__device__ __forceinline__ float group_sum(float v, int group) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1)
    if ((GROUP > 0 ? GROUP : group) > o) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// What a lane of a group holds of a head: NV vectors of VE components.  GROUP: lanes of a group that all have their vectors; 0:
// a.group lanes, some of them without.
template <typename T, int VE, int NV, int PAIRING, int GROUP>
struct Lane {
  static constexpr int N = NV * VE, M = N / 2;                // components, pairs of them as they are computed with
  int at[NV];                                                 // first component of each vector, -1: none
  int half;                                                   // pairs of a head
  int first_pair, paired;                                     // kApart: of this lane's components, and whether they turn

  __device__ __forceinline__ Lane(const HeadArgs& a, int g) : half(a.rd >> 1) {
    paired = g < half / VE;
    first_pair = g * VE;
#pragma unroll
    for (int s = 0; s < NV; ++s) {
      if constexpr (PAIRING == kApart) {
        const int lanes = half / VE;                          // that hold a vector of each half; the others, what stays
        at[s] = (paired ? g + s * lanes : 2 * lanes + 2 * (g - lanes) + s) * VE;
      } else if constexpr (VE > 1) {
        at[s] = (s * (GROUP > 0 ? GROUP : a.group) + g) * VE;
      } else {
        const int pair = (s / 2) * a.group + g;
        at[s] = pair >= half ? 2 * pair + s % 2 : a.neighbours ? 2 * pair + s % 2 : pair + s % 2 * half;
      }
      if (GROUP == 0 && at[s] + VE > a.hd) at[s] = -1;
    }
  }
  __device__ __forceinline__ bool has(int s) const { return GROUP > 0 || at[s] >= 0; }
  __device__ __forceinline__ int component(int i) const { return has(i / VE) ? at[i / VE] + i % VE : -1; }
  // kInside: the pair of components (2 i, 2 i + 1) of this lane, -1 where they stay
  __device__ __forceinline__ int pair(const HeadArgs& a, int g, int i) const {
    if constexpr (VE > 1) {
      const int c = component(2 * i);
      return c >= 0 && c < a.rd ? c >> 1 : -1;
    } else {
      const int p = i * a.group + g;
      return p < half ? p : -1;
    }
  }
};

// kCrossed: a warp's heads in shared memory, as they came, and where a lane finds the partners of its components there: byte
// offsets, two to a word; for components that stay that of a zero.  Heads are a word more than their length apart, for the banks.
constexpr int kCrossing = 32 * 2 * 4 + 32;                    // words of a warp; then the zero
template <typename T, int VE, int NV, int PAIRING, int GROUP>
struct Partners {
  using L = Lane<T, VE, NV, PAIRING, GROUP>;
  static constexpr int M = PAIRING == kCrossed ? L::M : 1;
  uint32_t from[M];
  uint32_t *warp, *own;                                       // the warp's heads, and this lane's

  __device__ __forceinline__ Partners(const HeadArgs& a, const L& lane, int in_warp, uint32_t* words) : warp(words) {
    if constexpr (PAIRING == kCrossed) {
      static_assert(NV == 2 && VE * sizeof(T) == 16, "kCrossing");
      const int start = in_warp * (a.hd * (int)sizeof(T) / 4 + 1);
      own = words + start;
      auto of = [&](int c) {
        if (c < 0 || c >= a.rd) return kCrossing * 4;
        return start * 4 + (c < lane.half ? c + lane.half : c - lane.half) * (int)sizeof(T);
      };
#pragma unroll
      for (int i = 0; i < M; ++i) from[i] = (uint32_t)of(lane.component(2 * i)) | (uint32_t)of(lane.component(2 * i + 1)) << 16;
    }
  }
  // u: the partners of r
  __device__ __forceinline__ void cross(const L& lane, const Pack<T, VE> (&r)[NV], uint64_t (&u)[L::M]) const {
    if constexpr (PAIRING == kCrossed) {
      __syncwarp();                                           // (the head before has been read)
#pragma unroll
      for (int s = 0; s < NV; ++s)
        if (lane.has(s)) {
          uint32_t* to = own + lane.at[s] * (int)sizeof(T) / 4;
          to[0] = r[s].v.x; to[1] = r[s].v.y; to[2] = r[s].v.z; to[3] = r[s].v.w;
        }
      __syncwarp();
      const uint8_t* base = reinterpret_cast<const uint8_t*>(warp);
#pragma unroll
      for (int i = 0; i < M; ++i)
        u[i] = pack_f32x2(to_f(*reinterpret_cast<const T*>(base + (from[i] & 0xffffu))),
                          to_f(*reinterpret_cast<const T*>(base + (from[i] >> 16))));
    }
  }
};

// Sine and cosine of a lane's pairs at a token's position, and the rotation of what it holds of a head by them.
template <typename T, int VE, int NV, int PAIRING, int GROUP>
struct Angles {
  using L = Lane<T, VE, NV, PAIRING, GROUP>;
  static constexpr int M = L::M, A = PAIRING == kApart ? M / 2 : PAIRING == kCrossed ? M : 1, I = PAIRING == kInside ? M : 1;
  // of two pairs (kApart; n2: the sines negated) or two components (kCrossed; s2 with the sign that they take their partner with)
  uint64_t c2[A], s2[A], n2[A];
  float c1[I], s1[I];                                         // kInside

  __device__ __forceinline__ void set(const HeadArgs& a, const double* turns, const L& lane, int g, unsigned token) {
    long long pos;
    const unsigned at = token % a.seq;
    if (a.positions == nullptr) pos = (at < a.split ? a.offset : a.offset_behind) + at;
    else if (a.wide_positions) pos = reinterpret_cast<const long long*>(a.positions)[at];
    else pos = reinterpret_cast<const int*>(a.positions)[at];
    const double place = (double)pos;
    auto angle = [&](int pair, float* c, float* s) {
      double t = place * turns[pair];
      t -= rint(t);
      sin_cos_turns<T>((float)t, s, c);
      *c *= a.magnitude;
      *s *= a.magnitude * a.sign;
    };
    if constexpr (PAIRING == kApart) {
#pragma unroll
      for (int i = 0; i < A; ++i) {
        float c[2] = {1.f, 1.f}, s[2] = {0.f, 0.f};
        if (lane.paired) {
          angle(lane.first_pair + 2 * i, &c[0], &s[0]);
          angle(lane.first_pair + 2 * i + 1, &c[1], &s[1]);
        }
        c2[i] = pack_f32x2(c[0], c[1]);
        s2[i] = pack_f32x2(s[0], s[1]);
        n2[i] = pack_f32x2(-s[0], -s[1]);
      }
    } else if constexpr (PAIRING == kCrossed) {
#pragma unroll
      for (int i = 0; i < A; ++i) {
        float c[2] = {1.f, 1.f}, s[2] = {0.f, 0.f};
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int at = lane.component(2 * i + e);
          if (at >= 0 && at < a.rd) {
            angle(at < lane.half ? at : at - lane.half, &c[e], &s[e]);
            if (at < lane.half) s[e] = -s[e];
          }
        }
        c2[i] = pack_f32x2(c[0], c[1]);
        s2[i] = pack_f32x2(s[0], s[1]);
      }
    } else {
#pragma unroll
      for (int i = 0; i < I; ++i) {
        const int p = lane.pair(a, g, i);
        if (p >= 0) angle(p, &c1[i], &s1[i]);
      }
    }
  }
  // u: the partners (kCrossed)
  __device__ __forceinline__ void rotate(const HeadArgs& a, const L& lane, int g, uint64_t (&v)[M], const uint64_t (&u)[M]) const {
    if constexpr (PAIRING == kCrossed) {
#pragma unroll
      for (int i = 0; i < A; ++i) v[i] = fma_f32x2(v[i], c2[i], mul_f32x2(u[i], s2[i]));
    } else if constexpr (PAIRING == kApart) {
      if (lane.paired) {
#pragma unroll
        for (int i = 0; i < A; ++i) {
          const uint64_t p = v[i], q = v[A + i];
          v[i] = fma_f32x2(p, c2[i], mul_f32x2(q, n2[i]));
          v[A + i] = fma_f32x2(q, c2[i], mul_f32x2(p, s2[i]));
        }
      }
    } else {
#pragma unroll
      for (int i = 0; i < I; ++i) {
        if (lane.pair(a, g, i) >= 0) {
          const float2 p = unpack_f32x2(v[i]);
          v[i] = pack_f32x2(p.x * c1[i] - p.y * s1[i], p.y * c1[i] + p.x * s1[i]);
        }
      }
    }
  }
};

template <int M>
__device__ __forceinline__ float dot(const uint64_t (&v)[M], const uint64_t (&u)[M]) {
  uint64_t sum[2] = {0, 0};
#pragma unroll
  for (int i = 0; i < M; ++i) sum[i & 1] = fma_f32x2(v[i], u[i], sum[i & 1]);
  const float2 f = unpack_f32x2(add_f32x2(sum[0], sum[1]));
  return f.x + f.y;
}

template <typename T>
__device__ __forceinline__ float weight_of(const HeadArgs& a, int kind, int c) {
  const void* w = kind == 0 ? a.wq : a.wk;
  if (w == nullptr || c < 0) return 1.f;
  return a.wide_weights ? reinterpret_cast<const float*>(w)[c] : to_f(reinterpret_cast<const T*>(w)[c]);
}

// The weights of a lane's components, from shared memory.
template <int VE, int NV, typename L>
__device__ __forceinline__ void weights_of(const float* weights, const L& lane, uint64_t (&w)[NV * VE / 2]) {
  if constexpr (VE > 1) {
#pragma unroll
    for (int i = 0; i < NV * VE / 2; i += 2) {
      const float4 f = *reinterpret_cast<const float4*>(&weights[lane.has(2 * i / VE) ? lane.at[2 * i / VE] + 2 * i % VE : 0]);
      w[i] = pack_f32x2(f.x, f.y);
      w[i + 1] = pack_f32x2(f.z, f.w);
    }
  } else {
#pragma unroll
    for (int i = 0; i < NV / 2; ++i)
      w[i] = pack_f32x2(weights[max(lane.at[2 * i], 0)], weights[max(lane.at[2 * i + 1], 0)]);
  }
}

// A unit of work of a warp: of its heads the group `in_warp` has every per_warp-th, from `head` on, `count` of them.
struct Unit {
  unsigned token;
  int head, count;
  __device__ __forceinline__ Unit(const HeadArgs& a, int kind, unsigned unit, int in_warp, int per_warp) {
    token = unit / (unsigned)a.chunks[kind];
    const int first = (int)(unit - token * (unsigned)a.chunks[kind]) * a.chunk[kind] + in_warp;
    const int end = min(first - in_warp + a.chunk[kind], a.heads[kind]);
    count = first < end ? (end - first + per_warp - 1) / per_warp : 0;
    head = first + (kind > 0 ? a.heads[0] : 0) + (kind > 1 ? a.heads[1] : 0);
  }
};

// The heads behind queries and keys, copied (forward: of x, backward: of dy).
template <typename T, int VE, int NV, typename L>
__device__ __forceinline__ void copy_rest(const HeadArgs& a, const L& lane, const void* from, long long row, long long head,
                                          unsigned unit, unsigned stride, int in_warp, int per_warp) {
  const unsigned units = a.tokens * (unsigned)a.chunks[2];
  const long long step = head * per_warp, out_step = a.out_head * per_warp;
  for (; unit < units; unit += stride) {
    const Unit u(a, 2, unit, in_warp, per_warp);
    const T* src = reinterpret_cast<const T*>(from) + (long long)u.token * row + u.head * head;
    T* out = reinterpret_cast<T*>(a.out) + (long long)u.token * a.out_row + u.head * a.out_head;
    constexpr int R = VE > 1 ? 4 : 2;
    for (int h = 0; h < u.count; h += R) {
      Pack<T, VE> r[R][NV];
#pragma unroll
      for (int k = 0; k < R; ++k)
#pragma unroll
        for (int s = 0; s < NV; ++s)
          if (h + k < u.count && lane.has(s)) r[k][s] = load_pack<T, VE>(src + (h + k) * step + lane.at[s]);
#pragma unroll
      for (int k = 0; k < R; ++k)
#pragma unroll
        for (int s = 0; s < NV; ++s)
          if (h + k < u.count && lane.has(s)) store_pack<T, VE>(out + (h + k) * out_step + lane.at[s], r[k][s]);
    }
  }
}

// Forward.  Four heads' loads are in flight together and four heads are worked on side by side: that hides more than a
// third or fourth CTA per SM or loads a step ahead would (16384 tokens, 48 heads of 128 bf16, us, rotation / norm and rotation:
// two heads and 4 / 3 CTAs 80.7 / 87.4, two and the next two on their way 75.5 / 72.3, four 64.7 / 67.6; with partners from other
// lanes two 77.1 / 95.7, four 71.5 / 105.5, which spill with the norm: two there).  Query and key heads
// are one kind here, which share their angles; their weights are in shared memory.
template <typename T, int VE, int NV, int PAIRING, int KIND, int GROUP>
__global__ void __launch_bounds__(kThreads, kCtasPerSm) heads_fwd_kernel(const __grid_constant__ HeadArgs a) {
  using L = Lane<T, VE, NV, PAIRING, GROUP>;
  constexpr bool CROSSED = PAIRING == kCrossed;
  constexpr int M = L::M, U = CROSSED && KIND == kNorm ? 2 : VE > 1 ? 4 : 1;
  __shared__ double turns[kMaxPairs];
  __shared__ __align__(16) float weights[KIND == kNorm ? 2 : 1][KIND == kNorm ? 2 * kMaxPairs : 4];
  // kCrossed: the weights of the components' partners
  __shared__ __align__(16) float opposite[CROSSED && KIND == kNorm ? 2 : 1][CROSSED && KIND == kNorm ? 2 * kMaxPairs : 4];
  __shared__ uint32_t crossing[CROSSED ? kThreads / 32 : 1][CROSSED ? kCrossing + 1 : 1];
  grid_dependency_launch();
  for (int i = threadIdx.x; i < a.rd / 2; i += kThreads) turns[i] = a.turns[i];
  if constexpr (KIND == kNorm) {
    for (int c = threadIdx.x; c < 2 * a.hd; c += kThreads)
      weights[c >= a.hd][c >= a.hd ? c - a.hd : c] = weight_of<T>(a, c >= a.hd, c >= a.hd ? c - a.hd : c);
    if constexpr (CROSSED) {
      for (int i = threadIdx.x; i < 2 * a.hd; i += kThreads) {
        const int which = i >= a.hd, c = which ? i - a.hd : i, half = a.rd / 2;
        opposite[which][c] = weight_of<T>(a, which, c < half ? c + half : c < a.rd ? c - half : c);
      }
    }
  }
  if (CROSSED && threadIdx.x < kThreads / 32) crossing[threadIdx.x][kCrossing] = 0u;
  __syncthreads();
  const int group = GROUP > 0 ? GROUP : a.group;
  const int warp = threadIdx.x >> 5, g = threadIdx.x & (group - 1);
  const int per_warp = 32 / group, in_warp = (threadIdx.x & 31) / group;
  const L lane(a, g);
  const Partners<T, VE, NV, PAIRING, GROUP> partners(a, lane, in_warp, crossing[CROSSED ? warp : 0]);
  const unsigned stride = gridDim.x * (kThreads / 32), units = a.tokens * (unsigned)a.chunks[0];
  const long long x_step = a.x_head * per_warp, out_step = a.out_head * per_warp;
  unsigned unit = blockIdx.x * (kThreads / 32) + warp;
  for (; unit < units; unit += stride) {
    // (every lane of the warp takes part in every step: a group whose heads have ended works on none)
    const Unit u(a, 0, unit, in_warp, per_warp);
    const int most = __shfl_sync(0xffffffffu, u.count, 0);    // (no group has more than the first)
    const T* x = reinterpret_cast<const T*>(a.x) + (long long)u.token * a.x_row + u.head * a.x_head;
    T* out = reinterpret_cast<T*>(a.out) + (long long)u.token * a.out_row + u.head * a.out_head;
    Pack<T, VE> raw[U][NV];
    auto fetch = [&](int h, auto heads) {
#pragma unroll
      for (int k = 0; k < heads(); ++k) {
#pragma unroll
        for (int s = 0; s < NV; ++s) {
          if (h + k < u.count && lane.has(s)) raw[k][s] = load_pack<T, VE>(x + lane.at[s]);
          else clear(raw[k][s]);
        }
        x += x_step;
      }
    };
    Angles<T, VE, NV, PAIRING, GROUP> angles;
    auto work = [&](int h, auto heads) {
#pragma unroll
      for (int k = 0; k < heads(); ++k) {
        uint64_t v[M], other[M];
        unpack<T, VE, NV>(raw[k], v);
        partners.cross(lane, raw[k], other);
        if constexpr (KIND == kNorm) {
          const float r = rsqrtf(group_sum<GROUP>(dot(v, v), a.group) * a.inv_hd + a.eps);
          const uint64_t r2 = pack_f32x2(r, r);
          const int which = u.head + (h + k) * per_warp >= a.queries;
          uint64_t w[M];
          weights_of<VE, NV>(weights[which], lane, w);
#pragma unroll
          for (int i = 0; i < M; ++i) v[i] = mul_f32x2(v[i], mul_f32x2(r2, w[i]));
          if constexpr (CROSSED) {
            weights_of<VE, NV>(opposite[which], lane, w);
#pragma unroll
            for (int i = 0; i < M; ++i) other[i] = mul_f32x2(other[i], mul_f32x2(r2, w[i]));
          }
        }
        angles.rotate(a, lane, g, v, other);
        if (h + k < u.count) {
          Pack<T, VE> res[NV];
          pack<T, VE, NV>(v, res);
#pragma unroll
          for (int s = 0; s < NV; ++s)
            if (lane.has(s)) store_pack<T, VE>(out + lane.at[s], res[s]);
        }
        out += out_step;
      }
    };
    // U heads at a time, the last ones of a unit (few tokens: its only one) in twos and singly
    const std::integral_constant<int, U> many;
    const std::integral_constant<int, (U > 1 ? 2 : 1)> two;
    const std::integral_constant<int, 1> one;
    int h = 0;
    if (most >= U) fetch(0, many);
    else if (most >= 2) fetch(0, two);
    else fetch(0, one);
    angles.set(a, turns, lane, g, u.token);                   // while the first heads are on their way
    for (; h + U <= most; h += U) {
      if (h > 0) fetch(h, many);
      work(h, many);
    }
    if (U > 2 && h + 2 <= most) {
      if (h > 0) fetch(h, two);
      work(h, two);
      h += 2;
    }
    if (h < most) {
      if (h > 0) fetch(h, one);
      work(h, one);
    }
  }
  copy_rest<T, VE, NV>(a, lane, a.x, a.x_row, a.x_head, unit - units, stride, in_warp, per_warp);
}

// 16 bytes global -> shared by a copy of this thread's own.
__device__ __forceinline__ void copy_async(void* to, const void* from) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem_u32(to)), "l"(from) : "memory");
}
__device__ __forceinline__ void copy_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int LEFT> __device__ __forceinline__ void copy_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(LEFT) : "memory"); }

constexpr int kBwdSteps = 4;                                  // heads in the ring
constexpr int kBwdRing = kBwdSteps * 4 * 16 * kThreads;

// Backward.  x and dy come through a ring in shared memory that every thread fills and reads for itself, three heads ahead
// and across the units' ends, and w stays there: the registers are needed for the sums of dw and a head's values (16384
// tokens, 48 heads of 128 bf16, us: loads into registers a head ahead 138, with w in shared memory 128, the ring 109, with two
// heads side by side, which spill, 149).
template <typename T, int VE, int NV, int PAIRING, int GROUP>
__global__ void __launch_bounds__(kThreads, kCtasPerSm) heads_bwd_kernel(const __grid_constant__ HeadArgs a) {
  using L = Lane<T, VE, NV, PAIRING, GROUP>;
  constexpr int N = L::N, M = L::M;
  constexpr bool RING = VE > 1;
  constexpr int R = RING ? kBwdSteps : 1;
  constexpr bool CROSSED = PAIRING == kCrossed;
  extern __shared__ __align__(16) uint8_t ring[];             // [R][2 NV][kThreads] vectors
  __shared__ double turns[kMaxPairs];
  __shared__ __align__(16) float weights[2 * kMaxPairs];
  __shared__ float reduced[kThreads / 32][2 * kMaxPairs];
  __shared__ uint32_t crossing[CROSSED ? kThreads / 32 : 1][CROSSED ? kCrossing + 1 : 1];
  grid_dependency_launch();
  for (int i = threadIdx.x; i < a.rd / 2; i += kThreads) turns[i] = a.turns[i];
  if (CROSSED && threadIdx.x < kThreads / 32) crossing[threadIdx.x][kCrossing] = 0u;
  const int group = GROUP > 0 ? GROUP : a.group;
  const int warp = threadIdx.x >> 5, g = threadIdx.x & (group - 1);
  const int per_warp = 32 / group, in_warp = (threadIdx.x & 31) / group;
  const L lane(a, g);
  const Partners<T, VE, NV, PAIRING, GROUP> partners(a, lane, in_warp, crossing[CROSSED ? warp : 0]);
  const unsigned stride = gridDim.x * (kThreads / 32);
  unsigned unit = blockIdx.x * (kThreads / 32) + warp;        // of the kind at hand
#pragma unroll 1
  for (int kind = 0; kind < 2; ++kind) {
    const unsigned units = a.tokens * (unsigned)a.chunks[kind];
    const int rounds = a.chunk[kind] / per_warp;              // of a unit, the same for all of them
    const long long x_step = a.x_head * per_warp, dy_step = a.dy_head * per_warp, out_step = a.out_head * per_warp;
    for (int c = threadIdx.x; c < a.hd; c += kThreads) weights[c] = weight_of<T>(a, kind, c);
    __syncthreads();
    uint64_t sums[M] = {};

    Pack<T, VE> rx[NV], rd[NV];
    // the copies' place in the units, ahead of the work's
    unsigned ahead = unit;
    int ahead_h = 0, ahead_count = 0;
    const T* x = nullptr;
    const T* dy = nullptr;
    auto fetch = [&](int slot) {
      if (ahead < units) {
        if (ahead_h == 0) {
          const Unit u(a, kind, ahead, in_warp, per_warp);
          ahead_count = u.count;
          x = reinterpret_cast<const T*>(a.x) + (long long)u.token * a.x_row + u.head * a.x_head;
          dy = reinterpret_cast<const T*>(a.dy) + (long long)u.token * a.dy_row + u.head * a.dy_head;
        }
#pragma unroll
        for (int s = 0; s < NV; ++s) {
          const bool read = ahead_h < ahead_count && lane.has(s);
          if constexpr (RING) {
            uint8_t* to = ring + ((slot * 2 * NV + s) * kThreads + threadIdx.x) * 16;
            if (read) {
              copy_async(to, x + lane.at[s]);
              copy_async(to + NV * kThreads * 16, dy + lane.at[s]);
            } else {
              *reinterpret_cast<uint4*>(to) = make_uint4(0u, 0u, 0u, 0u);
              *reinterpret_cast<uint4*>(to + NV * kThreads * 16) = make_uint4(0u, 0u, 0u, 0u);
            }
          } else {
            clear(rx[s]);
            clear(rd[s]);
            if (read) { rx[s] = load_pack<T, VE>(x + lane.at[s]); rd[s] = load_pack<T, VE>(dy + lane.at[s]); }
          }
        }
        x += x_step;
        dy += dy_step;
        if (++ahead_h == rounds) { ahead_h = 0; ahead += stride; }
      }
      if constexpr (RING) copy_commit();
    };
#pragma unroll
    for (int i = 0; i < R - 1; ++i) fetch(i);

    int slot = 0;
    for (; unit < units; unit += stride) {
      const Unit u(a, kind, unit, in_warp, per_warp);
      T* out = reinterpret_cast<T*>(a.out) + (long long)u.token * a.out_row + u.head * a.out_head;
      Angles<T, VE, NV, PAIRING, GROUP> angles;
      angles.set(a, turns, lane, g, u.token);
      for (int h = 0; h < rounds; ++h) {
        fetch(slot == 0 ? R - 1 : slot - 1);
        if constexpr (RING) {
          copy_wait<R - 1>();
#pragma unroll
          for (int s = 0; s < NV; ++s) {
            const uint8_t* from = ring + ((slot * 2 * NV + s) * kThreads + threadIdx.x) * 16;
            rx[s] = *reinterpret_cast<const Pack<T, VE>*>(from);
            rd[s] = *reinterpret_cast<const Pack<T, VE>*>(from + NV * kThreads * 16);
          }
          slot = slot == R - 1 ? 0 : slot + 1;
        }
        uint64_t v[M], d[M], gw[M];
        partners.cross(lane, rd, gw);
        unpack<T, VE, NV>(rx, v);
        unpack<T, VE, NV>(rd, d);
        angles.rotate(a, lane, g, d, gw);                     // (a.sign: backwards)
        weights_of<VE, NV>(weights, lane, gw);
#pragma unroll
        for (int i = 0; i < M; ++i) gw[i] = mul_f32x2(d[i], gw[i]);
        float q = dot(v, v), p = dot(gw, v);
        group_sums<GROUP>(q, p, a.group);
        const float r = rsqrtf(q * a.inv_hd + a.eps);
        const float mean = p * r * a.inv_hd;                // of g w u
        const uint64_t r2 = pack_f32x2(r, r), m2 = pack_f32x2(-mean * r, -mean * r);
        if (h < u.count) {
#pragma unroll
          for (int i = 0; i < M; ++i) {
            const uint64_t unit_x = mul_f32x2(v[i], r2);
            sums[i] = fma_f32x2(d[i], unit_x, sums[i]);
            v[i] = fma_f32x2(unit_x, m2, mul_f32x2(gw[i], r2));
          }
          Pack<T, VE> res[NV];
          pack<T, VE, NV>(v, res);
#pragma unroll
          for (int s = 0; s < NV; ++s)
            if (lane.has(s)) store_pack<T, VE>(out + lane.at[s], res[s]);
        }
        out += out_step;
      }
    }
    if constexpr (RING) copy_wait<0>();                       // (empty groups: the ring is free for the next kind)
    unit -= units;                                            // as in the forward pass
    if (a.partial != nullptr) {
      // the lanes that hold the same components: over the warp by shuffles, over the warps in their order
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const float2 f = unpack_f32x2(sums[i / 2]);
        float v = i % 2 ? f.y : f.x;
        for (int o = group; o < 32; o <<= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
        if (in_warp == 0 && lane.component(i) >= 0) reduced[warp][lane.component(i)] = v;
      }
    }
    __syncthreads();                                          // (also: everybody is done with this kind's weights)
    if (a.partial != nullptr) {
      for (int c = threadIdx.x; c < a.hd; c += kThreads) {
        float v = 0.f;
        for (int k = 0; k < kThreads / 32; ++k) v += reduced[k][c];
        a.partial[((size_t)blockIdx.x * 2 + kind) * a.hd + c] = v;
      }
      __syncthreads();
    }
  }
  copy_rest<T, VE, NV>(a, lane, a.dy, a.dy_row, a.dy_head, unit, stride, in_warp, per_warp);
}

// dw[c] = sum over the CTAs of partial[cta][which][c], always in the same order: a block per 32 columns, its 32 warps take
// every 32nd row.
template <typename W>
__global__ void __launch_bounds__(1024) heads_dw_kernel(const float* partial, int parts, int hd, W* dwq, W* dwk,
                                                        int accumulate) {
  __shared__ float red[32][33];
  const int lane = threadIdx.x & 31, row = threadIdx.x >> 5;
  const int c = blockIdx.x * 32 + lane;                       // of the two weights' 2 * hd
  float v = 0.f;
  grid_dependency_wait();                                     // (launched ahead of the end of the kernel before it)
  grid_dependency_launch();
  if (c < 2 * hd) {
#pragma unroll 10
    for (int p = row; p < parts; p += 32) v += partial[(size_t)p * 2 * hd + c];
  }
  red[row][lane] = v;
  __syncthreads();
  if (row == 0 && c < 2 * hd) {
    v = 0.f;
#pragma unroll
    for (int k = 0; k < 32; ++k) v += red[k][lane];
    W* dst = c < hd ? dwq : dwk;
    if (dst != nullptr) {
      dst += c < hd ? c : c - hd;
      *dst = from_f<W>(accumulate ? to_f(*dst) + v : v);
    }
  }
}

// Heads of a group per unit at most.  More of them share a lane's angles, fewer give more units (as many as leave every warp of
// the grid two) and keep what the warps are at closer together in memory, which three streams want most (us, as above, 16 / 8 /
// 4 heads: rotation 65.7 / 71.7 / 70.4, backward 106.4 / 106.6 / 97.0).
constexpr int kMostRounds = 16, kMostRoundsBackward = 4;

enum Pass { kRotate = 0, kForward = 1, kBackward = 2 };

template <typename T, int VE, int NV, int PAIRING, int GROUP, int PASS>
int launch(const HeadArgs& a, int ctas, cudaStream_t stream) {
  if constexpr (PASS == kBackward) {
    auto* kernel = heads_bwd_kernel<T, VE, NV, PAIRING, GROUP>;
    const int smem = VE > 1 ? kBwdRing : 0;
    static bool configured[64] = {false};
    int dev = 0;
    cudaGetDevice(&dev);
    if (smem > 0 && !configured[dev & 63]) {
      const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
      if (e != cudaSuccess) return (int)e;
      configured[dev & 63] = true;
    }
    kernel<<<ctas, kThreads, smem, stream>>>(a);
  } else {
    heads_fwd_kernel<T, VE, NV, PAIRING, PASS == kRotate ? kRope : kNorm, GROUP><<<ctas, kThreads, 0, stream>>>(a);
  }
  return (int)cudaGetLastError();
}

inline bool aligned(const void* p, long long row, long long head, int size) {
  return p == nullptr || (reinterpret_cast<uintptr_t>(p) % 16 == 0 && row * size % 16 == 0 && head * size % 16 == 0);
}

template <typename T, int PASS>
int dispatch(HeadArgs& a, int* parts, cudaStream_t stream) {
  constexpr int VE = 16 / sizeof(T);
  const int size = sizeof(T);
  // in place nothing but what turns is touched (3062 tokens, 32 heads of 80 fp16, 32 of them turned: 8.7 -> 6.7 us)
  if (PASS == kRotate && a.x == a.out && a.rd < a.hd) a.hd = a.hd % VE == 0 ? (a.rd + VE - 1) / VE * VE : a.rd;
  if (a.hd == 0) return DD_OK;
  // whole vectors need heads of whole vectors at 16-byte addresses and two vectors per lane of a warp; else single components,
  // sixteen per lane
  const bool vectors = a.hd % VE == 0 && a.hd <= 64 * VE && aligned(a.x, a.x_row, a.x_head, size) &&
                       aligned(a.dy, a.dy_row, a.dy_head, size) && aligned(a.out, a.out_row, a.out_head, size);
  // halves that are not whole vectors (rd / 2 = 25, say): partners by way of shared memory, 16384 tokens, 48 heads of 128 bf16 of
  // which 50 components turn, us, rotation / in place / norm and rotation / backward: 72 / 39 / 96 / 174 (4 heads per unit 188),
  // single components 131 / 93 / 137 / 272
  const bool crossed = vectors && !a.neighbours && a.rd % (2 * VE) != 0;
  for (a.group = 1; a.group * (vectors ? 2 * VE : 16) < a.hd; a.group *= 2) {}
  const int most = current_sm_count() * kCtasPerSm, warps = kThreads / 32, per_warp = 32 / a.group;
  long long units;
  for (int rounds = PASS == kBackward && !crossed ? kMostRoundsBackward : kMostRounds;; rounds /= 2) {
    units = 0;
    for (int k = 0; k < 3; ++k) {
      a.chunk[k] = rounds * per_warp;
      if (a.chunk[k] > a.heads[k]) a.chunk[k] = (a.heads[k] + per_warp - 1) / per_warp * per_warp;
      a.chunks[k] = a.heads[k] > 0 ? (a.heads[k] + a.chunk[k] - 1) / a.chunk[k] : 0;
      units += (long long)a.tokens * a.chunks[k];
    }
    if (rounds == 1 || units >= 2LL * most * warps) break;
  }
  if (units > 0x3fffffffLL) return DD_ERR_TOO_LARGE;
  const long long want = (units + warps - 1) / warps;
  const int ctas = (int)(want < most ? want : most);
  *parts = ctas;
  if (!vectors) return launch<T, 1, 16, kInside, 0, PASS>(a, ctas, stream);
  // groups of 4 to 32 lanes that all have their vectors know their size beforehand: shuffles and addresses without questions
  // (backward 108 -> 98 us when it was added; 96 now)
  const int full = a.hd == 2 * VE * a.group ? a.group : 0;
  if (a.neighbours) {
    if (full == 4) return launch<T, VE, 2, kInside, 4, PASS>(a, ctas, stream);
    if (full == 8) return launch<T, VE, 2, kInside, 8, PASS>(a, ctas, stream);
    if (full == 16) return launch<T, VE, 2, kInside, 16, PASS>(a, ctas, stream);
    if (full == 32) return launch<T, VE, 2, kInside, 32, PASS>(a, ctas, stream);
    return launch<T, VE, 2, kInside, 0, PASS>(a, ctas, stream);
  }
  if (crossed) return launch<T, VE, 2, kCrossed, 0, PASS>(a, ctas, stream);
  if (full == 4) return launch<T, VE, 2, kApart, 4, PASS>(a, ctas, stream);
  if (full == 8) return launch<T, VE, 2, kApart, 8, PASS>(a, ctas, stream);
  if (full == 16) return launch<T, VE, 2, kApart, 16, PASS>(a, ctas, stream);
  if (full == 32) return launch<T, VE, 2, kApart, 32, PASS>(a, ctas, stream);
  return launch<T, VE, 2, kApart, 0, PASS>(a, ctas, stream);
}

template <int PASS>
int dispatch_type(HeadArgs& a, int dtype, int* parts, cudaStream_t stream) {
  if (dtype == 0) return dispatch<__nv_bfloat16, PASS>(a, parts, stream);
  if (dtype == 1) return dispatch<__half, PASS>(a, parts, stream);
  if (dtype == 2) return dispatch<float, PASS>(a, parts, stream);
  return DD_ERR_BAD_ARG;
}

}  // namespace

// CTAs (and rows of the backward pass's scratch) at most.
DD_API int dd_heads_parts() { return current_sm_count() * kCtasPerSm; }

// A call, packed by the caller: ctypes takes longer for thirty arguments than a launch does.  Tensors [tokens, hq + hk + rest,
// hd] by address, token and head stride (in elements; unit stride inside a head), dtype 0 bf16, 1 fp16, 2 fp32.
//   pass 0 (rotation)  out = x with the first hq heads turned (sign -1: backwards); the others are copied, or with out == x left
//                      alone (hk is 0)
//   pass 1 (norm)      out = x with the first hq heads normed with wq and turned, the next hk with wk, the others as above
//   pass 2 (backward)  out = dx from x and dy (out of place); dwq, dwk [hd] of the weights' type (null: not wanted), or with
//                      accumulate added to what is there, fp32; partial: dd_heads_parts() * 2 * hd floats where they are wanted
// Weights [hd] of x's type, or fp32 with wide_weights, or null.  turns [rd / 2]: frequencies in turns per position (host
// memory); positions [seq] on the device (4 or, wide_positions, 8 bytes each) of token % seq, or null for offset + token % seq.
// Where a second range of positions follows the first in every sequence, two more numbers stand behind the call: the place it begins
// at, and what is added to its positions.
struct HeadsCall {
  const void *x, *dy;
  void* out;
  const void *wq, *wk;
  void *dwq, *dwk;
  float* partial;
  const void* positions;
  const double* turns;
  long long x_row, x_head, dy_row, dy_head, out_row, out_head, tokens, offset, seq;
  int pass, dtype, hq, hk, rest, hd, rd, neighbours, wide_weights, wide_positions, accumulate;
  float magnitude, sign, eps;
};
static_assert(sizeof(HeadsCall) == 19 * 8 + 14 * 4, "packed without holes");
struct SecondRange { long long split, jump; };

DD_API int dd_heads(const void* packed, int bytes, void* stream) {
  HeadsCall c;
  SecondRange second = {0x7fffffffLL, 0};
  const bool two = bytes == (int)(sizeof c + sizeof second);
  if (packed == nullptr || (bytes != (int)sizeof c && !two)) return DD_ERR_BAD_ARG;
  memcpy(&c, packed, sizeof c);
  if (two) memcpy(&second, static_cast<const char*>(packed) + sizeof c, sizeof second);
  if (second.split < 0) return DD_ERR_BAD_ARG;
  const bool back = c.pass == kBackward;
  if (c.pass < kRotate || c.pass > kBackward || (c.pass == kRotate && c.hk != 0)) return DD_ERR_BAD_ARG;
  if (c.tokens < 0 || c.hq < 0 || c.hk < 0 || c.rest < 0 || c.hd < 1 || c.rd < 0 || c.rd > c.hd || c.rd % 2 != 0)
    return DD_ERR_BAD_ARG;
  if (c.rd > 0 && (c.turns == nullptr || c.seq < 1)) return DD_ERR_BAD_ARG;
  if (c.dtype < 0 || c.dtype > 2) return DD_ERR_BAD_ARG;
  if (c.hd > 2 * kMaxPairs || c.tokens > 0x3fffffffLL) return DD_ERR_TOO_LARGE;
  const bool weights = back && (c.dwq != nullptr || c.dwk != nullptr);
  if (weights && c.partial == nullptr) return DD_ERR_BAD_ARG;
  HeadArgs a = {};
  a.x = c.x; a.x_row = c.x_row; a.x_head = c.x_head;
  a.out = c.out; a.out_row = c.out_row; a.out_head = c.out_head;
  a.tokens = (unsigned)c.tokens;
  a.seq = c.seq < 1 ? 1u : c.seq > 0x3fffffffLL ? 0x3fffffffu : (unsigned)c.seq;
  a.heads[0] = back ? c.hq : c.hq + c.hk;
  a.heads[1] = back ? c.hk : 0;
  a.heads[2] = !back && c.x == c.out ? 0 : c.rest;
  a.queries = c.hq;
  a.hd = c.hd; a.rd = c.rd; a.neighbours = c.neighbours;
  a.positions = c.positions; a.wide_positions = c.wide_positions; a.offset = c.offset;
  a.split = second.split > 0x7fffffffLL ? 0x7fffffffu : (unsigned)second.split; a.offset_behind = c.offset + second.jump;
  a.magnitude = c.magnitude;
  a.inv_hd = 1.f / (float)c.hd;
  a.sign = back ? -1.f : c.pass == kRotate ? c.sign : 1.f;
  for (int i = 0; i < c.rd / 2; ++i) a.turns[i] = c.turns[i];
  if (c.pass != kRotate) { a.wq = c.wq; a.wk = c.wk; a.wide_weights = c.wide_weights; a.eps = c.eps; }
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  int parts = 0;
  if (c.tokens > 0 && a.heads[0] + a.heads[1] + a.heads[2] > 0) {
    if (c.x == nullptr || c.out == nullptr || (back && c.dy == nullptr)) return DD_ERR_BAD_ARG;
    if (back) {
      a.dy = c.dy; a.dy_row = c.dy_row; a.dy_head = c.dy_head;
      a.partial = weights ? c.partial : nullptr;
    }
    const int e = c.pass == kRotate    ? dispatch_type<kRotate>(a, c.dtype, &parts, st)
                  : c.pass == kForward ? dispatch_type<kForward>(a, c.dtype, &parts, st)
                                       : dispatch_type<kBackward>(a, c.dtype, &parts, st);
    if (e) return e;
  }
  if (!weights) return DD_OK;
  const int grid = (2 * c.hd + 31) / 32;                      // (no tokens: parts = 0, zeros)
  auto add = [&](auto* dwq, auto* dwk, int accumulate) {
    using W = std::remove_pointer_t<decltype(dwq)>;
    return launch_ahead(heads_dw_kernel<W>, dim3(grid), dim3(1024), 0, st, true, (const float*)c.partial, parts, c.hd, dwq, dwk,
                        accumulate);
  };
  if (c.accumulate || c.wide_weights || c.dtype == 2) return add((float*)c.dwq, (float*)c.dwk, c.accumulate);
  if (c.dtype == 1) return add((__half*)c.dwq, (__half*)c.dwk, 0);
  return add((__nv_bfloat16*)c.dwq, (__nv_bfloat16*)c.dwk, 0);
}
