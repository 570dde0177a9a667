// Routing of tokens to experts in its general form: softmax or sigmoid scores, a bias that takes part in the choice only,
// choice within the best groups of experts, weights renormalised or not; up to 512 experts, 32 of them per token.  (The plain
// softmax form for up to 64 bf16 experts is in moe.cu.)
//
//   score    s = softmax(l) or 1 / (1 + e^-l) over the E logits of a token;  p = s / sum s
//   choice   c = s + bias; of the groups (E / groups experts each) the top_groups with the largest value (the largest c, or the
//            sum of the two largest), of their experts the k largest c; ties go to the lowest number
//   weights  w = scale * s, or scale * s / (sum of the chosen s)
//   backward with g on w and q on sum_t p:  d s_i of the chosen from g, d p from q, and ds / dl = s (1 - s) (sigmoid),
//            written out per case at the kernel
//
// An expert whose logit or bias is -inf is never chosen; a token with fewer than k others has -1 and weight 0 in the places left,
// one with none of them routes nowhere and adds nothing.  A NaN (softmax: also +inf) makes the weights of its token, its p and
// its gradient NaN, and counts as the best, so that a token of NaN alone is not lost either.
//
// The choice is that of exact arithmetic.  Experts are compared as integers: 23 bits of value over 9 bits that favour the
// lower number.  16-bit logits that decide themselves (no bias, no sums of scores) fit into them; everything else is cut to
// steps of 2^-23 of the token's range, and where one of the chosen and another expert are closer than their errors (and not
// alike in logit and bias), or a sum of two holds a value below the range, those that matter are decided in 64 bits: some tokens
// in a thousand.  So neither the order of sums nor the fast
// exponential shows in the experts.
//
// A warp works on a token, its lanes on C consecutive experts each, which they sort; the k best are then the largest of the
// lanes' first ones, k times, one warp-wide integer maximum each.  Above some thousand tokens instructions that follow from one
// another bound it, 580 (softmax, no bias) to 840 (sigmoid, bias, 8 groups) per token of 256 experts: 16384 tokens 23 to 30 us
// with the slots (with the experts unsorted and the winner's place looked for by ballot and shuffle 1 130 to 1 920, 40 to 66
// us); below, a latency.  Slots follow in a second kernel (route_slot_kernel): a pair's
// slot is its rank in pair order among the pairs of its expert, so nothing depends on how CTAs are scheduled; sums of p are
// formed per chunk of tokens and then over the chunks, always in the same order.
#include "common.cuh"
#include "runtime.cuh"

#include <cuda_fp16.h>

#include <cfloat>
#include <cstring>

using namespace dd;

namespace {

constexpr int kMaxExperts = 512, kMaxChoices = 32, kMaxGroups = 32;
constexpr int kWarps = 8;
constexpr int kMostRows = 256;                                // tokens of a chunk (a CTA of the first kernel) at most
constexpr int kSlotThreads = 1024;                            // of a CTA of the second kernel, which takes whole chunks

// Tokens of a chunk: a token per warp while that gives every SM up to three CTAs, then so many that it still does.
inline int rows_of(int tokens) {
  const int per_warp = (tokens - 1) / (kWarps * 3 * 148) + 1;
  return kWarps * (per_warp < kMostRows / kWarps ? per_warp : kMostRows / kWarps);
}

struct RouteArgs {
  const void* logits;       // [tokens, ld]
  const float* bias;        // [E] or null
  int* ids;                 // [tokens, k]
  float* w;                 // [tokens, k]
  int* hist;                // [chunks][E4]: pairs per expert
  float* psum;              // [chunks][E4]: sums of p
  int ld, tokens, rows, E, E4, k;
  int groups, top_groups, size;                               // size: experts of a group
  int lanes;                                                  // of a group, where it begins and ends with a lane's; else 0
  bool group_sum, sigmoid, renormalize, by_logit, vectors;
  float scale;
};

template <typename T> __device__ __forceinline__ float to_f(T v);
template <> __device__ __forceinline__ float to_f(float v) { return v; }
template <> __device__ __forceinline__ float to_f(__half v) { return __half2float(v); }
template <> __device__ __forceinline__ float to_f(__nv_bfloat16 v) { return __bfloat162float(v); }
template <typename T> __device__ __forceinline__ T from_f(float v);
template <> __device__ __forceinline__ float from_f(float v) { return v; }
template <> __device__ __forceinline__ __half from_f(float v) { return __float2half_rn(v); }
template <> __device__ __forceinline__ __nv_bfloat16 from_f(float v) { return __float2bfloat16_rn(v); }

// C values of one lane in memory, moved in pieces of up to 16 bytes.
template <typename T, int C> struct alignas(C * sizeof(T) < 16 ? C * sizeof(T) : 16) Row { T v[C]; };

// Where a value of each expert stands in shared memory, so that the lanes' loads of up to 16 bytes lie side by side.
template <int C> __device__ __forceinline__ int place_of(int lane, int j) {
  constexpr int V = C < 4 ? C : 4;
  return lane * V + j / V * 32 * V + j % V;
}

template <typename T, int C>
__device__ __forceinline__ void load_row(const T* p, bool vectors, int left, float (&l)[C]) {
  if (vectors && left >= C) {
    const Row<T, C> r = *reinterpret_cast<const Row<T, C>*>(p);
#pragma unroll
    for (int j = 0; j < C; ++j) l[j] = to_f(r.v[j]);
  } else {
#pragma unroll
    for (int j = 0; j < C; ++j) l[j] = j < left ? to_f(p[j]) : -INFINITY;
  }
}

// Order-preserving: a < b as floats, ordered(a) < ordered(b) as integers.
__device__ __forceinline__ unsigned ordered(float v) {
  unsigned u = __float_as_uint(v);
  if (u == 0x80000000u) u = 0u;                               // -0 is 0
  return u ^ ((unsigned)((int)u >> 31) | 0x80000000u);
}
// Largest and smallest value of a warp; a NaN is the largest.
__device__ __forceinline__ float top_of_warp(float v) {
  float r;
  asm("redux.sync.max.NaN.f32 %0, %1, 0xffffffff;" : "=f"(r) : "f"(v));
  return r;
}
__device__ __forceinline__ float low_of_warp(float v) {
  float r;
  asm("redux.sync.min.f32 %0, %1, 0xffffffff;" : "=f"(r) : "f"(v));
  return r;
}
__device__ __forceinline__ float max_or_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
// Keys: value (23 bits) << 9 | 511 - expert, 0 for an expert that may not be chosen.
constexpr float kSteps = 8388600.f;
constexpr unsigned kBad = 0xfffffe00u;

// Falling, by Batcher's odd-even merges.
template <int C>
__device__ __forceinline__ void sort_falling(unsigned (&key)[C]) {
#pragma unroll
  for (int p = 1; p < C; p *= 2)
#pragma unroll
    for (int q = p; q >= 1; q /= 2)
#pragma unroll
      for (int j = q % p; j + q < C; j += 2 * q)
#pragma unroll
        for (int i = 0; i < q; ++i)
          if (i + j + q < C && (i + j) / (2 * p) == (i + j + q) / (2 * p)) {
            const unsigned x = key[i + j], y = key[i + j + q];
            key[i + j] = max(x, y);
            key[i + j + q] = min(x, y);
          }
}
// The two largest values of every group of experts, each in all lanes that `step` lanes of a group share; V: int or double.
// best: this lane's own two, where groups begin and end with a lane's experts (a.lanes), else all values by expert in shared
// memory, `none` where there is no expert.  Returns the group of this lane.
template <typename V>
__device__ __forceinline__ int best_of_groups(const RouteArgs& a, const V* values, V none, V& b0, V& b1, int& step) {
  const int lane = threadIdx.x & 31;
  if (a.lanes > 0) {
    step = a.lanes;
  } else {
    step = a.groups > 16 ? 1 : a.groups > 8 ? 2 : a.groups > 4 ? 4 : a.groups > 2 ? 8 : 16;
    b0 = b1 = none;
    if (lane / step < a.groups)
      for (int i = lane % step; i < a.size; i += step) {
        const V v = values[lane / step * a.size + i];
        b1 = max(b1, min(b0, v));
        b0 = max(b0, v);
      }
  }
  for (int o = 1; o < step; o <<= 1) {
    const V o0 = __shfl_xor_sync(0xffffffffu, b0, o), o1 = __shfl_xor_sync(0xffffffffu, b1, o);
    b1 = max(max(b1, o1), min(b0, o0));
    b0 = max(b0, o0);
  }
  return lane / step;
}
// Whether the group of this lane is among the best, the lower numbers first where they are alike.
template <typename V>
__device__ __forceinline__ bool among_best(const RouteArgs& a, V value, int g, int step) {
  int place = 0;
  for (int i = 0; i < a.groups; ++i) {
    const V v = __shfl_sync(0xffffffffu, value, i * step);
    place += v > value || (v == value && i < g);
  }
  return g < a.groups && place < a.top_groups;
}
// Clears what a lane holds of groups that are not kept.
template <typename V, int C>
__device__ __forceinline__ void clear_others(const RouteArgs& a, V (&v)[C], V none, bool in, int first, int left, int step) {
  if (a.lanes > 0) {
    if (!in) {
#pragma unroll
      for (int j = 0; j < C; ++j) v[j] = none;
    }
  } else {
    const unsigned kept = __ballot_sync(0xffffffffu, in);
    int of = first / a.size, at = first - of * a.size;
#pragma unroll
    for (int j = 0; j < C; ++j) {
      if (j >= left || !((kept >> (of * step)) & 1u)) v[j] = none;
      if (++at == a.size) { at = 0; ++of; }
    }
  }
}

// What an expert is chosen by, in 64 bits (softmax scores: choose_in_64_bits).  T: of the logits.
template <typename T>
__device__ __forceinline__ double value_in_64_bits(const RouteArgs& a, const T* from, int e) {
  const double l = to_f(from[e]);
  return (a.by_logit ? l : 1.0 / (1.0 + exp(-l))) + (a.bias != nullptr ? (double)a.bias[e] : 0.0);
}
// Whether this lane's group is among the best, in 64 bits: of a lane's sorted keys those that can be one of its group's two best
// (its best), their value >= least.  (What decides few tokens is kept short: others wait at the end for the one that is fetching
// instructions.  With all experts in 64 bits 16384 tokens took 34 us, with those that matter 29.)
template <typename T, int C>
__device__ __noinline__ bool groups_in_64_bits(const RouteArgs& a, const unsigned* key, int least, const T* from) {
  double b0 = -INFINITY, b1 = -INFINITY;
#pragma unroll 1
  for (int j = 0; j < C; ++j) {
    const bool in = key[j] != 0u && (int)(key[j] >> 9) >= least;
    if (!__any_sync(0xffffffffu, in)) break;
    const double v = in ? value_in_64_bits<T>(a, from, 511 - (int)(key[j] & 511u)) : -INFINITY;
    b1 = fmax(b1, fmin(b0, v));
    b0 = fmax(b0, v);
  }
  int step;
  const int g = best_of_groups<double>(a, nullptr, -INFINITY, b0, b1, step);
  return among_best(a, a.group_sum && b1 > -INFINITY ? b0 + b1 : b0, g, step);
}
// The first k of n candidates, the i-th key in lane i (0: none), in the order of 64 bits.
template <typename T>
__device__ __noinline__ int order_in_64_bits(const RouteArgs& a, unsigned mine, int n, const T* from) {
  const int lane = threadIdx.x & 31, e = mine != 0u ? 511 - (int)(mine & 511u) : kMaxExperts;
  const double c = mine != 0u ? value_in_64_bits<T>(a, from, e) : -INFINITY;
  int place = 0;
#pragma unroll 1
  for (int i = 0; i < n; ++i) {
    const double other = __shfl_sync(0xffffffffu, c, i);
    const int f = __shfl_sync(0xffffffffu, e, i);
    place += other > c || (other == c && f < e);
  }
  int chosen = -1;
#pragma unroll 1
  for (int i = 0; i < n; ++i) {
    const int f = __shfl_sync(0xffffffffu, e, i);
    if (__shfl_sync(0xffffffffu, place, i) == lane && f < kMaxExperts) chosen = f;
  }
  return lane < a.k ? chosen : -1;
}

// The choice of one token from the keys of its experts: lane i gets the i-th expert, -1 where there is none.  `close` is set
// where values within `near` of one another (near < 0: all values are exact) decide, are not those of experts alike in logit
// and bias, and are not decided here (`here`: where they can be).  Values up to `floor` may stand for any below them.
template <typename T, int C>
__device__ __forceinline__ int choose(const RouteArgs& a, unsigned (&key)[C], int first, int left, int near, int floor, bool here,
                                      bool& close, int* values, const T* from) {
  const int lane = threadIdx.x & 31;
  if (a.groups > 1) {
    int b0, b1, step;
    if (a.lanes > 0) {
      sort_falling<C>(key);
      b0 = (int)(key[0] >> 9);
      b1 = C > 1 ? (int)(key[C > 1] >> 9) : 0;
    } else {
#pragma unroll
      for (int j = 0; j < C; ++j)
        if (j < left) values[first + j] = (int)(key[j] >> 9);
      __syncwarp();
    }
    const int g = best_of_groups<int>(a, values, 0, b0, b1, step);
    // value (24 bits) over what favours the lower number: the best groups one by one, as the experts below
    unsigned group = g < a.groups ? (unsigned)(a.group_sum ? b0 + b1 : b0) << 5 | (unsigned)(31 - g) : 0u, worst = 0u;
    bool in = false;
    for (int i = 0; i < a.top_groups; ++i) {
      worst = __reduce_max_sync(0xffffffffu, group);
      if (group == worst) { in = g < a.groups; group = 0u; }
    }
    if (near >= 0) {
      const int least = (int)(worst >> 5), most = (int)(__reduce_max_sync(0xffffffffu, group) >> 5);
      // (of a group with one expert only its value itself would have to be known, and of a sum that is among the best
      // both values: one that may be any below counts for too much)
      close = (most > 0 && least - most <= (a.group_sum ? 2 * near : near)) ||
              __any_sync(0xffffffffu, g < a.groups && a.group_sum && a.size > 1 && b0 > 0 && b1 <= (in ? floor : 0));
      if (close && here && a.lanes > 0) {
        unsigned sorted[C];
#pragma unroll
        for (int j = 0; j < C; ++j) sorted[j] = key[j];
        in = groups_in_64_bits<T, C>(a, sorted, (a.group_sum ? b1 : b0) - near, from);
        close = false;
      }
    }
    clear_others<unsigned, C>(a, key, 0u, in, first, left, step);
    if (a.lanes == 0) {
      __syncwarp();
      sort_falling<C>(key);
    }
  } else {
    sort_falling<C>(key);
  }
  // the k best one by one: lane i keeps the i-th key
  unsigned mine = 0u;
  for (int i = 0; i < a.k; ++i) {
    const unsigned top = __reduce_max_sync(0xffffffffu, key[0]);
    if (lane == i) mine = top;
    if (key[0] == top) {
#pragma unroll
      for (int j = 0; j + 1 < C; ++j) key[j] = key[j + 1];
      key[C - 1] = 0u;
    }
  }
  if (near >= 0) {                                            // none may be close to the next, the first left out included
    const unsigned next = __shfl_down_sync(0xffffffffu, mine, 1);
    unsigned out = __reduce_max_sync(0xffffffffu, key[0]), last = __shfl_sync(0xffffffffu, mine, a.k - 1);
    // (two alike in logit and bias are alike, and in order)
    auto same = [&](unsigned x, unsigned y) {
      const int e = 511 - (int)(x & 511u), f = 511 - (int)(y & 511u);
      return to_f(from[f]) == to_f(from[e]) && (a.bias == nullptr || a.bias[f] == a.bias[e]);
    };
    bool alike = true;
    if (lane < a.k - 1 && next != 0u && (int)(mine >> 9) - (int)(next >> 9) <= near) alike = same(mine, next);
    // of those left out all that are close, not the next one alone: behind some that are alike there may be others
    if (out != 0u && (int)(last >> 9) - (int)(out >> 9) <= near) {
#pragma unroll
      for (int j = 0; j < C; ++j)
        if (key[j] != 0u && (int)(last >> 9) - (int)(key[j] >> 9) <= near) alike = alike && same(last, key[j]);
    }
    if (__any_sync(0xffffffffu, !alike)) {
      if (!here || close) { close = true; return -1; }
      // all that may be among the k best: up to the first that is not close to the one before it
      int n = a.k;
      while (out != 0u && (int)(last >> 9) - (int)(out >> 9) <= near) {
        if (n == 32) { close = true; return -1; }
        if (lane == n) mine = out;
        ++n;
        last = out;
        if (key[0] == out) {
#pragma unroll
          for (int j = 0; j + 1 < C; ++j) key[j] = key[j + 1];
          key[C - 1] = 0u;
        }
        out = __reduce_max_sync(0xffffffffu, key[0]);
      }
      return order_in_64_bits<T>(a, mine, n, from);
    }
  }
  const int chosen = lane < a.k && mine != 0u ? 511 - (int)(mine & 511u) : -1;
  return chosen;
}

__device__ __forceinline__ double warp_sum_d(double v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}
// Order-preserving, as ordered(); 0: -inf.
__device__ __forceinline__ unsigned long long ordered_d(double v) {
  if (!(v > -INFINITY)) return 0ull;
  const unsigned long long u = (unsigned long long)__double_as_longlong(v + 0.0);
  return u ^ ((unsigned long long)((long long)u >> 63) | 0x8000000000000000ull);
}

// The choice of a token in 64 bits.  l_in: this lane's logits (-inf: not to be chosen, or bad: the best); top: the token's
// largest.
template <int C>
__device__ __noinline__ int choose_in_64_bits(const RouteArgs& a, const float* l_in, float top, unsigned bad, int first, int left,
                                              double* values) {
  const int lane = threadIdx.x & 31;
  double c[C], z = 0.0;
#pragma unroll
  for (int j = 0; j < C; ++j) {
    const double l = l_in[j];
    c[j] = a.by_logit ? l : a.sigmoid ? 1.0 / (1.0 + exp(-l)) : exp(l - (double)top);
    z += c[j];
  }
  if (!a.by_logit && !a.sigmoid) z = warp_sum_d(z);
#pragma unroll
  for (int j = 0; j < C; ++j) {
    if (!a.by_logit && !a.sigmoid) c[j] /= z;
    if (a.bias != nullptr && j < left) c[j] += (double)a.bias[first + j];
    if (!(l_in[j] > -INFINITY) || c[j] != c[j]) c[j] = (bad >> j) & 1u ? INFINITY : -INFINITY;
    else c[j] = fmin(c[j], DBL_MAX);                          // (+inf from a sigmoid or a bias: below what is no number)
  }
  if (a.groups > 1) {
    double b0 = -INFINITY, b1 = -INFINITY;
    int step;
    if (a.lanes > 0) {
#pragma unroll
      for (int j = 0; j < C; ++j) {
        b1 = fmax(b1, fmin(b0, c[j]));
        b0 = fmax(b0, c[j]);
      }
    } else {
#pragma unroll
      for (int j = 0; j < C; ++j)
        if (j < left) values[first + j] = c[j];
      __syncwarp();
    }
    const int g = best_of_groups<double>(a, values, -INFINITY, b0, b1, step);
    const double value = a.group_sum && b1 > -INFINITY && b0 < INFINITY ? fmin(b0 + b1, DBL_MAX) : b0;
    const bool in = among_best(a, value, g, step);
    clear_others<double, C>(a, c, -INFINITY, in, first, left, step);
    __syncwarp();
  }
  unsigned long long key[C];
#pragma unroll
  for (int j = 0; j < C; ++j) key[j] = ordered_d(c[j]);
  int chosen = -1;
  for (int i = 0; i < a.k; ++i) {
    unsigned long long best = 0ull;
    int e = 0;
#pragma unroll
    for (int j = 0; j < C; ++j)
      if (key[j] > best) { best = key[j]; e = first + j; }
    const unsigned hi = __reduce_max_sync(0xffffffffu, (unsigned)(best >> 32));
    const unsigned lo = __reduce_max_sync(0xffffffffu, (unsigned)(best >> 32) == hi ? (unsigned)best : 0u);
    const unsigned long long most = (unsigned long long)hi << 32 | lo;
    if (most == 0ull) break;
    e = __shfl_sync(0xffffffffu, e, __ffs(__ballot_sync(0xffffffffu, best == most)) - 1);
    if (lane == i) chosen = e;
#pragma unroll
    for (int j = 0; j < C; ++j)
      if (first + j == e) key[j] = 0ull;
  }
  return chosen;
}

// The largest logit of a token.  Logits without a number (NaN; softmax: +inf) are taken out of a lane's, as bits of `bad`;
// `nan`: whether the token has any.
template <int C>
__device__ __forceinline__ float top_logit(float (&l)[C], bool sigmoid, unsigned& bad, bool& nan) {
  float top = l[0];
#pragma unroll
  for (int j = 1; j < C; ++j) top = max_or_nan(top, l[j]);
  top = top_of_warp(top);
  nan = top != top || (!sigmoid && top == INFINITY);
  if (nan) {
    top = -INFINITY;
#pragma unroll
    for (int j = 0; j < C; ++j) {
      if (l[j] != l[j] || (!sigmoid && l[j] == INFINITY)) {
        bad |= 1u << j;
        l[j] = -INFINITY;
      }
      top = fmaxf(top, l[j]);
    }
    top = top_of_warp(top);
  }
  return top;
}

// e^x for x <= 0, within 2^-21 however far below zero: x log2 e as a product and what its rounding leaves (Dekker's two-product by
// fma, and the rest of the constant), the second by its first-order term.  (__expf forms the product alone, which is off by
// |x| 2^-24; 16384 tokens of 256 experts 22.6 -> 23.6 us.)
__device__ __forceinline__ float exp_of(float x) {
  constexpr double kLog2e = 1.4426950408889634;
  constexpr float kHigh = (float)kLog2e, kRest = (float)(kLog2e - (double)kHigh), kLn2 = 0.6931471805599453f;
  x = fmaxf(x, -200.f);                                       // (0 from -104 on; -inf has no remainder)
  const float t = x * kHigh, rest = fmaf(x, kRest, fmaf(x, kHigh, -t));
  const float e = exp2f(t);
  return fmaf(e, rest * kLn2, e);
}

// Scores of a token, p = s / sum s (0 in rows without an expert), from the largest logit.  Sigmoids take the fast exponential: a
// score is off by 2^-22 + (1 - s) |l| 2^-23 of itself, so that only scores that count for nothing beside others lose bits.
template <int C>
struct Scores {
  float inv;                // p = part * inv
  float part[C];            // softmax: e^(l - top); sigmoid: s / e^min(top, 0), which does not underflow in whole rows

  __device__ __forceinline__ void set(const float (&l)[C], bool sigmoid, float top) {
    const bool none = top == -INFINITY;
    float z = 0.f;
    if (!sigmoid) {
      const float shift = none ? 0.f : top;
#pragma unroll
      for (int j = 0; j < C; ++j) part[j] = exp_of(l[j] - shift);
    } else if (top >= 0.f) {
#pragma unroll
      for (int j = 0; j < C; ++j) part[j] = __fdividef(1.f, 1.f + __expf(-l[j]));   // (e^88: 0, as e^-88)
    } else {
      const float shift = none ? 0.f : top;
#pragma unroll
      for (int j = 0; j < C; ++j) part[j] = __fdividef(__expf(l[j] - shift), 1.f + __expf(l[j]));
    }
#pragma unroll
    for (int j = 0; j < C; ++j) z += part[j];
    inv = none ? 0.f : __fdividef(1.f, warp_sum(z));
  }
};

template <typename T, int C>
__global__ void __launch_bounds__(kWarps * 32, C <= 8 ? 3 : 2) route_kernel(const __grid_constant__ RouteArgs a) {
  __shared__ int s_hist[kMaxExperts];
  __shared__ __align__(16) float s_bias[32 * C];
  __shared__ __align__(16) double s_row[kWarps][32 * C];      // a warp's values by expert; at the end its sums of p
  grid_dependency_launch();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  for (int e = threadIdx.x; e < a.E; e += kWarps * 32) s_hist[e] = 0;
  for (int e = threadIdx.x; e < 32 * C; e += kWarps * 32)
    s_bias[place_of<C>(e / C, e % C)] = a.bias != nullptr && e < a.E ? a.bias[e] : 0.f;
  __syncthreads();
  const int first = lane * C;
  const int left = min(max(a.E - first, 0), C);               // experts of this lane
  const bool exact = a.by_logit && sizeof(T) == 2;            // the logits fit into a key's value
  float sums[C];
#pragma unroll
  for (int j = 0; j < C; ++j) sums[j] = 0.f;

  for (int row = warp; row < a.rows; row += kWarps) {
    const int t = blockIdx.x * a.rows + row;
    if (t >= a.tokens) break;
    const T* from = reinterpret_cast<const T*>(a.logits) + (size_t)t * a.ld;
    float l[C];
    load_row<T, C>(from + first, a.vectors, left, l);
    unsigned bad = 0u;                                        // this lane's experts without a number
    bool nan;
    const float top_l = top_logit<C>(l, a.sigmoid, bad, nan);
    Scores<C> s;
    s.set(l, a.sigmoid, top_l);
    unsigned key[C];
    int near = -1, floor = 0;                                 // differences, and values, up to here say nothing
    if (exact) {
#pragma unroll
      for (int j = 0; j < C; ++j) key[j] = l[j] > -INFINITY ? (ordered(l[j]) & ~511u) | (511 - first - j) : 0u;
    } else {
      float v[C], hi = -INFINITY, lo = INFINITY;
      const float back = a.by_logit ? 0.f : a.sigmoid ? __expf(fminf(top_l, 0.f)) : s.inv;
#pragma unroll
      for (int j = 0; j < C; ++j) {
        v[j] = a.by_logit ? l[j] : s.part[j] * back + s_bias[place_of<C>(lane, j)];
        if (!(l[j] > -INFINITY)) v[j] = -INFINITY;            // (a bias of -inf takes an expert out, too)
        hi = fmaxf(hi, v[j]);
        lo = fminf(lo, v[j]);
      }
      hi = top_of_warp(hi);
      // (values far below the largest, -inf among them, are not told apart: should they decide, they are close)
      const float low = low_of_warp(lo);
      lo = fmaxf(low, hi - (a.by_logit ? 64.f : 8.f));
      floor = low < lo;
      const float range = hi - lo, steps = range > 1e-25f ? __fdividef(kSteps, range) : 0.f;
      // scores: sigmoid 4e-7 off at most (its slope times the exponential's error, a division), softmax 4e-6 of the largest,
      // the bias's addition; the cut itself: a step each way
      const float off = a.by_logit ? 0.f : (a.sigmoid ? 2e-6f : 8e-6f * s.inv) + 4e-7f * fmaxf(fabsf(hi), fabsf(lo));
      near = (int)fminf(off * steps + 3.f, 8388607.f);
#pragma unroll
      for (int j = 0; j < C; ++j)
        // (2^23 + a whole number: the number is the mantissa, and the shift drops the rest)
        key[j] = v[j] > -INFINITY ? (__float_as_uint(fmaf(fmaxf(v[j] - lo, 0.f), steps, 8388609.f)) << 9) + (511 - first - j) : 0u;
    }
    if (nan) {
#pragma unroll
      for (int j = 0; j < C; ++j)
        if ((bad >> j) & 1u) key[j] = kBad | (511 - first - j);
    }
    bool close = false;
    int chosen = choose<T, C>(a, key, first, left, near, floor, !nan && (a.by_logit || a.sigmoid), close,
                              reinterpret_cast<int*>(s_row[warp]), from);
    close = close || (nan && a.groups > 1 && a.group_sum);    // (what is no number is the best, whatever is added to it)
    if (close) {                                              // (the same on every lane)
      float again[C];
#pragma unroll
      for (int j = 0; j < C; ++j) again[j] = l[j];
      chosen = choose_in_64_bits<C>(a, again, top_l, bad, first, left, s_row[warp]);
    }
    // the weights, from the chosen logits: sums of k lanes, shifted so that the largest does not underflow
    float weight = 0.f;
    {
      const float lc = chosen >= 0 && !nan ? to_f(from[chosen]) : -INFINITY;
      const float top = a.renormalize ? top_of_warp(lc) : top_l;
      float v;
      if (a.sigmoid) {
        const float shift = a.renormalize ? fminf(top, 0.f) : 0.f, e = __expf(-fabsf(lc));
        v = __fdividef(lc > 0.f ? 1.f : shift == 0.f ? e : __expf(lc - shift), 1.f + e);
      } else {
        v = exp_of(lc - top);
      }
      if (chosen < 0) v = 0.f;
      if (a.renormalize) v = __fdividef(v, warp_sum(v));
      else if (!a.sigmoid) v *= s.inv;
      weight = chosen < 0 ? 0.f : a.scale * v;
      if (nan && chosen >= 0) weight = __int_as_float(0x7fffffff);
    }
    if (lane < a.k) {
      a.ids[(size_t)t * a.k + lane] = chosen;
      a.w[(size_t)t * a.k + lane] = weight;
      if (chosen >= 0) atomicAdd(&s_hist[chosen], 1);
    }
    const float inv = nan ? __int_as_float(0x7fffffff) : s.inv;
#pragma unroll
    for (int j = 0; j < C; ++j) sums[j] += s.part[j] * inv;
  }
  __syncwarp();
  float* s_sums = reinterpret_cast<float*>(&s_row[0][0]);     // [kWarps][64 C], the first halves
#pragma unroll
  for (int j = 0; j < C; ++j) s_sums[warp * 64 * C + first + j] = sums[j];
  __syncthreads();
  for (int e = threadIdx.x; e < a.E4; e += kWarps * 32) {
    float v = 0.f;
    for (int k = 0; k < kWarps; ++k) v += s_sums[k * 64 * C + e];
    a.psum[(size_t)blockIdx.x * a.E4 + e] = e < a.E ? v : 0.f;
    a.hist[(size_t)blockIdx.x * a.E4 + e] = e < a.E ? s_hist[e] : 0;
  }
}

// slot[pair] = rank of the pair among those of its expert in pair order, -1 from the capacity on (and for -1 in ids).  The
// experts of a token differ, so that the rank is the number of earlier tokens: whole CTAs before (sums over the chunks'
// histograms), words of 32 tokens before, lower bits in the word.
__global__ void __launch_bounds__(kSlotThreads)
route_slot_kernel(const int* ids, int tokens, int k, int E, int E4, int capacity, const int* hist, const float* psum, int chunks,
                  int chunk, int per_cta, int* counts, float* prob_sum, int* slot) {
  constexpr int W = kMostRows / 32, kOwn = 2;                 // kOwn: pairs of a thread whose experts are fetched at once
  __shared__ unsigned s_mask[W][kMaxExperts];
  __shared__ __align__(16) int s_part[kSlotThreads * 4];      // sums before this CTA; then [W][kMaxExperts] bases
  const int tid = threadIdx.x, lane = tid & 31;
  for (int i = tid; i < W * kMaxExperts; i += kSlotThreads) (&s_mask[0][0])[i] = 0u;
  const int quads = E4 / 4, lanes = kSlotThreads / quads;     // threads per four experts
  const int before = blockIdx.x * per_cta, t0 = before * chunk;          // chunks and tokens before this CTA's
  const int pairs = min(tokens - t0, per_cta * chunk) * k;
  grid_dependency_wait();                                     // (launched ahead of the end of the kernel before it)
  grid_dependency_launch();
  // everything that is read, first: a latency is all that this kernel is made of
  const int* own = ids + (size_t)t0 * k;
  int e_of[kOwn];
#pragma unroll
  for (int i = 0; i < kOwn; ++i) e_of[i] = tid + i * kSlotThreads < pairs ? own[tid + i * kSlotThreads] : -1;
  const int q_sum = blockIdx.x + (tid >> 5) * gridDim.x;      // sums of p: a warp of the grid per four experts
  float4 p_sum = make_float4(0.f, 0.f, 0.f, 0.f);
  if (q_sum < quads) {
#pragma unroll 8
    for (int r = lane; r < chunks; r += 32) {
      const float4 v = *reinterpret_cast<const float4*>(psum + (size_t)r * E4 + q_sum * 4);
      p_sum.x += v.x; p_sum.y += v.y; p_sum.z += v.z; p_sum.w += v.w;
    }
  }
  {
    const int q = tid % quads, r0 = tid / quads;
    int4 sum = make_int4(0, 0, 0, 0);
    if (r0 < lanes) {
#pragma unroll 8
      for (int r = r0; r < before; r += lanes) {
        const int4 v = *reinterpret_cast<const int4*>(hist + (size_t)r * E4 + q * 4);
        sum.x += v.x; sum.y += v.y; sum.z += v.z; sum.w += v.w;
      }
      *reinterpret_cast<int4*>(&s_part[(r0 * quads + q) * 4]) = sum;
    }
  }
  __syncthreads();
  auto each_pair = [&](auto visit) {
#pragma unroll
    for (int i = 0; i < kOwn; ++i)
      if (tid + i * kSlotThreads < pairs) visit(tid + i * kSlotThreads, e_of[i]);
    for (int p = tid + kOwn * kSlotThreads; p < pairs; p += kSlotThreads) visit(p, own[p]);
  };
  each_pair([&](int p, int e) {
    if (e >= 0 && e < E) atomicOr(&s_mask[(p / k) >> 5][e], 1u << ((p / k) & 31));
  });
  int run = 0;
  if (tid < E)
    for (int r = 0; r < min(lanes, before); ++r) run += s_part[r * E4 + tid];
  __syncthreads();
  if (tid < E) {
    for (int w = 0; w < W; ++w) {
      s_part[w * kMaxExperts + tid] = run;
      run += __popc(s_mask[w][tid]);
    }
    if (blockIdx.x == gridDim.x - 1) counts[tid] = run;
  }
  __syncthreads();
  each_pair([&](int p, int e) {
    const int tok = p / k;
    int s = -1;
    if (e >= 0 && e < E) {
      s = s_part[(tok >> 5) * kMaxExperts + e] + __popc(s_mask[tok >> 5][e] & ((1u << (tok & 31)) - 1u));
      if (s >= capacity) s = -1;
    }
    slot[(size_t)t0 * k + p] = s;
  });
  for (int q = q_sum; q < quads; q += gridDim.x * (kSlotThreads / 32)) {
    if (q != q_sum) {                                         // (few CTAs: few chunks as well)
      p_sum = make_float4(0.f, 0.f, 0.f, 0.f);
      for (int r = lane; r < chunks; r += 32) {
        const float4 v = *reinterpret_cast<const float4*>(psum + (size_t)r * E4 + q * 4);
        p_sum.x += v.x; p_sum.y += v.y; p_sum.z += v.z; p_sum.w += v.w;
      }
    }
    const float out[4] = {warp_sum(p_sum.x), warp_sum(p_sum.y), warp_sum(p_sum.z), warp_sum(p_sum.w)};
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (lane == i && q * 4 + i < E) prob_sum[q * 4 + i] = out[i];
  }
}

// dl of a token.  With w = scale * what the weights are without it, D = sum over the chosen of (w / scale) dw:
//   renormalised: G_i = w_i (dw_i - D) for the chosen i;  else G_i = w_i dw_i (softmax: and -p_e scale D for all e)
//   dl_e = f_e (G_e + p_e (q_e - sum p q)),  f = 1 (softmax) or 1 - s_e (sigmoid)
template <typename T, int C>
__global__ void __launch_bounds__(kWarps * 32)
route_bwd_kernel(const __grid_constant__ RouteArgs a, const float* __restrict__ dw, const float* __restrict__ dprob,
                 T* __restrict__ dlogits) {
  __shared__ __align__(16) float s_row[kWarps][32 * C];
  grid_dependency_launch();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int first = lane * C, left = min(max(a.E - first, 0), C);
  float coef[C];
#pragma unroll
  for (int j = 0; j < C; ++j) coef[j] = dprob != nullptr && j < left ? dprob[first + j] : 0.f;
  float next_l[C], next_w = 0.f, next_g = 0.f;
  int next_id = -1;
  auto fetch = [&](int t) {
    load_row<T, C>(reinterpret_cast<const T*>(a.logits) + (size_t)t * a.ld + first, a.vectors, left, next_l);
    if (lane < a.k) {
      next_id = a.ids[(size_t)t * a.k + lane];
      next_w = a.w[(size_t)t * a.k + lane];
      if (dw != nullptr) next_g = dw[(size_t)t * a.k + lane];
    }
  };
  const int stride = gridDim.x * kWarps, start = blockIdx.x * kWarps + warp;
  constexpr bool kAhead = C >= 8;
  if (kAhead && start < a.tokens) fetch(start);
  for (int t = start; t < a.tokens; t += stride) {
    if (!kAhead) fetch(t);
    float l[C];
#pragma unroll
    for (int j = 0; j < C; ++j) l[j] = next_l[j];
    const int id = next_id;
    const float w = next_w, g = id >= 0 ? next_g : 0.f;
    if (kAhead && a.tokens - t > stride) fetch(t + stride);
#pragma unroll
    for (int j = 0; j < C; ++j) s_row[warp][place_of<C>(lane, j)] = 0.f;
    const float wd = warp_sum(id >= 0 ? w * g : 0.f);         // scale * D
    const float grad = a.renormalize ? w * (g - __fdividef(wd, a.scale)) : w * g;
    __syncwarp();
    if (id >= 0 && id < a.E) s_row[warp][place_of<C>(id / C, id % C)] = grad;
    unsigned bad = 0u;
    bool nan;
    const float top_l = top_logit<C>(l, a.sigmoid, bad, nan);
    Scores<C> s;
    s.set(l, a.sigmoid, top_l);
    float p[C], pq = 0.f;
#pragma unroll
    for (int j = 0; j < C; ++j) { p[j] = s.part[j] * s.inv; pq += p[j] * coef[j]; }
    pq = warp_sum(pq);
    const float all = !a.renormalize && !a.sigmoid ? wd : 0.f;
    __syncwarp();
    Row<T, C> out;
#pragma unroll
    for (int j = 0; j < C; ++j) {
      const float f = a.sigmoid ? __fdividef(1.f, 1.f + __expf(l[j])) : 1.f;
      const float v = f * (s_row[warp][place_of<C>(lane, j)] + p[j] * (coef[j] - pq - all));
      out.v[j] = from_f<T>(j >= left ? 0.f : nan ? __int_as_float(0x7fffffff) : v);
    }
    T* to = dlogits + (size_t)t * a.ld;
    if (a.vectors) {
      if (first < a.ld) *reinterpret_cast<Row<T, C>*>(to + first) = out;
    } else {
#pragma unroll
      for (int j = 0; j < C; ++j)
        if (first + j < a.ld) to[first + j] = out.v[j];
    }
    for (int e = 32 * C + lane; e < a.ld; e += 32) to[e] = from_f<T>(0.f);
    __syncwarp();
  }
}

bool fill(RouteArgs& a, const void* logits, int ld, int size, int tokens, int E, int k, int sigmoid, int renormalize,
          float scale, int* c) {
  if (E < 1 || E > kMaxExperts || k < 1 || k > kMaxChoices || k > E || ld < E || tokens < 1 || logits == nullptr) return false;
  if ((long long)tokens * k > 0x7fffffffLL) return false;
  a.logits = logits;
  a.ld = ld; a.tokens = tokens; a.E = E; a.k = k;
  a.E4 = (E + 3) / 4 * 4;
  a.sigmoid = sigmoid != 0; a.renormalize = renormalize != 0; a.scale = scale;
  a.rows = rows_of(tokens);
  int C = 1;
  while (32 * C < E) C *= 2;
  *c = C;
  // rows of whole lanes at addresses that a lane's values can be moved at in one piece (or in pieces of 16 bytes)
  const int piece = C * size < 16 ? C * size : 16;
  a.vectors = ld % C == 0 && (long long)ld * size % piece == 0 && reinterpret_cast<uintptr_t>(logits) % piece == 0;
  return true;
}

template <typename T>
int forward(const RouteArgs& a, int C, int chunks, cudaStream_t s) {
  constexpr int threads = kWarps * 32;
  if (C == 1) route_kernel<T, 1><<<chunks, threads, 0, s>>>(a);
  else if (C == 2) route_kernel<T, 2><<<chunks, threads, 0, s>>>(a);
  else if (C == 4) route_kernel<T, 4><<<chunks, threads, 0, s>>>(a);
  else if (C == 8) route_kernel<T, 8><<<chunks, threads, 0, s>>>(a);
  else route_kernel<T, 16><<<chunks, threads, 0, s>>>(a);
  return (int)cudaGetLastError();
}
template <typename T>
int backward(const RouteArgs& a, int C, const float* dw, const float* dprob, void* dlogits, cudaStream_t s) {
  constexpr int threads = kWarps * 32;
  // (8 and 16 experts per lane: as many CTAs as an SM holds, each token's loads a token ahead; 16384 tokens of 256 13.1 -> 10.2 us.
  // Fewer: as many warps as there are tokens; 128 experts 6.5 us, with five CTAs per SM and the loads ahead 6.9)
  const int want = (a.tokens + kWarps - 1) / kWarps, most = 148 * (C == 16 ? 2 : C == 8 ? 4 : 32), grid = want < most ? want : most;
  T* d = reinterpret_cast<T*>(dlogits);
  if (C == 1) route_bwd_kernel<T, 1><<<grid, threads, 0, s>>>(a, dw, dprob, d);
  else if (C == 2) route_bwd_kernel<T, 2><<<grid, threads, 0, s>>>(a, dw, dprob, d);
  else if (C == 4) route_bwd_kernel<T, 4><<<grid, threads, 0, s>>>(a, dw, dprob, d);
  else if (C == 8) route_bwd_kernel<T, 8><<<grid, threads, 0, s>>>(a, dw, dprob, d);
  else route_bwd_kernel<T, 16><<<grid, threads, 0, s>>>(a, dw, dprob, d);
  return (int)cudaGetLastError();
}

}  // namespace

// Words of scratch of dd_route_fwd (a multiple of 4).
DD_API int dd_route_words(int tokens, int E) {
  if (tokens < 1 || E < 1 || E > kMaxExperts) return 0;
  return 2 * ((tokens - 1) / rows_of(tokens) + 1) * ((E + 3) / 4 * 4);
}

// A call, packed by the caller (ctypes takes longer for twenty arguments than a launch does).  logits [tokens, ld], the first E
// columns (dtype 0 bf16, 1 fp16, 2 fp32); bias [E] fp32 or null; ids, w, slot [tokens * k]; counts, prob_sum [E]; scratch:
// `words` words, dd_route_words or more, 16-byte aligned.
struct RouteCall {
  const void* logits;
  const float* bias;
  int* ids;
  float* w;
  int *slot, *counts;
  float* prob_sum;
  int* scratch;
  long long words;
  int ld, dtype, tokens, E, k, capacity, groups, top_groups, group_sum, sigmoid, renormalize;
  float scale;
};
static_assert(sizeof(RouteCall) == 9 * 8 + 12 * 4, "packed without holes");

DD_API int dd_route_fwd(const void* packed, int bytes, void* stream) {
  RouteCall c;
  if (packed == nullptr || bytes != (int)sizeof c) return DD_ERR_BAD_ARG;
  memcpy(&c, packed, sizeof c);
  RouteArgs a = {};
  int C;
  const int size = c.dtype == 2 ? 4 : 2;
  if (c.dtype < 0 || c.dtype > 2 || !fill(a, c.logits, c.ld, size, c.tokens, c.E, c.k, c.sigmoid, c.renormalize, c.scale, &C))
    return DD_ERR_BAD_ARG;
  if (c.groups < 1 || c.groups > kMaxGroups || c.E % c.groups != 0 || c.top_groups < 1 || c.top_groups > c.groups)
    return DD_ERR_BAD_ARG;
  if (c.ids == nullptr || c.w == nullptr || c.slot == nullptr || c.counts == nullptr || c.prob_sum == nullptr ||
      c.scratch == nullptr)
    return DD_ERR_BAD_ARG;
  if (reinterpret_cast<uintptr_t>(c.scratch) % 16 != 0) return DD_ERR_ALIGN;
  const int chunks = (c.tokens - 1) / a.rows + 1;
  if (c.words < 2LL * chunks * a.E4) return DD_ERR_BAD_ARG;
  a.bias = c.bias;
  a.groups = c.top_groups == c.groups ? 1 : c.groups;         // (all groups: no choice among them)
  a.top_groups = c.top_groups; a.size = c.E / c.groups; a.group_sum = c.group_sum != 0;
  a.by_logit = c.bias == nullptr && !(a.groups > 1 && a.group_sum && a.size > 1);
  const int lanes = a.size / C;
  a.lanes = a.size % C == 0 && (lanes & (lanes - 1)) == 0 ? lanes : 0;
  a.ids = c.ids; a.w = c.w;
  a.hist = c.scratch;
  a.psum = reinterpret_cast<float*>(c.scratch + (size_t)chunks * a.E4);
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  const int e = c.dtype == 0   ? forward<__nv_bfloat16>(a, C, chunks, s)
                : c.dtype == 1 ? forward<__half>(a, C, chunks, s)
                               : forward<float>(a, C, chunks, s);
  if (e) return e;
  const int per_cta = kMostRows / a.rows;
  return launch_ahead(route_slot_kernel, dim3((chunks - 1) / per_cta + 1), dim3(kSlotThreads), 0, s, true, (const int*)c.ids,
                      c.tokens, c.k, c.E, a.E4, c.capacity, (const int*)a.hist, (const float*)a.psum, chunks, a.rows, per_cta,
                      c.counts, c.prob_sum, c.slot);
}

// dlogits [tokens, ld] from the gradients of w (dw [tokens, k], or null) and of prob_sum (dprob [E], or null).
DD_API int dd_route_bwd(const void* logits, int ld, int dtype, int tokens, int E, int k, int sigmoid, int renormalize,
                        float scale, const int* ids, const float* w, const float* dw, const float* dprob, void* dlogits,
                        void* stream) {
  RouteArgs a = {};
  int C;
  const int size = dtype == 2 ? 4 : 2;
  if (dtype < 0 || dtype > 2 || !fill(a, logits, ld, size, tokens, E, k, sigmoid, renormalize, scale, &C)) return DD_ERR_BAD_ARG;
  if (ids == nullptr || w == nullptr || dlogits == nullptr) return DD_ERR_BAD_ARG;
  if (reinterpret_cast<uintptr_t>(dlogits) % 16 != 0) return DD_ERR_ALIGN;
  a.ids = const_cast<int*>(ids);
  a.w = const_cast<float*>(w);
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  if (dtype == 0) return backward<__nv_bfloat16>(a, C, dw, dprob, dlogits, s);
  if (dtype == 1) return backward<__half>(a, C, dw, dprob, dlogits, s);
  return backward<float>(a, C, dw, dprob, dlogits, s);
}
