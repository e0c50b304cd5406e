// Routing tokens to experts: from a router's logits to every token's experts and their weights.
//
// s = softmax(z) over the token's experts, or sigmoid(z) each; c = s + bias (a bias for balance, which takes part in the choice only). With
// groups (consecutive experts, all of one size), a group's score is the sum of its `group_best` (1 or 2) largest c, the `top_groups` groups with
// the largest score stay. Of the experts that stay, the `top` with the largest c are chosen, in that order; weight = s, divided by (the sum of
// the chosen s + 1e-20) if renormalised, times a scale. The smaller index wins among equals, of groups and of experts.
//
// An expert whose logit is -infinity or NaN, or whose bias is -infinity or NaN, is never chosen, and a group of such experts never stays; a token
// with fewer than `top` experts left gets -1 (and weight 0) in the places that remain. A logit of +infinity counts as the largest float.
#include <cfloat>

#include "common.cuh"
#include "step_ops.h"

SB_DEFINE_LAST_ERROR()

namespace {

constexpr int kMaxExperts = 1024;
constexpr int kMaxGroups = 32;

struct Routing {
  const float* logits;
  int64_t ldz;
  const float* bias;          // [E] or null
  int32_t* choice;            // [n][top]
  float* weights;             // [top][ldw]: pair k of token t at k ldw + t
  int64_t ldw;
  int n, E, top, groups, top_groups, group_best;
  int softmax, renormalise;
  float scale;
  int size;                   // experts of a group, and 2^32 / size rounded up: e / size = the upper half of e times it, for e and size below 2^11
  uint32_t inverse_size;
};
__device__ __forceinline__ int group_of(const Routing& r, int e) { return r.size == 1 ? e : __umulhi(e, r.inverse_size); }

// float -> a word whose unsigned order is the values' (no NaN comes here).
__device__ __forceinline__ uint32_t order_key(float v) {
  const uint32_t b = __float_as_uint(v);
  return (b & 0x80000000u) ? ~b : (b | 0x80000000u);
}
__device__ __forceinline__ float warp_max(float v) {
  for (int o = 16; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
  return v;
}
template <class T>
__device__ __forceinline__ T warp_sum(T v) {
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}
// e^(z - top): the difference with what its rounding dropped, so that far logits keep their relative accuracy too.
__device__ __forceinline__ float exp_difference(float z, float top) {
  const float d = z - top, back = d + top, dropped = (z - back) + ((back - d) - top);
  return fabsf(dropped) < 1.0f ? expf(d) * (1.0f + dropped) : expf(d);
}

__device__ __forceinline__ double sigmoid_64(float z) { return 1.0 / (1.0 + exp(-static_cast<double>(z))); }

// This lane's values of a row of E: places lane PER .. lane PER + PER - 1 (`other` beyond). VEC: the row begins at a 16-byte border.
template <int PER, bool VEC>
__device__ __forceinline__ void load_lane(const float* row, int E, int lane, float other, float* v) {
  if (VEC && (lane + 1) * PER <= E) {
#pragma unroll
    for (int i = 0; i < PER; i += 4) {
      const float4 a = *reinterpret_cast<const float4*>(row + lane * PER + i);
      v[i] = a.x, v[i + 1] = a.y, v[i + 2] = a.z, v[i + 3] = a.w;
    }
  } else {
#pragma unroll
    for (int i = 0; i < PER; ++i) v[i] = lane * PER + i < E ? row[lane * PER + i] : other;
  }
}

// The scores s of this lane's experts from their logits; bit i of the result: the logit allows a choice. T: double, or float, then of a softmax only.
template <class T, int PER>
__device__ __forceinline__ uint32_t scores(const Routing& r, const float* logits, T* s) {
  uint32_t open = 0;
  float v[PER];
  float top = -INFINITY;
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    if (logits[i] > -INFINITY) open |= 1u << i;              // (not NaN either)
    v[i] = fminf(logits[i], FLT_MAX);
    if ((open >> i) & 1u) top = fmaxf(top, v[i]);
  }
  if (sizeof(T) == 4 || r.softmax) {
    top = warp_max(top);
    T sum = 0;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      s[i] = 0;
      if ((open >> i) & 1u) {
        if constexpr (sizeof(T) == 8) s[i] = exp(static_cast<double>(v[i]) - static_cast<double>(top));
        else s[i] = exp_difference(v[i], top);
      }
      sum += s[i];
    }
    sum = warp_sum(sum);
#pragma unroll
    for (int i = 0; i < PER; ++i) s[i] = sum > 0 ? s[i] / sum : T(0);
  } else {
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const double all = sigmoid_64(v[i]);         // (of all: without branches they overlap)
      s[i] = (open >> i) & 1u ? all : 0.0;
    }
  }
  return open;
}

// Whether a lane's experts are of one group, and a group's lanes a power of two.
template <int PER>
__device__ __forceinline__ bool whole_groups(const Routing& r) {
  return r.size % PER == 0 && (r.size / PER & (r.size / PER - 1)) == 0;
}

template <int PER>
__device__ __forceinline__ int lanes_of_group(const Routing& r, bool whole) {
  if (whole) return __ffs(r.size / PER) - 1;
  int shift = 0;
  while ((2 << shift) * r.groups <= 32) ++shift;
  return shift;
}

// The experts whose groups stay, as bits. c: -infinity where an expert may not be chosen. held: the warp's own E values of shared memory. a, b: a
// lane's two largest c, if `given`. gap (of float): the score of the last group that stays minus the best that does not. 1 << shift neighbouring
// lanes look through a group.
template <class T, int PER>
__device__ __forceinline__ uint32_t keep_groups(const Routing& r, int lane, const T* c, T* held, T& gap, bool whole, int shift, bool given, T a, T b) {
  const int size = r.size;
  if (!given) {
    a = b = -INFINITY;
#pragma unroll
    for (int i = 0; i < PER; ++i)
      if (lane * PER + i < r.E) held[lane * PER + i] = c[i];
    __syncwarp();
    const int g = lane >> shift, share = 1 << shift;
    if (g < r.groups) {
      const T* from = held + g * size;
      for (int j = lane & (share - 1); j < size; j += share) {
        const T v = from[j];
        b = v > a ? a : (v > b ? v : b);
        a = v > a ? v : a;
      }
    }
  }
  for (int o = 1; o < 1 << shift; o <<= 1) {
    const T oa = __shfl_xor_sync(0xffffffffu, a, o), ob = __shfl_xor_sync(0xffffffffu, b, o);
    b = oa > a ? (a > ob ? a : ob) : (oa > b ? oa : b);
    a = oa > a ? oa : a;
  }
  a = __shfl_sync(0xffffffffu, a, (lane << shift) & 31), b = __shfl_sync(0xffffffffu, b, (lane << shift) & 31);      // lane g: group g's
  if (lane >= r.groups) a = b = -INFINITY;
  __syncwarp();
  T mine = a;
  if (r.group_best > 1 && b > static_cast<T>(-INFINITY)) {
    mine = a + b;
    if (sizeof(T) == 4) mine = fmax(mine, static_cast<T>(-FLT_MAX));      // (a sum beyond the floats is no empty group: those alone are -infinity)
  }
  int before = 0;                              // groups that come before this lane's
#pragma unroll 4
  for (int g = 0; g < r.groups; ++g) {
    const T other = __shfl_sync(0xffffffffu, mine, g);
    before += other > mine || (other == mine && g < lane);
  }
  const unsigned kept = __ballot_sync(0xffffffffu, lane < r.groups && before < r.top_groups);
  const unsigned last = __ballot_sync(0xffffffffu, lane < r.groups && before == r.top_groups - 1);
  const unsigned next = __ballot_sync(0xffffffffu, lane < r.groups && before == r.top_groups);
  const T score = __shfl_sync(0xffffffffu, mine, __ffs(last) - 1);
  gap = next != 0 ? score - __shfl_sync(0xffffffffu, mine, __ffs(next) - 1) : static_cast<T>(INFINITY);
  if (score == static_cast<T>(-INFINITY)) gap = INFINITY;       // (groups with nothing in them: it does not matter which)
  if (whole) return (kept >> (lane >> shift)) & 1u ? 0xffffffffu : 0u;
  uint32_t stay = 0;
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    const int g = group_of(r, lane * PER + i);
    if (g < 32 && ((kept >> g) & 1u)) stay |= 1u << i;
  }
  return stay;
}

__device__ __forceinline__ void write_row(const Routing& r, int row, int lane, int e, double weight) {
  if (lane < r.top) {
    r.choice[static_cast<int64_t>(row) * r.top + lane] = e;
    r.weights[static_cast<int64_t>(lane) * r.ldw + row] = static_cast<float>(weight);
  }
}

// A token in 64-bit.
template <int PER>
__device__ __noinline__ void route_row_64(const Routing& r, int row, int lane, double* held) {
  double s[PER], c[PER], gap;
  float z[PER], bias[PER];
  load_lane<PER, false>(r.logits + row * r.ldz, r.E, lane, -INFINITY, z);
#pragma unroll
  for (int i = 0; i < PER; ++i) bias[i] = r.bias != nullptr && lane * PER + i < r.E ? r.bias[lane * PER + i] : 0.0f;
  uint32_t open = scores<double, PER>(r, z, s);
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    if (!(bias[i] > -INFINITY)) open &= ~(1u << i);
    c[i] = s[i] + static_cast<double>(bias[i]);
  }
  if (r.groups > 1) {
    const bool whole = whole_groups<PER>(r);
    double a = -INFINITY, b = -INFINITY;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      if (!((open >> i) & 1u)) c[i] = -INFINITY;
      b = c[i] > a ? a : (c[i] > b ? c[i] : b);
      a = c[i] > a ? c[i] : a;
    }
    open &= keep_groups<double, PER>(r, lane, c, held, gap, whole, lanes_of_group<PER>(r, whole), whole, a, b);
  }
  double sum = 0.0, kept_s = 0.0;
  int kept_e = -1;
  for (int k = 0; k < r.top; ++k) {
    double best = 0.0, score = 0.0;
    int at = 0x7fffffff;
#pragma unroll
    for (int i = 0; i < PER; ++i)
      if (((open >> i) & 1u) && (at == 0x7fffffff || c[i] > best)) best = c[i], at = lane * PER + i, score = s[i];
    for (int o = 16; o > 0; o >>= 1) {
      const double ob = __shfl_xor_sync(0xffffffffu, best, o), os = __shfl_xor_sync(0xffffffffu, score, o);
      const int oa = __shfl_xor_sync(0xffffffffu, at, o);
      if (oa != 0x7fffffff && (at == 0x7fffffff || ob > best || (ob == best && oa < at))) best = ob, at = oa, score = os;
    }
    if (at == 0x7fffffff) at = -1, score = 0.0;
#pragma unroll
    for (int i = 0; i < PER; ++i)
      if (at == lane * PER + i) open &= ~(1u << i);
    sum += score;
    if (lane == k) kept_s = score, kept_e = at;      // (at most 32 choices)
  }
  write_row(r, row, lane, kept_e, r.renormalise ? kept_s * r.scale / (sum + 1e-20) : kept_s * r.scale);
}

// A key's value, without the bits that its place took. Below the lowest float's key: -infinity.
constexpr uint32_t kLowestKey = 0x00800000u;

// A row's largest logit and, in the order of `scores`, the 64-bit sum of its exponentials.
struct Softmax64 {
  float top;
  double sum;
};
template <int PER>
__device__ __noinline__ Softmax64 softmax_64(const float* logits, int E, int lane) {
  float z[PER], top = -INFINITY;
  load_lane<PER, false>(logits, E, lane, -INFINITY, z);
#pragma unroll
  for (int i = 0; i < PER; ++i)
    if (z[i] > -INFINITY) top = fmaxf(top, fminf(z[i], FLT_MAX));
  top = warp_max(top);
  double sum = 0.0;
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    const double all = exp(static_cast<double>(fminf(z[i], FLT_MAX)) - static_cast<double>(top));
    sum += z[i] > -INFINITY ? all : 0.0;
  }
  return {top, warp_sum(sum)};
}
// An expert's 64-bit score with its bias, as `route_row_64` has it.
__device__ __forceinline__ double score_64(const Routing& r, const float* logits, int e, const Softmax64& of) {
  const float v = fminf(logits[e], FLT_MAX);
  const double s = !r.softmax ? sigmoid_64(v) : of.sum > 0 ? exp(static_cast<double>(v) - static_cast<double>(of.top)) / of.sum : 0.0;
  return s + (r.bias != nullptr ? static_cast<double>(r.bias[e]) : 0.0);
}
template <int PER>
__device__ __forceinline__ float key_value(uint32_t key) {
  const uint32_t k = key & ~(PER - 1u);
  return key < kLowestKey ? -INFINITY : __uint_as_float((k & 0x80000000u) ? (k & 0x7FFFFFFFu) : ~k);
}

// By descending key: Batcher's merge exchanges.
template <int N, int P, int K>
__device__ __forceinline__ void merge_exchange(uint32_t* key) {
#pragma unroll
  for (int a = 0; a + K < N; ++a) {
    constexpr int kFirst = K % P;
    const int b = a + K;
    if (a >= kFirst && (a - kFirst) % (2 * K) < K && a / (2 * P) == b / (2 * P)) {
      const uint32_t low = min(key[a], key[b]);
      key[a] = max(key[a], key[b]), key[b] = low;
    }
  }
  if constexpr (K > 1) merge_exchange<N, P, K / 2>(key);
  else if constexpr (2 * P < N) merge_exchange<N, 2 * P, 2 * P>(key);
}
template <int N>
__device__ __forceinline__ void sort_descending(uint32_t* key) {
  if constexpr (N > 1) merge_exchange<N, 1, 1>(key);
}

// A warp a token. In 32-bit first, where a score is off by less than a known share of the largest: a sigmoid by 2^-20 (its approximated exponential is
// off by 2 + 1.2 |z| units in the last place, of which a quarter counts at most near and above 1/2, its division by two; 2^-16 where all scores
// are small), a softmax by PER + 16 times 2^-24 (PER + 4 additions, four units in the last place of the exponential, a division); a sum with a bias
// by 2^-23 of its size more, and a key by PER - 1 times that, whose last bits hold the place of the lane's expert. (The sizes of the two that are
// compared: what lies further down may be off by more, but lies further away by more than that.) Candidates that are closer to their
// neighbours than both can be off are taken on beyond the last that is chosen, until one is not, and ranked again by 64-bit scores, a candidate a lane;
// so are groups, if the last that stays is too close to the first that does not. What that does not settle (more than 32 candidates, a group whose
// third expert is as close to its second) is routed again in 64-bit as a whole. So the choice is that of 64-bit scores always, at the price of
// 32-bit ones. (One token in 64-bit takes 10 us, and of thousands one is always among the last.)
// 16,384 tokens of 256 experts in eight groups, eight chosen: everything in 64-bit 87 us, the close ones as a whole 30, so 18.7 (900 GB/s; issue slots
// bound it, 950 instructions a token, issued in 73% of the cycles: seven times the time of its bytes); one token 12.6 and 2.7; 8,192 of 160, six chosen of
// three groups of eight, 12.9 by sigmoids and 17.0 to 17.8 by softmax.
template <int PER>
__device__ __forceinline__ void route_row(const Routing& r, int row, int lane, const float* z, const float* bias, double* held, float* held_scores) {
  float c[PER], high_s = 0.0f;                   // c: -infinity if never to be chosen
  {
    float s[PER];
    uint32_t open = 0;
    if (r.softmax) {
      open = scores<float, PER>(r, z, s);
    } else {
#pragma unroll
      for (int i = 0; i < PER; ++i) s[i] = __fdividef(1.0f, 1.0f + __expf(fminf(-z[i], 80.0f)));      // (to choose by; a chosen one's weight is computed anew)
    }
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      c[i] = z[i] > -INFINITY && bias[i] > -INFINITY ? s[i] + bias[i] : -INFINITY;
      high_s = fmaxf(high_s, s[i]);
      held_scores[lane * PER + i] = r.softmax ? s[i] : z[i];
    }
  }
  high_s = __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(high_s)));      // (not negative: their bits are ordered as they are)
  const float near = 2.0f * high_s * (r.softmax ? (PER + 16) * 0x1p-24f : high_s > 0.125f ? 0x1p-20f : 0x1p-16f) + 0x1p-113f;      // (e^-80, where a sigmoid ends)
  constexpr float kShare = PER * 0x1p-23f;
  const bool grouped = r.groups > 1, whole = whole_groups<PER>(r);
  const float* logits = r.logits + row * r.ldz;
  Softmax64 of = {0.0f, -1.0};                   // (once it is needed)
  bool sure = true;
  uint32_t key[PER];                             // this lane's candidates, largest first: the order of c's bits, the last of them the place
#pragma unroll
  for (int i = 0; i < PER; ++i) key[i] = (order_key(c[i]) & ~(PER - 1u)) | i;
  if (grouped) {
    const int shift = lanes_of_group<PER>(r, whole);
    float a = 0.0f, b = 0.0f, gap, high_c = 0.0f;
    if (whole) {
      sort_descending<PER>(key);
      a = key_value<PER>(key[0]), b = PER > 1 ? key_value<PER>(key[PER > 1]) : -INFINITY;
      high_c = fmaxf(a > -INFINITY ? fabsf(a) : 0.0f, b > -INFINITY ? fabsf(b) : 0.0f);
    } else {
#pragma unroll
      for (int i = 0; i < PER; ++i)
        if (c[i] > -INFINITY) high_c = fmaxf(high_c, fabsf(c[i]));
    }
    uint32_t stay = keep_groups<float, PER>(r, lane, c, reinterpret_cast<float*>(held), gap, whole, shift, whole, a, b);
    high_c = __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(high_c)));
    if (!(gap > 2.0f * near + 4.0f * kShare * high_c)) {           // (sums of two)
      // the groups again by 64-bit sums of the lanes' largest two, if no lane's third is too close to its second
      float high[3] = {-INFINITY, -INFINITY, -INFINITY};
      int at[2] = {0, 0};
      if (whole) {
        high[0] = a, high[1] = b, high[2] = PER > 2 ? key_value<PER>(key[PER > 2 ? 2 : 0]) : -INFINITY;
        at[0] = lane * PER + static_cast<int>(key[0] & (PER - 1u)), at[1] = lane * PER + static_cast<int>(key[PER > 1] & (PER - 1u));
      } else {
        const float* from = reinterpret_cast<float*>(held);
        const int g = lane >> shift, share = 1 << shift;
#pragma unroll 1
        for (int e = g * r.size + (lane & (share - 1)); e < (g + 1) * r.size && g < r.groups; e += share) {
          const float v = from[e];
          if (v > high[0]) high[2] = high[1], high[1] = high[0], at[1] = at[0], high[0] = v, at[0] = e;
          else if (v > high[1]) high[2] = high[1], high[1] = v, at[1] = e;
          else if (v > high[2]) high[2] = v;
        }
      }
      const bool clear = high[2] == -INFINITY || high[1] - high[2] > near + kShare * (fabsf(high[1]) + fabsf(high[2]));
      sure = __all_sync(0xffffffffu, clear);
      if (r.softmax) of = softmax_64<PER>(logits, r.E, lane);
      const double a64 = high[0] > -INFINITY ? score_64(r, logits, at[0], of) : -INFINITY, b64 = high[1] > -INFINITY ? score_64(r, logits, at[1], of) : -INFINITY;
      double gap_64;
      stay = keep_groups<double, PER>(r, lane, nullptr, nullptr, gap_64, whole, shift, true, fmax(a64, b64), fmin(a64, b64));
    }
#pragma unroll
    for (int i = 0; i < PER; ++i)
      if (whole ? stay == 0u : !((stay >> i) & 1u)) key[i] = 0u;
  }
  if (!grouped || !whole) sort_descending<PER>(key);
  __syncwarp();
  float before = INFINITY;
  int kept_e = -1, count = 0;
  bool close = false;
  while (sure) {
    const uint32_t best = __reduce_max_sync(0xffffffffu, key[0]);
    if (best < kLowestKey) break;
    const float value = key_value<PER>(best);
    const bool apart = count == 0 || before - value > near + kShare * (fabsf(before) + fabsf(value));
    if (count >= r.top && apart) break;
    close = close || !apart;
    if (count == 32) sure = false;
    const int owner = __ffs(__ballot_sync(0xffffffffu, key[0] == best)) - 1;
    if (lane == count) kept_e = owner * PER + static_cast<int>(best & (PER - 1u));
    if (lane == owner) {
#pragma unroll
      for (int i = 0; i + 1 < PER; ++i) key[i] = key[i + 1];
      key[PER - 1] = 0;
    }
    before = value, ++count;
  }
  if (sure && close) {
    if (r.softmax && of.sum < 0.0) of = softmax_64<PER>(logits, r.E, lane);
    const double mine = kept_e >= 0 ? score_64(r, logits, kept_e, of) : -INFINITY;
    int rank = 0, from = 0;
    for (int j = 0; j < count; ++j) {
      const double other = __shfl_sync(0xffffffffu, mine, j);
      const int e = __shfl_sync(0xffffffffu, kept_e, j);
      rank += other > mine || (other == mine && e < kept_e);
    }
    for (int j = 0; j < count; ++j)
      if (__shfl_sync(0xffffffffu, rank, j) == lane) from = j;
    const int e = __shfl_sync(0xffffffffu, kept_e, from);
    kept_e = lane < min(count, r.top) ? e : -1;
  }
  float kept_s = 0.0f, sum = 0.0f;
  if (kept_e >= 0) {
    kept_s = held_scores[kept_e];
    if (!r.softmax) kept_s = kept_s < -80.0f ? expf(kept_s) : 1.0f / (1.0f + expf(-fminf(kept_s, FLT_MAX)));      // (e^88 and more would leave nothing of it)
  }
  if (r.renormalise) sum = warp_sum(kept_s);
  if (r.renormalise && kept_e >= 0 && sum < 0x1p-50f) sure = false;      // (scores below the smallest floats count where all are)
  sure = __all_sync(0xffffffffu, sure);
  if (!sure) {
    __syncwarp();
    return route_row_64<PER>(r, row, lane, held);
  }
  write_row(r, row, lane, kept_e, r.renormalise ? kept_s * (r.scale / (sum + 1e-20f)) : kept_s * r.scale);
}

constexpr int kWarps = 4;
template <int PER, bool VEC>
__global__ void __launch_bounds__(32 * kWarps, PER <= 8 ? 8 : 1) route_kernel(const Routing r) {
  __shared__ double held_s[kWarps][32 * PER];       // (64-bit scores, or 32-bit sums with the bias in front of 32-bit scores)
  sb::grid_launch_dependents();
  const int lane = threadIdx.x & 31, row = blockIdx.x * kWarps + (threadIdx.x >> 5);
  sb::grid_dependency_wait();
  if (row >= r.n) return;
  double* held = held_s[threadIdx.x >> 5];
  float bias[PER], z[PER];
#pragma unroll
  for (int i = 0; i < PER; ++i) bias[i] = 0.0f;
  load_lane<PER, VEC>(r.logits + row * r.ldz, r.E, lane, -INFINITY, z);
  if (r.bias != nullptr) load_lane<PER, VEC>(r.bias, r.E, lane, 0.0f, bias);
  route_row<PER>(r, row, lane, z, bias, held, reinterpret_cast<float*>(held) + 32 * PER);
}

int launch(Routing r, cudaStream_t st) {
  if (r.n < 0 || r.E < 1 || r.E > kMaxExperts || r.top < 1 || r.top > 32 || r.top > r.E || r.ldz < r.E || r.ldw < r.n)
    return sb::fail("route_experts: %d of %d experts (at most 32 of %d), %d tokens, rows of %lld logits, of %lld weights", r.top, r.E, kMaxExperts, r.n,
                    (long long)r.ldz, (long long)r.ldw);
  if (r.groups < 1 || r.groups > kMaxGroups || r.E % r.groups || r.top_groups < 1 || r.top_groups > r.groups || r.group_best < 1 || r.group_best > 2)
    return sb::fail("route_experts: %d of %d groups (at most %d) of %d experts, judged by their best %d (1 or 2)", r.top_groups, r.groups, kMaxGroups, r.E, r.group_best);
  if (r.top > r.top_groups * (r.E / r.groups)) return sb::fail("route_experts: %d experts of %d groups of %d", r.top, r.top_groups, r.E / r.groups);
  if (r.n == 0) return 0;
  r.size = r.E / r.groups, r.inverse_size = r.size == 1 ? 0u : static_cast<uint32_t>((0x100000000ull + r.size - 1) / r.size);
  const int per = (r.E + 31) / 32;
  const dim3 grid((r.n + kWarps - 1) / kWarps), block(32 * kWarps);
  const bool vec = r.ldz % 4 == 0 && ((reinterpret_cast<uintptr_t>(r.logits) | reinterpret_cast<uintptr_t>(r.bias)) & 15) == 0;
  if (per <= 1) sb::launch_pdl(route_kernel<1, false>, grid, block, 0, st, r);
  else if (per <= 2) sb::launch_pdl(route_kernel<2, false>, grid, block, 0, st, r);
  else if (per <= 4) vec ? sb::launch_pdl(route_kernel<4, true>, grid, block, 0, st, r) : sb::launch_pdl(route_kernel<4, false>, grid, block, 0, st, r);
  else if (per <= 8) vec ? sb::launch_pdl(route_kernel<8, true>, grid, block, 0, st, r) : sb::launch_pdl(route_kernel<8, false>, grid, block, 0, st, r);
  else if (per <= 16) vec ? sb::launch_pdl(route_kernel<16, true>, grid, block, 0, st, r) : sb::launch_pdl(route_kernel<16, false>, grid, block, 0, st, r);
  else vec ? sb::launch_pdl(route_kernel<32, true>, grid, block, 0, st, r) : sb::launch_pdl(route_kernel<32, false>, grid, block, 0, st, r);
  return sb::check_launch("route_experts");
}

}  // namespace

// logits [n][ldz] float32, bias [E] float32 or null, choice [n][top] int32, weights [top][ldw] float32. score: 0 sigmoid, 1 softmax.
typedef struct SbRouteCall {
  const float* logits;
  int64_t ldz;
  const float* bias;
  int32_t* choice;
  float* weights;
  int64_t ldw;
  int32_t n, experts, top, score, groups, top_groups, group_best, renormalise;
  float scale;
} SbRouteCall;

SB_EXPORT int sb_route_experts(const SbRouteCall* call, void* stream) {
  const SbRouteCall c = *call;
  const Routing r = {c.logits, c.ldz, c.bias, c.choice, c.weights, c.ldw, c.n, c.experts, c.top, c.groups, c.top_groups, c.group_best, c.score,
                     c.renormalise, c.scale};
  return launch(r, static_cast<cudaStream_t>(stream));
}

// i: 0 logits, 1 ldz, 2 bias (or 0), 3 choice [n][top], 4 weights [top][n], 5 experts, 6 top, 7 score, 8 groups, 9 top_groups, 10 group_best,
// 11 renormalise. f: 0 scale
SB_EXPORT int sb_op_route_experts(const SbOp* op, const SbStep* s, void* stream) {
  using namespace sbstep;
  if (s->n <= 0) return SB_OP_SKIPPED;
  const Routing r = {ptr<float>(op->i[0]), op->i[1], ptr<float>(op->i[2]), ptr<int32_t>(op->i[3]), ptr<float>(op->i[4]), s->n, s->n, (int)op->i[5],
                     (int)op->i[6], (int)op->i[8], (int)op->i[9], (int)op->i[10], (int)op->i[7], (int)op->i[11], (float)op->f[0]};
  return launch(r, static_cast<cudaStream_t>(stream)) != 0 ? SB_OP_FAILED : SB_OP_LAUNCHED;
}
