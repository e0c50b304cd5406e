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
};

__device__ __forceinline__ double warp_max(double v) {
  for (int o = 16; o > 0; o >>= 1) v = fmax(v, __shfl_xor_sync(0xffffffffu, v, o));
  return v;
}
__device__ __forceinline__ double warp_sum(double v) {
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// A warp a token; lane L holds experts L, L + 32, ...: PER of them. Scores are in 64-bit: in 32, experts whose scores differ by less than a
// rounding would be told apart by it.
template <int PER>
__global__ void __launch_bounds__(128) route_kernel(const Routing r) {
  sb::grid_launch_dependents();
  sb::grid_dependency_wait();
  const int row = blockIdx.x * 4 + (threadIdx.x >> 5), lane = threadIdx.x & 31;
  if (row >= r.n) return;
  const float* z = r.logits + row * r.ldz;
  double s[PER], c[PER];
  bool open[PER];
  double top_logit = -INFINITY;
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    const int e = lane + 32 * i;
    const float v = e < r.E ? fminf(z[e], FLT_MAX) : -INFINITY;       // (fminf(NaN, x) = x: NaN is looked for in the logit itself)
    open[i] = e < r.E && z[e] > -INFINITY;
    s[i] = v;
    if (open[i]) top_logit = fmax(top_logit, s[i]);
  }
  if (r.softmax) {
    top_logit = warp_max(top_logit);
    double sum = 0.0;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      s[i] = open[i] ? exp(s[i] - top_logit) : 0.0;
      sum += s[i];
    }
    sum = warp_sum(sum);
#pragma unroll
    for (int i = 0; i < PER; ++i) s[i] = sum > 0.0 ? s[i] / sum : 0.0;
  } else {
#pragma unroll
    for (int i = 0; i < PER; ++i) s[i] = open[i] ? 1.0 / (1.0 + exp(-s[i])) : 0.0;
  }
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    const int e = lane + 32 * i;
    c[i] = s[i];
    if (open[i] && r.bias != nullptr) {
      const float b = r.bias[e];
      open[i] = b > -INFINITY;
      c[i] += static_cast<double>(b);
    }
  }
  if (r.groups > 1) {
    const int size = r.E / r.groups;
    double mine = -INFINITY;                  // lane g: the score of group g
    for (int g = 0; g < r.groups; ++g) {
      double a = -INFINITY, b = -INFINITY;    // the two largest of the group
#pragma unroll
      for (int i = 0; i < PER; ++i) {
        const int e = lane + 32 * i;
        if (open[i] && e >= g * size && e < (g + 1) * size) {
          if (c[i] > a) b = a, a = c[i];
          else if (c[i] > b) b = c[i];
        }
      }
      for (int o = 16; o > 0; o >>= 1) {
        const double oa = __shfl_xor_sync(0xffffffffu, a, o), ob = __shfl_xor_sync(0xffffffffu, b, o);
        b = fmax(fmin(a, oa), fmax(b, ob));
        a = fmax(a, oa);
      }
      if (lane == g) mine = r.group_best > 1 && b > -INFINITY ? a + b : a;
    }
    int before = 0;                           // groups that come before this lane's
    for (int g = 0; g < r.groups; ++g) {
      const double other = __shfl_sync(0xffffffffu, mine, g);
      before += other > mine || (other == mine && g < lane);
    }
    const unsigned kept = __ballot_sync(0xffffffffu, lane < r.groups && before < r.top_groups);
#pragma unroll
    for (int i = 0; i < PER; ++i)
      if (open[i]) open[i] = (kept >> ((lane + 32 * i) / size)) & 1u;
  }
  double sum = 0.0, kept_s = 0.0;
  int kept_e = -1;
  for (int k = 0; k < r.top; ++k) {
    double best = 0.0, score = 0.0;
    int at = 0x7fffffff;
#pragma unroll
    for (int i = 0; i < PER; ++i)
      if (open[i] && (at == 0x7fffffff || c[i] > best)) best = c[i], at = lane + 32 * i, score = s[i];
    for (int o = 16; o > 0; o >>= 1) {
      const double ob = __shfl_xor_sync(0xffffffffu, best, o), os = __shfl_xor_sync(0xffffffffu, score, o);
      const int oa = __shfl_xor_sync(0xffffffffu, at, o);
      if (oa != 0x7fffffff && (at == 0x7fffffff || ob > best || (ob == best && oa < at))) best = ob, at = oa, score = os;
    }
    if (at == 0x7fffffff) at = -1, score = 0.0;
#pragma unroll
    for (int i = 0; i < PER; ++i)
      if (at == lane + 32 * i) open[i] = false;
    sum += score;
    if (lane == k) kept_s = score, kept_e = at;      // (at most 32 choices)
  }
  const double factor = r.renormalise ? static_cast<double>(r.scale) / (sum + 1e-20) : static_cast<double>(r.scale);
  if (lane < r.top) {
    r.choice[static_cast<int64_t>(row) * r.top + lane] = kept_e;
    r.weights[static_cast<int64_t>(lane) * r.ldw + row] = static_cast<float>(kept_s * factor);
  }
}

int launch(const Routing& r, cudaStream_t st) {
  if (r.n < 0 || r.E < 1 || r.E > kMaxExperts || r.top < 1 || r.top > 32 || r.top > r.E || r.ldz < r.E || r.ldw < r.n)
    return sb::fail("route_experts: %d of %d experts (at most 32 of %d), %d tokens, rows of %lld logits, of %lld weights", r.top, r.E, kMaxExperts, r.n,
                    (long long)r.ldz, (long long)r.ldw);
  if (r.groups < 1 || r.groups > kMaxGroups || r.E % r.groups || r.top_groups < 1 || r.top_groups > r.groups || r.group_best < 1 || r.group_best > 2)
    return sb::fail("route_experts: %d of %d groups (at most %d) of %d experts, judged by their best %d (1 or 2)", r.top_groups, r.groups, kMaxGroups, r.E, r.group_best);
  if (r.top > r.top_groups * (r.E / r.groups)) return sb::fail("route_experts: %d experts of %d groups of %d", r.top, r.top_groups, r.E / r.groups);
  if (r.n == 0) return 0;
  const dim3 grid((r.n + 3) / 4), block(128);
  const int per = (r.E + 31) / 32;
  if (per <= 1) sb::launch_pdl(route_kernel<1>, grid, block, 0, st, r);
  else if (per <= 2) sb::launch_pdl(route_kernel<2>, grid, block, 0, st, r);
  else if (per <= 4) sb::launch_pdl(route_kernel<4>, grid, block, 0, st, r);
  else if (per <= 8) sb::launch_pdl(route_kernel<8>, grid, block, 0, st, r);
  else if (per <= 16) sb::launch_pdl(route_kernel<16>, grid, block, 0, st, r);
  else sb::launch_pdl(route_kernel<32>, grid, block, 0, st, r);
  return sb::check_launch("route_experts");
}

}  // namespace

// logits [n][ldz] float32, bias [E] float32 or null, choice [n][top] int32, weights [top][ldw] float32. score: 0 sigmoid, 1 softmax.
SB_EXPORT int sb_route_experts(const float* logits, int64_t ldz, const float* bias, int32_t* choice, float* weights, int64_t ldw, int n, int E, int top,
                               int score, int groups, int top_groups, int group_best, int renormalise, float scale, void* stream) {
  const Routing r = {logits, ldz, bias, choice, weights, ldw, n, E, top, groups, top_groups, group_best, score, renormalise, scale};
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
