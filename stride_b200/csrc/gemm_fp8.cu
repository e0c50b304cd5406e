// Linear layers with 8-bit weights, out = x . W^T: W in e4m3 with one float32 scale per block of 128 rows and 128 columns, x quantised on the
// way in, one scale per token and block of 128 columns.
//
// `quantize_kernel`: with a = max |x_j| of a token's block, s = 2^e, e = max(ceil(log2(a / 448)), -100) (448 is the largest e4m3 value) and
// q_j = e4m3(x_j / s), to nearest even. A power of two, because then x / s and q s are exact: what is lost is the one rounding to e4m3, the
// same however it is computed (a scale a / 448 uses up to one more bit of the largest elements' range, but rounds the quotient twice). A block
// with an infinity or a NaN gets the scale NaN, so the token's whole result is NaN.
//
// The product: y[t, m] = sum over blocks b of columns of s[t, b] w_s[m / 128, b] (sum of q w over the block). The inner sum runs on the tensor cores
// (tcgen05.mma kind::f8f6f4, float32 accumulators): every block of 128 columns, one row of the 128-byte swizzle, is a fresh accumulator in
// tensor memory, of which there is a ring; the epilogue's warps take it from there and add it, times its two scales, to the tile's sum in
// registers, one fused multiply-add an element, in 32 bits. That addition is what bounds large products beside the power limit (one multiply-add an
// element and block beside 128 products on the tensor cores: 4,096 tokens through 28,672 gate and up rows of 4,096 take 470 us in a burst of
// 20 calls, 2.05 PFLOP/s, and 510 to 560 in a long run of them, at the clock that the limit leaves; a trial without the additions 393 and 440), the
// weights' bytes the small ones. Times here are of the kernels in a row, in a recorded graph or a burst; a call among others from Python adds up to
// 3 us to short ones.
//
// K is cut into ranges, a function of the weight's shape alone (`fp8_ranges`): few weight tiles leave SMs without work. The sum of a range
// starts from zero, the ranges are added in ascending order. With few tokens, and with more where that takes fewer rounds, the ranges are shared out
// among the CTAs of a cluster, which add up through distributed shared memory; else one CTA walks them all. So a token's bits depend neither on the
// step it is part of nor on the tile, nor on which of the forms made them:
//   `gemm_fp8_kernel`        up to 64 tokens: 128 weight rows by 16, 32 or 64 tokens; of 16 it may quantise its input itself
//   `gemm_fp8_token_kernel`  up to 128, and more where that takes fewer rounds: tokens are the product's rows
//   `gemm_fp8_pair_kernel`   many, and the experts': tokens are the product's rows, CTAs or pairs of CTAs walk the tiles
// An expert's products are those of a tile of its rows (`expert_order_kernel` sorts the choices by expert).
#include <algorithm>
#include <type_traits>

#include "gemm_tc_tile.cuh"
#include "step_ops.h"

SB_DEFINE_LAST_ERROR()

namespace {

using namespace sb::tc5;
using sb::gemm_tile::bf16;
using sb::gemm_tile::Gate;
using sb::gemm_tile::gated_product;
using sb::gemm_tile::kGateSilu;
using sb::gemm_tile::silu_fast;

// (No kernel here promises that its inputs are read by it alone (__restrict__): the compiler may take loads of such an input in front of the wait
// for the kernel that writes it.)
constexpr int kBlock = 128;            // columns (and weight rows) of a scale
constexpr int kStageA = kBlock * 128;  // bytes of a weight tile's block
constexpr int kMaxStages = 8;
constexpr int kMaxRanges = 4;
constexpr int kSmemBudget = 200 * 1024;

enum Epilogue { kStore = 0, kAdd = 1, kGated = 2 };

// ------------------------------------------------------------------ quantisation
// The scale's exponent: amax = 1.m 2^E -> E - 8 if 1.m <= 1.75 (448 = 1.75 2^8), else E - 7; never below -100.
__device__ __forceinline__ int scale_exponent(uint32_t amax_bits) {
  return max(static_cast<int>((amax_bits + 0x1FFFFFu) >> 23) - 127 - 8, -100);
}
__device__ __forceinline__ float power_of_two(int e) { return __uint_as_float(static_cast<uint32_t>(e + 127) << 23); }   // -126 <= e <= 127
__device__ __forceinline__ uint32_t e4m3x2(float lo, float hi) {
  uint16_t r;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %2, %1;" : "=h"(r) : "f"(lo), "f"(hi));
  return r;
}

// Eight columns of a row, k .. k + 7 of K (zeros behind). VEC: the row begins at a 16-byte border.
template <class T, bool VEC>
__device__ __forceinline__ void load8(const T* from, int k, int K, float* v) {
  if (VEC && k + 8 <= K) {
    if (sizeof(T) == 2) {
      const uint4 raw = *reinterpret_cast<const uint4*>(from);
      const uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
#pragma unroll
      for (int i = 0; i < 4; ++i) v[2 * i] = __uint_as_float(w[i] << 16), v[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u);
    } else {
      const float4 a = reinterpret_cast<const float4*>(from)[0], b = reinterpret_cast<const float4*>(from)[1];
      v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w, v[4] = b.x, v[5] = b.y, v[6] = b.z, v[7] = b.w;
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = k + i < K ? sb::widen(from[i]) : 0.0f;
  }
}

// x [n][ldx] -> q bytes [rows][ldq], scales [ceil(K / 128)][lds]. Sixteen lanes take a block of 128 columns of a row, a warp two blocks; the CTA's
// warps take neighbouring rows, whose scales lie side by side. place (or null): a row is stored `copies` times, as rows place[row copies + i] (left out where that is negative).
template <class T, bool VEC>
__global__ void __launch_bounds__(256) quantize_kernel(const T* x, int64_t ldx, const int32_t* place,
                                                       int copies, int n, int K, int blocks, uint8_t* q, int64_t ldq,
                                                       float* scales, int64_t lds) {
  sb::grid_launch_dependents();
  sb::grid_dependency_wait();
  const int row = blockIdx.x * 8 + (threadIdx.x >> 5), lane = threadIdx.x & 31, b = blockIdx.y * 2 + (lane >> 4), k = b * kBlock + (lane & 15) * 8;
  if (row >= n) return;
  alignas(16) float v[8];
  if constexpr (VEC || sizeof(T) == 2) {
    load8<T, VEC>(x + static_cast<int64_t>(row) * ldx + k, k, K, v);
  } else {
    // a column a lane at a time, then eight neighbours each from shared memory (2,055 rows of 4,023: 11.8 us, so 8.5; bfloat16 is no faster so)
    __shared__ __align__(16) float line[8][256];
    float* mine = line[threadIdx.x >> 5];
    const int first = blockIdx.y * 256, left = K - first;
    const T* from = x + static_cast<int64_t>(row) * ldx + first;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int c = lane + 32 * i;
      mine[c] = c < left ? from[c] : 0.0f;
    }
    __syncwarp();
#pragma unroll
    for (int i = 0; i < 8; i += 4) *reinterpret_cast<float4*>(v + i) = *reinterpret_cast<const float4*>(mine + 8 * lane + i);
  }
  uint32_t amax = 0;               // (the bit patterns of |x| are ordered as the values are, infinity and NaN above them)
#pragma unroll
  for (int i = 0; i < 8; ++i) amax = max(amax, __float_as_uint(v[i]) & 0x7FFFFFFFu);
#pragma unroll
  for (int o = 1; o < 16; o <<= 1) amax = max(amax, __shfl_xor_sync(0xffffffffu, amax, o));
  const bool finite = amax < 0x7F800000u;
  const int e = finite ? scale_exponent(amax) : 0;
  const float inverse = power_of_two(-e), scale = finite ? power_of_two(e) : __uint_as_float(0x7FC00000u);
  const uint32_t lo = e4m3x2(v[0] * inverse, v[1] * inverse) | (e4m3x2(v[2] * inverse, v[3] * inverse) << 16);
  const uint32_t hi = e4m3x2(v[4] * inverse, v[5] * inverse) | (e4m3x2(v[6] * inverse, v[7] * inverse) << 16);
  if (b >= blocks) return;
  for (int i = 0; i < copies; ++i) {
    const int at = place != nullptr ? place[static_cast<int64_t>(row) * copies + i] : row;
    if (at < 0) continue;
    uint8_t* to = q + static_cast<int64_t>(at) * ldq + k;
    if (k + 8 <= K) {
      *reinterpret_cast<uint2*>(to) = make_uint2(lo, hi);            // (rows of q start 16-byte aligned)
    } else {
      for (int j = 0; k + j < K; ++j) to[j] = static_cast<uint8_t>((j < 4 ? lo : hi) >> (8 * (j & 3)));
    }
    if ((lane & 15) == 0) scales[static_cast<int64_t>(b) * lds + at] = scale;
  }
}

// ------------------------------------------------------------------ the product
struct Fp8Params {
  void* out;                 // kStore: [n][ldo] of OUT; kAdd: float32 [n][ldo]; kGated: OUT [n][ldo]
  int64_t ldo;
  const float* x_scales;     // [blocks][ldxs]
  int64_t ldxs;
  const void* x;             // for the forms that quantise it themselves: float32 (x_f32) or bfloat16 [n][ldx], rows 16-byte aligned
  int64_t ldx;
  int x_f32, x_gathered;     // x_gathered: row i is token order[i]
  int quant_warps;           // how many of the warps quantise
  const float* w_scales;     // [blocks of rows][blocks]
  int n, M, K, blocks;       // M: rows of the weight (of one expert); kGated: gate rows, then up rows
  int half_rows;
  int scale_rows;            // blocks of rows of one expert's scales
  int ranges, range_blocks;  // K ranges and blocks of columns in each
  int split;                 // the ranges of a CTA, if they run on CTAs of their own; else 0
  int stages;
  int tiles_m, tiles_n, vec_out;      // (kernels that walk tiles; vec_out: the result takes 16-byte stores)
  const int32_t* tiles;      // experts: the list of `expert_order_kernel`; else null
  const int32_t* order;      // experts: row -> token
  const int32_t* choice;     // experts, few choices: every warp puts them in order itself (`FewChoices`), `tiles` and `order` are null
  int choices, top, experts; // with it
  float* z_scales;           // experts, gated products quantised by the epilogue: [blocks of features][ldxs]
  Gate gate;
  int* status;
};

__device__ __forceinline__ uint32_t instr_desc_e4m3(int n) {      // D float32, A and B e4m3, both K-major, M = 128
  return (1u << 4) | (static_cast<uint32_t>(n >> 3) << 17) | (static_cast<uint32_t>(kBlock >> 4) << 24);
}
// One block of 128 columns: four products of 32 columns (32 bytes of both operands' rows each) into a fresh accumulator, by one thread of a warp
// that is here as a whole, as it is for the signals behind them. Descriptors and addresses are then values of the warp, not of a thread: issued
// from a branch of one thread, moving them takes longer than the tensor cores do (4,096 tokens through 28,672 gate and up rows 545 us, so 470; 64 tokens
// through [4096, 14336] 19.7, so 16.4).
template <bool PAIR>
__device__ __forceinline__ void issue_products(uint32_t tmem_d, uint64_t da, uint64_t db, uint32_t idesc) {
#define SB_PRODUCT(GROUP, STEP, ACCUMULATE)                                                                                                  \
  asm volatile("{\n\t.reg .pred e, p;\n\telect.sync _|e, 0xffffffff;\n\tsetp.ne.b32 p, %4, 0;\n\t"                                             \
               "@e tcgen05.mma.cta_group::" GROUP ".kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}" ::"r"(tmem_d), "l"(da + 2 * STEP), "l"(db + 2 * STEP), \
               "r"(idesc), "n"(ACCUMULATE)                                                                                                   \
               : "memory")
  if (PAIR) {
    SB_PRODUCT("2", 0, 0);
    SB_PRODUCT("2", 1, 1);
    SB_PRODUCT("2", 2, 1);
    SB_PRODUCT("2", 3, 1);
  } else {
    SB_PRODUCT("1", 0, 0);
    SB_PRODUCT("1", 1, 1);
    SB_PRODUCT("1", 2, 1);
    SB_PRODUCT("1", 3, 1);
  }
#undef SB_PRODUCT
}
// Arrives on the barrier (of both CTAs of a pair) once the products issued so far are done.
template <bool PAIR>
__device__ __forceinline__ void issue_signal(uint32_t bar) {
  if (PAIR)
    asm volatile("{\n\t.reg .pred e;\n\telect.sync _|e, 0xffffffff;\n\t"
                 "@e tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;\n\t}" ::"r"(bar),
                 "h"(static_cast<unsigned short>(3))
                 : "memory");
  else
    asm volatile("{\n\t.reg .pred e;\n\telect.sync _|e, 0xffffffff;\n\t"
                 "@e tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}" ::"r"(bar)
                 : "memory");
}
// The same for loads: by one thread of a warp that is here as a whole, with addresses and coordinates that are values of the warp.
__device__ __forceinline__ void issue_expect(uint32_t bar, uint32_t bytes) {
  asm volatile("{\n\t.reg .pred e;\n\telect.sync _|e, 0xffffffff;\n\t@e mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;\n\t}" ::"r"(bar), "r"(bytes)
               : "memory");
}
template <bool PAIR>
__device__ __forceinline__ void issue_load(uint32_t dst, const CUtensorMap* map, uint32_t bar, int x, int y) {
  if (PAIR)
    asm volatile("{\n\t.reg .pred e;\n\telect.sync _|e, 0xffffffff;\n\t"
                 "@e cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], [%2];\n\t}" ::"r"(dst),
                 "l"(reinterpret_cast<uint64_t>(map)), "r"(bar & kPeerBitMask), "r"(x), "r"(y)
                 : "memory");
  else
    asm volatile("{\n\t.reg .pred e;\n\telect.sync _|e, 0xffffffff;\n\t"
                 "@e cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], [%2];\n\t}" ::"r"(dst),
                 "l"(reinterpret_cast<uint64_t>(map)), "r"(bar), "r"(x), "r"(y)
                 : "memory");
}
// Whether a barrier's phase is over, asked ahead of the wait for it: the answer is on its way while other work is issued (a wait that finds its phase
// over takes some hundred cycles, as long as a quarter of a block).
__device__ __forceinline__ bool mbar_over(uint32_t bar, uint32_t parity) {
  uint32_t ok;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "mbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(ok)
      : "r"(bar), "r"(parity)
      : "memory");
  return ok != 0;
}
// `mbar_wait` by a warp that leaves it as a whole, as loads from tensor memory need it: its lanes go on once all have seen the phase end. (A
// wait of each lane's own and a `__syncwarp` behind it: 4,096 tokens through 28,672 gate and up rows 558 to 566 us in a recorded graph, so 546 to 551.)
__device__ __forceinline__ bool mbar_wait_warp(uint32_t bar, uint32_t parity, int* status, int code) {
  long long began = 0;
  for (int spins = 1; !__all_sync(0xffffffffu, mbar_try_wait(bar, parity)); ++spins) {
    if ((spins & 255) != 0) continue;
    if (began == 0) began = clock64();
    const bool late = clock64() - began > kWaitCycles;
    if (late) atomicCAS(status, 0, code);
    if (__any_sync(0xffffffffu, late || *reinterpret_cast<volatile int*>(status) != 0)) return false;
  }
  return true;
}
// Waits for this warp's loads from tensor memory; what they brought passes through, so that no use of it can be moved in front of the wait.
__device__ __forceinline__ void tmem_arrived16(uint32_t* r) {
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]), "+r"(r[8]), "+r"(r[9]), "+r"(r[10]),
                 "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15])
               :
               : "memory");
}
__device__ __forceinline__ void tmem_arrived32(uint32_t* r) {
  tmem_arrived16(r);
  tmem_arrived16(r + 16);            // (nothing is left to wait for)
}
// sum[c] += v[c] * f[c], N sums of a thread.
template <int N>
__device__ __forceinline__ void add_scaled(float* sum, const uint32_t* v, const float* f) {
#pragma unroll
  for (int c = 0; c < N; c += 4) {
    const float4 s = *reinterpret_cast<const float4*>(f + c);
    sum[c] = fmaf(__uint_as_float(v[c]), s.x, sum[c]);
    sum[c + 1] = fmaf(__uint_as_float(v[c + 1]), s.y, sum[c + 1]);
    sum[c + 2] = fmaf(__uint_as_float(v[c + 2]), s.z, sum[c + 2]);
    sum[c + 3] = fmaf(__uint_as_float(v[c + 3]), s.w, sum[c + 3]);
  }
}
template <int N>
__device__ __forceinline__ void add_scaled(float* sum, const uint32_t* v, float f) {
#pragma unroll
  for (int c = 0; c < N; c += 2)           // (two of them an instruction)
    asm("{\n\t.reg .b64 s, v, f;\n\t"
        "mov.b64 s, {%0, %1};\n\tmov.b64 v, {%2, %3};\n\tmov.b64 f, {%4, %4};\n\t"
        "fma.rn.f32x2 s, v, f, s;\n\t"
        "mov.b64 {%0, %1}, s;\n\t}"
        : "+f"(sum[c]), "+f"(sum[c + 1])
        : "f"(__uint_as_float(v[c])), "f"(__uint_as_float(v[c + 1])), "f"(f));
}
// Sixteen bytes from global to shared memory on their own, the last 16 - `bytes` as zeros.
__device__ __forceinline__ void copy16_async(uint32_t to, const void* from, int bytes) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to), "l"(from), "r"(bytes) : "memory");
}
__device__ __forceinline__ void copies_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int LEFT>
__device__ __forceinline__ void copies_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(LEFT) : "memory");
}
__device__ __forceinline__ float cluster_load_float(uint32_t addr) {
  float v;
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(addr) : "memory");
  return v;
}

// Up to 32 choices of experts: a lane each, and every warp knows all about them without a kernel that puts them in order (one token's six through
// experts of 2,048 x 1,408: 22.7 us with it, 20.4 without, 20.0 by now). Rows in the order of the experts, an expert's in the choices' order.
constexpr int kMaxExperts = 1024;
constexpr int kFewChoices = 32;
struct FewChoices {
  uint32_t expert;          // of the lane's choice; kNone: of none
  uint32_t less, same;      // the choices of experts before it, and of the same
  int place;                // its row
  static constexpr uint32_t kNone = 2 * kMaxExperts - 1;
  __device__ __forceinline__ FewChoices(const int32_t* choice, int choices, int experts, int lane) {
    expert = lane < choices ? static_cast<uint32_t>(choice[lane]) : kNone;
    if (expert >= static_cast<uint32_t>(experts)) expert = kNone;
    less = 0, same = 0xFFFFFFFFu;
#pragma unroll
    for (uint32_t bit = kMaxExperts; bit != 0; bit >>= 1) {
      const uint32_t set = __ballot_sync(0xffffffffu, (expert & bit) != 0);
      if (expert & bit) less |= same & ~set;
      same &= expert & bit ? set : ~set;
    }
    place = __popc(less) + __popc(same & ((1u << lane) - 1u));
  }
  // Tile `at` of `rows` rows, 16 or more, as the list of `expert_order_kernel` has it; its row r is choice `of_row(left, r)`. False: there is none.
  __device__ __forceinline__ bool tile(int at, int rows, int lane, int& e, int& first, int& end, uint32_t& left) const {
    const int count = __popc(same);
    const bool leads = expert != kNone && lane == __ffs(same) - 1;
    const uint32_t one = __ballot_sync(0xffffffffu, leads), two = __ballot_sync(0xffffffffu, leads && count > rows);      // (of 32, no expert has three)
    const int before = __popc(one & less) + __popc(two & less);
    const uint32_t hit = __ballot_sync(0xffffffffu, leads && (before == at || (before + 1 == at && count > rows)));
    if (hit == 0) return false;
    const int from = __ffs(hit) - 1, start = __shfl_sync(0xffffffffu, place, from), skip = rows * (at - __shfl_sync(0xffffffffu, before, from));
    e = static_cast<int>(__shfl_sync(0xffffffffu, expert, from));
    left = __shfl_sync(0xffffffffu, same, from);
    first = start + skip, end = start + __popc(left);
    for (int i = 0; i < skip; ++i) left &= left - 1;
    return true;
  }
  static __device__ __forceinline__ int of_row(uint32_t left, int r) {
    for (int i = 0; i < r; ++i) left &= left - 1;
    return __ffs(left) - 1;
  }
};

template <int BN>
struct Shape {
  static constexpr int kEpilogueWarps = BN >= 64 ? 16 : BN >= 32 ? 8 : 4;
  static constexpr int kColumns = 16;                                  // columns of a thread's row of the tile
  static_assert(kColumns * kEpilogueWarps == 4 * BN, "four warps see all 128 rows");
  static constexpr int threads(bool quant) { return 128 + 32 * kEpilogueWarps + (quant ? 192 : 0); }
  static constexpr int kSlots = BN <= 32 ? 8 : 4;                      // accumulators under way
  static constexpr int kStage = kStageA + BN * 128;
  static constexpr int kTmem = kSlots * BN;                            // (a power of two)
  static constexpr int kCtas = BN <= 32 ? 2 : 1;                       // of an SM: with few tokens one fills its ring while the other drains
};

// blockIdx = (weight tile, token tile, K range: the rank in the cluster when SPLIT; else there is one range). Warp 0 loads, warp 1 issues the
// products, warps 2 and 3 multiply the scales, the others are the epilogue: four of them see all 128 rows, of 16 tokens. QUANT (tiles of 16 tokens): the
// input comes as it is, and eight warps quantise it, the same arithmetic as `quantize_kernel`, straight into the ring's stages. A block is one
// warp's, so that eight (of float32, where two CTAs share an SM's memory, four, of as many warps) are on their way at a time; all warps on one block at a
// time took 1.2 us for it. A lane copies the columns that it reads. A warp meets a stage's barrier only now and then, and could take one phase for the
// one two further on: it looks there only once its accumulator, of which there are eight, is free, and with it the last but one block of that stage.
constexpr int kQuantWarps = 8, kQuantRows = 16;
template <int EPI, int BN, class OUT, bool GROUPED, bool SPLIT, bool QUANT>
__global__ void __launch_bounds__(Shape<BN>::threads(QUANT), Shape<BN>::kCtas)
gemm_fp8_kernel(const __grid_constant__ CUtensorMap map_w, const __grid_constant__ CUtensorMap map_x, const Fp8Params p) {
  using S = Shape<BN>;
  static_assert(!QUANT || BN == kQuantRows, "two lanes a row of the input");
  constexpr int kScaleWarps = QUANT ? kQuantWarps : 2, kFirst = 2 + kScaleWarps;        // the epilogue's first warp
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  __shared__ __align__(8) uint64_t full_bar[kMaxStages], empty_bar[kMaxStages];
  __shared__ __align__(8) uint64_t accum_full[S::kSlots], scale_full[S::kSlots], slot_empty[S::kSlots];
  __shared__ __align__(16) float factor[S::kSlots][2][BN];
  __shared__ uint32_t tmem_base_s;

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t smem0 = (smem_u32(smem_raw) + 1023u) & ~1023u;
  uint8_t* smem0_p = smem_raw + (smem0 - smem_u32(smem_raw));
  const int tile_m = blockIdx.x;
  const int b0 = SPLIT ? blockIdx.z * p.range_blocks : 0;
  const int iters = (SPLIT ? min(p.blocks, b0 + p.range_blocks) : p.blocks) - b0;

  if (threadIdx.x == 0) {
    prefetch_tensormap(&map_w);
    prefetch_tensormap(&map_x);
    for (int s = 0; s < p.stages; ++s) mbar_init(smem_u32(&full_bar[s]), QUANT ? 2 : 1), mbar_init(smem_u32(&empty_bar[s]), 1);
    for (int s = 0; s < S::kSlots; ++s) {
      mbar_init(smem_u32(&accum_full[s]), 1);
      mbar_init(smem_u32(&scale_full[s]), QUANT ? 1 : 64);
      mbar_init(smem_u32(&slot_empty[s]), S::kEpilogueWarps);
    }
    mbar_init_fence();
  }
  if (warp == 1) tmem_alloc(smem_u32(&tmem_base_s), S::kTmem);
  fence_before_sync();
  __syncthreads();
  fence_after_sync();
  const uint32_t tmem_base = tmem_base_s;
  sb::grid_launch_dependents();        // (behind the allocation: a kernel let in before it could take the columns and wait for this one)
  int expert = 0, n0 = blockIdx.y * BN, end = p.n;
  uint32_t few = 0;
  bool empty = false;
  if (GROUPED) {
    sb::grid_dependency_wait();        // whose rows this tile holds is an earlier kernel's result
    if (QUANT && p.choice != nullptr) {
      empty = !FewChoices(p.choice, p.choices, p.experts, lane).tile(blockIdx.y, BN, lane, expert, n0, end, few);
    } else {
      empty = static_cast<int>(blockIdx.y) >= p.tiles[0];
      if (!empty) expert = p.tiles[2 + 3 * blockIdx.y], n0 = p.tiles[3 + 3 * blockIdx.y], end = p.tiles[4 + 3 * blockIdx.y];
    }
  }

  if (empty) {
  } else if (warp == 0) {
    const int row_w = expert * p.M + tile_m * (EPI == kGated ? 64 : kBlock);
    auto load_w = [&](int i, int st) {
      const uint32_t bar = smem_u32(&full_bar[st]), a = smem0 + st * S::kStage;
      issue_expect(bar, QUANT ? kStageA : S::kStage);
      issue_load<false>(a, &map_w, bar, (b0 + i) * kBlock, row_w);
      if (EPI == kGated) issue_load<false>(a + kStageA / 2, &map_w, bar, (b0 + i) * kBlock, row_w + p.half_rows);
    };
    auto load_x = [&](int i, int st) {
      if (!QUANT) issue_load<false>(smem0 + st * S::kStage + kStageA, &map_x, smem_u32(&full_bar[st]), (b0 + i) * kBlock, n0);
    };
    // (the weights are nobody's result: the first ring of them is under way before the kernels in front have ended)
    const int ahead = min(iters, p.stages);
    for (int i = 0; i < ahead; ++i) load_w(i, i);
    if (!GROUPED && !QUANT) sb::grid_dependency_wait();
    for (int i = 0; i < ahead; ++i) load_x(i, i);
    int st = ahead == p.stages ? 0 : ahead;
    uint32_t par = 0;
    for (int i = ahead; i < iters; ++i) {
      mbar_wait(smem_u32(&empty_bar[st]), par, p.status, 41);
      __syncwarp();
      load_w(i, st);
      load_x(i, st);
      if (++st == p.stages) st = 0, par ^= 1;
    }
  } else if (warp == 1) {
    const uint32_t idesc = instr_desc_e4m3(BN);
    const uint64_t first = smem_desc_sw128(smem0);
    int st = 0, slot = 0;
    uint32_t par = 0, slot_par = 1;
    bool ready = false;
    for (int i = 0; i < iters; ++i) {
      if (!__all_sync(0xffffffffu, ready)) {
        mbar_wait(smem_u32(&slot_empty[slot]), slot_par, p.status, 42);
        mbar_wait(smem_u32(&full_bar[st]), par, p.status, 43);
        __syncwarp();
      }
      fence_after_sync();
      const uint64_t da = first + static_cast<uint64_t>(st * (S::kStage >> 4));
      issue_products<false>(tmem_base + slot * BN, da, da + (kStageA >> 4), idesc);
      issue_signal<false>(smem_u32(&empty_bar[st]));
      issue_signal<false>(smem_u32(&accum_full[slot]));
      if (++st == p.stages) st = 0, par ^= 1;
      if (++slot == S::kSlots) slot = 0, slot_par ^= 1;
      ready = mbar_over(smem_u32(&slot_empty[slot]), slot_par) && mbar_over(smem_u32(&full_bar[st]), par);
    }
  } else if (warp < kFirst) {
    // the scales' products, a column a thread; four blocks are read ahead of their turn
    constexpr int kAhead = 4;
    const int t = threadIdx.x - 64;
    const float* ws0 = p.w_scales + static_cast<int64_t>(expert * p.scale_rows + (EPI == kGated ? tile_m / 2 : tile_m)) * p.blocks + b0;
    const float* ws1 = EPI == kGated ? ws0 + static_cast<int64_t>(p.scale_rows / 2) * p.blocks : ws0;
    if (!GROUPED) sb::grid_dependency_wait();
    if constexpr (QUANT) {
      constexpr int kPerRow = 2, kColumns = 128 / kPerRow;            // lanes of a row of the tile, columns of a lane
      const int r = lane / kPerRow, part = lane % kPerRow, first = warp - 2, warps = p.quant_warps, size = p.x_f32 ? 4 : 2,
                pieces = kColumns * size / 16;
      const bool live = n0 + r < end;
      int64_t row = !live ? 0 : n0 + r;
      if (GROUPED && p.x_gathered && live) row = p.choice != nullptr ? FewChoices::of_row(few, r) / p.top : p.order[n0 + r];
      const uint8_t* from = static_cast<const uint8_t*>(p.x) + (row * p.ldx + b0 * kBlock + part * kColumns) * size;
      const int columns = live ? p.K - b0 * kBlock - part * kColumns : 0;        // what the row has from there on
      const int mine = p.stages * S::kStage + first * pieces * 512 + lane * 16;      // this lane's pieces, 32 x 16 bytes from one to the next
      auto copy = [&](int i) {
        if (i < iters) {
          for (int j = 0; j < pieces; ++j) {
            const int there = (columns - i * kBlock) * size - 16 * j;
            copy16_async(smem0 + mine + j * 512, there > 0 ? from + i * kBlock * size + 16 * j : static_cast<const uint8_t*>(p.x),
                         min(max(there, 0), 16));
          }
        }
        copies_commit();
      };
      if (first < warps) copy(first);
      for (int i = first; i < iters && first < warps; i += warps) {
        const float w0 = __ldg(ws0 + i), w1 = EPI == kGated ? __ldg(ws1 + i) : 0.0f;
        copies_wait<0>();
        const uint8_t* piece = smem0_p + mine;
        uint32_t amax = 0;
        if (p.x_f32) {
#pragma unroll 8
          for (int j = 0; j < kColumns / 4; ++j) {
            const uint4 a = *reinterpret_cast<const uint4*>(piece + j * 512);
            amax = max(max(amax, max(a.x & 0x7FFFFFFFu, a.y & 0x7FFFFFFFu)), max(a.z & 0x7FFFFFFFu, a.w & 0x7FFFFFFFu));
          }
        } else {
#pragma unroll 4
          for (int j = 0; j < kColumns / 8; ++j) {
            const uint4 a = *reinterpret_cast<const uint4*>(piece + j * 512);
            const uint32_t w[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
            for (int k = 0; k < 4; ++k) amax = max(amax, max((w[k] << 16) & 0x7FFFFFFFu, w[k] & 0x7FFF0000u));
          }
        }
        amax = max(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
        const bool finite = amax < 0x7F800000u;
        const int e = finite ? scale_exponent(amax) : 0, st = i % p.stages, slot = i % S::kSlots;
        const float inverse = power_of_two(-e), scale = finite ? power_of_two(e) : __uint_as_float(0x7FC00000u);
        mbar_wait(smem_u32(&slot_empty[slot]), ((i / S::kSlots) & 1) ^ 1, p.status, 44);
        mbar_wait(smem_u32(&empty_bar[st]), ((i / p.stages) & 1) ^ 1, p.status, 47);
        uint8_t* to = smem0_p + st * S::kStage + kStageA + r * 128;
#pragma unroll 2
        for (int h = 0; h < kColumns / 16; ++h) {
          float v[16];
          if (p.x_f32) {
#pragma unroll
            for (int j = 0; j < 4; ++j) *reinterpret_cast<float4*>(v + 4 * j) = *reinterpret_cast<const float4*>(piece + (4 * h + j) * 512);
          } else {
#pragma unroll
            for (int j = 0; j < 2; ++j) {
              const uint4 a = *reinterpret_cast<const uint4*>(piece + (2 * h + j) * 512);
              const uint32_t w[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
              for (int k = 0; k < 4; ++k) v[8 * j + 2 * k] = __uint_as_float(w[k] << 16), v[8 * j + 2 * k + 1] = __uint_as_float(w[k] & 0xFFFF0000u);
            }
          }
          uint32_t q[4];
#pragma unroll
          for (int j = 0; j < 4; ++j)
            q[j] = e4m3x2(v[4 * j] * inverse, v[4 * j + 1] * inverse) | (e4m3x2(v[4 * j + 2] * inverse, v[4 * j + 3] * inverse) << 16);
          *reinterpret_cast<uint4*>(to + (((part * (kColumns / 16) + h) ^ (r & 7)) << 4)) = make_uint4(q[0], q[1], q[2], q[3]);      // (the 128-byte swizzle)
        }
        fence_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(smem_u32(&full_bar[st]));
        copy(i + warps);
        if (part == 0) {
          factor[slot][0][r] = scale * w0;
          if (EPI == kGated) factor[slot][1][r] = scale * w1;
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(smem_u32(&scale_full[slot]));
      }
    } else {
    float xs[kAhead], w0[kAhead], w1[kAhead];
    auto fetch = [&](int i, int a) {
      if (i >= iters) return;
      w0[a] = __ldg(ws0 + i), w1[a] = EPI == kGated ? __ldg(ws1 + i) : 0.0f;
      xs[a] = t < BN && n0 + t < end ? p.x_scales[static_cast<int64_t>(b0 + i) * p.ldxs + n0 + t] : 0.0f;
    };
#pragma unroll
    for (int a = 0; a < kAhead; ++a) fetch(a, a);
    int slot = 0;
    uint32_t slot_par = 1;
    for (int i0 = 0; i0 < iters; i0 += kAhead) {
#pragma unroll
      for (int a = 0; a < kAhead; ++a) {
        const int i = i0 + a;
        if (i >= iters) break;
        mbar_wait(smem_u32(&slot_empty[slot]), slot_par, p.status, 44);
        if (t < BN) {
          factor[slot][0][t] = xs[a] * w0[a];
          if (EPI == kGated) factor[slot][1][t] = xs[a] * w1[a];
        }
        mbar_arrive(smem_u32(&scale_full[slot]));
        fetch(i + kAhead, a);
        if (++slot == S::kSlots) slot = 0, slot_par ^= 1;
      }
    }
    }
  } else {
    const int quarter = warp & 3, half = (warp - kFirst) >> 2, row = quarter * 32 + lane;
    constexpr int C = S::kColumns;
    float acc[C];
#pragma unroll
    for (int c = 0; c < C; ++c) acc[c] = 0.0f;
    bool ok = true;
    int slot = 0;
    uint32_t slot_par = 0;
    bool ready = false;
    for (int i = 0; i < iters; ++i) {
      if (!__all_sync(0xffffffffu, ready)) {
        ok = mbar_wait(smem_u32(&accum_full[slot]), slot_par, p.status, 45) && ok;
        ok = mbar_wait(smem_u32(&scale_full[slot]), slot_par, p.status, 46) && ok;
        __syncwarp();
      }
      fence_after_sync();
      const uint32_t from = tmem_base + (static_cast<uint32_t>(quarter * 32) << 16) + slot * BN + half * C;
      const float* f = factor[slot][EPI == kGated && quarter >= 2 ? 1 : 0] + half * C;
      uint32_t v[C];
      tmem_load16_nowait(from, v);
      tmem_arrived16(v);
      add_scaled<C>(acc, v, f);
      fence_before_sync();
      __syncwarp();
      if (lane == 0) mbar_arrive(smem_u32(&slot_empty[slot]));
      if (++slot == S::kSlots) slot = 0, slot_par ^= 1;
      ready = mbar_over(smem_u32(&accum_full[slot]), slot_par) && mbar_over(smem_u32(&scale_full[slot]), slot_par);
    }
    // the tile's sums to shared memory, [token][row]: every load has arrived and every product that reads the ring is done
    float* tile = reinterpret_cast<float*>(smem0_p);
    if (ok) {
#pragma unroll
      for (int c = 0; c < C; ++c) tile[(half * C + c) * kBlock + row] = acc[c];
    }
    if (!ok) tile = nullptr;
    asm volatile("bar.sync 1, %0;" ::"r"(32 * S::kEpilogueWarps) : "memory");
    if (!GROUPED) sb::grid_dependency_wait();
    if (!SPLIT) {
      const int thread = threadIdx.x - 32 * kFirst;
      constexpr int kFeatures = EPI == kGated ? 64 : kBlock, kStride = 32 * S::kEpilogueWarps / kFeatures;
      const int j = thread % kFeatures, m = tile_m * kFeatures + j;
      if (tile != nullptr && m < (EPI == kGated ? p.half_rows : p.M)) {
        for (int c = thread / kFeatures; c < BN && n0 + c < end; c += kStride) {
          float v = tile[c * kBlock + j];
          if (EPI == kGated) v = gated_product(v, tile[c * kBlock + 64 + j], p.gate);
          OUT* o = static_cast<OUT*>(p.out) + static_cast<int64_t>(n0 + c) * p.ldo + m;
          if (EPI == kAdd) v += sb::widen(*o);
          *o = sb::narrow<OUT>(v);
        }
      }
    }
  }
  if (SPLIT) {
    sb::cluster_sync();
    if (warp >= kFirst) {
      const int thread = threadIdx.x - 32 * kFirst, rank = static_cast<int>(sb::cluster_rank());
      constexpr int kFeatures = EPI == kGated ? 64 : kBlock, kStride = 32 * S::kEpilogueWarps / kFeatures;
      const int j = thread % kFeatures, m = tile_m * kFeatures + j;
      const bool ok = *reinterpret_cast<volatile int*>(p.status) == 0;       // (a range that lost a signal has left no sums)
      if (ok && m < (EPI == kGated ? p.half_rows : p.M)) {
        const uint32_t here = smem0 + 4 * j;
        for (int c = rank + p.ranges * (thread / kFeatures); c < BN && n0 + c < end; c += p.ranges * kStride) {
          float v = 0.0f, u = 0.0f;
          for (int r = 0; r < p.ranges; ++r) {
            uint32_t peer;
            asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(peer) : "r"(here + c * kBlock * 4), "r"(r));
            const float a = cluster_load_float(peer);
            v = r == 0 ? a : v + a;
            if (EPI == kGated) {
              const float b = cluster_load_float(peer + 64 * 4);
              u = r == 0 ? b : u + b;
            }
          }
          if (EPI == kGated) v = gated_product(v, u, p.gate);
          OUT* o = static_cast<OUT*>(p.out) + static_cast<int64_t>(n0 + c) * p.ldo + m;
          if (EPI == kAdd) v += sb::widen(*o);
          *o = sb::narrow<OUT>(v);
        }
      }
    }
    sb::cluster_sync();                // (nobody leaves while another reads its sums)
  }
  fence_before_sync();
  __syncthreads();
  if (warp == 1) {
    fence_after_sync();
    tmem_dealloc(tmem_base, S::kTmem);
  }
}

// The same for many tokens, on pairs of CTAs (a cluster of two, cta_group::2) that walk tiles, with the operands' places changed: the 256 rows
// of a product are tokens, 128 a CTA, its columns are weight rows. A thread of the epilogue then holds one token's sums, and the scales of a
// block are one factor a thread and 128 weight rows instead of one a sum. (With weight rows as the product's rows, a factor from shared memory
// for every four sums, the gated product of 4,096 tokens, 2 x 14,336 rows of 4,096, took 870 us.) WIDE: 256 weight rows a tile, or 128 gate rows
// and their 128 up rows: each CTA loads 128 of them and 128 tokens, 32 KB a block for 512 cycles of the tensor cores. A weight with several K
// ranges needs its totals beside the sums in registers and has 128 rows a tile.
//
// A block's product is issued as two chains, each with half of both CTAs' weight rows (of a gated product: a feature's gate row and its up row
// in the same chain) and accumulators of its own, and the epilogue's warps as two sets, one a chain: a set's way from one accumulator to the
// next (signals, first loads) then falls into the other's additions. Each chain has a warp that issues it: one for both took longer than the
// tensor cores (574 us, with a warp each 524, when that was measured).
//
// PAIR false (experts, whose rows rarely fill 256, and dense products that need fewer rounds so): one CTA with the pair's weight rows and 128
// tokens, 48 KB a block for the same 512 cycles (2,000 tokens through 64 experts, six each: 280 us on pairs, 238 so, in bursts;
// in a long run of calls 265 to 277 so). The weight rows lie in
// shared memory as the pair's CTAs would have them, 64 of the first chain's each, then the second's.
constexpr int kPairTokens = 256;
constexpr int kPairThreads = 640;                // a warp that loads, two that issue the products, one for the scales, sixteen of the epilogue
constexpr int kBatch = 4, kBatches = 3;          // blocks whose factors are handed over together; batches under way
template <bool WIDE, bool PAIR>
struct PairShape {
  static constexpr int kRows = WIDE ? 256 : 128;             // weight rows of a tile
  static constexpr int kColumns = kRows / 2;                 // of a chain
  static constexpr int kTokens = PAIR ? 256 : 128;
  static constexpr int kStage = kStageA + (PAIR ? kRows / 2 : kRows) * 128;
  static constexpr int kChainB = (PAIR ? kColumns / 2 : kColumns) * 128;      // bytes from one chain's weight rows to the other's
  static constexpr int kSlots = 512 / kColumns;              // accumulators under way, all of tensor memory; even ones are the first chain's
  __host__ __device__ static constexpr int stages(bool staged) { return !PAIR ? (staged ? 3 : 4) : WIDE ? 5 : 6; }
};

// The tiles of a launch in the order in which the pairs walk them. Dense: the tiles of tokens first, so that the pairs of a round share few weight
// rows and every tile of tokens (which stay in L2); experts: the weight tiles of a tile of rows first.
struct PairTile {
  int tile_m, expert, n0, end;
  __device__ __forceinline__ PairTile(const Fp8Params& p, bool grouped, int tile, int tokens) {
    if (grouped) {
      const int t = tile / p.tiles_m;
      tile_m = tile - t * p.tiles_m;
      expert = p.tiles[2 + 3 * t], n0 = p.tiles[3 + 3 * t], end = p.tiles[4 + 3 * t];
    } else {
      tile_m = tile / p.tiles_n;
      expert = 0, n0 = (tile - tile_m * p.tiles_n) * tokens, end = p.n;
    }
  }
};

// A warp's results, a token a lane, 32 features m .. m + 31 of M each, to rows first .. of `out`, of which `count` exist. They pass through shared
// memory (`staged`, 32 rows of kPitch bytes), 64 bytes a token at a time, so that a store of the warp fills whole sectors of eight tokens: stored from
// the registers, half a sector a lane of 32 tokens, a tile's stores took as long as eight of its blocks.
constexpr int kPitch = 80;
constexpr int kStaged = 16 * 32 * kPitch;       // of all the epilogue's warps
template <int EPI, class OUT>
__device__ __forceinline__ void store_rows(OUT* out, int64_t ldo, int64_t first, int count, int m, int M, bool vec, const float* v, uint8_t* staged, int lane) {
  constexpr int kPer = 16 / sizeof(OUT), kChunk = 4 * kPer;      // elements of a piece of 16 bytes, of a token's 64 bytes
#pragma unroll
  for (int c0 = 0; c0 < 32; c0 += kChunk) {
    __syncwarp();
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      alignas(16) OUT r[kPer];
#pragma unroll
      for (int i = 0; i < kPer; ++i) r[i] = sb::narrow<OUT>(v[c0 + j * kPer + i]);
      *reinterpret_cast<uint4*>(staged + lane * kPitch + j * 16) = *reinterpret_cast<const uint4*>(r);
    }
    __syncwarp();
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int token = j * 8 + (lane >> 2), at = m + c0 + (lane & 3) * kPer;
      if (token >= count || at >= M) continue;
      uint4 raw = *reinterpret_cast<const uint4*>(staged + token * kPitch + (lane & 3) * 16);
      OUT* to = out + (first + token) * ldo + at;
      if (vec && at + kPer <= M) {
        if (EPI == kAdd) {
          const uint4 old = *reinterpret_cast<const uint4*>(to);
#pragma unroll
          for (int i = 0; i < kPer; ++i)
            reinterpret_cast<OUT*>(&raw)[i] = sb::narrow<OUT>(sb::widen(reinterpret_cast<const OUT*>(&raw)[i]) + sb::widen(reinterpret_cast<const OUT*>(&old)[i]));
        }
        *reinterpret_cast<uint4*>(to) = raw;
      } else {
#pragma unroll
        for (int i = 0; i < kPer; ++i)
          if (at + i < M) to[i] = EPI == kAdd ? sb::narrow<OUT>(sb::widen(reinterpret_cast<const OUT*>(&raw)[i]) + sb::widen(to[i])) : reinterpret_cast<const OUT*>(&raw)[i];
      }
    }
  }
}

template <int EPI, bool WIDE, class OUT, bool GROUPED, bool PAIR>
__global__ void __launch_bounds__(kPairThreads, 1)
gemm_fp8_pair_kernel(const __grid_constant__ CUtensorMap map_w, const __grid_constant__ CUtensorMap map_x, const Fp8Params p) {
  using S = PairShape<WIDE, PAIR>;
  constexpr bool kQuantised = std::is_same<OUT, uint8_t>::value;       // the gated products leave as e4m3 with scales of their own
  constexpr int kStages = S::stages(!kQuantised);
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  __shared__ __align__(8) uint64_t full_bar[kStages];      // used in the leader: both CTAs' tiles have landed
  __shared__ __align__(8) uint64_t empty_bar[kStages];     // in each CTA: the products that read its stage are done
  __shared__ __align__(8) uint64_t accum_full[S::kSlots];     // in each CTA
  __shared__ __align__(8) uint64_t accum_empty[S::kSlots];    // used in the leader: both CTAs have taken an accumulator's sums
  __shared__ __align__(8) uint64_t factor_full[kBatches], factor_empty[kBatches];      // in each CTA, its own
  __shared__ float factor[kBatches][kBatch][WIDE ? 2 : 1][kBlock];                     // by token
  __shared__ uint32_t largest[kQuantised ? 2 : 1][4][kQuantised ? kBlock : 1];
  __shared__ uint32_t tmem_base_s;

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int rank = PAIR ? static_cast<int>(sb::cluster_rank()) : 0;
  const uint32_t smem0 = (smem_u32(smem_raw) + 1023u) & ~1023u;
  uint8_t* smem0_p = smem_raw + (smem0 - smem_u32(smem_raw));
  const int pair = PAIR ? blockIdx.x >> 1 : blockIdx.x, pairs = PAIR ? gridDim.x >> 1 : gridDim.x;
  if (threadIdx.x == 0) {
    prefetch_tensormap(&map_w);
    prefetch_tensormap(&map_x);
    for (int s = 0; s < kStages; ++s) mbar_init(smem_u32(&full_bar[s]), 1), mbar_init(smem_u32(&empty_bar[s]), 2);      // (both chains')
    for (int s = 0; s < S::kSlots; ++s) {
      mbar_init(smem_u32(&accum_full[s]), 1);
      mbar_init(smem_u32(&accum_empty[s]), PAIR ? 2 * 8 : 8);       // one arrival a warp of either CTA's set
    }
    for (int s = 0; s < kBatches; ++s) mbar_init(smem_u32(&factor_full[s]), 32), mbar_init(smem_u32(&factor_empty[s]), 16);
    mbar_init_fence();
  }
  if (warp == 1) {
    if (PAIR) tmem_alloc_pair(smem_u32(&tmem_base_s), 512);
    else tmem_alloc(smem_u32(&tmem_base_s), 512);
  }
  fence_before_sync();
  __syncthreads();
  if (PAIR) sb::cluster_sync();          // the peer's barriers exist before anything signals them
  fence_after_sync();
  const uint32_t tmem_base = tmem_base_s;
  sb::grid_launch_dependents();
  sb::grid_dependency_wait();
  const int total = p.tiles_m * (GROUPED ? p.tiles[0] : p.tiles_n);

  if (warp == 0) {
    int st = 0;
    uint32_t par = 1;
    PairTile t(p, GROUPED, max(min(pair, total - 1), 0), S::kTokens);
    for (int tile = pair; tile < total; tile += pairs) {
      const PairTile next(p, GROUPED, min(tile + pairs, total - 1), S::kTokens);        // (on its way while this one is loaded)
      const int row = t.expert * p.M + (EPI == kGated ? t.tile_m * kBlock + rank * p.half_rows : t.tile_m * S::kRows + rank * (S::kRows / 2));
      const int token = t.n0 + rank * kBlock;
      for (int i = 0; i < p.blocks; ++i) {
        mbar_wait(smem_u32(&empty_bar[st]), par, p.status, 51);
        __syncwarp();
        const uint32_t bar = smem_u32(&full_bar[st]), a = smem0 + st * S::kStage;
        if (rank == 0) issue_expect(bar, (PAIR ? 2 : 1) * S::kStage);
        issue_load<PAIR>(a, &map_x, bar, i * kBlock, token);
        issue_load<PAIR>(a + kStageA, &map_w, bar, i * kBlock, row);
        if (!PAIR) {           // (boxes of 64 rows: the first chain's of the first and of the second half, then the second chain's)
          const int second = row + (EPI == kGated ? p.half_rows : kBlock);
          issue_load<false>(a + kStageA + 64 * 128, &map_w, bar, i * kBlock, second);
          issue_load<false>(a + kStageA + 128 * 128, &map_w, bar, i * kBlock, row + 64);
          issue_load<false>(a + kStageA + 192 * 128, &map_w, bar, i * kBlock, second + 64);
        }
        if (++st == kStages) st = 0, par ^= 1;
      }
      t = next;
    }
  } else if (warp < 3) {
    if (rank == 0) {
      const int chain = warp - 1;
      const uint64_t first = smem_desc_sw128(smem0);
      const uint32_t idesc = (1u << 4) | (static_cast<uint32_t>(S::kColumns >> 3) << 17) | (static_cast<uint32_t>(S::kTokens >> 4) << 24);
      int st = 0, slot = chain;
      uint32_t par = 0, slot_par = 1;
      bool ready = false;
      for (int tile = pair; tile < total; tile += pairs) {
        for (int i = 0; i < p.blocks; ++i) {
          if (WIDE || !__all_sync(0xffffffffu, ready)) {
            mbar_wait(smem_u32(&accum_empty[slot]), slot_par, p.status, 52);
            mbar_wait(smem_u32(&full_bar[st]), par, p.status, 53);
            __syncwarp();
          }
          fence_after_sync();
          const uint64_t da = first + static_cast<uint64_t>(st * (S::kStage >> 4));
          issue_products<PAIR>(tmem_base + slot * S::kColumns, da, da + (kStageA >> 4) + chain * (S::kChainB >> 4), idesc);
          issue_signal<PAIR>(smem_u32(&empty_bar[st]));
          issue_signal<PAIR>(smem_u32(&accum_full[slot]));
          if (++st == kStages) st = 0, par ^= 1;
          if ((slot += 2) >= S::kSlots) slot = chain, slot_par ^= 1;
          if (!WIDE) ready = mbar_over(smem_u32(&accum_empty[slot]), slot_par) && mbar_over(smem_u32(&full_bar[st]), par);
        }
      }
    }
  } else if (warp == 3) {
    // the scales' products, four tokens a lane, a batch ahead of those that wait in shared memory (a trip to L2 takes longer than a block)
    int slot = 0;
    uint32_t slot_par = 1;
    PairTile t(p, GROUPED, max(min(pair, total - 1), 0), S::kTokens);
    for (int tile = pair; tile < total; tile += pairs) {
      const PairTile next(p, GROUPED, min(tile + pairs, total - 1), S::kTokens);
      const int last = (EPI == kGated ? p.scale_rows / 2 : p.scale_rows) - 1;      // (rows beyond the weight: their sums are nobody's)
      const float* base = p.w_scales + static_cast<int64_t>(t.expert) * p.scale_rows * p.blocks;
      const float* ws0 = base + static_cast<int64_t>(min(EPI == kGated || !WIDE ? t.tile_m : 2 * t.tile_m, last)) * p.blocks;
      const float* ws1 = EPI == kGated ? ws0 + static_cast<int64_t>(p.scale_rows / 2) * p.blocks : base + static_cast<int64_t>(min(2 * t.tile_m + 1, last)) * p.blocks;
      const int token = t.n0 + rank * kBlock + lane;
      const float* xs = p.x_scales + token;
      float x[kBatch][4], w0[kBatch], w1[kBatch];
      auto fetch = [&](int i0) {
#pragma unroll
        for (int a = 0; a < kBatch; ++a) {
          const int i = i0 + a;
          const bool there = i < p.blocks;
          w0[a] = there ? __ldg(ws0 + i) : 0.0f, w1[a] = WIDE && there ? __ldg(ws1 + i) : 0.0f;
#pragma unroll
          for (int c = 0; c < 4; ++c) x[a][c] = there && token + 32 * c < t.end ? xs[i * p.ldxs + 32 * c] : 0.0f;
        }
      };
      fetch(0);
      for (int i0 = 0; i0 < p.blocks; i0 += kBatch) {
        mbar_wait(smem_u32(&factor_empty[slot]), slot_par, p.status, 54);
#pragma unroll
        for (int a = 0; a < kBatch; ++a)
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            factor[slot][a][0][lane + 32 * c] = x[a][c] * w0[a];
            if (WIDE) factor[slot][a][WIDE ? 1 : 0][lane + 32 * c] = x[a][c] * w1[a];
          }
        mbar_arrive(smem_u32(&factor_full[slot]));
        fetch(i0 + kBatch);
        if (++slot == kBatches) slot = 0, slot_par ^= 1;
      }
      t = next;
    }
  } else {
    // a token a thread; WIDE: 32 weight rows of each CTA, else 32 of the CTA `part`
    const int quarter = warp & 3, set = (warp - 4) >> 3, part = ((warp - 4) >> 2) & 1;
    float acc[32], other[32];            // the sums; WIDE: of the second 128 rows, else: the ranges' totals
    int slot = set, batch = 0;
    uint32_t slot_par = 0, batch_par = 0;
    bool ready = false;
    PairTile t(p, GROUPED, max(min(pair, total - 1), 0), S::kTokens);
    for (int tile = pair; tile < total; tile += pairs) {
      const PairTile next(p, GROUPED, min(tile + pairs, total - 1), S::kTokens);
      const int token = t.n0 + rank * kBlock + quarter * 32 + lane, blocks = p.blocks;
#pragma unroll
      for (int c = 0; c < 32; ++c) acc[c] = 0.0f, other[c] = WIDE ? 0.0f : -0.0f;
      bool ok = true;
      int left = p.range_blocks;
#pragma unroll 1
      for (int i = 0, in_batch = 0; i < blocks; ++i) {
        if (in_batch == 0) ok = mbar_wait(smem_u32(&factor_full[batch]), batch_par, p.status, 56) && ok;
        const float f0 = factor[batch][in_batch][0][quarter * 32 + lane], f1 = factor[batch][in_batch][WIDE ? 1 : 0][quarter * 32 + lane];
        if (WIDE) {
          ok = mbar_wait_warp(smem_u32(&accum_full[slot]), slot_par, p.status, 55) && ok;
        } else {
          if (!__all_sync(0xffffffffu, ready)) ok = mbar_wait(smem_u32(&accum_full[slot]), slot_par, p.status, 55) && ok;
          __syncwarp();
        }
        fence_after_sync();
        const uint32_t from = tmem_base + (static_cast<uint32_t>(quarter * 32) << 16) + slot * S::kColumns + part * 32;
        uint32_t v[16];
#pragma unroll
        for (int c0 = 0; c0 < (WIDE ? 64 : 32); c0 += 16) {
          tmem_load16_nowait(from + (c0 & 31) + (c0 & 32 ? 64 : 0), v);
          tmem_arrived16(v);
          if (c0 + 16 == (WIDE ? 64 : 32)) {         // (the last of them: the accumulator is free)
            fence_before_sync();
            __syncwarp();
            if (lane == 0) {
              if (PAIR) mbar_arrive_leader(smem_u32(&accum_empty[slot]));
              else mbar_arrive(smem_u32(&accum_empty[slot]));
            }
            if ((slot += 2) >= S::kSlots) slot = set, slot_par ^= 1;
            if (!WIDE) ready = mbar_over(smem_u32(&accum_full[slot]), slot_par);       // (WIDE: two accumulators a set, the next is never there yet)
          }
          add_scaled<16>((c0 & 32 ? other : acc) + (c0 & 31), v, c0 & 32 ? f1 : f0);
        }
        if (!WIDE && (--left == 0 || i + 1 == blocks)) {
          left = p.range_blocks;
#pragma unroll
          for (int c = 0; c < 32; ++c) other[c] += acc[c], acc[c] = 0.0f;
        }
        if (++in_batch == kBatch || i + 1 == blocks) {
          in_batch = 0;
          __syncwarp();
          if (lane == 0) mbar_arrive(smem_u32(&factor_empty[batch]));
          if (++batch == kBatches) batch = 0, batch_par ^= 1;
        }
      }
      if (EPI == kGated) {
        if (p.gate.act == kGateSilu) {       // (one gate for all, outside the loop)
#pragma unroll
          for (int c = 0; c < 32; ++c) acc[c] = silu_fast(acc[c]) * other[c];
        } else {
#pragma unroll
          for (int c = 0; c < 32; ++c) acc[c] = gated_product(acc[c], other[c], p.gate);
        }
      }
      if constexpr (kQuantised) {
        // the gated products are the next product's input: a block of 128 features is four threads' (both sets, both parts)
        const int m = t.tile_m * kBlock + set * 64 + part * 32, buffer = (tile / pairs) & 1, mine = quarter * 32 + lane;
        uint32_t amax = 0;
#pragma unroll
        for (int c = 0; c < 32; ++c) amax = m + c < p.half_rows ? max(amax, __float_as_uint(acc[c]) & 0x7FFFFFFFu) : amax;
        largest[buffer][set * 2 + part][mine] = amax;
        asm volatile("bar.sync 1, 512;" ::: "memory");           // (the buffers alternate: who writes one again has passed the barrier behind its readers)
#pragma unroll
        for (int j = 0; j < 4; ++j) amax = max(amax, largest[buffer][j][mine]);
        const bool finite = amax < 0x7F800000u;
        const int e = finite ? scale_exponent(amax) : 0;
        const float inverse = power_of_two(-e);
        if (ok && token < t.end) {
          uint8_t* to = static_cast<uint8_t*>(p.out) + static_cast<int64_t>(token) * p.ldo + m;
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            uint32_t q[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              const float* f = acc + 16 * h + 4 * j;
              q[j] = e4m3x2(f[0] * inverse, f[1] * inverse) | (e4m3x2(f[2] * inverse, f[3] * inverse) << 16);
            }
            if (m + 16 * h < p.ldo) *reinterpret_cast<uint4*>(to + 16 * h) = make_uint4(q[0], q[1], q[2], q[3]);      // (rows are padded to 16 bytes)
          }
          if (set + part == 0) p.z_scales[static_cast<int64_t>(t.tile_m) * p.ldxs + token] = finite ? power_of_two(e) : __uint_as_float(0x7FC00000u);
        }
      } else if (__all_sync(0xffffffffu, ok)) {
        OUT* out = static_cast<OUT*>(p.out);
        uint8_t* staged = smem0_p + kStages * S::kStage + (warp - 4) * 32 * kPitch;
        const int first = token - lane, count = min(t.end - first, 32);
        if (EPI == kGated) {
          store_rows<kStore>(out, p.ldo, first, count, t.tile_m * kBlock + set * 64 + part * 32, p.half_rows, p.vec_out, acc, staged, lane);
        } else {
          const int m = t.tile_m * S::kRows + (WIDE ? set * 64 + part * 32 : part * 64 + set * 32);
          store_rows<EPI>(out, p.ldo, first, count, m, p.M, p.vec_out, WIDE ? acc : other, staged, lane);
          if (WIDE) store_rows<EPI>(out, p.ldo, first, count, m + kBlock, p.M, p.vec_out, other, staged, lane);
        }
      }
      __syncwarp();
      t = next;
    }
  }
  fence_before_sync();
  __syncthreads();
  if (PAIR) sb::cluster_sync();          // neither CTA frees the pair's tensor memory, or leaves, while the other still works
  if (warp == 1) {
    fence_after_sync();
    if (PAIR) tmem_dealloc_pair(tmem_base, 512);
    else tmem_dealloc(tmem_base, 512);
  }
}

// The same for more tokens than a few and fewer than many, with tokens as the product's rows too (with weight rows as the product's rows [6144, 4096] of
// 128 tokens took 20.4 us, so 13.9): up to 128 tokens by 128
// weight rows, or 64 gate rows and their 64 up rows. SPLIT: the K ranges are shared out among the
// CTAs of a cluster, one or two each (0: one CTA has them all). Warp 0 loads, warp 1 issues the
// products, warp 2 multiplies the scales, sixteen warps are the epilogue, a token a lane and 32 columns each; those without tokens pass over.
constexpr int kTokenThreads = 640, kTokenRows = 128, kTokenSlots = 4;
constexpr int kRowPitch = 132;                   // floats from a token's sums to the next one's: 16-byte pieces of eight tokens meet in no bank
constexpr int kTokenStage = 2 * kStageA, kTokenStages = 6;

template <int EPI, class OUT, int SPLIT>
__global__ void __launch_bounds__(kTokenThreads, 1)
gemm_fp8_token_kernel(const __grid_constant__ CUtensorMap map_w, const __grid_constant__ CUtensorMap map_x, const Fp8Params p) {
  constexpr int kStages = SPLIT == 2 ? kTokenStages - 2 : kTokenStages;         // (two make room for the first range's sums)
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  __shared__ __align__(8) uint64_t full_bar[kStages], empty_bar[kStages];
  __shared__ __align__(8) uint64_t accum_full[kTokenSlots], accum_empty[kTokenSlots];
  __shared__ __align__(8) uint64_t factor_full[kBatches], factor_empty[kBatches];
  __shared__ float factor[kBatches][kBatch][EPI == kGated ? 2 : 1][kTokenRows];
  __shared__ uint32_t tmem_base_s;

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t smem0 = (smem_u32(smem_raw) + 1023u) & ~1023u;
  uint8_t* smem0_p = smem_raw + (smem0 - smem_u32(smem_raw));
  const int tile_m = blockIdx.x;
  const int b0 = SPLIT ? blockIdx.z * SPLIT * p.range_blocks : 0;
  const int iters = (SPLIT ? min(p.blocks, b0 + SPLIT * p.range_blocks) : p.blocks) - b0;

  if (warp == 1) tmem_alloc(smem_u32(&tmem_base_s), 512);
  __syncthreads();
  sb::grid_launch_dependents();        // (behind the allocation, as above)
  const int n0 = blockIdx.y * kTokenRows;
  const int count = min(p.n - n0, kTokenRows), quarters = (count + 31) / 32;        // the tile's tokens, and the lanes' quarters that have some
  if (threadIdx.x == 0) {
    prefetch_tensormap(&map_w);
    prefetch_tensormap(&map_x);
    for (int s = 0; s < kStages; ++s) mbar_init(smem_u32(&full_bar[s]), 1), mbar_init(smem_u32(&empty_bar[s]), 1);
    for (int s = 0; s < kTokenSlots; ++s) mbar_init(smem_u32(&accum_full[s]), 1), mbar_init(smem_u32(&accum_empty[s]), 4 * quarters);
    for (int s = 0; s < kBatches; ++s) mbar_init(smem_u32(&factor_full[s]), 32), mbar_init(smem_u32(&factor_empty[s]), 4 * quarters);
    mbar_init_fence();
  }
  fence_before_sync();
  __syncthreads();
  fence_after_sync();
  const uint32_t tmem_base = tmem_base_s;
  float* sums = reinterpret_cast<float*>(smem0_p);
  constexpr int kFirstSums = SPLIT == 2 ? kStages * kTokenStage / 4 : 0;         // SPLIT 2: where the first range's are, the second's are `sums`

  if (warp == 0) {
    const int row_w = tile_m * (EPI == kGated ? 64 : kBlock);
    auto load_w = [&](int i, int st) {
      const uint32_t bar = smem_u32(&full_bar[st]), to = smem0 + st * kTokenStage + kStageA;
      issue_expect(bar, kTokenStage);
      issue_load<false>(to, &map_w, bar, (b0 + i) * kBlock, row_w);
      if (EPI == kGated) issue_load<false>(to + kStageA / 2, &map_w, bar, (b0 + i) * kBlock, row_w + p.half_rows);
    };
    auto load_x = [&](int i, int st) { issue_load<false>(smem0 + st * kTokenStage, &map_x, smem_u32(&full_bar[st]), (b0 + i) * kBlock, n0); };
    // (the weights are nobody's result: the first ring of them is under way before the kernels in front have ended)
    const int ahead = min(iters, kStages);
    for (int i = 0; i < ahead; ++i) load_w(i, i);
    sb::grid_dependency_wait();
    for (int i = 0; i < ahead; ++i) load_x(i, i);
    int st = ahead == kStages ? 0 : ahead;
    uint32_t par = 0;
    for (int i = ahead; i < iters; ++i) {
      mbar_wait(smem_u32(&empty_bar[st]), par, p.status, 61);
      __syncwarp();
      load_w(i, st);
      load_x(i, st);
      if (++st == kStages) st = 0, par ^= 1;
    }
  } else if (warp == 1) {
    const uint32_t idesc = instr_desc_e4m3(kBlock);
    const uint64_t first = smem_desc_sw128(smem0);
    int st = 0, slot = 0;
    uint32_t par = 0, slot_par = 1;
    bool ready = false;
    for (int i = 0; i < iters; ++i) {
      if (!__all_sync(0xffffffffu, ready)) {
        mbar_wait(smem_u32(&accum_empty[slot]), slot_par, p.status, 62);
        mbar_wait(smem_u32(&full_bar[st]), par, p.status, 63);
        __syncwarp();
      }
      fence_after_sync();
      const uint64_t da = first + static_cast<uint64_t>(st * (kTokenStage >> 4));
      issue_products<false>(tmem_base + slot * kBlock, da, da + (kStageA >> 4), idesc);
      issue_signal<false>(smem_u32(&empty_bar[st]));
      issue_signal<false>(smem_u32(&accum_full[slot]));
      if (++st == kStages) st = 0, par ^= 1;
      if (++slot == kTokenSlots) slot = 0, slot_par ^= 1;
      ready = mbar_over(smem_u32(&accum_empty[slot]), slot_par) && mbar_over(smem_u32(&full_bar[st]), par);
    }
  } else if (warp == 2) {
    // the scales' products, four tokens a lane, a batch ahead of those that wait in shared memory
    const float* ws0 = p.w_scales + static_cast<int64_t>(EPI == kGated ? tile_m / 2 : tile_m) * p.blocks + b0;
    const float* ws1 = ws0 + static_cast<int64_t>(EPI == kGated ? p.scale_rows / 2 : 0) * p.blocks;
    const float* xs = p.x_scales + b0 * p.ldxs + n0 + lane;
    sb::grid_dependency_wait();
    float x[kBatch][4], w0[kBatch], w1[kBatch];
    auto fetch = [&](int i0) {
#pragma unroll
      for (int a = 0; a < kBatch; ++a) {
        const int i = i0 + a;
        const bool there = i < iters;
        w0[a] = there ? __ldg(ws0 + i) : 0.0f, w1[a] = EPI == kGated && there ? __ldg(ws1 + i) : 0.0f;
#pragma unroll
        for (int c = 0; c < 4; ++c) x[a][c] = there && lane + 32 * c < count ? xs[i * p.ldxs + 32 * c] : 0.0f;
      }
    };
    fetch(0);
    int slot = 0;
    uint32_t slot_par = 1;
    for (int i0 = 0; i0 < iters; i0 += kBatch) {
      mbar_wait(smem_u32(&factor_empty[slot]), slot_par, p.status, 64);
#pragma unroll
      for (int a = 0; a < kBatch; ++a)
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          factor[slot][a][0][lane + 32 * c] = x[a][c] * w0[a];
          if (EPI == kGated) factor[slot][a][EPI == kGated ? 1 : 0][lane + 32 * c] = x[a][c] * w1[a];
        }
      mbar_arrive(smem_u32(&factor_full[slot]));
      fetch(i0 + kBatch);
      if (++slot == kBatches) slot = 0, slot_par ^= 1;
    }
  } else if (warp >= 4 && (warp & 3) < quarters) {
    const int quarter = warp & 3, part = (warp - 4) >> 2, token = quarter * 32 + lane;
    float acc[32], total[SPLIT ? 1 : 32];
#pragma unroll
    for (int c = 0; c < 32; ++c) acc[c] = 0.0f;
    if (!SPLIT) {
#pragma unroll
      for (int c = 0; c < 32; ++c) total[c] = -0.0f;          // (the first range is added to nothing: -0 + v = v, signs of zeros too)
    }
    int slot = 0, batch = 0, left = p.range_blocks;
    uint32_t slot_par = 0, batch_par = 0;
    bool ready = false;
#pragma unroll 1
    for (int i = 0, in_batch = 0; i < iters; ++i) {
      if (in_batch == 0) mbar_wait(smem_u32(&factor_full[batch]), batch_par, p.status, 66);
      const float f = factor[batch][in_batch][EPI == kGated && part >= 2 ? 1 : 0][token];
      if (!__all_sync(0xffffffffu, ready)) mbar_wait(smem_u32(&accum_full[slot]), slot_par, p.status, 65);
      __syncwarp();
      fence_after_sync();
      const uint32_t from = tmem_base + (static_cast<uint32_t>(quarter * 32) << 16) + slot * kBlock + part * 32;
      constexpr int kChunk = SPLIT ? 32 : 16;          // (the totals leave fewer registers)
      uint32_t v[kChunk];
#pragma unroll
      for (int c0 = 0; c0 < 32; c0 += kChunk) {
        if (kChunk == 32) tmem_load32_nowait(from, v), tmem_arrived32(v);
        else tmem_load16_nowait(from + c0, v), tmem_arrived16(v);
        if (c0 + kChunk == 32) {
          fence_before_sync();
          __syncwarp();
          if (lane == 0) mbar_arrive(smem_u32(&accum_empty[slot]));
          if (++slot == kTokenSlots) slot = 0, slot_par ^= 1;
          ready = mbar_over(smem_u32(&accum_full[slot]), slot_par);
        }
        add_scaled<kChunk>(acc + c0, v, f);
      }
      if (++in_batch == kBatch || i + 1 == iters) {
        in_batch = 0;
        __syncwarp();
        if (lane == 0) mbar_arrive(smem_u32(&factor_empty[batch]));
        if (++batch == kBatches) batch = 0, batch_par ^= 1;
      }
      if (!SPLIT && (--left == 0 || i + 1 == iters)) {
        left = p.range_blocks;
#pragma unroll
        for (int c = 0; c < 32; ++c) total[c] += acc[c], acc[c] = 0.0f;
      }
      if (SPLIT == 2 && i + 1 == min(p.range_blocks, iters)) {
        float* to = sums + kFirstSums + token * kRowPitch + part * 32;
#pragma unroll
        for (int c = 0; c < 32; c += 4)
          *reinterpret_cast<float4*>(to + c) = make_float4(acc[c], acc[c + 1], acc[c + 2], acc[c + 3]), acc[c] = acc[c + 1] = acc[c + 2] = acc[c + 3] = 0.0f;
      }
    }
    // the sums to shared memory, a row a token: every load has arrived and every product that reads the ring is done
    float* to = sums + token * kRowPitch + part * 32;
    const float* done = SPLIT ? acc : total;
#pragma unroll
    for (int c = 0; c < 32; c += 4) *reinterpret_cast<float4*>(to + c) = make_float4(done[c], done[c + 1], done[c + 2], done[c + 3]);
  }
  __syncwarp();
  if (SPLIT) sb::cluster_sync();
  else __syncthreads();
  if (warp >= 4 && *reinterpret_cast<volatile int*>(p.status) == 0) {      // (a wait that gave up has left no sums)
    sb::grid_dependency_wait();
    const int rank = SPLIT ? static_cast<int>(sb::cluster_rank()) : 0, ranges = SPLIT ? p.ranges : 1;
    const int ctas = SPLIT ? gridDim.z : 1;
    constexpr int kPer = EPI == kGated ? 2 : 4;                  // features of a lane
    const int m = tile_m * (EPI == kGated ? 64 : kBlock) + lane * kPer, M = EPI == kGated ? p.half_rows : p.M;
    for (int t = rank + ctas * (warp - 4); t < count; t += ctas * 16) {
      float v[kPer], u[EPI == kGated ? 2 : 1];
      const uint32_t here = smem0 + (t * kRowPitch + lane * kPer) * 4;
      for (int r = 0; r < ranges; ++r) {
        float a[kPer], b[2] = {0.0f, 0.0f};
        if (SPLIT) {
          uint32_t peer;
          asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(peer) : "r"(here + (SPLIT == 2 && (r & 1) == 0 ? 4 * kFirstSums : 0)), "r"(SPLIT == 2 ? r >> 1 : r));
#pragma unroll
          for (int i = 0; i < kPer; i += 2) {
            const float2 x = sb::cluster_load_float2(peer + 4 * i);
            a[i] = x.x, a[i + 1] = x.y;
          }
          if (EPI == kGated) {
            const float2 x = sb::cluster_load_float2(peer + 64 * 4);
            b[0] = x.x, b[1] = x.y;
          }
        } else {
          const float* at = sums + t * kRowPitch + lane * kPer;
#pragma unroll
          for (int i = 0; i < kPer; ++i) a[i] = at[i];
          if (EPI == kGated) b[0] = at[64], b[1] = at[65];
        }
#pragma unroll
        for (int i = 0; i < kPer; ++i) v[i] = r == 0 ? a[i] : v[i] + a[i];
        if (EPI == kGated) {
#pragma unroll
          for (int i = 0; i < 2; ++i) u[EPI == kGated ? i : 0] = r == 0 ? b[i] : u[EPI == kGated ? i : 0] + b[i];
        }
      }
      if (EPI == kGated) {
#pragma unroll
        for (int i = 0; i < kPer; ++i) v[i] = gated_product(v[i], u[EPI == kGated ? i : 0], p.gate);
      }
      OUT* o = static_cast<OUT*>(p.out) + static_cast<int64_t>(n0 + t) * p.ldo + m;
      if (p.vec_out && m + kPer <= M) {
        struct alignas(kPer * sizeof(OUT)) Piece {
          OUT e[kPer];
        } piece;
        if (EPI == kAdd) {
          piece = *reinterpret_cast<const Piece*>(o);
#pragma unroll
          for (int i = 0; i < kPer; ++i) v[i] += sb::widen(piece.e[i]);
        }
#pragma unroll
        for (int i = 0; i < kPer; ++i) piece.e[i] = sb::narrow<OUT>(v[i]);
        *reinterpret_cast<Piece*>(o) = piece;
      } else {
#pragma unroll
        for (int i = 0; i < kPer; ++i)
          if (m + i < M) o[i] = sb::narrow<OUT>(EPI == kAdd ? v[i] + sb::widen(o[i]) : v[i]);
      }
    }
  }
  if (SPLIT) sb::cluster_sync();       // (nobody leaves while another reads its sums)
  fence_before_sync();
  __syncthreads();
  if (warp == 1) {
    fence_after_sync();
    tmem_dealloc(tmem_base, 512);
  }
}

// ------------------------------------------------------------------ experts
// choice [n][top] -> the choices' tokens in expert order, the row of every choice (place [n][top]; -1: none), and the row tiles of the
// products. An id outside [0, E) is no expert: it is left out. list: [0] tiles, [1] rows, then (expert, first row, end row) of every tile.
// (Which of an expert's rows comes first does not matter: every row is computed on its own.) One CTA; a thread holds kHeld choices, loaded
// together, and reads those beyond twice.
constexpr int kOrderThreads = 1024, kHeld = 16;
__global__ void __launch_bounds__(kOrderThreads) expert_order_kernel(const int32_t* choice, int n, int top, int E, int tile,
                                                                     int32_t* order, int32_t* place, int32_t* list) {
  __shared__ int count[kMaxExperts], next[kMaxExperts], tile_at[kMaxExperts], rows;
  __shared__ __align__(4) uint16_t sorted[kHeld * kOrderThreads];      // the tokens of held choices by row (stored to memory one by one they took 6 us)
  sb::grid_launch_dependents();
  for (int e = threadIdx.x; e < E; e += blockDim.x) count[e] = 0;
  __syncthreads();
  sb::grid_dependency_wait();
  const int pairs = n * top, t = threadIdx.x;
  uint32_t held[kHeld];
#pragma unroll
  for (int j = 0; j < kHeld; ++j) held[j] = t + j * kOrderThreads < pairs ? static_cast<uint32_t>(choice[t + j * kOrderThreads]) : 0xFFFFFFFFu;
  int rank[kHeld];                       // a held choice's place among its expert's
#pragma unroll
  for (int j = 0; j < kHeld; ++j) rank[j] = held[j] < static_cast<uint32_t>(E) ? atomicAdd(&count[held[j]], 1) : 0;
  __syncthreads();
  int* held_of = reinterpret_cast<int*>(sorted);         // (of more choices than those: how many of an expert's are held)
  if (pairs > kHeld * kOrderThreads) {
    for (int e = t; e < E; e += kOrderThreads) held_of[e] = count[e];
    __syncthreads();
    for (int i = t + kHeld * kOrderThreads; i < pairs; i += kOrderThreads) {
      const uint32_t e = static_cast<uint32_t>(choice[i]);
      if (e < static_cast<uint32_t>(E)) atomicAdd(&count[e], 1);
    }
    __syncthreads();
  }
  if (threadIdx.x < 32) {
    const int lane = threadIdx.x;
    int rows_before = 0, tiles_before = 0;
    for (int e0 = 0; e0 < E; e0 += 32) {
      const int e = e0 + lane, c = e < E ? count[e] : 0, ct = (c + tile - 1) / tile;
      int cs = c, ts = ct;
      for (int o = 1; o < 32; o <<= 1) {
        const int a = __shfl_up_sync(0xffffffffu, cs, o), b = __shfl_up_sync(0xffffffffu, ts, o);
        if (lane >= o) cs += a, ts += b;
      }
      if (e < E) next[e] = rows_before + cs - c, tile_at[e] = tiles_before + ts - ct;
      rows_before += __shfl_sync(0xffffffffu, cs, 31), tiles_before += __shfl_sync(0xffffffffu, ts, 31);
    }
    if (lane == 0) list[0] = tiles_before, list[1] = rows = rows_before;
  }
  __syncthreads();
  for (int e = threadIdx.x; e < E; e += blockDim.x) {
    const int first = next[e], end = first + count[e];
    int32_t* to = list + 2 + 3 * static_cast<int64_t>(tile_at[e]);
    for (int r = first; r < end; r += tile, to += 3) to[0] = e, to[1] = r, to[2] = end;
  }
#pragma unroll
  for (int j = 0; j < kHeld; ++j) {
    const int i = t + j * kOrderThreads;
    if (i >= pairs) break;
    const bool there = held[j] < static_cast<uint32_t>(E);
    const int at = there ? next[held[j]] + rank[j] : -1;
    if (there && pairs <= kHeld * kOrderThreads) sorted[at] = static_cast<uint16_t>(i / top);
    else if (there) order[at] = i / top;
    place[i] = at;
  }
  __syncthreads();
  if (pairs <= kHeld * kOrderThreads) {
    for (int i = t; i < rows; i += kOrderThreads) order[i] = sorted[i];
    return;
  }
  for (int e = t; e < E; e += kOrderThreads) next[e] += held_of[e];
  __syncthreads();
  for (int i = t + kHeld * kOrderThreads; i < pairs; i += kOrderThreads) {
    const uint32_t e = static_cast<uint32_t>(choice[i]);
    const int at = e < static_cast<uint32_t>(E) ? atomicAdd(&next[e], 1) : -1;
    if (at >= 0) order[at] = i / top;
    place[i] = at;
  }
}

// out[t] = the sum over the token's choices, in their order, of weight times result: parts [rows][ldp], rows 16-byte aligned, by `place` [n][top] (-1:
// no expert, no term; null: `FewChoices` of `choice`), weights [top][n]. Twice four features a thread (VEC: the result takes them together), the loads of several choices under way.
template <class OUT, bool VEC>
__global__ void __launch_bounds__(128) expert_combine_kernel(const float* parts, int64_t ldp, const int32_t* place, const int32_t* choice, int experts, const float* weights,
                                                             int n, int top, int W, OUT* out, int64_t ldo) {
  sb::grid_launch_dependents();
  sb::grid_dependency_wait();
  const int t = blockIdx.x, m0 = (blockIdx.y * 2 * blockDim.x + threadIdx.x) * 4;
  const int32_t* mine = place + static_cast<int64_t>(t) * top;
  int few = -1;                      // the row of the lane's choice
  if (place == nullptr) {
    const FewChoices all(choice, n * top, experts, threadIdx.x & 31);
    few = all.expert != FewChoices::kNone ? all.place : -1;
  }
  float sum[2][4] = {};
  constexpr int kTogether = 4;
  for (int k0 = 0; k0 < top; k0 += kTogether) {
    float4 v[kTogether][2];
    float w[kTogether];
    int row[kTogether];
#pragma unroll
    for (int k = 0; k < kTogether; ++k) {
      row[k] = place == nullptr ? __shfl_sync(0xffffffffu, few, (t * top + k0 + k) & 31) : k0 + k < top ? mine[k0 + k] : -1;
      if (k0 + k >= top) row[k] = -1;
      w[k] = k0 + k < top ? weights[static_cast<int64_t>(k0 + k) * n + t] : 0.0f;
    }
#pragma unroll
    for (int k = 0; k < kTogether; ++k)
#pragma unroll
      for (int h = 0; h < 2; ++h)
        if (row[k] >= 0 && m0 + h * 512 < W) v[k][h] = *reinterpret_cast<const float4*>(parts + row[k] * ldp + m0 + h * 512);
#pragma unroll
    for (int k = 0; k < kTogether; ++k)
#pragma unroll
      for (int h = 0; h < 2; ++h)
        if (row[k] >= 0 && m0 + h * 512 < W) {
          sum[h][0] = fmaf(w[k], v[k][h].x, sum[h][0]), sum[h][1] = fmaf(w[k], v[k][h].y, sum[h][1]);
          sum[h][2] = fmaf(w[k], v[k][h].z, sum[h][2]), sum[h][3] = fmaf(w[k], v[k][h].w, sum[h][3]);
        }
  }
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const int m = m0 + h * 512;
    if (m >= W) break;
    OUT* to = out + static_cast<int64_t>(t) * ldo + m;
    if (VEC && m + 4 <= W) {
      alignas(16) OUT r[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) r[i] = sb::narrow<OUT>(sum[h][i]);
      if (sizeof(OUT) == 4) *reinterpret_cast<uint4*>(to) = *reinterpret_cast<const uint4*>(r);
      else *reinterpret_cast<uint2*>(to) = *reinterpret_cast<const uint2*>(r);
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (m + i < W) to[i] = sb::narrow<OUT>(sum[h][i]);
    }
  }
}

// ------------------------------------------------------------------ host side
// Tensor map of bytes [rows][K] (row stride ld, a multiple of 16) in boxes of 128 columns by `box_rows`, 128-byte swizzle, zeros beyond.
bool byte_map(const void* base, int64_t rows, int64_t K, int64_t ld, int box_rows, CUtensorMap* out) {
  EncodeTiledFn fn = encode_fn();
  if (!fn) return false;
  const cuuint64_t dims[2] = {static_cast<cuuint64_t>(K), static_cast<cuuint64_t>(rows)}, strides[1] = {static_cast<cuuint64_t>(ld)};
  const cuuint32_t box[2] = {128, static_cast<cuuint32_t>(box_rows)}, one[2] = {1, 1};
  return fn(out, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void*>(base), dims, strides, box, one, CU_TENSOR_MAP_INTERLEAVE_NONE,
            CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// K ranges of a weight of `tiles` tiles of 128 rows and `blocks` blocks of columns: as many CTAs as there are SMs, four ranges at most (of eight, a
// cluster's CTAs found places late: [2048, 2048] of 40 tokens 10.5 us, in four ranges 7.1).
int fp8_ranges(int tiles, int blocks) {
  int s = 1;
  while (s < kMaxRanges && tiles * s * 2 <= 148 && blocks >= s * 4) s *= 2;
  return (blocks + (blocks + s - 1) / s - 1) / ((blocks + s - 1) / s);        // (no empty range)
}

// Up to `kQuantRows` rows of a tile the product can quantise its input itself. Of a dense product it does where a CTA has up to this many blocks: that
// saves a launch, but a block takes longer (2,048 x 2,048 of one token 7.7 us with a launch, 4.6 without; 16,384 x 2,048, 16 blocks a CTA, of eight
// 10.1 and 12.1). The experts' two inputs would need two launches.
constexpr int kQuantBlocks = 6;

template <int EPI, int BN, class OUT, bool GROUPED>
int launch_tile(const void* w, int64_t rows_w, int64_t ldw, const void* q, int64_t rows_q, int64_t ldq, Fp8Params p, int tiles_m, int tiles_n,
                cudaStream_t st) {
  using S = Shape<BN>;
  const bool quant = BN <= kQuantRows && p.x != nullptr;
  CUtensorMap map_w, map_x;
  if (!byte_map(w, rows_w, p.K, ldw, EPI == kGated ? 64 : kBlock, &map_w) || (!quant && !byte_map(q, rows_q, p.K, ldq, BN, &map_x)))
    return sb::fail("gemm_fp8: no tensor map for a weight of %lld x %d (stride %lld)", (long long)rows_w, p.K, (long long)ldw);
  if (quant) map_x = map_w;                  // (not read)
  const bool split = !GROUPED && p.split;
  const dim3 grid(tiles_m, tiles_n, split ? p.ranges : 1);
  // (few CTAs have an SM each: the longest ring then brings most of the weights on their way while the kernel in front still runs. Else two share
  // one where they can. Quantising: at least half as many stages as accumulators, see the kernel)
  const bool alone = static_cast<long long>(tiles_m) * tiles_n * grid.z <= sb::sm_count();
  p.quant_warps = p.x_f32 && !alone ? kQuantWarps / 2 : kQuantWarps;
  const int copies = quant ? p.quant_warps * BN * kBlock * (p.x_f32 ? 4 : 2) : 0;
  const int room = (alone || S::kCtas == 1 ? kSmemBudget : quant ? 4 * S::kStage + copies : 100 * 1024) - copies;
  p.stages = std::min(kMaxStages, room / S::kStage);
  const size_t smem = static_cast<size_t>(p.stages) * S::kStage + copies + 1024;
  auto run = [&](auto kernel, sb::DeviceOnce& once) {
    if (once.needed()) {
      if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmemBudget + 1024) != cudaSuccess) return sb::check_launch("gemm_fp8");
      once.done();
    }
    if (split) sb::launch_pdl_cluster(kernel, grid, dim3(S::threads(quant)), smem, st, dim3(1, 1, p.ranges), map_w, map_x, p);
    else sb::launch_pdl(kernel, grid, dim3(S::threads(quant)), smem, st, map_w, map_x, p);
    return sb::check_launch("gemm_fp8");
  };
  static sb::DeviceOnce once[4];
  if constexpr (BN <= kQuantRows) {
    if (quant) {
      if constexpr (!GROUPED) {
        if (split) return run(gemm_fp8_kernel<EPI, BN, OUT, GROUPED, true, true>, once[0]);
      }
      return run(gemm_fp8_kernel<EPI, BN, OUT, GROUPED, false, true>, once[1]);
    }
  }
  if constexpr (!GROUPED) {
    if (split) return run(gemm_fp8_kernel<EPI, BN, OUT, GROUPED, true, false>, once[2]);
  }
  return run(gemm_fp8_kernel<EPI, BN, OUT, GROUPED, false, false>, once[3]);
}

template <int EPI, class OUT>
int launch_token(const void* w, int64_t rows_w, int64_t ldw, const void* q, int64_t rows_q, int64_t ldq, Fp8Params p, int tiles_m, int tiles_n, cudaStream_t st) {
  CUtensorMap map_w, map_x;
  if (!byte_map(w, rows_w, p.K, ldw, EPI == kGated ? 64 : kBlock, &map_w) || !byte_map(q, rows_q, p.K, ldq, kTokenRows, &map_x))
    return sb::fail("gemm_fp8: no tensor map for a weight of %lld x %d (stride %lld)", (long long)rows_w, p.K, (long long)ldw);
  const int piece = (EPI == kGated ? 2 : 4) * static_cast<int>(sizeof(OUT));
  p.vec_out = p.ldo * sizeof(OUT) % piece == 0 && (reinterpret_cast<uintptr_t>(p.out) & (piece - 1)) == 0;
  const size_t smem = static_cast<size_t>(kTokenStages) * kTokenStage + (p.split == 2 ? kTokenRows * kRowPitch * 4 - 2 * kTokenStage : 0) + 1024;
  const int ctas = p.split ? (p.ranges + p.split - 1) / p.split : 1;
  const dim3 grid(tiles_m, tiles_n, ctas);
  static sb::DeviceOnce once[3];
  auto run = [&](auto kernel, sb::DeviceOnce& first) {
    if (first.needed()) {
      if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(smem)) != cudaSuccess) return sb::check_launch("gemm_fp8");
      first.done();
    }
    if (p.split) sb::launch_pdl_cluster(kernel, grid, dim3(kTokenThreads), smem, st, dim3(1, 1, ctas), map_w, map_x, p);
    else sb::launch_pdl(kernel, grid, dim3(kTokenThreads), smem, st, map_w, map_x, p);
    return sb::check_launch("gemm_fp8");
  };
  if (p.split == 2) return run(gemm_fp8_token_kernel<EPI, OUT, 2>, once[2]);
  return p.split ? run(gemm_fp8_token_kernel<EPI, OUT, 1>, once[0]) : run(gemm_fp8_token_kernel<EPI, OUT, 0>, once[1]);
}

template <int EPI, bool WIDE, class OUT, bool GROUPED, bool PAIR>
int launch_pair(const void* w, int64_t rows_w, int64_t ldw, const void* q, int64_t rows_q, int64_t ldq, Fp8Params p, int tiles_n, cudaStream_t st) {
  using S = PairShape<WIDE, PAIR>;
  CUtensorMap map_w, map_x;
  if (!byte_map(w, rows_w, p.K, ldw, PAIR ? S::kRows / 2 : 64, &map_w) || !byte_map(q, rows_q, p.K, ldq, kBlock, &map_x))
    return sb::fail("gemm_fp8: no tensor map for a weight of %lld x %d (stride %lld)", (long long)rows_w, p.K, (long long)ldw);
  p.tiles_m = EPI == kGated ? (p.half_rows + kBlock - 1) / kBlock : (p.M + S::kRows - 1) / S::kRows;
  p.tiles_n = tiles_n;
  p.vec_out = p.ldo * sizeof(OUT) % 16 == 0 && (reinterpret_cast<uintptr_t>(p.out) & 15) == 0;
  const long long tiles = static_cast<long long>(p.tiles_m) * tiles_n;
  if (tiles > (1ll << 30)) return sb::fail("gemm_fp8: too many tiles");
  auto kernel = gemm_fp8_pair_kernel<EPI, WIDE, OUT, GROUPED, PAIR>;
  constexpr bool kThrough = !std::is_same<OUT, uint8_t>::value;          // results pass through shared memory
  const size_t smem = static_cast<size_t>(S::stages(kThrough)) * S::kStage + (kThrough ? kStaged : 0) + 1024;
  static sb::DeviceOnce once;
  if (once.needed()) {
    if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(smem)) != cudaSuccess) return sb::check_launch("gemm_fp8");
    once.done();
  }
  const int units = static_cast<int>(std::min<long long>(tiles, PAIR ? sb::sm_count() / 2 : sb::sm_count()));
  if (PAIR) sb::launch_pdl_cluster(kernel, dim3(2 * units), dim3(kPairThreads), smem, st, dim3(2, 1, 1), map_w, map_x, p);
  else sb::launch_pdl(kernel, dim3(units), dim3(kPairThreads), smem, st, map_w, map_x, p);
  return sb::check_launch("gemm_fp8");
}

template <int EPI, class OUT, bool GROUPED>
int launch_product(const void* w, int64_t rows_w, int64_t ldw, const void* q, int64_t rows_q, int64_t ldq, const Fp8Params& p, int tile_n, int tiles_n,
                   cudaStream_t st) {
  const int tiles_m = EPI == kGated ? (p.half_rows + 63) / 64 : (p.M + kBlock - 1) / kBlock;
  if (tile_n == 16) return launch_tile<EPI, 16, OUT, GROUPED>(w, rows_w, ldw, q, rows_q, ldq, p, tiles_m, tiles_n, st);
  if constexpr (!GROUPED) {
    if (tile_n == 32) return launch_tile<EPI, 32, OUT, false>(w, rows_w, ldw, q, rows_q, ldq, p, tiles_m, tiles_n, st);
    if (tile_n == 64) return launch_tile<EPI, 64, OUT, false>(w, rows_w, ldw, q, rows_q, ldq, p, tiles_m, tiles_n, st);
    if (tile_n == kTokenRows) return launch_token<EPI, OUT>(w, rows_w, ldw, q, rows_q, ldq, p, tiles_m, tiles_n, st);
    if (p.ranges == 1) {
      // (a round of tiles takes pairs and single CTAs the same, within 5%, single CTAs a little longer: they are for where they need fewer of them.
      // [12000, 4096] of 300 tokens: 46 us on pairs, two rounds, 27.7 on single CTAs)
      const long long sms = sb::sm_count(), wide = EPI == kGated ? (p.half_rows + kBlock - 1) / kBlock : (p.M + 255) / 256;
      const int single_n = (p.n + kTokenRows - 1) / kTokenRows;
      if ((wide * single_n + sms - 1) / sms < (wide * tiles_n + sms / 2 - 1) / (sms / 2))
        return launch_pair<EPI, true, OUT, false, false>(w, rows_w, ldw, q, rows_q, ldq, p, single_n, st);
      return launch_pair<EPI, true, OUT, false, true>(w, rows_w, ldw, q, rows_q, ldq, p, tiles_n, st);
    }
    if constexpr (EPI != kGated) return launch_pair<EPI, false, OUT, false, true>(w, rows_w, ldw, q, rows_q, ldq, p, tiles_n, st);
  }
  return sb::fail("gemm_fp8: no form for tiles of %d tokens", tile_n);
}

int launch_quantize(const void* x, int xdtype, int64_t ldx, const int32_t* place, int copies, int n, int K, void* q, int64_t ldq,
                    float* scales, int64_t lds, cudaStream_t st) {
  const int blocks = (K + kBlock - 1) / kBlock;
  const dim3 grid((n + 7) / 8, (blocks + 1) / 2), block(256);
  if (grid.y > 65535) return sb::fail("quantize_fp8: %d columns are too many", K);
  const bool vec = ldx * (xdtype == 0 ? 4 : 2) % 16 == 0 && (reinterpret_cast<uintptr_t>(x) & 15) == 0;
  uint8_t* to = static_cast<uint8_t*>(q);
  auto run = [&](auto kernel, auto from) {
    sb::launch_pdl(kernel, grid, block, 0, st, from, ldx, place, copies, n, K, blocks, to, ldq, scales, lds);
    return sb::check_launch("quantize_fp8");
  };
  if (xdtype == 0) return vec ? run(quantize_kernel<float, true>, static_cast<const float*>(x)) : run(quantize_kernel<float, false>, static_cast<const float*>(x));
  return vec ? run(quantize_kernel<bf16, true>, static_cast<const bf16*>(x)) : run(quantize_kernel<bf16, false>, static_cast<const bf16*>(x));
}

// Tokens of a tile of the product; sets `split`, the K ranges of a CTA where they run on CTAs of their own (0: they do not). Up to 128 tokens they do,
// one each. More are for pairs of CTAs (gated with ranges, whose sums and totals would not fit a pair's registers: for single ones), unless a weight
// of several ranges has so few tiles that a cluster's CTAs, with one or two ranges each, are done sooner: in microseconds, a block of columns costs
// a pair some 0.38, a single CTA 0.42, a cluster's CTA 0.34; a pass of pairs begins and ends in 4, a round of single CTAs in 2.3, of clusters in 4.8
// gated, else in 6.6, with two ranges 7.5 (the first 6 of a further round). 256 tokens, [4096, 14336]: 49.7 us on pairs, 38.5 with a range each in
// two rounds, 31.9 with two each; [4096, 4096] 23.9, 24.1, 16.7; [2048, 4096] gated 19.6 on single ones, 11.4 with a range each; [2500, 2056] 13.0 on
// pairs, 14.2 with two each; 333 tokens, [6144, 4096]: 32.8 on pairs, 26.1 with a range each.
//
// More than 32 tokens of a weight with more tiles than SMs: walked too if the wide tiles then take half the rounds (a round of those takes half as
// long again). 64 tokens, [20000, 2048]: 19.8 and 15.6 us, [28000, 4096]: 31.2 and 26.6; [14000, 8192], one round either way: 27.1 and 39.6.
int token_tile(Fp8Params& p, int epilogue) {
  const bool gated = epilogue == kGated;
  const long long sms = sb::sm_count();
  p.split = p.ranges > 1;
  if (p.n <= 32) return p.n <= 16 ? 16 : 32;
  if (p.n <= kTokenRows) {
    const int rows = gated ? p.half_rows : p.M, narrow = gated ? 64 : kBlock;
    const long long tiles = (rows + narrow - 1) / narrow, wide = (rows + 2 * narrow - 1) / (2 * narrow);
    if (p.ranges == 1 && (tiles + sms - 1) / sms >= 2 * ((wide + sms - 1) / sms)) return kPairTokens;
    return p.n <= 64 ? 64 : kTokenRows;
  }
  if (p.ranges > 1) {
    const long long tiles = gated ? (p.half_rows + 63) / 64 : (p.M + kBlock - 1) / kBlock, of_tokens = (p.n + kTokenRows - 1) / kTokenRows;
    const long long pair_rounds = (tiles * ((p.n + kPairTokens - 1) / kPairTokens) + sms / 2 - 1) / (sms / 2);
    auto rounds = [&](int ctas) { return (tiles * of_tokens * ctas + sms - 1) / sms; };
    long long best = gated ? rounds(1) * (42 * p.blocks + 230) : pair_rounds * 38 * p.blocks + 400;
    p.split = 0;
    for (int each = 1; each <= 2 && each < p.ranges; ++each) {
      const long long c = rounds((p.ranges + each - 1) / each) * (34 * each * p.range_blocks + (gated ? 480 : 600)) + (gated ? 0 : each == 1 ? 60 : 150);
      if (c < best) best = c, p.split = each;
    }
    if (gated || p.split != 0) return kTokenRows;
  }
  return kPairTokens;
}

// The input as it is, for the forms that quantise it themselves: they copy 16 bytes at a time.
bool copied_input(const void* x, int xdtype, int64_t ldx) { return ldx % (xdtype == 0 ? 4 : 8) == 0 && (reinterpret_cast<uintptr_t>(x) & 15) == 0; }
void set_input(Fp8Params& p, const void* x, int xdtype, int64_t ldx) {
  p.x = x, p.ldx = ldx, p.x_f32 = xdtype == 0;
}

// Whether a layer's product of n tokens quantises its input itself.
bool quantises_itself(const void* x, int xdtype, int64_t ldx, int n, int M, int K) {
  if (n > kQuantRows || !copied_input(x, xdtype, ldx)) return false;
  const int blocks = (K + kBlock - 1) / kBlock, ranges = fp8_ranges((M + kBlock - 1) / kBlock, blocks);
  return (blocks + ranges - 1) / ranges <= kQuantBlocks;
}

// One product; x: the input that it quantises itself, or null: q and xs hold it. out_dtype 0 float32, 1 bfloat16.
int launch_gemm(const void* x, int xdtype, int64_t ldx, const void* q, int64_t ldq, const float* xs, int64_t ldxs, const void* w, int64_t ldw, const float* ws, void* out, int out_dtype,
                int64_t ldo, int n, int M, int K, int epilogue, int half_rows, const Gate& gate, cudaStream_t st) {
  Fp8Params p = {};
  p.out = out, p.ldo = ldo, p.x_scales = xs, p.ldxs = ldxs, p.w_scales = ws;
  p.n = n, p.M = M, p.K = K, p.blocks = (K + kBlock - 1) / kBlock, p.half_rows = half_rows;
  p.scale_rows = epilogue == kGated ? 2 * ((half_rows + kBlock - 1) / kBlock) : (M + kBlock - 1) / kBlock;
  p.ranges = fp8_ranges((M + kBlock - 1) / kBlock, p.blocks);
  p.range_blocks = (p.blocks + p.ranges - 1) / p.ranges;
  p.gate = gate;
  if (x != nullptr) set_input(p, x, xdtype, ldx);
  p.status = status_word();
  if (p.status == nullptr) return sb::fail("gemm_fp8: no status word on this device");
  const int tile = token_tile(p, epilogue), tiles_n = (n + tile - 1) / tile;
  if (tiles_n > 65535) return sb::fail("gemm_fp8: %d tokens are too many", n);
  if (epilogue == kAdd) return launch_product<kAdd, float, false>(w, M, ldw, q, n, ldq, p, tile, tiles_n, st);
  if (epilogue == kStore)
    return out_dtype == 0 ? launch_product<kStore, float, false>(w, M, ldw, q, n, ldq, p, tile, tiles_n, st)
                          : launch_product<kStore, bf16, false>(w, M, ldw, q, n, ldq, p, tile, tiles_n, st);
  return out_dtype == 0 ? launch_product<kGated, float, false>(w, M, ldw, q, n, ldq, p, tile, tiles_n, st)
                        : launch_product<kGated, bf16, false>(w, M, ldw, q, n, ldq, p, tile, tiles_n, st);
}
int check_quantized(const char* who, const void* q, int64_t ldq, int64_t ldxs, int n, int K) {
  if (n < 0 || K <= 0) return sb::fail("%s: %d rows of %d columns", who, n, K);
  if (ldq < K || ldq % 16 || (reinterpret_cast<uintptr_t>(q) & 15)) return sb::fail("%s: rows of 8-bit values are 16-byte aligned (stride %lld, %d columns)", who, (long long)ldq, K);
  if (ldxs < n) return sb::fail("%s: %lld scales for %d rows", who, (long long)ldxs, n);
  return 0;
}
int check_product(const char* who, const void* w, int64_t ldw, int out_dtype, int64_t ldo, int M, int K, int epilogue, int half_rows) {
  if (M <= 0 || epilogue < kStore || epilogue > kGated) return sb::fail("%s: %d weight rows, epilogue %d", who, M, epilogue);
  if (ldw < K || ldw % 16 || (reinterpret_cast<uintptr_t>(w) & 15)) return sb::fail("%s: weight rows are 16-byte aligned (stride %lld, %d columns)", who, (long long)ldw, K);
  if (epilogue == kGated && (half_rows <= 0 || 2 * half_rows != M)) return sb::fail("%s: a gated product has as many gate rows as up rows (%d of %d)", who, half_rows, M);
  if (out_dtype < 0 || out_dtype > 1 || (epilogue == kAdd && out_dtype != 0)) return sb::fail("%s: results are float32 or bfloat16, sums float32", who);
  if (ldo < (epilogue == kGated ? half_rows : M)) return sb::fail("%s: rows of %lld results for %d weight rows", who, (long long)ldo, M);
  return 0;
}

// Rows of a tile of the experts' products (a row's result does not depend on it). 16, quantised on the way in, where an expert gets few, else 128 on
// CTAs that walk tiles, which pays from nine or so on average if there are many pairs in all (64 experts of 2,048 x 1,408, six a token: 100 tokens
// 131 us in tiles of 16, 123 walked, 150 tokens 157 and 127; 20 tokens, two of four experts of 1,024 x 512: 24.3 and 28.2). Tiles of 256 on pairs
// of CTAs were no faster even with 1,000 rows an expert (82.6 us, 80.4 walked by single ones).
int64_t most_in_tiles_of_16(int64_t E) { return std::max<int64_t>(8 * E, std::min<int64_t>(16 * E, 256)); }
int expert_tile(int pairs, int E) { return pairs <= most_in_tiles_of_16(E) ? 16 : kTokenRows; }
int most_tiles(int pairs, int E, int tile) { return std::min(pairs, pairs / tile + std::min(pairs, E)); }

// Where an expert call's intermediate results lie in its scratch buffer, every one 256-byte aligned. z is for the products on tiles of 16 rows (the others
// quantise it as they make it), so for as many choices as those have at most: of 8,192 tokens, eight of 256 experts of 7,168 x 2,048, 16 MB and not 512. With more
// tokens every part is as large or larger: a buffer for some serves fewer.
struct ExpertScratch {
  int64_t order, place, list, xq, xs, z, zq, zs, parts, bytes, ldx, ldz, ldp;
};
ExpertScratch expert_scratch(int64_t n, int64_t top, int64_t E, int64_t W, int64_t F) {
  ExpertScratch s;
  const int64_t pairs = n * top;
  int64_t at = 0;
  auto take = [&](int64_t bytes) {
    const int64_t here = at;
    at += (bytes + 255) / 256 * 256;
    return here;
  };
  s.ldx = (W + 15) / 16 * 16, s.ldz = (F + 15) / 16 * 16, s.ldp = (W + 3) / 4 * 4;
  s.order = take(4 * pairs), s.place = take(4 * pairs), s.list = take(4 * (2 + 3 * pairs));
  s.xq = take(pairs * s.ldx), s.xs = take(4 * pairs * ((W + kBlock - 1) / kBlock));
  s.z = take(4 * std::min(pairs, most_in_tiles_of_16(E)) * s.ldz), s.zq = take(pairs * s.ldz), s.zs = take(4 * pairs * ((F + kBlock - 1) / kBlock));
  s.parts = take(4 * pairs * s.ldp);
  s.bytes = at;
  return s;
}

}  // namespace

SB_EXPORT void sb_gemm_fp8_use_status_word(int* device_word) { status_word_given() = device_word; }
// 0 if every wait of these kernels completed, else where one gave up; resets it. Until then the clustered and the token form store nothing.
SB_EXPORT int sb_gemm_fp8_status() {
  int* status = status_word();
  if (!status) return -1;
  int host = 0;
  if (cudaMemcpy(&host, status, sizeof(int), cudaMemcpyDeviceToHost) != cudaSuccess) return -2;
  if (host != 0) cudaMemset(status, 0, sizeof(int));
  return host;
}

// x [n][ldx] float32 (0) or bfloat16 (1) -> q [n][ldq] e4m3, scales [ceil(K / 128)][lds] float32.
SB_EXPORT int sb_quantize_fp8(const void* x, int xdtype, int64_t ldx, void* q, int64_t ldq, float* scales, int64_t lds, int n, int K, void* stream) {
  if (int rc = check_quantized("quantize_fp8", q, ldq, lds, n, K)) return rc;
  if (xdtype < 0 || xdtype > 1 || ldx < K) return sb::fail("quantize_fp8: rows of %lld elements, %d columns", (long long)ldx, K);
  if (n == 0) return 0;
  return launch_quantize(x, xdtype, ldx, nullptr, 1, n, K, q, ldq, scales, lds, static_cast<cudaStream_t>(stream));
}

// out = x . w^T of quantised x; epilogue 0 store, 1 add, 2 gated (w: half_rows gate rows, then as many up rows; act, limit, slope: the gate).
SB_EXPORT int sb_gemm_fp8(const void* q, int64_t ldq, const float* xs, int64_t ldxs, const void* w, int64_t ldw, const float* ws, void* out, int out_dtype,
                          int64_t ldo, int n, int M, int K, int epilogue, int half_rows, int act, float limit, float slope, void* stream) {
  if (int rc = check_quantized("gemm_fp8", q, ldq, ldxs, n, K)) return rc;
  if (int rc = check_product("gemm_fp8", w, ldw, out_dtype, ldo, M, K, epilogue, half_rows)) return rc;
  if (n == 0) return 0;
  Gate gate;
  gate.act = act, gate.limit = limit, gate.slope = slope;
  return launch_gemm(nullptr, 0, 0, q, ldq, xs, ldxs, w, ldw, ws, out, out_dtype, ldo, n, M, K, epilogue, half_rows, gate, static_cast<cudaStream_t>(stream));
}

// What a layer hands over with every call: buffers for the quantised input, q [rows][ldq] and x_scales [ceil(K / 128)][ldxs], and the weight.
typedef struct SbFp8Layer {
  void* q;
  int64_t ldq;
  float* x_scales;
  int64_t ldxs;
  const void* w;
  int64_t ldw;
  const float* w_scales;
  int32_t M, K, half_rows;
} SbFp8Layer;

// x is quantised, of few tokens perhaps on the way into the product (which leaves the buffers alone), and multiplied.
typedef struct SbFp8Call {
  const SbFp8Layer* layer;
  const void* x;
  int64_t ldx;
  void* out;
  int64_t ldo;
  int32_t x_dtype, out_dtype, n, epilogue, act;
  float limit, slope;
} SbFp8Call;

SB_EXPORT int sb_linear_fp8(const SbFp8Call* call, void* stream) {
  const SbFp8Call c = *call;
  const SbFp8Layer* l = c.layer;
  const void* x = c.x;
  void* out = c.out;
  const int64_t ldx = c.ldx, ldo = c.ldo;
  const int xdtype = c.x_dtype, out_dtype = c.out_dtype, n = c.n, epilogue = c.epilogue;
  if (int rc = check_quantized("linear_fp8", l->q, l->ldq, l->ldxs, n, l->K)) return rc;
  if (int rc = check_product("linear_fp8", l->w, l->ldw, out_dtype, ldo, l->M, l->K, epilogue, l->half_rows)) return rc;
  if (xdtype < 0 || xdtype > 1 || ldx < l->K) return sb::fail("linear_fp8: rows of %lld elements, %d columns", (long long)ldx, l->K);
  if (n == 0) return 0;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const bool itself = quantises_itself(x, xdtype, ldx, n, l->M, l->K);
  if (!itself) {
    if (int rc = launch_quantize(x, xdtype, ldx, nullptr, 1, n, l->K, l->q, l->ldq, l->x_scales, l->ldxs, st)) return rc;
  }
  Gate gate;
  gate.act = c.act, gate.limit = c.limit, gate.slope = c.slope;
  return launch_gemm(itself ? x : nullptr, xdtype, ldx, l->q, l->ldq, l->x_scales, l->ldxs, l->w, l->ldw, l->w_scales, out, out_dtype, ldo, n, l->M, l->K, epilogue,
                     epilogue == kGated ? l->half_rows : 0, gate, st);
}

// Bytes of scratch that `sb_experts_fp8` needs for n tokens.
SB_EXPORT int64_t sb_experts_fp8_scratch(int n, int top, int E, int W, int F) { return expert_scratch(n, top, E, W, F).bytes; }

// out[t] = sum over k of weights[k][t] D_e (silu(G_e x_t) * (U_e x_t)), e = choice[t][k] (no expert: no term). gate_up [E 2F][ldg] e4m3 (an
// expert's gate rows, then its up rows) with scales [E 2 ceil(F / 128)][ceil(W / 128)], down [E W][ldd] with [E ceil(W / 128)][ceil(F / 128)].
// The gated products stay in 32-bit until they are quantised.
typedef struct SbFp8Experts {
  const void* gate_up;
  int64_t ldg;
  const float* gate_up_scales;
  const void* down;
  int64_t ldd;
  const float* down_scales;
  int32_t experts, width, inner;
} SbFp8Experts;

typedef struct SbFp8ExpertsCall {
  const SbFp8Experts* experts;
  const void* x;
  int64_t ldx;
  const int32_t* choice;
  const float* weights;
  void* out;
  int64_t ldo;
  void* scratch;
  int64_t scratch_bytes;
  int32_t x_dtype, out_dtype, n, top;
} SbFp8ExpertsCall;

SB_EXPORT int sb_experts_fp8(const SbFp8ExpertsCall* call, void* stream) {
  const SbFp8ExpertsCall c = *call;
  const SbFp8Experts* l = c.experts;
  const void* x = c.x;
  const int32_t* choice = c.choice;
  const float* weights = c.weights;
  void *out = c.out, *scratch = c.scratch;
  const int64_t ldx = c.ldx, ldo = c.ldo, scratch_bytes = c.scratch_bytes;
  const int xdtype = c.x_dtype, out_dtype = c.out_dtype, n = c.n, top = c.top;
  const void *gate_up = l->gate_up, *down = l->down;
  const float *gate_up_scales = l->gate_up_scales, *down_scales = l->down_scales;
  const int64_t ldg = l->ldg, ldd = l->ldd;
  const int E = l->experts, W = l->width, F = l->inner;
  const char* who = "experts_fp8";
  if (n < 0 || top < 1 || E < 1 || E > kMaxExperts || W < 1 || F < 1) return sb::fail("%s: %d of %d experts (at most %d), %d tokens, sizes %d and %d", who, top, E, kMaxExperts, n, W, F);
  if (static_cast<int64_t>(n) * top > (1 << 24) || static_cast<int64_t>(E) * std::max(2 * F, W) > 0x7FFFFFFF)
    return sb::fail("%s: %d tokens with %d choices, %d experts of %d x %d: too many rows", who, n, top, E, F, W);
  if (xdtype < 0 || xdtype > 1 || ldx < W || out_dtype < 0 || out_dtype > 1 || ldo < W) return sb::fail("%s: rows of %lld and %lld elements for a width of %d", who, (long long)ldx, (long long)ldo, W);
  if (int rc = check_product(who, gate_up, ldg, 0, F, 2 * F, W, kGated, F)) return rc;
  if (int rc = check_product(who, down, ldd, 0, W, W, F, kStore, 0)) return rc;
  const ExpertScratch s = expert_scratch(n, top, E, W, F);
  if (scratch_bytes < s.bytes || (reinterpret_cast<uintptr_t>(scratch) & 15)) return sb::fail("%s: %lld bytes of scratch where %lld are needed", who, (long long)scratch_bytes, (long long)s.bytes);
  if (n == 0) return 0;
  int* status = status_word();
  if (status == nullptr) return sb::fail("%s: no status word on this device", who);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  uint8_t* base = static_cast<uint8_t*>(scratch);
  int32_t *order = reinterpret_cast<int32_t*>(base + s.order), *place = reinterpret_cast<int32_t*>(base + s.place), *list = reinterpret_cast<int32_t*>(base + s.list);
  float *xs = reinterpret_cast<float*>(base + s.xs), *z = reinterpret_cast<float*>(base + s.z), *zs = reinterpret_cast<float*>(base + s.zs);
  float* parts = reinterpret_cast<float*>(base + s.parts);
  const int pairs = n * top, tile = expert_tile(pairs, E), tiles = most_tiles(pairs, E, tile);
  if (tiles > 65535) return sb::fail("%s: %d tiles of rows are too many", who, tiles);
  const bool quant_x = tile <= kQuantRows && copied_input(x, xdtype, ldx), few = quant_x && pairs <= kFewChoices;
  if (!few) {
    sb::launch_pdl(expert_order_kernel, dim3(1), dim3(kOrderThreads), 0, st, choice, n, top, E, tile, order, place, list);
    if (int rc = sb::check_launch(who)) return rc;
  }
  if (!quant_x) {
    if (int rc = launch_quantize(x, xdtype, ldx, place, top, n, W, base + s.xq, s.ldx, xs, pairs, st)) return rc;
  }
  Fp8Params p = {};
  if (quant_x) set_input(p, x, xdtype, ldx), p.x_gathered = 1;
  if (few) p.choice = choice, p.choices = pairs, p.top = top, p.experts = E;
  else p.tiles = list, p.order = order;
  p.status = status, p.n = n, p.ranges = 1;
  p.out = z, p.ldo = s.ldz, p.x_scales = xs, p.ldxs = pairs, p.w_scales = gate_up_scales, p.M = 2 * F, p.K = W, p.half_rows = F;
  p.blocks = p.range_blocks = (W + kBlock - 1) / kBlock, p.scale_rows = 2 * ((F + kBlock - 1) / kBlock);
  const int64_t rows_g = static_cast<int64_t>(E) * 2 * F, rows_d = static_cast<int64_t>(E) * W;
  const bool walks = tile == kTokenRows;          // (those quantise the gated products themselves)
  if (walks) {
    p.out = base + s.zq, p.ldo = s.ldz, p.z_scales = zs;
    if (int rc = launch_pair<kGated, true, uint8_t, true, false>(gate_up, rows_g, ldg, base + s.xq, pairs, s.ldx, p, tiles, st)) return rc;
  } else {
    if (int rc = launch_product<kGated, float, true>(gate_up, rows_g, ldg, base + s.xq, pairs, s.ldx, p, tile, tiles, st)) return rc;
    set_input(p, z, 0, s.ldz), p.x_gathered = 0;
  }
  p.out = parts, p.ldo = s.ldp, p.x_scales = zs, p.w_scales = down_scales, p.M = W, p.K = F, p.half_rows = 0;
  p.blocks = p.range_blocks = (F + kBlock - 1) / kBlock, p.scale_rows = (W + kBlock - 1) / kBlock;
  if (int rc = walks ? launch_pair<kStore, true, float, true, false>(down, rows_d, ldd, base + s.zq, pairs, s.ldz, p, tiles, st)
                     : launch_product<kStore, float, true>(down, rows_d, ldd, base + s.zq, pairs, s.ldz, p, tile, tiles, st))
    return rc;
  const dim3 grid(n, (W + 1023) / 1024);
  if (grid.y > 65535) return sb::fail("%s: %d features are too many", who, W);
  auto combine = [&](auto kernel, auto to) {
    sb::launch_pdl(kernel, grid, dim3(128), 0, st, static_cast<const float*>(parts), s.ldp, few ? static_cast<const int32_t*>(nullptr) : place, choice,
                   E, weights, n, top, W, to, ldo);
  };
  const int size = out_dtype == 0 ? 4 : 2;
  const bool vec = ldo % 4 == 0 && (reinterpret_cast<uintptr_t>(out) & (4 * size - 1)) == 0;
  if (out_dtype == 0) vec ? combine(expert_combine_kernel<float, true>, static_cast<float*>(out)) : combine(expert_combine_kernel<float, false>, static_cast<float*>(out));
  else vec ? combine(expert_combine_kernel<bf16, true>, static_cast<bf16*>(out)) : combine(expert_combine_kernel<bf16, false>, static_cast<bf16*>(out));
  return sb::check_launch(who);
}

// i: 0 q, 1 ldq, 2 x scales, 3 ldxs, 4 w, 5 ldw, 6 w scales, 7 M, 8 K, 9 half_rows, 10 x, 11 x dtype, 12 ldx, 13 out, 14 out dtype, 15 ldo,
// 16 epilogue, 17 act, 18 wanted rows (else the step's tokens). f: 0 limit, 1 slope
SB_EXPORT int sb_op_linear_fp8(const SbOp* op, const SbStep* s, void* stream) {
  using namespace sbstep;
  const int n = op->i[18] != 0 ? s->wanted : s->n;
  if (n <= 0) return SB_OP_SKIPPED;
  const SbFp8Layer l = {ptr<void>(op->i[0]), op->i[1], ptr<float>(op->i[2]), op->i[3], ptr<void>(op->i[4]), op->i[5], ptr<float>(op->i[6]),
                        (int)op->i[7], (int)op->i[8], (int)op->i[9]};
  const SbFp8Call c = {&l, ptr<void>(op->i[10]), op->i[12], ptr<void>(op->i[13]), op->i[15], (int)op->i[11], (int)op->i[14], n, (int)op->i[16], (int)op->i[17],
                       (float)op->f[0], (float)op->f[1]};
  return sb_linear_fp8(&c, stream) != 0 ? SB_OP_FAILED : SB_OP_LAUNCHED;
}

// i: 0 gate_up, 1 ldg, 2 gate_up scales, 3 down, 4 ldd, 5 down scales, 6 experts, 7 width, 8 inner, 9 x, 10 x dtype, 11 ldx, 12 choice [n][top],
// 13 weights [top][n], 14 out, 15 out dtype, 16 ldo, 17 top, 18 scratch, 19 its bytes
SB_EXPORT int sb_op_experts_fp8(const SbOp* op, const SbStep* s, void* stream) {
  using namespace sbstep;
  if (s->n <= 0) return SB_OP_SKIPPED;
  const SbFp8Experts l = {ptr<void>(op->i[0]), op->i[1], ptr<float>(op->i[2]), ptr<void>(op->i[3]), op->i[4], ptr<float>(op->i[5]), (int)op->i[6],
                          (int)op->i[7], (int)op->i[8]};
  const SbFp8ExpertsCall c = {&l, ptr<void>(op->i[9]), op->i[11], ptr<int32_t>(op->i[12]), ptr<float>(op->i[13]), ptr<void>(op->i[14]), op->i[16],
                              ptr<void>(op->i[18]), op->i[19], (int)op->i[10], (int)op->i[15], s->n, (int)op->i[17]};
  return sb_experts_fp8(&c, stream) != 0 ? SB_OP_FAILED : SB_OP_LAUNCHED;
}
