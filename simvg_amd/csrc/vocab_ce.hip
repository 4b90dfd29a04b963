// simvg-build-flags: -Wno-inline-asm
// Softmax cross entropy over a large vocabulary without its logits, forward and backward.
//
//   z = x w^T + b  [M, V],  lse_i = log sum_v exp(z_iv),  loss_i = lse_i - z_i,target(i)          (0 where the target is ignored)
//   backward, for the gradients g_i of the rows' losses:  e_iv = exp(z_iv - lse_i) - [v = target(i)]
//     dx_i = g_i sum_v e_iv w_v,   dw_v = sum_i e_iv g_i x_i,   db_v = sum_i g_i e_iv
//
// Bound by the matrix pipes (2 M V K forward, 6 M V K backward: the logits are computed again, they are never kept), for few rows by
// reading w once.  Forward: a matrix product whose epilogue keeps, for each row and each 128 or 256 words, the maximum and the sum of the
// exponentials; a second kernel joins them.  Backward, in pieces of the vocabulary: (1) the logits of the piece again, as e rounded to
// 16 bits into a workspace that stays near the caches; (2) its share of dx, added to sums in 32 bits; (3) its rows of dw.  (2) and (3)
// are products over the vocabulary and over the rows: their operands lie "the other way round" in memory and are read from LDS with
// the transposing ds_read_b64_tr_b16, so that nothing is ever laid out twice.
//
// Measured, medians, at 8191 rows, 64010 words, K = 1024, bf16: forward 0.94 ms (1.15 PFLOP/s; the library's product alone, which writes
// the logits, 1.05 ms), backward 2.96 ms (1.09) in four pieces of e 273, dx 243 and dw 212 us (the library's products of a piece: 285 and
// 291 us for the last two); the best of several runs were 0.90 and 2.87 ms.  Half of the time the matrix pipes work, at 1.75 to 1.83 GHz, which they themselves bring down; the rest is the
// start and the epilogue of a tile (28 us, of which 18 are products), which one workgroup to a compute unit cannot cover.  20 rows, 64010
// words, K = 768: 17 us for 98 MB of w, 5.7 TB/s.
//
// Rounding to 16 bits, by choice: e (one rounding, relative 2^-9 bf16 / 2^-12 fp16; in fp16 times 2^14, so that a probability of 2^-28
// keeps all its bits) and g x / max|g| where the rows' gradients differ (where they are equal or 0 the factor is 1 or 0: exact).
// Everything that is summed is summed in 32 bits; db is summed before the rounding.
#include <type_traits>
#include <utility>

#include "seq.h"

struct simvg_vocab_ce_args {
  int dtype, M, V, K;
  const void* x; long ldx;                                   // [M][K]
  const void* w; long ldw;                                   // [V][K]
  const float* bias;                                         // [V] or null
  const long* target; long ignore_index;                     // [M]
  float *loss, *lse;                                         // [M]; lse: backward input
  const float* dloss;                                        // [M]
  void* dx; long lddx; void* dw; long lddw; float* dbias;    // backward outputs; dbias null with bias null
  void* ws; long ws_bytes;
};

namespace {
using namespace seq;

constexpr float LOG2E = 1.44269504088896340736f;
constexpr float NEG_INF = -__builtin_huge_valf();
constexpr float FAR = 4096.f;                                // logits beyond it have their maximum subtracted before the scaling, not in its fma
constexpr int BK = 64;                                       // contracted values of a stage: a row's are one line of 128 bytes

__device__ __forceinline__ f32x16 zero16() { return (f32x16){0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f}; }
__device__ __forceinline__ int acc_row(int r, int lane) { return (r >> 2) * 8 + (lane >> 5) * 4 + (r & 3); }
// in a branch that few tiles take: keeps hipcc from computing it for all of them and selecting
__device__ __forceinline__ void stay_a_branch() { asm volatile(""); }

// ------------------------------------------------------------------------------------------------- the matrix product
// A wave's tile of 128 x 64 is 128 accumulators and 6 fragments of 1 KiB for 8 MFMAs of 32 cycles; eight waves make 256 x 256, one
// workgroup to a compute unit.  (256 x 128 in four waves, two workgroups to a compute unit with stages of 32 values, so that one's
// epilogue runs beside the other's products: 1.08 against 1.01 ms at the time for the forward pass at 8191 x 64010 x 1024, bound by the
// L2's requests: half lines, and half as many products for each.)
//
// One operand of a workgroup's tile: R rows (or columns) of the result by BK contracted values per stage.
//   T = false: memory [R][contracted], a stage is R rows of 128 bytes;  T = true: memory [contracted][R], BK rows of 2 R bytes.
// In LDS, slots of 16 bytes are permuted within a row so that the fragment reads touch every bank once: 16 rows of one slot
// (ds_read_b128) or 4 rows of 4 neighbouring slots (ds_read_b64_tr_b16) are one cycle's.
template <int R, bool T, int WAVES> struct Operand {
  static constexpr int BYTES = R * BK * 2, ROW = T ? R * 2 : BK * 2, PIECES = BYTES / 1024 / WAVES;
  static_assert(PIECES >= 1 && (!T || R >= 128) && WAVES % 2 == 0, "tile of an operand");
  static __device__ __forceinline__ int at(int row, int slot) {
    return row * ROW + ((slot ^ (T ? (row & 3) << 2 : (row >> 1 & 1) << 2 | (row >> 2 & 3))) << 4);
  }

  // what a lane adds to a stage's start for its part of a fragment; the rest of an address is a constant in the instruction
  typedef __attribute__((address_space(3))) const char* Lds;
  Lds lane_at[T ? 4 : BK / 16];
  // the wave's fragments are first .. (in units of 32 rows); `base`: where the operand's stages start
  __device__ __forceinline__ void init_reads(const char* base, int first, int lane) {
    const Lds b = (Lds)(const __attribute__((address_space(3))) void*)LDS_PTR(base);
    if constexpr (T) {
      const int i = lane & 15, row = 8 * (lane >> 5) + (i >> 2);
#pragma unroll
      for (int f = 0; f < 4; ++f) {
        const int col = (first + f) * 32 + (lane >> 4 & 1) * 16 + 4 * (i & 3);
        lane_at[f] = b + at(row, col >> 3) + (col & 7) * 2;
      }
    } else {
#pragma unroll
      for (int ks = 0; ks < BK / 16; ++ks) lane_at[ks] = b + at(first * 32 + (lane & 31), ks * 2 + (lane >> 5));
    }
  }
  // fragment f of the wave's, contracted values 16 ks .. of stage `st`
  __device__ __forceinline__ lpx8_t frag(int st, int f, int ks) const {
    if constexpr (T) {
      typedef __attribute__((address_space(3))) lpx4_t* P;
      const lpx4_t lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((P)(lane_at[f] + st * BYTES + ks * 16 * ROW));
      const lpx4_t hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((P)(lane_at[f] + st * BYTES + (ks * 16 + 4) * ROW));
      return (lpx8_t){lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
    } else {
      return *(const __attribute__((address_space(3))) lpx8_t*)(lane_at[ks] + st * BYTES + f * 32 * ROW);
    }
  }

  // HBM -> LDS, 1 KiB a piece, wave w's pieces are w, w + WAVES ..
  unsigned off[PIECES], lds, step;
  unsigned long next;                                        // the next stage's first value
  int inner, left;                                           // the lane's first contracted value of a stage (T: of its first piece); how many are left
  // rows: what there is of the tile's rows, depth: of contracted values from `base` on
  __device__ __forceinline__ void init_stages(const unsigned short* base, long ld, int rows, int depth, const char* to, int wave, int lane) {
    next = (unsigned long)base;
    step = T ? (unsigned)(BK * 2) * (unsigned)ld : BK * 2;
    lds = lds_addr(to) + wave * 1024;
    left = depth;
#pragma unroll
    for (int i = 0; i < PIECES; ++i) {
      const int byte = (i * WAVES + wave) * 1024 + lane * 16, row = byte / ROW;
      const int slot = (at(row, byte % ROW / 16) - row * ROW) >> 4;            // the permutation is its own inverse
      if (i == 0) inner = T ? row : slot * 8;                // T = false: the same in every piece (whole eights of rows apart)
      off[i] = (T ? slot * 8 < rows : row < rows) ? (unsigned)row * (unsigned)ld * 2 + slot * 16 : DMA_NOTHING;
    }
  }
  // half Q of the next stage's pieces, to place ST
  template <int ST, int Q> __device__ __forceinline__ void half() {
    constexpr int FROM = PIECES * Q / 2, N = PIECES * (Q + 1) / 2 - FROM;
    const u32x4_t b = {(unsigned)next, (unsigned)(next >> 32) & 0xffffu, DMA_NOTHING - 1, 0x00020000u};
    unsigned o[N > 0 ? N : 1];
#pragma unroll
    for (int i = 0; i < N; ++i) o[i] = off[FROM + i];
    if (left < BK) {                                         // zeros behind the last contracted value
      stay_a_branch();
#pragma unroll
      for (int i = 0; i < N; ++i)
        if (inner + (T ? (FROM + i) * WAVES * 1024 / ROW : 0) >= left) o[i] = DMA_NOTHING;
    }
    issue<ST, FROM>(b, o, std::make_integer_sequence<int, N>{});
    if (Q == 1) {
      next += step;
      left -= BK;
    }
  }
  template <int ST, int FROM, int... I> __device__ __forceinline__ void issue(u32x4_t b, const unsigned* o, std::integer_sequence<int, I...>) {
    (dma16_at<ST * BYTES + (FROM + I) * WAVES * 1024>(b, lds, o[I]), ...);
  }
};

// acc[i][j] += A rows (WA of the wave's, 32 i ..) x B rows (WB, 32 j ..): registers run over A's rows, lanes over B's
template <class E, int RA, bool TA, int RB, bool TB, int WA, int WB, int STAGES>
struct Product {
  static constexpr int WAVES = (RA / WA) * (RB / WB), THREADS = WAVES * 64, NA = WA / 32, NB = WB / 32;
  using OA = Operand<RA, TA, WAVES>;
  using OB = Operand<RB, TB, WAVES>;
  static constexpr int B_AT = STAGES * OA::BYTES, LDS = B_AT + STAGES * OB::BYTES, IN_FLIGHT = OA::PIECES + OB::PIECES;
  static __device__ __forceinline__ int wave_a(int wave) { return wave / (RB / WB) * WA; }
  static __device__ __forceinline__ int wave_b(int wave) { return wave % (RB / WB) * WB; }

  // The fragments of a step are read while the step before is multiplied, across the stages' border too: the barrier that makes a stage
  // visible stands before the products of the last step of the stage before, whose fragments have all been read by then -- so the
  // matrix pipes have work behind it, and the stage's place in LDS is free for the one STAGES further on.
  static __device__ __forceinline__ void run(f32x16 (&acc)[NA][NB], OA& oa, OB& ob, int stages) {
    if (stages <= 0) return;
    lpx8_t a[2][NA], b[2][NB];
    auto ask = [&](auto st, auto q) __attribute__((always_inline)) {
      oa.template half<decltype(st)::value, decltype(q)::value>();
      ob.template half<decltype(st)::value, decltype(q)::value>();
    };
    using I0 = std::integral_constant<int, 0>;
    using I1 = std::integral_constant<int, 1>;
    using I2 = std::integral_constant<int, 2>;
    auto ask_all = [&](auto st) __attribute__((always_inline)) { ask(st, I0{}); ask(st, I1{}); };
    auto read = [&](auto st, int ks) __attribute__((always_inline)) {
      constexpr int S = decltype(st)::value;
#pragma unroll
      for (int j = 0; j < NB; ++j) b[ks & 1][j] = ob.frag(S, j, ks);
#pragma unroll
      for (int i = 0; i < NA; ++i) a[ks & 1][i] = oa.frag(S, i, ks);
    };
    // the products of one step
    auto multiply = [&](int k) __attribute__((always_inline)) {
#pragma unroll
      for (int i = 0; i < NA; ++i)
#pragma unroll
        for (int j = 0; j < NB; ++j) acc[i][j] = E::mfma(a[k][i], b[k][j], acc[i][j]);
      __builtin_amdgcn_sched_barrier(0);
    };
    ask_all(I0{});
    if (stages > 1) ask_all(I1{});
    if (STAGES == 3 && stages > 2) ask_all(I2{});
    if (stages >= STAGES) dma_wait<(STAGES - 1) * IN_FLIGHT>(); else dma_wait<0>();
    wave_barrier_only();
    read(I0{}, 0);
    // what goes to the place of the stage before is asked for in two halves, in two steps: the eight waves' pieces at once fill the
    // queue of the load unit, and a wave that waits there multiplies nothing (forward pass 934 -> 900 us)
    auto stage = [&](int kt, auto st) __attribute__((always_inline)) {
      constexpr int S = decltype(st)::value;
      const std::integral_constant<int, (S + STAGES - 1) % STAGES> before;
      const bool more = kt > 0 && kt - 1 + STAGES < stages;
      read(st, 1);
      if (more) ask(before, I1{});
      multiply(0);
      read(st, 2);
      multiply(1);
      read(st, 3);
      multiply(0);
      if (kt + 1 < stages) {
        if (kt + STAGES - 1 < stages) dma_wait<(STAGES - 2) * IN_FLIGHT>(); else dma_wait<0>();
        wave_barrier_only();
        read(std::integral_constant<int, (S + 1) % STAGES>{}, 0);
        if (kt + STAGES < stages) ask(st, I0{});
      }
      multiply(1);
    };
    for (int kt = 0;;) {
      stage(kt, I0{});
      if (++kt >= stages) break;
      stage(kt, I1{});
      if (++kt >= stages) break;
      if constexpr (STAGES == 3) {
        stage(kt, I2{});
        if (++kt >= stages) break;
      }
    }
    __syncthreads();                                         // the epilogues use the LDS
  }
  static __device__ __forceinline__ void zero(f32x16 (&acc)[NA][NB]) {
#pragma unroll
    for (int i = 0; i < NA; ++i)
#pragma unroll
      for (int j = 0; j < NB; ++j) acc[i][j] = zero16();
  }
};

// Tiles in bands of `band` tiles of the inner direction: the workgroups that run at the same time on an XCD (bid mod 8) are neighbours
// in this order and share their operands in its L2.
__device__ __forceinline__ void tile_of(int id, int n, int outer, int inner, int band, int& to, int& ti) {
  const int q = n >> 3, r = n & 7, xcd = id & 7;
  id = (xcd < r ? xcd * (q + 1) : r * (q + 1) + (xcd - r) * q) + (id >> 3);
  const int per = outer * band, g = id / per, width = min(band, inner - g * band), l = id - g * per;
  to = l / width;
  ti = g * band + l % width;
}

// a row takes part if its target is a word; otherwise (ignored, or no word at all) its gradient is nothing
__device__ __forceinline__ bool is_word(const simvg_vocab_ce_args& a, long t) { return t != a.ignore_index && t >= 0 && t < a.V; }

// the words' bias: to LDS before the products, and added behind them (64 loads a lane, whose wait nothing covers there, are 16 reads)
template <int RA>
__device__ __forceinline__ void bias_to_lds(const simvg_vocab_ce_args& a, int v0, const char* to, int wave, int lane) {
  const unsigned long p = (unsigned long)(a.bias + v0);
  const u32x4_t b = {(unsigned)p, (unsigned)(p >> 32) & 0xffffu, DMA_NOTHING - 1, 0x00020000u};
  if (wave < RA / 64) dma4(b, lds_addr(to) + wave * 256, v0 + wave * 64 + lane < a.V ? (wave * 64 + lane) * 4u : DMA_NOTHING);
}
template <int NA, int NB>
__device__ __forceinline__ void add_bias(f32x16 (&acc)[NA][NB], const char* from, int lane) {       // from: the wave's first word's
#pragma unroll
  for (int i = 0; i < NA; ++i)
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const f32x4_t b = *(const f32x4_t*)(from + (i * 32 + q * 8 + (lane >> 5) * 4) * 4);
#pragma unroll
      for (int j = 0; j < NB; ++j)
#pragma unroll
        for (int r = 0; r < 4; ++r) acc[i][j][4 * q + r] += b[r];
    }
}

// ------------------------------------------------------------------------------------------------------------- forward
// words in registers, rows in lanes: [tile of RA words][M] (maximum, sum of exp2) and the targets' logits
template <class E, int RA, int RB, int WA, int WB, int STAGES>
__global__ __launch_bounds__((RA / WA) * (RB / WB) * 64, 2) void ce_fwd_kernel(simvg_vocab_ce_args a, float2* part, float* zt) {
  using P = Product<E, RA, false, RB, false, WA, WB, STAGES>;
  extern __shared__ __attribute__((aligned(16))) char smem[];
  const int tv = cdiv(a.V, RA), tm = cdiv(a.M, RB);
  int iv, im;
  tile_of(blockIdx.x, tv * tm, tv, tm, 4, iv, im);
  const int v0 = iv * RA, m0 = im * RB, lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  f32x16 acc[P::NA][P::NB];
  P::zero(acc);
  typename P::OA oa;
  typename P::OB ob;
  oa.init_stages((const unsigned short*)a.w + (long)v0 * a.ldw, a.ldw, min(RA, a.V - v0), a.K, smem, wave, lane);
  ob.init_stages((const unsigned short*)a.x + (long)m0 * a.ldx, a.ldx, min(RB, a.M - m0), a.K, smem + P::B_AT, wave, lane);
  oa.init_reads(smem, P::wave_a(wave) / 32, lane);
  ob.init_reads(smem + P::B_AT, P::wave_b(wave) / 32, lane);
  if (a.bias) bias_to_lds<RA>(a, v0, smem + P::LDS, wave, lane);
  P::run(acc, oa, ob, cdiv(a.K, BK));
  const int wv = v0 + P::wave_a(wave), wm = P::wave_b(wave);
  if (a.bias) add_bias(acc, smem + P::LDS + P::wave_a(wave) * 4, lane);
  if (wv + WA > a.V) {
    stay_a_branch();
#pragma unroll
    for (int i = 0; i < P::NA; ++i)
#pragma unroll
      for (int r = 0; r < 16; ++r)
#pragma unroll
        for (int j = 0; j < P::NB; ++j)
          if (wv + i * 32 + acc_row(r, lane) >= a.V) acc[i][j][r] = NEG_INF;
  }
  float2* joined = (float2*)smem;                            // [RA / WA][RB]
#pragma unroll
  for (int j = 0; j < P::NB; ++j) {
    const int mr = wm + j * 32 + (lane & 31), m = m0 + mr;
    const long t = m < a.M ? a.target[m] : -1;
    const int local = t >= wv && t < wv + WA && t < a.V ? (int)(t - wv) : -1;
    if (__any(local >= 0)) {
      stay_a_branch();
#pragma unroll
      for (int i = 0; i < P::NA; ++i)
#pragma unroll
        for (int r = 0; r < 16; ++r)
          if (local == i * 32 + acc_row(r, lane)) zt[m] = acc[i][j][r];
    }
    float top = NEG_INF, sum = 0.f;
#pragma unroll
    for (int i = 0; i < P::NA; ++i)
#pragma unroll
      for (int r = 0; r < 16; ++r) top = fmaxf(top, acc[i][j][r]);
    top = fmaxf(top, __shfl_xor(top, 32, 64));
    float ref = top == NEG_INF ? 0.f : top * LOG2E;
    // `ref` is rounded, and off by hundreds of powers of two in a tile of words that a bias of -1e10 takes out, by all of them at -1e38:
    // the exponentials there would be inf, not 1
    if (__any(fabsf(ref) > FAR)) {
      stay_a_branch();
      const bool far = fabsf(ref) > FAR;                     // each row by itself: what another one is far off changes no bit of it
#pragma unroll
      for (int i = 0; i < P::NA; ++i)
#pragma unroll
        for (int r = 0; r < 16; ++r) acc[i][j][r] -= far ? top : 0.f;
      if (far) ref = 0.f;
    }
#pragma unroll
    for (int i = 0; i < P::NA; ++i)
#pragma unroll
      for (int r = 0; r < 16; ++r) sum += __builtin_amdgcn_exp2f(fmaf(acc[i][j][r], LOG2E, -ref));
    sum += __shfl_xor(sum, 32, 64);
    if (lane < 32) joined[wave / (RB / WB) * RB + mr] = make_float2(top, sum);
  }
  __syncthreads();
  if (threadIdx.x < RB && m0 + (int)threadIdx.x < a.M) {
    float top = NEG_INF, sum = 0.f;
#pragma unroll
    for (int w = 0; w < RA / WA; ++w) top = fmaxf(top, joined[w * RB + threadIdx.x].x);
    const float ref = top == NEG_INF ? 0.f : top;
#pragma unroll
    for (int w = 0; w < RA / WA; ++w) {
      const float2 p = joined[w * RB + threadIdx.x];
      sum += p.y * __builtin_amdgcn_exp2f((p.x - ref) * LOG2E);
    }
    part[(long)iv * a.M + m0 + threadIdx.x] = make_float2(top, sum);
  }
}
// 8 rows and 128 strands of word tiles to a workgroup
__global__ __launch_bounds__(1024) void ce_join_kernel(simvg_vocab_ce_args a, const float2* part, const float* zt, int groups) {
  __shared__ float tops[128][9], sums[128][9];
  const int c = threadIdx.x & 7, s = threadIdx.x >> 3, m = blockIdx.x * 8 + c;
  float top = NEG_INF, sum = 0.f;
  if (m < a.M) {
#pragma unroll 4
    for (int g = s; g < groups; g += 128) {
      const float2 p = part[(long)g * a.M + m];
      const float to = fmaxf(top, p.x), ref = to == NEG_INF ? 0.f : to;
      sum = sum * __builtin_amdgcn_exp2f((top - ref) * LOG2E) + p.y * __builtin_amdgcn_exp2f((p.x - ref) * LOG2E);
      top = to;
    }
  }
  tops[s][c] = top;
  sums[s][c] = sum;
  __syncthreads();
  for (int n = 64; n > 0; n >>= 1) {
    if (s < n) {
      const float t1 = tops[s + n][c], to = fmaxf(top, t1), ref = to == NEG_INF ? 0.f : to;
      sum = sum * __builtin_amdgcn_exp2f((top - ref) * LOG2E) + sums[s + n][c] * __builtin_amdgcn_exp2f((t1 - ref) * LOG2E);
      top = to;
      tops[s][c] = top;
      sums[s][c] = sum;
    }
    __syncthreads();
  }
  if (s == 0 && m < a.M) {
    const float lse = (top == NEG_INF ? 0.f : top) + __builtin_logf(sum);
    const long target = a.target[m];
    a.lse[m] = lse;
    // a target that is neither a word nor ignored is a mistake of the caller's: its loss says so
    a.loss[m] = target == a.ignore_index ? 0.f : is_word(a, target) ? lse - zt[m] : __builtin_nanf("");
  }
}

// The rows' losses to one: their sum, or their mean over the rows that are not ignored, and how many those are (1 for a sum: what a
// row's gradient is divided by).  One workgroup, every run adds in the same order, in 64 bits; no counters to be cleared, so that a captured
// graph holds nothing but kernels (torch's sum over some hundred thousand rows clears one by a memset).
__global__ __launch_bounds__(1024) void ce_reduce_kernel(const float* loss, const long* target, long ignore_index, int M, int mean, float* total,
                                                         float* count) {
  __shared__ double sums[16];
  __shared__ int counts[16];
  double sum = 0.;
  int n = 0;
#pragma unroll 8
  for (int m = threadIdx.x; m < M; m += 1024) {
    sum += loss[m];
    n += target[m] != ignore_index;
  }
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) {
    sum += __shfl_xor(sum, o, 64);
    n += __shfl_xor(n, o, 64);
  }
  if ((threadIdx.x & 63) == 0) { sums[threadIdx.x >> 6] = sum; counts[threadIdx.x >> 6] = n; }
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int i = 1; i < 16; ++i) { sum += sums[i]; n += counts[i]; }
    *total = (float)(mean ? sum / n : sum);
    *count = mean ? (float)n : 1.f;
  }
}

// ------------------------------------------------------------------------------------------------------------ backward
// Only the rows that take part are computed: the list of them, made on the device, is as long as `kept` says there (masked-word training
// ignores most rows), and the kernels below go by that length; their launches and the workspace are laid out for all M.
// ws: head | list: row of each kept one [M] | place of each row in the list or -1 [M] | g / max|g| of the kept [M] | kept rows of x, times
// that [M][K] 16 bit | kept rows of x as they are [M][K] | e [M][piece] 16 bit | dx sums [splits][kept][K] | db sums [waves' rows][V]
struct Head { float gmax; int kept; };
struct Plan { int piece, grid_dx, small; long o_list, o_place, o_factor, o_x, o_xk, o_e, o_dx, o_db, bytes; };
constexpr long E_BYTES = 256L << 20;                         // of e at a time: what the memory-side cache holds
constexpr int SMALL_M = 64;                                  // up to here one tile of 64 rows, beyond tiles of 256

Plan ce_plan(int M, int V, int K, bool bias) {
  Plan p;
  p.small = M <= SMALL_M;
  const long words = cdiv(V, 256) * 256L;
  long piece = E_BYTES / 2 / M / 256 * 256;
  if (piece < 1024) piece = 1024;
  if (piece > words) piece = words;
  const long n = (words + piece - 1) / piece;                // even pieces
  p.piece = (int)(((words + n - 1) / n + 255) / 256 * 256);
  const int rows = p.small ? 64 : 256, tiles = cdiv(K, 256) * cdiv(M, rows);
  p.grid_dx = max(256, tiles);                               // see dx_splits
  auto up = [](long n) { return (n + 255) / 256 * 256; };
  long o = 256;
  p.o_list = o; o += up(M * 4L);
  p.o_place = o; o += up(M * 4L);
  p.o_factor = o; o += up(M * 4L);
  p.o_x = o; o += up((long)M * K * 2);
  p.o_xk = o; o += up((long)M * K * 2);
  p.o_e = o; o += up((long)M * p.piece * 2);
  p.o_dx = o; o += (long)p.grid_dx * rows * 256 * 4;
  p.o_db = o; o += bias ? up((long)cdiv(M, 64) * V * 4) : 0;
  p.bytes = o;
  return p;
}
// dx is kept x K: few tiles.  A piece's words are shared out in `splits`, so that each of the chip's 256 compute units has a tile, of 256
// words at least, and eights of them go to the eight XCDs: the tiles of a split read the same words and e, through one L2
__device__ __forceinline__ int dx_splits(int grid, int tiles, int piece) {
  const int n = max(1, min(grid / max(1, tiles), piece / 256));
  return n < 8 ? n : n & ~7;
}

// A workgroup of 1024 counts the rows that take part, a stretch of rows to a thread: the thread's first place in their list, how many
// there are, and the largest |gradient| among them
struct Counted { int m0, m1, at, kept; float g; };
// f(row, whether it takes part, its gradient) of rows m0 .. m1 - 1, the loads of four at a time
template <class F> __device__ __forceinline__ void each_row(const simvg_vocab_ce_args& a, int m0, int m1, F f) {
  for (int m = m0; m < m1; m += 4) {
    long t[4];
    float d[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      t[i] = a.target[min(m + i, m1 - 1)];
      d[i] = a.dloss[min(m + i, m1 - 1)];
    }
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (m + i < m1) f(m + i, is_word(a, t[i]), d[i]);
  }
}
__device__ __forceinline__ Counted count_rows(const simvg_vocab_ce_args& a) {
  __shared__ float most[16];
  __shared__ int counts[16];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, per = cdiv(a.M, 1024);
  Counted c = {min(tid * per, a.M), min(tid * per + per, a.M), 0, 0, 0.f};
  int n = 0;
  each_row(a, c.m0, c.m1, [&](int, bool on, float d) {
    if (!on) return;
    c.g = fmaxf(c.g, fabsf(d));
    ++n;
  });
  c.g = wave_max(c.g);
  int upto = n;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const int before = __shfl_up(upto, o, 64);
    if (lane >= o) upto += before;
  }
  if (lane == 63) { most[wave] = c.g; counts[wave] = upto; }
  __syncthreads();
  c.at = upto - n;
  c.g = most[0];
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    c.g = fmaxf(c.g, most[i]);
    if (i < wave) c.at += counts[i];
    c.kept += counts[i];
  }
  return c;
}
__device__ __forceinline__ float row_factor(float d, float g) { return d == 0.f ? 0.f : d / g; }
// the list of the rows that take part, in their order: one workgroup
__global__ __launch_bounds__(1024) void ce_rows_kernel(simvg_vocab_ce_args a, Head* head, int* list, int* place, float* factor) {
  const Counted c = count_rows(a);
  int at = c.at;
  each_row(a, c.m0, c.m1, [&](int m, bool on, float d) {
    place[m] = on ? at : -1;
    if (on) {
      list[at] = m;
      factor[at++] = row_factor(d, c.g);
    }
  });
  if (threadIdx.x == 0) { head->gmax = c.g; head->kept = c.kept; }
}
// eight values of kept row r, row m of x: as they are, and times the row's factor
template <class E>
__device__ __forceinline__ void gather8(const simvg_vocab_ce_args& a, int r, int m, int c, float f, unsigned short* xs, unsigned short* xk) {
  u32x4_t v = *(const u32x4_t*)((const unsigned short*)a.x + (long)m * a.ldx + c);
  *(u32x4_t*)(xk + (long)r * a.K + c) = v;
  if (f != 1.f) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      float lo, hi;
      unpack2<E>(v[j], lo, hi);
      v[j] = E::pack(lo * f, hi * f);
    }
  }
  *(u32x4_t*)(xs + (long)r * a.K + c) = v;
}
template <class E>
__global__ __launch_bounds__(256) void ce_gather_kernel(simvg_vocab_ce_args a, const Head* head, const int* list, const float* factor,
                                                        unsigned short* xs, unsigned short* xk) {
  const int per = a.K / 8;
  for (long i = blockIdx.x * 256L + threadIdx.x; i < (long)head->kept * per; i += gridDim.x * 256L) {
    const int r = (int)(i / per);
    gather8<E>(a, r, list[r], (int)(i % per) * 8, factor[r], xs, xk);
  }
}
// Both in one launch: every workgroup counts for itself, the first one writes the list down.  (Up to a few thousand rows the count costs less
// than a launch: backward pass of 1280 rows 215 -> 211 us, of 40 rows, 8003 words 40.5 -> 37.9.)
constexpr int ROWS_AT_ONCE = 4096;
template <class E>
__global__ __launch_bounds__(1024) void ce_rows_gather_kernel(simvg_vocab_ce_args a, Head* head, int* list, int* place, float* factor,
                                                              unsigned short* xs, unsigned short* xk) {
  __shared__ int rows[ROWS_AT_ONCE];
  __shared__ float factors[ROWS_AT_ONCE];
  const Counted c = count_rows(a);
  const bool first = blockIdx.x == 0;
  int at = c.at;
  each_row(a, c.m0, c.m1, [&](int m, bool on, float d) {
    if (first) place[m] = on ? at : -1;
    if (on) {
      const float f = row_factor(d, c.g);
      rows[at] = m;
      factors[at] = f;
      if (first) { list[at] = m; factor[at] = f; }
      ++at;
    }
  });
  if (first && threadIdx.x == 0) { head->gmax = c.g; head->kept = c.kept; }
  __syncthreads();
  const int per = a.K / 8;
  for (int i = blockIdx.x * 1024 + threadIdx.x; i < c.kept * per; i += gridDim.x * 1024) {
    const int r = i / per;
    gather8<E>(a, r, rows[r], i % per * 8, factors[r], xs, xk);
  }
}

constexpr float E_POWER = 14.f;
template <class E> __device__ __forceinline__ float e_scale() { return E::kScaled ? 16384.f : 1.f; }

// the sum of v over a half wave's 16-lane row, in all its lanes' last
template <int CTRL> __device__ __forceinline__ float dpp_add(float v) {
  return v + __uint_as_float((unsigned)__builtin_amdgcn_update_dpp(0, (int)__float_as_uint(v), CTRL, 0xf, 0xf, true));
}
__device__ __forceinline__ float row16_sum(float v) {
  v = dpp_add<0xb1>(v);                                      // lane ^ 1 (quad_perm 1, 0, 3, 2)
  v = dpp_add<0x4e>(v);                                      // lane ^ 2 (quad_perm 2, 3, 0, 1)
  v = dpp_add<0x141>(v);                                     // the other four of eight (row_half_mirror)
  return dpp_add<0x140>(v);                                  // the other eight (row_mirror)
}

// A wave's block, WB rows (lanes) of WA values (registers) times `mul`, through LDS at `mine`, so that rows leave in whole lines (from the
// registers they would leave in halves of 16 bytes): store(row, first column, eight values).  Rows there are 16 bytes longer than the values.
constexpr int e_ld(int values) { return values * 2 + 16; }
constexpr int max_of(int x, int y) { return x > y ? x : y; }
template <class E, int WA, int WB, class Store>
__device__ __forceinline__ void block_rows(const f32x16 (&acc)[WA / 32][WB / 32], float mul, char* mine, int lane, Store store) {
  constexpr int LD = e_ld(WA), PER = WA / 8, ROWS = 64 / PER;  // lanes to a row, rows at a time
#pragma unroll
  for (int j = 0; j < WB / 32; ++j)
#pragma unroll
    for (int i = 0; i < WA / 32; ++i)
#pragma unroll
      for (int q = 0; q < 4; ++q)
        *(u32x2_t*)(mine + (j * 32 + (lane & 31)) * LD + (i * 32 + q * 8 + (lane >> 5) * 4) * 2) =
            (u32x2_t){E::pack(acc[i][j][4 * q] * mul, acc[i][j][4 * q + 1] * mul), E::pack(acc[i][j][4 * q + 2] * mul, acc[i][j][4 * q + 3] * mul)};
#pragma unroll 4
  for (int r = 0; r < WB; r += ROWS) {
    const int row = r + lane / PER, col = lane % PER * 8;
    store(row, col, *(const u32x4_t*)(mine + row * LD + col * 2));
  }
}

template <class P> constexpr int e_lds() { return max_of(P::LDS, P::WAVES * P::NB * 32 * e_ld(P::NA * 32)); }      // of (1), without the bias

// (1) words in registers, kept rows in lanes: e of words [v_begin, v_begin + piece), and db's sums over the wave's rows
template <class E, int RA, int RB, int WA, int WB, int STAGES, bool BIAS>
__global__ __launch_bounds__((RA / WA) * (RB / WB) * 64, 2) void ce_e_kernel(simvg_vocab_ce_args a, const Head* head, const int* list,
                                                                             const float* factor, const unsigned short* xk, unsigned short* e,
                                                                             int piece, int v_begin, float* db) {
  using P = Product<E, RA, false, RB, false, WA, WB, STAGES>;
  extern __shared__ __attribute__((aligned(16))) char smem[];
  constexpr int BIAS_AT = e_lds<P>();
  const int kept = head->kept, tv = piece / RA, tm = cdiv(kept, RB);
  if ((int)blockIdx.x >= tv * tm) return;
  int iv, im;
  tile_of(blockIdx.x, tv * tm, tv, tm, 4, iv, im);
  const int l0 = iv * RA, v0 = v_begin + l0, m0 = im * RB, lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  f32x16 acc[P::NA][P::NB];
  P::zero(acc);
  const int words = min(RA, a.V - v0);                       // may be <= 0 in the last piece: e is zeros there
  if (words > 0) {
    typename P::OA oa;
    typename P::OB ob;
    oa.init_stages((const unsigned short*)a.w + (long)v0 * a.ldw, a.ldw, words, a.K, smem, wave, lane);
    ob.init_stages(xk + (long)m0 * a.K, a.K, min(RB, kept - m0), a.K, smem + P::B_AT, wave, lane);
    oa.init_reads(smem, P::wave_a(wave) / 32, lane);
    ob.init_reads(smem + P::B_AT, P::wave_b(wave) / 32, lane);
    if (BIAS) bias_to_lds<RA>(a, v0, smem + BIAS_AT, wave, lane);
    P::run(acc, oa, ob, cdiv(a.K, BK));
    if (BIAS) add_bias(acc, smem + BIAS_AT + P::wave_a(wave) * 4, lane);
  }
  const int wl = P::wave_a(wave), wv = v0 + wl, wm = P::wave_b(wave);
  float less[P::NB], g[P::NB];
  int local[P::NB];
  bool any = false;
#pragma unroll
  for (int j = 0; j < P::NB; ++j) {
    const int r = m0 + wm + j * 32 + (lane & 31), m = list[min(r, kept - 1)];
    const bool on = r < kept;
    const long t = a.target[m];
    const float lse = a.lse[m], power = E::kScaled ? E_POWER : 0.f;
    less[j] = on ? power - lse * LOG2E : NEG_INF;
    const bool far = on && fabsf(lse) > FAR;
    if (__any(far)) {                                        // as in the forward pass
      stay_a_branch();
#pragma unroll
      for (int i = 0; i < P::NA; ++i)
#pragma unroll
        for (int q = 0; q < 16; ++q) acc[i][j][q] -= far ? lse : 0.f;
      if (far) less[j] = power;
    }
    g[j] = BIAS && on ? factor[r] : 0.f;
    local[j] = on && t >= wv && t < wv + WA ? (int)(t - wv) : -1;
    any = any || local[j] >= 0;
  }
#pragma unroll
  for (int i = 0; i < P::NA; ++i)
#pragma unroll
    for (int j = 0; j < P::NB; ++j)
#pragma unroll
      for (int r = 0; r < 16; ++r) acc[i][j][r] = __builtin_amdgcn_exp2f(fmaf(acc[i][j][r], LOG2E, less[j]));
  if (wv + WA > a.V) {
    stay_a_branch();
#pragma unroll
    for (int i = 0; i < P::NA; ++i)
#pragma unroll
      for (int j = 0; j < P::NB; ++j)
#pragma unroll
        for (int r = 0; r < 16; ++r)
          if (wv + i * 32 + acc_row(r, lane) >= a.V) acc[i][j][r] = 0.f;
  }
  if (__any(any)) {                                          // a target of the wave's rows is among the wave's words
    stay_a_branch();
#pragma unroll
    for (int i = 0; i < P::NA; ++i)
#pragma unroll
      for (int j = 0; j < P::NB; ++j)
#pragma unroll
        for (int r = 0; r < 16; ++r)
          if (local[j] == i * 32 + acc_row(r, lane)) acc[i][j][r] -= e_scale<E>();
  }
  if (BIAS && a.dbias) {
    const float down = 1.f / e_scale<E>();
#pragma unroll
    for (int i = 0; i < P::NA; ++i)
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        float s = 0.f;
#pragma unroll
        for (int j = 0; j < P::NB; ++j) s += acc[i][j][r] * g[j];
        s = row16_sum(s);
        s += __shfl_xor(s, 16, 64);
        const int v = wv + i * 32 + acc_row(r, lane);
        if ((lane & 31) == 0 && v < a.V && m0 + wm < kept) db[(long)((m0 + wm) / WB) * a.V + v] = s * down;
      }
  }
  block_rows<E, WA, WB>(acc, 1.f, smem + wave * WB * e_ld(WA), lane, [&](int row, int col, u32x4_t v) {
    const int m = m0 + wm + row;
    if (m < kept) *(u32x4_t*)(e + (long)m * piece + l0 + wl + col) = v;
  });
}
constexpr int dx_ld(int values) { return values * 4 + 16; }    // bytes of a row of a wave's sums in LDS
// (2) K in registers, rows in lanes: the piece's share of dx into this split's sums
template <class E, int RB, int WA, int WB, int STAGES>
__global__ __launch_bounds__((256 / WA) * (RB / WB) * 64, 2) void ce_dx_kernel(simvg_vocab_ce_args a, const Head* head,
                                                                               const unsigned short* e, int piece, int v_begin, float* sums) {
  using P = Product<E, 256, true, RB, false, WA, WB, STAGES>;
  extern __shared__ __attribute__((aligned(16))) char smem[];
  const int kept = head->kept, tk = cdiv(a.K, 256), tm = cdiv(kept, RB), tiles = tk * tm, splits = dx_splits(gridDim.x, tiles, piece);
  if ((int)blockIdx.x >= tiles * splits) return;
  int ik, im;
  int split, slot = blockIdx.x / 8;
  if (splits >= 8) {
    split = slot / tiles * 8 + blockIdx.x % 8;
    slot %= tiles;
    im = slot / tk;
    ik = slot % tk;
  } else {
    split = blockIdx.x / tiles;
    tile_of(blockIdx.x % tiles, tiles, tm, tk, tk, im, ik);
  }
  const int k0 = ik * 256, m0 = im * RB, lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  f32x16 acc[P::NA][P::NB];
  P::zero(acc);
  const int words = min(piece, a.V - v_begin), stages = cdiv(words, BK);
  const int s0 = (int)((long)stages * split / splits), s1 = (int)((long)stages * (split + 1) / splits);
  typename P::OA oa;
  typename P::OB ob;
  oa.init_stages((const unsigned short*)a.w + ((long)v_begin + s0 * BK) * a.ldw + k0, a.ldw, min(256, a.K - k0), words - s0 * BK, smem, wave, lane);
  ob.init_stages(e + (long)m0 * piece + s0 * BK, piece, min(RB, kept - m0), words - s0 * BK, smem + P::B_AT, wave, lane);
  oa.init_reads(smem, P::wave_a(wave) / 32, lane);
  ob.init_reads(smem + P::B_AT, P::wave_b(wave) / 32, lane);
  P::run(acc, oa, ob, s1 - s0);
  const int wk = k0 + P::wave_a(wave), wm = m0 + P::wave_b(wave);
  // through LDS, so that rows leave in whole lines, 32 of the wave at a time
  constexpr int LD = dx_ld(WA), PER = WA / 4, ROWS = 64 / PER;
  char* mine = smem + wave * 32 * LD;
#pragma unroll
  for (int j = 0; j < P::NB; ++j) {
#pragma unroll
    for (int i = 0; i < P::NA; ++i)
#pragma unroll
      for (int g = 0; g < 4; ++g)
        *(f32x4_t*)(mine + (lane & 31) * LD + (i * 32 + g * 8 + (lane >> 5) * 4) * 4) =
            (f32x4_t){acc[i][j][4 * g], acc[i][j][4 * g + 1], acc[i][j][4 * g + 2], acc[i][j][4 * g + 3]};
#pragma unroll 4
    for (int r = 0; r < 32; r += ROWS) {
      const int row = r + lane / PER, m = wm + j * 32 + row, k = wk + lane % PER * 4;
      f32x4_t v = *(const f32x4_t*)(mine + row * LD + lane % PER * 16);
      if (m >= kept || k >= a.K) continue;
      f32x4_t* at = (f32x4_t*)(sums + ((long)split * kept + m) * a.K + k);
      if (v_begin > 0) v += *at;
      *at = v;
    }
  }
}
// (3) K in registers, words in lanes: the piece's rows of dw
template <class E>
__global__ __launch_bounds__(512, 2) void ce_dw_kernel(simvg_vocab_ce_args a, const Head* head, const unsigned short* xs, const unsigned short* e,
                                                       int piece, int v_begin) {
  constexpr int RB = 256;
  using P = Product<E, 256, true, RB, true, 128, 64, 2>;
  extern __shared__ __attribute__((aligned(16))) char smem[];
  const int kept = head->kept, words = min(piece, a.V - v_begin), tk = cdiv(a.K, 256), tv = cdiv(words, RB);
  int ik, iv;
  tile_of(blockIdx.x, tk * tv, tv, tk, tk, iv, ik);
  const int k0 = ik * 256, l0 = iv * RB, lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  f32x16 acc[P::NA][P::NB];
  P::zero(acc);
  typename P::OA oa;
  typename P::OB ob;
  oa.init_stages(xs + k0, a.K, min(256, a.K - k0), kept, smem, wave, lane);
  ob.init_stages(e + l0, piece, min(RB, piece - l0), kept, smem + P::B_AT, wave, lane);
  oa.init_reads(smem, P::wave_a(wave) / 32, lane);
  ob.init_reads(smem + P::B_AT, P::wave_b(wave) / 32, lane);
  P::run(acc, oa, ob, cdiv(kept, BK));
  const int wk = k0 + P::wave_a(wave), wl = l0 + P::wave_b(wave);
  const float mul = head->gmax / e_scale<E>();
  block_rows<E, 128, 64>(acc, mul, smem + wave * 64 * e_ld(128), lane, [&](int row, int col, u32x4_t v) {
    if (wl + row < words && wk + col < a.K) *(u32x4_t*)((unsigned short*)a.dw + (long)(v_begin + wl + row) * a.lddw + wk + col) = v;
  });
}
// dx: the splits' sums, and zeros for the rows that take no part
template <class E>
__global__ __launch_bounds__(256) void ce_dx_join_kernel(simvg_vocab_ce_args a, const Head* head, const int* place, const float* sums, int grid_dx,
                                                         int rows, int piece) {
  const int per = a.K / 4, kept = head->kept, splits = dx_splits(grid_dx, cdiv(a.K, 256) * cdiv(kept, rows), piece);
  for (long i = blockIdx.x * 256L + threadIdx.x; i < (long)a.M * per; i += gridDim.x * 256L) {
    const int m = (int)(i / per), c = (int)(i % per) * 4, r = place[m];
    f32x4_t v = {0.f, 0.f, 0.f, 0.f};
    if (r >= 0) {
#pragma unroll 8
      for (int s = 0; s < splits; ++s) v += *(const f32x4_t*)(sums + ((long)s * kept + r) * a.K + c);
      v *= a.dloss[m] / e_scale<E>();
    }
    *(u32x2_t*)((unsigned short*)a.dx + (long)m * a.lddx + c) = (u32x2_t){E::pack(v[0], v[1]), E::pack(v[2], v[3])};
  }
}
__global__ __launch_bounds__(256) void ce_db_join_kernel(simvg_vocab_ce_args a, const Head* head, const float* db) {
  const int v = blockIdx.x * 256 + threadIdx.x, groups = cdiv(head->kept, 64);
  if (v >= a.V) return;
  float s = 0.f;
#pragma unroll 8
  for (int g = 0; g < groups; ++g) s += db[(long)g * a.V + v];
  a.dbias[v] = s * head->gmax;
}

// ---------------------------------------------------------------------------------------------------------------- host
bool rows16(const void* p, long ld) { return p && (uintptr_t)p % 16 == 0 && ld % 8 == 0; }

int ce_check(const simvg_vocab_ce_args* a, bool bwd) {
  SIMVG_CHECK_ARG(a, "vocab_ce: null argument block");
  SIMVG_CHECK_ARG(a->dtype == SEQ_F16 || a->dtype == SEQ_BF16, "vocab_ce: dtype must be fp16 or bf16");
  SIMVG_CHECK_ARG(a->M >= 0 && a->V >= 1 && a->K >= 8, "vocab_ce: needs M >= 0, V >= 1, K >= 8");
  SIMVG_CHECK_ARG(a->K % 8 == 0, "vocab_ce: K must be a multiple of 8");
  SIMVG_CHECK_ARG(a->M <= 1 << 22 && a->V <= 1 << 24 && a->K <= 1 << 16, "vocab_ce: M, V or K too large");
  SIMVG_CHECK_ARG((long)cdiv(a->V, 256) * cdiv(a->M, 256) < 1L << 23, "vocab_ce: too many tiles for one launch");
  SIMVG_CHECK_ARG(a->ldx >= a->K && a->ldw >= a->K && a->ldx < 1 << 21 && a->ldw < 1 << 21, "vocab_ce: row strides must be at least K and below 2^21");
  SIMVG_CHECK_ARG(rows16(a->w, a->ldw), "vocab_ce: rows of w must start at multiples of 16 bytes");
  SIMVG_CHECK_ARG(a->M == 0 || rows16(a->x, a->ldx), "vocab_ce: rows of x must start at multiples of 16 bytes");
  SIMVG_CHECK_ARG(a->M == 0 || (a->target && a->lse), "vocab_ce: null pointer");
  SIMVG_CHECK_ARG(bwd || a->M == 0 || a->loss, "vocab_ce: null pointer");
  if (bwd) {
    SIMVG_CHECK_ARG((a->M == 0 || (a->dloss && a->dx)) && a->dw, "vocab_ce: null pointer");
    SIMVG_CHECK_ARG((a->M == 0 || rows16(a->dx, a->lddx)) && rows16(a->dw, a->lddw) && a->lddx >= a->K && a->lddw >= a->K,
                    "vocab_ce: rows of the gradients must start at multiples of 16 bytes and hold K values");
    SIMVG_CHECK_ARG(!a->dbias || a->bias, "vocab_ce: a gradient for a bias that is not there");
  }
  return SIMVG_OK;
}

#define CE_LAUNCH(THREADS, LDS, KERNEL, GRID, ...)                                   \
  do {                                                                               \
    static std::atomic<unsigned long> done{0};                                       \
    allow_lds((const void*)(KERNEL), LDS, done);                                     \
    hipLaunchKernelGGL((KERNEL), dim3(GRID), dim3(THREADS), LDS, s, __VA_ARGS__);    \
  } while (0)

int ce_fwd_groups(int V, int M) { return cdiv(V, M <= SMALL_M ? 128 : 256); }

template <class E>
int ce_fwd(const simvg_vocab_ce_args& a, hipStream_t s) {
  const int groups = ce_fwd_groups(a.V, a.M);
  float* zt = (float*)a.ws;
  float2* part = (float2*)((char*)a.ws + (a.M * 4L + 255) / 256 * 256);
  if (a.M <= SMALL_M) {                                      // a row of tiles, bound by reading w: twice as many, half as high, two to a compute unit
    using P = Product<E, 128, false, 64, false, 32, 64, 3>;
    CE_LAUNCH(P::THREADS, P::LDS + 128 * 4, (ce_fwd_kernel<E, 128, 64, 32, 64, 3>), groups, a, part, zt);
  } else {
    using P = Product<E, 256, false, 256, false, 128, 64, 2>;
    CE_LAUNCH(P::THREADS, P::LDS + 256 * 4, (ce_fwd_kernel<E, 256, 256, 128, 64, 2>), groups * cdiv(a.M, 256), a, part, zt);
  }
  SIMVG_LAUNCH_CHECK();
  hipLaunchKernelGGL(ce_join_kernel, dim3(cdiv(a.M, 8)), dim3(1024), 0, s, a, part, zt, groups);
  SIMVG_LAUNCH_CHECK();
  return SIMVG_OK;
}

__global__ void ce_zero_kernel(unsigned short* dw, long lddw, int V, int K, float* db) {
  const long n = (long)V * K;
  for (long i = blockIdx.x * 256L + threadIdx.x; i < n; i += (long)gridDim.x * 256) dw[i / K * lddw + i % K] = 0;
  if (db)
    for (long i = blockIdx.x * 256L + threadIdx.x; i < V; i += (long)gridDim.x * 256) db[i] = 0.f;
}

template <class E>
int ce_bwd(const simvg_vocab_ce_args& a, hipStream_t s) {
  const Plan p = ce_plan(a.M, a.V, a.K, a.dbias != nullptr);
  char* ws = (char*)a.ws;
  Head* head = (Head*)ws;
  int *list = (int*)(ws + p.o_list), *place = (int*)(ws + p.o_place);
  float *factor = (float*)(ws + p.o_factor), *sums = (float*)(ws + p.o_dx), *db = (float*)(ws + p.o_db);
  unsigned short *xs = (unsigned short*)(ws + p.o_x), *xk = (unsigned short*)(ws + p.o_xk), *e = (unsigned short*)(ws + p.o_e);
  if (a.M <= ROWS_AT_ONCE) {
    hipLaunchKernelGGL(ce_rows_gather_kernel<E>, dim3(min(256, cdiv(a.M * (a.K / 8), 1024))), dim3(1024), 0, s, a, head, list, place, factor, xs, xk);
  } else {
    hipLaunchKernelGGL(ce_rows_kernel, dim3(1), dim3(1024), 0, s, a, head, list, place, factor);
    hipLaunchKernelGGL(ce_gather_kernel<E>, dim3(min(2048, cdiv(a.M, 2))), dim3(256), 0, s, a, head, list, factor, xs, xk);
  }
  SIMVG_LAUNCH_CHECK();
  const int tk = cdiv(a.K, 256);
  const auto piece = [&](auto bias, int v) {
    constexpr bool B = decltype(bias)::value;
    const int words = min(p.piece, a.V - v);
    if (p.small) {
      using P1 = Product<E, 128, false, 64, false, 32, 64, 3>;
      using P2 = Product<E, 256, true, 64, false, 64, 64, 2>;
      static_assert(P2::WAVES * 32 * dx_ld(64) <= P2::LDS, "the waves' blocks of results");
      CE_LAUNCH(P1::THREADS, e_lds<P1>() + 128 * 4, (ce_e_kernel<E, 128, 64, 32, 64, 3, B>), p.piece / 128, a, head, list, factor, xk, e, p.piece, v, db);
      CE_LAUNCH(P2::THREADS, P2::LDS, (ce_dx_kernel<E, 64, 64, 64, 2>), p.grid_dx, a, head, e, p.piece, v, sums);
    } else {
      using P1 = Product<E, 256, false, 256, false, 128, 64, 2>;
      using P2 = Product<E, 256, true, 256, false, 128, 64, 2>;
      CE_LAUNCH(P1::THREADS, e_lds<P1>() + 256 * 4, (ce_e_kernel<E, 256, 256, 128, 64, 2, B>), cdiv(a.M, 256) * (p.piece / 256), a, head, list, factor, xk, e,
                p.piece, v, db);
      CE_LAUNCH(P2::THREADS, max_of(P2::LDS, P2::WAVES * 32 * dx_ld(128)), (ce_dx_kernel<E, 256, 128, 64, 2>), p.grid_dx, a, head, e, p.piece, v, sums);
    }
    using P3 = Product<E, 256, true, 256, true, 128, 64, 2>;
    CE_LAUNCH(P3::THREADS, max_of(P3::LDS, P3::WAVES * 64 * e_ld(128)), ce_dw_kernel<E>, tk * cdiv(words, 256), a, head, xs, e, p.piece, v);
  };
  for (int v = 0; v < a.V; v += p.piece) {
    if (a.bias) piece(std::true_type{}, v); else piece(std::false_type{}, v);
    SIMVG_LAUNCH_CHECK();
  }
  hipLaunchKernelGGL(ce_dx_join_kernel<E>, dim3(min(2048, cdiv(a.M, 2))), dim3(256), 0, s, a, head, place, sums, p.grid_dx, p.small ? 64 : 256,
                     p.piece);
  if (a.dbias) hipLaunchKernelGGL(ce_db_join_kernel, dim3(cdiv(a.V, 256)), dim3(256), 0, s, a, head, db);
  SIMVG_LAUNCH_CHECK();
  return SIMVG_OK;
}
}  // namespace

extern "C" long simvg_vocab_ce_ws_bytes(int M, int V, int K, int with_bias, int backward) {
  if (M <= 0 || V <= 0 || K <= 0) return 0;
  if (backward) return ce_plan(M, V, K, with_bias != 0).bytes;
  return (M * 4L + 255) / 256 * 256 + (long)ce_fwd_groups(V, M) * M * 8;
}
extern "C" int simvg_vocab_ce_fwd(const simvg_vocab_ce_args* args, hipStream_t stream) {
  const int rc = ce_check(args, false);
  if (rc || args->M == 0) return rc;
  const long need = simvg_vocab_ce_ws_bytes(args->M, args->V, args->K, args->bias != nullptr, 0);
  SIMVG_CHECK_ARG(args->ws && (uintptr_t)args->ws % 256 == 0 && args->ws_bytes >= need, "vocab_ce: the workspace is too small or misaligned");
  return args->dtype == SEQ_F16 ? ce_fwd<F16>(*args, stream) : ce_fwd<BF16>(*args, stream);
}
extern "C" int simvg_vocab_ce_reduce(const float* loss, const long* target, long ignore_index, int M, int mean, float* total, float* count,
                                     hipStream_t stream) {
  SIMVG_CHECK_ARG(M >= 0 && M <= 1 << 22, "vocab_ce_reduce: M must be between 0 and 2^22");
  SIMVG_CHECK_ARG((M == 0 || (loss && target)) && total && count, "vocab_ce_reduce: null pointer");
  hipLaunchKernelGGL(ce_reduce_kernel, dim3(1), dim3(1024), 0, stream, loss, target, ignore_index, M, mean, total, count);
  SIMVG_LAUNCH_CHECK();
  return SIMVG_OK;
}
extern "C" int simvg_vocab_ce_bwd(const simvg_vocab_ce_args* args, hipStream_t stream) {
  const int rc = ce_check(args, true);
  if (rc) return rc;
  if (args->M == 0) {                                        // sums of nothing
    hipLaunchKernelGGL(ce_zero_kernel, dim3(1024), dim3(256), 0, stream, (unsigned short*)args->dw, args->lddw, args->V, args->K, args->dbias);
    SIMVG_LAUNCH_CHECK();
    return SIMVG_OK;
  }
  const long need = simvg_vocab_ce_ws_bytes(args->M, args->V, args->K, args->dbias != nullptr, 1);
  SIMVG_CHECK_ARG(args->ws && (uintptr_t)args->ws % 256 == 0 && args->ws_bytes >= need, "vocab_ce: the workspace is too small or misaligned");
  return args->dtype == SEQ_F16 ? ce_bwd<F16>(*args, stream) : ce_bwd<BF16>(*args, stream);
}
