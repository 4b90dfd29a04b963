// simvg-build-flags: -Wno-inline-asm
// Softmax cross entropy over a large vocabulary without its logits, forward and backward.
//
//   z = x w^T + b  [M, V],  lse_i = log sum_v exp(z_iv),  loss_i = lse_i - z_i,target(i)          (0 where the target is ignored)
//   backward, for the gradients g_i of the rows' losses:  e_iv = exp(z_iv - lse_i) - [v = target(i)]
//     dx_i = g_i sum_v e_iv w_v,   dw_v = sum_i e_iv g_i x_i,   db_v = sum_i g_i e_iv
//
// Bound by the matrix pipes (2 M V K forward, 6 M V K backward: the logits are computed again, they are never kept), for few rows by
// reading w once.  Forward: a matrix product whose epilogue keeps, for each row and each 32..128 words, the maximum and the sum of the
// exponentials; a second kernel joins them.  Backward, in pieces of the vocabulary: (1) the logits of the piece again, as e rounded to
// 16 bits into a workspace that stays near the caches; (2) its share of dx, added to sums in 32 bits; (3) its rows of dw.  (2) and (3)
// are products over the vocabulary and over the rows: their operands lie "the other way round" in memory and are read from LDS with
// the transposing ds_read_b64_tr_b16, so that nothing is ever laid out twice.
//
// Rounding to 16 bits, by choice: e (one rounding, relative 2^-9 bf16 / 2^-12 fp16; in fp16 times 2^14, so that a probability of 2^-28
// keeps all its bits) and g x / max|g| where the rows' gradients differ (where they are equal or 0 the factor is 1 or 0: exact).
// Everything that is summed is summed in 32 bits; db is summed before the rounding.
#include <atomic>

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

constexpr float LOG2E = 1.44269504088896340736f, LN2 = 0.69314718055994530942f;
constexpr float NEG_INF = -__builtin_huge_valf();
constexpr int BK = 64;                                       // contracted values of a stage

__device__ __forceinline__ f32x16 zero16() { return (f32x16){0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f}; }
__device__ __forceinline__ int acc_row(int r, int lane) { return (r >> 2) * 8 + (lane >> 5) * 4 + (r & 3); }

// ------------------------------------------------------------------------------------------------- the matrix product
// One operand of a workgroup's tile: R rows (or columns) of the result by BK contracted values per stage.
//   T = false: memory [R][contracted], a stage is R rows of 128 bytes;  T = true: memory [contracted][R], BK rows of 2 R bytes.
// In LDS, slots of 16 bytes are permuted within a row so that the fragment reads touch every bank once: 16 rows of one slot
// (ds_read_b128) or 4 rows of 4 neighbouring slots (ds_read_b64_tr_b16) are one cycle's.
template <int R, bool T> struct Operand {
  static constexpr int BYTES = R * BK * 2;
  static constexpr int ROW = T ? R * 2 : BK * 2;
  static __device__ __forceinline__ int at(int row, int slot) {
    int x;
    if (T && R >= 128) x = (row & 3) << 2;
    else x = (row >> 1 & 1) << 2 | (row >> 2 & 3);            // rows of 128 bytes: a pair of rows shares the banks' 256
    return row * ROW + ((slot ^ x) << 4);
  }
  // the 32 x 16 fragment `f` (rows 32 f ..) of contracted values 16 ks ..
  static __device__ __forceinline__ lpx8_t frag(const char* lds, int f, int ks, int lane) {
    if constexpr (!T) {
      return *(const lpx8_t*)(lds + at(f * 32 + (lane & 31), ks * 2 + (lane >> 5)));
    } else {
      const int i = lane & 15, col = f * 32 + (lane >> 4 & 1) * 16 + 4 * (i & 3);
      const int row = ks * 16 + 8 * (lane >> 5) + (i >> 2);
      const lpx4_t lo = lds_read_tr16(lds + at(row, col >> 3) + (col & 7) * 2);
      const lpx4_t hi = lds_read_tr16(lds + at(row + 4, col >> 3) + (col & 7) * 2);
      return (lpx8_t){lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
    }
  }
};
// The source of an operand: base of the tile's first row / column, what is there of rows (R direction) and of contracted values
struct Source { const unsigned short* base; long ld; int rows, depth; };

template <int R, bool T, int WAVES> struct Stager {
  using Op = Operand<R, T>;
  static constexpr int PIECES = Op::BYTES / 1024 / WAVES;    // 1 KiB each
  static_assert(PIECES >= 1, "a wave stages at least one piece");
  unsigned off[PIECES];
  int inner[PIECES];                                         // T = false: first contracted value of the lane's 16 bytes
  __device__ __forceinline__ void init(const Source& s, int wave, int lane) {
#pragma unroll
    for (int i = 0; i < PIECES; ++i) {
      const int byte = (wave * PIECES + i) * 1024 + lane * 16, row = byte / Op::ROW, phys = byte % Op::ROW / 16;
      const int slot = (Op::at(row, phys) - row * Op::ROW) >> 4;               // the permutation is its own inverse
      inner[i] = slot * 8;
      if (T) off[i] = slot * 8 < s.rows ? (unsigned)(row * s.ld * 2 + slot * 16) : DMA_NOTHING;
      else off[i] = row < s.rows ? (unsigned)(row * s.ld * 2 + slot * 16) : DMA_NOTHING;
    }
  }
  // stage `kt` of the contraction into LDS at `lds`
  __device__ __forceinline__ void issue(const Source& s, int kt, unsigned lds, int wave) {
    const int left = s.depth - kt * BK;                      // contracted values from this stage on
    if (T) {
      // rows past the depth lie past the buffer; columns past the tile's were ruled out in init
      const unsigned bytes = left > 0 ? (unsigned)((min(left, BK) - 1) * s.ld * 2 + ((s.rows + 7) & ~7) * 2) : 0u;
      const u32x4_t b = dma_buffer(s.base + (long)kt * BK * s.ld, bytes);
#pragma unroll
      for (int i = 0; i < PIECES; ++i) dma16(b, lds + (wave * PIECES + i) * 1024, off[i]);
    } else {
      const u32x4_t b = dma_buffer(s.base + kt * BK, left > 0 ? (unsigned)((s.rows - 1) * s.ld * 2 + ((min(left, BK) + 7) & ~7) * 2) : 0u);
      if (left >= BK) {
#pragma unroll
        for (int i = 0; i < PIECES; ++i) dma16(b, lds + (wave * PIECES + i) * 1024, off[i]);
      } else {                                               // the row's tail: what follows it is another row
#pragma unroll
        for (int i = 0; i < PIECES; ++i) dma16(b, lds + (wave * PIECES + i) * 1024, inner[i] < left ? off[i] : DMA_NOTHING);
      }
    }
  }
};

// acc[i][j] += A rows (wa + 32 i ..) x B rows (wb + 32 j ..) over stages [k0, k1): registers run over A's rows, lanes over B's
template <class E, int RA, bool TA, int RB, bool TB, int WA, int WB>
struct Product {
  static constexpr int WAVES = (RA / WA) * (RB / WB), THREADS = WAVES * 64, NA = WA / 32, NB = WB / 32;
  using OA = Operand<RA, TA>;
  using OB = Operand<RB, TB>;
  static constexpr int STAGE = OA::BYTES + OB::BYTES, LDS = 2 * STAGE;
  static __device__ __forceinline__ void run(f32x16 (&acc)[NA][NB], const Source& sa, const Source& sb, int k0, int k1, char* smem) {
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int fa = wave / (RB / WB) * NA, fb = wave % (RB / WB) * NB;
    Stager<RA, TA, WAVES> ga;
    Stager<RB, TB, WAVES> gb;
    ga.init(sa, wave, lane);
    gb.init(sb, wave, lane);
    const unsigned lds = lds_addr(smem);
    if (k0 < k1) {
      ga.issue(sa, k0, lds, wave);
      gb.issue(sb, k0, lds + OA::BYTES, wave);
    }
    for (int kt = k0; kt < k1; ++kt) {
      const int buf = (kt - k0) & 1;
      dma_wait<0>();                                         // this wave's pieces of the stage
      wave_barrier_only();                                   // everybody's; and everybody is done with the other buffer
      if (kt + 1 < k1) {
        ga.issue(sa, kt + 1, lds + (buf ^ 1) * STAGE, wave);
        gb.issue(sb, kt + 1, lds + (buf ^ 1) * STAGE + OA::BYTES, wave);
      }
      const char *la = smem + buf * STAGE, *lb = la + OA::BYTES;
#pragma unroll
      for (int ks = 0; ks < BK / 16; ++ks) {
        lpx8_t a[NA], b[NB];
#pragma unroll
        for (int j = 0; j < NB; ++j) b[j] = OB::frag(lb, fb + j, ks, lane);
#pragma unroll
        for (int i = 0; i < NA; ++i) a[i] = OA::frag(la, fa + i, ks, lane);
#pragma unroll
        for (int i = 0; i < NA; ++i)
#pragma unroll
          for (int j = 0; j < NB; ++j) acc[i][j] = E::mfma(a[i], b[j], acc[i][j]);
      }
    }
    __syncthreads();                                         // the epilogues use the LDS
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

// ------------------------------------------------------------------------------------------------------------- forward
// words in registers, rows in lanes: [word group of WA][M] (maximum, sum of exp2) and the targets' logits
template <class E, int RB, int WA, int WB>
__global__ __launch_bounds__((256 / WA) * (RB / WB) * 64) void ce_fwd_kernel(simvg_vocab_ce_args a, float2* part, float* zt) {
  using P = Product<E, 256, false, RB, false, WA, WB>;
  extern __shared__ __attribute__((aligned(16))) char smem[];
  const int tv = cdiv(a.V, 256), tm = cdiv(a.M, RB);
  int iv, im;
  tile_of(blockIdx.x, tv * tm, tv, tm, 4, iv, im);
  const int v0 = iv * 256, m0 = im * RB;
  f32x16 acc[P::NA][P::NB];
#pragma unroll
  for (int i = 0; i < P::NA; ++i)
#pragma unroll
    for (int j = 0; j < P::NB; ++j) acc[i][j] = zero16();
  const Source sa = {(const unsigned short*)a.w + (long)v0 * a.ldw, a.ldw, min(256, a.V - v0), a.K};
  const Source sb = {(const unsigned short*)a.x + (long)m0 * a.ldx, a.ldx, min(RB, a.M - m0), a.K};
  P::run(acc, sa, sb, 0, cdiv(a.K, BK), smem);
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int wv = v0 + wave / (RB / WB) * WA, wm = m0 + wave % (RB / WB) * WB;
#pragma unroll
  for (int i = 0; i < P::NA; ++i)
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      const int v = wv + i * 32 + acc_row(r, lane);
      const float b = a.bias && v < a.V ? a.bias[v] : 0.f;
#pragma unroll
      for (int j = 0; j < P::NB; ++j) acc[i][j][r] = v < a.V ? acc[i][j][r] + b : NEG_INF;
    }
#pragma unroll
  for (int j = 0; j < P::NB; ++j) {
    const int m = wm + j * 32 + (lane & 31);
    const long t = m < a.M ? a.target[m] : -1;
    const int local = t >= wv && t < wv + WA && t < a.V ? (int)(t - wv) : -1;
    if (__any(local >= 0)) {
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
    const float ref = top == NEG_INF ? 0.f : top * LOG2E;
#pragma unroll
    for (int i = 0; i < P::NA; ++i)
#pragma unroll
      for (int r = 0; r < 16; ++r) sum += __builtin_amdgcn_exp2f(fmaf(acc[i][j][r], LOG2E, -ref));
    sum += __shfl_xor(sum, 32, 64);
    if (lane < 32 && m < a.M && wv < a.V) part[(long)(wv / WA) * a.M + m] = make_float2(top, sum);
  }
}
// 32 rows and 32 strands of word groups to a workgroup
__global__ __launch_bounds__(1024) void ce_join_kernel(simvg_vocab_ce_args a, const float2* part, const float* zt, int groups) {
  __shared__ float tops[32][33], sums[32][33];
  const int c = threadIdx.x & 31, s = threadIdx.x >> 5, m = blockIdx.x * 32 + c;
  float top = NEG_INF, sum = 0.f;
  if (m < a.M)
    for (int g = s; g < groups; g += 32) {
      const float2 p = part[(long)g * a.M + m];
      const float to = fmaxf(top, p.x), ref = to == NEG_INF ? 0.f : to;
      sum = sum * __builtin_amdgcn_exp2f((top - ref) * LOG2E) + p.y * __builtin_amdgcn_exp2f((p.x - ref) * LOG2E);
      top = to;
    }
  tops[s][c] = top;
  sums[s][c] = sum;
  __syncthreads();
  if (s == 0 && m < a.M) {
    float t = NEG_INF;
    for (int i = 0; i < 32; ++i) t = fmaxf(t, tops[i][c]);
    const float ref = t == NEG_INF ? 0.f : t;
    float total = 0.f;
    for (int i = 0; i < 32; ++i) total += sums[i][c] * __builtin_amdgcn_exp2f((tops[i][c] - ref) * LOG2E);
    const float lse = ref + __builtin_logf(total);
    const long target = a.target[m];
    a.lse[m] = lse;
    // a target that is neither a word nor ignored is a mistake of the caller's: its loss says so
    a.loss[m] = target == a.ignore_index ? 0.f : is_word(a, target) ? lse - zt[m] : __builtin_nanf("");
  }
}

// ------------------------------------------------------------------------------------------------------------ backward
// ws: max|g| | row factors g / max|g| [M] | g x / max|g| [M][K] 16 bit | e [M][piece] 16 bit | dx sums [splits][M][K] | db sums [rows / RA][V]
struct Plan { int piece, splits, small; long o_factor, o_x, o_e, o_dx, o_db, bytes; };
constexpr long E_BYTES = 256L << 20;                         // of e at a time: what the memory-side cache holds

Plan ce_plan(int M, int V, int K, bool bias) {
  Plan p;
  p.small = M <= 64;
  const long words = cdiv(V, 256) * 256L;
  long piece = E_BYTES / 2 / M / 256 * 256;
  if (piece < 1024) piece = 1024;
  if (piece > words) piece = words;
  const long n = (words + piece - 1) / piece;                // even pieces
  p.piece = (int)(((words + n - 1) / n + 255) / 256 * 256);
  // dx is M x K: few tiles.  The piece's words are shared out so that the chip's 256 compute units have a tile each
  const int tiles = cdiv(K, 256) * cdiv(M, p.small ? 64 : 256), most = p.piece / 256;
  p.splits = 256 / tiles < 1 ? 1 : 256 / tiles > most ? most : 256 / tiles;
  auto up = [](long n) { return (n + 255) / 256 * 256; };
  long o = 256;
  p.o_factor = o; o += up(M * 4L);
  p.o_x = o; o += up((long)M * K * 2);
  p.o_e = o; o += up((long)M * p.piece * 2);
  p.o_dx = o; o += up((long)p.splits * M * K * 4);
  p.o_db = o; o += bias ? up((long)cdiv(M, 64) * V * 4) : 0;
  p.bytes = o;
  return p;
}

__global__ __launch_bounds__(1024) void ce_gmax_kernel(simvg_vocab_ce_args a, float* gmax, float* factor) {
  __shared__ float red[16];
  float g = 0.f;
  for (int m = threadIdx.x; m < a.M; m += 1024)
    if (is_word(a, a.target[m])) g = fmaxf(g, fabsf(a.dloss[m]));
  g = wave_max(g);
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = g;
  __syncthreads();
  g = red[0];
  for (int i = 1; i < 16; ++i) g = fmaxf(g, red[i]);
  if (threadIdx.x == 0) gmax[0] = g;
  for (int m = threadIdx.x; m < a.M; m += 1024) factor[m] = !is_word(a, a.target[m]) ? 0.f : a.dloss[m] == 0.f ? 0.f : a.dloss[m] / g;
}
template <class E>
__global__ __launch_bounds__(256) void ce_scale_kernel(simvg_vocab_ce_args a, const float* factor, unsigned short* xs) {
  const int per = a.K / 8;
  for (long i = blockIdx.x * 256L + threadIdx.x; i < (long)a.M * per; i += (long)gridDim.x * 256) {
    const int m = (int)(i / per), c = (int)(i % per) * 8;
    u32x4_t v = *(const u32x4_t*)((const unsigned short*)a.x + (long)m * a.ldx + c);
    const float f = factor[m];
    if (!is_word(a, a.target[m])) v = (u32x4_t){0u, 0u, 0u, 0u};               // whatever an ignored row holds
    else if (f != 1.f) {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        float lo, hi;
        unpack2<E>(v[j], lo, hi);
        v[j] = E::pack(lo * f, hi * f);
      }
    }
    *(u32x4_t*)(xs + (long)m * a.K + c) = v;
  }
}

constexpr float E_POWER = 14.f;
template <class E> __device__ __forceinline__ float e_scale() { return E::kScaled ? 16384.f : 1.f; }

// (1) rows in registers, words in lanes: e of words [v_begin, v_begin + piece) and db's sums over the workgroup's rows
template <class E, int RA, int WA, int WB>
__global__ __launch_bounds__((RA / WA) * (256 / WB) * 64) void ce_e_kernel(simvg_vocab_ce_args a, const float* factor, unsigned short* e,
                                                                           int piece, int v_begin, float* db) {
  using P = Product<E, RA, false, 256, false, WA, WB>;
  extern __shared__ __attribute__((aligned(16))) char smem[];
  const int tv = piece / 256, tm = cdiv(a.M, RA);
  int iv, im;
  tile_of(blockIdx.x, tv * tm, tv, tm, 4, iv, im);
  const int l0 = iv * 256, v0 = v_begin + l0, m0 = im * RA;
  f32x16 acc[P::NA][P::NB];
#pragma unroll
  for (int i = 0; i < P::NA; ++i)
#pragma unroll
    for (int j = 0; j < P::NB; ++j) acc[i][j] = zero16();
  const int words = min(256, a.V - v0);                      // may be <= 0 in the last piece: e is zeros there
  const Source sa = {(const unsigned short*)a.x + (long)m0 * a.ldx, a.ldx, min(RA, a.M - m0), a.K};
  const Source sb = {(const unsigned short*)a.w + (words > 0 ? (long)v0 * a.ldw : 0L), a.ldw, max(words, 0), a.K};
  if (words > 0) P::run(acc, sa, sb, 0, cdiv(a.K, BK), smem);
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int wl = wave % (256 / WB) * WB, wm = m0 + wave / (256 / WB) * WA;
  const float up = e_scale<E>();
  float bias[P::NB], sum[P::NB];
#pragma unroll
  for (int j = 0; j < P::NB; ++j) {
    const int v = v0 + wl + j * 32 + (lane & 31);
    bias[j] = a.bias && v < a.V ? a.bias[v] : 0.f;
    sum[j] = 0.f;
  }
#pragma unroll
  for (int i = 0; i < P::NA; ++i)
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      const int m = wm + i * 32 + acc_row(r, lane), mc = min(m, a.M - 1);
      const long t = a.target[mc];
      const bool on = m < a.M && is_word(a, t);
      const float lse = a.lse[mc] * LOG2E, g = a.dbias ? factor[mc] : 0.f;
#pragma unroll
      for (int j = 0; j < P::NB; ++j) {
        const int v = v0 + wl + j * 32 + (lane & 31);
        float p = __builtin_amdgcn_exp2f(fmaf(acc[i][j][r] + bias[j], LOG2E, -lse));
        if (t == v) p -= 1.f;
        p = on && v < a.V ? p : 0.f;
        sum[j] += on ? p * g : 0.f;
        if (m < a.M) e[(long)m * piece + l0 + wl + j * 32 + (lane & 31)] = (unsigned short)E::pack(p * up, 0.f);
      }
    }
  if (a.dbias) {
#pragma unroll
    for (int j = 0; j < P::NB; ++j) {
      const int v = v0 + wl + j * 32 + (lane & 31);
      sum[j] += __shfl_xor(sum[j], 32, 64);
      if (lane < 32 && v < a.V && wm < a.M) db[(long)(wm / WA) * a.V + v] = sum[j];
    }
  }
}
// (2) K in registers, rows in lanes: the piece's share of dx into this split's sums
template <class E, int RB, int WA, int WB>
__global__ __launch_bounds__((256 / WA) * (RB / WB) * 64) void ce_dx_kernel(simvg_vocab_ce_args a, const unsigned short* e, int piece,
                                                                            int v_begin, int splits, float* sums) {
  using P = Product<E, 256, true, RB, false, WA, WB>;
  extern __shared__ __attribute__((aligned(16))) char smem[];
  const int tk = cdiv(a.K, 256), tm = cdiv(a.M, RB), tiles = tk * tm;
  int ik, im;
  const int split = blockIdx.x / tiles;
  tile_of(blockIdx.x % tiles, tiles, tm, tk, tk, im, ik);
  const int k0 = ik * 256, m0 = im * RB;
  f32x16 acc[P::NA][P::NB];
#pragma unroll
  for (int i = 0; i < P::NA; ++i)
#pragma unroll
    for (int j = 0; j < P::NB; ++j) acc[i][j] = zero16();
  const int words = min(piece, a.V - v_begin), stages = cdiv(words, BK);
  const int s0 = (int)((long)stages * split / splits), s1 = (int)((long)stages * (split + 1) / splits);
  const Source sa = {(const unsigned short*)a.w + (long)v_begin * a.ldw + k0, a.ldw, min(256, a.K - k0), words};
  const Source sb = {e + (long)m0 * piece, piece, min(RB, a.M - m0), words};
  P::run(acc, sa, sb, s0, s1, smem);
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int wk = k0 + wave / (RB / WB) * WA, wm = m0 + wave % (RB / WB) * WB;
#pragma unroll
  for (int j = 0; j < P::NB; ++j) {
    const int m = wm + j * 32 + (lane & 31);
    if (m >= a.M) continue;
#pragma unroll
    for (int i = 0; i < P::NA; ++i)
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        const int k = wk + i * 32 + g * 8 + (lane >> 5) * 4;
        if (k >= a.K) continue;
        f32x4_t* at = (f32x4_t*)(sums + ((long)split * a.M + m) * a.K + k);
        f32x4_t v = {acc[i][j][4 * g], acc[i][j][4 * g + 1], acc[i][j][4 * g + 2], acc[i][j][4 * g + 3]};
        if (v_begin > 0) v += *at;
        *at = v;
      }
  }
}
// (3) K in registers, words in lanes: the piece's rows of dw
template <class E, int RB, int WA, int WB>
__global__ __launch_bounds__((256 / WA) * (RB / WB) * 64) void ce_dw_kernel(simvg_vocab_ce_args a, const unsigned short* xs,
                                                                            const unsigned short* e, int piece, int v_begin, const float* gmax) {
  using P = Product<E, 256, true, RB, true, WA, WB>;
  extern __shared__ __attribute__((aligned(16))) char smem[];
  const int words = min(piece, a.V - v_begin), tk = cdiv(a.K, 256), tv = cdiv(words, RB);
  int ik, iv;
  tile_of(blockIdx.x, tk * tv, tv, tk, tk, iv, ik);
  const int k0 = ik * 256, l0 = iv * RB;
  f32x16 acc[P::NA][P::NB];
#pragma unroll
  for (int i = 0; i < P::NA; ++i)
#pragma unroll
    for (int j = 0; j < P::NB; ++j) acc[i][j] = zero16();
  const Source sa = {xs + k0, a.K, min(256, a.K - k0), a.M};
  const Source sb = {e + l0, piece, min(RB, piece - l0), a.M};
  P::run(acc, sa, sb, 0, cdiv(a.M, BK), smem);
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int wk = k0 + wave / (RB / WB) * WA, wl = l0 + wave % (RB / WB) * WB;
  const float mul = gmax[0] / e_scale<E>();
#pragma unroll
  for (int j = 0; j < P::NB; ++j) {
    const int v = wl + j * 32 + (lane & 31);
    if (v >= words) continue;
    unsigned short* out = (unsigned short*)a.dw + (long)(v_begin + v) * a.lddw;
#pragma unroll
    for (int i = 0; i < P::NA; ++i)
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        const int k = wk + i * 32 + g * 8 + (lane >> 5) * 4;
        if (k < a.K)
          *(u32x2_t*)(out + k) = (u32x2_t){E::pack(acc[i][j][4 * g] * mul, acc[i][j][4 * g + 1] * mul),
                                           E::pack(acc[i][j][4 * g + 2] * mul, acc[i][j][4 * g + 3] * mul)};
      }
  }
}
template <class E>
__global__ __launch_bounds__(256) void ce_dx_join_kernel(simvg_vocab_ce_args a, const float* sums, int splits) {
  const int per = a.K / 4;
  for (long i = blockIdx.x * 256L + threadIdx.x; i < (long)a.M * per; i += (long)gridDim.x * 256) {
    const int m = (int)(i / per), c = (int)(i % per) * 4;
    f32x4_t v = {0.f, 0.f, 0.f, 0.f};
    for (int s = 0; s < splits; ++s) v += *(const f32x4_t*)(sums + ((long)s * a.M + m) * a.K + c);
    const bool on = is_word(a, a.target[m]);
    const float g = on ? a.dloss[m] / e_scale<E>() : 0.f;
    if (!on) v = (f32x4_t){0.f, 0.f, 0.f, 0.f};
    *(u32x2_t*)((unsigned short*)a.dx + (long)m * a.lddx + c) = (u32x2_t){E::pack(v[0] * g, v[1] * g), E::pack(v[2] * g, v[3] * g)};
  }
}
__global__ __launch_bounds__(256) void ce_db_join_kernel(simvg_vocab_ce_args a, const float* db, int groups, const float* gmax) {
  const int v = blockIdx.x * 256 + threadIdx.x;
  if (v >= a.V) return;
  float s = 0.f;
  for (int g = 0; g < groups; ++g) s += db[(long)g * a.V + v];
  a.dbias[v] = s * gmax[0];
}

// ---------------------------------------------------------------------------------------------------------------- host
bool rows16(const void* p, long ld) { return p && (uintptr_t)p % 16 == 0 && ld % 8 == 0; }

int ce_check(const simvg_vocab_ce_args* a, bool bwd) {
  SIMVG_CHECK_ARG(a, "vocab_ce: null argument block");
  SIMVG_CHECK_ARG(a->dtype == SEQ_F16 || a->dtype == SEQ_BF16, "vocab_ce: dtype must be fp16 or bf16");
  SIMVG_CHECK_ARG(a->M >= 0 && a->V >= 1 && a->K >= 8, "vocab_ce: needs M >= 0, V >= 1, K >= 8");
  SIMVG_CHECK_ARG(a->K % 8 == 0, "vocab_ce: K must be a multiple of 8");
  SIMVG_CHECK_ARG(a->M <= 1 << 22 && a->V <= 1 << 24 && a->K <= 1 << 16, "vocab_ce: M, V or K too large");
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

// more than 64 KiB of LDS has to be asked for, once on each device
void allow_lds(const void* kernel, int bytes, std::atomic<unsigned long>& done) {
  int device = 0;
  if (hipGetDevice(&device) != hipSuccess || (device < 64 && done.load() >> device & 1)) return;
  if (hipFuncSetAttribute(kernel, hipFuncAttributeMaxDynamicSharedMemorySize, bytes) == hipSuccess && device < 64) done |= 1ul << device;
}
#define CE_LAUNCH(P, KERNEL, GRID, ...)                                                  \
  do {                                                                                   \
    static std::atomic<unsigned long> done{0};                                           \
    allow_lds((const void*)(KERNEL), P::LDS, done);                                      \
    hipLaunchKernelGGL((KERNEL), dim3(GRID), dim3(P::THREADS), P::LDS, s, __VA_ARGS__);  \
  } while (0)

long ce_fwd_groups(int V, bool small) { return (long)cdiv(V, 256) * (small ? 8 : 2); }

template <class E>
int ce_fwd(const simvg_vocab_ce_args& a, hipStream_t s) {
  const bool small = a.M <= 64;
  const int wa = small ? 32 : 128, groups = cdiv(a.V, wa);
  float* zt = (float*)a.ws;
  float2* part = (float2*)((char*)a.ws + (a.M * 4L + 255) / 256 * 256);
  if (small) {
    using P = Product<E, 256, false, 64, false, 32, 64>;
    CE_LAUNCH(P, (ce_fwd_kernel<E, 64, 32, 64>), cdiv(a.V, 256) * cdiv(a.M, 64), a, part, zt);
  } else {
    using P = Product<E, 256, false, 256, false, 128, 64>;
    CE_LAUNCH(P, (ce_fwd_kernel<E, 256, 128, 64>), cdiv(a.V, 256) * cdiv(a.M, 256), a, part, zt);
  }
  SIMVG_LAUNCH_CHECK();
  hipLaunchKernelGGL(ce_join_kernel, dim3(cdiv(a.M, 32)), dim3(1024), 0, s, a, part, zt, groups);
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
  float *gmax = (float*)ws, *factor = (float*)(ws + p.o_factor), *sums = (float*)(ws + p.o_dx), *db = (float*)(ws + p.o_db);
  unsigned short *xs = (unsigned short*)(ws + p.o_x), *e = (unsigned short*)(ws + p.o_e);
  hipLaunchKernelGGL(ce_gmax_kernel, dim3(1), dim3(1024), 0, s, a, gmax, factor);
  hipLaunchKernelGGL(ce_scale_kernel<E>, dim3(min(2048, cdiv(a.M, 2) )), dim3(256), 0, s, a, factor, xs);
  SIMVG_LAUNCH_CHECK();
  const int tk = cdiv(a.K, 256);
  for (int v = 0; v < a.V; v += p.piece) {
    const int words = min(p.piece, a.V - v);
    if (p.small) {
      using P1 = Product<E, 64, false, 256, false, 64, 32>;
      using P2 = Product<E, 256, true, 64, false, 32, 64>;
      CE_LAUNCH(P1, (ce_e_kernel<E, 64, 64, 32>), cdiv(a.M, 64) * (p.piece / 256), a, factor, e, p.piece, v, db);
      CE_LAUNCH(P2, (ce_dx_kernel<E, 64, 32, 64>), cdiv(a.M, 64) * tk * p.splits, a, e, p.piece, v, p.splits, sums);
    } else {
      using P1 = Product<E, 256, false, 256, false, 128, 64>;
      using P2 = Product<E, 256, true, 256, false, 128, 64>;
      CE_LAUNCH(P1, (ce_e_kernel<E, 256, 128, 64>), cdiv(a.M, 256) * (p.piece / 256), a, factor, e, p.piece, v, db);
      CE_LAUNCH(P2, (ce_dx_kernel<E, 256, 128, 64>), cdiv(a.M, 256) * tk * p.splits, a, e, p.piece, v, p.splits, sums);
    }
    using P3 = Product<E, 256, true, 256, true, 128, 64>;
    CE_LAUNCH(P3, (ce_dw_kernel<E, 256, 128, 64>), tk * cdiv(words, 256), a, xs, e, p.piece, v, gmax);
    SIMVG_LAUNCH_CHECK();
  }
  hipLaunchKernelGGL(ce_dx_join_kernel<E>, dim3(min(2048, cdiv(a.M, 2))), dim3(256), 0, s, a, sums, p.splits);
  if (a.dbias) hipLaunchKernelGGL(ce_db_join_kernel, dim3(cdiv(a.V, 256)), dim3(256), 0, s, a, db, cdiv(a.M, p.small ? 64 : 128), gmax);
  SIMVG_LAUNCH_CHECK();
  return SIMVG_OK;
}
}  // namespace

extern "C" long simvg_vocab_ce_ws_bytes(int M, int V, int K, int with_bias, int backward) {
  if (M <= 0 || V <= 0 || K <= 0) return 0;
  if (backward) return ce_plan(M, V, K, with_bias != 0).bytes;
  return (M * 4L + 255) / 256 * 256 + ce_fwd_groups(V, M <= 64) * M * 8;
}
extern "C" int simvg_vocab_ce_fwd(const simvg_vocab_ce_args* args, hipStream_t stream) {
  const int rc = ce_check(args, false);
  if (rc || args->M == 0) return rc;
  SIMVG_CHECK_ARG(args->ws && (uintptr_t)args->ws % 256 == 0 && args->ws_bytes >= simvg_vocab_ce_ws_bytes(args->M, args->V, args->K, args->bias != nullptr, 0),
                  "vocab_ce: the workspace is too small or misaligned");
  return args->dtype == SEQ_F16 ? ce_fwd<F16>(*args, stream) : ce_fwd<BF16>(*args, stream);
}
extern "C" int simvg_vocab_ce_bwd(const simvg_vocab_ce_args* args, hipStream_t stream) {
  const int rc = ce_check(args, true);
  if (rc) return rc;
  if (args->M == 0) {                                        // sums of nothing
    hipLaunchKernelGGL(ce_zero_kernel, dim3(1024), dim3(256), 0, stream, (unsigned short*)args->dw, args->lddw, args->V, args->K, args->dbias);
    SIMVG_LAUNCH_CHECK();
    return SIMVG_OK;
  }
  SIMVG_CHECK_ARG(args->ws && (uintptr_t)args->ws % 256 == 0 && args->ws_bytes >= simvg_vocab_ce_ws_bytes(args->M, args->V, args->K, args->dbias != nullptr, 1),
                  "vocab_ce: the workspace is too small or misaligned");
  return args->dtype == SEQ_F16 ? ce_bwd<F16>(*args, stream) : ce_bwd<BF16>(*args, stream);
}
