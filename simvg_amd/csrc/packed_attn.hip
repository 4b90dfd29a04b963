// simvg-build-flags: -Wno-inline-asm
// Attention over packed sequences, forward and backward: rows [cu[s], cu[s + 1]) of q, k, v are sequence s.  A row sees the keys of its
// own sequence, under `causal` those up to itself; Hq heads of q share Hkv heads of k and v, G = Hq / Hkv neighbours each.
//
//   S = scale q k^T,  lse_i = log sum_j exp(S_ij),  P = exp(S - lse),  O = P V
//   backward: D_i = sum_d dO_id O_id;  dV = P^T dO;  dP = dO V^T;  dS = P (dP - D);  dQ = scale dS K;  dK = scale dS^T Q
//
// Bound by the matrix pipes (4 D products per visible pair forward, 10 D backward).  One workgroup takes 128 rows of one sequence and
// head, a wave 32 of them, in tiles of 64 keys (queries, for dK and dV) that pass through LDS once for the workgroup.  All scores are
// computed transposed, S^T = K Q^T by 32x32x16 MFMAs: a lane then holds ONE query's scores (keys in its registers), so that the
// softmax needs a single exchange, between the two halves of the wave, and what the next product takes as its B operand is what the
// lane already has -- the order of the contraction's keys is free, and the transposed reads (ds_read_b64_tr_b16) that fetch V^T use
// the order in which the accumulator holds them.  P and dS never leave registers.
//
// Measured, medians, of 1.46 (fp16) and 1.44 (bf16) PFLOP/s that a library product of 8192^3 reaches: one sequence of 16384 rows, 16 heads
// of 128 on 2, causal, bf16, forward 1.00 ms (1.05 on a slower card), 1.10 PFLOP/s; nine of up to 4097 rows, 32 heads on 8: forward 0.49 ms,
// 0.92; dQ 0.69 ms and dK, dV 1.05 ms, 0.99 and 0.86 of what each computes (6 D and 8 D: both need the scores).  Half of the time the matrix
// pipes work (the clock falls to 1.7 GHz under them), a third goes to the exponentials and the rest of the vector work, which one or two
// waves to a SIMD cover in part.  Heads of 64 (64 x 411 rows, 12 heads, no mask, fp16): forward 66 us, delta and norms 24, dQ 91, dK and dV
// 133: vector work, as much for half the products, and for dK and dV start and end of workgroups of seven tiles, about half of their time.
//
// Which rows a workgroup takes stands in a plan that the caller has built once for a batch (packed_plan_kernel): one entry for each
// tile of 128 rows of each sequence, tiles far down a sequence first, because under `causal` they cost most and the last workgroups to
// start should be the short ones.
//
// Masks: rows and keys past a sequence are zeros in LDS and are never stored, so nothing of a neighbour is read.  In a tile that the
// diagonal crosses, P is an exact 0 above it, and 0 x inf in the matrix product would still carry a later row's inf or NaN to an
// earlier one: such a tile is looked through for values that are not finite, and if there are any they are added, as themselves, to the
// rows that do see them and taken out of the tile (`add_nonfinite`, `tile_clean`).
#include <algorithm>
#include <type_traits>
#include <utility>

#include "seq.h"

struct simvg_packed_attn_args {
  int dtype, T, nseq, Hq, Hkv, D, causal, fill_tail;        // fill_tail: rows past the last sequence become zeros (else: as they were); 2: lse's alone
  float scale;
  const int* plan;
  const void* q; long q_ts, q_hs; const void* k; long k_ts, k_hs; const void* v; long v_ts, v_hs;
  void* o; long o_ts, o_hs;                                  // forward: output; backward: the forward's output
  float* lse; long lse_hs;                                   // [Hq][T]: head stride, rows are neighbours
  const void* d_o; long do_ts, do_hs;                        // backward
  void* dq; long dq_ts, dq_hs; void* dk; long dk_ts, dk_hs; void* dv; long dv_ts, dv_hs;
  float* ws;                                                 // simvg_packed_attn_ws_floats() floats
};

namespace {
using namespace seq;

constexpr int QT = 128;                                      // rows of a plan entry
constexpr int KT = 64;                                       // rows of a tile in LDS
// Up to this many tiles of keys to a workgroup's queries (queries to its keys) P and dS go into their products in two parts, as rounded to
// 16 bits and what that took off: a result of few terms, in a batch of few and short sequences, shows their rounding beside its own
// (154 sequences of two rows: dQ off by 1.53 of what its last rounding costs, bf16), longer sums keep sqrt(2) of it.
constexpr int FEW = 2;
constexpr float LOG2E = 1.44269504088896340736f;
constexpr float NEG_INF = -__builtin_huge_valf();
constexpr float FAR = 4096.f;                                // exponents beyond it: the reference is subtracted before the scaling, not in its fma

// ---------------------------------------------------------------------------------------------------------------- the plan
// ints: [0] entries, [1] the row after the last sequence (-1: `cu` is no such list, there are no entries), [2..3] unused, then int4
// {first row, rows, tile of the sequence, tiles of all sequences before} per entry, tiles far down their sequence first, then the same
// entries in their natural order, then nseq + 1 prefix sums of tiles (used while building).  A list that does not start at 0, falls, or
// passes T is found here, so the kernels below stay inside their tensors
// whatever it holds.
constexpr int FILL_LSE = 2;                                  // fill_tail of a forward pass into a result of the caller's
constexpr int PLAN_HEAD = 4, PLAN_BINS = 1024;
// one more than the tiles of any valid list: what a launch has left over is enough for the tiles behind the last sequence
__host__ __device__ __forceinline__ int plan_capacity(int T, int nseq) { return T / QT + nseq + 1; }

// sum of the values of threads 0 .. tid, and of all 1024
__device__ __forceinline__ int scan1024(int v, int (&waves)[16], int tid, int& total) {
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const int up = __shfl_up(v, o, 64);
    if ((tid & 63) >= o) v += up;
  }
  if ((tid & 63) == 63) waves[tid >> 6] = v;
  __syncthreads();
  total = 0;
#pragma unroll
  for (int w = 0; w < 16; ++w) {
    if (w < tid >> 6) v += waves[w];
    total += waves[w];
  }
  __syncthreads();
  return v;
}
__global__ __launch_bounds__(1024) void packed_plan_kernel(const int* cu, int nseq, int T, int* plan) {
  __shared__ int waves[16], bins[PLAN_BINS];
  const int tid = threadIdx.x, cap = plan_capacity(T, nseq);
  int *natural = plan + PLAN_HEAD + 4 * cap, *base = natural + 4 * cap;
  int bad = cu[0] != 0;
  for (int s = tid; s < nseq; s += 1024) bad |= cu[s + 1] < cu[s] || cu[s + 1] > T;
  if (__syncthreads_or(bad)) {
    if (tid == 0) { plan[0] = 0; plan[1] = -1; }
    return;
  }
  int total = 0;
  for (int s0 = 0; s0 < nseq; s0 += 1024) {                  // prefix sums of the sequences' tiles
    const int s = s0 + tid, mine = s < nseq ? (cu[s + 1] - cu[s] + QT - 1) / QT : 0;
    int all;
    const int upto = scan1024(mine, waves, tid, all);
    if (s < nseq) base[s] = total + upto - mine;
    total += all;
  }
  if (tid == 0) { base[nseq] = total; plan[0] = total; plan[1] = cu[nseq]; }
  bins[tid] = 0;
  __threadfence_block();
  __syncthreads();
  // tiles far down their sequence first: count them by their place, then hand out the places from the back
  for (int pass = 0; pass < 2; ++pass) {
    for (int i = tid; i < total; i += 1024) {
      int lo = 0, hi = nseq;                                 // the sequence with base[s] <= i < base[s + 1]
      while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (base[mid] <= i) lo = mid; else hi = mid;
      }
      const int t = i - base[lo], bin = PLAN_BINS - 1 - min(t, PLAN_BINS - 1);
      const int at = atomicAdd(&bins[bin], 1);               // the order within a bin changes which workgroup does a tile, not what it does
      if (pass) {
        const int first = cu[lo], len = cu[lo + 1] - first;
        int *e = plan + PLAN_HEAD + 4 * at, *f = natural + 4 * i;
        e[0] = f[0] = first; e[1] = f[1] = len; e[2] = f[2] = t; e[3] = f[3] = base[lo];
      }
    }
    __syncthreads();
    if (!pass) {                                             // counts to starting places
      int all;
      const int mine = bins[tid], upto = scan1024(mine, waves, tid, all);
      bins[tid] = upto - mine;
      __syncthreads();
    }
  }
}

// --------------------------------------------------------------------------------------------------- tiles and fragments
// A tile in LDS: rows of DP 16-bit values, in slots of 16 bytes.  Slot s of row r lies at s ^ swizzle(r): the row-wise fragments read
// 16 rows of one slot in a cycle (ds_read_b128), the transposed ones 4 rows of four neighbouring slots, and both then touch every bank
// once.
template <int DP>
__device__ __forceinline__ int tile_at(int row, int slot) {
  const int x = DP == 128 ? ((row & 3) << 2 | (row >> 2 & 3)) : ((row >> 1 & 1) << 2 | (row >> 2 & 3));
  return row * (DP * 2) + ((slot ^ x) << 4);
}

// in a branch that few tiles take: keeps hipcc from computing it for all of them and selecting
__device__ __forceinline__ void stay_a_branch() { asm volatile(""); }

// Brings tiles of KT rows of a head from HBM to LDS (LDS-DMA, seq.h), one after the other, the work of four waves: zeros past the
// sequence's rows and past D.  LDS0: where the array's tiles of this operand start.
template <int DP, int LDS0> struct Stager {
  static constexpr int PIECES = KT * DP * 2 / 4096;
  unsigned off[PIECES], lds;                                 // lds: of the wave's first piece
  unsigned long base;                                        // the next tile's first row
  unsigned step;                                             // bytes from tile to tile
  int row, left;                                             // the lane's row of its first piece; the sequence's rows from the next tile on
  unsigned place = 0;                                        // added to LDS0, where the buffer's number is no constant
  __device__ __forceinline__ void init(const void* first, long ts, int rows, int D, const char* smem, int wave, int lane) {
    const int r0 = (wave * 1024 + lane * 16) / (DP * 2);
    base = (unsigned long)first;
    step = (unsigned)(KT * 2) * (unsigned)ts;
    lds = lds_addr(smem) + LDS0 + wave * 1024;
    left = rows;
    row = r0;
#pragma unroll
    for (int i = 0; i < PIECES; ++i) {
      const int byte = (i * 4 + wave) * 1024 + lane * 16, r = byte / (DP * 2);
      const int slot = (tile_at<DP>(r, byte % (DP * 2) / 16) - r * DP * 2) >> 4;       // the permutation is its own inverse
      off[i] = slot * 8 < D ? (unsigned)(r * (int)ts * 2 + slot * 16) : DMA_NOTHING;
    }
  }
  template <int BUF> __device__ __forceinline__ void next() {
    const u32x4_t b = {(unsigned)base, (unsigned)(base >> 32) & 0xffffu, DMA_NOTHING - 1, 0x00020000u};
    unsigned o[PIECES];
#pragma unroll
    for (int i = 0; i < PIECES; ++i) o[i] = off[i];
    if (left < KT) {
      stay_a_branch();
#pragma unroll
      for (int i = 0; i < PIECES; ++i)
        if (row + i * (2048 / DP) >= left) o[i] = DMA_NOTHING;
    }
    issue<BUF>(b, o, std::make_integer_sequence<int, PIECES>{});
    base += step;
    left -= KT;
  }
  template <int BUF, int... I> __device__ __forceinline__ void issue(u32x4_t b, const unsigned (&o)[PIECES], std::integer_sequence<int, I...>) {
    (dma16_at<BUF * KT * DP * 2 + I * 4096>(b, lds + place, o[I]), ...);
  }
};
// What a lane adds to a tile's start for its part of a fragment; everything else of an address is a constant in the instruction.
//   row(rb, ks): A operand from rows: row 32 rb + (lane & 31), columns 16 ks + 8 (lane >> 5) ..
//   col(rk, cb): A operand from columns: column 32 cb + (lane & 31), the 16 rows 16 rk .. in the order of a 32x32 accumulator's registers
template <int DP> struct Lanes {
  static constexpr int ROWB = DP * 2;
  typedef __attribute__((address_space(3))) const char* Lds;
  Lds r[DP / 16], c[DP / 32][2];
  __device__ __forceinline__ void init(const char* smem, int lane) {
    const int i = lane & 15, row = 4 * (lane >> 5) + (i >> 2);
    const Lds base = (Lds)(const __attribute__((address_space(3))) void*)LDS_PTR(smem);
#pragma unroll
    for (int ks = 0; ks < DP / 16; ++ks) r[ks] = base + tile_at<DP>(lane & 31, ks * 2 + (lane >> 5));
#pragma unroll
    for (int cb = 0; cb < DP / 32; ++cb) {
      const int col = cb * 32 + (lane >> 4 & 1) * 16 + 4 * (i & 3);
      c[cb][0] = base + tile_at<DP>(row, col >> 3) + (col & 7) * 2;
      c[cb][1] = base + tile_at<DP>(row + 8, col >> 3) + (col & 7) * 2;
    }
  }
  // `tile`: bytes from the start of the LDS array
  __device__ __forceinline__ lpx8_t row(int tile, int rb, int ks) const {
    return *(const __attribute__((address_space(3))) lpx8_t*)(r[ks] + tile + rb * 32 * ROWB);
  }
  __device__ __forceinline__ lpx8_t col(int tile, int rk, int cb) const {
    typedef __attribute__((address_space(3))) lpx4_t* P;
    const lpx4_t lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((P)(c[cb][0] + tile + rk * 16 * ROWB));
    const lpx4_t hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((P)(c[cb][1] + tile + rk * 16 * ROWB));
    return (lpx8_t){lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
  }
};
// B operand kept in registers: row `row` of a head (zeros past D), columns 16 ks + 8 (lane >> 5) ..
__device__ __forceinline__ lpx8_t global_frag(const unsigned short* base, int ks, int D, int lane) {
  const int col = ks * 16 + 8 * (lane >> 5);
  return col < D ? *(const lpx8_t*)(base + col) : (lpx8_t){0, 0, 0, 0, 0, 0, 0, 0};
}
// Loaded before a loop that has DMA in flight: taken here, so that hipcc's wait for the load stands here and not at the first use in
// the loop, where it would wait for the tile that has just been asked for, at every tile
template <int N> __device__ __forceinline__ void arrived(lpx8_t (&f)[N]) {
#pragma unroll
  for (int i = 0; i < N; ++i) asm volatile("" : "+v"(f[i]));
}
__device__ __forceinline__ void arrived(float& f) { asm volatile("" : "+v"(f)); }
// registers 8 rk .. 8 rk + 7 of an accumulator as the B operand of a product over its rows
template <class E>
__device__ __forceinline__ lpx8_t acc_frag(const f32x16& p, int rk) {
  const u32x4_t u = {E::pack(p[8 * rk], p[8 * rk + 1]), E::pack(p[8 * rk + 2], p[8 * rk + 3]), E::pack(p[8 * rk + 4], p[8 * rk + 5]),
                     E::pack(p[8 * rk + 6], p[8 * rk + 7])};
  return __builtin_bit_cast(lpx8_t, u);
}
// what that rounding took off them: the registers less what the operand holds
template <class E>
__device__ __forceinline__ lpx8_t acc_rest(f32x16& p, int rk) {
#pragma unroll
  for (int r = 8 * rk; r < 8 * rk + 8; r += 2) {
    float a, b;
    unpack2<E>(E::pack(p[r], p[r + 1]), a, b);
    p[r] -= a;
    p[r + 1] -= b;
  }
  return acc_frag<E>(p, rk);
}
// the other half of the wave's value of v (lane ^ 32), joined with this half's
__device__ __forceinline__ float max_halves(float v) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float add_halves(float v) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}
// row of a 32x32 accumulator's register r: a constant, and 4 more in the upper half of the wave
__device__ __forceinline__ constexpr int reg_row(int r) { return (r >> 2) * 8 + (r & 3); }
__device__ __forceinline__ int acc_row(int r, int lane) { return reg_row(r) + (lane >> 5) * 4; }
__device__ __forceinline__ f32x16 zero16() { return (f32x16){0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f}; }

// ---- values that are not finite in a tile that the mask crosses
// (integer arithmetic and no comparisons: unrolled, their results would fill the scalar registers)
template <class E>
__device__ __forceinline__ unsigned finite_mask(unsigned u) {          // all bits of each half that holds a finite value
  const int lo = (int)(u & 0x7fffu) - E::kInf, hi = (int)(u >> 16 & 0x7fffu) - E::kInf;
  return ((unsigned)(lo >> 31) & 0xffffu) | ((unsigned)(hi >> 31) << 16);
}
// a fragment with zeros where values are not finite
template <class E>
__device__ __forceinline__ lpx8_t finite(lpx8_t f) {
  u32x4_t v = __builtin_bit_cast(u32x4_t, f);
#pragma unroll
  for (int j = 0; j < 4; ++j) v[j] &= finite_mask<E>(v[j]);
  return __builtin_bit_cast(lpx8_t, v);
}
// The workgroup's 256 threads look through a tile, each its share; the same answer in all of them.  (The barrier inside also waits for
// the tile that is on its way: this is done for the two or three tiles of a workgroup that a mask crosses, not for the others.)
template <class E, int DP>
__device__ __forceinline__ bool tile_nonfinite(const char* lds) {
  unsigned bad = 0;
#pragma unroll
  for (int i = 0; i < KT * DP * 2 / 4096; ++i) {
    const u32x4_t v = *(const u32x4_t*)(lds + (i * 256 + threadIdx.x) * 16);
#pragma unroll
    for (int j = 0; j < 4; ++j) bad |= ~finite_mask<E>(v[j]);
  }
  return __syncthreads_or(bad != 0);
}
// ... and put zeros where values are not finite, once every wave has read what it needs of them
template <class E, int DP>
__device__ __forceinline__ void tile_clean(char* lds) {
  __syncthreads();
  for (int i = 0; i < KT * DP * 2 / 4096; ++i) {
    u32x4_t* at = (u32x4_t*)(lds + (i * 256 + threadIdx.x) * 16);
    u32x4_t v = *at;
#pragma unroll
    for (int j = 0; j < 4; ++j) v[j] &= finite_mask<E>(v[j]);
    *at = v;
  }
  __syncthreads();
}
// acc[cb] holds columns 32 cb .. of the lane's row; `sees(j)`: whether that row sees row j of the tile.  What `tile_clean` will take out
// is added here: as itself where it multiplies a probability, as NaN where it multiplies dS, whose sign says nothing.
template <class E, int DP, bool NAN_ONLY, class Sees>
__device__ __forceinline__ void add_nonfinite(f32x16 (&acc)[DP / 32], const char* lds, int lane, Sees sees) {
#pragma unroll 1
  for (int j = 0; j < KT; ++j) {
    if (!sees(j)) continue;
#pragma unroll
    for (int cb = 0; cb < DP / 32; ++cb)
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        const int col = cb * 32 + acc_row(r, lane);
        const unsigned short b = *(const unsigned short*)(lds + tile_at<DP>(j, col >> 3) + (col & 7) * 2);
        const float x = E::to_f32((unsigned short)(b & ~finite_mask<E>(b)));           // 0 where it is finite
        acc[cb][r] += NAN_ONLY ? x - x : x;
      }
  }
}

// Workgroup j of the Hq of a tile runs on XCD j mod 8 if 8 divides Hq: heads that share a key head go to the same one, whose L2 then
// holds that head's k and v and not everybody's
__device__ __forceinline__ int head_of(int j, int Hq) { return Hq % 8 ? j : j % 8 * (Hq / 8) + j / 8; }

struct Tile { int first, len, t, base; };
__device__ __forceinline__ bool plan_entry(const simvg_packed_attn_args& a, int id, Tile& e) {
  const int* p = a.plan + PLAN_HEAD + 4 * id;                // the grid is as long as the table: the entry is read beside the count
  int n = a.plan[0], first = p[0], len = p[1], t = p[2], base = p[3];
  asm volatile("" : "+s"(n), "+s"(first), "+s"(len), "+s"(t), "+s"(base));
  e.first = first; e.len = len; e.t = t; e.base = base;
  return id < n;
}
// Which tile, head and part of the work a workgroup takes; false: it has none, and `id` - plan[0] counts those.  Where costs differ
// (`causal`) or work is cut, the order is the plan's, heads next to each other.  Otherwise an XCD (workgroup number mod 8) takes a
// contiguous eighth of (head, sequence, tile): the tiles of a sequence and head read the same rows, at the same time, from one L2 (64 x 411
// rows, 12 heads of 64: forward 69 -> 66 us, backward 255 -> 250).
template <bool CAUSAL>
__device__ __forceinline__ bool workgroup(const simvg_packed_attn_args& a, int H, int parts, int& h, int& part, int& id, Tile& e) {
  const int b = blockIdx.x;
  if (CAUSAL || parts > 1) {
    h = head_of(b % H, H);
    part = b / H % parts;
    id = b / H / parts;
    return plan_entry(a, id, e);
  }
  const int n = a.plan[0], all = n * H;
  part = 0;
  if (b >= all) {
    h = (b - all) % H;
    id = n + (b - all) / H;
    return false;
  }
  const int q = all >> 3, r = all & 7, xcd = b & 7, u = xcd * q + min(xcd, r) + (b >> 3);
  h = u / n;
  id = u % n;
  const int* p = a.plan + PLAN_HEAD + 4 * (plan_capacity(a.T, a.nseq) + id);
  e.first = p[0]; e.len = p[1]; e.t = p[2]; e.base = p[3];
  return true;
}
// a workgroup without an entry: its tile of the rows behind the last sequence, zeros; NaN everywhere where there is no valid plan
__device__ __forceinline__ void fill_tail(const simvg_packed_attn_args& a, int id, void* out, long ts, long hs, int h, float* lse) {
  if (!a.fill_tail || (a.fill_tail == FILL_LSE && !lse)) return;
  const bool invalid = a.plan[1] < 0;
  const long row0 = (invalid ? 0L : a.plan[1]) + (id - a.plan[0]) * (long)QT;
  const int rows = (int)min((long)QT, a.T - row0);
  const unsigned short value = invalid ? 0x7fff : 0;         // a NaN in fp16 and in bf16
  if (a.fill_tail != FILL_LSE)
    for (int i = threadIdx.x; i < rows * a.D; i += 256) ((unsigned short*)out)[(row0 + i / a.D) * ts + (long)h * hs + i % a.D] = value;
  if (lse)
    for (int i = threadIdx.x; i < rows; i += 256) lse[(long)h * a.lse_hs + row0 + i] = invalid ? __builtin_nanf("") : 0.f;
}
// the 32 x DP block that a wave holds transposed (lane = row, registers = columns) to its rows of `out`
template <class E, int DP>
__device__ __forceinline__ void store_rows(const f32x16 (&acc)[DP / 32], float mul, unsigned short* out, int D, bool valid, int lane) {
#pragma unroll
  for (int cb = 0; cb < DP / 32; ++cb)
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      const int col = cb * 32 + g * 8 + (lane >> 5) * 4;
      if (valid && col < D)
        *(u32x2_t*)(out + col) = (u32x2_t){E::pack(acc[cb][4 * g] * mul, acc[cb][4 * g + 1] * mul),
                                           E::pack(acc[cb][4 * g + 2] * mul, acc[cb][4 * g + 3] * mul)};
    }
}

// ... in 32 bits
template <int DP>
__device__ __forceinline__ void store_sums(const f32x16 (&acc)[DP / 32], float mul, float* out, int D, bool valid, int lane) {
#pragma unroll
  for (int cb = 0; cb < DP / 32; ++cb)
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      const int col = cb * 32 + g * 8 + (lane >> 5) * 4;
      if (valid && col < D) *(f32x4_t*)(out + col) = (f32x4_t){acc[cb][4 * g], acc[cb][4 * g + 1], acc[cb][4 * g + 2], acc[cb][4 * g + 3]} * mul;
    }
}

// ------------------------------------------------------------------------------------------------------------- forward
// ws, where the keys are cut into parts: (reference, sum) [parts][T][Hq], a multiple of 16 bytes, then numerators [parts][T][Hq][D]
__host__ __device__ __forceinline__ long ws_stats(long parts, long T, long Hq) { return (2 * parts * T * Hq + 3) / 4 * 4; }
template <class E, int DP, bool CAUSAL, bool SHORT>
__global__ __launch_bounds__(256, DP == 64 ? 3 : 2) void packed_attn_fwd_kernel(simvg_packed_attn_args a, int parts) {
  extern __shared__ __attribute__((aligned(16))) char smem[];
  constexpr int TILE = KT * DP * 2, DB = DP / 32, KS = DP / 16;
  int h, part, id;
  Tile e;
  if (!workgroup<CAUSAL>(a, a.Hq, parts, h, part, id, e)) {
    if (part == 0) fill_tail(a, id, a.o, a.o_ts, a.o_hs, h, a.lse);
    return;
  }
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
  const int hk = h / (a.Hq / a.Hkv);
  const int row = e.t * QT + wave * 32 + (lane & 31);        // the lane's query
  const bool valid = row < e.len;
  const unsigned short* qp = (const unsigned short*)a.q + (long)(e.first + min(row, e.len - 1)) * a.q_ts + (long)h * a.q_hs;
  const unsigned short* kp = (const unsigned short*)a.k + (long)e.first * a.k_ts + (long)hk * a.k_hs;
  const unsigned short* vp = (const unsigned short*)a.v + (long)e.first * a.v_ts + (long)hk * a.v_hs;
  // the tiles of keys, and this part's of them: [kt0, tiles)
  const int keys = CAUSAL ? min(e.len, (e.t + 1) * QT) : e.len, all_tiles = (keys + KT - 1) / KT;
  const int kt0 = all_tiles * part / parts, tiles = all_tiles * (part + 1) / parts;
  const bool few = SHORT && all_tiles <= FEW;
  const int wave_first = e.t * QT + wave * 32;               // the wave's first query
  // tiles that no mask touches come first, then those that the diagonal or the sequence's end crosses, then (for the wave) nothing
  const int whole = min(tiles, min(CAUSAL ? (e.t * QT + 1) / KT : tiles, e.len / KT));         // of all four waves
  const int wave_whole = min(CAUSAL ? (wave_first + 1) / KT : tiles, e.len / KT);
  const bool live = wave_first < e.len;                      // a wave without a row only brings its pieces of the tiles
  const int wave_tiles = !live ? 0 : CAUSAL ? min(tiles, (wave_first + 32 + KT - 1) / KT) : tiles;

  Stager<DP, 0> gk;
  Stager<DP, 2 * TILE> gv;
  gk.init(kp + (long)kt0 * KT * a.k_ts, a.k_ts, e.len - kt0 * KT, a.D, smem, wave, lane);
  gv.init(vp + (long)kt0 * KT * a.v_ts, a.v_ts, e.len - kt0 * KT, a.D, smem, wave, lane);
  if (kt0 < tiles) {
    gk.template next<0>();
    gv.template next<0>();
  }
  if (few && kt0 + 1 < tiles) {
    gk.template next<1>();
    gv.template next<1>();
  }
  lpx8_t qf[KS];
#pragma unroll
  for (int ks = 0; ks < KS; ++ks) qf[ks] = global_frag(qp, ks, a.D, lane);
  arrived(qf);
  Lanes<DP> at;
  at.init(smem, lane);
  f32x16 o[DB];
#pragma unroll
  for (int i = 0; i < DB; ++i) o[i] = zero16();
  const float c = a.scale * LOG2E;
  float m = NEG_INF, l = 0.f;                                // reference of the exponentials (raw scores), sum over this half's keys

  // One tile.  The buffer's number is a constant, so that every LDS address is a lane's register and a constant; MASKED: a mask crosses
  // it for some wave.
  auto tile = [&](int kt, auto which, auto crossed) {
    constexpr int BUF = decltype(which)::value, K0 = BUF * TILE, V0 = (2 + BUF) * TILE;
    constexpr bool MASKED = decltype(crossed)::value;
    dma_wait<0>();                                           // this wave's pieces of the tile
    wave_barrier_only();                                     // everybody's; and everybody is done with the other buffer
    if (kt + 1 < tiles) {
      gk.template next<BUF ^ 1>();
      gv.template next<BUF ^ 1>();
    }
    const bool odd = MASKED && tile_nonfinite<E, DP>(smem + V0), mine = MASKED ? kt < wave_tiles : live;
    const int last = (CAUSAL ? min(row, e.len - 1) : e.len - 1) - kt * KT;     // of the tile's keys, the last that the lane's query sees
    const int last4 = last - (lane >> 5) * 4;                // against a register's constant
    f32x16 s[2];
    if (mine) {
      s[0] = s[1] = zero16();                                // two chains of products, one waits for its own result less often
#pragma unroll
      for (int ks = 0; ks < KS; ++ks)
#pragma unroll
        for (int kb = 0; kb < 2; ++kb) s[kb] = E::mfma(at.row(K0, kb, ks), qf[ks], s[kb]);
      if (MASKED && kt >= wave_whole) {
#pragma unroll
        for (int kb = 0; kb < 2; ++kb)
#pragma unroll
          for (int r = 0; r < 16; ++r)
            if (kb * 32 + reg_row(r) > last4) s[kb][r] = NEG_INF;
      }
      float top = NEG_INF;
#pragma unroll
      for (int kb = 0; kb < 2; ++kb)
#pragma unroll
        for (int r = 0; r < 16; ++r) top = fmaxf(top, s[kb][r]);
      top = max_halves(top);
      // the reference follows the maximum only where it has grown by more than 2^8: the exponentials stay below 2^8, and what is
      // left of O and l need not be scaled at every tile.  (Each row by itself: its neighbours in the wave change no bit of it.)
      if (__any((top - m) * c > 8.f || fabsf(m * c) > FAR)) {
        const float to = (top - m) * c > 8.f ? top : m, f = m == to ? 1.f : __builtin_amdgcn_exp2f((m - to) * c);
        m = to;
        l *= f;
#pragma unroll
        for (int i = 0; i < DB; ++i) o[i] *= f;
        // m c is rounded, and off by hundreds of powers of two while a row has seen nothing but scores of -1e10 (keys that a feature takes
        // out): its exponentials would be inf, not 1
        const bool far = fabsf(m * c) > FAR && m != NEG_INF;
        if (__any(far)) {
          stay_a_branch();
#pragma unroll
          for (int kb = 0; kb < 2; ++kb) s[kb] -= far ? m : 0.f;
        }
      }
    }
    if (odd) {
      if (mine) add_nonfinite<E, DP, false>(o, smem + V0, lane, [&](int j) { return j <= last; });
      tile_clean<E, DP>(smem + V0);
    }
    if (mine) {
      // the exponentials of 16 keys and the products of the 16 before: vector and matrix pipes at the same time
      const float mc = fabsf(m * c) > FAR ? 0.f : m * c;     // (nothing but scores of -inf so far: exponentials of 0, not NaN)
      lpx8_t p[4];
      auto exps = [&](int rk) {
        f32x16& x = s[rk >> 1];
#pragma unroll
        for (int r = 8 * (rk & 1); r < 8 * (rk & 1) + 8; ++r) {
          x[r] = __builtin_amdgcn_exp2f(fmaf(x[r], c, -mc));
          l += x[r];
        }
        p[rk] = acc_frag<E>(x, rk & 1);
      };
      exps(0);
#pragma unroll
      for (int rk = 0; rk < 4; ++rk) {
        lpx8_t v[DB];
#pragma unroll
        for (int cb = 0; cb < DB; ++cb) v[cb] = at.col(V0, rk, cb);
#pragma unroll
        for (int cb = 0; cb < DB; ++cb) o[cb] = E::mfma(v[cb], p[rk], o[cb]);
        if (rk < 3) exps(rk + 1);
      }
    }
  };
  auto finish = [&] {
    l += __shfl_xor(l, 32, 64);
    const auto z = late_args<simvg_packed_attn_args>();
    if (parts == 1) {
      unsigned short* out = (unsigned short*)z->o + (long)(e.first + row) * z->o_ts + (long)h * z->o_hs;
      store_rows<E, DP>(o, 1.f / l, out, z->D, valid, lane);
      if (valid && lane < 32) z->lse[(long)h * z->lse_hs + e.first + row] = m * z->scale + __builtin_logf(l);
    } else {
      const long n = (long)z->T * z->Hq, at = (long)(e.first + row) * z->Hq + h;
      store_sums<DP>(o, 1.f, z->ws + ws_stats(parts, z->T, z->Hq) + (part * n + at) * z->D, z->D, valid, lane);
      if (valid && lane < 32) ((float2*)z->ws)[part * n + at] = make_float2(m, l);
    }
  };
  if (few) {
    // Both tiles are in LDS, one behind the other: 32 keys at a time, the maximum first, then exponentials and products
    dma_wait<0>();
    wave_barrier_only();
    bool odd = false;
    for (int kt = 0; kt < tiles - kt0; ++kt) odd |= tile_nonfinite<E, DP>(smem + (2 + kt) * TILE);
    const int last = (CAUSAL ? min(row, e.len - 1) : e.len - 1) - kt0 * KT;
    const int wave_last = (CAUSAL ? min(wave_first + 31, e.len - 1) : e.len - 1) - kt0 * KT;
    const int blocks = live ? min(2 * (tiles - kt0), (wave_last >> 5) + 1) : 0;
    auto scores = [&](int b) {
      const int last4 = last - b * 32 - (lane >> 5) * 4;
      f32x16 s = zero16();
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) s = E::mfma(at.row(b * 32 * DP * 2, 0, ks), qf[ks], s);
#pragma unroll
      for (int r = 0; r < 16; ++r)
        if (reg_row(r) > last4) s[r] = NEG_INF;
      return s;
    };
#pragma unroll 1
    for (int b = 0; b < blocks; ++b) {
      const f32x16 s = scores(b);
#pragma unroll
      for (int r = 0; r < 16; ++r) m = fmaxf(m, s[r]);
    }
    m = max_halves(m);
    if (odd && live)
      for (int kt = 0; kt < tiles - kt0; ++kt)
        add_nonfinite<E, DP, false>(o, smem + (2 + kt) * TILE, lane, [&](int j) { return j <= last - kt * KT; });
    const bool far = fabsf(m * c) > FAR;                     // as in a tile of many
    const float mc = far ? 0.f : m * c, base = far && m != NEG_INF ? m : 0.f;
#pragma unroll 1
    for (int b = 0; b < blocks; ++b) {
      f32x16 s = scores(b);
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        s[r] = __builtin_amdgcn_exp2f(fmaf(s[r] - base, c, -mc));
        l += s[r];
      }
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int rk = 0; rk < 2; ++rk) {
        const lpx8_t p = acc_frag<E>(s, rk), rest = acc_rest<E>(s, rk);
#pragma unroll
        for (int cb = 0; cb < DB; ++cb) {
          lpx8_t v = at.col(2 * TILE + b * 32 * DP * 2, rk, cb);
          if (odd) v = finite<E>(v);
          o[cb] = E::mfma(v, p, o[cb]);
          o[cb] = E::mfma(v, rest, o[cb]);
        }
        __builtin_amdgcn_sched_barrier(0);
      }
    }
    return finish();
  }
  int kt = kt0;
  for (; kt + 1 < whole; kt += 2) {
    tile(kt, std::integral_constant<int, 0>{}, std::false_type{});
    tile(kt + 1, std::integral_constant<int, 1>{}, std::false_type{});
  }
  for (; kt < tiles; kt += 2) {                              // a few tiles more
    tile(kt, std::integral_constant<int, 0>{}, std::true_type{});
    if (kt + 1 < tiles) tile(kt + 1, std::integral_constant<int, 1>{}, std::true_type{});
  }
  finish();
}
// the parts of a row joined: out = sum O_p 2^((m_p - m) c) / sum l_p 2^((m_p - m) c), c = scale log2(e); 16 lanes a row
template <class E>
__global__ __launch_bounds__(256) void packed_attn_fwd_join_kernel(simvg_packed_attn_args a, int parts) {
  const int c = (threadIdx.x & 15) * 8;
  const long n = (long)a.T * a.Hq, rows = (long)a.plan[1] * a.Hq;
  const float2* stat = (const float2*)a.ws;
  const float scale2 = a.scale * LOG2E;
  for (long at = blockIdx.x * 16L + (threadIdx.x >> 4); at < rows; at += gridDim.x * 16L) {
    float m = NEG_INF, l = 0.f;
    for (int p = 0; p < parts; ++p) m = fmaxf(m, stat[p * n + at].x);
    f32x4_t lo = {0.f, 0.f, 0.f, 0.f}, hi = lo;
    for (int p = 0; p < parts; ++p) {
      const float2 s = stat[p * n + at];
      const float f = s.y == 0.f ? 0.f : __builtin_amdgcn_exp2f((s.x - m) * scale2);       // a part without keys has no reference
      l += s.y * f;
      if (c < a.D) {
        const float* src = a.ws + ws_stats(parts, a.T, a.Hq) + (p * n + at) * a.D + c;
        const f32x4_t x = *(const f32x4_t*)src, y = *(const f32x4_t*)(src + 4);
        lo += x * f;
        hi += y * f;
      }
    }
    const long row = at / a.Hq, h = at % a.Hq;
    const float r = 1.f / l;
    if (c < a.D)
      *(u32x4_t*)((unsigned short*)a.o + row * a.o_ts + h * a.o_hs + c) = (u32x4_t){E::pack(lo[0] * r, lo[1] * r), E::pack(lo[2] * r, lo[3] * r),
                                                                                   E::pack(hi[0] * r, hi[1] * r), E::pack(hi[2] * r, hi[3] * r)};
    if (c == 0) a.lse[h * a.lse_hs + row] = m * a.scale + __builtin_logf(l);
  }
}

// ------------------------------------------------------------------------------------------------------------ backward
// For fp16: delta_i = sum_d dO_id O_id, and the largest norms of dO's and V's rows in a tile and head: |dP_ij| and |delta_i| are at most
// |dO_i| |V_j|, so with them dS can be brought to where fp16 has all its bits (`grad_power`).  (bf16: the dQ kernel takes delta along.)
// ws: -delta [Hq][T] | lse log2(e) less P's power [Hq][T] | norms of dO [tiles][Hq] | norms of V [tiles][Hkv] |
// the parts' sums: dQ [parts][T][Hq][D], then dK and dV [parts][2][T][Hkv][D]
__host__ __device__ __forceinline__ long ws_fixed(int T, int nseq, int Hq, int Hkv) {
  return (2L * Hq * T + (long)plan_capacity(T, nseq) * (Hq + Hkv) + 3) / 4 * 4;
}
struct Ws { float *less, *lse2, *ndo, *nv; };
__device__ __forceinline__ Ws ws_of(const simvg_packed_attn_args& a) {
  Ws w;
  w.less = a.ws;
  w.lse2 = a.ws + (long)a.Hq * a.T;
  w.ndo = w.lse2 + (long)a.Hq * a.T;
  w.nv = w.ndo + (long)plan_capacity(a.T, a.nseq) * a.Hq;
  return w;
}
template <class E>
__device__ __forceinline__ float dot8(u32x4_t x, u32x4_t y, float s) {
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    float a0, a1, b0, b1;
    unpack2<E>(x[j], a0, a1);
    unpack2<E>(y[j], b0, b1);
    s = fmaf(a0, b0, s);
    s = fmaf(a1, b1, s);
  }
  return s;
}
template <class E>
__global__ __launch_bounds__(256) void packed_attn_delta_kernel(simvg_packed_attn_args a) {
  __shared__ float most[2][4];
  const int h = blockIdx.x % a.Hq, G = a.Hq / a.Hkv;
  Tile e;
  if (!plan_entry(a, blockIdx.x / a.Hq, e)) return;
  const Ws w = ws_of(a);
  const int lane16 = threadIdx.x & 15, n = min(QT, e.len - e.t * QT);
  const bool with_v = h % G == 0;
  float mdo = 0.f, mv = 0.f;
  // 16 lanes a row, 8 columns each: D <= 128
  for (int r = threadIdx.x >> 4; r < QT; r += 16) {
    const long row = e.first + e.t * QT + min(r, n - 1);
    const int col = lane16 * 8;
    float d = 0.f, sd = 0.f, sv = 0.f;
    if (col < a.D) {
      const u32x4_t x = *(const u32x4_t*)((const unsigned short*)a.d_o + row * a.do_ts + (long)h * a.do_hs + col);
      const u32x4_t y = *(const u32x4_t*)((const unsigned short*)a.o + row * a.o_ts + (long)h * a.o_hs + col);
      d = dot8<E>(x, y, 0.f);
      sd = dot8<E>(x, x, 0.f);
      if (with_v) {
        const u32x4_t z = *(const u32x4_t*)((const unsigned short*)a.v + row * a.v_ts + (long)(h / G) * a.v_hs + col);
        sv = dot8<E>(z, z, 0.f);
      }
    }
#pragma unroll
    for (int o = 8; o > 0; o >>= 1) {
      d += __shfl_xor(d, o, 64);
      sd += __shfl_xor(sd, o, 64);
      sv += __shfl_xor(sv, o, 64);
    }
    if (r < n && lane16 == 0) w.less[(long)h * a.T + row] = -d;
    if (__builtin_isfinite(sd)) mdo = fmaxf(mdo, sd);        // a row that is not finite has no gradient that a scale could save
    if (__builtin_isfinite(sv)) mv = fmaxf(mv, sv);
  }
  mdo = wave_max(mdo);
  mv = wave_max(mv);
  if ((threadIdx.x & 63) == 0) { most[0][threadIdx.x >> 6] = mdo; most[1][threadIdx.x >> 6] = mv; }
  __syncthreads();
  if (threadIdx.x == 0) {
    const long tile = e.base + e.t;
    w.ndo[tile * a.Hq + h] = sqrtf(fmaxf(fmaxf(most[0][0], most[0][1]), fmaxf(most[0][2], most[0][3])));
    if (with_v) w.nv[tile * a.Hkv + h / G] = sqrtf(fmaxf(fmaxf(most[1][0], most[1][1]), fmaxf(most[1][2], most[1][3])));
  }
}
// fp16: what is rounded to 16 bits is P 2^14 (P <= 1: the largest is 2^14) and dS 2^14 2^-x with 2^x at least the sequence's and key
// head's largest |dO_i| |V_j|: at most 2^15.  A probability of 2^-28 then still has all its bits.  Both powers are exact and come out
// of the sums in 32 bits.  bf16 has fp32's exponents: no scale.
constexpr float P_POWER = 14.f;
template <class E>
__device__ __forceinline__ float grad_power(const simvg_packed_attn_args& a, const Tile& e, int hk, float* red) {
  if constexpr (!E::kScaled) return 0.f;
  const Ws w = ws_of(a);
  const int tiles = (e.len + QT - 1) / QT, G = a.Hq / a.Hkv;
  float mdo = 0.f, mv = 0.f;
  for (int i = threadIdx.x; i < tiles * G; i += 256) mdo = fmaxf(mdo, w.ndo[(long)(e.base + i / G) * a.Hq + hk * G + i % G]);
  for (int i = threadIdx.x; i < tiles; i += 256) mv = fmaxf(mv, w.nv[(long)(e.base + i) * a.Hkv + hk]);
  mdo = wave_max(mdo);
  mv = wave_max(mv);
  if ((threadIdx.x & 63) == 0) { red[threadIdx.x >> 6] = mdo; red[4 + (threadIdx.x >> 6)] = mv; }
  __syncthreads();
  mdo = fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3]));
  mv = fmaxf(fmaxf(red[4], red[5]), fmaxf(red[6], red[7]));
  const float most = mdo * mv;
  if (!(most > 0.f)) return 0.f;
  return fminf(fmaxf(-ceilf(__builtin_log2f(most) + 1e-3f), -60.f), 60.f);
}

// dQ: a workgroup's 128 queries against the tiles of their keys, as in the forward pass
template <class E, int DP, bool CAUSAL>
__global__ __launch_bounds__(256, DP == 64 ? 3 : 2) void packed_attn_dq_kernel(simvg_packed_attn_args a, int parts) {
  extern __shared__ __attribute__((aligned(16))) char smem[];
  __shared__ float red[8];
  constexpr int TILE = KT * DP * 2, DB = DP / 32, KS = DP / 16;
  int h, part, id;
  Tile e;
  if (!workgroup<CAUSAL>(a, a.Hq, parts, h, part, id, e)) {
    if (part == 0) fill_tail(a, id, a.dq, a.dq_ts, a.dq_hs, h, nullptr);
    return;
  }
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
  const int hk = h / (a.Hq / a.Hkv);
  const int row = e.t * QT + wave * 32 + (lane & 31);
  const bool valid = row < e.len;
  const long here = e.first + min(row, e.len - 1);
  const unsigned short* qp = (const unsigned short*)a.q + here * a.q_ts + (long)h * a.q_hs;
  const unsigned short* dop = (const unsigned short*)a.d_o + here * a.do_ts + (long)h * a.do_hs;
  const unsigned short* kp = (const unsigned short*)a.k + (long)e.first * a.k_ts + (long)hk * a.k_hs;
  const unsigned short* vp = (const unsigned short*)a.v + (long)e.first * a.v_ts + (long)hk * a.v_hs;
  // the tiles of keys, and this part's of them: [kt0, tiles)
  const int keys = CAUSAL ? min(e.len, (e.t + 1) * QT) : e.len, all_tiles = (keys + KT - 1) / KT;
  // Where a row sees at most 128 keys delta is summed here, P dP over its keys, from the scores and not from the output, whose rounding
  // would show: dS of a row that sees n keys alike is off by its own rounding and by about 1 / sqrt(n) of it for delta's, and the few rows
  // with few keys hold the largest gradients (a sequence of 100 rows: dK 1.62 times as far off as its last rounding alone, and 1.42, what
  // dS's own rounding costs, with this).  Both tiles stay in LDS for the second pass.
  const bool few = all_tiles <= FEW;
  const int kt0 = few ? (part ? all_tiles : 0) : all_tiles * part / parts, tiles = few ? all_tiles : all_tiles * (part + 1) / parts;
  const int wave_first = e.t * QT + wave * 32;
  const int whole = min(tiles, min(CAUSAL ? (e.t * QT + 1) / KT : tiles, e.len / KT));         // of all four waves
  const int wave_whole = min(CAUSAL ? (wave_first + 1) / KT : tiles, e.len / KT);
  const bool live = wave_first < e.len;                      // a wave without a row only brings its pieces of the tiles
  const int wave_tiles = !live ? 0 : CAUSAL ? min(tiles, (wave_first + 32 + KT - 1) / KT) : tiles;
  Stager<DP, 0> gk;
  Stager<DP, 2 * TILE> gv;
  gk.init(kp + (long)kt0 * KT * a.k_ts, a.k_ts, e.len - kt0 * KT, a.D, smem, wave, lane);
  gv.init(vp + (long)kt0 * KT * a.v_ts, a.v_ts, e.len - kt0 * KT, a.D, smem, wave, lane);
  if (kt0 < tiles) {
    gk.template next<0>();
    gv.template next<0>();
  }
  if (few && kt0 + 1 < tiles) {
    gk.template next<1>();
    gv.template next<1>();
  }
  const float power = grad_power<E>(a, e, hk, red), up = __builtin_amdgcn_exp2f(power), shift = E::kScaled ? P_POWER : 0.f;
  lpx8_t qf[KS], dof[KS];
#pragma unroll
  for (int ks = 0; ks < KS; ++ks) { qf[ks] = global_frag(qp, ks, a.D, lane); dof[ks] = global_frag(dop, ks, a.D, lane); }
  Lanes<DP> at;
  at.init(smem, lane);
  const float c = a.scale * LOG2E;
  float lse2 = a.lse[(long)h * a.lse_hs + here] * LOG2E - shift, delta = 0.f;
  if (few) {
    dma_wait<0>();
    wave_barrier_only();
#pragma unroll 1
    for (int half = 2 * kt0; half < 2 * wave_tiles; ++half) {
      const int tile = (half >> 1) * TILE, kb = half & 1, last4 = (CAUSAL ? min(row, e.len - 1) : e.len - 1) - half * 32 - (lane >> 5) * 4;
      f32x16 s = zero16(), dp = zero16();
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) {
        s = E::mfma(at.row(tile, kb, ks), qf[ks], s);
        dp = E::mfma(at.row(2 * TILE + tile, kb, ks), dof[ks], dp);
      }
#pragma unroll
      for (int r = 0; r < 16; ++r)
        if (reg_row(r) <= last4) delta = fmaf(__builtin_amdgcn_exp2f(fmaf(s[r], c, -lse2)), dp[r], delta);
    }
    delta = add_halves(delta) * __builtin_amdgcn_exp2f(-shift);
  } else if constexpr (E::kScaled) {
    delta = -ws_of(a).less[(long)h * a.T + here];
  } else {                                                   // dO's row is here already: delta needs no kernel of its own
    const unsigned short* op = (const unsigned short*)a.o + here * a.o_ts + (long)h * a.o_hs;
#pragma unroll
    for (int ks = 0; ks < KS; ++ks)
      delta = dot8<E>(__builtin_bit_cast(u32x4_t, dof[ks]), __builtin_bit_cast(u32x4_t, global_frag(op, ks, a.D, lane)), delta);
    delta = add_halves(delta);
  }
  if (part == 0 && valid && lane < 32) {                     // for dK and dV
    if (few || !E::kScaled) ws_of(a).less[(long)h * a.T + here] = -delta;
    ws_of(a).lse2[(long)h * a.T + here] = lse2;
  }
  arrived(qf);
  arrived(dof);
  arrived(lse2);
  arrived(delta);
  f32x16 dq[DB];
#pragma unroll
  for (int i = 0; i < DB; ++i) dq[i] = zero16();

  auto tile = [&](int kt, auto which, auto crossed) {
    constexpr int BUF = decltype(which)::value, K0 = BUF * TILE, V0 = (2 + BUF) * TILE;
    constexpr bool MASKED = decltype(crossed)::value;
    dma_wait<0>();
    wave_barrier_only();
    if (kt + 1 < tiles) {
      gk.template next<BUF ^ 1>();
      gv.template next<BUF ^ 1>();
    }
    const bool odd = MASKED && tile_nonfinite<E, DP>(smem + K0), mine = MASKED ? kt < wave_tiles : live;
    const int last = (CAUSAL ? min(row, e.len - 1) : e.len - 1) - kt * KT;
    const int last4 = last - (lane >> 5) * 4;                // against a register's constant
    lpx8_t ds[4];
    f32x16 s, dp;
    auto scores = [&](int kb) {
      s = dp = zero16();
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) {
        s = E::mfma(at.row(K0, kb, ks), qf[ks], s);
        dp = E::mfma(at.row(V0, kb, ks), dof[ks], dp);
      }
    };
    auto gradients = [&](int kb) {
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        const float p = __builtin_amdgcn_exp2f(fmaf(s[r], c, -lse2));
        s[r] = E::kScaled ? p * ((dp[r] - delta) * up) : p * (dp[r] - delta);
      }
      if (MASKED && kt >= wave_whole) {
#pragma unroll
        for (int r = 0; r < 16; ++r)
          if (kb * 32 + reg_row(r) > last4) s[r] = 0.f;
      }
      ds[2 * kb] = acc_frag<E>(s, 0);
      ds[2 * kb + 1] = acc_frag<E>(s, 1);
    };
    auto products = [&](int kb) {
#pragma unroll
      for (int rk = 2 * kb; rk < 2 * kb + 2; ++rk)
#pragma unroll
        for (int cb = 0; cb < DB; ++cb) dq[cb] = E::mfma(at.col(K0, rk, cb), ds[rk], dq[cb]);
    };
    if (mine) { scores(0); gradients(0); }
    if (MASKED) {                                            // both halves' dS before the tile may be cleaned
      if (mine) { scores(1); gradients(1); }
      if (odd) {
        if (mine) add_nonfinite<E, DP, true>(dq, smem + K0, lane, [&](int j) { return j <= last; });
        tile_clean<E, DP>(smem + K0);
      }
      if (mine) { products(0); products(1); }
    } else if (mine) {
      products(0);
      scores(1);
      gradients(1);
      products(1);
    }
  };
  if (few) {                                                 // as in the forward pass
    bool odd = false;
    for (int kt = 0; kt < tiles - kt0; ++kt) odd |= tile_nonfinite<E, DP>(smem + kt * TILE);
    const int last = CAUSAL ? min(row, e.len - 1) : e.len - 1;
    if (odd && live)
      for (int kt = 0; kt < tiles - kt0; ++kt)
        add_nonfinite<E, DP, true>(dq, smem + kt * TILE, lane, [&](int j) { return j <= last - kt * KT; });
#pragma unroll 1
    for (int b = 2 * kt0; b < 2 * wave_tiles; ++b) {
      const int at_b = b * 32 * DP * 2, last4 = last - b * 32 - (lane >> 5) * 4;
      f32x16 s = zero16(), dp = zero16();
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) {
        s = E::mfma(at.row(at_b, 0, ks), qf[ks], s);
        dp = E::mfma(at.row(2 * TILE + at_b, 0, ks), dof[ks], dp);
      }
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        const float p = __builtin_amdgcn_exp2f(fmaf(s[r], c, -lse2));
        s[r] = reg_row(r) > last4 ? 0.f : E::kScaled ? p * ((dp[r] - delta) * up) : p * (dp[r] - delta);
      }
#pragma unroll
      for (int rk = 0; rk < 2; ++rk) {
        const lpx8_t ds = acc_frag<E>(s, rk), rest = acc_rest<E>(s, rk);
#pragma unroll
        for (int cb = 0; cb < DB; ++cb) {
          lpx8_t k = at.col(at_b, rk, cb);
          if (odd) k = finite<E>(k);
          dq[cb] = E::mfma(k, ds, dq[cb]);
          dq[cb] = E::mfma(k, rest, dq[cb]);
        }
      }
    }
  } else {
    int kt = kt0;
    for (; kt + 1 < whole; kt += 2) {
      tile(kt, std::integral_constant<int, 0>{}, std::false_type{});
      tile(kt + 1, std::integral_constant<int, 1>{}, std::false_type{});
    }
    for (; kt < tiles; kt += 2) {
      tile(kt, std::integral_constant<int, 0>{}, std::true_type{});
      if (kt + 1 < tiles) tile(kt + 1, std::integral_constant<int, 1>{}, std::true_type{});
    }
  }
  const auto z = late_args<simvg_packed_attn_args>();
  const float mul = z->scale * __builtin_amdgcn_exp2f(-power - shift);
  if (parts == 1) store_rows<E, DP>(dq, mul, (unsigned short*)z->dq + (long)(e.first + row) * z->dq_ts + (long)h * z->dq_hs, z->D, valid, lane);
  else
    store_sums<DP>(dq, mul, z->ws + ws_fixed(z->T, z->nseq, z->Hq, z->Hkv) + ((part * (long)z->T + e.first + row) * z->Hq + h) * z->D, z->D,
                   valid, lane);
}

// Four stages: with two, asked for one tile ahead, a quarter of the time went to waiting for them (documents' backward pass 1842 us,
// 1630 with the sending left out; 1761 with four stages and the tiles' order below).
constexpr int DKV_STAGES = 4;
// dK, dV: a workgroup's 128 keys against the tiles of the queries that see them, of all heads that share the key head, one after the
// other: the sum over heads stays in the accumulators and needs no atomics.  Where that makes few workgroups (long sequences, few key
// heads) each of them is cut into `parts` of equal length, whose sums in 32 bits go to the workspace and are joined in their order.
template <class E, int DP, bool CAUSAL>
__global__ __launch_bounds__(256, DP == 64 ? 2 : 1) void packed_attn_dkv_kernel(simvg_packed_attn_args a, int parts) {
  extern __shared__ __attribute__((aligned(16))) char smem[];
  __shared__ float red[8];
  constexpr bool PIPED = DP == 128;
  constexpr int TILE = KT * DP * 2, DB = DP / 32, KS = DP / 16, STAGE = 2 * TILE, STAT0 = DKV_STAGES * STAGE, STAT = 2 * KT * 4;
  const int G = a.Hq / a.Hkv;
  int hk, part, id;
  Tile e;
  if (!workgroup<CAUSAL>(a, a.Hkv, parts, hk, part, id, e)) {
    if (part) return;
    fill_tail(a, id, a.dk, a.dk_ts, a.dk_hs, hk, nullptr);
    return fill_tail(a, id, a.dv, a.dv_ts, a.dv_hs, hk, nullptr);
  }
  const int ntile = (e.len + QT - 1) / QT;
  if (CAUSAL) e.t = ntile - 1 - e.t;                         // the plan's order is by cost: the first keys are seen by the most queries
  const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63;
  const int key = e.t * QT + wave * 32 + (lane & 31);        // the lane's key
  const bool valid = key < e.len;
  const long here = e.first + min(key, e.len - 1);
  const unsigned short* kp = (const unsigned short*)a.k + here * a.k_ts + (long)hk * a.k_hs;
  const unsigned short* vp = (const unsigned short*)a.v + here * a.v_ts + (long)hk * a.v_hs;
  // Step i of the G heads' tiles: the sequence's tile of queries all - 1 - i / G, head hk G + i % G; this part's are [s0, s1).  From the
  // last tile backwards, all heads of a tile: the workgroups of a sequence's keys, which all see its end, read the same rows at the same
  // time and find them in the L2.
  const int first = CAUSAL ? e.t * QT / KT : 0, all = (e.len + KT - 1) / KT, tiles = all - first;
  const int wave_first = e.t * QT + wave * 32, s0 = (int)((long)G * tiles * part / parts), s1 = (int)((long)G * tiles * (part + 1) / parts);
  const int steps = s1 - s0, g0 = s0 % G, t0 = all - 1 - s0 / G;
  const long row_first = e.first + (long)t0 * KT;
  Stager<DP, 0> gq;
  Stager<DP, TILE> gd;
  gq.init((const unsigned short*)a.q + row_first * a.q_ts + (long)(hk * G + g0) * a.q_hs, a.q_ts, e.len - t0 * KT, a.D, smem, wave, lane);
  gd.init((const unsigned short*)a.d_o + row_first * a.do_ts + (long)(hk * G + g0) * a.do_hs, a.do_ts, e.len - t0 * KT, a.D, smem, wave, lane);
  // from the last head of a tile to the first of the one before (`next` has gone one tile on)
  const long q_head = a.q_hs * 2 - (long)gq.step, d_head = a.do_hs * 2 - (long)gd.step;
  const long q_back = -(long)gq.step - G * (a.q_hs * 2), d_back = -(long)gd.step - G * (a.do_hs * 2);
  // the rows' lse and delta, from two waves
  unsigned long stat_at = (unsigned long)((wave ? ws_of(a).less : ws_of(a).lse2) + (long)(hk * G + g0) * a.T + row_first);
  const long stat_head = a.T * 4L, stat_back = -G * (a.T * 4L) - KT * 4L;
  const unsigned stat_lds = lds_addr(smem) + STAT0 + wave * KT * 4;
  int send_g = g0, send_to = 0;                              // of the next step that is sent for: its head and its place
  auto send = [&] {
    gq.place = gd.place = send_to * STAGE;
    if (wave < 2) {
      const u32x4_t b = {(unsigned)stat_at, (unsigned)(stat_at >> 32) & 0xffffu, DMA_NOTHING - 1, 0x00020000u};
      dma4(b, stat_lds + send_to * STAT, lane < gq.left ? lane * 4u : DMA_NOTHING);
    }
    gq.template next<0>();
    gd.template next<0>();
    gq.base += q_head;
    gd.base += d_head;
    gq.left += KT;
    gd.left += KT;
    stat_at += stat_head;
    if (++send_g == G) {                                     // the tile before
      send_g = 0;
      gq.base += q_back;
      gd.base += d_back;
      gq.left += KT;
      gd.left += KT;
      stat_at += stat_back;
    }
    if (++send_to == DKV_STAGES) send_to = 0;
  };
  for (int i = 0; i < DKV_STAGES - 1 && i < steps; ++i) send();
  const float power = grad_power<E>(a, e, hk, red), up = __builtin_amdgcn_exp2f(power), shift = E::kScaled ? P_POWER : 0.f;
  lpx8_t kf[KS], vf[KS];
#pragma unroll
  for (int ks = 0; ks < KS; ++ks) { kf[ks] = global_frag(kp, ks, a.D, lane); vf[ks] = global_frag(vp, ks, a.D, lane); }
  arrived(kf);
  arrived(vf);
  Lanes<DP> at;
  at.init(smem, lane);
  const float c = a.scale * LOG2E;
  f32x16 dk[DB], dv[DB];
#pragma unroll
  for (int i = 0; i < DB; ++i) { dk[i] = zero16(); dv[i] = zero16(); }

  int row0 = t0 * KT, g_now = g0, now = 0;                   // of the step that is multiplied: its first row, head and place
  // A step's tile becomes visible: every wave's pieces are in LDS, nobody reads the one before any more, and to its place goes the one
  // DKV_STAGES further on
  auto arrive = [&](int i, int row0, int place) {
    constexpr int PIECES = 2 * Stager<DP, 0>::PIECES, AHEAD = DKV_STAGES - 2;
    if (i + AHEAD >= steps) dma_wait<0>();
    else if (wave < 2) dma_wait<AHEAD * (PIECES + 1)>();
    else dma_wait<AHEAD * PIECES>();
    wave_barrier_only();
    if (i + DKV_STAGES - 1 < steps) send();
    // Rows that are not finite lose nothing by being cleaned before the scores: their lse (of q) or delta (of dO) is not finite either,
    // and carries that to P and dS of every key they see
    if (CAUSAL && row0 < e.t * QT + QT - 1) {
      char *lq = smem + place * STAGE, *ld = lq + TILE;
      const bool mine = row0 + KT > wave_first;
      const int from = key - row0;
      const bool odd_q = tile_nonfinite<E, DP>(lq), odd_d = tile_nonfinite<E, DP>(ld);
      if (odd_d) {
        if (mine) add_nonfinite<E, DP, false>(dv, ld, lane, [&](int j) { return j >= from; });
        tile_clean<E, DP>(ld);
      }
      if (odd_q) {
        if (mine) add_nonfinite<E, DP, true>(dk, lq, lane, [&](int j) { return j >= from; });
        tile_clean<E, DP>(lq);
      }
    }
  };
  // A block of 32 rows takes A: S and dP; B: P and dS from them, rounded; C: their products into dV and dK, each in N groups of two MFMAs.
  // Heads of 128 leave one wave to a SIMD (its accumulators and its keys' operands are 192 registers): nobody else covers its waits or
  // its vector work, so a tile's two blocks go through in four phases, A0, A1 beside B0, C0 beside B1, C1, and each group asks for the
  // operands of its like in the next phase, the last one for the next step's first rows.  Smaller heads have two waves to a SIMD,
  // which cover each other, and no room for the second block's registers: one block after the other.
  constexpr int N = DP / 16, PER = 16 / N;
  lpx8_t x[N], y[N];                                         // operands of q and dO, by rows (A) or columns (C)
  auto rows = [&](int g, int stage, int qb) {
    x[g] = at.row(stage, qb, g);
    y[g] = at.row(stage + TILE, qb, g);
  };
  auto cols = [&](int g, int stage, int qb) {
    x[g] = at.col(stage, qb * 2 + g / DB, g % DB);
    y[g] = at.col(stage + TILE, qb * 2 + g / DB, g % DB);
  };
  auto step = [&](int i) {
    const int stage = now * STAGE;
    const float* stat = (const float*)(smem + STAT0 + now * STAT) + (lane >> 5) * 4;
    // (without a mask row0 + KT is always above 0: a branch all the same, or hipcc keeps the operands of two steps at once and spills)
    const bool mine = wave_first < e.len && row0 + KT > (CAUSAL ? wave_first : 0), whole = row0 + KT <= e.len && (!CAUSAL || row0 >= wave_first + 31);
    u32x4_t p[2], ds[2];
    auto products = [&](int g) {
      const int rk = g / DB, cb = g % DB;
      dv[cb] = E::mfma(y[g], __builtin_bit_cast(lpx8_t, p[rk]), dv[cb]);
      dk[cb] = E::mfma(x[g], __builtin_bit_cast(lpx8_t, ds[rk]), dk[cb]);
    };
    if (mine) {
      f32x16 s[2], dp[2];
      f32x4_t ls[2][4];
      u32x4_t np[2], nds[2];
      auto start = [&](int qb) {                             // dP's products start from -delta
        s[qb] = zero16();
#pragma unroll
        for (int g = 0; g < 4; ++g) {
          ls[qb][g] = *(const f32x4_t*)(stat + qb * 32 + g * 8);
          const f32x4_t d = *(const f32x4_t*)(stat + KT + qb * 32 + g * 8);
#pragma unroll
          for (int r = 0; r < 4; ++r) dp[qb][4 * g + r] = d[r];
        }
      };
      auto scores = [&](int g, int qb) {
        s[qb] = E::mfma(x[g], kf[g], s[qb]);
        dp[qb] = E::mfma(y[g], vf[g], dp[qb]);
      };
      auto gradients = [&](int g, int qb) {                  // registers PER g ..
#pragma unroll
        for (int r = PER * g; r < PER * (g + 1); r += 2) {
          const float p0 = __builtin_amdgcn_exp2f(fmaf(s[qb][r], c, -ls[qb][r / 4][r % 4]));
          const float p1 = __builtin_amdgcn_exp2f(fmaf(s[qb][r + 1], c, -ls[qb][r / 4][r % 4 + 1]));
          np[r / 8][r % 8 / 2] = E::pack(p0, p1);
          nds[r / 8][r % 8 / 2] = E::kScaled ? E::pack(p0 * (dp[qb][r] * up), p1 * (dp[qb][r + 1] * up))
                                             : E::pack(p0 * dp[qb][r], p1 * dp[qb][r + 1]);
        }
      };
      auto rounded = [&](int qb) {
        if (!whole) {                                        // bits, not products: what is masked may be NaN
          stay_a_branch();
          // the rows of the tile that see the lane's key, up to the sequence's end (rows past it are zeros; times a key of -inf, NaN)
          const int from4 = (CAUSAL ? key - row0 : 0) - (lane >> 5) * 4, rows4 = e.len - row0 - (lane >> 5) * 4;
#pragma unroll
          for (int r = 0; r < 16; r += 2) {
            const int row = qb * 32 + reg_row(r);
            const unsigned m = (row >= from4 && row < rows4 ? 0xffffu : 0u) | (row + 1 >= from4 && row + 1 < rows4 ? 0xffff0000u : 0u);
            np[r / 8][r % 8 / 2] &= m;
            nds[r / 8][r % 8 / 2] &= m;
          }
        }
        p[0] = np[0]; p[1] = np[1]; ds[0] = nds[0]; ds[1] = nds[1];
      };
      if (tiles <= FEW) {                                    // what the rounding of P and dS will take off, first
        stay_a_branch();
#pragma unroll 1
        for (int qb = 0; qb < 2; ++qb) {
#pragma unroll
          for (int g = 0; g < N; ++g) rows(g, stage, qb);
          start(0);
#pragma unroll
          for (int g = 0; g < N; ++g) scores(g, 0);
#pragma unroll
          for (int g = 0; g < N; ++g) cols(g, stage, qb);
#pragma unroll
          for (int r = 0; r < 16; r += 2) {
            float p0 = __builtin_amdgcn_exp2f(fmaf(s[0][r], c, -ls[0][r / 4][r % 4])), p1 = __builtin_amdgcn_exp2f(fmaf(s[0][r + 1], c, -ls[0][r / 4][r % 4 + 1]));
            float d0 = E::kScaled ? p0 * (dp[0][r] * up) : p0 * dp[0][r], d1 = E::kScaled ? p1 * (dp[0][r + 1] * up) : p1 * dp[0][r + 1], a0, a1;
            unpack2<E>(E::pack(p0, p1), a0, a1);
            np[r / 8][r % 8 / 2] = E::pack(p0 - a0, p1 - a1);
            unpack2<E>(E::pack(d0, d1), a0, a1);
            nds[r / 8][r % 8 / 2] = E::pack(d0 - a0, d1 - a1);
          }
          rounded(qb);
#pragma unroll
          for (int g = 0; g < N; ++g) products(g);
          stat += 32;
        }
        stat -= 64;
        if constexpr (PIPED) {
#pragma unroll
          for (int g = 0; g < N; ++g) rows(g, stage, 0);
        }
      }
      if constexpr (PIPED) {
        start(0);
#pragma unroll
        for (int g = 0; g < N; ++g) {
          scores(g, 0);
          rows(g, stage, 1);
          __builtin_amdgcn_sched_barrier(0);
        }
        start(1);
#pragma unroll
        for (int g = 0; g < N; ++g) {
          scores(g, 1);
          cols(g, stage, 0);
          gradients(g, 0);
          __builtin_amdgcn_sched_barrier(0);
        }
        rounded(0);
#pragma unroll
        for (int g = 0; g < N; ++g) {
          products(g);
          cols(g, stage, 1);
          gradients(g, 1);
          __builtin_amdgcn_sched_barrier(0);
        }
        rounded(1);
      } else {
#pragma unroll
        for (int qb = 0; qb < 2; ++qb) {
#pragma unroll
          for (int g = 0; g < N; ++g) rows(g, stage, qb);
          start(0);
#pragma unroll
          for (int g = 0; g < N; ++g) scores(g, 0);
#pragma unroll
          for (int g = 0; g < N; ++g) cols(g, stage, qb);
#pragma unroll
          for (int g = 0; g < N; ++g) gradients(g, 0);
          rounded(qb);
#pragma unroll
          for (int g = 0; g < N; ++g) products(g);
          stat += 32;
        }
      }
    }
    if (++g_now == G) {
      g_now = 0;
      row0 -= KT;
    }
    if (++now == DKV_STAGES) now = 0;
    if (i + 1 < steps) arrive(i + 1, row0, now);
    if constexpr (PIPED) {
      if (mine) {
#pragma unroll
        for (int g = 0; g < N; ++g) {
          products(g);
          rows(g, now * STAGE, 0);
          __builtin_amdgcn_sched_barrier(0);
        }
      } else {
#pragma unroll
        for (int g = 0; g < N; ++g) rows(g, now * STAGE, 0);
      }
    }
  };
  if (steps > 0) {
    arrive(0, row0, 0);
    if constexpr (PIPED) {
#pragma unroll
      for (int g = 0; g < N; ++g) rows(g, 0, 0);
    }
  }
  for (int i = 0; i < steps; ++i) step(i);
  const auto z = late_args<simvg_packed_attn_args>();
  const float mk = z->scale * __builtin_amdgcn_exp2f(-power - shift), mv = __builtin_amdgcn_exp2f(-shift);
  if (parts == 1) {
    store_rows<E, DP>(dv, mv, (unsigned short*)z->dv + (long)(e.first + key) * z->dv_ts + (long)hk * z->dv_hs, z->D, valid, lane);
    store_rows<E, DP>(dk, mk, (unsigned short*)z->dk + (long)(e.first + key) * z->dk_ts + (long)hk * z->dk_hs, z->D, valid, lane);
  } else {
    const long n = (long)z->T * z->Hkv * z->D;
    float* out = z->ws + ws_fixed(z->T, z->nseq, z->Hq, z->Hkv) + 2 * part * n + ((long)(e.first + key) * z->Hkv + hk) * z->D;
    store_sums<DP>(dk, mk, out, z->D, valid, lane);
    store_sums<DP>(dv, mv, out + n, z->D, valid, lane);
  }
}
// the parts of a gradient, joined: sums [part][T][H][D], `stride` apart, one thread for 8 columns of a row (rows behind the last
// sequence were done by the parts' kernel)
template <class E>
__global__ __launch_bounds__(256) void packed_attn_join_kernel(const int* plan, const float* sums, long stride, int parts, int H, int D,
                                                               unsigned short* out, long ts, long hs) {
  const int per = D / 8;
  for (long i = blockIdx.x * 256L + threadIdx.x; i < (long)plan[1] * H * per; i += gridDim.x * 256L) {
    const int c = (int)(i % per) * 8, h = (int)(i / per % H);
    const long row = i / per / H;
    const float* src = sums + (row * H + h) * D + c;
    f32x4_t lo = {0.f, 0.f, 0.f, 0.f}, hi = lo;
#pragma unroll 4
    for (int p = 0; p < parts; ++p) {
      lo += *(const f32x4_t*)(src + p * stride);
      hi += *(const f32x4_t*)(src + p * stride + 4);
    }
    *(u32x4_t*)(out + row * ts + h * hs + c) = (u32x4_t){E::pack(lo[0], lo[1]), E::pack(lo[2], lo[3]), E::pack(hi[0], hi[1]), E::pack(hi[2], hi[3])};
  }
}

// ---------------------------------------------------------------------------------------------------------------- host
// rows in 16-byte chunks; a tile's offsets fit 31 bits
bool rows16(const void* p, long ts, long hs) { return p && (uintptr_t)p % 16 == 0 && ts % 8 == 0 && hs % 8 == 0; }
bool in_reach(long ts) { return ts >= 0 && ts < 1L << 24; }

// How many parts a workgroup's work is cut into where a launch has few workgroups: so many that there are two for each of the 256
// compute units, four under `causal`, where they are of very different length, and each of at least eight tiles on average.  (One
// sequence of 8192 rows, 4 heads of 128 on 1, causal: forward 152 us uncut and 99 cut, backward 1091 and 335; 16384 rows, 16 heads on 2:
// backward 5.14 and 3.79 ms; 2048 rows, 8 heads of 128, no mask: 41 and 40 us, 124 and 118; 8192 rows, 4 heads, no mask, are 264 equal
// workgroups and stay uncut: three parts took 519 us where one took 501.)
int parts_of(long groups, long tiles, int causal) {
  return (int)std::max(1L, std::min(std::min((causal ? 1024 : 512) / groups, tiles / (causal ? 2 : 1) / 8), 32L));
}
// ... of a tile of queries, over its keys (forward pass and dQ)
int row_parts(int T, int nseq, int Hq, int causal) {
  return parts_of((long)plan_capacity(T, nseq) * Hq, (long)T / std::max(nseq, 1) / KT, causal);
}
// ... of a tile of keys, over the queries and heads that see it (dK, dV)
int key_parts(int T, int nseq, int Hq, int Hkv, int causal) {
  return parts_of((long)plan_capacity(T, nseq) * Hkv, (long)T / std::max(nseq, 1) / KT * (Hq / Hkv), causal);
}
// Whether a forward pass looks for workgroups with few tiles (FEW): where sequences are of 128 rows or less on average, or few rows at
// all.  The path for them takes registers from the others' (64 x 411 rows, 12 heads of 64: 65.0 us without and 66.6 with it; one sequence of
// 16384 rows, 16 heads of 128: 1013 and 1022); dQ, dK and dV have it at no cost.
bool short_rows(int T, int nseq) { return T <= (long)QT * std::max(nseq, 16); }
// the parts' sums of the backward pass: dQ's and then dK's and dV's use the same room
long bwd_sums(int T, int nseq, int Hq, int Hkv, int D, int causal) {
  const int r = row_parts(T, nseq, Hq, causal), k = key_parts(T, nseq, Hq, Hkv, causal);
  return std::max(r > 1 ? (long)r * T * Hq * D : 0L, k > 1 ? 2L * k * T * Hkv * D : 0L);
}
long fwd_sums(int T, int nseq, int Hq, int D, int causal) {
  const int r = row_parts(T, nseq, Hq, causal);
  return r > 1 ? ws_stats(r, T, Hq) + (long)r * T * Hq * D : 0L;
}
int attn_check(const simvg_packed_attn_args* a, bool bwd) {
  SIMVG_CHECK_ARG(a->dtype == SEQ_F16 || a->dtype == SEQ_BF16, "packed_attn: dtype must be fp16 or bf16");
  SIMVG_CHECK_ARG(a->T >= 0 && a->nseq >= 0 && a->nseq <= 1 << 24, "packed_attn: T and nseq must not be negative");
  SIMVG_CHECK_ARG(a->Hkv >= 1 && a->Hq >= a->Hkv && a->Hq % a->Hkv == 0, "packed_attn: the heads of q must be a multiple of those of k and v");
  SIMVG_CHECK_ARG(a->D >= 8 && a->D <= 128 && a->D % 8 == 0, "packed_attn: the head size must be a multiple of 8 and at most 128");
  SIMVG_CHECK_ARG(a->scale > 0.f && a->scale < __builtin_huge_valf(), "packed_attn: scale must be positive and finite");
  SIMVG_CHECK_ARG((long)plan_capacity(a->T, a->nseq) * a->Hq < 1L << 24, "packed_attn: too many tiles for one launch");
  if (a->T == 0) return SIMVG_OK;
  SIMVG_CHECK_ARG(a->plan && a->lse, "packed_attn: null pointer");
  SIMVG_CHECK_ARG((uintptr_t)a->plan % 4 == 0, "packed_attn: misaligned plan");
  SIMVG_CHECK_ARG(rows16(a->q, a->q_ts, a->q_hs) && rows16(a->k, a->k_ts, a->k_hs) && rows16(a->v, a->v_ts, a->v_hs) &&
                  rows16(a->o, a->o_ts, a->o_hs), "packed_attn: rows of q, k, v and out must start at multiples of 16 bytes");
  SIMVG_CHECK_ARG(in_reach(a->q_ts) && in_reach(a->k_ts) && in_reach(a->v_ts) && (!bwd || in_reach(a->do_ts)),
                  "packed_attn: token strides must be below 2^24 elements");
  SIMVG_CHECK_ARG(bwd || fwd_sums(a->T, a->nseq, a->Hq, a->D, a->causal) == 0 || (a->ws && (uintptr_t)a->ws % 16 == 0),
                  "packed_attn: this forward pass needs a workspace, aligned to 16 bytes");
  if (bwd) {
    SIMVG_CHECK_ARG(rows16(a->d_o, a->do_ts, a->do_hs) && rows16(a->dq, a->dq_ts, a->dq_hs) && rows16(a->dk, a->dk_ts, a->dk_hs) &&
                    rows16(a->dv, a->dv_ts, a->dv_hs), "packed_attn: rows of the gradients must start at multiples of 16 bytes");
    SIMVG_CHECK_ARG(a->ws && (uintptr_t)a->ws % 16 == 0, "packed_attn: the backward pass needs a workspace, aligned to 16 bytes");
  }
  // the operands are read by many workgroups until the last one is done: results have memory of their own
  const int T = a->T, Hq = a->Hq, Hkv = a->Hkv;
  const Rows in[] = {{a->q, a->q_ts, a->q_hs, T, Hq}, {a->k, a->k_ts, a->k_hs, T, Hkv}, {a->v, a->v_ts, a->v_hs, T, Hkv},
                     {a->o, a->o_ts, a->o_hs, T, Hq}, {a->d_o, a->do_ts, a->do_hs, T, Hq}};
  const Rows out[] = {{a->dq, a->dq_ts, a->dq_hs, T, Hq}, {a->dk, a->dk_ts, a->dk_hs, T, Hkv}, {a->dv, a->dv_ts, a->dv_hs, T, Hkv}};
  const auto apart = [&](const Rows& x, const Rows& y) { return rows_apart(x, y, T, a->D, 2); };
  for (int i = 0; i < 5; ++i)
    for (int j = 0; j < 3; ++j)
      SIMVG_CHECK_ARG(bwd ? apart(in[i], out[j]) : i || apart(in[j], in[3]), "packed_attn: a result overlaps an operand or another result");
  SIMVG_CHECK_ARG(!bwd || (apart(out[0], out[1]) && apart(out[0], out[2]) && apart(out[1], out[2])),
                  "packed_attn: a result overlaps an operand or another result");
  return SIMVG_OK;
}

template <class E>
void join(const simvg_packed_attn_args& a, const float* sums, long stride, int parts, int H, void* out, long ts, long hs, hipStream_t s) {
  const long work = (long)a.T * H * a.D / 8;
  hipLaunchKernelGGL((packed_attn_join_kernel<E>), dim3((int)min((work + 255) / 256, 4096L)), dim3(256), 0, s, a.plan, sums, stride, parts, H, a.D,
                     (unsigned short*)out, ts, hs);
}

constexpr int dkv_lds(int DP) { return DKV_STAGES * (2 * KT * DP * 2 + 2 * KT * 4); }

template <class E, int DP, bool CAUSAL>
void attn_launch(const simvg_packed_attn_args& a, bool bwd, hipStream_t s) {
  static std::atomic<unsigned long> done[4] = {{0}, {0}, {0}, {0}};               // the tiles of 128 columns and the kernels' own few bytes pass 64 KiB
  if (!bwd) allow_lds((const void*)packed_attn_fwd_kernel<E, DP, CAUSAL, false>, 4 * KT * DP * 2, done[0]);
  else {
    allow_lds((const void*)packed_attn_dq_kernel<E, DP, CAUSAL>, 4 * KT * DP * 2, done[1]);
    allow_lds((const void*)packed_attn_dkv_kernel<E, DP, CAUSAL>, dkv_lds(DP), done[2]);
  }
  const int entries = plan_capacity(a.T, a.nseq), lds = 4 * KT * DP * 2, rparts = row_parts(a.T, a.nseq, a.Hq, a.causal);
  if (!bwd) {
    if (short_rows(a.T, a.nseq)) {
      allow_lds((const void*)packed_attn_fwd_kernel<E, DP, CAUSAL, true>, lds, done[3]);
      hipLaunchKernelGGL((packed_attn_fwd_kernel<E, DP, CAUSAL, true>), dim3(entries * a.Hq * rparts), dim3(256), lds, s, a, rparts);
    } else {
      hipLaunchKernelGGL((packed_attn_fwd_kernel<E, DP, CAUSAL, false>), dim3(entries * a.Hq * rparts), dim3(256), lds, s, a, rparts);
    }
    if (rparts > 1)
      hipLaunchKernelGGL((packed_attn_fwd_join_kernel<E>), dim3((int)min(((long)a.T * a.Hq + 15) / 16, 8192L)), dim3(256), 0, s, a, rparts);
    return;
  }
  float* sums = a.ws + ws_fixed(a.T, a.nseq, a.Hq, a.Hkv);
  if constexpr (E::kScaled) hipLaunchKernelGGL((packed_attn_delta_kernel<E>), dim3(entries * a.Hq), dim3(256), 0, s, a);
  hipLaunchKernelGGL((packed_attn_dq_kernel<E, DP, CAUSAL>), dim3(entries * a.Hq * rparts), dim3(256), lds, s, a, rparts);
  if (rparts > 1) join<E>(a, sums, (long)a.T * a.Hq * a.D, rparts, a.Hq, a.dq, a.dq_ts, a.dq_hs, s);
  const int kparts = key_parts(a.T, a.nseq, a.Hq, a.Hkv, a.causal);
  hipLaunchKernelGGL((packed_attn_dkv_kernel<E, DP, CAUSAL>), dim3(entries * a.Hkv * kparts), dim3(256), dkv_lds(DP), s, a, kparts);
  if (kparts > 1) {
    const long n = (long)a.T * a.Hkv * a.D;
    join<E>(a, sums, 2 * n, kparts, a.Hkv, a.dk, a.dk_ts, a.dk_hs, s);
    join<E>(a, sums + n, 2 * n, kparts, a.Hkv, a.dv, a.dv_ts, a.dv_hs, s);
  }
}
template <class E>
void attn_dispatch(const simvg_packed_attn_args& a, bool bwd, hipStream_t s) {
  if (a.D <= 64) a.causal ? attn_launch<E, 64, true>(a, bwd, s) : attn_launch<E, 64, false>(a, bwd, s);
  else a.causal ? attn_launch<E, 128, true>(a, bwd, s) : attn_launch<E, 128, false>(a, bwd, s);
}
int attn_run(const simvg_packed_attn_args* args, bool bwd, hipStream_t s) {
  SIMVG_CHECK_ARG(args, "packed_attn: null argument block");
  simvg_packed_attn_args a = *args;
  // the token stride of one token and the head stride of one head are never walked: whatever a view has there is no reason to refuse it
  if (a.T == 1) a.q_ts = a.k_ts = a.v_ts = a.o_ts = a.do_ts = a.dq_ts = a.dk_ts = a.dv_ts = 0;
  if (a.Hq == 1) a.q_hs = a.o_hs = a.do_hs = a.dq_hs = 0;
  if (a.Hkv == 1) a.k_hs = a.v_hs = a.dk_hs = a.dv_hs = 0;
  const int rc = attn_check(&a, bwd);
  if (rc || a.T == 0) return rc;
  if (a.dtype == SEQ_F16) attn_dispatch<F16>(a, bwd, s);
  else attn_dispatch<BF16>(a, bwd, s);
  SIMVG_LAUNCH_CHECK();
  return SIMVG_OK;
}
}  // namespace

extern "C" long simvg_packed_plan_ints(int T, int nseq) {
  return T < 0 || nseq < 0 ? 0 : PLAN_HEAD + 8L * plan_capacity(T, nseq) + nseq + 1;
}
extern "C" int simvg_packed_plan(const int* cu_seqlens, int nseq, int T, int* plan, hipStream_t stream) {
  SIMVG_CHECK_ARG(T >= 0 && nseq >= 0 && nseq <= 1 << 24, "packed_plan: T and nseq must not be negative");
  SIMVG_CHECK_ARG(cu_seqlens && plan, "packed_plan: null pointer");
  hipLaunchKernelGGL(packed_plan_kernel, dim3(1), dim3(1024), 0, stream, cu_seqlens, nseq, T, plan);
  SIMVG_LAUNCH_CHECK();
  return SIMVG_OK;
}
extern "C" long simvg_packed_attn_ws_floats(int T, int nseq, int Hq, int Hkv, int D, int causal, int backward) {
  if (T <= 0 || nseq < 0 || Hkv < 1 || Hq < Hkv || D < 0) return 0;
  return backward ? ws_fixed(T, nseq, Hq, Hkv) + bwd_sums(T, nseq, Hq, Hkv, D, causal != 0) : fwd_sums(T, nseq, Hq, D, causal != 0);
}
extern "C" int simvg_packed_attn_fwd(const simvg_packed_attn_args* args, hipStream_t stream) { return attn_run(args, false, stream); }
extern "C" int simvg_packed_attn_bwd(const simvg_packed_attn_args* args, hipStream_t stream) { return attn_run(args, true, stream); }
