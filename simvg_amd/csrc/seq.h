// Shared by the sequence operators (rope.hip, packed_attn.hip, vocab_ce.hip): element types chosen per call, 32x32 MFMA fragments.
// The encoder's kernels are built for ONE 16-bit format (common.h, "lp"); these take either of the two as an argument, because what
// they read comes from a caller's language model and not from this library's encoder.  Rounding to 16 bits is round-to-nearest-even
// and does not saturate: an overflow is an inf, as in torch, and a loss scaler can see it.
#pragma once
#include <climits>

#include <algorithm>
#include <atomic>
#include <cstdlib>
#include <numeric>

#include "common.h"

// element types of the `dtype` arguments (include/simvg_hip.h: SIMVG_F32, SIMVG_F16, SIMVG_BF16)
enum { SEQ_F32 = 0, SEQ_F16 = 1, SEQ_BF16 = 2 };

namespace seq {

typedef __attribute__((ext_vector_type(16))) float f32x16;
typedef _Float16 half8 __attribute__((ext_vector_type(8)));
typedef _Float16 half2v __attribute__((ext_vector_type(2)));
typedef __bf16 bf8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf2 __attribute__((ext_vector_type(2)));
typedef __attribute__((ext_vector_type(2))) float f32x2;

struct F16 {
  static constexpr bool kScaled = true;                 // 5 exponent bits: what a backward pass rounds is brought into range first
  static constexpr int kInf = 0x7c00;
  static __device__ __forceinline__ float to_f32(unsigned short v) { return (float)__builtin_bit_cast(_Float16, v); }
  static __device__ __forceinline__ unsigned pack(float a, float b) {
    return __builtin_bit_cast(unsigned, __builtin_convertvector((f32x2){a, b}, half2v));
  }
  static __device__ __forceinline__ f32x16 mfma(lpx8_t a, lpx8_t b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(half8, a), __builtin_bit_cast(half8, b), c, 0, 0, 0);
  }
};
struct BF16 {
  static constexpr bool kScaled = false;
  static constexpr int kInf = 0x7f80;
  static __device__ __forceinline__ float to_f32(unsigned short v) { return __uint_as_float((unsigned)v << 16); }
  static __device__ __forceinline__ unsigned pack(float a, float b) {
    return __builtin_bit_cast(unsigned, __builtin_convertvector((f32x2){a, b}, bf2));
  }
  static __device__ __forceinline__ f32x16 mfma(lpx8_t a, lpx8_t b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf8, a), __builtin_bit_cast(bf8, b), c, 0, 0, 0);
  }
};

template <class E>
__device__ __forceinline__ void unpack2(unsigned u, float& lo, float& hi) {
  lo = E::to_f32((unsigned short)(u & 0xffffu));
  hi = E::to_f32((unsigned short)(u >> 16));
}

// ---- HBM -> LDS without registers (LDS-DMA), 16 bytes a lane: LDS bytes [lds, lds + 1024) of the wave get what its lanes' offsets
// name, in the lanes' order; an offset at or past `bytes` of the buffer reads zeros.  The instruction is written in asm because hipcc
// puts `s_waitcnt vmcnt(0)` in front of every LDS read that may alias a DMA it knows of, which would wait for the tile that has just
// been asked for; it has no register output, so nothing can be taken before it has arrived.  The caller counts: `dma_wait<N>` leaves
// the N youngest in flight, and a barrier makes the others' pieces visible.
// (LDS byte `lds` + PLUS: one scalar register serves all pieces of a wave.  A buffer: address, 48 bits | bytes | 0x00020000.)
template <int PLUS>
__device__ __forceinline__ void dma16_at(u32x4_t buffer, unsigned lds, unsigned offset) {
  asm volatile("s_add_u32 m0, %0, %3\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds" ::"s"(lds), "v"(offset), "s"(buffer), "n"(PLUS)
               : "memory", "m0", "scc");
}
// 4 bytes a lane: LDS bytes [lds, lds + 256)
__device__ __forceinline__ void dma4(u32x4_t buffer, unsigned lds, unsigned offset) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dword %1, %2, 0 offen lds" ::"s"(lds), "v"(offset), "s"(buffer) : "memory", "m0");
}
// The kernel's arguments read again from the kernarg segment: what only the end of a kernel needs does not sit in scalar registers
// through its loop (hipcc loads all arguments at the start and then spills them)
template <class A>
__device__ __forceinline__ const __attribute__((address_space(4))) A* late_args() {
  auto p = (const __attribute__((address_space(4))) A*)__builtin_amdgcn_kernarg_segment_ptr();
  asm volatile("" : "+s"(p));
  return p;
}
constexpr unsigned DMA_NOTHING = 0x80000000u;          // an offset past every buffer (which is at most one byte shorter): zeros
template <int N>
__device__ __forceinline__ void dma_wait() { asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory"); }
// a barrier that does not drain this wave's DMA (what `__syncthreads` would wait for is the caller's business here)
__device__ __forceinline__ void wave_barrier_only() { asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory"); }

// ---- where an operand [T][H][D] lies, for the host's checks that results have memory of their own
struct Rows {
  const void* p; long ts, hs; int H;
  Rows(const void* p, long ts, long hs, int T, int H) : p(p), ts(T > 1 ? ts : 0), hs(H > 1 ? hs : 0), H(H) {}       // (strides that are never walked)
  bool same(const Rows& o) const { return p == o.p && ts == o.ts && hs == o.hs && H == o.H; }
};
// Whether two operands of the same T, D and size of a value have no value in common.  Slices of one buffer lie in each other's range and
// are told apart by their rows: the distance of two heads' rows is d + i ts for tokens i apart.  Exact where the token strides are the
// same; where they are not, rows that could meet in an endless tensor (a multiple of the strides' common divisor apart) count as meeting.
inline bool rows_apart(const Rows& a, const Rows& b, int T, int D, int size) {
  if (T <= 0 || !a.p || !b.p) return true;
  const long start = (intptr_t)b.p - (intptr_t)a.p, row = (long)D * size;
  const auto low = [&](const Rows& r) { return std::min(0L, (T - 1) * r.ts * size) + std::min(0L, (r.H - 1) * r.hs * size); };
  const auto high = [&](const Rows& r) { return std::max(0L, (T - 1) * r.ts * size) + std::max(0L, (r.H - 1) * r.hs * size) + row; };
  if (start + low(b) >= high(a) || low(a) >= start + high(b)) return true;
  const long step = std::gcd(a.ts, b.ts) * size, reach = a.ts == b.ts ? T - 1 : LONG_MAX;
  const auto meet = [&](long d) {                            // some |i| <= reach with |d + i step| < row
    if (step == 0) return std::abs(d) < row;
    const long i = std::abs(d) / step, rest = std::abs(d) % step;
    return (i <= reach && rest < row) || (i < reach && step - rest < row) || (i > reach && std::abs(d) - reach * step < row);
  };
  if (a.hs == b.hs) {                                        // the heads' distances are few
    for (long h = 1 - a.H; h < b.H; ++h)
      if (meet(start + h * b.hs * size)) return false;
    return true;
  }
  if ((long)a.H * b.H > 1 << 16) return false;
  for (int i = 0; i < a.H; ++i)
    for (int j = 0; j < b.H; ++j)
      if (meet(start + (j * b.hs - i * a.hs) * size)) return false;
  return true;
}

// more than 64 KiB of LDS has to be asked for, once on each device
inline void allow_lds(const void* kernel, int bytes, std::atomic<unsigned long>& done) {
  int device = 0;
  if (hipGetDevice(&device) != hipSuccess || (device < 64 && done.load() >> device & 1)) return;
  if (hipFuncSetAttribute(kernel, hipFuncAttributeMaxDynamicSharedMemorySize, bytes) == hipSuccess && device < 64) done |= 1ul << device;
}

}  // namespace seq
