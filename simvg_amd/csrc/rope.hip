// Norms of queries and keys for each head with the rotation by several position axes in the same pass, forward and backward.
//
//   n = x / sqrt(mean(x^2) + eps),  z = g * n          (a head's row of D values; g shared by the heads of q, another one by k's)
//   y[a_j] = z[a_j] cos t_j - z[b_j] sin t_j,  y[b_j] = z[a_j] sin t_j + z[b_j] cos t_j     for the P = sum(sections) rotated pairs
//   t_j = pos[row, axis(j)] * inv_freq[j];  (a_j, b_j) = (j, j + P) or, interleaved, (2j, 2j + 1);  values from 2P on are not rotated
//
//   backward: dz = the rotation by -t of dy;  dg = sum over rows and heads of dz * n;  dn = g * dz;
//             dx = (dn - n mean(dn n)) / sqrt(mean(x^2) + eps)       (n is computed again from x, which has to be read anyway)
//
// Bound by HBM: one read and one write of q and k forward, two reads and one write backward.  A wave takes one token: 64 lanes
// compute its P angles once (the angle is a product in 64 bits, reduced to a part of a turn there: an axis position of 2^20 times a
// frequency keeps 2^-32 of a turn, in 32 bits it would keep 2^-4) and leave (cos, sin) in LDS for all heads; then groups of lanes
// take a head's row each, a lane holding the two chunks of 16 bytes whose values are each other's partners, so that nothing but the
// sum of squares crosses lanes.
//
// Measured, medians (a copy of 4 GiB reaches 4.7 TB/s, one that stays in the 256 MB memory-side cache 7.2): 26944 tokens, 24 heads of 64,
// fp16, forward: 36 us, 4.6 TB/s; 16384 tokens, 40 heads of 128, bf16: forward 60 us, 5.6 TB/s, backward 116 us and the join of the weights'
// gradients 5, 4.2 TB/s; one token: 4 us.  Rows that start anywhere, a value at a time: 144 us where chunks take 48 (26944 tokens, fp16,
// the call included), backward 292 and 87.
#include "seq.h"

struct simvg_qk_norm_rope_args {
  int dtype, T, Hq, Hkv, D, n_axes, sections[4], interleaved, pos_is_64;
  float eps;
  const void* pos; long pos_ld;
  const double* inv_freq;
  const float *gq, *gk;                                     // both or neither: without them the rows are only rotated
  const void* q; long q_ts, q_hs; const void* k; long k_ts, k_hs;             // inputs (token and head strides in elements)
  void* q_out; long qo_ts, qo_hs; void* k_out; long ko_ts, ko_hs;             // forward: outputs; backward: gradients of the inputs
  const void* dq; long dq_ts, dq_hs; const void* dk; long dk_ts, dk_hs;       // backward: gradients of the outputs
  float *dgq, *dgk, *ws;                                    // backward, with norms: [D] each, and the partial sums' workspace
};

namespace {
using namespace seq;

constexpr int ROPE_MAX_D = 256;
// Workgroups of the backward pass, one partial sum of (dgq | dgk) each: as many as the chip holds at once (three to a compute unit with
// 16-bit values, four with 32-bit ones), each walking its share of the tokens.  16384 tokens, 40 heads of 128, bf16, in turn on one card: 110
// us with 768, 134 with 1024, 121 with 2048; 4099 tokens, fp32: 17.9, 17.0, 18.8.  (The kernels for single values would fit six to a
// compute unit; they were not measured with other numbers.)
constexpr int ROPE_BWD_BLOCKS = 1024;
int rope_bwd_blocks(int T, int dtype) { return min(cdiv(T, 4), dtype == SEQ_F32 ? ROPE_BWD_BLOCKS : 768); }

// V consecutive values: 16 bytes of 16-bit values, or of 32-bit ones, or a single value
template <int DT, int V> struct Chunk;
template <> struct Chunk<SEQ_F32, 4> {
  static __device__ __forceinline__ void load(const void* p, long i, float (&x)[4]) {
    const f32x4_t v = *(const f32x4_t*)((const float*)p + i);
    x[0] = v[0]; x[1] = v[1]; x[2] = v[2]; x[3] = v[3];
  }
  static __device__ __forceinline__ void store(void* p, long i, const float (&x)[4]) {
    *(f32x4_t*)((float*)p + i) = (f32x4_t){x[0], x[1], x[2], x[3]};
  }
};
template <> struct Chunk<SEQ_F32, 1> {
  static __device__ __forceinline__ void load(const void* p, long i, float (&x)[1]) { x[0] = ((const float*)p)[i]; }
  static __device__ __forceinline__ void store(void* p, long i, const float (&x)[1]) { ((float*)p)[i] = x[0]; }
};
template <class E> struct Chunk16 {
  static __device__ __forceinline__ void load8(const void* p, long i, float (&x)[8]) {
    const u32x4_t v = *(const u32x4_t*)((const unsigned short*)p + i);
#pragma unroll
    for (int j = 0; j < 4; ++j) unpack2<E>(v[j], x[2 * j], x[2 * j + 1]);
  }
  static __device__ __forceinline__ void store8(void* p, long i, const float (&x)[8]) {
    *(u32x4_t*)((unsigned short*)p + i) =
        (u32x4_t){E::pack(x[0], x[1]), E::pack(x[2], x[3]), E::pack(x[4], x[5]), E::pack(x[6], x[7])};
  }
};
template <> struct Chunk<SEQ_F16, 8> : Chunk16<F16> {
  static __device__ __forceinline__ void load(const void* p, long i, float (&x)[8]) { load8(p, i, x); }
  static __device__ __forceinline__ void store(void* p, long i, const float (&x)[8]) { store8(p, i, x); }
};
template <> struct Chunk<SEQ_BF16, 8> : Chunk16<BF16> {
  static __device__ __forceinline__ void load(const void* p, long i, float (&x)[8]) { load8(p, i, x); }
  static __device__ __forceinline__ void store(void* p, long i, const float (&x)[8]) { store8(p, i, x); }
};
template <> struct Chunk<SEQ_F16, 1> {
  static __device__ __forceinline__ void load(const void* p, long i, float (&x)[1]) { x[0] = F16::to_f32(((const unsigned short*)p)[i]); }
  static __device__ __forceinline__ void store(void* p, long i, const float (&x)[1]) {
    ((unsigned short*)p)[i] = (unsigned short)F16::pack(x[0], 0.f);
  }
};
template <> struct Chunk<SEQ_BF16, 1> {
  static __device__ __forceinline__ void load(const void* p, long i, float (&x)[1]) { x[0] = BF16::to_f32(((const unsigned short*)p)[i]); }
  static __device__ __forceinline__ void store(void* p, long i, const float (&x)[1]) {
    ((unsigned short*)p)[i] = (unsigned short)BF16::pack(x[0], 0.f);
  }
};

// what a lane of a row's group holds: the two chunks of index c (of D / 2V): partners of a rotation, or two neighbours past 2P
struct Place { int first, second, pair; bool rotated; };
__device__ __forceinline__ Place place(const simvg_qk_norm_rope_args& a, int P, int V, int c) {
  Place p;
  p.pair = c * V;
  p.rotated = c * V < P;
  if (!p.rotated || a.interleaved) { p.first = 2 * V * c; p.second = p.first + V; }
  else { p.first = c * V; p.second = P + c * V; }
  return p;
}

// (cos, sin) of the wave's token into its LDS row
__device__ __forceinline__ void angles(const simvg_qk_norm_rope_args& a, int P, long t, int lane, float2* cs) {
  for (int j = lane; j < P; j += 64) {
    int axis = 0, edge = a.sections[0];
    while (j >= edge) edge += a.sections[++axis];            // j < P = the sections' sum
    const long at = t * a.pos_ld + axis;
    const long pos = a.pos_is_64 ? ((const long*)a.pos)[at] : (long)((const int*)a.pos)[at];
    const double turns = (double)pos * a.inv_freq[j] * 0.15915494309189533577;        // 1 / 2 pi
    float s, c;
    sincospif((float)(2.0 * (turns - rint(turns))), &s, &c);
    cs[j] = make_float2(c, s);
  }
}

// the wave's own LDS row: written and read by this wave alone, whose LDS accesses are done in their order
__device__ __forceinline__ void own_row_written() { asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory"); }

// the rotation of one lane's two chunks by +t (forward) or -t (backward).  Partners are (lo[i], hi[i]), or neighbours of 2V
// consecutive values in lo, hi
template <int V>
__device__ __forceinline__ void rotate(float (&lo)[V], float (&hi)[V], const float2* cs, bool interleaved, float sign) {
  if (V == 1 || !interleaved) {
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const float2 w = cs[i];
      const float s = sign * w.y, x = lo[i], y = hi[i];
      lo[i] = x * w.x - y * s;
      hi[i] = x * s + y * w.x;
    }
  } else {
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const float2 w = cs[i];
      float& px = 2 * i < V ? lo[(2 * i) % V] : hi[(2 * i) % V];
      float& py = 2 * i < V ? lo[(2 * i + 1) % V] : hi[(2 * i + 1) % V];
      const float s = sign * w.y, x = px, y = py;
      px = x * w.x - y * s;
      py = x * s + y * w.x;
    }
  }
}

// LPR lanes (a power of two) per row, NP chunk pairs per lane: NP * LPR >= D / 2V.  `wpt` waves of a workgroup share a token.
template <int DT, int V, int LPR, int NP>
__global__ __launch_bounds__(256) void rope_fwd_kernel(simvg_qk_norm_rope_args a, int P, int wpt) {
  using C = Chunk<DT, V>;
  __shared__ float2 cs_all[4][ROPE_MAX_D / 2];
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  const long t = (long)blockIdx.x * (4 / wpt) + wave / wpt;
  float2* cs = cs_all[wave];
  if (t >= a.T) return;
  angles(a, P, t, lane, cs);
  own_row_written();
  constexpr int GROUPS = 64 / LPR;
  const int group = lane / LPR, l = lane % LPR, n = a.D / (2 * V);
  const float inv_d = 1.f / (float)a.D;
  for (int h = (wave % wpt) * GROUPS + group; h < a.Hq + a.Hkv; h += GROUPS * wpt) {
    const bool is_q = h < a.Hq;
    const void* src = is_q ? a.q : a.k;
    void* dst = is_q ? a.q_out : a.k_out;
    const float* g = is_q ? a.gq : a.gk;
    const long hh = is_q ? h : h - a.Hq;
    const long in0 = t * (is_q ? a.q_ts : a.k_ts) + hh * (is_q ? a.q_hs : a.k_hs);
    const long out0 = t * (is_q ? a.qo_ts : a.ko_ts) + hh * (is_q ? a.qo_hs : a.ko_hs);
    float lo[NP][V], hi[NP][V];
    float sq = 0.f;
#pragma unroll
    for (int i = 0; i < NP; ++i) {
      const int c = l + i * LPR;
      if (c < n) {
        const Place p = place(a, P, V, c);
        C::load(src, in0 + p.first, lo[i]);
        C::load(src, in0 + p.second, hi[i]);
#pragma unroll
        for (int j = 0; j < V; ++j) sq += lo[i][j] * lo[i][j] + hi[i][j] * hi[i][j];
      }
    }
    float r = 1.f;
    if (g) {
#pragma unroll
      for (int o = LPR / 2; o > 0; o >>= 1) sq += __shfl_xor(sq, o, 64);
      r = rsqrtf(sq * inv_d + a.eps);
    }
#pragma unroll
    for (int i = 0; i < NP; ++i) {
      const int c = l + i * LPR;
      if (c < n) {
        const Place p = place(a, P, V, c);
        if (g) {
#pragma unroll
          for (int j = 0; j < V; ++j) {
            lo[i][j] *= r * g[p.first + j];
            hi[i][j] *= r * g[p.second + j];
          }
        }
        if (p.rotated) rotate<V>(lo[i], hi[i], cs + p.pair, a.interleaved != 0, 1.f);
        C::store(dst, out0 + p.first, lo[i]);
        C::store(dst, out0 + p.second, hi[i]);
      }
    }
  }
}

// The sums over rows and heads for dgq, dgk stay in registers while a wave walks its tokens; the workgroup's sum goes to its row of
// the workspace and rope_dg_kernel adds the rows in their order: the same bits at every run.
template <int DT, int V, int LPR, int NP>
__global__ __launch_bounds__(256) void rope_bwd_kernel(simvg_qk_norm_rope_args a, int P) {
  using C = Chunk<DT, V>;
  __shared__ float2 cs_all[4][ROPE_MAX_D / 2];
  __shared__ float sum[4][2 * ROPE_MAX_D];
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  float2* cs = cs_all[wave];
  constexpr int GROUPS = 64 / LPR;
  const int group = lane / LPR, l = lane % LPR, n = a.D / (2 * V);
  const float inv_d = 1.f / (float)a.D;
  float acc[2][NP][2 * V];
#pragma unroll
  for (int w = 0; w < 2; ++w)
#pragma unroll
    for (int i = 0; i < NP; ++i)
#pragma unroll
      for (int j = 0; j < 2 * V; ++j) acc[w][i][j] = 0.f;
  for (long t = (long)blockIdx.x * 4 + wave; t < a.T; t += (long)gridDim.x * 4) {
    angles(a, P, t, lane, cs);
    own_row_written();
#pragma unroll
    for (int w = 0; w < 2; ++w) {
      const int H = w ? a.Hkv : a.Hq;
      const float* g = w ? a.gk : a.gq;
      const void *src = w ? a.k : a.q, *grad = w ? a.dk : a.dq;
      void* dst = w ? a.k_out : a.q_out;
      for (int h = group; h < H; h += GROUPS) {
        const long in0 = t * (w ? a.k_ts : a.q_ts) + h * (w ? a.k_hs : a.q_hs);
        const long gr0 = t * (w ? a.dk_ts : a.dq_ts) + h * (w ? a.dk_hs : a.dq_hs);
        const long out0 = t * (w ? a.ko_ts : a.qo_ts) + h * (w ? a.ko_hs : a.qo_hs);
        float xl[NP][V], xh[NP][V], gl[NP][V], gh[NP][V];
        float sq = 0.f, dot = 0.f;
#pragma unroll
        for (int i = 0; i < NP; ++i) {
          const int c = l + i * LPR;
          if (c < n) {
            const Place p = place(a, P, V, c);
            C::load(grad, gr0 + p.first, gl[i]);
            C::load(grad, gr0 + p.second, gh[i]);
            if (g) {
              C::load(src, in0 + p.first, xl[i]);
              C::load(src, in0 + p.second, xh[i]);
            }
          }
        }
#pragma unroll
        for (int i = 0; i < NP; ++i) {
          const int c = l + i * LPR;
          if (c < n) {
            const Place p = place(a, P, V, c);
            if (p.rotated) rotate<V>(gl[i], gh[i], cs + p.pair, a.interleaved != 0, -1.f);
            if (g) {
#pragma unroll
              for (int j = 0; j < V; ++j) {
                sq += xl[i][j] * xl[i][j] + xh[i][j] * xh[i][j];
                dot += gl[i][j] * g[p.first + j] * xl[i][j] + gh[i][j] * g[p.second + j] * xh[i][j];
              }
            }
          }
        }
        if (!g) {
#pragma unroll
          for (int i = 0; i < NP; ++i) {
            const int c = l + i * LPR;
            if (c < n) {
              const Place p = place(a, P, V, c);
              C::store(dst, out0 + p.first, gl[i]);
              C::store(dst, out0 + p.second, gh[i]);
            }
          }
          continue;
        }
#pragma unroll
        for (int o = LPR / 2; o > 0; o >>= 1) {
          sq += __shfl_xor(sq, o, 64);
          dot += __shfl_xor(dot, o, 64);
        }
        const float r = rsqrtf(sq * inv_d + a.eps);
        const float m = r * r * dot * inv_d;                 // dx = r (g dz - n mean(g dz n)) = r g dz - r (r^2 dot / D) x
#pragma unroll
        for (int i = 0; i < NP; ++i) {
          const int c = l + i * LPR;
          if (c < n) {
            const Place p = place(a, P, V, c);
#pragma unroll
            for (int j = 0; j < V; ++j) {
              acc[w][i][j] += gl[i][j] * (xl[i][j] * r);
              acc[w][i][V + j] += gh[i][j] * (xh[i][j] * r);
              gl[i][j] = r * (gl[i][j] * g[p.first + j] - xl[i][j] * m);
              gh[i][j] = r * (gh[i][j] * g[p.second + j] - xh[i][j] * m);
            }
            C::store(dst, out0 + p.first, gl[i]);
            C::store(dst, out0 + p.second, gh[i]);
          }
        }
      }
    }
  }
  if (!a.gq) return;
#pragma unroll
  for (int w = 0; w < 2; ++w)
#pragma unroll
    for (int i = 0; i < NP; ++i) {
      const int c = l + i * LPR;
      const Place p = place(a, P, V, c);
#pragma unroll
      for (int j = 0; j < 2 * V; ++j) {
        float v = acc[w][i][j];
#pragma unroll
        for (int o = 32; o >= LPR; o >>= 1) v += __shfl_xor(v, o, 64);
        if (group == 0 && c < n) sum[wave][w * a.D + (j < V ? p.first + j : p.second + j - V)] = v;
      }
    }
  __syncthreads();
  for (int i = threadIdx.x; i < 2 * a.D; i += 256)
    a.ws[(long)blockIdx.x * 2 * a.D + i] = (sum[0][i] + sum[1][i]) + (sum[2][i] + sum[3][i]);
}

// dgq | dgk = the sum of `rows` partial rows: 16 columns per workgroup, 64 strands of rows, joined in order
__global__ __launch_bounds__(1024) void rope_dg_kernel(const float* ws, int rows, int D, float* dgq, float* dgk) {
  __shared__ float part[64][17];
  const int c = blockIdx.x * 16 + (threadIdx.x & 15), s = threadIdx.x >> 4;
  float v = 0.f;
  if (c < 2 * D) {
#pragma unroll 8
    for (int r = s; r < rows; r += 64) v += ws[(long)r * 2 * D + c];
  }
  part[s][threadIdx.x & 15] = v;
  __syncthreads();
  const int l = threadIdx.x & 15;
  if (s < 16) part[s][l] = (part[s][l] + part[s + 16][l]) + (part[s + 32][l] + part[s + 48][l]);
  __syncthreads();
  if (s == 0 && c < 2 * D) {
    float total = 0.f;
#pragma unroll
    for (int i = 0; i < 16; ++i) total += part[i][threadIdx.x];
    (c < D ? dgq[c] : dgk[c - D]) = total;
  }
}

bool aligned16(const void* p, long ts, long hs, int size) {
  return (uintptr_t)p % 16 == 0 && ts * size % 16 == 0 && hs * size % 16 == 0;
}

int rope_check(const simvg_qk_norm_rope_args* a, bool bwd, int& P) {
  SIMVG_CHECK_ARG(a, "qk_norm_rope: null argument block");
  SIMVG_CHECK_ARG(a->dtype == SEQ_F32 || a->dtype == SEQ_F16 || a->dtype == SEQ_BF16, "qk_norm_rope: dtype must be fp32, fp16 or bf16");
  SIMVG_CHECK_ARG(a->T >= 0 && a->Hq >= 1 && a->Hkv >= 1, "qk_norm_rope: needs T >= 0 and at least one head of q and of k");
  SIMVG_CHECK_ARG(a->T < 1 << 26, "qk_norm_rope: too many tokens for one launch");
  SIMVG_CHECK_ARG(a->D >= 2 && a->D <= ROPE_MAX_D && a->D % 2 == 0, "qk_norm_rope: the head size must be even and at most 256");
  SIMVG_CHECK_ARG(a->n_axes >= 1 && a->n_axes <= 4, "qk_norm_rope: one to four position axes");
  P = 0;
  for (int i = 0; i < a->n_axes; ++i) {
    SIMVG_CHECK_ARG(a->sections[i] >= 0 && a->sections[i] <= ROPE_MAX_D, "qk_norm_rope: a negative section");
    P += a->sections[i];
  }
  SIMVG_CHECK_ARG(P >= 1 && 2 * P <= a->D, "qk_norm_rope: the sections must sum to between one and D / 2 pairs");
  SIMVG_CHECK_ARG((a->gq == nullptr) == (a->gk == nullptr), "qk_norm_rope: norm weights for both q and k, or for neither");
  SIMVG_CHECK_ARG(a->T == 0 || (a->pos && a->inv_freq && a->q_out && a->k_out), "qk_norm_rope: null pointer");
  SIMVG_CHECK_ARG(a->T == 0 || (a->q && a->k) || (bwd && !a->gq), "qk_norm_rope: null pointer");
  SIMVG_CHECK_ARG(!bwd || a->T == 0 || (a->dq && a->dk), "qk_norm_rope: null pointer");
  SIMVG_CHECK_ARG(!bwd || !a->gq || (a->dgq && a->dgk && a->ws), "qk_norm_rope: the weights' gradients need outputs and a workspace");
  SIMVG_CHECK_ARG(a->pos_ld >= a->n_axes || a->T <= 1, "qk_norm_rope: rows of positions are shorter than the axes");
  // a row is read whole before it is written: results may lie where their own operands do, row on row, and nowhere else on an operand
  const Rows q(a->q, a->q_ts, a->q_hs, a->T, a->Hq), k(a->k, a->k_ts, a->k_hs, a->T, a->Hkv), dq(a->dq, a->dq_ts, a->dq_hs, a->T, a->Hq),
      dk(a->dk, a->dk_ts, a->dk_hs, a->T, a->Hkv), qo(a->q_out, a->qo_ts, a->qo_hs, a->T, a->Hq), ko(a->k_out, a->ko_ts, a->ko_hs, a->T, a->Hkv);
  const auto apart = [&](const Rows& x, const Rows& y) { return rows_apart(x, y, a->T, a->D, a->dtype == SEQ_F32 ? 4 : 2); };
  const auto over = [&](const Rows& out, const Rows& in) { return out.same(in) || apart(out, in); };
  SIMVG_CHECK_ARG(apart(qo, ko) && over(qo, q) && over(ko, k) && apart(qo, k) && apart(ko, q),
                  "qk_norm_rope: a result overlaps another result or an operand (only its own one, row on row, may it replace)");
  SIMVG_CHECK_ARG(!bwd || (over(qo, dq) && over(ko, dk) && apart(qo, dk) && apart(ko, dq)),
                  "qk_norm_rope: a result overlaps another result or an operand (only its own one, row on row, may it replace)");
  return SIMVG_OK;
}

// chunks of 16 bytes where every row, pair and start allows them, single values otherwise
bool rope_wide(const simvg_qk_norm_rope_args& a, int P, bool bwd) {
  const int size = a.dtype == SEQ_F32 ? 4 : 2, V = 16 / size;
  bool ok = a.D % (2 * V) == 0 && P % V == 0 && aligned16(a.q_out, a.qo_ts, a.qo_hs, size) && aligned16(a.k_out, a.ko_ts, a.ko_hs, size);
  if (a.q && a.k) ok = ok && aligned16(a.q, a.q_ts, a.q_hs, size) && aligned16(a.k, a.k_ts, a.k_hs, size);
  if (bwd) ok = ok && aligned16(a.dq, a.dq_ts, a.dq_hs, size) && aligned16(a.dk, a.dk_ts, a.dk_hs, size);
  return ok;
}

template <int DT, int V, int LPR, int NP>
void rope_launch(const simvg_qk_norm_rope_args& a, int P, bool bwd, hipStream_t s) {
  if (!bwd) {
    // with fewer tokens than waves on the chip (a decoder's single tokens) the heads of a token are shared by a workgroup's waves
    const int wpt = a.T < 1024 ? 4 : 1;
    hipLaunchKernelGGL((rope_fwd_kernel<DT, V, LPR, NP>), dim3(cdiv(a.T, 4 / wpt)), dim3(256), 0, s, a, P, wpt);
  } else {
    hipLaunchKernelGGL((rope_bwd_kernel<DT, V, LPR, NP>), dim3(rope_bwd_blocks(a.T, a.dtype)), dim3(256), 0, s, a, P);
  }
}
template <int DT, int V>
void rope_dispatch(const simvg_qk_norm_rope_args& a, int P, bool wide, bool bwd, hipStream_t s) {
  if (!wide) return rope_launch<DT, 1, 64, 2>(a, P, bwd, s);
  const int n = a.D / (2 * V);
  if (n <= 2) return rope_launch<DT, V, 2, 1>(a, P, bwd, s);
  if (n <= 4) return rope_launch<DT, V, 4, 1>(a, P, bwd, s);
  if (n <= 8) return rope_launch<DT, V, 8, 1>(a, P, bwd, s);
  if (n <= 16) return rope_launch<DT, V, 16, 1>(a, P, bwd, s);
  if constexpr (V == 4) return rope_launch<DT, V, 32, 1>(a, P, bwd, s);
}

int rope_run(const simvg_qk_norm_rope_args* args, bool bwd, hipStream_t s) {
  int P = 0;
  const int rc = rope_check(args, bwd, P);
  if (rc) return rc;
  const simvg_qk_norm_rope_args& a = *args;
  if (a.T > 0) {
    const bool wide = rope_wide(a, P, bwd);
    if (a.dtype == SEQ_F32) rope_dispatch<SEQ_F32, 4>(a, P, wide, bwd, s);
    else if (a.dtype == SEQ_F16) rope_dispatch<SEQ_F16, 8>(a, P, wide, bwd, s);
    else rope_dispatch<SEQ_BF16, 8>(a, P, wide, bwd, s);
    SIMVG_LAUNCH_CHECK();
  }
  if (bwd && a.gq) {                                          // without a token the gradients are sums of nothing: zeros
    hipLaunchKernelGGL(rope_dg_kernel, dim3(cdiv(2 * a.D, 16)), dim3(1024), 0, s, a.ws, rope_bwd_blocks(a.T, a.dtype), a.D, a.dgq, a.dgk);
    SIMVG_LAUNCH_CHECK();
  }
  return SIMVG_OK;
}
}  // namespace

extern "C" long simvg_qk_norm_rope_ws_floats(int T, int D) {
  return T < 0 || D < 0 ? 0 : (long)min(cdiv(T, 4), ROPE_BWD_BLOCKS) * 2 * D;
}
extern "C" int simvg_qk_norm_rope_fwd(const simvg_qk_norm_rope_args* args, hipStream_t stream) { return rope_run(args, false, stream); }
extern "C" int simvg_qk_norm_rope_bwd(const simvg_qk_norm_rope_args* args, hipStream_t stream) { return rope_run(args, true, stream); }
