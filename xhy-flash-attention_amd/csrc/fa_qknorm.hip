// Per-head RMS norm of queries and keys with the rotary embedding in the same pass (gfx950).
//
// For each (batch, token, head) row x of d elements, gains w, and a token's angles (cos, sin)[p]:
//     r = 1 / sqrt(mean(x^2) + eps),   n = x r,   z = w n,
//     y = z with the pairs of its first rotary_dim columns rotated: (z1 c - z2 s, z1 s + z2 c).
// Backward, g = the rotation's transpose applied to dy:
//     dw = sum over rows of g n,       dx = r (g w - n mean(g w n)).
// Everything is fp32 between the loads and the one rounding of each output.
//
// HBM-bound: x is read once and y written once (backward: x, dy read, dx written; the norm is
// recomputed from x, so the forward saves nothing).  So the layout serves the memory pipe:
//   * a row is spread over LPR lanes and a lane holds two W-element pieces of it, chosen so that a
//     rotation pair never crosses lanes (halves: piece i of either half; adjacent pairs: any piece).
//     The row sum is log2(LPR) cross-lane adds, the rotation is lane-local;
//   * a lane keeps one token's angles in registers for up to NH heads of it, and issues all of their
//     row loads before the first use;
//   * W = 8 (16-byte pieces) where strides, rotary_dim and the tables allow it; W = 1 takes every
//     other shape with 64 lanes per row (4 x 8192 tokens, 32 + 8 heads of 128, rotary_dim 24, 40 or 54: 328 us
//     forward and 1005 backward against 125 and 205);
//   * the backward is one round of resident workgroups over the rows, each with its partial of dw.
// Measured on those 4 x 8192 tokens, bf16: forward 124 us (0.67 GB, 5.4 TB/s, what a copy reaches),
// backward 205 + 6 us (1.0 GB, 4.8 TB/s); 16 tokens: 4.0 us, a launch.
// The weight gradient is reduced in registers over a lane's rows, over the workgroup through LDS,
// and over workgroups by a second kernel in a fixed order: no atomics, bitwise deterministic.
#include <stdexcept>
#include <string>

#include "fa_common.h"
#include "fa_params.h"

namespace fa {

typedef unsigned short u16;
static constexpr int kThreads = 256;

template <bool BF16>
__device__ inline u16 to_elt(float x) { return (u16)(Elt<BF16>::pack2(x, 0.f) & 0xffffu); }

template <bool BF16, int W>
__device__ inline void load_elts(const void* p, float (&x)[W], bool ok) {
  if constexpr (W == 8) {
    const u32x4_t v = ld16(p, ok);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      x[2 * i] = Elt<BF16>::to_f32((u16)(v[i] & 0xffffu));
      x[2 * i + 1] = Elt<BF16>::to_f32((u16)(v[i] >> 16));
    }
  } else {
    static_assert(W == 1, "pieces of 8 or 1");
    x[0] = ok ? Elt<BF16>::to_f32(*(const u16*)p) : 0.f;
  }
}

template <bool BF16, int W>
__device__ inline void store_elts(void* p, const float (&x)[W], bool ok) {
  if (!ok) return;
  if constexpr (W == 8) {
    u32x4_t v;
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = Elt<BF16>::pack2(x[2 * i], x[2 * i + 1]);
    *(u32x4_t*)p = v;
  } else {
    *(u16*)p = to_elt<BF16>(x[0]);
  }
}

// N consecutive values of a table or gain vector in fp32 (element type: fp32, or the input's)
template <bool BF16, int N>
__device__ inline void load_table(const void* base, int64_t at, bool f32, float* x) {
  if (f32) {
    const float* p = (const float*)base + at;
    if constexpr (N % 4 == 0) {
#pragma unroll
      for (int i = 0; i < N / 4; ++i) {
        const f32x4_t v = *(const f32x4_t*)(p + 4 * i);
#pragma unroll
        for (int e = 0; e < 4; ++e) x[4 * i + e] = v[e];
      }
    } else {
#pragma unroll
      for (int i = 0; i < N; ++i) x[i] = p[i];
    }
  } else {
    const u16* p = (const u16*)base + at;
    if constexpr (N % 4 == 0) {
#pragma unroll
      for (int i = 0; i < N / 4; ++i) {
        const u32x2_t v = *(const u32x2_t*)(p + 4 * i);
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          x[4 * i + 2 * e] = Elt<BF16>::to_f32((u16)(v[e] & 0xffffu));
          x[4 * i + 2 * e + 1] = Elt<BF16>::to_f32((u16)(v[e] >> 16));
        }
      }
    } else {
#pragma unroll
      for (int i = 0; i < N; ++i) x[i] = Elt<BF16>::to_f32(p[i]);
    }
  }
}

// The two pieces of a row that slot t holds: their first columns, and which rotation applies.
//   pair (halves, and W = 1): element e of piece a turns with element e of piece b, angle angle_a + e
//   else (adjacent pairs, W = 8): elements 2i, 2i+1 of either piece turn, angles angle_a + i, angle_b + i
template <int W>
struct Pieces {
  int a, b, angle_a, angle_b;
  bool has_a, has_b, turn_a, turn_b;
  __device__ inline Pieces(int t, int d, int rd, bool interleaved) {
    const int half = rd / 2;
    if (interleaved && W == 1) {
      a = 2 * t; b = a + 1;
      angle_a = angle_b = t;
      turn_a = turn_b = a < rd;
    } else if (interleaved) {
      a = t * W; b = (t + (d / W + 1) / 2) * W;
      if (t >= (d / W + 1) / 2) a = b = d;   // a slot past the row
      angle_a = a / 2; angle_b = b / 2;
      turn_a = a < rd; turn_b = b < rd;
    } else {
      const int nh = half / W;
      turn_a = turn_b = t < nh;
      a = turn_a ? t * W : rd + 2 * (t - nh) * W;
      b = turn_a ? a + half : a + W;
      angle_a = a; angle_b = a;
    }
    has_a = a < d; has_b = b < d;
  }
};

// c, s of a slot: W angles (adjacent pairs with W = 8: four for each piece); (1, 0) where nothing turns
template <bool BF16, int W>
__device__ inline void load_angles(const QkNormParams& p, const Pieces<W>& pc, int64_t row, float (&c)[W],
                                   float (&s)[W]) {
#pragma unroll
  for (int e = 0; e < W; ++e) { c[e] = 1.f; s[e] = 0.f; }
  const int64_t at = row * p.cs_row;
  if (W == 8 && p.interleaved) {
    if (pc.turn_a && pc.has_a) {
      load_table<BF16, (W + 1) / 2>(p.cos, at + pc.angle_a, p.table_f32, c);
      load_table<BF16, (W + 1) / 2>(p.sin, at + pc.angle_a, p.table_f32, s);
    }
    if (pc.turn_b && pc.has_b) {
      load_table<BF16, (W + 1) / 2>(p.cos, at + pc.angle_b, p.table_f32, c + W / 2);
      load_table<BF16, (W + 1) / 2>(p.sin, at + pc.angle_b, p.table_f32, s + W / 2);
    }
  } else if (pc.turn_a && pc.has_a) {
    load_table<BF16, W>(p.cos, at + pc.angle_a, p.table_f32, c);
    load_table<BF16, W>(p.sin, at + pc.angle_a, p.table_f32, s);
  }
}

// rotates the pieces in place (dir = 1: forward, -1: the transpose)
template <int W>
__device__ inline void turn(float (&xa)[W], float (&xb)[W], const float (&c)[W], const float (&s)[W], float dir,
                            bool adjacent) {
  if (W == 8 && adjacent) {
#pragma unroll
    for (int i = 0; i < W / 2; ++i) {
      const float a0 = xa[2 * i], a1 = xa[(2 * i + 1) % W], b0 = xb[2 * i], b1 = xb[(2 * i + 1) % W];
      const float sa = dir * s[i], sb = dir * s[(W / 2 + i) % W];
      xa[2 * i] = a0 * c[i] - a1 * sa;
      xa[(2 * i + 1) % W] = a0 * sa + a1 * c[i];
      xb[2 * i] = b0 * c[(W / 2 + i) % W] - b1 * sb;
      xb[(2 * i + 1) % W] = b0 * sb + b1 * c[(W / 2 + i) % W];
    }
  } else {
#pragma unroll
    for (int e = 0; e < W; ++e) {
      const float a = xa[e], b = xb[e], se = dir * s[e];
      xa[e] = a * c[e] - b * se;
      xb[e] = a * se + b * c[e];
    }
  }
}

template <int LPR>
__device__ inline float row_sum(float x) {
#pragma unroll
  for (int off = 1; off < LPR; off <<= 1) x += __shfl_xor(x, off);
  return x;
}

// gains of a slot's pieces (1 without a gain vector, 0 past the row)
template <bool BF16, int W>
__device__ inline void load_gains(const void* w, const Pieces<W>& pc, bool f32, float (&ga)[W], float (&gb)[W]) {
#pragma unroll
  for (int e = 0; e < W; ++e) { ga[e] = 1.f; gb[e] = 1.f; }
  if (w == nullptr) return;
  if (pc.has_a) load_table<BF16, W>(w, pc.a, f32, ga);
  if (pc.has_b) load_table<BF16, W>(w, pc.b, f32, gb);
}

// table row of a token, or -1 when its position is outside the table (the row's outputs become NaN)
__device__ inline int64_t table_row(const QkNormParams& p, int bi, int si) {
  if (p.cos == nullptr) return 0;
  const int64_t r = p.positions ? (int64_t)p.positions[(int64_t)bi * p.pos_batch + si] : (int64_t)si;
  return r >= 0 && r < p.table_rows ? r : -1;
}

// One group of LPR lanes takes a token's heads [NH hb, NH hb + NH) of q or k.
template <bool BF16, int W, int LPR, int NP, int NH>
__global__ void __launch_bounds__(kThreads) qk_norm_fwd_kernel(const QkNormParams p) {
  const int lane = threadIdx.x % LPR;
  const int64_t item = (int64_t)blockIdx.x * (kThreads / LPR) + threadIdx.x / LPR;
  const int hbq = (p.h + NH - 1) / NH, hbs = hbq + (p.hk + NH - 1) / NH;
  const int64_t token = item / hbs;
  if (token >= (int64_t)p.b * p.seqlen) return;
  int hb = (int)(item - token * hbs);
  const int bi = (int)(token / p.seqlen), si = (int)(token - (int64_t)bi * p.seqlen);
  const bool is_k = hb >= hbq;
  if (is_k) hb -= hbq;
  const int heads = is_k ? p.hk : p.h;
  const QkNormTensor in = is_k ? p.k : p.q, out = is_k ? p.k_out : p.q_out;
  const u16* x0 = (const u16*)in.ptr + bi * in.batch + si * in.row;
  u16* y0 = (u16*)out.ptr + bi * out.batch + si * out.row;

  float xa[NP][NH][W], xb[NP][NH][W];
#pragma unroll
  for (int j = 0; j < NP; ++j) {
    const Pieces<W> pc(lane + j * LPR, p.d, p.rd, p.interleaved);
#pragma unroll
    for (int n = 0; n < NH; ++n) {
      const int head = hb * NH + n;
      const u16* x = x0 + (int64_t)(head < heads ? head : 0) * in.head;
      load_elts<BF16, W>(x + (pc.has_a ? pc.a : 0), xa[j][n], pc.has_a && head < heads);
      load_elts<BF16, W>(x + (pc.has_b ? pc.b : 0), xb[j][n], pc.has_b && head < heads);
    }
  }
  const int64_t trow = table_row(p, bi, si);
  float r[NH];
#pragma unroll
  for (int n = 0; n < NH; ++n) {
    float sum = 0.f;
#pragma unroll
    for (int j = 0; j < NP; ++j)
#pragma unroll
      for (int e = 0; e < W; ++e) sum += xa[j][n][e] * xa[j][n][e] + xb[j][n][e] * xb[j][n][e];
    r[n] = 1.f / sqrtf(row_sum<LPR>(sum) * p.inv_d + p.eps);
    if (trow < 0) r[n] = __builtin_nanf("");
  }
#pragma unroll
  for (int j = 0; j < NP; ++j) {
    const Pieces<W> pc(lane + j * LPR, p.d, p.rd, p.interleaved);
    float c[W], s[W], ga[W], gb[W];
    load_angles<BF16, W>(p, pc, trow < 0 ? 0 : trow, c, s);
    load_gains<BF16, W>(is_k ? p.wk : p.wq, pc, p.weight_f32, ga, gb);
#pragma unroll
    for (int n = 0; n < NH; ++n) {
      const int head = hb * NH + n;
#pragma unroll
      for (int e = 0; e < W; ++e) { xa[j][n][e] *= r[n] * ga[e]; xb[j][n][e] *= r[n] * gb[e]; }
      turn<W>(xa[j][n], xb[j][n], c, s, 1.f, p.interleaved);
      u16* y = y0 + (int64_t)head * out.head;
      store_elts<BF16, W>(y + pc.a, xa[j][n], pc.has_a && head < heads);
      store_elts<BF16, W>(y + pc.b, xb[j][n], pc.has_b && head < heads);
    }
  }
}

// Workgroups [0, blocks_q) take q's items, the others k's; a workgroup's partial weight gradient
// goes to dw_part[block][d].
template <bool BF16, int W, int LPR, int NP, int NH>
__global__ void __launch_bounds__(kThreads) qk_norm_bwd_kernel(const QkNormParams p) {
  constexpr int GROUPS = kThreads / LPR;
  const int lane = threadIdx.x % LPR, group = threadIdx.x / LPR;
  const bool is_k = blockIdx.x >= (unsigned)p.blocks_q;
  const int block = is_k ? (int)blockIdx.x - p.blocks_q : (int)blockIdx.x;
  const int blocks = is_k ? (int)gridDim.x - p.blocks_q : p.blocks_q;
  const int heads = is_k ? p.hk : p.h;
  const int hbs = (heads + NH - 1) / NH;
  const QkNormTensor in = is_k ? p.k : p.q, dout = is_k ? p.k_grad : p.q_grad, dx = is_k ? p.k_out : p.q_out;
  const int64_t items = (int64_t)p.b * p.seqlen * hbs;

  float ga[NP][W], gb[NP][W], wa[NP][W], wb[NP][W];
#pragma unroll
  for (int j = 0; j < NP; ++j) {
    const Pieces<W> pc(lane + j * LPR, p.d, p.rd, p.interleaved);
    load_gains<BF16, W>(is_k ? p.wk : p.wq, pc, p.weight_f32, ga[j], gb[j]);
#pragma unroll
    for (int e = 0; e < W; ++e) wa[j][e] = wb[j][e] = 0.f;
  }
  for (int64_t item = (int64_t)block * GROUPS + group; item < items; item += (int64_t)blocks * GROUPS) {
    const int64_t token = item / hbs;
    const int hb = (int)(item - token * hbs);
    const int bi = (int)(token / p.seqlen), si = (int)(token - (int64_t)bi * p.seqlen);
    const u16* x0 = (const u16*)in.ptr + bi * in.batch + si * in.row;
    const u16* g0 = (const u16*)dout.ptr + bi * dout.batch + si * dout.row;
    u16* d0 = (u16*)dx.ptr + bi * dx.batch + si * dx.row;
    const int64_t trow = table_row(p, bi, si);
    float xa[NP][NH][W], xb[NP][NH][W], ya[NP][NH][W], yb[NP][NH][W];
#pragma unroll
    for (int j = 0; j < NP; ++j) {
      const Pieces<W> pc(lane + j * LPR, p.d, p.rd, p.interleaved);
#pragma unroll
      for (int n = 0; n < NH; ++n) {
        const int head = hb * NH + n;
        const bool ok = head < heads;
        const u16* x = x0 + (int64_t)(ok ? head : 0) * in.head;
        const u16* g = g0 + (int64_t)(ok ? head : 0) * dout.head;
        load_elts<BF16, W>(x + (pc.has_a ? pc.a : 0), xa[j][n], pc.has_a && ok);
        load_elts<BF16, W>(x + (pc.has_b ? pc.b : 0), xb[j][n], pc.has_b && ok);
        load_elts<BF16, W>(g + (pc.has_a ? pc.a : 0), ya[j][n], pc.has_a && ok);
        load_elts<BF16, W>(g + (pc.has_b ? pc.b : 0), yb[j][n], pc.has_b && ok);
      }
    }
    float sum[NH], dot[NH];
#pragma unroll
    for (int n = 0; n < NH; ++n) sum[n] = dot[n] = 0.f;
#pragma unroll
    for (int j = 0; j < NP; ++j) {
      const Pieces<W> pc(lane + j * LPR, p.d, p.rd, p.interleaved);
      float c[W], s[W];
      load_angles<BF16, W>(p, pc, trow < 0 ? 0 : trow, c, s);
#pragma unroll
      for (int n = 0; n < NH; ++n) {
        turn<W>(ya[j][n], yb[j][n], c, s, -1.f, p.interleaved);
#pragma unroll
        for (int e = 0; e < W; ++e) {
          sum[n] += xa[j][n][e] * xa[j][n][e] + xb[j][n][e] * xb[j][n][e];
          dot[n] += ya[j][n][e] * ga[j][e] * xa[j][n][e] + yb[j][n][e] * gb[j][e] * xb[j][n][e];
        }
      }
    }
#pragma unroll
    for (int n = 0; n < NH; ++n) {
      float r = 1.f / sqrtf(row_sum<LPR>(sum[n]) * p.inv_d + p.eps);
      if (trow < 0) r = __builtin_nanf("");
      const float k = row_sum<LPR>(dot[n]) * r * r * p.inv_d;   // mean(g w n) r
      const int head = hb * NH + n;
#pragma unroll
      for (int j = 0; j < NP; ++j) {
        const Pieces<W> pc(lane + j * LPR, p.d, p.rd, p.interleaved);
        float oa[W], ob[W];
#pragma unroll
        for (int e = 0; e < W; ++e) {
          // a head past the last: x = g = 0, but r = 1 / sqrt(eps) may be infinite
          if (head < heads) {
            wa[j][e] += ya[j][n][e] * xa[j][n][e] * r;
            wb[j][e] += yb[j][n][e] * xb[j][n][e] * r;
          }
          oa[e] = r * (ya[j][n][e] * ga[j][e] - xa[j][n][e] * k);
          ob[e] = r * (yb[j][n][e] * gb[j][e] - xb[j][n][e] * k);
        }
        u16* dst = d0 + (int64_t)head * dx.head;
        store_elts<BF16, W>(dst + pc.a, oa, pc.has_a && head < heads);
        store_elts<BF16, W>(dst + pc.b, ob, pc.has_b && head < heads);
      }
    }
  }
  if (p.dw_part == nullptr) return;
  // lanes of a wave with the same slot, then the four waves
  __shared__ float part[kThreads / 64][256];
  const int wave = threadIdx.x >> 6;
#pragma unroll
  for (int j = 0; j < NP; ++j) {
    const Pieces<W> pc(lane + j * LPR, p.d, p.rd, p.interleaved);
#pragma unroll
    for (int e = 0; e < W; ++e) {
      float a = wa[j][e], b = wb[j][e];
#pragma unroll
      for (int off = LPR; off < 64; off <<= 1) { a += __shfl_xor(a, off); b += __shfl_xor(b, off); }
      if ((threadIdx.x & 63) < LPR) {
        if (pc.has_a) part[wave][pc.a + e] = a;
        if (pc.has_b) part[wave][pc.b + e] = b;
      }
    }
  }
  __syncthreads();
  for (int i = threadIdx.x; i < p.d; i += kThreads) {
    float sum = 0.f;
#pragma unroll
    for (int w = 0; w < kThreads / 64; ++w) sum += part[w][i];
    p.dw_part[(int64_t)blockIdx.x * p.d + i] = sum;
  }
}

// dw[i] = sum over the workgroups' partials: 16 columns x 64 partial rows per workgroup
// (blockIdx.y: q or k)
template <bool BF16>
__global__ void __launch_bounds__(1024) qk_norm_dw_kernel(const QkNormParams p, int blocks) {
  const bool is_k = blockIdx.y != 0;
  const int first = is_k ? p.blocks_q : 0, last = is_k ? blocks : p.blocks_q;
  void* dw = is_k ? p.dwk : p.dwq;
  if (dw == nullptr) return;
  const int col = threadIdx.x & 15, row = threadIdx.x >> 4;
  const int i = blockIdx.x * 16 + col;
  float sum = 0.f;
  if (i < p.d)
    for (int r = first + row; r < last; r += 64) sum += p.dw_part[(int64_t)r * p.d + i];
  __shared__ float part[64][17];
  part[row][col] = sum;
  __syncthreads();
  for (int off = 32; off > 0; off >>= 1) {
    if (row < off) part[row][col] += part[row + off][col];
    __syncthreads();
  }
  if (row == 0 && i < p.d) {
    if (p.weight_f32) ((float*)dw)[i] = part[0][col];
    else ((u16*)dw)[i] = to_elt<BF16>(part[0][col]);
  }
}

// 16-byte pieces: aligned bases and strides, whole pieces, rotation pairs in whole pieces
static bool vector_ok(const QkNormParams& p, bool backward) {
  auto aligned = [](const QkNormTensor& t) {
    return (uintptr_t)t.ptr % 16 == 0 && t.batch % 8 == 0 && t.row % 8 == 0 && t.head % 8 == 0;
  };
  auto based = [](const void* q) { return (uintptr_t)q % 16 == 0; };
  bool ok = p.d % 8 == 0 && p.rd % 16 == 0 && aligned(p.q) && aligned(p.k) && aligned(p.q_out) && aligned(p.k_out);
  ok = ok && based(p.wq) && based(p.wk) && based(p.cos) && based(p.sin) && p.cs_row % 8 == 0;
  if (backward) ok = ok && aligned(p.q_grad) && aligned(p.k_grad);
  return ok;
}

// Heads a group of lanes takes of one token: more share the angles' loads and keep more row loads in
// flight, fewer spread a decoding step over more CUs.  Forward: four, or one where four leave CUs without a
// workgroup (32 + 8 heads of 128, bf16; 4 x 8192 tokens: four 124 us, two 132, one 138; 16 tokens: four
// 5.2 us, two 4.5, one 4.0).  Backward: two (one and four are within 3 % at their best numbers of workgroups).
static constexpr int kHeadsFwd = 4, kHeadsBwd = 2;

template <bool BF16, int W, int LPR, int NP, int NH>
static bool run_forward(const QkNormParams& p, int64_t least, hipStream_t stream) {
  constexpr int groups = kThreads / LPR;
  const int hbs = (p.h + NH - 1) / NH + (p.hk + NH - 1) / NH;
  const int64_t grid = ((int64_t)p.b * p.seqlen * hbs + groups - 1) / groups;
  if (grid < least) return false;
  if (grid > 0x7fffffff) throw std::runtime_error("qk_norm_rotary: too many rows for one launch");
  hipLaunchKernelGGL((qk_norm_fwd_kernel<BF16, W, LPR, NP, NH>), dim3((unsigned)grid), dim3(kThreads), 0, stream, p);
  return true;
}

template <bool BF16, int W, int LPR, int NP>
static void run(QkNormParams& p, bool backward, hipStream_t stream) {
  constexpr int groups = kThreads / LPR;
  const int64_t tokens = (int64_t)p.b * p.seqlen;
  if (!backward) {
    if (!run_forward<BF16, W, LPR, NP, kHeadsFwd>(p, 256, stream)) run_forward<BF16, W, LPR, NP, 1>(p, 0, stream);
    return;
  }
  const int64_t gq = (tokens * ((p.h + kHeadsBwd - 1) / kHeadsBwd) + groups - 1) / groups;
  const int64_t gk = (tokens * ((p.hk + kHeadsBwd - 1) / kHeadsBwd) + groups - 1) / groups;
  // workgroups in proportion to the items of q and k, one round of them at most (1024, with a round of a
  // third behind three workgroups a CU: 227 us instead of 205)
  const int64_t total = gq + gk < kQkNormMaxBlocks ? gq + gk : kQkNormMaxBlocks;
  int64_t bq = (total * gq + (gq + gk) / 2) / (gq + gk);
  if (bq < 1) bq = 1;
  if (bq > total - 1) bq = total - 1;
  p.blocks_q = (int)bq;
  hipLaunchKernelGGL((qk_norm_bwd_kernel<BF16, W, LPR, NP, kHeadsBwd>), dim3((unsigned)total), dim3(kThreads), 0, stream,
                     p);
  if (p.dw_part != nullptr)
    hipLaunchKernelGGL((qk_norm_dw_kernel<BF16>), dim3((p.d + 15) / 16, 2), dim3(1024), 0, stream, p, (int)total);
}

template <bool BF16>
static void dispatch(QkNormParams& p, bool backward, hipStream_t stream) {
  if (!vector_ok(p, backward)) return run<BF16, 1, 64, 2>(p, backward, stream);
  if (p.d <= 32) return run<BF16, 8, 2, 1>(p, backward, stream);
  if (p.d <= 64) return run<BF16, 8, 4, 1>(p, backward, stream);
  if (p.d <= 128) return run<BF16, 8, 8, 1>(p, backward, stream);
  return run<BF16, 8, 16, 1>(p, backward, stream);
}

void launch_qk_norm(QkNormParams p, bool backward, bool is_bf16, hipStream_t stream) {
  if (p.b == 0 || p.seqlen == 0) return;
  if (is_bf16) dispatch<true>(p, backward, stream);
  else dispatch<false>(p, backward, stream);
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) throw std::runtime_error(std::string("qk_norm_rotary launch: ") + hipGetErrorString(e));
}

}  // namespace fa
