// Attention of drafted tokens over a key/value cache (gfx950): sq rows a sequence (1: plain decoding).
//
// Row i of sequence b sees the lens[b] cached keys and, of the sq drafted keys behind them, those its
// mask row names (without a mask: drafted keys 0 .. i).  O = softmax(scale q k) v, LSE = its logarithm.
//
// MI355X mapping.  With few rows the call is bound by reading K and V once, so the work is split over
// the keys until the chip is full, and every wave streams its own keys:
//   * the G query heads of a kv head and the sq tokens are packed as rows (row = token G + head), so a
//     kv head's K/V is read once for all of them; a workgroup takes 32 WM rows (WM = 1, 2, 4) of a
//     (sequence, kv head, key split);
//   * a step of the workgroup is 128 keys, 32 a wave: a wave loads its 32 K and V rows one step ahead
//     into registers (16 bytes a lane, whole rows; the compiler's counted waits keep them in flight
//     over the step's compute) and hands them over through its own LDS tile, which MFMA operands
//     are then read from (row reads for K, transposing reads for V);
//   * WM = 1: the four waves take different keys and no barrier is needed; WM = 4: they take
//     different rows of the same 128 keys; WM = 2: two by two.  Waves that share rows merge their
//     (max, sum, O) through LDS at the end; key splits through fp32 partials and a second kernel;
//   * S^T = K Q^T and O^T = V^T P^T as in fa_fwd.hip: a lane holds one row, so the softmax is lane-local
//     plus one half swap, and P is the next product's operand without moving.
// P is rounded to 16 bits for the product with V (half a step of the type relative to each weight;
// the sum that divides is of the unrounded P); scores, statistics, O and the partials are fp32.
//
// A row's result depends on what it sees alone: non-finite values of a drafted V row, which the product
// would multiply by the zero weights of the rows that do not see it, are taken out of the tile and
// added to the rows that do (a rare path, looked for in steps with drafted keys only).
// Keys past a sequence's end load as zeros, so no slot behind it reaches a result.  A sequence whose
// length does not leave room for the drafted tokens, or that names a page outside the cache, gives NaN.
#include <algorithm>
#include <stdexcept>
#include <string>

#include "fa_kvcache.h"

namespace fa {

typedef unsigned short u16;
static constexpr int kStep = 128;   // keys a workgroup takes at a time, 32 a wave

__device__ inline int64_t shfl64(int64_t x, int lane) {
  const unsigned lo = (unsigned)__shfl((int)(unsigned)x, lane), hi = (unsigned)__shfl((int)(x >> 32), lane);
  return (int64_t)(((uint64_t)hi << 32) | lo);
}

// A wave's 32 K and V rows in flight: lane -> (row, 16-byte chunk), whole rows per instruction, and
// within it four rows of a 64-byte panel per 16 lanes (the LDS writes then fill whole bank lines)
template <int D>
struct Stage {
  static constexpr int CPR = D / 8, RPI = 64 / CPR, NI = 32 / RPI, RQ = RPI < 4 ? RPI : 4;
  u32x4_t k[NI], v[NI];
  static __device__ inline int row(int i, int lane) {
    const int q = lane >> 2;
    return i * RPI + (q / RQ) / (CPR / 4) * RQ + q % RQ;
  }
  static __device__ inline int chunk(int lane) { return ((lane >> 2) / RQ) % (CPR / 4) * 4 + (lane & 3); }
};

// infinities and NaN of two packed elements
template <bool BF16>
__device__ inline unsigned odd_pair(unsigned u) {
  constexpr unsigned m = BF16 ? 0x7f80u : 0x7c00u;
  return ((u & m) == m ? 0xffffu : 0u) | ((u & (m << 16)) == (m << 16) ? 0xffff0000u : 0u);
}

template <bool BF16, int D, int WM>
__global__ void __launch_bounds__(256, D <= 128 ? 2 : 1) kv_attn_kernel(const KvAttnParams p) {
  using E = Elt<BF16>;
  using St = Stage<D>;
  constexpr int KS = D / 16, NP = D / 32, WK = 4 / WM;
  constexpr int TILE = 32 * D * 2;                 // bytes of one wave's K (or V) rows
  __shared__ __attribute__((aligned(16))) char smem[4 * 2 * TILE];
  __shared__ float sm_m[4][32], sm_l[4][32];
  __shared__ int sm_bad[4], sm_odd[4];
  const KvCache& c = p.c;
  const int tid = threadIdx.x, lane = tid & 63, wave = wave_uniform(tid >> 6);
  const int r = lane & 31, hh = lane >> 5;
  const LdsBases lb(lane);

  // (split, sequence, kv head) units; a unit's row tiles sit 8 workgroups apart: the same XCD, whose L2
  // then serves K/V to all of them
  const int per = 8 * p.m_tiles;
  const int oct = blockIdx.x / per, rem = blockIdx.x - oct * per;
  const int mt = rem >> 3, unit = oct * 8 + (rem & 7);
  const int nbh = c.b * c.hk;
  if (unit >= nbh * p.splits) return;
  const int split = unit / nbh, bh = unit - split * nbh;
  const int bidb = bh / c.hk, kvh = bh - bidb * c.hk;

  const int len = c.lens[bidb];
  const bool ok_seq = seq_ok(c, len, p.sq);
  const int total = ok_seq ? len + p.sq : 0;
  // the sequence's steps, dealt evenly to the splits
  const int steps = (total + kStep - 1) / kStep;
  const int per_split = (steps + p.splits - 1) / p.splits;
  const int s0 = split * per_split, s1 = min(steps, s0 + per_split);
  if (p.splits > 1 && s0 >= s1) return;            // the merge knows which splits have keys

  const int wm = wave % WM, wk = wave / WM;
  const int row0 = (mt * WM + wm) * 32;
  const int row = row0 + r;                        // this lane's row
  const bool row_ok = row < p.rows;
  const int tok = (row_ok ? row : 0) / p.group, gh = (row_ok ? row : 0) - tok * p.group;

  i16x8_t qf[KS];
  {
    const u16* q = (const u16*)p.q + (int64_t)bidb * p.q_batch + (int64_t)tok * p.q_row +
                   (int64_t)(kvh * p.group + gh) * p.q_head;
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) {
      const int d0 = 16 * ks + 8 * hh;
      qf[ks] = __builtin_bit_cast(i16x8_t, ld16(q + (d0 < c.d ? d0 : 0), row_ok && d0 < c.d));
    }
  }

  const u16* kc = (const u16*)c.k + (int64_t)kvh * c.head;
  const u16* vc = (const u16*)c.v + (int64_t)kvh * c.head;
  const bool has_new = p.k_new != nullptr;
  const u16* kn = (const u16*)p.k_new + (int64_t)bidb * p.kn_batch + (int64_t)kvh * p.kn_head;
  const u16* vn = (const u16*)p.v_new + (int64_t)bidb * p.vn_batch + (int64_t)kvh * p.vn_head;
  const int chunk = St::chunk(lane) * 8;
  const bool chunk_ok = chunk < c.d;
  bool bad = false;

  St st;
  // page of key (step, r) of this wave, looked up one step before its rows are loaded
  auto key_offset = [&](int step) -> int64_t {
    const int j = step * kStep + wave * 32 + r;
    return j < total ? slot_offset(c, bidb, j, bad) : 0;
  };
  auto load = [&](int step, int64_t off_r) {
    const int j0 = step * kStep + wave * 32;
    if (j0 + 32 <= (has_new ? len : total)) {      // all from the cache
#pragma unroll
      for (int i = 0; i < St::NI; ++i) {
        const int64_t off = shfl64(off_r, St::row(i, lane)) + chunk;
        st.k[i] = ld16(kc + off, chunk_ok);
        st.v[i] = ld16(vc + off, chunk_ok);
      }
    } else {
#pragma unroll
      for (int i = 0; i < St::NI; ++i) {
        const int jr = St::row(i, lane), j = j0 + jr;
        const int64_t off = shfl64(off_r, jr) + chunk;
        const bool fresh = has_new && j >= len;
        const u16* kp = fresh ? kn + (int64_t)(j - len) * p.kn_row + chunk : kc + off;
        const u16* vp = fresh ? vn + (int64_t)(j - len) * p.vn_row + chunk : vc + off;
        st.k[i] = ld16(kp, chunk_ok && j < total);
        st.v[i] = ld16(vp, chunk_ok && j < total);
      }
    }
  };
  bool found_odd = false;                          // wave-uniform
  char* const mine = smem + wave * 2 * TILE;       // [K rows][V rows] of this wave
  auto hand_over = [&](int step) {
#pragma unroll
    for (int i = 0; i < St::NI; ++i) {
      const int off = panel_off(St::row(i, lane), St::chunk(lane), 32);
      *(u32x4_t*)(mine + off) = st.k[i];
      *(u32x4_t*)(mine + TILE + off) = st.v[i];
    }
    if (step * kStep + wave * 32 + 32 > len) {     // drafted keys among them
      unsigned odd = 0;
#pragma unroll 1
      for (int i = lane; i < TILE / 8; i += 64) {  // (rare steps: through LDS, sparing the registers)
        u32x2_t* const x = (u32x2_t*)(mine + TILE) + i;
        const unsigned m0 = odd_pair<BF16>((*x)[0]), m1 = odd_pair<BF16>((*x)[1]);
        if (m0 | m1) *x = u32x2_t{(*x)[0] & ~m0, (*x)[1] & ~m1};
        odd |= m0 | m1;
      }
      found_odd = found_odd || __any(odd != 0);
    }
  };

  float m_run = kNegInf, l_run = 0.f;
  f32x16_t o[NP];
#pragma unroll
  for (int t = 0; t < NP; ++t)
#pragma unroll
    for (int g = 0; g < 16; ++g) o[t][g] = 0.f;
  const float cs = p.scale_log2;

  // whether token t sees key j (branch-free: every byte of a step is on its way before the first is used)
  auto sees = [&](int t, int j) {
    const int u = max(0, min(j - len, p.sq - 1));
    const bool drafted = p.mask ? p.mask[(int64_t)bidb * p.mask_batch + (int64_t)t * p.mask_row + u] != 0 : u <= t;
    return (j < total) & ((j < len) | drafted);
  };
  // one 32-key subtile in LDS: wave `sub`'s, first key j0
  auto compute = [&](int sub, int j0) {
    if (j0 >= total) return;
    const int tile = sub * 2 * TILE;
    const TileAddr ta(lb, tile);
    f32x16_t s;
#pragma unroll
    for (int g = 0; g < 16; ++g) s[g] = 0.f;
    static_for<0, KS>([&](auto K) {
      constexpr int ks = decltype(K)::value;
      s = E::mfma(row_read_c<32, 0, 2 * ks>(smem, ta), qf[ks], s);
    });
    if (j0 + 32 > len) {                           // drafted keys, or the end
#pragma unroll
      for (int g = 0; g < 16; ++g) {
        s[g] = sees(tok, j0 + acc_row(g, hh)) ? s[g] : kNegInf;
      }
    }
    float mt4[4] = {kNegInf, kNegInf, kNegInf, kNegInf};
#pragma unroll
    for (int g = 0; g < 16; ++g) mt4[g & 3] = fmaxf(mt4[g & 3], s[g]);
    const float m_new = fmaxf(m_run, half_swap_max(fmaxf(fmaxf(mt4[0], mt4[1]), fmaxf(mt4[2], mt4[3]))) * cs);
    if (__any(m_new != m_run)) {
      const float alpha = m_new == kNegInf ? 1.f : fast_exp2(m_run - m_new);
      l_run *= alpha;
#pragma unroll
      for (int t = 0; t < NP; ++t)
#pragma unroll
        for (int g = 0; g < 16; ++g) o[t][g] *= alpha;
      m_run = m_new;
    }
    const float ms = m_run == kNegInf ? 0.f : m_run;
    float ls[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int g = 0; g < 16; ++g) {
      s[g] = fast_exp2(fmaf(s[g], cs, -ms));
      ls[g & 3] += s[g];
    }
    l_run += (ls[0] + ls[1]) + (ls[2] + ls[3]);
    const i16x8_t p0 = pack_frag<BF16>(s, 0), p1 = pack_frag<BF16>(s, 1);
    const TileAddr tv(lb, tile + TILE);
    static_for<0, NP>([&](auto T) {
      constexpr int t = decltype(T)::value;
      o[t] = E::mfma(tr_frag_c<32, 0, t>(smem, tv), p0, o[t]);
      o[t] = E::mfma(tr_frag_c<32, 16, t>(smem, tv), p1, o[t]);
    });
  };

  if (s0 < s1) {
    load(s0, key_offset(s0));
    int64_t next_off = s0 + 1 < s1 ? key_offset(s0 + 1) : 0;
    for (int step = s0; step < s1; ++step) {
      hand_over(step);
      if (step + 1 < s1) {
        const int64_t off = next_off;
        if (step + 2 < s1) next_off = key_offset(step + 2);
        load(step + 1, off);
      }
      if constexpr (WM == 1) {
        __builtin_amdgcn_wave_barrier();           // the wave reads its own tile: LDS order suffices
        compute(wave, step * kStep + wave * 32);
        __builtin_amdgcn_wave_barrier();
      } else {
        lds_barrier();
#pragma unroll 1
        for (int t = 0; t < WM; ++t) {
          const int sub = wk * WM + t;
          compute(sub, step * kStep + sub * 32);
        }
        lds_barrier();
      }
    }
  }

  // ---- merge the WK waves that share rows: (m, l) and O through LDS, rows of D floats whose 16-byte
  // chunks are XORed with the row (32 lanes of one column then hit distinct banks) ----
  l_run = half_swap_sum(l_run);
  if constexpr (WM == 1) lds_barrier();            // every wave is done with its tiles
  constexpr int CH = D / 4;
  float* osm = (float*)smem + wave * 32 * D;
#pragma unroll
  for (int t = 0; t < NP; ++t)
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const int ch = t * 8 + 2 * q + hh;           // columns 32 t + 8 q + 4 hh ..
      f32x4_t x;
#pragma unroll
      for (int e = 0; e < 4; ++e) x[e] = o[t][4 * q + e];
      *(f32x4_t*)(osm + r * D + ((ch ^ (r & (CH - 1))) << 2)) = x;
    }
  if (hh == 0) { sm_m[wave][r] = m_run; sm_l[wave][r] = l_run; }
  const bool any_bad = __any(bad);
  if (lane == 0) { sm_bad[wave] = any_bad; sm_odd[wave] = found_odd; }
  lds_barrier();

  const int rows_here = min(32 * WM, p.rows - mt * WM * 32);
  for (int i = tid; i < rows_here * CH; i += 256) {
    const int rl = i / CH, ch = i - rl * CH;
    const int w0 = rl >> 5, rr = rl & 31;          // waves w0, w0 + WM, ... hold the row
    float m = kNegInf, l = 0.f;
#pragma unroll
    for (int k = 0; k < WK; ++k) m = fmaxf(m, sm_m[w0 + k * WM][rr]);
    f32x4_t acc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int k = 0; k < WK; ++k) {
      const int w = w0 + k * WM;
      const float f = m == kNegInf ? 0.f : fast_exp2(sm_m[w][rr] - m);
      l += f * sm_l[w][rr];
      const f32x4_t x = *(const f32x4_t*)((const float*)smem + w * 32 * D + rr * D + ((ch ^ (rr & (CH - 1))) << 2));
#pragma unroll
      for (int e = 0; e < 4; ++e) acc[e] += f * x[e];
    }
    if (!ok_seq || (sm_bad[0] | sm_bad[1] | sm_bad[2] | sm_bad[3])) l = __builtin_nanf("");
    const float inv = l == 0.f ? 0.f : 1.f / l;
#pragma unroll
    for (int e = 0; e < 4; ++e) acc[e] *= inv;
    const int rg = mt * WM * 32 + rl;
    if (sm_odd[0] | sm_odd[1] | sm_odd[2] | sm_odd[3]) {
      const int t = rg / p.group;
      for (int j = max(len, s0 * kStep); j < min(total, s1 * kStep); ++j) {
        bool out = false;
        const u16* v = has_new ? vn + (int64_t)(j - len) * p.vn_row : vc + slot_offset(c, bidb, j, out);
        if (ch * 4 >= c.d || !sees(t, j)) continue;
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (odd_pair<BF16>(v[ch * 4 + e])) acc[e] += E::to_f32(v[ch * 4 + e]);
      }
    }
    if (l != l) acc[0] = acc[1] = acc[2] = acc[3] = l;
    const float lse2 = l == 0.f ? kNegInf : m + __log2f(l);
    if (p.splits > 1) {
      const int64_t at = ((int64_t)bh * p.splits + split) * p.rows + rg;
      if (ch * 4 < c.d) *(f32x4_t*)(p.part_o + at * c.d + ch * 4) = acc;
      if (ch == 0) p.part_lse[at] = lse2;
    } else {
      const int t = rg / p.group, head = kvh * p.group + rg - t * p.group;
      if (ch * 4 < c.d) {
        u32x2_t u = {E::pack2(acc[0], acc[1]), E::pack2(acc[2], acc[3])};
        *(u32x2_t*)((u16*)p.o + (int64_t)bidb * p.o_batch + (int64_t)t * p.o_row + (int64_t)head * p.o_head + ch * 4) = u;
      }
      if (ch == 0) p.lse[((int64_t)bidb * p.h + head) * p.sq + t] = l == 0.f ? -kNegInf : lse2 * kLn2;
    }
  }

  // ---- append the drafted keys of this split (nobody reads their slots: rows come from k_new) ----
  if (has_new && mt == 0 && ok_seq) {
    const int first = max(len, s0 * kStep), last = min(total, s1 * kStep);
    const int cpr = c.d / 8;
    for (int i = tid; i < (last - first) * cpr; i += 256) {
      const int jr = i / cpr, ch = (i - jr * cpr) * 8, j = first + jr;
      bool out = false;
      const int64_t off = slot_offset(c, bidb, j, out) + ch;
      if (out) continue;
      *(u32x4_t*)((u16*)c.k + (int64_t)kvh * c.head + off) = *(const u32x4_t*)(kn + (int64_t)(j - len) * p.kn_row + ch);
      *(u32x4_t*)((u16*)c.v + (int64_t)kvh * c.head + off) = *(const u32x4_t*)(vn + (int64_t)(j - len) * p.vn_row + ch);
    }
  }
}

// Merges the splits of one row: one workgroup a row, D / 4 lanes of 4 columns x the splits dealt to
// the 256 / (D / 4) lane groups, then a tree over the groups in LDS.
template <bool BF16, int D>
__global__ void __launch_bounds__(256) kv_merge_kernel(const KvAttnParams p) {
  using E = Elt<BF16>;
  constexpr int CH = D / 4, GROUPS = 256 / CH;
  const KvCache& c = p.c;
  const int row = blockIdx.x % p.rows, bh = blockIdx.x / p.rows;
  const int bidb = bh / c.hk, kvh = bh - bidb * c.hk;
  const int t = row / p.group, head = kvh * p.group + row - t * p.group;
  const int ch = threadIdx.x % CH, grp = threadIdx.x / CH;
  const int len = c.lens[bidb];
  const bool ok_seq = seq_ok(c, len, p.sq);
  const int steps = ok_seq ? (len + p.sq + kStep - 1) / kStep : 0;
  const int per_split = (steps + p.splits - 1) / p.splits;
  const int live = per_split > 0 ? (steps + per_split - 1) / per_split : 0;

  const float* pl = p.part_lse + (int64_t)bh * p.splits * p.rows + row;
  float m = kNegInf;
  for (int s = threadIdx.x & 63; s < live; s += 64) m = fmaxf(m, pl[(int64_t)s * p.rows]);
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) m = fmaxf(m, __shfl_xor(m, off));
  float l = 0.f;
  f32x4_t acc = {0.f, 0.f, 0.f, 0.f};
  for (int s = grp; s < live; s += GROUPS) {
    const float x = pl[(int64_t)s * p.rows];
    const float f = x == kNegInf ? 0.f : fast_exp2(x - m);   // NaN stays
    l += f;
    if (ch * 4 < c.d) {
      const f32x4_t v = *(const f32x4_t*)(p.part_o + (((int64_t)bh * p.splits + s) * p.rows + row) * c.d + ch * 4);
#pragma unroll
      for (int e = 0; e < 4; ++e) acc[e] += f * v[e];
    }
  }
  __shared__ float sl[GROUPS];
  __shared__ f32x4_t sa[GROUPS][CH];
  if (ch == 0) sl[grp] = l;
  sa[grp][ch] = acc;
  __syncthreads();
  if (grp != 0) return;
#pragma unroll
  for (int g = 1; g < GROUPS; ++g) {
    l += sl[g];
    const f32x4_t v = sa[g][ch];
#pragma unroll
    for (int e = 0; e < 4; ++e) acc[e] += v[e];
  }
  if (!ok_seq) l = __builtin_nanf("");
  const float inv = l == 0.f ? 0.f : 1.f / l;
  if (ch * 4 < c.d) {
    u32x2_t u = {E::pack2(acc[0] * inv, acc[1] * inv), E::pack2(acc[2] * inv, acc[3] * inv)};
    *(u32x2_t*)((u16*)p.o + (int64_t)bidb * p.o_batch + (int64_t)t * p.o_row + (int64_t)head * p.o_head + ch * 4) = u;
  }
  if (ch == 0) p.lse[((int64_t)bidb * p.h + head) * p.sq + t] = l == 0.f ? -kNegInf : (m + __log2f(l)) * kLn2;
}

// weight[b][kvh][j] += sum over the kv head's rows of exp(scale q k_j - LSE): 32 keys a wave, the key on
// the lane (S = Q K^T), so the sum over rows is lane-local.  One owner a key: no atomics.
template <bool BF16, int D>
__global__ void __launch_bounds__(256) kv_weight_kernel(const KvAttnParams p) {
  using E = Elt<BF16>;
  constexpr int KS = D / 16;
  const KvCache& c = p.c;
  const int lane = threadIdx.x & 63, wave = wave_uniform(threadIdx.x >> 6);
  const int r = lane & 31, hh = lane >> 5;
  const int bh = blockIdx.x, bidb = bh / c.hk, kvh = bh - bidb * c.hk;
  const int len = c.lens[bidb];
  if (!seq_ok(c, len, p.sq)) return;
  const int total = len + p.sq, j0 = blockIdx.y * 128 + wave * 32;
  if (j0 >= total) return;
  const int j = j0 + r;
  bool bad = false;
  const int64_t off = (j < total ? slot_offset(c, bidb, j, bad) : 0) + (int64_t)kvh * c.head;
  i16x8_t kf[KS];
#pragma unroll
  for (int ks = 0; ks < KS; ++ks) {
    const int d0 = 16 * ks + 8 * hh;
    kf[ks] = __builtin_bit_cast(i16x8_t, ld16((const u16*)c.k + off + (d0 < c.d ? d0 : 0), j < total && d0 < c.d));
  }
  float sum = 0.f;
  for (int row0 = 0; row0 < p.rows; row0 += 32) {
    const int row = row0 + r;
    const bool ok = row < p.rows;
    const int tok = (ok ? row : 0) / p.group, head = kvh * p.group + (ok ? row : 0) - tok * p.group;
    const u16* q = (const u16*)p.q + (int64_t)bidb * p.q_batch + (int64_t)tok * p.q_row + (int64_t)head * p.q_head;
    f32x16_t s;
#pragma unroll
    for (int g = 0; g < 16; ++g) s[g] = 0.f;
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) {
      const int d0 = 16 * ks + 8 * hh;
      s = E::mfma(__builtin_bit_cast(i16x8_t, ld16(q + (d0 < c.d ? d0 : 0), ok && d0 < c.d)), kf[ks], s);
    }
    const float lse = ok ? p.lse[((int64_t)bidb * p.h + head) * p.sq + tok] * kLog2e : 0.f;
#pragma unroll
    for (int g = 0; g < 16; ++g) {
      const int rr = acc_row(g, hh), rg = row0 + rr;
      const float le = __shfl(lse, rr);
      bool see = rg < p.rows;
      if (j0 + 32 > len) {                         // drafted keys, or the end
        const int tk = min(rg, p.rows - 1) / p.group, u = max(0, min(j - len, p.sq - 1));
        const bool drafted = p.mask ? p.mask[(int64_t)bidb * p.mask_batch + (int64_t)tk * p.mask_row + u] != 0 : u <= tk;
        see = see & (j < total) & ((j < len) | drafted);
      }
      sum += see ? fast_exp2(fmaf(s[g], p.scale_log2, -le)) : 0.f;
    }
  }
  sum = half_swap_sum(sum);
  if (hh == 0 && j < total) p.weight[(int64_t)bidb * p.w_batch + (int64_t)kvh * p.w_head + j] += sum;
}

// Rows tiles of 32 WM and key splits: enough workgroups for several rounds of the chip's 512 resident
// ones (ragged sequences then balance), at least two steps each so that loads run ahead.
static int rows_per_block(int rows) { return rows <= 32 ? 32 : rows <= 64 ? 64 : 128; }

void kv_attn_plan(KvAttnParams& p) {
  const int per = rows_per_block(p.rows);
  p.m_tiles = (p.rows + per - 1) / per;
  const int64_t base = (int64_t)p.c.b * p.c.hk * p.m_tiles;
  const int64_t most = (p.c.slots + 2 * kStep - 1) / (2 * kStep);
  const int64_t want = (2048 + base - 1) / base;
  p.splits = (int)std::max<int64_t>(1, std::min(most, want));
}

size_t kv_attn_workspace(const KvAttnParams& p) {
  if (p.splits <= 1) return 0;
  return (size_t)p.c.b * p.c.hk * p.splits * p.rows * (size_t)(p.c.d + 1) * sizeof(float);
}

template <bool BF16, int D>
static void run_attn(const KvAttnParams& p, hipStream_t stream) {
  const int64_t units = (int64_t)p.c.b * p.c.hk * p.splits;
  const int64_t grid = (units + 7) / 8 * 8 * p.m_tiles;
  if (grid > 0x7fffffff) throw std::runtime_error("kvcache attention: too many workgroups for one launch");
  const dim3 g((unsigned)grid), t(256);
  switch (rows_per_block(p.rows)) {
    case 32: hipLaunchKernelGGL((kv_attn_kernel<BF16, D, 1>), g, t, 0, stream, p); break;
    case 64: hipLaunchKernelGGL((kv_attn_kernel<BF16, D, 2>), g, t, 0, stream, p); break;
    default: hipLaunchKernelGGL((kv_attn_kernel<BF16, D, 4>), g, t, 0, stream, p); break;
  }
  if (p.splits > 1)
    hipLaunchKernelGGL((kv_merge_kernel<BF16, D>), dim3((unsigned)(p.c.b * p.c.hk * p.rows)), t, 0, stream, p);
  if (p.weight != nullptr)
    hipLaunchKernelGGL((kv_weight_kernel<BF16, D>), dim3((unsigned)(p.c.b * p.c.hk), (unsigned)((p.c.slots + 127) / 128)), t,
                       0, stream, p);
}

template <bool BF16>
static void dispatch_attn(const KvAttnParams& p, hipStream_t stream) {
  if (p.c.d <= 64) run_attn<BF16, 64>(p, stream);
  else if (p.c.d <= 128) run_attn<BF16, 128>(p, stream);
  else run_attn<BF16, 256>(p, stream);
}

static void check_launch(const char* what) {
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) throw std::runtime_error(std::string(what) + " launch: " + hipGetErrorString(e));
}

void launch_kv_attn(KvAttnParams p, void* workspace, bool is_bf16, hipStream_t stream) {
  if (p.splits > 1) {
    p.part_o = (float*)workspace;
    p.part_lse = p.part_o + (int64_t)p.c.b * p.c.hk * p.splits * p.rows * p.c.d;
  }
  if (is_bf16) dispatch_attn<true>(p, stream);
  else dispatch_attn<false>(p, stream);
  check_launch("kvcache attention");
}

}  // namespace fa
