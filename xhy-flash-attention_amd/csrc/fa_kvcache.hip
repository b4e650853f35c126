// Attention of drafted tokens over a key/value cache (gfx950): sq rows a sequence (1: plain decoding).
//
// Row i of sequence b sees the lens[b] cached keys and, of the sq drafted keys behind them, those its
// mask row names (without a mask: drafted keys 0 .. i).  O = softmax(scale q k) v, LSE = its logarithm.
//
// MI355X mapping.  With few rows the call is bound by reading K and V once, and the lengths are known on
// the device only, so the work is dealt out there:
//   * the G query heads of a kv head and the sq tokens are packed as rows (row = token G + head), so a
//     kv head's K/V is read once for all of them; a unit is (sequence, kv head, 32 WM rows), WM = 1, 2, 4;
//   * a step is 128 keys.  The steps of all sequences, in order, are cut into equal shares, and a share
//     has one resident workgroup for every kv head and row tile: whatever the lengths, every CU streams the
//     same number of bytes, and the heads of a key, neighbours in memory, are read at the same time.  A
//     workgroup walks the pieces of sequences in its share; a unit that lies in one share is written at
//     once, the pieces of the others go through fp32 partials and a merge kernel;
//   * a wave loads its 32 keys of a step (K and V rows, 16 bytes a lane) one step ahead into
//     registers: range-checked loads off a wave-uniform row base when the 32 keys are evenly strided (a
//     cache without pages, or pages of whole 32 keys), else one address a lane.  It hands them over through
//     its own LDS tile, which MFMA operands are then read from (row reads for K, transposing reads for V);
//   * WM = 1: the four waves take different keys and no barrier is needed; WM = 4: they take
//     different rows of the same 128 keys; WM = 2: two by two.  Waves that share rows merge their
//     (max, sum, O) through LDS at the end of a piece;
//   * S^T = K Q^T and O^T = V^T P^T as in fa_fwd.hip: a lane holds one row, so the softmax is lane-local
//     plus one half swap, and P is the next product's operand without moving;
//   * attention weights: with few rows (rows <= d / 4) the kernel also stores each key's scores, fp32 (a
//     row's 4 bytes a key against the 4 d of its K and V), and the merge launch turns them into
//     probabilities once the LSE is known; with more rows K is read again (kv_weight_kernel).
// P is rounded to 16 bits for the product with V (half a step of the type relative to each weight;
// the sum that divides is of the unrounded P); scores, statistics, O and the partials are fp32.
//
// A row's result depends on what it sees alone: non-finite values of a drafted V row, which the product
// would multiply by the zero weights of the rows that do not see it, are taken out of the tile and
// added, times their weight, to the rows that do (a rare path, looked for in steps with drafted keys, and gone
// for keys that some row of the unit does not see: a tree's, or those around a prompt's diagonal).
// Keys past a sequence's end load as zeros, so no slot behind it reaches a result.  A sequence whose
// length does not leave room for the drafted tokens, or that names a page outside the cache, gives NaN.
//
// Measured, 32 / 8 heads of 128: 8 sequences of 20k to 32k keys with weights 201 + 13 us (4.5 TB/s of K and V; a
// step's hand-over through LDS and its products keep a workgroup from more); 4k keys of one sequence 13 + 4 us
// (latency: one key takes 11.8, by three reads of the lengths, Q, the keys, LDS and the merge one after another); 48
// drafted tokens over 16 sequences of up to 8k keys in pages of 64: 164 + 12 us under the profiler, 146 in all
// without it (softmax and products of 96-row tiles: the fourth wave stages keys only).  A prompt is slow here: 8192
// tokens 20.5 ms, against 0.42 of the causal forward (all keys for every row tile, and one share is one XCD).
#include <algorithm>
#include <stdexcept>
#include <string>

#include "fa_kvcache.h"

namespace fa {

typedef unsigned short u16;
static constexpr int kStep = 128;       // keys a workgroup takes at a time, 32 a wave
static constexpr int kScoreRows = 32;   // most rows whose scores are stored for the attention weights
static constexpr int kFar = 0x7ffffff0;   // a byte offset outside every range-checked load

__device__ inline int64_t shfl64(int64_t x, int lane) {
  const unsigned lo = (unsigned)__shfl((int)(unsigned)x, lane), hi = (unsigned)__shfl((int)(x >> 32), lane);
  return (int64_t)(((uint64_t)hi << 32) | lo);
}

// (readfirstlane on both parts: what the compiler cannot prove uniform it would load lane group by group)
__device__ inline buf_rsrc_t uniform_rsrc(const void* base, int bytes) {
  return make_rsrc(uniform_ptr((const char*)base), wave_uniform(bytes));
}
__device__ inline u32x4_t load16(buf_rsrc_t r, int off) {
  return __builtin_bit_cast(u32x4_t, __builtin_amdgcn_raw_buffer_load_b128(r, off, 0, 0));
}

// ---- the shares ----
// Steps of a sequence: its keys in kStep's; one, without keys, where the length is none (the units then
// write NaN)
__device__ inline int seq_steps(const KvAttnParams& p, int len) {
  return seq_ok(p.c, len, p.sq) ? (len + p.sq + kStep - 1) / kStep : 1;
}
// What a wave's scan over the lengths tells of the shares
struct Shares {
  int total, share;   // steps of all sequences, and of a share
  __device__ inline Shares(const KvAttnParams& p, int lane) {
    total = before(p, lane, p.c.b);
    share = wave_uniform((total + p.shares - 1) / p.shares);
  }
  // steps before sequence b
  static __device__ inline int before(const KvAttnParams& p, int lane, int b) {
    int sum = 0;
    for (int i = lane; i < b; i += 64) sum += seq_steps(p, p.c.lens[i]);
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) sum += __shfl_xor(sum, off);
    return wave_uniform(sum);
  }
  // the sequence of step `at` < total, and the steps before it
  static __device__ inline int find(const KvAttnParams& p, int lane, int at, int& seq_at) {
    seq_at = 0;
    for (int b0 = 0;; b0 += 64) {
      const int b = b0 + lane;
      int x = b < p.c.b ? seq_steps(p, p.c.lens[b]) : 0;
      const int own = x;
#pragma unroll
      for (int off = 1; off < 64; off <<= 1) {
        const int y = __shfl_up(x, off);
        if (lane >= off) x += y;
      }
      const uint64_t m = __ballot(seq_at + x > at);
      if (m != 0) {
        const int l = __builtin_ctzll(m);
        seq_at = wave_uniform(seq_at + __shfl(x - own, l));
        return wave_uniform(b0 + l);
      }
      seq_at += wave_uniform(__shfl(x, 63));
    }
  }
};

// A wave's 32 K and V rows in flight: lane -> (row, 16-byte chunk), whole rows one after another.
// NR: the panels of the LDS tile are shifted against each other by 64 bytes (128 at two panels), so that the
// 16 lanes of a row, or of two, write to distinct banks; reads stay within a panel.
template <int D>
struct Stage {
  static constexpr int CPR = D / 8, RPI = 64 / CPR, NI = 32 / RPI, NR = D == 64 ? 34 : 33;
  static constexpr int TILE = D / 32 * NR * 64;   // bytes
  u32x4_t k[NI], v[NI];
  static __device__ inline int row(int i, int lane) { return i * RPI + lane / CPR; }
  static __device__ inline int chunk(int lane) { return lane % CPR; }
};

// four operands in registers at this point: without it the scheduler reads each from LDS right before its
// product and waits for it there
__device__ inline void keep4(i16x8_t& a, i16x8_t& b, i16x8_t& c, i16x8_t& d) {
  asm volatile("" : "+v"(a), "+v"(b), "+v"(c), "+v"(d));
}

// infinities and NaN of two packed elements
template <bool BF16>
__device__ inline unsigned odd_pair(unsigned u) {
  constexpr unsigned m = BF16 ? 0x7f80u : 0x7c00u;
  return ((u & m) == m ? 0xffffu : 0u) | ((u & (m << 16)) == (m << 16) ? 0xffff0000u : 0u);
}

// The first drafted key that some row of the unit does not see, rounded down to a tile of 32 keys (without a mask
// the unit's first token sees the drafted keys up to itself)
__device__ inline int first_hidden(const KvAttnParams& p, int len, int mt) {
  return max(len, p.mask != nullptr ? len : (len + mt * p.tile_rows / p.group + 1) & ~31);
}

// Workgroups a CU, and steps in flight.  Few rows: one workgroup of up to 512 registers a wave and two
// steps; row tiles that are bound by the softmax and the products want two waves a SIMD instead.  (8
// sequences of 26k keys, 32 / 8 heads of 128: 205 us, against 218 with two workgroups of one step each, and
// 219 with one workgroup of eight waves.)
constexpr int groups_per_cu(int d, int wm) { return d <= 128 && wm > 1 ? 2 : 1; }
constexpr int steps_ahead(int d, int wm) { return d <= 128 && wm == 1 ? 2 : 1; }

template <bool BF16, int D, int WM>
__global__ void __launch_bounds__(256, groups_per_cu(D, WM)) kv_attn_kernel(const KvAttnParams p) {
  using E = Elt<BF16>;
  using St = Stage<D>;
  constexpr int KS = D / 16, NP = D / 32, WK = 4 / WM;
  constexpr int TILE = St::TILE, NR = St::NR;      // one wave's K (or V) rows
  constexpr int CH = D / 4;
  __shared__ __attribute__((aligned(16))) char smem[4 * 2 * TILE];
  __shared__ float sm_m[4][32], sm_l[4][32];
  __shared__ int sm_bad[4], sm_odd[4];
  const KvCache& c = p.c;
  const int tid = threadIdx.x, lane = tid & 63, wave = wave_uniform(tid >> 6);
  const int r = lane & 31, hh = lane >> 5;
  const LdsBases lb(lane);
  const int wm = wave % WM, wk = wave / WM;
  const float cs = p.scale_log2;
  const bool has_new = p.k_new != nullptr;
  const int chunk = St::chunk(lane) * 8;
  const bool chunk_ok = chunk < c.d;
  char* const mine = smem + wave * 2 * TILE;       // [K rows][V rows] of this wave

  // The units of a share sit 8 workgroups apart, on one XCD: the heads of a key, neighbours in memory, then
  // spread over all channels of its L2 (one head an XCD would use one in hk of them), and the row tiles
  // of a head read K/V through the same L2
  const int units = c.hk * p.m_tiles;
  const int oct = (blockIdx.x >> 3) / units, unit = (blockIdx.x >> 3) - oct * units;
  const int share = oct * 8 + (blockIdx.x & 7);
  const int mt = unit / c.hk, kvh = unit - mt * c.hk;
  if (share >= p.shares) return;                   // (of the last eight)
  const Shares sh(p, lane);
  int at = share * sh.share;
  const int end = min(sh.total, at + sh.share);
  if (at >= end) return;
  int seq_at;
  int bidb = Shares::find(p, lane, at, seq_at);

  while (at < end) {
    // ---- the piece: steps [s0, s1) of sequence bidb ----
    const int len = wave_uniform(c.lens[bidb]);    // (all of this is: the loads' row bases are scalar)
    const int steps = seq_steps(p, len);
    const int s0 = at - seq_at, s1 = min(steps, s0 + end - at);
    const bool ok_seq = seq_ok(c, len, p.sq);
    const int total = ok_seq ? len + p.sq : 0;
    const int old = has_new ? min(len, total) : total;   // keys that come from the cache
    const int bh = bidb * c.hk + kvh;

    const int rows_here = min(p.tile_rows, p.rows - mt * p.tile_rows);
    const int row = mt * p.tile_rows + wm * 32 + r;   // this lane's row
    const bool row_ok = wm * 32 + r < rows_here;
    const int tok = row_ok ? row / p.group : 0, gh = row_ok ? row - tok * p.group : 0;

    i16x8_t qf[KS];
    {
      const buf_rsrc_t rq = uniform_rsrc((const u16*)p.q + (int64_t)bidb * p.q_batch + (int64_t)kvh * p.group * p.q_head, kFar);
      const int q0 = row_ok ? (int)(tok * p.q_row + gh * p.q_head) * 2 + 16 * hh : kFar;
#pragma unroll
      for (int ks = 0; ks < KS; ++ks)
        qf[ks] = __builtin_bit_cast(i16x8_t, load16(rq, 16 * ks + 8 * hh < c.d ? q0 + 32 * ks : kFar));
    }

    const u16* kc = (const u16*)c.k + (int64_t)kvh * c.head;
    const u16* vc = (const u16*)c.v + (int64_t)kvh * c.head;
    const u16* kn = (const u16*)p.k_new + (int64_t)bidb * p.kn_batch + (int64_t)kvh * p.kn_head;
    const u16* vn = (const u16*)p.v_new + (int64_t)bidb * p.vn_batch + (int64_t)kvh * p.vn_head;
    bool bad = false, found_odd = false;

    const int row_off = chunk_ok ? (St::row(0, lane) * (int)c.row + chunk) * 2 : (1 << 31);
    constexpr int DEPTH = steps_ahead(D, WM);
    St stage[DEPTH];
    // the wave's keys of a step: where the first one's row is (even strides), or lane r's row is
    auto locate = [&](int step) -> int64_t {
      const int j = step * kStep + wave * 32 + (p.even ? 0 : r);
      return j < total ? slot_offset(c, bidb, j, bad) : 0;
    };
    // plain: the step's 32 keys of the wave are evenly strided rows of the cache; the range check zeroes
    // rows past the end and chunks past d.  Else (drafted keys among them, or odd pages) every lane has
    // a valid address of its own and hand_over zeroes.
    auto plain = [&](int j0) { return p.even && (j0 + 32 <= old || !has_new); };
    auto load = [&](St& st, int step, int64_t where) {
      const int j0 = step * kStep + wave * 32;
      if (plain(j0)) {
        const int64_t base = uniform64(where);
        const int bytes = max(0, min(32, total - j0)) * (int)c.row * 2;
        const buf_rsrc_t rk = uniform_rsrc(kc + base, bytes), rv = uniform_rsrc(vc + base, bytes);
        int off = opaque(row_off);                 // (opaque: no register kept for each offset)
#pragma unroll
        for (int i = 0; i < St::NI; ++i) {
          st.k[i] = load16(rk, off);
          st.v[i] = load16(rv, off);
          off += St::RPI * (int)c.row * 2;
        }
      } else {
        const int ln = opaque(lane), ck = chunk_ok ? chunk : 0;
        int64_t at_row[St::NI];                    // (all looked up before the first load)
        if (p.even) {
#pragma unroll
          for (int i = 0; i < St::NI; ++i) at_row[i] = where + (j0 + St::row(i, ln) < len ? St::row(i, ln) * c.row : 0);
        } else {
#pragma unroll
          for (int i = 0; i < St::NI; ++i) at_row[i] = shfl64(where, St::row(i, ln));
        }
#pragma unroll
        for (int i = 0; i < St::NI; ++i) {
          const int u = j0 + St::row(i, ln) - len;
          const int64_t off = at_row[i] + ck;
          const int64_t fresh = has_new && u >= 0 ? -1 : 0;   // (selected by bits: no branches)
          const int64_t uc = min(max(u, 0), p.sq - 1);
          const int64_t ka = (int64_t)(kc + off), kb = (int64_t)(kn + uc * p.kn_row + ck);
          const int64_t va = (int64_t)(vc + off), vb = (int64_t)(vn + uc * p.vn_row + ck);
          st.k[i] = *(const u32x4_t*)(ka ^ ((ka ^ kb) & fresh));
          st.v[i] = *(const u32x4_t*)(va ^ ((va ^ vb) & fresh));
        }
      }
    };
    auto hand_over = [&](St& st, int step) {
      const int j0 = step * kStep + wave * 32;
      const int ln = opaque(lane);
      unsigned odd = 0;
      if (plain(j0) && j0 + 32 <= len) {
#pragma unroll
        for (int i = 0; i < St::NI; ++i) {
          const int off = panel_off(St::row(i, ln), St::chunk(ln), NR);
          *(u32x4_t*)(mine + off) = st.k[i];
          *(u32x4_t*)(mine + TILE + off) = st.v[i];
        }
      } else {
#pragma unroll
        for (int i = 0; i < St::NI; ++i) {
          const int off = panel_off(St::row(i, ln), St::chunk(ln), NR);
          const unsigned keep = chunk_ok && j0 + St::row(i, ln) < total ? ~0u : 0u;
          // (cached keys' values may take the path below, too, where it changes nothing for them.  Asking first: tree
          // of 48 over 16 x 8k keys 148 us, 157 without; at d = 256 it spills: decoding 8 x 26k keys 617, 441 without)
          const unsigned drafted = D == 256 || j0 + St::row(i, ln) >= len ? ~0u : 0u;
          u32x4_t kx, vx;
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            kx[e] = st.k[i][e] & keep;
            vx[e] = st.v[i][e] & keep;
            odd |= odd_pair<BF16>(vx[e]) & drafted;
          }
          *(u32x4_t*)(mine + off) = kx;
          *(u32x4_t*)(mine + TILE + off) = vx;
        }
        if (__builtin_expect(j0 + 32 > len && __any(odd != 0), 0)) {    // (rare: through LDS, sparing the registers)
          found_odd = true;
          const int first = first_hidden(p, len, opaque(mt));
#pragma unroll 1
          for (int i = lane; i < D / 32 * 256; i += 64) {   // 256 pairs of words a panel, 8 a row
            if (j0 + ((i & 255) >> 3) < first) continue;
            u32x2_t* const x = (u32x2_t*)(mine + TILE + (i >> 8) * NR * 64) + (i & 255);
            *x = u32x2_t{(*x)[0] & ~odd_pair<BF16>((*x)[0]), (*x)[1] & ~odd_pair<BF16>((*x)[1])};
          }
        }
      }
    };

    float m_run = kNegInf, l_run = 0.f;
    f32x16_t o[NP];
#pragma unroll
    for (int t = 0; t < NP; ++t)
#pragma unroll
      for (int g = 0; g < 16; ++g) o[t][g] = 0.f;
    const buf_rsrc_t score_rsrc =
        uniform_rsrc(p.scores != nullptr ? p.scores + (int64_t)bh * p.rows * p.score_pitch : p.lse,
                  p.scores != nullptr ? (int)(p.rows * p.score_pitch * 4) : 0);

    // whether token t sees key j: its mask byte (branch-free; keys that are not drafted are asked for too, and
    // read nothing), and what to make of it
    const buf_rsrc_t rmask = uniform_rsrc(p.mask + (int64_t)bidb * p.mask_batch,
                                          p.mask != nullptr ? mask_bytes(p.sq, (int)p.mask_row) : 0);
    auto mask_byte = [&](int t, int j) {
      return (unsigned)__builtin_amdgcn_raw_buffer_load_b8(rmask, mask_offset(t, j, len, total, (int)p.mask_row, kFar), 0, 0);
    };
    auto sees = [&](int t, int j, unsigned byte) {
      return (j < total) & ((j < len) | (byte != 0) | ((p.mask == nullptr) & (j - len <= t)));
    };
    // one 32-key subtile in LDS: wave `sub`'s, first key j0
    auto compute = [&](int sub, int j0) {
      if (WM > 1 && (j0 >= total || wm * 32 >= rows_here)) return;   // (WM = 1: every step stores, see below)
      const int tile = sub * 2 * TILE;
      const TileAddr ta(lb, tile);
      f32x16_t s;
#pragma unroll
      for (int g = 0; g < 16; ++g) s[g] = 0.f;
      static_for<0, KS / 4>([&](auto K) {          // four operands on their way, then their products
        constexpr int k0 = decltype(K)::value * 4;
        i16x8_t ka[4];
        static_for<0, 4>([&](auto I) { ka[decltype(I)::value] = row_read_c<NR, 0, 2 * (k0 + decltype(I)::value)>(smem, ta); });
        keep4(ka[0], ka[1], ka[2], ka[3]);
#pragma unroll
        for (int i = 0; i < 4; ++i) s = E::mfma(ka[i], qf[k0 + i], s);
      });
      if (j0 + 32 > len) {                         // drafted keys, or the end
        unsigned byte[16];
#pragma unroll
        for (int g = 0; g < 16; ++g) byte[g] = mask_byte(tok, j0 + acc_row(g, hh));
#pragma unroll
        for (int g = 0; g < 16; ++g) asm volatile("" : "+v"(byte[g]));   // all on their way first
#pragma unroll
        for (int g = 0; g < 16; ++g) s[g] = sees(tok, j0 + acc_row(g, hh), byte[g]) ? s[g] : kNegInf;
      }
      if constexpr (WM == 1) {
        // Range-checked, and in every step: with no scores to store, or no keys, every lane is out of range.
        // The counted waits for the next step's loads, issued before these, then leave the stores in
        // flight; behind a branch they would have to wait for them too.
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const f32x4_t x = {s[4 * q] * cs, s[4 * q + 1] * cs, s[4 * q + 2] * cs, s[4 * q + 3] * cs};
          __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4_t, x), score_rsrc,
                                                 row_ok && j0 < total ? (int)((row * p.score_pitch + j0 + 4 * hh + 8 * q) * 4) : kFar,
                                                 0, 0);
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
      static_for<0, NP / 2>([&](auto T) {
        constexpr int t = decltype(T)::value * 2;
        i16x8_t v0 = tr_frag_c<NR, 0, t>(smem, tv), v1 = tr_frag_c<NR, 0, t + 1>(smem, tv);
        i16x8_t v2 = tr_frag_c<NR, 16, t>(smem, tv), v3 = tr_frag_c<NR, 16, t + 1>(smem, tv);
        keep4(v0, v1, v2, v3);
        o[t] = E::mfma(v0, p0, o[t]);
        o[t + 1] = E::mfma(v1, p0, o[t + 1]);
        o[t] = E::mfma(v2, p1, o[t]);
        o[t + 1] = E::mfma(v3, p1, o[t + 1]);
      });
    };

    // one step: its rows to LDS, those of step + DEPTH on their way, and the products
    auto advance = [&](St& st, int step, int64_t& next) {
      hand_over(st, step);
      if (step + DEPTH < s1) {
        const int64_t where = next;
        if (step + DEPTH + 1 < s1) next = locate(step + DEPTH + 1);   // looked up before the loads in between
        load(st, step + DEPTH, where);
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
    };
    if (ok_seq) {
      load(stage[0], s0, locate(s0));
      if constexpr (DEPTH == 2) {
        wait_vmem_all();   // Q counts as landed: no wait for it inside the loop, where later loads are in flight
        if (s0 + 1 < s1) load(stage[1], s0 + 1, locate(s0 + 1));
        int64_t next = s0 + 2 < s1 ? locate(s0 + 2) : 0;
#pragma unroll 1
        for (int step = s0; step < s1; step += 2) {
          advance(stage[0], step, next);
          if (step + 1 < s1) advance(stage[1], step + 1, next);
        }
      } else {
        int64_t next = s0 + 1 < s1 ? locate(s0 + 1) : 0;
        wait_vmem_all();   // (as above)
#pragma unroll 1
        for (int step = s0; step < s1; ++step) advance(stage[0], step, next);
      }
    }

    // ---- merge the WK waves that share rows: (m, l) and O through LDS, rows of D floats whose 16-byte
    // chunks are XORed with the row (32 lanes of one column then hit distinct banks) ----
    l_run = half_swap_sum(l_run);
    if constexpr (WM == 1) lds_barrier();          // every wave is done with its tiles
    float* osm = (float*)smem + wave * 32 * D;
#pragma unroll
    for (int t = 0; t < NP; ++t)
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const int ch = t * 8 + 2 * q + hh;         // columns 32 t + 8 q + 4 hh ..
        f32x4_t x;
#pragma unroll
        for (int e = 0; e < 4; ++e) x[e] = o[t][4 * q + e];
        *(f32x4_t*)(osm + r * D + ((ch ^ (r & (CH - 1))) << 2)) = x;
      }
    if (hh == 0) { sm_m[wave][r] = m_run; sm_l[wave][r] = l_run; }
    const bool any_bad = __any(bad);
    if (lane == 0) { sm_bad[wave] = any_bad; sm_odd[wave] = found_odd; }
    lds_barrier();

    const bool whole = s0 == 0 && s1 == steps;     // else a partial: slot 1 where the unit begins, 0 behind
    const int64_t slot = ((int64_t)share * units + unit) * 2 + (s0 == 0 ? 1 : 0);
    for (int i = tid; i < rows_here * CH; i += 256) {
      const int rl = i / CH, ch = i - rl * CH;
      const int w0 = rl >> 5, rr = rl & 31;        // waves w0, w0 + WM, ... hold the row
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
      const int rg = mt * p.tile_rows + rl, t = rg / p.group;
      const float lse2 = l == 0.f ? kNegInf : m + __log2f(l);
      if (__builtin_expect(sm_odd[0] | sm_odd[1] | sm_odd[2] | sm_odd[3], 0)) {
        // The CH lanes of a row go through its drafted keys together, each with 4 columns of V and of the score.
        // (opaque, unroll 1: else lane constants are made before the loop over the steps and spill there: d = 256
        // decoding 525 us, 440 so)
        const int col = opaque(ch) * 4;
        const bool in = col < c.d;
        const u16* q = (const u16*)p.q + (int64_t)bidb * p.q_batch + (int64_t)t * p.q_row +
                       (int64_t)(kvh * p.group + rg - t * p.group) * p.q_head;
        auto four = [&](const u16* row) { return in ? *(const u32x2_t*)(row + col) : u32x2_t{0u, 0u}; };
        auto elt = [](u32x2_t x, int e) { return E::to_f32((u16)(x[e >> 1] >> (e & 1) * 16)); };
        const int ln = opaque(lane);
        auto of_row = [&](bool x) { return __ballot(x) >> (ln & ~(CH - 1)) & (~0ull >> (64 - CH)); };
        const u32x2_t qx = four(q);
        const int last = min(p.mask == nullptr ? min(total, len + t + 1) : total, s1 * kStep);
        for (int j = max(first_hidden(p, len, mt), s0 * kStep); j < last; ++j) {
          if (!sees(t, j, mask_byte(t, j))) continue;
          bool out = false;
          const int64_t off = has_new ? 0 : slot_offset(c, bidb, j, out);
          const u32x2_t v = four(has_new ? vn + (int64_t)(j - len) * p.vn_row : vc + off);
          const unsigned odd[2] = {odd_pair<BF16>(v[0]), odd_pair<BF16>(v[1])};
          if (of_row((odd[0] | odd[1]) != 0) == 0) continue;
          const u32x2_t k = four(has_new ? kn + (int64_t)(j - len) * p.kn_row : kc + off);
          float dot = 0.f;
#pragma unroll
          for (int e = 0; e < 4; ++e) dot += elt(qx, e) * elt(k, e);
#pragma unroll 1
          for (int x = 1; x < CH; x <<= 1) dot += __shfl_xor(dot, opaque(x));
          const float weight = fast_exp2(fmaf(dot, cs, -lse2));
          bool done = true;                        // (NaN already: no key changes that)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            if (odd[e >> 1] >> (e & 1) * 16 & 1) acc[e] += weight * elt(v, e);
            done = done && acc[e] != acc[e];
          }
          if (of_row(in && !done) == 0) break;
        }
      }
      if (l != l) acc[0] = acc[1] = acc[2] = acc[3] = l;
      if (!whole) {
        const int64_t prow = slot * p.tile_rows + rl;
        if (ch * 4 < c.d) *(f32x4_t*)(p.part_o + prow * c.d + ch * 4) = acc;
        if (ch == 0) p.part_lse[prow] = lse2;
      } else {
        const int head = kvh * p.group + rg - t * p.group;
        if (ch * 4 < c.d) {
          u32x2_t u = {E::pack2(acc[0], acc[1]), E::pack2(acc[2], acc[3])};
          *(u32x2_t*)((u16*)p.o + (int64_t)bidb * p.o_batch + (int64_t)t * p.o_row + (int64_t)head * p.o_head + ch * 4) = u;
        }
        if (ch == 0) p.lse[((int64_t)bidb * p.h + head) * p.sq + t] = l == 0.f ? -kNegInf : lse2 * kLn2;
      }
    }

    // ---- append the drafted keys of this piece (nobody reads their slots: rows come from k_new) ----
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

    // ---- next ----
    at += s1 - s0;
    if (s1 == steps) { seq_at = at; ++bidb; }
    if (at < end) lds_barrier();                   // the merge is done with LDS
  }
}

// The pieces of a sequence: shares [first, last]; a row's partials of each
struct Pieces {
  int first, last;
  __device__ inline Pieces(const KvAttnParams& p, const Shares& sh, int lane, int bidb, int len) {
    const int at = Shares::before(p, lane, bidb);
    first = at / sh.share;
    last = (at + seq_steps(p, len) - 1) / sh.share;
  }
  __device__ inline int64_t row(const KvAttnParams& p, int share, int unit, int rl) const {
    return (((int64_t)share * p.c.hk * p.m_tiles + unit) * 2 + (share == first ? 1 : 0)) * p.tile_rows + rl;
  }
};

// Workgroups [0, merges): the pieces of RPB rows are merged, 256 / RPB threads a row, D / 4 lanes of 4
// columns x the pieces dealt to the groups of so many lanes, then the groups through LDS.  The others:
// 1024 keys of a (sequence, kv head) each, 4 a thread, whose weight grows by the sum over the rows of
// 2^(stored score - LSE).
template <bool BF16, int D, int RPB>
__global__ void __launch_bounds__(256) kv_merge_kernel(const KvAttnParams p, int merges, int chunks) {
  using E = Elt<BF16>;
  constexpr int CH = D / 4, TPR = 256 / RPB, GROUPS = TPR / CH;
  static_assert(GROUPS >= 1, "a row has at least D / 4 threads");
  const KvCache& c = p.c;
  const int lane = threadIdx.x & 63;
  const Shares sh(p, lane);

  if ((int)blockIdx.x >= merges) {
    const int wg = blockIdx.x - merges, bh = wg / chunks;
    const int bidb = bh / c.hk, kvh = bh - bidb * c.hk;
    const int len = c.lens[bidb];
    const int total = seq_ok(c, len, p.sq) ? len + p.sq : 0;
    const int j0 = (wg - bh * chunks) * 1024, j = j0 + 4 * (int)threadIdx.x;
    if (j0 >= total) return;
    const Pieces pc(p, sh, lane, bidb, len);       // (stored scores: one tile of rows, unit = kv head)
    __shared__ float s_lse[kScoreRows];
    // the first rows' scores and the weights are on their way over the LSE
    constexpr int kAhead = 4;
    const bool has = j < total;
    const float* sc = p.scores + (int64_t)bh * p.rows * p.score_pitch + (has ? j : 0);
    float* w = p.weight + (int64_t)bidb * p.w_batch + (int64_t)kvh * p.w_head + (has ? j : 0);
    f32x4_t ahead[kAhead], sum;
#pragma unroll
    for (int i = 0; i < kAhead; ++i) ahead[i] = *(const f32x4_t*)(sc + (int64_t)min(i, p.rows - 1) * p.score_pitch);
#pragma unroll
    for (int e = 0; e < 4; ++e) sum[e] = j + e < total ? w[e] : 0.f;
    // eight threads a row, all rows at once
    const int r = threadIdx.x >> 3, g = threadIdx.x & 7;
    static_assert(kScoreRows <= 256 / 8, "a row has eight threads");
    float m = kNegInf, l = 0.f;
    auto join = [&](float m2, float l2) {          // (equal maxima, both -inf among them: no difference taken; NaN stays)
      const float top = fmaxf(m, m2);
      l = l * (m == top ? 1.f : fast_exp2(m - top)) + l2 * (m2 == top ? 1.f : fast_exp2(m2 - top));
      m = top;
    };
    if (pc.first < pc.last) {
      if (r < p.rows)
        for (int s = pc.first + g; s <= pc.last; s += 8) {
          const float y = p.part_lse[pc.row(p, s, kvh, r)];
          if (y != kNegInf) join(y, 1.f);
        }
#pragma unroll
      for (int off = 4; off > 0; off >>= 1) {
        const float m2 = __shfl_xor(m, off), l2 = __shfl_xor(l, off);
        join(m2, l2);
      }
      if (g == 0 && r < p.rows) s_lse[r] = l == 0.f ? kNegInf : m + __log2f(l);
    } else if (g == 0 && r < p.rows) {
      const int t = r / p.group, head = kvh * p.group + r - t * p.group;
      const float x = p.lse[((int64_t)bidb * p.h + head) * p.sq + t] * kLog2e;
      s_lse[r] = x == -kNegInf ? kNegInf : x;
    }
    __syncthreads();
    if (!has) return;
    f32x4_t add = {0.f, 0.f, 0.f, 0.f};
    auto row_adds = [&](const f32x4_t& x, float le) {
#pragma unroll
      for (int e = 0; e < 4; ++e) add[e] += x[e] == kNegInf ? 0.f : fast_exp2(x[e] - le);
    };
#pragma unroll
    for (int i = 0; i < kAhead; ++i)
      if (i < p.rows) row_adds(ahead[i], s_lse[i]);
#pragma unroll 4
    for (int i = kAhead; i < p.rows; ++i) row_adds(*(const f32x4_t*)(sc + (int64_t)i * p.score_pitch), s_lse[i]);
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (j + e < total) w[e] = sum[e] + add[e];
    return;
  }

  const int rblocks = (p.rows + RPB - 1) / RPB;
  const int bh = blockIdx.x / rblocks, row = (blockIdx.x - bh * rblocks) * RPB + (int)threadIdx.x / TPR;
  const int bidb = bh / c.hk, kvh = bh - bidb * c.hk;
  const int ch = threadIdx.x % CH, grp = threadIdx.x % TPR / CH;
  const int mt = min(row, p.rows - 1) / p.tile_rows, rl = min(row, p.rows - 1) - mt * p.tile_rows;
  const Pieces pc(p, sh, lane, bidb, c.lens[bidb]);
  const bool split = pc.first < pc.last && row < p.rows;
  float m = kNegInf, l = 0.f;
  f32x4_t acc = {0.f, 0.f, 0.f, 0.f};
  if (split) {
    for (int s = pc.first + grp; s <= pc.last; s += GROUPS) {   // running maximum: one read of the pieces
      const int64_t prow = pc.row(p, s, mt * c.hk + kvh, rl);
      const float x = p.part_lse[prow];
      f32x4_t v = {0.f, 0.f, 0.f, 0.f};
      if (ch * 4 < c.d) v = *(const f32x4_t*)(p.part_o + prow * c.d + ch * 4);
      if (x == kNegInf) continue;
      const float mn = fmaxf(m, x), a = m == kNegInf ? 0.f : fast_exp2(m - mn), f = fast_exp2(x - mn);   // NaN stays
      l = l * a + f;
#pragma unroll
      for (int e = 0; e < 4; ++e) acc[e] = acc[e] * a + f * v[e];
      m = mn;
    }
  }
  if constexpr (GROUPS > 1) {
    __shared__ float sl[RPB * GROUPS], sm[RPB * GROUPS];
    __shared__ f32x4_t sa[RPB * GROUPS][CH];
    const int me = (int)threadIdx.x / CH;
    if (ch == 0) { sl[me] = l; sm[me] = m; }
    sa[me][ch] = acc;
    __syncthreads();
    if (grp != 0 || !split) return;
    float top = m;
#pragma unroll
    for (int g = 1; g < GROUPS; ++g) top = fmaxf(top, sm[me + g]);
    const float a = m == kNegInf ? 0.f : fast_exp2(m - top);
    l *= a;
#pragma unroll
    for (int e = 0; e < 4; ++e) acc[e] *= a;
#pragma unroll
    for (int g = 1; g < GROUPS; ++g) {
      const float f = sm[me + g] == kNegInf ? 0.f : fast_exp2(sm[me + g] - top);
      l += f * sl[me + g];
      const f32x4_t v = sa[me + g][ch];
#pragma unroll
      for (int e = 0; e < 4; ++e) acc[e] += f * v[e];
    }
    m = top;
  }
  if (!split) return;
  const int t = row / p.group, head = kvh * p.group + row - t * p.group;
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

// Rows of a unit, and the shares: as many as make the units the resident workgroups of the chip, four
// rounds of them when a share alone has more than a quarter; fewer when there are not as many steps.
// (Two or four rounds of smaller shares balance better but pay each a start and a merge: 5 to 10 % slower.)
// Rows of several tiles are dealt evenly, in wholes of a wave's 32; the waves left over stage their keys only
// (48 tokens x 4 heads, 16 sequences of up to 8k keys: 96 + 96 rows 163 us, 128 + 64 171, and 183 with those waves computing
// too; three tiles of 64 250).
static int rows_per_unit(int rows) { return rows <= 32 ? 32 : rows <= 64 ? 64 : 128; }

void kv_attn_plan(KvAttnParams& p) {
  const int per = rows_per_unit(p.rows);
  p.m_tiles = (p.rows + per - 1) / per;
  p.tile_rows = std::min(p.rows, ((p.rows + p.m_tiles - 1) / p.m_tiles + 31) / 32 * 32);
  const int64_t units = (int64_t)p.c.hk * p.m_tiles, steps = (int64_t)p.c.b * ((p.c.slots + kStep - 1) / kStep);
  if (steps > 0x7fff0000 || units > 0xffffff) throw std::runtime_error("kvcache attention: too many keys for one launch");
  const int dd = p.c.d <= 64 ? 64 : p.c.d <= 128 ? 128 : 256;
  const int64_t resident = 256 * groups_per_cu(dd, per / 32);
  p.shares = (int)std::min(steps, units <= resident / 4 ? resident / units : (4 * resident + units - 1) / units);
  p.score_pitch = (p.c.slots + 127) & ~127;
  // a wave's 32 keys evenly strided, their rows apart and within a range check's 31 bits
  p.even = p.c.page % 32 == 0 && p.c.row >= p.c.d && p.c.row <= (1 << 24);
}

// scores are stored where that is at most a quarter of the cache's bytes (and 32-bit offsets reach them)
static bool store_scores(const KvAttnParams& p) {
  return p.weight != nullptr && p.rows <= kScoreRows && 4 * p.rows <= p.c.d && p.rows * p.score_pitch < (1 << 29);
}

// a sequence of one step is never cut, nor any where all steps are one share (a prompt's row tiles fill the chip)
static bool may_cut(const KvAttnParams& p) { return p.c.slots > kStep && p.shares > 1; }

static size_t part_floats(const KvAttnParams& p) {
  return may_cut(p) ? ((size_t)p.shares * p.c.hk * p.m_tiles * 2 * p.tile_rows * (p.c.d + 1) + 3) / 4 * 4 : 0;
}

size_t kv_attn_workspace(const KvAttnParams& p) {
  const size_t scores = store_scores(p) ? (size_t)p.c.b * p.c.hk * p.rows * (size_t)p.score_pitch : 0;
  return (part_floats(p) + scores) * sizeof(float);
}

template <bool BF16, int D>
static void run_attn(const KvAttnParams& p, hipStream_t stream) {
  const int64_t bh = (int64_t)p.c.b * p.c.hk;
  // many rows are cut into few pieces each (their tiles make the units): fewer threads a row
  constexpr int kFewPieces = 1024 / D;
  const bool many = p.rows > 32;
  const int chunks = p.scores != nullptr ? (p.c.slots + 1023) / 1024 : 0;
  const int64_t merges = !may_cut(p) ? 0 : bh * (many ? (p.rows + kFewPieces - 1) / kFewPieces : p.rows);
  const int64_t tail = merges + bh * chunks;
  const int weight_chunks = p.weight != nullptr && p.scores == nullptr ? (p.c.slots + 127) / 128 : 0;
  if (tail > 0x7fffffff || weight_chunks > 65535)
    throw std::runtime_error("kvcache attention: too many workgroups for one launch");
  const dim3 g((unsigned)((p.shares + 7) / 8 * 8 * p.c.hk * p.m_tiles)), t(256), gt((unsigned)tail);
  switch (rows_per_unit(p.rows)) {
    case 32: hipLaunchKernelGGL((kv_attn_kernel<BF16, D, 1>), g, t, 0, stream, p); break;
    case 64: hipLaunchKernelGGL((kv_attn_kernel<BF16, D, 2>), g, t, 0, stream, p); break;
    default: hipLaunchKernelGGL((kv_attn_kernel<BF16, D, 4>), g, t, 0, stream, p); break;
  }
  if (tail > 0 && many) hipLaunchKernelGGL((kv_merge_kernel<BF16, D, kFewPieces>), gt, t, 0, stream, p, (int)merges, chunks);
  else if (tail > 0) hipLaunchKernelGGL((kv_merge_kernel<BF16, D, 1>), gt, t, 0, stream, p, (int)merges, chunks);
  if (weight_chunks > 0)
    hipLaunchKernelGGL((kv_weight_kernel<BF16, D>), dim3((unsigned)bh, (unsigned)weight_chunks), t, 0, stream, p);
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
  p.part_o = (float*)workspace;
  p.part_lse = p.part_o + (int64_t)p.shares * p.c.hk * p.m_tiles * 2 * p.tile_rows * p.c.d;
  if (store_scores(p)) p.scores = (float*)workspace + part_floats(p);
  if (is_bf16) dispatch_attn<true>(p, stream);
  else dispatch_attn<false>(p, stream);
  check_launch("kvcache attention");
}

}  // namespace fa
