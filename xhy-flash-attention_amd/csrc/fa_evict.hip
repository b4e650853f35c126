// Compaction of a key/value cache in place (gfx950): eviction by accumulated attention weight, and the
// commit of the accepted drafted tokens.
//
// Eviction, for each (sequence, kv head) of n > budget keys with weights w: keep the first `sink` keys,
// the last `recent`, and of the others the budget - sink - recent with the largest w (equal weights:
// the lowest index); the kept keys move to places 0 .. budget - 1 in their order.  Two kernels:
//   * select: one workgroup a (sequence, kv head), which holds up to 32k weights in registers.  The
//     smallest kept weight is found by a radix select over order-preserving 32-bit images of the weights,
//     8 + 12 + 12 bits from the top, each pass a histogram in LDS of the keys that agree with the prefix
//     found so far.  Weights crowd in a few exponents, so the first histogram has a copy for every two
//     lanes.  One more pass counts, per wave over consecutive keys, those above and those equal;
//     their prefix sums give every kept key its place, so the result is a function of the weights alone;
//   * move: place i receives key kept[i] >= i.  A workgroup owns all rows of a 64- or 128-byte column slice of K
//     or V of one (sequence, kv head) and walks the places upwards in chunks: the chunk's rows are in
//     registers in every thread (barrier) before any of its places is written, and places below
//     a chunk are never read by a later one, so in place needs no second buffer: each kept row
//     is read once and written once.  The next chunk's rows are on their way over the barrier.
// Commit is the move kernel with the list of the accepted drafted tokens, built in LDS by the workgroup
// itself, at places lens[b] ...
// Measured: 8 heads of 4.2k keys to 2k: select 15.7 us, bound by its passes' barriers on one CU a head, move
// 6.5; 64 heads of 9k to 32k keys to 8k (paged, d = 128, fp16): select 38 us, move 129 us (0.54 GB, 4.2 TB/s in
// scattered 256-byte rows, a copy's 5.2 in whole pages); commit of 128 x 64 drafted 8.8 us, of one sequence 3.0.
#include <stdexcept>
#include <string>

#include "fa_kvcache.h"

namespace fa {

static constexpr int kSelThreads = 1024, kSelWaves = kSelThreads / 64;
static constexpr int kSelCopies = 32, kSelPitch = 257;   // histograms of the first pass, by lane (see below)

// 32-bit image of a weight: unsigned order = numeric order, NaN above +inf, -0 = +0
__device__ inline unsigned ordered(float x) {
  if (x != x) return 0xffffffffu;
  const unsigned u = __builtin_bit_cast(unsigned, x == 0.f ? 0.f : x);
  return (u >> 31) ? ~u : (u | 0x80000000u);
}

__device__ inline int wave_count(bool x) { return __popcll(__ballot(x)); }
__device__ inline int lanes_below(bool x, int lane) { return __popcll(__ballot(x) & ((1ull << lane) - 1)); }

// BATCH: keys a thread holds
template <int BATCH>
__global__ void __launch_bounds__(kSelThreads) kv_select_kernel(const KvEvictParams p) {
  constexpr int CHUNK = kSelThreads * BATCH;
  const KvCache& c = p.c;
  const int tid = threadIdx.x, lane = tid & 63, wave = wave_uniform(tid >> 6);
  const int kvh = blockIdx.x, bidb = blockIdx.y;
  const int bh = bidb * c.hk + kvh;
  const int n = c.lens[bidb];
  const bool ok = seq_ok(c, n, 0);
  const float* __restrict__ w = p.weight + (int64_t)bidb * p.w_batch + (int64_t)kvh * p.w_head;
  float* __restrict__ wo = p.weight_out + (int64_t)bidb * p.wo_batch + (int64_t)kvh * p.wo_head;
  int* __restrict__ kept = p.kept + (int64_t)bh * p.budget;
  if (kvh == 0 && tid == 0) p.lens_out[bidb] = ok ? min(n, p.budget) : n;

  if (!ok || n <= p.budget) {   // nothing moves; a length outside the cache leaves everything as it was
    for (int i = tid; i < p.budget; i += kSelThreads) kept[i] = ok && i < n ? i : -1;
    for (int i = tid; i < c.slots; i += kSelThreads) wo[i] = !ok || i < n ? w[i] : 0.f;
    if (tid == 0) p.first[bh] = p.budget;
    return;
  }

  __shared__ int hist[kSelCopies * kSelPitch];     // pass 0: copies of 256 bins; then one of 4096
  __shared__ int wave_sum[2][kSelWaves], wave_sum2[2][kSelWaves];
  __shared__ int s_digit, s_need, s_first;
  const int lo = p.sink, hi = n - p.recent;       // the keys that compete
  int need = p.budget - p.sink - p.recent;        // how many of them stay
  unsigned prefix = 0;
  int shift = 32;
  if (tid == 0) s_first = n;
  // The weights go by in chunks of consecutive keys, a wave 64 `used` of a chunk, all on their way at
  // once; a head of one chunk keeps them in registers over all passes.
  float x[BATCH];
  unsigned image[BATCH];
  int held = -1;
  auto at = [&](int c0, int used, int u) { return c0 + (wave * used + u) * 64 + lane; };
  auto competes = [&](int i) { return (unsigned)(i - lo) < (unsigned)(hi - lo); };   // (hi > lo: n > budget)
  auto fetch = [&](int c0) {
    const int used = min(BATCH, (n - c0 + kSelThreads - 1) / kSelThreads);
    if (held != c0) {
#pragma unroll
      for (int u = 0; u < BATCH; ++u)
        if (u < used) x[u] = w[min(at(c0, used, u), n - 1)];
#pragma unroll
      for (int u = 0; u < BATCH; ++u)
        if (u < used) image[u] = ordered(x[u]);
      held = c0;
    }
    return used;
  };
#pragma unroll 1
  for (int pass = 0; pass < 3 && need > 0; ++pass) {
    const int bits = pass == 0 ? 8 : 12;
    for (int i = tid; i < kSelCopies * kSelPitch; i += kSelThreads) hist[i] = 0;
    __syncthreads();
    const int top = shift;
    shift -= bits;
    for (int c0 = 0; c0 < n; c0 += CHUNK) {
      const int used = fetch(c0);
      if (pass == 0) {
#pragma unroll
        for (int u = 0; u < BATCH; ++u)
          if (u < used && competes(at(c0, used, u)))
            atomicAdd(&hist[lane % kSelCopies * kSelPitch + (image[u] >> 24)], 1);
      } else {
#pragma unroll
        for (int u = 0; u < BATCH; ++u)
          if (u < used && competes(at(c0, used, u)) && (image[u] >> top) == prefix)
            atomicAdd(&hist[(image[u] >> shift) & 4095u], 1);
      }
    }
    __syncthreads();
    // a thread holds 4 bins (pass 0: the first 256 threads one), the highest first: keys above a bin by
    // a prefix sum over the threads
    const int b0 = pass == 0 ? 255 - tid : 4095 - 4 * tid;
    int own[4] = {0, 0, 0, 0};
    if (pass > 0) {
#pragma unroll
      for (int k = 0; k < 4; ++k) own[k] = hist[b0 - k];
    } else if (tid < 256) {
#pragma unroll
      for (int v = 0; v < kSelCopies; ++v) own[0] += hist[v * kSelPitch + b0];
    }
    const int mine = own[0] + own[1] + own[2] + own[3];
    int sum = mine;
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) {
      const int y = __shfl_up(sum, off);
      if (lane >= off) sum += y;
    }
    if (lane == 63) wave_sum[0][wave] = sum;
    __syncthreads();
    int above = sum - mine;
#pragma unroll
    for (int i = 0; i < kSelWaves; ++i) above += i < wave ? wave_sum[0][i] : 0;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      if (above < need && above + own[k] >= need) { s_digit = b0 - k; s_need = need - above; }
      above += own[k];
    }
    __syncthreads();
    prefix = (prefix << bits) | (unsigned)s_digit;
    need = s_need;
    __syncthreads();
  }
  // kept of [lo, hi): images above `prefix`, and the first `need` equal to it (none at all when no
  // key of the middle stays): every wave counts its own, the counts meet in LDS, and the keys go to
  // their places.
  const bool some = p.budget > p.sink + p.recent;
  int above0 = 0, equal0 = 0, dropped_first = n;   // kept above / equal before this chunk
  for (int c0 = 0, turn = 0; c0 < n; c0 += CHUNK, turn ^= 1) {
    const int used = fetch(c0);
    unsigned gt = 0, eq = 0;                       // bit u: this lane's key u
    int above = 0, equal = 0;
#pragma unroll
    for (int u = 0; u < BATCH; ++u)
      if (u < used) {
        const int i = at(c0, used, u);
        const bool mid = competes(i);
        const bool g = i < n && (!mid || (some && image[u] > prefix)), e = mid && some && image[u] == prefix;
        gt |= (unsigned)g << u;
        eq |= (unsigned)e << u;
        above += wave_count(g);
        equal += wave_count(e);
      }
    if (lane == 0) { wave_sum[turn][wave] = above; wave_sum2[turn][wave] = equal; }
    __syncthreads();                               // (the two turns' counts alternate: one barrier a chunk)
    int ga = above0, ea = equal0;
#pragma unroll
    for (int v = 0; v < kSelWaves; ++v) {
      const int a = wave_sum[turn][v], e = wave_sum2[turn][v];
      ga += v < wave ? a : 0;
      ea += v < wave ? e : 0;
      above0 += a;
      equal0 += e;
    }
#pragma unroll
    for (int u = 0; u < BATCH; ++u)
      if (u < used) {
        const int i = at(c0, used, u);
        const bool g = (gt >> u) & 1, e = (eq >> u) & 1;
        const int erank = ea + lanes_below(e, lane);
        const int place = ga + lanes_below(g, lane) + min(erank, need);
        const bool keep = g || (e && erank < need);
        if (keep) { kept[place] = i; wo[place] = x[u]; }
        if (i < n && !keep) dropped_first = min(dropped_first, i);
        ga += wave_count(g);
        ea += wave_count(e);
      }
  }
  if (dropped_first < n) atomicMin(&s_first, dropped_first);
  lds_barrier();                                   // (leaves the stores in flight)
  if (tid == 0) p.first[bh] = min(s_first, p.budget);   // keys below the first dropped one stay put
  for (int i = p.budget + tid; i < c.slots; i += kSelThreads) wo[i] = 0.f;
}

// Threads and rows a thread: eviction walks thousands of rows (64 heads of 8k: 1024 threads 129 us, 512 172; two
// or six rows 134), commit the accepted ones of a few dozen (128 x 64 drafted: 256 threads with one row
// 8.8 us, with four 9.5; 512 with two 11.6, 1024 16.8).
static constexpr int kEvictThreads = 1024, kEvictRows = 4, kCommitThreads = 256, kCommitLanes = 16, kCommitRows = 1;

// Moves rows list(i) -> base + i for i in [first, count) of one column slice; list(i) is a key >= base + i,
// ascending.  LANES lanes of 16 bytes a row, U rows a thread in flight, two chunks deep.
template <int THREADS, int LANES, int U, typename List>
__device__ inline void move_rows(const KvCache& c, char* base_ptr, int bidb, int col, int base, int first, int count,
                                 List list) {
  constexpr int ROWS = THREADS / LANES, CHUNK = ROWS * U;
  const int rl = threadIdx.x / LANES;
  const int64_t cb = (int64_t)(col + 8 * (threadIdx.x % LANES)) * 2;
  const bool col_ok = col + 8 * ((int)threadIdx.x % LANES) < c.d;
  bool ok[2][U];
  u32x4_t x[2][U];
  int from[U];                                     // the next chunk's keys, read a chunk before their rows
  auto look_up = [&](int i0) {
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int i = i0 + u * ROWS + rl;
      from[u] = i < count ? list(i) : -1;
    }
  };
  auto load = [&](int b) {
#pragma unroll
    for (int u = 0; u < U; ++u) {
      bool bad = false;
      ok[b][u] = from[u] >= 0 && col_ok;
      if (!ok[b][u]) continue;
      const int64_t off = slot_offset(c, bidb, from[u], bad);
      ok[b][u] = !bad;
      if (!bad) x[b][u] = *(const u32x4_t*)(base_ptr + off * 2 + cb);
    }
  };
  auto store = [&](int i0, int b) {
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (!ok[b][u]) continue;
      bool bad = false;
      const int64_t off = slot_offset(c, bidb, base + i0 + u * ROWS + rl, bad);
      if (!bad) *(u32x4_t*)(base_ptr + off * 2 + cb) = x[b][u];
    }
  };
  auto landed = [&](int b) {   // the chunk's rows are in this thread's registers
#pragma unroll
    for (int u = 0; u < U; ++u) asm volatile("" : "+v"(x[b][u]) :: "memory");
  };
#pragma unroll
  for (int u = 0; u < U; ++u) x[0][u] = x[1][u] = u32x4_t{0u, 0u, 0u, 0u};
  look_up(first);
  load(0);
  look_up(first + CHUNK);
  for (int i0 = first; i0 < count; i0 += 2 * CHUNK) {
    load(1);
    look_up(i0 + 2 * CHUNK);
    landed(0);
    lds_barrier();
    store(i0, 0);
    load(0);
    look_up(i0 + 3 * CHUNK);
    landed(1);
    lds_barrier();
    store(i0 + CHUNK, 1);
  }
}

// Column slices of LANES 16-byte pieces; the slices of a (sequence, kv head) sit 8 workgroups apart: the same
// XCD, so lines that two of them share are fetched once
template <int LANES>
__global__ void __launch_bounds__(kEvictThreads) kv_evict_move_kernel(const KvEvictParams p, int slices) {
  const KvCache& c = p.c;
  const int per = 8 * 2 * slices;
  const int oct = blockIdx.x / per, rem = blockIdx.x - oct * per;
  const int bh = oct * 8 + (rem & 7), part = rem >> 3;
  if (bh >= c.b * c.hk) return;
  const int bidb = bh / c.hk, kvh = bh - bidb * c.hk;
  const int n = c.lens[bidb];
  if (!seq_ok(c, n, 0)) return;
  const int first = p.first[bh], count = min(n, p.budget);
  if (first >= count) return;
  char* base = (char*)(part >= slices ? c.v : c.k) + (int64_t)kvh * c.head * 2;
  const int* kept = p.kept + (int64_t)bh * p.budget;
  move_rows<kEvictThreads, LANES, kEvictRows>(c, base, bidb, part % slices * LANES * 8, 0, first, count,
                            [&](int i) { return kept[i]; });
}

__global__ void __launch_bounds__(kCommitThreads) kv_commit_kernel(const KvCommitParams p, int slices) {
  const KvCache& c = p.c;
  extern __shared__ int list[];                   // the accepted tokens, ascending
  __shared__ int s_count;
  const int per = 2 * slices;
  const int bh = blockIdx.x / per, part = blockIdx.x - bh * per;
  const int bidb = bh / c.hk, kvh = bh - bidb * c.hk;
  const int lane = threadIdx.x & 63, len = c.lens[bidb];
  const bool ok = seq_ok(c, len, p.sq);
  if (threadIdx.x < 64) {
    int count = 0;
    for (int i0 = 0; i0 < p.sq; i0 += 64) {
      const bool a = i0 + lane < p.sq && p.accepted[(int64_t)bidb * p.acc_batch + i0 + lane] != 0;
      if (a) list[count + lanes_below(a, lane)] = i0 + lane;
      count += wave_count(a);
    }
    if (lane == 0) s_count = count;
  }
  __syncthreads();
  const int count = s_count;
  if (part == 0 && kvh == 0 && threadIdx.x == 0) p.lens_out[bidb] = ok ? len + count : len;
  if (!ok) return;
  char* base = (char*)(part >= slices ? c.v : c.k) + (int64_t)kvh * c.head * 2;
  move_rows<kCommitThreads, kCommitLanes, kCommitRows>(c, base, bidb, part % slices * kCommitLanes * 8, len, 0, count,
                             [&](int i) { return len + list[i]; });
  if (p.weight != nullptr && part == 0) {
    float* w = p.weight + (int64_t)bidb * p.w_batch + (int64_t)kvh * p.w_head + len;
    for (int i0 = 0; i0 < p.sq; i0 += kCommitThreads) {
      const int i = i0 + (int)threadIdx.x;
      const float x = i < count ? w[list[i]] : 0.f;
      __syncthreads();                            // (waits for the loads: sources lie at or above i)
      if (i < p.sq) w[i] = x;
    }
  }
}

void launch_kv_evict(const KvEvictParams& p, hipStream_t stream) {
  const KvCache& c = p.c;
  // 32 keys a thread unroll to code that a small cache does not earn back (4k slots, 8 heads: 8 keys a
  // thread 15.7 us, 32 keys 22.4; at 32k slots, 64 heads: 4 keys 47.8, 32 keys 38 us)
  const dim3 heads((unsigned)c.hk, (unsigned)c.b);
  if (c.slots <= 8 * kSelThreads) hipLaunchKernelGGL((kv_select_kernel<8>), heads, dim3(kSelThreads), 0, stream, p);
  else hipLaunchKernelGGL((kv_select_kernel<32>), heads, dim3(kSelThreads), 0, stream, p);
  // 128-byte slices (whole lines), or 64-byte ones where those leave CUs without a workgroup (64 heads of 8k
  // kept keys: 128 bytes 129 us, 64 bytes 160; 8 heads of 2k: 8.9, 6.5 us)
  const int64_t heads8 = ((int64_t)c.b * c.hk + 7) / 8 * 8;
  const bool wide = heads8 * 2 * ((c.d + 63) / 64) >= 256;
  const int slices = wide ? (c.d + 63) / 64 : (c.d + 31) / 32;
  const int64_t grid = heads8 * 2 * slices;
  if (grid > 0x7fffffff) throw std::runtime_error("kvcache evict: too many workgroups for one launch");
  if (wide) hipLaunchKernelGGL((kv_evict_move_kernel<8>), dim3((unsigned)grid), dim3(kEvictThreads), 0, stream, p, slices);
  else hipLaunchKernelGGL((kv_evict_move_kernel<4>), dim3((unsigned)grid), dim3(kEvictThreads), 0, stream, p, slices);
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) throw std::runtime_error(std::string("kvcache evict launch: ") + hipGetErrorString(e));
}

void launch_kv_commit(const KvCommitParams& p, hipStream_t stream) {
  const KvCache& c = p.c;
  const int slices = (c.d + 8 * kCommitLanes - 1) / (8 * kCommitLanes);
  const int64_t grid = (int64_t)c.b * c.hk * 2 * slices;
  if (grid > 0x7fffffff) throw std::runtime_error("kvcache commit: too many workgroups for one launch");
  hipLaunchKernelGGL(kv_commit_kernel, dim3((unsigned)grid), dim3(kCommitThreads), (unsigned)p.sq * sizeof(int), stream,
                     p, slices);
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) throw std::runtime_error(std::string("kvcache commit launch: ") + hipGetErrorString(e));
}

}  // namespace fa
