// Compaction of a key/value cache in place (gfx950): eviction by accumulated attention weight, and the
// commit of the accepted drafted tokens.
//
// Eviction, for each (sequence, kv head) of n > budget keys with weights w: keep the first `sink` keys,
// the last `recent`, and of the others the budget - sink - recent with the largest w (equal weights:
// the lowest index); the kept keys move to places 0 .. budget - 1 in their order.  Two kernels:
//   * select: one workgroup a (sequence, kv head).  The smallest kept weight is found by a radix
//     select over order-preserving 32-bit images of the weights, 11 + 11 + 10 bits from the top, each
//     pass a histogram in LDS of the keys that agree with the prefix found so far (the weights are
//     re-read from L2: 4 bytes a key against the 4 d of its K and V).  One more pass counts, per wave
//     over consecutive keys, those above and those equal; their prefix sums give every kept key its
//     place without atomics, so the result is a function of the weights alone;
//   * move: place i receives key kept[i] >= i.  A workgroup owns all rows of a 64-byte column slice of K
//     or V of one (sequence, kv head) and walks the places upwards in chunks: the chunk's rows are in
//     registers in every thread (barrier) before any of its places is written, and places below
//     a chunk are never read by a later one, so in place needs no second buffer: each kept row
//     is read once and written once.  The next chunk's rows are on their way over the barrier.
// Commit is the move kernel with the list of the accepted drafted tokens, built in LDS by the workgroup
// itself, at places lens[b] ...
#include <stdexcept>
#include <string>

#include "fa_kvcache.h"

namespace fa {

static constexpr int kSelThreads = 1024, kSelWaves = kSelThreads / 64;
static constexpr int kMoveThreads = 512;

// 32-bit image of a weight: unsigned order = numeric order, NaN above +inf, -0 = +0
__device__ inline unsigned ordered(float x) {
  if (x != x) return 0xffffffffu;
  const unsigned u = __builtin_bit_cast(unsigned, x == 0.f ? 0.f : x);
  return (u >> 31) ? ~u : (u | 0x80000000u);
}

__device__ inline int wave_count(bool x) { return __popcll(__ballot(x)); }
__device__ inline int lanes_below(bool x, int lane) { return __popcll(__ballot(x) & ((1ull << lane) - 1)); }

__global__ void __launch_bounds__(kSelThreads) kv_select_kernel(const KvEvictParams p) {
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

  __shared__ int hist[2048];
  __shared__ int wave_sum[kSelWaves], wave_sum2[kSelWaves];
  __shared__ int s_digit, s_need, s_first;
  const int lo = p.sink, hi = n - p.recent;       // the keys that compete
  int need = p.budget - p.sink - p.recent;        // how many of them stay
  unsigned prefix = 0;
  int shift = 32;
  if (tid == 0) s_first = n;
#pragma unroll 1
  for (int pass = 0; pass < 3 && need > 0; ++pass) {
    const int bits = pass < 2 ? 11 : 10;
    for (int i = tid; i < 2048; i += kSelThreads) hist[i] = 0;
    __syncthreads();
    const int top = shift;
    shift -= bits;
    for (int i = lo + tid; i < hi; i += kSelThreads) {
      const unsigned u = ordered(w[i]);
      if (pass == 0 || (u >> top) == prefix) atomicAdd(&hist[(u >> shift) & ((1u << bits) - 1)], 1);
    }
    __syncthreads();
    // thread t holds bins 2047 - 2t, 2046 - 2t: keys above a bin by a prefix sum over the threads
    const int b0 = 2047 - 2 * tid, n0 = hist[b0], n1 = hist[b0 - 1];
    int sum = n0 + n1;
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) {
      const int x = __shfl_up(sum, off);
      if (lane >= off) sum += x;
    }
    if (lane == 63) wave_sum[wave] = sum;
    __syncthreads();
    int above = sum - n0 - n1;
    for (int i = 0; i < wave; ++i) above += wave_sum[i];
    if (above < need && above + n0 >= need) { s_digit = b0; s_need = need - above; }
    else if (above + n0 < need && above + n0 + n1 >= need) { s_digit = b0 - 1; s_need = need - above - n0; }
    __syncthreads();
    prefix = (prefix << bits) | (unsigned)s_digit;
    need = s_need;
    __syncthreads();
  }
  // kept of [lo, hi): images above `prefix`, and the first `need` equal to it (none at all when no
  // key of the middle stays)
  const bool some = p.budget > p.sink + p.recent;
  const int per_wave = ((n + kSelWaves - 1) / kSelWaves + 63) & ~63;
  const int w0 = wave * per_wave, w1 = min(n, w0 + per_wave);
  int above = 0, equal = 0;
  for (int i0 = w0; i0 < w1; i0 += 64) {
    const int i = i0 + lane;
    const bool in = i < w1, mid = in && i >= lo && i < hi;
    const unsigned u = mid ? ordered(w[i]) : 0u;
    above += wave_count(in && (!mid || (some && u > prefix)));
    equal += wave_count(mid && some && u == prefix);
  }
  if (lane == 0) { wave_sum[wave] = above; wave_sum2[wave] = equal; }
  __syncthreads();
  int above0 = 0, equal0 = 0;
  for (int i = 0; i < wave; ++i) { above0 += wave_sum[i]; equal0 += wave_sum2[i]; }
  for (int i0 = w0; i0 < w1; i0 += 64) {
    const int i = i0 + lane;
    const bool in = i < w1, mid = in && i >= lo && i < hi;
    const float x = in ? w[i] : 0.f;
    const unsigned u = mid ? ordered(x) : 0u;
    const bool eq = mid && some && u == prefix;
    const bool gt = in && (!mid || (some && u > prefix));
    const int erank = equal0 + lanes_below(eq, lane);
    const bool keep = gt || (eq && erank < need);
    const int place = above0 + lanes_below(gt, lane) + min(erank, need);
    if (keep) { kept[place] = i; wo[place] = x; }
    const uint64_t dropped = __ballot(in && !keep);
    if (lane == 0 && dropped != 0) atomicMin(&s_first, i0 + __builtin_ctzll(dropped));
    above0 += wave_count(gt);
    equal0 += wave_count(eq);
  }
  for (int i = p.budget + tid; i < c.slots; i += kSelThreads) wo[i] = 0.f;
  __syncthreads();
  if (tid == 0) p.first[bh] = min(s_first, p.budget);   // keys below the first dropped one stay put
}

// Moves rows list(i) -> base + i for i in [first, count) of one column slice; list(i) is a key >= base + i,
// ascending.  LANES lanes of 16 bytes a row, U rows a thread in flight, two chunks deep.
template <int LANES, int U, typename List>
__device__ inline void move_rows(const KvCache& c, char* base_ptr, int bidb, int col, int base, int first, int count,
                                 List list) {
  constexpr int ROWS = kMoveThreads / LANES, CHUNK = ROWS * U;
  const int rl = threadIdx.x / LANES;
  const int64_t cb = (int64_t)(col + 8 * (threadIdx.x % LANES)) * 2;
  const bool col_ok = col + 8 * ((int)threadIdx.x % LANES) < c.d;
  bool ok[2][U];
  u32x4_t x[2][U];
  auto load = [&](int i0, int b) {
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int i = i0 + u * ROWS + rl;
      bool bad = false;
      ok[b][u] = i < count && col_ok;
      if (!ok[b][u]) continue;
      const int64_t off = slot_offset(c, bidb, list(i), bad);
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
  load(first, 0);
  for (int i0 = first; i0 < count; i0 += 2 * CHUNK) {
    load(i0 + CHUNK, 1);
    landed(0);
    lds_barrier();
    store(i0, 0);
    load(i0 + 2 * CHUNK, 0);
    landed(1);
    lds_barrier();
    store(i0 + CHUNK, 1);
  }
}

// 64-byte column slices; the slices of a (sequence, kv head) sit 8 workgroups apart: the same XCD, so the
// 128-byte lines that two of them share are fetched once
static constexpr int kEvictLanes = 4;
__global__ void __launch_bounds__(kMoveThreads) kv_evict_move_kernel(const KvEvictParams p, int slices) {
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
  move_rows<kEvictLanes, 4>(c, base, bidb, part % slices * kEvictLanes * 8, 0, first, count,
                            [&](int i) { return kept[i]; });
}

static constexpr int kCommitLanes = 16;
__global__ void __launch_bounds__(kMoveThreads) kv_commit_kernel(const KvCommitParams p, int slices) {
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
  move_rows<kCommitLanes, 2>(c, base, bidb, part % slices * kCommitLanes * 8, len, 0, count,
                             [&](int i) { return len + list[i]; });
  if (p.weight != nullptr && part == 0) {
    float* w = p.weight + (int64_t)bidb * p.w_batch + (int64_t)kvh * p.w_head + len;
    for (int i0 = 0; i0 < p.sq; i0 += kMoveThreads) {
      const int i = i0 + (int)threadIdx.x;
      const float x = i < count ? w[list[i]] : 0.f;
      __syncthreads();                            // (waits for the loads: sources lie at or above i)
      if (i < p.sq) w[i] = x;
    }
  }
}

void launch_kv_evict(const KvEvictParams& p, hipStream_t stream) {
  const KvCache& c = p.c;
  hipLaunchKernelGGL(kv_select_kernel, dim3((unsigned)c.hk, (unsigned)c.b), dim3(kSelThreads), 0, stream, p);
  const int slices = (c.d + 8 * kEvictLanes - 1) / (8 * kEvictLanes);
  const int64_t grid = ((int64_t)c.b * c.hk + 7) / 8 * 8 * 2 * slices;
  if (grid > 0x7fffffff) throw std::runtime_error("kvcache evict: too many workgroups for one launch");
  hipLaunchKernelGGL(kv_evict_move_kernel, dim3((unsigned)grid), dim3(kMoveThreads), 0, stream, p, slices);
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) throw std::runtime_error(std::string("kvcache evict launch: ") + hipGetErrorString(e));
}

void launch_kv_commit(const KvCommitParams& p, hipStream_t stream) {
  const KvCache& c = p.c;
  const int slices = (c.d + 8 * kCommitLanes - 1) / (8 * kCommitLanes);
  const int64_t grid = (int64_t)c.b * c.hk * 2 * slices;
  if (grid > 0x7fffffff) throw std::runtime_error("kvcache commit: too many workgroups for one launch");
  hipLaunchKernelGGL(kv_commit_kernel, dim3((unsigned)grid), dim3(kMoveThreads), (unsigned)p.sq * sizeof(int), stream,
                     p, slices);
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) throw std::runtime_error(std::string("kvcache commit launch: ") + hipGetErrorString(e));
}

}  // namespace fa
