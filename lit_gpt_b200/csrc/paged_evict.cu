// Sequences of a paged key-value cache cut down by the attention weight that their keys have received: per sequence and group the first, the last and the heaviest keys stay, in order, at
// the front of the sequence's pages.
//
// One launch where a sequence's weights, places and pages fit into shared memory: a cluster of CTAs per sequence and group.  Every CTA finds the smallest weight that stays by radix
// selection over the weights as ordered whole numbers (11, 11 and 10 bits) and the places that stay by a scan, a run of keys a thread (of long sequences the cluster's CTAs each have a part of
// the keys); then the cluster moves keys, values and weights in place.  A key moves to a lower index or stays: a cluster that goes through its rows in order, reads a tile of them before it
// writes them, and has a barrier between, never writes what is still to be read.  What does not fit: a launch that chooses (weights read for every digit, eight bits each, and scanned in
// rounds), a launch that moves.
//
// Bound: bytes of the rows that stay, read and written, behind the choice, which is a chain.  us in a captured graph: 1 sequence of 32 groups cut from 576 keys to 512 9.3 (choice and
// move in two launches 14.3); 16 of 8 groups from 3001 - 8001 to 2048 58, 4.7 TB/s (two launches 77; pieces of 32 bytes of a row a CTA 119); 1 of 12 groups, 64 numbers a head,
// from 30001 to 8191 33 (two launches 151).  512 threads with twice the rows each: 62 and 50 (of 38, each CTA choosing for itself).
#include "common.cuh"

namespace b200 {

namespace {

constexpr int kChThreads = 1024, kChWarps = kChThreads / 32, kHistCopies = 8;
constexpr int kMvThreads = 256, kMvUnroll = 8;

struct EvictParams {
  __nv_bfloat16* k; __nv_bfloat16* v; int64_t k_page, k_group, v_page, v_group;
  float* kw;
  const int* pages; int64_t pages_ld; int table_seqs, max_pages, pool, shift;
  const int* lengths; const int* rows; int* lengths_out; int n_seqs, n_groups, keep, first, recent, max_length;
  int* from;      // [n_seqs][n_groups][keep]: where what moves to each place comes from
  int* moved;     // [n_seqs]: places, 0: the sequence stays as it is
};

__device__ __forceinline__ uint32_t ordered(float w) {   // greater numbers, greater keys; the two zeros are one; NaN above all
  if (w != w) return 0xffffffffu;
  const uint32_t u = __float_as_uint(w + 0.0f);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}

__global__ void __launch_bounds__(kChThreads) paged_choose_kernel(const EvictParams p) {
  __shared__ int s_hist[kHistCopies][256];
  __shared__ int s_warp[2][kChWarps];
  __shared__ int s_pick[2];
  griddep_wait();
  griddep_launch();
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, s = blockIdx.x / p.n_groups, g = blockIdx.x - s * p.n_groups, page = 1 << p.shift;
  const int n = p.lengths[s], row = p.rows ? p.rows[s] : s;
  bool cut = n > p.keep && n <= p.max_length && row >= 0 && row < p.table_seqs;
  const int* const table = p.pages + (int64_t)(cut ? row : 0) * p.pages_ld;
  if (cut) {
    bool all = true;
    for (int i = tid; i < (n + page - 1) >> p.shift; i += kChThreads) all = all && table[i] >= 0 && table[i] < p.pool;
    cut = __syncthreads_and(all);
  }
  if (g == 0 && tid == 0) {
    p.lengths_out[s] = cut ? p.keep : n;
    p.moved[s] = cut ? p.keep : 0;
  }
  if (!cut) return;
  auto at = [&](int i) -> float* { return p.kw + (((int64_t)table[i >> p.shift] * p.n_groups + g) << p.shift) + (i & (page - 1)); };
  const int lo = p.first, hi = n - p.recent;
  // the need-th largest of the weights between: `high` are its leading bits
  int need = p.keep - p.first - p.recent;
  uint32_t high = 0;
  for (int shift = 24; shift >= 0 && need > 0; shift -= 8) {
    for (int i = tid; i < kHistCopies * 256; i += kChThreads) (&s_hist[0][0])[i] = 0;
    __syncthreads();
    for (int i = lo + tid; i < hi; i += kChThreads) {
      const uint32_t u = ordered(*at(i));
      if (shift == 24 || u >> (shift + 8) == high) atomicAdd(&s_hist[warp % kHistCopies][(u >> shift) & 255u], 1);
    }
    __syncthreads();
    if (warp == 0) {   // lane l has digits 255 - 8 l down to 248 - 8 l
      int c[8], sum = 0;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        c[j] = 0;
        for (int k = 0; k < kHistCopies; ++k) c[j] += s_hist[k][255 - 8 * lane - j];
        sum += c[j];
      }
      int inc = sum;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) { const int t = __shfl_up_sync(0xffffffffu, inc, o); if (lane >= o) inc += t; }
      int before = inc - sum;
      if (before < need && need <= inc) {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          if (before < need && need <= before + c[j]) { s_pick[0] = 255 - 8 * lane - j; s_pick[1] = need - before; }
          before += c[j];
        }
      }
    }
    __syncthreads();
    high = (high << 8) | (uint32_t)s_pick[0];
    need = s_pick[1];
    __syncthreads();
  }
  const bool any = p.keep > p.first + p.recent;   // all of those above `high` and the first `need` of those that equal it
  int* const from = p.from + (int64_t)blockIdx.x * p.keep;
  int done = 0, equal = 0;                        // places filled and equal ones met before this round
  for (int i0 = 0; i0 < n; i0 += kChThreads) {
    const int i = i0 + tid;
    const float w = i < n ? *at(i) : 0.f;
    const uint32_t u = ordered(w);
    const bool mid = any && i >= lo && i < hi, tie = mid && u == high;
    const unsigned ties = __ballot_sync(0xffffffffu, tie);
    if (lane == 0) s_warp[0][warp] = __popc(ties);
    __syncthreads();
    int before = equal, total = equal;
    for (int k = 0; k < kChWarps; ++k) { if (k < warp) before += s_warp[0][k]; total += s_warp[0][k]; }
    equal = total;
    const bool stays = i < n && (i < lo || i >= hi || (mid && u > high) || (tie && before + __popc(ties & ((1u << lane) - 1u)) < need));
    const unsigned kept = __ballot_sync(0xffffffffu, stays);
    if (lane == 0) s_warp[1][warp] = __popc(kept);
    __syncthreads();                              // (and: every weight of this round has been read)
    int place = done;
    for (int k = 0; k < kChWarps; ++k) { if (k < warp) place += s_warp[1][k]; done += s_warp[1][k]; }
    if (stays) {
      place += __popc(kept & ((1u << lane) - 1u));
      from[place] = i;
      *at(place) = w;
    }
  }
}

// ---- the same with the sequence's weights, and the places that stay, in shared memory ----
constexpr int kBins = 2048, kBinCopies = 2;

// a's sum over the threads before this one
template <int THREADS>
__device__ __forceinline__ int block_before(int a, int* s_warp) {
  constexpr int WARPS = THREADS / 32;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int inc = a;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) { const int t = __shfl_up_sync(0xffffffffu, inc, o); if (lane >= o) inc += t; }
  __syncthreads();                                 // (s_warp has been read)
  if (lane == 31) s_warp[warp] = inc;
  __syncthreads();
  int w = lane < WARPS ? s_warp[lane] : 0;
#pragma unroll
  for (int o = 1; o < WARPS; o <<= 1) { const int t = __shfl_up_sync(0xffffffffu, w, o); if (lane >= o) w += t; }
  const int before = __shfl_sync(0xffffffffu, w, max(warp - 1, 0));
  return inc - a + (warp ? before : 0);
}

struct Held {                                      // in dynamic shared memory
  float* w;                                        // weights: of all keys, or of this CTA's
  int* from;                                       // [keep] where what moves to each place comes from
  int* table;                                      // the sequence's pages
};

__device__ __forceinline__ void cluster_sync() {
  __syncwarp();
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ uint32_t smem_of(const void* at, int rank) {   // the same place in another CTA of the cluster
  uint32_t a;
  asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"((uint32_t)__cvta_generic_to_shared(at)), "r"(rank));
  return a;
}
__device__ __forceinline__ int2 other_pair(const int* at, int rank) {
  int2 v;
  asm volatile("ld.shared::cluster.v2.s32 {%0, %1}, [%2];" : "=r"(v.x), "=r"(v.y) : "r"(smem_of(at, rank)) : "memory");
  return v;
}

// Whether the sequence is cut down; if so, its pages, its weights and the places that stay.  By every CTA for itself; or, SPLIT, by the cluster: each CTA has as many keys' weights, one part behind
// the other, and counts their digits, all add up the counts; what comes to a place is told the CTA that moves it (places go round by `tile`), and the weights move at once.
template <int THREADS, bool SPLIT>
__device__ __forceinline__ bool choose(const EvictParams& p, int s, int g, const Held& h, int rank, int ctas, int tile) {
  __shared__ __align__(8) int s_hist[kBinCopies * kBins];   // copies; SPLIT: this digit's and the one's before
  __shared__ __align__(8) int s_counts[2];                  // of this CTA's keys: above, equal
  __shared__ int s_warp[THREADS / 32], s_pick[2];
  const int tid = threadIdx.x, warp = tid >> 5, page = 1 << p.shift;
  const int n = p.lengths[s], row = p.rows ? p.rows[s] : s;
  bool cut = n > p.keep && n <= p.max_length && row >= 0 && row < p.table_seqs;
  if (!cut) return false;
  const int* const table = p.pages + (int64_t)row * p.pages_ld;
  bool all = true;
#pragma unroll 4
  for (int i = tid; i < (n + page - 1) >> p.shift; i += THREADS) {
    const int id = table[i];
    h.table[i] = id;
    all = all && id >= 0 && id < p.pool;
  }
  cut = __syncthreads_and(all);
  if (!cut) return false;
  const int each = SPLIT ? (n + ctas - 1) / ctas : n, k0 = SPLIT ? min(rank * each, n) : 0, k1 = SPLIT ? min(k0 + each, n) : n;   // keys that this CTA looks at
  auto at = [&](int i) -> float* { return p.kw + (((int64_t)h.table[i >> p.shift] * p.n_groups + g) << p.shift) + (i & (page - 1)); };
#pragma unroll 8
  for (int i = k0 + tid; i < k1; i += THREADS) h.w[i - k0] = *at(i);
  const int lo = p.first, hi = n - p.recent;
  int need = p.keep - p.first - p.recent;
  const bool any = need > 0;
  uint32_t high = 0;
  // digits of 11, 11 and 10 bits
  for (int digit = 0; digit < 3 && any; ++digit) {
    const int shift = digit == 0 ? 21 : digit == 1 ? 10 : 0, bits = digit == 2 ? 10 : 11;
    int* const hist = SPLIT ? s_hist + (digit & 1) * kBins : s_hist;
    for (int i = tid; i < (SPLIT ? 1 : kBinCopies) * kBins; i += THREADS) hist[i] = 0;
    __syncthreads();                               // (and: the weights are there)
    int* const mine = SPLIT ? hist : hist + warp % kBinCopies * kBins;
#pragma unroll 4
    for (int i = max(lo, k0) + tid; i < min(hi, k1); i += THREADS) {
      const uint32_t u = ordered(h.w[i - k0]);
      if (digit == 0 || u >> (shift + bits) == high) atomicAdd(&mine[(u >> shift) & ((1u << bits) - 1u)], 1);
    }
    if (SPLIT) cluster_sync();                     // (who is past it has read the counts of the digit before)
    else __syncthreads();
    // a thread has two digits next to each other, the greater one first
    static_assert(kBins == 2 * THREADS, "two digits a thread");
    const int top = kBins - 1 - 2 * tid;
    int c[2] = {0, 0};
    if (SPLIT) {
#pragma unroll 8
      for (int k = 0; k < ctas; ++k) {
        const int2 v = other_pair(hist + top - 1, k);
        c[0] += v.y;
        c[1] += v.x;
      }
    } else {
#pragma unroll
      for (int k = 0; k < kBinCopies; ++k) {
        c[0] += hist[k * kBins + top];
        c[1] += hist[k * kBins + top - 1];
      }
    }
    int before = block_before<THREADS>(c[0] + c[1], s_warp);
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      if (before < need && need <= before + c[j]) { s_pick[0] = top - j; s_pick[1] = need - before; }
      before += c[j];
    }
    __syncthreads();
    high = (high << bits) | (uint32_t)s_pick[0];
    need = s_pick[1];
    __syncthreads();
  }
  if (!any) __syncthreads();                       // (the weights are there)
  // a run of keys a thread, an odd number of them so that the threads meet all banks: those above, and the first `need` of those that equal it
  const int run = ((k1 - k0 + THREADS - 1) / THREADS) | 1, begin = min(k1, k0 + tid * run), end = min(k1, begin + run);
  int above = 0, ties = 0;
#pragma unroll 4
  for (int i = begin; i < end; ++i) {
    const uint32_t u = ordered(h.w[i - k0]);
    const bool mid = i >= lo && i < hi;
    above += !mid || (any && u > high);
    ties += mid && any && u == high;
  }
  int above_before = block_before<THREADS>(above, s_warp);
  int equal = block_before<THREADS>(ties, s_warp);
  if (SPLIT) {
    if (tid == THREADS - 1) { s_counts[0] = above_before + above; s_counts[1] = equal + ties; }
    cluster_sync();                                // (and: every weight has been read)
    for (int k = 0; k < rank; ++k) {
      const int2 v = other_pair(s_counts, k);
      above_before += v.x;
      equal += v.y;
    }
  }
  int place = above_before + min(equal, need);
  for (int i = begin; i < end; ++i) {
    const float w = h.w[i - k0];
    const uint32_t u = ordered(w);
    const bool mid = i >= lo && i < hi, tie = mid && any && u == high;
    if (!mid || (any && u > high) || (tie && equal < need)) {
      if (SPLIT) {
        asm volatile("st.shared::cluster.s32 [%0], %1;" ::"r"(smem_of(h.from + place, place / tile % ctas)), "r"(i) : "memory");
        *at(place) = w;
      } else {
        h.from[place] = i;
      }
      ++place;
    }
    equal += tie;
  }
  if (SPLIT) cluster_sync();
  else __syncthreads();
  return true;
}
__device__ __forceinline__ Held held_of(const EvictParams& p, float* smem, int parts) {
  Held h;
  h.w = smem;
  h.from = reinterpret_cast<int*>(smem + (p.max_length + parts - 1) / parts);
  h.table = h.from + p.keep;
  return h;
}

// ---- the whole of it in one launch ----
// A cluster of CTAs per sequence and group: each of them chooses for itself, from weights that all have read before the first is written, or they choose together; then they share the rows.
constexpr int kEvThreads = 1024, kEvUnroll = 2;

template <int LANES, bool SPLIT>
__global__ void __launch_bounds__(kEvThreads) paged_evict_kernel(const EvictParams p, int ctas) {
  extern __shared__ __align__(16) float ev_smem[];
  griddep_launch();
  griddep_wait();
  const int tid = threadIdx.x, rank = blockIdx.x % ctas, item = blockIdx.x / ctas, s = item / p.n_groups, g = item - s * p.n_groups, page = 1 << p.shift;
  constexpr int ROWS = kEvThreads / LANES, TILE = ROWS * kEvUnroll;   // at once; of a tile
  const Held h = held_of(p, ev_smem, SPLIT ? ctas : 1);
  const bool cut = choose<kEvThreads, SPLIT>(p, s, g, h, rank, ctas, TILE);
  if (g == 0 && rank == 0 && tid == 0) p.lengths_out[s] = cut ? p.keep : p.lengths[s];
  if (!cut) return;                                // (the whole cluster)
  const float* const s_w = h.w;
  const int* const s_from = h.from;
  const int* const s_table = h.table;
  auto at = [&](int i) -> float* { return p.kw + (((int64_t)s_table[i >> p.shift] * p.n_groups + g) << p.shift) + (i & (page - 1)); };
  // ---- the rows.  A tile is read while the one before it is still in registers: its rows lie behind all places of that one ----
  const int keep = p.keep, hs = LANES * 8, first = rank * TILE + tid / LANES, step = ctas * TILE, lane8 = tid % LANES * 8;
  __nv_bfloat16* const kg = p.k + (int64_t)g * p.k_group + lane8;
  __nv_bfloat16* const vg = p.v + (int64_t)g * p.v_group + lane8;
  auto key_at = [&](int i) { return reinterpret_cast<uint4*>(kg + (int64_t)s_table[i >> p.shift] * p.k_page + (i & (page - 1)) * hs); };
  auto value_at = [&](int i) { return reinterpret_cast<uint4*>(vg + (int64_t)s_table[i >> p.shift] * p.v_page + (i & (page - 1)) * hs); };
  uint4 kx[kEvUnroll], vx[kEvUnroll];
  auto load = [&](int d0) {
#pragma unroll
    for (int j = 0; j < kEvUnroll; ++j) {
      const int d = d0 + first + j * ROWS;
      if (d < keep) {
        const int f = s_from[d];
        kx[j] = *key_at(f);
        vx[j] = *value_at(f);
      }
    }
  };
  load(0);
  for (int d0 = 0; d0 < keep; d0 += step) {        // (as many rounds in every thread)
    uint4 ky[kEvUnroll], vy[kEvUnroll];
#pragma unroll
    for (int j = 0; j < kEvUnroll; ++j) { ky[j] = kx[j]; vy[j] = vx[j]; }
    load(d0 + step);
    // this tile, and the first time the weights, have been read by all
    if (ctas == 1) __syncthreads();
    else cluster_sync();
    if (!SPLIT && d0 == 0) {
#pragma unroll 4
      for (int d = rank * kEvThreads + tid; d < keep; d += ctas * kEvThreads) *at(d) = s_w[s_from[d]];
    }
#pragma unroll
    for (int j = 0; j < kEvUnroll; ++j) {
      const int d = d0 + first + j * ROWS;
      if (d < keep) {
        *key_at(d) = ky[j];
        *value_at(d) = vy[j];
      }
    }
  }
}

// LANES lanes of 16 bytes each a row; the CTAs of a cluster share the rows of a sequence, group and tensor, a tile each at a time.  A tile is read while the one before it is still in
// registers: its rows lie behind all places of that one.
template <int LANES>
__global__ void __launch_bounds__(kMvThreads) paged_move_kernel(const EvictParams p, int ctas) {
  constexpr int ROWS = kMvThreads / LANES, TILE = ROWS * kMvUnroll;        // at once; of a tile
  griddep_launch();
  griddep_wait();
  const int rank = blockIdx.x % ctas, item = blockIdx.x / ctas, s = item / p.n_groups, g = item - s * p.n_groups, page = 1 << p.shift;
  const int keep = p.moved[s];
  if (keep == 0) return;
  const int hs = LANES * 8, row = rank * TILE + (int)threadIdx.x / LANES;
  const int* const table = p.pages + (int64_t)(p.rows ? p.rows[s] : s) * p.pages_ld;
  const int* const from = p.from + (int64_t)item * p.keep;
  const int64_t apart = blockIdx.y ? p.v_page : p.k_page;
  __nv_bfloat16* const base = (blockIdx.y ? p.v + (int64_t)g * p.v_group : p.k + (int64_t)g * p.k_group) + threadIdx.x % LANES * 8;
  auto at = [&](int i) { return reinterpret_cast<uint4*>(base + (int64_t)table[i >> p.shift] * apart + (int64_t)(i & (page - 1)) * hs); };
  uint4 x[kMvUnroll];
  int f[kMvUnroll];
  auto indices = [&](int d0) {
#pragma unroll
    for (int j = 0; j < kMvUnroll; ++j) {
      const int d = d0 + row + j * ROWS;
      f[j] = d < keep ? from[d] : -1;
    }
  };
  auto load = [&]() {
#pragma unroll
    for (int j = 0; j < kMvUnroll; ++j)
      if (f[j] >= 0) x[j] = *at(f[j]);
  };
  const int step = ctas * TILE;
  indices(0);
  load();
  indices(step);
  for (int d0 = 0; d0 < keep; d0 += step) {        // (as many rounds in every thread)
    uint4 y[kMvUnroll];
#pragma unroll
    for (int j = 0; j < kMvUnroll; ++j) y[j] = x[j];
    load();                                        // of the next tile
    indices(d0 + 2 * step);
    // this tile has been read by all
    if (ctas == 1) __syncthreads();
    else cluster_sync();
#pragma unroll
    for (int j = 0; j < kMvUnroll; ++j) {
      const int d = d0 + row + j * ROWS;
      if (d < keep) *at(d) = y[j];
    }
  }
}

constexpr int kHeldMax = 200 * 1024;              // shared memory for weights, places and pages
// Of more keys a cluster chooses together: its barriers and the counts' way between SMs are 10 us, a CTA's own choice of 30000 keys 22.  us, alone and together: 1 sequence of 8 groups from 8000 to
// 2000 17.7, 22.0; from 16384 to 4096 28.1, 28.3; 12 groups, 64 numbers a head, from 30001 to 8191 38.6, 32.9; 4 groups from 100000 to 4000 350 (two launches), 31.
constexpr int kSplitMin = 16384;

// Clusters of 2, 4, 8 CTAs that this device runs at once: what its SMs come in leaves some of them without (B200: 74, 33, 15 with a CTA an SM, and not 74, 37, 18; a cluster more and all wait for a
// second round: 36 groups cut from 3000 to 2000 in clusters of 4 35.9 us, of 2 27.5; 16 in clusters of 8 26.4, of 4 18.5).
constexpr int kDevices = 64;
std::atomic<int> g_clusters[kDevices][3];
cudaError_t evict_configure() {
  static PerDeviceOnce once;
  if (!once.need()) return cudaSuccess;
  for (auto* k : {paged_evict_kernel<8, false>, paged_evict_kernel<8, true>, paged_evict_kernel<16, false>, paged_evict_kernel<16, true>}) {
    const cudaError_t e = cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, kHeldMax);
    if (e != cudaSuccess) return e;
  }
  int device = 0;
  cudaError_t e = cudaGetDevice(&device);
  for (int i = 0; e == cudaSuccess && i < 3; ++i) {
    cudaLaunchAttribute attr = {};
    attr.id = cudaLaunchAttributeClusterDimension;
    attr.val.clusterDim.x = 2u << i;
    attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(2u << i);
    cfg.blockDim = dim3(kEvThreads);
    cfg.dynamicSmemBytes = kHeldMax;
    cfg.attrs = &attr;
    cfg.numAttrs = 1;
    int n = 0;
    e = cudaOccupancyMaxActiveClusters(&n, paged_evict_kernel<16, false>, &cfg);
    if (device < kDevices) g_clusters[device][i].store(n, std::memory_order_relaxed);
  }
  if (e == cudaSuccess) once.done();
  return e;
}
int clusters_at_once(int ctas) {
  int device = 0;
  if (cudaGetDevice(&device) != cudaSuccess || device >= kDevices) return 0;
  return g_clusters[device][ctas == 2 ? 0 : ctas == 4 ? 1 : 2].load(std::memory_order_relaxed);
}

int64_t evict_held(int64_t max_length, int64_t keep, int page, int parts) { return ((max_length + parts - 1) / parts + keep + (max_length + page - 1) / page) * 4; }
size_t evict_bytes(int n_seqs, int n_groups, int64_t keep, int64_t max_length, int page) {   // (more than a cluster needs that holds the weights together)
  return evict_held(max_length, keep, page, 1) <= kHeldMax ? 0 : ((size_t)n_seqs * n_groups * keep + n_seqs) * sizeof(int);
}

}  // namespace
}  // namespace b200

using namespace b200;

extern "C" {

size_t b200_evict_paged_workspace_bytes(int n_seqs, int n_groups, int64_t keep, int64_t max_length, int page) {
  if (n_seqs <= 0 || n_groups <= 0 || keep <= 0 || keep >= max_length || max_length >= (1 << 30) || page <= 0) return 0;
  return evict_bytes(n_seqs, n_groups, keep, max_length, page);
}

int b200_evict_paged(const b200_evict_paged_args* a, b200_stream_t stream) {
  B200_CHECK_ARG(a, "b200_evict_paged: null argument");
  B200_CHECK_ARG(a->head_size == 64 || a->head_size == 128, "b200_evict_paged: head size %d (64 or 128)", a->head_size);
  B200_CHECK_ARG(a->n_seqs > 0 && a->n_groups > 0 && (int64_t)a->n_seqs * a->n_groups < (1 << 24), "b200_evict_paged: %d sequences of %d groups", a->n_seqs, a->n_groups);
  B200_CHECK_ARG(a->page >= 16 && a->page <= 256 && (a->page & (a->page - 1)) == 0, "b200_evict_paged: pages of %d keys (16, 32, 64, 128 or 256)", a->page);
  B200_CHECK_ARG(a->pool > 0 && a->table_seqs > 0 && a->max_pages > 0 && a->pages_ld >= a->max_pages, "b200_evict_paged: no pages, or a bad page table");
  B200_CHECK_ARG(a->rows || a->table_seqs >= a->n_seqs, "b200_evict_paged: a page table of %d rows for %d sequences", a->table_seqs, a->n_seqs);
  B200_CHECK_ARG(a->max_length > 0 && a->max_length <= (int64_t)a->max_pages * a->page && a->max_length < (1 << 30), "b200_evict_paged: %lld keys in %d pages of %d",
                 (long long)a->max_length, a->max_pages, a->page);
  B200_CHECK_ARG(a->keep > 0 && a->first >= 0 && a->recent >= 0 && a->first <= a->keep && a->recent <= a->keep - a->first, "b200_evict_paged: %lld first and %lld recent keys of %lld to keep",
                 (long long)a->first, (long long)a->recent, (long long)a->keep);
  B200_CHECK_ARG(a->k_pages && a->v_pages && a->key_weights && a->pages && a->lengths && a->lengths_out, "b200_evict_paged: null pointer");
  B200_CHECK_ARG(a->lengths != a->lengths_out, "b200_evict_paged: lengths_out in the place of lengths");
  B200_CHECK_ARG((((uintptr_t)a->k_pages | (uintptr_t)a->v_pages) & 15) == 0 && ((a->k_page_stride | a->k_group_stride | a->v_page_stride | a->v_group_stride) & 7) == 0 &&
                     (((uintptr_t)a->key_weights | (uintptr_t)a->workspace) & 3) == 0,
                 "b200_evict_paged: pages must lie on 16-byte boundaries");
  if (a->keep >= a->max_length) {   // nothing is longer
    B200_CUDA(cudaMemcpyAsync(a->lengths_out, a->lengths, sizeof(int) * (size_t)a->n_seqs, cudaMemcpyDeviceToDevice, (cudaStream_t)stream));
    return B200_OK;
  }
  const size_t need = evict_bytes(a->n_seqs, a->n_groups, a->keep, a->max_length, a->page);
  B200_CHECK_ARG(a->workspace_bytes >= need && (a->workspace || need == 0), "b200_evict_paged: workspace too small");
  EvictParams p = {};
  p.k = (__nv_bfloat16*)a->k_pages; p.v = (__nv_bfloat16*)a->v_pages;
  p.k_page = a->k_page_stride; p.k_group = a->k_group_stride; p.v_page = a->v_page_stride; p.v_group = a->v_group_stride;
  p.kw = a->key_weights;
  p.pages = a->pages; p.pages_ld = a->pages_ld; p.table_seqs = a->table_seqs; p.max_pages = a->max_pages; p.pool = a->pool;
  for (p.shift = 4; (1 << p.shift) < a->page; ++p.shift) {}
  p.lengths = a->lengths; p.rows = a->rows; p.lengths_out = a->lengths_out; p.n_seqs = a->n_seqs; p.n_groups = a->n_groups;
  p.keep = (int)a->keep; p.first = (int)a->first; p.recent = (int)a->recent; p.max_length = (int)a->max_length;
  p.from = (int*)a->workspace;
  p.moved = p.from + (int64_t)a->n_seqs * a->n_groups * a->keep;
  const cudaStream_t st = (cudaStream_t)stream;
  const unsigned items = (unsigned)(a->n_seqs * a->n_groups);
  const int lanes = a->head_size / 8;
  B200_CUDA(evict_configure());
  // as many CTAs for a sequence and group as run at once, no more than they have tiles unless they choose together
  const int tile = kEvThreads / lanes * kEvUnroll;
  int ctas = 1;
  while (ctas < 8 && items <= (unsigned)clusters_at_once(2 * ctas) && (ctas * tile < a->keep || a->max_length > kSplitMin)) ctas *= 2;
  const bool split = ctas > 1 && a->max_length > kSplitMin;
  const int64_t held = evict_held(a->max_length, a->keep, a->page, split ? ctas : 1);
  if (held <= kHeldMax) {
    auto* const kernel = lanes == 8 ? (split ? paged_evict_kernel<8, true> : paged_evict_kernel<8, false>) : split ? paged_evict_kernel<16, true> : paged_evict_kernel<16, false>;
    B200_CUDA(launch_cluster(kernel, dim3(items * ctas), dim3(kEvThreads), ctas, (size_t)held, st, p, ctas));
    return B200_OK;
  }
  B200_CUDA(launch(paged_choose_kernel, dim3(items), dim3(kChThreads), 0, st, p));
  // as many CTAs for the rows of one tensor as leave none of the SMs without, no more than they have tiles
  const int rows = kMvThreads / lanes * kMvUnroll;
  ctas = 1;
  while (ctas < 8 && (int64_t)items * 2 * ctas < sm_count() && ctas * rows < a->keep) ctas *= 2;
  B200_CUDA(launch_cluster(lanes == 8 ? paged_move_kernel<8> : paged_move_kernel<16>, dim3(items * ctas, 2), dim3(kMvThreads), ctas, 0, st, p, ctas));
  return B200_OK;
}

}  // extern "C"
