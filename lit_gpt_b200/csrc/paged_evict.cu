// Sequences of a paged key-value cache cut down by the attention weight that their keys have received: per sequence and group the first, the last and the heaviest keys stay, in order, at
// the front of the sequence's pages.
//
// Two launches.  paged_choose_kernel, a CTA per sequence and group: the smallest weight that stays by radix selection over the weights as ordered whole numbers, eight bits at a time; then
// the indices that stay, in order, by a scan, and their weights moved.  paged_move_kernel: keys and values moved in place, a CTA per sequence, group, tensor and slice of the columns.
// A key moves to a lower index or stays, and slices of columns share nothing: a CTA that goes through its rows in order, reads a tile of them before it writes them, and has a
// barrier between, never writes what is still to be read.
//
// Bound: bytes of the rows that stay, read and written.
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

// LANES lanes of 16 bytes each a row
template <int LANES>
__global__ void __launch_bounds__(kMvThreads) paged_move_kernel(const EvictParams p) {
  constexpr int ROWS = kMvThreads / LANES;        // at once
  griddep_launch();
  griddep_wait();
  const int s = blockIdx.x / p.n_groups, g = blockIdx.x - s * p.n_groups, page = 1 << p.shift;
  const int keep = p.moved[s];
  if (keep == 0) return;
  const int hs = (int)gridDim.z * LANES * 8;
  const int* const table = p.pages + (int64_t)(p.rows ? p.rows[s] : s) * p.pages_ld;
  const int* const from = p.from + (int64_t)blockIdx.x * p.keep;
  const int64_t apart = blockIdx.y ? p.v_page : p.k_page;
  __nv_bfloat16* const base = (blockIdx.y ? p.v + (int64_t)g * p.v_group : p.k + (int64_t)g * p.k_group) + blockIdx.z * LANES * 8 + threadIdx.x % LANES * 8;
  auto at = [&](int i) { return reinterpret_cast<uint4*>(base + (int64_t)table[i >> p.shift] * apart + (int64_t)(i & (page - 1)) * hs); };
  for (int d0 = (int)threadIdx.x / LANES; d0 < keep + (int)threadIdx.x / LANES; d0 += ROWS * kMvUnroll) {   // (as many rounds in every thread)
    uint4 x[kMvUnroll];
#pragma unroll
    for (int j = 0; j < kMvUnroll; ++j) {
      const int d = d0 + j * ROWS;
      if (d < keep) x[j] = *at(from[d]);
    }
    __syncthreads();
#pragma unroll
    for (int j = 0; j < kMvUnroll; ++j) {
      const int d = d0 + j * ROWS;
      if (d < keep) *at(d) = x[j];
    }
  }
}

size_t evict_bytes(int n_seqs, int n_groups, int64_t keep) { return ((size_t)n_seqs * n_groups * keep + n_seqs) * sizeof(int); }

}  // namespace
}  // namespace b200

using namespace b200;

extern "C" {

size_t b200_evict_paged_workspace_bytes(int n_seqs, int n_groups, int64_t keep) {
  if (n_seqs <= 0 || n_groups <= 0 || keep <= 0 || keep >= (1 << 30)) return 0;
  return evict_bytes(n_seqs, n_groups, keep);
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
  B200_CHECK_ARG(a->k_pages && a->v_pages && a->key_weights && a->pages && a->lengths && a->lengths_out && a->workspace, "b200_evict_paged: null pointer");
  B200_CHECK_ARG(a->lengths != a->lengths_out, "b200_evict_paged: lengths_out in the place of lengths");
  B200_CHECK_ARG((((uintptr_t)a->k_pages | (uintptr_t)a->v_pages) & 15) == 0 && ((a->k_page_stride | a->k_group_stride | a->v_page_stride | a->v_group_stride) & 7) == 0 &&
                     (((uintptr_t)a->key_weights | (uintptr_t)a->workspace) & 3) == 0,
                 "b200_evict_paged: pages must lie on 16-byte boundaries");
  if (a->keep >= a->max_length) {   // nothing is longer
    B200_CUDA(cudaMemcpyAsync(a->lengths_out, a->lengths, sizeof(int) * (size_t)a->n_seqs, cudaMemcpyDeviceToDevice, (cudaStream_t)stream));
    return B200_OK;
  }
  B200_CHECK_ARG(a->workspace_bytes >= evict_bytes(a->n_seqs, a->n_groups, a->keep), "b200_evict_paged: workspace too small");
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
  B200_CUDA(launch(paged_choose_kernel, dim3(items), dim3(kChThreads), 0, st, p));
  B200_CUDA(launch(paged_move_kernel<2>, dim3(items, 2, (unsigned)(a->head_size / 16)), dim3(kMvThreads), 0, st, p));
  return B200_OK;
}

}  // extern "C"
