// A ragged step over a paged key-value cache: what its kernels (paged_attn.cu) are given.
#pragma once
#include "tc05.cuh"

namespace b200 {

constexpr int kMaxTiles = 1 << 29;          // of a step

constexpr int kCutNothing = -2;
struct PagedCut {                                           // what a CTA of paged_attn_tc05.cu goes on with that others began
  int first, last;                                          // the CTAs that have segments of it; last -1: it begins with an item of its own, kCutNothing: nothing was done
  int count, row, gi;                                       // its queries, its first row, its group
};

struct PagedWeightCut {                                     // a block of 128 keys that several CTAs of paged_weights.cu have parts of
  int first, last;                                          // those CTAs; last -1: none to join
  int s, table, cached, n, row, gi, block;                  // its sequence, and that one's first row
};

struct PagedParams {
  const __nv_bfloat16* qkv;
  const void* cos; const void* sin;
  int table_bf16, table_rows, table_presel, rope_n, wide;   // wide: rows of heads and tables allow accesses of HS / 32 numbers
  const void* row_pos; int pos64;                           // position of every row in the rotation's tables
  const int* row_seq;                                       // sequence of every row: one that is not the sequence's whose range holds it takes no part
  const int4* seqs; int n_seqs;                             // first row, rows, keys in the cache before the step, row of the page table
  const int* pages; int64_t pages_ld; int page_rows, max_pages, pool, shift;   // page table (page_rows, max_pages), pages there are, log2 of a page's keys
  __nv_bfloat16* k; __nv_bfloat16* v; int64_t k_page, k_group, v_page, v_group;
  float* kw;                                                // [pool][n_groups][page] attention weight that every key has received; null: not wanted
  __nv_bfloat16* out;
  int rows, n_head, n_groups, per, max_rows, max_length;
  __nv_bfloat16* q;                                         // the queries, turned: [n_groups][rows * per][HS]
  float* lse;                                               // [n_groups][rows * per] log2 of the sum of exponentials of a query's scores (with kw); inf: it sees no key; NaN: a score is
  int tile_rows;                                            // queries of an item
  int items;                                                // at most
  int workers, sms;                                         // warps that share the tiles, at most
  float* acc; float2* ml;                                   // results of key ranges: slots of tile_rows queries
  int2* where;                                              // per item: the first worker that has tiles of it, and how many workers have
  int mixed, list_ns, tensor_ns;                            // the list beside the tensor memory; what a tile of either takes
  int list_max;                                             // sequences of more queries a group are left to the tensor memory (paged_attn_tc05.cu)
  int tc_rows;                                              // rows of a block of theirs: 256 queries at most
  int tc_workers;                                           // CTAs that share their tiles, at most
  float* tc_acc; float2* tc_ml; PagedCut* cuts;             // their results: two slots of 256 queries a CTA
  float* scores; int score_rows, kept_max;                  // scores of the list's tiles, that many queries each; of sequences of up to kept_max queries a group (0: none are kept)
  int kw_workers; float* kw_part; PagedWeightCut* kw_cuts;  // CTAs that compute the others' again, their sums: two slots of 128 keys a CTA
  int* tile_base;                                           // per sequence: its first tile in the list; -1: nothing was done
  int* item_base;                                           // per sequence: its first item; -1 likewise
  int ways;                                                 // warps that join a head's results
  float scale_log2;
};

// A sequence of the step as the kernels use it: nothing in it reaches beyond the rows, the page table or max_length.
struct PagedSeq {
  int first, rows;   // its rows; none where the description does not fit
  int cached, n;     // keys before the step, keys behind it
  int table;
};
__device__ __forceinline__ PagedSeq paged_seq(const PagedParams& p, int s) {
  const int4 v = p.seqs[s];
  PagedSeq q;
  q.first = v.x;
  q.table = v.w;
  const bool fits = v.y > 0 && v.x >= 0 && v.x < p.rows && v.y <= p.rows - v.x && v.y <= p.max_rows && v.z >= 0 && v.w >= 0 && v.w < p.page_rows;
  q.rows = fits ? v.y : 0;
  q.cached = min(max(v.z, 0), p.max_length);
  q.n = fits ? min(q.cached + q.rows, p.max_length) : 0;
  return q;
}
__device__ __forceinline__ int seq_items(const PagedParams& p, const PagedSeq& s) {   // of the list, of a group
  return s.rows > 0 && s.rows * p.per <= p.list_max ? (s.rows * p.per + p.tile_rows - 1) / p.tile_rows : 0;
}
__device__ __forceinline__ int seq_tiles(const PagedSeq& s) { return (s.n + 31) / 32; }

// Single tokens beside chunks: the list and the tensor memory run at the same time, on SMs of their own, as many as their work (in ns, of a group) asks for.  Both kernels come to the same
// numbers, whole ones, each from its own look at the sequences.  What a step of either costs an SM: 16 KB of keys and values at 45 GB/s, 128 keys of 256 queries 3.4 us (beside the list; 2.1 alone); half heads 0.5 and
// 0.75 of it.  us in a captured graph, when this was chosen, one after the other and so: 32 tokens over 100 - 3001 keys beside 512 rows, 8 groups of 4 heads, 89, 75; 3 over 16000 beside 512 81, 78; 8
// over 300 beside 64, 32 groups, 32, 26; 64 over 500 beside 1000 rows behind 3000 131, 134; 2 over 100 beside 2048 103, 102.  (With 2.1 us 88, 98, 28, 142, 102; with 4.2 73, 73, 26, 150, 102.)  Since the
// tensor memory's waits are shorter code: 74, 75, 27, 125, 96.
struct Shares { unsigned long long list, tensor; };
__device__ __forceinline__ void add_work(const PagedParams& p, const PagedSeq& s, Shares& w) {
  w.list += (unsigned long long)seq_items(p, s) * seq_tiles(s) * p.list_ns;
  if (s.rows > 0 && s.rows * p.per > p.list_max) {
    const int blocks = (s.rows + p.tc_rows - 1) / p.tc_rows;
    w.tensor += (unsigned long long)blocks * (2 + (s.n - s.rows / 2 + 127) / 128) * p.tensor_ns;
  }
}
__device__ __forceinline__ int tensor_share(const PagedParams& p, const Shares& w) {   // of the SMs
  if (w.list == 0) return p.sms;
  if (w.tensor == 0) return 0;
  const double f = (double)w.tensor / ((double)w.tensor + (double)w.list);
  return min(max((int)(f * p.sms + 0.5), 1), p.sms - 1);
}

// the page of keys [index << shift, ...) of a row of the page table; -1: there is none
__device__ __forceinline__ int page_at(const PagedParams& p, int table, int index) {
  if (index >= p.max_pages) return -1;
  const int id = p.pages[(int64_t)table * p.pages_ld + index];
  return id >= 0 && id < p.pool ? id : -1;
}

// The page of key `key` of sequence s; -1: there is no such key, since it has no page or, of the step's own, its row is not the sequence's
__device__ __forceinline__ int whose_key(const PagedParams& p, int s, int cached, int first_row, int key) { return key < cached ? s : p.row_seq[first_row + key - cached]; }
__device__ __forceinline__ int key_page(const PagedParams& p, int s, int table, int cached, int first_row, int n, int key) {
  if (key >= n) return -1;
  const int whose = whose_key(p, s, cached, first_row, key), id = page_at(p, table, key >> p.shift);   // (both on their way at once)
  return whose == s ? id : -1;
}

__device__ __forceinline__ int capped(int64_t x) { return (int)(x < kMaxTiles ? x : kMaxTiles); }

// A box of 64 numbers of min(page, 128) keys, 128-byte-swizzled
__device__ __forceinline__ void load_page(uint32_t dst, const CUtensorMap* map, int x, int row, int group, int page, uint32_t bar) {
  asm volatile("cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], [%6];"
               ::"r"(dst), "l"(map), "r"(x), "r"(row), "r"(group), "r"(page), "r"(bar) : "memory");
}
inline bool page_map(CUtensorMap* map, const void* base, int hs, int page, int groups, int pool, int64_t group, int64_t apart) {
  const TensorMapEncodeFn enc = tensor_map_encoder();
  if (!enc) return false;
  // (a single group's, or a single page's, distance is not used, but has to be one)
  if (group == 0) group = (int64_t)page * hs;
  if (apart == 0) apart = (int64_t)page * hs;
  const cuuint64_t dim[4] = {(cuuint64_t)hs, (cuuint64_t)page, (cuuint64_t)groups, (cuuint64_t)pool};
  const cuuint64_t stride[3] = {(cuuint64_t)hs * 2, (cuuint64_t)group * 2, (cuuint64_t)apart * 2};
  const cuuint32_t box[4] = {64u, (cuuint32_t)(page < 128 ? page : 128), 1u, 1u};
  const cuuint32_t step[4] = {1u, 1u, 1u, 1u};
  return enc(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 4, const_cast<void*>(base), dim, stride, box, step, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
             CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

cudaError_t launch_paged_weights(const PagedParams& p, int head_size, cudaStream_t st);   // what the keys of sequences of more than kept_max queries a group receive
cudaError_t launch_paged_tc05(const PagedParams& p, int head_size, cudaStream_t st);   // rows of sequences of more than list_max queries a group

}  // namespace b200
