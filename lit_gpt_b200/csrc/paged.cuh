// A ragged step over a paged key-value cache: what its kernels (paged_attn.cu) are given.
#pragma once
#include "common.cuh"

namespace b200 {

constexpr int kMaxTiles = 1 << 29;          // of a step

struct PagedCut {                                           // what a CTA of paged_attn_tc05.cu goes on with that others began
  int first, last;                                          // the CTAs that have segments of it; last -1: it begins with an item of its own
  int count, row, gi;                                       // its queries, its first row, its group
};

struct PagedParams {
  const __nv_bfloat16* qkv;
  const void* cos; const void* sin;
  int table_bf16, table_rows, table_presel, rope_n, wide;   // wide: rows of heads and tables allow accesses of HS / 32 numbers
  const void* row_pos; int pos64;                           // position of every row in the rotation's tables
  const int* row_seq;                                       // sequence of every row
  const int4* seqs; int n_seqs;                             // first row, rows, keys in the cache before the step, row of the page table
  const int* pages; int64_t pages_ld; int page_rows, max_pages, pool, shift;   // page table (page_rows, max_pages), pages there are, log2 of a page's keys
  __nv_bfloat16* k; __nv_bfloat16* v; int64_t k_page, k_group, v_page, v_group;
  float* kw;                                                // [pool][n_groups][page] attention weight that every key has received; null: not wanted
  __nv_bfloat16* out;
  int rows, n_head, n_groups, per, max_length;
  __nv_bfloat16* q;                                         // the queries, turned: [n_groups][rows * per][HS]
  float* lse;                                               // [n_groups][rows * per] log2 of the sum of exponentials of a query's scores (with kw)
  int tile_rows;                                            // queries of an item
  int items;                                                // at most
  int workers, sms;                                         // warps that share the tiles, at most
  float* acc; float2* ml;                                   // results of key ranges: slots of tile_rows queries
  int2* where;                                              // per item: the first worker that has tiles of it, and how many workers have
  int list_max;                                             // sequences of more queries a group are left to the tensor memory (paged_attn_tc05.cu)
  int tc_rows;                                              // rows of a block of theirs: 256 queries at most
  int tc_workers;                                           // CTAs that share their tiles, at most
  float* tc_acc; float2* tc_ml; PagedCut* cuts;             // their results: two slots of 256 queries a CTA
  int* item_base;                                           // per sequence: its first item
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
  const bool fits = v.y > 0 && v.x >= 0 && v.x < p.rows && v.y <= p.rows - v.x && v.z >= 0 && v.w >= 0 && v.w < p.page_rows;
  q.rows = fits ? v.y : 0;
  q.cached = min(max(v.z, 0), p.max_length);
  q.n = fits ? min(q.cached + q.rows, p.max_length) : 0;
  return q;
}
// the page of keys [index << shift, ...) of a row of the page table; -1: there is none
__device__ __forceinline__ int page_at(const PagedParams& p, int table, int index) {
  if (index >= p.max_pages) return -1;
  const int id = p.pages[(int64_t)table * p.pages_ld + index];
  return id >= 0 && id < p.pool ? id : -1;
}

cudaError_t launch_paged_tc05(const PagedParams& p, int head_size, cudaStream_t st);   // rows of sequences of more than list_max queries a group

}  // namespace b200
