// A decode step of rows that share a prefix: what its kernels (attn_shared.cu, attn_shared_tc05.cu) are given.
#pragma once
#include "common.cuh"

namespace b200 {

struct SharedParams {
  const __nv_bfloat16* qkv;
  const void* cos; const void* sin;
  int table_bf16, table_rows, table_presel, rope_n, wide;   // wide: rows of heads and tables allow accesses of HS / 32 numbers
  const void* pos; int pos64, pos_each;      // pos_each: one position per row
  const void* plen; int plen64;              // null: prefix_rows
  __nv_bfloat16* kc; __nv_bfloat16* vc; int64_t kc_b, kc_g, vc_b, vc_g;
  const __nv_bfloat16* kp; const __nv_bfloat16* vp; int64_t kp_g, vp_g;
  __nv_bfloat16* out;
  int batch, n_head, n_groups, per, own_rows, prefix_rows;
  int head_tiles, row_tiles, tile_rows;      // tiles of 16 heads of a row's group; tiles of a group's query rows over the prefix, of so many rows
  __nv_bfloat16* q;                          // the queries, turned: [n_groups][batch * per][HS]
  int workers, sms;                          // warps that share the tiles, at most
  float* own_acc; float2* own_ml;            // results of key ranges of own items: slots of min(16, per) rows
  float* pre_acc; float2* pre_ml;            // of prefix items: slots of tile_rows rows
  int2* own_where; int2* pre_where;          // per item of the list: the first worker that has tiles of it, and how many workers have
  int ways;                                  // warps that join a head's results
  // On the tensor memory (attn_shared_tc05.cu) prefix items are 128 or 256 query rows of a group, with `pre_parts` results each, in slots of `pre_rows` rows, item after item;
  // row_tiles is 0 then.  pre_parts 0: the prefix is in the list of tiles.
  int pre_parts, pre_rows, pre_tiles;        // pre_tiles: items of a group
  float scale_log2;
};

__device__ __forceinline__ int64_t index_at(const void* p, int is64, int64_t i) {
  return is64 ? reinterpret_cast<const int64_t*>(p)[i] : (int64_t)reinterpret_cast<const int32_t*>(p)[i];
}
__device__ __forceinline__ int64_t row_pos(const SharedParams& p, int b) { return index_at(p.pos, p.pos64, p.pos_each ? b : 0); }
__device__ __forceinline__ int prefix_len(const SharedParams& p) {
  if (!p.plen) return p.prefix_rows;
  const int64_t n = index_at(p.plen, p.plen64, 0);
  return (int)(n < 0 ? 0 : (n > p.prefix_rows ? p.prefix_rows : n));
}

// Partial results of a group's query rows over the prefix, on the tensor memory.  splits: key ranges of an item; pair: 256 query rows a CTA, else 128
cudaError_t launch_attn_shared_prefix(const SharedParams& p, int head_size, bool pair, int splits, cudaStream_t st);

}  // namespace b200
