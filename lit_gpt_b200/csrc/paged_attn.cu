// A ragged step over a paged key-value cache: every sequence brings one token or a chunk of them, whose rotated keys and values join its pages, and
//   o_i = sum_j softmax_j(q_i . k_j / sqrt(hs)) v_j   over the keys j <= cached + i of its sequence that have a page.
// The rounding points are those of the model's step (lit_gpt/model.py:624-653, 767-773): q and k are bf16 after the rotation, the softmax is fp32 with a running maximum,
// the result is rounded once.  A row that sees no key has a result of zero.
//
// Few single tokens: one launch, a cluster of CTAs for a sequence and group (paged_cluster_kernel).  Else queries and new keys are turned and the new rows stored in their pages
// (paged_append_wide_kernel); sequences of few queries a group -- single tokens -- are the list's (paged_list_kernel), the others the tensor memory's (paged_attn_tc05.cu), at the same time where a
// step has both; their partial results are joined (paged_join_kernel).  No counter or flag is left between calls, and two calls at a time share nothing.
//
// The list: an item is a tile of queries of one sequence and group -- rows times heads of the group, row after row, so that the heads of a group share the keys that they read -- against
// the sequence's keys, in tiles of 32.  The tiles of all items are one list, cut evenly over the warps of all SMs (attn_list.cuh): requests of unequal lengths leave no SM without work.
//
// With the weights of keys wanted, the list keeps its scores beside the results, and a launch behind the join adds up what every key received: no key is read again.  What chunks' keys
// receive is computed from the joined sums (paged_weights.cu).
//
// Bound: single tokens by the bytes of their keys and values: 64 of 8 groups of 4 heads over 5 - 16000 keys, 2.1 GB, 325 us, 6.45 TB/s; 16 of 32 groups over 2047 with weights, 546 MB, 105 us, 83 of
// them the bytes: the rest the append's and the join's launches and the scores (with the keys read again for them 190).  Few of them by latency: 1 token of 32 groups over 300 keys 7.7 us (13.5 in
// three launches).  Beside chunks: 32 tokens over 100 - 3001 keys and 512 rows behind 1024 74 us, where either alone takes 40 and 30.
#include "attn_list.cuh"
#include "paged.cuh"

namespace b200 {

using namespace list;

namespace {

constexpr int kUnits = 3;                   // a warp's ring: units of 32 keys or 32 values

__device__ __forceinline__ int64_t paged_pos(const PagedParams& p, int row) {
  const int64_t at = p.table_presel ? row : p.pos64 ? reinterpret_cast<const int64_t*>(p.row_pos)[row] : (int64_t)reinterpret_cast<const int32_t*>(p.row_pos)[row];
  return at < 0 ? 0 : (at >= p.table_rows ? p.table_rows - 1 : at);
}

// ---- the queries and the new keys turned, the new rows stored ----
// A CTA takes a row, or some heads of one: HS / 16 threads a head, each with sixteen numbers of it, eight and the eight that they turn with (or, where nothing is turned, any sixteen), whose cosines
// and sines it keeps from head to head.  Needs rows of heads and tables for accesses of 16 bytes, and halves of the rotation that are multiples of eight numbers (or no rotation).
// Bound: bytes in flight behind the look-up of the row's place, three loads one after the other: 4096 rows of 32 groups of 1 head, 200 MB, 44 us, 4.6 TB/s (a head a warp 112; three
// CTAs an SM 48; three heads a thread on their way at a time, two CTAs an SM, 52).
template <int HS>
__global__ void __launch_bounds__(256, 4) paged_append_wide_kernel(const PagedParams p) {
  constexpr int TH = HS / 16, HEADS = 256 / TH;    // threads of a head; heads at once
  griddep_wait();     // (before the launch of what follows: the kernels behind read the step's description and the older keys ahead of their own wait)
  griddep_launch();
  const int row = blockIdx.x, heads = p.n_groups * (p.per + 2), n = p.rope_n, half = n >> 1;
  const int piece = threadIdx.x % TH;
  // numbers a .. a + 7 and b .. b + 7: pairs of the rotation first, then what it leaves
  const int turning = half >> 3, a = piece < turning ? piece * 8 : n + (piece - turning) * 16, b = piece < turning ? a + half : a + 8;
  const __nv_bfloat16* const x = p.qkv + (int64_t)row * heads * HS;
  int i = blockIdx.y * HEADS + threadIdx.x / TH;
  uint4 ra = {}, rb = {};
  auto load = [&](int h) {
    if (h < heads) {
      ra = *reinterpret_cast<const uint4*>(x + (int64_t)h * HS + a);
      rb = *reinterpret_cast<const uint4*>(x + (int64_t)h * HS + b);
    }
  };
  load(i);
  const int which = p.row_seq[row];
  float ca[8], sa[8], cb[8], sb[8];
  if (piece < turning) {
    const int64_t at = paged_pos(p, row) * n;
    auto get = [&](const void* t, int d, float (&f)[8]) {
      if (p.table_bf16) load8(reinterpret_cast<const __nv_bfloat16*>(t) + at + d, f);
      else load8(reinterpret_cast<const float*>(t) + at + d, f);
    };
    get(p.cos, a, ca);
    get(p.sin, a, sa);
    get(p.cos, b, cb);
    get(p.sin, b, sb);
  }
  PagedSeq s = {};
  if (which >= 0 && which < p.n_seqs) s = paged_seq(p, which);
  const int mine = row - s.first, key = s.cached + mine;
  const bool none = mine < 0 || mine >= s.rows;    // a row of no sequence
  const int id = none || key >= s.n ? -1 : page_at(p, s.table, key >> p.shift), in = key & ((1 << p.shift) - 1);   // (no room behind max_length)
  for (; i < heads; i += gridDim.y * HEADS) {
    const uint4 ua = ra, ub = rb;
    load(i + gridDim.y * HEADS);
    const int gi = i / (p.per + 2), h = i - gi * (p.per + 2);
    if (none) {
      if (h < p.per) {
        __nv_bfloat16* const to = p.out + ((int64_t)row * p.n_head + gi * p.per + h) * HS;
        *reinterpret_cast<uint4*>(to + a) = *reinterpret_cast<uint4*>(to + b) = make_uint4(0u, 0u, 0u, 0u);
        if (p.lse && piece == 0) p.lse[((int64_t)gi * p.rows + row) * p.per + h] = INFINITY;
      }
      continue;
    }
    if (h >= p.per && id < 0) continue;
    __nv_bfloat16* const to = h < p.per    ? p.q + (((int64_t)gi * p.rows + row) * p.per + h) * HS
                              : h == p.per ? p.k + (int64_t)id * p.k_page + (int64_t)gi * p.k_group + (int64_t)in * HS
                                           : p.v + (int64_t)id * p.v_page + (int64_t)gi * p.v_group + (int64_t)in * HS;
    uint4 wa = ua, wb = ub;
    if (piece < turning && h <= p.per) {
      const uint32_t xa[4] = {ua.x, ua.y, ua.z, ua.w}, xb[4] = {ub.x, ub.y, ub.z, ub.w};
      uint32_t ya[4], yb[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float al = bf16lo(xa[j]), ah = bf16hi(xa[j]), bl = bf16lo(xb[j]), bh = bf16hi(xb[j]);
        ya[j] = pack_bf16(turned(al, bl, true, ca[2 * j], sa[2 * j], p.table_bf16), turned(ah, bh, true, ca[2 * j + 1], sa[2 * j + 1], p.table_bf16));
        yb[j] = pack_bf16(turned(bl, al, false, cb[2 * j], sb[2 * j], p.table_bf16), turned(bh, ah, false, cb[2 * j + 1], sb[2 * j + 1], p.table_bf16));
      }
      wa = make_uint4(ya[0], ya[1], ya[2], ya[3]);
      wb = make_uint4(yb[0], yb[1], yb[2], yb[3]);
    }
    *reinterpret_cast<uint4*>(to + a) = wa;
    *reinterpret_cast<uint4*>(to + b) = wb;
    if (p.kw && h == p.per && piece == 0) p.kw[(((int64_t)id * p.n_groups + gi) << p.shift) + in] = 0.f;
  }
}

// Any rotation and alignment: a head a warp.
template <int HS>
__global__ void __launch_bounds__(256) paged_append_kernel(const PagedParams p) {
  constexpr int V = HS / 32;
  griddep_wait();
  griddep_launch();
  const int lane = threadIdx.x & 31, heads = p.n_groups * (p.per + 2);
  const int64_t at = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5);
  const int row = (int)(at / heads), i = (int)(at - (int64_t)row * heads), gi = i / (p.per + 2), h = i - gi * (p.per + 2);
  if (row >= p.rows) return;
  const int which = p.row_seq[row];
  PagedSeq s = {};
  if (which >= 0 && which < p.n_seqs) s = paged_seq(p, which);
  const int mine = row - s.first, key = s.cached + mine;
  if (mine < 0 || mine >= s.rows) {   // a row of no sequence
    if (h < p.per) {
      __nv_bfloat16* const to = p.out + ((int64_t)row * p.n_head + gi * p.per + h) * HS;
      for (int j = 0; j < V; ++j) to[lane * V + j] = __float2bfloat16_rn(0.f);
      if (p.lse && lane == 0) p.lse[((int64_t)gi * p.rows + row) * p.per + h] = INFINITY;
    }
    return;
  }
  const __nv_bfloat16* const x = p.qkv + at * HS;
  uint32_t v[HS / 64];
  if (h <= p.per) {
    turned_part<HS>(p, x, paged_pos(p, row), lane, v);
  } else {
    const uint16_t* const u = reinterpret_cast<const uint16_t*>(x + lane * V);
#pragma unroll
    for (int j = 0; j < V / 2; ++j) v[j] = (uint32_t)u[2 * j] | ((uint32_t)u[2 * j + 1] << 16);
  }
  __nv_bfloat16* to;
  if (h < p.per) {
    to = p.q + (((int64_t)gi * p.rows + row) * p.per + h) * HS;
  } else {
    if (key >= s.n) return;           // no room behind max_length
    const int id = page_at(p, s.table, key >> p.shift), in = key & ((1 << p.shift) - 1);
    if (id < 0) return;
    to = (h == p.per ? p.k + (int64_t)id * p.k_page + (int64_t)gi * p.k_group : p.v + (int64_t)id * p.v_page + (int64_t)gi * p.v_group) + (int64_t)in * HS;
    if (p.kw && h == p.per && lane == 0) p.kw[(((int64_t)id * p.n_groups + gi) << p.shift) + in] = 0.f;
  }
  if constexpr (V == 4) *reinterpret_cast<uint2*>(to + lane * V) = make_uint2(v[0], v[V / 2 - 1]);
  else *reinterpret_cast<uint32_t*>(to + lane * V) = v[0];
}

// Workers take runs of the list's tiles, sequence after sequence, there group after group and tile of queries after tile of queries.  The result of item i by worker w goes to slot
// i + w, which no other pair has, since either grows with the tiles.
struct Split {
  int all, workers;      // tiles; workers
  int each, more;        // every worker has `each` tiles, the first `more` of them one more
};
__device__ __forceinline__ int worker_of(int tile, const Split& s) {
  const int wide = s.more * (s.each + 1);
  return tile < wide ? tile / (s.each + 1) : s.more + (tile - wide) / s.each;
}
__device__ __forceinline__ int first_tile(int w, const Split& s) { return w * s.each + min(w, s.more); }

// Sequences are summed in runs of one per thread: sums[t] = tiles and items (of one group) of the sequences before run t, sums[THREADS] of all.
// `ctas`: the CTAs that take part.
template <int THREADS>
__device__ __forceinline__ Split make_split(const PagedParams& p, int2* sums, int2* s_warp, bool note, int& ctas) {
  __shared__ Shares s_shares[THREADS / 32];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, run = (p.n_seqs + THREADS - 1) / THREADS;
  // (a description whose sequences overlap can hold more tiles than fit the step's limits: then none is done)
  int2 here = make_int2(0, 0);
  Shares work = {0ull, 0ull};
  for (int i = tid * run; i < min(p.n_seqs, (tid + 1) * run); ++i) {
    const PagedSeq s = paged_seq(p, i);
    const int items = seq_items(p, s);
    if (p.mixed) add_work(p, s, work);
    here.x = capped(here.x + (int64_t)items * seq_tiles(s));
    here.y = capped((int64_t)here.y + items);
  }
  int2 inc = here;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int x = __shfl_up_sync(0xffffffffu, inc.x, o), y = __shfl_up_sync(0xffffffffu, inc.y, o);
    if (lane >= o) { inc.x = capped((int64_t)inc.x + x); inc.y = capped((int64_t)inc.y + y); }
  }
  if (lane == 31) s_warp[warp] = inc;
  if (p.mixed) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      work.list += __shfl_xor_sync(0xffffffffu, work.list, o);
      work.tensor += __shfl_xor_sync(0xffffffffu, work.tensor, o);
    }
    if (lane == 0) s_shares[warp] = work;
  }
  __syncthreads();
  if (p.mixed) {
    work = {0ull, 0ull};
    for (int w = 0; w < THREADS / 32; ++w) { work.list += s_shares[w].list; work.tensor += s_shares[w].tensor; }
    ctas = max(p.sms - tensor_share(p, work), 1);
  }
  int2 before = make_int2(inc.x - here.x, inc.y - here.y);
  for (int w = 0; w < warp; ++w) { before.x = capped((int64_t)before.x + s_warp[w].x); before.y = capped((int64_t)before.y + s_warp[w].y); }
  sums[tid] = before;
  if (tid == THREADS - 1) sums[THREADS] = make_int2(capped((int64_t)before.x + here.x), capped((int64_t)before.y + here.y));
  __syncthreads();
  Split s;
  const int64_t all = (int64_t)sums[THREADS].x * p.n_groups, items = (int64_t)sums[THREADS].y * p.n_groups;
  if (note) {                            // who joins the results, and who adds up the keys' weights, learns where a sequence's items and tiles begin
    const bool fits = all < kMaxTiles && items <= p.items;
    for (int i = tid * run; i < min(p.n_seqs, (tid + 1) * run); ++i) {
      const PagedSeq q = paged_seq(p, i);
      const int n = seq_items(p, q);
      __stcg(p.item_base + i, fits ? before.y * p.n_groups : -1);
      __stcg(p.tile_base + i, fits ? before.x * p.n_groups : -1);
      before.x += n * seq_tiles(q);
      before.y += n;
    }
  }
  s.all = all < kMaxTiles && items <= p.items ? (int)all : 0;
  // two tiles a worker at least, unless that leaves SMs without one
  s.workers = min(max(s.all / 2, min(s.all, ctas)), p.mixed ? p.workers / (int)gridDim.x * ctas : p.workers);
  s.each = s.workers ? s.all / s.workers : 0;
  s.more = s.all - s.each * s.workers;
  return s;
}

// A tile of a worker's range, and the item that it belongs to.
struct Tile {
  int index;                         // in the order of all tiles
  int s, gi, part;                   // sequence, group, tile of queries
  PagedSeq seq;
  int tile, tiles;                   // of the item
  int item;
  int id0, id1;                      // pages of its first and last sixteen keys
  uint32_t bits;                     // its keys that are there
  __device__ __forceinline__ int left() const { return tiles - 1 - tile; }
  __device__ __forceinline__ int key0() const { return tile * kShTile; }
};

struct Walk {
  const PagedParams& p;
  const int2* sums;
  int run, threads;

  __device__ __forceinline__ void pages(Tile& t) const {
    const int i = t.key0() >> p.shift;
    t.id0 = page_at(p, t.seq.table, i);
    t.id1 = p.shift == 4 && t.key0() + 16 < t.seq.n ? page_at(p, t.seq.table, i + 1) : t.id0;
    const int rest = t.seq.n - t.key0();
    t.bits = (rest >= 32 ? 0xffffffffu : (1u << rest) - 1u) & ((t.id0 >= 0 ? 0xffffu : 0u) | (t.id1 >= 0 ? 0xffff0000u : 0u));
  }
  __device__ __forceinline__ void locate(Tile& t) const {   // by a warp
    pages(t);
    if (t.seq.rows > 1 && t.key0() + kShTile > t.seq.cached) {   // (of a single token's key nobody asks whose it is: a result that is not the sequence's goes nowhere)
      const int key = t.key0() + (threadIdx.x & 31);
      t.bits &= __ballot_sync(0xffffffffu, key < t.seq.n && whose_key(p, t.s, t.seq.cached, t.seq.first, key) == t.s);
    }
  }
  __device__ __forceinline__ Tile find(int index) const {
    Tile t;
    t.index = index;
    int lo = 0, hi = threads;        // the run whose sequences hold it
    while (hi - lo > 1) {
      const int mid = (lo + hi) / 2;
      if (sums[mid].x * p.n_groups <= index) lo = mid; else hi = mid;
    }
    int rest = index - sums[lo].x * p.n_groups;
    t.item = sums[lo].y * p.n_groups;
    t.s = lo * run;
    for (;;) {                       // (one sequence a run unless there are many)
      t.seq = paged_seq(p, t.s);
      t.tiles = seq_tiles(t.seq);
      const int items = seq_items(p, t.seq), here = items * t.tiles * p.n_groups;
      if (rest < here) {
        const int item = rest / t.tiles;
        t.tile = rest - item * t.tiles;
        t.item += item;
        t.gi = item / items;
        t.part = item - t.gi * items;
        break;
      }
      rest -= here;
      t.item += items * p.n_groups;
      ++t.s;
    }
    locate(t);
    return t;
  }
  // the tile behind it (there is one)
  __device__ __forceinline__ void next(Tile& t) const {
    ++t.index;
    if (++t.tile == t.tiles) {
      t.tile = 0;
      ++t.item;
      if (++t.part == seq_items(p, t.seq)) {
        t.part = 0;
        if (++t.gi == p.n_groups) {
          t.gi = 0;
          do t.seq = paged_seq(p, ++t.s); while (seq_items(p, t.seq) == 0);
          t.tiles = seq_tiles(t.seq);
        }
      }
    }
    locate(t);
  }
  __device__ __forceinline__ int queries(const Tile& t) const { return min(p.tile_rows, t.seq.rows * p.per - t.part * p.tile_rows); }
  __device__ __forceinline__ int64_t query_row(const Tile& t) const { return ((int64_t)t.gi * p.rows + t.seq.first) * p.per + t.part * p.tile_rows; }
};

// 32 rows of a tile, zeros where there is no key: a weight of zero times whatever lies there must be zero
template <int HS>
__device__ __forceinline__ void load_tile(const PagedParams& p, const Tile& t, const __nv_bfloat16* base, int64_t page, int64_t group, uint32_t dst, int lane) {
  constexpr int CH = HS / 8, RP = 32 / CH;   // 16-byte pieces of a row, rows a warp copies at once
  const uint32_t bits = t.bits;
  const int c = lane % CH, in = t.key0() & ((1 << p.shift) - 1);
  const __nv_bfloat16* const g = base + (int64_t)t.gi * group + c * 8;
  const __nv_bfloat16* const a = g + (int64_t)max(t.id0, 0) * page + (int64_t)in * HS;
  const __nv_bfloat16* const b = p.shift == 4 ? g + (int64_t)max(t.id1, 0) * page - (int64_t)16 * HS : a;
#pragma unroll
  for (int j = 0; j < kShTile / RP; ++j) {
    const int r = j * RP + lane / CH;
    const bool ok = (bits >> r) & 1u;
    const __nv_bfloat16* const src = j * RP < 16 ? a : b;
    pf_cp16(dst + sw<HS>(r, c), ok ? src + r * HS : g, ok);
  }
}

// A warp's shared memory: a ring of units, the queries of two items.  One CTA an SM.  Queries come in eights, NQ of them.
template <int HS, int NQ>
struct PgSmem {
  static constexpr int kUnit = kShTile * HS * 2, kQ = 8 * NQ * HS * 2;
  static constexpr int kWarp = kUnits * kUnit + 2 * kQ;
  static constexpr int kWarps = HS == 64 ? (NQ == 4 ? 10 : 12) : (NQ == 4 ? 5 : 7);
  static constexpr int kBytes = kWarps * kWarp;
};

template <int HS, int NQ, bool KEEP>
__global__ void __launch_bounds__(PgSmem<HS, NQ>::kWarps * 32, 1) paged_list_kernel(const PagedParams p) {
  using C = PgSmem<HS, NQ>;
  constexpr int T = C::kWarps * 32, CH = HS / 8, RP = 32 / CH;
  extern __shared__ __align__(128) uint8_t pg_smem[];
  __shared__ int2 s_sums[T + 1], s_warp[C::kWarps];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, tq = lane & 3;
  griddep_launch();
  int ctas = gridDim.x;
  const Split s = make_split<T>(p, s_sums, s_warp, blockIdx.x == 0, ctas);
  const int w = warp * ctas + (int)blockIdx.x;             // (workers beside each other on different SMs)
  // Beside the tensor memory's kernel, which lets this one begin once the append kernel has ended, the wait is for that kernel: at the end, so that what comes next finds both done.
  const bool late = p.mixed;
  if (w >= s.workers || (int)blockIdx.x >= ctas) {
    griddep_wait();
    return;
  }
  const Walk walk{p, s_sums, (p.n_seqs + T - 1) / T, T};
  const uint32_t ring = pf_smem(pg_smem) + warp * C::kWarp, sq = ring + kUnits * C::kUnit;

  auto load_k = [&](uint32_t dst, const Tile& t) { load_tile<HS>(p, t, p.k, p.k_page, p.k_group, dst, lane); };
  auto load_v = [&](uint32_t dst, const Tile& t) { load_tile<HS>(p, t, p.v, p.v_page, p.v_group, dst, lane); };
  auto load_queries = [&](uint32_t dst, const Tile& t) {
    const __nv_bfloat16* const src = p.q + walk.query_row(t) * HS;
    const int valid = walk.queries(t);
#pragma unroll
    for (int j = 0; j < 8 * NQ / RP; ++j) {
      const int r = j * RP + lane / CH, c = lane % CH;
      const bool ok = r < valid;
      pf_cp16(dst + sw<HS>(r, c), src + (ok ? r * HS : 0) + c * 8, ok);
    }
  };
  const int first = first_tile(w, s), end = first_tile(w + 1, s);
  Tile cur = walk.find(first);
  Tile coming = cur;                                       // the tile behind it: its values are loaded next
  const bool two = cur.index + 1 < end;
  if (two) walk.next(coming);
  // What the append kernel writes, queries and new keys, is read behind the wait; everything else was there before.
  auto early = [&](bool now) {
    const bool c = now == (cur.key0() + kShTile <= cur.seq.cached), n = two && now == (coming.key0() + kShTile <= coming.seq.cached);
    if (c) {
      load_k(ring, cur);
      load_v(ring + C::kUnit, cur);
    }
    if (n) load_k(ring + 2 * C::kUnit, coming);
  };
  early(true);
  if (!late) griddep_wait();
  early(false);
  load_queries(sq, cur);
  int qb = 0, next_qb = 0;                                 // the query buffers of either
  if (two && cur.left() == 0) load_queries(sq + (next_qb = 1) * C::kQ, coming);
  pf_commit();
  pf_commit();
  pf_commit();

  Sums<HS, NQ> a;
  auto clear = [&]() {
#pragma unroll
    for (int t = 0; t < NQ; ++t) {
#pragma unroll
      for (int i = 0; i < HS / 16; ++i) a.o[i][t][0] = a.o[i][t][1] = a.o[i][t][2] = a.o[i][t][3] = 0.f;
      a.m[t][0] = a.m[t][1] = -INFINITY;
      a.l[t][0] = a.l[t][1] = 0.f;
    }
  };
  clear();
  int unit = 0;                                            // of the current tile's keys
  for (;;) {
    const uint32_t kb = ring + unit * C::kUnit;
    unit = unit == kUnits - 1 ? 0 : unit + 1;
    const uint32_t vb = ring + unit * C::kUnit;
    unit = unit == kUnits - 1 ? 0 : unit + 1;
    const bool more = cur.index + 1 < end;
    pf_wait<2>();
    __syncwarp();
    auto values = [&]() {
      __syncwarp();                                        // the keys have been read: the values of the next tile take their place
      if (more) load_v(kb, coming);
      pf_commit();
      pf_wait<2>();
      __syncwarp();
      return vb;
    };
    const uint32_t bits = cur.bits;
    const int key0 = cur.key0(), count = walk.queries(cur);
    float* const kept = KEEP ? p.scores + (int64_t)cur.index * p.score_rows * kShTile : nullptr;
    auto keep = [&](int key, int t, int c, float s) {
      if constexpr (KEEP) {
        const int m = t * 8 + 2 * tq + c;
        if (m < count) __stcg(kept + m * kShTile + key, s);
      }
    };
    if (key0 + kShTile > cur.seq.cached + 1 && cur.seq.rows > 1) {   // a chunk's own keys: every row sees those up to its own
      int lim[NQ][2];
#pragma unroll
      for (int t = 0; t < NQ; ++t)
#pragma unroll
        for (int c = 0; c < 2; ++c) lim[t][c] = cur.seq.cached + (cur.part * p.tile_rows + t * 8 + 2 * tq + c) / p.per - key0;
      attend_tile<HS, NQ, NQ>(a, sq + qb * C::kQ, 0, kb, p.scale_log2, lane, [&](int key, int t, int c) { return ((bits >> key) & 1u) && key <= lim[t][c]; }, keep, values);
    } else {
      auto seen = [bits](int key, int, int) { return ((bits >> key) & 1u) != 0u; };
      if (NQ == 1 || count > 8) attend_tile<HS, NQ, NQ>(a, sq + qb * C::kQ, 0, kb, p.scale_log2, lane, seen, keep, values);
      else attend_tile<HS, NQ, 1>(a, sq + qb * C::kQ, 0, kb, p.scale_log2, lane, seen, keep, values);
    }
    __syncwarp();                                          // the values have been read: the keys of the tile after the next take their place
    const bool ends = cur.left() == 0 || !more;
    const Tile was = cur;
    cur = coming;
    qb = next_qb;
    if (cur.index + 1 < end) {
      walk.next(coming);
      load_k(vb, coming);
      if (cur.left() == 0) load_queries(sq + (next_qb = qb ^ 1) * C::kQ, coming);
    }
    pf_commit();
    if (ends) {
      // ---- the item, or this worker's part of it, ends ----
      const int64_t slot = (int64_t)was.item + w;
      if (lane == 0 && was.index - was.tile >= first)      // it began here: who joins its results learns where they are
        __stcg(p.where + was.item, make_int2(w, worker_of(was.index + was.left(), s) - w + 1));
      store_sums<HS, NQ>(a, p.acc + slot * p.tile_rows * HS, p.ml + slot * p.tile_rows, walk.queries(was), lane);
      if (!more) break;
      clear();
    }
  }
  pf_wait<0>();
  if (late) griddep_wait();
}

// An item of the tensor memory's that several CTAs had segments of (paged_attn_tc05.cu): CTA (w, part) joins a share of its queries, 32 at a time, for the w-th worker's beginning within it.  A query a lane, HS / 8
// numbers a warp.
template <int HS>
__device__ __forceinline__ void join_cut(const PagedParams& p, int index, int parts) {
  constexpr int V = HS / 8;
  const int w = index / parts, part = index - w * parts, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const PagedCut c = p.cuts[w];
  if (c.last == kCutNothing && w == 0) {           // rows that were the tensor memory's see no key
    for (int row = part; row < p.rows; row += parts) {
      const int which = p.row_seq[row];
      if (which < 0 || which >= p.n_seqs || paged_seq(p, which).rows * p.per <= p.list_max) continue;
      for (int i = threadIdx.x; i < p.n_head * HS / 8; i += blockDim.x) reinterpret_cast<uint4*>(p.out + (int64_t)row * p.n_head * HS)[i] = make_uint4(0u, 0u, 0u, 0u);
      for (int i = threadIdx.x; p.lse && i < p.n_head; i += blockDim.x) p.lse[((int64_t)(i / p.per) * p.rows + row) * p.per + i % p.per] = INFINITY;
    }
  }
  if (c.last < 0) return;
  const int shares = (c.last - c.first) * parts, share = (w - c.first - 1) * parts + part;
  for (int m0 = share * 32; m0 < c.count; m0 += shares * 32) {
    const int m = m0 + lane;
    float top = -INFINITY, sum = 0.f, a[V] = {};
    for (int i0 = c.first; i0 <= c.last; i0 += 2) {
      float2 e[2];
      float4 v[2][V / 4];
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        e[u] = make_float2(-INFINITY, 0.f);
#pragma unroll
        for (int j = 0; j < V / 4; ++j) v[u][j] = make_float4(0.f, 0.f, 0.f, 0.f);
        if (i0 + u <= c.last && m < c.count) {
          const int64_t slot = 2 * (i0 + u) + (i0 + u == c.first);
          e[u] = __ldcg(p.tc_ml + slot * 256 + m);
#pragma unroll
          for (int j = 0; j < V / 4; ++j) v[u][j] = __ldcg(reinterpret_cast<const float4*>(p.tc_acc + slot * 256 * HS + (int64_t)(warp * V + 4 * j) * 256 + m * 4));
        }
      }
      const float now = fmaxf(top, fmaxf(e[0].x, e[1].x)), org = now == -INFINITY ? 0.f : now, shrink = ex2(top - org);
      top = now;
      sum *= shrink;
#pragma unroll
      for (int j = 0; j < V; ++j) a[j] *= shrink;
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const float f = ex2(e[u].x - org);
        sum += e[u].y * f;
        if (e[u].y != 0.f) {            // (a range that saw nothing has no result)
#pragma unroll
          for (int j = 0; j < V / 4; ++j) {
            a[4 * j] += v[u][j].x * f;
            a[4 * j + 1] += v[u][j].y * f;
            a[4 * j + 2] += v[u][j].z * f;
            a[4 * j + 3] += v[u][j].w * f;
          }
        }
      }
    }
    if (m >= c.count) continue;
    const int row = m / p.per, hh = m - row * p.per;
    const float inv = sum == 0.f ? 0.f : 1.f / sum;   // (a sum that is NaN stays one)
    __nv_bfloat16* const to = p.out + ((int64_t)(c.row + row) * p.n_head + c.gi * p.per + hh) * HS + warp * V;
#pragma unroll
    for (int j = 0; j < V; j += 8)
      *reinterpret_cast<uint4*>(to + j) = make_uint4(pack_bf16(a[j] * inv, a[j + 1] * inv), pack_bf16(a[j + 2] * inv, a[j + 3] * inv), pack_bf16(a[j + 4] * inv, a[j + 5] * inv),
                                                     pack_bf16(a[j + 6] * inv, a[j + 7] * inv));
    if (p.lse && warp == 0) p.lse[((int64_t)c.gi * p.rows + c.row) * p.per + m] = sum == 0.f ? INFINITY : top + log2f(sum);
  }
}

// The first CTAs join the tensor memory's cut items, kCutParts a worker; the others the list's results, `ways` warps a head, HS / 32 numbers a lane.
constexpr int kCutParts = 8;
template <int HS>
__global__ void __launch_bounds__(256) paged_join_kernel(const PagedParams p) {
  if ((int)blockIdx.x < p.tc_workers * kCutParts) {
    griddep_launch();
    griddep_wait();
    join_cut<HS>(p, blockIdx.x, kCutParts);
    return;
  }
  const int block = blockIdx.x - p.tc_workers * kCutParts;
  constexpr int V = HS / 32;
  __shared__ float s_acc[8][HS];
  __shared__ float2 s_ml[8];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, heads = 8 / p.ways, blocks = (p.n_head + heads - 1) / heads;
  const int row = block / blocks, h = (block - row * blocks) * heads + warp / p.ways, way = warp % p.ways;
  griddep_launch();
  const int which = p.row_seq[row];
  PagedSeq s = {};
  if (which >= 0 && which < p.n_seqs) s = paged_seq(p, which);
  const bool idle = row < s.first || row - s.first >= s.rows || s.rows * p.per > p.list_max;   // (or the tensor memory's)
  griddep_wait();
  float top = -INFINITY, sum = 0.f, a[V] = {};
  const int gi = h / p.per, m = (row - s.first) * p.per + h - gi * p.per;
  int item = -1;
  if (h < p.n_head && !idle && s.n > 0) item = __ldcg(p.item_base + which);
  if (item >= 0) {                 // (less where nothing was done: there is no result to read)
    item += gi * seq_items(p, s) + m / p.tile_rows;
    const int at = m % p.tile_rows;
    const int2 at_w = __ldcg(p.where + item);
    join_results<V>(way, p.ways, at_w.y, lane, top, sum, a, [&](int i, const float2*& ml, const float*& acc) {
      const int64_t slot = ((int64_t)item + at_w.x + i) * p.tile_rows + at;
      ml = p.ml + slot;
      acc = p.acc + slot * HS;
    });
  }
  if (p.ways > 1) {
    if (way > 0) {
#pragma unroll
      for (int j = 0; j < V; ++j) s_acc[warp][lane * V + j] = a[j];
      if (lane == 0) s_ml[warp] = make_float2(top, sum);
    }
    __syncthreads();
    if (way == 0) join_warps<HS>(s_acc[warp], s_ml + warp, p.ways, lane, top, sum, a);
  }
  if (way > 0 || h >= p.n_head || idle) return;
  store_result<HS>(p.out + ((int64_t)row * p.n_head + h) * HS, a, sum == 0.f ? 0.f : 1.f / sum, lane);
  if (p.lse && lane == 0) p.lse[((int64_t)gi * p.rows + row) * p.per + h - gi * p.per] = sum == 0.f ? INFINITY : top + log2f(sum);
}

// ---- few single tokens: a sequence and group's whole step by a cluster of CTAs, in one launch ----
// Every CTA turns the group's heads itself; the cluster's warps share the tiles, the new key and value come into their tile from shared memory; behind the cluster's barrier its CTAs
// join the results, a head at a time each.
template <int HS, int NQ>
struct ClSmem {
  static constexpr int kWarps = 4, kUnit = kShTile * HS * 2, kWarp = 2 * kUnit, kQ = 8 * NQ * HS * 2;   // keys and values of a tile; a warp's results in their place
  static constexpr int kBytes = kWarps * kWarp + kQ + 2 * HS * 2;
  static_assert(8 * NQ * HS * 4 <= kWarp, "a warp's results");
};

template <int HS, int NQ>
__global__ void __launch_bounds__(ClSmem<HS, NQ>::kWarps * 32) paged_cluster_kernel(const PagedParams p, int ctas) {
  using C = ClSmem<HS, NQ>;
  constexpr int W = C::kWarps, V = HS / 32;
  extern __shared__ __align__(128) uint8_t cl_smem[];
  __shared__ float2 s_ml[W][8 * NQ], s_cta[8 * NQ];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, rank = blockIdx.x % ctas, item = blockIdx.x / ctas, gi = item % p.n_groups;
  uint8_t* const s_q = cl_smem + W * C::kWarp;
  uint8_t* const s_new = s_q + C::kQ;              // the new key, the new value
  griddep_launch();
  griddep_wait();
  Tile t;
  t.seq = paged_seq(p, item / p.n_groups);
  // rows of no sequence
  for (int row = blockIdx.x; row < p.rows; row += gridDim.x) {
    const int which = p.row_seq[row];
    PagedSeq s = {};
    if (which >= 0 && which < p.n_seqs) s = paged_seq(p, which);
    if (row >= s.first && row - s.first < s.rows) continue;
    for (int i = threadIdx.x; i < p.n_head * HS / 8; i += W * 32) reinterpret_cast<uint4*>(p.out + (int64_t)row * p.n_head * HS)[i] = make_uint4(0u, 0u, 0u, 0u);
  }
  if (t.seq.rows == 0) return;                     // (the whole cluster)
  const int row = t.seq.first, key = t.seq.cached, step = ctas * W;
  const Walk walk{p, nullptr, 0, 0};
  t.gi = gi;
  t.tiles = seq_tiles(t.seq);
  t.tile = rank * W + warp;
  const uint32_t kb = pf_smem(cl_smem) + warp * C::kWarp, vb = kb + C::kUnit;
  // the new key is not read from its page: it comes from shared memory
  const int whose = p.row_seq[row];                // (where the row is another's, or none's, nothing of it is stored)
  const int fresh = key < t.seq.n && page_at(p, t.seq.table, key >> p.shift) >= 0 ? key : -1;
  auto load = [&](const Tile& x, const __nv_bfloat16* base, int64_t page, int64_t group, uint32_t dst) {
    Tile y = x;
    const int at = key - x.key0();
    if (at >= 0 && at < kShTile) y.bits &= ~(1u << at);
    load_tile<HS>(p, y, base, page, group, dst, lane);
    pf_commit();
  };
  if (t.tile < t.tiles) {
    walk.pages(t);
    load(t, p.k, p.k_page, p.k_group, kb);
    load(t, p.v, p.v_page, p.v_group, vb);
  }
  const int64_t trow = paged_pos(p, row);
  for (int h = warp; h < 8 * NQ + 2; h += W) {     // the queries (zeros behind them), the new key, the new value
    uint32_t v[HS / 64];
#pragma unroll
    for (int j = 0; j < V / 2; ++j) v[j] = 0u;
    const int head = h < 8 * NQ ? h : p.per + h - 8 * NQ;
    const __nv_bfloat16* const x = p.qkv + (((int64_t)row * p.n_groups + gi) * (p.per + 2) + head) * HS;
    if (h < p.per || h == 8 * NQ) {
      turned_part<HS>(p, x, trow, lane, v);
    } else if (h == 8 * NQ + 1) {
      const uint16_t* const u = reinterpret_cast<const uint16_t*>(x + lane * V);
#pragma unroll
      for (int j = 0; j < V / 2; ++j) v[j] = (uint32_t)u[2 * j] | ((uint32_t)u[2 * j + 1] << 16);
    }
    auto store = [&](void* at) {
      if constexpr (V == 4) *reinterpret_cast<uint2*>(at) = make_uint2(v[0], v[V / 2 - 1]);
      else *reinterpret_cast<uint32_t*>(at) = v[0];
    };
    store(h < 8 * NQ ? s_q + sw<HS>(h, lane * V / 8) + lane * V % 8 * 2 : s_new + (h - 8 * NQ) * HS * 2 + lane * V * 2);
    if (h >= 8 * NQ && rank == 0 && fresh >= 0 && whose == item / p.n_groups) {
      const int64_t id = page_at(p, t.seq.table, key >> p.shift), in = key & ((1 << p.shift) - 1);
      store((h == 8 * NQ ? p.k + id * p.k_page + (int64_t)gi * p.k_group : p.v + id * p.v_page + (int64_t)gi * p.v_group) + in * HS + lane * V);
    }
  }
  __syncthreads();
  Sums<HS, NQ> a;
#pragma unroll
  for (int u = 0; u < NQ; ++u) {
#pragma unroll
    for (int i = 0; i < HS / 16; ++i) a.o[i][u][0] = a.o[i][u][1] = a.o[i][u][2] = a.o[i][u][3] = 0.f;
    a.m[u][0] = a.m[u][1] = -INFINITY;
    a.l[u][0] = a.l[u][1] = 0.f;
  }
  while (t.tile < t.tiles) {
    Tile next = t;
    next.tile += step;
    const bool more = next.tile < t.tiles;
    if (more) walk.pages(next);
    const int at = fresh - t.key0();               // the new key's place in this tile
    auto patch = [&](uint32_t dst, int which) {
      if (at >= 0 && at < kShTile) {
        if (lane < HS / 8) {
          const uint4 x = *reinterpret_cast<const uint4*>(s_new + which * HS * 2 + lane * 16);
          asm volatile("st.shared.v4.u32 [%0], {%1,%2,%3,%4};" ::"r"(dst + sw<HS>(at, lane)), "r"(x.x), "r"(x.y), "r"(x.z), "r"(x.w) : "memory");
        }
        __syncwarp();
      }
    };
    pf_wait<1>();
    __syncwarp();
    patch(kb, 0);
    const uint32_t bits = t.bits;
    attend_tile<HS, NQ, NQ>(a, pf_smem(s_q), 0, kb, p.scale_log2, lane, [bits](int k, int, int) { return ((bits >> k) & 1u) != 0u; }, [](int, int, int, float) {}, [&]() {
      __syncwarp();
      if (more) load(next, p.k, p.k_page, p.k_group, kb); else pf_commit();
      pf_wait<1>();
      __syncwarp();
      patch(vb, 1);
      return vb;
    });
    __syncwarp();
    if (more) load(next, p.v, p.v_page, p.v_group, vb); else pf_commit();
    t = next;
  }
  pf_wait<0>();
  __syncwarp();
  // ---- the CTA's results, then the cluster's ----
  float* const mine = reinterpret_cast<float*>(cl_smem + warp * C::kWarp);
  const int g = lane >> 2, tq = lane & 3;
#pragma unroll
  for (int u = 0; u < NQ; ++u)
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      float l = a.l[u][c];
#pragma unroll
      for (int o = 4; o < 32; o <<= 1) l += __shfl_xor_sync(0xffffffffu, l, o);
      const int h = u * 8 + 2 * tq + c;
#pragma unroll
      for (int i = 0; i < HS / 16; ++i) {
        mine[h * HS + i * 16 + g] = a.o[i][u][c];
        mine[h * HS + i * 16 + 8 + g] = a.o[i][u][2 + c];
      }
      if (g == 0) s_ml[warp][h] = make_float2(a.m[u][c], l);
    }
  __syncthreads();
  float* const first = reinterpret_cast<float*>(cl_smem);
  for (int i = threadIdx.x; i < p.per * HS; i += W * 32) {
    const int h = i / HS;
    float top = -INFINITY, sum = 0.f, x = 0.f;
#pragma unroll
    for (int w = 0; w < W; ++w) top = fmaxf(top, s_ml[w][h].x);
    const float org = top == -INFINITY ? 0.f : top;
#pragma unroll
    for (int w = 0; w < W; ++w) {
      const float f = ex2(s_ml[w][h].x - org);
      sum += s_ml[w][h].y * f;
      x += s_ml[w][h].y == 0.f ? 0.f : reinterpret_cast<const float*>(cl_smem + w * C::kWarp)[i] * f;   // (a warp that saw nothing has no result)
    }
    first[i] = x;                                  // (read by this thread alone)
    if (i % HS == 0) s_cta[h] = make_float2(top, sum);
  }
  if (ctas > 1) asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
  else __syncthreads();
  auto remote = [](const void* at, int of) {
    uint32_t ra;
    float x;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(ra) : "r"(pf_smem(at)), "r"(of));
    asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(x) : "r"(ra) : "memory");
    return x;
  };
  for (int i = rank * W * 32 + threadIdx.x; i < p.per * HS; i += ctas * W * 32) {
    const int h = i / HS;
    float m[8], l[8], x[8], top = -INFINITY, sum = 0.f, y = 0.f;
#pragma unroll
    for (int u = 0; u < 8; ++u) {
      const bool in = u < ctas;
      m[u] = in ? remote(&s_cta[h].x, u) : -INFINITY;
      l[u] = in ? remote(&s_cta[h].y, u) : 0.f;
      x[u] = in ? remote(first + i, u) : 0.f;
      top = fmaxf(top, m[u]);
    }
    const float org = top == -INFINITY ? 0.f : top;
#pragma unroll
    for (int u = 0; u < 8; ++u) {
      const float f = ex2(m[u] - org);
      sum += l[u] * f;
      y += l[u] == 0.f ? 0.f : x[u] * f;
    }
    if (whose == item / p.n_groups) p.out[((int64_t)row * p.n_head + gi * p.per + h) * HS + i % HS] = __float2bfloat16_rn(sum == 0.f ? 0.f : y / sum);
  }
  // no CTA leaves, and frees its shared memory, before the others have read it
  if (ctas > 1) asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}

// ---- the weight that keys receive: blocks of keys that several CTAs of paged_weights.cu had parts of, in the CTAs' order; and the list's sequences', a key a thread, from the scores
// that were kept ----
__global__ void __launch_bounds__(256) paged_kept_kernel(const PagedParams p) {
  griddep_launch();
  if ((int)blockIdx.x < p.kw_workers) {
    griddep_wait();
    const PagedWeightCut c = p.kw_cuts[blockIdx.x];
    if (c.last < 0 || blockIdx.y > 0 || threadIdx.x >= 128) return;
    const int key = c.block * 128 + (int)threadIdx.x;
    float sum = 0.f;
    for (int w = c.first; w <= c.last; ++w) sum += __ldcg(p.kw_part + (2 * w + (w == c.first)) * 128 + threadIdx.x);
    const int id = key_page(p, c.s, c.table, c.cached, c.row, c.n, key);
    if (id >= 0) p.kw[(((int64_t)id * p.n_groups + c.gi) << p.shift) + (key & ((1 << p.shift) - 1))] += sum;
    return;
  }
  const int pair = blockIdx.x - p.kw_workers, which = pair / p.n_groups, gi = pair - which * p.n_groups;
  const PagedSeq s = paged_seq(p, which);
  const int items = seq_items(p, s);
  auto place = [&](int key) -> float* {
    const int id = key_page(p, which, s.table, s.cached, s.first, s.n, key);
    return id < 0 ? nullptr : p.kw + (((int64_t)id * p.n_groups + gi) << p.shift) + (key & ((1 << p.shift) - 1));
  };
  int key = blockIdx.y * 256 + threadIdx.x;
  float* at = items > 0 ? place(key) : nullptr;
  griddep_wait();
  if (items == 0) return;
  const int tiles = seq_tiles(s), count = s.rows * p.per;
  const int first = __ldcg(p.tile_base + which);
  if (first < 0) return;                           // (more than fits a step's limits: nothing was done)
  const float* const lse = p.lse + ((int64_t)gi * p.rows + s.first) * p.per;
  for (; key < s.n; key += gridDim.y * 256, at = place(key)) {
    if (!at) continue;
    const float before = *at;
    auto gains = [&](bool rare) {
      float sum = 0.f;
      for (int m0 = 0, index = first + gi * items * tiles + key / kShTile; m0 < count; m0 += p.tile_rows, index += tiles) {
        const float* const kept = p.scores + (int64_t)index * p.score_rows * kShTile + key % kShTile;
        const int n = min(p.tile_rows, count - m0);
        if (!rare) {
#pragma unroll 8
          for (int m = 0; m < n; ++m) sum += ex2(__ldcg(kept + m * kShTile) - __ldcg(lse + m0 + m));
        } else {
#pragma unroll 1
          for (int m = 0; m < n; ++m) {
            const float l = __ldcg(lse + m0 + m), x = ex2(__ldcg(kept + m * kShTile) - l);
            sum += l == INFINITY || m0 + m < max(key - s.cached, 0) * p.per ? 0.f : x;
          }
        }
      }
      return sum;
    };
    float sum = gains(false);
    if (sum != sum) sum = gains(true);             // of what is not a number only that counts which a row of the sequence that sees the key gives it
    *at = before + sum;
  }
}

// ---- host ----
struct PagedPlan {
  int nq, ctas, workers, ways;
  bool list, tensor;               // which kernels there is work for
  int cluster;                     // CTAs that a sequence and group's step takes in one launch; 0: the launches above
  int list_max, tc_workers;
  int64_t items, slots, q;
  int score_rows, kept_max, kw_workers;
  int64_t scores;
  int64_t steps;                   // bound of what any kernel counts in its list
  size_t bytes;
};
constexpr int64_t kScoresMax = (int64_t)1 << 28;   // scores that a step may keep: 1 GB

std::atomic<int> g_paged_path{0};
constexpr int kListMax = 32;       // queries of a sequence and group that the list of tiles takes

PagedPlan paged_plan(int64_t rows, int n_seqs, int n_groups, int per, int hs, int64_t max_rows, int64_t max_length, bool kw) {
  PagedPlan s;
  const int path = g_paged_path.load(std::memory_order_relaxed);
  // chunks of one length only: all go to the tensor memory (some of them may turn out shorter, or not there)
  // 17 to 32 queries: 8 groups of 4 heads, us of the list and of the tensor memory: 8 rows behind 500 keys 13.5, 16.2, behind 16000 40, 29; 16 times 8 rows behind 300 23, 22, behind 3000 86, 55
  const bool short_ = (int64_t)n_seqs * n_groups * max_length <= 60000;
  const int singles = per <= 8 ? 8 : per <= 16 ? 16 : kListMax;   // beside chunks the list takes single tokens, in items as small as they are
  s.list_max = path == 1 || path == 3 || per > 128 ? 0x3fffffff : path == 2 ? 0 : max_rows * per <= (short_ ? kListMax : 16) ? kListMax : rows == (int64_t)n_seqs * max_rows ? 0 : singles;
  s.tensor = max_rows * per > s.list_max;
  s.list = s.list_max > 0;
  const int64_t most = max_rows * per < s.list_max ? max_rows * per : s.list_max;   // queries of an item
  s.nq = most <= 8 ? 1 : most <= 16 ? 2 : 4;
  // (beside chunks, whose rows are none of the list's, an item holds the queries of any sequence and group that is)
  s.items = (int64_t)n_groups * (s.tensor && most <= 8 * s.nq ? n_seqs : (rows * per + 8 * s.nq - 1) / (8 * s.nq) + n_seqs);
  const int warps = hs == 64 ? (s.nq == 4 ? PgSmem<64, 4>::kWarps : PgSmem<64, 1>::kWarps) : (s.nq == 4 ? PgSmem<128, 4>::kWarps : PgSmem<128, 1>::kWarps);
  const int64_t tiles = s.items * ((max_length + kShTile - 1) / kShTile);
  s.ctas = sm_count();
  if (s.ctas > tiles && !(s.tensor && s.list)) s.ctas = (int)tiles;
  s.workers = s.ctas * warps < tiles || (s.tensor && s.list) ? s.ctas * warps : (int)tiles;
  s.slots = s.list ? (s.items + s.workers) * 8 * s.nq : 0;
  const int64_t blocks = s.tensor ? (int64_t)n_groups * (rows / (256 / per) + n_seqs) * ((max_length + 127) / 128) : 0;
  s.tc_workers = blocks < sm_count() && !(s.tensor && s.list) ? (int)blocks : sm_count();
  if (!s.tensor) s.tc_workers = 0;
  const int64_t tc_slots = (int64_t)s.tc_workers * 2 * 256;
  s.q = rows * per * n_groups * hs;
  s.score_rows = s.kept_max = s.kw_workers = 0;
  s.scores = 0;
  s.steps = s.list ? tiles : 0;
  const int64_t steps = (int64_t)n_groups * (rows / (per <= 256 ? 256 / per : 1) + n_seqs) * ((max_length + 127) / 128 + 2);
  if (s.tensor && steps > s.steps) s.steps = steps;
  if (kw) {
    const int64_t again = (int64_t)n_groups * ((max_length + 127) / 128) * ((rows * per + 127) / 128 + 2 * (int64_t)n_seqs);
    if (again > s.steps) s.steps = again;
    s.score_rows = (int)(most < 8 * s.nq ? most : 8 * s.nq);
    if (s.list && path != 3 && tiles * s.score_rows * kShTile <= kScoresMax) {
      s.scores = tiles * s.score_rows * kShTile;
      s.kept_max = s.list_max;
    }
    if (s.tensor || s.kept_max == 0) {
      const double blocks = (double)n_groups * n_seqs * ((max_length + 127) / 128) * ((max_rows * per + 127) / 128);
      s.kw_workers = blocks < sm_count() ? (int)blocks : sm_count();
    }
  }
  s.bytes = (size_t)s.slots * (hs + 2) * sizeof(float) + (size_t)s.q * 2 + (size_t)s.items * sizeof(int2) + (size_t)n_seqs * 2 * sizeof(int) +
            (kw ? (size_t)rows * per * n_groups * sizeof(float) : 0) + (size_t)s.scores * sizeof(float) + (size_t)s.kw_workers * (256 * sizeof(float) + sizeof(PagedWeightCut)) + (size_t)tc_slots * (hs + 2) * sizeof(float) + (size_t)s.tc_workers * sizeof(PagedCut);
  // A cluster where its warps have four tiles each at most, and all clusters run at once.  us of the list and of clusters: 1 token of 32 groups, 128 numbers a head, over 300 keys 13.5, 7.7, over
  // 2000 14.1, 10.7, over 8000 30.4, 28.3 (the list's all the same: more than four tiles a warp); of 8 groups of 4 heads over 8000 16.2, 16.8; 16 tokens of 32 groups over 300 18.3, 19.9; 64 of 8
  // groups over 100 15.1, 16.2; 7 of 12 groups, 64 numbers a head, over 500 12.3, 8.3; 16 of them over 1000 16.0, 18.0.
  s.cluster = 0;
  if (max_rows == 1 && !kw && per <= 16 && (path == 0 || path == 4)) {   // (then the list takes every sequence, and nq queries hold a group's heads)
    const int64_t key_tiles = (max_length + kShTile - 1) / kShTile, pairs = (int64_t)n_seqs * n_groups;
    int ctas = 1;
    while (ctas < 8 && (ctas * 4 < key_tiles || ctas * 4 < per) && pairs * 2 * ctas <= 2 * sm_count()) ctas *= 2;   // (its CTAs share the heads' joins, too)
    if (path == 4 || (key_tiles <= 16 * ctas && pairs * ctas <= (hs == 64 ? 6 : 3) * sm_count())) s.cluster = ctas;
  }
  if (s.cluster) s.bytes = 0;
  const int64_t results = 2 + (int64_t)s.workers / s.items;
  s.ways = 1;                      // four results a warp are one round; no more warps than the GPU has at once
  while (s.ways < 8 && results > 4 * s.ways && rows * n_groups * per * s.ways < 24 * sm_count()) s.ways *= 2;
  return s;
}

template <int HS, int NQ, bool KEEP>
cudaError_t launch_list_of(const PagedParams& p, const PagedPlan& s, cudaStream_t st) {
  using C = PgSmem<HS, NQ>;
  static PerDeviceOnce once;
  if (once.need()) {
    const cudaError_t e = cudaFuncSetAttribute(paged_list_kernel<HS, NQ, KEEP>, cudaFuncAttributeMaxDynamicSharedMemorySize, C::kBytes);
    if (e != cudaSuccess) return e;
    once.done();
  }
  return launch(paged_list_kernel<HS, NQ, KEEP>, dim3((unsigned)s.ctas), dim3(C::kWarps * 32), (size_t)C::kBytes, st, p);
}

template <int HS, int NQ>
cudaError_t launch_list(const PagedParams& p, const PagedPlan& s, cudaStream_t st) { return p.scores ? launch_list_of<HS, NQ, true>(p, s, st) : launch_list_of<HS, NQ, false>(p, s, st); }

template <int HS, int NQ>
cudaError_t launch_clusters(const PagedParams& p, const PagedPlan& s, cudaStream_t st) {
  using C = ClSmem<HS, NQ>;
  if (p.per > 8 * NQ) return cudaErrorInvalidValue;
  static PerDeviceOnce once;
  if (once.need()) {
    const cudaError_t e = cudaFuncSetAttribute(paged_cluster_kernel<HS, NQ>, cudaFuncAttributeMaxDynamicSharedMemorySize, C::kBytes);
    if (e != cudaSuccess) return e;
    once.done();
  }
  return launch_cluster(paged_cluster_kernel<HS, NQ>, dim3((unsigned)(p.n_seqs * p.n_groups * s.cluster)), dim3(C::kWarps * 32), s.cluster, (size_t)C::kBytes, st, p, s.cluster);
}

template <int HS>
cudaError_t launch_paged(const PagedParams& p, const PagedPlan& s, cudaStream_t st) {
  if (s.cluster) return s.nq == 1 ? launch_clusters<HS, 1>(p, s, st) : launch_clusters<HS, 2>(p, s, st);
  const int64_t warps = (int64_t)p.rows * p.n_groups * (p.per + 2);
  cudaError_t e;
  if (p.wide) {                    // few rows: a row's heads on several CTAs, as many as are at once
    const int turns = (p.n_groups * (p.per + 2) * (HS / 16) + 255) / 256, ctas = p.sms * 4 / p.rows;
    e = launch(paged_append_wide_kernel<HS>, dim3((unsigned)p.rows, (unsigned)(ctas < 1 ? 1 : ctas < turns ? ctas : turns)), dim3(256), 0, st, p);
  } else {
    e = launch(paged_append_kernel<HS>, dim3((unsigned)((warps + 7) / 8)), dim3(256), 0, st, p);
  }
  if (e != cudaSuccess) return e;
  if (s.tensor && (e = launch_paged_tc05(p, HS, st)) != cudaSuccess) return e;
  if (s.list) {
    e = s.nq == 4 ? launch_list<HS, 4>(p, s, st) : s.nq == 2 ? launch_list<HS, 2>(p, s, st) : launch_list<HS, 1>(p, s, st);
    if (e != cudaSuccess) return e;
  }
  const int heads = 8 / s.ways, joins = s.list ? p.rows * ((p.n_head + heads - 1) / heads) : 0;
  e = launch(paged_join_kernel<HS>, dim3((unsigned)(p.tc_workers * kCutParts + joins)), dim3(256), 0, st, p);
  if (e != cudaSuccess || !p.kw) return e;
  if (s.kw_workers > 0 && (e = launch_paged_weights(p, HS, st)) != cudaSuccess) return e;
  const int64_t pairs = p.scores ? (int64_t)p.n_seqs * p.n_groups : 0;
  const int64_t runs = p.scores ? (p.max_length + 255) / 256 : 1, most = 16 * p.sms / (pairs + 1) + 1;   // (a few rounds of CTAs at most)
  return launch(paged_kept_kernel, dim3((unsigned)(p.kw_workers + pairs), (unsigned)(runs < most ? runs : most)), dim3(256), 0, st, p);
}

}  // namespace
}  // namespace b200

using namespace b200;

extern "C" {

size_t b200_attn_paged_workspace_bytes(int64_t rows, int n_seqs, int n_head, int n_groups, int head_size, int64_t max_rows, int64_t max_length, int key_weights) {
  if (rows <= 0 || n_seqs <= 0 || n_groups <= 0 || n_head <= 0 || n_head % n_groups || max_rows <= 0 || max_rows > rows || max_length <= 0 || (head_size != 64 && head_size != 128) ||
      rows * n_head >= (1 << 24) || (int64_t)n_seqs * n_groups >= (1 << 24) || max_length >= (1 << 30))
    return 0;
  return paged_plan(rows, n_seqs, n_groups, n_head / n_groups, head_size, max_rows, max_length, key_weights != 0).bytes;
}

int b200_attn_paged_tune(int path) { return g_paged_path.exchange(path >= 1 && path <= 4 ? path : 0); }

int b200_attn_paged(const b200_attn_paged_args* a, b200_stream_t stream) {
  B200_CHECK_ARG(a, "b200_attn_paged: null argument");
  B200_CHECK_ARG(a->head_size == 64 || a->head_size == 128, "b200_attn_paged: head size %d (64 or 128)", a->head_size);
  B200_CHECK_ARG(a->rows > 0 && a->n_seqs > 0 && a->n_groups > 0 && a->n_head > 0 && a->n_head % a->n_groups == 0, "b200_attn_paged: bad rows, sequences, heads %d or groups %d",
                 a->n_head, a->n_groups);
  B200_CHECK_ARG(a->rows < (1 << 24) && a->rows * a->n_head < (1 << 24) && (int64_t)a->n_seqs * a->n_groups < (1 << 24), "b200_attn_paged: too many rows or sequences in a step");
  B200_CHECK_ARG(a->max_rows > 0 && a->max_rows <= a->rows, "b200_attn_paged: sequences of up to %lld rows, of %lld", (long long)a->max_rows, (long long)a->rows);
  B200_CHECK_ARG(a->page >= 16 && a->page <= 256 && (a->page & (a->page - 1)) == 0, "b200_attn_paged: pages of %d keys (16, 32, 64, 128 or 256)", a->page);
  B200_CHECK_ARG(a->pool > 0 && a->table_seqs > 0 && a->max_pages > 0 && a->pages_ld >= a->max_pages, "b200_attn_paged: no pages, or a bad page table");
  B200_CHECK_ARG(a->max_length > 0 && a->max_length <= (int64_t)a->max_pages * a->page && a->max_length < (1 << 30), "b200_attn_paged: %lld keys in %d pages of %d",
                 (long long)a->max_length, a->max_pages, a->page);
  B200_CHECK_ARG(a->qkv && a->row_pos && a->row_seq && a->seqs && a->pages && a->k_pages && a->v_pages && a->out, "b200_attn_paged: null pointer");
  B200_CHECK_ARG(a->rope_n_elem >= 0 && a->rope_n_elem <= a->head_size && a->rope_n_elem % 2 == 0, "b200_attn_paged: bad rope_n_elem %d", a->rope_n_elem);
  B200_CHECK_ARG(a->rope_n_elem == 0 || (a->cos && a->sin && a->table_rows > 0), "b200_attn_paged: no tables");
  B200_CHECK_ARG(!a->table_preselected || a->rope_n_elem == 0 || a->table_rows >= a->rows, "b200_attn_paged: %d preselected table rows for %lld rows", a->table_rows, (long long)a->rows);
  B200_CHECK_ARG(a->table_dtype == B200_F32 || a->table_dtype == B200_BF16, "b200_attn_paged: tables must be fp32 or bf16");
  const uintptr_t at = (uintptr_t)a->k_pages | (uintptr_t)a->v_pages | (uintptr_t)a->workspace | (uintptr_t)a->seqs;
  const int64_t strides = a->k_page_stride | a->k_group_stride | a->v_page_stride | a->v_group_stride;
  B200_CHECK_ARG((at & 15) == 0 && (strides & 7) == 0 && ((uintptr_t)a->out & 15) == 0 && ((uintptr_t)a->key_weights & 3) == 0,
                 "b200_attn_paged: pages, result, workspace and the sequences' description must lie on 16-byte boundaries");
  const int per = a->n_head / a->n_groups;
  const PagedPlan s = paged_plan(a->rows, a->n_seqs, a->n_groups, per, a->head_size, a->max_rows, a->max_length, a->key_weights != nullptr);
  B200_CHECK_ARG(s.steps < kMaxTiles, "b200_attn_paged: too many keys in a step");
  B200_CHECK_ARG(a->workspace_bytes >= s.bytes && (a->workspace || s.bytes == 0), "b200_attn_paged: workspace too small");
  if (s.tensor || s.kw_workers > 0) B200_CHECK_WAITS("b200_attn_paged");
  PagedParams p = {};
  p.qkv = (const __nv_bfloat16*)a->qkv;
  p.cos = a->cos; p.sin = a->sin; p.table_bf16 = a->table_dtype == B200_BF16; p.table_rows = a->table_rows; p.table_presel = a->table_preselected; p.rope_n = a->rope_n_elem;
  p.wide = (((uintptr_t)a->qkv | (uintptr_t)a->cos | (uintptr_t)a->sin) & 15) == 0 && a->rope_n_elem % 16 == 0;
  p.row_pos = a->row_pos; p.pos64 = a->pos_is_int64; p.row_seq = a->row_seq;
  p.seqs = (const int4*)a->seqs; p.n_seqs = a->n_seqs;
  p.pages = a->pages; p.pages_ld = a->pages_ld; p.page_rows = a->table_seqs; p.max_pages = a->max_pages; p.pool = a->pool;
  for (p.shift = 4; (1 << p.shift) < a->page; ++p.shift) {}
  p.k = (__nv_bfloat16*)a->k_pages; p.v = (__nv_bfloat16*)a->v_pages;
  p.k_page = a->k_page_stride; p.k_group = a->k_group_stride; p.v_page = a->v_page_stride; p.v_group = a->v_group_stride;
  p.kw = a->key_weights;
  p.out = (__nv_bfloat16*)a->out;
  p.rows = (int)a->rows; p.n_head = a->n_head; p.n_groups = a->n_groups; p.per = per; p.max_rows = (int)a->max_rows; p.max_length = (int)a->max_length;
  p.tile_rows = 8 * s.nq; p.items = (int)s.items; p.workers = s.workers; p.sms = sm_count(); p.ways = s.ways;
  // (every part of wide accesses begins on a 16-byte boundary: they come first)
  p.q = (__nv_bfloat16*)a->workspace;
  p.acc = (float*)(p.q + s.q);
  p.ml = (float2*)(p.acc + s.slots * a->head_size);
  p.mixed = s.tensor && s.list; p.list_ns = a->head_size == 64 ? 182 : 364; p.tensor_ns = a->head_size == 64 ? 2550 : 3400;
  p.list_max = s.list_max; p.tc_workers = s.tc_workers; p.tc_rows = per <= 256 ? 256 / per : 1;
  p.tc_acc = (float*)(p.ml + s.slots);
  p.tc_ml = (float2*)(p.tc_acc + (int64_t)s.tc_workers * 512 * a->head_size);
  p.where = (int2*)(p.tc_ml + (int64_t)s.tc_workers * 512);
  p.cuts = (PagedCut*)(p.where + s.items);
  p.item_base = (int*)(p.cuts + s.tc_workers);
  p.score_rows = s.score_rows; p.kept_max = s.kept_max; p.kw_workers = s.kw_workers;
  p.tile_base = p.item_base + a->n_seqs;
  p.kw_cuts = (PagedWeightCut*)(p.tile_base + a->n_seqs);
  p.kw_part = (float*)(p.kw_cuts + s.kw_workers);
  p.lse = p.kw ? p.kw_part + (int64_t)s.kw_workers * 256 : nullptr;
  p.scores = s.scores ? p.lse + (int64_t)p.rows * p.per * p.n_groups : nullptr;
  p.scale_log2 = 1.4426950408889634f / sqrtf((float)a->head_size);
  const cudaStream_t st = (cudaStream_t)stream;
  B200_CUDA((a->head_size == 128 ? launch_paged<128>(p, s, st) : launch_paged<64>(p, s, st)));
  return B200_OK;
}

}  // extern "C"
