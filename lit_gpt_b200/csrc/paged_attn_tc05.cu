// Chunks of new tokens over a paged key-value cache on the 5th-generation tensor cores (paged_attn.cu has the step, and says which sequences come here).
//
// An item is a block of up to 256 queries of one sequence and group -- whole rows, every head of the group -- against the keys that its last row sees, in tiles of 128.  The key tiles of
// all items are one list, cut evenly over the CTAs, one an SM: neither few rows over many keys nor chunks of unequal lengths leave SMs without work.  A CTA's part of an item is a segment.
// The result of an item that is one CTA's is stored at once; else every segment leaves maxima, sums and unscaled outputs, and the step's join (paged_attn.cu) puts them together.
//   * warps 0-3 and 4-7: the softmax of the block's first and second 128 queries, one per thread.  S (128 columns of tensor memory) is read into registers once, as many as the
//     other warps give up; the probabilities go back over it as bf16, the left operand of P V, in two halves so that P V starts on the first;
//   * warps 8-11: when a row's maximum grew, they shrink its O in tensor memory while its exponentials are still being taken;
//   * warp 12: one thread issues S = Q K^T and O += P V, 128 x 128 x 16 each, S of a tile's next step right behind its P V;
//   * warp 13 brings the keys and the queries, warp 14 the values, two stages each, 128-byte-swizzled: a page, or what of it lies in the tile, is one TMA box; values of a tile that
//     ends past the sequence's last key, or has no page somewhere, come row by row with cp.async, zeros where there is nothing.
// A row that is not the sequence's whose range holds it (row_seq) is computed from whatever lies in its place and not stored; there is no key in its place.
// A masked key has weight 0, and 0 times an infinite or NaN value is NaN: a value of the chunk that is not finite reaches the rows before its own, within its
// tile of 128 keys and 128 queries.
// Probabilities are rounded to bf16 as they multiply V; the running maximum is exact, so that the largest probability is 1 and loses nothing.  They are summed before the rounding: the
// keys' weights are taken from these sums (of rounded ones a result's error against 64 bits is 0.1 to 0.4 % smaller, a weight's thousands of times larger).
//
// Bound: a stream's chain of scores, maximum, exponentials and output, which the other stream fills in part: a tile of 256 queries takes 3300 clocks where its products and its exponentials take
// 2048 each.  4096 rows of 32 groups of 1 head 143 us, 0.96 PFLOP/s of the causal half; 613 rows behind 1500 keys, 8 groups of 4 heads, 32 us, 4 of them the way to the
// first tile.  The instruction cache takes part: the roles walk different code, and each wait that was unrolled 64 times cost them all (tc05.cuh, mbar_wait_loop).
// Not taken, measured while they were and the step with 4096 rows took 200 us and more: half of S read twice: products 163 -> 178; half of a query's scores a thread, sixteen softmax warps at 80
// registers: the step 223 -> 275; the scores of the next tile's keys 64 .. 127, whose place is free early, ahead of P V: 200 -> 222 (products of 64 columns cost shared memory nearly what those of 128
// do).  A segment's results stored a query a thread in whole rows: 4 us each; four numbers of 128 queries side by side: 2.
#include "attn_tmem.cuh"
#include "paged.cuh"

#include <type_traits>

namespace b200 {

namespace {

constexpr int kPtThreads = 512, kPtSegs = 16;

template <int HS>
struct PtTile {
  static constexpr int kPanels = HS / 64;                  // 128-byte-wide panels of a tile of 128 rows
  static constexpr int kBytes = kPanels * 128 * 128;       // one operand tile
  static constexpr int kSmem = 6 * kBytes + 1024;          // Q0 Q1 | K x 2 | V x 2
  static constexpr uint32_t kIdescS = (1u << 4) | (1u << 7) | (1u << 10) | ((uint32_t)(128 >> 3) << 17) | ((uint32_t)(128 >> 4) << 24);
  static constexpr uint32_t kIdescO = (1u << 4) | (1u << 7) | (1u << 10) | (1u << 16) | ((uint32_t)(HS >> 3) << 17) | ((uint32_t)(128 >> 4) << 24);
  static constexpr uint32_t kS = 0, kO = 256;              // tensor-memory columns: S0 S1 (P over them) | O0 O1
};

// ---- the list of key tiles ----
// The list is cut by steps: an item counts as its key tiles and kLead more, the time that its queries' way in and its results' way out take (4 to 5 us where a tile takes 2.2).
constexpr int kLead = 2;
struct Blocks {            // of a sequence
  int count;               // of a group; none where the sequence is the list's
  int rows_each, cached, rows, n;
  __device__ __forceinline__ int steps(int block) const { return block < count ? kLead + ((min(cached + min((block + 1) * rows_each, rows), n) + 127) >> 7) : 0; }
};
__device__ __forceinline__ Blocks blocks_of(const PagedParams& p, const PagedSeq& s) {
  Blocks b;
  b.rows_each = p.tc_rows;
  b.count = s.rows * p.per > p.list_max ? (s.rows + b.rows_each - 1) / b.rows_each : 0;
  b.cached = s.cached; b.rows = s.rows; b.n = s.n;
  return b;
}
// The steps of a group, by a whole warp.
__device__ __forceinline__ int steps_of(const Blocks& b, int lane) {
  int64_t s = 0;
  for (int i = lane; i < b.count; i += 32) s += b.steps(i);
  int c = capped(s);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) c = capped((int64_t)c + __shfl_xor_sync(0xffffffffu, c, o));
  return c;
}

struct Seg {
  int q0, count;           // first query in the workspace's order, queries
  int m0, first;           // its number within the sequence and group; the sequence's first row
  int s, cached, n, table, gi;
  int lo, hi, hi0;         // key tiles; those of the first 128 queries end at hi0
  int slot;                // place of its results; -1: the item is done here
};

struct ListAt {            // where the list of segments goes on
  int tile, end;
  int s, gi, block, lo;    // sequence, group, block, first key tile
};

template <int HS>
__global__ void __launch_bounds__(kPtThreads, 1)
paged_tc05_kernel(const PagedParams p, const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v, unsigned* err) {
  using C = PtTile<HS>;
  extern __shared__ __align__(1024) uint8_t pt_smem[];
  __shared__ __align__(8) uint64_t s_bars[27];
  __shared__ float s_shrink[256];         // per query: what its O and sum shrink by in this step
  __shared__ __align__(16) uint32_t s_bits[4][4];        // keys of a tile that have a page, of the last four tiles
  __shared__ Seg s_seg[kPtSegs];
  __shared__ ListAt s_at;
  __shared__ PagedCut s_cut;
  __shared__ int s_segs, s_more;
  __shared__ uint32_t s_tmem;
  __shared__ int s_sums[kPtThreads + 1], s_warp[kPtThreads / 32];
  __shared__ Shares s_shares[kPtThreads / 32];
  __shared__ long long s_held[kPtThreads / 32];          // rows that the sequences hold, by warps
  __shared__ int s_owned[kPtThreads / 32];               // and those that are the sequence's which holds them: as many unless rows are taken out of a sequence's range
  const int tid = threadIdx.x, lane = tid & 31, warp = __shfl_sync(0xffffffffu, tid >> 5, 0);
  const uint32_t smem = (tc::smem_u32(pt_smem) + 1023u) & ~1023u;
  const uint32_t sq_ = smem, sk_ = smem + 2 * C::kBytes, sv_ = smem + 4 * C::kBytes;
  const uint32_t bars = tc::smem_u32(s_bars);
  const uint32_t k_full = bars, v_full = bars + 16, k_empty = bars + 32, v_empty = bars + 48, s_full = bars + 64, p_half = bars + 80, p_full = bars + 96,
                 o_done = bars + 112, q_full = bars + 128, shrink = bars + 136, idle = bars + 200;   // shrink: one per softmax warp; idle: products that gave up

  if (!p.mixed) griddep_launch();
  // ---- this CTA's part of the list: from the step's description, which was there before the append kernel ----
  // (of up to 32 sequences by one warp: without the other warps' sums 1 to 2 us less)
  const bool few = p.n_seqs <= 32;
  const int run = (p.n_seqs + kPtThreads - 1) / kPtThreads, turns = few && warp > 0 ? 0 : run;
  int here = 0, owned = 0;
  long long held = 0;
  Shares work = {0ull, 0ull};
#pragma unroll 4
  for (int row = tid; row < p.rows; row += kPtThreads) {
    const int of = p.row_seq[row];
    const bool any = of >= 0 && of < p.n_seqs;
    const PagedSeq s = paged_seq(p, any ? of : 0);
    owned += any && row >= s.first && row - s.first < s.rows;
  }
  for (int k = 0; k < turns; ++k) {
    const int i = tid * run + k;
    Blocks mine = {};
    if (i < p.n_seqs) {
      const PagedSeq s = paged_seq(p, i);
      mine = blocks_of(p, s);
      held += s.rows;
      if (p.mixed) add_work(p, s, work);
    }
    if (mine.count <= 16) {
      for (int e = 0; e < mine.count; ++e) here = capped((int64_t)here + mine.steps(e));
    }
    for (unsigned left = __ballot_sync(0xffffffffu, mine.count > 16); left; left &= left - 1) {   // long ones: by all lanes, one after the other
      const int of = __ffs(left) - 1;
      Blocks b;
      b.rows_each = p.tc_rows;
      b.count = __shfl_sync(0xffffffffu, mine.count, of);
      b.cached = __shfl_sync(0xffffffffu, mine.cached, of);
      b.rows = __shfl_sync(0xffffffffu, mine.rows, of);
      b.n = __shfl_sync(0xffffffffu, mine.n, of);
      const int sum = steps_of(b, lane);
      if (lane == of) here = capped((int64_t)here + sum);
    }
  }
  int inc = here;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int x = __shfl_up_sync(0xffffffffu, inc, o);
    if (lane >= o) inc = capped((int64_t)inc + x);
  }
  if (few) {
    if (warp == 0) {
      s_sums[lane] = inc - here;
      if (lane == 31) s_sums[32] = s_sums[kPtThreads] = inc;
    }
  } else if (lane == 31) {
    s_warp[warp] = inc;
  }
  if (p.mixed) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      work.list += __shfl_xor_sync(0xffffffffu, work.list, o);
      work.tensor += __shfl_xor_sync(0xffffffffu, work.tensor, o);
    }
    if (lane == 0) s_shares[warp] = work;
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) held += __shfl_xor_sync(0xffffffffu, held, o);
  owned = __reduce_add_sync(0xffffffffu, owned);
  if (lane == 0) {
    s_held[warp] = held;
    s_owned[warp] = owned;
  }
  if (tid == kPtThreads - 32) {
    tc::mbar_init(q_full, 1);
    tc::mbar_init(idle, 1);
    for (int i = 0; i < 2; ++i) {
      tc::mbar_init(k_full + 8 * i, 1);
      tc::mbar_init(v_full + 8 * i, 1);
      tc::mbar_init(k_empty + 8 * i, 1);
      tc::mbar_init(v_empty + 8 * i, 1);
      tc::mbar_init(s_full + 8 * i, 1);
      tc::mbar_init(p_half + 8 * i, 8);   // the softmax and the shrinking warps
      tc::mbar_init(p_full + 8 * i, 4);
      tc::mbar_init(o_done + 8 * i, 1);
    }
    for (int i = 0; i < 8; ++i) tc::mbar_init(shrink + 8 * i, 1);
    tc::mbar_init_fence();
  }
  __syncthreads();
  if (!few) {
    int before = inc - here;
    for (int w = 0; w < warp; ++w) before = capped((int64_t)before + s_warp[w]);
    s_sums[tid] = before;
    if (tid == kPtThreads - 1) s_sums[kPtThreads] = capped((int64_t)before + here);
    __syncthreads();
  }
  const int64_t all64 = (int64_t)s_sums[kPtThreads] * p.n_groups;
  const int all = all64 < kMaxTiles ? (int)all64 : 0;      // (a description whose sequences overlap can hold more: then none is done)
  int ctas = gridDim.x;
  if (p.mixed) {                        // the list's kernel takes the other SMs: it may begin once the append kernel has ended
    work = {0ull, 0ull};
    for (int w = 0; w < kPtThreads / 32; ++w) { work.list += s_shares[w].list; work.tensor += s_shares[w].tensor; }
    ctas = tensor_share(p, work);
    if ((int)blockIdx.x >= ctas) {
      griddep_wait();
      griddep_launch();
      if (tid == 0) {
        PagedCut c = {};
        c.last = -1;
        p.cuts[blockIdx.x] = c;
      }
      return;
    }
  }
  if (warp == 0) {
    const int workers = min(max(all / 2, min(all, ctas)), ctas), w = blockIdx.x;
    const int each = workers ? all / workers : 0, more = all - each * workers;
    const int first = w * each + min(w, more), end = w < workers ? first + each + (w < more ? 1 : 0) : first;
    ListAt at = {};
    at.tile = first;
    at.end = end;
    PagedCut c = {};                    // for the launch that joins: the item that this CTA goes on with
    c.last = all64 < kMaxTiles ? -1 : kCutNothing;
    if (first < end) {
      int lo = 0, hi = few ? 32 : kPtThreads;
      while (hi - lo > 1) {
        const int mid = (lo + hi) / 2;
        if ((int64_t)s_sums[mid] * p.n_groups <= first) lo = mid; else hi = mid;
      }
      int rest = first - s_sums[lo] * p.n_groups, of_group;
      PagedSeq seq;
      Blocks blk;
      for (at.s = lo * run;; ++at.s) {
        seq = paged_seq(p, at.s);
        blk = blocks_of(p, seq);
        of_group = run == 1 ? s_sums[lo + 1] - s_sums[lo] : steps_of(blk, lane);
        if (rest < of_group * p.n_groups) break;
        rest -= of_group * p.n_groups;
      }
      at.gi = rest / of_group;
      rest -= at.gi * of_group;
      for (int b0 = 0;; b0 += 32) {     // the block that holds it
        const int t = blk.steps(b0 + lane);
        int sum = t;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) { const int x = __shfl_up_sync(0xffffffffu, sum, o); if (lane >= o) sum += x; }
        const unsigned behind = __ballot_sync(0xffffffffu, sum > rest);
        if (behind) {
          const int of = __ffs(behind) - 1;
          at.block = b0 + of;
          at.lo = rest - __shfl_sync(0xffffffffu, sum - t, of);
          break;
        }
        rest -= __shfl_sync(0xffffffffu, sum, 31);
      }
      if (at.lo > kLead) {
        const int m0 = at.block * blk.rows_each * p.per, wide = more * (each + 1);
        auto worker_of = [&](int tile) { return tile < wide ? tile / (each + 1) : more + (tile - wide) / each; };
        c.first = worker_of(first - at.lo + kLead);   // (whose part holds the first key tile)
        c.last = worker_of(first - at.lo + blk.steps(at.block) - 1);
        c.count = min(blk.rows_each * p.per, seq.rows * p.per - m0);
        c.row = seq.first + at.block * blk.rows_each;
        c.gi = at.gi;
      }
    }
    if (lane == 0) {
      s_cut = c;
      s_at = at;
    }
  }
  uint32_t tmem = 0;
  bool ok = true;
  // counted over all segments, so that every barrier's phase is known
  int tiles_done = 0, segs_done = 0;                       // loads and products
  uint32_t n[2] = {0u, 0u};                                // steps of either 128 queries

  auto list_segments = [&]() {            // by thread 0
    ListAt at = s_at;
    int c = 0;
    if (at.tile < at.end) {
      PagedSeq seq = paged_seq(p, at.s);
      Blocks blk = blocks_of(p, seq);
      for (; c < kPtSegs && at.tile < at.end; c += s_seg[c].hi > s_seg[c].lo) {   // (a part without a key tile is none)
        const int steps = blk.steps(at.block), m0 = at.block * blk.rows_each * p.per, count = min(blk.rows_each * p.per, seq.rows * p.per - m0);
        Seg& g = s_seg[c];
        g.q0 = (at.gi * p.rows + seq.first) * p.per + m0;
        g.count = count;
        g.m0 = m0;
        g.first = seq.first;
        g.s = at.s; g.cached = seq.cached; g.n = seq.n; g.table = seq.table; g.gi = at.gi;
        const int stop = min(steps, at.lo + at.end - at.tile);
        g.lo = max(at.lo - kLead, 0);
        g.hi = max(stop - kLead, 0);
        g.hi0 = min(g.hi, (min(seq.cached + (m0 + min(count, 128) - 1) / p.per + 1, seq.n) + 127) >> 7);
        g.slot = g.lo == 0 && stop == steps ? -1 : 2 * (int)blockIdx.x + (g.lo == 0);   // (of a CTA's segments only the first begins, only the last ends within an item)
        at.tile += stop - at.lo;
        if (at.tile >= at.end) continue;
        at.lo = 0;
        if (++at.block == blk.count) {
          at.block = 0;
          if (++at.gi == p.n_groups) {
            at.gi = 0;
            do {
              seq = paged_seq(p, ++at.s);
              blk = blocks_of(p, seq);
            } while (blk.count == 0);
          }
        }
      }
    }
    s_at = at;                                           // (in shared memory: the softmax has no registers for it)
    s_segs = c;
    s_more = at.tile < at.end;
  };
  if (tid == 0) list_segments();
  griddep_wait();                         // (tensor memory is taken behind the wait only)
  if (p.mixed) griddep_launch();
  if (warp == 12) tc::tmem_alloc<512>(tc::smem_u32(&s_tmem));
  if (tid == 0) p.cuts[blockIdx.x] = s_cut;
  tc::fence_before();
  __syncthreads();
  tc::fence_after();
  tmem = s_tmem;
  auto more_segments = [&]() {            // by all, behind a batch's segments
    ok = __syncthreads_and(ok);
    const bool more = ok && s_more;
    __syncthreads();                      // (everyone has read s_more)
    return more;
  };
  auto strangers = [&]() {                // whether a row is not the sequence's whose range holds it
    long long held = 0, owned = 0;
    for (int w = 0; w < kPtThreads / 32; ++w) { held += s_held[w]; owned += s_owned[w]; }
    return held != owned;
  };
  // A role has its loop over batches of segments to itself, so that its registers are its own: the softmax warps hold a query's 128 scores, and registers go from the others to them
  // (256 x 192 + 256 x 56 of the launch's 512 x 128).
  if (warp >= 12) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 56;");
    // (whose rows a tile's keys are is looked up only where some are not the sequence's: 613 rows behind 1500 42.6 us, with the look in every loop 42.9, a prompt of 4096 186, 192)
    auto loads = [&](auto strangers) {
      for (;;) {
        const int segs = s_segs;
      // ================================ loads ================================
      const bool keys = warp == 13;
      const uint32_t dst = keys ? sk_ : sv_, full = keys ? k_full : v_full, empty = keys ? k_empty : v_empty;
      const CUtensorMap* const map = keys ? &map_k : &map_v;
      const int parts = p.shift >= 7 ? 1 : 128 >> p.shift, part_rows = min(128, 1 << p.shift);
      for (int c = 0; c < segs && ok; ++c) {
        const Seg& g = s_seg[c];
        const int lo = g.lo, hi = g.hi, total = g.n, table = g.table, gi = g.gi;
        auto page_of = [&](int j) { return lane < parts ? page_at(p, table, ((j * 128) >> p.shift) + lane) : -1; };
        int id = page_of(lo);
        for (int j = lo; j < hi; ++j, ++tiles_done) {
          const int s = tiles_done & 1;
          const int next = j + 1 < hi ? page_of(j + 1) : -1;
          ok = __all_sync(0xffffffffu, tc::mbar_wait_loop(empty + 8 * s, ((uint32_t)(tiles_done >> 1) & 1u) ^ 1u));
          if (!ok) break;
          const uint32_t have = __ballot_sync(0xffffffffu, id >= 0);
          bool whole = have == (1u << parts) - 1u;
          uint32_t own = 0xffffffffu;   // lane l < 4: keys 32 l and on, but those of rows that are not the sequence's
          if constexpr (strangers.value) {
#pragma unroll 1
            for (int e = 0; e < 4; ++e) {
              const int key = j * 128 + 32 * e + lane;
              const uint32_t word = __ballot_sync(0xffffffffu, key >= total || whose_key(p, g.s, g.cached, g.first, key) == g.s);
              if (lane == e) own = word;
            }
            whole = whole && __all_sync(0xffffffffu, own == 0xffffffffu);
          }
          if (keys && lane < 4) {       // word l: keys 32 l and on
            uint32_t bits = 0u;
            if (p.shift >= 5) bits = (have >> ((lane * 32) >> min(p.shift, 7))) & 1u ? 0xffffffffu : 0u;
            else bits = ((have >> (2 * lane)) & 1u ? 0xffffu : 0u) | ((have >> (2 * lane + 1)) & 1u ? 0xffff0000u : 0u);
            s_bits[tiles_done & 3][lane] = strangers.value ? bits & own : bits;
          }
          const int row = p.shift >= 7 ? (j * 128) & ((1 << p.shift) - 1) : 0;
          if (keys || (whole && (j + 1) * 128 <= total)) {
            __syncwarp();               // (the words are written before the barrier that hands them over is arrived on)
            if (lane == 0) tc::mbar_expect_tx(full + 8 * s, (uint32_t)(__popc(have) * part_rows * HS * 2));
            __syncwarp();
            if (id >= 0) {
#pragma unroll
              for (int e = 0; e < C::kPanels; ++e)
                load_page(dst + s * C::kBytes + e * 16384u + (uint32_t)(lane * part_rows) * 128u, map, e * 64, row, gi, id, full + 8 * s);
            }
          } else {
            constexpr int CH = HS / 8, RP = 32 / CH;   // 16-byte pieces per row, rows per pass
            const int cc = lane % CH;
            const __nv_bfloat16* const base = p.v + (int64_t)gi * p.v_group + cc * 8;
            const uint32_t to = dst + s * C::kBytes + (uint32_t)(cc >> 3) * 16384u;
#pragma unroll 8
            for (int i = 0; i < 128 / RP; ++i) {
              const int r = i * RP + lane / CH, at = __shfl_sync(0xffffffffu, id, p.shift >= 7 ? 0 : r >> p.shift);
              bool in = at >= 0 && j * 128 + r < total;
              if constexpr (strangers.value) in = (__shfl_sync(0xffffffffu, own, r >> 5) >> (r & 31) & 1u) && in;
              cp16(to + (uint32_t)(r * 128 + (((cc & 7) ^ (r & 7)) << 4)), in ? base + (int64_t)at * p.v_page + (int64_t)((row + r) & ((1 << p.shift) - 1)) * HS : base, in);
            }
            asm volatile("cp.async.wait_all;" ::: "memory");
            tc::fence_smem_async();
            __syncwarp();
            if (lane == 0) tc::mbar_arrive(full + 8 * s);
          }
          if (keys && j == lo) {        // the queries, once the segment before has done its last product with the ones there
            if (tiles_done > 0) ok = __all_sync(0xffffffffu, tc::mbar_wait_loop(k_empty + 8 * (s ^ 1), (uint32_t)((tiles_done - 1) >> 1) & 1u));
            if (!ok) break;
            const int halves = g.count > 128 ? 2 : 1;
            if (lane == 0) {
              tc::mbar_expect_tx(q_full, halves * C::kBytes);
              for (int h = 0; h < halves; ++h)
#pragma unroll
                for (int e = 0; e < C::kPanels; ++e) tc::tma_load_2d(sq_ + h * C::kBytes + e * 16384u, &map_q, e * 64, g.q0 + h * 128, q_full);
            }
            __syncwarp();
          }
          id = next;
        }
        ++segs_done;
      }
        if (!more_segments()) break;
        __syncthreads();
      }
    };
    const bool loading = warp == 13 || warp == 14, checked = loading && strangers();
    if (loading && !checked) {
      loads(std::false_type{});
    } else if (warp == 12) {
      for (;;) {
        const int segs = s_segs;
      // ================================ products ================================
      if (tc::elect()) {
        const uint32_t q_low = tc::desc_sw128_low(sq_), k_low = tc::desc_sw128_low(sk_), v_low = desc_v_low(sv_);
        auto scores = [&](int t, int s) {                    // S of query tile t with the keys of stage s
          const uint32_t q = q_low + t * (C::kBytes >> 4), k = k_low + s * (C::kBytes >> 4);
#pragma unroll
          for (int e = 0; e < HS / 16; ++e) {
            const uint32_t off = ((uint32_t)(e >> 2) * 16384u + (uint32_t)(e & 3) * 32u) >> 4;
            mma_ss(tmem + C::kS + t * 128, tc::desc_of(q + off, tc::kDescSw128High), tc::desc_of(k + off, tc::kDescSw128High), C::kIdescS, e != 0);
          }
          tc::commit(s_full + 8 * t);
        };
        for (int c = 0; c < segs && ok; ++c) {
          const Seg& g = s_seg[c];
          const int lo = g.lo, hi = g.hi, hi0 = g.hi0, hi1 = g.count > 128 ? hi : lo;
          ok = tc::mbar_wait_loop(q_full, (uint32_t)segs_done & 1u) && tc::mbar_wait_loop(k_full + 8 * (tiles_done & 1), (uint32_t)(tiles_done >> 1) & 1u);
          if (!ok) break;
          tc::fence_after();
#pragma unroll
          for (int t = 0; t < 2; ++t)
            if (lo < (t ? hi1 : hi0)) scores(t, tiles_done & 1);
          tc::commit(k_empty + 8 * (tiles_done & 1));
          bool fresh[2] = {true, true};
          for (int j = lo; j < hi; ++j, ++tiles_done) {
            const int i = tiles_done, s = i & 1, s1 = s ^ 1;
            const bool more_keys = j + 1 < hi;
            ok = tc::mbar_wait_loop(v_full + 8 * s, (uint32_t)(i >> 1) & 1u) && (!more_keys || tc::mbar_wait_loop(k_full + 8 * s1, (uint32_t)((i + 1) >> 1) & 1u));
            if (!ok) break;
#pragma unroll
            for (int t = 0; t < 2; ++t) {
              const int stop = t ? hi1 : hi0;
              if (j < stop) {
                const uint32_t dv = v_low + s * (C::kBytes >> 4);
#pragma unroll
                for (int half = 0; half < 2; ++half) {
                  ok = ok && tc::mbar_wait_loop((half ? p_full : p_half) + 8 * t, n[t] & 1u);
                  if (!ok) break;
                  tc::fence_after();
#pragma unroll
                  for (int e = 4 * half; e < 4 * half + 4; ++e)
                    mma_ts(tmem + C::kO + t * HS, tmem + C::kS + t * 128 + e * 8, tc::desc_of(dv + 128 * e, tc::kDescSw128High), C::kIdescO, !fresh[t] || e != 0);
                }
                if (!ok) break;
                fresh[t] = false;
                tc::commit(o_done + 8 * t);
                ++n[t];
              }
              if (more_keys && j + 1 < stop) scores(t, s1);
            }
            if (!ok) break;
            tc::commit(v_empty + 8 * s);
            if (more_keys) tc::commit(k_empty + 8 * s1);
          }
          ++segs_done;
        }
        if (!ok) {
          tc::commit(idle);
          tc::mbar_wait_loop(idle, 0);
        }
      }
      ok = __all_sync(0xffffffffu, ok);
        if (!more_segments()) break;
        __syncthreads();
      }
    } else if (checked) {
      loads(std::true_type{});
    } else {
      while (more_segments()) __syncthreads();
    }
  } else if (warp >= 8) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 56;");
    for (;;) {
      const int segs = s_segs;
      // ================================ shrinking O ================================
      const int v = warp - 8;
      for (int c = 0; c < segs && ok; ++c) {
        const Seg& g = s_seg[c];
        const int lo = g.lo, hi = g.hi, hi0 = g.hi0, hi1 = g.count > 128 ? hi : lo;
        for (int j = lo; j < hi && ok; ++j) {
#pragma unroll
          for (int t = 0; t < 2; ++t) {
            if (j >= (t ? hi1 : hi0)) continue;
            ok = ok && __all_sync(0xffffffffu, tc::mbar_wait_loop(shrink + 8 * (4 * t + v), n[t] & 1u));
            if (!ok) break;
            const float f = s_shrink[t * 128 + v * 32 + lane];
            if (__any_sync(0xffffffffu, f != 1.0f)) {   // (S of this step is there, so P V of the last one is done; a segment's first step has f = 1)
              tc::fence_after();
              const uint32_t to = tmem + ((uint32_t)(v * 32) << 16) + C::kO + t * HS;
#pragma unroll 1
              for (int cc = 0; cc < HS; cc += 16) {
                uint32_t o[16];
                tc::ld16(o, to + cc);
                tc::wait_ld(o);
#pragma unroll
                for (int e = 0; e < 16; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * f);
                st16(to + cc, o);
              }
              wait_st();
              tc::fence_before();
            }
            __syncwarp();
            if (lane == 0) tc::mbar_arrive(p_half + 8 * t);
            ++n[t];
          }
        }
      }
      if (!more_segments()) break;
      __syncthreads();
    }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 192;");
    for (;;) {
      const int segs = s_segs;
      // ================================ softmax: a query per thread ================================
      const int t = warp >> 2;
      const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
      const uint32_t ts = tmem + lanes + C::kS + t * 128, to = tmem + lanes + C::kO + t * HS;
      const float sl = p.scale_log2;
      int tiles_before = tiles_done;                       // of this batch's segments before the current one
      for (int c = 0; c < segs && ok; ++c) {
        const Seg& g = s_seg[c];
        const int count = g.count, lo = g.lo, hi = t ? (count > 128 ? g.hi : lo) : g.hi0;
        const int row = (g.m0 + tid) / p.per;              // of the sequence
        const int lim = tid < count ? min(g.cached + row, g.n - 1) : -1;
        const int w_lim = __reduce_min_sync(0xffffffffu, lim < 0 ? 0x7fffffff : lim);
        float m = -INFINITY;
        f2 l2[2] = {0ull, 0ull};
        const uint32_t n0 = n[0];
        for (int j = lo; j < hi; ++j, ++n[0]) {
          ok = ok && __all_sync(0xffffffffu, tc::mbar_wait_loop(s_full + 8 * t, n[0] & 1u));
          if (!ok) break;
          tc::fence_after();
          const int j0 = j * 128;
          const uint4 bits = *reinterpret_cast<const uint4*>(s_bits[(tiles_before + j - lo) & 3]);
          const bool holes = (bits.x & bits.y & bits.z & bits.w) != 0xffffffffu;
          const bool masked = j0 + 127 > w_lim || holes;   // (queries past the segment's are computed and not stored)
          auto mask = [&](uint32_t (&s)[32], int i) {
            if (masked) {
              const uint32_t there = i == 0 ? bits.x : i == 1 ? bits.y : i == 2 ? bits.z : bits.w;
#pragma unroll
              for (int e = 0; e < 32; ++e) {
                const int key = j0 + i * 32 + e;
                if (key > lim || !((there >> e) & 1u)) s[e] = 0xff800000u;
              }
            }
          };
          auto most = [](const uint32_t (&s)[32], float mx) {
#pragma unroll
            for (int e = 0; e < 32; e += 2) mx = max3(mx, __uint_as_float(s[e]), __uint_as_float(s[e + 1]));
            return mx;
          };
          uint32_t v[4][32];
          float mx[4];
#pragma unroll
          for (int i = 0; i < 4; ++i) tc::ld32(v[i], ts + 32 * i);
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            tc::wait_ld(v[i]);
            mask(v[i], i);
            mx[i] = most(v[i], -INFINITY);
          }
          const float nm = fmaxf(m, fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])));
          const float f = m == -INFINITY ? 1.0f : ex2((m - nm) * sl);   // nothing seen so far: O and the sum are zero
          m = nm;
          s_shrink[tid] = f;
          __syncwarp();
          if (lane == 0) tc::mbar_arrive(shrink + 8 * warp);
          const f2 ff = pk2(f, f);
          l2[0] = fma2(l2[0], ff, 0ull);
          l2[1] = fma2(l2[1], ff, 0ull);
          const float org = m == -INFINITY ? 0.f : m * sl;   // queries with nothing visible yet: exp2(-inf) = 0
          const f2 sl2 = pk2(sl, sl), org2 = pk2(-org, -org);
          auto exps = [&](const uint32_t (&s)[32], int i) {
            uint32_t q[16];
#pragma unroll
            for (int e = 0; e < 16; ++e) {
              float a, b;
              un2(fma2(pk2(__uint_as_float(s[2 * e]), __uint_as_float(s[2 * e + 1])), sl2, org2), a, b);
              a = ex2(a);
              b = ex2(b);
              q[e] = pack_bf16(a, b);
              l2[e & 1] = add2(l2[e & 1], pk2(a, b));
            }
            st16(ts + i * 16, q);
          };
          auto hand_over = [&](uint32_t bar) {
            wait_st();
            tc::fence_before();
            __syncwarp();
            if (lane == 0) tc::mbar_arrive(bar + 8 * t);
          };
          exps(v[0], 0);
          exps(v[1], 1);
          hand_over(p_half);
          exps(v[2], 2);
          exps(v[3], 3);
          hand_over(p_full);
        }
        tiles_before += g.hi - lo;
        const int whose = tid < count ? p.row_seq[g.first + row] : -1;   // (of a row that is not the sequence's the queries are whatever lay there)
        const bool any = n[0] != n0;
        if (any && ok) {
          ok = __all_sync(0xffffffffu, tc::mbar_wait_loop(o_done + 8 * t, (n[0] - 1) & 1u));
          tc::fence_after();
        }
        if (!ok) break;
        if (t * 128 < count) {
          float a, b, d, e;
          un2(l2[0], a, b);
          un2(l2[1], d, e);
          const float l = (a + b) + (d + e);
          const int slot = g.slot;
          const int hh = g.m0 + tid - row * p.per;
          if (slot < 0) {
            const float inv = l > 0.f ? 1.0f / l : 0.f;   // (NaN: the output is NaN itself)
            const int64_t y_at = whose == g.s ? ((int64_t)(g.first + row) * p.n_head + g.gi * p.per + hh) * HS : -1;
#pragma unroll 1
            for (int c0 = 0; c0 < HS; c0 += 32) {
              uint32_t o[32], x[16];
              tc::ld32(o, to + c0);
              tc::wait_ld(o);
#pragma unroll
              for (int i = 0; i < 16; ++i) x[i] = any ? pack_bf16(__uint_as_float(o[2 * i]) * inv, __uint_as_float(o[2 * i + 1]) * inv) : 0u;
              // Four neighbouring lanes have 64 bytes of four rows, and swap so that each store has 64 bytes of eight rows and not sixteen of 32: piece i of lane l becomes piece l of the
              // row of lane i (the four stores of 16 bytes at one address a lane took 2.2 us a segment).
#pragma unroll
              for (int d = 1; d < 4; d <<= 1) {
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                  if (i & d) continue;
#pragma unroll
                  for (int e = 0; e < 4; ++e) {
                    const bool high = lane & d;
                    const uint32_t give = high ? x[4 * i + e] : x[4 * (i + d) + e];
                    const uint32_t got = __shfl_xor_sync(0xffffffffu, give, d);
                    if (high) x[4 * i + e] = got; else x[4 * (i + d) + e] = got;
                  }
                }
              }
#pragma unroll
              for (int i = 0; i < 4; ++i) {
                const int64_t to_row = __shfl_sync(0xffffffffu, y_at, (lane & ~3) + i);
                if (to_row >= 0) *reinterpret_cast<uint4*>(p.out + to_row + c0 + (lane & 3) * 8) = make_uint4(x[4 * i], x[4 * i + 1], x[4 * i + 2], x[4 * i + 3]);
              }
            }
            if (p.lse && whose == g.s) p.lse[g.q0 + tid] = l == 0.f ? INFINITY : m * sl + log2f(l);
          } else {
            float* const at = p.tc_acc + (int64_t)slot * 256 * HS + tid * 4;   // four numbers of every query side by side: a warp's stores are whole lines (a query's all together: 4 us a segment)
#pragma unroll 1
            for (int c0 = 0; c0 < HS; c0 += 32) {
              uint32_t o[32];
              tc::ld32(o, to + c0);
              tc::wait_ld(o);
              if (tid < count) {
#pragma unroll
                for (int i = 0; i < 32; i += 4) __stcg(reinterpret_cast<uint4*>(at + (int64_t)(c0 + i) * 256), make_uint4(o[i], o[i + 1], o[i + 2], o[i + 3]));
              }
            }
            if (tid < count) __stcg(p.tc_ml + (int64_t)slot * 256 + tid, whose != g.s ? make_float2(-INFINITY, 0.f) : make_float2(m == -INFINITY ? m : m * sl, any ? l : 0.f));
          }
          tc::fence_before();
        }
      }
      tiles_done = tiles_before;
      if (!more_segments()) break;
      if (tid == 0) list_segments();
      __syncthreads();
    }
  }
  if (!ok) {
    // copies on their way: neither stage may be written once this CTA has left
    if (warp == 13 || warp == 14) {
      const uint32_t full = warp == 13 ? k_full : v_full;
      for (int e = max(tiles_done - 2, 0); e < tiles_done; ++e) tc::mbar_wait_loop(full + 8 * (e & 1), (uint32_t)(e >> 1) & 1u);
      if (warp == 13 && segs_done > 0) tc::mbar_wait_loop(q_full, (uint32_t)(segs_done - 1) & 1u);
    }
    *err = 1u;
  }
  tc::fence_before();
  __syncthreads();
  if (warp == 12) {
    __syncwarp();
    tc::tmem_free<512>(tmem);
  }
}

template <int HS>
cudaError_t launch_hs(const PagedParams& p, cudaStream_t st) {
  constexpr int smem = PtTile<HS>::kSmem;
  static PerDeviceOnce once;
  if (once.need()) {
    const cudaError_t e = cudaFuncSetAttribute(paged_tc05_kernel<HS>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    if (e != cudaSuccess) return e;
    once.done();
  }
  alignas(64) CUtensorMap mq, mk, mv;
  const int page = 1 << p.shift;
  if (!tensor_map_2d(&mq, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, p.q, (int64_t)p.n_groups * p.rows * p.per, HS, HS * 2, 128) ||
      !page_map(&mk, p.k, HS, page, p.n_groups, p.pool, p.k_group, p.k_page) || !page_map(&mv, p.v, HS, page, p.n_groups, p.pool, p.v_group, p.v_page))
    return cudaErrorInvalidValue;
  unsigned* const err = wait_error_word();
  if (!err) return cudaErrorMemoryAllocation;
  return launch(paged_tc05_kernel<HS>, dim3((unsigned)p.tc_workers), dim3(kPtThreads), (size_t)smem, st, p, mq, mk, mv, err);
}

}  // namespace

cudaError_t launch_paged_tc05(const PagedParams& p, int head_size, cudaStream_t st) { return head_size == 128 ? launch_hs<128>(p, st) : launch_hs<64>(p, st); }

}  // namespace b200
