// The attention weight that the keys of a paged cache receive in a step (paged_attn.cu): per key and group the sum, over the step's rows and the group's heads, of
//   exp2(s - lse),   s the score and lse the logarithm of the row's sum of exponentials, both times log2(e).
//
// Sequences of the list of tiles leave their scores behind (a hundredth to a sixth of their keys' bytes); paged_kept_kernel (paged_attn.cu) adds up what they give, a key a thread.
//
// The others' are computed again on the 5th-generation tensor cores, paged_weights_kernel: S^T = K Q^T, 128 keys as the rows of tensor memory and 128 queries as its columns, so that a
// thread has a key, its sum stays in registers and nothing is reduced across threads.  An item is a block of 128 keys of a sequence and group against the tiles of queries that see it; the
// tiles of all items are one list, cut evenly over the CTAs.  The sums of an item that several CTAs have parts of are added by the same kernel, in the order of the CTAs.
//   * warps 0-3 and 4-7: the even and the odd tiles of queries, a key a thread: s in registers, a query's lse from shared memory (one address for all lanes), an exponential and an addition
//   * warp 8: one thread issues the products, four tiles of scores in tensor memory
//   * warp 9 brings keys (a page, or what of it lies in the block, is one TMA box), queries (four stages) and the queries' lse
// No atomics: one order of additions.
//
// Bound: the exponentials, 16 a clock and SM: 2048 clocks for two tiles of queries.  512 rows behind 2000 keys, 8 groups of 4 heads: 24 us, 10 of them the exponentials; the rest the way to the
// first tile (6), and the sums' way out (on mma.sync, a tile of 32 keys a warp, 137).
#include "attn_tmem.cuh"
#include "paged.cuh"

#include <type_traits>

namespace b200 {

namespace {

constexpr int kKwThreads = 320, kKwSegs = 16;
constexpr int kKwLead = 1;                // an item counts as its tiles of queries and so many more: its keys' way in

template <int HS>
struct KwTile {
  static constexpr int kPanels = HS / 64, kBytes = kPanels * 128 * 128;
  static constexpr int kSmem = 6 * kBytes + 1024;          // K x 2 | Q x 4
  static constexpr uint32_t kIdesc = (1u << 4) | (1u << 7) | (1u << 10) | ((uint32_t)(128 >> 3) << 17) | ((uint32_t)(128 >> 4) << 24);
};

struct KeyBlocks {                        // of a sequence
  int count, m;                           // blocks of 128 keys (none where its scores were kept); queries
  int cached, per;
  __device__ __forceinline__ int from(int block) const { return max(block * 128 - cached, 0) * per >> 7; }   // earlier tiles of queries see none of its keys
  __device__ __forceinline__ int steps(int block) const { return block < count ? kKwLead + ((m + 127) >> 7) - from(block) : 0; }
};
__device__ __forceinline__ KeyBlocks key_blocks(const PagedParams& p, const PagedSeq& s) {
  KeyBlocks b;
  b.m = s.rows * p.per;
  b.count = b.m > p.kept_max ? (s.n + 127) >> 7 : 0;
  b.cached = s.cached;
  b.per = p.per;
  return b;
}
__device__ __forceinline__ int steps_of(const KeyBlocks& b, int lane) {
  int64_t s = 0;
  for (int i = lane; i < b.count; i += 32) s += b.steps(i);
  int c = capped(s);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) c = capped((int64_t)c + __shfl_xor_sync(0xffffffffu, c, o));
  return c;
}

struct KwSeg {
  int s, row;                             // the sequence, its first row
  int q0, m;                              // the sequence's and group's first query in the workspace's order; queries
  int cached, n, table, gi;
  int block, lo, hi;                      // tiles of queries
  int slot;                               // place of its sums; -1: the item is done here
};
struct KwAt {
  int tile, end;
  int s, gi, block, lo;
};

template <int HS>
__global__ void __launch_bounds__(kKwThreads, 1)
paged_weights_kernel(const PagedParams p, const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_k, unsigned* err) {
  using C = KwTile<HS>;
  extern __shared__ __align__(1024) uint8_t kw_smem[];
  __shared__ __align__(8) uint64_t s_bars[29];
  __shared__ __align__(16) float s_lse[8][128];            // of the last eight tiles of queries, negative: tile i + 8's are written once the products of tile i + 4 are done, whose scores
                                                           // take the place of tile i's
  __shared__ int s_blind[8];                               // whether a query of theirs sees no key, or there are fewer than 128
  __shared__ float s_sum[128];
  __shared__ KwSeg s_seg[kKwSegs];
  __shared__ KwAt s_at;
  __shared__ PagedWeightCut s_cut;
  __shared__ int s_segs, s_more, s_sums[kKwThreads + 1], s_warp[kKwThreads / 32];
  __shared__ uint32_t s_tmem;
  const int tid = threadIdx.x, lane = tid & 31, warp = __shfl_sync(0xffffffffu, tid >> 5, 0);
  const uint32_t smem = (tc::smem_u32(kw_smem) + 1023u) & ~1023u, sk_ = smem, sq_ = smem + 2 * C::kBytes;
  const uint32_t bars = tc::smem_u32(s_bars);
  const uint32_t k_full = bars, k_empty = bars + 16, q_full = bars + 32, q_empty = bars + 64, s_full = bars + 96, s_empty = bars + 128, idle = bars + 160, x_full = bars + 168, x_empty = bars + 200;

  griddep_launch();
  // ---- this CTA's part of the list: from the step's description ----
  const bool few = p.n_seqs <= 32;        // by one warp
  const int run = (p.n_seqs + kKwThreads - 1) / kKwThreads, turns = few && warp > 0 ? 0 : run;
  int here = 0;
  for (int k = 0; k < turns; ++k) {
    const int i = tid * run + k;
    KeyBlocks mine = {};
    if (i < p.n_seqs) mine = key_blocks(p, paged_seq(p, i));
    if (mine.count <= 16) {
      for (int e = 0; e < mine.count; ++e) here = capped((int64_t)here + mine.steps(e));
    }
    for (unsigned left = __ballot_sync(0xffffffffu, mine.count > 16); left; left &= left - 1) {
      const int of = __ffs(left) - 1;
      KeyBlocks b;
      b.count = __shfl_sync(0xffffffffu, mine.count, of);
      b.m = __shfl_sync(0xffffffffu, mine.m, of);
      b.cached = __shfl_sync(0xffffffffu, mine.cached, of);
      b.per = p.per;
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
      if (lane == 31) s_sums[32] = s_sums[kKwThreads] = inc;
    }
  } else if (lane == 31) {
    s_warp[warp] = inc;
  }
  if (tid == kKwThreads - 32) {
    for (int i = 0; i < 2; ++i) {
      tc::mbar_init(k_full + 8 * i, 1);
      tc::mbar_init(k_empty + 8 * i, 1);
    }
    for (int i = 0; i < 4; ++i) {
      tc::mbar_init(q_full + 8 * i, 1);
      tc::mbar_init(q_empty + 8 * i, 1);
      tc::mbar_init(s_full + 8 * i, 1);
      tc::mbar_init(s_empty + 8 * i, 4);
      tc::mbar_init(x_full + 8 * i, 1);
      tc::mbar_init(x_empty + 8 * i, 1);
    }
    tc::mbar_init(idle, 1);
    tc::mbar_init_fence();
  }
  __syncthreads();
  if (!few) {
    int before = inc - here;
    for (int w = 0; w < warp; ++w) before = capped((int64_t)before + s_warp[w]);
    s_sums[tid] = before;
    if (tid == kKwThreads - 1) s_sums[kKwThreads] = capped((int64_t)before + here);
    __syncthreads();
  }
  if (warp == 0) {
    const int64_t all64 = (int64_t)s_sums[kKwThreads] * p.n_groups;
    const int all = all64 < kMaxTiles ? (int)all64 : 0;
    const int workers = min(max(all / 2, min(all, p.sms)), p.kw_workers), w = blockIdx.x;
    const int each = workers ? all / workers : 0, more = all - each * workers;
    const int first = w * each + min(w, more), end = w < workers ? first + each + (w < more ? 1 : 0) : first;
    KwAt at = {};
    at.tile = first;
    at.end = end;
    PagedWeightCut c = {};
    c.last = -1;
    if (first < end) {
      int lo = 0, hi = few ? 32 : kKwThreads;
      while (hi - lo > 1) {
        const int mid = (lo + hi) / 2;
        if ((int64_t)s_sums[mid] * p.n_groups <= first) lo = mid; else hi = mid;
      }
      int rest = first - s_sums[lo] * p.n_groups, of_group;
      PagedSeq seq;
      KeyBlocks blk;
      for (at.s = lo * run;; ++at.s) {
        seq = paged_seq(p, at.s);
        blk = key_blocks(p, seq);
        of_group = run == 1 ? s_sums[lo + 1] - s_sums[lo] : steps_of(blk, lane);
        if (rest < of_group * p.n_groups) break;
        rest -= of_group * p.n_groups;
      }
      at.gi = rest / of_group;
      rest -= at.gi * of_group;
      for (int b0 = 0;; b0 += 32) {
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
      const int wide = more * (each + 1);
      auto worker_of = [&](int tile) { return tile < wide ? tile / (each + 1) : more + (tile - wide) / each; };
      if (at.lo > kKwLead && worker_of(first - at.lo + kKwLead) == w - 1) {   // (the first of those that go on with it joins it)
        c.first = w - 1;
        c.last = worker_of(first - at.lo + blk.steps(at.block) - 1);
        c.s = at.s; c.row = seq.first; c.cached = seq.cached;
        c.table = seq.table; c.n = seq.n; c.gi = at.gi; c.block = at.block;
      }
    }
    if (lane == 0) {
      s_cut = c;
      s_at = at;
    }
  }
  uint32_t tmem = 0;
  bool ok = true, began = false;
  int segs_done = 0, tiles_done = 0;      // counted over all segments, so that every barrier's phase is known

  for (;;) {
    if (tid == 0) {
      KwAt at = s_at;
      int c = 0;
      if (at.tile < at.end) {
        PagedSeq seq = paged_seq(p, at.s);
        KeyBlocks blk = key_blocks(p, seq);
        for (; c < kKwSegs && at.tile < at.end; c += s_seg[c].hi > s_seg[c].lo) {   // (a part without a tile is none)
          const int steps = blk.steps(at.block), stop = min(steps, at.lo + at.end - at.tile), from = blk.from(at.block);
          KwSeg& g = s_seg[c];
          g.s = at.s; g.row = seq.first;
          g.q0 = (at.gi * p.rows + seq.first) * p.per;
          g.m = blk.m;
          g.cached = seq.cached; g.n = seq.n; g.table = seq.table; g.gi = at.gi;
          g.block = at.block;
          g.lo = from + max(at.lo - kKwLead, 0);
          g.hi = from + max(stop - kKwLead, 0);
          g.slot = at.lo <= kKwLead && stop == steps ? -1 : 2 * (int)blockIdx.x + (at.lo <= kKwLead);
          at.tile += stop - at.lo;
          if (at.tile >= at.end) continue;
          at.lo = 0;
          if (++at.block == blk.count) {
            at.block = 0;
            if (++at.gi == p.n_groups) {
              at.gi = 0;
              do {
                seq = paged_seq(p, ++at.s);
                blk = key_blocks(p, seq);
              } while (blk.count == 0);
            }
          }
        }
      }
      s_at = at;
      s_segs = c;
      s_more = at.tile < at.end;
    }
    if (!began) {                         // (tensor memory is taken behind the wait only)
      griddep_wait();
      if (warp == 8) tc::tmem_alloc<512>(tc::smem_u32(&s_tmem));
      if (tid == 0) p.kw_cuts[blockIdx.x] = s_cut;
      tc::fence_before();
    }
    __syncthreads();
    if (!began) {
      tc::fence_after();
      tmem = s_tmem;
      began = true;
    }
    const int segs = s_segs;

    if (warp == 9) {
      // ================================ loads ================================
      const int parts = p.shift >= 7 ? 1 : 128 >> p.shift, part_rows = min(128, 1 << p.shift);
      for (int c = 0; c < segs && ok; ++c, ++segs_done) {
        const KwSeg& g = s_seg[c];
        const int ks = segs_done & 1;
        const int id = lane < parts ? page_at(p, g.table, ((g.block * 128) >> p.shift) + lane) : -1;
        ok = __all_sync(0xffffffffu, tc::mbar_wait(k_empty + 8 * ks, ((uint32_t)(segs_done >> 1) & 1u) ^ 1u));
        if (!ok) break;
        const uint32_t have = __ballot_sync(0xffffffffu, id >= 0);
        if (lane == 0) tc::mbar_expect_tx(k_full + 8 * ks, (uint32_t)(__popc(have) * part_rows * HS * 2));
        __syncwarp();
        if (id >= 0) {
          const int row = p.shift >= 7 ? (g.block * 128) & ((1 << p.shift) - 1) : 0;
#pragma unroll
          for (int e = 0; e < C::kPanels; ++e) load_page(sk_ + ks * C::kBytes + e * 16384u + (uint32_t)(lane * part_rows) * 128u, &map_k, e * 64, row, g.gi, id, k_full + 8 * ks);
        }
        auto lse_of = [&](int j, float (&f)[4]) {
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int m = j * 128 + lane * 4 + i;
            f[i] = m < g.m ? -__ldcg(p.lse + g.q0 + m) : -INFINITY;
          }
        };
        float f[4];
        lse_of(g.lo, f);
        for (int j = g.lo; j < g.hi; ++j, ++tiles_done) {
          const int s = tiles_done & 3;
          ok = __all_sync(0xffffffffu, tc::mbar_wait(q_empty + 8 * s, ((uint32_t)(tiles_done >> 2) & 1u) ^ 1u));
          if (!ok) break;
          *reinterpret_cast<float4*>(&s_lse[tiles_done & 7][lane * 4]) = make_float4(f[0], f[1], f[2], f[3]);
          const int blind = __any_sync(0xffffffffu, f[0] == -INFINITY || f[1] == -INFINITY || f[2] == -INFINITY || f[3] == -INFINITY);
          if (lane == 0) s_blind[tiles_done & 7] = blind;
          __syncwarp();                   // (written before the barrier that hands them over is arrived on)
          if (lane == 0) {
            tc::mbar_expect_tx(q_full + 8 * s, C::kBytes);
#pragma unroll
            for (int e = 0; e < C::kPanels; ++e) tc::tma_load_2d(sq_ + s * C::kBytes + e * 16384u, &map_q, e * 64, g.q0 + j * 128, q_full + 8 * s);
          }
          __syncwarp();
          if (j + 1 < g.hi) lse_of(j + 1, f);
        }
      }
    } else if (warp == 8) {
      // ================================ products ================================
      if (tc::elect()) {
        const uint32_t q_low = tc::desc_sw128_low(sq_), k_low = tc::desc_sw128_low(sk_);
        for (int c = 0; c < segs && ok; ++c, ++segs_done) {
          const KwSeg& g = s_seg[c];
          const int ks = segs_done & 1, lo = g.lo, hi = g.hi;
          ok = tc::mbar_wait_here(k_full + 8 * ks, (uint32_t)(segs_done >> 1) & 1u);
          for (int j = lo; j < hi && ok; ++j, ++tiles_done) {
            const int s = tiles_done & 3;
            ok = tc::mbar_wait_here(q_full + 8 * s, (uint32_t)(tiles_done >> 2) & 1u) && tc::mbar_wait_here(s_empty + 8 * s, ((uint32_t)(tiles_done >> 2) & 1u) ^ 1u);
            if (!ok) break;
            tc::fence_after();
            const uint32_t q = q_low + s * (C::kBytes >> 4), k = k_low + ks * (C::kBytes >> 4);
#pragma unroll
            for (int e = 0; e < HS / 16; ++e) {
              const uint32_t off = ((uint32_t)(e >> 2) * 16384u + (uint32_t)(e & 3) * 32u) >> 4;
              mma_ss(tmem + s * 128, tc::desc_of(k + off, tc::kDescSw128High), tc::desc_of(q + off, tc::kDescSw128High), C::kIdesc, e != 0);
            }
            tc::commit(s_full + 8 * s);
            tc::commit(q_empty + 8 * s);
          }
          if (!ok) break;
          tc::commit(k_empty + 8 * ks);
        }
        if (!ok) {
          tc::commit(idle);
          tc::mbar_wait(idle, 0);
        }
      }
      ok = __all_sync(0xffffffffu, ok);
    } else {
      // ================================ sums: a key per thread ================================
      const int t = warp >> 2, mine = tid & 127;
      const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
      const float sl = p.scale_log2;
      const f2 sl2 = pk2(sl, sl);
      for (int c = 0; c < segs && ok; ++c) {
        const KwSeg& g = s_seg[c];
        const int key = g.block * 128 + mine, lo = g.lo, hi = g.hi;
        const int low = max(key - g.cached, 0) * p.per;    // queries before this one do not see the key
        const int w_low = max(g.block * 128 + 127 - g.cached, 0) * p.per;
        f2 sum[2] = {0ull, 0ull};
        for (int j = lo; j < hi; ++j, ++tiles_done) {
          if ((tiles_done & 1) != t) continue;
          const int s = tiles_done & 3;
          ok = ok && __all_sync(0xffffffffu, tc::mbar_wait(s_full + 8 * s, (uint32_t)(tiles_done >> 2) & 1u));
          if (!ok) break;
          tc::fence_after();
          const int m0 = j * 128;
          const float* const lse = s_lse[tiles_done & 7];
          uint32_t x[32], y[32];
          auto add = [&](uint32_t (&v)[32], int i, auto masked) {
#pragma unroll
            for (int e = 0; e < 32; e += 4) {
              const float4 l = *reinterpret_cast<const float4*>(lse + i * 32 + e);
              float a, b, d, h;
              un2(fma2(pk2(__uint_as_float(v[e]), __uint_as_float(v[e + 1])), sl2, pk2(l.x, l.y)), a, b);
              un2(fma2(pk2(__uint_as_float(v[e + 2]), __uint_as_float(v[e + 3])), sl2, pk2(l.z, l.w)), d, h);
              a = ex2(a);
              b = ex2(b);
              d = ex2(d);
              h = ex2(h);
              if constexpr (masked.value) {   // (behind the exponentials: what a query gives a key that it does not see is zero even where its sum is NaN)
                const int from = low - m0 - i * 32;
                if (e < from || l.x == -INFINITY) a = 0.f;
                if (e + 1 < from || l.y == -INFINITY) b = 0.f;
                if (e + 2 < from || l.z == -INFINITY) d = 0.f;
                if (e + 3 < from || l.w == -INFINITY) h = 0.f;
              }
              sum[0] = add2(sum[0], pk2(a, b));
              sum[1] = add2(sum[1], pk2(d, h));
            }
          };
          const uint32_t at = tmem + lanes + s * 128;
          auto add_all = [&](auto masked) {
            tc::ld32(x, at);
            tc::wait_ld(x);
            tc::ld32(y, at + 32);
            add(x, 0, masked);
            tc::wait_ld(y);
            tc::ld32(x, at + 64);
            add(y, 1, masked);
            tc::wait_ld(x);
            tc::ld32(y, at + 96);
            add(x, 2, masked);
            tc::wait_ld(y);
            add(y, 3, masked);
          };
          if (m0 < w_low || s_blind[tiles_done & 7]) add_all(std::true_type{});
          else add_all(std::false_type{});
          tc::fence_before();
          __syncwarp();
          if (lane == 0) tc::mbar_arrive(s_empty + 8 * s);   // (behind the last look at the queries' lse: their place is taken again four tiles after the scores')
        }
        if (!ok) break;
        float a, b, d, h;
        un2(sum[0], a, b);
        un2(sum[1], d, h);
        const float total = (a + b) + (d + h);
        // warp w + 4 hands its sums to warp w, which adds them: one order
        const int w = warp & 3;
        if (t == 1) {
          ok = __all_sync(0xffffffffu, tc::mbar_wait(x_empty + 8 * w, ((uint32_t)segs_done & 1u) ^ 1u));
          if (!ok) break;
          s_sum[mine] = total;
          __syncwarp();
          if (lane == 0) tc::mbar_arrive(x_full + 8 * w);
        } else {
          ok = __all_sync(0xffffffffu, tc::mbar_wait(x_full + 8 * w, (uint32_t)segs_done & 1u));
          if (!ok) break;
          const float both = total + s_sum[mine];
          __syncwarp();
          if (lane == 0) tc::mbar_arrive(x_empty + 8 * w);
          if (g.slot >= 0) {
            __stcg(p.kw_part + g.slot * 128 + mine, both);
          } else {
            const int id = key_page(p, g.s, g.table, g.cached, g.row, g.n, key);
            if (id >= 0) p.kw[(((int64_t)id * p.n_groups + g.gi) << p.shift) + (key & ((1 << p.shift) - 1))] += both;
          }
        }
        ++segs_done;
      }
    }
    ok = __syncthreads_and(ok);
    if (!ok || !s_more) break;
    __syncthreads();                      // (everyone has read s_more)
  }
  if (!ok) {
    if (warp == 9) {                      // copies on their way: no stage may be written once this CTA has left
      for (int e = max(tiles_done - 4, 0); e < tiles_done; ++e) tc::mbar_wait(q_full + 8 * (e & 3), (uint32_t)(e >> 2) & 1u);
      for (int e = max(segs_done - 1, 0); e <= segs_done; ++e) tc::mbar_wait(k_full + 8 * (e & 1), (uint32_t)(e >> 1) & 1u);
    }
    *err = 1u;
  }
  tc::fence_before();
  __syncthreads();
  if (warp == 8) {
    __syncwarp();
    tc::tmem_free<512>(tmem);
  }
}

template <int HS>
cudaError_t launch_hs(const PagedParams& p, cudaStream_t st) {
  constexpr int smem = KwTile<HS>::kSmem;
  static PerDeviceOnce once;
  if (once.need()) {
    const cudaError_t e = cudaFuncSetAttribute(paged_weights_kernel<HS>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    if (e != cudaSuccess) return e;
    once.done();
  }
  alignas(64) CUtensorMap mq, mk;
  if (!tensor_map_2d(&mq, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, p.q, (int64_t)p.n_groups * p.rows * p.per, HS, HS * 2, 128) ||
      !page_map(&mk, p.k, HS, 1 << p.shift, p.n_groups, p.pool, p.k_group, p.k_page))
    return cudaErrorInvalidValue;
  unsigned* const err = wait_error_word();
  if (!err) return cudaErrorMemoryAllocation;
  return launch(paged_weights_kernel<HS>, dim3((unsigned)p.kw_workers), dim3(kKwThreads), (size_t)smem, st, p, mq, mk, err);
}

}  // namespace

cudaError_t launch_paged_weights(const PagedParams& p, int head_size, cudaStream_t st) { return head_size == 128 ? launch_hs<128>(p, st) : launch_hs<64>(p, st); }

}  // namespace b200
