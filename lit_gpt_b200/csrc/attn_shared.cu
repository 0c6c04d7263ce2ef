// One decode step (T = 1) of B rows that share a prefix: rotation of q and of the new k, append of the new k / v to the row's own cache, and
//   o = sum_j softmax_j(q . k_j / sqrt(hs)) v_j   over the prefix's keys [0, P) and the row's own keys [0, pos - P].
// The rounding points are those of the model's step (attn_decode.cu; lit_gpt/model.py:624-653, 767-773): q and k are bf16 after the rotation, the softmax is
// fp32 with a running maximum, the result is rounded once.
//
// The prefix is read once for all rows: the B * (heads per group) query rows of a key-value group are the left operand of its products, a key tile serves them all.
// Three launches: the queries and new keys are turned and the new rows stored; warps compute partial results (maximum, sum, unscaled output) over tiles of 32 keys of the
// prefix for up to 32 query rows of a group (the prefix's larger products: attn_shared_tc05.cu), and of a row's own keys for its heads of a group; a head's partial
// results are joined.  Few rows a group: the whole of it in one launch, a cluster of CTAs a group.  No counter or flag is left between calls, and two calls at a time share nothing.
//
// Bound: a few short rows by latency: 2 rows of 32 heads over 96 shared keys take 7.2 us, 1.8 MB (10.0 in three launches).  Else by bytes: 16 rows of 32 heads over 2048 shared and 200 own
// keys, 87 MB, take 25 us (3.5 TB/s): 13 at the memory's rate, the rest the way to the first tile, the queries' launch before it and the join behind it.
//
// All tiles, of the prefix and of all rows' own keys, are one list that is cut evenly over the warps of all SMs, so that neither few rows over a long prefix nor many
// rows of unequal lengths leave SMs without work.  A warp keeps a ring of units of 32 keys or values, two of them on their way, and the queries of its next item behind them.
// S^T = K Q^T and O^T += V^T P^T on mma.sync.m16n8k16, eight queries a product (with the queries as the left operand's sixteen rows 64 x 16001 took 68 us, with eight
// 58).  P enters as two bf16 numbers, its leading bits and the rest, so that its rounding does not add to the result's own (with the nearest bf16 number alone the
// error against 64 bits is a fifth larger than that of the final rounding).  The rest is taken of the number above the weight: it is not zero, and an infinite value
// times it is infinite and not NaN.
#include <math.h>

#include "attn_body.cuh"
#include "attn_shared.cuh"
#include "mma_tile.cuh"
#include "tc05.cuh"

namespace b200 {

namespace {

constexpr int kShTile = 32;                 // keys of a tile
constexpr float kAbove = 1.00000012f;       // 1 + 2^-23: a weight's second number is never zero
constexpr int kShUnits = 3;                 // a warp's ring: units of 32 keys or 32 values

// index of a row's new key in its own cache; -1: the row takes no part
__device__ __forceinline__ int own_index(const SharedParams& p, int64_t pos, int plen) {
  if (pos < 0) return -1;
  const int64_t i = pos - plen;
  return (int)(i < 0 ? 0 : (i >= p.own_rows ? p.own_rows - 1 : i));
}
__device__ __forceinline__ int64_t table_row(const SharedParams& p, int b, int64_t pos) {
  const int64_t r = p.table_presel ? (p.pos_each ? b : 0) : pos;
  return r < 0 ? 0 : (r >= p.table_rows ? p.table_rows - 1 : r);
}
__device__ __forceinline__ float ex2(float x) { float r; asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x)); return r; }

// apply_rope (lit_gpt/model.py:767-773)
__device__ __forceinline__ float turned(float a, float other, bool low, float c, float s, int table_bf16) {
  const float rot = low ? -other : other;
  if (table_bf16) return __fadd_rn(round_bf16(__fmul_rn(a, c)), round_bf16(__fmul_rn(rot, s)));
  return __fadd_rn(__fmul_rn(a, c), __fmul_rn(rot, s));
}
// HS / 32 numbers of a head from lane * HS / 32 on, after the rotation
template <int HS>
__device__ __forceinline__ void turned_part(const SharedParams& p, const __nv_bfloat16* x, int64_t trow, int lane, uint32_t (&out)[HS / 64]) {
  constexpr int V = HS / 32;
  const int n = p.rope_n, half = n >> 1, d0 = lane * V;
  if (p.wide) {
    auto get = [&](int d, float (&f)[V]) {
      if constexpr (V == 4) {
        const uint2 w = *reinterpret_cast<const uint2*>(x + d);
        f[0] = bf16lo(w.x); f[1] = bf16hi(w.x); f[2] = bf16lo(w.y); f[3] = bf16hi(w.y);
      } else {
        const uint32_t w = *reinterpret_cast<const uint32_t*>(x + d);
        f[0] = bf16lo(w); f[1] = bf16hi(w);
      }
    };
    auto table = [&](const void* t, float (&f)[V]) {
      const int64_t at = trow * n + d0;
      if (p.table_bf16) {
#pragma unroll
        for (int i = 0; i < V; ++i) f[i] = __bfloat162float(reinterpret_cast<const __nv_bfloat16*>(t)[at + i]);
      } else if constexpr (V == 4) {
        const float4 w = *reinterpret_cast<const float4*>(reinterpret_cast<const float*>(t) + at);
        f[0] = w.x; f[1] = w.y; f[2] = w.z; f[3] = w.w;
      } else {
        const float2 w = *reinterpret_cast<const float2*>(reinterpret_cast<const float*>(t) + at);
        f[0] = w.x; f[1] = w.y;
      }
    };
    float a[V];
    get(d0, a);
    if (d0 < n) {
      const bool low = d0 < half;
      float o[V], c[V], s[V];
      get(low ? d0 + half : d0 - half, o);
      table(p.cos, c);
      table(p.sin, s);
#pragma unroll
      for (int i = 0; i < V; ++i) a[i] = turned(a[i], o[i], low, c[i], s[i], p.table_bf16);
    }
#pragma unroll
    for (int i = 0; i < V / 2; ++i) out[i] = pack_bf16(a[2 * i], a[2 * i + 1]);
  } else {
    float a[V];
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const int d = d0 + i;
      a[i] = __bfloat162float(x[d]);
      if (d < n) {
        const bool low = d < half;
        a[i] = turned(a[i], __bfloat162float(x[low ? d + half : d - half]), low, table_at(p.cos, p.table_bf16, trow * n + d), table_at(p.sin, p.table_bf16, trow * n + d),
                      p.table_bf16);
      }
    }
#pragma unroll
    for (int i = 0; i < V / 2; ++i) out[i] = pack_bf16(a[2 * i], a[2 * i + 1]);
  }
}

// The tiles of a step, one after the other: rows' own keys, row after row, there group after group and tile of heads after tile of heads, then the prefix, group after
// group and tile of query rows after tile of query rows.  An item is what one query tile sees of one of them.  Workers take runs of tiles; the result of item i by worker w goes to
// slot i + w, which no other pair has, since either grows with the tiles.
struct Split {
  int own, all;          // tiles of own keys; all tiles
  int prefix, workers;   // tiles of the prefix for one item; workers
  int each, more;        // every worker has `each` tiles, the first `more` of them one more
};
__device__ __forceinline__ int worker_of(int tile, const Split& s) {
  const int wide = s.more * (s.each + 1);
  return tile < wide ? tile / (s.each + 1) : s.more + (tile - wide) / s.each;
}
__device__ __forceinline__ int first_tile(int w, const Split& s) { return w * s.each + min(w, s.more); }

// Rows are summed in runs of one per thread: sums[t] = own tiles (of one group and tile of heads) of the rows before run t, sums[THREADS] of all.  mine[b]: own_index of the
// rows there is place for.
template <int THREADS>
__device__ __forceinline__ Split make_split(const SharedParams& p, int plen, int* sums, int* mine, int* s_warp) {
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, run = (p.batch + THREADS - 1) / THREADS;
  int here = 0;
  for (int b = tid * run; b < min(p.batch, (tid + 1) * run); ++b) {
    const int at = own_index(p, row_pos(p, b), plen);
    if (b < THREADS) mine[b] = at;
    here += (at + kShTile) / kShTile;
  }
  int inc = here;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) { const int t = __shfl_up_sync(0xffffffffu, inc, o); if (lane >= o) inc += t; }
  if (lane == 31) s_warp[warp] = inc;
  __syncthreads();
  int before = inc - here;
  for (int w = 0; w < warp; ++w) before += s_warp[w];
  sums[tid] = before;
  if (tid == THREADS - 1) sums[THREADS] = before + here;
  __syncthreads();
  Split s;
  s.own = sums[THREADS] * p.n_groups * p.head_tiles;
  s.prefix = p.row_tiles ? (plen + kShTile - 1) / kShTile : 0;
  s.all = s.own + s.prefix * p.n_groups * p.row_tiles;
  // two tiles a worker at least, unless that leaves SMs without one
  s.workers = min(max(s.all / 2, min(s.all, p.sms)), p.workers);
  s.each = s.workers ? s.all / s.workers : 0;
  s.more = s.all - s.each * s.workers;
  return s;
}

// A warp's shared memory: a ring of units, the queries of two items.  One CTA an SM.  Queries come in eights: NP of them over the prefix, NO over a row's own keys.
template <int HS, int NP>
struct ShSmem {
  static constexpr int kUnit = kShTile * HS * 2, kQ = 8 * (NP > 2 ? NP : 2) * HS * 2;
  static constexpr int kWarp = kShUnits * kUnit + 2 * kQ;
  static constexpr int kWarps = HS == 64 ? (NP == 4 ? 10 : 12) : (NP == 4 ? 5 : 7);
  static constexpr int kBytes = kWarps * kWarp;
};

// ---- the queries and the new keys turned, the new rows stored: a head a warp ----
template <int HS>
__global__ void __launch_bounds__(256) attn_shared_turn_kernel(const SharedParams p) {
  constexpr int V = HS / 32;
  griddep_wait();     // (before the launch of what follows: the kernels behind read positions, lengths and the prefix ahead of their own wait)
  griddep_launch();
  const int lane = threadIdx.x & 31, heads = p.n_groups * (p.per + 2);
  const int64_t at = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5);
  const int b = (int)(at / heads), i = (int)(at - (int64_t)b * heads), gi = i / (p.per + 2), h = i - gi * (p.per + 2);
  if (b >= p.batch) return;
  const int64_t pos = row_pos(p, b);
  const __nv_bfloat16* const x = p.qkv + at * HS;
  uint32_t v[HS / 64];
  if (h <= p.per) {
    turned_part<HS>(p, x, table_row(p, b, pos), lane, v);
  } else {
    const uint16_t* const u = reinterpret_cast<const uint16_t*>(x + lane * V);
#pragma unroll
    for (int j = 0; j < V / 2; ++j) v[j] = (uint32_t)u[2 * j] | ((uint32_t)u[2 * j + 1] << 16);
  }
  __nv_bfloat16* to;
  if (h < p.per) {
    to = p.q + ((int64_t)gi * p.batch * p.per + (int64_t)b * p.per + h) * HS;
    if (pos < 0)
#pragma unroll
      for (int j = 0; j < V / 2; ++j) v[j] = 0u;
  } else {
    const int mine = own_index(p, pos, prefix_len(p));
    if (mine < 0) return;
    to = (h == p.per ? p.kc + (int64_t)b * p.kc_b + (int64_t)gi * p.kc_g : p.vc + (int64_t)b * p.vc_b + (int64_t)gi * p.vc_g) + (int64_t)mine * HS;
  }
  if constexpr (V == 4) *reinterpret_cast<uint2*>(to + lane * V) = make_uint2(v[0], v[V / 2 - 1]);
  else *reinterpret_cast<uint32_t*>(to + lane * V) = v[0];
}

// A tile of a worker's range, and the item that it belongs to.
struct Tile {
  int index;                         // in the order of all tiles
  const __nv_bfloat16* k; const __nv_bfloat16* v;   // its first rows
  int valid;                         // rows of it
  int left;                          // tiles of the item behind this one
  int own;                           // an own item?
  int b, gi, part;                   // row, group, tile of heads (own); -, group, tile of query rows
  int at;                            // own: index of the new key
};

template <int HS, int NP>
struct Walk {
  const SharedParams& p;
  const Split& s;
  const int* sums;
  const int* mine_of;                // of the first `threads` rows
  int plen, run, threads;

  __device__ __forceinline__ int mine(int b) const { return b < threads ? mine_of[b] : own_index(p, row_pos(p, b), plen); }

  __device__ __forceinline__ void own_item(Tile& t, int mine, int tile) const {
    const int tiles = mine / kShTile + 1;
    t.own = 1;
    t.at = mine;
    t.left = tiles - 1 - tile;
    t.k = p.kc + (int64_t)t.b * p.kc_b + (int64_t)t.gi * p.kc_g + (int64_t)tile * kShTile * HS;
    t.v = p.vc + (int64_t)t.b * p.vc_b + (int64_t)t.gi * p.vc_g + (int64_t)tile * kShTile * HS;
    t.valid = min(kShTile, mine + 1 - tile * kShTile);
  }
  __device__ __forceinline__ void prefix_item(Tile& t, int tile) const {
    t.own = 0;
    t.left = s.prefix - 1 - tile;
    t.k = p.kp + (int64_t)t.gi * p.kp_g + (int64_t)tile * kShTile * HS;
    t.v = p.vp + (int64_t)t.gi * p.vp_g + (int64_t)tile * kShTile * HS;
    t.valid = min(kShTile, plen - tile * kShTile);
  }
  __device__ __forceinline__ Tile find(int index) const {
    Tile t;
    t.index = index;
    if (index < s.own) {
      const int each = p.n_groups * p.head_tiles;
      int lo = 0, hi = threads;      // the run whose rows hold it
      while (hi - lo > 1) {
        const int mid = (lo + hi) / 2;
        if (sums[mid] * each <= index) lo = mid; else hi = mid;
      }
      int rest = index - sums[lo] * each;
      int b = lo * run, at = mine(b);
      for (;;) {                     // (one row a run unless the batch is large)
        const int here = (at + kShTile) / kShTile * each;
        if (rest < here) break;
        rest -= here;
        at = mine(++b);
      }
      const int tiles = at / kShTile + 1, item = rest / tiles;
      t.b = b;
      t.gi = item / p.head_tiles;
      t.part = item - t.gi * p.head_tiles;
      own_item(t, at, rest - item * tiles);
    } else {
      const int rest = index - s.own, item = rest / s.prefix;
      t.b = 0;
      t.gi = item / p.row_tiles;
      t.part = item - t.gi * p.row_tiles;
      t.at = 0;
      prefix_item(t, rest - item * s.prefix);
    }
    return t;
  }
  // the tile behind it (there is one)
  __device__ __forceinline__ void next(Tile& t) const {
    ++t.index;
    if (t.left > 0) {
      --t.left;
      t.k += kShTile * HS;
      t.v += kShTile * HS;
      if (t.own) {
        const int done = t.at / kShTile - t.left;
        t.valid = min(kShTile, t.at + 1 - done * kShTile);
      } else {
        t.valid = min(kShTile, plen - (s.prefix - 1 - t.left) * kShTile);
      }
      return;
    }
    if (t.index == s.own) {
      t.gi = t.part = 0;
      prefix_item(t, 0);
    } else if (t.own) {
      int at = t.at;
      if (++t.part == p.head_tiles) {
        t.part = 0;
        if (++t.gi == p.n_groups) {
          t.gi = 0;
          do at = mine(++t.b); while (at < 0);
        }
      }
      own_item(t, at, 0);
    } else {
      if (++t.part == p.row_tiles) { t.part = 0; ++t.gi; }
      prefix_item(t, 0);
    }
  }
  __device__ __forceinline__ int64_t query_row(const Tile& t) const {
    return (int64_t)t.gi * p.batch * p.per + (t.own ? (int64_t)t.b * p.per + t.part * 16 : (int64_t)t.part * 8 * NP);
  }
  __device__ __forceinline__ int queries(const Tile& t) const { return t.own ? min(16, p.per - t.part * 16) : min(8 * NP, p.batch * p.per - t.part * 8 * NP); }
  __device__ __forceinline__ int tiles(const Tile& t) const { return t.own ? t.at / kShTile + 1 : s.prefix; }
  __device__ __forceinline__ int64_t item(const Tile& t) const {   // own items count with rows that take no part
    return t.own ? ((int64_t)t.b * p.n_groups + t.gi) * p.head_tiles + t.part : (int64_t)t.gi * p.row_tiles + t.part;
  }
};

// O^T: dimensions 16 i + g and 16 i + g + 8 of queries 8 t + 2 tq and 8 t + 2 tq + 1 (g = lane / 4, tq = lane % 4), and those queries' maxima and this lane's part of their sums
template <int HS, int NQ>
struct Sums {
  float o[HS / 16][NQ][4], m[NQ][2], l[NQ][2];
};

__device__ __forceinline__ uint32_t transposed(uint32_t v) {   // an 8 x 8 matrix of 16-bit numbers over a warp
  uint32_t r;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
  return r;
}

// 8 N queries, from row q0 of `q` on, and a tile of keys: S^T = K Q^T and O^T += V^T P^T, keys and dimensions as the rows of the products, so that few queries cost few of them.  `vb` of the
// values is what `values` gives, which waits for them.
template <int HS, int NQ, int N, typename Values>
__device__ __forceinline__ void attend_tile(Sums<HS, NQ>& a, uint32_t q, int q0, uint32_t kb, int valid, float scale_log2, int lane, Values values) {
  const int g = lane >> 2;
  float s[kShTile / 16][N][4];
#pragma unroll
  for (int i = 0; i < kShTile / 16; ++i)
#pragma unroll
    for (int t = 0; t < N; ++t) s[i][t][0] = s[i][t][1] = s[i][t][2] = s[i][t][3] = 0.f;
#pragma unroll
  for (int kp = 0; kp < HS / 32; ++kp) {
    uint32_t qf[N][4];
#pragma unroll
    for (int t = 0; t < N; ++t) ldsm_x4(qf[t], q + sw<HS>(q0 + t * 8 + (lane & 7), kp * 4 + (lane >> 3)));
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int i = 0; i < kShTile / 16; ++i) {
        uint32_t kf[4];
        ldsm_x4(kf, kb + sw<HS>(i * 16 + (lane & 15), kp * 4 + h * 2 + (lane >> 4)));
#pragma unroll
        for (int t = 0; t < N; ++t) pf_mma(s[i][t], kf, qf[t][2 * h], qf[t][2 * h + 1]);
      }
  }
  uint32_t hi[kShTile / 16][N][2], lo[kShTile / 16][N][2];
#pragma unroll
  for (int t = 0; t < N; ++t) {
    float top[2] = {a.m[t][0], a.m[t][1]}, org[2];
#pragma unroll
    for (int i = 0; i < kShTile / 16; ++i)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        s[i][t][e] = i * 16 + (e >> 1) * 8 + g < valid ? s[i][t][e] * scale_log2 : -INFINITY;
        top[e & 1] = fmaxf(top[e & 1], s[i][t][e]);
      }
#pragma unroll
    for (int c = 0; c < 2; ++c) {
#pragma unroll
      for (int o = 4; o < 32; o <<= 1) top[c] = fmaxf(top[c], __shfl_xor_sync(0xffffffffu, top[c], o));
      org[c] = top[c] == -INFINITY ? 0.f : top[c];   // (scores that are all -inf: weights of zero)
      const float shrink = ex2(a.m[t][c] - org[c]);
      a.m[t][c] = top[c];
      a.l[t][c] *= shrink;
#pragma unroll
      for (int i = 0; i < HS / 16; ++i) { a.o[i][t][c] *= shrink; a.o[i][t][2 + c] *= shrink; }
    }
#pragma unroll
    for (int i = 0; i < kShTile / 16; ++i)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const float x = ex2(s[i][t][2 * h] - org[0]), y = ex2(s[i][t][2 * h + 1] - org[1]);
        a.l[t][0] += x;
        a.l[t][1] += y;
        const uint32_t w = __byte_perm(__float_as_uint(x), __float_as_uint(y), 0x7632);   // the leading 16 bits of both
        hi[i][t][h] = transposed(w);
        lo[i][t][h] = transposed(pack_bf16(fmaf(x, kAbove, -bf16lo(w)), fmaf(y, kAbove, -bf16hi(w))));
      }
  }
  const uint32_t vb = values();
#pragma unroll
  for (int i = 0; i < kShTile / 16; ++i) {
#pragma unroll
    for (int d = 0; d < HS / 16; ++d) {
      uint32_t vf[4];
      ldsm_x4_t(vf, vb + sw<HS>(i * 16 + ((lane >> 4) << 3) + (lane & 7), d * 2 + ((lane >> 3) & 1)));
#pragma unroll
      for (int t = 0; t < N; ++t) {
        pf_mma(a.o[d][t], vf, hi[i][t][0], hi[i][t][1]);
        pf_mma(a.o[d][t], vf, lo[i][t][0], lo[i][t][1]);
      }
    }
  }
}

// The first `valid` queries' results to a slot
template <int HS, int NQ>
__device__ __forceinline__ void store_sums(const Sums<HS, NQ>& a, float* acc, float2* ml, int valid, int lane) {
  const int g = lane >> 2, tq = lane & 3;
#pragma unroll
  for (int t = 0; t < NQ; ++t)
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      float l = a.l[t][c];
#pragma unroll
      for (int o = 4; o < 32; o <<= 1) l += __shfl_xor_sync(0xffffffffu, l, o);
      const int r = t * 8 + 2 * tq + c;
      if (r < valid) {
#pragma unroll
        for (int i = 0; i < HS / 16; ++i) {
          __stcg(acc + r * HS + i * 16 + g, a.o[i][t][c]);
          __stcg(acc + r * HS + i * 16 + 8 + g, a.o[i][t][2 + c]);
        }
        if (g == 0) __stcg(ml + r, make_float2(a.m[t][c], l));
      }
    }
}

template <int HS, int NP, int NO>
__global__ void __launch_bounds__(ShSmem<HS, NP>::kWarps * 32, 1) attn_shared_kernel(const SharedParams p) {
  using C = ShSmem<HS, NP>;
  constexpr int NQ = NP > NO ? NP : NO;
  constexpr int T = C::kWarps * 32, CH = HS / 8, RP = 32 / CH;   // 16-byte pieces of a row, rows a warp copies at once
  extern __shared__ __align__(128) uint8_t sh_smem[];
  __shared__ int s_sums[T + 1], s_mine[T], s_warp[C::kWarps];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  griddep_launch();
  const int plen = prefix_len(p);
  const Split s = make_split<T>(p, plen, s_sums, s_mine, s_warp);
  const int w = warp * (int)gridDim.x + (int)blockIdx.x;   // (workers beside each other on different SMs)
  // Where the prefix's own kernel ran in between, the turning kernel ended before that one let this one begin: then the wait is for that kernel, so that what comes next
  // finds both done; one CTA waits for all.
  const bool late = p.pre_parts > 0;
  if (w >= s.workers) {
    if (!late || blockIdx.x == gridDim.x - 1) griddep_wait();
    return;
  }
  const Walk<HS, NP> walk{p, s, s_sums, s_mine, plen, (p.batch + T - 1) / T, T};
  const uint32_t ring = pf_smem(sh_smem) + warp * C::kWarp, sq = ring + kShUnits * C::kUnit;

  auto load = [&](uint32_t dst, const __nv_bfloat16* src, int valid) {   // 32 rows, zeros from `valid` on: a weight of zero times whatever lies there must be zero
#pragma unroll
    for (int j = 0; j < kShTile / RP; ++j) {
      const int r = j * RP + lane / CH, c = lane % CH;
      const bool ok = r < valid;
      pf_cp16(dst + sw<HS>(r, c), src + (ok ? r * HS : 0) + c * 8, ok);
    }
  };
  auto load_queries = [&](uint32_t dst, const Tile& t) {
    const __nv_bfloat16* const src = p.q + walk.query_row(t) * HS;
    const int valid = walk.queries(t);
#pragma unroll
    for (int j = 0; j < 8 * NQ / RP; ++j) {
      const int r = j * RP + lane / CH, c = lane % CH;
      if (8 * NQ % RP && r >= 8 * NQ) break;
      const bool ok = r < valid;
      pf_cp16(dst + sw<HS>(r, c), src + (ok ? r * HS : 0) + c * 8, ok);
    }
  };
  const int first = first_tile(w, s), end = first_tile(w + 1, s);
  Tile cur = walk.find(first);
  Tile coming = cur;                                       // the tile behind it: its values are loaded next
  const bool two = cur.index + 1 < end;
  if (two) walk.next(coming);
  // What the turning kernel writes, queries and the newest own row, the last of an item's, is read behind the wait; everything else was there before.
  auto early = [&](bool now) {
    const bool c = now == (!cur.own || cur.left > 0), n = two && now == (!coming.own || coming.left > 0);
    if (c) {
      load(ring, cur.k, cur.valid);
      load(ring + C::kUnit, cur.v, cur.valid);
    }
    if (n) load(ring + 2 * C::kUnit, coming.k, coming.valid);
  };
  early(true);
  if (!late) griddep_wait();
  early(false);
  load_queries(sq, cur);
  int qb = 0, next_qb = 0;                                 // the query buffers of either
  if (two && cur.left == 0) load_queries(sq + (next_qb = 1) * C::kQ, coming);
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
    unit = unit == kShUnits - 1 ? 0 : unit + 1;
    const uint32_t vb = ring + unit * C::kUnit;
    unit = unit == kShUnits - 1 ? 0 : unit + 1;
    const bool more = cur.index + 1 < end;
    pf_wait<2>();
    __syncwarp();
    auto values = [&]() {
      __syncwarp();                                        // the keys have been read: the values of the next tile take their place
      if (more) load(kb, coming.v, coming.valid);
      pf_commit();
      pf_wait<2>();
      __syncwarp();
      return vb;
    };
    if (NP == NO || cur.own) attend_tile<HS, NQ, NO>(a, sq + qb * C::kQ, 0, kb, cur.valid, p.scale_log2, lane, values);
    else attend_tile<HS, NQ, NP>(a, sq + qb * C::kQ, 0, kb, cur.valid, p.scale_log2, lane, values);
    __syncwarp();                                          // the values have been read: the keys of the tile after the next take their place
    const bool ends = cur.left == 0 || !more;
    Tile was = cur;
    cur = coming;
    qb = next_qb;
    if (cur.index + 1 < end) {
      walk.next(coming);
      load(vb, coming.k, coming.valid);
      if (cur.left == 0) load_queries(sq + (next_qb = qb ^ 1) * C::kQ, coming);
    }
    pf_commit();
    if (ends) {
      // ---- the item, or this worker's part of it, ends ----
      const int64_t item = walk.item(was), slot = item + w;
      const int begun = walk.tiles(was) - 1 - was.left;   // the item's tiles before the last one here
      if (lane == 0 && was.index - begun >= first) {       // it began here: who joins its results learns where they are
        int2* const where = was.own ? p.own_where : p.pre_where;
        __stcg(where + item, make_int2(w, worker_of(was.index + was.left, s) - w + 1));
      }
      const int rows = was.own ? min(16, p.per) : 8 * NP;
      store_sums<HS, NQ>(a, (was.own ? p.own_acc : p.pre_acc) + slot * rows * HS, (was.own ? p.own_ml : p.pre_ml) + slot * rows, walk.queries(was), lane);
      if (!more) break;
      clear();
    }
  }
  pf_wait<0>();
  if (late && blockIdx.x == gridDim.x - 1) griddep_wait();
}

// Results first, first + step, .. of n, V numbers a lane, four on their way at a time; where(i): the i-th result's maximum and sum, and its numbers
template <int V, typename Where>
__device__ __forceinline__ void join_results(int first, int step, int n, int lane, float& top, float& sum, float (&a)[V], Where where) {
  for (int i0 = first; i0 < n; i0 += 4 * step) {
    float2 e[4];
    float v[4][V];
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const int i = i0 + u * step;
      e[u] = make_float2(-INFINITY, 0.f);
#pragma unroll
      for (int j = 0; j < V; ++j) v[u][j] = 0.f;
      if (i < n) {
        const float2* ml;
        const float* acc;
        where(i, ml, acc);
        e[u] = __ldcg(ml);
        if constexpr (V == 4) {
          const float4 x = __ldcg(reinterpret_cast<const float4*>(acc + lane * V));
          v[u][0] = x.x; v[u][1] = x.y; v[u][V - 2] = x.z; v[u][V - 1] = x.w;
        } else {
          const float2 x = __ldcg(reinterpret_cast<const float2*>(acc + lane * V));
          v[u][0] = x.x; v[u][1] = x.y;
        }
      }
    }
    float now = top;
#pragma unroll
    for (int u = 0; u < 4; ++u) now = fmaxf(now, e[u].x);
    const float org = now == -INFINITY ? 0.f : now, shrink = ex2(top - org);
    top = now;
    sum *= shrink;
#pragma unroll
    for (int j = 0; j < V; ++j) a[j] *= shrink;
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const float c = ex2(e[u].x - org);
      sum += e[u].y * c;
#pragma unroll
      for (int j = 0; j < V; ++j) a[j] += e[u].y == 0.f ? 0.f : v[u][j] * c;   // (a range that saw nothing has no result)
    }
  }
}

// What the next ways - 1 warps left in shared memory, to the first one's
template <int HS>
__device__ __forceinline__ void join_warps(const float* acc, const float2* ml, int ways, int lane, float& top, float& sum, float (&a)[HS / 32]) {
  constexpr int V = HS / 32;
  float now = top;
  for (int u = 1; u < ways; ++u) now = fmaxf(now, ml[u].x);
  const float org = now == -INFINITY ? 0.f : now, c0 = ex2(top - org);
  sum *= c0;
#pragma unroll
  for (int j = 0; j < V; ++j) a[j] *= c0;
  for (int u = 1; u < ways; ++u) {
    const float c = ex2(ml[u].x - org);
    sum += ml[u].y * c;
#pragma unroll
    for (int j = 0; j < V; ++j) a[j] += acc[u * HS + lane * V + j] * c;
  }
}
template <int HS>
__device__ __forceinline__ void store_result(__nv_bfloat16* out, const float (&a)[HS / 32], float inv, int lane) {
  constexpr int V = HS / 32;
  if constexpr (V == 4) *reinterpret_cast<uint2*>(out + lane * V) = make_uint2(pack_bf16(a[0] * inv, a[1] * inv), pack_bf16(a[V - 2] * inv, a[V - 1] * inv));
  else *reinterpret_cast<uint32_t*>(out + lane * V) = pack_bf16(a[0] * inv, a[1] * inv);
}

// A head's results joined: `ways` warps a head, HS / 32 numbers a lane.
template <int HS>
__global__ void __launch_bounds__(256) attn_shared_join_kernel(const SharedParams p) {
  constexpr int V = HS / 32;
  __shared__ float s_acc[8][HS];
  __shared__ float2 s_ml[8];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, heads = 8 / p.ways, blocks = (p.n_head + heads - 1) / heads;
  const int b = blockIdx.x / blocks, h = (blockIdx.x - b * blocks) * heads + warp / p.ways, way = warp % p.ways;
  griddep_launch();
  const bool idle = row_pos(p, b) < 0;
  const int gi = h / p.per, hh = h - gi * p.per, row = b * p.per + hh, own_rows = min(16, p.per);
  const int64_t own_item = ((int64_t)b * p.n_groups + gi) * p.head_tiles + hh / 16, pre_item = (int64_t)gi * p.row_tiles + row / p.tile_rows;
  int2 pre = make_int2(0, p.pre_parts);
  int64_t pre_at = 0;
  if (p.pre_parts) pre_at = ((int64_t)gi * p.pre_tiles + row / p.pre_rows) * p.pre_parts * p.pre_rows + row % p.pre_rows;
  const int pre_step = p.pre_parts ? p.pre_rows : p.tile_rows;
  const bool listed = p.row_tiles > 0 && prefix_len(p) > 0;   // the prefix is in the list of tiles
  griddep_wait();
  float top = -INFINITY, sum = 0.f, a[V] = {};
  if (h < p.n_head && !idle) {
    const int2 own = __ldcg(p.own_where + own_item);
    if (listed) {
      pre = __ldcg(p.pre_where + pre_item);
      pre_at = (pre_item + pre.x) * p.tile_rows + row % p.tile_rows;
    }
    const int64_t own_at = (own_item + own.x) * own_rows + hh % 16;
    const int own_n = own.y, n = own_n + pre.y;
    join_results<V>(way, p.ways, n, lane, top, sum, a, [&](int i, const float2*& ml, const float*& acc) {
      const bool mine = i < own_n;
      const int64_t at = mine ? own_at + (int64_t)i * own_rows : pre_at + (int64_t)(i - own_n) * pre_step;
      ml = (mine ? p.own_ml : p.pre_ml) + at;
      acc = (mine ? p.own_acc : p.pre_acc) + at * HS;
    });
  }
  if (p.ways > 1) {
#pragma unroll
    for (int j = 0; j < V; ++j) s_acc[warp][lane * V + j] = a[j];
    if (lane == 0) s_ml[warp] = make_float2(top, sum);
    __syncthreads();
    if (way != 0) return;
    join_warps<HS>(s_acc[warp], s_ml + warp, p.ways, lane, top, sum, a);
  }
  if (h < p.n_head) store_result<HS>(p.out + ((int64_t)b * p.n_head + h) * HS, a, idle ? 0.f : 1.f / sum, lane);
}

// ---- few query rows a group: the step of a group by a cluster, in one launch ----
// The three launches above wait for one another, which is most of a short step's time.  Here each CTA of a group's cluster turns the group's few queries and new keys itself, its
// warps share the group's key tiles with those of the others, and behind the cluster's barrier they join the results.
constexpr int kClHeads = 32;   // heads that a CTA turns, queries, keys and values of all rows
constexpr int kClCtas = 8;

template <int HS, int NP>
struct ClSmem {
  static constexpr int kUnit = kShTile * HS * 2, kWarps = HS == 64 ? 12 : 7, kQRows = 16 * NP, kNew = kClHeads / 3;
  static constexpr int kQ = kWarps * kShUnits * kUnit, kNewKeys = kQ + kQRows * HS * 2, kNewValues = kNewKeys + kNew * HS * 2, kBytes = kNewValues + kNew * HS * 2;
};

template <int HS, int NP>
__global__ void __launch_bounds__(ClSmem<HS, NP>::kWarps * 32, 1) attn_shared_cluster_kernel(const SharedParams p, int ctas) {
  using C = ClSmem<HS, NP>;
  constexpr int W = C::kWarps, V = HS / 32, CH = HS / 8, RP = 32 / CH;
  extern __shared__ __align__(128) uint8_t sh_smem[];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, gi = blockIdx.x / ctas, rank = blockIdx.x - gi * ctas;
  const uint32_t smem = pf_smem(sh_smem), ring = smem + warp * kShUnits * C::kUnit, sq = smem + C::kQ;
  griddep_wait();
  griddep_launch();
  // lane b: row b's newest own key, the first of its tiles
  const int plen = prefix_len(p), rows = p.batch * p.per;
  const int64_t pos_of = lane < p.batch ? row_pos(p, lane) : -1;
  const int at = own_index(p, pos_of, plen), here = (at + kShTile) / kShTile;
  int inc = here;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) { const int t = __shfl_up_sync(0xffffffffu, inc, o); if (lane >= o) inc += t; }
  const int first = inc - here;
  Split s;
  s.own = __shfl_sync(0xffffffffu, inc, 31);
  s.prefix = (plen + kShTile - 1) / kShTile;
  s.all = s.own + s.prefix;
  s.workers = min(s.all, ctas * W);
  s.each = s.workers ? s.all / s.workers : 0;
  s.more = s.all - s.each * s.workers;
  const int w = warp * ctas + rank;
  const int begin = w < s.workers ? first_tile(w, s) : s.all, end = w < s.workers ? first_tile(w + 1, s) : s.all;

  struct Place { const __nv_bfloat16* k; const __nv_bfloat16* v; int stored, valid, own, b, last; };   // stored: rows that lie in the cache already; the newest one comes behind them
  auto find = [&](int t) {
    Place x;
    x.own = t < s.own;
    if (x.own) {
      x.b = __popc(__ballot_sync(0xffffffffu, lane < p.batch && first <= t)) - 1;
      const int newest = __shfl_sync(0xffffffffu, at, x.b), tile = t - __shfl_sync(0xffffffffu, first, x.b);
      x.k = p.kc + (int64_t)x.b * p.kc_b + (int64_t)gi * p.kc_g + (int64_t)tile * kShTile * HS;
      x.v = p.vc + (int64_t)x.b * p.vc_b + (int64_t)gi * p.vc_g + (int64_t)tile * kShTile * HS;
      x.last = tile == newest / kShTile;
      x.stored = x.last ? newest % kShTile : kShTile;
      x.valid = x.stored + x.last;
    } else {
      const int tile = t - s.own;
      x.b = 0;
      x.k = p.kp + (int64_t)gi * p.kp_g + (int64_t)tile * kShTile * HS;
      x.v = p.vp + (int64_t)gi * p.vp_g + (int64_t)tile * kShTile * HS;
      x.last = tile == s.prefix - 1;
      x.stored = x.valid = min(kShTile, plen - tile * kShTile);
    }
    return x;
  };
  auto load = [&](uint32_t dst, const __nv_bfloat16* src, int valid) {   // zeros from `valid` on
#pragma unroll
    for (int j = 0; j < kShTile / RP; ++j) {
      const int r = j * RP + lane / CH, c = lane % CH;
      const bool ok = r < valid;
      pf_cp16(dst + sw<HS>(r, c), src + (ok ? r * HS : 0) + c * 8, ok);
    }
  };
  Place cur = {}, coming = {};
  if (begin < end) {
    cur = find(begin);
    load(ring, cur.k, cur.stored);
    pf_commit();
    load(ring + C::kUnit, cur.v, cur.stored);
    pf_commit();
    if (begin + 1 < end) {
      coming = find(begin + 1);
      load(ring + 2 * C::kUnit, coming.k, coming.stored);
    }
    pf_commit();
  }

  // ---- the group's queries, keys and values of this step ----
  auto put = [&](uint32_t dst, const uint32_t (&v)[HS / 64]) {
    if constexpr (V == 4) asm volatile("st.shared.v2.u32 [%0], {%1, %2};" ::"r"(dst), "r"(v[0]), "r"(v[V / 2 - 1]) : "memory");
    else asm volatile("st.shared.u32 [%0], %1;" ::"r"(dst), "r"(v[0]) : "memory");
  };
  auto row_of = [&](uint32_t base, int r) { return base + sw<HS>(r, lane * V * 2 / 16) + lane * V * 2 % 16; };
  const int heads = p.batch * (p.per + 2);
#pragma unroll 1
  for (int i = warp; i < heads; i += W) {
    const int b = i / (p.per + 2), h = i - b * (p.per + 2), mine = __shfl_sync(0xffffffffu, at, b);
    const int64_t pos = __shfl_sync(0xffffffffu, pos_of, b);
    const __nv_bfloat16* const x = p.qkv + (((int64_t)b * p.n_groups + gi) * (p.per + 2) + h) * HS;
    uint32_t v[HS / 64];
    if (h <= p.per) {
      turned_part<HS>(p, x, table_row(p, b, pos), lane, v);
    } else {
      const uint16_t* const n = reinterpret_cast<const uint16_t*>(x + lane * V);
#pragma unroll
      for (int j = 0; j < V / 2; ++j) v[j] = (uint32_t)n[2 * j] | ((uint32_t)n[2 * j + 1] << 16);
    }
    if (h < p.per) {
      if (pos < 0)
#pragma unroll
        for (int j = 0; j < V / 2; ++j) v[j] = 0u;
      put(row_of(sq, b * p.per + h), v);
    } else {
      put(smem + (h == p.per ? C::kNewKeys : C::kNewValues) + (b * HS + lane * V) * 2, v);
      if (rank == 0 && mine >= 0) {
        __nv_bfloat16* const to = (h == p.per ? p.kc + (int64_t)b * p.kc_b + (int64_t)gi * p.kc_g : p.vc + (int64_t)b * p.vc_b + (int64_t)gi * p.vc_g) + (int64_t)mine * HS + lane * V;
        if constexpr (V == 4) *reinterpret_cast<uint2*>(to) = make_uint2(v[0], v[V / 2 - 1]);
        else *reinterpret_cast<uint32_t*>(to) = v[0];
      }
    }
  }
  for (int r = rows + warp; r < C::kQRows; r += W) {
    const uint32_t none[HS / 64] = {};
    put(row_of(sq, r), none);
  }
  __syncthreads();

  // ---- the key tiles ----
  const int own_rows = p.per, slots = p.batch + p.workers;   // (workers: the most of a cluster)
  if (begin < end) {
    auto newest = [&](uint32_t unit, uint32_t news) {   // the row that the caches do not hold yet
      if (cur.own && cur.last) {
        uint32_t v[HS / 64];
        const uint32_t src = smem + news + (cur.b * HS + lane * V) * 2;
        if constexpr (V == 4) asm volatile("ld.shared.v2.u32 {%0, %1}, [%2];" : "=r"(v[0]), "=r"(v[V / 2 - 1]) : "r"(src) : "memory");
        else asm volatile("ld.shared.u32 %0, [%1];" : "=r"(v[0]) : "r"(src) : "memory");
        put(row_of(unit, cur.stored), v);
      }
      __syncwarp();
    };
    Sums<HS, NP> a;
    auto clear = [&]() {
#pragma unroll
      for (int t = 0; t < NP; ++t) {
#pragma unroll
        for (int i = 0; i < HS / 16; ++i) a.o[i][t][0] = a.o[i][t][1] = a.o[i][t][2] = a.o[i][t][3] = 0.f;
        a.m[t][0] = a.m[t][1] = -INFINITY;
        a.l[t][0] = a.l[t][1] = 0.f;
      }
    };
    clear();
    int unit = 0;                                          // of the current tile's keys
    for (int t = begin;; ++t) {
      const uint32_t kb = ring + unit * C::kUnit;
      unit = unit == kShUnits - 1 ? 0 : unit + 1;
      const uint32_t vb = ring + unit * C::kUnit;
      unit = unit == kShUnits - 1 ? 0 : unit + 1;
      const bool more = t + 1 < end;
      pf_wait<2>();
      __syncwarp();
      newest(kb, C::kNewKeys);
      auto values = [&]() {
        __syncwarp();                                      // the keys have been read: the values of the next tile take their place
        if (more) load(kb, coming.v, coming.stored);
        pf_commit();
        pf_wait<2>();
        __syncwarp();
        newest(vb, C::kNewValues);
        return vb;
      };
      attend_tile<HS, NP, NP>(a, sq, cur.own ? cur.b * p.per : 0, kb, cur.valid, p.scale_log2, lane, values);   // (own keys with as many columns: the code of fewer is fetched, too)
      __syncwarp();                                        // the values have been read: the keys of the tile after the next take their place
      const bool ends = cur.last || !more;
      const int own = cur.own, b = cur.b;
      cur = coming;
      if (t + 2 < end) {
        coming = find(t + 2);
        load(vb, coming.k, coming.stored);
      }
      pf_commit();
      if (ends) {
        const int64_t slot = own ? (int64_t)gi * slots + b + w : (int64_t)gi * p.workers + w;
        const int size = own ? own_rows : 8 * NP;
        store_sums<HS, NP>(a, (own ? p.own_acc : p.pre_acc) + slot * size * HS, (own ? p.own_ml : p.pre_ml) + slot * size, own ? p.per : rows, lane);
        if (!more) break;
        clear();
      }
    }
    pf_wait<0>();
  }
  asm volatile("barrier.cluster.arrive.release;\n\tbarrier.cluster.wait.acquire;" ::: "memory");

  // ---- the results joined: heads in turn to the CTAs, there as many warps a head as there are for it ----
  const int joined = (rows + ctas - 1) / ctas, ways = joined < W ? W / joined : 1, once = W / ways, way = warp % ways;
  float* const s_acc = reinterpret_cast<float*>(sh_smem) + warp * HS;      // (over the ring, which nothing reads any more)
  float2* const s_ml = reinterpret_cast<float2*>(sh_smem + W * HS * sizeof(float)) + warp;
  for (int h0 = 0; h0 < joined; h0 += once) {
    const int r = rank + ctas * (h0 + warp / ways);
    const bool here = warp / ways < once && r < rows;
    const int b = here ? r / p.per : 0, newest = __shfl_sync(0xffffffffu, at, b), t0 = __shfl_sync(0xffffffffu, first, b);
    float top = -INFINITY, sum = 0.f, a[V] = {};
    if (here && newest >= 0) {
      const int own_w = worker_of(t0, s), own_n = worker_of(t0 + newest / kShTile, s) - own_w + 1;
      const int pre_w = s.prefix ? worker_of(s.own, s) : 0, n = own_n + (s.prefix ? worker_of(s.all - 1, s) - pre_w + 1 : 0);
      const int64_t own_at = ((int64_t)gi * slots + b + own_w) * own_rows + r - b * p.per, pre_at = ((int64_t)gi * p.workers + pre_w) * 8 * NP + r;
      join_results<V>(way, ways, n, lane, top, sum, a, [&](int i, const float2*& ml, const float*& acc) {
        const bool mine = i < own_n;
        const int64_t at = mine ? own_at + (int64_t)i * own_rows : pre_at + (int64_t)(i - own_n) * 8 * NP;
        ml = (mine ? p.own_ml : p.pre_ml) + at;
        acc = (mine ? p.own_acc : p.pre_acc) + at * HS;
      });
    }
    if (ways > 1) {
#pragma unroll
      for (int j = 0; j < V; ++j) s_acc[lane * V + j] = a[j];
      if (lane == 0) *s_ml = make_float2(top, sum);
      __syncthreads();
      if (here && way == 0) {
        join_warps<HS>(s_acc, s_ml, ways, lane, top, sum, a);
      }
    }
    if (here && way == 0) store_result<HS>(p.out + ((int64_t)b * p.n_head + gi * p.per + r - b * p.per) * HS, a, newest < 0 ? 0.f : 1.f / sum, lane);
  }
}

std::atomic<int> g_shared_path{0};   // b200_attn_decode_shared_tune

struct SharedPlan {
  int np, no, head_tiles, row_tiles, ctas, workers, ways;   // np, no: eights of queries of a prefix's item and of an own one
  int64_t own_slots, pre_slots;   // rows
  int64_t own_items, pre_items;   // in the list of tiles
  int64_t tiles, q;               // tiles at most; numbers of the turned queries
  size_t bytes;
  bool tensor, pair;              // the prefix on the tensor memory; 256 query rows a CTA instead of 128
  int splits;                     // its key ranges
  int pre_rows, pre_tiles, pre_parts;
  bool cluster;                   // a cluster a group, in one launch
};

// Whether a group's step goes to a cluster: it saves two launches, but a cluster's few CTAs turn all of the group's heads each, and have a group's tiles to themselves while
// others' SMs idle.  us of list and cluster, in a graph (call after call a cluster is 5 us of the host shorter):
//   rows x groups x heads of 128 each, prefix 96 to 200, 500, 1500, 2500 to 4000:  1 x 32 x 1  9.6 10.2 12.9 16.3, 8.1 8.4 11.9 15.1;  4 x 32 x 1  10.7 10.7 13.8 16.8, 8.3 9.3 13.6 16.4;
//   2 x 8 x 4  8.7 10.0 10.6 12.5, 7.9 8.7 9.6 12.8;  4 x 8 x 2  8.6 10.2 10.6 12.7, 7.9 9.2 10.1 12.9;  8 x 32 x 1  10.8 11.3 14.6 17.7, 10.0 12.0 16.5 18.8;
//   5 x 8 x 4 over 100 10.9, 14.3;  4 x 2 x 4 over 8000 15.4, 20.2;  of 64: 7 x 12 x 1 over 1001 11.0, 8.7;  8 x 24 x 2 over 300 11.6, 9.7
// So: no more than 16 heads of 128 or 32 of 64 to turn, and at most 1.25 tiles a warp more than in the list (own caches half full).
// The plan goes by prefix_rows, what the buffer has room for, since the length is on the device; these times and those at shared_plan are of prefixes that fill it.  In a buffer
// of 8192, rows x groups x heads over 500 and 2000 keys:  2 x 32 x 1  10.0 14.8 (filled 7.9 13.5);  16 x 32 x 1  15.0 19.9 (15.2 20.0);  16 x 8 x 4  19.0 22.7 (16.2 18.6);
// 64 x 8 x 4  26.8 28.0 (22.3 26.8).
bool few_rows(int batch, int n_groups, int per, int hs, int prefix_rows, int own_rows) {
  if (batch * (per + 2) * hs > 2048) return false;
  const int sms = sm_count(), ctas = sms / n_groups < 1 ? 1 : sms / n_groups < kClCtas ? sms / n_groups : kClCtas;
  const double tiles = (prefix_rows + 0.5 * batch * own_rows) / kShTile, warps = hs == 64 ? ClSmem<64, 1>::kWarps : ClSmem<128, 1>::kWarps;
  return tiles * (1.0 / ctas - (double)n_groups / sms) <= 1.25 * warps;
}

SharedPlan shared_plan(int batch, int n_groups, int per, int hs, int prefix_rows, int own_rows) {
  SharedPlan s;
  const int64_t rows = (int64_t)batch * per;
  // The prefix on the tensor memory from so much work on: its kernel reads a key once for 256 rows, the list once for 32, but it is a launch more.  List and tensor memory, us:
  // 48 rows of 8 groups x 2048 16.5, 19.5; 32 rows of 32 groups x 2048 26.3, 29.9; 24 rows of 8 groups x 8000 23.4, 23.5; 64 x 8000 34.1, 30.4; 32 x 16000 33.1, 29.2;
  // up to 16 rows a tile of the list has no more products than eights: 16 rows of 8 groups x 8000 20.0, 22.3.
  const int path = g_shared_path.load(std::memory_order_relaxed);
  s.cluster = per <= 16 && (int64_t)batch * (per + 2) <= kClHeads && (path == 3 || (path == 0 && few_rows(batch, n_groups, per, hs, prefix_rows, own_rows)));
  if (s.cluster) {
    s.np = rows > 16 ? 4 : rows > 8 ? 2 : 1;
    s.no = per > 8 ? 2 : 1;
    s.tensor = s.pair = false;
    s.splits = s.pre_rows = s.pre_tiles = s.pre_parts = s.head_tiles = s.row_tiles = s.ctas = 0;
    s.ways = 1;
    s.q = s.own_items = s.pre_items = 0;
    const int64_t tiles = (int64_t)batch * ((own_rows + kShTile - 1) / kShTile) + (prefix_rows + kShTile - 1) / kShTile;
    const int warps = hs == 64 ? ClSmem<64, 1>::kWarps : ClSmem<128, 1>::kWarps;
    s.tiles = tiles * n_groups;
    s.workers = kClCtas * warps < tiles ? kClCtas * warps : (int)tiles;
    s.own_slots = (int64_t)n_groups * (batch + s.workers) * per;
    s.pre_slots = prefix_rows > 0 ? (int64_t)n_groups * s.workers * 8 * s.np : 0;
    s.bytes = (size_t)(s.own_slots + s.pre_slots) * (hs + 2) * sizeof(float);
    return s;
  }
  s.tensor = prefix_rows > 0 && (path ? path == 2 : rows > 16 && (int64_t)prefix_rows * n_groups * ((rows + 31) / 32) > 100000);
  s.pair = rows > 128;
  s.splits = s.pre_rows = s.pre_tiles = s.pre_parts = 0;
  if (s.tensor) {
    s.pre_rows = s.pair ? 256 : 128;
    s.pre_tiles = (int)((rows + s.pre_rows - 1) / s.pre_rows);
    const int64_t items = (int64_t)n_groups * s.pre_tiles, ranges = ((int64_t)prefix_rows + 127) / 128;
    // SMs for the prefix's kernel: the kernel of the own keys begins beside it on the others, so each has the share of SMs that its work asks for (own caches half full): a tile
    // of 128 keys takes 2.15 us with 256 rows and 1.3 with 128, own keys come at 58 GB/s an SM.  64 rows x 16001 in 8 groups of 4 heads, up to 1000 own tokens, in 6, 9, 12, 18
    // ranges 69, 54, 55, 64 us; 10 own tokens 63, 50, 43, 46; 4000 shared and up to 1000 own ones 42, 43, 47, 51 (3 ranges 46).  (All of heads of 128; a tile of heads of 64,
    // half as large, is counted as much.)
    const double prefix_work = (double)items * ranges * (s.pair ? 2.15 : 1.3), own_work = (double)batch * n_groups * own_rows * hs * 2 / 58e3;
    const double share = sm_count() * prefix_work / (prefix_work + own_work) / items;
    s.splits = share < 1.0 ? 1 : share < (double)ranges ? (int)(share + 0.5) : (int)ranges;
    while (s.splits > 1 && s.splits * items > sm_count()) --s.splits;
    s.pre_parts = s.pair ? s.splits : 2 * s.splits;
    prefix_rows = 0;               // not in the list of tiles
  }
  s.no = per > 8 ? 2 : 1;
  s.np = prefix_rows == 0 ? s.no : rows > 16 ? 4 : rows > 8 ? 2 : 1;
  s.head_tiles = (per + 15) / 16;
  s.row_tiles = prefix_rows > 0 ? (int)((rows + 8 * s.np - 1) / (8 * s.np)) : 0;
  const int64_t own_items = (int64_t)batch * n_groups * s.head_tiles, pre_items = (int64_t)n_groups * s.row_tiles;
  const int64_t tiles = own_items * ((own_rows + kShTile - 1) / kShTile) + pre_items * ((prefix_rows + kShTile - 1) / kShTile);
  const int warps = hs == 64 ? (s.np == 4 ? ShSmem<64, 4>::kWarps : ShSmem<64, 1>::kWarps) : (s.np == 4 ? ShSmem<128, 4>::kWarps : ShSmem<128, 1>::kWarps);
  s.tiles = tiles;
  // a CTA an SM; beside the prefix's own kernel, which leaves SMs one by one, two shorter ones
  s.ctas = sm_count() * (s.tensor ? 2 : 1);
  if (s.ctas > tiles) s.ctas = (int)tiles;
  s.workers = s.ctas * warps < tiles ? s.ctas * warps : (int)tiles;
  s.own_slots = (own_items + s.workers) * (per < 16 ? per : 16);
  s.pre_slots = prefix_rows > 0 ? (pre_items + s.workers) * 8 * s.np : (int64_t)n_groups * s.pre_tiles * s.pre_parts * s.pre_rows;
  s.q = rows * n_groups * hs;
  s.own_items = own_items;
  s.pre_items = pre_items;
  s.bytes = (size_t)(s.own_slots + s.pre_slots) * (hs + 2) * sizeof(float) + (size_t)s.q * 2 + (size_t)(own_items + pre_items) * sizeof(int2);
  // results of a head: about those of a prefix item and of an own one
  const int64_t results = 2 + s.pre_parts + (int64_t)s.workers / (pre_items > 0 ? pre_items : own_items);
  s.ways = 1;                      // four results a warp are one round; no more warps than the GPU has at once
  while (s.ways < 8 && results > 4 * s.ways && (int64_t)batch * n_groups * per * s.ways < 24 * sm_count()) s.ways *= 2;
  return s;
}

template <int HS, int NP, int NO>
cudaError_t launch_tiles(const SharedParams& p, const SharedPlan& s, cudaStream_t st) {
  using C = ShSmem<HS, NP>;
  static PerDeviceOnce once;
  if (once.need()) {
    const cudaError_t e = cudaFuncSetAttribute(attn_shared_kernel<HS, NP, NO>, cudaFuncAttributeMaxDynamicSharedMemorySize, C::kBytes);
    if (e != cudaSuccess) return e;
    once.done();
  }
  return launch(attn_shared_kernel<HS, NP, NO>, dim3((unsigned)s.ctas), dim3(C::kWarps * 32), (size_t)C::kBytes, st, p);
}

// As many CTAs a cluster as let all groups' clusters run at once, no more than there are tiles for their warps.
template <int HS, int NP>
cudaError_t launch_clusters(const SharedParams& p, const SharedPlan& s, cudaStream_t st) {
  using C = ClSmem<HS, NP>;
  static std::atomic<int> known[64][kClCtas + 1];   // clusters at once
  static PerDeviceOnce once;
  if (once.need()) {
    const cudaError_t e = cudaFuncSetAttribute(attn_shared_cluster_kernel<HS, NP>, cudaFuncAttributeMaxDynamicSharedMemorySize, C::kBytes);
    if (e != cudaSuccess) return e;
    once.done();
  }
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) dev = 0;
  int ctas = (s.workers + C::kWarps - 1) / C::kWarps;
  for (; ctas > 1; --ctas) {
    if (ctas * p.n_groups > p.sms) continue;
    std::atomic<int>& n = known[dev & 63][ctas];
    int have = n.load(std::memory_order_relaxed);
    if (have == 0) {
      cudaLaunchConfig_t cfg = {};
      cfg.gridDim = dim3((unsigned)ctas);
      cfg.blockDim = dim3(C::kWarps * 32);
      cfg.dynamicSmemBytes = C::kBytes;
      cudaLaunchAttribute attr[1];
      attr[0].id = cudaLaunchAttributeClusterDimension;
      attr[0].val.clusterDim.x = (unsigned)ctas;
      attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
      cfg.attrs = attr;
      cfg.numAttrs = 1;
      if (cudaOccupancyMaxActiveClusters(&have, attn_shared_cluster_kernel<HS, NP>, &cfg) != cudaSuccess || have <= 0) {
        (void)cudaGetLastError();
        have = 1;
      }
      n.store(have, std::memory_order_relaxed);
    }
    if (have >= p.n_groups) break;
  }
  return launch_cluster(attn_shared_cluster_kernel<HS, NP>, dim3((unsigned)(p.n_groups * ctas)), dim3(C::kWarps * 32), ctas, (size_t)C::kBytes, st, p, ctas);
}

template <int HS>
cudaError_t launch_shared(const SharedParams& p, const SharedPlan& s, cudaStream_t st) {
  if (s.cluster) {
    return s.np == 4 ? launch_clusters<HS, 4>(p, s, st) : s.np == 2 ? launch_clusters<HS, 2>(p, s, st) : launch_clusters<HS, 1>(p, s, st);
  }
  const int64_t warps = (int64_t)p.batch * p.n_groups * (p.per + 2);
  cudaError_t e = launch(attn_shared_turn_kernel<HS>, dim3((unsigned)((warps + 7) / 8)), dim3(256), 0, st, p);
  if (e != cudaSuccess) return e;
  if (s.tensor && (e = launch_attn_shared_prefix(p, HS, s.pair, s.splits, st)) != cudaSuccess) return e;
  if (s.np == 4) e = s.no == 2 ? launch_tiles<HS, 4, 2>(p, s, st) : launch_tiles<HS, 4, 1>(p, s, st);
  else if (s.np == 2) e = s.no == 2 ? launch_tiles<HS, 2, 2>(p, s, st) : launch_tiles<HS, 2, 1>(p, s, st);
  else e = launch_tiles<HS, 1, 1>(p, s, st);
  if (e != cudaSuccess) return e;
  const int heads = 8 / s.ways;
  return launch(attn_shared_join_kernel<HS>, dim3((unsigned)(p.batch * ((p.n_head + heads - 1) / heads))), dim3(256), 0, st, p);
}

}  // namespace
}  // namespace b200

using namespace b200;

extern "C" {

size_t b200_attn_decode_shared_workspace_bytes(int batch, int n_head, int n_groups, int head_size, int prefix_rows, int own_rows) {
  if (batch <= 0 || n_groups <= 0 || n_head <= 0 || n_head % n_groups || prefix_rows < 0 || own_rows <= 0 || (head_size != 64 && head_size != 128)) return 0;
  const SharedPlan s = shared_plan(batch, n_groups, n_head / n_groups, head_size, prefix_rows, own_rows);
  return s.bytes;
}

int b200_attn_decode_shared_tune(int path) { return g_shared_path.exchange(path >= 1 && path <= 3 ? path : 0); }

int b200_attn_decode_shared(const b200_attn_decode_shared_args* a, b200_stream_t stream) {
  B200_CHECK_ARG(a, "b200_attn_decode_shared: null argument");
  B200_CHECK_ARG(a->head_size == 64 || a->head_size == 128, "b200_attn_decode_shared: head size %d (64 or 128)", a->head_size);
  B200_CHECK_ARG(a->batch > 0 && a->n_groups > 0 && a->n_head > 0 && a->n_head % a->n_groups == 0, "b200_attn_decode_shared: bad batch %d, heads %d or groups %d", a->batch,
                 a->n_head, a->n_groups);
  B200_CHECK_ARG((int64_t)a->batch * a->n_head < (1 << 24), "b200_attn_decode_shared: %d rows of %d heads", a->batch, a->n_head);
  B200_CHECK_ARG(a->own_rows > 0 && a->prefix_rows >= 0 && a->own_rows < (1 << 30) && a->prefix_rows < (1 << 30), "b200_attn_decode_shared: bad cache lengths");
  B200_CHECK_ARG(a->qkv && a->pos && a->k_cache && a->v_cache && a->out && a->workspace, "b200_attn_decode_shared: null pointer");
  B200_CHECK_ARG(a->prefix_rows == 0 || (a->k_prefix && a->v_prefix), "b200_attn_decode_shared: null prefix");
  B200_CHECK_ARG(a->rope_n_elem >= 0 && a->rope_n_elem <= a->head_size && a->rope_n_elem % 2 == 0, "b200_attn_decode_shared: bad rope_n_elem %d", a->rope_n_elem);
  B200_CHECK_ARG(a->rope_n_elem == 0 || (a->cos && a->sin && a->table_rows > 0), "b200_attn_decode_shared: no tables");
  B200_CHECK_ARG(a->table_dtype == B200_F32 || a->table_dtype == B200_BF16, "b200_attn_decode_shared: tables must be fp32 or bf16");
  B200_CHECK_ARG(a->pos_count == 1 || a->pos_count == a->batch, "b200_attn_decode_shared: %d positions for %d rows", a->pos_count, a->batch);
  const uintptr_t at = (uintptr_t)a->k_cache | (uintptr_t)a->v_cache | (uintptr_t)a->k_prefix | (uintptr_t)a->v_prefix | (uintptr_t)a->workspace;
  const int64_t strides = a->k_batch_stride | a->k_group_stride | a->v_batch_stride | a->v_group_stride | a->k_prefix_stride | a->v_prefix_stride;
  B200_CHECK_ARG((at & 15) == 0 && (strides & 7) == 0 && ((uintptr_t)a->out & 7) == 0, "b200_attn_decode_shared: caches and prefix must lie on 16-byte boundaries");
  const SharedPlan s = shared_plan(a->batch, a->n_groups, a->n_head / a->n_groups, a->head_size, a->prefix_rows, a->own_rows);
  B200_CHECK_ARG(s.tiles < (1 << 30), "b200_attn_decode_shared: caches of too many keys");
  B200_CHECK_ARG(a->workspace_bytes >= s.bytes, "b200_attn_decode_shared: workspace too small");
  if (s.tensor) B200_CHECK_WAITS("b200_attn_decode_shared");
  SharedParams p = {};
  p.qkv = (const __nv_bfloat16*)a->qkv;
  p.cos = a->cos; p.sin = a->sin; p.table_bf16 = a->table_dtype == B200_BF16; p.table_rows = a->table_rows; p.table_presel = a->table_preselected; p.rope_n = a->rope_n_elem;
  p.pos = a->pos; p.pos64 = a->pos_is_int64; p.pos_each = a->pos_count > 1;
  p.plen = a->prefix_len; p.plen64 = a->prefix_len_is_int64;
  p.kc = (__nv_bfloat16*)a->k_cache; p.vc = (__nv_bfloat16*)a->v_cache;
  p.kc_b = a->k_batch_stride; p.kc_g = a->k_group_stride; p.vc_b = a->v_batch_stride; p.vc_g = a->v_group_stride;
  p.kp = (const __nv_bfloat16*)a->k_prefix; p.vp = (const __nv_bfloat16*)a->v_prefix; p.kp_g = a->k_prefix_stride; p.vp_g = a->v_prefix_stride;
  p.out = (__nv_bfloat16*)a->out;
  p.batch = a->batch; p.n_head = a->n_head; p.n_groups = a->n_groups; p.per = a->n_head / a->n_groups; p.own_rows = a->own_rows; p.prefix_rows = a->prefix_rows;
  p.head_tiles = s.head_tiles; p.row_tiles = s.row_tiles; p.tile_rows = 8 * s.np; p.workers = s.workers; p.sms = sm_count(); p.ways = s.ways;
  p.pre_parts = s.pre_parts; p.pre_rows = s.pre_rows; p.pre_tiles = s.pre_tiles;
  const int n = a->rope_n_elem, part = a->head_size / 32;
  p.wide = ((uintptr_t)a->qkv & 15) == 0 && n % (2 * part) == 0 && (a->table_dtype == B200_BF16 || (((uintptr_t)a->cos | (uintptr_t)a->sin) & 15) == 0);
  // (every part of wide accesses begins on a 16-byte boundary: they come first)
  p.q = (__nv_bfloat16*)a->workspace;
  p.own_acc = (float*)(p.q + s.q);
  p.pre_acc = p.own_acc + s.own_slots * a->head_size;
  p.own_ml = (float2*)(p.pre_acc + s.pre_slots * a->head_size);
  p.pre_ml = p.own_ml + s.own_slots;
  p.own_where = (int2*)(p.pre_ml + s.pre_slots);
  p.pre_where = p.own_where + s.own_items;
  p.scale_log2 = 1.4426950408889634f / sqrtf((float)a->head_size);
  const cudaStream_t st = (cudaStream_t)stream;
  B200_CUDA((a->head_size == 128 ? launch_shared<128>(p, s, st) : launch_shared<64>(p, s, st)));
  return B200_OK;
}

}  // extern "C"
