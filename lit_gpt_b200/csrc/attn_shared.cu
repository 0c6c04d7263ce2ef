// One decode step (T = 1) of B rows that share a prefix: rotation of q and of the new k, append of the new k / v to the row's own cache, and
//   o = sum_j softmax_j(q . k_j / sqrt(hs)) v_j   over the prefix's keys [0, P) and the row's own keys [0, pos - P].
// The rounding points are those of the model's step (attn_decode.cu; lit_gpt/model.py:624-653, 767-773): q and k are bf16 after the rotation, the softmax is
// fp32 with a running maximum, the result is rounded once.
//
// The prefix is read once for all rows: the B * (heads per group) query rows of a key-value group are the left operand of its products, a key tile serves them all.
// Launch 1 computes partial results (maximum, sum, unscaled output) of key ranges, of the prefix for 16 * MT rows of a group and of a row's own keys for
// its heads of a group; launch 2 joins a row's partial results.  Both kinds of range run side by side in launch 1, so the step has no third launch, and neither has a
// counter that two calls at a time could share.
//
// A CTA has four warps; warp w takes the key tiles w, w + 4, .. of the CTA's range, double-buffered in its own shared-memory stages by cp.async.  S = Q K^T and
// O += P V on mma.sync.m16n8k16.  P enters as two bf16 numbers, its leading bits and the rest, so that its rounding does not add to the result's own (with the nearest
// bf16 number alone the error against 64 bits is a fifth larger than that of the final rounding).  The rest is kept above zero, so that an infinite value
// times it is infinite and not NaN.
#include <math.h>

#include "attn_body.cuh"
#include "mma_tile.cuh"

namespace b200 {

namespace {

constexpr int kShThreads = 128, kShTile = 32;

struct SharedParams {
  const __nv_bfloat16* qkv;
  const void* cos; const void* sin;
  int table_bf16, table_rows, table_presel, rope_n;
  const void* pos; int pos64, pos_each;      // pos_each: one position per row
  const void* plen; int plen64;              // null: prefix_rows
  __nv_bfloat16* kc; __nv_bfloat16* vc; int64_t kc_b, kc_g, vc_b, vc_g;
  const __nv_bfloat16* kp; const __nv_bfloat16* vp; int64_t kp_g, vp_g;
  __nv_bfloat16* out;
  int batch, n_head, n_groups, per, own_rows, prefix_rows;
  int tiles, prefix_splits, own_splits, head_tiles;   // query-row tiles of a group; key ranges; tiles of 16 heads of one row
  float* acc;                                // [batch][n_head][splits][HS]
  float2* ml;                                // [batch][n_head][splits]: maximum (log2 units), sum
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
// index of a row's new key in its own cache (pos >= 0)
__device__ __forceinline__ int own_index(const SharedParams& p, int64_t pos, int plen) {
  const int64_t i = pos - plen;
  return (int)(i < 0 ? 0 : (i >= p.own_rows ? p.own_rows - 1 : i));
}
__device__ __forceinline__ float ex2(float x) { float r; asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x)); return r; }

// apply_rope (lit_gpt/model.py:767-773) on element d of a head, for a position's table row
__device__ __forceinline__ __nv_bfloat16 turned(const SharedParams& p, const __nv_bfloat16* x, int d, int64_t row) {
  const int n = p.rope_n;
  if (d >= n) return x[d];
  const int half = n >> 1;
  const float a = __bfloat162float(x[d]), o = __bfloat162float(d < half ? x[d + half] : x[d - half]), rot = d < half ? -o : o;
  const float c = table_at(p.cos, p.table_bf16, row * n + d), s = table_at(p.sin, p.table_bf16, row * n + d);
  if (p.table_bf16) return __float2bfloat16_rn(__fadd_rn(round_bf16(__fmul_rn(a, c)), round_bf16(__fmul_rn(rot, s))));
  return __float2bfloat16_rn(__fadd_rn(__fmul_rn(a, c), __fmul_rn(rot, s)));
}
__device__ __forceinline__ int64_t table_row(const SharedParams& p, int b, int64_t pos) {
  const int64_t r = p.table_presel ? (p.pos_each ? b : 0) : pos;
  return r < 0 ? 0 : (r >= p.table_rows ? p.table_rows - 1 : r);
}

// Shared memory: four warps' key and value stages, then the query tile.
template <int HS, int MT>
struct ShSmem {
  static constexpr int kStage = 2 * kShTile * HS * 2, kWarp = 2 * kStage;     // K + V tile; two stages
  static constexpr int kQ = 16 * MT * HS * 2;
  static constexpr int kBytes = 4 * kWarp + kQ + 2 * HS * 2;
};

// The CTA's query tile against the keys [kbeg, kend) of one matrix of keys and values (rows HS apart), and the four warps' results joined.  `fresh` >= 0: that key's row
// and its value are in shared memory (nk, nv) and not yet in the matrix.  Results of row r go to slot(r); slot(r) < 0: nowhere.
template <int HS, int MT, typename Slot>
__device__ __forceinline__ void attend(const SharedParams& p, uint8_t* smem, uint8_t* sQ, const __nv_bfloat16* kg, const __nv_bfloat16* vg, int kbeg, int kend,
                                       int fresh, const __nv_bfloat16* nk, const __nv_bfloat16* nv, float (*s_m)[16 * MT], float (*s_l)[16 * MT], Slot slot) {
  constexpr int CH = HS / 8, RP = 32 / CH;   // 16-byte pieces of a row, rows a warp copies at once
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, tq = lane & 3;
  const uint32_t wbase = pf_smem(smem) + warp * ShSmem<HS, MT>::kWarp;
  const int ntiles = kend > kbeg ? (kend - kbeg + kShTile - 1) / kShTile : 0;

  auto load_tile = [&](int tile, int buf) {
    const int j0 = kbeg + tile * kShTile;
    const uint32_t kb = wbase + buf * ShSmem<HS, MT>::kStage, vb = kb + kShTile * HS * 2;
#pragma unroll
    for (int j = 0; j < kShTile / RP; ++j) {
      const int r = j * RP + lane / CH, c = lane % CH;
      const bool ok = j0 + r < kend && j0 + r != fresh;   // (zeros behind the range: a weight of zero times whatever lies there must be zero)
      const int64_t off = (int64_t)(ok ? j0 + r : kbeg) * HS + c * 8;
      pf_cp16(kb + sw<HS>(r, c), kg + off, ok);
      pf_cp16(vb + sw<HS>(r, c), vg + off, ok);
    }
    pf_commit();
  };

  float o[MT][HS / 8][4], m[MT][2], l[MT][2];
#pragma unroll
  for (int t = 0; t < MT; ++t) {
#pragma unroll
    for (int i = 0; i < HS / 8; ++i) o[t][i][0] = o[t][i][1] = o[t][i][2] = o[t][i][3] = 0.f;
    m[t][0] = m[t][1] = -INFINITY;
    l[t][0] = l[t][1] = 0.f;
  }
  if (warp < ntiles) load_tile(warp, 0);
  int it = 0;
  for (int tile = warp; tile < ntiles; tile += 4, ++it) {
    const int buf = it & 1;
    if (tile + 4 < ntiles) { load_tile(tile + 4, buf ^ 1); pf_wait<1>(); } else { pf_wait<0>(); }
    __syncwarp();
    const int j0 = kbeg + tile * kShTile;
    const uint32_t kb = wbase + buf * ShSmem<HS, MT>::kStage, vb = kb + kShTile * HS * 2;
    if (fresh >= j0 && fresh < j0 + kShTile) {
      if (lane < 2 * CH) {
        const int r = fresh - j0, c = lane % CH;
        const uint4 val = *reinterpret_cast<const uint4*>((lane < CH ? nk : nv) + c * 8);
        const uint32_t dst = (lane < CH ? kb : vb) + sw<HS>(r, c);
        asm volatile("st.shared.v4.u32 [%0], {%1,%2,%3,%4};" ::"r"(dst), "r"(val.x), "r"(val.y), "r"(val.z), "r"(val.w) : "memory");
      }
      __syncwarp();
    }
    float s[MT][kShTile / 8][4];
#pragma unroll
    for (int t = 0; t < MT; ++t)
#pragma unroll
      for (int i = 0; i < kShTile / 8; ++i) s[t][i][0] = s[t][i][1] = s[t][i][2] = s[t][i][3] = 0.f;
#pragma unroll
    for (int ks = 0; ks < HS / 16; ++ks) {
      uint32_t qf[MT][4];
#pragma unroll
      for (int t = 0; t < MT; ++t) ldsm_x4(qf[t], pf_smem(sQ) + sw<HS>(t * 16 + (lane & 15), ks * 2 + (lane >> 4)));
#pragma unroll
      for (int np = 0; np < kShTile / 16; ++np) {
        uint32_t kf[4];
        ldsm_x4(kf, kb + sw<HS>(np * 16 + ((lane >> 4) << 3) + (lane & 7), ks * 2 + ((lane >> 3) & 1)));
#pragma unroll
        for (int t = 0; t < MT; ++t) {
          pf_mma(s[t][2 * np], qf[t], kf[0], kf[1]);
          pf_mma(s[t][2 * np + 1], qf[t], kf[2], kf[3]);
        }
      }
    }
    uint32_t hi[MT][kShTile / 16][4], lo[MT][kShTile / 16][4];
#pragma unroll
    for (int t = 0; t < MT; ++t) {
      float top[2] = {m[t][0], m[t][1]};
#pragma unroll
      for (int i = 0; i < kShTile / 8; ++i) {
        const int j = j0 + i * 8 + 2 * tq;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          s[t][i][e] = (j + (e & 1) < kend) ? s[t][i][e] * p.scale_log2 : -INFINITY;
          top[e >> 1] = fmaxf(top[e >> 1], s[t][i][e]);
        }
      }
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        top[h] = fmaxf(top[h], __shfl_xor_sync(0xffffffffu, top[h], 1));
        top[h] = fmaxf(top[h], __shfl_xor_sync(0xffffffffu, top[h], 2));
        const float org = top[h] == -INFINITY ? 0.f : top[h];   // (scores that are all -inf: weights of zero)
        const float shrink = ex2(m[t][h] - org);
        m[t][h] = top[h];
        l[t][h] *= shrink;
#pragma unroll
        for (int i = 0; i < HS / 8; ++i) { o[t][i][2 * h] *= shrink; o[t][i][2 * h + 1] *= shrink; }
#pragma unroll
        for (int i = 0; i < kShTile / 8; ++i) {
          const float a = ex2(s[t][i][2 * h] - org), b = ex2(s[t][i][2 * h + 1] - org);
          l[t][h] += a + b;
          const uint32_t w = __byte_perm(__float_as_uint(a), __float_as_uint(b), 0x7632);   // the leading 16 bits of both
          hi[t][i >> 1][(i & 1) * 2 + h] = w;
          lo[t][i >> 1][(i & 1) * 2 + h] = pack_bf16(fmaxf(a - bf16lo(w), 1e-36f), fmaxf(b - bf16hi(w), 1e-36f));
        }
      }
    }
#pragma unroll
    for (int ks = 0; ks < kShTile / 16; ++ks) {
#pragma unroll
      for (int dp = 0; dp < HS / 16; ++dp) {
        uint32_t vf[4];
        ldsm_x4_t(vf, vb + sw<HS>(ks * 16 + (((lane >> 3) & 1) << 3) + (lane & 7), dp * 2 + (lane >> 4)));
#pragma unroll
        for (int t = 0; t < MT; ++t) {
          pf_mma(o[t][2 * dp], hi[t][ks], vf[0], vf[1]);
          pf_mma(o[t][2 * dp + 1], hi[t][ks], vf[2], vf[3]);
          pf_mma(o[t][2 * dp], lo[t][ks], vf[0], vf[1]);
          pf_mma(o[t][2 * dp + 1], lo[t][ks], vf[2], vf[3]);
        }
      }
    }
    __syncwarp();   // the stage just read is filled again by this warp's own copies
  }

  // the warp's result into its own stages, then all four joined
  float* const mine = reinterpret_cast<float*>(smem + warp * ShSmem<HS, MT>::kWarp);   // [16 * MT][HS]
#pragma unroll
  for (int t = 0; t < MT; ++t)
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      l[t][h] += __shfl_xor_sync(0xffffffffu, l[t][h], 1);
      l[t][h] += __shfl_xor_sync(0xffffffffu, l[t][h], 2);
      const int r = t * 16 + h * 8 + g;
#pragma unroll
      for (int i = 0; i < HS / 8; ++i) *reinterpret_cast<float2*>(mine + r * HS + i * 8 + 2 * tq) = make_float2(o[t][i][2 * h], o[t][i][2 * h + 1]);
      if (tq == 0) { s_m[warp][r] = m[t][h]; s_l[warp][r] = l[t][h]; }
    }
  __syncthreads();
  for (int i = tid; i < 16 * MT * (HS / 4); i += kShThreads) {
    const int r = i / (HS / 4), d = (i % (HS / 4)) * 4;
    const int64_t at = slot(r);
    if (at < 0) continue;
    const float top = fmaxf(fmaxf(s_m[0][r], s_m[1][r]), fmaxf(s_m[2][r], s_m[3][r])), org = top == -INFINITY ? 0.f : top;
    float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
    float sum = 0.f;
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      if (s_m[w][r] == -INFINITY && !(s_l[w][r] != 0.f)) continue;   // (nothing there)
      const float c = ex2(s_m[w][r] - org);
      const float4 v = *reinterpret_cast<const float4*>(reinterpret_cast<const float*>(smem + w * ShSmem<HS, MT>::kWarp) + r * HS + d);
      a.x += v.x * c; a.y += v.y * c; a.z += v.z * c; a.w += v.w * c;
      sum += s_l[w][r] * c;
    }
    __stcg(reinterpret_cast<float4*>(p.acc + at * HS + d), a);
    if (d == 0) __stcg(p.ml + at, make_float2(top, sum));
  }
}

template <int HS, int MT>
__global__ void __launch_bounds__(kShThreads, 1) attn_shared_kernel(const SharedParams p) {
  extern __shared__ __align__(128) uint8_t sh_smem[];
  __shared__ float s_m[4][16 * MT], s_l[4][16 * MT];
  uint8_t* const sQ = sh_smem + 4 * ShSmem<HS, MT>::kWarp;
  const int tid = threadIdx.x;
  griddep_launch();
  griddep_wait();
  const int plen = prefix_len(p), splits = p.prefix_splits + p.own_splits;
  int unit = blockIdx.x;
  const int own_units = p.batch * p.n_groups * p.head_tiles * p.own_splits;
  if (unit >= own_units) {
    // ---- rows of a group against a range of the prefix ----
    unit -= own_units;
    const int split = unit % p.prefix_splits, tile = (unit / p.prefix_splits) % p.tiles, gi = unit / (p.prefix_splits * p.tiles);
    const int per_range = (plen + p.prefix_splits - 1) / p.prefix_splits;
    const int kbeg = min(plen, split * per_range), kend = min(plen, kbeg + per_range);
    const int rows = p.batch * p.per;
    for (int i = tid; i < 16 * MT * HS; i += kShThreads) {
      const int r = i / HS, d = i % HS, row = tile * 16 * MT + r, b = row / p.per, h = row - b * p.per;
      __nv_bfloat16 v = __float2bfloat16_rn(0.f);
      if (row < rows) {
        const int64_t pos = row_pos(p, b);
        if (pos >= 0) v = turned(p, p.qkv + (((int64_t)b * p.n_groups + gi) * (p.per + 2) + h) * HS, d, table_row(p, b, pos));
      }
      *reinterpret_cast<__nv_bfloat16*>(sQ + sw<HS>(r, d >> 3) + (d & 7) * 2) = v;
    }
    __syncthreads();
    attend<HS, MT>(p, sh_smem, sQ, p.kp + (int64_t)gi * p.kp_g, p.vp + (int64_t)gi * p.vp_g, kbeg, kend, -1, nullptr, nullptr, s_m, s_l, [&](int r) -> int64_t {
      const int row = tile * 16 * MT + r, b = row / p.per;
      return row < rows ? ((int64_t)b * p.n_head + gi * p.per + (row - b * p.per)) * splits + split : (int64_t)-1;
    });
    return;
  }
  // ---- a row's heads of a group against a range of its own keys ----
  const int split = unit % p.own_splits;
  unit /= p.own_splits;
  const int ht = unit % p.head_tiles;
  unit /= p.head_tiles;
  const int gi = unit % p.n_groups, b = unit / p.n_groups;
  const int64_t pos = row_pos(p, b);
  if (pos < 0) return;
  const int mine = own_index(p, pos, plen), keys = mine + 1, per_range = (keys + p.own_splits - 1) / p.own_splits;
  const int kbeg = min(keys, split * per_range), kend = min(keys, kbeg + per_range);
  const bool fresh = mine >= kbeg && mine < kend;
  __nv_bfloat16* const nk = reinterpret_cast<__nv_bfloat16*>(sQ + ShSmem<HS, MT>::kQ);
  __nv_bfloat16* const nv = nk + HS;
  const __nv_bfloat16* const grp = p.qkv + ((int64_t)b * p.n_groups + gi) * (p.per + 2) * HS;
  const int64_t trow = table_row(p, b, pos);
  const int heads = min(16, p.per - ht * 16);
  for (int i = tid; i < 16 * HS; i += kShThreads) {
    const int r = i / HS, d = i % HS;
    *reinterpret_cast<__nv_bfloat16*>(sQ + sw<HS>(r, d >> 3) + (d & 7) * 2) = r < heads ? turned(p, grp + (int64_t)(ht * 16 + r) * HS, d, trow) : __float2bfloat16_rn(0.f);
  }
  if (fresh && tid < HS) {
    const __nv_bfloat16 k = turned(p, grp + (int64_t)p.per * HS, tid, trow), v = grp[(int64_t)(p.per + 1) * HS + tid];
    nk[tid] = k;
    nv[tid] = v;
    if (ht == 0) {   // (the other tiles of heads take the row from their own shared memory)
      p.kc[(int64_t)b * p.kc_b + (int64_t)gi * p.kc_g + (int64_t)mine * HS + tid] = k;
      p.vc[(int64_t)b * p.vc_b + (int64_t)gi * p.vc_g + (int64_t)mine * HS + tid] = v;
    }
  }
  __syncthreads();
  attend<HS, 1>(p, sh_smem, sQ, p.kc + (int64_t)b * p.kc_b + (int64_t)gi * p.kc_g, p.vc + (int64_t)b * p.vc_b + (int64_t)gi * p.vc_g, kbeg, kend, fresh ? mine : -1, nk, nv,
                reinterpret_cast<float (*)[16]>(s_m), reinterpret_cast<float (*)[16]>(s_l), [&](int r) -> int64_t {
                  return r < heads ? ((int64_t)b * p.n_head + gi * p.per + ht * 16 + r) * splits + p.prefix_splits + split : (int64_t)-1;
                });
}

// a (row, head) per HS / 4 threads
template <int HS>
__global__ void __launch_bounds__(256) attn_shared_join_kernel(const SharedParams p) {
  griddep_launch();
  griddep_wait();
  constexpr int T = HS / 4;
  const int64_t rh = (int64_t)blockIdx.x * (256 / T) + threadIdx.x / T;
  if (rh >= (int64_t)p.batch * p.n_head) return;
  const int d = (threadIdx.x % T) * 4;
  __nv_bfloat16* const out = p.out + rh * HS + d;
  if (row_pos(p, (int)(rh / p.n_head)) < 0) {
    *reinterpret_cast<uint2*>(out) = make_uint2(0u, 0u);
    return;
  }
  const int splits = p.prefix_splits + p.own_splits;
  const float2* const ml = p.ml + rh * splits;
  float top = -INFINITY;
  for (int i = 0; i < splits; ++i) top = fmaxf(top, __ldcg(ml + i).x);
  const float org = top == -INFINITY ? 0.f : top;
  float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
  float sum = 0.f;
  for (int i = 0; i < splits; ++i) {
    const float2 e = __ldcg(ml + i);
    if (e.x == -INFINITY && e.y == 0.f) continue;
    const float c = ex2(e.x - org);
    const float4 v = __ldcg(reinterpret_cast<const float4*>(p.acc + (rh * splits + i) * HS + d));
    a.x += v.x * c; a.y += v.y * c; a.z += v.z * c; a.w += v.w * c;
    sum += e.y * c;
  }
  const float inv = 1.f / sum;
  *reinterpret_cast<uint2*>(out) = make_uint2(pack_bf16(a.x * inv, a.y * inv), pack_bf16(a.z * inv, a.w * inv));
}

struct SharedPlan { int mt, tiles, prefix_splits, own_splits, head_tiles; };

SharedPlan shared_plan(int batch, int n_groups, int per, int prefix_rows, int own_rows) {
  SharedPlan s;
  const int rows = batch * per, fill = 2 * sm_count();
  s.mt = rows > 16 ? 2 : 1;
  s.tiles = (rows + 16 * s.mt - 1) / (16 * s.mt);
  s.head_tiles = (per + 15) / 16;
  auto ranges = [&](int units, int keys) {
    const int want = (fill + units - 1) / units, most = keys / 256;
    const int n = want < most ? want : most;
    return n < 1 ? 1 : (n > 64 ? 64 : n);
  };
  s.prefix_splits = prefix_rows > 0 ? ranges(s.tiles * n_groups, prefix_rows) : 0;
  s.own_splits = ranges(batch * n_groups * s.head_tiles, own_rows);
  return s;
}

template <int HS, int MT>
cudaError_t launch_shared(const SharedParams& p, cudaStream_t st) {
  constexpr int smem = ShSmem<HS, MT>::kBytes;
  static PerDeviceOnce once;
  if (once.need()) {
    const cudaError_t e = cudaFuncSetAttribute(attn_shared_kernel<HS, MT>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    if (e != cudaSuccess) return e;
    once.done();
  }
  const int64_t units = (int64_t)p.batch * p.n_groups * p.head_tiles * p.own_splits + (int64_t)p.n_groups * p.tiles * p.prefix_splits;
  const cudaError_t e = launch(attn_shared_kernel<HS, MT>, dim3((unsigned)units), dim3(kShThreads), (size_t)smem, st, p);
  if (e != cudaSuccess) return e;
  const int64_t heads = (int64_t)p.batch * p.n_head;
  constexpr int each = 256 / (HS / 4);
  return launch(attn_shared_join_kernel<HS>, dim3((unsigned)((heads + each - 1) / each)), dim3(256), 0, st, p);
}

}  // namespace
}  // namespace b200

using namespace b200;

extern "C" {

size_t b200_attn_decode_shared_workspace_bytes(int batch, int n_head, int n_groups, int head_size, int prefix_rows, int own_rows) {
  if (batch <= 0 || n_groups <= 0 || n_head <= 0 || n_head % n_groups || prefix_rows < 0 || own_rows <= 0 || (head_size != 64 && head_size != 128)) return 0;
  const SharedPlan s = shared_plan(batch, n_groups, n_head / n_groups, prefix_rows, own_rows);
  return (size_t)batch * n_head * (s.prefix_splits + s.own_splits) * (head_size + 2) * sizeof(float);
}

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
  const SharedPlan s = shared_plan(a->batch, a->n_groups, a->n_head / a->n_groups, a->prefix_rows, a->own_rows);
  const size_t slots = (size_t)a->batch * a->n_head * (s.prefix_splits + s.own_splits);
  B200_CHECK_ARG(a->workspace_bytes >= slots * (a->head_size + 2) * sizeof(float), "b200_attn_decode_shared: workspace too small");
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
  p.tiles = s.tiles; p.prefix_splits = s.prefix_splits; p.own_splits = s.own_splits; p.head_tiles = s.head_tiles;
  p.acc = (float*)a->workspace;
  p.ml = (float2*)(p.acc + slots * a->head_size);
  p.scale_log2 = 1.4426950408889634f / sqrtf((float)a->head_size);
  const cudaStream_t st = (cudaStream_t)stream;
  if (a->head_size == 128) B200_CUDA((s.mt == 2 ? launch_shared<128, 2>(p, st) : launch_shared<128, 1>(p, st)));
  else B200_CUDA((s.mt == 2 ? launch_shared<64, 2>(p, st) : launch_shared<64, 1>(p, st)));
  return B200_OK;
}

}  // extern "C"
