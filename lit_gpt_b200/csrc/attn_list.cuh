// What the attention kernels that walk a list of key tiles share (attn_shared.cu, paged_attn.cu): a warp's products over a tile of 32 keys, S^T = K Q^T and O^T += V^T P^T on
// mma.sync, its partial results, and how a head's partial results are joined; the rotation of a head by a warp.
#pragma once
#include <math.h>

#include "attn_body.cuh"
#include "mma_tile.cuh"

namespace b200 {
namespace list {

constexpr int kShTile = 32;                 // keys of a tile
constexpr float kAbove = 1.00000012f;       // 1 + 2^-23: a weight's second number is never zero

__device__ __forceinline__ float ex2(float x) { float r; asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x)); return r; }


// apply_rope (lit_gpt/model.py:767-773)
__device__ __forceinline__ float turned(float a, float other, bool low, float c, float s, int table_bf16) {
  const float rot = low ? -other : other;
  if (table_bf16) return __fadd_rn(round_bf16(__fmul_rn(a, c)), round_bf16(__fmul_rn(rot, s)));
  return __fadd_rn(__fmul_rn(a, c), __fmul_rn(rot, s));
}
// HS / 32 numbers of a head from lane * HS / 32 on, after the rotation
template <int HS, typename Params>
__device__ __forceinline__ void turned_part(const Params& p, const __nv_bfloat16* x, int64_t trow, int lane, uint32_t (&out)[HS / 64]) {
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

// 8 N queries, from row q0 of `q` on, and a tile of keys: S^T = K Q^T and O^T += V^T P^T, keys and dimensions as the rows of the products, so that few queries cost few of them.  seen(key,
// t, c): whether query 8 t + 2 tq + c sees that key of the tile; keep(key, t, c, s): for a
// use of its score times log2(e), -inf where it does not.  `vb` of the values is what `values` gives, which waits for them.
template <int HS, int NQ, int N, typename Seen, typename Keep, typename Values>
__device__ __forceinline__ void attend_tile(Sums<HS, NQ>& a, uint32_t q, int q0, uint32_t kb, float scale_log2, int lane, Seen seen, Keep keep, Values values) {
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
        s[i][t][e] = seen(i * 16 + (e >> 1) * 8 + g, t, e & 1) ? s[i][t][e] * scale_log2 : -INFINITY;
        keep(i * 16 + (e >> 1) * 8 + g, t, e & 1, s[i][t][e]);
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
  top = now;
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

}  // namespace list
}  // namespace b200
