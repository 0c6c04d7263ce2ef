// Logits of several rows on their way to a token: penalties for repeated tokens, biases and a mask of allowed tokens (b200_adjust_logits), and the draw of one
// token per row with the same rules applied on the way (b200_sample_rows).
//
//   n = counts[b, v]; where n > 0:  l = l > 0 ? l / repetition : l * repetition;  l = l - frequency * n;  l = l - presence
//   l = l + bias[v];  tokens that are not allowed: -inf                                 (fp32, every step rounded by itself)
//   kept   : the top_k largest l of a row, equal ones in the order of the tokens; never one of -inf
//   token  : argmax over the kept ones of (l - max) / T - ln e,  e ~ Exp(1) from the row's own Philox state or a caller-given row;  T <= 0: argmax of l
//   logprob: (l_token - max) / T - ln sum over the kept ones of exp((l - max) / T)      (T <= 0: over all, as with T = 1)
// The adjusted logits are compared as the fp32 numbers that they are.  The winner is found in fp32 and, among those within 1e-3 of it (rounding of a score
// near the top: 4e-5 at most), in 64 bits, so that it is the argmax of the formula, the lowest token of equal ones.
#include "philox.cuh"

namespace b200 {

namespace {

struct Rules {
  const void* logits; int64_t ld;
  const int32_t* counts; int64_t counts_ld;
  const float* repetition; const float* frequency; const float* presence;
  float repetition_all, frequency_all, presence_all;
  const float* bias; int64_t bias_ld;
  const uint32_t* allowed; int64_t allowed_ld;
  int rows, vocab;
};

// the row's pointers and penalties
template <typename LT>
struct RowRules {
  const LT* logits; const int32_t* counts; const float* bias; const uint32_t* allowed;
  float rep, freq, pres;
  __device__ __forceinline__ RowRules(const Rules& r, int b) {
    logits = reinterpret_cast<const LT*>(r.logits) + (int64_t)b * r.ld;
    counts = r.counts ? r.counts + (int64_t)b * r.counts_ld : nullptr;
    bias = r.bias ? r.bias + (int64_t)b * r.bias_ld : nullptr;
    allowed = r.allowed ? r.allowed + (int64_t)b * r.allowed_ld : nullptr;
    rep = r.repetition ? r.repetition[b] : r.repetition_all;
    freq = r.frequency ? r.frequency[b] : r.frequency_all;
    pres = r.presence ? r.presence[b] : r.presence_all;
  }
  __device__ __forceinline__ float penalised(float l, int n) const {
    if (n > 0) {
      l = l > 0.f ? __fdiv_rn(l, rep) : __fmul_rn(l, rep);
      l = __fsub_rn(__fsub_rn(l, __fmul_rn(freq, (float)n)), pres);
    }
    return l;
  }
  __device__ __forceinline__ float at(int v) const {
    float l = load_as_float<LT>(logits, v);
    if (counts) l = penalised(l, counts[v]);
    if (bias) l = __fadd_rn(l, bias[v]);
    if (allowed && !((allowed[v >> 5] >> (v & 31)) & 1u)) l = -INFINITY;
    return l;
  }
  // four tokens from v, a multiple of four, on: every pointer that is there allows the wide access (wide()), and v + 3 < vocab
  __device__ __forceinline__ void at4(int v, float (&l)[4]) const {
    if constexpr (sizeof(LT) == 2) {
      const uint2 w = *reinterpret_cast<const uint2*>(logits + v);
      l[0] = bf16lo(w.x); l[1] = bf16hi(w.x); l[2] = bf16lo(w.y); l[3] = bf16hi(w.y);
    } else {
      const float4 w = *reinterpret_cast<const float4*>(logits + v);
      l[0] = w.x; l[1] = w.y; l[2] = w.z; l[3] = w.w;
    }
    if (counts) {
      const int4 n = *reinterpret_cast<const int4*>(counts + v);
      l[0] = penalised(l[0], n.x); l[1] = penalised(l[1], n.y); l[2] = penalised(l[2], n.z); l[3] = penalised(l[3], n.w);
    }
    if (bias) {
      const float4 a = *reinterpret_cast<const float4*>(bias + v);
      l[0] = __fadd_rn(l[0], a.x); l[1] = __fadd_rn(l[1], a.y); l[2] = __fadd_rn(l[2], a.z); l[3] = __fadd_rn(l[3], a.w);
    }
    if (allowed) {
      const uint32_t w = allowed[v >> 5] >> (v & 31);
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (!((w >> e) & 1u)) l[e] = -INFINITY;
    }
  }
  __device__ __forceinline__ bool wide() const {
    return ((reinterpret_cast<uintptr_t>(logits) & (4 * sizeof(LT) - 1)) | ((reinterpret_cast<uintptr_t>(counts) | reinterpret_cast<uintptr_t>(bias)) & 15)) == 0;
  }
};

// ---- adjusted logits ----------------------------------------------------------------------------------------------------------------
constexpr int kAdjThreads = 256, kAdjQuads = 2;   // four tokens a quad

template <typename LT, typename OT>
__global__ void __launch_bounds__(kAdjThreads) adjust_kernel(const Rules r, OT* out, int64_t out_ld, int chunks) {
  griddep_launch();
  griddep_wait();
  const int b = blockIdx.x / chunks, chunk = blockIdx.x - b * chunks;
  const RowRules<LT> row(r, b);
  OT* const o = out + (int64_t)b * out_ld;
  const int v0 = chunk * kAdjThreads * kAdjQuads * 4;
  if (row.wide() && (reinterpret_cast<uintptr_t>(o) & (4 * sizeof(OT) - 1)) == 0) {
#pragma unroll
    for (int i = 0; i < kAdjQuads; ++i) {
      const int v = v0 + (i * kAdjThreads + (int)threadIdx.x) * 4;
      if (v + 3 < r.vocab) {
        float l[4];
        row.at4(v, l);
        if constexpr (sizeof(OT) == 2) *reinterpret_cast<uint2*>(o + v) = make_uint2(pack_bf16(l[0], l[1]), pack_bf16(l[2], l[3]));
        else *reinterpret_cast<float4*>(o + v) = make_float4(l[0], l[1], l[2], l[3]);
      } else {
        for (int e = v; e < r.vocab; ++e) store_from_float<OT>(o, e, row.at(e));
      }
    }
  } else {
#pragma unroll 4
    for (int i = 0; i < kAdjQuads * 4; ++i) {
      const int v = v0 + i * kAdjThreads + (int)threadIdx.x;
      if (v < r.vocab) store_from_float<OT>(o, v, row.at(v));
    }
  }
}

// ---- the draw -----------------------------------------------------------------------------------------------------------------------
// A row's tokens are cut into the slices of a cluster's CTAs; a slice's adjusted logits stay in shared memory (CACHED) and are read again by every later step.
constexpr int kSaThreads = 512, kSaBins = 2048;

struct DrawArgs {
  const float* temperature; float temperature_all;
  const int32_t* top_k; int top_k_all;
  int64_t* rng; const float* noise; int64_t noise_ld;
  void* token; int token64;
  float* logprob;
  int32_t* count;   // (the rules' counts, to be raised by the token drawn)
  void* pos; int pos64;
  void* history; int64_t history_ld, history_len;
  int slice;        // tokens of a CTA, a multiple of four
};

__device__ __forceinline__ uint32_t cta_rank() { uint32_t r; asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r)); return r; }
__device__ __forceinline__ uint32_t cta_count() { uint32_t r; asm volatile("mov.u32 %0, %%cluster_nctarank;" : "=r"(r)); return r; }
__device__ __forceinline__ void cluster_barrier() { asm volatile("barrier.cluster.arrive.release;\n\tbarrier.cluster.wait.acquire;" ::: "memory"); }
__device__ __forceinline__ uint32_t remote(const void* p, uint32_t rank) {
  uint32_t r;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"((uint32_t)__cvta_generic_to_shared(p)), "r"(rank));
  return r;
}
__device__ __forceinline__ float remote_f32(const float* p, uint32_t rank) {
  float v;
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(remote(p, rank)) : "memory");
  return v;
}
__device__ __forceinline__ double remote_f64(const double* p, uint32_t rank) {
  double v;
  asm volatile("ld.shared::cluster.f64 %0, [%1];" : "=d"(v) : "r"(remote(p, rank)) : "memory");
  return v;
}
__device__ __forceinline__ uint4 remote_u4(const void* p, uint32_t rank) {
  uint4 v;
  asm volatile("ld.shared::cluster.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(remote(p, rank)) : "memory");
  return v;
}

template <typename LT, bool CACHED>
__global__ void __launch_bounds__(kSaThreads) sample_rows_kernel(const Rules r, const DrawArgs a) {
  extern __shared__ __align__(16) float s_l[];                       // the slice's adjusted logits, then its scores
  __shared__ __align__(16) uint32_t s_hist[2][kSaBins];
  __shared__ uint32_t s_warp[16], s_bin, s_left, s_in_bin;
  __shared__ float s_red[16];
  __shared__ double s_redd[16], s_weights[16];
  __shared__ int s_redi[16];
  __shared__ float s_max;
  __shared__ double s_score, s_weight, s_sum;
  __shared__ int s_index;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const uint32_t rank = cta_rank(), ctas = cta_count();
  const int b = blockIdx.x / ctas;
  griddep_launch();
  griddep_wait();
  const RowRules<LT> row(r, b);
  const int V = r.vocab, v0 = (int)rank * a.slice, v1 = min(V, v0 + a.slice), quads = v1 > v0 ? (v1 - v0 + 3) / 4 : 0;
  const float T = a.temperature ? a.temperature[b] : a.temperature_all;
  const bool greedy = !(T > 0.f);
  const int k = a.top_k ? a.top_k[b] : a.top_k_all;
  const float* const noise = a.noise ? a.noise + (int64_t)b * a.noise_ld : nullptr;
  const uint64_t seed = a.rng ? (uint64_t)a.rng[2 * b] : 0ull, offset = a.rng ? (uint64_t)a.rng[2 * b + 1] : 0ull;
  const bool wide = row.wide(), noise_wide = noise && (reinterpret_cast<uintptr_t>(noise) & 15) == 0;

  // a NaN logit counts as -inf, a zero has no sign; tokens past the vocabulary are -inf
  auto fetch = [&](int q, float (&l)[4]) {
    const int v = v0 + 4 * q;
    if (wide && v + 3 < V) {
      row.at4(v, l);
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e) l[e] = v + e < V ? row.at(v + e) : -INFINITY;
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) l[e] = l[e] == l[e] ? l[e] + 0.f : -INFINITY;
  };
  auto logits4 = [&](int q, float (&l)[4]) {
    if constexpr (CACHED) {
      const float4 w = *reinterpret_cast<const float4*>(s_l + 4 * q);
      l[0] = w.x; l[1] = w.y; l[2] = w.z; l[3] = w.w;
    } else {
      fetch(q, l);
    }
  };
  // e of four tokens: between 0 and the largest number
  auto exponentials = [&](int q, float (&e)[4]) {
    const int v = v0 + 4 * q;
    if (noise) {
      if (noise_wide && v + 3 < V) {
        const float4 w = *reinterpret_cast<const float4*>(noise + v);
        e[0] = w.x; e[1] = w.y; e[2] = w.z; e[3] = w.w;
      } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) e[i] = v + i < V ? noise[v + i] : 1.f;
      }
    } else {
      uint32_t rnd[4];
      philox4x32_10((uint32_t)(v >> 2), 0u, (uint32_t)offset, (uint32_t)(offset >> 32), (uint32_t)seed, (uint32_t)(seed >> 32), rnd);
#pragma unroll
      for (int i = 0; i < 4; ++i) e[i] = -__logf(((float)(rnd[i] >> 8) + 0.5f) * (1.0f / 16777216.0f));
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) e[i] = fmaxf(fminf(e[i], 3.4028234e38f), 0.f);
  };

  // ---- adjusted logits and their maximum ----
  float top = -INFINITY;
  for (int q = tid; q < quads; q += kSaThreads) {
    float l[4];
    fetch(q, l);
    if constexpr (CACHED) *reinterpret_cast<float4*>(s_l + 4 * q) = make_float4(l[0], l[1], l[2], l[3]);
    top = fmaxf(fmaxf(top, fmaxf(l[0], l[1])), fmaxf(l[2], l[3]));
  }
  for (int i = tid; i < kSaBins; i += kSaThreads) s_hist[0][i] = 0u;
  top = warp_max(top);
  if (lane == 0) s_red[warp] = top;
  __syncthreads();
  if (warp == 0) {
    top = warp_max(lane < 16 ? s_red[lane] : -INFINITY);
    if (lane == 0) s_max = top;
  }
  cluster_barrier();
  float M = -INFINITY;
  for (uint32_t c = 0; c < ctas; ++c) M = fmaxf(M, remote_f32(&s_max, c));

  // ---- the k-th largest (logit, lowest token): a digit of the 62-bit key a pass, from the highest ----
  uint64_t bound = 0ull;   // kept: keys from here on
  auto key_of = [](float l, int v) { return ((uint64_t)order_key(l) << 30) | (uint64_t)((1u << 30) - 1u - (uint32_t)v); };
  if (!greedy && k > 0 && k < V && M > -INFINITY) {
    uint32_t left = (uint32_t)k;
    int pass = 0;
    for (int shift = 51, bits = 11; shift >= 0; ++pass) {
      uint32_t* const hist = s_hist[pass & 1];
      for (int q = tid; q < quads; q += kSaThreads) {
        float l[4];
        logits4(q, l);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const uint64_t key = key_of(l[e], v0 + 4 * q + e);
          if ((key >> (shift + bits)) == (bound >> (shift + bits)) && l[e] > -INFINITY) atomicAdd(&hist[(uint32_t)(key >> shift) & ((1u << bits) - 1u)], 1u);
        }
      }
      cluster_barrier();
      // every CTA adds the histograms up: four bins a thread, the highest bins first
      const int first = kSaBins - 4 * (tid + 1);
      uint4 n = make_uint4(0u, 0u, 0u, 0u);
      for (uint32_t c = 0; c < ctas; ++c) {
        const uint4 m = remote_u4(hist + first, c);
        n.x += m.x; n.y += m.y; n.z += m.z; n.w += m.w;
      }
      uint32_t* const other = s_hist[(pass & 1) ^ 1];   // (read by all before they came to the barrier)
      *reinterpret_cast<uint4*>(other + first) = make_uint4(0u, 0u, 0u, 0u);
      const uint32_t total = n.x + n.y + n.z + n.w;
      uint32_t inc = total;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) { const uint32_t t = __shfl_up_sync(0xffffffffu, inc, o); if (lane >= o) inc += t; }
      if (lane == 31) s_warp[warp] = inc;
      if (tid == 0) s_bin = 0xffffffffu;
      __syncthreads();
      uint32_t before = inc - total;
      for (int w = 0; w < warp; ++w) before += s_warp[w];
      if (before < left && before + total >= left) {   // one thread at most
        uint32_t cum = before, bin = (uint32_t)first + 3u, here = n.w;
        if (cum + here < left) { cum += here; here = n.z; --bin; }
        if (bin == (uint32_t)first + 2u && cum + here < left) { cum += here; here = n.y; --bin; }
        if (bin == (uint32_t)first + 1u && cum + here < left) { cum += here; here = n.x; --bin; }
        s_bin = bin;
        s_left = left - cum;
        s_in_bin = here;
      }
      __syncthreads();
      if (s_bin == 0xffffffffu) break;   // fewer than k are above -inf: all of them (first pass only)
      bound |= (uint64_t)s_bin << shift;
      left = s_left;
      if (s_in_bin == left) break;       // the bin's are all kept
      if (shift == 0) break;
      const int next = shift == 51 ? 11 : 10;
      shift -= next;
      bits = next;
      __syncthreads();
    }
  }

  // ---- weights, scores in fp32 ----
  const float inv = greedy ? 1.f : 1.f / T, inv2 = inv * 1.4426950408889634f;
  float sum = 0.f, best = -INFINITY;
  if (M > -INFINITY) {
    for (int q = tid; q < quads; q += kSaThreads) {
      float l[4], e[4], s[4];
      logits4(q, l);
      if (!greedy) exponentials(q, e);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        s[i] = -INFINITY;
        if (l[i] > -INFINITY && key_of(l[i], v0 + 4 * q + i) >= bound) {
          const float gap = l[i] == M ? 0.f : l[i] - M;
          sum += gap == 0.f ? 1.f : exp2f(gap * inv2);
          s[i] = greedy ? l[i] : (gap == 0.f ? 0.f : gap * inv) - __logf(e[i]);
          best = fmaxf(best, s[i]);
        }
      }
      if constexpr (CACHED) *reinterpret_cast<float4*>(s_l + 4 * q) = make_float4(s[0], s[1], s[2], s[3]);
    }
  }
  sum = warp_sum(sum);
  best = warp_max(best);
  __syncthreads();
  if (lane == 0) { s_red[warp] = best; s_redd[warp] = (double)sum; }
  __syncthreads();
  best = warp_max(lane < 16 ? s_red[lane] : -INFINITY);
  double all = 0.0;
  if (tid == 0)
    for (int w = 0; w < 16; ++w) all += s_redd[w];

  // ---- the best of the slice in 64 bits, of equal ones the lowest token ----
  double score = -INFINITY, weight = 0.0;
  int index = 0x7fffffff;
  if (best > -INFINITY) {
    const float near = greedy ? best : best - 1e-3f;
    for (int q = tid; q < quads; q += kSaThreads) {
      float s[4], l[4], e[4];
      bool any;
      if constexpr (CACHED) {
        const float4 w = *reinterpret_cast<const float4*>(s_l + 4 * q);
        s[0] = w.x; s[1] = w.y; s[2] = w.z; s[3] = w.w;
        any = fmaxf(fmaxf(s[0], s[1]), fmaxf(s[2], s[3])) >= near;
        if (!any) continue;
        fetch(q, l);
        if (!greedy) exponentials(q, e);
      } else {
        fetch(q, l);
        if (!greedy) exponentials(q, e);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float gap = l[i] == M ? 0.f : l[i] - M;
          s[i] = !(l[i] > -INFINITY) || key_of(l[i], v0 + 4 * q + i) < bound ? -INFINITY : greedy ? l[i] : (gap == 0.f ? 0.f : gap * inv) - __logf(e[i]);
        }
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if (!(s[i] >= near)) continue;
        const double w = l[i] == M ? 0.0 : ((double)l[i] - (double)M) / (greedy ? 1.0 : (double)T);
        const double exact = greedy ? w : w - log((double)e[i]);
        const int v = v0 + 4 * q + i;
        if (index == 0x7fffffff || exact > score || (exact == score && v < index)) { score = exact; weight = w; index = v; }
      }
    }
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const double os = __shfl_xor_sync(0xffffffffu, score, o), ow = __shfl_xor_sync(0xffffffffu, weight, o);
    const int oi = __shfl_xor_sync(0xffffffffu, index, o);
    if (oi != 0x7fffffff && (index == 0x7fffffff || os > score || (os == score && oi < index))) { score = os; weight = ow; index = oi; }
  }
  __syncthreads();
  if (lane == 0) { s_redd[warp] = score; s_redi[warp] = index; s_weights[warp] = weight; }
  __syncthreads();
  if (tid == 0) {
    for (int w = 1; w < 16; ++w)
      if (s_redi[w] != 0x7fffffff && (index == 0x7fffffff || s_redd[w] > score || (s_redd[w] == score && s_redi[w] < index))) {
        score = s_redd[w]; weight = s_weights[w]; index = s_redi[w];
      }
    s_score = score; s_weight = weight; s_index = index; s_sum = all;
  }
  cluster_barrier();
  if (rank == 0 && tid == 0) {
    for (uint32_t c = 1; c < ctas; ++c) {
      int oi;
      asm volatile("ld.shared::cluster.s32 %0, [%1];" : "=r"(oi) : "r"(remote(&s_index, c)) : "memory");
      const double os = remote_f64(&s_score, c);
      all += remote_f64(&s_sum, c);
      if (oi != 0x7fffffff && (index == 0x7fffffff || os > score || (os == score && oi < index))) { score = os; weight = remote_f64(&s_weight, c); index = oi; }
    }
    const bool none = index == 0x7fffffff;   // nothing is allowed
    const int64_t tok = none ? -1 : index;
    if (a.token64) reinterpret_cast<int64_t*>(a.token)[b] = tok;
    else reinterpret_cast<int32_t*>(a.token)[b] = (int32_t)tok;
    if (a.logprob) a.logprob[b] = none ? -INFINITY : (float)(weight - log(all));
    if (a.rng) a.rng[2 * b + 1] = (int64_t)(offset + 1ull);
    if (a.count && !none) a.count[(int64_t)b * r.counts_ld + tok] += 1;
    if (a.pos) {
      const int64_t np = (a.pos64 ? reinterpret_cast<const int64_t*>(a.pos)[b] : (int64_t)reinterpret_cast<const int32_t*>(a.pos)[b]) + 1;
      if (a.pos64) reinterpret_cast<int64_t*>(a.pos)[b] = np;
      else reinterpret_cast<int32_t*>(a.pos)[b] = (int32_t)np;
      if (a.history && np >= 0 && np < a.history_len) {
        if (a.token64) reinterpret_cast<int64_t*>(a.history)[(int64_t)b * a.history_ld + np] = tok;
        else reinterpret_cast<int32_t*>(a.history)[(int64_t)b * a.history_ld + np] = (int32_t)tok;
      }
    }
  }
  cluster_barrier();   // no CTA leaves before its shared memory was read
}

constexpr int kSaMaxSlice = 48 * 1024;   // floats: 192 KB beside 17 KB of histograms

template <typename LT>
cudaError_t launch_draw(const Rules& r, DrawArgs a, cudaStream_t st) {
  int ctas = 1;
  while (ctas < 8 && (r.rows * ctas < 2 * sm_count() || (r.vocab + ctas - 1) / ctas > kSaMaxSlice) && r.vocab / ctas > 2048) ctas *= 2;
  a.slice = ((r.vocab + ctas - 1) / ctas + 3) & ~3;
  const bool cached = a.slice <= kSaMaxSlice;
  const size_t smem = cached ? (size_t)a.slice * sizeof(float) : 0;
  if (cached) {
    static PerDeviceOnce once;
    if (once.need()) {
      const cudaError_t e = cudaFuncSetAttribute(sample_rows_kernel<LT, true>, cudaFuncAttributeMaxDynamicSharedMemorySize, kSaMaxSlice * (int)sizeof(float));
      if (e != cudaSuccess) return e;
      once.done();
    }
    return launch_cluster(sample_rows_kernel<LT, true>, dim3((unsigned)(r.rows * ctas)), dim3(kSaThreads), ctas, smem, st, r, a);
  }
  return launch_cluster(sample_rows_kernel<LT, false>, dim3((unsigned)(r.rows * ctas)), dim3(kSaThreads), ctas, smem, st, r, a);
}

int check_rules(const b200_logit_rules* a, const char* what, Rules* out) {
  B200_CHECK_ARG(a && (a->logits || a->rows == 0), "%s: null pointer", what);
  B200_CHECK_ARG(a->logits_dtype == B200_BF16 || a->logits_dtype == B200_F32, "%s: logits must be bf16 or fp32", what);
  B200_CHECK_ARG(a->rows >= 0 && a->rows <= (1 << 20) && a->vocab > 0 && a->vocab < (1 << 30), "%s: %lld rows of %lld logits", what, (long long)a->rows, (long long)a->vocab);
  B200_CHECK_ARG(a->ld >= 0 && a->counts_ld >= 0 && a->bias_ld >= 0 && a->allowed_ld >= 0, "%s: negative row distance", what);
  Rules r;
  r.logits = a->logits; r.ld = a->ld;
  r.counts = a->counts; r.counts_ld = a->counts_ld;
  r.repetition = a->repetition; r.frequency = a->frequency; r.presence = a->presence;
  r.repetition_all = a->repetition_all; r.frequency_all = a->frequency_all; r.presence_all = a->presence_all;
  r.bias = a->bias; r.bias_ld = a->bias_ld;
  r.allowed = reinterpret_cast<const uint32_t*>(a->allowed); r.allowed_ld = a->allowed_ld;
  r.rows = (int)a->rows; r.vocab = (int)a->vocab;
  *out = r;
  return B200_OK;
}

}  // namespace
}  // namespace b200

using namespace b200;

extern "C" {

int b200_adjust_logits(const b200_logit_rules* rules, void* out, int out_dtype, int64_t out_ld, b200_stream_t stream) {
  Rules r;
  if (const int rc = check_rules(rules, "b200_adjust_logits", &r)) return rc;
  B200_CHECK_ARG((out || r.rows == 0) && (out_dtype == B200_BF16 || out_dtype == B200_F32), "b200_adjust_logits: the result is bf16 or fp32");
  B200_CHECK_ARG(out_ld >= r.vocab || r.rows <= 1, "b200_adjust_logits: result rows overlap");
  if (r.rows == 0) return B200_OK;
  const int each = kAdjThreads * kAdjQuads * 4, chunks = (r.vocab + each - 1) / each;
  B200_CHECK_ARG((int64_t)chunks * r.rows < 0x7fffffff, "b200_adjust_logits: too many logits");
  const dim3 grid((unsigned)(chunks * r.rows)), block(kAdjThreads);
  const cudaStream_t st = (cudaStream_t)stream;
  B200_FLOAT_TYPES(rules->logits_dtype, LT, B200_FLOAT_TYPES(out_dtype, OT, B200_CUDA((launch(adjust_kernel<LT, OT>, grid, block, 0, st, r, (OT*)out, out_ld, chunks)))));
  return B200_OK;
}

int b200_sample_rows(const b200_logit_rules* rules, const b200_draw_args* a, b200_stream_t stream) {
  Rules r;
  if (const int rc = check_rules(rules, "b200_sample_rows", &r)) return rc;
  B200_CHECK_ARG(a && (a->token_out || r.rows == 0), "b200_sample_rows: null pointer");
  B200_CHECK_ARG(a->rng_state || a->noise || (!a->temperature && !(a->temperature_all > 0.f)), "b200_sample_rows: temperature > 0 needs rng_state or noise");
  B200_CHECK_ARG(a->noise_ld >= 0 && a->history_ld >= 0, "b200_sample_rows: negative row distance");
  B200_CHECK_ARG(!a->count || rules->counts, "b200_sample_rows: nothing to count in");
  B200_CHECK_ARG(!a->history || a->pos_inout, "b200_sample_rows: a history needs positions");
  if (r.rows == 0) return B200_OK;
  DrawArgs d = {};
  d.temperature = a->temperature; d.temperature_all = a->temperature_all;
  d.top_k = a->top_k; d.top_k_all = a->top_k_all;
  d.rng = a->rng_state; d.noise = a->noise; d.noise_ld = a->noise_ld;
  d.token = a->token_out; d.token64 = a->token_is_int64;
  d.logprob = a->logprob_out;
  d.count = a->count ? const_cast<int32_t*>(rules->counts) : nullptr;
  d.pos = a->pos_inout; d.pos64 = a->pos_is_int64;
  d.history = a->history; d.history_ld = a->history_ld; d.history_len = a->history_len;
  B200_FLOAT_TYPES(rules->logits_dtype, LT, B200_CUDA((launch_draw<LT>(r, d, (cudaStream_t)stream))));
  return B200_OK;
}

}  // extern "C"
