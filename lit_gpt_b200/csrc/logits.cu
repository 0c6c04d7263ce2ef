// Logits of several rows on their way to a token: penalties for repeated tokens, biases and a mask of allowed tokens (b200_adjust_logits), and the draw of one
// token per row with the same rules applied on the way (b200_sample_rows).
//
//   n = counts[b, v]; where n > 0:  l = l > 0 ? l / repetition : l * repetition;  l = l - frequency * n;  l = l - presence
//   l = l + bias[v];  tokens that are not allowed: -inf                                 (fp32, every step rounded by itself)
//   kept   : the top_k largest l of a row, equal ones in the order of the tokens; never one of -inf
//   token  : argmax over the kept ones of (l - max) / T - ln e,  e ~ Exp(1) from the row's own Philox state or a caller-given row;  T <= 0: argmax of l
//   logprob: (l_token - max) / T - ln sum over the kept ones of exp((l - max) / T)      (T <= 0: over all, as with T = 1)
// The adjusted logits are compared as the fp32 numbers that they are.  The winner is found in fp32 and, among those that come within 1e-3 of it (rounding of a score
// near the top: 4e-5 at most), in 64 bits, so that it is the argmax of the formula, the lowest token of equal ones.
//
// Bound: adjusting by bytes, 64 x 50304 fp32 with counts, a bias and a mask per row 52 MB in 9.6 us (5.4 TB/s).  The draw reads what the rules need once.  Of a few rows it is
// a chain of waits: 32000 bf16 logits 8 us, 14.5 with a top-k of 200: a histogram of the first ten bits of the keys over the cluster, then one CTA goes on with the 1024 tokens
// at most that are left (up to 512 of them ranked one by one instead of digit by digit: 11.6 against 11.0 for fp32, 16.0 against 12.7 for bf16 with its equal logits, k = 50).
// Two bins a power of two leave more than 1024 where the vocabulary is large; every digit is then a pass over the cluster.  us, 1 row, k = 200, normal logits of standard
// deviation 2, 3, 4: of 32000 bf16 tokens 13.8 14.0 14.7, of 50257 16.6 14.7 16.6 (at 3 some rows leave few), of 128256 21.3 19.3 23.9; 16 rows 19.0 18.9 19.1, 21.9 21.1 21.4, 31.5 25.3 31.4.
// Of many rows it is what a token takes, its rules, weight and score, 96 instructions that wait
// for one another: 96 x 50257 fp32 with counts, a bias, masks and noise, 58 MB, 32 us (1.8 TB/s) with 46 % of the issue slots taken by 24 warps an SM.  Without the weights, where
// no log-probability is asked for, draws were 0 to 4 % shorter, and with one 1 to 3 % longer.  From Philox states and without rules, noise given in brackets: 96 x 50257 bf16 28.0
// (27.2), 64 x 50304 bf16 18.9 (19.4), 16 x 32000 bf16 10.2 (9.3), with a top-k of 200 18.9 (16.7).
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
  // N tokens v, v + STEP, ..; with FULL all of them are there, else those below `end`.  Everything is on its way before any of it is used.
  template <int N, int STEP, bool FULL>
  __device__ __forceinline__ void some(int v, int end, float (&l)[N]) const {
    int n[N];
    float add[N];
    bool out[N];
#pragma unroll
    for (int i = 0; i < N; ++i) {
      l[i] = FULL || v + i * STEP < end ? load_as_float<LT>(logits + v, i * STEP) : -INFINITY;
      n[i] = 0;
      add[i] = 0.f;
      out[i] = false;
    }
    if (counts) {
#pragma unroll
      for (int i = 0; i < N; ++i)
        if (FULL || v + i * STEP < end) n[i] = (counts + v)[i * STEP];
    }
    if (bias) {
#pragma unroll
      for (int i = 0; i < N; ++i)
        if (FULL || v + i * STEP < end) add[i] = (bias + v)[i * STEP];
    }
    if (allowed) {
#pragma unroll
      for (int i = 0; i < N; ++i)
        if (FULL || v + i * STEP < end) out[i] = STEP % 32 == 0 ? !((allowed + (v >> 5))[i * (STEP / 32)] >> (v & 31) & 1u) : !(allowed[(v + i * STEP) >> 5] >> ((v + i * STEP) & 31) & 1u);
    }
#pragma unroll
    for (int i = 0; i < N; ++i) l[i] = penalised(l[i], n[i]);
    if (bias) {
#pragma unroll
      for (int i = 0; i < N; ++i) l[i] = __fadd_rn(l[i], add[i]);
    }
#pragma unroll
    for (int i = 0; i < N; ++i) l[i] = out[i] ? -INFINITY : l[i];
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
// A row's tokens are cut into the slices of a cluster's CTAs; a slice's adjusted logits stay in shared memory (CACHED) and are read again by the later steps.
// NT threads a CTA: 512, or 256, of which three CTAs fit an SM.
constexpr int kSaDigit = 10, kSaBins = 1 << kSaDigit, kSaCtas = 8;
constexpr int kSaGather = 1024;   // tokens that one CTA goes on with alone
constexpr float kNear = 1.5e-3f;  // scores, in powers of two, this close to the best are compared in 64 bits

__device__ __forceinline__ float ex2(float x) { float r; asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x)); return r; }
__device__ __forceinline__ float lg2(float x) { float r; asm("lg2.approx.f32 %0, %1;" : "=f"(r) : "f"(x)); return r; }

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
__device__ __forceinline__ uint32_t remote_u32(const void* p, uint32_t rank) {
  uint32_t v;
  asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(remote(p, rank)) : "memory");
  return v;
}
template <int N>
__device__ __forceinline__ void remote_bins(const uint32_t* p, uint32_t rank, uint32_t (&v)[N]) {
  if constexpr (N == 4) asm volatile("ld.shared::cluster.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[N - 1]) : "r"(remote(p, rank)) : "memory");
  else asm volatile("ld.shared::cluster.v2.u32 {%0,%1}, [%2];" : "=r"(v[0]), "=r"(v[1]) : "r"(remote(p, rank)) : "memory");
}
__device__ __forceinline__ void remote_store(const void* p, uint32_t rank, uint32_t v) {
  asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(remote(p, rank)), "r"(v) : "memory");
}
__device__ __forceinline__ uint32_t remote_add(const void* p, uint32_t rank, uint32_t v) {
  uint32_t old;
  asm volatile("atom.shared::cluster.add.u32 %0, [%1], %2;" : "=r"(old) : "r"(remote(p, rank)), "r"(v) : "memory");
  return old;
}

// Where counts, from bin 0 on or with DOWN from the last bin on, come to `left`: the bin, what is left of `left` in it, what it holds (0xffffffff: nowhere).  n: the
// counts of the thread's own bins, of as many neighbours a thread.  All threads call it; true in the one whose bin it is.
template <int NT, bool DOWN>
__device__ __forceinline__ bool find_bin(const uint32_t (&n)[kSaBins / NT], uint32_t left, uint32_t* s_warp, uint32_t (&s_found)[3]) {
  constexpr int N = kSaBins / NT;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  uint32_t total = 0u;
#pragma unroll
  for (int i = 0; i < N; ++i) total += n[i];
  uint32_t inc = total;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) { const uint32_t t = __shfl_up_sync(0xffffffffu, inc, o); if (lane >= o) inc += t; }
  if (lane == 31) s_warp[warp] = inc;
  if (tid == 0) s_found[0] = 0xffffffffu;
  __syncthreads();
  uint32_t sum = lane < NT / 32 && lane < warp ? s_warp[lane] : 0u;
  sum = __reduce_add_sync(0xffffffffu, sum) + inc - total;
  const bool mine = sum < left && sum + total >= left;   // one thread at most
  if (mine) {
    int at = -1;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const uint32_t c = n[DOWN ? N - 1 - i : i];
      if (at < 0 && sum + c >= left) {
        at = i;
        s_found[1] = left - sum;
        s_found[2] = c;
      }
      sum += at < 0 ? c : 0u;
    }
    s_found[0] = (uint32_t)(DOWN ? kSaBins - 1 - (N * tid + at) : N * tid + at);
  }
  __syncthreads();
  return mine;
}

template <typename LT, bool CACHED, bool WIDE, int NT>
__global__ void __launch_bounds__(NT, NT == 512 ? 2 : 3) sample_rows_kernel(const Rules r, const DrawArgs a) {
  constexpr int kSaThreads = NT, kSaWarps = NT / 32, N = kSaBins / NT;
  extern __shared__ __align__(16) float s_l[];                       // the slice's adjusted logits
  __shared__ __align__(16) uint32_t s_hist[2][kSaBins];
  __shared__ uint32_t s_warp[kSaWarps], s_found[3], s_ties[kSaCtas], s_gathered;
  __shared__ float s_gl[kSaGather], s_ge[kSaGather];                  // gathered in the first CTA: logits, their e, their tokens
  __shared__ int s_gv[kSaGather];
  __shared__ float s_top[kSaWarps], s_l_of[kSaWarps], s_max;
  __shared__ uint64_t s_sum[kSaWarps];
  __shared__ int s_index[kSaWarps], s_close;
  __shared__ double s_exact[kSaWarps];
  __shared__ uint32_t s_all[kSaCtas][5];                              // of every CTA, in the first one: best score, its token, its logit, sum
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const uint32_t rank = cta_rank(), ctas = cta_count();
  const int b = blockIdx.x / ctas;
#pragma unroll
  for (int i = 0; i < N; ++i) s_hist[0][N * tid + i] = 0u;
  if (tid == 0) { s_close = 0; s_gathered = 0u; }
  griddep_launch();
  griddep_wait();
  const RowRules<LT> row(r, b);
  const int V = r.vocab, v0 = (int)rank * a.slice, n = max(0, min(V - v0, a.slice)), quads = (n + 3) / 4;
  const float T = a.temperature ? a.temperature[b] : a.temperature_all;
  const bool greedy = !(T > 0.f);
  const int k = a.top_k ? a.top_k[b] : a.top_k_all;
  const bool select = !greedy && k > 0 && k < V;
  const float* const noise = a.noise ? a.noise + (int64_t)b * a.noise_ld : nullptr;
  const uint64_t seed = a.rng ? (uint64_t)a.rng[2 * b] : 0ull, offset = a.rng ? (uint64_t)a.rng[2 * b + 1] : 0ull;
  __syncthreads();

  // a NaN logit counts as -inf, a zero has no sign; tokens past the slice are -inf
  auto clean = [](float l) { return l == l ? l + 0.f : -INFINITY; };
  auto logits4 = [&](int q, float (&l)[4]) {
    if constexpr (CACHED) {
      const float4 w = *reinterpret_cast<const float4*>(s_l + 4 * q);
      l[0] = w.x; l[1] = w.y; l[2] = w.z; l[3] = w.w;
    } else {
      row.template some<4, 1, false>(v0 + 4 * q, v0 + n, l);
#pragma unroll
      for (int e = 0; e < 4; ++e) l[e] = clean(l[e]);
    }
  };
  // e of four tokens: at most the largest number
  auto exponentials = [&](int v, float (&e)[4]) {
    if (noise) {
      if (v + 3 < V) {
        if constexpr (WIDE) {
          const float4 w = *reinterpret_cast<const float4*>(noise + v);
          e[0] = w.x; e[1] = w.y; e[2] = w.z; e[3] = w.w;
        } else {
#pragma unroll
          for (int i = 0; i < 4; ++i) e[i] = (noise + v)[i];
        }
      } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) e[i] = v + i < V ? noise[v + i] : 1.f;
      }
    } else {
      uint32_t rnd[4];
      philox4x32_10((uint32_t)(v >> 2), 0u, (uint32_t)offset, (uint32_t)(offset >> 32), (uint32_t)seed, (uint32_t)(seed >> 32), rnd);
#pragma unroll
      for (int i = 0; i < 4; ++i) e[i] = fmaxf(-__logf(((float)(rnd[i] >> 8) + 0.5f) * (1.0f / 16777216.0f)), 2.98023224e-8f);   // (the last of 2^24 numbers is rounded to 1: not 0 but 2^-25)
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) e[i] = fminf(e[i], 3.4028234e38f);
  };
  auto exponential = [&](int v) {
    if (noise) return fminf(noise[v], 3.4028234e38f);
    float e[4];
    exponentials(v & ~3, e);
    const float lo = v & 1 ? e[1] : e[0], hi = v & 1 ? e[3] : e[2];
    return v & 2 ? hi : lo;
  };

  // ---- adjusted logits, their maximum, the first digit's histogram ----
  float top = -INFINITY;
  auto see = [&](const auto& l) {
    if (select) {
      for (const float x : l)
        if (x > -INFINITY) atomicAdd(&s_hist[0][order_key(x) >> (32 - kSaDigit)], 1u);
    }
  };
  if constexpr (CACHED && WIDE) {
#pragma unroll 2
    for (int q = tid; q < quads; q += kSaThreads) {
      float l[4];
      if (v0 + 4 * q + 3 < V) row.at4(v0 + 4 * q, l);
      else row.template some<4, 1, false>(v0 + 4 * q, v0 + n, l);
#pragma unroll
      for (int e = 0; e < 4; ++e) l[e] = clean(l[e]);
      *reinterpret_cast<float4*>(s_l + 4 * q) = make_float4(l[0], l[1], l[2], l[3]);
      top = fmaxf(fmaxf(top, fmaxf(l[0], l[1])), fmaxf(l[2], l[3]));
      see(l);
    }
  } else {
    constexpr int E = 8;
    for (int i0 = tid; i0 < 4 * quads; i0 += E * NT) {
      float l[E];
      if (i0 + (E - 1) * NT < n) row.template some<E, NT, true>(v0 + i0, v0 + n, l);
      else row.template some<E, NT, false>(v0 + i0, v0 + n, l);
#pragma unroll
      for (int e = 0; e < E; ++e) {
        const int i = i0 + e * NT;
        l[e] = clean(l[e]);
        if (CACHED && i < 4 * quads) s_l[i] = l[e];
        top = fmaxf(top, l[e]);
      }
      see(l);
    }
  }
  top = warp_max(top);
  if (lane == 0) s_top[warp] = top;
  __syncthreads();
  if (warp == 0) {
    top = warp_max(lane < kSaWarps ? s_top[lane] : -INFINITY);
    if (lane == 0) s_max = top;
  }
  cluster_barrier();
  float M = __uint_as_float(remote_u32(&s_max, min((uint32_t)lane, ctas - 1)));   // (its warp's maximum is taken below)

  // ---- the k-th largest logit, a digit of its key a pass; of those equal to it the lowest tokens ----
  uint32_t bound = 0u;      // kept: keys above it, and those equal to it, from bit `low` on, up to token `cut`
  int low = 0, cut = 0x7fffffff;
  bool alone = false;       // the first CTA goes on with what was gathered
  uint32_t gathered = 0u;
  if (select) {
    uint32_t left = (uint32_t)k;
    const bool short_keys = sizeof(LT) == 2 && !row.counts && !row.bias;   // bf16 numbers: bits 15 .. 0 of a key say nothing
#pragma unroll 1
    for (int pass = 0, shift = 32 - kSaDigit, bits = kSaDigit;; ++pass) {
      uint32_t* const hist = s_hist[pass & 1];
      if (pass > 0) {
        if (alone) {
#pragma unroll 1
          for (uint32_t i = tid; i < gathered; i += kSaThreads) {
            const uint32_t key = order_key(s_gl[i]);
            if (((key ^ bound) >> (shift + bits)) == 0u) atomicAdd(&hist[(key >> shift) & ((1u << bits) - 1u)], 1u);
          }
          __syncthreads();
        } else {
#pragma unroll 1
          for (int q = tid; q < quads; q += kSaThreads) {
            float l[4];
            logits4(q, l);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const uint32_t key = order_key(l[e]);
              if (((key ^ bound) >> (shift + bits)) == 0u && l[e] > -INFINITY) atomicAdd(&hist[(key >> shift) & ((1u << bits) - 1u)], 1u);
            }
          }
          cluster_barrier();
        }
      }
      // every CTA adds the histograms up, the highest bins first
      const int first = kSaBins - N * (tid + 1);
      uint32_t m[kSaCtas][N], sum[N] = {};
      if (alone) {
#pragma unroll
        for (int i = 0; i < N; ++i) sum[i] = hist[first + i];
      } else {
#pragma unroll
        for (uint32_t c = 0; c < kSaCtas; ++c)
          if (c < ctas) remote_bins(hist + first, c, m[c]);
#pragma unroll
        for (uint32_t c = 0; c < kSaCtas; ++c)
#pragma unroll
          for (int i = 0; i < N; ++i) sum[i] += c < ctas ? m[c][i] : 0u;
      }
#pragma unroll
      for (int i = 0; i < N; ++i) s_hist[(pass & 1) ^ 1][first + i] = 0u;   // (read by all before they came to the barrier)
      if (find_bin<NT, true>(sum, left, s_warp, s_found) && !alone) {
        const int at = (int)s_found[0] - first;
#pragma unroll
        for (uint32_t c = 0; c < kSaCtas; ++c)
#pragma unroll
          for (int i = 0; i < N; ++i)
            if (i == at && c < ctas) s_ties[c] = m[c][i];
      }
      __syncthreads();
      const uint32_t bin = s_found[0], in_bin = s_found[2];
      if (bin == 0xffffffffu) break;           // fewer than k are above -inf: all of them (in the first pass)
      const uint32_t above = left - s_found[1];   // in higher bins
      bound |= bin << shift;
      left = s_found[1];
      low = shift;
      if (in_bin == left && (alone || pass > 0)) break;           // the bin's are all kept
      if (pass == 0 && above + in_bin <= (uint32_t)kSaGather) {
        // few: the first CTA takes them all; a warp finds out how many it has and asks for as many places
        auto goes = [&](float l) { return l > -INFINITY && order_key(l) >> shift >= bin; };
        int have = 0;
#pragma unroll 1
        for (int q = tid; q < quads; q += NT) {
          float l[4];
          logits4(q, l);
          have += goes(l[0]) + goes(l[1]) + goes(l[2]) + goes(l[3]);
        }
        int upto = have;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) { const int t = __shfl_up_sync(0xffffffffu, upto, o); if (lane >= o) upto += t; }
        uint32_t at = 0u;
        if (lane == 31 && upto > 0) at = remote_add(&s_gathered, 0, (uint32_t)upto);
        at = __shfl_sync(0xffffffffu, at, 31) + (uint32_t)(upto - have);
#pragma unroll 1
        for (int q = tid; have > 0 && q < quads; q += NT) {
          float l[4];
          logits4(q, l);
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (goes(l[e])) {
              const int v = v0 + 4 * q + e;
              remote_store(s_gl + at, 0, __float_as_uint(l[e]));
              remote_store(s_gv + at, 0, (uint32_t)v);
              remote_store(s_ge + at, 0, __float_as_uint(exponential(v)));
              ++at;
              --have;
            }
        }
        M = warp_max(M);
        cluster_barrier();   // (behind it no CTA reads or writes another's shared memory)
        if (rank != 0) return;
        alone = true;
        gathered = above + in_bin;
        if (in_bin == left) break;
      } else if (in_bin == left) {
        break;
      }
      if (shift == 0 || (short_keys && shift <= 16)) {
        // equal logits: those of the first CTAs, then of one CTA those of the lowest tokens
        uint32_t have = in_bin, keep = left;
        if (!alone) {
          uint32_t before = 0u;
          for (uint32_t c = 0; c < rank; ++c) before += s_ties[c];
          have = s_ties[rank];
          keep = left <= before ? 0u : min(left - before, have);
        }
        if (keep < have) {
          cut = -1;
          if (keep > 0u) {
            uint32_t want = keep;
            uint32_t* const local = s_hist[(pass & 1) ^ 1];    // (empty, and no other CTA's business)
            int token = 0;
#pragma unroll 1
            for (int at = 2 * kSaDigit; at >= 0; at -= kSaDigit) {   // digits of the token
              if (V >> at == 0) continue;
              auto look = [&](float l, int v) {
                if (((order_key(l) ^ bound) >> low) == 0u && l > -INFINITY && (at == 2 * kSaDigit || v >> (at + kSaDigit) == token >> (at + kSaDigit)))
                  atomicAdd(&local[(v >> at) & (kSaBins - 1)], 1u);
              };
              if (alone) {
#pragma unroll 1
                for (uint32_t i = tid; i < gathered; i += kSaThreads) look(s_gl[i], s_gv[i]);
              } else {
#pragma unroll 1
                for (int q = tid; q < quads; q += kSaThreads) {
                  float l[4];
                  logits4(q, l);
#pragma unroll
                  for (int e = 0; e < 4; ++e) look(l[e], v0 + 4 * q + e);
                }
              }
              __syncthreads();
              uint32_t h[N];
#pragma unroll
              for (int i = 0; i < N; ++i) { h[i] = local[N * tid + i]; local[N * tid + i] = 0u; }
              find_bin<NT, false>(h, want, s_warp, s_found);
              token |= (int)(s_found[0] << at);
              want = s_found[1];
              __syncthreads();
            }
            cut = token;
          }
        }
        break;
      }
      const int next = min(shift, kSaDigit);
      shift -= next;
      bits = next;
      __syncthreads();
    }
  }
  if (!alone) M = warp_max(M);
  auto kept = [&](float l, int v) {
    const uint32_t key = order_key(l) >> low, edge = bound >> low;
    return l > -INFINITY && (!select || key > edge || (key == edge && v <= cut));
  };

  // ---- weights and scores; a thread's best and whether another of its own comes close ----
  // What threads have is added as whole numbers, and gathered tokens each: the sum does not depend on the order that they were gathered in.
  // powers of two: gap * log2(e) / T, and what the product and the quotient were rounded by, which a weight of 2^-20 would otherwise have 2e-6 of its own of
  const float t = greedy ? 1.f : T, inv2 = fminf(1.44269502f / t, 3.4028234e38f);
  const float inv2_rest = inv2 < 1e30f && t < 1e30f ? (fmaf(-inv2, t, 1.44269502f) + 1.925963e-8f) / t : 0.f;
  const float unit = __int_as_float((127 + __clz(V) + 30) << 23);   // 2^(30 + leading zeros): V of them stay below 2^63
  auto power_of = [&](float l) { return (l == M ? 0.f : l - M) * inv2; };
  auto score_of = [&](float l, float e) { return greedy ? l : power_of(l) - lg2(e); };
  const uint64_t one = __float2ull_rz(unit);                        // the largest logit's weight; beside it what is small keeps its digits
  uint64_t sum = 0ull;
  float best = -INFINITY, second = -INFINITY, best_l = 0.f;
  int index = 0x7fffffff;
  auto weigh = [&](float l, float e, int v) {
    const float power = power_of(l), s = greedy ? l : power - lg2(e);
    const bool first = s > best;      // (the tokens of a slice come to a thread in their order)
    second = fmaxf(second, first ? best : s);
    best = first ? s : best;
    best_l = first ? l : best_l;
    index = first ? v : index;
    const float gap = l == M ? 0.f : l - M, w = ex2(power), rest = fmaf(gap, inv2, -power) + gap * inv2_rest;
    return power > -126.f ? fmaf(w, rest * 0.693147181f, w) : 0.f;
  };
  if (alone) {
#pragma unroll 1
    for (uint32_t i = tid; i < gathered; i += kSaThreads) {
      const float l = s_gl[i];
      if (kept(l, s_gv[i])) sum += __float2ull_rz(weigh(l, s_ge[i], s_gv[i]) * unit);
    }
  } else if (M > -INFINITY) {
    float part = 0.f;
    int tops = 0;
    constexpr int G = 4;   // quads of a thread whose noise is on its way together
#pragma unroll 1
    for (int q0 = tid; q0 < quads; q0 += G * NT) {
      float e[G][4];
      const int last = q0 + (G - 1) * NT;
      if (noise && !greedy && last < quads && v0 + 4 * last + 3 < V) {
        const float* const from = noise + v0 + 4 * q0;
#pragma unroll
        for (int g = 0; g < G; ++g) {
          if constexpr (WIDE) {
            const float4 w = *reinterpret_cast<const float4*>(from + g * 4 * NT);
            e[g][0] = w.x; e[g][1] = w.y; e[g][2] = w.z; e[g][3] = w.w;
          } else {
#pragma unroll
            for (int i = 0; i < 4; ++i) e[g][i] = from[g * 4 * NT + i];
          }
        }
#pragma unroll
        for (int g = 0; g < G; ++g)
#pragma unroll
          for (int i = 0; i < 4; ++i) e[g][i] = fminf(e[g][i], 3.4028234e38f);
      } else {
#pragma unroll
        for (int g = 0; g < G; ++g) {
          e[g][0] = e[g][1] = e[g][2] = e[g][3] = 1.f;
          if (!greedy && q0 + g * NT < quads) exponentials(v0 + 4 * (q0 + g * NT), e[g]);
        }
      }
#pragma unroll
      for (int g = 0; g < G; ++g) {
        const int q = q0 + g * NT;
        if (q >= quads) break;
        float l[4];
        logits4(q, l);
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (select ? kept(l[i], v0 + 4 * q + i) : l[i] > -INFINITY) {
            const float w = weigh(l[i], e[g][i], v0 + 4 * q + i);
            tops += l[i] == M;
            part += l[i] == M ? 0.f : w;
          }
      }
    }
    sum = __float2ull_rz(part * unit) + (uint64_t)tops * one;
  }
  const float mine = best;
  // the warp's, then the warps'
#pragma unroll 1
  for (int half = 0; half < 2; ++half) {
#pragma unroll 1
    for (int o = 16; o > 0; o >>= 1) {
      const float ob = __shfl_xor_sync(0xffffffffu, best, o), ol = __shfl_xor_sync(0xffffffffu, best_l, o);
      const int oi = __shfl_xor_sync(0xffffffffu, index, o);
      sum += __shfl_xor_sync(0xffffffffu, sum, o);
      if (ob > best || (ob == best && oi < index)) { best = ob; best_l = ol; index = oi; }
    }
    if (half == 0) {
      if (lane == 0) { s_top[warp] = best; s_l_of[warp] = best_l; s_index[warp] = index; s_sum[warp] = sum; }
      __syncthreads();
      const bool there = lane < kSaWarps;
      best = there ? s_top[lane] : -INFINITY;
      best_l = there ? s_l_of[lane] : 0.f;
      index = there ? s_index[lane] : 0x7fffffff;
      sum = there ? s_sum[lane] : 0ull;
    }
  }
  // ---- others that come close to the slice's best: in 64 bits, of equal ones the lowest token ----
  auto exact_score = [&](float l, float e) { return (l == M ? 0.0 : ((double)l - (double)M) / (double)T) - log((double)e); };
  const float near = greedy ? best : best - kNear;
  if (!greedy && best > -INFINITY) {
    const int close = (mine >= near) + (second >= near);
    if (close) atomicAdd(&s_close, close);
  }
  __syncthreads();
  if (s_close > 1) {
    double score = -INFINITY;
    best_l = 0.f;
    index = 0x7fffffff;
    auto rival = [&](float l, float e, int v) {
      if (!kept(l, v) || !(score_of(l, e) >= near)) return;
      const double x = exact_score(l, e);
      if (x > score || index == 0x7fffffff || (x == score && v < index)) { score = x; best_l = l; index = v; }
    };
    if (alone) {
#pragma unroll 1
      for (uint32_t i = tid; i < gathered; i += kSaThreads) rival(s_gl[i], s_ge[i], s_gv[i]);
    } else {
#pragma unroll 1
      for (int q = tid; q < quads; q += kSaThreads) {
        float l[4], e[4];
        logits4(q, l);
        exponentials(v0 + 4 * q, e);
#pragma unroll
        for (int i = 0; i < 4; ++i) rival(l[i], e[i], v0 + 4 * q + i);
      }
    }
#pragma unroll 1
    for (int half = 0; half < 2; ++half) {
#pragma unroll 1
      for (int o = 16; o > 0; o >>= 1) {
        const double ox = __shfl_xor_sync(0xffffffffu, score, o);
        const float ol = __shfl_xor_sync(0xffffffffu, best_l, o);
        const int oi = __shfl_xor_sync(0xffffffffu, index, o);
        if (oi != 0x7fffffff && (index == 0x7fffffff || ox > score || (ox == score && oi < index))) { score = ox; best_l = ol; index = oi; }
      }
      if (half == 0) {
        if (lane == 0) { s_exact[warp] = score; s_l_of[warp] = best_l; s_index[warp] = index; }
        __syncthreads();
        score = lane < kSaWarps ? s_exact[lane] : -INFINITY;
        best_l = lane < kSaWarps ? s_l_of[lane] : 0.f;
        index = lane < kSaWarps ? s_index[lane] : 0x7fffffff;
      }
    }
  }

  // ---- the first CTA's first warp takes the slices' results ----
  if (!alone && ctas > 1) {
    if (tid == 0) {
      remote_store(&s_all[rank][0], 0, __float_as_uint(best));
      remote_store(&s_all[rank][1], 0, (uint32_t)index);
      remote_store(&s_all[rank][2], 0, __float_as_uint(best_l));
      remote_store(&s_all[rank][3], 0, (uint32_t)sum);
      remote_store(&s_all[rank][4], 0, (uint32_t)(sum >> 32));
    }
    cluster_barrier();   // (behind it no CTA reads or writes another's shared memory)
    if (rank != 0 || warp != 0) return;
    const bool there = lane < (int)ctas;
    best = there ? __uint_as_float(s_all[lane & 7][0]) : -INFINITY;
    index = there ? (int)s_all[lane & 7][1] : 0x7fffffff;
    best_l = there ? __uint_as_float(s_all[lane & 7][2]) : 0.f;
    sum = there ? (uint64_t)s_all[lane & 7][3] | (uint64_t)s_all[lane & 7][4] << 32 : 0ull;
#pragma unroll 1
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    const float most = warp_max(best);
    const unsigned rivals = __ballot_sync(0xffffffffu, index != 0x7fffffff && (greedy ? best == most : best >= most - kNear));
    bool wins = rivals >> lane & 1u;
    if (rivals & (rivals - 1u)) {
      double score = -INFINITY;
      if (wins) score = greedy ? 0.0 : exact_score(best_l, exponential(index));
      double highest = score;
#pragma unroll 1
      for (int o = 16; o > 0; o >>= 1) {
        const double ox = __shfl_xor_sync(0xffffffffu, highest, o);
        highest = ox > highest ? ox : highest;
      }
      wins = wins && score == highest;
      const int lowest = __reduce_min_sync(0xffffffffu, wins ? index : 0x7fffffff);
      wins = wins && index == lowest;
    }
    const unsigned winner = __ballot_sync(0xffffffffu, wins);
    const int from = winner ? __ffs(winner) - 1 : 0;
    index = __shfl_sync(0xffffffffu, index, from);
    best_l = __shfl_sync(0xffffffffu, best_l, from);
  }
  if (tid != 0) return;
  const bool none = index == 0x7fffffff;   // nothing is allowed
  const int64_t tok = none ? -1 : index;
  if (a.token64) reinterpret_cast<int64_t*>(a.token)[b] = tok;
  else reinterpret_cast<int32_t*>(a.token)[b] = (int32_t)tok;
  if (a.logprob) a.logprob[b] = none ? -INFINITY : (best_l == M ? 0.f : (greedy ? best_l - M : (best_l - M) / T)) - log1pf(__ull2float_rn(sum > one ? sum - one : 0ull) / unit);
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

constexpr int kSaMaxSlice = 48 * 1024;   // floats: 192 KB beside the histograms and gathered tokens
constexpr int kSaOwnBytes = 22 * 1024;   // those, rounded up

template <typename LT, bool CACHED, bool WIDE, int NT>
cudaError_t allow_slices() {
  static PerDeviceOnce once;
  if (!once.need()) return cudaSuccess;
  const cudaError_t e = cudaFuncSetAttribute(sample_rows_kernel<LT, CACHED, WIDE, NT>, cudaFuncAttributeMaxDynamicSharedMemorySize, kSaMaxSlice * (int)sizeof(float));
  if (e == cudaSuccess) once.done();
  return e;
}

// CTAs of NT threads that an SM has place for beside each other, by their slices
template <int NT>
int ctas_an_sm(int slice) {
  const int by_memory = 228 * 1024 / (slice * (int)sizeof(float) + kSaOwnBytes + 1024), most = NT == 512 ? 2 : 3;
  return by_memory < most ? by_memory : most;
}
// Clusters that the GPU has at once (a cluster's SMs are neighbours: of 8 CTAs, two an SM, 148 SMs have 33, not 37).  Asked once per device.
template <int NT>
int clusters_at_once(int dev, int sms, int ctas, int an_sm) {
  static std::atomic<int> known[64][kSaCtas + 1][4];
  std::atomic<int>& here = known[dev & 63][ctas][an_sm];
  int n = here.load(std::memory_order_relaxed);
  if (n > 0) return n;
  if (allow_slices<float, true, true, NT>() == cudaSuccess) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)ctas);
    cfg.blockDim = dim3(NT);
    cfg.dynamicSmemBytes = an_sm == 1 ? kSaMaxSlice * sizeof(float) : 228 * 1024 / an_sm - kSaOwnBytes - 1024;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = (unsigned)ctas;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    if (cudaOccupancyMaxActiveClusters(&n, sample_rows_kernel<float, true, true, NT>, &cfg) != cudaSuccess) {
      (void)cudaGetLastError();
      n = 0;
    }
  }
  if (n <= 0) n = sms * an_sm / ctas > 1 ? sms * an_sm / ctas : 1;
  here.store(n, std::memory_order_relaxed);
  return n;
}
// What a draw takes, us, but for what all of them take: 3.5 for each further round of clusters, and per round by the SM that has most of it: 0.5 per 1000 tokens, 0.58 with CTAs
// of 256 threads, 0.7 and 1.1 if it has one CTA only; more CTAs of a cluster or of an SM wait for one another a little longer.  Against 34 sizes, 1 to 600 rows of 1000 to 150000
// tokens with and without a top-k, the CTAs chosen take 1.035 times the time of the best ones on average, 1.22 at worst (48 x 32000).
template <int NT>
float draw_time(int dev, int sms, int rows, int ctas, int slice) {
  const int an_sm = ctas_an_sm<NT>(slice), once = clusters_at_once<NT>(dev, sms, ctas, an_sm), full = (rows - 1) / once, rest = rows - full * once;
  const int last = (rest * ctas + sms - 1) / sms;
  auto tokens = [&](int n) { return (n == 1 ? (NT == 512 ? 0.7f : 1.1f) : (NT == 512 ? 0.5f : 0.58f) * (float)n) * 1e-3f * (float)slice; };
  return 3.5f * (float)full + (float)full * tokens(an_sm) + tokens(last < an_sm ? last : an_sm) + (float)ctas * (0.15f + 0.5f * (float)rows / (float)sms);
}

template <typename LT, bool CACHED, bool WIDE, int NT>
cudaError_t launch_draw_as(const Rules& r, const DrawArgs& a, int ctas, cudaStream_t st) {
  if (CACHED) {
    const cudaError_t e = allow_slices<LT, CACHED, WIDE, NT>();
    if (e != cudaSuccess) return e;
  }
  return launch_cluster(sample_rows_kernel<LT, CACHED, WIDE, NT>, dim3((unsigned)(r.rows * ctas)), dim3(NT), ctas, CACHED ? (size_t)a.slice * sizeof(float) : 0, st, r, a);
}

template <typename LT>
cudaError_t launch_draw(const Rules& r, DrawArgs a, cudaStream_t st) {
  // The cluster's CTAs, each with 1024 tokens at least, and their threads: the shortest of draw_time.  us, bf16 from Philox states, k = 50, of clusters of 1, 2, 3, 4, 6, 8 CTAs of 512 threads, of 256:
  //   1 x 32000   25.5 17.7 15.6 14.3 13.1 12.7, 37.4 23.2 18.7 17.0 15.4 14.1;     38 x 50304   25.6 25.5 24.2 21.9 19.6 27.9, 35.8 35.8 28.5 26.1 23.4 22.1
  //   96 x 50257  47.2 47.4 38.0 38.6 42.6 47.8, 65.9 65.8 49.7 30.3 39.9 42.0;     200 x 32000  51.7 38.5 46.7 47.4 59.1 72.8, 77.1 51.6 42.9 41.9 52.7 62.5
  const int sizes = r.vocab / 1024, most = sizes < 1 ? 1 : sizes < kSaCtas ? sizes : kSaCtas, least = (r.vocab + kSaMaxSlice - 1) / kSaMaxSlice;
  auto slice_of = [&](int ctas) { return ((r.vocab + ctas - 1) / ctas + 3) & ~3; };
  int ctas = kSaCtas, dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) dev = 0;
  const int sms = sm_count();
  bool few = true;
  float best = INFINITY;
  for (int c = least; c <= most; ++c) {
    const float wide_cta = draw_time<512>(dev, sms, r.rows, c, slice_of(c)), narrow = draw_time<256>(dev, sms, r.rows, c, slice_of(c));
    if (wide_cta <= best) { best = wide_cta; ctas = c; few = true; }
    if (narrow < best) { best = narrow; ctas = c; few = false; }
  }
  a.slice = slice_of(ctas);
  // four tokens an access where every row of everything that is there begins on such a boundary
  auto whole = [&](const void* p, int64_t ld, int bytes) { return !p || (((uintptr_t)p & (4 * bytes - 1)) == 0 && (r.rows == 1 || (ld & 3) == 0)); };
  const bool wide = whole(r.logits, r.ld, (int)sizeof(LT)) && whole(r.counts, r.counts_ld, 4) && whole(r.bias, r.bias_ld, 4) && whole(a.noise, a.noise_ld, 4);
  if (a.slice > kSaMaxSlice) return launch_draw_as<LT, false, false, 512>(r, a, ctas, st);
  if (few) return wide ? launch_draw_as<LT, true, true, 512>(r, a, ctas, st) : launch_draw_as<LT, true, false, 512>(r, a, ctas, st);
  return wide ? launch_draw_as<LT, true, true, 256>(r, a, ctas, st) : launch_draw_as<LT, true, false, 256>(r, a, ctas, st);
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
  B200_CHECK_ARG(out != r.logits || (out_dtype == rules->logits_dtype && (out_ld == r.ld || r.rows <= 1)), "b200_adjust_logits: in place the result has the logits' type and distance");
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
