// Partial results of a decode step's query rows over the prefix that they share, on the 5th-generation tensor cores (attn_shared.cu has the step, and says from where on).
//
// One CTA = 128 or 256 query rows of a group (rows of the batch times heads of the group) against a range of the prefix's keys, in tiles of 128 keys.  Two streams of products
// and softmax, each with its scores and its output in tensor memory, fill each other's gaps: with 256 rows the halves of the rows, with 128 the even and the odd key tiles,
// whose results are joined as those of two ranges.
//   * warps 0-7 and 8-15: a stream's softmax, half of a row's 128 keys per thread: its 64 scores are read into registers, the row's maximum is joined through shared memory,
//     and the weights go back over the scores as two bf16 numbers, the leading bits and the rest (attn_shared.cu says why).  A row's maximum moves, and its output shrinks,
//     only when the maximum grew by 2^8: with the rest a weight of 256 is as exact as one of 1.  With a whole row per thread, four warps a stream, a tile took 4600
//     clocks: a warp a scheduler does not fill the exponentials' 1024 clocks.  Unrolled over a row the code was 15 KB, and a launch spent 10000 clocks on fetching it once.
//   * warp 16: S = Q K^T (operands in shared memory) and O += P V (P from tensor memory, V as it lies), 128 x 128 x 16 each
//   * warps 17 and 18 bring keys and values, two stages each: whole tiles by TMA, the prefix's last one row by row, zeros behind it.
// Bound: the prefix's bytes with up to 128 rows (a tile of 128 keys, 64 KB, is 2800 clocks of an SM's share of the memory's rate, its products 1536), with 256 rows the
// products: 3 x 1024 clocks a tile, a third of them for the weights' second numbers.  A tile of 256 rows takes 4100: a stream's chain of scores, maximum, weights and output, which
// the other stream fills in part.  64 rows of 8 groups of 4 heads over 16001 shared and up to 1000 own keys, 193 MB: 54 us the whole step, 3.6 TB/s.
#include "attn_shared.cuh"
#include "attn_tmem.cuh"

namespace b200 {

namespace {

constexpr int kSpThreads = 608;
constexpr float kAbove = 1.00000012f;   // 1 + 2^-23 (attn_shared.cu)

template <int HS>
struct SpTile {
  static constexpr int kPanels = HS / 64, kBytes = kPanels * 128 * 128;   // an operand tile: panels of 128 rows of 128 bytes
  static constexpr int kSmem = 6 * kBytes + 1024;                         // Q0 Q1 | K x 2 | V x 2
  static constexpr uint32_t kIdescS = (1u << 4) | (1u << 7) | (1u << 10) | ((uint32_t)(128 >> 3) << 17) | ((uint32_t)(128 >> 4) << 24);
  static constexpr uint32_t kIdescO = (1u << 4) | (1u << 7) | (1u << 10) | (1u << 16) | ((uint32_t)(HS >> 3) << 17) | ((uint32_t)(128 >> 4) << 24);
  static constexpr uint32_t kS = 0, kO = 256;                             // tensor-memory columns: S0 S1 (P over them) | O0 O1
};

__device__ __forceinline__ void load_box(uint32_t dst, const CUtensorMap* map, int x, int row, int group, uint32_t bar) {
  asm volatile("cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];"
               ::"r"(dst), "l"(map), "r"(x), "r"(row), "r"(group), "r"(bar) : "memory");
}

template <int HS, bool PAIR>
__global__ void __launch_bounds__(kSpThreads, 1)
attn_shared_prefix_kernel(const SharedParams p, const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v,
                          int splits, unsigned* err) {
  using C = SpTile<HS>;
  extern __shared__ __align__(1024) uint8_t sp_smem[];
  __shared__ __align__(8) uint64_t s_bars[18];
  __shared__ uint32_t s_tmem;
  __shared__ float s_both[2][2][2][128];   // step, stream, half: a row's maximum over half of a tile; at the end its sum
  const int tid = threadIdx.x, lane = tid & 31, warp = __shfl_sync(0xffffffffu, tid >> 5, 0);
  const int split = blockIdx.x % splits, item = blockIdx.x / splits, tile_of_rows = item % p.pre_tiles, gi = item / p.pre_tiles;
  const int rows = p.batch * p.per, r0 = tile_of_rows * p.pre_rows;
  const uint32_t smem = (tc::smem_u32(sp_smem) + 1023u) & ~1023u;
  const uint32_t sq_ = smem, sk_ = smem + 2 * C::kBytes, sv_ = smem + 4 * C::kBytes;
  const uint32_t bars = tc::smem_u32(s_bars);
  const uint32_t k_full = bars, v_full = bars + 16, k_empty = bars + 32, v_empty = bars + 48, s_full = bars + 64, p_full = bars + 80, o_done = bars + 96, q_full = bars + 112,
                 idle = bars + 120, p_half = bars + 128;   // idle: products that gave up
  const int plen = prefix_len(p), tiles = (plen + 127) / 128, each = (tiles + splits - 1) / splits;
  const int first = min(tiles, split * each), n = min(tiles, first + each) - first;   // this CTA's key tiles
  if (tid == 0) {
    for (int i = 0; i < 2; ++i) {
      tc::mbar_init(k_full + 8 * i, 1);
      tc::mbar_init(v_full + 8 * i, 1);
      tc::mbar_init(k_empty + 8 * i, 1);
      tc::mbar_init(v_empty + 8 * i, 1);
      tc::mbar_init(s_full + 8 * i, 1);
      tc::mbar_init(p_half + 8 * i, 8);
      tc::mbar_init(p_full + 8 * i, 4);
      tc::mbar_init(o_done + 8 * i, 1);
    }
    tc::mbar_init(q_full, 1);
    tc::mbar_init(idle, 1);
    tc::mbar_init_fence();
  }
  __syncthreads();
  // The prefix was there before the turning kernel: its copies begin ahead of the wait for that one.  Only behind its wait a CTA lets attn_shared_kernel begin, which
  // counts on the turning kernel's end.
  uint32_t tmem = 0;
  if (warp < 17) {
    griddep_wait();
    griddep_launch();
    if (warp == 16) tc::tmem_alloc<512>(tc::smem_u32(&s_tmem));
    tc::fence_before();
    asm volatile("bar.sync 1, 544;" ::: "memory");
    tc::fence_after();
    tmem = s_tmem;
  }
  bool ok = true;

  if (warp >= 17) {
    // ================================ loads ================================
    const bool keys = warp == 17;
    const __nv_bfloat16* const src = keys ? p.kp + (int64_t)gi * p.kp_g : p.vp + (int64_t)gi * p.vp_g;
    const uint32_t dst = keys ? sk_ : sv_, full = keys ? k_full : v_full, empty = keys ? k_empty : v_empty;
    if (lane == 0) tc::prefetch_map(keys ? &map_k : &map_v);
    auto behind_the_wait = [&]() {
      griddep_wait();
      griddep_launch();
      if (keys && n > 0 && tc::elect()) {
        tc::mbar_expect_tx(q_full, (PAIR ? 2 : 1) * C::kBytes);
#pragma unroll
        for (int e = 0; e < (PAIR ? 2 : 1) * C::kPanels; ++e) load_box(sq_ + e * 16384u, &map_q, e % C::kPanels * 64, r0 + e / C::kPanels * 128, gi, q_full);
      }
    };
    int j = 0;
    for (; j < n; ++j) {
      if (j == 1) behind_the_wait();
      const int s = j & 1, row = (first + j) * 128;
      ok = __all_sync(0xffffffffu, tc::mbar_wait(empty + 8 * s, ((uint32_t)(j >> 1) & 1u) ^ 1u));
      if (!ok) break;
      if (row + 128 <= plen) {
        if (tc::elect()) {
          tc::mbar_expect_tx(full + 8 * s, C::kBytes);
#pragma unroll
          for (int e = 0; e < C::kPanels; ++e) load_box(dst + s * C::kBytes + e * 16384u, keys ? &map_k : &map_v, e * 64, row, gi, full + 8 * s);
        }
      } else {
        copy_tile<HS, 32>(dst + s * C::kBytes, src, HS, row, plen, lane);
        asm volatile("cp.async.wait_all;" ::: "memory");
        tc::fence_smem_async();
        __syncwarp();
        if (lane == 0) tc::mbar_arrive(full + 8 * s);
      }
    }
    if (n <= 1) behind_the_wait();
    // no copy may land after the CTA has left
    if (keys && n > 0) ok = __all_sync(0xffffffffu, tc::mbar_wait(q_full, 0)) && ok;
    for (int i = max(j - 2, 0); i < j; ++i) ok = __all_sync(0xffffffffu, tc::mbar_wait(full + 8 * (i & 1), (uint32_t)(i >> 1) & 1u)) && ok;
  } else if (warp == 16) {
    // ================================ products ================================
    if (tc::elect() && n > 0) {
      const uint32_t q_low = tc::desc_sw128_low(sq_), k_low = tc::desc_sw128_low(sk_), v_low = desc_v_low(sv_);
      auto scores = [&](int t, int s) {                    // S of stream t with the keys of stage s
        const uint32_t q = q_low + (PAIR ? t : 0) * (C::kBytes >> 4), k = k_low + s * (C::kBytes >> 4);
#pragma unroll
        for (int e = 0; e < HS / 16; ++e) {
          const uint32_t off = ((uint32_t)(e >> 2) * 16384u + (uint32_t)(e & 3) * 32u) >> 4;
          mma_ss(tmem + C::kS + t * 128, tc::desc_of(q + off, tc::kDescSw128High), tc::desc_of(k + off, tc::kDescSw128High), C::kIdescS, e != 0);
        }
        tc::commit(s_full + 8 * t);
      };
      auto outputs = [&](int t, int s, int half, bool begins) {   // O of stream t with half of the values of stage s
        const uint32_t dv = v_low + s * (C::kBytes >> 4), d = tmem + C::kO + t * HS, pp = tmem + C::kS + t * 128;
#pragma unroll
        for (int e = 4 * half; e < 4 * half + 4; ++e) {          // 16 keys: their leading bits, their rests
          const uint64_t v = tc::desc_of(dv + 128 * e, tc::kDescSw128High);
          mma_ts(d, pp + (e >> 1) * 32 + (e & 1) * 8, v, C::kIdescO, !(begins && e == 0));
          mma_ts(d, pp + (e >> 1) * 32 + 16 + (e & 1) * 8, v, C::kIdescO, 1u);
        }
      };
      auto arrived = [&](uint32_t bar, int j) { return tc::mbar_wait_here(bar + 8 * (j & 1), (uint32_t)(j >> 1) & 1u); };   // the copies of tile j
      ok = tc::mbar_wait_here(q_full, 0) && arrived(k_full, 0);
      if (ok) {
        tc::fence_after();
        scores(0, 0);
        if (PAIR) scores(1, 0);
        tc::commit(k_empty);
        if (!PAIR && n > 1) {
          ok = arrived(k_full, 1);
          if (ok) {
            tc::fence_after();
            scores(1, 1);
            tc::commit(k_empty + 8);
          }
        }
      }
      constexpr int AHEAD = PAIR ? 1 : 2;                  // the tile whose scores follow a tile's outputs
      for (int j = 0; j < n && ok; ++j) {
        const int s = j & 1, next = j + AHEAD;
        ok = arrived(v_full, j) && (next >= n || arrived(k_full, next));
        if (!ok) break;
#pragma unroll
        for (int u = 0; u < (PAIR ? 2 : 1); ++u) {
          const int t = PAIR ? u : s;
#pragma unroll
          for (int half = 0; half < 2; ++half) {
            ok = ok && tc::mbar_wait_here((half ? p_full : p_half) + 8 * t, (uint32_t)(PAIR ? j : j >> 1) & 1u);
            if (!ok) break;
            tc::fence_after();
            outputs(t, s, half, PAIR ? j == 0 : j < 2);
          }
          if (!ok) break;
          if (next < n) scores(t, next & 1);
          else tc::commit(o_done + 8 * t);
        }
        if (!ok) break;
        tc::commit(v_empty + 8 * s);
        if (next < n) tc::commit(k_empty + 8 * (next & 1));
      }
      if (!ok) {
        tc::commit(idle);
        tc::mbar_wait(idle, 0);
      }
    }
  } else {
    // ================================ softmax: half of a row's keys per thread ================================
    const int t = warp >> 3, half = (warp >> 2) & 1, r = (warp & 3) * 32 + lane, row = r0 + (PAIR ? t * 128 : 0) + r;
    const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
    const uint32_t ts = tmem + lanes + C::kS + t * 128 + half * 64, to = tmem + lanes + C::kO + t * HS + half * (HS / 2);
    const float sl = p.scale_log2, room = 8.f / sl;
    auto both = [&](float mine, int step) {                // the other half's number of the row
      s_both[step][t][half][r] = mine;
      asm volatile("bar.sync %0, 64;" ::"r"(2 + t * 4 + (warp & 3)) : "memory");
      return s_both[step][t][half ^ 1][r];
    };
    float m = -INFINITY;
    f2 l2[2] = {0ull, 0ull};
    uint32_t steps = 0;
    for (int j = PAIR ? 0 : t; j < n; j += PAIR ? 1 : 2, ++steps) {
      ok = ok && __all_sync(0xffffffffu, tc::mbar_wait(s_full + 8 * t, steps & 1u));
      if (!ok) {       // (a warp that gave up a wait still meets the one that has the rows' other half)
        both(0.f, steps & 1);
        continue;
      }
      tc::fence_after();
      uint32_t v[2][32];
      tc::ld32(v[0], ts);
      tc::ld32(v[1], ts + 32);
      const int valid = plen - (first + j) * 128 - half * 64;
      float mx[2];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        tc::wait_ld(v[i]);
        if (32 * i + 32 > valid) {
#pragma unroll
          for (int e = 0; e < 32; ++e)
            if (32 * i + e >= valid) v[i][e] = 0xff800000u;
        }
        mx[i] = -INFINITY;
#pragma unroll
        for (int e = 0; e < 32; e += 2) mx[i] = max3(mx[i], __uint_as_float(v[i][e]), __uint_as_float(v[i][e + 1]));
      }
      const float here = fmaxf(mx[0], mx[1]), top = fmaxf(here, both(here, steps & 1));
      const bool grew = top > m + room || (m == -INFINITY && top > m);
      if (__any_sync(0xffffffffu, grew && steps > 0)) {   // (S of this step is there, so P V of the last one is done)
        const float f = !grew ? 1.f : m == -INFINITY ? 0.f : ex2((m - top) * sl);
        const f2 ff = pk2(f, f);
        l2[0] = fma2(l2[0], ff, 0ull);
        l2[1] = fma2(l2[1], ff, 0ull);
#pragma unroll 1
        for (int c = 0; c < HS / 2; c += 16) {
          uint32_t o[16];
          tc::ld16(o, to + c);
          tc::wait_ld(o);
#pragma unroll
          for (int e = 0; e < 16; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * f);
          st16(to + c, o);
        }
        wait_st();
      }
      if (half) {      // both halves' outputs have shrunk before any product
        tc::fence_before();
        __syncwarp();
        if (lane == 0) tc::mbar_arrive(p_half + 8 * t);
      }
      if (grew) m = top;
      const float org = m == -INFINITY ? 0.f : m * sl;
      const f2 sl2 = pk2(sl, sl), org2 = pk2(-org, -org);
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        uint32_t hi[16], lo[16];
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          float a, b;
          un2(fma2(pk2(__uint_as_float(v[i][2 * e]), __uint_as_float(v[i][2 * e + 1])), sl2, org2), a, b);
          a = ex2(a);
          b = ex2(b);
          l2[e & 1] = add2(l2[e & 1], pk2(a, b));
          hi[e] = __byte_perm(__float_as_uint(a), __float_as_uint(b), 0x7632);
          un2(fma2(pk2(a, b), pk2(kAbove, kAbove), pk2(-bf16lo(hi[e]), -bf16hi(hi[e]))), a, b);
          lo[e] = pack_bf16(a, b);
        }
        st16(ts + i * 32, hi);        // over their own scores: leading bits, rests
        st16(ts + i * 32 + 16, lo);
      }
      wait_st();
      tc::fence_before();
      __syncwarp();
      if (lane == 0) tc::mbar_arrive((half ? p_full : p_half) + 8 * t);
    }
    const int64_t slot = PAIR ? ((int64_t)item * splits + split) * 256 + t * 128 + r : (((int64_t)item * splits + split) * 2 + t) * 128 + r;
    if (steps > 0 && ok) {
      // The rows go through shared memory, where nothing is read any more once both streams are done, and from there a row at a time: stored from registers, a warp's
      // 16 bytes of 32 rows take 32 sectors each; by a bulk copy of every thread's own row, 256 copies took 4500 clocks.
      ok = __all_sync(0xffffffffu, tc::mbar_wait(o_done, 0) && (!(PAIR || n > 1) || tc::mbar_wait(o_done + 8, 0)));
      tc::fence_after();
      constexpr uint32_t LD = HS * 2 + 16;      // half a row
      const uint32_t mine = smem + (uint32_t)tid * LD;
#pragma unroll 1
      for (int c = 0; c < HS / 2 && ok; c += 32) {
        uint32_t o[32];
        tc::ld32(o, to + c);
        tc::wait_ld(o);
#pragma unroll
        for (int e = 0; e < 32; e += 4)
          asm volatile("st.shared.v4.u32 [%0], {%1,%2,%3,%4};" ::"r"(mine + (c + e) * 4), "r"(o[e]), "r"(o[e + 1]), "r"(o[e + 2]), "r"(o[e + 3]) : "memory");
      }
      __syncwarp();
      constexpr int LR = HS / 8, R = 32 / LR;   // lanes half a row, rows at once
      const uint32_t from = smem + (uint32_t)(tid - lane + lane / LR) * LD + lane % LR * 16;
      float* const acc = p.pre_acc + (slot - lane + lane / LR) * HS + half * (HS / 2) + lane % LR * 4;
      const int there = ok ? rows - (row - lane) - lane / LR : 0;
#pragma unroll 4
      for (int i = 0; i < 32; i += R) {
        uint4 x;
        asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(x.x), "=r"(x.y), "=r"(x.z), "=r"(x.w) : "r"(from + i * LD));
        if (i < there) __stcg(reinterpret_cast<uint4*>(acc + i * HS), x);
      }
    }
    float a, b, c, d;
    un2(l2[0], a, b);
    un2(l2[1], c, d);
    const float l = (a + b) + (c + d), all = l + both(l, steps & 1);   // (a step's buffer that no half still reads: the last one's was the other)
    if (row < rows && half == 0) __stcg(p.pre_ml + slot, make_float2(m == -INFINITY ? m : m * sl, all));
  }
  if (!ok) *err = 1u;
  tc::fence_before();
  __syncthreads();
  if (warp == 16) {
    __syncwarp();
    tc::tmem_free<512>(tmem);
  }
}

// [groups][rows][HS] in boxes of 128 rows x 64 numbers, 128-byte swizzle, zeros outside.  (Prefixes of fewer than 128 rows are not read through it.)
bool prefix_map(CUtensorMap* map, const void* base, int hs, int rows, int groups, int64_t group_stride) {
  const TensorMapEncodeFn enc = tensor_map_encoder();
  if (!enc) return false;
  const cuuint64_t dim[3] = {(cuuint64_t)hs, (cuuint64_t)rows, (cuuint64_t)groups};
  const cuuint64_t stride[2] = {(cuuint64_t)hs * 2, (cuuint64_t)(groups > 1 ? group_stride : (int64_t)rows * hs) * 2};
  const cuuint32_t box[3] = {64u, 128u, 1u}, step[3] = {1u, 1u, 1u};
  return enc(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, const_cast<void*>(base), dim, stride, box, step, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
             CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <int HS, bool PAIR>
cudaError_t launch_prefix(const SharedParams& p, int splits, cudaStream_t st) {
  constexpr int smem = SpTile<HS>::kSmem;
  static PerDeviceOnce once;
  if (once.need()) {
    const cudaError_t e = cudaFuncSetAttribute(attn_shared_prefix_kernel<HS, PAIR>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    if (e != cudaSuccess) return e;
    once.done();
  }
  alignas(64) CUtensorMap mq, mk, mv;
  if (!prefix_map(&mq, p.q, HS, p.batch * p.per, p.n_groups, (int64_t)p.batch * p.per * HS) || !prefix_map(&mk, p.kp, HS, p.prefix_rows, p.n_groups, p.kp_g) || !prefix_map(&mv, p.vp, HS, p.prefix_rows, p.n_groups, p.vp_g)) return cudaErrorInvalidValue;
  unsigned* const err = wait_error_word();
  if (!err) return cudaErrorMemoryAllocation;
  return launch(attn_shared_prefix_kernel<HS, PAIR>, dim3((unsigned)(p.n_groups * p.pre_tiles * splits)), dim3(kSpThreads), (size_t)smem, st, p, mq, mk, mv, splits, err);
}

}  // namespace

cudaError_t launch_attn_shared_prefix(const SharedParams& p, int head_size, bool pair, int splits, cudaStream_t st) {
  if (head_size == 128) return pair ? launch_prefix<128, true>(p, splits, st) : launch_prefix<128, false>(p, splits, st);
  return pair ? launch_prefix<64, true>(p, splits, st) : launch_prefix<64, false>(p, splits, st);
}

}  // namespace b200
