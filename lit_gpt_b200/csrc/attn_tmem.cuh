// What attention kernels on the 5th-generation tensor cores share (attn_tc05.cu, attn_shared_tc05.cu): products with both operands in shared memory or the left one in
// tensor memory, packed float arithmetic, operand tiles of 128 rows.
#pragma once
#include "tc05.cuh"

namespace b200 {

typedef unsigned long long f2;   // two packed floats
__device__ __forceinline__ f2 pk2(float a, float b) { f2 r; asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b)); return r; }
__device__ __forceinline__ void un2(f2 v, float& a, float& b) { asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(v)); }
__device__ __forceinline__ f2 fma2(f2 a, f2 b, f2 c) { f2 r; asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c)); return r; }
__device__ __forceinline__ f2 add2(f2 a, f2 b) { f2 r; asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b)); return r; }
__device__ __forceinline__ float ex2(float x) { float r; asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x)); return r; }

// S = Q K^T: both K-major in shared memory
__device__ __forceinline__ void mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
  asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\ttcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}"
               ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(accumulate) : "memory");
}
// O += P V: P in tensor memory
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
  asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\ttcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}"
               ::"r"(d), "r"(a), "l"(b), "r"(idesc), "r"(accumulate) : "memory");
}
__device__ __forceinline__ void st16(uint32_t addr, const uint32_t (&v)[16]) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};"
               ::"r"(addr), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]), "r"(v[9]), "r"(v[10]),
               "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15])
               : "memory");
}
__device__ __forceinline__ float max3(float a, float b, float c) { float r; asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c)); return r; }
__device__ __forceinline__ void wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void cp16(uint32_t dst, const void* src, bool valid) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(valid ? 16 : 0) : "memory");
}

// V tile as the right operand: N = HS contiguous (MN-major), 64 numbers per 128-byte row, one row per key: 8-key groups 1024 bytes apart
// (stride offset), the second panel of 64 numbers 16 KB on (leading offset).  +128 in the address field is 16 keys.
// The low word of the descriptor; the high one is tc::kDescSw128High.
__device__ __forceinline__ uint32_t desc_v_low(uint32_t addr) { return ((addr & 0x3FFFFu) >> 4) | ((16384u >> 4) << 16); }

// Rows [first, first + 128) of a matrix into a swizzled tile by N threads (this one `id`), zeros from row `end` on
template <int HS, int N>
__device__ __forceinline__ void copy_tile(uint32_t dst, const __nv_bfloat16* src, int64_t ld, int first, int end, int id) {
  constexpr int CH = HS / 8, RP = N / CH;   // 16-byte pieces per row, rows per pass
  const int c = id % CH, rr = id / CH;
  const __nv_bfloat16* p = src + (int64_t)(first + rr) * ld + c * 8;
  dst += (uint32_t)(c >> 3) * 16384u;
#pragma unroll 8
  for (int i = 0; i < 128 / RP; ++i) {
    const int r = rr + i * RP;
    const bool in = first + r < end;
    cp16(dst + (uint32_t)(r * 128 + (((c & 7) ^ (r & 7)) << 4)), in ? p + (int64_t)(i * RP) * ld : src, in);
  }
}

}  // namespace b200
