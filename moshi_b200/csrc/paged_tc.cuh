// What the tensor-core kernels of the paged 8-bit cache share (paged_prompt.cu, paged_tree.cu): TMEM reads and writes, pairs of fp32 operations, masks, the two products' operands.
#pragma once

#include "paged.cuh"

namespace b200 {
namespace paged {

using namespace tcp;

#define R32(r, o) "=r"((r)[o]), "=r"((r)[o + 1]), "=r"((r)[o + 2]), "=r"((r)[o + 3]), "=r"((r)[o + 4]), "=r"((r)[o + 5]), "=r"((r)[o + 6]), "=r"((r)[o + 7])
__device__ __forceinline__ void tmem_ld32(uint32_t taddr, uint32_t* r) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
      "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
      : R32(r, 0), R32(r, 8), R32(r, 16), R32(r, 24) : "r"(taddr));
}
#undef R32
// Waits for loads, these 32 among them: nothing that uses them may come in front.
#define R32(r, o) "+r"((r)[o]), "+r"((r)[o + 1]), "+r"((r)[o + 2]), "+r"((r)[o + 3]), "+r"((r)[o + 4]), "+r"((r)[o + 5]), "+r"((r)[o + 6]), "+r"((r)[o + 7])
__device__ __forceinline__ void tmem_ld_wait32(uint32_t* r) {
  asm volatile("tcgen05.wait::ld.sync.aligned;" : R32(r, 0), R32(r, 8), R32(r, 16), R32(r, 24) :: "memory");
}
__device__ __forceinline__ void tmem_ld_wait16(uint32_t* r) { asm volatile("tcgen05.wait::ld.sync.aligned;" : R32(r, 0), R32(r, 8) :: "memory"); }
__device__ __forceinline__ void tmem_ld_wait8(uint32_t* r) { asm volatile("tcgen05.wait::ld.sync.aligned;" : R32(r, 0) :: "memory"); }
#undef R32
#define R8(r, o) "r"((r)[o]), "r"((r)[o + 1]), "r"((r)[o + 2]), "r"((r)[o + 3]), "r"((r)[o + 4]), "r"((r)[o + 5]), "r"((r)[o + 6]), "r"((r)[o + 7])
__device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint32_t* r) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};"
               ::"r"(taddr), R8(r, 0), R8(r, 8) : "memory");
}
#undef R8
__device__ __forceinline__ void tmem_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ uint32_t pack_f16(float a, float b) {
  const __half2 v = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&v);
}
__device__ __forceinline__ uint32_t pack_bf16(float a, float b) {
  const __nv_bfloat162 v = __floats2bfloat162_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&v);
}
// two fp32 operations in one instruction
__device__ __forceinline__ uint64_t together(float a, float b) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ uint64_t two(float a) { return together(a, a); }
__device__ __forceinline__ void apart(uint64_t x, float& a, float& b) { asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(x)); }
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
// bits 0 .. x of 32
__device__ __forceinline__ uint32_t upto(int x) { return x < 0 ? 0u : x > 31 ? 0xffffffffu : 0xffffffffu >> (31 - x); }
__device__ __forceinline__ bool warp_wait(uint32_t bar, uint32_t parity, volatile int* quit) { return __all_sync(0xffffffffu, wait_or_quit(bar, parity, quit)); }

// kind::f16, f16 operands, fp32 accumulators, 128 rows by n columns; `tokens_first`: the second operand lies [k][n]
constexpr uint32_t idesc_f16(int n, bool tokens_first) { return (1u << 4) | (tokens_first ? 1u << 16 : 0u) | ((uint32_t)(n >> 3) << 17) | (8u << 24); }
// O += P V, 16 tokens: P in TMEM (8 columns of two f16), V [tokens][64 dims a half]: 8 tokens 1024 bytes on, the next 64 dims a half on
__device__ __forceinline__ void product_pv(uint32_t d, uint32_t p, uint32_t v_smem, uint32_t half, uint32_t idesc, uint32_t accumulate) {
  const uint64_t desc = (uint64_t)(((v_smem & 0x3FFFFu) >> 4) | ((half >> 4) << 16)) | (uint64_t)DESC_HIGH << 32;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}"
      ::"r"(d), "r"(p), "l"(desc), "r"(idesc), "r"(accumulate) : "memory");
}

}  // namespace paged
}  // namespace b200
