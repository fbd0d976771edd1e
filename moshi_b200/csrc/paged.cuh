// What the kernels of the paged 8-bit cache share (paged.cu: append, read, attention of few rows; paged_prompt.cu: attention of many rows of a sequence).
#pragma once

#include <cuda.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>

#include "common.cuh"
#include "tc_prims.cuh"

namespace b200 {
namespace paged {

constexpr int INT8 = 0, E4M3 = 1;            // template arguments; B200_KV_INT8 / B200_KV_FP8_E4M3 at the entry points
constexpr float LOG2E = 1.4426950408889634f;
constexpr float SCALE_MIN = 8.673617379884035e-19f;      // 2^-60, the least scale of a page
constexpr float MAGNITUDE = 1.8446744073709552e19f;      // 2^64, the largest magnitude that is stored

// ---- the step's sequences, as device memory has them: nothing is believed before it is checked ----
struct Batch {
  const int32_t *table, *before, *rows;
  long long table_ld;
  int S, T, width, max_rows;
};
struct Seq { int r0, n, before; bool ok; };
__device__ __forceinline__ Seq sequence(const Batch& b, int s, int P) {
  Seq q;
  q.r0 = b.rows[s];
  const int r1 = b.rows[s + 1];
  q.before = b.before[s];
  q.ok = q.r0 >= 0 && r1 >= q.r0 && r1 <= b.T && q.before >= 0 && r1 - q.r0 <= b.max_rows && (long long)q.before + (r1 - q.r0) <= (long long)b.width * P;
  q.n = r1 - q.r0;
  return q;
}
// The sequence that row r belongs to, S if there is none; the whole warp asks together (one load latency, where a binary search has seven for 128 sequences).  Of rows that do not rise it may be one
// that does not have row r: has_row says so, and a position is asked for behind it only, as that is what sequence() has bounded.
__device__ __forceinline__ int sequence_of_row(const Batch& b, int r) {
  int s = 0;
  for (int i = threadIdx.x & 31; i - (int)(threadIdx.x & 31) < b.S; i += 32) s += __popc(__ballot_sync(0xffffffffu, i < b.S && b.rows[i + 1] <= r));
  return r < b.rows[0] ? b.S : s;
}
__device__ __forceinline__ bool has_row(const Seq& q, int r) { return q.ok && r >= q.r0 && r - q.r0 < q.n; }
// One block of every call looks at all sequences: those that are left out are recorded, whether or not they have rows or pages that another block comes across.
__device__ __forceinline__ void record_sequences(const Batch& b, int P, int32_t* flags, int threads) {
  for (int s = threadIdx.x; s < b.S; s += threads)
    if (!sequence(b, s, P).ok) atomicOr(flags, B200_PAGED_BAD_BATCH);
}

// ---- codes ----
__device__ __forceinline__ uint32_t prmt(uint32_t a, uint32_t b, uint32_t sel) {
  uint32_t r;
  asm("prmt.b32 %0, %1, %2, %3;" : "=r"(r) : "r"(a), "r"(b), "r"(sel));
  return r;
}
// Two codes (bytes 2 * HI, 2 * HI + 1 of a word) as f16, exactly.  int8: the byte with its sign bit flipped is the mantissa of 1024 + 128 + code; words of int8
// go through ready() first.
template <int FMT>
__device__ __forceinline__ uint32_t ready(uint32_t w) { return FMT == INT8 ? w ^ 0x80808080u : w; }
template <int FMT, int HI>
__device__ __forceinline__ uint32_t half2_of(uint32_t w) {
  if constexpr (FMT == INT8) {
    const uint32_t u = prmt(w, 0x64646464u, HI ? 0x4342u : 0x4140u);
    const __half2 v = __hsub2(*reinterpret_cast<const __half2*>(&u), __half2half2(__ushort_as_half(0x6480)));
    return *reinterpret_cast<const uint32_t*>(&v);
  } else {
    uint32_t r;
    const uint16_t x = (uint16_t)(HI ? w >> 16 : w);
    asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(r) : "h"(x));
    return r;
  }
}
template <int FMT, int HI>
__device__ __forceinline__ float2 float2_of(uint32_t w) {
  const uint32_t r = half2_of<FMT, HI>(w);
  return __half22float2(*reinterpret_cast<const __half2*>(&r));
}
template <int FMT>
__device__ constexpr float code_max() { return FMT == INT8 ? 127.f : 448.f; }
// four values that are already divided by their scale -> four codes, each off by half a step at most
template <int FMT>
__device__ __forceinline__ uint32_t codes4(float a, float b, float c, float d) {
  if constexpr (FMT == INT8) {
    // to the nearest whole number, ties to the even one: the sum with 1.5 * 2^23 has it in its last bits
    auto one = [](float x) { return __float_as_uint(fminf(fmaxf(x, -127.f), 127.f) + 12582912.f); };
    return prmt(prmt(one(a), one(b), 0x0040u), prmt(one(c), one(d), 0x0040u), 0x5410u);
  } else {
    return (uint32_t)__nv_cvt_float2_to_fp8x2(make_float2(a, b), __NV_SATFINITE, __NV_E4M3) | (uint32_t)__nv_cvt_float2_to_fp8x2(make_float2(c, d), __NV_SATFINITE, __NV_E4M3) << 16;
  }
}

__device__ __forceinline__ float exp2_fast(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
// the greatest power of two in x > 0, but 2^-100 at least, so that 2^14 / it is a float
__device__ __forceinline__ float power_of_two_in(float x) { return __uint_as_float(max(__float_as_uint(x) & 0x7f800000u, (127u - 100u) << 23)); }

// ---- attention ----
// What a page's values count as in the exponent.  A page of zeros has the scale 0 and adds nothing to the sums but its share of the weights' total: it counts as the least scale, so that the running maximum,
// which is of score + log2(scale), stays that of the pages that have something to add.
__device__ __forceinline__ float value_scale(float s) { return s > 0.f ? s : SCALE_MIN; }
// Weights are P = 2^(score + log2(value scale) - M) in f16, whose numbers go from 2^-24 to 65504.  M is set 2^UNDER below the largest exponent and follows when one passes it by 2^SLACK: P reaches 2^15, and
// a weight (times its value's scale) is off by 2^-11 of itself or, under 2^-21 of the largest one, by 2^-32 of that.  exp2 ends at 2^-126: of pages whose value scales lie as far apart as 2^118, the whole
// range that scales have, the lower ones' weights count in the total down to 2^-15 of the largest.
constexpr float UNDER = 7.f, SLACK = 15.f;
struct AttnP {
  const uint8_t *k, *v;
  const float *k_scale, *v_scale;
  int32_t* flags;
  Batch b;
  const __nv_bfloat16* q;
  __nv_bfloat16* out;
  long long q_ld, out_ld;
  int pages, P, page_shift, H, G;            // tokens of a page = 1 << page_shift; kv heads; query heads of each
  int window, sinks;
  float scale2;                              // score scale * log2(e)
  // few rows
  int direct;                                // a CTA per unit
  float *part_o, *part_ml;                   // [CTAs][2][columns][D], [CTAs][2][columns][2]
  int2* parts;                               // [sequences][H]: first CTA and number of further ones of a unit
  // many rows
  int from_rows;                             // sequences of at least this many rows
  int q_tiles, nsplit;                       // units of a sequence and kv head; ranges of the keys
};

// Keys that the rows of positions pf .. pl see, in tiles of 1 << SHIFT tokens: `first` tiles from token 0 on (those of the sinks), then those from tile `from` on.
template <int SHIFT>
struct Tiles {
  int first, from, n;
  __device__ __forceinline__ Tiles(int pf, int pl, int window, int sinks) {
    const int begin = window > 0 ? max(0, pf + 1 - window) : 0;
    first = (min(sinks, begin) + (1 << SHIFT) - 1) >> SHIFT;
    from = max(begin >> SHIFT, first);
    n = first + (pl >> SHIFT) + 1 - from;
  }
  __device__ __forceinline__ int operator[](int i) const { return i < first ? i : from + i - first; }
};
__device__ __forceinline__ bool sees(int p, int j, int window, int sinks) { return j <= p && (window <= 0 || p - j < window || j < sinks); }

// A wait of ten seconds at most; `quit`: somebody of the block has waited that long, and nobody waits any more.
__device__ __forceinline__ bool wait_or_quit(uint32_t bar, uint32_t parity, volatile int* quit) {
  uint32_t done, spins = 0;
  uint64_t t0 = 0;
  for (;;) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(done) : "r"(bar), "r"(parity) : "memory");
    if (done) return true;
    if ((++spins & 1023u) == 0u) {
      if (*quit) return false;
      const uint64_t now = tcp::global_timer_ns();
      if (t0 == 0) t0 = now;
      else if (now - t0 > tcp::WAIT_LIMIT_NS) { *quit = 1; return false; }
    }
  }
}
// paged_prompt.cu
struct PromptPlan { int q_tiles, nsplit; long long units; };
PromptPlan prompt_plan(const b200_paged_cache* c, const b200_paged_batch* b, int G, int window, int sinks);
int64_t prompt_bytes(const PromptPlan& f, int D);
int prompt_attention(const AttnP& p, const PromptPlan& f, int fmt, int dim, cudaStream_t st);

}  // namespace paged
}  // namespace b200
