// Attention of many rows of a sequence over the paged 8-bit cache, on the 5th-generation tensor cores.
//
// A CTA owns one kv head and up to 256 rows (row of the sequence, query head of the group) as two tiles of 128, and walks the keys in tiles of 128 tokens.  Warps 8..14 bring the codes from memory
// through registers into f16 tiles (exact for both types) in SWIZZLE_128B, keys K-major and values as they lie, tokens by dims; warp 15 issues S_i = Q_i K^T and O_i += P_i V as
// tcgen05.mma with fp32 accumulators in TMEM (one place for the scores, O_0, O_1); warps 0..3 and 4..7 hold a row per thread, with all its 128 scores, and put P as f16 into TMEM,
// from where the second product reads it.  As soon as one tile's scores are in registers their place takes the other's.
//
// Scales as in paged.cu: that of a page's keys multiplies its 16 or more columns' scores, that of its values goes into the exponent.  O is rescaled only when a weight would pass 2^15.
//
// Bounds: the chain of a tile through its weight warps; the tensor pipe and the exponentials' unit are each active half the time (2048 rows on 6100 tokens, 32 heads on 8: 281 to 285 us, 0.84 PFLOP/s; a
// window of 1024 over 6000 rows of 16 heads on 4: 103 us).  The same statements in another order were up to 4 % slower.  A row's scores are read from TMEM once, and stay in 184 registers that setmaxnreg takes from the other warps
// (read twice, in 96, the first of these took 389 us when this took 365).
#include "paged.cuh"

#include <cfloat>

namespace b200 {
namespace paged {

namespace {

using namespace tcp;
typedef __nv_bfloat16 bf16;

constexpr int SOFT_WARPS = 8, CONVERT_WARPS = 7, THREADS = (SOFT_WARPS + CONVERT_WARPS + 1) * 32, ROWS = 256, KEYS = 128, INFOS = 8;

template <int D>
struct Smem {
  static constexpr uint32_t TILE = 128 * D * 2, HALF = 128 * 128;             // 128 rows of f16, in halves of 64 dims
  static constexpr uint32_t Q = 0, K = 2 * TILE, V = 4 * TILE, END = 6 * TILE, BYTES = END + 1024;
};

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
__device__ __forceinline__ uint32_t max2(uint32_t a, uint32_t b) {
  uint32_t r;
  asm("max.u16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}
// magnitudes of eight bf16: the largest of the even ones and that of the odd ones
__device__ __forceinline__ uint32_t largest8(const uint4& x) {
  constexpr uint32_t M = 0x7fff7fffu;
  return max2(max2(x.x & M, x.y & M), max2(x.z & M, x.w & M));
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

struct Unit {
  Seq q;
  int s, h, split, r0, rows, n_rows;         // first row of the unit, rows in it, rows of the sequence
  int pf, pl, t0, n;                         // first and last position; first tile and number of tiles of this range
};
__device__ __forceinline__ bool unit_of(const AttnP& p, Unit& u) {
  int x = (int)blockIdx.x;
  u.split = x % p.nsplit; x /= p.nsplit;
  u.h = x % p.H; x /= p.H;
  u.s = x % p.b.S;
  const int ct = p.q_tiles - 1 - x / p.b.S;  // the longest first
  u.q = sequence(p.b, u.s, p.P);
  if (!u.q.ok || u.q.n < p.from_rows) return false;
  u.n_rows = u.q.n * p.G;
  u.r0 = ct * ROWS;
  if (u.r0 >= u.n_rows) return false;
  u.rows = min(ROWS, u.n_rows - u.r0);
  u.pf = u.q.before + u.r0 / p.G;
  u.pl = u.q.before + (u.r0 + u.rows - 1) / p.G;
  const Tiles<7> tiles(u.pf, u.pl, p.window, p.sinks);
  const int per = (tiles.n + p.nsplit - 1) / p.nsplit;
  u.t0 = u.split * per;
  u.n = min(per, tiles.n - u.t0);
  return u.n > 0;
}

template <int D, int FMT>
__global__ void __launch_bounds__(THREADS, 1) prompt_kernel(const AttnP p) {
  typedef Smem<D> L;
  extern __shared__ uint8_t smem_raw[];
  __shared__ __align__(8) uint64_t bars[19 + INFOS];
  __shared__ float4 info[INFOS][8];          // per 16 keys: keys' scale, log2 and reciprocal of the values'; there: whether the page is
  __shared__ __align__(16) uint32_t there[INFOS][8];
  __shared__ uint32_t tmem_at;
  __shared__ volatile int quit;
  __shared__ float factors[ROWS];            // of a row: what turns a product of codes into a score in base 2, but for the keys' scale
  const uint32_t base = (smem_u32(smem_raw) + 1023u) & ~1023u;
  uint8_t* const smem = smem_raw + (base - smem_u32(smem_raw));
  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  const uint32_t bar = smem_u32(bars), k_full = bar, k_empty = bar + 16, v_full = bar + 32, v_empty = bar + 48, s_full = bar + 64, p_full = bar + 80, o_done = bar + 96, p_half = bar + 112, s_taken = bar + 128, q_full = bar + 144, i_full = bar + 152;
  if (threadIdx.x == 0) {
    quit = 0;
    for (int i = 0; i < 2; ++i) {
      mbar_init(k_full + 8 * i, 4); mbar_init(k_empty + 8 * i, 1); mbar_init(v_full + 8 * i, 4); mbar_init(v_empty + 8 * i, 1);
      mbar_init(s_full + 8 * i, 1); mbar_init(p_half + 8 * i, 4); mbar_init(s_taken + 8 * i, 4); mbar_init(p_full + 8 * i, 4); mbar_init(o_done + 8 * i, 1);
    }
    mbar_init(q_full, SOFT_WARPS);
    for (int i = 0; i < INFOS; ++i) mbar_init(i_full + 8 * i, 4);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  pdl_trigger();
  pdl_wait();
  if (blockIdx.x == 0)
    for (int i = threadIdx.x; i < p.b.S; i += THREADS)
      if (!sequence(p.b, i, p.P).ok) atomicOr(p.flags, B200_PAGED_BAD_BATCH);
  Unit u;
  if (!unit_of(p, u)) return;
  if (warp == SOFT_WARPS + CONVERT_WARPS) tmem_alloc(smem_u32(&tmem_at), 512);
  const int tiles_q = u.rows > 128 ? 2 : 1;
  const Tiles<7> tiles(u.pf, u.pl, p.window, p.sinks);

  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = tmem_at;
  const int n = u.n;

  // registers go to the warps that hold a row's scores: 8 x 184 + 8 x 72 = 16 x 128
  if (warp >= SOFT_WARPS) {
  asm volatile("setmaxnreg.dec.sync.aligned.u32 72;");
  if (warp < SOFT_WARPS + CONVERT_WARPS) {
    // ---- codes into f16 tiles: 32 tokens of a tile's keys or values at a time, eight such tasks a tile, which the warps take in turn ----
    constexpr int LANES = D / 16, STEP = 32 / LANES, LOADS = 32 / STEP;       // lanes a row, rows a load, loads
    const int row = lane / LANES, c = lane % LANES;
    // lanes of a row's second 64 dims take the neighbouring row, so that eight lanes' pieces of the f16 tile lie in different banks
    const int r_in = row ^ (D == 128 ? c >> 2 : 0);
    const int tasks = 8 * n;
    uint4 held[LOADS];                       // of the task to come
    float2 scales = make_float2(0.f, 1.f);   // of its pages: lane l has the one of token (l & 1) * 16
    auto look_up = [&](int task) {
      if (task >= tasks) return -1;
      const int j = (tiles[u.t0 + (task >> 3)] << 7) + 32 * (task & 3) + 16 * (lane & 1);
      int page = -1;
      if (j <= u.pl && (p.window <= 0 || u.pf - j - 15 < p.window || j < p.sinks)) {
        page = p.b.table[u.s * p.b.table_ld + (j >> p.page_shift)];
        if (page < 0 || page >= p.pages) { page = -1; atomicOr(p.flags, B200_PAGED_BAD_PAGE); }
      }
      return page;
    };
    auto load = [&](int task, int page) {
      if (task >= tasks) return;
      const bool keys = !(task & 4);
      const uint8_t* codes = keys ? p.k : p.v;
      const int j0 = (tiles[u.t0 + (task >> 3)] << 7) + 32 * (task & 3);
      if (keys && page >= 0) scales = make_float2(p.k_scale[(long long)page * p.H + u.h], p.v_scale[(long long)page * p.H + u.h]);
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        const int pg = __shfl_sync(0xffffffffu, page, half), j1 = j0 + 16 * half;
        const uint8_t* from = codes + (((long long)pg * p.H + u.h) * p.P + (j1 & (p.P - 1)) + r_in) * D + 16 * c;
        // values that no row sees may be anything; keys are masked
        const bool all = keys || (j1 + 15 <= u.pl && (p.window <= 0 || u.pf - j1 < p.window || j1 + 16 <= p.sinks));
#pragma unroll
        for (int x = 0; x < LOADS / 2; ++x) {
          const int j = j1 + x * STEP + r_in;
          const bool seen = pg >= 0 && (all || (j <= u.pl && (p.window <= 0 || u.pf - j < p.window || j < p.sinks)));
          held[half * (LOADS / 2) + x] = seen ? *reinterpret_cast<const uint4*>(from + x * STEP * D) : make_uint4(0, 0, 0, 0);
        }
      }
    };
    int task = warp - SOFT_WARPS, page = look_up(task), page_next = look_up(task + CONVERT_WARPS);
    load(task, page);
    for (; task < tasks; task += CONVERT_WARPS) {
      const int i = task >> 3, st = i & 1, w4 = task & 3;
      const bool keys = !(task & 4);
      if (keys) {                            // what the weights need to know of these keys' pages
        if (lane < 2) {
          const float vs = value_scale(scales.y);
          there[i % INFOS][2 * w4 + lane] = page >= 0 ? 1u : 0u;
          info[i % INFOS][2 * w4 + lane] = page >= 0 ? make_float4(scales.x > 0.f ? scales.x : 1.f, __log2f(vs), __frcp_rn(vs), 0.f) : make_float4(1.f, 0.f, 0.f, 0.f);
        }
        __syncwarp();
      }
      if (!warp_wait((keys ? k_empty : v_empty) + 8 * st, ((uint32_t)(i >> 1) & 1u) ^ 1u, &quit)) break;
      if (keys && lane == 0) mbar_arrive(i_full + 8 * (i % INFOS));
      uint8_t* const dst = smem + (keys ? L::K : L::V) + st * L::TILE + (c >> 2) * L::HALF;
#pragma unroll
      for (int x = 0; x < LOADS; ++x) {
        const int t = 32 * w4 + x * STEP + r_in;
        const uint32_t w[4] = {ready<FMT>(held[x].x), ready<FMT>(held[x].y), ready<FMT>(held[x].z), ready<FMT>(held[x].w)};
        uint8_t* r = dst + t * 128;
        *reinterpret_cast<uint4*>(r + (((2 * (c & 3)) ^ (t & 7)) << 4)) = make_uint4(half2_of<FMT, 0>(w[0]), half2_of<FMT, 1>(w[0]), half2_of<FMT, 0>(w[1]), half2_of<FMT, 1>(w[1]));
        *reinterpret_cast<uint4*>(r + (((2 * (c & 3) + 1) ^ (t & 7)) << 4)) = make_uint4(half2_of<FMT, 0>(w[2]), half2_of<FMT, 1>(w[2]), half2_of<FMT, 0>(w[3]), half2_of<FMT, 1>(w[3]));
      }
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      __syncwarp();
      if (lane == 0) mbar_arrive((keys ? k_full : v_full) + 8 * st);
      page = page_next;
      load(task + CONVERT_WARPS, page);
      page_next = look_up(task + 2 * CONVERT_WARPS);
    }
  } else {
    // ---- products ----
    constexpr uint32_t id_s = idesc_f16(KEYS, false), id_o = idesc_f16(D, true);
    auto scores = [&](int i, int x) {        // of tile x for queries i
      const uint32_t a = desc_low(base + L::Q + i * L::TILE), b = desc_low(base + L::K + (x & 1) * L::TILE);
      tc_fence_after();
#pragma unroll
      for (int half = 0; half < D / 64; ++half) umma_block<1>(tmem, a + half * (L::HALF >> 4), b - a, id_s, half > 0 ? 1u : 0u);
      commit_elected(s_full + 8 * i);
      if (i == tiles_q - 1) commit_elected(k_empty + 8 * (x & 1));
    };
    auto sums = [&](int i, int x) {          // over tile x for queries i, half of the keys behind the other: the second half's weights are made beside the first's product
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        if (!warp_wait((half ? p_full : p_half) + 8 * i, (uint32_t)x & 1u, &quit)) return false;
        tc_fence_after();
        if (elected()) {
#pragma unroll
          for (int k = half * KEYS / 32; k < (half + 1) * KEYS / 32; ++k)
            product_pv(tmem + 256 + 128 * i, tmem + 128 + 64 * i + 8 * k, base + L::V + (x & 1) * L::TILE + k * 2048, L::HALF, id_o, x > 0 || k > 0 ? 1u : 0u);
        }
        __syncwarp();
      }
      commit_elected(o_done + 8 * i);
      if (i == tiles_q - 1) commit_elected(v_empty + 8 * (x & 1));
      return true;
    };
    auto v_there = [&](int x) { return warp_wait(v_full + 8 * (x & 1), (uint32_t)(x >> 1) & 1u, &quit); };
    // The scores' place is free as soon as a tile's weight warps have them in registers, and then takes the other tile's: the next scores of a tile are made while its weights still are.
    // In turn: scores of 1, sum of 1 over the keys in front, scores of 0 over the next keys, sum of 0.
    bool ok = warp_wait(q_full, 0, &quit) && warp_wait(k_full, 0, &quit);
    if (ok) scores(0, 0);
    for (int x = 0; ok && x < n; ++x) {
      ok = warp_wait(s_taken, (uint32_t)x & 1u, &quit);
      if (tiles_q > 1) {
        if (ok) scores(1, x);
        if (x > 0) ok = ok && sums(1, x - 1);
        ok = ok && warp_wait(s_taken + 8, (uint32_t)x & 1u, &quit);
      }
      if (x + 1 < n) {
        ok = ok && warp_wait(k_full + 8 * ((x + 1) & 1), (uint32_t)((x + 1) >> 1) & 1u, &quit);
        if (ok) scores(0, x + 1);
      }
      ok = ok && v_there(x) && sums(0, x);
    }
    if (tiles_q > 1) ok = ok && sums(1, n - 1);
    __syncwarp();
  }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 184;");
    // ---- queries: f16 after a power of two for each row, as rows and heads of very different size may lie side by side ----
    constexpr int PIECES = D / 8, MINE = 2 * 128 * PIECES / (SOFT_WARPS * 32);          // 16-byte pieces of a row, and of this thread
    {
      uint4 raw[MINE];
      // the thread has piece c of every APART-th row from `at` on; token and head of a row by counting, not by division
      constexpr int APART = SOFT_WARPS * 32 / PIECES;
      const int c = threadIdx.x % PIECES, at = threadIdx.x / PIECES, step_i = APART / p.G, step_g = APART - step_i * p.G;
      int i = (u.r0 + at) / p.G, g = u.r0 + at - i * p.G;
      const bf16* const q0 = p.q + (long long)u.q.r0 * p.q_ld + (long long)u.h * p.G * D + c * 8;
#pragma unroll
      for (int k = 0; k < MINE; ++k) {
        raw[k] = at + k * APART < u.rows ? *reinterpret_cast<const uint4*>(q0 + i * p.q_ld + g * D) : make_uint4(0, 0, 0, 0);
        i += step_i; g += step_g;
        if (g >= p.G) { g -= p.G; ++i; }
      }
      // magnitudes as 16-bit numbers, which order like the values; two rows a word, k and k + MINE / 2
      uint32_t top[MINE / 2];
#pragma unroll
      for (int k = 0; k < MINE / 2; ++k) {
        const uint32_t a = largest8(raw[k]), b = largest8(raw[k + MINE / 2]);
        top[k] = max2(prmt(a, b, 0x5410u), prmt(a, b, 0x7632u));
      }
      // The lanes of a row have as many rows as they are: each step halves the rows that a lane answers for, until lane c has the c-th one's.
      static_assert(MINE == PIECES, "a row's lanes share its rows out");
#pragma unroll
      for (int h = MINE / 4; h > 0; h /= 2)
#pragma unroll
        for (int k = 0; k < h; ++k) {
          const bool upper = lane & h;
          const uint32_t theirs = __shfl_xor_sync(0xffffffffu, upper ? top[k] : top[k + h], h);
          top[k] = max2(upper ? top[k + h] : top[k], theirs);
        }
      top[0] = max2(top[0], __shfl_xor_sync(0xffffffffu, top[0], MINE / 2));
      const uint32_t largest = lane & MINE / 2 ? top[0] & 0xffff0000u : top[0] << 16;
      // A row that is not finite gets NaN, and no other: it asks as zeros, whose weights say whether it sees anything at all, and its factor tells the end of it.
      const bool odd = largest >= 0x7f800000u;
      const float power = largest ? power_of_two_in(__uint_as_float(largest)) : 1.f;
      const float up_mine = __uint_as_float((268u << 23) - __float_as_uint(power));            // 2^14 / power
      factors[at + c * APART] = odd ? NAN : power * (1.f / 16384.f) * p.scale2;
      if (__any_sync(0xffffffffu, odd)) {
#pragma unroll
        for (int k = 0; k < MINE; ++k)
          if (__shfl_sync(0xffffffffu, odd, k, PIECES)) raw[k] = make_uint4(0, 0, 0, 0);
      }
      asm volatile("bar.sync 1, %0;" ::"n"(SOFT_WARPS * 32) : "memory");      // all rows' factors
#pragma unroll
      for (int k = 0; k < MINE; ++k) {
        const int r = at + k * APART;
        const float up = __shfl_sync(0xffffffffu, up_mine, k, PIECES);
        const uint32_t v[4] = {raw[k].x, raw[k].y, raw[k].z, raw[k].w};
        uint32_t o[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) o[i] = pack_f16(__uint_as_float(v[i] << 16) * up, __uint_as_float(v[i] & 0xffff0000u) * up);
        *reinterpret_cast<uint4*>(smem + L::Q + (r >> 7) * L::TILE + (c >> 3) * L::HALF + (r & 127) * 128 + (((c & 7) ^ (r & 7)) << 4)) = make_uint4(o[0], o[1], o[2], o[3]);
      }
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      __syncwarp();
      if (lane == 0) mbar_arrive(q_full);
    }
    if ((warp >> 2) < tiles_q) {
    // ---- weights: a row per thread ----
    const int i = warp >> 2, q4 = warp & 3, row = 128 * i + q4 * 32 + lane, rr = u.r0 + row;
    const bool has = row < u.rows;
    const int pos = has ? u.q.before + rr / p.G : -1, lo = p.window > 0 ? pos - p.window : -1;      // sees j <= pos, j > lo or j < sinks
    const int pf = u.q.before + (u.r0 + 128 * i) / p.G, pl = u.q.before + (u.r0 + min(128 * i + 128, u.rows) - 1) / p.G;      // of this tile of queries
    const uint32_t lanes = (uint32_t)(q4 * 32) << 16, ts = tmem + lanes, tp = tmem + lanes + 128 + 64 * i, to = tmem + lanes + 256 + 128 * i;
    const float fac = factors[row];
    float m = -INFINITY, sum = 0.f;
    bool ok = true;
    for (int x = 0; x < n; ++x) {
      ok = wait_or_quit(i_full + 8 * (x % INFOS), (uint32_t)(x / INFOS) & 1u, &quit) && wait_or_quit(s_full + 8 * i, (uint32_t)x & 1u, &quit);
      if (!__all_sync(0xffffffffu, ok)) { ok = false; break; }
      tc_fence_after();
      const int j0 = tiles[u.t0 + x] << 7;
      const float4* ip = info[x % INFOS];
      const uint4 t0 = *reinterpret_cast<const uint4*>(there[x % INFOS]), t1 = *reinterpret_cast<const uint4*>(there[x % INFOS] + 4);
      const bool whole = ((t0.x & t0.y & t0.z & t0.w & t1.x & t1.y & t1.z & t1.w) != 0u) & (j0 + KEYS - 1 <= pf) & ((p.window <= 0) | (pl - j0 < p.window) | (j0 + KEYS <= p.sinks));
      uint32_t r[KEYS];                      // the row's scores: read once, as the registers have room for them
      float t = -INFINITY, by[8], lv[8];     // score in base 2 = product * by + lv; by > 0, so that the largest score of a page's keys is that of their largest product
      tmem_ld32(ts, r);
      tmem_ld_wait32(r);
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        if (c < 3) tmem_ld32(ts + 32 * c + 32, r + 32 * c + 32);
        if (!whole) {                        // keys that the row does not see: a bit for each of 32
          const int at = j0 + 32 * c;
          uint32_t seen = upto(pos - at) & (~upto(lo - at) | upto(p.sinks - 1 - at));
          if (!there[x % INFOS][2 * c]) seen &= 0xffff0000u;
          if (!there[x % INFOS][2 * c + 1]) seen &= 0xffffu;
#pragma unroll
          for (int e = 0; e < 32; ++e)
            if (!(seen >> e & 1u)) r[32 * c + e] = 0xff800000u;
        }
#pragma unroll
        for (int b = 2 * c; b < 2 * c + 2; ++b) {
          by[b] = fmaxf(ip[b].x * fac, FLT_MIN);                              // also where fac is NaN
          lv[b] = ip[b].y;
          float mx[2] = {__uint_as_float(r[16 * b]), __uint_as_float(r[16 * b + 1])};
#pragma unroll
          for (int e = 2; e < 16; ++e) mx[e & 1] = fmaxf(mx[e & 1], __uint_as_float(r[16 * b + e]));
          t = fmaxf(t, fmaf(fmaxf(mx[0], mx[1]), by[b], lv[b]));
        }
        if (c < 3) tmem_ld_wait32(r + 32 * c + 32);
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(s_taken + 8 * i);
      const bool grow = t > __fadd_rd(m, SLACK);       // rounded down: above 2^27 the sum would else round to the score itself, and its weight to infinity
      if (x > 0) {                           // the sum over the keys in front has read its weights and settled in O
        ok = wait_or_quit(o_done + 8 * i, (uint32_t)(x - 1) & 1u, &quit);
        if (!__all_sync(0xffffffffu, ok)) { ok = false; break; }
        tc_fence_after();
      }
      if (__any_sync(0xffffffffu, grow)) {
        const float now = t - UNDER, factor = grow ? exp2_fast(m - now) : 1.f;
        if (grow) { m = now; sum *= factor; }
        if (x > 0) {
#pragma unroll
          for (int c = 0; c < D / 16; ++c) {
            uint32_t o[16];
            tmem_ld16(to + 16 * c, o);
            tmem_ld_wait16(o);
#pragma unroll
            for (int e = 0; e < 16; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * factor);
            tmem_st16(to + 16 * c, o);
          }
        }
      }
      const float off = m == -INFINITY ? 0.f : m;
      // log2 s_v - M in one number is off by half a unit of M: only while that is no more than a quarter
      if (__any_sync(0xffffffffu, fabsf(off) > 4194304.f && off < INFINITY)) {
#pragma unroll
        for (int e = 0; e < KEYS; ++e) r[e] = __float_as_uint(fmaf(__uint_as_float(r[e]), by[e / 16], lv[e / 16]));
#pragma unroll
        for (int b = 0; b < 8; ++b) { by[b] = 1.f; lv[b] = 0.f; }
      }
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        uint32_t w[16];
#pragma unroll
        for (int b = 2 * c; b < 2 * c + 2; ++b) {
          const uint64_t by2 = two(by[b]), add = two(lv[b] - off);
          uint64_t part = 0;
#pragma unroll
          for (int e = 0; e < 16; e += 2) {
            float e0, e1;
            apart(fma2(together(__uint_as_float(r[16 * b + e]), __uint_as_float(r[16 * b + e + 1])), by2, add), e0, e1);
            e0 = exp2_fast(e0); e1 = exp2_fast(e1);
            part = add2(part, together(e0, e1));
            w[8 * (b & 1) + (e >> 1)] = pack_f16(e0, e1);
          }
          float s0, s1;
          apart(part, s0, s1);
          sum = fmaf(s0 + s1, ip[b].z, sum);
        }
        tmem_st16(tp + 16 * c, w);
        if (c & 1) {
          tmem_st_wait();
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive((c == 1 ? p_half : p_full) + 8 * i);
        }
      }
    }
    if (ok) {
      ok = wait_or_quit(o_done + 8 * i, (uint32_t)(n - 1) & 1u, &quit);
      ok = __all_sync(0xffffffffu, ok);
    }
    if (ok) {
      tc_fence_after();
      if (sum != 0.f && isnan(factors[row])) sum = NAN;
      const float inv = sum != 0.f ? 1.f / sum : 0.f;
      if (p.nsplit > 1) {
        const long long at = (long long)blockIdx.x * ROWS + row;
        if (has) *reinterpret_cast<float2*>(p.part_ml + 2 * at) = make_float2(m, sum);
#pragma unroll
        for (int c = 0; c < D / 32; ++c) {
          uint32_t o[32];
          __syncwarp();
          tmem_ld32(to + 32 * c, o);
          tmem_ld_wait32(o);
          if (has) {
#pragma unroll
            for (int e = 0; e < 32; e += 4) *reinterpret_cast<uint4*>(p.part_o + at * D + 32 * c + e) = make_uint4(o[e], o[e + 1], o[e + 2], o[e + 3]);
          }
        }
      } else {
        // through the queries' place, which nobody reads any more: whole rows go out, and not 16 bytes of 32 rows at a time
        uint8_t* const mine = smem + L::Q + (i * 4 + q4) * (32 * D * 2);
#pragma unroll
        for (int c = 0; c < D / 32; ++c) {
          uint32_t o[32];
          tmem_ld32(to + 32 * c, o);
          tmem_ld_wait32(o);
#pragma unroll
          for (int e = 0; e < 32; e += 8) {
            uint4 v;
            v.x = pack_bf16(__uint_as_float(o[e]) * inv, __uint_as_float(o[e + 1]) * inv);
            v.y = pack_bf16(__uint_as_float(o[e + 2]) * inv, __uint_as_float(o[e + 3]) * inv);
            v.z = pack_bf16(__uint_as_float(o[e + 4]) * inv, __uint_as_float(o[e + 5]) * inv);
            v.w = pack_bf16(__uint_as_float(o[e + 6]) * inv, __uint_as_float(o[e + 7]) * inv);
            const int piece = 4 * c + e / 8;
            *reinterpret_cast<uint4*>(mine + lane * D * 2 + ((piece ^ (lane & 7)) << 4)) = v;
          }
        }
        __syncwarp();
        constexpr int AT_ONCE = 32 / PIECES;
        const int c = lane % PIECES;
        bf16* const out0 = p.out + (long long)u.q.r0 * p.out_ld + (long long)u.h * p.G * D + c * 8;
#pragma unroll 4
        for (int k = 0; k < 32; k += AT_ONCE) {
          const int r = k + lane / PIECES, x = u.r0 + 128 * i + 32 * q4 + r, token = x / p.G;
          if (128 * i + 32 * q4 + r < u.rows)
            *reinterpret_cast<uint4*>(out0 + token * p.out_ld + (x - token * p.G) * D) = *reinterpret_cast<const uint4*>(mine + r * D * 2 + ((c ^ (r & 7)) << 4));
        }
      }
      tc_fence_before();
    }
    }
  }
  __syncthreads();
  tc_fence_after();
  if (warp == SOFT_WARPS + CONVERT_WARPS) tmem_dealloc(tmem, 512);
  if (threadIdx.x == 0 && quit) atomicOr(p.flags, B200_PAGED_WAIT);
}

// Joins the ranges of the keys: 16 threads a row.
template <int D>
__global__ void __launch_bounds__(128) prompt_join_kernel(const AttnP p) {
  pdl_trigger();
  pdl_wait();
  constexpr int PER = D / 16;
  const long long x = (long long)blockIdx.x * 8 + (threadIdx.x >> 4);
  const int row = (int)(x % ROWS), d0 = (threadIdx.x & 15) * PER;
  int unit = (int)(x / ROWS);
  const long long first = (long long)unit * p.nsplit * ROWS + row;
  const int h = unit % p.H; unit /= p.H;
  const int s = unit % p.b.S, ct = p.q_tiles - 1 - unit / p.b.S, rr = ct * ROWS + row;
  const Seq q = sequence(p.b, s, p.P);
  if (!q.ok || q.n < p.from_rows || rr >= q.n * p.G) return;
  const int rows = min(ROWS, q.n * p.G - ct * ROWS);
  const Tiles<7> tiles(q.before + ct * ROWS / p.G, q.before + (ct * ROWS + rows - 1) / p.G, p.window, p.sinks);
  const int per = (tiles.n + p.nsplit - 1) / p.nsplit, parts = (tiles.n + per - 1) / per;
  const float2* ml = reinterpret_cast<const float2*>(p.part_ml);
  float top = -INFINITY, sum = 0.f, acc[PER];
  for (int i = 0; i < parts; ++i) top = fmaxf(top, ml[first + (long long)i * ROWS].x);
#pragma unroll
  for (int e = 0; e < PER; ++e) acc[e] = 0.f;
  for (int i = 0; i < parts; ++i) {
    const float2 y = ml[first + (long long)i * ROWS];
    const float by = y.x == -INFINITY ? 0.f : exp2_fast(y.x - top);
    sum = fmaf(y.y, by, sum);
    const float4* o = reinterpret_cast<const float4*>(p.part_o + (first + (long long)i * ROWS) * D + d0);
#pragma unroll
    for (int e = 0; e < PER / 4; ++e) {
      const float4 v = o[e];
      acc[4 * e] = fmaf(v.x, by, acc[4 * e]); acc[4 * e + 1] = fmaf(v.y, by, acc[4 * e + 1]);
      acc[4 * e + 2] = fmaf(v.z, by, acc[4 * e + 2]); acc[4 * e + 3] = fmaf(v.w, by, acc[4 * e + 3]);
    }
  }
  const float by = sum != 0.f ? 1.f / sum : 0.f;
  const int token = rr / p.G;
  bf16* out = p.out + (long long)(q.r0 + token) * p.out_ld + (long long)(h * p.G + rr - token * p.G) * D + d0;
#pragma unroll
  for (int e = 0; e < PER; e += 4) *reinterpret_cast<uint2*>(out + e) = make_uint2(pack_bf16(acc[e] * by, acc[e + 1] * by), pack_bf16(acc[e + 2] * by, acc[e + 3] * by));
}

template <int D, int FMT>
int launch(const AttnP& p, long long units, cudaStream_t st) {
  static std::atomic<uint64_t> limits{0};
  static std::atomic<uint64_t> shares{0};
  B200_TRY(allow_smem(limits, (int)Smem<D>::BYTES, prompt_kernel<D, FMT>));
  B200_TRY(prefer_smem(shares, 100, prompt_kernel<D, FMT>, prompt_join_kernel<D>));
  B200_TRY(launch_early(prompt_kernel<D, FMT>, dim3((unsigned)(units * p.nsplit)), dim3(THREADS), Smem<D>::BYTES, st, p));
  if (p.nsplit > 1) B200_TRY(launch_early(prompt_join_kernel<D>, dim3((unsigned)(units * (ROWS / 8))), dim3(128), 0, st, p));
  return B200_OK;
}

}  // namespace

PromptPlan prompt_plan(const b200_paged_cache* c, const b200_paged_batch* b, int G, int window, int sinks) {
  PromptPlan f;
  f.q_tiles = (int)ceil_div64((long long)b->max_rows * G, ROWS);
  f.units = (long long)b->sequences * c->kv_heads * f.q_tiles;
  long long keys = (long long)b->table_width * c->page_tokens;
  if (window > 0 && (long long)window + sinks + ROWS / G < keys) keys = (long long)window + sinks + ROWS / G;
  const long long tiles = ceil_div64(keys, KEYS);
  long long n = f.units ? 148 / f.units : 1;
  if (n > tiles / 2) n = tiles / 2;          // ranges of two tiles at least
  f.nsplit = n < 1 ? 1 : (int)n;
  return f;
}
int64_t prompt_bytes(const PromptPlan& f, int D) { return f.nsplit > 1 ? f.units * f.nsplit * ROWS * (D + 2) * 4 : 0; }

int prompt_attention(const AttnP& p, const PromptPlan& f, int fmt, int dim, cudaStream_t st) {
  if (dim == 128) return fmt == INT8 ? launch<128, INT8>(p, f.units, st) : launch<128, E4M3>(p, f.units, st);
  return fmt == INT8 ? launch<64, INT8>(p, f.units, st) : launch<64, E4M3>(p, f.units, st);
}

}  // namespace paged
}  // namespace b200
