// Attention of trees of drafted tokens over the paged 8-bit cache: a row sees what its sequence has cached in front of the step, and of the step's own tokens itself and those that it comes behind.
//
// Columns are (row of the sequence, query head of the group).  A unit is C = 32, 64 or 128 of them with one kv head, and a CTA walks its keys in tiles of 128 tokens.  The tensor cores' tiles have 128 rows,
// and a tree has 20 to 100 columns as often as not: the rows are R = 128 / C copies of the columns, of which each weighs C of a tile's 128 keys.  So all threads of the weights have work whatever C is, with a
// running maximum of their own; the products of a copy's rows with the other copies' keys are thrown away (scores) or made of zeros (P is block-diagonal, and the zeros are written once).  Tiles go to
// two groups of weight warps in turn, with a sum O of each, so that the scores of one tile, the weights of another and the sum over a third are made at the same time.  At a unit's end its 2 R sums
// are joined through shared memory.
//
// Units lie one behind the other and are cut into equal runs, one per CTA, as in paged.cu.  Codes, scales, f16 tiles and the lazy maximum are those of paged_prompt.cu.
#include "paged_tc.cuh"

#include <cfloat>

namespace b200 {
namespace paged {

namespace {

typedef __nv_bfloat16 bf16;

// =========================================================================================================================
// the tree
// =========================================================================================================================
constexpr int MAX_NODES = 1024;              // of a sequence

struct BuildP {
  Batch b;
  const int32_t* parents;
  uint32_t* seen;                            // [rows][words]
  int32_t* position;
  int32_t* flags;
  int words;
};
// A block per sequence, a thread per token: from parent to parent through shared memory, a word of the mask at a time.  Parents have lower numbers, so the words come in falling order.
__global__ void __launch_bounds__(128) tree_build_kernel(const BuildP p) {
  pdl_trigger();
  pdl_wait();
  __shared__ int16_t parent[MAX_NODES];
  const int s = (int)blockIdx.x, r0 = p.b.rows[s], r1 = p.b.rows[s + 1], before = p.b.before[s];
  if (r0 < 0 || r1 < r0 || r1 > p.b.T || before < 0 || r1 - r0 > p.b.max_rows) {
    if (threadIdx.x == 0) atomicOr(p.flags, B200_PAGED_BAD_BATCH);
    return;
  }
  const int n = r1 - r0;
  for (int i = threadIdx.x; i < n; i += blockDim.x) {
    int x = p.parents[r0 + i];
    if (x < -1 || x >= i) { x = -1; atomicOr(p.flags, B200_PAGED_BAD_TREE); }
    parent[i] = (int16_t)x;
  }
  __syncthreads();
  for (int i = threadIdx.x; i < n; i += blockDim.x) {
    uint32_t* row = p.seen + (long long)(r0 + i) * p.words;
    for (int w = (i >> 5) + 1; w < p.words; ++w) row[w] = 0;
    int depth = -1, word = i >> 5;
    uint32_t bits = 0;
    for (int x = i; x >= 0; x = parent[x]) {
      for (; word > x >> 5; --word, bits = 0) row[word] = bits;
      bits |= 1u << (x & 31);
      ++depth;
    }
    for (; word >= 0; --word, bits = 0) row[word] = bits;
    p.position[r0 + i] = (int)((uint32_t)before + (uint32_t)depth);
  }
}

// =========================================================================================================================
// attention
// =========================================================================================================================
constexpr int SOFT_WARPS = 8, CONVERT_WARPS = 7, THREADS = (SOFT_WARPS + CONVERT_WARPS + 1) * 32, KEYS = 128, INFOS = 8;
constexpr int UNIT_COST = 6, MIN_RUN = 6;    // in tiles: what a unit costs beside its own, and the least of a CTA

struct TreeP : AttnP {
  const uint32_t* seen;                      // [rows][words]: bit i of a row: it sees the sequence's i-th token of the step
  const int32_t* position;                   // [rows]
  int words;
  int4* split;                               // per CTA: the unit that it begins and does not end (sequence, kv head, columns' number) and how many CTAs behind it have parts of that; 0: there is none
};

template <int D>
struct TreeSmem {
  static constexpr uint32_t TILE = 128 * D * 2, HALF = 128 * 128;             // 128 rows of f16, in halves of 64 dims
  static constexpr uint32_t Q = 0, K = TILE, V = 3 * TILE, JOIN = 5 * TILE, BYTES = JOIN + 256 * 128 + 1024;
};

// ---- the flattened work ----
template <int C>
__device__ __forceinline__ int units_of(const AttnP& p, const Seq& q) { return !q.ok || q.n == 0 ? 0 : p.H * ((q.n * p.G + C - 1) / C); }
// all units of a sequence take its whole range, from the first row's window on
__device__ __forceinline__ int places_of(const AttnP& p, const Seq& q) { return Tiles<7>(q.before, q.before + q.n - 1, p.window, p.sinks).n + UNIT_COST; }
template <int C>
__device__ __forceinline__ long long work_of(const AttnP& p, int s) {
  const Seq q = sequence(p.b, s, p.P);
  const int u = units_of<C>(p, q);
  return u ? (long long)u * places_of(p, q) : 0;
}
struct Run { long long from, to, base; int s; };      // this CTA's places; the sequence that it begins in and the places in front of that
// by all threads of the block
template <int C>
__device__ Run run_of(const AttnP& p) {
  constexpr int WARPS = THREADS / 32;
  __shared__ long long sums[WARPS];
  __shared__ Run found;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  long long mine = 0;
  for (int s = threadIdx.x; s < p.b.S; s += THREADS) mine += work_of<C>(p, s);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) mine += __shfl_xor_sync(0xffffffffu, mine, o);
  if (lane == 0) sums[warp] = mine;
  if (threadIdx.x == 0) found.s = -1;
  __syncthreads();
  long long total = 0;
#pragma unroll
  for (int w = 0; w < WARPS; ++w) total += sums[w];
  const long long run = max((total + gridDim.x - 1) / gridDim.x, (long long)MIN_RUN);
  Run r;
  r.from = run * blockIdx.x; r.to = min(r.from + run, total); r.s = -1; r.base = 0;
  if (r.from >= total) return r;
  long long base = 0;
  for (int s0 = 0; s0 < p.b.S; s0 += THREADS) {
    const int s = s0 + (int)threadIdx.x;
    const long long w = s < p.b.S ? work_of<C>(p, s) : 0;
    long long in = w;                        // inclusive sums of the warp, then of the block
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const long long x = __shfl_up_sync(0xffffffffu, in, o);
      if (lane >= o) in += x;
    }
    __syncthreads();
    if (lane == 31) sums[warp] = in;
    __syncthreads();
    long long all = 0;
#pragma unroll
    for (int i = 0; i < WARPS; ++i) {
      if (i < warp) in += sums[i];
      all += sums[i];
    }
    if (base + in - w <= r.from && r.from < base + in) { found.s = s; found.base = base + in - w; }
    __syncthreads();
    if (found.s >= 0) break;
    base += all;
  }
  r.s = found.s; r.base = found.base;
  return r;
}
// A part of a unit: places u0 .. u1 - 1 of n_pos, of which the first UNIT_COST are no tiles; tiles t0 .. t0 + n - 1 of the sequence's.
struct Part { Seq q; int s, h, ct, u0, u1, n_pos, t0, n; };
template <int C>
struct Walk {
  long long f, to, base;
  int s, units, places;
  Seq q;
  __device__ __forceinline__ void at(const AttnP& p) {
    q = sequence(p.b, s, p.P);
    units = units_of<C>(p, q);
    places = units ? places_of(p, q) : 1;
  }
  __device__ __forceinline__ Walk(const AttnP& p, const Run& r) : f(r.from), to(r.to), base(r.base), s(r.s) { at(p); }
  __device__ __forceinline__ bool next(const AttnP& p, Part& x) {
    if (f >= to) return false;
    while (f >= base + (long long)units * places && s + 1 < p.b.S) {          // the next sequence that has work
      base += (long long)units * places;
      ++s;
      at(p);
    }
    const long long o = f - base;
    const int u = o < 0x7fffffffll ? (int)((uint32_t)o / (uint32_t)places) : (int)(o / places), cts = units / p.H;
    x.q = q; x.s = s; x.h = u / cts; x.ct = u - x.h * cts; x.n_pos = places;
    x.u0 = (int)(o - (long long)u * places); x.u1 = (int)min((long long)places, x.u0 + (to - f));
    f += x.u1 - x.u0;
    x.t0 = max(x.u0 - UNIT_COST, 0); x.n = max(x.u1 - UNIT_COST, 0) - x.t0;
    return true;
  }
};

// registers of a weight thread and of the others: together those that the block was launched with
template <int C> constexpr int soft_regs() { return C == 128 ? 176 : 128; }

template <int D, int FMT, int C>
__global__ void __launch_bounds__(THREADS, 1) tree_kernel(const TreeP p) {
  typedef TreeSmem<D> L;
  constexpr int R = 128 / C;
  extern __shared__ uint8_t smem_raw[];
  __shared__ __align__(8) uint64_t bars[17 + INFOS];
  __shared__ float4 info[INFOS][8];          // per 16 keys: keys' scale, log2 and reciprocal of the values'; there: whether the page is
  __shared__ __align__(16) uint32_t there[INFOS][8];
  __shared__ uint32_t tmem_at;
  __shared__ volatile int quit;              // somebody has waited too long: nobody waits any more, and all go through to the end
  __shared__ float factors[C];               // of a column: what turns a product of codes into a score in base 2, but for the keys' scale
  __shared__ float2 ml[256], total[C];
  const uint32_t base = (smem_u32(smem_raw) + 1023u) & ~1023u;
  uint8_t* const smem = smem_raw + (base - smem_u32(smem_raw));
  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  const uint32_t bar = smem_u32(bars), k_full = bar, k_empty = bar + 16, v_full = bar + 32, v_empty = bar + 48, s_full = bar + 64, p_full = bar + 80, o_done = bar + 96, s_taken = bar + 112, q_full = bar + 128, i_full = bar + 136;
  if (threadIdx.x == 0) {
    quit = 0;
    for (int i = 0; i < 2; ++i) {
      mbar_init(k_full + 8 * i, 4); mbar_init(k_empty + 8 * i, 1); mbar_init(v_full + 8 * i, 4); mbar_init(v_empty + 8 * i, 1);
      mbar_init(s_full + 8 * i, 1); mbar_init(s_taken + 8 * i, 4); mbar_init(p_full + 8 * i, 4); mbar_init(o_done + 8 * i, 1);
    }
    mbar_init(q_full, SOFT_WARPS);
    for (int i = 0; i < INFOS; ++i) mbar_init(i_full + 8 * i, 4);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  pdl_trigger();
  pdl_wait();
  if (blockIdx.x == 0) record_sequences(p.b, p.P, p.flags, THREADS);
  if (threadIdx.x == 0) p.split[blockIdx.x] = make_int4(0, 0, 0, 0);
  const Run run = run_of<C>(p);
  if (run.s < 0) return;                     // the whole block
  if (warp == SOFT_WARPS + CONVERT_WARPS) tmem_alloc(smem_u32(&tmem_at), 512);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = tmem_at;
  Walk<C> walk(p, run);
  Part u;

  // Tiles are numbered through all parts, g = 0, 1, ..: tile g has the places g & 1 of keys and values, and the weight warps g & 1.
  if (warp >= SOFT_WARPS) {
  asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(256 - soft_regs<C>()));
  if (warp < SOFT_WARPS + CONVERT_WARPS) {
    // ---- codes into f16 tiles: 32 tokens of a tile's keys or values at a time, eight such tasks a tile, which the warps take in turn ----
    constexpr int LANES = D / 16, STEP = 32 / LANES, LOADS = 32 / STEP;       // lanes a row, rows a load, loads
    const int row = lane / LANES, c = lane % LANES;
    // lanes of a row's second 64 dims take the neighbouring row, so that eight lanes' pieces of the f16 tile lie in different banks
    const int r_in = row ^ (D == 128 ? c >> 2 : 0);
    struct Job { int task, j0, h, pf, pl, page; };      // task: numbered through all tiles, -1: none; page: lane l's, of tokens j0 + (l & 1) * 16 ..
    int at = warp - SOFT_WARPS, first = 0, count = 0;   // the next task, and the part's
    u.n = 0;
    auto next_job = [&]() {
      Job x;
      x.task = -1;
      while (at >= first + count) {
        first += count;
        if (!walk.next(p, u)) { count = 0; return x; }
        count = 8 * u.n;
      }
      const int t = at - first;
      const Tiles<7> tiles(u.q.before, u.q.before + u.q.n - 1, p.window, p.sinks);
      x.task = at; x.h = u.h; x.pf = u.q.before; x.pl = u.q.before + u.q.n - 1;
      x.j0 = (tiles[u.t0 + (t >> 3)] << 7) + 32 * (t & 3);
      const int j = x.j0 + 16 * (lane & 1);
      x.page = -1;
      if (j <= x.pl && (p.window <= 0 || x.pf - j - 15 < p.window || j < p.sinks)) {
        x.page = p.b.table[u.s * p.b.table_ld + (j >> p.page_shift)];
        if (x.page < 0 || x.page >= p.pages) { x.page = -1; atomicOr(p.flags, B200_PAGED_BAD_PAGE); }
      }
      at += CONVERT_WARPS;
      return x;
    };
    uint4 held[LOADS];                       // of the job to come
    float2 scales = make_float2(0.f, 1.f);
    auto load = [&](const Job& x) {
      if (x.task < 0) return;
      const bool keys = !(x.task & 4);
      const uint8_t* codes = keys ? p.k : p.v;
      if (keys && x.page >= 0) scales = make_float2(p.k_scale[(long long)x.page * p.H + x.h], p.v_scale[(long long)x.page * p.H + x.h]);
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        const int pg = __shfl_sync(0xffffffffu, x.page, half), j1 = x.j0 + 16 * half;
        const uint8_t* from = codes + (((long long)pg * p.H + x.h) * p.P + (j1 & (p.P - 1)) + r_in) * D + 16 * c;
        // values that no row sees may be anything; keys are masked
        const bool all = keys || (j1 + 15 <= x.pl && (p.window <= 0 || x.pf - j1 < p.window || j1 + 16 <= p.sinks));
#pragma unroll
        for (int i = 0; i < LOADS / 2; ++i) {
          const int j = j1 + i * STEP + r_in;
          const bool seen = pg >= 0 && (all || (j <= x.pl && (p.window <= 0 || x.pf - j < p.window || j < p.sinks)));
          held[half * (LOADS / 2) + i] = seen ? *reinterpret_cast<const uint4*>(from + i * STEP * D) : make_uint4(0, 0, 0, 0);
        }
      }
    };
    Job job = next_job();
    load(job);
    Job then = next_job();
    while (job.task >= 0) {
      const int g = job.task >> 3, st = g & 1, w4 = job.task & 3;
      const bool keys = !(job.task & 4);
      if (keys) {                            // what the weights need to know of these keys' pages
        if (lane < 2) {
          const float vs = value_scale(scales.y);
          there[g % INFOS][2 * w4 + lane] = job.page >= 0 ? 1u : 0u;
          info[g % INFOS][2 * w4 + lane] = job.page >= 0 ? make_float4(scales.x > 0.f ? scales.x : 1.f, __log2f(vs), __frcp_rn(vs), 0.f) : make_float4(1.f, 0.f, 0.f, 0.f);
        }
        __syncwarp();
      }
      warp_wait((keys ? k_empty : v_empty) + 8 * st, ((uint32_t)(g >> 1) & 1u) ^ 1u, &quit);
      if (keys && lane == 0) mbar_arrive(i_full + 8 * (g % INFOS));
      uint8_t* const dst = smem + (keys ? L::K : L::V) + st * L::TILE + (c >> 2) * L::HALF;
#pragma unroll
      for (int i = 0; i < LOADS; ++i) {
        const int t = 32 * w4 + i * STEP + r_in;
        const uint32_t w[4] = {ready<FMT>(held[i].x), ready<FMT>(held[i].y), ready<FMT>(held[i].z), ready<FMT>(held[i].w)};
        uint8_t* r = dst + t * 128;
        *reinterpret_cast<uint4*>(r + (((2 * (c & 3)) ^ (t & 7)) << 4)) = make_uint4(half2_of<FMT, 0>(w[0]), half2_of<FMT, 1>(w[0]), half2_of<FMT, 0>(w[1]), half2_of<FMT, 1>(w[1]));
        *reinterpret_cast<uint4*>(r + (((2 * (c & 3) + 1) ^ (t & 7)) << 4)) = make_uint4(half2_of<FMT, 0>(w[2]), half2_of<FMT, 1>(w[2]), half2_of<FMT, 0>(w[3]), half2_of<FMT, 1>(w[3]));
      }
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      __syncwarp();
      if (lane == 0) mbar_arrive((keys ? k_full : v_full) + 8 * st);
      job = then;
      load(job);
      then = next_job();
    }
  } else {
    // ---- products ----
    constexpr uint32_t id_s = idesc_f16(KEYS, false), id_o = idesc_f16(D, true);
    int g0 = 0, part = 0;                    // tiles and parts in front
    for (; walk.next(p, u); ++part) {
      warp_wait(q_full, (uint32_t)part & 1u, &quit);
      for (int x = 0; x <= u.n; ++x) {
        if (x < u.n) {
          const int g = g0 + x, st = g & 1;
          if (g > 0) warp_wait(s_taken + 8 * (st ^ 1), (uint32_t)((g - 1) >> 1) & 1u, &quit);
          warp_wait(k_full + 8 * st, (uint32_t)(g >> 1) & 1u, &quit);
          tc_fence_after();
          const uint32_t a = desc_low(base + L::Q), b = desc_low(base + L::K + st * L::TILE);
#pragma unroll
          for (int half = 0; half < D / 64; ++half) umma_block<1>(tmem, a + half * (L::HALF >> 4), b - a, id_s, half > 0 ? 1u : 0u);
          commit_elected(s_full + 8 * st);
          commit_elected(k_empty + 8 * st);
        }
        if (x > 0) {
          const int g = g0 + x - 1, st = g & 1;
          warp_wait(v_full + 8 * st, (uint32_t)(g >> 1) & 1u, &quit);
          warp_wait(p_full + 8 * st, (uint32_t)(g >> 1) & 1u, &quit);
          tc_fence_after();
          if (elected()) {
#pragma unroll
            for (int k = 0; k < KEYS / 16; ++k)
              product_pv(tmem + 256 + 128 * st, tmem + 128 + 64 * st + 8 * k, base + L::V + st * L::TILE + k * 2048, L::HALF, id_o, x > 2 || k > 0 ? 1u : 0u);
          }
          __syncwarp();
          commit_elected(o_done + 8 * st);
          commit_elected(v_empty + 8 * st);
        }
      }
      g0 += u.n;
    }
    __syncwarp();
  }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(soft_regs<C>()));
    // ---- weights: a row per thread, which is a column and C of a tile's keys ----
    const int i = warp >> 2, q4 = warp & 3, in = q4 * 32 + lane, rep = in / C, col = in % C;
    const uint32_t lanes = (uint32_t)(q4 * 32) << 16, ts = tmem + lanes + rep * C, tp = tmem + lanes + 128 + 64 * i, to = tmem + lanes + 256 + 128 * i;
    if constexpr (R > 1) {                   // other copies' keys have no weight here
      const uint32_t zero[16] = {};
#pragma unroll
      for (int k = 0; k < 4; ++k) tmem_st16(tp + 16 * k, zero);
      tmem_st_wait();
    }
    int g0 = 0;
    for (; walk.next(p, u); g0 += u.n) {
      // queries: f16 after a power of two for each column, as rows and heads of very different size may lie side by side
      constexpr int PIECES = D / 8, MINE = C * PIECES / (SOFT_WARPS * 32);
      const int n_cols = u.q.n * p.G - u.ct * C;                              // of this unit, and more
#pragma unroll
      for (int k = 0; k < MINE; ++k) {
        const int x = threadIdx.x + 256 * k, r = x / PIECES, c = x % PIECES, cc = u.ct * C + r, token = cc / p.G;
        uint4 raw = r < n_cols ? *reinterpret_cast<const uint4*>(p.q + (u.q.r0 + token) * p.q_ld + (long long)(u.h * p.G + cc - token * p.G) * D + 8 * c) : make_uint4(0, 0, 0, 0);
        const uint32_t v[4] = {raw.x, raw.y, raw.z, raw.w};
        uint32_t top = 0;                    // magnitudes as numbers, which order like the values
#pragma unroll
        for (int e = 0; e < 4; ++e) top = max(top, max(v[e] << 16 & 0x7fff0000u, v[e] & 0x7fff0000u));
#pragma unroll
        for (int o = PIECES / 2; o > 0; o >>= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
        // A column that is not finite gets NaN, and no other: it asks as zeros, whose weights say whether it sees anything at all, and its factor tells the end of it.
        const bool odd = top >= 0x7f800000u;
        const float power = top && !odd ? power_of_two_in(__uint_as_float(top)) : 1.f, up = 16384.f / power;
        if (c == 0) factors[r] = odd ? NAN : power * (1.f / 16384.f) * p.scale2;
        uint32_t o[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) o[e] = odd ? 0u : pack_f16(__uint_as_float(v[e] << 16) * up, __uint_as_float(v[e] & 0xffff0000u) * up);
#pragma unroll
        for (int y = r; y < 128; y += C)
          *reinterpret_cast<uint4*>(smem + L::Q + (c >> 3) * L::HALF + y * 128 + (((c & 7) ^ (y & 7)) << 4)) = make_uint4(o[0], o[1], o[2], o[3]);
      }
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      __syncwarp();
      if (lane == 0) mbar_arrive(q_full);
      asm volatile("bar.sync 1, %0;" ::"n"(SOFT_WARPS * 32) : "memory");      // all columns' factors
      const Tiles<7> tiles(u.q.before, u.q.before + u.q.n - 1, p.window, p.sinks);
      const int before = u.q.before, last = before + u.q.n - 1, token = (u.ct * C + col) / p.G;
      const bool has = col < n_cols;
      const int pos = has ? p.position[u.q.r0 + token] : -1, lo = p.window > 0 ? pos - p.window : -1;         // of what is cached: sees j > lo or j < sinks
      const uint32_t* const seen_row = p.seen + (long long)(u.q.r0 + token) * p.words;
      const float fac = factors[col];
      float m = -INFINITY, sum = 0.f;
      int done = 0;                          // tiles of this group of warps
      for (int x = (g0 + i) & 1; x < u.n; x += 2, ++done) {
        const int g = g0 + x;
        warp_wait(i_full + 8 * (g % INFOS), (uint32_t)(g / INFOS) & 1u, &quit);
        warp_wait(s_full + 8 * i, (uint32_t)(g >> 1) & 1u, &quit);
        tc_fence_after();
        const int j0 = tiles[u.t0 + x] << 7;
        const float4* ip = info[g % INFOS] + rep * (C / 16);
        const uint32_t* th = there[g % INFOS];
        const uint4 t0 = *reinterpret_cast<const uint4*>(th), t1 = *reinterpret_cast<const uint4*>(th + 4);
        const bool whole = ((t0.x & t0.y & t0.z & t0.w & t1.x & t1.y & t1.z & t1.w) != 0u) & (j0 + KEYS <= before) & ((p.window <= 0) | (last - j0 < p.window) | (j0 + KEYS <= p.sinks));
        uint32_t r[C];                       // the row's scores: read once, as the registers have room for them
        float t = -INFINITY, by[C / 16], lv[C / 16];    // score in base 2 = product * by + lv; by > 0, so that the largest score of a page's keys is that of their largest product
#pragma unroll
        for (int c = 0; c < C / 32; ++c) tmem_ld32(ts + 32 * c, r + 32 * c);
#pragma unroll
        for (int c = 0; c < C / 32; ++c) tmem_ld_wait32(r + 32 * c);
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(s_taken + 8 * i);
        if (!whole) {                        // keys that the row does not see: a bit for each of 32
#pragma unroll
          for (int c = 0; c < C / 32; ++c) {
            const int at = j0 + rep * C + 32 * c, off = at - before;
            uint32_t seen = has && at < before ? upto(before - 1 - at) & (~upto(lo - at) | upto(p.sinks - 1 - at)) : 0u;
            if (has && at + 31 >= before && at <= last) {                     // the step's own tokens
              const int w = off >> 5, sh = off & 31;
              const uint32_t a = w >= 0 && w < p.words ? seen_row[w] : 0u, b = w + 1 >= 0 && w + 1 < p.words ? seen_row[w + 1] : 0u;
              uint32_t own = __funnelshift_r(a, b, sh) & upto(last - at);
              if (p.window > 0 && pos - before >= p.window)                   // some of those in front may be too far away
                for (uint32_t left = own; left; left &= left - 1) {
                  const int e = __ffs(left) - 1, their = p.position[u.q.r0 + off + e];
                  if (!(pos - their < p.window || their < p.sinks)) own &= ~(1u << e);
                }
              seen |= own;
            }
            if (!th[rep * (C / 16) + 2 * c]) seen &= 0xffff0000u;
            if (!th[rep * (C / 16) + 2 * c + 1]) seen &= 0xffffu;
#pragma unroll
            for (int e = 0; e < 32; ++e)
              if (!(seen >> e & 1u)) r[32 * c + e] = 0xff800000u;
          }
        }
#pragma unroll
        for (int b = 0; b < C / 16; ++b) {
          by[b] = fmaxf(ip[b].x * fac, FLT_MIN);                              // also where fac is NaN
          lv[b] = ip[b].y;
          float mx[2] = {__uint_as_float(r[16 * b]), __uint_as_float(r[16 * b + 1])};
#pragma unroll
          for (int e = 2; e < 16; ++e) mx[e & 1] = fmaxf(mx[e & 1], __uint_as_float(r[16 * b + e]));
          t = fmaxf(t, fmaf(fmaxf(mx[0], mx[1]), by[b], lv[b]));
        }
        const bool grow = t > __fadd_rd(m, SLACK);     // rounded down: above 2^27 the sum would else round to the score itself, and its weight to infinity
        if (done > 0) {                      // the sum over this group's tile in front has read its weights and settled in O
          warp_wait(o_done + 8 * i, (uint32_t)((g - 2) >> 1) & 1u, &quit);
          tc_fence_after();
        }
        if (__any_sync(0xffffffffu, grow)) {
          const float now = t - UNDER, factor = grow ? exp2_fast(m - now) : 1.f;
          if (grow) { m = now; sum *= factor; }
          if (done > 0) {
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
          for (int e = 0; e < C; ++e) r[e] = __float_as_uint(fmaf(__uint_as_float(r[e]), by[e / 16], lv[e / 16]));
#pragma unroll
          for (int b = 0; b < C / 16; ++b) { by[b] = 1.f; lv[b] = 0.f; }
        }
#pragma unroll
        for (int c = 0; c < C / 32; ++c) {
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
          tmem_st16(tp + rep * (C / 2) + 16 * c, w);
        }
        tmem_st_wait();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(p_full + 8 * i);
      }
      if (done > 0) {
        const int g = g0 + ((g0 + i) & 1) + 2 * (done - 1);
        warp_wait(o_done + 8 * i, (uint32_t)(g >> 1) & 1u, &quit);
        tc_fence_after();
      }
      // join the column's 2 R rows
      const bool alone = u.u0 == 0 && u.u1 == u.n_pos;
      const int slot = 2 * (int)blockIdx.x + (u.u0 == 0 ? 1 : 0);
      if (u.u0 == 0 && !alone && threadIdx.x == 0) {
        const long long runs = run.to - run.from, left = u.n_pos - u.u1;
        p.split[blockIdx.x] = make_int4(u.s, u.h, u.ct, (int)((left + runs - 1) / runs));
      }
      ml[128 * i + in] = make_float2(m, sum);
      asm volatile("bar.sync 1, %0;" ::"n"(SOFT_WARPS * 32) : "memory");
      float top = -INFINITY, all = 0.f;
#pragma unroll
      for (int k = 0; k < 2 * R; ++k) top = fmaxf(top, ml[k * C + col].x);
#pragma unroll
      for (int k = 0; k < 2 * R; ++k) {
        const float2 y = ml[k * C + col];
        all = fmaf(y.y, y.x == -INFINITY ? 0.f : exp2_fast(y.x - top), all);
      }
      const float by = m == -INFINITY ? 0.f : exp2_fast(m - top);
      if (i == 0 && rep == 0) total[col] = make_float2(top, all != 0.f && isnan(fac) ? NAN : all);
      constexpr int TEAM = 2 * R, PER = 32 / TEAM;                            // threads of a column, dims of each
      const int c_out = threadIdx.x / TEAM, d_out = (threadIdx.x % TEAM) * PER, cc = u.ct * C + c_out, t_out = cc / p.G;
      uint8_t* const join = smem + L::JOIN;
#pragma unroll
      for (int c = 0; c < D / 32; ++c) {
        uint32_t o[32];
        if (done > 0) {
          tmem_ld32(to + 32 * c, o);
          tmem_ld_wait32(o);
        }
#pragma unroll
        for (int e = 0; e < 32; e += 4) {
          float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
          if (done > 0 && by != 0.f) v = make_float4(__uint_as_float(o[e]) * by, __uint_as_float(o[e + 1]) * by, __uint_as_float(o[e + 2]) * by, __uint_as_float(o[e + 3]) * by);
          *reinterpret_cast<float4*>(join + (128 * i + in) * 128 + (((e >> 2) ^ (in & 7)) << 4)) = v;
        }
        asm volatile("bar.sync 1, %0;" ::"n"(SOFT_WARPS * 32) : "memory");
        float acc[PER];
#pragma unroll
        for (int e = 0; e < PER; ++e) acc[e] = 0.f;
#pragma unroll
        for (int k = 0; k < 2 * R; ++k)
#pragma unroll
          for (int e = 0; e < PER; e += 4) {
            const float4 v = *reinterpret_cast<const float4*>(join + (k * C + c_out) * 128 + ((((d_out + e) >> 2) ^ (c_out & 7)) << 4));
            acc[e] += v.x; acc[e + 1] += v.y; acc[e + 2] += v.z; acc[e + 3] += v.w;
          }
        if (c_out < n_cols) {
          const float2 tl = total[c_out];
          if (alone) {
            const float inv = tl.y != 0.f ? 1.f / tl.y : 0.f;
            bf16* out = p.out + (u.q.r0 + t_out) * p.out_ld + (long long)(u.h * p.G + cc - t_out * p.G) * D + 32 * c + d_out;
#pragma unroll
            for (int e = 0; e < PER; e += 4) *reinterpret_cast<uint2*>(out + e) = make_uint2(pack_bf16(acc[e] * inv, acc[e + 1] * inv), pack_bf16(acc[e + 2] * inv, acc[e + 3] * inv));
          } else {
            const long long at = (long long)slot * C + c_out;
            if (c == 0 && d_out == 0) *reinterpret_cast<float2*>(p.part_ml + 2 * at) = tl;
#pragma unroll
            for (int e = 0; e < PER; e += 4) *reinterpret_cast<float4*>(p.part_o + at * D + 32 * c + d_out + e) = make_float4(acc[e], acc[e + 1], acc[e + 2], acc[e + 3]);
          }
        }
        asm volatile("bar.sync 1, %0;" ::"n"(SOFT_WARPS * 32) : "memory");
      }
      tc_fence_before();
    }
  }
  __syncthreads();
  tc_fence_after();
  if (warp == SOFT_WARPS + CONVERT_WARPS) tmem_dealloc(tmem, 512);
  if (threadIdx.x == 0 && quit) atomicOr(p.flags, B200_PAGED_WAIT);
}

// Joins the units that are cut: a block for two columns of the one that a CTA has begun, a column's four teams of sixteen threads take its parts in turn.
template <int D, int C>
__global__ void __launch_bounds__(128) tree_join_kernel(const TreeP p) {
  pdl_trigger();
  pdl_wait();
  constexpr int PER = D / 16;
  __shared__ float o_s[8][D + 4], m_s[8], l_s[8];
  const int cta = (int)blockIdx.x / (C / 2), col = 2 * ((int)blockIdx.x % (C / 2)) + (threadIdx.x >> 6), team = threadIdx.x >> 4, d0 = (threadIdx.x & 15) * PER;
  const int4 of = p.split[cta];
  if (of.w == 0) return;
  const Seq q = sequence(p.b, of.x, p.P);
  const int cc = of.z * C + col, token = cc / p.G;
  const bool has = cc < q.n * p.G;
  float top = -INFINITY, sum = 0.f, acc[PER];
#pragma unroll
  for (int e = 0; e < PER; ++e) acc[e] = 0.f;
  if (has) {
    // the first part is its run's last, the others are their runs' first
#pragma unroll 2
    for (int i = team & 3; i <= of.w; i += 4) {
      const long long at = (long long)(2 * (cta + i) + (i == 0 ? 1 : 0)) * C + col;
      const float2 y = reinterpret_cast<const float2*>(p.part_ml)[at];
      const float now = fmaxf(top, y.x), keep = now == -INFINITY ? 0.f : exp2_fast(top - now), by = now == -INFINITY ? 0.f : exp2_fast(y.x - now);
      const float4* o = reinterpret_cast<const float4*>(p.part_o + at * D + d0);
      top = now;
      sum = fmaf(sum, keep, y.y * by);
#pragma unroll
      for (int e = 0; e < PER / 4; ++e) {
        const float4 v = o[e];
        acc[4 * e] = fmaf(acc[4 * e], keep, v.x * by); acc[4 * e + 1] = fmaf(acc[4 * e + 1], keep, v.y * by);
        acc[4 * e + 2] = fmaf(acc[4 * e + 2], keep, v.z * by); acc[4 * e + 3] = fmaf(acc[4 * e + 3], keep, v.w * by);
      }
    }
  }
#pragma unroll
  for (int e = 0; e < PER; ++e) o_s[team][d0 + e] = acc[e];
  if ((threadIdx.x & 15) == 0) { m_s[team] = top; l_s[team] = sum; }
  __syncthreads();
  if ((team & 3) || !has) return;
  top = -INFINITY; sum = 0.f;
#pragma unroll
  for (int i = 0; i < 4; ++i) top = fmaxf(top, m_s[team + i]);
#pragma unroll
  for (int e = 0; e < PER; ++e) acc[e] = 0.f;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float by = m_s[team + i] == -INFINITY ? 0.f : exp2_fast(m_s[team + i] - top);
    sum = fmaf(l_s[team + i], by, sum);
#pragma unroll
    for (int e = 0; e < PER; ++e) acc[e] = fmaf(o_s[team + i][d0 + e], by, acc[e]);
  }
  const float inv = sum != 0.f ? 1.f / sum : 0.f;
  bf16* out = p.out + (q.r0 + token) * p.out_ld + (long long)(of.y * p.G + cc - token * p.G) * D + d0;
#pragma unroll
  for (int e = 0; e < PER; e += 4) *reinterpret_cast<uint2*>(out + e) = make_uint2(pack_bf16(acc[e] * inv, acc[e + 1] * inv), pack_bf16(acc[e + 2] * inv, acc[e + 3] * inv));
}

// =========================================================================================================================
// host
// =========================================================================================================================
struct TreePlan { int cols, ctas; };
TreePlan tree_plan(const b200_paged_cache* c, const b200_paged_batch* b, int G, int window, int sinks) {
  TreePlan f;
  const long long cols = (long long)b->max_rows * G;
  f.cols = cols <= 32 ? 32 : cols <= 64 ? 64 : 128;
  long long keys = (long long)b->table_width * c->page_tokens;
  if (window > 0 && (long long)window + sinks + b->max_rows < keys) keys = (long long)window + sinks + b->max_rows;
  const long long units = (long long)b->sequences * c->kv_heads * ceil_div64(cols, f.cols), runs = ceil_div64(units * (ceil_div64(keys, KEYS) + 1 + UNIT_COST), MIN_RUN);
  f.ctas = (int)(runs < 148 ? runs : 148);
  return f;
}
// sums and (maximum, sum of the weights) of two parts per CTA, and the units that are cut
int64_t tree_bytes(const TreePlan& f, int D) { return (int64_t)f.ctas * (2 * f.cols * (D + 2) * 4 + 16); }

template <int D, int FMT, int C>
int launch(const TreeP& p, int ctas, cudaStream_t st) {
  static std::atomic<uint64_t> limits{0};
  static std::atomic<uint64_t> shares{0};
  B200_TRY(allow_smem(limits, (int)TreeSmem<D>::BYTES, tree_kernel<D, FMT, C>));
  B200_TRY(prefer_smem(shares, 100, tree_kernel<D, FMT, C>, tree_join_kernel<D, C>));
  B200_TRY(launch_early(tree_kernel<D, FMT, C>, dim3((unsigned)ctas), dim3(THREADS), TreeSmem<D>::BYTES, st, p));
  return launch_early(tree_join_kernel<D, C>, dim3((unsigned)(ctas * (C / 2))), dim3(128), 0, st, p);
}
template <int D, int FMT>
int launch_cols(const TreeP& p, const TreePlan& f, cudaStream_t st) {
  return f.cols == 32 ? launch<D, FMT, 32>(p, f.ctas, st) : f.cols == 64 ? launch<D, FMT, 64>(p, f.ctas, st) : launch<D, FMT, 128>(p, f.ctas, st);
}

}  // namespace
}  // namespace paged
}  // namespace b200

using namespace b200;

extern "C" {

int b200_paged_tree_build(const b200_paged_batch* batch, const b200_paged_tree* tree, const int32_t* parents_dev, int32_t* flags_dev, int device, void* stream) {
  using namespace b200::paged;
  if (!batch || !batch->before_dev || !batch->rows_dev || !tree || !tree->seen_dev || !tree->position_dev || !parents_dev || !flags_dev) B200_FAIL(B200_ERR_INVALID, "paged_tree_build: null pointer");
  if (batch->sequences < 1 || batch->sequences > 65536 || batch->total_rows < 0 || batch->total_rows > (1 << 24) || batch->max_rows < 0 || batch->max_rows > MAX_NODES || tree->words < 1 ||
      (long long)tree->words * 32 < batch->max_rows || tree->words > MAX_NODES / 32)
    B200_FAIL(B200_ERR_SHAPE, "paged_tree_build: %d sequences of up to %d tokens (at most %d), masks of %d words", batch->sequences, batch->max_rows, MAX_NODES, tree->words);
  if (batch->total_rows == 0 || batch->max_rows == 0) return B200_OK;
  DeviceGuard guard(device);
  BuildP p;
  p.b.table = nullptr; p.b.before = batch->before_dev; p.b.rows = batch->rows_dev; p.b.table_ld = 0; p.b.S = batch->sequences; p.b.T = batch->total_rows; p.b.width = 0; p.b.max_rows = batch->max_rows;
  p.parents = parents_dev; p.seen = tree->seen_dev; p.position = tree->position_dev; p.flags = flags_dev; p.words = tree->words;
  EARLY_LAUNCH(tree_build_kernel, batch->sequences, 128, 0, static_cast<cudaStream_t>(stream), p);
  return check_launch("paged_tree_build");
}

int64_t b200_paged_tree_attention_bytes(const b200_paged_cache* cache, const b200_paged_batch* batch, int q_heads, int window, int sinks) {
  using namespace b200::paged;
  if (!cache || !batch || cache->kv_heads < 1 || q_heads < cache->kv_heads || q_heads % cache->kv_heads || window < 0 || sinks < 0 || batch->sequences < 1 || batch->max_rows <= 0 || batch->total_rows <= 0) return 0;
  return tree_bytes(tree_plan(cache, batch, q_heads / cache->kv_heads, window, sinks), cache->dim);
}

int b200_paged_tree_attention(const b200_paged_cache* cache, const b200_paged_batch* batch, const b200_paged_tree* tree, const void* q_dev, int64_t q_ld, void* out_dev, int64_t out_ld, int q_heads,
                              float scale, int window, int sinks, void* work_dev, int64_t work_bytes, void* stream) {
  using namespace b200::paged;
  TreeP p;
  B200_TRY(attention_arguments(&p, cache, batch, q_dev, q_ld, out_dev, out_ld, q_heads, scale, window, sinks, "paged_tree_attention"));
  if (!tree || !tree->seen_dev || !tree->position_dev) B200_FAIL(B200_ERR_INVALID, "paged_tree_attention: null pointer in the tree");
  if (batch->max_rows > MAX_NODES || tree->words < 1 || (long long)tree->words * 32 < batch->max_rows || tree->words > MAX_NODES / 32)
    B200_FAIL(B200_ERR_SHAPE, "paged_tree_attention: trees of up to %d tokens (at most %d), masks of %d words", batch->max_rows, MAX_NODES, tree->words);
  if (batch->total_rows == 0 || batch->max_rows == 0) return B200_OK;
  const TreePlan f = tree_plan(cache, batch, p.G, window, sinks);
  const int64_t need = tree_bytes(f, cache->dim);
  if (!work_dev || work_bytes < need || (reinterpret_cast<uintptr_t>(work_dev) & 15))
    B200_FAIL(B200_ERR_INVALID, "paged_tree_attention: a workspace of %lld bytes; b200_paged_tree_attention_bytes asks for %lld, on a 16-byte border", (long long)work_bytes, (long long)need);
  DeviceGuard guard(cache->device);
  p.seen = tree->seen_dev; p.position = tree->position_dev; p.words = tree->words;
  p.part_o = static_cast<float*>(work_dev);
  p.part_ml = p.part_o + (long long)f.ctas * 2 * f.cols * cache->dim;
  p.split = reinterpret_cast<int4*>(p.part_ml + (long long)f.ctas * 2 * f.cols * 2);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const bool i8 = cache->kv_dtype == B200_KV_INT8;
  if (cache->dim == 128) B200_TRY((i8 ? launch_cols<128, INT8>(p, f, st) : launch_cols<128, E4M3>(p, f, st)));
  else B200_TRY((i8 ? launch_cols<64, INT8>(p, f, st) : launch_cols<64, E4M3>(p, f, st)));
  return check_launch("paged_tree_attention");
}

}  // extern "C"
