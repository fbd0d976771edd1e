// Attention of trees of drafted tokens over the paged 8-bit cache: a row sees what its sequence has cached in front of the step, and of the step's own tokens itself and those that it comes behind.
//
// Columns are (row of the sequence, query head of the group).  A unit is C = 32, 64 or 128 of them with one kv head, and a CTA walks its keys in tiles of 64 tokens.  The tensor cores' tiles have 128 rows,
// and a tree has 20 to 100 columns as often as not: the rows are R = 128 / C copies of the columns, of which each weighs 64 / R of a tile's keys.  So all threads of the weights have work whatever C is, with a
// running maximum of their own; the products of a copy's rows with the other copies' keys are thrown away (scores) or made of zeros (P is block-diagonal, and the zeros are written once).  Tiles go to
// two groups of weight warps in turn, with a sum O of each, so that the scores of one tile, the weights of another and the sum over a third are made at the same time.  At a unit's end its 2 R sums
// are joined, both groups' where they lie in TMEM, the copies' through shared memory.
//
// Codes come as swizzled tensor copies (a producer warp, 72 KB on their way); six warps turn them into f16 tiles; one issues the products: S = Q K^T with Q in TMEM, O += P V with P there.  Units lie
// one behind the other and are cut into equal runs, one per CTA, as in paged.cu; a CTA finds its own at its start.  Codes, scales, f16 tiles and the lazy maximum are those of paged_prompt.cu.
//
// Bound: the chain of a tile, scores - weights - sum, beside the instructions around it: 950 clocks with 32 columns (products 512, three quarters of them thrown away or with zeros), 1350 with 128 (exponentials 512); and
// 7000 to 9000 clocks a unit, 7000 to a CTA's first scores, as its code is cold and the reads depend on one another (lengths, page, codes).  64 requests of 3000 tokens, 32 heads on 8: 32 columns 108 us (HBM: 62), 64 columns 119, 128
// columns 151.  Few columns go to paged.cu's kernel of few rows, in warps of their own (tree_plan).
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
constexpr int SOFT_WARPS = 8, CONVERT_WARPS = 6, PRODUCER = 14, ISSUER = 15, THREADS = 16 * 32, SHIFT = 6, KEYS = 1 << SHIFT, STAGES = 4, INFOS = 32;
// In tiles: what a unit costs beside its own (16 requests with 6, 8, 12, 16: 48.1, 48.0, 48.4, 50.6 us; 32 with 20 columns 46.4, 45.2, 45.9, 48.0), and the least of a CTA (9, 12, 16, 24: 40 columns on 3000 tokens, 8 heads 17.1,
// 16.9, 18.0, 21.4 us, one head 13.6, 14.9, 16.7, 20.3; 4 requests of 100 columns on 1000 tokens 20.1, 19.9, 19.9, 19.0).
constexpr int UNIT_COST = 8, MIN_RUN = 12;

struct TreeP : AttnP {
  int4* split;                               // per CTA: the unit that it begins and does not end, or has a middle of (sequence, kv head, columns' number); how many CTAs behind the first have parts of that, 0: there is
                                             // no such unit; and in the upper half how many CTAs back it begins
};

template <int D>
struct TreeSmem {
  static constexpr int SLOTS = CONVERT_WARPS * (D == 128 ? 3 : 6), PAIRS = SLOTS / 2;         // places of 32 tokens' codes; a place is always the same warp's; two of them side by side have a tile's keys or values
  static constexpr uint32_t HALF = KEYS * 128, TILE = HALF * (D / 64);        // a tile's f16 rows, in halves of 64 dims
  static constexpr uint32_t SLOT = 32 * D, K = 0, V = K + STAGES * TILE, CODES = V + STAGES * TILE, JOIN = CODES + SLOTS * SLOT, BYTES = JOIN + 256 * D / 2 + 1024;
};
// What is to be known of a tile: its first token, first and last position of the unit's rows, whether every row sees all of it (1) and whether all its tokens are there and may be seen (2); and of each 16
// tokens: keys' scale, log2 and reciprocal of the values', 1 where there is a page.
struct TileInfo { int j0, pf, pl, whole; float4 group[KEYS / 16]; };

// ---- the flattened work ----
template <int C>
__device__ __forceinline__ int units_of(const AttnP& p, const Seq& q) { return !q.ok || q.n == 0 ? 0 : p.H * ((q.n * p.G + C - 1) / C); }
// all units of a sequence take its whole range, from the first row's window on
__device__ __forceinline__ int places_of(const AttnP& p, const Seq& q) { return Tiles<SHIFT>(q.before, q.before + q.n - 1, p.window, p.sinks).n + UNIT_COST; }
// A sequence's units and the places of each.
struct Share {
  Seq q;
  int units, places;
  __device__ __forceinline__ long long work() const { return (long long)units * places; }
};
template <int C>
__device__ __forceinline__ Share share_of(const AttnP& p, int s) {
  Share x;
  x.q = sequence(p.b, s, p.P);
  x.units = units_of<C>(p, x.q);
  x.places = x.units ? places_of(p, x.q) : 1;
  return x;
}
// A part of a unit: places u0 .. u1 - 1 of n_pos, of which the first UNIT_COST are no tiles; tiles t0 .. t0 + n - 1 of the sequence's.
struct Part {
  Seq q;
  int s, h, ct, u0, u1, n_pos, t0, n;
  int first, from;                           // of the sequence's tiles: those in front of `first` are the first ones' (Tiles)
  __device__ __forceinline__ int tile(int x) const { const int i = t0 + x; return i < first ? i : from + i - first; }
};
// A warp's way through its CTA's parts.  It lies in shared memory, as every warp's roles have other uses for 20 registers.
struct Walk {
  long long f, to, base, run;                // places; run: the CTAs' equal share
  int s, now;                                // part[now]: the last one; the one in front of it lies beside it
  Share share;
  Part part[2];
};
// Where a CTA's walk begins, `run`: places of an equal share.  Where there is a CTA for every unit, and the longest is not much longer than a share, each has one whole: a unit that is cut costs a second start and the
// join.  (CUT_COST 0, 20, 60, on 80 columns of 8 heads: 16 requests of 3000 tokens 44.1, 39.9, 40.1 us, of 400 tokens 23.2, 15.9, 15.9, 8 of 3000 tokens 31.9, 31.9, 38.8; narrow heads under a window 24.6, 19.9, 19.9.)
constexpr int CUT_COST = 20, UNITS_MOST = 1 << 20;       // more units are as many as that: it is many either way
struct Shares {
  long long run, from;                       // from: the CTA's first place or, where it has one whole, its unit
  bool whole;
  __device__ __forceinline__ Shares(long long total, int units, int longest) {
    const long long up = total + gridDim.x - 1;
    run = max(up >> 32 ? up / gridDim.x : (long long)((uint32_t)up / gridDim.x), (long long)MIN_RUN);
    whole = units <= (int)gridDim.x && longest <= run + CUT_COST;
    from = whole ? blockIdx.x : run * blockIdx.x;
  }
};
// Sequence s, whose work (units, where CTAs have them whole) ends at `end` of all sequences', is the one that the CTA begins in.
__device__ __forceinline__ void begin_in(Walk& w, const Shares& x, int s, const Share& share, long long end, long long size, long long total) {
  w.now = 0; w.s = s; w.share = share; w.run = x.run;
  if (x.whole) {                             // places are counted from this sequence on
    w.base = 0;
    w.f = (x.from - (end - size)) * share.places; w.to = w.f + share.places;
  } else {
    w.base = end - size;
    w.f = x.from; w.to = min(x.from + x.run, total);
  }
}
// By a warp, for up to 32 sequences.
template <int C>
__device__ __forceinline__ void start_alone(const AttnP& p, Walk& w) {
  const int lane = threadIdx.x & 31;
  const Share x = share_of<C>(p, min(lane, p.b.S - 1));
  const bool is = lane < p.b.S;
  const long long work = is ? x.work() : 0;
  const int units = is ? min(x.units, UNITS_MOST) : 0, longest = __reduce_max_sync(0xffffffffu, units ? x.places : 0);
  long long in = work;                       // inclusive sums
  int units_in = units;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const long long y = __shfl_up_sync(0xffffffffu, in, o);
    const int z = __shfl_up_sync(0xffffffffu, units_in, o);
    if (lane >= o) { in += y; units_in += z; }
  }
  const long long total = __shfl_sync(0xffffffffu, in, 31);
  const Shares shares(total, __shfl_sync(0xffffffffu, units_in, 31), longest);
  const long long size = shares.whole ? units : work, end = shares.whole ? units_in : in;
  const bool here = end - size <= shares.from && shares.from < end;
  if (here) begin_in(w, shares, lane, x, end, size, total);
  if (!__any_sync(0xffffffffu, here) && lane == 0) w.f = w.to = 0;            // there is no work for this CTA
  __syncwarp();
}
// By all threads of the block, for any number.
template <int C>
__device__ __forceinline__ void start_together(const AttnP& p, Walk& found) {
  constexpr int WARPS = THREADS / 32;
  __shared__ long long sums[WARPS];
  __shared__ int unit_sums[WARPS], tops[WARPS];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, S = p.b.S;
  const Share mine = share_of<C>(p, min((int)threadIdx.x, S - 1));
  long long total = 0;
  int units = 0, longest = 0;
  for (int s = threadIdx.x; s < S; s += THREADS) {
    const Share x = s == (int)threadIdx.x ? mine : share_of<C>(p, s);
    total += x.work(); units = min(units + min(x.units, UNITS_MOST), UNITS_MOST);
    longest = max(longest, x.units ? x.places : 0);
  }
  units = min(__reduce_add_sync(0xffffffffu, units), UNITS_MOST);
  longest = __reduce_max_sync(0xffffffffu, longest);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) total += __shfl_xor_sync(0xffffffffu, total, o);
  if (lane == 0) { sums[warp] = total; unit_sums[warp] = units; tops[warp] = longest; }
  if (threadIdx.x == 0) found.s = -1;
  __syncthreads();
  total = lane < WARPS ? sums[lane] : 0;
  units = __reduce_add_sync(0xffffffffu, lane < WARPS ? unit_sums[lane] : 0);
  longest = __reduce_max_sync(0xffffffffu, lane < WARPS ? tops[lane] : 0);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) total += __shfl_xor_sync(0xffffffffu, total, o);
  const Shares shares(total, units, longest);
  long long base = 0;                        // in front of the round
  for (int s0 = 0; s0 < S; s0 += THREADS) {
    const int s = s0 + (int)threadIdx.x;
    const Share x = s0 == 0 ? mine : share_of<C>(p, min(s, S - 1));
    const long long size = s < S ? (shares.whole ? x.units : x.work()) : 0;
    long long in = size;                     // inclusive sums of the warp, then of the block
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const long long y = __shfl_up_sync(0xffffffffu, in, o);
      if (lane >= o) in += y;
    }
    __syncthreads();
    if (lane == 31) sums[warp] = in;
    __syncthreads();
    long long all = lane < WARPS ? sums[lane] : 0, front = lane < warp ? all : 0;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) { all += __shfl_xor_sync(0xffffffffu, all, o); front += __shfl_xor_sync(0xffffffffu, front, o); }
    const long long end = base + front + in;
    if (end - size <= shares.from && shares.from < end) begin_in(found, shares, s, x, end, size, total);
    __syncthreads();
    if (found.s >= 0) break;
    base += all;
  }
  if (threadIdx.x == 0 && found.s < 0) found.f = found.to = 0;                // there is no work for this CTA
  __syncthreads();
}
// by one lane
template <int C>
__device__ __forceinline__ bool walk_on(Walk& w, const AttnP& p) {
  long long f = w.f, base = w.base;
  const long long to = w.to;
  int s = w.s;
  Share x = w.share;
  if (f >= to) return false;
  if (f >= base + x.work()) {                // the next sequence that has work
    do {
      base += x.work();
      x = share_of<C>(p, ++s);
    } while (f >= base + x.work() && s + 1 < p.b.S);
    w.base = base; w.s = s; w.share = x;
  }
  const Tiles<SHIFT> tiles(x.q.before, x.q.before + x.q.n - 1, p.window, p.sinks);
  const long long o = f - base;
  const int u = o < 0x7fffffffll ? (int)((uint32_t)o / (uint32_t)x.places) : (int)(o / x.places), cts = x.units / p.H;
  Part y;
  y.q = x.q; y.s = s; y.h = u / cts; y.ct = u - y.h * cts; y.n_pos = x.places;
  y.u0 = (int)(o - (long long)u * x.places); y.u1 = (int)min((long long)x.places, y.u0 + (to - f));
  y.t0 = max(y.u0 - UNIT_COST, 0); y.n = max(y.u1 - UNIT_COST, 0) - y.t0;
  y.first = tiles.first; y.from = tiles.from;
  w.f = f + y.u1 - y.u0;
  w.now ^= 1;
  w.part[w.now] = y;
  return true;
}
// by the whole warp: the next part, null behind the last
template <int C>
__device__ __forceinline__ const Part* next_part(Walk& w, const AttnP& p) {
  __syncwarp();                              // the part before the one in front has been read
  bool more = false;
  if ((threadIdx.x & 31) == 0) more = walk_on<C>(w, p);
  more = __shfl_sync(0xffffffffu, more, 0);
  __syncwarp();                              // what lane 0 has written is there for all
  return more ? &w.part[w.now] : nullptr;
}

// The products of a tile, by one thread of the warp, and a commit behind them; A in TMEM, 8 columns of two f16 for 16 of k.
// S = Q K^T: K's rows [64 tokens][64 dims], swizzled; the next 16 dims 32 bytes on, the next 64 a half.
#define MMA(k, acc) "@q tcgen05.mma.cta_group::1.kind::f16 [%0], [a" #k "], w" #k ", %3, " acc ";\n\t"
#define ARG(k, by) "add.u32 a" #k ", %1, 8*" #k ";\n\tadd.u32 x, %2, " by ";\n\tmov.b64 w" #k ", {x, %5};\n\t"
#define REGS "{\n\t.reg .pred f, t, q;\n\t.reg .b32 x, a0, a1, a2, a3, a4, a5, a6, a7;\n\t.reg .b64 w0, w1, w2, w3, w4, w5, w6, w7;\n\t"
#define ELECT "setp.ne.b32 t, %5, 0;\n\tsetp.ne.b32 f, %6, 0;\n\telect.sync _|q, 0xffffffff;\n\t"
#define COMMIT "@q tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%4];\n\t}"
template <int D>
__device__ __forceinline__ void scores_of_tile(uint32_t s, uint32_t q, uint32_t k_smem, uint32_t idesc, uint32_t bar) {
  if constexpr (D == 128)
    asm volatile(REGS ARG(0, "0") ARG(1, "2") ARG(2, "4") ARG(3, "6") ARG(4, "512") ARG(5, "514") ARG(6, "516") ARG(7, "518") ELECT
                 MMA(0, "f") MMA(1, "t") MMA(2, "t") MMA(3, "t") MMA(4, "t") MMA(5, "t") MMA(6, "t") MMA(7, "t") COMMIT
                 ::"r"(s), "r"(q), "r"(desc_low(k_smem)), "r"(idesc), "r"(bar), "r"(DESC_HIGH), "r"(0u) : "memory");
  else
    asm volatile(REGS ARG(0, "0") ARG(1, "2") ARG(2, "4") ARG(3, "6") ELECT MMA(0, "f") MMA(1, "t") MMA(2, "t") MMA(3, "t") COMMIT
                 ::"r"(s), "r"(q), "r"(desc_low(k_smem)), "r"(idesc), "r"(bar), "r"(DESC_HIGH), "r"(0u) : "memory");
}
// O (+)= P V: V's rows [64 tokens][64 dims], 16 tokens 2048 bytes on, the next 64 dims a half
__device__ __forceinline__ void sums_of_tile(uint32_t o, uint32_t p, uint32_t v_smem, uint32_t half, uint32_t idesc, uint32_t bar, uint32_t accumulate) {
  asm volatile(REGS ARG(0, "0") ARG(1, "128") ARG(2, "256") ARG(3, "384") ELECT MMA(0, "f") MMA(1, "t") MMA(2, "t") MMA(3, "t") COMMIT
               ::"r"(o), "r"(p), "r"(((v_smem & 0x3FFFFu) >> 4) | ((half >> 4) << 16)), "r"(idesc), "r"(bar), "r"(DESC_HIGH), "r"(accumulate) : "memory");
}
#undef MMA
#undef ARG
#undef REGS
#undef ELECT
#undef COMMIT
#define R8(r, o) "r"((r)[o]), "r"((r)[o + 1]), "r"((r)[o + 2]), "r"((r)[o + 3]), "r"((r)[o + 4]), "r"((r)[o + 5]), "r"((r)[o + 6]), "r"((r)[o + 7])
__device__ __forceinline__ void tmem_st8(uint32_t taddr, const uint32_t* r) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"r"(taddr), R8(r, 0) : "memory");
}
#undef R8
// Two barriers, asked together.
__device__ __forceinline__ void wait_two(uint32_t bar, uint32_t parity, uint32_t bar2, uint32_t parity2, volatile int* quit) {
  uint32_t done;
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t"
      "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
      "mbarrier.try_wait.parity.shared::cta.b64 q, [%3], %4;\n\t"
      "and.pred p, p, q;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(done) : "r"(bar), "r"(parity), "r"(bar2), "r"(parity2) : "memory");
  if (__all_sync(0xffffffffu, done)) return;
  warp_wait(bar, parity, quit);
  warp_wait(bar2, parity2, quit);
}
// A barrier of some of the block's warps, by whole warps: it asks for all lanes of a warp together, which stores and loops of single lanes in front of it may have parted.
__device__ __forceinline__ void meet(int id, int threads) {
  __syncwarp();
  asm volatile("bar.sync %0, %1;" ::"r"(id), "r"(threads) : "memory");
}
template <int ID, int N>
__device__ __forceinline__ void meet() {
  __syncwarp();
  asm volatile("bar.sync %0, %1;" ::"n"(ID), "n"(N) : "memory");
}
// registers of a weight thread; with those of the others they are what the block was launched with
template <int C> constexpr int soft_regs() { return C == 128 ? 168 : 144; }

template <int D, int FMT, int C>
__global__ void __launch_bounds__(THREADS, 1) tree_kernel(const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v, const __grid_constant__ TreeP p) {
  typedef TreeSmem<D> L;
  constexpr int R = 128 / C, HOLD = KEYS / R, SLOTS = L::SLOTS, PAIRS = L::PAIRS;        // HOLD: scores of a weight thread
  // TMEM: scores and weights of the two groups of warps, their sums, the queries
  constexpr uint32_t P_AT = 2 * KEYS, O_AT = P_AT + KEYS, Q_AT = 512 - D / 2;
  static_assert(O_AT + 2 * D <= Q_AT, "TMEM");
  extern __shared__ uint8_t smem_raw[];
  __shared__ __align__(8) uint64_t bars[2 * PAIRS + 4 * STAGES + 5 + INFOS];
  __shared__ __align__(16) TileInfo infos[INFOS];
  __shared__ uint32_t tmem_at;
  __shared__ volatile int quit;              // somebody has waited too long: nobody waits any more, and all go through to the end
  __shared__ int end;                        // number of the converters' jobs, once it is known
  __shared__ float factors[C];               // of a column: what turns a product of codes into a score in base 2, but for the keys' scale
  __shared__ float2 ml[256], total[2][C];
  __shared__ Walk walks[SOFT_WARPS + 2];     // of the weights' warps, the producer and the issuer
  const uint32_t base = (smem_u32(smem_raw) + 1023u) & ~1023u;
  uint8_t* const smem = smem_raw + (base - smem_u32(smem_raw));
  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  const uint32_t bar = smem_u32(bars), c_full = bar, c_empty = c_full + 8 * PAIRS, k_full = c_empty + 8 * PAIRS, v_full = k_full + 8 * STAGES,
                 s_done = v_full + 8 * STAGES, o_done = s_done + 8 * STAGES, p_full = o_done + 8 * STAGES, s_taken = p_full + 16, q_full = s_taken + 16, i_full = q_full + 8;
  if (threadIdx.x == 0) {
    quit = 0;
    end = 0x7fffffff;
    for (int i = 0; i < PAIRS; ++i) { mbar_init(c_full + 8 * i, 1); mbar_init(c_empty + 8 * i, 2); }
    for (int i = 0; i < STAGES; ++i) { mbar_init(k_full + 8 * i, 2); mbar_init(v_full + 8 * i, 2); mbar_init(s_done + 8 * i, 1); mbar_init(o_done + 8 * i, 1); }
    for (int i = 0; i < 2; ++i) { mbar_init(s_taken + 8 * i, 4); mbar_init(p_full + 8 * i, 4); }
    mbar_init(q_full, 4);
    for (int i = 0; i < INFOS; ++i) mbar_init(i_full + 8 * i, 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  __syncthreads();                           // the barriers have begun
  pdl_trigger();
  pdl_wait();
  if (warp == ISSUER) tmem_alloc(smem_u32(&tmem_at), 512);
  Walk& walk = walks[warp < SOFT_WARPS ? warp : warp == PRODUCER ? SOFT_WARPS : SOFT_WARPS + 1];
  const bool walks_on = warp < SOFT_WARPS || warp >= PRODUCER;
  if (p.b.S <= 32) {                         // a warp finds its way without the others
    if (walks_on) start_alone<C>(p, walk);
  } else {
    __shared__ Walk start;
    start_together<C>(p, start);
    if (walks_on && lane == 0) walk = start;
  }
  __syncwarp();                              // registers are taken and given by whole warps
  auto tmem_ready = [&]() {                  // by the issuer and the weights' warps
    tc_fence_before();
    meet<4, (SOFT_WARPS + 1) * 32>();
    tc_fence_after();
    return tmem_at;
  };

  // Tiles are numbered through all parts, g = 0, 1, ..: tile g has the places g % STAGES of keys and values, and the weight warps g & 1; its codes are the jobs 4 g .. 4 g + 3, 32 tokens of keys or values each.
  if (warp >= SOFT_WARPS) {
  asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(256 - soft_regs<C>()));
  if (warp < PRODUCER) {
    // ---- codes into f16 tiles ----
    if (blockIdx.x == 0)                     // until the first come: what every call looks at
      for (int s = (int)threadIdx.x - SOFT_WARPS * 32; s < p.b.S; s += CONVERT_WARPS * 32)
        if (!sequence(p.b, s, p.P).ok) atomicOr(p.flags, B200_PAGED_BAD_BATCH);
    constexpr int LANES = D / 16, STEP = 32 / LANES;     // lanes a row, rows at a time
    const int c = lane % LANES;
    // lanes of a row's second 64 dims take the neighbouring row, so that eight lanes' pieces of the f16 tile lie in different banks
    const int r_in = lane / LANES ^ (D == 128 ? c >> 2 : 0);
    for (int j = warp - SOFT_WARPS;; j += CONVERT_WARPS) {
      const int slot = j % SLOTS, pair = slot >> 1, g = j >> 2, st = g % STAGES, half = j & 1;
      const bool values = j & 2;
      // the codes, and the f16 tile's place: where there are no more jobs, it is free as well
      wait_two(c_full + 8 * pair, (uint32_t)(j / SLOTS) & 1u, (values ? o_done : s_done) + 8 * st, ((uint32_t)(g / STAGES) & 1u) ^ 1u, &quit);
      if (__any_sync(0xffffffffu, quit || j >= *(volatile int*)&end)) break;
      const uint8_t* from = smem + L::CODES + slot * L::SLOT;
      uint8_t* const to = smem + (values ? L::V : L::K) + st * L::TILE + (c >> 2) * L::HALF;
      auto fetch = [&](int r) { return *reinterpret_cast<const uint4*>(from + (D == 128 ? r * 128 + ((c ^ (r & 7)) << 4) : r * 64 + ((c ^ (r >> 1 & 3)) << 4))); };
      auto put = [&](int r, const uint4& x) {
        const int n = 32 * half + r;
        const uint32_t w[4] = {ready<FMT>(x.x), ready<FMT>(x.y), ready<FMT>(x.z), ready<FMT>(x.w)};
        uint8_t* y = to + n * 128;
        *reinterpret_cast<uint4*>(y + (((2 * (c & 3)) ^ (n & 7)) << 4)) = make_uint4(half2_of<FMT, 0>(w[0]), half2_of<FMT, 1>(w[0]), half2_of<FMT, 0>(w[1]), half2_of<FMT, 1>(w[1]));
        *reinterpret_cast<uint4*>(y + (((2 * (c & 3) + 1) ^ (n & 7)) << 4)) = make_uint4(half2_of<FMT, 0>(w[2]), half2_of<FMT, 1>(w[2]), half2_of<FMT, 0>(w[3]), half2_of<FMT, 1>(w[3]));
      };
      const TileInfo& t = infos[g % INFOS];
      if (!values || (t.whole & 2)) {
        uint4 x[32 / STEP];
#pragma unroll
        for (int i = 0; i < 32 / STEP; ++i) x[i] = fetch(i * STEP + r_in);
#pragma unroll
        for (int i = 0; i < 32 / STEP; ++i) put(i * STEP + r_in, x[i]);
      } else {                               // values that no row sees may be anything; keys are masked
#pragma unroll 1
        for (int i = 0; i < 32 / STEP; ++i) {
          const int r = i * STEP + r_in, token = t.j0 + 32 * half + r;
          const bool seen = t.group[2 * half + (r >> 4)].w != 0.f && token <= t.pl && (p.window <= 0 || t.pf - token < p.window || token < p.sinks);
          put(r, seen ? fetch(r) : make_uint4(0, 0, 0, 0));
        }
      }
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      __syncwarp();
      if (lane == 0) { mbar_arrive(c_empty + 8 * pair); mbar_arrive((values ? v_full : k_full) + 8 * st); }
    }
  } else if (warp == PRODUCER) {
    // ---- copies: pages and scales are looked up for eight tiles at a time, a lane for each 16 tokens, and eight tiles ahead ----
    const int groups = min(p.P, KEYS) / 16;  // of 16 tokens, that a copy has
    int g = 0, pair = 0;
    uint32_t parity = 1;                     // of the places' turns: 1: they have not been used yet
    for (const Part* u; (u = next_part<C>(walk, p)) != nullptr;) {
      const int n = u->n, h = u->h, pf = u->q.before, pl = pf + u->q.n - 1;
      const int32_t* const table = p.b.table + u->s * p.b.table_ld;
      auto first_of = [&](int batch) { return (u->tile(8 * batch + (lane >> 2)) << SHIFT) + 16 * (lane & 3); };        // of the lane's tokens
      auto look_up = [&](int batch) {
        const int j = first_of(batch);
        if (8 * batch + (lane >> 2) >= n || j > pl || (p.window > 0 && pf - j - 15 >= p.window && j >= p.sinks)) return -1;
        const int page = table[j >> p.page_shift];
        if (page >= 0 && page < p.pages) return page;
        atomicOr(p.flags, B200_PAGED_BAD_PAGE);
        return -1;
      };
      auto scales_of = [&](int page) { return page < 0 ? make_float2(1.f, 1.f) : make_float2(p.k_scale[(long long)page * p.H + h], p.v_scale[(long long)page * p.H + h]); };
      int page = -1, row = 0, page_next = look_up(0);
      uint32_t there = 0, copies = 0;        // of the batch's groups: those that are there, and those of them that begin a copy
      float2 scale_next = scales_of(page_next);
      for (int x = 0; x < n; ++x, ++g) {
        const int tile = x & 7;
        if (tile == 0) {                     // a batch: a copy is made by the lane of its first group that is there; all of its groups lie in one page
          page = page_next;
          row = (page * p.H + h) * p.P + (first_of(x >> 3) & (p.P - 1) & -16 * groups);
          there = __ballot_sync(0xffffffffu, page >= 0);
          copies = __ballot_sync(0xffffffffu, page >= 0 && !(there & ((1u << lane) - (1u << (lane & -groups)))));
        }
        if (tile == 4) scale_next = scales_of(page_next);
        const int pair_v = pair + 1 == PAIRS ? 0 : pair + 1;
        const uint32_t parity_v = pair + 1 == PAIRS ? parity ^ 1u : parity;
        wait_two(c_empty + 8 * pair, parity, c_empty + 8 * pair_v, parity_v, &quit);
        const uint32_t bytes = (uint32_t)(__popc(copies >> 4 * tile & 15u) * groups * 16 * D);
        if (elected()) mbar_expect_tx(c_full + 8 * pair, bytes);
        __syncwarp();
        const bool makes = (lane >> 2) == tile && (copies >> lane & 1u);
        const uint32_t to = base + L::CODES + (lane & 3 & -groups) * 16 * D;
        if (makes) tma_load_2d(to + 2 * pair * L::SLOT, &map_k, c_full + 8 * pair, 0, row);
        if (tile == 0) {                     // what is to be known of the batch: behind its first keys, which do not wait for scales
          const int j = first_of(x >> 3), j0 = j & ~(KEYS - 1), mine = x + (lane >> 2);
          TileInfo& t = infos[(g + (lane >> 2)) % INFOS];
          const float vs = value_scale(scale_next.y);
          const bool all = (there >> (lane & 28) & 15u) == 15u;
          if (mine < n) {
            t.group[lane & 3] = page >= 0 ? make_float4(scale_next.x > 0.f ? scale_next.x : 1.f, __log2f(vs), __frcp_rn(vs), 1.f) : make_float4(1.f, 0.f, 0.f, 0.f);
            if ((lane & 3) == 0) {
              const bool whole = all && j0 + KEYS <= pf && (p.window <= 0 || pl - j0 < p.window || j0 + KEYS <= p.sinks);
              const bool seen = all && j0 + KEYS - 1 <= pl && (p.window <= 0 || pf - j0 < p.window || j0 + KEYS <= p.sinks);
              t.j0 = j0; t.pf = pf; t.pl = pl; t.whole = (whole ? 1 : 0) | (seen ? 2 : 0);
            }
          }
          __syncwarp();
          if (mine < n && (lane & 3) == 0) mbar_arrive(i_full + 8 * ((g + (lane >> 2)) % INFOS));
          page_next = look_up((x >> 3) + 1);
          __syncwarp();
        }
        // The values' only arrival, behind the infos: their converters read those, and a tile without pages has no copy that would hold the phase open.
        if (elected()) mbar_expect_tx(c_full + 8 * pair_v, bytes);
        __syncwarp();
        if (makes) tma_load_2d(to + 2 * pair_v * L::SLOT, &map_v, c_full + 8 * pair_v, 0, row);
        __syncwarp();
        pair += 2;
        if (pair >= PAIRS) { pair -= PAIRS; parity ^= 1u; }
      }
    }
    if (lane == 0) *(volatile int*)&end = 4 * g;
    __syncwarp();
    for (int k = 0; k < CONVERT_WARPS / 2; ++k) {                             // each converter finds that there is no more
      warp_wait(c_empty + 8 * pair, parity, &quit);
      if (lane == 0) mbar_arrive(c_full + 8 * pair);
      if (++pair == PAIRS) { pair = 0; parity ^= 1u; }
    }
  } else {
    // ---- products ----
    constexpr uint32_t id_s = idesc_f16(KEYS, false), id_o = idesc_f16(D, true);
    const uint32_t tmem = tmem_ready();
    int g0 = 0, part = 0;                    // tiles and parts in front
    for (const Part* u; (u = next_part<C>(walk, p)) != nullptr; ++part) {
      const int n = u->n;
      warp_wait(q_full, (uint32_t)part & 1u, &quit);
      // scores two tiles in front of the sums: a group of warps finds its next ones when it has made its weights
#pragma unroll 1
      for (int x = -2; x < n; ++x) {
        if (x + 2 < n) {
          const int g = g0 + x + 2, st = g % STAGES, i = g & 1;
          if (g >= 2) wait_two(s_taken + 8 * i, (uint32_t)((g - 2) >> 1) & 1u, k_full + 8 * st, (uint32_t)(g / STAGES) & 1u, &quit);
          else warp_wait(k_full + 8 * st, (uint32_t)(g / STAGES) & 1u, &quit);
          tc_fence_after();
          scores_of_tile<D>(tmem + KEYS * i, tmem + Q_AT, base + L::K + st * L::TILE, id_s, s_done + 8 * st);
        }
        if (x >= 0) {
          const int g = g0 + x, st = g % STAGES, i = g & 1;
          wait_two(v_full + 8 * st, (uint32_t)(g / STAGES) & 1u, p_full + 8 * i, (uint32_t)(g >> 1) & 1u, &quit);
          tc_fence_after();
          sums_of_tile(tmem + O_AT + D * i, tmem + P_AT + KEYS / 2 * i, base + L::V + st * L::TILE, L::HALF, id_o, o_done + 8 * st, x > 1 ? 1u : 0u);
        }
      }
      g0 += n;
    }
    __syncwarp();
  }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(soft_regs<C>()));
    // ---- weights: a row per thread, which is a column and HOLD of a tile's keys ----
    if (threadIdx.x == 0) p.split[blockIdx.x] = make_int4(0, 0, 0, 0);
    const uint32_t tmem = tmem_ready();
    const int i = warp >> 2, q4 = warp & 3, in = q4 * 32 + lane, rep = in / C, col = in % C;
    const uint32_t lanes = (uint32_t)(q4 * 32) << 16, ts = tmem + lanes + KEYS * i + rep * HOLD, tp = tmem + lanes + P_AT + KEYS / 2 * i, to = tmem + lanes + O_AT + D * i;
    if constexpr (R > 1) {                   // other copies' keys have no weight here
      const uint32_t zero[16] = {};
#pragma unroll
      for (int k = 0; k < KEYS / 32; ++k) tmem_st16(tp + 16 * k, zero);
      tmem_st_wait();
    }
    // The queries of a part, f16 after a power of two for each column, as rows and heads of very different size may lie side by side.  They come in whole rows, the thread's are piece c of every APART-th column
    // from r_at on (token and head by counting, not by division), go through the place of the joining, HERE columns at a time, and a row per thread into TMEM.
    constexpr int PIECES = D / 8, MINE = C * PIECES / (SOFT_WARPS * 32), APART = SOFT_WARPS * 32 / PIECES, HERE = C < 64 ? C : 64;
    const int c_q = threadIdx.x % PIECES, r_at = threadIdx.x / PIECES;
    uint8_t* const join = smem + L::JOIN;
    uint4 raw[MINE];
    auto load_queries = [&](const Part& u) {
      const int c0 = u.ct * C, n_cols = u.q.n * p.G - c0, step_t = APART / p.G, step_g = APART - step_t * p.G;
      int token = (c0 + r_at) / p.G, head = c0 + r_at - token * p.G;
      const bf16* const q0 = p.q + (long long)u.q.r0 * p.q_ld + (long long)u.h * p.G * D + 8 * c_q;
#pragma unroll
      for (int k = 0; k < MINE; ++k) {
        raw[k] = r_at + k * APART < n_cols ? *reinterpret_cast<const uint4*>(q0 + token * p.q_ld + head * D) : make_uint4(0, 0, 0, 0);
        token += step_t; head += step_g;
        if (head >= p.G) { head -= p.G; ++token; }
      }
    };
    auto put_queries = [&]() {
#pragma unroll
      for (int k = 0; k < MINE; ++k) {
        uint32_t v[4] = {raw[k].x, raw[k].y, raw[k].z, raw[k].w}, top = 0;    // magnitudes as numbers, which order like the values
#pragma unroll
        for (int e = 0; e < 4; ++e) top = max(top, max(v[e] << 16 & 0x7fff0000u, v[e] & 0x7fff0000u));
#pragma unroll
        for (int o = PIECES / 2; o > 0; o >>= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
        // A column that is not finite gets NaN, and no other: it asks as zeros, whose weights say whether it sees anything at all, and its factor tells the end of it.
        const bool odd = top >= 0x7f800000u;
        const float power = top && !odd ? power_of_two_in(__uint_as_float(top)) : 1.f, up = __uint_as_float((268u << 23) - __float_as_uint(power));     // 2^14 / power
        if (c_q == 0) factors[r_at + k * APART] = odd ? NAN : power * (1.f / 16384.f) * p.scale2;
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = odd ? 0u : pack_f16(__uint_as_float(v[e] << 16) * up, __uint_as_float(v[e] & 0xffff0000u) * up);
        raw[k] = make_uint4(v[0], v[1], v[2], v[3]);
      }
#pragma unroll
      for (int round = 0; round < C / HERE; ++round) {
#pragma unroll
        for (int k = round * (MINE * HERE / C); k < (round + 1) * (MINE * HERE / C); ++k) {
          const int r = r_at + k * APART - round * HERE;
          *reinterpret_cast<uint4*>(join + r * 2 * D + ((c_q ^ (r & 7)) << 4)) = raw[k];
        }
        meet<1, SOFT_WARPS * 32>();    // all columns' factors, too
        if (i == 0 && (C / HERE == 1 || warp / (4 / (C / HERE)) == round)) {
          const uint8_t* mine = join + col % HERE * 2 * D;
#pragma unroll 2
          for (int k = 0; k < PIECES; k += 4) {
            uint32_t v[16];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const uint4 x = *reinterpret_cast<const uint4*>(mine + (((k + e) ^ (col & 7)) << 4));
              v[4 * e] = x.x; v[4 * e + 1] = x.y; v[4 * e + 2] = x.z; v[4 * e + 3] = x.w;
            }
            tmem_st16(tmem + lanes + Q_AT + 4 * k, v);
          }
          tmem_st_wait();
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(q_full);
        }
        meet<1, SOFT_WARPS * 32>();    // the place is free again
      }
    };
    float fac = 0.f, m = -INFINITY, sum = 0.f;
    int g0 = 0, done = 0;                    // tiles in front of the part; this group of warps' of the part
    const Part* next = next_part<C>(walk, p);            // a run has a part at least
    for (const Part* now = nullptr;;) {
      // The next part's queries come in beside the end of this one, and its first scores are made while this one's rows are joined.
      if (next != nullptr) load_queries(*next);
      if (now != nullptr) {
        ml[128 * i + in] = make_float2(m, sum);
        meet<1, SOFT_WARPS * 32>();    // every score has been made
      }
      if (next != nullptr) put_queries();
      if (now != nullptr) {
        const Part& u = *now;
        const bool alone = u.u0 == 0 && u.u1 == u.n_pos;
        if (u.n > 0) {                       // the last tile's sum, and with it all in front
          const int g = g0 + u.n - 1;
          warp_wait(o_done + 8 * (g % STAGES), (uint32_t)(g / STAGES) & 1u, &quit);
        }
        tc_fence_after();
        // Join the column's 2 R rows.  Both groups' sums of a row lie in the row's lane: the first group of warps has half of the dims of both, the second the rest; the R copies go through shared memory.
        float top = -INFINITY, all = 0.f;
#pragma unroll
        for (int k = 0; k < 2 * R; ++k) top = fmaxf(top, ml[k * C + col].x);
#pragma unroll
        for (int k = 0; k < 2 * R; ++k) {
          const float2 y = ml[k * C + col];
          all = fmaf(y.y, y.x == -INFINITY ? 0.f : exp2_fast(y.x - top), all);
        }
        float by[2];
#pragma unroll
        for (int k = 0; k < 2; ++k) by[k] = ml[128 * k + in].x == -INFINITY ? 0.f : exp2_fast(ml[128 * k + in].x - top);
        if (all != 0.f && isnan(fac)) all = NAN;
        const int r0 = u.q.r0, c0 = u.ct * C, n_cols = u.q.n * p.G - c0, slot = 2 * (int)blockIdx.x + (u.u0 == 0 ? 1 : 0);
        constexpr int PIECE = D / 8;         // dims at a time
        uint32_t o[2][PIECE];
        auto fetch_sums = [&](int d0) {
#pragma unroll
          for (int k = 0; k < 2; ++k) {
            const uint32_t at = tmem + lanes + O_AT + D * k + d0;
            if constexpr (PIECE == 16) tmem_ld16(at, o[k]); else tmem_ld8(at, o[k]);
          }
        };
        auto both_sums = [&](float* v) {     // a group that has seen nothing may have anything there
#pragma unroll
          for (int k = 0; k < 2; ++k) { if constexpr (PIECE == 16) tmem_ld_wait16(o[k]); else tmem_ld_wait8(o[k]); }
#pragma unroll
          for (int e = 0; e < PIECE; ++e) {
            v[e] = by[0] != 0.f ? __uint_as_float(o[0][e]) * by[0] : 0.f;
            if (by[1] != 0.f) v[e] = fmaf(__uint_as_float(o[1][e]), by[1], v[e]);
          }
        };
        float4* const parts = reinterpret_cast<float4*>(p.part_o) + (long long)slot * (D / 4) * C;           // [D / 4][C]
        if constexpr (R == 1) {              // a thread has its column alone
          const int cc = c0 + col, t_out = cc / p.G;
          const float inv = all != 0.f ? 1.f / all : 0.f;
          bf16* const out = p.out + (r0 + t_out) * p.out_ld + (long long)(u.h * p.G + cc - t_out * p.G) * D;
          const long long at = (long long)slot * C + col;
          if (!alone && i == 0 && col < n_cols) *reinterpret_cast<float2*>(p.part_ml + 2 * at) = make_float2(top, all);
#pragma unroll 1
          for (int c = 0; c < 4; ++c) {
            const int d0 = (4 * i + c) * PIECE;
            float v[PIECE];
            __syncwarp();                    // sums are read by whole warps, and some lanes may have had a column in front of this
            fetch_sums(d0);
            both_sums(v);
            if (col < n_cols) {
#pragma unroll
              for (int e = 0; e < PIECE; e += 8) {
                if (alone) {
                  *reinterpret_cast<uint4*>(out + d0 + e) = make_uint4(pack_bf16(v[e] * inv, v[e + 1] * inv), pack_bf16(v[e + 2] * inv, v[e + 3] * inv), pack_bf16(v[e + 4] * inv, v[e + 5] * inv), pack_bf16(v[e + 6] * inv, v[e + 7] * inv));
                } else {
                  parts[(d0 + e) / 4 * C + col] = make_float4(v[e], v[e + 1], v[e + 2], v[e + 3]);
                  parts[(d0 + e + 4) / 4 * C + col] = make_float4(v[e + 4], v[e + 5], v[e + 6], v[e + 7]);
                }
              }
            }
          }
        } else {
          if (rep == 0) total[i][col] = make_float2(top, all);
          __syncwarp();
          // LINE threads a column, whose results lie side by side
          constexpr int LINE = PIECE / 4, AT_ONCE = 128 / LINE;
          auto place = [](int row, int e) { return row * PIECE * 4 + ((e ^ (D == 128 ? row >> 1 & 3 : row >> 2 & 1)) << 4); };
          const int d_out = in % LINE, c_first = in / LINE;
          uint8_t* const mine = join + i * (128 * PIECE * 4);
          fetch_sums(4 * i * PIECE);
#pragma unroll 1
          for (int c = 0; c < 4; ++c) {
            const int d0 = (4 * i + c) * PIECE;
            float v[PIECE];
            both_sums(v);
#pragma unroll
            for (int e = 0; e < LINE; ++e) *reinterpret_cast<float4*>(mine + place(in, e)) = make_float4(v[4 * e], v[4 * e + 1], v[4 * e + 2], v[4 * e + 3]);
            if (c < 3) fetch_sums(d0 + PIECE);           // on their way beside this piece
            meet(2 + i, 128);
#pragma unroll
            for (int c_out = c_first; c_out < C; c_out += AT_ONCE) {
              if (c_out >= n_cols) break;
              float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
              for (int k = 0; k < R; ++k) {
                const float4 y = *reinterpret_cast<const float4*>(mine + place(k * C + c_out, d_out));
                acc.x += y.x; acc.y += y.y; acc.z += y.z; acc.w += y.w;
              }
              const float2 tl = total[i][c_out];
              if (alone) {
                const int cc = c0 + c_out, t_out = cc / p.G;
                const float inv = tl.y != 0.f ? 1.f / tl.y : 0.f;
                bf16* out = p.out + (r0 + t_out) * p.out_ld + (long long)(u.h * p.G + cc - t_out * p.G) * D + d0 + 4 * d_out;
                *reinterpret_cast<uint2*>(out) = make_uint2(pack_bf16(acc.x * inv, acc.y * inv), pack_bf16(acc.z * inv, acc.w * inv));
              } else {
                const long long at = (long long)slot * C + c_out;
                if (i == 0 && c == 0 && d_out == 0) *reinterpret_cast<float2*>(p.part_ml + 2 * at) = tl;
                parts[(d0 / 4 + d_out) * C + c_out] = acc;
              }
            }
            meet(2 + i, 128);
          }
        }
        g0 += u.n;
        tc_fence_before();
        meet<1, SOFT_WARPS * 32>();    // both groups have read both sums
      }
      if (next == nullptr) break;
      now = next;
      const Part& u = *next;
      if (u.u1 < u.n_pos && threadIdx.x == 0) {
        const int runs = (int)min(walk.run, 1ll << 30), back = (u.u0 + runs - 1) / runs;
        p.split[blockIdx.x] = make_int4(u.s, u.h, u.ct, (back + (u.n_pos - u.u1 + runs - 1) / runs) | back << 16);
      }
      fac = factors[col]; m = -INFINITY; sum = 0.f; done = 0;
      next = next_part<C>(walk, p);
      if (next != nullptr) {                 // its queries into L2
        const int cc = next->ct * C + (int)threadIdx.x % C, token = cc / p.G;
        const bf16* row = p.q + (next->q.r0 + token) * p.q_ld + (long long)(next->h * p.G + cc - token * p.G) * D;
        if (cc < next->q.n * p.G && (int)threadIdx.x < C * (D / 64)) asm volatile("prefetch.global.L2 [%0];" ::"l"(row + (int)threadIdx.x / C * 64));
      }
      for (int x = (g0 + i) & 1; x < u.n; x += 2, ++done) {
        const int g = g0 + x;
        wait_two(i_full + 8 * (g % INFOS), (uint32_t)(g / INFOS) & 1u, s_done + 8 * (g % STAGES), (uint32_t)(g / STAGES) & 1u, &quit);
        tc_fence_after();
        const TileInfo& info = infos[g % INFOS];
        const float4* ip = info.group + rep * HOLD / 16;
        uint32_t r[HOLD];                    // the row's scores
        float t = -INFINITY, by[HOLD / 16], lv[HOLD / 16];  // score in base 2 = product * by + lv; by > 0, so that the largest score of a page's keys is that of their largest product
        if constexpr (HOLD == 16) {
          tmem_ld16(ts, r);
          tmem_ld_wait16(r);
        } else {
#pragma unroll
          for (int c = 0; c < HOLD; c += 32) tmem_ld32(ts + c, r + c);
#pragma unroll
          for (int c = 0; c < HOLD; c += 32) tmem_ld_wait32(r + c);
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(s_taken + 8 * i);
        if (!(info.whole & 1)) {             // keys that the row does not see: a bit for each of 32
          const int before = info.pf, last = info.pl, cc = u.ct * C + col, token = cc / p.G;
          const bool has = cc < u.q.n * p.G;
          const int pos = has ? p.position[u.q.r0 + token] : -1, lo = p.window > 0 ? pos - p.window : -1;     // of what is cached: sees j > lo or j < sinks
          const uint32_t* const seen_row = p.seen + (long long)(u.q.r0 + token) * p.words;
#pragma unroll
          for (int c = 0; c < HOLD; c += 32) {
            const int at = info.j0 + rep * HOLD + c, off = at - before;
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
            if (ip[c / 16].w == 0.f) seen &= 0xffff0000u;
            if (HOLD > 16 && ip[HOLD > 16 ? c / 16 + 1 : 0].w == 0.f) seen &= 0xffffu;
#pragma unroll
            for (int e = 0; e < 32 && e < HOLD; ++e)
              if (!(seen >> e & 1u)) r[c + e] = 0xff800000u;
          }
        }
#pragma unroll
        for (int b = 0; b < HOLD / 16; ++b) {
          by[b] = fmaxf(ip[b].x * fac, FLT_MIN);                              // also where fac is NaN
          lv[b] = ip[b].y;
          float mx[2] = {__uint_as_float(r[16 * b]), __uint_as_float(r[16 * b + 1])};
#pragma unroll
          for (int e = 2; e < 16; ++e) mx[e & 1] = fmaxf(mx[e & 1], __uint_as_float(r[16 * b + e]));
          t = fmaxf(t, fmaf(fmaxf(mx[0], mx[1]), by[b], lv[b]));
        }
        const bool grow = t > __fadd_rd(m, SLACK);     // rounded down: above 2^27 the sum would else round to the score itself, and its weight to infinity
        if (done > 0) {                      // the sum over this group's tile in front has read its weights and settled in O
          warp_wait(o_done + 8 * ((g - 2) % STAGES), (uint32_t)((g - 2) / STAGES) & 1u, &quit);
          tc_fence_after();
        }
        if (__any_sync(0xffffffffu, grow)) {
          const float now = t - UNDER, factor = grow ? exp2_fast(m - now) : 1.f;
          if (grow) { m = now; sum *= factor; }
          __syncwarp();
          if (done > 0) {
#pragma unroll 1
            for (int c = 0; c < D / 16; ++c) {           // seldom: short code
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
          for (int e = 0; e < HOLD; ++e) r[e] = __float_as_uint(fmaf(__uint_as_float(r[e]), by[e / 16], lv[e / 16]));
#pragma unroll
          for (int b = 0; b < HOLD / 16; ++b) { by[b] = 1.f; lv[b] = 0.f; }
        }
#pragma unroll
        for (int b = 0; b < HOLD / 16; ++b) {
          const uint64_t by2 = two(by[b]), add = two(lv[b] - off);
          uint64_t part = 0;
          uint32_t w[8];
#pragma unroll
          for (int e = 0; e < 16; e += 2) {
            float e0, e1;
            apart(fma2(together(__uint_as_float(r[16 * b + e]), __uint_as_float(r[16 * b + e + 1])), by2, add), e0, e1);
            e0 = exp2_fast(e0); e1 = exp2_fast(e1);
            part = add2(part, together(e0, e1));
            w[e >> 1] = pack_f16(e0, e1);
          }
          float s0, s1;
          apart(part, s0, s1);
          sum = fmaf(s0 + s1, ip[b].z, sum);
          tmem_st8(tp + rep * (HOLD / 2) + 8 * b, w);
        }
        tmem_st_wait();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(p_full + 8 * i);
      }
    }
  }
  __syncthreads();
  tc_fence_after();
  if (warp == ISSUER) tmem_dealloc(tmem_at, 512);
  if (quit) {                                // let copies in flight land before the block ends
    if (threadIdx.x == 0) atomicOr(p.flags, B200_PAGED_WAIT);
    const uint64_t since = global_timer_ns();
    while (global_timer_ns() - since < 2000000ull) {}
  }
}

// Joins the units that are cut, four dims of a column a thread (parts are [D / 4][C] of those; a warp has 4 columns and 8 such pieces, so that reads and writes are whole sectors).  A block has 16 columns of the unit that
// its CTA has begun; where there are many parts it has four, two or one of them, 4, 8 or 16 threads to a piece that take the parts in turn, and the blocks of the CTAs that have middles of the unit have the others.  (Many: four at least, as the blocks of
// fewer could not cover 16 columns each, four at a time.  With 4, 8, 16: 100 columns of one head on 3000 tokens 16.0, 16.7, 16.8 us, on 9500 16.8, 16.7, 19.6, on 131000 39.8, 39.6, 45.3; with none 97.)
constexpr int JOIN_COLS = 16, MANY_PARTS = 4;
template <int D, int C>
__global__ void __launch_bounds__(JOIN_COLS * D / 4) tree_join_kernel(const TreeP p) {
  pdl_trigger();
  pdl_wait();
  constexpr int QUADS = D / 4, BLOCKS = C / JOIN_COLS;   // pieces of a column; blocks of a CTA
  __shared__ float4 o_s[JOIN_COLS * QUADS];
  __shared__ float2 ml_s[JOIN_COLS * QUADS];
  const int4 of = p.split[blockIdx.x / BLOCKS];
  const int parts = of.w & 0xffff, back = of.w >> 16, block = (int)blockIdx.x % BLOCKS, cta = (int)blockIdx.x / BLOCKS - back;
  const bool many = parts >= MANY_PARTS;
  const int cols = parts >= 16 ? 1 : parts >= 8 ? 2 : 4, threads = QUADS * cols, teams = many ? JOIN_COLS / cols : 1;
  if (parts == 0 || (many ? (back * BLOCKS + block) * cols >= C : back > 0)) return;        // parts * BLOCKS * cols >= C
  const Seq q = sequence(p.b, of.x, p.P);
  const int n_cols = q.n * p.G - of.z * C, team = (int)threadIdx.x / threads, in = (int)threadIdx.x % threads, quad = in / cols;
  const int col = cols * (many ? back * BLOCKS + block : 4 * block + team) + in % cols;
  float top = -INFINITY, sum = 0.f;
  float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
  auto add = [&](float y_top, float y_sum, const float4& v) {
    const float now = fmaxf(top, y_top), keep = now == -INFINITY ? 0.f : exp2_fast(top - now), by = now == -INFINITY ? 0.f : exp2_fast(y_top - now);
    top = now;
    sum = fmaf(sum, keep, y_sum * by);
    acc.x = fmaf(acc.x, keep, v.x * by); acc.y = fmaf(acc.y, keep, v.y * by); acc.z = fmaf(acc.z, keep, v.z * by); acc.w = fmaf(acc.w, keep, v.w * by);
  };
  if (col < n_cols) {
    // the first part is its run's last, the others are their runs' first
#pragma unroll 2
    for (int i = many ? team : 0; i <= parts; i += teams) {
      const long long slot = 2 * (cta + i) + (i == 0 ? 1 : 0);
      const float2 y = reinterpret_cast<const float2*>(p.part_ml)[slot * C + col];
      add(y.x, y.y, reinterpret_cast<const float4*>(p.part_o)[(slot * QUADS + quad) * C + col]);
    }
  }
  if (many) {
    o_s[threadIdx.x] = acc; ml_s[threadIdx.x] = make_float2(top, sum);
    __syncthreads();
    if (team) return;
    for (int k = in + threads; k < JOIN_COLS * QUADS; k += threads) add(ml_s[k].x, ml_s[k].y, o_s[k]);
  }
  if (col >= n_cols) return;
  const int cc = of.z * C + col, token = cc / p.G;
  const float inv = sum != 0.f ? 1.f / sum : 0.f;
  bf16* out = p.out + (q.r0 + token) * p.out_ld + (long long)(of.y * p.G + cc - token * p.G) * D + 4 * quad;
  *reinterpret_cast<uint2*>(out) = make_uint2(pack_bf16(acc.x * inv, acc.y * inv), pack_bf16(acc.z * inv, acc.w * inv));
}

// =========================================================================================================================
// host
// =========================================================================================================================
struct TreePlan { int cols, ctas; FewPlan few; };      // few.units: the columns of a sequence are few enough for the kernel of few rows
// Up to few_cols columns go to the kernel of few rows, the border that steps without a tree have.  Both sides (there / as 32 columns here, us; int8, 3000 tokens, 32 heads on 8; 1, 16, 64 requests).  Head size 128: 8 columns
// 13.7, 29, 80 / 16, 34, 104; 16 columns 18.9, 42, 110 / 16.2, 34, 107; 48 sessions of 12 rows, 32 heads of their own, 200 / 189.  Head size 64: 8 columns 11.9, 23, 63 / 14.2, 28, 84; 16 columns 16.1, 30, 82 / 14.4, 28, 85;
// 32 columns 25, 47, 128 / 14.4, 29, 87.  For trees the border is thus too high: from 9 columns on (17 at head size 64) this side is the quicker one.
TreePlan tree_plan(const b200_paged_cache* c, const b200_paged_batch* b, int G, int window, int sinks) {
  TreePlan f;
  memset(&f, 0, sizeof(f));
  const long long cols = (long long)b->max_rows * G;
  if (cols <= few_cols(c->dim)) {
    f.few = few_plan(c, b, G, window, sinks, 0x7fffffff);
    return f;
  }
  f.cols = cols <= 32 ? 32 : cols <= 64 ? 64 : 128;
  long long keys = (long long)b->table_width * c->page_tokens;
  if (window > 0 && (long long)window + sinks + b->max_rows < keys) keys = (long long)window + sinks + b->max_rows;
  const long long units = (long long)b->sequences * c->kv_heads * ceil_div64(cols, f.cols), runs = ceil_div64(units * (ceil_div64(keys, KEYS) + 1 + UNIT_COST), MIN_RUN);
  f.ctas = (int)(runs < 148 ? runs : 148);
  return f;
}
// sums and (maximum, sum of the weights) of two parts per CTA, and the units that are cut
int64_t tree_bytes(const TreePlan& f, int D) { return f.few.units ? few_bytes(f.few, D) : (int64_t)f.ctas * (2 * f.cols * (D + 2) * 4 + 16); }

template <int D, int FMT, int C>
int launch(const TreeP& p, int ctas, cudaStream_t st) {
  static std::atomic<uint64_t> limits{0};
  static std::atomic<uint64_t> shares{0};
  CUtensorMap map_k, map_v;
  B200_TRY(code_map(&map_k, p.k, (long long)p.pages * p.H * p.P, D, p.P < KEYS ? p.P : KEYS));
  B200_TRY(code_map(&map_v, p.v, (long long)p.pages * p.H * p.P, D, p.P < KEYS ? p.P : KEYS));
  B200_TRY(allow_smem(limits, (int)TreeSmem<D>::BYTES, tree_kernel<D, FMT, C>));
  B200_TRY(prefer_smem(shares, 100, tree_kernel<D, FMT, C>, tree_join_kernel<D, C>));
  B200_TRY(launch_early(tree_kernel<D, FMT, C>, dim3((unsigned)ctas), dim3(THREADS), TreeSmem<D>::BYTES, st, map_k, map_v, p));
  return launch_early(tree_join_kernel<D, C>, dim3((unsigned)(ctas * (C / JOIN_COLS))), dim3(JOIN_COLS * D / 4), 0, st, p);
}
template <int D, int FMT>
int launch_cols(const TreeP& p, const TreePlan& f, cudaStream_t st) {
  if constexpr (few_cols(D) < 32)            // at head size 64 so few columns go to the kernel of few rows
    if (f.cols == 32) return launch<D, FMT, 32>(p, f.ctas, st);
  return f.cols == 64 ? launch<D, FMT, 64>(p, f.ctas, st) : launch<D, FMT, 128>(p, f.ctas, st);
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
  const bool empty = batch->total_rows == 0 || batch->max_rows == 0;
  if (!tree || (!empty && (!tree->seen_dev || !tree->position_dev))) B200_FAIL(B200_ERR_INVALID, "paged_tree_attention: null pointer in the tree");
  if (batch->max_rows > MAX_NODES || tree->words < 1 || (long long)tree->words * 32 < batch->max_rows || tree->words > MAX_NODES / 32)
    B200_FAIL(B200_ERR_SHAPE, "paged_tree_attention: trees of up to %d tokens (at most %d), masks of %d words", batch->max_rows, MAX_NODES, tree->words);
  if (empty) return B200_OK;
  const TreePlan f = tree_plan(cache, batch, p.G, window, sinks);
  const int64_t need = tree_bytes(f, cache->dim);
  if (f.few.units > 0x7fffffffll / 64) B200_FAIL(B200_ERR_SHAPE, "paged_tree_attention: %d sequences with %d heads in one call", batch->sequences, q_heads);
  if (need > 0 && (!work_dev || work_bytes < need || (reinterpret_cast<uintptr_t>(work_dev) & 15)))
    B200_FAIL(B200_ERR_INVALID, "paged_tree_attention: a workspace of %lld bytes; b200_paged_tree_attention_bytes asks for %lld, on a 16-byte border", (long long)work_bytes, (long long)need);
  DeviceGuard guard(cache->device);
  p.seen = tree->seen_dev; p.position = tree->position_dev; p.words = tree->words;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const bool i8 = cache->kv_dtype == B200_KV_INT8;
  if (f.few.units) {
    p.from_rows = 0x7fffffff;
    B200_TRY(few_attention(p, f.few, i8 ? INT8 : E4M3, cache->dim, true, work_dev, st));
    return check_launch("paged_tree_attention");
  }
  p.part_o = static_cast<float*>(work_dev);
  p.part_ml = p.part_o + (long long)f.ctas * 2 * f.cols * cache->dim;
  p.split = reinterpret_cast<int4*>(p.part_ml + (long long)f.ctas * 2 * f.cols * 2);
  if (cache->dim == 128) B200_TRY((i8 ? launch_cols<128, INT8>(p, f, st) : launch_cols<128, E4M3>(p, f, st)));
  else B200_TRY((i8 ? launch_cols<64, INT8>(p, f, st) : launch_cols<64, E4M3>(p, f, st)));
  return check_launch("paged_tree_attention");
}

}  // extern "C"
