// A cache of keys and values in 8 bits whose memory goes to sequences page by page: append with the position rotation on the way, reading back, and attention
// of few rows per sequence (decoding, drafts); long portions are paged_prompt.cu's.
//
// Codes lie as [pages][kv heads][tokens of a page][dim], int8 or e4m3, with one scale per page, head and side (keys, values): a page's tokens of one head are one
// run of memory.  A page's scale s is (largest magnitude) / (largest code) of the rows that began the page; rows that come later may need more, and then
// it is doubled until they fit and the older codes are halved as often.  Only doubling keeps a page that grows token by token within one step of its last scale:
// a half step from the first rounding, and halves, quarters .. of it from those before.  (Growing to the exact maximum each time, the roundings of a slowly growing page all have the
// same sign: 0.1 % a token never changes a code, and after 64 tokens the largest are 8 steps off.)  For e4m3 halving is exact but for subnormals.
#include "paged.cuh"

namespace b200 {
namespace paged {

namespace {

using tcp::pdl_trigger;
using tcp::pdl_wait;
typedef __nv_bfloat16 bf16;

__device__ __forceinline__ void flag(int32_t* flags, int bit) { atomicOr(flags, bit); }
__device__ __forceinline__ uint32_t pack_bf16(float a, float b) {
  const __nv_bfloat162 v = __floats2bfloat162_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&v);
}
__device__ __forceinline__ float2 unpack_bf16(uint32_t w) { return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u)); }

// =========================================================================================================================
// append
// =========================================================================================================================
struct AppendP {
  uint8_t *k_codes, *v_codes;
  float *k_scale, *v_scale;
  int32_t* flags;
  Batch b;
  const bf16 *k, *v, *q;
  bf16* q_out;
  long long k_ld, v_ld, q_ld, q_out_ld;
  const uint64_t* turns;                     // per pair of dimensions: turns per position as a 64-bit fraction; null: no rotation
  int rot, halves;                           // rotated dimensions; pairs are (j, j + rot / 2), else (2j, 2j + 1)
  const int32_t* positions;                  // positions of the rows' own: [axes][positions_ld]
  const uint8_t* pair_axis;                  // per pair: the axis whose position turns it; null: the first
  long long positions_ld;
  int axes;
  int pages, P, H, Hq, items, heads_per_block, page_ctas, q_rows;            // items: numbers of touched pages
};

// Sixteen dimensions of a row: eight from `lo` on and eight from `hi` on, so that a rotated pair is always in one thread's hands.
struct Chunk {
  int lo, hi;
  bool turned;
  __device__ __forceinline__ Chunk(int j, int rot, int halves) {
    turned = 16 * j < rot;
    const bool split = turned && halves;
    lo = split ? 8 * j : 16 * j;
    hi = split ? rot / 2 + 8 * j : 16 * j + 8;
  }
};
struct Turn { float sn[8], cs[8]; };
// The angle of a position is its product with the turns per position, of which only the fraction counts: 64-bit fixed point drops whole turns
// exactly, where an angle in fp32 is off by 0.03 at position 10^6.
__device__ __forceinline__ void turn_of(Turn& t, const uint64_t* turns, int j, int pos) {
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int part = (int)((turns[8 * j + i] * (uint64_t)pos) >> 32);
    sincospif((float)part * 4.656612873077393e-10f, &t.sn[i], &t.cs[i]);      // 2^-31: half turns
  }
}
// The same at positions of row r's own, one for each axis.
__device__ __forceinline__ void turn_of_row(Turn& t, const AppendP& p, int j, int r) {
  int at[4];
#pragma unroll
  for (int a = 0; a < 4; ++a) at[a] = a < p.axes ? p.positions[a * p.positions_ld + r] : 0;
  const uint2 which = p.pair_axis ? *reinterpret_cast<const uint2*>(p.pair_axis + 8 * j) : make_uint2(0, 0);
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const uint32_t a = (i < 4 ? which.x : which.y) >> (8 * (i & 3)) & 255u;
    const int pos = a == 1 ? at[1] : a == 2 ? at[2] : a == 3 ? at[3] : at[0];
    const int part = (int)((p.turns[8 * j + i] * (uint64_t)(int64_t)pos) >> 32);         // whole turns drop out of negative products likewise
    sincospif((float)part * 4.656612873077393e-10f, &t.sn[i], &t.cs[i]);
  }
}
// OWN: the rows have positions of their own, else a row's position is its place in the sequence.
template <bool OWN>
__device__ __forceinline__ void turn(Turn& t, const AppendP& p, int j, int pos, int r) {
  if constexpr (OWN) turn_of_row(t, p, j, r);
  else turn_of(t, p.turns, j, pos);
}
__device__ __forceinline__ void unpack16(float* x, const uint4* raw) {
  const uint32_t w[8] = {raw[0].x, raw[0].y, raw[0].z, raw[0].w, raw[1].x, raw[1].y, raw[1].z, raw[1].w};
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float2 f = unpack_bf16(w[i]);
    x[2 * i] = f.x; x[2 * i + 1] = f.y;
  }
}
__device__ __forceinline__ void load16(float* x, const bf16* row, const Chunk& c) {
  const uint4 raw[2] = {*reinterpret_cast<const uint4*>(row + c.lo), *reinterpret_cast<const uint4*>(row + c.hi)};
  unpack16(x, raw);
}
__device__ __forceinline__ void rotate16(float* x, const Turn& t, int halves) {
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    float& a = halves ? x[i] : x[2 * i];
    float& b = halves ? x[8 + i] : x[2 * i + 1];
    const float re = a * t.cs[i] - b * t.sn[i], im = a * t.sn[i] + b * t.cs[i];
    a = re; b = im;
  }
}

// Which sequence and page the step's touched page number `item` is.  They are numbered without a pass over the sequences: sequence s has the numbers from rows[s] / P + 2 s on, and n rows
// from any place in a page on touch at most n / P + 2 pages.  The whole warp asks together.
struct Page { int first, page, o, e, r; bool ok; };      // position of its first slot; slots o .. e - 1 are the step's, from batch row r on
__device__ __forceinline__ Page page_of(const AppendP& p, int item, bool tell) {
  const int lane = threadIdx.x & 31;
  int s = 0;                                            // the last sequence whose numbers begin at or in front of `item`
  for (int i = lane + 1; i - lane - 1 < p.b.S - 1; i += 32) s += __popc(__ballot_sync(0xffffffffu, i < p.b.S && (long long)p.b.rows[i] / p.P + 2ll * i <= item));
  const Seq q = sequence(p.b, s, p.P);
  Page g;
  g.ok = false;
  const int nth = item - (q.r0 / p.P + 2 * s);          // of the sequence's pages; negative for numbers in front of the first sequence's, and for some of rows out of order
  if (!q.ok || nth < 0) return g;
  const int block = q.before / p.P + nth;
  const long long first = (long long)block * p.P;
  if (q.n == 0 || first >= (long long)q.before + q.n) return g;
  g.page = p.b.table[s * p.b.table_ld + block];
  if (g.page < 0 || g.page >= p.pages) {
    if (tell) flag(p.flags, B200_PAGED_BAD_PAGE);
    return g;
  }
  g.first = (int)first;
  g.o = max(q.before - g.first, 0);
  g.e = (int)min((long long)q.before + q.n - first, (long long)p.P);
  g.r = q.r0 + (g.first + g.o - q.before);
  g.ok = true;
  return g;
}
// A page's scale for new rows whose largest magnitude is `top`; doublings: how often the older rows' codes are halved, -1: they become 0.
template <int FMT>
__device__ __forceinline__ float scale_for(float top, int older, float s_old, int* doublings) {
  const float need = top > 0.f ? fmaxf(top / code_max<FMT>(), SCALE_MIN) : 0.f;
  *doublings = 0;
  if (older == 0) return need;
  if (!(s_old > 0.f)) { *doublings = -1; return need; }
  if (!(need > s_old)) return s_old;
  const float ratio = need / s_old;                     // the least power of two with s_old * 2^k >= need
  int power;
  const float part = frexpf(ratio, &power);
  *doublings = part == 0.5f ? power - 1 : power;
  return ldexpf(s_old, *doublings);
}
template <int FMT>
__device__ __forceinline__ void store16(uint8_t* row, const Chunk& c, const float* x, float scale) {
  // x / scale, rounded like a division, by Markstein's correction (IBM Journal of Research and Development 34, 1990): a product with the rounded reciprocal, and what it left over, exact in an FMA, once more.
  // (Scales lie between 2^-60 and 2^58 and |x| <= 2^64: nothing overflows, and what underflows is 0 as a code.)
  const float div = scale > 0.f ? scale : 1.f, inv = 1.f / div;
  float y[16];
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    const float q = x[i] * inv;
    y[i] = fmaf(fmaf(-q, div, x[i]), inv, q);
  }
  *reinterpret_cast<uint2*>(row + c.lo) = make_uint2(codes4<FMT>(y[0], y[1], y[2], y[3]), codes4<FMT>(y[4], y[5], y[6], y[7]));
  *reinterpret_cast<uint2*>(row + c.hi) = make_uint2(codes4<FMT>(y[8], y[9], y[10], y[11]), codes4<FMT>(y[12], y[13], y[14], y[15]));
}
template <int FMT>
__device__ __forceinline__ void halve16(uint8_t* at, int doublings) {
  const float by = doublings >= 0 ? ldexpf(1.f, -doublings) : 0.f;
  const uint4 was = *reinterpret_cast<const uint4*>(at);
  const uint32_t w[4] = {was.x, was.y, was.z, was.w};
  uint32_t now[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 a = float2_of<FMT, 0>(ready<FMT>(w[i])), b = float2_of<FMT, 1>(ready<FMT>(w[i]));
    now[i] = doublings >= 0 ? codes4<FMT>(a.x * by, a.y * by, b.x * by, b.y * by) : 0u;
  }
  *reinterpret_cast<uint4*>(at) = make_uint4(now[0], now[1], now[2], now[3]);
}
// what is not finite, or larger than 2^64, becomes 0
__device__ __forceinline__ bool only_finite(float* x) {
  bool odd = false;
#pragma unroll
  for (int i = 0; i < 16; ++i)
    if (!(fabsf(x[i]) <= MAGNITUDE)) { x[i] = 0.f; odd = true; }
  return odd;
}
__device__ __forceinline__ float largest16(const float* x) {
  float top = 0.f;
#pragma unroll
  for (int i = 0; i < 16; ++i) top = fmaxf(top, fabsf(x[i]));
  return top;
}

// Queries: rotate, round, store.  `slots` rows of a head side by side in the block; q_rows rows of the batch, whose angles serve all heads.
template <int D, bool OWN>
__device__ void append_queries(const AppendP& p, int block) {
  constexpr int CHUNKS = D / 16;
  __shared__ int row_pos[8];
  const int tid = threadIdx.x, lane = tid & 31, warps = blockDim.x >> 5;
  const int slots = blockDim.x / CHUNKS / p.q_rows, r_first = block * p.q_rows;
  for (int i = tid >> 5; i < p.q_rows; i += warps) {
    const int r = r_first + i;
    int pos = -1;
    if (r < p.b.T) {
      const int s = sequence_of_row(p.b, r);
      if (s < p.b.S) {
        const Seq q = sequence(p.b, s, p.P);
        if (has_row(q, r)) pos = q.before + (r - q.r0);
      }
    }
    if (lane == 0) row_pos[i] = pos;
  }
  __syncthreads();
  const int slot = tid / CHUNKS, j = tid % CHUNKS, i = slot / slots, r = r_first + i, pos = row_pos[i];
  if (pos < 0) return;
  const Chunk c(j, p.rot, p.halves);
  Turn t;
  if (c.turned) turn<OWN>(t, p, j, pos, r);
  constexpr int ROUND = 4;                   // heads asked for together: results may lie over the queries, so the compiler keeps loads behind stores
  for (int h0 = slot % slots; h0 < p.Hq; h0 += ROUND * slots) {
    uint4 raw[ROUND][2];
#pragma unroll
    for (int k = 0; k < ROUND; ++k) {
      const bf16* row = p.q + r * p.q_ld + (long long)(h0 + k * slots) * D;
      if (h0 + k * slots < p.Hq) { raw[k][0] = *reinterpret_cast<const uint4*>(row + c.lo); raw[k][1] = *reinterpret_cast<const uint4*>(row + c.hi); }
    }
#pragma unroll
    for (int k = 0; k < ROUND; ++k) {
      if (h0 + k * slots >= p.Hq) break;
      float x[16];
      unpack16(x, raw[k]);
      if (c.turned) { if (p.halves) rotate16(x, t, 1); else rotate16(x, t, 0); }
      bf16* out = p.q_out + r * p.q_out_ld + (long long)(h0 + k * slots) * D;
      *reinterpret_cast<uint4*>(out + c.lo) = make_uint4(pack_bf16(x[0], x[1]), pack_bf16(x[2], x[3]), pack_bf16(x[4], x[5]), pack_bf16(x[6], x[7]));
      *reinterpret_cast<uint4*>(out + c.hi) = make_uint4(pack_bf16(x[8], x[9]), pack_bf16(x[10], x[11]), pack_bf16(x[12], x[13]), pack_bf16(x[14], x[15]));
    }
  }
}

// Few rows a sequence: a warp per (page that the step touches, kv head, side); rows past the first sweep of the warp are read twice, for the scale and for the codes.
// Bounds: the launch and a chain of four dependent reads (rows, table, scale, codes): 48 sequences of one row, 32 heads and their queries 8.6 us.
constexpr int APPEND_THREADS = 256;
template <int FMT, int D, bool OWN>
__global__ void __launch_bounds__(APPEND_THREADS) append_few_kernel(const AppendP p) {
  pdl_trigger();
  pdl_wait();
  constexpr int CHUNKS = D / 16, RPS = 32 / CHUNKS;
  if (blockIdx.x == gridDim.x - 1) { record_sequences(p.b, p.P, p.flags, blockDim.x); return; }
  if ((int)blockIdx.x >= p.page_ctas) { append_queries<D, OWN>(p, (int)blockIdx.x - p.page_ctas); return; }
  const int lane = threadIdx.x & 31, task = (int)blockIdx.x * (APPEND_THREADS / 32) + (threadIdx.x >> 5);
  if (task >= p.items * p.H * 2) return;
  const bool keys = !(task & 1);
  const int h = (task >> 1) % p.H;
  const Page g = page_of(p, (task >> 1) / p.H, lane == 0);
  if (!g.ok) return;
  const bf16* src = (keys ? p.k : p.v) + (long long)h * D;
  const long long ld = keys ? p.k_ld : p.v_ld;
  uint8_t* codes = (keys ? p.k_codes : p.v_codes) + ((long long)g.page * p.H + h) * p.P * D;
  float* scale_at = (keys ? p.k_scale : p.v_scale) + (long long)g.page * p.H + h;
  const float s_old = g.o > 0 ? *scale_at : 0.f;
  const int j = lane % CHUNKS, row0 = lane / CHUNKS;
  const Chunk c(j, keys ? p.rot : 0, p.halves);
  bool odd = false;
  auto fetch = [&](float* x, int slot) {
    load16(x, src + (g.r + slot - g.o) * ld, c);
    if (c.turned) {
      Turn t;
      turn<OWN>(t, p, j, g.first + slot, g.r + slot - g.o);
      if (p.halves) rotate16(x, t, 1); else rotate16(x, t, 0);
    }
    odd |= only_finite(x);
  };
  float kept[16], top = 0.f;
  if (g.o + row0 < g.e) { fetch(kept, g.o + row0); top = largest16(kept); }
  for (int slot = g.o + row0 + RPS; slot < g.e; slot += RPS) {
    float x[16];
    fetch(x, slot);
    top = fmaxf(top, largest16(x));
  }
  top = warp_max(top);
  if (__any_sync(0xffffffffu, odd) && lane == 0) flag(p.flags, B200_PAGED_NOT_FINITE);
  int doublings;
  const float sc = scale_for<FMT>(top, g.o, s_old, &doublings);
  __syncwarp();
  if (lane == 0) *scale_at = sc;
  if (g.o + row0 < g.e) store16<FMT>(codes + (long long)(g.o + row0) * D, c, kept, sc);
  for (int slot = g.o + row0 + RPS; slot < g.e; slot += RPS) {
    float x[16];
    fetch(x, slot);
    store16<FMT>(codes + (long long)slot * D, c, x, sc);
  }
  if (doublings != 0)
    for (int slot = row0; slot < g.o; slot += RPS) halve16<FMT>(codes + (long long)slot * D + 16 * j, doublings);
}

// Many rows: a block of P * D / 32 threads, two chunks each, has a page and goes through some of its heads, keys and values; the next head's rows are on their way while one is worked on, and
// the angles of the page's positions serve all heads.  Everything is read once, as the scale has to be known before the first code.
// Bounds: bytes, once the chain of reads in front is shared by several heads: 7887 rows of 8 heads 24 us (48 MB), with 32 heads of queries 41 (177 MB, 4.3 TB/s).  A head to a block took 40 and 69.
template <int FMT, int D, bool OWN>
__global__ void __launch_bounds__(512) append_many_kernel(const AppendP p) {
  pdl_trigger();
  pdl_wait();
  constexpr int CHUNKS = D / 16;
  if (blockIdx.x == gridDim.x - 1) { record_sequences(p.b, p.P, p.flags, blockDim.x); return; }
  if ((int)blockIdx.x >= p.page_ctas) { append_queries<D, OWN>(p, (int)blockIdx.x - p.page_ctas); return; }
  __shared__ float tops[2][16];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, warps = blockDim.x >> 5;
  const int groups = (p.H + p.heads_per_block - 1) / p.heads_per_block, item = (int)blockIdx.x / groups, h0 = ((int)blockIdx.x - item * groups) * p.heads_per_block;
  const Page g = page_of(p, item, tid == 0);
  if (!g.ok) return;                                    // the whole block
  const int j = tid % CHUNKS, row0 = tid / CHUNKS, half = p.P / 2, works = 2 * (min(h0 + p.heads_per_block, p.H) - h0);
  const int slot[2] = {row0, row0 + half};
  const bool mine[2] = {slot[0] >= g.o && slot[0] < g.e, slot[1] >= g.o && slot[1] < g.e};
  const Chunk ck(j, p.rot, p.halves), cv(j, 0, 0);
  Turn t[2];
  if (ck.turned) {
#pragma unroll
    for (int k = 0; k < 2; ++k) turn<OWN>(t[k], p, j, g.first + slot[k], mine[k] ? g.r + slot[k] - g.o : g.r);
  }
  uint4 raw[2][2];
  float s_next;
  auto ask = [&](int w) {
    if (w >= works) return;
    const int h = h0 + (w >> 1);
    const bool keys = !(w & 1);
    const bf16* src = (keys ? p.k : p.v) + (long long)h * D;
    const long long ld = keys ? p.k_ld : p.v_ld;
    const int lo = keys ? ck.lo : cv.lo, hi = keys ? ck.hi : cv.hi;
    s_next = g.o > 0 ? (keys ? p.k_scale : p.v_scale)[(long long)g.page * p.H + h] : 0.f;
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      const bf16* row = src + (g.r + slot[k] - g.o) * ld;
      raw[k][0] = mine[k] ? *reinterpret_cast<const uint4*>(row + lo) : make_uint4(0, 0, 0, 0);
      raw[k][1] = mine[k] ? *reinterpret_cast<const uint4*>(row + hi) : make_uint4(0, 0, 0, 0);
    }
  };
  ask(0);
  bool odd = false;
  for (int w = 0; w < works; ++w) {
    const int h = h0 + (w >> 1);
    const bool keys = !(w & 1);
    float x[2][16], top = 0.f;
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      unpack16(x[k], raw[k]);
      if (keys && ck.turned) { if (p.halves) rotate16(x[k], t[k], 1); else rotate16(x[k], t[k], 0); }
      odd |= only_finite(x[k]);
      top = fmaxf(top, largest16(x[k]));
    }
    const float s_old = s_next;
    ask(w + 1);
    top = warp_max(top);
    if (lane == 0) tops[w & 1][warp] = top;             // two places: the next round's maxima may come before the last thread has read these
    __syncthreads();
    for (int i = 0; i < warps; ++i) top = fmaxf(top, tops[w & 1][i]);
    int doublings;
    const float sc = scale_for<FMT>(top, g.o, s_old, &doublings);
    uint8_t* codes = (keys ? p.k_codes : p.v_codes) + ((long long)g.page * p.H + h) * p.P * D;
    if (tid == 0) (keys ? p.k_scale : p.v_scale)[(long long)g.page * p.H + h] = sc;
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      if (mine[k]) { if (keys) store16<FMT>(codes + slot[k] * D, ck, x[k], sc); else store16<FMT>(codes + slot[k] * D, cv, x[k], sc); }
      if (doublings != 0 && slot[k] < g.o) halve16<FMT>(codes + slot[k] * D + 16 * j, doublings);
    }
  }
  if (__any_sync(0xffffffffu, odd) && lane == 0) flag(p.flags, B200_PAGED_NOT_FINITE);
}

// =========================================================================================================================
// read back: the rows of the batch as bf16
// =========================================================================================================================
struct ReadP {
  const uint8_t *k_codes, *v_codes;
  const float *k_scale, *v_scale;
  int32_t* flags;
  Batch b;
  bf16 *k, *v;                               // [T][H][D]
  int pages, P, H;
};
constexpr int READ_THREADS = 256;

// A warp per row and side; four 16-byte pieces of codes in flight a lane.  Bounds: bytes, and for few rows the same chain of reads as append's: 8000 rows of 8 heads 11 us (50 MB).
template <int FMT, int D>
__global__ void __launch_bounds__(READ_THREADS) read_kernel(const ReadP p) {
  pdl_trigger();
  pdl_wait();
  if (blockIdx.x == gridDim.x - 1) { record_sequences(p.b, p.P, p.flags, blockDim.x); return; }
  const int lane = threadIdx.x & 31, task = (int)blockIdx.x * (READ_THREADS / 32) + (threadIdx.x >> 5), r = task >> 1, side = task & 1;
  if (r >= p.b.T) return;
  const int s = sequence_of_row(p.b, r);
  if (s >= p.b.S) return;
  const Seq q = sequence(p.b, s, p.P);
  if (!has_row(q, r)) return;
  const int pos = q.before + (r - q.r0), page = p.b.table[s * p.b.table_ld + pos / p.P], slot = pos % p.P;
  if (page < 0 || page >= p.pages) {
    if (lane == 0) flag(p.flags, B200_PAGED_BAD_PAGE);
    return;
  }
  constexpr int CHUNKS = D / 16, ROUND = 4;
  const int n = p.H * CHUNKS;
  const uint8_t* codes = (side ? p.v_codes : p.k_codes) + ((long long)page * p.H * p.P + slot) * D;
  const float* scales = (side ? p.v_scale : p.k_scale) + (long long)page * p.H;
  bf16* out = (side ? p.v : p.k) + (long long)r * p.H * D;
  for (int x0 = lane; x0 < n; x0 += 32 * ROUND) {
    uint4 c[ROUND];
    float sc[ROUND];
#pragma unroll
    for (int k = 0; k < ROUND; ++k) {
      const int x = x0 + 32 * k;
      if (x < n) {
        c[k] = *reinterpret_cast<const uint4*>(codes + (long long)(x / CHUNKS) * p.P * D + 16 * (x % CHUNKS));
        sc[k] = scales[x / CHUNKS];
      }
    }
#pragma unroll
    for (int k = 0; k < ROUND; ++k) {
      if (x0 + 32 * k >= n) break;
      const uint32_t w[4] = {c[k].x, c[k].y, c[k].z, c[k].w};
      uint32_t o[8];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float2 a = float2_of<FMT, 0>(ready<FMT>(w[i])), b = float2_of<FMT, 1>(ready<FMT>(w[i]));
        o[2 * i] = pack_bf16(a.x * sc[k], a.y * sc[k]);
        o[2 * i + 1] = pack_bf16(b.x * sc[k], b.y * sc[k]);
      }
      *reinterpret_cast<uint4*>(out + 16 * (x0 + 32 * k)) = make_uint4(o[0], o[1], o[2], o[3]);
      *reinterpret_cast<uint4*>(out + 16 * (x0 + 32 * k) + 8) = make_uint4(o[4], o[5], o[6], o[7]);
    }
  }
}

// =========================================================================================================================
// attention of few rows
// =========================================================================================================================
// Columns are (row of the sequence, query head of the group); a unit is 8 * NT of them with one kv head, over tiles of 32 tokens that a CTA's warps take in turn.  Both products have the cache as
// the first operand of mma.sync: S^T = K Q^T (tokens x columns) and O^T += V^T P^T (dims x columns), so that a single row of one head wastes tensor-core columns and not
// cache bytes.  Which dimension of K is which k of the product is free as long as Q has the same order, and so is which dimension of V is which row of O^T, and which token is which row of S^T and
// k of the other product: a lane reads its fragments as 16 neighbouring codes.  P^T comes out of S^T by movmatrix.
//
// Codes of both types are exact in f16, and so are bf16 queries after a power of two per column; the scale of a page's keys multiplies the
// scores; that of its values goes into the exponent, P = 2^(score + log2 s_v - M), with M behind the running maximum of the same, and the sum of the weights takes P / s_v: nothing is
// rounded on the way but P, which is f16.  M follows only when a score passes it by 2^15, as then no column has to be compared across lanes for most tiles.
//
// Bounds: HBM for large batches (48 sessions of 3000 tokens, 32 heads, e4m3: 184 us, 6.4 TB/s); for many short units what a unit costs beside its tiles (128 sessions under a window of 1024, 8 heads: 68 us, floor 36;
// a part's first copies, its queries and the joining of its warps are 7400 clocks beside 20000 for eight tiles a warp).
// Why this way:
// * tiles come as swizzled tensor copies, two in flight and two at work per warp: asked for lane by lane in the fragments' order, 16 bytes of eight rows an instruction, the same bytes came at 5.2 TB/s,
//   in whole lines at 7.1 (nothing but copies);
// * the scores of a tile and the values of the one in front do not wait for one another and are one stretch of code;
// * two CTAs of four warps an SM: four of two warps are faster for short units (that window 68 -> 62 us) and slower for few (one session of 375 tokens 8.5 -> 11.6 us, one request of 131072 tokens
//   53 -> 55); three of four do not fit with the values' second place.
constexpr int FEW_WARPS = 4, FEW_THREADS = FEW_WARPS * 32;
constexpr int FEW_PER_SM = 2;                // CTAs
constexpr int DIRECT_TILES = 64;             // units of more tiles are always cut
constexpr int MIN_RUN = 8;                    // tiles of a CTA

__device__ __forceinline__ void mma_f16(float* d, uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
               : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t transposed8x8(uint32_t a) {
  uint32_t r;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(a));
  return r;
}
__device__ __forceinline__ uint32_t pack_f16(float a, float b) {
  const __half2 v = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&v);
}

// a column's D / 16 sums from dimension d0 on, divided by the sum of the weights (0: nothing was seen)
template <int D>
__device__ __forceinline__ void store_row(const AttnP& p, const Seq& q, int h, int cc, int d0, const float* acc, float sum) {
  constexpr int PER = D / 16;
  const float by = sum != 0.f ? 1.f / sum : 0.f;
  const int i = cc / p.G;
  bf16* out = p.out + (long long)(q.r0 + i) * p.out_ld + (long long)(h * p.G + cc - i * p.G) * D + d0;
  uint32_t w[PER / 2];
#pragma unroll
  for (int e = 0; e < PER / 2; ++e) w[e] = pack_bf16(acc[2 * e] * by, acc[2 * e + 1] * by);
  if constexpr (PER == 8) *reinterpret_cast<uint4*>(out) = make_uint4(w[0], w[1], w[2], w[3]);
  else *reinterpret_cast<uint2*>(out) = make_uint2(w[0], w[1]);
}

// ---- the flattened work ----
// The tiles of all units (sequence, kv head) one behind the other are cut into equal runs, one per CTA: lengths of a batch may differ as they like.  A unit that lies in several runs
// is joined by join_kernel; a run has at most two parts of such units, one that the run begins inside of and one that it ends inside of.
__device__ __forceinline__ int units_of(const AttnP& p, const Seq& q) { return !q.ok || q.n == 0 || q.n >= p.from_rows ? 0 : p.H; }
// What joining the warps, the first loads and the queries cost a unit, in tiles: a run of many short units is shorter.
constexpr int UNIT_COST = 12;
__device__ __forceinline__ int tiles_of(const AttnP& p, const Seq& q) { return Tiles<5>(q.before, q.before + q.n - 1, p.window, p.sinks).n; }
__device__ __forceinline__ long long work_of(const AttnP& p, int s) {
  const Seq q = sequence(p.b, s, p.P);
  const int u = units_of(p, q);
  return u ? (long long)u * (tiles_of(p, q) + UNIT_COST) : 0;
}
struct Run { long long from, to, base; int s; };      // this CTA's tiles; the sequence that it begins in and the tiles in front of that
// by all threads of the block
__device__ __forceinline__ Run run_of(const AttnP& p) {
  if (p.direct) {                            // a CTA a unit
    const int s = (int)blockIdx.x / p.H, u = (int)blockIdx.x - s * p.H;
    const Seq q = sequence(p.b, s, p.P);
    Run r;
    r.s = u < units_of(p, q) ? s : -1; r.base = 0;
    const int n = r.s >= 0 ? tiles_of(p, q) + UNIT_COST : 0;
    r.from = (long long)u * n; r.to = r.from + n;
    return r;
  }
  __shared__ long long sums[FEW_WARPS];
  __shared__ Run found;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  long long mine = 0, first = 0;
  for (int s = threadIdx.x; s < p.b.S; s += FEW_THREADS) {
    const long long w = work_of(p, s);
    if (s == (int)threadIdx.x) first = w;
    mine += w;
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) mine += __shfl_xor_sync(0xffffffffu, mine, o);
  if (lane == 0) sums[warp] = mine;
  if (threadIdx.x == 0) found.s = -1;
  __syncthreads();
  long long total = 0;
#pragma unroll
  for (int w = 0; w < FEW_WARPS; ++w) total += sums[w];
  long long run = (total + gridDim.x - 1) / gridDim.x;
  run = max((run + FEW_WARPS - 1) / FEW_WARPS * FEW_WARPS, (long long)MIN_RUN);
  Run r;
  r.from = run * blockIdx.x; r.to = min(r.from + run, total); r.s = -1; r.base = 0;
  if (r.from >= total) return r;
  long long base = 0;
  for (int s0 = 0; s0 < p.b.S; s0 += FEW_THREADS) {
    const int s = s0 + (int)threadIdx.x;
    const long long w = s0 == 0 ? first : s < p.b.S ? work_of(p, s) : 0;
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
    for (int i = 0; i < FEW_WARPS; ++i) {
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

constexpr int SEEN = 1, IN_PART = 0, HIDDEN = -1;      // a half of a tile: by all columns, by some, by none

// Tiles lie in shared memory as the copies swizzle them: 16-byte piece n of row r.
template <int D>
__device__ __forceinline__ int piece(int r, int n) { return D == 128 ? r * 128 + ((n ^ (r & 7)) << 4) : r * 64 + ((n ^ ((r >> 1) & 3)) << 4); }
// Which token is row i (and i + 8) of the fragments: an order in which neither the keys' nor the values' reads meet in a bank.  Eight lanes read keys of rows token_of(2 m), token_of(2 m + 1),
// four pieces of each, and values of rows token_of(2 c) (or 2 c + 1), c = 0 .. 3, two pieces of each.
template <int D>
__device__ __forceinline__ int token_of(int i) { return (D == 128 ? 0x37156240u : 0x67542310u) >> (4 * i) & 7; }

// Of a tree's rows, whose own positions the columns have, token j of sequence q for row r: what is cached by the positions, the step's own by the row's mask.
__device__ __forceinline__ bool sees_in_tree(const AttnP& p, const Seq& q, int r, int pos, int j) {
  if (pos < 0) return false;
  const int off = j - q.before;
  if (off < 0) return p.window <= 0 || pos - j < p.window || j < p.sinks;
  if (off >= q.n || !(p.seen[(long long)r * p.words + (off >> 5)] >> (off & 31) & 1u)) return false;
  if (p.window <= 0 || pos - q.before < p.window) return true;
  const int their = p.position[q.r0 + off];
  return pos - their < p.window || their < p.sinks;
}

template <int D, int FMT, int NT, bool TREE>
__global__ void __launch_bounds__(FEW_THREADS, FEW_PER_SM) few_rows_kernel(const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v, const AttnP p) {
  constexpr int KS = D / 16, MT = D / 16, COLS = 8 * NT, SIDE = 32 * D;        // bytes of a tile's keys or values
  extern __shared__ uint8_t smem_raw[];
  uint8_t* const ring = smem_raw + ((1024u - (tcp::smem_u32(smem_raw) & 1023u)) & 1023u);       // [warp]: two tiles of keys, two of values, as the copies swizzle them
  __shared__ __align__(8) uint64_t bars[FEW_WARPS][4];                        // a ring's places
  __shared__ volatile int quit;
  __shared__ float4 meta[FEW_WARPS][64];                                      // per half of a tile: who sees it, keys' scale, log2 and reciprocal of the values'
  __shared__ int rows_at[FEW_WARPS][64];                                      // and the row of codes that it begins at
  __shared__ float m_s[FEW_WARPS][8], l_s[FEW_WARPS][8];
  typedef float Sums[8][D + 4];
  Sums* o_s = reinterpret_cast<Sums*>(ring + FEW_WARPS * 4 * SIDE);           // the warps' sums
  const int lane = threadIdx.x & 31, warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), g = lane >> 2, c = lane & 3;
  const uint32_t bar = tcp::smem_u32(&bars[warp][0]);
  if (lane < 4) tcp::mbar_init(bar + 8 * lane, 1);
  if (threadIdx.x == 0) quit = 0;
  asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  __syncthreads();                           // no warp waits before `quit` has its first value
  const int key_row = token_of<D>(g), val_row[2] = {token_of<D>(2 * c), token_of<D>(2 * c + 1)};
  pdl_trigger();
  pdl_wait();
  if (blockIdx.x == 0) record_sequences(p.b, p.P, p.flags, FEW_THREADS);
  const Run run = run_of(p);
  if (run.s < 0) return;

  // A part of a unit: its places of u0 .. u1 - 1 are the run's, of which the first UNIT_COST are no tiles.
  struct Part {
    Seq q;
    int s, h, u0, u1, n_pos, pf, pl, first, count, used;                  // this warp's tiles; used: how many went through its ring before
    Tiles<5> tiles;
  };
  long long f = run.from, base = run.base;
  int s_at = run.s;
  Seq q_at = sequence(p.b, s_at, p.P);
  int units_at = units_of(p, q_at), n_at = units_at ? tiles_of(p, q_at) + UNIT_COST : 1;
  auto next_part = [&](int used) {
    while (f >= base + (long long)units_at * n_at && s_at + 1 < p.b.S) {      // the next sequence that has work
      base += (long long)units_at * n_at;
      q_at = sequence(p.b, ++s_at, p.P);
      units_at = units_of(p, q_at);
      n_at = units_at ? tiles_of(p, q_at) + UNIT_COST : 1;
    }
    const long long at = f - base;
    const int h = at < 0x7fffffffll ? (int)((uint32_t)at / (uint32_t)n_at) : (int)(at / n_at);
    const int u0 = (int)(at - (long long)h * n_at), u1 = (int)min((long long)n_at, u0 + (run.to - f));
    f += u1 - u0;
    const int pf = q_at.before, pl = q_at.before + q_at.n - 1;
    Part w{q_at, s_at, h, u0, u1, n_at, pf, pl, 0, 0, used, Tiles<5>(pf, pl, p.window, p.sinks)};
    const int t0 = max(u0 - UNIT_COST, 0), t1 = max(u1 - UNIT_COST, 0);
    w.first = t0 + warp;
    w.count = w.first < t1 ? (t1 - w.first + FEW_WARPS - 1) / FEW_WARPS : 0;
    return w;
  };
  uint8_t* const my_ring = ring + warp * 4 * SIDE;
  const uint32_t ring_at = tcp::smem_u32(my_ring);
  auto fetch = [&](const Part& w, int i, const CUtensorMap& map, int side) {
    const int place = side + ((w.used + i) & 1);
    const int r0 = rows_at[warp][(2 * i) & 63], r1 = rows_at[warp][(2 * i + 1) & 63];
    if (tcp::elected()) {
      const uint32_t to = ring_at + place * SIDE, b = bar + 8 * place;
      tcp::mbar_expect_tx(b, (r0 >= 0 ? SIDE / 2 : 0) + (r1 >= 0 ? SIDE / 2 : 0));
      if (r0 >= 0) tcp::tma_load_2d(to, &map, b, 0, r0);
      if (r1 >= 0) tcp::tma_load_2d(to + SIDE / 2, &map, b, 0, r1);
    }
    __syncwarp();
  };
  // Every 16 tiles the lanes look up the pages of their halves; what the scores need of them comes behind the copies' start.
  auto look_up = [&](const Part& w, int i) {
    const int mine = i + (lane >> 1), j = mine < w.count ? (w.tiles[w.first + mine * FEW_WARPS] << 5) + 16 * (lane & 1) : 0;
    int page = -1;
    if (mine < w.count && j <= w.pl && (p.window <= 0 || w.pf - j - 15 < p.window || j < p.sinks)) {
      page = p.b.table[w.s * p.b.table_ld + (j >> p.page_shift)];
      if (page < 0 || page >= p.pages) { flag(p.flags, B200_PAGED_BAD_PAGE); page = -1; }
    }
    rows_at[warp][(2 * i + lane) & 63] = page < 0 ? -1 : (page * p.H + w.h) * p.P + (j & (p.P - 1));
    __syncwarp();
    return page;
  };
  auto tell = [&](const Part& w, int i, int page) {
    const int mine = i + (lane >> 1), j = mine < w.count ? (w.tiles[w.first + mine * FEW_WARPS] << 5) + 16 * (lane & 1) : 0;
    float4 x = make_float4(__int_as_float(HIDDEN), 0.f, -INFINITY, 0.f);
    if (page >= 0) {
      const bool all = j + 15 <= w.pf - (TREE ? 1 : 0) && (p.window <= 0 || w.pl - j < p.window || j + 16 <= p.sinks);
      x.x = __int_as_float(all ? SEEN : IN_PART);
      x.y = p.k_scale[(long long)page * p.H + w.h];
      const float vs = value_scale(p.v_scale[(long long)page * p.H + w.h]);
      x.z = __log2f(vs); x.w = __frcp_rn(vs);
    }
    meta[warp][(2 * i + lane) & 63] = x;
    __syncwarp();
  };
  // the part's i-th tile on its way into the ring
  auto issue_keys = [&](const Part& w, int i) {
    if (i >= w.count) return;
    if (i & 15) { fetch(w, i, map_k, 0); return; }
    const int page = look_up(w, i);
    fetch(w, i, map_k, 0);
    tell(w, i, page);
  };
  auto issue_values = [&](const Part& w, int i) {
    if (i < w.count) fetch(w, i, map_v, 2);
  };
  uint32_t raw[KS][2];                       // eight columns' queries of the part to come, as they are in memory
  auto load_queries = [&](const Part& w, int nt) {
    const int col = nt * 8 + g;
    const bool has = col < w.q.n * p.G;
    const int i = has ? col / p.G : 0;
    const bf16* row = p.q + (long long)(w.q.r0 + i) * p.q_ld + (long long)(w.h * p.G + (has ? col - i * p.G : 0)) * D;
#pragma unroll
    for (int b = 0; b < D / 64; ++b) {
      const uint4 x = has ? *reinterpret_cast<const uint4*>(row + 64 * b + 16 * c) : make_uint4(0, 0, 0, 0);
      const uint4 y = has ? *reinterpret_cast<const uint4*>(row + 64 * b + 16 * c + 8) : make_uint4(0, 0, 0, 0);
      raw[4 * b][0] = x.x; raw[4 * b][1] = x.y; raw[4 * b + 1][0] = x.z; raw[4 * b + 1][1] = x.w;
      raw[4 * b + 2][0] = y.x; raw[4 * b + 2][1] = y.y; raw[4 * b + 3][0] = y.z; raw[4 * b + 3][1] = y.w;
    }
  };
  // a part's first copies, which go out before the part in front of it is joined
  auto start = [&](const Part& w) {
    __syncwarp();
    if (w.count == 0) {
      if constexpr (NT == 1) load_queries(w, 0);
      return;
    }
    const int page = look_up(w, 0);
    fetch(w, 0, map_k, 0);
    fetch(w, 0, map_v, 2);
    if (w.count > 1) fetch(w, 1, map_k, 0);
    if constexpr (NT == 1) load_queries(w, 0);                                // their way is as long as the scales'
    tell(w, 0, page);
  };
  auto arrived = [&](const Part& w, int i, int side) {
    const uint32_t n = (uint32_t)(w.used + i);
    if (!wait_or_quit(bar + 8 * (side + (n & 1)), (n >> 1) & 1u, &quit)) flag(p.flags, B200_PAGED_WAIT);
    __syncwarp();
  };

  Part w = next_part(0);
  start(w);
  for (;;) {
    const Seq q = w.q;
    const int h = w.h, n_cols = q.n * p.G, pf = w.pf, pl = w.pl, first = w.first, count = w.count, used = w.used;
    const Tiles<5> tiles = w.tiles;

    // queries: lane (g, c) has of column 8 nt + g the dimensions 64 i + 16 c .. + 15
    uint32_t qf[NT][KS][2];
    float fac[NT][2];                        // of columns 8 nt + 2 c, + 1: what turns a product of codes into a score in base 2
    int pos[NT][2];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      if constexpr (NT > 1) load_queries(w, nt);
      float top = 0.f;                       // of the column's finite values; infinity if there are others
      bool odd = false;
#pragma unroll
      for (int k = 0; k < KS; ++k)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const float2 v = unpack_bf16(raw[k][e]);
          odd |= !(fabsf(v.x) < INFINITY) || !(fabsf(v.y) < INFINITY);
          top = fmaxf(top, fmaxf(fabsf(v.x), fabsf(v.y)));
        }
      if (odd) top = INFINITY;
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
      const float power = top > 0.f ? power_of_two_in(top) : 1.f;
      const float up = 16384.f / power;      // the column's largest lands in [2^14, 2^15)
#pragma unroll
      for (int k = 0; k < KS; ++k)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const float2 v = unpack_bf16(raw[k][e]);
          qf[nt][k][e] = pack_f16(v.x * up, v.y * up);
        }
      const float back = top < INFINITY ? power * (1.f / 16384.f) : NAN;         // such a column's results are NaN, and no other's
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        fac[nt][e] = __shfl_sync(0xffffffffu, back, (2 * c + e) * 4) * p.scale2;
        const int cc = nt * 8 + 2 * c + e;
        pos[nt][e] = cc >= n_cols ? -1 : TREE ? (p.window > 0 ? max(p.position[q.r0 + cc / p.G], 0) : q.before) : q.before + cc / p.G;
      }
    }

    float o[NT][MT][4], m[NT][2], l[NT][2];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
      for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) o[nt][i][e] = 0.f;
      m[nt][0] = m[nt][1] = -INFINITY;
      l[nt][0] = l[nt][1] = 0.f;
    }

    struct Tile { float4 x[2]; bool whole; };
    auto tile_at = [&](int i) {
      Tile t;
      t.x[0] = meta[warp][(2 * i) & 63];
      t.x[1] = meta[warp][(2 * i + 1) & 63];
      t.whole = __float_as_int(t.x[0].x) + __float_as_int(t.x[1].x) == 2 * SEEN;
      return t;
    };
    // scores in base 2, log2 of the values' scale added
    auto scores = [&](int i, const Tile& t, float (&sc)[2][NT][4]) {
      const uint8_t* from = my_ring + ((used + i) & 1) * SIDE;
#pragma unroll
      for (int half = 0; half < 2; ++half)
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) sc[half][nt][0] = sc[half][nt][1] = sc[half][nt][2] = sc[half][nt][3] = 0.f;
#pragma unroll
      for (int b = 0; b < D / 64; ++b)
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          const uint8_t* f_h = from + half * (SIDE / 2);
          const uint4 r0 = *reinterpret_cast<const uint4*>(f_h + piece<D>(key_row, 4 * b + c)), r1 = *reinterpret_cast<const uint4*>(f_h + piece<D>(key_row + 8, 4 * b + c));
          const uint32_t k0[4] = {r0.x, r0.y, r0.z, r0.w}, k1[4] = {r1.x, r1.y, r1.z, r1.w};
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const uint32_t w0 = ready<FMT>(k0[k]), w1 = ready<FMT>(k1[k]);
            const uint32_t a0 = half2_of<FMT, 0>(w0), a1 = half2_of<FMT, 0>(w1), a2 = half2_of<FMT, 1>(w0), a3 = half2_of<FMT, 1>(w1);
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) mma_f16(sc[half][nt], a0, a1, a2, a3, qf[nt][4 * b + k][0], qf[nt][4 * b + k][1]);
          }
        }
#pragma unroll
      for (int half = 0; half < 2; ++half)
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          const float by[2] = {t.x[half].y * fac[nt][0], t.x[half].y * fac[nt][1]};
#pragma unroll
          for (int e = 0; e < 4; ++e) sc[half][nt][e] = fmaf(sc[half][nt][e], by[e & 1], t.x[half].z);
        }
    };
    uint32_t pb[2][NT][2];                   // weights of the tile whose values come next
    // weights out of scores, and O and the sums brought to the maximum that they refer to
    auto weigh = [&](int i, const Tile& t, float (&sc)[2][NT][4]) {
      if (!t.whole) {
        const int j0 = tiles[first + i * FEW_WARPS] << 5;
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          const bool has = __float_as_int(t.x[half].x) != HIDDEN;
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const int j = j0 + 16 * half + key_row + 8 * (e >> 1);
              bool seen = has;
              if constexpr (TREE) seen = has && sees_in_tree(p, q, q.r0 + (nt * 8 + 2 * c + (e & 1)) / p.G, pos[nt][e & 1], j);
              else seen = has && sees(pos[nt][e & 1], j, p.window, p.sinks);
              if (!seen) sc[half][nt][e] = -INFINITY;
            }
        }
      }
      float top[NT][2];
      bool grow = false;
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          top[nt][e] = fmaxf(fmaxf(sc[0][nt][e], sc[0][nt][e + 2]), fmaxf(sc[1][nt][e], sc[1][nt][e + 2]));
          grow |= top[nt][e] > __fadd_rd(m[nt][e], SLACK);      // rounded down: above 2^27 the sum would else round to the score itself, and its weight to infinity
        }
      if (__any_sync(0xffffffffu, grow)) {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            float y = top[nt][e];
            y = fmaxf(y, __shfl_xor_sync(0xffffffffu, y, 4));
            y = fmaxf(y, __shfl_xor_sync(0xffffffffu, y, 8));
            y = fmaxf(y, __shfl_xor_sync(0xffffffffu, y, 16));
            const float now = fmaxf(m[nt][e], y - UNDER), by = now == -INFINITY ? 1.f : exp2_fast(m[nt][e] - now);
            m[nt][e] = now;
            l[nt][e] *= by;
#pragma unroll
            for (int k = 0; k < MT; ++k) { o[nt][k][e] *= by; o[nt][k][e + 2] *= by; }
          }
      }
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        const float off[2] = {m[nt][0] == -INFINITY ? 0.f : m[nt][0], m[nt][1] == -INFINITY ? 0.f : m[nt][1]};
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          float w[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) w[e] = exp2_fast(sc[half][nt][e] - off[e & 1]);
          l[nt][0] = fmaf(w[0] + w[2], t.x[half].w, l[nt][0]);
          l[nt][1] = fmaf(w[1] + w[3], t.x[half].w, l[nt][1]);
          pb[half][nt][0] = transposed8x8(pack_f16(w[0], w[1]));
          pb[half][nt][1] = transposed8x8(pack_f16(w[2], w[3]));
        }
      }
    };
    // codes of tokens that no column sees may be anything: this lane's become 0
    auto hide = [&](int i, const Tile& t) {
      const int j0 = tiles[first + i * FEW_WARPS] << 5;
#pragma unroll
      for (int half = 0; half < 2; ++half)
#pragma unroll
        for (int a = 0; a < 4; ++a) {
          const int r = val_row[a & 1] + 8 * (a >> 1), j = j0 + 16 * half + r;
          if (__float_as_int(t.x[half].x) != HIDDEN && j <= pl && (p.window <= 0 || pf - j < p.window || j < p.sinks)) continue;
          uint8_t* v = my_ring + (2 + ((used + i) & 1)) * SIDE + half * (SIDE / 2);
          if constexpr (D == 128) *reinterpret_cast<uint4*>(v + piece<D>(r, g)) = make_uint4(0, 0, 0, 0);
          else *reinterpret_cast<uint2*>(v + piece<D>(r, g >> 1) + 8 * (g & 1)) = make_uint2(0, 0);
        }
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");            // the next copy into this place comes behind these writes
      __syncwarp();                          // lanes with and without such tokens together again: the products ask for whole warps
    };
    auto add_values = [&](int i) {
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        const uint8_t* f_h = my_ring + (2 + ((used + i) & 1)) * SIDE + half * (SIDE / 2);
        uint32_t v[4][D / 32];
#pragma unroll
        for (int a = 0; a < 4; ++a) {
          const int r = val_row[a & 1] + 8 * (a >> 1);
          if constexpr (D == 128) {
            const uint4 w = *reinterpret_cast<const uint4*>(f_h + piece<D>(r, g));
            v[a][0] = w.x; v[a][1] = w.y; v[a][2] = w.z; v[a][3] = w.w;
          } else {
            const uint2 w = *reinterpret_cast<const uint2*>(f_h + piece<D>(r, g >> 1) + 8 * (g & 1));
            v[a][0] = w.x; v[a][1] = w.y;
          }
        }
#pragma unroll
        for (int j = 0; j < D / 32; ++j) {   // four dimensions of this lane's
          const uint32_t v0 = ready<FMT>(v[0][j]), v1 = ready<FMT>(v[1][j]), v2 = ready<FMT>(v[2][j]), v3 = ready<FMT>(v[3][j]);
          const uint32_t lo = prmt(v0, v1, 0x5140u), hi = prmt(v0, v1, 0x7362u), lo8 = prmt(v2, v3, 0x5140u), hi8 = prmt(v2, v3, 0x7362u);
          const uint32_t a[8] = {half2_of<FMT, 0>(lo), half2_of<FMT, 1>(lo), half2_of<FMT, 0>(lo8), half2_of<FMT, 1>(lo8),
                                 half2_of<FMT, 0>(hi), half2_of<FMT, 1>(hi), half2_of<FMT, 0>(hi8), half2_of<FMT, 1>(hi8)};
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) {
            mma_f16(o[nt][2 * j], a[0], a[1], a[2], a[3], pb[half][nt][0], pb[half][nt][1]);
            mma_f16(o[nt][2 * j + 1], a[4], a[5], a[6], a[7], pb[half][nt][0], pb[half][nt][1]);
          }
        }
      }
    };

    // The scores of tile i + 1 and the values of tile i do not wait for one another, and lie in one stretch of code; behind them the weights of tile i + 1.
    if (count) {
      Tile t = tile_at(0);
      float sc[2][NT][4];
      arrived(w, 0, 0);
      scores(0, t, sc);
      weigh(0, t, sc);
      for (int i = 0; i + 1 < count; ++i) {
        __syncwarp();                        // the places that these copies go to have been read
        issue_values(w, i + 1);
        issue_keys(w, i + 2);
        arrived(w, i, 2);
        if (!t.whole) hide(i, t);
        t = tile_at(i + 1);
        arrived(w, i + 1, 0);
        scores(i + 1, t, sc);
        add_values(i);
        weigh(i + 1, t, sc);
      }
      arrived(w, count - 1, 2);
      if (!t.whole) hide(count - 1, t);
      add_values(count - 1);
    }
    const Part now = w;
    const bool more = f < run.to;
    if (more) {
      w = next_part(used + count);
      start(w);
    }

    // join the warps, eight columns at a time
    const bool alone = now.u0 == 0 && now.u1 == now.n_pos;
    const int slot = 2 * (int)blockIdx.x + (now.u0 == 0 ? 1 : 0);
    if (!p.direct && now.u0 == 0 && threadIdx.x == 0) {                       // where the unit's parts are: this run's and so many after it
      const long long runs = run.to - run.from, left = now.n_pos - now.u1;
      p.parts[(long long)now.s * p.H + now.h] = make_int2((int)blockIdx.x, alone ? 0 : (int)((left + runs - 1) / runs));
    }
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      if (nt * 8 >= n_cols) break;
      __syncthreads();
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        float sum = l[nt][e];
        sum += __shfl_xor_sync(0xffffffffu, sum, 4);
        sum += __shfl_xor_sync(0xffffffffu, sum, 8);
        sum += __shfl_xor_sync(0xffffffffu, sum, 16);
        if (g == 0) { m_s[warp][2 * c + e] = m[nt][e]; l_s[warp][2 * c + e] = sum; }
      }
#pragma unroll
      for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int e = 0; e < 2; ++e) *reinterpret_cast<float2*>(&o_s[warp][2 * c + e][(D / 8) * g + 2 * i]) = make_float2(o[nt][i][e], o[nt][i][e + 2]);
      __syncthreads();
      constexpr int PER = D / 16;            // 16 threads a column
      const int d0 = (threadIdx.x & 15) * PER;
#pragma unroll
      for (int col = threadIdx.x >> 4; col < 8; col += FEW_THREADS / 16) {
        const int cc = nt * 8 + col;
        if (cc >= n_cols) break;
        float top = -INFINITY, sum = 0.f, acc[PER];
#pragma unroll
        for (int w = 0; w < FEW_WARPS; ++w) top = fmaxf(top, m_s[w][col]);
#pragma unroll
        for (int i = 0; i < PER; ++i) acc[i] = 0.f;
#pragma unroll
        for (int w = 0; w < FEW_WARPS; ++w) {
          const float by = m_s[w][col] == -INFINITY ? 0.f : exp2_fast(m_s[w][col] - top);
          sum = fmaf(l_s[w][col], by, sum);
#pragma unroll
          for (int i = 0; i < PER; ++i) acc[i] = fmaf(o_s[w][col][d0 + i], by, acc[i]);
        }
        if (alone) store_row<D>(p, q, h, cc, d0, acc, sum);
        else {
          const long long at = (long long)slot * COLS + nt * 8 + col;
          if ((threadIdx.x & 15) == 0) *reinterpret_cast<float2*>(p.part_ml + 2 * at) = make_float2(top, sum);
#pragma unroll
          for (int i = 0; i < PER; i += 4) *reinterpret_cast<float4*>(p.part_o + at * D + d0 + i) = make_float4(acc[i], acc[i + 1], acc[i + 2], acc[i + 3]);
        }
      }
    }
    if (!more) break;
  }
  if (quit) {                                // let copies in flight land before the block ends
    const uint64_t since = tcp::global_timer_ns();
    while (tcp::global_timer_ns() - since < 2000000ull) {}
  }
}

// Joins the parts of units that lie in several runs: a block a column, its eight teams of sixteen threads take the parts in turn (one thread after the other through 74 parts of a long request had
// taken 20 us).  Bounds: four dependent reads.
template <int D, int NT>
__global__ void __launch_bounds__(128) join_kernel(const AttnP p) {
  pdl_trigger();
  pdl_wait();
  constexpr int COLS = 8 * NT, PER = D / 16;
  __shared__ float o_s[8][D + 4], m_s[8], l_s[8];
  const int most = min(COLS, p.b.max_rows * p.G);       // columns of a unit
  const int cc = (int)(blockIdx.x % most), team = threadIdx.x >> 4, d0 = (threadIdx.x & 15) * PER;
  const long long unit = blockIdx.x / most;
  const int h = (int)(unit % p.H), s = (int)(unit / p.H);
  const Seq q = sequence(p.b, s, p.P);
  if (units_of(p, q) == 0 || cc >= q.n * p.G) return;
  const int2 parts = p.parts[unit];
  if (parts.y == 0) return;
  // the first part is its run's last, the others are their runs' first
  const float2* ml = reinterpret_cast<const float2*>(p.part_ml);
  float top = -INFINITY, sum = 0.f, acc[PER];
#pragma unroll
  for (int e = 0; e < PER; ++e) acc[e] = 0.f;
#pragma unroll 2
  for (int i = team; i <= parts.y; i += 8) {
    const long long at = (long long)(2 * (parts.x + i) + (i == 0 ? 1 : 0)) * COLS + cc;
    const float2 y = ml[at];
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
#pragma unroll
  for (int e = 0; e < PER; ++e) o_s[team][d0 + e] = acc[e];
  if ((threadIdx.x & 15) == 0) { m_s[team] = top; l_s[team] = sum; }
  __syncthreads();
  if (team) return;
  top = -INFINITY; sum = 0.f;
#pragma unroll
  for (int i = 0; i < 8; ++i) top = fmaxf(top, m_s[i]);
#pragma unroll
  for (int e = 0; e < PER; ++e) acc[e] = 0.f;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float by = m_s[i] == -INFINITY ? 0.f : exp2_fast(m_s[i] - top);
    sum = fmaf(l_s[i], by, sum);
#pragma unroll
    for (int e = 0; e < PER; ++e) acc[e] = fmaf(o_s[i][d0 + e], by, acc[e]);
  }
  store_row<D>(p, q, h, cc, d0, acc, sum);
}

// =========================================================================================================================
// host
// =========================================================================================================================
int check_cache(const b200_paged_cache* c, const char* what) {
  if (!c || !c->k_dev || !c->v_dev || !c->k_scale_dev || !c->v_scale_dev || !c->flags_dev) B200_FAIL(B200_ERR_INVALID, "%s: null pointer in the cache", what);
  if (c->kv_dtype != B200_KV_INT8 && c->kv_dtype != B200_KV_FP8_E4M3) B200_FAIL(B200_ERR_INVALID, "%s: kv_dtype %d", what, c->kv_dtype);
  if (c->dim != 64 && c->dim != 128) B200_FAIL(B200_ERR_SHAPE, "%s: head size %d (64 or 128)", what, c->dim);
  if (c->page_tokens != 16 && c->page_tokens != 32 && c->page_tokens != 64 && c->page_tokens != 128) B200_FAIL(B200_ERR_SHAPE, "%s: pages of %d tokens (16, 32, 64 or 128)", what, c->page_tokens);
  if (c->pages < 1 || c->kv_heads < 1 || c->kv_heads > 1024 || (long long)c->pages * c->kv_heads * c->page_tokens > 0x7fffff00ll) B200_FAIL(B200_ERR_SHAPE, "%s: %d pages, %d heads", what, c->pages, c->kv_heads);
  if ((reinterpret_cast<uintptr_t>(c->k_dev) | reinterpret_cast<uintptr_t>(c->v_dev)) & 15) B200_FAIL(B200_ERR_INVALID, "%s: the cache's codes must begin on a 16-byte border", what);
  return B200_OK;
}
int check_batch(const b200_paged_cache* c, const b200_paged_batch* b, const char* what) {
  if (!b || !b->table_dev || !b->before_dev || !b->rows_dev) B200_FAIL(B200_ERR_INVALID, "%s: null pointer in the batch", what);
  if (b->sequences < 1 || b->sequences > 65536 || b->total_rows < 0 || b->total_rows > (1 << 24) || b->max_rows < 0 || b->table_width < 1 || b->table_ld < b->table_width)
    B200_FAIL(B200_ERR_SHAPE, "%s: %d sequences, %d rows (%d of one), tables of %d pages", what, b->sequences, b->total_rows, b->max_rows, b->table_width);
  if ((long long)b->table_width * c->page_tokens > 0x7fffff00ll) B200_FAIL(B200_ERR_SHAPE, "%s: tables of %d pages reach past 2^31 tokens", what, b->table_width);
  return B200_OK;
}
Batch batch_of(const b200_paged_batch* b) {
  Batch x;
  x.table = b->table_dev; x.before = b->before_dev; x.rows = b->rows_dev; x.table_ld = b->table_ld;
  x.S = b->sequences; x.T = b->total_rows; x.width = b->table_width; x.max_rows = b->max_rows;
  return x;
}
bool rows_fit(const void* p, long long ld, int heads, int dim) { return p && !(reinterpret_cast<uintptr_t>(p) & 15) && ld >= (long long)heads * dim && ld % 8 == 0; }
int shift_of(int P) { return P == 16 ? 4 : P == 32 ? 5 : P == 64 ? 6 : 7; }

// Sequences of more than 16 columns (rows times heads of a group), at head size 64 of more than 32, go to the tensor cores' kernel of whole tiles, whose time hardly depends on how many of its 256 columns
// there are; the only sequence of a step goes there with all its rows if it may have that many.  (Here / there, 3000 tokens.  32 heads of 128 on 8: 16 requests of 16 columns 39 / 65 us, 64 of them 105 / 233, one 17.5 / 14.8;
// of 24 columns, as several units a sequence, 87 / 66, of 48 136 / 66.  24 heads of 64 on 4: 16 requests of 18, 24 and 30 columns 26, 26 and 28 / 31, of 24 on 1000 tokens 20 / 19, of 30 on 10000 50 / 81,
// 64 of 24 61 / 100, one 19 / 13; 32 heads on 8, 32 columns: 16 requests 42 / 53, 4 of them 23 / 21.5.)
struct Route { int from_rows; FewPlan few; PromptPlan prompt; int64_t few_bytes, prompt_bytes; };
Route route(const b200_paged_cache* c, const b200_paged_batch* b, int G, int window, int sinks) {
  Route r;
  memset(&r, 0, sizeof(r));
  const bool many = (long long)b->max_rows * G > few_cols(c->dim);
  r.from_rows = !many ? 0x7fffffff : b->sequences == 1 ? 1 : few_cols(c->dim) / G + 1;
  if (r.from_rows > 1) { r.few = few_plan(c, b, G, window, sinks, r.from_rows); r.few_bytes = (few_bytes(r.few, c->dim) + 15) / 16 * 16; }
  if (many) { r.prompt = prompt_plan(c, b, G, window, sinks); r.prompt_bytes = prompt_bytes(r.prompt, c->dim); }
  return r;
}

constexpr int WAVE = 148 * 3 / 2;
template <int FMT, int D, bool OWN>
int launch_append(AppendP& p, cudaStream_t st) {
  // Up to 16 rows of a sequence: a warp a page, head and side (32 heads, 48 sequences of 1 / 8 / 16 rows: 7.8 / 9.7 / 13.7 us, as blocks of whole pages 28 / 29 / 30; 8 heads, 8 sequences of
  // 32 / 64 rows: 6.8 / 9.6 us, as blocks 6.1 / 6.5).
  const bool few = p.b.max_rows <= 16;
  const int threads = few ? APPEND_THREADS : p.P * D / 32;
  // as many heads to a block as leave the chip a wave of blocks, two to an SM
  p.heads_per_block = 1;
  while (!few && p.heads_per_block < p.H && (long long)p.items * ceil_div(p.H, 2 * p.heads_per_block) >= WAVE) p.heads_per_block *= 2;
  p.page_ctas = few ? (int)ceil_div64((long long)p.items * p.H * 2, APPEND_THREADS / 32) : p.items * ceil_div(p.H, p.heads_per_block);
  // a block's queries: one row where there are few, else up to eight rows, whose angles then serve more heads
  const int slots = threads / (D / 16);
  p.q_rows = 1;
  while (p.q_rows < 8 && 2 * p.q_rows <= slots && (long long)p.b.T * p.Hq >= 148ll * 8 * slots * p.q_rows) p.q_rows *= 2;
  const dim3 grid((unsigned)(p.page_ctas + (p.Hq ? ceil_div(p.b.T, p.q_rows) : 0) + 1));       // the last one looks at the sequences
  if (few) return launch_early(append_few_kernel<FMT, D, OWN>, grid, dim3(threads), 0, st, p);
  return launch_early(append_many_kernel<FMT, D, OWN>, grid, dim3(threads), 0, st, p);
}

template <int D, int FMT, int NT, bool TREE>
int launch_few(const AttnP& p, const FewPlan& f, cudaStream_t st) {
  constexpr int ring = FEW_WARPS * 4 * 32 * D, sums = FEW_WARPS * 8 * (D + 4) * 4, smem = ring + sums + 1024;
  static std::atomic<uint64_t> limits{0};
  CUtensorMap map_k, map_v;
  B200_TRY(code_map(&map_k, p.k, (long long)p.pages * p.H * p.P, D, 16));
  B200_TRY(code_map(&map_v, p.v, (long long)p.pages * p.H * p.P, D, 16));
  B200_TRY(allow_smem(limits, smem, few_rows_kernel<D, FMT, NT, TREE>));
  // all of an SM's L1 as shared memory, also for what runs in between: left to the driver an SM keeps what the kernel in front left, and then holds one CTA and not two
  static std::atomic<uint64_t> shares{0};
  B200_TRY(prefer_smem(shares, 100, few_rows_kernel<D, FMT, NT, TREE>, join_kernel<D, NT>));
  B200_TRY(launch_early(few_rows_kernel<D, FMT, NT, TREE>, dim3((unsigned)f.ctas), dim3(FEW_THREADS), smem, st, map_k, map_v, p));
  if (f.direct) return B200_OK;
  const long long most = (long long)p.b.max_rows * p.G < 8 * NT ? (long long)p.b.max_rows * p.G : 8 * NT;
  return launch_early(join_kernel<D, NT>, dim3((unsigned)(f.units * most)), dim3(128), 0, st, p);
}
template <int D, int FMT, bool TREE>
int launch_few_nt(const AttnP& p, const FewPlan& f, cudaStream_t st) {
  if constexpr (few_cols(D) > 16)
    if (f.nt == 4) return launch_few<D, FMT, 4, TREE>(p, f, st);
  return f.nt == 1 ? launch_few<D, FMT, 1, TREE>(p, f, st) : launch_few<D, FMT, 2, TREE>(p, f, st);
}

}  // namespace

// CTAs of 8 * nt columns, a wave of them, fewer where the tables allow for less work than that.
FewPlan few_plan(const b200_paged_cache* c, const b200_paged_batch* b, int G, int window, int sinks, int few_rows) {
  FewPlan f;
  const long long rows = few_rows <= b->max_rows ? few_rows - 1 : b->max_rows, cols = rows * G;
  f.nt = cols <= 8 ? 1 : cols <= 16 ? 2 : 4;
  f.units = (long long)b->sequences * c->kv_heads;       // few_cols, and so all rows of a sequence that come here, fit into one
  long long keys = (long long)b->table_width * c->page_tokens;
  if (window > 0 && (long long)window + sinks + rows < keys) keys = (long long)window + sinks + rows;
  const long long tiles = ceil_div64(keys, 32) + 1, runs = ceil_div64(f.units * (tiles + 4), MIN_RUN), wave = 148 * FEW_PER_SM;
  // A CTA a unit, and nothing to join, where the chip holds all units at once and the longest is not much longer than an equal share: 7 us and 0.25 a tile, against 10.5 and 0.34 for every 296th part of all
  // tiles and 12 for each unit.  (One token, 32 heads on 8, uncut / cut: 1 request of 1000 tokens 13.4 / 11.3 us, 32 of them 18.2 / 23.7, 8 of 2000 23.3 / 16.7, 32 of them, past the limit, 28.8 / 34.6; 1
  // session of 374 tokens with 32 heads 8.7 / 11.3.)
  f.direct = f.units <= wave && tiles <= DIRECT_TILES && 250 * tiles < 3500 + f.units * (tiles + UNIT_COST) * 115 / 100;
  f.ctas = (int)(f.direct ? f.units : runs < wave ? runs : wave);
  return f;
}
// sums and (maximum, sum of the weights) of two parts per CTA, and where each unit's parts are
int64_t few_bytes(const FewPlan& f, int D) { return f.direct ? 0 : (int64_t)f.ctas * 2 * 8 * f.nt * (D + 2) * 4 + f.units * 8; }
int few_attention(AttnP p, const FewPlan& f, int fmt, int dim, bool tree, void* work, cudaStream_t st) {
  p.direct = f.direct;
  if (!f.direct) {
    p.part_o = static_cast<float*>(work);
    p.part_ml = p.part_o + (long long)f.ctas * 2 * 8 * f.nt * dim;
    p.parts = reinterpret_cast<int2*>(p.part_ml + (long long)f.ctas * 2 * 8 * f.nt * 2);
  }
  if (dim == 128) {
    if (tree) return fmt == INT8 ? launch_few_nt<128, INT8, true>(p, f, st) : launch_few_nt<128, E4M3, true>(p, f, st);
    return fmt == INT8 ? launch_few_nt<128, INT8, false>(p, f, st) : launch_few_nt<128, E4M3, false>(p, f, st);
  }
  if (tree) return fmt == INT8 ? launch_few_nt<64, INT8, true>(p, f, st) : launch_few_nt<64, E4M3, true>(p, f, st);
  return fmt == INT8 ? launch_few_nt<64, INT8, false>(p, f, st) : launch_few_nt<64, E4M3, false>(p, f, st);
}

int code_map(CUtensorMap* m, const void* codes, long long rows, int dim, int box_rows) {
  typedef CUresult (*EncodeFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave,
                               CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
  static const EncodeFn fn = [] {
    void* f = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &f, cudaEnableDefault, &q) != cudaSuccess || q != cudaDriverEntryPointSuccess) f = nullptr;
    return reinterpret_cast<EncodeFn>(f);
  }();
  if (!fn) B200_FAIL(B200_ERR_CUDA, "cuTensorMapEncodeTiled not available");
  cuuint64_t dims[2] = {(cuuint64_t)dim, (cuuint64_t)rows}, strides[1] = {(cuuint64_t)dim};
  cuuint32_t box[2] = {(cuuint32_t)dim, (cuuint32_t)box_rows}, est[2] = {1, 1};
  const CUresult r = fn(m, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void*>(codes), dims, strides, box, est, CU_TENSOR_MAP_INTERLEAVE_NONE,
                        dim == 128 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) B200_FAIL(B200_ERR_CUDA, "paged cache: tensor map of %lld rows of %d codes refused (%d)", rows, dim, (int)r);
  return B200_OK;
}
int checked_cache(const b200_paged_cache* cache, const char* what) { return check_cache(cache, what); }
int checked(const b200_paged_cache* cache, const b200_paged_batch* batch, const char* what) {
  B200_TRY(check_cache(cache, what));
  return check_batch(cache, batch, what);
}
int attention_arguments(AttnP* p, const b200_paged_cache* cache, const b200_paged_batch* batch, const void* q_dev, int64_t q_ld, void* out_dev, int64_t out_ld, int q_heads, float scale, int window,
                        int sinks, const char* what) {
  B200_TRY(checked(cache, batch, what));
  const int D = cache->dim, H = cache->kv_heads;
  if (q_heads < H || q_heads % H || q_heads / H > 256) B200_FAIL(B200_ERR_SHAPE, "%s: %d query heads on %d heads of the cache", what, q_heads, H);
  if (!(scale > 0.f && scale < INFINITY) || window < 0 || sinks < 0) B200_FAIL(B200_ERR_INVALID, "%s: scale %g, window %d, %d first tokens", what, (double)scale, window, sinks);
  if (batch->total_rows && batch->max_rows && (!rows_fit(q_dev, q_ld, q_heads, D) || !rows_fit(out_dev, out_ld, q_heads, D)))
    B200_FAIL(B200_ERR_INVALID, "%s: queries and results must begin on a 16-byte border, rows %lld and %lld elements apart", what, (long long)q_ld, (long long)out_ld);
  memset(p, 0, sizeof(*p));
  p->k = static_cast<const uint8_t*>(cache->k_dev); p->v = static_cast<const uint8_t*>(cache->v_dev); p->k_scale = cache->k_scale_dev; p->v_scale = cache->v_scale_dev;
  p->flags = cache->flags_dev; p->b = batch_of(batch); p->q = static_cast<const __nv_bfloat16*>(q_dev); p->out = static_cast<__nv_bfloat16*>(out_dev);
  p->q_ld = q_ld; p->out_ld = out_ld; p->pages = cache->pages; p->P = cache->page_tokens; p->page_shift = shift_of(p->P); p->H = H; p->G = q_heads / H;
  p->window = window; p->sinks = sinks; p->scale2 = scale * LOG2E;
  return B200_OK;
}

}  // namespace paged
}  // namespace b200

using namespace b200;

extern "C" {

static int append(const b200_paged_cache* cache, const b200_paged_batch* batch, const void* k_dev, int64_t k_ld, const void* v_dev, int64_t v_ld,
                  const void* q_dev, int64_t q_ld, void* q_out_dev, int64_t q_out_ld, int q_heads, const b200_rotary* rotary, const b200_paged_positions* at, void* stream) {
  using namespace b200::paged;
  B200_TRY(check_cache(cache, "paged_append"));
  B200_TRY(check_batch(cache, batch, "paged_append"));
  const int D = cache->dim;
  if (batch->total_rows == 0) return B200_OK;
  if (!rows_fit(k_dev, k_ld, cache->kv_heads, D) || !rows_fit(v_dev, v_ld, cache->kv_heads, D))
    B200_FAIL(B200_ERR_INVALID, "paged_append: keys and values must begin on a 16-byte border, rows %lld and %lld elements apart", (long long)k_ld, (long long)v_ld);
  if (q_dev && (q_heads < 1 || q_heads > 8192 || !rows_fit(q_dev, q_ld, q_heads, D) || !rows_fit(q_out_dev, q_out_ld, q_heads, D)))
    B200_FAIL(B200_ERR_INVALID, "paged_append: %d query heads, rows %lld and %lld elements apart, on a 16-byte border", q_heads, (long long)q_ld, (long long)q_out_ld);
  if (rotary && (!rotary->turns_dev || rotary->rot_dims < 16 || rotary->rot_dims % 16 || rotary->rot_dims > D || (rotary->pairing != B200_ROT_HALVES && rotary->pairing != B200_ROT_ADJACENT)))
    B200_FAIL(B200_ERR_INVALID, "paged_append: %d rotated dimensions (a multiple of 16, up to the head size), pairing %d", rotary->rot_dims, rotary->pairing);
  if (at && (!rotary || !at->positions_dev || at->axes < 1 || at->axes > 4 || at->ld < batch->total_rows || (at->axes > 1 && !at->pair_axis_dev) || (reinterpret_cast<uintptr_t>(at->pair_axis_dev) & 7)))
    B200_FAIL(B200_ERR_INVALID, "paged_append: positions of %d axes (1 to 4), %lld apart, of %d rows, with a rotation and an axis for each of its pairs on an 8-byte border", at->axes, (long long)at->ld, batch->total_rows);
  DeviceGuard guard(cache->device);
  AppendP p;
  p.k_codes = static_cast<uint8_t*>(cache->k_dev); p.v_codes = static_cast<uint8_t*>(cache->v_dev); p.k_scale = cache->k_scale_dev; p.v_scale = cache->v_scale_dev;
  p.flags = cache->flags_dev; p.b = batch_of(batch);
  p.k = static_cast<const __nv_bfloat16*>(k_dev); p.v = static_cast<const __nv_bfloat16*>(v_dev); p.q = static_cast<const __nv_bfloat16*>(q_dev);
  p.q_out = static_cast<__nv_bfloat16*>(q_out_dev); p.k_ld = k_ld; p.v_ld = v_ld; p.q_ld = q_ld; p.q_out_ld = q_out_ld;
  p.turns = rotary ? rotary->turns_dev : nullptr; p.rot = rotary ? rotary->rot_dims : 0; p.halves = rotary ? rotary->pairing == B200_ROT_HALVES : 0;
  p.positions = at ? at->positions_dev : nullptr; p.pair_axis = at ? at->pair_axis_dev : nullptr; p.positions_ld = at ? at->ld : 0; p.axes = at ? at->axes : 0;
  p.pages = cache->pages; p.P = cache->page_tokens; p.H = cache->kv_heads; p.Hq = q_dev ? q_heads : 0;
  const long long items = (long long)batch->total_rows / p.P + 2ll * batch->sequences;
  if (items * p.H * 2 > (1ll << 30)) B200_FAIL(B200_ERR_SHAPE, "paged_append: %d rows of %d sequences with %d heads in one call", batch->total_rows, batch->sequences, p.H);
  p.items = (int)items;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const bool i8 = cache->kv_dtype == B200_KV_INT8;
  int rc;
  if (at) {
    if (D == 128) rc = i8 ? launch_append<INT8, 128, true>(p, st) : launch_append<E4M3, 128, true>(p, st);
    else rc = i8 ? launch_append<INT8, 64, true>(p, st) : launch_append<E4M3, 64, true>(p, st);
  } else {
    if (D == 128) rc = i8 ? launch_append<INT8, 128, false>(p, st) : launch_append<E4M3, 128, false>(p, st);
    else rc = i8 ? launch_append<INT8, 64, false>(p, st) : launch_append<E4M3, 64, false>(p, st);
  }
  B200_TRY(rc);
  return check_launch("paged_append");
}
int b200_paged_append(const b200_paged_cache* cache, const b200_paged_batch* batch, const void* k_dev, int64_t k_ld, const void* v_dev, int64_t v_ld,
                      const void* q_dev, int64_t q_ld, void* q_out_dev, int64_t q_out_ld, int q_heads, const b200_rotary* rotary, void* stream) {
  return append(cache, batch, k_dev, k_ld, v_dev, v_ld, q_dev, q_ld, q_out_dev, q_out_ld, q_heads, rotary, nullptr, stream);
}
int b200_paged_append_at(const b200_paged_cache* cache, const b200_paged_batch* batch, const void* k_dev, int64_t k_ld, const void* v_dev, int64_t v_ld, const void* q_dev, int64_t q_ld,
                         void* q_out_dev, int64_t q_out_ld, int q_heads, const b200_rotary* rotary, const b200_paged_positions* positions, void* stream) {
  if (!positions) B200_FAIL(B200_ERR_INVALID, "paged_append_at: no positions");
  return append(cache, batch, k_dev, k_ld, v_dev, v_ld, q_dev, q_ld, q_out_dev, q_out_ld, q_heads, rotary, positions, stream);
}

int b200_paged_read(const b200_paged_cache* cache, const b200_paged_batch* batch, void* k_out_dev, void* v_out_dev, void* stream) {
  using namespace b200::paged;
  B200_TRY(check_cache(cache, "paged_read"));
  B200_TRY(check_batch(cache, batch, "paged_read"));
  if (batch->total_rows == 0) return B200_OK;
  const int D = cache->dim;
  if (!rows_fit(k_out_dev, (long long)cache->kv_heads * D, cache->kv_heads, D) || !rows_fit(v_out_dev, (long long)cache->kv_heads * D, cache->kv_heads, D))
    B200_FAIL(B200_ERR_INVALID, "paged_read: the results must begin on a 16-byte border");
  DeviceGuard guard(cache->device);
  ReadP p;
  p.k_codes = static_cast<const uint8_t*>(cache->k_dev); p.v_codes = static_cast<const uint8_t*>(cache->v_dev); p.k_scale = cache->k_scale_dev; p.v_scale = cache->v_scale_dev;
  p.flags = cache->flags_dev; p.b = batch_of(batch); p.k = static_cast<__nv_bfloat16*>(k_out_dev); p.v = static_cast<__nv_bfloat16*>(v_out_dev);
  p.pages = cache->pages; p.P = cache->page_tokens; p.H = cache->kv_heads;
  const dim3 grid((unsigned)ceil_div(batch->total_rows, READ_THREADS / 64) + 1);        // the last one looks at the sequences
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const bool i8 = cache->kv_dtype == B200_KV_INT8;
  if (D == 128) { if (i8) EARLY_LAUNCH((read_kernel<INT8, 128>), grid, READ_THREADS, 0, st, p); else EARLY_LAUNCH((read_kernel<E4M3, 128>), grid, READ_THREADS, 0, st, p); }
  else { if (i8) EARLY_LAUNCH((read_kernel<INT8, 64>), grid, READ_THREADS, 0, st, p); else EARLY_LAUNCH((read_kernel<E4M3, 64>), grid, READ_THREADS, 0, st, p); }
  return check_launch("paged_read");
}

int64_t b200_paged_attention_bytes(const b200_paged_cache* cache, const b200_paged_batch* batch, int q_heads, int window, int sinks) {
  using namespace b200::paged;
  if (!cache || !batch || cache->kv_heads < 1 || q_heads < cache->kv_heads || q_heads % cache->kv_heads || window < 0 || sinks < 0 || batch->sequences < 1 || batch->max_rows < 0) return 0;
  const int G = q_heads / cache->kv_heads;
  if (batch->total_rows <= 0 || batch->max_rows == 0) return 0;
  const Route r = route(cache, batch, G, window, sinks);
  return r.few_bytes + r.prompt_bytes;
}

int b200_paged_attention(const b200_paged_cache* cache, const b200_paged_batch* batch, const void* q_dev, int64_t q_ld, void* out_dev, int64_t out_ld, int q_heads,
                         float scale, int window, int sinks, void* work_dev, int64_t work_bytes, void* stream) {
  using namespace b200::paged;
  AttnP p;
  B200_TRY(attention_arguments(&p, cache, batch, q_dev, q_ld, out_dev, out_ld, q_heads, scale, window, sinks, "paged_attention"));
  if (batch->total_rows == 0 || batch->max_rows == 0) return B200_OK;
  DeviceGuard guard(cache->device);
  const int D = cache->dim;
  const Route r = route(cache, batch, p.G, window, sinks);
  if (r.few.units > 0x7fffffffll / 64 || r.prompt.units * (r.prompt.nsplit ? r.prompt.nsplit : 1) > 0x7fffffffll / 64 || (long long)batch->max_rows * p.G > 0x3fffffffll)
    B200_FAIL(B200_ERR_SHAPE, "paged_attention: %d sequences of up to %d rows with %d heads in one call", batch->sequences, batch->max_rows, q_heads);
  const int64_t need = r.few_bytes + r.prompt_bytes;
  if (need > 0 && (!work_dev || work_bytes < need || (reinterpret_cast<uintptr_t>(work_dev) & 15)))
    B200_FAIL(B200_ERR_INVALID, "paged_attention: a workspace of %lld bytes; b200_paged_attention_bytes asks for %lld, on a 16-byte border", (long long)work_bytes, (long long)need);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const int fmt = cache->kv_dtype == B200_KV_INT8 ? INT8 : E4M3;
  p.from_rows = r.from_rows;
  if (r.prompt.units) {
    AttnP x = p;
    x.q_tiles = r.prompt.q_tiles; x.nsplit = r.prompt.nsplit;
    if (r.prompt_bytes) {
      x.part_o = reinterpret_cast<float*>(static_cast<uint8_t*>(work_dev) + r.few_bytes);
      x.part_ml = x.part_o + r.prompt_bytes / 4 / (D + 2) * D;
    }
    B200_TRY(prompt_attention(x, r.prompt, fmt, D, st));
  }
  if (r.few.units) B200_TRY(few_attention(p, r.few, fmt, D, false, work_dev, st));
  return check_launch("paged_attention");
}

}  // extern "C"
