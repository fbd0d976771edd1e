// A cache of keys and values in 8 bits whose memory goes to sequences page by page: append with the position rotation on the way, reading back, and attention
// of few rows per sequence (decoding, drafts); long portions are paged_prompt.cu's.
//
// Codes lie as [pages][kv heads][tokens of a page][dim], int8 or e4m3, with one scale per page, head and side (keys, values): a page's tokens of one head are one
// run of memory.  A page's scale s is (largest magnitude) / (largest code) of the rows that began the page; rows that come later may need more, and then
// it is doubled until they fit and the older codes are halved as often.  Only doubling keeps a page that grows token by token within one step of its last scale:
// a half step from the first rounding, and halves, quarters .. of it from those before.  (Growing to the exact maximum each time, the roundings of a slowly growing page all have the
// same sign: 0.1 % a token never changes a code, and after 64 tokens the largest are 8 steps off.)  For e4m3 halving is exact but for subnormals.
#include "paged.cuh"

#include "tc_prims.cuh"

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
  int pages, P, H, Hq, page_tasks, page_ctas, q_rows;
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
__device__ __forceinline__ void load16(float* x, const bf16* row, const Chunk& c) {
  const uint4 a = *reinterpret_cast<const uint4*>(row + c.lo), b = *reinterpret_cast<const uint4*>(row + c.hi);
  const uint32_t w[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float2 f = unpack_bf16(w[i]);
    x[2 * i] = f.x; x[2 * i + 1] = f.y;
  }
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

constexpr int APPEND_THREADS = 256;

// A team of threads per (page that the step touches, kv head, side).  What the step adds to a page is read once and held in registers (KEEP sweeps of the team over the
// rows; further ones are read again), because the page's scale has to be known before its first code.  The queries' blocks come behind the pages'.
//
// The step's touched pages are numbered without a pass over the sequences: sequence s has the numbers from rows[s] / P + 2 s on, and n rows from any place in a page on
// touch at most n / P + 2 pages.
// Bounds: bytes for prompts, the launch and a chain of four dependent reads for a frame.
template <int FMT, int D, int TEAM, int KEEP>
__global__ void __launch_bounds__(APPEND_THREADS) append_kernel(const AppendP p) {
  pdl_trigger();
  pdl_wait();
  constexpr int CHUNKS = D / 16, RPS = TEAM / CHUNKS, TEAMS = APPEND_THREADS / TEAM;
  const int tid = threadIdx.x, lane = tid & 31;
  if ((int)blockIdx.x >= p.page_ctas) {                 // ---- queries: rotate, round, store ----
    __shared__ int row_pos[APPEND_THREADS / CHUNKS];
    const int slots = (APPEND_THREADS / CHUNKS) / p.q_rows;      // heads side by side
    const int r_first = ((int)blockIdx.x - p.page_ctas) * p.q_rows;
    for (int i = tid >> 5; i < p.q_rows; i += APPEND_THREADS / 32) {
      const int r = r_first + i;
      int pos = -1;
      if (r < p.b.T) {
        const int s = sequence_of_row(p.b, r);
        if (s < p.b.S) {
          const Seq q = sequence(p.b, s, p.P);
          if (q.ok && r >= q.r0) pos = q.before + r - q.r0;
        }
      }
      if (lane == 0) row_pos[i] = pos;
    }
    __syncthreads();
    const int slot = tid / CHUNKS, j = tid % CHUNKS, i = slot / slots, r = r_first + i, pos = row_pos[i];
    if (pos < 0) return;
    const Chunk c(j, p.rot, p.halves);
    Turn t;
    if (c.turned) turn_of(t, p.turns, j, pos);
    for (int h = slot % slots; h < p.Hq; h += slots) {
      float x[16];
      load16(x, p.q + r * p.q_ld + (long long)h * D, c);
      if (c.turned) { if (p.halves) rotate16(x, t, 1); else rotate16(x, t, 0); }
      bf16* out = p.q_out + r * p.q_out_ld + (long long)h * D;
      *reinterpret_cast<uint4*>(out + c.lo) = make_uint4(pack_bf16(x[0], x[1]), pack_bf16(x[2], x[3]), pack_bf16(x[4], x[5]), pack_bf16(x[6], x[7]));
      *reinterpret_cast<uint4*>(out + c.hi) = make_uint4(pack_bf16(x[8], x[9]), pack_bf16(x[10], x[11]), pack_bf16(x[12], x[13]), pack_bf16(x[14], x[15]));
    }
    return;
  }

  // ---- pages ----
  const int task = (int)blockIdx.x * TEAMS + tid / TEAM, me = tid % TEAM;
  if (task >= p.page_tasks) return;                     // whole teams
  const int side = task & 1, h = (task >> 1) % p.H, item = (task >> 1) / p.H;
  int s = 0;                                            // the last sequence whose numbers begin at or in front of `item`
  for (int i = lane + 1; i - lane - 1 < p.b.S - 1; i += 32) s += __popc(__ballot_sync(0xffffffffu, i < p.b.S && (long long)p.b.rows[i] / p.P + 2ll * i <= item));
  const Seq q = sequence(p.b, s, p.P);
  const int block = (q.ok ? q.before : 0) / p.P + item - (q.ok ? q.r0 / p.P + 2 * s : 0);
  if (!q.ok) {
    if (me == 0) flag(p.flags, B200_PAGED_BAD_BATCH);
    return;
  }
  const long long page_first = (long long)block * p.P;
  if (q.n == 0 || page_first >= (long long)q.before + q.n) return;
  const int page = p.b.table[s * p.b.table_ld + block];
  if (page < 0 || page >= p.pages) {
    if (me == 0) flag(p.flags, B200_PAGED_BAD_PAGE);
    return;
  }
  const int o = max(q.before - (int)page_first, 0), e = (int)min((long long)q.before + q.n - page_first, (long long)p.P);
  const int r = q.r0 + (int)(page_first + o - q.before);            // batch row of slot o
  const bool keys = side == 0;
  const int rot = keys ? p.rot : 0;
  const bf16* src = (keys ? p.k : p.v) + (long long)h * D;
  const long long ld = keys ? p.k_ld : p.v_ld;
  uint8_t* codes = (keys ? p.k_codes : p.v_codes) + ((long long)page * p.H + h) * p.P * D;
  float* scale_at = (keys ? p.k_scale : p.v_scale) + (long long)page * p.H + h;
  const float s_old = o > 0 ? *scale_at : 0.f;
  const int j = me % CHUNKS, row0 = me / CHUNKS;
  const Chunk c(j, rot, p.halves);
  float top = 0.f;
  bool odd = false;                                     // a value that is not finite, or too large
  auto fetch = [&](float* x, int slot) {
    load16(x, src + (r + slot - o) * ld, c);
    if (c.turned) {
      Turn t;
      turn_of(t, p.turns, j, (int)page_first + slot);
      if (p.halves) rotate16(x, t, 1); else rotate16(x, t, 0);
    }
#pragma unroll
    for (int i = 0; i < 16; ++i)
      if (!(fabsf(x[i]) <= MAGNITUDE)) { x[i] = 0.f; odd = true; }
  };
  float kept[KEEP][16];
#pragma unroll
  for (int k = 0; k < KEEP; ++k) {
    const int slot = o + row0 + k * RPS;
    if (slot < e) fetch(kept[k], slot);
    else {
#pragma unroll
      for (int i = 0; i < 16; ++i) kept[k][i] = 0.f;
    }
#pragma unroll
    for (int i = 0; i < 16; ++i) top = fmaxf(top, fabsf(kept[k][i]));
  }
  for (int slot = o + row0 + KEEP * RPS; slot < e; slot += RPS) {
    float x[16];
    fetch(x, slot);
#pragma unroll
    for (int i = 0; i < 16; ++i) top = fmaxf(top, fabsf(x[i]));
  }
  top = warp_max(top);
  if constexpr (TEAM > 32) {
    __shared__ float tops[TEAM / 32];
    if (lane == 0) tops[tid >> 5] = top;
    __syncthreads();                                    // one team: all threads of the block are here
#pragma unroll
    for (int i = 0; i < TEAM / 32; ++i) top = fmaxf(top, tops[i]);
  }
  if (__any_sync(0xffffffffu, odd) && lane == 0) flag(p.flags, B200_PAGED_NOT_FINITE);
  const float need = top > 0.f ? fmaxf(top / code_max<FMT>(), SCALE_MIN) : 0.f;
  float sc = need;
  int doublings = 0;
  if (s_old > 0.f) {
    sc = s_old;
    if (need > s_old) {                                 // the least power of two with s_old * 2^k >= need
      const float ratio = need / s_old;
      int power;
      const float part = frexpf(ratio, &power);
      doublings = part == 0.5f ? power - 1 : power;
      sc = ldexpf(s_old, doublings);
    }
  }
  __syncwarp();
  if (me == 0) *scale_at = sc;
  const float div = sc > 0.f ? sc : 1.f;
  auto store = [&](const float* x, int slot) {
    uint8_t* row = codes + (long long)slot * D;
    float y[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) y[i] = x[i] / div;
    *reinterpret_cast<uint2*>(row + c.lo) = make_uint2(codes4<FMT>(y[0], y[1], y[2], y[3]), codes4<FMT>(y[4], y[5], y[6], y[7]));
    *reinterpret_cast<uint2*>(row + c.hi) = make_uint2(codes4<FMT>(y[8], y[9], y[10], y[11]), codes4<FMT>(y[12], y[13], y[14], y[15]));
  };
#pragma unroll
  for (int k = 0; k < KEEP; ++k)
    if (o + row0 + k * RPS < e) store(kept[k], o + row0 + k * RPS);
  for (int slot = o + row0 + KEEP * RPS; slot < e; slot += RPS) {
    float x[16];
    fetch(x, slot);
    store(x, slot);
  }
  if (o > 0 && (doublings > 0 || !(s_old > 0.f))) {     // the older rows' codes in the new scale
    const float by = s_old > 0.f ? ldexpf(1.f, -doublings) : 0.f;
    for (int slot = row0; slot < o; slot += RPS) {
      uint4* at = reinterpret_cast<uint4*>(codes + (long long)slot * D + 16 * j);
      const uint4 was = *at;
      const uint32_t w[4] = {was.x, was.y, was.z, was.w};
      uint32_t now[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float2 a = float2_of<FMT, 0>(ready<FMT>(w[i])), b = float2_of<FMT, 1>(ready<FMT>(w[i]));
        now[i] = s_old > 0.f ? codes4<FMT>(a.x * by, a.y * by, b.x * by, b.y * by) : 0u;
      }
      *at = make_uint4(now[0], now[1], now[2], now[3]);
    }
  }
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
constexpr int READ_THREADS = 256, READ_ROWS = 4;

template <int FMT, int D>
__global__ void __launch_bounds__(READ_THREADS) read_kernel(const ReadP p) {
  pdl_trigger();
  pdl_wait();
  __shared__ int at[READ_ROWS][2];           // page and slot of the rows
  const int warp = threadIdx.x >> 5, r_first = (int)blockIdx.x * READ_ROWS;
  if (warp < READ_ROWS) {
    const int r = r_first + warp;
    int page = -1, slot = 0;
    if (r < p.b.T) {
      const int s = sequence_of_row(p.b, r);
      if (s < p.b.S) {
        const Seq q = sequence(p.b, s, p.P);
        if (q.ok && r >= q.r0) {
          const int pos = q.before + r - q.r0;
          page = p.b.table[s * p.b.table_ld + pos / p.P];
          slot = pos % p.P;
          if (page < 0 || page >= p.pages) { page = -1; if ((threadIdx.x & 31) == 0) flag(p.flags, B200_PAGED_BAD_PAGE); }
        } else if (!q.ok && (threadIdx.x & 31) == 0) flag(p.flags, B200_PAGED_BAD_BATCH);
      }
    }
    if ((threadIdx.x & 31) == 0) { at[warp][0] = page; at[warp][1] = slot; }
  }
  __syncthreads();
  constexpr int CHUNKS = D / 16;
  const int per_row = p.H * CHUNKS * 2;
  for (int i = threadIdx.x; i < per_row * READ_ROWS; i += READ_THREADS) {
    const int row = i / per_row, x = i - row * per_row, side = x >= per_row / 2, y = x - side * (per_row / 2), h = y / CHUNKS, j = y % CHUNKS;
    const int page = at[row][0];
    if (page < 0) continue;
    const long long ph = (long long)page * p.H + h;
    const float sc = (side ? p.v_scale : p.k_scale)[ph];
    const uint4 c = *reinterpret_cast<const uint4*>((side ? p.v_codes : p.k_codes) + (ph * p.P + at[row][1]) * D + 16 * j);
    const uint32_t w[4] = {c.x, c.y, c.z, c.w};
    uint32_t o[8];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const float2 a = float2_of<FMT, 0>(ready<FMT>(w[k])), b = float2_of<FMT, 1>(ready<FMT>(w[k]));
      o[2 * k] = pack_bf16(a.x * sc, a.y * sc);
      o[2 * k + 1] = pack_bf16(b.x * sc, b.y * sc);
    }
    bf16* out = (side ? p.v : p.k) + ((long long)(r_first + row) * p.H + h) * D + 16 * j;
    *reinterpret_cast<uint4*>(out) = make_uint4(o[0], o[1], o[2], o[3]);
    *reinterpret_cast<uint4*>(out + 8) = make_uint4(o[4], o[5], o[6], o[7]);
  }
}

// =========================================================================================================================
// attention of few rows
// =========================================================================================================================
// Columns are (row of the sequence, query head of the group); a CTA has 8 * NT of them, one kv head and a range of the keys, in tiles of 16 tokens that its warps take in
// turn.  Both products have the cache as the first operand of mma.m16n8k16: S^T = K Q^T (tokens x columns) and O^T += V^T P^T (dims x columns), so a single row of one head
// wastes tensor-core columns and not cache bytes.  Codes go from memory into registers as fragments, 16 bytes at a time: which dimension of K is which
// k of the product is free as long as Q has the same order, and so is which dimension of V is which row of O^T.  P^T comes out of S^T by movmatrix.
//
// Codes of both types are exact in f16, and so are bf16 queries after a power of two per column; P is f16 in (0, 2^8].  The scale of a page's keys multiplies the scores; that of its
// values goes into the exponent, P = 2^(score + log2 s_v - M), with M the running maximum of the same, and the sum of the weights takes P / s_v: nothing is rounded on the way but P.
// M follows only when a score passes it by 2^8, as then no column has to be compared across lanes for most tiles.
constexpr int FEW_WARPS = 4, FEW_THREADS = FEW_WARPS * 32;
constexpr float SLACK = 8.f;

__device__ __forceinline__ uint4 load_stream16(const void* p) {
  uint4 r;
  asm volatile("ld.global.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(r.x), "=r"(r.y), "=r"(r.z), "=r"(r.w) : "l"(p));
  return r;
}
__device__ __forceinline__ uint2 load_stream8(const void* p) {
  uint2 r;
  asm volatile("ld.global.L1::no_allocate.v2.u32 {%0, %1}, [%2];" : "=r"(r.x), "=r"(r.y) : "l"(p));
  return r;
}
__device__ __forceinline__ void mma_f16(float* d, uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
               : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t transposed8x8(uint32_t a) {
  uint32_t r;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(a));
  return r;
}
__device__ __forceinline__ uint32_t pack_f16(float a, float b) {
  const __half2 v = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&v);
}

template <int D>
struct Codes {                               // a warp's tile of 16 tokens, as its lanes hold it
  uint32_t k[2][D / 16], v[4][D / 32];
};

template <int D, int FMT, int NT>
__global__ void __launch_bounds__(FEW_THREADS, NT == 1 ? 4 : NT == 2 ? 3 : 2) few_rows_kernel(const AttnP p) {
  pdl_trigger();
  pdl_wait();
  constexpr int KS = D / 16, MT = D / 16, COLS = 8 * NT;
  __shared__ float o_s[FEW_WARPS][8][D + 4];
  __shared__ float m_s[FEW_WARPS][8], l_s[FEW_WARPS][8];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, c = lane & 3;
  int u = (int)blockIdx.x;
  const int split = u % p.nsplit; u /= p.nsplit;
  const int ct = u % p.ctiles; u /= p.ctiles;
  const int h = u % p.H, s = u / p.H;
  const Seq q = sequence(p.b, s, p.P);
  if (!q.ok) {
    if (threadIdx.x == 0) flag(p.flags, B200_PAGED_BAD_BATCH);
    return;
  }
  const int n_cols = q.n * p.G, c0 = ct * COLS;
  if (q.n >= p.from_rows || c0 >= n_cols) return;
  const int pf = q.before + c0 / p.G, pl = q.before + (min(c0 + COLS, n_cols) - 1) / p.G;
  const Tiles<4> tiles(pf, pl, p.window, p.sinks);
  const int per = (tiles.n + p.nsplit - 1) / p.nsplit, t0 = split * per, t1 = min(t0 + per, tiles.n);
  if (t0 >= t1) return;

  // queries: lane (g, c) has of column 8 nt + g the dimensions 64 i + 16 c .. + 15
  uint32_t qf[NT][KS][2];
  float fac[NT][2];                          // of columns 8 nt + 2 c, + 1: what turns a product of codes into a score in base 2
  int pos[NT][2];
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
    const int col = c0 + nt * 8 + g;
    const bool has = col < n_cols;
    const int i = has ? col / p.G : 0;
    const bf16* row = p.q + (long long)(q.r0 + i) * p.q_ld + (long long)(h * p.G + (has ? col - i * p.G : 0)) * D;
    uint32_t raw[KS][2];
    float top = 0.f;
#pragma unroll
    for (int b = 0; b < D / 64; ++b) {
      const uint4 x = has ? *reinterpret_cast<const uint4*>(row + 64 * b + 16 * c) : make_uint4(0, 0, 0, 0);
      const uint4 y = has ? *reinterpret_cast<const uint4*>(row + 64 * b + 16 * c + 8) : make_uint4(0, 0, 0, 0);
      raw[4 * b][0] = x.x; raw[4 * b][1] = x.y; raw[4 * b + 1][0] = x.z; raw[4 * b + 1][1] = x.w;
      raw[4 * b + 2][0] = y.x; raw[4 * b + 2][1] = y.y; raw[4 * b + 3][0] = y.z; raw[4 * b + 3][1] = y.w;
    }
#pragma unroll
    for (int k = 0; k < KS; ++k)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const float2 f = unpack_bf16(raw[k][e]);
        const float a = fabsf(f.x), b = fabsf(f.y);
        if (a < INFINITY) top = fmaxf(top, a);
        if (b < INFINITY) top = fmaxf(top, b);
      }
    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
    const float power = top > 0.f ? power_of_two_in(top) : 1.f;
    const float up = 16384.f / power;        // the column's largest lands in [2^14, 2^15)
#pragma unroll
    for (int k = 0; k < KS; ++k)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const float2 f = unpack_bf16(raw[k][e]);
        qf[nt][k][e] = pack_f16(f.x * up, f.y * up);
      }
    const float back = power * (1.f / 16384.f);
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      fac[nt][e] = __shfl_sync(0xffffffffu, back, (2 * c + e) * 4) * p.scale2;
      const int cc = c0 + nt * 8 + 2 * c + e;
      pos[nt][e] = cc < n_cols ? q.before + cc / p.G : -1;
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

  const int32_t* table = p.b.table + s * p.b.table_ld;
  const long long head = (long long)h * p.P, page_rows = (long long)p.H * p.P;
  // lane i has the page and scales of the warp's i-th tile from here on
  int my_page = -1;
  float my_ks = 0.f, my_vs = 1.f;
  auto look_up = [&](int t) {
    const int mine = t + lane * FEW_WARPS;
    my_page = -1; my_ks = 0.f; my_vs = 1.f;
    if (mine < t1) {
      const int page = table[(tiles[mine] << 4) >> p.page_shift];
      if (page >= 0 && page < p.pages) {
        my_page = page;
        my_ks = p.k_scale[(long long)page * p.H + h];
        const float v = p.v_scale[(long long)page * p.H + h];
        my_vs = v > 0.f ? v : 1.f;           // all codes of a page of zeros are 0
      } else flag(p.flags, B200_PAGED_BAD_PAGE);
    }
  };
  auto load = [&](Codes<D>& x, int t, int page) {
    if (page < 0) {
#pragma unroll
      for (int a = 0; a < 2; ++a)
#pragma unroll
        for (int b = 0; b < D / 16; ++b) x.k[a][b] = 0;
#pragma unroll
      for (int a = 0; a < 4; ++a)
#pragma unroll
        for (int b = 0; b < D / 32; ++b) x.v[a][b] = 0;
      return;
    }
    const long long at = (page * page_rows + head + ((tiles[t] << 4) & (p.P - 1))) * D;
    const uint8_t *k = p.k + at + 16 * c, *v = p.v + at + (D / 8) * g;
#pragma unroll
    for (int a = 0; a < 2; ++a)
#pragma unroll
      for (int b = 0; b < D / 64; ++b) {
        const uint4 w = load_stream16(k + (g + 8 * a) * D + 64 * b);
        x.k[a][4 * b] = w.x; x.k[a][4 * b + 1] = w.y; x.k[a][4 * b + 2] = w.z; x.k[a][4 * b + 3] = w.w;
      }
#pragma unroll
    for (int a = 0; a < 4; ++a) {
      const uint8_t* at_v = v + (2 * c + (a & 1) + 8 * (a >> 1)) * D;
      if constexpr (D == 128) {
        const uint4 w = load_stream16(at_v);
        x.v[a][0] = w.x; x.v[a][1] = w.y; x.v[a][2] = w.z; x.v[a][3] = w.w;
      } else {
        const uint2 w = load_stream8(at_v);
        x.v[a][0] = w.x; x.v[a][1] = w.y;
      }
    }
  };
  auto work = [&](Codes<D>& x, int t, int page, float ks, float vs) {
    float sc[NT][4];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) sc[nt][0] = sc[nt][1] = sc[nt][2] = sc[nt][3] = 0.f;
#pragma unroll
    for (int k = 0; k < KS; ++k) {
      const uint32_t w0 = ready<FMT>(x.k[0][k]), w1 = ready<FMT>(x.k[1][k]);
      const uint32_t a0 = half2_of<FMT, 0>(w0), a1 = half2_of<FMT, 0>(w1), a2 = half2_of<FMT, 1>(w0), a3 = half2_of<FMT, 1>(w1);
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) mma_f16(sc[nt], a0, a1, a2, a3, qf[nt][k][0], qf[nt][k][1]);
    }
    const float lv = __log2f(vs), inv = __frcp_rn(vs);
    const int j0 = tiles[t] << 4;
    const bool whole = page >= 0 && j0 + 15 <= pf && (p.window <= 0 || pl - j0 < p.window || j0 + 16 <= p.sinks);
    if (!whole) {                            // codes of tokens that no column sees may be anything
#pragma unroll
      for (int a = 0; a < 4; ++a) {
        const int j = j0 + 2 * c + (a & 1) + 8 * (a >> 1);
        if (!(j <= pl && (p.window <= 0 || pf - j < p.window || j < p.sinks))) {
#pragma unroll
          for (int b = 0; b < D / 32; ++b) x.v[a][b] = 0;
        }
      }
    }
    bool grow = false;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        float v = fmaf(sc[nt][e], ks * fac[nt][e & 1], lv);
        if (!whole && !(page >= 0 && sees(pos[nt][e & 1], j0 + g + 8 * (e >> 1), p.window, p.sinks))) v = -INFINITY;
        sc[nt][e] = v;
        grow |= v > m[nt][e & 1] + SLACK;
      }
    if (__any_sync(0xffffffffu, grow)) {
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          float top = fmaxf(sc[nt][e], sc[nt][e + 2]);
          top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 4));
          top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 8));
          top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 16));
          const float now = fmaxf(m[nt][e], top), by = now == -INFINITY ? 1.f : exp2_fast(m[nt][e] - now);
          m[nt][e] = now;
          l[nt][e] *= by;
#pragma unroll
          for (int i = 0; i < MT; ++i) { o[nt][i][e] *= by; o[nt][i][e + 2] *= by; }
        }
    }
    uint32_t b0[NT], b1[NT];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      float w[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) w[e] = exp2_fast(sc[nt][e] - (m[nt][e & 1] == -INFINITY ? 0.f : m[nt][e & 1]));
      l[nt][0] = fmaf(w[0] + w[2], inv, l[nt][0]);
      l[nt][1] = fmaf(w[1] + w[3], inv, l[nt][1]);
      b0[nt] = transposed8x8(pack_f16(w[0], w[1]));
      b1[nt] = transposed8x8(pack_f16(w[2], w[3]));
    }
#pragma unroll
    for (int j = 0; j < D / 32; ++j) {       // four dimensions of this lane's: words of tokens 2 c, 2 c + 1, 2 c + 8, 2 c + 9
      const uint32_t v0 = ready<FMT>(x.v[0][j]), v1 = ready<FMT>(x.v[1][j]), v2 = ready<FMT>(x.v[2][j]), v3 = ready<FMT>(x.v[3][j]);
      const uint32_t lo = prmt(v0, v1, 0x5140u), hi = prmt(v0, v1, 0x7362u), lo8 = prmt(v2, v3, 0x5140u), hi8 = prmt(v2, v3, 0x7362u);
      const uint32_t a[8] = {half2_of<FMT, 0>(lo), half2_of<FMT, 1>(lo), half2_of<FMT, 0>(lo8), half2_of<FMT, 1>(lo8),
                             half2_of<FMT, 0>(hi), half2_of<FMT, 1>(hi), half2_of<FMT, 0>(hi8), half2_of<FMT, 1>(hi8)};
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        mma_f16(o[nt][2 * j], a[0], a[1], a[2], a[3], b0[nt], b1[nt]);
        mma_f16(o[nt][2 * j + 1], a[4], a[5], a[6], a[7], b0[nt], b1[nt]);
      }
    }
  };

  // the next tile's codes are on their way while a tile is worked on
  Codes<D> x, y;
  int at = 0;
  const int first = t0 + warp;
  if (first < t1) {
    look_up(first);
    int page = __shfl_sync(0xffffffffu, my_page, 0);
    float ks = __shfl_sync(0xffffffffu, my_ks, 0), vs = __shfl_sync(0xffffffffu, my_vs, 0);
    load(x, first, page);
    for (int t = first; t < t1; t += FEW_WARPS) {
      const int next = t + FEW_WARPS;
      int page2 = -1;
      float ks2 = 0.f, vs2 = 1.f;
      if (next < t1) {
        if (++at == 32) { look_up(next); at = 0; }
        page2 = __shfl_sync(0xffffffffu, my_page, at);
        ks2 = __shfl_sync(0xffffffffu, my_ks, at);
        vs2 = __shfl_sync(0xffffffffu, my_vs, at);
        load(y, next, page2);
      }
      work(x, t, page, ks, vs);
      x = y; page = page2; ks = ks2; vs = vs2;
    }
  }

  // join the warps, eight columns at a time
  const int unit = (s * p.H + h) * p.ctiles + ct;
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
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
    constexpr int PER = D / 16;              // 16 threads a column
    const int col = threadIdx.x >> 4, d0 = (threadIdx.x & 15) * PER;
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
    const int cc = c0 + nt * 8 + col;
    if (p.nsplit > 1) {
      const long long at_part = ((long long)unit * p.nsplit + split) * COLS + nt * 8 + col;
      if ((threadIdx.x & 15) == 0) *reinterpret_cast<float2*>(p.part_ml + 2 * at_part) = make_float2(top, sum);
#pragma unroll
      for (int i = 0; i < PER; i += 4) *reinterpret_cast<float4*>(p.part_o + at_part * D + d0 + i) = make_float4(acc[i], acc[i + 1], acc[i + 2], acc[i + 3]);
    } else if (cc < n_cols) {
      const float by = sum != 0.f ? 1.f / sum : 0.f;
      const int i = cc / p.G;
      bf16* out = p.out + (long long)(q.r0 + i) * p.out_ld + (long long)(h * p.G + cc - i * p.G) * D + d0;
      uint32_t w[PER / 2];
#pragma unroll
      for (int e = 0; e < PER / 2; ++e) w[e] = pack_bf16(acc[2 * e] * by, acc[2 * e + 1] * by);
      if constexpr (PER == 8) *reinterpret_cast<uint4*>(out) = make_uint4(w[0], w[1], w[2], w[3]);
      else *reinterpret_cast<uint2*>(out) = make_uint2(w[0], w[1]);
    }
    __syncthreads();
  }
}

// Joins the ranges of the keys: eight columns of a unit per CTA.
template <int D, int NT>
__global__ void __launch_bounds__(128) join_kernel(const AttnP p) {
  pdl_trigger();
  pdl_wait();
  constexpr int COLS = 8 * NT, PER = D / 16;
  int u = (int)blockIdx.x;
  const int nt = u % NT; u /= NT;
  const int unit = u, ct = u % p.ctiles; u /= p.ctiles;
  const int h = u % p.H, s = u / p.H;
  const Seq q = sequence(p.b, s, p.P);
  const int n_cols = q.n * p.G, c0 = ct * COLS, col = threadIdx.x >> 4, cc = c0 + nt * 8 + col, d0 = (threadIdx.x & 15) * PER;
  if (!q.ok || q.n >= p.from_rows || cc >= n_cols) return;
  const Tiles<4> tiles(q.before + c0 / p.G, q.before + (min(c0 + COLS, n_cols) - 1) / p.G, p.window, p.sinks);
  const int per = (tiles.n + p.nsplit - 1) / p.nsplit, parts = (tiles.n + per - 1) / per;
  const float2* ml = reinterpret_cast<const float2*>(p.part_ml);
  const long long first = (long long)unit * p.nsplit * COLS + nt * 8 + col;
  float top = -INFINITY;
  for (int i = 0; i < parts; ++i) top = fmaxf(top, ml[first + (long long)i * COLS].x);
  float sum = 0.f, acc[PER];
#pragma unroll
  for (int e = 0; e < PER; ++e) acc[e] = 0.f;
#pragma unroll 4
  for (int i = 0; i < parts; ++i) {
    const float2 x = ml[first + (long long)i * COLS];
    const float by = x.x == -INFINITY ? 0.f : exp2_fast(x.x - top);
    sum = fmaf(x.y, by, sum);
    const float4* o = reinterpret_cast<const float4*>(p.part_o + (first + (long long)i * COLS) * D + d0);
#pragma unroll
    for (int e = 0; e < PER / 4; ++e) {
      const float4 v = o[e];
      acc[4 * e] = fmaf(v.x, by, acc[4 * e]); acc[4 * e + 1] = fmaf(v.y, by, acc[4 * e + 1]);
      acc[4 * e + 2] = fmaf(v.z, by, acc[4 * e + 2]); acc[4 * e + 3] = fmaf(v.w, by, acc[4 * e + 3]);
    }
  }
  const float by = sum != 0.f ? 1.f / sum : 0.f;
  const int i = cc / p.G;
  bf16* out = p.out + (long long)(q.r0 + i) * p.out_ld + (long long)(h * p.G + cc - i * p.G) * D + d0;
  uint32_t w[PER / 2];
#pragma unroll
  for (int e = 0; e < PER / 2; ++e) w[e] = pack_bf16(acc[2 * e] * by, acc[2 * e + 1] * by);
  if constexpr (PER == 8) *reinterpret_cast<uint4*>(out) = make_uint4(w[0], w[1], w[2], w[3]);
  else *reinterpret_cast<uint2*>(out) = make_uint2(w[0], w[1]);
}

// =========================================================================================================================
// host
// =========================================================================================================================
int check_cache(const b200_paged_cache* c, const char* what) {
  if (!c || !c->k_dev || !c->v_dev || !c->k_scale_dev || !c->v_scale_dev || !c->flags_dev) B200_FAIL(B200_ERR_INVALID, "%s: null pointer in the cache", what);
  if (c->kv_dtype != B200_KV_INT8 && c->kv_dtype != B200_KV_FP8_E4M3) B200_FAIL(B200_ERR_INVALID, "%s: kv_dtype %d", what, c->kv_dtype);
  if (c->dim != 64 && c->dim != 128) B200_FAIL(B200_ERR_SHAPE, "%s: head size %d (64 or 128)", what, c->dim);
  if (c->page_tokens != 16 && c->page_tokens != 32 && c->page_tokens != 64 && c->page_tokens != 128) B200_FAIL(B200_ERR_SHAPE, "%s: pages of %d tokens (16, 32, 64 or 128)", what, c->page_tokens);
  if (c->pages < 1 || c->kv_heads < 1 || c->kv_heads > 1024) B200_FAIL(B200_ERR_SHAPE, "%s: %d pages, %d heads", what, c->pages, c->kv_heads);
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

// How the keys of a step are cut.  CTAs of 8 * nt columns; ranges so that the chip has about one wave of CTAs (four to an SM, 148 SMs), none shorter than 16 tiles
// (two rounds of a CTA's warps, twice) by the longest that the tables allow.
struct FewPlan { int nt, ctiles, nsplit; long long units; };
FewPlan few_plan(const b200_paged_cache* c, const b200_paged_batch* b, int G, int window, int sinks, int few_rows) {
  FewPlan f;
  const long long rows = few_rows < b->max_rows ? few_rows : b->max_rows, cols = rows * G;
  f.nt = cols <= 8 ? 1 : cols <= 16 ? 2 : 4;
  f.ctiles = (int)ceil_div64(cols, 8 * f.nt);
  f.units = (long long)b->sequences * c->kv_heads * f.ctiles;
  long long keys = (long long)b->table_width * c->page_tokens;
  if (window > 0 && (long long)window + sinks + rows < keys) keys = (long long)window + sinks + rows;
  const long long tiles = ceil_div64(keys, 16), slots = 148 * (f.nt == 1 ? 4 : f.nt == 2 ? 3 : 2);
  long long n = f.units ? slots / f.units : 1;
  if (n > tiles / 16) n = tiles / 16;
  f.nsplit = n < 1 ? 1 : n > 256 ? 256 : (int)n;
  return f;
}

template <int D, int FMT, int NT>
int launch_few(const AttnP& p, long long units, cudaStream_t st) {
  B200_TRY(launch_early(few_rows_kernel<D, FMT, NT>, dim3((unsigned)(units * p.nsplit)), dim3(FEW_THREADS), 0, st, p));
  if (p.nsplit > 1) B200_TRY(launch_early(join_kernel<D, NT>, dim3((unsigned)(units * NT)), dim3(128), 0, st, p));
  return B200_OK;
}
template <int D, int FMT>
int launch_few_nt(const AttnP& p, const FewPlan& f, cudaStream_t st) {
  if (f.nt == 1) return launch_few<D, FMT, 1>(p, f.units, st);
  if (f.nt == 2) return launch_few<D, FMT, 2>(p, f.units, st);
  return launch_few<D, FMT, 4>(p, f.units, st);
}

template <int FMT, int D>
int launch_append(AppendP& p, int max_rows, int q_ctas_rows, cudaStream_t st) {
  // few rows to a page: a warp each; else a block, which holds whole pages in registers
  const bool few = max_rows <= 4;
  const long long ctas = ceil_div64(p.page_tasks, few ? APPEND_THREADS / 32 : 1);
  p.page_ctas = (int)ctas;
  const dim3 grid((unsigned)(ctas + q_ctas_rows));
  if (few) return launch_early(append_kernel<FMT, D, 32, 1>, grid, dim3(APPEND_THREADS), 0, st, p);
  return launch_early(append_kernel<FMT, D, 256, D / 32>, grid, dim3(APPEND_THREADS), 0, st, p);
}

}  // namespace
}  // namespace paged
}  // namespace b200

using namespace b200;

extern "C" {

int b200_paged_append(const b200_paged_cache* cache, const b200_paged_batch* batch, const void* k_dev, int64_t k_ld, const void* v_dev, int64_t v_ld,
                      const void* q_dev, int64_t q_ld, void* q_out_dev, int64_t q_out_ld, int q_heads, const b200_rotary* rotary, void* stream) {
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
  DeviceGuard guard(cache->device);
  AppendP p;
  p.k_codes = static_cast<uint8_t*>(cache->k_dev); p.v_codes = static_cast<uint8_t*>(cache->v_dev); p.k_scale = cache->k_scale_dev; p.v_scale = cache->v_scale_dev;
  p.flags = cache->flags_dev; p.b = batch_of(batch);
  p.k = static_cast<const __nv_bfloat16*>(k_dev); p.v = static_cast<const __nv_bfloat16*>(v_dev); p.q = static_cast<const __nv_bfloat16*>(q_dev);
  p.q_out = static_cast<__nv_bfloat16*>(q_out_dev); p.k_ld = k_ld; p.v_ld = v_ld; p.q_ld = q_ld; p.q_out_ld = q_out_ld;
  p.turns = rotary ? rotary->turns_dev : nullptr; p.rot = rotary ? rotary->rot_dims : 0; p.halves = rotary ? rotary->pairing == B200_ROT_HALVES : 0;
  p.pages = cache->pages; p.P = cache->page_tokens; p.H = cache->kv_heads; p.Hq = q_dev ? q_heads : 0;
  const long long tasks = ((long long)batch->total_rows / p.P + 2ll * batch->sequences) * p.H * 2;
  if (tasks > (1ll << 30)) B200_FAIL(B200_ERR_SHAPE, "paged_append: %d rows of %d sequences with %d heads in one call", batch->total_rows, batch->sequences, p.H);
  p.page_tasks = (int)tasks;
  // a block's queries: one row where there are few (all heads at once), else eight rows, whose angles then serve several heads
  const int slots = APPEND_THREADS / (D / 16);
  p.q_rows = (long long)batch->total_rows * q_heads >= 148ll * 8 * slots ? 8 : 1;
  const int q_ctas = q_dev ? ceil_div(batch->total_rows, p.q_rows) : 0;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const bool i8 = cache->kv_dtype == B200_KV_INT8;
  int rc;
  if (D == 128) rc = i8 ? launch_append<INT8, 128>(p, batch->max_rows, q_ctas, st) : launch_append<E4M3, 128>(p, batch->max_rows, q_ctas, st);
  else rc = i8 ? launch_append<INT8, 64>(p, batch->max_rows, q_ctas, st) : launch_append<E4M3, 64>(p, batch->max_rows, q_ctas, st);
  B200_TRY(rc);
  return check_launch("paged_append");
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
  const dim3 grid((unsigned)ceil_div(batch->total_rows, READ_ROWS));
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
  const FewPlan f = few_plan(cache, batch, G, window, sinks, 0x7fffffff);
  return f.nsplit > 1 ? f.units * f.nsplit * 8 * f.nt * (cache->dim + 2) * (int64_t)sizeof(float) : 0;
}

int b200_paged_attention(const b200_paged_cache* cache, const b200_paged_batch* batch, const void* q_dev, int64_t q_ld, void* out_dev, int64_t out_ld, int q_heads,
                         float scale, int window, int sinks, void* work_dev, int64_t work_bytes, void* stream) {
  using namespace b200::paged;
  B200_TRY(check_cache(cache, "paged_attention"));
  B200_TRY(check_batch(cache, batch, "paged_attention"));
  const int D = cache->dim, H = cache->kv_heads;
  if (q_heads < H || q_heads % H || q_heads / H > 256) B200_FAIL(B200_ERR_SHAPE, "paged_attention: %d query heads on %d heads of the cache", q_heads, H);
  if (!(scale > 0.f && scale < INFINITY) || window < 0 || sinks < 0) B200_FAIL(B200_ERR_INVALID, "paged_attention: scale %g, window %d, %d first tokens", (double)scale, window, sinks);
  if (batch->total_rows == 0 || batch->max_rows == 0) return B200_OK;
  if (!rows_fit(q_dev, q_ld, q_heads, D) || !rows_fit(out_dev, out_ld, q_heads, D))
    B200_FAIL(B200_ERR_INVALID, "paged_attention: queries and results must begin on a 16-byte border, rows %lld and %lld elements apart", (long long)q_ld, (long long)out_ld);
  DeviceGuard guard(cache->device);
  AttnP p;
  p.k = static_cast<const uint8_t*>(cache->k_dev); p.v = static_cast<const uint8_t*>(cache->v_dev); p.k_scale = cache->k_scale_dev; p.v_scale = cache->v_scale_dev;
  p.flags = cache->flags_dev; p.b = batch_of(batch); p.q = static_cast<const __nv_bfloat16*>(q_dev); p.out = static_cast<__nv_bfloat16*>(out_dev);
  p.q_ld = q_ld; p.out_ld = out_ld; p.pages = cache->pages; p.P = cache->page_tokens; p.page_shift = shift_of(p.P); p.H = H; p.G = q_heads / H;
  p.window = window; p.sinks = sinks; p.scale2 = scale * LOG2E;
  p.from_rows = 0x7fffffff; p.q_tiles = 0;
  const FewPlan f = few_plan(cache, batch, p.G, window, sinks, p.from_rows);
  if (f.units * f.nsplit > 0x7fffffffll / 4) B200_FAIL(B200_ERR_SHAPE, "paged_attention: %d sequences of up to %d rows with %d heads in one call", batch->sequences, batch->max_rows, q_heads);
  p.nsplit = f.nsplit; p.ctiles = f.ctiles; p.part_o = p.part_ml = nullptr;
  if (f.nsplit > 1) {
    const long long cols = f.units * f.nsplit * 8 * f.nt;
    if (!work_dev || work_bytes < cols * (D + 2) * (long long)sizeof(float) || (reinterpret_cast<uintptr_t>(work_dev) & 15))
      B200_FAIL(B200_ERR_INVALID, "paged_attention: a workspace of %lld bytes, b200_paged_attention_bytes asks for %lld on a 16-byte border", (long long)work_bytes, cols * (D + 2) * 4ll);
    p.part_o = static_cast<float*>(work_dev);
    p.part_ml = p.part_o + cols * D;
  }
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const bool i8 = cache->kv_dtype == B200_KV_INT8;
  if (D == 128) B200_TRY((i8 ? launch_few_nt<128, INT8>(p, f, st) : launch_few_nt<128, E4M3>(p, f, st)));
  else B200_TRY((i8 ? launch_few_nt<64, INT8>(p, f, st) : launch_few_nt<64, E4M3>(p, f, st)));
  return check_launch("paged_attention");
}

}  // extern "C"
