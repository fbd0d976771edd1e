// Rows that are kept of a tree of drafted tokens, and the pages of a pool: who holds them, copies before a shared one is written, the move of what is in use to the front.
//
// All layers' caches take their pages from the same tables, so that whatever moves codes goes through up to 64 caches in one launch.
#include "paged.cuh"

namespace b200 {
namespace paged {

namespace {

using tcp::pdl_trigger;
using tcp::pdl_wait;

constexpr int MAX_CACHES = 64;               // of a launch
struct Layer { uint8_t *k, *v; float *k_scale, *v_scale; };
struct Layers { Layer of[MAX_CACHES]; };

// =========================================================================================================================
// kept rows
// =========================================================================================================================
struct KeepP {
  Layers layers;
  Batch b;
  const int32_t *kept, *counts;              // [rows]: a sequence's first counts[s] are the numbers of its kept rows, rising
  int32_t* flags;
  int n_layers, pages, P, H;
};
constexpr int KEEP_THREADS = 256;

// The least number of doublings with which a page's largest code reaches `top`.  Both sides are products of a code and a scale, so that equal scales never double.
template <int FMT>
__device__ __forceinline__ int doublings_for(double top, float s_old) {
  const double limit = (double)s_old * (double)code_max<FMT>();
  if (!(top > limit)) return 0;
  int power;
  const double part = frexp(top / limit, &power);
  return part == 0.5 ? power - 1 : power;
}
template <int FMT>
__device__ __forceinline__ float largest_code(const uint4& x) {
  const uint32_t w[4] = {ready<FMT>(x.x), ready<FMT>(x.y), ready<FMT>(x.z), ready<FMT>(x.w)};
  float top = 0.f;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 a = float2_of<FMT, 0>(w[i]), b = float2_of<FMT, 1>(w[i]);
    top = fmaxf(top, fmaxf(fmaxf(fabsf(a.x), fabsf(a.y)), fmaxf(fabsf(b.x), fabsf(b.y))));
  }
  return top;
}
// codes * s / by, rounded like a division (Markstein's correction, as in paged.cu), as codes again
template <int FMT>
__device__ __forceinline__ uint4 converted(const uint4& x, float s, float by) {
  const float div = by > 0.f ? by : 1.f, inv = 1.f / div;
  auto one = [&](float c) {
    const float v = c * s, q = v * inv;
    return fmaf(fmaf(-q, div, v), inv, q);
  };
  const uint32_t w[4] = {ready<FMT>(x.x), ready<FMT>(x.y), ready<FMT>(x.z), ready<FMT>(x.w)};
  uint32_t o[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 a = float2_of<FMT, 0>(w[i]), b = float2_of<FMT, 1>(w[i]);
    o[i] = codes4<FMT>(one(a.x), one(a.y), one(b.x), one(b.y));
  }
  return make_uint4(o[0], o[1], o[2], o[3]);
}
// The same in 64 bits.  Where rows give a page its scale, quotients of their codes are ratios of whole numbers, and halves among them are common: in 32 bits it would be chance which way those go.
template <int FMT>
__device__ __forceinline__ uint4 converted_far(const uint4& x, double s, double by) {
  const double inv = 1.0 / by;
  auto one = [&](float c) {
    const double v = (double)c * s, q = v * inv;
    return fma(fma(-q, by, v), inv, q);
  };
  const uint32_t w[4] = {ready<FMT>(x.x), ready<FMT>(x.y), ready<FMT>(x.z), ready<FMT>(x.w)};
  uint32_t o[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 a = float2_of<FMT, 0>(w[i]), b = float2_of<FMT, 1>(w[i]);
    double q[4] = {one(a.x), one(a.y), one(b.x), one(b.y)};
    if constexpr (FMT == INT8)
#pragma unroll
      for (int e = 0; e < 4; ++e) q[e] = rint(q[e]);
    o[i] = codes4<FMT>((float)q[0], (float)q[1], (float)q[2], (float)q[3]);
  }
  return make_uint4(o[0], o[1], o[2], o[3]);
}
// codes / 2^doublings; -1: they become 0
template <int FMT>
__device__ __forceinline__ uint4 halved(const uint4& x, int doublings) {
  if (doublings == 0) return x;
  if (doublings < 0) return make_uint4(0, 0, 0, 0);
  const float by = ldexpf(1.f, -doublings);
  const uint32_t w[4] = {ready<FMT>(x.x), ready<FMT>(x.y), ready<FMT>(x.z), ready<FMT>(x.w)};
  uint32_t o[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 a = float2_of<FMT, 0>(w[i]), b = float2_of<FMT, 1>(w[i]);
    o[i] = codes4<FMT>(a.x * by, a.y * by, b.x * by, b.y * by);
  }
  return make_uint4(o[0], o[1], o[2], o[3]);
}

// A warp per (cache, sequence, kv head, side) goes through the pages that kept rows move to, in rising order: row i comes from place a_i >= i, so that what is read has not been written yet.
// Bound: a chain of dependent reads a page (list, table, scale, rows), 12 us for 8 caches of 16 sequences that keep 3 to 8 rows each; the bytes would be done in 0.5.
template <int FMT, int D>
__global__ void __launch_bounds__(KEEP_THREADS) keep_kernel(const __grid_constant__ KeepP p) {
  pdl_trigger();
  pdl_wait();
  if (blockIdx.x == gridDim.x - 1) { record_sequences(p.b, p.P, p.flags, KEEP_THREADS); return; }
  constexpr int CHUNKS = D / 16, RPS = 32 / CHUNKS;      // 16-byte pieces of a row; rows of a warp's sweep
  const int lane = threadIdx.x & 31;
  const long long task = (long long)blockIdx.x * (KEEP_THREADS / 32) + (threadIdx.x >> 5);
  if (task >= (long long)p.n_layers * p.b.S * p.H * 2) return;
  const int side = (int)(task & 1), h = (int)((task >> 1) % p.H), s = (int)((task >> 1) / p.H % p.b.S), layer = (int)((task >> 1) / p.H / p.b.S);
  const Seq q = sequence(p.b, s, p.P);
  if (!q.ok || q.n == 0) return;
  const int count = p.counts[s];
  const int32_t* kept = p.kept + q.r0;
  int moved = count;                                     // the first row that does not lie where it belongs
  bool bad = count < 0 || count > q.n;
  for (int i = lane; !bad && i - lane < count; i += 32) {
    if (i >= count) break;
    const int a = kept[i];
    bad = a < 0 || a >= q.n || (i > 0 && a <= kept[i - 1]);
    if (a != i) moved = min(moved, i);
  }
  if (__any_sync(0xffffffffu, bad)) {
    if (lane == 0) atomicOr(p.flags, B200_PAGED_BAD_BATCH);
    return;
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) moved = min(moved, __shfl_xor_sync(0xffffffffu, moved, o));
  if (moved >= count) return;
  const Layer& to = p.layers.of[layer];
  uint8_t* const codes = side ? to.v : to.k;
  float* const scales = side ? to.v_scale : to.k_scale;
  const int32_t* table = p.b.table + s * p.b.table_ld;
  const int c = lane % CHUNKS, row0 = lane / CHUNKS;
  auto at = [&](int page, int slot) { return codes + (((long long)page * p.H + h) * p.P + slot) * D + 16 * c; };
  auto page_at = [&](int block) {
    const int page = table[block];
    if (page >= 0 && page < p.pages) return page;
    if (lane == 0) atomicOr(p.flags, B200_PAGED_BAD_PAGE);
    return -1;
  };
  for (int block = (q.before + moved) / p.P; block <= (q.before + count - 1) / p.P; ++block) {
    const int page = page_at(block);
    if (page < 0) continue;                              // its rows are left out
    const int first = block * p.P, i0 = max(first - q.before, 0), i1 = (int)min((long long)first + p.P - q.before, (long long)count), older = max(q.before - first, 0);
    // the largest value that comes from another page
    double top = 0.0;
    bool far = false, near = false;
    for (int i = i0 + row0; i - row0 < i1; i += RPS) {
      if (i >= i1) continue;
      const int from = q.before + kept[i], b = from / p.P;
      if (b == block) { near = true; continue; }
      const int source = table[b];
      far = true;
      if (source < 0 || source >= p.pages) { atomicOr(p.flags, B200_PAGED_BAD_PAGE); continue; }
      top = fmax(top, (double)largest_code<FMT>(*reinterpret_cast<const uint4*>(at(source, from - b * p.P))) * (double)scales[(long long)source * p.H + h]);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) top = fmax(top, __shfl_xor_sync(0xffffffffu, top, o));
    far = __any_sync(0xffffffffu, far);
    const bool resident = older > 0 || __any_sync(0xffffffffu, near);
    const float s_old = scales[(long long)page * p.H + h];
    float sc = s_old;
    double own = 0.0;                                    // the scale that the rows themselves give the page
    int doublings = 0;
    if (far) {
      if (resident && s_old > 0.f) {
        doublings = doublings_for<FMT>(top, s_old);
        sc = ldexpf(s_old, doublings);
      } else {
        own = top > 0.0 ? fmax(top / (double)code_max<FMT>(), (double)SCALE_MIN) : 0.0;
        sc = (float)own;
        doublings = -1;
      }
    }
    __syncwarp();                                        // all lanes have read the scale
    if (far && lane == 0) scales[(long long)page * p.H + h] = sc;
    if (doublings != 0)
      for (int slot = row0; slot < older; slot += RPS) {
        uint4* x = reinterpret_cast<uint4*>(at(page, slot));
        *x = halved<FMT>(*x, doublings);
      }
    for (int i = i0 + row0; i - row0 < i1; i += RPS) {
      uint4 x = make_uint4(0, 0, 0, 0);
      bool put = false;
      if (i < i1) {
        const int from = q.before + kept[i], b = from / p.P;
        if (b == block) {
          put = kept[i] != i || doublings != 0;
          if (put) x = halved<FMT>(*reinterpret_cast<const uint4*>(at(page, from - first)), doublings);
        } else {
          const int source = table[b];
          put = source >= 0 && source < p.pages;
          if (put) {
            const uint4 was = *reinterpret_cast<const uint4*>(at(source, from - b * p.P));
            const float s_from = scales[(long long)source * p.H + h];
            x = own > 0.0 ? converted_far<FMT>(was, (double)s_from, own) : converted<FMT>(was, s_from, sc);
          }
        }
      }
      __syncwarp();                                      // rows of a sweep are read before one is written
      if (put) *reinterpret_cast<uint4*>(at(page, q.before + i - first)) = x;
      __syncwarp();
    }
  }
}

// =========================================================================================================================
// pages
// =========================================================================================================================
struct PoolP {
  int32_t *table, *lengths, *held, *refs, *flags;
  long long table_ld;
  int S, W, pages, P;
};
// What sequence s holds, and how many pages its tokens are in; -1 where that does not fit together.
__device__ __forceinline__ int pages_of(const PoolP& p, int s, int held) {
  const int n = p.lengths[s];
  if (n < 0 || held < 0 || held > p.W || n > (long long)held * p.P) return -1;
  return (n + p.P - 1) / p.P;
}

// ---- one block's sums ----
constexpr int ONE = 1024;                                // threads of the blocks that look at all pages
// Exclusive sums of the block's values in the order of its threads; *all: their total.
__device__ __forceinline__ int block_sums(int v, int* all) {
  __shared__ int sums[ONE / 32];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int in = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int x = __shfl_up_sync(0xffffffffu, in, o);
    if (lane >= o) in += x;
  }
  __syncthreads();                                       // the sums of the call in front have been read
  if (lane == 31) sums[warp] = in;
  __syncthreads();
  int before = 0, total = 0;
#pragma unroll 8
  for (int w = 0; w < ONE / 32; ++w) {
    if (w < warp) before += sums[w];
    total += sums[w];
  }
  *all = total;
  return before + in - v;
}

// ---- sequences change places ----
struct RearrangeP {
  PoolP o;
  const int32_t* source;
  int32_t *old_table, *old_pages, *old_lengths;          // [S][W], [S], [S]
};
// a source that names no sequence: the sequence stays what it is
__device__ __forceinline__ int source_of(const RearrangeP& p, int i) {
  const int s = p.source[i];
  return s >= -1 && s < p.o.S ? s : i;
}
// A block per sequence as it was: its pages get as many references as there are sequences that it becomes, and what it holds behind its tokens is given back; all of it, where its length is not one that its pages
// can have, as nobody could give them back later.
__global__ void __launch_bounds__(256) rearrange_count_kernel(const RearrangeP p) {
  pdl_trigger();
  pdl_wait();
  __shared__ int becomes;
  const int s = (int)blockIdx.x;
  if (threadIdx.x == 0) becomes = 0;
  __syncthreads();
  int mine = 0;
  for (int i = threadIdx.x; i < p.o.S; i += blockDim.x) {
    mine += source_of(p, i) == s;
    if (s == 0 && (p.source[i] < -1 || p.source[i] >= p.o.S)) atomicOr(p.o.flags, B200_PAGED_BAD_BATCH);
  }
  if (mine) atomicAdd(&becomes, mine);
  __syncthreads();
  const int held = min(p.o.held[s], p.o.W), fits = pages_of(p.o, s, p.o.held[s]), n = max(fits, 0);       // one whose length and pages do not fit together counts as empty
  if (threadIdx.x == 0) {
    if (fits < 0) atomicOr(p.o.flags, B200_PAGED_BAD_BATCH);
    p.old_pages[s] = n; p.old_lengths[s] = fits < 0 ? 0 : p.o.lengths[s];
  }
  for (int b = threadIdx.x; b < held; b += blockDim.x) {
    const int page = p.o.table[s * p.o.table_ld + b];
    if (b < n) p.old_table[(long long)s * p.o.W + b] = page;
    if (page < 0 || page >= p.o.pages) { atomicOr(p.o.flags, B200_PAGED_BAD_PAGE); continue; }
    const int more = (b < n ? becomes : 0) - 1;
    if (more) atomicAdd(p.o.refs + page, more);
  }
}
__global__ void __launch_bounds__(256) rearrange_take_kernel(const RearrangeP p) {
  pdl_trigger();
  pdl_wait();
  const int i = (int)blockIdx.x, s = source_of(p, i), n = s < 0 ? 0 : p.old_pages[s];
  if (threadIdx.x == 0) { p.o.held[i] = n; p.o.lengths[i] = s < 0 ? 0 : p.old_lengths[s]; }
  for (int b = threadIdx.x; b < p.o.W; b += blockDim.x) p.o.table[i * p.o.table_ld + b] = b < n ? p.old_table[(long long)s * p.o.W + b] : -1;
}

// Small tables by one block, through shared memory (64 sequences of 24 pages: 5.8 us, as two launches 9.3).
constexpr int SMALL_TABLE = 8192, SMALL_SEQUENCES = 1024;
__global__ void __launch_bounds__(ONE) rearrange_small_kernel(const RearrangeP p) {
  pdl_trigger();
  pdl_wait();
  __shared__ int32_t old[SMALL_TABLE];
  __shared__ int becomes[SMALL_SEQUENCES], tokens[SMALL_SEQUENCES], n_pages[SMALL_SEQUENCES];
  const int s = threadIdx.x, S = p.o.S, W = p.o.W;       // S <= ONE: a thread a sequence
  int from = -1, held = 0;
  becomes[s] = 0;
  __syncthreads();
  if (s < S) {
    from = source_of(p, s);
    held = p.o.held[s];
    const int n = pages_of(p.o, s, held);
    if (p.source[s] < -1 || p.source[s] >= S || n < 0) atomicOr(p.o.flags, B200_PAGED_BAD_BATCH);
    if (from >= 0) atomicAdd(becomes + from, 1);
    tokens[s] = n < 0 ? 0 : p.o.lengths[s];
    n_pages[s] = max(n, 0);                              // one whose length and pages do not fit together counts as empty
  }
  __syncthreads();
  for (int i = threadIdx.x; i < S * W; i += ONE) {
    const int x = i / W, b = i - x * W, n = n_pages[x];
    if (b >= p.o.held[x]) continue;
    const int page = p.o.table[x * p.o.table_ld + b];
    old[i] = page;
    if (page < 0 || page >= p.o.pages) { atomicOr(p.o.flags, B200_PAGED_BAD_PAGE); continue; }
    const int more = (b < n ? becomes[x] : 0) - 1;
    if (more) atomicAdd(p.o.refs + page, more);
  }
  __syncthreads();
  if (s < S) {
    p.o.held[s] = from < 0 ? 0 : n_pages[from];
    p.o.lengths[s] = from < 0 ? 0 : tokens[from];
    becomes[s] = from;
  }
  __syncthreads();
  for (int i = threadIdx.x; i < S * W; i += ONE) {
    const int x = i / W, b = i - x * W, y = becomes[x];
    p.o.table[x * p.o.table_ld + b] = y >= 0 && b < n_pages[y] ? old[y * W + b] : -1;
  }
}

// ---- pages for tokens to come ----
constexpr int MAX_SEQUENCES = 4096;                      // of a pool
struct ReserveP {
  PoolP o;
  const int32_t* add;
  int32_t* free_pages;                                   // [pages]: the lowest free ones that are needed
  int2* moves;                                           // [S]: pages to copy, and where to
  int32_t* n_moves;
};
// One block, as pages go out in order; bound by its few rounds of dependent reads and sums (6 us for 64 sequences).  Who needs what: sequence s wants its pages up to lengths + add tokens, and one more where the page that its next token goes to is shared.  Of the sequences that share one, all but the last get a copy.
__global__ void __launch_bounds__(ONE) reserve_kernel(const ReserveP p) {
  pdl_trigger();
  pdl_wait();
  constexpr int COPIED = -2, LEFT_OUT = -3;
  __shared__ int begun[MAX_SEQUENCES], from[MAX_SEQUENCES + 1];      // the shared page that a sequence goes on in, -1: none; its first place among all pages that are needed
  const int tid = threadIdx.x, S = p.o.S, P = p.o.P;
  auto want = [&](int s, int held) {                     // pages that the sequence is to hold; -1: left out
    const int n = p.o.lengths[s], add = p.add[s];
    if (pages_of(p.o, s, held) < 0 || add < 0 || (long long)n + add > (long long)p.o.W * P) return -1;
    return add ? max(held, (int)(((long long)n + add + P - 1) / P)) : held;
  };
  int refs[4];                               // of the first pages, on their way beside the sequences
#pragma unroll
  for (int k = 0; k < 4; ++k) refs[k] = 4 * tid + k < p.o.pages ? p.o.refs[4 * tid + k] : 1;
  for (int s = tid; s < S; s += ONE) {
    const int held = p.o.held[s], n = p.o.lengths[s], next = pages_of(p.o, s, held);      // next: its first page without tokens
    int page = -1;
    bool out = want(s, held) < 0;
    if (!out && p.add[s] > 0) {
      const int32_t* table = p.o.table + s * p.o.table_ld;
      const int spare = next < held ? table[next] : -1;
      if (n % P) {
        page = table[n / P];
        if (page < 0 || page >= p.o.pages) { atomicOr(p.o.flags, B200_PAGED_BAD_PAGE); page = -1; }
        else if (p.o.refs[page] <= 1) page = -1;
      }
      // a page that others have tokens in: the sequence was made shorter and not rearranged
      out = spare >= 0 && spare < p.o.pages && p.o.refs[spare] > 1;
    }
    if (out) atomicOr(p.o.flags, B200_PAGED_BAD_BATCH);
    begun[s] = out ? LEFT_OUT : page;
  }
  __syncthreads();
  int needed = 0, copied = 0;
  for (int s0 = 0; s0 < S; s0 += ONE) {
    const int s = s0 + tid;
    int need = 0, copy = 0;
    if (s < S) {
      const int held = p.o.held[s], page = begun[s];
      need = page == LEFT_OUT ? 0 : want(s, held) - held;
      if (page >= 0) {
        int rank = 0;
        for (int i = 0; i < s; ++i) rank += begun[i] == page;
        copy = p.o.refs[page] - rank > 1;
      }
    }
    int all, copies;
    const int at = block_sums(need + copy, &all), place = block_sums(copy, &copies);
    if (s < S) from[s] = needed + at;
    __syncthreads();                                     // all ranks of these sequences are known
    if (copy) p.moves[copied + place] = make_int2(begun[s], s);           // the page that it becomes is not known yet
    needed += all; copied += copies;
  }
  if (tid == 0) from[S] = needed;
  // the lowest free pages
  int found = 0;
  for (int p0 = 0; p0 < p.o.pages && found < needed; p0 += 4 * ONE) {
    int mine = 0, all;
    const int first = p0 + 4 * tid;
    bool is[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) mine += is[k] = p0 == 0 ? refs[k] == 0 : first + k < p.o.pages && p.o.refs[first + k] == 0;
    int at = found + block_sums(mine, &all);
#pragma unroll
    for (int k = 0; k < 4; ++k)
      if (is[k]) { if (at < needed) p.free_pages[at] = first + k; ++at; }
    found += all;
  }
  __syncthreads();
  if (found < needed) {                                  // nobody gets anything
    if (tid == 0) { atomicOr(p.o.flags, B200_PAGED_NO_PAGES); *p.n_moves = 0; }
    return;
  }
  if (tid == 0) *p.n_moves = copied;
  for (int i = tid; i < copied; i += ONE) {              // a copy is its sequence's first page
    const int2 x = p.moves[i];
    const int to = p.free_pages[from[x.y]];
    p.o.table[x.y * p.o.table_ld + p.o.lengths[x.y] / P] = to;
    p.o.refs[to] = 1;
    atomicSub(p.o.refs + x.x, 1);
    p.moves[i] = make_int2(x.x, to);
    begun[x.y] = COPIED;
  }
  __syncthreads();
  for (int i = tid; i < needed; i += ONE) {
    int lo = 0, hi = S;                                  // the sequence that place i belongs to
    while (hi - lo > 1) {
      const int mid = (lo + hi) / 2;
      if (from[mid] <= i) lo = mid; else hi = mid;
    }
    const int b = i - from[lo] - (begun[lo] == COPIED);
    if (b < 0) continue;
    const int page = p.free_pages[i];
    p.o.table[lo * p.o.table_ld + p.o.held[lo] + b] = page;
    p.o.refs[page] = 1;
  }
  __syncthreads();
  for (int s = tid; s < S; s += ONE) p.o.held[s] += from[s + 1] - from[s] - (begun[s] == COPIED);
}

// ---- what is in use to the front ----
struct CompactP {
  PoolP o;
  int32_t *holes, *now;                                  // [pages]: free pages below the number in use; what a page becomes
  int2* moves;                                           // [pages / 2]
  int32_t* n_moves;
  int renumber;                                          // the tables, too: they are small
};
__device__ __forceinline__ void renumber(const CompactP& p, int s, int b) {
  if (b >= p.o.held[s]) return;
  int32_t* at = p.o.table + s * p.o.table_ld + b;
  const int page = *at;
  if (page >= 0 && page < p.o.pages) *at = p.now[page];
  else atomicOr(p.o.flags, B200_PAGED_BAD_PAGE);
}
__global__ void __launch_bounds__(ONE) compact_kernel(const CompactP p) {
  pdl_trigger();
  pdl_wait();
  const int tid = threadIdx.x, n = p.o.pages;
  int used = 0;
  for (int i = tid; i < n; i += ONE) used += p.o.refs[i] > 0;
  block_sums(used, &used);
  int below = 0, above = 0;
  for (int p0 = 0; p0 < n; p0 += 4 * ONE) {
    int hole = 0, high = 0, holes, highs;
    const int first = p0 + 4 * tid;
    bool in[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const int i = first + k;
      in[k] = i < n && p.o.refs[i] > 0;
      hole += i < used && !in[k];
      high += i >= used && in[k];
    }
    int at_hole = below + block_sums(hole, &holes), at_high = above + block_sums(high, &highs);
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const int i = first + k;
      if (i >= n) break;
      p.now[i] = i;
      if (i < used && !in[k]) p.holes[at_hole++] = i;
      if (i >= used && in[k]) p.moves[at_high++] = make_int2(i, -1);
    }
    below += holes; above += highs;
  }
  __syncthreads();
  for (int i = tid; i < above; i += ONE) {
    const int src = p.moves[i].x, dst = p.holes[i];
    p.moves[i] = make_int2(src, dst);
    p.now[src] = dst;
    p.o.refs[dst] = p.o.refs[src];
    p.o.refs[src] = 0;
  }
  if (tid == 0) *p.n_moves = above;
  if (!p.renumber) return;
  __syncthreads();
  for (int i = tid; i < p.o.S * p.o.W; i += ONE) {
    const int x = i / p.o.W;
    renumber(p, x, i - x * p.o.W);
  }
}
__global__ void __launch_bounds__(256) renumber_kernel(const CompactP p) {
  pdl_trigger();
  pdl_wait();
  for (int b = threadIdx.x; b < p.o.W; b += blockDim.x) renumber(p, (int)blockIdx.x, b);
}

// ---- copies ----
struct CopyP {
  Layers layers;
  const int2* moves;
  const int32_t* n_moves;
  int most, n_layers, H, pages;
  long long bytes;                                       // of a page's codes, one side
};
constexpr int COPY_THREADS = 256, COPY_DEEP = 4, COPY_CHUNK = COPY_THREADS * 16 * COPY_DEEP, COPY_BLOCKS = 148 * 64;
// A page's codes are one run of memory per side: a block has a cache's side and takes 16 KB of a page at a time, four pieces in flight a thread; nobody reads them soon.  Bounds: bytes.
__global__ void __launch_bounds__(COPY_THREADS) copy_kernel(const __grid_constant__ CopyP p) {
  pdl_trigger();
  pdl_wait();
  const uint32_t n = (uint32_t)min(max(*p.n_moves, 0), p.most), chunks = (uint32_t)((p.bytes + COPY_CHUNK - 1) / COPY_CHUNK), tasks = n * chunks;
  const int side = blockIdx.y & 1;
  const Layer& l = p.layers.of[blockIdx.y >> 1];
  uint8_t* const codes = side ? l.v : l.k;
  float* const scales = side ? l.v_scale : l.k_scale;
  for (uint32_t t = blockIdx.x; t < tasks; t += gridDim.x) {
    const uint32_t i = t / chunks, chunk = t - i * chunks;
    const int2 x = p.moves[i];
    if (x.x < 0 || x.x >= p.pages || x.y < 0 || x.y >= p.pages) continue;
    const long long at = (long long)chunk * COPY_CHUNK + 16 * threadIdx.x;
    const uint8_t* src = codes + x.x * p.bytes + at;
    uint8_t* dst = codes + x.y * p.bytes + at;
    uint4 v[COPY_DEEP];
#pragma unroll
    for (int k = 0; k < COPY_DEEP; ++k)
      if (at + k * COPY_THREADS * 16 < p.bytes) v[k] = __ldcs(reinterpret_cast<const uint4*>(src + k * COPY_THREADS * 16));
#pragma unroll
    for (int k = 0; k < COPY_DEEP; ++k)
      if (at + k * COPY_THREADS * 16 < p.bytes) __stcs(reinterpret_cast<uint4*>(dst + k * COPY_THREADS * 16), v[k]);
    if (chunk == 0)
      for (int h = threadIdx.x; h < p.H; h += COPY_THREADS) scales[(long long)x.y * p.H + h] = scales[(long long)x.x * p.H + h];
  }
}

// =========================================================================================================================
// host
// =========================================================================================================================
int check_caches(const b200_paged_cache* caches, int n, const char* what) {
  if (!caches || n < 1) B200_FAIL(B200_ERR_INVALID, "%s: no caches", what);
  for (int i = 0; i < n; ++i) {
    B200_TRY(checked_cache(caches + i, what));
    const b200_paged_cache &a = caches[0], &c = caches[i];
    if (a.pages != c.pages || a.page_tokens != c.page_tokens || a.kv_heads != c.kv_heads || a.dim != c.dim || a.kv_dtype != c.kv_dtype || a.device != c.device)
      B200_FAIL(B200_ERR_SHAPE, "%s: cache %d is not like the first", what, i);
  }
  return B200_OK;
}
Layers layers_of(const b200_paged_cache* caches, int n) {
  Layers x;
  memset(&x, 0, sizeof(x));
  for (int i = 0; i < n; ++i) x.of[i] = {static_cast<uint8_t*>(caches[i].k_dev), static_cast<uint8_t*>(caches[i].v_dev), caches[i].k_scale_dev, caches[i].v_scale_dev};
  return x;
}
int check_pool(const b200_page_pool* o, const char* what) {
  if (!o || !o->table_dev || !o->lengths_dev || !o->held_dev || !o->refs_dev || !o->flags_dev) B200_FAIL(B200_ERR_INVALID, "%s: null pointer in the pool", what);
  if (o->sequences < 1 || o->sequences > MAX_SEQUENCES || o->table_width < 1 || o->table_ld < o->table_width || o->pages < 1 || o->pages > 0x7fff0000 || (long long)o->sequences * o->table_width > 0x7fff0000 ||
      (o->page_tokens != 16 && o->page_tokens != 32 && o->page_tokens != 64 && o->page_tokens != 128) || (long long)o->table_width * o->page_tokens > 0x7fffff00ll)
    B200_FAIL(B200_ERR_SHAPE, "%s: %d sequences (at most %d) with tables of %d pages, %d pages of %d tokens", what, o->sequences, MAX_SEQUENCES, o->table_width, o->pages, o->page_tokens);
  return B200_OK;
}
int check_pool_caches(const b200_page_pool* o, const b200_paged_cache* caches, int n, const char* what) {
  if (n == 0) return B200_OK;
  B200_TRY(check_caches(caches, n, what));
  if (caches->pages != o->pages || caches->page_tokens != o->page_tokens || caches->device != o->device) B200_FAIL(B200_ERR_SHAPE, "%s: the caches' pages are not the pool's", what);
  return B200_OK;
}
PoolP pool_of(const b200_page_pool* o) {
  PoolP p;
  p.table = o->table_dev; p.lengths = o->lengths_dev; p.held = o->held_dev; p.refs = o->refs_dev; p.flags = o->flags_dev; p.table_ld = o->table_ld;
  p.S = o->sequences; p.W = o->table_width; p.pages = o->pages; p.P = o->page_tokens;
  return p;
}
int copy_pages(const b200_paged_cache* caches, int n, const int2* moves, const int32_t* n_moves, int most, cudaStream_t st) {
  for (int first = 0; first < n && most > 0; first += MAX_CACHES) {
    const b200_paged_cache& c = caches[first];
    CopyP p;
    p.n_layers = n - first < MAX_CACHES ? n - first : MAX_CACHES;
    p.layers = layers_of(caches + first, p.n_layers);
    p.moves = moves; p.n_moves = n_moves; p.most = most; p.H = c.kv_heads; p.pages = c.pages;
    p.bytes = (long long)c.kv_heads * c.page_tokens * c.dim;
    const long long tasks = (long long)most * ceil_div64(p.bytes, COPY_CHUNK), blocks = ceil_div(COPY_BLOCKS, 2 * p.n_layers);
    B200_TRY(launch_early(copy_kernel, dim3((unsigned)(tasks < blocks ? tasks : blocks), 2 * p.n_layers), dim3(COPY_THREADS), 0, st, p));
  }
  return B200_OK;
}
// a call's workspace: pieces on 16-byte borders
struct Pieces {
  uint8_t* at;
  int64_t used = 0;
  template <typename T>
  T* take(int64_t n) {
    T* x = reinterpret_cast<T*>(at + used);
    used += (n * (int64_t)sizeof(T) + 15) / 16 * 16;
    return x;
  }
};
int check_work(const char* what, const void* work, int64_t bytes, int64_t need) {
  if (!work || bytes < need || (reinterpret_cast<uintptr_t>(work) & 15)) B200_FAIL(B200_ERR_INVALID, "%s: a workspace of %lld bytes; b200_page_pool_bytes asks for %lld, on a 16-byte border", what, (long long)bytes, (long long)need);
  return B200_OK;
}
int64_t bytes_of(const b200_page_pool* o) {
  const int64_t S = o->sequences, rearrange = S * o->table_width * 4 + S * 8, reserve = (int64_t)o->pages * 4 + S * 8, compact = (int64_t)o->pages * 12;
  const int64_t most = rearrange > reserve ? rearrange : reserve;
  return (most > compact ? most : compact) + 128;          // and the pieces' borders
}

}  // namespace
}  // namespace paged
}  // namespace b200

using namespace b200;

extern "C" {

int b200_paged_keep(const b200_paged_cache* caches, int n_caches, const b200_paged_batch* batch, const int32_t* kept_dev, const int32_t* counts_dev, void* stream) {
  using namespace b200::paged;
  B200_TRY(check_caches(caches, n_caches, "paged_keep"));
  B200_TRY(checked(caches, batch, "paged_keep"));
  if (batch->total_rows == 0 || batch->max_rows == 0) return B200_OK;
  if (!kept_dev || !counts_dev) B200_FAIL(B200_ERR_INVALID, "paged_keep: null pointer");
  if ((long long)batch->sequences * caches->kv_heads * 2 * MAX_CACHES > (1ll << 33)) B200_FAIL(B200_ERR_SHAPE, "paged_keep: %d sequences with %d heads in one call", batch->sequences, caches->kv_heads);
  DeviceGuard guard(caches->device);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const bool i8 = caches->kv_dtype == B200_KV_INT8;
  for (int first = 0; first < n_caches; first += MAX_CACHES) {
    KeepP p;
    p.n_layers = n_caches - first < MAX_CACHES ? n_caches - first : MAX_CACHES;
    p.layers = layers_of(caches + first, p.n_layers);
    p.b.table = batch->table_dev; p.b.before = batch->before_dev; p.b.rows = batch->rows_dev; p.b.table_ld = batch->table_ld;
    p.b.S = batch->sequences; p.b.T = batch->total_rows; p.b.width = batch->table_width; p.b.max_rows = batch->max_rows;
    p.kept = kept_dev; p.counts = counts_dev; p.flags = caches->flags_dev; p.pages = caches->pages; p.P = caches->page_tokens; p.H = caches->kv_heads;
    const dim3 grid((unsigned)ceil_div64((long long)p.n_layers * p.b.S * p.H * 2, KEEP_THREADS / 32) + 1);       // the last one looks at the sequences
    if (caches->dim == 128) B200_TRY((i8 ? launch_early(keep_kernel<INT8, 128>, grid, dim3(KEEP_THREADS), 0, st, p) : launch_early(keep_kernel<E4M3, 128>, grid, dim3(KEEP_THREADS), 0, st, p)));
    else B200_TRY((i8 ? launch_early(keep_kernel<INT8, 64>, grid, dim3(KEEP_THREADS), 0, st, p) : launch_early(keep_kernel<E4M3, 64>, grid, dim3(KEEP_THREADS), 0, st, p)));
  }
  return check_launch("paged_keep");
}

int64_t b200_page_pool_bytes(const b200_page_pool* pool) { return pool && pool->sequences > 0 && pool->table_width > 0 && pool->pages > 0 ? b200::paged::bytes_of(pool) : 0; }

int b200_page_pool_rearrange(const b200_page_pool* pool, const int32_t* source_dev, void* work_dev, int64_t work_bytes, void* stream) {
  using namespace b200::paged;
  B200_TRY(check_pool(pool, "page_pool_rearrange"));
  if (!source_dev) B200_FAIL(B200_ERR_INVALID, "page_pool_rearrange: null pointer");
  B200_TRY(check_work("page_pool_rearrange", work_dev, work_bytes, bytes_of(pool)));
  DeviceGuard guard(pool->device);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  Pieces w{static_cast<uint8_t*>(work_dev)};
  RearrangeP p;
  p.o = pool_of(pool); p.source = source_dev;
  p.old_table = w.take<int32_t>((int64_t)p.o.S * p.o.W); p.old_pages = w.take<int32_t>(p.o.S); p.old_lengths = w.take<int32_t>(p.o.S);
  if (p.o.S <= SMALL_SEQUENCES && (long long)p.o.S * p.o.W <= SMALL_TABLE) {
    EARLY_LAUNCH(rearrange_small_kernel, 1, ONE, 0, st, p);
    return check_launch("page_pool_rearrange");
  }
  EARLY_LAUNCH(rearrange_count_kernel, p.o.S, 256, 0, st, p);
  EARLY_LAUNCH(rearrange_take_kernel, p.o.S, 256, 0, st, p);
  return check_launch("page_pool_rearrange");
}

int b200_page_pool_reserve(const b200_page_pool* pool, const b200_paged_cache* caches, int n_caches, const int32_t* add_dev, void* work_dev, int64_t work_bytes, void* stream) {
  using namespace b200::paged;
  B200_TRY(check_pool(pool, "page_pool_reserve"));
  B200_TRY(check_pool_caches(pool, caches, n_caches, "page_pool_reserve"));
  if (!add_dev) B200_FAIL(B200_ERR_INVALID, "page_pool_reserve: null pointer");
  B200_TRY(check_work("page_pool_reserve", work_dev, work_bytes, bytes_of(pool)));
  DeviceGuard guard(pool->device);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  Pieces w{static_cast<uint8_t*>(work_dev)};
  ReserveP p;
  p.o = pool_of(pool); p.add = add_dev;
  p.free_pages = w.take<int32_t>(p.o.pages); p.moves = w.take<int2>(p.o.S); p.n_moves = w.take<int32_t>(1);
  EARLY_LAUNCH(reserve_kernel, 1, ONE, 0, st, p);
  B200_TRY(copy_pages(caches, n_caches, p.moves, p.n_moves, p.o.S, st));
  return check_launch("page_pool_reserve");
}

int b200_page_pool_compact(const b200_page_pool* pool, const b200_paged_cache* caches, int n_caches, void* work_dev, int64_t work_bytes, void* stream) {
  using namespace b200::paged;
  B200_TRY(check_pool(pool, "page_pool_compact"));
  B200_TRY(check_pool_caches(pool, caches, n_caches, "page_pool_compact"));
  B200_TRY(check_work("page_pool_compact", work_dev, work_bytes, bytes_of(pool)));
  DeviceGuard guard(pool->device);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  Pieces w{static_cast<uint8_t*>(work_dev)};
  CompactP p;
  p.o = pool_of(pool);
  p.holes = w.take<int32_t>(p.o.pages); p.now = w.take<int32_t>(p.o.pages); p.moves = w.take<int2>(p.o.pages / 2 + 1); p.n_moves = w.take<int32_t>(1);
  p.renumber = (long long)p.o.S * p.o.W <= SMALL_TABLE;
  EARLY_LAUNCH(compact_kernel, 1, ONE, 0, st, p);
  if (!p.renumber) EARLY_LAUNCH(renumber_kernel, p.o.S, 256, 0, st, p);
  B200_TRY(copy_pages(caches, n_caches, p.moves, p.n_moves, p.o.pages / 2, st));
  return check_launch("page_pool_compact");
}

}  // extern "C"
