// Attention of rows (one query token each) over the paged f16 KV cache, where the rows of a group share their first pages: decode
// batches behind one prompt, or the tokens of a prompt (a group whose rows share all pages and differ in length).
//
// Three kernels: attn_tile_kernel works on the shared pages, every K and V read once for 256 rows of (token, head) and multiplied by
// the 5th-generation tensor cores; attn_own_kernel reads the pages that a row has to itself and adds what the first found;
// attn_join_kernel adds up what several CTAs found of a row.  Sums travel as (m, l = sum of 2^(x - m), sum of 2^(x - m) v), x a score in
// the log2 domain: two of them add up after scaling by 2^(m - max).
#include <cuda_bf16.h>
#include <math.h>

#include "attn_shared.h"
#include "attn_tc.cuh"

namespace {

using namespace tc;

constexpr int kHD = 128, kPage = 16;
constexpr int kThreads = kOwnWarps * 32, kDepth = 2, kRing = kDepth * kOwnWarps;  // pages of a warp on their way
constexpr uint32_t kSlotBytes = 2 * kPage * kHD * 2;
constexpr int kHDP = kHD + 4;  // row stride of the warps' sums in shared memory: no bank conflicts
constexpr size_t kOwnSmem = kRing * kSlotBytes + 1024;
constexpr float kLog2e = 1.4426950408889634f;
// The largest weight of a row is 2^kHigh and more: the smallest that a f16 number holds at full precision is then 2^-21 of it.
constexpr float kHigh = 7.f;

// K and V of one (page, kv head): 32 rows as two halves of 64 dims, 128-byte swizzled; nobody else reads it
__device__ __forceinline__ void page_g2s(uint32_t dst, const CUtensorMap* map, int row, uint32_t bar) {
  uint64_t policy;
  asm("createpolicy.fractional.L2::evict_first.b64 %0;\n" : "=l"(policy));
  asm volatile("cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes.L2::cache_hint [%0], [%1, {%2, %3, %4}], [%5], %6;\n" ::"r"(dst), "l"(map),
               "r"(0), "r"(row), "r"(0), "r"(bar), "l"(policy)
               : "memory");
}
__device__ __forceinline__ void ldsm4(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];\n" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void ldsm4_t(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];\n" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ uint32_t transpose8x8(uint32_t a) {
  uint32_t d;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;\n" : "=r"(d) : "r"(a));
  return d;
}
__device__ __forceinline__ void mma16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
               : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
               : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ float rcp(float x) {
  float y;
  asm("rcp.approx.ftz.f32 %0, %1;\n" : "=f"(y) : "f"(x));
  return y;
}
// cap * tanh(y), cap2 x = 2 y log2(e): 1 - 2 / (e^2y + 1), its error 2^-22 of the cap, however small the score.  Weights of 11 bits
// are off by 2^-12 themselves: results of 16 bits take this form for caps up to kCoarseCap, where a score, and so a weight, is off by 2^-14.
constexpr float kCoarseCap = 256.f;
__device__ __forceinline__ float capped(float x, float cap2, float cap) { return fmaf(-2.f * cap, rcp(ex2(x * cap2) + 1.f), cap); }
// The same for f32 results and larger caps: below 0.6, where scores mostly are and the difference above cancels, y + y^3 P(y^2), P fitted at Chebyshev
// nodes (relative error 2^-23.6).  With it for all caps, calls of 16-bit results at a cap of 50 took 42 us for 37, 295 for 222 (256 rows
// behind 16384 tokens) and 1007 for 694 (seven prompts); with both forms in one kernel 38, 228 and 699.
__device__ __forceinline__ float capped_f32(float x, float cap2, float cap) {
  const float y = x * (cap2 * 0.34657359027997264f), z = y * y;  // ln(2) / 2
  float p = fmaf(-0.006276387721f, z, 0.02111621387f);
  p = fmaf(p, z, -0.05387513712f);
  p = fmaf(p, z, 0.1333292425f);
  p = fmaf(p, z, -0.3333333135f);
  const float big = fmaf(-2.f, rcp(ex2(fabsf(x * cap2)) + 1.f), 1.f);
  return cap * (fabsf(y) < 0.6f ? fmaf(y * z, p, y) : copysignf(big, y));
}
// address of 16-byte chunk c (0..15) of row r (16..31: V) of a page
__device__ __forceinline__ uint32_t chunk_at(int r, int c) { return (uint32_t)((c >> 3) * 4096 + r * 128 + (((c & 7) ^ (r & 7)) << 4)); }

// four values of row t, head hq, from dim d on
__device__ __forceinline__ void store4(const qeng_shared_attn& p, int t, int hq, int d, float4 v) {
  const size_t at = (size_t)t * p.ldo + (size_t)hq * kHD + d;
  if (p.out_dtype == QENG_F32) {
    *reinterpret_cast<float4*>(static_cast<float*>(p.out) + at) = v;
  } else if (p.out_dtype == QENG_F16) {
    *reinterpret_cast<uint2*>(static_cast<__half*>(p.out) + at) = make_uint2(pack_h2(v.x, v.y), pack_h2(v.z, v.w));
  } else {
    const __nv_bfloat162 a = __floats2bfloat162_rn(v.x, v.y), b = __floats2bfloat162_rn(v.z, v.w);
    *reinterpret_cast<uint2*>(static_cast<__nv_bfloat16*>(p.out) + at) = make_uint2(*reinterpret_cast<const uint32_t*>(&a), *reinterpret_cast<const uint32_t*>(&b));
  }
}

// eight of them
__device__ __forceinline__ void store8(const qeng_shared_attn& p, int t, int hq, int d, const float (&v)[8]) {
  if (p.out_dtype == QENG_F32) {
    store4(p, t, hq, d, make_float4(v[0], v[1], v[2], v[3]));
    store4(p, t, hq, d + 4, make_float4(v[4], v[5], v[6], v[7]));
    return;
  }
  uint32_t h[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const __nv_bfloat162 b = __floats2bfloat162_rn(v[2 * i], v[2 * i + 1]);
    h[i] = p.out_dtype == QENG_F16 ? pack_h2(v[2 * i], v[2 * i + 1]) : *reinterpret_cast<const uint32_t*>(&b);
  }
  *reinterpret_cast<uint4*>(static_cast<__half*>(p.out) + (size_t)t * p.ldo + (size_t)hq * kHD + d) = make_uint4(h[0], h[1], h[2], h[3]);
}

// ---- groups, rows and their units -----------------------------------------------------------------------------------------
struct Groups {
  int *first, *pages, *tile;  // [G + 1] each, in shared memory; tile: double tiles before a group
  __device__ Groups(int* at, int G) : first(at), pages(at + G + 1), tile(at + 2 * (G + 1)) {}
};
constexpr size_t groups_bytes(int64_t G) { return (size_t)(3 * (G + 1)) * sizeof(int); }

// Reads the groups into shared memory; false in every thread where their bounds do not ascend within the call's rows.
__device__ __forceinline__ bool read_groups(const qeng_shared_attn& p, const Groups& g) {
  bool bad = false;
  for (int i = threadIdx.x; i <= p.G; i += blockDim.x) {
    const int f = p.first[i];
    g.first[i] = f;
    if (i < p.G) {
      g.pages[i] = (int)min((long long)max(p.pages[i], 0), p.max_pages);
      bad = bad || p.first[i + 1] < f;
    }
    bad = bad || f < 0 || f > p.T;
  }
  if (__syncthreads_or(bad)) return false;
  if (threadIdx.x < 32) {
    const int lane = threadIdx.x;
    int sum = 0;
    for (int i = lane; i - lane < p.G; i += 32) {
      const int n = i < p.G && g.pages[i] > 0 ? (g.first[i + 1] - g.first[i] + 2 * p.tokens - 1) / (2 * p.tokens) : 0;
      int x = n;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int y = __shfl_up_sync(0xffffffffu, x, o);
        if (lane >= o) x += y;
      }
      if (i < p.G) g.tile[i] = sum + x - n;
      sum += __shfl_sync(0xffffffffu, x, 31);
    }
    if (lane == 0) g.tile[p.G] = sum;
  }
  __syncthreads();
  return true;
}

// last i in [0, n) with a[i] <= x (a ascends, a[0] <= x)
__device__ __forceinline__ int find(const int* a, int n, int x) {
  int lo = 0, hi = n;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (a[mid] <= x) lo = mid;
    else hi = mid;
  }
  return lo;
}

struct Row {
  int table_row, len, win0;  // table_row < 0: the row is not there
  int group;
  int page0, pages;          // its own pages: the first, how many
};

__device__ __forceinline__ int table_row_of(const qeng_shared_attn& p, int t) {
  const int row = p.rows ? __ldg(p.rows + t) : t;
  return row < p.table_rows ? row : -1;
}
__device__ __forceinline__ int len_of(const qeng_shared_attn& p, int t) { return (int)min((long long)max(__ldg(p.lens + t), 0), p.max_pages * kPage); }

__device__ __forceinline__ Row row_of(const qeng_shared_attn& p, const Groups& g, int t) {
  Row r;
  r.table_row = -1;
  r.len = r.win0 = r.group = r.page0 = r.pages = 0;
  if (t < g.first[0] || t >= g.first[p.G]) return r;
  r.group = find(g.first, p.G, t);
  r.table_row = table_row_of(p, t);
  if (r.table_row < 0) return r;
  r.len = len_of(p, t);
  r.win0 = p.window > 0 ? max(0, r.len - p.window) : 0;
  r.page0 = max(r.win0 / kPage, g.pages[r.group]);
  r.pages = max(0, (r.len + kPage - 1) / kPage - r.page0);
  return r;
}
// The CTAs (or warps) of a kernel divide its work evenly: CTA c has the units [c q, (c + 1) q) of `all`, q = share(all, n).
__device__ __forceinline__ long long divided(long long x, long long q) {  // of numbers that are not negative; most fit 32 bits
  return ((unsigned long long)(x | q) >> 32) == 0 ? (long long)((uint32_t)x / (uint32_t)q) : x / q;
}
__device__ __forceinline__ long long share(long long all, int n, int least = 1) { return max(divided(all + n - 1, n), (long long)least); }
// Work of attn_own_kernel: a (row, kv head) counts kStart pages more than it has, which is what its start and end cost (4 to 5 us, a
// page 1 us); a warp has kLeast at least, as cutting a pair costs, too.
constexpr int kStart = 4, kLeast = 6;
__device__ __forceinline__ int units_of(const Row& r) { return r.pages > 0 ? r.pages + kStart : 0; }
__device__ __forceinline__ long long own_share(const qeng_shared_attn& p) { return share(p.unit_first[p.T] * p.Hkv, p.own_warps, kLeast); }
// Adds up to 32 sums of one (row, head) to a running (M, L, O): lane i has the i-th, if any; its (m, l) and the place of its 128 values.
// The lanes' pairs are loaded together and so are the values, four dims a lane.
__device__ __forceinline__ void add_sums(int lane, bool have, const float2* ml_at, const float* o_at, float& M, float& L, float4& O) {
  const float2 ml = have ? *ml_at : make_float2(-INFINITY, 0.f);
  float m = ml.x;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
  m = fmaxf(m, M);
  // (m, l) = (-inf, NaN): scores of NaN alone; (-inf, 0): nothing attended, or scores of minus infinity alone
  const float f = ml.x == -INFINITY ? 0.f : exp2f(ml.x - m), a = M == -INFINITY ? 0.f : exp2f(M - m);
  float l = ml.x == -INFINITY ? ml.y : ml.y * f;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) l += __shfl_xor_sync(0xffffffffu, l, o);
  L = (M == -INFINITY ? L : L * a) + l;
  M = m;
  O.x *= a; O.y *= a; O.z *= a; O.w *= a;
  unsigned with = __ballot_sync(0xffffffffu, ml.x != -INFINITY);
  while (with != 0) {
    float4 v[4];
    float g[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int k = with != 0 ? __ffs(with) - 1 : -1;
      const float* const at = reinterpret_cast<const float*>(__shfl_sync(0xffffffffu, (unsigned long long)o_at, max(k, 0)));
      g[i] = __shfl_sync(0xffffffffu, f, max(k, 0));
      v[i] = make_float4(0.f, 0.f, 0.f, 0.f);
      if (k >= 0) v[i] = reinterpret_cast<const float4*>(at)[lane];
      else g[i] = 0.f;
      with &= with - 1;
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      O.x = fmaf(v[i].x, g[i], O.x); O.y = fmaf(v[i].y, g[i], O.y); O.z = fmaf(v[i].z, g[i], O.z); O.w = fmaf(v[i].w, g[i], O.w);
    }
  }
}

// The CTAs of attn_tile_kernel that worked on the double tile of row t and kv head h, c0 to c1; false: none did (no shared pages, or
// nobody in the double tile attends any).
__device__ __forceinline__ bool shared_ctas(const qeng_shared_attn& p, const Groups& g, const Row& r, int t, int h, int& c0, int& c1) {
  if (g.pages[r.group] == 0) return false;
  const int tile = g.tile[r.group] + (t - g.first[r.group]) / (2 * p.tokens), f0 = p.tile_first[tile], n = p.tile_first[tile + 1] - f0;
  if (n == 0) return false;
  const int q = (int)share((long long)p.tile_first[g.tile[p.G]] * p.Hkv, p.tile_ctas), x = f0 * p.Hkv + h * n;
  c0 = x / q;
  c1 = (x + n - 1) / q;
  return true;
}
// Adds the pieces of CTAs c0 to c1 of something cut between them, at `row` of `stride` rows for each piece.
__device__ __forceinline__ void add_pieces(int lane, int c0, int c1, const float* o, const float* ml, int stride, int row, float& M, float& L, float4& O) {
  for (int c = c0 + lane; c - lane <= c1; c += 32) {
    const size_t at = (size_t)(2 * c + (c == c0 ? 1 : 0)) * stride + row;  // the first CTA ends with it, the others begin with it
    add_sums(lane, c <= c1, reinterpret_cast<const float2*>(ml) + at, o + at * kHD, M, L, O);
  }
}

// ---- shared pages -------------------------------------------------------------------------------------------------------------
// A double tile is two tiles of 128 MMA rows, each of `tokens` tokens x the query heads of a kv head, against the same keys, 128 (eight
// pages) at a time.  Queries, K and V lie in shared memory, the scores S and the outputs O in tensor memory (256 columns
// a tile); the weights P take the place of the scores, as one f16 number or two (f32 results).  Warps 0-3 and 4-7 are the softmax of the
// two tiles, a lane a row; 8 issues the MMAs, 9 the copies, 10 and 11 look for values that are not finite.  The weights are handed over
// 64 keys at a time, the second ones first; the MMAs of one tile run beside the softmax of the other.  O is rescaled only when a row's
// maximum has grown by more than 2^kGrow since it was last.
//
// K and V tiles: [2 halves of 64 dims][128 keys][128 bytes], 128-byte swizzled; K is a K-major operand of 128 columns, V an MN-major one.
//
// Bound by the chain of a tile: 128 keys of both tiles take 3650 cycles, of which the MMAs need 2048 and the powers of two as many (16 a
// cycle and SM); a tile's softmax takes 2600 of them and then waits 1050 for its values and the next scores.  With two terms 7200 cycles.
// 256 rows behind 16384 tokens, 32 query and 8 kv heads: 78 us (69 GFLOP, 0.53 of the measured rate; the tensor pipe is busy for 44 % of
// the cycles), of which 3 us are the look at all rows in front.  Seven prompts of 7551 rows: 365 us.  A CTA's blocks are as many as another's,
// but from one (double tile, kv head) to the next takes 12000 cycles, and a CTA has 4 to 25 of them there: CTAs end between 40 and 372 us,
// half of them before 266, and the look at all rows takes 13 us (39 in the CTA that counts units).  What did not
// help, each measured against the kernel of its time: eight softmax warps a tile (96 registers and spills: 110 us, 92 without), a warp of
// its own for each tile's MMAs (the tiles fall into step and wait together: 4900 cycles for 128 keys), scores of 64 keys in two buffers
// (an MMA of 64 columns takes 74 cycles: 107 us, 92 without), part of the powers as polynomials on the FMA pipe (a call 133 us, 129
// without).
constexpr int kRows = 128, kKeys = 128;
constexpr uint32_t kTileBytes = kRows * kHD * 2, kHalf = kTileBytes / 2;
constexpr int kSoftWarps = 8, kMmaWarp = kSoftWarps, kLoadWarp = kMmaWarp + 1, kCheckWarp = kLoadWarp + 1, kCheckWarps = 2;
constexpr int kTileThreads = (kCheckWarp + kCheckWarps) * 32;
constexpr size_t kTileSmem = 6 * kTileBytes + 1024;
// Columns of a tile: scores at 0; the weights of 32 keys take the place of their scores, the second terms 16 columns behind the first.
constexpr uint32_t kO = 128;
// The MMAs cut the sums that they add to: 3e-7 of O a block with two terms.  For f32 results O starts anew every kFresh blocks, and what
// it held is added up in memory (in L2), rounded to nearest.
constexpr int kFresh = 2;
constexpr float kGrow = 8.f;   // weights reach 2^(kHigh + kGrow), below the largest f16 number

// Some blocks of a double tile.
struct Piece {
  int t0, ntok, tiles, h;
  int keys;                // shared keys of the group
  int page0, blocks;       // first page, blocks of 128 keys (none: no more pieces)
  int kv0, kv1;            // keys that any row attends: [kv0, kv1)
  int begin_max, end_min;  // keys that every row attends (which attends any)
  int table_row, whole, slot;
};
// whether some row does not attend some key of block j
__device__ __forceinline__ bool is_edge(const Piece& w, int j) {
  const int key0 = w.page0 * kPage + j * kKeys;
  return key0 < w.begin_max || key0 + kKeys > w.end_min;
}

// keys that the rows of a double tile attend among the shared ones, found by a warp
__device__ __forceinline__ void span_of(const qeng_shared_attn& p, int lane, Piece& w) {
  int kv0 = 0x7fffffff, kv1 = 0, begin_max = 0, end_min = 0x7fffffff, some = 0x7fffffff;
  for (int i = lane; i < w.ntok; i += 32) {
    const int t = w.t0 + i, len = len_of(p, t), begin = p.window > 0 ? max(0, len - p.window) : 0, end = min(len, w.keys);
    if (table_row_of(p, t) < 0 || begin >= end) continue;
    kv0 = min(kv0, begin);
    kv1 = max(kv1, end);
    begin_max = max(begin_max, begin);
    end_min = min(end_min, end);
    some = min(some, i);
  }
  w.kv0 = __reduce_min_sync(0xffffffffu, kv0);
  w.kv1 = __reduce_max_sync(0xffffffffu, kv1);
  w.begin_max = __reduce_max_sync(0xffffffffu, begin_max);
  w.end_min = __reduce_min_sync(0xffffffffu, end_min);
  some = __reduce_min_sync(0xffffffffu, some);
  w.table_row = some == 0x7fffffff ? -1 : table_row_of(p, w.t0 + some);
}
__device__ __forceinline__ void rows_of_tile(const qeng_shared_attn& p, const Groups& g, int tile, Piece& w) {
  const int k = find(g.tile, p.G, tile);  // the last group that begins here: the others are empty
  w.t0 = g.first[k] + (tile - g.tile[k]) * 2 * p.tokens;
  w.ntok = min(2 * p.tokens, g.first[k + 1] - w.t0);
  w.tiles = w.ntok > p.tokens ? 2 : 1;
  w.keys = (int)min((long long)g.pages[k] * kPage, 0x7fffffffll);
}
__device__ __forceinline__ int blocks_of(int kv0, int kv1) { return kv1 > kv0 ? (kv1 - kv0 / kPage * kPage + kKeys - 1) / kKeys : 0; }

// unit_first, by one CTA
__device__ __forceinline__ void count_units(const qeng_shared_attn& p, const Groups& g, long long* sums) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  long long before = 0;
  for (int t0 = 0; t0 < p.T; t0 += kTileThreads) {
    const int t = t0 + threadIdx.x;
    long long n = 0;
    if (t < p.T) {
      n = units_of(row_of(p, g, t));
      if (p.rows && t >= g.first[0] && t < g.first[p.G] && __ldg(p.rows + t) >= p.table_rows) atomicExch(p.status, 6);
    }
    long long x = n;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const long long y = __shfl_up_sync(0xffffffffu, x, o);
      if (lane >= o) x += y;
    }
    if (lane == 31) sums[warp] = x;
    __syncthreads();
    long long front = before;
    for (int w = 0; w < kTileThreads / 32; ++w) {
      const long long y = sums[w];
      if (w < warp) front += y;
      before += y;
    }
    if (t < p.T) p.unit_first[t] = front + x - n;
    __syncthreads();
  }
  if (threadIdx.x == 0) p.unit_first[p.T] = before;
}

struct TileShared {
  alignas(8) int first[kSharedTiles + 1];  // blocks (of one kv head) before a double tile
  Piece piece[2];
  uint32_t bad[2][4];           // of a V tile: keys with a value that is not finite
  int begun[2];                 // O of a tile holds sums before its first MMA
  uint32_t tmem;
  // full / empty: pieces' descriptions, queries, K and V tiles (even, odd); of a tile: scores done, the last values of a piece
  // added, weights ready (of the first, the second 64 keys); V looked through
  uint64_t pfull[2], pempty[2], qfull, qempty, full[4], empty[4], sdone[2], odone[2], pready[2][2], checked[2], drained;
};

template <bool kTwo, bool kFineCap>  // weights as two f16 numbers; scores capped by capped_f32
__global__ void __launch_bounds__(kTileThreads, 1) attn_tile_kernel(const qeng_shared_attn p, const __grid_constant__ CUtensorMap kvmap, const __grid_constant__ CUtensorMap qmap) {
  extern __shared__ unsigned char smem_raw[];
  const uint32_t qs = (smem_u32(smem_raw) + 1023u) & ~1023u, ring = qs + 2 * kTileBytes;
  __shared__ __align__(8) TileShared sh;
  const Groups groups(reinterpret_cast<int*>(smem_raw + kTileSmem), p.G);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, cta = blockIdx.x;
  if (tid == 0) {
    for (int i = 0; i < 2; ++i) {
      mbar_init(smem_u32(sh.pfull + i), 1);
      mbar_init(smem_u32(sh.pempty + i), kSoftWarps + 1 + kCheckWarps);
      mbar_init(smem_u32(sh.sdone + i), 1);
      for (int k = 0; k < 2; ++k) mbar_init(smem_u32(&sh.pready[i][k]), kSoftWarps / 2);
      mbar_init(smem_u32(sh.odone + i), 1);
      mbar_init(smem_u32(sh.checked + i), kCheckWarps);
    }
    for (int i = 0; i < 4; ++i) {
      mbar_init(smem_u32(sh.full + i), 1);
      mbar_init(smem_u32(sh.empty + i), i & 1 ? 1 + kCheckWarps : 1);
    }
    mbar_init(smem_u32(&sh.qfull), 1);
    mbar_init(smem_u32(&sh.qempty), 1);
    mbar_init(smem_u32(&sh.drained), 1);
    asm volatile("fence.mbarrier_init.release.cluster;\n" ::: "memory");
  }
  if (tid == 0) p.tile_jobs[cta].tokens = 0;
  if (warp == kLoadWarp && lane < 2) asm volatile("prefetch.tensormap [%0];\n" ::"l"(lane == 0 ? &kvmap : &qmap) : "memory");
  if (!read_groups(p, groups)) return;  // (attn_own_kernel reports it)
  if (cta == (int)gridDim.x - 1) count_units(p, groups, reinterpret_cast<long long*>(sh.first));  // it has least to do
  const int ntiles = groups.tile[p.G];
  {  // keys that the double tiles attend, a thread a row; the ring is not in use yet
    int* const kv0 = reinterpret_cast<int*>(smem_raw);
    int* const kv1 = kv0 + ntiles;
    for (int s = tid; s < ntiles; s += kTileThreads) {
      kv0[s] = 0x7fffffff;
      kv1[s] = 0;
    }
    __syncthreads();
#pragma unroll 4
    for (int t = groups.first[0] + tid; t < groups.first[p.G]; t += kTileThreads) {
      const int g = find(groups.first, p.G, t), len = len_of(p, t), begin = p.window > 0 ? max(0, len - p.window) : 0, end = min(len, groups.pages[g] * kPage);
      if (table_row_of(p, t) >= 0 && begin < end) {
        const int s = groups.tile[g] + (t - groups.first[g]) / (2 * p.tokens);
        atomicMin(kv0 + s, begin);
        atomicMax(kv1 + s, end);
      }
    }
    __syncthreads();
    for (int s = tid; s < ntiles; s += kTileThreads) sh.first[s + 1] = blocks_of(kv0[s], kv1[s]);
    asm volatile("fence.proxy.async.shared::cta;\n" ::: "memory");  // copies write there
  }
  if (tid == 0) sh.first[0] = 0;
  __syncthreads();
  if (warp == 0) {
    int sum = 0;
    for (int i = lane; i - lane < ntiles; i += 32) {
      int x = i < ntiles ? sh.first[i + 1] : 0;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int y = __shfl_up_sync(0xffffffffu, x, o);
        if (lane >= o) x += y;
      }
      if (i < ntiles) sh.first[i + 1] = sum + x;
      sum += __shfl_sync(0xffffffffu, x, 31);
    }
  } else if (warp == kMmaWarp) {
    tmem_alloc(smem_u32(&sh.tmem));
    asm volatile("griddepcontrol.launch_dependents;\n" ::: "memory");
  }
  fence_before();
  __syncthreads();
  fence_after();
  if (cta == 0)
    for (int s = tid; s <= ntiles; s += kTileThreads) p.tile_first[s] = sh.first[s];
  const uint32_t tmem = sh.tmem;
  const int all = sh.first[ntiles] * p.Hkv, q = (int)share(all, gridDim.x), u0 = min(all, cta * q), u1 = min(all, u0 + q);
  bool failed = false;

  // a warp of another role asks for the next piece's description, which stays until it asks again; null: no more
  int npiece = 0;
  const auto next_piece = [&]() -> const Piece* {
    if (npiece > 0) {  // done with the last one
      __syncwarp();
      if (lane == 0) mbar_arrive(smem_u32(sh.pempty + ((npiece - 1) & 1)));
    }
    const int e = npiece & 1;
    if (failed || !wait_warp(smem_u32(sh.pfull + e), (uint32_t)(npiece >> 1) & 1u)) {
      failed = true;
      return nullptr;
    }
    ++npiece;
    return sh.piece[e].blocks > 0 ? &sh.piece[e] : nullptr;
  };

  if (warp == kLoadWarp) {
    // ===== pieces and copies ============================================================================================
    int n = 0, b = 0;  // pieces, blocks so far
    int u = u0, s = u < u1 ? find(sh.first, ntiles, u / p.Hkv) : 0;
    for (;;) {
      Piece w;
      w.blocks = 0;
      if (u < u1) {
        while (sh.first[s + 1] * p.Hkv <= u) ++s;
        rows_of_tile(p, groups, s, w);
        span_of(p, lane, w);
        const int nb = sh.first[s + 1] - sh.first[s], at = u - sh.first[s] * p.Hkv;
        w.h = at / nb;
        const int k0 = at - w.h * nb;
        w.blocks = min(nb - k0, u1 - u);
        w.page0 = w.kv0 / kPage + k0 * (kKeys / kPage);
        w.whole = w.blocks == nb;
        w.slot = 2 * cta + (k0 == 0 ? 1 : 0);
        if (k0 == 0 && !w.whole && lane == 0) {  // cut: attn_join_kernel adds the pieces
          qeng_tile_job& job = p.tile_jobs[cta];
          job.t0 = w.t0;
          job.h = w.h;
          job.last = (u + nb - 1) / q;
          job.tokens = w.ntok;
        }
      }
      if (!wait_warp(smem_u32(sh.pempty + (n & 1)), ((uint32_t)(n >> 1) & 1u) ^ 1u)) { failed = true; break; }
      if (lane == 0) {
        sh.piece[n & 1] = w;
        mbar_arrive(smem_u32(sh.pfull + (n & 1)));
      }
      __syncwarp();
      if (w.blocks == 0) break;
      const int last_page = (w.kv1 - 1) / kPage;
      const int32_t* const ids = p.table + (size_t)w.table_row * p.max_pages;
      // lanes 2 i and 2 i + 1 copy the two halves of page i of the block
      const int pg = lane >> 1, half = lane & 1;
      const auto queries = [&] {  // half a tile at a time
        if (!wait_warp(smem_u32(&sh.qempty), ((uint32_t)n & 1u) ^ 1u)) {
          failed = true;
          return;
        }
        if (lane == 0) mbar_expect_tx(smem_u32(&sh.qfull), (uint32_t)(w.tiles * 2 * 128 * p.grp * p.tokens));
        __syncwarp();
        if (lane < 2 * w.tiles)
          asm volatile("cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];\n" ::"r"(
                           qs + (uint32_t)(lane >> 1) * kTileBytes + (uint32_t)half * kHalf),
                       "l"(&qmap), "r"(64 * half), "r"(w.h * p.grp), "r"(w.t0 + (lane >> 1) * p.tokens), "r"(smem_u32(&sh.qfull))
                       : "memory");
      };
      if (n == 0) queries();
      int id = lane < 16 && w.page0 + pg <= last_page ? ids[w.page0 + pg] : 0;
      for (int j = 0; j < w.blocks && !failed; ++j, ++b) {
        const int here = w.page0 + j * 8, pages = min(8, last_page - here + 1);
        int row = -64;  // in front of the pool: the copies bring zeros
        if ((unsigned)id < (unsigned)p.pool_pages) row = (id * p.Hkv + w.h) * 32;
        else atomicExch(p.status, 1);  // malformed page table
        if (lane < 16 && j + 1 < w.blocks && here + 8 + pg <= last_page) id = ids[here + 8 + pg];
        for (int kv = 0; kv < 2; ++kv) {
          const int slot = 2 * (b & 1) + kv;
          const uint32_t bar = smem_u32(sh.full + slot);
          if (!wait_warp(smem_u32(sh.empty + slot), ((uint32_t)(b >> 1) & 1u) ^ 1u)) { failed = true; break; }
          if (lane == 0) mbar_expect_tx(bar, (uint32_t)pages * 4096u);
          __syncwarp();
          if (lane < 2 * pages)
            asm volatile("cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];\n" ::"r"(
                             ring + (uint32_t)slot * kTileBytes + (uint32_t)half * kHalf + (uint32_t)pg * 2048u),
                         "l"(&kvmap), "r"(0), "r"(row + 16 * kv), "r"(half), "r"(bar)
                         : "memory");
        }
        if (j == 0 && n > 0 && !failed) queries();  // behind the first K and V: the last piece may still use theirs
      }
      if (failed) break;
      u += w.blocks;
      ++n;
    }
  } else if (warp == kMmaWarp) {
    // ===== MMA issue ====================================================================================================
    // f16 x f16 -> f32, M = N = 128; B of S K-major, of O MN-major
    constexpr uint32_t kIdescS = (1u << 4) | (16u << 17) | (8u << 24), kIdescO = kIdescS | (1u << 16);
    constexpr uint32_t kTwoTiles = 2 * kTileBytes >> 4;
    const uint32_t tm = __shfl_sync(0xffffffffu, tmem, 0), r0 = __shfl_sync(0xffffffffu, ring, 0);
    const uint64_t qd = make_desc(__shfl_sync(0xffffffffu, qs, 0), 16, 1024);
    const uint64_t kd = make_desc(r0, 16, 1024), vd = make_desc(r0 + kTileBytes, kHalf, 1024);  // + 2 tiles in the odd blocks
    int b = 0;                // blocks so far
    uint32_t turn = 0;        // parities of pready (bit 2 x + half) and of checked (bit 4 + slot)
    const bool leader = elect_one();
    const int who = __ffs(__ballot_sync(0xffffffffu, leader)) - 1;
    while (const Piece* const piece = next_piece()) {
      const int blocks = piece->blocks, tiles = piece->tiles, left0 = piece->kv1 - piece->page0 * kPage;
      bool lost = false;
      if (leader) {
        const auto full = [&](int kv, int blk) { return mbar_wait(smem_u32(sh.full + 2 * (blk & 1) + kv), (uint32_t)(blk >> 1) & 1u); };
        const auto scores = [&](int x, int blk, bool last) {
          const uint64_t q = qd + (kTileBytes >> 4) * x, k = kd + kTwoTiles * (blk & 1);
#pragma unroll
          for (int c = 0; c < 8; ++c) {
            const uint32_t at = (uint32_t)(c >> 2) * (kHalf >> 4) + (uint32_t)(c & 3) * 2u;
            umma_ss(tm + (uint32_t)x * 256u, q + at, k + at, kIdescS, c > 0);
          }
          umma_commit(smem_u32(sh.sdone + x));
          if (x + 1 == tiles) {
            umma_commit(smem_u32(sh.empty + 2 * (blk & 1)));
            if (last) umma_commit(smem_u32(&sh.qempty));
          }
        };
        lost = !mbar_wait(smem_u32(&sh.qfull), (uint32_t)(npiece - 1) & 1u) || !full(0, b);
        if (!lost) {
          fence_after();
          scores(0, b, blocks == 1);
          if (tiles == 2) scores(1, b, blocks == 1);
        }
        for (int j = 0; j < blocks && !lost; ++j) {
          const int blk = b + j, left = left0 - kKeys * j;
          const bool edge = is_edge(*piece, j);
          const uint64_t v = vd + kTwoTiles * (blk & 1);
#pragma unroll
          for (int x = 0; x < 2; ++x) {
            if (x >= tiles || lost) continue;
#pragma unroll
            for (int half = 1; half >= 0; --half) {  // the second 64 keys first
              if (lost || left <= 64 * half) continue;
              const bool first = half == 1 || left <= 64;
              if (!mbar_wait(smem_u32(&sh.pready[x][half]), (turn >> (2 * x + half)) & 1u)) { lost = true; continue; }
              turn ^= 1u << (2 * x + half);
              if (x == 0 && first) {
                if (!full(1, blk)) { lost = true; continue; }
                if (edge) {
                  if (!mbar_wait(smem_u32(sh.checked + (blk & 1)), (turn >> (4 + (blk & 1))) & 1u)) { lost = true; continue; }
                  turn ^= 16u << (blk & 1);
                }
              }
              fence_after();
              uint32_t acc = !first || (kTwo ? j % kFresh != 0 : j > 0) || *(volatile int*)&sh.begun[x];
              const int steps = (left - 64 * half + kPage - 1) / kPage;
#pragma unroll
              for (int k = 0; k < 4; ++k) {
                if (k >= steps) continue;
                const uint32_t w_at = tm + (uint32_t)x * 256u + 64u * half + 32u * (k >> 1) + 8u * (k & 1);
                umma_ts(tm + (uint32_t)x * 256u + kO, w_at, v + (uint32_t)(4 * half + k) * (2048u >> 4), kIdescO, acc);
                if (kTwo) umma_ts(tm + (uint32_t)x * 256u + kO, w_at + 16u, v + (uint32_t)(4 * half + k) * (2048u >> 4), kIdescO, 1u);
                acc = 1u;
              }
            }
            if (lost) continue;
            if (j + 1 < blocks) {
              if (x == 0) {
                if (!full(0, blk + 1)) { lost = true; continue; }
                fence_after();
              }
              scores(x, blk + 1, j + 2 == blocks);
            } else {
              umma_commit(smem_u32(sh.odone + x));
            }
            if (x + 1 == tiles) umma_commit(smem_u32(sh.empty + 2 * (blk & 1) + 1));
          }
        }
        if (lost) {  // what was issued still has to finish before tensor memory is freed
          umma_commit(smem_u32(&sh.drained));
          mbar_wait(smem_u32(&sh.drained), 0);
        }
      }
      lost = __shfl_sync(0xffffffffu, (int)lost, who);
      if (lost) { failed = true; break; }
      b += blocks;
    }
  } else if (warp >= kCheckWarp) {
    // ===== values that are not finite ===================================================================================
    // Where the rows of a block attend different keys, a value that is not finite would reach rows that do not attend it (their weight
    // is zero, but zero times infinity is NaN).  Such keys are cleared here, and their rows added by the softmax; keys that nobody
    // attends, and what no copy wrote, are cleared, too.
    int b = 0;
    while (const Piece* const piece = next_piece()) {
      const Piece& w = *piece;
      for (int j = 0; j < w.blocks && !failed; ++j, ++b) {
        // every tile is waited for, and let go: a parity says nothing to those who have missed a turn
        if (!wait_warp(smem_u32(sh.full + 2 * (b & 1) + 1), (uint32_t)(b >> 1) & 1u)) { failed = true; break; }
        if (!is_edge(w, j)) {
          if (lane == 0) mbar_arrive(smem_u32(sh.empty + 2 * (b & 1) + 1));
          continue;
        }
        const int key0 = (w.page0 + 8 * j) * kPage;
        const uint32_t v = ring + (uint32_t)(2 * (b & 1) + 1) * kTileBytes;
#pragma unroll 1
        for (int i = 0; i < 2; ++i) {
          const int r = (warp - kCheckWarp) * 64 + 32 * i + lane;
          const bool used = key0 + r >= w.kv0 && key0 + r < w.kv1;
          uint32_t worst = 0;  // largest magnitude bits of the halves: an exponent of all ones has 0x7c00 and more
          if (used) {
#pragma unroll
            for (int c = 0; c < 16; ++c) {
              uint4 y;
              asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];\n"
                           : "=r"(y.x), "=r"(y.y), "=r"(y.z), "=r"(y.w)
                           : "r"(v + (uint32_t)(c >> 3) * kHalf + (uint32_t)r * 128u + (uint32_t)(((c & 7) ^ (r & 7)) << 4))
                           : "memory");
              worst = __vmaxu2(worst, __vmaxu2(__vmaxu2(y.x & 0x7fff7fffu, y.y & 0x7fff7fffu), __vmaxu2(y.z & 0x7fff7fffu, y.w & 0x7fff7fffu)));
            }
          }
          const bool bad = (worst & 0xffffu) >= 0x7c00u || (worst >> 16) >= 0x7c00u;
          if (!used || bad) {
#pragma unroll
            for (int c = 0; c < 16; ++c)
              asm volatile("st.shared.v4.u32 [%0], {%1,%1,%1,%1};\n" ::"r"(v + (uint32_t)(c >> 3) * kHalf + (uint32_t)r * 128u + (uint32_t)((c & 7) << 4)), "r"(0u) : "memory");
          }
          const uint32_t mask = __ballot_sync(0xffffffffu, bad);
          if (lane == 0) sh.bad[b & 1][(warp - kCheckWarp) * 2 + i] = mask;
        }
        asm volatile("fence.proxy.async.shared::cta;\n" ::: "memory");
        __syncwarp();
        if (lane == 0) {
          mbar_arrive(smem_u32(sh.checked + (b & 1)));
          mbar_arrive(smem_u32(sh.empty + 2 * (b & 1) + 1));
        }
      }
    }
  } else {
    // ===== softmax: this lane's row of tile x ============================================================================
    const int x = warp >> 2, row = (warp & 3) * 32 + lane, tok = row / p.grp;
    const uint32_t mem = tmem + ((uint32_t)((warp & 3) * 32) << 16) + (uint32_t)x * 256u;
    const float sc = p.softcap > 0.f ? 1.f : p.scale * kLog2e;
    const float cap2 = 2.f * kLog2e * p.scale / p.softcap, cap = p.softcap * kLog2e;
    float4* const kept = reinterpret_cast<float4*>(p.kept_o) + (size_t)cta * 8192 + x * kRows + row;  // this lane's; [32 x 4 dims][256 rows] of a CTA
    int b = 0;
    uint32_t turn = 0;  // parities of sdone (bit 0), odone (1) and checked (4 + slot)
    while (const Piece* const piece = next_piece()) {
      const Piece& w = *piece;
      if (x >= w.tiles) {
        for (int j = 0; j < w.blocks; ++j)
          if (is_edge(w, j)) turn ^= 16u << ((b + j) & 1);
        b += w.blocks;
        continue;
      }
      const int i = x * p.tokens + tok, t = w.t0 + i, head = w.h * p.grp + row - tok * p.grp;
      bool live = tok < p.tokens && i < w.ntok;
      int len = 0;
      if (live) {
        live = table_row_of(p, t) >= 0;
        if (live) len = len_of(p, t);
      }
      const int win0 = p.window > 0 ? max(0, len - p.window) : 0;
      const bool some = live && win0 < min(len, w.keys);
      // a row that attends none of these keys attends everything, to nobody's use
      const int begin = some ? win0 : 0, end = some ? min(len, w.keys) : 0x7fffffff;
      float m_run = -INFINITY, l_run = 0.f;
      float scale_kept = 1.f;  // of what `kept` holds, since it was last written
#pragma unroll 1
      for (int j = 0; j < w.blocks; ++j, ++b) {
        const int key0 = (w.page0 + 8 * j) * kPage;
        const bool edge = is_edge(w, j), fresh = kTwo ? j % kFresh == 0 : j == 0;
        if (!wait_warp(smem_u32(sh.sdone + x), turn & 1u)) { failed = true; break; }
        turn ^= 1u;
        fence_after();
        const bool two = key0 + 64 < w.kv1;  // keys in the second half, too
        // 64 keys at a time, the second ones first.  The first ones' scores are read twice: what was handed over then runs beside
        // their weights, where the compiler would otherwise put those in front.
        float s[64];
        const auto scores = [&](int half) {
          __syncwarp();  // one lane has let the MMAs go on with the other half
          tmem_ld64(mem + 64 * half, reinterpret_cast<uint32_t*>(s));
          if (p.softcap > 0.f) {
#pragma unroll
            for (int k = 0; k < 64; ++k) s[k] = kFineCap ? capped_f32(s[k], cap2, cap) : capped(s[k], cap2, cap);
          }
          if (edge) {
            const int e = end - key0 - 64 * half, a = begin - key0 - 64 * half;
            if (__any_sync(0xffffffffu, e < 64)) {
#pragma unroll
              for (int k = 0; k < 64; ++k) s[k] = k < e ? s[k] : -INFINITY;
            }
            if (__any_sync(0xffffffffu, a > 0)) {
#pragma unroll
              for (int k = 0; k < 64; ++k) s[k] = k >= a ? s[k] : -INFINITY;
            }
          }
        };
        float mx = -INFINITY;
#pragma unroll 1
        for (int half = 0; half <= (two ? 1 : 0); ++half) {
          scores(half);
          float mx4[4] = {max3(mx, s[0], s[1]), s[2], s[3], max3(s[4], s[5], s[6])};
#pragma unroll
          for (int k = 7; k < 63; k += 2) mx4[(k >> 1) & 3] = max3(mx4[(k >> 1) & 3], s[k], s[k + 1]);
          mx = max3(max3(mx4[0], mx4[1], mx4[2]), mx4[3], s[63]);
        }
        // the reference of the row's weights moves when its maximum has left it far behind
        const bool moved = mx > m_run && (m_run == -INFINITY || (mx - m_run) * sc > kGrow);
        if (__any_sync(0xffffffffu, moved)) {
          const float alpha = !moved ? 1.f : m_run == -INFINITY ? 0.f : ex2((m_run - mx) * sc);
          if (moved) m_run = mx;
          l_run *= alpha;
          scale_kept *= alpha;
          if (j > 0) {  // the values of the block before are in (its scores came behind them), the next wait for this warp
            __syncwarp();  // not every lane's reference has moved
#pragma unroll 1
            for (int c = 0; c < 4; ++c) {
              uint32_t o[32];
              tmem_ld32(mem + kO + 32 * c, o);
#pragma unroll
              for (int k = 0; k < 32; ++k) o[k] = __float_as_uint(__uint_as_float(o[k]) * alpha);
              tmem_st32(mem + kO + 32 * c, o);
            }
          }
        }
        if (kTwo && fresh && j > 0) {
          st_wait();
          __syncwarp();
#pragma unroll 1
          for (int c = 0; c < 4; ++c) {
            float4 before[8];
            if (j > kFresh) {
#pragma unroll
              for (int d = 0; d < 8; ++d) before[d] = __ldcg(kept + (8 * c + d) * 256);
            }
            uint32_t o[32];
            tmem_ld32(mem + kO + 32 * c, o);
#pragma unroll
            for (int d = 0; d < 8; ++d) {
              float4 v = make_float4(__uint_as_float(o[4 * d]), __uint_as_float(o[4 * d + 1]), __uint_as_float(o[4 * d + 2]), __uint_as_float(o[4 * d + 3]));
              if (j > kFresh)
                v = make_float4(fmaf(before[d].x, scale_kept, v.x), fmaf(before[d].y, scale_kept, v.y), fmaf(before[d].z, scale_kept, v.z), fmaf(before[d].w, scale_kept, v.w));
              __stcg(kept + (8 * c + d) * 256, v);
            }
          }
          scale_kept = 1.f;
        }
        const float off = m_run == -INFINITY ? 0.f : kHigh - m_run * sc;  // nothing attended yet: all weights are zero
        float sum[8];
#pragma unroll
        for (int k = 0; k < 8; ++k) sum[k] = 0.f;
        bool zeroed = false;
#pragma unroll 1
        for (int half = two ? 1 : 0; half >= 0; --half) {
          if (half == 0 && two) scores(0);
#pragma unroll
          for (int c = 0; c < 2; ++c) {  // 32 keys at a time
            uint32_t hi[16], lo[16];
#pragma unroll
            for (int k = 0; k < 16; ++k) {
              float &a0 = s[32 * c + 2 * k], &a1 = s[32 * c + 2 * k + 1];
              fma2(a0, a1, sc, off);
              a0 = ex2(a0);
              a1 = ex2(a1);
              add2(sum[2 * (k & 3)], sum[2 * (k & 3) + 1], a0, a1);
              hi[k] = pack_h2(a0, a1);
              if (kTwo) {
                const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&hi[k]));
                lo[k] = pack_h2(a0 - f.x, a1 - f.y);
              }
            }
            tmem_st16(mem + 64 * half + 32 * c, hi);
            if (kTwo) tmem_st16(mem + 64 * half + 32 * c + 16, lo);
          }
          st_wait();
          if (half == 1 && !edge) {  // of an edge both wait for the values that are not finite
            if (fresh && tid % 128 == 0) *(volatile int*)&sh.begun[x] = 0;
            fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(smem_u32(&sh.pready[x][1]));
          }
        }
        l_run += ((sum[0] + sum[1]) + (sum[2] + sum[3])) + ((sum[4] + sum[5]) + (sum[6] + sum[7]));
        if (edge) {
          if (!wait_warp(smem_u32(sh.checked + (b & 1)), (turn >> (4 + (b & 1))) & 1u)) { failed = true; break; }
          turn ^= 16u << (b & 1);
#pragma unroll 1
          for (int q = 0; q < 4; ++q) {
#pragma unroll 1
            for (uint32_t mask = sh.bad[b & 1][q]; mask != 0; mask &= mask - 1) {  // the same in all lanes
              const int k = 32 * q + __ffs(mask) - 1, key = key0 + k;
              if (fresh && !zeroed) {
                uint32_t z[32];
#pragma unroll
                for (int d = 0; d < 32; ++d) z[d] = 0u;
#pragma unroll 1
                for (int c = 0; c < 4; ++c) tmem_st32(mem + kO + 32 * c, z);
                st_wait();
                zeroed = true;
              }
              float weight = 0.f;
#pragma unroll 1
              for (int c = 0; c <= (kTwo ? 16 : 0); c += 16) {
                const uint32_t y = tmem_ld1(mem + (k & ~31) + c + (k & 31) / 2);
                const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&y));
                weight += k & 1 ? f.y : f.x;
              }
              const bool on = key >= begin && key < end;
              const int id = p.table[(size_t)w.table_row * p.max_pages + key / kPage];
              if ((unsigned)id >= (unsigned)p.pool_pages) continue;  // (its place holds zeros, and is not looked up)
              const __half2* const val = reinterpret_cast<const __half2*>(p.pool + (((size_t)id * p.Hkv + w.h) * 32 + 16 + key % kPage) * kHD);
#pragma unroll 1
              for (int c = 0; c < 4; ++c) {
                uint32_t o[32];
                tmem_ld32(mem + kO + 32 * c, o);
#pragma unroll
                for (int d = 0; d < 16; ++d) {
                  const float2 f = __half22float2(val[16 * c + d]);
                  if (on) {
                    o[2 * d] = __float_as_uint(fmaf(weight, f.x, __uint_as_float(o[2 * d])));
                    o[2 * d + 1] = __float_as_uint(fmaf(weight, f.y, __uint_as_float(o[2 * d + 1])));
                  }
                }
                __syncwarp();
                tmem_st32(mem + kO + 32 * c, o);
              }
              st_wait();
            }
          }
        }
        fence_before();
        __syncwarp();
        if (lane == 0) {
          if (fresh && (warp & 3) == 0 && (edge || !two)) *(volatile int*)&sh.begun[x] = zeroed;
          if (edge && two) mbar_arrive(smem_u32(&sh.pready[x][1]));
          mbar_arrive(smem_u32(&sh.pready[x][0]));
        }
      }
      if (failed || !wait_warp(smem_u32(sh.odone + x), (turn >> 1) & 1u)) { failed = true; break; }
      turn ^= 2u;
      fence_after();
      // Whole and all that the row attends: its result.  Otherwise what has to be added to others' sums.
      const bool alone = max((len + kPage - 1) / kPage - max(win0 / kPage, w.keys / kPage), 0) == 0;
      const bool result = w.whole && alone;  // (attn_own_kernel writes the zeros of a row that attends nothing)
      const float inv = 1.f / l_run;
      const size_t place = w.whole ? (size_t)t * p.Hq + head : (size_t)w.slot * 256 + x * kRows + row;
      if (live && !(w.whole && alone)) {
        float* const ml = (w.whole ? p.row_ml : p.tile_ml) + 2 * place;
        // rows that attend nothing here have no weight
        *reinterpret_cast<float2*>(ml) = some ? make_float2(m_run == -INFINITY ? -INFINITY : m_run * sc - kHigh, l_run) : make_float2(-INFINITY, 0.f);
      }
#pragma unroll 1
      for (int c = 0; c < 4; ++c) {
        uint32_t o[32];
        __syncwarp();
        tmem_ld32(mem + kO + 32 * c, o);
        if (kTwo && w.blocks > kFresh) {
#pragma unroll
          for (int d = 0; d < 8; ++d) {
            const float4 v = __ldcg(kept + (8 * c + d) * 256);
            o[4 * d] = __float_as_uint(fmaf(v.x, scale_kept, __uint_as_float(o[4 * d])));
            o[4 * d + 1] = __float_as_uint(fmaf(v.y, scale_kept, __uint_as_float(o[4 * d + 1])));
            o[4 * d + 2] = __float_as_uint(fmaf(v.z, scale_kept, __uint_as_float(o[4 * d + 2])));
            o[4 * d + 3] = __float_as_uint(fmaf(v.w, scale_kept, __uint_as_float(o[4 * d + 3])));
          }
        }
        if (!live || (result && !some)) continue;
        if (result) {
#pragma unroll
          for (int d = 0; d < 32; d += 8) {
            float f[8];
#pragma unroll
            for (int k = 0; k < 8; ++k) f[k] = __uint_as_float(o[d + k]) * inv;
            store8(p, t, head, 32 * c + d, f);
          }
        } else {
          // a cut piece: [32 x 4 dims][256 rows]
          float4* const dst = reinterpret_cast<float4*>(w.whole ? p.row_o + place * kHD + 32 * c : p.tile_o + ((size_t)w.slot * 32 + 8 * c) * 1024 + 4 * (x * kRows + row));
          const int step = w.whole ? 1 : 256;
#pragma unroll
          for (int d = 0; d < 8; ++d) {
            const float4 v = make_float4(__uint_as_float(o[4 * d]), __uint_as_float(o[4 * d + 1]), __uint_as_float(o[4 * d + 2]), __uint_as_float(o[4 * d + 3]));
            dst[d * step] = some ? v : make_float4(0.f, 0.f, 0.f, 0.f);
          }
        }
      }
      __syncwarp();
    }
  }
  if (failed && lane == 0) atomicExch(p.status, 4);
  fence_before();
  if (__syncthreads_or(failed)) grace();
  if (warp == kMmaWarp) tmem_free(tmem);
}

// ---- a row's own pages ------------------------------------------------------------------------------------------------------
// Every warp has pages of its own, of one or several (row, kv head), and keeps two on their way.  HBM-bound where there are many pages:
// 256 rows of 1 to 256 tokens (134 MB) take 29 us (4.6 TB/s), 64 of 1 to 1024 27 us; below that a start and an end, 4 to 5 us, and 1 us
// a page.  Three CTAs fit on an SM up to about 840 groups, above that two, but the work is cut for three: 1000 rows of 1024 tokens take
// 718 us in as many groups, 661 in one.  With a (row, kv head) for the four warps of a CTA, merged in shared memory, these took 57 and 48 us.  The query heads of the
// kv head are the eight columns of every MMA, S^T = K Q^T and O^T = V^T P^T; P in two f16 terms.
__global__ void __launch_bounds__(kThreads, 3) attn_own_kernel(const qeng_shared_attn p, const __grid_constant__ CUtensorMap kvmap) {
  asm volatile("griddepcontrol.launch_dependents;\n" ::: "memory");
  extern __shared__ unsigned char smem_raw[];
  unsigned char* const ring = smem_raw + (1024u - (smem_u32(smem_raw) & 1023u)) % 1024u;
  const Groups groups(reinterpret_cast<int*>(smem_raw + kOwnSmem), p.G);
  __shared__ __align__(8) uint64_t full[kRing];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t4 = lane & 3, me = blockIdx.x * kOwnWarps + warp;
  if (tid == 0) {
    for (int i = 0; i < kRing; ++i) mbar_init(smem_u32(full + i), 1);
    asm volatile("fence.mbarrier_init.release.cluster;\n" ::: "memory");
  }
  const bool sound_groups = read_groups(p, groups);
  asm volatile("griddepcontrol.wait;\n" ::: "memory");  // for attn_tile_kernel; attn_join_kernel waits for both by waiting for this one
  if (lane == 0) p.own_jobs[me].t = -1;
  if (!sound_groups) {
    if (me == 0 && lane == 0) {
      atomicExch(p.status, 6);
      p.tile_list[0] = 0;
    }
    return;
  }
  __syncwarp();
  if (me == 0) {  // the CTAs of attn_tile_kernel that left a job, and how many in front: attn_join_kernel begins with them
    int n = 0;
    for (int c0 = 0; c0 < p.tile_ctas; c0 += 32) {
      const int c = c0 + lane;
      const unsigned with = __ballot_sync(0xffffffffu, c < p.tile_ctas && p.tile_jobs[min(c, p.tile_ctas - 1)].tokens > 0);
      if ((with >> lane) & 1u) p.tile_list[1 + n + __popc(with & ((1u << lane) - 1u))] = c;
      n += __popc(with);
    }
    if (lane == 0) p.tile_list[0] = n;
  }
  // rows that attend nothing
  for (int t0 = 32 * me; t0 < p.T; t0 += 32 * p.own_warps) {
    const Row r = row_of(p, groups, min(t0 + lane, p.T - 1));
    for (unsigned empty = __ballot_sync(0xffffffffu, t0 + lane < p.T && r.table_row >= 0 && r.len == 0); empty != 0; empty &= empty - 1)
      for (int hq = 0; hq < p.Hq; ++hq) store4(p, t0 + __ffs(empty) - 1, hq, 4 * lane, make_float4(0.f, 0.f, 0.f, 0.f));
  }
  const long long all = p.unit_first[p.T] * p.Hkv, q = own_share(p), u0 = min(all, me * q), u1 = min(all, u0 + q);
  unsigned char* const slot0 = ring + (size_t)(warp * kDepth) * kSlotBytes;
  const uint32_t slots = smem_u32(slot0), bars = smem_u32(full + warp * kDepth);
  float (*const sm_o)[kHDP] = reinterpret_cast<float (*)[kHDP]>(slot0);  // the warp's sums, when its slots are free
  const int krow = lane & 15, kc = lane >> 4, vrow = 16 + (lane & 7) + (lane >> 4) * 8, vc = (lane >> 3) & 1;
  const float sc = p.scale * kLog2e, cap2 = 2.f * kLog2e * p.scale / p.softcap, cap = p.softcap * kLog2e;
  int slot = 0;
  uint32_t ph = 0;
  bool failed = false;
  int t = -1, h = 0;
  long long pair0 = 0;  // units before the pair
  Row row;
  for (long long u = u0; u < u1 && !failed;) {
    if (t >= 0 && h + 1 < p.Hkv) {  // the last pair is done
      ++h;
    } else {
      // the row of unit u: unit_first[t] Hkv <= u < unit_first[t + 1] Hkv, 32 samples at a time
      t = 0;
      for (int hi = p.T; hi - t > 1;) {
        const int step = (hi - t + 31) / 32, at = min(t + (lane + 1) * step, hi);
        const unsigned beyond = __ballot_sync(0xffffffffu, p.unit_first[at] * p.Hkv > u);  // (the last one is)
        const int k = __ffs(beyond) - 1;
        hi = min(t + (k + 1) * step, hi);
        t += k * step;
      }
      row = row_of(p, groups, t);
      const long long at = p.unit_first[t] * p.Hkv;
      h = (int)divided(u - at, units_of(row));
      pair0 = at + (long long)h * units_of(row);
    }
    const long long end = min(u1, pair0 + units_of(row));
    const int past = max((int)(u - pair0) - kStart, 0), nw = (int)(end - pair0) - kStart - past, first = row.page0 + past;
    const bool begins = past == 0, ends = end == pair0 + units_of(row);
    if (nw <= 0) {  // what a start costs, and no page
      u = end;
      continue;
    }

    const int32_t* const ids = p.table + (size_t)row.table_row * p.max_pages + first;
    auto page_id = [&](int n) { return n < nw ? ids[n] : -1; };
    int pid_cur = page_id(lane), pid_next = page_id(32 + lane);
    auto fetch = [&](int n, int base, int s) {  // page n of the piece; base: the first page that pid_cur holds
      const int pj = __shfl_sync(0xffffffffu, n - base < 32 ? pid_cur : pid_next, n & 31);
      if (lane == 0) {
        if ((unsigned)pj >= (unsigned)p.pool_pages) {  // malformed page table: record, hand over an empty slot
          atomicExch(p.status, 1);
          mbar_arrive(bars + 8u * s);
        } else {
          mbar_expect_tx(bars + 8u * s, kSlotBytes);
          page_g2s(slots + (uint32_t)s * kSlotBytes, &kvmap, (pj * p.Hkv + h) * 32, bars + 8u * s);
        }
      }
    };
    for (int n = 0; n < kDepth && n < nw; ++n) fetch(n, 0, (slot + n) % kDepth);
    uint32_t qb[8][2];  // column g = query head h * grp + g (zero columns from grp on)
#pragma unroll
    for (int j = 0; j < 8; ++j) qb[j][0] = qb[j][1] = 0u;
    if (g < p.grp) {
      const uint32_t* qp = reinterpret_cast<const uint32_t*>(p.q + (size_t)t * p.ldq + ((size_t)h * p.grp + g) * kHD);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        qb[j][0] = qp[8 * j + t4];
        qb[j][1] = qp[8 * j + 4 + t4];
      }
    }
    float m_run[2] = {-INFINITY, -INFINITY}, l_run[2] = {0.f, 0.f};  // query heads 2 t4 and 2 t4 + 1 of the group
    float o[8][4];  // O^T: tile j, rows d = 16 j + g and + 8, columns = the lane's two heads
#pragma unroll
    for (int j = 0; j < 8; ++j)
#pragma unroll
      for (int i = 0; i < 4; ++i) o[j][i] = 0.f;
    for (int n = 0; n < nw; ++n) {
      if ((n & 31) == 0 && n > 0) {
        pid_cur = pid_next;
        pid_next = page_id(n + 32 + lane);
      }
      if (!failed) failed = !__all_sync(0xffffffffu, mbar_wait(bars + 8u * slot, ph));
      const bool sound = (unsigned)__shfl_sync(0xffffffffu, pid_cur, n & 31) < (unsigned)p.pool_pages;
      if (sound && !failed) {
        const uint32_t kv = slots + (uint32_t)slot * kSlotBytes;
        float sa[2][4];
#pragma unroll
        for (int i = 0; i < 4; ++i) sa[0][i] = sa[1][i] = 0.f;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          uint32_t ka[4];
          ldsm4(kv + chunk_at(krow, 2 * j + kc), ka);
          mma16816(sa[j & 1], ka, qb[j][0], qb[j][1]);
        }
        // log2 domain; lane: tokens g (i < 2) and g + 8, heads 2 t4 and 2 t4 + 1
        const int tok0 = (first + n) * kPage;
        const bool edge = tok0 + kPage > row.len || tok0 < row.win0;
        float sv[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          float x = sa[0][i] + sa[1][i];
          x = p.softcap > 0.f ? capped_f32(x, cap2, cap) : x * sc;
          if (edge) {
            const int tok = tok0 + g + (i >> 1) * 8;
            if (tok >= row.len || tok < row.win0) x = -INFINITY;
          }
          sv[i] = x;
        }
        float mx[2] = {fmaxf(sv[0], sv[2]), fmaxf(sv[1], sv[3])}, alpha[2], off[2];
#pragma unroll
        for (int o2 = 4; o2 <= 16; o2 <<= 1) {
          mx[0] = fmaxf(mx[0], __shfl_xor_sync(0xffffffffu, mx[0], o2));
          mx[1] = fmaxf(mx[1], __shfl_xor_sync(0xffffffffu, mx[1], o2));
        }
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const float m_new = fmaxf(m_run[i], mx[i]);
          alpha[i] = m_new == -INFINITY ? 1.f : ex2(m_run[i] - m_new);  // scores of minus infinity so far: weights of zero
          m_run[i] = m_new;
          off[i] = m_new == -INFINITY ? 0.f : m_new - kHigh;
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) sv[i] = ex2(sv[i] - off[i & 1]);
        l_run[0] = l_run[0] * alpha[0] + (sv[0] + sv[2]);
        l_run[1] = l_run[1] * alpha[1] + (sv[1] + sv[3]);
        if (__any_sync(0xffffffffu, alpha[0] != 1.0f || alpha[1] != 1.0f)) {
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            o[j][0] *= alpha[0]; o[j][1] *= alpha[1];
            o[j][2] *= alpha[0]; o[j][3] *= alpha[1];
          }
        }
        uint32_t hi2[2], lo2[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          hi2[i] = pack_h2(sv[2 * i], sv[2 * i + 1]);
          const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&hi2[i]));
          lo2[i] = transpose8x8(pack_h2(sv[2 * i] - f.x, sv[2 * i + 1] - f.y));
          hi2[i] = transpose8x8(hi2[i]);
        }
        // V rows that are not attended are zeroed (their weight is 0, but 0 * garbage may be NaN)
        uint32_t keep[2] = {0xffffffffu, 0xffffffffu};
        if (edge) {
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const int tok = tok0 + 8 * i + 2 * t4;
            keep[i] = (tok < row.len && tok >= row.win0 ? 0xffffu : 0u) | (tok + 1 < row.len && tok + 1 >= row.win0 ? 0xffff0000u : 0u);
          }
        }
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          uint32_t va[4];
          ldsm4_t(kv + chunk_at(vrow, 2 * j + vc), va);
          if (edge) {
            va[0] &= keep[0]; va[1] &= keep[0];
            va[2] &= keep[1]; va[3] &= keep[1];
          }
          // a page's values by themselves: the MMAs cut what they add to, which would show after some dozens
          float d[4] = {0.f, 0.f, 0.f, 0.f};
          mma16816(d, va, hi2[0], hi2[1]);
          mma16816(d, va, lo2[0], lo2[1]);
#pragma unroll
          for (int i = 0; i < 4; ++i) o[j][i] += d[i];
        }
      }
      __syncwarp();
      if (n + kDepth < nw && !failed) fetch(n + kDepth, n & ~31, slot);
      if (++slot == kDepth) { slot = 0; ph ^= 1u; }
    }
    if (failed) break;

    // ---- the piece's sums, a head's together: the slots are free
#pragma unroll
    for (int i = 0; i < 2; ++i) {
#pragma unroll
      for (int o2 = 4; o2 <= 16; o2 <<= 1) l_run[i] += __shfl_xor_sync(0xffffffffu, l_run[i], o2);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        sm_o[2 * t4 + i][16 * j + g] = o[j][i];
        sm_o[2 * t4 + i][16 * j + 8 + g] = o[j][2 + i];
      }
    }
    __syncwarp();
    const bool whole = begins && ends;
    int c0 = 0, c1 = 0;
    const bool shared = shared_ctas(p, groups, row, t, h, c0, c1);
    if (begins && !ends && !(shared && c0 != c1) && lane == 0) {  // cut, and no tile's job: attn_join_kernel adds the pieces
      qeng_own_job& job = p.own_jobs[me];
      job.t = t;
      job.h = h;
      job.last = (int)divided(pair0 + units_of(row) - 1, q);
      job.shared = shared;
    }
    for (int hh = 0; hh < p.grp; ++hh) {
      float M = __shfl_sync(0xffffffffu, hh & 1 ? m_run[1] : m_run[0], hh >> 1) - kHigh;
      float L = __shfl_sync(0xffffffffu, hh & 1 ? l_run[1] : l_run[0], hh >> 1);
      float4 O = *reinterpret_cast<const float4*>(&sm_o[hh][4 * lane]);
      const int hq = h * p.grp + hh;
      if (whole && !(shared && c0 != c1)) {
        const size_t place = (size_t)t * p.Hq + hq;
        if (shared) add_sums(lane, lane == 0, reinterpret_cast<const float2*>(p.row_ml) + place, p.row_o + place * kHD, M, L, O);
        const float inv = 1.f / L;
        store4(p, t, hq, 4 * lane, make_float4(O.x * inv, O.y * inv, O.z * inv, O.w * inv));
      } else {  // whole: a tile's job adds it to the pieces of the shared pages
        float* const o_at = whole ? p.row_o : p.cut_o;
        float* const ml_at = whole ? p.row_ml : p.cut_ml;
        const size_t place = whole ? (size_t)t * p.Hq + hq : (size_t)(2 * me + (begins ? 1 : 0)) * 8 + hh;
        reinterpret_cast<float4*>(o_at + place * kHD)[lane] = O;
        if (lane == 0) reinterpret_cast<float2*>(ml_at)[place] = make_float2(M, L);
      }
    }
    asm volatile("fence.proxy.async.shared::cta;\n" ::: "memory");  // the slots are written by copies again
    __syncwarp();
    u = end;
    pair0 = end;
  }
  if (failed) {
    if (lane == 0) atomicExch(p.status, 4);
    grace();
  }
}

// ---- what was cut: a CTA of attn_tile_kernel left a job for the double tile (and kv head) that it ends with, a warp of
// attn_own_kernel for its last (row, kv head).  A tile's job also takes its rows' own sums, cut or whole.
// Bound by the latency of its loads: 5 to 13 us.  80 registers hold four pieces on their way; 64 for one more CTA took a call of 64 rows
// behind 16384 tokens from 80 to 85 us, 128 for eight pieces one of seven prompts from 395 to 409.
constexpr int kJoinWarps = 8, kJoinParts = 16;  // CTAs to a tile's job: a warp has eight of its 256 rows and a quarter of their dims

__global__ void __launch_bounds__(kJoinWarps * 32, 3) attn_join_kernel(const qeng_shared_attn p) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  asm volatile("griddepcontrol.wait;\n" ::: "memory");
  if (blockIdx.x < p.tile_ctas * kJoinParts) {
    // Lane: row lane % 8 of the warp's eight; for the weights every fourth piece, for the values dims 32 (warp % 4) + 4 (lane / 8) + 16 k.
    const int index = blockIdx.x / kJoinParts;
    if (index >= p.tile_list[0]) return;
    const int cta = p.tile_list[1 + index], part = blockIdx.x % kJoinParts * kJoinWarps + warp, four = lane >> 3, c0 = 8 * (part & 3) + four;
    const qeng_tile_job job = p.tile_jobs[cta];
    const int r = (part >> 2) * 8 + (lane & 7), x = r >> 7, i = (r & 127) / p.grp, hh = (r & 127) - i * p.grp, at = x * p.tokens + i;
    const bool mine = i < p.tokens && at < job.tokens;
    if (!__any_sync(0xffffffffu, mine)) return;
    const int t = mine ? job.t0 + at : job.t0, hq = job.h * p.grp + (mine ? hh : 0);
    const long long u = p.unit_first[t], units = p.unit_first[t + 1] - u, q = own_share(p);
    const bool live = mine && table_row_of(p, t) >= 0 && len_of(p, t) > 0;
    int e0 = 0, own = 0;  // warps with pieces of the row's own pages
    if (units > 0) {
      const long long y = u * p.Hkv + job.h * units;
      e0 = (int)divided(y + kStart, q);
      own = (int)divided(y + units - 1, q) - e0 + 1;
    }
    const int shared = job.last - cta + 1;  // pieces of the shared pages, two at least
    const size_t place = (size_t)t * p.Hq + hq;
    // The first CTA (or warp) ends with what is cut, the others begin with it: the first piece, then those of every second slot.
    struct Pieces {
      const float2* ml;
      const float4* o;
      int ml_step, o_step;
    };
    const float2* const tile_ml = reinterpret_cast<const float2*>(p.tile_ml) + r;
    const float4* const tile_o = reinterpret_cast<const float4*>(p.tile_o) + r + 256 * c0;
    const float2* const cut_ml = reinterpret_cast<const float2*>(p.cut_ml) + hh;
    const float4* const cut_o = reinterpret_cast<const float4*>(p.cut_o) + hh * 32 + c0;
    const Pieces first = {tile_ml + (size_t)(2 * cta + 1) * 256, tile_o + (size_t)(2 * cta + 1) * 8192, 0, 0};
    const Pieces rest = {tile_ml + (size_t)(2 * cta + 2) * 256, tile_o + (size_t)(2 * cta + 2) * 8192, 512, 16384};
    const Pieces own_first = own == 1 ? Pieces{reinterpret_cast<const float2*>(p.row_ml) + place, reinterpret_cast<const float4*>(p.row_o) + place * 32 + c0, 0, 0}
                                      : Pieces{cut_ml + (size_t)(2 * e0 + 1) * 8, cut_o + (size_t)(2 * e0 + 1) * 256, 0, 0};
    const Pieces own_rest = {cut_ml + (size_t)(2 * e0 + 2) * 8, cut_o + (size_t)(2 * e0 + 2) * 256, 16, 512};
    float M = first.ml->x;
    if (own > 0) M = fmaxf(M, own_first.ml->x);
    const auto most = [&](const Pieces& a, int n) {  // every fourth piece
#pragma unroll 4
      for (int k = four; k < n; k += 4) M = fmaxf(M, a.ml[k * a.ml_step].x);
    };
    most(rest, shared - 1);
    most(own_rest, own - 1);
    M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, 8));
    M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, 16));
    float L = 0.f;
    float4 O[2] = {make_float4(0.f, 0.f, 0.f, 0.f), make_float4(0.f, 0.f, 0.f, 0.f)};
    const auto add = [&](float2 ml, const float4& v, const float4& w) {
      // (m, l) = (-inf, NaN): scores of NaN alone; (-inf, 0): nothing attended, or scores of minus infinity alone
      const bool any = ml.x != -INFINITY;
      const float f = any ? ex2(ml.x - M) : 0.f;
      L = any ? fmaf(ml.y, f, L) : L + ml.y;
      O[0].x = fmaf(v.x, f, O[0].x); O[0].y = fmaf(v.y, f, O[0].y); O[0].z = fmaf(v.z, f, O[0].z); O[0].w = fmaf(v.w, f, O[0].w);
      O[1].x = fmaf(w.x, f, O[1].x); O[1].y = fmaf(w.y, f, O[1].y); O[1].z = fmaf(w.z, f, O[1].z); O[1].w = fmaf(w.w, f, O[1].w);
    };
    const auto add_all = [&](Pieces a, int n, int four_dims) {  // four pieces at a time, their loads in front
      for (; n > 0; n -= 4) {
        float2 ml[4];
        float4 v[4], w[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const bool more = k < n;  // (behind the last one: no weight)
          ml[k] = more ? __ldcg(a.ml) : make_float2(-INFINITY, 0.f);
          v[k] = more ? __ldcg(a.o) : make_float4(0.f, 0.f, 0.f, 0.f);
          w[k] = more ? __ldcg(a.o + four_dims) : make_float4(0.f, 0.f, 0.f, 0.f);
          a.ml += a.ml_step;
          a.o += a.o_step;
        }
#pragma unroll
        for (int k = 0; k < 4; ++k) add(ml[k], v[k], w[k]);
      }
    };
    const float2 ml0 = *first.ml, ml1 = *own_first.ml;
    const float4 v0 = first.o[0], w0 = first.o[1024], v1 = own_first.o[0], w1 = own_first.o[4];
    add_all(rest, shared - 1, 1024);
    add_all(own_rest, own - 1, 4);
    add(ml0, v0, w0);
    if (own > 0) add(ml1, v1, w1);
    const float inv = 1.f / L;
#pragma unroll
    for (int k = 0; k < 2; ++k)
      if (live) store4(p, t, hq, 4 * c0 + 16 * k, make_float4(O[k].x * inv, O[k].y * inv, O[k].z * inv, O[k].w * inv));
  } else {
    const int me = (blockIdx.x - p.tile_ctas * kJoinParts) * kJoinWarps + warp;
    if (me >= p.own_warps) return;
    const qeng_own_job job = p.own_jobs[me];
    if (job.t < 0) return;
    for (int hh = 0; hh < p.grp; ++hh) {
      float M = -INFINITY, L = 0.f;
      float4 O = make_float4(0.f, 0.f, 0.f, 0.f);
      add_pieces(lane, me, job.last, p.cut_o, p.cut_ml, 8, hh, M, L, O);
      const int hq = job.h * p.grp + hh;
      const size_t place = (size_t)job.t * p.Hq + hq;
      if (job.shared) add_sums(lane, lane == 0, reinterpret_cast<const float2*>(p.row_ml) + place, p.row_o + place * kHD, M, L, O);
      const float inv = 1.f / L;
      store4(p, job.t, hq, 4 * lane, make_float4(O.x * inv, O.y * inv, O.z * inv, O.w * inv));
    }
  }
}

}  // namespace

// tensor maps of half a page's K or V (16 rows of 64 dims) and of half the queries of a tile ([tokens][grp] rows of 64 dims)
static int32_t tile_maps(qeng_ctx* ctx, const qeng_shared_attn& p, CUtensorMap* kv, CUtensorMap* q) {
  auto enc = reinterpret_cast<decltype(&cuTensorMapEncodeTiled)>(qeng_tensor_map_encoder());
  const cuuint32_t es[3] = {1, 1, 1};
  const cuuint64_t kdims[3] = {64, (cuuint64_t)p.pool_pages * p.Hkv * 32, 2}, kstrides[2] = {256, 128};
  const cuuint32_t kbox[3] = {64, kPage, 1};
  const cuuint64_t qdims[3] = {kHD, (cuuint64_t)p.Hq, (cuuint64_t)p.T}, qstrides[2] = {kHD * 2, (cuuint64_t)p.ldq * 2};
  const cuuint32_t qbox[3] = {64, (cuuint32_t)p.grp, (cuuint32_t)p.tokens};
  if (!enc ||
      enc(kv, CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 3, p.pool, kdims, kstrides, kbox, es, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
          CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) != CUDA_SUCCESS ||
      enc(q, CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 3, const_cast<__half*>(p.q), qdims, qstrides, qbox, es, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
          CU_TENSOR_MAP_L2_PROMOTION_L2_128B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) != CUDA_SUCCESS)
    return qeng_fail(ctx, QENG_ERR_CUDA, "attn_shared: tensor maps rejected");
  return QENG_OK;
}

extern "C" int32_t qeng_attn_shared(qeng_ctx* ctx, const qeng_kv_pool* pool, const uint16_t* q_f16, int64_t ldq, const int32_t* page_table, int64_t max_pages,
                                    int64_t table_rows, const int32_t* rows, const int32_t* lens, int64_t T, int64_t Hq, const int32_t* group_first,
                                    const int32_t* group_pages, int64_t G, float scale, float softcap, int32_t window, void* out, int32_t out_dtype,
                                    int64_t ldo, void* stream) {
  if (!ctx || !pool || !q_f16 || !page_table || !lens || !group_first || !group_pages || !out) return qeng_fail(ctx, QENG_ERR_ARG, "attn_shared: null argument");
  if (T <= 0 || Hq <= 0 || max_pages <= 0 || table_rows <= 0 || G <= 0) return qeng_fail(ctx, QENG_ERR_ARG, "attn_shared: T, Hq, G and the table's sizes must be positive");
  if (!(scale >= 0.f) || !(softcap >= 0.f) || window < 0) return qeng_fail(ctx, QENG_ERR_ARG, "attn_shared: scale, softcap and window must not be negative");
  if (softcap > 1e30f || (softcap > 0.f && !isfinite(2.f * kLog2e * scale / softcap)))
    return qeng_fail(ctx, QENG_ERR_ARG, "attn_shared: softcap of %g with a scale of %g leaves 32 bits", softcap, scale);
  if (out_dtype < QENG_F32 || out_dtype > QENG_BF16) return qeng_fail(ctx, QENG_ERR_ARG, "attn_shared: unknown type %d", out_dtype);
  if (Hq % pool->kv_heads != 0 || Hq / pool->kv_heads > 8)
    return qeng_fail(ctx, QENG_ERR_SHAPE, "attn_shared: query heads per kv head must divide evenly and be <= 8");
  if (G > kSharedGroups || T * Hq > (1 << 21) || max_pages > (1 << 26) || table_rows > (1 << 30) || pool->pages * pool->kv_heads >= (1 << 26))
    return qeng_fail(ctx, QENG_ERR_SHAPE, "attn_shared: at most %d groups, 2^21 rows times heads, less than 2^26 pages times kv heads", kSharedGroups);
  if (!rows && table_rows < T) return qeng_fail(ctx, QENG_ERR_SHAPE, "attn_shared: a table of %lld rows for %lld without their rows", (long long)table_rows, (long long)T);
  const int grp = (int)(Hq / pool->kv_heads), tokens = 128 / grp;
  const int64_t tiles = (T + 2 * tokens - 1) / (2 * tokens) + (G < T ? G : T);  // at most
  if (tiles > kSharedTiles || (max_pages / 8 + 2) * tiles * pool->kv_heads > 0x7fffffff)
    return qeng_fail(ctx, QENG_ERR_SHAPE, "attn_shared: rows / %d + groups exceed %d, or those times kv heads and pages 2^34", 2 * tokens, kSharedTiles);
  if (ldq < Hq * kHD || ldo < Hq * kHD) return qeng_fail(ctx, QENG_ERR_SHAPE, "attn_shared: rows of %lld and %lld values hold less than %lld heads", (long long)ldq, (long long)ldo, (long long)Hq);
  if (((reinterpret_cast<uintptr_t>(q_f16) | reinterpret_cast<uintptr_t>(out)) & 15) != 0 || ldq % 8 != 0 || ldo % (out_dtype == QENG_F32 ? 4 : 8) != 0)
    return qeng_fail(ctx, QENG_ERR_ALIGN, "attn_shared: rows of q and out must be 16-byte aligned");
  QENG_ENTER(ctx);
  const cudaStream_t st = (cudaStream_t)stream;
  static bool configured_on[64] = {};  // the opt-in shared-memory size is set per device
  bool& configured = configured_on[ctx->device & 63];
  if (!configured) {
    for (auto* const fn : {attn_tile_kernel<false, false>, attn_tile_kernel<false, true>, attn_tile_kernel<true, true>})
      QENG_CUDA(ctx, cudaFuncSetAttribute(fn, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)(kTileSmem + groups_bytes(kSharedGroups))));
    QENG_CUDA(ctx, cudaFuncSetAttribute(attn_own_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)(kOwnSmem + groups_bytes(kSharedGroups))));
    configured = true;
  }
  qeng_shared_attn p;
  p.q = reinterpret_cast<const __half*>(q_f16); p.ldq = ldq; p.table = page_table; p.max_pages = max_pages; p.table_rows = table_rows;
  p.rows = rows; p.lens = lens; p.first = group_first; p.pages = group_pages; p.out = out; p.ldo = ldo; p.out_dtype = out_dtype; p.status = ctx->status;
  p.pool = pool->data; p.T = (int)T; p.Hq = (int)Hq; p.Hkv = (int)pool->kv_heads; p.grp = grp; p.tokens = tokens; p.G = (int)G; p.pool_pages = (int)pool->pages;
  p.window = window; p.softcap = softcap;
  p.scale = scale > 0.f ? scale : 1e-30f;  // nothing, but a masked score (minus infinity) stays what it is
  p.own_warps = 3 * ctx->sm_count * kOwnWarps;
  p.tile_ctas = ctx->sm_count;
  CUtensorMap map, tile_map, q_map;
  int32_t rc = qeng_kv_map(ctx, pool->data, pool->pages * pool->kv_heads * 32, &map);
  if (rc != QENG_OK) return rc;
  rc = tile_maps(ctx, p, &tile_map, &q_map);
  if (rc != QENG_OK) return rc;
  qeng_scratch* sc = qeng_scratch_for(ctx, st);
  // tile_first, tile_o, tile_ml, row_o, row_ml, unit_first, cut_o, cut_ml, jobs
  const size_t cut = (size_t)2 * p.tile_ctas * 256, rows_heads = (size_t)T * Hq, own = (size_t)2 * p.own_warps * 8;
  const size_t need[12] = {(size_t)(tiles + 1) * 4, cut * kHD * 4, cut * 8, rows_heads * kHD * 4, rows_heads * 8, ((size_t)T + 1) * 8, own * kHD * 4, own * 8,
                           p.tile_ctas * sizeof(qeng_tile_job), p.own_warps * sizeof(qeng_own_job),
                           (size_t)(1 + p.tile_ctas) * 4, out_dtype == QENG_F32 ? (size_t)p.tile_ctas * 256 * kHD * 4 : 0};
  size_t at[13] = {0};
  for (int i = 0; i < 12; ++i) at[i + 1] = at[i] + ((need[i] + 255) & ~(size_t)255);
  rc = qeng_scratch_grow(ctx, sc, &sc->shared, at[12]);
  if (rc != QENG_OK) return rc;
  unsigned char* const mem = static_cast<unsigned char*>(sc->shared.ptr);
  p.tile_first = reinterpret_cast<int*>(mem);
  p.tile_o = reinterpret_cast<float*>(mem + at[1]);
  p.tile_ml = reinterpret_cast<float*>(mem + at[2]);
  p.row_o = reinterpret_cast<float*>(mem + at[3]);
  p.row_ml = reinterpret_cast<float*>(mem + at[4]);
  p.unit_first = reinterpret_cast<long long*>(mem + at[5]);
  p.cut_o = reinterpret_cast<float*>(mem + at[6]);
  p.cut_ml = reinterpret_cast<float*>(mem + at[7]);
  p.tile_jobs = reinterpret_cast<qeng_tile_job*>(mem + at[8]);
  p.own_jobs = reinterpret_cast<qeng_own_job*>(mem + at[9]);
  p.tile_list = reinterpret_cast<int*>(mem + at[10]);
  p.kept_o = reinterpret_cast<float*>(mem + at[11]);
  auto* const tile_kernel = out_dtype == QENG_F32 ? attn_tile_kernel<true, true> : softcap > kCoarseCap ? attn_tile_kernel<false, true> : attn_tile_kernel<false, false>;
  tile_kernel<<<(unsigned)p.tile_ctas, kTileThreads, kTileSmem + groups_bytes(G), st>>>(p, tile_map, q_map);
  QENG_LAUNCH_CHECK(ctx);
  // the other two may start as CTAs of the one in front leave
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.stream = st;
  cfg.attrs = attr;
  cfg.numAttrs = ctx->pdl ? 1 : 0;
  cfg.gridDim = dim3((unsigned)(p.own_warps / kOwnWarps));
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = kOwnSmem + groups_bytes(G);
  QENG_CUDA(ctx, cudaLaunchKernelEx(&cfg, attn_own_kernel, p, map));
  cfg.gridDim = dim3((unsigned)(p.tile_ctas * kJoinParts + (p.own_warps + kJoinWarps - 1) / kJoinWarps));
  cfg.blockDim = dim3(kJoinWarps * 32);
  cfg.dynamicSmemBytes = 0;
  QENG_CUDA(ctx, cudaLaunchKernelEx(&cfg, attn_join_kernel, p));
  return QENG_OK;
}
