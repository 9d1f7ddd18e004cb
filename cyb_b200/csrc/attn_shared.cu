// Attention of rows (one query token each) over the paged f16 KV cache, where the rows of a group share their first pages: decode
// batches behind one prompt, or the tokens of a prompt (a group whose rows share all pages and differ in length).
//
// Two kernels: attn_own_kernel reads the pages that a row has to itself, attn_join_kernel adds up what several CTAs found of a row.
// Sums travel as (log2 of the largest weight m, sum l of 2^(x - m), sum of 2^(x - m) v): two of them add up after scaling by
// 2^(m - max).
#include <cuda_bf16.h>
#include <math.h>

#include "attn_shared.h"

namespace {

constexpr int kHD = 128, kPage = 16;
constexpr int kThreads = kOwnWarps * 32, kDepth = 2, kRing = kDepth * kOwnWarps;  // pages of a warp on their way
constexpr uint32_t kSlotBytes = 2 * kPage * kHD * 2;
constexpr int kHDP = kHD + 4;  // row stride of the warps' sums in shared memory: no bank conflicts
constexpr size_t kOwnSmem = kRing * kSlotBytes + 1024;
constexpr float kLog2e = 1.4426950408889634f;
// The largest weight of a row is 2^kHigh: the smallest that a f16 number holds at full precision is then 2^-22 of it.
constexpr float kHigh = 8.f;

__device__ __forceinline__ uint32_t smem_u32(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }
__device__ __forceinline__ void mbar_init(uint32_t bar, uint32_t count) { asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;\n" ::"r"(bar), "r"(count)); }
__device__ __forceinline__ void mbar_arrive(uint32_t bar) { asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];\n" ::"r"(bar) : "memory"); }
__device__ __forceinline__ void mbar_expect_tx(uint32_t bar, uint32_t bytes) {
  asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;\n" ::"r"(bar), "r"(bytes) : "memory");
}
__device__ __forceinline__ bool mbar_try_wait(uint32_t bar, uint32_t parity) {
  uint32_t ok;
  asm volatile("{\n .reg .pred p;\n mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n selp.u32 %0, 1, 0, p;\n}\n" : "=r"(ok) : "r"(bar), "r"(parity) : "memory");
  return ok != 0;
}
// Bounded wait: gives up (false) two seconds after the first failed attempt.
__device__ __noinline__ bool mbar_wait_slow(uint32_t bar, uint32_t parity) {
  unsigned long long t0, t1;
  asm volatile("mov.u64 %0, %globaltimer;\n" : "=l"(t0));
  do {
    for (int i = 0; i < 64; ++i)
      if (mbar_try_wait(bar, parity)) return true;
    asm volatile("mov.u64 %0, %globaltimer;\n" : "=l"(t1));
  } while (t1 - t0 <= 2000000000ull);
  return false;
}
__device__ __forceinline__ bool mbar_wait(uint32_t bar, uint32_t parity) { return mbar_try_wait(bar, parity) || mbar_wait_slow(bar, parity); }
// K and V of one (page, kv head): 32 rows as two halves of 64 dims, 128-byte swizzled
__device__ __forceinline__ void page_g2s(uint32_t dst, const CUtensorMap* map, int row, uint32_t bar) {
  asm volatile("cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];\n" ::"r"(dst), "l"(map), "r"(0),
               "r"(row), "r"(0), "r"(bar)
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
__device__ __forceinline__ uint32_t pack_h2(float a, float b) {
  const __half2 h = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
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

// ---- groups, rows and their units -----------------------------------------------------------------------------------------
struct Groups {
  int first[kSharedGroups + 1], pages[kSharedGroups];
};

// Reads the groups into shared memory; false in every thread where their bounds do not ascend within the call's rows.
__device__ __forceinline__ bool read_groups(const qeng_shared_attn& p, Groups& g) {
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
  return !__syncthreads_or(bad);
}

struct Row {
  int table_row, len, win0;  // table_row < 0: the row is not there
  int group;
  int page0, pages;          // its own pages: the first, how many
};

__device__ __forceinline__ Row row_of(const qeng_shared_attn& p, const Groups& g, int t) {
  Row r;
  r.table_row = -1;
  r.len = r.win0 = r.group = r.page0 = r.pages = 0;
  if (t < g.first[0] || t >= g.first[p.G]) return r;
  int lo = 0, hi = p.G;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (g.first[mid] <= t) lo = mid;
    else hi = mid;
  }
  r.group = lo;
  const int row = p.rows ? p.rows[t] : t;
  if (row < 0) return r;
  if (row >= p.table_rows) {
    atomicExch(p.status, 6);
    return r;
  }
  r.table_row = row;
  r.len = (int)min((long long)max(p.lens[t], 0), p.max_pages * kPage);
  r.win0 = p.window > 0 ? max(0, r.len - p.window) : 0;
  r.page0 = r.win0 / kPage;
  r.pages = max(0, (r.len + kPage - 1) / kPage - r.page0);
  return r;
}
__device__ __forceinline__ int units_of(const Row& r) { return (r.pages + kOwnWarps - 1) / kOwnWarps; }

// first CTA of `n` whose share of `all` units holds unit x, the shares beginning at c all / n
__device__ __forceinline__ int cta_of(long long x, long long all, int n) { return (int)(((x + 1) * n - 1) / all); }

// ---- a row's own pages ------------------------------------------------------------------------------------------------------
// A warp looks after the pages it reads, two on their way.  The query heads of the kv head are the eight columns of every MMA,
// S^T = K Q^T and O^T = V^T P^T; P in two f16 terms.
__global__ void __launch_bounds__(kThreads, 3) attn_own_kernel(const qeng_shared_attn p, const __grid_constant__ CUtensorMap kvmap) {
  extern __shared__ unsigned char smem_raw[];
  unsigned char* const ring = smem_raw + (1024u - (smem_u32(smem_raw) & 1023u)) % 1024u;
  __shared__ Groups groups;
  __shared__ __align__(8) uint64_t full[kRing];
  __shared__ long long before[kThreads + 1];  // units before the rows of a thread
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t4 = lane & 3, cta = blockIdx.x;
  if (tid == 0) {
    for (int i = 0; i < kRing; ++i) mbar_init(smem_u32(full + i), 1);
    asm volatile("fence.mbarrier_init.release.cluster;\n" ::: "memory");
  }
  if (!read_groups(p, groups)) {
    if (cta == 0 && tid == 0) atomicExch(p.status, 6);
    return;
  }
  // units of all rows: a thread adds up neighbouring rows
  const int per = (p.T + kThreads - 1) / kThreads;
  {
    long long n = 0;
    for (int t = tid * per; t < min((tid + 1) * per, p.T); ++t) n += units_of(row_of(p, groups, t));
    before[tid + 1] = n;
    if (tid == 0) before[0] = 0;
    __syncthreads();
    if (warp == 0) {
      long long sum = 0;
      for (int i = 0; i < kOwnWarps; ++i) {
        long long x = before[1 + i * 32 + lane];
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const long long y = __shfl_up_sync(0xffffffffu, x, o);
          if (lane >= o) x += y;
        }
        before[1 + i * 32 + lane] = sum + x;
        sum += __shfl_sync(0xffffffffu, x, 31);
      }
    }
    __syncthreads();
  }
  if (cta == 0) {  // for attn_join_kernel
    long long n = before[tid];
    for (int t = tid * per; t < min((tid + 1) * per, p.T); ++t) {
      p.unit_first[t] = n;
      n += units_of(row_of(p, groups, t));
    }
    if (tid == 0) p.unit_first[p.T] = before[kThreads];
  }
  const long long all = before[kThreads] * p.Hkv, u0 = all * cta / gridDim.x, u1 = all * (cta + 1) / gridDim.x;

  float (*const sm_o)[8][kHDP] = reinterpret_cast<float (*)[8][kHDP]>(ring);
  float (*const sm_m)[8] = reinterpret_cast<float (*)[8]>(ring + sizeof(float) * kOwnWarps * 8 * kHDP);
  float (*const sm_l)[8] = sm_m + kOwnWarps;
  const uint32_t slots = smem_u32(ring) + (uint32_t)(warp * kDepth) * kSlotBytes, bars = smem_u32(full + warp * kDepth);
  const int krow = lane & 15, kc = lane >> 4, vrow = 16 + (lane & 7) + (lane >> 4) * 8, vc = (lane >> 3) & 1;
  const float sc = p.scale * kLog2e;
  int slot = 0;
  uint32_t ph = 0;
  bool failed = false;
  for (long long u = u0; u < u1;) {
    // the pair of unit u: its rows' thread, then the row among that thread's, 32 at a time
    int lo = 0, hi = kThreads;
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (before[mid] * p.Hkv <= u) lo = mid;
      else hi = mid;
    }
    int t = lo * per;
    long long at = before[lo] * p.Hkv;  // units before row t
    Row row;
    for (;; t += 32) {
      const bool there = t + lane < min((lo + 1) * per, p.T);
      long long n = there ? units_of(row_of(p, groups, t + lane)) : 0;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const long long y = __shfl_up_sync(0xffffffffu, n, o);
        if (lane >= o) n += y;
      }
      const unsigned beyond = __ballot_sync(0xffffffffu, at + n * p.Hkv > u);
      if (beyond != 0) {
        const int k = __ffs(beyond) - 1;
        at += (k > 0 ? __shfl_sync(0xffffffffu, n, k - 1) : 0) * p.Hkv;
        t += k;
        break;
      }
      at += __shfl_sync(0xffffffffu, n, 31) * p.Hkv;
    }
    row = row_of(p, groups, t);
    const int units = units_of(row), h = (int)((u - at) / units);
    const long long pair0 = at + (long long)h * units;       // the pair's units: [pair0, pair0 + units)
    const long long end = min(u1, pair0 + units);
    const int first = row.page0 + (int)(u - pair0) * kOwnWarps, last = min(row.page0 + row.pages, row.page0 + (int)(end - pair0) * kOwnWarps);
    const bool begins = u == pair0, ends = end == pair0 + units;

    // ---- pages first + warp, + kOwnWarps, ...
    const int nw = last - first > warp ? (last - first - warp + kOwnWarps - 1) / kOwnWarps : 0;
    const int32_t* const ids = p.table + (size_t)row.table_row * p.max_pages + first + warp;
    auto page_id = [&](int n) { return n < nw ? ids[n * kOwnWarps] : -1; };
    int pid_cur = page_id(lane), pid_next = page_id(32 + lane);
    auto fetch = [&](int n, int base, int s) {  // page n of the warp; base: the first page that pid_cur holds
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
    for (int n = 0; n < kDepth && n < nw && !failed; ++n) fetch(n, 0, (slot + n) % kDepth);
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
        const int tok0 = (first + warp + kOwnWarps * n) * kPage;
        const bool edge = tok0 + kPage > row.len || tok0 < row.win0;
        float sv[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          float x = sa[0][i] + sa[1][i];
          if (p.softcap > 0.f) x = p.softcap * tanhf(x * p.scale / p.softcap) * kLog2e;
          else x *= sc;
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
          alpha[i] = m_new == -INFINITY ? 1.f : exp2f(m_run[i] - m_new);  // scores of minus infinity so far: weights of zero
          m_run[i] = m_new;
          off[i] = m_new == -INFINITY ? 0.f : m_new - kHigh;
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) sv[i] = exp2f(sv[i] - off[i & 1]);
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
          mma16816(o[j], va, hi2[0], hi2[1]);
          mma16816(o[j], va, lo2[0], lo2[1]);
        }
      }
      __syncwarp();
      if (n + kDepth < nw && !failed) fetch(n + kDepth, n & ~31, slot);
      if (++slot == kDepth) { slot = 0; ph ^= 1u; }
    }
    if (failed) grace();  // copies on their way land before their place is used

    // ---- the warps' sums: the ring becomes their place ----
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 2; ++i) {
#pragma unroll
      for (int o2 = 4; o2 <= 16; o2 <<= 1) l_run[i] += __shfl_xor_sync(0xffffffffu, l_run[i], o2);
      const int hh = 2 * t4 + i;
      if (hh < p.grp) {
        if (g == 0) {
          sm_m[warp][hh] = m_run[i];
          sm_l[warp][hh] = l_run[i];
        }
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          sm_o[warp][hh][16 * j + g] = o[j][i];
          sm_o[warp][hh][16 * j + 8 + g] = o[j][2 + i];
        }
      }
    }
    __syncthreads();
    const bool whole = begins && ends;
    for (int hh = warp; hh < p.grp; hh += kOwnWarps) {
      float M = -INFINITY;
#pragma unroll
      for (int w = 0; w < kOwnWarps; ++w) M = fmaxf(M, sm_m[w][hh]);
      float L = 0.f;
      float4 O = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
      for (int w = 0; w < kOwnWarps; ++w) {
        const float f = sm_m[w][hh] == -INFINITY ? 0.f : exp2f(sm_m[w][hh] - M);  // a warp without pages
        const float4 v = *reinterpret_cast<const float4*>(&sm_o[w][hh][4 * lane]);
        L += sm_l[w][hh] * f;
        O.x += v.x * f; O.y += v.y * f; O.z += v.z * f; O.w += v.w * f;
      }
      if (whole) {
        const float inv = 1.f / L;
        store4(p, t, h * p.grp + hh, 4 * lane, make_float4(O.x * inv, O.y * inv, O.z * inv, O.w * inv));
      } else {
        const size_t at2 = (size_t)(2 * cta + (begins ? 1 : 0)) * 8 + hh;
        reinterpret_cast<float4*>(p.cut_o + at2 * kHD)[lane] = O;
        if (lane == 0) reinterpret_cast<float2*>(p.cut_ml)[at2] = make_float2(M, L);
      }
    }
    asm volatile("fence.proxy.async.shared::cta;\n" ::: "memory");  // the ring is written by copies again
    __syncthreads();
    u = end;
  }
  if (__syncthreads_or(failed) && tid == 0) atomicExch(p.status, 4);
}

// ---- what is left of a row: sums of several CTAs, or nothing to attend --------------------------------------------------------
constexpr int kJoinWarps = 8;

__global__ void __launch_bounds__(kJoinWarps * 32) attn_join_kernel(const qeng_shared_attn p) {
  __shared__ Groups groups;
  const int t = blockIdx.x, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (!read_groups(p, groups)) return;
  const Row row = row_of(p, groups, t);
  if (row.table_row < 0) return;
  const long long u = p.unit_first[t], all = p.unit_first[p.T] * p.Hkv, units = p.unit_first[t + 1] - u;
  for (int hq = warp; hq < p.Hq; hq += kJoinWarps) {
    if (units == 0) {
      store4(p, t, hq, 4 * lane, make_float4(0.f, 0.f, 0.f, 0.f));
      continue;
    }
    const int h = hq / p.grp, hh = hq - h * p.grp;
    const long long x = u * p.Hkv + h * units;
    const int c0 = cta_of(x, all, p.own_ctas), c1 = cta_of(x + units - 1, all, p.own_ctas);
    if (c0 == c1) continue;
    float M = -INFINITY, L = 0.f;
    float4 O = make_float4(0.f, 0.f, 0.f, 0.f);
    const auto add = [&](const float* o, float2 ml) {
      if (ml.x == -INFINITY) {  // nothing attended, or scores of minus infinity alone: no weight
        L += ml.y;
        return;
      }
      const float m = fmaxf(M, ml.x), a = M == -INFINITY ? 0.f : exp2f(M - m), f = exp2f(ml.x - m);
      const float4 v = reinterpret_cast<const float4*>(o)[lane];
      M = m;
      L = L * a + ml.y * f;
      O.x = O.x * a + v.x * f; O.y = O.y * a + v.y * f; O.z = O.z * a + v.z * f; O.w = O.w * a + v.w * f;
    };
    for (int c = c0; c <= c1; ++c) {
      if (all * c / p.own_ctas == all * (c + 1) / p.own_ctas) continue;  // no units
      const size_t at = (size_t)(2 * c + (c == c0 ? 1 : 0)) * 8 + hh;  // the first CTA ends with the pair, the others begin with it
      add(p.cut_o + at * kHD, reinterpret_cast<const float2*>(p.cut_ml)[at]);
    }
    const float inv = 1.f / L;
    store4(p, t, hq, 4 * lane, make_float4(O.x * inv, O.y * inv, O.z * inv, O.w * inv));
  }
}

}  // namespace

extern "C" int32_t qeng_attn_shared(qeng_ctx* ctx, const qeng_kv_pool* pool, const uint16_t* q_f16, int64_t ldq, const int32_t* page_table, int64_t max_pages,
                                    int64_t table_rows, const int32_t* rows, const int32_t* lens, int64_t T, int64_t Hq, const int32_t* group_first,
                                    const int32_t* group_pages, int64_t G, float scale, float softcap, int32_t window, void* out, int32_t out_dtype,
                                    int64_t ldo, void* stream) {
  if (!ctx || !pool || !q_f16 || !page_table || !lens || !group_first || !group_pages || !out) return qeng_fail(ctx, QENG_ERR_ARG, "attn_shared: null argument");
  if (T <= 0 || Hq <= 0 || max_pages <= 0 || table_rows <= 0 || G <= 0) return qeng_fail(ctx, QENG_ERR_ARG, "attn_shared: T, Hq, G and the table's sizes must be positive");
  if (!(softcap >= 0.f) || window < 0) return qeng_fail(ctx, QENG_ERR_ARG, "attn_shared: softcap and window must not be negative");
  if (out_dtype < QENG_F32 || out_dtype > QENG_BF16) return qeng_fail(ctx, QENG_ERR_ARG, "attn_shared: unknown type %d", out_dtype);
  if (Hq % pool->kv_heads != 0 || Hq / pool->kv_heads > 8)
    return qeng_fail(ctx, QENG_ERR_SHAPE, "attn_shared: query heads per kv head must divide evenly and be <= 8");
  if (G > kSharedGroups || T * Hq > (1 << 21) || max_pages > (1 << 26) || table_rows > (1 << 30) || pool->pages * pool->kv_heads >= (1 << 26))
    return qeng_fail(ctx, QENG_ERR_SHAPE, "attn_shared: at most %d groups, 2^21 rows times heads, less than 2^26 pages times kv heads", kSharedGroups);
  if (!rows && table_rows < T) return qeng_fail(ctx, QENG_ERR_SHAPE, "attn_shared: a table of %lld rows for %lld without their rows", (long long)table_rows, (long long)T);
  if (ldq < Hq * kHD || ldo < Hq * kHD) return qeng_fail(ctx, QENG_ERR_SHAPE, "attn_shared: rows of %lld and %lld values hold less than %lld heads", (long long)ldq, (long long)ldo, (long long)Hq);
  if (((reinterpret_cast<uintptr_t>(q_f16) | reinterpret_cast<uintptr_t>(out)) & 15) != 0 || ldq % 8 != 0 || ldo % (out_dtype == QENG_F32 ? 4 : 8) != 0)
    return qeng_fail(ctx, QENG_ERR_ALIGN, "attn_shared: rows of q and out must be 16-byte aligned");
  QENG_ENTER(ctx);
  const cudaStream_t st = (cudaStream_t)stream;
  static bool configured_on[64] = {};  // the opt-in shared-memory size is set per device
  bool& configured = configured_on[ctx->device & 63];
  if (!configured) {
    QENG_CUDA(ctx, cudaFuncSetAttribute(attn_own_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)kOwnSmem));
    configured = true;
  }
  qeng_shared_attn p;
  p.q = reinterpret_cast<const __half*>(q_f16); p.ldq = ldq; p.table = page_table; p.max_pages = max_pages; p.table_rows = table_rows;
  p.rows = rows; p.lens = lens; p.first = group_first; p.pages = group_pages; p.out = out; p.ldo = ldo; p.out_dtype = out_dtype; p.status = ctx->status;
  p.T = (int)T; p.Hq = (int)Hq; p.Hkv = (int)pool->kv_heads; p.grp = (int)(Hq / pool->kv_heads); p.G = (int)G; p.pool_pages = (int)pool->pages;
  p.window = window; p.scale = scale; p.softcap = softcap;
  p.own_ctas = 3 * ctx->sm_count;
  CUtensorMap map;
  int32_t rc = qeng_kv_map(ctx, pool->data, pool->pages * pool->kv_heads * 32, &map);
  if (rc != QENG_OK) return rc;
  qeng_scratch* sc = qeng_scratch_for(ctx, st);
  const size_t units = ((size_t)T + 1) * 8, cut = (size_t)2 * p.own_ctas * 8;
  auto up = [](size_t x) { return (x + 255) & ~(size_t)255; };
  rc = qeng_scratch_grow(ctx, sc, &sc->shared, up(units) + up(cut * kHD * 4) + up(cut * 8));
  if (rc != QENG_OK) return rc;
  unsigned char* at = static_cast<unsigned char*>(sc->shared.ptr);
  p.unit_first = reinterpret_cast<long long*>(at);
  p.cut_o = reinterpret_cast<float*>(at += up(units));
  p.cut_ml = reinterpret_cast<float*>(at += up(cut * kHD * 4));
  p.own_o = p.own_ml = nullptr;
  attn_own_kernel<<<(unsigned)p.own_ctas, kThreads, kOwnSmem, st>>>(p, map);
  QENG_LAUNCH_CHECK(ctx);
  attn_join_kernel<<<(unsigned)T, kJoinWarps * 32, 0, st>>>(p);
  QENG_LAUNCH_CHECK(ctx);
  return QENG_OK;
}
