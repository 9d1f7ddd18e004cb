// What a server does to the paged KV cache between "these requests get so many more tokens" and the attention of the batch: pages
// and slots for the new tokens, and the append that writes through them.
//
// kv_plan_kernel: everything follows from three exclusive sums over the requests (tokens, pages taken, pages given back), which
// every CTA computes for itself in shared memory; a token or page finds its request by bisection there.  One CTA, or a cluster of up
// to eight where the buffers are long: lengths and counters may be updated in place, so nobody writes them before every CTA has read
// them, and a cluster's barrier is the cheapest place to wait for that.  Bound by latency: 64 requests 5.6 us, 1000 with 131072 places
// for tokens 13.6 us (2 MB written; 26 us before a page id was asked for once for four tokens, stores had 16 bytes and blocks grew with the call).
//
// rope_append_slots_kernel: HBM-bound, (Hq + 2 Hkv) * 128 values read and written as f16 once.  A CTA has a token; sixteen lanes have
// a head (the pairs (i, i + 64) of a lane are eight values: 16-byte loads of f32 rows).  8192 rows of 48 f32 heads:
// 49.5 us, 6.1 TB/s (57 with the slot asked for before the row).
#include <math.h>

#include "qeng_internal.h"

#include <cuda_bf16.h>

namespace {

constexpr int kHD = 128, kPage = 16;
constexpr int kPlanThreads = 1024, kPlanRequests = 8192;

struct PlanParams {
  const int32_t *lens, *add, *keep;
  int32_t* table;
  int32_t* ring;
  const int64_t* ends;  // [2]: pages taken from the ring and given to it since the beginning
  int32_t* lens_out;
  int64_t* ends_out;
  int32_t *starts, *slots, *pos, *seen, *rows;
  int32_t* status;
  int R, capacity, pages, ctas;
  bool whole4;  // the tokens' arrays take 16-byte stores
  long long max_pages, ring_size;
};

__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.release.aligned;\n" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire.aligned;\n" ::: "memory"); }

// exclusive sums of three values over the block's threads; totals in tot
__device__ __forceinline__ void scan3(long long (&v)[3], long long (&tot)[3], long long (*warps)[32]) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, nw = blockDim.x >> 5;
  long long own[3];
#pragma unroll
  for (int i = 0; i < 3; ++i) {
    own[i] = v[i];
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const long long x = __shfl_up_sync(0xffffffffu, v[i], o);
      if (lane >= o) v[i] += x;
    }
    if (lane == 31) warps[i][warp] = v[i];
  }
  __syncthreads();
  if (warp < 3) {  // (four warps at least)
    long long x = lane < nw ? warps[warp][lane] : 0;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const long long y = __shfl_up_sync(0xffffffffu, x, o);
      if (lane >= o) x += y;
    }
    warps[warp][lane] = x;
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < 3; ++i) {
    v[i] = v[i] - own[i] + (warp > 0 ? warps[i][warp - 1] : 0);
    tot[i] = warps[i][31];
  }
  __syncthreads();  // `warps` may be written again
}

// of numbers that are not negative; most fit 32 bits
__device__ __forceinline__ long long remainder_of(long long x, long long n) { return ((x | n) >> 32) == 0 ? (long long)((uint32_t)x % (uint32_t)n) : x % n; }

// last r in [lo, n) with first[r] <= x (first ascends, first[lo] <= x)
__device__ __forceinline__ int find_row(const int* first, int lo, int n, int x) {
  int hi = n;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (first[mid] <= x) lo = mid;
    else hi = mid;
  }
  return lo;
}

__global__ void __launch_bounds__(kPlanThreads) kv_plan_kernel(const PlanParams p) {
  extern __shared__ int plan_smem[];
  int* const tok = plan_smem;          // [R + 1] first token of a request
  int* const page = tok + p.R + 1;     // [R + 1] first page it takes
  int* const back = page + p.R + 1;    // [R + 1] first page it gives back
  int* const len = back + p.R + 1;     // [R]
  __shared__ long long warps[3][32];
  __shared__ int cut;                  // first request that does not fit
  const int tid = threadIdx.x, nt = blockDim.x, cta = blockIdx.x;
  const long long limit = p.max_pages * kPage;
  long long head = p.ends[0], tail = p.ends[1];
  const bool sound = head >= 0 && tail >= head && tail - head <= p.ring_size;
  if (!sound) {
    if (cta == 0 && tid == 0) atomicExch(p.status, 6);
    head = tail = 0;
  }
  if (tid == 0) cut = p.R;
  __syncthreads();
  long long base[3] = {0, 0, 0};
  for (int r0 = 0; r0 < p.R; r0 += nt) {
    const int r = r0 + tid;
    long long v[3] = {0, 0, 0}, own[3], tot[3];
    if (r < p.R) {
      const int l = p.lens[r], a = p.add[r];
      const bool bad = l < 0 || l > limit;
      const long long old = bad ? 0 : (l + (long long)kPage - 1) / kPage;
      len[r] = l;
      if (!bad && a > 0 && l + (long long)a <= limit) {
        v[0] = a;
        v[1] = (l + (long long)a + kPage - 1) / kPage - old;
      } else if (a < 0) {
        const long long k = p.keep ? p.keep[r] : 0;
        v[2] = old - min(max(k, 0ll), old);
      }
      if ((bad || (a > 0 && v[0] == 0)) && cta == 0) atomicExch(p.status, 2);
    }
#pragma unroll
    for (int i = 0; i < 3; ++i) own[i] = v[i];
    scan3(v, tot, warps);
#pragma unroll
    for (int i = 0; i < 3; ++i) v[i] += base[i];
    if (r < p.R) {
      const bool fits = v[0] + own[0] <= p.capacity && v[1] + own[1] <= tail - head;
      if (own[0] > 0 && !fits) atomicMin(&cut, r);
      // beyond what fits the sums are not used: any large value will do
      tok[r] = (int)min(v[0], 0x7fffffffll);
      page[r] = (int)min(v[1], 0x7fffffffll);
      back[r] = (int)min(v[2], 0x7fffffffll);
    }
#pragma unroll
    for (int i = 0; i < 3; ++i) base[i] += tot[i];
  }
  if (tid == 0) {
    tok[p.R] = (int)min(base[0], 0x7fffffffll);
    page[p.R] = (int)min(base[1], 0x7fffffffll);
    back[p.R] = (int)min(base[2], 0x7fffffffll);
  }
  __syncthreads();
  // requests from `cut` on get nothing: their sums are those at the cut
  const int c = cut, tokens = tok[c], taken = page[c];
  __syncthreads();
  for (int r = c + tid; r <= p.R; r += nt) {
    tok[r] = tokens;
    page[r] = taken;
  }
  // pages given back lie behind the ring's tail: more than there is room for means that the caller's books are wrong
  const bool room = sound && tail - head + base[2] <= p.ring_size;
  const int given = room ? back[p.R] : 0;
  if (!room && base[2] > 0 && cta == 0 && tid == 0) atomicExch(p.status, 6);
  __syncthreads();
  if (p.ctas > 1) cluster_arrive();  // this CTA has read lengths and counters

  const long long h0 = remainder_of(head, p.ring_size), t0 = remainder_of(tail, p.ring_size);
  const auto ring_at = [&](long long at, long long i) {
    const long long x = at + i;  // i <= ring_size
    return x >= p.ring_size ? x - p.ring_size : x;
  };
  const int self = cta * nt + tid, all = p.ctas * nt;
  // tokens, four in a row to a thread: most of them share a page
  for (int t = 4 * self; t < p.capacity; t += 4 * all) {
    int slot[4], at[4], n[4], row[4];
    int r = t < tokens ? find_row(tok, 0, p.R, t) : 0, of = -1, id = -1;  // page `of` of request r
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int u = t + i;
      slot[i] = row[i] = -1;
      at[i] = n[i] = 0;
      if (u < tokens) {
        while (tok[r + 1] <= u) {
          ++r;
          of = -1;
        }
        row[i] = r;
        at[i] = len[r] + (u - tok[r]);
        n[i] = at[i] + 1;
        const int old = (len[r] + kPage - 1) / kPage, pg = at[i] / kPage;
        if (pg != of) {
          of = pg;
          id = pg < old ? p.table[(size_t)r * p.max_pages + pg] : p.ring[ring_at(h0, page[r] + (pg - old))];
          if ((unsigned)id >= (unsigned)p.pages) {
            id = -1;
            atomicExch(p.status, 1);
          }
        }
        if (id >= 0) slot[i] = id * kPage + at[i] % kPage;
      }
    }
    if (p.whole4) {
      *reinterpret_cast<int4*>(p.slots + t) = make_int4(slot[0], slot[1], slot[2], slot[3]);
      *reinterpret_cast<int4*>(p.pos + t) = make_int4(at[0], at[1], at[2], at[3]);
      *reinterpret_cast<int4*>(p.seen + t) = make_int4(n[0], n[1], n[2], n[3]);
      *reinterpret_cast<int4*>(p.rows + t) = make_int4(row[0], row[1], row[2], row[3]);
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (t + i < p.capacity) {
          p.slots[t + i] = slot[i];
          p.pos[t + i] = at[i];
          p.seen[t + i] = n[i];
          p.rows[t + i] = row[i];
        }
    }
  }
  for (int i = self; i < taken; i += all) {
    const int r = find_row(page, 0, p.R, i);
    p.table[(size_t)r * p.max_pages + (len[r] + kPage - 1) / kPage + (i - page[r])] = p.ring[ring_at(h0, i)];
  }
  for (int i = self; i < given; i += all) {
    const int r = find_row(back, 0, p.R, i);
    // the request's pages end with its last one
    const int id = p.table[(size_t)r * p.max_pages + (len[r] + kPage - 1) / kPage - (back[r + 1] - i)];
    if ((unsigned)id >= (unsigned)p.pages) atomicExch(p.status, 1);  // the counters go on, and so it stands in the ring
    p.ring[ring_at(t0, i)] = id;
  }
  for (int r = self; r <= p.R; r += all) p.starts[r] = tok[r];
  if (p.ctas > 1) cluster_wait();  // everybody has: they may be overwritten
  for (int r = self; r < p.R; r += all) {
    const int n = tok[r + 1] - tok[r], a = p.add[r];
    p.lens_out[r] = a < 0 && room && len[r] >= 0 && len[r] <= limit ? 0 : len[r] + n;
  }
  if (self == 0) {
    p.ends_out[0] = sound ? head + taken : p.ends[0];
    p.ends_out[1] = sound ? tail + given : p.ends[1];
  }
}

__device__ __forceinline__ float4 load4(const float* p) { return __ldcs(reinterpret_cast<const float4*>(p)); }
__device__ __forceinline__ float4 load4(const __half* p) {
  const uint2 v = __ldcs(reinterpret_cast<const uint2*>(p));
  const float2 a = __half22float2(*reinterpret_cast<const __half2*>(&v.x)), b = __half22float2(*reinterpret_cast<const __half2*>(&v.y));
  return make_float4(a.x, a.y, b.x, b.y);
}
__device__ __forceinline__ float4 load4(const __nv_bfloat16* p) {
  const uint2 v = __ldcs(reinterpret_cast<const uint2*>(p));
  return make_float4(__uint_as_float(v.x << 16), __uint_as_float(v.x & 0xffff0000u), __uint_as_float(v.y << 16), __uint_as_float(v.y & 0xffff0000u));
}
__device__ __forceinline__ uint2 half4(float a, float b, float c, float d) {
  const __half2 x = __floats2half2_rn(a, b), y = __floats2half2_rn(c, d);
  return make_uint2(*reinterpret_cast<const uint32_t*>(&x), *reinterpret_cast<const uint32_t*>(&y));
}

struct AppendParams {
  const void* x;
  long long ldx, ldq;
  const int32_t *pos, *slots;
  const float *qg, *kg;
  __half *q, *pool;
  int32_t* status;
  int Hq, Hkv;
  long long places;  // slots of the pool
  float eps;
  double log2_base;
};

constexpr int kAppendThreads = 256, kHeadLanes = 16, kAtOnce = 3;  // heads of a lane on their way together

template <typename T>
__global__ void __launch_bounds__(kAppendThreads, 4) rope_append_slots_kernel(const AppendParams p) {
  __shared__ float cs[2][64];
  const int tid = threadIdx.x, l = tid % kHeadLanes, lane_head = tid / kHeadLanes;
  constexpr int kStep = kAppendThreads / kHeadLanes;
  const size_t t = blockIdx.x;
  const int heads = p.Hq + 2 * p.Hkv;
  const T* const x = static_cast<const T*>(p.x) + t * p.ldx;
  float4 a[kAtOnce], b[kAtOnce];
  const auto load = [&](int h0) {
#pragma unroll
    for (int i = 0; i < kAtOnce; ++i) {
      const int h = h0 + i * kStep;
      if (h < heads) {
        a[i] = load4(x + h * kHD + 4 * l);
        b[i] = load4(x + h * kHD + 64 + 4 * l);
      }
    }
  };
  load(lane_head);  // on its way while the slot and the position are
  const int slot = p.slots[t], pos = p.pos[t];
  if (slot < 0) return;  // padding
  if (slot >= p.places) {
    if (tid == 0) atomicExch(p.status, 1);
    return;
  }
  if (tid < 64) {
    // whole turns leave the angle in 64 bits: in 32 a position of 10^5 would be off by 10^-3
    double turns = pos * exp2(-(double)tid / 64 * p.log2_base) * 0.15915494309189533577;
    turns -= rint(turns);
    float s, c;
    sincospif((float)(2 * turns), &s, &c);
    cs[0][tid] = c;
    cs[1][tid] = s;
  }
  __syncthreads();
  const float4 c = *reinterpret_cast<const float4*>(&cs[0][4 * l]), s = *reinterpret_cast<const float4*>(&cs[1][4 * l]);
  __half* const page = p.pool + (size_t)(slot / kPage) * p.Hkv * (2 * kPage * kHD) + slot % kPage * kHD + 4 * l;
  // both halves of a warp go round together, though with an odd number of heads the second has none at the end
  for (int h0 = lane_head; h0 - lane_head % 2 < heads; h0 += kAtOnce * kStep) {
    if (h0 != lane_head) load(h0);
#pragma unroll
    for (int i = 0; i < kAtOnce; ++i) {
      const int h = h0 + i * kStep;
      float4 u = a[i], v = b[i];
      const float* const gain = h < p.Hq ? p.qg : p.kg;
      if (gain != nullptr) {  // the shuffle is every lane's
        float ss = u.x * u.x + u.y * u.y + u.z * u.z + u.w * u.w + v.x * v.x + v.y * v.y + v.z * v.z + v.w * v.w;
#pragma unroll
        for (int o = kHeadLanes / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
        if (h < p.Hq + p.Hkv) {
          const float r = rsqrtf(ss / (float)kHD + p.eps);
          const float4 g = *reinterpret_cast<const float4*>(gain + 4 * l), k = *reinterpret_cast<const float4*>(gain + 64 + 4 * l);
          u = make_float4(u.x * r * g.x, u.y * r * g.y, u.z * r * g.z, u.w * r * g.w);
          v = make_float4(v.x * r * k.x, v.y * r * k.y, v.z * r * k.z, v.w * r * k.w);
        }
      }
      if (h >= heads) continue;
      __half* dst;
      if (h < p.Hq + p.Hkv) {
        const float4 w = u;
        u = make_float4(w.x * c.x - v.x * s.x, w.y * c.y - v.y * s.y, w.z * c.z - v.z * s.z, w.w * c.w - v.w * s.w);
        v = make_float4(v.x * c.x + w.x * s.x, v.y * c.y + w.y * s.y, v.z * c.z + w.z * s.z, v.w * c.w + w.w * s.w);
        dst = h < p.Hq ? p.q + t * p.ldq + h * kHD + 4 * l : page + (size_t)(h - p.Hq) * (2 * kPage * kHD);
      } else {
        dst = page + (size_t)(h - p.Hq - p.Hkv) * (2 * kPage * kHD) + kPage * kHD;
      }
      *reinterpret_cast<uint2*>(dst) = half4(u.x, u.y, u.z, u.w);
      *reinterpret_cast<uint2*>(dst + 64) = half4(v.x, v.y, v.z, v.w);
    }
  }
}

}  // namespace

extern "C" {

int32_t qeng_kv_plan(qeng_ctx* ctx, const qeng_kv_pool* pool, int64_t R, const int32_t* lens, const int32_t* add, const int32_t* keep,
                     int32_t* page_table, int64_t max_pages, int32_t* ring, int64_t ring_size, const int64_t* ends, int32_t* lens_out,
                     int64_t* ends_out, int32_t* starts, int32_t* slots, int32_t* pos, int32_t* seen, int32_t* rows, int64_t capacity, void* stream) {
  if (!ctx || !pool || !lens || !add || !page_table || !ring || !ends || !lens_out || !ends_out || !starts || !slots || !pos || !seen || !rows)
    return qeng_fail(ctx, QENG_ERR_ARG, "kv_plan: null argument");
  if (R <= 0 || max_pages <= 0 || ring_size <= 0 || capacity <= 0)
    return qeng_fail(ctx, QENG_ERR_ARG, "kv_plan: R, max_pages, ring_size and capacity must be positive");
  if (R > kPlanRequests) return qeng_fail(ctx, QENG_ERR_SHAPE, "kv_plan: %lld requests, %d at most", (long long)R, kPlanRequests);
  if (capacity > (1 << 30) || max_pages > (1 << 26) || ring_size > (1 << 30) || pool->pages > (1 << 26))
    return qeng_fail(ctx, QENG_ERR_SHAPE, "kv_plan: slots are 32-bit: at most 2^30 tokens and ring entries, 2^26 pages");
  if (((reinterpret_cast<uintptr_t>(ends) | reinterpret_cast<uintptr_t>(ends_out)) & 7) != 0)
    return qeng_fail(ctx, QENG_ERR_ALIGN, "kv_plan: ends must be 8-byte aligned");
  QENG_ENTER(ctx);
  PlanParams p;
  p.lens = lens; p.add = add; p.keep = keep; p.table = page_table; p.ring = ring; p.ends = ends; p.lens_out = lens_out; p.ends_out = ends_out;
  p.starts = starts; p.slots = slots; p.pos = pos; p.seen = seen; p.rows = rows; p.status = ctx->status;
  p.R = (int)R; p.capacity = (int)capacity; p.pages = (int)pool->pages; p.max_pages = max_pages; p.ring_size = ring_size;
  p.whole4 = capacity % 4 == 0 &&
             ((reinterpret_cast<uintptr_t>(slots) | reinterpret_cast<uintptr_t>(pos) | reinterpret_cast<uintptr_t>(seen) | reinterpret_cast<uintptr_t>(rows)) & 15) == 0;
  // a thread for every request and four tokens as far as a block has them (barriers of few warps are faster), clusters above
  p.ctas = 1;
  while (p.ctas < 8 && capacity > 4096ll * p.ctas) p.ctas *= 2;
  int threads = 128;
  while (threads < kPlanThreads && (threads < R || 4ll * threads < capacity)) threads *= 2;
  const size_t smem = (size_t)(4 * R + 3) * sizeof(int);
  static bool configured_on[64] = {};  // the opt-in shared-memory size is set per device
  bool& configured = configured_on[ctx->device & 63];
  if (!configured) {
    QENG_CUDA(ctx, cudaFuncSetAttribute(kv_plan_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)((4 * kPlanRequests + 3) * sizeof(int))));
    configured = true;
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)p.ctas);
  cfg.blockDim = dim3((unsigned)threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = (cudaStream_t)stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = (unsigned)p.ctas;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = p.ctas > 1 ? 1 : 0;
  QENG_CUDA(ctx, cudaLaunchKernelEx(&cfg, kv_plan_kernel, p));
  return QENG_OK;
}

int32_t qeng_rope_append(qeng_ctx* ctx, qeng_kv_pool* pool, const void* qkv, int32_t x_dtype, int64_t T, int64_t ldx, int64_t Hq, const float* q_gain,
                         const float* k_gain, float eps, const int32_t* pos, const int32_t* slots, float base, uint16_t* q_f16, int64_t ldq, void* stream) {
  if (!ctx || !pool || !qkv || !pos || !slots || !q_f16) return qeng_fail(ctx, QENG_ERR_ARG, "rope_append: null argument");
  if (x_dtype < QENG_F32 || x_dtype > QENG_BF16) return qeng_fail(ctx, QENG_ERR_ARG, "rope_append: unknown type %d", x_dtype);
  if (T <= 0 || Hq <= 0 || T > 0x7fffffff || Hq > 4096) return qeng_fail(ctx, QENG_ERR_SHAPE, "rope_append: T and Hq must be positive (Hq at most 4096)");
  if (!(base > 0.f)) return qeng_fail(ctx, QENG_ERR_ARG, "rope_append: base must be positive");
  if ((q_gain == nullptr) != (k_gain == nullptr)) return qeng_fail(ctx, QENG_ERR_ARG, "rope_append: gains of both q and k, or of neither");
  const int64_t size = x_dtype == QENG_F32 ? 4 : 2;
  if (ldx < (Hq + 2 * pool->kv_heads) * kHD || ldq < Hq * kHD)
    return qeng_fail(ctx, QENG_ERR_SHAPE, "rope_append: rows of %lld and %lld values do not hold %lld + 2 * %lld heads", (long long)ldx, (long long)ldq,
                     (long long)Hq, (long long)pool->kv_heads);
  if (((reinterpret_cast<uintptr_t>(qkv) | reinterpret_cast<uintptr_t>(q_f16) | reinterpret_cast<uintptr_t>(q_gain) | reinterpret_cast<uintptr_t>(k_gain)) & 15) != 0 ||
      ldx * size % 16 != 0 || ldq % 8 != 0)
    return qeng_fail(ctx, QENG_ERR_ALIGN, "rope_append: rows and gains must be 16-byte aligned");
  QENG_ENTER(ctx);
  AppendParams p;
  p.x = qkv; p.ldx = ldx; p.ldq = ldq; p.pos = pos; p.slots = slots; p.qg = q_gain; p.kg = k_gain; p.q = reinterpret_cast<__half*>(q_f16);
  p.pool = pool->data; p.status = ctx->status; p.Hq = (int)Hq; p.Hkv = (int)pool->kv_heads; p.places = pool->pages * kPage; p.eps = eps;
  p.log2_base = log2((double)base);
  auto* const fn = x_dtype == QENG_F32 ? rope_append_slots_kernel<float> : x_dtype == QENG_F16 ? rope_append_slots_kernel<__half> : rope_append_slots_kernel<__nv_bfloat16>;
  fn<<<(unsigned)T, kAppendThreads, 0, (cudaStream_t)stream>>>(p);
  QENG_LAUNCH_CHECK(ctx);
  return QENG_OK;
}

}  // extern "C"
