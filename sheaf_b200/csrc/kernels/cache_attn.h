// Parts shared by the kernels of attention over a key/value cache
// (cache_attention.cu, cache_attention_tile.cu, cache_attention_mma.cu,
// cache_attention_tc.cu).
// Included by .cu files only.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <cmath>

#include "kernels.h"
#include "pdl.h"
#include "tc_common.h"

namespace sb {
namespace cattn {

constexpr float kLog2e = 1.4426950408889634f;

// Two f32 rounded to packed bf16 or f16, and what the rounding left of them.
template <bool F16>
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
  uint32_t d;
  if (F16) asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(d) : "f"(hi), "f"(lo));
  else asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(d) : "f"(hi), "f"(lo));
  return d;
}
template <bool F16>
__device__ __forceinline__ float2 unpack2(uint32_t w) {
  if (F16) return __half22float2(*(const __half2*)&w);
  return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
}
template <bool F16>
__device__ __forceinline__ uint32_t take2(float& lo, float& hi) {
  const uint32_t w = pack2<F16>(lo, hi);
  const float2 f = unpack2<F16>(w);
  lo -= f.x;
  hi -= f.y;
  return w;
}

// Codes c in bytes 0 and 2 of t (bytes 1 and 3: anything) to two f16 values.
// 0x6400 + (c + 128) is 1024 + c + 128 as f16 (steps of 1 there): c exactly,
// after a subtraction.  (bf16 has no steps of 1 beyond 8 bits and would need
// twice the instructions, which bound the int8 kernel.)
__device__ __forceinline__ uint32_t codes(uint32_t t) {
  const uint32_t a = (t & 0x00ff00ffu) ^ 0x64806480u;
  __half2 x = __hsub2(*(const __half2*)&a, __half2half2(__ushort_as_half(0x6480)));
  return *(uint32_t*)&x;
}

struct Params {
  const void *k, *v;
  const float *ks, *vs;
  const int *positions, *parents;
  const void* q;
  void* out;
  int bf16;             // q and out
  int H, G, S, D;       // cache heads, query heads per cache head, tokens, head size
  int chunks;           // blocks of query rows (token x query head) per (slot, cache head)
  int64_t T;
  float scale2;         // scale * log2(e)
};

// The calls that go to the tensor cores (cache_attention_mma.cu and _tc.cu, heads
// padded to 64 or 128).  Heads up to 32 only from 4 rows on: one row of 64 x 12
// int8 caches of 512 keys of 32 takes 21.5 us there and 15.1 on the CUDA cores, 4
// rows of 19 x 4 of 6K keys 22 and 63, 160 rows of 15 x 4 of 1.5K bf16 keys 22 and
// 137; one row with heads of 48, 23.6 and 28.0.
inline bool on_tensor_cores(const CacheAttnArgs& a) {
  return a.cache.type != KvType::F32 && a.cache.D <= 128 && (a.cache.D > 32 || a.S * (a.Hq / a.cache.H) >= 4);
}

inline Params make_params(const CacheAttnArgs& a, int chunk_rows) {
  const KvCacheView& c = a.cache;
  const int G = (int)(a.Hq / c.H), rows = (int)a.S * G;
  return {c.k, c.v, c.k_scale, c.v_scale, a.positions, a.parents, a.q, a.out, a.bf16 ? 1 : 0, (int)c.H, G, (int)a.S,
          (int)c.D, (rows + chunk_rows - 1) / chunk_rows, c.T, a.scale * kLog2e};
}

inline int sm_count() {
  int dev = 0, n = 148;
  if (cudaGetDevice(&dev) == cudaSuccess) cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev);
  return n;
}

// CTAs of a cluster: 8 is what every GPU takes.  Twice that goes where a few
// long items would leave SMs idle, at most one CTA per SM: one sequence's 8 heads of
// 30K bf16 keys of 128, 34 us against 53, f32 keys 47 and 89; with 16 items, which
// 8 CTAs each spread over most SMs, it was slower (26 us, 21.5).
constexpr int kPortable = 8, kMaxCluster = 16;
inline bool may_double(int C, int64_t items) {
  return C < kPortable || (C < kMaxCluster && items * 2 * C <= sm_count());
}

template <typename... K, typename... A>
cudaError_t launch_cluster(void (*kern)(K...), int64_t blocks, int cluster, int threads, size_t smem,
                           cudaStream_t stream, A&&... args) {
  if (blocks > INT32_MAX) return cudaErrorInvalidValue;
  if (smem > 40 * 1024) {  // with the static part it may pass the default 48 KB
    cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
    if (e != cudaSuccess) return e;
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)blocks);
  cfg.blockDim = dim3((unsigned)threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute at[2];
  pdl_attribute(&at[0]);
  at[1].id = cudaLaunchAttributeClusterDimension;
  at[1].val.clusterDim.x = (unsigned)cluster;
  at[1].val.clusterDim.y = at[1].val.clusterDim.z = 1;
  cfg.attrs = at;
  cfg.numAttrs = 2;
  if (cluster > kPortable) {  // where the GPU has room for one
    cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
    if (e != cudaSuccess) return e;
    int fit = 0;
    e = cudaOccupancyMaxActiveClusters(&fit, kern, &cfg);
    if (e != cudaSuccess || fit < 1) {
      cudaGetLastError();
      cfg.gridDim.x = (unsigned)(blocks / cluster * kPortable);
      at[1].val.clusterDim.x = kPortable;
    }
  }
  launch_counter().fetch_add(1, std::memory_order_relaxed);
  return cudaLaunchKernelEx(&cfg, kern, std::forward<A>(args)...);
}

__device__ __forceinline__ uint32_t cluster_size() {
  uint32_t c;
  asm("mov.u32 %0, %%cluster_nctarank;" : "=r"(c));
  return c;
}

// Where a CTA stands: the (slot, cache head) and block of rows of its cluster,
// and the keys there: positions [0, pre) before the drafted tokens, and the
// drafted ones at [pos, end).
struct Place {
  uint32_t rank, C;
  int chunk, h;
  int64_t nh, n, pos, pre, end;
};
__device__ __forceinline__ Place find_place(const Params& p) {
  Place w;
  w.rank = tc::cluster_rank();
  w.C = cluster_size();
  const unsigned item = blockIdx.x / w.C;
  w.chunk = (int)(item % (unsigned)p.chunks);
  const unsigned nh = item / (unsigned)p.chunks;
  w.nh = nh;
  w.n = nh / (unsigned)p.H;
  w.h = (int)(nh % (unsigned)p.H);
  w.pos = p.positions[w.n];
  w.pre = w.pos < 0 ? 0 : min(w.pos, p.T);
  w.end = w.pos < 0 ? 0 : min(w.pos + p.S, p.T);
  return w;
}

// Element offset of row `row` (token row / G, query head h G + row % G) in q and out.
__device__ __forceinline__ int64_t row_at(const Params& p, const Place& w, int row) {
  const int s = row / p.G, g = row - s * p.G;
  return (((w.n * p.S + s) * p.H + w.h) * p.G + g) * p.D;
}

// Which of the S drafted tokens token s attends to: bit j of mask[s].  The
// parents' chains are closed by pointer doubling in shared memory (log2 S
// rounds).  One warp.
__device__ __forceinline__ void tree_masks(const int* parents, int S, int lane, unsigned long long* mask, int* jump) {
  for (int s = lane; s < S; s += 32) {
    const int q = parents ? parents[s] : s - 1;
    jump[s] = q >= 0 && q < s ? q : -1;
    mask[s] = 1ull << s;
  }
  __syncwarp();
  for (int d = 1; d < S; d *= 2) {
    unsigned long long m[2];
    int j[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int s = lane + 32 * i;
      if (s < S) {
        const int t = jump[s];
        m[i] = mask[s] | (t >= 0 ? mask[t] : 0ull);
        j[i] = t >= 0 ? jump[t] : -1;
      }
    }
    __syncwarp();
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int s = lane + 32 * i;
      if (s < S) mask[s] = m[i], jump[s] = j[i];
    }
    __syncwarp();
  }
}

// The drafted tokens that a token with mask `mask` sees and that fit the cache.
__device__ __forceinline__ unsigned long long drafted_seen(const Place& w, unsigned long long mask) {
  const int64_t fit = w.end - w.pos;
  return w.pos < 0 || fit <= 0 ? 0ull : fit >= 64 ? mask : mask & ((1ull << fit) - 1);
}

__device__ __forceinline__ float ld_remote(const float* p, uint32_t rank) {
  float x;
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(x) : "r"(tc::cluster_addr(p, rank)));
  return x;
}
__device__ __forceinline__ float4 ld_remote4(const float* p, uint32_t rank) {
  float4 x;
  asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
               : "=f"(x.x), "=f"(x.y), "=f"(x.z), "=f"(x.w)
               : "r"(tc::cluster_addr(p, rank)));
  return x;
}

__device__ __forceinline__ void store4(const Params& p, int64_t at, float4 y) {
  if (p.bf16) {
    __nv_bfloat162 h[2] = {__floats2bfloat162_rn(y.x, y.y), __floats2bfloat162_rn(y.z, y.w)};
    *(uint2*)((__nv_bfloat16*)p.out + at) = *(uint2*)h;
  } else {
    *(float4*)((float*)p.out + at) = y;
  }
}


// f16 operands for int8 caches.  A row of queries is scaled by a power of two to
// a largest value in [2^14, 2^15), which keeps what is 2^-38 of it: 2^(14 - e)
// for a largest value of exponent e, within f32's normal range; down = 1 / up.
__device__ __forceinline__ float f16_row_scale(float largest, float& down) {
  const int e = min(max((int)(__float_as_uint(largest) >> 23) - 127, -110), 127);
  down = __uint_as_float((uint32_t)(127 - 14 + e) << 23);
  return __uint_as_float((uint32_t)(127 + 14 - e) << 23);
}
// P times the value scales goes into f16 relative to a power of two, 2^vref, with
// steps of 2^-30 of it: at most 2^(8 + 6).  As long as the scales met so far lie
// within 2^kEven of one another, 2^vref is above the largest of them, for all rows
// alike.  Past that the scales are "wide", from that tile on: vref is a row's own,
// by the largest P times scale of the keys that the row sees, so that neither a key
// that it does not see nor one of little weight takes bits from the others.  (8 x 4
// caches of 16K keys of 128, 256 bf16 rows: 126 us, wide 312; 4 x 8 of 30K, 4 rows:
// 61 and 68.  So the limit is far above what the values of a text differ by, and
// leaves the smallest scale 22 bits.)
constexpr int kVrefFirst = -120;  // low enough for every normal scale; its factors are normal f32
constexpr int kVrefLast = 127;
constexpr int kEven = 8;
constexpr int kBigExponent = 100;  // wide too, and rows' maxima are not lazy: 2^8 times such a scale may pass f32's range
__device__ __forceinline__ float vref_down(int vref) { return __uint_as_float((uint32_t)(127 + 6 - vref) << 23); }
__device__ __forceinline__ float vref_up(int vref) { return __uint_as_float((uint32_t)(127 - 6 + vref) << 23); }
__device__ __forceinline__ float pow2(int e) {  // 0 below f32's normal range
  return e < -126 ? 0.f : __uint_as_float((uint32_t)(127 + min(e, 127)) << 23);
}
// The exponents of the scales met so far by a warp: 2^hi is above the largest, 2^(lo - 1) at most the smallest of the
// lane's.  Zeros (which need no bits) and scales that are not finite (which leave none) do not count.
struct ScaleRange {
  int hi = kVrefFirst, lane_hi = kVrefFirst, lo = kVrefLast + 1;
  bool wide = false;
  __device__ __forceinline__ void lane_adds(float s) {
    const uint32_t u = __float_as_uint(s) & 0x7fffffffu;
    const int e = max((int)(u >> 23) - 126, kVrefFirst);
    if (u - 1u < 0x7f800000u - 1u) lane_hi = max(lane_hi, e), lo = min(lo, e);
  }
  __device__ __forceinline__ bool big() const { return hi > kBigExponent; }
  __device__ __forceinline__ void join_lanes() {  // one vote as long as nothing changes
    if (!__any_sync(0xffffffffu, lane_hi > hi || lo < hi - kEven)) return;
    hi = __reduce_max_sync(0xffffffffu, lane_hi);
    wide = wide || big() || __any_sync(0xffffffffu, lo < hi - kEven);
  }
};
// A row's vref among wide scales; `largest`: of P times scale so far, relative to the row's present maximum.  It
// comes down at once, where the row's other keys need the bits, and goes up when f16 would not hold the next.
__device__ __forceinline__ int wide_vref(int vref, float largest) {
  const int e = min(max((int)(__float_as_uint(largest) >> 23) - 126, kVrefFirst), kVrefLast);
  return largest > 0.f && (e > vref + 8 || e < vref) ? max(e, vref - 120) : vref;
}

// The weights of N partial results with base-2 maxima m: f = 2^(m - max).
template <int N>
__device__ __forceinline__ float join_weights(const float* m, float* f) {
  float mx = -INFINITY;
#pragma unroll
  for (int j = 0; j < N; ++j) mx = fmaxf(mx, m[j]);
  const float base = mx == -INFINITY ? 0.f : mx;
#pragma unroll
  for (int j = 0; j < N; ++j) f[j] = exp2f(m[j] - base);
  return mx;
}
__device__ __forceinline__ void add_scaled(float4& a, const float4& x, float f) {
  a.x = fmaf(x.x, f, a.x);
  a.y = fmaf(x.y, f, a.y);
  a.z = fmaf(x.z, f, a.z);
  a.w = fmaf(x.w, f, a.w);
}

// The finished values d .. d + 3 of row r0 + r: o / l, or zeros for a row
// without keys.  `bad`: drafted bf16 values that are not finite were taken out
// of the products; they go to the rows that see them.
__device__ __forceinline__ void finish4(const Params& p, const Place& w, int row, int d, float4 o, float l,
                                        const unsigned long long* mask, bool bad) {
  if (d >= p.D) return;
  const unsigned long long seen = drafted_seen(w, mask[row / p.G]);
  float y[4] = {o.x / l, o.y / l, o.z / l, o.w / l};
  if (bad)
    for (int j = 0; j < p.S; ++j)
      if (seen >> j & 1ull)
        for (int i = 0; i < 4; ++i) {
          const float v = __bfloat162float(((const __nv_bfloat16*)p.v)[(w.nh * p.T + w.pos + j) * p.D + d + i]);
          if (!isfinite(v)) y[i] += v;
        }
  if (w.pre <= 0 && !seen) y[0] = y[1] = y[2] = y[3] = 0.f;
  store4(p, row_at(p, w, row) + d, make_float4(y[0], y[1], y[2], y[3]));
}

// The partial results of up to R rows, joined and written: first the PARTS of a
// CTA of NW warps, then the CTAs' of the cluster (rank c finishes every C-th piece
// of 4 values).  part_o [PARTS][R][DP], part_m, part_l [PARTS][R] in shared memory
// (m: base-2 maximum, l: sum); every thread of the CTA calls once it has written
// its parts.  cta_o [R][DP] (with one part, may be part_o) and cta_ml [2 R] are
// shared too; s_bad (may be null): see finish4.
template <int NW, int R, int DP, int PARTS = NW>
__device__ __forceinline__ void join_and_store(const Params& p, const Place& w, int r0, int rows,
                                               const float* part_o, const float* part_m, const float* part_l,
                                               float* cta_o, float* cta_ml, const unsigned long long* mask,
                                               const int* s_bad) {
  constexpr int V = DP / 4;
  const int tid = threadIdx.x;
  __syncthreads();
  for (int i = tid; i < rows * V; i += NW * 32) {
    const int r = i / V, d = (i % V) * 4;
    float m[PARTS], f[PARTS], l = 0.f;
    float4 x[PARTS], a = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int j = 0; j < PARTS; ++j) {
      m[j] = part_m[j * R + r];
      x[j] = *(const float4*)(part_o + (j * R + r) * DP + d);
    }
    const float mx = join_weights<PARTS>(m, f);
#pragma unroll
    for (int j = 0; j < PARTS; ++j) {
      add_scaled(a, x[j], f[j]);
      l = fmaf(part_l[j * R + r], f[j], l);
    }
    if (w.C == 1) {
      finish4(p, w, r0 + r, d, a, l, mask, s_bad && *s_bad);
    } else {
      *(float4*)(cta_o + r * DP + d) = a;
      if (d == 0) cta_ml[r] = mx, cta_ml[R + r] = l;
    }
  }
  if (w.C == 1) return;
  tc::cluster_sync();
  int bad = 0;
  if (s_bad)
    for (uint32_t c = 0; c < w.C; ++c) {
      int y;
      asm volatile("ld.shared::cluster.s32 %0, [%1];" : "=r"(y) : "r"(tc::cluster_addr(s_bad, c)));
      bad |= y;
    }
  for (int i = (int)w.rank * NW * 32 + tid; i < rows * V; i += (int)w.C * NW * 32) {
    const int r = i / V, d = (i % V) * 4;
    float m[kMaxCluster], l[kMaxCluster], f[kMaxCluster], sum = 0.f;
    float4 x[kMaxCluster], a = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (uint32_t c = 0; c < kMaxCluster; ++c) {
      m[c] = -INFINITY, l[c] = 0.f, x[c] = a;
      if (c < w.C) {
        m[c] = ld_remote(&cta_ml[r], c);
        l[c] = ld_remote(&cta_ml[R + r], c);
        x[c] = ld_remote4(cta_o + r * DP + d, c);
      }
    }
    join_weights<kMaxCluster>(m, f);
#pragma unroll
    for (int c = 0; c < kMaxCluster; ++c) {
      add_scaled(a, x[c], f[c]);
      sum = fmaf(l[c], f[c], sum);
    }
    finish4(p, w, r0 + r, d, a, sum, mask, bad);
  }
  tc::cluster_sync();  // no CTA leaves while another may read its shared memory
}

}  // namespace cattn
}  // namespace sb
