// Attention of a few tokens per sequence over a key/value cache, on the CUDA
// cores: one token (decoding), or a chain or tree of drafted tokens.
//
//   o_s = sum_t softmax_t(scale q_s . k_t) v_t   over the positions t < pos,
//         the token itself and its ancestors among the drafted tokens.
//
// Reading the cache once bounds it, so the work is laid out around the loads:
// a group of LPK lanes holds one cached row, 8 values a lane (one 32-byte load
// of f32, 16 of bf16, 8 of int8 codes), and a warp takes 32 / LPK rows at a
// time, U of them in flight for K and for V.  The scores of R query rows
// (tokens x query heads that share the cache head) are formed in one pass: R
// dot products per lane and a butterfly over the group leave every lane of the
// group with the scores of its row, which is all it needs for its part of the
// V sum.  Each group keeps its own running maximum m and sum l (base 2), so no
// lane waits for another inside the loop; int8 scales multiply the score and
// the probability, not the row.
//
// The positions are split over a cluster of C CTAs.  Each CTA joins its warps'
// (m, l, o) in shared memory, and after one cluster barrier every CTA adds up
// its slice of the outputs from all C shared memories in rank order.  So the
// split needs no workspace in memory and no atomics: results do not depend on
// timing, and graphs that run at the same time share nothing.
#include <cuda_bf16.h>

#include <cmath>

#include "kernels.h"
#include "pdl.h"
#include "tc_common.h"

namespace sb {
namespace {

constexpr int kWarps = 8, kThreads = kWarps * 32;
constexpr int EPL = 8;
constexpr float kLog2e = 1.4426950408889634f;

struct Params {
  const void *k, *v;
  const float *ks, *vs;
  const int *positions, *parents;
  const void* q;
  void* out;
  int bf16;  // q and out
  int H, G, S, D, chunks;  // chunks of R rows
  int64_t T;
  float scale2;  // scale * log2(e)
};

template <typename T>
struct Raw;  // 8 values as loaded
template <>
struct Raw<float> { float4 a, b; };
template <>
struct Raw<__nv_bfloat16> { uint4 a; };
template <>
struct Raw<int8_t> { uint2 a; };

__device__ __forceinline__ void load_raw(const float* p, Raw<float>& r) {
  asm volatile("ld.global.L1::no_allocate.v8.f32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
               : "=f"(r.a.x), "=f"(r.a.y), "=f"(r.a.z), "=f"(r.a.w), "=f"(r.b.x), "=f"(r.b.y), "=f"(r.b.z), "=f"(r.b.w)
               : "l"(p));
}
__device__ __forceinline__ void load_raw(const __nv_bfloat16* p, Raw<__nv_bfloat16>& r) {
  asm volatile("ld.global.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(r.a.x), "=r"(r.a.y), "=r"(r.a.z), "=r"(r.a.w) : "l"(p));
}
__device__ __forceinline__ void load_raw(const int8_t* p, Raw<int8_t>& r) {
  asm volatile("ld.global.L1::no_allocate.v2.u32 {%0,%1}, [%2];" : "=r"(r.a.x), "=r"(r.a.y) : "l"(p));
}

__device__ __forceinline__ void widen(const Raw<float>& r, float* x) {
  x[0] = r.a.x, x[1] = r.a.y, x[2] = r.a.z, x[3] = r.a.w, x[4] = r.b.x, x[5] = r.b.y, x[6] = r.b.z, x[7] = r.b.w;
}
__device__ __forceinline__ void widen(const Raw<__nv_bfloat16>& r, float* x) {
  const uint32_t w[4] = {r.a.x, r.a.y, r.a.z, r.a.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    x[2 * i] = __uint_as_float(w[i] << 16);
    x[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
  }
}
// Codes to f32 without the conversion unit: byte b of c ^ 0x80 (= c + 128)
// becomes the low mantissa byte of 2^23, and 2^23 + 128 is subtracted.
__device__ __forceinline__ void widen(const Raw<int8_t>& r, float* x) {
  const uint32_t w[2] = {r.a.x ^ 0x80808080u, r.a.y ^ 0x80808080u};
#pragma unroll
  for (int i = 0; i < 8; ++i)
    x[i] = __uint_as_float(__byte_perm(w[i / 4], 0x4b000000u, 0x7440 + (i & 3))) - 8388736.f;
}
template <typename CT>
__device__ __forceinline__ void zero_raw(Raw<CT>& r) {
  r = Raw<CT>{};
}

// Which of the S drafted tokens token s attends to: bit j of mask[s].  The
// parents' chains are closed by pointer doubling in shared memory (log2 S
// rounds).  One warp.
__device__ void tree_masks(const int* parents, int S, int lane, unsigned long long* mask, int* jump) {
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

template <typename CT, int LPK, int R, int U>
__global__ void __launch_bounds__(kThreads) cache_attn_kernel(const Params p) {
  pdl_prologue();
  constexpr int KPW = 32 / LPK;   // rows of the cache a warp loads at once
  constexpr int DP = LPK * EPL;   // head size, padded
  constexpr int TK = KPW * U;
  extern __shared__ float sm[];
  float* s_o = sm;                              // [kWarps][R][DP]; the CTA's sum replaces warp 0's
  float* s_m = sm + kWarps * R * DP;            // [kWarps][R]
  float* s_l = s_m + kWarps * R;
  __shared__ unsigned long long s_mask[kKvMaxTokens];
  __shared__ int s_jump[kKvMaxTokens];
  __shared__ float c_m[R], c_l[R];

  const uint32_t rank = tc::cluster_rank();
  uint32_t C;
  asm("mov.u32 %0, %%cluster_nctarank;" : "=r"(C));
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, gl = lane % LPK, grp = lane / LPK;
  const int64_t item = blockIdx.x / C;
  const int chunk = (int)(item % p.chunks);
  const int64_t nh = item / p.chunks, n = nh / p.H;
  const int h = (int)(nh % p.H);
  const int64_t pos = p.positions[n];
  // keys: [0, pre) before the drafted tokens, [pos, end) drafted
  const int64_t pre = pos < 0 ? 0 : min(pos, p.T), end = pos < 0 ? 0 : min(pos + p.S, p.T);
  if (warp == 0) tree_masks(p.parents ? p.parents + n * p.S : nullptr, p.S, lane, s_mask, s_jump);
  __syncthreads();

  const int rows = p.S * p.G, r0 = chunk * R;
  float q[R][EPL], o[R][EPL], m[R], l[R];
  int tok[R];
#pragma unroll
  for (int r = 0; r < R; ++r) {
    const int row = min(r0 + r, rows - 1);
    tok[r] = row / p.G;
    const int64_t at = ((n * p.S + tok[r]) * p.H * p.G + (int64_t)h * p.G + row % p.G) * p.D + gl * EPL;
#pragma unroll
    for (int i = 0; i < EPL; ++i) q[r][i] = o[r][i] = 0.f;
    if (gl * EPL < p.D) {
      if (p.bf16) {
        Raw<__nv_bfloat16> x;
        x.a = *(const uint4*)((const __nv_bfloat16*)p.q + at);
        widen(x, q[r]);
      } else {
        const float4* x = (const float4*)((const float*)p.q + at);
        Raw<float> y = {x[0], x[1]};
        widen(y, q[r]);
      }
    }
#pragma unroll
    for (int i = 0; i < EPL; ++i) q[r][i] *= p.scale2;
    m[r] = -INFINITY;
    l[r] = 0.f;
  }

  // this CTA's positions
  const int64_t per = (end + C - 1) / C, lo = min((int64_t)rank * per, end), hi = min(lo + per, end);
  const CT* kb = (const CT*)p.k + nh * p.T * p.D + gl * EPL;
  const CT* vb = (const CT*)p.v + nh * p.T * p.D + gl * EPL;
  const bool live_lane = gl * EPL < p.D;
  for (int64_t t0 = lo + warp * TK; t0 < hi; t0 += kWarps * TK) {
    Raw<CT> kr[U], vr[U];
    float ksc[U], vsc[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int64_t t = t0 + u * KPW + grp;
      zero_raw(kr[u]);
      zero_raw(vr[u]);
      ksc[u] = vsc[u] = 0.f;
      if (t < hi) {
        if (live_lane) {
          load_raw(kb + t * p.D, kr[u]);
          load_raw(vb + t * p.D, vr[u]);
        }
        if constexpr (sizeof(CT) == 1) {
          ksc[u] = p.ks[nh * p.T + t];
          vsc[u] = p.vs[nh * p.T + t];
        }
      }
    }
    float s[U][R];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      float x[EPL];
      widen(kr[u], x);
#pragma unroll
      for (int r = 0; r < R; ++r) {
        float a = 0.f;
#pragma unroll
        for (int i = 0; i < EPL; ++i) a = fmaf(q[r][i], x[i], a);
#pragma unroll
        for (int w = LPK / 2; w; w >>= 1) a += __shfl_xor_sync(0xffffffffu, a, w);
        if constexpr (sizeof(CT) == 1) a *= ksc[u];
        s[u][r] = a;
      }
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int64_t t = t0 + u * KPW + grp;
#pragma unroll
      for (int r = 0; r < R; ++r) {
        bool see = t < hi;
        if (t >= pre && t < hi) see = (s_mask[tok[r]] >> (t - pos)) & 1ull;
        if (!see) s[u][r] = -INFINITY;
      }
    }
#pragma unroll
    for (int r = 0; r < R; ++r) {
      float mx = m[r];
#pragma unroll
      for (int u = 0; u < U; ++u) mx = fmaxf(mx, s[u][r]);
      const float base = mx == -INFINITY ? 0.f : mx;
      const float a = exp2f(m[r] - base);
      m[r] = mx;
      l[r] *= a;
#pragma unroll
      for (int i = 0; i < EPL; ++i) o[r][i] *= a;
#pragma unroll
      for (int u = 0; u < U; ++u) {
        s[u][r] = exp2f(s[u][r] - base);
        l[r] += s[u][r];
      }
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      float x[EPL];
      widen(vr[u], x);
#pragma unroll
      for (int r = 0; r < R; ++r) {
        float w = s[u][r];
        if constexpr (sizeof(CT) == 1) w *= vsc[u];
        // a masked position holds anything, NaN included: it adds nothing
        if (s[u][r] != 0.f) {
#pragma unroll
          for (int i = 0; i < EPL; ++i) o[r][i] = fmaf(w, x[i], o[r][i]);
        }
      }
    }
  }

  // join the groups of the warp
#pragma unroll
  for (int r = 0; r < R; ++r) {
#pragma unroll
    for (int w = LPK; w < 32; w *= 2) {
      const float m2 = __shfl_xor_sync(0xffffffffu, m[r], w), l2 = __shfl_xor_sync(0xffffffffu, l[r], w);
      const float mx = fmaxf(m[r], m2), base = mx == -INFINITY ? 0.f : mx;
      const float a = exp2f(m[r] - base), b = exp2f(m2 - base);
      l[r] = l[r] * a + l2 * b;
#pragma unroll
      for (int i = 0; i < EPL; ++i) o[r][i] = o[r][i] * a + __shfl_xor_sync(0xffffffffu, o[r][i], w) * b;
      m[r] = mx;
    }
    if (grp == 0) {
#pragma unroll
      for (int i = 0; i < EPL; ++i) s_o[(warp * R + r) * DP + gl * EPL + i] = o[r][i];
      if (gl == 0) s_m[warp * R + r] = m[r], s_l[warp * R + r] = l[r];
    }
  }
  __syncthreads();
  // join the warps
  for (int i = tid; i < R * DP; i += kThreads) {
    const int r = i / DP;
    float mx = -INFINITY;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) mx = fmaxf(mx, s_m[w * R + r]);
    const float base = mx == -INFINITY ? 0.f : mx;
    float a = 0.f, b = 0.f;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      const float f = exp2f(s_m[w * R + r] - base);
      a += s_o[w * R * DP + i] * f;
      b += s_l[w * R + r] * f;
    }
    s_o[i] = a;
    if (i % DP == 0) c_m[r] = mx, c_l[r] = b;
  }
  tc::cluster_sync();
  // join the cluster: rank c of C finishes outputs i = c (mod C) in steps of a CTA
  for (int i = (int)rank * kThreads + tid; i < R * DP; i += (int)C * kThreads) {
    const int r = i / DP, d = i % DP;
    float mx = -INFINITY;
    for (uint32_t c = 0; c < C; ++c) {
      float x;
      asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(x) : "r"(tc::cluster_addr(&c_m[r], c)));
      mx = fmaxf(mx, x);
    }
    const float base = mx == -INFINITY ? 0.f : mx;
    float a = 0.f, b = 0.f;
    for (uint32_t c = 0; c < C; ++c) {
      float xm, xl, xo;
      asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(xm) : "r"(tc::cluster_addr(&c_m[r], c)));
      asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(xl) : "r"(tc::cluster_addr(&c_l[r], c)));
      asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(xo) : "r"(tc::cluster_addr(&s_o[i], c)));
      const float f = exp2f(xm - base);
      a += xo * f;
      b += xl * f;
    }
    const int row = r0 + r;
    if (row < rows && d < p.D) {
      const int t = row / p.G;
      // keys the token sees: the positions before, and its drafted ones that fit the cache
      const unsigned long long fit = end - pos >= 64 ? ~0ull : end > pos ? (1ull << (end - pos)) - 1 : 0ull;
      const bool any = pos >= 0 && (pre > 0 || (s_mask[t] & fit));
      const float y = any ? a / b : 0.f;
      const int64_t at = ((n * p.S + t) * p.H * p.G + (int64_t)h * p.G + row % p.G) * p.D + d;
      if (p.bf16) ((__nv_bfloat16*)p.out)[at] = __float2bfloat16_rn(y);
      else ((float*)p.out)[at] = y;
    }
  }
  tc::cluster_sync();  // no CTA leaves while another may read its shared memory
}

template <typename CT, int LPK, int R, int U>
cudaError_t launch(const CacheAttnArgs& a, cudaStream_t stream) {
  const KvCacheView& c = a.cache;
  const int G = (int)(a.Hq / c.H), rows = (int)a.S * G, chunks = (rows + R - 1) / R;
  Params p = {c.k, c.v, c.k_scale, c.v_scale, a.positions, a.parents, a.q, a.out, a.bf16 ? 1 : 0, (int)c.H, G, (int)a.S,
              (int)c.D, chunks, c.T, a.scale * kLog2e};
  const int64_t items = c.N * c.H * chunks;
  static const int sms = [] {
    int dev = 0, n = 148;
    if (cudaGetDevice(&dev) == cudaSuccess) cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev);
    return n;
  }();
  // split until every SM has two CTAs or a CTA has fewer than 64 positions
  int C = 1;
  while (C < 8 && items * C < 2 * sms && c.T / (2 * C) >= 32) C *= 2;
  if (items * C > INT32_MAX) return cudaErrorInvalidValue;
  const size_t smem = (size_t)(kWarps * R * (LPK * EPL + 2)) * sizeof(float);
  auto kern = cache_attn_kernel<CT, LPK, R, U>;
  if (smem > 48 * 1024) {
    cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
    if (e != cudaSuccess) return e;
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(items * C));
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute at[2];
  pdl_attribute(&at[0]);
  at[1].id = cudaLaunchAttributeClusterDimension;
  at[1].val.clusterDim.x = (unsigned)C;
  at[1].val.clusterDim.y = at[1].val.clusterDim.z = 1;
  cfg.attrs = at;
  cfg.numAttrs = 2;
  launch_counter().fetch_add(1, std::memory_order_relaxed);
  return cudaLaunchKernelEx(&cfg, kern, p);
}

template <typename CT, int LPK>
cudaError_t by_rows(const CacheAttnArgs& a, cudaStream_t stream) {
  const int64_t rows = a.S * (a.Hq / a.cache.H);
  if (rows <= 1) return launch<CT, LPK, 1, 4>(a, stream);
  if (rows <= 2) return launch<CT, LPK, 2, 4>(a, stream);
  if (rows <= 4) return launch<CT, LPK, 4, 4>(a, stream);
  return launch<CT, LPK, 8, 2>(a, stream);
}

template <typename CT>
cudaError_t by_dim(const CacheAttnArgs& a, cudaStream_t stream) {
  if (a.cache.D <= 16) return by_rows<CT, 2>(a, stream);
  if (a.cache.D <= 32) return by_rows<CT, 4>(a, stream);
  if (a.cache.D <= 64) return by_rows<CT, 8>(a, stream);
  if (a.cache.D <= 128) return by_rows<CT, 16>(a, stream);
  return by_rows<CT, 32>(a, stream);
}

}  // namespace

cudaError_t cache_attention(const CacheAttnArgs& a, cudaStream_t stream) {
  if (cache_attention_tc_takes(a)) return cache_attention_tc(a, stream);
  switch (a.cache.type) {
    case KvType::F32: return by_dim<float>(a, stream);
    case KvType::BF16: return by_dim<__nv_bfloat16>(a, stream);
    case KvType::I8: return by_dim<int8_t>(a, stream);
  }
  return cudaErrorInvalidValue;
}

}  // namespace sb
