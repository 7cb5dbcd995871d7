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
//
// It takes up to 8 rows over f32 caches, up to 3 over others of heads of 32 or less,
// and every call of heads over 128.
// One row of 4 x 8 f32 caches of 30K keys of 128: 148 us, 6.6 TB/s, as fast as a
// copy; of 64 x 12 caches of 512 keys of 64: 38 us, 5.4 TB/s; of one sequence of
// 200 keys, 6 heads: 4.1 us, launch and latency.  From 4 rows on the FMAs and the
// butterflies bound it (16 x 8 caches of 4K keys of 128, 4 rows: 119 us, 4.4 TB/s).
#include "cache_attn.h"

namespace sb {
namespace {

using namespace cattn;

constexpr int kWarps = 8, kThreads = kWarps * 32;
constexpr int EPL = 8;

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
  asm volatile("ld.global.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];"
               : "=r"(r.a.x), "=r"(r.a.y), "=r"(r.a.z), "=r"(r.a.w)
               : "l"(p));
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

template <typename CT, int LPK, int R, int U>
__global__ void __launch_bounds__(kThreads) cache_attn_kernel(const Params p) {
  pdl_prologue();
  constexpr int KPW = 32 / LPK;   // rows of the cache a warp loads at once
  constexpr int DP = LPK * EPL;   // head size, padded
  constexpr int TK = KPW * U;
  extern __shared__ __align__(16) float sm[];  // [kWarps + 1][R][DP]
  __shared__ unsigned long long s_mask[kKvMaxTokens];
  __shared__ int s_jump[kKvMaxTokens];
  __shared__ float s_m[kWarps * R], s_l[kWarps * R], s_ml[2 * R];
  const Place w = find_place(p);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, gl = lane % LPK, grp = lane / LPK;
  if (warp == 0) tree_masks(p.parents ? p.parents + w.n * p.S : nullptr, p.S, lane, s_mask, s_jump);
  __syncthreads();

  const int r0 = w.chunk * R, rows = min(R, p.S * p.G - r0);
  float q[R][EPL], o[R][EPL], m[R], l[R];
  int tok[R];
#pragma unroll
  for (int r = 0; r < R; ++r) {
    const int row = r0 + min(r, rows - 1);
    tok[r] = row / p.G;
    const int64_t at = row_at(p, w, row) + gl * EPL;
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
  const int64_t per = (w.end + w.C - 1) / w.C, lo = min((int64_t)w.rank * per, w.end), hi = min(lo + per, w.end);
  const CT* kb = (const CT*)p.k + w.nh * p.T * p.D + gl * EPL;
  const CT* vb = (const CT*)p.v + w.nh * p.T * p.D + gl * EPL;
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
          ksc[u] = p.ks[w.nh * p.T + t];
          vsc[u] = p.vs[w.nh * p.T + t];
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
    const bool masked = t0 + TK > w.pre || t0 + TK > hi;
    uint32_t hidden = 0;  // bit u R + r: row r does not see the position
    static_assert(U * R <= 32, "a bit each");
    if (masked) {
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int64_t t = t0 + u * KPW + grp;
#pragma unroll
        for (int r = 0; r < R; ++r) {
          const bool see = t < hi && (t < w.pre || (s_mask[tok[r]] >> (t - w.pos) & 1ull));
          if (!see) s[u][r] = -INFINITY, hidden |= 1u << (u * R + r);
        }
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
        float y = s[u][r];
        if constexpr (sizeof(CT) == 1) y *= vsc[u];
        // what a row does not see may hold anything, NaN included: it adds nothing
        if (!masked || !(hidden >> (u * R + r) & 1u)) {
#pragma unroll
          for (int i = 0; i < EPL; ++i) o[r][i] = fmaf(y, x[i], o[r][i]);
        }
      }
    }
  }

  // join the groups of the warp
#pragma unroll
  for (int r = 0; r < R; ++r) {
#pragma unroll
    for (int x = LPK; x < 32; x *= 2) {
      const float m2 = __shfl_xor_sync(0xffffffffu, m[r], x), l2 = __shfl_xor_sync(0xffffffffu, l[r], x);
      const float mx = fmaxf(m[r], m2), base = mx == -INFINITY ? 0.f : mx;
      const float a = exp2f(m[r] - base), b = exp2f(m2 - base);
      l[r] = l[r] * a + l2 * b;
#pragma unroll
      for (int i = 0; i < EPL; ++i) o[r][i] = o[r][i] * a + __shfl_xor_sync(0xffffffffu, o[r][i], x) * b;
      m[r] = mx;
    }
    if (grp == 0) {
#pragma unroll
      for (int i = 0; i < EPL; ++i) sm[(warp * R + r) * DP + gl * EPL + i] = o[r][i];
      if (gl == 0) s_m[warp * R + r] = m[r], s_l[warp * R + r] = l[r];
    }
  }
  join_and_store<kWarps, R, DP>(p, w, r0, rows, sm, s_m, s_l, sm + kWarps * R * DP, s_ml, s_mask,
                                nullptr);
}

template <typename CT, int LPK, int R, int U>
cudaError_t launch(const CacheAttnArgs& a, cudaStream_t stream) {
  const Params p = make_params(a, R);
  const int64_t items = a.cache.N * a.cache.H * p.chunks;
  // Split while every SM has at most two CTAs and a CTA has 32 positions, one step of a
  // warp or two.  (96 items of 600 keys of 64: 7.2 us; up to three or four CTAs per SM,
  // which the cluster's places do not allow at once, 10.7; 128 of 4K keys of 128, 81
  // and 84; 32 of 30K keys, 148, unsplit 615.)
  int C = 1;
  while (may_double(C, items) && items * 2 * C <= 2 * sm_count() && a.cache.T / (2 * C) >= 32) C *= 2;
  const size_t smem = (size_t)((kWarps + 1) * R * LPK * EPL) * sizeof(float);
  return launch_cluster(cache_attn_kernel<CT, LPK, R, U>, items * C, C, kThreads, smem, stream, p);
}

template <typename CT, int LPK>
cudaError_t by_rows(const CacheAttnArgs& a, cudaStream_t stream) {
  const int64_t rows = a.S * (a.Hq / a.cache.H);
  // Rows of the cache under way per group: four; eight for heads over 128, of which a
  // warp holds one at a time, in 8 or 16 bits (16 x 8 caches of 3K bf16 keys of 256: 62
  // us, 82 with four; f32, twice the bytes and registers, 125 and 117).  With four
  // query rows int8 codes leave no registers for eight (32 and 38 us).
  constexpr bool NARROW = LPK == 32 && sizeof(CT) < 4;
  if (rows <= 1) return launch<CT, LPK, 1, NARROW ? 8 : 4>(a, stream);
  if (rows <= 2) return launch<CT, LPK, 2, NARROW ? 8 : 4>(a, stream);
  if constexpr (sizeof(CT) == 4 || LPK == 32)
    if (rows > 4) return launch<CT, LPK, 8, 2>(a, stream);
  return launch<CT, LPK, 4, NARROW && sizeof(CT) == 2 ? 8 : 4>(a, stream);
}

template <typename CT>
cudaError_t by_dim(const CacheAttnArgs& a, cudaStream_t stream) {
  if (a.cache.D <= 16) return by_rows<CT, 2>(a, stream);
  if (a.cache.D <= 32) return by_rows<CT, 4>(a, stream);
  if constexpr (sizeof(CT) == 4) {
    if (a.cache.D <= 64) return by_rows<CT, 8>(a, stream);
    if (a.cache.D <= 128) return by_rows<CT, 16>(a, stream);
  }
  return by_rows<CT, 32>(a, stream);
}

}  // namespace

cudaError_t cache_attention(const CacheAttnArgs& a, cudaStream_t stream) {
  if (cache_attention_mma_takes(a)) return cache_attention_mma(a, stream);
  if (cache_attention_tc_takes(a)) return cache_attention_tc(a, stream);
  if (cache_attention_tile_takes(a)) return cache_attention_tile(a, stream);
  switch (a.cache.type) {
    case KvType::F32: return by_dim<float>(a, stream);
    case KvType::BF16: return by_dim<__nv_bfloat16>(a, stream);
    case KvType::I8: return by_dim<int8_t>(a, stream);
  }
  return cudaErrorInvalidValue;
}

}  // namespace sb
