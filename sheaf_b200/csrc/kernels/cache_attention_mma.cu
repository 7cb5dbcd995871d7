// Attention of few query rows over a bf16 or int8 cache: one token whose query
// heads share a cache head, or a short draft.  Same definition as
// cache_attention.cu.
//
// Reading the cache once bounds it; on the CUDA cores the products (2 FMA per
// value and row) pass that from 2 to 4 rows on.  Here a warp multiplies with
// m16n8k16 bf16 instructions straight from the registers it loads into: no
// shared memory, no barrier in the loop.  (A tcgen05 tile has 128 rows, of
// which up to 16 would be used, and needs every tile staged and converted in
// shared memory; cache_attention_tc.cu takes over where its rows fill.)
//
//   S = Q K^T  A = Q (16 rows), B = K: lane (g, c) = (lane / 4, lane % 4) holds
//              key g's values.  The head dimension may be summed in any order,
//              so a lane takes consecutive values (one 16-byte load: 8 bf16 or
//              16 codes) and Q is laid out to match.
//   O += P V   A = P: the accumulators of S are its operand layout already.  B
//              pairs two keys of one column: lane (g, c) loads consecutive
//              columns of keys 2c, 2c + 1, 2c + 8, 2c + 9 and pairs them by
//              byte permutation; the columns' order is undone at the end.
//
// f32 queries: a value is the sum of three bf16 parts, exactly.  With at most
// four rows the parts fill the 16 rows of A (0-3 first, 8-11 second, 4-7 third
// part), so f32 accuracy costs no more instructions; S is the sum over a
// lane's two rows and its partner's.  P is split the same way, and the parts'
// products accumulate apart.
//
// int8 codes become bf16 exactly (see codes below); key scales multiply S,
// value scales P.
#include "cache_attn.h"

namespace sb {
namespace {

using namespace cattn;

constexpr int kWarps = 4, kThreads = kWarps * 32;
constexpr float kLazy = 8.f;  // a row's maximum moves when it would grow by more than this (log2)

__device__ __forceinline__ void mma16816(float* d, const uint32_t* a, uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {
  uint32_t d;
  asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(d) : "f"(hi), "f"(lo));
  return d;
}
__device__ __forceinline__ float bf_lo(uint32_t w) { return __uint_as_float(w << 16); }
__device__ __forceinline__ float bf_hi(uint32_t w) { return __uint_as_float(w & 0xffff0000u); }

// Two codes, in bytes 0 and 2 of t (bytes 1 and 3: anything), to two bf16
// values.  A code's low 7 bits and its sign bit, each put under the exponent of
// 128 (bf16 steps of 1 from 128 to 256), differ by the code:
// (128 + low) - (128 or 256) = code, exactly.
__device__ __forceinline__ uint32_t codes(uint32_t t) {
  const uint32_t a = (t & 0x007f007fu) | 0x43004300u, b = (t & 0x00800080u) | 0x43004300u;
  __nv_bfloat162 x = __hsub2(*(const __nv_bfloat162*)&a, *(const __nv_bfloat162*)&b);
  return *(uint32_t*)&x;
}

__device__ __forceinline__ uint4 load16(const void* p) {
  uint4 r;
  asm volatile("ld.global.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];"
               : "=r"(r.x), "=r"(r.y), "=r"(r.z), "=r"(r.w)
               : "l"(p));
  return r;
}
__device__ __forceinline__ uint2 load8(const void* p) {
  uint2 r;
  asm volatile("ld.global.L1::no_allocate.v2.u32 {%0, %1}, [%2];" : "=r"(r.x), "=r"(r.y) : "l"(p));
  return r;
}

// Takes values that are not finite out of a word of two bf16.
__device__ __forceinline__ uint32_t finite_only(uint32_t w, bool& bad) {
  if ((w & 0x7f80u) == 0x7f80u) w &= 0xffff0000u, bad = true;
  if ((w & 0x7f800000u) == 0x7f800000u) w &= 0xffffu, bad = true;
  return w;
}

// DP: head size padded to 64 or 128.  Q32: f32 queries, at most 4 rows; else
// bf16 queries, at most 16.
template <int DP, bool I8, bool Q32>
struct MmaCfg {
  static constexpr int RMAX = Q32 ? 4 : 16, NR = Q32 ? 1 : 2;  // rows of the CTA, of a lane
  static constexpr int KB = I8 ? 32 : 16;                      // keys per step
  static constexpr int EK = I8 ? 16 : 8;                       // values of a lane's K load
  static constexpr int KL = DP / (4 * EK);                     // K loads per key
  static constexpr int EV = I8 ? DP / 8 : 8;                   // values of a lane's V load
  static constexpr int VL = DP / (8 * EV);                     // V loads per key
  static constexpr int SMEM = (kWarps + 1) * RMAX * DP * 4;
};

template <int DP, bool I8, bool Q32>
__global__ void __launch_bounds__(kThreads) cache_attn_mma(const Params p) {
  using F = MmaCfg<DP, I8, Q32>;
  constexpr int KB = F::KB, NB = KB / 8, KG = KB / 16, EK = F::EK, KL = F::KL, VL = F::VL, NR = F::NR, RMAX = F::RMAX;
  constexpr int ES = I8 ? 1 : 2;  // bytes per value
  pdl_prologue();
  extern __shared__ __align__(16) float sm[];
  __shared__ unsigned long long s_mask[kKvMaxTokens];
  __shared__ int s_jump[kKvMaxTokens];
  __shared__ float s_m[kWarps * RMAX], s_l[kWarps * RMAX], s_ml[2 * RMAX];
  __shared__ int s_bad;
  const Place w = find_place(p);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, c = lane & 3;
  const int r0 = w.chunk * RMAX, rows = min(RMAX, p.S * p.G - r0);
  // this CTA's keys, in whole steps of the warps' stride
  const int64_t per = ((w.end + w.C - 1) / w.C + KB - 1) / KB * KB;
  const int64_t lo = min((int64_t)w.rank * per, w.end), hi = min(lo + per, w.end);

  const uint8_t* kb = (const uint8_t*)p.k + w.nh * p.T * p.D * ES;
  const uint8_t* vb = (const uint8_t*)p.v + w.nh * p.T * p.D * ES;
  const float *ksb = I8 ? p.ks + w.nh * p.T : nullptr, *vsb = I8 ? p.vs + w.nh * p.T : nullptr;
  const int64_t rs = (int64_t)p.D * ES;
  uint4 kr[NB][KL];
  uint4 vr[KG][4][VL];
  float ks[NB][2], vs[NB][2];
  auto load_k = [&](int64_t t0) {
#pragma unroll
    for (int b = 0; b < NB; ++b) {
      const int64_t t = t0 + b * 8 + g;
#pragma unroll
      for (int i = 0; i < KL; ++i) {
        const int d = i * 4 * EK + c * EK;
        kr[b][i] = make_uint4(0, 0, 0, 0);
        if (t < hi && d < p.D) kr[b][i] = load16(kb + t * rs + d * ES);
      }
      if (I8) {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const int64_t t2 = t0 + b * 8 + 2 * c + i;
          ks[b][i] = t2 < hi ? ksb[t2] : 0.f;
        }
      }
    }
  };
  auto load_v = [&](int64_t t0) {
#pragma unroll
    for (int k = 0; k < KG; ++k)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int64_t t = t0 + k * 16 + 2 * c + (i & 1) + (i >> 1) * 8;
#pragma unroll
        for (int j = 0; j < VL; ++j) {
          const int d = j * 8 * F::EV + g * F::EV;
          vr[k][i][j] = make_uint4(0, 0, 0, 0);
          if (t < hi && d < p.D) {
            if (F::EV * ES == 8) {
              const uint2 x = load8(vb + t * rs + d * ES);
              vr[k][i][j].x = x.x, vr[k][i][j].y = x.y;
            } else {
              vr[k][i][j] = load16(vb + t * rs + d * ES);
            }
          }
        }
      }
    if (I8) {
#pragma unroll
      for (int b = 0; b < NB; ++b)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const int64_t t = t0 + b * 8 + 2 * c + i;
          vs[b][i] = t < hi ? vsb[t] : 0.f;
        }
    }
  };
  int64_t t0 = lo + warp * KB;
  load_k(t0);
  load_v(t0);
  if (warp == 0) tree_masks(p.parents ? p.parents + w.n * p.S : nullptr, p.S, lane, s_mask, s_jump);
  if (tid == 0) s_bad = 0;

  // Q: k-step s takes values d .. d + 3 of the lane's EK
  uint32_t q[DP / 16][4];
#pragma unroll
  for (int s = 0; s < DP / 16; ++s) {
    const int d = (s / (EK / 4)) * 4 * EK + c * EK + (s % (EK / 4)) * 4;
    if (Q32) {
      const int row = g & 3;
      float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
      if (row < rows && d < p.D) x = *(const float4*)((const float*)p.q + row_at(p, w, r0 + row) + d);
      const float y[4] = {x.x * p.scale2, x.y * p.scale2, x.z * p.scale2, x.w * p.scale2};
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const uint32_t a = pack_bf16(y[2 * i], y[2 * i + 1]);
        const float e0 = y[2 * i] - bf_lo(a), e1 = y[2 * i + 1] - bf_hi(a);
        const uint32_t b = pack_bf16(e0, e1), l3 = pack_bf16(e0 - bf_lo(b), e1 - bf_hi(b));
        q[s][2 * i] = g < 4 ? a : l3;
        q[s][2 * i + 1] = g < 4 ? b : 0u;
      }
    } else {
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        const int row = g + 8 * r;
        uint2 x = make_uint2(0, 0);
        if (row < rows && d < p.D) x = *(const uint2*)((const __nv_bfloat16*)p.q + row_at(p, w, r0 + row) + d);
        q[s][r] = x.x;
        q[s][2 + r] = x.y;
      }
    }
  }
  __syncthreads();
  unsigned long long seen[NR];
#pragma unroll
  for (int r = 0; r < NR; ++r) seen[r] = s_mask[min(r0 + (Q32 ? g & 3 : g + 8 * r), p.S * p.G - 1) / p.G];

  float o[DP / 8][4], m[NR], l[NR];
#pragma unroll
  for (int j = 0; j < DP / 8; ++j) o[j][0] = o[j][1] = o[j][2] = o[j][3] = 0.f;
#pragma unroll
  for (int r = 0; r < NR; ++r) m[r] = -INFINITY, l[r] = 0.f;

  for (; t0 < hi; t0 += kWarps * KB) {
    float s[NB][4];
#pragma unroll
    for (int b = 0; b < NB; ++b) s[b][0] = s[b][1] = s[b][2] = s[b][3] = 0.f;
#pragma unroll
    for (int k = 0; k < DP / 16; ++k)
#pragma unroll
      for (int b = 0; b < NB; ++b) {
        const uint4& x = kr[b][k / (EK / 4)];
        const uint32_t word[4] = {x.x, x.y, x.z, x.w};
        if (I8) {
          const uint32_t y = word[k % 4];
          mma16816(s[b], q[k], codes(__byte_perm(y, 0, 0x4140)), codes(__byte_perm(y, 0, 0x4342)));
        } else {
          mma16816(s[b], q[k], word[(k % 2) * 2], word[(k % 2) * 2 + 1]);
        }
      }
    // scores of the lane's NR rows and two keys per block, in units of log2
    float x[NB][NR][2];
#pragma unroll
    for (int b = 0; b < NB; ++b)
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        if (Q32) {
          const float y = s[b][i] + s[b][2 + i];
          x[b][0][i] = y + __shfl_xor_sync(0xffffffffu, y, 16);
        } else {
#pragma unroll
          for (int r = 0; r < NR; ++r) x[b][r][i] = s[b][2 * r + i] * p.scale2;
        }
        if (I8)
#pragma unroll
          for (int r = 0; r < NR; ++r) x[b][r][i] *= ks[b][i];
      }
    const int64_t tn = t0 + kWarps * KB;
    load_k(tn);  // under way during the softmax and the second product
    const bool masked = t0 + KB > w.pre || t0 + KB > hi;
    if (masked) {
      bool bad = false;
#pragma unroll
      for (int b = 0; b < NB; ++b)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const int64_t t = t0 + b * 8 + 2 * c + i;
#pragma unroll
          for (int r = 0; r < NR; ++r) {
            const bool see = t < hi && (t < w.pre || (seen[r] >> (t - w.pos) & 1ull));
            if (!see) x[b][r][i] = -INFINITY;
          }
        }
      if (!I8) {
#pragma unroll
        for (int k = 0; k < KG; ++k)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int64_t t = t0 + k * 16 + 2 * c + (i & 1) + (i >> 1) * 8;
            if (t >= w.pre)
#pragma unroll
              for (int j = 0; j < VL; ++j) {
                uint4& y = vr[k][i][j];
                y = make_uint4(finite_only(y.x, bad), finite_only(y.y, bad), finite_only(y.z, bad),
                               finite_only(y.w, bad));
              }
          }
        if (bad) s_bad = 1;
      }
    }
    float mx[NR];
    bool move = false;
#pragma unroll
    for (int r = 0; r < NR; ++r) {
      mx[r] = -INFINITY;
#pragma unroll
      for (int b = 0; b < NB; ++b) mx[r] = fmaxf(mx[r], fmaxf(x[b][r][0], x[b][r][1]));
      mx[r] = fmaxf(mx[r], __shfl_xor_sync(0xffffffffu, mx[r], 1));
      mx[r] = fmaxf(mx[r], __shfl_xor_sync(0xffffffffu, mx[r], 2));
      move |= mx[r] > m[r] + kLazy;
    }
    if (__any_sync(0xffffffffu, move)) {
#pragma unroll
      for (int r = 0; r < NR; ++r) {
        const float mn = fmaxf(m[r], mx[r]), f = mn == -INFINITY ? 0.f : tc::ex2(m[r] - mn);
        l[r] *= f;
        m[r] = mn;
#pragma unroll
        for (int j = 0; j < DP / 8; ++j) {
          o[j][2 * r] *= f, o[j][2 * r + 1] *= f;
          if (Q32) o[j][2] *= f, o[j][3] *= f;
        }
      }
    }
    uint32_t a[KG][4];
#pragma unroll
    for (int b = 0; b < NB; ++b)
#pragma unroll
      for (int r = 0; r < NR; ++r) {
        const float base = m[r] == -INFINITY ? 0.f : m[r];
        float y[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const float e = tc::ex2(x[b][r][i] - base);
          l[r] += e;
          y[i] = I8 ? (masked && x[b][r][i] == -INFINITY ? 0.f : e * vs[b][i]) : e;
        }
        uint32_t* dst = &a[b / 2][(b & 1) * 2];
        const uint32_t h1 = pack_bf16(y[0], y[1]);
        if (Q32) {
          const float e0 = y[0] - bf_lo(h1), e1 = y[1] - bf_hi(h1);
          const uint32_t h2 = pack_bf16(e0, e1), h3 = pack_bf16(e0 - bf_lo(h2), e1 - bf_hi(h2));
          dst[0] = g < 4 ? h1 : h3;
          dst[1] = g < 4 ? h2 : 0u;
        } else {
          dst[r] = h1;
        }
      }
#pragma unroll
    for (int k = 0; k < KG; ++k)
#pragma unroll
      for (int j = 0; j < VL; ++j) {
        uint32_t word[4][4];
#pragma unroll
        for (int i = 0; i < 4; ++i)
          word[i][0] = vr[k][i][j].x, word[i][1] = vr[k][i][j].y, word[i][2] = vr[k][i][j].z, word[i][3] = vr[k][i][j].w;
#pragma unroll
        for (int e = 0; e < F::EV; ++e) {
          uint32_t b[2];
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            if (I8) {
              const int by = e % 4;
              b[i] = codes(__byte_perm(word[2 * i][e / 4], word[2 * i + 1][e / 4], by * 0x11 | (by + 4) * 0x1100));
            } else {
              b[i] = __byte_perm(word[2 * i][e / 2], word[2 * i + 1][e / 2], e & 1 ? 0x7632 : 0x5410);
            }
          }
          mma16816(o[j * F::EV + e], a[k], b[0], b[1]);
        }
      }
    load_v(tn);
  }

  // the warp's parts: row, and columns 2c, 2c + 1 of block (j, e) = value (2c) EV + e of load j
#pragma unroll
  for (int r = 0; r < NR; ++r) {
    l[r] += __shfl_xor_sync(0xffffffffu, l[r], 1);
    l[r] += __shfl_xor_sync(0xffffffffu, l[r], 2);
    const int row = Q32 ? g & 3 : g + 8 * r;
    if (c == 0 && (!Q32 || g < 4)) s_m[warp * RMAX + row] = m[r], s_l[warp * RMAX + row] = l[r];
#pragma unroll
    for (int j = 0; j < DP / 8; ++j)
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        float y = o[j][2 * r + i];
        if (Q32) {
          y += o[j][2 + i];
          y += __shfl_xor_sync(0xffffffffu, y, 16);
        }
        const int d = (j / F::EV) * 8 * F::EV + (2 * c + i) * F::EV + j % F::EV;
        if (!Q32 || g < 4) sm[(warp * RMAX + row) * DP + d] = y;
      }
  }
  int bad = 0;
  if (!I8) {
    // a drafted value that is not finite reaches the rows that see it: whichever CTA read it
    __syncthreads();
    if (w.C > 1) tc::cluster_sync();
    for (uint32_t r = 0; r < w.C; ++r) {
      int y;
      asm volatile("ld.shared::cluster.s32 %0, [%1];" : "=r"(y) : "r"(tc::cluster_addr(&s_bad, r)));
      bad |= y;
    }
  }
  join_and_store<kWarps, RMAX, DP>(
      p, w, r0, rows, sm, s_m, s_l, sm + kWarps * RMAX * DP, s_ml, s_mask, [&](unsigned long long see, int d, float* y) {
        if (!bad) return;
        for (int j = 0; j < p.S; ++j)
          if (see >> j & 1ull)
            for (int i = 0; i < 4; ++i) {
              const float v = __bfloat162float(((const __nv_bfloat16*)p.v)[(w.nh * p.T + w.pos + j) * p.D + d + i]);
              if (!isfinite(v)) y[i] += v;
            }
      });
}

template <int DP, bool I8, bool Q32>
cudaError_t launch(const CacheAttnArgs& a, cudaStream_t stream) {
  using F = MmaCfg<DP, I8, Q32>;
  const Params p = make_params(a, F::RMAX);
  const int64_t items = a.cache.N * a.cache.H * p.chunks;
  // split until the SMs hold their CTAs twice over, or a warp would have one step
  int C = 1;
  while (C < kMaxCluster && items * C < 3 * sm_count() && a.cache.T / (2 * C) >= kWarps * F::KB) C *= 2;
  return launch_cluster(cache_attn_mma<DP, I8, Q32>, items * C, C, kThreads, F::SMEM, stream, p);
}

}  // namespace

bool cache_attention_mma_takes(const CacheAttnArgs& a) {
  return a.cache.type != KvType::F32 && a.cache.D >= 64 && a.cache.D <= 128 &&
         a.S * (a.Hq / a.cache.H) <= (a.bf16 ? 16 : 4);
}

cudaError_t cache_attention_mma(const CacheAttnArgs& a, cudaStream_t stream) {
  const bool i8 = a.cache.type == KvType::I8;
  if (a.cache.D <= 64) {
    if (a.bf16) return i8 ? launch<64, true, false>(a, stream) : launch<64, false, false>(a, stream);
    return i8 ? launch<64, true, true>(a, stream) : launch<64, false, true>(a, stream);
  }
  if (a.bf16) return i8 ? launch<128, true, false>(a, stream) : launch<128, false, false>(a, stream);
  return i8 ? launch<128, true, true>(a, stream) : launch<128, false, true>(a, stream);
}

}  // namespace sb
