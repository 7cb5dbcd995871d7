// Attention of many query rows over an f32 cache, whose products take all 24 bits,
// on the CUDA cores.  Same definition as cache_attention.cu.
//
// That kernel holds 8 query rows in registers and reads the cache once per 8
// rows.  Here a CTA of W warps takes 8 W rows, and tiles of 64 keys pass through two
// stages of asynchronous copies, each read once for all rows.
//   S: a lane has two keys and the warp's 8 rows; per 4 values of the head a
//      16-byte load per key and a broadcast per row feed 64 FMAs.
//   softmax: a row's maximum is the warp's (one redux); each lane sums its own
//      keys.  P goes to shared memory, 8 rows of a key together.
//   O: a lane has DP / 32 columns of the 8 rows; a key's P is two broadcasts.
// Shared memory's 128 bytes per cycle to registers bound it (a broadcast costs as
// much as any load).  Lanes of 8 rows x 4 keys halve those loads, but leave one
// warp per SM quarter, and were slower.  8 x 12 f32 caches of 663 keys of 64,
// 63 rows each (27 us of FMAs): 59 us, against 107 by the other kernel; 4 x 8
// caches of 8K keys of 128, 128 rows: 554 against 1374.
#include "cache_attn.h"

namespace sb {
namespace {

using namespace cattn;

constexpr int RW = 8;                  // rows of a warp
constexpr int KPL = 2, BN = 32 * KPL;  // keys of a lane and of a tile

template <int DP, int W>
struct TileCfg {
  static constexpr int DPL = DP / 32, R = W * RW;         // output columns of a lane, rows of the CTA
  static constexpr int ROW = DP * 4 + 16;   // bytes; lanes' rows start in different banks
  static constexpr int TILE = BN * ROW, STAGE = 2 * TILE;  // K and V
  static constexpr int KV_OFF = R * DP * 4, P_OFF = KV_OFF + 2 * STAGE, SMEM = P_OFF + W * BN * RW * 4;
};

// N consecutive values from shared memory.
template <int N>
__device__ __forceinline__ void take(const void* p, float* x) {
  struct alignas(N * 4) Vec {
    float v[N];
  };
  const Vec y = *(const Vec*)p;
#pragma unroll
  for (int i = 0; i < N; ++i) x[i] = y.v[i];
}

__device__ __forceinline__ float warp_max(float x) {
  float y;
  asm volatile("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(y) : "f"(x));
  return y;
}

template <int DP, int W>
__global__ void __launch_bounds__(W * 32) cache_attn_tile(const Params p) {
  using F = TileCfg<DP, W>;
  constexpr int DPL = F::DPL, R = F::R, ROW = F::ROW;
  pdl_prologue();
  extern __shared__ __align__(16) uint8_t sm[];
  __shared__ unsigned long long s_mask[kKvMaxTokens];
  __shared__ int s_jump[kKvMaxTokens], s_tok[R];
  __shared__ int64_t s_at[R];  // where a row stands in q
  __shared__ float s_m[R], s_l[R], s_ml[2 * R];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const Place w = find_place(p);
  const int r0 = w.chunk * R, rows = min(R, p.S * p.G - r0);
  float* const sq = (float*)sm;
  float* const sp = (float*)(sm + F::P_OFF) + warp * BN * RW;

  // this CTA's positions, in whole tiles
  const int64_t per = ((w.end + w.C - 1) / w.C + BN - 1) / BN * BN;
  const int64_t lo = min((int64_t)w.rank * per, w.end), hi = min(lo + per, w.end);
  const uint8_t* const kb = (const uint8_t*)p.k + w.nh * p.T * p.D * (int64_t)4;
  const uint8_t* const vb = (const uint8_t*)p.v + w.nh * p.T * p.D * (int64_t)4;
  constexpr int PIECES = DP * 4 / 16;  // 16-byte pieces of a row, padded
  const int u = tid % PIECES, key0 = tid / PIECES;
  constexpr int KSTEP = W * 32 / PIECES;
  static_assert(W * 32 % PIECES == 0, "whole rows per step");
  const bool has = u * 16 < p.D * 4;
  // Keys t .. t + BN into stage `st`, zeros behind the last one.
  auto fetch = [&](int64_t t, int st) {
    const uint32_t dst = tc::smem_u32(sm + F::KV_OFF + st * F::STAGE) + key0 * ROW + u * 16;
    const int64_t at = (t + key0) * p.D * (int64_t)4 + u * 16;
    if (!has) return;
#pragma unroll
    for (int k = 0; k < BN; k += KSTEP) {
      if (KSTEP > BN && key0 >= BN) break;
      const bool in = t + key0 + k < hi;
      const int64_t from = in ? at + (int64_t)k * p.D * 4 : 0;
      asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst + k * ROW), "l"(kb + from), "r"(in ? 16 : 0)
                   : "memory");
      asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst + F::TILE + k * ROW), "l"(vb + from),
                   "r"(in ? 16 : 0)
                   : "memory");
    }
  };
  auto commit = [] { asm volatile("cp.async.commit_group;" ::: "memory"); };
  if (tid < R) {
    s_tok[tid] = min(r0 + tid, p.S * p.G - 1) / p.G;
    s_at[tid] = row_at(p, w, r0 + min(tid, rows - 1));
  }
  if (lo < hi) fetch(lo, 0);
  commit();
  __syncthreads();
  // queries times scale log2(e)
#pragma unroll 4
  for (int i = tid; i < R * (DP / 4); i += W * 32) {
    const int r = i / (DP / 4), d = i % (DP / 4) * 4;
    float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
    if (r < rows && d < p.D) {
      const int64_t at = s_at[r] + d;
      if (p.bf16) {
        const uint2 z = *(const uint2*)((const __nv_bfloat16*)p.q + at);
        const float2 a = unpack2<false>(z.x), b = unpack2<false>(z.y);
        x = make_float4(a.x, a.y, b.x, b.y);
      } else {
        x = *(const float4*)((const float*)p.q + at);
      }
    }
    *(float4*)(sq + r * DP + d) = make_float4(x.x * p.scale2, x.y * p.scale2, x.z * p.scale2, x.w * p.scale2);
  }
  if (warp == 0) tree_masks(p.parents ? p.parents + w.n * p.S : nullptr, p.S, lane, s_mask, s_jump);

  float o[RW][DPL], m[RW], l[RW];
#pragma unroll
  for (int r = 0; r < RW; ++r) {
    m[r] = -INFINITY, l[r] = 0.f;
#pragma unroll
    for (int i = 0; i < DPL; ++i) o[r][i] = 0.f;
  }
  const int row0 = warp * RW;  // the warp's first row
  const float* const wq = sq + row0 * DP;
  int st = 0;
  for (int64_t t0 = lo; t0 < hi; t0 += BN, st ^= 1) {
    if (t0 + BN < hi) fetch(t0 + BN, st ^ 1);
    commit();
    asm volatile("cp.async.wait_group 1;" ::: "memory");
    __syncthreads();
    if (warp * RW < rows) {
      const uint8_t* const tk = sm + F::KV_OFF + st * F::STAGE;
      const uint8_t* const tv = tk + F::TILE + lane * DPL * 4;
      float s[RW][KPL];
#pragma unroll
      for (int r = 0; r < RW; ++r)
#pragma unroll
        for (int j = 0; j < KPL; ++j) s[r][j] = 0.f;
#pragma unroll 1
      for (int d0 = 0; d0 < p.D; d0 += 16)
#pragma unroll
        for (int d = d0; d < d0 + 16; d += 4) {
          float k[KPL][4];
#pragma unroll
          for (int j = 0; j < KPL; ++j) take<4>(tk + (32 * j + lane) * ROW + d * 4, k[j]);
#pragma unroll
          for (int r = 0; r < RW; ++r) {
            const float4 q = *(const float4*)(wq + r * DP + d);
#pragma unroll
            for (int j = 0; j < KPL; ++j) {
              s[r][j] = fmaf(q.x, k[j][0], s[r][j]);
              s[r][j] = fmaf(q.y, k[j][1], s[r][j]);
              s[r][j] = fmaf(q.z, k[j][2], s[r][j]);
              s[r][j] = fmaf(q.w, k[j][3], s[r][j]);
            }
          }
        }
      const bool masked = t0 + BN > w.pre || t0 + BN > hi;
#pragma unroll
      for (int r = 0; r < RW; ++r) {
        bool hidden[KPL] = {};
        if (masked) {
          const unsigned long long seen = s_mask[s_tok[row0 + r]];
#pragma unroll
          for (int j = 0; j < KPL; ++j) {
            const int64_t t = t0 + 32 * j + lane;
            hidden[j] = !(t < hi && (t < w.pre || (seen >> (t - w.pos) & 1ull)));
            if (hidden[j]) s[r][j] = -INFINITY;
          }
        }
        const float mx = warp_max(fmaxf(s[r][0], s[r][1]));
        if (mx > m[r]) {
          const float f = tc::ex2(m[r] - mx);
          l[r] *= f;
#pragma unroll
          for (int i = 0; i < DPL; ++i) o[r][i] *= f;
          m[r] = mx;
        }
        const float base = m[r] == -INFINITY ? 0.f : m[r];
#pragma unroll
        for (int j = 0; j < KPL; ++j) {
          s[r][j] = tc::ex2(s[r][j] - base);
          l[r] += s[r][j];
          if (masked && hidden[j]) s[r][j] = -0.f;  // no probability: what the position holds does not matter, NaN included
        }
      }
#pragma unroll
      for (int j = 0; j < KPL; ++j)
#pragma unroll
        for (int r = 0; r < RW; r += 4)
          *(float4*)(sp + (32 * j + lane) * RW + r) = make_float4(s[r][j], s[r + 1][j], s[r + 2][j], s[r + 3][j]);
      __syncwarp();
      auto add = [&](auto masked_tag) {
        constexpr bool MASK = decltype(masked_tag)::value;
#pragma unroll 4
        for (int key = 0; key < BN; ++key) {
          float v[DPL], y[RW];
          take<DPL>(tv + key * ROW, v);
          take<4>(sp + key * RW, y);
          take<4>(sp + key * RW + 4, y + 4);
#pragma unroll
          for (int r = 0; r < RW; ++r)
            if (!MASK || __float_as_uint(y[r]) != 0x80000000u)
#pragma unroll
              for (int i = 0; i < DPL; ++i) o[r][i] = fmaf(y[r], v[i], o[r][i]);
        }
      };
      if (masked) add(std::true_type{});
      else add(std::false_type{});
    }
    __syncthreads();  // the stage has been read
  }
  asm volatile("cp.async.wait_group 0;" ::: "memory");
  __syncthreads();  // the queries have been read too: their memory takes the partial outputs
#pragma unroll
  for (int r = 0; r < RW; ++r) {
#pragma unroll
    for (int x = 16; x; x >>= 1) l[r] += __shfl_xor_sync(0xffffffffu, l[r], x);
    if (lane == 0) s_m[row0 + r] = m[r], s_l[row0 + r] = l[r];
#pragma unroll
    for (int i = 0; i < DPL; ++i) sq[(row0 + r) * DP + lane * DPL + i] = o[r][i];
  }
  join_and_store<W, R, DP, 1>(p, w, r0, rows, sq, s_m, s_l, sq, s_ml, s_mask, nullptr);
}

template <int DP, int W>
cudaError_t launch(const CacheAttnArgs& a, cudaStream_t stream) {
  using F = TileCfg<DP, W>;
  const Params p = make_params(a, F::R);
  const int64_t items = a.cache.N * a.cache.H * p.chunks;
  // Split until the CTAs fill the SMs (228 KB of shared memory each) or have one
  // tile.  Clusters do not pack into every place: with more than three quarters of
  // them taken a second wave followed (96 items of 3 CTAs, 2 per SM: 77 us, of 2: 64).
  const int per_sm = (228 << 10) / (F::SMEM + (4 << 10));
  int C = 1;
  while (C < kPortable && items * (C + 1) * 4 <= (per_sm > 1 ? 3 * per_sm : 4) * sm_count() &&
         a.cache.T / (C + 1) >= BN)
    ++C;
  if (C == kPortable && may_double(C, items) && a.cache.T / (2 * C) >= BN) C *= 2;
  return launch_cluster(cache_attn_tile<DP, W>, items * C, C, W * 32, F::SMEM, stream, p);
}

}  // namespace

// 9 rows: 30 us against 37 (8 x 12 caches of 609 keys of 64), 9.0 against 8.0 for
// the smallest calls.
bool cache_attention_tile_takes(const CacheAttnArgs& a) {
  return a.cache.type == KvType::F32 && a.cache.D <= 128 && a.S * (a.Hq / a.cache.H) > 8;
}

cudaError_t cache_attention_tile(const CacheAttnArgs& a, cudaStream_t stream) {
  const bool few = a.S * (a.Hq / a.cache.H) <= 32;
  if (a.cache.D <= 32) return few ? launch<32, 4>(a, stream) : launch<32, 8>(a, stream);
  if (a.cache.D <= 64) return few ? launch<64, 4>(a, stream) : launch<64, 8>(a, stream);
  return few ? launch<128, 4>(a, stream) : launch<128, 8>(a, stream);
}

}  // namespace sb
