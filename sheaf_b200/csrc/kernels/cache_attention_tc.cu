// Attention of a chain or tree of drafted tokens over a bf16 or int8 cache on
// the tcgen05 tensor cores.  Same definition as cache_attention.cu; used where
// many query rows (tokens x query heads that share a cache head) read the same
// keys, so that the products and not the loads bound the CUDA cores.
//
// A cluster of C CTAs carries up to 256 rows of one (slot, cache head); the
// key tiles are split over its CTAs.  A CTA runs two softmax streams of four
// warps, each with its own S tile and O accumulator in TMEM:
//   more than 128 rows: stream a takes rows 128 a .., both read every tile;
//   otherwise:          stream a takes the tiles of parity a, both with the
//                       same rows (their results are joined at the end); with
//                       at most 64 rows stream 1 uses the upper half of the
//                       TMEM lanes, so the two use different SM quarters.
// While one stream turns S into P the tensor cores work for the other.  Warp
// roles: 8 softmax, 4 loading, 2 issuing the MMAs, 1 for copies and scales.
//
//   S = Q K^T   f32 queries are split exactly into three bf16 (f16) parts whose
//               products accumulate into the same f32 S, so S has f32 accuracy.
//               For int8 caches all operands are f16, which holds codes exactly
//               and takes half the instructions to make from them.  S has two
//               buffers: the tensor cores form the next one during the softmax.
//   P           exp2(S - m) times the value row's int8 scale, written back over
//               S in TMEM as parts: three for f32 output (f32 accuracy), two of
//               bf16 for bf16 output (2^-16 of each probability is left out; one
//               part, 2^-8, would be as far off as the output's own rounding, with
//               80 us for the 8 x 4 caches of 16K below in place of 95), one of f16
//               for bf16 output of int8 caches (2^-11 is left out, an eighth of the
//               output's rounding; a second part took 142 us in place of 122).
//   O += P V    the maximum m a row refers to moves only when it would grow by
//               more than 2^8, so O is rescaled in the first tiles and then
//               hardly ever; exact since P, O and the sum l share m.
//
// bf16 tiles arrive by TMA, int8 tiles through registers (codes to f16 on the way
// to swizzled shared memory).  Rows of V behind the last token are zeroed
// (0 x NaN would reach every row); a value of a drafted token that is not
// finite is taken out of the tile and added to the rows that attend to it when
// the outputs are joined.
//
// 8 x 4 caches of 16K keys of 128, 256 bf16 rows (69 GFLOP, 41 us of tensor time,
// 61 with both parts of P; bf16 cache 22 us of reading): 95 us from bf16; 124 us
// from int8, held by the softmax (two more multiplications per score) and the
// conversion.  f32 queries have three times the products: 198 and 294 us.  63 f32
// rows over 8 x 12 caches of 1K keys of 64: 22 and 30 us, of which 12 are there
// without a cache: the launch, the staging of the queries, the cluster's join.
//
// Every mbarrier wait is bounded.  TMEM is freed before the cluster barrier: a
// CTA that holds TMEM never waits for another CTA.
#include <type_traits>

#include "cache_attn.h"

namespace sb {
namespace {

using namespace cattn;
using namespace tc;

// warps 0-7 softmax, 8-11 loading (int8: conversion), 12 and 13 MMA issue (one
// per stream), 14 copies and scales; all but 12-14 stage the queries first, 15
// also builds the drafted tokens' masks
constexpr int kSoftWarps = 8, kLoadWarps = 4, kMmaWarp = 12, kFeedWarp = 14, kWarps = 16, kThreads = kWarps * 32;
constexpr int kStageWarps = kSoftWarps + kLoadWarps;
constexpr int kLoadThreads = kLoadWarps * 32;
constexpr int BN = 64;  // keys of a tile
// Sums of query x code stay below 2^30: times a key scale below this they are finite.
constexpr float kBigScale = 1.2379400392853803e27f;  // 2^90
constexpr float kLazy = 8.f;  // a row's maximum moves when it would grow by more than this (log2)

// MMAs and commits issued by one elected lane of a converged warp: the operands
// stay in uniform registers.  (Issued from a branch that one lane takes, each
// MMA cost about 95 cycles.)
__device__ __forceinline__ void mma_ss(uint32_t tmem_d, uint64_t ad, uint64_t bd, uint32_t idesc, uint32_t acc) {
  asm volatile(
      "{\n\t.reg .pred p, e;\n\t"
      "elect.sync _|e, 0xffffffff;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "@e tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(tmem_d),
      "l"(ad), "l"(bd), "r"(idesc), "r"(acc)
      : "memory");
}
// A in TMEM: 16-bit pairs, lane = row, column = two k.
__device__ __forceinline__ void mma_ts(uint32_t tmem_d, uint32_t tmem_a, uint64_t bd, uint32_t idesc, uint32_t acc) {
  asm volatile(
      "{\n\t.reg .pred p, e;\n\t"
      "elect.sync _|e, 0xffffffff;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "@e tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(tmem_d),
      "r"(tmem_a), "l"(bd), "r"(idesc), "r"(acc)
      : "memory");
}
__device__ __forceinline__ void commit(uint64_t* bar) {
  asm volatile(
      "{\n\t.reg .pred e;\n\t"
      "elect.sync _|e, 0xffffffff;\n\t"
      "@e tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}" ::"r"(smem_u32(bar))
      : "memory");
}

__device__ __forceinline__ void tmem_ld32_async(uint32_t taddr, uint32_t* r) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
      "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]),
        "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
        "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(taddr));
}
__device__ __forceinline__ void reg_fence32(uint32_t* r) {
#pragma unroll
  for (int i = 0; i < 32; ++i) asm volatile("" : "+r"(r[i]));
}
__device__ __forceinline__ void tmem_st16u(uint32_t taddr, const uint32_t* v) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};" ::"r"(
          taddr),
      "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]), "r"(v[9]),
      "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15])
      : "memory");
}

__device__ __forceinline__ void tmem_st8u(uint32_t taddr, const uint32_t* v) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"r"(taddr), "r"(v[0]),
               "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7])
               : "memory");
}

// Two f32 at once (sm_100 packed arithmetic).
__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
  float2 d;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(*(uint64_t*)&d) : "l"(*(uint64_t*)&a), "l"(*(uint64_t*)&b));
  return d;
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
  float2 d;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(*(uint64_t*)&d) : "l"(*(uint64_t*)&a), "l"(*(uint64_t*)&b));
  return d;
}
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
  float2 d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;"
      : "=l"(*(uint64_t*)&d)
      : "l"(*(uint64_t*)&a), "l"(*(uint64_t*)&b), "l"(*(uint64_t*)&c));
  return d;
}

// 16 codes to 16 f16 values; of four codes in a row the middle two change places.
__device__ __forceinline__ void codes_to_f16(const uint4& c, uint4* out) {
  out[0] = make_uint4(codes(c.x), codes(c.x >> 8), codes(c.y), codes(c.y >> 8));
  out[1] = make_uint4(codes(c.z), codes(c.z >> 8), codes(c.w), codes(c.w >> 8));
}

// kind::f16 instruction descriptor: D f32, A and B both bf16 or both f16,
// transpose bits, N>>3, M>>4.
__host__ __device__ constexpr uint32_t idesc_16(bool f16, int M, int N, int a_mn, int b_mn) {
  return (1u << 4) | (f16 ? 0u : (1u << 7) | (1u << 10)) | ((uint32_t)a_mn << 15) | ((uint32_t)b_mn << 16) |
         ((uint32_t)(N >> 3) << 17) | ((uint32_t)(M >> 4) << 24);
}

// 16-byte unit u (of 8 per 128-byte row and 64-value chunk) of row r in a
// 128-byte-swizzled tile of `rows` rows.
__device__ __forceinline__ uint32_t unit_at(int rows, int r, int unit) {
  return (uint32_t)((unit >> 3) * rows * 128 + r * 128 + (((unit & 7) ^ (r & 7)) << 4));
}

__device__ __forceinline__ void loaders_sync() { asm volatile("bar.sync 1, %0;" ::"n"(kLoadThreads) : "memory"); }

template <int DP, int QP, bool I8>
struct Cfg {
  static constexpr int MAXR = QP == 3 && DP == 128 ? 128 : 256;  // query rows of a CTA
  static constexpr int SB = QP == 3 && DP == 128 ? 1 : 2;        // buffers of S per stream
  static constexpr int PP = QP == 3 ? 3 : I8 ? 1 : 2;            // parts of P
  static constexpr int QTILE = 128 * DP * 2;                     // one part of 128 rows
  static constexpr int Q_BYTES = (MAXR / 128) * QP * QTILE;
  static constexpr int TILE = BN * DP * 2;
  static constexpr int NS = QP == 3 && DP == 128 ? 2 : 4;  // K and V tiles in flight
  // Groups of loading warps that take int8 tiles in turn.  Two, with four places: one
  // group converts while the other's loads are on their way (8 x 16K keys, 256
  // bf16 rows of 128: 124 us, against 134 with all four warps on each tile; short f32
  // calls lose, 63 rows over 1K keys of 64: 30 against 28).  With two places a group
  // would wait for its place longer.
  static constexpr int GROUPS = NS > 2 ? 2 : 1;
  static constexpr int NSC = 2 * NS;                       // rows of scales in flight (see the loader)
  static constexpr int K_OFF = Q_BYTES, V_OFF = K_OFF + NS * TILE, END = V_OFF + NS * TILE;
  static constexpr int LDO = DP + 4;  // padded row of the joined outputs, f32
  static constexpr int JOIN = 256 * LDO * 4;
  static constexpr int SMEM = END > JOIN ? END : JOIN;
  static constexpr uint32_t COLS = 512;
  // S (P's first two parts in place), O, P's third part; two streams each
  static constexpr uint32_t S_COL = 0, O_COL = 2 * SB * BN, T_COL = O_COL + 2 * DP;
  static_assert(T_COL + (QP == 3 ? SB * BN : 0) <= 512, "TMEM columns");
};

// Flags of a tile's scales.  A key scale is 2^90 or more; from this tile on rows have exponents of their own and the
// value scales stand as they are (see kEven); and rows' maxima are not lazy.
enum { kBigKey = 1, kWide = 2, kEager = 4 };

struct Shared {
  uint64_t k_full[4], k_free[4], v_full[4], v_free[4], sc_full[8], s_bar[2][2], p_bar[2][2], o_bar[2];
  uint64_t raw, mended, q_bar;
  uint32_t tslot;
  volatile int abort_flag;
  int bad;  // a drafted value that is not finite was taken out of a tile
  int q_row[256];  // query row of a staged row, in units of D values from the slot and head's first; -1: none
  // of a tile's scales: exponent that the value scales are relative to, times 8, and flags
  int sc_info[8];
  unsigned long long mask[kKvMaxTokens];
  int jump[kKvMaxTokens];
  float qs[256];                // what undoes the scaling of a query row (f16)
  float m[256], l[256], up[256];  // a row's maximum, sum, and factor of its O
  float wgt[256 * 2];  // rows of a rank x parts: at most 256 / C x C, or 128 / C x 2 C
};

// I8: int8 cache, else bf16.  QP: parts of a query (1: bf16, 3: f32).
template <int DP, int QP, bool I8>
__global__ void __launch_bounds__(kThreads, 1)
    cache_attn_tc(const __grid_constant__ CUtensorMap mK, const __grid_constant__ CUtensorMap mV, const Params p,
                  int* err) {
  using F = Cfg<DP, QP, I8>;
  constexpr bool F16 = I8;
  constexpr int SB = F::SB, NS = F::NS, NSC = F::NSC, PP = F::PP;
  pdl_prologue();
  extern __shared__ __align__(1024) uint8_t smem[];
  __shared__ Shared sh;
  __shared__ __align__(16) float sc_k[I8 ? NSC : 1][I8 ? BN : 4], sc_v[I8 ? NSC : 1][I8 ? BN : 4];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const Place w = find_place(p);
  const uint32_t rank = w.rank, C = w.C;
  const int64_t n = w.n, nh = w.nh, pos = w.pos, pre = w.pre, end = w.end;
  const int h = w.h, r0 = w.chunk * F::MAXR, rows = min(F::MAXR, p.S * p.G - r0);
  const bool split = rows > 128;                 // streams by rows, else by tiles
  const int up = !split && rows <= 64 ? 64 : 0;  // stream 1's first TMEM lane
  // this CTA's tiles [first, first + nt)
  const int tiles = (int)((end + BN - 1) / BN);
  const int first = (int)((int64_t)tiles * rank / C), nt = (int)((int64_t)tiles * (rank + 1) / C) - first;
  const bool aligned = !(smem_u32(smem) & 1023u);

  if (tid == 0) {
    for (int i = 0; i < NS; ++i) {
      mbar_init(&sh.k_full[i], I8 ? kLoadWarps / F::GROUPS : 1);
      mbar_init(&sh.v_full[i], I8 ? kLoadWarps / F::GROUPS : 1);
      mbar_init(&sh.k_free[i], split ? 2 : 1);  // the streams that read the tile
      mbar_init(&sh.v_free[i], split ? 2 : 1);
    }
    for (int i = 0; i < NSC; ++i) mbar_init(&sh.sc_full[i], 1);
    for (int a = 0; a < 2; ++a) {
      const int mine = split ? min(128, rows - 128 * a) : rows;
      for (int i = 0; i < 2; ++i) {
        mbar_init(&sh.s_bar[a][i], 1);
        mbar_init(&sh.p_bar[a][i], (uint32_t)((mine + 31) / 32));
      }
      mbar_init(&sh.o_bar[a], 1);
    }
    mbar_init(&sh.raw, 1);
    mbar_init(&sh.mended, 1);
    mbar_init(&sh.q_bar, kStageWarps + 1);
    sh.abort_flag = aligned ? 0 : 1;
    sh.bad = 0;
    if (!aligned) atomicExch(err, 50);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    fence_proxy_async();
  }
  if (warp == 0) tmem_alloc(&sh.tslot, F::COLS);
  if (tid < 256) {
    const int local = up ? tid & 63 : tid, row = r0 + local, s = row / p.G;
    sh.q_row[tid] = local < rows && tid < (split ? 256 : 128) ? s * p.H * p.G + row - s * p.G : -1;
  }
  fence_before();
  __syncthreads();
  fence_after();
  constexpr uint32_t tmem = 0;  // all 512 columns: the address is column 0
  if (tid == 0 && sh.tslot != 0) {
    atomicExch(err, 67);
    sh.abort_flag = 1;
  }
  volatile int* abort_flag = &sh.abort_flag;
  // tiles of stream a, and the i-th of them (relative to `first`)
  auto count = [&](int a) { return split ? nt : (nt - a + 1) / 2; };
  auto tile = [&](int a, int i) { return split ? i : 2 * i + a; };

  // Queries into swizzled K-major tiles: tile (row block, part) of 128 rows; one
  // block of rows repeated at lane `up` when stream 1 uses those lanes.
  // Warp `sw` of kStageWarps.  A negative scale of bf16 queries goes into their
  // signs, so that the softmax can take maxima before it scales.
  auto stage_q = [&](int sw) {
    // a thread keeps its 8-value column `u` and walks the rows
    constexpr int UNITS = DP / 8, RSTEP = kStageWarps * 32 / UNITS, LOADS = QP == 1 ? 1 : 2, BATCH = QP == 1 ? 4 : 2;
    static_assert(kStageWarps * 32 % UNITS == 0, "whole rows per step");
    const int u = lane % UNITS, total = nt > 0 && aligned ? (split ? 256 : 128) : 0;
    const uint8_t* q0 = (const uint8_t*)p.q + ((n * p.S * p.H + h) * p.G * p.D + u * 8) * (QP == 1 ? 2 : 4);
    const int row_bytes = p.D * (QP == 1 ? 2 : 4);
#pragma unroll 1
    for (int kw = sw * 32 / UNITS; kw < total; kw += BATCH * RSTEP) {  // the warp's first row of the batch
      const int k0 = kw + lane / UNITS;
      uint4 raw[BATCH][LOADS];
#pragma unroll
      for (int k = 0; k < BATCH; ++k) {
        const int at = k0 + k * RSTEP < total && u * 8 < p.D ? sh.q_row[k0 + k * RSTEP] : -1;
#pragma unroll
        for (int c = 0; c < LOADS; ++c) {
          raw[k][c] = make_uint4(0, 0, 0, 0);
          if (at >= 0) raw[k][c] = *(const uint4*)(q0 + (int64_t)at * row_bytes + 16 * c);
        }
      }
#pragma unroll
      for (int k = 0; k < BATCH; ++k) {
        const int i = k0 + k * RSTEP;
        uint8_t* dst = smem + (i >> 7) * QP * F::QTILE + unit_at(128, i & 127, u);
        if (QP == 1 && !F16) {
          const uint32_t flip = p.scale2 < 0.f ? 0x80008000u : 0u;
          const uint4 x = raw[k][0];
          if (i < total) *(uint4*)dst = make_uint4(x.x ^ flip, x.y ^ flip, x.z ^ flip, x.w ^ flip);
        } else {
          float x[8];
          if (QP == 1) {
            const uint32_t y[4] = {raw[k][0].x, raw[k][0].y, raw[k][0].z, raw[k][0].w};
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              const float2 f = unpack2<false>(y[j]);
              x[2 * j] = f.x, x[2 * j + 1] = f.y;
            }
          } else {
            *(uint4*)x = raw[k][0];
            *(uint4*)(x + 4) = raw[k][LOADS - 1];
          }
          float f = QP == 1 ? (p.scale2 < 0.f ? -1.f : 1.f) : p.scale2;
          if (F16) {
            float big = 0.f, down;
#pragma unroll
            for (int j = 0; j < 8; ++j) big = fmaxf(big, fabsf(x[j] * f));
#pragma unroll
            for (int o = UNITS / 2; o; o >>= 1) big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, o));
            const float rise = f16_row_scale(big, down);
            if (u == 0 && i < total) sh.qs[i] = QP == 1 ? down * fabsf(p.scale2) : down;
#pragma unroll
            for (int j = 0; j < 8; ++j) x[j] = x[j] * f * rise;
#pragma unroll
            for (int j = 0; j < 8; j += 4) {  // the order of the codes
              const float y = x[j + 1];
              x[j + 1] = x[j + 2], x[j + 2] = y;
            }
          } else {
#pragma unroll
            for (int j = 0; j < 8; ++j) x[j] *= f;
          }
          // x = part 0 + part 1 + part 2, each a rounding of what is left
#pragma unroll
          for (int part = 0; part < QP; ++part) {
            uint32_t y[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) y[j] = take2<F16>(x[2 * j], x[2 * j + 1]);
            if (i < total) *(uint4*)(dst + part * F::QTILE) = make_uint4(y[0], y[1], y[2], y[3]);
          }
        }
      }
    }
    fence_proxy_async();
    __syncwarp();
    if (lane == 0) mbar_arrive(&sh.q_bar);
  };

  if (warp < kSoftWarps) {
    // ------------------------------------------------------------ softmax
    stage_q(warp);
    const int a = warp >> 2, quad = warp & 3;
    const int lo_lane = split ? 0 : a * up;  // the stream's first TMEM lane
    const int mine = split ? min(128, rows - 128 * a) : rows;
    const int q0 = quad * 32 - lo_lane;  // first row of this warp within the stream
    if (q0 >= 0 && q0 < mine) {
      const int local = q0 + lane;  // row within the stream
      const int row = r0 + (split ? 128 * a : 0) + min(local, mine - 1);
      const uint32_t tl = (uint32_t)(quad * 32) << 16;
      const uint32_t tO = tmem + tl + F::O_COL + (uint32_t)(a * DP);
      float m = -INFINITY;
      float2 l2 = make_float2(0.f, 0.f);
      int vref = kVrefFirst;
      float big = 0.f;  // the row's largest P times scale, once they are wide
      const int cnt = count(a);
      // the drafted tokens' masks and every warp's part of the queries are there
      bool ok = mbar_wait(&sh.q_bar, 0, abort_flag, err, 61);
      const unsigned long long* const seen_at = &sh.mask[row / p.G];
      const int pos32 = (int)pos, pre32 = (int)pre, end32 = (int)end;  // a cache's positions are ints
      // S times the key's scale times f0: the scores in units of log2
      const float f0 = F16 ? sh.qs[(split ? 128 * a : 0) + quad * 32 + lane] : QP == 1 ? fabsf(p.scale2) : 1.f;
      auto ready = [&](int i) {  // S and the scales of the i-th tile
        const int t = tile(a, i);
        if (I8) ok = ok && mbar_wait(&sh.sc_full[t % NSC], (uint32_t)(t / NSC) & 1u, abort_flag, err, 51);
        ok = ok && mbar_wait(&sh.s_bar[a][i % SB], (uint32_t)(i / SB) & 1u, abort_flag, err, 52);
        ok = __all_sync(0xffffffffu, ok);
        fence_after();
        return ok;
      };
      auto turn = [&](int i, auto wide_tag) {  // S of the i-th tile into P
        constexpr bool WIDE = decltype(wide_tag)::value;
        const int t = tile(a, i), info = I8 ? sh.sc_info[t % NSC] : 0;
        const float lazy = WIDE && info & kEager ? 0.f : kLazy;
        const int t0 = (first + t) * BN;  // below `end`, which is an int's
        const float* fk = I8 ? sc_k[t % NSC] : nullptr;
        const float* fv = I8 ? sc_v[t % NSC] : nullptr;
        const uint32_t tS = tmem + tl + F::S_COL + (uint32_t)((a * SB + i % SB) * BN);
        const uint32_t tT = tmem + tl + F::T_COL + (uint32_t)((a * SB + i % SB) * BN / 2);
        auto scale_o = [&](float f) {
          if (i == 0) return;
          ok = __all_sync(0xffffffffu, mbar_wait(&sh.o_bar[a], (uint32_t)(i - 1) & 1u, abort_flag, err, 53));
          if (!ok) return;
          fence_after();
#pragma unroll
          for (int c = 0; c < DP; c += 32) {
            uint32_t r[32];
            tmem_ld32_async(tO + (uint32_t)c, r);
            tmem_wait_ld();
            reg_fence32(r);
#pragma unroll
            for (int j = 0; j < 32; ++j) r[j] = __float_as_uint(__uint_as_float(r[j]) * f);
            tmem_st16u(tO + (uint32_t)c, r);
            tmem_st16u(tO + (uint32_t)c + 16, r + 16);
          }
          tmem_wait_st();
        };
        // the row's maximum moves: O and l are rescaled
        auto rescale = [&](float mx) {
          const float mn = fmaxf(m, mx), f = mn == -INFINITY ? 0.f : ex2(m - mn);
          scale_o(f);
          l2.x *= f;
          l2.y *= f;
          if (WIDE) big *= f;
          m = mn;
        };
        // wide scales: the row's exponent for P times scale of at most `largest`; whether any row's moved
        auto reref = [&](float largest) {
          big = fmaxf(big, largest);
          const int next = wide_vref(vref, big);
          if (!__any_sync(0xffffffffu, next != vref)) return false;
          scale_o(pow2(vref - next));
          vref = next;
          return true;
        };
        if (I8 && !WIDE && info >> 3 > vref) {
          scale_o(ex2((float)(vref - (info >> 3))));
          if (!ok) return;
          vref = info >> 3;
        }
        auto moves = [&](float mx) { return __any_sync(0xffffffffu, mx > m + lazy); };
        // P of the tile from S; `vis`: the columns the row sees.  The masked way also
        // takes any scale: a row's factor f0 up to 1 goes before the key's, a larger
        // one after it, so that neither product passes f32's range unless the score does;
        // and wide scales.
        auto softmax = [&](auto mask_tag, const uint32_t* vis) {
          constexpr bool MASK = WIDE || decltype(mask_tag)::value;
          const float pre = MASK && I8 ? fminf(f0, 1.f) : 1.f, f1 = MASK && I8 ? fmaxf(f0, 1.f) : f0;
          if constexpr (QP == 1) {
            // One pass with the maximum as it stands: P is kept in registers
            // until the tile's own maximum is known.  If that moved too far
            // (always in the first tile) the pass runs again.
            for (;;) {
              const float base = m == -INFINITY ? 0.f : m;
              const float2 nb = make_float2(-base, -base);
              float mx = -INFINITY, largest = 0.f;
              const float down = WIDE ? vref_down(vref) : 1.f;
              float2 s2 = make_float2(0.f, 0.f);
              uint32_t w[BN / 2], w2[PP == 2 ? BN / 2 : 1];  // P, and what its rounding left
              uint32_t r[2][32];
              tmem_ld32_async(tS, r[0]);
#pragma unroll
              for (int c = 0; c < BN; c += 32) {
                uint32_t* x = r[(c / 32) & 1];
                tmem_wait_ld();
                reg_fence32(x);
                if (c + 32 < BN) tmem_ld32_async(tS + (uint32_t)(c + 32), r[(c / 32 + 1) & 1]);
#pragma unroll
                for (int j = 0; j < 32; j += 4) {
                  float4 f = make_float4(1.f, 1.f, 1.f, 1.f), e = f;
                  if (I8) f = *(const float4*)(fk + c + j), e = *(const float4*)(fv + c + j);
                  const float2 g[2] = {make_float2(f.x, f.y), make_float2(f.z, f.w)};
                  const float2 h2[2] = {make_float2(e.x, e.y), make_float2(e.z, e.w)};
#pragma unroll
                  for (int k = 0; k < 2; ++k) {
                    float2 s = make_float2(__uint_as_float(x[j + 2 * k]), __uint_as_float(x[j + 2 * k + 1]));
                    const bool v0 = !MASK || (vis[c / 32] >> (j + 2 * k) & 1u);
                    const bool v1 = !MASK || (vis[c / 32] >> (j + 2 * k + 1) & 1u);
                    if (I8 && MASK) s = mul2(s, make_float2(pre, pre));
                    if (I8) s = mul2(s, g[k]);
                    if (MASK) s.x = v0 ? s.x : -INFINITY, s.y = v1 ? s.y : -INFINITY;
                    mx = fmaxf(mx, fmaxf(s.x, s.y));
                    s = fma2(s, make_float2(f1, f1), nb);
                    float2 y = make_float2(ex2(s.x), ex2(s.y));
                    if (MASK) y.x = v0 ? y.x : 0.f, y.y = v1 ? y.y : 0.f;  // f1 may be 0
                    s2 = add2(s2, y);
                    if (I8) {
                      y = mul2(y, h2[k]);
                      if (MASK) y.x = v0 ? y.x : 0.f, y.y = v1 ? y.y : 0.f;
                      if (WIDE) {
                        largest = fmaxf(largest, fmaxf(fabsf(y.x), fabsf(y.y)));
                        y = mul2(y, make_float2(down, down));
                      }
                    }
                    w[(c + j) / 2 + k] = take2<F16>(y.x, y.y);
                    if (PP == 2) w2[(c + j) / 2 + k] = pack2<F16>(y.x, y.y);
                  }
                }
              }
              if (mx != -INFINITY) mx *= f1;
              if (moves(mx)) {
                rescale(mx);
                if (!ok) return;
                continue;
              }
              if (WIDE && reref(largest)) {
                if (!ok) return;
                continue;
              }
              l2 = add2(l2, s2);
#pragma unroll
              for (int c = 0; c < BN / 32; ++c) {
                tmem_st16u(tS + (uint32_t)(32 * c), w + 16 * c);
                if (PP == 2) tmem_st16u(tS + (uint32_t)(32 * c + 16), w2 + 16 * c);
              }
              return;
            }
          } else {
            float mx = -INFINITY;
#pragma unroll
            for (int c = 0; c < BN; c += 32) {
              uint32_t r[32];
              tmem_ld32_async(tS + (uint32_t)c, r);
              tmem_wait_ld();
              reg_fence32(r);
#pragma unroll
              for (int j = 0; j < 32; j += 4) {
                float4 f = make_float4(1.f, 1.f, 1.f, 1.f);
                if (I8) f = *(const float4*)(fk + c + j);
                const float g[4] = {f.x, f.y, f.z, f.w};
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                  float s = __uint_as_float(r[j + k]);
                  if (I8) s = s * pre * g[k];
                  if (MASK && !(vis[c / 32] >> (j + k) & 1u)) s = -INFINITY;
                  mx = fmaxf(mx, s);
                }
              }
            }
            if (mx != -INFINITY) mx *= f1;
            if (moves(mx)) {
              rescale(mx);
              if (!ok) return;
            }
            const float base = m == -INFINITY ? 0.f : m;
            if (WIDE) {
              float largest = 0.f;
#pragma unroll 1
              for (int c = 0; c < BN; c += 32) {
                uint32_t r[32];
                tmem_ld32_async(tS + (uint32_t)c, r);
                tmem_wait_ld();
                reg_fence32(r);
#pragma unroll
                for (int j = 0; j < 32; ++j)
                  if (vis[c / 32] >> j & 1u)
                    largest = fmaxf(largest, ex2(fmaf(__uint_as_float(r[j]) * pre * fk[c + j], f1, -base)) * fabsf(fv[c + j]));
              }
              do {
                reref(largest);
                if (!ok) return;
              } while (__any_sync(0xffffffffu, wide_vref(vref, big) != vref));
            }
            const float down = WIDE ? vref_down(vref) : 1.f;
#pragma unroll
            for (int c = 0; c < BN; c += 32) {
              uint32_t r[32];
              tmem_ld32_async(tS + (uint32_t)c, r);
              tmem_wait_ld();
              reg_fence32(r);
#pragma unroll
              for (int half = 0; half < 32; half += 16) {
                float x[16];
#pragma unroll
                for (int j = 0; j < 16; j += 4) {
                  float4 f = make_float4(1.f, 1.f, 1.f, 1.f), e = f;
                  if (I8) f = *(const float4*)(fk + c + half + j), e = *(const float4*)(fv + c + half + j);
                  const float g[4] = {f.x, f.y, f.z, f.w}, h4[4] = {e.x, e.y, e.z, e.w};
                  float y[4];
#pragma unroll
                  for (int k = 0; k < 4; ++k) {
                    const bool see = !MASK || (vis[c / 32] >> (half + j + k) & 1u);
                    const float s = __uint_as_float(r[half + j + k]);
                    y[k] = ex2(I8 ? fmaf(s * pre * g[k], f1, -base) : s - base);
                    if (MASK) y[k] = see ? y[k] : 0.f;
                    x[j + k] = y[k];
                    if (I8 && see) x[j + k] = WIDE ? x[j + k] * h4[k] * down : x[j + k] * h4[k];
                  }
                  l2 = add2(l2, add2(make_float2(y[0], y[1]), make_float2(y[2], y[3])));
                }
#pragma unroll
                for (int part = 0; part < QP; ++part) {
                  uint32_t w[8];
#pragma unroll
                  for (int j = 0; j < 8; ++j) w[j] = take2<F16>(x[2 * j], x[2 * j + 1]);
                  tmem_st8u((part < 2 ? tS + (uint32_t)(c + 16 * part) : tT + (uint32_t)(c / 2)) + half / 2, w);
                }
              }
            }
          }
        };
        if (WIDE || pre32 - t0 < BN || (I8 && info & kBigKey)) {
          uint32_t vis[BN / 32];
          const int before = pre32 - t0, fit = end32 - t0;  // columns in front of the drafted tokens, and in all
          const unsigned long long seen = pos < p.T ? *seen_at : 0ull;
#pragma unroll
          for (int vw = 0; vw < BN / 32; ++vw) {
            const int c0 = vw * 32, j0 = c0 - (pos32 - t0);  // drafted token at the word's first column
            const uint32_t b = before >= c0 + 32 ? ~0u : before <= c0 ? 0u : (1u << (before - c0)) - 1u;
            const uint32_t d = j0 >= 64 || j0 <= -32 ? 0u : (uint32_t)(j0 >= 0 ? seen >> j0 : seen << -j0);
            vis[vw] = (b | d) & (fit >= c0 + 32 ? ~0u : fit <= c0 ? 0u : (1u << (fit - c0)) - 1u);
          }
          softmax(std::true_type{}, vis);
        } else {
          softmax(std::false_type{}, nullptr);
        }
        if (!ok) return;
        tmem_wait_st();
        fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&sh.p_bar[a][i % SB]);
      };
      int i = 0;
      for (; i < cnt && ready(i); ++i) {
        if (I8 && sh.sc_info[tile(a, i) % NSC] & kWide) break;
        turn(i, std::false_type{});
        if (!ok) break;
      }
      if constexpr (I8) {
        big = m == -INFINITY ? 0.f : pow2(vref);
        for (; i < cnt && ok && ready(i); ++i) turn(i, std::true_type{});
      }
      const float l = l2.x + l2.y;
      const int at = (split ? 128 * a : a * 128) + local;
      if (local < mine) sh.m[at] = m, sh.l[at] = l, sh.up[at] = I8 ? vref_up(vref) : 1.f;
    }
  } else if (warp < kSoftWarps + kLoadWarps) {
    // ------------------------------------------------------------ loading
    stage_q(warp);
    const int lt = tid - kSoftWarps * 32;
    auto slot_free = [&](uint64_t* bars, int t, int code) {
      return t < NS || mbar_wait(&bars[t % NS], (uint32_t)(t / NS - 1) & 1u, abort_flag, err, code);
    };
    if constexpr (I8) {
      constexpr int THREADS = kLoadThreads / F::GROUPS;
      constexpr int UNITS = DP / 16;                  // 16-code pieces of a row
      constexpr int PER = BN * UNITS / THREADS;  // per thread and tile
      constexpr int RSTEP = THREADS / UNITS;     // rows between a thread's pieces (a multiple of 8)
      static_assert(RSTEP % 8 == 0, "a thread's pieces share a swizzle phase");
      // Eight lanes that store together take four pieces of two rows, whose
      // swizzles put them into different banks.
      const int group = lt / THREADS, gt = lt % THREADS;
      const int u = UNITS == 8 ? (lane & 3) | (lane >> 1 & 4) : gt % UNITS;
      const int row0 = UNITS == 8 ? (gt >> 5) * 4 + (lane >> 2 & 1) + (lane >> 3 & 2) : gt / UNITS;
      const bool has = u * 16 < p.D;
      const int64_t at0 = (nh * p.T + (int64_t)first * BN + row0) * p.D + u * 16;
      const uint32_t put0 = unit_at(BN, row0, 2 * u), put1 = unit_at(BN, row0, 2 * u + 1);
      uint4 rk[PER], rv[PER];
      // Loads of the group's next tile.  They go out right behind the fence that
      // publishes a tile: a fence waits for the thread's outstanding loads.
      auto fetch = [&](const void* base, int t, uint4* r) {
        const int8_t* src = (const int8_t*)base + at0 + (int64_t)t * BN * p.D;
        const int left = t < nt ? (int)min((int64_t)BN, end - (int64_t)(first + t) * BN) : 0;  // rows of the tile
#pragma unroll
        for (int j = 0; j < PER; ++j) {
          r[j] = make_uint4(0, 0, 0, 0);
          if (has && row0 + j * RSTEP < left) r[j] = *(const uint4*)(src + (int64_t)(j * RSTEP) * p.D);
        }
      };
      auto put = [&](uint8_t* dst, const uint4* r) {
#pragma unroll
        for (int j = 0; j < PER; ++j) {
          uint4 o[2];
          codes_to_f16(r[j], o);
          *(uint4*)(dst + put0 + j * RSTEP * 128) = o[0];
          *(uint4*)(dst + put1 + j * RSTEP * 128) = o[1];
        }
      };
      fetch(p.k, group, rk);
      fetch(p.v, group, rv);
      for (int t = group; t < nt; t += F::GROUPS) {
        if (!__all_sync(0xffffffffu, slot_free(sh.k_free, t, 54))) break;
        put(smem + F::K_OFF + (t % NS) * F::TILE, rk);
        if (!__all_sync(0xffffffffu, slot_free(sh.v_free, t, 55))) break;
        put(smem + F::V_OFF + (t % NS) * F::TILE, rv);
        fence_proxy_async();
        fetch(p.k, t + F::GROUPS, rk);
        fetch(p.v, t + F::GROUPS, rv);
        __syncwarp();
        if (lane == 0) {
          mbar_arrive(&sh.k_full[t % NS]);
          mbar_arrive(&sh.v_full[t % NS]);
        }
      }
    } else {
      // Tiles with drafted tokens or the end of the sequence are mended before
      // the MMAs may read them.  Every loading thread passes every such tile's
      // barrier, whatever was aborted (an aborted wait returns at once), so none
      // is left waiting.
      int mended = 0;
      for (int t = (int)max((int64_t)0, pre / BN - first); t < nt; ++t) {
        const int64_t t0 = (int64_t)(first + t) * BN;
        if (t0 + BN <= pre) continue;
        uint8_t* dv = smem + F::V_OFF + t % NS * F::TILE;
        mbar_wait(&sh.raw, (uint32_t)mended & 1u, abort_flag, err, 56);
        ++mended;
        for (int i = lt; i < BN * (DP / 8); i += kLoadThreads) {
          const int row = i / (DP / 8);
          uint4* x = (uint4*)(dv + unit_at(BN, row, i % (DP / 8)));
          if (t0 + row >= end) {
            *x = make_uint4(0, 0, 0, 0);
          } else if (t0 + row >= pre) {
            uint32_t w[4] = {x->x, x->y, x->z, x->w};
            bool bad = false;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              if ((w[j] & 0x7f80u) == 0x7f80u) w[j] &= 0xffff0000u, bad = true;
              if ((w[j] & 0x7f800000u) == 0x7f800000u) w[j] &= 0xffffu, bad = true;
            }
            if (bad) {
              *x = make_uint4(w[0], w[1], w[2], w[3]);
              sh.bad = 1;
            }
          }
        }
        fence_proxy_async();
        loaders_sync();
        if (lt == 0) {
          mbar_arrive(&sh.mended);
          mbar_arrive(&sh.v_full[t % NS]);
        }
      }
    }
  } else if (warp == kFeedWarp) {
    // ------------------------------------------------------------ copies and scales
    auto slot_free = [&](uint64_t* bars, int t, int code) {
      return t < NS || mbar_wait(&bars[t % NS], (uint32_t)(t / NS - 1) & 1u, abort_flag, err, code);
    };
    if constexpr (I8) {
      // Scales of keys lane and lane + 32, one tile ahead.
      // Value scales are stored relative to 2^range.hi, above the largest so far, until they are wide.
      float ck[2], cv[2];
      ScaleRange range;
      auto fetch_scales = [&](int t) {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const int64_t at = (int64_t)(first + t) * BN + i * 32 + lane;
          ck[i] = cv[i] = 0.f;
          if (t < nt && at < end) ck[i] = p.ks[nh * p.T + at], cv[i] = p.vs[nh * p.T + at];
        }
      };
      fetch_scales(0);
      for (int t = 0; t < nt; ++t) {
        // The slot of these scales was last used by tile t - NSC, whose softmax is
        // over once PV of tile t - NS has left its place.
        if (!__all_sync(0xffffffffu, slot_free(sh.v_free, t, 68))) break;
        range.lane_adds(cv[0]);
        range.lane_adds(cv[1]);
        range.join_lanes();
        const float down = range.wide ? 1.f : vref_down(range.hi);
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          sc_k[t % NSC][i * 32 + lane] = ck[i];
          sc_v[t % NSC][i * 32 + lane] = cv[i] * down;
        }
        const bool big = __any_sync(0xffffffffu, !(ck[0] < kBigScale && ck[1] < kBigScale));
        if (lane == 0)
          sh.sc_info[t % NSC] = range.hi * 8 + (big ? kBigKey : 0) + (range.wide ? kWide : 0) + (range.big() ? kEager : 0);
        __syncwarp();
        if (lane == 0) mbar_arrive(&sh.sc_full[t % NSC]);
        fetch_scales(t + 1);
      }
    } else if (lane == 0 && aligned) {
      int mend_sent = 0, sent_k = 0, sent_v = 0;
      bool ok = true;
      for (int t = 0; t < nt && ok; ++t) {
        const int64_t t0 = (int64_t)(first + t) * BN;
        const int s = t % NS;
        uint8_t *dk = smem + F::K_OFF + s * F::TILE, *dv = smem + F::V_OFF + s * F::TILE;
        const bool mend = t0 + BN > pre;  // drafted tokens or the end of the sequence
        // the queries' loads are not to queue behind more tiles than the streams start with
        if (t == 2) ok = mbar_wait(&sh.q_bar, 0, abort_flag, err, 70);
        ok = ok && slot_free(sh.k_free, t, 54);
        if (!ok) break;
        mbar_expect_tx(&sh.k_full[s], F::TILE);
#pragma unroll
        for (int c = 0; c < DP / 64; ++c)
          tma_load_3d(dk + c * BN * 128, &mK, &sh.k_full[s], c * 64, (int)t0, (int)nh);
        sent_k = t + 1;
        ok = slot_free(sh.v_free, t, 55);
        // one tile at a time is on its way to the mending warps
        if (ok && mend && mend_sent > 0) ok = mbar_wait(&sh.mended, (uint32_t)(mend_sent - 1) & 1u, abort_flag, err, 69);
        if (!ok) break;
        uint64_t* bar = mend ? &sh.raw : &sh.v_full[s];
        mbar_expect_tx(bar, F::TILE);
#pragma unroll
        for (int c = 0; c < DP / 64; ++c) tma_load_3d(dv + c * BN * 128, &mV, bar, c * 64, (int)t0, (int)nh);
        if (mend) ++mend_sent;
        else sent_v = t + 1;
      }
      // After an abort: no copy of this CTA may still be in flight when it
      // leaves.  The MMA warps may not have waited for the last ones.
      if (*abort_flag) {
        const unsigned long long t1 = now_ns() + kTimeoutNs;
        for (int s = max(0, sent_k - NS); s < sent_k; ++s)
          while (!mbar_try_wait(&sh.k_full[s % NS], (uint32_t)(s / NS) & 1u) && now_ns() < t1) {}
        for (int s = max(0, sent_v - NS); s < sent_v; ++s)
          while (!mbar_try_wait(&sh.v_full[s % NS], (uint32_t)(s / NS) & 1u) && now_ns() < t1) {}
        while (mend_sent && !mbar_try_wait(&sh.raw, (uint32_t)(mend_sent - 1) & 1u) && now_ns() < t1) {}
      }
    }
  } else {
    const int a = warp - kMmaWarp;
    if (a > 1) {
      tree_masks(p.parents ? p.parents + n * p.S : nullptr, p.S, lane, sh.mask, sh.jump);
      __syncwarp();
      if (lane == 0) mbar_arrive(&sh.q_bar);
    } else {
      // ---------------------------------------------------------- MMA issue of stream a
      const uint32_t id_s = idesc_16(F16, 128, BN, 0, 0), id_o = idesc_16(F16, 128, DP, 0, 1);
      const uint32_t sq = smem_u32(smem) + (split ? (uint32_t)(a * QP * F::QTILE) : 0u);
      const uint32_t sk = smem_u32(smem) + F::K_OFF, sv = smem_u32(smem) + F::V_OFF;
      const uint32_t to = tmem + F::O_COL + (uint32_t)(a * DP);
      const int cnt = count(a);
      bool ok = __all_sync(0xffffffffu, mbar_wait(&sh.q_bar, 0, abort_flag, err, 62));
      auto issue_s = [&](int i) {
        const int t = tile(a, i);
        if (!__all_sync(0xffffffffu, mbar_wait(&sh.k_full[t % NS], (uint32_t)(t / NS) & 1u, abort_flag, err, 57)))
          return false;
        fence_after();
        const uint32_t ts = tmem + F::S_COL + (uint32_t)((a * SB + i % SB) * BN);
        const uint64_t qd = smem_desc(sq, 16, 1024, 2);
        const uint64_t kd = smem_desc(sk + (uint32_t)((t % NS) * F::TILE), 16, 1024, 2);
#pragma unroll
        for (int part = QP - 1; part >= 0; --part)  // the accumulator truncates: small products first
#pragma unroll
          for (int kk = 0; kk < DP / 16; ++kk)
            mma_ss(ts, qd + ((part * F::QTILE + (kk / 4) * 128 * 128 + (kk % 4) * 32) >> 4),
                   kd + (((kk / 4) * BN * 128 + (kk % 4) * 32) >> 4), id_s, part < QP - 1 || kk > 0 ? 1u : 0u);
        commit(&sh.s_bar[a][i % SB]);
        commit(&sh.k_free[t % NS]);
        return true;
      };
      for (int i = 0; i < SB && i < cnt && ok; ++i) ok = issue_s(i);
      // O of tile i, then S of tile i + SB: tcgen05 MMAs of one thread run in issue
      // order, so that S overwrites P of tile i after O has read it
      for (int i = 0; i < cnt && ok; ++i) {
        const int t = tile(a, i);
        ok = __all_sync(0xffffffffu, mbar_wait(&sh.p_bar[a][i % SB], (uint32_t)(i / SB) & 1u, abort_flag, err, 58) &&
                                         mbar_wait(&sh.v_full[t % NS], (uint32_t)(t / NS) & 1u, abort_flag, err, 59));
        if (!ok) break;
        fence_after();
        const uint32_t ts = tmem + F::S_COL + (uint32_t)((a * SB + i % SB) * BN);
        const uint32_t tt = tmem + F::T_COL + (uint32_t)((a * SB + i % SB) * BN / 2);
        const uint64_t bd = smem_desc(sv + (uint32_t)((t % NS) * F::TILE), BN * 128, 1024, 2);
#pragma unroll
        for (int kk = 0; kk < BN / 16; ++kk) {
          const uint32_t pc = ts + (uint32_t)((kk / 2) * 32 + (kk % 2) * 8);
          mma_ts(to, pc, bd + kk * (2048 >> 4), id_o, i > 0 || kk > 0 ? 1u : 0u);
          if (PP > 1) mma_ts(to, pc + 16, bd + kk * (2048 >> 4), id_o, 1u);
          if (PP > 2) mma_ts(to, tt + (uint32_t)(kk * 8), bd + kk * (2048 >> 4), id_o, 1u);
        }
        commit(&sh.o_bar[a]);
        commit(&sh.v_free[t % NS]);
        if (i + SB < cnt) ok = issue_s(i + SB);
      }
      // the accumulator is final, and no MMA of the stream reads shared memory, once this passes
      if (ok && cnt > 0) mbar_wait(&sh.o_bar[a], (uint32_t)(cnt - 1) & 1u, abort_flag, err, 60);
    }
  }
  __syncwarp();
  fence_before();
  __syncthreads();
  fence_after();
  const bool failed = sh.abort_flag != 0;

  // outputs of the two streams to shared memory: row a * 128 + local
  float* so = (float*)smem;
  if (warp < kSoftWarps && !failed) {
    const int a = warp >> 2, quad = warp & 3;
    const int mine = split ? min(128, rows - 128 * a) : rows, q0 = quad * 32 - (split ? 0 : a * up);
    if (q0 >= 0 && q0 < mine) {
      const int local = q0 + lane;
      const uint32_t tO = tmem + ((uint32_t)(quad * 32) << 16) + F::O_COL + (uint32_t)(a * DP);
#pragma unroll
      for (int c = 0; c < DP; c += 32) {
        uint32_t r[32];
        tmem_ld32_async(tO + (uint32_t)c, r);
        tmem_wait_ld();
        reg_fence32(r);
        if (local < mine)
#pragma unroll
          for (int j = 0; j < 32; j += 4)
            *(uint4*)(so + (a * 128 + local) * F::LDO + c + j) =
                count(a) == 0 ? make_uint4(0, 0, 0, 0)
                : I8          ? make_uint4(r[j], r[j + 2], r[j + 1], r[j + 3])  // the order of the codes
                              : make_uint4(r[j], r[j + 1], r[j + 2], r[j + 3]);
      }
    }
  }
  fence_before();
  __syncthreads();
  if (warp == 0) {
    fence_after();
    tmem_dealloc(sh.tslot, F::COLS);
  }
  __syncthreads();
  cluster_sync();
  if (!failed) {
    // Rank c joins rows c, c + C, ..  First a thread per row turns the parts'
    // maxima and sums into weights (part j: CTA j when split, else CTA j / 2,
    // stream j % 2), then the outputs are summed with every load of a thread's
    // values under way at once.
    const int np = split ? (int)C : 2 * (int)C, mine = rows > (int)rank ? (rows - (int)rank + (int)C - 1) / (int)C : 0;
    float* wgt = sh.wgt;
    for (int k = tid; k < mine; k += kThreads) {
      const int i = k * (int)C + (int)rank;
      float pm[16], pl[16], pu[16], mx = -INFINITY, l = 0.f;
#pragma unroll
      for (int j = 0; j < 16; ++j) {
        pm[j] = -INFINITY, pl[j] = 0.f, pu[j] = 1.f;
        if (j < np) {
          const uint32_t c = (uint32_t)(split ? j : j / 2);
          const int at = split ? i : (j & 1) * 128 + i;
          asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(pm[j]) : "r"(cluster_addr(&sh.m[at], c)));
          asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(pl[j]) : "r"(cluster_addr(&sh.l[at], c)));
          if (I8) asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(pu[j]) : "r"(cluster_addr(&sh.up[at], c)));
        }
      }
#pragma unroll
      for (int j = 0; j < 16; ++j) mx = fmaxf(mx, pm[j]);
      const float base = mx == -INFINITY ? 0.f : mx;
#pragma unroll
      for (int j = 0; j < 16; ++j) {
        pm[j] = ex2(pm[j] - base);
        l = fmaf(pl[j], pm[j], l);
      }
      // A part without keys has no meaning for its row.  No part has one where the scores are -inf or NaN
      // throughout, which gives NaN as in the formula, or where there are no keys (see finish4).
      const float none = mx == -INFINITY ? NAN : 0.f;
#pragma unroll
      for (int j = 0; j < 16; ++j)
        if (j < np) wgt[k * np + j] = pm[j] == 0.f ? none : pm[j] / l * pu[j];
    }
    int bad = 0;
    if (!I8 && lane < (int)C)
      asm volatile("ld.shared::cluster.s32 %0, [%1];" : "=r"(bad) : "r"(cluster_addr(&sh.bad, (uint32_t)lane)));
    bad = __any_sync(0xffffffffu, bad);
    __syncthreads();
    constexpr int LPR = DP / 4;
    const int gl = tid % LPR;
    constexpr int ROWS = kThreads / LPR;
    for (int k0 = tid / LPR; k0 < mine; k0 += 2 * ROWS) {
      float4 acc[2] = {make_float4(0.f, 0.f, 0.f, 0.f), make_float4(0.f, 0.f, 0.f, 0.f)};
      for (int j0 = 0; j0 < np; j0 += 4) {
        float4 x[2][4];
#pragma unroll
        for (int r = 0; r < 2; ++r)
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            x[r][j] = make_float4(0.f, 0.f, 0.f, 0.f);
            const int k = k0 + r * ROWS;
            if (j0 + j < np && k < mine) {
              const int i = k * (int)C + (int)rank, part = j0 + j;
              x[r][j] = ld_remote4(so + (split ? i : (part & 1) * 128 + i) * F::LDO + gl * 4,
                                   (uint32_t)(split ? part : part / 2));
            }
          }
#pragma unroll
        for (int r = 0; r < 2; ++r)
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const int k = k0 + r * ROWS;
            if (j0 + j < np && k < mine) {
              const float f = wgt[k * np + j0 + j];
              if (f != 0.f) add_scaled(acc[r], x[r][j], f);
            }
          }
      }
#pragma unroll
      for (int r = 0; r < 2; ++r)
        if (k0 + r * ROWS < mine)
          finish4(p, w, r0 + (k0 + r * ROWS) * (int)C + (int)rank, gl * 4, acc[r], 1.f, sh.mask, bad);
    }
  }
  cluster_sync();
}

template <int DP, int QP, bool I8>
cudaError_t launch(const CacheAttnArgs& a, cudaStream_t stream) {
  using F = Cfg<DP, QP, I8>;
  const KvCacheView& c = a.cache;
  const Params p = make_params(a, F::MAXR);
  CUtensorMap mk{}, mv{};
  if (!I8) {
    const uint64_t dims[3] = {(uint64_t)c.D, (uint64_t)c.T, (uint64_t)(c.N * c.H)};
    const uint64_t strides[2] = {(uint64_t)c.D * 2, (uint64_t)(c.T * c.D) * 2};
    if (!tc_make_map_bf16(&mk, c.k, 3, dims, strides, BN) || !tc_make_map_bf16(&mv, c.v, 3, dims, strides, BN))
      return cudaErrorNotSupported;
  }
  int* err = tc_error_word();
  if (!err) return cudaErrorMemoryAllocation;
  const int64_t items = c.N * c.H * p.chunks;
  // One CTA fits an SM (shared memory, and all of its TMEM): split until the CTAs
  // fill the SMs once, or a CTA has four tiles, since a second wave would repeat the
  // 10 us that a CTA takes without keys.  (8 items of 128 rows over 8K keys of 128:
  // 28 us, unsplit 94; 32 of 256 rows over 16K: 95 and 289; 24 of 63 rows over 1K of
  // 64: 14 and 20.)
  int C = 1;
  while (C < kPortable && items * (C + 1) <= sm_count() && c.T / (C + 1) >= 4 * BN) ++C;
  // The accumulators truncate, so an output falls short by a little with every MMA added
  // to it: of f32 calls, with three parts of P, some 1.5e-7 of itself per tile of a
  // stream.  So a stream takes at most 32 of their tiles, whatever that costs in waves
  // (12 x 8 caches of 12K keys of 64, 20 rows: off by 5e-6 at 3 CTAs each, 1.4e-5 at 1),
  // up to the 8 CTAs of 32K keys.
  const int64_t streams = a.S * (a.Hq / c.H) > 128 && F::MAXR > 128 ? 1 : 2;
  while (QP == 3 && C < kPortable && (c.T + BN - 1) / BN > 32 * streams * C) ++C;
  return launch_cluster(cache_attn_tc<DP, QP, I8>, items * C, C, kThreads, F::SMEM, stream, mk, mv, p, err);
}

}  // namespace

bool cache_attention_tc_takes(const CacheAttnArgs& a) {
  return on_tensor_cores(a) && !cache_attention_mma_takes(a);
}

cudaError_t cache_attention_tc(const CacheAttnArgs& a, cudaStream_t stream) {
  const bool i8 = a.cache.type == KvType::I8;
  if (a.cache.D <= 64) {
    if (a.bf16) return i8 ? launch<64, 1, true>(a, stream) : launch<64, 1, false>(a, stream);
    return i8 ? launch<64, 3, true>(a, stream) : launch<64, 3, false>(a, stream);
  }
  if (a.bf16) return i8 ? launch<128, 1, true>(a, stream) : launch<128, 1, false>(a, stream);
  return i8 ? launch<128, 3, true>(a, stream) : launch<128, 3, false>(a, stream);
}

}  // namespace sb
