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
// roles: 8 softmax, 4 loading, 2 issuing the MMAs (one thread needs about 80
// cycles per tcgen05.mma, more than the 64 that one takes), 2 helpers.
//
//   S = Q K^T   bf16 operands.  f32 queries are split exactly into three bf16
//               parts (8 mantissa bits each) whose products accumulate into
//               the same f32 S, so S has f32 accuracy; cache values are bf16
//               or int8 codes, which bf16 holds exactly.
//   P           exp2(S - m) times the value row's int8 scale, written back over
//               S in TMEM as bf16 (bf16 output: one rounding, as large as the
//               output's own) or as three bf16 parts (f32 output: f32 accuracy;
//               two parts would leave 2^-16 of each probability).
//   O += P V    the maximum m a row refers to moves only when it would grow by
//               more than 2^8, so O is rescaled in the first tiles and then
//               hardly ever; exact since P, O and the sum l share m.
//
// bf16 tiles arrive by TMA, int8 tiles through registers (codes to bf16 on the
// way to swizzled shared memory).  Rows of V behind the last token are zeroed
// (0 x NaN would reach every row); a value of a drafted token that is not
// finite is taken out of the tile and added to the rows that attend to it when
// the outputs are joined.
//
// Every mbarrier wait is bounded.  TMEM is freed before the cluster barrier: a
// CTA that holds TMEM never waits for another CTA.
#include <type_traits>

#include "cache_attn.h"

namespace sb {
namespace {

using namespace cattn;
using namespace tc;

// warps 0-7 softmax, 8-11 loading, 12 and 13 MMA issue (one per stream), 14, 15
// and the softmax warps stage the queries
constexpr int kSoftWarps = 8, kLoadWarps = 4, kMmaWarp = 12, kWarps = 16, kThreads = kWarps * 32;
constexpr int kStageWarps = kWarps - kLoadWarps - 2;
// Registers per thread of the four warpgroups: 2 softmax, loading, the rest.
// They add up to the launch's 4 x 128.
constexpr int kRegsSoft = 168, kRegsLoad = 104, kRegsRest = 72, kRegsLaunch = 128;
static_assert(2 * kRegsSoft + kRegsLoad + kRegsRest == 4 * kRegsLaunch, "register shares");
template <int N>
__device__ __forceinline__ void regs_inc() { asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N)); }
template <int N>
__device__ __forceinline__ void regs_dec() { asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N)); }
constexpr int kLoadThreads = kLoadWarps * 32;
constexpr int NS = 2;   // K and V tiles in flight
constexpr int NSC = 4;  // rows of scales in flight (see the loader)
constexpr float kLazy = 8.f;  // a row's maximum moves when it would grow by more than this (log2)

// D (TMEM) (+)= A (TMEM, bf16 pairs: lane = row, column = two k) * B.
__device__ __forceinline__ void mma_bf16_ts(uint32_t tmem_d, uint32_t tmem_a, uint64_t bd, uint32_t idesc, uint32_t acc) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(tmem_d),
      "r"(tmem_a), "l"(bd), "r"(idesc), "r"(acc)
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

// (lo, hi) f32 to packed bf16, rounded to nearest even
__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {
  uint32_t d;
  asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(d) : "f"(hi), "f"(lo));
  return d;
}
__device__ __forceinline__ float bf_lo(uint32_t w) { return __uint_as_float(w << 16); }
__device__ __forceinline__ float bf_hi(uint32_t w) { return __uint_as_float(w & 0xffff0000u); }

// 16 codes to 16 bf16 values.  A code's low 7 bits and its sign bit, each put
// under the exponent of 128 (bf16 steps of 1 from 128 to 256), differ by the
// code: (128 + low) - (128 or 256) = code, exactly.
__device__ __forceinline__ void codes_to_bf16(const uint4& c, uint4* out) {
  const uint32_t w[4] = {c.x, c.y, c.z, c.w};
  uint32_t o[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const uint32_t t = __byte_perm(w[i / 2], 0, i & 1 ? 0x4342 : 0x4140);
    const uint32_t a = (t & 0x007f007fu) | 0x43004300u, b = (t & 0x00800080u) | 0x43004300u;
    __nv_bfloat162 x = __hsub2(*(const __nv_bfloat162*)&a, *(const __nv_bfloat162*)&b);
    o[i] = *(uint32_t*)&x;
  }
  out[0] = make_uint4(o[0], o[1], o[2], o[3]);
  out[1] = make_uint4(o[4], o[5], o[6], o[7]);
}

// 16-byte unit u (of 8 per 128-byte row and 64-value chunk) of row r in a
// 128-byte-swizzled tile of `rows` rows.
__device__ __forceinline__ uint32_t unit_at(int rows, int r, int unit) {
  return (uint32_t)((unit >> 3) * rows * 128 + r * 128 + (((unit & 7) ^ (r & 7)) << 4));
}

__device__ __forceinline__ void loaders_sync() { asm volatile("bar.sync 1, %0;" ::"n"(kLoadThreads) : "memory"); }

template <int DP, int BN, int QP>
struct Cfg {
  static constexpr int MAXR = QP == 3 && DP == 128 ? 128 : 256;  // query rows of a CTA
  static constexpr int QTILE = 128 * DP * 2;                     // one part of 128 rows
  static constexpr int Q_BYTES = (MAXR / 128) * QP * QTILE;
  static constexpr int TILE = BN * DP * 2;
  static constexpr int K_OFF = Q_BYTES, V_OFF = K_OFF + NS * TILE, END = V_OFF + NS * TILE;
  static constexpr int LDO = DP + 4;  // padded row of the joined outputs, f32
  static constexpr int JOIN = 256 * LDO * 4;
  static constexpr int SMEM = END > JOIN ? END : JOIN;
  static constexpr uint32_t COLS = 512;
  // S (P's first two parts in place), O, P's third part; two streams each
  static constexpr uint32_t S_COL = 0, O_COL = 2 * BN, T_COL = O_COL + 2 * DP;
  static_assert(2 * BN + 2 * DP + (QP == 3 ? BN : 0) <= 512, "TMEM columns");
};

struct Shared {
  uint64_t k_full[NS], k_free[NS], v_full[NS], v_free[NS], sc_full[NSC], s_bar[2], p_bar[2], o_bar[2], raw, q_bar;
  uint32_t tslot;
  volatile int abort_flag;
  int bad;  // a drafted value that is not finite was taken out of a tile
  unsigned long long mask[kKvMaxTokens];
  int jump[kKvMaxTokens];
  float m[256], l[256];
  float wgt[256 * 2];  // rows of a rank x parts: at most 256 / C x C, or 128 / C x 2 C
};

// I8: int8 cache, else bf16.  QP: parts of a query (1: bf16, 3: f32).
template <int DP, int BN, int QP, bool I8>
__global__ void __launch_bounds__(kThreads, 1)
    cache_attn_tc(const __grid_constant__ CUtensorMap mK, const __grid_constant__ CUtensorMap mV, const Params p,
                  int* err) {
  using F = Cfg<DP, BN, QP>;
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
      mbar_init(&sh.k_full[i], I8 ? kLoadWarps : 1);
      mbar_init(&sh.v_full[i], I8 ? kLoadWarps : 1);
      mbar_init(&sh.k_free[i], split ? 2 : 1);  // the streams that read the tile
      mbar_init(&sh.v_free[i], split ? 2 : 1);
    }
    for (int i = 0; i < NSC; ++i) mbar_init(&sh.sc_full[i], kLoadWarps);
    for (int a = 0; a < 2; ++a) {
      const int mine = split ? min(128, rows - 128 * a) : rows;
      mbar_init(&sh.s_bar[a], 1);
      mbar_init(&sh.p_bar[a], (uint32_t)((mine + 31) / 32));
      mbar_init(&sh.o_bar[a], 1);
    }
    mbar_init(&sh.raw, 1);
    mbar_init(&sh.q_bar, kStageWarps);
    sh.abort_flag = aligned ? 0 : 1;
    sh.bad = 0;
    if (!aligned) atomicExch(err, 50);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    fence_proxy_async();
  }
  if (warp == 0) tmem_alloc(&sh.tslot, F::COLS);
  fence_before();
  __syncthreads();
  fence_after();
  const uint32_t tmem = sh.tslot;
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
    constexpr int UNITS = DP / 8, RSTEP = kStageWarps * 32 / UNITS, LOADS = QP == 1 ? 1 : 2, BATCH = QP == 1 ? 8 : 4;
    static_assert(kStageWarps * 32 % UNITS == 0, "whole rows per step");
    const int u = (sw * 32 + lane) % UNITS, total = nt > 0 && aligned ? (split ? 256 : 128) : 0;
    const int64_t q0 = (n * p.S * p.H + h) * p.G * p.D + u * 8;
    const int64_t token = (int64_t)p.H * p.G * p.D;
#pragma unroll 1
    for (int k0 = (sw * 32 + lane) / UNITS; k0 < total; k0 += BATCH * RSTEP) {
      uint4 raw[BATCH][LOADS];
#pragma unroll
      for (int k = 0; k < BATCH; ++k) {
        const int i = k0 + k * RSTEP, local = up ? i & 63 : i;
#pragma unroll
        for (int c = 0; c < LOADS; ++c) raw[k][c] = make_uint4(0, 0, 0, 0);
        if (i < total && local < rows && u * 8 < p.D) {
          const int row = r0 + local, s = row / p.G, g = row - s * p.G;
          const int64_t at = q0 + s * token + g * p.D;
#pragma unroll
          for (int c = 0; c < LOADS; ++c)
            raw[k][c] = *(const uint4*)((const uint8_t*)p.q + (at + 4 * c) * (QP == 1 ? 2 : 4));
        }
      }
#pragma unroll
      for (int k = 0; k < BATCH; ++k) {
        const int i = k0 + k * RSTEP;
        if (i >= total) continue;
        uint8_t* dst = smem + (i >> 7) * QP * F::QTILE + unit_at(128, i & 127, u);
        if (QP == 1) {
          const uint32_t flip = p.scale2 < 0.f ? 0x80008000u : 0u;
          const uint4 x = raw[k][0];
          *(uint4*)dst = make_uint4(x.x ^ flip, x.y ^ flip, x.z ^ flip, x.w ^ flip);
        } else {
          // x = part 0 + part 1 + part 2, each a bf16 rounding of what is left
          float x[8];
          *(uint4*)x = raw[k][0];
          *(uint4*)(x + 4) = raw[k][LOADS - 1];
#pragma unroll
          for (int j = 0; j < 8; ++j) x[j] *= p.scale2;
#pragma unroll
          for (int part = 0; part < QP; ++part) {
            uint32_t y[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              y[j] = pack_bf16(x[2 * j], x[2 * j + 1]);
              x[2 * j] -= bf_lo(y[j]);
              x[2 * j + 1] -= bf_hi(y[j]);
            }
            *(uint4*)(dst + part * F::QTILE) = make_uint4(y[0], y[1], y[2], y[3]);
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
    regs_inc<kRegsSoft>();
    stage_q(warp);
    const int a = warp >> 2, quad = warp & 3;
    const int lo_lane = split ? 0 : a * up;  // the stream's first TMEM lane
    const int mine = split ? min(128, rows - 128 * a) : rows;
    const int q0 = quad * 32 - lo_lane;  // first row of this warp within the stream
    if (q0 >= 0 && q0 < mine) {
      const int local = q0 + lane;  // row within the stream
      const int row = r0 + (split ? 128 * a : 0) + min(local, mine - 1);
      const uint32_t tl = (uint32_t)(quad * 32) << 16;
      const uint32_t tS = tmem + tl + F::S_COL + (uint32_t)(a * BN), tO = tmem + tl + F::O_COL + (uint32_t)(a * DP);
      const uint32_t tT = tmem + tl + F::T_COL + (uint32_t)(a * BN / 2);
      const float f0 = fabsf(p.scale2);  // bf16 queries over a bf16 cache: scaled here
      float m = -INFINITY;
      float2 l2 = make_float2(0.f, 0.f);
      const int cnt = count(a);
      // the drafted tokens' masks and every warp's part of the queries are there
      bool ok = mbar_wait(&sh.q_bar, 0, abort_flag, err, 61);
      const unsigned long long seen = sh.mask[row / p.G];
      for (int i = 0; i < cnt; ++i) {
        const int t = tile(a, i);
        const int64_t t0 = (int64_t)(first + t) * BN;
        if (I8) ok = ok && mbar_wait(&sh.sc_full[t % NSC], (uint32_t)(t / NSC) & 1u, abort_flag, err, 51);
        ok = ok && mbar_wait(&sh.s_bar[a], (uint32_t)i & 1u, abort_flag, err, 52);
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) break;
        fence_after();
        const float* fk = I8 ? sc_k[t % NSC] : nullptr;
        const float* fv = I8 ? sc_v[t % NSC] : nullptr;
        // the row's maximum moves to mn: O and l are rescaled
        auto rescale = [&](float mx) {
          const float mn = fmaxf(m, mx), f = mn == -INFINITY ? 0.f : ex2(m - mn);
          if (i > 0) {
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
          }
          l2.x *= f;
          l2.y *= f;
          m = mn;
        };
        auto moves = [&](float mx) { return __any_sync(0xffffffffu, mx > m + kLazy); };
        // P of the tile from S; `vis`: the columns the row sees
        auto softmax = [&](auto mask_tag, const uint32_t* vis) {
          constexpr bool MASK = decltype(mask_tag)::value;
          if constexpr (QP == 1) {
            // One pass with the maximum as it stands: P is kept in registers
            // until the tile's own maximum is known.  If that moved too far
            // (always in the first tile) the pass runs again.
            for (;;) {
              const float base = m == -INFINITY ? 0.f : m;
              const float2 nb = make_float2(-base, -base);
              float mx = -INFINITY;
              float2 s2 = make_float2(0.f, 0.f);
              uint32_t w[BN / 2];
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
                  float4 f = make_float4(f0, f0, f0, f0), e = f;
                  if (I8) f = *(const float4*)(fk + c + j), e = *(const float4*)(fv + c + j);
                  const float2 g[2] = {make_float2(f.x, f.y), make_float2(f.z, f.w)};
                  const float2 h2[2] = {make_float2(e.x, e.y), make_float2(e.z, e.w)};
#pragma unroll
                  for (int k = 0; k < 2; ++k) {
                    float2 s = make_float2(__uint_as_float(x[j + 2 * k]), __uint_as_float(x[j + 2 * k + 1]));
                    const bool v0 = !MASK || (vis[c / 32] >> (j + 2 * k) & 1u);
                    const bool v1 = !MASK || (vis[c / 32] >> (j + 2 * k + 1) & 1u);
                    if (I8) s = mul2(s, g[k]);
                    if (MASK) s.x = v0 ? s.x : -INFINITY, s.y = v1 ? s.y : -INFINITY;
                    mx = fmaxf(mx, fmaxf(s.x, s.y));
                    s = I8 ? add2(s, nb) : fma2(s, g[k], nb);
                    float2 y = make_float2(ex2(s.x), ex2(s.y));
                    if (MASK && !I8) y.x = v0 ? y.x : 0.f, y.y = v1 ? y.y : 0.f;  // f0 may be 0
                    s2 = add2(s2, y);
                    if (I8) {
                      y = mul2(y, h2[k]);
                      if (MASK) y.x = v0 ? y.x : 0.f, y.y = v1 ? y.y : 0.f;
                    }
                    w[(c + j) / 2 + k] = pack_bf16(y.x, y.y);
                  }
                }
              }
              if (!I8 && mx != -INFINITY) mx *= f0;
              if (moves(mx)) {
                rescale(mx);
                if (!ok) return;
                continue;
              }
              l2 = add2(l2, s2);
#pragma unroll
              for (int c = 0; c < BN / 32; ++c) tmem_st16u(tS + (uint32_t)(32 * c), w + 16 * c);
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
                  if (I8) s *= g[k];
                  if (MASK && !(vis[c / 32] >> (j + k) & 1u)) s = -INFINITY;
                  mx = fmaxf(mx, s);
                }
              }
            }
            if (moves(mx)) {
              rescale(mx);
              if (!ok) return;
            }
            const float base = m == -INFINITY ? 0.f : m;
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
                    y[k] = ex2(I8 ? fmaf(s, g[k], -base) : s - base);
                    if (MASK) y[k] = see ? y[k] : 0.f;
                    x[j + k] = y[k];
                    if (I8 && see) x[j + k] *= h4[k];
                  }
                  l2 = add2(l2, add2(make_float2(y[0], y[1]), make_float2(y[2], y[3])));
                }
#pragma unroll
                for (int part = 0; part < QP; ++part) {
                  uint32_t w[8];
#pragma unroll
                  for (int j = 0; j < 8; ++j) {
                    w[j] = pack_bf16(x[2 * j], x[2 * j + 1]);
                    if (part + 1 < QP) x[2 * j] -= bf_lo(w[j]), x[2 * j + 1] -= bf_hi(w[j]);
                  }
                  tmem_st8u((part < 2 ? tS + (uint32_t)(c + 16 * part) : tT + (uint32_t)(c / 2)) + half / 2, w);
                }
              }
            }
          }
        };
        if (t0 + BN > pre) {
          uint32_t vis[BN / 32];
          const int64_t off = pos - t0;  // column of drafted token 0
#pragma unroll
          for (int vw = 0; vw < BN / 32; ++vw) {
            const int64_t c0 = vw * 32;
            const uint32_t before = pre - t0 >= c0 + 32 ? ~0u : pre - t0 <= c0 ? 0u : (1u << (pre - t0 - c0)) - 1u;
            const int64_t j0 = c0 - off;  // drafted token at the word's first column
            uint32_t d = 0;
            if (j0 >= 0) d = j0 < 64 ? (uint32_t)(seen >> j0) : 0u;
            else if (j0 > -32) d = (uint32_t)(seen << -j0);
            const uint32_t fit = end - t0 >= c0 + 32 ? ~0u : end - t0 <= c0 ? 0u : (1u << (end - t0 - c0)) - 1u;
            vis[vw] = (before | (pos < p.T ? d : 0u)) & fit;
          }
          softmax(std::true_type{}, vis);
        } else {
          softmax(std::false_type{}, nullptr);
        }
        if (!ok) break;
        tmem_wait_st();
        fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&sh.p_bar[a]);
      }
      const float l = l2.x + l2.y;
      const int at = (split ? 128 * a : a * 128) + local;
      if (local < mine) sh.m[at] = m, sh.l[at] = l;
    }
    __syncwarp();
    regs_dec<kRegsLaunch>();
  } else if (warp < kSoftWarps + kLoadWarps) {
    // ------------------------------------------------------------ loading
    regs_dec<kRegsLoad>();
    const int lt = tid - kSoftWarps * 32;
    auto slot_free = [&](uint64_t* bars, int t, int code) {
      return t < NS || mbar_wait(&bars[t % NS], (uint32_t)(t / NS - 1) & 1u, abort_flag, err, code);
    };
    if constexpr (I8) {
      constexpr int UNITS = DP / 16;                  // 16-code pieces of a row
      constexpr int PER = BN * UNITS / kLoadThreads;  // per thread and tile
      constexpr int RSTEP = kLoadThreads / UNITS;     // rows between a thread's pieces (a multiple of 8)
      static_assert(RSTEP % 8 == 0, "a thread's pieces share a swizzle phase");
      const int u = lt % UNITS, row0 = lt / UNITS;
      const bool has = u * 16 < p.D;
      const int64_t at0 = (nh * p.T + (int64_t)first * BN + row0) * p.D + u * 16;
      const uint32_t put0 = unit_at(BN, row0, 2 * u), put1 = unit_at(BN, row0, 2 * u + 1);
      uint4 rk[PER], rv[PER];
      float nk = 0.f, nv = 0.f;
      auto fetch = [&](const void* base, int t, uint4* r) {
        const int8_t* src = (const int8_t*)base + at0 + (int64_t)t * BN * p.D;
        const int left = t < nt ? (int)min((int64_t)BN, end - (int64_t)(first + t) * BN) : 0;  // rows of the tile
#pragma unroll
        for (int j = 0; j < PER; ++j) {
          r[j] = make_uint4(0, 0, 0, 0);
          if (has && row0 + j * RSTEP < left) r[j] = *(const uint4*)(src + (int64_t)(j * RSTEP) * p.D);
        }
      };
      auto fetch_scales = [&](int t) {
        const int64_t at = (int64_t)(first + t) * BN + lt;
        nk = nv = 0.f;
        if (lt < BN && t < nt && at < end) nk = p.ks[nh * p.T + at], nv = p.vs[nh * p.T + at];
      };
      auto put = [&](uint8_t* dst, const uint4* r) {
#pragma unroll
        for (int j = 0; j < PER; ++j) {
          uint4 o[2];
          codes_to_bf16(r[j], o);
          *(uint4*)(dst + put0 + j * RSTEP * 128) = o[0];
          *(uint4*)(dst + put1 + j * RSTEP * 128) = o[1];
        }
      };
      fetch(p.k, 0, rk);
      fetch(p.v, 0, rv);
      fetch_scales(0);
      for (int t = 0; t < nt; ++t) {
        if (!__all_sync(0xffffffffu, slot_free(sh.k_free, t, 54))) break;
        put(smem + F::K_OFF + (t % NS) * F::TILE, rk);
        // The slot of these scales was last used by tile t - NSC.  Its softmax
        // is over: V of tile t - 1 went into a slot that PV of tile t - 1 - NS
        // had left, and V of tile t - 2 into that of tile t - 2 - NS = t - NSC.
        if (lt < BN) {
          sc_k[t % NSC][lt] = QP == 1 ? nk * fabsf(p.scale2) : nk;
          sc_v[t % NSC][lt] = nv;
        }
        fetch(p.k, t + 1, rk);
        fetch_scales(t + 1);
        fence_proxy_async();
        __syncwarp();
        if (lane == 0) {
          mbar_arrive(&sh.k_full[t % NS]);
          mbar_arrive(&sh.sc_full[t % NSC]);
        }
        if (!__all_sync(0xffffffffu, slot_free(sh.v_free, t, 55))) break;
        put(smem + F::V_OFF + (t % NS) * F::TILE, rv);
        fetch(p.v, t + 1, rv);
        fence_proxy_async();
        __syncwarp();
        if (lane == 0) mbar_arrive(&sh.v_full[t % NS]);
      }
    } else {
      // Every loading thread passes every mended tile's barrier, whatever was
      // aborted (an aborted wait returns at once), so none is left waiting.
      int mended = 0, sent_k = 0, sent_v = 0, sent_raw = 0;
      for (int t = 0; t < nt; ++t) {
        const int64_t t0 = (int64_t)(first + t) * BN;
        const int s = t % NS;
        uint8_t *dk = smem + F::K_OFF + s * F::TILE, *dv = smem + F::V_OFF + s * F::TILE;
        const bool mend = t0 + BN > pre;  // drafted tokens or the end of the sequence
        bool ok = true;
        if (lt == 0) {
          ok = slot_free(sh.k_free, t, 54);
          if (ok) {
            mbar_expect_tx(&sh.k_full[s], F::TILE);
#pragma unroll
            for (int c = 0; c < DP / 64; ++c)
              tma_load_3d(dk + c * BN * 128, &mK, &sh.k_full[s], c * 64, (int)t0, (int)nh);
            sent_k = t + 1;
            ok = slot_free(sh.v_free, t, 55);
          }
          if (ok) {
            uint64_t* bar = mend ? &sh.raw : &sh.v_full[s];
            mbar_expect_tx(bar, F::TILE);
#pragma unroll
            for (int c = 0; c < DP / 64; ++c) tma_load_3d(dv + c * BN * 128, &mV, bar, c * 64, (int)t0, (int)nh);
            if (mend) ++sent_raw;
            else sent_v = t + 1;
          }
        }
        if (mend) {
          ok = mbar_wait(&sh.raw, (uint32_t)mended & 1u, abort_flag, err, 56) && ok;
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
          if (lt == 0) mbar_arrive(&sh.v_full[s]);
        }
      }
      // After an abort: no copy of this CTA may still be in flight when it
      // leaves.  The MMA warp may not have waited for the last ones.
      if (lt == 0 && *abort_flag) {
        const unsigned long long t1 = now_ns() + kTimeoutNs;
        for (int s = max(0, sent_k - NS); s < sent_k; ++s)
          while (!mbar_try_wait(&sh.k_full[s % NS], (uint32_t)(s / NS) & 1u) && now_ns() < t1) {}
        for (int s = max(0, sent_v - NS); s < sent_v; ++s)
          while (!mbar_try_wait(&sh.v_full[s % NS], (uint32_t)(s / NS) & 1u) && now_ns() < t1) {}
        while (sent_raw && !mbar_try_wait(&sh.raw, (uint32_t)(sent_raw - 1) & 1u) && now_ns() < t1) {}
      }
    }
  } else {
    regs_dec<kRegsRest>();
    const int a = warp - kMmaWarp;
    if (a > 1) {
      if (a == 2) tree_masks(p.parents ? p.parents + n * p.S : nullptr, p.S, lane, sh.mask, sh.jump);
      stage_q(warp - kLoadWarps - 2);
    } else if (lane == 0) {
      // ---------------------------------------------------------- MMA issue of stream a
      const uint32_t id_s = idesc_bf16(128, BN, 0, 0), id_o = idesc_bf16(128, DP, 0, 1);
      const uint32_t sq = smem_u32(smem) + (split ? (uint32_t)(a * QP * F::QTILE) : 0u);
      const uint32_t sk = smem_u32(smem) + F::K_OFF, sv = smem_u32(smem) + F::V_OFF;
      const uint32_t ts = tmem + F::S_COL + (uint32_t)(a * BN), to = tmem + F::O_COL + (uint32_t)(a * DP);
      const uint32_t tt = tmem + F::T_COL + (uint32_t)(a * BN / 2);
      const int cnt = count(a);
      bool ok = mbar_wait(&sh.q_bar, 0, abort_flag, err, 62);
      // S of tile i, then O of it: tcgen05 MMAs of one thread run in issue
      // order, so S of tile i + 1 overwrites P of tile i after O has read it
      for (int i = 0; i <= cnt && ok; ++i) {
        if (i > 0) {
          const int t = tile(a, i - 1);
          ok = mbar_wait(&sh.p_bar[a], (uint32_t)(i - 1) & 1u, abort_flag, err, 58) &&
               mbar_wait(&sh.v_full[t % NS], (uint32_t)(t / NS) & 1u, abort_flag, err, 59);
          if (!ok) break;
          fence_after();
          const uint64_t bd = smem_desc(sv + (uint32_t)((t % NS) * F::TILE), BN * 128, 1024, 2);
#pragma unroll
          for (int kk = 0; kk < BN / 16; ++kk) {
            const uint32_t pc = ts + (uint32_t)((kk / 2) * 32 + (kk % 2) * 8);
            mma_bf16_ts(to, pc, bd + kk * (2048 >> 4), id_o, i > 1 || kk > 0 ? 1u : 0u);
            if (QP == 3) {
              mma_bf16_ts(to, pc + 16, bd + kk * (2048 >> 4), id_o, 1u);
              mma_bf16_ts(to, tt + (uint32_t)(kk * 8), bd + kk * (2048 >> 4), id_o, 1u);
            }
          }
          mma_commit(&sh.o_bar[a]);
          mma_commit(&sh.v_free[t % NS]);
        }
        if (i < cnt) {
          const int t = tile(a, i);
          ok = mbar_wait(&sh.k_full[t % NS], (uint32_t)(t / NS) & 1u, abort_flag, err, 57);
          if (!ok) break;
          fence_after();
          const uint64_t qd = smem_desc(sq, 16, 1024, 2);
          const uint64_t kd = smem_desc(sk + (uint32_t)((t % NS) * F::TILE), 16, 1024, 2);
#pragma unroll
          for (int part = QP - 1; part >= 0; --part)  // the accumulator truncates: small products first
#pragma unroll
            for (int kk = 0; kk < DP / 16; ++kk)
              mma_bf16(ts, qd + ((part * F::QTILE + (kk / 4) * 128 * 128 + (kk % 4) * 32) >> 4),
                       kd + (((kk / 4) * BN * 128 + (kk % 4) * 32) >> 4), id_s, part < QP - 1 || kk > 0 ? 1u : 0u);
          mma_commit(&sh.s_bar[a]);
          mma_commit(&sh.k_free[t % NS]);
        }
      }
      // the accumulator is final, and no MMA of the stream reads shared memory, once this passes
      if (ok && cnt > 0) mbar_wait(&sh.o_bar[a], (uint32_t)(cnt - 1) & 1u, abort_flag, err, 60);
    }
  }
  // Registers go back to the launch's share: the loading and MMA warpgroups take
  // theirs only once every softmax warp has had and returned its own (before
  // that, a warpgroup that is done early could take what a softmax warp still
  // waits for, and neither would go on).
  __syncwarp();
  fence_before();
  __syncthreads();
  if (warp >= kSoftWarps) regs_inc<kRegsLaunch>();
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
                count(a) > 0 ? make_uint4(r[j], r[j + 1], r[j + 2], r[j + 3]) : make_uint4(0, 0, 0, 0);
      }
    }
  }
  fence_before();
  __syncthreads();
  if (warp == 0) {
    fence_after();
    tmem_dealloc(tmem, F::COLS);
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
      float pm[16], pl[16], mx = -INFINITY, l = 0.f;
#pragma unroll
      for (int j = 0; j < 16; ++j) {
        pm[j] = -INFINITY, pl[j] = 0.f;
        if (j < np) {
          const uint32_t c = (uint32_t)(split ? j : j / 2);
          const int at = split ? i : (j & 1) * 128 + i;
          asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(pm[j]) : "r"(cluster_addr(&sh.m[at], c)));
          asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(pl[j]) : "r"(cluster_addr(&sh.l[at], c)));
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
#pragma unroll
      for (int j = 0; j < 16; ++j)
        if (j < np) wgt[k * np + j] = pm[j] / l;
    }
    int bad = 0;
    if (!I8)
      for (uint32_t c = 0; c < C; ++c) {
        int x;
        asm volatile("ld.shared::cluster.s32 %0, [%1];" : "=r"(x) : "r"(cluster_addr(&sh.bad, c)));
        bad |= x;
      }
    __syncthreads();
    constexpr int LPR = DP / 4;
    const int gl = tid % LPR;
    for (int k = tid / LPR; k < mine; k += kThreads / LPR) {
      const int i = k * (int)C + (int)rank;
      float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
      for (int j0 = 0; j0 < np; j0 += 8) {
        float4 x[8];
#pragma unroll
        for (int j = 0; j < 8; ++j)
          if (j0 + j < np) {
            const uint32_t c = (uint32_t)(split ? j0 + j : (j0 + j) / 2);
            const int at = split ? i : (j & 1) * 128 + i;
            asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
                         : "=f"(x[j].x), "=f"(x[j].y), "=f"(x[j].z), "=f"(x[j].w)
                         : "r"(cluster_addr(so + at * F::LDO + gl * 4, c)));
          }
#pragma unroll
        for (int j = 0; j < 8; ++j)
          if (j0 + j < np) {
            const float w = wgt[k * np + j0 + j];
            if (w != 0.f) {  // a part without keys has no meaning for its row
              acc.x = fmaf(x[j].x, w, acc.x);
              acc.y = fmaf(x[j].y, w, acc.y);
              acc.z = fmaf(x[j].z, w, acc.z);
              acc.w = fmaf(x[j].w, w, acc.w);
            }
          }
      }
      finish4(p, w, r0 + i, gl * 4, acc, 1.f, sh.mask, bad);
    }
  }
  cluster_sync();
}

template <int DP, int BN, int QP, bool I8>
cudaError_t launch(const CacheAttnArgs& a, cudaStream_t stream) {
  using F = Cfg<DP, BN, QP>;
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
  // one CTA fits an SM: split until the CTAs fill the SMs once, or a CTA has two tiles
  int C = 1;
  while (C < kMaxCluster && items * (C + 1) <= sm_count() && c.T / (C + 1) >= 2 * BN) ++C;
  return launch_cluster(cache_attn_tc<DP, BN, QP, I8>, items * C, C, kThreads, F::SMEM, stream, mk, mv, p, err);
}

}  // namespace

bool cache_attention_tc_takes(const CacheAttnArgs& a) {
  return a.cache.type != KvType::F32 && a.cache.D >= 64 && a.cache.D <= 128 && a.S * (a.Hq / a.cache.H) > (a.bf16 ? 16 : 4);
}

cudaError_t cache_attention_tc(const CacheAttnArgs& a, cudaStream_t stream) {
  const bool i8 = a.cache.type == KvType::I8;
  if (a.cache.D <= 64) {
    if (a.bf16) return i8 ? launch<64, 128, 1, true>(a, stream) : launch<64, 128, 1, false>(a, stream);
    return i8 ? launch<64, 128, 3, true>(a, stream) : launch<64, 128, 3, false>(a, stream);
  }
  if (a.bf16) return i8 ? launch<128, 128, 1, true>(a, stream) : launch<128, 128, 1, false>(a, stream);
  return i8 ? launch<128, 64, 3, true>(a, stream) : launch<128, 64, 3, false>(a, stream);
}

}  // namespace sb
