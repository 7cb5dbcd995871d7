// Attention of few query rows over a bf16 or int8 cache: one token whose query
// heads share a cache head, or a short draft.  Same definition as
// cache_attention.cu.
//
// Reading the cache once bounds it; on the CUDA cores the products (2 FMA per
// value and row) pass that from 2 to 4 rows on.  Here a warp multiplies with
// m16n8k16 bf16 instructions.  (A tcgen05 tile has 128 rows, of which up to 16
// would be used, and needs every tile converted and swizzled in shared memory;
// cache_attention_tc.cu takes over where its rows fill.)
//
// Each warp streams its steps of keys through its own ring of stages in shared
// memory, filled by TMA (one lane issues 2 to 4 copies a step; loads into
// registers kept too few bytes under way, and asynchronous copies per lane cost
// too many instructions).  There is no barrier between warps in the loop.
//
//   S = Q K^T  A = Q (16 rows), B = K: lane (g, c) = (lane / 4, lane % 4) holds
//              key g's values.  The head dimension may be summed in any order,
//              so a lane takes consecutive values (one 16-byte piece: 8 bf16
//              or 16 codes) and Q is laid out to match.
//   O += P V   A = P: the accumulators of S are its operand layout already.  B
//              pairs two keys of one column: lane (g, c) loads consecutive
//              columns of keys 2c, 2c + 1, 2c + 8, 2c + 9 and pairs them by
//              byte permutation; the columns' order is undone at the end.
//
// f32 queries: a value is the sum of three bf16 (f16) parts, exactly.  With at
// most four rows the parts fill the 16 rows of A (0-3 first, 8-11 second, 4-7
// third part), so f32 accuracy costs no more instructions; S is the sum over a
// lane's two rows and its partner's.  P is split the same way, and the parts'
// products accumulate apart.
//
// int8 codes become f16 exactly (see codes below), and Q and P are f16 there
// too; key scales multiply S, value scales P.
#include <type_traits>

#include "cache_attn.h"

namespace sb {
namespace {

using namespace cattn;

constexpr int NW = 4;        // warps of a CTA
constexpr float kLazy = 8.f;  // a row's maximum moves when it would grow by more than this (log2)

// D += A B, 16 x 8 x 16, of bf16 or f16 values.
template <bool F16>
__device__ __forceinline__ void mma16816(float* d, const uint32_t* a, uint32_t b0, uint32_t b1) {
  if (F16)
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// (c + 128) 2^-24, a subnormal f16, in one instruction: for the first product,
// where sum q (c + 128) - 128 sum q costs one or two of 24 bits.
__device__ __forceinline__ uint32_t codes_plus_128(uint32_t t) { return (t & 0x00ff00ffu) ^ 0x00800080u; }

// Four bytes to shared memory, asynchronously; zero where `in` is false.
__device__ __forceinline__ void copy4(uint32_t dst, const void* src, bool in) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst), "l"(src), "r"(in ? 4 : 0) : "memory");
}
__device__ __forceinline__ void copies_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void copies_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

// Takes values that are not finite out of a word of two bf16.
__device__ __forceinline__ uint32_t finite_only(uint32_t w, bool& bad) {
  if ((w & 0x7f80u) == 0x7f80u) w &= 0xffff0000u, bad = true;
  if ((w & 0x7f800000u) == 0x7f800000u) w &= 0xffffu, bad = true;
  return w;
}

// DP: head size padded to 64 or 128.  MODE: bf16 queries of at most 16 rows
// (kRows16) or 8 (kRows8: rows 8-15 of the second product hold what bf16 left of
// P, so P has 16 bits), f32 queries in blocks of 4 rows (kF32).
enum Mode { kRows16, kRows8, kF32 };
template <int DP, bool I8, int MODE, int ST>
struct MmaCfg {
  static constexpr int RMAX = MODE == kF32 ? 4 : MODE == kRows8 ? 8 : 16;  // rows of the CTA
  static constexpr int NR = MODE == kRows16 ? 2 : 1;                       // of a lane
  static constexpr int KB = 4096 / (DP * (I8 ? 1 : 2));        // keys per step: 4 KB of K, 4 KB of V
  static constexpr int EK = I8 ? 16 : 8;                       // values of a lane's 16-byte piece of K
  static constexpr int KL = DP / (4 * EK);                     // such pieces per key
  static constexpr int EV = I8 ? DP / 8 : 8;                   // values of a lane's piece of V
  static constexpr int VL = DP / (8 * EV);                     // such pieces per key
  static constexpr int RB = DP * (I8 ? 1 : 2) < 128 ? 64 : 128;  // bytes of a row in a TMA box
  static constexpr int BOXES = DP * (I8 ? 1 : 2) / RB, BOX = KB * RB;
  // a warp's stage: K boxes, V boxes; its scales stand behind all stages
  static constexpr int STAGE = 2 * BOXES * BOX, STAGES = ST;
  static constexpr int SC_OFF = NW * STAGES * STAGE, END = SC_OFF + (I8 ? NW * STAGES * KB * 8 : 0);
  static constexpr int THREADS = NW * 32;
  static constexpr int JOIN = (NW + 1) * RMAX * DP * 4;
  static constexpr int SMEM = END > JOIN ? END : JOIN;
};

// The keys of a block of 8 in the order in which the fragments' columns take
// them, so that the 16-byte pieces that a quarter of a warp reads together lie
// in different banks of the swizzled boxes, for K (two keys, four pieces each)
// and V (four keys, two pieces each).
template <int RB>
__device__ __forceinline__ int key_of(int x) {
  if (RB == 128) return x & 1 ? (x - 1) ^ 5 : x;  // 0 5 2 7 4 1 6 3
  const int e = ((x >> 1) & 1) | ((x >> 1) & 2) << 1;
  return x & 1 ? e ^ 3 : e;  // 0 3 1 2 4 7 5 6
}
// Byte of piece u (16 bytes) of row `key` in a box, as TMA swizzles it.
template <int RB>
__device__ __forceinline__ int piece_at(int key, int u) {
  return key * RB + ((RB == 128 ? u ^ (key & 7) : u ^ (key >> 1 & 3)) << 4);
}

template <int DP, bool I8, int MODE, int ST>
__global__ void __launch_bounds__(NW * 32)
    cache_attn_mma(const __grid_constant__ CUtensorMap mK, const __grid_constant__ CUtensorMap mV, const Params p,
                   int* err) {
  using F = MmaCfg<DP, I8, MODE, ST>;
  constexpr bool Q32 = MODE == kF32;
  constexpr bool F16 = I8;  // operands: f16 for int8 caches, bf16 for bf16 ones
  // 9 to 16 bf16 rows fill A, so the second part of P takes products of its own: over
  // bf16 caches, which reading bounds (8 x 12 caches of 465 keys 9.2 us, 9.0 with one
  // part, that is with 2^-8 of each probability left out in place of 2^-16).  f16 leaves
  // 2^-11 out, an eighth of the output's rounding, and keeps one (4 x 8 int8 caches of
  // 30K keys of 128: 68 us, 76 with two).
  constexpr bool P2 = MODE == kRows16 && !I8;
  constexpr int KB = F::KB, NB = KB / 8, KG = KB / 16, EK = F::EK, KL = F::KL, VL = F::VL, NR = F::NR, RMAX = F::RMAX;
  constexpr int RB = F::RB, BOX = F::BOX, STAGES = F::STAGES;
  extern __shared__ __align__(1024) float sm[];  // the warps' stages, later their partial outputs
  __shared__ uint64_t s_full[NW][F::STAGES];
  __shared__ volatile int s_abort;
  __shared__ unsigned long long s_mask[kKvMaxTokens];
  __shared__ int s_jump[kKvMaxTokens];
  __shared__ float s_m[NW * RMAX], s_l[NW * RMAX], s_ml[2 * RMAX];
  __shared__ int s_bad;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, c = lane & 3;
  // nothing of the previous kernel is needed for this
  if (tid == 0) {
    asm volatile("prefetch.tensormap [%0];" ::"l"(&mK) : "memory");
    asm volatile("prefetch.tensormap [%0];" ::"l"(&mV) : "memory");
    for (int i = 0; i < NW * STAGES; ++i) tc::mbar_init(&s_full[0][i], 1);
    s_bad = 0;
    s_abort = tc::smem_u32(sm) & 1023u ? 1 : 0;
    if (s_abort) atomicExch(err, 63);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    tc::fence_proxy_async();
  }
  __syncthreads();
  pdl_prologue();
  const Place w = find_place(p);
  const int r0 = w.chunk * RMAX, rows = min(RMAX, p.S * p.G - r0);
  // this CTA's keys, in whole steps of the warps' stride
  const int64_t per = ((w.end + w.C - 1) / w.C + KB - 1) / KB * KB;
  const int64_t lo = min((int64_t)w.rank * per, w.end), hi = min(lo + per, w.end);

  const float *ksb = I8 ? p.ks + w.nh * p.T : nullptr, *vsb = I8 ? p.vs + w.nh * p.T : nullptr;
  uint8_t* const ring = (uint8_t*)sm + warp * STAGES * F::STAGE;
  float* const scales = (float*)((uint8_t*)sm + F::SC_OFF) + warp * STAGES * KB * 2;
  uint64_t* const full = s_full[warp];
  // One step's keys into stage `st` of this warp: boxes by TMA (rows behind the
  // cache's capacity arrive as zeros), scales by asynchronous copies.
  auto fetch = [&](int64_t t, int st) {
    if (lane == 0 && !s_abort) {
      tc::mbar_expect_tx(&full[st], F::STAGE);
      uint8_t* dst = ring + st * F::STAGE;
      if (F::BOXES == 1 || p.D == DP) {
        tc::tma_load_4d(dst, &mK, &full[st], 0, (int)t, 0, (int)w.nh);
        tc::tma_load_4d(dst + F::BOXES * BOX, &mV, &full[st], 0, (int)t, 0, (int)w.nh);
      } else {
#pragma unroll
        for (int i = 0; i < F::BOXES; ++i) {
          tc::tma_load_4d(dst + i * BOX, &mK, &full[st], i * (RB / (I8 ? 1 : 2)), (int)t, 0, (int)w.nh);
          tc::tma_load_4d(dst + (F::BOXES + i) * BOX, &mV, &full[st], i * (RB / (I8 ? 1 : 2)), (int)t, 0, (int)w.nh);
        }
      }
    }
    if (I8) {
#pragma unroll
      for (int i = 0; i < KB / 32; ++i) {
        const bool in = t + i * 32 + lane < w.end;
        const uint32_t at = tc::smem_u32(scales + st * KB * 2 + i * 32 + lane);
        copy4(at, in ? ksb + t + i * 32 + lane : ksb, in);
        copy4(at + KB * 4, in ? vsb + t + i * 32 + lane : vsb, in);
      }
    }
  };
  // the queries' loads go out first, then the first steps' copies
  float y[NR][DP / 16][4];
#pragma unroll
  for (int r = 0; r < NR; ++r) {
    const int row = Q32 ? g & 3 : g + 8 * r;
    const bool in = row < rows;
    const int64_t at = in ? row_at(p, w, r0 + row) : 0;
#pragma unroll
    for (int s = 0; s < DP / 16; ++s) {
      const int d = (s / (EK / 4)) * 4 * EK + c * EK + (s % (EK / 4)) * 4;
      float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
      if (in && d < p.D) {
        if (Q32) {
          x = *(const float4*)((const float*)p.q + at + d);
        } else {
          const uint2 z = *(const uint2*)((const __nv_bfloat16*)p.q + at + d);
          const float2 a = unpack2<false>(z.x), b = unpack2<false>(z.y);
          x = make_float4(a.x, a.y, b.x, b.y);
        }
      }
      y[r][s][0] = x.x, y[r][s][1] = x.y, y[r][s][2] = x.z, y[r][s][3] = x.w;
    }
  }
  int64_t t0 = lo + warp * KB;
  constexpr int STRIDE = NW * KB;
#pragma unroll
  for (int i = 0; i < STAGES; ++i) {
    if (t0 + i * STRIDE < hi) fetch(t0 + i * STRIDE, i);
    if (I8) copies_commit();
  }
  if (warp == 0) tree_masks(p.parents ? p.parents + w.n * p.S : nullptr, p.S, lane, s_mask, s_jump);

  // Q: k-step s takes values d .. d + 3 of the lane's EK, as the pairs of an
  // int8 word (bytes 0 and 2, bytes 1 and 3) or of consecutive bf16 values.
  // For f16 a row is scaled (f16_row_scale); S is multiplied back by `fs`.
  uint32_t q[DP / 16][4];
  float fs[NR], pre[NR], sum_q[NR];
#pragma unroll
  for (int r = 0; r < NR; ++r) {
    float up = 1.f;
    fs[r] = p.scale2;
    pre[r] = 1.f;
    sum_q[r] = 0.f;
    if (F16) {
      float big = 0.f;
#pragma unroll
      for (int s = 0; s < DP / 16; ++s)
#pragma unroll
        for (int i = 0; i < 4; ++i) big = fmaxf(big, fabsf(y[r][s][i]));
      big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, 1));
      big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, 2));
      float down;
      up = f16_row_scale(big, down);
      fs[r] = p.scale2 * down;
      // A row's factor up to 1 goes before the key's scale, a larger one after it:
      // neither product passes f32's range unless the score does.
      if (fabsf(fs[r]) <= 1.f) pre[r] = fs[r], fs[r] = 1.f;
    }
#pragma unroll
    for (int s = 0; s < DP / 16; ++s) {
      float2 a = make_float2(y[r][s][0] * up, y[r][s][I8 ? 2 : 1] * up),
             b = make_float2(y[r][s][I8 ? 1 : 2] * up, y[r][s][3] * up);
      if (Q32) {
        const uint32_t a1 = take2<F16>(a.x, a.y), b1 = take2<F16>(b.x, b.y);
        const uint32_t a2 = take2<F16>(a.x, a.y), b2 = take2<F16>(b.x, b.y);
        const uint32_t a3 = pack2<F16>(a.x, a.y), b3 = pack2<F16>(b.x, b.y);
        q[s][0] = g < 4 ? a1 : a3;
        q[s][1] = g < 4 ? a2 : 0u;
        q[s][2] = g < 4 ? b1 : b3;
        q[s][3] = g < 4 ? b2 : 0u;
      } else {
        q[s][r] = pack2<F16>(a.x, a.y);
        q[s][2 + r] = pack2<F16>(b.x, b.y);
        if (MODE == kRows8) q[s][1] = q[s][3] = 0u;
        if (F16) {
          const float2 a1 = unpack2<F16>(q[s][r]), b1 = unpack2<F16>(q[s][2 + r]);
          sum_q[r] += (a1.x + a1.y) + (b1.x + b1.y);
        }
      }
    }
    if (F16 && !Q32) {
      sum_q[r] += __shfl_xor_sync(0xffffffffu, sum_q[r], 1);
      sum_q[r] += __shfl_xor_sync(0xffffffffu, sum_q[r], 2);
      sum_q[r] *= 128.f * pre[r];  // acc = 2^-24 sum q (c + 128):  S = (acc 2^24 - 128 sum q) pre fs
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

  const int kg = key_of<RB>(g), kc[2] = {key_of<RB>(2 * c), key_of<RB>(2 * c + 1)};
  int st = 0, vref[NR];
  uint32_t phase = 0;
  float vdown[NR], top[NR];  // top: a row's largest P times scale, once they are wide
  ScaleRange range;
#pragma unroll
  for (int r = 0; r < NR; ++r) vref[r] = kVrefFirst, vdown[r] = vref_down(kVrefFirst), top[r] = 0.f;
  auto ready = [&] {  // the keys at t0, and the range of their scales
    if (I8) {  // a lane's copies of scales are there for the others once the warp has met
      copies_wait<STAGES - 1>();
      __syncwarp();
#pragma unroll
      for (int i = 0; i < KB / 32; ++i) range.lane_adds(scales[(st * 2 + 1) * KB + i * 32 + lane]);
      range.join_lanes();
    }
    return __all_sync(0xffffffffu, tc::mbar_wait(&full[st], phase, &s_abort, err, 64)) != 0;
  };
  auto turn = [&](auto wide_tag) {
    constexpr bool WIDE = decltype(wide_tag)::value;
    const uint8_t *const stage = ring + st * F::STAGE, *const stage_v = stage + F::BOXES * BOX;
    const float* const sc = scales + st * KB * 2;
    float s[NB][4];
#pragma unroll
    for (int b = 0; b < NB; ++b) s[b][0] = s[b][1] = s[b][2] = s[b][3] = 0.f;
#pragma unroll
    for (int i = 0; i < KL; ++i) {
      uint4 x[NB];
#pragma unroll
      for (int b = 0; b < NB; ++b)
        x[b] = *(const uint4*)(stage + (i * 4 * 16 / RB) * BOX + piece_at<RB>(b * 8 + kg, (i * 4) % (RB / 16) + c));
#pragma unroll
      for (int k = 0; k < EK / 4; ++k)
#pragma unroll
        for (int b = 0; b < NB; ++b) {
          const uint32_t word[4] = {x[b].x, x[b].y, x[b].z, x[b].w};
          const uint32_t* a = q[i * (EK / 4) + k];
          if (I8 && Q32) mma16816<F16>(s[b], a, codes(word[k]), codes(word[k] >> 8));
          else if (I8) mma16816<F16>(s[b], a, codes_plus_128(word[k]), codes_plus_128(word[k] >> 8));
          else mma16816<F16>(s[b], a, word[(k % 2) * 2], word[(k % 2) * 2 + 1]);
        }
    }
    // scores of the lane's NR rows and two keys per block, in units of log2
    float x[NB][NR][2];
#pragma unroll
    for (int b = 0; b < NB; ++b) {
      float2 f = make_float2(1.f, 1.f);
      if (I8) f = make_float2(sc[b * 8 + kc[0]], sc[b * 8 + kc[1]]);
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        if (Q32) {
          const float y = s[b][i] + s[b][2 + i];
          x[b][0][i] = (y + __shfl_xor_sync(0xffffffffu, y, 16)) * (I8 ? pre[0] : 1.f);
        } else {
#pragma unroll
          for (int r = 0; r < NR; ++r)
            x[b][r][i] = I8 ? fmaf(s[b][2 * r + i], 16777216.f * pre[r], -sum_q[r]) : s[b][2 * r + i];
        }
#pragma unroll
        for (int r = 0; r < NR; ++r) x[b][r][i] = (I8 ? x[b][r][i] * (i ? f.y : f.x) : x[b][r][i]) * fs[r];
      }
    }
    const bool masked = t0 + KB > w.pre || t0 + KB > hi;
    if (masked) {
#pragma unroll
      for (int b = 0; b < NB; ++b)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const int64_t t = t0 + b * 8 + kc[i];
#pragma unroll
          for (int r = 0; r < NR; ++r) {
            const bool see = t < hi && (t < w.pre || (seen[r] >> (t - w.pos) & 1ull));
            if (!see) x[b][r][i] = -INFINITY;
          }
        }
    }
    const float lazy = WIDE && range.big() ? 0.f : kLazy;
    float mx[NR];
    bool move = false;
#pragma unroll
    for (int r = 0; r < NR; ++r) {
      mx[r] = -INFINITY;
#pragma unroll
      for (int b = 0; b < NB; ++b) mx[r] = fmaxf(mx[r], fmaxf(x[b][r][0], x[b][r][1]));
      mx[r] = fmaxf(mx[r], __shfl_xor_sync(0xffffffffu, mx[r], 1));
      mx[r] = fmaxf(mx[r], __shfl_xor_sync(0xffffffffu, mx[r], 2));
      move |= mx[r] > m[r] + lazy;
    }
    if (__any_sync(0xffffffffu, move)) {
#pragma unroll
      for (int r = 0; r < NR; ++r) {
        const float mn = fmaxf(m[r], mx[r]), f = mn == -INFINITY ? 0.f : tc::ex2(m[r] - mn);
        l[r] *= f;
        if (WIDE) top[r] *= f;
        m[r] = mn;
#pragma unroll
        for (int j = 0; j < DP / 8; ++j) {
          o[j][2 * r] *= f, o[j][2 * r + 1] *= f;
          if (MODE != kRows16) o[j][2] *= f, o[j][3] *= f;
        }
      }
    }
    if (I8 && (WIDE || range.hi > vref[0])) {
      int next[NR];
      bool change = !WIDE;
#pragma unroll
      for (int r = 0; r < NR; ++r) {
        next[r] = range.hi;
        if (WIDE) {
          const float base = m[r] == -INFINITY ? 0.f : m[r];
          float big = 0.f;
#pragma unroll
          for (int b = 0; b < NB; ++b)
#pragma unroll
            for (int i = 0; i < 2; ++i)
              if (x[b][r][i] != -INFINITY) big = fmaxf(big, tc::ex2(x[b][r][i] - base) * fabsf(sc[KB + b * 8 + kc[i]]));
          big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, 1));
          big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, 2));
          top[r] = fmaxf(top[r], big);
          next[r] = wide_vref(vref[r], top[r]);
          change |= next[r] != vref[r];
        }
      }
      if (__any_sync(0xffffffffu, change)) {
#pragma unroll
        for (int r = 0; r < NR; ++r) {
          const float f = pow2(vref[r] - next[r]);
#pragma unroll
          for (int j = 0; j < DP / 8; ++j) {
            o[j][2 * r] *= f, o[j][2 * r + 1] *= f;
            if (MODE != kRows16) o[j][2] *= f, o[j][3] *= f;
          }
          vref[r] = next[r];
          vdown[r] = vref_down(vref[r]);
        }
      }
    }
    uint32_t a[KG][4], a2[KG][4];  // P, and with P2 what its rounding left
#pragma unroll
    for (int b = 0; b < NB; ++b)
#pragma unroll
      for (int r = 0; r < NR; ++r) {
        const float base = m[r] == -INFINITY ? 0.f : m[r];
        float2 f = make_float2(1.f, 1.f);
        if (I8) f = make_float2(sc[KB + b * 8 + kc[0]], sc[KB + b * 8 + kc[1]]);
        float y[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const float e = tc::ex2(x[b][r][i] - base);
          l[r] += e;
          y[i] = I8 ? (masked && x[b][r][i] == -INFINITY ? 0.f : e * (i ? f.y : f.x) * vdown[r]) : e;
        }
        uint32_t* dst = &a[b / 2][(b & 1) * 2];
        if (Q32) {
          const uint32_t h1 = take2<F16>(y[0], y[1]), h2 = take2<F16>(y[0], y[1]), h3 = pack2<F16>(y[0], y[1]);
          dst[0] = g < 4 ? h1 : h3;
          dst[1] = g < 4 ? h2 : 0u;
        } else if (MODE == kRows8) {
          dst[0] = take2<F16>(y[0], y[1]);
          dst[1] = pack2<F16>(y[0], y[1]);
        } else {
          dst[r] = take2<F16>(y[0], y[1]);
          if (P2) a2[b / 2][(b & 1) * 2 + r] = pack2<F16>(y[0], y[1]);
        }
      }
#pragma unroll
    for (int k = 0; k < KG; ++k)
#pragma unroll
      for (int j = 0; j < VL; ++j) {
        uint32_t word[4][4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int key = k * 16 + kc[i & 1] + (i >> 1) * 8;
          if (F::EV * (I8 ? 1 : 2) == 8) {
            const uint2 x2 = *(const uint2*)(stage_v + piece_at<RB>(key, g >> 1) + (g & 1) * 8);
            word[i][0] = x2.x, word[i][1] = x2.y;
          } else {
            const uint4 x4 = *(const uint4*)(stage_v + j * BOX + piece_at<RB>(key, g));
            word[i][0] = x4.x, word[i][1] = x4.y, word[i][2] = x4.z, word[i][3] = x4.w;
          }
          if (!I8 && masked && t0 + key >= w.pre) {
            bool bad = false;
#pragma unroll
            for (int e = 0; e < 4; ++e) word[i][e] = finite_only(word[i][e], bad);
            if (bad && t0 + key < w.end) s_bad = 1;
          }
        }
#pragma unroll
        for (int e = 0; e < F::EV; ++e) {
          uint32_t b[2];
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            if (I8) {  // bytes e of the two keys to bytes 0 and 2
              const uint32_t y = __byte_perm(word[2 * i][e / 4], word[2 * i + 1][e / 4], e & 2 ? 0x7632 : 0x5410);
              b[i] = codes(e & 1 ? y >> 8 : y);
            } else {
              b[i] = __byte_perm(word[2 * i][e / 2], word[2 * i + 1][e / 2], e & 1 ? 0x7632 : 0x5410);
            }
          }
          mma16816<F16>(o[j * F::EV + e], a[k], b[0], b[1]);
          if (P2) mma16816<F16>(o[j * F::EV + e], a2[k], b[0], b[1]);
        }
      }
    __syncwarp();  // the stage has been read
    if (t0 + STAGES * STRIDE < hi) fetch(t0 + STAGES * STRIDE, st);
    if (I8) copies_commit();
    if (++st == STAGES) st = 0, phase ^= 1u;
    t0 += STRIDE;
  };
  while (t0 < hi && ready() && !range.wide) turn(std::false_type{});
  if constexpr (I8) {
#pragma unroll
    for (int r = 0; r < NR; ++r) top[r] = m[r] == -INFINITY ? 0.f : pow2(vref[r]);
    while (t0 < hi && ready()) turn(std::true_type{});
  }
  if (I8) copies_wait<0>();
  if (s_abort && lane == 0 && t0 < hi) {  // the boxes of the steps that were not taken may still be on their way
    const unsigned long long give_up = tc::now_ns() + tc::kTimeoutNs;
    for (int i = 0; i < STAGES && t0 < hi; ++i, t0 += STRIDE) {
      while (!tc::mbar_try_wait(&full[st], phase) && tc::now_ns() < give_up) {}
      if (++st == STAGES) st = 0, phase ^= 1u;
    }
  }
  __syncthreads();  // every warp has read its last stage: the memory takes the partial outputs

  // the warp's parts: row, and columns 2c, 2c + 1 of block (j, e) = value (2c) EV + e of load j
#pragma unroll
  for (int r = 0; r < NR; ++r) {
    const float vup = vref_up(vref[r]);
    l[r] += __shfl_xor_sync(0xffffffffu, l[r], 1);
    l[r] += __shfl_xor_sync(0xffffffffu, l[r], 2);
    const int row = Q32 ? g & 3 : g + 8 * r;
    if (c == 0 && (!Q32 || g < 4)) s_m[warp * RMAX + row] = m[r], s_l[warp * RMAX + row] = l[r];
#pragma unroll
    for (int j = 0; j < DP / 8; ++j)
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        float y = o[j][2 * r + i];
        if (MODE != kRows16) y += o[j][2 + i];
        if (Q32) y += __shfl_xor_sync(0xffffffffu, y, 16);
        if (I8) y *= vup;
        const int d = (j / F::EV) * 8 * F::EV + (2 * c + i) * F::EV + j % F::EV;
        if (!Q32 || g < 4) sm[(warp * RMAX + row) * DP + d] = y;
      }
  }
  join_and_store<NW, RMAX, DP>(p, w, r0, rows, sm, s_m, s_l, sm + NW * RMAX * DP, s_ml, s_mask, I8 ? nullptr : &s_bad);
}

template <int DP, bool I8, int MODE, int ST>
cudaError_t launch(const CacheAttnArgs& a, int C, cudaStream_t stream) {
  using F = MmaCfg<DP, I8, MODE, ST>;
  const Params p = make_params(a, F::RMAX);
  const KvCacheView& c = a.cache;
  CUtensorMap mk, mv;
  const uint32_t blocks = c.D == DP ? F::BOXES : 1;
  if (!tc_make_map_rows(&mk, c.k, I8, c.D, c.T, c.N * c.H, F::RB, F::KB, blocks) ||
      !tc_make_map_rows(&mv, c.v, I8, c.D, c.T, c.N * c.H, F::RB, F::KB, blocks))
    return cudaErrorNotSupported;
  int* err = tc_error_word();
  if (!err) return cudaErrorMemoryAllocation;
  return launch_cluster(cache_attn_mma<DP, I8, MODE, ST>, c.N * c.H * p.chunks * C, C, F::THREADS, F::SMEM, stream, mk,
                        mv, p, err);
}

template <int DP, bool I8, int MODE>
cudaError_t by_items(const CacheAttnArgs& a, cudaStream_t stream) {
  const int64_t items = a.cache.N * a.cache.H;
  constexpr int KB = MmaCfg<DP, I8, MODE, 3>::KB;
  const int64_t row = a.cache.D * (I8 ? 1 : 2);  // bytes
  // Items are split while the CTAs are one wave of three per SM and a warp keeps
  // two steps; and, for batches of uneven lengths, which would end with their longest
  // items alone, until no CTA has more than 256 KB of K (64 x 8 items of up to 4K
  // bf16 keys of 128: 91 us, unsplit 96).
  int C = 1;
  while (may_double(C, items) && a.cache.T / (2 * C) >= 4 * KB &&
         (items * 2 * C <= 3 * sm_count() || a.cache.T * row > C * (256 << 10)))
    C *= 2;
  // An SM holds two CTAs of three stages, or three of two (replayed graphs: 64 x 12
  // items of up to 1K int8 keys of 64, 25.6 us, 28.7 with three stages; 128 x 4 of up to
  // 2K bf16 keys of 128, 53 and 58; but 32 x 8 of 3.8K int8 keys of 128 as one wave of two
  // per SM, 87 and 64).
  if (items * C > 2 * sm_count()) return launch<DP, I8, MODE, 2>(a, C, stream);
  return launch<DP, I8, MODE, 3>(a, C, stream);
}

}  // namespace

// As many bf16 rows as the instruction has, and f32 rows in two blocks of 4, whose
// second reading of the cache is from L2.  There it is the faster one (in replayed
// graphs): 16 bf16 rows of 4 x 8 caches of 30K keys of 128 take 86 us from bf16 and 69
// from int8, on tcgen05 101 and 130; of 8 x 12 caches of 465 keys of 64, 9.1 and 9.8,
// 13.2 and 15.3; 8 f32 rows of 8 x 12 caches of 6K keys of 128, 83 and 83, 136 and 200
// (three blocks, 12 rows: 123 and 120, but of 300 keys 29 and 34, 17 and 23).  Two
// blocks of bf16 rows lose it: 32 rows of 6K keys, 104 us from bf16, 81 on tcgen05
// (from int8 88 and 114, but of 632 keys of 64 19 and 17).  4 f32 rows of 16 x 8 caches
// of 4K keys of 128, 57 and 39 us, on the CUDA cores 125 and 241.
//
// Reading the cache bounds the long bf16 calls (one bf16 row of 4 x 8 x 30K keys of
// 128: 83 us, 6.0 TB/s); int8 ones (60 us, 4.2 TB/s) the conversion of codes and of P,
// some five half-rate instructions per word of four codes; short ones their set-up
// and joining, some 5 us.
bool cache_attention_mma_takes(const CacheAttnArgs& a) {
  return on_tensor_cores(a) && a.S * (a.Hq / a.cache.H) <= (a.bf16 ? 16 : 8);
}

cudaError_t cache_attention_mma(const CacheAttnArgs& a, cudaStream_t stream) {
  const bool i8 = a.cache.type == KvType::I8, wide = a.cache.D > 64;
  if (!a.bf16) {
    if (i8) return wide ? by_items<128, true, kF32>(a, stream) : by_items<64, true, kF32>(a, stream);
    return wide ? by_items<128, false, kF32>(a, stream) : by_items<64, false, kF32>(a, stream);
  }
  if (a.S * (a.Hq / a.cache.H) > 8) {
    if (i8) return wide ? by_items<128, true, kRows16>(a, stream) : by_items<64, true, kRows16>(a, stream);
    return wide ? by_items<128, false, kRows16>(a, stream) : by_items<64, false, kRows16>(a, stream);
  }
  if (i8) return wide ? by_items<128, true, kRows8>(a, stream) : by_items<64, true, kRows8>(a, stream);
  return wide ? by_items<128, false, kRows8>(a, stream) : by_items<64, false, kRows8>(a, stream);
}

}  // namespace sb
