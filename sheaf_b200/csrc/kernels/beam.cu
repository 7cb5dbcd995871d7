// Beam search: the selection of the W best continuations of each group of W
// beams (beam_select) and the rearrangement of per-beam state to follow it
// (beam_reorder).
//
//   cand(w, v) = score_w + (z_wv - lse_w),  lse_w = log sum_v exp z_wv
//   selected: the W largest of the W x V candidates, by (value, then lowest
//   w V + v).
//
// Reading the logits once bounds the selection, so the pass over them does as
// little as it can: a cluster of C CTAs carries a group, each warp streams
// pieces of one beam's row, and a lane keeps its largest value, that value's
// lowest index and its sum of exponentials.  Lanes meet only at the end.  A
// lane's best is a 64-bit key (order-preserving image of the logit above the
// complemented index: unique, so equal logits order by index and every step
// has one answer), and of a beam's W best values none can lie in a lane whose
// best is not among the W best of all its lanes.  So each warp sends its W best
// keys; after a cluster barrier CTA r finds the W best of beams r, r + C, ..,
// reads the few values of those W lanes again (from L2) for others above the
// W-th, and sends the result to every CTA; after a second barrier each CTA
// orders the W x W survivors.  Lists cross CTAs through distributed shared
// memory: no workspace, no atomics on memory and no second launch.
//
// Within a beam the order is the logits' own.  Between beams it needs lse.  The
// first round sums f32 exponentials, off by less than kFastError; if two
// neighbours of the result from different beams, or its last candidate and any
// that was not selected from another beam, are closer than twice that (or tie),
// the group's sums are taken again in f64, whose exponentials would otherwise
// bound the kernel.  So the order is that of f64 sums in every case.
//
// 32 x 8 beams over 50304 f32 logits (52 MB, 7.9 us of reading): 19.3 us, 17.3 in a
// replayed graph (172 us with every sum in f64).  About 10 us of that are not the
// pass but what 4 beams over 65 values take as well (10.7 us): the launch, two
// cluster barriers, the join and the second look at the W best lanes.
//
// The reordering moves bytes: 64 beams' caches of 12 layers, 12 heads, 1K positions
// of 64 bf16 values (a third to nine tenths of them live): 395 us, 5.4 TB/s
// written and read; a thread reads its 16 bytes of all beams before it writes any.
#include <cuda_bf16.h>

#include <cmath>

#include "kernels.h"
#include "pdl.h"
#include "tc_common.h"

namespace sb {
namespace {

constexpr int kSelWarps = 16, kSelThreads = kSelWarps * 32;
// Bound on the error of an lse from f32 exponentials of V <= 2^31 values.  A
// term 2^-t (t: what the value is below its warp's base, in units of log2) has a
// relative error of at most 2^-22 (ex2) + 2^-23.4 |t| (its argument, two
// roundings), and terms with t > 32 + log2 of the sum of the others' number are
// below it.  A base is at most the row's maximum, so the mean of t by the sum's
// weight is at most log2(V); and at least the warp's less kBaseRoom - log2(V), so
// the mean of |t| is at most kBaseRoom.  32 terms are added in f32 (at most 9
// additions each), the rest in f64, in which sums also pass from one base to
// another: 2^-22 + kBaseRoom * 2^-23.4 + 9 * 2^-24 < 4e-6.
constexpr double kFastError = 4e-6, kBaseRoom = 35;
constexpr int EPC = 32;              // values per lane and piece
constexpr int kPiece = EPC * 32;     // values per warp and piece
constexpr int W_MAX = (int)kBeamMax;
using u64 = unsigned long long;
constexpr float kLog2e = 1.4426950408889634f;

struct SelectParams {
  const void* logits;
  const float* scores;
  const int* finished;
  float* out_scores;
  int *out_parents, *out_tokens, *out_finished;
  int64_t V, total;  // total: values of the whole logits buffer
  int W, eos;
  float step;  // a value this far above its warp's base moves the base
};

// Order-preserving image of an f32 that is not NaN; one image for both zeros, which are equal.
__device__ __forceinline__ uint32_t ordered(float x) {
  const uint32_t u = __float_as_uint(x + 0.f);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float unordered(uint32_t u) {
  return __uint_as_float(u & 0x80000000u ? u & 0x7fffffffu : ~u);
}
__device__ __forceinline__ u64 shfl64(u64 x, int src) { return __shfl_sync(0xffffffffu, x, src); }

// The N = 4 (f32) or 8 (bf16) values of a 16-byte load.
template <bool BF>
__device__ __forceinline__ void load_vec(const void* buf, int64_t at, float* x) {
  const uint4 r = *(const uint4*)((const uint8_t*)buf + at * (BF ? 2 : 4));
  const uint32_t w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if (BF) {
      x[2 * i] = __uint_as_float(w[i] << 16);
      x[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    } else {
      x[i] = __uint_as_float(w[i]);
    }
  }
}

// Values at .. at + N - 1 of the logits buffer (at: a multiple of N) where they
// belong to the row [base, base + V), -inf elsewhere.  `inside`: all of them do.
// The buffer's last values are loaded one by one where the 16 bytes would pass its
// end.
template <bool BF>
__device__ __forceinline__ void load_piece(const void* buf, bool inside, int64_t at, int64_t base, int64_t V,
                                           int64_t total, float* x) {
  constexpr int N = BF ? 8 : 4;
  if (inside) {
    load_vec<BF>(buf, at, x);
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) x[i] = -INFINITY;
    if (at < base + V && at + N <= total) {
      load_vec<BF>(buf, at, x);
    } else if (at < base + V) {
      for (int i = 0; i < N; ++i)
        if (at + i < total)
          x[i] = BF ? __bfloat162float(((const __nv_bfloat16*)buf)[at + i]) : ((const float*)buf)[at + i];
    }
#pragma unroll
    for (int i = 0; i < N; ++i)
      if (at + i < base || at + i >= base + V) x[i] = -INFINITY;
  }
}

struct SelectShared {
  u64 list[kSelWarps][W_MAX];  // a warp's best lanes' keys, in order
  double s[kSelWarps];
  float m[kSelWarps];
  // the beams that this CTA joins: the keys of all their lists, the W best of
  // them, and the other keys of those lanes that are above the W-th (a warp
  // ranks its lanes' keys in its part of the pool before that)
  u64 pool[kSelThreads];
  u64 top[W_MAX][W_MAX];
  u64 more[W_MAX][W_MAX * W_MAX];
  int more_count[W_MAX];
  double lse[W_MAX];
  // the candidates of every beam, best first (each CTA has them all)
  double cand[W_MAX][W_MAX + 1];  // padded: threads read down the columns
  int token[W_MAX][W_MAX + 1];
  int done[W_MAX];
  int rank[W_MAX * W_MAX];
  double best[W_MAX + 1];  // the first W + 1 of them, and their beams
  int beam[W_MAX + 1], pick[W_MAX];
};

__device__ __forceinline__ u64 ld_remote64(const void* p, uint32_t rank) {
  u64 x;
  asm volatile("ld.shared::cluster.u64 %0, [%1];" : "=l"(x) : "r"(tc::cluster_addr(p, rank)));
  return x;
}
__device__ __forceinline__ float ld_remote_f(const float* p, uint32_t rank) {
  float x;
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(x) : "r"(tc::cluster_addr(p, rank)));
  return x;
}
__device__ __forceinline__ void st_remote64(const void* p, uint32_t rank, u64 x) {
  asm volatile("st.shared::cluster.u64 [%0], %1;" ::"r"(tc::cluster_addr(p, rank)), "l"(x) : "memory");
}
__device__ __forceinline__ void st_remote32(const void* p, uint32_t rank, uint32_t x) {
  asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(tc::cluster_addr(p, rank)), "r"(x) : "memory");
}

// A beam's row in the logits: elements [base, base + V) of the buffer, streamed
// in pieces from `first`, the 16-byte boundary at or before it.
struct Row {
  int64_t base, first, pieces;
};
template <bool BF>
__device__ __forceinline__ Row row_of(const SelectParams& p, int64_t row) {
  Row r;
  r.base = row * p.V;
  r.first = r.base & ~(int64_t)((BF ? 8 : 4) - 1);
  r.pieces = (r.base + p.V - r.first + kPiece - 1) / kPiece;
  return r;
}
template <bool BF>
__device__ __forceinline__ void load_row(const SelectParams& p, const Row& r, int64_t c, int lane, float* x) {
  constexpr int N = BF ? 8 : 4;
  const int64_t at0 = r.first + c * kPiece + lane * N;
  if (r.first + c * kPiece >= r.base && r.first + (c + 1) * kPiece <= r.base + p.V) {
#pragma unroll
    for (int i = 0; i < EPC / N; ++i) load_vec<BF>(p.logits, at0 + i * 32 * N, x + i * N);
  } else {  // the row begins or ends in this piece: all loads first, then what does not belong to it
#pragma unroll
    for (int i = 0; i < EPC / N; ++i) {
      const int64_t at = at0 + i * 32 * N;
#pragma unroll
      for (int k = 0; k < N; ++k) x[i * N + k] = -INFINITY;
      if (at < r.base + p.V && at + N <= p.total) load_vec<BF>(p.logits, at, x + i * N);
    }
#pragma unroll
    for (int i = 0; i < EPC / N; ++i) {
      const int64_t at = at0 + i * 32 * N;
      if (at < r.base + p.V && at + N > p.total) load_piece<BF>(p.logits, false, at, r.base, p.V, p.total, x + i * N);
#pragma unroll
      for (int k = 0; k < N; ++k)
        if (at + k < r.base || at + k >= r.base + p.V) x[i * N + k] = -INFINITY;
    }
  }
}
// Whether the order of two candidates of different beams may be other than that of exact sums.
__device__ __forceinline__ bool too_close(double ahead, double behind) {
  return behind != -INFINITY && ahead - behind < 2 * kFastError + 1e-15 * fabs(ahead);
}
__device__ __forceinline__ u64 key_of(float x, int64_t idx) {
  return (u64)ordered(x) << 32 | (uint32_t)~(uint32_t)idx;
}

template <bool BF>
__global__ void __launch_bounds__(kSelThreads, 1) select_kernel(const SelectParams p) {
  __shared__ SelectShared sh;
  constexpr int N = BF ? 8 : 4;
  const uint32_t crank = tc::cluster_rank();
  uint32_t C;
  asm("mov.u32 %0, %%cluster_nctarank;" : "=r"(C));
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int W = p.W;
  const int64_t g = blockIdx.x / C;
  // warps of the cluster per beam; warp `gid` streams every `per`-th piece of its beam
  const int warps = (int)C * kSelWarps, per = warps / W;
  const int gid = (int)crank * kSelWarps + warp, beam = gid / per, sub = gid % per;
  const Row row = row_of<BF>(p, g * W + min(beam, W - 1));
  // beams b = crank + q C that this CTA joins, and the keys of one's lists
  const int joins = (int)crank < W ? (W - 1 - (int)crank) / (int)C + 1 : 0, keys = per * W;
  pdl_prologue();
  float x[EPC], y[EPC];
  if (beam < W && sub < row.pieces) load_row<BF>(p, row, sub, lane, x);
  const bool mine = beam < W && !(p.eos >= 0 && p.finished[g * W + beam]);
  float wm = -INFINITY;  // what the warp's sums are relative to (base)

  for (int round = 0;; ++round) {
    double sum = 0.;
    if (round == 0) {
      float best = -INFINITY;  // the lane's
      int at = -1;
      if (mine) {
        auto piece = [&](const float* x, int64_t c) {
          float top = fmaxf(x[0], -INFINITY);  // NaN counts as -inf, in every one of the values too
#pragma unroll
          for (int i = 1; i < EPC; ++i) top = fmaxf(top, x[i]);
          if (__any_sync(0xffffffffu, top > wm + p.step)) {  // the first piece, and hardly ever again
            float up = top;
#pragma unroll
            for (int o = 16; o; o >>= 1) up = fmaxf(up, __shfl_xor_sync(0xffffffffu, up, o));
            if (wm != -INFINITY) sum *= exp((double)wm - (double)up);
            wm = up;
          }
          if (top > best || at < 0) {
            const int64_t at0 = row.first + c * kPiece + lane * N - row.base;
            int found = -1;
            if (top > -INFINITY) {
#pragma unroll
              for (int i = EPC - 1; i >= 0; --i)
                if (x[i] == top) found = (i / N) * 32 * N + i % N;
            } else {  // values outside the row are -inf too
              for (int i = EPC - 1; i >= 0; --i) {
                const int64_t idx = at0 + (i / N) * 32 * N + i % N;
                if (idx >= 0 && idx < p.V) found = (i / N) * 32 * N + i % N;
              }
            }
            if (found >= 0) best = top, at = (int)(at0 + found);
          }
          const float b = wm == -INFINITY ? 0.f : wm;
          auto sum_up = [&](bool clean) {
            float e[4];
#pragma unroll
            for (int i = 0; i < EPC; ++i) {
              const float v = tc::ex2(((clean ? fmaxf(x[i], -INFINITY) : x[i]) - b) * kLog2e);
              e[i % 4] = i < 4 ? v : e[i % 4] + v;
            }
            return (e[0] + e[1]) + (e[2] + e[3]);
          };
          float s = sum_up(false);
          if (s != s) s = sum_up(true);  // NaN counts as -inf (a sum that stays NaN has an infinity)
          sum += (double)s;
        };
        for (int64_t c = sub; c < row.pieces; c += 2 * per) {  // the next piece is under way during one
          if (c + per < row.pieces) load_row<BF>(p, row, c + per, lane, y);
          piece(x, c);
          if (c + per >= row.pieces) break;
          if (c + 2 * per < row.pieces) load_row<BF>(p, row, c + 2 * per, lane, x);
          piece(y, c + per);
        }
      }
      // the W best of the lanes' keys, in order
      const u64 key = at < 0 ? 0 : key_of(best, at);
      sh.pool[tid] = key;
      __syncwarp();
      int ahead = 0;
#pragma unroll
      for (int i = 0; i < 32; ++i) {
        const u64 k = sh.pool[warp * 32 + i];
        ahead += k > key || (k == key && i < lane);
      }
      if (ahead < W) sh.list[warp][ahead] = key;
    } else if (mine && wm != -INFINITY) {  // again, in f64
#pragma unroll 1
      for (int64_t c = sub; c < row.pieces; c += per) {
#pragma unroll 1
        for (int i = 0; i < EPC / N; ++i) {
          float x[N];
          load_piece<BF>(p.logits, false, row.first + c * kPiece + (i * 32 + lane) * N, row.base, p.V, p.total, x);
#pragma unroll
          for (int k = 0; k < N; ++k) sum += exp((double)fmaxf(x[k], -INFINITY) - (double)wm);
        }
      }
    }
#pragma unroll
    for (int o = 16; o; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    if (lane == 0) sh.m[warp] = wm, sh.s[warp] = sum;
    tc::cluster_sync();

    // CTA r joins beams r, r + C, ..
    if (round == 0) {
      if (tid < joins * keys) {
        const int q = tid / keys, k = tid - q * keys, id = ((int)crank + q * (int)C) * per + k / W;
        sh.pool[tid] = ld_remote64(&sh.list[id % kSelWarps][k % W], id / kSelWarps);
      }
      if (tid < W_MAX) sh.more_count[tid] = 0;
      if (tid < W_MAX * W_MAX) (&sh.top[0][0])[tid] = 0;
    }
    for (int q = kSelWarps - 1 - warp; q < joins; q += kSelWarps) {  // the sums, by the last warps
      const int b = (int)crank + q * (int)C;
      constexpr int PARTS = 8 * kSelWarps / 32;  // of a lane: k, k + 32, ..
      float top = -INFINITY;
#pragma unroll
      for (int i = 0; i < PARTS; ++i) {
        const int k = lane + 32 * i, id = b * per + k;
        if (k < per) top = fmaxf(top, ld_remote_f(&sh.m[id % kSelWarps], id / kSelWarps));
      }
#pragma unroll
      for (int o = 16; o; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
      double ps = 0.;
#pragma unroll 1
      for (int i = 0; i < PARTS && lane + 32 * i < per; ++i) {
        const int id = b * per + lane + 32 * i;
        const double s2 = __longlong_as_double((long long)ld_remote64(&sh.s[id % kSelWarps], id / kSelWarps));
        const float m2 = ld_remote_f(&sh.m[id % kSelWarps], id / kSelWarps);
        if (m2 != -INFINITY) ps += s2 * exp((double)m2 - (double)top);
      }
#pragma unroll
      for (int o = 16; o; o >>= 1) ps += __shfl_xor_sync(0xffffffffu, ps, o);
      if (lane == 0) sh.lse[q] = (double)top + log(ps);
    }
    __syncthreads();
    if (round == 0) {
      // the W best of a beam's keys: each key counts those above it, four lanes a key
      for (int i0 = 0; i0 < 4 * joins * keys; i0 += kSelThreads) {
        const int i = i0 + tid, k = min(i >> 2, joins * keys - 1), q = k / keys;
        const u64 key = sh.pool[k], *pool = sh.pool + q * keys;
        int ahead = 0;
#pragma unroll 8
        for (int j = tid & 3; j < keys; j += 4) ahead += pool[j] > key;
        ahead += __shfl_xor_sync(0xffffffffu, ahead, 1);
        ahead += __shfl_xor_sync(0xffffffffu, ahead, 2);
        if (key && ahead < W && !(i & 3) && i < 4 * joins * keys) sh.top[q][ahead] = key;
      }
      __syncthreads();
      // other values of those lanes: the 16-byte loads of the lane that holds the j-th key, 32 at a time
      for (int e = warp; e < joins * W; e += kSelWarps) {
        const int q = e / W;
        const u64 key = sh.top[q][e - q * W], bar = sh.top[q][W - 1];
        if (!key) continue;
        const Row r = row_of<BF>(p, g * W + (int)crank + q * (int)C);
        const int64_t where = r.base - r.first + (uint32_t)~(uint32_t)key, piece = where / kPiece;
        const int sub2 = (int)(piece % per), lane2 = (int)(where - piece * kPiece) / N % 32;
        const int64_t loads = ((r.pieces - sub2 + per - 1) / per) * (EPC / N);
        u64 list = 0;  // lane j < W: the j-th best, for a beam with more than W of them in this lane
        for (int64_t v0 = 0; v0 < loads; v0 += 32) {
          const int64_t v = v0 + lane;
          const int64_t at = r.first + (sub2 + v / (EPC / N) * per) * kPiece + (v % (EPC / N) * 32 + lane2) * N;
          float z[N];
#pragma unroll
          for (int k = 0; k < N; ++k) z[k] = -INFINITY;
          if (v < loads)
            load_piece<BF>(p.logits, at >= r.base && at + N <= r.base + p.V, at, r.base, p.V, p.total, z);
          u64 k2[N];
          bool any = false;
#pragma unroll
          for (int k = 0; k < N; ++k) {
            const int64_t idx = at + k - r.base;
            k2[k] = v < loads && idx >= 0 && idx < p.V ? key_of(fmaxf(z[k], -INFINITY), idx) : 0;
            if (k2[k] == key || k2[k] <= bar) k2[k] = 0;
            any |= k2[k] != 0;
          }
          if (!__any_sync(0xffffffffu, any)) continue;
#pragma unroll
          for (int k = 0; k < N; ++k)
            for (uint32_t hit = __ballot_sync(0xffffffffu, k2[k] != 0); hit; hit &= hit - 1) {
              const u64 in = shfl64(k2[k], __ffs(hit) - 1);
              const int place = __popc(__ballot_sync(0xffffffffu, lane < W && list > in));
              const u64 up = __shfl_up_sync(0xffffffffu, list, 1);
              if (lane < W && lane >= place) list = lane == place ? in : up;
            }
        }
        if (lane < W && list) sh.more[q][atomicAdd(&sh.more_count[q], 1)] = list;
      }
    }
    __syncthreads();
    // the W best of both, as candidates, to every CTA
    const int per_beam = W + W * W;
    for (int i = tid; i < joins * per_beam; i += kSelThreads) {
      const int q = i / per_beam, k = i - q * per_beam, b = (int)crank + q * (int)C, n = sh.more_count[q];
      if (k >= W + n) continue;
      const float score = p.scores[g * W + b];
      const bool fin = p.eos >= 0 && p.finished[g * W + b], exists = k < p.V;
      double value = -INFINITY;
      int token = exists ? k : -1, place = k;
      if (!isfinite(score) || (!fin && !isfinite(sh.lse[q]))) {
        // no candidate is better than another: the lowest tokens
        if (k >= W) continue;
      } else if (fin) {
        // the end token alone, then the others from the lowest
        if (k >= W) continue;
        if (k == 0) value = score;
        if (exists) token = k == 0 ? p.eos : k - 1 + (k - 1 >= p.eos);
      } else {
        const u64 key = k < W ? sh.top[q][k] : sh.more[q][k - W];
        place = 0;
        for (int j = 0; j < W; ++j) place += sh.top[q][j] > key;
        for (int j = 0; j < n; ++j) place += sh.more[q][j] > key;
        if (!key) {  // fewer than W values: the places behind the last
          if (k < W && exists) continue;
          place = k;
          token = -1;
        } else {
          token = (int)~(uint32_t)key;
          value = (double)score + ((double)unordered((uint32_t)(key >> 32)) - sh.lse[q]);
        }
      }
      if (place >= W) continue;
      for (uint32_t c = 0; c < C; ++c) {
        st_remote64(&sh.cand[b][place], c, (u64)__double_as_longlong(value));
        st_remote32(&sh.token[b][place], c, (uint32_t)token);
        if (place == 0) st_remote32(&sh.done[b], c, fin ? 1u : 0u);
      }
    }
    if (tid <= W) sh.beam[tid] = -1;
    for (int i = tid; i < W * W; i += kSelThreads) sh.rank[i] = i % W;  // a survivor's place in its own list
    tc::cluster_sync();
    // plus those ahead of it in every other list (among equals the lower beam comes first)
    for (int i = tid; i < W * W * W; i += kSelThreads) {
      const int s = i / W, b2 = i - s * W, b = s / W, j = s - b * W;
      if (b2 == b || sh.token[b][j] < 0) continue;
      const double v = sh.cand[b][j];
      int n = 0;
#pragma unroll 8
      for (int k = 0; k < W; ++k) {
        const double v2 = sh.cand[b2][k];
        n += sh.token[b2][k] >= 0 && (v2 > v || (v2 == v && b2 < b));
      }
      if (n) atomicAdd(&sh.rank[s], n);
    }
    __syncthreads();
    for (int i = tid; i < W * W; i += kSelThreads) {
      const int b = i / W, j = i - b * W, rank = sh.rank[i];
      if (sh.token[b][j] < 0 || rank > W) continue;
      sh.best[rank] = sh.cand[b][j], sh.beam[rank] = b;
      if (rank < W) sh.pick[rank] = sh.token[b][j];
    }
    __syncthreads();
    bool close = false;
    if (round == 0 && tid < W) {
      const int b1 = sh.beam[tid], b2 = sh.beam[tid + 1];
      // finished beams' candidates and -inf are exact
      close = b1 >= 0 && b2 >= 0 && b1 != b2 && too_close(sh.best[tid], sh.best[tid + 1]);
    }
    // behind the last place another beam's candidates may stand after several of its own beam's
    if (round == 0)
      for (int i = tid; i < W * W; i += kSelThreads) {
        const int b = i / W, j = i - b * W;
        close |= sh.rank[i] >= W && sh.token[b][j] >= 0 && b != sh.beam[W - 1] &&
                 too_close(sh.best[W - 1], sh.cand[b][j]);
      }
    if (__syncthreads_or(close)) {
      tc::cluster_sync();  // every CTA has read the candidates before they are written again
      continue;
    }
    if (crank == 0 && tid < W) {
      const int64_t o = g * W + tid;
      const int b = sh.beam[tid], tok = sh.pick[tid];
      p.out_scores[o] = (float)sh.best[tid];
      p.out_parents[o] = b;
      p.out_tokens[o] = tok;
      if (p.eos >= 0) p.out_finished[o] = sh.done[b] || tok == p.eos;
    }
    return;
  }
}

struct ReorderParams {
  struct State {
    uint8_t* p;
    int64_t row_bytes, T, inner;
    int64_t units;      // pieces of `unit` bytes per row
    int64_t first;      // first block of the state
    int unit;
  };
  static constexpr int kStates = 48;
  State s[kStates];
  int count;
  const int *parents, *lengths;
  int W;
};

constexpr int kReThreads = 256;

template <typename U, int W>
__device__ __forceinline__ void reorder_piece(const ReorderParams::State& s, int64_t g, int64_t u, const int* src,
                                              const int64_t* live, int w) {
  if (u >= s.units) return;
  // entry of the time axis; -1: whole rows
  int64_t t = -1;
  if (s.T) {
    const int64_t at = u * (int64_t)sizeof(U);
    t = s.row_bytes <= UINT32_MAX ? (uint32_t)at / (uint32_t)s.inner % (uint32_t)s.T : at / s.inner % s.T;
  }
  uint8_t* row0 = s.p + g * w * s.row_bytes + u * (int64_t)sizeof(U);
  U v[W];
  // every read comes before the first write: this thread alone touches these bytes of the group's rows
#pragma unroll
  for (int j = 0; j < W; ++j)
    if (j < w && src[j] != j && (t < 0 || t < live[j])) v[j] = *(const U*)(row0 + src[j] * s.row_bytes);
#pragma unroll
  for (int j = 0; j < W; ++j)
    if (j < w && src[j] != j && (t < 0 || t < live[j])) *(U*)(row0 + j * s.row_bytes) = v[j];
}

template <int W>
__global__ void __launch_bounds__(kReThreads) reorder_kernel(const __grid_constant__ ReorderParams p) {
  pdl_prologue();
  __shared__ int src[W];
  __shared__ int64_t live[W];  // entries to take over
  int lo = 0, hi = p.count - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) / 2;
    if ((int64_t)blockIdx.x >= p.s[mid].first) lo = mid;
    else hi = mid - 1;
  }
  const ReorderParams::State& s = p.s[lo];
  const int64_t per_group = (s.units + kReThreads - 1) / kReThreads;
  const int64_t b = (int64_t)blockIdx.x - s.first, g = b / per_group, u = (b % per_group) * kReThreads + threadIdx.x;
  if (threadIdx.x < W) {
    const int j = threadIdx.x;
    int q = j < p.W ? p.parents[g * p.W + j] : j;
    if (q < 0 || q >= p.W) q = j;
    src[j] = q;
    live[j] = p.lengths && j < p.W ? (int64_t)p.lengths[g * p.W + q] : s.T;
  }
  __syncthreads();
  switch (s.unit) {
    case 16: reorder_piece<uint4, W>(s, g, u, src, live, p.W); break;
    case 8: reorder_piece<uint2, W>(s, g, u, src, live, p.W); break;
    case 4: reorder_piece<uint32_t, W>(s, g, u, src, live, p.W); break;
    case 2: reorder_piece<uint16_t, W>(s, g, u, src, live, p.W); break;
    default: reorder_piece<uint8_t, W>(s, g, u, src, live, p.W); break;
  }
}

}  // namespace

cudaError_t beam_select(const BeamSelectArgs& a, cudaStream_t stream) {
  if (a.G == 0) return cudaSuccess;
  SelectParams p = {a.logits, a.scores, a.finished, a.out_scores, a.out_parents, a.out_tokens, a.out_finished,
                    a.V, a.G * a.W * a.V, (int)a.W, (int)a.eos,
                    (float)((kBaseRoom - std::log2((double)a.V)) * std::log(2.))};
  // One CTA fits an SM: split while the CTAs stay one wave and a warp has a piece (32
  // groups of 8 beams over 50304 values: 1 CTA each 47 us, 2: 26, 4: 17, 8: 37).
  const int64_t pieces = a.W * ((a.V + kPiece - 1) / kPiece);
  int dev = 0, sms = 148, C = 1;
  if (cudaGetDevice(&dev) == cudaSuccess) cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
  while (C < 8 && a.G * 2 * C <= sms && pieces > C * kSelWarps) C *= 2;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(a.G * C));
  cfg.blockDim = dim3(kSelThreads);
  cfg.stream = stream;
  cudaLaunchAttribute at[2];
  pdl_attribute(&at[0]);
  at[1].id = cudaLaunchAttributeClusterDimension;
  at[1].val.clusterDim.x = (unsigned)C;
  at[1].val.clusterDim.y = at[1].val.clusterDim.z = 1;
  cfg.attrs = at;
  cfg.numAttrs = 2;
  launch_counter().fetch_add(1, std::memory_order_relaxed);
  return a.bf16 ? cudaLaunchKernelEx(&cfg, select_kernel<true>, p) : cudaLaunchKernelEx(&cfg, select_kernel<false>, p);
}

cudaError_t beam_reorder(const BeamState* states, int64_t count, const int* parents, const int* lengths, int64_t G,
                         int64_t W, cudaStream_t stream) {
  for (int64_t at = 0; at < count;) {
    ReorderParams p;
    p.count = 0;
    p.parents = parents;
    p.lengths = lengths;
    p.W = (int)W;
    int64_t blocks = 0;
    for (; at < count && p.count < ReorderParams::kStates; ++at) {
      const BeamState& s = states[at];
      if (s.row_bytes == 0) continue;
      int unit = 16;
      while (s.inner % unit) unit /= 2;
      const int64_t units = s.row_bytes / unit, more = G * ((units + kReThreads - 1) / kReThreads);
      if (more > INT32_MAX) return cudaErrorInvalidValue;
      if (blocks + more > INT32_MAX) break;
      p.s[p.count++] = {(uint8_t*)s.p, s.row_bytes, s.T, s.inner, units, blocks, unit};
      blocks += more;
    }
    if (p.count == 0) continue;
    const dim3 grid((unsigned)blocks), block(kReThreads);
    cudaError_t e = W <= 2   ? launch_pdl(reorder_kernel<2>, grid, block, 0, stream, p)
                    : W <= 4 ? launch_pdl(reorder_kernel<4>, grid, block, 0, stream, p)
                    : W <= 8 ? launch_pdl(reorder_kernel<8>, grid, block, 0, stream, p)
                             : launch_pdl(reorder_kernel<16>, grid, block, 0, stream, p);
    if (e != cudaSuccess) return e;
  }
  return cudaSuccess;
}

}  // namespace sb
