// Beam search: the selection of the W best continuations of each group of W
// beams (beam_select) and the rearrangement of per-beam state to follow it
// (beam_reorder).
//
//   cand(w, v) = score_w + (z_wv - lse_w),  lse_w = log sum_v exp z_wv
//   selected: the W largest of the W x V candidates, by (value, then lowest
//   w V + v).
//
// Reading the logits once bounds the selection.  A cluster of C CTAs carries a
// group; each warp streams pieces of one beam's row and keeps in its lanes the
// W best of what it has seen as 64-bit keys (order-preserving image of the
// logit above the complemented index: unique, so equal logits order by index
// and every step has one answer).  The list starts as the W best of the lanes'
// best keys in the first piece; after that few values pass the best W-th key
// that any warp of the CTA has for the beam, and they are inserted one by one
// (a lane offers its next value only if its second largest passes too).  After
// a cluster barrier CTA r joins the lists
// of beams r, r + C, .. and sends them to every CTA; after a second one each CTA
// orders the W x W survivors.  Lists cross CTAs through distributed shared
// memory, so there is no workspace, no atomic and no second launch.
//
// Within a beam the order is the logits' own.  Between beams it needs lse.  The
// first round sums f32 exponentials, off by less than kFastError; if two
// neighbours of the result from different beams are closer than twice that (or
// tie), the group's sums are taken again in f64, whose exponentials would
// otherwise bound the kernel.  So the order is that of f64 sums in every case.
#include <cuda_bf16.h>

#include <cmath>

#include "kernels.h"
#include "pdl.h"
#include "tc_common.h"

namespace sb {
namespace {

constexpr int kSelWarps = 16, kSelThreads = kSelWarps * 32;
// Bound on the error of an lse from f32 exponentials of V <= 2^31 values.  A
// term 2^-t has a relative error of at most 2^-22 (ex2) + 2^-23.4 t (its
// argument, two roundings), and terms with t > 32 + log2 of the sum of the
// others' number are below it; the mean t of the sum's weight is at most
// log2(V) < 32; 16 terms are added in f32 (at most 4 additions each), the rest
// in f64: 2^-22 + 32 * 2^-23.4 + 4 * 2^-24 < 4e-6.
constexpr double kFastError = 4e-6;
constexpr int EPC = 16;              // values per lane and piece
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
};

// Order-preserving image of an f32 that is not NaN.
__device__ __forceinline__ uint32_t ordered(float x) {
  const uint32_t u = __float_as_uint(x);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float unordered(uint32_t u) {
  return __uint_as_float(u & 0x80000000u ? u & 0x7fffffffu : ~u);
}
__device__ __forceinline__ u64 shfl64(u64 x, int src) { return __shfl_sync(0xffffffffu, x, src); }

// A warp's list: lane j < W holds the j-th largest key, 0 where there is none
// (every real key is above 0).
__device__ __forceinline__ void insert(u64& list, u64 key, int lane, int W) {
  const int rank = __popc(__ballot_sync(0xffffffffu, lane < W && list > key));
  const u64 up = __shfl_up_sync(0xffffffffu, list, 1);
  if (lane < W && lane >= rank) list = lane == rank ? key : up;
}

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
// belong to the row [base, base + V), -inf elsewhere and for NaN.  `inside`: all
// of them do.  The buffer's last values are loaded one by one where the 16
// bytes would pass its end.
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
#pragma unroll
  for (int i = 0; i < N; ++i) x[i] = fmaxf(x[i], -INFINITY);  // the number of the two
}

struct SelectShared {
  u64 list[kSelWarps][W_MAX];
  u64 sort[kSelWarps][32];  // a warp's first list
  u64 bar[W_MAX];           // per beam: a key that W keys of the CTA reach
  double s[kSelWarps];
  float m[kSelWarps];
  // the candidates of every beam, best first (each CTA has them all)
  double cand[W_MAX][W_MAX];
  int token[W_MAX][W_MAX];
  int done[W_MAX];
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

template <bool BF>
__global__ void __launch_bounds__(kSelThreads, 2) select_kernel(const SelectParams p) {
  pdl_prologue();
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
  const bool mine = beam < W && !(p.eos >= 0 && p.finished[g * W + beam]);
  const int64_t base = (g * W + (mine ? beam : 0)) * p.V;
  const int64_t first = base - base % N;  // 16-byte boundary at or before the row
  const int64_t pieces = (base + p.V - first + kPiece - 1) / kPiece;
  u64 list = 0;
  float m = -INFINITY;
  if (tid < W_MAX) sh.bar[tid] = 0;
  __syncthreads();

  for (int round = 0;; ++round) {
    double sum = 0.;
    if (mine && round == 0) {
      for (int64_t c = sub; c < pieces; c += per) {
        const int64_t at0 = first + c * kPiece + lane * N;
        const bool inside = first + c * kPiece >= base && first + (c + 1) * kPiece <= base + p.V;
        float x[EPC];
#pragma unroll
        for (int i = 0; i < EPC / N; ++i)
          load_piece<BF>(p.logits, inside, at0 + i * 32 * N, base, p.V, p.total, x + i * N);
        // the lane's two largest values
        float mx = x[0], m2 = -INFINITY;
#pragma unroll
        for (int i = 1; i < EPC; ++i) {
          m2 = fmaxf(m2, fminf(mx, x[i]));
          mx = fmaxf(mx, x[i]);
        }
        float wm = mx;
#pragma unroll
        for (int o = 16; o; o >>= 1) wm = fmaxf(wm, __shfl_xor_sync(0xffffffffu, wm, o));
        const float mn = fmaxf(m, wm);
        if (mn != -INFINITY) {
          if (mn > m) sum *= (double)exp2f((m - mn) * kLog2e);
          m = mn;
          float e[8];
#pragma unroll
          for (int i = 0; i < EPC; ++i) {
            const float y = tc::ex2((x[i] - m) * kLog2e);
            e[i % 8] = i < 8 ? y : e[i % 8] + y;
          }
#pragma unroll
          for (int w = 4; w; w >>= 1)
#pragma unroll
            for (int i = 0; i < w; ++i) e[i] += e[i + w];
          sum += (double)e[0];  // per lane
        }
        // The best that any warp of this CTA has W of for the beam bars the rest.
        u64 bar = shfl64(list, W - 1);
        const u64 shared_bar = shfl64(*(volatile u64*)&sh.bar[beam], 0);
        if (shared_bar > bar) bar = shared_bar;
        float barf = bar ? unordered((uint32_t)(bar >> 32)) : -INFINITY;
        if (!__any_sync(0xffffffffu, mx >= barf)) continue;
        // the lane's best key: its largest value at the lowest index; then the next ones
        u64 last = ~0ull;
        auto next = [&]() {
          u64 best = 0;
#pragma unroll
          for (int i = 0; i < EPC; ++i) {
            const int64_t idx = at0 + (i / N) * 32 * N + i % N - base;
            if (idx < 0 || idx >= p.V || x[i] < barf) continue;
            const u64 key = (u64)ordered(x[i]) << 32 | (uint32_t)~(uint32_t)idx;
            if (key < last && key > best) best = key;
          }
          last = best;
          return best;
        };
        u64 key = 0;
        if (mx >= barf) key = next();
        if (!shfl64(list, 0)) {
          // the first piece: the list starts as the W best of the lanes' best keys
          u64* mine_keys = sh.sort[warp];
          mine_keys[lane] = key;
          __syncwarp();
          int ahead = 0;
#pragma unroll
          for (int i = 0; i < 32; ++i) ahead += mine_keys[i] > key || (mine_keys[i] == key && i < lane);
          __syncwarp();
          mine_keys[ahead] = key;
          __syncwarp();
          list = lane < W ? mine_keys[lane] : 0;
          if (shfl64(list, W - 1) > bar) bar = shfl64(list, W - 1);
          barf = bar ? unordered((uint32_t)(bar >> 32)) : -INFINITY;
          if (ahead < W) key = m2 >= barf ? next() : 0;  // that one is in
        }
        // keys that pass, one by one; a lane whose key went in offers its next
        for (uint32_t hit; (hit = __ballot_sync(0xffffffffu, key > bar)) != 0;) {
          const int src = __ffs(hit) - 1;
          insert(list, shfl64(key, src), lane, W);
          const u64 b2 = shfl64(list, W - 1);
          if (b2 > bar) bar = b2, barf = unordered((uint32_t)(bar >> 32));
          if (lane == src) key = m2 >= barf ? next() : 0;
        }
        if (lane == 0 && bar > shared_bar) atomicMax(&sh.bar[beam], bar);
      }
      if (lane < W_MAX) sh.list[warp][lane] = lane < W ? list : 0;
    } else if (mine) {  // again, in f64; m is the warp's maximum
      for (int64_t c = sub; c < pieces; c += per) {
        const int64_t at0 = first + c * kPiece + lane * N;
#pragma unroll 1
        for (int i = 0; i < EPC / N; ++i) {
          float x[N];
          load_piece<BF>(p.logits, false, at0 + i * 32 * N, base, p.V, p.total, x);
          if (m != -INFINITY)
#pragma unroll
            for (int k = 0; k < N; ++k) sum += exp((double)x[k] - (double)m);
        }
      }
    } else if (round == 0 && lane < W_MAX) {
      sh.list[warp][lane] = 0;
    }
#pragma unroll
    for (int o = 16; o; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    if (lane == 0) sh.m[warp] = m, sh.s[warp] = sum;
    tc::cluster_sync();

    // CTA r joins beams r, r + C, ..: one warp each
    for (int b = (int)crank + (int)C * warp; b < W; b += (int)C * kSelWarps) {
      u64 best = 0;
      float pm = -INFINITY;  // lane k (and k + 32, ..): the parts of the sum
      double ps = 0.;
      for (int k0 = 0; k0 < per; k0 += 8) {
        u64 part[8];
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          const int id = b * per + k0 + k;
          part[k] = k0 + k < per && lane < W ? ld_remote64(&sh.list[id % kSelWarps][lane], id / kSelWarps) : 0;
        }
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          if (k0 + k == 0) {
            best = part[k];
            continue;
          }
          for (int j = 0; j < W; ++j) {  // sorted: stop at the first that does not get in
            const u64 key = shfl64(part[k], j);
            if (key <= shfl64(best, W - 1)) break;
            insert(best, key, lane, W);
          }
        }
      }
      for (int k = lane; k < per; k += 32) {
        const int id = b * per + k;
        const float m2 = ld_remote_f(&sh.m[id % kSelWarps], id / kSelWarps);
        const double s2 = __longlong_as_double((long long)ld_remote64(&sh.s[id % kSelWarps], id / kSelWarps));
        const float mx = fmaxf(pm, m2);
        if (mx != -INFINITY) {
          ps = ps * exp((double)pm - (double)mx) + s2 * exp((double)m2 - (double)mx);
          pm = mx;
        }
      }
      float top = pm;
#pragma unroll
      for (int o = 16; o; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
      ps = pm == -INFINITY ? 0. : ps * exp((double)pm - (double)top);
#pragma unroll
      for (int o = 16; o; o >>= 1) ps += __shfl_xor_sync(0xffffffffu, ps, o);
      const float score = p.scores[g * W + b];
      const bool fin = p.eos >= 0 && p.finished[g * W + b];
      const double lse = (double)top + log(ps);
      const int have = (int)min((int64_t)W, p.V);
      double value = -INFINITY;
      int token = lane;
      if (isfinite(score) && fin) {
        // the end token alone, then the others from the lowest
        value = lane == 0 ? (double)score : -INFINITY;
        token = lane == 0 ? p.eos : lane - 1 + (lane - 1 >= p.eos);
      } else if (isfinite(score) && isfinite(lse)) {
        token = (int)~(uint32_t)best;
        value = (double)score + ((double)unordered((uint32_t)(best >> 32)) - lse);
      }
      if (lane < W) {
        if (lane >= have) value = -INFINITY, token = -1;  // no such candidate
        for (uint32_t c = 0; c < C; ++c) {
          st_remote64(&sh.cand[b][lane], c, (u64)__double_as_longlong(value));
          st_remote32(&sh.token[b][lane], c, (uint32_t)token);
          if (lane == 0) st_remote32(&sh.done[b], c, fin ? 1u : 0u);
        }
      }
    }
    if (tid <= W) sh.beam[tid] = -1;
    tc::cluster_sync();
    // rank of each survivor: its place in its own list, and in every other by
    // bisection (among equals the lower beam comes first)
    for (int i = tid; i < W * W; i += kSelThreads) {
      const int b = i / W, j = i % W, tok = sh.token[b][j];
      if (tok < 0) continue;
      const double v = sh.cand[b][j];
      int rank = j;
      for (int b2 = 0; b2 < W; ++b2) {
        if (b2 == b) continue;
        int n = 0;
#pragma unroll
        for (int step = W_MAX; step; step >>= 1)
          if (n + step <= W && sh.token[b2][n + step - 1] >= 0 &&
              (sh.cand[b2][n + step - 1] > v || (sh.cand[b2][n + step - 1] == v && b2 < b)))
            n += step;
        rank += n;
      }
      if (rank <= W) sh.best[rank] = v, sh.beam[rank] = b;
      if (rank < W) sh.pick[rank] = tok;
    }
    __syncthreads();
    bool close = false;
    if (round == 0 && tid < W) {
      const int b1 = sh.beam[tid], b2 = sh.beam[tid + 1];
      // finished beams' candidates and -inf are exact
      close = b1 >= 0 && b2 >= 0 && b1 != b2 && sh.best[tid + 1] != -INFINITY &&
              sh.best[tid] - sh.best[tid + 1] < 2 * kFastError + 1e-15 * fabs(sh.best[tid]);
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
                    a.V, a.G * a.W * a.V, (int)a.W, (int)a.eos};
  // split while the CTAs (two per SM) stay one wave and every warp has two pieces
  const int64_t pieces = a.W * ((a.V + kPiece - 1) / kPiece);
  int dev = 0, sms = 148, C = 1;
  if (cudaGetDevice(&dev) == cudaSuccess) cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
  while (C < 8 && a.G * 2 * C <= 2 * sms && pieces > 2 * C * kSelWarps) C *= 2;
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
