// Key/value cache rows: writing new tokens (kv_cache_write) and reading back
// the values a range of the cache stands for (kv_cache_read).
//
// A cache is [N, H, T, D]: slots, heads, capacity, head size.  An f32 or bf16
// cache holds the values (bf16: rounded to nearest even).  An int8 cache holds
// codes c in [-127, 127] and one f32 scale s per row (slot, head, position):
//   s = amax(|x|) / 127 rounded to f32,   c = x / s rounded to the nearest
//   integer, ties to even, in exact arithmetic,   value = c * s.
// One scale per row keeps a row's error below s / 2 whatever other rows hold,
// and attention can apply it to a score or a probability instead of a row.
// A NaN is written as 0 and an infinity as the largest finite f32, so that one
// bad value leaves the row's other codes usable.
#include <cuda_bf16.h>

#include <cfloat>

#include "kernels.h"
#include "pdl.h"

namespace sb {
namespace {

constexpr int kThreads = 256;
constexpr int EPL = 8;  // values per lane: one 16-byte load of bf16, two of f32, one 8-byte load of codes

template <typename T>
__device__ __forceinline__ void load8(const T* p, float* x);
template <>
__device__ __forceinline__ void load8<float>(const float* p, float* x) {
  const float4 a = *(const float4*)p, b = *(const float4*)(p + 4);
  x[0] = a.x, x[1] = a.y, x[2] = a.z, x[3] = a.w, x[4] = b.x, x[5] = b.y, x[6] = b.z, x[7] = b.w;
}
template <>
__device__ __forceinline__ void load8<__nv_bfloat16>(const __nv_bfloat16* p, float* x) {
  const uint4 a = *(const uint4*)p;
  const uint32_t w[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    x[2 * i] = __uint_as_float(w[i] << 16);
    x[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
  }
}
template <>
__device__ __forceinline__ void load8<int8_t>(const int8_t* p, float* x) {
  const uint2 a = *(const uint2*)p;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    x[i] = (float)(int8_t)(a.x >> (8 * i));
    x[4 + i] = (float)(int8_t)(a.y >> (8 * i));
  }
}

template <typename T>
__device__ __forceinline__ void store8(T* p, const float* x);
template <>
__device__ __forceinline__ void store8<float>(float* p, const float* x) {
  *(float4*)p = make_float4(x[0], x[1], x[2], x[3]);
  *(float4*)(p + 4) = make_float4(x[4], x[5], x[6], x[7]);
}
template <>
__device__ __forceinline__ void store8<__nv_bfloat16>(__nv_bfloat16* p, const float* x) {
  __nv_bfloat162 h[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) h[i] = __floats2bfloat162_rn(x[2 * i], x[2 * i + 1]);
  *(uint4*)p = *(uint4*)h;
}

// The integer nearest to x / s, ties to even, in exact arithmetic.  The f32
// quotient is within one step of it; the remainder x - q s is exact in one
// fma (a multiple of half an ulp of s, below 2^24 of them), so comparing it
// with s / 2 settles the last step.
__device__ __forceinline__ int nearest_code(float x, float s) {
  float q = rintf(__fdiv_rn(x, s));
  const float r = 2.f * fmaf(-q, s, x);
  if (r > s || (r == s && ((int)q & 1))) q += 1.f;
  if (r < -s || (r == -s && ((int)q & 1))) q -= 1.f;
  return (int)fminf(fmaxf(q, -127.f), 127.f);
}

struct WriteParams {
  const void* src[2];  // k, v [N, S, H, D]
  void* dst[2];        // the caches
  float* scale[2];
  const int* pos;
  int64_t rows;  // N * S * H of one of the two
  int64_t T;
  int S, H, D;
};

// A group of LPR lanes carries one row: with 8 values a lane the row's largest
// magnitude is a butterfly of log2(LPR) shuffles.
template <typename TI, typename TC, int LPR>
__global__ void __launch_bounds__(kThreads) write_kernel(const WriteParams p) {
  pdl_prologue();
  const int lane = threadIdx.x % LPR;
  const int64_t r2 = (int64_t)blockIdx.x * (kThreads / LPR) + threadIdx.x / LPR;
  const int which = r2 >= p.rows;
  const int64_t r = r2 - (which ? p.rows : 0);
  const int64_t h = r % p.H, ns = r / p.H, s = ns % p.S, n = ns / p.S;
  const bool row = r < p.rows;
  const int64_t first = row ? p.pos[n] : -1, t = first + s;
  const bool in = first >= 0 && t < p.T && lane * EPL < p.D;
  float x[EPL];
#pragma unroll
  for (int i = 0; i < EPL; ++i) x[i] = 0.f;
  if (in) load8((const TI*)p.src[which] + r * p.D + lane * EPL, x);
  const int64_t at = (n * p.H + h) * p.T + t;
  if constexpr (sizeof(TC) == 1) {
    float m = 0.f;
#pragma unroll
    for (int i = 0; i < EPL; ++i) {
      x[i] = x[i] != x[i] ? 0.f : fminf(fmaxf(x[i], -FLT_MAX), FLT_MAX);
      m = fmaxf(m, fabsf(x[i]));
    }
#pragma unroll
    for (int o = LPR / 2; o; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
    const float sc = __fdiv_rn(m, 127.f);
    if (in) {
      uint32_t w[2] = {0, 0};
      if (sc > 0.f) {
#pragma unroll
        for (int i = 0; i < EPL; ++i) w[i / 4] |= (uint32_t)(nearest_code(x[i], sc) & 255) << (8 * (i % 4));
      }
      *(uint2*)((int8_t*)p.dst[which] + at * p.D + lane * EPL) = make_uint2(w[0], w[1]);
      if (lane == 0) p.scale[which][at] = sc;
    }
  } else {
    if (in) store8((TC*)p.dst[which] + at * p.D + lane * EPL, x);
  }
}

struct ReadParams {
  const void* src[2];
  const float* scale[2];
  void* dst[2];  // [N, H, S, D]
  const int *starts, *counts;
  int64_t units;  // 8-value pieces of one of the two outputs
  int64_t T, S;
  int H, D;
};

template <typename TC, typename TO>
__global__ void __launch_bounds__(kThreads) read_kernel(const ReadParams p) {
  pdl_prologue();
  const int64_t u2 = (int64_t)blockIdx.x * kThreads + threadIdx.x;
  const int which = u2 >= p.units;
  const int64_t u = u2 - (which ? p.units : 0);
  if (u >= p.units) return;
  const int per = p.D / EPL;
  const int64_t row = u / per, i = row % p.S, nh = row / p.S, n = nh / p.H;
  const int64_t t = (p.starts ? (int64_t)p.starts[n] : 0) + i;
  if (t < 0 || t >= p.T || (p.counts && i >= p.counts[n])) return;
  const int64_t at = nh * p.T + t;
  const int d = (int)(u % per) * EPL;
  float x[EPL];
  load8((const TC*)p.src[which] + at * p.D + d, x);
  if constexpr (sizeof(TC) == 1) {
    const float s = p.scale[which][at];
#pragma unroll
    for (int j = 0; j < EPL; ++j) x[j] *= s;
  }
  store8((TO*)p.dst[which] + row * p.D + d, x);
}

template <typename TI, typename TC, int LPR>
cudaError_t launch_write(const WriteParams& p, cudaStream_t stream) {
  const int64_t per = kThreads / LPR, blocks = (2 * p.rows + per - 1) / per;
  if (blocks > INT32_MAX) return cudaErrorInvalidValue;
  return launch_pdl(write_kernel<TI, TC, LPR>, dim3((unsigned)blocks), dim3(kThreads), 0, stream, p);
}

template <typename TI, typename TC>
cudaError_t write_rows(const WriteParams& p, cudaStream_t stream) {
  if (p.D <= 16) return launch_write<TI, TC, 2>(p, stream);
  if (p.D <= 32) return launch_write<TI, TC, 4>(p, stream);
  if (p.D <= 64) return launch_write<TI, TC, 8>(p, stream);
  if (p.D <= 128) return launch_write<TI, TC, 16>(p, stream);
  return launch_write<TI, TC, 32>(p, stream);
}

template <typename TC, typename TO>
cudaError_t read_rows(const ReadParams& p, cudaStream_t stream) {
  const int64_t blocks = (2 * p.units + kThreads - 1) / kThreads;
  if (blocks > INT32_MAX) return cudaErrorInvalidValue;
  return launch_pdl(read_kernel<TC, TO>, dim3((unsigned)blocks), dim3(kThreads), 0, stream, p);
}

}  // namespace

cudaError_t kv_cache_write(const KvCacheView& c, const int* positions, const void* k, const void* v, bool in_bf16,
                           int64_t S, cudaStream_t stream) {
  WriteParams p = {{k, v}, {c.k, c.v}, {c.k_scale, c.v_scale}, positions, c.N * S * c.H, c.T, (int)S, (int)c.H,
                   (int)c.D};
  using bf = __nv_bfloat16;
  switch (c.type) {
    case KvType::F32: return in_bf16 ? write_rows<bf, float>(p, stream) : write_rows<float, float>(p, stream);
    case KvType::BF16: return in_bf16 ? write_rows<bf, bf>(p, stream) : write_rows<float, bf>(p, stream);
    case KvType::I8: return in_bf16 ? write_rows<bf, int8_t>(p, stream) : write_rows<float, int8_t>(p, stream);
  }
  return cudaErrorInvalidValue;
}

cudaError_t kv_cache_read(const KvCacheView& c, const int* starts, const int* counts, void* k_out, void* v_out,
                          bool out_bf16, int64_t S, cudaStream_t stream) {
  ReadParams p = {{c.k, c.v}, {c.k_scale, c.v_scale}, {k_out, v_out}, starts, counts, c.N * c.H * S * (c.D / EPL), c.T,
                  S, (int)c.H, (int)c.D};
  using bf = __nv_bfloat16;
  switch (c.type) {
    case KvType::F32: return out_bf16 ? read_rows<float, bf>(p, stream) : read_rows<float, float>(p, stream);
    case KvType::BF16: return out_bf16 ? read_rows<bf, bf>(p, stream) : read_rows<bf, float>(p, stream);
    case KvType::I8: return out_bf16 ? read_rows<int8_t, bf>(p, stream) : read_rows<int8_t, float>(p, stream);
  }
  return cudaErrorInvalidValue;
}

}  // namespace sb
