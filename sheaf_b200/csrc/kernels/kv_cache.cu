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
// bad value leaves the row's other codes usable (the scale of such a row rounds up,
// so that f32 reads the code 127 back as an infinity).
//
// Bytes bound both.  8 x 1024 tokens of 12 heads of 64, f32 to int8, and the read
// back to f32 (128 MB): 27.4 us, 4.7 TB/s (much of it stays in L2 between the two);
// a ragged read of 24 slots of 4K positions, int8 to f32 (430 MB): 72 us, 6.0
// TB/s, 0.92 of a copy; one token of one sequence: 4 us, the latency of a launch.
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
__device__ __forceinline__ void load8<float>(const float* p, float* x) {  // p: 32-byte aligned
  asm volatile("ld.global.L1::no_allocate.v8.f32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
               : "=f"(x[0]), "=f"(x[1]), "=f"(x[2]), "=f"(x[3]), "=f"(x[4]), "=f"(x[5]), "=f"(x[6]), "=f"(x[7])
               : "l"(p));
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

template <typename T>
__device__ __forceinline__ void store8(T* p, const float* x);
template <>
__device__ __forceinline__ void store8<float>(float* p, const float* x) {  // p: 32-byte aligned
  asm volatile("st.global.v8.f32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(p), "f"(x[0]), "f"(x[1]), "f"(x[2]),
               "f"(x[3]), "f"(x[4]), "f"(x[5]), "f"(x[6]), "f"(x[7])
               : "memory");
}
template <>
__device__ __forceinline__ void store8<__nv_bfloat16>(__nv_bfloat16* p, const float* x) {
  __nv_bfloat162 h[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) h[i] = __floats2bfloat162_rn(x[2 * i], x[2 * i + 1]);
  *(uint4*)p = *(uint4*)h;
}

// The integer nearest to x / s, ties to even, in exact arithmetic, |x / s| <= 190.
// The f32 quotient is within one step of it; the remainder x - q s is exact in
// one fma (a multiple of half an ulp of s, below 2^24 of them), so comparing it
// with s / 2 settles the last step.
__device__ __forceinline__ int nearest_code(float x, float s) {
  float q = rintf(__fdiv_rn(x, s));
  const float r = 2.f * fmaf(-q, s, x);
  if (r > s || (r == s && ((int)q & 1))) q += 1.f;
  if (r < -s || (r == -s && ((int)q & 1))) q -= 1.f;
  return (int)fminf(fmaxf(q, -127.f), 127.f);
}

// Codes of 8 values (finite, at most 127 (1 + 2^-24) s) as 8 bytes.  The common
// way has no division: x (1 / s) is within 2^-15 of x / s, adding 1.5 2^23
// rounds it to an integer q and leaves q in the sum's low byte, and where the
// remainder is below s / 2 that q is the nearest.  Any other value of a lane
// sends its 8 through nearest_code; so does a scale whose reciprocal or half
// is not normal.
__device__ __forceinline__ uint2 codes8(const float* x, float s) {
  const float inv = __frcp_rn(s), half = 0.5f * s;
  bool sure = s > 1e-36f && s < 1e36f;
  uint32_t b[EPL];
#pragma unroll
  for (int i = 0; i < EPL; ++i) {
    const float y = fmaf(x[i], inv, 12582912.f);
    b[i] = __float_as_uint(y);
    sure = sure && fabsf(fmaf(-(y - 12582912.f), s, x[i])) < half;
  }
  if (!sure) {
#pragma unroll
    for (int i = 0; i < EPL; ++i) b[i] = s > 0.f ? (uint32_t)nearest_code(x[i], s) : 0u;
  }
  uint2 w;
  w.x = __byte_perm(__byte_perm(b[0], b[1], 0x0040), __byte_perm(b[2], b[3], 0x0040), 0x5410);
  w.y = __byte_perm(__byte_perm(b[4], b[5], 0x0040), __byte_perm(b[6], b[7], 0x0040), 0x5410);
  return w;
}

struct WriteParams {
  const void* src[2];  // k, v [N, S, H, D]
  void* dst[2];        // the caches
  float* scale[2];
  const int* pos;
  int64_t T;
  unsigned rows;    // S * H: a slot's rows of one of the two
  unsigned blocks;  // per slot
  int H, D;
};

// A group of LPR lanes carries one row: with 8 values a lane the row's largest
// magnitude is a butterfly of log2(LPR) shuffles.  The groups of a block take rows
// of one slot's keys, then values.  (Four rows per group, their loads first, were no
// faster for a prompt, 13.1 us against 13.0, and slower for less: 8 x 64 tokens 3.3
// and 2.4.)
template <typename TI, typename TC, int LPR>
__global__ void __launch_bounds__(kThreads) write_kernel(const WriteParams p) {
  pdl_prologue();
  const int lane = threadIdx.x % LPR;
  const unsigned n = blockIdx.x / p.blocks;
  unsigned r = blockIdx.x % p.blocks * (kThreads / LPR) + threadIdx.x / LPR;
  const unsigned which = r >= p.rows;
  if (which) r -= p.rows;
  const unsigned s = r / p.H, h = r - s * p.H;
  const int64_t first = p.pos[n], t = first + s;
  const bool in = r < p.rows && first >= 0 && t < p.T && lane * EPL < p.D;
  const int64_t at = ((int64_t)n * p.H + h) * p.T + t;
  float x[EPL];
#pragma unroll
  for (int i = 0; i < EPL; ++i) x[i] = 0.f;
  if (in) load8((const TI*)(which ? p.src[1] : p.src[0]) + ((int64_t)n * p.rows + r) * p.D + lane * EPL, x);
  if constexpr (sizeof(TC) == 1) {
    float m = 0.f, odd = 0.f;  // odd: NaN unless all values are finite
#pragma unroll
    for (int i = 0; i < EPL; ++i) {
      odd = fmaf(x[i], 0.f, odd);
      m = fmaxf(m, fabsf(x[i]));
    }
    if (odd != 0.f) {
      m = 0.f;
#pragma unroll
      for (int i = 0; i < EPL; ++i) {
        x[i] = x[i] != x[i] ? 0.f : fminf(fmaxf(x[i], -FLT_MAX), FLT_MAX);
        m = fmaxf(m, fabsf(x[i]));
      }
    }
#pragma unroll
    for (int o = LPR / 2; o; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
    const float sc = __fdiv_rn(m, 127.f);
    if (in) {
      *(uint2*)((int8_t*)(which ? p.dst[1] : p.dst[0]) + at * p.D + lane * EPL) = codes8(x, sc);
      if (lane == 0) (which ? p.scale[1] : p.scale[0])[at] = sc;
    }
  } else {
    if (in) store8((TC*)(which ? p.dst[1] : p.dst[0]) + at * p.D + lane * EPL, x);
  }
}

struct ReadParams {
  const void* src[2];
  const float* scale[2];
  void* dst[2];  // [N, H, S, D]
  const int *starts, *counts;
  int64_t T, S;
  unsigned blocks;  // per (slot, head) of one of the two
  int H, D;
};

constexpr int kReadUnits = 4;  // 16-byte pieces of the cache per thread

// For one (slot, head) both sides are contiguous: rows i of the output are rows
// starts[n] + i of the cache, so a block copies a range of pieces and clips it to
// the rows that exist and are counted.  A thread's loads all come first: they
// are what is under way while the block waits.
template <typename TC, typename TO>
__global__ void __launch_bounds__(kThreads) read_kernel(const ReadParams p) {
  pdl_prologue();
  constexpr int PV = 16 / sizeof(TC);  // values of a piece
  const unsigned b = blockIdx.x % p.blocks, item = blockIdx.x / p.blocks, which = item & 1, nh = item >> 1;
  const unsigned n = nh / p.H;
  const int64_t start = p.starts ? p.starts[n] : 0;
  const int64_t lo = max((int64_t)0, -start);
  int64_t hi = min(p.S, p.T - start);
  if (p.counts) hi = min(hi, (int64_t)p.counts[n]);
  const int per = p.D / PV;
  const int64_t u0 = (int64_t)b * (kThreads * kReadUnits) + threadIdx.x, u_lo = lo * per, u_hi = hi * per;
  const TC* src = (const TC*)(which ? p.src[1] : p.src[0]) + ((int64_t)nh * p.T + start) * p.D;
  TO* dst = (TO*)(which ? p.dst[1] : p.dst[0]) + (int64_t)nh * p.S * p.D;
  const float* scale = sizeof(TC) == 1 ? (which ? p.scale[1] : p.scale[0]) + (int64_t)nh * p.T + start : nullptr;
  uint4 raw[kReadUnits];
  float s[kReadUnits];
#pragma unroll
  for (int k = 0; k < kReadUnits; ++k) {
    const int64_t u = u0 + k * kThreads;
    s[k] = 1.f;
    if (u >= u_lo && u < u_hi) {
      asm volatile("ld.global.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];"
                   : "=r"(raw[k].x), "=r"(raw[k].y), "=r"(raw[k].z), "=r"(raw[k].w)
                   : "l"(src + u * PV));
      if constexpr (sizeof(TC) == 1)
        s[k] = scale[u <= UINT32_MAX ? (int64_t)((uint32_t)u / (uint32_t)per) : u / per];
    }
  }
#pragma unroll
  for (int k = 0; k < kReadUnits; ++k) {
    const int64_t u = u0 + k * kThreads;
    if (u < u_lo || u >= u_hi) continue;
    const uint32_t w[4] = {raw[k].x, raw[k].y, raw[k].z, raw[k].w};
    float x[PV];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (sizeof(TC) == 1) {
        // byte c ^ 0x80 = c + 128 under 2^23, less 2^23 + 128: no conversion instruction
        const uint32_t y = w[i] ^ 0x80808080u;
#pragma unroll
        for (int j = 0; j < 4; ++j)
          x[4 * i + j] = (__uint_as_float(__byte_perm(y, 0x4b000000u, 0x7440 + j)) - 8388736.f) * s[k];
      } else if constexpr (sizeof(TC) == 2) {
        x[2 * i] = __uint_as_float(w[i] << 16);
        x[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
      } else {
        x[i] = __uint_as_float(w[i]);
      }
    }
    TO* to = dst + u * PV;
    if constexpr (PV >= 8) {
#pragma unroll
      for (int i = 0; i < PV; i += 8) store8(to + i, x + i);
    } else if constexpr (sizeof(TO) == 4) {
      *(uint4*)to = raw[k];
    } else {
      __nv_bfloat162 h[2] = {__floats2bfloat162_rn(x[0], x[1]), __floats2bfloat162_rn(x[2], x[3])};
      *(uint2*)to = *(uint2*)h;
    }
  }
}

template <typename TI, typename TC, int LPR>
cudaError_t launch_write(WriteParams p, int64_t N, cudaStream_t stream) {
  constexpr int64_t per = kThreads / LPR;
  const int64_t blocks = (2 * (int64_t)p.rows + per - 1) / per;
  if (blocks * N > INT32_MAX) return cudaErrorInvalidValue;
  p.blocks = (unsigned)blocks;
  return launch_pdl(write_kernel<TI, TC, LPR>, dim3((unsigned)(blocks * N)), dim3(kThreads), 0, stream, p);
}

template <typename TI, typename TC>
cudaError_t write_rows(const WriteParams& p, int64_t N, cudaStream_t stream) {
  if (p.D <= 16) return launch_write<TI, TC, 2>(p, N, stream);
  if (p.D <= 32) return launch_write<TI, TC, 4>(p, N, stream);
  if (p.D <= 64) return launch_write<TI, TC, 8>(p, N, stream);
  if (p.D <= 128) return launch_write<TI, TC, 16>(p, N, stream);
  return launch_write<TI, TC, 32>(p, N, stream);
}

template <typename TC, typename TO>
cudaError_t read_rows(ReadParams p, int64_t N, cudaStream_t stream) {
  constexpr int64_t per = kThreads * kReadUnits;
  const int64_t units = p.S * (p.D * (int64_t)sizeof(TC) / 16), blocks = (units + per - 1) / per;
  if (blocks * 2 * N * p.H > INT32_MAX) return cudaErrorInvalidValue;
  p.blocks = (unsigned)blocks;
  return launch_pdl(read_kernel<TC, TO>, dim3((unsigned)(blocks * 2 * N * p.H)), dim3(kThreads), 0, stream, p);
}

}  // namespace

cudaError_t kv_cache_write(const KvCacheView& c, const int* positions, const void* k, const void* v, bool in_bf16,
                           int64_t S, cudaStream_t stream) {
  if (S * c.H > INT32_MAX) return cudaErrorInvalidValue;
  const WriteParams p = {{k, v}, {c.k, c.v}, {c.k_scale, c.v_scale}, positions, c.T, (unsigned)(S * c.H), 0,
                         (int)c.H, (int)c.D};
  using bf = __nv_bfloat16;
  switch (c.type) {
    case KvType::F32: return in_bf16 ? write_rows<bf, float>(p, c.N, stream) : write_rows<float, float>(p, c.N, stream);
    case KvType::BF16: return in_bf16 ? write_rows<bf, bf>(p, c.N, stream) : write_rows<float, bf>(p, c.N, stream);
    case KvType::I8: return in_bf16 ? write_rows<bf, int8_t>(p, c.N, stream) : write_rows<float, int8_t>(p, c.N, stream);
  }
  return cudaErrorInvalidValue;
}

cudaError_t kv_cache_read(const KvCacheView& c, const int* starts, const int* counts, void* k_out, void* v_out,
                          bool out_bf16, int64_t S, cudaStream_t stream) {
  const ReadParams p = {{c.k, c.v}, {c.k_scale, c.v_scale}, {k_out, v_out}, starts, counts, c.T, S, 0, (int)c.H,
                        (int)c.D};
  using bf = __nv_bfloat16;
  switch (c.type) {
    case KvType::F32: return out_bf16 ? read_rows<float, bf>(p, c.N, stream) : read_rows<float, float>(p, c.N, stream);
    case KvType::BF16: return out_bf16 ? read_rows<bf, bf>(p, c.N, stream) : read_rows<bf, float>(p, c.N, stream);
    case KvType::I8: return out_bf16 ? read_rows<int8_t, bf>(p, c.N, stream) : read_rows<int8_t, float>(p, c.N, stream);
  }
  return cudaErrorInvalidValue;
}

}  // namespace sb
