// Rows of one head of one token: loading, rotating and quantising them, a lane holding 8 neighbouring channels
// (so D/8 lanes, 2 to 32, hold a row).  Shared by the rotation and the paged cache's append.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "intfa_internal.h"
#include "intfa_ptx.cuh"

namespace intfa {

// 8 channels as they lie in memory
template <typename T>
struct Raw {
  static constexpr int W = sizeof(T) * 2;             // 32-bit words
  uint32_t w[W];
  __device__ __forceinline__ void load(const T* p) {
#pragma unroll
    for (int i = 0; i < W; i += 4) {
      const uint4 x = *reinterpret_cast<const uint4*>(reinterpret_cast<const uint32_t*>(p) + i);
      w[i] = x.x; w[i + 1] = x.y; w[i + 2] = x.z; w[i + 3] = x.w;
    }
  }
  __device__ __forceinline__ void store(T* p) const {
#pragma unroll
    for (int i = 0; i < W; i += 4) *reinterpret_cast<uint4*>(reinterpret_cast<uint32_t*>(p) + i) = make_uint4(w[i], w[i + 1], w[i + 2], w[i + 3]);
  }
  __device__ __forceinline__ void zero() {
#pragma unroll
    for (int i = 0; i < W; ++i) w[i] = 0u;
  }
};
template <typename T>
__device__ __forceinline__ void widen(const Raw<T>& r, float (&x)[8]) {
#pragma unroll
  for (int i = 0; i < 8; i += 2) {
    if constexpr (sizeof(T) == 4) {
      x[i] = __uint_as_float(r.w[i]);
      x[i + 1] = __uint_as_float(r.w[i + 1]);
    } else if constexpr (__is_same(T, __half)) {
      const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&r.w[i / 2]));
      x[i] = f.x;
      x[i + 1] = f.y;
    } else {
      x[i] = __uint_as_float(r.w[i / 2] << 16);
      x[i + 1] = __uint_as_float(r.w[i / 2] & 0xffff0000u);
    }
  }
}
template <typename T>
__device__ __forceinline__ void narrow(const float (&x)[8], Raw<T>& r) {
#pragma unroll
  for (int i = 0; i < 8; i += 2) {
    if constexpr (sizeof(T) == 4) {
      r.w[i] = __float_as_uint(x[i]);
      r.w[i + 1] = __float_as_uint(x[i + 1]);
    } else if constexpr (__is_same(T, __half)) {
      const __half2 h = __floats2half2_rn(x[i], x[i + 1]);
      r.w[i / 2] = *reinterpret_cast<const uint32_t*>(&h);
    } else {
      const __nv_bfloat162 h = __floats2bfloat162_rn(x[i], x[i + 1]);
      r.w[i / 2] = *reinterpret_cast<const uint32_t*>(&h);
    }
  }
}
template <typename T>
__device__ __forceinline__ float widen1(T x) {
  if constexpr (sizeof(T) == 4) return x;
  else if constexpr (__is_same(T, __half)) return __half2float(x);
  else return __bfloat162float(x);
}

// The rotation of one lane's 8 channels at one position: pair j of the first rot channels, (a, b) = channels (j, j + rot/2), or
// (2j, 2j + 1) interleaved, becomes (a c - b s, b c + a s) with (c, s) = table[position][j].  The products are rounded one by one (no
// fma): the same bits as the same expression in single tensor operations.
// What a lane needs of the table stays in registers for all heads of the token.
struct Turn {
  float c[8], s[8];                  // half layout: of the lane's channels; interleaved: of its 4 pairs (the first 4)
  int kind;                          // 0: not rotated; 1, 2: half layout, the lane holds the a's, the b's; 3: interleaved; 4: half layout whose
                                     // border lies inside a lane's 8 channels (rot no multiple of 16): element by element
  __device__ __forceinline__ void load(const float* table, long long pos, int rot, bool interleaved, bool inverse, int e0) {
    const int half = rot >> 1;
    const float2* row = reinterpret_cast<const float2*>(table) + pos * half;
    kind = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) c[i] = s[i] = 0.f;
    if (e0 >= rot) {
      if (!interleaved && (half & 7)) kind = 4;        // (its lanes all take the same way)
    } else if (interleaved) {
      kind = 3;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float2 f = e0 + 2 * i < rot ? row[(e0 >> 1) + i] : make_float2(1.f, 0.f);
        c[i] = f.x;
        s[i] = inverse ? -f.y : f.y;
      }
    } else if ((half & 7) == 0) {
      kind = e0 < half ? 1 : 2;
      const float4* r4 = reinterpret_cast<const float4*>(row + (e0 < half ? e0 : e0 - half));
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float4 f = r4[i];
        c[2 * i] = f.x; s[2 * i] = inverse ? -f.y : f.y;
        c[2 * i + 1] = f.z; s[2 * i + 1] = inverse ? -f.w : f.w;
      }
    } else {
      kind = 4;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int e = e0 + i;
        const float2 f = e < rot ? row[e < half ? e : e - half] : make_float2(1.f, 0.f);
        c[i] = f.x;
        s[i] = inverse ? -f.y : f.y;
      }
    }
  }
  // x: the lane's channels, r: as loaded, row: the row in memory, e0: the lane's first channel.  All lanes of the warp call this together;
  // a row with turn = false is left alone.
  template <typename T>
  __device__ __forceinline__ void apply(float (&x)[8], const Raw<T>& r, const T* row, bool row_ok, int rot, bool interleaved, int e0, bool turn = true) const {
    const int kind = turn ? this->kind : 0;
    if (interleaved) {
      if (kind == 3) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          if (e0 + 2 * i >= rot) break;
          const float a = x[2 * i], b = x[2 * i + 1];
          x[2 * i] = __fsub_rn(__fmul_rn(a, c[i]), __fmul_rn(b, s[i]));
          x[2 * i + 1] = __fadd_rn(__fmul_rn(b, c[i]), __fmul_rn(a, s[i]));
        }
      }
      return;
    }
    const int half = rot >> 1;
    float y[8];
    if ((half & 7) == 0) {
      const int lane = threadIdx.x & 31, other = kind == 1 ? lane + (half >> 3) : kind == 2 ? lane - (half >> 3) : lane;
      Raw<T> o;
#pragma unroll
      for (int i = 0; i < Raw<T>::W; ++i) o.w[i] = __shfl_sync(0xffffffffu, r.w[i], other);
      widen(o, y);
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int e = e0 + i;
        y[i] = row_ok && e < rot ? widen1(row[e < half ? e + half : e - half]) : 0.f;
      }
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float p = __fmul_rn(x[i], c[i]), q = __fmul_rn(y[i], s[i]);
      if (kind == 1) x[i] = __fsub_rn(p, q);
      else if (kind == 2) x[i] = __fadd_rn(p, q);
      else if (kind == 4 && e0 + i < rot) x[i] = e0 + i < half ? __fsub_rn(p, q) : __fadd_rn(p, q);
    }
  }
};

// largest magnitude, a NaN if there is one
__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float absmax8(const float (&x)[8]) {
  float m = fabsf(x[0]);
#pragma unroll
  for (int i = 1; i < 8; ++i) m = max_nan(m, fabsf(x[i]));
  return m;
}
// ... of a row held by LPR neighbouring lanes
template <int LPR>
__device__ __forceinline__ float row_max(float m) {
#pragma unroll
  for (int o = LPR / 2; o > 0; o >>= 1) m = max_nan(m, __shfl_xor_sync(0xffffffffu, m, o));
  return m;
}
// the scale of values up to `most`, rounded to fp32; 0, infinite or NaN where there is none
__device__ __forceinline__ float scale_of(float most) { return __fdiv_rn(most, 127.0f); }

// 8 values as int8 codes: x/scale, rounded to fp32 and then to the nearest whole number (ties to even); zeros where the scale is 0 or not
// finite.  The quotient is formed with the reciprocal, whose error of less than 127 * 2^-22 decides nothing unless it is that near to
// a border of two codes: then, which is once in 10 000 values, by a division.
__device__ __forceinline__ uint2 codes8(const float (&x)[8], float scale, float inverse) {
  constexpr float kMagic = 12582912.0f;               // 1.5 * 2^23: the sum's low byte is the whole number
  if (!(scale > 0.f && scale <= 3.402823466e38f)) return make_uint2(0u, 0u);
  uint32_t b[8];
  float off = 0.f;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float q = __fmul_rn(x[i], inverse), t = __fadd_rn(q, kMagic);
    off = fmaxf(off, fabsf(__fsub_rn(q, __fsub_rn(t, kMagic))));
    b[i] = __float_as_uint(t);
  }
  // (a scale whose reciprocal overflows or is rounded as a subnormal, an `off` that is not small: the careful way)
  if (!(off < 0.4999f && scale > 1e-37f && inverse > 1e-37f)) {
#pragma unroll
    for (int i = 0; i < 8; ++i) b[i] = __float_as_uint(__fadd_rn(fminf(fmaxf(__fdiv_rn(x[i], scale), -127.f), 127.f), kMagic));
  }
  uint2 r;
  r.x = __byte_perm(__byte_perm(b[0], b[1], 0x0040), __byte_perm(b[2], b[3], 0x0040), 0x5410);
  r.y = __byte_perm(__byte_perm(b[4], b[5], 0x0040), __byte_perm(b[6], b[7], 0x0040), 0x5410);
  return r;
}

// largest i in [0, n) with f(i) <= x, by the lanes of a warp together (f grows, f(0) <= x)
template <typename F>
__device__ __forceinline__ int find_last(int n, long long x, F f) {
  int lo = 0;
  const int lane = threadIdx.x & 31;
  while (n > 1) {
    const int step = (n + 31) / 32, i = lane * step;
    const unsigned ok = __ballot_sync(0xffffffffu, i < n && f(lo + i) <= x);
    const int last = ok ? 31 - __clz(ok) : 0;
    lo += last * step;
    n = min(step, n - last * step);
  }
  return lo;
}

}  // namespace intfa
