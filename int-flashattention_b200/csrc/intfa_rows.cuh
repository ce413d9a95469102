// Rows of one head of one token: loading, rotating and quantising them, a lane holding two pieces of 8 channels
// (so D/16 lanes, 1 to 16, hold a row).  Shared by the rotation and the paged cache's append.
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

// How a row is rotated.  kHalf: pair j is channels (j, j + rot/2), rot a multiple of 16; kAny: the same for other rot, element by element
// with the partner read from memory once more; kPairs: channels (2j, 2j + 1).
enum Spin { kNone, kHalf, kAny, kPairs };

// Which 16 channels of a row lane j of D/16 holds, as two pieces of 8.  kHalf: both halves of the same pairs, so that a rotation stays
// within the lane; the pieces that are not rotated two by two.  Else neighbours.
struct Pieces {
  int a, b;                          // first channel of each
  template <int SPIN>
  __device__ __forceinline__ void place(int j, int rot) {
    const int h8 = rot >> 4;
    if (SPIN == kHalf) {
      a = j < h8 ? 8 * j : 16 * j;   // (16 h8 + 16 (j - h8))
      b = j < h8 ? 8 * (j + h8) : a + 8;
    } else {
      a = 16 * j;
      b = a + 8;
    }
  }
};
template <typename T>
struct Row16 {
  Raw<T> a, b;
  __device__ __forceinline__ void load(const T* row, const Pieces& at) {
    a.load(row + at.a);
    b.load(row + at.b);
  }
  __device__ __forceinline__ void zero() {
    a.zero();
    b.zero();
  }
};
template <typename T>
__device__ __forceinline__ void widen16(const Row16<T>& r, float (&x)[16]) {
  widen(r.a, reinterpret_cast<float(&)[8]>(x[0]));
  widen(r.b, reinterpret_cast<float(&)[8]>(x[8]));
}

// The rotation of a lane's channels at one position: (a, b) of pair j becomes (a c - b s, b c + a s) with (c, s) = table[position][j].
// The products are rounded one by one (no fma, and no packed pairs, which the compiler does contract): the same bits as the same expression
// in single tensor operations.  What a lane needs of the table stays in registers for all heads of the token.
template <int SPIN>
struct Turn {
  float c[SPIN == kAny ? 16 : 8], s[SPIN == kAny ? 16 : 8];      // kHalf: of the lane's 8 pairs; kPairs: 4 of each piece; kAny: of its channels
  __device__ __forceinline__ void load(const float* table, long long pos, int rot, bool inverse, const Pieces& at) {
    if constexpr (SPIN == kNone) return;
    const int half = rot >> 1;
    const float2* row = reinterpret_cast<const float2*>(table) + pos * half;
    auto put = [&](int i, float2 f) {
      c[i] = f.x;
      s[i] = inverse ? -f.y : f.y;
    };
    if constexpr (SPIN == kHalf) {
#pragma unroll
      for (int i = 0; i < 8; ++i) c[i] = s[i] = 0.f;
      if (at.a >= half) return;
      const float4* r4 = reinterpret_cast<const float4*>(row + at.a);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float4 f = r4[i];
        put(2 * i, make_float2(f.x, f.y));
        put(2 * i + 1, make_float2(f.z, f.w));
      }
    } else if constexpr (SPIN == kPairs) {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int e = (i < 4 ? at.a : at.b) + 2 * (i & 3);
        put(i, e < rot ? row[e >> 1] : make_float2(1.f, 0.f));
      }
    } else {
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const int e = (i < 8 ? at.a : at.b) + (i & 7);
        put(i, e < rot ? row[e < half ? e : e - half] : make_float2(1.f, 0.f));
      }
    }
  }
  // x: the lane's channels; row: the row in memory
  template <typename T>
  __device__ __forceinline__ void apply(float (&x)[16], const T* row, int rot, const Pieces& at) const {
    const int half = rot >> 1;
    if constexpr (SPIN == kHalf) {
      if (at.a >= half) return;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float a = x[i], b = x[8 + i];
        x[i] = __fsub_rn(__fmul_rn(a, c[i]), __fmul_rn(b, s[i]));
        x[8 + i] = __fadd_rn(__fmul_rn(b, c[i]), __fmul_rn(a, s[i]));
      }
    } else if constexpr (SPIN == kPairs) {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int e = (i < 4 ? at.a : at.b) + 2 * (i & 3), k = 2 * i;
        if (e < rot) {
          const float a = x[k], b = x[k + 1];
          x[k] = __fsub_rn(__fmul_rn(a, c[i]), __fmul_rn(b, s[i]));
          x[k + 1] = __fadd_rn(__fmul_rn(b, c[i]), __fmul_rn(a, s[i]));
        }
      }
    } else if constexpr (SPIN == kAny) {
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const int e = (i < 8 ? at.a : at.b) + (i & 7);
        if (e < rot) {
          const float y = widen1(row[e < half ? e + half : e - half]);
          const float u = __fmul_rn(x[i], c[i]), v = __fmul_rn(y, s[i]);
          x[i] = e < half ? __fsub_rn(u, v) : __fadd_rn(u, v);
        }
      }
    }
  }
};

// largest magnitude, a NaN if there is one
__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float max_nan3(float a, float b, float c) {
  float r;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}
__device__ __forceinline__ float absmax16(const float (&x)[16]) {
  float m = fabsf(x[0]), n = fabsf(x[1]);
#pragma unroll
  for (int i = 2; i < 14; i += 4) {
    m = max_nan3(m, fabsf(x[i]), fabsf(x[i + 1]));
    n = max_nan3(n, fabsf(x[i + 2]), fabsf(x[i + 3]));
  }
  return max_nan3(max_nan(m, n), fabsf(x[14]), fabsf(x[15]));
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

// Values as int8 codes: x/scale, rounded to fp32 and then to the nearest whole number (ties to even); zeros where the scale is 0 or not
// finite.  Without a division: the reciprocal is approximate (2^-23), a little more and a little less of it (1 +- 2^-21, and 2^-24 of rounding)
// are on either side of every quotient that the division could give.  Where both round to the same code it is that one; where they do not, once
// in some 25 000 values, by a division.
template <int N>
__device__ __forceinline__ void codes(const float (&x)[N], float scale, uint32_t (&out)[N / 4]) {
  constexpr float kMagic = 12582912.0f;               // 1.5 * 2^23: the sum's low byte is the whole number
  const bool ok = scale > 0.f && scale <= 3.402823466e38f;
  float inverse;
  asm("rcp.approx.f32 %0, %1;" : "=f"(inverse) : "f"(scale));
  const float more = inverse * (1.f + 4.76837158e-7f), less = inverse * (1.f - 4.76837158e-7f);
  const uint64_t more2 = f2_pack(more, more), less2 = f2_pack(less, less), magic2 = f2_pack(kMagic, kMagic);
  uint32_t b[N], differ = 0u;
#pragma unroll
  for (int i = 0; i < N; i += 2) {
    const uint64_t q = f2_pack(x[i], x[i + 1]);
    uint32_t m0, m1;
    f2_unpacku(f2_fma(q, more2, magic2), m0, m1);
    f2_unpacku(f2_fma(q, less2, magic2), b[i], b[i + 1]);
    differ |= m0 ^ b[i];
    differ |= m1 ^ b[i + 1];
  }
  // (a scale whose reciprocal is not a normal number: the careful way)
  if (ok && !(differ == 0u && scale > 1e-37f && scale < 1e37f)) {
#pragma unroll
    for (int i = 0; i < N; ++i) b[i] = __float_as_uint(__fadd_rn(fminf(fmaxf(__fdiv_rn(x[i], scale), -127.f), 127.f), kMagic));
  }
#pragma unroll
  for (int i = 0; i < N / 4; ++i)
    out[i] = ok ? __byte_perm(__byte_perm(b[4 * i], b[4 * i + 1], 0x0040), __byte_perm(b[4 * i + 2], b[4 * i + 3], 0x0040), 0x5410) : 0u;
}

// 16 bytes to shared memory, zeros unless ok
__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, bool ok = true) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(ok ? 16 : 0) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_async_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

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
