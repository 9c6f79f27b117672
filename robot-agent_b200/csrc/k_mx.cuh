// Microscaled rows: 32 values of a row share a power of two, each value is kept in 4 bits (e2m1)
// or 8 bits (e4m3).
//
// Block rule: with m the largest magnitude, e = floor(log2 m) - emax (emax = 2 for e2m1, whose
// largest value is 1.5 * 2^2; 8 for e4m3, 1.75 * 2^8), clamped to -127..127; the codes are the
// nearest values of the format to x / 2^e, ties to even, saturating.  floor(log2 m) is m's exponent
// field; m itself is taken as the largest magnitude BIT pattern, an unsigned maximum, under which
// an infinity is above every number and a NaN above an infinity, so that such a block is seen and
// gets the scale NaN (255) whatever its other values are.  x / 2^e is an exact product (2^-e is
// a normal float for every e that a block can have), so the only rounding is the conversion's.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "../../include/smg.h"

#ifndef DEV
#define DEV __device__ __forceinline__
#endif

// ---- 8 consecutive values of a row <-> 8 floats ----
template <int TYPE>
struct Elem;
template <>
struct Elem<SMG_EMB_F32> {
  typedef float T;
  static DEV float up(float v) { return v; }
  static DEV float down(float v) { return v; }
};
template <>
struct Elem<SMG_EMB_BF16> {
  typedef __nv_bfloat16 T;
  static DEV float up(__nv_bfloat16 v) { return __bfloat162float(v); }
  static DEV __nv_bfloat16 down(float v) { return __float2bfloat16_rn(v); }
};
template <>
struct Elem<SMG_EMB_F16> {
  typedef __half T;
  static DEV float up(__half v) { return __half2float(v); }
  static DEV __half down(float v) { return __float2half_rn(v); }
};

// p: the first of 8 values, of which n (<= 8, may be <= 0) exist; vec: p is 16-byte aligned
template <int TYPE>
DEV void load8(const typename Elem<TYPE>::T* p, int n, bool vec, float (&v)[8]) {
  typedef typename Elem<TYPE>::T T;
  if (vec && n >= 8) {
    union { uint4 q[sizeof(T) / 2]; T t[8]; } u;
    const uint4* s = (const uint4*)p;
#pragma unroll
    for (int i = 0; i < (int)sizeof(T) / 2; ++i) u.q[i] = __ldg(s + i);
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = Elem<TYPE>::up(u.t[i]);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = i < n ? Elem<TYPE>::up(p[i]) : 0.f;
  }
}

// The same in two steps, for kernels that first issue all of a row's loads: 8 values as they lie in
// memory (none past n: zero bits are the value 0), and the floats they are.  VEC: p on 16 bytes, n a multiple of 8.
template <int TYPE>
struct Raw8 {
  typedef typename Elem<TYPE>::T T;
  union { uint4 q[sizeof(T) / 2]; T t[8]; };
  template <bool VEC>
  DEV void load(const T* p, int n) {
    if constexpr (VEC) {
#pragma unroll
      for (int i = 0; i < (int)sizeof(T) / 2; ++i) q[i] = n > 0 ? __ldg((const uint4*)p + i) : make_uint4(0, 0, 0, 0);
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) t[i] = i < n ? p[i] : Elem<TYPE>::down(0.f);
    }
  }
  DEV float get(int i) const { return Elem<TYPE>::up(t[i]); }
};

template <int TYPE>
DEV void store8(typename Elem<TYPE>::T* p, int n, bool vec, const float (&v)[8]) {
  typedef typename Elem<TYPE>::T T;
  if (vec && n >= 8) {
    union { uint4 q[sizeof(T) / 2]; T t[8]; } u;
#pragma unroll
    for (int i = 0; i < 8; ++i) u.t[i] = Elem<TYPE>::down(v[i]);
#pragma unroll
    for (int i = 0; i < (int)sizeof(T) / 2; ++i) ((uint4*)p)[i] = u.q[i];
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (i < n) p[i] = Elem<TYPE>::down(v[i]);
  }
}

// 2^e, -127 <= e <= 127
DEV float mx_two(int e) { return __int_as_float(e > -127 ? (e + 127) << 23 : 1 << 22); }

// scale byte of a block whose largest magnitude has the bit pattern m
template <int BITS>
DEV uint32_t mx_scale(uint32_t m) {
  if (m >= 0x7f800000u) return 255u;
  const int s = (int)(m >> 23) - (BITS == 4 ? 2 : 8);
  return (uint32_t)(s < 0 ? 0 : s);
}

// 8 values (already over 2^e) to codes: 4 bytes (4 bits) or 8 bytes
template <int BITS>
DEV void mx_codes(const float (&u)[8], uint32_t (&c)[2]) {
  if (BITS == 4) {
    uint16_t h[2];
#pragma unroll
    for (int i = 0; i < 2; ++i)
      asm("{\n\t.reg .b8 a, b;\n\t"
          "cvt.rn.satfinite.e2m1x2.f32 a, %2, %1;\n\t"
          "cvt.rn.satfinite.e2m1x2.f32 b, %4, %3;\n\t"
          "mov.b16 %0, {a, b};\n\t}"
          : "=h"(h[i])
          : "f"(u[4 * i]), "f"(u[4 * i + 1]), "f"(u[4 * i + 2]), "f"(u[4 * i + 3]));
    c[0] = (uint32_t)h[0] | (uint32_t)h[1] << 16;
    c[1] = 0;
  } else {
#pragma unroll
    for (int h = 0; h < 2; ++h)
      asm("{\n\t.reg .b16 a, b;\n\t"
          "cvt.rn.satfinite.e4m3x2.f32 a, %2, %1;\n\t"
          "cvt.rn.satfinite.e4m3x2.f32 b, %4, %3;\n\t"
          "mov.b32 %0, {a, b};\n\t}"
          : "=r"(c[h])
          : "f"(u[4 * h]), "f"(u[4 * h + 1]), "f"(u[4 * h + 2]), "f"(u[4 * h + 3]));
  }
}

// Codes of 8 values back to floats (without the scale).  An e2m1 code's 3 magnitude bits, put at the
// border of a float's exponent and mantissa, are the value times 2^-126 (subnormal ones too).
template <int BITS>
DEV void mx_decode(const uint32_t (&c)[2], float (&u)[8]) {
  if constexpr (BITS == 4) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const uint32_t n = c[0] >> (4 * i);
      u[i] = __uint_as_float((n & 7u) << 22 | (n & 8u) << 28) * __uint_as_float(253u << 23);
    }
  } else {
#pragma unroll
    for (int q = 0; q < 2; ++q) {
      uint32_t h[2];
      asm("{\n\t.reg .b16 a, b;\n\t"
          "mov.b32 {a, b}, %2;\n\t"
          "cvt.rn.f16x2.e4m3x2 %0, a;\n\t"
          "cvt.rn.f16x2.e4m3x2 %1, b;\n\t}"
          : "=r"(h[0]), "=r"(h[1])
          : "r"(c[q]));
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const __half2 p = *(const __half2*)&h[i];
        u[4 * q + 2 * i] = __low2float(p);
        u[4 * q + 2 * i + 1] = __high2float(p);
      }
    }
  }
}

struct MxOut {
  uint8_t* codes;      // rows of kb * 32 * bits / 8 bytes
  uint8_t* scales;     // rows of pitch bytes
  __nv_bfloat16* values;
  int dim, kb, pitch;  // values a row, its blocks, bytes of a row of scales (blocks rounded up to 4)
};

// Codes, scale and values of the 8 values v at 8 * j of `row`; 4 neighbouring lanes (j = 4b .. 4b + 3)
// hold one block and all 32 lanes of the warp call this together.  v is zero past dim.
template <int BITS>
DEV void mx_emit(const MxOut& o, int64_t row, int j, const float (&v)[8]) {
  uint32_t m = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) m = max(m, __float_as_uint(v[i]) & 0x7fffffffu);
  m = max(m, __shfl_xor_sync(0xffffffffu, m, 1));
  m = max(m, __shfl_xor_sync(0xffffffffu, m, 2));
  const int b = j >> 2;
  if (b >= o.pitch) return;
  const uint32_t s = mx_scale<BITS>(m);
  if (o.scales && !(j & 3)) o.scales[row * o.pitch + b] = (uint8_t)(b < o.kb ? s : 0u);
  if (b >= o.kb) return;
  const float inv = mx_two(s == 255u ? 0 : 127 - (int)s);
  float u[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) u[i] = v[i] * inv;
  uint32_t c[2];
  mx_codes<BITS>(u, c);
  if (o.codes) {
    uint8_t* d = o.codes + (row * o.kb * 4 + j) * BITS;   // 8 values are BITS bytes
    if (BITS == 4) *(uint32_t*)d = c[0];
    else *(uint2*)d = make_uint2(c[0], c[1]);
  }
  if (o.values) {
    mx_decode<BITS>(c, u);
    const float two = s == 255u ? __int_as_float(0x7fc00000) : mx_two((int)s - 127);
#pragma unroll
    for (int i = 0; i < 8; ++i) u[i] *= two;
    store8<SMG_EMB_BF16>(o.values + row * o.dim + 8 * j, o.dim - 8 * j, !(o.dim & 7), u);
  }
}

// Row and place of the t-th of a matrix's 8-value parts, `per` a row; 32-bit division where it does.
DEV void mx_place(int64_t t, int64_t n, int per, int64_t& row, int& j) {
  if (n <= 0x7fffffff) {
    const uint32_t r = (uint32_t)t / (uint32_t)per;
    row = r;
    j = (int)((uint32_t)t - r * (uint32_t)per);
  } else {
    row = t / per;
    j = (int)(t - row * per);
  }
}

// MX_EACH parts of 8 values a thread, a block's width apart; all loads first.  Bound by memory: per value
// it reads the input once and writes bits / 8 + 1/32 bytes (and 2 with `values`).
#define MX_EACH 4
template <int TYPE, int BITS, bool VEC>
__global__ void __launch_bounds__(256) k_mx_quantise(const typename Elem<TYPE>::T* x, int64_t ldx, int64_t n, MxOut o) {
  const int per = o.pitch * 4;   // parts a row
  const int64_t t0 = (int64_t)blockIdx.x * (256 * MX_EACH) + threadIdx.x;
  Raw8<TYPE> raw[MX_EACH];
  int64_t row;
  int j;
  mx_place(t0, n, per, row, j);
  int64_t r = row;
  int c = j;
#pragma unroll
  for (int i = 0; i < MX_EACH; ++i) {
    const bool live = t0 + i * 256 < n;
    raw[i].template load<VEC>(live ? x + r * ldx + 8 * c : x, live ? o.dim - 8 * c : 0);
    for (c += 256; c >= per; c -= per) ++r;
  }
#pragma unroll
  for (int i = 0; i < MX_EACH; ++i) {
    float v[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = raw[i].get(e);
    // n and `per` are multiples of 4, so the lanes of a block of 32 are all in or all out of range
    mx_emit<BITS>(o, row, t0 + i * 256 < n ? j : o.pitch * 4, v);
    for (j += 256; j >= per; j -= per) ++row;
  }
}

// MX_EACH parts of 8 values a thread
template <int TYPE, int BITS>
__global__ void __launch_bounds__(256) k_mx_values(MxOut o, int64_t n, typename Elem<TYPE>::T* out, int64_t ld, bool vec) {
  const int per = o.kb * 4;
  const int64_t t0 = (int64_t)blockIdx.x * (256 * MX_EACH) + threadIdx.x;
  int64_t row;
  int j;
  mx_place(t0, n, per, row, j);
#pragma unroll
  for (int i = 0; i < MX_EACH; ++i) {
    if (t0 + i * 256 >= n) return;
    const uint8_t* d = o.codes + (row * per + j) * BITS;
    uint32_t c[2];
    c[0] = __ldg((const uint32_t*)d);
    c[1] = BITS == 8 ? __ldg((const uint32_t*)d + 1) : 0u;
    const uint32_t s = o.scales[row * o.pitch + (j >> 2)];
    float u[8];
    mx_decode<BITS>(c, u);
    const float two = s == 255u ? __int_as_float(0x7fc00000) : mx_two((int)s - 127);
#pragma unroll
    for (int e = 0; e < 8; ++e) u[e] *= two;
    store8<TYPE>(out + row * ld + 8 * j, o.dim - 8 * j, vec, u);
    for (j += 256; j >= per; j -= per) ++row;
  }
}
