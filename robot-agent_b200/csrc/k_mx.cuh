// Microscaled rows: 32 values of a row share a power of two, each value is kept in 4 bits (e2m1)
// or 8 bits (e4m3).
//
// Block rule: with m the largest magnitude, e = floor(log2 m) - emax (emax = 2 for e2m1, whose
// largest value is 1.5 * 2^2; 8 for e4m3, 1.75 * 2^8), clamped to -127..127; the codes are the
// nearest values of the format to x / 2^e, ties to even, saturating.  floor(log2 m) is m's exponent
// field; m is taken with the maximum that hands NaN on, so that a block with an infinity or NaN is seen
// and gets the scale NaN (255) whatever its other values are.  x / 2^e is an exact product (2^-e is
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

// Programmatic launch: a kernel may be set up while the one before it in the stream still runs.  It
// touches global memory only after heads_wait(), which returns when that one is complete, its writes included, and
// reads it with ordinary loads: the read-only path (__ldg) is for memory that nobody writes in a kernel's lifetime,
// which begins before the wait.
DEV void heads_wait() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
DEV void heads_next() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }

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

// 8 values of a row as they lie in memory (zeros past n, which may be <= 0), and the floats they are: in two
// steps, so that a kernel can issue all of its loads first.  VEC: p on 16 bytes, n a multiple of 8.
template <int TYPE>
struct Raw8 {
  typedef typename Elem<TYPE>::T T;
  union { uint4 q[sizeof(T) / 2]; T t[8]; uint32_t w[2 * sizeof(T)]; };
  template <bool VEC>
  DEV void load(const T* p, int n) {   // p is used only where n > 0
    if constexpr (VEC) {
#pragma unroll
      for (int i = 0; i < (int)sizeof(T) / 2; ++i) q[i] = n > 0 ? ((const uint4*)p)[i] : make_uint4(0, 0, 0, 0);
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) t[i] = i < n ? p[i] : Elem<TYPE>::down(0.f);
    }
  }
  DEV float get(int i) const { return Elem<TYPE>::up(t[i]); }
};

// N words of w + `bytes` (0 .. 15): w has N + 4
template <int N>
DEV void words_from(const uint32_t (&w)[N + 4], uint32_t bytes, uint32_t (&out)[N]) {
  uint32_t a[N + 2], b[N + 1];
#pragma unroll
  for (int i = 0; i < N + 2; ++i) a[i] = bytes & 8u ? w[i + 2] : w[i];
#pragma unroll
  for (int i = 0; i < N + 1; ++i) b[i] = bytes & 4u ? a[i + 1] : a[i];
#pragma unroll
  for (int i = 0; i < N; ++i) out[i] = __funnelshift_r(b[i], b[i + 1], (bytes & 3u) * 8);
}

// The same of rows that start anywhere (a matrix of odd length): the 16-byte words around the 8 values, as far
// as they lie within the matrix (lo .. hi), then a shift; value by value at its two ends.
template <int TYPE>
struct Any8 {
  typedef typename Elem<TYPE>::T T;
  static constexpr int V = sizeof(T) / 2;   // 16-byte words of 8 values
  uint32_t w[4 * V + 4];
  const T* p;
  int n;
  bool in;
  DEV void begin(const T* at, int left, uintptr_t lo, uintptr_t hi) {
    p = at;
    n = left;
    const uintptr_t a = (uintptr_t)at & ~(uintptr_t)15;
    in = n > 0 && a >= lo && a + 16 * (V + 1) <= hi;
#pragma unroll
    for (int i = 0; i <= V; ++i) {
      const uint4 q = in ? ((const uint4*)a)[i] : make_uint4(0, 0, 0, 0);
      w[4 * i] = q.x; w[4 * i + 1] = q.y; w[4 * i + 2] = q.z; w[4 * i + 3] = q.w;
    }
  }
  DEV void end(Raw8<TYPE>& r) const {
    if (in) {
      words_from<4 * V>(w, (uint32_t)((uintptr_t)p & 15), r.w);
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (i >= n) r.t[i] = Elem<TYPE>::down(0.f);
    } else {
      r.template load<false>(p, n);
    }
  }
};

// One past the last byte of a matrix
template <typename T>
DEV uintptr_t rows_end(const void* p, int64_t rows, int64_t ld, int dim) {
  return (uintptr_t)p + ((rows - 1) * ld + dim) * sizeof(T);
}

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

// 8 16-bit values (as 4 words) to p, n of them there; the lanes' places j count along a row, and all 32 lanes
// call this together.  Off 16 bytes a lane stores the aligned 16 bytes that begin in its values and end in its
// neighbour's; what no such store takes (the ends of a row and of the warp) goes value by value.
DEV void store8_any(uint16_t* p, int n, int j, const uint32_t (&c)[4]) {
  const uint32_t sh = (uint32_t)(uintptr_t)p & 15u, lane = threadIdx.x & 31;
  uint32_t w[8], out[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    w[i] = c[i];
    w[4 + i] = __shfl_down_sync(0xffffffffu, c[i], 1);
  }
  const int nj = __shfl_down_sync(0xffffffffu, j, 1), nn = __shfl_down_sync(0xffffffffu, n, 1), pj = __shfl_up_sync(0xffffffffu, j, 1);
  if (n <= 0) return;
  if (sh == 0 && n >= 8) {
    *(uint4*)p = make_uint4(c[0], c[1], c[2], c[3]);
    return;
  }
  const int head = (int)(16 - sh) / 2;   // values before the aligned 16 bytes
  const bool mine = sh && lane < 31 && nj == j + 1 && nn >= head && n >= 8;
  const bool before = sh && lane > 0 && pj == j - 1 && n >= head;   // the neighbour's store takes my first ones
  if (mine) {
    words_from<4>(w, 16 - sh, out);
    *(uint4*)(p + head) = make_uint4(out[0], out[1], out[2], out[3]);
  }
  const int from = before ? head : 0, to = mine ? head : n < 8 ? n : 8;
#pragma unroll
  for (int i = 0; i < 8; ++i)
    if (i >= from && i < to) p[i] = (uint16_t)(c[i >> 1] >> (16 * (i & 1)));
}

DEV float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

// scale byte of a block whose largest magnitude is m
template <int BITS>
DEV uint32_t mx_scale(float m) {
  const uint32_t b = __float_as_uint(m);
  if (b >= 0x7f800000u) return 255u;
  const int s = (int)(b >> 23) - (BITS == 4 ? 2 : 8);
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

// Codes of 8 e2m1 values to 8 bf16 ones (without the scale) times 2^-126: a code's 3 magnitude bits,
// put at the border of exponent and mantissa, are that (subnormal ones too).
DEV void mx_e2m1_bf16(uint32_t c, uint32_t (&p)[4]) {
  const uint32_t lo = c & 0x0f0f0f0fu, hi = c >> 4 & 0x0f0f0f0fu;   // even and odd values, a byte each
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    uint32_t w;   // value 2i in the low half, 2i + 1 in the high one
    if (i == 0) w = __byte_perm(lo, hi, 0x7470) & 0x000f000fu;
    else if (i == 1) w = __byte_perm(lo, hi, 0x7571) & 0x000f000fu;
    else if (i == 2) w = __byte_perm(lo, hi, 0x7672) & 0x000f000fu;
    else w = __byte_perm(lo, hi, 0x7773) & 0x000f000fu;
    p[i] = (w << 6 & 0x01c001c0u) | (w << 12 & 0x80008000u);
  }
}

DEV __nv_bfloat162 bf162(uint32_t bits) { return *(const __nv_bfloat162*)&bits; }
DEV __nv_bfloat162 bf162_all(uint32_t one) { return bf162(one | one << 16); }

// Codes of 8 values to the bf16 values they stand for, with the block's scale byte.  Products of
// powers of two and values of 4 bits or fewer of mantissa: exact, but below 2^-126.
template <int BITS>
DEV void mx_values8(const uint32_t (&c)[2], uint32_t scale, uint32_t (&out)[4]) {
  // 2^(scale - 127) in bf16 (subnormal for 0), or NaN
  const uint32_t two = scale == 255u ? 0x7fc0u : scale ? scale << 7 : 0x40u;
  if constexpr (BITS == 4) {
    mx_e2m1_bf16(c[0], out);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const __nv_bfloat162 v = __hmul2(__hmul2(bf162(out[i]), bf162_all(253u << 7)), bf162_all(two));
      out[i] = *(const uint32_t*)&v;
    }
  } else {
    const float f = __uint_as_float(two << 16);
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
        const __nv_bfloat162 v = __floats2bfloat162_rn(__low2float(p) * f, __high2float(p) * f);
        out[2 * q + i] = *(const uint32_t*)&v;
      }
    }
  }
}

// Division of a place below 2^31 by `per`: (t * mul) >> (31 + shift), mul = ceil(2^(31 + shift) / per),
// shift = ceil(log2 per)
struct MxDiv {
  uint32_t per, mul;
  int shift;
};

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
  float m = fabsf(v[0]);
#pragma unroll
  for (int i = 1; i < 8; ++i) m = max_nan(m, fabsf(v[i]));
  m = max_nan(m, __shfl_xor_sync(0xffffffffu, m, 1));
  m = max_nan(m, __shfl_xor_sync(0xffffffffu, m, 2));
  const int b = j >> 2;
  const bool there = b < o.kb;
  const uint32_t s = mx_scale<BITS>(m);
  if (o.scales && !(j & 3) && b < o.pitch) o.scales[row * o.pitch + b] = (uint8_t)(there ? s : 0u);
  const float inv = __uint_as_float(s == 255u ? 0x3f800000u : (254u - s) << 23);
  float u[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) u[i] = v[i] * inv;
  uint32_t c[2];
  mx_codes<BITS>(u, c);
  if (o.codes && there) {
    uint8_t* d = o.codes + (row * o.kb * 4 + j) * BITS;   // 8 values are BITS bytes
    if (BITS == 4) *(uint32_t*)d = c[0];
    else *(uint2*)d = make_uint2(c[0], c[1]);
  }
  if (o.values) {
    uint32_t q[4];
    mx_values8<BITS>(c, s, q);
    uint16_t* d = (uint16_t*)o.values + row * o.dim + 8 * j;
    const int n = o.dim - 8 * j;
    if (!(o.dim & 7)) {
      if (n > 0) *(uint4*)d = make_uint4(q[0], q[1], q[2], q[3]);
    } else {
      store8_any(d, n, j, q);
    }
  }
}

// Row and place of the t-th of a matrix's n 8-value parts
DEV void mx_place(int64_t t, int64_t n, const MxDiv& d, int64_t& row, int& j) {
  if (n <= 0x7fffffff) {
    const uint32_t r = (uint32_t)((uint64_t)(uint32_t)t * d.mul >> (31 + d.shift));
    row = r;
    j = (int)((uint32_t)t - r * d.per);
  } else {
    row = t / d.per;
    j = (int)(t - row * d.per);
  }
}

// MX_EACH parts of 8 values a thread, a block's width apart; all loads first.  Bound by memory: per value
// it reads the input once and writes bits / 8 + 1/32 bytes (and 2 with `values`).  Measured on 16384 x 1152 bf16 in 4 bits
// with values: 16 us, 5.3 TB/s (81% of a copy's; the rest is the launch: 65536 rows run at 5.4); a form with one
// part a thread, a 64-bit division and codes decoded one by one had 235 instructions a part and took 20.
#define MX_EACH 4
template <int TYPE, int BITS, bool VEC>
__global__ void __launch_bounds__(256) k_mx_quantise(const typename Elem<TYPE>::T* x, int64_t ldx, int rows, int64_t n, MxDiv div, MxOut o) {
  heads_next();
  heads_wait();
  const int64_t t0 = (int64_t)blockIdx.x * (256 * MX_EACH) + threadIdx.x;
  Raw8<TYPE> raw[MX_EACH];
  Any8<TYPE> any[VEC ? 1 : MX_EACH];
  int64_t row[MX_EACH];
  int j[MX_EACH];
  const uintptr_t hi = rows_end<typename Elem<TYPE>::T>(x, rows, ldx, o.dim);
#pragma unroll
  for (int i = 0; i < MX_EACH; ++i) {
    mx_place(t0 + i * 256, n, div, row[i], j[i]);
    // n and a row's parts are multiples of 4, so the lanes of a block of 32 are all in or all out of range
    if (t0 + i * 256 >= n) { row[i] = 0; j[i] = o.pitch * 4; }
    const typename Elem<TYPE>::T* p = x + row[i] * ldx + 8 * j[i];
    if constexpr (VEC) raw[i].template load<true>(p, o.dim - 8 * j[i]);
    else any[i].begin(p, o.dim - 8 * j[i], (uintptr_t)x, hi);
  }
  if constexpr (!VEC) {
#pragma unroll
    for (int i = 0; i < MX_EACH; ++i) any[i].end(raw[i]);
  }
#pragma unroll
  for (int i = 0; i < MX_EACH; ++i) {
    float v[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = raw[i].get(e);
    mx_emit<BITS>(o, row[i], j[i], v);
  }
}

// MX_EACH parts of 8 values a thread.  Measured on 16384 x 1152 (replayed on one set): to bf16 9.8 us, to f32 21.5.
template <int TYPE, int BITS>
__global__ void __launch_bounds__(256) k_mx_values(MxOut o, int64_t n, MxDiv div, typename Elem<TYPE>::T* out, int64_t ld, bool vec) {
  heads_next();
  heads_wait();
  const int64_t t0 = (int64_t)blockIdx.x * (256 * MX_EACH) + threadIdx.x;
#pragma unroll
  for (int i = 0; i < MX_EACH; ++i) {
    if (t0 + i * 256 >= n) return;
    int64_t row;
    int j;
    mx_place(t0 + i * 256, n, div, row, j);
    const uint8_t* d = o.codes + (row * o.kb * 4 + j) * BITS;
    uint32_t c[2], q[4];
    c[0] = ((const uint32_t*)d)[0];
    c[1] = BITS == 8 ? ((const uint32_t*)d)[1] : 0u;
    const uint32_t s = o.scales[row * o.pitch + (j >> 2)];
    float u[8];
    if (TYPE == SMG_EMB_BF16) {
      mx_values8<BITS>(c, s, q);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        u[2 * e] = __uint_as_float(q[e] << 16);
        u[2 * e + 1] = __uint_as_float(q[e] & 0xffff0000u);
      }
    } else {   // the values without the scale are exact in bf16; the scale is applied in 32 bits
      mx_values8<BITS>(c, 127, q);
      const float two = s == 255u ? __int_as_float(0x7fc00000) : mx_two((int)s - 127);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        u[2 * e] = __uint_as_float(q[e] << 16) * two;
        u[2 * e + 1] = __uint_as_float(q[e] & 0xffff0000u) * two;
      }
    }
    store8<TYPE>(out + row * ld + 8 * j, o.dim - 8 * j, vec, u);
  }
}
