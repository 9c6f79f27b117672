// Ragged products by group: y = x w_g^T, dx = dy w_g, dw_g = dy_g^T x_g, and the same first form of
// microscaled rows.  One thread per output value.
#pragma once
#include "k_mx.cuh"

struct ProdArgs {
  const int32_t* off;
  int n_groups, rows, n, k;
  const void *a, *b;              // x and w | dy and w | dy and x
  int64_t lda, ldb, b_stride;
  const uint8_t *sa, *sb;         // scales of microscaled a and b
  int pitch, row_bytes;
  void* y;
  int64_t ldy, y_stride;
  int y_type;
  int32_t* err;
};

DEV int prod_group(const ProdArgs& g, int row) {
  if (!g.off) return 0;
  int f = -1;
  for (int i = 0; i < g.n_groups; ++i)
    if (g.off[i] <= row && row < g.off[i + 1]) f = i;
  return f;
}

DEV void prod_put(const ProdArgs& g, int64_t at, float v) {
  if (g.y_type == SMG_EMB_F32) ((float*)g.y)[at] = v;
  else if (g.y_type == SMG_EMB_BF16) ((__nv_bfloat16*)g.y)[at] = __float2bfloat16_rn(v);
  else ((__half*)g.y)[at] = __float2half_rn(v);
}

DEV void prod_check(const ProdArgs& g) {
  if (!g.off || !g.err || blockIdx.x) return;
  for (int i = threadIdx.x; i < g.n_groups; i += blockDim.x) {
    const int p = g.off[i], q = g.off[i + 1];
    if (p < 0 || q < p || q > g.rows || (i == 0 && p) || (i == g.n_groups - 1 && q != g.rows)) atomicOr(g.err, SMG_PROD_OFFSETS);
  }
}

template <int TYPE>
__global__ void __launch_bounds__(256) k_prod_y(ProdArgs g) {
  typedef typename Elem<TYPE>::T T;
  prod_check(g);
  for (int64_t t = (int64_t)blockIdx.x * 256 + threadIdx.x; t < (int64_t)g.rows * g.n; t += (int64_t)gridDim.x * 256) {
    const int row = (int)(t / g.n), j = (int)(t % g.n), q = prod_group(g, row);
    if (q < 0) continue;
    const T *a = (const T*)g.a + row * g.lda, *b = (const T*)g.b + q * g.b_stride + j * g.ldb;
    float s = 0.f;
    for (int i = 0; i < g.k; ++i) s = __fmaf_rn(Elem<TYPE>::up(a[i]), Elem<TYPE>::up(b[i]), s);
    prod_put(g, row * g.ldy + j, s);
  }
}

template <int TYPE>
__global__ void __launch_bounds__(256) k_prod_dx(ProdArgs g) {
  typedef typename Elem<TYPE>::T T;
  prod_check(g);
  for (int64_t t = (int64_t)blockIdx.x * 256 + threadIdx.x; t < (int64_t)g.rows * g.k; t += (int64_t)gridDim.x * 256) {
    const int row = (int)(t / g.k), i = (int)(t % g.k), q = prod_group(g, row);
    if (q < 0) continue;
    const T *a = (const T*)g.a + row * g.lda, *b = (const T*)g.b + q * g.b_stride + i;
    float s = 0.f;
    for (int j = 0; j < g.n; ++j) s = __fmaf_rn(Elem<TYPE>::up(a[j]), Elem<TYPE>::up(b[j * g.ldb]), s);
    prod_put(g, row * g.ldy + i, s);
  }
}

template <int TYPE>
__global__ void __launch_bounds__(256) k_prod_dw(ProdArgs g) {
  typedef typename Elem<TYPE>::T T;
  prod_check(g);
  const int64_t per = (int64_t)g.n * g.k;
  for (int64_t t = (int64_t)blockIdx.x * 256 + threadIdx.x; t < per * g.n_groups; t += (int64_t)gridDim.x * 256) {
    const int q = (int)(t / per), j = (int)(t % per / g.k), i = (int)(t % g.k);
    int r0 = g.off ? g.off[q] : 0, r1 = g.off ? g.off[q + 1] : g.rows;
    if (r0 < 0 || r1 < r0 || r1 > g.rows) r1 = r0 = 0;
    float s = 0.f;
    for (int64_t r = r0; r < r1; ++r)
      s = __fmaf_rn(Elem<TYPE>::up(((const T*)g.a)[r * g.lda + j]), Elem<TYPE>::up(((const T*)g.b)[r * g.ldb + i]), s);
    prod_put(g, q * g.y_stride + j * g.ldy + i, s);
  }
}

template <int BITS>
__global__ void __launch_bounds__(256) k_prod_mx(ProdArgs g) {
  prod_check(g);
  for (int64_t t = (int64_t)blockIdx.x * 256 + threadIdx.x; t < (int64_t)g.rows * g.n; t += (int64_t)gridDim.x * 256) {
    const int row = (int)(t / g.n), j = (int)(t % g.n), q = prod_group(g, row);
    if (q < 0) continue;
    const int64_t br = (int64_t)q * g.n + j;
    float s = 0.f;
    for (int v = 0; v < g.row_bytes / BITS; ++v) {   // 8 values are BITS bytes
      uint32_t c[2] = {0, 0}, d[2] = {0, 0};
      const uint32_t* p = (const uint32_t*)((const uint8_t*)g.a + (int64_t)row * g.row_bytes + v * BITS);
      const uint32_t* w = (const uint32_t*)((const uint8_t*)g.b + br * g.row_bytes + v * BITS);
#pragma unroll
      for (int i = 0; i < BITS / 4; ++i) { c[i] = p[i]; d[i] = w[i]; }
      float x[8], y[8], e = 0.f;
      mx_decode<BITS>(c, x);
      mx_decode<BITS>(d, y);
#pragma unroll
      for (int i = 0; i < 8; ++i) e = __fmaf_rn(x[i], y[i], e);
      const int sx = g.sa[(int64_t)row * g.pitch + (v >> 2)], sy = g.sb[br * g.pitch + (v >> 2)];
      s += sx == 255 || sy == 255 ? __int_as_float(0x7fc00000) : e * mx_two(sx - 127) * mx_two(sy - 127);
    }
    prod_put(g, row * g.ldy + j, s);
  }
}
