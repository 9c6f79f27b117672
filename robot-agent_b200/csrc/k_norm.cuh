// Root-mean-square norm with the residual's addition, its rows written in microscaled codes, and
// its gradients.
//
//   h = x + r,  rstd = 1 / sqrt(mean(h^2) + eps),  y = h * rstd * gain
//   n = h * rstd,  u = dy * gain,  dx = rstd * (u - n * mean(u * n)) + dh,  dgain = sum_rows dy * n
//
// A row is held in registers (8 values a lane and step, h in 32 bits) between the sum of squares
// and the outputs, so every input is read once and every output written once; both kernels are bound by
// memory.  WARPS warps share a row: one for short rows, so that no row waits on a block barrier.
#pragma once
#include "k_mx.cuh"

struct NormArgs {
  const void *x, *r, *dy, *dh;
  int64_t ldx, ldr, ldy, ldh_in;
  const float* gain;
  void *h, *dx;
  int64_t ldh, lddx;
  float *rstd, *part;
  int rows, dim;
  float eps;
  bool vec;     // every row of x, r, dy, dh, h and dx starts on 16 bytes
  bool gvec;    // gain starts on 16 bytes
  MxOut mx;
};

DEV float warp_sum(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// sum over the WARPS warps that share a row; scr: WARPS floats of the row's group of warps
template <int WARPS>
DEV float row_sum(float v, float* scr) {
  v = warp_sum(v);
  if (WARPS == 1) return v;
  const int w = (threadIdx.x >> 5) % WARPS;
  __syncthreads();
  if ((threadIdx.x & 31) == 0) scr[w] = v;
  __syncthreads();
  v = 0.f;
#pragma unroll
  for (int i = 0; i < WARPS; ++i) v += scr[i];
  return v;
}

#define NORM_THREADS 256
#define NORM_ROWS(WARPS) (8 / (WARPS))   // rows a block works on at a time

template <int TYPE, int BITS, int WARPS, int NV>
__global__ void __launch_bounds__(NORM_THREADS) k_norm_add(NormArgs a) {
  typedef typename Elem<TYPE>::T T;
  __shared__ float scr[NORM_ROWS(WARPS)][WARPS];
  const int sub = threadIdx.x / (32 * WARPS), t = threadIdx.x % (32 * WARPS);
  const int64_t row = (int64_t)blockIdx.x * NORM_ROWS(WARPS) + sub;
  const bool live = row < a.rows;   // uniform over the row's warps; with WARPS > 1 no early exit before a barrier
  float h[NV][8];
  float ss = 0.f;
  if (live) {
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = 8 * (t + i * 32 * WARPS), n = a.dim - c;
      load8<TYPE>((const T*)a.x + row * a.ldx + c, n, a.vec, h[i]);
      if (a.r) {
        float r[8];
        load8<TYPE>((const T*)a.r + row * a.ldr + c, n, a.vec, r);
#pragma unroll
        for (int k = 0; k < 8; ++k) h[i][k] += r[k];
      }
    }
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
      for (int k = 0; k < 8; ++k) ss = __fmaf_rn(h[i][k], h[i][k], ss);
  }
  ss = row_sum<WARPS>(ss, scr[sub]);
  if (!live) return;
  const float rstd = 1.f / sqrtf(ss / (float)a.dim + a.eps);
  if (a.rstd && t == 0) a.rstd[row] = rstd;
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int j = t + i * 32 * WARPS, c = 8 * j, n = a.dim - c;
    if (a.h) store8<TYPE>((T*)a.h + row * a.ldh + c, n, a.vec, h[i]);
    if (BITS) {
      float g[8];
      load8<SMG_EMB_F32>(a.gain + c, n, a.gvec, g);
#pragma unroll
      for (int k = 0; k < 8; ++k) h[i][k] = h[i][k] * rstd * g[k];
      mx_emit<BITS>(a.mx, row, j, h[i]);
    }
  }
}

// Gradients.  The blocks walk the rows with a stride; each lane keeps the dgain of its columns in
// registers, a block joins its rows' sums at the end (in warp order) and writes one partial row,
// which k_norm_dgain adds up in block order.
template <int TYPE, int WARPS, int NV>
__global__ void __launch_bounds__(NORM_THREADS) k_norm_add_bwd(NormArgs a) {
  typedef typename Elem<TYPE>::T T;
  __shared__ float scr[NORM_ROWS(WARPS)][WARPS];
  extern __shared__ float acc[];   // dim floats (NORM_ROWS > 1)
  const int sub = threadIdx.x / (32 * WARPS), t = threadIdx.x % (32 * WARPS);
  float dg[NV][8];
#pragma unroll
  for (int i = 0; i < NV; ++i)
#pragma unroll
    for (int k = 0; k < 8; ++k) dg[i][k] = 0.f;
  const int64_t step = (int64_t)gridDim.x * NORM_ROWS(WARPS);
  for (int64_t r0 = (int64_t)blockIdx.x * NORM_ROWS(WARPS); r0 < a.rows; r0 += step) {
    const int64_t row = r0 + sub;
    const bool live = row < a.rows;
    float n[NV][8], u[NV][8];
    float dot = 0.f, rstd = 0.f;
    if (live) {
      rstd = a.rstd[row];
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const int c = 8 * (t + i * 32 * WARPS), left = a.dim - c;
        load8<TYPE>((const T*)a.x + row * a.ldx + c, left, a.vec, n[i]);
        load8<TYPE>((const T*)a.dy + row * a.ldy + c, left, a.vec, u[i]);
        if (a.r) {
          float r[8];
          load8<TYPE>((const T*)a.r + row * a.ldr + c, left, a.vec, r);
#pragma unroll
          for (int k = 0; k < 8; ++k) n[i][k] += r[k];
        }
      }
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const int c = 8 * (t + i * 32 * WARPS);
        float g[8];
        load8<SMG_EMB_F32>(a.gain + c, a.dim - c, a.gvec, g);
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          n[i][k] *= rstd;
          dg[i][k] = __fmaf_rn(u[i][k], n[i][k], dg[i][k]);
          u[i][k] *= g[k];
          dot = __fmaf_rn(u[i][k], n[i][k], dot);
        }
      }
    }
    dot = row_sum<WARPS>(dot, scr[sub]) / (float)a.dim;
    if (live) {
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const int c = 8 * (t + i * 32 * WARPS), left = a.dim - c;
        float d[8] = {0, 0, 0, 0, 0, 0, 0, 0};
        if (a.dh) load8<TYPE>((const T*)a.dh + row * a.ldh_in + c, left, a.vec, d);
#pragma unroll
        for (int k = 0; k < 8; ++k) d[k] = __fmaf_rn(rstd, __fmaf_rn(-n[i][k], dot, u[i][k]), d[k]);
        store8<TYPE>((T*)a.dx + row * a.lddx + c, left, a.vec, d);
      }
    }
  }
  float* part = a.part + (int64_t)blockIdx.x * a.dim;
  if constexpr (NORM_ROWS(WARPS) == 1) {
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        const int c = 8 * (t + i * 32 * WARPS) + k;
        if (c < a.dim) part[c] = dg[i][k];
      }
  } else {
    for (int s = 0; s < NORM_ROWS(WARPS); ++s) {   // one row's warps after the other
      if (sub == s) {
#pragma unroll
        for (int i = 0; i < NV; ++i)
#pragma unroll
          for (int k = 0; k < 8; ++k) {
            const int c = 8 * (t + i * 32 * WARPS) + k;
            if (c < a.dim) {
              const float v = (s ? acc[c] : 0.f) + dg[i][k];
              if (s == NORM_ROWS(WARPS) - 1) part[c] = v;
              else acc[c] = v;
            }
          }
      }
      __syncthreads();
    }
  }
}

// dgain[c] = sum of the parts, in order: 32 columns x 8 spans of parts a block
__global__ void __launch_bounds__(256) k_norm_dgain(const float* part, int n_part, int dim, float* dgain) {
  __shared__ float s[8][32];
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5, c = blockIdx.x * 32 + lane;
  float v = 0.f;
  if (c < dim)
    for (int p = w; p < n_part; p += 8) v += part[(int64_t)p * dim + c];
  s[w][lane] = v;
  __syncthreads();
  if (w == 0 && c < dim) {
    v = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) v += s[i][lane];
    dgain[c] = v;
  }
}
