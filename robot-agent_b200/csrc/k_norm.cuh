// Root-mean-square norm with the residual's addition, its rows written in microscaled codes, and
// its gradients.
//
//   h = x + r,  rstd = 1 / sqrt(mean(h^2) + eps),  y = h * rstd * gain
//   n = h * rstd,  u = dy * gain,  dx = rstd * (u - n * mean(u * n)) + dh,  dgain = sum_rows dy * n
//
// A row is held in registers (8 values a lane and step, h in 32 bits) between the sum of squares
// and the outputs, so every input is read once and every output written once; both kernels are bound by
// memory.  WARPS warps share a row: one for short rows, so that no row waits on a block barrier.  Measured on
// 65536 x 1152 bf16: forward with codes and values 108 us on the device (6.3 TB/s, 96% of a copy's rate), gradient 140 us (5.4 TB/s: its
// column sums leave registers for two blocks an SM); one row 2.0 us.  With the loads of a row in branches (rows off
// 16 bytes value by value) the same took 177 and 731.  Read-only loads leave the forward 64 registers in place of 80 and
// took 104 us, but are not for inputs that the kernel before still writes (heads_wait).
#pragma once
#include <math.h>

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
  MxOut mx;
};

#define NORM_THREADS 256
#define NORM_ROWS(WARPS) (8 / (WARPS))   // rows a block works on at a time

// sum (MAX: maximum) over the WARPS warps that share a row (their own named barrier; scr: WARPS floats of theirs)
template <int WARPS, bool MAX = false>
DEV float row_sum(float v, float* scr, int sub) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const float u = __shfl_xor_sync(0xffffffffu, v, o);
    v = MAX ? fmaxf(v, u) : v + u;
  }
  if constexpr (WARPS > 1) {
    const int w = (threadIdx.x >> 5) % WARPS;
    asm volatile("bar.sync %0, %1;" ::"r"(sub + 1), "r"(WARPS * 32) : "memory");   // the last sum has been read
    if ((threadIdx.x & 31) == 0) scr[w] = v;
    asm volatile("bar.sync %0, %1;" ::"r"(sub + 1), "r"(WARPS * 32) : "memory");
    v = 0.f;
#pragma unroll
    for (int i = 0; i < WARPS; ++i) v = MAX ? fmaxf(v, scr[i]) : v + scr[i];
  }
  return v;
}

// a lane's values of `row` of two matrices, all loads first (a null matrix gives zeros)
template <int TYPE, int WARPS, int NV, bool VEC>
DEV void row_load2(Raw8<TYPE> (&q)[NV], const void* p, int64_t ldp, Raw8<TYPE> (&u)[NV], const void* o, int64_t ldo, int64_t row, int t,
                   const NormArgs& a) {
  typedef typename Elem<TYPE>::T T;
  const T *ap = (const T*)p + (p ? row * ldp : 0), *ao = (const T*)o + (o ? row * ldo : 0);
  const int dp = p ? a.dim : 0, dn = o ? a.dim : 0;
  if constexpr (VEC) {
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = 8 * (t + i * 32 * WARPS);
      q[i].template load<true>(ap + c, dp - c);
      u[i].template load<true>(ao + c, dn - c);
    }
  } else {
    const uintptr_t hp = rows_end<T>(p, a.rows, ldp, a.dim), ho = rows_end<T>(o, a.rows, ldo, a.dim);
    Any8<TYPE> w[NV], v[NV];
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = 8 * (t + i * 32 * WARPS);
      w[i].begin(ap + c, dp - c, (uintptr_t)p, hp);
      v[i].begin(ao + c, dn - c, (uintptr_t)o, ho);
    }
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      w[i].end(q[i]);
      v[i].end(u[i]);
    }
  }
}

// 8 values at c of a row; all lanes of the warp together
template <int TYPE, bool VEC>
DEV void row_store(typename Elem<TYPE>::T* p, int c, int dim, const float (&v)[8]) {
  if constexpr (VEC || TYPE == SMG_EMB_F32) {
    store8<TYPE>(p + c, dim - c, VEC, v);
  } else {
    Raw8<TYPE> q;
#pragma unroll
    for (int i = 0; i < 8; ++i) q.t[i] = Elem<TYPE>::down(v[i]);
    store8_any((uint16_t*)(p + c), dim - c, c >> 3, q.w);
  }
}

// 1 / sqrt(ss / dim + eps) as a float and what it lacks (both together good to about 2^-45): the float's
// residual 1 - (v + ve) r^2, with v + ve the argument before its roundings, halved, corrects it (one Newton step).
DEV float rstd_of(float ss, float dim, float eps, float& low) {
  const float q = ss / dim, qe = __fmaf_rn(-q, dim, ss) / dim;
  const float v = q + eps, b = v - q, ve = ((q - (v - b)) + (eps - b)) + qe;
  const float r = 1.f / sqrtf(v), t = v * r, te = __fmaf_rn(v, r, -t);
  const float e = __fmaf_rn(-ve * r, r, __fmaf_rn(-te, r, __fmaf_rn(-t, r, 1.f)));
  low = r > 0.f ? 0.5f * r * e : 0.f;   // an infinity in the row: 1 / rms is 0 and lacks nothing
  return r;
}

// gain of 8 columns (VEC: on 16 bytes and n a multiple of 8)
template <bool VEC>
DEV void gain8(const float* p, int n, float (&g)[8]) {
  Raw8<SMG_EMB_F32> q;
  if (VEC || (n >= 8 && !((uintptr_t)p & 15))) q.template load<true>(p, n);
  else q.template load<false>(p, n);
#pragma unroll
  for (int i = 0; i < 8; ++i) g[i] = q.get(i);
}

template <int TYPE, int BITS, int WARPS, int NV, bool VEC>
__global__ void __launch_bounds__(NORM_THREADS) k_norm_add(NormArgs a) {
  typedef typename Elem<TYPE>::T T;
  __shared__ float scr[NORM_ROWS(WARPS)][WARPS];
  const int sub = threadIdx.x / (32 * WARPS), t = threadIdx.x % (32 * WARPS);
  const int64_t row = (int64_t)blockIdx.x * NORM_ROWS(WARPS) + sub;
  if (row >= a.rows) return;   // all warps of a row together
  heads_next();
  heads_wait();
  float h[NV][8];
  {
    Raw8<TYPE> x[NV], r[NV];
    row_load2<TYPE, WARPS, NV, VEC>(x, a.x, a.ldx, r, a.r, a.ldr, row, t, a);
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
      for (int k = 0; k < 8; ++k) h[i][k] = a.r ? x[i].get(k) + r[i].get(k) : x[i].get(k);
  }
  const auto squares = [&](float by) {   // sum of the row's (h * by)^2
    float sq[8];   // 8 short sums, then their tree: fewer roundings than one long sum
#pragma unroll
    for (int k = 0; k < 8; ++k) sq[k] = (h[0][k] * by) * (h[0][k] * by);
#pragma unroll
    for (int i = 1; i < NV; ++i)
#pragma unroll
      for (int k = 0; k < 8; ++k) sq[k] = __fmaf_rn(h[i][k] * by, h[i][k] * by, sq[k]);
    return row_sum<WARPS>(((sq[0] + sq[1]) + (sq[2] + sq[3])) + ((sq[4] + sq[5]) + (sq[6] + sq[7])), scr[sub], sub);
  };
  const float ss = squares(1.f);
  // The codes' rounding turns an error of the last place into one of a code, so 1 / rms goes in two parts: what
  // remains are the two products' own roundings (carrying those on too changed next to no code).
  float low;
  float rstd = rstd_of(ss, (float)a.dim, a.eps, low);
  if constexpr (TYPE != SMG_EMB_F16) {
    // Squares beyond 2^127, or so small that those below 2^-126 are missed (f16 has neither): once more with the row over a
    // power of two, by its largest magnitude or the root of eps, whichever is more.  All threads of a row together.
    if (!(rstd > 0.f && rstd < 0x1p40f)) {
      float m = 0.f;
#pragma unroll
      for (int i = 0; i < NV; ++i)
#pragma unroll
        for (int k = 0; k < 8; ++k) m = fmaxf(m, fabsf(h[i][k]));
      m = fmaxf(row_sum<WARPS, true>(m, scr[sub], sub), sqrtf(a.eps));
      if (m < INFINITY) {
        const float by = mx_two(127 - (int)(__float_as_uint(m) >> 23));
        rstd = rstd_of(squares(by), (float)a.dim, a.eps * by * by, low) * by;
        low *= by;
      }
    }
  }
  if (a.rstd && t == 0) a.rstd[row] = rstd;
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int j = t + i * 32 * WARPS, c = 8 * j, n = a.dim - c;
    if (a.h) row_store<TYPE, VEC>((T*)a.h + row * a.ldh, c, a.dim, h[i]);
    float g[8];
    gain8<VEC>(a.gain + c, n, g);
#pragma unroll
    for (int k = 0; k < 8; ++k) h[i][k] = __fmaf_rn(h[i][k], rstd, h[i][k] * low) * g[k];
    mx_emit<BITS>(a.mx, row, j, h[i]);
  }
}

// Gradients.  The blocks walk the rows with a stride; each lane keeps the dgain of its columns in
// registers, a block adds up its rows' sums at the end (in order) and writes one partial row, which
// k_norm_dgain adds up in block order.
template <int TYPE, int WARPS, int NV, bool VEC>
__global__ void __launch_bounds__(NORM_THREADS, NV <= 3 ? 2 : 1) k_norm_add_bwd(NormArgs a) {
  typedef typename Elem<TYPE>::T T;
  __shared__ float scr[NORM_ROWS(WARPS)][WARPS];
  extern __shared__ float acc[];   // NORM_ROWS x dim (WARPS < 8)
  const int sub = threadIdx.x / (32 * WARPS), t = threadIdx.x % (32 * WARPS);
  float dg[NV][8];
#pragma unroll
  for (int i = 0; i < NV; ++i)
#pragma unroll
    for (int k = 0; k < 8; ++k) dg[i][k] = 0.f;
  heads_next();
  heads_wait();
  const int64_t step = (int64_t)gridDim.x * NORM_ROWS(WARPS);
  for (int64_t row = (int64_t)blockIdx.x * NORM_ROWS(WARPS) + sub; row < a.rows; row += step) {
    Raw8<TYPE> x[NV], r[NV], y[NV], d[NV];
    row_load2<TYPE, WARPS, NV, VEC>(x, a.x, a.ldx, y, a.dy, a.ldy, row, t, a);
    row_load2<TYPE, WARPS, NV, VEC>(r, a.r, a.ldr, d, a.dh, a.ldh_in, row, t, a);
    const float rstd = a.rstd[row];
    float dot = 0.f;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = 8 * (t + i * 32 * WARPS);
      float g[8];
      gain8<VEC>(a.gain + c, a.dim - c, g);
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        const float n = (x[i].get(k) + r[i].get(k)) * rstd, dy = y[i].get(k);
        dg[i][k] = __fmaf_rn(dy, n, dg[i][k]);
        dot = __fmaf_rn(dy * g[k], n, dot);
      }
    }
    dot = row_sum<WARPS>(dot, scr[sub], sub) / (float)a.dim;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = 8 * (t + i * 32 * WARPS);
      float g[8], o[8];
      gain8<VEC>(a.gain + c, a.dim - c, g);
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        const float n = (x[i].get(k) + r[i].get(k)) * rstd;
        o[k] = __fmaf_rn(rstd, __fmaf_rn(-n, dot, y[i].get(k) * g[k]), d[i].get(k));
      }
      row_store<TYPE, VEC>((T*)a.dx + row * a.lddx, c, a.dim, o);
    }
  }
  float* part = a.part + (int64_t)blockIdx.x * a.dim;
  float* own = WARPS < 8 ? acc + sub * a.dim : part;
#pragma unroll
  for (int i = 0; i < NV; ++i)
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const int c = 8 * (t + i * 32 * WARPS) + k;
      if (c < a.dim) own[c] = dg[i][k];
    }
  if constexpr (WARPS < 8) {
    __syncthreads();
    for (int c = threadIdx.x; c < a.dim; c += NORM_THREADS) {
      float v = 0.f;
#pragma unroll
      for (int s = 0; s < NORM_ROWS(WARPS); ++s) v += acc[s * a.dim + c];
      part[c] = v;
    }
  }
}

// dgain[c] = sum of the parts: 32 columns a block, the parts over 32 warps, each in order
__global__ void __launch_bounds__(1024) k_norm_dgain(const float* part, int n_part, int dim, float* dgain) {
  __shared__ float s[32][33];
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5, c = blockIdx.x * 32 + lane;
  heads_next();
  heads_wait();
  float v = 0.f;
  if (c < dim)
    for (int p = w; p < n_part; p += 32) v += part[(int64_t)p * dim + c];
  s[w][lane] = v;
  __syncthreads();
  if (w == 0 && c < dim) {
    v = 0.f;
#pragma unroll
    for (int i = 0; i < 32; ++i) v += s[i][lane];
    dgain[c] = v;
  }
}
