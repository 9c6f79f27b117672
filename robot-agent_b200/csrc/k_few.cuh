// y = x w_g^T for a few rows per group: one pass over w, straight from memory into mma fragments.
//
// With r rows a group every weight is used r times, 2 r operations for 2 bytes: the time is that of
// reading w, and what the tcgen05 form sets up (tensor memory, barriers, tensor maps, a ring through shared
// memory) is what remains to be saved.  A block takes 16 rows of w_g and up to 8 rows of x at a time; its
// warps share the k axis, 32 values a step.  The order of k within an mma is free as long as both operands
// have the same: lane l holds 8 consecutive values (one 16-byte load) of rows l / 4 and l / 4 + 8 of w, and of row l / 4 of
// x, at 8 (l % 4), and they serve as the fragments of two m16n8k16 products.  The warps' sums are added in warp order.
// Larger groups than 8 rows go round again (w_g's rows then come from the cache), one round after the other: 512 rows all
// in one of 64 groups of 512 x 768 take 66 us, 8 in each 14.  Measured: one row, k = 768, n = 256: 2.1 us (the tcgen05
// form 7.3); 24 groups of 512 x 1152 (28 MB): 9.1 us from memory, 6.3 where L2 holds them.
#pragma once
#include "k_mx.cuh"

#define FEW_W 16
#define FEW_WARPS 8
#define FEW_ROWS 8
#define FEW_STEPS 5   // loads in flight: 5 x 3 x 16 bytes a lane, 1280 values of k a block

struct FewArgs {
  const int32_t* off;
  int n_groups, rows, n, k;
  const void *x, *w;
  int64_t ldx, ldw, w_stride;
  void* y;
  int64_t ldy;
  int y_type;
  int32_t* err;
};

template <int TYPE>
DEV void few_mma(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  if constexpr (TYPE == SMG_EMB_BF16)
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  else
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// 8 values at c of a row of k (16-byte aligned); zeros past k and where the row is not there
template <int TYPE>
DEV uint4 few_load(const typename Elem<TYPE>::T* row, int c, int k, bool there) {
  if (!there || c >= k) return make_uint4(0, 0, 0, 0);
  if (c + 8 <= k) return *(const uint4*)(row + c);
  Raw8<TYPE> q;
  q.template load<false>(row + c, k - c);
  return q.q[0];
}

template <int TYPE>
__global__ void __launch_bounds__(FEW_WARPS * 32) k_few(FewArgs a) {
  typedef typename Elem<TYPE>::T T;
  __shared__ float part[FEW_WARPS][FEW_ROWS][FEW_W + 1];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = blockIdx.y, j0 = blockIdx.x * FEW_W;
  heads_next();
  heads_wait();
  int r0 = 0, r1 = a.rows;
  if (a.off) {
    r0 = a.off[g];
    r1 = a.off[g + 1];
    const bool good = r0 >= 0 && r1 >= r0 && r1 <= a.rows;
    if (blockIdx.x == 0 && threadIdx.x == 0 && a.err && (!good || (g == 0 && r0 != 0) || (g == a.n_groups - 1 && r1 != a.rows)))
      atomicOr(a.err, SMG_PROD_OFFSETS);
    if (!good) return;
  }
  const int q = lane >> 2;
  const T* w = (const T*)a.w + g * a.w_stride;
  // a row of w past the last is read as the last and not stored
  const T *w0 = w + (int64_t)min(j0 + q, a.n - 1) * a.ldw, *w1 = w + (int64_t)min(j0 + q + 8, a.n - 1) * a.ldw;
  for (int r = r0; r < r1; r += FEW_ROWS) {
    const bool there = r + q < r1;
    const T* x = (const T*)a.x + (int64_t)(there ? r + q : r) * a.ldx;
    float d[4] = {0.f, 0.f, 0.f, 0.f};
    // by warp, not by lane: an mma needs all 32 lanes
    for (int k0 = warp * 32; k0 < a.k; k0 += FEW_STEPS * FEW_WARPS * 32) {
      uint4 u[FEW_STEPS], v[FEW_STEPS], b[FEW_STEPS];
#pragma unroll
      for (int i = 0; i < FEW_STEPS; ++i) {   // all loads first
        const int c = k0 + i * FEW_WARPS * 32 + (lane & 3) * 8;
        u[i] = few_load<TYPE>(w0, c, a.k, true);
        v[i] = few_load<TYPE>(w1, c, a.k, true);
        b[i] = few_load<TYPE>(x, c, a.k, there);
      }
      __syncwarp();
#pragma unroll
      for (int i = 0; i < FEW_STEPS; ++i) {
        few_mma<TYPE>(d, u[i].x, v[i].x, u[i].y, v[i].y, b[i].x, b[i].y);
        few_mma<TYPE>(d, u[i].z, v[i].z, u[i].w, v[i].w, b[i].z, b[i].w);
      }
    }
    // d: rows q and q + 8 of w, rows 2 (l % 4) and the next of x
    const int n = (lane & 3) * 2;
    part[warp][n][q] = d[0];
    part[warp][n + 1][q] = d[1];
    part[warp][n][q + 8] = d[2];
    part[warp][n + 1][q + 8] = d[3];
    __syncthreads();
    if (threadIdx.x < FEW_ROWS * FEW_W) {
      const int row = threadIdx.x / FEW_W, j = threadIdx.x % FEW_W;
      float s = 0.f;
#pragma unroll
      for (int i = 0; i < FEW_WARPS; ++i) s += part[i][row][j];
      if (r + row < r1 && j0 + j < a.n) {
        const int64_t o = (int64_t)(r + row) * a.ldy + j0 + j;
        if (a.y_type == SMG_EMB_F32) ((float*)a.y)[o] = s;
        else if (a.y_type == SMG_EMB_BF16) ((__nv_bfloat16*)a.y)[o] = __float2bfloat16_rn(s);
        else ((__half*)a.y)[o] = __float2half_rn(s);
      }
    }
    __syncthreads();
  }
}
