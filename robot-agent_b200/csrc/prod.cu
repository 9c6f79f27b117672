// C ABI of the embedding heads' products (include/smg.h): ragged products by group, products of
// microscaled rows.
#include <algorithm>
#include <atomic>
#include <cmath>

#include "heads_host.h"
#include "k_few.cuh"
#include "k_prod.cuh"

#include <cudaTypedefs.h>

extern "C" PFN_cuTensorMapEncodeTiled_v12000 smg_tmap_encoder();   // smg.cu

// ------------------------------------------------------------------ ragged products
// sizes and offsets, the same for every product
static int prod_args(const char* who, const int32_t* off, int n_groups, int rows, int n, int k, int type, int out_type) {
  if (n_groups < 1 || rows < 0 || n < 1 || k < 1 || (!off && n_groups != 1))
    return fail(SMG_ERR_ARGS, "%s: bad sizes (n_groups %d, rows %d, n %d, k %d%s)", who, n_groups, rows, n, k, off ? "" : ", no offsets");
  // tiles and stages are counted in 32 bits, the last one whole
  if (rows > 0x7ffffe00) return fail(SMG_ERR_CAPACITY, "%s: too many rows for one call", who);
  if (n > 0x7ffffe00 || k > 0x7ffffe00) return fail(SMG_ERR_CAPACITY, "%s: too wide for one call (n %d, k %d)", who, n, k);
  if (n_groups > SMG_PROD_MAX_GROUPS) return fail(SMG_ERR_CAPACITY, "%s: %d groups, at most %d", who, n_groups, SMG_PROD_MAX_GROUPS);
  if (type != SMG_EMB_BF16 && type != SMG_EMB_F16) return fail(SMG_ERR_ARGS, "%s: inputs must be bf16 or f16", who);
  if (!type_ok(out_type)) return fail(SMG_ERR_ARGS, "%s: bad output type", who);
  return SMG_OK;
}

// a row operand of `len` elements a row: aligned for the tensor-core loads
static int operand(const char* who, const char* name, const void* p, int64_t ld, int64_t len, int64_t rows) {
  if (rows > 0 && !p) return fail(SMG_ERR_ARGS, "%s: %s is null", who, name);
  if (ld < len) return fail(SMG_ERR_ARGS, "%s: rows of %s overlap (leading dimension %lld, %lld values)", who, name, (long long)ld, (long long)len);
  if (!rows16(p, ld, SMG_EMB_BF16)) return fail(SMG_ERR_ARGS, "%s: %s must start on 16 bytes in every row", who, name);
  return SMG_OK;
}

// SMs of the current device, and which it is; 0 without one
static int sm_count(int* device) {
  static std::atomic<int> known[64];
  int dev = 0, n = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) return 0;
  *device = dev;
  if (dev < 64 && (n = known[dev].load(std::memory_order_relaxed)) > 0) return n;
  if (cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess) return 0;
  if (dev < 64) known[dev].store(n, std::memory_order_relaxed);
  return n;
}

// Rows for the tensor-core loads: `outer` groups of `rows` rows of `len` values (microscaled rows: bytes),
// boxes of 128 bytes x box_rows, 128-byte swizzle, zeros outside the array.
static int encode(const char* who, CUtensorMap* m, const void* p, bool bytes, int64_t len, int64_t rows, int64_t outer, int64_t ld,
                  int64_t outer_stride, int box_rows) {
  PFN_cuTensorMapEncodeTiled_v12000 fn = smg_tmap_encoder();
  if (!fn) return fail(SMG_ERR_DEVICE, "%s: cuTensorMapEncodeTiled unavailable", who);
  const int size = bytes ? 1 : 2;
  const cuuint64_t dim[3] = {(cuuint64_t)len, (cuuint64_t)std::max<int64_t>(rows, 1), (cuuint64_t)std::max<int64_t>(outer, 1)};
  const cuuint64_t str[2] = {(cuuint64_t)ld * size, (cuuint64_t)outer_stride * size};
  const cuuint32_t box[3] = {(cuuint32_t)(128 / size), (cuuint32_t)box_rows, 1};
  const cuuint32_t est[3] = {1, 1, 1};
  const CUresult r = fn(m, bytes ? CU_TENSOR_MAP_DATA_TYPE_UINT8 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, outer ? 3 : 2, const_cast<void*>(p),
                        dim, str, box, est, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                        CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) return fail(SMG_ERR_ARGS, "%s: tensor map refused (%d): a row or group is too far from the next", who, (int)r);
  return SMG_OK;
}

// A product's operands: A has the packed rows, B the groups' fixed rows (DW: the packed rows of x)
struct Operands {
  const void *a, *b;
  int64_t lda, ldb, b_stride;
  int64_t a_len, b_len;   // values of a row (microscaled: bytes)
};

template <int KIND, int BN, int FORM, bool PAIR = false>
static int launch(const char* who, const Operands& o, ProdArgs g, int type, cudaStream_t st) {
  using S = ProdShape<KIND, BN, PAIR>;
  constexpr bool bytes = KIND != 16;
  const int wide = FORM == FORM_Y || FORM == FORM_YT ? g.n : g.k;
  const int pr = PAIR ? 2 * PR_BM : PR_BM;   // rows of P in a tile
  g.p_tiles = FORM == FORM_YT || FORM == FORM_DW ? (g.n + pr - 1) / pr : 1;
  g.q_tiles = FORM == FORM_YT ? 1 : (wide + BN - 1) / BN;
  const int64_t per = (int64_t)g.p_tiles * g.q_tiles, rt = FORM == FORM_YT ? BN : pr;
  const int64_t row_tiles = FORM == FORM_DW ? g.n_groups : g.rows / rt + std::min(g.n_groups, g.rows);   // at most
  if (row_tiles * per > 0x7ff00000) return fail(SMG_ERR_CAPACITY, "%s: too many tiles for one call", who);
  CUtensorMap tA, tB;
  int r;
  if (FORM == FORM_DW) {
    r = encode(who, &tA, o.a, bytes, o.a_len, g.rows, 0, o.lda, 0, 64);
    if (!r) r = encode(who, &tB, o.b, bytes, o.b_len, g.rows, 0, o.ldb, 0, 64);
  } else {
    r = encode(who, &tA, o.a, bytes, o.a_len, g.rows, 0, o.lda, 0, FORM == FORM_YT ? BN : PR_BM);
    if (!r) r = encode(who, &tB, o.b, bytes, o.b_len, g.n, g.n_groups, o.ldb, g.n_groups > 1 ? o.b_stride : o.ldb * (int64_t)g.n,
                       FORM == FORM_Y ? S::QR : FORM == FORM_YT ? PR_BM : 64);
  }
  if (r) return r;
  // instruction descriptor: operand types (f16 0, bf16 1 with 32-bit sums in bits 4-5; e4m3 0, e2m1 1 with
  // power-of-two scales in bit 23) at 7 and 10, MN-major P and Q at 15 and 16, BN / 8 at 17, 128 / 16 at 24
  const uint32_t fmt = KIND == 16 ? (type == SMG_EMB_BF16) : KIND == 4;
  g.idesc = fmt << 7 | fmt << 10 | (uint32_t)(BN >> 3) << 17 | (uint32_t)(pr >> 4) << 24 | (KIND == 16 ? 1u << 4 : 1u << 23) |
            (FORM == FORM_DW ? 1u << 15 : 0u) | (FORM == FORM_DX || FORM == FORM_DW ? 1u << 16 : 0u);
  g.y_vec = rows16(g.y, g.ldy, g.y_type) && (FORM != FORM_DW || g.y_stride * size_of(g.y_type) % 16 == 0);
  static std::atomic<uint64_t> ready{0};   // devices on which this kernel has its shared memory
  int dev = 0;
  const int sms = sm_count(&dev);
  if (!sms) return fail(SMG_ERR_DEVICE, "%s: no usable device (%s)", who, cudaGetErrorString(cudaGetLastError()));
  if (dev > 63 || !(ready.load(std::memory_order_relaxed) >> dev & 1)) {
    const cudaError_t e = cudaFuncSetAttribute(k_prod<KIND, BN, FORM, PAIR>, cudaFuncAttributeMaxDynamicSharedMemorySize, S::SMEM);
    if (e != cudaSuccess) return fail(SMG_ERR_DEVICE, "%s: %s", who, cudaGetErrorString(e));
    if (dev < 64) ready.fetch_or(1ull << dev, std::memory_order_relaxed);
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(PAIR ? 2 * std::min<int64_t>(sms / 2, row_tiles * per) : std::min<int64_t>(sms, row_tiles * per)));
  cfg.blockDim = dim3(PR_THREADS(KIND, PAIR));
  cfg.dynamicSmemBytes = S::SMEM;
  cfg.stream = st;
  cudaLaunchAttribute at[2];
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;   // as launch_next
  at[0].val.programmaticStreamSerializationAllowed = 1;
  at[1].id = cudaLaunchAttributeClusterDimension;
  at[1].val.clusterDim.x = 2;
  at[1].val.clusterDim.y = at[1].val.clusterDim.z = 1;
  cfg.attrs = at;
  cfg.numAttrs = PAIR ? 2 : 1;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, k_prod<KIND, BN, FORM, PAIR>, tA, tB, g);
  if (e != cudaSuccess) return fail(SMG_ERR_DEVICE, "%s: %s", who, cudaGetErrorString(e));
  return SMG_OK;
}

static ProdArgs prod_fill(const int32_t* off, int n_groups, int rows, int n, int k, void* y, int64_t ldy, int64_t y_stride, int y_type,
                          int32_t* err) {
  ProdArgs g = {};
  g.off = off; g.n_groups = n_groups; g.rows = rows; g.n = n; g.k = k;
  g.y = y; g.ldy = ldy; g.y_stride = y_stride; g.y_type = y_type; g.err = err;
  return g;
}

// Which tile: the one with the least estimated time, (rounds of tiles over the SMs) x (rows of operands
// that a CTA loads for a tile) / (bytes a cycle that it gets), since every form is held up by its loads and their
// way through shared memory: the 128 x 256 tile of one CTA takes its 384 rows at 55 bytes a cycle
// and SM, the pair's 256 rows at 45; the MMAs would take 100.  The groups'
// sizes are known on the device only: they are taken to be spread about their mean, half a tile of each
// group left over.
struct TileCost {
  int64_t rows;
  int groups, sms;
  double of(int rt, int64_t fixed, int units, int loaded) const {
    const double full = (double)std::min<int64_t>(groups, rows), m = rows / full;
    const double row_tiles = groups == 1 ? std::ceil(m / rt) : full * std::max(1.0, m / rt + 0.5);
    return std::ceil(row_tiles * fixed / units) * loaded;
  }
  double narrow(int64_t wide, int bn) const { return of(bn, (wide + PR_BM - 1) / PR_BM, sms, PR_BM + bn); }    // FORM_YT
  double single(int64_t wide, int bn) const { return of(PR_BM, (wide + bn - 1) / bn, sms, PR_BM + bn); }
  double pair(int64_t wide, int bn) const { return of(2 * PR_BM, (wide + bn - 1) / bn, sms / 2, PR_BM + bn / 2) * 55 / 45; }
};

extern "C" {

int smg_group_product(const void* x, int64_t ldx, const void* w, int64_t ldw, int64_t w_stride, const int32_t* off, int n_groups,
                      int rows, int n, int k, int type, void* y, int64_t ldy, int y_type, int32_t* err, void* stream) {
  const char* who = "smg_group_product";
  if (int r = prod_args(who, off, n_groups, rows, n, k, type, y_type)) return r;
  if (int r = operand(who, "x", x, ldx, k, rows)) return r;
  if (int r = operand(who, "w", w, ldw, k, n)) return r;
  if (n_groups > 1)
    if (int r = operand(who, "w (from group to group)", w, w_stride, (int64_t)(n - 1) * ldw + k, n)) return r;
  if (int r = out_rows(who, y, ldy, n, rows)) return r;
  if (rows == 0) return SMG_OK;
  const ProdArgs g = prod_fill(off, n_groups, rows, n, k, y, ldy, 0, y_type, err);
  const Operands o = {x, w, ldx, ldw, w_stride, k, k};
  const cudaStream_t st = (cudaStream_t)stream;
  // Up to 8 rows a group in the mean, and weights that do not make it a matter of bandwidth.  Both sides measured with
  // the weights in L2 (one set, replayed): on 1 to 8 rows of one group (n = k = 1152) 2.6 us against 6.8, on 24
  // groups of 512 x 1152 (28 MB) 7.2 against 7.5, on 42 (50 MB) 11.3 against 11.7; on 64 groups (75 MB) 15.2 against
  // 12.3, and on 64 of 1152 x 1152 42 against 31.  From memory (sets in turn) this side takes 9.1 us on 24 groups and
  // 14.5 on 42, the other 15.7 on 64: where the two meet then was not measured.
  if ((int64_t)rows <= FEW_ROWS * (int64_t)n_groups && (int64_t)n_groups * n * k <= 24ll << 20) {
    const FewArgs a = {off, n_groups, rows, n, k, x, w, ldx, ldw, w_stride, y, ldy, y_type, err};
    const dim3 grid((n + FEW_W - 1) / FEW_W, n_groups);
    return launch_next(who, type == SMG_EMB_BF16 ? k_few<SMG_EMB_BF16> : k_few<SMG_EMB_F16>, grid, FEW_WARPS * 32, 0, st, a);
  }
  int dev;
  const TileCost c = {rows, n_groups, std::max(sm_count(&dev), 2)};
  const double t[] = {c.narrow(n, 32), c.narrow(n, 64), c.narrow(n, 128), c.single(n, 192), c.single(n, 256), c.pair(n, 256)};
  switch (std::min_element(t, t + 6) - t) {
    case 0: return launch<16, 32, FORM_YT>(who, o, g, type, st);
    case 1: return launch<16, 64, FORM_YT>(who, o, g, type, st);
    case 2: return launch<16, 128, FORM_YT>(who, o, g, type, st);
    case 3: return launch<16, 192, FORM_Y>(who, o, g, type, st);
    case 4: return launch<16, 256, FORM_Y>(who, o, g, type, st);
    default: return launch<16, 256, FORM_Y, true>(who, o, g, type, st);
  }
}

int smg_group_product_dx(const void* dy, int64_t lddy, const void* w, int64_t ldw, int64_t w_stride, const int32_t* off,
                         int n_groups, int rows, int n, int k, int type, void* dx, int64_t lddx, int dx_type, int32_t* err,
                         void* stream) {
  const char* who = "smg_group_product_dx";
  if (int r = prod_args(who, off, n_groups, rows, n, k, type, dx_type)) return r;
  if (int r = operand(who, "dy", dy, lddy, n, rows)) return r;
  if (int r = operand(who, "w", w, ldw, k, n)) return r;
  if (n_groups > 1)
    if (int r = operand(who, "w (from group to group)", w, w_stride, (int64_t)(n - 1) * ldw + k, n)) return r;
  if (int r = out_rows(who, dx, lddx, k, rows)) return r;
  if (rows == 0) return SMG_OK;
  const ProdArgs g = prod_fill(off, n_groups, rows, n, k, dx, lddx, 0, dx_type, err);
  const Operands o = {dy, w, lddy, ldw, w_stride, n, k};
  const cudaStream_t st = (cudaStream_t)stream;
  int dev;
  const TileCost c = {rows, n_groups, std::max(sm_count(&dev), 2)};
  const double t[] = {c.single(k, 128), c.single(k, 192), c.single(k, 256), c.pair(k, 256)};
  switch (std::min_element(t, t + 4) - t) {
    case 0: return launch<16, 128, FORM_DX>(who, o, g, type, st);
    case 1: return launch<16, 192, FORM_DX>(who, o, g, type, st);
    case 2: return launch<16, 256, FORM_DX>(who, o, g, type, st);
    default: return launch<16, 256, FORM_DX, true>(who, o, g, type, st);
  }
}

int smg_group_product_dw(const void* dy, int64_t lddy, const void* x, int64_t ldx, const int32_t* off, int n_groups, int rows,
                         int n, int k, int type, void* dw, int64_t lddw, int64_t dw_stride, int dw_type, int32_t* err,
                         void* stream) {
  const char* who = "smg_group_product_dw";
  if (int r = prod_args(who, off, n_groups, rows, n, k, type, dw_type)) return r;
  if (int r = operand(who, "dy", dy, lddy, n, rows)) return r;
  if (int r = operand(who, "x", x, ldx, k, rows)) return r;
  if (int r = out_rows(who, dw, lddw, k, n)) return r;
  if (n_groups > 1 && dw_stride < (int64_t)(n - 1) * lddw + k) return fail(SMG_ERR_ARGS, "%s: the groups of dw overlap", who);
  ProdArgs g = prod_fill(off, n_groups, rows, n, k, dw, lddw, dw_stride, dw_type, err);
  Operands o = {dy, x, lddy, ldx, 0, n, k};
  if (rows == 0) {   // every group is empty and nothing is loaded: dw itself stands in for the operands
    if (!on16(dw)) return fail(SMG_ERR_ARGS, "%s: without rows dw must start on 16 bytes", who);
    o.a = o.b = dw;
    o.lda = (n + 7) / 8 * 8;
    o.ldb = (k + 7) / 8 * 8;
  }
  // every group has the same tiles, only their lengths differ
  const cudaStream_t st = (cudaStream_t)stream;
  int dev;
  const int sms = std::max(sm_count(&dev), 2);
  const auto cost = [&](int rt, int bn, int units, int loaded) {
    return std::ceil((double)n_groups * ((n + rt - 1) / rt) * ((k + bn - 1) / bn) / units) * loaded;
  };
  const double t[] = {cost(128, 128, sms, 256), cost(128, 256, sms, 384), cost(256, 256, sms / 2, 256) * 55 / 45};
  switch (std::min_element(t, t + 3) - t) {
    case 0: return launch<16, 128, FORM_DW>(who, o, g, type, st);
    case 1: return launch<16, 256, FORM_DW>(who, o, g, type, st);
    default: return launch<16, 256, FORM_DW, true>(who, o, g, type, st);
  }
}

int smg_mx_product(const uint8_t* a_codes, const uint8_t* a_scales, const uint8_t* b_codes, const uint8_t* b_scales,
                   const int32_t* off, int n_groups, int rows, int n, int k, int bits, void* y, int64_t ldy, int y_type,
                   int32_t* err, void* stream) {
  const char* who = "smg_mx_product";
  if (int r = prod_args(who, off, n_groups, rows, n, k, SMG_EMB_BF16, y_type)) return r;
  if (int r = mx_args(who, rows, k, bits, a_codes, a_scales)) return r;
  if (int r = mx_args(who, n, k, bits, b_codes, b_scales)) return r;
  if (int r = out_rows(who, y, ldy, n, rows)) return r;
  if (rows == 0) return SMG_OK;
  if (!a_codes || !b_codes) return fail(SMG_ERR_ARGS, "%s: no codes", who);
  ProdArgs g = prod_fill(off, n_groups, rows, n, k, y, ldy, 0, y_type, err);
  const MxOut m = mx_rows(k, nullptr, nullptr, nullptr);
  g.sa = a_scales; g.sb = b_scales; g.pitch = m.pitch;
  const int64_t len = (int64_t)m.kb * 4 * bits;
  const Operands o = {a_codes, b_codes, len, len, len * n, len, len};
  const cudaStream_t st = (cudaStream_t)stream;
  int dev;
  const TileCost c = {rows, n_groups, std::max(sm_count(&dev), 2)};
  const double t[] = {c.narrow(n, 32), c.narrow(n, 64), c.narrow(n, 128), c.single(n, 192), c.pair(n, 192)};
  switch (std::min_element(t, t + 5) - t) {
    case 0: return bits == 4 ? launch<4, 32, FORM_YT>(who, o, g, 0, st) : launch<8, 32, FORM_YT>(who, o, g, 0, st);
    case 1: return bits == 4 ? launch<4, 64, FORM_YT>(who, o, g, 0, st) : launch<8, 64, FORM_YT>(who, o, g, 0, st);
    case 2: return bits == 4 ? launch<4, 128, FORM_YT>(who, o, g, 0, st) : launch<8, 128, FORM_YT>(who, o, g, 0, st);
    case 3: return bits == 4 ? launch<4, 192, FORM_Y>(who, o, g, 0, st) : launch<8, 192, FORM_Y>(who, o, g, 0, st);
    default: return bits == 4 ? launch<4, 192, FORM_Y, true>(who, o, g, 0, st) : launch<8, 192, FORM_Y, true>(who, o, g, 0, st);
  }
}

}   // extern "C"
