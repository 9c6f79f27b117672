// C ABI of the embedding heads (include/smg.h): ragged products by group, microscaled rows, the
// residual norm.
#include <cuda_runtime.h>
#include <stdarg.h>
#include <stdio.h>

#include "k_norm.cuh"
#include "k_prod.cuh"

int smg_set_error(int code, const char* msg);   // smg.cu: records msg for smg_last_error

static int fail(int code, const char* fmt, ...) {
  char msg[256];
  va_list ap;
  va_start(ap, fmt);
  vsnprintf(msg, sizeof msg, fmt, ap);
  va_end(ap);
  return smg_set_error(code, msg);
}

static int launched(const char* who) {
  const cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? SMG_OK : fail(SMG_ERR_DEVICE, "%s: %s", who, cudaGetErrorString(e));
}

static bool on16(const void* p) { return !((uintptr_t)p & 15); }
static bool type_ok(int t) { return t == SMG_EMB_F32 || t == SMG_EMB_BF16 || t == SMG_EMB_F16; }
static int size_of(int t) { return t == SMG_EMB_F32 ? 4 : 2; }
// rows of ld elements starting at p all start on 16 bytes
static bool rows16(const void* p, int64_t ld, int type) { return on16(p) && ld * size_of(type) % 16 == 0; }

// ------------------------------------------------------------------ ragged products
// sizes and offsets, the same for every product
static int prod_args(const char* who, const int32_t* off, int n_groups, int rows, int n, int k, int type, int out_type) {
  if (n_groups < 1 || rows < 0 || n < 1 || k < 1 || (!off && n_groups != 1))
    return fail(SMG_ERR_ARGS, "%s: bad sizes (n_groups %d, rows %d, n %d, k %d%s)", who, n_groups, rows, n, k, off ? "" : ", no offsets");
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

static int out_rows(const char* who, const void* p, int64_t ld, int64_t len, int64_t rows) {
  if (rows > 0 && !p) return fail(SMG_ERR_ARGS, "%s: the output is null", who);
  if (ld < len) return fail(SMG_ERR_ARGS, "%s: the output's rows overlap", who);
  return SMG_OK;
}

static ProdArgs prod_fill(const int32_t* off, int n_groups, int rows, int n, int k, const void* a, int64_t lda, const void* b, int64_t ldb,
                          int64_t b_stride, void* y, int64_t ldy, int64_t y_stride, int y_type, int32_t* err) {
  ProdArgs g = {};
  g.off = off; g.n_groups = n_groups; g.rows = rows; g.n = n; g.k = k;
  g.a = a; g.lda = lda; g.b = b; g.ldb = ldb; g.b_stride = b_stride;
  g.y = y; g.ldy = ldy; g.y_stride = y_stride; g.y_type = y_type; g.err = err;
  return g;
}

static int grid_for(int64_t threads) {
  const int64_t b = (threads + 255) / 256;
  return (int)(b < 1 ? 1 : b > 148 * 64 ? 148 * 64 : b);
}

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
  const ProdArgs g = prod_fill(off, n_groups, rows, n, k, x, ldx, w, ldw, w_stride, y, ldy, 0, y_type, err);
  const int grid = grid_for((int64_t)rows * n);
  if (type == SMG_EMB_BF16) k_prod_y<SMG_EMB_BF16><<<grid, 256, 0, (cudaStream_t)stream>>>(g);
  else k_prod_y<SMG_EMB_F16><<<grid, 256, 0, (cudaStream_t)stream>>>(g);
  return launched(who);
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
  const ProdArgs g = prod_fill(off, n_groups, rows, n, k, dy, lddy, w, ldw, w_stride, dx, lddx, 0, dx_type, err);
  const int grid = grid_for((int64_t)rows * k);
  if (type == SMG_EMB_BF16) k_prod_dx<SMG_EMB_BF16><<<grid, 256, 0, (cudaStream_t)stream>>>(g);
  else k_prod_dx<SMG_EMB_F16><<<grid, 256, 0, (cudaStream_t)stream>>>(g);
  return launched(who);
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
  const ProdArgs g = prod_fill(off, n_groups, rows, n, k, dy, lddy, x, ldx, 0, dw, lddw, dw_stride, dw_type, err);
  const int grid = grid_for((int64_t)n_groups * n * k);
  if (type == SMG_EMB_BF16) k_prod_dw<SMG_EMB_BF16><<<grid, 256, 0, (cudaStream_t)stream>>>(g);
  else k_prod_dw<SMG_EMB_F16><<<grid, 256, 0, (cudaStream_t)stream>>>(g);
  return launched(who);
}

// ------------------------------------------------------------------ microscaled rows
static MxOut mx_rows(int k, const uint8_t* codes, const uint8_t* scales, uint16_t* values) {
  MxOut o;
  o.codes = const_cast<uint8_t*>(codes); o.scales = const_cast<uint8_t*>(scales); o.values = (__nv_bfloat16*)values;
  o.dim = k; o.kb = (k + 31) / 32; o.pitch = (o.kb + 3) / 4 * 4;
  return o;
}

static int mx_args(const char* who, int rows, int k, int bits, const uint8_t* codes, const uint8_t* scales) {
  if (rows < 0 || k < 1 || k > (1 << 24)) return fail(SMG_ERR_ARGS, "%s: bad sizes (rows %d, %d values a row)", who, rows, k);
  if (bits != 4 && bits != 8) return fail(SMG_ERR_ARGS, "%s: bits must be 4 or 8", who);
  if (rows > 0 && (!codes != !scales)) return fail(SMG_ERR_ARGS, "%s: codes and scales go together", who);
  if (!on16(codes) || !on16(scales)) return fail(SMG_ERR_ARGS, "%s: codes and scales must start on 16 bytes", who);
  return SMG_OK;
}

static int blocks256(const char* who, int64_t threads, unsigned* grid) {
  const int64_t b = (threads + 255) / 256;
  if (b > 0x7fffffff) return fail(SMG_ERR_CAPACITY, "%s: too many values for one call", who);
  *grid = (unsigned)b;
  return SMG_OK;
}

#define BY_TYPE(type, CALL)                               \
  do {                                                    \
    if ((type) == SMG_EMB_F32) { CALL(SMG_EMB_F32); }     \
    else if ((type) == SMG_EMB_BF16) { CALL(SMG_EMB_BF16); } \
    else { CALL(SMG_EMB_F16); }                           \
  } while (0)

int smg_mx_quantise(const void* x, int64_t ldx, int rows, int k, int type, int bits, uint8_t* codes, uint8_t* scales,
                    uint16_t* values, void* stream) {
  const char* who = "smg_mx_quantise";
  if (int r = mx_args(who, rows, k, bits, codes, scales)) return r;
  if (!type_ok(type)) return fail(SMG_ERR_ARGS, "%s: bad input type", who);
  if (rows == 0) return SMG_OK;
  if (!x || (!codes && !values) || (values && ((uintptr_t)values & (k % 8 ? 1 : 15))))
    return fail(SMG_ERR_ARGS, "%s: no input, no output, or values off their alignment", who);
  const MxOut o = mx_rows(k, codes, scales, values);
  const int64_t n = (int64_t)rows * o.pitch * 4;
  const bool vec = rows16(x, ldx, type);
  unsigned grid;
  if (int r = blocks256(who, n, &grid)) return r;
#define CALL(TY)                                                                                                           \
  if (bits == 4) k_mx_quantise<TY, 4><<<grid, 256, 0, (cudaStream_t)stream>>>((const Elem<TY>::T*)x, ldx, n, vec, o);        \
  else k_mx_quantise<TY, 8><<<grid, 256, 0, (cudaStream_t)stream>>>((const Elem<TY>::T*)x, ldx, n, vec, o)
  BY_TYPE(type, CALL);
#undef CALL
  return launched(who);
}

int smg_mx_values(const uint8_t* codes, const uint8_t* scales, int rows, int k, int bits, void* out, int64_t ld, int out_type,
                  void* stream) {
  const char* who = "smg_mx_values";
  if (int r = mx_args(who, rows, k, bits, codes, scales)) return r;
  if (!type_ok(out_type)) return fail(SMG_ERR_ARGS, "%s: bad output type", who);
  if (int r = out_rows(who, out, ld, k, rows)) return r;
  if (rows == 0) return SMG_OK;
  if (!codes) return fail(SMG_ERR_ARGS, "%s: no codes", who);
  const MxOut o = mx_rows(k, codes, scales, nullptr);
  const int64_t n = (int64_t)rows * o.kb * 4;
  const bool vec = rows16(out, ld, out_type);
  unsigned grid;
  if (int r = blocks256(who, n, &grid)) return r;
#define CALL(TY)                                                                                                  \
  if (bits == 4) k_mx_values<TY, 4><<<grid, 256, 0, (cudaStream_t)stream>>>(o, n, (Elem<TY>::T*)out, ld, vec);      \
  else k_mx_values<TY, 8><<<grid, 256, 0, (cudaStream_t)stream>>>(o, n, (Elem<TY>::T*)out, ld, vec)
  BY_TYPE(out_type, CALL);
#undef CALL
  return launched(who);
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
  ProdArgs g = prod_fill(off, n_groups, rows, n, k, a_codes, 0, b_codes, 0, 0, y, ldy, 0, y_type, err);
  const MxOut o = mx_rows(k, nullptr, nullptr, nullptr);
  g.sa = a_scales; g.sb = b_scales; g.pitch = o.pitch; g.row_bytes = o.kb * 4 * bits;
  const int grid = grid_for((int64_t)rows * n);
  if (bits == 4) k_prod_mx<4><<<grid, 256, 0, (cudaStream_t)stream>>>(g);
  else k_prod_mx<8><<<grid, 256, 0, (cudaStream_t)stream>>>(g);
  return launched(who);
}

// ------------------------------------------------------------------ residual norm
// Warps a row and register steps of 8 values a lane: the smallest that hold the row.  One warp up
// to 2048 values; then the row goes over 4 or 8 warps, so that a lane keeps to 64 values.
#define NORM_MAX_DIM 16384
#define NORM_PARTS 296   // blocks of the gradient kernel, two an SM

#define BY_DIM(lanes8, CALL)                    \
  do {                                          \
    const int s_ = ((lanes8) + 31) / 32;        \
    if (s_ <= 1) { CALL(1, 1); }                \
    else if (s_ <= 2) { CALL(1, 2); }           \
    else if (s_ <= 3) { CALL(1, 3); }           \
    else if (s_ <= 4) { CALL(1, 4); }           \
    else if (s_ <= 5) { CALL(1, 5); }           \
    else if (s_ <= 6) { CALL(1, 6); }           \
    else if (s_ <= 8) { CALL(1, 8); }           \
    else if (s_ <= 16) { CALL(4, 4); }          \
    else if (s_ <= 32) { CALL(8, 4); }          \
    else { CALL(8, 8); }                        \
  } while (0)

int smg_norm_add(const void* x, int64_t ldx, const void* r, int64_t ldr, const float* gain, int rows, int dim, int type, float eps,
                 void* h, int64_t ldh, float* rstd, int bits, uint8_t* codes, uint8_t* scales, uint16_t* values, void* stream) {
  const char* who = "smg_norm_add";
  if (int e = mx_args(who, rows, dim, bits, codes, scales)) return e;
  if (!type_ok(type)) return fail(SMG_ERR_ARGS, "%s: bad input type", who);
  if (dim > NORM_MAX_DIM) return fail(SMG_ERR_CAPACITY, "%s: %d values a row, at most %d", who, dim, NORM_MAX_DIM);
  if (h && ldh < dim) return fail(SMG_ERR_ARGS, "%s: the rows of h overlap", who);
  if (rows == 0) return SMG_OK;
  if (!x || (!gain && (codes || values))) return fail(SMG_ERR_ARGS, "%s: x or gain is null", who);
  if (values && ((uintptr_t)values & (dim % 8 ? 1 : 15))) return fail(SMG_ERR_ARGS, "%s: values off their alignment", who);
  NormArgs a = {};
  a.x = x; a.ldx = ldx; a.r = r; a.ldr = ldr; a.gain = gain; a.h = h; a.ldh = ldh; a.rstd = rstd;
  a.rows = rows; a.dim = dim; a.eps = eps;
  a.vec = rows16(x, ldx, type) && (!r || rows16(r, ldr, type)) && (!h || rows16(h, ldh, type));
  a.gvec = on16(gain);
  a.mx = mx_rows(dim, codes, scales, values);
  const int b = codes || values ? bits : 0;
  const int lanes = a.mx.pitch * 4;   // lanes that the row's blocks need, the scales' padding with them
#define LAUNCH(T, W, NV)                                                                                       \
  const unsigned grid = (unsigned)((rows + NORM_ROWS(W) - 1) / NORM_ROWS(W));                                  \
  if (b == 4) k_norm_add<T, 4, W, NV><<<grid, NORM_THREADS, 0, (cudaStream_t)stream>>>(a);                    \
  else if (b == 8) k_norm_add<T, 8, W, NV><<<grid, NORM_THREADS, 0, (cudaStream_t)stream>>>(a);               \
  else k_norm_add<T, 0, W, NV><<<grid, NORM_THREADS, 0, (cudaStream_t)stream>>>(a)
#define CALL32(W, NV) LAUNCH(SMG_EMB_F32, W, NV)
#define CALLBF(W, NV) LAUNCH(SMG_EMB_BF16, W, NV)
#define CALLHF(W, NV) LAUNCH(SMG_EMB_F16, W, NV)
  if (type == SMG_EMB_F32) BY_DIM(lanes, CALL32);
  else if (type == SMG_EMB_BF16) BY_DIM(lanes, CALLBF);
  else BY_DIM(lanes, CALLHF);
#undef LAUNCH
  return launched(who);
}

int64_t smg_norm_add_bwd_work(int dim) { return dim < 1 ? 0 : (int64_t)NORM_PARTS * dim * 4; }

int smg_norm_add_bwd(const void* dy, int64_t lddy, const void* x, int64_t ldx, const void* r, int64_t ldr, const float* rstd,
                     const float* gain, const void* dh, int64_t lddh, int rows, int dim, int type, void* dx, int64_t lddx,
                     float* dgain, void* work, void* stream) {
  const char* who = "smg_norm_add_bwd";
  if (rows < 0 || dim < 1) return fail(SMG_ERR_ARGS, "%s: bad sizes (rows %d, dim %d)", who, rows, dim);
  if (!type_ok(type)) return fail(SMG_ERR_ARGS, "%s: bad type", who);
  if (dim > NORM_MAX_DIM) return fail(SMG_ERR_CAPACITY, "%s: %d values a row, at most %d", who, dim, NORM_MAX_DIM);
  if (!dgain || !gain || (rows > 0 && (!dy || !x || !rstd || !dx || !work))) return fail(SMG_ERR_ARGS, "%s: a pointer is null", who);
  if (!on16(work)) return fail(SMG_ERR_ARGS, "%s: work must start on 16 bytes", who);
  if (lddx < dim) return fail(SMG_ERR_ARGS, "%s: the rows of dx overlap", who);
  NormArgs a = {};
  a.x = x; a.ldx = ldx; a.r = r; a.ldr = ldr; a.dy = dy; a.ldy = lddy; a.dh = dh; a.ldh_in = lddh;
  a.gain = gain; a.rstd = const_cast<float*>(rstd); a.dx = dx; a.lddx = lddx; a.part = (float*)work;
  a.rows = rows; a.dim = dim;
  a.vec = rows16(x, ldx, type) && (!r || rows16(r, ldr, type)) && rows16(dy, lddy, type) && (!dh || rows16(dh, lddh, type)) &&
          rows16(dx, lddx, type);
  a.gvec = on16(gain);
  const cudaStream_t st = (cudaStream_t)stream;
  int parts = 0;
  if (rows > 0) {
#define LAUNCH(T, W, NV)                                                                            \
  parts = (rows + NORM_ROWS(W) - 1) / NORM_ROWS(W);                                                 \
  if (parts > NORM_PARTS) parts = NORM_PARTS;                                                       \
  k_norm_add_bwd<T, W, NV><<<parts, NORM_THREADS, NORM_ROWS(W) > 1 ? dim * 4 : 0, st>>>(a)
    if (type == SMG_EMB_F32) BY_DIM((dim + 7) / 8, CALL32);
    else if (type == SMG_EMB_BF16) BY_DIM((dim + 7) / 8, CALLBF);
    else BY_DIM((dim + 7) / 8, CALLHF);
#undef LAUNCH
  }
  k_norm_dgain<<<(dim + 31) / 32, 256, 0, st>>>(a.part, parts, dim, dgain);
  return launched(who);
}

}   // extern "C"
