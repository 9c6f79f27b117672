// C ABI of the embedding heads' row operators (include/smg.h): microscaled rows, the residual norm
// and its gradients.
#include <algorithm>

#include "heads_host.h"
#include "k_norm.cuh"

extern "C" {

// ------------------------------------------------------------------ microscaled rows
static int mx_blocks(const char* who, int64_t parts, unsigned* grid) {
  const int64_t b = (parts + 256 * MX_EACH - 1) / (256 * MX_EACH);
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
  const bool vec = rows16(x, ldx, type) && k % 8 == 0;
  unsigned grid;
  if (int r = mx_blocks(who, n, &grid)) return r;
  const cudaStream_t st = (cudaStream_t)stream;
#define CALL(TY)                                                                                              \
  const auto f = bits == 4 ? (vec ? k_mx_quantise<TY, 4, true> : k_mx_quantise<TY, 4, false>)                 \
                           : (vec ? k_mx_quantise<TY, 8, true> : k_mx_quantise<TY, 8, false>);                \
  return launch_next(who, f, grid, 256, 0, st, (const Elem<TY>::T*)x, ldx, rows, n, mx_div(o.pitch * 4), o)
  BY_TYPE(type, CALL);
#undef CALL
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
  if (int r = mx_blocks(who, n, &grid)) return r;
#define CALL(TY)                                                                                              \
  return launch_next(who, bits == 4 ? k_mx_values<TY, 4> : k_mx_values<TY, 8>, grid, 256, 0, (cudaStream_t)stream, o, n, \
                     mx_div(o.kb * 4), (Elem<TY>::T*)out, ld, vec)
  BY_TYPE(out_type, CALL);
#undef CALL
}

// ------------------------------------------------------------------ residual norm
// Warps a row and register steps of 8 values a lane, for a row of `steps` x 256 values: as many steps
// as leave two or more blocks an SM their registers (forward: two 16-bit inputs in 5 steps,
// or 32-bit ones in 3; the gradient with its four inputs and its column sums: 3 and 2), then more
// warps a row.  Rows off 16 bytes take the same shape, so that the order of the sums is the same.
#define NORM_MAX_DIM 16384
#define NORM_PARTS 296   // blocks of the gradient kernel, two an SM
#define NORM_FEW 1184    // rows (forward) up to which a row of at most 2048 values gets a block's 8 warps, one step a lane
                         // instead of up to five in turn (1 x 1152: 2.0 us against 4.0; 1184: 5.1 against 6.3; 2368: 9.3, 7.7)

#define BY_STEPS5(steps, CALL)                     \
  do {                                             \
    if (steps <= 1) { CALL(1, 1); }                \
    else if (steps <= 2) { CALL(1, 2); }           \
    else if (steps <= 3) { CALL(1, 3); }           \
    else if (steps <= 4) { CALL(1, 4); }           \
    else if (steps <= 5) { CALL(1, 5); }           \
    else if (steps <= 10) { CALL(2, 5); }          \
    else if (steps <= 20) { CALL(4, 5); }          \
    else if (steps <= 40) { CALL(8, 5); }          \
    else { CALL(8, 8); }                           \
  } while (0)
#define BY_STEPS3(steps, CALL)                     \
  do {                                             \
    if (steps <= 1) { CALL(1, 1); }                \
    else if (steps <= 2) { CALL(1, 2); }           \
    else if (steps <= 3) { CALL(1, 3); }           \
    else if (steps <= 6) { CALL(2, 3); }           \
    else if (steps <= 12) { CALL(4, 3); }          \
    else if (steps <= 24) { CALL(8, 3); }          \
    else { CALL(8, 8); }                           \
  } while (0)
#define BY_STEPS2(steps, CALL)                     \
  do {                                             \
    if (steps <= 1) { CALL(1, 1); }                \
    else if (steps <= 2) { CALL(1, 2); }           \
    else if (steps <= 4) { CALL(2, 2); }           \
    else if (steps <= 8) { CALL(4, 2); }           \
    else if (steps <= 16) { CALL(8, 2); }          \
    else { CALL(8, 8); }                           \
  } while (0)

int smg_norm_add(const void* x, int64_t ldx, const void* r, int64_t ldr, const float* gain, int rows, int dim, int type, float eps,
                 void* h, int64_t ldh, float* rstd, int bits, uint8_t* codes, uint8_t* scales, uint16_t* values, void* stream) {
  const char* who = "smg_norm_add";
  if (int e = mx_args(who, rows, dim, bits, codes, scales)) return e;
  if (!type_ok(type)) return fail(SMG_ERR_ARGS, "%s: bad input type", who);
  if (dim > NORM_MAX_DIM) return fail(SMG_ERR_CAPACITY, "%s: %d values a row, at most %d", who, dim, NORM_MAX_DIM);
  if (h && ldh < dim) return fail(SMG_ERR_ARGS, "%s: the rows of h overlap", who);
  if (rows == 0) return SMG_OK;
  if (!x || !gain || (!codes && !values)) return fail(SMG_ERR_ARGS, "%s: x, gain, or codes and values are null", who);
  if (values && ((uintptr_t)values & (dim % 8 ? 1 : 15))) return fail(SMG_ERR_ARGS, "%s: values off their alignment", who);
  NormArgs a = {};
  a.x = x; a.ldx = ldx; a.r = r; a.ldr = ldr; a.gain = gain; a.h = h; a.ldh = ldh; a.rstd = rstd;
  a.rows = rows; a.dim = dim; a.eps = eps;
  const bool vec = dim % 8 == 0 && rows16(x, ldx, type) && (!r || rows16(r, ldr, type)) && (!h || rows16(h, ldh, type)) && on16(gain);
  a.mx = mx_rows(dim, codes, scales, values);
  const int steps = (a.mx.pitch * 4 + 31) / 32;   // of 256 values, the scales' padding included
#define LAUNCH(T, W, NV)                                                                                      \
  const auto f = bits == 4 ? (vec ? k_norm_add<T, 4, W, NV, true> : k_norm_add<T, 4, W, NV, false>)           \
                           : (vec ? k_norm_add<T, 8, W, NV, true> : k_norm_add<T, 8, W, NV, false>);          \
  return launch_next(who, f, (unsigned)(((int64_t)rows + NORM_ROWS(W) - 1) / NORM_ROWS(W)), NORM_THREADS, 0, (cudaStream_t)stream, a)
#define CALL32(W, NV) LAUNCH(SMG_EMB_F32, W, NV)
#define CALLBF(W, NV) LAUNCH(SMG_EMB_BF16, W, NV)
#define CALLHF(W, NV) LAUNCH(SMG_EMB_F16, W, NV)
  if (rows <= NORM_FEW && steps > 1 && steps <= 8) {
    if (type == SMG_EMB_F32) { CALL32(8, 1); }
    else if (type == SMG_EMB_BF16) { CALLBF(8, 1); }
    else { CALLHF(8, 1); }
  }
  if (type == SMG_EMB_F32) BY_STEPS3(steps, CALL32);
  else if (type == SMG_EMB_BF16) BY_STEPS5(steps, CALLBF);
  else BY_STEPS5(steps, CALLHF);
#undef LAUNCH
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
  const bool vec = dim % 8 == 0 && rows16(x, ldx, type) && (!r || rows16(r, ldr, type)) && rows16(dy, lddy, type) &&
                   (!dh || rows16(dh, lddh, type)) && rows16(dx, lddx, type) && on16(gain);
  const cudaStream_t st = (cudaStream_t)stream;
  const int steps = (dim + 255) / 256;
  int parts = 0, e = SMG_OK;
  if (rows > 0) {
#define LAUNCH(T, W, NV)                                                                         \
  parts = (int)std::min<int64_t>(((int64_t)rows + NORM_ROWS(W) - 1) / NORM_ROWS(W), NORM_PARTS); \
  const int sm = W < 8 ? NORM_ROWS(W) * dim * 4 : 0;                                             \
  e = launch_next(who, vec ? k_norm_add_bwd<T, W, NV, true> : k_norm_add_bwd<T, W, NV, false>, parts, NORM_THREADS, sm, st, a)
    if (type == SMG_EMB_F32) BY_STEPS2(steps, CALL32);
    else if (type == SMG_EMB_BF16) BY_STEPS3(steps, CALLBF);
    else BY_STEPS3(steps, CALLHF);
#undef LAUNCH
  }
  if (e) return e;
  return launch_next(who, k_norm_dgain, (dim + 31) / 32, 1024, 0, st, a.part, parts, dim, dgain);
}

}   // extern "C"
