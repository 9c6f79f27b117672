// What the host sides of the embedding heads (prod.cu, rows.cu) share: errors, alignment and argument
// checks.
#pragma once
#include <cuda_runtime.h>
#include <stdarg.h>
#include <stdio.h>

#include "k_mx.cuh"

int smg_set_error(int code, const char* msg);              // smg.cu: records msg for smg_last_error

static inline int fail(int code, const char* fmt, ...) {
  char msg[256];
  va_list ap;
  va_start(ap, fmt);
  vsnprintf(msg, sizeof msg, fmt, ap);
  va_end(ap);
  return smg_set_error(code, msg);
}

static inline bool on16(const void* p) { return !((uintptr_t)p & 15); }
static inline bool type_ok(int t) { return t == SMG_EMB_F32 || t == SMG_EMB_BF16 || t == SMG_EMB_F16; }
static inline int size_of(int t) { return t == SMG_EMB_F32 ? 4 : 2; }
// rows of ld elements starting at p all start on 16 bytes
static inline bool rows16(const void* p, int64_t ld, int type) { return on16(p) && ld * size_of(type) % 16 == 0; }

static inline int out_rows(const char* who, const void* p, int64_t ld, int64_t len, int64_t rows) {
  if (rows > 0 && !p) return fail(SMG_ERR_ARGS, "%s: the output is null", who);
  if (ld < len) return fail(SMG_ERR_ARGS, "%s: the output's rows overlap", who);
  return SMG_OK;
}

static inline MxOut mx_rows(int k, const uint8_t* codes, const uint8_t* scales, uint16_t* values) {
  MxOut o;
  o.codes = const_cast<uint8_t*>(codes); o.scales = const_cast<uint8_t*>(scales); o.values = (__nv_bfloat16*)values;
  o.dim = k; o.kb = (k + 31) / 32; o.pitch = (o.kb + 3) / 4 * 4;
  return o;
}

static inline int mx_args(const char* who, int rows, int k, int bits, const uint8_t* codes, const uint8_t* scales) {
  if (rows < 0 || k < 1 || k > (1 << 24)) return fail(SMG_ERR_ARGS, "%s: bad sizes (rows %d, %d values a row)", who, rows, k);
  if (bits != 4 && bits != 8) return fail(SMG_ERR_ARGS, "%s: bits must be 4 or 8", who);
  if (rows > 0 && (!codes != !scales)) return fail(SMG_ERR_ARGS, "%s: codes and scales go together", who);
  // the products' tensor maps want the codes on 16 bytes (rows of them are multiples of it); scales are copied 4 at a time
  if (!on16(codes) || ((uintptr_t)scales & 3)) return fail(SMG_ERR_ARGS, "%s: codes must start on 16 bytes, scales on 4", who);
  return SMG_OK;
}

static inline MxDiv mx_div(int per) {
  int shift = 0;
  while ((1ll << shift) < per) ++shift;
  const MxDiv d = {(uint32_t)per, (uint32_t)(((1ull << (31 + shift)) + (uint32_t)per - 1) / (uint32_t)per), shift};
  return d;
}

// A launch that may be set up while the kernel before it in the stream still runs (heads_wait).
template <typename... P, typename... A>
static inline int launch_next(const char* who, void (*kernel)(P...), dim3 grid, int threads, size_t smem, cudaStream_t st, A... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = at;
  cfg.numAttrs = 1;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, P(args)...);
  return e == cudaSuccess ? SMG_OK : fail(SMG_ERR_DEVICE, "%s: %s", who, cudaGetErrorString(e));
}
