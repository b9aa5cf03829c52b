// Rows in four bits with a scale, and optionally a middle, per group of 32, 64 or 128 columns: encoding, decoding, and the
// products of a few vectors with all rows.  The int8 quantiser (sq8.cu) has one scale per column or per matrix, as the reference's
// ScalarQuantizer does (Quantization/ScalarQuantizer.swift:251-270,389-451); a group's own scale is what makes four bits usable.
//
//   symmetric   s = half(float(amax / 7)),          value = s (c - 8)
//   min / max   s = half(float((hi - lo) / 15)),    m = half(float(lo + 8 s)),   value = s (c - 8) + m
//   code        c = clip(rint((x - m) / s) + 8, 0, 15), the quotient in 64 bits, ties to even; s = 0 gives c = 8
//   product     y[q, r] = sum_g ( s[r,g] sum_{i in g} (c[r,i] - 8) x[q,i] + m[r,g] sum_{i in g} x[q,i] )
//
// Two codes a byte, the even column in the low half.
#include <cuda_bf16.h>
#include <math_constants.h>

#include <algorithm>

#include "int4.cuh"

namespace vsk {
namespace {

template <typename T> __device__ __forceinline__ float to_float(T v);
template <> __device__ __forceinline__ float to_float<float>(float v) { return v; }
template <> __device__ __forceinline__ float to_float<__half>(__half v) { return __half2float(v); }
template <> __device__ __forceinline__ float to_float<__nv_bfloat16>(__nv_bfloat16 v) { return __bfloat162float(v); }

// ---- encoding -----------------------------------------------------------------------------------------------------------
// One warp per 128 columns of a row, four columns per lane: a group of G columns is G / 4 lanes, its extremes a few shuffles.

// The whole number nearest to away / step in 64 bits, ties to even.  The fp32 quotient is off by less than 1e-5 where the code is not
// clipped anyway (|quotient| < 9, three roundings of 2^-24 each): only quotients that near to a half are divided in 64 bits.
__device__ __forceinline__ int nearest_code(float x, float mid, float inv, float step) {
  const float u = (x - mid) * inv;
  float r = rintf(u);
  if (fabsf(u) < 9.0f && fabsf(u - r) > 0.5f - 1e-5f) r = (float)rint(((double)x - (double)mid) / (double)step);
  return (int)fminf(fmaxf(r, -8.0f), 7.0f) + 8;
}

template <typename T>
__global__ void __launch_bounds__(256) q4_encode_kernel(const T* __restrict__ rows, int64_t n, int dim, int64_t row_stride, int group,
                                                        int groups, int symmetric, int wide, uint8_t* __restrict__ codes,
                                                        int64_t code_stride, __half* __restrict__ scales,
                                                        __half* __restrict__ middles) {
  const int lane = threadIdx.x & 31;
  const int pieces = (dim + 127) / 128;
  const int64_t item = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5);
  if (item >= n * pieces) return;   // (whole warps)
  const int64_t row = item / pieces;
  const int col = (int)(item - row * pieces) * 128 + lane * 4;
  const T* src = rows + row * row_stride + col;
  float v[4];
  const int have = max(0, min(4, dim - col));
  if (wide && have == 4) {
    if constexpr (sizeof(T) == 4) {
      const float4 f = __ldg(reinterpret_cast<const float4*>(src));
      v[0] = f.x; v[1] = f.y; v[2] = f.z; v[3] = f.w;
    } else {
      const uint2 f = __ldg(reinterpret_cast<const uint2*>(src));
      const T* h = reinterpret_cast<const T*>(&f);
#pragma unroll
      for (int j = 0; j < 4; ++j) v[j] = to_float<T>(h[j]);
    }
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j) v[j] = j < have ? to_float<T>(*VSK_CHK(src + j)) : 0.f;
  }
  float hi = -CUDART_INF_F, lo = CUDART_INF_F;
#pragma unroll
  for (int j = 0; j < 4; ++j)
    if (j < have) {
      hi = fmaxf(hi, v[j]);
      lo = fminf(lo, v[j]);
    }
  for (int o = group / 8; o > 0; o >>= 1) {
    hi = fmaxf(hi, __shfl_xor_sync(0xffffffffu, hi, o));
    lo = fminf(lo, __shfl_xor_sync(0xffffffffu, lo, o));
  }
  if (have == 0) return;   // (no shuffles behind this)
  // two roundings, to fp32 and to fp16, as a host computes them
  float step, mid = 0.f;
  if (symmetric) {
    step = (float)((double)fmaxf(hi, -lo) / 7.0);
  } else {
    step = (float)(((double)hi - (double)lo) / 15.0);
  }
  const __half hs = __float2half_rn(fminf(step, 65504.f));
  step = __half2float(hs);
  const int64_t slot = row * groups + col / group;
  const bool first = (col % group) == 0;
  if (!symmetric) {
    const float m = (float)((double)lo + 8.0 * (double)step);
    const __half hm = __float2half_rn(fminf(fmaxf(m, -65504.f), 65504.f));
    mid = __half2float(hm);
    if (first) *VSK_CHK_W(middles + slot) = hm;
  }
  if (first) *VSK_CHK_W(scales + slot) = hs;
  const float inv = 1.0f / step;
  int c[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) c[j] = (j < have && step > 0.f) ? nearest_code(v[j], mid, inv, step) : 8;
  uint8_t* dst = codes + row * code_stride + (col >> 1);
  const uint8_t b0 = (uint8_t)(c[0] | (c[1] << 4)), b1 = (uint8_t)(c[2] | (c[3] << 4));
  if (have > 2 && (code_stride & 1) == 0 && (reinterpret_cast<uintptr_t>(codes) & 1) == 0) {
    *VSK_CHK_W(reinterpret_cast<uint16_t*>(dst)) = (uint16_t)(b0 | (b1 << 8));
  } else {
    *VSK_CHK_W(dst) = b0;
    if (have > 2) *VSK_CHK_W(dst + 1) = b1;
  }
}

// ---- decoding: one thread per eight columns --------------------------------------------------------------------------------
__global__ void __launch_bounds__(256) q4_decode_kernel(const uint8_t* __restrict__ codes, int64_t code_stride,
                                                        const __half* __restrict__ scales, const __half* __restrict__ middles,
                                                        int64_t scale_stride, int64_t n, int dim, int group,
                                                        float* __restrict__ out) {
  const int pieces = (dim + 7) / 8;
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (i >= n * pieces) return;
  const int64_t row = i / pieces;
  const int col = (int)(i - row * pieces) * 8;
  const uint8_t* src = codes + row * code_stride + (col >> 1);
  const int have = min(8, dim - col);
  uint32_t w = 0;
  if (have == 8 && (reinterpret_cast<uintptr_t>(src) & 3) == 0) {
    w = __ldg(reinterpret_cast<const uint32_t*>(src));
  } else {
    for (int j = 0; j < (have + 1) / 2; ++j) w |= (uint32_t)*VSK_CHK(src + j) << (8 * j);
  }
  const int64_t slot = row * scale_stride + col / group;
  const float s = __half2float(*VSK_CHK(scales + slot));
  const float m = middles ? __half2float(*VSK_CHK(middles + slot)) : 0.f;
  float v[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    v[j] = s * (float)((int)((w >> (4 * j)) & 15) - 8);   // exact: 11 + 4 bits
    if (middles) v[j] = __fadd_rn(v[j], m);
  }
  float* dst = out + row * dim + col;
  if (have == 8 && (reinterpret_cast<uintptr_t>(dst) & 15) == 0) {
    reinterpret_cast<float4*>(VSK_CHK_W(dst))[0] = make_float4(v[0], v[1], v[2], v[3]);
    reinterpret_cast<float4*>(VSK_CHK_W(dst + 4))[0] = make_float4(v[4], v[5], v[6], v[7]);
  } else {
    for (int j = 0; j < have; ++j) *VSK_CHK_W(dst + j) = v[j];
  }
}

int32_t check_ctx(vsk_ctx* c, Ctx** ctx) {
  *ctx = reinterpret_cast<Ctx*>(c);
  if (!*ctx) return VSK_ERR_INVALID_INPUT;
  cudaSetDevice((*ctx)->device);
  return VSK_OK;
}

int32_t check_shape(Ctx* ctx, int64_t n, int32_t dim, int32_t group) {
  if (n <= 0) return fail(ctx, VSK_ERR_EMPTY_INPUT, "no rows");
  if (n > (1ll << 40)) return fail(ctx, VSK_ERR_INVALID_BUFFER_SIZE, "too many rows");
  if (dim <= 0 || dim > (1 << 24)) return fail(ctx, VSK_ERR_DIMENSION_MISMATCH, "dimension must be in [1, 2^24]");
  if (group != 32 && group != 64 && group != 128)
    return fail(ctx, VSK_ERR_UNSUPPORTED_OPERATION, "groups of %d columns are not supported (32, 64 or 128)", group);
  return VSK_OK;
}

int32_t check_rows(Ctx* ctx, const vsk_q4_rows* r) {
  if (!r) return fail(ctx, VSK_ERR_INVALID_INPUT, "null rows");
  VSK_TRY(check_shape(ctx, r->n, r->dim, r->group));
  if (!r->codes || !r->scales) return fail(ctx, VSK_ERR_INVALID_INPUT, "null codes or scales");
  if (r->code_stride < ((int64_t)r->dim + 1) / 2) return fail(ctx, VSK_ERR_INVALID_BUFFER_SIZE, "code rows are shorter than %d columns", r->dim);
  if (r->scale_stride < ceil_div(r->dim, r->group)) return fail(ctx, VSK_ERR_INVALID_BUFFER_SIZE, "scale rows are shorter than the groups of %d columns", r->dim);
  if ((reinterpret_cast<uintptr_t>(r->scales) & 1) || (reinterpret_cast<uintptr_t>(r->middles) & 1))
    return fail(ctx, VSK_ERR_INVALID_INPUT, "scales and middles must be aligned to two bytes");
  return VSK_OK;
}

int dtype_size(int32_t t) { return t == VSK_DTYPE_F32 ? 4 : (t == VSK_DTYPE_F16 || t == VSK_DTYPE_BF16) ? 2 : 0; }

int32_t encode(Ctx* ctx, const void* rows, int32_t dtype, int64_t n, int32_t dim, int64_t row_stride, int32_t group, int32_t symmetric,
               uint8_t* codes, int64_t code_stride, void* scales, void* middles) {
  const int es = dtype_size(dtype);
  const int64_t items = n * ceil_div(dim, 128), blocks = ceil_div(items, 8);
  if (blocks > 0x7fffffffLL) return fail(ctx, VSK_ERR_INVALID_BUFFER_SIZE, "too many rows in one call");
  const int groups = (int)ceil_div(dim, group);
  const int wide = ((reinterpret_cast<uintptr_t>(rows) | (uintptr_t)(row_stride * es)) & (uintptr_t)(4 * es - 1)) == 0;
  auto go = [&](auto* x) {
    using T = std::remove_const_t<std::remove_pointer_t<decltype(x)>>;
    q4_encode_kernel<T><<<(unsigned)blocks, 256, 0, ctx->stream>>>(x, n, dim, row_stride, group, groups, symmetric, wide, codes,
                                                                   code_stride, (__half*)scales, (__half*)middles);
  };
  if (dtype == VSK_DTYPE_F32) go((const float*)rows);
  else if (dtype == VSK_DTYPE_F16) go((const __half*)rows);
  else go((const __nv_bfloat16*)rows);
  ctx->stats.kernel_launches++;
  VSK_CUDA(ctx, cudaGetLastError());
  return VSK_OK;
}

int32_t decode(Ctx* ctx, const vsk_q4_rows* r, float* out) {
  const int64_t blocks = ceil_div(r->n * ceil_div(r->dim, 8), 256);
  if (blocks > 0x7fffffffLL) return fail(ctx, VSK_ERR_INVALID_BUFFER_SIZE, "too many rows in one call");
  q4_decode_kernel<<<(unsigned)blocks, 256, 0, ctx->stream>>>(r->codes, r->code_stride, (const __half*)r->scales,
                                                              (const __half*)r->middles, r->scale_stride, r->n, r->dim, r->group, out);
  ctx->stats.kernel_launches++;
  VSK_CUDA(ctx, cudaGetLastError());
  return VSK_OK;
}

int32_t check_encode(Ctx* ctx, const void* rows, int32_t dtype, int64_t n, int32_t dim, int64_t row_stride, int32_t group,
                     int32_t symmetric, uint8_t* codes, int64_t code_stride, void* scales, void* middles) {
  VSK_TRY(check_shape(ctx, n, dim, group));
  const int es = dtype_size(dtype);
  if (es == 0) return fail(ctx, VSK_ERR_UNSUPPORTED_OPERATION, "element type %d is not supported", dtype);
  if (!rows || !codes || !scales || (!symmetric && !middles)) return fail(ctx, VSK_ERR_INVALID_INPUT, "null pointer");
  if (row_stride < dim) return fail(ctx, VSK_ERR_INVALID_BUFFER_SIZE, "rows are shorter than %d columns", dim);
  if (code_stride < ((int64_t)dim + 1) / 2) return fail(ctx, VSK_ERR_INVALID_BUFFER_SIZE, "code rows are shorter than %d columns", dim);
  if ((reinterpret_cast<uintptr_t>(rows) & (uintptr_t)(es - 1)) || (reinterpret_cast<uintptr_t>(scales) & 1) ||
      (reinterpret_cast<uintptr_t>(middles) & 1))
    return fail(ctx, VSK_ERR_INVALID_INPUT, "a pointer is not aligned to its element");
  return VSK_OK;
}

// Device copies of one host-pointer call, freed when it goes out of scope.
struct Staged {
  Ctx* ctx;
  void* p[4] = {};
  int used = 0;
  explicit Staged(Ctx* c) : ctx(c) {}
  ~Staged() {
    for (void* q : p) dev_free(q);
  }
  int32_t get(size_t bytes, void** out) {
    VSK_TRY(dev_alloc(ctx, &p[used], bytes));
    *out = p[used++];
    return VSK_OK;
  }
};

}  // namespace
}  // namespace vsk

using namespace vsk;

extern "C" {

int32_t vsk_q4_encode_dev(vsk_ctx* c, const void* rows, int32_t dtype, int64_t n, int32_t dim, int64_t row_stride, int32_t group,
                          int32_t symmetric, uint8_t* codes, int64_t code_stride, void* scales, void* middles) {
  VSK_TRACE("vsk_q4_encode_dev");
  Ctx* ctx;
  VSK_TRY(check_ctx(c, &ctx));
  VSK_TRY(check_encode(ctx, rows, dtype, n, dim, row_stride, group, symmetric, codes, code_stride, scales, middles));
  drain_stale_error("vsk_q4_encode_dev");
  VSK_TRY(encode(ctx, rows, dtype, n, dim, row_stride, group, symmetric, codes, code_stride, scales, middles));
  VSK_CUDA(ctx, cudaStreamSynchronize(ctx->stream));
  return VSK_OK;
}

int32_t vsk_q4_encode(vsk_ctx* c, const float* rows, int64_t n, int32_t dim, int32_t group, int32_t symmetric, uint8_t* codes,
                      int64_t code_stride, void* scales, void* middles) {
  VSK_TRACE("vsk_q4_encode");
  Ctx* ctx;
  VSK_TRY(check_ctx(c, &ctx));
  VSK_TRY(check_encode(ctx, rows, VSK_DTYPE_F32, n, dim, dim, group, symmetric, codes, code_stride, scales, middles));
  drain_stale_error("vsk_q4_encode");
  const size_t in = (size_t)n * dim * 4, held = (size_t)n * code_stride, per = (size_t)n * ceil_div(dim, group) * 2;
  Staged s(ctx);
  void *dx, *dc, *ds, *dm = nullptr;
  VSK_TRY(s.get(in, &dx));
  VSK_TRY(s.get(held, &dc));
  VSK_TRY(s.get(per, &ds));
  if (!symmetric) VSK_TRY(s.get(per, &dm));
  VSK_CUDA(ctx, cudaMemcpyAsync(dx, rows, in, cudaMemcpyHostToDevice, ctx->stream));
  // (bytes of a code row behind its columns are the caller's: they go back as zeros of this copy)
  VSK_CUDA(ctx, cudaMemsetAsync(dc, 0, held, ctx->stream));
  VSK_TRY(encode(ctx, dx, VSK_DTYPE_F32, n, dim, dim, group, symmetric, (uint8_t*)dc, code_stride, ds, dm));
  VSK_CUDA(ctx, cudaMemcpyAsync(codes, dc, held, cudaMemcpyDeviceToHost, ctx->stream));
  VSK_CUDA(ctx, cudaMemcpyAsync(scales, ds, per, cudaMemcpyDeviceToHost, ctx->stream));
  if (!symmetric) VSK_CUDA(ctx, cudaMemcpyAsync(middles, dm, per, cudaMemcpyDeviceToHost, ctx->stream));
  VSK_CUDA(ctx, cudaStreamSynchronize(ctx->stream));
  ctx->stats.h2d_bytes += (int64_t)in;
  ctx->stats.d2h_bytes += (int64_t)(held + per + (symmetric ? 0 : per));
  return VSK_OK;
}

int32_t vsk_q4_decode_dev(vsk_ctx* c, const vsk_q4_rows* rows, float* out) {
  VSK_TRACE("vsk_q4_decode_dev");
  Ctx* ctx;
  VSK_TRY(check_ctx(c, &ctx));
  VSK_TRY(check_rows(ctx, rows));
  if (!out) return fail(ctx, VSK_ERR_INVALID_INPUT, "null pointer");
  drain_stale_error("vsk_q4_decode_dev");
  VSK_TRY(decode(ctx, rows, out));
  VSK_CUDA(ctx, cudaStreamSynchronize(ctx->stream));
  return VSK_OK;
}

int32_t vsk_q4_decode(vsk_ctx* c, const vsk_q4_rows* rows, float* out) {
  VSK_TRACE("vsk_q4_decode");
  Ctx* ctx;
  VSK_TRY(check_ctx(c, &ctx));
  VSK_TRY(check_rows(ctx, rows));
  if (!out) return fail(ctx, VSK_ERR_INVALID_INPUT, "null pointer");
  drain_stale_error("vsk_q4_decode");
  const int64_t groups = ceil_div(rows->dim, rows->group);
  // the last row's stride is not the caller's to read behind
  const size_t held = (size_t)(rows->n - 1) * rows->code_stride + (size_t)(rows->dim + 1) / 2;
  const size_t per = ((size_t)(rows->n - 1) * rows->scale_stride + groups) * 2, outb = (size_t)rows->n * rows->dim * 4;
  Staged s(ctx);
  vsk_q4_rows r = *rows;
  void *dc, *ds, *dm = nullptr, *dx;
  VSK_TRY(s.get(held, &dc));
  VSK_TRY(s.get(per, &ds));
  if (rows->middles) VSK_TRY(s.get(per, &dm));
  VSK_TRY(s.get(outb, &dx));
  VSK_CUDA(ctx, cudaMemcpyAsync(dc, rows->codes, held, cudaMemcpyHostToDevice, ctx->stream));
  VSK_CUDA(ctx, cudaMemcpyAsync(ds, rows->scales, per, cudaMemcpyHostToDevice, ctx->stream));
  if (dm) VSK_CUDA(ctx, cudaMemcpyAsync(dm, rows->middles, per, cudaMemcpyHostToDevice, ctx->stream));
  r.codes = (const uint8_t*)dc;
  r.scales = ds;
  r.middles = dm;
  VSK_TRY(decode(ctx, &r, (float*)dx));
  VSK_CUDA(ctx, cudaMemcpyAsync(out, dx, outb, cudaMemcpyDeviceToHost, ctx->stream));
  VSK_CUDA(ctx, cudaStreamSynchronize(ctx->stream));
  ctx->stats.h2d_bytes += (int64_t)(held + per * (dm ? 2 : 1));
  ctx->stats.d2h_bytes += (int64_t)outb;
  return VSK_OK;
}

int32_t vsk_q4_product_dev(vsk_ctx* c, const vsk_q4_rows* rows, const void* x, int32_t x_dtype, int64_t nq, int64_t x_stride, void* y,
                           int32_t y_dtype, int64_t y_stride) {
  VSK_TRACE("vsk_q4_product_dev");
  Ctx* ctx;
  VSK_TRY(check_ctx(c, &ctx));
  VSK_TRY(check_rows(ctx, rows));
  if (nq <= 0) return fail(ctx, VSK_ERR_EMPTY_INPUT, "no vectors");
  if (nq > (1 << 24)) return fail(ctx, VSK_ERR_INVALID_BUFFER_SIZE, "too many vectors");
  if (!x || !y) return fail(ctx, VSK_ERR_INVALID_INPUT, "null pointer");
  const int xs = dtype_size(x_dtype), ys = dtype_size(y_dtype);
  if (!xs || !ys) return fail(ctx, VSK_ERR_UNSUPPORTED_OPERATION, "element type %d is not supported", xs ? y_dtype : x_dtype);
  if (x_stride < rows->dim) return fail(ctx, VSK_ERR_DIMENSION_MISMATCH, "vectors are shorter than %d columns", rows->dim);
  if (y_stride < rows->n) return fail(ctx, VSK_ERR_INVALID_BUFFER_SIZE, "result rows are shorter than the rows of the matrix");
  if ((reinterpret_cast<uintptr_t>(x) & (uintptr_t)(xs - 1)) || (reinterpret_cast<uintptr_t>(y) & (uintptr_t)(ys - 1)))
    return fail(ctx, VSK_ERR_INVALID_INPUT, "a pointer is not aligned to its element");
  drain_stale_error("vsk_q4_product_dev");
  // 200 000 x 2 048, groups of 128 / of 32 with middles: five fp16 vectors take 75 / 130 us in whole numbers and 91 / 142 in 16 bits, six
  // 99 / 175 and 91 / 143 (a third tile of digits).  fp32 vectors have no 16-bit form.
  if (x_dtype == VSK_DTYPE_F32 || nq <= 5) VSK_TRY(q4_product_digits(ctx, *rows, x, x_dtype, nq, x_stride, y, y_dtype, y_stride));
  else VSK_TRY(q4_product(ctx, *rows, x, x_dtype, nq, x_stride, y, y_dtype, y_stride));
  VSK_CUDA(ctx, cudaStreamSynchronize(ctx->stream));
  return VSK_OK;
}

}  // extern "C"
