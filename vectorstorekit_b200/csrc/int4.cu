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
// Eight columns per lane: a group of G columns is G / 8 lanes, its extremes a few shuffles.  `lanes` neighbouring lanes share a row (short
// rows leave several to a warp) and walk along it, the next columns' load under way.  100 000 x 768 fp32, groups of 32, min / max
// (307 MB in): 93 us, issue slots 84 % busy: bound by the instructions of a value and of its group's scale, which every lane of the group makes (a few
// of them in 64 bits; quotients in 64 bits are taken only next to a border).

// (float)(d / 15) with the quotient in 64 bits.  The product with the rounded reciprocal is off by less than 2 of its last bits: it
// rounds to the same fp32 number unless it lies that near to the middle between two.
__device__ __forceinline__ float fifteenth(double d) {
  const double q = d * (1.0 / 15.0);
  const int rest = (int)(__double2loint(q) & 0x1fffffff) - 0x10000000;   // the 29 bits that fp32 drops (normal numbers)
  if (abs(rest) < 8 || !(q > 1.2e-38)) return (float)(d / 15.0);
  return (float)q;
}

// Eight codes, the first in the lowest four bits: the whole numbers nearest to (x - mid) / step in 64 bits, ties to even, within -8 .. 7.  The
// fp32 quotient is off by less than 1e-5 there (a few roundings of 2^-24 each): only where one lies that near to a half are they divided
// in 64 bits.  Rounding and conversion are an addition of 1.5 2^23: the unit that has instructions for them takes a quarter of the rate.
__device__ __forceinline__ unsigned nearest_codes(const float (&x)[8], float mid, float inv, float step) {
  unsigned t[8];
  float far = 0.f;
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const float u = fminf(fmaxf((x[j] - mid) * inv, -8.f), 7.f), r = u + 12582912.f;
    far = fmaxf(far, fabsf(u - (r - 12582912.f)));
    t[j] = __float_as_uint(r);
  }
  if (far > 0.5f - 1e-5f) {
#pragma unroll
    for (int j = 0; j < 8; ++j) t[j] = (unsigned)(int)fmin(fmax(rint(((double)x[j] - (double)mid) / (double)step), -8.0), 7.0);
  }
  unsigned c = 0x88888888u;
#pragma unroll
  for (int j = 0; j < 8; ++j) c ^= (t[j] & 15u) << (4 * j);
  return c;
}

template <typename T, bool SYMMETRIC, bool WIDE>
__global__ void __launch_bounds__(256) q4_encode_kernel(const T* __restrict__ rows, int64_t n, int dim, int64_t row_stride, int group,
                                                        int groups, int lanes, int columns, uint8_t* __restrict__ codes,
                                                        int64_t code_stride, __half* __restrict__ scales,
                                                        __half* __restrict__ middles) {
  const int lane = threadIdx.x & (lanes - 1), per_block = 256 / lanes;
  const int64_t row = (int64_t)blockIdx.x * per_block + threadIdx.x / lanes;
  const bool inside = row < n;   // (whole warps walk together)
  const T* const src = rows + (inside ? row : 0) * row_stride;
  uint8_t* const dst = codes + (inside ? row : 0) * code_stride;
  const bool words = (code_stride & 3) == 0 && (reinterpret_cast<uintptr_t>(codes) & 3) == 0;
  const int first = blockIdx.y * columns, end = min(dim, first + columns), stride = 8 * lanes;
  const int group_shift = group == 32 ? 5 : group == 64 ? 6 : 7;

  // Rows that do not begin at 16-byte boundaries: aligned vectors around the lane's eight columns, shifted together.  They may reach into a
  // neighbouring row, never out of the rows' memory.
  const int off = (int)(reinterpret_cast<uintptr_t>(src) & 15);
  const uint8_t* const begin = reinterpret_cast<const uint8_t*>(rows);
  const uint8_t* const finish = reinterpret_cast<const uint8_t*>(rows + (n - 1) * row_stride + dim);
  auto load = [&](int col, float (&v)[8]) {
    const int have = inside ? min(8, end - col) : 0;
    constexpr int kWords = 2 * (int)sizeof(T);   // of eight columns
    const uint8_t* const from = reinterpret_cast<const uint8_t*>(src + col) - off;
    if (!WIDE && have == 8 && from >= begin && from + 4 * kWords + 16 <= finish) {
      uint32_t w[kWords + 4];
#pragma unroll
      for (int i = 0; i < kWords + 4; i += 4) {
        const uint4 u = __ldg(reinterpret_cast<const uint4*>(from + 4 * i));
        w[i] = u.x; w[i + 1] = u.y; w[i + 2] = u.z; w[i + 3] = u.w;
      }
#pragma unroll
      for (int i = 0; i < kWords + 2; ++i) w[i] = (off & 8) ? w[i + 2] : w[i];
#pragma unroll
      for (int i = 0; i < kWords + 1; ++i) w[i] = (off & 4) ? w[i + 1] : w[i];
      if constexpr (sizeof(T) == 2) {
#pragma unroll
        for (int i = 0; i < kWords; ++i) w[i] = __funnelshift_r(w[i], w[i + 1], 8 * (off & 2));
      }
      T h[8];
      memcpy(h, w, sizeof(h));
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] = to_float<T>(h[j]);
    } else if (WIDE && have == 8) {
      if constexpr (sizeof(T) == 4) {
#pragma unroll
        for (int j = 0; j < 8; j += 4) {
          const float4 f = __ldg(reinterpret_cast<const float4*>(src + col + j));
          v[j] = f.x; v[j + 1] = f.y; v[j + 2] = f.z; v[j + 3] = f.w;
        }
      } else {
        const uint4 f = __ldg(reinterpret_cast<const uint4*>(src + col));
        const T* h = reinterpret_cast<const T*>(&f);
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = to_float<T>(h[j]);
      }
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] = j < have ? to_float<T>(*VSK_CHK(src + col + j)) : j == 0 ? 0.f : v[0];   // (no other extremes)
    }
  };
  float next[8];
  load(first + lane * 8, next);
  for (int base = first; base < end; base += stride) {
    const int col = base + lane * 8;
    float v[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = next[j];
    if (base + stride < end) load(col + stride, next);
    const int have = inside ? min(8, end - col) : 0;
    float hi = v[0], lo = v[0];
#pragma unroll
    for (int j = 1; j < 8; ++j) {
      hi = fmaxf(hi, v[j]);
      lo = fminf(lo, v[j]);
    }
    if (have <= 0) {
      hi = -CUDART_INF_F;
      lo = CUDART_INF_F;
    }
    if (SYMMETRIC) hi = fmaxf(hi, -lo);
    for (int o = group / 16; o > 0; o >>= 1) {
      hi = fmaxf(hi, __shfl_xor_sync(0xffffffffu, hi, o));
      if (!SYMMETRIC) lo = fminf(lo, __shfl_xor_sync(0xffffffffu, lo, o));
    }
    if (have <= 0) continue;
    // Two roundings, to fp32 and to fp16, as a host computes them from the quotient in 64 bits.  (A seventh of an fp32 number is never
    // nearer than 2^-28 of it to the middle between two: one division in fp32 rounds alike.)
    float step, mid = 0.f;
    if (SYMMETRIC) step = __fdiv_rn(hi, 7.0f);
    else step = fifteenth((double)hi - (double)lo);
    const __half hs = __float2half_rn(fminf(step, 65504.f));
    step = __half2float(hs);
    const int64_t slot = row * groups + (col >> group_shift);
    const bool leads = (col & (group - 1)) == 0;
    if (!SYMMETRIC) {
      const float m = (float)((double)lo + 8.0 * (double)step);
      const __half hm = __float2half_rn(fminf(fmaxf(m, -65504.f), 65504.f));
      mid = __half2float(hm);
      if (leads) *VSK_CHK_W(middles + slot) = hm;
    }
    if (leads) *VSK_CHK_W(scales + slot) = hs;
    const float inv = step > 0.f ? __fdividef(1.0f, step) : 0.f;   // (of an fp16 number: in range)
    unsigned c = nearest_codes(v, mid, inv, step);
    uint8_t* const at = dst + (col >> 1);
    if (have == 8 && words) {
      *VSK_CHK_W(reinterpret_cast<uint32_t*>(at)) = c;
    } else {
      if (have & 1) c = (c & ~(15u << (4 * have))) | (8u << (4 * have));   // the half behind an odd last column
      for (int j = 0; j < (have + 1) / 2; ++j) *VSK_CHK_W(at + j) = (uint8_t)(c >> (8 * j));
    }
  }
}

// ---- decoding: eight columns per thread, `lanes` threads along a row (100 000 x 768 to fp32, 48 MB in and 307 MB out: 76 us, 4.7 TB/s asked for) -------
constexpr int kDecodeSteps = 4;
__global__ void __launch_bounds__(256) q4_decode_kernel(const uint8_t* __restrict__ codes, int64_t code_stride,
                                                        const __half* __restrict__ scales, const __half* __restrict__ middles,
                                                        int64_t scale_stride, int64_t n, int dim, int group_shift, int lanes, int columns,
                                                        float* __restrict__ out) {
  __shared__ __align__(16) float staged[8][256];   // what a warp writes at once, where rows do not begin at 16-byte boundaries
  const int64_t row = (int64_t)blockIdx.x * (256 / lanes) + threadIdx.x / lanes;
  const bool inside = row < n;   // (whole warps walk together)
  const bool apart = ((reinterpret_cast<uintptr_t>(out) | (uintptr_t)(4 * dim)) & 15) != 0;
  const uint8_t* const line = codes + row * code_stride;
  const __half* const s_line = scales + row * scale_stride;
  const __half* const m_line = middles + row * scale_stride;
  float* const to = out + row * dim;
  const int end = min(dim, ((int)blockIdx.y + 1) * columns), first = blockIdx.y * columns + (threadIdx.x & (lanes - 1)) * 8;
  // everything that a thread needs is asked for before anything is stored (`columns` are at most as many strides)
  uint32_t w[kDecodeSteps];
  __half s[kDecodeSteps], m[kDecodeSteps];
#pragma unroll
  for (int i = 0; i < kDecodeSteps; ++i) {
    const int col = first + i * lanes * 8, have = inside ? min(8, end - col) : 0;
    w[i] = 0;
    s[i] = m[i] = __half(0.f);
    if (have <= 0) continue;
    const uint8_t* src = line + (col >> 1);
    if (have == 8 && (reinterpret_cast<uintptr_t>(src) & 3) == 0) {
      w[i] = __ldg(reinterpret_cast<const uint32_t*>(src));
    } else {
      for (int j = 0; j < (have + 1) / 2; ++j) w[i] |= (uint32_t)*VSK_CHK(src + j) << (8 * j);
    }
    s[i] = *VSK_CHK(s_line + (col >> group_shift));
    if (middles) m[i] = *VSK_CHK(m_line + (col >> group_shift));
  }
#pragma unroll
  for (int i = 0; i < kDecodeSteps; ++i) {
    const int col = first + i * lanes * 8, have = inside ? min(8, end - col) : 0;
    const int base = blockIdx.y * columns + i * lanes * 8;   // of this step, the same for the whole warp
    if (base >= end) break;
    const float scale = __half2float(s[i]), middle = __half2float(m[i]);
    float v[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      v[j] = scale * (float)((int)((w[i] >> (4 * j)) & 15) - 8);   // exact: 11 + 4 bits
      if (middles) v[j] = __fadd_rn(v[j], middle);
    }
    float* dst = to + col;
    if (have == 8 && !apart) {
      *VSK_CHK_W(reinterpret_cast<float4*>(dst)) = make_float4(v[0], v[1], v[2], v[3]);
      *VSK_CHK_W(reinterpret_cast<float4*>(dst + 4)) = make_float4(v[4], v[5], v[6], v[7]);
    } else if (!apart) {
      for (int j = 0; j < have; ++j) *VSK_CHK_W(dst + j) = v[j];
    } else {
      // A warp's rows of this step follow one another in memory: a part of one row, or (short rows) several whole ones.
      const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, span = min(lanes * 8, end - base);
      float* const at = staged[warp] + (lane / lanes) * span + (col - base);
      for (int j = 0; j < have; ++j) at[j] = v[j];
      __syncwarp();
      const int64_t row0 = row - lane / lanes;   // the warp's first
      const int rows = (int)min((int64_t)(32 / lanes), max((int64_t)0, n - row0));
      float* const all = out + row0 * dim + base;
      for (int e = lane; e < rows * span; e += 32) *VSK_CHK_W(all + e) = staged[warp][e];
      __syncwarp();
    }
  }
}

int32_t check_ctx(vsk_ctx* c, Ctx** ctx) {
  *ctx = reinterpret_cast<Ctx*>(c);
  if (!*ctx) return VSK_ERR_INVALID_INPUT;
  cudaSetDevice((*ctx)->device);
  return VSK_OK;
}

// Elements of one array, and bytes that rows reach over: no size in bytes is computed past 64 bits.
constexpr int64_t kMost = 1ll << 56;

int32_t check_shape(Ctx* ctx, int64_t n, int32_t dim, int32_t group) {
  if (n <= 0) return fail(ctx, VSK_ERR_EMPTY_INPUT, "no rows");
  if (n > (1ll << 40)) return fail(ctx, VSK_ERR_INVALID_BUFFER_SIZE, "too many rows");
  if (dim <= 0 || dim > (1 << 24)) return fail(ctx, VSK_ERR_DIMENSION_MISMATCH, "dimension must be in [1, 2^24]");
  if (group != 32 && group != 64 && group != 128)
    return fail(ctx, VSK_ERR_UNSUPPORTED_OPERATION, "groups of %d columns are not supported (32, 64 or 128)", group);
  if (n > kMost / dim) return fail(ctx, VSK_ERR_INVALID_BUFFER_SIZE, "too many rows of %d columns", dim);
  return VSK_OK;
}

int32_t check_rows(Ctx* ctx, const vsk_q4_rows* r) {
  if (!r) return fail(ctx, VSK_ERR_INVALID_INPUT, "null rows");
  VSK_TRY(check_shape(ctx, r->n, r->dim, r->group));
  if (!r->codes || !r->scales) return fail(ctx, VSK_ERR_INVALID_INPUT, "null codes or scales");
  if (r->code_stride < ((int64_t)r->dim + 1) / 2) return fail(ctx, VSK_ERR_INVALID_BUFFER_SIZE, "code rows are shorter than %d columns", r->dim);
  if (r->scale_stride < ceil_div(r->dim, r->group)) return fail(ctx, VSK_ERR_INVALID_BUFFER_SIZE, "scale rows are shorter than the groups of %d columns", r->dim);
  if (r->n > 1 && std::max(r->code_stride, r->scale_stride) > kMost / r->n)
    return fail(ctx, VSK_ERR_INVALID_BUFFER_SIZE, "the distance of code or scale rows is too large");
  if ((reinterpret_cast<uintptr_t>(r->scales) & 1) || (reinterpret_cast<uintptr_t>(r->middles) & 1))
    return fail(ctx, VSK_ERR_INVALID_INPUT, "scales and middles must be aligned to two bytes");
  return VSK_OK;
}

int dtype_size(int32_t t) { return t == VSK_DTYPE_F32 ? 4 : (t == VSK_DTYPE_F16 || t == VSK_DTYPE_BF16) ? 2 : 0; }

int32_t encode(Ctx* ctx, const void* rows, int32_t dtype, int64_t n, int32_t dim, int64_t row_stride, int32_t group, int32_t symmetric,
               uint8_t* codes, int64_t code_stride, void* scales, void* middles) {
  const int es = dtype_size(dtype);
  const int groups = (int)ceil_div(dim, group);
  const int wide = ((reinterpret_cast<uintptr_t>(rows) | (uintptr_t)(row_stride * es)) & 15) == 0;
  int lanes = group / 8;
  while (lanes < 32 && lanes * 8 < dim) lanes *= 2;
  const int columns = 1024;   // of a thread's walk: a multiple of every stride and group
  const int64_t blocks = ceil_div(n, 256 / lanes), along = ceil_div(dim, columns);
  if (blocks > 0x7fffffffLL) return fail(ctx, VSK_ERR_INVALID_BUFFER_SIZE, "too many rows in one call");
  auto go = [&](auto* x) {
    using T = std::remove_const_t<std::remove_pointer_t<decltype(x)>>;
    const dim3 grid((unsigned)blocks, (unsigned)along);
    auto kernel = symmetric ? (wide ? q4_encode_kernel<T, true, true> : q4_encode_kernel<T, true, false>)
                            : (wide ? q4_encode_kernel<T, false, true> : q4_encode_kernel<T, false, false>);
    kernel<<<grid, 256, 0, ctx->stream>>>(x, n, dim, row_stride, group, groups, lanes, columns, codes, code_stride, (__half*)scales, (__half*)middles);
  };
  if (dtype == VSK_DTYPE_F32) go((const float*)rows);
  else if (dtype == VSK_DTYPE_F16) go((const __half*)rows);
  else go((const __nv_bfloat16*)rows);
  ctx->stats.kernel_launches++;
  VSK_CUDA(ctx, cudaGetLastError());
  return VSK_OK;
}

int32_t decode(Ctx* ctx, const vsk_q4_rows* r, float* out) {
  int lanes = 1;
  while (lanes < 32 && lanes * 8 < r->dim) lanes *= 2;
  const int columns = kDecodeSteps * lanes * 8;
  const int64_t blocks = ceil_div(r->n, 256 / lanes);
  if (blocks > 0x7fffffffLL) return fail(ctx, VSK_ERR_INVALID_BUFFER_SIZE, "too many rows in one call");
  q4_decode_kernel<<<dim3((unsigned)blocks, (unsigned)ceil_div(r->dim, columns)), 256, 0, ctx->stream>>>(
      r->codes, r->code_stride, (const __half*)r->scales, (const __half*)r->middles, r->scale_stride, r->n, r->dim,
      r->group == 32 ? 5 : r->group == 64 ? 6 : 7, lanes, columns, out);
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
  tl_mark(ctx, "q4_encode");
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
  const int64_t width = (dim + 1) / 2;
  const size_t in = (size_t)n * dim * 4, held = (size_t)n * width, per = (size_t)n * ceil_div(dim, group) * 2;
  Staged s(ctx);
  void *dx, *dc, *ds, *dm = nullptr;
  VSK_TRY(s.get(in, &dx));
  VSK_TRY(s.get(held, &dc));
  VSK_TRY(s.get(per, &ds));
  if (!symmetric) VSK_TRY(s.get(per, &dm));
  VSK_CUDA(ctx, cudaMemcpyAsync(dx, rows, in, cudaMemcpyHostToDevice, ctx->stream));
  VSK_TRY(encode(ctx, dx, VSK_DTYPE_F32, n, dim, dim, group, symmetric, (uint8_t*)dc, width, ds, dm));
  // (bytes of a code row behind its columns are the caller's)
  VSK_CUDA(ctx, cudaMemcpy2DAsync(codes, (size_t)code_stride, dc, (size_t)width, (size_t)width, (size_t)n, cudaMemcpyDeviceToHost, ctx->stream));
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
  if (reinterpret_cast<uintptr_t>(out) & 3) return fail(ctx, VSK_ERR_INVALID_INPUT, "a pointer is not aligned to its element");
  drain_stale_error("vsk_q4_decode_dev");
  VSK_TRY(decode(ctx, rows, out));
  tl_mark(ctx, "q4_decode");
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
  // 200 000 x 2 048, groups of 128 / of 32 with middles: four fp16 vectors take 74 / 123 us in whole numbers and 91 / 143 in 16 bits, six
  // 99 / 175 and 91 / 143 (they no longer fit two tiles of digits).  fp32 vectors have no 16-bit form.
  if (x_dtype == VSK_DTYPE_F32 || nq <= 4) VSK_TRY(q4_product_digits(ctx, *rows, x, x_dtype, nq, x_stride, y, y_dtype, y_stride));
  else if (q4_fits_tensor(ctx, *rows, nq)) return q4_product_tensor(ctx, *rows, x, x_dtype, nq, x_stride, y, y_dtype, y_stride);
  else VSK_TRY(q4_product(ctx, *rows, x, x_dtype, nq, x_stride, y, y_dtype, y_stride));
  tl_mark(ctx, "q4_product");
  VSK_CUDA(ctx, cudaStreamSynchronize(ctx->stream));
  return VSK_OK;
}

}  // extern "C"
