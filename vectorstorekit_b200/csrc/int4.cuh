// Products with rows in four bits: what int4.cu (checks, entry points) asks of the other files.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>
#include <type_traits>

#include "common.cuh"

namespace vsk {

// y[q * y_stride + r] = sum over columns of (value of row r) x[q * x_stride + column]; arguments checked by the caller.
int32_t q4_product(Ctx* ctx, const vsk_q4_rows& rows, const void* x, int32_t x_dtype, int64_t nq, int64_t x_stride, void* y,
                   int32_t y_dtype, int64_t y_stride);

// The same in whole numbers, for a few vectors (int4_digits.cu).
int32_t q4_product_digits(Ctx* ctx, const vsk_q4_rows& rows, const void* x, int32_t x_dtype, int64_t nq, int64_t x_stride, void* y,
                          int32_t y_dtype, int64_t y_stride);

// The same on the tensor cores' block form, for more than 16 vectors and rows at 16-byte places that fill the machine (int4_tensor.cu).
bool q4_fits_tensor(Ctx* ctx, const vsk_q4_rows& rows, int64_t nq);
int32_t q4_product_tensor(Ctx* ctx, const vsk_q4_rows& rows, const void* x, int32_t x_dtype, int64_t nq, int64_t x_stride, void* y,
                          int32_t y_dtype, int64_t y_stride);

__device__ __forceinline__ void copy16(uint32_t dst, const void* src, int bytes) {   // bytes behind `bytes` become zeros
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void copy4(uint32_t dst, const void* src, int bytes) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void copy_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N> __device__ __forceinline__ void copy_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }
__device__ __forceinline__ void wait_for_launches_before() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
__device__ __forceinline__ void let_the_next_launch_begin() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }

// The vectors as the caller has them, for products that are taken one by one.
struct Vectors {
  const void* x;
  int64_t stride;
  int dtype;
  __device__ __forceinline__ float at(int64_t q, int64_t column) const {
    const int64_t e = q * stride + column;
    if (dtype == VSK_DTYPE_F32) return *VSK_CHK((const float*)x + e);
    if (dtype == VSK_DTYPE_F16) return __half2float(*VSK_CHK((const __half*)x + e));
    return __bfloat162float(*VSK_CHK((const __nv_bfloat16*)x + e));
  }
};

// The product of one row with a vector that holds an infinity or a NaN, from the definition: each value s (c - 8) + m first.  (The sums of
// s (c - 8) x and of m x are two infinities that need not agree, or 0 times one.)
template <typename Args>
__device__ __noinline__ float plain_product(const Args& a, const Vectors& x, int64_t row, int64_t q) {
  float sum = 0.f;
  for (int i = 0; i < a.dim; ++i) {
    const uint8_t b = *VSK_CHK(a.codes + row * a.code_stride + (i >> 1));
    const int c = (int)((i & 1) ? b >> 4 : b & 15) - 8;
    float v = __half2float(*VSK_CHK(a.scales + row * a.scale_stride + i / a.group)) * (float)c;
    if (a.middles) v += __half2float(*VSK_CHK(a.middles + row * a.scale_stride + i / a.group));
    sum = fmaf(v, x.at(q, i), sum);
  }
  return sum;
}

__device__ __forceinline__ uint32_t and_or(uint32_t w, uint32_t mask, uint32_t bits) {   // (w & mask) | bits, in one instruction
  uint32_t r;
  asm("lop3.b32 %0, %1, %2, %3, 0xea;" : "=r"(r) : "r"(w), "r"(mask), "r"(bits));
  return r;
}

// Eight codes to four pairs (code j, code j + 4) of the numbers code - 8, exactly: the code under the exponent of 1024 (fp16) or 128 (bf16)
// is that power plus the code, and the difference needs no rounding.
template <typename T>
__device__ __forceinline__ void unpack(uint32_t w, uint32_t (&p)[4]) {
  if constexpr (std::is_same<T, __half>::value) {
    const __half2 base = __half2half2(__ushort_as_half(0x6408)), scale = __half2half2(__ushort_as_half(0x2c00)),   // 1032, 1/16
                  high = __half2half2(__ushort_as_half(0xd480));                                                    // -72
    const uint32_t v = w >> 8;
    uint32_t q[4] = {and_or(w, 0x000f000fu, 0x64006400u), and_or(w, 0x00f000f0u, 0x64006400u), and_or(v, 0x000f000fu, 0x64006400u),
                     and_or(v, 0x00f000f0u, 0x64006400u)};
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      __half2 h = *reinterpret_cast<__half2*>(&q[j]);
      h = (j & 1) ? __hfma2(h, scale, high) : __hsub2(h, base);   // (1024 + 16 c) / 16 - 72 = c - 8
      p[j] = *reinterpret_cast<uint32_t*>(&h);
    }
  } else {
    const __nv_bfloat162 base = __bfloat162bfloat162(__ushort_as_bfloat16(0x4308));   // 136
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      uint32_t q = and_or(w >> (4 * j), 0x000f000fu, 0x43004300u);
      __nv_bfloat162 h = __hsub2(*reinterpret_cast<__nv_bfloat162*>(&q), base);
      p[j] = *reinterpret_cast<uint32_t*>(&h);
    }
  }
}

// Warps of a block that share a tile's columns: what leaves the busiest warp the fewest steps (a tile's end counts as one), tiles being dealt
// out to `slots` warps.  39 865 x 7 680, one fp16 vector: one warp each 60 steps for half the warps, eight 5 x 8.
inline int q4_team(int64_t tiles, int ksteps, int64_t slots, int most) {
  int best = 1;
  int64_t least = 0;
  for (int team = 1; team <= most && (team == 1 || team <= ksteps); team *= 2) {
    const int64_t cost = ceil_div(tiles, std::max<int64_t>(1, slots / team)) * (ceil_div(ksteps, team) + 1);
    if (team == 1 || cost < least) {
      least = cost;
      best = team;
    }
  }
  return best;
}

}  // namespace vsk
