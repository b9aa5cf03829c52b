// Products with rows in four bits: what int4.cu (checks, entry points) asks of int4_product.cu.
#pragma once
#include <algorithm>

#include "common.cuh"

namespace vsk {

// y[q * y_stride + r] = sum over columns of (value of row r) x[q * x_stride + column]; arguments checked by the caller.
int32_t q4_product(Ctx* ctx, const vsk_q4_rows& rows, const void* x, int32_t x_dtype, int64_t nq, int64_t x_stride, void* y,
                   int32_t y_dtype, int64_t y_stride);

// The same in whole numbers, for a few vectors (int4_digits.cu).
int32_t q4_product_digits(Ctx* ctx, const vsk_q4_rows& rows, const void* x, int32_t x_dtype, int64_t nq, int64_t x_stride, void* y,
                          int32_t y_dtype, int64_t y_stride);

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
