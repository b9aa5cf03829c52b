// Products of a few vectors with rows held in four bits (int4.cu has the format).
//
// A decoding step multiplies one token, or the beams of a search, with all rows: every code is read once and used for a handful
// of products, so the call is bound by the bytes of the codes and scales.  The fp32 pipes would not keep up with them - 13 000
// billion codes a second are 46 per SM and clock, and a conversion, a multiply-add and the unpacking are three to four instructions each
// of the 128 a clock - so the products run on the tensor cores' warp form (m16n8k16, fp32 sums): a code becomes an exact 16-bit number
// in about one instruction, and eight vectors, or three parts of two fp32 ones, share it.
//
//   codes    16 (or 32) rows x 128 columns at a time into a ring in shared memory that belongs to ONE warp: asynchronous 16-byte
//            copies, no block-wide barrier.  The four 16-byte pieces of a row are stored in the order piece ^ (row / 2 % 4), so that the
//            four-byte reads of eight rows fall into 32 different banks.
//   x        in 16 bits as it is, or, for fp32, as three bf16 parts of 8 bits whose sum is the value: the products are exact and the
//            result is the fp32 one.  The parts are columns of their own and are added at the end.
//   scales   each group's sum is taken in fp32 registers, multiplied by the scale there and added to the row's total: codes are never
//            multiplied by a rounded weight.
#include <cuda_bf16.h>

#include <algorithm>

#include "int4.cuh"

namespace vsk {
namespace {

constexpr int kWarps = 8;

struct ProductArgs {
  const uint8_t* codes;
  int64_t code_stride;
  const __half* scales;
  const __half* middles;      // or null
  int64_t scale_stride;
  int64_t n;
  int dim, groups, ksteps;    // ksteps: steps of 128 columns
  int copy;                   // bytes of one asynchronous copy of codes: 16 or 4; 1 = plain byte loads
  int pair_scales;            // the scales of a step can be read with one load
  const void* x;              // [cols][x_stride], 16 bits
  int64_t x_stride;
  const float* xsum;          // [groups][sum_stride]: sums of x over a group, 0 in columns that are not a vector's first part
  int sum_stride;
  int x_pad;                  // columns of x that may be read (zeros behind dim)
  int64_t nq;
  int parts, per_launch;      // columns per vector; vectors per grid row
  void* y;
  int64_t y_stride;
  int y_dtype;
  int team;                   // warps that share a tile's columns (1, 2, 4 or 8)
};

__device__ __forceinline__ void copy16(uint32_t dst, const void* src, int bytes) {   // bytes behind `bytes` become zeros
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void copy4(uint32_t dst, const void* src, int bytes) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void copy_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N> __device__ __forceinline__ void copy_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

template <typename T>
__device__ __forceinline__ void mma(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  if constexpr (std::is_same<T, __half>::value) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  } else {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  }
}

// Eight codes to four pairs (code j, code j + 4) of the numbers code - 8, exactly: the code under the exponent of 1024 (fp16) or 128 (bf16)
// is that power plus the code, and the difference needs no rounding.
template <typename T>
__device__ __forceinline__ void unpack(uint32_t w, uint32_t (&p)[4]) {
  if constexpr (std::is_same<T, __half>::value) {
    const __half2 base = __half2half2(__ushort_as_half(0x6408)), scale = __half2half2(__ushort_as_half(0x2c00)),   // 1032, 1/16
                  high = __half2half2(__ushort_as_half(0xd480));                                                    // -72
    const uint32_t v = w >> 8;
    uint32_t q[4] = {(w & 0x000f000fu) | 0x64006400u, (w & 0x00f000f0u) | 0x64006400u, (v & 0x000f000fu) | 0x64006400u,
                     (v & 0x00f000f0u) | 0x64006400u};
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
      uint32_t q = ((w >> (4 * j)) & 0x000f000fu) | 0x43004300u;
      __nv_bfloat162 h = __hsub2(*reinterpret_cast<__nv_bfloat162*>(&q), base);
      p[j] = *reinterpret_cast<uint32_t*>(&h);
    }
  }
}

// GW groups per 128 columns.  (a step's scales of one row, as fp32)
template <int GW>
__device__ __forceinline__ void load_scales(const __half* __restrict__ p, int first, int groups, int pair, float (&out)[GW]) {
  if (pair && first + GW <= groups) {
    if constexpr (GW == 4) {
      const uint2 v = __ldg(reinterpret_cast<const uint2*>(p + first));
      const __half2* h = reinterpret_cast<const __half2*>(&v);
      const float2 a = __half22float2(h[0]), b = __half22float2(h[1]);
      out[0] = a.x; out[1] = a.y; out[2] = b.x; out[3] = b.y;
      return;
    } else if constexpr (GW == 2) {
      const uint32_t v = __ldg(reinterpret_cast<const uint32_t*>(p + first));
      const float2 a = __half22float2(*reinterpret_cast<const __half2*>(&v));
      out[0] = a.x; out[1] = a.y;
      return;
    }
  }
#pragma unroll
  for (int g = 0; g < GW; ++g) out[g] = first + g < groups ? __half2float(*VSK_CHK(p + first + g)) : 0.f;
}

__device__ __forceinline__ void store_y(const ProductArgs& a, int64_t at, float v) {
  if (a.y_dtype == VSK_DTYPE_F32) *VSK_CHK_W((float*)a.y + at) = v;
  else if (a.y_dtype == VSK_DTYPE_F16) *VSK_CHK_W((__half*)a.y + at) = __float2half_rn(v);
  else *VSK_CHK_W((__nv_bfloat16*)a.y + at) = __float2bfloat16_rn(v);
}

// NT tiles of eight columns of x, MT tiles of sixteen rows per warp step.
template <int NT, int MT>
struct Shape {
  static constexpr int kRows = 16 * MT;
  static constexpr int kStage = kRows * 64;
  static constexpr int kStages = MT == 1 ? 8 : 6;
  static constexpr int kLine = 8 * NT + 1;    // floats of a row of the epilogue's buffer
  static constexpr size_t kRing = (size_t)kWarps * kStages * kStage;
  static constexpr size_t kShared = kRing + (size_t)kWarps * kRows * kLine * 4;
};

template <typename T, int NT, int MT, int GW, bool MID>
__global__ void __launch_bounds__(32 * kWarps) q4_product_kernel(const ProductArgs a) {
  using S = Shape<NT, MT>;
  extern __shared__ __align__(128) uint8_t smem[];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int g = lane >> 2, t = lane & 3;   // row (and column of x) and quarter of the fragments
  const int team = a.team, teams = kWarps / team, wk = warp % team;
  uint8_t* const ring = smem + (size_t)warp * S::kStages * S::kStage;
  const uint32_t ring_addr = (uint32_t)__cvta_generic_to_shared(ring);
  float* const red = reinterpret_cast<float*>(smem + S::kRing) + (size_t)(warp / team) * team * S::kRows * S::kLine;

  const int64_t q0 = (int64_t)blockIdx.y * a.per_launch;
  const int nq = (int)min((int64_t)a.per_launch, a.nq - q0), cols = nq * a.parts;
  const T* const x = reinterpret_cast<const T*>(a.x) + q0 * a.parts * a.x_stride;

  const int64_t tiles = (a.n + S::kRows - 1) / S::kRows;
  const int64_t stride = (int64_t)gridDim.x * teams;
  const int64_t tile0 = (int64_t)blockIdx.x * teams + warp / team;
  const int64_t mine = tile0 < tiles ? (tiles - tile0 + stride - 1) / stride : 0;
  const int k0 = (int)((int64_t)a.ksteps * wk / team), k1 = (int)((int64_t)a.ksteps * (wk + 1) / team), per_tile = k1 - k0;
  const int64_t total = mine * per_tile;
  const int row_bytes = (a.dim + 1) / 2;

  // one step's codes into a stage of the ring (rows behind the last one repeat it, bytes behind a row's end are zeros: their columns of x are)
  int64_t f_tile = tile0;
  int f_k = k0, f_slot = 0;
  int64_t fetched = 0;
  auto fetch = [&]() {
    if (fetched < total) {
      const int64_t row0 = f_tile * S::kRows;
      const int byte0 = f_k * 64;
      const uint32_t stage = ring_addr + f_slot * S::kStage;
      if (a.copy == 16) {
#pragma unroll
        for (int j = 0; j < 2 * MT; ++j) {
          const int id = lane + 32 * j, r = id >> 2, piece = id & 3, at = byte0 + piece * 16;
          const int64_t row = min(row0 + r, a.n - 1);
          const int have = max(0, min(16, row_bytes - at));
          const uint8_t* src = a.codes + row * a.code_stride + (have ? at : 0);
          copy16(stage + r * 64 + ((piece ^ (r >> 1)) & 3) * 16, have == 16 ? (const void*)VSK_CHK((const uint4*)src) : src, have);
        }
      } else if (a.copy == 4) {
#pragma unroll
        for (int j = 0; j < 8 * MT; ++j) {
          const int id = lane + 32 * j, r = id >> 4, word = id & 15, at = byte0 + word * 4;
          const int64_t row = min(row0 + r, a.n - 1);
          const int have = max(0, min(4, row_bytes - at));
          const uint8_t* src = a.codes + row * a.code_stride + (have ? at : 0);
          copy4(stage + r * 64 + (((word >> 2) ^ (r >> 1)) & 3) * 16 + (word & 3) * 4, have == 4 ? (const void*)VSK_CHK((const uint32_t*)src) : src,
                have);
        }
      } else {
        for (int j = 0; j < 8 * MT; ++j) {
          const int id = lane + 32 * j, r = id >> 4, word = id & 15, at = byte0 + word * 4;
          const int64_t row = min(row0 + r, a.n - 1);
          const uint8_t* src = a.codes + row * a.code_stride + at;
          uint32_t w = 0;
          for (int b = 0; b < 4; ++b)
            if (at + b < row_bytes) w |= (uint32_t)*VSK_CHK(src + b) << (8 * b);
          *reinterpret_cast<uint32_t*>(ring + f_slot * S::kStage + r * 64 + (((word >> 2) ^ (r >> 1)) & 3) * 16 + (word & 3) * 4) = w;
        }
      }
      if (++f_k == k1) {
        f_k = k0;
        f_tile += stride;
      }
      if (++f_slot == S::kStages) f_slot = 0;
    }
    ++fetched;
    copy_commit();   // (an empty group keeps the count of groups in step)
  };
#pragma unroll
  for (int s = 0; s < S::kStages - 1; ++s) fetch();

  // scales of the step at hand and of the next one, per row of the fragments
  float sc[MT][2][GW], sc_next[MT][2][GW], md[MT][2][GW], md_next[MT][2][GW];
  auto read_scales = [&](int64_t tile, int k, float (&s)[MT][2][GW], float (&m)[MT][2][GW]) {
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int64_t row = min(tile * S::kRows + i * 16 + h * 8 + g, a.n - 1);
        load_scales<GW>(a.scales + row * a.scale_stride, k * GW, a.groups, a.pair_scales, s[i][h]);
        if constexpr (MID) load_scales<GW>(a.middles + row * a.scale_stride, k * GW, a.groups, a.pair_scales, m[i][h]);
      }
  };

  float tot[MT][NT][4];
  int64_t tile = tile0;
  int k = k0, slot = 0;
  if (total > 0) read_scales(tile, k, sc_next, md_next);
  for (int64_t step = 0; step < total; ++step) {
    if (k == k0) {
#pragma unroll
      for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int j = 0; j < NT; ++j)
#pragma unroll
          for (int e = 0; e < 4; ++e) tot[i][j][e] = 0.f;
    }
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int e = 0; e < GW; ++e) {
          sc[i][h][e] = sc_next[i][h][e];
          if constexpr (MID) md[i][h][e] = md_next[i][h][e];
        }
    const bool last = k + 1 == k1;
    if (step + 1 < total) read_scales(last ? tile + stride : tile, last ? k0 : k + 1, sc_next, md_next);

    copy_wait<S::kStages - 2>();
    __syncwarp();   // everybody's copies of this step have landed, and everybody is done with the stage that is filled next
    fetch();

    const uint8_t* stage = ring + slot * S::kStage;
    if (++slot == S::kStages) slot = 0;
    float acc[MT][NT][4];
#pragma unroll
    for (int sub = 0; sub < 4; ++sub) {   // 32 columns
      constexpr int kSub = 4 / GW;
      if (sub % kSub == 0) {
#pragma unroll
        for (int i = 0; i < MT; ++i)
#pragma unroll
          for (int j = 0; j < NT; ++j)
#pragma unroll
            for (int e = 0; e < 4; ++e) acc[i][j][e] = 0.f;
      }
      const int col = k * 128 + sub * 32 + t * 8;
      uint32_t b[NT][4];
#pragma unroll
      for (int j = 0; j < NT; ++j) {
        const int c = j * 8 + g;
        uint4 v = make_uint4(0u, 0u, 0u, 0u);
        if (c < cols && col < a.x_pad) v = __ldg(reinterpret_cast<const uint4*>(x + c * a.x_stride + col));
        b[j][0] = __byte_perm(v.x, v.z, 0x5410);   // (0, 4)
        b[j][1] = __byte_perm(v.x, v.z, 0x7632);   // (1, 5)
        b[j][2] = __byte_perm(v.y, v.w, 0x5410);
        b[j][3] = __byte_perm(v.y, v.w, 0x7632);
      }
#pragma unroll
      for (int i = 0; i < MT; ++i) {
        uint32_t lo[4], hi[4];
        const int r = i * 16 + g, place = ((sub ^ (r >> 1)) & 3) * 16 + t * 4;   // (r and r + 8 share it)
        unpack<T>(*reinterpret_cast<const uint32_t*>(stage + r * 64 + place), lo);
        unpack<T>(*reinterpret_cast<const uint32_t*>(stage + (r + 8) * 64 + place), hi);
#pragma unroll
        for (int j = 0; j < NT; ++j) {
          mma<T>(acc[i][j], lo[0], hi[0], lo[1], hi[1], b[j][0], b[j][1]);
          mma<T>(acc[i][j], lo[2], hi[2], lo[3], hi[3], b[j][2], b[j][3]);
        }
      }
      if (sub % kSub == kSub - 1) {
        const int gi = sub / kSub;
#pragma unroll
        for (int j = 0; j < NT; ++j) {
          float x0 = 0.f, x1 = 0.f;
          if constexpr (MID) {
            const int c = j * 8 + 2 * t;
            if (k * GW + gi < a.groups) {
              const float* p = a.xsum + (int64_t)(k * GW + gi) * a.sum_stride + q0 * a.parts + c;
              if (c < cols) x0 = __ldg(p);
              if (c + 1 < cols) x1 = __ldg(p + 1);
            }
          }
#pragma unroll
          for (int i = 0; i < MT; ++i) {
            tot[i][j][0] = fmaf(sc[i][0][gi], acc[i][j][0], tot[i][j][0]);
            tot[i][j][1] = fmaf(sc[i][0][gi], acc[i][j][1], tot[i][j][1]);
            tot[i][j][2] = fmaf(sc[i][1][gi], acc[i][j][2], tot[i][j][2]);
            tot[i][j][3] = fmaf(sc[i][1][gi], acc[i][j][3], tot[i][j][3]);
            if constexpr (MID) {
              tot[i][j][0] = fmaf(md[i][0][gi], x0, tot[i][j][0]);
              tot[i][j][1] = fmaf(md[i][0][gi], x1, tot[i][j][1]);
              tot[i][j][2] = fmaf(md[i][1][gi], x0, tot[i][j][2]);
              tot[i][j][3] = fmaf(md[i][1][gi], x1, tot[i][j][3]);
            }
          }
        }
      }
    }

    if (last) {
      // the warps' sums meet in shared memory: columns of x in a row's line, parts and the team's shares are added on the way out
      float* const own = red + (size_t)wk * S::kRows * S::kLine;
#pragma unroll
      for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int j = 0; j < NT; ++j)
#pragma unroll
          for (int e = 0; e < 4; ++e) own[(i * 16 + g + (e >> 1) * 8) * S::kLine + j * 8 + 2 * t + (e & 1)] = tot[i][j][e];
      const int bar = 1 + warp / team;
      auto meet = [&]() {
        if (team == 1) __syncwarp();
        else asm volatile("bar.sync %0, %1;" ::"r"(bar), "r"(team * 32) : "memory");
      };
      meet();
      const int64_t row0 = tile * S::kRows;
      const int rows = (int)min((int64_t)S::kRows, a.n - row0);
      for (int o = wk * 32 + lane; o < nq * S::kRows; o += team * 32) {
        const int r = o % S::kRows, q = o / S::kRows;
        float v = 0.f;
        for (int p = a.parts - 1; p >= 0; --p)   // the small parts first
          for (int w = 0; w < team; ++w) v += red[((size_t)w * S::kRows + r) * S::kLine + q * a.parts + p];
        if (r < rows) store_y(a, (q0 + q) * a.y_stride + row0 + r, v);
      }
      meet();
      tile += stride;
      k = k0;
    } else {
      ++k;
    }
  }
}

// x to 16-bit columns of whole steps (zeros behind dim), and its sums over the groups.  One thread per eight columns of one vector.
template <typename X, typename T>
__global__ void __launch_bounds__(128) q4_prepare_kernel(const X* __restrict__ x, int64_t x_stride, int dim, int padded, int parts, int group,
                                                         int groups, T* __restrict__ out, float* __restrict__ sums, int sum_stride) {
  const int64_t q = blockIdx.y;
  const int col = ((int)blockIdx.x * 128 + (int)threadIdx.x) * 8;
  float v[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    v[j] = 0.f;
    if (col + j < dim) {
      const X e = *VSK_CHK(x + q * x_stride + col + j);
      if constexpr (std::is_same<X, float>::value) v[j] = e;
      else if constexpr (std::is_same<X, __half>::value) v[j] = __half2float(e);
      else v[j] = __bfloat162float(e);
    }
  }
  if (sums) {
    float s = ((v[0] + v[1]) + (v[2] + v[3])) + ((v[4] + v[5]) + (v[6] + v[7]));
    for (int o = group / 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
    if (col % group == 0 && col / group < groups) {
      float* at = sums + (int64_t)(col / group) * sum_stride + q * parts;
      for (int p = 0; p < parts; ++p) *VSK_CHK_W(at + p) = p == 0 ? s : 0.f;
    }
  }
  if (col >= padded) return;
  for (int p = 0; p < parts; ++p) {
    __align__(16) T h[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      if constexpr (std::is_same<X, float>::value) {
        // the leading eight bits, cut off rather than rounded: what is left is exact, and the largest numbers stay finite
        const float top = __uint_as_float(__float_as_uint(v[j]) & 0xffff0000u);
        h[j] = __float2bfloat16_rn(top);
        v[j] = isfinite(top) ? v[j] - top : 0.f;   // (an infinity or a NaN is all in the first part)
        if (p == 0 && !isfinite(top)) h[j] = __float2bfloat16_rn(__uint_as_float(__float_as_uint(x[q * x_stride + col + j])));
      } else {
        h[j] = (col + j < dim) ? x[q * x_stride + col + j] : T(0.f);
      }
    }
    *VSK_CHK_W(reinterpret_cast<uint4*>(out + (q * parts + p) * padded + col)) = *reinterpret_cast<const uint4*>(h);
  }
}

template <typename T, int NT, int MT, int GW, bool MID>
int32_t launch(Ctx* ctx, const ProductArgs& a0) {
  using S = Shape<NT, MT>;
  ProductArgs a = a0;
  auto kernel = q4_product_kernel<T, NT, MT, GW, MID>;
  VSK_CUDA(ctx, opt_in_shared(ctx, kernel, S::kShared));
  a.per_launch = 8 * NT / a.parts;
  const int64_t chunks = ceil_div(a.nq, a.per_launch);
  const int per_sm = resident_blocks(ctx, kernel, 32 * kWarps, S::kShared);
  const int64_t slots = (int64_t)ctx->prop.multiProcessorCount * per_sm * kWarps;   // warps that run at once
  const int64_t tiles = ceil_div(a.n, S::kRows);
  // few rows: warps of a block share a tile's columns until the device is full
  a.team = 1;
  while (a.team < kWarps && 2 * a.team <= a.ksteps && tiles * a.team * chunks < slots) a.team *= 2;
  const int64_t blocks = std::min(ceil_div(tiles, kWarps / a.team), std::max<int64_t>(1, slots / kWarps / chunks));
  for (int64_t c = 0; c < chunks; c += 65535) {
    const int64_t here = std::min<int64_t>(65535, chunks - c);
    ProductArgs b = a;
    const int64_t q = c * a.per_launch;
    b.nq = std::min(a.nq - q, here * a.per_launch);
    b.x = (const uint16_t*)a.x + q * a.parts * a.x_stride;
    if (MID) b.xsum = a.xsum + q * a.parts;
    b.y = (uint8_t*)a.y + q * a.y_stride * (a.y_dtype == VSK_DTYPE_F32 ? 4 : 2);
    kernel<<<dim3((unsigned)blocks, (unsigned)here), 32 * kWarps, S::kShared, ctx->stream>>>(b);
    ctx->stats.kernel_launches++;
    VSK_CUDA(ctx, cudaGetLastError());
  }
  return VSK_OK;
}

template <typename T, int NT, int MT>
int32_t by_group(Ctx* ctx, const ProductArgs& a, int group) {
  const bool mid = a.middles != nullptr;
  switch (group) {
    case 32: return mid ? launch<T, NT, MT, 4, true>(ctx, a) : launch<T, NT, MT, 4, false>(ctx, a);
    case 64: return mid ? launch<T, NT, MT, 2, true>(ctx, a) : launch<T, NT, MT, 2, false>(ctx, a);
    default: return mid ? launch<T, NT, MT, 1, true>(ctx, a) : launch<T, NT, MT, 1, false>(ctx, a);
  }
}

template <typename T>
int32_t by_columns(Ctx* ctx, const ProductArgs& a, int group) {
  const int64_t cols = a.nq * a.parts;
  if (cols <= 8) return by_group<T, 1, 1>(ctx, a, group);
  if (cols <= 16) return by_group<T, 2, 2>(ctx, a, group);
  return by_group<T, 4, 2>(ctx, a, group);
}

}  // namespace

int32_t q4_product(Ctx* ctx, const vsk_q4_rows& rows, const void* x, int32_t x_dtype, int64_t nq, int64_t x_stride, void* y,
                   int32_t y_dtype, int64_t y_stride) {
  ProductArgs a{};
  a.codes = rows.codes;
  a.code_stride = rows.code_stride;
  a.scales = (const __half*)rows.scales;
  a.middles = (const __half*)rows.middles;
  a.scale_stride = rows.scale_stride;
  a.n = rows.n;
  a.dim = rows.dim;
  a.groups = (int)ceil_div(rows.dim, rows.group);
  a.ksteps = (int)ceil_div(rows.dim, 128);
  const uintptr_t code_bits = reinterpret_cast<uintptr_t>(rows.codes) | (uintptr_t)rows.code_stride;
  a.copy = (code_bits & 15) == 0 ? 16 : (code_bits & 3) == 0 ? 4 : 1;
  const int gw = 128 / rows.group;
  const uintptr_t scale_bits = reinterpret_cast<uintptr_t>(rows.scales) | reinterpret_cast<uintptr_t>(rows.middles) | (uintptr_t)(2 * rows.scale_stride);
  a.pair_scales = (scale_bits & (uintptr_t)(2 * gw - 1)) == 0;
  a.nq = nq;
  a.y = y;
  a.y_stride = y_stride;
  a.y_dtype = y_dtype;
  a.parts = x_dtype == VSK_DTYPE_F32 ? 3 : 1;
  const bool as_is = x_dtype != VSK_DTYPE_F32 && !rows.middles && rows.dim % 8 == 0 && x_stride % 8 == 0 &&
                     (reinterpret_cast<uintptr_t>(x) & 15) == 0;
  if (as_is) {
    a.x = x;
    a.x_stride = x_stride;
    a.x_pad = rows.dim;
  } else {
    const int padded = a.ksteps * 128;
    const int64_t cols = nq * a.parts;
    void *p, *s = nullptr;
    VSK_TRY(scratch(ctx, SLOT_Q16, (size_t)cols * padded * 2, &p));
    a.sum_stride = (int)((cols + 3) / 4 * 4);
    if (rows.middles) VSK_TRY(scratch(ctx, SLOT_QAUX, (size_t)a.groups * a.sum_stride * 4, &s));
    for (int64_t q = 0; q < nq; q += 65535) {
      const dim3 grid((unsigned)ceil_div(padded / 8, 128), (unsigned)std::min<int64_t>(65535, nq - q));
      float* sums = s ? (float*)s + q * a.parts : nullptr;
      uint16_t* to = (uint16_t*)p + q * a.parts * padded;
      if (x_dtype == VSK_DTYPE_F32)
        q4_prepare_kernel<float, __nv_bfloat16><<<grid, 128, 0, ctx->stream>>>((const float*)x + q * x_stride, x_stride, a.dim, padded, 3,
                                                                              rows.group, a.groups, (__nv_bfloat16*)to, sums, a.sum_stride);
      else if (x_dtype == VSK_DTYPE_F16)
        q4_prepare_kernel<__half, __half><<<grid, 128, 0, ctx->stream>>>((const __half*)x + q * x_stride, x_stride, a.dim, padded, 1, rows.group,
                                                                        a.groups, (__half*)to, sums, a.sum_stride);
      else
        q4_prepare_kernel<__nv_bfloat16, __nv_bfloat16><<<grid, 128, 0, ctx->stream>>>((const __nv_bfloat16*)x + q * x_stride, x_stride, a.dim,
                                                                                      padded, 1, rows.group, a.groups, (__nv_bfloat16*)to, sums,
                                                                                      a.sum_stride);
      ctx->stats.kernel_launches++;
      VSK_CUDA(ctx, cudaGetLastError());
    }
    a.x = p;
    a.x_stride = padded;
    a.x_pad = padded;
    a.xsum = (const float*)s;
  }
  return x_dtype == VSK_DTYPE_F16 ? by_columns<__half>(ctx, a, rows.group) : by_columns<__nv_bfloat16>(ctx, a, rows.group);
}

}  // namespace vsk
