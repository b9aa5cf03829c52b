// Products of a few vectors with rows held in four bits, in whole numbers (int4.cu has the format, int4_product.cu the form for more vectors).
//
// With one vector the call is bound by the bytes of the rows as long as unpacking keeps up with them: 6.5 TB/s are 46 codes per SM and
// clock.  A code in the high half of a byte, its top bit turned, IS the signed byte 16 (code - 8): eight codes take three
// instructions, a third of what any 16-bit form takes.  So x comes in whole numbers too.  Each vector is scaled by a power of two until
// its largest element fills four signed bytes and rounded there, by at most 2^-31 of that element: an fp32 sum that contains it rounds by
// a hundred times as much.  (A row with no weight there sees that rounding alone: elements below it are lost to such a row.)  The bytes are columns of their own in m16n8k32 products, a tile of eight holds two vectors; group sums are exact
// whole numbers, become fp32 (a magic constant is the products' starting value: its difference is the number) and meet the scale there.
// A vector with an infinity or a NaN has no such form: its products are taken one by one in fp32.
//
//   codes   32 rows x 128 columns (2 KB) per step into a ring in shared memory that belongs to ONE warp, by asynchronous 16-byte copies.  A
//           lane's words of a group lie side by side where the group is that wide (one read of 16 bytes for groups of 128 columns, two of
//           8, four of 4), and the pieces of a row are turned so that the rows read together fall into different banks
//   digits  prepared by a kernel of their own in the order of the fragments: 32 bytes per lane, step and eight of them, from L1 a step ahead.
//           The product kernel is launched with it and has its first codes under way before it waits for it.
//   scales  asked for by the row's lane two steps ahead, handed to the fragments' lanes as fp32 numbers in shared memory
//   middles a row's middles times the vectors' group sums, in the row's lane
//
// 1 000 000 x 768, groups of 32 with middles, one fp32 vector (480 MB): 96 us, 5.0 TB/s, 0.77 of a copy's rate, issue slots 65 % busy (150
// instructions for 16 rows x 128 columns: 24 unpack, 40 scale and sum the four groups).  200 000 x 2 048, groups of 128, one fp16 vector:
// 43 us, 4.9 TB/s.  16-bit products of the same shape took three times as long, 32 rows with digits on the left side 1.2 times.
#include <cuda_bf16.h>

#include <algorithm>
#include <climits>

#include "int4.cuh"

namespace vsk {
namespace {

constexpr int kWarps = 8;
constexpr int kDigits = 4;           // of a vector's numbers
constexpr int kMagic = 0x4b400000;   // the bits of 1.5 2^23: that many more as a whole number is as much more as an fp32 number

struct VectorInfo {
  int exponent;    // the vector's numbers are its digits times 2^exponent; INT_MIN: not finite
};

struct DigitArgs {
  const uint8_t* codes;
  int64_t code_stride;
  const __half* scales;
  const __half* middles;      // or null
  int64_t scale_stride;
  int64_t n;
  int dim, groups, ksteps, group;
  int copy;                   // bytes of one asynchronous copy of codes: 16 or 4; 1 = plain byte loads
  int pair_scales;            // a step's scales (and middles) of a row can be read at once
  const uint4* frags;         // [chunk][kstep][tile of 8 columns][2][32 lanes]
  const float* sums;          // [vector][sum_stride]: sums of x over the groups (zeros behind the last)
  int sum_stride;
  const VectorInfo* info;     // [vector]
  Vectors x;                  // for those that are not finite
  int64_t nq;
  int per_launch;             // vectors per grid row
  void* y;
  int64_t y_stride;
  int y_dtype;
  int team;                   // warps that share a tile's columns (1, 2, 4 or 8)
};


// codes (16 rows x 32 columns) times digits (32 columns x 8 of them)
__device__ __forceinline__ void mma(int (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1, const int (&c)[4]) {
  asm volatile("mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%11,%12,%13};"
               : "=r"(d[0]), "=r"(d[1]), "=r"(d[2]), "=r"(d[3])
               : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "r"(c[0]), "r"(c[1]), "r"(c[2]), "r"(c[3]));
}

// Two fp32 numbers in one register pair: one instruction for both.
typedef unsigned long long f32x2;
__device__ __forceinline__ f32x2 pair_of(float lo, float hi) {
  f32x2 r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(lo), "f"(hi));
  return r;
}
__device__ __forceinline__ void unpair(f32x2 v, float& lo, float& hi) { asm("mov.b64 {%0, %1}, %2;" : "=f"(lo), "=f"(hi) : "l"(v)); }
__device__ __forceinline__ f32x2 add2(f32x2 a, f32x2 b) {
  f32x2 r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ f32x2 fma2(f32x2 a, f32x2 b, f32x2 c) {
  f32x2 r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}

__device__ __forceinline__ void store_y(const DigitArgs& a, int64_t at, float v) {
  if (a.y_dtype == VSK_DTYPE_F32) *VSK_CHK_W((float*)a.y + at) = v;
  else if (a.y_dtype == VSK_DTYPE_F16) *VSK_CHK_W((__half*)a.y + at) = __float2half_rn(v);
  else *VSK_CHK_W((__nv_bfloat16*)a.y + at) = __float2bfloat16_rn(v);
}

__device__ __forceinline__ uint32_t masked_turned(uint32_t w) {   // (w & 0xf0f0f0f0) ^ 0x80808080, in one instruction
  uint32_t r;
  asm("lop3.b32 %0, %1, %2, %3, 0x6a;" : "=r"(r) : "r"(w), "r"(0xf0f0f0f0u), "r"(0x80808080u));
  return r;
}

// DT tiles of eight digits; 32 rows per warp step.
template <int DT>
struct Shape {
  static constexpr int kStage = 32 * 64;
  static constexpr int kStages = DT == 4 ? 6 : 4;
  static constexpr int kVectors = DT * 8 / kDigits;
  static constexpr int kLine = 8 * DT + kVectors + 1;        // floats of a row of the epilogue's buffer: digits, then middles' share per vector
  static constexpr int kScales = 2 * 32 * 4;                 // two steps' scales
  static constexpr size_t kRing = (size_t)kWarps * kStages * kStage;
  static constexpr size_t kShared = kRing + (size_t)kWarps * (kScales + 32 * kLine) * 4;
};

// The place of a row's 16-byte piece in a stage.
template <int GW>
__device__ __forceinline__ int turned(int row, int piece) {
  return GW == 2 ? piece ^ (((row >> 2) & 1) | (row & 2)) : (piece ^ (row >> 1)) & 3;
}

// GW groups per 128 columns.  WIDE: codes by 16-byte copies (addresses and distances of rows are multiples of 16), else by words or bytes.
template <int DT, int GW, bool MID, bool WIDE>
__global__ void __launch_bounds__(32 * kWarps, DT == 4 ? 1 : 2) q4_digits_kernel(const __grid_constant__ DigitArgs a) {
  using S = Shape<DT>;
  extern __shared__ __align__(128) uint8_t smem[];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int g = lane >> 2, t = lane & 3;   // row (and digit) and quarter of the fragments
  const int team = a.team, wk = warp & (team - 1), in_block = warp / team;
  uint8_t* const ring = smem + warp * (S::kStages * S::kStage);
  float* const scales = reinterpret_cast<float*>(smem + S::kRing) + warp * S::kScales;   // [2][32 rows][GW]
  float* const red = reinterpret_cast<float*>(smem + S::kRing) + kWarps * S::kScales + in_block * team * 32 * S::kLine;

  const int64_t q0 = (int64_t)blockIdx.y * a.per_launch;
  const int nq = (int)min((int64_t)a.per_launch, a.nq - q0);

  const int tiles = (int)((a.n + 31) / 32);   // (the host keeps their number and one more stride below 2^31)
  const int stride = gridDim.x * (kWarps / team);
  const int tile0 = blockIdx.x * (kWarps / team) + in_block;
  const int k0 = a.ksteps * wk / team, k1 = a.ksteps * (wk + 1) / team;
  const int row_bytes = (a.dim + 1) / 2;

  // the codes of one step after the other: this lane's rows (eight apart) and its place in them.  Rows behind the last one repeat it, bytes
  // behind a row's end are zeros: their digits are.
  const int f_piece = lane & 3;
  const uint8_t* f_src[WIDE ? 4 : 1];
  int f_tile = tile0, f_k = k0, f_slot = 0;
  const int tail = max(0, min(16, row_bytes - (a.ksteps - 1) * 64 - f_piece * 16));   // this lane's bytes in a row's last step
  const uint32_t f_dst = (uint32_t)__cvta_generic_to_shared(ring) + g * 64 + turned<GW>(g, f_piece) * 16;   // (the same place eight rows on)
  auto aim = [&]() {
    if constexpr (WIDE) {
#pragma unroll
      for (int j = 0; j < 4; ++j) f_src[j] = a.codes + min((int64_t)f_tile * 32 + g + 8 * j, a.n - 1) * a.code_stride + (k0 * 64 + f_piece * 16);
    }
  };
  aim();
  auto fetch = [&]() {
    if (f_tile < tiles) {
      if constexpr (WIDE) {
        const int have = f_k == a.ksteps - 1 ? tail : 16;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
#ifdef VSK_CHECKED
          const void* src = have == 16 ? (const void*)VSK_CHK((const uint4*)f_src[j]) : have ? (const void*)f_src[j] : a.codes;
#else
          const void* src = f_src[j];   // (of a copy of no bytes nothing is read)
#endif
          copy16(f_dst + f_slot * S::kStage + j * 512, src, have);
          f_src[j] += 64;
        }
      } else {
        const int at = f_k * 64 + (lane & 15) * 4, have = max(0, min(4, row_bytes - at));
        for (int j = 0; j < 16; ++j) {
          const int r = (lane >> 4) + 2 * j;
          const uint8_t* src = a.codes + min((int64_t)f_tile * 32 + r, a.n - 1) * a.code_stride + (have ? at : 0);
          uint8_t* to = ring + f_slot * S::kStage + r * 64 + turned<GW>(r, (lane >> 2) & 3) * 16 + (lane & 3) * 4;
          if (a.copy == 4) {
            copy4((uint32_t)__cvta_generic_to_shared(to), have == 4 ? (const void*)VSK_CHK((const uint32_t*)src) : src, have);
          } else {
            uint32_t w = 0;
            for (int b = 0; b < have; ++b) w |= (uint32_t)*VSK_CHK(src + b) << (8 * b);
            *reinterpret_cast<uint32_t*>(to) = w;
          }
        }
      }
      f_slot = f_slot + 1 == S::kStages ? 0 : f_slot + 1;
      if (++f_k == k1) {
        f_k = k0;
        f_tile += stride;
        aim();
      }
    }
    copy_commit();   // (an empty group keeps the count of groups in step)
  };
#pragma unroll 1
  for (int s = 0; s < S::kStages - 1; ++s) fetch();

  // Scales and middles of row `lane`, two steps ahead; behind the last tile they are the last row's.
  struct Held {
    __half s[GW], m[MID ? GW : 1];
  };
  int h_tile = tile0, h_k = k0, h_left = a.groups - k0 * GW;   // groups from this step's first on
  const __half *h_s, *h_m;
  auto aim_scales = [&]() {
    const int64_t at = min((int64_t)h_tile * 32 + lane, a.n - 1) * a.scale_stride + k0 * GW;
    h_s = a.scales + at;
    if constexpr (MID) h_m = a.middles + at;
  };
  aim_scales();
  auto read_scales = [&](Held& h) {
    bool whole = GW == 1;
    if constexpr (GW == 4) {
      if (a.pair_scales && h_left >= 4) {
        const uint2 v = __ldg(reinterpret_cast<const uint2*>(h_s));
        memcpy(h.s, &v, 8);
        if constexpr (MID) {
          const uint2 u = __ldg(reinterpret_cast<const uint2*>(h_m));
          memcpy(h.m, &u, 8);
        }
        whole = true;
      }
    } else if constexpr (GW == 2) {
      if (a.pair_scales && h_left >= 2) {
        const uint32_t v = __ldg(reinterpret_cast<const uint32_t*>(h_s));
        memcpy(h.s, &v, 4);
        if constexpr (MID) {
          const uint32_t u = __ldg(reinterpret_cast<const uint32_t*>(h_m));
          memcpy(h.m, &u, 4);
        }
        whole = true;
      }
    } else {
      h.s[0] = *VSK_CHK(h_s);   // (every step has its group)
      if constexpr (MID) h.m[0] = *VSK_CHK(h_m);
    }
    if (!whole) {
#pragma unroll
      for (int e = 0; e < GW; ++e) {
        h.s[e] = e < h_left ? *VSK_CHK(h_s + e) : __half(0.f);
        if constexpr (MID) h.m[e] = e < h_left ? *VSK_CHK(h_m + e) : __half(0.f);
      }
    }
    h_s += GW;
    if constexpr (MID) h_m += GW;
    h_left -= GW;
    if (++h_k == k1) {
      h_k = k0;
      h_left = a.groups - k0 * GW;
      h_tile += stride;
      aim_scales();
    }
  };
  auto put_scales = [&](const Held& h, int buffer) {
    float* at = scales + (buffer * 32 + lane) * GW;
    if constexpr (GW == 4) *reinterpret_cast<float4*>(at) = make_float4(__half2float(h.s[0]), __half2float(h.s[1]), __half2float(h.s[2]), __half2float(h.s[3]));
    else if constexpr (GW == 2) *reinterpret_cast<float2*>(at) = make_float2(__half2float(h.s[0]), __half2float(h.s[1]));
    else *at = __half2float(h.s[0]);
  };
  Held now, next, after;
  read_scales(now);
  read_scales(next);
  put_scales(now, 0);
  int buffer = 0;
  wait_for_launches_before();   // the digits

  const uint4* const frags = a.frags + ((int64_t)blockIdx.y * a.ksteps + k0) * (DT * 64) + lane;
  const int magic[4] = {kMagic, kMagic, kMagic, kMagic};
  const f32x2 less = pair_of(-12582912.f, -12582912.f);
  int slot = 0;
  uint4 x[DT][2], x_next[DT][2];
  const uint4* step = frags;
  int x_k = k0;
  auto read_digits = [&](uint4 (&to)[DT][2]) {
#pragma unroll
    for (int j = 0; j < DT; ++j)
#pragma unroll
      for (int h = 0; h < 2; ++h) to[j][h] = *VSK_CHK(step + j * 64 + h * 32);
    step += DT * 64;
    if (++x_k == k1) {
      x_k = k0;
      step = frags;
    }
  };
  read_digits(x_next);
  for (int tile = tile0; tile < tiles; tile += stride) {
    f32x2 tot[2][DT][2];   // digits 8 j + 2 t and the next of rows 16 i + g and 8 more
    float mid[S::kVectors];
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int j = 0; j < DT; ++j) tot[i][j][0] = tot[i][j][1] = 0ull;
    if constexpr (MID) {
#pragma unroll
      for (int v = 0; v < S::kVectors; ++v) mid[v] = 0.f;
    }
    const float* sums = MID ? a.sums + q0 * a.sum_stride + k0 * GW : nullptr;
#pragma unroll 1
    for (int k = k0; k < k1; ++k) {
#pragma unroll
      for (int j = 0; j < DT; ++j)
#pragma unroll
        for (int h = 0; h < 2; ++h) x[j][h] = x_next[j][h];
      read_digits(x_next);
      read_scales(after);

      copy_wait<S::kStages - 2>();
      __syncwarp();   // everybody's copies and scales of this step are there, and everybody is done with what is filled next
      fetch();
      put_scales(next, buffer ^ 1);

      if constexpr (MID) {
#pragma unroll
        for (int v = 0; v < S::kVectors; ++v)
          if (v < nq) {
            float of[GW];
            if constexpr (GW == 4) {
              const float4 f = *VSK_CHK(reinterpret_cast<const float4*>(sums + v * a.sum_stride));
              of[0] = f.x; of[1] = f.y; of[2] = f.z; of[3] = f.w;
            } else {
#pragma unroll
              for (int e = 0; e < GW; ++e) of[e] = *VSK_CHK(sums + v * a.sum_stride + e);
            }
#pragma unroll
            for (int e = 0; e < GW; ++e) mid[v] = fmaf(__half2float(now.m[e]), of[e], mid[v]);
          }
        sums += GW;
      }
      now = next;
      next = after;

      const uint8_t* stage = ring + slot * S::kStage + g * 64;
      slot = slot + 1 == S::kStages ? 0 : slot + 1;
      const float* of_row = scales + (buffer * 32 + g) * GW;
      buffer ^= 1;
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        // rows 16 i + g and eight more: the lane's four words, in the order of the groups
        uint32_t lo[4], hi[4];
        const uint8_t* line = stage + i * 1024;
        if constexpr (GW == 4) {
#pragma unroll
          for (int sub = 0; sub < 4; ++sub) {
            const int at = turned<GW>(g, sub) * 16 + t * 4;
            lo[sub] = *reinterpret_cast<const uint32_t*>(line + at);
            hi[sub] = *reinterpret_cast<const uint32_t*>(line + 512 + at);
          }
        } else if constexpr (GW == 2) {
#pragma unroll
          for (int p = 0; p < 2; ++p) {
            const int at = turned<GW>(g, 2 * p + (t >> 1)) * 16 + (t & 1) * 8;
            const uint2 u = *reinterpret_cast<const uint2*>(line + at), v = *reinterpret_cast<const uint2*>(line + 512 + at);
            lo[2 * p] = u.x; lo[2 * p + 1] = u.y;
            hi[2 * p] = v.x; hi[2 * p + 1] = v.y;
          }
        } else {
          const int at = turned<GW>(g, t) * 16;
          const uint4 u = *reinterpret_cast<const uint4*>(line + at), v = *reinterpret_cast<const uint4*>(line + 512 + at);
          lo[0] = u.x; lo[1] = u.y; lo[2] = u.z; lo[3] = u.w;
          hi[0] = v.x; hi[1] = v.y; hi[2] = v.z; hi[3] = v.w;
        }
        float s_lo[GW], s_hi[GW];
        if constexpr (GW == 4) {
          const float4 u = *reinterpret_cast<const float4*>(of_row + i * 64), v = *reinterpret_cast<const float4*>(of_row + i * 64 + 32);
          s_lo[0] = u.x; s_lo[1] = u.y; s_lo[2] = u.z; s_lo[3] = u.w;
          s_hi[0] = v.x; s_hi[1] = v.y; s_hi[2] = v.z; s_hi[3] = v.w;
        } else if constexpr (GW == 2) {
          const float2 u = *reinterpret_cast<const float2*>(of_row + i * 32), v = *reinterpret_cast<const float2*>(of_row + i * 32 + 16);
          s_lo[0] = u.x; s_lo[1] = u.y;
          s_hi[0] = v.x; s_hi[1] = v.y;
        } else {
          s_lo[0] = of_row[i * 16];
          s_hi[0] = of_row[i * 16 + 8];
        }
        int acc[DT][4];
#pragma unroll
        for (int sub = 0; sub < 4; ++sub) {
          constexpr int kSub = 4 / GW;
          // even columns from the low halves, odd ones from the high halves: 16 (code - 8) as signed bytes
          const uint32_t a0 = masked_turned(lo[sub] << 4), a1 = masked_turned(hi[sub] << 4), a2 = masked_turned(lo[sub]), a3 = masked_turned(hi[sub]);
#pragma unroll
          for (int j = 0; j < DT; ++j) {
            const uint4 v = x[j][sub >> 1];
            const uint32_t b0 = (sub & 1) ? v.z : v.x, b1 = (sub & 1) ? v.w : v.y;
            if (sub % kSub == 0) mma(acc[j], a0, a1, a2, a3, b0, b1, magic);
            else mma(acc[j], a0, a1, a2, a3, b0, b1, acc[j]);
          }
          if (sub % kSub == kSub - 1) {
            const int gi = sub / kSub;
            const f32x2 s0 = pair_of(s_lo[gi], s_lo[gi]), s1 = pair_of(s_hi[gi], s_hi[gi]);
#pragma unroll
            for (int j = 0; j < DT; ++j) {
              tot[i][j][0] = fma2(s0, add2(pair_of(__int_as_float(acc[j][0]), __int_as_float(acc[j][1])), less), tot[i][j][0]);
              tot[i][j][1] = fma2(s1, add2(pair_of(__int_as_float(acc[j][2]), __int_as_float(acc[j][3])), less), tot[i][j][1]);
            }
          }
        }
      }
    }

    // the warps' sums meet in shared memory; digits and the team's shares are added on the way out
    float* const own = red + wk * (32 * S::kLine);
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int j = 0; j < DT; ++j)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          float* at = own + (i * 16 + h * 8 + g) * S::kLine + j * 8 + 2 * t;
          unpair(tot[i][j][h], at[0], at[1]);
        }
    if constexpr (MID) {
#pragma unroll
      for (int v = 0; v < S::kVectors; ++v) own[lane * S::kLine + 8 * DT + v] = mid[v];
    }
    auto meet = [&]() {
      __syncwarp();
      if (team > 1) asm volatile("bar.sync %0, %1;" ::"r"(1 + in_block), "r"(team * 32) : "memory");
    };
    meet();
    const int64_t row = (int64_t)tile * 32 + lane;
    for (int q = wk; q < nq; q += team) {
      const int exponent = VSK_CHK(a.info + q0 + q)->exponent;
      float v = 0.f, m = 0.f;
#pragma unroll
      for (int d = 0; d < kDigits; ++d) {   // the small digits first
        float part = 0.f;
        for (int w = 0; w < team; ++w) part += red[(w * 32 + lane) * S::kLine + q * kDigits + d];
        v = fmaf(v, 1.f / 256.f, part);
      }
      if constexpr (MID)
        for (int w = 0; w < team; ++w) m += red[(w * 32 + lane) * S::kLine + 8 * DT + q];
      // (the digits' numbers are 16 times the products, and the last one added counts 256^3)
      v = ldexpf(v, exponent + 8 * (kDigits - 1) - 4) + m;
      if (row < a.n) {
        if (exponent == INT_MIN) v = plain_product(a, a.x, row, q0 + q);
        store_y(a, (q0 + q) * a.y_stride + row, v);
      }
    }
    meet();
  }
}

// One block per vector: its largest element, then digits in the order of the fragments, and its sums over the groups.  Eight columns per
// thread; of vectors of up to 8 192 nothing is read twice.
constexpr int kToDigits = 512, kKept = 2;
template <typename X>
__global__ void __launch_bounds__(kToDigits) q4_to_digits_kernel(const X* __restrict__ x, int64_t x_stride, int wide, int dim, int ksteps,
                                                                 int per_launch, int tiles, int group, uint2* __restrict__ frags,
                                                                 float* __restrict__ sums, int sum_stride, VectorInfo* __restrict__ info) {
  __shared__ float warp_top[kToDigits / 32];
  __shared__ int wrong;
  let_the_next_launch_begin();
  const int64_t q = blockIdx.x;
  const X* src = x + q * x_stride;
  auto to_f32 = [](X e) {
    if constexpr (std::is_same<X, float>::value) return e;
    else if constexpr (std::is_same<X, __half>::value) return __half2float(e);
    else return __bfloat162float(e);
  };
  auto load = [&](int col, float (&v)[8]) {
    if (wide && col + 8 <= dim) {
      constexpr int kVec = 16 / sizeof(X);
#pragma unroll
      for (int j = 0; j < 8; j += kVec) {
        const uint4 u = __ldg(reinterpret_cast<const uint4*>(src + col + j));
        const X* h = reinterpret_cast<const X*>(&u);
#pragma unroll
        for (int e = 0; e < kVec; ++e) v[j + e] = to_f32(h[e]);
      }
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] = col + j < dim ? to_f32(*VSK_CHK(src + col + j)) : 0.f;
    }
  };
  if (threadIdx.x == 0) wrong = 0;
  __syncthreads();
  float top = 0.f;
  bool bad = false;
  float kept[kKept][8];
  auto look = [&](const float (&v)[8]) {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      bad |= !isfinite(v[j]);
      top = fmaxf(top, fabsf(v[j]));
    }
  };
#pragma unroll
  for (int i = 0; i < kKept; ++i) {
    load((i * kToDigits + (int)threadIdx.x) * 8, kept[i]);
    look(kept[i]);
  }
  for (int col = (kKept * kToDigits + (int)threadIdx.x) * 8; col < dim; col += kToDigits * 8) {
    float v[8];
    load(col, v);
    look(v);
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
  if (bad) wrong = 1;
  if ((threadIdx.x & 31) == 0) warp_top[threadIdx.x >> 5] = top;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kToDigits / 32; ++w) top = fmaxf(top, warp_top[w]);
  const bool finite = wrong == 0;
  // the largest power of two that keeps |top| within 127 256^3 + 127 256^2 + 127 256 + 127
  int shift = 0;
  if (finite && top > 0.f) {
    shift = 30 - ilogbf(top);      // top 2^shift in [2^30, 2^31)
    if (ldexpf(top, shift) > 2139062016.f) --shift;
  }
  if (threadIdx.x == 0) info[q] = VectorInfo{finite ? -shift : INT_MIN};
  // a power of two beyond fp32's range is taken in two steps
  const float up0 = ldexpf(1.f, max(-126, min(127, shift))), up1 = ldexpf(1.f, shift - max(-126, min(127, shift)));
  const int64_t chunk = q / per_launch;
  const int first_col = (int)(q % per_launch) * kDigits;
  auto put = [&](int p, const float (&v)[8]) {   // (whole warps together, for the sums)
    const int col = p * 8;
    const bool inside = p < ksteps * 16;
    uint32_t even[kDigits] = {}, odd[kDigits] = {};
    float s = 0.f;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      s += v[j];
      int n = __float2int_rn(v[j] * up0 * up1);
#pragma unroll
      for (int d = 0; d < kDigits; ++d) {
        const int low = (int)(int8_t)(n & 0xff);
        n = (n - low) >> 8;
        if (j & 1) odd[d] |= (uint32_t)(low & 0xff) << (8 * (j >> 1));
        else even[d] |= (uint32_t)(low & 0xff) << (8 * (j >> 1));
      }
    }
    // which of the lane's four words of a step these eight columns meet, and in which lane (q4_digits_kernel)
    const int k = p >> 4, sub = group == 32 ? (p >> 2) & 3 : group == 64 ? ((p >> 2) & 2) | (p & 1) : p & 3;
    const int t = group == 32 ? p & 3 : group == 64 ? (p >> 1) & 3 : (p >> 2) & 3;
#pragma unroll
    for (int d = 0; d < kDigits; ++d) {
      const int c = first_col + d, lane = (c & 7) * 4 + t;
      // [chunk][kstep][tile][sub / 2][lane][sub & 1]
      const int64_t at = ((((chunk * ksteps + k) * tiles + (c >> 3)) * 2 + (sub >> 1)) * 32 + lane) * 2 + (sub & 1);
      if (inside) *VSK_CHK_W(frags + at) = make_uint2(even[d], odd[d]);
    }
    if (sums) {   // (neighbouring threads hold a group's parts)
      for (int o = group / 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
      if (inside && col % group == 0) *VSK_CHK_W(sums + q * sum_stride + col / group) = s;
    }
  };
#pragma unroll
  for (int i = 0; i < kKept; ++i) {
    if (!finite) {
#pragma unroll
      for (int j = 0; j < 8; ++j) kept[i][j] = 0.f;   // (the product kernel does without)
    }
    if (i * kToDigits < ksteps * 16) put(i * kToDigits + (int)threadIdx.x, kept[i]);
  }
  for (int p0 = kKept * kToDigits; p0 < ksteps * 16; p0 += kToDigits) {
    float v[8];
    load((p0 + (int)threadIdx.x) * 8, v);
    if (!finite) {
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] = 0.f;
    }
    put(p0 + (int)threadIdx.x, v);
  }
}

template <int DT, int GW, bool MID, bool WIDE>
int32_t launch(Ctx* ctx, DigitArgs a) {
  using S = Shape<DT>;
  auto kernel = q4_digits_kernel<DT, GW, MID, WIDE>;
  VSK_CUDA(ctx, opt_in_shared(ctx, kernel, S::kShared));
  const int64_t chunks = ceil_div(a.nq, a.per_launch);
  const int64_t slots = (int64_t)ctx->prop.multiProcessorCount * resident_blocks(ctx, kernel, 32 * kWarps, S::kShared) * kWarps;
  const int64_t tiles = ceil_div(a.n, 32);
  if (tiles > 1 << 30) return fail(ctx, VSK_ERR_INVALID_BUFFER_SIZE, "too many rows in one call");
  a.team = q4_team(tiles, a.ksteps, std::max<int64_t>(1, slots / chunks), kWarps);
  const int64_t blocks = std::min(ceil_div(tiles, kWarps / a.team), std::max<int64_t>(1, slots / kWarps / chunks));
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((unsigned)blocks, (unsigned)chunks);
  cfg.blockDim = dim3(32 * kWarps);
  cfg.dynamicSmemBytes = S::kShared;
  cfg.stream = ctx->stream;
  cudaLaunchAttribute attr{};
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  VSK_CUDA(ctx, cudaLaunchKernelEx(&cfg, kernel, a));
  ctx->stats.kernel_launches++;
  return VSK_OK;
}

template <int DT, int GW>
int32_t by_layout(Ctx* ctx, const DigitArgs& a) {
  if (a.copy == 16) return a.middles ? launch<DT, GW, true, true>(ctx, a) : launch<DT, GW, false, true>(ctx, a);
  return a.middles ? launch<DT, GW, true, false>(ctx, a) : launch<DT, GW, false, false>(ctx, a);
}
template <int DT>
int32_t by_group(Ctx* ctx, const DigitArgs& a) {
  return a.group == 32 ? by_layout<DT, 4>(ctx, a) : a.group == 64 ? by_layout<DT, 2>(ctx, a) : by_layout<DT, 1>(ctx, a);
}

}  // namespace

int32_t q4_product_digits(Ctx* ctx, const vsk_q4_rows& rows, const void* x, int32_t x_dtype, int64_t nq, int64_t x_stride, void* y,
                          int32_t y_dtype, int64_t y_stride) {
  DigitArgs a{};
  a.codes = rows.codes;
  a.code_stride = rows.code_stride;
  a.scales = (const __half*)rows.scales;
  a.middles = (const __half*)rows.middles;
  a.scale_stride = rows.scale_stride;
  a.n = rows.n;
  a.dim = rows.dim;
  a.group = rows.group;
  a.groups = (int)ceil_div(rows.dim, rows.group);
  a.ksteps = (int)ceil_div(rows.dim, 128);
  const uintptr_t code_bits = reinterpret_cast<uintptr_t>(rows.codes) | (uintptr_t)rows.code_stride;
  a.copy = (code_bits & 15) == 0 ? 16 : (code_bits & 3) == 0 ? 4 : 1;
  const int gw = 128 / rows.group;
  const uintptr_t scale_bits = reinterpret_cast<uintptr_t>(rows.scales) | reinterpret_cast<uintptr_t>(rows.middles) | (uintptr_t)(2 * rows.scale_stride);
  a.pair_scales = (scale_bits & (uintptr_t)(2 * gw - 1)) == 0;
  a.x = Vectors{x, x_stride, x_dtype};
  a.nq = nq;
  a.y = y;
  a.y_stride = y_stride;
  a.y_dtype = y_dtype;
  const int tiles = nq <= 2 ? 1 : nq <= 4 ? 2 : 4;
  a.per_launch = 8 * tiles / kDigits;
  const int64_t chunks = ceil_div(nq, a.per_launch);
  if (chunks > 65535) return fail(ctx, VSK_ERR_INVALID_BUFFER_SIZE, "too many vectors");
  const size_t frag_bytes = (size_t)chunks * a.ksteps * tiles * 1024;
  a.sum_stride = a.ksteps * gw;
  const size_t sum_bytes = rows.middles ? (size_t)nq * a.sum_stride * 4 : 0;
  void* p;
  VSK_TRY(scratch(ctx, SLOT_Q16, frag_bytes + sum_bytes + (size_t)nq * sizeof(VectorInfo), &p));
  a.frags = (const uint4*)p;
  float* sums = sum_bytes ? (float*)((uint8_t*)p + frag_bytes) : nullptr;
  VectorInfo* info = (VectorInfo*)((uint8_t*)p + frag_bytes + sum_bytes);
  a.sums = sums;
  a.info = info;
  auto prepare = [&](auto* v) {
    using X = std::remove_const_t<std::remove_pointer_t<decltype(v)>>;
    const int wide = ((reinterpret_cast<uintptr_t>(v) | (uintptr_t)(x_stride * sizeof(X))) & 15) == 0;
    q4_to_digits_kernel<X><<<(unsigned)nq, kToDigits, 0, ctx->stream>>>(v, x_stride, wide, a.dim, a.ksteps, a.per_launch, tiles, a.group, (uint2*)p, sums,
                                                                  a.sum_stride, info);
  };
  if (x_dtype == VSK_DTYPE_F32) prepare((const float*)x);
  else if (x_dtype == VSK_DTYPE_F16) prepare((const __half*)x);
  else prepare((const __nv_bfloat16*)x);
  ctx->stats.kernel_launches++;
  VSK_CUDA(ctx, cudaGetLastError());
  return tiles == 1 ? by_group<1>(ctx, a) : tiles == 2 ? by_group<2>(ctx, a) : by_group<4>(ctx, a);
}

}  // namespace vsk
