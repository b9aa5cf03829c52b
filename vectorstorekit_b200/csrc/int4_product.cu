// Products of tens of vectors with rows held in four bits (int4.cu has the format, int4_digits.cu the form for a few vectors).
//
// Here x stays in its 16 bits and the codes become exact 16-bit numbers, so that the call is bound by the tensor cores' warp form
// (m16n8k16, fp32 sums) rather than by four digits' worth of columns: a code under the exponent of 1024 (fp16) or 128 (bf16) is that power
// plus the code, and taking the power and 8 away needs no rounding.  A group's sum is taken in fp32 registers, multiplied by the
// scale there and added to the row's total: codes are never multiplied by a rounded weight.
//
// More than 16 vectors, with rows that fill the machine at 16-byte places, go to int4_tensor.cu.  131 072 x 2 048, groups of 128, 32 bf16 vectors, here: 104 us,
// where the warp form's rate would allow 31: tensor pipe 33 %, issue slots 32 %, each warp alternating between unpacking and products.  Four tiles
// of rows per warp, 2 - 6 stages, two blocks per SM, sixteen warps in step with x in shared memory were all within 7 %.
//
//   codes   32 rows x 128 columns (2 KB) per step into a ring in shared memory that belongs to ONE warp, by asynchronous 16-byte copies.  A
//           lane's words of a group lie side by side where the group is that wide, and the pieces of a row are turned so that the rows read
//           together fall into different banks
//   x       in the order of the fragments (16 bytes per lane, 32 columns and eight vectors), prepared by a kernel of its own; the product kernel
//           is launched with it and has its first codes under way before it waits for it
//   scales  asked for by the row's lane two steps ahead, handed to the fragments' lanes as fp32 numbers in shared memory; middles likewise,
//           times the vectors' sums over the group
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
  int dim, groups, ksteps, group;   // ksteps: steps of 128 columns
  int copy;                   // bytes of one asynchronous copy of codes: 16 or 4; 1 = plain byte loads
  int pair_scales;            // a step's scales (and middles) of a row can be read at once
  const uint4* frags;         // [chunk][kstep][32 columns][tile of 8 vectors][32 lanes]
  const float* sums;          // [chunk][kstep * groups of it][8 * tiles]: sums of x over the groups
  Vectors x;                  // for those that are not finite
  int64_t nq;
  int per_launch;             // vectors per grid row
  void* y;
  int64_t y_stride;
  int y_dtype;
  int team;                   // warps that share a tile's columns (1, 2, 4 or 8)
};


template <typename T>
__device__ __forceinline__ void mma(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1, const float (&c)[4]) {
  if constexpr (std::is_same<T, __half>::value) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%11,%12,%13};"
                 : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(c[0]), "f"(c[1]), "f"(c[2]), "f"(c[3]));
  } else {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%11,%12,%13};"
                 : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(c[0]), "f"(c[1]), "f"(c[2]), "f"(c[3]));
  }
}

__device__ __forceinline__ void store_y(const ProductArgs& a, int64_t at, float v) {
  if (a.y_dtype == VSK_DTYPE_F32) *VSK_CHK_W((float*)a.y + at) = v;
  else if (a.y_dtype == VSK_DTYPE_F16) *VSK_CHK_W((__half*)a.y + at) = __float2half_rn(v);
  else *VSK_CHK_W((__nv_bfloat16*)a.y + at) = __float2bfloat16_rn(v);
}

// NT tiles of eight vectors; 32 rows per warp step.
template <int NT>
struct Shape {
  static constexpr int kStage = 32 * 64;
  static constexpr int kStages = NT == 4 ? 6 : 4;
  static constexpr int kLine = 8 * NT + 1;                   // floats of a row of the epilogue's buffer
  static constexpr int kScales = 2 * 2 * 32 * 4;             // two steps' scales and middles
  static constexpr size_t kRing = (size_t)kWarps * kStages * kStage;
  static constexpr size_t kShared = kRing + (size_t)kWarps * (kScales + 32 * kLine) * 4;
};

// The place of a row's 16-byte piece in a stage.
template <int GW>
__device__ __forceinline__ int turned(int row, int piece) {
  return GW == 2 ? piece ^ (((row >> 2) & 1) | (row & 2)) : (piece ^ (row >> 1)) & 3;
}

// GW groups per 128 columns.  WIDE: codes by 16-byte copies (addresses and distances of rows are multiples of 16), else by words or bytes.
template <typename T, int NT, int GW, bool MID, bool WIDE>
__global__ void __launch_bounds__(32 * kWarps, NT == 4 ? 1 : 2) q4_product_kernel(const __grid_constant__ ProductArgs a) {
  using S = Shape<NT>;
  extern __shared__ __align__(128) uint8_t smem[];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int g = lane >> 2, t = lane & 3;   // row (and vector) and quarter of the fragments
  const int team = a.team, wk = warp & (team - 1), in_block = warp / team;
  uint8_t* const ring = smem + warp * (S::kStages * S::kStage);
  float* const scales = reinterpret_cast<float*>(smem + S::kRing) + warp * S::kScales;   // [2][scales, middles][32 rows][GW]
  float* const red = reinterpret_cast<float*>(smem + S::kRing) + kWarps * S::kScales + in_block * team * 32 * S::kLine;

  const int64_t q0 = (int64_t)blockIdx.y * a.per_launch;
  const int nq = (int)min((int64_t)a.per_launch, a.nq - q0);

  const int tiles = (int)((a.n + 31) / 32);   // (the host keeps their number and one more stride below 2^31)
  const int stride = gridDim.x * (kWarps / team);
  const int tile0 = blockIdx.x * (kWarps / team) + in_block;
  const int k0 = a.ksteps * wk / team, k1 = a.ksteps * (wk + 1) / team;
  const int row_bytes = (a.dim + 1) / 2;

  // the codes of one step after the other: this lane's rows (eight apart) and its place in them.  Rows behind the last one repeat it; bytes
  // behind a row's end are zeros, and so are the vectors' columns there.
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
  auto put = [&](const __half* h, float* at) {
    if constexpr (GW == 4) *reinterpret_cast<float4*>(at) = make_float4(__half2float(h[0]), __half2float(h[1]), __half2float(h[2]), __half2float(h[3]));
    else if constexpr (GW == 2) *reinterpret_cast<float2*>(at) = make_float2(__half2float(h[0]), __half2float(h[1]));
    else *at = __half2float(h[0]);
  };
  auto put_scales = [&](const Held& h, int buffer) {
    put(h.s, scales + (buffer * 64 + lane) * GW);
    if constexpr (MID) put(h.m, scales + (buffer * 64 + 32 + lane) * GW);
  };
  Held next, after;
  read_scales(next);
  put_scales(next, 0);
  read_scales(next);
  int buffer = 0;
  wait_for_launches_before();   // x

  const uint4* const frags = a.frags + ((int64_t)blockIdx.y * a.ksteps + k0) * (NT * 128) + lane;
  const float* const sums = MID ? a.sums + ((int64_t)blockIdx.y * a.ksteps + k0) * (GW * 8 * NT) + 2 * t : nullptr;
  int slot = 0;
  for (int tile = tile0; tile < tiles; tile += stride) {
    float tot[2][NT][4];   // vectors 8 j + 2 t and the next of rows 16 i + g and 8 more
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int j = 0; j < NT; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) tot[i][j][e] = 0.f;
    const uint4* step = frags;
    const float* sum = sums;
#pragma unroll 1
    for (int k = k0; k < k1; ++k) {
      read_scales(after);

      copy_wait<S::kStages - 2>();
      __syncwarp();   // everybody's copies and scales of this step are there, and everybody is done with what is filled next
      fetch();
      put_scales(next, buffer ^ 1);
      next = after;

      const uint8_t* stage = ring + slot * S::kStage + g * 64;
      slot = slot + 1 == S::kStages ? 0 : slot + 1;
      const float* of_row = scales + (buffer * 64 + g) * GW;
      buffer ^= 1;
      float acc[2][NT][4];
      const float zero[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int sub = 0; sub < 4; ++sub) {
        constexpr int kSub = 4 / GW;
        uint4 x[NT];
#pragma unroll
        for (int j = 0; j < NT; ++j) x[j] = *VSK_CHK(step + (sub * NT + j) * 32);
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          // the word of rows 16 i + g and eight more, in the order of the groups
          const int piece = GW == 4 ? sub : GW == 2 ? (sub & 2) + (t >> 1) : t;
          const int in_piece = GW == 4 ? t * 4 : GW == 2 ? (t & 1) * 8 + (sub & 1) * 4 : sub * 4;
          const uint8_t* word = stage + i * 1024 + turned<GW>(g, piece) * 16 + in_piece;
          uint32_t lo[4], hi[4];
          unpack<T>(*reinterpret_cast<const uint32_t*>(word), lo);
          unpack<T>(*reinterpret_cast<const uint32_t*>(word + 512), hi);
#pragma unroll
          for (int j = 0; j < NT; ++j) {
            if (sub % kSub == 0) mma<T>(acc[i][j], lo[0], hi[0], lo[1], hi[1], x[j].x, x[j].y, zero);
            else mma<T>(acc[i][j], lo[0], hi[0], lo[1], hi[1], x[j].x, x[j].y, acc[i][j]);
            mma<T>(acc[i][j], lo[2], hi[2], lo[3], hi[3], x[j].z, x[j].w, acc[i][j]);
          }
        }
        if (sub % kSub == kSub - 1) {
          const int gi = sub / kSub;
          float2 xs[MID ? NT : 1];
          if constexpr (MID) {
#pragma unroll
            for (int j = 0; j < NT; ++j) xs[j] = *VSK_CHK(reinterpret_cast<const float2*>(sum + gi * (8 * NT) + j * 8));
          }
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const float s_lo = of_row[i * (16 * GW) + gi], s_hi = of_row[i * (16 * GW) + 8 * GW + gi];
#pragma unroll
            for (int j = 0; j < NT; ++j) {
              tot[i][j][0] = fmaf(s_lo, acc[i][j][0], tot[i][j][0]);
              tot[i][j][1] = fmaf(s_lo, acc[i][j][1], tot[i][j][1]);
              tot[i][j][2] = fmaf(s_hi, acc[i][j][2], tot[i][j][2]);
              tot[i][j][3] = fmaf(s_hi, acc[i][j][3], tot[i][j][3]);
            }
            if constexpr (MID) {
              const float m_lo = of_row[32 * GW + i * (16 * GW) + gi], m_hi = of_row[32 * GW + i * (16 * GW) + 8 * GW + gi];
#pragma unroll
              for (int j = 0; j < NT; ++j) {
                tot[i][j][0] = fmaf(m_lo, xs[j].x, tot[i][j][0]);
                tot[i][j][1] = fmaf(m_lo, xs[j].y, tot[i][j][1]);
                tot[i][j][2] = fmaf(m_hi, xs[j].x, tot[i][j][2]);
                tot[i][j][3] = fmaf(m_hi, xs[j].y, tot[i][j][3]);
              }
            }
          }
        }
      }
      step += NT * 128;
      if constexpr (MID) sum += GW * 8 * NT;
    }

    // the warps' sums meet in shared memory; the team's shares are added on the way out
    float* const own = red + wk * (32 * S::kLine);
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int j = 0; j < NT; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) own[(i * 16 + (e >> 1) * 8 + g) * S::kLine + j * 8 + 2 * t + (e & 1)] = tot[i][j][e];
    auto meet = [&]() {
      __syncwarp();
      if (team > 1) asm volatile("bar.sync %0, %1;" ::"r"(1 + in_block), "r"(team * 32) : "memory");
    };
    meet();
    const int64_t row = (int64_t)tile * 32 + lane;
    for (int q = wk; q < nq; q += team) {
      float v = 0.f;
      for (int w = 0; w < team; ++w) v += red[(w * 32 + lane) * S::kLine + q];
      if (row < a.n) {
        if (MID && !isfinite(v)) v = plain_product(a, a.x, row, q0 + q);   // (without middles both orders answer alike)
        store_y(a, (q0 + q) * a.y_stride + row, v);
      }
    }
    meet();
  }
}

// x in the order of the fragments, zeros behind dim and behind the last vector, and its sums over the groups.  One thread per eight columns
// of one vector.
template <typename T>
__global__ void __launch_bounds__(128) q4_to_fragments_kernel(const T* __restrict__ x, int64_t x_stride, int64_t nq, int dim, int ksteps, int tiles,
                                                              int group, uint4* __restrict__ frags, float* __restrict__ sums) {
  let_the_next_launch_begin();
  const int64_t q = blockIdx.y;
  const int p = blockIdx.x * 128 + threadIdx.x, col = p * 8;
  __align__(16) T v[8];
  float s = 0.f;
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    v[j] = q < nq && col + j < dim ? *VSK_CHK(x + q * x_stride + col + j) : T(0.f);
    if constexpr (std::is_same<T, __half>::value) s += __half2float(v[j]);
    else s += __bfloat162float(v[j]);
  }
  for (int o = group / 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
  if (p >= ksteps * 16) return;
  // which of the lane's four words of a step these eight columns meet, and in which lane (q4_product_kernel)
  const int k = p >> 4, sub = group == 32 ? (p >> 2) & 3 : group == 64 ? ((p >> 2) & 2) | (p & 1) : p & 3;
  const int t = group == 32 ? p & 3 : group == 64 ? (p >> 1) & 3 : (p >> 2) & 3;
  const int64_t chunk = q / (8 * tiles);
  const int c = (int)(q % (8 * tiles));
  // pairs (j, j + 4), as the codes of a word are taken apart
  __align__(16) T w[8] = {v[0], v[4], v[1], v[5], v[2], v[6], v[3], v[7]};
  *VSK_CHK_W(frags + (((chunk * ksteps + k) * 4 + sub) * tiles + (c >> 3)) * 32 + (c & 7) * 4 + t) = *reinterpret_cast<const uint4*>(w);
  if (sums && col % group == 0) *VSK_CHK_W(sums + (chunk * ksteps * (128 / group) + col / group) * (8 * tiles) + c) = s;
}

template <typename T, int NT, int GW, bool MID, bool WIDE>
int32_t launch(Ctx* ctx, ProductArgs a) {
  using S = Shape<NT>;
  auto kernel = q4_product_kernel<T, NT, GW, MID, WIDE>;
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

template <typename T, int NT, int GW>
int32_t by_layout(Ctx* ctx, const ProductArgs& a) {
  if (a.copy == 16) return a.middles ? launch<T, NT, GW, true, true>(ctx, a) : launch<T, NT, GW, false, true>(ctx, a);
  return a.middles ? launch<T, NT, GW, true, false>(ctx, a) : launch<T, NT, GW, false, false>(ctx, a);
}
template <typename T, int NT>
int32_t by_group(Ctx* ctx, const ProductArgs& a) {
  return a.group == 32 ? by_layout<T, NT, 4>(ctx, a) : a.group == 64 ? by_layout<T, NT, 2>(ctx, a) : by_layout<T, NT, 1>(ctx, a);
}

template <typename T>
int32_t prepare_and_launch(Ctx* ctx, const ProductArgs& a, const T* x, int64_t x_stride, int tiles) {
  const int64_t vectors = ceil_div(a.nq, a.per_launch) * a.per_launch;
  for (int64_t q = 0; q < vectors; q += 65535 / 32 * 32) {
    const int64_t here = std::min<int64_t>(65535 / 32 * 32, vectors - q), chunk = q / a.per_launch;
    q4_to_fragments_kernel<T><<<dim3((unsigned)ceil_div(a.ksteps * 16, 128), (unsigned)here), 128, 0, ctx->stream>>>(
        x + q * x_stride, x_stride, a.nq - q, a.dim, a.ksteps, tiles, a.group, (uint4*)a.frags + chunk * a.ksteps * 4 * tiles * 32,
        a.sums ? (float*)a.sums + chunk * a.ksteps * (128 / a.group) * 8 * tiles : nullptr);
    ctx->stats.kernel_launches++;
    VSK_CUDA(ctx, cudaGetLastError());
  }
  return tiles == 2 ? by_group<T, 2>(ctx, a) : by_group<T, 4>(ctx, a);
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
  const int tiles = nq <= 16 ? 2 : 4;
  a.per_launch = 8 * tiles;
  const int64_t chunks = ceil_div(nq, a.per_launch);
  if (chunks > 65535) return fail(ctx, VSK_ERR_INVALID_BUFFER_SIZE, "too many vectors");
  const size_t frag_bytes = (size_t)chunks * a.ksteps * tiles * 2048, sum_bytes = rows.middles ? (size_t)chunks * a.ksteps * gw * 32 * tiles : 0;
  void* p;
  VSK_TRY(scratch(ctx, SLOT_Q16, frag_bytes + sum_bytes, &p));
  a.frags = (const uint4*)p;
  a.sums = sum_bytes ? (const float*)((uint8_t*)p + frag_bytes) : nullptr;
  return x_dtype == VSK_DTYPE_F16 ? prepare_and_launch(ctx, a, (const __half*)x, x_stride, tiles)
                                  : prepare_and_launch(ctx, a, (const __nv_bfloat16*)x, x_stride, tiles);
}

}  // namespace vsk
