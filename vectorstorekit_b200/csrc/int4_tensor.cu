// Products of tens of 16-bit vectors with many rows held in four bits, on tcgen05 (int4_product.cu has the warp form and its reasons).
//
// A wait that runs out ends the block's part with what it has: the call returns VSK_ERR_TIMEOUT.
//
// A block takes 128 rows (the matrix instruction's M) and NV = 32 vectors (its N).  Per step of 64 columns
//   codes     32 bytes per row, copied to a warp's part of a ring by two lanes a row, four steps ahead; a thread takes its row's, which become exact
//             16-bit numbers (code - 8) in tensor memory, the instruction's left side.  A word of eight codes is four columns there, in the
//             order 0 4 1 5 2 6 3 7, which the vectors' tile has too
//   vectors   NV rows of 128 bytes, brought into that order and turned by the row (128-byte swizzle) once by a kernel of its own; a step's tile
//             is copied to the ring as it is
//   products  four instructions of 16 columns, sums of one group of columns per accumulator in tensor memory
//   scales    a thread owns a row: it reads the group's sums of its row, multiplies by the scale in fp32 and adds to the row's NV totals, while
//             the next step's products run; middles likewise, times the vectors' sums over the group, which come with the step's copies.
//             Accumulators, operands and barriers are double
// Codes are never multiplied by a rounded weight: every product is exact, sums are fp32.
//
// 131 072 x 2 048, groups of 128, 32 bf16 vectors: the call takes 84 us, 127 with the warp form.  Bound by a step's chain (copies - numbers - tensor
// memory - products - sums: 0.57 us for a block alone, 18 944 x 8 192 in 72.5 us; four blocks to an SM) and by 1 024 tiles on 592 blocks: kernel 61 us, issue
// slots 59 %, tensor pipe 15 %.  Codes to shared memory
// instead of tensor memory: 97 against 93 us, then codes and vectors asked for through registers two and one steps ahead instead of copies: 93 against 84.
#include "int4.cuh"
#include "tc_ptx.cuh"

namespace vsk {
namespace {
using namespace tc;

constexpr int kThreads = 128, NV = 32;
constexpr int kStages = 5;
constexpr int kSumStages = kStages + 1;   // of the vectors' sums, which other threads may still read when the next copies begin
constexpr int kCodes = 4096 + 16;   // of a stage: even rows, 16 bytes, odd rows (so that the rows of a read lie in different banks)
constexpr int kLeft = 32;           // columns of tensor memory that a step's codes take: 64 numbers of 16 bits


struct TensorArgs {
  const uint8_t* codes;
  int64_t code_stride;
  const __half* scales;
  const __half* middles;          // or null
  int64_t scale_stride;
  int64_t n;
  int dim, group;
  int row_bytes, groups, steps;   // steps of 64 columns
  int quads;                      // four scales of a row can be read at once
  const uint4* x;                 // [chunk][step][NV][8 pieces, turned]
  const float* sums;              // [chunk][group][NV]: sums of x over the groups, if there are middles
  Vectors vectors;                // for those that are not finite
  int64_t nq;
  void* y;
  int64_t y_stride;
  int y_dtype;
  int* err;                       // pinned: a wait ran out
};

template <int GROUP>
struct Shape {
  static constexpr int kPer = GROUP == 32 ? 2 : 1;                         // groups that end in a step, at most
  static constexpr int kSums = 2 * NV * kPer;                              // columns of tensor memory, 64 or 128, behind two steps' codes
  static constexpr int kColumns = 2 * kLeft + kSums <= 128 ? 128 : 256;
  static constexpr int kBlocks = 512 / kColumns;                           // per SM
  static constexpr int kTile = NV * 128;
  // so much that no further block would have to wait for tensor memory
  static constexpr int kAsked = kBlocks == 4 ? 47 * 1024 : 78 * 1024;
  static_assert(kStages * (kTile + kCodes) + kSumStages * kPer * NV * 4 + 1024 <= kAsked, "the ring");
};

// 32 columns of this thread's lane; done behind a tcgen05.wait::st.
__device__ __forceinline__ void store_codes(uint32_t at, const uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], "
      "{%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, "
      "%17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, %32};" ::"r"(at),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]),
      "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]), "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]),
      "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]), "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31])
      : "memory");
}

// Sums (+)= left (tensor memory, 128 rows of 16 numbers in eight columns) x right (shared memory): one instruction.
__device__ __forceinline__ void multiply(uint32_t sums, uint32_t left, uint64_t right, uint32_t instruction, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(sums),
      "r"(left), "l"(right), "r"(instruction), "r"(accumulate)
      : "memory");
}

__device__ __forceinline__ void add_pair(float& a, float& b, float by, float x, float y) {
  const float2 r = __ffma2_rn(make_float2(by, by), make_float2(x, y), make_float2(a, b));
  a = r.x;
  b = r.y;
}

// False when the limit of looks has run out.
__device__ __forceinline__ bool wait_for(uint64_t* bar, uint32_t parity) {
  for (uint32_t i = 0; i < WAIT_LIMIT; ++i) {
    if (mbar_try_wait(bar, parity)) return true;
    if (i > 64) __nanosleep(64);
  }
  return false;
}

template <typename T, int GROUP, bool MID>
__global__ void __launch_bounds__(kThreads, (Shape<GROUP>::kBlocks)) q4_tensor_kernel(const __grid_constant__ TensorArgs a) {
  using S = Shape<GROUP>;
  extern __shared__ uint8_t raw[];
  __shared__ uint64_t done[2];
  __shared__ uint32_t tmem_at;
  __shared__ int gave_up;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  uint8_t* const x_at = raw + ((1024 - (smem_u32(raw) & 1023)) & 1023);   // (the swizzle counts from multiples of 1 024)
  if (threadIdx.x == 0) {
    mbar_init(&done[0], 1);
    mbar_init(&done[1], 1);
    gave_up = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 0) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&tmem_at)), "r"(S::kColumns) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  uint8_t* const codes_at = x_at + kStages * S::kTile;
  float* const sums_of = reinterpret_cast<float*>(codes_at + kStages * kCodes);   // [kSumStages][groups of a step][NV]
  const uint32_t tmem = tmem_at, own_lanes = (uint32_t)(warp * 32) << 16, sums_at = tmem + 2 * kLeft;

  const int64_t q0 = (int64_t)blockIdx.y * NV;
  const int nq = (int)min((int64_t)NV, a.nq - q0);
  const int tiles = (int)((a.n + 127) / 128);
  const int mine = (int)blockIdx.x < tiles ? (tiles - 1 - (int)blockIdx.x) / (int)gridDim.x + 1 : 0;
  const int64_t total = (int64_t)mine * a.steps;

  // Codes and vectors of one step after the other: this lane's half of its own row and of its neighbour's, its pieces of the vectors' tile.  Rows
  // behind the last repeat it; bytes behind a row's end are zeros, whose columns of the vectors are zero.
  const int half = lane & 1;
  int f_tile = blockIdx.x, f_step = 0, f_slot = 0, f_sums = 0;
  const uint8_t* f_src[2];
  auto aim = [&]() {
#pragma unroll
    for (int j = 0; j < 2; ++j)
      f_src[j] = a.codes + min((int64_t)f_tile * 128 + (threadIdx.x & ~1) + j, a.n - 1) * a.code_stride + half * 16;
  };
  aim();
  const uint4* const x0 = a.x + (int64_t)blockIdx.y * a.steps * (NV * 8) + threadIdx.x;
  const uint32_t to_codes = smem_u32(codes_at) + threadIdx.x * 16, to_x = smem_u32(x_at) + threadIdx.x * 16;
  auto fetch = [&]() {
    if (f_tile < tiles) {
      const int have = max(0, min(16, a.row_bytes - f_step * 32 - half * 16));
#pragma unroll
      for (int j = 0; j < 2; ++j) {
#ifdef VSK_CHECKED
        const void* src = have == 16 ? (const void*)VSK_CHK((const uint4*)f_src[j]) : have ? (const void*)f_src[j] : a.codes;
#else
        const void* src = f_src[j];   // (of a copy of no bytes nothing is read)
#endif
        copy16(to_codes + f_slot * kCodes + j * (2048 + 16), src, have);
        f_src[j] += 32;
      }
#pragma unroll
      for (int j = 0; j < NV / 16; ++j) copy16(to_x + f_slot * S::kTile + j * (kThreads * 16), VSK_CHK(x0 + (int64_t)f_step * (NV * 8) + j * kThreads), 16);
      if constexpr (MID) {
        const int e = threadIdx.x / (NV / 4), g = GROUP == 32 ? 2 * f_step + e : GROUP == 64 ? f_step : f_step >> 1;
        if (e < S::kPer && g < a.groups)
          copy16(smem_u32(sums_of + f_sums * (S::kPer * NV)) + threadIdx.x * 16,
                 VSK_CHK(reinterpret_cast<const uint4*>(a.sums + ((int64_t)blockIdx.y * a.groups + g) * NV) + threadIdx.x % (NV / 4)), 16);
        f_sums = f_sums + 1 == kSumStages ? 0 : f_sums + 1;
      }
      f_slot = f_slot + 1 == kStages ? 0 : f_slot + 1;
      if (++f_step == a.steps) {
        f_step = 0;
        f_tile += gridDim.x;
        aim();
      }
    }
    copy_commit();   // (an empty group keeps the count of groups in step)
  };

  // the scales (and middles) of this thread's row, four groups at a time, the next four under way
  struct Four {
    uint2 s, m;
    __device__ __forceinline__ static float of(uint2 v, int group) {
      const uint32_t pair = (group & 2) ? v.y : v.x;
      return __half2float(__ushort_as_half((unsigned short)((group & 1) ? pair >> 16 : pair)));
    }
  };
  int s_tile = blockIdx.x, s_group = 0;
  auto four = [&](const __half* at) {
    if (a.quads && s_group + 4 <= a.groups) return *VSK_CHK(reinterpret_cast<const uint2*>(at));
    uint32_t h[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) h[e] = s_group + e < a.groups ? __half_as_ushort(*VSK_CHK(at + e)) : 0;
    return make_uint2(h[0] | h[1] << 16, h[2] | h[3] << 16);
  };
  auto next_four = [&]() {
    Four v{};
    if (s_tile < tiles) {
      const int64_t at = min((int64_t)s_tile * 128 + threadIdx.x, a.n - 1) * a.scale_stride + s_group;
      v.s = four(a.scales + at);
      if constexpr (MID) v.m = four(a.middles + at);
      s_group += 4;
      if (s_group >= a.groups) {
        s_group = 0;
        s_tile += gridDim.x;
      }
    }
    return v;
  };
  Four now{}, next = next_four();

  float tot[NV];
#pragma unroll
  for (int q = 0; q < NV; ++q) tot[q] = 0.f;

  wait_for_launches_before();   // x
#pragma unroll 1
  for (int s = 0; s < kStages - 1; ++s) fetch();

  bool ok = true;
  int group = 0;              // of the row: the next one whose sums are taken
  int sums_now = 0;           // the stage of the step's sums of vectors
  int issued = 0, taken = 0;  // groups so far: their accumulators alternate
  // The sums of the step before `at` steps: waits for its products, and takes the groups that ended with them.
  auto finish = [&](int64_t at, bool ends) {
    if (ok) ok = wait_for(&done[at & 1], (uint32_t)(at >> 1) & 1u);
    __syncwarp();
    tc_fence_after();
    const int sum_slot = sums_now;
    if constexpr (MID) sums_now = sums_now + 1 == kSumStages ? 0 : sums_now + 1;
    if (!ends) return;
    const uint32_t from = sums_at + own_lanes + (taken & 1) * (NV * S::kPer);
#pragma unroll
    for (int e = 0; e < S::kPer; ++e) {
      float v[NV];
      tc_ld32(from + e * NV, v);
      if ((group & 3) == 0) {
        now = next;
        next = next_four();
      }
      if (group < a.groups) {
        const float s = Four::of(now.s, group);
#pragma unroll
        for (int q = 0; q < NV; q += 2) add_pair(tot[q], tot[q + 1], s, v[q], v[q + 1]);
        if constexpr (MID) {
          const float m = Four::of(now.m, group);
          const float4* x = reinterpret_cast<const float4*>(sums_of + sum_slot * (S::kPer * NV) + e * NV);
#pragma unroll
          for (int q = 0; q < NV; q += 4) {
            const float4 xs = x[q / 4];
            add_pair(tot[q], tot[q + 1], m, xs.x, xs.y);
            add_pair(tot[q + 2], tot[q + 3], m, xs.z, xs.w);
          }
        }
        ++group;
      }
    }
    ++taken;
  };
  // whether a step is its group's (or groups') last
  auto ends_group = [&](int step) { return GROUP != 128 || (step & 1) || step == a.steps - 1; };

  constexpr uint32_t kType = std::is_same<T, __half>::value ? 0u : 1u;
  constexpr uint32_t kInstruction = (1u << 4) | (kType << 7) | (kType << 10) | ((uint32_t)(NV >> 3) << 17) | ((uint32_t)(128 >> 4) << 24);
  int step = 0;
  int64_t tile = blockIdx.x;
  int slot = 0;
#pragma unroll 1
  for (int64_t at = 0; at < total; ++at) {
    const int b = (int)(at & 1);
    copy_wait<kStages - 2>();
    __syncwarp();
    {
      const uint4* own = reinterpret_cast<const uint4*>(codes_at + slot * kCodes + (lane & 1) * (2048 + 16) + (threadIdx.x & ~1) * 16);
      uint32_t p[32];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const uint4 v = own[h];
        const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          uint32_t four[4];
          unpack<T>(w[i], four);
#pragma unroll
          for (int e = 0; e < 4; ++e) p[h * 16 + i * 4 + e] = four[e];
        }
      }
      store_codes(tmem + own_lanes + b * kLeft, p);
    }
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
    tc_fence_before();
    __syncthreads();
    if (warp == 0) {
      tc_fence_after();
      if (elect_one() && ok) {
        const uint32_t lo_b = desc_lo(smem_u32(x_at + slot * S::kTile)), to = sums_at + (issued & 1) * (NV * S::kPer);
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const uint32_t more = GROUP == 128 ? (uint32_t)(k > 0 || (step & 1)) : GROUP == 64 ? (uint32_t)(k > 0) : (uint32_t)(k & 1);
          multiply(GROUP == 32 ? to + (k >> 1) * NV : to, tmem + b * kLeft + k * 8, desc_pack(lo_b + k * 2, kDescHi), kInstruction, more);
        }
        tc_commit(&done[b]);
      }
      __syncwarp();
    }
    if (step > 0) finish(at - 1, ends_group(step - 1));
    fetch();   // into the stage of the step before, whose products are done
    slot = slot + 1 == kStages ? 0 : slot + 1;
    if (ends_group(step)) ++issued;
    if (++step < a.steps) continue;
    // the tile's end: the last step's sums, and the results
    finish(at, true);
    const int64_t row = tile * 128 + threadIdx.x;
    if (row < a.n) {
      auto put = [&](auto* y, auto&& rounded) {
        auto* p = y + q0 * a.y_stride + row;
#pragma unroll
        for (int q = 0; q < NV; ++q) {
          if (q < nq) *VSK_CHK_W(p) = rounded(tot[q]);
          p += a.y_stride;
        }
      };
      if (a.y_dtype == VSK_DTYPE_F32) put((float*)a.y, [](float v) { return v; });
      else if (a.y_dtype == VSK_DTYPE_F16) put((__half*)a.y, [](float v) { return __float2half_rn(v); });
      else put((__nv_bfloat16*)a.y, [](float v) { return __float2bfloat16_rn(v); });
      if constexpr (MID) {   // (without middles both orders answer alike)
        uint32_t wrong = 0;
#pragma unroll
        for (int q = 0; q < NV; ++q) wrong |= (q < nq && !isfinite(tot[q])) ? 1u << q : 0u;
        for (; wrong; wrong &= wrong - 1) {
          const int q = __ffs(wrong) - 1;
          const float v = plain_product(a, a.vectors, row, q0 + q);
          const int64_t at_y = (q0 + q) * a.y_stride + row;
          if (a.y_dtype == VSK_DTYPE_F32) *VSK_CHK_W((float*)a.y + at_y) = v;
          else if (a.y_dtype == VSK_DTYPE_F16) *VSK_CHK_W((__half*)a.y + at_y) = __float2half_rn(v);
          else *VSK_CHK_W((__nv_bfloat16*)a.y + at_y) = __float2bfloat16_rn(v);
        }
      }
    }
#pragma unroll
    for (int q = 0; q < NV; ++q) tot[q] = 0.f;
    // (four scales are taken when a row's groups begin anew)
    group = 0;
    step = 0;
    tile += gridDim.x;
  }
  if (!ok) {
    gave_up = 1;
    wait_for(&done[(total - 1) & 1], (uint32_t)((total - 1) >> 1) & 1u);   // what is still under way, with the same limit
  }
  tc_fence_before();
  __syncthreads();
  if (threadIdx.x == 0 && gave_up) *reinterpret_cast<volatile int*>(a.err) = 1;
  if (warp == 0) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(S::kColumns) : "memory");
  }
}

// x as the steps' tiles, zeros behind dim and behind the last vector, and its sums over the groups: a thread per eight columns of one vector.
template <typename T>
__global__ void __launch_bounds__(128) q4_to_tiles_kernel(const T* __restrict__ x, int64_t x_stride, int64_t nq, int64_t q_first, int dim, int steps,
                                                          int group, int groups, uint4* __restrict__ out, float* __restrict__ sums) {
  let_the_next_launch_begin();
  const int64_t q = q_first + blockIdx.y;
  const int p = blockIdx.x * 128 + threadIdx.x, col = p * 8;
  __align__(16) T v[8];
  float s = 0.f;
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    v[j] = q < nq && col + j < dim ? *VSK_CHK(x + q * x_stride + col + j) : T(0.f);
    s += (float)v[j];
  }
  for (int o = group / 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
  const int64_t chunk = q / NV;
  const int c = (int)(q % NV);
  if (sums && col % group == 0 && col < dim) *VSK_CHK_W(sums + (chunk * groups + col / group) * NV + c) = s;
  if (p >= steps * 8) return;
  __align__(16) T w[8] = {v[0], v[4], v[1], v[5], v[2], v[6], v[3], v[7]};   // as the codes of a word are taken apart
  *VSK_CHK_W(out + ((chunk * steps + (p >> 3)) * NV + c) * 8 + ((p & 7) ^ (c & 7))) = *reinterpret_cast<const uint4*>(w);
}

template <typename T, int GROUP, bool MID>
int32_t launch(Ctx* ctx, const TensorArgs& a) {
  using S = Shape<GROUP>;
  auto kernel = q4_tensor_kernel<T, GROUP, MID>;
  VSK_CUDA(ctx, opt_in_shared(ctx, kernel, S::kAsked));
  const int64_t chunks = ceil_div(a.nq, NV), tiles = ceil_div(a.n, 128);
  const int64_t blocks = std::min(tiles, std::max<int64_t>(1, (int64_t)ctx->prop.multiProcessorCount * S::kBlocks / chunks));
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((unsigned)blocks, (unsigned)chunks);
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = S::kAsked;
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

template <typename T, int GROUP>
int32_t by_middles(Ctx* ctx, const TensorArgs& a) {
  return a.middles ? launch<T, GROUP, true>(ctx, a) : launch<T, GROUP, false>(ctx, a);
}
template <typename T>
int32_t prepare_and_launch(Ctx* ctx, const TensorArgs& a, const T* x, int64_t x_stride, int dim, int group) {
  const int64_t vectors = ceil_div(a.nq, NV) * NV;
  for (int64_t q = 0; q < vectors; q += 65535) {
    q4_to_tiles_kernel<T><<<dim3((unsigned)ceil_div(a.steps * 8, 128), (unsigned)std::min<int64_t>(65535, vectors - q)), 128, 0, ctx->stream>>>(
        x, x_stride, a.nq, q, dim, a.steps, group, a.groups, (uint4*)a.x, (float*)a.sums);
    ctx->stats.kernel_launches++;
    VSK_CUDA(ctx, cudaGetLastError());
  }
  return group == 32 ? by_middles<T, 32>(ctx, a) : group == 64 ? by_middles<T, 64>(ctx, a) : by_middles<T, 128>(ctx, a);
}

}  // namespace

// More than 16 vectors, and a tile of 128 rows and 32 vectors for every SM: warp form / this one, us, symmetric: 19 000 x 4 096, 32 vectors 56 / 57;
// 28 000 63 / 60; 152 000 229 / 161; 10 000 x 1 024, 64 vectors 35 / 28; 4 000 x 512, 200 vectors 29 / 24; fewer: 10 000 x 4 096, 32 vectors
// 44 / 56.  Middles: 152 000 x 2 048, groups of 128, 32 vectors 158 / 102; 152 000 x 148, groups of 32: 75 / 43.  Groups of 32 have two blocks to an SM
// (accumulators of both of a step's groups, double): 152 000 x 4 096, 17 vectors 240 / 246.  Up to 16 vectors the warp form does half the work and this one the same: 152 000 x 4 096, 16 vectors, groups of 32: 154 / 177.
bool q4_fits_tensor(Ctx* ctx, const vsk_q4_rows& rows, int64_t nq) {
  const uintptr_t code_bits = reinterpret_cast<uintptr_t>(rows.codes) | (uintptr_t)rows.code_stride;
  const int64_t tiles = ceil_div(rows.n, 128), chunks = ceil_div(nq, NV);
  return nq > 16 && (code_bits & 15) == 0 && tiles < (1 << 30) && chunks <= 65535 && tiles * chunks >= ctx->prop.multiProcessorCount;
}

int32_t q4_product_tensor(Ctx* ctx, const vsk_q4_rows& rows, const void* x, int32_t x_dtype, int64_t nq, int64_t x_stride, void* y,
                          int32_t y_dtype, int64_t y_stride) {
  TensorArgs a{};
  a.codes = rows.codes;
  a.code_stride = rows.code_stride;
  a.scales = (const __half*)rows.scales;
  a.scale_stride = rows.scale_stride;
  a.n = rows.n;
  a.dim = rows.dim;
  a.group = rows.group;
  a.row_bytes = (rows.dim + 1) / 2;
  a.groups = (int)ceil_div(rows.dim, rows.group);
  a.steps = (int)ceil_div(rows.dim, 64);
  a.middles = (const __half*)rows.middles;
  a.quads = ((reinterpret_cast<uintptr_t>(rows.scales) | reinterpret_cast<uintptr_t>(rows.middles) | (uintptr_t)(2 * rows.scale_stride)) & 7) == 0;
  a.vectors = Vectors{x, x_stride, x_dtype};
  a.nq = nq;
  a.y = y;
  a.y_stride = y_stride;
  a.y_dtype = y_dtype;
  const int64_t vectors = ceil_div(nq, NV) * NV;
  const size_t tile_bytes = (size_t)vectors * a.steps * 128, sum_bytes = rows.middles ? (size_t)vectors * a.groups * 4 : 0;
  void* p;
  VSK_TRY(scratch(ctx, SLOT_Q16, tile_bytes + sum_bytes, &p));
  a.x = (const uint4*)p;
  a.sums = sum_bytes ? (const float*)((uint8_t*)p + tile_bytes) : nullptr;
  VSK_TRY(pinned_reserve(ctx, &ctx->host_flags[0], sizeof(int)));
  volatile int* gave_up = (volatile int*)ctx->host_flags[0].p;
  *gave_up = 0;
  a.err = (int*)ctx->host_flags[0].p;
  VSK_TRY(x_dtype == VSK_DTYPE_F16 ? prepare_and_launch(ctx, a, (const __half*)x, x_stride, rows.dim, rows.group)
                                   : prepare_and_launch(ctx, a, (const __nv_bfloat16*)x, x_stride, rows.dim, rows.group));
  tl_mark(ctx, "q4_product");
  VSK_CUDA(ctx, cudaStreamSynchronize(ctx->stream));
  if (*gave_up) return fail(ctx, VSK_ERR_TIMEOUT, "products with rows in four bits: a bounded wait ran out");
  return VSK_OK;
}

}  // namespace vsk
