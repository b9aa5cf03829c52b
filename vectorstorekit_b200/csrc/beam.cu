// A beam search's step: the k best (beam, token) continuations of every batch entry, and the beams' states moved after their parents.
//
// Selection.  Candidate (j, v) of a live beam j has the total  score_j + (l_jv - lse_j)  (lse_j = log of the sum of exp of row j), or
// score_j + l_jv without normalisation, in 64 bits; the k largest are wanted, equal totals by the lowest (j, v).  The logits are
// read once: a warp takes a piece of 1 024 of them and leaves its maximum and its sum of exponentials (a second look at registers
// instead of running maxima).  The k best candidates lie in the k pieces with the best maxima, since a piece outside those has k
// better maxima before every one of its candidates: one block per batch entry finds a bound that at least k pieces reach and reads
// those pieces again, from L2, for the candidates that reach it too.  Few candidates are staged in shared memory instead and need
// no pieces.
#include <cuda_bf16.h>
#include <math_constants.h>

#include <algorithm>
#include <new>
#include <vector>

#include "common.cuh"
#include "strided.cuh"

namespace vsk {
namespace {

constexpr int kPiece = 1024;
constexpr int kMaxBeams = 64;
constexpr int kMaxBeamK = 128;
constexpr int kListed = 1024;     // candidates that a selection can order at once
constexpr int kChosen = 512;      // pieces that it reads again
// Candidates of a batch entry that are staged in shared memory.  1 000 entries of 4 x 400: 49 us staged, 69 in pieces; 100 of 4 x 500: 46
// and 42; 500 of 8 x 1 000: 76 and 60 (the calls, normalised fp32).
constexpr int kSmall = 2048;

struct BeamArgs {
  const void* logits;
  int64_t batch, batch_stride, beam_stride, vocab;
  int64_t first_batch;            // of a launch of beam_pieces_kernel
  int beams, k, normalize;
  const float* scores;            // [batch][beams]
  const uint8_t* finished;        // [batch][beams] or null
  int64_t end_token;
  float2* stats;                  // [batch * beams][pieces]: maximum, sum of exp(x - maximum)
  float* parts;                   // [batch * beams][pieces][parts of one]: maxima of what one load of a warp brings, or null
  int pieces, per_warp;
  float* out_scores;
  int64_t* out_beams;
  int64_t* out_tokens;
};

__device__ __forceinline__ void wait_for_launches_before() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
__device__ __forceinline__ void let_the_next_launch_begin() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }

template <typename T> __device__ __forceinline__ float as_float(T v);
template <> __device__ __forceinline__ float as_float<float>(float v) { return v; }
template <> __device__ __forceinline__ float as_float<__half>(__half v) { return __half2float(v); }
template <> __device__ __forceinline__ float as_float<__nv_bfloat16>(__nv_bfloat16 v) { return __bfloat162float(v); }

// (x - from) first: it is exact near the maximum, however large the logits are.
__device__ __forceinline__ float exp_of(float x, float from) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"((x - from) * 1.4426950408889634f));
  return r;
}
__device__ __forceinline__ float reference_of(float top) { return top == -CUDART_INF_F ? 0.f : top; }

__device__ __forceinline__ float warp_max(float x) { return ordered_to_float(__reduce_max_sync(0xffffffffu, float_to_ordered(x))); }

// ---- pieces -------------------------------------------------------------------------------------------------------------------
template <typename T> __device__ __forceinline__ T lowest();
template <> __device__ __forceinline__ float lowest<float>() { return -CUDART_INF_F; }
template <> __device__ __forceinline__ __half lowest<__half>() { return __ushort_as_half(0xfc00); }
template <> __device__ __forceinline__ __nv_bfloat16 lowest<__nv_bfloat16>() { return __ushort_as_bfloat16(0xff80); }

// Sixteen bytes of a row: elements at .. at + kVec - 1, -inf behind its end.  ALIGNED: the row begins at a 16-byte boundary.  Others are read as words
// of four bytes; with 16-bit elements five of them, of which the first and the last count half where the row begins in the middle of a word.
template <typename T, bool ALIGNED>
struct RowVector {
  static constexpr int kVec = 16 / (int)sizeof(T);
  static constexpr bool kHalves = !ALIGNED && sizeof(T) == 2;
  uint4 v;
  uint32_t last;
  // `shift`: bits of the row's first word that are not its own (shift_of)
  __device__ __forceinline__ void load(const T* row, int64_t at, int64_t vocab, int shift) {
    const int before = kHalves ? shift >> 4 : 0;
    if (at >= before && at + kVec + (kHalves ? 2 : 0) <= vocab) {
      if constexpr (ALIGNED) {
        v = __ldg(reinterpret_cast<const uint4*>(row + at));
      } else {
        const uint32_t* const w = reinterpret_cast<const uint32_t*>(row + (at - before));
        v = make_uint4(__ldg(w), __ldg(w + 1), __ldg(w + 2), __ldg(w + 3));
        if constexpr (kHalves) last = __ldg(w + 4);
      }
    } else {
      __align__(16) T h[kVec];
#pragma unroll
      for (int j = 0; j < kVec; ++j) h[j] = at + j < vocab ? *VSK_CHK(row + at + j) : lowest<T>();
      v = *reinterpret_cast<const uint4*>(h);
      if constexpr (kHalves) {   // as if they had been read like that
        last = __funnelshift_l(v.w, 0u, shift);
        v = make_uint4(v.x << shift, __funnelshift_l(v.x, v.y, shift), __funnelshift_l(v.y, v.z, shift), __funnelshift_l(v.z, v.w, shift));
      }
    }
  }
  __device__ __forceinline__ uint4 whole(int shift) const {
    if constexpr (!kHalves) return v;
    else return make_uint4(__funnelshift_r(v.x, v.y, shift), __funnelshift_r(v.y, v.z, shift), __funnelshift_r(v.z, v.w, shift), __funnelshift_r(v.w, last, shift));
  }
};
template <typename T>
__device__ __forceinline__ int shift_of(const T* row) { return (int)(reinterpret_cast<uintptr_t>(row) & 2) * 8; }

// A warp takes a.per_warp pieces of a row one after the other, the next one's loads under way.  Pieces are counted from the row's first logit, and
// which of its logits a lane adds never changes: equal rows have equal sums, bit for bit, at whatever addresses they lie.
// 32 x 8 x 131 072 bf16 logits (67 MB): 20 us, 3.3 TB/s, issue slots 61 % busy: bound by the instructions of a logit (convert, maximum,
// convert, subtract, multiply, power, add).  ALIGNED: all rows begin at 16-byte boundaries.
template <typename T, bool ALIGNED>
__global__ void __launch_bounds__(256) beam_pieces_kernel(const BeamArgs a) {
  constexpr int kVec = 16 / sizeof(T), kLoads = kPiece / (32 * kVec);
  let_the_next_launch_begin();
  const int lane = threadIdx.x & 31;
  int piece = (blockIdx.x * 8 + (threadIdx.x >> 5)) * a.per_warp;
  if (piece >= a.pieces) return;
  const int end = min(piece + a.per_warp, a.pieces);
  const int64_t b = a.first_batch + blockIdx.z, row = b * a.beams + blockIdx.y;
  if (!isfinite(__ldg(a.scores + row)) || (a.finished && __ldg(a.finished + row))) return;   // not looked at again
  const T* base = reinterpret_cast<const T*>(a.logits) + b * a.batch_stride + blockIdx.y * a.beam_stride;
  const int shift = shift_of(base);
  RowVector<T, ALIGNED> next[kLoads];
  auto load = [&](int p) {
    const int64_t first = (int64_t)p * kPiece + lane * kVec;
#pragma unroll
    for (int i = 0; i < kLoads; ++i) next[i].load(base, first + i * 32 * kVec, a.vocab, shift);
  };
  load(piece);
  for (; piece < end; ++piece) {
    uint4 raw[kLoads];
#pragma unroll
    for (int i = 0; i < kLoads; ++i) raw[i] = next[i].whole(shift);
    if (piece + 1 < end) load(piece + 1);
    float own[kLoads], top = -CUDART_INF_F;
#pragma unroll
    for (int i = 0; i < kLoads; ++i) {
      const T* h = reinterpret_cast<const T*>(&raw[i]);
      own[i] = -CUDART_INF_F;
#pragma unroll
      for (int j = 0; j < kVec; ++j) own[i] = fmaxf(own[i], as_float<T>(h[j]));   // (a NaN is passed over)
      top = fmaxf(top, own[i]);
    }
    top = warp_max(top);
    const int64_t item = row * a.pieces + piece;
    if (a.parts) {
#pragma unroll
      for (int i = 0; i < kLoads; ++i) {
        const float m = warp_max(own[i]);
        if (lane == i) *VSK_CHK_W(a.parts + item * kLoads + i) = m;
      }
    }
    float sum = 0.f;
    if (a.normalize) {
      const float from = reference_of(top);   // (+inf stays: its row's sum becomes NaN, and so does a NaN's)
#pragma unroll
      for (int i = 0; i < kLoads; ++i) {
        const T* h = reinterpret_cast<const T*>(&raw[i]);
#pragma unroll
        for (int j = 0; j < kVec; ++j) sum += exp_of(as_float<T>(h[j]), from);
      }
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    }
    if (lane == 0) *VSK_CHK_W(a.stats + item) = make_float2(top, sum);
  }
}

// ---- selection --------------------------------------------------------------------------------------------------------------
struct Key {
  double total;
  int64_t at;
};
__device__ __forceinline__ Key no_key() { return Key{-CUDART_INF, 0x7fffffffffffffffLL}; }
__device__ __forceinline__ bool before(const Key& a, const Key& b) { return a.total > b.total || (a.total == b.total && a.at < b.at); }

// Descending bitonic sort of P = 2^i keys.
__device__ __forceinline__ void sort_keys(Key* s, int P) {
  for (int size = 2; size <= P; size <<= 1)
    for (int stride = size >> 1; stride > 0; stride >>= 1) {
      for (int i = threadIdx.x; i < (P >> 1); i += blockDim.x) {
        const int pos = 2 * i - (i & (stride - 1)), other = pos + stride;
        const Key x = s[pos], y = s[other];
        if (before(y, x) == ((pos & size) == 0)) {
          s[pos] = y;
          s[other] = x;
        }
      }
      __syncthreads();
    }
}

// The k best keys of `items`, in order, into list[0 .. return value) (at most k).  key_of(i) may be asked several times.
// A thread's own best keys are as many as there are threads, so the k-th best of them bounds the k-th best of all from below, and
// only the k threads with better ones hold keys above it: rarely more than a few times k, and if they are more than the list
// takes (as many good keys in one thread's share), the best are taken out one by one.
template <int THREADS, typename F>
__device__ int best_keys(int64_t items, int k, Key* list, int* count, F key_of) {
  Key own = no_key();
  for (int64_t i = threadIdx.x; i < items; i += THREADS) {
    const Key x = key_of(i);
    if (before(x, own)) own = x;
  }
  list[threadIdx.x] = own;
  if (threadIdx.x == 0) *count = 0;
  __syncthreads();
  sort_keys(list, THREADS);
  const Key bound = list[k - 1];   // (no_key() where fewer threads have one)
  __syncthreads();
  for (int64_t i = threadIdx.x; i < items; i += THREADS) {
    const Key x = key_of(i);
    if (x.total > -CUDART_INF && !before(bound, x)) {
      const int slot = atomicAdd(count, 1);
      if (slot < kListed) list[slot] = x;
    }
  }
  __syncthreads();
  const int found = *count;
  __syncthreads();
  if (found <= kListed) {
    int P = 2;
    while (P < found) P <<= 1;
    for (int i = found + threadIdx.x; i < P; i += THREADS) list[i] = no_key();
    __syncthreads();
    sort_keys(list, P);
    return min(found, k);
  }
  // one by one: the best key behind the last one taken
  Key last{CUDART_INF, -1};
  for (int r = 0; r < k; ++r) {
    own = no_key();
    for (int64_t i = threadIdx.x; i < items; i += THREADS) {
      const Key x = key_of(i);
      if (before(last, x) && before(x, own)) own = x;
    }
    Key* room = list + kMaxBeamK;   // (behind the answers)
    room[threadIdx.x] = own;
    __syncthreads();
    for (int o = THREADS / 2; o > 0; o >>= 1) {
      if (threadIdx.x < o && before(room[threadIdx.x + o], room[threadIdx.x])) room[threadIdx.x] = room[threadIdx.x + o];
      __syncthreads();
    }
    last = room[0];
    if (threadIdx.x == 0) list[r] = last;
    __syncthreads();
  }
  return k;
}

// The largest bound that at least k threads' keys reach, or nearly the largest (at most half as many again do, if the keys differ enough);
// 1 where fewer than k threads have one.  Keys are the order of fp32 numbers, 0: none.
template <int THREADS>
__device__ unsigned bound_of(unsigned own, int k, unsigned* shared) {
  if (threadIdx.x == 0) {
    shared[0] = 0xffffffffu;
    shared[1] = 0u;
  }
  const int real = __syncthreads_count(own != 0u);
  if (real <= k) return 1u;
  const unsigned low = __reduce_min_sync(0xffffffffu, own ? own : 0xffffffffu), high = __reduce_max_sync(0xffffffffu, own);
  if ((threadIdx.x & 31) == 0) {
    atomicMin(&shared[0], low);
    atomicMax(&shared[1], high);
  }
  __syncthreads();
  unsigned lo = shared[0], hi = shared[1];   // at least k reach lo; hi may be too much
  while (lo < hi) {
    const unsigned mid = lo + (hi - lo + 1) / 2;
    const int reach = __syncthreads_count(own >= mid);
    if (reach >= k) {
      lo = mid;
      if (reach <= k + k / 2) break;
    } else {
      hi = mid - 1;
    }
  }
  return lo;
}

// One block per batch entry.  SMALL: the candidates are staged in shared memory; otherwise their pieces are ranked first.  A chain of short
// dependent steps, bound by their latency: 12 us for one entry of 4 x 32 768, 19 for 32 of 8 x 131 072, 15 for 1 000 of 8 x 100 (SMALL).
template <typename T, int THREADS, bool SMALL>
__global__ void __launch_bounds__(THREADS) beam_choose_kernel(const BeamArgs a) {
  __shared__ Key list[kListed];
  __shared__ double lse[kMaxBeams], score[kMaxBeams];
  __shared__ uint8_t kind[kMaxBeams];           // 0: offers nothing, 1: its tokens, 2: finished
  __shared__ int64_t chosen[kMaxBeamK];
  __shared__ int piece_list[SMALL ? 1 : kChosen];
  __shared__ int count, taken_pieces;
  __shared__ unsigned range[2];
  extern __shared__ float staged[];             // SMALL: [beams][vocab]
  static_assert(kMaxBeamK + THREADS <= kListed, "best_keys keeps the answers and the threads' keys side by side");
  static_assert(THREADS >= kMaxBeamK, "the k-th best of the threads' keys");
  const int64_t b = blockIdx.x;
  const T* base = reinterpret_cast<const T*>(a.logits) + b * a.batch_stride;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const unsigned width = (unsigned)a.vocab;

  if constexpr (!SMALL) wait_for_launches_before();   // the pieces
  if constexpr (SMALL) {
    for (int j = 0; j < a.beams; ++j)
      for (unsigned v = threadIdx.x; v < width; v += THREADS) staged[j * width + v] = as_float<T>(*VSK_CHK(base + j * a.beam_stride + v));
    __syncthreads();
  }
  for (int j = warp; j < a.beams; j += THREADS / 32) {
    const int64_t row = b * a.beams + j;
    const float s = __ldg(a.scores + row);
    int what = !isfinite(s) ? 0 : (a.finished && __ldg(a.finished + row)) ? 2 : 1;
    double total = 0.0;
    if (what == 1 && a.normalize) {
      float top = -CUDART_INF_F;
      double sum = 0.0;
      if constexpr (SMALL) {
        for (unsigned v = lane; v < width; v += 32) top = fmaxf(top, staged[j * width + v]);
        top = warp_max(top);
        const float from = reference_of(top);
        float part = 0.f;
        for (unsigned v = lane; v < width; v += 32) part += exp_of(staged[j * width + v], from);
        sum = part;
      } else {
        const float2* stats = a.stats + row * a.pieces;
        float2 held[4];   // the first 128 pieces' are read once
#pragma unroll
        for (int i = 0; i < 4; ++i) held[i] = lane + 32 * i < a.pieces ? *VSK_CHK(stats + lane + 32 * i) : make_float2(-CUDART_INF_F, 0.f);
#pragma unroll
        for (int i = 0; i < 4; ++i) top = fmaxf(top, held[i].x);
        for (int p = lane + 128; p < a.pieces; p += 32) top = fmaxf(top, VSK_CHK(stats + p)->x);
        top = warp_max(top);
        const float from = reference_of(top);
        // (a piece of nothing but -inf and NaN: its sum is 0 or NaN)
        auto share = [&](const float2& v) { sum += v.x == -CUDART_INF_F ? (double)v.y : (double)v.y * (double)exp_of(v.x, from); };
#pragma unroll
        for (int i = 0; i < 4; ++i) share(held[i]);
        for (int p = lane + 128; p < a.pieces; p += 32) share(*VSK_CHK(stats + p));
      }
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
      if (!(sum > 0.0) || !isfinite(sum)) what = 0;   // nothing but -inf, or a NaN or +inf among the logits
      else total = (double)top + log(sum);
    }
    if (lane == 0) {
      kind[j] = (uint8_t)what;
      score[j] = (double)s;
      lse[j] = total;
    }
  }
  if (threadIdx.x == 0) count = taken_pieces = 0;
  __syncthreads();

  auto total_of = [&](int j, float x) { return score[j] + ((double)x - lse[j]); };   // (lse is 0 without normalisation)
  // the order of a total as fp32, 0: no candidate.  (Rounding keeps the order, up to equality.)
  auto order_of = [&](int j, float x) -> unsigned { return x > -CUDART_INF_F ? float_to_ordered((float)total_of(j, x) + 0.f) : 0u; };   // (not a NaN either)
  auto token_key = [&](int j, int64_t v, float x) { return x > -CUDART_INF_F ? Key{total_of(j, x), j * a.vocab + v} : no_key(); };
  auto add = [&](const Key& x) {
    const int slot = atomicAdd(&count, 1);
    if (slot < kListed) list[slot] = x;
  };
  const unsigned pieces = (unsigned)a.pieces;
  constexpr int kVec = 16 / sizeof(T), kParts = kPiece / (32 * kVec);
  const unsigned per_piece = !SMALL && a.parts ? kParts : 1;
  // part i of the pieces (all parts, or whole pieces)
  auto part_order = [&](unsigned i) -> unsigned {
    const unsigned at = i / per_piece, j = at / pieces;
    if (kind[j] == 2) return i % (per_piece * pieces) == 0 ? float_to_ordered((float)score[j] + 0.f) : 0u;
    if (kind[j] == 0) return 0u;
    const int64_t of = b * a.beams * pieces;
    return order_of(j, a.parts ? *VSK_CHK(a.parts + of * kParts + i) : VSK_CHK(a.stats + of + i)->x);
  };

  // A bound that at least k candidates reach; those that do.
  bool fits = true;
  if constexpr (SMALL) {
    const unsigned items = (unsigned)a.beams * width;
    auto element = [&](unsigned i) -> unsigned {
      const unsigned j = i / width;
      if (kind[j] == 1) return order_of(j, staged[i]);
      return kind[j] == 2 && i % width == 0 ? float_to_ordered((float)score[j] + 0.f) : 0u;
    };
    unsigned own = 0u;
    for (unsigned i = threadIdx.x; i < items; i += THREADS) own = max(own, element(i));
    const unsigned bound = bound_of<THREADS>(own, a.k, range);
    if (own >= bound)
      for (unsigned i = threadIdx.x; i < items; i += THREADS)
        if (element(i) >= bound) {
          const unsigned j = i / width;
          add(kind[j] == 2 ? Key{score[j], j * a.vocab + a.end_token} : token_key(j, i % width, staged[i]));
        }
  } else {
    const unsigned items = (unsigned)a.beams * pieces * per_piece;
    unsigned own = 0u;
#pragma unroll 4
    for (unsigned i = threadIdx.x; i < items; i += THREADS) own = max(own, part_order(i));
    const unsigned bound = bound_of<THREADS>(own, a.k, range);
    if (own >= bound)
      for (unsigned i = threadIdx.x; i < items; i += THREADS)
        if (items <= THREADS || part_order(i) >= bound) {
          const int slot = atomicAdd(&taken_pieces, 1);
          if (slot < kChosen) piece_list[slot] = (int)i;
        }
    __syncthreads();
    fits = taken_pieces <= kChosen;
    if (fits) {
      // a warp per part: what one of its loads brings, or all loads of a whole piece
      for (int s = warp; s < taken_pieces; s += THREADS / 32) {
        const unsigned i = (unsigned)piece_list[s], at = i / per_piece, j = at / pieces;
        if (kind[j] == 2) {
          if (lane == 0) add(Key{score[j], j * a.vocab + a.end_token});
          continue;
        }
        const T* row = base + j * a.beam_stride;
        const int64_t first = (int64_t)(at % pieces) * kPiece;
        const int l0 = a.parts ? (int)(i % per_piece) : 0, l1 = a.parts ? l0 + 1 : kParts;
        const bool aligned = (reinterpret_cast<uintptr_t>(row) & 15) == 0;
        const int shift = shift_of(row);
#pragma unroll 4
        for (int l = l0; l < l1; ++l) {
          const int64_t v0 = first + (l * 32 + lane) * kVec;
          uint4 u;
          if (aligned && v0 + kVec <= a.vocab) {
            u = __ldg(reinterpret_cast<const uint4*>(row + v0));
          } else {
            RowVector<T, false> r;
            r.load(row, v0, a.vocab, shift);
            u = r.whole(shift);
          }
          const T* h = reinterpret_cast<const T*>(&u);
          float x[kVec];
#pragma unroll
          for (int e = 0; e < kVec; ++e) x[e] = as_float<T>(h[e]);
          float top = x[0];
#pragma unroll
          for (int e = 1; e < kVec; ++e) top = fmaxf(top, x[e]);
          if (top > -CUDART_INF_F && order_of(j, top) >= bound) {
#pragma unroll
            for (int e = 0; e < kVec; ++e)
              if (order_of(j, x[e]) >= bound) add(token_key(j, v0 + e, x[e]));
          }
        }
      }
    }
  }
  __syncthreads();
  const int reach = count;

  auto put = [&](int r, const Key& x) {
    const bool has = x.total > -CUDART_INF;
    *VSK_CHK_W(a.out_scores + b * a.k + r) = has ? (float)x.total : -CUDART_INF_F;
    *VSK_CHK_W(a.out_beams + b * a.k + r) = has ? x.at / a.vocab : -1;
    *VSK_CHK_W(a.out_tokens + b * a.k + r) = has ? x.at % a.vocab : -1;
  };
  if (fits && reach <= kListed) {
    // a candidate's place is the number of those before it
    for (int i = threadIdx.x; i < reach; i += THREADS) {
      const Key x = list[i];
      int place = 0;
      for (int j = 0; j < reach; ++j) place += before(list[j], x);
      if (place < a.k) put(place, x);
    }
    for (int r = reach + threadIdx.x; r < a.k; r += THREADS) put(r, no_key());
    return;
  }

  // Many equal totals, many candidates in few places, or hardly more parts than k (every candidate reaches the bound then: one row of 8 000 with
  // k = 64 takes 90 us with cold caches, four of 32 768 with k = 8 take 46): exact keys throughout.
  int found;
  __syncthreads();
  if constexpr (SMALL) {
    found = best_keys<THREADS>((int64_t)a.beams * width, a.k, list, &count, [&](int64_t i) {
      const int j = (int)((unsigned)i / width);
      const unsigned v = (unsigned)i % width;
      if (kind[j] == 1) return token_key(j, v, staged[i]);
      return kind[j] == 2 && v == 0 ? Key{score[j], j * a.vocab + a.end_token} : no_key();
    });
  } else {
    const int taken = best_keys<THREADS>((int64_t)a.beams * pieces, a.k, list, &count, [&](int64_t i) {
      const int j = (int)((unsigned)i / pieces), p = (int)((unsigned)i % pieces);
      if (kind[j] == 2) return p == 0 ? Key{score[j], i} : no_key();
      if (kind[j] == 0) return no_key();
      const float top = VSK_CHK(a.stats + b * a.beams * pieces + i)->x;
      return top > -CUDART_INF_F ? Key{total_of(j, top), i} : no_key();
    });
    if (threadIdx.x < taken) chosen[threadIdx.x] = list[threadIdx.x].at;
    __syncthreads();
    found = best_keys<THREADS>((int64_t)taken * kPiece, a.k, list, &count, [&](int64_t i) {
      const unsigned at = (unsigned)chosen[i / kPiece];
      const int j = (int)(at / pieces), p = (int)(at % pieces), e = (int)(i % kPiece);
      if (kind[j] == 2) return e == 0 ? Key{score[j], j * a.vocab + a.end_token} : no_key();
      const int64_t v = (int64_t)p * kPiece + e;
      return v < a.vocab ? token_key(j, v, as_float<T>(*VSK_CHK(base + j * a.beam_stride + v))) : no_key();
    });
  }
  for (int r = threadIdx.x; r < a.k; r += THREADS) put(r, r < found ? list[r] : no_key());
}

template <typename T>
int32_t select(Ctx* ctx, BeamArgs a) {
  const int64_t candidates = a.beams * a.vocab;
  if (candidates <= kSmall) {
    // 1 000 entries of 8 x 100 and 4 x 400: 46 and 49 us with four warps to an entry, 60 and 57 with sixteen; 100 of 4 x 500: 46 and 40
    beam_choose_kernel<T, 128, true><<<(unsigned)a.batch, 128, (size_t)candidates * sizeof(float), ctx->stream>>>(a);
    ctx->stats.kernel_launches++;
    VSK_CUDA(ctx, cudaGetLastError());
    return VSK_OK;
  }
  constexpr int kParts = kPiece * (int)sizeof(T) / 512;
  a.pieces = (int)ceil_div(a.vocab, kPiece);
  const int64_t items = a.batch * a.beams * a.pieces;
  // Parts of pieces where whole ones are few against k: the bound then leaves fewer candidates.  Four rows of 50 000, k = 64: 48 us with
  // parts, 180 without (more candidates than a list orders); 64 beams of 65 536, k = 128: 119 and 93.
  const bool parts = (int64_t)a.beams * a.pieces < 16 * (int64_t)a.k;
  void* p;
  VSK_TRY(scratch(ctx, SLOT_BEAM, (size_t)items * (sizeof(float2) + (parts ? kParts * sizeof(float) : 0)), &p));
  a.stats = (float2*)p;
  a.parts = parts ? (float*)(a.stats + items) : nullptr;
  // as many pieces per warp as leave two rounds of warps (32 x 8 x 131 072 fp32: 84 us, one piece each: 87)
  a.per_warp = (int)std::max<int64_t>(1, std::min<int64_t>(8, items / ((int64_t)ctx->prop.multiProcessorCount * 64)));
  const uintptr_t bits = reinterpret_cast<uintptr_t>(a.logits) |
                         (uintptr_t)((int64_t)sizeof(T) * ((a.batch > 1 ? a.batch_stride : 0) | (a.beams > 1 ? a.beam_stride : 0)));
  auto* const pieces_kernel = (bits & 15) == 0 ? beam_pieces_kernel<T, true> : beam_pieces_kernel<T, false>;
  for (int64_t f = 0; f < a.batch; f += 65535) {
    a.first_batch = f;
    pieces_kernel<<<dim3((unsigned)ceil_div(a.pieces, 8 * a.per_warp), (unsigned)a.beams, (unsigned)std::min<int64_t>(65535, a.batch - f)), 256, 0, ctx->stream>>>(a);
    ctx->stats.kernel_launches++;
    VSK_CUDA(ctx, cudaGetLastError());
  }
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((unsigned)a.batch);
  cfg.blockDim = dim3(512);
  cfg.stream = ctx->stream;
  cudaLaunchAttribute attr{};
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  VSK_CUDA(ctx, cudaLaunchKernelEx(&cfg, beam_choose_kernel<T, 512, false>, a));
  ctx->stats.kernel_launches++;
  VSK_CUDA(ctx, cudaGetLastError());
  return VSK_OK;
}

// ---- states ---------------------------------------------------------------------------------------------------------------------
// A thread owns vectors of W bytes, each at one place of all the rows of a batch entry: it loads what every slot takes from its parent and only
// then stores, so rows may change places in place, in any permutation.  Four such places per thread: a block's look at the parents and its
// place in the list of states cost as much as moving 4 KB (27 states of 3 x 8 x 766 x 128 fp32: 160 -> 131 us).  Eight states of
// 64 x 8 x 1 024 x 128 bf16 into a second set: 205 us for 1.15 GB read and written, 5.6 TB/s, 0.86 of a copy's rate.
constexpr int kPlaces = 4;
constexpr int kStatesPerLaunch = 32;
struct StateMove {
  const uint8_t* src;
  uint8_t* dst;
  int64_t src_row, dst_row, src_outer, dst_outer;   // bytes between rows / between the outer parts of a row
  int64_t outer, inner;                             // outer parts, bytes of one
  int64_t step;                                     // bytes of a time step, 0: no time axis
  unsigned first_block, tiles;                      // blocks before this state's, blocks along one part
};
struct StateArgs {
  StateMove move[kStatesPerLaunch];
  int count, beams;
  int64_t batch;
  const int64_t* parents;     // [batch][beams]
  const int64_t* lengths;     // [batch] or null
  int* bad;                   // pinned host memory
};

template <typename V, int SLOTS>
__global__ void __launch_bounds__(256) reorder_kernel(const __grid_constant__ StateArgs a) {
  constexpr int kAtOnce = SLOTS <= 8 ? 2 : 1;   // places under way
  __shared__ int from[kMaxBeams];
  __shared__ int moving, wrong;
  int s = 0;
  while (s + 1 < a.count && blockIdx.x >= a.move[s + 1].first_block) ++s;
  const StateMove& m = a.move[s];
  unsigned at = blockIdx.x - m.first_block;
  const unsigned tile = at % m.tiles;
  at /= m.tiles;
  const int64_t part = at % (unsigned)m.outer, b = at / (unsigned)m.outer;   // (the host keeps their product below 2^31)
  if (threadIdx.x == 0) moving = wrong = 0;
  __syncthreads();
  int64_t live = m.inner;
  if (m.step && a.lengths) {
    const int64_t len = __ldg(a.lengths + b);
    live = len <= 0 ? 0 : len >= m.inner / m.step ? m.inner : len * m.step;
  }
  if (threadIdx.x < a.beams) {
    const int i = threadIdx.x;
    const int64_t p = __ldg(a.parents + b * a.beams + i);
    const bool ok = p >= -1 && p < a.beams, moves = ok && p >= 0 && (p != i || m.src != m.dst);
    from[i] = moves ? (int)p : -1;
    if (!ok) wrong = 1;
    if (moves) moving = 1;
  }
  __syncthreads();
  if (wrong) {   // every block of this batch entry sees it: none of its rows moves
    if (threadIdx.x == 0) *reinterpret_cast<volatile int*>(a.bad) = 1;
    return;
  }
  if (!moving) return;
  const uint8_t* const src = m.src + b * a.beams * m.src_row + part * m.src_outer;
  uint8_t* const dst = m.dst + b * a.beams * m.dst_row + part * m.dst_outer;
  const int64_t first = ((int64_t)tile * (256 * kPlaces) + threadIdx.x) * (int64_t)sizeof(V);
#pragma unroll 1
  for (int place = 0; place < kPlaces; place += kAtOnce) {
    int64_t off[kAtOnce];
#pragma unroll
    for (int u = 0; u < kAtOnce; ++u) off[u] = first + (place + u) * (256 * (int64_t)sizeof(V));
    if (off[0] >= live) return;
    // in place, SLOTS >= beams: everything is loaded before anything is stored
    for (int i0 = 0; i0 < a.beams; i0 += SLOTS) {
      V v[kAtOnce][SLOTS];
#pragma unroll
      for (int u = 0; u < kAtOnce; ++u)
#pragma unroll
        for (int i = 0; i < SLOTS; ++i)
          if (off[u] < live && i0 + i < a.beams && from[i0 + i] >= 0) v[u][i] = *VSK_CHK(reinterpret_cast<const V*>(src + from[i0 + i] * m.src_row + off[u]));
#pragma unroll
      for (int u = 0; u < kAtOnce; ++u)
#pragma unroll
        for (int i = 0; i < SLOTS; ++i)
          if (off[u] < live && i0 + i < a.beams && from[i0 + i] >= 0) *VSK_CHK_W(reinterpret_cast<V*>(dst + (i0 + i) * m.dst_row + off[u])) = v[u][i];
    }
  }
}

// The largest vector that every address and length of a state is a multiple of.
int vector_bytes(const vsk_state& s) {
  const uintptr_t bits = reinterpret_cast<uintptr_t>(s.src) | reinterpret_cast<uintptr_t>(s.dst) | (uintptr_t)s.src_row_stride |
                         (uintptr_t)s.dst_row_stride | (s.outer > 1 ? (uintptr_t)(s.src_outer_stride | s.dst_outer_stride) : 0) |
                         (uintptr_t)s.step_bytes;
  return (bits & 15) == 0 ? 16 : (bits & 7) == 0 ? 8 : (bits & 3) == 0 ? 4 : (bits & 1) == 0 ? 2 : 1;
}

// Blocks of a state that moves vectors of `width` bytes; more than a launch has: -1.
int64_t blocks_of(const vsk_state& s, int width, int64_t batch) {
  const int64_t tiles = ceil_div(s.steps * s.step_bytes, 256 * kPlaces * (int64_t)width);
  if (tiles > 0x7fffffffLL || s.outer > 0x7fffffffLL || batch * s.outer > 0x7fffffffLL / tiles) return -1;
  return batch * s.outer * tiles;
}
int move_width(const vsk_state& s, int beams) {
  const int w = vector_bytes(s);
  return w == 16 && s.src == s.dst && beams > 32 ? 8 : w;   // (sixty-four vectors of 16 bytes do not fit the registers)
}

template <typename V>
int32_t reorder(Ctx* ctx, StateArgs& a, bool in_place, int64_t blocks) {
  if (!in_place || a.beams <= 8) reorder_kernel<V, 8><<<(unsigned)blocks, 256, 0, ctx->stream>>>(a);
  else if (a.beams <= 16) reorder_kernel<V, 16><<<(unsigned)blocks, 256, 0, ctx->stream>>>(a);
  else if (a.beams <= 32) reorder_kernel<V, 32><<<(unsigned)blocks, 256, 0, ctx->stream>>>(a);
  else if constexpr (sizeof(V) <= 8) reorder_kernel<V, 64><<<(unsigned)blocks, 256, 0, ctx->stream>>>(a);   // (wider ones come as two)
  ctx->stats.kernel_launches++;
  VSK_CUDA(ctx, cudaGetLastError());
  return VSK_OK;
}

// No memory is written that another row, part or state is read from or written to: blocks move them in any order.
int32_t check_apart(Ctx* ctx, const vsk_state* states, int32_t count, int64_t rows) {
  struct Range {
    Strided of;
    int32_t state;
    bool written;
  };
  std::vector<Range> ranges;
  ranges.reserve(2 * (size_t)count);
  for (int32_t i = 0; i < count; ++i) {
    const vsk_state& s = states[i];
    const int64_t inner = s.steps * s.step_bytes, src_part = s.outer > 1 ? s.src_outer_stride : 0, dst_part = s.outer > 1 ? s.dst_outer_stride : 0;
    for (const auto& [row, part] : {std::pair{s.src_row_stride, src_part}, std::pair{s.dst_row_stride, dst_part}})
      if ((double)rows * (double)row + (double)s.outer * (double)part > 0x1p60) return fail(ctx, VSK_ERR_INVALID_BUFFER_SIZE, "state %d is too large", i);
    ranges.push_back({{(int64_t)s.dst, rows, s.dst_row_stride, s.outer, dst_part, inner}, i, true});
    if (meets_itself(ranges.back().of)) return fail(ctx, VSK_ERR_INVALID_BUFFER_SIZE, "state %d: rows overlap", i);
    if (s.src != s.dst) ranges.push_back({{(int64_t)s.src, rows, s.src_row_stride, s.outer, src_part, inner}, i, false});
  }
  std::sort(ranges.begin(), ranges.end(), [](const Range& a, const Range& b) { return a.of.at < b.of.at; });
  // Rows side by side in wider ones (a model's caches in one block) lie apart from one another as soon as each begins behind the one before it
  // and the last ends before the first's next row: only what is behind such a run is looked at pair by pair.
  for (size_t first = 0, behind; first < ranges.size(); first = behind) {
    const int64_t row = ranges[first].of.row, next_row = ranges[first].of.at + row;
    for (behind = first + 1; behind < ranges.size(); ++behind) {
      const Strided &a = ranges[behind - 1].of, &b = ranges[behind].of;
      if (b.row != row || b.at < a.at + a.in_row() || b.at + b.in_row() > next_row) break;
    }
    for (size_t i = first; i < behind; ++i) {
      const int64_t end = ranges[i].of.last();
      for (size_t j = behind; j < ranges.size() && ranges[j].of.at < end; ++j)
        if ((ranges[i].written || ranges[j].written) && meet(ranges[i].of, ranges[j].of))
          return fail(ctx, VSK_ERR_INVALID_INPUT, "memory of states %d and %d overlaps", ranges[i].state, ranges[j].state);
    }
  }
  return VSK_OK;
}

int32_t check_ctx(vsk_ctx* c, Ctx** ctx) {
  *ctx = reinterpret_cast<Ctx*>(c);
  if (!*ctx) return VSK_ERR_INVALID_INPUT;
  cudaSetDevice((*ctx)->device);
  return VSK_OK;
}

}  // namespace
}  // namespace vsk

using namespace vsk;

extern "C" {

int32_t vsk_beam_select_dev(vsk_ctx* c, const void* logits, int32_t dtype, int64_t batch, int32_t beams, int64_t vocab, int64_t batch_stride,
                            int64_t beam_stride, const float* scores, const uint8_t* finished, int64_t end_token, int32_t normalize, int32_t k,
                            float* out_scores, int64_t* out_beams, int64_t* out_tokens) {
  VSK_TRACE("vsk_beam_select_dev");
  Ctx* ctx;
  VSK_TRY(check_ctx(c, &ctx));
  if (batch <= 0 || beams <= 0 || vocab <= 0) return fail(ctx, VSK_ERR_EMPTY_INPUT, "no candidates");
  if (beams > kMaxBeams) return fail(ctx, VSK_ERR_INVALID_INPUT, "at most %d beams", kMaxBeams);
  if (k <= 0 || k > kMaxBeamK) return fail(ctx, VSK_ERR_INVALID_INPUT, "k must be in [1, %d]", kMaxBeamK);
  if (vocab > 0x7fffffffLL || batch > 0x7fffffffLL) return fail(ctx, VSK_ERR_INVALID_BUFFER_SIZE, "vocabulary and batch must be below 2^31");
  if (!logits || !scores || !out_scores || !out_beams || !out_tokens) return fail(ctx, VSK_ERR_INVALID_INPUT, "null pointer");
  if (batch_stride < 0 || beam_stride < 0) return fail(ctx, VSK_ERR_INVALID_INPUT, "negative stride");
  if (finished && (end_token < 0 || end_token >= vocab)) return fail(ctx, VSK_ERR_INVALID_INPUT, "the end token must be in [0, %lld)", (long long)vocab);
  if (dtype != VSK_DTYPE_F32 && dtype != VSK_DTYPE_F16 && dtype != VSK_DTYPE_BF16)
    return fail(ctx, VSK_ERR_UNSUPPORTED_OPERATION, "element type %d is not supported", dtype);
  if (reinterpret_cast<uintptr_t>(logits) & (dtype == VSK_DTYPE_F32 ? 3 : 1)) return fail(ctx, VSK_ERR_INVALID_INPUT, "logits are not aligned to their element");
  if (((reinterpret_cast<uintptr_t>(scores) | reinterpret_cast<uintptr_t>(out_scores)) & 3) ||
      ((reinterpret_cast<uintptr_t>(out_beams) | reinterpret_cast<uintptr_t>(out_tokens)) & 7))
    return fail(ctx, VSK_ERR_INVALID_INPUT, "scores, beams or tokens are not aligned to their element");
  drain_stale_error("vsk_beam_select_dev");
  BeamArgs a{};
  a.logits = logits;
  a.batch = batch;
  a.batch_stride = batch_stride;
  a.beam_stride = beam_stride;
  a.vocab = vocab;
  a.beams = beams;
  a.k = k;
  a.normalize = normalize != 0;
  a.scores = scores;
  a.finished = finished;
  a.end_token = end_token;
  a.out_scores = out_scores;
  a.out_beams = out_beams;
  a.out_tokens = out_tokens;
  VSK_TRY(dtype == VSK_DTYPE_F32 ? select<float>(ctx, a) : dtype == VSK_DTYPE_F16 ? select<__half>(ctx, a) : select<__nv_bfloat16>(ctx, a));
  tl_mark(ctx, "beam_select");
  VSK_CUDA(ctx, cudaStreamSynchronize(ctx->stream));
  return VSK_OK;
}

int32_t vsk_reorder_states_dev(vsk_ctx* c, const vsk_state* states, int32_t count, int64_t batch, int32_t beams, const int64_t* parents,
                               const int64_t* lengths) {
  VSK_TRACE("vsk_reorder_states_dev");
  Ctx* ctx;
  VSK_TRY(check_ctx(c, &ctx));
  if (count <= 0 || batch <= 0 || beams <= 0) return fail(ctx, VSK_ERR_EMPTY_INPUT, "no states");
  if (beams > kMaxBeams) return fail(ctx, VSK_ERR_INVALID_INPUT, "at most %d beams", kMaxBeams);
  if (batch > 0x7fffffffLL) return fail(ctx, VSK_ERR_INVALID_BUFFER_SIZE, "batch must be below 2^31");
  if (!states || !parents) return fail(ctx, VSK_ERR_INVALID_INPUT, "null pointer");
  if ((reinterpret_cast<uintptr_t>(parents) | reinterpret_cast<uintptr_t>(lengths)) & 7)
    return fail(ctx, VSK_ERR_INVALID_INPUT, "parents or lengths are not aligned to their element");
  for (int32_t i = 0; i < count; ++i) {
    const vsk_state& s = states[i];
    if (!s.src || !s.dst) return fail(ctx, VSK_ERR_INVALID_INPUT, "state %d: null pointer", i);
    if (s.outer <= 0 || s.steps <= 0 || s.step_bytes <= 0) return fail(ctx, VSK_ERR_EMPTY_INPUT, "state %d is empty", i);
    if (s.steps > (1ll << 48) / s.step_bytes || s.outer > (1ll << 48) / (s.steps * s.step_bytes))
      return fail(ctx, VSK_ERR_INVALID_BUFFER_SIZE, "state %d is too large", i);
    const int64_t inner = s.steps * s.step_bytes;
    if (s.src_row_stride < 0 || s.src_outer_stride < 0 || s.dst_row_stride < inner || (s.outer > 1 && s.dst_outer_stride < inner))
      return fail(ctx, VSK_ERR_INVALID_BUFFER_SIZE, "state %d: rows overlap", i);
    if (s.src == s.dst && (s.src_row_stride != s.dst_row_stride || (s.outer > 1 && s.src_outer_stride != s.dst_outer_stride)))
      return fail(ctx, VSK_ERR_INVALID_INPUT, "state %d: in place, but with other strides", i);
    if (blocks_of(s, move_width(s, beams), batch) < 0) return fail(ctx, VSK_ERR_INVALID_BUFFER_SIZE, "state %d is too large", i);
    const double last = (double)(batch * beams - 1) * s.dst_row_stride + (double)(s.outer - 1) * (s.outer > 1 ? s.dst_outer_stride : 0) + inner;
    auto inside = [&](const int64_t* p, int64_t numbers) {
      const double from = (double)((intptr_t)p - (intptr_t)s.dst);
      return p && from < last && from + 8. * numbers > 0.;
    };
    if (inside(parents, batch * beams) || inside(lengths, batch))
      return fail(ctx, VSK_ERR_INVALID_INPUT, "parents or lengths lie in state %d, which moves", i);
  }
  try {
    VSK_TRY(check_apart(ctx, states, count, batch * beams));
  } catch (const std::bad_alloc&) {
    return fail(ctx, VSK_ERR_OUT_OF_MEMORY, "out of host memory");
  }
  drain_stale_error("vsk_reorder_states_dev");
  VSK_TRY(pinned_reserve(ctx, &ctx->host_flags[0], sizeof(int)));
  volatile int* bad = (volatile int*)ctx->host_flags[0].p;
  *bad = 0;
  // one launch for the states of one vector width that are moved the same way, up to kStatesPerLaunch
  for (int width = 16; width >= 1; width >>= 1)
    for (int in_place = 0; in_place < 2; ++in_place) {
      StateArgs a{};
      a.beams = beams;
      a.batch = batch;
      a.parents = parents;
      a.lengths = lengths;
      a.bad = (int*)ctx->host_flags[0].p;
      int64_t blocks = 0;
      auto launch = [&]() -> int32_t {
        if (a.count == 0) return VSK_OK;
        VSK_TRY(width == 16  ? reorder<uint4>(ctx, a, in_place, blocks)
                : width == 8 ? reorder<uint2>(ctx, a, in_place, blocks)
                : width == 4 ? reorder<uint32_t>(ctx, a, in_place, blocks)
                : width == 2 ? reorder<uint16_t>(ctx, a, in_place, blocks)
                             : reorder<uint8_t>(ctx, a, in_place, blocks));
        a.count = 0;
        blocks = 0;
        return VSK_OK;
      };
      for (int32_t i = 0; i < count; ++i) {
        const vsk_state& s = states[i];
        if (move_width(s, beams) != width || (s.src == s.dst) != (in_place == 1)) continue;
        const int64_t more = blocks_of(s, width, batch);
        if (a.count == kStatesPerLaunch || blocks + more > 0x7fffffffLL) VSK_TRY(launch());
        StateMove& m = a.move[a.count++];
        m.src = (const uint8_t*)s.src;
        m.dst = (uint8_t*)s.dst;
        m.src_row = s.src_row_stride;
        m.dst_row = s.dst_row_stride;
        m.src_outer = s.src_outer_stride;
        m.dst_outer = s.dst_outer_stride;
        m.outer = s.outer;
        m.inner = s.steps * s.step_bytes;
        m.step = s.timed ? s.step_bytes : 0;
        m.first_block = (unsigned)blocks;
        m.tiles = (unsigned)(more / (batch * s.outer));
        blocks += more;
      }
      VSK_TRY(launch());
    }
  tl_mark(ctx, "reorder_states");
  VSK_CUDA(ctx, cudaStreamSynchronize(ctx->stream));
  if (*bad) return fail(ctx, VSK_ERR_INVALID_INPUT, "a parent is outside [-1, %d): its batch entry's states were left as they were", beams);
  return VSK_OK;
}

}  // extern "C"
