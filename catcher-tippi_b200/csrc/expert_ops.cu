// Kernels of the fp8 linear and the linears of experts; see expert_ops.hpp.
#include "expert_ops.hpp"

#include <algorithm>

#include "fp8.cuh"
#include "launch.hpp"

namespace cq {

namespace {

// ------------------------------------------------------------------ rows to e4m3

// A CTA takes 16 rows times four blocks of 128 values, a half warp one row:
// its four blocks are loaded (a kilobyte next to each other for 16-bit rows)
// before the first is looked at, eight values a lane; the largest magnitude by
// shuffles, then the codes, eight bytes a lane.  The scales leave as runs of 16
// rows: written one by one they were scattered over as many sectors and cost as
// much as the codes.  Bound by memory: (2 + 1) bytes a value for 16-bit rows
// (16384 x 4096: 35 us, 31 of bytes at the copy rate).
constexpr int kQuantThreads = 256, kQuantRows = kQuantThreads / 16;
constexpr int kQuantBlocks = 4;

template <int DT>
__global__ void __launch_bounds__(kQuantThreads) quantize_rows_kernel(const QuantizeRowsArgs a) {
  __shared__ float scale_s[kQuantBlocks][kQuantRows];
  pdl_wait();
  pdl_launch_dependents();  // in this order: the product after it may rely on the offsets
  constexpr int kSize = DT == kF32 ? 4 : 2;
  const int blocks = (a.cols + kFp8Block - 1) / kFp8Block;
  const bool aligned = ((a.ldx * kSize) & 15) == 0 && (reinterpret_cast<uintptr_t>(a.x) & 15) == 0;
  const int half = threadIdx.x >> 4, lane = threadIdx.x & 15;
  const int groups = (blocks + kQuantBlocks - 1) / kQuantBlocks;
  const int64_t row0 = static_cast<int64_t>(blockIdx.x / groups) * kQuantRows, row = row0 + half;
  const int b0 = static_cast<int>(blockIdx.x % groups) * kQuantBlocks;
  int64_t src = row < a.rows ? row : -1;
  if (src >= 0 && a.row_index != nullptr) src = a.row_index[row];
  const bool live = src >= 0 && src < a.x_rows;
  const char* from = reinterpret_cast<const char*>(a.x) + src * a.ldx * kSize;
  Raw8<DT> raw[kQuantBlocks];
#pragma unroll
  for (int u = 0; u < kQuantBlocks; ++u) {
    raw[u] = Raw8<DT>{};
    if (live && b0 + u < blocks) raw[u] = load_row8<DT>(from, (b0 + u) * kFp8Block + lane * 8, a.cols, aligned);
  }
#pragma unroll
  for (int u = 0; u < kQuantBlocks; ++u) {
    int e;
    const uint2 out = quantize8<DT>(raw[u], e);
    const int k = (b0 + u) * kFp8Block + lane * 8;
    if (live && b0 + u < blocks && k < a.ld) *reinterpret_cast<uint2*>(a.codes + row * a.ld + k) = out;
    if (lane == 0) scale_s[u][half] = pow2f(e);
  }
  __syncthreads();
  const int u = threadIdx.x / kQuantRows, r = threadIdx.x % kQuantRows;
  if (u < kQuantBlocks && b0 + u < blocks && row0 + r < a.rows)
    a.scales[static_cast<int64_t>(b0 + u) * a.rows + row0 + r] = scale_s[u][r];
}

// One CTA per 128 x 128 block of a weight; used when a layer is made.  4096 x 4096:
// 46 us, where its bytes take 13 (it reads a block twice and stores single bytes).
__global__ void __launch_bounds__(kQuantThreads)
    quantize_weight_kernel(const float* w, int rows, int cols, uint8_t* codes, float* scales) {
  const int n0 = blockIdx.y * kFp8Block, k0 = blockIdx.x * kFp8Block;
  const int n1 = min(n0 + kFp8Block, rows), k1 = min(k0 + kFp8Block, cols);
  __shared__ uint32_t most;
  if (threadIdx.x == 0) most = 0;
  __syncthreads();
  const int c = threadIdx.x % kFp8Block, r0 = threadIdx.x / kFp8Block;
  constexpr int kStep = kQuantThreads / kFp8Block;
  uint32_t top = 0;
  if (k0 + c < k1)
    for (int n = n0 + r0; n < n1; n += kStep)
      top = max(top, finite_magnitude(w[static_cast<int64_t>(n) * cols + k0 + c]));
  atomicMax(&most, top);
  __syncthreads();
  const int e = fp8_scale_exponent(most);
  const float inv = pow2f(-e);
  if (k0 + c < k1)
    for (int n = n0 + r0; n < n1; n += kStep) {
      const int64_t i = static_cast<int64_t>(n) * cols + k0 + c;
      codes[i] = static_cast<uint8_t>(e4m3x2(w[i] * inv, 0.0f));
    }
  if (threadIdx.x == 0) scales[static_cast<int64_t>(blockIdx.y) * gridDim.x + blockIdx.x] = pow2f(e);
}

template <int DT>
__global__ void __launch_bounds__(256) round_kernel(const float* v, int64_t n, void* out) {
  for (int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x; i < n; i += static_cast<int64_t>(gridDim.x) * 256)
    st_t<DT>(out, i, v[i]);
}

// ------------------------------------------------------------------ gather

// 16-bit rows to 16-byte aligned rows, eight values a thread: the order of a
// row list, or rows whose own alignment a tile copy cannot take.
__global__ void __launch_bounds__(256) gather_rows_kernel(const GatherRowsArgs a) {
  pdl_wait();
  pdl_launch_dependents();  // in this order: the product after it may rely on the offsets
  const int chunks = (a.cols + 7) / 8;
  const bool aligned = (a.ldx & 7) == 0 && (reinterpret_cast<uintptr_t>(a.x) & 15) == 0;
  const int64_t items = static_cast<int64_t>(a.rows) * chunks;
  for (int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x; i < items;
       i += static_cast<int64_t>(gridDim.x) * 256) {
    const int64_t row = i / chunks;
    const int c = static_cast<int>(i - row * chunks) * 8;
    const int64_t src = a.row_index != nullptr ? a.row_index[row] : row;
    if (src < 0 || src >= a.x_rows) continue;
    const uint16_t* from = reinterpret_cast<const uint16_t*>(a.x) + src * a.ldx + c;
    uint4 v;
    if (aligned && c + 8 <= a.cols) {
      v = *reinterpret_cast<const uint4*>(from);
    } else {
      uint16_t h[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) h[j] = c + j < a.cols ? from[j] : static_cast<uint16_t>(0);
      v = make_uint4(h[0] | h[1] << 16, h[2] | h[3] << 16, h[4] | h[5] << 16, h[6] | h[7] << 16);
    }
    *reinterpret_cast<uint4*>(reinterpret_cast<uint16_t*>(a.out) + row * a.ld + c) = v;
  }
}

// ------------------------------------------------------------------ router

// A block takes kRouteTokens tokens, eight lanes a token.  A logit and its
// expert become one integer, the higher the better (equal logits: the lower
// expert), so that choosing is sorting: each lane keeps the best K of its
// experts as a sorted list in registers (an insertion is K maxima and minima,
// no branches), and the lanes' lists are merged pairwise (the best K of two
// sorted lists are max(a[i], b[K - 1 - i]), a bitonic sequence).  One warp
// maximum a round and token instead took 33.6 us for both kernels against 19.3
// (16384 tokens, 128 experts, 8 best, bf16).  Bound by latency and occupancy, not by
// memory: of these 19 us the choice takes 11 and the places 9, each on 128 CTAs, one an
// SM with half of its warps, issuing 0.6 and 0.4 instructions a cycle and scheduler.
// f32 logits take 22.8 us; more than 8 best, whose lists of 32 keys do not fit a
// thread's registers, 27 to 34 us for bf16 and 76 to 83 for f32.  Which tokens of the block
// chose an expert is a bit mask per expert in shared memory, so that a pair's
// rank inside the block is a population count, the same in every run.  One
// block does it all where the tokens fit one; otherwise a second kernel adds up
// the blocks' counts.
constexpr int kRouteTokens = 128;
constexpr int kRouteThreads = 1024;
constexpr int kRouteWords = kRouteTokens / 32;
static_assert(kRouteThreads == kRouteTokens * 8 && kRouteThreads >= kMaxExperts, "eight lanes a token, a thread an expert");

constexpr int kRouteLanes = 8;

// A logit's order above the complement of its expert: 32 bits for 16-bit
// logits, 64 for f32; 0 for -infinity and NaN.
template <int DT>
struct RouteKey {
  using Type = uint32_t;
  static __device__ __forceinline__ Type make(uint32_t bits, int e) {
    const float v = DT == kBF16 ? __uint_as_float(bits << 16) : __half2float(__ushort_as_half(static_cast<uint16_t>(bits)));
    if (!(v > -INFINITY)) return 0u;
    const uint32_t u = bits == 0x8000u ? 0u : bits;  // -0 and +0 are equal
    return (((u & 0x8000u) ? (~u & 0xFFFFu) : (u | 0x8000u)) << 16) | static_cast<uint32_t>(0xFFFF - e);
  }
  static __device__ __forceinline__ int expert(Type k) { return 0xFFFF - static_cast<int>(k & 0xFFFFu); }
  static __device__ __forceinline__ float value(Type k) {
    const uint32_t o = k >> 16, u = (o & 0x8000u) ? (o & 0x7FFFu) : (~o & 0xFFFFu);
    return DT == kBF16 ? __uint_as_float(u << 16) : __half2float(__ushort_as_half(static_cast<uint16_t>(u)));
  }
};
template <>
struct RouteKey<kF32> {
  using Type = unsigned long long;
  static __device__ __forceinline__ Type make(uint32_t bits, int e) {
    const float v = __uint_as_float(bits);
    if (!(v > -INFINITY)) return 0ull;
    const uint32_t u = __float_as_uint(v + 0.0f);  // -0 and +0 are equal
    const uint32_t o = (u & 0x80000000u) ? ~u : (u | 0x80000000u);
    return (static_cast<Type>(o) << 32) | static_cast<uint32_t>(0xFFFF - e);
  }
  static __device__ __forceinline__ int expert(Type k) { return 0xFFFF - static_cast<int>(k & 0xFFFFu); }
  static __device__ __forceinline__ float value(Type k) {
    const uint32_t o = static_cast<uint32_t>(k >> 32);
    return __uint_as_float((o & 0x80000000u) ? (o & 0x7FFFFFFFu) : ~o);
  }
};

__device__ __forceinline__ float route_share(float v, float most) {
  return most == INFINITY ? (v == INFINITY ? 1.0f : 0.0f) : expf(v - most);
}

// f(logit's bits, expert) for each logit of a lane's share of the token: eight
// (f32: four) neighbours at a time where they can be loaded at once.
template <int DT, class F>
__device__ __forceinline__ void each_logit(const RouteArgs& a, int64_t t, int lane, F&& f) {
  constexpr int kSize = DT == kF32 ? 4 : 2, kPer = 16 / kSize;
  const char* row = reinterpret_cast<const char*>(a.logits) + t * a.ld * kSize;
  if ((reinterpret_cast<uintptr_t>(row) & 15) == 0 && a.experts % kPer == 0) {
#pragma unroll 2
    for (int e = lane * kPer; e < a.experts; e += kRouteLanes * kPer) {
      const uint4 u = *reinterpret_cast<const uint4*>(row + e * kSize);
      const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
      for (int i = 0; i < kPer; ++i) f(DT == kF32 ? w[i % 4] : (w[i / 2] >> (16 * (i & 1))) & 0xFFFFu, e + i);
    }
  } else {
#pragma unroll 4
    for (int e = lane; e < a.experts; e += kRouteLanes)
      f(DT == kF32 ? reinterpret_cast<const uint32_t*>(row)[e] : reinterpret_cast<const uint16_t*>(row)[e], e);
  }
}

// Token t, the slot-th of its block, by eight neighbouring lanes: expert and
// weight, the masks, and (where `chosen` is given) the block's note of them
// [kRouteTokens][top].  All lanes of the warp; `there`: the token exists.
template <int DT, int K>
__device__ __forceinline__ void route_token(const RouteArgs& a, int64_t t, int slot, bool there, int lane,
                                            uint32_t* masks, int16_t* chosen) {
  using Key = typename RouteKey<DT>::Type;
  Key best[K] = {};
  if (there)
    each_logit<DT>(a, t, lane, [&](uint32_t bits, int e) {
      Key x = RouteKey<DT>::make(bits, e);
#pragma unroll
      for (int i = 0; i < K; ++i) {
        const Key high = max(best[i], x);
        x = min(best[i], x);
        best[i] = high;
      }
    });
#pragma unroll
  for (int o = 1; o < kRouteLanes; o <<= 1) {
    Key other[K];
#pragma unroll
    for (int i = 0; i < K; ++i) other[i] = __shfl_xor_sync(0xFFFFFFFFu, best[K - 1 - i], o);
#pragma unroll
    for (int i = 0; i < K; ++i) best[i] = max(best[i], other[i]);
#pragma unroll
    for (int d = K / 2; d > 0; d >>= 1)
#pragma unroll
      for (int i = 0; i < K; ++i)
        if ((i & d) == 0) {
          const Key high = max(best[i], best[i + d]);
          best[i + d] = min(best[i], best[i + d]);
          best[i] = high;
        }
  }
  const float most = RouteKey<DT>::value(best[0]);
  constexpr int kMine = (K + kRouteLanes - 1) / kRouteLanes;  // choices that a lane writes
  float share[kMine], sum = 0.0f;
  int expert[kMine];
#pragma unroll
  for (int m = 0; m < kMine; ++m) {
    share[m] = 0.0f;
    expert[m] = -1;
#pragma unroll
    for (int i = m * kRouteLanes; i < K && i < (m + 1) * kRouteLanes; ++i)
      if (i % kRouteLanes == lane && i < a.top && best[i] != 0) {
        expert[m] = RouteKey<DT>::expert(best[i]);
        share[m] = route_share(RouteKey<DT>::value(best[i]), most);
      }
    sum += share[m];
  }
  if (!a.renormalize) {
    // the denominator over every expert that can be taken
    sum = 0.0f;
    if (there)
      each_logit<DT>(a, t, lane, [&](uint32_t bits, int e) {
        const Key x = RouteKey<DT>::make(bits, e);
        if (x != 0) sum += route_share(RouteKey<DT>::value(x), most);
      });
  }
#pragma unroll
  for (int o = 1; o < kRouteLanes; o <<= 1) sum += __shfl_xor_sync(0xFFFFFFFFu, sum, o);
  if (!there) return;
#pragma unroll
  for (int m = 0; m < kMine; ++m) {
    const int j = m * kRouteLanes + lane;
    if (j >= a.top) break;
    a.expert[t * a.top + j] = expert[m];
    a.weight[t * a.top + j] = expert[m] >= 0 ? share[m] / sum : 0.0f;
    if (chosen != nullptr) chosen[slot * a.top + j] = static_cast<int16_t>(expert[m]);
    if (expert[m] >= 0) atomicOr(&masks[expert[m] * kRouteWords + (slot >> 5)], 1u << (slot & 31));
  }
}

__device__ __forceinline__ int mask_count(const uint32_t* m) {
  int n = 0;
#pragma unroll
  for (int w = 0; w < kRouteWords; ++w) n += __popc(m[w]);
  return n;
}

__device__ __forceinline__ int mask_rank(const uint32_t* m, int slot) {
  int n = 0;
#pragma unroll
  for (int w = 0; w < kRouteWords; ++w) {
    if (w < (slot >> 5)) n += __popc(m[w]);
    else if (w == (slot >> 5)) n += __popc(m[w] & ((1u << (slot & 31)) - 1u));
  }
  return n;
}

// base[e] (shared, kMaxExperts values) -> the exclusive sum before e; returns
// the total.  All threads of the block; experts <= kRouteThreads.
__device__ __forceinline__ int exclusive_sum(int* base, int experts, int* scratch) {
  const int t = threadIdx.x, lane = t & 31, warp = t >> 5;
  int v = t < experts ? base[t] : 0, sum = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int up = __shfl_up_sync(0xFFFFFFFFu, sum, o);
    if (lane >= o) sum += up;
  }
  if (lane == 31) scratch[warp] = sum;
  __syncthreads();
  if (warp == 0) {
    int s = lane < kRouteThreads / 32 ? scratch[lane] : 0;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int up = __shfl_up_sync(0xFFFFFFFFu, s, o);
      if (lane >= o) s += up;
    }
    scratch[lane] = s;
  }
  __syncthreads();
  const int before = warp ? scratch[warp - 1] : 0;
  if (t < experts) base[t] = before + sum - v;
  const int total = scratch[31];
  __syncthreads();
  return total;
}

// Writes the sorted rows of the block's pairs from base[e], the first row that
// the block has in expert e.
__device__ __forceinline__ void place_pairs(const RouteArgs& a, int t0, int n, const int* base, const uint32_t* masks,
                                            const int16_t* chosen) {
  for (int i = threadIdx.x; i < n * a.top; i += kRouteThreads) {
    const int slot = i / a.top;
    const int e = chosen[i];
    int row = -1;
    if (e >= 0) {
      row = base[e] + mask_rank(masks + e * kRouteWords, slot);
      a.token[row] = t0 + slot;
    }
    a.position[static_cast<int64_t>(t0) * a.top + i] = row;
  }
}

__device__ __forceinline__ void write_tail(const RouteArgs& a, int total, int first, int step) {
  for (int64_t p = static_cast<int64_t>(total) + first; p < static_cast<int64_t>(a.tokens) * a.top; p += step)
    a.token[p] = -1;
}

template <int DT, int K, bool ONE>
__global__ void __launch_bounds__(kRouteThreads) route_choose_kernel(const RouteArgs a) {
  extern __shared__ uint32_t route_smem[];
  uint32_t* masks = route_smem;                                         // [experts][kRouteWords]
  int* base = reinterpret_cast<int*>(masks + a.experts * kRouteWords);  // [experts] (ONE)
  int16_t* chosen = reinterpret_cast<int16_t*>(base + a.experts);       // [kRouteTokens][top] (ONE)
  __shared__ int scratch[32];
  for (int i = threadIdx.x; i < a.experts * kRouteWords; i += kRouteThreads) masks[i] = 0u;
  __syncthreads();
  pdl_launch_dependents();
  pdl_wait();
  const int t0 = blockIdx.x * kRouteTokens;
  const int n = min(kRouteTokens, a.tokens - t0);
  const int slot = threadIdx.x / kRouteLanes, lane = threadIdx.x % kRouteLanes;
  if ((threadIdx.x & ~31) / kRouteLanes < n)  // the warp has a token
    route_token<DT, K>(a, t0 + slot, slot, slot < n, lane, masks, ONE ? chosen : nullptr);
  __syncthreads();
  if constexpr (ONE) {
    for (int e = threadIdx.x; e < a.experts; e += kRouteThreads) base[e] = mask_count(masks + e * kRouteWords);
    __syncthreads();
    const int total = exclusive_sum(base, a.experts, scratch);
    for (int e = threadIdx.x; e <= a.experts; e += kRouteThreads) a.offsets[e] = e < a.experts ? base[e] : total;
    place_pairs(a, t0, n, base, masks, chosen);
    write_tail(a, total, threadIdx.x, kRouteThreads);
  } else {
    for (int e = threadIdx.x; e < a.experts; e += kRouteThreads)
      a.counts[static_cast<int64_t>(blockIdx.x) * a.experts + e] = mask_count(masks + e * kRouteWords);
  }
}

// The rows of each block's pairs: the counts of the blocks before it and of
// all experts before, from the counts of all blocks.
__global__ void __launch_bounds__(kRouteThreads) route_place_kernel(const RouteArgs a) {
  extern __shared__ uint32_t route_smem[];
  uint32_t* masks = route_smem;
  int* base = reinterpret_cast<int*>(masks + a.experts * kRouteWords);  // [experts]
  int* before = base + a.experts;                                       // [experts]
  int16_t* chosen = reinterpret_cast<int16_t*>(before + a.experts);
  __shared__ int scratch[32];
  pdl_launch_dependents();
  for (int i = threadIdx.x; i < a.experts * kRouteWords; i += kRouteThreads) masks[i] = 0u;
  for (int i = threadIdx.x; i < a.experts; i += kRouteThreads) base[i] = before[i] = 0;
  __syncthreads();
  pdl_wait();
  const int t0 = blockIdx.x * kRouteTokens;
  const int n = min(kRouteTokens, a.tokens - t0);
  for (int i = threadIdx.x; i < n * a.top; i += kRouteThreads) {
    const int e = a.expert[static_cast<int64_t>(t0) * a.top + i], slot = i / a.top;
    chosen[i] = static_cast<int16_t>(e);
    if (e >= 0) atomicOr(&masks[e * kRouteWords + (slot >> 5)], 1u << (slot & 31));
  }
  // threads that share an expert split the blocks
  const int lanes = kRouteThreads / a.experts;
  if (static_cast<int>(threadIdx.x) < lanes * a.experts) {
    const int e = threadIdx.x % a.experts;
    int all = 0, mine = 0;
#pragma unroll 8
    for (int b = threadIdx.x / a.experts; b < static_cast<int>(gridDim.x); b += lanes) {
      const int c = a.counts[static_cast<int64_t>(b) * a.experts + e];
      all += c;
      mine += b < static_cast<int>(blockIdx.x) ? c : 0;
    }
    atomicAdd(&base[e], all);
    atomicAdd(&before[e], mine);
  }
  __syncthreads();
  const int total = exclusive_sum(base, a.experts, scratch);
  if (blockIdx.x == 0)
    for (int e = threadIdx.x; e <= a.experts; e += kRouteThreads) a.offsets[e] = e < a.experts ? base[e] : total;
  for (int e = threadIdx.x; e < a.experts; e += kRouteThreads) before[e] += base[e];
  __syncthreads();
  place_pairs(a, t0, n, before, masks, chosen);
  write_tail(a, total, blockIdx.x * kRouteThreads + threadIdx.x, gridDim.x * kRouteThreads);
}

template <int DT, int K>
cudaError_t route_typed(const RouteArgs& a, cudaStream_t stream, bool pdl) {
  const int blocks = (a.tokens + kRouteTokens - 1) / kRouteTokens;
  const size_t masks = static_cast<size_t>(a.experts) * kRouteWords * 4;
  const size_t pairs = static_cast<size_t>(kRouteTokens) * a.top;
  const size_t one = masks + a.experts * 4 + pairs * 2, place = masks + a.experts * 8 + pairs * 2;
  if (blocks <= 1)
    return launch(route_choose_kernel<DT, K, true>, dim3(1), dim3(kRouteThreads), one, stream, pdl, a);
  cudaError_t e = launch(route_choose_kernel<DT, K, false>, dim3(blocks), dim3(kRouteThreads), masks, stream, pdl, a);
  if (e != cudaSuccess) return e;
  return launch(route_place_kernel, dim3(blocks), dim3(kRouteThreads), place, stream, pdl, a);
}

template <int DT>
cudaError_t route_dtype(const RouteArgs& a, cudaStream_t stream, bool pdl) {
  if (a.top <= 2) return route_typed<DT, 2>(a, stream, pdl);
  if (a.top <= 8) return route_typed<DT, 8>(a, stream, pdl);
  return route_typed<DT, 32>(a, stream, pdl);
}

// ------------------------------------------------------------------ combine

// A thread sums eight columns of one token.  Bound by memory: the rows of z
// once, y once.  Four experts' rows are on their way before the first is
// added.  `VEC`: every row is 16-byte aligned and dims a multiple of 8 (16384 tokens of 8
// experts, 2048 columns: 98 us); the other rows are read value by value, one expert
// after another (2047 columns: 172 us).
template <int T>
__device__ __forceinline__ void add_raw8(const Raw8<T>& r, float w, float (&acc)[8]) {
  float v[8];
  widen8<T>(r, v);
#pragma unroll
  for (int j = 0; j < 8; ++j) acc[j] = fmaf(w, v[j], acc[j]);
}

template <int DT, int ZT, bool VEC>
__global__ void __launch_bounds__(256) combine_kernel(const CombineArgs a) {
  pdl_launch_dependents();
  pdl_wait();
  constexpr int kSize = ZT == kF32 ? 4 : 2;
  const uint32_t chunks = (a.dims + 7) / 8;
  const int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
  if (i >= static_cast<int64_t>(a.tokens) * chunks) return;
  const int64_t t = i / chunks;
  const int d = static_cast<int>(i - t * chunks) * 8;
  const int32_t* position = a.position + t * a.top;
  const float* weight = a.weight + t * a.top;
  float acc[8] = {};
  for (int j0 = 0; j0 < a.top; j0 += 4) {
    if constexpr (VEC) {
      Raw8<ZT> raw[4];
      float w[4];
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const int p = j0 + u < a.top ? __ldg(position + j0 + u) : -1;
        const bool ok = p >= 0 && p < a.rows;
        w[u] = ok ? __ldg(weight + j0 + u) : 0.0f;
        const uint4* from = reinterpret_cast<const uint4*>(reinterpret_cast<const char*>(a.z) + (p * a.ldz + d) * kSize);
#pragma unroll
        for (int h = 0; h < (ZT == kF32 ? 2 : 1); ++h) raw[u].u[h] = ok ? from[h] : make_uint4(0, 0, 0, 0);
      }
#pragma unroll
      for (int u = 0; u < 4; ++u) add_raw8<ZT>(raw[u], w[u], acc);
    } else {
      for (int j = j0; j < min(j0 + 4, a.top); ++j) {
        const int p = __ldg(position + j);
        if (p < 0 || p >= a.rows) continue;
        const float w = __ldg(weight + j);
#pragma unroll
        for (int c = 0; c < 8; ++c)
          if (d + c < a.dims) acc[c] = fmaf(w, ld_t<ZT>(reinterpret_cast<const char*>(a.z) + p * a.ldz * kSize, d + c), acc[c]);
      }
    }
  }
  uint16_t* out = reinterpret_cast<uint16_t*>(a.y) + t * a.ldy + d;
  if constexpr (VEC) {
    uint32_t u[4];
#pragma unroll
    for (int c = 0; c < 4; ++c) u[c] = pack_t<DT>(acc[2 * c], acc[2 * c + 1]);
    *reinterpret_cast<uint4*>(out) = make_uint4(u[0], u[1], u[2], u[3]);
  } else {
    for (int c = 0; c < 8; ++c)
      if (d + c < a.dims) st_t<DT>(out, c, acc[c]);
  }
}

template <int DT, int ZT>
cudaError_t combine_typed(const CombineArgs& a, cudaStream_t stream, bool pdl) {
  const int64_t items = static_cast<int64_t>(a.tokens) * ((a.dims + 7) / 8);
  const dim3 grid(static_cast<unsigned>((items + 255) / 256));
  const int64_t bytes = ZT == kF32 ? 4 : 2;
  const bool vec = a.dims % 8 == 0 && (a.ldz * bytes) % 16 == 0 && a.ldy % 8 == 0 &&
                   (reinterpret_cast<uintptr_t>(a.z) & 15) == 0 && (reinterpret_cast<uintptr_t>(a.y) & 15) == 0;
  return vec ? launch(combine_kernel<DT, ZT, true>, grid, dim3(256), 0, stream, pdl, a)
             : launch(combine_kernel<DT, ZT, false>, grid, dim3(256), 0, stream, pdl, a);
}

}  // namespace

cudaError_t launch_quantize_rows(int dtype, const QuantizeRowsArgs& a, cudaStream_t stream, bool pdl) {
  if (a.rows == 0) return cudaSuccess;
  const int blocks = (a.cols + kFp8Block - 1) / kFp8Block;
  const int64_t grid = static_cast<int64_t>((a.rows + kQuantRows - 1) / kQuantRows) * ((blocks + kQuantBlocks - 1) / kQuantBlocks);
  if (grid > INT32_MAX) return cudaErrorInvalidValue;  // rows of 256 GB
  switch (dtype) {
    case kF16: return launch(quantize_rows_kernel<kF16>, dim3(static_cast<unsigned>(grid)), dim3(kQuantThreads), 0, stream, pdl, a);
    case kBF16: return launch(quantize_rows_kernel<kBF16>, dim3(static_cast<unsigned>(grid)), dim3(kQuantThreads), 0, stream, pdl, a);
    case kF32: return launch(quantize_rows_kernel<kF32>, dim3(static_cast<unsigned>(grid)), dim3(kQuantThreads), 0, stream, pdl, a);
    default: return cudaErrorInvalidValue;
  }
}

cudaError_t launch_quantize_weight(const float* w, int rows, int cols, uint8_t* codes, float* scales,
                                   cudaStream_t stream) {
  const dim3 grid((cols + kFp8Block - 1) / kFp8Block, (rows + kFp8Block - 1) / kFp8Block);
  return launch(quantize_weight_kernel, grid, dim3(kQuantThreads), 0, stream, false, w, rows, cols, codes, scales);
}

cudaError_t launch_round(int dtype, const float* v, int64_t n, void* out, cudaStream_t stream) {
  const int grid = static_cast<int>(std::min<int64_t>((n + 255) / 256, 1024));
  return dtype == kF16 ? launch(round_kernel<kF16>, dim3(grid), dim3(256), 0, stream, false, v, n, out)
                       : launch(round_kernel<kBF16>, dim3(grid), dim3(256), 0, stream, false, v, n, out);
}

cudaError_t launch_gather_rows(const GatherRowsArgs& a, cudaStream_t stream, bool pdl) {
  const int64_t items = static_cast<int64_t>(a.rows) * ((a.cols + 7) / 8);
  if (items == 0) return cudaSuccess;
  const int grid = static_cast<int>(std::min<int64_t>((items + 255) / 256, 148 * 16));
  return launch(gather_rows_kernel, dim3(grid), dim3(256), 0, stream, pdl, a);
}

size_t route_workspace(int tokens, int experts) {
  const size_t blocks = (static_cast<size_t>(tokens) + kRouteTokens - 1) / kRouteTokens;
  return blocks <= 1 ? 0 : blocks * experts * sizeof(int32_t);
}

cudaError_t launch_route(int dtype, const RouteArgs& a, cudaStream_t stream, bool pdl) {
  switch (dtype) {
    case kF16: return route_dtype<kF16>(a, stream, pdl);
    case kBF16: return route_dtype<kBF16>(a, stream, pdl);
    case kF32: return route_dtype<kF32>(a, stream, pdl);
    default: return cudaErrorInvalidValue;
  }
}

cudaError_t launch_combine(int dtype, const CombineArgs& a, cudaStream_t stream, bool pdl) {
  if (a.tokens == 0) return cudaSuccess;
  if (a.z_f32) return dtype == kF16 ? combine_typed<kF16, kF32>(a, stream, pdl) : combine_typed<kBF16, kF32>(a, stream, pdl);
  return dtype == kF16 ? combine_typed<kF16, kF16>(a, stream, pdl) : combine_typed<kBF16, kBF16>(a, stream, pdl);
}

}  // namespace cq
