// The fp8 linear for few rows: y[r] = act(W x[r] + b).
//
// Bound by the bytes of the weights, so everything serves their stream: a warp
// owns 16 weight rows and a slice of k and asks for all of it at once, 32 bytes
// a lane and row (a quad reads the 128 bytes of one k block of one row), before
// it looks at x.  The lane's bytes are used as the A fragment of mma.sync as
// they come: which k a fragment slot holds does not matter as long as x, the B
// fragment, is permuted alike, and both are read as the same 32 bytes of a
// block.  mma.sync, not tcgen05: at so few rows the products take less
// than a tenth of the time of the weights' bytes, and this path has no
// tensor-memory set-up and no copy into shared memory before it can start.
//
// A CTA is kBands bands of 16 weight rows times kSlices slices of k; with few
// bands a cluster splits k further, the partial sums meeting in the first
// CTA's shared memory.  Each CTA brings its slice of the rows of x to e4m3
// itself (a few KB from L2), which saves a launch.
//
// n 4096, k 1024 (4.2 MB of weights, 0.66 us of memory), each call on weights that
// are not in L2: 3.6 us for one row, 4.2 for 8, 5.3 for 14 (4.7 where they come as
// codes, so 0.6 us are their way to e4m3).  One row's time is the launch, the
// first loads' latency and the join; what the others add is each CTA's own work on its
// slice of the rows.  The INT8 linear takes 3.5 us for the 14.
#include "expert_gemv.hpp"

#include <algorithm>

#include "fp8.cuh"
#include "launch.hpp"

namespace cq {

namespace {

constexpr int kThreads = 256, kWarps = 8;
constexpr int kMaxRows = kGemvMaxRows, kTiles = kMaxRows / 8;
constexpr int kAhead = 4;       // k blocks a warp has in flight
constexpr int kSmemMax = 200 * 1024;


__device__ __forceinline__ void mma_e4m3(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                         uint32_t b1) {
  asm("mma.sync.aligned.m16n8k32.row.col.f32.e4m3.e4m3.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

__device__ __forceinline__ void st_dsmem_f32(uint32_t addr, float v) {
  asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(addr), "f"(v) : "memory");
}

__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); }

// Blocks [kb0, kb1) of the rows of x into shared memory: codes, `pitch` bytes a
// row, and their scales [block][kMaxRows].
template <int DT, int SRC>
__device__ __forceinline__ void stage_x(const ExpertGemvArgs& a, int kb0, int kb1, uint8_t* xs, int pitch, float* sx) {
  const int n = a.rows, blocks = kb1 - kb0;
  if constexpr (SRC == kSourceT) {
    const bool aligned = ((a.ldx * 2) & 15) == 0 && (reinterpret_cast<uintptr_t>(a.x) & 15) == 0;
    // half warps share the rows out, a power of two of them to a row, each
    // with up to four of its blocks on their way
    const int half = threadIdx.x >> 4, lane = threadIdx.x & 15;
    constexpr int kHalves = kThreads / 16, kFlight = 4;
    const int shift = n > 8 ? 0 : n > 4 ? 1 : n > 2 ? 2 : n > 1 ? 3 : 4;  // log2 of half warps to a row
    for (int r0 = 0; r0 < n; r0 += kHalves >> shift) {
      const int r = r0 + (half >> shift);
      const char* row = reinterpret_cast<const char*>(a.x) + r * a.ldx * 2;
      // the same turns in every half warp: the shuffles below are the warp's
      for (int b0 = 0; b0 < blocks; b0 += kFlight << shift) {
        Raw8<DT> raw[kFlight];
#pragma unroll
        for (int u = 0; u < kFlight; ++u) {
          const int b = b0 + (u << shift) + (half & ((1 << shift) - 1));
          raw[u] = Raw8<DT>{};
          if (r < n && b < blocks) raw[u] = load_row8<DT>(row, (kb0 + b) * kFp8Block + lane * 8, a.K, aligned);
        }
#pragma unroll
        for (int u = 0; u < kFlight; ++u) {
          const int b = b0 + (u << shift) + (half & ((1 << shift) - 1));
          if (b0 + (u << shift) >= blocks) break;
          int e;
          const uint2 out = quantize8<DT>(raw[u], e);
          if (r < n && b < blocks) {
            *reinterpret_cast<uint2*>(xs + r * pitch + b * 128 + lane * 8) = out;
            if (lane == 0) sx[b * kMaxRows + r] = pow2f(e);
          }
        }
      }
    }
  } else {
    // 16 bytes a thread; the rows of codes are 16-byte aligned
    const int pieces = blocks * 8;
    for (int i = threadIdx.x; i < n * pieces; i += kThreads) {
      const int r = i / pieces, p = i - r * pieces;
      const int k = kb0 * kFp8Block + p * 16;
      uint4 v = make_uint4(0, 0, 0, 0);
      const uint8_t* from = reinterpret_cast<const uint8_t*>(a.x) + r * a.ldx + k;
      if (k + 16 <= a.K) {
        v = *reinterpret_cast<const uint4*>(from);
      } else {
        uint32_t w[4] = {0, 0, 0, 0};
#pragma unroll
        for (int j = 0; j < 16; ++j)
          if (k + j < a.K) w[j / 4] |= static_cast<uint32_t>(from[j]) << (8 * (j & 3));
        v = make_uint4(w[0], w[1], w[2], w[3]);
      }
      *reinterpret_cast<uint4*>(xs + r * pitch + p * 16) = v;
    }
    for (int i = threadIdx.x; i < n * blocks; i += kThreads) {
      const int b = i / n, r = i - b * n;
      sx[b * kMaxRows + r] = a.x_scales[static_cast<int64_t>(kb0 + b) * n + r];
    }
  }
}

__host__ __device__ inline int x_pitch(int blocks) { return blocks * 128 + 16; }  // quads of a row pair miss each other's banks

template <int DT, int SRC, int BANDS>
__global__ void __launch_bounds__(kThreads) expert_gemv_kernel(const ExpertGemvArgs a, int splits) {
  constexpr int SLICES = kWarps / BANDS, ROWS = 16 * BANDS;
  extern __shared__ __align__(16) uint8_t gemv_smem[];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int band = warp % BANDS, slice = warp / BANDS;
  const int g = lane >> 2, q = lane & 3;
  const int KB = (a.K + kFp8Block - 1) / kFp8Block;
  const int rank = splits > 1 ? static_cast<int>(cluster_ctarank()) : 0;
  const int per = (KB + splits - 1) / splits;
  const int kb0 = rank * per, kb1 = min(KB, kb0 + per);
  // this warp's blocks of the CTA's
  const int wper = (per + SLICES - 1) / SLICES;
  const int wb0 = min(kb0 + slice * wper, kb1), wb1 = min(wb0 + wper, kb1);
  const int n0 = blockIdx.x / splits * ROWS;
  const int staged = (a.rows + 7) & ~7;
  const int pitch = x_pitch(per);
  uint8_t* xs = gemv_smem;
  float* sx = reinterpret_cast<float*>(xs + staged * pitch);       // [per][kMaxRows]
  float* red = sx + per * kMaxRows;                                // [SLICES][kMaxRows][ROWS + 1]
  float* clus = red + SLICES * kMaxRows * (ROWS + 1);             // [splits][kMaxRows][ROWS], in rank 0
  if (splits > 1) cluster_arrive();  // the CTAs of the cluster run

  pdl_launch_dependents();
  // weights are nobody's result: all of the warp's first blocks at once, while
  // the kernel before still runs.  Rows past N read the last row; what they make
  // is not stored.
  const char* w_lo = reinterpret_cast<const char*>(a.w) + min(n0 + band * 16 + g, a.N - 1) * a.ldw + q * 32;
  const char* w_hi = reinterpret_cast<const char*>(a.w) + min(n0 + band * 16 + g + 8, a.N - 1) * a.ldw + q * 32;
  const float* sw = a.w_scales + static_cast<int64_t>(min(n0 + band * 16, a.N - 1) / kFp8Block) * KB;
  uint4 w[kAhead][4];
#pragma unroll
  for (int i = 0; i < kAhead; ++i) {
    if (wb0 + i < wb1) {
      ld_global_cg_v8(w_lo + static_cast<int64_t>(wb0 + i) * 128, w[i][0], w[i][1]);
      ld_global_cg_v8(w_hi + static_cast<int64_t>(wb0 + i) * 128, w[i][2], w[i][3]);
    }
  }
  pdl_wait();

  const int n = a.rows, tiles = (n + 7) >> 3;
  stage_x<DT, SRC>(a, kb0, kb1, xs, pitch, sx);
  __syncthreads();
  float acc[kTiles][4] = {};
  for (int b0 = wb0; b0 < wb1; b0 += kAhead) {
    if (b0 != wb0) {
#pragma unroll
      for (int i = 0; i < kAhead; ++i) {
        if (b0 + i < wb1) {
          ld_global_cg_v8(w_lo + static_cast<int64_t>(b0 + i) * 128, w[i][0], w[i][1]);
          ld_global_cg_v8(w_hi + static_cast<int64_t>(b0 + i) * 128, w[i][2], w[i][3]);
        }
      }
    }
#pragma unroll
    for (int i = 0; i < kAhead; ++i) {
      if (b0 + i >= wb1) break;
      const uint32_t lo[8] = {w[i][0].x, w[i][0].y, w[i][0].z, w[i][0].w, w[i][1].x, w[i][1].y, w[i][1].z, w[i][1].w};
      const uint32_t hi[8] = {w[i][2].x, w[i][2].y, w[i][2].z, w[i][2].w, w[i][3].x, w[i][3].y, w[i][3].z, w[i][3].w};
      const int b = b0 + i - kb0;
      const float scale = __ldg(sw + b0 + i);
#pragma unroll
      for (int t = 0; t < kTiles; ++t) {
        if (t < tiles) {
          const uint4* xp = reinterpret_cast<const uint4*>(xs + (t * 8 + g) * pitch + b * 128 + q * 32);
          const uint4 x0 = xp[0], x1 = xp[1];
          const uint32_t x[8] = {x0.x, x0.y, x0.z, x0.w, x1.x, x1.y, x1.z, x1.w};
          float p[4] = {};
#pragma unroll
          for (int s = 0; s < 4; ++s) mma_e4m3(p, lo[2 * s], hi[2 * s], lo[2 * s + 1], hi[2 * s + 1], x[2 * s], x[2 * s + 1]);
          const float2 f = *reinterpret_cast<const float2*>(sx + b * kMaxRows + t * 8 + q * 2);
          const float f0 = f.x * scale, f1 = f.y * scale;
          acc[t][0] = fmaf(p[0], f0, acc[t][0]);
          acc[t][1] = fmaf(p[1], f1, acc[t][1]);
          acc[t][2] = fmaf(p[2], f0, acc[t][2]);
          acc[t][3] = fmaf(p[3], f1, acc[t][3]);
        }
      }
    }
  }
  // the slices' sums, row by row of the tile
#pragma unroll
  for (int t = 0; t < kTiles; ++t) {
    if (t < tiles) {
#pragma unroll
      for (int i = 0; i < 4; ++i)
        red[(slice * kMaxRows + t * 8 + q * 2 + (i & 1)) * (ROWS + 1) + band * 16 + g + (i >> 1) * 8] = acc[t][i];
    }
  }
  __syncthreads();
  if (splits > 1) cluster_wait();
  for (int i = threadIdx.x; i < n * ROWS; i += kThreads) {
    const int r = i / ROWS, c = i % ROWS;
    float v = 0.0f;
#pragma unroll
    for (int s = 0; s < SLICES; ++s) v += red[(s * kMaxRows + r) * (ROWS + 1) + c];
    if (splits > 1) {
      st_dsmem_f32(mapa_shared(smem_u32(clus + (rank * kMaxRows + r) * ROWS + c), 0), v);
    } else if (n0 + c < a.N) {
      if (a.bias != nullptr) v += ld_t<DT>(a.bias, n0 + c);
      v = activate(v, a.act);
      st_t<DT>(a.y, r * a.ldy + n0 + c, v);
    }
  }
  if (splits > 1) {
    cluster_sync_all();
    if (rank == 0) {
      for (int i = threadIdx.x; i < n * ROWS; i += kThreads) {
        const int r = i / ROWS, c = i % ROWS;
        if (n0 + c >= a.N) continue;
        float v = 0.0f;
        for (int s = 0; s < splits; ++s) v += clus[(s * kMaxRows + r) * ROWS + c];
        if (a.bias != nullptr) v += ld_t<DT>(a.bias, n0 + c);
        v = activate(v, a.act);
        st_t<DT>(a.y, r * a.ldy + n0 + c, v);
      }
    }
  }
}

struct GemvPlan {
  int bands, splits, smem;
};

int smem_of(int rows, int KB, int bands, int splits) {
  const int per = (KB + splits - 1) / splits;
  const int staged = (rows + 7) & ~7;
  int bytes = staged * x_pitch(per) + per * kMaxRows * 4;
  bytes += kWarps / bands * kMaxRows * (16 * bands + 1) * 4;
  if (splits > 1) bytes += splits * kMaxRows * 16 * bands * 4;
  return bytes;
}

GemvPlan plan(int rows, int N, int K, int num_sms) {
  const int KB = (K + kFp8Block - 1) / kFp8Block;
  GemvPlan p{2, 1, 0};
  if ((N + 31) / 32 < num_sms / 2) p.bands = 1;
  const int64_t ctas = (N + 16 * p.bands - 1) / (16 * p.bands);
  const int slices = kWarps / p.bands;
  // split k while a warp still has a block of its own and the GPU has room, or
  // while the rows of x do not fit
  for (int s : {2, 4, 8}) {
    const int per = (KB + s - 1) / s;
    if ((s - 1) * per >= KB) break;
    const bool room = ctas * s <= 2 * num_sms && per >= slices;
    if (room || smem_of(rows, KB, p.bands, p.splits) > 56 * 1024) p.splits = s;
  }
  p.smem = smem_of(rows, KB, p.bands, p.splits);
  return p;
}

template <int DT, int SRC, int BANDS>
cudaError_t launch_typed(const GemvPlan& p, const ExpertGemvArgs& a, cudaStream_t stream, bool pdl) {
  static SharedMemoryOptIn opt_in;
  auto kernel = expert_gemv_kernel<DT, SRC, BANDS>;
  const cudaError_t e = opt_in.ensure(reinterpret_cast<const void*>(kernel), kSmemMax);
  if (e != cudaSuccess) return e;
  const int tiles = (a.N + 16 * BANDS - 1) / (16 * BANDS);
  return launch_clustered(kernel, dim3(tiles * p.splits), dim3(kThreads), p.smem, stream, pdl, p.splits, a, p.splits);
}

template <int DT>
cudaError_t launch_dtype(int source, const ExpertGemvArgs& a, int num_sms, cudaStream_t stream, bool pdl) {
  const GemvPlan p = plan(a.rows, a.N, a.K, num_sms);
  if (source == kSourceT)
    return p.bands == 1 ? launch_typed<DT, kSourceT, 1>(p, a, stream, pdl) : launch_typed<DT, kSourceT, 2>(p, a, stream, pdl);
  return p.bands == 1 ? launch_typed<DT, kSourceCodes, 1>(p, a, stream, pdl)
                      : launch_typed<DT, kSourceCodes, 2>(p, a, stream, pdl);
}

}  // namespace

bool expert_gemv_fits(int rows, int N, int K) {
  // Every CTA brings the rows to e4m3 for itself, so the work beside the weights'
  // stream is as rows * N * K, while tiles on the tensor cores start later and
  // take a second launch.  us on the GPU here / there (n x k):
  //   rows          8          16          24
  //   4096 x 1024   4.2/7.6    5.5/7.4     7.4/7.3
  //   1024 x 4096   4.6/12.0   6.5/12.0    9.7/12.0
  //   2048 x 2048   4.7/8.8    6.5/8.8     9.6/8.8
  //   4096 x 4096   8.4/13.9   14.8/12.4   30.3/12.1
  // A call from Python takes 7.7 us of host time here and 12.2 there, so that up to
  // 24 rows it is the faster one here at each of the first three; replayed from a graph,
  // 17 to 24 rows lose up to a tenth at 2048 x 2048 by that.
  if (rows > kMaxRows || (rows > 8 && static_cast<int64_t>(N) * K > (1 << 23))) return false;
  const int KB = (K + kFp8Block - 1) / kFp8Block;
  int splits = 1;
  for (int s : {2, 4, 8})
    if ((s - 1) * ((KB + s - 1) / s) < KB) splits = s;
    else break;
  return smem_of(rows, KB, 2, splits) <= kSmemMax && smem_of(rows, KB, 1, splits) <= kSmemMax;
}

cudaError_t launch_expert_gemv(int dtype, int source, const ExpertGemvArgs& a, int num_sms, cudaStream_t stream, bool pdl) {
  if (!expert_gemv_fits(a.rows, a.N, a.K)) return cudaErrorInvalidValue;
  return dtype == kF16 ? launch_dtype<kF16>(source, a, num_sms, stream, pdl)
                       : launch_dtype<kBF16>(source, a, num_sms, stream, pdl);
}

}  // namespace cq
