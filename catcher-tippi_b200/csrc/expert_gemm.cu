// The grouped product y[r] = act(W[e] x[r] + b[e]) on the 5th-generation
// tensor cores, for rows sorted by expert; one expert and no offsets make it a
// plain linear.
//
// Rows of x are the MMA's M (128 tensor-memory lanes per CTA), weight rows its
// N, so that one thread of the epilogue holds a run of one row's outputs: its
// row's scale is one register, its stores are whole 32-byte sectors, and the
// largest magnitude of a 128-wide block of outputs (for codes) is found inside
// the thread.
//
// e4m3: kind::f8f6f4 sums one k block of 128 into tensor memory; the epilogue
// warps multiply that partial sum by scale(x) * scale(w) and add it to f32
// registers, while the tensor cores work on the next block in another
// tensor-memory buffer.  16-bit: kind::f16 sums all of k in tensor memory, and
// the epilogue of a tile overlaps the next tile's products.
//
// Persistent: a CTA (a pair of CTAs, or a cluster that splits k) takes every
// W-th tile of all experts' tiles; the tile list follows from the offsets,
// which only the device knows.
//   warp 0      copies tiles of x and W (TMA, 128-byte swizzle) into a ring
//   warp 1      issues tcgen05.mma
//   warp 2      owns the tensor memory
//   warp 3      e4m3: fetches the scales, eight k blocks ahead
//   warps 4-11  epilogue: two groups of four warps, each half of the columns
#include "expert_gemm.hpp"

#include <algorithm>

#include "fp8.cuh"
#include "launch.hpp"

namespace cq {

namespace {

constexpr int kThreads = 384;
constexpr int kEpiWarp0 = 4, kEpiWarps = 8, kEpiThreads = kEpiWarps * 32;
constexpr int kRowBytes = 128;                       // a k block of one row
constexpr int kXBytes = kGemmRows * kRowBytes;       // a stage's rows of x
constexpr int kMaxStages = 8;
constexpr uint32_t kTmemCols = 512;
constexpr int kSmemLimit = 227 * 1024;
constexpr int kMaxBuffers = 4;  // tensor-memory accumulators

enum Format : int { kFmtE4M3 = 0, kFmtF16 = 1, kFmtBF16 = 2 };

constexpr int kScaleBlocks = 8;  // k blocks of scales fetched at a time
constexpr int kScaleSlots = 2;
constexpr int kScaleBytes = kScaleBlocks * (kGemmRows + 2) * 4;
constexpr int kStageOut = kStoreRows * kStoreBytes;  // one of a warp's two tile stores

struct SmemPlan {
  int stage_bytes, stages, out_off, part_off, scale_off, list_off, bar_off, bytes;
};

__host__ __device__ inline SmemPlan plan_smem(bool e4m3, int bn, int pair, int splits, int experts) {
  SmemPlan p{};
  p.stage_bytes = kXBytes + bn / pair * kRowBytes;
  const int part = splits > 1 ? bn * kGemmRows * 4 : 0;
  const int list = (2 * (experts + 2) * 4 + 15) / 16 * 16;
  const int bars = (2 * kMaxStages + 2 * kMaxBuffers + 2 * kScaleSlots + 2) * 8 + 16;
  const int scales = e4m3 ? kScaleSlots * kScaleBytes : 0;
  const int rest = kEpiWarps * 2 * kStageOut + part + scales + list + bars;
  p.stages = (kSmemLimit - 2048 - rest) / p.stage_bytes;  // 2048: alignment, and the bias
  if (p.stages > kMaxStages) p.stages = kMaxStages;
  p.out_off = p.stages * p.stage_bytes;
  p.part_off = p.out_off + kEpiWarps * 2 * kStageOut;
  p.scale_off = p.part_off + part;
  p.list_off = p.scale_off + scales;
  p.bar_off = p.list_off + list;
  p.bytes = p.bar_off + bars + 1024;  // + alignment
  return p;
}

// --------------------------------------------------------------- tcgen05

template <int CG>
__device__ __forceinline__ void tmem_alloc(uint32_t* dst, uint32_t cols) {
  if constexpr (CG == 2)
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(dst)), "r"(cols) : "memory");
  else
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(dst)), "r"(cols) : "memory");
}

template <int CG>
__device__ __forceinline__ void tmem_release(uint32_t taddr, uint32_t cols) {
  if constexpr (CG == 2) {
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(taddr), "r"(cols) : "memory");
  } else {
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(taddr), "r"(cols) : "memory");
  }
}

__device__ __forceinline__ void tc_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }

template <int FMT, int CG>
__device__ __forceinline__ void tc_mma(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
  if constexpr (FMT == kFmtE4M3 && CG == 2)
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\ttcgen05.mma.cta_group::2.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}" ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(accumulate) : "memory");
  else if constexpr (FMT == kFmtE4M3)
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\ttcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}" ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(accumulate) : "memory");
  else if constexpr (CG == 2)
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\ttcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(accumulate) : "memory");
  else
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\ttcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(accumulate) : "memory");
}

// Arrives on `bar` when the MMAs issued so far are done; with a pair, on the
// barrier at that place in both CTAs.
template <int CG>
__device__ __forceinline__ void tc_commit(uint64_t* bar) {
  if constexpr (CG == 2)
    asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(smem_u32(bar)), "h"(static_cast<uint16_t>(3)) : "memory");
  else
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_u32(bar)) : "memory");
}

// 32 lanes x 32 columns: thread i of the warp gets its lane's 32 columns.
__device__ __forceinline__ void tmem_ld32(uint32_t taddr, uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,"
      "%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]),
        "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
        "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(taddr)
      : "memory");
}
// Two sums at once: a += s * x, b += s * y.
__device__ __forceinline__ void fma2(float& a, float& b, uint32_t x, uint32_t y, float s) {
  asm("{\n\t.reg .b64 p, q, t;\n\tmov.b64 p, {%2, %3};\n\tmov.b64 q, {%4, %4};\n\tmov.b64 t, {%0, %1};\n\t"
      "fma.rn.f32x2 t, p, q, t;\n\tmov.b64 {%0, %1}, t;\n\t}"
      : "+f"(a), "+f"(b) : "r"(x), "r"(y), "f"(s));
}
// Waits for the warp's tensor-memory loads.  The loaded registers pass through
// it, so that no use of them can be scheduled before it.
__device__ __forceinline__ void tmem_wait_ld(uint32_t (&r)[32]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]),
               "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15]),
               "+r"(r[16]), "+r"(r[17]), "+r"(r[18]), "+r"(r[19]), "+r"(r[20]), "+r"(r[21]), "+r"(r[22]), "+r"(r[23]),
               "+r"(r[24]), "+r"(r[25]), "+r"(r[26]), "+r"(r[27]), "+r"(r[28]), "+r"(r[29]), "+r"(r[30]), "+r"(r[31])
               :
               : "memory");
}

// Shared-memory matrix descriptor, K-major, 128-byte swizzle: 8-row atoms of
// 128-byte rows, 1024 bytes apart.
__device__ __forceinline__ uint64_t sw128_desc(uint32_t saddr) {
  return static_cast<uint64_t>((saddr >> 4) & 0x3FFFu) | (static_cast<uint64_t>(1) << 16) |
         (static_cast<uint64_t>(1024 >> 4) << 32) | (static_cast<uint64_t>(1) << 46) | (static_cast<uint64_t>(2) << 61);
}

// Instruction descriptor: f32 sums, both operands K-major.
template <int FMT, int CG>
__device__ __forceinline__ uint32_t mma_idesc(int n) {
  constexpr uint32_t type = FMT == kFmtBF16 ? 1u : 0u;  // f16 kind: 0 f16, 1 bf16; f8f6f4 kind: 0 e4m3
  return (1u << 4) | (type << 7) | (type << 10) | (static_cast<uint32_t>(n >> 3) << 17) |
         (static_cast<uint32_t>(kGemmRows * CG >> 4) << 24);
}

// TMA load into this CTA's shared memory; with a pair the bytes are counted on
// the leader's barrier (`bar` is a shared::cluster address).
template <int CG>
__device__ __forceinline__ void load_tile(void* dst, const CUtensorMap* map, int x, int y, uint32_t bar, uint64_t policy) {
  if constexpr (CG == 2)
    asm volatile(
        "cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes.cta_group::2.L2::cache_hint "
        "[%0], [%1, {%2, %3}], [%4], %5;" ::"r"(smem_u32(dst)), "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y),
        "r"(bar), "l"(policy) : "memory");
  else
    asm volatile(
        "cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes.L2::cache_hint "
        "[%0], [%1, {%2, %3}], [%4], %5;" ::"r"(smem_u32(dst)), "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y),
        "r"(bar), "l"(policy) : "memory");
}

// --------------------------------------------------------------- cluster barriers

__device__ __forceinline__ void mbar_arrive_cluster(uint32_t addr) {
  asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(addr) : "memory");
}
// An arrival that publishes no memory (a tensor-memory buffer has been read,
// which tcgen05.fence orders): release at cluster scope would cost a fence of
// all outstanding stores for every k block (568 -> 415 us at 16384 x 4096 x 4096).
__device__ __forceinline__ void mbar_arrive_remote(uint32_t addr) {
  asm volatile("mbarrier.arrive.shared::cluster.b64 _, [%0];" ::"r"(addr) : "memory");
}
__device__ __forceinline__ bool mbar_try_wait_cluster(uint64_t* bar, uint32_t parity) {
  uint32_t ok;
  asm volatile("{\n\t.reg .pred p;\n\tmbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2;\n\tselp.u32 %0, 1, 0, p;\n\t}"
               : "=r"(ok) : "r"(smem_u32(bar)), "r"(parity) : "memory");
  return ok != 0;
}
// Waits as mbar_wait_bounded does, but inline: a kernel that moves registers
// between its warps (setmaxnreg) makes no calls.
template <bool CLUSTER>
__device__ __forceinline__ bool wait_phase(uint64_t* bar, uint32_t parity, int* status) {
  uint64_t t0 = 0;
  for (uint32_t i = 0;; ++i) {
    if (CLUSTER ? mbar_try_wait_cluster(bar, parity) : mbar_try_wait(bar, parity)) return true;
    if ((i & 31) == 0) {
      const uint64_t now = globaltimer_ns();
      if (t0 == 0) t0 = now;
      if (now - t0 > kWaitLimitNs) {
        atomicOr(status, kStatusWaitTimeout);
        return false;
      }
    }
  }
}

// One lane of a converged warp.
__device__ __forceinline__ bool elect_one() {
  uint32_t ok;
  asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(ok));
  return ok != 0;
}

// --------------------------------------------------------------- tile list

// Tiles of all experts in order: start[e] is the first row of expert e, tile[e]
// its first tile.  start[experts] is the first row of no expert.
struct TileList {
  int* start;
  int* tile;
};

// One warp.  Offsets are cut to [0, rows] and made to rise, so that whatever
// the array holds no tile reaches outside the rows.
__device__ __forceinline__ void build_list(const ExpertGemmArgs& a, TileList l, int tile_rows, int tiles_n, int lane) {
  if (a.offsets == nullptr) {
    if (lane == 0) {
      l.start[0] = 0;
      l.start[1] = a.rows;
      l.tile[0] = 0;
      l.tile[1] = (a.rows + tile_rows - 1) / tile_rows * tiles_n;
    }
    return;
  }
  int row = 0, tile = 0;
  for (int e0 = 0; e0 < a.experts; e0 += 32) {
    const int e = e0 + lane;
    int end = e < a.experts ? min(max(a.offsets[e + 1], row), a.rows) : row;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int up = __shfl_up_sync(0xFFFFFFFFu, end, o);
      if (lane >= o) end = max(end, up);
    }
    int begin = __shfl_up_sync(0xFFFFFFFFu, end, 1);
    if (lane == 0) begin = row;
    const int mine = (end - begin + tile_rows - 1) / tile_rows * tiles_n;
    int sum = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int up = __shfl_up_sync(0xFFFFFFFFu, sum, o);
      if (lane >= o) sum += up;
    }
    if (e < a.experts) {
      l.start[e] = begin;
      l.tile[e] = tile + sum - mine;
    }
    row = __shfl_sync(0xFFFFFFFFu, end, 31);
    tile += __shfl_sync(0xFFFFFFFFu, sum, 31);
  }
  if (lane == 0) {
    l.start[a.experts] = row;
    l.tile[a.experts] = tile;
  }
}

struct Tile {
  int expert, m0, end, n0;
};

// A place in a ring of barriers and the parity of its next phase.
struct Ring {
  int at = 0;
  uint32_t phase = 0;
  __device__ __forceinline__ void next(int size) {
    if (++at == size) {
      at = 0;
      phase ^= 1u;
    }
  }
};

// The t-th tile; `e` only moves forward.
__device__ __forceinline__ Tile find_tile(const TileList& l, int t, int tile_rows, int tiles_n, int bn, int& e) {
  while (t >= l.tile[e + 1]) ++e;
  const int i = t - l.tile[e];
  return Tile{e, l.start[e] + i / tiles_n * tile_rows, l.start[e + 1], i % tiles_n * bn};
}

constexpr int kBoxBytes = kGemmBoxRows * kRowBytes;
__device__ __forceinline__ int row_boxes(int rows) {
  return min(max(rows + kGemmBoxRows - 1, 0) / kGemmBoxRows, kGemmRows / kGemmBoxRows);
}

// --------------------------------------------------------------- epilogue

// 32-byte store of eight words.
__device__ __forceinline__ void store32(void* p, const uint32_t* w) {
  asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(p), "r"(w[0]), "r"(w[1]), "r"(w[2]),
               "r"(w[3]), "r"(w[4]), "r"(w[5]), "r"(w[6]), "r"(w[7]) : "memory");
}

// 64 bytes of each of a warp's 32 rows: through the warp's shared memory
// (16-byte pieces in the 64-byte swizzle, free of bank conflicts) to one tile
// store.  Whole sectors leave the SM in few requests; a store by each lane to
// its own row touches 32 lines an instruction.  Two buffers take turns, so that
// a piece waits for the one before the last.
__device__ __forceinline__ void store_piece(uint8_t* out_s, int& turn, int lane, const uint32_t* w,
                                            const CUtensorMap* ymap, int n, int row) {
  uint8_t* buf = out_s + turn * kStageOut;
  turn ^= 1;
  if (lane == 0) asm volatile("cp.async.bulk.wait_group.read 1;" ::: "memory");
  __syncwarp();
#pragma unroll
  for (int p = 0; p < 4; ++p)
    *reinterpret_cast<uint4*>(buf + lane * kStoreBytes + ((p ^ ((lane >> 1) & 3)) << 4)) =
        make_uint4(w[4 * p], w[4 * p + 1], w[4 * p + 2], w[4 * p + 3]);
  fence_proxy_async_shared();
  __syncwarp();
  if (lane == 0) {
    asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.tile.bulk_group [%0, {%1, %2}], [%3];" ::"l"(
                     reinterpret_cast<uint64_t>(ymap)), "r"(n), "r"(row), "r"(smem_u32(buf)) : "memory");
    asm volatile("cp.async.bulk.commit_group;" ::: "memory");
  }
}

// The same for rows that a tile store cannot take: the last rows of a group,
// or rows of y that are not 16-byte aligned.  From shared memory the warp
// writes row by row, so that its lanes' addresses are next to each other.
// `size`: bytes of a value; `values`: how many of the piece are inside N.
__device__ __forceinline__ void store_piece_by_rows(uint8_t* buf, int lane, const uint32_t* w, uint8_t* y, int64_t pitch,
                                                    int size, int rows, int values, bool aligned) {
  if (lane == 0) asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");
  __syncwarp();
#pragma unroll
  for (int p = 0; p < 4; ++p)
    *reinterpret_cast<uint4*>(buf + lane * kStoreBytes + ((p ^ ((lane >> 1) & 3)) << 4)) =
        make_uint4(w[4 * p], w[4 * p + 1], w[4 * p + 2], w[4 * p + 3]);
  __syncwarp();
  if (aligned && values * size == kStoreBytes) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int r = i * 8 + (lane >> 2), p = lane & 3;
      if (r < rows)
        *reinterpret_cast<uint4*>(y + r * pitch + p * 16) =
            *reinterpret_cast<const uint4*>(buf + r * kStoreBytes + ((p ^ ((r >> 1) & 3)) << 4));
    }
  } else {
    const int per_row = kStoreBytes / size, step = 32 / per_row;  // 32 T or 16 f32 values a row
    const int c = lane % per_row, byte = c * size;
    for (int r = lane / per_row; r < rows; r += step) {
      const uint8_t* from = buf + r * kStoreBytes + ((((byte >> 4) ^ (r >> 1)) & 3) << 4) + (byte & 15);
      if (c < values) {
        if (size == 4) *reinterpret_cast<uint32_t*>(y + r * pitch + byte) = *reinterpret_cast<const uint32_t*>(from);
        else *reinterpret_cast<uint16_t*>(y + r * pitch + byte) = *reinterpret_cast<const uint16_t*>(from);
      }
    }
  }
}

// The four warps of an epilogue group.
__device__ __forceinline__ void group_sync(int half) {
  if (half == 0) asm volatile("bar.sync 1, 128;" ::: "memory");
  else asm volatile("bar.sync 2, 128;" ::: "memory");
}

// --------------------------------------------------------------- kernel

template <int FMT, int DT, int CG, int BN>
__global__ void __launch_bounds__(kThreads, 1)
    expert_gemm_kernel(const __grid_constant__ CUtensorMap xmap, const __grid_constant__ CUtensorMap xmap_part,
                       const __grid_constant__ CUtensorMap wmap,
                       const __grid_constant__ CUtensorMap ymap, const ExpertGemmArgs a) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
  const int S = CG == 2 || BN == 256 ? 1 : a.splits;
  const SmemPlan L = plan_smem(FMT == kFmtE4M3, BN, CG, S, a.experts);
  const int stages = L.stages;
  constexpr int buffers = static_cast<int>(kTmemCols) / BN < kMaxBuffers ? static_cast<int>(kTmemCols) / BN : kMaxBuffers;
  float* part = reinterpret_cast<float*>(smem + L.part_off);
  TileList list{reinterpret_cast<int*>(smem + L.list_off), reinterpret_cast<int*>(smem + L.list_off) + a.experts + 2};
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + L.bar_off);
  uint64_t* empty = full + kMaxStages;
  uint64_t* acc_full = empty + kMaxStages;
  uint64_t* acc_empty = acc_full + kMaxBuffers;
  uint64_t* part_full = acc_empty + kMaxBuffers;
  uint64_t* part_empty = part_full + 1;
  uint64_t* scale_full = part_empty + 1;
  uint64_t* scale_empty = scale_full + kScaleSlots;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(scale_empty + kScaleSlots);
  // [slot][k block][row], then [slot][k block][column half]
  float* scale_x = reinterpret_cast<float*>(smem + L.scale_off);
  float* scale_w = scale_x + kScaleSlots * kScaleBlocks * kGemmRows;
  __shared__ __align__(16) float bias_s[256];

  // the same in all lanes, and known to be
  const int warp = __shfl_sync(0xFFFFFFFFu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  const int rank = CG == 2 || S > 1 ? static_cast<int>(cluster_ctarank()) : 0;
  const int worker = blockIdx.x / (CG * S), workers = gridDim.x / (CG * S);
  const int tile_rows = kGemmRows * CG, tiles_n = (a.N + BN - 1) / BN;
  constexpr int kElems = FMT == kFmtE4M3 ? 128 : 64;  // values of a k block
  const int KB = (a.K + kElems - 1) / kElems;
  const int per = (KB + S - 1) / S;
  const int kb0 = CG == 2 ? 0 : rank * per, kb1 = min(KB, kb0 + per);  // every slice holds a block (host)

  if (threadIdx.x == 0) {
    prefetch_tensormap(&xmap);
    prefetch_tensormap(&xmap_part);
    prefetch_tensormap(&wmap);
    prefetch_tensormap(&ymap);
    for (int s = 0; s < kMaxStages; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    for (int b = 0; b < kMaxBuffers; ++b) {
      mbar_init(&acc_full[b], 1);
      mbar_init(&acc_empty[b], CG * kEpiWarps);
    }
    mbar_init(part_full, S * kEpiWarps);
    mbar_init(part_empty, S * kEpiWarps);
    for (int b = 0; b < kScaleSlots; ++b) {
      mbar_init(&scale_full[b], 32);
      mbar_init(&scale_empty[b], kEpiWarps);
    }
    fence_mbar_init();
  }
  if (warp == 2) tmem_alloc<CG>(tmem_slot, kTmemCols);
  pdl_launch_dependents();
  pdl_wait();  // offsets, rows and scales are other kernels' results
  if (warp == 3) build_list(a, list, tile_rows, tiles_n, lane);
  tc_fence_before();
  __syncthreads();
  if (CG == 2 || S > 1) cluster_sync_all();  // barriers of the other CTAs are ready
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  const int groups = a.offsets == nullptr ? 1 : a.experts;
  const int total = list.tile[groups];
  bool ok = true;

  if (warp < 4) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 72;");
    if (warp == 0) {
      // ---------------------------------------------------------- copies
      const uint64_t keep = l2_policy_evict_normal();
      int e = 0, issued = 0;
      Ring ring;
      for (int t = worker; t < total && ok; t += workers) {
        const Tile tile = find_tile(list, t, tile_rows, tiles_n, BN, e);
        // only the rows that there are, by 32: a small group's tile is mostly weights
        const int m = tile.m0 + (CG == 2 ? rank * kGemmRows : 0);
        const int boxes = row_boxes(tile.end - m);
        const int all_boxes = CG == 2 ? row_boxes(tile.end - tile.m0) + row_boxes(tile.end - tile.m0 - kGemmRows) : boxes;
        const uint32_t bytes = static_cast<uint32_t>(all_boxes * kBoxBytes + BN * kRowBytes);
        const int w = tile.expert * a.N + tile.n0 + (CG == 2 ? rank * (BN / 2) : 0);
        for (int kb = kb0; kb < kb1; ++kb) {
          if (!wait_phase<false>(&empty[ring.at], ring.phase ^ 1u, a.status)) {
            ok = false;
            break;
          }
          uint8_t* st = smem + ring.at * L.stage_bytes;
          uint32_t bar = smem_u32(&full[ring.at]);
          if (CG == 2) bar = mapa_shared(bar, 0);
          if (elect_one()) {
            if (rank == 0 || CG == 1) mbar_arrive_expect_tx(&full[ring.at], bytes);
            if (boxes == kGemmRows / kGemmBoxRows) {
              load_tile<CG>(st, &xmap, kb * kElems, m, bar, keep);
            } else {
              for (int b = 0; b < boxes; ++b)
                load_tile<CG>(st + b * kBoxBytes, &xmap_part, kb * kElems, m + b * kGemmBoxRows, bar, keep);
            }
            load_tile<CG>(st + kXBytes, &wmap, kb * kElems, w, bar, keep);
          }
          __syncwarp();
          ring.next(stages);
          ++issued;
        }
      }
      if (!ok && (rank == 0 || CG == 1))  // a wait ran out: let the copies in flight land before the CTA ends
        for (int i = max(0, issued - stages); i < issued; ++i) wait_phase<false>(&full[i % stages], (i / stages) & 1, a.status);
    } else if (warp == 1 && (CG == 1 || rank == 0)) {
      // ---------------------------------------------------------- products
      const uint32_t idesc = mma_idesc<FMT, CG>(BN);
      // The tensor pipe queues few products, so this loop's scalar work has to
      // fit under four of them: the whole warp runs it, with values that are
      // the same in all lanes, and one lane issues; ring places by counters,
      // descriptors by adds (every address field stays below 2^14).
      const uint64_t base = sw128_desc(smem_u32(smem));
      const uint32_t stage_units = static_cast<uint32_t>(L.stage_bytes) >> 4;
      Ring ring, acc;
      for (int t = worker; t < total && ok; t += workers) {
        for (int kb = kb0; kb < kb1; ++kb) {
          const bool first = FMT == kFmtE4M3 || kb == kb0, last = FMT == kFmtE4M3 || kb == kb1 - 1;
          if (first) ok = wait_phase<false>(&acc_empty[acc.at], acc.phase ^ 1u, a.status);
          ok = ok && wait_phase<false>(&full[ring.at], ring.phase, a.status);
          if (!ok) break;
          tc_fence_after();
          const uint64_t da = base + ring.at * stage_units;
          const uint64_t db = da + (kXBytes >> 4);
          const uint32_t d = tmem + static_cast<uint32_t>(acc.at * BN);
          if (elect_one()) {
            tc_mma<FMT, CG>(d, da, db, idesc, !first);
            tc_mma<FMT, CG>(d, da + 2, db + 2, idesc, 1);
            tc_mma<FMT, CG>(d, da + 4, db + 4, idesc, 1);
            tc_mma<FMT, CG>(d, da + 6, db + 6, idesc, 1);
            tc_commit<CG>(&empty[ring.at]);
            if (last) tc_commit<CG>(&acc_full[acc.at]);
          }
          __syncwarp();
          ring.next(stages);
          if (last) acc.next(buffers);
        }
      }
    } else if (FMT == kFmtE4M3 && warp == 3) {
      // ---------------------------------------------------------- scales
      const int NBLK = (a.N + kFp8Block - 1) / kFp8Block;
      int e = 0;
      Ring ring;
      for (int t = worker; t < total && ok; t += workers) {
        const Tile tile = find_tile(list, t, tile_rows, tiles_n, BN, e);
        const int row0 = tile.m0 + (CG == 2 ? rank * kGemmRows : 0) + lane;
        const float* sw = a.w_scales + static_cast<int64_t>(tile.expert) * NBLK * KB;
        const int blk0 = min(tile.n0 / kFp8Block, NBLK - 1), blk1 = min((tile.n0 + BN / 2) / kFp8Block, NBLK - 1);
        for (int kb = kb0; kb < kb1; kb += kScaleBlocks) {
          ok = wait_phase<false>(&scale_empty[ring.at], ring.phase ^ 1u, a.status);
          if (!ok) break;
          float v[kScaleBlocks][4];
#pragma unroll
          for (int i = 0; i < kScaleBlocks; ++i) {
            const int k = min(kb + i, kb1 - 1);
#pragma unroll
            for (int j = 0; j < 4; ++j)
              v[i][j] = __ldg(a.x_scales + static_cast<int64_t>(k) * a.rows + min(row0 + 32 * j, a.rows - 1));
          }
          float* sx = scale_x + ring.at * kScaleBlocks * kGemmRows + lane;
          if (lane < 2 * kScaleBlocks)
            scale_w[ring.at * 2 * kScaleBlocks + lane] =
                __ldg(sw + static_cast<int64_t>(lane & 1 ? blk1 : blk0) * KB + min(kb + (lane >> 1), kb1 - 1));
#pragma unroll
          for (int i = 0; i < kScaleBlocks; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j) sx[i * kGemmRows + 32 * j] = v[i][j];
          mbar_arrive(&scale_full[ring.at]);
          ring.next(kScaleSlots);
        }
      }
    }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 216;");
    // ------------------------------------------------------------ epilogue
    const int quarter = warp & 3, half = (warp - kEpiWarp0) >> 2;
    constexpr int W = BN / 2;  // columns of this warp group
    const uint32_t lane_base = tmem + (static_cast<uint32_t>(quarter * 32) << 16) + static_cast<uint32_t>(half * W);
    const uint32_t acc_empty0 = CG == 2 ? mapa_shared(smem_u32(acc_empty), 0) : smem_u32(acc_empty);
    const int local = quarter * 32 + lane;  // row of the tile's 128
    uint8_t* out_s = smem + L.out_off + (warp - kEpiWarp0) * 2 * kStageOut;
    int turn_out = 0;

    // rows of no expert are zeros
    if (a.out != kOutCodes) {
      const int size = a.out == kOutF32 ? 4 : 2;
      for (int64_t r = list.start[groups] + static_cast<int64_t>(blockIdx.x); r < a.rows; r += gridDim.x) {
        char* p = reinterpret_cast<char*>(a.y) + r * a.ldy * size;
        for (int i = threadIdx.x - kEpiWarp0 * 32; i < a.N; i += kEpiThreads) {
          if (size == 4) reinterpret_cast<float*>(p)[i] = 0.0f;
          else reinterpret_cast<uint16_t*>(p)[i] = 0;
        }
      }
    }

    int e = 0, turn = 0;
    Ring ring, scales;
    for (int t = worker; t < total && ok; t += workers, ++turn) {
      const Tile tile = find_tile(list, t, tile_rows, tiles_n, BN, e);
      const int64_t row = tile.m0 + (CG == 2 ? rank * kGemmRows : 0) + local;
      const bool live = row < tile.end;
      const int row_w = tile.m0 + (CG == 2 ? rank * kGemmRows : 0) + quarter * 32;  // the warp's first row
      const bool idle = row_w >= tile.end;  // a warp without rows only hands buffers back
      const int n0 = tile.n0 + half * W;
      float acc[W];
#pragma unroll
      for (int i = 0; i < W; ++i) acc[i] = 0.0f;
      if (a.bias != nullptr) {
        // the group's columns of the bias, one a thread
        group_sync(half);  // the tile before has been read
        if (local < W) {
          const int n = n0 + local;
          bias_s[half * 128 + local] = n < a.N ? ld_t<DT>(a.bias, static_cast<int64_t>(tile.expert) * a.N + n) : 0.0f;
        }
        group_sync(half);
      }

      if constexpr (FMT == kFmtE4M3) {
        for (int kb = kb0; kb < kb1; kb += kScaleBlocks) {
          ok = ok && wait_phase<false>(&scale_full[scales.at], scales.phase, a.status);
          const float* sx = scale_x + scales.at * kScaleBlocks * kGemmRows + local;
          const float* sw = scale_w + scales.at * 2 * kScaleBlocks + half;
          const int blocks = min(kScaleBlocks, kb1 - kb);
#pragma unroll 1
          for (int i = 0; i < blocks; ++i) {
            ok = ok && wait_phase<false>(&acc_full[ring.at], ring.phase, a.status);
            tc_fence_after();
            const uint32_t src = lane_base + static_cast<uint32_t>(ring.at * BN);
            if (idle) {
              if (lane == 0) mbar_arrive_remote(acc_empty0 + ring.at * 8);
              ring.next(buffers);
              continue;
            }
            // the next columns are on their way while these are added
            uint32_t r[2][32];
            tmem_ld32(src, r[0]);
            const float scale = sx[i * kGemmRows] * sw[2 * i];
#pragma unroll
            for (int c = 0; c < W; c += 32) {
              tmem_wait_ld(r[(c / 32) & 1]);
              if (c + 32 < W) {
                tmem_ld32(src + c + 32, r[(c / 32 + 1) & 1]);
              } else {
                // all read: the buffer goes back before the last sums
                tc_fence_before();
                if (lane == 0) mbar_arrive_remote(acc_empty0 + ring.at * 8);
              }
              const uint32_t(&v)[32] = r[(c / 32) & 1];
#pragma unroll
              for (int j = 0; j < 32; j += 2) fma2(acc[c + j], acc[c + j + 1], v[j], v[j + 1], scale);
            }
            ring.next(buffers);
          }
          __syncwarp();
          if (lane == 0) mbar_arrive(&scale_empty[scales.at]);
          scales.next(kScaleSlots);
        }
      } else {
        ok = ok && wait_phase<false>(&acc_full[ring.at], ring.phase, a.status);
        tc_fence_after();
        const uint32_t src = lane_base + static_cast<uint32_t>(ring.at * BN);
#pragma unroll
        for (int c = 0; c < W; c += 32) {
          if (idle) break;
          uint32_t r[32];
          tmem_ld32(src + c, r);
          tmem_wait_ld(r);
#pragma unroll
          for (int j = 0; j < 32; ++j) acc[c + j] = __uint_as_float(r[j]);
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive_remote(acc_empty0 + ring.at * 8);
        ring.next(buffers);
      }
      if (!ok) break;

      if (S > 1) {
        // each CTA of the cluster parks its sums [column][row], then finishes
        // its share of the columns over all CTAs' sums, in rank order
        ok = wait_phase<true>(part_empty, (turn & 1) ^ 1, a.status);
#pragma unroll
        for (int c = 0; c < W; ++c) part[(half * W + c) * kGemmRows + local] = acc[c];
        __syncwarp();
        if (lane < S) mbar_arrive_cluster(mapa_shared(smem_u32(part_full), lane));
        ok = wait_phase<true>(part_full, turn & 1, a.status) && ok;
        const int mine = BN / S / 2, c0 = rank * (BN / S) + half * mine;
        for (int c = c0; c < c0 + mine; c += 4) {
          float v[4] = {};
          for (int r = 0; r < S; ++r) {
            const uint32_t from = mapa_shared(smem_u32(part), r);
#pragma unroll
            for (int j = 0; j < 4; ++j) v[j] += ld_dsmem_f32(from + static_cast<uint32_t>((c + j) * kGemmRows + local) * 4u);
          }
          if (live) {
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              const int n = tile.n0 + c + j;
              if (n < a.N) {
                float o = v[j];
                if (a.bias != nullptr) o += ld_t<DT>(a.bias, static_cast<int64_t>(tile.expert) * a.N + n);
                o = activate(o, a.act);
                if (a.out == kOutF32) st_t<kF32>(a.y, row * a.ldy + n, o);
                else st_t<DT>(a.y, row * a.ldy + n, o);
              }
            }
          }
        }
        __syncwarp();
        if (lane < S) mbar_arrive_cluster(mapa_shared(smem_u32(part_empty), lane));
        continue;
      }
      if (idle) continue;
#pragma unroll
      for (int c = 0; c < W; c += 32) {
        if (a.bias != nullptr) {
          const float4* b4 = reinterpret_cast<const float4*>(bias_s + half * 128 + c);
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            const float4 b = b4[j];
            acc[c + 4 * j] += b.x, acc[c + 4 * j + 1] += b.y, acc[c + 4 * j + 2] += b.z, acc[c + 4 * j + 3] += b.w;
          }
        }
        if (a.act != kActNone) {
#pragma unroll
          for (int j = 0; j < 32; j += 2) activate2(acc[c + j], acc[c + j + 1], a.act);
        }
      }
      const bool whole = a.tile_store && row_w + 32 <= tile.end;
      if constexpr (BN == 256 && FMT == kFmtE4M3) {
        if (a.out == kOutCodes) {
          // the thread's 128 columns are one block of its row
          if (n0 >= a.N) continue;
          if (n0 + W > a.N) {
#pragma unroll
            for (int i = 0; i < W; ++i) acc[i] = n0 + i < a.N ? acc[i] : 0.0f;
          }
          uint32_t top = 0;
#pragma unroll
          for (int i = 0; i < W; ++i) top = max(top, __float_as_uint(acc[i]) & 0x7FFFFFFFu);
          int ex = fp8_scale_exponent(top);
          if (top >= 0x7F800000u) {
            // not all finite: the scale comes from those that are, the others become NaN
            top = 0;
#pragma unroll
            for (int i = 0; i < W; ++i) {
              const uint32_t m = finite_magnitude(acc[i]);
              top = max(top, m);
              if (m == 0 && acc[i] != 0.0f) acc[i] = __uint_as_float(0x7FC00000u);
            }
            ex = fp8_scale_exponent(top);
          }
          const float inv = pow2f(-ex);
          if (live) a.y_scales[static_cast<int64_t>(n0 / kFp8Block) * a.rows + row] = pow2f(ex);
          // rows of codes are padded to whole blocks
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            uint32_t w[16];
#pragma unroll
            for (int i = 0; i < 16; ++i) {
              const float* v = acc + 64 * h + 4 * i;
              w[i] = e4m3x2_finite(v[0] * inv, v[1] * inv) | (e4m3x2_finite(v[2] * inv, v[3] * inv) << 16);
            }
            if (whole) {
              store_piece(out_s, turn_out, lane, w, &ymap, n0 + 64 * h, row_w);
            } else if (live) {
              uint8_t* p = reinterpret_cast<uint8_t*>(a.y) + row * a.ldy + n0 + 64 * h;
              store32(p, w);
              store32(p + 32, w + 8);
            }
          }
          continue;
        }
      }
      const int rows_w = min(32, tile.end - row_w);
      const int size = a.out == kOutF32 ? 4 : 2;
#pragma unroll
      for (int c = 0; c < W; c += 16) {
        // 64 bytes: 16 f32 values, or 32 of T
        if (n0 + c >= a.N) break;
        uint32_t w[16];
        if (a.out == kOutF32) {
#pragma unroll
          for (int i = 0; i < 16; ++i) w[i] = __float_as_uint(acc[c + i]);
        } else {
          if (c % 32 != 0) continue;
#pragma unroll
          for (int i = 0; i < 16; ++i) w[i] = pack_t<DT>(acc[(c + 2 * i) % W], acc[(c + 2 * i + 1) % W]);
        }
        if (whole) {
          store_piece(out_s, turn_out, lane, w, &ymap, n0 + c, row_w);
        } else {
          store_piece_by_rows(out_s, lane, w, reinterpret_cast<uint8_t*>(a.y) + (row_w * a.ldy + n0 + c) * size,
                              a.ldy * size, size, rows_w, min(kStoreBytes / size, a.N - n0 - c), a.tile_store != 0);
        }
      }
    }
    // the tile stores have read their shared memory
    asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");
  }

  __syncwarp();
  tc_fence_before();
  __syncthreads();
  if (CG == 2 || S > 1) cluster_sync_all();  // no CTA ends while another reads or signals its memory
  if (warp == 2) {
    tc_fence_after();
    tmem_release<CG>(tmem, kTmemCols);
  }
}

template <int FMT, int DT, int CG, int BN>
cudaError_t launch_typed(const CUtensorMap& xmap, const CUtensorMap& xmap_part, const CUtensorMap& wmap, const CUtensorMap& ymap, const ExpertGemmArgs& a, int num_sms,
                         cudaStream_t stream, bool pdl) {
  auto kernel = expert_gemm_kernel<FMT, DT, CG, BN>;
  static SharedMemoryOptIn opt_in;
  const cudaError_t configured = opt_in.ensure(reinterpret_cast<const void*>(kernel), kSmemLimit - 1024);
  if (configured != cudaSuccess) return configured;
  const SmemPlan p = plan_smem(FMT == kFmtE4M3, BN, CG, a.splits, a.experts);
  const int cluster = CG * a.splits;
  // at most one tile list per cluster; no more clusters than tiles there can be
  const int64_t tile_rows = kGemmRows * CG;
  const int64_t groups = a.offsets == nullptr ? 1 : std::min(a.experts, a.rows);
  const int64_t tiles = ((a.rows + tile_rows - 1) / tile_rows + groups) * ((a.N + BN - 1) / BN);
  const int clusters = static_cast<int>(std::min<int64_t>(tiles, num_sms / cluster));
  return launch_clustered(kernel, dim3(clusters * cluster), dim3(kThreads), p.bytes, stream, pdl, cluster, xmap, xmap_part, wmap, ymap, a);
}

template <int FMT, int DT>
cudaError_t launch_config(const ExpertGemmConfig& cfg, const CUtensorMap& xmap, const CUtensorMap& xmap_part,
                          const CUtensorMap& wmap, const CUtensorMap& ymap, const ExpertGemmArgs& a, int num_sms, cudaStream_t stream, bool pdl) {
  if (cfg.pair == 2) return launch_typed<FMT, DT, 2, 256>(xmap, xmap_part, wmap, ymap, a, num_sms, stream, pdl);
  if (cfg.bn == 256) return launch_typed<FMT, DT, 1, 256>(xmap, xmap_part, wmap, ymap, a, num_sms, stream, pdl);
  if (cfg.bn == 128) return launch_typed<FMT, DT, 1, 128>(xmap, xmap_part, wmap, ymap, a, num_sms, stream, pdl);
  return launch_typed<FMT, DT, 1, 64>(xmap, xmap_part, wmap, ymap, a, num_sms, stream, pdl);
}

}  // namespace

cudaError_t launch_expert_gemm(int dtype, bool e4m3, const CUtensorMap& xmap, const CUtensorMap& xmap_part,
                               const CUtensorMap& wmap, const CUtensorMap& ymap, const ExpertGemmConfig& cfg, ExpertGemmArgs a, int num_sms, cudaStream_t stream,
                               bool pdl) {
  a.splits = cfg.splits;
  const int KB = (a.K + (e4m3 ? 127 : 63)) / (e4m3 ? 128 : 64);
  const bool pair = cfg.pair == 2;
  if (cfg.bn != 64 && cfg.bn != 128 && cfg.bn != 256) return cudaErrorInvalidValue;
  if (cfg.splits != 1 && cfg.splits != 2 && cfg.splits != 4 && cfg.splits != 8) return cudaErrorInvalidValue;
  if (cfg.splits > 1 && (pair || cfg.bn > 128 || a.out == kOutCodes)) return cudaErrorInvalidValue;
  if ((cfg.splits - 1) * ((KB + cfg.splits - 1) / cfg.splits) >= KB) return cudaErrorInvalidValue;
  if (pair && cfg.bn != 256) return cudaErrorInvalidValue;
  if (e4m3)
    return dtype == kF16 ? launch_config<kFmtE4M3, kF16>(cfg, xmap, xmap_part, wmap, ymap, a, num_sms, stream, pdl)
                         : launch_config<kFmtE4M3, kBF16>(cfg, xmap, xmap_part, wmap, ymap, a, num_sms, stream, pdl);
  return dtype == kF16 ? launch_config<kFmtF16, kF16>(cfg, xmap, xmap_part, wmap, ymap, a, num_sms, stream, pdl)
                       : launch_config<kFmtBF16, kBF16>(cfg, xmap, xmap_part, wmap, ymap, a, num_sms, stream, pdl);
}

ExpertGemmConfig plan_expert_gemm(bool e4m3, int rows, int experts, int N, int K, bool codes_out, int num_sms) {
  const int KB = (K + (e4m3 ? 127 : 63)) / (e4m3 ? 128 : 64);
  const int groups = std::min(experts, rows);
  const auto tiles = [&](int tile_rows, int bn) {
    // a group of the mean size; ragged groups have about half a tile more
    const int64_t mean = rows / groups;
    return static_cast<int64_t>(groups) * ((mean + tile_rows - 1) / tile_rows) * ((N + bn - 1) / bn);
  };
  if (rows / groups >= 512 && tiles(256, 256) * 2 >= num_sms) return {2, 256, 1};
  if (codes_out || tiles(128, 256) >= num_sms) return {1, 256, 1};
  const int bn = tiles(128, 128) >= num_sms ? 128 : 64;
  int splits = 1;
  for (int s : {2, 4, 8})
    if (tiles(128, bn) * s <= num_sms && (KB + s - 1) / s >= 8 && (s - 1) * ((KB + s - 1) / s) < KB) splits = s;
  return {1, bn, splits};
}

}  // namespace cq
