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
// the epilogue of a tile overlaps the next tile's products.  Rows of x that come
// as the sum of two 16-bit parts (h of the feed-forward module) meet each k block
// of the weights twice; narrow tiles have both parts in one stage, with one copy
// of the weights.
//
// Wide tiles are bound by the copies from L2: a 128 x 256 tile takes 48 KB a k
// block, 1100 cycles at the rate that all SMs have together.
//
// Persistent: a CTA takes every W-th tile of all experts' tiles; the
// tile list follows from the offsets, which only the device knows.
//   warps 0, 2  copy tiles of x and of W (TMA, 128-byte swizzle) into a ring
//   warp 1      issues tcgen05.mma
//               (warp 2 also owns the tensor memory)
//   warp 3      e4m3: fetches the scales, eight k blocks ahead
//   warps 4-    epilogue: one set of eight warps or two, in a set two groups of
//               four warps, each half of the columns
#include "expert_gemm.hpp"

#include <algorithm>
#include <cmath>

#include "fp8.cuh"
#include "launch.hpp"

namespace cq {

namespace {

constexpr int kEpiWarp0 = 4, kSetWarps = 8;
// Sets of eight epilogue warps.  Narrow tiles have two that take turns, so that
// one set's last pass over a tile (activation, rounding or codes, stores) runs
// beside the other's sums of the next tile: with one set that pass took as long
// as the copies of a whole tile.
__host__ __device__ constexpr int epi_sets(int bn) { return bn < 256 ? 2 : 1; }
__host__ __device__ constexpr int gemm_threads(int bn) { return (kEpiWarp0 + kSetWarps * epi_sets(bn)) * 32; }
constexpr int kRowBytes = 128;                       // a k block of one row
constexpr int kXBytes = kGemmRows * kRowBytes;       // a stage's rows of x
constexpr int kMaxStages = 8;
constexpr uint32_t kTmemCols = 512;
constexpr int kSmemLimit = 227 * 1024;
constexpr int kGroups = 2;  // of tensor-memory accumulators
constexpr int kGroupCols = static_cast<int>(kTmemCols) / kGroups;

enum Format : int { kFmtE4M3 = 0, kFmtF16 = 1, kFmtBF16 = 2 };

constexpr int kScaleBlocks = 8;  // k blocks of scales fetched at a time
constexpr int kScaleSlots = 2;
constexpr int kScaleBytes = kScaleBlocks * (kGemmRows + 2) * 4;
constexpr int kStageOut = kStoreRows * kStoreBytes;  // a warp's tile store
constexpr int kStageOuts = 16;                        // two for each of one set's warps, one for each of two sets'

// k blocks of one stage: two where a block's products are so short that the
// waits and signals of a stage would outlast them.
__host__ __device__ constexpr int stage_blocks(int bn) { return bn < 256 ? 2 : 1; }

constexpr int kStaticBytes = 1024 + 4096;  // the bias, and the largest magnitudes of a block's halves

struct SmemPlan {
  int stage_bytes, stages, out_off, scale_off, list_off, bar_off, bytes;
};

__host__ __device__ inline SmemPlan plan_smem(bool e4m3, int bn, int experts) {
  SmemPlan p{};
  p.stage_bytes = stage_blocks(bn) * (kXBytes + bn * kRowBytes);
  const int list = (2 * (experts + 2) * 4 + 15) / 16 * 16;
  const int bars = (2 * kMaxStages + 2 * kGroups + 2 * kScaleSlots + 2) * 8 + 16;
  const int scales = e4m3 ? kScaleSlots * kScaleBytes : 0;
  const int rest = kStageOuts * kStageOut + scales + list + bars;
  p.stages = (kSmemLimit - kStaticBytes - 1024 - rest) / p.stage_bytes;  // 1024: alignment
  if (p.stages > kMaxStages) p.stages = kMaxStages;
  p.out_off = p.stages * p.stage_bytes;
  p.scale_off = p.out_off + kStageOuts * kStageOut;
  p.list_off = p.scale_off + scales;
  p.bar_off = p.list_off + list;
  p.bytes = p.bar_off + bars + 1024;  // + alignment
  return p;
}

// --------------------------------------------------------------- tcgen05

__device__ __forceinline__ void tmem_alloc(uint32_t* dst, uint32_t cols) {
  asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(dst)), "r"(cols) : "memory");
  asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
}
__device__ __forceinline__ void tmem_release(uint32_t taddr, uint32_t cols) {
  asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(taddr), "r"(cols) : "memory");
}

__device__ __forceinline__ void tc_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }

template <int FMT>
__device__ __forceinline__ void tc_mma(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
  if constexpr (FMT == kFmtE4M3)
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\ttcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}" ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(accumulate) : "memory");
  else
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\ttcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(accumulate) : "memory");
}

// Arrives on the barrier at `bar` when the MMAs issued so far are done.
__device__ __forceinline__ void tc_commit(uint32_t bar) {
  asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar) : "memory");
}

// 32 lanes x 32 (or 16) columns: thread i of the warp gets its lane's columns.
__device__ __forceinline__ void tmem_ld(uint32_t taddr, uint32_t (&r)[32]) {
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
__device__ __forceinline__ void tmem_ld(uint32_t taddr, uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(taddr)
      : "memory");
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

__device__ __forceinline__ void tmem_wait_ld(uint32_t (&r)[16]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]),
                 "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15])
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
template <int FMT>
__device__ __forceinline__ uint32_t mma_idesc(int n) {
  constexpr uint32_t type = FMT == kFmtBF16 ? 1u : 0u;  // f16 kind: 0 f16, 1 bf16; f8f6f4 kind: 0 e4m3
  return (1u << 4) | (type << 7) | (type << 10) | (static_cast<uint32_t>(n >> 3) << 17) |
         (static_cast<uint32_t>(kGemmRows >> 4) << 24);
}

// TMA load into this CTA's shared memory, counted on the barrier at `bar`.
__device__ __forceinline__ void load_tile(uint32_t dst, const CUtensorMap* map, int x, int y, uint32_t bar, uint64_t policy) {
  asm volatile(
      "cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes.L2::cache_hint "
      "[%0], [%1, {%2, %3}], [%4], %5;" ::"r"(dst), "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(bar),
      "l"(policy) : "memory");
}

__device__ __forceinline__ void load_tile(uint32_t dst, const CUtensorMap* map, int x, int y, int z, uint32_t bar,
                                          uint64_t policy) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes.L2::cache_hint "
      "[%0], [%1, {%2, %3, %4}], [%5], %6;" ::"r"(dst), "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(z),
      "r"(bar), "l"(policy) : "memory");
}

// --------------------------------------------------------------- barriers

// Barriers go by their shared-memory addresses: the loops that issue copies and
// products have a few hundred cycles a turn, and address arithmetic counts.
__device__ __forceinline__ void arrive(uint32_t bar) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ void arrive_expect(uint32_t bar, uint32_t bytes) {
  asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(bytes) : "memory");
}

// Tests a phase, asleep for up to kSuspendNs until it completes: without the
// hint a waiting warp polls, and the polls of a CTA's waiting warps hold up
// the shared-memory instructions of the ones at work.
constexpr uint32_t kSuspendNs = 20000;
__device__ __forceinline__ bool phase_done(uint32_t bar, uint32_t parity) {
  uint32_t ok;
  asm volatile("{\n\t.reg .pred p;\n\tmbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2, %3;\n\tselp.u32 %0, 1, 0, p;\n\t}"
               : "=r"(ok) : "r"(bar), "r"(parity), "r"(kSuspendNs) : "memory");
  return ok != 0;
}

// Waits as mbar_wait_bounded does, but inline: a kernel that moves registers
// between its warps (setmaxnreg) makes no calls.
__device__ __forceinline__ bool wait_phase(uint32_t bar, uint32_t parity, int* status) {
  if (phase_done(bar, parity)) return true;
  const uint64_t t0 = globaltimer_ns();
  while (!phase_done(bar, parity)) {
    if (globaltimer_ns() - t0 > kWaitLimitNs) {
      atomicOr(status, kStatusWaitTimeout);
      return false;
    }
  }
  return true;
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
    int end = e < a.experts ? min(max(__ldcg(a.offsets + e + 1), row), a.rows) : row;
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
  Ring() = default;
  // after `used` places
  __device__ __forceinline__ Ring(int used, int size) : at(used % size), phase((used / size) & 1) {}
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
// its own row touches 32 lines an instruction.  Where there are two buffers they
// take turns, and a piece waits for the one before the last.  `PARTS`: y's map
// has parts, of which this is one's.
template <int BUFFERS, bool PARTS>
__device__ __forceinline__ void store_piece(uint8_t* out_s, int& turn, int lane, const uint32_t* w,
                                            const CUtensorMap* ymap, int n, int row, int part) {
  uint8_t* buf = out_s + turn * kStageOut;
  if constexpr (BUFFERS == 2) {
    turn ^= 1;
    if (lane == 0) asm volatile("cp.async.bulk.wait_group.read 1;" ::: "memory");
  } else {
    if (lane == 0) asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");
  }
  __syncwarp();
#pragma unroll
  for (int p = 0; p < 4; ++p)
    *reinterpret_cast<uint4*>(buf + lane * kStoreBytes + ((p ^ ((lane >> 1) & 3)) << 4)) =
        make_uint4(w[4 * p], w[4 * p + 1], w[4 * p + 2], w[4 * p + 3]);
  fence_proxy_async_shared();
  __syncwarp();
  if (lane == 0) {
    if constexpr (PARTS)
      asm volatile("cp.async.bulk.tensor.3d.global.shared::cta.tile.bulk_group [%0, {%1, %2, %3}], [%4];" ::"l"(
                       reinterpret_cast<uint64_t>(ymap)), "r"(n), "r"(row), "r"(part), "r"(smem_u32(buf)) : "memory");
    else
      asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.tile.bulk_group [%0, {%1, %2}], [%3];" ::"l"(
                       reinterpret_cast<uint64_t>(ymap)), "r"(n), "r"(row), "r"(smem_u32(buf)) : "memory");
    asm volatile("cp.async.bulk.commit_group;" ::: "memory");
  }
}

// The same for the last rows of a group, which a tile store would write past:
// each lane stores its own row.
__device__ __forceinline__ void store_piece_by_lanes(const uint32_t* w, uint8_t* row) {
  if ((reinterpret_cast<uintptr_t>(row) & 31) == 0) {
    store32(row, w);
    store32(row + 32, w + 8);
  } else {
#pragma unroll
    for (int p = 0; p < 4; ++p)
      *reinterpret_cast<uint4*>(row + 16 * p) = make_uint4(w[4 * p], w[4 * p + 1], w[4 * p + 2], w[4 * p + 3]);
  }
}

// The same for rows of y that are not 16-byte aligned, or the last columns of a
// group's last rows: from shared memory the warp writes row by row, so that its
// lanes' addresses are next to each other.  `size`: bytes of a value; `values`:
// how many of the piece are inside N.
__device__ __forceinline__ void store_piece_by_rows(uint8_t* buf, int lane, const uint32_t* w, uint8_t* y, int64_t pitch,
                                                    int size, int rows, int values) {
  if (lane == 0) asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");
  __syncwarp();
#pragma unroll
  for (int p = 0; p < 4; ++p)
    *reinterpret_cast<uint4*>(buf + lane * kStoreBytes + ((p ^ ((lane >> 1) & 3)) << 4)) =
        make_uint4(w[4 * p], w[4 * p + 1], w[4 * p + 2], w[4 * p + 3]);
  __syncwarp();
  const int per_row = kStoreBytes / size, step = 32 / per_row;  // 32 T or 16 f32 values a row
  const int c = lane % per_row, byte = c * size;
  if (c >= values) rows = 0;
  uint8_t* to = y + byte;
  if (size == 4) {
#pragma unroll 8
    for (int r = lane / per_row; r < rows; r += step)
      *reinterpret_cast<uint32_t*>(to + r * pitch) =
          *reinterpret_cast<const uint32_t*>(buf + r * kStoreBytes + ((((byte >> 4) ^ (r >> 1)) & 3) << 4) + (byte & 15));
  } else {
#pragma unroll 8
    for (int r = lane / per_row; r < rows; r += step)
      *reinterpret_cast<uint16_t*>(to + r * pitch) =
          *reinterpret_cast<const uint16_t*>(buf + r * kStoreBytes + ((((byte >> 4) ^ (r >> 1)) & 3) << 4) + (byte & 15));
  }
  __syncwarp();
}

// The four warps of an epilogue group, and the eight of a set.
__device__ __forceinline__ void group_sync(int group) {
  if (group == 0) asm volatile("bar.sync 1, 128;" ::: "memory");
  else if (group == 1) asm volatile("bar.sync 2, 128;" ::: "memory");
  else if (group == 2) asm volatile("bar.sync 3, 128;" ::: "memory");
  else asm volatile("bar.sync 4, 128;" ::: "memory");
}
__device__ __forceinline__ void set_sync(int set) {
  if (set == 0) asm volatile("bar.sync 5, 256;" ::: "memory");
  else asm volatile("bar.sync 6, 256;" ::: "memory");
}

// --------------------------------------------------------------- kernel

template <int FMT, int DT, int BN>
__global__ void __launch_bounds__(gemm_threads(BN), 1)
    expert_gemm_kernel(const __grid_constant__ CUtensorMap xmap, const __grid_constant__ CUtensorMap xmap_part,
                       const __grid_constant__ CUtensorMap wmap,
                       const __grid_constant__ CUtensorMap ymap, const ExpertGemmArgs a) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
  const SmemPlan L = plan_smem(FMT == kFmtE4M3, BN, a.experts);
  const int stages = L.stages;
  // Tensor memory is two groups of accumulators that go back and forth between
  // the products and the epilogue: of kPer k blocks' partial sums each (e4m3),
  // or of one tile's sums.
  constexpr int kSets = epi_sets(BN), kEpiThreads = kSets * kSetWarps * 32;
  constexpr int kStageBlocks = stage_blocks(BN);
  constexpr int kPer = FMT == kFmtE4M3 ? static_cast<int>(kTmemCols) / kGroups / BN : 1;
  static_assert(FMT != kFmtE4M3 || kPer % kStageBlocks == 0, "a stage's blocks are of one group");
  TileList list{reinterpret_cast<int*>(smem + L.list_off), reinterpret_cast<int*>(smem + L.list_off) + a.experts + 2};
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + L.bar_off);
  const uint32_t full = smem_u32(bars), empty = full + kMaxStages * 8;
  const uint32_t acc_full = empty + kMaxStages * 8, acc_empty = acc_full + kGroups * 8;
  const uint32_t scale_full = acc_empty + kGroups * 8, scale_empty = scale_full + kScaleSlots * 8;
  const uint32_t token = scale_empty + kScaleSlots * 8;
  constexpr int kBarriers = 2 * kMaxStages + 2 * kGroups + 2 * kScaleSlots + 2;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + kBarriers);
  // [slot][k block][row], then [slot][k block][column half]
  float* scale_x = reinterpret_cast<float*>(smem + L.scale_off);
  float* scale_w = scale_x + kScaleSlots * kScaleBlocks * kGemmRows;
  __shared__ __align__(16) float bias_s[256];  // [set][column]
  __shared__ uint32_t top_s[2][4][kSets == 2 && BN >= kFp8Block && FMT == kFmtE4M3 ? kGemmRows : 1];  // [tile's parity][group][row]

  // the same in all lanes, and known to be
  const int warp = __shfl_sync(0xFFFFFFFFu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  const int worker = blockIdx.x, workers = gridDim.x;
  const int tiles_n = (a.N + BN - 1) / BN;
  constexpr int kElems = FMT == kFmtE4M3 ? 128 : 64;  // values of a k block
  const int parts = FMT == kFmtE4M3 ? 1 : a.x_parts;
  const int KB = (a.K + kElems - 1) / kElems * parts;  // block kb: part kb % parts of x
  const bool shared_w = kStageBlocks == 2 && parts == 2;  // a stage's two blocks are one block's parts

  if (threadIdx.x == 0) {
    prefetch_tensormap(&xmap);
    prefetch_tensormap(&xmap_part);
    prefetch_tensormap(&wmap);
    prefetch_tensormap(&ymap);
    // arrivals: full by the two copying warps, acc_empty, scale_empty and token
    // by a set's warps, scale_full by the lanes of the scale warp
    uint64_t* b = bars;
    const auto init = [&](int count, int arrivals) {
      for (int i = 0; i < count; ++i) mbar_init(b++, arrivals);
    };
    init(kMaxStages, 2);
    init(kMaxStages, 1);
    init(kGroups, 1);
    init(kGroups, kSetWarps);
    init(kScaleSlots, 32);
    init(kScaleSlots, kSetWarps);
    init(2, kSetWarps);
    fence_mbar_init();
  }
  if (warp == 2) tmem_alloc(tmem_slot, kTmemCols);
  // Weights are nobody's result, and the offsets may be known to be there: then
  // the weights' stream starts while the kernel before still runs.  What reads
  // rows or scales, or writes y, waits for it.
  if (warp == 3) {
    if (a.offsets != nullptr && !a.offsets_ready) pdl_wait();
    build_list(a, list, kGemmRows, tiles_n, lane);
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  const int groups = a.offsets == nullptr ? 1 : a.experts;
  const int total = list.tile[groups];
  bool ok = true;

  if (warp < 4) {
    if constexpr (kSets == 2) asm volatile("setmaxnreg.dec.sync.aligned.u32 56;");  // of 640 threads of 96
    else asm volatile("setmaxnreg.dec.sync.aligned.u32 72;");                       // of 384 threads of 168
    if (warp == 0 || warp == 2) {
      // ---------------------------------------------------------- copies
      // warp 0: rows of x, only those that there are, by 32 (a small group's
      // tile is mostly weights); warp 2: weights
      const uint64_t keep = l2_policy_evict_normal();
      const uint32_t dst0 = smem_u32(smem) + (warp == 0 ? 0 : kStageBlocks * kXBytes);
      if (warp == 0) {
        pdl_wait();
        // every kernel before this one is done: the next may rely on that
        pdl_launch_dependents();
      }
      int e = 0, issued = 0;
      Ring ring;
      for (int t = worker; t < total && ok; t += workers) {
        const Tile tile = find_tile(list, t, kGemmRows, tiles_n, BN, e);
        const int boxes = row_boxes(tile.end - tile.m0);
        const int bytes = warp == 0 ? boxes * kBoxBytes : BN * kRowBytes;
        const int w = tile.expert * a.N + tile.n0;
        for (int kb = 0; kb < KB; kb += kStageBlocks, ++issued) {
          if (!wait_phase(empty + ring.at * 8, ring.phase ^ 1u, a.status)) {
            ok = false;
            break;
          }
          const uint32_t bar = full + ring.at * 8;
          const uint32_t dst = dst0 + ring.at * L.stage_bytes;
          const int blocks = warp == 2 && shared_w ? 1 : min(kStageBlocks, KB - kb);
          if (elect_one()) {
            arrive_expect(bar, blocks * bytes);
#pragma unroll
            for (int j = 0; j < kStageBlocks; ++j) {
              if (j >= blocks) break;
              const int part = parts == 2 ? (kb + j) & 1 : 0;
              const int k = (parts == 2 ? (kb + j) >> 1 : kb + j) * kElems;
              const auto load_x = [&](uint32_t to, const CUtensorMap* map, int row) {
                if constexpr (FMT == kFmtE4M3) load_tile(to, map, k, row, bar, keep);
                else load_tile(to, map, k, row, part, bar, keep);
              };
              if (warp == 2) {
                load_tile(dst + j * BN * kRowBytes, &wmap, k, w, bar, keep);
              } else if (boxes == kGemmRows / kGemmBoxRows) {
                load_x(dst + j * kXBytes, &xmap, tile.m0);
              } else {
                for (int b = 0; b < boxes; ++b)
                  load_x(dst + j * kXBytes + b * kBoxBytes, &xmap_part, tile.m0 + b * kGemmBoxRows);
              }
            }
          }
          __syncwarp();
          ring.next(stages);
        }
      }
      // The last stages' releases come from the tensor cores and nobody else
      // waits for them; the barriers have to be there until they have come.
      for (int i = 0; i < stages && ok; ++i) {
        ok = wait_phase(empty + ring.at * 8, ring.phase ^ 1u, a.status);
        ring.next(stages);
      }
      if (!ok)  // a wait ran out: let the copies in flight land before the CTA ends
        for (int i = max(0, issued - stages); i < issued; ++i) wait_phase(full + i % stages * 8, (i / stages) & 1, a.status);
    } else if (warp == 1) {
      // ---------------------------------------------------------- products
      const uint32_t idesc = mma_idesc<FMT>(BN);
      // The tensor pipe queues few products, so this loop's scalar work has to
      // fit under them: the whole warp runs it, with values that are the same
      // in all lanes, and one lane issues; ring places by counters,
      // descriptors by adds (every address field stays below 2^14).
      const uint64_t base = sw128_desc(smem_u32(smem));
      const uint32_t stage_units = static_cast<uint32_t>(L.stage_bytes) >> 4;
      const uint32_t w_step = shared_w ? 0 : BN * kRowBytes >> 4;  // from a stage's block of weights to the next
      Ring ring, acc;
      for (int t = worker; t < total && ok; t += workers) {
        int sub = 0;  // e4m3: every k block starts a sum of its own, kPer of them to a group
        for (int kb = 0; kb < KB; kb += kStageBlocks) {
          if (sub == 0 && (FMT == kFmtE4M3 || kb == 0)) ok = wait_phase(acc_empty + acc.at * 8, acc.phase ^ 1u, a.status);
          ok = ok && wait_phase(full + ring.at * 8, ring.phase, a.status);
          if (!ok) break;
          tc_fence_after();
          const uint64_t da = base + ring.at * stage_units;
          const uint32_t d = tmem + static_cast<uint32_t>(acc.at * kGroupCols + sub * BN);
          const int blocks = min(kStageBlocks, KB - kb);
          if (FMT == kFmtE4M3) sub += blocks;
          const bool closes = kb + blocks >= KB || (FMT == kFmtE4M3 && sub == kPer);
          if (elect_one()) {
#pragma unroll
            for (int j = 0; j < kStageBlocks; ++j) {
              if (j >= blocks) break;
              const uint64_t a0 = da + j * (kXBytes >> 4);
              const uint64_t b0 = da + kStageBlocks * (kXBytes >> 4) + j * w_step;
              const uint32_t to = FMT == kFmtE4M3 ? d + j * BN : d;
              tc_mma<FMT>(to, a0, b0, idesc, FMT != kFmtE4M3 && (kb != 0 || j != 0));
              tc_mma<FMT>(to, a0 + 2, b0 + 2, idesc, 1);
              tc_mma<FMT>(to, a0 + 4, b0 + 4, idesc, 1);
              tc_mma<FMT>(to, a0 + 6, b0 + 6, idesc, 1);
            }
            tc_commit(empty + ring.at * 8);
            if (closes) tc_commit(acc_full + acc.at * 8);
          }
          __syncwarp();
          ring.next(stages);
          if (closes) {
            sub = 0;
            acc.next(kGroups);
          }
        }
      }
    } else if (FMT == kFmtE4M3 && warp == 3) {
      // ---------------------------------------------------------- scales
      pdl_wait();
      const int NBLK = (a.N + kFp8Block - 1) / kFp8Block;
      int e = 0;
      Ring ring;
      for (int t = worker; t < total && ok; t += workers) {
        const Tile tile = find_tile(list, t, kGemmRows, tiles_n, BN, e);
        const int row0 = tile.m0 + lane;
        const float* sw = a.w_scales + static_cast<int64_t>(tile.expert) * NBLK * KB;
        const int blk0 = min(tile.n0 / kFp8Block, NBLK - 1), blk1 = min((tile.n0 + BN / 2) / kFp8Block, NBLK - 1);
        for (int kb = 0; kb < KB; kb += kScaleBlocks) {
          ok = wait_phase(scale_empty + ring.at * 8, ring.phase ^ 1u, a.status);
          if (!ok) break;
          float v[kScaleBlocks][4];
#pragma unroll
          for (int i = 0; i < kScaleBlocks; ++i) {
            const int k = min(kb + i, KB - 1);
#pragma unroll
            for (int j = 0; j < 4; ++j)
              v[i][j] = __ldg(a.x_scales + static_cast<int64_t>(k) * a.rows + min(row0 + 32 * j, a.rows - 1));
          }
          float* sx = scale_x + ring.at * kScaleBlocks * kGemmRows + lane;
          if (lane < 2 * kScaleBlocks)
            scale_w[ring.at * 2 * kScaleBlocks + lane] =
                __ldg(sw + static_cast<int64_t>(lane & 1 ? blk1 : blk0) * KB + min(kb + (lane >> 1), KB - 1));
#pragma unroll
          for (int i = 0; i < kScaleBlocks; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j) sx[i * kGemmRows + 32 * j] = v[i][j];
          arrive(scale_full + ring.at * 8);
          ring.next(kScaleSlots);
        }
      }
    }
  } else {
    if constexpr (kSets == 2) asm volatile("setmaxnreg.inc.sync.aligned.u32 104;");
    else asm volatile("setmaxnreg.inc.sync.aligned.u32 216;");
    // ------------------------------------------------------------ epilogue
    pdl_wait();
    const int quarter = warp & 3, half = ((warp - kEpiWarp0) >> 2) & 1, set = (warp - kEpiWarp0) / kSetWarps;
    constexpr int W = BN / 2;  // columns of this warp group
    const uint32_t lane_base = tmem + (static_cast<uint32_t>(quarter * 32) << 16) + static_cast<uint32_t>(half * W);
    const int local = quarter * 32 + lane;  // row of the tile's 128
    constexpr int kOuts = kStageOuts / (kSets * kSetWarps);
    uint8_t* out_s = smem + L.out_off + (warp - kEpiWarp0) * kOuts * kStageOut;
    int turn_out = 0, turn = 0;
    const int tile_groups = FMT == kFmtE4M3 ? (KB + kPer - 1) / kPer : 1;  // of accumulators, per tile
    const int tile_slots = (KB + kScaleBlocks - 1) / kScaleBlocks;         // of scales, per tile

    const auto hand_back = [&](int group) { arrive(acc_empty + group * 8); };

    // rows of no expert are zeros (codes and parts are the module's own: it does not read those rows)
    if (a.out == kOutT || a.out == kOutF32) {
      const int size = a.out == kOutF32 ? 4 : 2;
      for (int64_t r = list.start[groups] + static_cast<int64_t>(blockIdx.x); r < a.rows; r += gridDim.x) {
        char* p = reinterpret_cast<char*>(a.y) + r * a.ldy * size;
        for (int i = threadIdx.x - kEpiWarp0 * 32; i < a.N; i += kEpiThreads) {
          if (size == 4) reinterpret_cast<float*>(p)[i] = 0.0f;
          else reinterpret_cast<uint16_t*>(p)[i] = 0;
        }
      }
    }

    // A warp whose wait ran out (ok false) waits, sums and stores no more, but it
    // goes through all of its tiles: the others may have seen that phase complete
    // just in time, and meet it at the named barriers of every tile.
    int e = 0;
    for (int t = worker + set * workers, seq = set; t < total; t += kSets * workers, seq += kSets) {
      const Tile tile = find_tile(list, t, kGemmRows, tiles_n, BN, e);
      Ring ring(seq * tile_groups, kGroups), scales(seq * tile_slots, kScaleSlots);
      // The sets' sums follow one another: a set that waited for its accumulators
      // while the other's are still to come would take a phase of theirs, of the
      // same parity, for its own.
      if (kSets == 2 && seq > 0) ok = ok && wait_phase(token + set * 8, ((seq - 1) / 2) & 1, a.status);
      const int64_t row = tile.m0 + local;
      const bool live = row < tile.end;
      const int row_w = tile.m0 + quarter * 32;  // the warp's first row
      const bool idle = row_w >= tile.end;  // a warp without rows only hands buffers back
      const int n0 = tile.n0 + half * W;
      float acc[FMT == kFmtE4M3 ? W : 1];
#pragma unroll
      for (int i = 0; i < (FMT == kFmtE4M3 ? W : 1); ++i) acc[i] = 0.0f;
      if (a.bias != nullptr) {
        // the group's columns of the bias, one a thread
        group_sync(set * 2 + half);  // the tile before has been read
        if (local < W) {
          const int n = n0 + local;
          bias_s[set * BN + half * W + local] = n < a.N ? ld_t<DT>(a.bias, static_cast<int64_t>(tile.expert) * a.N + n) : 0.0f;
        }
        group_sync(set * 2 + half);
      }

      if constexpr (FMT == kFmtE4M3) {
        for (int kb = 0; kb < KB; kb += kScaleBlocks) {
          ok = ok && wait_phase(scale_full + scales.at * 8, scales.phase, a.status);
          if (!ok) break;
          const float* sx = scale_x + scales.at * kScaleBlocks * kGemmRows + local;
          const float* sw = scale_w + scales.at * 2 * kScaleBlocks + half;
          const int blocks = min(kScaleBlocks, KB - kb);
#pragma unroll 1
          for (int i = 0; i < blocks; i += kPer) {
            ok = wait_phase(acc_full + ring.at * 8, ring.phase, a.status);
            if (!ok) break;
            tc_fence_after();
            const uint32_t src = lane_base + static_cast<uint32_t>(ring.at * kGroupCols);
            if (idle) {
              if (lane == 0) hand_back(ring.at);
              ring.next(kGroups);
              continue;
            }
            // some columns at a time over the group's blocks, the next on their
            // way while these are added; a block past the end of k holds an
            // old group's sums and is left out
            float scale[kPer];
#pragma unroll
            for (int g = 0; g < kPer; ++g) scale[g] = i + g < blocks ? sx[(i + g) * kGemmRows] * sw[2 * (i + g)] : 0.0f;
            constexpr int kCols = kSets == 2 ? 16 : 32;  // what the registers hold of it
            constexpr int kRun = W / kCols, kSteps = kPer * kRun;
            constexpr int kDeep = kSets == 2 ? 1 : 2;   // loads in flight (two sets' warps hide each other's)
            uint32_t r[kDeep][kCols];
            if (kDeep == 2) tmem_ld(src, r[0]);
#pragma unroll
            for (int t = 0; t < kSteps; ++t) {
              const int g = t / kRun, c = t % kRun * kCols;
              if (kDeep == 1) tmem_ld(src + g * BN + c, r[0]);
              tmem_wait_ld(r[t % kDeep]);
              if (t + 1 == kSteps) {
                // all read: the group goes back before the last sums
                tc_fence_before();
                if (lane == 0) hand_back(ring.at);
              } else if (kDeep == 2) {
                tmem_ld(src + (t + 1) / kRun * BN + (t + 1) % kRun * kCols, r[(t + 1) % kDeep]);
              }
              if (g == 0 || i + g < blocks) {
                const uint32_t(&v)[kCols] = r[t % kDeep];
#pragma unroll
                for (int j = 0; j < kCols; ++j) acc[c + j] = fmaf(__uint_as_float(v[j]), scale[g], acc[c + j]);
              }
            }
            ring.next(kGroups);
          }
          if (!ok) break;
          __syncwarp();
          if (lane == 0) arrive(scale_empty + scales.at * 8);
          scales.next(kScaleSlots);
        }
      } else {
        ok = ok && wait_phase(acc_full + ring.at * 8, ring.phase, a.status);
        tc_fence_after();
      }
      ok = __all_sync(0xFFFFFFFFu, ok);
      if (kSets == 2 && ok && lane == 0) arrive(token + (set ^ 1) * 8);

      const uint32_t src = lane_base + static_cast<uint32_t>(ring.at * kGroupCols);
      const auto take = [&](int c, float(&v)[32]) {
        if constexpr (FMT == kFmtE4M3) {
#pragma unroll
          for (int j = 0; j < 32; ++j) v[j] = acc[c + j];
        } else {
          uint32_t r[32];
          tmem_ld(src + c, r);
          tmem_wait_ld(r);
#pragma unroll
          for (int j = 0; j < 32; ++j) v[j] = __uint_as_float(r[j]);
          if (c + 32 >= W) {
            tc_fence_before();
            __syncwarp();
            if (lane == 0) hand_back(ring.at);
          }
        }
      };
      const auto finish = [&](int c, float(&v)[32]) {
        if (a.bias != nullptr) {
          const float4* b4 = reinterpret_cast<const float4*>(bias_s + set * BN + half * W + c);
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            const float4 b = b4[j];
            v[4 * j] += b.x, v[4 * j + 1] += b.y, v[4 * j + 2] += b.z, v[4 * j + 3] += b.w;
          }
        }
        if (a.act == kActSilu) {
#pragma unroll
          for (int j = 0; j < 32; j += 2) silu2(v[j], v[j + 1]);
        } else if (a.act == kActRelu) {
#pragma unroll
          for (int j = 0; j < 32; ++j) v[j] = v[j] < 0.0f ? 0.0f : v[j];
        }
      };
      const int size = a.out == kOutF32 ? 4 : 2;
      const int rows_w = min(32, tile.end - row_w);
      const bool whole = a.tile_store && rows_w == 32;

      if constexpr (BN >= kFp8Block && FMT == kFmtE4M3) {
        if (a.out == kOutCodes) {
          // a row's block of 128 columns is one thread's, or two threads' halves:
          // its largest finite magnitude, then the codes (infinities made NaN)
          uint32_t top = 0;
          if (ok && !idle && n0 < a.N) {
            float most = 0.0f;
#pragma unroll
            for (int c = 0; c < W; c += 32) {
              float v[32];
              take(c, v);
              finish(c, v);
              if (n0 + c + 32 > a.N) {
#pragma unroll
                for (int j = 0; j < 32; ++j) v[j] = n0 + c + j < a.N ? v[j] : 0.0f;
              }
#pragma unroll
              for (int j = 0; j < 32; ++j) {
                most = fmaxf(most, fabsf(v[j]));
                acc[c + j] = v[j];
              }
            }
            top = __float_as_uint(most);
            if (top >= 0x7F800000u) {
              // (a NaN is not in the maximum, and converts to one)
              top = 0;
#pragma unroll
              for (int i = 0; i < W; ++i) {
                const uint32_t m = finite_magnitude(acc[i]);
                top = max(top, m);
                if (m == 0 && acc[i] != 0.0f) acc[i] = __uint_as_float(0x7FC00000u);
              }
            }
          }
          if constexpr (W < kFp8Block) {
            top_s[turn][set * 2 + half][local] = top;
            set_sync(set);
            top = max(top, top_s[turn][set * 2 + (half ^ 1)][local]);
            turn ^= 1;
          }
          if (!ok || idle || n0 >= a.N) continue;
          const int ex = fp8_scale_exponent(top);
          const float inv = pow2f(-ex);
          if (live && n0 % kFp8Block == 0) a.y_scales[static_cast<int64_t>(n0 / kFp8Block) * a.rows + row] = pow2f(ex);
#pragma unroll
          for (int h = 0; h < W; h += 64) {
            uint32_t w[16];
#pragma unroll
            for (int i = 0; i < 16; ++i) {
              const float* v = acc + h + 4 * i;
              w[i] = e4m3x2_finite(v[0] * inv, v[1] * inv) | (e4m3x2_finite(v[2] * inv, v[3] * inv) << 16);
            }
            if (whole) {
              store_piece<kOuts, false>(out_s, turn_out, lane, w, &ymap, n0 + h, row_w, 0);
            } else if (live) {
              store_piece_by_lanes(w, reinterpret_cast<uint8_t*>(a.y) + row * a.ldy + n0 + h);
            }
          }
          continue;
        }
      }
      if (!ok) continue;
      if (idle || n0 >= a.N) {
        if constexpr (FMT != kFmtE4M3) {
          if (lane == 0) hand_back(ring.at);
        }
        continue;
      }
#pragma unroll
      for (int c = 0; c < W; c += 32) {
        float v[32];
        take(c, v);
        if (n0 + c >= a.N) continue;
        finish(c, v);
        // 64 bytes a piece: 16 f32 values, or 32 of T; of parts the low one second
        uint32_t w[16];
        const int pieces = a.out == kOutT ? 1 : 2;
#pragma unroll 1
        for (int p = 0; p < pieces; ++p) {
          const int n = n0 + c + (a.out == kOutF32 ? 16 * p : 0);
          const int part = FMT != kFmtE4M3 && a.out == kOutParts ? p : 0;
          if (n >= a.N) break;
          if (a.out == kOutF32) {
#pragma unroll
            for (int i = 0; i < 16; ++i) w[i] = __float_as_uint(p == 0 ? v[i] : v[16 + i]);
          } else {
            if (part == 1) {
#pragma unroll
              for (int i = 0; i < 16; ++i) take_rest_t<DT>(w[i], v[2 * i], v[2 * i + 1]);
            }
#pragma unroll
            for (int i = 0; i < 16; ++i) w[i] = pack_t<DT>(v[2 * i], v[2 * i + 1]);
          }
          uint8_t* y = reinterpret_cast<uint8_t*>(a.y) + part * (a.rows * a.ldy * size);
          if (whole) {
            store_piece<kOuts, FMT != kFmtE4M3>(out_s, turn_out, lane, w, &ymap, n, row_w, part);
          } else if (a.tile_store && n + kStoreBytes / size <= a.N) {
            if (live) store_piece_by_lanes(w, y + (row * a.ldy + n) * size);
          } else {
            store_piece_by_rows(out_s, lane, w, y + (row_w * a.ldy + n) * size, a.ldy * size, size, rows_w,
                                min(kStoreBytes / size, a.N - n));
          }
        }
      }
    }
    // the tile stores have read their shared memory
    asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");
  }

  __syncwarp();
  tc_fence_before();
  __syncthreads();
  if (warp == 2) {
    tc_fence_after();
    tmem_release(tmem, kTmemCols);
  }
}

template <int FMT, int DT, int BN>
cudaError_t launch_typed(const ExpertGemmMaps& m, const ExpertGemmArgs& a, int num_sms, cudaStream_t stream, bool pdl) {
  auto kernel = expert_gemm_kernel<FMT, DT, BN>;
  static SharedMemoryOptIn opt_in;
  const cudaError_t configured = opt_in.ensure(reinterpret_cast<const void*>(kernel), kSmemLimit - kStaticBytes);
  if (configured != cudaSuccess) return configured;
  const SmemPlan p = plan_smem(FMT == kFmtE4M3, BN, a.experts);
  // no more CTAs than tiles there can be
  const int64_t groups = a.offsets == nullptr ? 1 : std::min(a.experts, a.rows);
  const int64_t tiles = ((a.rows + kGemmRows - 1) / kGemmRows + groups) * ((a.N + BN - 1) / BN);
  const int ctas = static_cast<int>(std::min<int64_t>(tiles, num_sms));
  return launch(kernel, dim3(ctas), dim3(gemm_threads(BN)), p.bytes, stream, pdl, m.x, m.x_part, m.w, m.y, a);
}

template <int FMT, int DT>
cudaError_t launch_cut(int bn, const ExpertGemmMaps& m, const ExpertGemmArgs& a, int num_sms, cudaStream_t stream, bool pdl) {
  if (bn == 256) return launch_typed<FMT, DT, 256>(m, a, num_sms, stream, pdl);
  if (bn == 128) return launch_typed<FMT, DT, 128>(m, a, num_sms, stream, pdl);
  return launch_typed<FMT, DT, 64>(m, a, num_sms, stream, pdl);
}

}  // namespace

cudaError_t launch_expert_gemm(int dtype, bool e4m3, int bn, const ExpertGemmMaps& maps,
                               const ExpertGemmArgs& a, int num_sms, cudaStream_t stream, bool pdl) {
  if (bn != 64 && bn != 128 && bn != 256) return cudaErrorInvalidValue;
  if (a.out == kOutCodes && (!e4m3 || bn < kFp8Block)) return cudaErrorInvalidValue;
  if ((a.out == kOutParts || a.x_parts != 1) && e4m3) return cudaErrorInvalidValue;
  if (e4m3)
    return dtype == kF16 ? launch_cut<kFmtE4M3, kF16>(bn, maps, a, num_sms, stream, pdl)
                         : launch_cut<kFmtE4M3, kBF16>(bn, maps, a, num_sms, stream, pdl);
  return dtype == kF16 ? launch_cut<kFmtF16, kF16>(bn, maps, a, num_sms, stream, pdl)
                       : launch_cut<kFmtBF16, kBF16>(bn, maps, a, num_sms, stream, pdl);
}

int plan_expert_gemm(bool e4m3, int rows, int experts, int N, int K, int x_parts, int act, int out, int num_sms) {
  // The cut with the least estimated time, in cycles: the last pass over a tile
  // (activation, codes, stores) and for each wave of tiles the sums of its k
  // blocks, a wave's last pass beside the next wave's sums where two sets of
  // epilogue warps take turns.  A k block takes the longer of a CTA's own time
  // and its weights' share of the memory's rate (which the tiles of one group
  // share: the second finds them in L2).  Fitted to nineteen calls of 16 to 16384
  // rows, 1 to 64 experts, n and k 520 to 18944, each with all three cuts: the
  // cut taken is the fastest of them or within 1 % for seventeen, 3 % (n 4096, k
  // 1024, 16-bit) and 7 % (8192 rows, k 1024, e4m3) behind it for two.  Both sides:
  //   64 rows, k 4096, n 1024, 8 experts, e4m3   14.1 us at 64, 18.3 at 128, 23.0 at 256
  //   1792 rows, n 4096, k 1024, 32, e4m3, SiLU  46.5           43.8         70.4
  //   8192 rows, n 2048, k 1024, 16, 16-bit      67.2           57.8         44.7
  // Two parts of x count as twice the k blocks: for the second product of seven
  // 16-bit modules of 1 to 4096 tokens the cut taken is the fastest five times, and 5 %
  // (4096 tokens, 4 experts, 512-1000) and 10 % (300, 4, 512-2048) behind it twice.  The
  // module's us, as far as they differ by that product alone:
  //   14 tokens, 8 experts, 1024-4096            61.2 at 64, 76.9 at 128, 88.6 at 256
  //   896 tokens, 32 experts, 1024-4096         189           171         148
  struct Cut {
    int bn;
    double block_e4m3, block_16, last_e4m3, last_16;
  };
  static constexpr Cut kCuts[] = {{64, 515, 480, 4300, 300}, {128, 820, 780, 7400, 600}, {256, 1020, 1140, 9900, 800}};
  constexpr double kMemoryBytes = 18.7;  // a cycle and SM
  constexpr double kActivation = 1.44;   // of SiLU or codes on the last pass
  const int KB = (K + (e4m3 ? 127 : 63)) / (e4m3 ? 128 : 64) * x_parts;
  const bool codes = out == kOutCodes;
  // experts that have rows, were the choice of expert even
  const double groups = experts * (1.0 - std::pow(1.0 - 1.0 / experts, rows)), mean = rows / groups;
  int best = 256;
  double least = 0.0;
  for (const Cut& c : kCuts) {
    if (codes && c.bn < kFp8Block) continue;
    // ragged groups have half a tile more than their mean size
    double per_group = std::ceil(mean / kGemmRows);
    if (experts > 1 && mean > kGemmRows / 2) per_group = mean / kGemmRows + 0.5;
    const double tiles = groups * per_group * ((N + c.bn - 1) / c.bn), busy = std::min(1.0, tiles / num_sms);
    const double block = std::max(e4m3 ? c.block_e4m3 : c.block_16, c.bn * kRowBytes / kMemoryBytes * busy / per_group);
    const double sums = KB * block;
    const double last = (e4m3 ? c.last_e4m3 : c.last_16) * (codes || act == kActSilu ? kActivation : 1.0);
    // (16-bit sums of the next tile begin while this one's are read)
    double wave = std::max(sums, last);
    if (e4m3) wave = epi_sets(c.bn) == 2 ? std::max(sums, (sums + last) / 2) : sums + last;
    const double waves = std::max(1.0, std::ceil(tiles / num_sms - 1e-9));
    const double time = sums + last + (waves - 1) * wave;
    if (least == 0.0 || time < least) {
      least = time;
      best = c.bn;
    }
  }
  return best;
}

}  // namespace cq
