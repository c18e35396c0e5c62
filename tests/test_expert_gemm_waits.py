"""The grouped product's epilogue when a bounded wait runs out, on the host.

The epilogue's tile loop is taken from the kernel's source and compiled as host code, a thread for each warp, with
stand-ins for the device's functions: waits that answer as the test says, and named barriers that notice a warp that
never comes.  One warp's wait runs out while every other warp sees its phases complete; whichever wait that is, all
warps have to reach the end of the loop, and that warp stores nothing more.
"""
from __future__ import annotations

import os
import re
import subprocess


from conftest import ROOT

SOURCE = os.path.join(ROOT, "catcher-tippi_b200", "csrc", "expert_gemm.cu")

HEAD = r"""
#include <math.h>
#include <stdint.h>
#include <stdio.h>
#include <string.h>
#include <unistd.h>
#include <algorithm>
#include <chrono>
#include <condition_variable>
#include <mutex>
#include <thread>
#include <vector>
using std::min; using std::max;
struct float4 { float x, y, z, w; };
enum { kFmtE4M3, kFmtF16, kFmtBF16 };
enum { kOutT, kOutF32, kOutCodes, kOutParts };
enum { kActNone, kActSilu, kActRelu };
constexpr int kGemmRows = 128, kGroups = 2, kGroupCols = 256, kScaleBlocks = 8, kScaleSlots = 2, kFp8Block = 128, kStoreBytes = 64;
constexpr int kEpiWarp0 = 4, kSetWarps = 8, kStageOuts = 16, kStageOut = 2048;
struct Args { const void* bias; int N, rows, out, act, tile_store; void* y; float* y_scales; int64_t ldy; int* status; };
struct Tile { int expert, m0, end, n0; };
struct Ring {
  int at = 0; uint32_t phase = 0;
  Ring(int used, int size) : at(used % size), phase((used / size) & 1) {}
  void next(int size) { if (++at == size) { at = 0; phase ^= 1u; } }
};
struct Named {  // a named barrier of `want` warps
  std::mutex m; std::condition_variable c; int want = 0, came = 0; long turn = 0;
  void sync() {
    std::unique_lock<std::mutex> l(m);
    const long mine = turn;
    if (++came == want) { came = 0; ++turn; c.notify_all(); return; }
    if (!c.wait_for(l, std::chrono::seconds(2), [&] { return turn != mine; })) { printf("a warp never came to its barrier\n"); fflush(stdout); _exit(3); }
  }
};
static Named group_bar[4], set_bar[2];
static int victim, fail_at;                // the warp whose wait runs out, and which of its waits
static thread_local int warp_, waits_;
static thread_local bool failed_;
static int waits_of[32];
static void fail(const char* what) { printf("%s\n", what); fflush(stdout); _exit(4); }
static bool wait_phase(uint32_t, uint32_t, int*) {
  if (failed_) fail("a warp that gave up waits again");
  if (warp_ == victim && waits_ == fail_at) { failed_ = true; return false; }
  ++waits_; ++waits_of[warp_];
  return true;
}
static void group_sync(int g) { group_bar[g].sync(); }
static void set_sync(int s) { set_bar[s].sync(); }
static void arrive(uint32_t) { if (failed_) fail("a warp that gave up signals"); }
static void tc_fence_before() {} static void tc_fence_after() {} static void __syncwarp() {}
static bool __all_sync(uint32_t, bool v) { return v; }
template <int N> static void tmem_ld(uint32_t, uint32_t (&r)[N]) { if (failed_) fail("a warp that gave up reads"); for (auto& v : r) v = 0; }
template <int N> static void tmem_wait_ld(uint32_t (&)[N]) {}
static float __uint_as_float(uint32_t u) { float f; memcpy(&f, &u, 4); return f; }
static uint32_t __float_as_uint(float f) { uint32_t u; memcpy(&u, &f, 4); return u; }
template <int DT> static float ld_t(const void*, int64_t) { return 0.0f; }
static void silu2(float&, float&) {}
static uint32_t finite_magnitude(float) { return 0; }
static int fp8_scale_exponent(uint32_t) { return 0; }
static float pow2f(int) { return 1.0f; }
static uint32_t e4m3x2_finite(float, float) { return 0; }
template <int DT> static uint32_t pack_t(float, float) { return 0; }
template <int DT> static void take_rest_t(uint32_t, float&, float&) {}
static void store() { if (failed_) fail("a warp that gave up stores"); }
template <int B, bool P, class... A> static void store_piece(A&&...) { store(); }
template <class... A> static void store_piece_by_lanes(A&&...) { store(); }
template <class... A> static void store_piece_by_rows(A&&...) { store(); }
struct List {};
static Tile find_tile(const List&, int t, int, int tiles_n, int bn, int&) {
  // one tile in three has rows for half of the warps only
  return Tile{0, t / tiles_n * 128, t / tiles_n * 128 + (t % 3 == 2 ? 64 : 128), t % tiles_n * bn};
}
constexpr int epi_sets(int bn) { return bn < 256 ? 2 : 1; }

template <int FMT, int DT, int BN>
void epilogue(const Args& a, int warp, int KB, int total, float* bias_s, float* scale_x, float* scale_w, uint32_t (*top_s)[4][128]) {
  constexpr int kSets = epi_sets(BN), W = BN / 2;
  constexpr int kPer = FMT == kFmtE4M3 ? 512 / kGroups / BN : 1;
  constexpr int kOuts = kStageOuts / (kSets * kSetWarps);
  const int lane = 0, worker = 0, workers = 1, tiles_n = (a.N + BN - 1) / BN;
  const uint32_t token = 0, scale_full = 0, scale_empty = 0, acc_full = 0, acc_empty = 0, lane_base = 0;
  const int quarter = warp & 3, half = ((warp - kEpiWarp0) >> 2) & 1, set = (warp - kEpiWarp0) / kSetWarps;
  const int local = quarter * 32 + lane;
  const List list;
  const int ymap = 0;
  uint8_t* out_s = nullptr;
  int turn_out = 0, turn = 0;
  (void)turn; (void)turn_out; (void)top_s; (void)scale_x; (void)scale_w; (void)acc_empty;
  const int tile_groups = FMT == kFmtE4M3 ? (KB + kPer - 1) / kPer : 1, tile_slots = (KB + kScaleBlocks - 1) / kScaleBlocks;
  const auto hand_back = [&](int group) { arrive(acc_empty + group * 8); };
  bool ok = true;
"""

TAIL = r"""
}

template <int FMT, int DT, int BN>
void all(int KB, int total, int N, int out, bool bias) {
  constexpr int warps = epi_sets(BN) * kSetWarps;
  static float bias_s[256], scale_x[2 * 8 * 128], scale_w[64], y_scales[1 << 16];
  static uint32_t top_s[2][4][128];
  const auto run = [&](int v, int at) {
    victim = v; fail_at = at;
    memset(waits_of, 0, sizeof waits_of);
    Args a{bias ? bias_s : nullptr, N, 4096, out, kActSilu, 1, nullptr, y_scales, 1 << 14, nullptr};
    std::vector<std::thread> t;
    for (int w = 0; w < warps; ++w) t.emplace_back([&, w] {
      warp_ = kEpiWarp0 + w; waits_ = 0; failed_ = false;
      epilogue<FMT, DT, BN>(a, warp_, KB, total, bias_s, scale_x, scale_w, top_s);
    });
    for (auto& x : t) x.join();
  };
  for (auto& b : group_bar) b.want = 4;
  for (auto& b : set_bar) b.want = 8;
  run(-1, 0);
  int count[32];
  memcpy(count, waits_of, sizeof count);
  for (int v : {kEpiWarp0, kEpiWarp0 + warps - 2})
    for (int at = 0; at < count[v]; ++at) run(v, at);
  printf("%d %d: %d waits of warp 4\n", FMT, BN, count[kEpiWarp0]);
}

int main() {
  for (bool bias : {false, true}) {
    for (int out : {kOutT, kOutF32, kOutCodes}) {
      if (out != kOutCodes) all<kFmtE4M3, 1, 64>(5, 6, 300, out, bias);
      all<kFmtE4M3, 1, 128>(11, 6, 300, out, bias);
      all<kFmtE4M3, 1, 256>(9, 4, 500, out, bias);
    }
    for (int out : {kOutT, kOutF32, kOutParts}) {
      all<kFmtBF16, 1, 64>(3, 6, 300, out, bias);
      all<kFmtBF16, 1, 128>(3, 6, 300, out, bias);
      all<kFmtBF16, 1, 256>(3, 4, 500, out, bias);
    }
  }
}
"""


def test_a_wait_that_runs_out_leaves_no_warp_waiting(tmp_path):
    text = open(SOURCE).read()
    loop = re.search(r"^    int e = 0;\n    for \(int t = worker \+ set \* workers, seq = set;.*?(?=^    // the tile stores have read)",
                     text, flags=re.S | re.M)
    assert loop, "the epilogue's tile loop is not where it was"
    src, exe = tmp_path / "epilogue.cpp", tmp_path / "epilogue"
    src.write_text(HEAD + loop.group(0).replace("&ymap", "ymap") + TAIL)
    built = subprocess.run(["g++", "-std=c++17", "-O1", "-w", "-pthread", str(src), "-o", str(exe)], capture_output=True, text=True)
    assert built.returncode == 0, built.stderr[:3000]
    ran = subprocess.run([str(exe)], capture_output=True, text=True, timeout=300)
    assert ran.returncode == 0, ran.stdout[-500:] + ran.stderr[-500:]
