// Which tile and how many K splits a matrix product of mma.h takes: the choice with the smallest estimated time.
//
// A block's K step takes `alone` microseconds when it has a CU to itself (a latency: barrier, transfer, LDS) and costs the CU
// `share` microseconds when blocks overlap.  Measured on 1024 x 1024 x 4096 (one block per CU or less) and 2048^3 .. 8192^2 x
// 2048 (CUs full), less 5 us per launch, per step of 64 bf16 / fp16, 32 values in two planes, 128 int8:
//                          one plane            two planes
//                       alone   share        alone   share
//   64 x 64              0.50    0.21         0.52    0.23
//   96 x 96              0.56    0.39         0.62    0.43
//   64 x 128             0.58    0.37         0.60    0.37
//   128 x 128            0.72    0.58         0.85    0.62
//   256 x 256            1.22    1.75         1.72    2.10
// e.g. 2048^3 in two planes: 64 x 64 64 us, 64 x 128 52, 128 x 128 61, 256 x 256 121; 8192^2 x 2048: 128 x 128 632, 256 x 256 570.
// Splitting K writes and reads fp32 partial sums (about 3.5 TB/s) and shortens the chain of steps.
#pragma once
#include <stdint.h>

#include <algorithm>

namespace suave {
namespace mma {

enum TileId : int { kT64 = 0, kT96 = 1, kT64x128 = 2, kT128 = 3, kT256 = 4, kTileIds = 5 };
constexpr int kTileM[kTileIds] = {64, 96, 64, 128, 256};
constexpr int kTileN[kTileIds] = {64, 96, 128, 128, 256};
constexpr double kAlone[2][kTileIds] = {{0.50, 0.56, 0.58, 0.72, 1.22}, {0.52, 0.62, 0.60, 0.85, 1.72}};
constexpr double kShare[2][kTileIds] = {{0.21, 0.39, 0.37, 0.58, 1.75}, {0.23, 0.43, 0.37, 0.62, 2.10}};
constexpr int kCUs = 256;

inline int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }

// One product: `tiles` tiles of `steps` K steps
struct Work {
  int64_t tiles, steps;
  double sum_bytes;  // of one fp32 result: what each split writes and a later launch reads
};
// microseconds of n products that share a launch, product i with its K cut into split[i] blocks per tile
inline double estimate_us(TileId t, int planes, const Work* w, const int* split, int n) {
  double cu = 0, chain = 0, bytes = 0;
  for (int i = 0; i < n; ++i) {
    const double steps = (double)ceil_div(w[i].steps, split[i]);
    const double blocks = (double)(w[i].tiles * split[i]) / kCUs;
    // whole blocks per CU while there are few
    cu += (blocks < 6 ? (double)ceil_div(w[i].tiles * split[i], kCUs) : blocks) * steps * kShare[planes - 1][t];
    chain = std::max(chain, steps * kAlone[planes - 1][t]);
    if (split[i] > 1) bytes += 2.0 * split[i] * w[i].sum_bytes;
  }
  return std::max(cu, chain) + bytes / 3.5e6 + (bytes > 0 ? 4.0 : 0.0);
}

}  // namespace mma
}  // namespace suave
