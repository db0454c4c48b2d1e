// The layer products' launchers, one per element type (layer_gemm.hip), and which tile shape a product gets.
#pragma once
#include <algorithm>
#include <cmath>
#include "layer_rows.hpp"

namespace smrt {
namespace layers {

// chunks of groups larger than one (layer_common.hpp); with the groups of one chunk that many workgroups more
inline int64_t max_slabs(int64_t rows, int64_t chunk, int64_t groups) { return groups == 1 ? (rows > chunk ? (rows + chunk - 1) / chunk : 0) : rows / chunk + std::min(groups, rows / chunk); }
inline int64_t max_chunks(bool ends, int64_t rows, int64_t chunk, int64_t groups) { return ends ? max_slabs(rows, chunk, groups) + groups : (rows + chunk - 1) / chunk; }

enum Tile : int { TILE_LARGE = 0, TILE_MEDIUM = 1, TILE_SMALL = 2, TILE_ROWS = 3 };
struct GemmPlan { int tile, chunk; };      // chunk: dW's rows a workgroup

// The kernels for a few rows (layer_rows.hpp) read W once per row.  Forward they end where their workgroups, one per row and 64 columns, are two a
// CU for the 16-bit types and five for fp32.  Row kernel | 64x64 tile, a call in us: fp32 1 x 1024 x 1024 7.4 | 24.6, 96 x 450 x 784 (1248 workgroups) 9.3 |
// 14.2, 128 x 784 x 450 (1024) 13 | 20, 183 x 1792 x 64 7.5 | 36.8, 256 x 128 x 1024 (4096) 20.9 | 7.4; bf16 128 x 1024 x 256 (512) 7.5 | 8.1, 183 x 1792 x 64 8.3
// | 10.9, 96 x 784 x 450 (768) 9.2 | 8.7.
inline bool few_rows(bool f32, int64_t rows, int64_t n) { return rows * ((n + 63) / 64) <= (f32 ? 1280 : 512); }
// Backward, where they save two launches, they take 8 us, 0.012 a workgroup of dx and 0.07 a row of a group (dW's); the tiles 17 us, 4 more for a join over groups, and
// what dx's chain over n is longer than the other launches.  Row kernels | tiles, a call in us: fp32 66 x 64 x 64 12.5 | 17.3, 128 x 784 x 450 35 | 24, 200 x 300 x 300 36 |
// 21, 183 x 64 x 1792 22 | 46; bf16 66 x 64 x 64 12.6 | 17.4, 183 x 64 x 1792 22 | 22.
inline bool few_rows_backward(bool f32, int64_t rows, int64_t k, int64_t n, int64_t groups) {
    const double own = 8.0 + 0.012 * (double)rows * (double)((k + 63) / 64) + 0.07 * (double)rows / (double)groups;
    const double chain = (f32 ? 24.0 : 10.5) * (double)n / 1024.0 - (f32 ? 6.0 : 10.0);
    return rows <= 256 && own <= 17.0 + (groups > 1 ? 4.0 : 0.0) + std::max(chain, 0.0);
}

// 16-bit types have 256x256 (8 waves, one workgroup a CU), 128x128 (4 or 8 waves) and 64x64 tiles whose 4 waves split the
// summed index; fp32, whose three parts fill the registers sooner, the last two.  A launch takes its share of rounds over the 256 CUs, and at
// least as long as one tile's chain of loads and products.  Measured per 1024 summed indices, in us (one tile's chain | a round):
//             16 bit: 256x256  30 | 40     128x128  17   | 11.7     64x64  10.5 | 5.6
//             fp32:                        128x128  54   | 45       64x64  24   | 15.5
// so 65536 x 1024 x 1024 in bf16 took 152 / 155 / 269 us on the three, 4096 x 1024 x 1024 35 / 21 / 25, 40000 x 784 x 450 61 / 51 / 90,
// 1024 x 784 x 450 28 / 19 / 12; in fp32 65536 x 1024 x 1024 702 / 976 us on the two, 1024 x 784 x 450 48 / 25.
// The forward epilogue of the 256x256 tile has nothing beside it on its CU: 6 us a round, 9 with the 8-bit form (bf16, 256x256 | 128x128: 32768 x 256 x 1024 relu
// 40 | 33 us, 65536 x 512 x 1024 sigmoid 108 | 95, 32768 x 1024 x 1024 elu in 8 bits 104 | 99, 65536 x 2000 x 1024 relu 282 | 325).
// k: forward, the summed index.
inline GemmPlan plan_gemm(int layout, bool f32, int64_t rows, int64_t m, int64_t n, int64_t groups, int64_t k = 0, bool packed = false) {
    constexpr int side[3] = {256, 128, 64};
    constexpr double chain[2][3] = {{30, 17, 10.5}, {1e9, 54, 24}}, round[2][3] = {{40, 11.7, 5.6}, {1e9, 45, 15.5}};
    if (layout == LAYOUT_FORWARD && few_rows(f32, rows, n)) return {TILE_ROWS, 0};
    GemmPlan best = {TILE_SMALL, 512};
    double best_us = 1e30;
    for (int t = f32 ? 1 : 0; t < 3; ++t) {
        const int64_t tn = (n + side[t] - 1) / side[t];
        GemmPlan p = {t, 0};
        double us;
        if (layout == LAYOUT_DW) {
            // the weight gradient sums over the rows: few tiles, so the rows are cut into chunks, a workgroup a tile and chunk, whose
            // sums are joined afterwards (the slabs pass through memory twice); 512 rows at least, so that a chunk outweighs its slab, and
            // no second chunk, which costs a launch more, for the rows of a mini-batch (whole step, one chunk | two: 520 x 784 x 450 fp32 27
            // | 34 us, bf16 18 | 24; 1000 rows fp32 40 | 35, bf16 23 | 25)
            const int64_t tiles = (m + side[t] - 1) / side[t] * tn, all = (t == TILE_LARGE ? 256 : 512) / std::max<int64_t>(tiles, 1);
            // one round of the CUs, with the half chunk that a group's end adds on average
            const int64_t want = std::max<int64_t>({all - (groups > 1 ? (groups + 1) / 2 : 0), all / 2, 1});
            const int64_t one = f32 ? 768 : 1024, chunk = std::max<int64_t>(rows <= one ? one : 512, (rows + want - 1) / want + 127) / 128 * 128;
            p.chunk = (int)std::min<int64_t>(chunk, 1 << 30);
            const double chunks = groups == 1 ? (double)((rows + chunk - 1) / chunk) : (double)rows / chunk + 0.5 * groups;
            const double part = std::min((double)chunk, std::max(1.0, (double)rows / groups)) / 1024.0;
            us = part * std::max(chain[f32][t], round[f32][t] * std::ceil(tiles * chunks / 256.0));
            us += 2.0 * (double)max_slabs(rows, chunk, groups) * m * n * 4.0 / 5e6;
        } else {
            const int64_t tiles = (groups == 1 ? (rows + side[t] - 1) / side[t] : rows / side[t] + groups / 2) * tn;     // about half a tile a group is empty
            const double epilogue = layout == LAYOUT_FORWARD && t == TILE_LARGE ? (packed ? 9.0 : 6.0) * 1024.0 / (double)std::max<int64_t>(k, 1) : 0.0;
            us = std::max(chain[f32][t], round[f32][t] * (double)((tiles + 255) / 256)) + epilogue * (double)((tiles + 255) / 256);
        }
        if (us < best_us) { best_us = us; best = p; }
    }
    return best;
}

hipError_t layer_gemm_f32(int layout, const GemmPlan& p, const GemmArgs& g, hipStream_t stream);
hipError_t layer_gemm_f32(const GemmArgs& dx, const GemmArgs& dw, const JoinPart& db, hipStream_t stream);      // all in one launch, in 64x64 tiles
hipError_t layer_gemm_f32(const RowsBackward& p, hipStream_t stream);
hipError_t layer_gemm_bf16(int layout, const GemmPlan& p, const GemmArgs& g, hipStream_t stream);
hipError_t layer_gemm_bf16(const GemmArgs& dx, const GemmArgs& dw, const JoinPart& db, hipStream_t stream);      // all in one launch, in 64x64 tiles
hipError_t layer_gemm_bf16(const RowsBackward& p, hipStream_t stream);
hipError_t layer_gemm_f16(int layout, const GemmPlan& p, const GemmArgs& g, hipStream_t stream);
hipError_t layer_gemm_f16(const GemmArgs& dx, const GemmArgs& dw, const JoinPart& db, hipStream_t stream);      // all in one launch, in 64x64 tiles
hipError_t layer_gemm_f16(const RowsBackward& p, hipStream_t stream);
}  // namespace layers
}  // namespace smrt
