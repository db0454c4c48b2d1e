// The product kernels of one element type; built once per type (LAYER_T, LAYER_NAME).
#include "layer_gemm.hpp"
#include "layers.hpp"

namespace smrt {
namespace layers {

// fills in tiles_n; as many workgroups as any ends need
template <int LAYOUT, int BM, int BN> static int64_t workgroups(GemmArgs& g) {
    g.tiles_n = (g.N + BN - 1) / BN;
    const int64_t tiles_m = LAYOUT == LAYOUT_DW ? (int64_t)((g.M + BM - 1) / BM) * max_chunks(g.ends != nullptr, g.rows, g.chunk, g.groups)
                          : g.ends             ? (int64_t)g.rows / BM + g.groups + 1
                                               : (g.rows + BM - 1) / BM;
    return tiles_m * g.tiles_n;
}

template <class T, int LAYOUT, bool PACKED, int BM, int BN, int BK, int WAVES_M, int WAVES_N, int WAVES_K, int BUFS>
static hipError_t run(const GemmArgs& in, hipStream_t stream) {
    GemmArgs g = in;
    const int64_t blocks = workgroups<LAYOUT, BM, BN>(g);
    if (blocks <= 0) return hipSuccess;
    if (blocks > 0x7fffffff) return hipErrorInvalidConfiguration;
    hipLaunchKernelGGL((layer_gemm_kernel<T, LAYOUT, PACKED, BM, BN, BK, WAVES_M, WAVES_N, WAVES_K, BUFS>), dim3((unsigned)blocks),
                       dim3(WAVES_M * WAVES_N * WAVES_K * 64), 0, stream, g);
    return hipGetLastError();
}

template <class T, int LAYOUT, bool PACKED> static hipError_t run_tile(int tile, const GemmArgs& g, hipStream_t stream) {
    if constexpr (sizeof(T) == 4) {
        // 8 waves a 128x128 tile hide more of each other's waits than 4 where a CU has one tile (8192 x 784 x 450 forward 47 us against 53) and
        // do as well where it has many (65536 x 1024 x 1024 718 / 713, dx 702 / 700); where both operands are turned they do worse (817 / 723)
        if (tile == TILE_SMALL) return run<T, LAYOUT, PACKED, 64, 64, 64, 1, 1, 4, 1>(g, stream);
        return run<T, LAYOUT, PACKED, 128, 128, 32, 2, LAYOUT == LAYOUT_DW ? 2 : 4, 1, 1>(g, stream);
    } else {
        if (tile == TILE_LARGE) return run<T, LAYOUT, PACKED, 256, 256, 32, 2, 4, 1, 3>(g, stream);
        if constexpr (LAYOUT != LAYOUT_DW) {
            // the same with up to a tile a CU (8192 x 784 x 450 forward 17.9 us against 20.0, 1024 x 784 x 450 15.7 / 18.6), but with more of them
            // 4 waves do better (16384 x 1024 x 1024 45.6 us against 46.8, 65536 x 1024 x 1024 159 / 171)
            const bool one_a_cu = (int64_t)((g.rows + 127) / 128) * ((g.N + 127) / 128) <= 256;
            if (tile == TILE_MEDIUM && one_a_cu) return run<T, LAYOUT, PACKED, 128, 128, 64, 2, 4, 1, 1>(g, stream);
        }
        if (tile == TILE_MEDIUM) return run<T, LAYOUT, PACKED, 128, 128, 64, 2, 2, 1, 1>(g, stream);
        return run<T, LAYOUT, PACKED, 64, 64, 128, 1, 1, 4, 1>(g, stream);
    }
}

hipError_t LAYER_NAME(const RowsBackward& p, hipStream_t stream) {
    const int64_t blocks = p.dx_blocks + (p.dw || p.db ? (int64_t)p.groups * p.tiles_k * p.tiles_n : 0);
    if (blocks <= 0) return hipSuccess;
    if (blocks > 0x7fffffff) return hipErrorInvalidConfiguration;
    hipLaunchKernelGGL((rows_backward_kernel<LAYER_T>), dim3((unsigned)blocks), dim3(ROWS_THREADS), 0, stream, p);
    return hipGetLastError();
}

template <class T, bool PACKED> static hipError_t run_pair(const GemmArgs& in_dx, const GemmArgs& in_dw, const JoinPart& db, hipStream_t stream) {
    GemmArgs dx = in_dx, dw = in_dw;
    const int64_t dx_blocks = (workgroups<LAYOUT_DX, 64, 64>(dx) + 7) / 8 * 8, dw_blocks = workgroups<LAYOUT_DW, 64, 64>(dw), blocks = dx_blocks + dw_blocks + db.blocks;
    if (blocks > 0x7fffffff) return hipErrorInvalidConfiguration;
    hipLaunchKernelGGL((layer_gemm_pair_kernel<T, PACKED, 64, 64, sizeof(T) == 4 ? 64 : 128>), dim3((unsigned)blocks), dim3(256), 0, stream, dx, dw, db,
                       (int)dx_blocks, (int)dw_blocks);
    return hipGetLastError();
}
hipError_t LAYER_NAME(const GemmArgs& dx, const GemmArgs& dw, const JoinPart& db, hipStream_t stream) {
    return dw.A_scale ? run_pair<LAYER_T, true>(dx, dw, db, stream) : run_pair<LAYER_T, false>(dx, dw, db, stream);
}

hipError_t LAYER_NAME(int layout, const GemmPlan& p, const GemmArgs& g, hipStream_t stream) {
    if (p.tile == TILE_ROWS) {
        GemmArgs r = g;
        r.tiles_n = (g.N + 63) / 64;
        hipLaunchKernelGGL((rows_forward_kernel<LAYER_T>), dim3((unsigned)(g.rows * r.tiles_n)), dim3(ROWS_THREADS), 0, stream, r);
        return hipGetLastError();
    }
    if (layout == LAYOUT_FORWARD) return run_tile<LAYER_T, LAYOUT_FORWARD, false>(p.tile, g, stream);
    if (layout == LAYOUT_DX) return run_tile<LAYER_T, LAYOUT_DX, false>(p.tile, g, stream);
    return g.A_scale ? run_tile<LAYER_T, LAYOUT_DW, true>(p.tile, g, stream) : run_tile<LAYER_T, LAYOUT_DW, false>(p.tile, g, stream);
}

}  // namespace layers
}  // namespace smrt
