// The product kernels of one element type; built once per type (LAYER_T, LAYER_NAME).
#include "layer_gemm.hpp"
#include "layers.hpp"

namespace smrt {
namespace layers {

template <class T, int LAYOUT, bool PACKED> static hipError_t run(const GemmArgs& in, hipStream_t stream) {
    constexpr int BM = 128, BN = 128, BK = sizeof(T) == 4 ? 32 : 64;
    GemmArgs g = in;
    g.tiles_n = (g.N + BN - 1) / BN;
    const int64_t tiles_m = LAYOUT == LAYOUT_DW ? (int64_t)((g.M + BM - 1) / BM) * g.groups * g.splits
                          : g.ends             ? (int64_t)g.rows / BM + g.groups + 1
                                               : (g.rows + BM - 1) / BM;
    const int64_t blocks = tiles_m * g.tiles_n;
    if (blocks <= 0) return hipSuccess;
    if (blocks > 0x7fffffff) return hipErrorInvalidConfiguration;
    hipLaunchKernelGGL((layer_gemm_kernel<T, LAYOUT, PACKED, BM, BN, BK, 2, 2>), dim3((unsigned)blocks), dim3(256), 0, stream, g);
    return hipGetLastError();
}

hipError_t LAYER_NAME(int layout, const GemmArgs& g, hipStream_t stream) {
    if (layout == LAYOUT_FORWARD) return run<LAYER_T, LAYOUT_FORWARD, false>(g, stream);
    if (layout == LAYOUT_DX) return run<LAYER_T, LAYOUT_DX, false>(g, stream);
    return g.A_scale ? run<LAYER_T, LAYOUT_DW, true>(g, stream) : run<LAYER_T, LAYOUT_DW, false>(g, stream);
}

}  // namespace layers
}  // namespace smrt
