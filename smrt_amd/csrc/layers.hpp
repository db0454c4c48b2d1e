// Launchers of the layer products, one per element type (layer_gemm.hip).
#pragma once
#include "layer_gemm.hpp"

namespace smrt {
namespace layers {
hipError_t layer_gemm_f32(int layout, const GemmArgs& g, hipStream_t stream);
hipError_t layer_gemm_bf16(int layout, const GemmArgs& g, hipStream_t stream);
hipError_t layer_gemm_f16(int layout, const GemmArgs& g, hipStream_t stream);
}  // namespace layers
}  // namespace smrt
