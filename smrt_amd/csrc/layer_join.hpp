// Joining of partial sums over rows (weight and bias gradients).
#pragma once
#include "layer_common.hpp"

namespace smrt {
namespace layers {

// out[group][row][col] = sum over the group's slabs (group_slabs), in their order: the result does not depend on timing.
// A group of one chunk has its result already, one without rows gets zeros.
struct JoinPart {
    const float* slab; int64_t slab_stride;          // slab s at s * slab_stride: [out_rows][cols]
    const int64_t* ends; int32_t groups, rows, chunk;
    int32_t out_rows, cols; void* out; int64_t ld, group_stride;
    int32_t out_f32, share, group_blocks, blocks;    // workgroups a group and altogether; 0: nothing to join
};
// A piece of 8 columns has `share` threads (a power of two) that go over its slabs side by side, about eight each, where
// the pieces alone do not fill the GPU (a gradient of 90 x 113 over 73 slabs: 35 us with a thread a piece, 9 with eight).
template <class T> __device__ __forceinline__ void join(const JoinPart& p, int block, float (*lds)[8]) {
    const int pieces = 256 / p.share, group = block / p.group_blocks;
    const Slabs slabs = group_slabs(p.ends, p.groups, p.rows, group, p.chunk);
    if (slabs.count == 1) return;
    const uint32_t per_row = (uint32_t)(p.cols + 7) / 8;
    const int part = threadIdx.x / pieces, own = threadIdx.x % pieces;
    const uint32_t piece = (uint32_t)(block - group * p.group_blocks) * pieces + own, row = piece / per_row;
    const int col = (int)(piece - row * per_row) * 8, valid = row < (uint32_t)p.out_rows ? p.cols - col : 0;
    const float* src = p.slab + slabs.first * p.slab_stride + (int64_t)row * p.cols + col;
    float sum[8] = {};
    if (valid >= 8) {
#pragma unroll 8
        for (int s = part; s < slabs.count; s += p.share) {
            float v[8];
            load8(src + s * p.slab_stride, 8, v);
#pragma unroll
            for (int j = 0; j < 8; ++j) sum[j] += v[j];
        }
    } else if (valid > 0) {
        for (int s = part; s < slabs.count; s += p.share) {
            float v[8];
            load8(src + s * p.slab_stride, valid, v);
#pragma unroll
            for (int j = 0; j < 8; ++j) sum[j] += v[j];
        }
    }
    for (int half = p.share / 2; half; half /= 2) {
        if (part >= half && part < 2 * half)
#pragma unroll
            for (int j = 0; j < 8; ++j) lds[threadIdx.x][j] = sum[j];
        __syncthreads();
        if (part < half)
#pragma unroll
            for (int j = 0; j < 8; ++j) sum[j] += lds[(part + half) * pieces + own][j];
    }
    if (part) return;
    if (valid <= 0) return;
    const int64_t at = (int64_t)group * p.group_stride + (int64_t)row * p.ld + col;
    if (p.out_f32) store8((float*)p.out + at, valid, sum);
    else store8f((T*)p.out + at, valid, sum);
}

}  // namespace layers
}  // namespace smrt
