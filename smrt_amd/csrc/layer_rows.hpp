// The dense layer on a few rows, forward and backward.  Rows share nothing but W, and a tile of the matrix cores would be padding: 64-row
// tiles took 10.8 us (bf16) and 24.6 us (fp32, whose padding is even split into parts) for one row of 1024 x 1024, this 6.8 and 7.4, most
// of it the launch.  W goes straight from memory into fused multiply-adds in fp32, in which products of the 16-bit types are exact; what
// bounds it is the round trips to memory, so every lane requests all it can before it waits.
#pragma once
#include "layer_gemm.hpp"

namespace smrt {
namespace layers {

constexpr int ROWS_THREADS = 512;

// A workgroup has 64 columns of one row; its 64 summing lanes (8 a wave) take every 64th row of W each, 8 requested at a time.
template <class T> __global__ void __launch_bounds__(ROWS_THREADS, 2) rows_forward_kernel(GemmArgs g) {
    constexpr int LANES_K = 64, U = 8;
    __shared__ float sums[8][64];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int n0 = (int)(blockIdx.x % (unsigned)g.tiles_n) * 64, row = (int)(blockIdx.x / (unsigned)g.tiles_n);
    const int group = g.ends ? __builtin_amdgcn_readfirstlane(row_group(g.ends, g.groups, g.rows, row)) : 0;
    const bool rest = group < 0;                        // a row of no group: zeros
    const int K = rest ? 0 : g.K;
    const T* const w = (const T*)g.B + (int64_t)(rest ? 0 : group) * g.strideB;
    const T* const x = (const T*)g.A + (int64_t)row * g.lda;
    const int kl = wave * 8 + (lane >> 3), col = n0 + (lane & 7) * 8, valid = g.N - col;
    float acc[8] = {};
    for (int k0 = 0; k0 < K; k0 += LANES_K * U) {
        T wv[U][8], xv[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int k = k0 + u * LANES_K + kl;
            load8(w + (int64_t)k * g.ldb + col, k < K ? valid : 0, wv[u]);
            xv[u] = k < K ? x[k] : (T)0.0f;
        }
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int j = 0; j < 8; ++j) acc[j] = fmaf((float)xv[u], (float)wv[u][j], acc[j]);
    }
    // the wave's eight summing lanes, by halves, then the waves in their order
#pragma unroll
    for (int j = 0; j < 8; ++j)
#pragma unroll
        for (int d = 8; d < 64; d <<= 1) acc[j] += __shfl_xor(acc[j], d);
    if (lane < 8) {
#pragma unroll
        for (int j = 0; j < 8; ++j) sums[wave][lane * 8 + j] = acc[j];
    }
    __syncthreads();
    if (wave) return;
    const int c = n0 + lane;
    const bool in = c < g.N;
    float v = 0.0f;
#pragma unroll
    for (int i = 0; i < 8; ++i) v += sums[i][lane];
    if (g.bias && in && !rest) v += (float)((const T*)g.bias)[(int64_t)group * g.stride_bias + c];
    layer_act<T, 1>(g.act, &v);
    if (rest) v = 0.0f;
    if (g.q_out) {
        const float one[8] = {in ? (float)(T)v : 0.0f};
        uint32_t top = pack_top<1>(one);
#pragma unroll
        for (int d = 1; d < 32; d <<= 1) { const uint32_t o = (uint32_t)__shfl_xor((int)top, d); top = top > o ? top : o; }
        const int byte = pack_scale<T>(top);
        if ((c & -PACK_BLOCK) < g.N) {
            g.q_out[(int64_t)row * g.ldq + c] = (int8_t)(pack_bytes<T>(one, byte)[0] & 255u);
            if ((lane & 31) == 0) g.q_scale[(int64_t)row * g.ldq_scale + c / PACK_BLOCK] = (uint8_t)byte;
        }
    }
    if (!in) return;
    if (g.act_out) ((T*)g.act_out)[(int64_t)row * g.ld_act + c] = (T)v;
    if (g.residual && !rest) v += (float)((const T*)g.residual)[(int64_t)row * g.ldr + c];
    if (!(rest && g.keep_rest)) ((T*)g.C)[(int64_t)row * g.ldc + c] = (T)v;
}

struct RowsBackward {
    const void* grad; int64_t ldg;
    const void* a; int64_t lda; const uint8_t* a_scale; int64_t ld_a_scale;      // a_scale not null: the 8-bit form; likewise x
    const void* x; int64_t ldx; const uint8_t* x_scale; int64_t ld_x_scale;
    const void* w; int64_t ldw, w_stride;
    void* dx; int64_t lddx; void* dw; int64_t lddw, dw_stride; void* db; int64_t db_stride;      // each may be null
    const int64_t* ends; int32_t groups, keep_rest, rows, k, n, act;     // keep_rest: dx of rows of no group stays as it is
    int32_t tiles_k, tiles_n, dx_blocks;            // of 64; dx_blocks = rows * tiles_k, or 0 without dx
};

// 8 columns of a matrix of T or of its 8-bit form
template <class T> __device__ __forceinline__ void load_kept(const void* p, int64_t ld, const uint8_t* scale, int64_t ld_scale, int row, int col, int valid, float (&f)[8]) {
    if (!scale) { load8f((const T*)p + (int64_t)row * ld + col, valid, f); return; }
    u32x2 q = {0u, 0u};
    int byte = 0;
    if (valid > 0) {                                    // the 8-bit rows are padded to whole blocks with zeros
        __builtin_memcpy(&q, (const int8_t*)p + (int64_t)row * ld + col, 8);
        byte = scale[(int64_t)row * ld_scale + col / PACK_BLOCK];
    }
    unpack8(q, unpack_scale(byte), f);
#pragma unroll
    for (int j = 0; j < 8; ++j) f[j] = j < valid ? f[j] : 0.0f;
}
template <class T> __device__ __forceinline__ void load_dz(const RowsBackward& p, int row, int col, int valid, float (&g)[8]) {
    load8f((const T*)p.grad + (int64_t)row * p.ldg + col, valid, g);
    if (p.act == ACT_IDENTITY) return;
    float a[8];
    load_kept<T>(p.a, p.lda, p.a_scale, p.ld_a_scale, row, col, valid, a);
    layer_act_grad8(p.act, a, g);
#pragma unroll
    for (int j = 0; j < 8; ++j) g[j] = j < valid ? g[j] : 0.0f;
}

// One launch for all three gradients, dz in fp32 on the way and nowhere in memory.  The first workgroups have 64 columns of one row of
// dx each: a wave takes 8 rows of W, whose products with dz its lanes sum.  The others have a tile of 64 x 64 of one group's
// dw each, and those of the first 64 rows of W also db.
template <class T> __global__ void __launch_bounds__(ROWS_THREADS, 2) rows_backward_kernel(RowsBackward p) {
    constexpr int STEP = 32;
    __shared__ float dz[STEP][64], xs[STEP][64];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    int bid = blockIdx.x;
    if (bid < p.dx_blocks) {
        const int row = bid / p.tiles_k, k0 = (bid % p.tiles_k) * 64 + wave * 8;
        int group = 0;
        if (p.ends) group = __builtin_amdgcn_readfirstlane(row_group(p.ends, p.groups, p.rows, row));
        if (group < 0 && p.keep_rest) return;
        const T* const w = (const T*)p.w + (int64_t)(group < 0 ? 0 : group) * p.w_stride;
        float acc[8] = {};
        for (int n0 = 0; n0 < (group < 0 ? 0 : p.n); n0 += 512) {
            const int col = n0 + lane * 8, valid = p.n - col;
            T wv[8][8];
#pragma unroll
            for (int i = 0; i < 8; ++i) load8(w + (int64_t)(k0 + i) * p.ldw + col, k0 + i < p.k ? valid : 0, wv[i]);
            float g[8];
            load_dz<T>(p, row, col, valid, g);
#pragma unroll
            for (int i = 0; i < 8; ++i)
#pragma unroll
                for (int j = 0; j < 8; ++j) acc[i] = fmaf(g[j], (float)wv[i][j], acc[i]);
        }
        float mine = 0.0f;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
#pragma unroll
            for (int d = 32; d; d >>= 1) acc[i] += __shfl_xor(acc[i], d);
            mine = lane == i ? acc[i] : mine;
        }
        if (lane < 8 && k0 + lane < p.k) ((T*)p.dx)[(int64_t)row * p.lddx + k0 + lane] = (T)mine;
        return;
    }
    bid -= p.dx_blocks;
    const int n0 = (bid % p.tiles_n) * 64;
    bid /= p.tiles_n;
    const int k0 = (bid % p.tiles_k) * 64, group = bid / p.tiles_k;
    int r0 = 0, r1 = p.rows;
    if (p.ends) { const RowSpan s = group_rows(p.ends, p.groups, p.rows, group); r0 = s.r0; r1 = s.r1; }
    const int piece = (threadIdx.x & 7) * 8, k = threadIdx.x >> 3;           // this thread: row k of the tile, 8 of its columns
    float acc[8] = {}, sum = 0.0f;
    for (int first = r0; first < r1; first += STEP) {
        __syncthreads();
        {
            // half of the threads fetch dz, half x: a row's 64 columns are 8 threads
            const int r = (threadIdx.x & 255) >> 3, row = first + r;
            float f[8];
            if (threadIdx.x < 256) load_dz<T>(p, row, n0 + piece, row < r1 ? p.n - n0 - piece : 0, f);
            else load_kept<T>(p.x, p.ldx, p.x_scale, p.ld_x_scale, row, k0 + piece, row < r1 && p.dw ? p.k - k0 - piece : 0, f);
            float* const to = threadIdx.x < 256 ? &dz[r][piece] : &xs[r][piece];
#pragma unroll
            for (int j = 0; j < 8; ++j) to[j] = f[j];
        }
        __syncthreads();
        const int count = r1 - first < STEP ? r1 - first : STEP;
        for (int r = 0; r < count; ++r) {
            const float x = xs[r][k];
#pragma unroll
            for (int j = 0; j < 8; ++j) acc[j] = fmaf(x, dz[r][piece + j], acc[j]);
            if (threadIdx.x < 64) sum += dz[r][threadIdx.x];
        }
    }
    if (p.dw && k0 + k < p.k && n0 + piece < p.n)
        store8f((T*)p.dw + (int64_t)group * p.dw_stride + (int64_t)(k0 + k) * p.lddw + n0 + piece, p.n - n0 - piece, acc);
    if (p.db && k0 == 0 && threadIdx.x < 64 && n0 + (int)threadIdx.x < p.n) ((T*)p.db)[(int64_t)group * p.db_stride + n0 + threadIdx.x] = (T)sum;
}

}  // namespace layers
}  // namespace smrt
