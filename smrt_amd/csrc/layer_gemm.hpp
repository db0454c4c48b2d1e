// The matrix products of the dense layers: forward  y = act(x W + b) + r,  input gradient  dx = dz W^T,  weight gradient
// dW = x^T dz, each over one group of rows or over many (one weight per group).
//
// All three read row-major matrices in place.  A product tile needs its operands along the summed index; what lies
// otherwise in memory (W in the forward product, both operands of the weight gradient) is staged as it lies and turned on
// the way from LDS into registers (ds_read_b64_tr_b16).
//
// fp32.  The matrix cores multiply 16-bit numbers at 16 times the rate of 32-bit ones.  An fp32 number is the exact sum
// of three bf16 numbers (8 + 8 + 8 bits of significand, cut off, so all parts have its sign): x = h + m + l.  A product is
// then hh + (hm + mh) + (hl + mm + lh) + terms below 2^-24 of it, six bf16 products summed in fp32 -- the accuracy of an fp32
// product at 2.6 times its peak rate.  hh is summed apart from the small terms: the small ones keep their bits, and where
// hh alone is an infinity or NaN (whose parts m, l are NaN) it is the answer.
#pragma once
#include "layer_common.hpp"

namespace smrt {
namespace layers {

enum Layout : int { LAYOUT_FORWARD = 0, LAYOUT_DX = 1, LAYOUT_DW = 2 };

struct GemmArgs {
    const void* A; int64_t lda;                    // forward, dW: x [rows][k];  dx: dz [rows][n]
    const uint8_t* A_scale; int64_t lds_scale;     // x in its 8-bit form: A is int8, its scale bytes here
    const void* B; int64_t ldb, strideB;           // forward, dx: W [k][n] per group;  dW: dz [rows][n]
    void* C; int64_t ldc, strideC;                 // y, dx or dW (per group)
    float* slab;                                   // dW with splits: [splits][groups][M][N] partial sums
    const void* bias; int64_t stride_bias;         // forward only, may be null
    const void* residual; int64_t ldr;             // forward only, may be null
    void* act_out; int64_t ld_act;                 // forward only, may be null: act(z) where it is not y
    int8_t* q_out; int64_t ldq; uint8_t* q_scale; int64_t ldq_scale;     // forward only, may be null: act(z) in 8 bits
    const int64_t* ends; int32_t groups, keep_rest; // ends null: one group of all rows
    int32_t rows;                                  // of x
    int32_t M, N, K;                               // of the product (dW: M = k, N = n, K = rows)
    int32_t splits;                                // dW: slices of a group's rows
    int32_t act;
    int32_t tiles_n;
};

template <class T> struct Planes { static constexpr int n = 1; typedef T half; };
template <> struct Planes<float> { static constexpr int n = 3; typedef bf16 half; };

__device__ __forceinline__ uint32_t pack_hi(float a, float b) {     // the upper 16 bits of two floats
    return __builtin_amdgcn_perm(__float_as_uint(b), __float_as_uint(a), 0x07060302u);
}

// ---- staging.  A tile is ROWS x COLS elements of a row-major matrix, moved in pieces of 8 columns.  In LDS a row keeps its
// order but its pieces are exchanged by an XOR with row bits, so that the lanes that one LDS cycle serves meet all banks:
// along the summed index (READ_ALONG) 8 rows x one piece, across it 4 rows x 32 bytes.
template <int COLS, bool ALONG> struct Swizzle {
    static constexpr int CH = COLS / 8;
    __device__ static __forceinline__ int at(int row, int piece) {
        if (ALONG) {
            constexpr int per = CH >= 8 ? 1 : 8 / CH;
            constexpr int mask = CH >= 8 ? 7 : CH - 1;
            return row * CH + (piece ^ ((row / per) & mask));
        }
        return CH >= 16 ? row * CH + (piece ^ ((row & 3) << 2)) : row * CH + (piece ^ (((row >> 1) & 1) << 2));
    }
};

template <class T, bool PACKED> struct Raw { u32x4 v; };
template <> struct Raw<float, false> { u32x4 v[2]; };
template <class T> struct Raw<T, true> { u32x2 q; uint32_t scale; };

template <class T, bool PACKED, int ROWS, int COLS, int THREADS, bool ALONG> struct Stage {
    static constexpr int PIECES = ROWS * COLS / 8;
    static constexpr int PER = PIECES / THREADS;
    static constexpr int PLANES = PACKED ? 1 : Planes<T>::n;
    typedef typename Planes<T>::half half;
    static_assert(PIECES % THREADS == 0, "pieces of a tile over the threads");
    Raw<T, PACKED> raw[PER];

    // rows [row0, row_end), columns [col0, col_end) of the matrix; what lies outside is zero
    __device__ __forceinline__ void load(const void* base, int64_t ld, const uint8_t* scale, int64_t ld_scale, int row0, int row_end,
                                         int col0, int col_end) {
#pragma unroll
        for (int i = 0; i < PER; ++i) {
            const int p = threadIdx.x + i * THREADS, row = row0 + p / (COLS / 8), col = col0 + (p % (COLS / 8)) * 8;
            const int valid = row < row_end ? col_end - col : 0;
            if constexpr (PACKED) {
                raw[i].q = u32x2{0u, 0u};
                raw[i].scale = 0u;
                if (valid > 0) {                 // the 8-bit rows are padded to whole blocks with zeros
                    __builtin_memcpy(&raw[i].q, (const int8_t*)base + (int64_t)row * ld + col, 8);
                    raw[i].scale = scale[(int64_t)row * ld_scale + col / PACK_BLOCK];
                }
            } else {
                const T* src = (const T*)base + (int64_t)row * ld + col;
                if (valid >= 8) {
                    __builtin_memcpy(&raw[i], src, 8 * sizeof(T));
                } else {
                    T v[8];
#pragma unroll
                    for (int j = 0; j < 8; ++j) v[j] = j < valid ? src[j] : (T)0.0f;
                    __builtin_memcpy(&raw[i], v, 8 * sizeof(T));
                }
            }
        }
    }
    // into LDS: one plane of 16-bit values, or the three parts of fp32 numbers
    __device__ __forceinline__ void store(half* lds) const {
#pragma unroll
        for (int i = 0; i < PER; ++i) {
            const int p = threadIdx.x + i * THREADS;
            u32x4* dst = (u32x4*)lds + Swizzle<COLS, ALONG>::at(p / (COLS / 8), p % (COLS / 8));
            if constexpr (PACKED) {
                float f[8];
                unpack8(raw[i].q, unpack_scale((int)raw[i].scale), f);
                half h[8];
#pragma unroll
                for (int j = 0; j < 8; ++j) h[j] = (half)f[j];
                __builtin_memcpy(dst, h, 16);
            } else if constexpr (sizeof(T) == 2) {
                *dst = raw[i].v;
            } else {
                float x[8];
                __builtin_memcpy(x, &raw[i], 32);
#pragma unroll
                for (int pl = 0; pl < 3; ++pl) {
                    u32x4 w;
#pragma unroll
                    for (int j = 0; j < 4; ++j) w[j] = pack_hi(x[2 * j], x[2 * j + 1]);
                    dst[pl * PIECES] = w;
                    if (pl < 2) {
#pragma unroll
                        for (int j = 0; j < 8; ++j) x[j] -= __uint_as_float(__float_as_uint(x[j]) & 0xffff0000u);
                    }
                }
            }
        }
    }
};

template <class half> struct Mfma;
template <> struct Mfma<bf16> {
    typedef bf16 frag __attribute__((ext_vector_type(8)));
    __device__ static __forceinline__ f32x16 mul(frag a, frag b, f32x16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0); }
};
template <> struct Mfma<f16> {
    typedef f16 frag __attribute__((ext_vector_type(8)));
    __device__ static __forceinline__ f32x16 mul(frag a, frag b, f32x16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0); }
};

// The operand of a 32x32x16 product: lane l holds 8 successive summed indices from 8 * (l / 32), at row (column) l % 32 of the tile.
template <class half, int COLS, bool ALONG>
__device__ __forceinline__ typename Mfma<half>::frag read_frag(const half* lds, int base, int ks, int lane) {
    if constexpr (ALONG) {
        const u32x4 w = ((const u32x4*)lds)[Swizzle<COLS, true>::at(base + (lane & 31), ks * 2 + (lane >> 5))];
        return __builtin_bit_cast(typename Mfma<half>::frag, w);
    } else {
        // 16 lanes turn 4 summed rows x 16 columns: lane s of them points at row s / 4, columns 4 * (s % 4)
        s16x4 part[2];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const int row = ks * 16 + (lane >> 5) * 8 + h * 4 + ((lane & 15) >> 2);
            const int col = base + ((lane >> 4) & 1) * 16 + (lane & 3) * 4;
            const half* at = lds + Swizzle<COLS, false>::at(row, col >> 3) * 8 + (col & 7);
            part[h] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)at);
        }
        const s16x8 w = __builtin_shufflevector(part[0], part[1], 0, 1, 2, 3, 4, 5, 6, 7);
        return __builtin_bit_cast(typename Mfma<half>::frag, w);
    }
}

// Workgroups b, b + 8, b + 16 .. share an XCD and its L2: give each XCD a run of neighbouring tiles, which share rows of A.
__device__ __forceinline__ int xcd_tile(int b, int total) {
    const int per = total >> 3, rest = total & 7, x = b & 7, i = b >> 3;
    return x * per + (x < rest ? x : rest) + i;
}

template <class T, int LAYOUT, bool PACKED_A, int BM, int BN, int BK, int WAVES_M, int WAVES_N>
__global__ void __launch_bounds__(WAVES_M * WAVES_N * 64, 2) layer_gemm_kernel(GemmArgs g) {
    constexpr int THREADS = WAVES_M * WAVES_N * 64;
    constexpr int WM = BM / WAVES_M, WN = BN / WAVES_N, MI = WM / 32, NI = WN / 32;
    constexpr bool SPLIT3 = Planes<T>::n == 3;
    constexpr bool A_ALONG = LAYOUT != LAYOUT_DW, B_ALONG = LAYOUT == LAYOUT_DX;
    typedef typename Planes<T>::half half;
    typedef typename Mfma<half>::frag frag;
    typedef Stage<T, PACKED_A, A_ALONG ? BM : BK, A_ALONG ? BK : BM, THREADS, A_ALONG> StageA;
    typedef Stage<T, false, B_ALONG ? BN : BK, B_ALONG ? BK : BN, THREADS, B_ALONG> StageB;
    constexpr int PA = StageA::PLANES, PB = StageB::PLANES;
    constexpr int LDS_A = PA * BM * BK, LDS_B = PB * BN * BK;
    constexpr int EPI_LD = WN + 4;
    constexpr int EPI = WAVES_M * WAVES_N * 32 * EPI_LD * 4, MAIN = (LDS_A + LDS_B) * 2;
    __shared__ __attribute__((aligned(16))) char smem[EPI > MAIN ? EPI : MAIN];
    half* const lds_a = (half*)smem;
    half* const lds_b = lds_a + LDS_A;

    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int wm = (wave / WAVES_N) * WM, wn = (wave % WAVES_N) * WN;

    // which tile, of which group
    int bid = xcd_tile(blockIdx.x, gridDim.x);
    const int tn = bid % g.tiles_n;
    bid /= g.tiles_n;
    int m0, m_end, k0 = 0, k_end = g.K, group = 0, slice = 0;
    if constexpr (LAYOUT == LAYOUT_DW) {
        const int tiles_m = (g.M + BM - 1) / BM;
        m0 = (bid % tiles_m) * BM;
        m_end = g.M;
        bid /= tiles_m;
        group = bid % g.groups;
        slice = bid / g.groups;
        int r0 = 0, r1 = g.rows;
        if (g.ends) { const RowSpan s = group_rows(g.ends, group, g.rows); r0 = s.r0; r1 = s.r1; }
        int per = (r1 - r0 + g.splits - 1) / g.splits;
        per = (per + BK - 1) / BK * BK;
        const long b0 = r0 + (long)slice * per;
        k0 = b0 < r1 ? (int)b0 : r1;
        k_end = r1 - k0 > per ? k0 + per : r1;
    } else {
        if (g.ends) {
            const RowSpan s = tile_rows(g.ends, g.groups, g.rows, bid, BM);
            group = s.group; m0 = s.r0; m_end = s.r1;
            if (m0 >= m_end) return;
        } else {
            m0 = bid * BM;
            m_end = g.rows;
        }
    }
    const int n0 = tn * BN;
    const bool rest = group < 0;                     // rows of no group: zeros
    if (rest) k_end = k0;

    f32x16 acc[MI][NI] = {}, low[SPLIT3 ? MI : 1][SPLIT3 ? NI : 1] = {};
    const char* Bg = (const char*)g.B;
    if (LAYOUT != LAYOUT_DW) Bg += (int64_t)(rest ? 0 : group) * g.strideB * (int64_t)sizeof(T);

    StageA sa;
    StageB sb;
    auto fetch = [&](int k) {
        if constexpr (A_ALONG) sa.load(g.A, g.lda, g.A_scale, g.lds_scale, m0, m_end, k, k_end);
        else                   sa.load(g.A, g.lda, g.A_scale, g.lds_scale, k, k_end, m0, m_end);
        if constexpr (B_ALONG) sb.load(Bg, g.ldb, nullptr, 0, n0, g.N, k, k_end);
        else                   sb.load(Bg, g.ldb, nullptr, 0, k, k_end, n0, g.N);
    };
    if (k0 < k_end) fetch(k0);
    for (int k = k0; k < k_end; k += BK) {
        __syncthreads();
        sa.store(lds_a);
        sb.store(lds_b);
        __syncthreads();
        if (k + BK < k_end) fetch(k + BK);
#pragma unroll
        for (int ks = 0; ks < BK / 16; ++ks) {
            frag fa[PA][MI], fb[PB][NI];
#pragma unroll
            for (int p = 0; p < PA; ++p)
#pragma unroll
                for (int i = 0; i < MI; ++i) fa[p][i] = read_frag<half, A_ALONG ? BK : BM, A_ALONG>(lds_a + p * BM * BK, wm + i * 32, ks, lane);
#pragma unroll
            for (int p = 0; p < PB; ++p)
#pragma unroll
                for (int j = 0; j < NI; ++j) fb[p][j] = read_frag<half, B_ALONG ? BK : BN, B_ALONG>(lds_b + p * BN * BK, wn + j * 32, ks, lane);
#pragma unroll
            for (int i = 0; i < MI; ++i)
#pragma unroll
                for (int j = 0; j < NI; ++j) {
                    if constexpr (SPLIT3) {
#pragma unroll
                        for (int s = 2; s >= 1; --s)                      // smallest terms first
#pragma unroll
                            for (int p = 0; p <= s; ++p)
                                if (p < PA && s - p < PB) low[i][j] = Mfma<half>::mul(fa[p][i], fb[s - p][j], low[i][j]);
                    }
                    acc[i][j] = Mfma<half>::mul(fa[0][i], fb[0][j], acc[i][j]);
                }
        }
    }
    __syncthreads();

    // ---- epilogue: 32 rows of the wave's tile at a time through LDS, so that a lane ends up with 8 columns of a row
    float* const tile = (float*)smem + wave * 32 * EPI_LD;
    const int64_t out0 = LAYOUT == LAYOUT_DW ? (int64_t)group * g.strideC : 0;
#pragma unroll
    for (int i = 0; i < MI; ++i) {
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
#pragma unroll
        for (int j = 0; j < NI; ++j)
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                float v = acc[i][j][r];
                if constexpr (SPLIT3) { const float w = v + low[i][j][r]; v = __builtin_isfinite(v) ? w : v; }
                tile[((r >> 2) * 8 + (lane >> 5) * 4 + (r & 3)) * EPI_LD + j * 32 + (lane & 31)] = v;
            }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
#pragma unroll 1
        for (int it = 0; it < 32 * WN / 8 / 64; ++it) {
            const int p = it * 64 + lane, tr = p / (WN / 8), col = n0 + wn + (p % (WN / 8)) * 8;
            const int row = m0 + wm + i * 32 + tr;
            const int valid = row < m_end ? g.N - col : 0;
            float v[8];
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const f32x4 w = *(const f32x4*)(tile + tr * EPI_LD + (p % (WN / 8)) * 8 + 4 * h);
#pragma unroll
                for (int j = 0; j < 4; ++j) v[4 * h + j] = w[j];
            }
            if constexpr (LAYOUT == LAYOUT_DW) {
                if (valid <= 0) continue;
                if (g.slab) store8(g.slab + (((int64_t)slice * g.groups + group) * g.M + row) * g.N + col, valid, v);
                else        store8f((T*)g.C + out0 + (int64_t)row * g.ldc + col, valid, v);
            } else if constexpr (LAYOUT == LAYOUT_DX) {
                if (valid > 0 && !(rest && g.keep_rest)) store8f((T*)g.C + (int64_t)row * g.ldc + col, valid, v);
            } else {
                if (g.bias && !rest && valid > 0) {
                    float b[8];
                    load8f((const T*)g.bias + (int64_t)group * g.stride_bias + col, valid, b);
#pragma unroll
                    for (int j = 0; j < 8; ++j) v[j] += b[j];
                }
                layer_act8(g.act, v);
                if (rest) {
#pragma unroll
                    for (int j = 0; j < 8; ++j) v[j] = 0.0f;
                }
                if (g.q_out) {
                    float a[8];
#pragma unroll
                    for (int j = 0; j < 8; ++j) a[j] = j < valid ? (float)(T)v[j] : 0.0f;      // the 8-bit form of the value in T
                    pack_block<T>(a, lane, row < m_end && col < ((g.N + PACK_BLOCK - 1) & -PACK_BLOCK), g.q_out + (int64_t)row * g.ldq + col,
                                  g.q_scale + (int64_t)row * g.ldq_scale + col / PACK_BLOCK);
                }
                if (valid > 0) {
                    if (g.act_out) store8f((T*)g.act_out + (int64_t)row * g.ld_act + col, valid, v);
                    if (g.residual && !rest) {
                        float b[8];
                        load8f((const T*)g.residual + (int64_t)row * g.ldr + col, valid, b);
#pragma unroll
                        for (int j = 0; j < 8; ++j) v[j] += b[j];
                    }
                    if (!(rest && g.keep_rest)) store8f((T*)g.C + (int64_t)row * g.ldc + col, valid, v);
                }
            }
        }
    }
}

}  // namespace layers
}  // namespace smrt
