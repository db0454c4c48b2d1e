// The matrix products of the dense layers: forward  y = act(x W + b) + r,  input gradient  dx = dz W^T,  weight gradient
// dW = x^T dz, each over one group of rows or over many (one weight per group).
//
// All three read row-major matrices in place.  A product tile needs its operands along the summed index; what lies
// otherwise in memory (W in the forward product, both operands of the weight gradient) is staged as it lies and turned on
// the way from LDS into registers (ds_read_b64_tr_b16).
//
// fp32.  The matrix cores multiply 16-bit numbers at 16 times the rate of 32-bit ones.  An fp32 number is the sum of three bf16
// numbers, x = h + m + l: h is x cut off after 8 bits (so no number becomes an infinity), m the next 8, l the rest -- exact while x's last bit is a number
// of bf16, which it is from |x| = 2^-110 up; below, the products keep an absolute 2^-133.  A product is hh + (hm + mh) + (hl + mm + lh) + (ml + lm + ll):
// six bf16 products summed in fp32, at 2.6 times the fp32 product's peak rate; the last three are left out.  In A m is cut off, in B it is rounded away from zero,
// so that l has x's sign in A and the other in B, and ml and lm have different signs: together they are below 2^-22 of the product (4 u, u = 2^-24) and
// 0 on average, 0.37 u in the root mean square over random numbers, where rounding an fp32 product is 0.42 u.  (With m cut off in both they reach 7.8 u, always of the product's
// sign, 0.63 u on average; a step of 40000 x 784 x 450 in 8 groups 921 us, this 933, both rounded to nearest 946.)
// hh is summed apart from the small terms: the small ones keep their bits, and where
// hh alone is an infinity or NaN (whose parts m, l are NaN) it is the answer.  (h of a NaN that has no bit of its payload in the upper half, which no operation
// yields, is an infinity.)
#pragma once
#include "layer_join.hpp"

namespace smrt {
namespace layers {

enum Layout : int { LAYOUT_FORWARD = 0, LAYOUT_DX = 1, LAYOUT_DW = 2 };

struct GemmArgs {
    const void* A; int64_t lda;                    // forward, dW: x [rows][k];  dx: dz [rows][n]
    const uint8_t* A_scale; int64_t lds_scale;     // x in its 8-bit form: A is int8, its scale bytes here
    const void* B; int64_t ldb, strideB;           // forward, dx: W [k][n] per group;  dW: dz [rows][n]
    void* C; int64_t ldc, strideC;                 // y, dx or dW (per group)
    float* slab;                                   // dW: [chunks of the larger groups][M][N] sums
    const void* bias; int64_t stride_bias;         // forward only, may be null
    const void* residual; int64_t ldr;             // forward only, may be null
    void* act_out; int64_t ld_act;                 // forward only, may be null: act(z) where it is not y
    int8_t* q_out; int64_t ldq; uint8_t* q_scale; int64_t ldq_scale;     // forward only, may be null: act(z) in 8 bits
    const int64_t* ends; int32_t groups, keep_rest; // ends null: one group of all rows
    int32_t rows;                                  // of x
    int32_t M, N, K;                               // of the product (dW: M = k, N = n, K = rows)
    int32_t chunk;                                 // dW: rows a workgroup sums over (chunk_rows)
    int32_t act;
    int32_t tiles_n;
};

template <class T> struct Planes { static constexpr int n = 1; typedef T half; };
template <> struct Planes<float> { static constexpr int n = 3; typedef bf16 half; };

__device__ __forceinline__ uint32_t pack_hi(uint32_t a, uint32_t b) {     // the upper halves of two words
    return __builtin_amdgcn_perm(b, a, 0x07060302u);
}

// ---- staging.  A tile is ROWS x COLS elements of a row-major matrix, moved in pieces of 8 columns.  In LDS a row keeps its
// order but its pieces are exchanged by an XOR with row bits, so that the lanes that one LDS cycle serves (256 bytes) meet all
// 64 banks: along the summed index (ALONG) 16 rows x one piece, across it 4 rows x 64 bytes.
template <int COLS, bool ALONG> struct Swizzle {
    static constexpr int CH = COLS / 8;
    __device__ static __forceinline__ int at(int row, int piece) {
        if (ALONG) {
            constexpr int per = CH >= 16 ? 1 : 16 / CH, mask = CH >= 16 ? 15 : CH - 1;
            return row * CH + (piece ^ ((row / per) & mask));
        }
        return CH >= 16 ? row * CH + (piece ^ ((row & 3) << 2)) : row * CH + (piece ^ (((row >> 1) & 1) << 2));
    }
};

template <class T, bool PACKED> struct Raw { u32x4 v; };
template <> struct Raw<float, false> { u32x4 v[2]; };
template <class T> struct Raw<T, true> { u32x2 q; uint32_t scale; };

// UP: of an fp32 number's three parts the second is rounded away from zero (operand B)
template <class T, bool PACKED, int ROWS, int COLS, int THREADS, bool ALONG, bool UP> struct Stage {
    static constexpr int CH = COLS / 8, PIECES = ROWS * CH, PER = PIECES / THREADS, STEP = THREADS / CH;
    static constexpr int PLANES = PACKED ? 1 : Planes<T>::n;
    static constexpr int ESZ = PACKED ? 1 : sizeof(T);
    typedef typename Planes<T>::half half;
    static_assert(PIECES % THREADS == 0 && THREADS % CH == 0, "a thread keeps its columns");
    static constexpr int BACK = 8;                   // columns before the tile's first where the loads' base lies: a piece may begin there
    Raw<T, PACKED> raw[PER];
    uint32_t off[PER], soff[PACKED ? PER : 1];       // bytes from the base (of the scale bytes: from the tile's first)
    int shift;                                       // elements by which a piece that an end cuts is read earlier

    // rows and cols: what the tile has of the matrix along its own index (rows for ALONG, columns otherwise).  Nothing else needs a
    // test: every load stays inside the matrix, so the loop that issues them has no branch and keeps them in flight.  Rows behind the
    // end read the last row and columns behind the end the last ones, which only reaches results that are never stored.
    __device__ __forceinline__ void init(int64_t ld, int64_t ld_scale, int rows, int cols) {
        const int row = threadIdx.x / CH;
        int col = (threadIdx.x % CH) * 8;
        shift = 0;
        if (!ALONG && col + 8 > cols) {
            const int c = PACKED ? (cols - 1) & -8 : cols - 8;
            shift = !PACKED && col < cols ? col - c : 0;
            col = c;
        }
#pragma unroll
        for (int i = 0; i < PER; ++i) {
            int r = row + i * STEP;
            if (ALONG) r = r < rows ? r : rows - 1;
            off[i] = (uint32_t)r * (uint32_t)ld * ESZ + (uint32_t)(col + BACK) * ESZ;
            if constexpr (PACKED) soff[i] = (uint32_t)r * (uint32_t)ld_scale + (uint32_t)col / PACK_BLOCK;
        }
    }
    // before the last step is requested, which has only `has` of its summed indices
    __device__ __forceinline__ void to_last(int64_t ld, int64_t ld_scale, int has) {
        const int row = threadIdx.x / CH, col = (threadIdx.x % CH) * 8;
        if constexpr (ALONG) {
            if (col + 8 > has) {
                shift = col < has ? col - (has - 8) : 0;
#pragma unroll
                for (int i = 0; i < PER; ++i) off[i] -= (uint32_t)(col - (has - 8)) * ESZ;
            }
        } else {
#pragma unroll
            for (int i = 0; i < PER; ++i) {
                const int over = row + i * STEP - (has - 1);
                if (over > 0) {
                    off[i] -= (uint32_t)over * (uint32_t)ld * ESZ;
                    if constexpr (PACKED) soff[i] -= (uint32_t)over * (uint32_t)ld_scale;
                }
            }
        }
    }
    // a step; base (and scale) are the same in all lanes
    __device__ __forceinline__ void load(const char* base, const uint8_t* scale) {
#pragma unroll
        for (int i = 0; i < PER; ++i) {
            if constexpr (PACKED) {
                __builtin_memcpy(&raw[i].q, base + off[i], 8);
                raw[i].scale = scale[soff[i]];
            } else {
                __builtin_memcpy(&raw[i], base + off[i], 8 * sizeof(T));
            }
        }
    }
    // pieces that were read `shift` elements early, moved to their place; what comes in behind is zero
    __device__ __forceinline__ void unshift() {
        if constexpr (!PACKED) {
            constexpr int W = 2 * sizeof(T);         // words of a piece
#pragma unroll
            for (int i = 0; i < PER; ++i) {
                uint32_t w[W];
                __builtin_memcpy(w, &raw[i], 4 * W);
#pragma unroll
                for (int step = 4; step >= 1; step >>= 1) {
                    const bool on = shift & step;
                    if (sizeof(T) == 2 && step == 1) {
#pragma unroll
                        for (int j = 0; j < W; ++j) w[j] = on ? __builtin_amdgcn_alignbit(j + 1 < W ? w[j + 1] : 0u, w[j], 16) : w[j];
                    } else {
                        const int by = step * (int)sizeof(T) / 4;
#pragma unroll
                        for (int j = 0; j < W; ++j) w[j] = on ? (j + by < W ? w[j + by] : 0u) : w[j];
                    }
                }
                __builtin_memcpy(&raw[i], w, 4 * W);
            }
        }
    }
    // the last step: what lies behind its `has` summed indices becomes zero
    __device__ __forceinline__ void clear_last(int has) {
        if (ALONG) unshift();
#pragma unroll
        for (int i = 0; i < PER; ++i)
            if (ALONG ? (int)(threadIdx.x % CH) * 8 >= has : (int)(threadIdx.x / CH) + i * STEP >= has) raw[i] = {};
    }
    // any step of a matrix of fewer than 8 columns, which has no whole piece: rows x cols is what there is of the tile, the rest is zero
    __device__ __forceinline__ void load_narrow(const char* base, const uint8_t* scale, int64_t ld, int64_t ld_scale, int rows, int cols) {
#pragma unroll
        for (int i = 0; i < PER; ++i) {
            const int row = threadIdx.x / CH + i * STEP, col = (threadIdx.x % CH) * 8, valid = row < rows ? cols - col : 0;
            if constexpr (PACKED) {
                raw[i].q = u32x2{0u, 0u};
                raw[i].scale = 0u;
                if (valid > 0) {                     // the 8-bit rows are padded to whole blocks with zeros
                    __builtin_memcpy(&raw[i].q, base + (int64_t)row * ld + col, 8);
                    raw[i].scale = scale[(int64_t)row * ld_scale + col / PACK_BLOCK];
                }
            } else {
                T v[8];
                load8((const T*)base + (int64_t)row * ld + col, valid, v);
                __builtin_memcpy(&raw[i], v, 8 * sizeof(T));
            }
        }
    }
    // into LDS: one plane of 16-bit values, or the three parts of fp32 numbers
    __device__ __forceinline__ void store(half* lds) const {
#pragma unroll
        for (int i = 0; i < PER; ++i) {
            u32x4* dst = (u32x4*)lds + Swizzle<COLS, ALONG>::at(threadIdx.x / CH + i * STEP, threadIdx.x % CH);
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
                    // what the part is cut from: adding 2^16 - 1 to the bits takes the cut part away from zero
                    uint32_t from[8];
#pragma unroll
                    for (int j = 0; j < 8; ++j) from[j] = __float_as_uint(x[j]) + (UP && pl == 1 ? 0xffffu : 0u);
                    u32x4 w;
#pragma unroll
                    for (int j = 0; j < 4; ++j) w[j] = pack_hi(from[2 * j], from[2 * j + 1]);
                    dst[pl * PIECES] = w;
                    if (pl < 2) {
#pragma unroll
                        for (int j = 0; j < 8; ++j) x[j] -= __uint_as_float(from[j] & 0xffff0000u);
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

// All waves have written their part of LDS and read what they needed.  Loads from global memory go on.
__device__ __forceinline__ void lds_barrier() {
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup", "local");
    __builtin_amdgcn_s_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup", "local");
}

// BUFS = 1: two barriers a step, and the other workgroups of the CU multiply meanwhile (three of 128x128 with 4 waves in the 16-bit types, two in
// fp32, whose parts fill three times the LDS).  BUFS = 3, for the tile that leaves room for one workgroup a CU: while one step of BK is multiplied the one
// after the next goes from registers into LDS and the one behind that is requested from memory; one barrier a step.
// WAVES_K > 1: the waves share a small tile and split each step's summed indices between them; their sums are joined in LDS.
template <class T, int LAYOUT, bool PACKED_A, int BM, int BN, int BK, int WAVES_M, int WAVES_N, int WAVES_K, int BUFS> struct Product {
    static constexpr int WAVES = WAVES_M * WAVES_N * WAVES_K, THREADS = WAVES * 64;
    static constexpr int WM = BM / WAVES_M, WN = BN / WAVES_N, MI = WM / 32, NI = WN / 32, KS = BK / 16 / WAVES_K;
    static constexpr bool SPLIT3 = Planes<T>::n == 3;
    static constexpr bool A_ALONG = LAYOUT != LAYOUT_DW, B_ALONG = LAYOUT == LAYOUT_DX;
    typedef typename Planes<T>::half half;
    typedef typename Mfma<half>::frag frag;
    typedef Stage<T, PACKED_A, A_ALONG ? BM : BK, A_ALONG ? BK : BM, THREADS, A_ALONG, false> StageA;
    typedef Stage<T, false, B_ALONG ? BN : BK, B_ALONG ? BK : BN, THREADS, B_ALONG, true> StageB;
    static constexpr int PA = StageA::PLANES, PB = StageB::PLANES;
    static constexpr int LDS_A = PA * BM * BK, LDS_B = PB * BN * BK, LDS_STEP = LDS_A + LDS_B;
    static constexpr int EPI_LD = WN + 4, EPI_ROWS = WAVES_K > 1 ? WM : 32, EPI = WAVES * EPI_ROWS * EPI_LD * 4, MAIN = LDS_STEP * 2 * BUFS;
    static constexpr int SMEM = EPI > MAIN ? EPI : MAIN;
    __device__ static __forceinline__ void run(const GemmArgs& g, int block, char* smem);
};
template <class T, int LAYOUT, bool PACKED_A, int BM, int BN, int BK, int WAVES_M, int WAVES_N, int WAVES_K, int BUFS>
__device__ __forceinline__ void Product<T, LAYOUT, PACKED_A, BM, BN, BK, WAVES_M, WAVES_N, WAVES_K, BUFS>::run(const GemmArgs& g, int block, char* smem) {
    half* const lds = (half*)smem;

    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int wk = wave / (WAVES_M * WAVES_N), wm = (wave / WAVES_N % WAVES_M) * WM, wn = (wave % WAVES_N) * WN;

    // Which tile, of which group.  The grid is as large as any ends need; the workgroups too many are the last ones, so that every
    // XCD has as much to do.
    const int tiles_m = (g.M + BM - 1) / BM;
    const int count = LAYOUT == LAYOUT_DW ? count_chunks(g.ends, g.groups, g.rows, g.chunk) * tiles_m : count_tiles(g.ends, g.groups, g.rows, BM);
    const int total = __builtin_amdgcn_readfirstlane(count) * g.tiles_n;
    if (block >= total) return;
    int bid = xcd_tile(block, total);
    const int tn = bid % g.tiles_n;
    bid /= g.tiles_n;
    int m0, m_end, k0 = 0, k_end = g.K, group = 0, slab = -1;
    if constexpr (LAYOUT == LAYOUT_DW) {
        m0 = (bid % tiles_m) * BM;
        m_end = g.M;
        const Chunk c = chunk_rows(g.ends, g.groups, g.rows, bid / tiles_m, g.chunk);
        group = __builtin_amdgcn_readfirstlane(c.group);
        if (group < 0) return;
        k0 = __builtin_amdgcn_readfirstlane(c.r0);
        k_end = __builtin_amdgcn_readfirstlane(c.r1);
        slab = __builtin_amdgcn_readfirstlane(c.slab);
    } else {
        if (g.ends) {
            const RowSpan s = tile_rows(g.ends, g.groups, g.rows, bid, BM);
            group = __builtin_amdgcn_readfirstlane(s.group);
            m0 = __builtin_amdgcn_readfirstlane(s.r0);
            m_end = __builtin_amdgcn_readfirstlane(s.r1);
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
    StageA sa;
    StageB sb;
    // the tiles' first elements, and how far a step along the summed index is
    const int64_t esa = StageA::ESZ, esb = sizeof(T);
    const char* pa = (const char*)g.A + (A_ALONG ? m0 * g.lda + k0 : k0 * g.lda + m0) * esa;
    const uint8_t* psc = PACKED_A ? g.A_scale + (int64_t)k0 * g.lds_scale + m0 / PACK_BLOCK : nullptr;
    const char* pb = (const char*)g.B + ((LAYOUT == LAYOUT_DW || rest ? 0 : group) * g.strideB + (B_ALONG ? n0 * g.ldb + k0 : k0 * g.ldb + n0)) * esb;
    const int64_t step_a = (A_ALONG ? BK : BK * g.lda) * esa, step_b = (B_ALONG ? BK : BK * g.ldb) * esb, step_sc = PACKED_A ? BK * g.lds_scale : 0;
    const int m_has = m_end - m0, n_has = g.N - n0;
    const int steps = (k_end - k0 + BK - 1) / BK, last_has = k_end - k0 - (steps - 1) * BK;
    const bool partial = last_has < BK;              // of the summed index, the last step
    // a piece that an end cuts reaches back over at most 8 columns; a matrix that has not so many is loaded with tests
    const bool narrow = ((A_ALONG ? g.K : g.M) < 8 && !PACKED_A) || (B_ALONG ? g.K : g.N) < 8;
    int fetched = 0;
    // requests the next step, or the last one again (its pieces then go into a part of LDS that nothing reads)
    auto fetch = [&] {
        if (partial && fetched == steps - 1) {
            sa.to_last(g.lda, g.lds_scale, last_has);
            sb.to_last(g.ldb, 0, last_has);
        }
        sa.load(pa - StageA::BACK * esa, psc);
        sb.load(pb - StageB::BACK * esb, nullptr);
        asm volatile("" ::: "memory");               // the loads stay here: what uses them is a step away, and the compiler would move them there
        const bool more = ++fetched < steps;
        pa += more ? step_a : 0;
        pb += more ? step_b : 0;
        if (PACKED_A) psc += more ? step_sc : 0;
    };
    auto put = [&](int t, half* to, auto edge) {
        if constexpr (decltype(edge)::value) {
            if (!A_ALONG) sa.unshift();
            if (!B_ALONG) sb.unshift();
        }
        if (partial && t == steps - 1) { sa.clear_last(last_has); sb.clear_last(last_has); }
        sa.store(to);
        sb.store(to + LDS_A);
    };
    frag fa[2][PA][MI], fb[2][PB][NI];
    auto read = [&](const half* from, int ks) {
        frag (&a)[PA][MI] = fa[ks & 1];
        frag (&b)[PB][NI] = fb[ks & 1];
#pragma unroll
        for (int p = 0; p < PA; ++p)
#pragma unroll
            for (int i = 0; i < MI; ++i) a[p][i] = read_frag<half, A_ALONG ? BK : BM, A_ALONG>(from + p * BM * BK, wm + i * 32, wk * KS + ks, lane);
#pragma unroll
        for (int p = 0; p < PB; ++p)
#pragma unroll
            for (int j = 0; j < NI; ++j) b[p][j] = read_frag<half, B_ALONG ? BK : BN, B_ALONG>(from + LDS_A + p * BN * BK, wn + j * 32, wk * KS + ks, lane);
    };
    auto multiply = [&](int ks) {
        frag (&a)[PA][MI] = fa[ks & 1];
        frag (&b)[PB][NI] = fb[ks & 1];
#pragma unroll
        for (int i = 0; i < MI; ++i)
#pragma unroll
            for (int j = 0; j < NI; ++j) {
                if constexpr (SPLIT3) {
#pragma unroll
                    for (int s = 2; s >= 1; --s)                              // smallest terms first
#pragma unroll
                        for (int p = 0; p <= s; ++p)
                            if (p < PA && s - p < PB) low[i][j] = Mfma<half>::mul(b[s - p][j], a[p][i], low[i][j]);
                }
                acc[i][j] = Mfma<half>::mul(b[0][j], a[0][i], acc[i][j]);
            }
    };
    auto sum = [&](auto edge) {
        sa.init(g.lda, g.lds_scale, m_has, m_has);
        sb.init(g.ldb, 0, n_has, n_has);
        fetch();
        if constexpr (BUFS == 1) {
            for (int t = 0; t < steps; ++t) {
                lds_barrier();
                put(t, lds, edge);
                lds_barrier();
                fetch();
#pragma unroll
                for (int ks = 0; ks < KS; ++ks) { read(lds, ks); multiply(ks); }
            }
        } else {
            // Three parts of LDS go round: step t multiplies part t, the first operands of step t + 1 are read from the next part before
            // step t ends, the third is filled from the registers, which then request the step behind it.  The one barrier of a
            // step is met with operands in hand.
            static_assert(KS % 2 == 0, "the operands' two sets of registers alternate");
            half *cur = lds, *next = lds + LDS_STEP, *third = lds + 2 * LDS_STEP;
            put(0, cur, edge);
            fetch();
            put(1, next, edge);
            fetch();
            lds_barrier();
            read(cur, 0);
            for (int t = 0; t < steps; ++t) {
#pragma unroll
                for (int ks = 0; ks < KS; ++ks) {
                    if (ks + 1 < KS) read(cur, ks + 1);
                    else read(next, 0);
                    multiply(ks);
                    if (ks == 0) {
                        put(t + 2, third, edge);
                        fetch();
                    }
                }
                lds_barrier();
                half* const free = cur;
                cur = next;
                next = third;
                third = free;
            }
        }
    };
    if (steps > 0) {
        if (narrow) {
            for (int t = 0; t < steps; ++t) {
                const int k_has = k_end - k0 - t * BK;
                lds_barrier();
                sa.load_narrow(pa + t * step_a, psc + t * step_sc, g.lda, g.lds_scale, A_ALONG ? m_has : k_has, A_ALONG ? k_has : m_has);
                sb.load_narrow(pb + t * step_b, nullptr, g.ldb, 0, B_ALONG ? n_has : k_has, B_ALONG ? k_has : n_has);
                sa.store(lds);
                sb.store(lds + LDS_A);
                lds_barrier();
#pragma unroll
                for (int ks = 0; ks < KS; ++ks) { read(lds, ks); multiply(ks); }
            }
        } else if ((!A_ALONG && m_has < BM && (m_has & 7)) || (!B_ALONG && n_has < BN && (n_has & 7))) {
            sum(std::true_type());
        } else {
            sum(std::false_type());
        }
    }

    // ---- epilogue: 32 rows of the wave's tile at a time through LDS, so that a lane ends up with 8 columns of a row, the same
    // ones for all its rows.  What it reads besides (bias, residual) is requested two passes ahead, into the registers that the
    // operands have left.
    // With WAVES_K > 1 every wave puts its sums of the whole tile there, and takes a share of the rows.
    constexpr int PASS_ROWS = WAVES_K > 1 ? WM / WAVES_K : 32, PASSES = WAVES_K > 1 ? 1 : MI;
    constexpr int ROWP = WN / 8, STEPS = PASS_ROWS * ROWP / 64, ROWS_PER = 64 / ROWP;
    static_assert(64 % ROWP == 0 && STEPS > 0 && (WAVES_K == 1 || WAVES_M * WAVES_N == 1), "a lane keeps its columns");
    // (the products were taken as B^T A^T: a lane has one row and, in four registers next to each other, four columns)
    auto put_sums = [&](int i, float* to) {
#pragma unroll
        for (int j = 0; j < NI; ++j)
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                f32x4 v;
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    float x = acc[i][j][4 * q + e];
                    if constexpr (SPLIT3) { const float y = x + low[i][j][4 * q + e]; x = __builtin_isfinite(x) ? y : x; }
                    v[e] = x;
                }
                *(f32x4*)(to + (lane & 31) * EPI_LD + j * 32 + q * 8 + (lane >> 5) * 4) = v;
            }
    };
    float* const tile = (float*)smem + wave * EPI_ROWS * EPI_LD;
    const int ccol = (lane % ROWP) * 8, col = n0 + wn + ccol, cvalid = g.N - col;
    float bias[8] = {};
    if constexpr (LAYOUT == LAYOUT_FORWARD) {
        if (g.bias && !rest && cvalid > 0) load8f((const T*)g.bias + (int64_t)group * g.stride_bias + col, cvalid, bias);
    }
    const int row_first = m0 + (WAVES_K > 1 ? wk * PASS_ROWS : wm) + lane / ROWP;
    T res[2][STEPS][8];
    auto fetch_residual = [&](int i) {
        if constexpr (LAYOUT == LAYOUT_FORWARD) {
            if (g.residual && !rest && i < PASSES) {
#pragma unroll
                for (int it = 0; it < STEPS; ++it) {
                    const int row = row_first + i * 32 + it * ROWS_PER;
                    load8((const T*)g.residual + (int64_t)row * g.ldr + col, row < m_end ? cvalid : 0, res[i & 1][it]);
                }
            }
        }
    };
    fetch_residual(0);
    fetch_residual(1);
    __syncthreads();
    if constexpr (WAVES_K > 1) {
#pragma unroll
        for (int i = 0; i < MI; ++i) put_sums(i, tile + i * 32 * EPI_LD);
        __syncthreads();
    }
#pragma unroll
    for (int i = 0; i < PASSES; ++i) {
        const int row0 = row_first + i * 32;
        if constexpr (WAVES_K == 1) {
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
            __builtin_amdgcn_wave_barrier();
            put_sums(i, tile);
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
            __builtin_amdgcn_wave_barrier();
        }
        float v[STEPS][8] = {};
#pragma unroll
        for (int it = 0; it < STEPS; ++it)
#pragma unroll
            for (int w = 0; w < WAVES_K; ++w) {
                const float* from = WAVES_K > 1 ? (const float*)smem + (w * EPI_ROWS + wk * PASS_ROWS) * EPI_LD : tile;
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const f32x4 s = *(const f32x4*)(from + (it * ROWS_PER + lane / ROWP) * EPI_LD + ccol + 4 * h);
#pragma unroll
                    for (int j = 0; j < 4; ++j) v[it][4 * h + j] += s[j];
                }
            }
        if constexpr (LAYOUT == LAYOUT_FORWARD) {
#pragma unroll
            for (int it = 0; it < STEPS; ++it)
#pragma unroll
                for (int j = 0; j < 8; ++j) v[it][j] += bias[j];
            layer_act<T, STEPS * 8>(g.act, &v[0][0]);
            if (rest) {
#pragma unroll
                for (int it = 0; it < STEPS; ++it)
#pragma unroll
                    for (int j = 0; j < 8; ++j) v[it][j] = 0.0f;
            }
        }
#pragma unroll
        for (int it = 0; it < STEPS; ++it) {
            const int row = row0 + it * ROWS_PER, valid = row < m_end ? cvalid : 0;
            if constexpr (LAYOUT == LAYOUT_DW) {
                if (valid <= 0) continue;
                if (slab >= 0) store8(g.slab + ((int64_t)slab * g.M + row) * g.N + col, valid, v[it]);
                else           store8f((T*)g.C + (int64_t)group * g.strideC + (int64_t)row * g.ldc + col, valid, v[it]);
            } else if constexpr (LAYOUT == LAYOUT_DX) {
                if (valid > 0 && !(rest && g.keep_rest)) store8f((T*)g.C + (int64_t)row * g.ldc + col, valid, v[it]);
            } else {
                if (g.q_out) {
                    float a[8];
#pragma unroll
                    for (int j = 0; j < 8; ++j) a[j] = j < valid ? (float)(T)v[it][j] : 0.0f;      // the 8-bit form of the value in T
                    pack_block<T>(a, lane, row < m_end && (col & -PACK_BLOCK) < g.N, g.q_out + (int64_t)row * g.ldq + col,
                                  g.q_scale + (int64_t)row * g.ldq_scale + col / PACK_BLOCK);
                }
                if (valid > 0) {
                    if (g.act_out) store8f((T*)g.act_out + (int64_t)row * g.ld_act + col, valid, v[it]);
                    if (g.residual && !rest) {
#pragma unroll
                        for (int j = 0; j < 8; ++j) v[it][j] += (float)res[i & 1][it][j];
                    }
                    if (!(rest && g.keep_rest)) store8f((T*)g.C + (int64_t)row * g.ldc + col, valid, v[it]);
                }
            }
        }
        fetch_residual(i + 2);
    }
}

template <class T, int LAYOUT, bool PACKED_A, int BM, int BN, int BK, int WAVES_M, int WAVES_N, int WAVES_K, int BUFS>
__global__ void __launch_bounds__(WAVES_M * WAVES_N * WAVES_K * 64, 2) layer_gemm_kernel(GemmArgs g) {
    typedef Product<T, LAYOUT, PACKED_A, BM, BN, BK, WAVES_M, WAVES_N, WAVES_K, BUFS> P;
    __shared__ __attribute__((aligned(16))) char smem[P::SMEM];
    P::run(g, blockIdx.x, smem);
}
// Both gradients of a small layer in one launch: dx in the first workgroups (a multiple of 8, so that the others keep their XCDs), then dW,
// then the join of db's partial sums where dW needs none.  A launch costs 3.5 us of host time, as much as either product of a mini-batch.
template <class T, bool PACKED_A, int BM, int BN, int BK>
__global__ void __launch_bounds__(256, 2) layer_gemm_pair_kernel(GemmArgs dx, GemmArgs dw, JoinPart db, int dx_blocks, int dw_blocks) {
    typedef Product<T, LAYOUT_DX, false, BM, BN, BK, 1, 1, 4, 1> X;
    typedef Product<T, LAYOUT_DW, PACKED_A, BM, BN, BK, 1, 1, 4, 1> W;
    static_assert(X::THREADS == 256 && W::THREADS == 256 && X::SMEM >= (int)sizeof(float[256][8]), "join's threads and memory");
    __shared__ __attribute__((aligned(16))) char smem[X::SMEM > W::SMEM ? X::SMEM : W::SMEM];
    const int block = blockIdx.x;
    if (block < dx_blocks) X::run(dx, block, smem);
    else if (block < dx_blocks + dw_blocks) W::run(dw, block - dx_blocks, smem);
    else join<T>(db, block - dx_blocks - dw_blocks, (float(*)[8])smem);
}

}  // namespace layers
}  // namespace smrt
