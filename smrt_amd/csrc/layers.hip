// The layer operators of the C ABI (include/smrt_hip.h: smrt_dense_*, smrt_layer_norm_*, smrt_pack_rows, smrt_unpack_rows):
// argument checks, workspaces, launches, and the kernels beside the products (layer_gemm.hpp).
#include <algorithm>
#include <initializer_list>
#include <string>
#include "layers.hpp"
#include "../../include/smrt_hip.h"

int smrt_set_error(int code, const std::string& m);      // api.hip: the thread's error text

namespace smrt {
namespace layers {
namespace {

constexpr int64_t MAX_ROWS = 0x7fffffff - 4096, MAX_COLS = 1 << 30, MAX_LD = 1 << 21;     // a product tile of 256 rows spans less than 2^31 bytes
constexpr int MAX_GROUPS = 65535;

// ------------------------------------------------------------------------------------------------ dz = g * act'(a), column sums
// One pass over g (and a): writes dz for the two products that read it, and sums its columns into db on the way (in fp32, from
// the values before they are rounded to T).  dz itself is rounded to T, because the matrix cores take 16-bit operands: two parts of it would
// double both products and the bytes between the launches.  From the result in 64 bits, dx and dW of 32768 x 1024 x 1024 bf16 elu are off by 1.86e-3 of their norm, where rounding them alone
// is 1.66e-3 (sigmoid 2.3e-3; relu and the identity, whose dz is g or 0, 1.66e-3).  The kernels for a few rows multiply dz in fp32 (layer_rows.hpp).  A workgroup has 256 columns of a chunk of DZ_CHUNK rows (chunk_rows), 8 rows x 4 at a time.
// (with chunks of 256 rows, which need no join at 256 x 784 x 450, the step's three launches there took 35 us instead of 21)
constexpr int DZ_CHUNK = 64;
struct DzArgs {
    const void* grad; int64_t ldg;
    const void* a; int64_t lda; const uint8_t* a_scale; int64_t ld_a_scale;
    void* dz; int64_t ld_dz;                       // null: the identity, whose dz is g
    float* part;                                   // [chunks of the larger groups][n]
    void* db; int64_t db_stride;                   // null: not wanted
    const int64_t* ends; int32_t groups, rows, n, act, col_blocks;
};

template <class T, bool PACKED> __global__ void __launch_bounds__(256) dz_kernel(DzArgs p) {
    __shared__ float sums[8][256];
    const int cb = blockIdx.x % p.col_blocks;
    const Chunk chunk = chunk_rows(p.ends, p.groups, p.rows, blockIdx.x / p.col_blocks, DZ_CHUNK);
    if (chunk.group < 0) return;
    const int lo = chunk.r0, hi = chunk.r1;
    int col = cb * 256 + (threadIdx.x & 31) * 8, valid = p.n - col, lead = 0;
    if (!PACKED && valid > 0 && valid < 8 && p.n >= 8) {
        // the piece that the row's end cuts is the row's last 8 columns instead: its first `lead` are its neighbour's too, who
        // stores the same values, and only count in the neighbour's sums
        lead = 8 - valid;
        col -= lead;
        valid = 8;
    }
    float sum[8] = {};
    if (valid > 0) {
        constexpr int U = sizeof(T) == 2 ? 4 : 2;      // rows in flight a thread: their pieces are a round trip to memory
        for (int row = lo + (threadIdx.x >> 5); row < hi; row += 8 * U) {
            // (held as they lie in memory until they are used: as floats they fill the registers, and 40001 x 450 bf16 took 39 us instead of 34)
            T graw[U][8], araw[PACKED ? 1 : U][8];
            u32x2 q[PACKED ? U : 1];
            uint8_t byte[PACKED ? U : 1];
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int r = row + 8 * u, has = r < hi ? valid : 0;
                load8((const T*)p.grad + (int64_t)r * p.ldg + col, has, graw[u]);
                if constexpr (PACKED) {
                    q[u] = u32x2{0u, 0u};
                    byte[u] = 0;
                    if (p.dz && has > 0) {
                        __builtin_memcpy(&q[u], (const int8_t*)p.a + (int64_t)r * p.lda + col, 8);
                        byte[u] = p.a_scale[(int64_t)r * p.ld_a_scale + col / PACK_BLOCK];
                    }
                } else {
                    load8((const T*)p.a + (int64_t)r * p.lda + col, p.dz ? has : 0, araw[u]);
                }
            }
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int r = row + 8 * u;
                float g[8], a[8];
#pragma unroll
                for (int j = 0; j < 8; ++j) g[j] = (float)graw[u][j];
                if (p.dz) {
                    if constexpr (PACKED) unpack8(q[u], unpack_scale(byte[u]), a);
#pragma unroll
                    for (int j = 0; j < 8; ++j) if constexpr (!PACKED) a[j] = (float)araw[u][j];
                    layer_act_grad8(p.act, a, g);
                    if (r < hi) store8f((T*)p.dz + (int64_t)r * p.ld_dz + col, valid, g);
                }
#pragma unroll
                for (int j = 0; j < 8; ++j) sum[j] += g[j];
            }
        }
    }
    if (!p.db) return;
#pragma unroll
    for (int j = 0; j < 8; ++j) if (j >= lead) sums[threadIdx.x >> 5][(threadIdx.x & 31) * 8 + j - lead] = sum[j];
    __syncthreads();
    const int c = cb * 256 + threadIdx.x;
    if (c < p.n) {
        float s = 0.0f;
#pragma unroll
        for (int i = 0; i < 8; ++i) s += sums[i][threadIdx.x];
        if (chunk.slab >= 0) p.part[(int64_t)chunk.slab * p.n + c] = s;
        else ((T*)p.db)[(int64_t)chunk.group * p.db_stride + c] = (T)s;
    }
}

// ------------------------------------------------------------------------------------------------ joining of partial sums (layer_join.hpp)
template <class T> __global__ void __launch_bounds__(256) join_kernel(JoinPart a, JoinPart b) {
    __shared__ float lds[256][8];
    if ((int)blockIdx.x < a.blocks) join<T>(a, blockIdx.x, lds);
    else join<T>(b, blockIdx.x - a.blocks, lds);
}
// fills in share, group_blocks and blocks; false where that is more than a launch takes
bool join_blocks(JoinPart& p) {
    const int64_t slabs = p.rows / ((int64_t)p.chunk * p.groups) + 1, pieces = (int64_t)p.out_rows * ((p.cols + 7) / 8);
    p.share = 1;
    while (p.share < 64 && p.share * 8 < slabs && p.share * pieces * p.groups < 65536) p.share *= 2;
    const int64_t per = 256 / p.share, blocks = (pieces + per - 1) / per;
    if (pieces > 0x7fffffff || blocks * p.groups > 0x3fffffff) return false;
    p.group_blocks = (int32_t)blocks;
    p.blocks = (int32_t)blocks * p.groups;
    return true;
}

// ------------------------------------------------------------------------------------------------ layer norm
// A row lives in the registers of TPR lanes (8 columns each, CH times): one read, the mean, then the squares of the differences
// from it.  Rows go round the workgroups, so a lane keeps its columns: weight and bias are read once, and in the backward
// pass the sums of their gradients stay in registers until the end.
struct NormArgs {
    const void* x; int64_t ldx; const uint8_t* x_scale; int64_t ld_x_scale;
    const void* weight; const void* bias; int32_t w_f32;
    void* y; int64_t ldy; float* mean; float* rstd;
    const void* grad; int64_t ldg; void* dx; int64_t lddx; void* dw; void* db; float* part;
    int32_t rows, n; float eps;
};

// Sums of N values over the TPR lanes of a row.  With more than a wave a row the waves' shares meet in LDS, and all threads of the workgroup take
// part; two parts of LDS take turns, so a sum has one barrier: a part is written again only behind the next sum's, which no wave passes
// before all have read it.
template <int TPR, int THREADS, int N> struct RowSum {
    static constexpr int WAVES = TPR > 64 ? TPR / 64 : 0, SLOTS = WAVES ? THREADS / 64 : 1;
    float (*lds)[SLOTS][N];                          // [2]
    int turn = 0;
    __device__ __forceinline__ void operator()(float (&v)[N]) {
#pragma unroll
        for (int i = 0; i < N; ++i)
#pragma unroll
            for (int d = (TPR < 64 ? TPR : 64) / 2; d; d >>= 1) v[i] += __shfl_xor(v[i], d);
        if constexpr (WAVES > 0) {
            const int wave = threadIdx.x >> 6, first = wave / WAVES * WAVES;
            if ((threadIdx.x & 63) == 0)
#pragma unroll
                for (int i = 0; i < N; ++i) lds[turn][wave][i] = v[i];
            __syncthreads();
#pragma unroll
            for (int i = 0; i < N; ++i) {
                v[i] = 0.0f;
#pragma unroll
                for (int w = 0; w < WAVES; ++w) v[i] += lds[turn][first + w][i];
            }
            turn ^= 1;
        }
    }
};
template <class T> __device__ __forceinline__ void load_weight(const void* p, int w_f32, int col, int valid, float fill, float (&w)[8]) {
#pragma unroll
    for (int j = 0; j < 8; ++j) w[j] = fill;
    if (!p || valid <= 0) return;
    if (w_f32) load8f((const float*)p + col, valid, w);
    else load8f((const T*)p + col, valid, w);
}

template <class T, int TPR, int CH>
__global__ void __launch_bounds__(TPR > 256 ? TPR : 256) norm_forward_kernel(NormArgs p) {
    constexpr int THREADS = TPR > 256 ? TPR : 256, ROWS = THREADS / TPR;
    typedef RowSum<TPR, THREADS, 1> Sum;
    __shared__ float lds[2][Sum::SLOTS][1];
    Sum row_sum = {lds};
    const int lane = threadIdx.x % TPR;
    float w[CH][8], b[CH][8];
#pragma unroll
    for (int c = 0; c < CH; ++c) {
        const int col = (c * TPR + lane) * 8;
        load_weight<T>(p.weight, p.w_f32, col, p.n - col, 1.0f, w[c]);
        load_weight<T>(p.bias, p.w_f32, col, p.n - col, 0.0f, b[c]);
    }
    const float inv_n = 1.0f / (float)p.n;
    for (int64_t row0 = (int64_t)blockIdx.x * ROWS; row0 < p.rows; row0 += (int64_t)gridDim.x * ROWS) {
        const int64_t row = row0 + threadIdx.x / TPR;
        const bool live = row < p.rows;
        float x[CH][8], sum[1] = {};
#pragma unroll
        for (int c = 0; c < CH; ++c) {
            const int col = (c * TPR + lane) * 8;
            load8f((const T*)p.x + row * p.ldx + col, live ? p.n - col : 0, x[c]);
#pragma unroll
            for (int j = 0; j < 8; ++j) sum[0] += x[c][j];
        }
        row_sum(sum);
        const float mean = sum[0] * inv_n;
        float sq[1] = {};
#pragma unroll
        for (int c = 0; c < CH; ++c) {
            const int valid = p.n - (c * TPR + lane) * 8;
#pragma unroll
            for (int j = 0; j < 8; ++j) { x[c][j] -= mean; sq[0] += j < valid ? x[c][j] * x[c][j] : 0.0f; }
        }
        row_sum(sq);
        const float rstd = 1.0f / sqrtf(sq[0] * inv_n + p.eps);
        if (!live) continue;
#pragma unroll
        for (int c = 0; c < CH; ++c) {
            const int col = (c * TPR + lane) * 8;
#pragma unroll
            for (int j = 0; j < 8; ++j) x[c][j] = x[c][j] * rstd * w[c][j] + b[c][j];
            if (p.n - col > 0) store8f((T*)p.y + row * p.ldy + col, p.n - col, x[c]);
        }
        if (lane == 0) { p.mean[row] = mean; p.rstd[row] = rstd; }
    }
}

template <class T, bool PACKED, int TPR, int CH>
__global__ void __launch_bounds__(TPR > 256 ? TPR : 256) norm_backward_kernel(NormArgs p) {
    constexpr int THREADS = TPR > 256 ? TPR : 256, ROWS = THREADS / TPR;
    typedef RowSum<TPR, THREADS, 2> Sum;
    __shared__ float lds[2][Sum::SLOTS][2];
    Sum row_sum = {lds};
    __shared__ float sums[ROWS > 1 ? ROWS : 1][ROWS > 1 ? TPR * 8 : 1];
    const int lane = threadIdx.x % TPR;
    float w[CH][8], dw[CH][8] = {}, db[CH][8] = {};
#pragma unroll
    for (int c = 0; c < CH; ++c) { const int col = (c * TPR + lane) * 8; load_weight<T>(p.weight, p.w_f32, col, p.n - col, 1.0f, w[c]); }
    const float inv_n = 1.0f / (float)p.n;
    // A row is requested while the one before it is worked on; where there are no registers left for that, at its turn (32000 x 2000 bf16, four
    // pieces a lane: 83 us, against 102 with one wave a SIMD).
    constexpr bool EARLY = TPR < 1024 && CH < 4;
    T g_in[CH][8], x_in[PACKED ? 1 : CH][8];
    u32x2 q_in[PACKED ? CH : 1];
    uint8_t scale_in[PACKED ? CH : 1];
    float mean_in, rstd_in;
    auto request = [&](int64_t row) {
        const bool live = row < p.rows;
        mean_in = live ? p.mean[row] : 0.0f;
        rstd_in = live ? p.rstd[row] : 0.0f;
#pragma unroll
        for (int c = 0; c < CH; ++c) {
            const int col = (c * TPR + lane) * 8, valid = live ? p.n - col : 0;
            load8((const T*)p.grad + row * p.ldg + col, valid, g_in[c]);
            if constexpr (PACKED) {
                q_in[c] = u32x2{0u, 0u};
                scale_in[c] = 0;
                if (valid > 0) {
                    __builtin_memcpy(&q_in[c], (const int8_t*)p.x + row * p.ldx + col, 8);
                    scale_in[c] = p.x_scale[row * p.ld_x_scale + col / PACK_BLOCK];
                }
            } else {
                load8((const T*)p.x + row * p.ldx + col, valid, x_in[c]);
            }
        }
    };
    const int64_t first = (int64_t)blockIdx.x * ROWS, stride = (int64_t)gridDim.x * ROWS;
    if (EARLY) request(first + threadIdx.x / TPR);
    for (int64_t row0 = first; row0 < p.rows; row0 += stride) {
        const int64_t row = row0 + threadIdx.x / TPR;
        const bool live = row < p.rows;
        if (!EARLY) request(row);
        const float mean = mean_in, rstd = rstd_in;
        float h[CH][8], g[CH][8], s[2] = {};
#pragma unroll
        for (int c = 0; c < CH; ++c) {
            if constexpr (PACKED) unpack8(q_in[c], unpack_scale(scale_in[c]), h[c]);
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                g[c][j] = (float)g_in[c][j];
                if constexpr (!PACKED) h[c][j] = (float)x_in[c][j];
            }
        }
        if (EARLY) request(row + stride);
#pragma unroll
        for (int c = 0; c < CH; ++c) {
            const int valid = live ? p.n - (c * TPR + lane) * 8 : 0;
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                h[c][j] = j < valid ? (h[c][j] - mean) * rstd : 0.0f;
                dw[c][j] += g[c][j] * h[c][j];
                db[c][j] += g[c][j];
                g[c][j] *= w[c][j];
                s[0] += g[c][j];
                s[1] += g[c][j] * h[c][j];
            }
        }
        row_sum(s);
        const float s1 = s[0] * inv_n, s2 = s[1] * inv_n;
        if (!live || !p.dx) continue;
#pragma unroll
        for (int c = 0; c < CH; ++c) {
            const int col = (c * TPR + lane) * 8;
#pragma unroll
            for (int j = 0; j < 8; ++j) g[c][j] = rstd * (g[c][j] - s1 - h[c][j] * s2);
            if (p.n - col > 0) store8f((T*)p.dx + row * p.lddx + col, p.n - col, g[c]);
        }
    }
    // this workgroup's share of the weight's and the bias's gradient: to `part` [workgroups][2][n], or out at once where it is the only one
#pragma unroll
    for (int which = 0; which < 2; ++which) {
        void* out = which ? p.db : p.dw;
        if (!out) continue;
#pragma unroll
        for (int c = 0; c < CH; ++c) {
            const int col = (c * TPR + lane) * 8, valid = p.n - col;
            float v[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) v[j] = which ? db[c][j] : dw[c][j];
            if constexpr (ROWS > 1) {
                __syncthreads();
#pragma unroll
                for (int j = 0; j < 8; ++j) sums[threadIdx.x / TPR][lane * 8 + j] = v[j];
                __syncthreads();
                if (threadIdx.x >= TPR) continue;
                for (int i = 1; i < ROWS; ++i)
#pragma unroll
                    for (int j = 0; j < 8; ++j) v[j] += sums[i][lane * 8 + j];
            }
            if (valid <= 0) continue;
            if (p.part) store8(p.part + ((int64_t)blockIdx.x * 2 + which) * p.n + col, valid, v);
            else if (p.w_f32) store8((float*)out + col, valid, v);
            else store8f((T*)out + col, valid, v);
        }
    }
}

// ------------------------------------------------------------------------------------------------ the 8-bit form on its own
struct PackArgs { const void* x; int64_t ldx; int8_t* q; int64_t ldq; uint8_t* scale; int64_t ld_scale; int64_t rows; int32_t n; void* out; };

// I: an index type that holds the number of pieces (a 64-bit division costs more than the rest of a piece)
template <class T, class I> __global__ void __launch_bounds__(256) pack_kernel(PackArgs p) {
    const I per_row = (I)((p.n + PACK_BLOCK - 1) / PACK_BLOCK) * 4, total = (I)p.rows * per_row;       // whole blocks: four lanes
    for (I i = (I)blockIdx.x * 256 + threadIdx.x; i < total; i += (I)gridDim.x * 256) {                // stay together
        const I row = i / per_row;
        const int col = (int)(i - row * per_row) * 8;
        float f[8];
        load8f((const T*)p.x + (int64_t)row * p.ldx + col, p.n - col, f);
        pack_block<T>(f, (int)(i & 3), true, p.q + (int64_t)row * p.ldq + col, p.scale + (int64_t)row * p.ld_scale + col / PACK_BLOCK);
    }
}
template <class T, class I> __global__ void __launch_bounds__(256) unpack_kernel(PackArgs p) {
    const I per_row = (I)((p.n + 7) / 8), total = (I)p.rows * per_row;
    for (I i = (I)blockIdx.x * 256 + threadIdx.x; i < total; i += (I)gridDim.x * 256) {
        const I row = i / per_row;
        const int col = (int)(i - row * per_row) * 8;
        u32x2 q;
        __builtin_memcpy(&q, p.q + (int64_t)row * p.ldq + col, 8);
        float f[8];
        unpack8(q, unpack_scale(p.scale[(int64_t)row * p.ld_scale + col / PACK_BLOCK]), f);
        store8f((T*)p.out + (int64_t)row * p.ldx + col, p.n - col, f);
    }
}

// ------------------------------------------------------------------------------------------------ host side
int fail(const char* who, const char* what) { return smrt_set_error(-1, std::string(who) + ": " + what); }
int launched(const char* who, hipError_t e) { return e == hipSuccess ? 0 : smrt_set_error(-2, std::string(who) + ": " + hipGetErrorString(e)); }
int elem_size(int dtype) { return dtype == SMRT_F32 ? 4 : 2; }
int64_t pad(int64_t v, int64_t to) { return (v + to - 1) / to * to; }

int64_t span(int64_t rows, int64_t ld, int64_t cols) { return rows > 0 ? (rows - 1) * ld + cols : 0; }
// What a matrix occupies: `row` bytes every `pitch` bytes (pitch 0: one piece).
struct Span { const void* p; int64_t bytes, pitch, row; };
Span matrix(const void* p, int64_t rows, int64_t ld, int64_t cols, int64_t es) { return {p, span(rows, ld, cols) * es, ld * es, cols * es}; }
Span piece(const void* p, int64_t bytes) { return {p, bytes, 0, bytes}; }
bool overlap(const Span& a, const Span& b) {
    const uintptr_t x = (uintptr_t)a.p, y = (uintptr_t)b.p;
    if (!x || !y || a.bytes <= 0 || a.row <= 0 || b.bytes <= 0 || b.row <= 0 || x >= y + (uintptr_t)b.bytes || y >= x + (uintptr_t)a.bytes) return false;
    if (a.pitch <= 0 || a.pitch != b.pitch) return true;
    // rows of the same pitch may be different columns of one buffer
    const int64_t from_a = (int64_t)((y > x ? y - x : a.pitch - (x - y) % a.pitch) % a.pitch);
    return from_a < a.row || from_a + b.row > a.pitch;
}
// whether an output shares memory with an input or with another output
bool any_overlap(std::initializer_list<Span> outs, std::initializer_list<Span> ins) {
    for (const Span* o = outs.begin(); o != outs.end(); ++o) {
        for (const Span& i : ins) if (overlap(*o, i)) return true;
        for (const Span* q = o + 1; q != outs.end(); ++q) if (overlap(*o, *q)) return true;
    }
    return false;
}

Span weights(const void* p, int64_t groups, int64_t stride, int64_t k, int64_t ld, int64_t n, int64_t es) {
    return groups == 1 ? matrix(p, k, ld, n, es) : piece(p, ((groups - 1) * stride + span(k, ld, n)) * es);
}

// scale bytes of an 8-bit form (null: the matrix is not in 8 bits)
Span scales(const uint8_t* p, int64_t rows, int64_t ld, int64_t n) { return matrix(p, rows, ld, (n + PACK_BLOCK - 1) / PACK_BLOCK, 1); }
// a matrix that an earlier pass kept, of dtype or in 8 bits
Span kept(const void* p, const uint8_t* scale, int64_t rows, int64_t ld, int64_t n, int64_t es) {
    return scale ? matrix(p, rows, ld, pad(n, PACK_BLOCK), 1) : matrix(p, rows, ld, n, es);
}
Span ends_of(const smrt_dense* p) { return piece(p->ends, p->groups * 8); }

int check_dense(const smrt_dense* p, const char* who) {
    if (!p) return fail(who, "null argument");
    if (p->dtype < 0 || p->dtype > SMRT_F16) return fail(who, "dtype must be SMRT_F32, SMRT_BF16 or SMRT_F16");
    if (p->activation < 0 || p->activation > SMRT_ACT_TANH) return fail(who, "bad activation id");
    if (p->rows < 0 || p->rows > MAX_ROWS || p->k < 0 || p->k > MAX_COLS || p->n < 0 || p->n > MAX_COLS) return fail(who, "bad sizes");
    if (p->groups < 1 || p->groups > MAX_GROUPS) return fail(who, "groups must be in [1, 65535]");
    if (p->groups > 1 && !p->ends) return fail(who, "more than one group needs ends");
    if (p->ldx < p->k || p->ldw < p->n) return fail(who, "a leading dimension is below its columns");
    if (p->ldx > MAX_LD || p->ldw > MAX_LD || p->ldg > MAX_LD || p->ld_x_scale > MAX_LD) return fail(who, "a leading dimension is above 2^21");
    if (p->groups > 1 && p->w_stride < span(p->k, p->ldw, p->n)) return fail(who, "the groups' weights overlap");
    if (p->w_stride < 0) return fail(who, "bad sizes");
    if (p->groups > 1 && (p->bias || p->db) && p->bias_stride < p->n) return fail(who, "the groups' biases overlap");
    const bool product = p->rows && p->n && p->k;
    if (product && (!p->x || !p->w)) return fail(who, "null pointer");
    return 0;
}

hipError_t gemm(int dtype, int layout, const GemmPlan& p, const GemmArgs& g, hipStream_t s) {
    return dtype == SMRT_F32 ? layer_gemm_f32(layout, p, g, s) : dtype == SMRT_BF16 ? layer_gemm_bf16(layout, p, g, s) : layer_gemm_f16(layout, p, g, s);
}

hipError_t gemm_pair(int dtype, const GemmArgs& dx, const GemmArgs& dw, const JoinPart& db, hipStream_t s) {
    return dtype == SMRT_F32 ? layer_gemm_f32(dx, dw, db, s) : dtype == SMRT_BF16 ? layer_gemm_bf16(dx, dw, db, s) : layer_gemm_f16(dx, dw, db, s);
}

struct BackwardPlan {
    bool rows, need_dz, need_sum;
    GemmPlan dw;
    int64_t ld_dz, dz_bytes, slab_off, slab_bytes, part_off, part_bytes, total;
};
BackwardPlan plan_backward(const smrt_dense* p) {
    BackwardPlan b = {};
    b.rows = p->rows && p->n && few_rows_backward(p->dtype == SMRT_F32, p->rows, p->k, p->n, p->groups);
    if (b.rows) return b;
    const int64_t es = elem_size(p->dtype), G = p->groups;
    b.need_dz = p->activation != SMRT_ACT_IDENTITY && (p->dx || p->dw || p->db);
    b.need_sum = p->db != nullptr;
    b.ld_dz = pad(p->n, 8);
    b.dz_bytes = b.need_dz ? pad(p->rows * b.ld_dz * es, 256) : 0;
    b.part_bytes = b.need_sum ? pad(max_slabs(p->rows, DZ_CHUNK, G) * p->n * 4, 256) : 0;
    b.dw = plan_gemm(LAYOUT_DW, p->dtype == SMRT_F32, p->rows, p->k, p->n, G);
    b.slab_bytes = p->dw ? pad(max_slabs(p->rows, b.dw.chunk, G) * p->k * p->n * 4, 256) : 0;
    b.slab_off = b.dz_bytes;
    b.part_off = b.slab_off + b.slab_bytes;
    b.total = b.part_off + b.part_bytes;
    return b;
}

template <class F> hipError_t by_type(int dtype, F f) {
    return dtype == SMRT_F32 ? f((float)0) : dtype == SMRT_BF16 ? f((bf16)0.0f) : f((f16)0.0f);
}

hipError_t rows_backward(float, const RowsBackward& r, hipStream_t s) { return layer_gemm_f32(r, s); }
hipError_t rows_backward(bf16, const RowsBackward& r, hipStream_t s) { return layer_gemm_bf16(r, s); }
hipError_t rows_backward(f16, const RowsBackward& r, hipStream_t s) { return layer_gemm_f16(r, s); }

template <class T> hipError_t launch_dz(const DzArgs& d, hipStream_t s) {
    const int64_t blocks = (int64_t)d.col_blocks * max_chunks(d.ends != nullptr, d.rows, DZ_CHUNK, d.groups);
    if (blocks == 0) return hipSuccess;
    if (blocks > 0x7fffffff) return hipErrorInvalidConfiguration;
    if (d.a_scale) hipLaunchKernelGGL((dz_kernel<T, true>), dim3((unsigned)blocks), dim3(256), 0, s, d);
    else hipLaunchKernelGGL((dz_kernel<T, false>), dim3((unsigned)blocks), dim3(256), 0, s, d);
    return hipGetLastError();
}

int norm_blocks(int64_t rows, int rows_per_block, int most) { return (int)std::max<int64_t>(1, std::min<int64_t>((rows + rows_per_block - 1) / rows_per_block, most)); }
constexpr int NORM_MAX_COLS = 1024 * 8 * 4;
// lanes of a row and pieces of a lane, by the row's width
template <bool BACKWARD, class F> hipError_t by_width(int64_t n, F f) {
    if (n <= 64) return f(std::integral_constant<int, 8>(), std::integral_constant<int, 1>());
    if (n <= 128) return f(std::integral_constant<int, 16>(), std::integral_constant<int, 1>());
    if (n <= 256) return f(std::integral_constant<int, 32>(), std::integral_constant<int, 1>());
    if (n <= 512) return f(std::integral_constant<int, 64>(), std::integral_constant<int, 1>());
    if (n <= 1024) return f(std::integral_constant<int, 64>(), std::integral_constant<int, 2>());
    // a wave a row as far as registers go, then two: more waves wait for each other at every row (46700 x 1437 bf16 backward 262 us with four
    // waves a row, 109 with one)
    if (n <= 1536) return f(std::integral_constant<int, 64>(), std::integral_constant<int, 3>());
    if (n <= 2048) return f(std::integral_constant<int, 64>(), std::integral_constant<int, 4>());
    // (20000 x 2500 bf16, two waves a row | four: backward 92 | 122 us, forward, which keeps no sums, 50 | 45)
    if (n <= 4096) return f(std::integral_constant<int, BACKWARD ? 128 : 256>(), std::integral_constant<int, BACKWARD ? 4 : 2>());
    if (n <= 8192) return f(std::integral_constant<int, 256>(), std::integral_constant<int, 4>());
    if (n <= 16384) return f(std::integral_constant<int, 1024>(), std::integral_constant<int, 2>());
    return f(std::integral_constant<int, 1024>(), std::integral_constant<int, 4>());
}
int norm_rows_per_block(int64_t n) { return n <= 64 ? 32 : n <= 128 ? 16 : n <= 256 ? 8 : n <= 2048 ? 4 : n <= 4096 ? 2 : 1; }      // of the backward pass
// Workgroups of the forward pass: four turns each, so that weight and bias are read once for them, where that leaves eight a CU
int norm_forward_blocks(int64_t rows, int per) { return std::max(norm_blocks(rows, per, 2048), norm_blocks(rows, 4 * per, 4096)); }
// Workgroups of the backward pass: four turns each up to two a CU, which with the next row in flight reach the rate of a copy (65536 x
// 1024 bf16: 78 us, with four a CU, whose partial sums are twice as many, 87); one, which needs no join, as long as four turns do.
int norm_backward_blocks(int64_t rows, int64_t n) {
    const int per = norm_rows_per_block(n);
    return rows <= 4 * per ? 1 : norm_blocks(rows, 4 * per, 512);
}

int check_norm(const smrt_layer_norm* p, const char* who) {
    if (!p) return fail(who, "null argument");
    if (p->dtype < 0 || p->dtype > SMRT_F16) return fail(who, "dtype must be SMRT_F32, SMRT_BF16 or SMRT_F16");
    if (p->rows < 0 || p->rows > MAX_ROWS) return fail(who, "bad sizes");
    if (p->n < 1 || p->n > NORM_MAX_COLS) return fail(who, "n must be in [1, 32768]");
    if (p->ldx < p->n) return fail(who, "a leading dimension is below its columns");
    if (p->rows && (!p->x || !p->mean || !p->rstd)) return fail(who, "null pointer");
    return 0;
}
NormArgs norm_args(const smrt_layer_norm* p) {
    NormArgs a = {};
    a.x = p->x; a.ldx = p->ldx; a.x_scale = p->x_scale; a.ld_x_scale = p->ld_x_scale;
    a.weight = p->weight; a.bias = p->bias; a.w_f32 = p->weight_f32 || p->dtype == SMRT_F32;
    a.y = p->y; a.ldy = p->ldy; a.mean = p->mean; a.rstd = p->rstd;
    a.grad = p->grad; a.ldg = p->ldg; a.dx = p->dx; a.lddx = p->lddx; a.dw = p->dw; a.db = p->db;
    a.rows = (int32_t)p->rows; a.n = (int32_t)p->n; a.eps = p->eps;
    return a;
}

int check_pack(const char* who, int dtype, const void* x, int64_t ldx, int64_t rows, int64_t n, const void* q, int64_t ldq, const void* scale, int64_t ld_scale) {
    if (dtype < 0 || dtype > SMRT_F16) return fail(who, "dtype must be SMRT_F32, SMRT_BF16 or SMRT_F16");
    if (rows < 0 || rows > MAX_ROWS || n < 0 || n > MAX_COLS) return fail(who, "bad sizes");
    if (ldx < n || ldq < pad(n, PACK_BLOCK) || ld_scale < (n + PACK_BLOCK - 1) / PACK_BLOCK) return fail(who, "a leading dimension is below its columns");
    if (rows && n && (!x || !q || !scale)) return fail(who, "null pointer");
    if (any_overlap({matrix(x, rows, ldx, n, elem_size(dtype)), matrix(q, rows, ldq, pad(n, PACK_BLOCK), 1), scales((const uint8_t*)scale, rows, ld_scale, n)}, {}))
        return fail(who, "the matrix and its 8-bit form overlap");
    return 0;
}
constexpr int64_t SMALL_INDEX = 0xffffffffll - 256 * 256 * 64;       // an index and the grid's stride stay below 2^32
unsigned grid_of(int64_t items) { return (unsigned)std::max<int64_t>(1, std::min<int64_t>((items + 255) / 256, 256 * 32)); }

}  // namespace
}  // namespace layers
}  // namespace smrt

using namespace smrt::layers;

extern "C" int smrt_dense_forward(const smrt_dense* p, void* hip_stream) {
    const char* who = "smrt_dense_forward";
    if (int rc = check_dense(p, who)) return rc;
    if (p->x_scale) return fail(who, "x must be a matrix of dtype: the forward product does not read the 8-bit form");
    if (p->ldy < p->n || (p->residual && p->ldr < p->n)) return fail(who, "a leading dimension is below its columns");
    if (p->a && (p->a_scale ? p->lda < pad(p->n, PACK_BLOCK) || p->ld_a_scale < (p->n + PACK_BLOCK - 1) / PACK_BLOCK : p->lda < p->n))
        return fail(who, "a leading dimension is below its columns");
    if (p->rows == 0 || p->n == 0) return 0;
    if (!p->y) return fail(who, "null pointer");
    const int64_t es = elem_size(p->dtype);
    const Span y = matrix(p->y, p->rows, p->ldy, p->n, es), residual = matrix(p->residual, p->rows, p->ldr, p->n, es);
    const Span a = kept(p->a, p->a_scale, p->rows, p->lda, p->n, es), a_scale = scales(p->a ? p->a_scale : nullptr, p->rows, p->ld_a_scale, p->n);
    const Span bias = p->groups == 1 ? piece(p->bias, p->n * es) : matrix(p->bias, p->groups, p->bias_stride, p->n, es);
    const bool in_place = p->residual == p->y && p->ldr == p->ldy;
    if (any_overlap({y, a, a_scale}, {matrix(p->x, p->rows, p->ldx, p->k, es), weights(p->w, p->groups, p->w_stride, p->k, p->ldw, p->n, es), bias, ends_of(p),
                                      in_place ? Span{} : residual}))
        return fail(who, "an output overlaps an input or another output (y may only be the residual itself)");
    GemmArgs g = {};
    g.A = p->x; g.lda = p->ldx; g.B = p->w; g.ldb = p->ldw; g.strideB = p->w_stride; g.C = p->y; g.ldc = p->ldy;
    g.bias = p->bias; g.stride_bias = p->bias_stride; g.residual = p->residual; g.ldr = p->ldr;
    if (p->a && p->a_scale) { g.q_out = (int8_t*)p->a; g.ldq = p->lda; g.q_scale = p->a_scale; g.ldq_scale = p->ld_a_scale; }
    else if (p->a) { g.act_out = p->a; g.ld_act = p->lda; }
    g.ends = p->ends; g.groups = p->groups; g.keep_rest = p->keep_rest; g.rows = (int32_t)p->rows;
    g.M = (int32_t)p->rows; g.N = (int32_t)p->n; g.K = (int32_t)p->k; g.act = p->activation;
    return launched(who, gemm(p->dtype, LAYOUT_FORWARD, plan_gemm(LAYOUT_FORWARD, p->dtype == SMRT_F32, p->rows, p->rows, p->n, p->groups, p->k, g.q_out != nullptr), g, (hipStream_t)hip_stream));
}

extern "C" int64_t smrt_dense_backward_workspace(const smrt_dense* p) {
    if (check_dense(p, "smrt_dense_backward_workspace")) return -1;
    return plan_backward(p).total;
}

extern "C" int smrt_dense_backward(const smrt_dense* p, void* workspace, int64_t workspace_bytes, void* hip_stream) {
    const char* who = "smrt_dense_backward";
    if (int rc = check_dense(p, who)) return rc;
    const hipStream_t stream = (hipStream_t)hip_stream;
    const bool packed_a = p->a_scale != nullptr;
    if (p->ldg < p->n || (p->dx && p->lddx < p->k) || (p->dw && p->lddw < p->n)) return fail(who, "a leading dimension is below its columns");
    if (p->x_scale && (p->ldx < pad(p->k, PACK_BLOCK) || p->ld_x_scale < (p->k + PACK_BLOCK - 1) / PACK_BLOCK))
        return fail(who, "a leading dimension is below its columns");
    if (p->dw && p->groups > 1 && p->dw_stride < span(p->k, p->lddw, p->n)) return fail(who, "the groups' weight gradients overlap");
    const BackwardPlan b = plan_backward(p);
    if (p->activation != SMRT_ACT_IDENTITY && p->rows && p->n) {
        if (!p->a) return fail(who, "the activation's value is needed");
        if (packed_a ? p->lda < pad(p->n, PACK_BLOCK) || p->ld_a_scale < (p->n + PACK_BLOCK - 1) / PACK_BLOCK : p->lda < p->n)
            return fail(who, "a leading dimension is below its columns");
    }
    if (p->rows && p->n && !p->grad) return fail(who, "null pointer");
    const int64_t es = elem_size(p->dtype);
    const bool reads_a = p->activation != SMRT_ACT_IDENTITY;
    if (any_overlap({matrix(p->dx, p->rows, p->lddx, p->k, es), weights(p->dw, p->groups, p->dw_stride, p->k, p->lddw, p->n, es),
                     piece(p->db, ((p->groups - 1) * p->bias_stride + p->n) * es), piece(workspace, b.total)},
                    {matrix(p->grad, p->rows, p->ldg, p->n, es), weights(p->w, p->groups, p->w_stride, p->k, p->ldw, p->n, es), ends_of(p),
                     kept(p->x, p->x_scale, p->rows, p->ldx, p->k, es), scales(p->x_scale, p->rows, p->ld_x_scale, p->k),
                     kept(reads_a ? p->a : nullptr, p->a_scale, p->rows, p->lda, p->n, es), scales(reads_a ? p->a_scale : nullptr, p->rows, p->ld_a_scale, p->n)}))
        return fail(who, "an output or the workspace overlaps an input or another output");
    if (b.total > workspace_bytes || (b.total && !workspace)) return fail(who, "the workspace is smaller than smrt_dense_backward_workspace says");
    if (b.rows) {
        RowsBackward r = {};
        r.grad = p->grad; r.ldg = p->ldg; r.a = p->a; r.lda = p->lda; r.a_scale = p->a_scale; r.ld_a_scale = p->ld_a_scale;
        r.x = p->x; r.ldx = p->ldx; r.x_scale = p->x_scale; r.ld_x_scale = p->ld_x_scale; r.w = p->w; r.ldw = p->ldw; r.w_stride = p->w_stride;
        r.dx = p->k ? p->dx : nullptr; r.lddx = p->lddx; r.dw = p->k ? p->dw : nullptr; r.lddw = p->lddw; r.dw_stride = p->dw_stride; r.db = p->db; r.db_stride = p->bias_stride;
        r.ends = p->ends; r.groups = p->groups; r.keep_rest = p->keep_rest; r.rows = (int32_t)p->rows; r.k = (int32_t)p->k; r.n = (int32_t)p->n; r.act = p->activation;
        const int32_t tiles_k = (int32_t)((p->k + 63) / 64);
        r.dx_blocks = r.dx ? r.rows * tiles_k : 0;
        r.tiles_k = r.dw || r.dx ? tiles_k : 1;
        r.tiles_n = (int32_t)((p->n + 63) / 64);
        return launched(who, by_type(p->dtype, [&](auto t) { return rows_backward(t, r, stream); }));
    }
    char* const ws = (char*)workspace;
    const void* dz = p->grad;
    int64_t ld_dz = p->ldg;
    if (p->n && (b.need_dz || b.need_sum)) {
        DzArgs d = {};
        d.grad = p->grad; d.ldg = p->ldg; d.a = p->a; d.lda = p->lda;
        d.a_scale = b.need_dz ? p->a_scale : nullptr; d.ld_a_scale = p->ld_a_scale;
        if (b.need_dz) { d.dz = ws; d.ld_dz = b.ld_dz; dz = ws; ld_dz = b.ld_dz; }
        d.part = (float*)(ws + b.part_off); d.db = p->db; d.db_stride = p->bias_stride;
        d.ends = p->ends; d.groups = p->groups; d.rows = (int32_t)p->rows; d.n = (int32_t)p->n; d.act = p->activation;
        d.col_blocks = (int32_t)((p->n + 255) / 256);
        if (hipError_t e = by_type(p->dtype, [&](auto t) { return launch_dz<decltype(t)>(d, stream); }); e != hipSuccess) return launched(who, e);
    }
    GemmArgs x = {}, w = {};
    x.ends = w.ends = p->ends; x.groups = w.groups = p->groups; x.keep_rest = p->keep_rest; x.rows = w.rows = (int32_t)p->rows;
    x.A = dz; x.lda = ld_dz; x.B = p->w; x.ldb = p->ldw; x.strideB = p->w_stride; x.C = p->dx; x.ldc = p->lddx;
    x.M = (int32_t)p->rows; x.N = (int32_t)p->k; x.K = (int32_t)p->n;
    w.A = p->x; w.lda = p->ldx; w.A_scale = p->x_scale; w.lds_scale = p->ld_x_scale; w.B = dz; w.ldb = ld_dz;
    w.C = p->dw; w.ldc = p->lddw; w.strideC = p->dw_stride; w.slab = (float*)(ws + b.slab_off);
    w.M = (int32_t)p->k; w.N = (int32_t)p->n; w.K = (int32_t)p->rows; w.chunk = b.dw.chunk;
    const bool dx = p->dx && p->rows && p->k, dw = p->dw && p->k && p->n;
    const GemmPlan dx_plan = plan_gemm(LAYOUT_DX, p->dtype == SMRT_F32, p->rows, p->rows, p->k, p->groups);
    // one group with exactly one chunk has nothing to join; groups may be empty or larger
    JoinPart jw = {}, jb = {};
    if (dw && !(p->groups == 1 && !p->ends && p->rows > 0 && p->rows <= b.dw.chunk)) {
        jw = {(const float*)(ws + b.slab_off), p->k * p->n, p->ends, p->groups, (int32_t)p->rows, b.dw.chunk, (int32_t)p->k, (int32_t)p->n, p->dw, p->lddw,
              p->dw_stride, false};
        if (!join_blocks(jw)) return fail(who, "the weight gradient is too large");
    }
    if (p->db && p->n && !(p->groups == 1 && !p->ends && p->rows > 0 && p->rows <= DZ_CHUNK)) {
        jb = {(const float*)(ws + b.part_off), p->n, p->ends, p->groups, (int32_t)p->rows, DZ_CHUNK, 1, (int32_t)p->n, p->db, 0, p->bias_stride, false};
        if (!join_blocks(jb)) return fail(who, "the bias gradient is too large");
    }
    hipError_t e = hipSuccess;
    if (dx && dw && dx_plan.tile == TILE_SMALL && b.dw.tile == TILE_SMALL) {
        // where dW has nothing to join, db's join, whose sums are there already, goes along
        e = gemm_pair(p->dtype, x, w, jw.blocks ? JoinPart{} : jb, stream);
        if (!jw.blocks) jb.blocks = 0;
    } else {
        if (dx) e = gemm(p->dtype, LAYOUT_DX, dx_plan, x, stream);
        if (dw && e == hipSuccess) e = gemm(p->dtype, LAYOUT_DW, b.dw, w, stream);
    }
    if (e != hipSuccess) return launched(who, e);
    if (jw.blocks + jb.blocks == 0) return 0;
    return launched(who, by_type(p->dtype, [&](auto t) {
        hipLaunchKernelGGL((join_kernel<decltype(t)>), dim3(jw.blocks + jb.blocks), dim3(256), 0, stream, jw, jb);
        return hipGetLastError();
    }));
}

extern "C" int smrt_layer_norm_forward(const smrt_layer_norm* p, void* hip_stream) {
    const char* who = "smrt_layer_norm_forward";
    if (int rc = check_norm(p, who)) return rc;
    if (p->x_scale) return fail(who, "x must be a matrix of dtype: the forward pass does not read the 8-bit form");
    if (p->ldy < p->n) return fail(who, "a leading dimension is below its columns");
    if (p->rows == 0) return 0;
    if (!p->y) return fail(who, "null pointer");
    if (!(p->eps >= 0.0f)) return fail(who, "eps must be >= 0");
    const int64_t es = elem_size(p->dtype);
    const Span x = matrix(p->x, p->rows, p->ldx, p->n, es);
    if ((p->x != p->y || p->ldx != p->ldy) && overlap(matrix(p->y, p->rows, p->ldy, p->n, es), x))
        return fail(who, "y overlaps x (it may only be x itself)");
    const int64_t ws = p->n * (p->weight_f32 ? 4 : es);
    const Span mean = piece(p->mean, p->rows * 4), rstd = piece(p->rstd, p->rows * 4);
    if (any_overlap({matrix(p->y, p->rows, p->ldy, p->n, es), mean, rstd}, {piece(p->weight, ws), piece(p->bias, ws)}) || any_overlap({mean, rstd}, {x}))
        return fail(who, "an output overlaps an input or another output");
    const NormArgs a = norm_args(p);
    return launched(who, by_type(p->dtype, [&](auto t) {
        return by_width<false>(p->n, [&](auto tpr, auto ch) {
            constexpr int TPR = decltype(tpr)::value, THREADS = TPR > 256 ? TPR : 256;
            hipLaunchKernelGGL((norm_forward_kernel<decltype(t), TPR, decltype(ch)::value>), dim3(norm_forward_blocks(p->rows, THREADS / TPR)), dim3(THREADS), 0,
                               (hipStream_t)hip_stream, a);
            return hipGetLastError();
        });
    }));
}

extern "C" int64_t smrt_layer_norm_backward_workspace(const smrt_layer_norm* p) {
    if (check_norm(p, "smrt_layer_norm_backward_workspace")) return -1;
    const int blocks = norm_backward_blocks(p->rows, p->n);
    return blocks > 1 && (p->dw || p->db) ? (int64_t)blocks * 2 * p->n * 4 : 0;
}

extern "C" int smrt_layer_norm_backward(const smrt_layer_norm* p, void* workspace, int64_t workspace_bytes, void* hip_stream) {
    const char* who = "smrt_layer_norm_backward";
    if (int rc = check_norm(p, who)) return rc;
    const hipStream_t stream = (hipStream_t)hip_stream;
    if (p->ldg < p->n || (p->dx && p->lddx < p->n)) return fail(who, "a leading dimension is below its columns");
    if (p->x_scale && (p->ldx < pad(p->n, PACK_BLOCK) || p->ld_x_scale < (p->n + PACK_BLOCK - 1) / PACK_BLOCK))
        return fail(who, "a leading dimension is below its columns");
    if (p->rows && !p->grad) return fail(who, "null pointer");
    const int64_t need = smrt_layer_norm_backward_workspace(p);
    const int64_t es = elem_size(p->dtype), ws = p->n * (p->weight_f32 ? 4 : es);
    if (any_overlap({matrix(p->dx, p->rows, p->lddx, p->n, es), piece(p->dw, ws), piece(p->db, ws), piece(workspace, need)},
                    {matrix(p->grad, p->rows, p->ldg, p->n, es), kept(p->x, p->x_scale, p->rows, p->ldx, p->n, es), scales(p->x_scale, p->rows, p->ld_x_scale, p->n), piece(p->weight, ws),
                     piece(p->mean, p->rows * 4), piece(p->rstd, p->rows * 4)}))
        return fail(who, "an output or the workspace overlaps an input or another output");
    if (need > workspace_bytes || (need && !workspace)) return fail(who, "the workspace is smaller than smrt_layer_norm_backward_workspace says");
    NormArgs a = norm_args(p);
    const int blocks = norm_backward_blocks(p->rows, p->n);
    a.part = need ? (float*)workspace : nullptr;
    hipError_t e = by_type(p->dtype, [&](auto t) {
        return by_width<true>(p->n, [&](auto tpr, auto ch) {
            constexpr int TPR = decltype(tpr)::value, CH = decltype(ch)::value, THREADS = TPR > 256 ? TPR : 256;
            if (p->x_scale) hipLaunchKernelGGL((norm_backward_kernel<decltype(t), true, TPR, CH>), dim3(blocks), dim3(THREADS), 0, stream, a);
            else hipLaunchKernelGGL((norm_backward_kernel<decltype(t), false, TPR, CH>), dim3(blocks), dim3(THREADS), 0, stream, a);
            return hipGetLastError();
        });
    });
    if (e == hipSuccess && a.part) {
        // slabs of 2 n: the weight's half, then the bias's
        JoinPart jw = {}, jb = {};
        const int32_t n = (int32_t)p->n;
        if (p->dw) { jw = {a.part, 2 * p->n, nullptr, 1, blocks, 1, 1, n, p->dw, 0, 0, a.w_f32}; join_blocks(jw); }
        if (p->db) { jb = {a.part + n, 2 * p->n, nullptr, 1, blocks, 1, 1, n, p->db, 0, 0, a.w_f32}; join_blocks(jb); }
        e = by_type(p->dtype, [&](auto t) {
            hipLaunchKernelGGL((join_kernel<decltype(t)>), dim3(jw.blocks + jb.blocks), dim3(256), 0, stream, jw, jb);
            return hipGetLastError();
        });
    }
    return launched(who, e);
}

extern "C" int smrt_pack_rows(int32_t dtype, const void* x, int64_t ldx, int64_t rows, int64_t n, int8_t* q, int64_t ldq, uint8_t* scale,
                              int64_t ld_scale, void* hip_stream) {
    const char* who = "smrt_pack_rows";
    if (int rc = check_pack(who, dtype, x, ldx, rows, n, q, ldq, scale, ld_scale)) return rc;
    if (rows == 0 || n == 0) return 0;
    const PackArgs a = {x, ldx, q, ldq, scale, ld_scale, rows, (int32_t)n, nullptr};
    return launched(who, by_type(dtype, [&](auto t) {
        const int64_t pieces = rows * (pad(n, PACK_BLOCK) / 8);
        if (pieces < SMALL_INDEX) hipLaunchKernelGGL((pack_kernel<decltype(t), uint32_t>), dim3(grid_of(pieces)), dim3(256), 0, (hipStream_t)hip_stream, a);
        else hipLaunchKernelGGL((pack_kernel<decltype(t), uint64_t>), dim3(grid_of(pieces)), dim3(256), 0, (hipStream_t)hip_stream, a);
        return hipGetLastError();
    }));
}

extern "C" int smrt_unpack_rows(int32_t dtype, const int8_t* q, int64_t ldq, const uint8_t* scale, int64_t ld_scale, int64_t rows, int64_t n,
                                void* x, int64_t ldx, void* hip_stream) {
    const char* who = "smrt_unpack_rows";
    if (int rc = check_pack(who, dtype, x, ldx, rows, n, q, ldq, scale, ld_scale)) return rc;
    if (rows == 0 || n == 0) return 0;
    const PackArgs a = {nullptr, ldx, (int8_t*)q, ldq, (uint8_t*)scale, ld_scale, rows, (int32_t)n, x};
    return launched(who, by_type(dtype, [&](auto t) {
        const int64_t pieces = rows * ((n + 7) / 8);
        if (pieces < SMALL_INDEX) hipLaunchKernelGGL((unpack_kernel<decltype(t), uint32_t>), dim3(grid_of(pieces)), dim3(256), 0, (hipStream_t)hip_stream, a);
        else hipLaunchKernelGGL((unpack_kernel<decltype(t), uint64_t>), dim3(grid_of(pieces)), dim3(256), 0, (hipStream_t)hip_stream, a);
        return hipGetLastError();
    }));
}
