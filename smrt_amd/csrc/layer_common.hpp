// Shared by the layer operators (dense, layer norm, 8-bit checkpoints): element types, activations, groups of rows.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>
#include <type_traits>
#include "device_utils.hpp"

namespace smrt {
namespace layers {

typedef __bf16 bf16;
typedef _Float16 f16;
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef short s16x8 __attribute__((ext_vector_type(8)));

constexpr int PACK_BLOCK = 32;            // columns of a row that share one scale byte of the 8-bit form

// Rows move in pieces of 8 columns.  The tensors are a user's: rows may start at any element, so the pieces are read and
// written as memory of the element's own alignment (global loads and stores take any address on gfx950 at the same rate; 16
// bytes stay one instruction).  The piece that a row's end cuts is made of four, two and one elements, whichever there are: a lane of
// every wave has one, and eight single elements took longer than the rest of the row (450 columns against 448).
typedef uint32_t Words4 __attribute__((ext_vector_type(4), aligned(2), may_alias));
typedef uint32_t Words2 __attribute__((ext_vector_type(2), aligned(2), may_alias));
typedef uint32_t Words1 __attribute__((aligned(2), may_alias));
typedef uint16_t Halves1 __attribute__((may_alias));

template <class T> __device__ __forceinline__ void load8(const T* __restrict__ p, int valid, T (&v)[8]) {
    const char* const at = (const char*)p;
    u32x4 lo = {0u, 0u, 0u, 0u}, up = {0u, 0u, 0u, 0u};
    if (valid >= 8) {
        lo = *(const Words4*)at;
        if constexpr (sizeof(T) == 4) up = *(const Words4*)(at + 16);
    } else if (valid > 0) {
        const bool four = valid & 4, two = valid & 2, one = valid & 1;
        if constexpr (sizeof(T) == 4) {
            u32x4 a = {0u, 0u, 0u, 0u};
            u32x2 b = {0u, 0u};
            uint32_t c = 0u;
            if (four) a = *(const Words4*)at;
            if (two) b = *(const Words2*)(at + (four ? 16 : 0));
            if (one) c = *(const Words1*)(at + (four ? 16 : 0) + (two ? 8 : 0));
            const u32x4 rest = {two ? b[0] : c, two ? b[1] : 0u, two ? c : 0u, 0u};
            lo = four ? a : rest;
            up = four ? rest : u32x4{0u, 0u, 0u, 0u};
        } else {
            u32x2 a = {0u, 0u};
            uint32_t b = 0u, c = 0u;
            if (four) a = *(const Words2*)at;
            if (two) b = *(const Words1*)(at + (four ? 8 : 0));
            if (one) c = *(const Halves1*)(at + (four ? 8 : 0) + (two ? 4 : 0));
            const uint32_t r0 = two ? b : c, r1 = two ? c : 0u;
            lo = u32x4{four ? a[0] : r0, four ? a[1] : r1, four ? r0 : 0u, four ? r1 : 0u};
        }
    }
    __builtin_memcpy(v, &lo, 16);
    if constexpr (sizeof(T) == 4) __builtin_memcpy((char*)v + 16, &up, 16);
}
template <class T> __device__ __forceinline__ void store8(T* p, int valid, const T (&v)[8]) {
    char* const at = (char*)p;
    u32x4 lo, up = {0u, 0u, 0u, 0u};
    __builtin_memcpy(&lo, v, 16);
    if constexpr (sizeof(T) == 4) __builtin_memcpy(&up, (const char*)v + 16, 16);
    if (valid >= 8) {
        *(Words4*)at = lo;
        if constexpr (sizeof(T) == 4) *(Words4*)(at + 16) = up;
    } else if (valid > 0) {
        const bool four = valid & 4, two = valid & 2, one = valid & 1;
        if constexpr (sizeof(T) == 4) {
            const u32x4 rest = four ? up : lo;
            if (four) *(Words4*)at = lo;
            if (two) *(Words2*)(at + (four ? 16 : 0)) = u32x2{rest[0], rest[1]};
            if (one) *(Words1*)(at + (four ? 16 : 0) + (two ? 8 : 0)) = two ? rest[2] : rest[0];
        } else {
            const uint32_t r0 = four ? lo[2] : lo[0], r1 = four ? lo[3] : lo[1];
            if (four) *(Words2*)at = u32x2{lo[0], lo[1]};
            if (two) *(Words1*)(at + (four ? 8 : 0)) = r0;
            if (one) *(Halves1*)(at + (four ? 8 : 0) + (two ? 4 : 0)) = (uint16_t)(two ? r1 : r0);
        }
    }
}
template <class T> __device__ __forceinline__ void load8f(const T* __restrict__ p, int valid, float (&f)[8]) {
    T v[8];
    load8(p, valid, v);
#pragma unroll
    for (int j = 0; j < 8; ++j) f[j] = (float)v[j];
}
template <class T> __device__ __forceinline__ void store8f(T* p, int valid, const float (&f)[8]) {
    T v[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = (T)f[j];
    store8(p, valid, v);
}

// Activations.  Unlike act_fwd these hand a NaN on (relu of the training kernels is fmaxf, which drops it: there the loss
// reports it; here the value is the user's).
// e^v - 1 for v <= 0 in a dozen instructions (the library's takes several times that, which no memory traffic hides in a
// product's epilogue): near 0, where the difference would cancel, the exponential's series, elsewhere the exponential itself, whose
// error stays within a few units of 2^-24.  For fp32 the series goes to v^7 (next term below 2^-28 of v at 0.3); a result that is
// rounded to 16 bits needs it to v^3 only (next term below 2^-19 of v at 0.03, the difference's error 2^-18 of it).
template <class T> __device__ __forceinline__ float fast_expm1(float v) {
    const float e = __builtin_amdgcn_exp2f(1.4426950408889634f * v) - 1.0f;
    if constexpr (sizeof(T) == 2) {
        const float s = fmaf(v, 1.0f / 6.0f, 0.5f);
        return v > -0.03f ? fmaf(s * v, v, v) : e;
    } else {
        float s = fmaf(v, 1.0f / 5040.0f, 1.0f / 720.0f);
        s = fmaf(s, v, 1.0f / 120.0f);
        s = fmaf(s, v, 1.0f / 24.0f);
        s = fmaf(s, v, 1.0f / 6.0f);
        s = fmaf(s, v, 0.5f);
        return v > -0.3f ? fmaf(s * v, v, v) : e;
    }
}
// tanh |v| = -m / (m + 2) with m = e^(-2 |v|) - 1
template <class T> __device__ __forceinline__ float fast_tanh(float v) {
    const float m = fast_expm1<T>(-2.0f * fabsf(v));
    return copysignf(-m * __builtin_amdgcn_rcpf(m + 2.0f), v);
}

template <class T, int N> __device__ __forceinline__ void layer_act(int act, float* v) {
    switch (act) {
        case ACT_SIGMOID:
#pragma unroll
            for (int j = 0; j < N; ++j) v[j] = fast_sigmoid(v[j]);
            break;
        case ACT_TANH:
#pragma unroll
            for (int j = 0; j < N; ++j) v[j] = fast_tanh<T>(v[j]);
            break;
        case ACT_RELU:
#pragma unroll
            for (int j = 0; j < N; ++j) v[j] = v[j] < 0.0f ? 0.0f : v[j];
            break;
        case ACT_ELU:
#pragma unroll
            for (int j = 0; j < N; ++j) v[j] = v[j] > 0.0f ? v[j] : fast_expm1<T>(v[j]);
            break;
        default: break;
    }
}
// g := g * d act(z) / dz, from a = act(z); a NaN in a is handed on
__device__ __forceinline__ void layer_act_grad8(int act, const float (&a)[8], float (&g)[8]) {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        const float nan = a[j] != a[j] ? a[j] : 0.0f;
        switch (act) {
            case ACT_SIGMOID: g[j] *= a[j] * (1.0f - a[j]); break;
            case ACT_TANH:    g[j] *= 1.0f - a[j] * a[j]; break;
            case ACT_RELU:    g[j] = a[j] > 0.0f ? g[j] : nan; break;
            case ACT_ELU:     g[j] = a[j] >= 0.0f ? g[j] : g[j] * (a[j] + 1.0f); break;
            default:          break;
        }
    }
}

// ---- the 8-bit form.  32 columns of a row share 2^e; a value is a whole number q in [-127, 127] times 2^e, e the smallest
// exponent with max|x| <= 127 * 2^e.  q * 2^e has 7 significant bits: EXACT in bf16 (and, with e >= -24, in f16), so what the
// backward products read is the value itself, with no second rounding.  The scale byte is e + 127; 255 marks a block that
// held an infinity or a NaN: all its values stand for NaN.
template <class T> struct PackRange { static constexpr int lo = -126, hi = 122; };      // 64 * 2^122 is 2^128
template <> struct PackRange<f16> { static constexpr int lo = -24, hi = 10; };          // 64 * 2^10 is 2^16
// scale byte for the largest magnitude of a block (given as the bits of |x|, where NaN is above infinity above all numbers)
template <class T> __device__ __forceinline__ int pack_scale(uint32_t top_bits) {
    if (top_bits >= 0x7f800000u) return 255;
    int e = (int)(top_bits >> 23) - 127 - 6;                                  // top in [64, 128) * 2^e
    if ((top_bits & 0x7fffffu) > 0x7e0000u) ++e;                              // over 127 * 2^e
    return (e < PackRange<T>::lo ? PackRange<T>::lo : e) + 127;
}
// bits of the largest magnitude of N values
template <int N> __device__ __forceinline__ uint32_t pack_top(const float* f) {
    uint32_t top = 0;
#pragma unroll
    for (int j = 0; j < N; ++j) { const uint32_t b = __float_as_uint(f[j]) & 0x7fffffffu; top = top > b ? top : b; }
    return top;
}
// the eight q of a block with that scale byte.  x * 2^-e is exact, and adding 1.5 * 2^23 rounds it to a whole number, halves to
// even, whose two's complement is the low byte of the sum's bits.  |q| <= 127 by the choice of e.
template <class T> __device__ __forceinline__ u32x2 pack_bytes(const float (&f)[8], int byte) {
    const float magic = 12582912.0f;
    // 2^-e, a normal number for e in [-126, 122]; a block that stands for NaN has q = 0
    const float inv = byte == 255 ? 0.0f : __uint_as_float((uint32_t)(254 - byte) << 23);
    uint32_t b[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) b[j] = __float_as_uint(fmaf(f[j], inv, magic));
    if (byte == PackRange<T>::hi + 127) {                                     // 64 * 2^hi would be an infinity of T
#pragma unroll
        for (int j = 0; j < 8; ++j) b[j] = __float_as_uint(fminf(fmaxf(__uint_as_float(b[j]), magic - 63.0f), magic + 63.0f));
    }
    u32x2 w;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        const uint32_t lo = __builtin_amdgcn_perm(b[4 * h + 1], b[4 * h], 0x0c0c0400u), up = __builtin_amdgcn_perm(b[4 * h + 3], b[4 * h + 2], 0x04000c0cu);
        w[h] = byte == 255 ? 0u : lo | up;
    }
    return w;
}
__device__ __forceinline__ float unpack_scale(int byte) {
    return byte == 255 ? __uint_as_float(0x7fc00000u) : __uint_as_float((uint32_t)byte << 23);
}
__device__ __forceinline__ void unpack8(u32x2 q, float scale, float (&f)[8]) {
#pragma unroll
    for (int j = 0; j < 8; ++j) f[j] = (float)((int)(q[j / 4] << (24 - 8 * (j % 4))) >> 24) * scale;
}
// Four neighbouring lanes hold a block (8 columns each; columns behind the row's end are zero): writes its 8 bytes of q and,
// from the first of the four, the scale byte.
template <class T> __device__ __forceinline__ void pack_block(const float (&f)[8], int lane, bool store, int8_t* q, uint8_t* scale) {
    uint32_t top = pack_top<8>(f);
#pragma unroll
    for (int d = 1; d <= 2; d <<= 1) { const uint32_t o = (uint32_t)__shfl_xor((int)top, d); top = top > o ? top : o; }
    const int byte = pack_scale<T>(top);
    const u32x2 w = pack_bytes<T>(f, byte);
    if (!store) return;
    __builtin_memcpy(q, &w, 8);
    if ((lane & 3) == 0) *scale = (uint8_t)byte;
}

// ---- groups of rows.  ends[g] is where group g's rows end (it begins where g - 1 ends, group 0 at row 0).  The array is
// device memory that the host never sees, so every kernel makes it sound for itself: an end is clamped to [0, rows] and
// never lies before an earlier one.  Whatever the array holds, groups are then disjoint and inside the matrix.
// All 64 lanes of a wave call these together; the results are the same in all lanes.
struct RowSpan { int group; int r0, r1; };      // group -1: rows that no group has; r0 >= r1: nothing

__device__ __forceinline__ int clamp_end(const int64_t* __restrict__ ends, int g, int n_groups, int rows) {
    if (g >= n_groups) return 0;
    const int64_t e = ends[g];
    return e < 0 ? 0 : e > rows ? rows : (int)e;
}
__device__ __forceinline__ int wave_max_scan(int v) {
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) { const int o = __shfl_up(v, d); if ((int)(threadIdx.x & 63) >= d && o > v) v = o; }
    return v;
}
__device__ __forceinline__ int wave_sum_scan(int v) {
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) { const int o = __shfl_up(v, d); if ((int)(threadIdx.x & 63) >= d) v += o; }
    return v;
}
// Calls f(group, begin, end) for 64 groups at a time, a group a lane, in order, until f returns true.  Lanes behind the last group see an empty one.
template <class F> __device__ __forceinline__ int walk_groups(const int64_t* __restrict__ ends, int n_groups, int rows, F f) {
    int end0 = 0;
    for (int base = 0; base < n_groups; base += 64) {
        const int g = base + (int)(threadIdx.x & 63);
        int e = wave_max_scan(clamp_end(ends, g, n_groups, rows));
        e = e > end0 ? e : end0;
        int begin = __shfl_up(e, 1);
        if ((threadIdx.x & 63) == 0) begin = end0;
        if (f(g, begin, e)) return end0;
        end0 = __shfl(e, 63);
    }
    return end0;
}
// rows of group g: it begins at the largest of the ends before its own, a maximum that no lane waits for another in (a workgroup for each of
// thousands of groups spent most of its time in the scans of walk_groups)
__device__ __forceinline__ RowSpan group_rows(const int64_t* __restrict__ ends, int n_groups, int rows, int group) {
    int begin = 0;
#pragma unroll 4
    for (int g = (int)(threadIdx.x & 63); g < group; g += 64) { const int e = clamp_end(ends, g, n_groups, rows); begin = e > begin ? e : begin; }
#pragma unroll
    for (int d = 32; d; d >>= 1) { const int o = __shfl_xor(begin, d); begin = o > begin ? o : begin; }
    const int end = clamp_end(ends, group, n_groups, rows);
    return {group, begin, end > begin ? end : begin};
}
// the group of a row, -1 for none
__device__ __forceinline__ int row_group(const int64_t* __restrict__ ends, int n_groups, int rows, int row) {
    int group = -1;
    walk_groups(ends, n_groups, rows, [&](int g, int begin, int end) {
        const unsigned long long hit = __ballot(begin <= row && row < end);
        if (hit) group = __shfl(g, __builtin_ctzll(hit));
        return hit != 0;
    });
    return group;
}
// the t-th tile of `tile` rows, where no tile crosses from one group into the next; behind the last group come the rows
// that no group has
__device__ __forceinline__ RowSpan tile_rows(const int64_t* __restrict__ ends, int n_groups, int rows, int t, int tile) {
    RowSpan s = {-1, 0, rows};
    int tiles0 = 0;
    const int last = walk_groups(ends, n_groups, rows, [&](int g, int begin, int end) {
        const int own = (end - begin + tile - 1) / tile, sum = tiles0 + wave_sum_scan(own);
        const unsigned long long hit = __ballot(t < sum);
        if (hit) {
            const int f = __builtin_ctzll(hit);
            s = {__shfl(g, f), __shfl(begin, f) + (t - __shfl(sum - own, f)) * tile, __shfl(end, f)};
        }
        tiles0 = __shfl(sum, 63);
        return hit != 0;
    });
    if (s.group < 0) {
        const long r0 = (long)last + (long)(t - tiles0) * tile;
        s.r0 = r0 < rows ? (int)r0 : rows;
    }
    return s;
}

// how many tiles there are, the ones of rows that no group has among them
__device__ __forceinline__ int count_tiles(const int64_t* __restrict__ ends, int n_groups, int rows, int tile) {
    if (!ends) return (rows + tile - 1) / tile;
    int n = 0;
    const int last = walk_groups(ends, n_groups, rows, [&](int, int begin, int end) { n += (end - begin + tile - 1) / tile; return false; });
#pragma unroll
    for (int d = 32; d; d >>= 1) n += __shfl_xor(n, d);
    return n + (rows - last + tile - 1) / tile;
}

// ---- sums over a group's rows.  The rows are cut into chunks of `chunk`, none across groups, so that a large group does not
// make one workgroup late.  A group of one chunk has its result written at once; the chunks of the larger groups are numbered one
// after the other, each fills the slab of its number, and the join adds a group's slabs in their order.  A group
// without rows has no chunk, and zeros from the join.  Larger groups have at most rows / chunk + min(groups, rows / chunk) chunks.
struct Chunk { int group, r0, r1, slab; };       // slab -1: the group's only chunk; group -1: nothing
struct Slabs { int first, count; };              // count 0: no rows, 1: written at once

// chunk c: those of the larger groups first, then the groups of one chunk
__device__ __forceinline__ Chunk chunk_rows(const int64_t* __restrict__ ends, int n_groups, int rows, int c, int chunk) {
    Chunk r = {-1, 0, 0, -1};
    if (!ends) {
        const long r0 = (long)c * chunk;
        if (r0 < rows) r = {0, (int)r0, rows - r0 > chunk ? (int)r0 + chunk : rows, rows > chunk ? c : -1};
        return r;
    }
    int before = 0;
#pragma unroll 1
    for (int single = 0; single < 2 && r.group < 0; ++single)
        walk_groups(ends, n_groups, rows, [&](int g, int begin, int end) {
            const int n = end - begin, own = single ? (n > 0 && n <= chunk) : n > chunk ? (n - 1) / chunk + 1 : 0;
            const int sum = before + wave_sum_scan(own);
            const unsigned long long hit = __ballot(c < sum);
            if (hit) {
                const int f = __builtin_ctzll(hit);
                const int r0 = __shfl(begin, f) + (c - __shfl(sum - own, f)) * chunk, r1 = __shfl(end, f);
                r = {__shfl(g, f), r0, r1 - r0 > chunk ? r0 + chunk : r1, single ? -1 : c};
            }
            before = __shfl(sum, 63);
            return hit != 0;
        });
    return r;
}
__device__ __forceinline__ int count_chunks(const int64_t* __restrict__ ends, int n_groups, int rows, int chunk) {
    if (!ends) return (rows + chunk - 1) / chunk;
    int n = 0;
    walk_groups(ends, n_groups, rows, [&](int, int begin, int end) { n += (end - begin + chunk - 1) / chunk; return false; });
#pragma unroll
    for (int d = 32; d; d >>= 1) n += __shfl_xor(n, d);
    return n;
}
__device__ __forceinline__ Slabs group_slabs(const int64_t* __restrict__ ends, int n_groups, int rows, int group, int chunk) {
    if (!ends) return {0, (rows + chunk - 1) / chunk};
    Slabs s = {0, 0};
    int before = 0;
    walk_groups(ends, n_groups, rows, [&](int g, int begin, int end) {
        const int n = end - begin, own = n > chunk ? (n - 1) / chunk + 1 : 0, sum = before + wave_sum_scan(own);
        const unsigned long long hit = __ballot(g == group);
        if (hit) {
            const int f = __builtin_ctzll(hit), rows_f = __shfl(n, f);
            s = {__shfl(sum - own, f), rows_f > chunk ? __shfl(own, f) : rows_f > 0};
        }
        before = __shfl(sum, 63);
        return hit != 0;
    });
    return s;
}

}  // namespace layers
}  // namespace smrt
