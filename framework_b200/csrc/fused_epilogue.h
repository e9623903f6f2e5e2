// Epilogues of products from 16-bit planes that never leave their result in memory as f32.  Each epilogue thread holds 128
// neighbouring columns of one row of a 256 x 256 tile in registers when they begin, and the tensor pipe is at the next tile already.
//
//   logit_pairs   z = product + bias -> (maximum, sum of exponentials) of the 128 columns, and the target's logit: 8 bytes for 128
//                 logits instead of 512 written and read again
//   logit_grads   z -> exp(z - lse) - [class = target], in planes for the two products that follow: 4 bytes instead of 4 + 4 + 4 + 4
//                 through f32 logits, f32 gradients and a pass that splits them
//   polynomial    alpha * product + beta * add -> planes, above and below the diagonal where the result is symmetric
//
// Planes are written row by row, 32 bytes a store of one thread: whole sectors.  Scales are fixed, not looked for: a gradient of
// logits is at most one, what a polynomial makes is bounded on the host.
#pragma once

#include <cuda_fp16.h>

#include "internal.h"

namespace mni {
namespace {

struct FusedTile {
    int row, rows;                 // this thread's row, of so many
    int col, cols;                 // its first column, of so many
    int batch;
    int stretch;                   // index of the 128 columns
    bool off_diagonal;
    int lane;
};

__device__ __forceinline__ long long fused_target(const Targets &t, int row) {
    return t.bytes == 8 ? __ldg(static_cast<const long long *>(t.ptr) + row) : __ldg(static_cast<const int *>(t.ptr) + row);
}

// z = x * unscale + bias; columns past the last: -inf.
__device__ __forceinline__ void logits_of(const FusedArgs &f, const FusedTile &at, uint32_t (&run)[4][32], float unscale) {
    const bool whole = at.col + 128 <= at.cols;
    if (!f.bias && whole) {
#pragma unroll
        for (int c = 0; c < 4; ++c)
#pragma unroll
            for (int e = 0; e < 32; ++e) run[c][e] = __float_as_uint(__uint_as_float(run[c][e]) * unscale);
        return;
    }
    const float *const bias = f.bias + f.first_class + at.col;
#pragma unroll
    for (int c = 0; c < 4; ++c)
#pragma unroll
        for (int e = 0; e < 32; ++e) {
            const int j = c * 32 + e;
            const bool there = at.col + j < at.cols;
            const float b = f.bias && there ? __ldg(bias + j) : 0.f;
            run[c][e] = __float_as_uint(there ? fmaf(__uint_as_float(run[c][e]), unscale, b) : -INFINITY);
        }
}

__device__ __forceinline__ void logit_pairs(const FusedArgs &f, const FusedTile &at, uint32_t (&run)[4][32], float unscale) {
    if (at.col >= at.cols) return;                 // the same for the whole warp
    logits_of(f, at, run, unscale);
    const bool live = at.row < at.rows;
    float m[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
    for (int e = 0; e < 32; ++e)
#pragma unroll
        for (int c = 0; c < 4; ++c) m[c] = fmaxf(m[c], __uint_as_float(run[c][e]));
    const float top = fmaxf(fmaxf(m[0], m[1]), fmaxf(m[2], m[3]));
    const float shift = isinf(top) ? 0.f : top;
    float s[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int e = 0; e < 32; ++e)
#pragma unroll
        for (int c = 0; c < 4; ++c) s[c] += exp2f((__uint_as_float(run[c][e]) - shift) * 1.44269504f);
    if (live) f.pairs[static_cast<long long>(at.stretch) * at.rows + at.row] = make_float2(top, (s[0] + s[1]) + (s[2] + s[3]));
    // the target's logit, in the few tiles that hold one of these rows'
    const long long t = live ? fused_target(f.targets, at.row) - f.first_class - at.col : -1;
    const bool mine = t >= 0 && t < 128 && at.col + t < at.cols;
    if (__any_sync(0xffffffffu, mine)) {
        float z = 0.f;
#pragma unroll
        for (int c = 0; c < 4; ++c)
#pragma unroll
            for (int e = 0; e < 32; ++e) z = t == c * 32 + e ? __uint_as_float(run[c][e]) : z;
        if (mine) f.at_target[at.row] = z;
    }
}

__device__ __forceinline__ void store_planes16(uint16_t *at, const uint32_t (&v)[8]) {
    asm volatile("st.global.v8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"l"(at), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]),
                 "r"(v[6]), "r"(v[7])
                 : "memory");
}
__device__ __forceinline__ void load_planes16(const uint16_t *at, uint32_t (&v)[8]) {
    asm volatile("ld.global.v8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
                 : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7])
                 : "l"(at));
}
// x = hi + lo * 2^-kHalfLoShift, two elements
__device__ __forceinline__ void split_pair(float a, float b, uint32_t &hi, uint32_t &lo) {
    const __half2 h = __floats2half2_rn(a, b);
    const float2 back = __half22float2(h);
    constexpr float up = 1 << kHalfLoShift;
    const __half2 l = __floats2half2_rn((a - back.x) * up, (b - back.y) * up);
    hi = *reinterpret_cast<const uint32_t *>(&h);
    lo = *reinterpret_cast<const uint32_t *>(&l);
}

// WIDE: as three bf16, unscaled, for operands whose range f16 does not hold (an MMA's two operands have one type).
template <bool WIDE>
__device__ __forceinline__ void logit_grads(const FusedArgs &f, const FusedTile &at, uint32_t (&run)[4][32], float unscale) {
    if (at.col >= f.dst_pitch || at.row >= at.rows) return;
    logits_of(f, at, run, unscale);
    const float lse = __ldg(f.lse + at.row);
    const long long t = fused_target(f.targets, at.row);
    const long long rel = t - f.first_class - at.col;
    // a row left out has no gradient, whatever it holds; a target that is no class makes its row's NaN
    const float scale = t < f.classes ? (WIDE ? 1.f : static_cast<float>(1 << kGradExponent)) : NAN;
    uint16_t *const dst = f.dst + at.row * f.dst_pitch + at.col;
#pragma unroll
    for (int c = 0; c < 4; ++c)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const int j0 = c * 32 + h * 16;
            if (at.col + j0 >= f.dst_pitch) return;
            float d[16];
#pragma unroll
            for (int e = 0; e < 16; ++e) {
                const float p = expf(__uint_as_float(run[c][h * 16 + e]) - lse) - (rel == j0 + e ? 1.f : 0.f);
                d[e] = t >= 0 && at.col + j0 + e < at.cols ? p * scale : 0.f;
            }
            uint32_t x[3][8];
            if constexpr (WIDE) {
#pragma unroll
                for (int plane = 0; plane < 3; ++plane) {
#pragma unroll
                    for (int e = 0; e < 16; e += 2) {
                        const uint32_t a = __float_as_uint(d[e]) & 0xffff0000u, b = __float_as_uint(d[e + 1]) & 0xffff0000u;
                        x[plane][e / 2] = (a >> 16) | b;
                        d[e] -= __uint_as_float(a);
                        d[e + 1] -= __uint_as_float(b);
                    }
                    store_planes16(dst + plane * f.dst_plane + j0, x[plane]);
                }
            } else {
#pragma unroll
                for (int e = 0; e < 16; e += 2) split_pair(d[e], d[e + 1], x[0][e / 2], x[1][e / 2]);
                store_planes16(dst + j0, x[0]);
                store_planes16(dst + f.dst_plane + j0, x[1]);
            }
        }
}

__device__ __forceinline__ void polynomial(const FusedArgs &f, const FusedTile &at, uint32_t (&run)[4][32]) {
    const bool live = at.row < at.rows;
    const uint16_t *const add = f.add + at.batch * f.add_matrix + at.row * f.add_pitch + at.col;
    uint16_t *const out = f.dst + at.batch * f.dst_matrix;
#pragma unroll
    for (int c = 0; c < 4; ++c)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const int j0 = c * 32 + h * 16;
            if (at.col + j0 >= at.cols) return;    // the same for the whole warp; pitches are multiples of 64
            uint32_t hi[8] = {}, lo[8] = {};
            if (f.add && live) {
                load_planes16(add + j0, hi);
                load_planes16(add + f.add_plane + j0, lo);
            }
            float v[16];
#pragma unroll
            for (int e = 0; e < 16; e += 2) {
                const float2 a = __half22float2(*reinterpret_cast<const __half2 *>(&hi[e / 2])), b = __half22float2(*reinterpret_cast<const __half2 *>(&lo[e / 2]));
                constexpr float down = 1.f / (1 << kHalfLoShift);
                v[e] = fmaf(f.alpha, __uint_as_float(run[c][h * 16 + e]), f.beta * fmaf(b.x, down, a.x));
                v[e + 1] = fmaf(f.alpha, __uint_as_float(run[c][h * 16 + e + 1]), f.beta * fmaf(b.y, down, a.y));
            }
            if (f.final) {
#pragma unroll
                for (int e = 0; e < 16; ++e) run[c][h * 16 + e] = __float_as_uint(v[e]);
                continue;
            }
#pragma unroll
            for (int e = 0; e < 16; e += 2) split_pair(v[e], v[e + 1], hi[e / 2], lo[e / 2]);
            if (live) {
                store_planes16(out + at.row * f.dst_pitch + at.col + j0, hi);
                store_planes16(out + f.dst_plane + at.row * f.dst_pitch + at.col + j0, lo);
            }
            if (f.mirror && at.off_diagonal) {
                // Columns become rows.  Lanes of two neighbouring rows trade one of two columns, so that each writes two elements
                // of one row of the result: a warp's store covers 64 bytes of each of two rows.
                const bool odd = at.lane & 1;
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    const uint32_t even_col = __byte_perm(hi[e], lo[e], 0x5410), odd_col = __byte_perm(hi[e], lo[e], 0x7632);   // (hi, lo) of a column
                    const uint32_t got = __shfl_xor_sync(0xffffffffu, odd ? even_col : odd_col, 1);
                    const uint32_t first = odd ? got : even_col, second = odd ? odd_col : got;       // of rows row & ~1 and row | 1
                    const int col = at.col + j0 + 2 * e + (odd ? 1 : 0), row = at.row & ~1;
                    if (col < at.cols && row < at.rows) {          // an element past the last row goes into the pitch
                        uint16_t *const to = out + static_cast<long long>(col) * f.dst_pitch + row;
                        *reinterpret_cast<uint32_t *>(to) = __byte_perm(first, second, 0x5410);
                        *reinterpret_cast<uint32_t *>(to + f.dst_plane) = __byte_perm(first, second, 0x7632);
                    }
                }
            }
        }
}

}  // namespace
}  // namespace mni
