// Epilogues of products from 16-bit planes that never leave their result in memory as f32.  A thread holds columns of one row of the
// tile in registers when they begin, 32 of them a chunk, and the tensor pipe is at the next tile already.
//
//   PairSum       z = product + bias -> (maximum, sum of exponentials) of a thread's columns, and the target's logit: 8 bytes for
//                 128 logits instead of 512 written and read again
//   grad_chunk    z -> exp(z - lse) - [class = target], in planes for the two products that follow: 4 bytes instead of 4 + 4 + 4 + 4
//                 through f32 logits, f32 gradients and a pass that splits them
//
// The kernel calls them chunk after chunk in a loop that is not unrolled, and moves the registers down in between: unrolled over 128
// columns their code (40 KB, executed once a tile) came from beyond the instruction caches, and a tile's epilogue took 12 us.
//
// Planes are written row by row, 32 bytes a store of one thread: whole sectors.  The scale of f16 planes is fixed, 2^14, not looked for: a
// gradient d of logits is at most one.  So hi is subnormal below 2^-28, where the two planes begin to hold fewer than 22 bits, and nothing is left
// below 2^-51; with the lo * lo that products leave out, what a product takes of a d is off by an absolute 2^-50 (a row's weight is not in d
// yet).  A class of probability 1e-10 in every row has dw and dbias to 1e-5 of their size, one of 1e-13 to 1e-2.  It is a choice: beside what the
// row's own target adds (1 - p) it is 2^-50 of the row's gradient, and three bf16 planes, which would keep f32's range, are six products for three.
// Nor is their range looked at as an operand's is (half.cu): most classes are improbable in most rows, so that most calls would take six.
//
// exp: ex2.approx of the argument times log2(e).  That product's rounding makes a term off by (max - z) 2^-24 of itself at most, either way; a row's sum
// averages it over its terms, and the logits' own error (1e-6 of what they are summed from) is more.  In d it would be the result's, and is
// carried along.
#pragma once

#include <cuda_fp16.h>

#include "internal.h"

namespace mni {
namespace {

struct FusedTile {
    int row, rows;                 // this thread's row, of so many
    int col, cols;                 // its first column, of so many
    int stretch;                   // index of its columns' stretch
    int lane;
    float *patch;                  // 4 KB of shared memory of the warp's own
};

__device__ __forceinline__ float exp2_approx(float x) {     // 2 ulp; results below 2^-126 are zero
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
constexpr float kLog2e = 1.4426950408889634f;

// What is added to the logits of a chunk, in the warp's patch: bias, -inf past the last column.  Returns whether there is anything.
__device__ __forceinline__ bool stage_bias(const FusedArgs &f, const FusedTile &at, int col) {
    if (!f.bias && col + 32 <= at.cols) return false;
    const int j = col + at.lane;
    __syncwarp();
    at.patch[at.lane] = j < at.cols ? (f.bias ? __ldg(f.bias + f.first_class + j) : 0.f) : -INFINITY;
    __syncwarp();
    return true;
}
// z = x * unscale (+ the patch)
__device__ __forceinline__ void logits_of(bool biased, const FusedTile &at, uint32_t (&v)[32], float unscale) {
    if (biased) {
#pragma unroll
        for (int e = 0; e < 32; e += 4) {
            const float4 b = *reinterpret_cast<const float4 *>(at.patch + e);
            v[e] = __float_as_uint(fmaf(__uint_as_float(v[e]), unscale, b.x));
            v[e + 1] = __float_as_uint(fmaf(__uint_as_float(v[e + 1]), unscale, b.y));
            v[e + 2] = __float_as_uint(fmaf(__uint_as_float(v[e + 2]), unscale, b.z));
            v[e + 3] = __float_as_uint(fmaf(__uint_as_float(v[e + 3]), unscale, b.w));
        }
    } else {
#pragma unroll
        for (int e = 0; e < 32; ++e) v[e] = __float_as_uint(__uint_as_float(v[e]) * unscale);
    }
}
// The target of a thread's row, relative to column `col` of the launch; anything negative where it is not there.
__device__ __forceinline__ long long target_of(const FusedArgs &f, const FusedTile &at) {
    const Targets &t = f.targets;
    return t.bytes == 8 ? __ldg(static_cast<const long long *>(t.ptr) + at.row) : __ldg(static_cast<const int *>(t.ptr) + at.row);
}

struct PairSum {
    float m, s;
    int rel;                       // the target, relative to the thread's first column (-1: elsewhere)
    __device__ __forceinline__ void begin(const FusedArgs &f, const FusedTile &at, int columns) {
        m = -INFINITY;
        s = 0.f;
        const long long t = at.row < at.rows ? target_of(f, at) - f.first_class - at.col : -1;
        rel = t >= 0 && t < columns && at.col + t < at.cols ? static_cast<int>(t) : -1;
    }
    __device__ __forceinline__ void chunk(const FusedArgs &f, const FusedTile &at, uint32_t (&v)[32], int c, float unscale) {
        const int col = at.col + 32 * c;
        if (col >= at.cols) return;                // the same for the whole warp
        logits_of(stage_bias(f, at, col), at, v, unscale);
        float top[4] = {m, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
        for (int e = 0; e < 32; ++e) top[e & 3] = fmaxf(top[e & 3], __uint_as_float(v[e]));
        const float next = fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3]));
        const float shift = isinf(next) ? 0.f : next;
        float sum[4] = {m == next || m == -INFINITY ? s : s * exp2_approx((m - shift) * kLog2e), 0.f, 0.f, 0.f};
#pragma unroll
        for (int e = 0; e < 32; ++e) sum[e & 3] += exp2_approx((__uint_as_float(v[e]) - shift) * kLog2e);
        m = next;
        s = (sum[0] + sum[1]) + (sum[2] + sum[3]);
        // the target's logit, in the few chunks that hold one of these rows'
        const int r = rel - 32 * c;
        const bool mine = static_cast<unsigned>(r) < 32u;
        if (__any_sync(0xffffffffu, mine)) {
            float z = 0.f;
#pragma unroll
            for (int e = 0; e < 32; ++e) z = r == e ? __uint_as_float(v[e]) : z;
            if (mine) f.at_target[at.row] = z;
        }
    }
    __device__ __forceinline__ void end(const FusedArgs &f, const FusedTile &at) const {
        if (at.col < at.cols && at.row < at.rows) f.pairs[static_cast<long long>(at.stretch) * at.rows + at.row] = make_float2(m, s);
    }
};

__device__ __forceinline__ void store_planes16(uint16_t *at, const uint32_t *v) {
    asm volatile("st.global.v8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"l"(at), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]),
                 "r"(v[6]), "r"(v[7])
                 : "memory");
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

struct GradRow {
    float lse, scale;
    int rel;
    bool kept, live;
    // a row left out has no gradient, whatever it holds; a target that is no class makes its row's NaN
    __device__ __forceinline__ void begin(const FusedArgs &f, const FusedTile &at, bool wide) {
        live = at.row < at.rows;
        const long long t = live ? target_of(f, at) : -1, r = t - f.first_class - at.col;
        lse = live ? __ldg(f.lse + at.row) : 0.f;
        kept = t >= 0;
        scale = t < f.classes ? (wide ? 1.f : static_cast<float>(1 << kGradExponent)) : NAN;
        rel = r >= 0 && r < (1 << 20) ? static_cast<int>(r) : -1;
    }
};
// wide: as three bf16, unscaled, for operands whose range f16 does not hold (an MMA's two operands have one type).
__device__ __forceinline__ void grad_chunk(const FusedArgs &f, const FusedTile &at, const GradRow &g, uint32_t (&v)[32], int c, float unscale, bool wide) {
    const int col = at.col + 32 * c;
    if (col >= f.dst_pitch) return;                // the same for the whole warp; pitches are multiples of 64
    logits_of(stage_bias(f, at, col), at, v, unscale);
    const int r = g.rel - 32 * c;
#pragma unroll
    for (int e = 0; e < 32; ++e) {
        // the product with log2(e) carried out to where its rounding does not show: an error of 2^-24 of it would be one of the result
        const float u = __uint_as_float(v[e]) - g.lse, d = u < -200.f ? -200.f : u, y = d * kLog2e;      // (NaN stays)
        const float p = exp2_approx(y) * fmaf(fmaf(d, kLog2e, -y), 0.6931472f, 1.f);
        const float x = (e == r ? p - 1.f : p) * g.scale;
        v[e] = __float_as_uint(g.kept ? x : 0.f);
    }
    if (!g.live) return;
    uint16_t *const dst = f.dst + at.row * f.dst_pitch + col;
    if (wide) {
#pragma unroll 1
        for (int plane = 0; plane < 3; ++plane) {
            uint32_t x[16];
#pragma unroll
            for (int e = 0; e < 32; e += 2) {
                const uint32_t a = v[e] & 0xffff0000u, b = v[e + 1] & 0xffff0000u;
                x[e / 2] = (a >> 16) | b;
                v[e] = __float_as_uint(__uint_as_float(v[e]) - __uint_as_float(a));
                v[e + 1] = __float_as_uint(__uint_as_float(v[e + 1]) - __uint_as_float(b));
            }
            store_planes16(dst + plane * f.dst_plane, x);
            store_planes16(dst + plane * f.dst_plane + 16, x + 8);
        }
        return;
    }
    uint32_t hi[16], lo[16];
#pragma unroll
    for (int e = 0; e < 32; e += 2) split_pair(__uint_as_float(v[e]), __uint_as_float(v[e + 1]), hi[e / 2], lo[e / 2]);
    store_planes16(dst, hi);
    store_planes16(dst + 16, hi + 8);
    store_planes16(dst + f.dst_plane, lo);
    store_planes16(dst + f.dst_plane + 16, lo + 8);
}

}  // namespace
}  // namespace mni
