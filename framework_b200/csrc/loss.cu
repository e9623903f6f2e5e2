// Softmax cross entropy of a projection, z = x.w (+ bias), without its logits in the caller's memory, and its gradient.
//
//   lse[r] = log sum_j exp z[r, j],  loss[r] = lse[r] - z[r, t[r]],  d[r, j] = exp(z[r, j] - lse[r]) - [j = t[r]]
//   dx = diag(g) d w^T,  dw = (diag(g) x)^T d,  dbias = sum_r g[r] d[r, :]
//
// A row's sum of exponentials is kept as pairs (m, s), the sum being s * exp(m): one pair for each stretch of classes, joined by
// loss_finish_kernel.  m is the stretch's maximum; a stretch of nothing but -inf has s = 0 and m = -inf, one with +inf has
// m = +inf (and lse = +inf), NaN stays in s.  Sums of exponentials are in f32 over a stretch and in f32 over its stretches,
// sums over rows in f64, both in a fixed order.
//
// A target below zero leaves its row out: loss 0, no gradient, whatever the row of x holds.  One that is no class makes the
// row's loss, and with it the gradients, NaN: a mistake that shows, where a check would have to wait for the device.
#include "internal.h"

#include <cuda_fp16.h>

#include <algorithm>
#include <cmath>

namespace mni {

namespace {

constexpr int kThreads = 256;
constexpr int kStretch = kLogitStretch;            // classes per block of the kernel for logits in memory
constexpr int kPer = kStretch / kThreads;

__device__ __forceinline__ long long target_at(const Targets &t, long long row) {
    return t.bytes == 8 ? static_cast<const long long *>(t.ptr)[row] : static_cast<const int *>(t.ptr)[row];
}

__device__ __forceinline__ float warp_max(float v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
    return v;
}
template <class T>
__device__ __forceinline__ T warp_sum(T v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}

// s * exp(m - to), 0 where there is nothing to add; NaN in s stays.
__device__ __forceinline__ float rescaled(float m, float s, float to) {
    return m == to ? s : (m == -INFINITY ? s : s * expf(m - to));
}

// Pairs (m, s) of stretches of the logits z[rows, n] of classes first .. first + n, and the targets' logits.  One block per
// row and stretch, whose elements stay in registers between the maximum and the sum.  Bound by memory, 4 bytes an element.
__global__ void __launch_bounds__(kThreads)
logit_stats_kernel(const float *__restrict__ z, int rows, int n, FastDiv stretches, Targets targets, float2 *__restrict__ pairs,
                   float *__restrict__ at_target) {
    __shared__ float red[8];
    grid_dependency_trigger();
    grid_dependency_wait();
    const int row = fd_div(blockIdx.x, stretches), stretch = static_cast<int>(blockIdx.x - row * stretches.d), c0 = stretch * kStretch;
    const float *src = z + static_cast<long long>(row) * n;
    float v[kPer];
    float m = -INFINITY;
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
        const int c = c0 + i * kThreads + threadIdx.x;
        v[i] = c < n ? src[c] : -INFINITY;
        m = fmaxf(m, v[i]);
    }
    m = warp_max(m);
    if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = m;
    __syncthreads();
    m = red[0];
#pragma unroll
    for (int w = 1; w < 8; ++w) m = fmaxf(m, red[w]);
    const float shift = isinf(m) ? 0.f : m;
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < kPer; ++i) s += expf(v[i] - shift);
    s = warp_sum(s);
    __syncthreads();
    if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = s;
    __syncthreads();
    if (threadIdx.x == 0) {
        s = red[0];
#pragma unroll
        for (int w = 1; w < 8; ++w) s += red[w];
        pairs[static_cast<long long>(stretch) * rows + row] = make_float2(m, s);
        const long long t = target_at(targets, row);
        if (t >= c0 && t < min(n, c0 + kStretch)) at_target[row] = src[t];
    }
}

// Joins the pairs of 32 rows a block, `parts` of them each, eight warps taking every eighth.  sums: a pair (sum of losses, rows
// counted) per block; with one block the reduced loss is written here, else by loss_sum_kernel.
__global__ void __launch_bounds__(kThreads)
loss_finish_kernel(const float2 *__restrict__ pairs, int parts, int rows, int classes, Targets targets, const float *__restrict__ at_target,
                   int reduction, float *__restrict__ loss, float *__restrict__ lse, double2 *__restrict__ sums) {
    __shared__ float2 part[8][32];
    grid_dependency_trigger();
    grid_dependency_wait();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int row = blockIdx.x * 32 + lane;
    float m = -INFINITY, s = 0.f;
    if (row < rows) {
        for (int p0 = warp; p0 < parts; p0 += 64) {            // eight loads on their way together
            float2 x[8];
#pragma unroll
            for (int u = 0; u < 8; ++u) {
                const int p = p0 + 8 * u;
                x[u] = p < parts ? __ldcg(pairs + static_cast<long long>(p) * rows + row) : make_float2(-INFINITY, 0.f);
            }
            float top = m;
#pragma unroll
            for (int u = 0; u < 8; ++u) top = fmaxf(top, x[u].x);
            s = rescaled(m, s, top);
#pragma unroll
            for (int u = 0; u < 8; ++u) s += rescaled(x[u].x, x[u].y, top);
            m = top;
        }
    }
    part[warp][lane] = make_float2(m, s);
    __syncthreads();
    if (warp != 0) return;
    double l = 0.0;
    int counted = 0;
    if (row < rows) {
        float top = m;
#pragma unroll
        for (int w = 1; w < 8; ++w) top = fmaxf(top, part[w][lane].x);
        s = rescaled(m, s, top);
#pragma unroll
        for (int w = 1; w < 8; ++w) s += rescaled(part[w][lane].x, part[w][lane].y, top);
        const float total = top == -INFINITY ? logf(s) : top + logf(s);
        lse[row] = total;
        const long long t = target_at(targets, row);
        float one = 0.f;
        if (t >= 0) {
            one = t < classes ? total - __ldcg(at_target + row) : NAN;
            counted = 1;
            l = one;
        }
        if (reduction == 0) loss[row] = one;
    }
    if (reduction == 0) return;
    l = warp_sum(l);
    counted = __reduce_add_sync(0xffffffffu, counted);
    if (lane == 0) {
        if (gridDim.x == 1) loss[0] = static_cast<float>(reduction == 2 ? l / counted : l);
        else sums[blockIdx.x] = make_double2(l, counted);
    }
}

__global__ void __launch_bounds__(kThreads)
loss_sum_kernel(const double2 *__restrict__ sums, int count, int reduction, float *__restrict__ loss) {
    __shared__ double2 red[8];
    grid_dependency_trigger();
    grid_dependency_wait();
    double l = 0.0, n = 0.0;
    for (int i = threadIdx.x; i < count; i += kThreads) {
        const double2 x = sums[i];
        l += x.x;
        n += x.y;
    }
    l = warp_sum(l);
    n = warp_sum(n);
    if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = make_double2(l, n);
    __syncthreads();
    if (threadIdx.x != 0) return;
    for (int w = 1; w < 8; ++w) {
        l += red[w].x;
        n += red[w].y;
    }
    loss[0] = static_cast<float>(reduction == 2 ? l / n : l);
}

// Rows that count, of the whole batch (blocks that do not count for themselves wait for this).
constexpr int kCountRows = 4096;
__device__ int count_rows(const Targets &targets, int rows, int *red) {
    int n = 0;
    for (int i = threadIdx.x; i < rows; i += blockDim.x) n += target_at(targets, i) >= 0;
    n = __reduce_add_sync(0xffffffffu, n);
    if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = n;
    __syncthreads();
    n = 0;
    for (int w = 0; w < static_cast<int>(blockDim.x) / 32; ++w) n += red[w];
    return n;
}
__global__ void __launch_bounds__(1024)
count_rows_kernel(Targets targets, int rows, int *count) {
    __shared__ int red[32];
    grid_dependency_trigger();
    grid_dependency_wait();
    const int n = count_rows(targets, rows, red);
    if (threadIdx.x == 0) *count = n;
}

// Weights of the rows' losses in the result's gradient, g = grad, or grad / rows counted, 0 for rows left out; and a copy of x
// whose rows are multiplied by them (scaled), or left out where they are zero.  A block takes rows in turn.
__global__ void __launch_bounds__(kThreads)
row_weights_kernel(const __grid_constant__ RowsIn x, Targets targets, int reduction, const float *__restrict__ grad, const int *count,
                   float *__restrict__ weights, float *__restrict__ copy, int scaled, int *grad_exponent) {
    __shared__ int red[32];
    grid_dependency_trigger();
    grid_dependency_wait();
    if (grad_exponent && blockIdx.x == 0 && threadIdx.x == 0) *grad_exponent = kGradExponent;
    float all = 1.f;
    if (reduction != 0) {
        all = grad[0];
        if (reduction == 2) all /= static_cast<float>(count ? *count : count_rows(targets, x.rows, red));
    }
    for (int row = blockIdx.x; row < x.rows; row += gridDim.x) {
        const bool kept = target_at(targets, row) >= 0;
        const float g = kept ? (reduction == 0 ? grad[row] : all) : 0.f;
        if (threadIdx.x == 0) weights[row] = g;
        if (!copy) continue;
        const float *src = x.ptr + x.offset(row);
        float *dst = copy + static_cast<long long>(row) * x.cols;
        const float f = scaled ? g : 1.f;
        for (int c = threadIdx.x; c < x.cols; c += kThreads) dst[c] = kept ? src[c * x.col_stride] * f : 0.f;
    }
}

// Logits of a row that a block computes itself, for few logits of short rows: a pair and the target's logit (GRAD false), or the weighted
// gradient g * (exp(z - lse) - [j = t]) and the copy of x that dw is made of, zero in rows left out.  Each column is summed by `256 >> shift`
// threads, whose sums are added in order.  Bound by latency: one launch where product, logits' pass and (GRAD) weights are two or three.
template <bool GRAD>
__global__ void __launch_bounds__(kThreads)
small_logits_kernel(const __grid_constant__ RowsIn x, const float *__restrict__ w, long long w_k, long long w_n, const float *__restrict__ bias, int n,
                    int shift, Targets targets, float2 *__restrict__ pairs, float *__restrict__ at_target, int reduction, const float *__restrict__ lse,
                    const float *__restrict__ grad, float *__restrict__ d, float *__restrict__ copy) {
    extern __shared__ float row_of[];
    __shared__ float part[kThreads];
    __shared__ int red[32];
    float *const xs = row_of, *const zs = row_of + x.cols;
    grid_dependency_trigger();
    grid_dependency_wait();
    const int row = blockIdx.x;
    const long long t = target_at(targets, row);
    const bool kept = !GRAD || t >= 0;
    const float *const src = x.ptr + x.offset(row);
    for (int c = threadIdx.x; c < x.cols; c += kThreads) {
        const float v = kept ? src[c * x.col_stride] : 0.f;
        xs[c] = v;
        if (GRAD) copy[static_cast<long long>(row) * x.cols + c] = v;
    }
    float g = 0.f;
    if (GRAD) {
        g = reduction == 0 ? grad[row] : grad[0];
        if (reduction == 2) g /= static_cast<float>(count_rows(targets, x.rows, red));
    }
    __syncthreads();
    const int cols = 1 << shift, groups = kThreads >> shift, col = threadIdx.x & (cols - 1), group = threadIdx.x >> shift;
    for (int j0 = 0; j0 < n; j0 += cols) {
        const int j = j0 + col;
        float z = 0.f;
        if (j < n) {
            const float *const at = w + j * w_n;
#pragma unroll 8
            for (int k = group; k < x.cols; k += groups) z = fmaf(xs[k], __ldg(at + k * w_k), z);
        }
        if (groups > 1) {                          // (the row is one round of columns then)
            part[threadIdx.x] = z;
            __syncthreads();
            for (int i = 1; i < groups; ++i) z += part[(i << shift) + col];
        }
        if (group == 0 && j < n) zs[j] = bias ? z + __ldg(bias + j) : z;
    }
    __syncthreads();
    if (GRAD) {
        const float l = lse[row];
        for (int c = threadIdx.x; c < n; c += kThreads) {
            const float e = expf(zs[c] - l) - (c == t ? 1.f : 0.f);
            d[static_cast<long long>(row) * n + c] = t < 0 ? 0.f : t < n ? e * g : NAN;
        }
        return;
    }
    float m = -INFINITY;
    for (int c = threadIdx.x; c < n; c += kThreads) m = fmaxf(m, zs[c]);
    m = warp_max(m);
    if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = m;
    __syncthreads();
    m = part[0];
#pragma unroll
    for (int i = 1; i < 8; ++i) m = fmaxf(m, part[i]);
    const float to = isinf(m) ? 0.f : m;
    float s = 0.f;
    for (int c = threadIdx.x; c < n; c += kThreads) s += expf(zs[c] - to);
    s = warp_sum(s);
    __syncthreads();
    if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = s;
    __syncthreads();
    if (threadIdx.x != 0) return;
    for (int i = 1; i < 8; ++i) s += part[i];
    pairs[row] = make_float2(m, s);
    if (t >= 0 && t < n) at_target[row] = zs[t];
}

// z -> g * (exp(z - lse) - [j = t]), in place.
__global__ void __launch_bounds__(kThreads)
logit_grad_kernel(float *__restrict__ z, int n, FastDiv stretches, Targets targets, const float *__restrict__ lse,
                  const float *__restrict__ weights) {
    grid_dependency_trigger();
    grid_dependency_wait();
    const int row = fd_div(blockIdx.x, stretches), c0 = static_cast<int>(blockIdx.x - row * stretches.d) * kStretch;
    float *src = z + static_cast<long long>(row) * n;
    const long long t = target_at(targets, row);
    const float l = lse[row], g = weights[row];
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
        const int c = c0 + i * kThreads + threadIdx.x;
        if (c >= n) break;
        float d = expf(src[c] - l) - (c == t ? 1.f : 0.f);
        src[c] = t < 0 ? 0.f : t < n ? d * g : NAN;
    }
}

// dx (+)= weights * sums, row by row.
__global__ void __launch_bounds__(kThreads)
scale_rows_kernel(const float *__restrict__ sums, int ld, const float *__restrict__ weights, float *__restrict__ dx, long long n, FastDiv cols,
                  int accumulate) {
    grid_dependency_trigger();
    grid_dependency_wait();
    for (long long i = static_cast<long long>(blockIdx.x) * kThreads + threadIdx.x; i < n; i += static_cast<long long>(gridDim.x) * kThreads) {
        const long long row = n < 0x7fffffffLL ? fd_div(static_cast<int>(i), cols) : i / cols.d;
        const float w = weights[row];
        // nothing of a row left out: 0 * NaN would be NaN
        const float v = w == 0.f ? 0.f : sums[row * ld + (i - row * cols.d)] * w;
        dx[i] = accumulate ? dx[i] + v : v;
    }
}

// Column sums of logit gradients in planes (three bf16 where `status` says so), rows multiplied by their weights: 64 columns and a
// stretch of rows a block, 8 columns a thread; partial[stretch][columns].
constexpr int kSumCols = 64;
__global__ void __launch_bounds__(kThreads)
grad_column_sums_kernel(const uint16_t *__restrict__ planes, long long pitch, long long plane, int rows, int n, const float *__restrict__ weights,
                        const unsigned *__restrict__ status, float *__restrict__ partial, int stretch) {
    __shared__ float red[32][kSumCols];
    grid_dependency_trigger();
    grid_dependency_wait();
    const bool wide = (__ldcg(status) & 1u) != 0;
    const int col = blockIdx.x * kSumCols + (threadIdx.x & 7) * 8, lane_row = threadIdx.x >> 3;
    const int r0 = blockIdx.y * stretch, r1 = min(rows, r0 + stretch);
    float sum[8] = {};
    for (int r = r0 + lane_row; r < r1; r += 32) {
        const float w = weights[r];
        const uint16_t *at = planes + r * pitch + col;
        const uint4 a = __ldcg(reinterpret_cast<const uint4 *>(at)), b = __ldcg(reinterpret_cast<const uint4 *>(at + plane));
        const unsigned *const x = &a.x, *const y = &b.x;
        if (wide) {
            const uint4 d = __ldcg(reinterpret_cast<const uint4 *>(at + 2 * plane));
            const unsigned *const z = &d.x;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                auto part = [i](unsigned v) { return __uint_as_float(i & 1 ? v & 0xffff0000u : v << 16); };
                sum[i] = fmaf(w, part(x[i / 2]) + (part(y[i / 2]) + part(z[i / 2])), sum[i]);
            }
        } else {
#pragma unroll
            for (int i = 0; i < 8; i += 2) {
                const float2 h = __half22float2(*reinterpret_cast<const __half2 *>(&x[i / 2])), l = __half22float2(*reinterpret_cast<const __half2 *>(&y[i / 2]));
                constexpr float lo = 1.f / (1 << kHalfLoShift), unit = 1.f / (1 << kGradExponent);
                sum[i] = fmaf(w, fmaf(l.x, lo, h.x) * unit, sum[i]);
                sum[i + 1] = fmaf(w, fmaf(l.y, lo, h.y) * unit, sum[i + 1]);
            }
        }
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) red[lane_row][(threadIdx.x & 7) * 8 + i] = sum[i];
    __syncthreads();
    if (threadIdx.x < kSumCols && static_cast<int>(blockIdx.x * kSumCols + threadIdx.x) < n) {
        float s = red[0][threadIdx.x];
        for (int r = 1; r < 32; ++r) s += red[r][threadIdx.x];
        partial[static_cast<long long>(blockIdx.y) * n + blockIdx.x * kSumCols + threadIdx.x] = s;
    }
}
__global__ void __launch_bounds__(kThreads)
add_stretches_kernel(const float *__restrict__ partial, int stretches, int n, float *__restrict__ out, int accumulate) {
    grid_dependency_trigger();
    grid_dependency_wait();
    const int c = blockIdx.x * kThreads + threadIdx.x;
    if (c >= n) return;
    float s = partial[c];
    for (int i = 1; i < stretches; ++i) s += partial[static_cast<long long>(i) * n + c];
    out[c] = accumulate ? out[c] + s : s;
}

}  // namespace

int launch_scale_rows(const float *sums, int64_t ld, const float *weights, float *dx, int64_t rows, int64_t cols, bool accumulate, int sm_count,
                      cudaStream_t stream) {
    const unsigned blocks = static_cast<unsigned>(std::min<int64_t>((rows * cols + kThreads - 1) / kThreads, 8ll * sm_count));
    const cudaError_t e = launch_dependent(scale_rows_kernel, dim3(blocks), dim3(kThreads), 0, stream, sums, static_cast<int>(ld), weights, dx,
                                           static_cast<long long>(rows * cols), make_fastdiv(cols), accumulate ? 1 : 0);
    if (e != cudaSuccess) return fail(MNI_B200_ERR_CUDA, "scale_rows_kernel launch failed: %s", cudaGetErrorString(e));
    MNI_LAUNCH_CHECK("scale_rows_kernel");
    return MNI_B200_OK;
}

// Rows of a stretch: enough blocks for two rounds of four a SM, 64 stretches at most.
static int64_t sum_stretch(int64_t rows, int64_t n, int sm_count) {
    const int64_t want = std::max<int64_t>(1, std::min<int64_t>(64, 8ll * sm_count / ((n + kSumCols - 1) / kSumCols)));
    return std::max<int64_t>(32, ((rows + want - 1) / want + 31) / 32 * 32);
}
size_t grad_column_sums_bytes(int64_t rows, int64_t n, int sm_count) {
    const int64_t stretch = sum_stretch(rows, n, sm_count);
    return static_cast<size_t>((rows + stretch - 1) / stretch * n) * sizeof(float);
}
int launch_grad_column_sums(const uint16_t *planes, int64_t pitch, int64_t plane, int64_t rows, int64_t n, const float *weights, const unsigned *status,
                            float *partial, float *out, bool accumulate, int sm_count, cudaStream_t stream) {
    const int64_t stretch = sum_stretch(rows, n, sm_count), stretches = (rows + stretch - 1) / stretch;
    cudaError_t e = launch_dependent(grad_column_sums_kernel, dim3(static_cast<unsigned>((n + kSumCols - 1) / kSumCols), static_cast<unsigned>(stretches)),
                                     dim3(kThreads), 0, stream, planes, static_cast<long long>(pitch), static_cast<long long>(plane),
                                     static_cast<int>(rows), static_cast<int>(n), weights, status, partial, static_cast<int>(stretch));
    if (e != cudaSuccess) return fail(MNI_B200_ERR_CUDA, "grad_column_sums_kernel launch failed: %s", cudaGetErrorString(e));
    MNI_LAUNCH_CHECK("grad_column_sums_kernel");
    e = launch_dependent(add_stretches_kernel, dim3(static_cast<unsigned>((n + kThreads - 1) / kThreads)), dim3(kThreads), 0, stream, partial,
                         static_cast<int>(stretches), static_cast<int>(n), out, accumulate ? 1 : 0);
    if (e != cudaSuccess) return fail(MNI_B200_ERR_CUDA, "add_stretches_kernel launch failed: %s", cudaGetErrorString(e));
    MNI_LAUNCH_CHECK("add_stretches_kernel");
    return MNI_B200_OK;
}

int launch_logit_stats(const float *z, int64_t rows, int64_t n, const Targets &targets, float2 *pairs, float *at_target, cudaStream_t stream) {
    const int64_t stretches = (n + kStretch - 1) / kStretch;
    const dim3 grid(static_cast<unsigned>(rows * stretches));
    const cudaError_t e = launch_dependent(logit_stats_kernel, grid, dim3(kThreads), 0, stream, z, static_cast<int>(rows), static_cast<int>(n),
                                           make_fastdiv(stretches), targets, pairs, at_target);
    if (e != cudaSuccess) return fail(MNI_B200_ERR_CUDA, "logit_stats_kernel launch failed: %s", cudaGetErrorString(e));
    MNI_LAUNCH_CHECK("logit_stats_kernel");
    return MNI_B200_OK;
}

size_t loss_sums_bytes(int64_t rows) { return static_cast<size_t>((rows + 31) / 32) * sizeof(double2); }

int launch_loss_finish(const float2 *pairs, int64_t parts, int64_t rows, int64_t classes, const Targets &targets, const float *at_target,
                       int reduction, float *loss, float *lse, double2 *sums, cudaStream_t stream) {
    const unsigned blocks = static_cast<unsigned>((rows + 31) / 32);
    cudaError_t e = launch_dependent(loss_finish_kernel, dim3(blocks), dim3(kThreads), 0, stream, pairs, static_cast<int>(parts),
                                     static_cast<int>(rows), static_cast<int>(classes), targets, at_target, reduction, loss, lse, sums);
    if (e != cudaSuccess) return fail(MNI_B200_ERR_CUDA, "loss_finish_kernel launch failed: %s", cudaGetErrorString(e));
    MNI_LAUNCH_CHECK("loss_finish_kernel");
    if (reduction == 0 || blocks == 1) return MNI_B200_OK;
    e = launch_dependent(loss_sum_kernel, dim3(1), dim3(kThreads), 0, stream, sums, static_cast<int>(blocks), reduction, loss);
    if (e != cudaSuccess) return fail(MNI_B200_ERR_CUDA, "loss_sum_kernel launch failed: %s", cudaGetErrorString(e));
    MNI_LAUNCH_CHECK("loss_sum_kernel");
    return MNI_B200_OK;
}

int launch_row_weights(const RowsIn &x, const Targets &targets, int reduction, const float *grad, int *count, float *weights, float *copy,
                       bool scaled, int *grad_exponent, int sm_count, cudaStream_t stream) {
    const int *counted = nullptr;
    if (reduction == 2 && x.rows > kCountRows) {
        const cudaError_t e = launch_dependent(count_rows_kernel, dim3(1), dim3(1024), 0, stream, targets, x.rows, count);
        if (e != cudaSuccess) return fail(MNI_B200_ERR_CUDA, "count_rows_kernel launch failed: %s", cudaGetErrorString(e));
        MNI_LAUNCH_CHECK("count_rows_kernel");
        counted = count;
    }
    const unsigned blocks = static_cast<unsigned>(std::min<int64_t>(x.rows, 8ll * sm_count));
    const cudaError_t e = launch_dependent(row_weights_kernel, dim3(blocks), dim3(kThreads), 0, stream, x, targets, reduction, grad, counted,
                                           weights, copy, scaled ? 1 : 0, grad_exponent);
    if (e != cudaSuccess) return fail(MNI_B200_ERR_CUDA, "row_weights_kernel launch failed: %s", cudaGetErrorString(e));
    MNI_LAUNCH_CHECK("row_weights_kernel");
    return MNI_B200_OK;
}

static int small_shift(int64_t n) {
    int shift = 5;
    while (shift < 8 && (1 << shift) < n) ++shift;
    return shift;
}
// What small_logits_kernel takes: rows whose threads wait for weights four times at most (eight loads at a time).  us, product and passes / this: a
// step of 32 rows, 64 features and 96 classes 28.5 / 21.9; from a graph its gradient 10.4 / 8.3 and the loss 7.8 / 7.8.  With eight waits (128
// features, 128 classes) 9.7 / 10.9 for the loss and 12.4 / 11.1 for the gradient, with sixteen (1024 features, 16 classes) 8.9 / 16.2 and
// 11.1 / 14.1.
bool small_logits(int64_t rows, int64_t k, int64_t n) {
    const int64_t cols = int64_t{1} << small_shift(n), groups = kThreads / cols;
    return rows <= kCountRows && (n + cols - 1) / cols * ((k + 8 * groups - 1) / (8 * groups)) <= 4;
}

int launch_small_logits(const RowsIn &x, const float *w, int64_t w_k, int64_t w_n, const float *bias, int64_t n, const Targets &targets, float2 *pairs,
                        float *at_target, cudaStream_t stream) {
    const cudaError_t e = launch_dependent(small_logits_kernel<false>, dim3(static_cast<unsigned>(x.rows)), dim3(kThreads),
                                           static_cast<size_t>(x.cols + n) * sizeof(float), stream, x, w, static_cast<long long>(w_k),
                                           static_cast<long long>(w_n), bias, static_cast<int>(n), small_shift(n), targets, pairs, at_target, 0, nullptr,
                                           nullptr, nullptr, nullptr);
    if (e != cudaSuccess) return fail(MNI_B200_ERR_CUDA, "small_logits_kernel launch failed: %s", cudaGetErrorString(e));
    MNI_LAUNCH_CHECK("small_logits_kernel");
    return MNI_B200_OK;
}
int launch_small_grads(const RowsIn &x, const float *w, int64_t w_k, int64_t w_n, const float *bias, int64_t n, const Targets &targets, int reduction,
                       const float *lse, const float *grad, float *d, float *copy, cudaStream_t stream) {
    const cudaError_t e = launch_dependent(small_logits_kernel<true>, dim3(static_cast<unsigned>(x.rows)), dim3(kThreads),
                                           static_cast<size_t>(x.cols + n) * sizeof(float), stream, x, w, static_cast<long long>(w_k),
                                           static_cast<long long>(w_n), bias, static_cast<int>(n), small_shift(n), targets, nullptr, nullptr, reduction, lse,
                                           grad, d, copy);
    if (e != cudaSuccess) return fail(MNI_B200_ERR_CUDA, "small_logits_kernel launch failed: %s", cudaGetErrorString(e));
    MNI_LAUNCH_CHECK("small_logits_kernel");
    return MNI_B200_OK;
}

int launch_logit_grad(float *z, int64_t rows, int64_t n, const Targets &targets, const float *lse, const float *weights, cudaStream_t stream) {
    const int64_t stretches = (n + kStretch - 1) / kStretch;
    const dim3 grid(static_cast<unsigned>(rows * stretches));
    const cudaError_t e = launch_dependent(logit_grad_kernel, grid, dim3(kThreads), 0, stream, z, static_cast<int>(n), make_fastdiv(stretches),
                                           targets, lse, weights);
    if (e != cudaSuccess) return fail(MNI_B200_ERR_CUDA, "logit_grad_kernel launch failed: %s", cudaGetErrorString(e));
    MNI_LAUNCH_CHECK("logit_grad_kernel");
    return MNI_B200_OK;
}

}  // namespace mni
