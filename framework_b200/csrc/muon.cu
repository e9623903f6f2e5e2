// Updates of matrices by their orthogonalised momentum: the kernels around the Newton-Schulz products.
//
//   m <- mu m + g;  u = g + mu m (nesterov), or m;  x0 = u / (|u|_F + eps)
//   five times x <- a x + (b A + c A^2) x with A = x x^T (the other way round for matrices with more rows than columns)
//   p <- decay p - scale x
//
// As in optimizer.cu the unit of work is a chunk of whichever matrix, and one launch covers a list of them.  Bound by memory: 12
// bytes an element for the momentum (read g and m, write m), 8 to 12 for the normalised update, 12 for the parameter.  Norms are
// summed in f64, in a fixed order.
#include "internal.h"

#include <cuda_fp16.h>

#include <algorithm>
#include <cmath>

namespace mni {

namespace {

constexpr int kThreads = 256;
constexpr int kMaxList = 256;                  // matrices per launch
constexpr int kMaxChunks = 512;                // of one matrix: what a block adds up for the norm
constexpr int kChunk = 4096;

struct List {
    float *param[kMaxList], *momentum[kMaxList], *x[kMaxList];
    const float *grad[kMaxList];
    long long n[kMaxList];
    float scale[kMaxList];
    uint16_t *planes[kMaxList];
    long long plane[kMaxList];
    int rows[kMaxList], cols[kMaxList];
    FastDiv vectors[kMaxList];                 // of 8 columns, in a row of the planes
    unsigned first[kMaxList + 1];              // index of a matrix's first chunk
    int chunk[kMaxList];                       // elements of one
    int count;
};

__device__ __forceinline__ int find(const List &list, unsigned chunk) {
    int lo = 0, hi = list.count;
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (list.first[mid] <= chunk) lo = mid; else hi = mid;
    }
    return lo;
}

__device__ __forceinline__ float update_of(float g, float m, float mu, bool nesterov) { return nesterov ? fmaf(mu, m, g) : m; }

__global__ void __launch_bounds__(kThreads)
muon_momentum_kernel(const __grid_constant__ List list, float mu, bool nesterov, double *__restrict__ partial, unsigned *counters, int words) {
    __shared__ double red[8];
    grid_dependency_trigger();
    grid_dependency_wait();
    if (blockIdx.x == 0)
        for (int i = threadIdx.x; i < words; i += kThreads) counters[i] = 0u;
    const int t = find(list, blockIdx.x);
    const long long base = static_cast<long long>(blockIdx.x - list.first[t]) * list.chunk[t], end = min(list.n[t], base + list.chunk[t]);
    float *const m = list.momentum[t];
    const float *const g = list.grad[t];
    double sum = 0.0;
    auto one = [&](float gi, float &mi) {
        float u = gi;
        if (m) {
            mi = fmaf(mu, mi, gi);
            u = update_of(gi, mi, mu, nesterov);
        }
        sum += static_cast<double>(u) * u;
    };
    const bool vec = ((reinterpret_cast<uintptr_t>(m) | reinterpret_cast<uintptr_t>(g)) & 15) == 0;
    long long i = base;
    if (vec) {
        for (; i + kThreads * 4 <= end; i += kThreads * 4) {
            const long long at = i + threadIdx.x * 4;
            const float4 gi = *reinterpret_cast<const float4 *>(g + at);
            float4 mi = m ? *reinterpret_cast<const float4 *>(m + at) : gi;
            one(gi.x, mi.x); one(gi.y, mi.y); one(gi.z, mi.z); one(gi.w, mi.w);
            if (m) *reinterpret_cast<float4 *>(m + at) = mi;
        }
    }
    for (i += threadIdx.x; i < end; i += kThreads) {
        float mi = m ? m[i] : 0.f;
        one(g[i], mi);
        if (m) m[i] = mi;
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = sum;
    __syncthreads();
    if (threadIdx.x == 0) {
        for (int w = 1; w < 8; ++w) sum += red[w];
        partial[blockIdx.x] = sum;
    }
}

// 1 / (norm + eps) of matrix t, from its chunks' sums, as two factors near its root: of matrices whose norm or its inverse is beyond f32's normal
// range neither they nor what has been multiplied by the first is.  The same in every block that asks.
struct Inverse {
    float first, second;
};
__device__ Inverse inverse_norm(const List &list, int t, const double *partial, float eps, double *red) {
    double sum = 0.0;
    for (unsigned i = list.first[t] + threadIdx.x; i < list.first[t + 1]; i += kThreads) sum += __ldcg(partial + i);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = sum;
    __syncthreads();
    sum = red[0];
    for (int w = 1; w < 8; ++w) sum += red[w];
    const double inverse = 1.0 / (sqrt(sum) + static_cast<double>(eps));
    if (!(inverse > 0.0) || isinf(inverse)) return Inverse{1.f, static_cast<float>(inverse)};
    const double first = ldexp(1.0, ilogb(inverse) / 2);
    return Inverse{static_cast<float>(first), static_cast<float>(inverse / first)};
}

__global__ void __launch_bounds__(kThreads)
muon_normalise_kernel(const __grid_constant__ List list, float mu, bool nesterov, float eps, const double *__restrict__ partial) {
    __shared__ double red[8];
    grid_dependency_trigger();
    grid_dependency_wait();
    const int t = find(list, blockIdx.x);
    const Inverse inverse = inverse_norm(list, t, partial, eps, red);
    const long long base = static_cast<long long>(blockIdx.x - list.first[t]) * list.chunk[t], end = min(list.n[t], base + list.chunk[t]);
    const float *const m = list.momentum[t], *const g = list.grad[t];
    float *const x = list.x[t];
    for (long long i = base + threadIdx.x; i < end; i += kThreads) x[i] = (m ? update_of(g[i], m[i], mu, nesterov) : g[i]) * inverse.first * inverse.second;
}

__global__ void __launch_bounds__(kThreads)
muon_update_kernel(const __grid_constant__ List list, float decay) {
    grid_dependency_trigger();
    grid_dependency_wait();
    const int t = find(list, blockIdx.x);
    const long long base = static_cast<long long>(blockIdx.x - list.first[t]) * list.chunk[t], end = min(list.n[t], base + list.chunk[t]);
    float *const p = list.param[t];
    const float *const x = list.x[t];
    const float scale = list.scale[t];
    for (long long i = base + threadIdx.x; i < end; i += kThreads) p[i] = fmaf(-scale, x[i], decay * p[i]);
}

// x in f16 planes, hi + lo * 2^-12, 8 columns a thread.  Bound by memory: 8 bytes read (4 without a momentum), 4 written.  scale: 2^exponent.
// A block takes the same chunk of a matrix as above, counted in vectors.
__global__ void __launch_bounds__(kThreads)
muon_planes_kernel(const __grid_constant__ List list, float mu, bool nesterov, float eps, const double *__restrict__ partial, float scale) {
    __shared__ double red[8];
    grid_dependency_trigger();
    grid_dependency_wait();
    const int t = find(list, blockIdx.x), rows = list.rows[t], cols = list.cols[t];
    const Inverse inverse = inverse_norm(list, t, partial, eps, red);
    const float first = inverse.first, second = inverse.second * scale;
    const float *const m = list.momentum[t], *const g = list.grad[t];
    uint16_t *const dst = list.planes[t];
    const FastDiv per_row = list.vectors[t];
    const int vectors = static_cast<int>(per_row.d) * rows, blocks = static_cast<int>(list.first[t + 1] - list.first[t]);
    const int per_block = ((vectors + blocks - 1) / blocks + kThreads - 1) / kThreads * kThreads;
    const int v0 = static_cast<int>(min(static_cast<long long>(vectors), static_cast<long long>(blockIdx.x - list.first[t]) * per_block)), v1 = min(vectors, v0 + per_block);
    const bool vec = ((reinterpret_cast<uintptr_t>(m) | reinterpret_cast<uintptr_t>(g)) & 15) == 0 && cols % 4 == 0;
    for (int v = v0 + threadIdx.x; v < v1; v += kThreads) {
        const int row = fd_div(v, per_row), col = (v - row * static_cast<int>(per_row.d)) * 8;
        const long long at = static_cast<long long>(row) * cols + col;
        float x[8], y[8];
        if (vec && col + 8 <= cols) {
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const float4 a = __ldg(reinterpret_cast<const float4 *>(g + at) + h);
                x[4 * h] = a.x; x[4 * h + 1] = a.y; x[4 * h + 2] = a.z; x[4 * h + 3] = a.w;
                if (m) {
                    const float4 b = __ldcg(reinterpret_cast<const float4 *>(m + at) + h);
                    y[4 * h] = b.x; y[4 * h + 1] = b.y; y[4 * h + 2] = b.z; y[4 * h + 3] = b.w;
                }
            }
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                x[i] = col + i < cols ? __ldg(g + at + i) : 0.f;
                if (m) y[i] = col + i < cols ? __ldcg(m + at + i) : 0.f;
            }
        }
        uint4 hi, lo;
        unsigned *const h = &hi.x, *const l = &lo.x;
#pragma unroll
        for (int i = 0; i < 8; i += 2) {
            const float a = (m ? update_of(x[i], y[i], mu, nesterov) : x[i]) * first * second, b = (m ? update_of(x[i + 1], y[i + 1], mu, nesterov) : x[i + 1]) * first * second;
            const __half2 top = __floats2half2_rn(a, b);
            const float2 back = __half22float2(top);
            constexpr float up = 1 << kHalfLoShift;
            const __half2 rest = __floats2half2_rn((a - back.x) * up, (b - back.y) * up);
            h[i / 2] = *reinterpret_cast<const unsigned *>(&top);
            l[i / 2] = *reinterpret_cast<const unsigned *>(&rest);
        }
        uint16_t *const to = dst + static_cast<long long>(v) * 8;
        *reinterpret_cast<uint4 *>(to) = hi;
        *reinterpret_cast<uint4 *>(to + list.plane[t]) = lo;
    }
}

int64_t chunk_of(int64_t n) {
    const int64_t each = (n + kMaxChunks - 1) / kMaxChunks;
    return std::max<int64_t>(kChunk, (each + kChunk - 1) / kChunk * kChunk);
}
int64_t chunks_of(int64_t n) { return (n + chunk_of(n) - 1) / chunk_of(n); }

// Calls launch(list, chunks, chunks before) for stretches of the entries that fit a launch.
template <class Launch>
int for_lists(const MuonEntry *e, int64_t count, Launch launch) {
    int64_t before = 0;
    for (int64_t at = 0; at < count;) {
        List list;
        int64_t chunks = 0;
        int k = 0;
        for (; at < count && k < kMaxList; ++at) {
            if (e[at].n == 0) continue;
            list.param[k] = e[at].param;
            list.momentum[k] = e[at].momentum;
            list.x[k] = e[at].x;
            list.grad[k] = e[at].grad;
            list.n[k] = e[at].n;
            list.scale[k] = e[at].scale;
            list.planes[k] = e[at].planes;
            list.plane[k] = e[at].plane;
            list.vectors[k] = make_fastdiv(std::max<int64_t>(1, e[at].pitch / 8));
            list.rows[k] = static_cast<int>(e[at].rows);
            list.cols[k] = static_cast<int>(e[at].cols);
            list.chunk[k] = static_cast<int>(chunk_of(e[at].n));
            list.first[k] = static_cast<unsigned>(chunks);
            chunks += chunks_of(e[at].n);
            ++k;
        }
        if (k == 0) break;
        list.first[k] = static_cast<unsigned>(chunks);
        list.count = k;
        const int rc = launch(list, static_cast<unsigned>(chunks), before);
        if (rc) return rc;
        before += chunks;
    }
    return MNI_B200_OK;
}

}  // namespace

size_t muon_partial_bytes(const MuonEntry *e, int64_t count) {
    int64_t chunks = 0;
    for (int64_t i = 0; i < count; ++i) chunks += e[i].n ? chunks_of(e[i].n) : 0;
    return static_cast<size_t>(chunks) * sizeof(double);
}

int launch_muon_start(const MuonEntry *e, int64_t count, float mu, bool nesterov, float eps, double *partial, int exponent, unsigned *counters,
                      int words, cudaStream_t stream) {
    int rc = for_lists(e, count, [&](const List &list, unsigned chunks, int64_t before) -> int {
        const cudaError_t r = launch_dependent(muon_momentum_kernel, dim3(chunks), dim3(kThreads), 0, stream, list, mu, nesterov, partial + before,
                                               counters, words);
        if (r != cudaSuccess) return fail(MNI_B200_ERR_CUDA, "muon_momentum_kernel launch failed: %s", cudaGetErrorString(r));
        MNI_LAUNCH_CHECK("muon_momentum_kernel");
        return MNI_B200_OK;
    });
    if (rc) return rc;
    return for_lists(e, count, [&](const List &list, unsigned chunks, int64_t before) -> int {
        const double *const sums = partial + before;
        const cudaError_t r = list.planes[0]
                                  ? launch_dependent(muon_planes_kernel, dim3(chunks), dim3(kThreads), 0, stream, list, mu, nesterov, eps, sums, ldexpf(1.f, exponent))
                                  : launch_dependent(muon_normalise_kernel, dim3(chunks), dim3(kThreads), 0, stream, list, mu, nesterov, eps, sums);
        if (r != cudaSuccess) return fail(MNI_B200_ERR_CUDA, "muon_planes_kernel launch failed: %s", cudaGetErrorString(r));
        MNI_LAUNCH_CHECK("muon_planes_kernel");
        return MNI_B200_OK;
    });
}

int launch_muon_update(const MuonEntry *e, int64_t count, float decay, cudaStream_t stream) {
    return for_lists(e, count, [&](const List &list, unsigned chunks, int64_t) -> int {
        const cudaError_t r = launch_dependent(muon_update_kernel, dim3(chunks), dim3(kThreads), 0, stream, list, decay);
        if (r != cudaSuccess) return fail(MNI_B200_ERR_CUDA, "muon_update_kernel launch failed: %s", cudaGetErrorString(r));
        MNI_LAUNCH_CHECK("muon_update_kernel");
        return MNI_B200_OK;
    });
}

}  // namespace mni
