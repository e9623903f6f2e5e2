// Newton-Schulz steps on a list of matrices in one launch:  A = x x^T, R = b + c A;  Q = a + A R;  x <- Q x  (A = x^T x and x <- x Q for
// matrices with more rows than columns), `steps` times.  All matrices are in 16-bit planes (hi + lo * 2^-12, half.cu) at scales that are
// known beforehand; products are three passes of tcgen05.mma.kind::f16 with the large terms drained from their accumulator every 128
// elements (gemm_tcgen05.cu: kHalfDrain).
//
// A unit is one output tile of one of a step's three products of one matrix.  Units are numbered step by step, product by product, and
// CTAs (pairs) draw them in that order from a counter; a unit waits until the units of its matrix's product before have been counted as
// done.  It waits only for units of lower numbers, which have been drawn already, so the lowest unfinished one can always run.  So
// products of different matrices, steps and shapes fill each other's gaps: as one launch for each product and shape, each waiting
// for the one before, thirty matrices of 512 x 512 and 512 x 2048 took 1290 us, of which the pipe worked 260.
//
//   warp 0, 1   TMA producers of A and of B (both wait for the unit's matrix, then order the other CTAs' stores before their copies)
//   warp 2      issues the MMAs (of a pair: the leader's; the peer's draws the units)
//   warp 3      pair: relays "landed" to the leader; lone CTA: draws the units
//   warp 4-11   epilogue: planes of the result, by TMA from the warp's patch, or f32: the orthogonal matrix, or the parameter that it
//               updates.  Plain stores of a thread's own row (32 rows a store) took 70 clocks each, 11000 for a 256 x 256 tile, in which
//               nobody drained the next tile's accumulators.
//
// Of a symmetric result only the tiles on and above the diagonal are computed, and only they are written: a block of 64 contraction elements
// that lies below is loaded from above and given to the tensor core as what it is, MN-major.
//
// Tiles: 256 x 256 of a pair (24.4 clocks an element of the contraction: the pipe's 24), 128 x 128 of a lone CTA (24: its shared memory
// feeds half of the pipe) or 128 x 64 (15, 20 with its operands from L2).  The smaller ones have less to do in the chain of a single matrix,
// the large ones do twice as much a clock: tiling() weighs the two.
//
// What bounds it.  One matrix: the chain of 15 products, each of which takes its contraction (16000 clocks at 768), 1200 for the first operands,
// 700 for the accumulators, 2500 for the planes, 1500 until they are counted and 2000 until the others see that; 768 x 768 takes 201 us,
// 64 x 32 62 to 66; of a thin one the long side is one contraction of one or a few tiles (128 x 4096 304, 64 x 8192 523).  Many: thirty matrices of 512 x 512 and 512 x 2048 take 725 us as a whole step in a loop.  This launch by itself is 570 of them, the
// pipe busy for 45 %, L2 at 8.1 TB/s, 1.2 GB from and to DRAM (their planes are 220 MB, more than L2 holds): a tile of 512 elements takes 12500 clocks of the pipe and 10000 of its epilogue, during which the next tile's
// accumulators can only fill once.
#include "fused_epilogue.h"
#include "internal.h"
#include "tcgen05.h"

#include <algorithm>
#include <atomic>
#include <cmath>
#include <cstdlib>

namespace mni {

namespace {

constexpr int BM = 128, BK = 64, kStagesMax = 8, kEpiWarps = 8, kPatchBytes = 4096, kRing = 2;
constexpr int kPieceBlocks = 2;                    // k-blocks whose large terms share an accumulator's chain: 128 elements
constexpr int kThreads = 32 * (4 + kEpiWarps);
constexpr int kLaunchRegs = 168;                   // a thread has at launch; launch() checks that the compiler took no fewer
constexpr int kIssueRegs = 56, kEpiRegs = 224;
static_assert(kThreads * kLaunchRegs <= 65536 && kIssueRegs + 2 * kEpiRegs <= 3 * kLaunchRegs, "more registers than the launch has");
static_assert(2 * 25 * kNewtonLongest <= kWaitCycles, "a wait for one tile may run out");
constexpr int kBars = 3 * kStagesMax + 4 + 2 * kRing + 1;
constexpr int kFixedSmem = 1024 + kEpiWarps * kPatchBytes + kBars * 8 + 64;

struct Group {
    CUtensorMap a1[2], b1[2], x3[2];               // x, by the step's parity
    CUtensorMap a2[2], b2[2], q3[2];               // A, R and Q, contraction along rows and along columns
    CUtensorMap to_x[2], to_a, to_r, to_q;         // what the epilogue writes
    int rows, cols, side, count, tall;
    int first_matrix;
    int tiles1, tn1, tm3, tn3;                     // tiles of a symmetric product (on and above the diagonal), its columns of tiles; of x
    int begin[3];                                  // index of the group's first unit in each product
};
struct Step {
    float a, r, r_diagonal, q, q_diagonal, x;
};
struct Args {
    Group g[kNewtonGroups];
    Step step[kNewtonSteps];
    float *out[kNewtonMatrices];
    float scale[kNewtonMatrices];
    int groups, steps, units[3];
    int update;                                    // out is a parameter: out = decay * out - scale * x
    float decay;
    unsigned *ticket, *done;                       // done[3 * matrix + product]: warps that have written their part of a tile
    unsigned *err;
    long long wait_cycles;
    int withhold_at;                               // test hook, as KParams::withhold_at
    int stages;
};

struct Unit {
    int step, product, matrix, tm, tn;             // matrix: within the group
    const Group *g;
};
template <int RATIO>
__device__ __forceinline__ Unit decode(const Args &p, int u) {
    Unit t;
    const int per_step = p.units[0] + p.units[1] + p.units[2];
    t.step = u / per_step;
    int r = u - t.step * per_step;
    t.product = 0;
    while (r >= p.units[t.product]) r -= p.units[t.product++];
    int at = 0;
    while (at + 1 < p.groups && r >= p.g[at + 1].begin[t.product]) ++at;
    t.g = &p.g[at];
    r -= t.g->begin[t.product];
    if (t.product < 2) {
        t.matrix = r / t.g->tiles1;
        r -= t.matrix * t.g->tiles1;
        t.tm = 0;
        for (int row = t.g->tn1; r >= row; row -= RATIO) {
            r -= row;
            ++t.tm;
        }
        t.tn = RATIO * t.tm + r;
    } else {
        const int tiles = t.g->tm3 * t.g->tn3;
        t.matrix = r / tiles;
        r -= t.matrix * tiles;
        t.tn = r / t.g->tm3;
        t.tm = r - t.tn * t.g->tm3;
    }
    return t;
}
__device__ __forceinline__ int contraction(const Unit &t) {
    return t.product == 0 ? (t.g->tall ? t.g->rows : t.g->cols) : t.g->side;
}

// How an operand's block of 64 contraction elements lies in memory.  Of a symmetric matrix the blocks of `TM` rows below the diagonal are
// never written: they are read as what lies above it, turned.
struct Major {
    bool symmetric, mn;
    int block;                                     // of TM rows
    template <int TM>
    __device__ __forceinline__ bool mn_at(int it) const { return symmetric ? it / (TM / BK) < block : mn; }
};
template <int RATIO>
__device__ __forceinline__ Major major_of(const Unit &t, bool of_a) {
    const bool tall = t.g->tall != 0;
    Major m;
    m.symmetric = t.product == 1 || (t.product == 2 && tall != of_a);
    m.mn = t.product == 0 ? tall : !of_a;          // (of x: behind Q it is read along its rows, before Q along its columns)
    m.block = of_a ? t.tm : t.tn / RATIO;
    return m;
}

// Waits with the reach of a cluster, for what another CTA of it has stored before it arrived.
__device__ __forceinline__ bool wait_cluster(uint32_t bar, uint32_t parity, volatile uint32_t *abort_flag, unsigned *err, uint32_t code, long long limit) {
    long long t0 = 0;
    for (uint32_t spins = 0;; ++spins) {
        uint32_t ok;
        asm volatile(
            "{\n\t.reg .pred p;\n\t"
            "mbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2;\n\t"
            "selp.u32 %0, 1, 0, p;\n\t}"
            : "=r"(ok)
            : "r"(bar), "r"(parity)
            : "memory");
        if (ok) return true;
        if (spins == 0) t0 = clock64();
        if ((spins & 63u) == 63u) {
            if (*abort_flag) return false;
            if (clock64() - t0 > limit) {
                *abort_flag = 1u;
                atomicCAS(err, 0u, code);
                return false;
            }
        }
    }
}
__device__ __forceinline__ uint32_t in_cta(uint32_t addr, uint32_t cta) {
    uint32_t r;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(addr), "r"(cta));
    return r;
}
__device__ __forceinline__ void arrive_cluster(uint32_t cluster_addr) {
    asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(cluster_addr) : "memory");
}

template <int BN, int CG>
__global__ void __launch_bounds__(kThreads, 1)
newton_schulz_kernel(const __grid_constant__ Args p) {
    constexpr int TM = BM * CG, RATIO = TM / BN, BNL = BN / CG;
    static_assert(TM % BN == 0 && (BNL == 128 || BNL == 64), "tiles of a symmetric product nest, boxes are 64 or 128 rows");
    constexpr uint32_t A_BYTES = BM * BK * 2, B_BYTES = BNL * BK * 2, STAGE = A_BYTES + B_BYTES, STAGE16 = STAGE >> 4;
    constexpr int CHUNKS = BN / 64;                // of 32 columns, of each of the two warps of a lane quarter
    constexpr uint32_t TMEM_COLS = 2 * BN;         // large and small terms

    extern __shared__ uint8_t smem_raw[];
    uint8_t *const smem = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
    uint8_t *const patches = smem + static_cast<size_t>(p.stages) * STAGE;
    uint64_t *const bars = reinterpret_cast<uint64_t *>(patches + kEpiWarps * kPatchBytes);
    const uint32_t bar_full = smem_u32(bars), bar_ready = bar_full + 8u * kStagesMax, bar_empty = bar_ready + 8u * kStagesMax,
                   acc_full = bar_empty + 8u * kStagesMax, acc_empty = acc_full + 16u, unit_full = acc_empty + 16u, unit_empty = unit_full + 8u * kRing,
                   issued = unit_empty + 8u * kRing;
    volatile int *const ring = reinterpret_cast<int *>(bars + kBars);
    uint32_t *const tmem_slot = reinterpret_cast<uint32_t *>(bars + kBars) + kRing;
    volatile uint32_t *const abort_flag = tmem_slot + 1;

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t rank = CG == 2 ? cluster_ctarank() : 0u;
    constexpr uint32_t kDrawer = CG - 1;           // the CTA that draws the units

    if (threadIdx.x == 0) {
        grid_dependency_trigger();
        for (int s = 0; s < p.stages; ++s) {
            mbar_init(bar_full + 8u * s, 1);
            mbar_init(bar_ready + 8u * s, CG);
            mbar_init(bar_empty + 8u * s, 1);
        }
        for (int i = 0; i < 2; ++i) {
            mbar_init(acc_full + 8u * i, 1);
            mbar_init(acc_empty + 8u * i, CG * kEpiWarps);
        }
        // readers of a drawn unit: both producers and the epilogue; the MMA issuer of the leader; the relays of a pair
        for (int i = 0; i < kRing; ++i) {
            mbar_init(unit_full + 8u * i, 1);
            mbar_init(unit_empty + 8u * i, CG * (2 + kEpiWarps) + 1 + (CG == 2 ? 2 : 0));
        }
        mbar_init(issued, 1);
        *abort_flag = 0u;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    }
    if (warp == 2) {
        if constexpr (CG == 2) {
            asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)), "r"(TMEM_COLS) : "memory");
            asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
        } else {
            asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)), "r"(TMEM_COLS) : "memory");
            asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
        }
    }
    tc_fence_before();
    __syncthreads();
    if constexpr (CG == 2) cluster_sync_all();
    tc_fence_after();
    const uint32_t tmem_base = *tmem_slot;
    grid_dependency_wait();

    const int total = p.steps * (p.units[0] + p.units[1] + p.units[2]);
    long long unused = 0;
    // The next unit of this CTA (pair), -1 at the end (and when giving up).  n: how many this warp has had.
    auto next_unit = [&](int n) {
        const int slot = n % kRing;
        bool ok = wait_cluster(unit_full + 8u * slot, (n / kRing) & 1, abort_flag, p.err, 0x700u | slot, p.wait_cycles);
        ok = __all_sync(0xffffffffu, ok);
        const int u = ok ? ring[slot] : -1;
        __syncwarp();
        if (lane == 0) arrive_cluster(in_cta(unit_empty + 8u * slot, kDrawer));
        return u;
    };

    if (warp >= 4) {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kEpiRegs));
        // ------------------------------------------------------------ epilogue
        const int ew = warp - 4, quarter = warp & 3, half = ew >> 2;
        float *const patch = reinterpret_cast<float *>(patches + ew * kPatchBytes);
        const uint32_t large = tmem_base + (static_cast<uint32_t>(quarter * 32) << 16) + half * (BN / 2), small = large + BN;
        uint32_t run[CHUNKS][32];
        int pieces_seen = 0;
        bool ok = true;
        auto wait_full = [&](int slot, uint32_t phase) {
            ok = mbar_wait_warp(acc_full + 8u * slot, phase, abort_flag, p.err, 0x500u | slot, unused, false, p.wait_cycles);
            tc_fence_after();
            return ok;
        };
        auto release = [&](int slot) {
            tc_fence_before();
            __syncwarp();
            if (lane == 0) {
                if (CG == 2 && rank != 0) mbar_arrive_cta(acc_empty + 8u * slot, 0u);
                else mbar_arrive(acc_empty + 8u * slot);
            }
        };
        auto take = [&](uint32_t from, float scale, bool add) {
#pragma unroll
            for (int c = 0; c < 2 * CHUNKS; ++c) {
                uint32_t x[16];
                tmem_ld16_issue(from + c * 16, x);
                tmem_ld_wait();
#pragma unroll
                for (int e = 0; e < 16; ++e) {
                    uint32_t &r = run[c / 2][(c & 1) * 16 + e];
                    r = __float_as_uint(fmaf(__uint_as_float(x[e]), scale, add ? __uint_as_float(r) : 0.f));
                }
            }
        };
        // alpha * (the first chunk of run) + beta on the diagonal, in planes, to where `map` lies: a half of the patch each
        auto put = [&](const CUtensorMap *map, float alpha, float beta, int diagonal, int col, int row, int matrix) {
            uint32_t x[2][16];
#pragma unroll
            for (int e = 0; e < 32; e += 2)
                split_pair(fmaf(alpha, __uint_as_float(run[0][e]), diagonal == e ? beta : 0.f),
                           fmaf(alpha, __uint_as_float(run[0][e + 1]), diagonal == e + 1 ? beta : 0.f), x[0][e / 2], x[1][e / 2]);
#pragma unroll
            for (int plane = 0; plane < 2; ++plane) {
                if (lane == 0) asm volatile("cp.async.bulk.wait_group.read 1;" ::: "memory");      // what this half held has been read
                __syncwarp();
                uint8_t *const to = reinterpret_cast<uint8_t *>(patch) + plane * (kPatchBytes / 2) + lane * 64;
#pragma unroll
                for (int k = 0; k < 4; ++k)
                    *reinterpret_cast<uint4 *>(to + ((k ^ ((lane >> 1) & 3)) * 16)) = make_uint4(x[plane][4 * k], x[plane][4 * k + 1], x[plane][4 * k + 2], x[plane][4 * k + 3]);
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                __syncwarp();
                if (lane == 0) {
                    tma_store_planes(map, smem_u32(patch) + plane * (kPatchBytes / 2), col, row, matrix, plane);
                    asm volatile("cp.async.bulk.commit_group;" ::: "memory");
                }
            }
        };
        for (int n = 0; ok; ++n) {
            const int u = next_unit(n);
            if (u < 0) break;
            const Unit t = decode<RATIO>(p, u);
            const Group &g = *t.g;
            const int blocks = (contraction(t) + BK - 1) / BK, pieces = (blocks + kPieceBlocks - 1) / kPieceBlocks;
            for (int i = 0; ok && i < pieces; ++i) {
                if (i + 1 == pieces) {
                    if (!wait_full(1, n & 1)) break;
                    take(small, 1.f / (1 << kHalfLoShift), i > 0);
                    release(1);
                }
                if (!wait_full(0, pieces_seen & 1)) break;
                take(large, 1.f, i > 0 || i + 1 == pieces);
                release(0);
                ++pieces_seen;
            }
            if (!ok) break;
            const bool of_x = t.product == 2, last = of_x && t.step + 1 == p.steps;
            const int rows = of_x ? g.rows : g.side, cols = of_x ? g.cols : g.side;
            const int row0 = t.tm * TM + static_cast<int>(rank) * BM + quarter * 32;
            const int col0 = t.tn * BN + half * (BN / 2);
            const Step &s = p.step[t.step];
            const int m = g.first_matrix + t.matrix;
            if (row0 < rows) {
#pragma unroll 1
                for (int c = 0; c < CHUNKS; ++c) {
                    const int col = col0 + 32 * c;
                    if (col >= cols) break;
                    if (!last) {
                        const int diagonal = row0 + lane - col;
                        if (t.product == 0) {
                            put(&g.to_a, s.a, 0.f, diagonal, col, row0, t.matrix);
                            put(&g.to_r, s.r, s.r_diagonal, diagonal, col, row0, t.matrix);
                        } else if (t.product == 1) {
                            put(&g.to_q, s.q, s.q_diagonal, diagonal, col, row0, t.matrix);
                        } else {
                            put(&g.to_x[(t.step + 1) & 1], s.x, 0.f, diagonal, col, row0, t.matrix);
                        }
                    } else {
                        // the result in f32: turned in the patch, so that a store covers 32 neighbouring columns whatever the alignment
                        float *const out = p.out[m] + static_cast<long long>(row0) * cols + col + lane;
                        const float scale = p.scale[m];
                        const int live = col + lane < cols ? min(32, rows - row0) : 0;
                        __syncwarp();
#pragma unroll
                        for (int e = 0; e < 32; ++e) patch[lane * 32 + (e ^ lane)] = __uint_as_float(run[0][e]) * s.x;
                        __syncwarp();
                        constexpr int AT_ONCE = CHUNKS > 2 ? 16 : 32;              // loads in flight: as registers allow
#pragma unroll
                        for (int r0 = 0; r0 < 32; r0 += AT_ONCE) {
                            float y[AT_ONCE];
                            if (p.update) {
#pragma unroll
                                for (int r = 0; r < AT_ONCE; ++r) y[r] = r0 + r < live ? out[static_cast<long long>(r0 + r) * cols] : 0.f;
                            }
#pragma unroll
                            for (int r = 0; r < AT_ONCE; ++r) {
                                const float v = patch[(r0 + r) * 32 + (lane ^ (r0 + r))];
                                if (r0 + r < live) out[static_cast<long long>(r0 + r) * cols] = p.update ? fmaf(-scale, v, p.decay * y[r]) : v;
                            }
                        }
                    }
#pragma unroll
                    for (int d = 1; d < CHUNKS; ++d)
#pragma unroll
                        for (int e = 0; e < 32; ++e) run[d - 1][e] = run[d][e];
                }
            }
            if (!last) {                           // this warp's part is written, before the count
                if (lane == 0) {
                    asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
                    asm volatile("red.release.gpu.global.add.u32 [%0], 1;" ::"l"(p.done + 3 * m + t.product) : "memory");
                }
                __syncwarp();
            }
        }
    } else {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kIssueRegs));
        if (warp < 2) {
            // ------------------------------------------------------------ TMA producers: warp 0 of A, warp 1 of B
            const bool loads_a = warp == 0;
            const uint32_t base = smem_u32(smem) + (loads_a ? 0u : A_BYTES);
            int stage = 0, armed = 0;
            uint32_t phase = 0;
            bool ok = true;
            for (int n = 0; ok; ++n) {
                const int u = next_unit(n);
                if (u < 0) break;
                const Unit t = decode<RATIO>(p, u);
                const Group &g = *t.g;
                // what the unit reads: x of this step, A and R, or Q
                if (t.product > 0 || t.step > 0) {
                    const int before = t.product == 0 ? 2 : t.product - 1;
                    const unsigned tiles = static_cast<unsigned>(before == 2 ? g.tm3 * g.tn3 : g.tiles1);
                    const unsigned want = tiles * static_cast<unsigned>(t.product == 0 ? t.step : t.step + 1) * (CG * kEpiWarps);
                    // Every lane acquires the count itself, as any of them may issue the copies; the vote orders no memory.  (Lane 0 alone and a
                    // __syncwarp: 768 x 768 207 us for 201.)
                    const unsigned *const done = p.done + 3 * (g.first_matrix + t.matrix) + before;
                    const long long t0 = clock64();
                    while (true) {
                        unsigned seen;
                        asm volatile("ld.acquire.gpu.global.u32 %0, [%1];" : "=r"(seen) : "l"(done) : "memory");
                        if (seen >= want) break;
                        if (*abort_flag || clock64() - t0 > p.wait_cycles) {
                            *abort_flag = 1u;
                            atomicCAS(p.err, 0u, 0x800u | static_cast<unsigned>(t.product));
                            ok = false;
                            break;
                        }
                    }
                    ok = __all_sync(0xffffffffu, ok);
                    if (!ok) break;
                    asm volatile("fence.proxy.async;" ::: "memory");       // their stores before the copies of whichever lane issues them
                }
                const int blocks = (contraction(t) + BK - 1) / BK, parity = t.step & 1;
                const Major major = major_of<RATIO>(t, loads_a);
                const CUtensorMap *const along = loads_a ? (t.product == 0 ? &g.a1[parity] : t.product == 1 ? &g.a2[0] : g.tall ? &g.x3[parity] : &g.q3[0])
                                                         : (t.product == 0 ? &g.b1[parity] : t.product == 1 ? &g.b2[0] : g.tall ? &g.q3[0] : &g.x3[parity]);
                const int row = loads_a ? t.tm * TM + static_cast<int>(rank) * BM : t.tn * BN + static_cast<int>(rank) * BNL;
                for (int it = 0; ok && it < blocks; ++it) {
                    const bool mn = major.mn_at<TM>(it);
                    const CUtensorMap *const map = along + (major.symmetric && mn ? 1 : 0);
                    for (int plane = 0; plane < 2; ++plane) {
                        ok = mbar_wait_warp(bar_empty + 8u * stage, phase ^ 1u, abort_flag, p.err, 0x100u | stage, unused, false, p.wait_cycles);
                        if (!ok) break;
                        const uint32_t full = bar_full + 8u * stage;
                        ++armed;
                        if (elect_one()) {
                            if (loads_a) mbar_arrive_expect_tx(full, STAGE);
                            if (armed != p.withhold_at) {
                                const uint32_t dst = base + stage * STAGE;
                                if (mn) tma_load_5d(dst, map, full, 0, it * BK, row >> 6, t.matrix, plane);
                                else tma_load_5d(dst, map, full, it * BK, row, t.matrix, plane, 0);
                            }
                        }
                        if (++stage == p.stages) { stage = 0; phase ^= 1u; }
                    }
                }
                if (!loads_a && rank == kDrawer && lane == 0) mbar_arrive(issued);
            }
            if (!ok) {                             // giving up: copies already issued land before the CTA exits
                const int pending = min(armed, p.stages);
                for (int i = 0; i < pending; ++i) {
                    if (--stage < 0) { stage = p.stages - 1; phase ^= 1u; }
                    const long long t0 = clock64();
                    while (!mbar_try_wait(bar_full + 8u * stage, phase) && clock64() - t0 < p.wait_cycles / 8) {}
                }
            }
        } else if (warp == 2 && rank == 0) {
            // ------------------------------------------------------------ MMA issuer
            const uint32_t desc_hi = ((1024u >> 4) & 0x3FFFu) | (1u << 14) | (2u << 29);           // SBO 1024, version 1, SWIZZLE_128B
            const uint32_t sa = (smem_u32(smem) >> 4) & 0x3FFFu, sb = ((smem_u32(smem) + A_BYTES) >> 4) & 0x3FFFu;
            const uint32_t ready = CG == 1 ? bar_full : bar_ready;
            int stage = 0, pieces_seen = 0;
            uint32_t phase = 0;
            bool ok = true;
            for (int n = 0; ok; ++n) {
                const int u = next_unit(n);
                if (u < 0) break;
                const Unit t = decode<RATIO>(p, u);
                const Major a_major = major_of<RATIO>(t, true), b_major = major_of<RATIO>(t, false);
                const int blocks = (contraction(t) + BK - 1) / BK;
                for (int it = 0; it < blocks; ++it) {
                    const bool a_mn = a_major.mn_at<TM>(it), b_mn = b_major.mn_at<TM>(it);
                    const uint32_t lbo = static_cast<uint32_t>((BK * 128) >> 4) << 16;             // MN-major: chunks of 64 rows
                    const uint32_t a0 = sa | (a_mn ? lbo : 0u), b0 = sb | (b_mn ? lbo : 0u), a_ks = a_mn ? 128u : 2u, b_ks = b_mn ? 128u : 2u;
                    const uint32_t idesc = (1u << 4) | (a_mn ? 1u << 15 : 0u) | (b_mn ? 1u << 16 : 0u) | (static_cast<uint32_t>(BN >> 3) << 17) |
                                           (static_cast<uint32_t>(TM >> 4) << 24);
                    const int in_piece = it % kPieceBlocks;
                    const bool begins = in_piece == 0, last = it + 1 == blocks, ends = last || in_piece + 1 == kPieceBlocks, large_first = ends && !last;
                    ok = mbar_wait_warp(ready + 8u * stage, phase, abort_flag, p.err, 0x300u | stage, unused, false, p.wait_cycles);
                    if (!ok) break;
                    const uint32_t hi_stage = static_cast<uint32_t>(stage), ah = a0 + hi_stage * STAGE16, bh = b0 + hi_stage * STAGE16;
                    auto large = [&] {
                        if (begins) {
                            ok = mbar_wait_warp(acc_empty, (pieces_seen & 1) ^ 1u, abort_flag, p.err, 0x200u, unused, false, p.wait_cycles);
                            if (!ok) return;
                        }
                        tc_fence_after();
                        if (elect_one()) {
#pragma unroll
                            for (int ks = 0; ks < BK / 16; ++ks)
                                umma_f16<CG>(tmem_base, ah + ks * a_ks, desc_hi, bh + ks * b_ks, desc_hi, idesc, begins && ks == 0 ? 0u : 1u);
                            if (ends) commit_to<CG>(acc_full);
                        }
                        __syncwarp();
                    };
                    if (large_first) {
                        large();
                        if (!ok) break;
                    }
                    if (++stage == p.stages) { stage = 0; phase ^= 1u; }
                    if (it == 0) {
                        ok = mbar_wait_warp(acc_empty + 8u, (n & 1) ^ 1u, abort_flag, p.err, 0x201u, unused, false, p.wait_cycles);
                        if (!ok) break;
                    }
                    ok = mbar_wait_warp(ready + 8u * stage, phase, abort_flag, p.err, 0x300u | stage, unused, false, p.wait_cycles);
                    if (!ok) break;
                    tc_fence_after();
                    if (elect_one()) {
                        const uint32_t al = a0 + stage * STAGE16, bl = b0 + stage * STAGE16;
#pragma unroll
                        for (int ks = 0; ks < BK / 16; ++ks) {
                            umma_f16<CG>(tmem_base + BN, al + ks * a_ks, desc_hi, bh + ks * b_ks, desc_hi, idesc, it == 0 && ks == 0 ? 0u : 1u);
                            umma_f16<CG>(tmem_base + BN, ah + ks * a_ks, desc_hi, bl + ks * b_ks, desc_hi, idesc, 1u);
                        }
                        commit_to<CG>(bar_empty + 8u * stage);
                        if (large_first) commit_to<CG>(bar_empty + 8u * hi_stage);
                        if (last) commit_to<CG>(acc_full + 8u);
                    }
                    __syncwarp();
                    if (++stage == p.stages) { stage = 0; phase ^= 1u; }
                    if (!large_first) {
                        large();
                        if (!ok) break;
                        if (elect_one()) commit_to<CG>(bar_empty + 8u * hi_stage);
                        __syncwarp();
                    }
                    if (ends) ++pieces_seen;
                }
            }
        } else if (warp == 2 ? CG == 2 : CG == 1) {
            // ------------------------------------------------------------ draws the units
            // One at a time, when the copies of the one before are on their way: a CTA that held two tiles of a matrix's product while others
            // had none made the chain of a single matrix half as long again (one of 256 x 256: 204 us).
            bool ok = true;
            for (int n = 0; ok; ++n) {
                if (n > 0) {
                    ok = mbar_wait_warp(issued, (n - 1) & 1, abort_flag, p.err, 0xa00u, unused, false, p.wait_cycles);
                    if (!ok) break;
                }
                const int slot = n % kRing;
                ok = wait_cluster(unit_empty + 8u * slot, ((n / kRing) & 1) ^ 1u, abort_flag, p.err, 0x900u | slot, p.wait_cycles);
                ok = __all_sync(0xffffffffu, ok);
                if (!ok) break;
                int u = 0;
                if (lane == 0) {
                    const unsigned drawn = atomicAdd(p.ticket, 1u);
                    u = drawn < static_cast<unsigned>(total) ? static_cast<int>(drawn) : -1;
                    for (uint32_t cta = 0; cta < CG; ++cta) {
                        const uint32_t to = in_cta(smem_u32(const_cast<int *>(ring) + slot), cta);
                        asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(to), "r"(u) : "memory");
                        arrive_cluster(in_cta(unit_full + 8u * slot, cta));
                    }
                }
                u = __shfl_sync(0xffffffffu, u, 0);
                if (u < 0) break;
            }
        } else if (CG == 2 && warp == 3) {
            // ------------------------------------------------------------ tells the leader what has landed here
            int stage = 0;
            uint32_t phase = 0;
            bool ok = true;
            for (int n = 0; ok; ++n) {
                const int u = next_unit(n);
                if (u < 0) break;
                const int stages = 2 * ((contraction(decode<RATIO>(p, u)) + BK - 1) / BK);
                for (int i = 0; i < stages; ++i) {
                    ok = mbar_wait_warp(bar_full + 8u * stage, phase, abort_flag, p.err, 0x400u | stage, unused, false, p.wait_cycles);
                    if (!ok) break;
                    if (lane == 0) {
                        if (rank != 0) mbar_arrive_cta(bar_ready + 8u * stage, 0u);
                        else mbar_arrive(bar_ready + 8u * stage);
                    }
                    __syncwarp();
                    if (++stage == p.stages) { stage = 0; phase ^= 1u; }
                }
            }
        }
    }

    tc_fence_before();
    __syncthreads();
    if constexpr (CG == 2) cluster_sync_all();     // both CTAs are done with the pair's tensor memory and barriers
    if (warp == 2) {
        __syncwarp();
        tc_fence_after();
        if constexpr (CG == 2) asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"(TMEM_COLS) : "memory");
        else asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"(TMEM_COLS) : "memory");
    }
}

// ------------------------------------------------------------------ host side
struct Tiling {
    int bn, cg;
    double clocks_k, round;        // of a unit: per contraction element (with operands from L2), and beside its main loop where units follow one another
    double chain;                  // of a product in the chain of one matrix: count, first operands, epilogue
};
constexpr Tiling kTilings[] = {{256, 2, 24.4, 8000, 17000}, {128, 1, 24.0, 5000, 9500}, {64, 1, 20.0, 3000, 9500}};

int64_t symmetric_tiles(int64_t side, int tm, int bn) {
    const int64_t m = (side + tm - 1) / tm, n = (side + bn - 1) / bn, ratio = tm / bn;
    int64_t tiles = 0;
    for (int64_t i = 0; i < m; ++i) tiles += std::max<int64_t>(0, n - ratio * i);
    return tiles;
}

// The tiling whose estimate is least: the rounds of all units, or the chain of the longest matrix, whichever is more, and some of the other.
// us with tiles of 64 / 128 / 256 columns: one matrix of 256 x 256 118 / 144 / 203, 768 206 / 241 / 303, 1024 258 / 294 / 356, 1536 639 / 414 /
// 469, 2048 1071 / 670 / 614; three of 1001 x 333 182 / 215 / 271; twenty of 512 x 512 and ten of 512 x 2048 and turned 1130 / 839 / 736; six of
// 2048 x 2048 to 2048 x 8192 10000 / 7020 / 5180.
const Tiling &tiling(const NewtonProblem *g, int count, int sm_count) {
    const int env = env_int("MNI_B200_NEWTON_TILE", 0);
    const Tiling *best = nullptr;
    double least = 1e300;
    for (const Tiling &t : kTilings) {
        if (env == t.bn) return t;
        const int tm = BM * t.cg;
        const double slots = std::max(1, sm_count / t.cg);
        double work = 0, chain = 0;
        for (int i = 0; i < count; ++i) {
            const double side = static_cast<double>(g[i].side()), longer = static_cast<double>(std::max(g[i].rows, g[i].cols));
            const double t1 = static_cast<double>(symmetric_tiles(g[i].side(), tm, t.bn)),
                         t3 = static_cast<double>((g[i].rows + tm - 1) / tm) * static_cast<double>((g[i].cols + t.bn - 1) / t.bn);
            auto unit = [&](double k) { return t.clocks_k * std::max(k, 64.0) + t.round; };
            // (products of several shapes fill each other's last round)
            auto rounds = [&](double units) { return count == 1 ? std::ceil(units / slots) : units / slots; };
            const double n = static_cast<double>(g[i].count);
            work += rounds(t1 * n) * (unit(longer) + unit(side)) + rounds(t3 * n) * unit(side);
            chain = std::max(chain, t.clocks_k * (longer + 2 * side) + 3 * t.chain);
        }
        const double time = std::max(work, chain) + 0.3 * std::min(work, chain);
        if (time < least) {
            least = time;
            best = &t;
        }
    }
    return *best;
}

template <int BN, int CG>
cudaError_t launch(const Args &args, int units, size_t smem, int sm_count, cudaStream_t stream) {
    static std::atomic<uint64_t> opted_in{0};      // a bit per device ordinal, as in gemm_tcgen05.cu
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    const uint64_t bit = 1ull << (dev & 63);
    if ((opted_in.load(std::memory_order_acquire) & bit) == 0) {
        e = cudaFuncSetAttribute(newton_schulz_kernel<BN, CG>, cudaFuncAttributeMaxDynamicSharedMemorySize, 227 * 1024);
        if (e != cudaSuccess) return e;
        e = check_launch_registers(reinterpret_cast<const void *>(newton_schulz_kernel<BN, CG>), kLaunchRegs);
        if (e != cudaSuccess) return e;
        opted_in.fetch_or(bit, std::memory_order_release);
    }
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(static_cast<unsigned>(std::min(units, std::max(1, sm_count / CG)) * CG));
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cudaLaunchAttribute attrs[2];
    attrs[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attrs[0].val.programmaticStreamSerializationAllowed = pdl_enabled() ? 1 : 0;
    attrs[1].id = cudaLaunchAttributeClusterDimension;
    attrs[1].val.clusterDim.x = CG;
    attrs[1].val.clusterDim.y = 1;
    attrs[1].val.clusterDim.z = 1;
    cfg.attrs = attrs;
    cfg.numAttrs = CG == 2 ? 2 : 1;
    return cudaLaunchKernelEx(&cfg, newton_schulz_kernel<BN, CG>, args);
}

}  // namespace

int launch_newton_schulz(const NewtonProblem *problems, int count, const NewtonStep *steps, int step_count, float *const *out, const float *scale, bool update,
                         float decay, unsigned *counters, uint32_t *err_word, int sm_count, cudaStream_t stream) {
    if (count > kNewtonGroups || step_count > kNewtonSteps) return fail(MNI_B200_ERR_ARG, "internal: too many groups or steps for a launch");
    const Tiling &t = tiling(problems, count, sm_count);
    const int tm = BM * t.cg;
    Args args;
    args.groups = count;
    args.steps = step_count;
    args.units[0] = args.units[1] = args.units[2] = 0;
    int matrices = 0;
    int64_t units[3] = {0, 0, 0}, most = 0;
    for (int i = 0; i < count; ++i) {
        const NewtonProblem &n = problems[i];
        Group &g = args.g[i];
        const int64_t t1 = symmetric_tiles(n.side(), tm, t.bn), tm3 = (n.rows + tm - 1) / tm, tn3 = (n.cols + t.bn - 1) / t.bn;
        if ((t1 + tm3 * tn3) * n.count * step_count > 0x3fffffffLL || std::max(t1, tm3 * tn3) * step_count * 2 * kEpiWarps > 0x7fffffffLL)
            return fail(MNI_B200_ERR_TOO_LARGE, "matrices of %lld x %lld exceed the kernels' int32 indexing", (long long)n.rows, (long long)n.cols);
        g.rows = static_cast<int>(n.rows);
        g.cols = static_cast<int>(n.cols);
        g.side = static_cast<int>(n.side());
        g.count = static_cast<int>(n.count);
        g.tall = n.tall() ? 1 : 0;
        g.first_matrix = matrices;
        matrices += g.count;
        g.tiles1 = static_cast<int>(t1);
        g.tn1 = static_cast<int>((n.side() + t.bn - 1) / t.bn);
        g.tm3 = static_cast<int>(tm3);
        g.tn3 = static_cast<int>(tn3);
        const int64_t mine[3] = {t1 * n.count, t1 * n.count, tm3 * tn3 * n.count};
        for (int k = 0; k < 3; ++k) {
            g.begin[k] = static_cast<int>(units[k]);
            units[k] += mine[k];
        }
        auto operand = [&](const uint16_t *ptr, bool of_x, bool k_major) {
            HalfOperand o;
            const int64_t rows = of_x ? n.rows : n.side(), cols = of_x ? n.cols : n.side();
            o.ptr = ptr;
            o.k_major = k_major;
            o.rows = k_major ? rows : cols;
            o.kdim = k_major ? cols : rows;
            o.pitch = of_x ? n.x_pitch : n.s_pitch;
            o.matrix = rows * o.pitch;
            o.plane = o.matrix * n.count;
            o.batch = n.count;
            o.planes = 2;
            return o;
        };
        const int b_rows = t.bn / t.cg;
        int rc = MNI_B200_OK;
        auto map = [&](CUtensorMap *to, const uint16_t *ptr, bool of_x, bool k_major, int box_rows) {
            if (rc == MNI_B200_OK) rc = half_operand_map(to, operand(ptr, of_x, k_major), box_rows);
        };
        for (int k = 0; k < 2; ++k) {
            map(&g.a1[k], n.x[k], true, !n.tall(), 128);
            map(&g.b1[k], n.x[k], true, !n.tall(), b_rows);
            map(&g.x3[k], n.x[k], true, n.tall(), n.tall() ? 128 : b_rows);
            map(&g.a2[k], n.a, false, k == 0, 128);
            map(&g.b2[k], n.r, false, k == 0, b_rows);
            map(&g.q3[k], n.q, false, k == 0, n.tall() ? b_rows : 128);
            map(&g.to_x[k], n.x[k], true, true, 32);
        }
        map(&g.to_a, n.a, false, true, 32);
        map(&g.to_r, n.r, false, true, 32);
        map(&g.to_q, n.q, false, true, 32);
        if (rc) return rc;
    }
    if (matrices > kNewtonMatrices) return fail(MNI_B200_ERR_ARG, "internal: too many matrices for a launch");
    if ((units[0] + units[1] + units[2]) * step_count > 0x3fffffffLL) return fail(MNI_B200_ERR_TOO_LARGE, "the list has too many tiles");
    for (int k = 0; k < 3; ++k) {
        args.units[k] = static_cast<int>(units[k]);
        most = std::max(most, units[k]);
    }
    for (int k = 0; k < step_count; ++k) args.step[k] = Step{steps[k].a, steps[k].r, steps[k].r_diagonal, steps[k].q, steps[k].q_diagonal, steps[k].x};
    std::copy(out, out + matrices, args.out);
    std::copy(scale, scale + matrices, args.scale);
    args.update = update ? 1 : 0;
    args.decay = decay;
    args.ticket = counters;
    args.done = counters + 1;
    args.err = err_word;
    const char *w = env_value("MNI_B200_WAIT_CYCLES");
    const long long wc = w ? atoll(w) : 0;
    args.wait_cycles = wc > 0 ? wc : kWaitCycles;
    args.withhold_at = args.wait_cycles <= 200000000LL ? env_int("MNI_B200_TEST_WITHHOLD_KBLOCK", 0) : 0;
    const size_t stage = static_cast<size_t>(BM + t.bn / t.cg) * BK * 2;
    args.stages = static_cast<int>(std::min<size_t>(kStagesMax, (227 * 1024 - kFixedSmem) / stage));
    const size_t smem = kFixedSmem + static_cast<size_t>(args.stages) * stage;
    const int u = static_cast<int>(most);
    const cudaError_t e = t.bn == 256 ? launch<256, 2>(args, u, smem, sm_count, stream)
                          : t.bn == 128 ? launch<128, 1>(args, u, smem, sm_count, stream)
                                        : launch<64, 1>(args, u, smem, sm_count, stream);
    if (e != cudaSuccess) return fail(MNI_B200_ERR_CUDA, "newton_schulz_kernel set-up failed: %s", cudaGetErrorString(e));
    MNI_LAUNCH_CHECK("newton_schulz_kernel");
    return MNI_B200_OK;
}

}  // namespace mni
