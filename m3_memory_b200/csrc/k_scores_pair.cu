// k_scores_pair.cu -- scores of many queries (more than 64) against every row, two CTAs
// a tile.
//
// As in k_scores_tc.cu the rows of x lie along M and the queries along N.  A tile of
// 128 rows and 240 queries takes 46 KB of operands from L2 for every 128 bytes of K,
// 92 bytes a cycle at the tensor cores' rate where L2 gives an SM about 40.  Here a
// cluster of two CTAs (one TPC) computes 256 rows x 240 queries with
// tcgen05.mma.cta_group::2: each CTA holds 128 rows and half of the queries, 31 KB a
// slice, and each keeps its own rows' scores in its own TMEM and stores them.
//
// The first CTA's warp 1 issues every MMA; the second's copies, scale words and
// epilogue report to the first CTA's barriers (copies by complete_tx, threads by
// remote arrivals), and commits arrive at both CTAs' barriers.  The scale bytes of all
// queries are in both CTAs' TMEM, each row's in its own.
#include <cuda_bf16.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <atomic>

#include "scores_tc.cuh"

namespace m3g {
namespace {

constexpr int kN = 240, kHalf = kN / 2;  // queries a tile, and of them in each CTA
constexpr int kQBytes = kHalf * kSlice;
constexpr int kBox = 40;                 // queries a copy: three are a half
constexpr int kStages = 6;
constexpr int kEpi0 = 4, kEpiWarps = 8, kScale0 = 12, kScaleWarps = 4;
constexpr int kThreads = (kScale0 + kScaleWarps) * 32;
constexpr int kAcc = 256, kSf = 2, kSf0 = 240, kSfStep = 256;  // TMEM columns

struct alignas(1024) Smem {
    unsigned char x[kStages][kXBytes];
    unsigned char q[kStages][kQBytes];
    uint64_t full[kStages];   // first CTA: both CTAs' copies of the stage have landed
    uint64_t empty[kStages];  // each CTA: the stage's MMAs are done
    uint64_t accfull[2];      // each CTA
    uint64_t accempty[2];     // first CTA: both epilogues have read it
    uint64_t sffull[kSf];     // first CTA: both CTAs' scale words are in TMEM
    uint64_t sfempty[kSf];    // each CTA
    uint64_t drain;
    uint32_t tmem;
    int abort;
};

struct Params {
    int64_t nq, nx;
    int nk, row_bytes;
    const uint8_t *qs, *xs;
    int64_t lqs, lxs, ld_out;
    float alpha, beta;
    int64_t xtiles, qtiles;
    int per;  // queries a tile (a multiple of 16)
    int* err;
};

__device__ __forceinline__ uint32_t cta_rank() {
    uint32_t r;
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}
__device__ __forceinline__ void cluster_sync() {
    asm volatile("barrier.cluster.arrive.aligned;" ::: "memory");
    asm volatile("barrier.cluster.wait.aligned;" ::: "memory");
}
// The first CTA's copy of a shared variable.
__device__ __forceinline__ uint32_t in_first(const void* p) {
    uint32_t r;
    asm volatile("mapa.shared::cluster.u32 %0, %1, 0;" : "=r"(r) : "r"(smem_u32(p)));
    return r;
}
__device__ __forceinline__ void arrive_at(uint32_t bar) {
    asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(bar)
                 : "memory");
}
// Bounded wait that sees what the other CTA did before it arrived.
__device__ __forceinline__ bool wait_cluster(uint64_t* bar, uint32_t parity, int* abort) {
    uint64_t t0 = 0;
    for (;;) {
        uint32_t ok;
        asm volatile(
            "{\n\t.reg .pred p;\n\t"
            "mbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2, %3;\n\t"
            "selp.u32 %0, 1, 0, p;\n\t}"
            : "=r"(ok)
            : "r"(smem_u32(bar)), "r"(parity), "r"(20000u)
            : "memory");
        if (ok) return true;
        if (*(volatile int*)abort != 0) return false;
        const uint64_t now = global_ns();
        if (t0 == 0) t0 = now;
        if (now - t0 > kWaitLimitNs) break;
    }
    atomicCAS(abort, 0, (int)kErrWaitTimeout);
    return false;
}

// A tile into this CTA's shared memory, counted on the first CTA's barrier.
__device__ __forceinline__ void load_pair(void* dst, const CUtensorMap* map, int x, int y,
                                          uint32_t bar) {
    asm volatile(
        "cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes"
        ".cta_group::2 [%0], [%1, {%2, %3}], [%4];" ::"r"(smem_u32(dst)),
        "l"(map), "r"(x), "r"(y), "r"(bar)
        : "memory");
}

__device__ __forceinline__ void mma_mx2(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc,
                                        uint32_t sfa, uint32_t sfb, bool accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %6, 0;\n\t"
        "tcgen05.mma.cta_group::2.kind::mxf8f6f4.block_scale.scale_vec::1X "
        "[%0], %1, %2, %3, [%4], [%5], p;\n\t}" ::"r"(d),
        "l"(a), "l"(b), "r"(idesc), "r"(sfa), "r"(sfb), "r"((uint32_t)accumulate)
        : "memory");
}
__device__ __forceinline__ void mma_f16_2(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc,
                                          bool accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
        "l"(a), "l"(b), "r"(idesc), "r"((uint32_t)accumulate)
        : "memory");
}
// Arrives at both CTAs' barriers once the MMAs issued so far are done.
__device__ __forceinline__ void commit_both(uint64_t* bar) {
    asm volatile(
        "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64"
        " [%0], %1;" ::"r"(smem_u32(bar)),
        "h"((uint16_t)3)
        : "memory");
}

template <bool F8, class O>
__global__ void __launch_bounds__(kThreads, 1) __cluster_dims__(2, 1, 1)
    scores_pair_kernel(const __grid_constant__ CUtensorMap map_x,
                       const __grid_constant__ CUtensorMap map_q, O* __restrict__ out,
                       const __grid_constant__ Params p) {
    extern __shared__ unsigned char smem_raw[];
    // (the same offset in both CTAs: they run the same kernel)
    Smem& sm = *reinterpret_cast<Smem*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) &
                                        ~uintptr_t(1023));
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t rank = cta_rank();
    if (warp == 0) {
        asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(
                         smem_u32(&sm.tmem)),
                     "r"(512)
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
    }
    if (threadIdx.x == 32) {
        for (int s = 0; s < kStages; ++s) {
            mbar_init(&sm.full[s], 1);
            mbar_init(&sm.empty[s], 1);
        }
        for (int s = 0; s < 2; ++s) {
            mbar_init(&sm.accfull[s], 1);
            mbar_init(&sm.accempty[s], 2 * kEpiWarps);
        }
        for (int s = 0; s < kSf; ++s) {
            mbar_init(&sm.sffull[s], 2 * kScaleWarps);
            mbar_init(&sm.sfempty[s], 1);
        }
        mbar_init(&sm.drain, 1);
        sm.abort = 0;
        fence_mbar_init();
    }
    if (threadIdx.x == 0) {
        prefetch_tensormap(&map_x);
        prefetch_tensormap(&map_q);
    }
    tc_fence_before();
    __syncthreads();
    cluster_sync();
    tc_fence_after();
    const uint32_t tmem = sm.tmem;

    // Tiles t, t + clusters, ..: queries fastest, so the clusters that run at the same
    // time share rows in L2.
    const int64_t tiles = p.xtiles * p.qtiles, clusters = gridDim.x / 2;
    const int64_t first = blockIdx.x / 2;
    struct Tile {
        int64_t x0;  // this CTA's first row (may be past the last)
        int nx, q0, nq, n;
    };
    auto tile_of = [&](int64_t t) {
        Tile r;
        const int64_t xt = t / p.qtiles;
        r.x0 = xt * 2 * kM + rank * kM;
        r.nx = (int)max((int64_t)0, min((int64_t)kM, p.nx - r.x0));
        r.q0 = (int)(t - xt * p.qtiles) * p.per;
        r.nq = (int)min((int64_t)p.per, p.nq - r.q0);
        r.n = (r.nq + 15) & ~15;
        return r;
    };

    if (warp == 0) {
        // ---- loads of this CTA's rows and half of the queries
        const bool leader = elect_one();
        Ring<kStages> ring;
        bool ok = true;
        for (int64_t t = first; ok && t < tiles; t += clusters) {
            const Tile r = tile_of(t);
            const int boxes = (r.n / 2 + kBox - 1) / kBox;
            const int x0 = (int)min(r.x0, (int64_t)INT32_MAX);
            const int q0 = r.q0 + (int)rank * (r.n / 2);
            for (int kt = 0; kt < p.nk; ++kt) {
                if (ring.n >= kStages &&
                    !__all_sync(0xffffffffu,
                                wait_cluster(&sm.empty[ring.i], ring.phase ^ 1u, &sm.abort))) {
                    ok = false;
                    break;
                }
                if (leader) {
                    const uint32_t bar = in_first(&sm.full[ring.i]);
                    const int x = kt * (F8 ? kSlice : kSlice / 2);
                    if (rank == 0)
                        mbar_arrive_expect_tx(&sm.full[ring.i],
                                              2u * (kXBytes + (uint32_t)boxes * kBox * kSlice));
                    load_pair(sm.x[ring.i], &map_x, x, x0, bar);
                    for (int b = 0; b < boxes; ++b)
                        load_pair(sm.q[ring.i] + b * kBox * kSlice, &map_q, x, q0 + b * kBox, bar);
                }
                __syncwarp();
                ring.next();
            }
        }
        // no copy of either CTA may still be landing when they leave
        if (leader && rank == 0)
            for (uint32_t k = ring.n > kStages ? ring.n - kStages : 0u; k < ring.n; ++k)
                mbar_drain(&sm.full[k % kStages], (k / kStages) & 1u);
        __syncwarp();
    } else if (warp == 1) {
        if (rank == 0) {
            // ---- MMAs of both CTAs: tile i accumulates in TMEM half i & 1
            const bool leader = elect_one();
            const uint64_t dx0 = sw128_desc(smem_u32(sm.x[0]));
            const uint64_t dq0 = sw128_desc(smem_u32(sm.q[0]));
            Ring<kStages> ring;
            Ring<kSf> sf;
            int64_t i = 0;
            bool ok = true;
            for (int64_t t = first; ok && t < tiles; t += clusters, ++i) {
                const int h = (int)(i & 1), n = tile_of(t).n;
                if (i >= 2 &&
                    !__all_sync(0xffffffffu,
                                wait_cluster(&sm.accempty[h], (uint32_t)((i >> 1) - 1) & 1u,
                                             &sm.abort)))
                    break;
                const uint32_t d = tmem + (uint32_t)(h * kAcc);
                const uint32_t idesc =
                    F8 ? mx_idesc(2 * kM, n)
                       : (tc_idesc_m128(n, 1) & ~(31u << 24)) | ((uint32_t)(2 * kM >> 4) << 24);
                for (int kt = 0; kt < p.nk; ++kt) {
                    const bool begin = F8 && (kt & 3) == 0, end = kt + 1 == p.nk;
                    const bool last = F8 && ((kt & 3) == 3 || end);
                    const uint32_t tsf = tmem + (uint32_t)(kSf0 + (int)sf.i * kSfStep);
                    bool go = true;
                    if (begin) go = wait_cluster(&sm.sffull[sf.i], sf.phase, &sm.abort);
                    go = go && wait_cluster(&sm.full[ring.i], ring.phase, &sm.abort);
                    if (!__all_sync(0xffffffffu, go)) {
                        ok = false;
                        break;
                    }
                    tc_fence_after();
                    if (leader) {
                        auto mma = [&](int k) {
                            const uint64_t a = dx0 + ring.i * (kXBytes >> 4) + 2 * k;
                            const uint64_t b = dq0 + ring.i * (kQBytes >> 4) + 2 * k;
                            if (F8)
                                mma_mx2(d, a, b, mx_idesc_byte(idesc, kt & 3), tsf, tsf + 4,
                                        (kt | k) != 0);
                            else
                                mma_f16_2(d, a, b, idesc, (kt | k) != 0);
                        };
                        const int left = p.row_bytes - kt * kSlice;  // bytes
                        if (left >= kSlice) {
#pragma unroll
                            for (int k = 0; k < kSlice / 32; ++k) mma(k);
                        } else {
                            for (int k = 0; 32 * k < left; ++k) mma(k);
                        }
                        commit_both(&sm.empty[ring.i]);
                        if (last) commit_both(&sm.sfempty[sf.i]);
                        if (end) commit_both(&sm.accfull[h]);
                    }
                    __syncwarp();
                    ring.next();
                    if (last) sf.next();
                }
            }
            if (leader) {
                // fires once every MMA issued above has completed (also on an error path)
                asm volatile(
                    "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.b64 "
                    "[%0];" ::"r"(smem_u32(&sm.drain))
                    : "memory");
                mbar_drain(&sm.drain, 0);
            }
            __syncwarp();
        }
    } else if (warp >= kScale0) {
        if constexpr (F8) {
            // ---- scale words, read one chunk ahead: four columns for this CTA's rows,
            // eight for all queries of the tile, the same in each lane quarter
            const uint32_t quarter = tmem + ((uint32_t)((warp & 3) * 32) << 16);
            const uint8_t* ptr[12];
            uint32_t next[12];
            Ring<kSf> sf;
            int64_t t = first;
            auto load = [&](int kt) {
#pragma unroll
                for (int u = 0; u < 12; ++u)
                    next[u] = ptr[u] ? __ldg(reinterpret_cast<const uint32_t*>(ptr[u] + kt))
                                     : 0x7F7F7F7Fu;  // ones
            };
            auto open = [&] {
                if (t >= tiles) return false;
                const Tile r = tile_of(t);
                t += clusters;
#pragma unroll
                for (int u = 0; u < 12; ++u) {
                    const int i = lane + 32 * (u < 4 ? u : u - 4);
                    ptr[u] = u < 4 ? (i < r.nx ? p.xs + (r.x0 + i) * p.lxs : nullptr)
                                   : (i < r.nq ? p.qs + (int64_t)(r.q0 + i) * p.lqs : nullptr);
                }
                load(0);
                return true;
            };
            bool ok = open();
            for (int kt = 0; ok; sf.next()) {
                uint32_t w[12];
#pragma unroll
                for (int u = 0; u < 12; ++u) w[u] = next[u];
                kt += 4;
                bool more = true;
                if (kt < p.nk) {
                    load(kt);
                } else {
                    kt = 0;
                    more = open();
                }
                if (sf.n >= kSf) ok = wait_cluster(&sm.sfempty[sf.i], sf.phase ^ 1u, &sm.abort);
                ok = __all_sync(0xffffffffu, ok);
                if (!ok) break;
                tc_fence_after();
                const uint32_t at = quarter + (uint32_t)(kSf0 + (int)sf.i * kSfStep);
#pragma unroll
                for (int u = 0; u < 12; u += 4)
                    tmem_st4(at + u, w[u], w[u + 1], w[u + 2], w[u + 3]);
                tmem_st_wait();
                tc_fence_before();
                __syncwarp();
                if (lane == 0) arrive_at(in_first(&sm.sffull[sf.i]));
                ok = more;
            }
        }
    } else if (warp >= kEpi0) {
        // ---- epilogue: warp w holds TMEM lanes 32 (w & 3) .. of the CTA's rows, and
        // every other 16 columns
        const int quarter = warp & 3, half = (warp - kEpi0) >> 2;
        const int row = quarter * 32 + lane;
        int64_t i = 0;
        for (int64_t t = first; t < tiles; t += clusters, ++i) {
            const int h = (int)(i & 1);
            const Tile r = tile_of(t);
            const bool ok = wait_cluster(&sm.accfull[h], (uint32_t)(i >> 1) & 1u, &sm.abort);
            if (!__all_sync(0xffffffffu, ok)) break;
            tc_fence_after();
            const uint32_t acc = tmem + ((uint32_t)(quarter * 32) << 16) + (uint32_t)(h * kAcc);
            if (quarter * 32 < r.nx) {
                store_columns(out + (int64_t)r.q0 * p.ld_out + r.x0 + row, p.ld_out, acc, half,
                              r.nq, row < r.nx, p.alpha, p.beta);
            }
            tc_fence_before();
            __syncwarp();
            if (lane == 0) arrive_at(in_first(&sm.accempty[h]));
        }
    }
    tc_fence_before();
    __syncthreads();
    if (threadIdx.x == 0 && sm.abort) atomicOr(p.err + kScoreTimeout, 1);
    cluster_sync();  // neither leaves while the other uses its memory
    if (warp == 0) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512)
                     : "memory");
    }
}

template <bool F8, class O>
cudaError_t launch(const m3g_rows& q, const m3g_rows& x, const Params& p, void* out,
                   unsigned grid, cudaStream_t st) {
    constexpr size_t smem = sizeof(Smem) + 1024;
    static_assert(smem <= 227 * 1024, "shared memory of a CTA");
    auto kernel = scores_pair_kernel<F8, O>;
    static std::atomic<uint64_t> set{0};  // a bit a device
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    const uint64_t bit = dev < 64 ? uint64_t(1) << dev : 0;
    if (!(set.load() & bit)) {
        e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
        if (e != cudaSuccess) return e;
        set |= bit;
    }
    CUtensorMap mx, mq;
    row_map(&mx, x, kM);
    row_map(&mq, q, kBox);
    kernel<<<grid, kThreads, smem, st>>>(mx, mq, static_cast<O*>(out), p);
    return cudaGetLastError();
}

}  // namespace

cudaError_t launch_pair_scores(const m3g_rows& q, const m3g_rows& x, float alpha, float beta,
                               void* out, int out_dtype, int64_t ld_out, int* err, int sms,
                               cudaStream_t st) {
    Params p{};
    p.nq = q.n;
    p.nx = x.n;
    p.row_bytes = x.dim * (x.dtype == M3G_E4M3 ? 1 : 2);
    p.nk = (p.row_bytes + kSlice - 1) / kSlice;
    p.qs = q.scales;
    p.xs = x.scales;
    p.lqs = q.ld_scales;
    p.lxs = x.ld_scales;
    p.ld_out = ld_out;
    p.alpha = alpha;
    p.beta = beta;
    p.err = err;
    const int64_t parts = (q.n + kN - 1) / kN;
    p.per = (int)(((q.n + parts - 1) / parts + 15) / 16 * 16);
    p.qtiles = (q.n + p.per - 1) / p.per;
    p.xtiles = (x.n + 2 * kM - 1) / (2 * kM);
    const unsigned grid = 2 * (unsigned)std::min<int64_t>(p.xtiles * p.qtiles, sms / 2);
    if (x.dtype == M3G_E4M3)
        return out_dtype == M3G_F32 ? launch<true, float>(q, x, p, out, grid, st)
                                    : launch<true, __nv_bfloat16>(q, x, p, out, grid, st);
    return out_dtype == M3G_F32 ? launch<false, float>(q, x, p, out, grid, st)
                                : launch<false, __nv_bfloat16>(q, x, p, out, grid, st);
}

}  // namespace m3g
