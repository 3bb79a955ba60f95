// k_scores_tc.cu -- scores of queries against rows on the tensor cores: every row
// (dense) or the rows of each query's probed lists (grouped, ragged both ways).
//
// out[pair][j] = alpha * sum_i q_i x_ji + beta.  The rows lie along the MMA's M
// (128 rows of x a tile) and the queries along N, so a tile takes just as many
// columns as its list has queries (16 .. NT, a multiple of 16): with few queries a
// list the rows' bytes bound the kernel, and padding the queries to 128 would
// triple the operand traffic.  TMEM then holds one row of x per lane and one query
// per column, so a warp stores 32 neighbouring scores of one query: full lines
// without a detour through shared memory.
//
// 8-bit rows use kind::mxf8f6f4 with block scales: the hardware multiplies each
// 32-deep product by 2^(sx + sq - 254), both scale bytes read from TMEM.  One byte
// covers 128 dims, so the four MMAs of a 128-byte slice share it, and the four
// slices of a 512-dim chunk take bytes 0..3 of the same TMEM words.  bf16 rows use
// kind::f16.  Sums are fp32 in TMEM.
//
// A launch is one CTA per SM.  A tile is 128 rows of a group and up to NT of its
// queries, queries fastest, so the rows come from L2 after their first tile.  Warp 0
// loads rows and warp 12 queries (TMA; those of a group are gathered by warps 12-15),
// warp 1 issues the MMAs, warp 3 walks the groups and queues tiles, warps 4-11 store,
// warps 16-19 bring scale words.  Every wait is bounded.
//
// What bounds it, and what it measured (launches by themselves; back to back the clock
// falls, and dense products take up to a tenth longer):
//   few queries a row: the rows' bytes.  One query against 1M x 1024 8-bit rows 157 us
//     (6.6 TB/s); 1024 queries x 32 of 4096 lists, 1M x 1024 8-bit rows 186 us (5.5);
//     4096 x 16 of 4096 lists, 1M x 768 bf16 rows 257 us (5.9; partly filled tiles cost
//     the MMA warp as much as full ones, and a tile of 8-bit rows has fewer bytes).
//   many queries: the operands through L2, 46 KB for 128 bytes of K of a 128 x 240 tile,
//     beside the scores' own bytes.  1024 queries x 100096 rows x 1024 dims 142 us (1480
//     TFLOP/s; 37 bytes of operands a cycle and SM), 4096 x 16384 x 768 bf16 94 us (1100;
//     49).  CTA pairs (cta_group::2, 31 KB of operands a CTA) took 150 and 88 us, so the
//     operands are not all of it; staging the scores through shared memory for 16-byte
//     stores 164: neither was kept.  Rows of scores that do not start on 32-byte
//     boundaries cost up to twice their time: every 32-row store ends inside sectors (x
//     128 dims: 83 us for n = 100000, 160 for 100003).
#include <cuda_bf16.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <atomic>
#include <type_traits>

#include "common.cuh"
#include "kernels.h"
#include "kernels_scores.h"
#include "tc.cuh"

namespace m3g {
namespace {

constexpr int kM = 128;                 // rows of x a tile
constexpr int kSlice = 128;             // bytes of a row a swizzled tile holds (128 8-bit or 64 bf16 dims)
constexpr int kXBytes = kM * kSlice;
constexpr int kEpiWarps = 8;            // two for each quarter of the TMEM lanes
constexpr int kQueryWarps = 4;          // each gathers every fourth stage's queries
constexpr int kScaleWarps = 4;          // one for each quarter of the TMEM lanes
constexpr int kThreads = (4 + kEpiWarps + kQueryWarps + kScaleWarps) * 32;
constexpr int kEpi0 = 4;                // first epilogue warp (a multiple of 4)
constexpr int kQuery0 = kEpi0 + kEpiWarps;
constexpr int kScale0 = kQuery0 + kQueryWarps;  // (a multiple of 4)
constexpr int kItems = 8;               // tiles queued ahead

// The launch shapes: up to NT queries a tile.  Rows and queries have rings of their
// own (kX and kQ stages of kSlices slices; two slices a stage where the rows are read
// for few queries, as a stage costs the MMA warp some 400 cycles beside its MMAs).
// Lists of up to 32 queries a tile take a fifth stage of rows, as many of their tiles
// are partly filled (1024 x 32 of 4096 lists 185 us for 191); the dense form measured
// better with four (158 us for 168, one query against 1M rows).
template <int NT, bool GROUP>
struct Shape;
template <bool GROUP>
struct Shape<32, GROUP> {
    static constexpr int kX = GROUP ? 5 : 4, kQ = GROUP ? 6 : 8, kSlices = 2, kBox = 16,
                         kAcc = 32, kTmem = 128, kSf = 4, kSf0 = 64, kSfStep = 8;
};
template <bool GROUP>
struct Shape<64, GROUP> {
    static constexpr int kX = 4, kQ = 4, kSlices = 2, kBox = 16, kAcc = 64, kTmem = 256,
                         kSf = 4, kSf0 = 128, kSfStep = 8;
};
template <bool GROUP>
struct Shape<240, GROUP> {  // each accumulator's scales in the 16 columns behind it
    static constexpr int kX = 4, kQ = 4, kSlices = 1, kBox = 48, kAcc = 256, kTmem = 512,
                         kSf = 2, kSf0 = 240, kSfStep = 256;
};

template <bool GROUP>
struct Shape<112, GROUP> {  // many queries, bf16 rows and fp32 scores: see parts_of
    static constexpr int kX = 6, kQ = 6, kSlices = 1, kBox = 56, kAcc = 112, kTmem = 256,
                         kSf = 2, kSf0 = 224, kSfStep = 16;
};

// Accumulators a tile.  The tensor core cuts a sum's low bits where it could round, once
// a MMA, so a sum of K dims comes out low by about K 2^-30 of itself for bf16 products
// (K 2^-34 for e4m3 ones, whose sums seldom need the bits): 1e-6 at 1024 dims, 2.1e-6 at
// 2048, where fp32 sums are within 4e-7.  fp32 scores of bf16 rows are added up from
// sums of every fourth slice (4.7e-7 at 2048 dims).  With many queries that costs width:
// 240 queries a tile have room for one sum, 112 for two, and L2 then gives the rows
// twice (4096 x 16384 x 768: 147 us for 95), so the width goes by the dims: one sum up to
// 512 (4.7e-7), two up to 1536 (7.2e-7), 64 queries with four above.
template <bool F8, int NT, class O>
constexpr int parts_of() {
    return F8 || sizeof(O) != 4 || NT == 240 ? 1 : NT == 112 ? 2 : 4;
}

struct Item {
    int32_t x0, nx;  // first row of x, rows (0: no more tiles)
    int32_t q0, nq;  // first pair, pairs
    int64_t j0;      // the first row's place in its list
    int64_t len;     // rows of the list
};

template <int NT, bool GROUP>
struct alignas(1024) Smem {
    using S = Shape<NT, GROUP>;
    unsigned char x[S::kX][S::kSlices][kXBytes];
    unsigned char q[S::kQ][S::kSlices][NT * kSlice];
    int64_t at[kItems][NT];  // where each column's scores start; -1: nowhere
    alignas(16) int32_t row[kItems][NT];  // each column's row of q (0 where there is none)
    int64_t prefix[kThreads + 1];
    Item items[kItems];
    uint64_t xfull[S::kX], xempty[S::kX];
    uint64_t qfull[S::kQ], qempty[S::kQ];
    uint64_t accfull[2], accempty[2], sffull[S::kSf], sfempty[S::kSf];
    uint64_t itemfull[kItems], itemempty[kItems], drain;
    int64_t warp_sum[kThreads / 32];
    uint32_t tmem;
    int abort;
};

struct Params {
    int64_t nq, nx;  // rows of q and x
    int nk;          // slices of a row
    int row_bytes;   // bytes of a row that hold dims
    const void* q;
    int64_t ldq;  // bytes
    const uint8_t *qs, *xs;
    int64_t lqs, lxs;
    float alpha, beta;
    int64_t ld_out;  // dense form
    ScoreGroups g;   // group form
    int* err;
};

// 16 bytes global -> shared, those past the first `size` filled with zeros.  Through
// L1: a list's next tile gathers the same rows (215 us for 195 without, 1024 x 32 of
// 4096 lists).
__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, uint32_t size) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(size)
                 : "memory");
}
__device__ __forceinline__ void cp_async_wait_all() {
    asm volatile("cp.async.wait_all;" ::: "memory");
}

__device__ __forceinline__ void tc_mma_mx(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc,
                                          uint32_t sfa, uint32_t sfb, bool accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %6, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::mxf8f6f4.block_scale.scale_vec::1X "
        "[%0], %1, %2, %3, [%4], [%5], p;\n\t}" ::"r"(d),
        "l"(a), "l"(b), "r"(idesc), "r"(sfa), "r"(sfb), "r"((uint32_t)accumulate)
        : "memory");
}

// One word a lane into each of four TMEM columns of the warp's lane quarter.
__device__ __forceinline__ void tmem_st4(uint32_t taddr, uint32_t a, uint32_t b, uint32_t c,
                                         uint32_t d) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x4.b32 [%0], {%1, %2, %3, %4};" ::"r"(taddr),
                 "r"(a), "r"(b), "r"(c), "r"(d)
                 : "memory");
}
__device__ __forceinline__ void tmem_st_wait() {
    asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
}

// kind::mxf8f6f4: both operands e4m3 (0) and K-major, N >> 3 at bits 17-22, ue8m0
// scales (bit 23), M >> 7 at bits 27-28; the scale byte of the words: bits 4-5 (B)
// and 29-30 (A).
__device__ __forceinline__ uint32_t mx_idesc(int n) {
    return ((uint32_t)(n >> 3) << 17) | (1u << 23) | (1u << 27);
}
__device__ __forceinline__ uint32_t mx_idesc_byte(uint32_t idesc, int byte) {
    return idesc | ((uint32_t)byte << 4) | ((uint32_t)byte << 29);
}

// A position in a ring of N slots and the parity of its current round.
template <int N>
struct Ring {
    __device__ static constexpr uint32_t slots() { return N; }
    uint32_t i = 0, phase = 0, n = 0;
    __device__ __forceinline__ void next() {
        ++n;
        if (++i == N) {
            i = 0;
            phase ^= 1u;
        }
    }
};

__device__ __forceinline__ void put_score(float* p, float v) { *p = v; }
__device__ __forceinline__ void put_score(__nv_bfloat16* p, float v) { *p = __float2bfloat16_rn(v); }

// 16 columns of the warp's TMEM lanes, waited for by tmem_ld_wait.
__device__ __forceinline__ void tmem_ld16_start(uint32_t taddr, uint32_t (&r)[16]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, "
        "%11, %12, %13, %14, %15}, [%16];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]),
          "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]),
          "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
        : "r"(taddr));
}
// The values of r are there after it (and not read before it).
__device__ __forceinline__ void tmem_ld_wait(uint32_t (&r)[16]) {
    asm volatile("tcgen05.wait::ld.sync.aligned;"
                 : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]),
                   "+r"(r[6]), "+r"(r[7]), "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]),
                   "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15])
                 :
                 : "memory");
}

// 16 columns of the warp's TMEM lanes, added up over the first n of P accumulators that
// are `step` columns apart.
template <int P>
__device__ __forceinline__ void tmem_ld16_sum(uint32_t taddr, int step, int n, uint32_t (&r)[16]) {
    tmem_ld16(taddr, r);
#pragma unroll
    for (int a = 1; a < P; ++a) {
        if (a >= n) break;
        uint32_t s[16];
        tmem_ld16(taddr + (uint32_t)(a * step), s);
#pragma unroll
        for (int u = 0; u < 16; ++u)
            r[u] = __float_as_uint(__uint_as_float(r[u]) + __uint_as_float(s[u]));
    }
}

// Every other 16 of a tile's nq columns, from 16 * half on: a lane stores its row's
// score of column c at mine[c * ld].  The next columns are on their way from TMEM while
// these are stored (a load waited for at once, and a multiplication for each address,
// cost 690 cycles for 16 columns where the stores take 400).
template <class O>
__device__ __forceinline__ void store_columns(O* mine, int64_t ld, uint32_t acc, int half, int nq,
                                              bool in, float alpha, float beta) {
    uint32_t cur[16], next[16];
    int c = 16 * half;
    if (c >= nq) return;
    O* at = mine + c * ld;
    tmem_ld16_start(acc + (uint32_t)c, cur);
#pragma unroll 1
    for (; c < nq; c += 32) {
        tmem_ld_wait(cur);
        if (c + 32 < nq) tmem_ld16_start(acc + (uint32_t)(c + 32), next);
        if (c + 16 <= nq) {
#pragma unroll
            for (int u = 0; u < 16; ++u) {
                if (in) put_score(at, fmaf(alpha, __uint_as_float(cur[u]), beta));
                at += ld;
            }
        } else {
#pragma unroll
            for (int u = 0; u < 16; ++u) {
                if (in && c + u < nq) put_score(at, fmaf(alpha, __uint_as_float(cur[u]), beta));
                at += ld;
            }
        }
        at += 16 * ld;
        tmem_ld_wait(next);
#pragma unroll
        for (int u = 0; u < 16; ++u) cur[u] = next[u];
    }
}

// A group's tiles: its rows in 128s (nx) times its pairs in nqt parts of `per`, the
// pairs fastest.  CTAs take runs of equal weight: with few queries, where loading it is
// most of its time, a tile of 128 rows weighs 9 and a list's last one, of r rows,
// 1 + (r + 31) / 16 (whole numbers: 3 to 10; by 32-row boxes, 1 + 2 ceil(r / 32), 4096 x
// 16 of 4096 lists took 266 us for 263); the same always with many, where the MMAs are.
template <int NT>
struct Tiles {
    int64_t nx;
    int32_t per, nqt;
    int32_t w, wlast;  // weight of a tile of 128 rows, and of the last rows' tiles

    __device__ __forceinline__ Tiles(int64_t len, int64_t m) {
        nx = len > 0 && m > 0 ? (len + kM - 1) / kM : 0;
        uint32_t n = (uint32_t)m;  // pairs number less than 2^31
        if (n > (uint32_t)NT) {
            const uint32_t parts = (n + NT - 1) / NT;
            n = (n + parts - 1) / parts;
        }
        per = (int32_t)max((n + 15u) & ~15u, 16u);
        nqt = n == (uint32_t)m ? 1 : (int32_t)(((uint32_t)m + per - 1) / (uint32_t)per);
        w = NT > 64 ? 1 : 9;
        wlast = NT > 64 ? 1 : 1 + ((int32_t)(len - (nx - 1) * kM) + 31) / 16;
    }
    __device__ __forceinline__ int64_t count() const { return nx * nqt; }
    __device__ __forceinline__ int64_t weight() const {
        return nx > 0 ? ((nx - 1) * w + wlast) * nqt : 0;
    }
    // The first tile that starts at or after `at` (a weight from the group's start).
    __device__ __forceinline__ int64_t first(int64_t at) const {
        if (at <= 0) return 0;
        if (at >= weight()) return count();
        const int64_t whole = (nx - 1) * nqt, last = at - whole * w;
        return last <= 0 ? (at + w - 1) / w : whole + (last + wlast - 1) / wlast;
    }
};

// The group's rows and pairs; false (and nothing in it) when they are out of range.
struct GroupAt {
    int64_t l0, len, p0, m;
};
__device__ __forceinline__ bool load_group(const Params& p, int64_t i, GroupAt* o) {
    const ScoreGroups& g = p.g;
    const int64_t a = g.pair_off[i], b = g.pair_off[i + 1];
    o->l0 = g.list_off[i];
    o->len = g.list_len[i];
    o->p0 = a;
    o->m = b - a;
    const bool bad = a < 0 || b < a || b > g.npair || o->len < 0 || o->l0 < 0 ||
                     o->l0 > p.nx || o->len > p.nx - o->l0;
    if (bad) o->len = o->m = 0;
    return !bad || a == b;
}

template <bool F8, int NT, bool GROUP, class O>
__global__ void __launch_bounds__(kThreads, 1)
    scores_tc_kernel(const __grid_constant__ CUtensorMap map_x,
                     const __grid_constant__ CUtensorMap map_x32,
                     const __grid_constant__ CUtensorMap map_q, O* __restrict__ out,
                     const __grid_constant__ Params p) {
    using S = Shape<NT, GROUP>;
    // (a gathering warp meets its stages' slots at least a round apart: its waits by
    // parity would not tell rounds apart otherwise)
    static_assert(S::kQ >= kQueryWarps, "");
    extern __shared__ unsigned char smem_raw[];
    auto& sm = *reinterpret_cast<Smem<NT, GROUP>*>(
        (reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

    constexpr int P = parts_of<F8, NT, O>();
    constexpr int kAcc = P > 1 ? P * NT : S::kAcc;  // columns from one tile's to the next's
    constexpr int kTmem = P == 1 ? S::kTmem : 2 * kAcc > 256 ? 512 : 256;
    static_assert(P == 1 || 2 * kAcc <= 512, "");
    static_assert(!F8 || NT != 112, "");
    if (warp == 0) tmem_alloc(&sm.tmem, kTmem);
    if (threadIdx.x == 32) {
        for (int s = 0; s < S::kX; ++s) {
            mbar_init(&sm.xfull[s], 1);
            mbar_init(&sm.xempty[s], 1);
        }
        for (int s = 0; s < S::kQ; ++s) {
            mbar_init(&sm.qfull[s], 1);
            mbar_init(&sm.qempty[s], 1);
        }
        for (int s = 0; s < 2; ++s) {
            mbar_init(&sm.accfull[s], 1);
            mbar_init(&sm.accempty[s], kEpiWarps);
        }
        for (int s = 0; s < S::kSf; ++s) {
            mbar_init(&sm.sffull[s], kScaleWarps);
            mbar_init(&sm.sfempty[s], 1);
        }
        for (int s = 0; s < kItems; ++s) {
            mbar_init(&sm.itemfull[s], 1);
            // its readers' warps: rows, MMAs, scales, epilogue, queries
            mbar_init(&sm.itemempty[s], 2 + (F8 ? kScaleWarps : 0) + kEpiWarps +
                                            (GROUP && p.g.pair_row ? kQueryWarps : 1));
        }
        mbar_init(&sm.drain, 1);
        sm.abort = 0;
        fence_mbar_init();
    }
    if (threadIdx.x == 0) {
        prefetch_tensormap(&map_x);
        prefetch_tensormap(&map_x32);
        prefetch_tensormap(&map_q);
    }

    // This CTA's tiles.  Grouped: a run of the launch's weight, which is added up first:
    // runs of `chunk` groups by warps, then over the runs by threads.  Dense: every
    // gridDim.x-th tile.
    int64_t total;
    int64_t chunk = 0;  // groups of a run (a multiple of 32)
    if constexpr (GROUP) {
        chunk = 32 * ((p.g.ngroup + 32 * kThreads - 1) / (32 * (int64_t)kThreads));
        sm.prefix[threadIdx.x] = 0;
        __syncthreads();
        bool ok = true;
#pragma unroll 4
        for (int64_t b = warp; b < kThreads; b += kThreads / 32) {
            if (b * chunk >= p.g.ngroup) break;
            int64_t sum = 0;
            for (int64_t i = b * chunk + lane; i < min((b + 1) * chunk, p.g.ngroup); i += 32) {
                GroupAt at;
                ok &= load_group(p, i, &at);
                sum += Tiles<NT>(at.len, at.m).weight();
            }
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
            if (lane == 0) sm.prefix[b] = sum;
        }
        __syncthreads();
        const int64_t mine = sm.prefix[threadIdx.x];
        if (!ok && blockIdx.x == 0) atomicOr(p.err + kScoreBadItem, 1);
        int64_t incl = mine;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int64_t v = __shfl_up_sync(0xffffffffu, incl, o);
            if (lane >= o) incl += v;
        }
        if (lane == 31) sm.warp_sum[warp] = incl;
        __syncthreads();
        int64_t before = 0;
        for (int w = 0; w < warp; ++w) before += sm.warp_sum[w];
        sm.prefix[threadIdx.x] = before + incl - mine;
        if (threadIdx.x == kThreads - 1) sm.prefix[kThreads] = before + incl;
    } else {
        total = Tiles<NT>(p.nx, p.nq).count();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    if constexpr (GROUP) total = sm.prefix[kThreads];
    const int64_t t0 = total / gridDim.x * blockIdx.x +
                       total % gridDim.x * blockIdx.x / gridDim.x;
    const int64_t t1 = total / gridDim.x * (blockIdx.x + 1) +
                       total % gridDim.x * (blockIdx.x + 1) / gridDim.x;
    const uint32_t tmem = sm.tmem;

    // The next queued tile; false: none left, or the launch gave up.  done_with()
    // hands its slot back.
    auto next_item = [&](int64_t i, Item* it) {
        const int s = (int)(i % kItems);
        const bool ok = mbar_wait(&sm.itemfull[s], (uint32_t)(i / kItems) & 1u, &sm.abort);
        if (ok) *it = sm.items[s];
        __syncwarp();
        if (!__all_sync(0xffffffffu, ok)) return false;
        return it->nx > 0;
    };
    auto done_with = [&](int64_t i) {
        __syncwarp();
        if (lane == 0) mbar_arrive(&sm.itemempty[i % kItems]);
    };
    const bool gather = GROUP && p.g.pair_row != nullptr;
    auto columns = [](const Item& it) { return (it.nq + 15) & ~15; };

    if (warp >= kQuery0 && warp < kScale0 && gather) {
        // ---- a group's queries, gathered with 16-byte copies (TMA's gather4 takes
        // some 230 cycles for its four rows): eight lanes a row, four rows a copy, in
        // the 128-byte swizzle the MMA reads.  The copies are made visible to the
        // tensor core by a fence that waits for all of the warp's, so each warp has
        // one stage in flight and the warps take the stages in turn.
        const unsigned char* src = static_cast<const unsigned char*>(p.q) + 16 * (lane & 7);
        Ring<S::kQ> ring;
        bool ok = true;
        Item item;
        for (int64_t i = 0; ok && next_item(i, &item); ++i) {
            const int n = columns(item);
            const int32_t* rows = sm.row[i % kItems];
            for (int kt = 0; kt < p.nk; kt += S::kSlices, ring.next()) {
                if (ring.n % kQueryWarps != (uint32_t)(warp - kQuery0)) continue;
                if (ring.n >= S::kQ &&
                    !__all_sync(0xffffffffu,
                                mbar_wait(&sm.qempty[ring.i], ring.phase ^ 1u, &sm.abort))) {
                    ok = false;
                    break;
                }
#pragma unroll
                for (int s = 0; s < S::kSlices; ++s) {
                    if (kt + s >= p.nk) break;
                    const uint32_t dst = smem_u32(sm.q[ring.i][s]);
                    const int off = (kt + s) * kSlice;
                    const int left = p.row_bytes - off - 16 * (lane & 7);
                    const uint32_t size = left >= 16 ? 16u : left > 0 ? (uint32_t)left : 0u;
                    // (a copy of no bytes fills zeros; it is given an address in the row)
                    const unsigned char* at = src + (size ? off : -16 * (lane & 7));
#pragma unroll 4
                    for (int r = lane >> 3; r < n; r += 4)
                        cp_async16(dst + (uint32_t)(r * kSlice) + (((lane & 7) ^ (r & 7)) << 4),
                                   at + rows[r] * p.ldq, size);
                }
                cp_async_wait_all();
                fence_proxy_async_smem();
                __syncwarp();
                if (lane == 0) mbar_arrive(&sm.qfull[ring.i]);
            }
            done_with(i);
        }
    } else if (warp == 0 || warp == kQuery0) {
        // ---- loads by TMA: warp 0 the rows, the other the queries (a copy takes
        // its issuer some 100 cycles).  The warp walks the tiles with warp-uniform
        // values, so the copies' operands stay in uniform registers; the elected lane
        // issues.
        const bool leader = elect_one();
        auto load = [&](auto ring, uint64_t* full, uint64_t* empty, auto boxes_of, auto copy) {
            constexpr uint32_t N = decltype(ring)::slots();
            bool ok = true;
            Item item;
            for (int64_t i = 0; ok && next_item(i, &item); ++i) {
                done_with(i);
                const uint32_t bytes = (uint32_t)kSlice * boxes_of(item);
                for (int kt = 0; kt < p.nk; kt += S::kSlices) {
                    if (ring.n >= N &&
                        !__all_sync(0xffffffffu,
                                    mbar_wait(&empty[ring.i], ring.phase ^ 1u, &sm.abort))) {
                        ok = false;
                        break;
                    }
                    if (leader) {
                        const int ns = min(S::kSlices, p.nk - kt);
                        mbar_arrive_expect_tx(&full[ring.i], bytes * ns);
                        for (int s = 0; s < ns; ++s)
                            copy(item, ring.i, s, (kt + s) * (F8 ? kSlice : kSlice / 2));
                    }
                    __syncwarp();
                    ring.next();
                }
            }
            // no copy may still be landing when the CTA leaves
            if (leader)
                for (uint32_t k = ring.n > N ? ring.n - N : 0u; k < ring.n; ++k)
                    mbar_drain(&full[k % N], (k / N) & 1u);
            __syncwarp();
        };
        if (warp == 0) {
            // the 32-row boxes of a tile of less than four (0: one box of 128 rows)
            auto small = [](const Item& it) { return it.nx > 96 ? 0 : (it.nx + 31) / 32; };
            load(
                Ring<S::kX>(), sm.xfull, sm.xempty,
                [&](const Item& it) { return small(it) ? 32 * small(it) : kM; },
                [&](const Item& it, uint32_t slot, int s, int x) {
                    const int n = small(it);
                    if (n == 0) tma_load_2d(sm.x[slot][s], &map_x, x, it.x0, &sm.xfull[slot]);
                    for (int b = 0; b < n; ++b)
                        tma_load_2d(sm.x[slot][s] + b * 32 * kSlice, &map_x32, x, it.x0 + 32 * b,
                                    &sm.xfull[slot]);
                });
        } else {
            auto boxes = [&](const Item& it) { return (columns(it) + S::kBox - 1) / S::kBox; };
            load(
                Ring<S::kQ>(), sm.qfull, sm.qempty,
                [&](const Item& it) { return boxes(it) * S::kBox; },
                [&](const Item& it, uint32_t slot, int s, int x) {
                    for (int b = 0; b < boxes(it); ++b)
                        tma_load_2d(sm.q[slot][s] + b * S::kBox * kSlice, &map_q, x,
                                    it.q0 + b * S::kBox, &sm.qfull[slot]);
                });
        }
    } else if (warp == 1) {
        // ---- MMAs: tile i accumulates in TMEM half i & 1.  Warp-uniform like the loads.
        const bool leader = elect_one();
        // descriptors of the first stages; an offset of b bytes adds b >> 4
        const uint64_t dx0 = sw128_desc(smem_u32(sm.x[0][0]));
        const uint64_t dq0 = sw128_desc(smem_u32(sm.q[0][0]));
        Ring<S::kX> rx;
        Ring<S::kQ> rq;
        Ring<S::kSf> sf;
        bool ok = true;
        Item item;
        for (int64_t i = 0; ok && next_item(i, &item); ++i) {
            const int h = (int)(i & 1), n = columns(item);
            done_with(i);
            if (i >= 2 &&
                !__all_sync(0xffffffffu, mbar_wait(&sm.accempty[h], (uint32_t)((i >> 1) - 1) & 1u,
                                                   &sm.abort)))
                break;
            tc_fence_after();
            const uint32_t d = tmem + (uint32_t)(h * kAcc);
            const uint32_t idesc = F8 ? mx_idesc(n) : tc_idesc_m128(n, 1);
            for (int kt = 0; kt < p.nk; kt += S::kSlices) {
                const bool first = F8 && (kt & 3) == 0;
                const bool end = kt + S::kSlices >= p.nk;
                const bool last = F8 && (((kt + S::kSlices) & 3) == 0 || end);
                const uint32_t tsf = tmem + (uint32_t)(S::kSf0 + (int)sf.i * S::kSfStep);
                bool go = true;
                if (first) go = mbar_wait(&sm.sffull[sf.i], sf.phase, &sm.abort);
                go = go && mbar_wait(&sm.qfull[rq.i], rq.phase, &sm.abort);
                go = go && mbar_wait(&sm.xfull[rx.i], rx.phase, &sm.abort);
                if (!__all_sync(0xffffffffu, go)) {
                    ok = false;
                    break;
                }
                tc_fence_after();
                if (leader) {
                    auto mma = [&](int s, int k, uint32_t id) {
                        const uint64_t a =
                            dx0 + (rx.i * S::kSlices + s) * (kXBytes >> 4) + 2 * k;
                        const uint64_t b =
                            dq0 + (rq.i * S::kSlices + s) * (NT * kSlice >> 4) + 2 * k;
                        const uint32_t to = d + (uint32_t)((kt + s) % P * NT);
                        const bool more = kt + s >= P || k > 0;
                        if (F8) tc_mma_mx(to, a, b, id, tsf, tsf + 4, more);
                        else tc_mma_f16(to, a, b, id, more);
                    };
#pragma unroll
                    for (int s = 0; s < S::kSlices; ++s) {
                        const int left = p.row_bytes - (kt + s) * kSlice;  // bytes
                        const uint32_t id = F8 ? mx_idesc_byte(idesc, (kt + s) & 3) : idesc;
                        if (left >= kSlice) {
#pragma unroll
                            for (int k = 0; k < kSlice / 32; ++k) mma(s, k, id);
                        } else {
                            for (int k = 0; 32 * k < left; ++k) mma(s, k, id);
                        }
                    }
                    tc_commit(&sm.xempty[rx.i]);
                    tc_commit(&sm.qempty[rq.i]);
                    if (last) tc_commit(&sm.sfempty[sf.i]);
                    if (end) tc_commit(&sm.accfull[h]);
                }
                __syncwarp();
                rx.next();
                rq.next();
                if (last) sf.next();
            }
        }
        if (leader) {
            // fires once every MMA issued above has completed (also on an error path)
            tc_commit(&sm.drain);
            mbar_drain(&sm.drain, 0);
        }
        __syncwarp();
    } else if (warp >= kScale0) {
        if constexpr (F8) {
            // ---- scale words, read one chunk ahead of the one being handed over, from
            // global memory to TMEM: the four columns of 128 rows hold rows r, r + 32,
            // r + 64, r + 96 in lane r, the same in each lane quarter, so each of these
            // warps stores the same words to its own.
            constexpr int W = 4 + (NT > 128 ? 8 : 4);
            const uint8_t* ptr[W];
            uint32_t next[W];
            const uint32_t quarter = tmem + ((uint32_t)((warp & 3) * 32) << 16);
            Ring<S::kSf> sf;
            Item item;
            int64_t i = 0;
            auto load = [&](int kt) {
#pragma unroll
                for (int u = 0; u < W; ++u)
                    next[u] = ptr[u] ? __ldg(reinterpret_cast<const uint32_t*>(ptr[u] + kt))
                                     : 0x7F7F7F7Fu;  // ones
            };
            auto open = [&] {
                if (!next_item(i, &item)) return false;
#pragma unroll
                for (int u = 0; u < 4; ++u) {
                    const int r = lane + 32 * u;
                    ptr[u] = r < item.nx ? p.xs + (item.x0 + r) * p.lxs : nullptr;
                }
#pragma unroll
                for (int u = 0; u < W - 4; ++u) {
                    const int c = lane + 32 * u;
                    // (the queued row: a pair that is out of range has row 0)
                    const int64_t r = GROUP ? (c < item.nq ? sm.row[i % kItems][c] : 0)
                                            : (int64_t)item.q0 + c;
                    ptr[4 + u] = c < item.nq ? p.qs + r * p.lqs : nullptr;
                }
                done_with(i++);
                load(0);
                return true;
            };
            bool ok = open();
            for (int kt = 0; ok; sf.next()) {
                uint32_t w[W];
#pragma unroll
                for (int u = 0; u < W; ++u) w[u] = next[u];
                kt += 4;
                bool more = true;
                if (kt < p.nk) {
                    load(kt);
                } else {
                    kt = 0;
                    more = open();
                }
                if (sf.n >= S::kSf)
                    ok = mbar_wait(&sm.sfempty[sf.i], sf.phase ^ 1u, &sm.abort);
                ok = __all_sync(0xffffffffu, ok);
                if (!ok) break;
                tc_fence_after();
                const uint32_t at = quarter + (uint32_t)(S::kSf0 + (int)sf.i * S::kSfStep);
#pragma unroll
                for (int u = 0; u < W; u += 4)
                    tmem_st4(at + u, w[u], w[u + 1], w[u + 2], w[u + 3]);
                tmem_st_wait();
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(&sm.sffull[sf.i]);
                ok = more;
            }
        }
    } else if (warp == 3) {
        // ---- tiles t0 .. t1 - 1, 32 groups at a time, queued for the others
        int64_t i = 0;
        bool ok = true;
        auto queue = [&](const Item& item) {
            const int s = (int)(i % kItems);
            if (i >= kItems)
                ok = mbar_wait(&sm.itemempty[s], (uint32_t)((i / kItems) - 1) & 1u, &sm.abort);
            ok = __all_sync(0xffffffffu, ok);
            if (!ok) return;
            if constexpr (F8) {
                // the rows' scale words, into L2 before they are read: a range where lines
                // hold several rows', row by row where what lies between is not theirs
                const uint8_t* b = p.xs + (int64_t)item.x0 * p.lxs;
                auto prefetch = [](const uint8_t* at) {
                    asm volatile("prefetch.global.L2 [%0];" ::"l"(at));
                };
                if (p.lxs <= 128) {
                    const int n = (item.nx - 1) * (int)p.lxs + p.nk;
                    for (int o = 128 * lane; o < n; o += 128 * 32) prefetch(b + o);
                } else {
                    for (int r = lane; r < item.nx; r += 32)
                        for (int o = 0; o < p.nk; o += 128) prefetch(b + r * p.lxs + o);
                }
            }
            if constexpr (GROUP) {
                for (int c = lane; c < columns(item); c += 32) {
                    if (c >= item.nq) {
                        sm.row[s][c] = 0;
                        continue;
                    }
                    const int64_t pr = (int64_t)item.q0 + c;
                    const int64_t row = gather ? (int64_t)p.g.pair_row[pr] : pr;
                    const int64_t at = p.g.out_off[pr];
                    // (by the whole list's length: a pair's tiles decide alike)
                    const bool in = row >= 0 && row < p.nq && at >= 0 &&
                                    at <= p.g.out_n - item.len;
                    if (!in && row != -1) atomicOr(p.err + kScoreBadItem, 1);
                    sm.row[s][c] = in ? (int32_t)row : 0;
                    sm.at[s][c] = in ? at + item.j0 : -1;
                }
                __syncwarp();
            }
            if (lane == 0) {
                sm.items[s] = item;
                mbar_arrive(&sm.itemfull[s]);
            }
            __syncwarp();
            ++i;
        };
        // tiles from, from + step, .. of a group
        auto queue_group = [&](const GroupAt& at, const Tiles<NT>& g, int64_t from, int64_t to,
                               unsigned step) {
            for (int64_t t = from; ok && t < to; t += step) {
                int64_t xt = t;
                int32_t qt = 0;
                if (g.nqt > 1) {
                    xt = t / g.nqt;
                    qt = (int32_t)(t - xt * g.nqt);
                }
                Item item;
                item.j0 = xt * kM;
                item.len = at.len;
                item.x0 = (int32_t)(at.l0 + item.j0);
                item.nx = (int32_t)min((int64_t)kM, at.len - item.j0);
                item.q0 = (int32_t)(at.p0 + (int64_t)qt * g.per);
                item.nq = (int32_t)min((int64_t)g.per, at.m - (int64_t)qt * g.per);
                queue(item);
            }
        };
        if constexpr (GROUP) {
            if (t0 < t1) {
                int lo = 0, hi = kThreads;  // the last run that starts at or before t0
                while (hi - lo > 1) {
                    const int mid = (lo + hi) / 2;
                    if (sm.prefix[mid] <= t0) lo = mid;
                    else hi = mid;
                }
                int64_t first = sm.prefix[lo];
                for (int64_t g = lo * chunk; ok && g < p.g.ngroup && first < t1; g += 32) {
                    GroupAt at{0, 0, 0, 0};
                    if (g + lane < p.g.ngroup) load_group(p, g + lane, &at);
                    const int64_t weight = Tiles<NT>(at.len, at.m).weight();
                    int64_t incl = weight;
#pragma unroll
                    for (int o = 1; o < 32; o <<= 1) {
                        const int64_t v = __shfl_up_sync(0xffffffffu, incl, o);
                        if (lane >= o) incl += v;
                    }
                    const int64_t end = first + incl;
                    unsigned todo = __ballot_sync(0xffffffffu,
                                                  weight > 0 && end > t0 && end - weight < t1);
                    while (ok && todo) {
                        const int l = __ffs(todo) - 1;
                        todo &= todo - 1;
                        GroupAt o;
                        o.l0 = __shfl_sync(0xffffffffu, at.l0, l);
                        o.len = __shfl_sync(0xffffffffu, at.len, l);
                        o.p0 = __shfl_sync(0xffffffffu, at.p0, l);
                        o.m = __shfl_sync(0xffffffffu, at.m, l);
                        const int64_t b = __shfl_sync(0xffffffffu, end - weight, l);
                        const Tiles<NT> tiles(o.len, o.m);
                        queue_group(o, tiles, tiles.first(t0 - b), tiles.first(t1 - b), 1);
                    }
                    first = __shfl_sync(0xffffffffu, end, 31);
                }
            }
        } else {
            queue_group(GroupAt{0, p.nx, 0, p.nq}, Tiles<NT>(p.nx, p.nq), blockIdx.x, total,
                        gridDim.x);
        }
        if (ok) queue(Item{0, 0, 0, 0, 0, 0});
    } else if (warp >= kEpi0 && warp < kQuery0) {
        // ---- epilogue: warp w holds TMEM lanes 32 (w & 3) .. of the tile's rows, and
        // every other 16 columns
        const int quarter = warp & 3, half = (warp - kEpi0) >> 2;
        const int row = quarter * 32 + lane;
        Item item;
        for (int64_t i = 0; next_item(i, &item); ++i) {
            const int h = (int)(i & 1);
            const bool ok = mbar_wait(&sm.accfull[h], (uint32_t)(i >> 1) & 1u, &sm.abort);
            if (!__all_sync(0xffffffffu, ok)) break;
            tc_fence_after();
            const uint32_t acc =
                tmem + ((uint32_t)(quarter * 32) << 16) + (uint32_t)(h * kAcc);
            if (quarter * 32 < item.nx) {
                const bool in = row < item.nx;
                if constexpr (GROUP || P > 1) {
                    const int64_t* at = sm.at[i % kItems];
#pragma unroll 1
                    for (int c0 = 16 * half; c0 < item.nq; c0 += 32) {
                        uint32_t r[16];
                        tmem_ld16_sum<P>(acc + (uint32_t)c0, NT, p.nk, r);
#pragma unroll
                        for (int u = 0; u < 16; ++u) {
                            if (c0 + u >= item.nq) break;
                            const int64_t o = GROUP ? at[c0 + u]
                                                    : (item.q0 + c0 + u) * p.ld_out + item.j0;
                            if (in && o >= 0)
                                put_score(out + o + row,
                                          fmaf(p.alpha, __uint_as_float(r[u]), p.beta));
                        }
                    }
                } else {
                    store_columns(out + (int64_t)item.q0 * p.ld_out + item.j0 + row, p.ld_out,
                                  acc, half, item.nq, in, p.alpha, p.beta);
                }
            }
            done_with(i);
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&sm.accempty[h]);
        }
    }
    tc_fence_before();
    __syncthreads();
    if (threadIdx.x == 0 && sm.abort) atomicOr(p.err + kScoreTimeout, 1);
    if (warp == 0) {
        __syncwarp();
        tc_fence_after();
        tmem_dealloc(tmem, kTmem);
    }
}

void row_map(CUtensorMap* m, const m3g_rows& r, int box_rows) {
    const bool f8 = r.dtype == M3G_E4M3;
    encode_tma_2d(m, f8 ? CU_TENSOR_MAP_DATA_TYPE_UINT8 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, r.data,
                  (uint64_t)r.dim, (uint64_t)r.n, (uint64_t)r.ld * (f8 ? 1 : 2),
                  (uint32_t)(f8 ? kSlice : kSlice / 2), (uint32_t)box_rows,
                  CU_TENSOR_MAP_SWIZZLE_128B);
}

template <bool F8, int NT, bool GROUP, class O>
cudaError_t launch(const m3g_rows& q, const m3g_rows& x, const Params& p, void* out,
                   unsigned grid, cudaStream_t st) {
    constexpr size_t smem = sizeof(Smem<NT, GROUP>) + 1024;
    static_assert(smem <= 227 * 1024, "shared memory of a CTA");
    auto kernel = scores_tc_kernel<F8, NT, GROUP, O>;
    // once a device (a bit each; devices past 64 set it every time)
    static std::atomic<uint64_t> set{0};
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    const uint64_t bit = dev < 64 ? uint64_t(1) << dev : 0;
    if (!(set.load() & bit)) {
        e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
        if (e != cudaSuccess) return e;
        set |= bit;
    }
    CUtensorMap mx, mx32, mq;
    row_map(&mx, x, kM);
    row_map(&mx32, x, 32);
    row_map(&mq, q, Shape<NT, GROUP>::kBox);
    kernel<<<grid, kThreads, smem, st>>>(mx, mx32, mq, static_cast<O*>(out), p);
    return cudaGetLastError();
}

template <bool GROUP>
cudaError_t launch_any(const m3g_rows& q, const m3g_rows& x, const Params& p, int64_t queries,
                       void* out, int out_dtype, unsigned grid, cudaStream_t st) {
    const bool f32 = out_dtype == M3G_F32;
    auto with = [&](auto nt) {
        constexpr int NT = decltype(nt)::value;
        if constexpr (NT == 112)
            return launch<false, NT, GROUP, float>(q, x, p, out, grid, st);
        else if (x.dtype == M3G_E4M3)
            return f32 ? launch<true, NT, GROUP, float>(q, x, p, out, grid, st)
                       : launch<true, NT, GROUP, __nv_bfloat16>(q, x, p, out, grid, st);
        else
            return f32 ? launch<false, NT, GROUP, float>(q, x, p, out, grid, st)
                       : launch<false, NT, GROUP, __nv_bfloat16>(q, x, p, out, grid, st);
    };
    if (queries <= 32) return with(std::integral_constant<int, 32>());
    const bool sums = f32 && x.dtype == M3G_BF16;
    if (queries <= 64 || (sums && x.dim > 1536)) return with(std::integral_constant<int, 64>());
    if (sums && x.dim > 512) return with(std::integral_constant<int, 112>());
    return with(std::integral_constant<int, 240>());
}

Params params_of(const m3g_rows& q, const m3g_rows& x, float alpha, float beta, int* err) {
    Params p{};
    p.nq = q.n;
    p.nx = x.n;
    p.row_bytes = x.dim * (x.dtype == M3G_E4M3 ? 1 : 2);
    p.nk = (p.row_bytes + kSlice - 1) / kSlice;
    p.q = q.data;
    p.ldq = q.ld * (q.dtype == M3G_E4M3 ? 1 : 2);
    p.qs = q.scales;
    p.xs = x.scales;
    p.lqs = q.ld_scales;
    p.lxs = x.ld_scales;
    p.alpha = alpha;
    p.beta = beta;
    p.err = err;
    return p;
}

__global__ void take_score_errors_kernel(int* words, int* taken) {
    if (threadIdx.x < kScoreErrWords)
        taken[threadIdx.x] = atomicExch(words + threadIdx.x, 0);
}

}  // namespace

cudaError_t launch_take_score_errors(int* words, int* taken, cudaStream_t st) {
    take_score_errors_kernel<<<1, 32, 0, st>>>(words, taken);
    return cudaGetLastError();
}

cudaError_t launch_row_scores(const m3g_rows& q, const m3g_rows& x, float alpha, float beta,
                              void* out, int out_dtype, int64_t ld_out, int* err, int sms,
                              cudaStream_t st) {
    Params p = params_of(q, x, alpha, beta, err);
    p.ld_out = ld_out;
    const int64_t tiles = (x.n + kM - 1) / kM * ((q.n + 15) / 16);  // at least as many as there are
    return launch_any<false>(q, x, p, q.n, out, out_dtype,
                             (unsigned)std::min<int64_t>(tiles, sms), st);
}

cudaError_t launch_list_scores(const m3g_rows& q, const m3g_rows& x, const ScoreGroups& g,
                               float alpha, float beta, void* out, int out_dtype, int* err,
                               int sms, cudaStream_t st) {
    Params p = params_of(q, x, alpha, beta, err);
    p.g = g;
    return launch_any<true>(q, x, p, g.npair / g.ngroup, out, out_dtype, (unsigned)sms, st);
}

}  // namespace m3g
