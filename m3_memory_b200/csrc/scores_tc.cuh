// scores_tc.cuh -- what the tensor-core score kernels share: block-scaled MMAs, scale
// words in TMEM, rings.
#pragma once

#include <cuda_bf16.h>

#include "kernels.h"
#include "kernels_scores.h"
#include "tc.cuh"

namespace m3g {

constexpr int kM = 128;      // rows of x a CTA's tile
constexpr int kSlice = 128;  // bytes of a row a swizzled tile holds (128 8-bit or 64 bf16 dims)
constexpr int kXBytes = kM * kSlice;

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
__device__ __forceinline__ uint32_t mx_idesc(int m, int n) {
    return ((uint32_t)(n >> 3) << 17) | (1u << 23) | ((uint32_t)(m >> 7) << 27);
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

// The map of rows in boxes of a slice and box_rows rows, 128-byte swizzle.
inline void row_map(CUtensorMap* m, const m3g_rows& r, int box_rows) {
    const bool f8 = r.dtype == M3G_E4M3;
    encode_tma_2d(m, f8 ? CU_TENSOR_MAP_DATA_TYPE_UINT8 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, r.data,
                  (uint64_t)r.dim, (uint64_t)r.n, (uint64_t)r.ld * (f8 ? 1 : 2),
                  (uint32_t)(f8 ? kSlice : kSlice / 2), (uint32_t)box_rows,
                  CU_TENSOR_MAP_SWIZZLE_128B);
}

}  // namespace m3g
