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

// The map of rows in boxes of a slice and box_rows rows, 128-byte swizzle.
inline void row_map(CUtensorMap* m, const m3g_rows& r, int box_rows) {
    const bool f8 = r.dtype == M3G_E4M3;
    encode_tma_2d(m, f8 ? CU_TENSOR_MAP_DATA_TYPE_UINT8 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, r.data,
                  (uint64_t)r.dim, (uint64_t)r.n, (uint64_t)r.ld * (f8 ? 1 : 2),
                  (uint32_t)(f8 ? kSlice : kSlice / 2), (uint32_t)box_rows,
                  CU_TENSOR_MAP_SWIZZLE_128B);
}

}  // namespace m3g
