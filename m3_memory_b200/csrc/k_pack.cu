// k_pack.cu -- rows packed to 8 bits: e4m3 codes and one power-of-two scale per 128
// dims.
#include <cuda_bf16.h>
#include <cuda_fp8.h>
#include <cuda_runtime.h>

#include <algorithm>

#include "common.cuh"
#include "kernels_scores.h"

namespace m3g {
namespace {

// The exponent e of a block's scale from the bits of its largest finite |x|
// (A <= 448 * 2^e = 1.75 * 2^(e + 8), e >= -126): A's own exponent less 8, one
// more when its mantissa is above 1.75.  Subnormal A fall below the floor.
__device__ __forceinline__ int scale_exponent(uint32_t amax_bits) {
    const int x = (int)(amax_bits >> 23) - 127;
    const int e = x - 8 + ((amax_bits & 0x7FFFFFu) > 0x600000u ? 1 : 0);
    return max(e, -126);
}

__device__ __forceinline__ float pow2f(int e) {  // 2^e, -126 <= e <= 127
    return __int_as_float((e + 127) << 23);
}

__device__ __forceinline__ uint32_t finite_abs_bits(float v) {
    const uint32_t u = __float_as_uint(v) & 0x7FFFFFFFu;
    return u < 0x7F800000u ? u : 0u;
}

__device__ __forceinline__ float load_in(const float* p) { return *p; }
__device__ __forceinline__ float load_in(const __nv_bfloat16* p) { return __bfloat162float(*p); }

// One warp per block of 128 dims.
template <class T>
__global__ void __launch_bounds__(256)
    pack_rows_kernel(const T* __restrict__ x, int64_t n, int dim, int64_t ldx, int nblk,
                     uint8_t* __restrict__ codes, int64_t ld, uint8_t* __restrict__ scales,
                     int64_t lds) {
    const int lane = threadIdx.x & 31;
    const int64_t total = n * nblk;
    const int64_t step = (int64_t)gridDim.x * (blockDim.x >> 5);
    for (int64_t b = (int64_t)blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5); b < total;
         b += step) {
        const int64_t row = b / nblk;
        const int d0 = (int)(b - row * nblk) * kScaleDims;
        float v[4];
        uint32_t m = 0;
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            const int d = d0 + 4 * lane + u;
            v[u] = d < dim ? load_in(x + row * ldx + d) : 0.f;
            m = max(m, finite_abs_bits(v[u]));
        }
        m = __reduce_max_sync(0xffffffffu, m);
        const int e = scale_exponent(m);
        const float s = pow2f(-e);
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            const int d = d0 + 4 * lane + u;
            if (d < dim)
                codes[row * ld + d] = __nv_cvt_float_to_fp8(v[u] * s, __NV_SATFINITE, __NV_E4M3);
        }
        if (lane == 0) scales[row * lds + d0 / kScaleDims] = (uint8_t)(e + 127);
    }
}

}  // namespace

cudaError_t launch_pack_rows(const void* x, int dtype, int64_t n, int dim, int64_t ldx,
                             uint8_t* codes, int64_t ld, uint8_t* scales, int64_t lds,
                             cudaStream_t st) {
    const int nblk = (dim + kScaleDims - 1) / kScaleDims;
    const unsigned grid = (unsigned)std::min<int64_t>((n * nblk + 7) / 8, 148 * 8);
    if (dtype == M3G_F32)
        pack_rows_kernel<<<grid, 256, 0, st>>>(static_cast<const float*>(x), n, dim, ldx, nblk,
                                               codes, ld, scales, lds);
    else
        pack_rows_kernel<<<grid, 256, 0, st>>>(static_cast<const __nv_bfloat16*>(x), n, dim, ldx,
                                               nblk, codes, ld, scales, lds);
    return cudaGetLastError();
}

}  // namespace m3g
