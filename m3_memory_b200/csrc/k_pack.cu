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

__device__ __forceinline__ float load_in(const float* p) { return *p; }
__device__ __forceinline__ float load_in(const __nv_bfloat16* p) { return __bfloat162float(*p); }

// 16 bytes of a row (4 fp32 or 8 bf16 values) from dim d on, zeros past dim.
template <class T, int E, bool VEC>
__device__ __forceinline__ void load_values(const T* row, int d, int dim, float* v) {
    if (VEC && d + E <= dim) {
        const uint4 r = __ldcs(reinterpret_cast<const uint4*>(row + d));
        const uint32_t w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if constexpr (E == 4) {
                v[i] = __uint_as_float(w[i]);
            } else {
                v[2 * i] = __uint_as_float(w[i] << 16);
                v[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u);
            }
        }
        return;
    }
#pragma unroll
    for (int i = 0; i < E; ++i) v[i] = d + i < dim ? load_in(row + d + i) : 0.f;
}

__device__ __forceinline__ float max_of_8_lanes(float m) {
#pragma unroll
    for (int o = 4; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
    return m;
}

// Eight lanes a block of 128 dims, 16 values a lane in 16-byte loads eight lanes wide
// (with a lane for each 16 bytes of fp32, four values, the work a block costs beside
// its values took more time than the bytes: 1396 us where this takes 862); kU blocks
// in flight a lane.  The bytes bound it: 1M x 1024 fp32 rows at 5.9 TB/s.  VEC: rows on
// 16-byte boundaries; else value by value.
template <class T, bool VEC>
__global__ void __launch_bounds__(256)
    pack_rows_kernel(const T* __restrict__ x, int64_t n, int dim, int64_t ldx, int nblk,
                     uint8_t* __restrict__ codes, int64_t ld, uint8_t* __restrict__ scales,
                     int64_t lds) {
    constexpr int E = 16 / (int)sizeof(T), J = 16 / E;  // values a load, loads a block
    constexpr int kU = VEC ? 2 : 1;
    const int l = threadIdx.x & 7;
    const int64_t total = n * nblk;
    // this lane's blocks are `step` apart; the next one is found without a division
    const int64_t step = (int64_t)gridDim.x * (blockDim.x / 8);
    const int64_t first = ((int64_t)blockIdx.x * blockDim.x + threadIdx.x) / 8;
    const int64_t step_rows = step / nblk;
    const int step_blk = (int)(step - step_rows * nblk);
    int64_t row = first / nblk;
    int blk = (int)(first - row * nblk);
    // whole warps stay in the loop: a block past the last is computed and not stored
    const int64_t warp_first = first & ~int64_t(3);
    for (int64_t b = warp_first; b < total; b += step * kU) {
        float v[kU][16];
        int64_t rows[kU];
        int blks[kU];
#pragma unroll
        for (int u = 0; u < kU; ++u) {
            rows[u] = row;
            blks[u] = blk;
            const bool in = row < n;
#pragma unroll
            for (int j = 0; j < J; ++j)
                load_values<T, E, VEC>(x + (in ? row : 0) * ldx, blk * kScaleDims + (l + 8 * j) * E,
                                       in ? dim : 0, v[u] + j * E);
            row += step_rows;
            blk += step_blk;
            if (blk >= nblk) {
                blk -= nblk;
                ++row;
            }
        }
#pragma unroll
        for (int u = 0; u < kU; ++u) {
            float m = 0.f;
#pragma unroll
            for (int i = 0; i < 16; ++i) m = fmaxf(m, fabsf(v[u][i]));  // (skips NaN)
            m = max_of_8_lanes(m);
            if (__any_sync(0xffffffffu, m == __int_as_float(0x7f800000))) {
                m = 0.f;  // the finite values alone
#pragma unroll
                for (int i = 0; i < 16; ++i)
                    if (fabsf(v[u][i]) < __int_as_float(0x7f800000)) m = fmaxf(m, fabsf(v[u][i]));
                m = max_of_8_lanes(m);
            }
            const int e = scale_exponent(__float_as_uint(m));
            const float s = pow2f(-e);
            if (rows[u] >= n) continue;
            uint8_t* o = codes + rows[u] * ld + blks[u] * kScaleDims;
#pragma unroll
            for (int j = 0; j < J; ++j) {
                uint32_t w[E / 4];
#pragma unroll
                for (int i = 0; i < E; i += 4) {
                    const float* p = v[u] + j * E + i;
                    const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(p[0] * s, p[1] * s),
                                                                 __NV_SATFINITE, __NV_E4M3);
                    const uint32_t hi = __nv_cvt_float2_to_fp8x2(make_float2(p[2] * s, p[3] * s),
                                                                 __NV_SATFINITE, __NV_E4M3);
                    w[i / 4] = lo | hi << 16;
                }
                const int at = (l + 8 * j) * E, d = blks[u] * kScaleDims + at;
                if (d + E <= dim) {  // (rows of codes are on 16-byte boundaries)
                    if constexpr (E == 4) *reinterpret_cast<uint32_t*>(o + at) = w[0];
                    else *reinterpret_cast<uint2*>(o + at) = make_uint2(w[0], w[1]);
                } else {
#pragma unroll
                    for (int i = 0; i < E; ++i)
                        if (d + i < dim) o[at + i] = (uint8_t)(w[i / 4] >> (8 * (i % 4)));
                }
            }
            if (l == 0) scales[rows[u] * lds + blks[u]] = (uint8_t)(e + 127);
        }
    }
}

template <class T>
void launch_typed(const T* x, int64_t n, int dim, int64_t ldx, uint8_t* codes, int64_t ld,
                  uint8_t* scales, int64_t lds, int sms, cudaStream_t st) {
    const int nblk = (dim + kScaleDims - 1) / kScaleDims;
    const unsigned grid = (unsigned)std::min<int64_t>((n * nblk + 31) / 32, sms * 4);
    if ((reinterpret_cast<uintptr_t>(x) & 15) == 0 && ldx * sizeof(T) % 16 == 0)
        pack_rows_kernel<T, true><<<grid, 256, 0, st>>>(x, n, dim, ldx, nblk, codes, ld, scales,
                                                        lds);
    else
        pack_rows_kernel<T, false><<<grid, 256, 0, st>>>(x, n, dim, ldx, nblk, codes, ld, scales,
                                                         lds);
}

}  // namespace

cudaError_t launch_pack_rows(const void* x, int dtype, int64_t n, int dim, int64_t ldx,
                             uint8_t* codes, int64_t ld, uint8_t* scales, int64_t lds, int sms,
                             cudaStream_t st) {
    if (dtype == M3G_F32)
        launch_typed(static_cast<const float*>(x), n, dim, ldx, codes, ld, scales, lds, sms,
                     st);
    else
        launch_typed(static_cast<const __nv_bfloat16*>(x), n, dim, ldx, codes, ld, scales, lds,
                     sms, st);
    return cudaGetLastError();
}

}  // namespace m3g
