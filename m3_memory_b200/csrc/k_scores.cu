// k_scores.cu -- rows packed to 8 bits, and the scores of queries against rows:
// every row (dense) or the rows of each query's probed lists (grouped).
#include <cuda_bf16.h>
#include <cuda_fp8.h>
#include <cuda_runtime.h>

#include <algorithm>

#include "common.cuh"
#include "kernels_scores.h"

namespace m3g {
namespace {

// ---------------- packing ----------------

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

// ---------------- scores ----------------

__device__ __forceinline__ float row_value(const m3g_rows& r, int64_t row, int d) {
    if (r.dtype == M3G_BF16)
        return __bfloat162float(static_cast<const __nv_bfloat16*>(r.data)[row * r.ld + d]);
    const uint8_t c = static_cast<const uint8_t*>(r.data)[row * r.ld + d];
    const __half h = __nv_cvt_fp8_to_halfraw(c, __NV_E4M3);
    const uint8_t s = r.scales[row * r.ld_scales + d / kScaleDims];
    return __half2float(h) * __int_as_float((int)s << 23);
}

__device__ __forceinline__ void store_out(float* p, float v) { *p = v; }
__device__ __forceinline__ void store_out(__nv_bfloat16* p, float v) {
    *p = __float2bfloat16_rn(v);
}

// A 32 x 32 tile of products, queries along y: qrow[.] and xrow0 + . are rows.
template <class O, class QRow, class Out>
__device__ void score_tile(const m3g_rows& q, const m3g_rows& x, int64_t xrow0, int nx, int nqt,
                           float alpha, float beta, QRow qrow, Out out) {
    __shared__ float sq[32][33], sx[32][33];
    const int tx = threadIdx.x & 31, ty = threadIdx.x >> 5;  // 8 rows of 32 threads
    float acc[4] = {0.f, 0.f, 0.f, 0.f};
    for (int d0 = 0; d0 < q.dim; d0 += 32) {
        __syncthreads();
        for (int r = ty; r < 32; r += 8) {
            const int d = d0 + tx;
            const int64_t qr = r < nqt ? qrow(r) : -1;
            sq[r][tx] = qr >= 0 && qr < q.n && d < q.dim ? row_value(q, qr, d) : 0.f;
            sx[r][tx] = r < nx && d < q.dim ? row_value(x, xrow0 + r, d) : 0.f;
        }
        __syncthreads();
        for (int d = 0; d < 32; ++d)
#pragma unroll
            for (int u = 0; u < 4; ++u) acc[u] = fmaf(sq[ty + 8 * u][d], sx[tx][d], acc[u]);
    }
    for (int u = 0; u < 4; ++u) {
        const int r = ty + 8 * u;
        if (r < nqt && tx < nx) {
            O* p = out(r);
            if (p) store_out(p + tx, fmaf(alpha, acc[u], beta));
        }
    }
}

template <class O>
__global__ void __launch_bounds__(256)
    row_scores_kernel(m3g_rows q, m3g_rows x, float alpha, float beta, O* out, int64_t ld_out) {
    const int64_t tx = (x.n + 31) / 32, ty = (q.n + 31) / 32;
    for (int64_t t = blockIdx.x; t < tx * ty; t += gridDim.x) {
        const int64_t x0 = (t / ty) * 32, q0 = (t % ty) * 32;
        score_tile<O>(
            q, x, x0, (int)min((int64_t)32, x.n - x0), (int)min((int64_t)32, q.n - q0), alpha,
            beta, [&](int r) { return q0 + r; },
            [&](int r) { return out + (q0 + r) * ld_out + x0; });
    }
}

template <class O>
__global__ void __launch_bounds__(256)
    list_scores_kernel(m3g_rows q, m3g_rows x, ScoreGroups g, float alpha, float beta, O* out,
                       int* err) {
    for (int64_t i = blockIdx.x; i < g.ngroup; i += gridDim.x) {
        const int64_t p0 = g.pair_off[i], p1 = g.pair_off[i + 1];
        const int64_t l0 = g.list_off[i], len = g.list_len[i];
        if (p0 == p1 || len == 0) continue;
        if (p0 < 0 || p1 < p0 || p1 > g.npair || l0 < 0 || len < 0 || l0 + len > x.n) {
            if (threadIdx.x == 0) atomicOr(err + kScoreBadItem, 1);
            continue;
        }
        for (int64_t x0 = 0; x0 < len; x0 += 32)
            for (int64_t q0 = p0; q0 < p1; q0 += 32)
                score_tile<O>(
                    q, x, l0 + x0, (int)min((int64_t)32, len - x0),
                    (int)min((int64_t)32, p1 - q0), alpha, beta,
                    [&](int r) { return g.pair_row ? (int64_t)g.pair_row[q0 + r] : q0 + r; },
                    [&](int r) -> O* {
                        const int64_t row = g.pair_row ? (int64_t)g.pair_row[q0 + r] : q0 + r;
                        const int64_t o = g.out_off[q0 + r];
                        if (row == -1) return nullptr;
                        if (row < 0 || row >= q.n || o < 0 || o > g.out_n - len) {
                            atomicOr(err + kScoreBadItem, 1);
                            return nullptr;
                        }
                        return out + o + x0;
                    });
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

cudaError_t launch_row_scores(const m3g_rows& q, const m3g_rows& x, float alpha, float beta,
                              void* out, int out_dtype, int64_t ld_out, int* err, int sms,
                              cudaStream_t st) {
    const int64_t tiles = ((x.n + 31) / 32) * ((q.n + 31) / 32);
    const unsigned grid = (unsigned)std::min<int64_t>(tiles, (int64_t)sms * 8);
    if (out_dtype == M3G_F32)
        row_scores_kernel<<<grid, 256, 0, st>>>(q, x, alpha, beta, static_cast<float*>(out),
                                                ld_out);
    else
        row_scores_kernel<<<grid, 256, 0, st>>>(q, x, alpha, beta,
                                                static_cast<__nv_bfloat16*>(out), ld_out);
    return cudaGetLastError();
}

cudaError_t launch_list_scores(const m3g_rows& q, const m3g_rows& x, const ScoreGroups& g,
                               float alpha, float beta, void* out, int out_dtype, int* err,
                               int sms, cudaStream_t st) {
    const unsigned grid = (unsigned)std::min<int64_t>(g.ngroup, (int64_t)sms * 8);
    if (out_dtype == M3G_F32)
        list_scores_kernel<<<grid, 256, 0, st>>>(q, x, g, alpha, beta, static_cast<float*>(out),
                                                 err);
    else
        list_scores_kernel<<<grid, 256, 0, st>>>(q, x, g, alpha, beta,
                                                 static_cast<__nv_bfloat16*>(out), err);
    return cudaGetLastError();
}

}  // namespace m3g
