// k_probs.cu -- scores as probabilities: log-sum-exp, entropy, the log
// probability of given entries and the k most probable ones.
#include <cuda_bf16.h>
#include <cuda_runtime.h>

#include <algorithm>

#include "common.cuh"
#include "kernels_scores.h"

namespace m3g {
namespace {

__device__ __forceinline__ float load_score(const float* p) { return *p; }
__device__ __forceinline__ float load_score(const __nv_bfloat16* p) { return __bfloat162float(*p); }

// Scores oriented so that larger is more probable: t = score for scale > 0, -score
// else, with c = |scale|; l = c t.  An entry takes part if l is not NaN or -inf.
__device__ __forceinline__ bool takes_part(float t, float c) {
    return c * t > __int_as_float(0xff800000);
}

// One block per row; 256 threads.
template <class T>
__global__ void __launch_bounds__(256) score_probs_kernel(ProbsArgs a) {
    __shared__ float red[256], red2[256];
    __shared__ unsigned long long redk[256];
    const int tid = threadIdx.x;
    const float c = fabsf(a.scale), sgn = a.scale > 0.f ? 1.f : -1.f;
    for (int64_t row = blockIdx.x; row < a.nq; row += gridDim.x) {
        int64_t b = row * a.ld, len = a.n;
        if (a.row_off) {
            b = max((int64_t)0, min(a.row_off[row], a.n));
            len = max((int64_t)0, min(a.row_off[row + 1], a.n) - b);
        }
        const T* s = static_cast<const T*>(a.scores) + b;
        float m = __int_as_float(0xff800000);
        for (int64_t i = tid; i < len; i += 256) {
            const float t = sgn * load_score(s + i);
            if (takes_part(t, c)) m = fmaxf(m, t);
        }
        red[tid] = m;
        __syncthreads();
        for (int h = 128; h > 0; h >>= 1) {
            if (tid < h) red[tid] = fmaxf(red[tid], red[tid + h]);
            __syncthreads();
        }
        m = red[0];
        __syncthreads();
        // sums relative to cm = c m as rounded: exact for any reference value.  An
        // entry more than 1000 below it adds nothing (exp is 0 from -104 on).
        const float cm = c * m;
        const bool inf = cm == __int_as_float(0x7f800000);
        float z = 0.f, w = 0.f;
        for (int64_t i = tid; i < len; i += 256) {
            const float t = sgn * load_score(s + i);
            if (!takes_part(t, c)) continue;
            const float d = fmaxf(fmaf(c, t, -cm), -1000.f), p = expf(d);
            z += p;
            w += p * d;
        }
        red[tid] = z;
        red2[tid] = w;
        __syncthreads();
        for (int h = 128; h > 0; h >>= 1) {
            if (tid < h) {
                red[tid] += red[tid + h];
                red2[tid] += red2[tid + h];
            }
            __syncthreads();
        }
        z = red[0];
        w = red2[0];
        __syncthreads();
        const float logz = logf(z);  // -inf for a row with nothing left
        if (tid == 0) {
            a.lse[row] = inf || !(z > 0.f) ? cm : cm + logz;  // cm = -inf: nothing left
            a.entropy[row] = inf ? __int_as_float(0x7fc00000) : z > 0.f ? logz - w / z : 0.f;
        }
        auto logp = [&](float t) {
            if (!takes_part(t, c)) return __int_as_float(0xff800000);
            if (inf) return __int_as_float(c * t == cm ? 0x7fc00000 : 0xff800000);
            return fmaf(c, t, -cm) - logz;
        };
        for (int j = tid; j < a.ngiven; j += 256) {
            const int64_t at = a.given[row * a.ngiven + j];
            a.out_given[row * a.ngiven + j] =
                at >= 0 && at < len ? logp(sgn * load_score(s + at)) : __int_as_float(0xff800000);
        }
        // key: (descending score, ascending place); ~0 for none
        unsigned long long last = 0;
        for (int j = 0; j < a.k; ++j) {
            unsigned long long best = ~0ull;
            for (int64_t i = tid; i < len; i += 256) {
                const float t = sgn * load_score(s + i);
                if (!takes_part(t, c)) continue;
                const unsigned long long key =
                    ((unsigned long long)float_key(-t) << 32) | (uint32_t)i;
                if ((j == 0 || key > last) && key < best) best = key;
            }
            redk[tid] = best;
            __syncthreads();
            for (int h = 128; h > 0; h >>= 1) {
                if (tid < h) redk[tid] = min(redk[tid], redk[tid + h]);
                __syncthreads();
            }
            last = redk[0];
            __syncthreads();
            if (tid == 0) {
                const int64_t at = (int64_t)(uint32_t)last;
                a.top_index[row * a.k + j] = last == ~0ull ? -1 : at;
                a.top[row * a.k + j] = last == ~0ull ? __int_as_float(0xff800000)
                                                     : logp(sgn * load_score(s + at));
            }
        }
    }
}

}  // namespace

int64_t score_probs_work(int64_t, int64_t, bool, int, int) { return 0; }

cudaError_t launch_score_probs(const ProbsArgs& a, int sms, cudaStream_t st) {
    const unsigned grid = (unsigned)std::min<int64_t>(a.nq, (int64_t)sms * 8);
    if (a.dtype == M3G_F32)
        score_probs_kernel<float><<<grid, 256, 0, st>>>(a);
    else
        score_probs_kernel<__nv_bfloat16><<<grid, 256, 0, st>>>(a);
    return cudaGetLastError();
}

}  // namespace m3g
