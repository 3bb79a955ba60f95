// k_probs.cu -- scores as probabilities: log-sum-exp, entropy, the log probability
// of given entries and the k most probable ones, in one pass over the scores.
//
// With t = score (scale > 0) or -score, c = |scale| and l = c t, a part of a row is
// summed up as (m, z, w): its largest t, z = sum e^d and w = sum d e^d, where
// d = c t - c m.  Parts join by M = max m, z' = e^(c m - c M) z and
// w' = e^(c m - c M) (w + (c m - c M) z); then logsumexp = c M + log z and
// entropy = log z - w / z.  d is one fma on c m as rounded, so the formulas hold
// exactly whatever that rounding was.  Entries that are NaN, or -inf after scaling,
// come out of max(d, -1000) with e^d = 0.
//
// The best k of a row pass through a buffer in shared memory: a thread offers the
// entries of its 16 that reach the current bound tau, a lower bound of the k-th
// best.  tau first comes from the threads' own maxima (at least k of them reach the
// smallest of the warps' ceil(k / 8)-th largest), later from the buffer itself, which
// is cut to its best k when it could overflow.
//
// The scores' bytes bound it.  A block of 256 threads takes a row, or one of P parts
// of it where rows are few; parts leave (m, z, w) and their best k in the caller's
// scratch and a second kernel joins them.
#include <cuda_bf16.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <cmath>

#include "common.cuh"
#include "kernels_scores.h"

namespace m3g {
namespace {

constexpr int kThreads = 256, kWarps = kThreads / 32;
constexpr int kPer = 16;                      // entries a thread holds of a tile
constexpr int kTile = kThreads * kPer;
constexpr int kBuf = kTile + kProbsMaxK;      // a tile always fits behind the best k
constexpr unsigned long long kNone = ~0ull;   // no entry

__device__ __forceinline__ float ninf() { return __int_as_float(0xff800000); }

struct Sums {
    float m, z, w;
};
__device__ __forceinline__ Sums no_sums() { return {ninf(), 0.f, 0.f}; }

// e^d within 2^-22 and |d| 2^-23 of its value; 0 below 2^-126
__device__ __forceinline__ float exp_of(float d) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(d * 1.4426950408889634f));
    return r;
}

// Two fp32 values in one register pair: sm_100 has packed fma, mul and add.
__device__ __forceinline__ uint64_t pack2(float a, float b) {
    uint64_t r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ void unpack2(uint64_t v, float& a, float& b) {
    asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(v));
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
    uint64_t r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
    uint64_t r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
    uint64_t r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}

// a part's sums taken to another reference value
__device__ __forceinline__ void rebase(Sums& s, float c, float m) {
    if (s.m == m || s.z == 0.f) {
        s.m = m;
        return;
    }
    const float d = fmaxf(c * s.m - c * m, -1000.f), f = exp_of(d);
    s.w = f * fmaf(d, s.z, s.w);
    s.z *= f;
    s.m = m;
}
__device__ __forceinline__ Sums join(Sums a, Sums b, float c) {
    const float m = fmaxf(a.m, b.m);
    rebase(a, c, m);
    rebase(b, c, m);
    a.z += b.z;
    a.w += b.w;
    return a;
}

struct Shared {
    unsigned long long buf[kBuf], best[kProbsMaxK];
    Sums sums[kWarps];
    float offer[kWarps];
    int count;
};

// One value for each warp, the sums of all its lanes in fixed order.
__device__ __forceinline__ Sums warp_join(Sums s, float c) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        Sums b;
        b.m = __shfl_xor_sync(0xffffffffu, s.m, o);
        b.z = __shfl_xor_sync(0xffffffffu, s.z, o);
        b.w = __shfl_xor_sync(0xffffffffu, s.w, o);
        s = join(s, b, c);
    }
    return s;
}

__device__ __forceinline__ Sums block_join(Sums s, float c, Shared& sm) {
    s = warp_join(s, c);
    __syncthreads();
    if ((threadIdx.x & 31) == 0) sm.sums[threadIdx.x >> 5] = s;
    __syncthreads();
    s = sm.sums[0];
#pragma unroll
    for (int i = 1; i < kWarps; ++i) s = join(s, sm.sums[i], c);
    return s;
}

// Bitonic sort of one float a lane, descending.
__device__ __forceinline__ float warp_sort_desc(float v) {
    const int lane = threadIdx.x & 31;
#pragma unroll
    for (int k = 2; k <= 32; k <<= 1)
#pragma unroll
        for (int j = k >> 1; j > 0; j >>= 1) {
            const float p = __shfl_xor_sync(0xffffffffu, v, j);
            v = (((lane & k) == 0) == ((lane & j) == 0)) ? fmaxf(v, p) : fminf(v, p);
        }
    return v;
}

// A value that at least k of the threads' v reach (all of them if fewer than k are
// above -inf): the smallest of the warps' ceil(k / kWarps)-th largest.
__device__ __forceinline__ float offered_bound(float v, int k, Shared& sm) {
    v = warp_sort_desc(v);
    const int nth = (k + kWarps - 1) / kWarps - 1;
    if ((threadIdx.x & 31) == nth) sm.offer[threadIdx.x >> 5] = v;
    __syncthreads();
    float b = sm.offer[0];
#pragma unroll
    for (int i = 1; i < kWarps; ++i) b = fminf(b, sm.offer[i]);
    __syncthreads();
    return b;
}

// Keys order entries best first: descending t, then ascending place.
__device__ __forceinline__ unsigned long long key_of(float t, uint32_t place) {
    return ((unsigned long long)float_key(-t) << 32) | place;
}
__device__ __forceinline__ float t_of(unsigned long long key) {
    return -key_float((uint32_t)(key >> 32));
}

// Appends the keys a thread passes (any of them kNone) to the buffer.
__device__ __forceinline__ void append(unsigned long long key, Shared& sm) {
    if (key != kNone) sm.buf[atomicAdd(&sm.count, 1)] = key;
}

// Cuts the buffer's n entries to their best min(k, n), sorted, and returns the
// number.  Every entry's place is the number of better ones, counted among the
// entries that reach a bound of the k-th best: first the warps' offers of the
// threads' best ones, then, where many entries still reach that (rows in ascending
// order), the exact k-th of them.
__device__ __noinline__ int best_of_buffer(int n, int k, Shared& sm) {
    const int tid = threadIdx.x;
    for (int pass = 0; pass < 2 && n > kThreads && n > 4 * k; ++pass) {
        unsigned long long mine[kBuf / kThreads + 1], best = kNone;
#pragma unroll
        for (int u = 0; u < kBuf / kThreads + 1; ++u) {
            const int i = tid + u * kThreads;
            mine[u] = i < n ? sm.buf[i] : kNone;
            best = min(best, mine[u]);
        }
        unsigned long long bound = kNone;  // entries above it are dropped
        if (pass == 0) {
            const float b = offered_bound(best == kNone ? ninf() : t_of(best), k, sm);
            if (b > ninf()) bound = key_of(b, 0xFFFFFFFFu);
        } else {
            __syncthreads();
            sm.buf[tid] = best;
            __syncthreads();
            int better = 0;
            for (int i = 0; i < kThreads; ++i) better += sm.buf[i] < best;
            // (n > kThreads, so every thread has a best one and they are distinct)
            if (better == k - 1) sm.buf[kThreads] = best;
            __syncthreads();
            bound = sm.buf[kThreads];
        }
        __syncthreads();
        if (tid == 0) sm.count = 0;
        __syncthreads();
#pragma unroll
        for (int u = 0; u < kBuf / kThreads + 1; ++u)
            append(mine[u] <= bound ? mine[u] : kNone, sm);
        __syncthreads();
        n = sm.count;
        __syncthreads();
    }
    // places among the n entries that are left
    const int kept = min(n, k);
    for (int i0 = tid; i0 < n; i0 += kThreads) {
        const unsigned long long key = sm.buf[i0];
        int better = 0;
        for (int i = 0; i < n; ++i) better += sm.buf[i] < key;
        if (better < k) sm.best[better] = key;
    }
    __syncthreads();
    if (tid < kept) sm.buf[tid] = sm.best[tid];
    if (tid == 0) sm.count = kept;
    __syncthreads();
    return kept;
}

// ---------------- a part of a row ----------------

template <class T>
struct Vec;
template <>
struct Vec<float> {
    static constexpr int kN = 4;
    __device__ static void unpack(const uint4& r, float* o) {
        o[0] = __uint_as_float(r.x);
        o[1] = __uint_as_float(r.y);
        o[2] = __uint_as_float(r.z);
        o[3] = __uint_as_float(r.w);
    }
};
template <>
struct Vec<__nv_bfloat16> {
    static constexpr int kN = 8;
    __device__ static void unpack(const uint4& r, float* o) {
        const uint32_t w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            o[2 * i] = __uint_as_float(w[i] << 16);
            o[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u);
        }
    }
};

__device__ __forceinline__ float load_score(const float* p) { return *p; }
__device__ __forceinline__ float load_score(const __nv_bfloat16* p) { return __bfloat162float(*p); }

struct RowAt {
    int64_t first, len;
};
__device__ __forceinline__ RowAt row_at(const ProbsArgs& a, int64_t row) {
    if (!a.row_off) return {row * a.ld, a.n};
    const int64_t b = max((int64_t)0, min(a.row_off[row], a.n));
    const int64_t len = max((int64_t)0, min(a.row_off[row + 1], a.n) - b);
    return {b, min(len, (int64_t)INT32_MAX)};
}

// l = c t, or the reference value where that is infinite
__device__ __forceinline__ float log_prob(float t, float c, float cm, float logz) {
    const float l = c * t;
    if (!(l > ninf())) return ninf();  // left out
    if (cm == __int_as_float(0x7f800000)) return l == cm ? __int_as_float(0x7fc00000) : ninf();
    return fmaf(c, t, -cm) - logz;
}

// The answer of a row from its sums and its best entries (in sm.buf, sorted).
template <class T>
__device__ void finish_row(const ProbsArgs& a, int64_t row, const RowAt& at, const Sums& s,
                           int kept, float c, float sgn, Shared& sm) {
    const float cm = s.z > 0.f || s.m > ninf() ? c * s.m : ninf();
    const bool inf = cm == __int_as_float(0x7f800000);
    const float logz = logf(s.z);
    if (threadIdx.x == 0) {
        a.lse[row] = inf || !(s.z > 0.f) ? cm : cm + logz;
        a.entropy[row] = inf          ? __int_as_float(0x7fc00000)
                         : s.z > 0.f ? fmaxf(logz - s.w / s.z, 0.f)  // (roundings aside)
                                     : 0.f;
    }
    const T* x = static_cast<const T*>(a.scores) + at.first;
    for (int j = threadIdx.x; j < a.ngiven; j += kThreads) {
        const int64_t g = a.given[row * a.ngiven + j];
        a.out_given[row * a.ngiven + j] =
            g >= 0 && g < at.len ? log_prob(sgn * load_score(x + g), c, cm, logz) : ninf();
    }
    for (int j = threadIdx.x; j < a.k; j += kThreads) {
        const unsigned long long key = j < kept ? sm.buf[j] : kNone;
        a.top_index[row * a.k + j] = key == kNone ? -1 : (int64_t)(uint32_t)key;
        a.top[row * a.k + j] = key == kNone ? ninf() : log_prob(t_of(key), c, cm, logz);
    }
    __syncthreads();
}

// A part's place in the scratch (on an 8-byte boundary): its sums, then its best k
// keys.
__device__ __forceinline__ unsigned char* part_at(const ProbsArgs& a, int64_t unit) {
    return static_cast<unsigned char*>(a.work) + unit * (16 + 8 * (int64_t)a.k);
}

template <class T>
__global__ void __launch_bounds__(kThreads, 3) score_probs_kernel(ProbsArgs a, int parts) {
    constexpr int V = Vec<T>::kN, kVecs = kPer / V;
    __shared__ Shared sm;
    const int tid = threadIdx.x;
    const float c = fabsf(a.scale), sgn = a.scale > 0.f ? 1.f : -1.f;
    const uint32_t flip = a.scale > 0.f ? 0u : 0x80000000u;
    for (int64_t unit = blockIdx.x; unit < a.nq * parts; unit += gridDim.x) {
        const int64_t row = unit / parts;
        const int part = (int)(unit - row * parts);
        const RowAt at = row_at(a, row);
        const T* x = static_cast<const T*>(a.scores) + at.first;
        // the row: `head` entries up to a 16-byte boundary, whole granules of 16 bytes,
        // the rest; a part has its share of the granules, the first one the others too
        const int len = (int)at.len;
        const int head = min(
            (int)((16 - (reinterpret_cast<uintptr_t>(x) & 15)) % 16 / sizeof(T)), len);
        const int ngran = (len - head) / V;
        const int g0 = (int)((int64_t)ngran * part / parts);
        const int g1 = (int)((int64_t)ngran * (part + 1) / parts);
        const uint4* gran = reinterpret_cast<const uint4*>(x + head);
        Sums s = no_sums();
        float tau = ninf();  // entries below it are not among the best k
        if (tid == 0) sm.count = 0;
        uint4 raw[kVecs];
        auto load = [&](int g) {
#pragma unroll
            for (int v = 0; v < kVecs; ++v) {
                const int i = g + v * kThreads + tid;
                raw[v] = i < g1 ? __ldcs(gran + i) : make_uint4(~0u, ~0u, ~0u, ~0u);  // NaNs
            }
        };
        load(g0);
        __syncthreads();
        // a tile: t[u] (NaN for none) is the row's entry place(u)
        auto tile = [&](float(&t)[kPer], auto place) {
            float m = ninf();
#pragma unroll
            for (int u = 0; u < kPer; ++u) {
                t[u] = __uint_as_float(__float_as_uint(t[u]) ^ flip);
                m = fmaxf(m, t[u]);
            }
            const bool some = c * m > ninf();
            if (some) {
                if (m > s.m) rebase(s, c, m);
                const float cm = c * s.m;
                const uint64_t cc = pack2(c, c), mm = pack2(-cm, -cm);
                const uint64_t l2 = pack2(1.4426950408889634f, 1.4426950408889634f);
                uint64_t z = 0, w = 0;
#pragma unroll
                for (int u = 0; u < kPer; u += 2) {
                    float d0, d1, e0, e1;
                    unpack2(fma2(cc, pack2(t[u], t[u + 1]), mm), d0, d1);
                    const uint64_t d = pack2(fmaxf(d0, -1000.f), fmaxf(d1, -1000.f));
                    unpack2(mul2(d, l2), d0, d1);
                    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e0) : "f"(d0));
                    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e1) : "f"(d1));
                    const uint64_t e = pack2(e0, e1);
                    z = add2(z, e);
                    w = fma2(e, d, w);
                }
                float z0, z1, w0, w1;
                unpack2(z, z0, z1);
                unpack2(w, w0, w1);
                s.z += z0 + z1;
                s.w += w0 + w1;
            }
            if (a.k > 0) {
                int n = sm.count;  // (read by all before any can append)
                const int able = __syncthreads_count(some && m >= tau);
                if (able == 0) return;
                if (n > 4 * a.k + 64 || n + able * kPer > kTile / 2) {
                    // much to append (the first tile, for one): a better bound first
                    if (n > a.k) {
                        n = best_of_buffer(n, a.k, sm);
                        if (n == a.k) tau = fmaxf(tau, t_of(sm.buf[n - 1]));
                    }
                    if (n + able * kPer > kTile / 2)
                        tau = fmaxf(tau, offered_bound(some ? m : ninf(), a.k, sm));
                    else
                        __syncthreads();
                }
                if (some && m >= tau) {
#pragma unroll
                    for (int u = 0; u < kPer; ++u)
                        if (t[u] >= tau && c * t[u] > ninf())
                            append(key_of(t[u], (uint32_t)place(u)), sm);
                }
                __syncthreads();
            }
        };
        float t[kPer];
        if (part == 0 && V * ngran < len) {  // entries outside whole granules
            const int tail = head + V * ngran;
            const int i = tid < head ? tid : tail + tid - head;
#pragma unroll
            for (int u = 0; u < kPer; ++u) t[u] = __int_as_float(0x7fc00000);
            if (tid < head || (tid < 2 * V && i < len)) t[0] = load_score(x + i);
            tile(t, [&](int) { return i; });
        }
        for (int g = g0; g < g1; g += kVecs * kThreads) {
#pragma unroll
            for (int v = 0; v < kVecs; ++v) Vec<T>::unpack(raw[v], t + v * V);
            load(g + kVecs * kThreads);
            tile(t, [&](int u) { return head + (g + (u / V) * kThreads + tid) * V + u % V; });
        }
        s = block_join(s, c, sm);
        int kept = 0;
        if (a.k > 0) kept = best_of_buffer(sm.count, a.k, sm);
        if (parts == 1) {
            finish_row<T>(a, row, at, s, kept, c, sgn, sm);
        } else {
            unsigned char* o = part_at(a, unit);
            if (tid == 0) {
                reinterpret_cast<float2*>(o)[0] = make_float2(s.m, s.z);
                reinterpret_cast<float2*>(o)[1] = make_float2(s.w, 0.f);
            }
            for (int j = tid; j < a.k; j += kThreads)
                reinterpret_cast<unsigned long long*>(o + 16)[j] = j < kept ? sm.buf[j] : kNone;
            __syncthreads();
        }
    }
}

// Joins a row's parts: their sums in a fixed order, their best keys through the
// same buffer.
template <class T>
__global__ void __launch_bounds__(kThreads) join_parts_kernel(ProbsArgs a, int parts) {
    __shared__ Shared sm;
    const int tid = threadIdx.x;
    const float c = fabsf(a.scale), sgn = a.scale > 0.f ? 1.f : -1.f;
    for (int64_t row = blockIdx.x; row < a.nq; row += gridDim.x) {
        const RowAt at = row_at(a, row);
        if (tid == 0) sm.count = 0;
        Sums s = no_sums();
        for (int i = tid; i < parts; i += kThreads) {
            const float2* v =
                reinterpret_cast<const float2*>(part_at(a, row * parts + i));
            s = join(s, Sums{v[0].x, v[0].y, v[1].x}, c);
        }
        s = block_join(s, c, sm);
        int kept = 0;
        if (a.k > 0) {
            unsigned long long tau = kNone;
            const int64_t total = (int64_t)parts * a.k;
            for (int64_t b = 0; b < total; b += kTile) {
                for (int64_t i = b + tid; i < min(b + kTile, total); i += kThreads) {
                    const int p = (int)(i / a.k), j = (int)(i - (int64_t)p * a.k);
                    const unsigned long long key = reinterpret_cast<const unsigned long long*>(
                        part_at(a, row * parts + p) + 16)[j];
                    append(key <= tau ? key : kNone, sm);
                }
                __syncthreads();
                kept = best_of_buffer(sm.count, a.k, sm);
                if (kept == a.k) tau = sm.buf[kept - 1];
                __syncthreads();
            }
        }
        finish_row<T>(a, row, at, s, kept, c, sgn, sm);
    }
}

// Parts a row: enough units that the blocks the GPU holds at once (three an SM) finish
// together, each unit worth at least a tile.  A row's fixed work (its first bound,
// its final order) is taken as a tile.
int parts_of(int64_t nq, int64_t n, bool ragged, int sms) {
    const int64_t slots = 3 * (int64_t)sms;
    const int64_t len = ragged ? n / std::max<int64_t>(nq, 1) : n;
    const int64_t most = std::min<int64_t>(std::max<int64_t>(len / kTile, 1), slots);
    int best = 1;
    double cost = 0;
    for (int64_t p = 1; p <= most; p += 1 + p / 8) {
        const double c = (double)((nq * p + slots - 1) / slots) * ((double)len / p + kTile);
        if (p == 1 || c < 0.95 * cost) {
            best = (int)p;
            cost = c;
        }
        if (nq * p > 8 * slots) break;
    }
    return best;
}

}  // namespace

int64_t score_probs_work(int64_t nq, int64_t n, bool ragged, int k, int sms) {
    const int parts = parts_of(nq, n, ragged, sms);
    return parts == 1 ? 0 : nq * parts * (16 + 8 * (int64_t)k);
}

cudaError_t launch_score_probs(const ProbsArgs& a, int sms, cudaStream_t st) {
    const int parts = parts_of(a.nq, a.n, a.row_off != nullptr, sms);
    const unsigned grid = (unsigned)std::min<int64_t>(a.nq * parts, (int64_t)1 << 30);
    const unsigned rows = (unsigned)std::min<int64_t>(a.nq, (int64_t)1 << 30);
    if (a.dtype == M3G_F32) {
        score_probs_kernel<float><<<grid, kThreads, 0, st>>>(a, parts);
        if (parts > 1) join_parts_kernel<float><<<rows, kThreads, 0, st>>>(a, parts);
    } else {
        score_probs_kernel<__nv_bfloat16><<<grid, kThreads, 0, st>>>(a, parts);
        if (parts > 1) join_parts_kernel<__nv_bfloat16><<<rows, kThreads, 0, st>>>(a, parts);
    }
    return cudaGetLastError();
}

}  // namespace m3g
