// k_probs.cu -- scores as probabilities: log-sum-exp, entropy, the log probability
// of given entries and the k most probable ones, in one pass over the scores.
//
// With t = score (scale > 0) or -score, c = |scale| and l = c t, a part of a row is
// summed up as (m, z, w): its largest t, z = sum e^d and w = sum d e^d, where
// d = c t - c m.  Parts join by M = max m, z' = e^(c m - c M) z and
// w' = e^(c m - c M) (w + (c m - c M) z); then logsumexp = c M + log z and
// entropy = log z - w / z.  d is one fma on c m as rounded, so the formulas hold
// exactly whatever that rounding was, as long as e^(what it cut off) is near one: a part
// whose |c m| is 2^24 or more is summed up again from c m in two words (ref_of; in the
// first pass the second word cost 3% of every row's time).  Entries that are NaN, or
// -inf after scaling, come out of max(d, -1000) with e^d = 0; a.lowest is the least t
// that is neither.
//
// A warp takes a row, or one of P parts of it where rows are few, on its own: no warp
// waits for another, and one's latencies (row offsets, the final order, the outputs)
// pass behind the others' work.  Its scores come through a ring of two 4 KB bulk
// copies, so 160 KB an SM are in flight whatever the warps do.  Parts leave (m, z, w)
// and their best k in the caller's scratch and a second kernel joins them.
//
// The best k pass through a buffer of the warp's: entries that reach the bound tau, a
// lower bound of the k-th best.  tau first comes from the maxima of a stage's granules
// (16 bytes, eight a lane): at least k of the 256 reach the smallest of the eight
// rounds' ceil(k / 8)-th largest.  The buffer is cut to its best k, which sharpens tau,
// whenever it holds twice as many, and before it could overflow.
//
// The scores' bytes bound it without the best k (1024 rows x 100003 fp32: 67 us, 6.1
// TB/s); the best k add work that each warp does in turn: 89 us for k = 10, 177 for 100;
// 4096 rows of 3904 bf16 scores 16 us, and 36 and 73.  A row of 1000003 is latency: 9 us
// for its 488 parts and 6 to join them, k = 10.  Blocks of 256 threads a row, all of a
// row's best k through one buffer, took 107 us (k = 0) and 198 (10) for the first shape.
#include <cuda_bf16.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <atomic>
#include <cmath>
#include <type_traits>

#include "common.cuh"
#include "kernels_scores.h"
#include "tc.cuh"
#include "topk.cuh"

namespace m3g {
namespace {

constexpr unsigned long long kNone = ~0ull;   // no entry

// The warps of the first kernel, as many as shared memory holds: their latencies, not
// the bytes, are what the best k cost.  KW: k <= 32 KW.
constexpr int kStages = 2, kStageBytes = 4096, kRounds = kStageBytes / 512;
constexpr __host__ __device__ int warps_of(int kw) { return kw == 1 ? 20 : 16; }
// keys a warp's buffer holds: fewer than 2 k + 8, and a round (32 granules of up to 8)
constexpr __host__ __device__ int cap_of(int kw) { return 64 * kw + 32 + 256; }

// the block that joins a row's parts
constexpr int kThreads = 256, kJoinWarps = kThreads / 32;
constexpr int kTile = 4096;
constexpr int kBuf = kTile + kProbsMaxK;

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

// The value hi + lo that a part's z and w refer to: c m as rounded (not fused into what
// it is subtracted from) and, where that may be off by 1/2 and more, what the rounding
// cut off (exact).  With hi alone, at c m = 3e9, the largest entry's e^d could be e^128.
struct Ref {
    float hi, lo;
};
__device__ __forceinline__ Ref ref_of(float c, float m) {
    const float hi = __fmul_rn(c, m), a = fabsf(hi);
    return {hi, a >= 16777216.f && a < __int_as_float(0x7f800000) ? fmaf(c, m, -hi) : 0.f};
}
// c t less the reference value.  Next to a c m that was rounded by lo there are no
// entries nearer than lo / 2, so the two roundings are within 2^-22 of the result.  (A
// branch: subtracted always, 4096 ragged rows' best 10 took 38 us for 36.)
__device__ __forceinline__ float from_ref(float c, float t, const Ref& ref) {
    float d = fmaf(c, t, -ref.hi);
    if (__builtin_expect(ref.lo != 0.f, 0)) d -= ref.lo;
    return d;
}

// a part's sums taken to another reference value; LO: of two words
template <bool LO = true>
__device__ __forceinline__ void rebase(Sums& s, float c, float m) {
    if (s.m == m || s.z == 0.f) {
        s.m = m;
        return;
    }
    float d = __fmul_rn(c, s.m) - __fmul_rn(c, m);
    if (LO) d += ref_of(c, s.m).lo - ref_of(c, m).lo;
    d = fmaxf(d, -1000.f);
    const float f = exp_of(d);
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

// The sums of all lanes, in fixed order, in every lane.
template <bool LO = true>
__device__ __forceinline__ Sums warp_join(Sums s, float c) {
    float m = s.m;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
    rebase<LO>(s, c, m);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        s.z += __shfl_xor_sync(0xffffffffu, s.z, o);
        s.w += __shfl_xor_sync(0xffffffffu, s.w, o);
    }
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

// Keys order entries best first: descending t, then ascending place.
__device__ __forceinline__ unsigned long long key_of(float t, uint32_t place) {
    return ((unsigned long long)float_key(-t) << 32) | place;
}
__device__ __forceinline__ float t_of(unsigned long long key) {
    return -key_float((uint32_t)(key >> 32));
}

struct Shared {  // of the joining block
    unsigned long long buf[kBuf], best[kProbsMaxK];
    Sums sums[kJoinWarps];
    float offer[kJoinWarps];
    int count;
};

__device__ __forceinline__ Sums block_join(Sums s, float c, Shared& sm) {
    s = warp_join(s, c);
    __syncthreads();
    if ((threadIdx.x & 31) == 0) sm.sums[threadIdx.x >> 5] = s;
    __syncthreads();
    s = sm.sums[0];
#pragma unroll
    for (int i = 1; i < kJoinWarps; ++i) s = join(s, sm.sums[i], c);
    return s;
}

// A value that at least k of the threads' v reach (all of them if fewer than k are
// above -inf): the smallest of the warps' ceil(k / 8)-th largest.
__device__ __forceinline__ float offered_bound(float v, int k, Shared& sm) {
    v = warp_sort_desc(v);
    const int nth = (k + kJoinWarps - 1) / kJoinWarps - 1;
    if ((threadIdx.x & 31) == nth) sm.offer[threadIdx.x >> 5] = v;
    __syncthreads();
    float b = sm.offer[0];
#pragma unroll
    for (int i = 1; i < kJoinWarps; ++i) b = fminf(b, sm.offer[i]);
    __syncthreads();
    return b;
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
            if (tid == 0) sm.buf[kThreads] = kNone;
            __syncthreads();
            int better = 0;
            for (int i = 0; i < kThreads; ++i) better += sm.buf[i] < best;
            __syncthreads();
            if (best != kNone && better == k - 1) sm.buf[kThreads] = best;
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
    if (tid < kProbsMaxK) sm.best[tid] = kNone;
    __syncthreads();
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
    const int64_t b = a.row_off[row], e = a.row_off[row + 1];
    if (b >= 0 && b <= e && e <= a.n && e - b <= kProbsMaxRow) return {b, e - b};
    atomicOr(a.err + kScoreBadItem, 1);
    return {0, 0};
}

// l = c t, or the reference value where that is infinite
__device__ __forceinline__ float log_prob(float t, float c, const Ref& ref, float logz) {
    const float l = c * t;
    if (!(l > ninf())) return ninf();  // left out
    if (ref.hi == __int_as_float(0x7f800000))
        return l == ref.hi ? __int_as_float(0x7fc00000) : ninf();
    return from_ref(c, t, ref) - logz;
}

// The answer of a row from its sums and its best entries (keys, sorted, kept of them),
// by `threads` threads; ref is of s.m.
template <class T>
__device__ __forceinline__ void finish_row(const ProbsArgs& a, int64_t row, const RowAt& at,
                                           const Sums& s, const Ref& ref,
                                           const unsigned long long* keys, int kept, float c,
                                           float sgn, int tid, int threads) {
    const bool inf = ref.hi == __int_as_float(0x7f800000);
    const float logz = logf(s.z);
    if (tid == 0) {
        a.lse[row] = inf || !(s.z > 0.f) ? ref.hi : ref.hi + (ref.lo + logz);
        a.entropy[row] = inf          ? __int_as_float(0x7fc00000)
                         : s.z > 0.f ? fmaxf(logz - s.w / s.z, 0.f)  // (roundings aside)
                                     : 0.f;
    }
    const T* x = static_cast<const T*>(a.scores) + at.first;
    for (int j = tid; j < a.ngiven; j += threads) {
        const int64_t g = a.given[row * a.ngiven + j];
        a.out_given[row * a.ngiven + j] =
            g >= 0 && g < at.len ? log_prob(sgn * load_score(x + g), c, ref, logz) : ninf();
    }
    for (int j = tid; j < a.k; j += threads) {
        const unsigned long long key = j < kept ? keys[j] : kNone;
        a.top_index[row * a.k + j] = key == kNone ? -1 : (int64_t)(uint32_t)key;
        a.top[row * a.k + j] = key == kNone ? ninf() : log_prob(t_of(key), c, ref, logz);
    }
}

// A part's place in the scratch (on an 8-byte boundary): its sums, then its best k
// keys.
__device__ __forceinline__ unsigned char* part_at(const ProbsArgs& a, int64_t unit) {
    return static_cast<unsigned char*>(a.work) + unit * (16 + 8 * (int64_t)a.k);
}

// ---------------- the warps ----------------

template <int KW>
struct alignas(128) WarpShared {
    unsigned char stage[kStages][kStageBytes];
    unsigned long long buf[cap_of(KW)];
    uint64_t full[kStages];
    int lost;  // a wait gave up
};

// The number of all lanes' words that are at most v.
template <int W>
__device__ __forceinline__ int count_to(const uint32_t (&w)[W], uint32_t v) {
    int c = 0;
#pragma unroll
    for (int r = 0; r < W; ++r) c += w[r] <= v;
    return __reduce_add_sync(0xffffffffu, c);
}

// Cuts the warp's buffer of n keys to its best min(k, n), sorted; returns their number.
// Keys past the 32 KW that the sort holds are dropped first, by bisection on the high
// words for one that at least k and at most 32 KW keys reach and, where more than those
// share the k-th place's high word, on the low ones (their places).  Entries from `raw`
// on are not keys yet: their high word is t itself.
template <int KW>
__device__ __noinline__ int cut(unsigned long long* buf, int raw, int n, int k) {
    constexpr int W = cap_of(KW) / 32;
    const int lane = threadIdx.x & 31;
    __syncwarp();
    for (int i = raw + lane; i < n; i += 32)
        buf[i] = key_of(__uint_as_float((uint32_t)(buf[i] >> 32)), (uint32_t)buf[i]);
    __syncwarp();
    if (n > 32 * KW) {
        // (no key's high word is ~0: that is where float_key puts NaN)
        uint32_t w[W], lo = 0xFFFFFFFFu, hi = 0;
#pragma unroll
        for (int r = 0; r < W; ++r) {
            w[r] = 0xFFFFFFFFu;
            if (32 * r + lane < n) {
                w[r] = (uint32_t)(buf[32 * r + lane] >> 32);
                lo = min(lo, w[r]);
                hi = max(hi, w[r]);
            }
        }
        lo = __reduce_min_sync(0xffffffffu, lo);
        hi = __reduce_max_sync(0xffffffffu, hi);
        int c = n;  // keys up to hi
        while (c > 32 * KW && lo < hi) {
            const uint32_t mid = lo + (hi - lo) / 2;
            const int m = count_to(w, mid);
            if (m >= k) {
                hi = mid;
                c = m;
            } else {
                lo = mid + 1;
            }
        }
        const uint32_t high = hi;
        uint32_t low = 0xFFFFFFFFu;
        if (c > 32 * KW) {
            // places, plus one, of the keys of that high word; 0 for those before it
#pragma unroll
            for (int r = 0; r < W; ++r)
                if (32 * r + lane < n)
                    w[r] = w[r] < high    ? 0u
                           : w[r] == high ? (uint32_t)buf[32 * r + lane] + 1u
                                          : 0xFFFFFFFFu;
            uint32_t a = 0, b = 0xFFFFFFFEu;  // (places are below 2^31)
            while (c > 32 * KW) {
                const uint32_t mid = a + (b - a) / 2;
                const int m = count_to(w, mid);
                if (m >= k) {
                    b = mid;
                    c = m;
                } else {
                    a = mid + 1;
                }
            }
            low = b - 1u;
        }
        const unsigned long long last = ((unsigned long long)high << 32) | low;
        int m = 0;
#pragma unroll 1
        for (int b = 0; b < n; b += 32) {
            const unsigned long long key = b + lane < n ? buf[b + lane] : kNone;
            const bool keep = b + lane < n && key <= last;
            const unsigned ball = __ballot_sync(0xffffffffu, keep);
            if (keep) buf[m + __popc(ball & ((1u << lane) - 1u))] = key;  // (at or before b + lane)
            m += __popc(ball);
            __syncwarp();
        }
        n = m;
    }
    // bitonic sort of 32 KW keys, key 32 r + lane in v[r]
    unsigned long long v[KW];
#pragma unroll
    for (int r = 0; r < KW; ++r) v[r] = 32 * r + lane < n ? buf[32 * r + lane] : kNone;
    auto step = [&](int size, int j) {
#pragma unroll
        for (int r = 0; r < KW; ++r) {
            const unsigned long long p = shfl_xor_u64(v[r], j);
            const bool up = ((32 * r + lane) & size) == 0, lower = (lane & j) == 0;
            v[r] = lower == up ? min(v[r], p) : max(v[r], p);
        }
    };
    if constexpr (KW == 1) {
#pragma unroll
        for (int size = 2; size <= 32; size <<= 1)
#pragma unroll
            for (int j = size >> 1; j > 0; j >>= 1) step(size, j);
    } else {
        // rolled: unrolled it is most of the kernel's code, and a fourth of the time of
        // 4096 rows' best 100 went into fetching that
        static_assert(KW == 4, "");
        auto order = [](unsigned long long& a, unsigned long long& b, bool up) {
            const unsigned long long x = min(a, b), y = max(a, b);
            a = up ? x : y;
            b = up ? y : x;
        };
#pragma unroll 1
        for (int size = 2; size <= 128; size <<= 1) {
            if (size == 128) {
                order(v[0], v[2], true);
                order(v[1], v[3], true);
            }
            if (size >= 64) {
                order(v[0], v[1], true);
                order(v[2], v[3], size == 128);
            }
#pragma unroll 1
            for (int j = min(size >> 1, 16); j > 0; j >>= 1) step(size, j);
        }
    }
    n = min(n, k);
    __syncwarp();
#pragma unroll
    for (int r = 0; r < KW; ++r)
        if (32 * r + lane < n) buf[32 * r + lane] = v[r];
    __syncwarp();
    return n;
}

// A warp's unit: a row's part p of P.  The row: `head` entries up to a 16-byte
// boundary, whole granules of 16 bytes, the rest; a part has its share of the
// granules, the first one the other entries too.
template <class T>
struct Unit {
    int64_t row;
    RowAt at;
    int head, ngran, g0, g1, part;

    __device__ __forceinline__ void set(const ProbsArgs& a, int64_t unit, int parts, RowAt r) {
        constexpr int V = Vec<T>::kN;
        row = unit / parts;
        part = (int)(unit - row * parts);
        at = r;
        const uintptr_t x =
            reinterpret_cast<uintptr_t>(static_cast<const T*>(a.scores) + at.first);
        head = min((int)((16 - (x & 15)) % 16 / sizeof(T)), (int)at.len);
        ngran = ((int)at.len - head) / V;
        g0 = (int)((int64_t)ngran * part / parts);
        g1 = (int)((int64_t)ngran * (part + 1) / parts);
    }
    __device__ __forceinline__ const T* base(const ProbsArgs& a) const {
        return static_cast<const T*>(a.scores) + at.first;
    }
};

// A part's n entries from x on, and one a lane besides, summed up again from a reference
// value in two words; m is their largest score.  In blocks of sixteen a lane, so that a
// long row's sums lose no more than the first pass's.
template <class T>
__device__ __noinline__ Sums sums_of_far(const T* x, int n, float edge, float c, float sgn,
                                         float m) {
    const Ref ref = ref_of(c, m);
    Sums s{m, 0.f, 0.f};
    auto add = [&](float t, float& z, float& w) {
        const float d = fmaxf(from_ref(c, t, ref), -1000.f), e = exp_of(d);
        z += e;
        w = fmaf(e, d, w);
    };
    for (int64_t b = threadIdx.x & 31; b < n; b += 32 * 16) {
        float z = 0.f, w = 0.f;
#pragma unroll 4
        for (int u = 0; u < 16; ++u)
            if (b + 32 * u < n) add(sgn * load_score(x + b + 32 * u), z, w);
        s.z += z;
        s.w += w;
    }
    add(sgn * edge, s.z, s.w);
    return warp_join<false>(s, c);
}

template <class T, int KW>
__global__ void __launch_bounds__(warps_of(KW) * 32, 1)
    score_probs_kernel(ProbsArgs a, int parts) {
    constexpr int V = Vec<T>::kN;
    extern __shared__ unsigned char smem_raw[];
    const int lane = threadIdx.x & 31;
    WarpShared<KW>& sm = reinterpret_cast<WarpShared<KW>*>(
        (reinterpret_cast<uintptr_t>(smem_raw) + 127) & ~uintptr_t(127))[threadIdx.x >> 5];
    const float c = fabsf(a.scale), sgn = a.scale > 0.f ? 1.f : -1.f;
    const uint32_t flip = a.scale > 0.f ? 0u : 0x80000000u;
    const int64_t units = a.nq * parts, step = (int64_t)gridDim.x * warps_of(KW);
    // a block's warps take units far apart, so that a few units use every SM
    const int64_t first = (int64_t)(threadIdx.x >> 5) * gridDim.x + blockIdx.x;
    if (lane == 0) {
        for (int s = 0; s < kStages; ++s) mbar_init(&sm.full[s], 1);
        fence_mbar_init();
        sm.lost = 0;
    }
    __syncwarp();
    bool lost = false;  // a wait gave up: nothing more is read or written

    // the copies run ahead of the work by up to kStages, into later units too
    Unit<T> load;
    int64_t load_unit = first;
    RowAt load_next = {0, 0};  // the row after it, fetched early
    int load_g = 0;
    uint32_t issued = 0, used = 0;
    auto row_of = [&](int64_t unit) {
        return unit < units ? row_at(a, unit / parts) : RowAt{0, 0};
    };
    auto open_load = [&](RowAt r) {
        if (load_unit < units) {
            load.set(a, load_unit, parts, r);
            load_g = load.g0;
            load_next = row_of(load_unit + step);
        }
    };
    auto issue = [&] {
        while (issued - used < kStages && load_unit < units) {
            if (load_g >= load.g1) {
                load_unit += step;
                open_load(load_next);
                continue;
            }
            const int n = min(load.g1 - load_g, kStageBytes / 16);
            const uint32_t s = issued % kStages;
            if (lane == 0) {
                mbar_arrive_expect_tx(&sm.full[s], (uint32_t)n * 16);
                bulk_g2s(sm.stage[s], load.base(a) + load.head + (int64_t)load_g * V,
                         (uint32_t)n * 16, &sm.full[s]);
            }
            load_g += n;
            ++issued;
        }
    };
    open_load(row_of(load_unit));
    issue();

    RowAt next_row = row_of(first);
    for (int64_t unit = first; unit < units && !lost; unit += step) {
        Unit<T> u;
        u.set(a, unit, parts, next_row);
        next_row = row_of(unit + step);
        const T* x = u.base(a);
        const int len = (int)u.at.len;
        // the entries outside whole granules, one a lane, used last
        float edge = __int_as_float(0x7fc00000);
        const int edge_at = lane < u.head ? lane : u.head + V * u.ngran + lane - u.head;
        if (u.part == 0 && edge_at < len && (lane < u.head || edge_at >= u.head + V * u.ngran))
            edge = load_score(x + edge_at);
        Sums s = no_sums();
        float tau = a.lowest;  // entries below it are not among the best k
        int n = 0, keys = 0;  // entries in the buffer, and how many of them are keys
        auto sharpen = [&] {
            n = keys = cut<KW>(sm.buf, keys, n, a.k);
            if (n == a.k) tau = fmaxf(tau, t_of(sm.buf[n - 1]));
        };
        // Appends the lanes' entries (E each) that reach tau.
        auto offer = [&](const auto& t, int place) {
            constexpr int E = sizeof(t) / sizeof(float);
            if (n + 32 * E > cap_of(KW)) sharpen();
#pragma unroll
            for (int i = 0; i < E; ++i) {
                const bool hit = t[i] >= tau;
                const unsigned ball = __ballot_sync(0xffffffffu, hit);
                if (hit)
                    sm.buf[n + __popc(ball & ((1u << lane) - 1u))] =
                        (unsigned long long)__float_as_uint(t[i]) << 32 | (uint32_t)(place + i);
                n += __popc(ball);
            }
        };
        for (int g = u.g0; g < u.g1; g += kStageBytes / 16) {
            const uint32_t slot = used % kStages;
            const bool ok = mbar_wait(&sm.full[slot], (used / kStages) & 1u, &sm.lost);
            if (!__all_sync(0xffffffffu, ok)) {
                lost = true;
                break;
            }
            const uint4* st = reinterpret_cast<const uint4*>(sm.stage[slot]);
            const int left = u.g1 - g;  // granules
            // the lane's granule of round r, oriented, NaN past the last one
            auto granule = [&](int r, float(&v)[V]) {
                const uint4 nan = make_uint4(~0u, ~0u, ~0u, ~0u);
                Vec<T>::unpack(r * 32 + lane < left ? st[r * 32 + lane] : nan, v);
#pragma unroll
                for (int i = 0; i < V; ++i)
                    v[i] = __uint_as_float(__float_as_uint(v[i]) ^ flip);
            };
            // the sums, half of the stage's entries at a time in registers
            float m = ninf(), top[kRounds];
            auto half = [&](auto from) {
            constexpr int R0 = decltype(from)::value, R1 = R0 + kRounds / 2;
            float t[kRounds / 2][V], hm = ninf();
#pragma unroll
            for (int r = R0; r < R1; ++r) {
                granule(r, t[r - R0]);
                top[r] = ninf();
#pragma unroll
                for (int i = 0; i < V; ++i) top[r] = fmaxf(top[r], t[r - R0][i]);
                hm = fmaxf(hm, top[r]);
            }
            m = fmaxf(m, hm);
            if (hm >= a.lowest) {
                if (hm > s.m) rebase<false>(s, c, hm);
                const float cm = __fmul_rn(c, s.m);
                const uint64_t cc = pack2(c, c), mm = pack2(-cm, -cm);
                const uint64_t l2 = pack2(1.4426950408889634f, 1.4426950408889634f);
                uint64_t z = 0, w = 0;
#pragma unroll
                for (int r = 0; r < kRounds / 2; ++r)
#pragma unroll
                    for (int i = 0; i < V; i += 2) {
                        float d0, d1, e0, e1;
                        unpack2(fma2(cc, pack2(t[r][i], t[r][i + 1]), mm), d0, d1);
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
            };
            half(std::integral_constant<int, 0>());
            half(std::integral_constant<int, kRounds / 2>());
            if (a.k > 0 && __any_sync(0xffffffffu, m >= tau)) {
                if (g == u.g0) {
                    if (KW == 1) {
                        tau = fmaxf(tau, __shfl_sync(0xffffffffu, warp_sort_desc(m), a.k - 1));
                    } else {
                        const int nth = (a.k + kRounds - 1) / kRounds - 1;
                        float b = __int_as_float(0x7f800000);
#pragma unroll 1
                        for (int r = 0; r < kRounds; ++r) {
                            float v[V], best = ninf();
                            granule(r, v);
#pragma unroll
                            for (int i = 0; i < V; ++i) best = fmaxf(best, v[i]);
                            b = fminf(b, __shfl_sync(0xffffffffu, warp_sort_desc(best), nth));
                        }
                        tau = fmaxf(tau, b);
                    }
                }
                unsigned act = 0;
#pragma unroll
                for (int r = 0; r < kRounds; ++r)
                    act |= __any_sync(0xffffffffu, top[r] >= tau) ? 1u << r : 0u;
                // (read again, round by round, in a short loop)
#pragma unroll 1
                for (; act; act &= act - 1) {
                    const int r = __ffs(act) - 1;
                    float v[V];
                    granule(r, v);
                    offer(v, u.head + (g + r * 32 + lane) * V);
                }
                if (n >= 2 * a.k + 8) sharpen();
            }
            __syncwarp();
            ++used;
            issue();
        }
        if (lost) break;
        if (__any_sync(0xffffffffu, edge == edge)) {
            const float t[1] = {__uint_as_float(__float_as_uint(edge) ^ flip)};
            if (t[0] >= a.lowest) {
                if (t[0] > s.m) rebase<false>(s, c, t[0]);
                const float d = fmaxf(fmaf(c, t[0], -__fmul_rn(c, s.m)), -1000.f), e = exp_of(d);
                s.z += e;
                s.w = fmaf(e, d, s.w);
            }
            if (a.k > 0) offer(t, edge_at);
        }
        s = warp_join<false>(s, c);
        const Ref ref = ref_of(c, s.m);
        // c m has a second word, or an early m had, and left an infinite sum (times 0) that
        // a masked run of entries made (all of this is the same in every lane)
        if (__builtin_expect(ref.lo != 0.f || !(fabsf(s.w) < __int_as_float(0x7f800000)), 0))
            s = sums_of_far(x + u.head + (int64_t)u.g0 * V, (u.g1 - u.g0) * V, edge, c, sgn, s.m);
        int kept = 0;
        if (a.k > 0) kept = cut<KW>(sm.buf, keys, n, a.k);
        if (parts == 1) {
            finish_row<T>(a, u.row, u.at, s, ref, sm.buf, kept, c, sgn, lane, 32);
        } else {
            unsigned char* o = part_at(a, unit);
            if (lane == 0) {
                reinterpret_cast<float2*>(o)[0] = make_float2(s.m, s.z);
                reinterpret_cast<float2*>(o)[1] = make_float2(s.w, 0.f);
            }
            for (int j = lane; j < a.k; j += 32)
                reinterpret_cast<unsigned long long*>(o + 16)[j] = j < kept ? sm.buf[j] : kNone;
        }
        __syncwarp();
    }
    if (lost) {
        // no copy may still be landing when the warp leaves
        if (lane == 0) {
            atomicOr(a.err + kScoreTimeout, 1);
            for (uint32_t k = used; k != issued; ++k)
                mbar_drain(&sm.full[k % kStages], (k / kStages) & 1u);
        }
        __syncwarp();
    }
}

// The sums and keys of the first kernel, visible to one launched to start before its
// end.
__device__ __forceinline__ void after_first_kernel() { cudaGridDependencySynchronize(); }

// Joins a row's parts: their sums in a fixed order, their best keys through the
// block's buffer.
template <class T>
__global__ void __launch_bounds__(kThreads) join_parts_kernel(ProbsArgs a, int parts) {
    __shared__ Shared sm;
    const int tid = threadIdx.x;
    const float c = fabsf(a.scale), sgn = a.scale > 0.f ? 1.f : -1.f;
    after_first_kernel();
    for (int64_t row = blockIdx.x; row < a.nq; row += gridDim.x) {
        const RowAt at = row_at(a, row);
        Sums s = no_sums();
        for (int i = tid; i < parts; i += kThreads) {
            const float2* v = reinterpret_cast<const float2*>(part_at(a, row * parts + i));
            s = join(s, Sums{v[0].x, v[0].y, v[1].x}, c);
        }
        auto key_at = [&](int p, int j) {
            return reinterpret_cast<const unsigned long long*>(part_at(a, row * parts + p) +
                                                               16)[j];
        };
        int kept = 0, n = kBuf + 1;
        if (a.k > 0 && parts >= 2 * a.k) {
            // many parts: only those whose best key reaches a bound of the k-th best of
            // all the parts' best ones have any of the row's best k
            unsigned long long head = kNone;
            for (int i = tid; i < parts; i += kThreads) head = min(head, key_at(i, 0));
            if (tid == 0) sm.count = 0;
            const float b = offered_bound(head == kNone ? ninf() : t_of(head), a.k, sm);
            const unsigned long long bound = b > ninf() ? key_of(b, 0xFFFFFFFFu) : kNone - 1;
            for (int i = tid; i < parts; i += kThreads)
                for (int j = 0; j < a.k; ++j) {
                    const unsigned long long key = key_at(i, j);
                    if (key > bound) break;
                    const int at = atomicAdd(&sm.count, 1);
                    if (at < kBuf) sm.buf[at] = key;
                }
            __syncthreads();
            n = sm.count;
            __syncthreads();
            if (n <= kBuf) kept = best_of_buffer(n, a.k, sm);
        }
        if (n > kBuf) {
            const int total = parts * a.k;
            for (int b = 0; b < total; b += kTile) {
                const int m = min(kTile, total - b);
                for (int i = tid; i < m; i += kThreads) {
                    const int p = (b + i) / a.k;
                    sm.buf[kept + i] = key_at(p, (b + i) - p * a.k);
                }
                __syncthreads();
                kept = best_of_buffer(kept + m, a.k, sm);
            }
        }
        s = block_join(s, c, sm);
        finish_row<T>(a, row, at, s, ref_of(c, s.m), sm.buf, kept, c, sgn, tid, kThreads);
        __syncthreads();
    }
}

// The same by a warp a row, where all the parts' keys fit a warp's buffer.
template <class T, int KW>
__global__ void __launch_bounds__(128) join_few_parts_kernel(ProbsArgs a, int parts) {
    __shared__ unsigned long long bufs[4][cap_of(KW)];
    const int lane = threadIdx.x & 31;
    unsigned long long* buf = bufs[threadIdx.x >> 5];
    const float c = fabsf(a.scale), sgn = a.scale > 0.f ? 1.f : -1.f;
    after_first_kernel();
    for (int64_t row = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 5); row < a.nq;
         row += (int64_t)gridDim.x * 4) {
        const RowAt at = row_at(a, row);
        Sums s = no_sums();
        for (int i = lane; i < parts; i += 32) {
            const float2* v = reinterpret_cast<const float2*>(part_at(a, row * parts + i));
            s = join(s, Sums{v[0].x, v[0].y, v[1].x}, c);
        }
        int n = 0;
        for (int b = 0; b < parts * a.k; b += 32) {
            const int i = b + lane, p = i / max(a.k, 1);
            const unsigned long long key =
                i < parts * a.k ? reinterpret_cast<const unsigned long long*>(
                                      part_at(a, row * parts + p) + 16)[i - p * a.k]
                                : kNone;
            const unsigned ball = __ballot_sync(0xffffffffu, key != kNone);
            if (key != kNone) buf[n + __popc(ball & ((1u << lane) - 1u))] = key;
            n += __popc(ball);
        }
        s = warp_join(s, c);
        const int kept = a.k > 0 ? cut<KW>(buf, n, n, a.k) : 0;
        finish_row<T>(a, row, at, s, ref_of(c, s.m), buf, kept, c, sgn, lane, 32);
        __syncwarp();
    }
}

// Parts a row: twelve units an SM are enough warps to keep the copies in flight (with
// fewer, larger ones less of the work on the best k); none shorter than two stages.
int parts_of(int64_t nq, int64_t n, bool ragged, int esize, int sms) {
    const int64_t len = ragged ? n / std::max<int64_t>(nq, 1) : n;
    const int64_t want = (12 * (int64_t)sms + nq - 1) / std::max<int64_t>(nq, 1);
    return (int)std::max<int64_t>(std::min(want, len / (2 * kStageBytes / esize)), 1);
}

// A kernel that may start before the one before it on the stream has ended.
template <class... P, class... A>
cudaError_t launch_after(void (*kernel)(P...), unsigned grid, unsigned threads, cudaStream_t st,
                         A... args) {
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(grid);
    cfg.blockDim = dim3(threads);
    cfg.stream = st;
    cudaLaunchAttribute early{};
    early.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    early.val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = &early;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, kernel, args...);
}

template <class T, int KW>
cudaError_t launch_kw(const ProbsArgs& a, int parts, int sms, cudaStream_t st) {
    constexpr int smem = (int)sizeof(WarpShared<KW>) * warps_of(KW) + 128;
    static_assert(smem <= 227 * 1024, "shared memory of a CTA");
    static std::atomic<uint64_t> set{0};  // a bit a device
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    const uint64_t bit = dev < 64 ? uint64_t(1) << dev : 0;
    if (!(set.load() & bit)) {
        e = cudaFuncSetAttribute(score_probs_kernel<T, KW>,
                                 cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
        if (e != cudaSuccess) return e;
        set |= bit;
    }
    const unsigned grid = (unsigned)std::min<int64_t>(a.nq * parts, sms);
    score_probs_kernel<T, KW><<<grid, warps_of(KW) * 32, smem, st>>>(a, parts);
    e = cudaGetLastError();
    if (e != cudaSuccess || parts == 1) return e;
    if ((int64_t)parts * a.k <= cap_of(KW) && parts <= 256)
        return launch_after(join_few_parts_kernel<T, KW>, (unsigned)((a.nq + 3) / 4), 128, st, a,
                            parts);
    return launch_after(join_parts_kernel<T>, (unsigned)a.nq, kThreads, st, a, parts);
}

int element_size(int dtype) { return dtype == M3G_F32 ? 4 : 2; }

}  // namespace

int64_t score_probs_work(int64_t nq, int64_t n, bool ragged, int dtype, int k, int sms) {
    const int parts = parts_of(nq, n, ragged, element_size(dtype), sms);
    return parts == 1 ? 0 : nq * parts * (16 + 8 * (int64_t)k);
}

cudaError_t launch_score_probs(const ProbsArgs& a, int sms, cudaStream_t st) {
    const int parts = parts_of(a.nq, a.n, a.row_off != nullptr, element_size(a.dtype), sms);
    if (a.dtype == M3G_F32)
        return a.k <= 32 ? launch_kw<float, 1>(a, parts, sms, st)
                         : launch_kw<float, 4>(a, parts, sms, st);
    return a.k <= 32 ? launch_kw<__nv_bfloat16, 1>(a, parts, sms, st)
                     : launch_kw<__nv_bfloat16, 4>(a, parts, sms, st);
}

}  // namespace m3g
