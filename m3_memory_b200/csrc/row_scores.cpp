// row_scores.cpp -- host side of the row-score calls: argument checks (before any
// device work), the error words, launches.
#include <cmath>
#include <limits>
#include <string>

#include "engine.h"

namespace m3g {
namespace {

bool aligned(const void* p, uintptr_t a) { return (reinterpret_cast<uintptr_t>(p) & (a - 1)) == 0; }

// Strides and sizes stay far from where bytes or 16-byte units would overflow.
constexpr int64_t kMaxLd = int64_t(1) << 36;

void check_rows(const char* who, const char* name, const m3g_rows* r) {
    const std::string at = std::string(who) + ": " + name + ": ";
    if (!r) fail(M3G_EINVAL, at + "missing");
    if (r->dtype != M3G_BF16 && r->dtype != M3G_E4M3)
        fail(M3G_EINVAL, at + "rows are bf16 or e4m3");
    if (r->n < 0 || r->dim <= 0) fail(M3G_EINVAL, at + "bad sizes");
    if (r->n > INT32_MAX) fail(M3G_EUNSUPPORTED, at + "2^31 rows or more");
    if (r->dim > kScoreMaxDim) fail(M3G_EUNSUPPORTED, at + "more than 2^20 dims");
    const int64_t esize = r->dtype == M3G_BF16 ? 2 : 1;
    if (r->ld < r->dim || r->ld > kMaxLd || (r->ld * esize) % 16 != 0)
        fail(M3G_EINVAL, at + "ld must be at least dim and a multiple of 16 bytes");
    if (r->n > 0 && (!r->data || !aligned(r->data, 16)))
        fail(M3G_EINVAL, at + "data must start on a 16-byte boundary");
    if (r->dtype == M3G_E4M3) {
        const int64_t nblk = (r->dim + kScaleDims - 1) / kScaleDims;
        if (r->ld_scales < nblk || r->ld_scales > kMaxLd || r->ld_scales % 4 != 0)
            fail(M3G_EINVAL,
                 at + "ld_scales must be a multiple of 4 and hold one scale per 128 dims");
        if (r->n > 0 && (!r->scales || !aligned(r->scales, 4)))
            fail(M3G_EINVAL, at + "scales must start on a 4-byte boundary");
    }
}

void check_pair(const char* who, const m3g_rows* q, const m3g_rows* x, int out_dtype, float alpha,
                float beta) {
    check_rows(who, "queries", q);
    check_rows(who, "rows", x);
    if (q->dtype != x->dtype || q->dim != x->dim)
        fail(M3G_EINVAL, std::string(who) + ": queries and rows differ in type or dim");
    if (out_dtype != M3G_F32 && out_dtype != M3G_BF16)
        fail(M3G_EINVAL, std::string(who) + ": scores are fp32 or bf16");
    if (!std::isfinite(alpha) || !std::isfinite(beta))
        fail(M3G_EINVAL, std::string(who) + ": alpha and beta must be finite");
}

void check_out(const char* who, const void* out, int out_dtype) {
    if (!out || !aligned(out, out_dtype == M3G_F32 ? 4 : 2))
        fail(M3G_EINVAL, std::string(who) + ": output missing or misaligned");
}

// The least t with c * t > -inf in fp32 (c > 0): -FLT_MAX, or about -FLT_MAX / c.
float lowest_score(float c) {
    const float most = std::numeric_limits<float>::max(), none = -INFINITY;
    volatile float p;  // rounded to fp32
    float t = c <= 1.f ? -most : -most / c;
    while (p = c * t, p == none) t = std::nextafter(t, 0.f);
    while (t > -most && (p = c * std::nextafter(t, none), p != none)) t = std::nextafter(t, none);
    return t;
}

// This thread's allocations and waits are allowed while a stream captures.
struct CaptureRelaxed {
    cudaStreamCaptureMode mode = cudaStreamCaptureModeRelaxed;
    CaptureRelaxed() { M3G_CK(cudaThreadExchangeStreamCaptureMode(&mode)); }
    ~CaptureRelaxed() { cudaThreadExchangeStreamCaptureMode(&mode); }
};
struct OwnStream {
    cudaStream_t st = nullptr;
    OwnStream() { M3G_CK(cudaStreamCreateWithFlags(&st, cudaStreamNonBlocking)); }
    ~OwnStream() { cudaStreamDestroy(st); }
};

void fail_on(const int* w) {
    if (w[kScoreTimeout]) fail(M3G_ETIMEOUT, "row scores: a device-side wait gave up");
    if (w[kScoreBadItem])
        fail(M3G_ERANGE, "row scores: a list, pair or row of scores out of range was left out");
}

}  // namespace

int* Engine::score_err() {
    if (int* words = score_err_.load()) return words;
    std::lock_guard lk(score_mu_);
    if (!score_err_.load()) {
        // (on a stream of its own: the call may be captured, by another stream's capture)
        CaptureRelaxed relaxed;
        DBuf<int> w;
        w.alloc(3 * kScoreErrWords);
        OwnStream st;
        M3G_CK(cudaMemsetAsync(w.p, 0, 3 * kScoreErrWords * sizeof(int), st.st));
        M3G_CK(cudaStreamSynchronize(st.st));
        score_words_.swap(w);
        score_err_ = score_words_.p;
    }
    return score_err_.load();
}

void Engine::row_score_errors() {
    int* words = score_err_.load();
    if (!words) return;
    std::lock_guard lk(score_read_mu_);
    M3G_CK(cudaDeviceSynchronize());
    int* taken = words + 2 * kScoreErrWords;
    M3G_CK(launch_take_score_errors(words, taken, cudaStreamLegacy));
    int w[kScoreErrWords];
    M3G_CK(cudaMemcpy(w, taken, sizeof(w), cudaMemcpyDeviceToHost));
    fail_on(w);
}

template <class F>
void Engine::launch_scores(cudaStream_t ext, F launch) {
    int* words = score_err();
    if (ext) {
        M3G_CK(launch(words));
        return;
    }
    std::lock_guard lk(score_wait_mu_);
    words += kScoreErrWords;
    M3G_CK(launch(words));
    M3G_CK(cudaStreamSynchronize(ext));
    int w[kScoreErrWords];
    M3G_CK(cudaMemcpy(w, words, sizeof(w), cudaMemcpyDeviceToHost));
    if (w[kScoreTimeout] || w[kScoreBadItem]) M3G_CK(cudaMemset(words, 0, sizeof(w)));
    fail_on(w);
}

void Engine::pack_rows(const void* dX, int dtype, int64_t n, int dim, int64_t ldx,
                       const m3g_rows* out, cudaStream_t ext) {
    check_rows("pack_rows", "packed rows", out);
    if (out->dtype != M3G_E4M3) fail(M3G_EINVAL, "pack_rows: rows are packed to e4m3");
    if (dtype != M3G_F32 && dtype != M3G_BF16)
        fail(M3G_EINVAL, "pack_rows: vectors are fp32 or bf16");
    if (out->n != n || out->dim != dim) fail(M3G_EINVAL, "pack_rows: n or dim differ");
    if (ldx < dim || ldx > kMaxLd) fail(M3G_EINVAL, "pack_rows: ldx must be at least dim");
    if (n == 0) return;
    if (!dX || !aligned(dX, dtype == M3G_F32 ? 4 : 2))
        fail(M3G_EINVAL, "pack_rows: vectors missing or misaligned");
    DeviceGuard g(device_);
    M3G_CK(launch_pack_rows(dX, dtype, n, dim, ldx,
                            static_cast<uint8_t*>(const_cast<void*>(out->data)), out->ld,
                            const_cast<uint8_t*>(out->scales), out->ld_scales, num_sms_, ext));
    if (!ext) M3G_CK(cudaStreamSynchronize(ext));
}

void Engine::row_scores(const m3g_rows* q, const m3g_rows* x, float alpha, float beta,
                        void* d_out, int out_dtype, int64_t ld_out, cudaStream_t ext) {
    check_pair("row_scores", q, x, out_dtype, alpha, beta);
    if (ld_out < x->n || ld_out > kMaxLd)
        fail(M3G_EINVAL, "row_scores: ld_out must be at least the number of rows");
    if (q->n == 0 || x->n == 0) return;
    check_out("row_scores", d_out, out_dtype);
    DeviceGuard g(device_);
    launch_scores(ext, [&](int* err) {
        return launch_row_scores(*q, *x, alpha, beta, d_out, out_dtype, ld_out, err, num_sms_, ext);
    });
}

void Engine::list_scores(const m3g_rows* q, const m3g_rows* x, const ScoreGroups& groups,
                         float alpha, float beta, void* d_out, int out_dtype, cudaStream_t ext) {
    check_pair("list_scores", q, x, out_dtype, alpha, beta);
    const ScoreGroups& s = groups;
    if (s.ngroup < 0 || s.npair < 0 || s.out_n < 0) fail(M3G_EINVAL, "list_scores: bad sizes");
    if (s.ngroup > kScoreMaxGroups || s.npair > INT32_MAX)
        fail(M3G_EUNSUPPORTED, "list_scores: more than 2^22 lists, or 2^31 pairs");
    if (s.ngroup == 0 || s.npair == 0 || q->n == 0 || x->n == 0 || s.out_n == 0) return;
    if (!s.list_off || !s.list_len || !s.pair_off || !s.out_off)
        fail(M3G_EINVAL, "list_scores: buffers missing");
    if (!aligned(s.list_off, 8) || !aligned(s.list_len, 4) || !aligned(s.pair_off, 8) ||
        !aligned(s.out_off, 8) || !aligned(s.pair_row, 4))
        fail(M3G_EINVAL, "list_scores: misaligned buffers");
    check_out("list_scores", d_out, out_dtype);
    DeviceGuard g(device_);
    launch_scores(ext, [&](int* err) {
        return launch_list_scores(*q, *x, s, alpha, beta, d_out, out_dtype, err, num_sms_, ext);
    });
}

int64_t Engine::score_probs_work(int64_t nq, int64_t n, bool ragged, int dtype, int k) {
    if (dtype != M3G_F32 && dtype != M3G_BF16)
        fail(M3G_EINVAL, "score_probs_work: scores are fp32 or bf16");
    if (nq < 0 || n < 0 || k < 0) fail(M3G_EINVAL, "score_probs_work: bad sizes");
    return m3g::score_probs_work(nq, n, ragged, dtype, k, num_sms_);
}

void Engine::score_probs(ProbsArgs a, int64_t work_bytes, cudaStream_t ext) {
    if (a.dtype != M3G_F32 && a.dtype != M3G_BF16)
        fail(M3G_EINVAL, "score_probs: scores are fp32 or bf16");
    if (a.nq < 0 || a.n < 0 || a.ngiven < 0 || a.k < 0)
        fail(M3G_EINVAL, "score_probs: bad sizes");
    if (a.k > kProbsMaxK)
        fail(M3G_EUNSUPPORTED,
             "score_probs: k > " + std::to_string(kProbsMaxK) + " is not supported");
    if (a.nq > INT32_MAX || (!a.row_off && a.n > kProbsMaxRow) || a.n > kMaxLd)
        fail(M3G_EUNSUPPORTED, "score_probs: 2^31 - 2^16 entries in a row, or 2^31 rows");
    if (!a.row_off && (a.ld < a.n || a.ld > kMaxLd))
        fail(M3G_EINVAL, "score_probs: ld must be at least n");
    if (!std::isfinite(a.scale) || a.scale == 0.f)
        fail(M3G_EINVAL, "score_probs: scale must be finite and not 0");
    if (a.nq == 0) return;
    if ((a.n > 0 && !a.scores) || !a.lse || !a.entropy ||
        (a.ngiven > 0 && (!a.given || !a.out_given)) || (a.k > 0 && (!a.top_index || !a.top)))
        fail(M3G_EINVAL, "score_probs: buffers missing");
    if (!aligned(a.scores, a.dtype == M3G_F32 ? 4 : 2) || !aligned(a.row_off, 8) ||
        !aligned(a.given, 8) || !aligned(a.top_index, 8) || !aligned(a.lse, 4) ||
        !aligned(a.entropy, 4) || !aligned(a.out_given, 4) || !aligned(a.top, 4))
        fail(M3G_EINVAL, "score_probs: misaligned buffers");
    const int64_t need = score_probs_work(a.nq, a.n, a.row_off != nullptr, a.dtype, a.k);
    if (need > 0 && (!a.work || work_bytes < need || !aligned(a.work, 8)))
        fail(M3G_EINVAL, "score_probs: work needs " + std::to_string(need) +
                             " bytes on an 8-byte boundary");
    DeviceGuard g(device_);
    a.lowest = lowest_score(std::fabs(a.scale));
    launch_scores(ext, [&](int* err) {
        a.err = err;
        return launch_score_probs(a, num_sms_, ext);
    });
}

}  // namespace m3g
