// kernels_scores.h -- launchers of the row-score kernels (k_pack.cu, k_scores_tc.cu,
// k_probs.cu).
#pragma once

#include <cuda_runtime.h>
#include <stdint.h>

#include "m3gpu.h"

namespace m3g {

constexpr int kScaleDims = 128;  // dims that share one scale byte

// Error words of the row-score calls: a pair for an engine's enqueued calls, one for
// those that wait (one at a time), and one to which the first are taken.
enum ScoreError : int { kScoreTimeout = 0, kScoreBadItem = 1, kScoreErrWords = 2 };

// Moves a pair of words, leaving zeros: kernels that set them meanwhile lose none.
cudaError_t launch_take_score_errors(int* words, int* taken, cudaStream_t st);

// The group form's lists and pairs (all null / 0 in the dense form).
struct ScoreGroups {
    int64_t ngroup = 0, npair = 0, out_n = 0;
    const int64_t* list_off = nullptr;
    const int32_t* list_len = nullptr;
    const int64_t* pair_off = nullptr;
    const int32_t* pair_row = nullptr;
    const int64_t* out_off = nullptr;
};

cudaError_t launch_pack_rows(const void* x, int dtype, int64_t n, int dim, int64_t ldx,
                             uint8_t* codes, int64_t ld, uint8_t* scales, int64_t lds, int sms,
                             cudaStream_t st);
cudaError_t launch_row_scores(const m3g_rows& q, const m3g_rows& x, float alpha, float beta,
                              void* out, int out_dtype, int64_t ld_out, int* err, int sms,
                              cudaStream_t st);
cudaError_t launch_list_scores(const m3g_rows& q, const m3g_rows& x, const ScoreGroups& g,
                               float alpha, float beta, void* out, int out_dtype, int* err,
                               int sms, cudaStream_t st);

constexpr int kScoreMaxDim = 1 << 20;        // dims of a row
constexpr int64_t kScoreMaxGroups = 1 << 22; // lists of a call: one warp may walk them all
constexpr int kProbsMaxK = 128;
constexpr int64_t kProbsMaxRow = 0x7FFF0000;  // entries of a row: places in it are ints
int64_t score_probs_work(int64_t nq, int64_t n, bool ragged, int dtype, int k, int sms);
struct ProbsArgs {
    const void* scores;
    int dtype;
    int64_t nq, n, ld;
    const int64_t* row_off;
    float scale;
    float lowest;  // the least oriented score whose product with |scale| is not -inf
    const int64_t* given;
    int ngiven, k;
    float *lse, *entropy, *out_given;
    int64_t* top_index;
    float* top;
    void* work;
    int* err;
};
cudaError_t launch_score_probs(const ProbsArgs& a, int sms, cudaStream_t st);

}  // namespace m3g
