// sc_train.hpp -- launch interface of the training kernels over a mined
// sample matrix (sc_lr.hip: weak-learner responses, their gradient and the
// logistic loss; sc_sample.hip: draws from scores).
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>

namespace sc {

constexpr int kDesc = 32;  // values per descriptor (CalcFeature's 4 cells x 8 channels)

struct LrArgs {
    // sample matrix: sample i, patch p at x + i*ld + 32*p (elements)
    const void *x;
    long long ld;
    int n, n_patches, dtype;
    const int *rows;  // row r reads sample rows[r] (NULL: sample r); out of range: absent
    int R;
    // weak learners: m of them, h parameter sets each
    int M, H;
    const int *patch;  // NULL: learner m reads patch m; out of range: absent
    const float *w, *b;
    int act;
    float alpha, beta;
    // response
    const float *res;
    int res_kind;
    long long res_ld;
    float *y;
    long long y_ld;
    // gradient of a response
    const float *dy;
    long long dy_ld;
    float *dres;
    long long dres_ld;
    // loss
    const float *target, *weight;  // by sample; weight NULL: 1
    // gradient / loss outputs
    float *dw, *db, *loss;
    float *part;        // partial sums per row chunk (NULL: one chunk, results written directly)
    double *acc;        // sums over the launches so far (NULL: one launch)
    int row0;           // first row of a launch
    int chunks;         // its row chunks (grid y)
    int rows_per_wave;  // rows a wave walks
};

constexpr int kPartWords = kDesc + 2;  // per learner and set: dW, db, loss

// The launch shape of the gradient / loss kernels: the rows in `chunks`, of
// which a launch has `at_once`.  Workspace: acc, then part.
struct LrPlan {
    int chunks, at_once, rows_per_wave;
    size_t acc_bytes, part_bytes;
};
LrPlan lr_plan(const LrArgs &a);

void launch_lr_response(const LrArgs &a, hipStream_t s);
// sums per chunk, their join, and dres (acc, part and the launch shape from the plan)
void launch_lr_grad(const LrArgs &a, const LrPlan &p, void *ws, bool loss, hipStream_t s);

struct SampleArgs {
    const void *scores;
    int dtype, B, V;
    long long ld;
    const int *lens;  // NULL: V each; clamped to [0, V]
    double temperature, top_p, min_p;
    int top_k;
    int shift;  // a weight of 1 is 2^shift units of mass (sample_shift; rows of one workgroup)
    const double *u;
    int S;
    long long u_ld;
    int *index;
    long long index_ld;
    int *kept;  // may be NULL
    void *ws;   // sample_plan's bytes (NULL: none)
};

// the launch shape of the draws, from their sizes and trims; the most that any
// trims need without one (temperature above 0, top_k 0)
struct SamplePlan {
    size_t ws_bytes;
};
SamplePlan sample_plan(const SampleArgs &a);

constexpr int kMaxPool = 1 << 26;

// Masses are 64-bit integers, so that sums do not depend on their order: a
// weight w in [0, 1] is rint(w * 2^shift), with sums below 2^62 and a shift of 51
// at most (a double's mantissa).  Rows of one workgroup, 32768 scores at most, take
// the largest that V weights of 1 leave room for; longer ones (many workgroups)
// measure their own sum of weights first.
inline int sample_shift(int V) {
    int lg = 0;
    while ((1 << lg) < V) lg++;
    return 62 - lg < 51 ? 62 - lg : 51;
}

void launch_sample(const SampleArgs &a, hipStream_t s);

}  // namespace sc
