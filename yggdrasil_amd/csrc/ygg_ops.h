// The output head's operators: log-probabilities of given tokens (ygg_logprobs.hip), products of routed experts
// (ygg_experts.hip) and the int8 projection of float rows (ygg_int8.hip); and a recurrent block's: layer norm (ygg_norm.hip), the
// gated recurrence (ygg_gated_scan.hip), the gated projections (ygg_gated.hip) and clipping by the global norm (ygg_clip.hip).
// Every launcher is called with checked sizes.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

namespace ygg {

enum OpType { kOpF32 = 0, kOpBf16 = 1, kOpF16 = 2 };
inline int op_bytes(int type) { return type == kOpF32 ? 4 : 2; }

constexpr int kMostTop = 64;   // most alternatives of a row

// Workgroups that a launch takes: it holds less than 2^32 threads along a dimension. Rows of logits past that go in several
// launches, a product's sizes that make more are refused with kTooLarge (HIP's own answer to such a launch).
constexpr int64_t most_blocks(int threads) { return UINT32_MAX / (uint32_t)threads; }
constexpr hipError_t kTooLarge = hipErrorInvalidConfiguration;

struct LogprobsArgs {
    const void *x;             // rows of V logits, `stride` values apart
    int64_t rows, stride;
    int V, top, target_bytes;  // target_bytes: 4, 8, or 0 without targets
    const void *targets;
    float *logp, *entropy, *top_logp;
    int32_t *top_ids;
    float2 *stats;             // a row's maximum and the log of its sum of exp(x - maximum); NULL: not kept
};
struct LogprobsGradArgs {
    const void *x;
    int64_t rows, stride;
    int V, top, target_bytes;
    const void *targets;
    const float *entropy;
    const int32_t *top_ids;
    const float2 *stats;
    const float *g_logp, *g_entropy, *g_top;   // NULL: no gradient comes from that output
    void *dx;                                  // rows of V, contiguous
};
int64_t logprobs_scratch(int type, int64_t rows, int V, int top);
hipError_t launch_logprobs(int type, const LogprobsArgs &a, void *scratch, hipStream_t stream);
hipError_t launch_logprobs_grad(int type, const LogprobsGradArgs &a, hipStream_t stream);

// M rows in the order of their experts: expert e has the places offsets[e] .. offsets[e + 1] - 1 (offsets[0] counts as
// 0), place p is row order[p] (NULL: p). Values outside [0, M] are clamped, rows outside are skipped.
struct Groups {
    const int32_t *offsets, *order;
    int M, E;
};
hipError_t launch_grouped_matmul(int type, const void *x, const void *w, const Groups &g, int N, int K, void *y,
                                 hipStream_t stream);
hipError_t launch_grouped_grad_x(int type, const void *dy, const void *w, const Groups &g, int N, int K, void *dx,
                                 hipStream_t stream);
hipError_t launch_grouped_grad_w(int type, const void *dy, const void *x, const Groups &g, int N, int K, void *dw,
                                 hipStream_t stream);

int64_t int8_scratch(int M, int N, int K);
hipError_t launch_int8_linear(int type, const void *x, const int8_t *w, const float *w_scale, int M, int N, int K, void *y,
                              void *scratch, hipStream_t stream);

struct NormArgs {
    const void *x;                // rows of n values, `stride` values apart
    int64_t rows, stride;
    int n;
    bool wide;                    // weight and bias in f32, else in x's type; NULL: ones, zeros
    const void *weight, *bias;
    float eps;
    void *y;                      // rows of n, contiguous
    float *stats;                 // a row's mean and 1 / sqrt(variance + eps); NULL: not kept
    bool past = false;            // the launcher's: results past the caches
};
struct NormGradArgs {
    const void *x;
    int64_t rows, stride;
    int n;
    bool wide;
    const void *weight;
    const float *stats;
    const void *dy;               // rows of n, contiguous, as dx is
    void *dx, *dw, *db;           // NULL: not wanted
    bool past = false;
};
int64_t norm_grad_scratch(int type, int64_t rows, int n);
bool norm_grad_wide(int n);      // rows whose own gradient wants scratch too
hipError_t launch_norm(int type, const NormArgs &a, hipStream_t stream);
hipError_t launch_norm_grad(int type, const NormGradArgs &a, void *scratch, hipStream_t stream);

// h_t = gate_t h_{t-1} + x_t over T steps of B sequences of n channels; h, dh, dx and dgate (B, T, n) are contiguous
struct ScanArgs {
    const void *gate, *x;
    int64_t gate_b, gate_t, x_b, x_t;     // values from a sequence, a step, to the next
    int64_t B, T;
    int n;
    const float *state;                   // (B, n); NULL: zeros
    void *h;
    float *last;                          // (B, n)
    float *kept;                          // what the gates' gradient wants, scan_kept bytes; NULL: nothing
    bool past = false;                    // the launcher's: results past the caches
};
struct ScanGradArgs {
    const void *gate, *x, *dh;            // dh NULL: zeros
    int64_t gate_b, gate_t, x_b, x_t;
    int64_t B, T;
    int n;
    const float *state, *dlast, *kept;    // NULL: zeros; x, state and kept are read for dgate alone
    void *dx, *dgate;                     // NULL: not wanted
    float *dstate;
    bool past = false;
};
int64_t scan_kept(int64_t B, int64_t T, int n);
int64_t scan_scratch(int type, int gate_type, int64_t B, int64_t T, int n);
hipError_t launch_scan(int type, int gate_type, const ScanArgs &a, void *scratch, hipStream_t stream);
hipError_t launch_scan_grad(int type, int gate_type, const ScanGradArgs &a, void *scratch, hipStream_t stream);

// With x (M, K) and w (2, N, K): g = x w[0]^T, u = x w[1]^T, y (M, N) = act(g) u
enum Activation { kSilu = 0, kGelu = 1, kSigmoid = 2 };
hipError_t launch_gated(int type, int act, const void *x, const void *w, int M, int N, int K, void *y, void *gu, hipStream_t stream);
int64_t gated_kept(int type, int M, int N);    // bytes of gu
int64_t gated_grad_scratch(int type, int M, int N, int K);
hipError_t launch_gated_grad(int type, int act, const void *x, const void *w, const void *gu, const void *dy, int M, int N, int K,
                             void *dx, void *dw, void *scratch, hipStream_t stream);

// The norm of `count` tensors' values together; out (NULL: the norm alone) gets them times min(1, most / norm)
int64_t clip_scratch(const int64_t *sizes, int count);
hipError_t launch_clip(const void *const *tensors, const int64_t *sizes, const int *types, int count, double most, void *const *out,
                       float *norm, void *scratch, hipStream_t stream);

}  // namespace ygg
