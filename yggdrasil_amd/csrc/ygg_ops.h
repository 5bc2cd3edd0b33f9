// The output head's operators: log-probabilities of given tokens (ygg_logprobs.hip), products of routed experts
// (ygg_experts.hip) and the int8 projection of float rows (ygg_int8.hip). Every launcher is called with checked sizes.
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

}  // namespace ygg
