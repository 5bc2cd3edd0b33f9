// Log-probabilities of given tokens, entropies and most likely tokens of rows of logits, and their gradient.
//
// For a row x of V logits with m = max x, n the number of entries equal to m, r = sum of exp(x_c - m) over the others
// and s = sum of exp(x_c - m) (x_c - m) over them:
//   log Z = log1p(n - 1 + r)      (Z = sum exp(x - m); without cancellation where one token holds nearly everything)
//   logp_c = (x_c - m) - log Z
//   entropy = log Z - s / Z       (two terms of the same sign)
// A row whose every entry is -inf has logp -inf and entropy 0; one with a NaN or +inf is NaN throughout.
#include "ygg_ops.h"
#include "ygg_optype.h"

namespace ygg {
namespace {

constexpr float kLog2e = 1.4426950408889634f;

__device__ __forceinline__ float exp_of(float d) { return __builtin_amdgcn_exp2f(d * kLog2e); }

// the float's order as an unsigned integer's, and a row's entry as a key: larger first, then the lower index
__device__ __forceinline__ uint32_t ordered(float v) {
    const uint32_t u = __builtin_bit_cast(uint32_t, v);
    return u ^ ((uint32_t)((int32_t)u >> 31) | 0x80000000u);
}
__device__ __forceinline__ uint64_t key_of(float v, int c) { return (uint64_t)ordered(v + 0.0f) << 32 | (uint32_t)~c; }

template <class T> __device__ T block_reduce(T v, T *tmp, T (*join)(T, T)) {
    for (int o = 32; o; o >>= 1) v = join(v, __shfl_xor(v, o));
    __syncthreads();
    if ((threadIdx.x & 63) == 0) tmp[threadIdx.x >> 6] = v;
    __syncthreads();
    T all = tmp[0];
    for (int w = 1; w < (int)blockDim.x / 64; w++) all = join(all, tmp[w]);
    return all;
}
__device__ float add_f(float a, float b) { return a + b; }
__device__ float max_f(float a, float b) { return fmaxf(a, b); }
__device__ int or_i(int a, int b) { return a | b; }
__device__ uint64_t max_u(uint64_t a, uint64_t b) { return a > b ? a : b; }

__device__ __forceinline__ int64_t target_at(const void *t, int bytes, int64_t row) {
    return bytes == 8 ? ((const int64_t *)t)[row] : ((const int32_t *)t)[row];
}

template <class T> __global__ __launch_bounds__(256) void logprobs_kernel(LogprobsArgs a) {
    __shared__ float tf[4];
    __shared__ int ti[4];
    __shared__ uint64_t tu[4];
    const int64_t row = blockIdx.x;
    const T *x = (const T *)a.x + row * a.stride;
    const int tid = threadIdx.x;
    float m = -INFINITY;
    int bad = 0;
    for (int c = tid; c < a.V; c += 256) {
        const float v = to_f32(x[c]);
        bad |= !(v < INFINITY);
        m = fmaxf(m, v);
    }
    m = block_reduce(m, tf, max_f);
    bad = block_reduce(bad, ti, or_i);
    float n = 0, r = 0, s = 0;
    for (int c = tid; c < a.V; c += 256) {
        const float d = to_f32(x[c]) - m, e = exp_of(d);
        if (d == 0) n += 1;
        else if (e > 0) r += e, s += e * d;
    }
    n = block_reduce(n, tf, add_f);
    r = block_reduce(r, tf, add_f);
    s = block_reduce(s, tf, add_f);
    const bool none = m == -INFINITY && !bad;
    const float nan = __builtin_nanf("");
    const float logz = bad ? nan : none ? 0.0f : log1pf(n - 1 + r);
    if (bad) m = nan;
    if (tid == 0) {
        a.entropy[row] = none ? 0.0f : logz - s / (n + r);
        if (a.stats) a.stats[row] = make_float2(m, logz);
        if (a.target_bytes) {
            const int64_t t = target_at(a.targets, a.target_bytes, row);
            float v = 0;
            if (t != -1) v = t < 0 || t >= a.V ? nan : none ? -INFINITY : to_f32(x[t]) - m - logz;
            a.logp[row] = v;
        }
    }
    uint64_t last = ~0ull;
    for (int k = 0; k < a.top; k++) {
        uint64_t best = 0;
        for (int c = tid; c < a.V && !bad; c += 256) {
            const float v = to_f32(x[c]);
            const uint64_t key = key_of(v, c);
            if (v > -INFINITY && key < last && key > best) best = key;
        }
        best = block_reduce(best, tu, max_u);
        last = best;
        if (tid == 0) {
            const int c = best ? (int)~(uint32_t)best : -1;
            a.top_ids[row * a.top + k] = c;
            a.top_logp[row * a.top + k] = bad ? nan : c < 0 ? -INFINITY : to_f32(x[c]) - m - logz;
        }
    }
}

// dx_c = [c = t] g - p_c (g + sum_k g_k) + sum_k [c = id_k] g_k - g_H p_c (logp_c + H), one workgroup a row
template <class T> __global__ __launch_bounds__(256) void logprobs_grad_kernel(LogprobsGradArgs a) {
    const int64_t row = blockIdx.x;
    const T *x = (const T *)a.x + row * a.stride;
    T *dx = (T *)a.dx + row * a.V;
    const float2 st = a.stats[row];
    const float H = a.entropy[row], gh = a.g_entropy ? a.g_entropy[row] : 0.0f;
    int64_t t = a.g_logp ? target_at(a.targets, a.target_bytes, row) : -1;
    float g = 0;
    if (t != -1) g = t < 0 || t >= a.V ? __builtin_nanf("") : a.g_logp[row];
    float all = g;
    if (a.g_top)
        for (int k = 0; k < a.top; k++)
            if (a.top_ids[row * a.top + k] >= 0) all += a.g_top[row * a.top + k];
    const bool none = st.x == -INFINITY;
    for (int c = threadIdx.x; c < a.V; c += 256) {
        const float lp = to_f32(x[c]) - st.x - st.y, p = exp_of(lp);
        float d = p == 0 ? 0.0f : -p * (all + gh * (lp + H));
        if (c == t) d += g;
        if (a.g_top)
            for (int k = 0; k < a.top; k++)
                if (a.top_ids[row * a.top + k] == c) d += a.g_top[row * a.top + k];
        dx[c] = from_f32<T>(none ? 0.0f : d);
    }
}

}  // namespace

int64_t logprobs_scratch(int, int64_t, int, int) { return 0; }

hipError_t launch_logprobs(int type, const LogprobsArgs &a, void *, hipStream_t st) {
    const dim3 grid((unsigned)a.rows), block(256);
    if (type == kOpF32) hipLaunchKernelGGL(logprobs_kernel<float>, grid, block, 0, st, a);
    else if (type == kOpBf16) hipLaunchKernelGGL(logprobs_kernel<bf16_t>, grid, block, 0, st, a);
    else hipLaunchKernelGGL(logprobs_kernel<f16_t>, grid, block, 0, st, a);
    return hipGetLastError();
}

hipError_t launch_logprobs_grad(int type, const LogprobsGradArgs &a, hipStream_t st) {
    const dim3 grid((unsigned)a.rows), block(256);
    if (type == kOpF32) hipLaunchKernelGGL(logprobs_grad_kernel<float>, grid, block, 0, st, a);
    else if (type == kOpBf16) hipLaunchKernelGGL(logprobs_grad_kernel<bf16_t>, grid, block, 0, st, a);
    else hipLaunchKernelGGL(logprobs_grad_kernel<f16_t>, grid, block, 0, st, a);
    return hipGetLastError();
}

}  // namespace ygg
