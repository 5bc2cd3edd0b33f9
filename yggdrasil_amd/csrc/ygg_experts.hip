// Products of routed experts: rows x_i times the (N, K) matrix of the expert that row i takes, y_i = W[e_i] x_i, and the
// gradients dx_i = W[e_i]^T dy_i and dW[e] = sum over e's rows of dy_i x_i^T. Sums are held in f32, each output is rounded
// once.
#include "ygg_ops.h"
#include "ygg_optype.h"

namespace ygg {
namespace {

__device__ __forceinline__ int clamp_at(int v, int M) { return v < 0 ? 0 : v > M ? M : v; }
__device__ __forceinline__ int first_of(const Groups &g, int e) { return e == 0 ? 0 : clamp_at(g.offsets[e], g.M); }
__device__ __forceinline__ int end_of(const Groups &g, int e) { return clamp_at(g.offsets[e + 1], g.M); }
// the row of a place, or -1
__device__ __forceinline__ int row_of(const Groups &g, int place) {
    if (!g.order) return place;
    const int r = g.order[place];
    return r >= 0 && r < g.M ? r : -1;
}
// the expert of a place: the last whose first place is at most it; -1: none takes it
__device__ __forceinline__ int expert_of(const Groups &g, int place) {
    int lo = 0, hi = g.E - 1;
    while (lo < hi) {
        const int mid = (lo + hi + 1) / 2;
        if (first_of(g, mid) <= place) lo = mid;
        else hi = mid - 1;
    }
    return place < end_of(g, lo) ? lo : -1;
}

// out[row][o] = sum over i of in[row][i] * (TR ? w[e][i][o] : w[e][o][i]), a thread an output
template <class T, bool TR>
__global__ __launch_bounds__(256) void rows_kernel(const T *in, const T *w, Groups g, int O, int I, T *out) {
    const int place = blockIdx.x, o = blockIdx.y * 256 + threadIdx.x;
    const int e = expert_of(g, place), row = row_of(g, place);
    if (o >= O || row < 0) return;
    float acc = 0;
    if (e >= 0) {
        const T *we = w + (int64_t)e * O * I;
        for (int i = 0; i < I; i++)
            acc += to_f32(in[(int64_t)row * I + i]) * to_f32(TR ? we[(int64_t)i * O + o] : we[(int64_t)o * I + i]);
    }
    out[(int64_t)row * O + o] = from_f32<T>(acc);
}

template <class T> __global__ __launch_bounds__(256) void grad_w_kernel(const T *dy, const T *x, Groups g, int N, int K, T *dw) {
    const int e = blockIdx.x, n = blockIdx.y;
    const int first = first_of(g, e), end = end_of(g, e);
    for (int k = threadIdx.x; k < K; k += 256) {
        float acc = 0;
        for (int p = first; p < end; p++) {
            const int row = row_of(g, p);
            if (row >= 0) acc += to_f32(dy[(int64_t)row * N + n]) * to_f32(x[(int64_t)row * K + k]);
        }
        dw[((int64_t)e * N + n) * K + k] = from_f32<T>(acc);
    }
}

template <class T, bool TR>
hipError_t go_rows(const void *in, const void *w, const Groups &g, int O, int I, void *out, hipStream_t st) {
    hipLaunchKernelGGL((rows_kernel<T, TR>), dim3(g.M, (O + 255) / 256), dim3(256), 0, st, (const T *)in, (const T *)w, g,
                       O, I, (T *)out);
    return hipGetLastError();
}
template <class T>
hipError_t go_grad_w(const void *dy, const void *x, const Groups &g, int N, int K, void *dw, hipStream_t st) {
    hipLaunchKernelGGL(grad_w_kernel<T>, dim3(g.E, N), dim3(256), 0, st, (const T *)dy, (const T *)x, g, N, K, (T *)dw);
    return hipGetLastError();
}

}  // namespace

hipError_t launch_grouped_matmul(int type, const void *x, const void *w, const Groups &g, int N, int K, void *y,
                                 hipStream_t st) {
    if (type == kOpF32) return go_rows<float, false>(x, w, g, N, K, y, st);
    if (type == kOpBf16) return go_rows<bf16_t, false>(x, w, g, N, K, y, st);
    return go_rows<f16_t, false>(x, w, g, N, K, y, st);
}
hipError_t launch_grouped_grad_x(int type, const void *dy, const void *w, const Groups &g, int N, int K, void *dx,
                                 hipStream_t st) {
    if (type == kOpF32) return go_rows<float, true>(dy, w, g, K, N, dx, st);
    if (type == kOpBf16) return go_rows<bf16_t, true>(dy, w, g, K, N, dx, st);
    return go_rows<f16_t, true>(dy, w, g, K, N, dx, st);
}
hipError_t launch_grouped_grad_w(int type, const void *dy, const void *x, const Groups &g, int N, int K, void *dw,
                                 hipStream_t st) {
    if (type == kOpF32) return go_grad_w<float>(dy, x, g, N, K, dw, st);
    if (type == kOpBf16) return go_grad_w<bf16_t>(dy, x, g, N, K, dw, st);
    return go_grad_w<f16_t>(dy, x, g, N, K, dw, st);
}

}  // namespace ygg
