// The int8 projection of float rows: row i is quantised with its own scale, s_i = max(max |x_i| / 127, 2^-126),
// q = x / s_i rounded to nearest with ties to even, and multiplied by an int8 matrix with a scale for each of its rows,
// y_in = (sum_k q_ik w_nk) ws_n s_i (multiplied in this order: a row's scale may be near the ends of f32's range). The integer sums are exact in 32 bits (K <= 131072). A row with a NaN or an infinity
// has a NaN scale, so it is NaN throughout.
#include "ygg_ops.h"
#include "ygg_optype.h"

namespace ygg {
namespace {

constexpr float kLeastScale = 1.17549435e-38f;   // 2^-126

// a workgroup a row: its scale, and its integers, zero from K to Kp
template <class T>
__global__ __launch_bounds__(256) void quantize_kernel(const T *x, int K, int Kp, int8_t *q, float *scale) {
    __shared__ uint32_t tmp[4];
    const int64_t row = blockIdx.x;
    x += row * K;
    q += row * Kp;
    uint32_t most = 0;    // of the magnitudes' bits, among which infinities and NaN come last
    for (int k = threadIdx.x; k < K; k += 256)
        most = max(most, __builtin_bit_cast(uint32_t, to_f32(x[k])) & 0x7fffffffu);
    for (int o = 32; o; o >>= 1) most = max(most, (uint32_t)__shfl_xor((int)most, o));
    if ((threadIdx.x & 63) == 0) tmp[threadIdx.x >> 6] = most;
    __syncthreads();
    most = max(max(tmp[0], tmp[1]), max(tmp[2], tmp[3]));
    const bool bad = most >= 0x7f800000u;
    const float s = bad ? __builtin_nanf("") : fmaxf(__builtin_bit_cast(float, most) / 127.0f, kLeastScale);
    if (threadIdx.x == 0) scale[row] = s;
    for (int k = threadIdx.x; k < Kp; k += 256)
        q[k] = k < K && !bad ? (int8_t)(int)__builtin_rintf(to_f32(x[k]) / s) : (int8_t)0;
}

template <class T>
__global__ __launch_bounds__(256) void int8_kernel(const int8_t *q, const float *scale, const int8_t *w, const float *ws,
                                                   int N, int K, int Kp, T *y) {
    const int64_t row = blockIdx.x;
    const int n = blockIdx.y * 256 + threadIdx.x;
    if (n >= N) return;
    int acc = 0;
    for (int k = 0; k < K; k++) acc += (int)q[row * Kp + k] * (int)w[(int64_t)n * K + k];
    y[row * N + n] = from_f32<T>((float)acc * ws[n] * scale[row]);
}

int padded(int K) { return (K + 127) / 128 * 128; }

template <class T>
hipError_t go(const void *x, const int8_t *w, const float *ws, int M, int N, int K, void *y, void *scratch, hipStream_t st) {
    float *scale = (float *)scratch;
    int8_t *q = (int8_t *)scratch + ((int64_t)M * 4 + 255) / 256 * 256;
    hipLaunchKernelGGL(quantize_kernel<T>, dim3(M), dim3(256), 0, st, (const T *)x, K, padded(K), q, scale);
    hipLaunchKernelGGL(int8_kernel<T>, dim3(M, (N + 255) / 256), dim3(256), 0, st, q, scale, w, ws, N, K, padded(K), (T *)y);
    return hipGetLastError();
}

}  // namespace

int64_t int8_scratch(int M, int, int K) { return ((int64_t)M * 4 + 255) / 256 * 256 + (int64_t)M * padded(K); }

hipError_t launch_int8_linear(int type, const void *x, const int8_t *w, const float *w_scale, int M, int N, int K, void *y,
                              void *scratch, hipStream_t st) {
    if (type == kOpF32) return go<float>(x, w, w_scale, M, N, K, y, scratch, st);
    if (type == kOpBf16) return go<bf16_t>(x, w, w_scale, M, N, K, y, scratch, st);
    return go<f16_t>(x, w, w_scale, M, N, K, y, scratch, st);
}

}  // namespace ygg
