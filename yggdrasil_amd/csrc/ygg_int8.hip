// The int8 projection of float rows: row i is quantised with its own scale, s_i = max(max |x_i| / 127, 2^-126),
// q = x / s_i rounded to nearest with ties to even, and multiplied by an int8 matrix with a scale for each of its rows,
// y_in = (sum_k q_ik w_nk) ws_n s_i (multiplied in this order: a row's scale may be near the ends of f32's range). The
// integer sums are exact in 32 bits (K <= 131072). A row with a NaN or an infinity has a NaN scale, so it is NaN throughout.
#include "ygg_gemm.h"
#include "ygg_ops.h"

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

// A tile of rows and w's rows: the integers' products on the matrix cores, then a row's and a column's scale
template <class T, int FI, int FO, int WI, int WO, int kBufs>
__global__ __launch_bounds__(64 * WI * WO) void int8_kernel(const int8_t *q, const float *scale, const int8_t *w, const float *ws,
                                                            int M, int N, int K, int Kp, T *y, int cols, int band) {
    constexpr int kThreads = 64 * WI * WO, kI = 16 * FI * WI, kO = 16 * FO * WO;
    typedef Along<int8_t, kI, kThreads, FI, true> A;
    typedef Along<int8_t, kO, kThreads, FO, false> B;
    typedef Tile<int8_t, FI, FO, WI, WO, kBufs, A, B> Tl;
    __shared__ __align__(128) char lds[Tl::kLds];
    const Place t = place_of(tile_of(blockIdx.x, gridDim.x), gridDim.x / cols, cols, band);
    const int i0 = t.row * kI, o0 = t.col * kO;
    Tl tile;
    A a;
    B b;
    a.begin([&](int i) { return q + (int64_t)min(i0 + i, M - 1) * Kp; });
    b.begin([&](int o) { return w + (int64_t)min(o0 + o, N - 1) * K; });
    tile.run(a, b, lds, (K + 127) / 128, [&](int s) {
        a.load(s * 128, Kp);
        b.load(s * 128, K);
    });
    tile.template each<true>([&](int i, int o, const i32x4 *v, auto n) {
        constexpr int kN = decltype(n)::value;
        const int row = i0 + i, col = o0 + o;
        if (row >= M || col >= N) return;
        const float s = scale[row];
        float f[kN];
#pragma unroll
        for (int j = 0; j < kN; j++) f[j] = (float)v[j / 4][j % 4] * ws[min(col + j, N - 1)] * s;
        store_run<T, kN>(y + (int64_t)row * N + col, f, N - col);
    });
}

// The same where K is a multiple of 16 and the integers of x and of w have less than 2 GiB
template <class T, int FI, int FO, int WI, int WO>
__global__ __launch_bounds__(512) void int8_turn_kernel(const int8_t *q, const float *scale, const int8_t *w, const float *ws, int M,
                                                        int N, int K, int Kp, T *y, int cols, int band) {
    constexpr int kI = 16 * FI * WI, kO = 16 * FO * WO;
    typedef AlongLds<int8_t, FI, WI, true> A;
    typedef AlongLds<int8_t, FO, WO, false> B;
    typedef TurnTile<int8_t, FI, FO, WI, WO, A, B> Tl;
    __shared__ __align__(1024) char lds[Tl::kLds];
    const Place t = place_of(tile_of(blockIdx.x, gridDim.x), gridDim.x / cols, cols, band);
    const int i0 = t.row * kI, o0 = t.col * kO;
    Tl tile;
    A a;
    B b;
    a.begin(q, (uint32_t)M * Kp, Kp, [&](int i) { return (uint32_t)min(i0 + i, M - 1) * Kp; });
    b.begin(w, (uint32_t)N * K, K, [&](int o) { return (uint32_t)min(o0 + o, N - 1) * K; });
    tile.clear();
    tile.run(lds, (K + 127) / 128, [&](auto h, int s, uint32_t to) { a.template load<decltype(h)::value>(s, to); },
             [&](auto h, int s, uint32_t to) { b.template load<decltype(h)::value>(s, to); }, [](int) {});
    tile.template each<true>([&](int i, int o, const i32x4 *v, auto n) {
        constexpr int kN = decltype(n)::value;
        const int row = i0 + i, col = o0 + o;
        if (row >= M || col >= N) return;
        const float s = scale[row];
        float f[kN];
#pragma unroll
        for (int j = 0; j < kN; j++) f[j] = (float)v[j / 4][j % 4] * ws[min(col + j, N - 1)] * s;
        store_run<T, kN>(y + (int64_t)row * N + col, f, N - col);
    });
}

int padded(int K) { return (K + 127) / 128 * 128; }

template <class T>
hipError_t go(const void *x, const int8_t *w, const float *ws, int M, int N, int K, void *y, void *scratch, hipStream_t st) {
    float *scale = (float *)scratch;
    int8_t *q = (int8_t *)scratch + ((int64_t)M * 4 + 255) / 256 * 256;
    hipLaunchKernelGGL(quantize_kernel<T>, dim3(M), dim3(256), 0, st, (const T *)x, K, padded(K), q, scale);
    // tiles of 256 x 256 straight to LDS where there are enough of them: 8192 x 4096 x 8192 228 us against 424
    const int64_t big = (int64_t)((M + 255) / 256) * ((N + 255) / 256);
    if (K % 16 == 0 && (uintptr_t)w % 16 == 0 && (int64_t)M * padded(K) < 0x78000000 && (int64_t)N * K < 0x78000000 && big >= 256 &&
        big <= INT32_MAX) {
        hipLaunchKernelGGL((int8_turn_kernel<T, 8, 4, 2, 4>), dim3((unsigned)big), dim3(512), 0, st, q, scale, w, ws, M, N, K,
                           padded(K), (T *)y, (N + 255) / 256, 16);
        return hipGetLastError();
    }
    constexpr int FI = 4, FO = 4, WI = 2, WO = 2, kBufs = 1, kI = 16 * FI * WI, kO = 16 * FO * WO;
    const int cols = (N + kO - 1) / kO;
    const int64_t tiles = (int64_t)((M + kI - 1) / kI) * cols;
    if (tiles > INT32_MAX) return hipErrorInvalidValue;
    hipLaunchKernelGGL((int8_kernel<T, FI, FO, WI, WO, kBufs>), dim3((unsigned)tiles), dim3(64 * WI * WO), 0, st, q, scale, w,
                       ws, M, N, K, padded(K), (T *)y, cols, 8);
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
