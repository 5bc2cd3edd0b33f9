// The int8 projection of float rows: row i is quantised with its own scale, s_i = max(max |x_i| / 127, 2^-126),
// q = x / s_i rounded to nearest with ties to even, and multiplied by an int8 matrix with a scale for each of its rows,
// y_in = (sum_k q_ik w_nk) ws_n s_i (multiplied in this order: a row's scale may be near the ends of f32's range). The
// integer sums are exact in 32 bits (K <= 131072). A row with a NaN or an infinity has a NaN scale, so it is NaN throughout.
#include <algorithm>

#include "../../include/ygg_hip.h"
#include "ygg_gemm.h"
#include "ygg_ops.h"

namespace ygg {
namespace {

constexpr float kLeastScale = 1.17549435e-38f;   // 2^-126

// the largest magnitude of 16 bytes as bits, among which infinities and NaN come last
template <class T> __device__ __forceinline__ uint32_t most_of(u32x4 v) {
    constexpr int kE = 16 / sizeof(T);
    float f[kE];
    unpack(v, f, T{});
    uint32_t most = 0;
#pragma unroll
    for (int j = 0; j < kE; j++) most = max(most, __builtin_bit_cast(uint32_t, f[j]) & 0x7fffffffu);
    return most;
}
__device__ __forceinline__ float scale_of(uint32_t most) {
    return most >= 0x7f800000u ? __builtin_nanf("") : fmaxf(__builtin_bit_cast(float, most) / 127.0f, kLeastScale);
}
// the integers of 16 bytes; a NaN scale makes them 0
template <class T> __device__ __forceinline__ void put_integers(u32x4 v, float s, int8_t *q) {
    constexpr int kE = 16 / sizeof(T);
    float f[kE];
    unpack(v, f, T{});
    uint32_t out[kE / 4] = {};
#pragma unroll
    for (int j = 0; j < kE; j++) {
        const float r = s == s ? __builtin_rintf(f[j] / s) : 0.0f;
        out[j / 4] |= ((uint32_t)(int)r & 0xffu) << 8 * (j % 4);
    }
    __builtin_memcpy(__builtin_assume_aligned(q, kE), out, kE);
}
// piece i of a row of K values (16 bytes; what is past the row is zero)
template <class T> __device__ __forceinline__ u32x4 piece(const T *x, int K, int i) {
    constexpr int kE = 16 / sizeof(T);
    return K >= kE ? load16_end(x + i * kE, K - i * kE) : load16(x + min(i * kE, K - 1), K - i * kE);
}

// a workgroup a row: its scale, and its integers, zero from K to Kp. Up to kHold pieces of 16 bytes a thread stay in
// registers; longer rows are read twice. 8192 rows of 4096 bf16: 28 us, 3.6 TB/s, the VALU 84% busy.
template <class T> __global__ __launch_bounds__(256) void quantize_kernel(const T *x, int K, int Kp, int8_t *q, float *scale) {
    constexpr int kE = 16 / sizeof(T), kHold = 4;
    __shared__ uint32_t tmp[4];
    const int64_t row = blockIdx.x;
    const int tid = threadIdx.x, pieces = Kp / kE;
    x += row * K;
    q += row * Kp;
    u32x4 v[kHold];
    uint32_t most = 0;
#pragma unroll
    for (int u = 0; u < kHold; u++) v[u] = piece(x, K, min(tid + u * 256, pieces - 1));
#pragma unroll
    for (int u = 0; u < kHold; u++) most = max(most, most_of<T>(v[u]));
    for (int i = tid + kHold * 256; i < pieces; i += 256) most = max(most, most_of<T>(piece(x, K, i)));
    for (int o = 32; o; o >>= 1) most = max(most, (uint32_t)__shfl_xor((int)most, o));
    if ((tid & 63) == 0) tmp[tid >> 6] = most;
    __syncthreads();
    const float s = scale_of(max(max(tmp[0], tmp[1]), max(tmp[2], tmp[3])));
    if (tid == 0) scale[row] = s;
#pragma unroll
    for (int u = 0; u < kHold; u++)
        if (tid + u * 256 < pieces) put_integers<T>(v[u], s, q + (tid + u * 256) * kE);
    for (int i = tid + kHold * 256; i < pieces; i += 256) put_integers<T>(piece(x, K, i), s, q + i * kE);
}

// Few rows: 16 FI of them by 16 of w's rows a workgroup, whose 4 waves take a quarter of K each, w straight from memory with
// 8 pieces in flight a lane. kFused (FI 1): the rows are quantised here, by every workgroup, while its first pieces of w are
// on their way: one launch, and x is small beside w.
constexpr int kFusedBytes = 24576, kFusedPieces = 8;
int padded(int K) { return (K + 127) / 128 * 128; }
template <class T> bool fits_fused(int M, int K) {
    int rows = 1;
    while (rows < M) rows *= 2;
    return rows <= 8 && M * (padded(K) + 16) <= kFusedBytes && padded(K) / (int)(16 / sizeof(T)) <= kFusedPieces * (256 / rows);
}
template <class T, int FI, bool kFused>
__global__ __launch_bounds__(256) void few_int8_kernel(const T *x, const int8_t *q, const float *scale, const int8_t *w, const float *ws,
                                                       int M, int N, int K, int Kp, T *y, int cols) {
    constexpr int kU = 8, kE = 16 / sizeof(T);
    __shared__ i32x4 parts[4][FI][64];
    __shared__ __align__(16) int8_t mine[kFused ? kFusedBytes : 16];
    __shared__ uint32_t tmp[4];
    __shared__ float scales[16];
    const int t = tile_of(blockIdx.x, gridDim.x), o0 = t % cols * 16, i0 = t / cols * 16 * FI;
    const int tid = threadIdx.x, l = tid & 63, wave = tid >> 6, d = l & 15, g = l >> 4;
    const int steps = (K + 63) / 64, per = (steps + 3) / 4, begin = min(per * wave, steps), end = min(begin + per, steps);
    const int8_t *wp = w + (int64_t)min(o0 + d, N - 1) * K + g * 16;
    const int last = K - g * 16;
    // K >= 16; past the wave's part: of the row, and multiplied by zeros
    auto load_w = [&](u32x4 *a, int s) {
        if (s + kU <= end && (s + kU) * 64 <= K) {
#pragma unroll
            for (int u = 0; u < kU; u++) a[u] = load16(wp + (s + u) * 64);
        } else {
#pragma unroll
            for (int u = 0; u < kU; u++) a[u] = load16_end(wp + min(s + u, steps - 1) * 64, last - min(s + u, steps - 1) * 64);
        }
    };
    u32x4 a[kU];
    i32x4 acc[FI];
#pragma unroll
    for (int i = 0; i < FI; i++) acc[i] = i32x4{0, 0, 0, 0};
    const int8_t *from[FI];
    if constexpr (kFused) {
        int rows = 1;
        while (rows < M) rows *= 2;
        const int threads = 256 / rows, r = tid / threads, at = tid % threads, pieces = Kp / kE;
        const T *xr = x + (int64_t)min(r, M - 1) * K;
        u32x4 v[kFusedPieces];
#pragma unroll
        for (int u = 0; u < kFusedPieces; u++)
            if (u * threads < pieces) v[u] = piece(xr, K, min(at + u * threads, pieces - 1));
        load_w(a, begin);
        uint32_t most = 0;
#pragma unroll
        for (int u = 0; u < kFusedPieces; u++)
            if (u * threads < pieces) most = max(most, most_of<T>(v[u]));
        for (int o = min(threads, 64) / 2; o; o >>= 1) most = max(most, (uint32_t)__shfl_xor((int)most, o));
        if (l == 0) tmp[wave] = most;
        __syncthreads();
        if (threads == 128) most = max(tmp[wave & 2], tmp[wave | 1]);
        if (threads == 256) most = max(max(tmp[0], tmp[1]), max(tmp[2], tmp[3]));
        const float s = scale_of(most);
        if (r < M) {
            if (at == 0) scales[r] = s;
#pragma unroll
            for (int u = 0; u < kFusedPieces; u++)
                if (at + u * threads < pieces) put_integers<T>(v[u], s, mine + r * (Kp + 16) + (at + u * threads) * kE);
        }
        __syncthreads();
        from[0] = mine + min(d, M - 1) * (Kp + 16) + g * 16;
    } else {
        load_w(a, begin);
#pragma unroll
        for (int i = 0; i < FI; i++) from[i] = q + (int64_t)min(i0 + 16 * i + d, M - 1) * Kp + g * 16;
    }
    for (int s = begin; s < end; s += kU) {
        u32x4 now[kU];
#pragma unroll
        for (int u = 0; u < kU; u++) now[u] = a[u];
        if (s + kU < end) load_w(a, s + kU);
#pragma unroll
        for (int i = 0; i < FI; i++) {
            u32x4 b[kU];
#pragma unroll
            for (int u = 0; u < kU; u++) b[u] = *(const u32x4 *)(from[i] + min(s + u, steps - 1) * 64);
#pragma unroll
            for (int u = 0; u < kU; u++)
                acc[i] = Mma<int8_t>::run(now[u], s + u < end ? b[u] : u32x4{0, 0, 0, 0}, acc[i]);
        }
    }
#pragma unroll
    for (int i = 0; i < FI; i++) parts[wave][i][l] = acc[i];
    __syncthreads();
    for (int i = wave; i < FI; i += 4) {
        const i32x4 v = parts[0][i][l] + parts[1][i][l] + parts[2][i][l] + parts[3][i][l];
        const int row = i0 + 16 * i + d, col = o0 + 4 * g;
        if (row >= M || col >= N) continue;
        const float sr = kFused ? scales[row] : scale[row];
        float f[4];
#pragma unroll
        for (int j = 0; j < 4; j++) f[j] = (float)v[j] * ws[min(col + j, N - 1)] * sr;
        store_run<T, 4>(y + (int64_t)row * N + col, f, N - col);
    }
}

// A tile of rows and w's rows: the integers' products on the matrix cores, then a row's and a column's scale
template <class T, int FI, int FO, int WI, int WO>
__global__ __launch_bounds__(64 * WI * WO) void int8_kernel(const int8_t *q, const float *scale, const int8_t *w, const float *ws,
                                                            int M, int N, int K, int Kp, T *y, int cols, int band) {
    constexpr int kThreads = 64 * WI * WO, kI = 16 * FI * WI, kO = 16 * FO * WO;
    typedef Along<int8_t, kI, kThreads, FI, true> A;
    typedef Along<int8_t, kO, kThreads, FO, false> B;
    typedef Tile<int8_t, FI, FO, WI, WO, A, B> Tl;
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

template <class T>
hipError_t go(const void *x, const int8_t *w, const float *ws, int M, int N, int K, void *y, void *scratch, hipStream_t st) {
    float *scale = (float *)scratch;
    int8_t *q = (int8_t *)scratch + ((int64_t)M * 4 + 255) / 256 * 256;
    auto few = [&](auto fi, auto fused) {
        constexpr int FI = decltype(fi)::value;
        const int cols = (N + 15) / 16;
        const int64_t tiles = (int64_t)((M + 16 * FI - 1) / (16 * FI)) * cols;
        if (tiles > most_blocks(256)) return kTooLarge;
        hipLaunchKernelGGL((few_int8_kernel<T, FI, decltype(fused)::value>), dim3((unsigned)tiles), dim3(256), 0, st, (const T *)x,
                           q, scale, w, ws, M, N, K, padded(K), (T *)y, cols);
        return hipGetLastError();
    };
    using std::integral_constant;
    if (K >= 16 && fits_fused<T>(M, K)) return few(integral_constant<int, 1>(), std::true_type());
    const int half = YGG_MOST_ROWS / 2;     // 2^32 threads are too many for a launch
    for (int i = 0; i < M; i += half)
        hipLaunchKernelGGL(quantize_kernel<T>, dim3(std::min(M - i, half)), dim3(256), 0, st, (const T *)x + (int64_t)i * K, K,
                           padded(K), q + (int64_t)i * padded(K), scale + i);
    // w is read once for 16 or 32 rows, by four waves a workgroup; more rows, or a short K, go by tiles (8192 x 4096: 16 rows
    // 10 us for 20, 32 rows 14 for 20, 64 rows 25 for 21), but where there are few of those (77 rows, 1000 x 4096: 8 for 17)
    const int64_t tiles64 = (int64_t)((M + 63) / 64) * ((N + 63) / 64);
    if (K >= 16 && M <= 16) return few(integral_constant<int, 1>(), std::false_type());
    if ((K >= 1024 && M <= 32) || (K >= 2048 && tiles64 < 64)) return few(integral_constant<int, 2>(), std::false_type());
    // tiles of 256 x 256 straight to LDS where there are enough of them: 8192 x 4096 x 8192 259 us a call against 391
    const int64_t big = (int64_t)((M + 255) / 256) * ((N + 255) / 256);
    if (K % 16 == 0 && (uintptr_t)w % 16 == 0 && (int64_t)M * padded(K) < 0x78000000 && (int64_t)N * K < 0x78000000 && big >= 256 &&
        big <= most_blocks(512)) {
        hipLaunchKernelGGL((int8_turn_kernel<T, 8, 4, 2, 4>), dim3((unsigned)big), dim3(512), 0, st, q, scale, w, ws, M, N, K,
                           padded(K), (T *)y, (N + 255) / 256, 16);
        return hipGetLastError();
    }
    auto tiles = [&](auto fi, auto wo) {
        constexpr int FI = decltype(fi)::value, WO = decltype(wo)::value, kI = 32 * FI, kO = 64 * WO;
        const int cols = (N + kO - 1) / kO;
        const int64_t tiles = (int64_t)((M + kI - 1) / kI) * cols;
        if (tiles > most_blocks(128 * WO)) return kTooLarge;
        hipLaunchKernelGGL((int8_kernel<T, FI, 4, 2, WO>), dim3((unsigned)tiles), dim3(128 * WO), 0, st, q, scale, w, ws, M, N, K,
                           padded(K), (T *)y, cols, 16);
        return hipGetLastError();
    };
    // smaller tiles where there are few (512 x 4096 x 8192: 64 x 64 33 us, 64 x 128 30, 128 x 128 33; 77 x 1000 x 5003: 8, 10, 13)
    if (tiles64 <= 512) return tiles(integral_constant<int, 2>(), integral_constant<int, 1>());
    if (tiles64 <= 2048) return tiles(integral_constant<int, 2>(), integral_constant<int, 2>());
    return tiles(integral_constant<int, 4>(), integral_constant<int, 2>());
}

}  // namespace

int64_t int8_scratch(int M, int, int K) {
    if (K >= 16 && fits_fused<float>(M, K)) return 0;    // then every type does
    return ((int64_t)M * 4 + 255) / 256 * 256 + (int64_t)M * padded(K);
}

hipError_t launch_int8_linear(int type, const void *x, const int8_t *w, const float *w_scale, int M, int N, int K, void *y,
                              void *scratch, hipStream_t st) {
    if (type == kOpF32) return go<float>(x, w, w_scale, M, N, K, y, scratch, st);
    if (type == kOpBf16) return go<bf16_t>(x, w, w_scale, M, N, K, y, scratch, st);
    return go<f16_t>(x, w, w_scale, M, N, K, y, scratch, st);
}

}  // namespace ygg
