// The gated projections of a feed-forward block: with g = x Wg^T and u = x Wu^T, y = act(g) u in one kernel; and their gradients
//   dg = dy u act'(g), du = dy act(g);  dx = dg Wg + du Wu,  dWg = dg^T x, dWu = du^T x.
//
// A tile computes g and u of the same columns: a wave's 64 columns of the columns' operand are 32 rows of Wg and the 32 rows of
// Wu below them, so a lane ends up with 8 neighbouring values of g and the same 8 of u, in f32, and takes their product there. For a
// backward pass g and u are kept in the inputs' type (a rounding more in dy's factors, the size of the one that dg and du take
// to enter the matrix cores), one row of 2 N values each: dg and du are laid out alike, so that with w as (2 N, K) both
// gradients are single products, those of ygg_experts.hip with one expert that takes every row.
#include <algorithm>

#include "ygg_gemm.h"
#include "ygg_ops.h"

namespace ygg {
namespace {

// act(g) and, of the backward pass, act'(g)
template <int kAct> __device__ __forceinline__ float act_of(float g, float *slope = nullptr) {
    if constexpr (kAct == kGelu) {
        const float phi = 0.5f * (1.0f + erff(g * 0.70710678118654752f));
        if (slope) *slope = __builtin_fmaf(g, 0.3989422804014327f * expf(-0.5f * g * g), phi);
        return g * phi;
    } else {
        const float p = 1.0f / (1.0f + expf(-g));
        if constexpr (kAct == kSilu) {
            if (slope) *slope = p * __builtin_fmaf(g, 1.0f - p, 1.0f);
            return g * p;
        } else {
            if (slope) *slope = p * (1.0f - p);
            return p;
        }
    }
}
// f(an integral_constant of the activation)
template <class F> __host__ __device__ __forceinline__ auto with_act(int act, F f) {
    if (act == kSilu) return f(std::integral_constant<int, kSilu>());
    if (act == kGelu) return f(std::integral_constant<int, kGelu>());
    return f(std::integral_constant<int, kSigmoid>());
}

// the row of w of a tile's column o, the tile's outputs beginning at n0
__device__ __forceinline__ int row_of_w(int o, int n0, int N) { return (o & 32 ? N : 0) + min(n0 + (o >> 6) * 32 + (o & 31), N - 1); }

// kN neighbouring outputs of a row
template <class T, int kAct, int kN>
__device__ __forceinline__ void put_outputs(const float *g, const float *u, int row, int n, int N, T *y, T *gu) {
    float v[kN];
#pragma unroll
    for (int j = 0; j < kN; j++) v[j] = act_of<kAct>(g[j]) * u[j];
    store_run<T, kN>(y + (int64_t)row * N + n, v, N - n);
    if (gu) {
        T *p = gu + (int64_t)row * 2 * N + n;
        store_run<T, kN>(p, g, N - n);
        store_run<T, kN>(p + N, u, N - n);
    }
}
template <class T, int kAct, int FI, class Acc>
__device__ __forceinline__ void put_tile(Acc (&acc)[FI][4], int row0, int part, int M, int n0, int N, T *y, T *gu, int i0) {
    const int l = threadIdx.x & 63, n = n0 + part * 32 + 8 * (l >> 4);
    if (n >= N) return;
#pragma unroll
    for (int i = 0; i < FI; i++) {
        const int row = i0 + row0 + 16 * i + (l & 15);
        if (row < M) put_outputs<T, kAct, 8>((const float *)&acc[i][0], (const float *)&acc[i][2], row, n, N, y, gu);
    }
}

template <class T, int FI, int WI, int WO, int kAct>
__global__ __launch_bounds__(64 * WI * WO) void gated_kernel(const T *x, const T *w, int M, int N, int K, T *y, T *gu, int cols, int band) {
    constexpr int kThreads = 64 * WI * WO, kI = 16 * FI * WI, kO = 64 * WO;
    typedef Along<T, kI, kThreads, FI, true> A;
    typedef Along<T, kO, kThreads, 4, false> B;
    typedef Tile<T, FI, 4, WI, WO, A, B> Tl;
    __shared__ __align__(128) char lds[Tl::kLds];
    const Place t = place_of(tile_of(blockIdx.x, gridDim.x), gridDim.x / cols, cols, band);
    const int i0 = t.row * kI, n0 = t.col * (kO / 2);
    Tl tile;
    A a;
    B b;
    a.begin([&](int i) { return x + (int64_t)min(i0 + i, M - 1) * K; });
    b.begin([&](int o) { return w + (int64_t)row_of_w(o, n0, N) * K; });
    tile.run(a, b, lds, (K + A::kStep - 1) / A::kStep, [&](int s) {
        a.load(s * A::kStep, K);
        b.load(s * A::kStep, K);
    });
    put_tile<T, kAct>(tile.acc, Tl::row0(), Tl::col0() / 64, M, n0, N, y, gu, i0);
}

// Aligned rows, straight to LDS
template <class T, int kAct>
__global__ __launch_bounds__(512) void gated_turn_kernel(const T *x, const T *w, int M, int N, int K, T *y, T *gu, int cols, int band) {
    typedef AlongLds<T, 8, 2, true> A;
    typedef AlongLds<T, 4, 4, false> B;
    typedef TurnTile<T, 8, 4, 2, 4, A, B> Tl;
    __shared__ __align__(1024) char lds[Tl::kLds];
    const Place t = place_of(tile_of(blockIdx.x, gridDim.x), gridDim.x / cols, cols, band);
    const int i0 = t.row * 256, n0 = t.col * 128, bytes = K * (int)sizeof(T);
    Tl tile;
    A a;
    B b;
    a.begin(x, (uint32_t)M * bytes, bytes, [&](int i) { return i0 + i < M ? (uint32_t)(i0 + i) * bytes : kFar; });
    b.begin(w, 2 * (uint32_t)N * bytes, bytes, [&](int o) { return (uint32_t)row_of_w(o, n0, N) * bytes; });
    tile.clear();
    tile.run(lds, (bytes + 127) / 128, [&](auto h, int s, uint32_t to) { a.template load<decltype(h)::value>(s, to); },
             [&](auto h, int s, uint32_t to) { b.template load<decltype(h)::value>(s, to); }, [](int) {}, min(M - i0, 256));
    put_tile<T, kAct>(tile.acc, Tl::row0(), Tl::col0() / 64, M, n0, N, y, gu, i0);
}

// Few rows: 16 of them by 16 outputs a workgroup, whose kW waves take a part of K each, fragments straight from memory
template <class T, int kW, int kAct>
__global__ __launch_bounds__(64 * kW) void gated_few_kernel(const T *x, const T *w, int M, int N, int K, T *y, T *gu, int cols) {
    constexpr int kE = 16 / sizeof(T), kStep = 4 * kE, kU = 4;
    __shared__ f32x4 parts[kW][2][64];
    const int t = tile_of(blockIdx.x, gridDim.x), n0 = t % cols * 16, l = threadIdx.x & 63, wave = threadIdx.x >> 6, d = l & 15, q = l >> 4;
    const int row = t / cols * 16 + d;
    f32x4 acc[2] = {{0, 0, 0, 0}, {0, 0, 0, 0}};
    const int steps = (K + kStep - 1) / kStep, per = (steps + kW - 1) / kW, end = min(per * (wave + 1), steps);
    const T *gp = w + (int64_t)min(n0 + d, N - 1) * K + q * kE, *up = gp + (int64_t)N * K, *xp = x + (int64_t)min(row, M - 1) * K + q * kE;
    const int last = K - q * kE;
    int s = per * wave;
    for (; s + kU <= end && (s + kU) * kStep <= K; s += kU) {
        u32x4 a[kU], b[kU], c[kU];
#pragma unroll
        for (int k = 0; k < kU; k++) {
            a[k] = load16(gp + (s + k) * kStep);
            b[k] = load16(up + (s + k) * kStep);
        }
#pragma unroll
        for (int k = 0; k < kU; k++) c[k] = load16(xp + (s + k) * kStep);
#pragma unroll
        for (int k = 0; k < kU; k++) {
            acc[0] = Mma<T>::run(a[k], c[k], acc[0]);
            acc[1] = Mma<T>::run(b[k], c[k], acc[1]);
        }
    }
    for (; s < end; s++) {
        const int n = last - s * kStep;
        u32x4 a, b, c;
        if (K >= kE) {
            a = load16_end(gp + s * kStep, n);
            b = load16_end(up + s * kStep, n);
            c = load16_end(xp + s * kStep, n);
        } else {
            a = load16(gp + s * kStep, n);
            b = load16(up + s * kStep, n);
            c = load16(xp + s * kStep, n);
        }
        acc[0] = Mma<T>::run(a, c, acc[0]);
        acc[1] = Mma<T>::run(b, c, acc[1]);
    }
    parts[wave][0][l] = acc[0];
    parts[wave][1][l] = acc[1];
    __syncthreads();
    if (wave) return;
#pragma unroll
    for (int i = 1; i < kW; i++) {
        acc[0] += parts[i][0][l];
        acc[1] += parts[i][1][l];
    }
    const int n = n0 + 4 * q;
    if (row < M && n < N) put_outputs<T, kAct, 4>((const float *)&acc[0], (const float *)&acc[1], row, n, N, y, gu);
}

// dg and du of pieces of 16 bytes of dy; and the one expert's offsets
template <class T, int kAct>
__global__ __launch_bounds__(256) void gated_slope_kernel(const T *gu, const T *dy, int M, int N, T *dgu, int32_t *offsets) {
    constexpr int kE = 16 / sizeof(T);
    const int per = (N + kE - 1) / kE;
    const int64_t id = (int64_t)blockIdx.x * 256 + threadIdx.x, row = id / per;
    if (id == 0) {
        offsets[0] = 0;
        offsets[1] = M;
    }
    if (row >= M) return;
    const int n = (int)(id % per) * kE, left = N - n;
    const T *p = gu + row * 2 * N + n, *q = dy + row * N + n;
    float g[kE], u[kE], d[kE];
    unpack(load16(p, left), g, T());
    unpack(load16(p + N, left), u, T());
    unpack(load16(q, left), d, T());
#pragma unroll
    for (int j = 0; j < kE; j++) {
        float slope;
        const float a = act_of<kAct>(g[j], &slope);
        g[j] = d[j] * u[j] * slope;
        u[j] = d[j] * a;
    }
    T *out = dgu + row * 2 * N + n;
    store_run<T, kE>(out, g, left);
    store_run<T, kE>(out + N, u, left);
}

bool aligned16(const void *p, int64_t row_bytes) { return (uintptr_t)p % 16 == 0 && row_bytes % 16 == 0; }
constexpr int64_t kMostBytes = 0x78000000;   // of an operand with 32-bit offsets: kFar and a few steps stay past it
constexpr int kBand = 16;

template <class T, int kAct> hipError_t go(const void *x, const void *w, int M, int N, int K, void *y, void *gu, hipStream_t st) {
    const int64_t row = (int64_t)K * sizeof(T);
    if constexpr (sizeof(T) == 2) {
        const int cols = (N + 127) / 128;
        const int64_t tiles = ((int64_t)M + 255) / 256 * cols;
        if (aligned16(x, row) && aligned16(w, row) && M * row < kMostBytes && 2 * N * row < kMostBytes && tiles >= 256 &&
            tiles <= most_blocks(512)) {
            hipLaunchKernelGGL((gated_turn_kernel<T, kAct>), dim3((unsigned)tiles), dim3(512), 0, st, (const T *)x, (const T *)w, M, N, K,
                               (T *)y, (T *)gu, cols, kBand);
            return hipGetLastError();
        }
    }
    if (M <= 16) {
        const int cols = (N + 15) / 16;
        hipLaunchKernelGGL((gated_few_kernel<T, 4, kAct>), dim3((unsigned)cols), dim3(256), 0, st, (const T *)x, (const T *)w, M, N, K,
                           (T *)y, (T *)gu, cols);
        return hipGetLastError();
    }
    auto tiles = [&](auto fi, auto wi, auto wo) {
        constexpr int FI = decltype(fi)::value, WI = decltype(wi)::value, WO = decltype(wo)::value, kI = 16 * FI * WI;
        const int cols = (N + 32 * WO - 1) / (32 * WO);
        const int64_t all = ((int64_t)M + kI - 1) / kI * cols;
        if (all > most_blocks(64 * WI * WO)) return kTooLarge;
        hipLaunchKernelGGL((gated_kernel<T, FI, WI, WO, kAct>), dim3((unsigned)all), dim3(64 * WI * WO), 0, st, (const T *)x,
                           (const T *)w, M, N, K, (T *)y, (T *)gu, cols, kBand);
        return hipGetLastError();
    };
    constexpr std::integral_constant<int, 2> two{};
    constexpr std::integral_constant<int, 4> four{};
    const int64_t tiles128 = ((int64_t)M + 127) / 128 * ((N + 63) / 64);
    return tiles128 >= 512 ? tiles(four, two, two) : tiles(two, two, two);
}
template <class T, int kAct> hipError_t go_slope(const void *gu, const void *dy, int M, int N, void *dgu, int32_t *offsets, hipStream_t st) {
    constexpr int kE = 16 / sizeof(T);
    const int64_t blocks = std::max<int64_t>(((int64_t)M * ((N + kE - 1) / kE) + 255) / 256, 1);   // without rows for the offsets
    if (blocks > most_blocks(256)) return kTooLarge;
    hipLaunchKernelGGL((gated_slope_kernel<T, kAct>), dim3((unsigned)blocks), dim3(256), 0, st, (const T *)gu, (const T *)dy, M, N, (T *)dgu,
                       offsets);
    return hipGetLastError();
}
template <class F> hipError_t with_type(int type, F f) {
    if (type == kOpF32) return f(float());
    if (type == kOpBf16) return f(bf16_t());
    return f(f16_t());
}

}  // namespace

hipError_t launch_gated(int type, int act, const void *x, const void *w, int M, int N, int K, void *y, void *gu, hipStream_t st) {
    return with_type(type, [&](auto one) {
        return with_act(act, [&](auto k) { return go<decltype(one), decltype(k)::value>(x, w, M, N, K, y, gu, st); });
    });
}
int64_t gated_grad_scratch(int type, int M, int N, int) { return 256 + (int64_t)M * 2 * N * op_bytes(type); }
hipError_t launch_gated_grad(int type, int act, const void *x, const void *w, const void *gu, const void *dy, int M, int N, int K,
                             void *dx, void *dw, void *scratch, hipStream_t st) {
    int32_t *offsets = (int32_t *)scratch;
    void *dgu = (char *)scratch + 256;
    hipError_t e = with_type(type, [&](auto one) {
        return with_act(act, [&](auto k) { return go_slope<decltype(one), decltype(k)::value>(gu, dy, M, N, dgu, offsets, st); });
    });
    const Groups g = {offsets, nullptr, M, 1};
    if (e == hipSuccess && dx) e = launch_grouped_grad_x(type, dgu, w, g, 2 * N, K, dx, st);
    if (e == hipSuccess && dw) e = launch_grouped_grad_w(type, dgu, x, g, 2 * N, K, dw, st);
    return e;
}

}  // namespace ygg
