// Products of routed experts: rows x_i times the (N, K) matrix of the expert that row i takes, y_i = W[e_i] x_i, and the
// gradients dx_i = W[e_i]^T dy_i and dW[e] = sum over e's rows of dy_i x_i^T. Sums are held in f32, each output is rounded
// once.
#include "ygg_gemm.h"
#include "ygg_ops.h"

namespace ygg {
namespace {

__device__ __forceinline__ int clamp_at(int v, int M) { return v < 0 ? 0 : v > M ? M : v; }
// the first place of expert e; of e = E: of the rows that no expert takes
__device__ __forceinline__ int first_of(const Groups &g, int e) { return e == 0 ? 0 : clamp_at(g.offsets[e], g.M); }
__device__ __forceinline__ int end_of(const Groups &g, int e) { return e == g.E ? g.M : clamp_at(g.offsets[e + 1], g.M); }
// the row of a place, or -1
__device__ __forceinline__ int row_of(const Groups &g, int place) {
    if (!g.order) return place;
    const int r = g.order[place];
    return r >= 0 && r < g.M ? r : -1;
}

// Rows are cut into tiles of kI by expert, expert e's j th tile at the slot first_of(e) / kI + e + j: no two share one (e
// takes at most n_e / kI + 1 slots, and the next expert's begin after them), so a workgroup finds its tile from the offsets
// alone. Expert E is the rows that no expert takes. At most M / kI + E + 2 slots.
struct Piece {
    int e, first, count;    // count <= 0: the slot holds nothing
};
// a wave searches 64 experts at a time
template <int kI> __device__ __forceinline__ Piece piece_at(const Groups &g, int slot) {
    const int lane = threadIdx.x & 63;
    int lo = 0, n = g.E + 1;
    while (n > 1) {
        const int step = (n + 63) / 64, e = lane * step;
        const bool before = e < n && (e == 0 || first_of(g, lo + e) / kI + lo + e <= slot);
        const int at = (63 - __builtin_clzll(__ballot(before))) * step;
        lo += at;
        n = min(step, n - at);
    }
    lo = __builtin_amdgcn_readfirstlane(lo);
    const int first = first_of(g, lo), j = slot - first / kI - lo;
    const int64_t at = first + (int64_t)j * kI;
    const int left = (int)min((int64_t)end_of(g, lo) - at, (int64_t)kI);
    return {lo, (int)at, left};
}

// out[row][o] = sum over r of in[row][r] * (TR ? w[e][r][o] : w[e][o][r]): dimensions O and R
template <class T, int FI, int FO, int WI, int WO, int kBufs, bool TR> struct RowsTile {
    static constexpr int kThreads = 64 * WI * WO, kI = 16 * FI * WI, kO = 16 * FO * WO;
    typedef Along<T, kI, kThreads, FI, true> A;
    typedef std::conditional_t<TR, Across<T, kO, kThreads>, Along<T, kO, kThreads, FO, false>> B;
    typedef Tile<T, FI, FO, WI, WO, kBufs, A, B> Tl;
    static __device__ __forceinline__ void run(char *lds, const T *in, const T *w, const Groups &g, int O, int R, T *out,
                                               int slot, int o0) {
        const Piece pc = piece_at<kI>(g, slot);
        if (pc.count <= 0) return;
        Tl tile;
        A a;
        B b;
        const T *we = w + (int64_t)pc.e * O * R;
        if (pc.e < g.E) {
            a.begin([&](int i) {
                const int row = row_of(g, pc.first + min(i, pc.count - 1));
                return in + (int64_t)max(row, 0) * R;
            });
            if constexpr (TR) b.begin(we + o0, O - o0);
            else b.begin([&](int o) { return we + (int64_t)min(o0 + o, O - 1) * R; });
        }
        const int steps = pc.e < g.E ? (R + A::kStep - 1) / A::kStep : 0;
        tile.run(a, b, lds, steps, [&](int t) {
            const int r0 = t * A::kStep;
            a.load(r0, R);
            if constexpr (TR) b.load([&](int i) {
                const int r = r0 + B::r_of(i);
                return r < R ? (int64_t)r * O : -1;
            });
            else b.load(r0, R);
        });
        tile.template each<!TR>([&](int i, int o, const typename Tl::Acc *v, auto n) {
            if (i >= pc.count || o0 + o >= O) return;
            const int row = row_of(g, pc.first + i);
            if (row >= 0) store_run<T, decltype(n)::value>(out + (int64_t)row * O + o0 + o, (const float *)v, O - o0 - o);
        });
    }
};
template <class T, int FI, int FO, int WI, int WO, int kBufs, bool TR>
__global__ __launch_bounds__(64 * WI * WO) void rows_kernel(const T *in, const T *w, Groups g, int O, int R, T *out, int cols, int band) {
    typedef RowsTile<T, FI, FO, WI, WO, kBufs, TR> K;
    __shared__ __align__(128) char lds[K::Tl::kLds];
    const Place t = place_of(tile_of(blockIdx.x, gridDim.x), gridDim.x / cols, cols, band);
    K::run(lds, in, w, g, O, R, out, t.row, t.col * K::kO);
}

// dw[e][n][k] = sum over e's rows of dy[row][n] x[row][k], a tile of (n, k)
template <class T, int FI, int FO, int WI, int WO, int kBufs>
__global__ __launch_bounds__(64 * WI * WO) void grad_w_kernel(const T *dy, const T *x, Groups g, int N, int K, T *dw, int tn,
                                                              int tk) {
    constexpr int kThreads = 64 * WI * WO, kI = 16 * FI * WI, kO = 16 * FO * WO;
    typedef Across<T, kI, kThreads> A;
    typedef Across<T, kO, kThreads> B;
    typedef Tile<T, FI, FO, WI, WO, kBufs, A, B> Tl;
    __shared__ __align__(128) char lds[Tl::kLds];
    const int t = tile_of(blockIdx.x, gridDim.x);
    const int e = t / (tn * tk), n0 = t / tk % tn * kI, k0 = t % tk * kO;
    const int first = first_of(g, e), count = max(end_of(g, e) - first, 0);
    Tl tile;
    A a;
    B b;
    a.begin(dy + n0, N - n0);
    b.begin(x + k0, K - k0);
    const int steps = (count + A::kStep - 1) / A::kStep;
    tile.run(a, b, lds, steps, [&](int s) {
        a.load([&](int i) {
            const int r = s * A::kStep + A::r_of(i), row = r < count ? row_of(g, first + r) : -1;
            return row < 0 ? -1 : (int64_t)row * N;
        });
        b.load([&](int i) {
            const int r = s * B::kStep + B::r_of(i), row = r < count ? row_of(g, first + r) : -1;
            return row < 0 ? -1 : (int64_t)row * K;
        });
    });
    T *out = dw + (int64_t)e * N * K;
    tile.template each<false>([&](int i, int o, const typename Tl::Acc *v, auto n) {
        if (n0 + i >= N || k0 + o >= K) return;
        store_run<T, decltype(n)::value>(out + (int64_t)(n0 + i) * K + k0 + o, (const float *)v, K - k0 - o);
    });
}

// The same where rows are 16-byte aligned and the operands (of w one expert's matrix) small enough for 32-bit offsets
template <class T, int FI, int FO, int WI, int WO, bool TR>
__global__ __launch_bounds__(512) void rows_turn_kernel(const T *in, const T *w, Groups g, int O, int R, T *out, int cols, int band) {
    constexpr int kI = 16 * FI * WI, kO = 16 * FO * WO;
    typedef AlongLds<T, FI, WI, true> A;
    typedef std::conditional_t<TR, AcrossLds<T, FO, WO>, AlongLds<T, FO, WO, false>> B;
    typedef TurnTile<T, FI, FO, WI, WO, A, B> Tl;
    __shared__ __align__(1024) char lds[Tl::kLds];
    const Place t = place_of(tile_of(blockIdx.x, gridDim.x), gridDim.x / cols, cols, band);
    const int o0 = t.col * kO;
    const Piece pc = piece_at<kI>(g, t.row);
    if (pc.count <= 0) return;
    Tl tile;
    A a;
    B b;
    const int bytes_r = R * (int)sizeof(T), e = min(pc.e, g.E - 1);
    const T *we = w + (int64_t)e * O * R;
    a.begin(in, (uint32_t)g.M * bytes_r, bytes_r, [&](int i) {
        return (uint32_t)max(row_of(g, pc.first + min(i, pc.count - 1)), 0) * bytes_r;
    });
    if constexpr (TR) b.begin(we, (uint32_t)O * bytes_r, o0 * (int)sizeof(T), (O - o0) * (int)sizeof(T));
    else b.begin(we, (uint32_t)O * bytes_r, bytes_r, [&](int o) { return (uint32_t)min(o0 + o, O - 1) * bytes_r; });
    tile.clear();
    tile.run(lds, pc.e < g.E ? (bytes_r + 127) / 128 : 0,
             [&](auto h, int s, uint32_t to) { a.template load<decltype(h)::value>(s, to); },
             [&](auto h, int s, uint32_t to) {
                 if constexpr (TR) b.template load<decltype(h)::value>(to, [&](int i) {
                     const int r = s * B::kStep + B::r_of(i);
                     return r < R ? (uint32_t)r * (O * (int)sizeof(T)) : kFar;
                 });
                 else b.template load<decltype(h)::value>(s, to);
             },
             [](int) {});
    tile.template each<!TR>([&](int i, int o, const typename Tl::Acc *v, auto n) {
        if (i >= pc.count || o0 + o >= O) return;
        const int row = row_of(g, pc.first + i);
        if (row >= 0) store_run<T, decltype(n)::value>(out + (int64_t)row * O + o0 + o, (const float *)v, O - o0 - o);
    });
}
constexpr int kHeld = 7168;    // rows' numbers held in LDS at a time: a multiple of every step
constexpr int kAfter = 192;    // and how far past them a step that is fetched ahead reaches
template <class T, int FI, int FO, int WI, int WO>
__global__ __launch_bounds__(512) void grad_w_turn_kernel(const T *dy, const T *x, Groups g, int N, int K, T *dw, int tn, int tk) {
    constexpr int kI = 16 * FI * WI, kO = 16 * FO * WO, kSize = sizeof(T);
    typedef AcrossLds<T, FI, WI> A;
    typedef AcrossLds<T, FO, WO> B;
    typedef TurnTile<T, FI, FO, WI, WO, A, B> Tl;
    __shared__ __align__(1024) char lds[Tl::kLds];
    __shared__ int rows[kHeld + kAfter];
    const int t = tile_of(blockIdx.x, gridDim.x);
    const int e = t / (tn * tk), n0 = t / tk % tn * kI, k0 = t % tk * kO;
    const int first = first_of(g, e), count = max(end_of(g, e) - first, 0);
    Tl tile;
    A a;
    B b;
    a.begin(dy, (uint32_t)g.M * (N * kSize), n0 * kSize, (N - n0) * kSize);
    b.begin(x, (uint32_t)g.M * (K * kSize), k0 * kSize, (K - k0) * kSize);
    tile.clear();
    for (int from = 0; from < count; from += kHeld) {
        const int some = min(count - from, kHeld);
        __syncthreads();
        for (int i = threadIdx.x; i < some + kAfter; i += 512) rows[i] = i < some ? row_of(g, first + from + i) : -1;
        __syncthreads();
        // the thread's rows of the step to be loaded next: of both operands, whose loads lie alike
        static_assert(A::kN == B::kN && A::kWide == B::kWide, "");
        int row[A::kN];
        auto at = [&](int i, uint32_t size) { return row[i] < 0 ? kFar : (uint32_t)row[i] * size; };
        tile.run(lds, (some + A::kStep - 1) / A::kStep,
                 [&](auto h, int, uint32_t to) {
                     a.template load<decltype(h)::value>(to, [&](int i) { return at(i, N * kSize); });
                 },
                 [&](auto h, int, uint32_t to) {
                     b.template load<decltype(h)::value>(to, [&](int i) { return at(i, K * kSize); });
                 },
                 [&](int s) {
#pragma unroll
                     for (int i = 0; i < A::kN; i++) row[i] = rows[s * A::kStep + A::r_of(i)];
                 });
    }
    T *out = dw + (int64_t)e * N * K;
    tile.template each<false>([&](int i, int o, const typename Tl::Acc *v, auto n) {
        if (n0 + i >= N || k0 + o >= K) return;
        store_run<T, decltype(n)::value>(out + (int64_t)(n0 + i) * K + k0 + o, (const float *)v, K - k0 - o);
    });
}

bool aligned16(const void *p, int64_t row_bytes) { return (uintptr_t)p % 16 == 0 && row_bytes % 16 == 0; }
constexpr int64_t kMostBytes = 0x78000000;   // of an operand with 32-bit offsets: kFar and a few steps stay past it

// Tiles of 256 x 256 straight to LDS pay where an expert's rows fill half of one and there are tiles for the 256 CUs: on
// 16384 x 4096 x 4096 f16 over 8 experts 416 us against 655 of the 128 x 128 tiles through registers, which take the rest.
template <class T, bool TR>
hipError_t go_rows(const void *in, const void *w, const Groups &g, int O, int R, void *out, hipStream_t st) {
    const int64_t in_row = (int64_t)R * sizeof(T), w_row = TR ? (int64_t)O * sizeof(T) : in_row;
    if constexpr (sizeof(T) == 2) {
        const int cols = (O + 255) / 256;
        const int64_t rows = (int64_t)g.M / 256 + g.E + 2;
        if (aligned16(in, in_row) && aligned16(w, w_row) && g.M * in_row < kMostBytes && O * in_row < kMostBytes &&
            g.M >= 128 * (int64_t)g.E && (rows - g.E / 2) * cols >= 256 && rows * cols <= INT32_MAX) {
            hipLaunchKernelGGL((rows_turn_kernel<T, 8, 4, 2, 4, TR>), dim3((unsigned)(rows * cols)), dim3(512), 0, st,
                               (const T *)in, (const T *)w, g, O, R, (T *)out, cols, 16);
            return hipGetLastError();
        }
    }
    constexpr int FI = 4, FO = 4, WI = 2, WO = 2, kBufs = 1, kI = 16 * FI * WI, kO = 16 * FO * WO;
    const int cols = (O + kO - 1) / kO;
    const int64_t tiles = ((int64_t)g.M / kI + g.E + 2) * cols;
    if (tiles > INT32_MAX) return hipErrorInvalidValue;
    hipLaunchKernelGGL((rows_kernel<T, FI, FO, WI, WO, kBufs, TR>), dim3((unsigned)tiles), dim3(64 * WI * WO), 0, st,
                       (const T *)in, (const T *)w, g, O, R, (T *)out, cols, 16);
    return hipGetLastError();
}
template <class T>
hipError_t go_grad_w(const void *dy, const void *x, const Groups &g, int N, int K, void *dw, hipStream_t st) {
    if constexpr (sizeof(T) == 2) {
        const int tn = (N + 255) / 256, tk = (K + 255) / 256;
        const int64_t tiles = (int64_t)g.E * tn * tk, dy_row = (int64_t)N * sizeof(T), x_row = (int64_t)K * sizeof(T);
        if (aligned16(dy, dy_row) && aligned16(x, x_row) && g.M * dy_row < kMostBytes && g.M * x_row < kMostBytes &&
            tiles >= 256 && tiles <= INT32_MAX && N >= 192 && K >= 192) {
            hipLaunchKernelGGL((grad_w_turn_kernel<T, 8, 4, 2, 4>), dim3((unsigned)tiles), dim3(512), 0, st, (const T *)dy,
                               (const T *)x, g, N, K, (T *)dw, tn, tk);
            return hipGetLastError();
        }
    }
    constexpr int FI = 4, FO = 4, WI = 2, WO = 2, kBufs = 1, kI = 16 * FI * WI, kO = 16 * FO * WO;
    const int tn = (N + kI - 1) / kI, tk = (K + kO - 1) / kO;
    const int64_t tiles = (int64_t)g.E * tn * tk;
    if (tiles > INT32_MAX) return hipErrorInvalidValue;
    hipLaunchKernelGGL((grad_w_kernel<T, FI, FO, WI, WO, kBufs>), dim3((unsigned)tiles), dim3(64 * WI * WO), 0, st,
                       (const T *)dy, (const T *)x, g, N, K, (T *)dw, tn, tk);
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
