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
__global__ __launch_bounds__(64 * WI * WO) void rows_kernel(const T *in, const T *w, Groups g, int O, int R, T *out, int cols) {
    typedef RowsTile<T, FI, FO, WI, WO, kBufs, TR> K;
    __shared__ __align__(128) char lds[K::Tl::kLds];
    const int t = tile_of(blockIdx.x, gridDim.x);
    K::run(lds, in, w, g, O, R, out, t / cols, t % cols * K::kO);
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

template <class T, bool TR>
hipError_t go_rows(const void *in, const void *w, const Groups &g, int O, int R, void *out, hipStream_t st) {
    constexpr int FI = 4, FO = 4, WI = 2, WO = 2, kBufs = 1, kI = 16 * FI * WI, kO = 16 * FO * WO;
    const int cols = (O + kO - 1) / kO;
    const int64_t tiles = ((int64_t)g.M / kI + g.E + 2) * cols;
    if (tiles > INT32_MAX) return hipErrorInvalidValue;
    hipLaunchKernelGGL((rows_kernel<T, FI, FO, WI, WO, kBufs, TR>), dim3((unsigned)tiles), dim3(64 * WI * WO), 0, st,
                       (const T *)in, (const T *)w, g, O, R, (T *)out, cols);
    return hipGetLastError();
}
template <class T>
hipError_t go_grad_w(const void *dy, const void *x, const Groups &g, int N, int K, void *dw, hipStream_t st) {
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
