// Products of routed experts: rows x_i times the (N, K) matrix of the expert that row i takes, y_i = W[e_i] x_i, and the
// gradients dx_i = W[e_i]^T dy_i and dW[e] = sum over e's rows of dy_i x_i^T. Sums are held in f32, each output is rounded
// once.
#include <algorithm>

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

// The tiles by place, for fewer rows than experts: the tile that begins at this place, if one does
template <int kI> __device__ __forceinline__ Piece piece_from(const Groups &g, int place) {
    const int lane = threadIdx.x & 63;
    int lo = 0, n = g.E + 1;
    for (;;) {
        // the last step has a lane for every expert left and for the one after: the owner's ends too
        const int step = (n + 62) / 63, e = lane * step, at = lo + e;
        const int v = at == 0 ? 0 : at <= g.E ? clamp_at(g.offsets[at], g.M) : g.M;
        const int k = 63 - __builtin_clzll(__ballot(e < n && (e == 0 || v <= place)));
        if (step == 1) {
            const int first = __builtin_amdgcn_readlane(v, k), end = __builtin_amdgcn_readlane(v, k + 1);
            return {__builtin_amdgcn_readfirstlane(lo + k), place, place >= first && (place - first) % kI == 0 ? min(end - place, kI) : 0};
        }
        lo += k * step;
        n = min(step, n - k * step);
    }
}

// out[row][o] = sum over r of in[row][r] * (TR ? w[e][r][o] : w[e][o][r]): dimensions O and R
template <class T, int FI, int FO, int WI, int WO, bool TR> struct RowsTile {
    static constexpr int kThreads = 64 * WI * WO, kI = 16 * FI * WI, kO = 16 * FO * WO;
    typedef Along<T, kI, kThreads, FI, true> A;
    typedef std::conditional_t<TR, Across<T, kO, kThreads>, Along<T, kO, kThreads, FO, false>> B;
    typedef Tile<T, FI, FO, WI, WO, A, B> Tl;
    static __device__ __forceinline__ void run(char *lds, const T *in, const T *w, const Groups &g, int O, int R, T *out,
                                               const Piece &pc, int o0) {
        Tl tile;
        A a;
        B b;
        const T *we = w + (int64_t)pc.e * O * R;
        if (pc.e < g.E) {
            a.begin([&](int i) {
                const int row = row_of(g, pc.first + min(i, pc.count - 1));
                return in + (int64_t)max(row, 0) * R;
            });
            if constexpr (TR) b.begin(we, o0, O);
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
template <class T, int FI, int FO, int WI, int WO, bool TR>
__global__ __launch_bounds__(64 * WI * WO) void rows_kernel(const T *in, const T *w, Groups g, int O, int R, T *out, int cols, int band,
                                                            bool by_place) {
    typedef RowsTile<T, FI, FO, WI, WO, TR> K;
    __shared__ __align__(128) char lds[K::Tl::kLds];
    const Place t = place_of(tile_of(blockIdx.x, gridDim.x), gridDim.x / cols, cols, band);
    const Piece pc = by_place ? piece_from<K::kI>(g, t.row) : piece_at<K::kI>(g, t.row);
    if (pc.count > 0) K::run(lds, in, w, g, O, R, out, pc, t.col * K::kO);
}

// dw[e][n][k] = sum over e's rows of dy[row][n] x[row][k], a tile of (n, k)
template <class T, int FI, int FO, int WI, int WO>
__global__ __launch_bounds__(64 * WI * WO) void grad_w_kernel(const T *dy, const T *x, Groups g, int N, int K, T *dw, int tn,
                                                              int tk) {
    constexpr int kThreads = 64 * WI * WO, kI = 16 * FI * WI, kO = 16 * FO * WO;
    typedef Across<T, kI, kThreads> A;
    typedef Across<T, kO, kThreads> B;
    typedef Tile<T, FI, FO, WI, WO, A, B> Tl;
    __shared__ __align__(128) char lds[Tl::kLds];
    const int t = tile_of(blockIdx.x, gridDim.x);
    const int e = t / (tn * tk), n0 = t / tk % tn * kI, k0 = t % tk * kO;
    const int first = first_of(g, e), count = max(end_of(g, e) - first, 0);
    Tl tile;
    A a;
    B b;
    a.begin(dy, n0, N);
    b.begin(x, k0, K);
    const int steps = (count + A::kStep - 1) / A::kStep;
    // the rows of the step to be loaded next: their numbers come a step ahead
    int ra[A::kN], rb[B::kN];
    auto fetch = [&](int s) {
#pragma unroll
        for (int i = 0; i < A::kN; i++) {
            const int r = s * A::kStep + A::r_of(i);
            ra[i] = r < count ? row_of(g, first + r) : -1;
        }
#pragma unroll
        for (int i = 0; i < B::kN; i++) {
            const int r = s * B::kStep + B::r_of(i);
            rb[i] = r < count ? row_of(g, first + r) : -1;
        }
    };
    fetch(0);
    tile.run(a, b, lds, steps, [&](int s) {
        a.load([&](int i) { return ra[i] < 0 ? -1 : (int64_t)ra[i] * N; });
        b.load([&](int i) { return rb[i] < 0 ? -1 : (int64_t)rb[i] * K; });
        fetch(s + 1);
    });
    T *out = dw + (int64_t)e * N * K;
    tile.template each<false>([&](int i, int o, const typename Tl::Acc *v, auto n) {
        if (n0 + i >= N || k0 + o >= K) return;
        store_run<T, decltype(n)::value>(out + (int64_t)(n0 + i) * K + k0 + o, (const float *)v, K - k0 - o);
    });
}

// Few rows an expert: y (not its transpose) of 16 rows by 16 columns a workgroup, whose kW waves take a part of r each; the
// fragments come straight from memory, 8 of each operand in flight a lane. A row that there is not is row 0: it reaches only
// results that are not stored.
template <class T, int kW>
__global__ __launch_bounds__(64 * kW) void few_rows_kernel(const T *in, const T *w, Groups g, int O, int R, T *out, int cols,
                                                           bool by_place) {
    constexpr int kE = 16 / sizeof(T), kStep = 4 * kE, kU = 8;
    __shared__ f32x4 parts[kW][64];
    const int t = tile_of(blockIdx.x, gridDim.x), o0 = t % cols * 16;
    const int l = threadIdx.x & 63, wave = threadIdx.x >> 6, d = l & 15, q = l >> 4;
    // by place the rows' numbers need not wait for the search
    int row = by_place && t / cols + d < g.M ? row_of(g, t / cols + d) : -1;
    const Piece pc = by_place ? piece_from<16>(g, t / cols) : piece_at<16>(g, t / cols);
    if (pc.count <= 0) return;
    if (!by_place && d < pc.count) row = row_of(g, pc.first + d);
    if (d >= pc.count) row = -1;
    f32x4 acc = {0, 0, 0, 0};
    if (pc.e < g.E) {
        const int steps = (R + kStep - 1) / kStep, per = (steps + kW - 1) / kW, end = min(per * (wave + 1), steps);
        const T *wp = w + ((int64_t)pc.e * O + min(o0 + d, O - 1)) * R + q * kE, *xp = in + (int64_t)max(row, 0) * R + q * kE;
        const int last = R - q * kE;
        int s = per * wave;
        for (; s + kU <= end && (s + kU) * kStep <= R; s += kU) {
            u32x4 a[kU], b[kU];
#pragma unroll
            for (int u = 0; u < kU; u++) a[u] = load16(wp + (s + u) * kStep);
#pragma unroll
            for (int u = 0; u < kU; u++) b[u] = load16(xp + (s + u) * kStep);
#pragma unroll
            for (int u = 0; u < kU; u++) acc = Mma<T>::run(a[u], b[u], acc);
        }
        for (; s < end && R >= kE; s += 4) {
            u32x4 a[4], b[4];
#pragma unroll
            for (int u = 0; u < 4; u++) a[u] = load16_end(wp + (s + u) * kStep, last - (s + u) * kStep);
#pragma unroll
            for (int u = 0; u < 4; u++) b[u] = load16_end(xp + (s + u) * kStep, last - (s + u) * kStep);
#pragma unroll
            for (int u = 0; u < 4; u++)
                if (s + u >= end) a[u] = b[u] = u32x4{0, 0, 0, 0};
#pragma unroll
            for (int u = 0; u < 4; u++) acc = Mma<T>::run(a[u], b[u], acc);
        }
        for (; s < end; s++) {
            const int n = last - s * kStep;
            const u32x4 a = load16(wp + s * kStep, n), b = load16(xp + s * kStep, row >= 0 ? n : 0);
            acc = Mma<T>::run(a, b, acc);
        }
    }
    if constexpr (kW > 1) {
        parts[wave][l] = acc;
        __syncthreads();
        if (wave) return;
#pragma unroll
        for (int i = 1; i < kW; i++) acc += parts[i][l];
    }
    const int o = o0 + 4 * q;
    if (row >= 0 && o < O) store_run<T, 4>(out + (int64_t)row * O + o, (const float *)&acc, O - o);
}

// kF consecutive values, p being n before its row's end; those past it come as zero. Rows of kF or more (inner: n >= kF).
template <class T, int kF> __device__ __forceinline__ void load_few(const T *p, int n, bool inner, float *f) {
    T t[kF];
    if (inner) {
        __builtin_memcpy(t, p, sizeof(t));
#pragma unroll
        for (int j = 0; j < kF; j++) f[j] = to_f32(t[j]);
    } else {
        __builtin_memcpy(t, p + min(n - kF, 0), sizeof(t));
        const int by = max(kF - n, 0);
#pragma unroll
        for (int j = 0; j < kF; j++) {
            f[j] = 0.0f;
#pragma unroll
            for (int i = j; i < kF; i++) f[j] = i - j == by ? to_f32(t[i]) : f[j];
        }
    }
}

// dw of small matrices, in f32 products whatever the type (they are few; 16-bit values are exact in f32): a workgroup of 4
// waves takes 16 FN x 64 of one expert's (n, k), a wave every fourth 16 rows, straight from memory: lane (q, d) holds values
// FN d .. of dy and 4 d .. of x at the rows 4 j + q, so instruction j multiplies row 4 j + q's, and fragment f's d th n is
// FN d + f. kDepth blocks of 16 rows are in flight a wave. The waves' sums are joined in their order.
template <class T, int FN, int kDepth>
__device__ __forceinline__ void grad_w_small(f32x4 (*parts)[4][64], const T *dy, const T *x, const Groups &g, int N, int K, T *out,
                                             int first, int count, int n0, int k0) {
    const int l = threadIdx.x & 63, d = l & 15, q = l >> 4, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
    auto put = [&](int n, const float *v) {
        const int k = k0 + 4 * d;
        if (n < N && k < K) store_run<T, 4>(out + (int64_t)n * K + k, v, K - k);
    };
    if (count <= 0) {
        const float zero[4] = {};
        for (int n = n0 + (threadIdx.x >> 4); n < n0 + 16 * FN; n += 16) put(n, zero);
        return;
    }
    if (count <= 16 && wave) return;
    const int nn = N - n0 - FN * d, nk = K - k0 - 4 * d;
    const T *dyp = dy + n0 + FN * d, *xp = x + k0 + 4 * d;
    const bool in_n = n0 + 16 * FN <= N, in_k = k0 + 64 <= K;
    f32x4 acc[FN][4];
#pragma unroll
    for (int i = 0; i < FN; i++)
#pragma unroll
        for (int o = 0; o < 4; o++) acc[i][o] = f32x4{0, 0, 0, 0};
    // blocks in flight, and the rows' numbers of those to be loaded in their place
    struct {
        int row[4];
        bool none[4];
        float a[4][FN], b[4][4];
    } in[kDepth];
    auto rows = [&](int h, int at) {
#pragma unroll
        for (int j = 0; j < 4; j++) in[h].row[j] = at + 4 * j + q < count ? row_of(g, first + at + 4 * j + q) : -1;
    };
    auto load = [&](int h) {
#pragma unroll
        for (int j = 0; j < 4; j++) {
            const int row = in[h].row[j];
            in[h].none[j] = row < 0;
            load_few<T, FN>(dyp + (int64_t)max(row, 0) * N, nn, in_n, in[h].a[j]);
            load_few<T, 4>(xp + (int64_t)max(row, 0) * K, nk, in_k, in[h].b[j]);
        }
    };
#pragma unroll
    for (int h = 0; h < kDepth; h++) rows(h, 16 * wave + 64 * h);
#pragma unroll
    for (int h = 0; h < kDepth; h++) load(h);
#pragma unroll
    for (int h = 0; h < kDepth; h++) rows(h, 16 * wave + 64 * (h + kDepth));
    for (int at = 16 * wave; at < count; at += 64 * kDepth) {
#pragma unroll
        for (int h = 0; h < kDepth; h++) {
            float a[4][FN], b[4][4];
#pragma unroll
            for (int j = 0; j < 4; j++) {
#pragma unroll
                for (int i = 0; i < FN; i++) a[j][i] = in[h].none[j] ? 0.0f : in[h].a[j][i];
#pragma unroll
                for (int o = 0; o < 4; o++) b[j][o] = in[h].none[j] ? 0.0f : in[h].b[j][o];
            }
            if (kDepth > 1 || at + 64 < count) {
                load(h);
                rows(h, at + 64 * (h + 2 * kDepth));
            }
#pragma unroll
            for (int j = 0; j < 4; j++)
#pragma unroll
                for (int i = 0; i < FN; i++)
#pragma unroll
                    for (int o = 0; o < 4; o++) acc[i][o] = __builtin_amdgcn_mfma_f32_16x16x4f32(a[j][i], b[j][o], acc[i][o], 0, 0, 0);
        }
    }
    if (count <= 16) {
#pragma unroll
        for (int i = 0; i < FN; i++)
#pragma unroll
            for (int j = 0; j < 4; j++) {
                const float v[4] = {acc[i][0][j], acc[i][1][j], acc[i][2][j], acc[i][3][j]};
                put(n0 + FN * (4 * q + j) + i, v);
            }
        return;
    }
#pragma unroll
    for (int i = 0; i < FN; i++) {
        if (i) __syncthreads();
#pragma unroll
        for (int j = 0; j < 4; j++) parts[wave][j][l] = f32x4{acc[i][0][j], acc[i][1][j], acc[i][2][j], acc[i][3][j]};
        __syncthreads();
        const f32x4 v = ((parts[0][wave][l] + parts[1][wave][l]) + parts[2][wave][l]) + parts[3][wave][l];
        put(n0 + FN * (4 * q + wave) + i, (const float *)&v);
    }
}
// An expert of kLong rows or more takes a multiple of a tile's time, most of it memory's latency, so the grid's first `early`
// workgroups are for such experts (one holds a place that kLong divides, and the first of those names it), in tiles of 16 x 64
// with two blocks in flight: with half of 65536 rows at 16 of 1024 experts (256 x 64 f32) 75 us for 104 (even loads 47 for 42).
constexpr int kLong = 256;
template <class T, int FN>
__global__ __launch_bounds__(256) void grad_w_small_kernel(const T *dy, const T *x, Groups g, int N, int K, T *dw, int tk, int early) {
    __shared__ f32x4 parts[4][4][64];
    const int b = blockIdx.x;
    if (b < early) {
        const int tn = (N + 15) / 16, t = tile_of(b, early), place = t / (tn * tk) * kLong;
        const Piece pc = piece_from<1>(g, place);
        if (pc.count <= 0 || pc.e >= g.E) return;
        const int first = first_of(g, pc.e), count = end_of(g, pc.e) - first;
        if (count < kLong || (place > 0 && first <= place - kLong)) return;
        grad_w_small<T, 1, 2>(parts, dy, x, g, N, K, dw + (int64_t)pc.e * N * K, first, count, t / tk % tn * 16, t % tk * 64);
    } else {
        const int tn = (N + 16 * FN - 1) / (16 * FN), t = tile_of(b - early, gridDim.x - early), e = t / (tn * tk);
        const int first = first_of(g, e), count = end_of(g, e) - first;
        if (count >= kLong) return;
        grad_w_small<T, FN, 1>(parts, dy, x, g, N, K, dw + (int64_t)e * N * K, first, count, t / tk % tn * 16 * FN, t % tk * 64);
    }
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
        const int row = i < pc.count ? row_of(g, pc.first + i) : -1;
        return row < 0 ? kFar : (uint32_t)row * bytes_r;     // brings zeros
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
             [](int) {}, pc.count);
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

constexpr std::integral_constant<int, 1> one{};
constexpr std::integral_constant<int, 2> two{};
constexpr std::integral_constant<int, 4> four{};

bool aligned16(const void *p, int64_t row_bytes) { return (uintptr_t)p % 16 == 0 && row_bytes % 16 == 0; }
constexpr int64_t kMostBytes = 0x78000000;   // of an operand with 32-bit offsets: kFar and a few steps stay past it

// Tiles of 256 x 256 straight to LDS pay where an expert's rows fill half of one and there are tiles for the 256 CUs: on
// 16384 x 4096 x 4096 f16 over 8 experts 502 us a call against 692 with the 128 x 128 tiles through registers, which take the
// rest (a quarter of the rows go to two of the experts, the others anywhere; even loads 532 against 704).
template <class T, bool TR>
hipError_t go_rows(const void *in, const void *w, const Groups &g, int O, int R, void *out, hipStream_t st) {
    const int64_t in_row = (int64_t)R * sizeof(T), w_row = TR ? (int64_t)O * sizeof(T) : in_row;
    if constexpr (sizeof(T) == 2) {
        const int cols = (O + 255) / 256;
        const int64_t rows = (int64_t)g.M / 256 + g.E + 2;
        if (aligned16(in, in_row) && aligned16(w, w_row) && g.M * in_row < kMostBytes && O * in_row < kMostBytes &&
            g.M >= 128 * (int64_t)g.E && (rows - g.E / 2) * cols >= 256 && rows * cols <= most_blocks(512)) {
            hipLaunchKernelGGL((rows_turn_kernel<T, 8, 4, 2, 4, TR>), dim3((unsigned)(rows * cols)), dim3(512), 0, st,
                               (const T *)in, (const T *)w, g, O, R, (T *)out, cols, 16);
            return hipGetLastError();
        }
    }
    auto tiles = [&](auto fi, auto wi, auto wo) {
        constexpr int FI = decltype(fi)::value, WI = decltype(wi)::value, WO = decltype(wo)::value, kI = 16 * FI * WI, kO = 64 * WO;
        const int cols = (O + kO - 1) / kO;
        const int64_t slots = (int64_t)g.M / kI + g.E + 2, rows = std::min<int64_t>(slots, g.M);
        if (rows * cols > most_blocks(64 * WI * WO)) return kTooLarge;
        hipLaunchKernelGGL((rows_kernel<T, FI, 4, WI, WO, TR>), dim3((unsigned)(rows * cols)), dim3(64 * WI * WO), 0, st,
                           (const T *)in, (const T *)w, g, O, R, (T *)out, cols, 16, slots > g.M);
        return hipGetLastError();
    };
    // Measured with 64 experts of 1528 x 2040 and M / 64 rows each, bf16 / f32, us:
    //   rows of each                           1          7         31         62        125        250
    //   y   few_rows                      75/148    111/212    216/461    920/812
    //       16 x 64, 1 wave               75/144    118/224    177/366    288/600    400/893
    //       32 x 64, 1                    75/179    101/207    146/319    224/526    297/805
    //       64 x 64, 2                    77/315     96/329    143/452    174/437    227/812    434/1341
    //       64 x 128, 4                   86/301     99/312    133/385    158/452    183/683    331/1147
    //       128 x 128, 4                 101/559    115/564    136/719    186/740    167/750    290/1276
    //   dx  16 x 64, 1                   121/297    156/331    213/454    316/615    407/919
    //       64 x 64, 2                   115/372    131/432    146/510    201/541    246/848    404/1342
    //       64 x 128, 4                   94/354    138/437    149/487    169/544    212/842    343/1298
    // f32's matrix instructions are 1/16 of bf16's rate, so rows that a tile lacks cost it more. Matrices of 64 values along a
    // side keep to the 16-row tiles: with loads as uneven as a router's most experts have fewer rows than the mean.
    const int64_t mean = g.M / g.E;
    const bool f32 = sizeof(T) == 4, small = O <= 64 || R <= 64;
    if constexpr (!TR) {
        if (mean < 4 || g.M < 64 || (small && mean < 16)) {
            // off 16 bytes a row's 64 take two or three lines each, which tiles' whole 128 bytes feel less: 22 rows through 27
            // experts of 1702 x 1543 bf16 24 us for 57 (1704 x 1544: 23 and 27; 16 through 64 of 1536 x 2048: 23 and 18).
            // They do not split r, so there have to be enough of them.
            if (!small && !(aligned16(in, in_row) && aligned16(w, w_row)) && (int64_t)g.M * ((O + 63) / 64) >= 256) return tiles(one, one, one);
            const int cols = (O + 15) / 16;
            const int64_t slots = (int64_t)g.M / 16 + g.E + 2, rows = std::min<int64_t>(slots, g.M);
            if (rows * cols > most_blocks(in_row <= 1024 ? 64 : 256)) return kTooLarge;
            if (in_row <= 1024)
                hipLaunchKernelGGL((few_rows_kernel<T, 1>), dim3((unsigned)(rows * cols)), dim3(64), 0, st, (const T *)in,
                                   (const T *)w, g, O, R, (T *)out, cols, slots > g.M);
            else
                hipLaunchKernelGGL((few_rows_kernel<T, 4>), dim3((unsigned)(rows * cols)), dim3(256), 0, st, (const T *)in,
                                   (const T *)w, g, O, R, (T *)out, cols, slots > g.M);
            return hipGetLastError();
        }
        if constexpr (sizeof(T) == 4) {
            if (small && mean <= 128) return tiles(one, one, one);
            if (mean < 48) return tiles(two, one, one);
        } else if (mean >= 96 && O > 64) {
            return tiles(four, two, two);
        }
        return mean < 48 || O <= 64 ? tiles(two, two, one) : tiles(two, two, two);
    } else {
        if (small && mean <= (f32 ? 128 : 16)) return tiles(one, one, one);
        if (f32 && mean < 48) return tiles(one, one, one);
        return O <= 64 ? tiles(two, two, one) : tiles(two, two, two);
    }
}
template <class T>
hipError_t go_grad_w(const void *dy, const void *x, const Groups &g, int N, int K, void *dw, hipStream_t st) {
    if constexpr (sizeof(T) == 2) {
        const int tn = (N + 255) / 256, tk = (K + 255) / 256;
        const int64_t tiles = (int64_t)g.E * tn * tk, dy_row = (int64_t)N * sizeof(T), x_row = (int64_t)K * sizeof(T);
        if (aligned16(dy, dy_row) && aligned16(x, x_row) && g.M * dy_row < kMostBytes && g.M * x_row < kMostBytes &&
            tiles >= 256 && tiles <= most_blocks(512) && N >= 192 && K >= 192) {
            hipLaunchKernelGGL((grad_w_turn_kernel<T, 8, 4, 2, 4>), dim3((unsigned)tiles), dim3(512), 0, st, (const T *)dy,
                               (const T *)x, g, N, K, (T *)dw, tn, tk);
            return hipGetLastError();
        }
    }
    // us of 64 experts of 1528 x 2040 as above: f32 1 row of each 210 (64 x 128 tiles 262), 7 rows 247 (276), 31 rows 419 (315)
    if (N >= 4 && K >= 4 && (N <= 64 || (sizeof(T) == 4 && g.M < 16 * (int64_t)g.E))) {
        auto small = [&](auto fn) {
            constexpr int FN = decltype(fn)::value;
            const int tn = (N + 16 * FN - 1) / (16 * FN), tk = (K + 63) / 64;
            const int64_t early = g.M >= kLong ? ((int64_t)g.M / kLong + 1) * ((N + 15) / 16) * tk : 0;
            const int64_t tiles = (int64_t)g.E * tn * tk + early;
            if (tiles > most_blocks(256)) return kTooLarge;
            hipLaunchKernelGGL((grad_w_small_kernel<T, FN>), dim3((unsigned)tiles), dim3(256), 0, st, (const T *)dy, (const T *)x, g, N,
                               K, (T *)dw, tk, (int)early);
            return hipGetLastError();
        };
        return N <= 16 ? small(one) : N <= 32 ? small(two) : small(four);
    }
    auto tiles = [&](auto fi, auto wi, auto wo) {
        constexpr int FI = decltype(fi)::value, WI = decltype(wi)::value, WO = decltype(wo)::value, kI = 16 * FI * WI, kO = 64 * WO;
        const int tn = (N + kI - 1) / kI, tk = (K + kO - 1) / kO;
        const int64_t tiles = (int64_t)g.E * tn * tk;
        if (tiles > most_blocks(64 * WI * WO)) return kTooLarge;
        hipLaunchKernelGGL((grad_w_kernel<T, FI, 4, WI, WO>), dim3((unsigned)tiles), dim3(64 * WI * WO), 0, st, (const T *)dy,
                           (const T *)x, g, N, K, (T *)dw, tn, tk);
        return hipGetLastError();
    };
    // 64 x 128, 128 x 128 and (16 waves) 256 x 256: 4 experts of 1000 x 1000 bf16 74, 81 and 120 us; 64 of 1527 x 2041, 250 rows of
    // each, bf16 413, 372 and 349, f32 1345 and 1250; 8 of 3001 x 2999 bf16 1379, 1157 and 936
    const int64_t tiles128 = (int64_t)g.E * ((N + 127) / 128) * ((K + 127) / 128);
    if constexpr (sizeof(T) == 2) {
        if (tiles128 >= 2048) return tiles(four, four, four);
    }
    return tiles128 >= 512 ? tiles(four, two, two) : tiles(two, two, two);
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
