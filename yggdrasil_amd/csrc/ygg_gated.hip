// The gated projections of a feed-forward block: with g = x Wg^T and u = x Wu^T, y = act(g) u in one kernel; and their gradients
//   dg = dy u act'(g), du = dy act(g);  dx = dg Wg + du Wu,  dWg = dg^T x, dWu = du^T x.
//
// A tile computes g and u of the same columns: a wave's 64 columns of the columns' operand are 32 rows of Wg and the 32 rows of
// Wu below them, so a lane ends up with 8 neighbouring values of g and the same 8 of u, in f32, and takes their product there. For a
// backward pass g and u are kept: of 16-bit types the upper 24 bits of f32, so that the only roundings that the gradients have and
// g and u's own do not are those of dg and du on their way into the matrix cores and the results'. dg and du lie in rows of
// 2 N values: with w as (2 N, K) each gradient is a single product,
//   dx = [dg du] w,  dw = [dg du]^T x,
// of operands in tiles of their own; where the tiles are few for the 256 CUs the reduction is cut too, and the parts, in f32, are
// added in their order.
//
// f16 holds 40 powers of two, and dg and du may lie past them though what comes of them does not (u = dy = 300: dg about 90000; a loss in
// parts of 2^-20: dg 0). So the kernel that takes them also takes the largest of each row, which dx sums along, and of each column, which
// dw does, by maxima, which come out the same in any order. Where every one that is not 0 lies in f16 from 2^-3 on, dg and du are right as
// they are: off by 2^-11 of themselves or by 2^-22 of the largest that is summed with them. Else they are taken once more, into a copy for
// dx and one for dw, multiplied by powers of two of their rows and columns that bring the largest to 2^14 or more (2^-39 of the largest then),
// which are undone in f32 behind the sums; the card decides, and the products read which. 16384 x 2048 x 4096 f16, forward and
// backward, takes 1618 us without all that, 1675 with it and 1900 where the copies are made; 1001 x 1000 x 2003 97, 112 and 126. bf16
// reaches as far as f32.
//
// The matrix cores bound large products (16384 x 2048 x 4096 bf16 forward 490 us of kernels with g and u kept, 1.1 PFLOP/s at the 1.8 GHz
// that the card falls to; dg and du 145, by the memory; dx 440 and dw 500), the weights' reading few rows (1 x 4096 x 8192 bf16 24 us,
// 5.7 TB/s), the launches and the tiles' first loads what lies between.
#include <algorithm>

#include "ygg_gemm.h"
#include "ygg_ops.h"

namespace ygg {
namespace {

// act(g) and, of the backward pass, act'(g)
template <int kAct> __device__ __forceinline__ float act_of(float g, float *slope = nullptr) {
    if constexpr (kAct == kGelu) {
        const float phi = 0.5f * erfcf(g * -0.70710678118654752f);      // 1 + erf has no digits left where g is far below 0
        if (slope) *slope = __builtin_fmaf(g, 0.3989422804014327f * expf(-0.5f * g * g), phi);
        return g * phi;
    } else {
        const float e = expf(-g), p = 1.0f / (1.0f + e);
        if constexpr (kAct == kSilu) {
            if (slope) *slope = p * __builtin_fmaf(g, 1.0f - p, 1.0f);
            return g * p;
        } else {
            if (slope) *slope = p * (g > 0.0f ? e * p : 1.0f - p);      // 1 - p, which has no digits left where p is near 1
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

constexpr int kBand = 16;     // rows of tiles of a band

// the row of w of a tile's column o, the tile's outputs beginning at n0
__device__ __forceinline__ int row_of_w(int o, int n0, int N) { return (o & 32 ? N : 0) + min(n0 + (o >> 6) * 32 + (o & 31), N - 1); }

// What is kept of rows of N values lies `half` values apart, N up to a multiple of 8, so that it is read and written aligned and in whole
// runs of a lane's 8 results
__host__ __device__ constexpr int half_of(int N) { return (N + 7) / 8 * 8; }

// g and u of M rows, kept for the backward pass, in rows of 2 half values: f32, or its upper 24 bits, first all values' 16 and then their 8
// (in 16 bits alone the gradients were 1.8 times as far off as a rounding, in 24 1.4; the 16384 x 4096 of a bf16 case take the memory
// 134 MB longer on the way out and in)
template <class T> struct Kept {
    static constexpr int kBytes = sizeof(T) == 4 ? 4 : 3;
    char *p;
    int64_t count;
    // kN values from place `at` on, which may go on behind the row's N
    template <int kN> __device__ __forceinline__ void put(int64_t at, const float *v) const {
        if constexpr (sizeof(T) == 4) {
            store_run<float, kN>((float *)p + at, v, kN);
        } else {
            uint32_t b[kN];
#pragma unroll
            for (int j = 0; j < kN; j++)      // to nearest; a NaN must not carry into the sign
                b[j] = v[j] == v[j] ? __builtin_bit_cast(uint32_t, v[j]) + 0x80u : 0x7fc00000u;
            typedef uint32_t hi_t __attribute__((ext_vector_type(kN / 2)));
            typedef uint32_t lo_t __attribute__((ext_vector_type(kN / 4)));
            hi_t h;
            lo_t l;
#pragma unroll
            for (int j = 0; j < kN / 2; j++) h[j] = b[2 * j] >> 16 | (b[2 * j + 1] & 0xffff0000u);
#pragma unroll
            for (int j = 0; j < kN / 4; j++)
                l[j] = (b[4 * j] >> 8 & 0xffu) | (b[4 * j + 1] & 0xff00u) | (b[4 * j + 2] & 0xff00u) << 8 | (b[4 * j + 3] & 0xff00u) << 16;
            *(hi_t *)(p + 2 * at) = h;
            *(lo_t *)(p + 2 * count + at) = l;
        }
    }
    // what is kept of 16 bytes of values, as it lies there; kPast: past the caches, which would not hold it until it is read again
    struct Piece {
        u32x4 hi;
        u32x2 lo;
    };
    template <bool kPast> __device__ __forceinline__ Piece load(int64_t at) const {
        Piece v = {};
        const u32x4 *hi = (const u32x4 *)(p + at * (sizeof(T) == 4 ? 4 : 2));
        v.hi = kPast ? __builtin_nontemporal_load(hi) : *hi;
        if constexpr (sizeof(T) == 2) {
            const u32x2 *lo = (const u32x2 *)(p + 2 * count + at);
            v.lo = kPast ? __builtin_nontemporal_load(lo) : *lo;
        }
        return v;
    }
    static __device__ __forceinline__ void values(const Piece &v, float *f) {
#pragma unroll
        for (int j = 0; j < 16 / (int)sizeof(T); j++)
            f[j] = __builtin_bit_cast(float, sizeof(T) == 4 ? v.hi[j] : (v.hi[j / 2] >> 16 * (j % 2)) << 16 | (v.lo[j / 4] >> 8 * (j % 4) & 0xffu) << 8);
    }
};

// kN neighbouring outputs of a row
template <class T, int kAct, int kN>
__device__ __forceinline__ void put_outputs(const float *g, const float *u, int row, int n, int N, T *y, const Kept<T> &gu) {
    float v[kN];
#pragma unroll
    for (int j = 0; j < kN; j++) v[j] = act_of<kAct>(g[j]) * u[j];
    store_run<T, kN>(y + (int64_t)row * N + n, v, N - n);
    if (gu.p) {
        const int half = half_of(N);
        const int64_t at = (int64_t)row * 2 * half + n;
        gu.template put<kN>(at, g);
        gu.template put<kN>(at + half, u);
    }
}
template <class T, int kAct, int FI, class Acc>
__device__ __forceinline__ void put_tile(Acc (&acc)[FI][4], int row0, int part, int M, int n0, int N, T *y, const Kept<T> &gu, int i0) {
    const int l = threadIdx.x & 63, n = n0 + part * 32 + 8 * (l >> 4);
    if (n >= N) return;
#pragma unroll
    for (int i = 0; i < FI; i++) {
        const int row = i0 + row0 + 16 * i + (l & 15);
        if (row < M) put_outputs<T, kAct, 8>((const float *)&acc[i][0], (const float *)&acc[i][2], row, n, N, y, gu);
    }
}

template <class T, int FI, int WI, int WO, int kAct>
__global__ __launch_bounds__(64 * WI * WO) void gated_kernel(const T *x, const T *w, int M, int N, int K, T *y, Kept<T> gu, int cols, int band) {
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
__global__ __launch_bounds__(512) void gated_turn_kernel(const T *x, const T *w, int M, int N, int K, T *y, Kept<T> gu, int cols, int band) {
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

// Few tiles: 16 FR rows by 16 FC outputs a workgroup, whose four waves take a part of K each, fragments straight from memory
template <class T, int FR, int FC, int kAct>
__global__ __launch_bounds__(256) void gated_few_kernel(const T *x, const T *w, int M, int N, int K, T *y, Kept<T> gu, int cols) {
    constexpr int kE = 16 / sizeof(T), kStep = 4 * kE, kU = FR == 1 ? 4 : 2;
    __shared__ f32x4 parts[4][FR * FC][2][64];
    // the rows' tiles of a column of outputs follow each other: they share its weights
    const int t = tile_of(blockIdx.x, gridDim.x), tall = gridDim.x / cols, n0 = t / tall * 16 * FC, m0 = t % tall * 16 * FR;
    const int l = threadIdx.x & 63, wave = threadIdx.x >> 6, d = l & 15, q = l >> 4;
    f32x4 acc[FR][FC][2];
#pragma unroll
    for (int i = 0; i < FR; i++)
#pragma unroll
        for (int o = 0; o < FC; o++) acc[i][o][0] = acc[i][o][1] = f32x4{0, 0, 0, 0};
    const int steps = (K + kStep - 1) / kStep, per = (steps + 3) / 4, end = min(per * (wave + 1), steps);
    const T *wp[FC], *xp[FR];
    const int64_t to_u = (int64_t)N * K;
#pragma unroll
    for (int o = 0; o < FC; o++) wp[o] = w + (int64_t)min(n0 + 16 * o + d, N - 1) * K + q * kE;
#pragma unroll
    for (int i = 0; i < FR; i++) xp[i] = x + (int64_t)min(m0 + 16 * i + d, M - 1) * K + q * kE;
    int s = per * wave;
    for (; s + kU <= end && (s + kU) * kStep <= K; s += kU) {
        u32x4 a[kU][FC][2], c[kU][FR];
#pragma unroll
        for (int k = 0; k < kU; k++)
#pragma unroll
            for (int o = 0; o < FC; o++) {
                a[k][o][0] = load16(wp[o] + (s + k) * kStep);
                a[k][o][1] = load16(wp[o] + to_u + (s + k) * kStep);
            }
#pragma unroll
        for (int k = 0; k < kU; k++)
#pragma unroll
            for (int i = 0; i < FR; i++) c[k][i] = load16(xp[i] + (s + k) * kStep);
#pragma unroll
        for (int k = 0; k < kU; k++)
#pragma unroll
            for (int i = 0; i < FR; i++)
#pragma unroll
                for (int o = 0; o < FC; o++) {
                    acc[i][o][0] = Mma<T>::run(a[k][o][0], c[k][i], acc[i][o][0]);
                    acc[i][o][1] = Mma<T>::run(a[k][o][1], c[k][i], acc[i][o][1]);
                }
    }
    const int last = K - q * kE;
    auto load_end = [&](const T *p) { return K >= kE ? load16_end(p + s * kStep, last - s * kStep) : load16(p + s * kStep, last - s * kStep); };
    for (; s < end; s++) {
        u32x4 c[FR];
#pragma unroll
        for (int i = 0; i < FR; i++) c[i] = load_end(xp[i]);
#pragma unroll
        for (int o = 0; o < FC; o++) {
            const u32x4 a = load_end(wp[o]), b = load_end(wp[o] + to_u);
#pragma unroll
            for (int i = 0; i < FR; i++) {
                acc[i][o][0] = Mma<T>::run(a, c[i], acc[i][o][0]);
                acc[i][o][1] = Mma<T>::run(b, c[i], acc[i][o][1]);
            }
        }
    }
#pragma unroll
    for (int i = 0; i < FR; i++)
#pragma unroll
        for (int o = 0; o < FC; o++) {
            parts[wave][i * FC + o][0][l] = acc[i][o][0];
            parts[wave][i * FC + o][1][l] = acc[i][o][1];
        }
    __syncthreads();
    for (int f = wave; f < FR * FC; f += 4) {
        f32x4 g = parts[0][f][0][l], u = parts[0][f][1][l];
#pragma unroll
        for (int k = 1; k < 4; k++) {
            g += parts[k][f][0][l];
            u += parts[k][f][1][l];
        }
        const int row = m0 + 16 * (f / FC) + d, n = n0 + 16 * (f % FC) + 4 * q;
        if (row < M && n < N) put_outputs<T, kAct, 4>((const float *)&g, (const float *)&u, row, n, N, y, gu);
    }
}

// dg and du come with the powers of two of their rows or columns, where they want them
template <class T> constexpr bool kScaled = std::is_same_v<T, f16_t>;
// e with 2^14 <= v / 2^e < 2^15, from v's bits; 0 of no value
__device__ __forceinline__ int power_of(uint32_t bits) { return bits ? (int)(bits >> 23) - 127 - 14 : 0; }
__device__ __forceinline__ float times_power(float v, int e) { return __builtin_amdgcn_ldexpf(v, e); }

// 16 bytes of a row's columns from n on: what is kept of them and dy, then dg and du, zeros behind N
template <class T, int kAct, bool kPast> struct Slope {
    static constexpr int kE = 16 / sizeof(T);
    typename Kept<T>::Piece gp, up;
    u32x4 dp;
    __device__ __forceinline__ void load(const Kept<T> &gu, const T *dy, int64_t row, int N, int half, int n) {
        const int64_t at = row * 2 * half + n;
        gp = gu.template load<kPast>(at);
        up = gu.template load<kPast>(at + half);
        dp = N - n >= kE ? load16(dy + row * N + n) : load16(dy + row * N + n, N - n);
    }
    __device__ __forceinline__ void values(float *g, float *u, int left) const {
        float d[kE];
        Kept<T>::values(gp, g);
        Kept<T>::values(up, u);
        unpack(dp, d, T());
#pragma unroll
        for (int j = 0; j < kE; j++) {
            float slope;
            const float a = act_of<kAct>(g[j], &slope);
            g[j] = j < left ? d[j] * u[j] * slope : 0.0f;      // what lies behind N may be anything
            u[j] = j < left ? d[j] * a : 0.0f;
        }
    }
};

// dg and du lie as g and u do, so that the products' loads are aligned, zeros behind N. A thread: 16 bytes of each
template <class T, int kAct, bool kPast>
__global__ __launch_bounds__(256) void gated_slope_kernel(Kept<T> gu, const T *dy, int M, int N, T *dgu) {
    constexpr int kE = 16 / sizeof(T);
    const int half = half_of(N), per = half / kE;
    const int64_t id = (int64_t)blockIdx.x * 256 + threadIdx.x, row = id / per;
    if (row >= M) return;
    const int n = (int)(id % per) * kE;
    float g[kE], u[kE];
    Slope<T, kAct, kPast> s;
    s.load(gu, dy, row, N, half, n);
    s.values(g, u, N - n);
    T *out = dgu + row * 2 * half + n;
    store_run<T, kE>(out, g, kE, kPast);
    store_run<T, kE>(out + half, u, kE, kPast);
}

// f16: dg and du as they are, and the bits of the largest finite magnitudes of the rows and columns; `range` is 1 where those do not let
// them be. by_col: room for dw's copy then
struct Reach {
    uint32_t *rows, *cols, *range;
    void *by_col;
};
__global__ __launch_bounds__(256) void zero_kernel(uint32_t *p, int64_t count) {
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (i < count) p[i] = 0;
}
// A workgroup: `band` rows of 64 pieces of columns, each of its waves a row at a time. Workgroups of 16 waves, so that the maxima of a band's
// columns in memory are few (1001 x 2003 16.4 us, with 8 waves 25; 16384 x 4096 190 with either: the activations and the reading)
constexpr int kReachWaves = 16;
template <class T, int kAct, bool kPast>
__global__ __launch_bounds__(64 * kReachWaves)
void gated_reach_kernel(Kept<T> gu, const T *dy, int M, int N, int band, int slabs, T *dgu, Reach to) {
    constexpr int kE = 16 / sizeof(T), kC = 64 * kE;
    __shared__ uint32_t lds[kReachWaves][2 * kE][65];
    const int half = half_of(N), lane = threadIdx.x & 63, wave = threadIdx.x >> 6, c0 = (int)(blockIdx.x % slabs) * kC, n = c0 + lane * kE;
    const int first = (int)(blockIdx.x / slabs) * band, end = min(first + band, M);
    auto bits = [](float v) {
        const uint32_t b = __builtin_bit_cast(uint32_t, v) & 0x7fffffffu;
        return b < 0x7f800000u ? b : 0u;
    };
    uint32_t most[2 * kE] = {};
    for (int row = first + wave; row < end; row += kReachWaves) {
        uint32_t all = 0;
        if (n < half) {
            float g[kE], u[kE];
            Slope<T, kAct, kPast> s;
            s.load(gu, dy, row, N, half, n);
            s.values(g, u, N - n);
            T *out = dgu + (int64_t)row * 2 * half + n;
            store_run<T, kE>(out, g, kE, kPast);
            store_run<T, kE>(out + half, u, kE, kPast);
#pragma unroll
            for (int j = 0; j < kE; j++) {
                most[j] = max(most[j], bits(g[j]));
                most[kE + j] = max(most[kE + j], bits(u[j]));
                all = max(all, max(bits(g[j]), bits(u[j])));
            }
        }
        all = join<64>(all, [](uint32_t a, uint32_t b) { return max(a, b); });
        if (lane == 0 && all) atomicMax(to.rows + row, all);
    }
#pragma unroll
    for (int j = 0; j < 2 * kE; j++) lds[wave][j][lane] = most[j];
    __syncthreads();
    // neighbouring lanes take neighbouring columns; most maxima are not new ones
    for (int i = threadIdx.x; i < 2 * kC; i += 64 * kReachWaves) {
        const int c = i % kC, j = i / kC * kE + c % kE;
        if (c0 + c >= half) continue;
        uint32_t *at = to.cols + (i < kC ? 0 : half) + c0 + c, all = 0;
        for (int w = 0; w < kReachWaves; w++) all = max(all, lds[w][j][c / kE]);
        if (all > *(volatile uint32_t *)at) atomicMax(at, all);
    }
}
// the rows' and columns' largest lie one behind the other, `count` in all
__global__ __launch_bounds__(256) void gated_range_kernel(const uint32_t *most, int64_t count, uint32_t *range) {
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
    const uint32_t v = i < count ? most[i] : 0;
    if (v && (v < 0x3e000000u || v > 0x477fe000u)) *range = 1;      // 2^-3, 65504
}
// Where they are out of range: the two copies, by rows into dgu and by columns
template <class T, int kAct, bool kPast>
__global__ __launch_bounds__(256) void gated_rescale_kernel(Kept<T> gu, const T *dy, int M, int N, T *dgu, Reach to) {
    if (!*to.range) return;
    constexpr int kE = 16 / sizeof(T);
    const int half = half_of(N), per = half / kE;
    const int64_t all = (int64_t)M * per, hop = (int64_t)gridDim.x * 256;
    for (int64_t id = (int64_t)blockIdx.x * 256 + threadIdx.x; id < all; id += hop) {
        const int64_t row = id / per;
        const int n = (int)(id % per) * kE, e = power_of(to.rows[row]);
        const int64_t at = row * 2 * half + n;
        float g[kE], u[kE], t[kE];
        Slope<T, kAct, kPast> s;
        s.load(gu, dy, row, N, half, n);
        s.values(g, u, N - n);
#pragma unroll
        for (int j = 0; j < kE; j++) t[j] = times_power(g[j], -e);
        store_run<T, kE>(dgu + at, t, kE, kPast);
#pragma unroll
        for (int j = 0; j < kE; j++) t[j] = times_power(u[j], -e);
        store_run<T, kE>(dgu + at + half, t, kE, kPast);
        if (!to.by_col) continue;
        T *out = (T *)to.by_col + at;
#pragma unroll
        for (int j = 0; j < kE; j++) t[j] = times_power(g[j], -power_of(to.cols[n + j]));
        store_run<T, kE>(out, t, kE, kPast);
#pragma unroll
        for (int j = 0; j < kE; j++) t[j] = times_power(u[j], -power_of(to.cols[half + n + j]));
        store_run<T, kE>(out + half, t, kE, kPast);
    }
}

// ---- the gradients' products: out (I, O) = sum over r of A(i, r) b(r, o), b's rows `pitch` values apart. kRows: A is a (I, 2 half), the r's
// those of dg and du; else a^T, a (R, 2 half), the i's those of dg and du. A workgroup takes the steps of its part of the reduction; of more
// than one part, the sums go to `sums` in f32, part after part.
struct Dense {
    const void *a, *b;
    int I, O, R, pitch;
    int N, half;
    void *out;
    float *sums;
    int tiles, cols, per;       // tiles of a part, tiles along O, steps of a part
    // kScaled, NULL without rows: where *range, A is `scaled` instead, its row i by the power of two of most[i]
    const uint32_t *range, *most;
    const void *scaled;
    __device__ __forceinline__ bool is_scaled() const { return range && *range; }
    // the row of w that a column of dg and du belongs to, or -1
    __device__ __forceinline__ int place(int k) const { return k < N ? k : k >= half && k < half + N ? k - half + N : -1; }
};
template <class T, bool kRows> struct DenseOut {
    const Dense &g;
    int part, i0, o0;
    bool scaled;
    template <class N> __device__ __forceinline__ void operator()(int i, int o, const float *v, N) const {
        const int row = kRows ? (i0 + i < g.I ? i0 + i : -1) : g.place(i0 + i);
        if (row < 0 || o0 + o >= g.O) return;
        const int64_t at = (int64_t)row * g.O + o0 + o;
        float t[N::value];
        if constexpr (kScaled<T>) {
            const int e = scaled ? power_of(g.most[i0 + i]) : 0;
#pragma unroll
            for (int j = 0; j < N::value; j++) t[j] = times_power(v[j], e);
            v = t;
        }
        if (g.sums) store_run<float, N::value>(g.sums + (int64_t)part * g.I * g.O + at, v, g.O - o0 - o);
        else store_run<T, N::value>((T *)g.out + at, v, g.O - o0 - o);
    }
};
template <class T, int FI, int WI, int WO, bool kRows>
__global__ __launch_bounds__(64 * WI * WO) void dense_kernel(const Dense g) {
    constexpr int kThreads = 64 * WI * WO, kI = 16 * FI * WI, kO = 64 * WO;
    typedef std::conditional_t<kRows, Along<T, kI, kThreads, FI, true>, Across<T, kI, kThreads>> A;
    typedef Across<T, kO, kThreads> B;
    typedef Tile<T, FI, 4, WI, WO, A, B> Tl;
    __shared__ __align__(128) char lds[Tl::kLds];
    const int part = blockIdx.x / g.tiles, wide = 2 * g.half, R = kRows ? wide : g.R;
    const Place t = place_of(tile_of(blockIdx.x % g.tiles, g.tiles), g.tiles / g.cols, g.cols, kBand);
    const int i0 = t.row * kI, o0 = t.col * kO, steps = (R + A::kStep - 1) / A::kStep, first = part * g.per;
    const bool scaled = kScaled<T> && g.is_scaled();
    const void *const from = scaled ? g.scaled : g.a;
    Tl tile;
    A a;
    B b;
    if constexpr (kRows) a.begin([&](int i) { return (const T *)from + (int64_t)min(i0 + i, g.I - 1) * wide; });
    else a.begin((const T *)from, i0, wide);
    b.begin((const T *)g.b, o0, g.O);
    tile.run(a, b, lds, min(g.per, steps - first), [&](int s) {
        const int r0 = (first + s) * A::kStep;
        if constexpr (kRows) {
            a.load(r0, R);
            b.load([&](int i) {
                const int r = g.place(r0 + B::r_of(i));
                return r >= 0 ? (int64_t)r * g.pitch : -1;
            });
        } else {
            a.load([&](int i) { return r0 + A::r_of(i) < R ? (int64_t)(r0 + A::r_of(i)) * wide : -1; });
            b.load([&](int i) { return r0 + B::r_of(i) < R ? (int64_t)(r0 + B::r_of(i)) * g.pitch : -1; });
        }
    });
    const DenseOut<T, kRows> put = {g, part, i0, o0, scaled};
    tile.template each<false>([&](int i, int o, const typename Tl::Acc *v, auto n) { put(i, o, (const float *)v, n); });
}
template <class T, bool kRows> __global__ __launch_bounds__(512) void dense_turn_kernel(const Dense g) {
    constexpr int kSize = sizeof(T);
    typedef std::conditional_t<kRows, AlongLds<T, 8, 2, true>, AcrossLds<T, 8, 2>> A;
    typedef AcrossLds<T, 4, 4> B;
    typedef TurnTile<T, 8, 4, 2, 4, A, B> Tl;
    __shared__ __align__(1024) char lds[Tl::kLds];
    const int part = blockIdx.x / g.tiles, wide = 2 * g.half, R = kRows ? wide : g.R;
    const Place t = place_of(tile_of(blockIdx.x % g.tiles, g.tiles), g.tiles / g.cols, g.cols, kBand);
    const int i0 = t.row * 256, o0 = t.col * 256, steps = (R + B::kStep - 1) / B::kStep, first = part * g.per;
    const uint32_t a_row = wide * kSize, b_row = g.pitch * kSize;
    const bool scaled = kScaled<T> && g.is_scaled();
    const void *const from = scaled ? g.scaled : g.a;
    Tl tile;
    A a;
    B b;
    if constexpr (kRows) a.begin(from, g.I * a_row, a_row, [&](int i) { return i0 + i < g.I ? (uint32_t)(i0 + i) * a_row : kFar; });
    else a.begin(from, g.R * a_row, i0 * kSize, (wide - i0) * kSize);
    b.begin(g.b, (kRows ? 2 * g.N : g.R) * b_row, o0 * kSize, (g.O - o0) * kSize);
    tile.clear();
    auto row = [&](int r, uint32_t bytes) { return r >= 0 && r < R ? (uint32_t)r * bytes : kFar; };
    tile.run(lds, min(g.per, steps - first),
             [&](auto h, int s, uint32_t to) {
                 if constexpr (kRows) a.template load<decltype(h)::value>(first + s, to);
                 else a.template load<decltype(h)::value>(to, [&](int i) { return row((first + s) * B::kStep + A::r_of(i), a_row); });
             },
             [&](auto h, int s, uint32_t to) {
                 b.template load<decltype(h)::value>(to, [&](int i) {
                     const int r = (first + s) * B::kStep + B::r_of(i);
                     return row(kRows ? g.place(r) : r, b_row);
                 });
             },
             [](int) {}, kRows ? min(g.I - i0, 256) : 256);
    const DenseOut<T, kRows> put = {g, part, i0, o0, scaled};
    tile.template each<false>([&](int i, int o, const typename Tl::Acc *v, auto n) { put(i, o, (const float *)v, n); });
}
// rows of n values, `pitch` of whole 16 bytes apart
template <class T> __global__ __launch_bounds__(256) void spaced_kernel(const T *in, int64_t rows, int n, int pitch, T *out) {
    constexpr int kE = 16 / sizeof(T);
    const int per = pitch / kE;
    const int64_t id = (int64_t)blockIdx.x * 256 + threadIdx.x, row = id / per;
    if (row >= rows) return;
    const int c = (int)(id % per) * kE;
    *(u32x4 *)(out + row * pitch + c) = load16(in + row * n + c, n - c);
}
// the parts' sums, added in their order
template <class T> __global__ __launch_bounds__(256) void parts_kernel(const float *sums, int parts, int64_t count, T *out) {
    const int64_t at = ((int64_t)blockIdx.x * 256 + threadIdx.x) * 4;
    if (at >= count) return;
    const int left = (int)min(count - at, (int64_t)4);
    float v[4], p[4];
    unpack(load16(sums + at, left), v, 0.0f);
    for (int k = 1; k < parts; k++) {
        unpack(load16(sums + k * count + at, left), p, 0.0f);
#pragma unroll
        for (int j = 0; j < 4; j++) v[j] += p[j];
    }
    store_run<T, 4>(out + at, v, left);
}

bool aligned16(const void *p, int64_t row_bytes) { return (uintptr_t)p % 16 == 0 && row_bytes % 16 == 0; }
constexpr int64_t kMostBytes = 0x78000000;   // of an operand with 32-bit offsets: kFar and a few steps stay past it
template <class T, int kAct> hipError_t go(const void *x, const void *w, int M, int N, int K, void *y, void *kept, hipStream_t st) {
    const Kept<T> gu = {(char *)kept, (int64_t)M * 2 * half_of(N)};
    const int64_t row = (int64_t)K * sizeof(T);
    if constexpr (sizeof(T) == 2) {
        const int cols = (N + 127) / 128;
        const int64_t tiles = ((int64_t)M + 255) / 256 * cols;
        if (aligned16(x, row) && aligned16(w, row) && M * row < kMostBytes && 2 * N * row < kMostBytes && tiles >= 256 &&
            tiles <= most_blocks(512)) {
            hipLaunchKernelGGL((gated_turn_kernel<T, kAct>), dim3((unsigned)tiles), dim3(512), 0, st, (const T *)x, (const T *)w, M, N, K,
                               (T *)y, gu, cols, kBand);
            return hipGetLastError();
        }
    }
    auto few = [&](auto fr, auto fc) {
        constexpr int FR = decltype(fr)::value, FC = decltype(fc)::value;
        const int cols = (N + 16 * FC - 1) / (16 * FC);
        hipLaunchKernelGGL((gated_few_kernel<T, FR, FC, kAct>), dim3((unsigned)(cols * ((M + 16 * FR - 1) / (16 * FR)))), dim3(256), 0, st,
                           (const T *)x, (const T *)w, M, N, K, (T *)y, gu, cols);
        return hipGetLastError();
    };
    constexpr std::integral_constant<int, 1> one{};
    constexpr std::integral_constant<int, 2> two{};
    constexpr std::integral_constant<int, 4> four{};
    // Few tiles, as long as they are no more than the CUs: the smallest that are. bf16, in the tiles below and in these: 32 x 4096 x 1024
    // (rows, K, N) 34 and 16.5 us, 128 x 4096 x 1024 34 and 17, 256 x 4096 x 1024 35 and 25, 32 x 4096 x 8192 46 and 26, 64 x 4096 x 8192
    // 46 and 35; of twice as many as the CUs 128 x 4096 x 8192 46 and 60. The largest is no gain for 16-bit rows
    // off an alignment of 16 bytes (512 x 777 x 1001 13 and 17; f32 36 and 22).
    auto fits = [&](int fr, int fc) { return ((int64_t)M + 16 * fr - 1) / (16 * fr) * ((N + 16 * fc - 1) / (16 * fc)) <= 256; };
    if (M <= 16) return few(one, one);
    if (fits(2, 1)) return few(two, one);
    if (fits(2, 2)) return few(two, two);
    if (fits(4, 2) && (sizeof(T) == 4 || row % 16 == 0)) return few(four, two);
    auto tiles = [&](auto fi, auto wi, auto wo) {
        constexpr int FI = decltype(fi)::value, WI = decltype(wi)::value, WO = decltype(wo)::value, kI = 16 * FI * WI;
        const int cols = (N + 32 * WO - 1) / (32 * WO);
        const int64_t all = ((int64_t)M + kI - 1) / kI * cols;
        if (all > most_blocks(64 * WI * WO)) return kTooLarge;
        hipLaunchKernelGGL((gated_kernel<T, FI, WI, WO, kAct>), dim3((unsigned)all), dim3(64 * WI * WO), 0, st, (const T *)x,
                           (const T *)w, M, N, K, (T *)y, gu, cols, kBand);
        return hipGetLastError();
    };
    const int64_t tiles128 = ((int64_t)M + 127) / 128 * ((N + 63) / 64);
    // 128 rows a tile where there are more than one for each CU: 3000 x 2222 x 1111 (rows, K, N) bf16, 432 of them, 48 us, 65 with 64 rows;
    // 1001 x 1000 x 2003, 256 of them, 19.8 and 19.1
    return tiles128 >= 384 ? tiles(four, two, two) : tiles(two, two, two);
}
template <class T, int kAct> hipError_t go_slope(const void *gu, const void *dy, int M, int N, void *dgu, const Reach &to, hipStream_t st) {
    constexpr int kE = 16 / sizeof(T);
    const int half = half_of(N);
    const int64_t blocks = ((int64_t)M * (half / kE) + 255) / 256;
    if (blocks == 0) return hipSuccess;
    if (blocks > most_blocks(256)) return kTooLarge;
    const Kept<T> kept = {(char *)gu, (int64_t)M * 2 * half};
    auto launch = [&](auto past) {
        constexpr bool kPast = decltype(past)::value;
        if constexpr (kScaled<T>) {
            const int64_t count = (int64_t)M + 2 * half;      // rows, cols and range lie one behind the other
            const int slabs = (half / kE + 63) / 64, bands = std::max(512 / slabs, 1);
            const int band = ((M + bands - 1) / bands + kReachWaves - 1) / kReachWaves * kReachWaves;
            hipLaunchKernelGGL(zero_kernel, dim3((unsigned)((count + 256) / 256)), dim3(256), 0, st, to.rows, count + 1);
            hipLaunchKernelGGL((gated_reach_kernel<T, kAct, kPast>), dim3((unsigned)(slabs * ((M + band - 1) / band))), dim3(64 * kReachWaves), 0, st,
                               kept, (const T *)dy, M, N, band, slabs, (T *)dgu, to);
            hipLaunchKernelGGL(gated_range_kernel, dim3((unsigned)((count + 255) / 256)), dim3(256), 0, st, to.rows, count, to.range);
            // 2048: as many as the chip holds, so that they are soon gone where there is nothing to do
            hipLaunchKernelGGL((gated_rescale_kernel<T, kAct, kPast>), dim3((unsigned)std::min<int64_t>(blocks, 2048)), dim3(256), 0, st, kept,
                               (const T *)dy, M, N, (T *)dgu, to);
        } else {
            hipLaunchKernelGGL((gated_slope_kernel<T, kAct, kPast>), dim3((unsigned)blocks), dim3(256), 0, st, kept, (const T *)dy, M, N, (T *)dgu);
        }
    };
    // 16384 x 4096 bf16: 184 us with the caches, 145 past them
    if (kept.count * Kept<T>::kBytes >= kPastBytes) launch(std::true_type());
    else launch(std::false_type());
    return hipGetLastError();
}

// How a product is cut: 256 x 256 tiles straight to LDS (`turn`), which wants b's rows aligned: of a width that is no multiple of 16
// bytes they are laid out anew (`spaced`); else kI rows of a tile
struct Plan {
    bool turn, large, spaced;
    int cols, parts, per, pitch;
    int64_t tiles;
};
// rows: out (M, K) over 2 half r's; else out (2 N, K) over M
Plan plan_of(int size, bool rows, int M, int N, int K, bool aligned) {
    const int half = half_of(N), step = 128 / size, I = rows ? M : 2 * half, R = rows ? 2 * half : M, steps = (R + step - 1) / step;
    Plan p = {};
    auto cut = [&](int ti, int to, int64_t want, int least) {
        p.cols = (K + to - 1) / to;
        p.tiles = ((int64_t)I + ti - 1) / ti * p.cols;
        const int64_t parts = std::max<int64_t>(std::min<int64_t>(want / std::max<int64_t>(p.tiles, 1), steps / least), 1);
        p.per = (int)std::max<int64_t>((steps + parts - 1) / parts, 1);
        p.parts = std::max((steps + p.per - 1) / p.per, 1);      // without rows there is still the weights' gradient, zero
    };
    // 256 x 256 tiles where both sides fill most of one, and where tiles and parts come to 96 workgroups or more. Forward and one gradient of bf16
    // (rows, N, K) by those and by the smaller ones, us: 8192 x 2048 of K = 192 dx 108 and 128, dw 111 and 132, of K = 128 96 and 95, 100
    // and 95; 128 x 8192 x 4096 dx 96 and 91. 112 of them, 1001 x 2003 x 1000 dx 62 and 68, dw 63 and 67; 64 of them, 1024 x 1024 x 1024 47 and
    // 39, 49 and 39, 192 x 2048 x 2048 dx 47 and 41; 128, 256 x 4096 x 2048 dx 62 and 57
    p.pitch = half_of(K);
    const int64_t a_bytes = (int64_t)M * 2 * half * size, b_bytes = (int64_t)(rows ? 2 * N : M) * p.pitch * size;
    p.spaced = p.pitch != K;
    if (size == 2 && (aligned || p.spaced) && a_bytes < kMostBytes && b_bytes < kMostBytes && I >= 192 && K >= 192) {
        cut(256, 256, 256, 8);
        p.turn = p.tiles * p.parts >= 96;
        if (p.turn) return p;
    }
    p.spaced = false;
    p.pitch = K;
    p.large = ((int64_t)I + 127) / 128 * ((K + 127) / 128) >= 512;
    // two parts of tiles that are a few for each CU, so that the CUs end together: 3000 x 2222 x 1111 f32, of 846 and 630 tiles, both
    // gradients 826 us with one part and 670 with two
    const int64_t small = ((int64_t)I + 63) / 64 * ((K + 127) / 128);
    cut(p.large ? 128 : 64, 128, !p.large && small >= 600 ? 2 * small : 768, 6);
    return p;
}
// device memory of a product, behind each other: b laid out anew, the parts' sums
int64_t spaced_bytes(const Plan &p, int size, bool rows, int M, int N) {
    return p.spaced ? ((int64_t)(rows ? 2 * N : M) * p.pitch * size + 255) / 256 * 256 : 0;
}
int64_t part_bytes(const Plan &p, bool rows, int M, int N, int K) { return p.parts > 1 ? (int64_t)p.parts * (rows ? M : 2 * N) * K * 4 : 0; }
template <class T, bool kRows>
hipError_t go_dense(const void *a, const Reach &to, const void *b, int M, int N, int K, void *out, void *scratch, hipStream_t st) {
    const Plan p = plan_of(sizeof(T), kRows, M, N, K, (uintptr_t)b % 16 == 0);
    float *sums = (float *)((char *)scratch + spaced_bytes(p, sizeof(T), kRows, M, N));
    const int64_t blocks = p.tiles * p.parts, I = kRows ? M : 2 * N, count = I * K;
    if (blocks > most_blocks(512)) return kTooLarge;
    if (p.spaced) {
        constexpr int kE = 16 / sizeof(T);
        const int64_t rows = kRows ? 2 * N : M, pieces = (rows * (p.pitch / kE) + 255) / 256;
        if (pieces > most_blocks(256)) return kTooLarge;
        if (pieces) hipLaunchKernelGGL(spaced_kernel<T>, dim3((unsigned)pieces), dim3(256), 0, st, (const T *)b, rows, K, p.pitch, (T *)scratch);
        const hipError_t e = hipGetLastError();
        if (e != hipSuccess) return e;
        b = scratch;
    }
    const Dense g = {a, b, (int)I, K, M, p.pitch, N, half_of(N), out, p.parts > 1 ? sums : nullptr, (int)p.tiles, p.cols, p.per,
                     to.range, kRows ? to.rows : to.cols, kRows ? a : to.by_col};
    if (p.turn) {
        if constexpr (sizeof(T) == 2) hipLaunchKernelGGL((dense_turn_kernel<T, kRows>), dim3((unsigned)blocks), dim3(512), 0, st, g);
    } else if (p.large) {
        hipLaunchKernelGGL((dense_kernel<T, 4, 2, 2, kRows>), dim3((unsigned)blocks), dim3(256), 0, st, g);
    } else {
        hipLaunchKernelGGL((dense_kernel<T, 2, 2, 2, kRows>), dim3((unsigned)blocks), dim3(256), 0, st, g);
    }
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess || p.parts == 1) return e;
    hipLaunchKernelGGL(parts_kernel<T>, dim3((unsigned)((count + 1023) / 1024)), dim3(256), 0, st, (const float *)sums, p.parts, count, (T *)out);
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
int64_t gated_kept(int type, int M, int N) { return (int64_t)M * 2 * half_of(N) * (type == kOpF32 ? 4 : 3); }
// dg and du (f16: a copy for each product, the rows' and columns' largest and what is made of them), then what one product at a time takes;
// whether its operand turns out to be aligned or not
int64_t up_to_256(int64_t bytes) { return (bytes + 255) / 256 * 256; }
int64_t dgu_copy(int type, int M, int N) { return up_to_256((int64_t)M * 2 * half_of(N) * op_bytes(type)); }
int64_t dgu_bytes(int type, int M, int N) {
    const int64_t copy = dgu_copy(type, M, N);
    return type == kOpF16 && M ? 2 * copy + up_to_256(((int64_t)M + 2 * half_of(N) + 1) * 4) : copy;
}
int64_t gated_grad_scratch(int type, int M, int N, int K) {
    const int size = op_bytes(type);
    int64_t most = 0;
    for (bool aligned : {false, true})
        for (bool rows : {false, true}) {
            const Plan p = plan_of(size, rows, M, N, K, aligned);
            most = std::max(most, spaced_bytes(p, size, rows, M, N) + part_bytes(p, rows, M, N, K));
        }
    return dgu_bytes(type, M, N) + most;
}
hipError_t launch_gated_grad(int type, int act, const void *x, const void *w, const void *gu, const void *dy, int M, int N, int K,
                             void *dx, void *dw, void *scratch, hipStream_t st) {
    char *const at = (char *)scratch, *rest = at + dgu_bytes(type, M, N);
    const int64_t copy = dgu_copy(type, M, N);
    Reach to = {};
    if (type == kOpF16 && M) {
        to.rows = (uint32_t *)(at + 2 * copy);
        to.cols = to.rows + M;
        to.range = to.cols + 2 * half_of(N);
        to.by_col = dw ? at + copy : nullptr;
    }
    hipError_t e = with_type(type, [&](auto one) {
        return with_act(act, [&](auto k) { return go_slope<decltype(one), decltype(k)::value>(gu, dy, M, N, at, to, st); });
    });
    if (e != hipSuccess) return e;
    return with_type(type, [&](auto one) {
        typedef decltype(one) T;
        hipError_t e = hipSuccess;
        if (dx) e = go_dense<T, true>(at, to, w, M, N, K, dx, rest, st);
        if (e == hipSuccess && dw) e = go_dense<T, false>(at, to, x, M, N, K, dw, rest, st);
        return e;
    });
}

}  // namespace ygg
