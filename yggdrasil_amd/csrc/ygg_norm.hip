// Layer norm of rows and its gradients. With m and v a row's mean and variance and z = (x - m) / sqrt(v + eps):
//   y = z w + b;   q = w dy, dx = (q - mean(q) - z mean(q z)) / sqrt(v + eps);   dw = sum over rows of dy z, db = of dy.
//
// A row is held in the registers of 1 to 64 lanes or of a workgroup, 16 bytes a load, so that it is read once: the mean and
// then the squares about it are joined in f32. A workgroup's waves first take each its own mean and squares M2 and are joined by
//   m = sum n_i m_i / n,  M2 = sum M2_i + n_i (m_i - m)^2,
// which takes one barrier instead of two and cancels nothing. z is (x - m) times the inverse deviation, as it stands: with m times that
// rounded by itself, x rstd + (-m rstd) in one operation, rows far from zero lose half a step of |m| rstd, and rows of one value are not 0. The backward pass reads x and dy once, writes dx, and keeps its
// columns' sums of dy z and dy in registers over all of a workgroup's rows; the workgroups' sums are added in their order by a
// second kernel, so that they come out the same every time. Rows wider than the registers hold are read again: past 65536 values of
// f32, and in the backward pass, which holds the columns' sums too, past 16384.
//
// The memory bounds it: 65536 x 2048 bf16 forward 94 us (5.7 TB/s of reading and writing), backward 157 (5.1) and 5 for the join.
// 281 MB at other widths: forward 4.2 to 6.5 TB/s, backward 4.0 to 5.3, past 16384 values 2.9 to 3.4 of a single reading's bytes.
#include <algorithm>

#include "ygg_lanes.h"
#include "ygg_ops.h"
#include "ygg_optype.h"

namespace ygg {
namespace {

template <class T> constexpr int kEach = 16 / (int)sizeof(T);    // values of a piece

// A row of n values in pieces: piece i of lane `lane` of kL. The last piece of a row that it does not fill begins earlier, so that
// nothing in the rows' loop is cut: its first `skip` values are the piece's before it, computed and written twice alike and left
// out of the sums. kTiny: rows of less than a piece, one lane's.
template <class T, int kL, bool kTiny> struct Pieces {
    static constexpr int kE = kEach<T>;
    int n, lane;
    __device__ __forceinline__ int at(int i) const { return (i * kL + lane) * kE; }
    __device__ __forceinline__ int column(int i) const { return kTiny ? 0 : min(at(i), n - kE); }
    __device__ __forceinline__ bool some(int i) const { return at(i) < n; }
    __device__ __forceinline__ int skip(int i) const { return at(i) - column(i); }
    // columns and masks are worked out again from here on: those of many pieces held more registers than the values
    __device__ __forceinline__ void anew() { asm volatile("" : "+v"(lane)); }
    // all lanes' pieces are whole and their own
    __device__ __forceinline__ bool whole(int i) const { return !kTiny && (i + 1) * kL * kE <= n; }
    // value j of piece i is summed here
    __device__ __forceinline__ bool own(int i, int j) const { return kTiny ? lane == 0 && j < n : j >= skip(i); }
    __device__ __forceinline__ u32x4 load(const T *p, int i) const { return kTiny ? load16(p, n) : load16(p + column(i)); }
    template <class O> __device__ __forceinline__ void store(O *p, const float *f, int i, bool past) const {
        if (some(i)) store_run<O, kE>(p + column(i), f, kTiny ? n : kE, past);
    }
};

// What was unpacked from these before is not held until it is wanted again, but unpacked again
template <int kP> __device__ __forceinline__ void let_go(u32x4 (&v)[kP]) {
#pragma unroll
    for (int i = 0; i < kP; i++) asm volatile("" : "+v"(v[i])::"memory");
}

// kN values of a weight from column c on, in f32; `other` where there are none
template <class T, int kN> __device__ __forceinline__ void load_weight(float *f, const T *p, int c, int n, float other) {
    if (!p) {
#pragma unroll
        for (int j = 0; j < kN; j++) f[j] = other;
        return;
    }
    constexpr int kE = kEach<T>;
#pragma unroll
    for (int k = 0; k < kN; k += kE) {
        u32x4 v;
        if (c + k + kE <= n) v = load16(p + c + k);
        else v = load16(p + min(c + k, n - 1), n - c - k);
        float t[kE];
        unpack(v, t, T());
#pragma unroll
        for (int j = 0; j < kE && j < kN; j++) f[k + j] = t[j];
    }
}
template <class T, int kN>
__device__ __forceinline__ void load_weight(float *f, const void *p, bool wide, int c, int n, float other) {
    if (wide) load_weight<float, kN>(f, (const float *)p, c, n, other);
    else load_weight<T, kN>(f, (const T *)p, c, n, other);
}

// a piece that is all there
template <class T> __device__ __forceinline__ void whole_weight(float *f, const void *p, bool wide, int c, float other) {
    constexpr int kE = kEach<T>;
    if (!p) {
#pragma unroll
        for (int j = 0; j < kE; j++) f[j] = other;
    } else if (wide) {
#pragma unroll
        for (int k = 0; k < kE; k += 4) unpack(load16((const float *)p + c + k), f + k, 0.0f);
    } else {
        unpack(load16((const T *)p + c), f, T());
    }
}

// The mean and 1 / sqrt(variance + eps) of a row held by kL lanes. waves: LDS of a workgroup of more than a wave, another one
// than the row before's.
template <class T, int kL, bool kTiny, int kP>
__device__ __forceinline__ float2 moments(u32x4 (&x)[kP], const Pieces<T, kL, kTiny> &at, float eps, float2 *waves) {
    constexpr int kE = kEach<T>, kIn = kL < 64 ? kL : 64;
    const int n = at.n;
    // f(a value of the row that is this lane's)
    auto each = [&](auto f) {
#pragma unroll
        for (int i = 0; i < kP; i++) {
            float v[kE];
            unpack(x[i], v, T());
            if (at.whole(i)) {
#pragma unroll
                for (int j = 0; j < kE; j++) f(v[j], true);
            } else {
#pragma unroll
                for (int j = 0; j < kE; j++) f(v[j], at.own(i, j));
            }
            if constexpr (kP > 4) __builtin_amdgcn_sched_barrier(0);     // a piece at a time, for the registers
        }
    };
    float sum = 0.0f, squares = 0.0f;
    each([&](float v, bool own) { sum += own ? v : 0.0f; });
    // the values that a wave holds
    auto held = [&](int w) {
        int h = 0;
#pragma unroll
        for (int i = 0; i < kP; i++) h += min(max(n - (i * kL + w * 64) * kE, 0), 64 * kE);
        return (float)h;
    };
    const int wave = at.lane / 64;
    float mean = sum_of<kIn>(sum) / fmaxf(kL <= 64 ? (float)n : held(wave), 1.0f);
    let_go(x);
    each([&](float v, bool own) {
        const float d = own ? v - mean : 0.0f;
        squares = __builtin_fmaf(d, d, squares);
    });
    squares = sum_of<kIn>(squares);
    if constexpr (kL > 64) {
        if (at.lane % 64 == 0) waves[wave] = make_float2(mean, squares);
        __syncthreads();
        float total = 0.0f;
#pragma unroll
        for (int w = 0; w < kL / 64; w++) total = __builtin_fmaf(held(w), waves[w].x, total);
        mean = total / (float)n;
        squares = 0.0f;
#pragma unroll
        for (int w = 0; w < kL / 64; w++) {
            const float d = waves[w].x - mean;
            squares += __builtin_fmaf(held(w) * d, d, waves[w].y);
        }
    }
    return make_float2(mean, 1.0f / sqrtf(squares / (float)n + eps));
}

// A weight in f32 in LDS, in the order its lanes read it, 16 bytes each: in registers it would hold the rows off the CU
template <class T, int kL, int kP> struct Held {
    static constexpr int kE = kEach<T>;
    float v[kP][kE / 4][kL][4];
    template <int kThreads, bool kTiny> __device__ __forceinline__ void fill(const void *p, bool wide, int n, float other) {
        for (int k = threadIdx.x; k < kP * kL; k += kThreads) {
            const Pieces<T, kL, kTiny> at = {n, k % kL};
            float f[kE];
            load_weight<T, kE>(f, p, wide, at.column(k / kL), n, other);
#pragma unroll
            for (int j = 0; j < kE; j++) v[k / kL][j / 4][k % kL][j % 4] = f[j];
        }
    }
    __device__ __forceinline__ void get(float *f, int i, int lane) const {
#pragma unroll
        for (int j = 0; j < kE; j++) f[j] = v[i][j / 4][lane][j % 4];
    }
};

// kL lanes a row, kP pieces a lane; the next row's loads are on their way while a row is normed
template <class T, int kL, int kP, bool kTiny>
__global__ __launch_bounds__(kL > 256 ? kL : 256) void norm_kernel(const NormArgs a) {
    constexpr int kThreads = kL > 256 ? kL : 256, kRows = kThreads / kL, kE = kEach<T>;
    __shared__ float2 waves[2][kThreads / 64];
    constexpr bool kHeld = kL <= 256;      // wider rows' weights come from the caches for each row, so that LDS holds off no workgroup
    __shared__ Held<T, kHeld ? kL : 1, kHeld ? kP : 1> w, b;
    Pieces<T, kL, kTiny> at = {a.n, (int)threadIdx.x % kL};
    const int64_t hop = (int64_t)gridDim.x * kRows;
    int64_t row = (int64_t)blockIdx.x * kRows + threadIdx.x / kL;
    constexpr bool kAhead = kL <= 256 || kP <= 4;     // more pieces leave no registers for the next row's
    u32x4 x[kP], next[kAhead ? kP : 1];
    auto load = [&](u32x4 *v, int64_t r) {
        if (r >= a.rows) return;
#pragma unroll
        for (int i = 0; i < kP; i++) v[i] = at.load((const T *)a.x + r * a.stride, i);
    };
    if constexpr (kAhead) load(next, row);
    if constexpr (kHeld) {
        w.template fill<kThreads, kTiny>(a.weight, a.wide, a.n, 1.0f);
        b.template fill<kThreads, kTiny>(a.bias, a.wide, a.n, 0.0f);
        __syncthreads();
    }
    for (int turn = 0; row < a.rows; row += hop, turn ^= 1) {
        if constexpr (kAhead) {
#pragma unroll
            for (int i = 0; i < kP; i++) x[i] = next[i];
            load(next, row + hop);
        } else {
            load(x, row);
            at.anew();
        }
        const float2 s = moments(x, at, a.eps, waves[turn]);
        if (a.stats && at.lane == 0) ((float2 *)a.stats)[row] = s;
        let_go(x);
        if constexpr (!kAhead || (kL == 1024 && sizeof(T) == 2)) at.anew();
        T *y = (T *)a.y + row * a.n;
#pragma unroll
        for (int i = 0; i < kP; i++) {
            float f[kE], wf[kE], bf[kE];
            unpack(x[i], f, T());
            if constexpr (kHeld) {
                w.get(wf, i, at.lane);
                b.get(bf, i, at.lane);
            } else {
                whole_weight<T>(wf, a.weight, a.wide, at.column(i), 1.0f);
                whole_weight<T>(bf, a.bias, a.wide, at.column(i), 0.0f);
            }
#pragma unroll
            for (int j = 0; j < kE; j++) f[j] = __builtin_fmaf((f[j] - s.x) * s.y, wf[j], bf[j]);
            at.store(y, f, i, a.past);
            if constexpr (kP > 4) __builtin_amdgcn_sched_barrier(0);
        }
    }
}

// values joined over a workgroup of kThreads, the same in each thread
template <int kThreads> __device__ __forceinline__ float sum_all(float v, float *lds) {
    v = sum_of<64>(v);
    __syncthreads();
    if (threadIdx.x % 64 == 0) lds[threadIdx.x / 64] = v;
    __syncthreads();
    v = 0.0f;
#pragma unroll
    for (int w = 0; w < kThreads / 64; w++) v += lds[w];
    return v;
}
// f(column, values of x (and dy, where there is one), how many of them exist) over a row's pieces
template <class T, int kThreads, class F> __device__ __forceinline__ void each_piece(const T *x, const T *dy, int n, F f) {
    constexpr int kE = kEach<T>;
    for (int c = threadIdx.x * kE; c < n; c += kThreads * kE) {
        float v[kE], d[kE];
        unpack(load16(x + c, n - c), v, T());
        if (dy) unpack(load16(dy + c, n - c), d, T());
        f(c, v, d, n - c);
    }
}
// Rows wider than the registers of a workgroup: three readings, the later ones from the caches where they hold the row
template <class T> __global__ __launch_bounds__(1024) void norm_wide_kernel(const NormArgs a) {
    constexpr int kE = kEach<T>;
    __shared__ float lds[16];
    const int n = a.n;
    for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
        const T *x = (const T *)a.x + row * a.stride;
        float sum = 0.0f, squares = 0.0f;
        each_piece<T, 1024>(x, (const T *)nullptr, n, [&](int, const float *v, const float *, int) {
#pragma unroll
            for (int j = 0; j < kE; j++) sum += v[j];
        });
        const float mean = sum_all<1024>(sum, lds) / (float)n;
        each_piece<T, 1024>(x, (const T *)nullptr, n, [&](int, const float *v, const float *, int left) {
#pragma unroll
            for (int j = 0; j < kE; j++) {
                const float d = j < left ? v[j] - mean : 0.0f;
                squares = __builtin_fmaf(d, d, squares);
            }
        });
        const float inv = 1.0f / sqrtf(sum_all<1024>(squares, lds) / (float)n + a.eps);
        if (a.stats && threadIdx.x == 0) ((float2 *)a.stats)[row] = make_float2(mean, inv);
        T *y = (T *)a.y + row * n;
        each_piece<T, 1024>(x, (const T *)nullptr, n, [&](int c, const float *v, const float *, int left) {
            float w[kE], b[kE], f[kE];
            load_weight<T, kE>(w, a.weight, a.wide, c, n, 1.0f);
            load_weight<T, kE>(b, a.bias, a.wide, c, n, 0.0f);
#pragma unroll
            for (int j = 0; j < kE; j++) f[j] = __builtin_fmaf((v[j] - mean) * inv, w[j], b[j]);
            store_run<T, kE>(y + c, f, left);
        });
    }
}

// ---- backward: dx, and a workgroup's sums of dy z and dy over its rows into part[blockIdx][2][n]
template <class T, int kL, int kP, bool kTiny>
__global__ __launch_bounds__(kL > 256 ? kL : 256, 2) void norm_grad_kernel(const NormGradArgs a, float *part) {
    constexpr int kThreads = kL > 256 ? kL : 256, kRows = kThreads / kL, kE = kEach<T>, kIn = kL < 64 ? kL : 64;
    __shared__ float2 waves[2][kThreads / 64];
    __shared__ float sums[kL <= 64 ? 2 : 1][kL <= 64 ? kL * kP * kE : 1];
    // the widest rows: the weight comes from the caches for each row, and the sums of dy lie in LDS, each thread's its own
    constexpr bool kWide = kL > 512;
    __shared__ Held<T, kWide ? 1 : kL, kWide ? 1 : kP> w;
    __shared__ Held<T, kWide ? kL : 1, kWide ? kP : 1> b;
    const int n = a.n;
    Pieces<T, kL, kTiny> at = {n, (int)threadIdx.x % kL};
    float aw[kP][kE], ab[kWide ? 1 : kP][kE];
#pragma unroll
    for (int i = 0; i < kP; i++)
#pragma unroll
        for (int j = 0; j < kE; j++) {
            aw[i][j] = 0.0f;
            if constexpr (kWide) b.v[i][j / 4][threadIdx.x][j % 4] = 0.0f;
            else ab[i][j] = 0.0f;
        }
    const int64_t hop = (int64_t)gridDim.x * kRows;
    int64_t row = (int64_t)blockIdx.x * kRows + threadIdx.x / kL;
    u32x4 x[kP], dy[kP], next_x[kP], next_dy[kP];
    float2 s = {0, 0}, next_s = {0, 0};
    auto load = [&](int64_t r) {
        if (r >= a.rows) return;
#pragma unroll
        for (int i = 0; i < kP; i++) next_x[i] = at.load((const T *)a.x + r * a.stride, i);
#pragma unroll
        for (int i = 0; i < kP; i++) next_dy[i] = at.load((const T *)a.dy + r * n, i);
        next_s = ((const float2 *)a.stats)[r];
    };
    load(row);
    if constexpr (!kWide) w.template fill<kThreads, kTiny>(a.weight, a.wide, n, 1.0f);
    __syncthreads();
    for (int turn = 0; row < a.rows; row += hop, turn ^= 1) {
        if constexpr (kWide) load(row);
#pragma unroll
        for (int i = 0; i < kP; i++) {
            x[i] = next_x[i];
            dy[i] = next_dy[i];
        }
        s = next_s;
        if constexpr (kWide) at.anew();
        else load(row + hop);
        float q1 = 0.0f, q2 = 0.0f;
#pragma unroll
        for (int i = 0; i < kP; i++) {
            float f[kE], d[kE], wf[kE];
            unpack(x[i], f, T());
            unpack(dy[i], d, T());
            if constexpr (kWide) whole_weight<T>(wf, a.weight, a.wide, at.column(i), 1.0f);
            else w.get(wf, i, at.lane);
            if (!at.whole(i)) {
#pragma unroll
                for (int j = 0; j < kE; j++) d[j] = at.own(i, j) ? d[j] : 0.0f;
            }
#pragma unroll
            for (int j = 0; j < kE; j++) {
                const float z = (f[j] - s.x) * s.y, q = wf[j] * d[j];
                aw[i][j] = __builtin_fmaf(d[j], z, aw[i][j]);
                if constexpr (kWide) b.v[i][j / 4][threadIdx.x][j % 4] += d[j];
                else ab[i][j] += d[j];
                q1 += q;
                q2 = __builtin_fmaf(q, z, q2);
            }
            __builtin_amdgcn_sched_barrier(0);     // a piece at a time, for the registers
        }
        q1 = sum_of<kIn>(q1);
        q2 = sum_of<kIn>(q2);
        if constexpr (kL > 64) {
            if (at.lane % 64 == 0) waves[turn][at.lane / 64] = make_float2(q1, q2);
            __syncthreads();
            q1 = q2 = 0.0f;
#pragma unroll
            for (int k = 0; k < kL / 64; k++) {
                q1 += waves[turn][k].x;
                q2 += waves[turn][k].y;
            }
        }
        if (!a.dx) continue;       // not before the joins: the compiler would hold all the values that they add until then
        q1 /= (float)n;
        q2 /= -(float)n;
        let_go(x);
        let_go(dy);
        if constexpr (kWide) at.anew();
        T *dx = (T *)a.dx + row * n;
#pragma unroll
        for (int i = 0; i < kP; i++) {
            float f[kE], d[kE], wf[kE];
            unpack(x[i], f, T());
            unpack(dy[i], d, T());
            if constexpr (kWide) whole_weight<T>(wf, a.weight, a.wide, at.column(i), 1.0f);
            else w.get(wf, i, at.lane);
#pragma unroll
            for (int j = 0; j < kE; j++) {
                const float z = (f[j] - s.x) * s.y;
                f[j] = __builtin_fmaf(z, q2, wf[j] * d[j] - q1) * s.y;     // the deviation last: equal q cancel wholly
            }
            at.store(dx, f, i, a.past);
            __builtin_amdgcn_sched_barrier(0);
        }
    }
    if (!part) return;
    float *out = part + (int64_t)blockIdx.x * 2 * n;
    if constexpr (kL > 64) {
#pragma unroll
        for (int i = 0; i < kP; i++)
#pragma unroll
            for (int j = 0; j < kE; j++) {
                if (!at.some(i) || !at.own(i, j)) continue;
                out[at.column(i) + j] = aw[i][j];
                if constexpr (kWide) out[n + at.column(i) + j] = b.v[i][j / 4][threadIdx.x][j % 4];
                else out[n + at.column(i) + j] = ab[i][j];
            }
    } else {
        // the wave's groups of lanes, then the waves one after the other
#pragma unroll
        for (int i = 0; i < kP; i++)
#pragma unroll
            for (int j = 0; j < kE; j++)
#pragma unroll
                for (int o = kL; o < 64; o *= 2) {
                    aw[i][j] += __shfl_xor(aw[i][j], o);
                    ab[i][j] += __shfl_xor(ab[i][j], o);
                }
        for (int k = 0; k < kThreads / 64; k++) {
            if ((int)threadIdx.x / 64 == k && (int)threadIdx.x % 64 < kL) {
#pragma unroll
                for (int i = 0; i < kP; i++)
#pragma unroll
                    for (int j = 0; j < kE; j++) {
                        if (!at.some(i) || !at.own(i, j)) continue;
                        const int c = at.column(i) + j;
                        sums[0][c] = k ? sums[0][c] + aw[i][j] : aw[i][j];
                        sums[kL <= 64][c] = k ? sums[kL <= 64][c] + ab[i][j] : ab[i][j];
                    }
            }
            __syncthreads();
        }
        for (int c = threadIdx.x; c < n; c += kThreads) {
            out[c] = sums[0][c];
            out[n + c] = sums[kL <= 64][c];
        }
    }
}

// Wider rows, in two readings. The columns' sums by workgroups of a slab of columns and every groups-th row, which also leave each
// wave's part of a row's sums of q and q z, as (rows, waves, 2); then dx by a workgroup a row, which adds those.
template <class T> __host__ __device__ constexpr int waves_of(int n) { return (n + 64 * kEach<T> - 1) / (64 * kEach<T>); }
template <class T> __global__ __launch_bounds__(1024) void norm_grad_wide_kernel(const NormGradArgs a, const float2 *given) {
    constexpr int kE = kEach<T>;
    __shared__ float lds[16];
    const int n = a.n;
    for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
        const T *x = (const T *)a.x + row * a.stride, *dy = (const T *)a.dy + row * n;
        const float2 s = ((const float2 *)a.stats)[row];
        float q1 = 0.0f, q2 = 0.0f;
        for (int i = threadIdx.x; i < waves_of<T>(n); i += 1024) {
            const float2 q = given[row * waves_of<T>(n) + i];
            q1 += q.x;
            q2 += q.y;
        }
        q1 = sum_all<1024>(q1, lds) / (float)n;
        q2 = sum_all<1024>(q2, lds) / (float)n;
        T *dx = (T *)a.dx + row * n;
        each_piece<T, 1024>(x, dy, n, [&](int c, const float *v, const float *d, int left) {
            float w[kE], f[kE];
            load_weight<T, kE>(w, a.weight, a.wide, c, n, 1.0f);
#pragma unroll
            for (int j = 0; j < kE; j++) f[j] = (w[j] * d[j] - q1 - (v[j] - s.x) * s.y * q2) * s.y;
            store_run<T, kE>(dx + c, f, left, a.past);
        });
    }
}
template <class T> __global__ __launch_bounds__(256) void norm_columns_kernel(const NormGradArgs a, float *part, int groups, float2 *given) {
    constexpr int kE = kEach<T>, kU = 4;
    const int n = a.n, g = blockIdx.x % groups, c = (blockIdx.x / groups * 256 + threadIdx.x) * kE, left = n - c;
    const int wave = blockIdx.x / groups * 4 + threadIdx.x / 64, waves = waves_of<T>(n);
    if (wave >= waves) return;      // lanes past the end go on with zeros
    float aw[kE], ab[kE], w[kE];
#pragma unroll
    for (int j = 0; j < kE; j++) aw[j] = ab[j] = 0.0f;
    load_weight<T, kE>(w, a.weight, a.wide, min(c, n - 1), n, 1.0f);
    for (int64_t first = g; first < a.rows; first += kU * (int64_t)groups) {
        u32x4 x[kU], dy[kU];
        float2 s[kU];
#pragma unroll
        for (int k = 0; k < kU; k++) {
            const int64_t row = min(first + k * (int64_t)groups, a.rows - 1);
            const T *xp = (const T *)a.x + row * a.stride, *dp = (const T *)a.dy + row * n;
            if (left >= kE) {
                x[k] = load16(xp + c);
                dy[k] = load16(dp + c);
            } else {
                x[k] = load16(xp + min(c, n), left);
                dy[k] = load16(dp + min(c, n), left);
            }
            s[k] = ((const float2 *)a.stats)[row];
        }
#pragma unroll
        for (int k = 0; k < kU; k++) {
            const int64_t row = first + k * (int64_t)groups;
            if (row >= a.rows) break;
            float v[kE], d[kE], q1 = 0.0f, q2 = 0.0f;
            unpack(x[k], v, T());
            unpack(dy[k], d, T());
#pragma unroll
            for (int j = 0; j < kE; j++) {
                const float z = (v[j] - s[k].x) * s[k].y, q = w[j] * d[j];
                aw[j] = __builtin_fmaf(d[j], z, aw[j]);
                ab[j] += d[j];
                q1 += j < left ? q : 0.0f;
                q2 += j < left ? q * z : 0.0f;
            }
            if (!given) continue;
            q1 = sum_of<64>(q1);
            q2 = sum_of<64>(q2);
            if (threadIdx.x % 64 == 0) given[row * waves + wave] = make_float2(q1, q2);
        }
    }
    if (left <= 0 || !part) return;
    float *out = part + (int64_t)g * 2 * n + c;
    store_run<float, kE>(out, aw, left);
    store_run<float, kE>(out + n, ab, left);
}

// The groups' sums of a column, 16 runs of them side by side
template <class W> __global__ __launch_bounds__(1024) void norm_join_kernel(const float *part, int groups, int n, W *dw, W *db) {
    __shared__ float sums[16][64];
    const int col = threadIdx.x % 64, run = threadIdx.x / 64;
    const int64_t c = (int64_t)blockIdx.x * 64 + col;
    float sum = 0.0f;
    if (c < 2 * (int64_t)n) {
        const int per = (groups + 15) / 16, end = min((run + 1) * per, groups);
        int g = run * per;
        for (; g + 4 <= end; g += 4) {
            float v[4];
#pragma unroll
            for (int k = 0; k < 4; k++) v[k] = part[(int64_t)(g + k) * 2 * n + c];
#pragma unroll
            for (int k = 0; k < 4; k++) sum += v[k];
        }
        for (; g < end; g++) sum += part[(int64_t)g * 2 * n + c];
    }
    sums[run][col] = sum;
    __syncthreads();
    if (run || c >= 2 * (int64_t)n) return;
#pragma unroll
    for (int k = 1; k < 16; k++) sum += sums[k][col];
    if (c < n && dw) dw[c] = from_f32<W>(sum);
    if (c >= n && db) db[c - n] = from_f32<W>(sum);
}

// The form that holds rows of n values: f(lanes, pieces, whether rows are less than a piece), or false past all of them
template <class T, class F> bool with_form(int n, F f) {
    auto is = [&](auto l, auto p, auto tiny) {
        constexpr int kL = decltype(l)::value, kP = decltype(p)::value;
        if (n > (decltype(tiny)::value ? kEach<T> - 1 : kL * kP * kEach<T>)) return false;
        f(l, p, tiny);
        return true;
    };
    constexpr std::integral_constant<int, 1> one{};
    constexpr std::integral_constant<int, 2> two{};
    constexpr std::integral_constant<int, 3> three{};
    constexpr std::integral_constant<int, 4> four{};
    constexpr std::integral_constant<int, 16> l16{};
    constexpr std::integral_constant<int, 64> l64{};
    constexpr std::integral_constant<int, 256> l256{};
    constexpr std::false_type no{};
    return is(one, one, std::true_type()) || is(one, one, no) || is(four, one, no) || is(four, two, no) || is(l16, one, no) ||
           is(l16, two, no) || is(l16, four, no) || is(l64, two, no) || is(l64, three, no) || is(l64, four, no) || is(l256, two, no) || is(l256, three, no) || is(l256, four, no);
}
// values of the widest rows that a backward pass's workgroup holds with their columns' sums: f32 in 1024 lanes, 16-bit types in 512
// (1024 by 3 pieces of those spilled: 20000 bf16 303 us, in two readings 280)
constexpr int kWidest = 16384;
bool wide_rows(int n) { return n > kWidest; }
constexpr int kFewGroups = 512;     // workgroups of a backward pass: two on each CU
int64_t groups_of(int64_t rows, int lanes) {
    const int each = lanes >= 256 ? 1 : 256 / lanes;
    return std::min<int64_t>((rows + each - 1) / each, kFewGroups);
}
template <class T> int64_t grad_groups(int64_t rows, int n) {
    int64_t g = 0;
    if (!with_form<T>(n, [&](auto l, auto, auto) { g = groups_of(rows, decltype(l)::value); }) && !wide_rows(n))
        g = std::min<int64_t>(rows, n <= 512 * 4 * kEach<T> ? kFewGroups : kFewGroups / 2);
    // the columns' kernel: a thousand workgroups or so
    if (!g) g = std::min<int64_t>(rows, std::max(1, 1024 / ((n + 256 * kEach<T> - 1) / (256 * kEach<T>))));
    return g;
}

// Short rows that end inside a cache line are written with the caches all the same, which join the lines' parts: 250 f32 116 us with
// them, 128 past them
template <class T> bool writes_past(int64_t rows, int n) {
    const int64_t row = n * (int64_t)sizeof(T);
    return rows * row >= kPastBytes && (row % 128 == 0 || row >= 4096);
}

template <class T> hipError_t go(NormArgs a, hipStream_t st) {
    a.past = writes_past<T>(a.rows, a.n);
    auto launch = [&](auto kernel, int threads, int64_t blocks, int most) {
        hipLaunchKernelGGL(kernel, dim3((unsigned)std::min<int64_t>(blocks, most)), dim3(threads), 0, st, a);
    };
    if (!with_form<T>(a.n, [&](auto l, auto p, auto tiny) {
            // as many workgroups as the weights in LDS let the CUs hold together, so that all begin and end at once
            constexpr int kL = decltype(l)::value, kRows = 256 / kL, kLds = 2 * kL * decltype(p)::value * kEach<T> * 4 + 64;
            launch(norm_kernel<T, kL, decltype(p)::value, decltype(tiny)::value>, 256, (a.rows + kRows - 1) / kRows,
                   256 * std::min(8, 160 * 1024 / kLds));
        })) {
        constexpr int kE = kEach<T>;
        if (a.n <= 512 * 3 * kE) launch(norm_kernel<T, 512, 3, false>, 512, a.rows, 512);
        else if (a.n <= 512 * 4 * kE) launch(norm_kernel<T, 512, 4, false>, 512, a.rows, 512);
        else if (a.n <= 1024 * 4 * kE) launch(norm_kernel<T, 1024, 4, false>, 1024, a.rows, 256);
        else if (a.n <= 1024 * 8 * kE) launch(norm_kernel<T, 1024, 8, false>, 1024, a.rows, 256);
        else if (a.n <= 1024 * 16 * kE) launch(norm_kernel<T, 1024, 16, false>, 1024, a.rows, 256);
        else if constexpr (sizeof(T) == 4) launch(norm_wide_kernel<T>, 1024, a.rows, 1024);     // 16-bit rows end before
    }
    return hipGetLastError();
}
template <class T> hipError_t go_grad(NormGradArgs a, void *scratch, hipStream_t st) {
    a.past = writes_past<T>(a.rows, a.n);
    const bool sums = a.dw || a.db;
    float *part = sums ? (float *)scratch : nullptr;
    const int64_t groups = grad_groups<T>(a.rows, a.n);
    if (a.rows && !with_form<T>(a.n, [&](auto l, auto p, auto tiny) {
            hipLaunchKernelGGL((norm_grad_kernel<T, decltype(l)::value, decltype(p)::value, decltype(tiny)::value>), dim3((unsigned)groups), dim3(256), 0, st,
                               a, part);
        })) {
        constexpr int kE = kEach<T>;
        if (a.n <= 512 * 4 * kE) {
            hipLaunchKernelGGL((norm_grad_kernel<T, 512, 4, false>), dim3((unsigned)groups), dim3(512), 0, st, a, part);
        } else if (sizeof(T) == 4 && !wide_rows(a.n)) {
            if constexpr (sizeof(T) == 4)
                hipLaunchKernelGGL((norm_grad_kernel<T, 1024, 4, false>), dim3((unsigned)groups), dim3(1024), 0, st, a, part);
        } else {
            const int slabs = (a.n + 256 * kE - 1) / (256 * kE);
            float2 *given = a.dx ? (float2 *)((char *)scratch + groups * 2 * a.n * 4) : nullptr;
            hipLaunchKernelGGL(norm_columns_kernel<T>, dim3((unsigned)(groups * slabs)), dim3(256), 0, st, a, part, (int)groups, given);
            if (a.dx)
                hipLaunchKernelGGL(norm_grad_wide_kernel<T>, dim3((unsigned)std::min<int64_t>(a.rows, 1024)), dim3(1024), 0, st, a,
                                   (const float2 *)given);
        }
    }
    hipError_t e = hipGetLastError();
    if (e != hipSuccess || !sums) return e;
    const unsigned blocks = (unsigned)((2 * (int64_t)a.n + 63) / 64);
    if (a.wide)
        hipLaunchKernelGGL(norm_join_kernel<float>, dim3(blocks), dim3(1024), 0, st, part, (int)groups, a.n, (float *)a.dw, (float *)a.db);
    else
        hipLaunchKernelGGL(norm_join_kernel<T>, dim3(blocks), dim3(1024), 0, st, part, (int)groups, a.n, (T *)a.dw, (T *)a.db);
    return hipGetLastError();
}

}  // namespace

template <class T> int64_t scratch_of(int64_t rows, int n) {
    return grad_groups<T>(rows, n) * 2 * n * 4 + (wide_rows(n) ? rows * waves_of<T>(n) * 8 : 0);
}
int64_t norm_grad_scratch(int type, int64_t rows, int n) {
    return type == kOpF32 ? scratch_of<float>(rows, n) : scratch_of<bf16_t>(rows, n);
}
bool norm_grad_wide(int n) { return wide_rows(n); }
hipError_t launch_norm(int type, const NormArgs &a, hipStream_t st) {
    if (type == kOpF32) return go<float>(a, st);
    if (type == kOpBf16) return go<bf16_t>(a, st);
    return go<f16_t>(a, st);
}
hipError_t launch_norm_grad(int type, const NormGradArgs &a, void *scratch, hipStream_t st) {
    if (type == kOpF32) return go_grad<float>(a, scratch, st);
    if (type == kOpBf16) return go_grad<bf16_t>(a, scratch, st);
    return go_grad<f16_t>(a, scratch, st);
}

}  // namespace ygg
