// The tiled matrix product that the output head's products share: out[i][o] = sum over r of A[i][r] B[o][r] on the matrix
// cores, a workgroup a tile of kBI rows i by kBO columns o.
//
// Either operand lies with its reduction index r contiguous ("along": the rows of x, an expert's rows) or strided ("across":
// dy and x in the weights' gradient, an expert's matrix in the rows' gradient). Both are staged through registers into LDS,
// 16 bytes a thread, a step of 128 bytes of r ("along") or as many r's ("across") at a time; the loads of a step are issued
// before the products of the step before it. Rows may begin at any address of their element's alignment (a 16-byte load of
// global memory needs no more here), and what a row's end or the reduction's end leaves of 16 bytes is loaded element by
// element, so nothing outside the operands is read.
//
// A fragment of the 16-row matrix instructions is 16 bytes a lane: lane l holds row l % 16 and the l / 16 th quarter of 64
// bytes of r. bf16 and f16 take 32 r's in one instruction, int8 64, f32 16 in four (instruction j takes the j th element of
// every quarter). The columns' operand is the instruction's first, so that a lane's results are of one row i; the columns
// of an "along" operand are dealt to the fragments so that a lane has 4 FO consecutive ones: column 4 FO (l / 16) + 4 f + j
// for fragment f's j th.
//
// LDS: "along" rows of 128 bytes whose 16-byte pieces are exchanged by the row's number, so that the 16 rows that a fragment
// reads at one r lie in different banks; "across" rows of all the tile's i or o at one r, 32-byte pieces exchanged likewise,
// read with the transposing 8-byte load (16-bit types) or by element (f32).
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#include <type_traits>

#include "ygg_optype.h"

namespace ygg {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));

// D += A B^T of 16 rows each: lane l's results are D's rows 4 (l / 16) + j (A's row), column l % 16 (B's row)
template <class T> struct Mma;
template <> struct Mma<bf16_t> {
    typedef f32x4 Acc;
    static __device__ __forceinline__ Acc run(u32x4 a, u32x4 b, Acc c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
    }
};
template <> struct Mma<f16_t> {
    typedef f32x4 Acc;
    static __device__ __forceinline__ Acc run(u32x4 a, u32x4 b, Acc c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
    }
};
template <> struct Mma<float> {
    typedef f32x4 Acc;
    static __device__ __forceinline__ Acc run(u32x4 a, u32x4 b, Acc c) {
        const f32x4 x = __builtin_bit_cast(f32x4, a), y = __builtin_bit_cast(f32x4, b);
#pragma unroll
        for (int j = 0; j < 4; j++) c = __builtin_amdgcn_mfma_f32_16x16x4f32(x[j], y[j], c, 0, 0, 0);
        return c;
    }
};
template <> struct Mma<int8_t> {
    typedef i32x4 Acc;
    static __device__ __forceinline__ Acc run(u32x4 a, u32x4 b, Acc c) {
        return __builtin_amdgcn_mfma_i32_16x16x64_i8(__builtin_bit_cast(i32x4, a), __builtin_bit_cast(i32x4, b), c, 0, 0, 0);
    }
};

// 16 bytes from an address of T's alignment
template <class T> __device__ __forceinline__ u32x4 load16(const T *p) {
    typedef uint32_t any __attribute__((ext_vector_type(4), aligned(1)));
    return *(const any *)p;
}
// of which the first n elements exist; the others come as zero
template <class T> __device__ __forceinline__ u32x4 load16(const T *p, int n) {
    constexpr int kE = 16 / sizeof(T);
    if (n >= kE) return load16(p);
    u32x4 v = {0, 0, 0, 0};
    if (n <= 0) return v;
    if constexpr (sizeof(T) == 4) {
#pragma unroll
        for (int j = 0; j < 3; j++)
            if (j < n) v[j] = ((const uint32_t *)p)[j];
    } else if constexpr (sizeof(T) == 2) {
#pragma unroll
        for (int j = 0; j < 7; j++)
            if (j < n) v[j / 2] |= (uint32_t)((const uint16_t *)p)[j] << 16 * (j % 2);
    } else {
#pragma unroll
        for (int j = 0; j < 15; j++)
            if (j < n) v[j / 4] |= (uint32_t)((const uint8_t *)p)[j] << 8 * (j % 4);
    }
    return v;
}

// An operand whose reduction index is contiguous: kB rows of 128 bytes a step. kRow: its fragments are 16 rows in order (the
// rows' operand), else 4 kF columns are dealt to kF fragments (the columns' operand).
template <class T, int kB, int kThreads, int kF, bool kRow> struct Along {
    static constexpr int kN = kB * 8 / kThreads, kE = 16 / sizeof(T), kStep = 128 / sizeof(T), kBytes = kB * 128;
    static_assert(kN * kThreads == kB * 8, "");
    const T *p[kN];
    u32x4 v[kN];
    // the row's part of a piece's place: the 8 rows that 8 lanes read at once differ in it
    static __device__ __forceinline__ int turn(int row) {
        if constexpr (kRow || kF == 1) return row & 7;
        else return (row & 3) | (row / (4 * kF) & 1) << 2;
    }
    // at(i): the address of tile row i's values
    template <class F> __device__ __forceinline__ void begin(F at) {
#pragma unroll
        for (int i = 0; i < kN; i++) p[i] = at((int)(threadIdx.x + i * kThreads) >> 3) + (threadIdx.x & 7) * kE;
    }
    // the step that begins at r0, of R values in all
    __device__ __forceinline__ void load(int r0, int R) {
        if (r0 + kStep <= R) {
#pragma unroll
            for (int i = 0; i < kN; i++) v[i] = load16(p[i] + r0);
        } else {
            const int n = R - r0 - (threadIdx.x & 7) * kE;
#pragma unroll
            for (int i = 0; i < kN; i++) v[i] = load16(p[i] + r0, n);
        }
    }
    __device__ __forceinline__ void store(char *lds) const {
#pragma unroll
        for (int i = 0; i < kN; i++) {
            const int row = (int)(threadIdx.x + i * kThreads) >> 3;
            *(u32x4 *)(lds + row * 128 + (((threadIdx.x & 7) ^ turn(row)) << 4)) = v[i];
        }
    }
    // fragment f of the wave's part that begins at tile row `base`; half: which 64 bytes
    static __device__ __forceinline__ u32x4 frag(const char *lds, int base, int f, int half) {
        const int l = threadIdx.x & 63, d = l & 15;
        const int row = base + (kRow ? 16 * f + d : 4 * kF * (d >> 2) + 4 * f + (d & 3));
        return *(const u32x4 *)(lds + row * 128 + (((half * 4 + (l >> 4)) ^ turn(row)) << 4));
    }
};

// An operand whose reduction index is strided: kStep r's a step, kB elements each; its fragments are 16 elements in order.
template <class T, int kB, int kThreads> struct Across {
    static constexpr int kE = 16 / sizeof(T), kStep = 128 / sizeof(T), kBytes = kB * 128, kWide = kB * sizeof(T);
    static constexpr int kPer = kB / kE;             // 16-byte pieces of one r
    static constexpr int kN = kB * 8 / kThreads, kHop = kThreads / kPer;
    static_assert(kN * kThreads == kB * 8 && kHop * kPer == kThreads && kWide >= 256, "");
    const T *p;
    int n;              // how many elements of the thread's pieces exist
    u32x4 v[kN];
    // base: the address of the tile's first element at r = 0; left: elements from there to the row's end
    __device__ __forceinline__ void begin(const T *base, int left) {
        const int c = (int)threadIdx.x % kPer * kE;
        p = base + c;
        n = left - c;
    }
    // the r in the step of the thread's i th piece
    static __device__ __forceinline__ int r_of(int i) { return (int)threadIdx.x / kPer + i * kHop; }
    // offset(i): how far from r = 0 the i th piece's r lies, in elements, or -1: it counts as zero
    template <class F> __device__ __forceinline__ void load(F offset) {
#pragma unroll
        for (int i = 0; i < kN; i++) {
            const int64_t o = offset(i);
            v[i] = load16(p + (o < 0 ? 0 : o), o < 0 ? 0 : n);
        }
    }
    // exchanges pieces of 32 bytes (16-bit types) or 64 (f32): the r's that one read takes together differ
    static __device__ __forceinline__ int turn(int r) {
        if constexpr (sizeof(T) == 2) return ((r & 3) | (r >> 3 & 1) << 2) << 5;
        else return (r >> 2 & 3) << 6;
    }
    __device__ __forceinline__ void store(char *lds) const {
#pragma unroll
        for (int i = 0; i < kN; i++) {
            const int r = r_of(i);
            *(u32x4 *)(lds + r * kWide + (((int)threadIdx.x % kPer * 16) ^ turn(r))) = v[i];
        }
    }
    static __device__ __forceinline__ u32x4 frag(const char *lds, int base, int f, int half) {
        const int l = threadIdx.x & 63, d = l & 15, q = l >> 4;
        u32x4 v;
        if constexpr (sizeof(T) == 2) {
            // the transposing load: lane d of 16 gives the address of 4 elements at r = d / 4, and gets element d of four r's
            typedef __attribute__((address_space(3))) s16x4 *Shared;
            const int c = (base + 16 * f + 4 * (d & 3)) * 2;
#pragma unroll
            for (int h = 0; h < 2; h++) {
                const int r = half * 32 + 8 * q + 4 * h + (d >> 2);
                const u32x2 x = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((Shared)(lds + r * kWide + (c ^ turn(r)))));
                v[2 * h] = x[0];
                v[2 * h + 1] = x[1];
            }
        } else {
            const int c = (base + 16 * f + d) * 4;
#pragma unroll
            for (int j = 0; j < 4; j++) {
                const int r = half * 16 + 4 * q + j;
                v[j] = *(const uint32_t *)(lds + r * kWide + (c ^ turn(r)));
            }
        }
        return v;
    }
};

// A workgroup's tile: WI x WO waves, each 16 FI rows by 16 FO columns. a.load and b.load are called by load(step); kBufs 2:
// a step is stored while the one before it is read, one barrier a step and twice the LDS; 1: two barriers, and other
// workgroups of the CU work meanwhile.
template <class T, int FI, int FO, int WI, int WO, int kBufs, class A, class B> struct Tile {
    static constexpr int kI = 16 * FI * WI, kO = 16 * FO * WO, kThreads = 64 * WI * WO;
    static constexpr int kLds = kBufs * (A::kBytes + B::kBytes);
    typedef typename Mma<T>::Acc Acc;
    Acc acc[FI][FO];
    static __device__ __forceinline__ int row0() { return ((int)threadIdx.x >> 6) / WO * 16 * FI; }
    static __device__ __forceinline__ int col0() { return ((int)threadIdx.x >> 6) % WO * 16 * FO; }
    __device__ __forceinline__ void products(const char *a, const char *b) {
#pragma unroll
        for (int half = 0; half < 2; half++) {
            u32x4 y[FO];
#pragma unroll
            for (int o = 0; o < FO; o++) y[o] = B::frag(b, col0(), o, half);
#pragma unroll
            for (int i = 0; i < FI; i++) {
                const u32x4 x = A::frag(a, row0(), i, half);
#pragma unroll
                for (int o = 0; o < FO; o++) acc[i][o] = Mma<T>::run(y[o], x, acc[i][o]);
            }
        }
    }
    template <class F> __device__ __forceinline__ void run(A &a, B &b, char *lds, int steps, F load) {
#pragma unroll
        for (int i = 0; i < FI; i++)
#pragma unroll
            for (int o = 0; o < FO; o++) acc[i][o] = Acc{0, 0, 0, 0};
        if (steps <= 0) return;
        load(0);
        if constexpr (kBufs == 1) {
            for (int t = 0; t < steps; t++) {
                __syncthreads();
                a.store(lds);
                b.store(lds + A::kBytes);
                __syncthreads();
                if (t + 1 < steps) load(t + 1);
                __builtin_amdgcn_sched_barrier(0);
                products(lds, lds + A::kBytes);
            }
        } else {
            a.store(lds);
            b.store(lds + A::kBytes);
            __syncthreads();
            for (int t = 0; t < steps; t++) {
                if (t + 1 < steps) load(t + 1);
                __builtin_amdgcn_sched_barrier(0);
                const char *now = lds + (t & 1) * (A::kBytes + B::kBytes);
                products(now, now + A::kBytes);
                __builtin_amdgcn_sched_barrier(0);
                if (t + 1 < steps) {
                    char *next = lds + (~t & 1) * (A::kBytes + B::kBytes);
                    a.store(next);
                    b.store(next + A::kBytes);
                }
                __syncthreads();
            }
        }
    }
    // The lane's results: of tile row row0() + 16 i + lane % 16, runs of consecutive columns. put(row, column, values, count)
    // for each; dealt: the columns' operand is Along.
    template <bool kDealt, class F> __device__ __forceinline__ void each(F put) const {
        const int l = threadIdx.x & 63;
#pragma unroll
        for (int i = 0; i < FI; i++) {
            const int row = row0() + 16 * i + (l & 15);
            if constexpr (kDealt) {
                put(row, col0() + 4 * FO * (l >> 4), &acc[i][0], std::integral_constant<int, 4 * FO>());
            } else {
#pragma unroll
                for (int o = 0; o < FO; o++) put(row, col0() + 16 * o + 4 * (l >> 4), &acc[i][o], std::integral_constant<int, 4>());
            }
        }
    }
};

// kN consecutive values rounded to T at an address of T's alignment, of which the first `left` exist
template <class T, int kN, class V> __device__ __forceinline__ void store_run(T *p, const V *v, int left) {
    constexpr int kE = kN * sizeof(T) < 16 ? kN : 16 / sizeof(T);
    typedef uint32_t any __attribute__((ext_vector_type(kE * sizeof(T) / 4), aligned(1)));
    if (left >= kN) {
#pragma unroll
        for (int k = 0; k < kN; k += kE) {
            T t[kE];
#pragma unroll
            for (int j = 0; j < kE; j++) t[j] = from_f32<T>(v[k + j]);
            any a;
            __builtin_memcpy(&a, t, sizeof(a));
            *(any *)(p + k) = a;
        }
    } else {
#pragma unroll
        for (int k = 0; k < kN; k++)
            if (k < left) p[k] = from_f32<T>(v[k]);
    }
}

// Workgroups go round the 8 XCDs in turn, each with an L2 of its own: a run of neighbouring tiles to each
__device__ __forceinline__ int tile_of(int id, int tiles) {
    const int most = (tiles + 7) / 8, full = tiles - (most - 1) * 8;   // the first `full` XCDs have `most`
    const int x = id & 7;
    return (x < full ? x * most : full * most + (x - full) * (most - 1)) + (id >> 3);
}

}  // namespace ygg
