// The tiled matrix product that the output head's products share: out[i][o] = sum over r of A[i][r] B[o][r] on the matrix
// cores, a workgroup a tile of kBI rows i by kBO columns o.
//
// Either operand lies with its reduction index r contiguous ("along": the rows of x, an expert's rows) or strided ("across":
// dy and x in the weights' gradient, an expert's matrix in the rows' gradient). Both are staged through registers into LDS,
// 16 bytes a thread, a step of 128 bytes of r ("along") or as many r's ("across") at a time; the loads of a step are issued
// before the products of the step before it. Rows may begin at any address of their element's alignment (a 16-byte load of
// global memory needs no more here), and where fewer than 16 bytes are left of a row its last 16 are loaded and moved down,
// so nothing outside the operands is read.
//
// A fragment of the 16-row matrix instructions is 16 bytes a lane: lane l holds row l % 16 and the l / 16 th quarter of 64
// bytes of r. bf16 and f16 take 32 r's in one instruction, int8 64, f32 16 in four (instruction j takes the j th element of
// every quarter). The columns' operand is the instruction's first, so that a lane's results are of one row i; the columns
// of an "along" operand are dealt to pairs of fragments so that a lane has 8 consecutive ones: fragment f's j th is column
// 32 (f / 2) + 8 (l / 16) + 4 (f % 2) + j.
//
// LDS: "along" rows of 128 bytes whose 16-byte pieces are exchanged by the row's number, so that the 16 rows that a fragment
// reads at one r lie in different banks; "across" rows of all the tile's i or o at one r, 32-byte pieces exchanged likewise,
// read with the transposing 8-byte load (16-bit types) or by element (f32).
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#include <type_traits>

#include "ygg_lanes.h"
#include "ygg_optype.h"

namespace ygg {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));

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

// the column of fragment f's row d
__device__ __forceinline__ int dealt(int f, int d) { return 32 * (f >> 1) + 8 * (d >> 2) + 4 * (f & 1) + (d & 3); }

// An operand whose reduction index is contiguous: kB rows of 128 bytes a step. kRow: its fragments are 16 rows in order (the
// rows' operand), else its columns are dealt to the fragments (the columns' operand).
template <class T, int kB, int kThreads, int kF, bool kRow> struct Along {
    static constexpr int kN = kB * 8 / kThreads, kE = 16 / sizeof(T), kStep = 128 / sizeof(T), kBytes = kB * 128;
    static_assert(kN * kThreads == kB * 8, "");
    const T *p[kN];
    u32x4 v[kN];
    // the row's part of a piece's place: the 8 rows that 8 lanes read at once differ in it
    static __device__ __forceinline__ int turn(int row) {
        return kRow ? row & 7 : (row & 3) | (row >> 3 & 1) << 2;
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
            if (R >= kE) {
#pragma unroll
                for (int i = 0; i < kN; i++) v[i] = load16_end(p[i] + r0, n);
            } else {
#pragma unroll
                for (int i = 0; i < kN; i++) v[i] = load16(p[i] + r0, n);
            }
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
        const int row = base + (kRow ? 16 * f + d : dealt(f, d));
        return *(const u32x4 *)(lds + row * 128 + (((half * 4 + (l >> 4)) ^ turn(row)) << 4));
    }
};

// An operand whose reduction index is strided: kStep r's a step, kB elements each; its fragments are 16 elements in order.
template <class T, int kB, int kThreads> struct Across {
    static constexpr int kE = 16 / sizeof(T), kStep = 128 / sizeof(T), kBytes = kB * 128, kWide = kB * sizeof(T);
    static constexpr int kPer = kB / kE;             // 16-byte pieces of one r
    static constexpr int kN = kB * 8 / kThreads, kHop = kThreads / kPer;
    static_assert(kN * kThreads == kB * 8 && kHop * kPer == kThreads && kWide >= (sizeof(T) == 2 ? 128 : 256), "");
    const T *p;
    int n;              // how many elements of the thread's pieces exist
    bool inner, tiny;   // all the tile's elements exist; rows shorter than 16 bytes
    u32x4 v[kN];
    bool none[kN];
    // rows from base on, the tile's elements from `first` on of `width`
    __device__ __forceinline__ void begin(const T *base, int first, int width) {
        const int c = first + (int)threadIdx.x % kPer * kE;
        p = base + c;
        n = width - c;
        inner = first + kB <= width;
        tiny = width < kE;
    }
    // the r in the step of the thread's i th piece
    static __device__ __forceinline__ int r_of(int i) { return (int)threadIdx.x / kPer + i * kHop; }
    // offset(i): how far from r = 0 the i th piece's r lies, in elements, or -1: it counts as zero
    template <class F> __device__ __forceinline__ void load(F offset) {
        int64_t o[kN];
#pragma unroll
        for (int i = 0; i < kN; i++) o[i] = offset(i);
        if (inner) {
#pragma unroll
            for (int i = 0; i < kN; i++) v[i] = load16(p + max(o[i], (int64_t)0));
        } else if (!tiny) {
#pragma unroll
            for (int i = 0; i < kN; i++) v[i] = load16_end(p + max(o[i], (int64_t)0), n);
        } else {
#pragma unroll
            for (int i = 0; i < kN; i++) v[i] = load16(p + max(o[i], (int64_t)0), n);
        }
#pragma unroll
        for (int i = 0; i < kN; i++) none[i] = o[i] < 0;
    }
    // exchanges pieces of 32 bytes (16-bit types) or 64 (f32): the r's that one read takes together differ
    static __device__ __forceinline__ int turn(int r) {
        if constexpr (sizeof(T) == 2) return ((r & 3) | (kWide >= 256 ? (r >> 3 & 1) << 2 : 0)) << 5;
        else return (r >> 2 & 3) << 6;
    }
    __device__ __forceinline__ void store(char *lds) const {
#pragma unroll
        for (int i = 0; i < kN; i++) {
            const int r = r_of(i);
            *(u32x4 *)(lds + r * kWide + (((int)threadIdx.x % kPer * 16) ^ turn(r))) = none[i] ? u32x4{0, 0, 0, 0} : v[i];
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

// Two fragments' results, a and b, of 4 columns a group of 16 lanes each: group q gets 8 of the pair's 32 in order, 8 q .. 8 q + 7
__device__ __forceinline__ void trade(float &a, float &b) {
    u32x2 r = __builtin_bit_cast(u32x2, __builtin_amdgcn_permlane32_swap(__builtin_bit_cast(uint32_t, a), __builtin_bit_cast(uint32_t, b),
                                                                         false, false));
    r = __builtin_bit_cast(u32x2, __builtin_amdgcn_permlane16_swap(r[0], r[1], false, false));
    a = __builtin_bit_cast(float, (uint32_t)r[0]);
    b = __builtin_bit_cast(float, (uint32_t)r[1]);
}

// The lane's results, of tile row row0 + 16 i + lane % 16: put(row, column, values, count) for runs of consecutive columns.
// dealt: the columns' operand is Along, runs of 8. Otherwise a lane has 4 of a fragment's 16; stores of 4 16-bit values were
// 5 us a workgroup of 256 x 256, so there the groups of lanes trade for runs of 8.
template <class T, bool kDealt, int FI, int FO, class Acc, class F>
__device__ __forceinline__ void each_run(Acc (&acc)[FI][FO], int row0, int col0, F put) {
    static_assert(FO % 2 == 0, "");
    const int l = threadIdx.x & 63, q = l >> 4;
#pragma unroll
    for (int i = 0; i < FI; i++) {
        const int row = row0 + 16 * i + (l & 15);
        if constexpr (kDealt) {
#pragma unroll
            for (int o = 0; o < FO; o += 2) put(row, col0 + 16 * o + 8 * q, &acc[i][o], std::integral_constant<int, 8>());
        } else if constexpr (sizeof(T) == 2) {
#pragma unroll
            for (int o = 0; o < FO; o += 2) {
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    float a = acc[i][o][j], b = acc[i][o + 1][j];
                    trade(a, b);
                    acc[i][o][j] = a;
                    acc[i][o + 1][j] = b;
                }
                put(row, col0 + 16 * o + 8 * q, &acc[i][o], std::integral_constant<int, 8>());
            }
        } else {
#pragma unroll
            for (int o = 0; o < FO; o++) put(row, col0 + 16 * o + 4 * q, &acc[i][o], std::integral_constant<int, 4>());
        }
    }
}

// A workgroup's tile: WI x WO waves, each 16 FI rows by 16 FO columns, a step in LDS at a time while the next one's loads are
// on their way; the CU's other workgroups (three of four waves, by registers) fill the two barriers a step. With two steps in
// LDS and one barrier 16384 x 4096 x 4096 f16 over 8 experts took 7% longer.
template <class T, int FI, int FO, int WI, int WO, class A, class B> struct Tile {
    static constexpr int kI = 16 * FI * WI, kO = 16 * FO * WO, kThreads = 64 * WI * WO, kLds = A::kBytes + B::kBytes;
    typedef typename Mma<T>::Acc Acc;
    Acc acc[FI][FO];
    static __device__ __forceinline__ int row0() { return ((int)threadIdx.x >> 6) / WO * 16 * FI; }
    static __device__ __forceinline__ int col0() { return ((int)threadIdx.x >> 6) % WO * 16 * FO; }
    // load(step) calls a.load and b.load
    template <class F> __device__ __forceinline__ void run(A &a, B &b, char *lds, int steps, F load) {
#pragma unroll
        for (int i = 0; i < FI; i++)
#pragma unroll
            for (int o = 0; o < FO; o++) acc[i][o] = Acc{0, 0, 0, 0};
        if (steps <= 0) return;
        load(0);
        for (int t = 0; t < steps; t++) {
            __syncthreads();
            a.store(lds);
            b.store(lds + A::kBytes);
            __syncthreads();
            if (t + 1 < steps) load(t + 1);
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int half = 0; half < 2; half++) {
                u32x4 y[FO];
#pragma unroll
                for (int o = 0; o < FO; o++) y[o] = B::frag(lds + A::kBytes, col0(), o, half);
#pragma unroll
                for (int i = 0; i < FI; i++) {
                    const u32x4 x = A::frag(lds, row0(), i, half);
#pragma unroll
                    for (int o = 0; o < FO; o++) acc[i][o] = Mma<T>::run(y[o], x, acc[i][o]);
                }
            }
        }
    }
    template <bool kDealt, class F> __device__ __forceinline__ void each(F put) { each_run<T, kDealt>(acc, row0(), col0(), put); }
};

// The same product for operands whose rows are 16-byte aligned, straight from memory into LDS (no registers, no stores), for
// 16-bit types and int8.
//
// 8 waves, two a SIMD, in two groups that take turns: while one reads fragments and issues loads, the other's matrix
// instructions run; a barrier after every turn. A step of 128 bytes is two turns, half the wave's rows each, so that half the
// rows' fragments are held. Of the two LDS buffers each half operand (a region) is filled anew as soon as both groups have
// read it, two steps ahead of its use: three turns pass between a load and its first use, and no wait drains the queue.
//
//   turn 0 reads a0, b0, b1, loads a1 of the step before's place;  products a0 b0, a0 b1
//   turn 1 reads a1, loads a0, b0, b1;                             products a1 b0, a1 b1
//
// A buffer load whose lane lies past the descriptor's size brings zeros: what the reduction's end leaves of a step, and rows
// that there are not (those may bring others' values past the reduction's end: they reach no result that is stored).
//
// 256 x 256 tiles move 64 KB a step through L2 and LDS for 64 matrix instructions a wave, 1024 cycles of each SIMD's 2048: 1.35 us
// a step at the largest sizes, 1.3 PFLOP/s bf16 (16384 x 2112 x 4096) and 2.4 POP/s int8; four turns a step with a quarter of
// the tile each took 4% longer, tiles of 128 x 256 17%.
typedef uint32_t Rsrc __attribute__((ext_vector_type(4)));
__device__ __forceinline__ Rsrc rsrc_of(const void *p, uint32_t bytes) {
    const uint64_t a = (uint64_t)p;
    return Rsrc{(uint32_t)__builtin_amdgcn_readfirstlane((int)a), (uint32_t)__builtin_amdgcn_readfirstlane((int)(a >> 32)) & 0xffffu,
                (uint32_t)__builtin_amdgcn_readfirstlane((int)bytes), 0x00020000u};
}
constexpr uint32_t kFar = 0x80000000u;   // past every descriptor's size
// 16 bytes a lane to LDS from `lds` on (a wave's number: the same for all its lanes), lane after lane. The load has no output
// registers; the caller waits for it. It takes the LDS address in m0: as an operand, so that the compiler knows what m0 holds.
__device__ __forceinline__ void load_lds(Rsrc r, uint32_t offset, uint32_t lds) {
    lds = __builtin_amdgcn_readfirstlane((int)lds);
    asm volatile("s_nop 0\n\tbuffer_load_dwordx4 %0, %1, 0 offen lds" ::"v"(offset), "s"(r), "{m0}"(lds) : "memory");
}
template <int kCount> __device__ __forceinline__ void wait_loads() { asm volatile("s_waitcnt vmcnt(%0)" ::"n"(kCount) : "memory"); }
__device__ __forceinline__ void turn_over() {
    __builtin_amdgcn_sched_barrier(0);
    asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
    __builtin_amdgcn_sched_barrier(0);
}

// An operand whose reduction index is contiguous, kW wave parts of 16 kF rows each: two regions of kW * 8 kF rows of 128
// bytes, in the order of the fragments. kRow as for Along.
template <class T, int kF, int kW, bool kRow> struct AlongLds {
    static constexpr int kRows = kW * 8 * kF, kBytes = kRows * 128, kN = kRows / 64;   // loads of a region a thread
    static_assert(kF % 2 == 0 && kN * 64 == kRows, "");
    Rsrc src;
    uint32_t at[2][kN];
    int end;       // bytes of the reduction from the lane's piece on
    // offset(i): where tile row i begins, in bytes from base; bytes: of the whole operand, bytes_r: of a row
    template <class F> __device__ __forceinline__ void begin(const void *base, uint32_t bytes, int bytes_r, F offset) {
        const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, piece = ((lane & 7) ^ (lane >> 3)) * 16;
        src = rsrc_of(base, bytes);
        end = bytes_r - piece;
#pragma unroll
        for (int h = 0; h < 2; h++)
#pragma unroll
            for (int i = 0; i < kN; i++) {
                const int row = (i * 8 + wave) * 8 + (lane >> 3);
                const int part = row / (8 * kF), f = row / 16 % (kF / 2) + h * (kF / 2), d = row & 15;
                at[h][i] = offset(part * 16 * kF + (kRow ? 16 * f + d : dealt(f, d))) + piece;
            }
    }
    template <int h> __device__ __forceinline__ void load(int step, uint32_t lds) const {
        const uint32_t add = step * 128 < end ? step * 128 : kFar;
#pragma unroll
        for (int i = 0; i < kN; i++) load_lds(src, at[h][i] + add, lds + (i * 8 + (threadIdx.x >> 6)) * 1024);
    }
    // fragment f (of kF / 2) of wave part `part`
    static __device__ __forceinline__ u32x4 frag(const char *lds, int part, int f, int half) {
        const int d = threadIdx.x & 15, q = threadIdx.x >> 4 & 3;
        return *(const u32x4 *)(lds + part * (8 * kF * 128) + f * 2048 + d * 128 + (((half * 4 + q) ^ (d & 7)) << 4));
    }
};

// A 16-bit operand whose reduction index is strided: two regions of kStep r's of kW parts of 8 kF elements each
template <class T, int kF, int kW> struct AcrossLds {
    static constexpr int kWide = kW * 8 * kF * sizeof(T), kStep = 128 / sizeof(T), kBytes = kStep * kWide, kN = kBytes / 8192;
    static constexpr int kPer = 1024 / kWide;        // r's of one load of a wave
    static_assert(kN * 8192 == kBytes && kWide == 256 && sizeof(T) == 2, "");
    Rsrc src;
    uint32_t at[2];
    static __device__ __forceinline__ int turn(int r) { return Across<T, 256, 512>::turn(r); }
    // the r in the step of the thread's i th load
    static __device__ __forceinline__ int r_of(int i) {
        return (i * 8 + (int)(threadIdx.x >> 6)) * kPer + (int)(threadIdx.x & 63) / (kWide / 16);
    }
    // the tile's elements begin `left` bytes before a row's end, `first` bytes from base
    __device__ __forceinline__ void begin(const void *base, uint32_t bytes, uint32_t first, int left) {
        const int c = (((int)threadIdx.x * 16) & (kWide - 1)) ^ turn(r_of(0));    // the same for every load
        constexpr int kPart = 8 * kF * sizeof(T);
        src = rsrc_of(base, bytes);
#pragma unroll
        for (int h = 0; h < 2; h++) {
            const int col = c / kPart * 2 * kPart + h * kPart + c % kPart;
            at[h] = col < left ? first + col : kFar;
        }
    }
    // row(i): bytes from base to the row of the thread's i th r, or kFar
    template <int h, class F> __device__ __forceinline__ void load(uint32_t lds, F row) const {
#pragma unroll
        for (int i = 0; i < kN; i++) {
            const uint32_t r = row(i);
            load_lds(src, max(at[h], r) >= kFar ? kFar : at[h] + r, lds + (i * 8 + (threadIdx.x >> 6)) * 1024);
        }
    }
    static __device__ __forceinline__ u32x4 frag(const char *lds, int part, int f, int half) {
        const int l = threadIdx.x & 63, d = l & 15, q = l >> 4, base = part * 8 * kF + 16 * f;
        const int c = (base + 4 * (d & 3)) * 2;
        typedef __attribute__((address_space(3))) s16x4 *Shared;
        u32x4 v;
#pragma unroll
        for (int h = 0; h < 2; h++) {
            const int r = half * 32 + 8 * q + 4 * h + (d >> 2);
            const u32x2 x = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((Shared)(lds + r * kWide + (c ^ turn(r)))));
            v[2 * h] = x[0];
            v[2 * h + 1] = x[1];
        }
        return v;
    }
};

template <class T, int FI, int FO, int WI, int WO, class A, class B> struct TurnTile {
    static constexpr int kI = 16 * FI * WI, kO = 16 * FO * WO, kThreads = 64 * WI * WO;
    static constexpr int kBuf = 2 * (A::kBytes + B::kBytes), kLds = 2 * kBuf;
    static constexpr int kA = A::kN, kB = B::kN, kStep = 2 * (kA + kB);
    static_assert(WI * WO == 8, "");
    typedef typename Mma<T>::Acc Acc;
    Acc acc[FI][FO];
    static __device__ __forceinline__ int wave() { return __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6); }
    static __device__ __forceinline__ int row0() { return wave() / WO * 16 * FI; }
    static __device__ __forceinline__ int col0() { return wave() % WO * 16 * FO; }
    __device__ __forceinline__ void clear() {
#pragma unroll
        for (int i = 0; i < FI; i++)
#pragma unroll
            for (int o = 0; o < FO; o++) acc[i][o] = Acc{0, 0, 0, 0};
    }
    template <int i0> __device__ __forceinline__ void products(const u32x4 (&x)[2][FI / 2], const u32x4 (&y)[2][FO]) {
        __builtin_amdgcn_s_setprio(1);
#pragma unroll
        for (int half = 0; half < 2; half++)
#pragma unroll
            for (int i = 0; i < FI / 2; i++)
#pragma unroll
                for (int o = 0; o < FO; o++) acc[i0 + i][o] = Mma<T>::run(y[half][o], x[half][i], acc[i0 + i][o]);
        __builtin_amdgcn_s_setprio(0);
    }
    // lds: the workgroup's kLds bytes, at an LDS address of its own
    // load_a(half, step, LDS address) and load_b issue a region's loads, half an integral_constant; fetch(step) comes a turn
    // or more before a step's first loads, so that what they need from LDS is there. count: rows that there are, of the wave's
    // 64-row halves without any no products are taken
    template <class LA, class LB, class F>
    __device__ __forceinline__ void run(char *lds, int steps, LA load_a, LB load_b, F fetch, int count = kI) {
        typedef __attribute__((address_space(3))) char *Shared;
        const uint32_t base = __builtin_amdgcn_readfirstlane((int)(uint32_t)(uintptr_t)(Shared)lds);
        constexpr int kA0 = 0, kA1 = A::kBytes, kB0 = 2 * A::kBytes, kB1 = kB0 + B::kBytes;
        const int w = wave(), wi = w / WO, wo = w % WO;
        constexpr std::integral_constant<int, 0> k0{};
        constexpr std::integral_constant<int, 1> k1{};
        if (steps <= 0) return;
#pragma unroll
        for (int t = 0; t < 2; t++) {
            const uint32_t buf = base + t * kBuf;
            fetch(t);
            load_a(k0, t, buf + kA0);
            load_b(k0, t, buf + kB0);
            load_b(k1, t, buf + kB1);
            load_a(k1, t, buf + kA1);
        }
        wait_loads<kA + kStep>();
        turn_over();
        if (w >= 4) turn_over();
        const bool some = wi * 16 * FI < count, more = wi * 16 * FI + 8 * FI < count;
        auto turns = [&](auto all) {
            for (int t = 0; t < steps; t++) {
                const char *now = lds + (t & 1) * kBuf;
                const uint32_t buf = base + (t & 1) * kBuf;
                u32x4 x[2][FI / 2], y[2][FO];
#pragma unroll
                for (int half = 0; half < 2; half++) {
#pragma unroll
                    for (int o = 0; o < FO; o++) y[half][o] = B::frag(now + (o < FO / 2 ? kB0 : kB1), wo, o % (FO / 2), half);
#pragma unroll
                    for (int i = 0; i < FI / 2; i++) x[half][i] = A::frag(now + kA0, wi, i, half);
                }
                if (t > 0) load_a(k1, t + 1, base + (~t & 1) * kBuf + kA1);
                fetch(t + 2);
                wait_loads<kStep>();
                turn_over();
                if (decltype(all)::value || some) products<0>(x, y);
                turn_over();
#pragma unroll
                for (int half = 0; half < 2; half++)
#pragma unroll
                    for (int i = 0; i < FI / 2; i++) x[half][i] = A::frag(now + kA1, wi, i, half);
                load_a(k0, t + 2, buf + kA0);
                load_b(k0, t + 2, buf + kB0);
                load_b(k1, t + 2, buf + kB1);
                wait_loads<kStep>();
                turn_over();
                if (decltype(all)::value || more) products<FI / 2>(x, y);
                turn_over();
            }
        };
        // a loop of its own for whole tiles: the branches cost it 3%
        if (count >= kI) turns(std::true_type());
        else turns(std::false_type());
        if (w < 4) turn_over();
        wait_loads<0>();    // those of the steps past the last write LDS too
    }
    template <bool kDealt, class F> __device__ __forceinline__ void each(F put) { each_run<T, kDealt>(acc, row0(), col0(), put); }
};

// Tile t of rows x cols of them, by bands of `band` rows, down each column of a band: neighbours share both operands
struct Place {
    int row, col;
};
__device__ __forceinline__ Place place_of(int t, int rows, int cols, int band) {
    const int b = t / (band * cols), in = t - b * band * cols, high = min(band, rows - b * band);
    return {b * band + in % high, in / high};
}

}  // namespace ygg
