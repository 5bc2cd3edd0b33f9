// The gated recurrence h_t = a_t h_{t-1} + x_t of every channel, over long sequences, and its gradients
//   e_t = dh_t + a_{t+1} e_{t+1} (of the last step with the final state's gradient),  dx_t = e_t,  da_t = e_t h_{t-1},
//   dstate = a_0 e_0.
//
// A run of steps maps the state before it to the one after it, h -> A h + H with A the product of its gates and H its result from
// zero; two runs join to (A2 A1, A2 H1 + H2). A workgroup takes a slab of kCols groups of channels, 16 or 8 bytes of gates each, and goes
// through time by chunks of kParts parts: each thread holds a part, kSteps steps, in registers, so that its loads are all in flight
// together and values are read once; the four parts of a wave are joined by exchanging its rows of lanes, the waves' maps in LDS,
// and each thread then computes its steps again from the state it begins with. (With all 16 parts' maps in LDS the backward pass of
// 16 x 4096 x 2048 bf16 took 338 us, 276 like this: each thread read them all.) The next chunk's loads are issued before that.
//
// The backward pass is the same from the end: f_t = a_t e_t is what step t hands to the one before, e_t = dh_t + f_{t+1}. da wants
// h_{t-1} in f32, and the h that went out is rounded to its type: so the forward pass leaves the state before every kKeep-th step
// (1/64 of the values, in f32), and the backward pass computes a chunk's states again from it and from x, which reads as much as h
// would. (From h: 268 us, and the gates' gradient off by a rounding of h.)
//
// Where the slabs are too few for the chip, time is cut into segments too: a first kernel takes the map of each, and
// every workgroup of the second joins those before its own. That reads the gates and x (or dh) twice, so the second kernel goes
// through the segments from the last one, whose values the memory's cache still holds, and neighbouring segments are one XCD's.
// States, maps and their joins are in f32; h, dx and da are rounded to their types once, on the way out.
//
// The memory bounds it. 16 x 4096 x 2048 bf16: forward 155 us (2 readings and a writing of 268 MB, 5.2 TB/s), backward 273 us (3 and
// 2, 4.9 TB/s); 131072 x 256 bf16 with gates in f32: 30 us for the segments' maps, 44 for the states. Workgroups of 512 threads
// (295 us backward) and of half as many channels (300) were slower.
#include <algorithm>

#include "ygg_lanes.h"
#include "ygg_ops.h"
#include "ygg_optype.h"

namespace ygg {
namespace {

// kV consecutive values as they lie in memory, in words: of 16-bit values by themselves the compiler gives each a register
template <class T, int kV> struct Few {
    static constexpr int kW = (kV * (int)sizeof(T) + 3) / 4;
    typedef uint32_t any __attribute__((ext_vector_type(kW), aligned(1)));
    uint32_t w[kW];
    __device__ __forceinline__ float operator[](int j) const {
        if constexpr (sizeof(T) == 4) return __builtin_bit_cast(float, w[j]);
        else return to_f32(__builtin_bit_cast(T, (uint16_t)(w[j / 2] >> 16 * (j % 2))));
    }
    __device__ __forceinline__ void set(const float *f) {
        if constexpr (sizeof(T) == 4) {
#pragma unroll
            for (int j = 0; j < kV; j++) w[j] = __builtin_bit_cast(uint32_t, f[j]);
        } else {
#pragma unroll
            for (int j = 0; j < kW; j++) w[j] = 0;
#pragma unroll
            for (int j = 0; j < kV; j++) w[j / 2] |= half_of(f[j]) << 16 * (j % 2);
        }
    }
    __device__ __forceinline__ static uint32_t half_of(float v) {
        if constexpr (sizeof(T) == 2) return __builtin_bit_cast(uint16_t, from_f32<T>(v));
        return 0;
    }
    __device__ __forceinline__ void load(const T *p) {
        if constexpr (kV == 1 && sizeof(T) == 2) {
            w[0] = __builtin_bit_cast(uint16_t, *p);
        } else {
            const any a = *(const any *)p;
            __builtin_memcpy(w, &a, sizeof(w));
        }
    }
    __device__ __forceinline__ void store(T *p, bool past) const {
        if constexpr (kV == 1 && sizeof(T) == 2) {
            *p = __builtin_bit_cast(T, (uint16_t)w[0]);
        } else {
            any a;
            __builtin_memcpy(&a, w, sizeof(w));
            if (past) store_past(a, p);
            else *(any *)p = a;
        }
    }
    // `other` in the place of each
    __device__ __forceinline__ void fill(float other) {
        const uint32_t one = sizeof(T) == 4 ? __builtin_bit_cast(uint32_t, other) : half_of(other) * 0x10001u;
#pragma unroll
        for (int j = 0; j < kW; j++) w[j] = one;
    }
    __device__ __forceinline__ void fill_unless(bool is, float other) {
        Few f;
        f.fill(other);
#pragma unroll
        for (int j = 0; j < kW; j++) w[j] = is ? w[j] : f.w[j];
    }
    // what was made of these before is not held until it is wanted again, but made again: unpacked to f32 they take twice the registers
    __device__ __forceinline__ void let_go() {
        if constexpr (sizeof(T) == 2) {
#pragma unroll
            for (int j = 0; j < kW; j++) asm volatile("" : "+v"(w[j]));
        }
    }
};

// p + at, computed anew in each turn of a loop: the addresses of all steps and tensors, which the compiler would carry on from turn to
// turn, held more registers than the values
template <class T> __device__ __forceinline__ T *anew(T *p, int64_t at) {
    asm volatile("" : "+v"(at));
    return p + at;
}

// a workgroup's threads: 16 channels or groups of them by 16 parts, a row of lanes each
constexpr int kCols = 16, kParts = 16, kWaves = kCols * kParts / 64;

// A thread's channels: the last ones of a row that they do not fill begin earlier, and compute some a second time
template <int kV> struct Place {
    int64_t b;
    int c, part;
    bool some;
    __device__ __forceinline__ static Place of(int64_t slab, int slabs, int n) {
        const int col = (int)(slab % slabs * kCols) + (int)threadIdx.x % kCols;
        return {slab / slabs, max(min(col * kV, n - kV), 0), (int)threadIdx.x / kCols, col * kV < n};
    }
};
// The values of a wave's rows 0 and 1 in its first half, of 2 and 3 in its second, in all lanes; and those of its halves
struct Two {
    float lo, hi;
};
__device__ __forceinline__ Two of_rows(float v) {
    const uint32_t b = __builtin_bit_cast(uint32_t, v);
    const auto r = __builtin_amdgcn_permlane16_swap(b, b, false, false);
    return {__builtin_bit_cast(float, (uint32_t)r[0]), __builtin_bit_cast(float, (uint32_t)r[1])};
}
__device__ __forceinline__ Two of_halves(float v) {
    const uint32_t b = __builtin_bit_cast(uint32_t, v);
    const auto r = __builtin_amdgcn_permlane32_swap(b, b, false, false);
    return {__builtin_bit_cast(float, (uint32_t)r[0]), __builtin_bit_cast(float, (uint32_t)r[1])};
}
// A map of each part of a wave: of the parts before a lane's own (A, H), and of all of them (all_A, all_H). kAfter: also of maps B
// with the same products that go the other way, (after_A, after_B) those of the parts after it and all_B.
template <bool kAfter> struct Scan {
    float A, H, all_A, all_H, after_A, after_B, all_B;
    __device__ __forceinline__ Scan(float a, float h, float b) {
        const bool odd = threadIdx.x & 16, high = threadIdx.x & 32;
        Two ta = of_rows(a), th = of_rows(h), tb = {0.0f, 0.0f};
        A = odd ? ta.lo : 1.0f;
        H = odd ? th.lo : 0.0f;
        all_H = __builtin_fmaf(ta.hi, th.lo, th.hi);
        if constexpr (kAfter) {
            tb = of_rows(b);
            after_A = odd ? 1.0f : ta.hi;
            after_B = odd ? 0.0f : tb.hi;
            all_B = __builtin_fmaf(ta.lo, tb.hi, tb.lo);
        }
        ta = of_halves(ta.lo * ta.hi);
        th = of_halves(all_H);
        H = __builtin_fmaf(A, high ? th.lo : 0.0f, H);
        A *= high ? ta.lo : 1.0f;
        all_A = ta.lo * ta.hi;
        all_H = __builtin_fmaf(ta.hi, th.lo, th.hi);
        if constexpr (kAfter) {
            tb = of_halves(all_B);
            after_B = __builtin_fmaf(after_A, high ? 0.0f : tb.hi, after_B);
            after_A *= high ? 1.0f : ta.hi;
            all_B = __builtin_fmaf(ta.lo, tb.hi, tb.lo);
        }
    }
};
// The waves' maps, in LDS
template <int kV> struct Maps {
    float v[kWaves][kCols * kV];
    __device__ __forceinline__ void put(int j, float f) {
        if (threadIdx.x % 64 < kCols) v[threadIdx.x / 64][threadIdx.x % kCols * kV + j] = f;
    }
    __device__ __forceinline__ float get(int wave, int j) const { return v[wave][threadIdx.x % kCols * kV + j]; }
};
// carry: what the chunk begins with, then what it ends with; in: what the wave begins with. kBack: the waves in the other order
template <bool kBack, int kV> __device__ __forceinline__ void join_waves(const Maps<kV> &a, const Maps<kV> &h, float *carry, float *in) {
    const int wave = threadIdx.x / 64;
#pragma unroll
    for (int i = 0; i < kWaves; i++) {
        const int q = kBack ? kWaves - 1 - i : i;
#pragma unroll
        for (int j = 0; j < kV; j++) {
            in[j] = q == wave ? carry[j] : in[j];
            carry[j] = __builtin_fmaf(a.get(q, j), carry[j], h.get(q, j));
        }
    }
}
// carry: what the first segment begins with, then what the one after the `count` of these maps does. The maps lie `hop` values apart; each
// part takes its share of them, side by side, and the parts are joined as those of a chunk (one after the other those of 131072 x 256
// took 5 us longer)
template <int kV>
__device__ __forceinline__ void join_segments(const float *maps, int64_t hop, int n, int count, Maps<kV> &lds_a, Maps<kV> &lds_h, float *carry) {
    if (count == 0) return;
    const int per = (count + kParts - 1) / kParts, first = threadIdx.x / kCols * per, end = min(first + per, count);
    float A[kV], H[kV], in[kV];
#pragma unroll
    for (int j = 0; j < kV; j++) A[j] = 1.0f, H[j] = 0.0f;
#pragma unroll 4
    for (int s = first; s < end; s++) {
        Few<float, kV> a, h;
        a.load(maps + s * hop);
        h.load(maps + s * hop + n);
#pragma unroll
        for (int j = 0; j < kV; j++) {
            H[j] = __builtin_fmaf(a[j], H[j], h[j]);
            A[j] *= a[j];
        }
    }
#pragma unroll
    for (int j = 0; j < kV; j++) {
        const Scan<false> w(A[j], H[j], 0.0f);
        lds_a.put(j, w.all_A);
        lds_h.put(j, w.all_H);
    }
    __syncthreads();
    join_waves<false>(lds_a, lds_h, carry, in);
}

// How a call is cut: `slabs` of a sequence, `segments` of `per` steps each
struct Cut {
    int slabs, segments;
    int64_t per, steps;     // steps: all, up to whole chunks
};

// the maps of the segments, (B, segments, 2, n): each part goes through its share of the segment by itself. kBack: time runs
// backwards (places and segments count from the end of the last chunk, place i is step cut.steps - 1 - i), the map is that of f
// from dh.
template <class TX, class TG, int kV, int kSteps, bool kBack>
__global__ __launch_bounds__(kCols *kParts) void segment_kernel(const TG *gate, const TX *x, int64_t gate_b, int64_t gate_t, int64_t x_b,
                                                                int64_t x_t, int64_t T, int n, Cut cut, float *maps) {
    __shared__ Maps<kV> lds_a, lds_h;
    const int s = blockIdx.x % (cut.segments - 1);     // nobody asks for the last one's
    const Place<kV> at = Place<kV>::of(blockIdx.x / (cut.segments - 1), cut.slabs, n);
    const int64_t from = s * cut.per, share = cut.per / kParts;      // a segment that is not the last is whole
    const TG *g = gate + at.b * gate_b + at.c;
    const TX *xp = x ? x + at.b * x_b + at.c : nullptr;
    auto step = [&](int64_t i) { return kBack ? cut.steps - 1 - i : i; };
    float A[kV], H[kV];
#pragma unroll
    for (int j = 0; j < kV; j++) A[j] = 1.0f, H[j] = 0.0f;
    int64_t i = from + at.part * share;
    const int64_t end = i + share;
    for (; i < end; i += kSteps) {     // share is a multiple of kSteps
        Few<TG, kV> a[kSteps];
        Few<TX, kV> v[kSteps];
        const int64_t top = kBack ? min(step(i), T - 1) : i;
        const int less = kBack ? (int)min(step(i) - top, (int64_t)kSteps) : 0;     // the first ones are none
        const TG *gp = anew(g, top * gate_t);
        const TX *vp = anew(xp, top * x_t);
#pragma unroll
        for (int k = 0; k < kSteps; k++) {
            const int hop = kBack ? -max(k - less, 0) : k;
            a[k].load(gp + hop * gate_t);
            if (xp) v[k].load(vp + hop * x_t);
            else v[k].fill(0.0f);
            if (kBack) {
                a[k].fill_unless(k >= less, 1.0f);
                v[k].fill_unless(k >= less, 0.0f);
            }
        }
#pragma unroll
        for (int k = 0; k < kSteps; k++)
#pragma unroll
            for (int j = 0; j < kV; j++) {
                const float gt = a[k][j], xt = v[k][j];
                H[j] = kBack ? gt * (xt + H[j]) : __builtin_fmaf(gt, H[j], xt);
                A[j] *= gt;
            }
    }
#pragma unroll
    for (int j = 0; j < kV; j++) {
        const Scan<false> w(A[j], H[j], 0.0f);
        lds_a.put(j, w.all_A);
        lds_h.put(j, w.all_H);
    }
    __syncthreads();
    if (at.part || !at.some) return;
    float all_A[kV], all_H[kV];
#pragma unroll
    for (int j = 0; j < kV; j++) all_A[j] = lds_a.get(0, j), all_H[j] = lds_h.get(0, j);
#pragma unroll
    for (int q = 1; q < kWaves; q++)
#pragma unroll
        for (int j = 0; j < kV; j++) {
            all_H[j] = __builtin_fmaf(lds_a.get(q, j), all_H[j], lds_h.get(q, j));
            all_A[j] *= lds_a.get(q, j);
        }
    float *out = maps + (at.b * cut.segments + s) * 2 * n + at.c;
#pragma unroll
    for (int j = 0; j < kV; j++) {
        out[j] = all_A[j];
        out[n + j] = all_H[j];
    }
}

constexpr int kKeep = 64;      // steps from one state that is kept to the next
__host__ __device__ constexpr int64_t kept_of(int64_t T) { return T > 0 ? (T - 1) / kKeep : 0; }

template <class TX, class TG, int kV, int kSteps>
__global__ __launch_bounds__(kCols *kParts, 2) void scan_kernel(const ScanArgs a, Cut cut, const float *maps) {
    constexpr int kChunk = kParts * kSteps;
    __shared__ Maps<kV> lds_a[2], lds_h[2];
    const int id = gridDim.x - 1 - tile_of(blockIdx.x, gridDim.x), s = id % cut.segments, n = a.n;
    const Place<kV> at = Place<kV>::of(id / cut.segments, cut.slabs, n);
    const int64_t from = s * cut.per, end = min(from + cut.per, a.T);
    const TG *g = (const TG *)a.gate + at.b * a.gate_b + at.c;
    const TX *x = (const TX *)a.x + at.b * a.x_b + at.c;
    TX *h = (TX *)a.h + at.b * a.T * n + at.c;
    Few<TG, kV> ga[kSteps], next_g[kSteps];
    Few<TX, kV> xa[kSteps], next_x[kSteps];
    auto load = [&](int64_t chunk) {
        const int64_t first = min(chunk + at.part * kSteps, end - 1);
        const int left = (int)min(end - 1 - first, (int64_t)kSteps);
        const TG *gp = anew(g, first * a.gate_t);
        const TX *xp = anew(x, first * a.x_t);
#pragma unroll
        for (int k = 0; k < kSteps; k++) {
            next_g[k].load(gp + min(k, left) * a.gate_t);
            next_x[k].load(xp + min(k, left) * a.x_t);
        }
    };
    load(from);
    float carry[kV];
#pragma unroll
    for (int j = 0; j < kV; j++) carry[j] = a.state ? a.state[at.b * n + at.c + j] : 0.0f;
    join_segments<kV>(maps + at.b * cut.segments * 2 * n + at.c, 2 * n, n, s, lds_a[1], lds_h[1], carry);     // the chunks begin with [0]
    int buf = 0;
    for (int64_t chunk = from; chunk < end; chunk += kChunk, buf ^= 1) {
        const int64_t t0 = chunk + at.part * kSteps;
#pragma unroll
        for (int k = 0; k < kSteps; k++) {
            ga[k] = next_g[k];
            xa[k] = next_x[k];
            ga[k].fill_unless(t0 + k < end, 1.0f);     // steps past the end change nothing
            xa[k].fill_unless(t0 + k < end, 0.0f);
        }
        if (chunk + kChunk < end) load(chunk + kChunk);
        float A[kV], H[kV];
#pragma unroll
        for (int j = 0; j < kV; j++) A[j] = 1.0f, H[j] = 0.0f;
#pragma unroll
        for (int k = 0; k < kSteps; k++)
#pragma unroll
            for (int j = 0; j < kV; j++) {
                H[j] = __builtin_fmaf(ga[k][j], H[j], xa[k][j]);
                A[j] *= ga[k][j];
            }
#pragma unroll
        for (int j = 0; j < kV; j++) {
            const Scan<false> w(A[j], H[j], 0.0f);
            A[j] = w.A, H[j] = w.H;
            lds_a[buf].put(j, w.all_A);
            lds_h[buf].put(j, w.all_H);
        }
        __syncthreads();
        float in[kV];
        join_waves<false>(lds_a[buf], lds_h[buf], carry, in);
#pragma unroll
        for (int j = 0; j < kV; j++) in[j] = __builtin_fmaf(A[j], in[j], H[j]);
#pragma unroll
        for (int k = 0; k < kSteps; k++) {
            ga[k].let_go();
            xa[k].let_go();
        }
        if (a.kept && t0 % kKeep == 0 && t0 > 0 && t0 < end && at.some) {
            Few<float, kV> out;
            out.set(in);
            out.store(a.kept + (at.b * kept_of(a.T) + t0 / kKeep - 1) * n + at.c, false);
        }
        TX *to = anew(h, t0 * n);
#pragma unroll
        for (int k = 0; k < kSteps; k++) {
            Few<TX, kV> out;
#pragma unroll
            for (int j = 0; j < kV; j++) in[j] = __builtin_fmaf(ga[k][j], in[j], xa[k][j]);
            out.set(in);
            if (at.some && t0 + k < end) out.store(to + (int64_t)k * n, a.past);
        }
    }
    if (s == cut.segments - 1 && at.part == 0 && at.some) {
#pragma unroll
        for (int j = 0; j < kV; j++) a.last[at.b * n + at.c + j] = carry[j];
    }
}

// Few steps: a thread takes its channels through all of them
template <class TX, class TG, int kV> __global__ __launch_bounds__(256) void step_kernel(const ScanArgs a) {
    const int n = a.n, cols = (n + kV - 1) / kV;
    const int64_t id = (int64_t)blockIdx.x * 256 + threadIdx.x, b = id / cols;
    if (b >= a.B) return;
    const int c = max(min((int)(id % cols) * kV, n - kV), 0);
    const TG *g = (const TG *)a.gate + b * a.gate_b + c;
    const TX *x = (const TX *)a.x + b * a.x_b + c;
    TX *h = (TX *)a.h + b * a.T * n + c;
    float s[kV];
#pragma unroll
    for (int j = 0; j < kV; j++) s[j] = a.state ? a.state[b * n + c + j] : 0.0f;
    for (int64_t t = 0; t < a.T; t++) {
        Few<TG, kV> gt;
        Few<TX, kV> xt, out;
        gt.load(g + t * a.gate_t);
        xt.load(x + t * a.x_t);
#pragma unroll
        for (int j = 0; j < kV; j++) s[j] = __builtin_fmaf(gt[j], s[j], xt[j]);
        out.set(s);
        out.store(h + t * n, false);
    }
#pragma unroll
    for (int j = 0; j < kV; j++) a.last[b * n + c + j] = s[j];
}

// backward; places count from the end of the last chunk: place i is step cut.steps - 1 - i, and the first ones may be none
// kGate: the gates' gradient is wanted
template <class TX, class TG, int kV, int kSteps, bool kGate>
__global__ __launch_bounds__(kCols *kParts, 2) void scan_grad_kernel(const ScanGradArgs a, Cut cut, const float *maps) {
    constexpr int kChunk = kParts * kSteps;
    static_assert(kChunk % kKeep == 0, "a chunk begins where a state is kept");
    __shared__ Maps<kV> lds_a[2], lds_f[2], lds_h[2];      // lds_h: of the states, with the same products of gates
    const int id = gridDim.x - 1 - tile_of(blockIdx.x, gridDim.x), s = id % cut.segments, n = a.n;
    const Place<kV> at = Place<kV>::of(id / cut.segments, cut.slabs, n);
    const int64_t T = a.T, from = s * cut.per, end = min(from + cut.per, cut.steps), row = at.b * T * n + at.c;
    const TG *g = (const TG *)a.gate + at.b * a.gate_b + at.c;
    const TX *dh = a.dh ? (const TX *)a.dh + row : nullptr, *x = kGate ? (const TX *)a.x + at.b * a.x_b + at.c : nullptr;
    TX *dx = a.dx ? (TX *)a.dx + row : nullptr;
    TG *dg = kGate ? (TG *)a.dgate + row : nullptr;
    const float *first = a.state ? a.state + at.b * n + at.c : nullptr;
    float carry[kV];     // what the steps after this chunk hand to it
#pragma unroll
    for (int j = 0; j < kV; j++) carry[j] = a.dlast ? a.dlast[at.b * n + at.c + j] : 0.0f;
    Few<TG, kV> ga[kSteps], next_g[kSteps];
    Few<TX, kV> da[kSteps], next_d[kSteps], xa[kSteps], next_x[kSteps];
    Few<float, kV> begin, next_b;        // the state before a chunk's first step
#pragma unroll
    for (int k = 0; k < kSteps; k++) next_d[k].fill(0.0f);
    auto load = [&](int64_t chunk) {
        const int64_t t0 = cut.steps - 1 - (chunk + at.part * kSteps), top = min(t0, T - 1);
        const int less = (int)min(t0 - top, (int64_t)kSteps);    // the step of k is top - (k - less), the first `less` ones are none
        const TG *gp = anew(g, top * a.gate_t);
#pragma unroll
        for (int k = 0; k < kSteps; k++) next_g[k].load(gp - max(k - less, 0) * a.gate_t);
        if (dh) {
            const TX *dp = anew(dh, top * n);
#pragma unroll
            for (int k = 0; k < kSteps; k++) next_d[k].load(dp - (int64_t)max(k - less, 0) * n);
        }
        if constexpr (kGate) {
            const TX *xp = anew(x, top * a.x_t);
#pragma unroll
            for (int k = 0; k < kSteps; k++) next_x[k].load(xp - max(k - less, 0) * a.x_t);
            const int64_t before = (cut.steps - chunk) / kChunk - 1;    // chunks
            const float *p = before ? a.kept + (at.b * kept_of(T) + before * (kChunk / kKeep) - 1) * n + at.c : first;
            if (p) next_b.load(p);
            else next_b.fill(0.0f);
        }
    };
    if (from < end) load(from);     // there may be no step at all
    join_segments<kV>(maps + at.b * cut.segments * 2 * n + at.c, 2 * n, n, s, lds_a[1], lds_f[1], carry);
    int buf = 0;
    for (int64_t chunk = from; chunk < end; chunk += kChunk, buf ^= 1) {
        const int64_t t0 = cut.steps - 1 - (chunk + at.part * kSteps);     // the step of k is t0 - k
#pragma unroll
        for (int k = 0; k < kSteps; k++) {
            ga[k] = next_g[k];
            da[k] = next_d[k];
            xa[k] = next_x[k];
            ga[k].fill_unless(t0 - k < T, 1.0f);       // steps that there are not change nothing
            da[k].fill_unless(t0 - k < T, 0.0f);
        }
        begin = next_b;
        if (chunk + kChunk < end) load(chunk + kChunk);
        float A[kV], F[kV], H[kV];
#pragma unroll
        for (int j = 0; j < kV; j++) A[j] = 1.0f, F[j] = 0.0f, H[j] = 0.0f;
#pragma unroll
        for (int k = 0; k < kSteps; k++)
#pragma unroll
            for (int j = 0; j < kV; j++) {
                F[j] = ga[k][j] * (da[k][j] + F[j]);
                A[j] *= ga[k][j];
            }
        if constexpr (kGate) {
            // steps that there are not come after all others: what they make of the states, nobody asks for
#pragma unroll
            for (int k = kSteps - 1; k >= 0; k--)
#pragma unroll
                for (int j = 0; j < kV; j++) H[j] = __builtin_fmaf(ga[k][j], H[j], xa[k][j]);
        }
        float after_A[kV];
#pragma unroll
        for (int j = 0; j < kV; j++) {
            const Scan<kGate> w(A[j], F[j], H[j]);
            A[j] = w.A, F[j] = w.H;
            lds_a[buf].put(j, w.all_A);
            lds_f[buf].put(j, w.all_H);
            if constexpr (kGate) {
                after_A[j] = w.after_A, H[j] = w.after_B;
                lds_h[buf].put(j, w.all_B);
            }
        }
        __syncthreads();
        float f[kV], before[kSteps][kV];
        join_waves<false>(lds_a[buf], lds_f[buf], carry, f);
#pragma unroll
        for (int j = 0; j < kV; j++) f[j] = __builtin_fmaf(A[j], f[j], F[j]);
#pragma unroll
        for (int k = 0; k < kSteps; k++) {
            ga[k].let_go();
            da[k].let_go();
            xa[k].let_go();
        }
        if constexpr (kGate) {
            float h[kV], state[kV];
#pragma unroll
            for (int j = 0; j < kV; j++) state[j] = begin[j];
            join_waves<true>(lds_a[buf], lds_h[buf], state, h);
#pragma unroll
            for (int j = 0; j < kV; j++) h[j] = __builtin_fmaf(after_A[j], h[j], H[j]);
#pragma unroll
            for (int k = kSteps - 1; k >= 0; k--)
#pragma unroll
                for (int j = 0; j < kV; j++) {
                    before[k][j] = h[j];
                    h[j] = __builtin_fmaf(ga[k][j], h[j], xa[k][j]);
                }
#pragma unroll
            for (int k = 0; k < kSteps; k++) ga[k].let_go();
        }
        TX *to_x = anew(dx, t0 * n);
        TG *to_g = anew(dg, t0 * n);
#pragma unroll
        for (int k = 0; k < kSteps; k++) {
            Few<TX, kV> ox;
            Few<TG, kV> og;
            float e[kV], eh[kV];
#pragma unroll
            for (int j = 0; j < kV; j++) {
                e[j] = da[k][j] + f[j];
                if constexpr (kGate) eh[j] = e[j] * before[k][j];
                f[j] = ga[k][j] * e[j];
            }
            ox.set(e);
            if constexpr (kGate) og.set(eh);
            if (at.some && t0 - k < T) {
                if (dx) ox.store(to_x - (int64_t)k * n, a.past);
                if constexpr (kGate) og.store(to_g - (int64_t)k * n, a.past);
            }
        }
    }
    if (a.dstate && s == cut.segments - 1 && at.part == 0 && at.some) {
#pragma unroll
        for (int j = 0; j < kV; j++) a.dstate[at.b * n + at.c + j] = carry[j];
    }
}

constexpr int kAlone = 160;          // slabs from which on time is not cut
constexpr int kMostSegments = 256;   // maps that a workgroup of the second kernel joins
// want: workgroups that fill the chip
Cut cut_of(int64_t B, int64_t T, int n, int wide, int chunk, int want) {
    Cut c;
    c.slabs = (n + wide - 1) / wide;
    const int64_t columns = B * c.slabs, chunks = std::max<int64_t>((T + chunk - 1) / chunk, 1);
    // a segment is of two chunks or more; one alone from kAlone slabs on, which keep the memory busy by themselves (sequences of 4096 x 2048 bf16
    // with one segment and with as many as fill the chip, us: forward of 160 slabs 130 and 141, of 192 143 and 195, of 128 in wide slabs 126 and
    // 111; backward of 128 235 and 181, of 144 232 and 214, of 160 242 and 244, of 176 245 and 308, of 192 242 and 317)
    int64_t segments = columns >= kAlone ? 1 : std::min<int64_t>(std::min<int64_t>((want + columns - 1) / columns, kMostSegments), chunks / 2);
    segments = std::max<int64_t>(segments, 1);
    const int64_t per = (chunks + segments - 1) / segments;
    c.per = per * chunk;
    c.steps = T > 0 ? chunks * chunk : 0;
    c.segments = (int)((chunks + per - 1) / per);
    return c;
}
// Channels of a thread: 16 bytes of gates, or 8 where that makes slabs enough of too few (half; forward 4 x 4096 x 2048 f32 106 us with 16
// bytes and segments, 82 with 8 and none, 20 x 1000 x 300 f32 25 and 17; f32 backward 177 and 145; but of bf16 with f32 gates backward 113
// and 155, as the joins of a chunk take twice their share, and wide enough slabs are better off with 16: 6 x 4096 x 2048 125 and 144)
template <class TG, class F> auto with_width(int64_t B, int n, bool half, F f) {
    constexpr std::integral_constant<int, 16 / sizeof(TG)> wide{};
    constexpr std::integral_constant<int, 8 / sizeof(TG)> narrow{};
    constexpr std::integral_constant<int, 1> one{};
    auto slabs = [&](int v) { return B * ((n + kCols * v - 1) / (kCols * v)); };
    if (n < decltype(wide)::value) return f(one);
    if (half && slabs(decltype(wide)::value) < kAlone && slabs(decltype(narrow)::value) >= kAlone) return f(narrow);
    return f(wide);
}
template <class TX> constexpr bool half_of(bool back) { return !back || sizeof(TX) == 4; }
constexpr int steps_of(bool back) { return back ? 4 : 8; }     // of a thread
// Two workgroups on each CU, by the registers, three of the forward kernel of 16-bit values with gates in f32 (131072 x 256 bf16: 74 us of
// kernels, 80 with two; the backward kernel of 5 x 1001 x 1003 f32 18 us with two and 20 with three)
template <class TX, class TG> Cut cut_for(int64_t B, int64_t T, int n, bool back) {
    const int want = !back && sizeof(TX) == 2 && sizeof(TG) == 4 ? 768 : 512;
    return with_width<TG>(B, n, half_of<TX>(back), [&](auto v) { return cut_of(B, T, n, kCols * decltype(v)::value, kParts * steps_of(back), want); });
}

bool writes_past(int64_t B, int64_t T, int n, int size) { return B * T * n * size >= kPastBytes; }

template <class TX, class TG> hipError_t go(ScanArgs a, void *scratch, hipStream_t st) {
    a.past = writes_past(a.B, a.T, a.n, sizeof(TX));
    return with_width<TG>(a.B, a.n, half_of<TX>(false), [&](auto v) {
        constexpr int kV = decltype(v)::value, kSteps = steps_of(false);
        // by steps as long as the parts of a chunk would have few: 64 x 256 f32 of 8 steps 3.5 us and 4.2 by parts, of 12 4.1 and 4.2, of 16 4.7 and
        // 4.3; 16 x 2048 f32 3.6 and 5.2, 4.3 and 5.1, 5.0 and 5.1. (Channels enough to fill the chip are faster by steps further on:
        // 256 x 4096 bf16 of 16 18 us and 82, of 32 32 and 84.)
        if (a.T <= 8) {
            const int64_t threads = a.B * ((a.n + kV - 1) / kV);
            if ((threads + 255) / 256 > most_blocks(256)) return kTooLarge;
            hipLaunchKernelGGL((step_kernel<TX, TG, kV>), dim3((unsigned)((threads + 255) / 256)), dim3(256), 0, st, a);
            return hipGetLastError();
        }
        const Cut cut = cut_for<TX, TG>(a.B, a.T, a.n, false);
        const int64_t blocks = a.B * cut.slabs * cut.segments;
        if (blocks > most_blocks(256)) return kTooLarge;
        if (cut.segments > 1) {
            hipLaunchKernelGGL((segment_kernel<TX, TG, kV, kSteps, false>), dim3((unsigned)(blocks - a.B * cut.slabs)),
                               dim3(256), 0, st, (const TG *)a.gate, (const TX *)a.x, a.gate_b, a.gate_t, a.x_b, a.x_t, a.T, a.n, cut,
                               (float *)scratch);
        }
        hipLaunchKernelGGL((scan_kernel<TX, TG, kV, kSteps>), dim3((unsigned)blocks), dim3(256), 0, st, a, cut,
                           (const float *)scratch);
        return hipGetLastError();
    });
}
template <class TX, class TG> hipError_t go_grad(ScanGradArgs a, void *scratch, hipStream_t st) {
    a.past = writes_past(a.B, a.T, a.n, sizeof(TX));
    return with_width<TG>(a.B, a.n, half_of<TX>(true), [&](auto v) {
        constexpr int kV = decltype(v)::value, kSteps = steps_of(true);
        const Cut cut = cut_for<TX, TG>(a.B, a.T, a.n, true);
        const int64_t blocks = a.B * cut.slabs * cut.segments;
        if (blocks > most_blocks(256)) return kTooLarge;
        if (cut.segments > 1) {
            hipLaunchKernelGGL((segment_kernel<TX, TG, kV, kSteps, true>), dim3((unsigned)(blocks - a.B * cut.slabs)),
                               dim3(256), 0, st, (const TG *)a.gate, (const TX *)a.dh, a.gate_b, a.gate_t, a.T * a.n, (int64_t)a.n, a.T,
                               a.n, cut, (float *)scratch);
        }
        if (a.dgate)
            hipLaunchKernelGGL((scan_grad_kernel<TX, TG, kV, kSteps, true>), dim3((unsigned)blocks), dim3(256), 0, st, a,
                               cut, (const float *)scratch);
        else
            hipLaunchKernelGGL((scan_grad_kernel<TX, TG, kV, kSteps, false>), dim3((unsigned)blocks), dim3(256), 0, st,
                               a, cut, (const float *)scratch);
        return hipGetLastError();
    });
}
// f(a value of x's type, one of the gates')
template <class F> auto with_types(int type, int gate_type, F f) {
    if (type == kOpF32) return f(float(), float());
    if (type == kOpBf16) return gate_type == kOpF32 ? f(bf16_t(), float()) : f(bf16_t(), bf16_t());
    return gate_type == kOpF32 ? f(f16_t(), float()) : f(f16_t(), f16_t());
}

}  // namespace

int64_t scan_kept(int64_t B, int64_t T, int n) { return B * kept_of(T) * n * 4; }
int64_t scan_scratch(int type, int gate_type, int64_t B, int64_t T, int n) {
    const int64_t most = with_types(type, gate_type, [&](auto x, auto g) {
        auto segments = [&](bool back) { return cut_for<decltype(x), decltype(g)>(B, T, n, back).segments; };
        return std::max(segments(false), segments(true));
    });
    return most > 1 ? B * most * 2 * n * 4 : 0;
}
hipError_t launch_scan(int type, int gate_type, const ScanArgs &a, void *scratch, hipStream_t st) {
    return with_types(type, gate_type, [&](auto x, auto g) { return go<decltype(x), decltype(g)>(a, scratch, st); });
}
hipError_t launch_scan_grad(int type, int gate_type, const ScanGradArgs &a, void *scratch, hipStream_t st) {
    return with_types(type, gate_type, [&](auto x, auto g) { return go_grad<decltype(x), decltype(g)>(a, scratch, st); });
}

}  // namespace ygg
