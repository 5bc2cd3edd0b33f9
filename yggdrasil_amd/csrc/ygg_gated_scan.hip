// The gated recurrence h_t = a_t h_{t-1} + x_t of every channel, over long sequences, and its gradients
//   e_t = dh_t + a_{t+1} e_{t+1} (of the last step with the final state's gradient),  dx_t = e_t,  da_t = e_t h_{t-1},
//   dstate = a_0 e_0.
//
// A run of steps maps the state before it to the one after it, h -> A h + H with A the product of its gates and H its result from
// zero; two runs join to (A2 A1, A2 H1 + H2). A workgroup takes a slab of kCols * kV channels and goes through time by chunks of
// kParts * kSteps steps: each thread holds kSteps steps of kV channels in registers, so that its loads are all in flight
// together and values are read once; the parts' maps are joined in LDS, in the order of time, and each thread then computes its
// steps again from the state it begins with. The next chunk's loads are issued before that. The backward pass is the same from
// the end: f_t = a_t e_t is what step t hands to the one before, e_t = dh_t + f_{t+1}.
//
// Where the slabs are too few for the chip, time is cut into segments too: a first kernel takes the map of each, and
// every workgroup of the second joins those before its own. That reads the gates and x (or dh) twice, so the second kernel goes
// through the segments from the last one, whose values the memory's cache still holds. States, maps and their joins are in f32;
// h, dx and da are rounded to their types on the way out, and da takes the rounded h_{t-1}: it is off by that rounding and its own.
#include <algorithm>

#include "ygg_ops.h"
#include "ygg_optype.h"

namespace ygg {
namespace {

// kV consecutive values as they lie in memory
template <class T, int kV> struct Few {
    T v[kV];
    __device__ __forceinline__ void load(const T *p) {
        if constexpr (kV == 1) {
            v[0] = *p;
        } else {
            typedef uint32_t any __attribute__((ext_vector_type(kV * sizeof(T) / 4), aligned(1)));
            const any a = *(const any *)p;
            __builtin_memcpy(v, &a, sizeof(v));
        }
    }
    __device__ __forceinline__ void store(T *p) const {
        if constexpr (kV == 1) {
            *p = v[0];
        } else {
            typedef uint32_t any __attribute__((ext_vector_type(kV * sizeof(T) / 4), aligned(1)));
            any a;
            __builtin_memcpy(&a, v, sizeof(v));
            *(any *)p = a;
        }
    }
};

// A thread's channels: the last ones of a row that they do not fill begin earlier, and compute some a second time
template <int kV> struct Place {
    int64_t b;
    int c, part;
    bool some;
    template <int kCols> __device__ __forceinline__ static Place of(int64_t slab, int slabs, int n) {
        const int col = (int)(slab % slabs * kCols) + (int)threadIdx.x % kCols;
        return {slab / slabs, max(min(col * kV, n - kV), 0), (int)threadIdx.x / kCols, col * kV < n};
    }
};
// The map of a part of a chunk, in LDS
template <int kV, int kCols, int kParts> struct Maps {
    float a[kParts][kCols * kV], h[kParts][kCols * kV];
    __device__ __forceinline__ void put(int part, int col, const float *A, const float *H) {
#pragma unroll
        for (int j = 0; j < kV; j++) {
            a[part][col * kV + j] = A[j];
            h[part][col * kV + j] = H[j];
        }
    }
    // carry: the state at the chunk's begin, then at its end; in: at the begin of part `part`
    __device__ __forceinline__ void join(int part, int col, float *carry, float *in) const {
#pragma unroll
        for (int q = 0; q < kParts; q++) {
#pragma unroll
            for (int j = 0; j < kV; j++) {
                in[j] = q == part ? carry[j] : in[j];
                carry[j] = __builtin_fmaf(a[q][col * kV + j], carry[j], h[q][col * kV + j]);
            }
        }
    }
};
// the state at the begin of a segment: what `begin` is after the segments before it, whose maps lie `hop` values apart
template <int kV> __device__ __forceinline__ void join_segments(const float *maps, int64_t hop, int n, int count, float *carry) {
#pragma unroll 8
    for (int s = 0; s < count; s++) {
        float A[kV], H[kV];
#pragma unroll
        for (int j = 0; j < kV; j++) {
            A[j] = maps[s * hop + j];
            H[j] = maps[s * hop + n + j];
        }
#pragma unroll
        for (int j = 0; j < kV; j++) carry[j] = __builtin_fmaf(A[j], carry[j], H[j]);
    }
}

// How a call is cut: `slabs` of a sequence, `segments` of `per` steps each
struct Cut {
    int slabs, segments;
    int64_t per;
};

// the maps of the segments, (B, segments, 2, n): each part goes through its share of the segment by itself. kBack: time runs
// backwards (places and segments count from the end), the map is that of f from dh.
template <class TX, class TG, int kV, int kCols, int kParts, int kSteps, bool kBack>
__global__ __launch_bounds__(kCols *kParts) void segment_kernel(const TG *gate, const TX *x, int64_t gate_b, int64_t gate_t, int64_t x_b,
                                                                int64_t x_t, int64_t T, int n, Cut cut, float *maps) {
    __shared__ Maps<kV, kCols, kParts> lds;
    const int s = blockIdx.x % (cut.segments - 1);     // nobody asks for the last one's
    const Place<kV> at = Place<kV>::template of<kCols>(blockIdx.x / (cut.segments - 1), cut.slabs, n);
    const int64_t from = s * cut.per, share = cut.per / kParts;      // a segment that is not the last is whole
    const TG *g = gate + at.b * gate_b + at.c;
    const TX *xp = x ? x + at.b * x_b + at.c : nullptr;
    auto step = [&](int64_t i) { return kBack ? T - 1 - i : i; };
    float A[kV], H[kV];
#pragma unroll
    for (int j = 0; j < kV; j++) A[j] = 1.0f, H[j] = 0.0f;
    int64_t i = from + at.part * share;
    const int64_t end = i + share;
    for (; i < end; i += kSteps) {     // share is a multiple of kSteps
        Few<TG, kV> a[kSteps];
        Few<TX, kV> v[kSteps];
#pragma unroll
        for (int k = 0; k < kSteps; k++) {
            a[k].load(g + step(i + k) * gate_t);
            if (xp) v[k].load(xp + step(i + k) * x_t);
        }
#pragma unroll
        for (int k = 0; k < kSteps; k++)
#pragma unroll
            for (int j = 0; j < kV; j++) {
                const float gt = to_f32(a[k].v[j]), xt = xp ? to_f32(v[k].v[j]) : 0.0f;
                H[j] = kBack ? gt * (xt + H[j]) : __builtin_fmaf(gt, H[j], xt);
                A[j] *= gt;
            }
    }
    lds.put(at.part, threadIdx.x % kCols, A, H);
    __syncthreads();
    if (at.part || !at.some) return;
    const int col = threadIdx.x % kCols;
#pragma unroll
    for (int q = 1; q < kParts; q++)
#pragma unroll
        for (int j = 0; j < kV; j++) {
            H[j] = __builtin_fmaf(lds.a[q][col * kV + j], H[j], lds.h[q][col * kV + j]);
            A[j] *= lds.a[q][col * kV + j];
        }
    float *out = maps + (at.b * cut.segments + s) * 2 * n + at.c;
#pragma unroll
    for (int j = 0; j < kV; j++) {
        out[j] = A[j];
        out[n + j] = H[j];
    }
}

template <class TX, class TG, int kV, int kCols, int kParts, int kSteps>
__global__ __launch_bounds__(kCols *kParts) void scan_kernel(const ScanArgs a, Cut cut, const float *maps) {
    constexpr int kChunk = kParts * kSteps;
    __shared__ Maps<kV, kCols, kParts> lds[2];
    const int id = gridDim.x - 1 - blockIdx.x, s = id % cut.segments, n = a.n, col = threadIdx.x % kCols;
    const Place<kV> at = Place<kV>::template of<kCols>(id / cut.segments, cut.slabs, n);
    const int64_t from = s * cut.per, end = min(from + cut.per, a.T);
    const TG *g = (const TG *)a.gate + at.b * a.gate_b + at.c;
    const TX *x = (const TX *)a.x + at.b * a.x_b + at.c;
    TX *h = (TX *)a.h + at.b * a.T * n + at.c;
    Few<TG, kV> ga[kSteps], next_g[kSteps];
    Few<TX, kV> xa[kSteps], next_x[kSteps];
    auto load = [&](int64_t chunk) {
#pragma unroll
        for (int k = 0; k < kSteps; k++) {
            const int64_t t = min(chunk + at.part * kSteps + k, end - 1);
            next_g[k].load(g + t * a.gate_t);
            next_x[k].load(x + t * a.x_t);
        }
    };
    load(from);
    float carry[kV];
#pragma unroll
    for (int j = 0; j < kV; j++) carry[j] = a.state ? a.state[at.b * n + at.c + j] : 0.0f;
    join_segments<kV>(maps + at.b * cut.segments * 2 * n + at.c, 2 * n, n, s, carry);
    int buf = 0;
    for (int64_t chunk = from; chunk < end; chunk += kChunk, buf ^= 1) {
        const int64_t t0 = chunk + at.part * kSteps;
#pragma unroll
        for (int k = 0; k < kSteps; k++) {
            ga[k] = next_g[k];
            xa[k] = next_x[k];
        }
        if (chunk + kChunk < end) load(chunk + kChunk);
        float A[kV], H[kV];
#pragma unroll
        for (int j = 0; j < kV; j++) A[j] = 1.0f, H[j] = 0.0f;
#pragma unroll
        for (int k = 0; k < kSteps; k++)
#pragma unroll
            for (int j = 0; j < kV; j++) {
                const bool is = t0 + k < end;      // steps past the end change nothing
                const float gt = to_f32(ga[k].v[j]);
                H[j] = is ? __builtin_fmaf(gt, H[j], to_f32(xa[k].v[j])) : H[j];
                A[j] = is ? A[j] * gt : A[j];
            }
        lds[buf].put(at.part, col, A, H);
        __syncthreads();
        float in[kV];
        lds[buf].join(at.part, col, carry, in);
#pragma unroll
        for (int k = 0; k < kSteps; k++) {
            Few<TX, kV> out;
#pragma unroll
            for (int j = 0; j < kV; j++) {
                in[j] = __builtin_fmaf(to_f32(ga[k].v[j]), in[j], to_f32(xa[k].v[j]));
                out.v[j] = from_f32<TX>(in[j]);
            }
            if (at.some && t0 + k < end) out.store(h + (t0 + k) * n);
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
        for (int j = 0; j < kV; j++) {
            s[j] = __builtin_fmaf(to_f32(gt.v[j]), s[j], to_f32(xt.v[j]));
            out.v[j] = from_f32<TX>(s[j]);
        }
        out.store(h + t * n);
    }
#pragma unroll
    for (int j = 0; j < kV; j++) a.last[b * n + c + j] = s[j];
}

// backward; places count from the end: place i is step T - 1 - i
template <class TX, class TG, int kV, int kCols, int kParts, int kSteps>
__global__ __launch_bounds__(kCols *kParts) void scan_grad_kernel(const ScanGradArgs a, Cut cut, const float *maps) {
    constexpr int kChunk = kParts * kSteps;
    __shared__ Maps<kV, kCols, kParts> lds[2];
    const int id = gridDim.x - 1 - blockIdx.x, s = id % cut.segments, n = a.n, col = threadIdx.x % kCols;
    const Place<kV> at = Place<kV>::template of<kCols>(id / cut.segments, cut.slabs, n);
    const int64_t T = a.T, from = s * cut.per, end = min(from + cut.per, T), row = at.b * T * n + at.c;
    const TG *g = (const TG *)a.gate + at.b * a.gate_b + at.c;
    const TX *dh = a.dh ? (const TX *)a.dh + row : nullptr, *h = (const TX *)a.h + row;
    TX *dx = a.dx ? (TX *)a.dx + row : nullptr;
    TG *dg = a.dgate ? (TG *)a.dgate + row : nullptr;
    float first[kV], carry[kV];     // the state before the first step, and what the steps after this chunk hand to it
#pragma unroll
    for (int j = 0; j < kV; j++) {
        first[j] = a.state ? a.state[at.b * n + at.c + j] : 0.0f;
        carry[j] = a.dlast ? a.dlast[at.b * n + at.c + j] : 0.0f;
    }
    Few<TG, kV> ga[kSteps], next_g[kSteps];
    Few<TX, kV> da[kSteps], next_d[kSteps], ha[kSteps], next_h[kSteps];
    auto load = [&](int64_t chunk) {
#pragma unroll
        for (int k = 0; k < kSteps; k++) {
            const int64_t t = T - 1 - min(chunk + at.part * kSteps + k, end - 1);
            next_g[k].load(g + t * a.gate_t);
            if (dh) next_d[k].load(dh + t * n);
            if (dg) next_h[k].load(h + max(t - 1, (int64_t)0) * n);
        }
    };
    if (from < end) load(from);     // there may be no step at all
    join_segments<kV>(maps + at.b * cut.segments * 2 * n + at.c, 2 * n, n, s, carry);
    int buf = 0;
    for (int64_t chunk = from; chunk < end; chunk += kChunk, buf ^= 1) {
        const int64_t i0 = chunk + at.part * kSteps;
#pragma unroll
        for (int k = 0; k < kSteps; k++) {
            ga[k] = next_g[k];
            da[k] = next_d[k];
            ha[k] = next_h[k];
        }
        if (chunk + kChunk < end) load(chunk + kChunk);
        float A[kV], F[kV];
#pragma unroll
        for (int j = 0; j < kV; j++) A[j] = 1.0f, F[j] = 0.0f;
#pragma unroll
        for (int k = 0; k < kSteps; k++)
#pragma unroll
            for (int j = 0; j < kV; j++) {
                const bool is = i0 + k < end;
                const float gt = to_f32(ga[k].v[j]), e = (dh ? to_f32(da[k].v[j]) : 0.0f) + F[j];
                F[j] = is ? gt * e : F[j];
                A[j] = is ? A[j] * gt : A[j];
            }
        lds[buf].put(at.part, col, A, F);
        __syncthreads();
        float f[kV];
        lds[buf].join(at.part, col, carry, f);
#pragma unroll
        for (int k = 0; k < kSteps; k++) {
            const int64_t t = T - 1 - (i0 + k);
            Few<TX, kV> ox;
            Few<TG, kV> og;
#pragma unroll
            for (int j = 0; j < kV; j++) {
                const float e = (dh ? to_f32(da[k].v[j]) : 0.0f) + f[j];
                ox.v[j] = from_f32<TX>(e);
                og.v[j] = from_f32<TG>(e * (t > 0 ? to_f32(ha[k].v[j]) : first[j]));
                f[j] = to_f32(ga[k].v[j]) * e;
            }
            if (at.some && i0 + k < end) {
                if (dx) ox.store(dx + t * n);
                if (dg) og.store(dg + t * n);
            }
        }
    }
    if (a.dstate && s == cut.segments - 1 && at.part == 0 && at.some) {
#pragma unroll
        for (int j = 0; j < kV; j++) a.dstate[at.b * n + at.c + j] = carry[j];
    }
}

constexpr int kWant = 512;           // workgroups that fill the chip: two on each CU
constexpr int kMostSegments = 128;   // maps that a workgroup of the second kernel joins
Cut cut_of(int64_t B, int64_t T, int n, int wide, int chunk) {
    Cut c;
    c.slabs = (n + wide - 1) / wide;
    const int64_t columns = B * c.slabs, chunks = std::max<int64_t>((T + chunk - 1) / chunk, 1);
    // a segment is of two chunks or more
    int64_t segments = columns >= kWant / 2 ? 1 : std::min<int64_t>(std::min<int64_t>((kWant + columns - 1) / columns, kMostSegments), chunks / 2);
    segments = std::max<int64_t>(segments, 1);
    const int64_t per = (chunks + segments - 1) / segments;
    c.per = per * chunk;
    c.segments = (int)((chunks + per - 1) / per);
    return c;
}
template <class TG> constexpr int vector_of() { return 16 / (int)sizeof(TG); }
// values of a thread, and of a slab, by the row's length
template <class TG, class F> auto with_width(int n, F f) {
    constexpr std::integral_constant<int, vector_of<TG>()> wide{};
    constexpr std::integral_constant<int, 1> one{};
    return n >= vector_of<TG>() ? f(wide) : f(one);
}
constexpr int kCols = 16, kParts = 16, kSteps = 8, kBackSteps = 4;
template <class TG> Cut cut_for(int64_t B, int64_t T, int n, bool back) {
    return with_width<TG>(n, [&](auto v) { return cut_of(B, T, n, kCols * decltype(v)::value, kParts * (back ? kBackSteps : kSteps)); });
}

template <class TX, class TG> hipError_t go(const ScanArgs &a, void *scratch, hipStream_t st) {
    return with_width<TG>(a.n, [&](auto v) {
        constexpr int kV = decltype(v)::value;
        if (a.T <= 8) {
            const int64_t threads = a.B * ((a.n + kV - 1) / kV);
            if ((threads + 255) / 256 > most_blocks(256)) return kTooLarge;
            hipLaunchKernelGGL((step_kernel<TX, TG, kV>), dim3((unsigned)((threads + 255) / 256)), dim3(256), 0, st, a);
            return hipGetLastError();
        }
        const Cut cut = cut_for<TG>(a.B, a.T, a.n, false);
        const int64_t blocks = a.B * cut.slabs * cut.segments;
        if (blocks > most_blocks(256)) return kTooLarge;
        if (cut.segments > 1) {
            hipLaunchKernelGGL((segment_kernel<TX, TG, kV, kCols, kParts, kSteps, false>), dim3((unsigned)(blocks - a.B * cut.slabs)),
                               dim3(256), 0, st, (const TG *)a.gate, (const TX *)a.x, a.gate_b, a.gate_t, a.x_b, a.x_t, a.T, a.n, cut,
                               (float *)scratch);
        }
        hipLaunchKernelGGL((scan_kernel<TX, TG, kV, kCols, kParts, kSteps>), dim3((unsigned)blocks), dim3(256), 0, st, a, cut,
                           (const float *)scratch);
        return hipGetLastError();
    });
}
template <class TX, class TG> hipError_t go_grad(const ScanGradArgs &a, void *scratch, hipStream_t st) {
    return with_width<TG>(a.n, [&](auto v) {
        constexpr int kV = decltype(v)::value;
        const Cut cut = cut_for<TG>(a.B, a.T, a.n, true);
        const int64_t blocks = a.B * cut.slabs * cut.segments;
        if (blocks > most_blocks(256)) return kTooLarge;
        if (cut.segments > 1) {
            hipLaunchKernelGGL((segment_kernel<TX, TG, kV, kCols, kParts, kBackSteps, true>), dim3((unsigned)(blocks - a.B * cut.slabs)),
                               dim3(256), 0, st, (const TG *)a.gate, (const TX *)a.dh, a.gate_b, a.gate_t, a.T * a.n, (int64_t)a.n, a.T,
                               a.n, cut, (float *)scratch);
        }
        hipLaunchKernelGGL((scan_grad_kernel<TX, TG, kV, kCols, kParts, kBackSteps>), dim3((unsigned)blocks), dim3(256), 0, st, a, cut,
                           (const float *)scratch);
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

int64_t scan_scratch(int type, int gate_type, int64_t B, int64_t T, int n) {
    const bool wide = type == kOpF32 || gate_type == kOpF32;
    int64_t most = 1;
    for (bool back : {false, true})
        most = std::max<int64_t>(most, (wide ? cut_for<float>(B, T, n, back) : cut_for<bf16_t>(B, T, n, back)).segments);
    return most > 1 ? B * most * 2 * n * 4 : 0;
}
hipError_t launch_scan(int type, int gate_type, const ScanArgs &a, void *scratch, hipStream_t st) {
    return with_types(type, gate_type, [&](auto x, auto g) { return go<decltype(x), decltype(g)>(a, scratch, st); });
}
hipError_t launch_scan_grad(int type, int gate_type, const ScanGradArgs &a, void *scratch, hipStream_t st) {
    return with_types(type, gate_type, [&](auto x, auto g) { return go_grad<decltype(x), decltype(g)>(a, scratch, st); });
}

}  // namespace ygg
