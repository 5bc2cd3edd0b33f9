// The norm of many tensors' values together and their clipping by it: norm = sqrt(sum v^2), v times min(1, most / norm).
//
// A workgroup sums the squares of a chunk of one tensor; the chunks' sums are added in their order, by every workgroup of the second
// kernel where they are few, by a kernel between where they are many, so that the norm comes out the same every time; then each
// chunk is read again and written, from the last one, as the memory's cache still holds the end. Squares are taken and summed in 64
// bits: those of values past 2^64 or below 2^-63 leave f32's range, and the memory is far slower than the 64-bit units. The
// tensors' addresses and sizes go with the launch, kTensors at a time, so that nothing is copied to the device and a captured call
// keeps its own.
//
// The memory bounds large calls (120 million values of three types, 320 MB: 48 us for the squares, 6.6 TB/s, 5 for the norm, 109 for
// the values, 5.9 TB/s), the two launches small ones (70000 f32: 4 and 5 us).
#include <algorithm>

#include "ygg_ops.h"
#include "ygg_optype.h"

namespace ygg {
namespace {

constexpr int kThreads = 256, kMostChunk = 16384, kLeastChunk = 2048;    // values of a chunk
constexpr int kFewChunks = 1024;    // whose sums every workgroup adds: 8 KB from its L2, 2 us less than a launch between
constexpr int kTensors = 128;
struct Table {
    const void *in[kTensors];
    void *out[kTensors];
    int64_t size[kTensors];
    uint32_t first[kTensors + 1];   // a tensor's first workgroup
    uint8_t type[kTensors];
    int count, chunk;
    bool past;                      // the results, past the caches
};
static_assert(sizeof(Table) < 4000, "more than a launch's arguments");
struct Share {
    int t;
    int64_t from;
    int count;
};
// workgroup `id`'s chunk: by a search for the last tensor that begins no later
__device__ __forceinline__ Share share_of(const Table &tab, uint32_t id) {
    int lo = 0, n = tab.count;
    while (n > 1) {
        const int half = n / 2;
        if (tab.first[lo + half] <= id) lo += half, n -= half;
        else n = half;
    }
    const int64_t from = (int64_t)(id - tab.first[lo]) * tab.chunk;
    return {lo, from, (int)min(tab.size[lo] - from, (int64_t)tab.chunk)};
}
// f(the call for a type) by the tensor's
template <class F> __device__ __forceinline__ void by_type(int type, F f) {
    if (type == kOpF32) f(float());
    else if (type == kOpBf16) f(bf16_t());
    else f(f16_t());
}

// a sum over the workgroup, in thread 0
template <int kN> __device__ __forceinline__ double sum_all(double sum, double *lds) {
#pragma unroll
    for (int o = 32; o; o >>= 1) sum += __shfl_xor(sum, o);
    if (threadIdx.x % 64 == 0) lds[threadIdx.x / 64] = sum;
    __syncthreads();
#pragma unroll
    for (int w = 1; w < kN / 64; w++) sum += lds[w];
    return sum;
}
__global__ __launch_bounds__(kThreads) void squares_kernel(const Table tab, double *part) {
    __shared__ double lds[kThreads / 64];
    const Share s = share_of(tab, blockIdx.x);
    double sum[4] = {};
    by_type(tab.type[s.t], [&](auto one) {
        typedef decltype(one) T;
        constexpr int kE = 16 / sizeof(T), kU = 8;
        const T *p = (const T *)tab.in[s.t] + s.from;
        auto add = [&](u32x4 v) {
            float f[kE];
            unpack(v, f, T());
#pragma unroll
            for (int j = 0; j < kE; j++) sum[j % 4] = __builtin_fma((double)f[j], (double)f[j], sum[j % 4]);
        };
        int c = threadIdx.x * kE;
        for (; c + (kU - 1) * kThreads * kE + kE <= s.count; c += kU * kThreads * kE) {
            u32x4 v[kU];
#pragma unroll
            for (int u = 0; u < kU; u++) v[u] = load16(p + c + u * kThreads * kE);
#pragma unroll
            for (int u = 0; u < kU; u++) add(v[u]);
        }
        for (; c < s.count; c += kThreads * kE) add(load16(p + c, s.count - c));
    });
    const double all = sum_all<kThreads>((sum[0] + sum[1]) + (sum[2] + sum[3]), lds);
    if (threadIdx.x == 0) part[blockIdx.x] = all;
}

// v for a later rounding to T, so that both together are one: f32 itself, else towards zero with the last bit set where anything is lost
// (f32 has 13 bits more than f16, and 16 more than bf16, so what is no value of f32 stays on its side of their middles)
template <class T> __device__ __forceinline__ float to_odd(double v) {
    const float f = (float)v;
    if constexpr (sizeof(T) == 4) return f;
    const double back = (double)f;
    const uint32_t b = __builtin_bit_cast(uint32_t, f);
    return back == v ? f : __builtin_bit_cast(float, (b - (__builtin_fabs(back) > __builtin_fabs(v))) | 1u);
}

// in thread 0: the norm, and what the values are multiplied by. A norm that is no finite number changes nothing.
struct Norm {
    double norm, by;
};
template <int kN> __device__ __forceinline__ Norm norm_of(const double *part, int64_t count, double most, double *lds) {
    double sum = 0.0;
    for (int64_t i = threadIdx.x; i < count; i += kN) sum += part[i];
    const double all = sqrt(sum_all<kN>(sum, lds));
    return {all, all > most && all < __builtin_huge_val() ? most / all : 1.0};
}
__global__ __launch_bounds__(1024) void norm_of_kernel(const double *part, int64_t count, double most, float *norm, double *by) {
    __shared__ double lds[16];
    const Norm n = norm_of<1024>(part, count, most, lds);
    if (threadIdx.x) return;
    *norm = (float)n.norm;
    *by = n.by;
}

// few > 0: the chunks' sums, `few` of them, are added here; else `by` holds what comes of them
__global__ __launch_bounds__(kThreads) void scale_kernel(const Table tab, const double *by, const double *part, int few, double most, float *norm) {
    __shared__ double lds[kThreads / 64], shared;
    double f;
    if (few) {
        const Norm n = norm_of<kThreads>(part, few, most, lds);
        if (threadIdx.x == 0) {
            shared = n.by;
            if (norm && blockIdx.x == 0) *norm = (float)n.norm;
        }
        __syncthreads();
        f = shared;
    } else {
        f = *by;
    }
    const Share s = share_of(tab, gridDim.x - 1 - blockIdx.x);
    if (f == 1.0 && tab.in[s.t] == tab.out[s.t]) return;
    by_type(tab.type[s.t], [&](auto one) {
        typedef decltype(one) T;
        constexpr int kE = 16 / sizeof(T), kU = 4;
        const T *p = (const T *)tab.in[s.t] + s.from;
        T *out = (T *)tab.out[s.t] + s.from;
        auto put = [&](int c, u32x4 v) {
            float t[kE];
            unpack(v, t, T());
#pragma unroll
            for (int j = 0; j < kE; j++) t[j] = to_odd<T>((double)t[j] * f);
            store_run<T, kE>(out + c, t, s.count - c, tab.past);
        };
        int c = threadIdx.x * kE;
        for (; c + (kU - 1) * kThreads * kE + kE <= s.count; c += kU * kThreads * kE) {
            u32x4 v[kU];
#pragma unroll
            for (int u = 0; u < kU; u++) v[u] = load16(p + c + u * kThreads * kE);
#pragma unroll
            for (int u = 0; u < kU; u++) put(c + u * kThreads * kE, v[u]);
        }
        for (; c < s.count; c += kThreads * kE) put(c, load16(p + c, s.count - c));
    });
}

// 2048 values where there are few in all (a thread's one load or two), so that more CUs take part: 70000 f32 in 8 chunks 10.0 us of
// kernels, in 35 chunks 7.6
int chunk_of(const int64_t *sizes, int count) {
    int64_t all = 0;
    for (int i = 0; i < count; i++) all += sizes[i];
    int chunk = kLeastChunk;
    while (chunk < kMostChunk && all > (int64_t)chunk * kFewChunks) chunk *= 2;
    return chunk;
}
int64_t chunks_of(int64_t size, int chunk) { return (size + chunk - 1) / chunk; }

}  // namespace

int64_t clip_scratch(const int64_t *sizes, int count) {
    const int chunk = chunk_of(sizes, count);
    int64_t chunks = 0;
    for (int i = 0; i < count; i++) chunks += chunks_of(sizes[i], chunk);
    return 8 * (chunks + 1);
}
hipError_t launch_clip(const void *const *tensors, const int64_t *sizes, const int *types, int count, double most, void *const *out,
                       float *norm, void *scratch, hipStream_t st) {
    double *by = (double *)scratch, *part = by + 1;
    const int chunk = chunk_of(sizes, count);
    int64_t bytes = 0;
    for (int i = 0; i < count; i++) bytes += sizes[i] * op_bytes(types[i]);
    // f(a table of up to kTensors tensors, its workgroups, those before them)
    auto tables = [&](auto f) {
        int64_t before = 0;
        for (int i = 0; i < count;) {
            Table tab;
            int n = 0;
            int64_t blocks = 0;
            for (; i < count && n < kTensors; i++) {
                const int64_t chunks = chunks_of(sizes[i], chunk);
                if (chunks == 0) continue;
                if (chunks > most_blocks(kThreads)) return kTooLarge;
                if (blocks + chunks > most_blocks(kThreads)) break;
                tab.in[n] = tensors[i];
                tab.out[n] = out ? out[i] : nullptr;
                tab.size[n] = sizes[i];
                tab.type[n] = (uint8_t)types[i];
                tab.first[n++] = (uint32_t)blocks;
                blocks += chunks;
            }
            if (!n) continue;
            tab.first[n] = (uint32_t)blocks;
            tab.count = n;
            tab.chunk = chunk;
            tab.past = bytes >= kPastBytes;
            f(tab, (unsigned)blocks, before);
            const hipError_t e = hipGetLastError();
            if (e != hipSuccess) return e;
            before += blocks;
        }
        return hipSuccess;
    };
    int64_t all = 0;
    for (int i = 0; i < count; i++) all += chunks_of(sizes[i], chunk);
    hipError_t e = tables([&](const Table &tab, unsigned blocks, int64_t before) {
        hipLaunchKernelGGL(squares_kernel, dim3(blocks), dim3(kThreads), 0, st, tab, part + before);
    });
    if (e != hipSuccess) return e;
    const int few = out && all > 0 && all <= kFewChunks ? (int)all : 0;
    if (!few) {
        hipLaunchKernelGGL(norm_of_kernel, dim3(1), dim3(1024), 0, st, (const double *)part, all, most, norm, by);
        e = hipGetLastError();
        if (e != hipSuccess || !out) return e;
    }
    return tables([&](const Table &tab, unsigned blocks, int64_t before) {
        hipLaunchKernelGGL(scale_kernel, dim3(blocks), dim3(kThreads), 0, st, tab, (const double *)by, (const double *)part, few, most,
                           before == 0 ? norm : nullptr);
    });
}

}  // namespace ygg
