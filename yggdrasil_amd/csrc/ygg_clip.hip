// The norm of many tensors' values together and their clipping by it: norm = sqrt(sum v^2), v times min(1, most / norm).
//
// A workgroup sums the squares of a chunk of one tensor, one more adds the chunks' sums in their order, so that the norm comes out
// the same every time; then each chunk is read again and written. Squares are taken and summed in 64 bits: those of values
// past 2^64 or below 2^-63 leave f32's range, and the memory is far slower than the 64-bit units. The tensors' addresses
// and sizes go with the launch, kTensors at a time, so that nothing is copied to the device and a captured call keeps its own.
#include <algorithm>

#include "ygg_ops.h"
#include "ygg_optype.h"

namespace ygg {
namespace {

constexpr int kThreads = 256, kChunk = 16384;    // values of a chunk
constexpr int kTensors = 128;
struct Table {
    const void *in[kTensors];
    void *out[kTensors];
    int64_t size[kTensors];
    uint32_t first[kTensors + 1];   // a tensor's first workgroup
    uint8_t type[kTensors];
};
static_assert(sizeof(Table) < 4000, "more than a launch's arguments");
struct Share {
    int t;
    int64_t from;
    int count;
};
// the workgroup's chunk: by a search for the last tensor that begins no later
__device__ __forceinline__ Share share_of(const Table &tab, int count) {
    int lo = 0, n = count;
    while (n > 1) {
        const int half = n / 2;
        if (tab.first[lo + half] <= blockIdx.x) lo += half, n -= half;
        else n = half;
    }
    const int64_t from = (int64_t)(blockIdx.x - tab.first[lo]) * kChunk;
    return {lo, from, (int)min(tab.size[lo] - from, (int64_t)kChunk)};
}
// f(the call for a type) by the tensor's
template <class F> __device__ __forceinline__ void by_type(int type, F f) {
    if (type == kOpF32) f(float());
    else if (type == kOpBf16) f(bf16_t());
    else f(f16_t());
}

__global__ __launch_bounds__(kThreads) void squares_kernel(const Table tab, int count, double *part) {
    __shared__ double sums[kThreads / 64];
    const Share s = share_of(tab, count);
    double sum = 0.0;
    by_type(tab.type[s.t], [&](auto one) {
        typedef decltype(one) T;
        constexpr int kE = 16 / sizeof(T), kU = 4;
        const T *p = (const T *)tab.in[s.t] + s.from;
        int c = threadIdx.x * kE;
        for (; c + (kU - 1) * kThreads * kE + kE <= s.count; c += kU * kThreads * kE) {
            u32x4 v[kU];
#pragma unroll
            for (int u = 0; u < kU; u++) v[u] = load16(p + c + u * kThreads * kE);
#pragma unroll
            for (int u = 0; u < kU; u++) {
                float f[kE];
                unpack(v[u], f, T());
#pragma unroll
                for (int j = 0; j < kE; j++) sum = __builtin_fma((double)f[j], (double)f[j], sum);
            }
        }
        for (; c < s.count; c += kThreads * kE) {
            float f[kE];
            unpack(load16(p + c, s.count - c), f, T());
#pragma unroll
            for (int j = 0; j < kE; j++) sum = __builtin_fma((double)f[j], (double)f[j], sum);
        }
    });
#pragma unroll
    for (int o = 32; o; o >>= 1) sum += __shfl_xor(sum, o);
    if (threadIdx.x % 64 == 0) sums[threadIdx.x / 64] = sum;
    __syncthreads();
    if (threadIdx.x) return;
#pragma unroll
    for (int w = 1; w < kThreads / 64; w++) sum += sums[w];
    part[blockIdx.x] = sum;
}

// part[0 .. count - 1] -> the norm, and what the values are multiplied by. A norm that is no finite number changes nothing.
__global__ __launch_bounds__(1024) void norm_of_kernel(const double *part, int64_t count, double most, float *norm, double *by) {
    __shared__ double sums[16];
    double sum = 0.0;
    for (int64_t i = threadIdx.x; i < count; i += 1024) sum += part[i];
#pragma unroll
    for (int o = 32; o; o >>= 1) sum += __shfl_xor(sum, o);
    if (threadIdx.x % 64 == 0) sums[threadIdx.x / 64] = sum;
    __syncthreads();
    if (threadIdx.x) return;
#pragma unroll
    for (int w = 1; w < 16; w++) sum += sums[w];
    const double all = sqrt(sum);
    *norm = (float)all;
    *by = all > most && all < __builtin_huge_val() ? most / all : 1.0;
}

__global__ __launch_bounds__(kThreads) void scale_kernel(const Table tab, int count, const double *by) {
    const double f = *by;
    const Share s = share_of(tab, count);
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
            for (int j = 0; j < kE; j++) t[j] = (float)((double)t[j] * f);
            store_run<T, kE>(out + c, t, s.count - c);
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

int64_t chunks_of(int64_t size) { return (size + kChunk - 1) / kChunk; }

}  // namespace

int64_t clip_scratch(const int64_t *sizes, int count) {
    int64_t chunks = 0;
    for (int i = 0; i < count; i++) chunks += chunks_of(sizes[i]);
    return 8 * (chunks + 1);
}
hipError_t launch_clip(const void *const *tensors, const int64_t *sizes, const int *types, int count, double most, void *const *out,
                       float *norm, void *scratch, hipStream_t st) {
    double *by = (double *)scratch, *part = by + 1;
    // f(a table of up to kTensors tensors, how many, their workgroups, those before them)
    auto tables = [&](auto f) {
        int64_t before = 0;
        for (int i = 0; i < count;) {
            Table tab;
            int n = 0;
            int64_t blocks = 0;
            for (; i < count && n < kTensors; i++) {
                const int64_t chunks = chunks_of(sizes[i]);
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
            f(tab, n, (unsigned)blocks, before);
            const hipError_t e = hipGetLastError();
            if (e != hipSuccess) return e;
            before += blocks;
        }
        return hipSuccess;
    };
    int64_t all = 0;
    for (int i = 0; i < count; i++) all += chunks_of(sizes[i]);
    hipError_t e = tables([&](const Table &tab, int n, unsigned blocks, int64_t before) {
        hipLaunchKernelGGL(squares_kernel, dim3(blocks), dim3(kThreads), 0, st, tab, n, part + before);
    });
    if (e != hipSuccess) return e;
    hipLaunchKernelGGL(norm_of_kernel, dim3(1), dim3(1024), 0, st, (const double *)part, all, most, norm, by);
    e = hipGetLastError();
    if (e != hipSuccess || !out) return e;
    return tables([&](const Table &tab, int n, unsigned blocks, int64_t) {
        hipLaunchKernelGGL(scale_kernel, dim3(blocks), dim3(kThreads), 0, st, tab, n, (const double *)by);
    });
}

}  // namespace ygg
