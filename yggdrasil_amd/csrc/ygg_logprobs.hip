// Log-probabilities of given tokens, entropies and most likely tokens of rows of logits, and their gradient.
//
// For a row x of V logits with m = max x, n the number of entries equal to m, r = sum of exp(x_c - m) over the others
// and s = sum of exp(x_c - m) (x_c - m) over them:
//   log Z = log1p(n - 1 + r)      (Z = sum exp(x - m); without cancellation where one token holds nearly everything)
//   logp_c = (x_c - m) - log Z
//   entropy = log Z - s / Z       (two terms of the same sign)
// Two parts of a row join in their larger maximum: the other's n, r, s become, with d the difference of the maxima (<= 0) and
// f = exp d: n 0, r f (r + n), s f (s + (r + n) d). A row whose every entry is -inf has logp -inf and entropy 0; one with a
// NaN or +inf is NaN throughout (its r is: m is the largest number, and +inf - m or NaN - m joins the sum).
//
// The most likely tokens: every lane's largest value is known from the maximum's pass, and of the 16 or 64 of them the
// top-th largest is a bound that at least `top` entries reach and few others; those are gathered in LDS and each counts the
// keys (value, then lower index) above its own: its place. Where too many reach the bound (values in an order that hurts,
// or equal, also masked ones of a finite value where fewer than `top` are left), the places are found one by one, a pass each:
// 20 of 8 x 131072 equal bf16 46 us for 13, 5 of 4095 x 50257 464 for 119.
#include "ygg_ops.h"
#include "ygg_optype.h"

namespace ygg {
namespace {

constexpr float kLog2e = 1.4426950408889634f, kLowest = -3.402823466e38f;
constexpr float kGone = -1000.0f;    // exp of it is 0 in f32, and a count times it is finite

__device__ __forceinline__ float exp_of(float d) { return __builtin_amdgcn_exp2f(d * kLog2e); }

// the float's order as an unsigned integer's, and a row's entry as a key: larger first, then the lower index
__device__ __forceinline__ uint32_t ordered(float v) {
    const uint32_t u = __builtin_bit_cast(uint32_t, v);
    return u ^ ((uint32_t)((int32_t)u >> 31) | 0x80000000u);
}
__device__ __forceinline__ float unordered(uint32_t u) {
    return __builtin_bit_cast(float, u ^ ((uint32_t)((int32_t)~u >> 31) | 0x80000000u));
}
__device__ __forceinline__ uint64_t key_of(float v, int c) { return (uint64_t)ordered(v + 0.0f) << 32 | (uint32_t)~c; }
__device__ __forceinline__ int index_of(uint64_t key) { return (int)~(uint32_t)key; }

// A value joined over groups of kG lanes (16 or 64), the same in each of them
template <int kControl> __device__ __forceinline__ uint32_t rotated(uint32_t v) {
    return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, kControl, 0xf, 0xf, true);
}
template <int kG, class V, class F> __device__ __forceinline__ V join(V v, F f) {
    static_assert(sizeof(V) == 4, "");
    auto turn = [&](uint32_t o) { v = f(v, __builtin_bit_cast(V, o)); };
    turn(rotated<0x128>(__builtin_bit_cast(uint32_t, v)));    // row_ror of 8, 4, 2, 1
    turn(rotated<0x124>(__builtin_bit_cast(uint32_t, v)));
    turn(rotated<0x122>(__builtin_bit_cast(uint32_t, v)));
    turn(rotated<0x121>(__builtin_bit_cast(uint32_t, v)));
    if constexpr (kG == 64) {
        uint32_t u = __builtin_bit_cast(uint32_t, v);
        u32x2 r = __builtin_bit_cast(u32x2, __builtin_amdgcn_permlane16_swap(u, u, false, false));
        v = f(__builtin_bit_cast(V, (uint32_t)r[0]), __builtin_bit_cast(V, (uint32_t)r[1]));
        u = __builtin_bit_cast(uint32_t, v);
        r = __builtin_bit_cast(u32x2, __builtin_amdgcn_permlane32_swap(u, u, false, false));
        v = f(__builtin_bit_cast(V, (uint32_t)r[0]), __builtin_bit_cast(V, (uint32_t)r[1]));
    }
    return v;
}
template <int kG> __device__ __forceinline__ float sum_of(float v) { return join<kG>(v, [](float a, float b) { return a + b; }); }
template <int kG> __device__ __forceinline__ float max_of(float v) {
    return join<kG>(v, [](float a, float b) { return __builtin_fmaxf(a, b); });
}

__device__ __forceinline__ int64_t target_at(const void *t, int bytes, int64_t row) {
    return bytes == 8 ? ((const int64_t *)t)[row] : ((const int32_t *)t)[row];
}

struct Sums {
    float m, n, r, s;
    __device__ __forceinline__ void clear() { m = kLowest, n = r = s = 0; }
    // to the maximum `to`, at least m, and by far so where entries are masked by the type's lowest value: w d must not overflow,
    // as f would make it 0 times infinity
    __device__ __forceinline__ void move(float to) {
        const float d = __builtin_fmaxf(m - to, kGone), f = exp_of(d), w = r + n;
        const bool same = m == to;
        s = same ? s : f * __builtin_fmaf(w, d, s);
        r = same ? r : f * w;
        n = same ? n : 0.0f;
        m = to;
    }
    // values none of which is above m; -inf ones add nothing
    template <int kN> __device__ __forceinline__ void add(const float *v) {
        int count = 0;
#pragma unroll
        for (int j = 0; j < kN; j++) {
            const float d = v[j] - m, e = exp_of(d);
            const bool at = d == 0.0f;
            count += at;
            r += at ? 0.0f : e;
            s = __builtin_fmaf(e, __builtin_fmaxf(d, kLowest), s);
        }
        n += (float)count;
    }
    template <int kG> __device__ __forceinline__ void join_lanes() {
        move(max_of<kG>(m));
        n = sum_of<kG>(n);
        r = sum_of<kG>(r);
        s = sum_of<kG>(s);
    }
};

// What a row's sums give
struct Row {
    float m, logz, entropy;
    bool bad, none;
    __device__ __forceinline__ void of(const Sums &a) {
        bad = !(a.r == a.r);
        none = !bad && a.n + a.r == 0;
        const float nan = __builtin_nanf("");
        logz = bad ? nan : none ? 0.0f : log1pf(a.n - 1 + a.r);
        entropy = none ? 0.0f : logz - a.s / (a.n + a.r);
        m = bad ? nan : none ? -INFINITY : a.m;
    }
    __device__ __forceinline__ float logp(float v) const { return v - m - logz; }
};
// by one lane: a row's outputs but its alternatives; v: the target's logit
__device__ __forceinline__ void put_row(const LogprobsArgs &a, int64_t row, const Row &o, int64_t t, float v) {
    a.entropy[row] = o.entropy;
    if (a.stats) a.stats[row] = make_float2(o.m, o.logz);
    if (a.target_bytes) {
        const float nan = __builtin_nanf("");
        a.logp[row] = t == -1 ? 0.0f : t < 0 || t >= a.V ? nan : o.none ? -INFINITY : o.logp(v);
    }
}
// the alternative at place k, or that there is none (key 0)
__device__ __forceinline__ void put_top(const LogprobsArgs &a, int64_t row, int k, uint64_t key, const Row &o) {
    a.top_ids[row * a.top + k] = key ? index_of(key) : -1;
    a.top_logp[row * a.top + k] = o.bad ? __builtin_nanf("") : key ? o.logp(unordered((uint32_t)(key >> 32))) : -INFINITY;
}

// the wave's own writes to LDS before its reads after
__device__ __forceinline__ void wave_sync() {
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
}
__device__ __forceinline__ uint64_t max_key(uint64_t v, int lanes) {
    for (int o = lanes / 2; o; o >>= 1) {
        const uint64_t u = __shfl_xor(v, o);
        v = u > v ? u : v;
    }
    return v;
}

// The top-th largest of 16 lanes' values, ties by lane (-inf: there are fewer), the same in each of them
__device__ __forceinline__ float bound_of_16(float most, int top) {
    const int l = threadIdx.x & 15;
    int above = 0;
    auto turn = [&](uint32_t u, int by) {
        const float w = __builtin_bit_cast(float, u);
        above += w > most || (w == most && (l - by & 15) < l);     // row_ror by `by`: lane l has lane l - by's
    };
    const uint32_t u = __builtin_bit_cast(uint32_t, most);
    turn(rotated<0x121>(u), 1), turn(rotated<0x122>(u), 2), turn(rotated<0x123>(u), 3), turn(rotated<0x124>(u), 4);
    turn(rotated<0x125>(u), 5), turn(rotated<0x126>(u), 6), turn(rotated<0x127>(u), 7), turn(rotated<0x128>(u), 8);
    turn(rotated<0x129>(u), 9), turn(rotated<0x12a>(u), 10), turn(rotated<0x12b>(u), 11), turn(rotated<0x12c>(u), 12);
    turn(rotated<0x12d>(u), 13), turn(rotated<0x12e>(u), 14), turn(rotated<0x12f>(u), 15);
    return max_of<16>(above == top - 1 ? most : -INFINITY);
}
// of a wave's 64
__device__ __forceinline__ float bound_of_64(float most, int top) {
    const int l = threadIdx.x & 63;
    int above = 0;
#pragma unroll
    for (int i = 0; i < 64; i++) {
        const float w = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, most), i));
        above += w > most || (w == most && i < l);
    }
    return max_of<64>(above == top - 1 ? most : -INFINITY);
}
// the largest of lanes l, l + 16, l + 32, l + 48
__device__ __forceinline__ float max_of_rows(float v) {
    uint32_t u = __builtin_bit_cast(uint32_t, v);
    u32x2 r = __builtin_bit_cast(u32x2, __builtin_amdgcn_permlane16_swap(u, u, false, false));
    v = __builtin_fmaxf(__builtin_bit_cast(float, (uint32_t)r[0]), __builtin_bit_cast(float, (uint32_t)r[1]));
    u = __builtin_bit_cast(uint32_t, v);
    r = __builtin_bit_cast(u32x2, __builtin_amdgcn_permlane32_swap(u, u, false, false));
    return __builtin_fmaxf(__builtin_bit_cast(float, (uint32_t)r[0]), __builtin_bit_cast(float, (uint32_t)r[1]));
}

// Rows of up to kG kC kU entries, kG lanes a row with the row in their registers: a wave's arithmetic runs while the others' rows
// are on their way. 262144 rows of 256 f32 with 5 alternatives, 4 rows a wave: 67 us for 55 at a large copy's rate, VALU and
// reading both busy.
template <class T, int kG, int kU> __global__ __launch_bounds__(256) void narrow_kernel(LogprobsArgs a) {
    constexpr int kC = 16 / sizeof(T), kN = kU * kC, kRows = 256 / kG;
    __shared__ uint64_t keys[256];
    const int l = threadIdx.x % kG, at = threadIdx.x - l;
    const int64_t mine = (int64_t)blockIdx.x * kRows + threadIdx.x / kG, row = min(mine, a.rows - 1);
    const bool live = mine < a.rows;
    const T *x = (const T *)a.x + row * a.stride;
    int64_t t = -1;
    if (a.target_bytes) t = target_at(a.targets, a.target_bytes, row);
    float v[kN];
    if (a.V == kG * kN) {
        u32x4 c[kU];
#pragma unroll
        for (int u = 0; u < kU; u++) c[u] = load16(x + (u * kG + l) * kC);
#pragma unroll
        for (int u = 0; u < kU; u++) unpack(c[u], v + u * kC, T{});
    } else {
#pragma unroll
        for (int u = 0; u < kU; u++) {
            const int first = (u * kG + l) * kC, n = a.V - first;
            unpack(a.V >= kC ? load16_end(x + first, n) : load16(x + min(first, a.V - 1), n), v + u * kC, T{});
#pragma unroll
            for (int j = 0; j < kC; j++) v[u * kC + j] = j < n ? v[u * kC + j] : -INFINITY;
        }
    }
    const float vt = t >= 0 && t < a.V ? to_f32(x[t]) : 0.0f;
    float most = v[0];
#pragma unroll
    for (int j = 1; j < kN; j++) most = __builtin_fmaxf(most, v[j]);
    Sums z;
    z.clear();
    z.m = max_of<kG>(__builtin_fmaxf(most, kLowest));
    z.add<kN>(v);
    z.n = sum_of<kG>(z.n);
    z.r = sum_of<kG>(z.r);
    z.s = sum_of<kG>(z.s);
    Row o;
    o.of(z);
    if (live && l == 0) put_row(a, row, o, t, vt);
    if (!a.top) return;
    const float bound = kG == 16 || a.top <= 8 ? bound_of_16(kG == 16 ? most : max_of_rows(most), a.top) : bound_of_64(most, a.top);
    uint32_t reach = 0;
#pragma unroll
    for (int j = 0; j < kN; j++) reach |= (v[j] >= bound && v[j] > -INFINITY ? 1u : 0u) << j;
    if (o.bad) reach = 0;
    // how many reach it in the lanes before mine, and in all: sums over the lanes to the left, row_shr of 1, 2, 4, 8 (zeros come
    // in) and, past 16 lanes, the rows' last ones to the rows after (row_bcast 15 and 31)
    const int count = __popc(reach);
    int place = count, all;
    place += (int)__builtin_amdgcn_update_dpp(0, place, 0x111, 0xf, 0xf, true);
    place += (int)__builtin_amdgcn_update_dpp(0, place, 0x112, 0xf, 0xf, true);
    place += (int)__builtin_amdgcn_update_dpp(0, place, 0x114, 0xf, 0xf, true);
    place += (int)__builtin_amdgcn_update_dpp(0, place, 0x118, 0xf, 0xf, true);
    if constexpr (kG == 16) {
        all = join<16>(place, [](int p, int q) { return max(p, q); });
    } else {
        place += (int)__builtin_amdgcn_update_dpp(0, place, 0x142, 0xa, 0xf, false);
        place += (int)__builtin_amdgcn_update_dpp(0, place, 0x143, 0xc, 0xf, false);
        all = __builtin_amdgcn_readlane(place, 63);
    }
    place -= count;
    if (__all(all <= kG)) {
        while (__any(reach != 0)) {
            if (reach) {
                const int j = __builtin_ctz(reach);
                keys[at + place] = (j / kC * kG + l) * kC + j % kC;
                reach &= reach - 1;
                place++;
            }
        }
        wave_sync();
        int c = 0;
        uint64_t key = 0;
        if (l < all) {
            c = (int)keys[threadIdx.x];
            key = key_of(to_f32(x[c]), c);
        }
        wave_sync();
        keys[threadIdx.x] = key;
        wave_sync();
        int rank = 0;
        const int longest = kG == 64 ? all : max(max(__builtin_amdgcn_readlane(all, 0), __builtin_amdgcn_readlane(all, 16)),
                                                 max(__builtin_amdgcn_readlane(all, 32), __builtin_amdgcn_readlane(all, 48)));
        for (int i = 0; i < longest; i++) rank += keys[at + i] > key;
        if (live) {
            if (l < all && rank < a.top) put_top(a, row, rank, key, o);
            for (int i = l; i < a.top; i += kG)
                if (i >= all) put_top(a, row, i, 0, o);
        }
        return;
    }
    uint64_t last = ~0ull;
    for (int k = 0; k < a.top; k++) {
        uint64_t best = 0;
        for (int c = l; c < a.V; c += kG) {      // from the cache: the registers are not held for this
            const float u = to_f32(x[c]);
            const uint64_t key = key_of(u, c);
            if (u > -INFINITY && key < last && key > best) best = key;
        }
        last = max_key(o.bad ? 0 : best, kG);
        if (live && l == 0) put_top(a, row, k, last, o);
    }
}

// Wide rows: a workgroup of 256 takes a row, or one of `parts` parts of `width` entries, in one pass (and a second over what
// the L2 holds, for the alternatives); wide_join_kernel joins the parts.
constexpr int kHold = 1024;    // entries gathered at most
struct Wide {
    int parts, width;
    float4 *sums;       // (rows, parts)
    uint64_t *keys;     // (rows, parts, top), falling, then zeros
};

// calls f(values, index of the first, count) for the row's entries from c0 to c1, kU pieces of 16 bytes a thread at a time, and
// what is left by one
template <class T, int kU, class F> __device__ __forceinline__ void for_pieces(const T *x, int c0, int c1, F f) {
    constexpr int kC = 16 / sizeof(T), kN = kU * kC, kSpan = 256 * kN;
    const int l = threadIdx.x;
    int c = c0;
    for (; c + kSpan <= c1; c += kSpan) {
        u32x4 p[kU];
        float v[kN];
#pragma unroll
        for (int u = 0; u < kU; u++) p[u] = load16(x + c + (u * 256 + l) * kC);
#pragma unroll
        for (int u = 0; u < kU; u++) unpack(p[u], v + u * kC, T{});
        f(v, c + l * kC, std::integral_constant<int, kN>());
    }
    for (; c < c1; c += 256 * kC) {
        float v[kC];
        const int first = c + l * kC, n = c1 - first;
        unpack(load16_end(x + first, n), v, T{});      // c1 is past a whole piece of the row
#pragma unroll
        for (int j = 0; j < kC; j++) v[j] = j < n ? v[j] : -INFINITY;
        f(v, first, std::integral_constant<int, kC>());
    }
}

struct TopShared {
    uint64_t keys[kHold];
    uint64_t best[4];
    float most[256];
    int count;
};
// the keys' places among each other: put(place, key), then put(place, 0) up to top
template <class F> __device__ __forceinline__ void put_ranked(const TopShared &sh, int count, int top, F put) {
    for (int i = threadIdx.x; i < count; i += 256) {
        const uint64_t key = sh.keys[i];
        int rank = 0;
        for (int j = 0; j < count; j++) rank += sh.keys[j] > key;
        if (rank < top) put(rank, key);
    }
    for (int i = count + threadIdx.x; i < top; i += 256) put(i, 0);
}

template <class T, int kU> __global__ __launch_bounds__(256) void wide_kernel(LogprobsArgs a, Wide w) {
    constexpr int kC = 16 / sizeof(T);
    __shared__ Sums waves[4];
    __shared__ TopShared sh;
    const int64_t row = blockIdx.x / w.parts;
    const int part = blockIdx.x % w.parts, tid = threadIdx.x;
    const T *x = (const T *)a.x + row * a.stride;
    const int c0 = min((int64_t)part * w.width, (int64_t)a.V), c1 = (int)min((int64_t)c0 + w.width, (int64_t)a.V);
    Sums z;
    z.clear();
    for_pieces<T, kU>(x, c0, c1, [&](const float *v, int, auto count) {
        constexpr int kN = decltype(count)::value;
        float most = v[0];
#pragma unroll
        for (int j = 1; j < kN; j++) most = __builtin_fmaxf(most, v[j]);
        z.move(__builtin_fmaxf(z.m, most));
        z.add<kN>(v);
    });
    const float most = z.n > 0 ? z.m : -INFINITY;     // the thread's largest value
    z.join_lanes<64>();
    if ((tid & 63) == 0) waves[tid >> 6] = z;
    if (a.top) {
        sh.most[tid] = most;
        if (tid == 0) sh.count = 0;
    }
    __syncthreads();
    float m = waves[0].m;
#pragma unroll
    for (int i = 1; i < 4; i++) m = __builtin_fmaxf(m, waves[i].m);
    z = waves[0];
    z.move(m);
#pragma unroll
    for (int i = 1; i < 4; i++) {
        Sums y = waves[i];
        y.move(m);
        z.n += y.n;
        z.r += y.r;
        z.s += y.s;
    }
    Row o;
    o.of(z);
    if (tid == 0) {
        if (w.parts > 1) {
            w.sums[row * w.parts + part] = make_float4(z.m, z.n, z.r, z.s);
        } else {
            int64_t t = -1;
            if (a.target_bytes) t = target_at(a.targets, a.target_bytes, row);
            put_row(a, row, o, t, t >= 0 && t < a.V ? to_f32(x[t]) : 0.0f);
        }
    }
    if (!a.top) return;
    uint64_t *keys = w.keys + (row * w.parts + part) * a.top;
    auto put = [&](int k, uint64_t key) {
        if (w.parts > 1) keys[k] = key;
        else put_top(a, row, k, key, o);
    };
    // the top-th largest of 64 maxima, those of the threads tid, tid + 64, ...
    const int l = tid & 63;
    const float mine = __builtin_fmaxf(__builtin_fmaxf(sh.most[l], sh.most[l + 64]), __builtin_fmaxf(sh.most[l + 128], sh.most[l + 192]));
    const float bound = a.top <= 8 ? bound_of_16(max_of_rows(mine), a.top) : bound_of_64(mine, a.top);
    if (!o.bad && most >= bound) {      // few threads have an entry that reaches it
        for_pieces<T, kU>(x, c0, c1, [&](const float *v, int c, auto count) {
            constexpr int kN = decltype(count)::value;
#pragma unroll
            for (int j = 0; j < kN; j++) {
                if (v[j] >= bound && v[j] > -INFINITY) {
                    const int i = atomicAdd(&sh.count, 1);
                    if (i < kHold) sh.keys[i] = key_of(v[j], c + j / kC * 256 * kC + j % kC);
                }
            }
        });
    }
    __syncthreads();
    const int count = sh.count;
    if (count <= kHold) {
        put_ranked(sh, count, a.top, put);
        return;
    }
    uint64_t last = ~0ull;
    for (int k = 0; k < a.top; k++) {
        uint64_t best = 0;
        for_pieces<T, 1>(x, c0, c1, [&](const float *v, int c, auto) {
#pragma unroll
            for (int j = 0; j < kC; j++) {
                const uint64_t key = key_of(v[j], c + j);
                if (v[j] > -INFINITY && key < last && key > best) best = key;
            }
        });
        best = max_key(best, 64);
        __syncthreads();
        if ((tid & 63) == 0) sh.best[tid >> 6] = best;
        __syncthreads();
        last = max(max(sh.best[0], sh.best[1]), max(sh.best[2], sh.best[3]));
        if (tid == 0) put(k, last);
    }
}

// A row's parts, at most 64, joined by a workgroup. Each part's keys fall; with j = ceil(top / parts), the top-th largest of
// the parts' first keys (j = 1) or the least of their j th bounds the row's: at least `top` of the parts' keys reach it.
template <class T> __global__ __launch_bounds__(256) void wide_join_kernel(LogprobsArgs a, Wide w) {
    constexpr int kFirst = 4;
    __shared__ TopShared sh;
    const int64_t row = blockIdx.x;
    const int tid = threadIdx.x, l = tid & 63;
    const T *x = (const T *)a.x + row * a.stride;
    const uint64_t *keys = w.keys + row * w.parts * a.top;
    const int j = (a.top + w.parts - 1) / w.parts, all = w.parts * a.top;
    // every load that waits for none: together
    int64_t t = -1;
    if (a.target_bytes) t = target_at(a.targets, a.target_bytes, row);
    const float4 s = w.sums[row * w.parts + min(l, w.parts - 1)];
    uint64_t mine = 0, first[kFirst] = {};
    if (a.top) {
        mine = keys[min(l, w.parts - 1) * a.top + j - 1];
#pragma unroll
        for (int i = 0; i < kFirst; i++) first[i] = keys[min(tid + 256 * i, all - 1)];
    }
    if (tid == 0) sh.count = 0;
    const float vt = t >= 0 && t < a.V ? to_f32(x[t]) : 0.0f;
    Sums z;
    z.clear();
    if (l < w.parts) z.m = s.x, z.n = s.y, z.r = s.z, z.s = s.w;
    else mine = 0;
    z.join_lanes<64>();
    Row o;
    o.of(z);
    if (tid == 0) put_row(a, row, o, t, vt);
    if (!a.top) return;
    uint64_t bound;
    if (j == 1) {
        int above = 0;
        for (int i = 0; i < w.parts; i++) {
            const uint64_t v = (uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(mine >> 32), i) << 32 |
                               (uint32_t)__builtin_amdgcn_readlane((int)mine, i);
            above += v > mine || (v == mine && i < l);
        }
        bound = max_key(l < w.parts && above == a.top - 1 ? mine : 0, 64);
    } else {
        bound = ~max_key(l < w.parts ? ~mine : 0, 64);
    }
    __syncthreads();
    auto keep = [&](uint64_t key) {
        if (key && key >= bound) {
            const int at = atomicAdd(&sh.count, 1);
            if (at < kHold) sh.keys[at] = key;
        }
    };
    if (!o.bad) {
#pragma unroll
        for (int i = 0; i < kFirst; i++)
            if (tid + 256 * i < all) keep(first[i]);
        for (int i = tid + 256 * kFirst; i < all; i += 256) keep(keys[i]);
    }
    __syncthreads();
    const int count = sh.count;
    auto put = [&](int k, uint64_t key) { put_top(a, row, k, key, o); };
    if (count <= kHold) {
        put_ranked(sh, count, a.top, put);
        return;
    }
    uint64_t last = ~0ull;
    for (int k = 0; k < a.top; k++) {
        uint64_t best = 0;
        for (int i = tid; i < all; i += 256) {
            const uint64_t key = keys[i];
            if (key < last && key > best) best = key;
        }
        best = max_key(best, 64);
        __syncthreads();
        if (l == 0) sh.best[tid >> 6] = best;
        __syncthreads();
        last = max(max(sh.best[0], sh.best[1]), max(sh.best[2], sh.best[3]));
        if (tid == 0) put(k, last);
    }
}

// dx_c = [c = t] g - p_c (g + sum_k g_k) + sum_k [c = id_k] g_k - g_H p_c (logp_c + H). 2^shift threads a row, or `blocks`
// workgroups of them (shift 8); a thread takes kU pieces of 16 bytes.
template <class T, int kU> __global__ __launch_bounds__(256) void grad_kernel(LogprobsGradArgs a, int shift, int blocks) {
    constexpr int kC = 16 / sizeof(T);
    const int64_t row = ((int64_t)(blockIdx.x / blocks) << (8 - shift)) + (threadIdx.x >> shift);
    if (row >= a.rows) return;
    const int l = threadIdx.x & ((1 << shift) - 1), c0 = (blockIdx.x % blocks * kU * 256 + l) * kC;
    const T *x = (const T *)a.x + row * a.stride;
    T *dx = (T *)a.dx + row * a.V;
    const float2 st = a.stats[row];
    const float H = a.entropy[row], gh = a.g_entropy ? a.g_entropy[row] : 0.0f;
    const int64_t t = a.g_logp ? target_at(a.targets, a.target_bytes, row) : -1;
    float g = 0;
    if (t != -1) g = t < 0 || t >= a.V ? __builtin_nanf("") : a.g_logp[row];
    float all = g;
    if (a.g_top)
        for (int k = 0; k < a.top; k++)
            if (a.top_ids[row * a.top + k] >= 0) all += a.g_top[row * a.top + k];
    const bool none = st.x == -INFINITY, bad = all != all;
    u32x4 p[kU];
    if (blocks > 1 && (int)(blockIdx.x % blocks + 1) * kU * 256 * kC <= a.V) {
#pragma unroll
        for (int u = 0; u < kU; u++) p[u] = load16(x + c0 + (u * kC << shift));
    } else {
#pragma unroll
        for (int u = 0; u < kU; u++) {
            const int c = c0 + (u * kC << shift);
            p[u] = a.V >= kC ? load16_end(x + c, a.V - c) : load16(x + min(c, a.V - 1), a.V - c);
        }
    }
#pragma unroll
    for (int u = 0; u < kU; u++) {
        const int c = c0 + (u * kC << shift);
        if (c >= a.V) break;
        float v[kC];
        unpack(p[u], v, T{});
#pragma unroll
        for (int j = 0; j < kC; j++) {
            const float lp = v[j] - st.x - st.y, q = exp_of(lp);
            const float d = -q * __builtin_fmaf(gh, lp + H, all);
            v[j] = q == 0 && !bad ? 0.0f : d;
        }
        if (t >= c && t < c + kC) {
#pragma unroll
            for (int j = 0; j < kC; j++) v[j] += c + j == t ? g : 0.0f;
        }
        if (a.g_top) {
            for (int k = 0; k < a.top; k++) {
                const int id = a.top_ids[row * a.top + k] - c;
                if (id < 0 || id >= kC) continue;
                const float gk = a.g_top[row * a.top + k];
#pragma unroll
                for (int j = 0; j < kC; j++) v[j] += j == id ? gk : 0.0f;
            }
        }
        if (none) {
#pragma unroll
            for (int j = 0; j < kC; j++) v[j] = 0.0f;
        }
        store_run<T, kC>(dx + c, v, a.V - c);
    }
}

constexpr int kNarrow = 2048;    // most entries of a row held in registers

// Parts of a wide row: enough workgroups for 4 a CU, each of at least 4096 entries. Rows of up to 32768 are not worth the second
// launch (16 rows of 10426: 15 us in parts, 10 whole).
int parts_of(int64_t rows, int V) {
    if (V <= 32768) return 1;
    const int64_t want = (1024 + rows - 1) / rows, most = (V + 4095) / 4096;
    return (int)(want < most ? want < 64 ? want : 64 : most < 64 ? most : 64);
}

// the arguments from row n on
template <class P> void move_on(P *&p, int64_t n) {
    if (p) p += n;
}
void move_on(const void *&p, int64_t bytes) { p = p ? (const char *)p + bytes : p; }
void skip_rows(LogprobsArgs &a, int64_t n, int size) {
    move_on(a.x, n * a.stride * size), move_on(a.targets, n * a.target_bytes);
    move_on(a.logp, n), move_on(a.entropy, n), move_on(a.stats, n);
    move_on(a.top_logp, n * a.top), move_on(a.top_ids, n * a.top);
}
void skip_rows(LogprobsGradArgs &a, int64_t n, int size) {
    move_on(a.x, n * a.stride * size), move_on(a.targets, n * a.target_bytes);
    move_on(a.entropy, n), move_on(a.stats, n), move_on(a.top_ids, n * a.top);
    move_on(a.g_logp, n), move_on(a.g_entropy, n), move_on(a.g_top, n * a.top);
    a.dx = (char *)a.dx + n * a.V * size;
}
// launch(a) for up to `most` rows at a time: what one launch takes
template <class T, class A, class F> hipError_t by_rows(A a, int64_t most, F launch) {
    const int64_t rows = a.rows;
    for (int64_t done = 0;; skip_rows(a, most, sizeof(T))) {     // only to rows that there are: a single one may have any stride
        a.rows = rows - done < most ? rows - done : most;
        launch(a);
        if (hipError_t e = hipGetLastError()) return e;
        done += a.rows;
        if (done == rows) return hipSuccess;
    }
}

template <class T> hipError_t go(const LogprobsArgs &a, void *scratch, hipStream_t st) {
    constexpr int kC = 16 / sizeof(T);
    auto narrow = [&](auto g, auto u) {
        constexpr int kG = decltype(g)::value, kU = decltype(u)::value, kRows = 256 / kG;
        return by_rows<T>(a, most_blocks(256) * kRows, [&](const LogprobsArgs &b) {
            hipLaunchKernelGGL((narrow_kernel<T, kG, kU>), dim3((unsigned)((b.rows + kRows - 1) / kRows)), dim3(256), 0, st, b);
        });
    };
    using std::integral_constant;
    // 16 lanes hold 8 alternatives with room for as many more that reach the bound, or all of 16 classes
    if ((a.V <= 256 && a.top <= 8) || a.V <= 16) {
        if (a.V <= 16 * kC) return narrow(integral_constant<int, 16>(), integral_constant<int, 1>());
        return narrow(integral_constant<int, 16>(), integral_constant<int, 16 / kC>());
    }
    if (a.V <= 64 * kC) return narrow(integral_constant<int, 64>(), integral_constant<int, 1>());
    if (kC == 4 && a.V <= 512) return narrow(integral_constant<int, 64>(), integral_constant<int, 2>());
    if (a.V <= 1024) return narrow(integral_constant<int, 64>(), integral_constant<int, 16 / kC>());
    if (a.V <= kNarrow) return narrow(integral_constant<int, 64>(), integral_constant<int, 32 / kC>());
    Wide w;
    w.parts = parts_of(a.rows, a.V);
    w.width = ((a.V + w.parts - 1) / w.parts + kC - 1) / kC * kC;
    w.sums = (float4 *)scratch;
    w.keys = (uint64_t *)((char *)scratch + (a.rows * w.parts * 16 + 255) / 256 * 256);
    const dim3 block(256);
    if (w.parts == 1) {
        return by_rows<T>(a, most_blocks(256), [&](const LogprobsArgs &b) {
            hipLaunchKernelGGL((wide_kernel<T, 4>), dim3((unsigned)b.rows), block, 0, st, b, w);
        });
    }
    // fewer than 1024 rows; 4096 entries at a time: a part
    hipLaunchKernelGGL((wide_kernel<T, 16 / kC>), dim3((unsigned)(a.rows * w.parts)), block, 0, st, a, w);
    hipLaunchKernelGGL(wide_join_kernel<T>, dim3((unsigned)a.rows), block, 0, st, a, w);
    return hipGetLastError();
}

template <class T> hipError_t go_grad(const LogprobsGradArgs &a, hipStream_t st) {
    constexpr int kC = 16 / sizeof(T), kU = 4;
    const int pieces = (a.V + kC - 1) / kC;
    int shift = 0;
    while (shift < 8 && (kU << shift) < pieces) shift++;
    const int blocks = shift < 8 ? 1 : (pieces + kU * 256 - 1) / (kU * 256);
    return by_rows<T>(a, most_blocks(256) / blocks << (8 - shift), [&](const LogprobsGradArgs &b) {
        const int64_t grid = ((b.rows + (1 << (8 - shift)) - 1) >> (8 - shift)) * blocks;
        hipLaunchKernelGGL((grad_kernel<T, kU>), dim3((unsigned)grid), dim3(256), 0, st, b, shift, blocks);
    });
}

}  // namespace

int64_t logprobs_scratch(int, int64_t rows, int V, int top) {
    const int64_t parts = parts_of(rows, V);
    return parts == 1 ? 0 : (rows * parts * 16 + 255) / 256 * 256 + rows * parts * top * 8;
}

hipError_t launch_logprobs(int type, const LogprobsArgs &a, void *scratch, hipStream_t st) {
    if (type == kOpF32) return go<float>(a, scratch, st);
    if (type == kOpBf16) return go<bf16_t>(a, scratch, st);
    return go<f16_t>(a, scratch, st);
}

hipError_t launch_logprobs_grad(int type, const LogprobsGradArgs &a, hipStream_t st) {
    if (type == kOpF32) return go_grad<float>(a, st);
    if (type == kOpBf16) return go_grad<bf16_t>(a, st);
    return go_grad<f16_t>(a, st);
}

}  // namespace ygg
