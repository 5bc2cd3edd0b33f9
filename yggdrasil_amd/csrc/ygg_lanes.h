// Values joined over the lanes of a wave, in the lanes' registers, and the order of workgroups.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "ygg_optype.h"

namespace ygg {

// A value joined over groups of kG lanes (1, 4, 16 or 64), the same in each of them
template <int kControl> __device__ __forceinline__ uint32_t rotated(uint32_t v) {
    return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, kControl, 0xf, 0xf, true);
}
template <int kG, class V, class F> __device__ __forceinline__ V join(V v, F f) {
    static_assert(sizeof(V) == 4, "");
    auto turn = [&](uint32_t o) { v = f(v, __builtin_bit_cast(V, o)); };
    if constexpr (kG == 1) return v;
    if constexpr (kG == 4) {
        turn(rotated<0xb1>(__builtin_bit_cast(uint32_t, v)));     // quad_perm 1 0 3 2, 2 3 0 1
        turn(rotated<0x4e>(__builtin_bit_cast(uint32_t, v)));
        return v;
    }
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

// Workgroups go round the 8 XCDs in turn, each with an L2 of its own: a run of neighbouring tiles to each
__device__ __forceinline__ int tile_of(int id, int tiles) {
    const int most = (tiles + 7) / 8, full = tiles - (most - 1) * 8;   // the first `full` XCDs have `most`
    const int x = id & 7;
    return (x < full ? x * most : full * most + (x - full) * (most - 1)) + (id >> 3);
}

}  // namespace ygg
