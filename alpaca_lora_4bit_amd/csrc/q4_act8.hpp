// Blocks of 32 values in 8 bits (q4_act8.hip): a block's scale, and the values that codes stand for.
#pragma once
#include "q4_common.hpp"
#include "q4_gptq.h"

namespace q4 {

__host__ __device__ __forceinline__ long act8_blocks(long n) { return (n + 31) / 32; }

// Largest of the quad's four values, in all four lanes.
__device__ __forceinline__ uint32_t quad_max(uint32_t v) {
    uint32_t o = (uint32_t)__builtin_amdgcn_mov_dpp((int)v, 0xB1, 0xF, 0xF, true);       // lanes 1 0 3 2
    v = o > v ? o : v;
    o = (uint32_t)__builtin_amdgcn_mov_dpp((int)v, 0x4E, 0xF, 0xF, true);                // lanes 2 3 0 1
    return o > v ? o : v;
}

// Bits (as fp32, the low 16 zero) of the least bfloat16 s with 127 s >= a for the magnitude a of these bits; NaN where that is none.
// a / 127 rounded up may be one bfloat16 off either way, for its own rounding; 127 s is exact and decides.
__device__ __forceinline__ uint32_t act8_scale(uint32_t top) {
    if (top > 0x7F7FFFFFu) return 0x7FC00000u;
    const float a = __uint_as_float(top);
    const uint32_t up = (__float_as_uint(a * (1.f / 127.f)) + 0xFFFFu) & 0xFFFF0000u;
    if (127.f * __uint_as_float(up) < a) return up + 0x10000u;
    return up != 0 && 127.f * __uint_as_float(up - 0x10000u) >= a ? up - 0x10000u : up;
}

template <typename T> struct TypeMax;
template <> struct TypeMax<half_t> { static constexpr float value = 65504.f; };
template <> struct TypeMax<__bf16> { static constexpr float value = 0x1.FEp127f; };
template <> struct TypeMax<float> { static constexpr float value = 0x1.FFFFFEp127f; };

// Values of a block: code * scale, no further out than T's largest number (127 s may be, where the block reaches to T's end); NaN for a scale of NaN.
template <typename T>
struct Decode {
    float s, nan;
    __device__ __forceinline__ explicit Decode(uint16_t bits) : s(__uint_as_float((uint32_t)bits << 16)), nan(0.f * s) {}
    __device__ __forceinline__ float value(uint2_t w, int e) const {
        const float q = (float)(int8_t)((e < 4 ? w.x : w.y) >> (8 * (e % 4)));
        return __builtin_amdgcn_fmed3f(q * s, -TypeMax<T>::value, TypeMax<T>::value) + nan;      // the middle one drops a NaN, the sum brings it back
    }
};

}  // namespace q4
