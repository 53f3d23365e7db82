// Activations held in 8 bits between forward and backward: packed and read back, and a gated block's silu(gate) * up that keeps its operands so.
//
// n values in blocks of 32 neighbours, the last one as short as it comes: s = the least bfloat16 with 127 s >= the largest magnitude, q = x / s to
// the nearest whole number (ties to the even one); the value held is q * s, off by at most s / 2.  A block's scale has a code's own precision to spare
// (8 leading bits), so 127 * s and q * s are exact in fp32.  A block with an infinity or NaN has s = NaN and reads back as NaN: training must see it.
//
// HBM-bound: a lane takes 8 neighbours (one 16-byte load of 16-bit values), a block is the four lanes of a quad, its maximum two lane exchanges; one such
// piece a lane and 256 threads a workgroup (512 and 1024: the same or slower; codes stored past the caches: forward 19.3 -> 18.1 us at 1024 x 11008, but what
// reads them soon then waits for HBM, 2 us).  us and TB/s moved, operands from HBM: 16384 x 5120 fp32 packed 72 (5.8), read back 74 (5.6), call after call;
// packed and read back in turn 162 (5.1: each finds the caches full of what the other wrote).  8192 x 13824 bfloat16 through silu(gate) * up 160 (5.6), backward 158 (5.7);
// a large copy reaches 5.13.
#include <type_traits>
#include "q4_act8.hpp"

namespace q4 {

constexpr int kAct8Threads = 256;

template <typename T>
struct Act8Eight { T v[8]; };
struct Words4 { uint4_t w[1]; };
struct Words8 { uint4_t w[2]; };
template <typename T> using WordsOf = std::conditional_t<sizeof(T) == 4, Words8, Words4>;

template <typename T>
__device__ __forceinline__ Act8Eight<T> load_eight(const T* __restrict__ p, long i, long n) {
    if (i + 8 <= n) {
        WordsOf<T> w;
#pragma unroll
        for (int k = 0; k < (int)(sizeof(w) / 16); ++k) w.w[k] = reinterpret_cast<const uint4_t*>(p + i)[k];
        return __builtin_bit_cast(Act8Eight<T>, w);
    }
    Act8Eight<T> r;
#pragma unroll
    for (int e = 0; e < 8; ++e) r.v[e] = i + e < n ? p[i + e] : (T)0.f;
    return r;
}
template <typename T>
__device__ __forceinline__ void store_eight(T* __restrict__ p, long i, long n, const Act8Eight<T>& r) {
    if (i + 8 <= n) {
        const WordsOf<T> w = __builtin_bit_cast(WordsOf<T>, r);
#pragma unroll
        for (int k = 0; k < (int)(sizeof(w) / 16); ++k) reinterpret_cast<uint4_t*>(p + i)[k] = w.w[k];
        return;
    }
#pragma unroll
    for (int e = 0; e < 8; ++e)
        if (i + e < n) p[i + e] = r.v[e];
}
// eight codes are 8 bytes; a code array is 16-byte aligned and i a multiple of 8
__device__ __forceinline__ uint2_t load_codes(const int8_t* __restrict__ p, long i, long n) {
    if (i + 8 <= n) return *reinterpret_cast<const uint2_t*>(p + i);
    uint32_t w[2] = {0, 0};
#pragma unroll
    for (int e = 0; e < 8; ++e)
        if (i + e < n) w[e / 4] |= (uint32_t)(uint8_t)p[i + e] << (8 * (e % 4));
    return uint2_t{w[0], w[1]};
}
__device__ __forceinline__ void store_codes(int8_t* __restrict__ p, long i, long n, uint2_t w) {
    if (i + 8 <= n) {
        *reinterpret_cast<uint2_t*>(p + i) = w;
        return;
    }
#pragma unroll
    for (int e = 0; e < 8; ++e)
        if (i + e < n) p[i + e] = (int8_t)((e < 4 ? w.x : w.y) >> (8 * (e % 4)));
}

// Codes and scale of the quad's block from this lane's eight values; all four lanes take part.
template <typename T>
__device__ __forceinline__ uint2_t encode(const Act8Eight<T>& r, uint32_t* scale) {
    float x[8];
    uint32_t top = 0;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        x[e] = (float)r.v[e];
        const uint32_t mag = __float_as_uint(x[e]) & 0x7FFFFFFFu;            // as whole numbers magnitudes keep their order, infinity and NaN on top
        top = mag > top ? mag : top;
    }
    top = quad_max(top);
    const uint32_t sb = act8_scale(top);
    *scale = sb;
    float s = __uint_as_float(sb);
    const bool some = s > 0.f;                                               // neither zero nor NaN
    if constexpr (!__is_same(T, half_t)) {                 // fp16 has no values so small that 1 / s is out of range
        const float lift = s < 0x1p-100f ? 0x1p64f : 1.f;
        s *= lift;
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e] *= lift;
    }
    const float inv = 1.f / s, half = 0.5f * s;
    uint32_t w[2] = {0, 0};
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        // x * inv is the quotient to 2^-16: its nearest whole number is right, or one off beside a tie; x - q s is exact and tells
        float q = rintf(x[e] * inv);
        const float rest = fmaf(-q, s, x[e]), off = fabsf(rest);
        const bool odd = ((int)q & 1) != 0;
        if (off > half || (off == half && odd)) q += copysignf(1.f, rest);
        const uint32_t code = some ? (uint32_t)(int)q & 0xFFu : 0u;
        w[e / 4] |= code << (8 * (e % 4));
    }
    return uint2_t{w[0], w[1]};
}

template <typename T>
__global__ __launch_bounds__(kAct8Threads) void act8_pack_kernel(const T* __restrict__ x, int8_t* __restrict__ codes, uint16_t* __restrict__ scales, long n) {
    const long c = (long)blockIdx.x * kAct8Threads + threadIdx.x;
    if (c >= act8_blocks(n) * 4) return;                                     // quads stay together
    uint32_t sb;
    const uint2_t w = encode(load_eight(x, 8 * c, n), &sb);
    store_codes(codes, 8 * c, n, w);
    if (c % 4 == 0) scales[c / 4] = (uint16_t)(sb >> 16);
}

template <typename T>
__global__ __launch_bounds__(kAct8Threads) void act8_unpack_kernel(const int8_t* __restrict__ codes, const uint16_t* __restrict__ scales, T* __restrict__ x, long n) {
    const long c = (long)blockIdx.x * kAct8Threads + threadIdx.x;
    if (8 * c >= n) return;
    const Decode<T> d(scales[c / 4]);
    const uint2_t w = load_codes(codes, 8 * c, n);
    Act8Eight<T> r;
#pragma unroll
    for (int e = 0; e < 8; ++e) r.v[e] = (T)d.value(w, e);
    store_eight(x, 8 * c, n, r);
}

// 1 / (1 + exp(-x)); zero where it would be less than the least normal fp32, below -87
__device__ __forceinline__ float sigmoid(float x) { return __builtin_amdgcn_rcpf(1.f + __expf(-x)); }

// out = silu(gate) * up from the operands as they are, in fp32 and rounded once; KEEP: both operands kept in 8 bits.
template <typename T, bool KEEP>
__global__ __launch_bounds__(kAct8Threads) void silu_mul_act8_kernel(const T* __restrict__ gate, const T* __restrict__ up, T* __restrict__ out, q4_act8_t kg, q4_act8_t ku,
                                                                     long n) {
    const long c = (long)blockIdx.x * kAct8Threads + threadIdx.x;
    if (c >= act8_blocks(n) * 4) return;
    const Act8Eight<T> g = load_eight(gate, 8 * c, n), u = load_eight(up, 8 * c, n);
    Act8Eight<T> o;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        const float x = (float)g.v[e];
        o.v[e] = (T)(x * sigmoid(x) * (float)u.v[e]);
    }
    store_eight(out, 8 * c, n, o);
    if constexpr (KEEP) {
        uint32_t gs, us;
        const uint2_t gw = encode(g, &gs), uw = encode(u, &us);
        store_codes((int8_t*)kg.codes, 8 * c, n, gw);
        store_codes((int8_t*)ku.codes, 8 * c, n, uw);
        if (c % 4 == 0) {
            ((uint16_t*)kg.scales)[c / 4] = (uint16_t)(gs >> 16);
            ((uint16_t*)ku.scales)[c / 4] = (uint16_t)(us >> 16);
        }
    }
}

// d/dgate and d/dup of silu(gate) * up at the values held: dout * up * s (1 + gate (1 - s)) and dout * gate * s with s = sigmoid(gate).
template <typename T>
__global__ __launch_bounds__(kAct8Threads) void silu_mul_act8_bwd_kernel(const T* __restrict__ dout, const int8_t* __restrict__ gate_codes,
                                                                         const uint16_t* __restrict__ gate_scales, const int8_t* __restrict__ up_codes,
                                                                         const uint16_t* __restrict__ up_scales, T* __restrict__ dgate, T* __restrict__ dup,
                                                                         long n) {
    const long c = (long)blockIdx.x * kAct8Threads + threadIdx.x;
    if (8 * c >= n) return;
    const Decode<T> dg(gate_scales[c / 4]), du(up_scales[c / 4]);
    const uint2_t gw = load_codes(gate_codes, 8 * c, n), uw = load_codes(up_codes, 8 * c, n);
    const Act8Eight<T> d = load_eight(dout, 8 * c, n);
    Act8Eight<T> a, b;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        const float x = dg.value(gw, e), y = (float)d.v[e], s = sigmoid(x);
        a.v[e] = (T)(y * (du.value(uw, e) * (s * fmaf(x, 1.f - s, 1.f))));   // the factor within (-0.1, 1.1) first: nothing overflows on the way
        b.v[e] = (T)(y * (x * s));
    }
    store_eight(dgate, 8 * c, n, a);
    store_eight(dup, 8 * c, n, b);
}

inline dim3 act8_grid(long n) { return dim3((unsigned)((act8_blocks(n) * 4 + kAct8Threads - 1) / kAct8Threads)); }

template <typename F>
int by_type16(int type, F&& launch) {
    if (type == Q4_TYPE_BF16) launch((__bf16)0.f);
    else launch((half_t)0.f);
    return hipGetLastError() == hipSuccess ? 0 : -4;
}
template <typename F>
int by_type(int type, F&& launch) {
    if (type != Q4_TYPE_F32) return by_type16(type, launch);
    launch(0.f);
    return hipGetLastError() == hipSuccess ? 0 : -4;
}

}  // namespace q4

int q4_launch_act8_pack(const void* x, int type, void* codes, void* scales, long n, hipStream_t stream) {
    using namespace q4;
    return by_type(type, [&](auto t) {
        hipLaunchKernelGGL(act8_pack_kernel<decltype(t)>, act8_grid(n), dim3(kAct8Threads), 0, stream, (const decltype(t)*)x, (int8_t*)codes,
                           (uint16_t*)scales, n);
    });
}

int q4_launch_act8_unpack(const void* codes, const void* scales, void* x, int type, long n, hipStream_t stream) {
    using namespace q4;
    return by_type(type, [&](auto t) {
        hipLaunchKernelGGL(act8_unpack_kernel<decltype(t)>, act8_grid(n), dim3(kAct8Threads), 0, stream, (const int8_t*)codes, (const uint16_t*)scales,
                           (decltype(t)*)x, n);
    });
}

int q4_launch_silu_mul_act8(const void* gate, const void* up, int type, void* out, const q4_act8_t* g, const q4_act8_t* u, long n, hipStream_t stream) {
    using namespace q4;
    return by_type16(type, [&](auto t) {
        using T = decltype(t);
        if (g) hipLaunchKernelGGL((silu_mul_act8_kernel<T, true>), act8_grid(n), dim3(kAct8Threads), 0, stream, (const T*)gate, (const T*)up, (T*)out, *g, *u, n);
        else hipLaunchKernelGGL((silu_mul_act8_kernel<T, false>), act8_grid(n), dim3(kAct8Threads), 0, stream, (const T*)gate, (const T*)up, (T*)out, q4_act8_t{}, q4_act8_t{}, n);
    });
}

int q4_launch_silu_mul_act8_bwd(const void* dout, int type, const q4_act8_t* g, const q4_act8_t* u, void* dgate, void* dup, long n, hipStream_t stream) {
    using namespace q4;
    return by_type16(type, [&](auto t) {
        using T = decltype(t);
        hipLaunchKernelGGL(silu_mul_act8_bwd_kernel<T>, act8_grid(n), dim3(kAct8Threads), 0, stream, (const T*)dout, (const int8_t*)g->codes,
                           (const uint16_t*)g->scales, (const int8_t*)u->codes, (const uint16_t*)u->scales, (T*)dgate, (T*)dup, n);
    });
}
