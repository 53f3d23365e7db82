// Appending to the 4-bit key/value cache (layout in q4_kv4.hpp) and reading places of it back.
//
//   append:  k' = R(pos) k,  scale = rn16(max|k'| / 6) over a group (10912 at most where that fits fp16),  code = nearest(k' / scale);  v likewise without R;  q' = R(pos) q
//   read:    rn16(code * scale)
//
// R turns the first `rot` dimensions by pairs, (x_i, x_{i + rot/2}) or (x_{2i}, x_{2i+1}), with cosine and sine from a float32 table
// [position][rot/2][2] (angles of far positions and stretched frequencies are the table's).  The rotation and the division are
// float32 with one rounding each; q' is rounded once, k' not at all before its code.
//
// Eight dimensions a lane (one 16-byte load), D/8 lanes a token; a wavefront takes 64*8/D neighbouring tokens of ONE head, so that the codes of
// four tokens, which lie side by side, leave together.  HBM-bound for prompts, latency for a decoded token (table row, length, page: three loads
// that wait for each other).  A prompt's wavefront takes `turns` heads one after the other: where its tokens go and their angles are looked up once.
#include "q4_kv4.hpp"

namespace q4 {

template <bool VEC>
__device__ __forceinline__ void kv4_load8(const half_t* p, float* x) {
    if constexpr (VEC) {
        const half8_t h = *reinterpret_cast<const half8_t*>(p);
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e] = (float)h[e];
    } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e] = (float)p[e];
    }
}

// What turns eight dimensions 8*j .. of a token's rows, for all heads.
struct Kv4Turn {
    float c[8], s[8];         // of each dimension (interleaved: of each pair, four of them), the sine with its sign
    int mate;                 // where the other halves of the pairs are; -1 interleaved, -2: these dimensions are not turned
};

__device__ __forceinline__ Kv4Turn kv4_turn(const Kv4Append& a, int j, int pos) {
    Kv4Turn r;
    r.mate = -2;
    if (8 * j >= a.rot) return r;
    const int half = a.rot / 2;                                            // a multiple of 8
    const bool lower = 8 * j < half;
    r.mate = a.interleaved ? -1 : lower ? 8 * j + half : 8 * j - half;
    const float* cs = a.rope + 2 * (size_t)pos * half;
    if (a.interleaved) {
        const float4_t* t = reinterpret_cast<const float4_t*>(cs + 8 * j);
#pragma unroll
        for (int e = 0; e < 4; ++e) { r.c[e] = t[e / 2][2 * (e % 2)]; r.s[e] = t[e / 2][2 * (e % 2) + 1]; }
    } else {
        const float4_t* t = reinterpret_cast<const float4_t*>(cs + 2 * (lower ? 8 * j : 8 * j - half));
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            r.c[e] = t[e / 2][2 * (e % 2)];
            const float w = t[e / 2][2 * (e % 2) + 1];
            r.s[e] = lower ? -w : w;
        }
    }
    return r;
}

// Eight dimensions 8*j .. of a row, turned.
template <bool VEC>
__device__ __forceinline__ void kv4_turned8(const Kv4Turn& r, const half_t* row, int j, float* x) {
    kv4_load8<VEC>(row + 8 * j, x);
    if (r.mate == -1) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const float u = x[2 * e], v = x[2 * e + 1];
            x[2 * e] = u * r.c[e] - v * r.s[e];
            x[2 * e + 1] = v * r.c[e] + u * r.s[e];
        }
    } else if (r.mate >= 0) {
        float y[8];
        kv4_load8<VEC>(row + r.mate, y);
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e] = x[e] * r.c[e] + y[e] * r.s[e];
    }
}

// Magnitudes are compared as integers: an infinity or a NaN among them is the largest and reaches the scale.
__device__ __forceinline__ uint32_t kv4_bits(float x) { return __builtin_bit_cast(uint32_t, x) & 0x7FFFFFFFu; }
// A group that fits fp16 has a scale of 10912 at most: 65504 / 6 rounds up to 10920, whose sixfold is none of fp16's numbers.
__device__ __forceinline__ half_t kv4_scale(uint32_t bits) {
    const float x = __builtin_bit_cast(float, bits), s = x / 6.0f;
    return (half_t)(x <= 65504.0f ? fminf(s, 10912.0f) : s);
}
__device__ __forceinline__ float kv4_over(float x, float scale) { return scale > 0.0f ? x / scale : 0.0f; }

template <int D, int NG, bool VEC>
__global__ __launch_bounds__(256) void kv4_append_kernel(Kv4Append a) {
    constexpr int L = D / 8, TPW = 64 / L, G = D / NG, H = D / 16, W = D / 8;
    const int lane = threadIdx.x & 63, j = lane % L, heads = a.c.heads;
    const int t = blockIdx.x * TPW + lane / L;
    const int first = blockIdx.y * 4 * a.turns + (threadIdx.x >> 6);
    if (first >= 2 * heads + a.hq) return;                                 // uniform over the wavefront
    Kv4Place w = kv4_place<L>(a.c, a.p, t);
    if (a.rot && w.pos >= a.rope_rows) w.ok = false;
    const int pos = w.ok ? w.pos : 0;
    Kv4Turn turn;
    turn.mate = -2;
    if (a.turns > 1 || first < heads || first >= 2 * heads) turn = kv4_turn(a, j, pos);
    for (int i = 0; i < a.turns; ++i) {
        int h = first + 4 * i;
        if (h >= 2 * heads + a.hq) return;
        if (h >= 2 * heads) {
            h -= 2 * heads;
            if (!w.mine) continue;
            float x[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
            if (w.ok) kv4_turned8<VEC>(turn, a.q + t * a.q_t + h * a.q_h, j, x);
            half8_t o;
#pragma unroll
            for (int e = 0; e < 8; ++e) o[e] = (half_t)x[e];
            *reinterpret_cast<half8_t*>(a.q_out + ((size_t)t * a.hq + h) * D + 8 * j) = o;
            continue;
        }
        const int row = w.ok ? t : 0;                                          // lanes without a place work on row 0 and write nothing
        const bool is_k = h < heads;
        if (!is_k) h -= heads;
        const size_t at = (size_t)w.page * heads + h;
        if (is_k) {
            float x[8];
            kv4_turned8<VEC>(turn, a.k + row * a.k_t + h * a.k_h, j, x);
            uint32_t m = 0;
#pragma unroll
            for (int e = 0; e < 8; ++e) m = max(m, kv4_bits(x[e]));
#pragma unroll
            for (int s = 1; s < G / 8; s <<= 1) m = max(m, (uint32_t)__shfl_xor((int)m, s));
            const half_t sc = kv4_scale(m);
#pragma unroll
            for (int e = 0; e < 8; ++e) x[e] = kv4_over(x[e], (float)sc);
            if (!w.ok) continue;
            a.c.kc[(at * a.c.page + w.off) * W + (j % 4) * (D / 32) + j / 4] = kv4_codes(x);
            if (j % (G / 8) == 0) a.c.ks[(at * NG + j / (G / 8)) * a.c.page + w.off] = sc;
        } else {
            // lane j holds word j: dimensions 16*i + W*r + j, loaded one by one (32 contiguous bytes per half of the lanes)
            float x[8];
            const half_t* p = a.v + row * a.v_t + h * a.v_h + j;
#pragma unroll
            for (int n = 0; n < 8; ++n) x[n] = (float)p[16 * (n % H) + W * (n / H)];
            half_t sc[NG];
#pragma unroll
            for (int g = 0; g < NG; ++g) {
                uint32_t m = 0;
#pragma unroll
                for (int n = 0; n < 8; ++n)
                    if (n % H * 16 / G == g) m = max(m, kv4_bits(x[n]));
#pragma unroll
                for (int s = 1; s < L; s <<= 1) m = max(m, (uint32_t)__shfl_xor((int)m, s));
                sc[g] = kv4_scale(m);
            }
#pragma unroll
            for (int n = 0; n < 8; ++n) x[n] = kv4_over(x[n], (float)sc[n % H * 16 / G]);
            if (!w.ok) continue;
            a.c.vc[((at * (a.c.page / 4) + w.off / 4) * W + j) * 4 + w.off % 4] = kv4_codes(x);
#pragma unroll
            for (int g = 0; g < NG; ++g)
                if (j == g) a.c.vs[(at * NG + g) * a.c.page + w.off] = sc[g];
        }
    }
}

template <int D, int NG>
__global__ __launch_bounds__(256) void kv4_read_kernel(Kv4Read a) {
    constexpr int L = D / 8, TPW = 64 / L, G = D / NG, W = D / 8;
    const int lane = threadIdx.x & 63, j = lane % L, heads = a.c.heads;
    const int t = blockIdx.x * TPW + lane / L;
    const int first = blockIdx.y * 4 * a.turns + (threadIdx.x >> 6);
    if (first >= 2 * heads) return;
    const Kv4Place w = kv4_place<L>(a.c, a.p, t);
    if (t >= a.p.T) return;                                                // a row of no sequence has no place
    for (int i = 0; i < a.turns; ++i) {
        int h = first + 4 * i;
        if (h >= 2 * heads) return;
        const bool is_k = h < heads;
        if (!is_k) h -= heads;
        half8_t o = {};
        if (w.ok) {
            const size_t at = (size_t)w.page * heads + h;
            half8_t x;
            if (is_k) {
                x = kv4_word(a.c.kc[(at * a.c.page + w.off) * W + (j % 4) * (D / 32) + j / 4]);
            } else {                                                           // dimensions 8*j .. + 7: one nibble of eight words
                const uint32_t* p = a.c.vc + (at * (a.c.page / 4) + w.off / 4) * W * 4 + w.off % 4;
                const int first = D == 128 ? 8 * (j % 2) : 0, nib = D == 128 ? j / 2 : j / 2 + 4 * (j % 2);
                uint32_t word = 0;
#pragma unroll
                for (int e = 0; e < 8; ++e) word |= ((p[4 * (first + e)] >> (4 * nib)) & 15u) << (4 * e);
                x = kv4_word(word);
            }
            const float s = (float)(is_k ? a.c.ks : a.c.vs)[(at * NG + 8 * j / G) * a.c.page + w.off];
#pragma unroll
            for (int e = 0; e < 8; ++e) o[e] = (half_t)((float)x[e] * s);
        }
        *reinterpret_cast<half8_t*>((is_k ? a.k : a.v) + ((size_t)t * heads + h) * D + 8 * j) = o;
    }
}

}  // namespace q4

// Heads a wavefront takes: four where two workgroups for every compute unit are left (4096 tokens of 32 + 2 * 8 heads, stored and read back: 41.9 us with
// one, 34.3 with two, 31.3 with four, 30.5 with eight), one for the few rows of a decode step (16 of 32 + 2 * 32: 10.8 us with one, 16.1 with eight).
static int kv4_turns(int T, int per, int heads) { return (long)((T + per - 1) / per) * ((heads + 15) / 16) >= 512 ? 4 : 1; }

template <int D, int NG>
static void launch_append(q4::Kv4Append a, bool vec, hipStream_t stream) {
    const int per = 64 / (D / 8), heads = 2 * a.c.heads + a.hq;
    a.turns = kv4_turns(a.p.T, per, heads);
    const dim3 grid((a.p.T + per - 1) / per, (heads + 4 * a.turns - 1) / (4 * a.turns));
    if (vec) hipLaunchKernelGGL((q4::kv4_append_kernel<D, NG, true>), grid, dim3(256), 0, stream, a);
    else hipLaunchKernelGGL((q4::kv4_append_kernel<D, NG, false>), grid, dim3(256), 0, stream, a);
}

int q4_launch_kv4_append(const q4::Kv4Append& a, int D, int group, bool vec, hipStream_t stream) {
    switch (D / group + (D == 64 ? 8 : 0)) {
        case 1: launch_append<128, 1>(a, vec, stream); break;
        case 2: launch_append<128, 2>(a, vec, stream); break;
        case 4: launch_append<128, 4>(a, vec, stream); break;
        case 9: launch_append<64, 1>(a, vec, stream); break;
        default: launch_append<64, 2>(a, vec, stream); break;
    }
    return hipGetLastError() == hipSuccess ? 0 : -4;
}

template <int D, int NG>
static void launch_read(q4::Kv4Read a, hipStream_t stream) {
    const int per = 64 / (D / 8), heads = 2 * a.c.heads;
    a.turns = kv4_turns(a.p.T, per, heads);
    hipLaunchKernelGGL((q4::kv4_read_kernel<D, NG>), dim3((a.p.T + per - 1) / per, (heads + 4 * a.turns - 1) / (4 * a.turns)), dim3(256), 0, stream, a);
}

int q4_launch_kv4_read(const q4::Kv4Read& a, int D, int group, hipStream_t stream) {
    switch (D / group + (D == 64 ? 8 : 0)) {
        case 1: launch_read<128, 1>(a, stream); break;
        case 2: launch_read<128, 2>(a, stream); break;
        case 4: launch_read<128, 4>(a, stream); break;
        case 9: launch_read<64, 1>(a, stream); break;
        default: launch_read<64, 2>(a, stream); break;
    }
    return hipGetLastError() == hipSuccess ? 0 : -4;
}
