// Attention of a batch's new tokens over the 4-bit key/value cache (layout in q4_kv4.hpp):
//
//   out[t, h] = sum_j p_j v_j,   p = softmax_j(scale * q[t, h] . k_j)   over the keys j at or before the token's own position
//
// One pass over the keys with the running maximum m and sum l of the softmax in fp32.  Codes go to the matrix instructions as the exact
// fp16 values that they stand for; the keys' scales multiply the fp32 scores, the values' scales the probabilities, whose rounding to
// fp16 is the only one before the output's (prompts round more, see there).  What it costs beside the output's own rounding: nothing that shows for values' scales
// of 0.3 down to 1e-5 over 100000 keys (root mean square 2.1e-4 to 8.8e-4 with it and without).
#include "q4_kv4.hpp"
#include <algorithm>
#include <type_traits>

namespace q4 {

// Probabilities are formed as 2^10 * exp(s - m): times a value's scale they then stay clear of fp16's subnormals down to 1e-7 of the
// largest for scales of 0.1, and below its largest number for scales up to 32; for larger scales the maximum is raised.
constexpr float kBoost = 10.0f, kMostScale = 32.0f;
constexpr uint32_t kMostScaleBits = 0x5000u;          // 32 in fp16

__device__ __forceinline__ void wave_lds_fence() {
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

// Maximum over the four lanes r, r + 16, r + 32, r + 48: rows of 16 lanes change places in registers.  (The results are copied out of their vector
// first: a bit cast straight from its second element reads the first.)
__device__ __forceinline__ float max_of_rows(float x) {
    uint32_t u = __builtin_bit_cast(uint32_t, x);
    const auto a = __builtin_amdgcn_permlane32_swap(u, u, false, false);
    const uint32_t a0 = a[0], a1 = a[1];
    u = __builtin_bit_cast(uint32_t, fmaxf(__builtin_bit_cast(float, a0), __builtin_bit_cast(float, a1)));
    const auto b = __builtin_amdgcn_permlane16_swap(u, u, false, false);
    const uint32_t b0 = b[0], b1 = b[1];
    return fmaxf(__builtin_bit_cast(float, b0), __builtin_bit_cast(float, b1));
}

__device__ __forceinline__ float max_of_halves(float x) {
    const uint32_t u = __builtin_bit_cast(uint32_t, x);
    const auto a = __builtin_amdgcn_permlane32_swap(u, u, false, false);
    const uint32_t a0 = a[0], a1 = a[1];
    return fmaxf(__builtin_bit_cast(float, a0), __builtin_bit_cast(float, a1));
}

typedef float float2_t __attribute__((ext_vector_type(2)));
__device__ __forceinline__ uint32_t rounded_pair(float a, float b) { return as_u32(__builtin_convertvector(float2_t{a, b}, half2_t)); }

__device__ __forceinline__ uint32_t magnitude_bits(half_t x) { return __builtin_bit_cast(uint16_t, x) & 0x7FFFu; }
__device__ __forceinline__ bool finite_bits(half_t x) { return (__builtin_bit_cast(uint16_t, x) & 0x7C00u) != 0x7C00u; }

typedef unsigned short ushort2_t __attribute__((ext_vector_type(2)));
__device__ __forceinline__ uint32_t pk_max_u16(uint32_t a, uint32_t b) {
    return __builtin_bit_cast(uint32_t, __builtin_elementwise_max(__builtin_bit_cast(ushort2_t, a), __builtin_bit_cast(ushort2_t, b)));
}

// ---- up to 16 rows a workgroup ------------------------------------------------------------------
// A row is a query head of a token; the `share` heads that read one key head and the tokens of a sequence lie side by side.  Workgroup = one
// key head, 16 rows, one share of the keys; its four wavefronts take tiles of 64 keys in turn and meet once, in LDS, at the end.
// v_mfma_f32_16x16x32_f16 throughout:
//   S^T = K Q^T:   A = 16 keys x 32 dimensions, row 4*b + i of tile u is key 16*b + 4*u + i; B = 32 dimensions x 16 rows.  Lane (r, kk) gets
//                  the scores of row r for keys 16*kk + 4*u + (0..3)
//   O^T = V^T P^T: B = 32 keys x 16 rows: exactly these scores' probabilities, in the lane that holds them; A = 16 dimensions x 32 keys, the
//                  4 x 4 words of keys 16*kk ..: neighbouring keys' nibbles side by side by two operations per four pairs
// so no operand passes through LDS, and maximum, sum and rescaling belong to the lane.
template <int D, int NG>
__global__ __launch_bounds__(256, 3) void kv4_attn_rows_kernel(Kv4Attn a) {
    constexpr int S = D / 32, H = D / 16, SG = S / NG, HG = H / NG, W = D / 8;
    __shared__ __attribute__((aligned(16))) half_t scales[4][2][NG][64];
    __shared__ __attribute__((aligned(16))) float red[4][16][D + 4];
    __shared__ float red_ml[4][16][2];
    const int lane = threadIdx.x & 63, r = lane & 15, kk = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    int id = blockIdx.x;
    const int split = id % a.nsplit;
    id /= a.nsplit;
    const int h = id % a.c.heads;
    id /= a.c.heads;
    const int b = id / a.blocks;
    const int first = a.p.starts ? a.p.starts[b] : b * (a.p.T / a.p.B);
    const int n = min((a.p.starts ? a.p.starts[b + 1] : (b + 1) * (a.p.T / a.p.B)) - first, a.p.T);
    const int len = kv4_length(a.p, b), cap = a.p.width * a.c.page, p16 = a.c.page / 16;
    const int* table = a.p.table + (size_t)b * a.p.width;
    const int rows = n * a.share;

    for (int row0 = (id % a.blocks) * 16; row0 < rows; row0 += a.blocks * 16) {
        const int row = row0 + r;
        const int tok = first + row / a.share, qh = h * a.share + row % a.share;
        const bool live = row < rows && tok >= 0 && tok < a.p.T;
        // keys 0 .. limit - 1 are seen by this lane's row, 0 .. kmin - 1 by all rows, kend by any
        const int limit = live ? max(0, min(len - n + row / a.share + 1, cap)) : 0;
        const int kmin = max(0, min(len - n + row0 / a.share + 1, cap));
        const int kend = max(0, min(len - n + min(row0 + 15, rows - 1) / a.share + 1, cap));
        const int tiles = (kend + 63) / 64, per = (tiles + a.nsplit - 1) / a.nsplit;
        const int t_end = min((split + 1) * per, tiles);

        half8_t qf[S];
#pragma unroll
        for (int s = 0; s < S; ++s) {
            qf[s] = half8_t{};
            if (live) qf[s] = *reinterpret_cast<const half8_t*>(a.q + tok * a.q_t + qh * a.q_h + 32 * s + 8 * kk);
        }
        float4_t o[H];
#pragma unroll
        for (int i = 0; i < H; ++i) o[i] = float4_t{0.f, 0.f, 0.f, 0.f};
        float m = -INFINITY, l = 0.f;

        // Of a tile's four runs of 16 keys, lane c looks run c % 4 up: its place in units of 16 keys, in a head's codes and (second word) in its
        // scales.  The top bit marks a run that the sequence does not reach or whose page is none; it is read from page 0 and masked.
        auto look_up = [&](int tile) {
            const int run = tile * 4 + (lane & 3);
            const int idx = a.page_magic ? (int)__umulhi((uint32_t)run, a.page_magic) : run;
            const bool in = run * 16 < kend;
            int page = in ? table[idx] : -1;
            const bool ok = page >= 0 && page < a.c.pages;
            const uint32_t head = (uint32_t)(ok ? page : 0) * a.c.heads + h, off = ok ? run - idx * p16 : 0;
            uint2_t w;
            w.x = (head * p16 + off) | (ok ? 0u : 0x80000000u);
            w.y = head * NG * p16 + off;
            return w;
        };
        // Registers of one tile: the keys' are requested again as soon as the scores are formed, the values' as soon as they are multiplied.
        uint32_t xk[4][S];
        uint4_t xv[4], xs = {0u, 0u, 0u, 0u};                              // xs: eight scales, lane = (keys or values, group, eighth of the tile)
        auto load_keys = [&](uint2_t at) {
            const uint32_t kr = (uint32_t)__shfl((int)at.x, r >> 2) & 0x7FFFFFFFu;
            const uint32_t* kp = a.c.kc + (size_t)kr * (16 * W) + (r & 3) * W + kk * S;
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                if constexpr (S == 4) *reinterpret_cast<uint4_t*>(xk[u]) = __builtin_nontemporal_load(reinterpret_cast<const uint4_t*>(kp + u * 4 * W));
                else *reinterpret_cast<uint2_t*>(xk[u]) = __builtin_nontemporal_load(reinterpret_cast<const uint2_t*>(kp + u * 4 * W));
            }
            const int piece = lane & 7, g = (lane >> 3) % NG;
            const uint32_t sr = (uint32_t)__shfl((int)at.y, piece >> 1);
            if (lane < 16 * NG)
                xs = *reinterpret_cast<const uint4_t*>((lane < 8 * NG ? a.c.ks : a.c.vs) + ((size_t)sr + g * p16) * 16 + 8 * (piece & 1));
        };
        auto load_values = [&](uint2_t at) {
            const uint32_t vr = (uint32_t)__shfl((int)at.x, kk) & 0x7FFFFFFFu;
            const uint32_t* vp = a.c.vc + (size_t)vr * (16 * W) + (r % W) * 4;
#pragma unroll
            for (int u = 0; u < 4; ++u) xv[u] = __builtin_nontemporal_load(reinterpret_cast<const uint4_t*>(vp + u * 4 * W));
        };
        float s[16];
        auto scores = [&] {
            if (lane < 16 * NG) *reinterpret_cast<uint4_t*>(&scales[wave][0][0][0] + 8 * lane) = xs;
            wave_lds_fence();
#pragma unroll
            for (int g = 0; g < NG; ++g) {
                float4_t acc[4];
#pragma unroll
                for (int u = 0; u < 4; ++u) acc[u] = float4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int st = g * SG; st < (g + 1) * SG; ++st) {
                    __builtin_amdgcn_sched_barrier(0);                     // or all operands are built first, in registers that are not there
#pragma unroll
                    for (int u = 0; u < 4; ++u)
                        acc[u] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kv4_word(xk[u][st]), qf[st], acc[u], 0, 0, 0);
                }
                const half8_t k0 = *reinterpret_cast<const half8_t*>(&scales[wave][0][g][16 * kk]);
                const half8_t k1 = *reinterpret_cast<const half8_t*>(&scales[wave][0][g][16 * kk + 8]);
#pragma unroll
                for (int e = 0; e < 16; ++e) {
                    const float ks = (float)(e < 8 ? k0[e & 7] : k1[e & 7]);
                    s[e] = g == 0 ? acc[e >> 2][e & 3] * ks : fmaf(acc[e >> 2][e & 3], ks, s[e]);
                    asm volatile("" : "+v"(s[e]));                         // here, not where it is used: one group's sums at a time
                }
            }
        };
        auto weigh = [&](bool masked, int seen, bool unusual) {
            if (masked) {                                                  // whatever a place that is not seen holds, it counts nothing
#pragma unroll
                for (int e = 0; e < 16; ++e) s[e] = e < seen ? s[e] : -INFINITY;
            }
            float mx = s[0];
#pragma unroll
            for (int e = 1; e < 16; ++e) mx = fmaxf(mx, s[e]);
            float mn = max_of_rows(mx) * a.scale;
            if (unusual) {
                // Scales above kMostScale raise the maximum.  One that is no number makes the row none that sees it; it is zero for the others, whose
                // weight of nothing times it would not be nothing.
                float big = kMostScale;
#pragma unroll 1
                for (int i = 0; i < 16 * NG; ++i) {
                    const half_t x = scales[wave][1][i >> 4][16 * kk + (i & 15)];
                    if ((i & 15) < seen) {
                        if (finite_bits(x)) big = fmaxf(big, fabsf((float)x));
                        else l = NAN;
                    }
                }
                mn += log2f(max_of_rows(big) / kMostScale);
                wave_lds_fence();
                if (lane >= 8 * NG && lane < 16 * NG) {
                    half_t* x = &scales[wave][0][0][0] + 8 * lane;
#pragma unroll 1
                    for (int e = 0; e < 8; ++e)
                        if (!finite_bits(x[e])) x[e] = (half_t)0.f;
                }
                wave_lds_fence();
            }
            mn = fmaxf(m, mn);
            const float base = mn == -INFINITY ? 0.f : mn;
            if (__any(mn > m)) {
                const float f = __builtin_amdgcn_exp2f(m - base);
                l *= f;
#pragma unroll
                for (int i = 0; i < H; ++i) o[i] *= f;
                m = mn;
            }
#pragma unroll
            for (int e = 0; e < 16; ++e) {
                s[e] = __builtin_amdgcn_exp2f(fmaf(s[e], a.scale, kBoost - base));
                l += s[e];
            }
#pragma unroll
            for (int v = 0; v < 2; ++v) {
                __builtin_amdgcn_sched_barrier(0);
                uint32_t lo[4], hi[4];                                     // even and odd nibbles of two keys side by side
#pragma unroll
                for (int c = 0; c < 4; ++c) {
                    const uint4_t w = xv[2 * v + (c >> 1)];
                    uint32_t wa = c & 1 ? w.z : w.x, wb = c & 1 ? w.w : w.y;
                    if constexpr (D == 64) { wa >>= 16 * (r >> 3); wb >>= 16 * (r >> 3); }
                    lo[c] = (wa & 0x0F0F0F0Fu) | ((wb << 4) & 0xF0F0F0F0u);
                    hi[c] = ((wa >> 4) & 0x0F0F0F0Fu) | (wb & 0xF0F0F0F0u);
                }
#pragma unroll
                for (int g = 0; g < NG; ++g) {
                    if (NG > 1) __builtin_amdgcn_sched_barrier(0);
                    const half8_t sv = *reinterpret_cast<const half8_t*>(&scales[wave][1][g][16 * kk + 8 * v]);
                    uint4_t pw;
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        pw[e] = rounded_pair(fmaf(s[8 * v + 2 * e], (float)sv[2 * e], 0.f), fmaf(s[8 * v + 2 * e + 1], (float)sv[2 * e + 1], 0.f));
                    const half8_t pb = __builtin_bit_cast(half8_t, pw);
#pragma unroll
                    for (int i = g * HG; i < (g + 1) * HG; ++i) {
                        uint4_t vw;
#pragma unroll
                        for (int c = 0; c < 4; ++c) {
                            const uint32_t w = i & 1 ? hi[c] : lo[c];
                            vw[c] = as_u32(i / 2 == 0 ? kv4_pair<0>(w) : i / 2 == 1 ? kv4_pair<1>(w) : i / 2 == 2 ? kv4_pair<2>(w) : kv4_pair<3>(w));
                        }
                        o[i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(half8_t, vw), pb, o[i], 0, 0, 0);
                    }
                }
            }
        };

        // tiles wave, wave + 4, ... of the share; the page entries are looked up one tile further ahead
        int t = split * per + wave;
        uint2_t at = {0u, 0u}, next = {0u, 0u};
        if (t < t_end) {
            at = look_up(t);
            next = look_up(t + 4);
            load_keys(at);
            load_values(at);
        }
        while (t < t_end) {
            const bool more = t + 4 < t_end;
            scores();
            // whether a value's scale is above kMostScale or no number, seen or not, by its bits, where the tile's scales lie eight in a lane
            uint32_t most = pk_max_u16(pk_max_u16(xs.x, xs.y), pk_max_u16(xs.z, xs.w));
            most = lane >= 8 * NG && lane < 16 * NG ? max(most >> 16, most & 0xFFFFu) : 0u;
            const bool bad = (uint32_t)__shfl((int)at.x, kk) >> 31;
            at = next;
            if (more) {
                next = look_up(t + 8);
                load_keys(at);
            }
            weigh(t * 64 + 64 > kmin || __any(bad), bad ? 0 : limit - (t * 64 + 16 * kk), __any(most > kMostScaleBits));
            if (more) load_values(at);
            t += 4;
        }

        l += __shfl_xor(l, 16);
        l += __shfl_xor(l, 32);
        if (live) {
#pragma unroll
            for (int i = 0; i < H; ++i) *reinterpret_cast<float4_t*>(&red[wave][r][16 * i + 4 * kk]) = o[i];
            if (kk == 0) { red_ml[wave][r][0] = m; red_ml[wave][r][1] = l; }
        }
        __syncthreads();
        const int here = min(16, rows - row0);
        for (int i = threadIdx.x; i < here * (D / 4); i += 256) {
            const int rr = i / (D / 4), d = i % (D / 4) * 4;
            const int tk = first + (row0 + rr) / a.share;
            if (tk < 0 || tk >= a.p.T) continue;
            float top = red_ml[0][rr][0];
#pragma unroll
            for (int w = 1; w < 4; ++w) top = fmaxf(top, red_ml[w][rr][0]);
            float sum = 0.f;
            float4_t v = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int w = 0; w < 4; ++w) {
                const float f = red_ml[w][rr][0] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(red_ml[w][rr][0] - top);
                sum = fmaf(f, red_ml[w][rr][1], sum);
                const float4_t ov = *reinterpret_cast<const float4_t*>(&red[w][rr][d]);
#pragma unroll
                for (int e = 0; e < 4; ++e) v[e] = fmaf(f, ov[e], v[e]);
            }
            const size_t at = (size_t)tk * a.hq + h * a.share + (row0 + rr) % a.share;
            if (a.nsplit == 1) {
                half4_t y;
#pragma unroll
                for (int e = 0; e < 4; ++e) y[e] = (half_t)(sum == 0.f ? 0.f : v[e] / sum);
                *reinterpret_cast<half4_t*>(a.out + at * D + d) = y;
            } else {
                const size_t all = (size_t)a.p.T * a.hq;
                *reinterpret_cast<float4_t*>(a.part + (split * all + at) * D + d) = v;
                if (d == 0) {
                    float* ml = a.part + a.nsplit * all * D + (split * all + at) * 2;
                    ml[0] = top;
                    ml[1] = sum;
                }
            }
        }
        __syncthreads();
    }
}

// ---- prompts: 128 rows a workgroup -----------------------------------------------------------------
// Four wavefronts of 32 rows on the same tiles of 64 keys.  The workgroup turns a tile's codes into fp16 values (values: one rounding each, of code * scale) in LDS,
// in the order in which v_mfma_f32_32x32x16_f16 takes them: pieces of 16 bytes, lane after lane, so that neither side meets a bank conflict.  Two tiles: the next one
// is written, and the two behind it requested, while one is multiplied; one barrier a tile.  As above S^T = K Q^T and O^T = V^T P^T, lane (r, h) holding row r:
//   keys' piece (kb, st, lane): key 32*kb + r, dimensions 16*st + 8*h .. + 7
//   values' piece (kb, p, db, lane): dimension 32*db + r of keys 32*kb + 16*p + 4*h + (0..3) and + 8, the keys of the scores in that lane's registers 8*p .. + 7
// The maximum that weights refer to is raised only when a score lies 2^kSlack above it: weights then stay below 2^15.
//
// Blocks of rows whose last one sees up to kFewKeys keys get the keys' codes as they are, and each group's fp32 sums times its keys' scales; in blocks that see more, code * scale is
// rounded once like the values.  Root mean square error of a whole output against float64, relative: 2.6e-4 so, 3.1e-4 with all rounded for the prompt of 2048 tokens, 2.6e-4 and 3.4e-4
// for one of 128, 2.3e-4 for parts of prompts that see thousands (2.1e-4 are the output's own rounding); exact keys cost 5, 15 and 40 per cent at 1, 2 and 4 groups.
//
// What bounds it: a wavefront starts an operation in about eight cycles, and two of them share a SIMD, whose vector operations (230 a tile and wavefront) and matrix
// operations (32 of 32 cycles) take 1900 of the 3700 cycles that a tile of both lasts at 2.1 GHz.  The whole prompt of 2048 tokens, 32 heads of 128: 59 us, of which the
// last block's 32 tiles are 55; parts of four prompts (509, 434, 360, 286 tokens at 8191, 5062, 1933, 6995; 8 key heads of 4): 196 us, 128 tiles one after the other.
// Eight wavefronts on 256 rows, half turning keys, half values: 69 and 216 us, for all are at the same step; splitting the keys of whole prompts costs the join more
// than the balance gives (parts: 271 us in two shares).
//
// Values beyond fp16 (a scale above 10912, whose sixfold passes it; append writes none) would be infinite in LDS, and nothing times infinity is no number
// for the rows that do not see them.  The staging finds such a scale, and the rows are gone through a second time with an eighth of every value, which holds all of them.  (Once per block of rows that has such a
// value; the test for it replaces one for infinities, operation for operation; that there may be a second pass costs the others under 1 per cent.)
// Rounded keys are eighths always (a rotation takes pairs of large numbers beyond fp16; the conversion from codes multiplies by a power of two for nothing), and the softmax
// scale is eightfold; keys below 2^-11 lose up to three bits by it.
constexpr uint32_t kMostValueScale = 0x7154u;          // 10912 in fp16
constexpr uint32_t kAboveMost = (0x7FFFu - kMostValueScale) * 0x10001u;      // added to two magnitudes: the sign of one that is greater
constexpr float kLessen = 0.125f;
constexpr float kSlack = 5.0f;
constexpr int kPromptRows = 128;
constexpr int kFewKeys = 1024;

constexpr int kHalfPiece = 36;                                             // keys: 32 pieces and room for four, so that a key's quarters are written to banks of their own

template <int D>
struct Kv4Staged {
    uint4_t k[4 * D / 16 * kHalfPiece], v[4 * D / 32 * 64];
};

template <int D, int NG>
__global__ __launch_bounds__(256, 2) void kv4_attn_prompt_kernel(Kv4Attn a) {
    constexpr int S = D / 32, ST = D / 16, DB = D / 32, W = D / 8, SG = S / NG, H = D / 16, HG = H / NG, NV = D / 16;   // NV: nibbles of a word a thread takes
    __shared__ __attribute__((aligned(16))) Kv4Staged<D> tiles_lds[2];
    __shared__ __attribute__((aligned(16))) float key_scales[2][NG][64];
    __shared__ int poison;                                                 // first key seen whose values are no numbers
    __shared__ int large;                                                  // whether a value seen is beyond fp16
    __shared__ int there[2][4];                                            // whether the tile's runs of 16 keys lie on pages of the cache
    const int lane = threadIdx.x & 63, r = lane & 31, h32 = lane >> 5;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    int id = blockIdx.x;
    const int h = id % a.c.heads;                                          // workgroups on one head's keys lie on one chiplet where heads are a multiple of 8
    id /= a.c.heads;
    const int split = id % a.nsplit;
    id /= a.nsplit;
    // The rows with the most keys first.  Of up to 64 sequences the longest comes first with all its rows, so that its workgroups find compute units of their
    // own and the short ones come beside them (parts of four prompts at 8191, 6995, 5062 and 1933 tokens: 238 us in turns, 195 sorted).
    int b = id % a.p.B, block0 = a.blocks - 1 - id / a.p.B;
    if (a.p.B > 1 && a.p.B <= 64) {
        int mine = 0, length = -1, before = 0;                             // lane: a sequence, its blocks, and those of longer ones
        if (lane < a.p.B) {
            const int rows = (a.p.starts ? a.p.starts[lane + 1] - a.p.starts[lane] : a.p.T / a.p.B) * a.share;
            mine = min((max(rows, 0) + kPromptRows - 1) / kPromptRows, a.blocks);
            length = a.p.lengths[lane];
        }
        for (int k = 0; k < a.p.B; ++k) {
            const int other = __builtin_amdgcn_readlane(length, k), blocks = __builtin_amdgcn_readlane(mine, k);
            before += other > length || (other == length && k < lane) ? blocks : 0;
        }
        const uint64_t found = __ballot(lane < a.p.B && id >= before && id < before + mine);
        if (!found) return;
        b = __builtin_ctzll(found);
        block0 = __builtin_amdgcn_readlane(before + mine, b) - 1 - id;
    }
    const int first = a.p.starts ? a.p.starts[b] : b * (a.p.T / a.p.B);
    const int n = min((a.p.starts ? a.p.starts[b + 1] : (b + 1) * (a.p.T / a.p.B)) - first, a.p.T);
    const int len = kv4_length(a.p, b), cap = a.p.width * a.c.page, p16 = a.c.page / 16;
    const int* table = a.p.table + (size_t)b * a.p.width;
    const int rows = n * a.share;

    float lessen = 1.f;                                                    // of the values; kLessen while rows are gone through a second time
    for (int row0 = block0 * kPromptRows; row0 < rows;) {
        const int row = row0 + 32 * wave + r;
        const int tok = first + row / a.share, qh = h * a.share + row % a.share;
        const bool live = row < rows && tok >= 0 && tok < a.p.T;
        const int limit = live ? max(0, min(len - n + row / a.share + 1, cap)) : 0;
        // 0 .. kmin - 1 are seen by all rows of this wavefront, kend by any of the workgroup's
        const int kmin = max(0, min(len - n + (row0 + 32 * wave) / a.share + 1, cap));
        const int kend = max(0, min(len - n + min(row0 + kPromptRows - 1, rows - 1) / a.share + 1, cap));
        const int tiles = (kend + 63) / 64, per = (tiles + a.nsplit - 1) / a.nsplit;
        const int t0 = split * per, t_end = min(t0 + per, tiles);
        if (threadIdx.x == 0) { poison = 0x7FFFFFFF; large = 0; }

        half8_t qf[ST];
#pragma unroll
        for (int s = 0; s < ST; ++s) {
            qf[s] = half8_t{};
            if (live) qf[s] = *reinterpret_cast<const half8_t*>(a.q + tok * a.q_t + qh * a.q_h + 16 * s + 8 * h32);
        }
        float16_t o[DB];
#pragma unroll
        for (int i = 0; i < DB; ++i)
#pragma unroll
            for (int e = 0; e < 16; ++e) o[i][e] = 0.f;
        float m = -INFINITY, l = 0.f;

        // This thread's part of a tile: quarter lane % 4 of the words of key 16*wave + lane / 4, and word c of the four keys of block 4*wave + kk: all in run
        // `wave`, a contiguous kilobyte each.
        // Two tiles are on their way, and the page of the one behind them.
        const int c = lane & 15, kk = lane >> 4, kc = lane >> 2, kq = lane & 3;
        struct Raw {
            uint32_t k[S];
            uint4_t v;
            half_t ks[NG];
            half4_t vs[NG];
            int have;                                                      // -1 or 0
        } raw[2];
        int page = -1;                                                     // of the next tile to be requested
        int zero;                                                          // opaque: the page is loaded into a vector register and waited for where it is used
        asm volatile("v_mov_b32 %0, 0" : "=v"(zero));
        const int single = a.page_magic ? 0 : -1;                          // no branch in a tile's way: a taken one costs what fifty operations do
        auto index_of = [&](int run) __attribute__((always_inline)) { return (int)__umulhi((uint32_t)run, a.page_magic) | (run & single); };
        auto page_of = [&](int tile) __attribute__((always_inline)) { return table[index_of(min(tile * 4 + wave, (kend - 1) / 16)) + zero]; };   // of the tile's run, or of the last run there is
        size_t words = 0, halves = 0;                                      // where the tile's run lies in a head's codes and scales
        auto request_keys = [&](Raw& x, int tile) __attribute__((always_inline)) {
            const int run = tile * 4 + wave, pg = __builtin_amdgcn_readfirstlane(page);
            const int ok = -(int)((tile < t_end) & (run * 16 < kend) & ((uint32_t)pg < (uint32_t)a.c.pages));
            x.have = ok;
            const uint32_t head = (uint32_t)(pg & ok) * a.c.heads + h, off = (run - index_of(run) * p16) & ok;
            page = page_of(tile + 1);
            words = (size_t)(head * p16 + off) * (16 * W);
            halves = ((size_t)head * NG * p16 + off) * 16;
            const uint32_t* kp = a.c.kc + words + kc * W + kq * S;
            if constexpr (S == 4) *reinterpret_cast<uint4_t*>(x.k) = *reinterpret_cast<const uint4_t*>(kp);
            else *reinterpret_cast<uint2_t*>(x.k) = *reinterpret_cast<const uint2_t*>(kp);
#pragma unroll
            for (int g = 0; g < NG; ++g) x.ks[g] = a.c.ks[halves + (size_t)g * a.c.page + kc];
        };
        auto request_values = [&](Raw& x) __attribute__((always_inline)) { x.v = *reinterpret_cast<const uint4_t*>(a.c.vc + words + (kk * W + c % W) * 4); };
        auto request_scales = [&](Raw& x) __attribute__((always_inline)) {
#pragma unroll
            for (int g = 0; g < NG; ++g) x.vs[g] = *reinterpret_cast<const half4_t*>(a.c.vs + halves + (size_t)g * a.c.page + 4 * kk);
        };
        auto request = [&](Raw& x, int tile) __attribute__((always_inline)) {
            request_keys(x, tile);
            request_values(x);
            request_scales(x);
        };
        // What no row of the workgroup sees is nothing, and a value's scale that is no number makes the rows none that see it.
        auto look = [&](Raw& x, int buf, int tile) __attribute__((always_inline)) {
            const int key = tile * 64 + 16 * wave;
            there[buf][wave] = x.have | -(int)(key >= kend);
            uint32_t odd = 0;                                              // the sign of a half: a magnitude above kMostValueScale, or no number
#pragma unroll
            for (int g = 0; g < NG; ++g) {
                const uint2_t w = __builtin_bit_cast(uint2_t, x.vs[g]);
                odd |= ((w.x & 0x7FFF7FFFu) + kAboveMost) | ((w.y & 0x7FFF7FFFu) + kAboveMost);
            }
            if (__builtin_expect((key + 16 <= kend) & (__ballot((odd & 0x80008000u) != 0) == 0) & (x.have != 0), 1)) return;
            const int ks_in = x.have ? kend - key - kc : 0, vs_in = x.have ? kend - key - 4 * kk : 0;
            int strange = 0x7FFFFFFF;
            uint32_t most = 0;
#pragma unroll
            for (int g = 0; g < NG; ++g) {
                if (ks_in <= 0) x.ks[g] = (half_t)0.f;
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const bool finite = finite_bits(x.vs[g][e]);
                    if (e < vs_in && !finite) strange = min(strange, key + 4 * kk + e);
                    if (e >= vs_in || !finite) x.vs[g][e] = (half_t)0.f;
                    most = max(most, magnitude_bits(x.vs[g][e]));
                }
            }
            if (__any(strange != 0x7FFFFFFF)) atomicMin(&poison, strange);
            if (__any(most > kMostValueScale)) large = 1;
        };
        const int kb_w = wave >> 1;                                        // the half of a tile that this wavefront's keys lie in
        const int kr_w = 16 * (wave & 1) + kc;
        auto stage_keys = [&](auto exact, const Raw& x, int buf, int s) __attribute__((always_inline)) {  // dimensions 32*s + 8*kq .. + 7
            uint4_t y;
            if constexpr (decltype(exact)::value) {
                y = __builtin_bit_cast(uint4_t, kv4_word(x.k[s]));
                if (s % SG == 0) key_scales[buf][s / SG][16 * wave + kc] = (float)x.ks[s / SG];
            } else {
                const half2_t f = {x.ks[s / SG], x.ks[s / SG]};
                y = uint4_t{as_u32(kv4_pair<0>(x.k[s], kLessen) * f), as_u32(kv4_pair<1>(x.k[s], kLessen) * f), as_u32(kv4_pair<2>(x.k[s], kLessen) * f),
                            as_u32(kv4_pair<3>(x.k[s], kLessen) * f)};
            }
            tiles_lds[buf].k[((kb_w * ST + 2 * s) * 2 + kq) * kHalfPiece + kr_w] = y;
        };
        uint32_t pr[2][2];                                                 // [pair of keys][even, odd nibbles]
        auto pair_values = [&](const Raw& x) __attribute__((always_inline)) {
            uint32_t wd[4] = {x.v.x, x.v.y, x.v.z, x.v.w};
            if constexpr (D == 64) {
#pragma unroll
                for (int e = 0; e < 4; ++e) wd[e] >>= 16 * (c >> 3);
            }
#pragma unroll
            for (int q = 0; q < 2; ++q) {
                pr[q][0] = (wd[2 * q] & 0x0F0F0F0Fu) | ((wd[2 * q + 1] << 4) & 0xF0F0F0F0u);
                pr[q][1] = ((wd[2 * q] >> 4) & 0x0F0F0F0Fu) | (wd[2 * q + 1] & 0xF0F0F0F0u);
            }
        };
        // dimension 16*i + c of block 4*wave + kk of the tile: keys 4*kk .. of this half of its 32; piece p = wave & 1, h = kk & 1, half of it kk >> 1
        auto stage_values = [&](const Raw& x, int buf, int i) __attribute__((always_inline)) {
            uint2_t y;
#pragma unroll
            for (int q = 0; q < 2; ++q) {
                const uint32_t w = pr[q][i & 1];
                const half2_t f = {x.vs[i / HG][2 * q], x.vs[i / HG][2 * q + 1]};
                const half2_t d = i / 2 == 0 ? kv4_pair<0>(w, lessen) : i / 2 == 1 ? kv4_pair<1>(w, lessen) : i / 2 == 2 ? kv4_pair<2>(w, lessen) : kv4_pair<3>(w, lessen);
                y[q] = as_u32(d * f);
            }
            uint4_t* at = &tiles_lds[buf].v[((kb_w * 2 + (wave & 1)) * DB + i / 2) * 64 + 32 * (kk & 1) + 16 * (i & 1) + c];
            reinterpret_cast<uint2_t*>(at)[kk >> 1] = y;
        };
        // Tile t from half BUF, while t + 1 goes to the other one; behind the last tile that is written once more, for nobody.  What goes between the
        // products stands there: the compiler alone reads an operand, waits for it and multiplies.
        auto step = [&](auto exact, auto half, int t) __attribute__((always_inline)) {
            constexpr bool EXACT = decltype(exact)::value;
            constexpr int BUF = decltype(half)::value, N = 2 * ST, AHEAD = 3;   // N products of keys, and N of values
            const Kv4Staged<D>& x = tiles_lds[BUF];
            Raw& next = raw[BUF ^ 1];
            half8_t op[AHEAD];
            auto operand = [&](int i) __attribute__((always_inline)) {                                    // of product i: keys' (st, kb), then values' (kb, p, i)
                op[i % AHEAD] = __builtin_bit_cast(half8_t, i < N ? x.k[((i & 1) * ST + (i >> 1)) * 2 * kHalfPiece + lane + h32 * (kHalfPiece - 32)] : x.v[(i - N) * 64 + lane]);
            };
#pragma unroll
            for (int i = 0; i < AHEAD; ++i) operand(i);
            const int mine = there[BUF][lane & 3];
            look(next, BUF ^ 1, t + 1);
            float16_t s[2], sum[2];
            constexpr int RUN = EXACT ? N / NG : N;                        // products of a group's dimensions, then its scales
#pragma unroll
            for (int i = 0; i < N; ++i) {
                float16_t& y = EXACT ? sum[i & 1] : s[i & 1];
                if (i % RUN < 2) {
#pragma unroll
                    for (int e = 0; e < 16; ++e) y[e] = 0.f;
                }
                y = __builtin_amdgcn_mfma_f32_32x32x16_f16(op[i % AHEAD], qf[i >> 1], y, 0, 0, 0);
                operand(i + AHEAD);
                if (i % 4 == 3) stage_keys(exact, next, BUF ^ 1, i / 4);
                __builtin_amdgcn_sched_barrier(0);
                if (EXACT && i % RUN == RUN - 1) {
#pragma unroll
                    for (int e = 0; e < 32; e += 4) {
                        const float4_t f = *reinterpret_cast<const float4_t*>(&key_scales[BUF][i / RUN][32 * (e >> 4) + 2 * (e & 15) + 4 * h32]);
#pragma unroll
                        for (int d = 0; d < 4; ++d) {
                            const float z = sum[e >> 4][(e & 15) + d];
                            s[e >> 4][(e & 15) + d] = i < RUN ? z * f[d] : fmaf(z, f[d], s[e >> 4][(e & 15) + d]);
                        }
                    }
                }
            }
            const uint32_t gone = (uint32_t)__ballot(!mine) & 15u;         // runs that are not there
            if (__builtin_expect((t * 64 + 64 > kmin) | (gone != 0), 0)) {  // register e of block kb: key 32*kb + 8*(e/4) + 4*h32 + e%4
                const int seen = limit - (t * 64 + 4 * h32);
#pragma unroll
                for (int kb = 0; kb < 2; ++kb)
#pragma unroll
                    for (int e = 0; e < 16; ++e) {
                        const int until = gone >> (2 * kb + (e >> 3)) & 1 ? 0 : seen;
                        s[kb][e] = 32 * kb + 8 * (e >> 2) + (e & 3) < until ? s[kb][e] : -INFINITY;
                    }
            }
            const float scale = EXACT ? a.scale : a.scale8;
            float mx = s[0][0];
#pragma unroll
            for (int e = 1; e < 32; ++e) mx = fmaxf(mx, s[e >> 4][e & 15]);
            mx = max_of_halves(mx) * scale;
            if (__builtin_expect(__any(mx > m + kSlack), 0)) {
                const float mn = fmaxf(m, mx), f = mn == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(m - mn);
                l *= f;
#pragma unroll
                for (int i = 0; i < DB; ++i) o[i] *= f;
                m = mn;
            }
            const float base = kBoost - (m == -INFINITY ? 0.f : m);
            uint4_t pw[4];
            auto weights = [&](int e) __attribute__((always_inline)) {                                    // e, e + 1 of the 32
                float p[2];
#pragma unroll
                for (int d = 0; d < 2; ++d) {
                    p[d] = __builtin_amdgcn_exp2f(fmaf(s[e >> 4][(e & 15) + d], scale, base));
                    l += p[d];
                }
                pw[e >> 3][(e & 7) >> 1] = rounded_pair(p[0], p[1]);
            };
#pragma unroll
            for (int e = 0; e < 8; e += 2) weights(e);
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int i = 0; i < N; ++i) {
                o[i % DB] = __builtin_amdgcn_mfma_f32_32x32x16_f16(op[(N + i) % AHEAD], __builtin_bit_cast(half8_t, pw[i / DB]), o[i % DB], 0, 0, 0);
                if (i + AHEAD < N) operand(N + i + AHEAD);
                if (i < 3 * DB) {
#pragma unroll
                    for (int e = 0; e < 8 / DB; e += 2) weights(8 + i * (8 / DB) + e);
                    asm volatile("" : "+v"(l));                            // the sum here, not behind all products
                }
                if (i == N / 2 - 1) pair_values(next);
                if (i >= N / 2) stage_values(next, BUF ^ 1, i - N / 2);
                if (i == 1) request_keys(next, t + 3);                     // their registers are free, and later those of the values
                if (i == N / 2) request_values(next);
                __builtin_amdgcn_sched_barrier(0);
            }
            request_scales(next);
            __syncthreads();
        };

        __syncthreads();
        auto all = [&](auto exact) __attribute__((always_inline)) {
            if (t0 < t_end) {
                page = page_of(t0);
                request(raw[0], t0);
                request(raw[1], t0 + 1);
                look(raw[0], 0, t0);
#pragma unroll
                for (int s = 0; s < S; ++s) stage_keys(exact, raw[0], 0, s);
                pair_values(raw[0]);
#pragma unroll
                for (int i = 0; i < NV; ++i) stage_values(raw[0], 0, i);
                request(raw[0], t0 + 2);
            }
#pragma unroll
            for (int s = 0; s < ST; ++s) asm volatile("" : "+v"(qf[s]));   // the queries have arrived: the loop does not wait for them
            __syncthreads();
            int t = t0;
            for (; t + 1 < t_end; t += 2) {                                // (a way out between the two would have every step wait for all requests)
                step(exact, std::integral_constant<int, 0>{}, t);
                step(exact, std::integral_constant<int, 1>{}, t + 1);
            }
            if (t < t_end) step(exact, std::integral_constant<int, 0>{}, t);
        };
        if (kend <= kFewKeys) all(std::true_type{});
        else all(std::false_type{});
        if (__builtin_expect((large != 0) & (lessen == 1.f), 0)) {            // the same for all: the last write to it lies before the last barrier
            lessen = kLessen;
            __syncthreads();
            continue;
        }
        if (limit > poison) l = NAN;
        {
            const uint32_t lb = __builtin_bit_cast(uint32_t, l);
            const auto x = __builtin_amdgcn_permlane32_swap(lb, lb, false, false);
            const uint32_t x0 = x[0], x1 = x[1];
            l = __builtin_bit_cast(float, x0) + __builtin_bit_cast(float, x1);
        }
        if (live) {                                                        // o[i][e]: dimension 32*i + 8*(e/4) + 4*h32 + e%4
            const size_t at = (size_t)tok * a.hq + qh, all = (size_t)a.p.T * a.hq;
            const float up = 1.f / lessen, f = l == 0.f ? 0.f : up / l;
#pragma unroll
            for (int i = 0; i < DB; ++i)
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    const int d = 32 * i + 8 * q + 4 * h32;
                    if (a.nsplit == 1) {
                        half4_t y;
#pragma unroll
                        for (int e = 0; e < 4; ++e) y[e] = (half_t)(o[i][4 * q + e] * f);
                        *reinterpret_cast<half4_t*>(a.out + at * D + d) = y;
                    } else {
                        float4_t y;
#pragma unroll
                        for (int e = 0; e < 4; ++e) y[e] = o[i][4 * q + e] * up;
                        *reinterpret_cast<float4_t*>(a.part + (split * all + at) * D + d) = y;
                    }
                }
            if (a.nsplit > 1 && h32 == 0) {
                float* ml = a.part + a.nsplit * all * D + (split * all + at) * 2;
                ml[0] = m;
                ml[1] = l;
            }
        }
        row0 += a.blocks * kPromptRows;
        lessen = 1.f;
        __syncthreads();
    }
}

// ---- joining the shares of the keys --------------------------------------------------------------
// One workgroup a row; 256 / (D/4) shares at a time.
template <int D>
__global__ __launch_bounds__(256) void kv4_attn_join_kernel(Kv4Attn a) {
    constexpr int DV = D / 4, PER = 256 / DV;
    __shared__ float wt[256];
    __shared__ float red[8];
    __shared__ __attribute__((aligned(16))) float acc[PER][D];
    const size_t all = (size_t)a.p.T * a.hq, row = blockIdx.x;
    const int t = (int)(row / a.hq);
    if (a.p.starts && (t < a.p.starts[0] || t >= a.p.starts[a.p.B])) return;      // uniform: a row behind the last sequence
    const float* ml = a.part + a.nsplit * all * D + row * 2;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    float m = -INFINITY, l = 0.f;
    if ((int)threadIdx.x < a.nsplit) { m = ml[threadIdx.x * all * 2]; l = ml[threadIdx.x * all * 2 + 1]; }
    float top = m;
#pragma unroll
    for (int s = 1; s < 64; s <<= 1) top = fmaxf(top, __shfl_xor(top, s));
    if (lane == 0) red[wave] = top;
    __syncthreads();
    top = fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3]));
    const float f = m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m - top);
    wt[threadIdx.x] = f;
    float sum = f * l;
#pragma unroll
    for (int s = 1; s < 64; s <<= 1) sum += __shfl_xor(sum, s);
    if (lane == 0) red[4 + wave] = sum;
    __syncthreads();
    sum = (red[4] + red[5]) + (red[6] + red[7]);
    const int d = threadIdx.x % DV * 4, s0 = threadIdx.x / DV;
    float4_t v = {0.f, 0.f, 0.f, 0.f};
    for (int s = s0; s < a.nsplit; s += 4 * PER) {
        float4_t x[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) x[k] = *reinterpret_cast<const float4_t*>(a.part + (min(s + k * PER, a.nsplit - 1) * all + row) * D + d);
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const float w = s + k * PER < a.nsplit ? wt[s + k * PER] : 0.f;
#pragma unroll
            for (int e = 0; e < 4; ++e) v[e] = fmaf(w, w == 0.f ? 0.f : x[k][e], v[e]);
        }
    }
    *reinterpret_cast<float4_t*>(&acc[s0][d]) = v;
    __syncthreads();
    if ((int)threadIdx.x < D) {
        float y = 0.f;
#pragma unroll
        for (int s = 0; s < PER; ++s) y += acc[s][threadIdx.x];
        a.out[row * D + threadIdx.x] = (half_t)(sum == 0.f ? 0.f : y / sum);
    }
}

// ---- plan ----------------------------------------------------------------------------------------
struct Kv4AttnPlan { bool prompt; int blocks, nsplit; };

// Above 64 rows a key head and sequence the prompt kernel, below it 16 rows a workgroup.
// Prompts: the keys are split into shares of 256 at least while no more than two workgroups stand for every compute unit, for the ones beyond would wait for all
// (189 tokens at 7227, 8 key heads of 4: 46.4 us in eleven shares, 42.9 in ten).
// Rows: the shares, of 256 keys at least (a tile per wavefront), make two workgroups of one sequence for every compute unit (131072 tokens of one: 31.9 us with 512
// workgroups, 34.1 with 1024, 39.1 with 2048, for the shares are joined), eight of four sequences or more, whose lengths differ (32 of up to 16384: 101.7, 82.3 and
// 77.2 us); where there are 1024 workgroups without, a share has 1024 keys at least (35 requests of 40 heads and up to 265 tokens: 38.7 us in two shares, 25.7 in one).
inline Kv4AttnPlan plan_kv4_attn(int B, int heads, int D, int share, int T, int max_tokens, int max_length) {
    Kv4AttnPlan p;
    const long rows = (long)max_tokens * share;
    p.prompt = rows > 64;
    const int per = p.prompt ? kPromptRows : 16;
    p.blocks = (int)std::max(1l, std::min((rows + per - 1) / per, (1l << 22) / ((long)B * heads)));   // a workgroup takes several where a launch has no room
    const long groups = (long)B * heads * p.blocks, wanted = p.prompt ? 512 : std::min(512l * B, 2048l);
    const long keys = !p.prompt && groups >= 1024 ? 1024 : 256, most = std::max(1l, (max_length + keys - 1) / keys);
    // bounds that are right ask for 200 MB at most; others must not ask for all memory, nor for more rows than the join can be launched for
    const long room = (1l << 30) / ((long)T * heads * share * (D + 2) * (long)sizeof(float));
    p.nsplit = (int)std::max(1l, std::min({most, (p.prompt ? wanted : wanted + groups - 1) / groups, 256l, room}));
    return p;
}

}  // namespace q4

size_t q4_kv4_attn_workspace(int B, int heads, int D, int share, int T, int max_tokens, int max_length) {
    const q4::Kv4AttnPlan p = q4::plan_kv4_attn(B, heads, D, share, T, max_tokens, max_length);
    return p.nsplit == 1 ? 0 : (size_t)p.nsplit * T * heads * share * (D + 2) * sizeof(float);
}

template <int D, int NG>
static void launch_attn(const q4::Kv4Attn& a, bool prompt, hipStream_t stream) {
    const dim3 grid((unsigned)((long)a.p.B * a.blocks * a.c.heads * a.nsplit));
    if (prompt) hipLaunchKernelGGL((q4::kv4_attn_prompt_kernel<D, NG>), grid, dim3(256), 0, stream, a);
    else hipLaunchKernelGGL((q4::kv4_attn_rows_kernel<D, NG>), grid, dim3(256), 0, stream, a);
    if (a.nsplit > 1)
        hipLaunchKernelGGL((q4::kv4_attn_join_kernel<D>), dim3((unsigned)((long)a.p.T * a.hq)), dim3(256), 0, stream, a);
}

int q4_launch_kv4_attn(q4::Kv4Attn& a, int D, int group, int max_tokens, int max_length, hipStream_t stream) {
    const q4::Kv4AttnPlan p = q4::plan_kv4_attn(a.p.B, a.c.heads, D, a.share, a.p.T, max_tokens, max_length);
    a.scale8 = a.scale * (1.f / q4::kLessen);
    a.blocks = p.blocks;
    a.nsplit = p.nsplit;
    const uint32_t p16 = a.c.page / 16;
    a.page_magic = p16 == 1 ? 0u : (uint32_t)(((1ull << 32) + p16 - 1) / p16);
    switch (D / group + (D == 64 ? 8 : 0)) {
        case 1: launch_attn<128, 1>(a, p.prompt, stream); break;
        case 2: launch_attn<128, 2>(a, p.prompt, stream); break;
        case 4: launch_attn<128, 4>(a, p.prompt, stream); break;
        case 9: launch_attn<64, 1>(a, p.prompt, stream); break;
        default: launch_attn<64, 2>(a, p.prompt, stream); break;
    }
    return hipGetLastError() == hipSuccess ? 0 : -4;
}
