// Attention of a batch's new tokens over the 4-bit key/value cache (layout in q4_kv4.hpp):
//
//   out[t, h] = sum_j p_j v_j,   p = softmax_j(scale * q[t, h] . k_j)   over the keys j at or before the token's own position
//
// One pass over the keys with the running maximum m and sum l of the softmax in fp32.  Codes go to the matrix instructions as the exact
// fp16 values that they stand for; the keys' scales multiply the fp32 scores, the values' scales the probabilities, whose rounding to
// fp16 is the only one before the output's.
#include "q4_kv4.hpp"
#include <algorithm>

namespace q4 {

// Probabilities are formed as 2^10 * exp(s - m): times a value's scale they then stay clear of fp16's subnormals down to 1e-7 of the
// largest for scales of 0.1, and below its largest number for scales up to 32; for larger scales the maximum is raised.
constexpr float kBoost = 10.0f, kMostScale = 32.0f;

__device__ __forceinline__ void wave_lds_fence() {
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
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
struct Kv4Tile {
    uint32_t k[4][D / 32];
    uint4_t v[4];
    uint4_t sc;               // eight scales: lane (kv, group, eighth of the tile)
};

template <int D, int NG>
__global__ __launch_bounds__(256, 2) void kv4_attn_rows_kernel(Kv4Attn a) {
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
    const int len = a.p.lengths[b], cap = a.p.width * a.c.page, p16 = a.c.page / 16;
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
        auto load = [&](Kv4Tile<D, NG>& x, uint2_t at) {
            const uint32_t kr = (uint32_t)__shfl((int)at.x, r >> 2) & 0x7FFFFFFFu, vr = (uint32_t)__shfl((int)at.x, kk) & 0x7FFFFFFFu;
            const uint32_t* kp = a.c.kc + (size_t)kr * (16 * W) + (r & 3) * W + kk * S;
            const uint32_t* vp = a.c.vc + (size_t)vr * (16 * W) + (r % W) * 4;
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                if constexpr (S == 4) *reinterpret_cast<uint4_t*>(x.k[u]) = __builtin_nontemporal_load(reinterpret_cast<const uint4_t*>(kp + u * 4 * W));
                else *reinterpret_cast<uint2_t*>(x.k[u]) = __builtin_nontemporal_load(reinterpret_cast<const uint2_t*>(kp + u * 4 * W));
            }
#pragma unroll
            for (int u = 0; u < 4; ++u) x.v[u] = __builtin_nontemporal_load(reinterpret_cast<const uint4_t*>(vp + u * 4 * W));
            const int piece = lane & 7, g = (lane >> 3) % NG;
            const uint32_t sr = (uint32_t)__shfl((int)at.y, piece >> 1);
            if (lane < 16 * NG)
                x.sc = *reinterpret_cast<const uint4_t*>((lane < 8 * NG ? a.c.ks : a.c.vs) + ((size_t)sr + g * p16) * 16 + 8 * (piece & 1));
        };
        auto compute = [&](const Kv4Tile<D, NG>& x, uint2_t at, int tile) {
            if (lane < 16 * NG) *reinterpret_cast<uint4_t*>(&scales[wave][0][0][0] + 8 * lane) = x.sc;
            wave_lds_fence();
            float s[16];
#pragma unroll
            for (int g = 0; g < NG; ++g) {
                float4_t acc[4];
#pragma unroll
                for (int u = 0; u < 4; ++u) acc[u] = float4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int st = g * SG; st < (g + 1) * SG; ++st)
#pragma unroll
                    for (int u = 0; u < 4; ++u)
                        acc[u] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kv4_word(x.k[u][st]), qf[st], acc[u], 0, 0, 0);
                const half8_t k0 = *reinterpret_cast<const half8_t*>(&scales[wave][0][g][16 * kk]);
                const half8_t k1 = *reinterpret_cast<const half8_t*>(&scales[wave][0][g][16 * kk + 8]);
#pragma unroll
                for (int e = 0; e < 16; ++e) {
                    const float ks = (float)(e < 8 ? k0[e & 7] : k1[e & 7]);
                    s[e] = g == 0 ? acc[e >> 2][e & 3] * ks : fmaf(acc[e >> 2][e & 3], ks, s[e]);
                }
            }
            half8_t sv[NG][2];
#pragma unroll
            for (int g = 0; g < NG; ++g)
#pragma unroll
                for (int v = 0; v < 2; ++v) sv[g][v] = *reinterpret_cast<const half8_t*>(&scales[wave][1][g][16 * kk + 8 * v]);
            __builtin_amdgcn_wave_barrier();
            const bool bad = (uint32_t)__shfl((int)at.x, kk) >> 31;
            if (tile * 64 + 64 > kmin || __any(bad)) {                     // whatever a place that is not seen holds, it counts nothing
                const int seen = bad ? 0 : limit - (tile * 64 + 16 * kk);
#pragma unroll
                for (int e = 0; e < 16; ++e) {
                    s[e] = e < seen ? s[e] : -INFINITY;
#pragma unroll
                    for (int g = 0; g < NG; ++g) sv[g][e >> 3][e & 7] = e < seen ? sv[g][e >> 3][e & 7] : (half_t)0.f;
                }
            }
            float mx = s[0];
#pragma unroll
            for (int e = 1; e < 16; ++e) mx = fmaxf(mx, s[e]);
            half8_t big8 = sv[0][0];
#pragma unroll
            for (int g = 0; g < NG; ++g)
#pragma unroll
                for (int v = 0; v < 2; ++v) big8 = __builtin_elementwise_max(big8, sv[g][v]);
            half_t bigh = big8[0];
#pragma unroll
            for (int e = 1; e < 8; ++e) bigh = __builtin_elementwise_max(bigh, big8[e]);
            float big = (float)bigh;
            mx = fmaxf(mx, __shfl_xor(mx, 16));
            mx = fmaxf(mx, __shfl_xor(mx, 32));
            float mn = mx * a.scale;
            if (__any(big > kMostScale)) {
                big = fmaxf(big, __shfl_xor(big, 16));
                big = fmaxf(big, __shfl_xor(big, 32));
                mn += log2f(fmaxf(big, kMostScale) / kMostScale);
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
            float p[16];
#pragma unroll
            for (int e = 0; e < 16; ++e) {
                p[e] = __builtin_amdgcn_exp2f(fmaf(s[e], a.scale, kBoost - base));
                l += p[e];
            }
#pragma unroll
            for (int v = 0; v < 2; ++v) {
                uint32_t lo[4], hi[4];                                     // even and odd nibbles of two keys side by side
#pragma unroll
                for (int c = 0; c < 4; ++c) {
                    const uint4_t w = x.v[2 * v + (c >> 1)];
                    uint32_t wa = c & 1 ? w.z : w.x, wb = c & 1 ? w.w : w.y;
                    if constexpr (D == 64) { wa >>= 16 * (r >> 3); wb >>= 16 * (r >> 3); }
                    lo[c] = (wa & 0x0F0F0F0Fu) | ((wb << 4) & 0xF0F0F0F0u);
                    hi[c] = ((wa >> 4) & 0x0F0F0F0Fu) | (wb & 0xF0F0F0F0u);
                }
#pragma unroll
                for (int g = 0; g < NG; ++g) {
                    half8_t pb;
#pragma unroll
                    for (int e = 0; e < 8; ++e) pb[e] = (half_t)(p[8 * v + e] * (float)sv[g][v][e]);
#pragma unroll
                    for (int i = g * HG; i < (g + 1) * HG; ++i) {
                        half8_t va;
#pragma unroll
                        for (int c = 0; c < 4; ++c) {
                            const uint32_t w = i & 1 ? hi[c] : lo[c];
                            const half2_t d = i / 2 == 0 ? kv4_pair<0>(w) : i / 2 == 1 ? kv4_pair<1>(w) : i / 2 == 2 ? kv4_pair<2>(w) : kv4_pair<3>(w);
                            va[2 * c] = d[0];
                            va[2 * c + 1] = d[1];
                        }
                        o[i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(va, pb, o[i], 0, 0, 0);
                    }
                }
            }
        };

        // tiles wave, wave + 4, ... of the share; while one is worked on, the next one's codes and the page entries of the one behind it are on their way
        Kv4Tile<D, NG> xa, xb;
        int t = split * per + wave;
        uint2_t pa = {0u, 0u}, pb = {0u, 0u};
        if (t < t_end) { pa = look_up(t); load(xa, pa); pb = look_up(t + 4); }
        for (; t < t_end; t += 8) {
            uint2_t pc = {0u, 0u};
            if (t + 4 < t_end) { load(xb, pb); pc = look_up(t + 8); }
            compute(xa, pa, t);
            if (t + 4 >= t_end) break;
            pa = pc;
            uint2_t pd = {0u, 0u};
            if (t + 8 < t_end) { load(xa, pa); pd = look_up(t + 12); }
            compute(xb, pb, t + 4);
            pb = pd;
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
                for (int e = 0; e < 4; ++e) y[e] = (half_t)(top == -INFINITY ? 0.f : v[e] / sum);
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
    for (int s = s0; s < a.nsplit; s += PER) {
        const float w = wt[s];
        if (w == 0.f) continue;
        const float4_t x = *reinterpret_cast<const float4_t*>(a.part + (s * all + row) * D + d);
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = fmaf(w, x[e], v[e]);
    }
    *reinterpret_cast<float4_t*>(&acc[s0][d]) = v;
    __syncthreads();
    if ((int)threadIdx.x < D) {
        float y = 0.f;
#pragma unroll
        for (int s = 0; s < PER; ++s) y += acc[s][threadIdx.x];
        a.out[row * D + threadIdx.x] = (half_t)(top == -INFINITY ? 0.f : y / sum);
    }
}

// ---- plan ----------------------------------------------------------------------------------------
struct Kv4AttnPlan { int blocks, nsplit; };

// Row blocks of 16 for the longest run of new tokens; the keys in shares until about four workgroups stand for every compute unit, a share
// of 256 keys (a tile per wavefront) at least.
inline Kv4AttnPlan plan_kv4_attn(int B, int heads, int share, int max_tokens, int max_length) {
    Kv4AttnPlan p;
    p.blocks = (int)(((long)max_tokens * share + 15) / 16);
    const long groups = (long)B * heads * p.blocks;
    const long most = std::max(1, (max_length + 255) / 256);
    p.nsplit = (int)std::max(1l, std::min({most, (1024 + groups - 1) / groups, 256l}));
    return p;
}

}  // namespace q4

size_t q4_kv4_attn_workspace(int B, int heads, int D, int share, int T, int max_tokens, int max_length) {
    const q4::Kv4AttnPlan p = q4::plan_kv4_attn(B, heads, share, max_tokens, max_length);
    return p.nsplit == 1 ? 0 : (size_t)p.nsplit * T * heads * share * (D + 2) * sizeof(float);
}

template <int D, int NG>
static void launch_rows(const q4::Kv4Attn& a, hipStream_t stream) {
    const dim3 grid((unsigned)((long)a.p.B * a.blocks * a.c.heads * a.nsplit));
    hipLaunchKernelGGL((q4::kv4_attn_rows_kernel<D, NG>), grid, dim3(256), 0, stream, a);
    if (a.nsplit > 1)
        hipLaunchKernelGGL((q4::kv4_attn_join_kernel<D>), dim3((unsigned)((long)a.p.T * a.hq)), dim3(256), 0, stream, a);
}

int q4_launch_kv4_attn(q4::Kv4Attn& a, int D, int group, int max_tokens, int max_length, hipStream_t stream) {
    const q4::Kv4AttnPlan p = q4::plan_kv4_attn(a.p.B, a.c.heads, a.share, max_tokens, max_length);
    a.blocks = p.blocks;
    a.nsplit = p.nsplit;
    const uint32_t p16 = a.c.page / 16;
    a.page_magic = p16 == 1 ? 0u : (uint32_t)(((1ull << 32) + p16 - 1) / p16);
    switch (D / group + (D == 64 ? 8 : 0)) {
        case 1: launch_rows<128, 1>(a, stream); break;
        case 2: launch_rows<128, 2>(a, stream); break;
        case 4: launch_rows<128, 4>(a, stream); break;
        case 9: launch_rows<64, 1>(a, stream); break;
        default: launch_rows<64, 2>(a, stream); break;
    }
    return hipGetLastError() == hipSuccess ? 0 : -4;
}
