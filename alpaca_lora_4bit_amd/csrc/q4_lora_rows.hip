// The low-rank adapters of many requests at once, added onto a product that all of them share:
//
//   y[m] += scaling[a] * (x[m] @ A[a]^T) @ B[a]^T in place,   a = index[m / per], none where a lies outside 0 .. n - 1
//
// for up to four layers that share x and the index (q | k | v).  The adapters of a layer are one bank, A [n, R, K] and B [n, N, R].
// Two launches: `down` leaves fp32 partial sums of x @ A^T for shares of K, `up` adds them in a fixed order and makes the update.  A workgroup
// has a tile of 1 to 16 rows, in any order, and goes through the adapters that occur among them: the rows of one prompt have one, a tile of a
// decode batch as many as rows.  Products are full 16-row tiles of v_mfma_f32_16x16x32_f16 either way; what a row's adapter did not make is not
// written.  HBM-bound: x and the used adapters are read once, y once and written once; the second and later reads of an adapter by other tiles come
// from the caches.  x @ A^T * scaling goes to the matrix instructions as two fp16 numbers, the rounded one and what it left (ranks up to 16
// have the room in one instruction), so the update is rounded once, onto y.
#include "q4_common.hpp"
#include "q4_gptq.h"
#include <algorithm>

namespace q4 {

constexpr int kRowsProbs = 4, kRowsWaves = 4;
constexpr int kRowsFar = 0x70000000;      // beyond any buffer here: such loads return zero, no traffic

struct RowsProb {
    const half_t *a, *b;      // [n, R, K], [n, N, R]
    const float* scaling;     // [n]
    half_t* y;                // [M, N]
    int N;
};
struct RowsArgs {
    RowsProb p[kRowsProbs];
    const half_t* x;          // [M, K]
    const int* index;         // [ceil(M / per)]
    float* part;              // [problem][split][M][R]
    int M, K, R, n, per, rows, splits;
};

// Adapter of each of a tile's rows (lane % 16 is the row), -1 for none, and the rows that have one as a mask.
__device__ __forceinline__ int rows_adapter(const RowsArgs& a, int m0, uint32_t* pending) {
    const int r = threadIdx.x & 15, m = m0 + r;
    int idx = -1;
    if (r < a.rows && m < a.M) idx = a.index[m / a.per];
    if (idx >= a.n) idx = -1;
    *pending = (uint32_t)__ballot(idx >= 0) & 0xFFFFu;
    return idx;
}

template <int RB>             // 16-row blocks of A
__global__ __launch_bounds__(64 * kRowsWaves) void lora_rows_down_kernel(RowsArgs ra) {
    constexpr int UN = RB == 1 ? 8 : RB == 2 ? 4 : 2;                      // steps of 32 columns whose loads go out together
    __shared__ float red[kRowsWaves][RB][256];
    const RowsProb& p = ra.p[blockIdx.z];
    const int lane = threadIdx.x & 63, c = lane & 15, kk = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int m0 = blockIdx.x * ra.rows, rows = min(ra.rows, ra.M - m0);
    uint32_t pending;
    const int idx = rows_adapter(ra, m0, &pending);
    const int steps = ra.K / 32, parts = ra.splits * kRowsWaves, part = blockIdx.y * kRowsWaves + wave;
    const int s0 = (int)((long)steps * part / parts), s1 = (int)((long)steps * (part + 1) / parts);
    const rsrc_t rs_x = make_rsrc(ra.x + (size_t)m0 * ra.K, (unsigned)rows * (unsigned)ra.K * 2u);
    const int voff = (c * ra.K + 8 * kk) * 2;
    float* out = ra.part + ((size_t)blockIdx.z * ra.splits + blockIdx.y) * ra.M * ra.R;
    while (pending) {                                                      // the same in every wavefront
        const int ad = __builtin_amdgcn_readlane(idx, __builtin_ctz(pending));
        const uint32_t mine = (uint32_t)__ballot(idx == ad) & 0xFFFFu;
        pending &= ~mine;
        const rsrc_t rs_a = make_rsrc(p.a + (size_t)ad * ra.R * ra.K, (unsigned)ra.R * (unsigned)ra.K * 2u);   // rows past R read as zero
        float4_t acc[RB];
#pragma unroll
        for (int b = 0; b < RB; ++b) acc[b] = float4_t{0.f, 0.f, 0.f, 0.f};
        for (int s = s0; s < s1; s += UN) {
            uint4_t xv[UN], av[UN][RB];
#pragma unroll
            for (int u = 0; u < UN; ++u) {
                const int soff = s + u < s1 ? (s + u) * 64 : kRowsFar;
                xv[u] = buf_load128(rs_x, voff, soff);
#pragma unroll
                for (int b = 0; b < RB; ++b) av[u][b] = buf_load128(rs_a, voff + b * 32 * ra.K, soff);
            }
#pragma unroll
            for (int u = 0; u < UN; ++u)
#pragma unroll
                for (int b = 0; b < RB; ++b)
                    acc[b] = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(half8_t, xv[u]), __builtin_bit_cast(half8_t, av[u][b]),
                                                                    acc[b], 0, 0, 0);
        }
        // acc[b][e]: row 4*kk + e, column 16*b + c
#pragma unroll
        for (int b = 0; b < RB; ++b)
#pragma unroll
            for (int e = 0; e < 4; ++e) red[wave][b][(4 * kk + e) * 16 + c] = acc[b][e];
        __syncthreads();
#pragma unroll
        for (int b = 0; b < RB; ++b) {
            const int i = threadIdx.x, row = i >> 4, j = 16 * b + (i & 15);
            const float v = (red[0][b][i] + red[1][b][i]) + (red[2][b][i] + red[3][b][i]);
            if ((mine >> row & 1) && j < ra.R) out[(size_t)(m0 + row) * ra.R + j] = v;
        }
        __syncthreads();
    }
}

template <int RS>             // steps of 32: the 2 * R / 8 pieces of eight of (rounded, rest) in fours
__global__ __launch_bounds__(64 * kRowsWaves) void lora_rows_up_kernel(RowsArgs ra) {
    constexpr int RM = 16 * RS;
    __shared__ __attribute__((aligned(16))) float sx[16][RM + 4];
    const RowsProb& p = ra.p[blockIdx.z];
    if ((int)blockIdx.y * 256 >= p.N) return;                              // uniform: past a narrower layer of the launch
    const int lane = threadIdx.x & 63, r = lane & 15, kk = lane >> 4;
    const int m0 = blockIdx.x * ra.rows;
    uint32_t pending;
    const int idx = rows_adapter(ra, m0, &pending);
    if (!pending) return;
    const int n0 = blockIdx.y * 256 + (threadIdx.x >> 6) * 64;
    const bool live = idx >= 0 && n0 < p.N;
    // this lane's outputs: row m0 + r, columns n0 + 16*kk .. + 15
    half_t* y = p.y + (size_t)(m0 + r) * p.N + n0 + 16 * kk;
    half8_t y0 = {}, y1 = {};
    if (live) { y0 = *reinterpret_cast<const half8_t*>(y); y1 = *reinterpret_cast<const half8_t*>(y + 8); }
    const float* part = ra.part + (size_t)blockIdx.z * ra.splits * ra.M * ra.R;
    const int rv = ra.R / 4;
    for (int i = threadIdx.x; i < 16 * rv; i += 256) {
        const int row = i / rv, j = i % rv * 4;
        if (!(pending >> row & 1)) continue;
        float4_t v = {0.f, 0.f, 0.f, 0.f};
        for (int s = 0; s < ra.splits; ++s) v += *reinterpret_cast<const float4_t*>(part + ((size_t)s * ra.M + m0 + row) * ra.R + j);
        const float f = p.scaling[ra.index[(m0 + row) / ra.per]];
        *reinterpret_cast<float4_t*>(&sx[row][j]) = v * f;
    }
    __syncthreads();
    if (n0 >= p.N) return;
    const int pieces = ra.R / 8;
    float4_t acc[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) acc[u] = float4_t{0.f, 0.f, 0.f, 0.f};
    while (pending) {
        const int ad = __builtin_amdgcn_readlane(idx, __builtin_ctz(pending));
        pending &= ~((uint32_t)__ballot(idx == ad) & 0xFFFFu);
        const half_t* bank = p.b + ((size_t)ad * p.N + n0 + 16 * (r >> 2) + (r & 3)) * ra.R;
#pragma unroll
        for (int st = 0; st < RS; ++st) {
            const int q = 4 * st + kk;                                     // piece of (rounded | rest)
            const int seg = q < pieces ? q : q - pieces;
            const bool any = q < 2 * pieces;
            half8_t xb = {};
            if (any && idx == ad) {
                const float4_t f0 = *reinterpret_cast<const float4_t*>(&sx[r][8 * seg]), f1 = *reinterpret_cast<const float4_t*>(&sx[r][8 * seg + 4]);
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    const float f = e < 4 ? f0[e & 3] : f1[e & 3];
                    const half_t hi = (half_t)f;
                    xb[e] = q < pieces ? hi : __builtin_isinf((float)hi) ? (half_t)0.f : (half_t)(f - (float)hi);
                }
            }
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                half8_t bv = {};
                if (any) bv = *reinterpret_cast<const half8_t*>(bank + (size_t)(4 * u) * ra.R + 8 * seg);
                acc[u] = __builtin_amdgcn_mfma_f32_16x16x32_f16(bv, xb, acc[u], 0, 0, 0);
            }
        }
    }
    if (!live) return;
#pragma unroll
    for (int e = 0; e < 8; ++e) {                                          // acc[u][i]: column 16*kk + 4*u + i
        y0[e] = (half_t)((float)y0[e] + acc[e >> 2][e & 3]);
        y1[e] = (half_t)((float)y1[e] + acc[2 + (e >> 2)][e & 3]);
    }
    *reinterpret_cast<half8_t*>(y) = y0;
    *reinterpret_cast<half8_t*>(y + 8) = y1;
}

struct RowsPlan { int down_rows, up_rows, splits; };
// Shares of K of about 1024 columns (eight steps a wavefront, all their loads at once); the tiles of a few rows are made smaller until about
// two workgroups stand for every compute unit.
inline RowsPlan plan_rows(int M, int K, int probs, int n_max) {
    RowsPlan p;
    p.splits = std::max(1, (K + 1023) / 1024);
    p.down_rows = p.up_rows = 16;
    while (p.down_rows > 1 && (long)((M + p.down_rows - 1) / p.down_rows) * p.splits * probs < 512) p.down_rows >>= 1;
    while (p.up_rows > 1 && (long)((M + p.up_rows - 1) / p.up_rows) * ((n_max + 255) / 256) * probs < 512) p.up_rows >>= 1;
    return p;
}

}  // namespace q4

size_t q4_lora_rows_workspace(int M, int K, int R, int probs) {
    return (size_t)probs * q4::plan_rows(M, K, probs, 256).splits * M * R * sizeof(float);
}

template <int RB>
static void launch_rows(q4::RowsArgs a, const q4::RowsPlan& p, int probs, int n_max, hipStream_t stream) {
    const dim3 block(64 * q4::kRowsWaves);
    a.splits = p.splits;
    a.rows = p.down_rows;
    hipLaunchKernelGGL(q4::lora_rows_down_kernel<RB>, dim3((a.M + a.rows - 1) / a.rows, a.splits, probs), block, 0, stream, a);
    a.rows = p.up_rows;
    hipLaunchKernelGGL(q4::lora_rows_up_kernel<RB>, dim3((a.M + a.rows - 1) / a.rows, (n_max + 255) / 256, probs), block, 0, stream, a);
}

int q4_launch_lora_rows(const q4_lora_rows_t* probs, int count, const void* x, const int32_t* index, int per, int M, int K, int R, int n,
                        void* workspace, hipStream_t stream) {
    using namespace q4;
    RowsArgs a;
    int n_max = 0;
    for (int i = 0; i < count; ++i) {
        const q4_lora_rows_t& g = probs[i];
        a.p[i] = {reinterpret_cast<const half_t*>(g.a), reinterpret_cast<const half_t*>(g.b), g.scaling, reinterpret_cast<half_t*>(g.y), g.N};
        n_max = std::max(n_max, g.N);
    }
    a.x = reinterpret_cast<const half_t*>(x);
    a.index = index;
    a.part = reinterpret_cast<float*>(workspace);
    a.M = M; a.K = K; a.R = R; a.n = n; a.per = per;
    const RowsPlan p = plan_rows(M, K, count, n_max);
    switch ((R + 15) / 16) {
        case 1: launch_rows<1>(a, p, count, n_max, stream); break;
        case 2: launch_rows<2>(a, p, count, n_max, stream); break;
        case 3: launch_rows<3>(a, p, count, n_max, stream); break;
        default: launch_rows<4>(a, p, count, n_max, stream); break;
    }
    return hipGetLastError() == hipSuccess ? 0 : -4;
}
