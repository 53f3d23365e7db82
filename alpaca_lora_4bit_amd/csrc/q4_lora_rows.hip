// The low-rank adapters of many requests at once, added onto a product that all of them share:
//
//   y[m] += scaling[a] * (x[m] @ A[a]^T) @ B[a]^T in place,   a = index[m / per], none where a lies outside 0 .. n - 1
//
// for up to four layers that share x and the index (q | k | v).  The adapters of a layer are one bank, A [n, R, K] and B [n, N, R].
// Two launches: `down` leaves x @ A^T in fp32, as one sum or as sums over a few shares of K, `up` adds those in a fixed order and makes the update.  A
// tile of 1 to 32 rows, in any order, is gone through adapter by adapter: the rows of one prompt have one, a tile of a decode batch as many as
// rows.  Products are full 16-row tiles of v_mfma_f32_16x16x32_f16 either way; what a row's adapter did not make is not written.  HBM-bound: x and the used
// adapters are read once, y once and written once; the second and later reads of an adapter by other tiles come from the caches.
// x @ A^T * scaling goes to the matrix instructions as two fp16 numbers, the rounded one and what it left (ranks up to 16 have the room in one
// instruction), times a power of two of the row's own that takes its largest between 2^14 and 2^15: sums far beyond fp16, or far below, lose nothing.  So the
// update is rounded once, onto y.
#include "q4_common.hpp"
#include "q4_gptq.h"
#include <algorithm>

namespace q4 {

constexpr int kRowsProbs = 4;
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
    float* part;              // [problem][split][M][RP], RP = R filled up to 16, 32 or 64
    int M, K, R, n, per;
    int rows, splits, cols;   // rows of a tile (at most 32); shares of K; blocks of 256 columns (up)
};

// Adapter of each of a tile's rows (the lane is the row), -1 for none, and the rows that have one as a mask.
__device__ __forceinline__ int rows_adapter(const RowsArgs& a, int m0, uint64_t* pending) {
    const int r = threadIdx.x & 63, m = m0 + r;
    int idx = -1;
    if (r < a.rows && m < a.M) idx = a.index[m / a.per];
    if (idx >= a.n) idx = -1;
    *pending = __ballot(idx >= 0);
    return idx;
}
// The next adapter of a tile and its rows; the same in every wavefront.
__device__ __forceinline__ int rows_next(int idx, uint64_t* pending, uint64_t* mine) {
    const int ad = __builtin_amdgcn_readlane(idx, __builtin_ctzll(*pending));
    *mine = __ballot(idx == ad);
    *pending &= ~*mine;
    return ad;
}

// ---- x @ A^T ----------------------------------------------------------------------------------------
// Workgroup = 4 wavefronts on a tile and a share of K, which they take in chunks of 128 columns in turn; their products meet in LDS.  A chunk's rows
// are loaded 256 bytes by 16 neighbouring lanes (an operand's own order, a row a lane, costs the address unit four times the cycles: 701 rows of 11008
// features at rank 64 24 us) and pass to that order through LDS of the wavefront's own; the next chunk is on its way meanwhile.
constexpr int kRowsWaves = 4, kRowsChunk = 128;
template <int RB, int MT>     // 16-row blocks of A, filled up to 1, 2 or 4, and of the tile
__global__ __launch_bounds__(64 * kRowsWaves) void lora_rows_down_kernel(RowsArgs ra) {
    constexpr int NR = 16 * (RB + MT), LD = 4 * (RB + MT);                 // rows of a chunk: A's, then the tile's; four to a load
    constexpr int kTile = NR * (kRowsChunk + 8) * 2, kRed = MT * RB * 1024;
    __shared__ __attribute__((aligned(16))) char lds[kRowsWaves * (kTile > kRed ? kTile : kRed)];
    const RowsProb& p = ra.p[blockIdx.z];
    const int lane = threadIdx.x & 63, c = lane & 15, kk = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int m0 = blockIdx.x * ra.rows, rows = min(ra.rows, ra.M - m0);
    uint64_t pending, mine;
    const int idx = rows_adapter(ra, m0, &pending);
    const int chunks = (ra.K + kRowsChunk - 1) / kRowsChunk;
    const int c0 = (int)((long)chunks * blockIdx.y / ra.splits), c1 = (int)((long)chunks * (blockIdx.y + 1) / ra.splits);
    const rsrc_t rs_x = make_rsrc(ra.x + (size_t)m0 * ra.K, (unsigned)rows * (unsigned)ra.K * 2u);
    half_t (*tile)[kRowsChunk + 8] = reinterpret_cast<half_t(*)[kRowsChunk + 8]>(lds + wave * kTile);
    float (*red)[MT * RB][256] = reinterpret_cast<float(*)[MT * RB][256]>(lds);
    float* out = ra.part + ((size_t)blockIdx.z * ra.splits + blockIdx.y) * ra.M * (16 * RB);
    const int lr = lane >> 4, lc = 8 * (lane & 15);                        // row and column of this lane's piece of a load
    while (pending) {
        const int ad = rows_next(idx, &pending, &mine);
        const rsrc_t rs_a = make_rsrc(p.a + (size_t)ad * ra.R * ra.K, (unsigned)ra.R * (unsigned)ra.K * 2u);   // rows past R read as zero
        float4_t acc[MT][RB];
#pragma unroll
        for (int t = 0; t < MT; ++t)
#pragma unroll
            for (int b = 0; b < RB; ++b) acc[t][b] = float4_t{0.f, 0.f, 0.f, 0.f};
        uint4_t v[LD];
        auto request = [&](int ch) {
            const int col = ch * kRowsChunk + lc;
            const int at = ch < c1 && col < ra.K ? (lr * ra.K + col) * 2 : kRowsFar;      // what is not there comes as zero
#pragma unroll
            for (int i = 0; i < 4 * RB; ++i) v[i] = buf_load128(rs_a, at + 8 * i * ra.K, 0);
#pragma unroll
            for (int i = 0; i < 4 * MT; ++i)                               // four rows without this adapter: no traffic
                v[4 * RB + i] = buf_load128(rs_x, mine >> (4 * i) & 15u ? at + 8 * i * ra.K : kRowsFar, 0);
        };
        request(c0 + wave);
        for (int ch = c0 + wave; ch < c1; ch += kRowsWaves) {
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int i = 0; i < LD; ++i) *reinterpret_cast<uint4_t*>(&tile[4 * i + lr][lc]) = v[i];
            __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
            __builtin_amdgcn_wave_barrier();
            __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
            request(ch + kRowsWaves);
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int u = 0; u < kRowsChunk / 32; ++u) {
                half8_t av[RB], xv[MT];
#pragma unroll
                for (int b = 0; b < RB; ++b) av[b] = *reinterpret_cast<const half8_t*>(&tile[16 * b + c][32 * u + 8 * kk]);
#pragma unroll
                for (int t = 0; t < MT; ++t) xv[t] = *reinterpret_cast<const half8_t*>(&tile[16 * (RB + t) + c][32 * u + 8 * kk]);
#pragma unroll
                for (int t = 0; t < MT; ++t)
#pragma unroll
                    for (int b = 0; b < RB; ++b) acc[t][b] = __builtin_amdgcn_mfma_f32_16x16x32_f16(xv[t], av[b], acc[t][b], 0, 0, 0);
            }
            __builtin_amdgcn_wave_barrier();
        }
        __syncthreads();                                                   // the sums take the chunks' place
        // acc[t][b][e]: row 16*t + 4*kk + e, column 16*b + c
#pragma unroll
        for (int t = 0; t < MT; ++t)
#pragma unroll
            for (int b = 0; b < RB; ++b)
#pragma unroll
                for (int e = 0; e < 4; ++e) red[wave][t * RB + b][(4 * kk + e) * 16 + c] = acc[t][b][e];
        __syncthreads();
#pragma unroll
        for (int tb = 0; tb < MT * RB; ++tb) {
            const int e = threadIdx.x, row = 16 * (tb / RB) + (e >> 4), j = 16 * (tb % RB) + (e & 15);
            const float s = (red[0][tb][e] + red[1][tb][e]) + (red[2][tb][e] + red[3][tb][e]);
            if (mine >> row & 1) out[(size_t)(m0 + row) * (16 * RB) + j] = s;
        }
        __syncthreads();
    }
}

// Maximum over P (2, 4 or 8) neighbouring lanes, all of them active.
template <int P>
__device__ __forceinline__ uint32_t max_of_pieces(uint32_t x) {
    x = max(x, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0xB1, 0xF, 0xF, false));                   // lanes 1, 0, 3, 2 of four
    if constexpr (P > 2) x = max(x, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0x4E, 0xF, 0xF, false));     // lanes 2, 3, 0, 1
    if constexpr (P > 4) x = max(x, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0x141, 0xF, 0xF, false));    // lanes 7 .. 0 of eight
    return x;
}

// ---- the update -------------------------------------------------------------------------------------
// Workgroup = 256 columns, 64 a wavefront, of a tile of up to 16 * MT rows.  The sums become (rounded, rest) once, for all four; a wavefront's 64 rows of B and
// its products pass through LDS too, so that every access to memory is of whole lines by neighbouring lanes.  y is requested first of all.
template <int RB, int MT>     // 16 * RB = RP: pieces of eight 0 .. 2 * RB - 1, twice (rounded, rest), four to an instruction
__global__ __launch_bounds__(64 * kRowsWaves) void lora_rows_up_kernel(RowsArgs ra) {
    constexpr int P = 2 * RB, NS = RB == 4 ? 2 : 1;                        // NS pieces of B a lane, for RB instructions
    __shared__ half8_t sx[16 * MT][2 * P + 1];
    __shared__ half8_t sb[kRowsWaves][64][P + 1];
    __shared__ __attribute__((aligned(16))) float so[kRowsWaves][16][68];
    __shared__ float back[16 * MT];                                        // what takes a row's products to their own size again
    const RowsProb& p = ra.p[blockIdx.z];
    const int lane = threadIdx.x & 63, r = lane & 15, kk = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int m0 = (int)(blockIdx.x / ra.cols) * ra.rows, nb = blockIdx.x % ra.cols, n0 = nb * 256 + wave * 64;
    if (nb * 256 >= p.N) return;                                           // uniform: past a narrower layer of the launch
    const bool on = n0 < p.N;
    // this lane's outputs: rows m0 + 16*t + 8*i + lane/8, eight columns
    const int yr = lane >> 3, yc = n0 + 8 * (lane & 7), rows = min(ra.rows, ra.M - m0);
    half8_t y[MT][2];
#pragma unroll
    for (int t = 0; t < MT; ++t)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const int row = 16 * t + 8 * i + yr;
            y[t][i] = half8_t{};
            if (on && row < rows) y[t][i] = *reinterpret_cast<const half8_t*>(p.y + (size_t)(m0 + row) * p.N + yc);
        }
    uint64_t pending, mine;
    const int idx = rows_adapter(ra, m0, &pending);
    if (!pending) return;
    const uint64_t some = pending;
    const float factor = idx >= 0 ? p.scaling[idx] : 0.f;
    half8_t bw[P];                                                         // 64 rows of B, R / 8 pieces each, one after the other
    auto load_bank = [&](int ad) {
        const half8_t* bank = reinterpret_cast<const half8_t*>(p.b + ((size_t)ad * p.N + n0) * ra.R);
#pragma unroll
        for (int i = 0; i < P; ++i)
            if (on && 8 * i < ra.R) bw[i] = bank[64 * i + lane];
    };
    load_bank(__builtin_amdgcn_readlane(idx, __builtin_ctzll(pending)));
    const float* part = ra.part + ((size_t)blockIdx.z * ra.splits * ra.M + m0) * (8 * P);
    const size_t step = (size_t)ra.M * (8 * P);
    for (int i0 = 0; i0 < 16 * MT * P; i0 += 256) {
        const int i = i0 + threadIdx.x, row = min(i / P, 16 * MT - 1), j = i % P;
        const float f = __shfl(factor, row);
        if (i >= 16 * MT * P || !(some >> row & 1)) continue;
        const float* src = part + (size_t)row * (8 * P) + 8 * j;
        float4_t v = *reinterpret_cast<const float4_t*>(src), w = *reinterpret_cast<const float4_t*>(src + 4);
        int s = 1;
        for (; s + 3 <= ra.splits; s += 3) {                               // six loads on their way together
            float4_t a[3], b[3];
#pragma unroll
            for (int u = 0; u < 3; ++u) {
                a[u] = *reinterpret_cast<const float4_t*>(src + (s + u) * step);
                b[u] = *reinterpret_cast<const float4_t*>(src + (s + u) * step + 4);
            }
#pragma unroll
            for (int u = 0; u < 3; ++u) { v += a[u]; w += b[u]; }
        }
        for (; s < ra.splits; ++s) {
            v += *reinterpret_cast<const float4_t*>(src + s * step);
            w += *reinterpret_cast<const float4_t*>(src + s * step + 4);
        }
        v *= f;
        w *= f;
        uint32_t top = 0;                                                  // the row's largest magnitude; its P pieces lie in neighbouring lanes
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const float z = e < 4 ? v[e & 3] : w[e & 3];
            top = max(top, __builtin_bit_cast(uint32_t, z) & 0x7FFFFFFFu);
        }
        top = max_of_pieces<P>(top);
        const int shift = top >= 0x7F800000u ? 0 : min(127 + 14 - (int)(top >> 23), 100);
        const float grow = __builtin_bit_cast(float, (uint32_t)(127 + shift) << 23);
        if (j == 0) back[row] = __builtin_bit_cast(float, (uint32_t)(127 - shift) << 23);
        half8_t hi, lo;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const float x = (e < 4 ? v[e & 3] : w[e & 3]) * grow;
            hi[e] = (half_t)x;
            lo[e] = __builtin_isinf((float)hi[e]) ? (half_t)0.f : (half_t)(x - (float)hi[e]);
        }
        sx[row][j] = hi;
        sx[row][P + j] = lo;
    }
    __syncthreads();
    if (!on) return;
    float4_t acc[MT][4];
    float unit[MT];
#pragma unroll
    for (int t = 0; t < MT; ++t) {
        unit[t] = back[16 * t + r];                                        // of rows without an adapter: whatever, they are not written
#pragma unroll
        for (int u = 0; u < 4; ++u) acc[t][u] = float4_t{0.f, 0.f, 0.f, 0.f};
    }
    const int pieces = ra.R / 8;
    while (pending) {
        rows_next(idx, &pending, &mine);
#pragma unroll
        for (int i = 0; i < P; ++i)
            if (i < pieces) {
                const int at = 64 * i + lane;
                sb[wave][at / pieces][at % pieces] = bw[i];
            }
        __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
        __builtin_amdgcn_wave_barrier();
        __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
        if (pending) load_bank(__builtin_amdgcn_readlane(idx, __builtin_ctzll(pending)));
        half8_t bv[NS][4];
#pragma unroll
        for (int q = 0; q < NS; ++q) {
            const int seg = (4 * q + kk) % P;
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                bv[q][u] = half8_t{};
                if (seg < pieces) bv[q][u] = sb[wave][16 * u + r][seg];
            }
        }
        __builtin_amdgcn_wave_barrier();
#pragma unroll
        for (int t = 0; t < MT; ++t) {
            if (MT > 1 && !(mine >> (16 * t) & 0xFFFFu)) continue;
            // the lane's row takes the products of its own adapter only: zeros times an infinity of another one would be no zeros
            const bool own = mine >> (16 * t + r) & 1;
            float4_t sum[4];
#pragma unroll
            for (int u = 0; u < 4; ++u) sum[u] = float4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int i = 0; i < RB; ++i) {
                half8_t xb = {};
                if (own) xb = sx[16 * t + r][4 * i + kk];
#pragma unroll
                for (int u = 0; u < 4; ++u) sum[u] = __builtin_amdgcn_mfma_f32_16x16x32_f16(bv[i % NS][u], xb, sum[u], 0, 0, 0);
            }
#pragma unroll
            for (int u = 0; u < 4; ++u) acc[t][u] = own ? sum[u] : acc[t][u];
        }
    }
#pragma unroll
    for (int t = 0; t < MT; ++t) {                                         // acc[t][u]: row 16*t + r, columns 16*u + 4*kk ..
#pragma unroll
        for (int u = 0; u < 4; ++u) *reinterpret_cast<float4_t*>(&so[wave][r][16 * u + 4 * kk]) = acc[t][u] * unit[t];
        __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
        __builtin_amdgcn_wave_barrier();
        __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const int row = 16 * t + 8 * i + yr;
            const float4_t v = *reinterpret_cast<const float4_t*>(&so[wave][8 * i + yr][8 * (lane & 7)]);
            const float4_t w = *reinterpret_cast<const float4_t*>(&so[wave][8 * i + yr][8 * (lane & 7) + 4]);
            half8_t o;
#pragma unroll
            for (int e = 0; e < 8; ++e) o[e] = (half_t)((float)y[t][i][e] + (e < 4 ? v[e & 3] : w[e & 3]));
            if (some >> row & 1) *reinterpret_cast<half8_t*>(p.y + (size_t)(m0 + row) * p.N + yc) = o;
        }
        __builtin_amdgcn_wave_barrier();
    }
}

struct RowsPlan { int down_rows, splits, up_rows; };

// Up to 256 rows may be as many requests: their tiles are made smaller, a row each if need be, until the tiles and shares of 512 columns give 1024
// workgroups (64 rows of q, k and v, 32 adapters: 15.7 us at 256, 14.5 at 512, 13.7 at 1024); more rows are prompts' runs, 32 a tile, so that A is read less often
// (701 rows at rank 64: 26.3 us in tiles of 16, 24.3 of 32).  K is shared by as many workgroups as give 512 (tiles of whole blocks: 256, for every
// share leaves sums that all column blocks add up: 29.2 us at 512).  The update's tiles are made smaller until 512 workgroups stand (1024: 15.4 for 13.7 us).
inline RowsPlan plan_rows(int M, int K, int count, int n_max) {
    RowsPlan p;
    auto tiles = [&](int rows) { return ((long)M + rows - 1) / rows; };
    const long shares = (K + 511) / 512, cols = (n_max + 255) / 256;
    p.down_rows = 32;
    if (M <= 256)
        for (p.down_rows = 16; p.down_rows > 1 && tiles(p.down_rows) * count * shares < 1024;) p.down_rows >>= 1;
    p.splits = (int)std::max(1l, std::min(shares, (p.down_rows < 16 ? 512 : 256) / (tiles(p.down_rows) * count)));
    for (p.up_rows = 32; p.up_rows > 1 && tiles(p.up_rows) * cols * count < 512;) p.up_rows >>= 1;
    return p;
}

}  // namespace q4

size_t q4_lora_rows_workspace(int M, int K, int R, int count) {
    return (size_t)count * q4::plan_rows(M, K, count, 256).splits * M * (R <= 16 ? 16 : R <= 32 ? 32 : 64) * sizeof(float);
}

template <int RB>
static void launch_rows(q4::RowsArgs a, const q4::RowsPlan& p, int count, int n_max, hipStream_t stream) {
    const dim3 block(64 * q4::kRowsWaves);
    a.splits = p.splits;
    a.rows = p.down_rows;
    const dim3 down((a.M + a.rows - 1) / a.rows, a.splits, count);
    if (a.rows > 16) hipLaunchKernelGGL((q4::lora_rows_down_kernel<RB, 2>), down, block, 0, stream, a);
    else hipLaunchKernelGGL((q4::lora_rows_down_kernel<RB, 1>), down, block, 0, stream, a);
    a.rows = p.up_rows;
    a.cols = (n_max + 255) / 256;
    const dim3 up((unsigned)((long)((a.M + a.rows - 1) / a.rows) * a.cols), 1, count);
    if (a.rows > 16) hipLaunchKernelGGL((q4::lora_rows_up_kernel<RB, 2>), up, block, 0, stream, a);
    else hipLaunchKernelGGL((q4::lora_rows_up_kernel<RB, 1>), up, block, 0, stream, a);
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
        default: launch_rows<4>(a, p, count, n_max, stream); break;
    }
    return hipGetLastError() == hipSuccess ? 0 : -4;
}
