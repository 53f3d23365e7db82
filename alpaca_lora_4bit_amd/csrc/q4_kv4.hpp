// The 4-bit key/value cache: its layout, the places of a batch's tokens in it, and the conversions of its codes.
//
// A value is code * scale.  Codes are 4-bit floats (1 sign, 2 exponent, 1 mantissa bit: 0, 0.5, 1, 1.5, 2, 3, 4, 6), which this
// chip converts from and to by single instructions, two values at a time; the scale is one fp16 number, largest magnitude / 6,
// for `group` = D / NG dimensions of one token and head.  Pages hold `page` tokens (a multiple of 16) of all heads:
//
//   k_codes  [pages][heads][page][D/8]        word kk*(D/32) + s of a token, kk < 4: dimensions 32*s + 8*kk .. + 7, lowest nibble first
//   v_codes  [pages][heads][page/4][D/8][4]   word j of four tokens side by side; with H = D/16, nibble i + H*r of word j is dimension
//                                             16*i + (D/8)*r + j
//   scales   [pages][heads][NG][page]
//
// So one 16-byte load of a lane (8 bytes for the keys of 64-wide heads) is an operand of the matrix instructions: the keys' words lie along
// the head's dimensions, over which q . k sums, with every step of 32 inside one group, and the values' words side by side for four tokens,
// over which p . v sums.  A token's codes share no word with another token's: appending one token reads nothing back.
#pragma once
#include "q4_common.hpp"

namespace q4 {

struct Kv4Cache {
    uint32_t *kc, *vc;
    half_t *ks, *vs;
    int pages, page, heads;
};

// Where the rows of a batch belong: sequence b holds rows starts[b] .. starts[b + 1] - 1 (null: T / B each) at the last places of its
// lengths[b] tokens, whose pages are table[b][0 .. width - 1].
struct Kv4Batch {
    const int *table, *lengths, *starts;
    int width, B, T;
};

// What the launches take.
struct Kv4Append {
    Kv4Cache c;
    Kv4Batch p;
    const half_t *k, *v, *q;          // q null: none
    half_t* q_out;                    // [T, hq, D]
    long k_t, k_h, v_t, v_h, q_t, q_h;
    const float* rope;                // [rope_rows][rot/2][2]; rot 0: no rotation
    int rope_rows, rot, interleaved, hq;
    int turns;                        // heads a wavefront takes one after the other
};

struct Kv4Read {
    Kv4Cache c;
    Kv4Batch p;
    half_t *k, *v;                    // [T, heads, D]
    int turns;
};

struct Kv4Attn {
    Kv4Cache c;
    Kv4Batch p;
    const half_t* q;
    long q_t, q_h;
    half_t* out;              // [T, hq, D]
    float* part;              // [nsplit][T * hq][D] sums, then [nsplit][T * hq][2] maxima and sums of weights; null: nsplit 1
    float scale, scale8;      // softmax scale * log2(e), and eight times that
    int hq, share, nsplit, blocks;    // share = hq / heads; row blocks in the grid
    uint32_t page_magic;      // ceil(2^32 / (page / 16)), 0 for pages of 16
};

// A sequence's length, so far inside 32 bits that a batch's rows can be added and taken away: at most 2^26 places and 2^24 rows can matter.
__device__ __forceinline__ int kv4_length(const Kv4Batch& p, int b) { return min(max(p.lengths[b], -(1 << 25)), 1 << 28); }

struct Kv4Place {
    int pos, page, off;       // position in the sequence, page and offset in it
    bool mine, ok;            // the row belongs to a sequence; it has a place in the cache
};

// Place of row t, looked up by LANES neighbouring lanes together (all of them ask for the same t).
template <int LANES>
__device__ __forceinline__ Kv4Place kv4_place(const Kv4Cache& c, const Kv4Batch& p, int t) {
    Kv4Place r{0, 0, 0, false, false};
    int b, first, end;
    if (p.starts == nullptr) {
        const int n = p.T / p.B;
        b = t / n;
        first = b * n;
        end = first + n;
        r.mine = t < p.T;
    } else {
        int count = 0;                                     // sequences that end at or before t; starts do not fall
        for (int i = threadIdx.x % LANES; i < p.B; i += LANES) count += p.starts[i + 1] <= t;
#pragma unroll
        for (int m = 1; m < LANES; m <<= 1) count += __shfl_xor(count, m);
        b = count;
        r.mine = t < p.T && b < p.B;
        if (!r.mine) return r;
        first = p.starts[b];
        end = p.starts[b + 1];
        r.mine = t >= first;
    }
    if (!r.mine) return r;
    r.pos = kv4_length(p, b) - end + t;
    if (r.pos < 0 || r.pos / c.page >= p.width) return r;
    r.page = p.table[(size_t)b * p.width + r.pos / c.page];
    r.off = r.pos % c.page;
    r.ok = r.page >= 0 && r.page < c.pages;
    return r;
}

// two of the four code bytes' values, times `factor`, a power of two: byte SEL of w, low nibble first
template <int SEL>
__device__ __forceinline__ half2_t kv4_pair(uint32_t w, float factor = 1.0f) {
    return __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, factor, SEL);
}
__device__ __forceinline__ half8_t kv4_word(uint32_t w) {
    const uint4_t x = {as_u32(kv4_pair<0>(w)), as_u32(kv4_pair<1>(w)), as_u32(kv4_pair<2>(w)), as_u32(kv4_pair<3>(w))};
    return __builtin_bit_cast(half8_t, x);
}
// codes of eight values, to nearest, ties to the even code, beyond 6 to 6
__device__ __forceinline__ uint32_t kv4_codes(const float* y) {
    uint32_t w = 0;
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, y[0], y[1], 1.0f, 0);
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, y[2], y[3], 1.0f, 1);
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, y[4], y[5], 1.0f, 2);
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, y[6], y[7], 1.0f, 3);
    return w;
}

}  // namespace q4

int q4_launch_kv4_append(const q4::Kv4Append& a, int D, int group, bool vec, hipStream_t stream);
int q4_launch_kv4_read(const q4::Kv4Read& a, int D, int group, hipStream_t stream);
size_t q4_kv4_attn_workspace(int B, int heads, int D, int share, int T, int max_tokens, int max_length);
int q4_launch_kv4_attn(q4::Kv4Attn& a, int D, int group, int max_tokens, int max_length, hipStream_t stream);
