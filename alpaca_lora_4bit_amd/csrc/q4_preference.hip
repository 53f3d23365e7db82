// Log-probabilities of the tokens of answers from logits, their gradient, and the loss of pairs of answers (paired log ratios).
//
//   logp = x_l - L        L = m + log(sum of exp(x - m)) for any m        dx = c (1[l] - exp(x - L))
//
// HBM-bound: one pass over a row's logits, backward one pass more from the L that forward left (an answer's factor c needs all of its tokens first).
// Rows whose label is not one of the V words are no tokens of an answer (a prompt, padding): they are not read, and their gradient is zero.
// Exponentials in fp32, their sums and what follows in fp64: a log ratio is the small difference of sums of some hundred log-probabilities, and an
// error in one direction grows with the answer (over answers of 2048 tokens 1.1e-9 a token at most).  us and TB/s moved, 16 pairs of 1024 places of 32000
// words in fp16 of which 17370 are tokens: forward 186 (6.0), log ratios and loss 10, backward 527 (6.1); a large copy reaches 5.15.
#include "q4_common.hpp"
#include "q4_gptq.h"
#include "q4_preference.hpp"

namespace q4 {

constexpr float kLog2eHi = 0x1.715476p+0f, kLog2eLo = 0x1.4ae0c0p-26f;       // log2(e) in two parts
// v_exp_f32 is short by so much of itself on average: 1.24e-9 for arguments of 1 and more, 3.42e-9 for -1 and less, over all fp32 numbers of each power of
// two's range up to 128; what is left, 1.1e-9, is that of a row whose words all lie on one side of its label.
constexpr double kExpShort = 2.33e-9;

// exp(d).  With one fp32 factor log2(e) every exponent is short by 1.3e-8 of itself: all in one direction, which a log ratio over a
// long answer adds up.
__device__ __forceinline__ float exp_of(float d) { return __builtin_amdgcn_exp2f(fmaf(d, kLog2eHi, d * kLog2eLo)); }

template <typename T>
struct Pack {
    static constexpr int N = 16 / sizeof(T);
    T v[N];
};
// a 16-byte load from any value's address
template <typename T>
__device__ __forceinline__ Pack<T> load_pack(const T* p) {
    Pack<T> r;
    __builtin_memcpy(&r, p, 16);
    return r;
}
template <typename T>
__device__ __forceinline__ void store_pack(T* p, const Pack<T>& r) { *reinterpret_cast<uint4_t*>(p) = __builtin_bit_cast(uint4_t, r); }
// past the caches: a gradient of long rows is more than they hold
template <bool PAST, typename T>
__device__ __forceinline__ void store_grad(T* p, const Pack<T>& r) {
    if constexpr (PAST) __builtin_nontemporal_store(__builtin_bit_cast(uint4_t, r), reinterpret_cast<uint4_t*>(p));
    else store_pack(p, r);
}

// Values of a row before the first 16-byte boundary, packs behind it, values left.
template <typename T>
struct Split {
    int head, packs, tail;
    __device__ __forceinline__ Split(const T* row, int V) {
        const int to = (int)((0u - (unsigned)reinterpret_cast<uintptr_t>(row)) & 15u) / (int)sizeof(T);
        head = to < V ? to : V;
        packs = (V - head) / Pack<T>::N;
        tail = V - head - packs * Pack<T>::N;
    }
};

// Sum of exp(x - at) of a lane's values, in fp64: beside a word that has most of the weight the many small ones would each lose up to half a unit of an fp32 sum, all
// in one direction (a word 18.5 above 32000 others, sums of packs in fp32 and of those with Kahan's: 3e-8 a token).  us, fp32 / fp64: 32768 rows of 32000 fp16, 0.55
// of them tokens, 200 / 199; 8192 of bfloat16 90.5 / 90.3; 32768 of 1600 28.7 / 29.8, of 320 17.3 / 17.8.
struct Sum {
    double s = 0.0;
    template <typename T, int N>
    __device__ __forceinline__ void add(const T (&x)[N], float at) {
        double part[N];
#pragma unroll
        for (int e = 0; e < N; ++e) part[e] = (double)exp_of((float)x[e] - at);
#pragma unroll
        for (int w = N / 2; w >= 1; w /= 2)
#pragma unroll
            for (int e = 0; e < w; ++e) part[e] += part[e + w];
        s += part[0];
    }
};

__device__ __forceinline__ float wave_max(float v) {
#pragma unroll
    for (int d = 1; d < 64; d *= 2) v = fmaxf(v, __shfl_xor(v, d));
    return v;
}
__device__ __forceinline__ double wave_sum(double v) {
#pragma unroll
    for (int d = 1; d < 64; d *= 2) v += __shfl_xor(v, d);
    return v;
}

template <typename T>
__device__ __forceinline__ const T* row_of(const LogitsView& a, long row) {
    const long b = row / a.S, t = row - b * a.S;
    return reinterpret_cast<const T*>(a.x) + b * a.sb + t * a.st;
}

template <int WAVES>
__device__ __forceinline__ float group_max(float v, float* lds) {
    v = wave_max(v);
    if constexpr (WAVES > 1) {
        __syncthreads();
        if (threadIdx.x % 64 == 0) lds[threadIdx.x / 64] = v;
        __syncthreads();
#pragma unroll
        for (int w = 0; w < WAVES; ++w) v = fmaxf(v, lds[w]);
    }
    return v;
}
template <int WAVES>
__device__ __forceinline__ double group_sum(double v, double* lds) {
    v = wave_sum(v);
    if constexpr (WAVES > 1) {
        __syncthreads();
        if (threadIdx.x % 64 == 0) lds[threadIdx.x / 64] = v;
        __syncthreads();
        v = 0.0;
#pragma unroll
        for (int w = 0; w < WAVES; ++w) v += lds[w];
    }
    return v;
}

// A row's sum of exp(x - at), at = the label's own logit: exponents need no maximum first, and what follows is -log(sum).  Where the label's logit is
// so far below others that this leaves fp32 (by 80 and more), or is -infinity, or the row has a NaN or +infinity, the row is read again for its maximum and once more
// for the sum beside it; -infinity elsewhere is no weight at the first reading.  `logps` or `wide` (the other is null) takes the log-probability: in fp32 for a caller, in fp64 for the log ratios.
template <typename T, int THREADS>
__global__ __launch_bounds__(THREADS) void token_logps_kernel(LogitsView a, const long long* __restrict__ labels, float* __restrict__ logps, double* __restrict__ wide,
                                                              float2* __restrict__ stats) {
    constexpr int N = Pack<T>::N, WAVES = THREADS / 64, U = THREADS == 256 ? 8 : 4;
    __shared__ float sm[WAVES];
    __shared__ double ss[WAVES];
    const int tid = threadIdx.x;
    const long rows = (long)a.B * a.S;
    for (long row = blockIdx.x; row < rows; row += gridDim.x) {
        const long long label = labels[row];
        if (label < 0 || label >= a.V) {
            if (tid == 0) {
                if (logps) logps[row] = 0.f;
                else wide[row] = 0.0;
                stats[row] = float2{0.f, 0.f};
            }
            continue;
        }
        const T* x = row_of<T>(a, row);
        const float mine = (float)x[label];
        const int packs = a.V / N, tail = a.V - packs * N;
        Sum r;
        for (int i = tid; i < packs; i += U * THREADS) {
            Pack<T> p[U];
#pragma unroll
            for (int u = 0; u < U; ++u) {                                    // all on their way, the ones behind the end from the last place
                const int k = i + u * THREADS;
                p[u] = load_pack(x + (long)(k < packs ? k : packs - 1) * N);
            }
#pragma unroll
            for (int u = 0; u < U; ++u)
                if (i + u * THREADS < packs) r.add(p[u].v, mine);
        }
        if (tid < tail) { const T one[1] = {x[(long)packs * N + tid]}; r.add(one, mine); }
        double s = group_sum<WAVES>(r.s, ss);
        float at = mine;
        if (!(s < 0x1p115)) {                                                // the same in all threads
            at = -0x1.FFFFFEp127f;                                           // rows of this number or of -infinity give what their definition gives
            for (long i = tid; i < a.V; i += THREADS) at = fmaxf(at, (float)x[i]);
            at = group_max<WAVES>(at, sm);
            Sum again;
            for (long i = tid; i < a.V; i += THREADS) { const T one[1] = {x[i]}; again.add(one, at); }
            s = group_sum<WAVES>(again.s, ss);
        }
        if (tid == 0) {
            // one term of the sum, exp(0), is exact; the fp32 logarithm would be 3e-7 short on average
            const double total = log(s + kExpShort * (s - 1.0)), lp = ((double)mine - (double)at) - total;
            if (logps) logps[row] = (float)lp;
            else wide[row] = lp;
            // what backward takes: L in two parts, so that logits near it lose nothing when it is taken off (a row of the lowest number has all of
            // the sum's logarithm in the second)
            const float most = (float)((double)at + total);
            stats[row] = float2{most, (float)(total - ((double)most - (double)at))};
        }
    }
}

template <typename T, int THREADS>
__global__ __launch_bounds__(THREADS) void token_logps_bwd_kernel(LogitsView a, const long long* __restrict__ labels, const float2* __restrict__ stats,
                                                                  const float* __restrict__ coef, int per, const float* __restrict__ factor, T* __restrict__ dx) {
    constexpr int N = Pack<T>::N, U = 4;
    constexpr bool PAST = THREADS == 1024;
    const int tid = threadIdx.x;
    const long rows = (long)a.B * a.S;
    for (long row = blockIdx.x; row < rows; row += gridDim.x) {
        const long long label = labels[row];
        T* out = dx + row * a.V;
        const Split<T> so(out, a.V);                                         // stores from 16-byte boundaries on, loads from wherever that is
        if (label < 0 || label >= a.V) {
            Pack<T> zero;
#pragma unroll
            for (int e = 0; e < N; ++e) zero.v[e] = (T)0.f;
            for (int i = tid; i < so.packs; i += THREADS) store_grad<PAST>(out + so.head + (long)i * N, zero);
            if (tid < so.head) out[tid] = (T)0.f;
            if (tid < so.tail) out[so.head + (long)so.packs * N + tid] = (T)0.f;
            continue;
        }
        const T* x = row_of<T>(a, row);
        const float2 st = stats[row];
        const float c = (factor ? *factor : 1.f) * coef[row / per];
        // In fp32: the distance to L is off by half a unit of itself, its exponent by 1.3e-8 (one log2(e)), together 1e-6 of a probability of e^-16 and less of larger
        // ones: below the rounding to 16 bits, and in fp32 what softmax's own gradient has; no sum of these needs more.
        auto share = [&](T v) { return (T)(-c * __expf(((float)v - st.x) - st.y)); };
        // the label's own gradient c (1 - p), formed without that difference
        auto own = [&](T v) { return (T)(-c * expm1f(((float)v - st.x) - st.y)); };
        for (int i = tid; i < so.packs; i += U * THREADS) {
            Pack<T> p[U];
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int k = i + u * THREADS;
                p[u] = load_pack(x + so.head + (long)(k < so.packs ? k : so.packs - 1) * N);
            }
#pragma unroll
            for (int u = 0; u < U; ++u) {
                if (i + u * THREADS >= so.packs) break;
                const long at = so.head + (long)(i + u * THREADS) * N;
                Pack<T> g;
#pragma unroll
                for (int e = 0; e < N; ++e) g.v[e] = share(p[u].v[e]);
                if ((unsigned long)(label - at) < N) {
#pragma unroll
                    for (int e = 0; e < N; ++e)
                        if (label == at + e) g.v[e] = own(p[u].v[e]);
                }
                store_grad<PAST>(out + at, g);
            }
        }
        if (tid < so.head) out[tid] = tid == label ? own(x[tid]) : share(x[tid]);
        const long at = so.head + (long)so.packs * N + tid;
        if (tid < so.tail) out[at] = at == label ? own(x[at]) : share(x[at]);
    }
}

constexpr int kRatioThreads = 256, kPairThreads = 1024;

// This thread's share of an answer's log ratio, threads apart; four places on their way.
__device__ __forceinline__ double ratio_share(const double* __restrict__ logps, const float* __restrict__ ref, const long long* __restrict__ labels, int S, int V, int first,
                                              int apart) {
    double sum = 0.0;
    for (int t = first; t < S; t += 4 * apart) {
        long long l[4];
        double x[4];
        float y[4];
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            const int k = t + u * apart < S ? t + u * apart : S - 1;
            l[u] = t + u * apart < S ? labels[k] : -1;
            x[u] = logps[k];
            y[u] = ref[k];
        }
#pragma unroll
        for (int u = 0; u < 4; ++u)
            if (l[u] >= 0 && l[u] < V) sum += x[u] - (double)y[u];           // what the reference says elsewhere is not looked at
    }
    return sum;
}

__global__ __launch_bounds__(kRatioThreads) void answer_ratio_kernel(const double* __restrict__ logps, const float* __restrict__ ref, const long long* __restrict__ labels,
                                                                     int B, int S, int V, double* __restrict__ ratios) {
    __shared__ double lds[kRatioThreads / 64];
    for (int b = blockIdx.x; b < B; b += gridDim.x) {
        const long base = (long)b * S;
        const double r = group_sum<kRatioThreads / 64>(ratio_share(logps + base, ref + base, labels + base, S, V, threadIdx.x, kRatioThreads), lds);
        if (threadIdx.x == 0) ratios[b] = r;
    }
}

// One workgroup: the pairs' losses, their mean, and what the gradient of the mean with respect to each answer's log-probabilities is.  SUMS: also
// the answers' log ratios, a wavefront an answer.
template <bool SUMS>
__global__ __launch_bounds__(kPairThreads) void preference_pairs_kernel(const double* __restrict__ logps, const float* __restrict__ ref, const long long* __restrict__ labels,
                                                                        int P, int S, int V, double beta, double smoothing, double* ratios, float* __restrict__ loss,
                                                                        float* __restrict__ rewards, float* __restrict__ coef) {
    __shared__ double lds[kPairThreads / 64];
    if constexpr (SUMS) {
        for (int b = threadIdx.x / 64; b < 2 * P; b += kPairThreads / 64) {
            const long base = (long)b * S;
            const double r = wave_sum(ratio_share(logps + base, ref + base, labels + base, S, V, threadIdx.x % 64, 64));
            if (threadIdx.x % 64 == 0) ratios[b] = r;
        }
        __syncthreads();
    }
    double sum = 0.0;
    for (int p = threadIdx.x; p < P; p += kPairThreads) {
        const double good = ratios[p], bad = ratios[p + P], z = beta * (good - bad);
        const double e = exp(-fabs(z)), soft = log1p(e), sure = 1.0 / (1.0 + e);
        const double pos = z >= 0.0 ? sure : e * sure, neg = z >= 0.0 ? e * sure : sure;      // sigmoid(z), sigmoid(-z)
        double one = (1.0 - smoothing) * (soft + fmax(-z, 0.0));
        if (smoothing > 0.0) one += smoothing * (soft + fmax(z, 0.0));       // z may be infinite
        const double dz = (smoothing * pos - (1.0 - smoothing) * neg) * (beta / P);
        rewards[p] = (float)(beta * good);
        rewards[p + P] = (float)(beta * bad);
        coef[p] = (float)dz;
        coef[p + P] = (float)-dz;
        sum += one;
    }
    sum = group_sum<kPairThreads / 64>(sum, lds);
    if (threadIdx.x == 0) *loss = (float)(sum / P);
}

constexpr long kMostGroups = 1 << 20;                                        // workgroups of a launch; they go on to further rows

template <typename F>
int by_type(int type, F&& launch) {
    switch (type) {
        case Q4_TYPE_F16: launch((half_t)0.f); break;
        case Q4_TYPE_BF16: launch((__bf16)0.f); break;
        default: launch(0.f); break;
    }
    return hipGetLastError() == hipSuccess ? 0 : -4;
}

}  // namespace q4

// Threads of a row's workgroup, by the bytes of a row and, forward, how many rows there are (with those that have no label, for labels are device memory).  us, fp16:
//   64 / 256 threads (a wavefront by itself, or four), up to 4 KB a row.  32768 rows of 2, 4, 8 KB: forward 24 / 62, 31 / 67, 52 / 91, backward 26 / 52, 47 / 64,
//     94 / 92; 2048 rows of 4 KB 5.1 / 6.5 and 5.5 / 6.4; 256 rows the same.  Forward a wavefront would win beyond 4 KB, where this does not take it.
//   forward 256 / 512, beyond 512 rows of less than 192 KB.  64 KB a row: 37 rows 5.5 / 5.2, 256 7.4 / 6.6, 512 9.4 / 9.3, 768 13.5 / 13.6, 1024 17.1 / 18.2,
//     2048 27.4 / 28.1, 32768 of which 0.55 are tokens 190 / 218; 2048 rows of 16 KB 10.2 / 12.1.  1024 and 4096 rows of 128 KB 28.4 / 29.5 and 97 / 93, of 192 KB 40.1 / 41.3
//     and 144 / 136, of 256 KB 51 / 54 and 186 / 179.  256 with eight loads a thread on their way (four: 198 for 190); 1024 threads wait for each other (415).
//   backward, where nothing waits, 256 / 1024 past the caches / 1024 through them, up to 48 KB.  16384 rows of 32 KB 189 / 215 / 216, of 48 KB 296 / 263 / 268, of 64 KB 402 /
//     331 / 339; 1024 rows of 48 KB 21.8 / 20.3 / 22.8, 37 of 64 KB 6.2 / 5.0 / 5.0.  With a kernel behind it that reads the gradient: 1024 rows of 48 KB 35.2 / 37.6 / 36.6,
//     of 64 KB 46.9 / 47.0 / 45.2, 16384 rows of 64 KB 741 / 671 / 677.
namespace {
template <typename F>
void by_width(bool forward, long rows, long bytes, F&& launch) {
    const dim3 grid((unsigned)(rows < q4::kMostGroups ? rows : q4::kMostGroups));
    if (bytes <= 4096) launch(std::integral_constant<int, 64>{}, grid);
    else if (forward && (rows <= 512 || bytes >= 192 * 1024)) launch(std::integral_constant<int, 512>{}, grid);
    else if (!forward && bytes >= 48 * 1024) launch(std::integral_constant<int, 1024>{}, grid);
    else launch(std::integral_constant<int, 256>{}, grid);
}
}  // namespace

int q4_launch_token_logps(const q4::LogitsView& a, int type, const long long* labels, float* logps, double* wide, float* stats, hipStream_t stream) {
    using namespace q4;
    return by_type(type, [&](auto t) {
        using T = decltype(t);
        by_width(true, (long)a.B * a.S, (long)a.V * sizeof(T), [&](auto threads, dim3 grid) {
            constexpr int TH = decltype(threads)::value;
            if constexpr (TH < 1024)
                hipLaunchKernelGGL((token_logps_kernel<T, TH>), grid, dim3(TH), 0, stream, a, labels, logps, wide, (float2*)stats);
        });
    });
}

int q4_launch_token_logps_bwd(const q4::LogitsView& a, int type, const long long* labels, const float* stats, const float* coef, int per, const float* factor,
                              void* dx, hipStream_t stream) {
    using namespace q4;
    return by_type(type, [&](auto t) {
        using T = decltype(t);
        by_width(false, (long)a.B * a.S, (long)a.V * sizeof(T), [&](auto threads, dim3 grid) {
            constexpr int TH = decltype(threads)::value;
            if constexpr (TH != 512)
                hipLaunchKernelGGL((token_logps_bwd_kernel<T, TH>), grid, dim3(TH), 0, stream, a, labels, (const float2*)stats, coef, per, factor, (T*)dx);
        });
    });
}

int q4_launch_preference_pairs(const double* logps, const float* ref, const long long* labels, int P, int S, int V, double beta, double smoothing, float* loss,
                               float* rewards, float* coef, double* ratios, hipStream_t stream) {
    using namespace q4;
    // One launch where a wavefront has one or two answers of 256 places to add up (us, one / two launches: 1 pair of 48 places 3.6 / 5.3, 16 of 256
    // 5.8 / 6.0, 4 of 2048 7.6 / 5.9, 16 of 1024 11.9 / 5.8).
    if ((2l * P + 15) / 16 * ((S + 255l) / 256) <= 2) {
        hipLaunchKernelGGL(preference_pairs_kernel<true>, dim3(1), dim3(kPairThreads), 0, stream, logps, ref, labels, P, S, V, beta, smoothing, ratios, loss, rewards, coef);
    } else {
        const unsigned groups = (unsigned)(2l * P < kMostGroups ? 2l * P : kMostGroups);
        hipLaunchKernelGGL(answer_ratio_kernel, dim3(groups), dim3(kRatioThreads), 0, stream, logps, ref, labels, 2 * P, S, V, ratios);
        hipLaunchKernelGGL(preference_pairs_kernel<false>, dim3(1), dim3(kPairThreads), 0, stream, logps, ref, labels, P, S, V, beta, smoothing, ratios, loss, rewards, coef);
    }
    return hipGetLastError() == hipSuccess ? 0 : -4;
}
