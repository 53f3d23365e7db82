// Launches of the preference loss's kernels (q4_preference.hip).
#pragma once
#include <hip/hip_runtime.h>
#include <type_traits>

namespace q4 {
// Logits [B, S, V] with strides in elements, a row's V values side by side.
struct LogitsView {
    const void* x;
    long sb, st;
    int B, S, V;
};
}  // namespace q4

int q4_launch_token_logps(const q4::LogitsView& a, int type, const long long* labels, float* logps, double* wide, float* stats, hipStream_t stream);
int q4_launch_token_logps_bwd(const q4::LogitsView& a, int type, const long long* labels, const float* stats, const float* coef, int per, const float* factor,
                              void* dx, hipStream_t stream);
int q4_launch_preference_pairs(const double* logps, const float* ref, const long long* labels, int P, int S, int V, double beta, double smoothing, float* loss,
                               float* rewards, float* coef, double* ratios, hipStream_t stream);
