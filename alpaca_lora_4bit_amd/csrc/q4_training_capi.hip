// C ABI of the 8-bit activations and the preference loss (declared in include/q4_gptq.h): argument validation + kernel launches.
// No torch types, no allocation, no synchronisation.
#include <hip/hip_runtime.h>
#include <math.h>
#include <stdint.h>
#include "q4_gptq.h"
#include "q4_preference.hpp"

int q4_launch_act8_pack(const void*, int, void*, void*, long, hipStream_t);
int q4_launch_act8_unpack(const void*, const void*, void*, int, long, hipStream_t);
int q4_launch_silu_mul_act8(const void*, const void*, int, void*, const q4_act8_t*, const q4_act8_t*, long, hipStream_t);
int q4_launch_silu_mul_act8_bwd(const void*, int, const q4_act8_t*, const q4_act8_t*, void*, void*, long, hipStream_t);

namespace {
inline bool misaligned(const void* p, uintptr_t to = 16) { return (reinterpret_cast<uintptr_t>(p) & (to - 1)) != 0; }
inline bool fits(long long n) { return n >= 1 && n < (1ll << 35) - 2048; }        // 2^32 threads a launch, 8 values each
inline bool known(int type) { return type == Q4_TYPE_F16 || type == Q4_TYPE_BF16 || type == Q4_TYPE_F32; }
inline int size_of(int type) { return type == Q4_TYPE_F32 ? 4 : 2; }

int check_kept(const q4_act8_t* a) {
    if (!a || !a->codes || !a->scales) return Q4_ERR_NULL_POINTER;
    return misaligned(a->codes) || misaligned(a->scales) ? Q4_ERR_MISALIGNED : Q4_OK;
}

int check_logits(const void* logits, int type, long long sb, long long st, int B, int S, int V, const long long* labels) {
    if (!logits || !labels) return Q4_ERR_NULL_POINTER;
    if (!known(type) || B < 1 || S < 1 || V < 1 || V >= (1 << 30) || (double)B * S > 2147483647.0) return Q4_ERR_BAD_SHAPE;
    if (sb < 0 || st < 0 || sb > (1ll << 50) || st > (1ll << 50)) return Q4_ERR_BAD_SHAPE;
    return misaligned(logits, size_of(type)) || misaligned(labels, 8) ? Q4_ERR_MISALIGNED : Q4_OK;
}
}  // namespace

extern "C" int q4_act8_pack(const void* x, int type, void* codes, void* scales, long long n, void* stream) {
    if (!x || !codes || !scales) return Q4_ERR_NULL_POINTER;
    if (!known(type) || !fits(n)) return Q4_ERR_BAD_SHAPE;
    if (misaligned(x) || misaligned(codes) || misaligned(scales)) return Q4_ERR_MISALIGNED;
    return q4_launch_act8_pack(x, type, codes, scales, (long)n, (hipStream_t)stream);
}

extern "C" int q4_act8_unpack(const void* codes, const void* scales, void* x, int type, long long n, void* stream) {
    if (!x || !codes || !scales) return Q4_ERR_NULL_POINTER;
    if (!known(type) || !fits(n)) return Q4_ERR_BAD_SHAPE;
    if (misaligned(x) || misaligned(codes) || misaligned(scales)) return Q4_ERR_MISALIGNED;
    return q4_launch_act8_unpack(codes, scales, x, type, (long)n, (hipStream_t)stream);
}

extern "C" int q4_silu_mul_act8(const void* gate, const void* up, int type, void* out, const q4_act8_t* kept_gate, const q4_act8_t* kept_up, long long n,
                                void* stream) {
    if (!gate || !up || !out) return Q4_ERR_NULL_POINTER;
    if ((type != Q4_TYPE_F16 && type != Q4_TYPE_BF16) || !fits(n)) return Q4_ERR_BAD_SHAPE;
    if (misaligned(gate) || misaligned(up) || misaligned(out)) return Q4_ERR_MISALIGNED;
    if (!kept_gate && !kept_up) return q4_launch_silu_mul_act8(gate, up, type, out, nullptr, nullptr, (long)n, (hipStream_t)stream);
    int rc = check_kept(kept_gate);
    if (rc == Q4_OK) rc = check_kept(kept_up);
    return rc != Q4_OK ? rc : q4_launch_silu_mul_act8(gate, up, type, out, kept_gate, kept_up, (long)n, (hipStream_t)stream);
}

extern "C" int q4_silu_mul_act8_bwd(const void* dout, int type, const q4_act8_t* kept_gate, const q4_act8_t* kept_up, void* dgate, void* dup, long long n,
                                    void* stream) {
    if (!dout || !dgate || !dup) return Q4_ERR_NULL_POINTER;
    if ((type != Q4_TYPE_F16 && type != Q4_TYPE_BF16) || !fits(n)) return Q4_ERR_BAD_SHAPE;
    if (misaligned(dout) || misaligned(dgate) || misaligned(dup)) return Q4_ERR_MISALIGNED;
    int rc = check_kept(kept_gate);
    if (rc == Q4_OK) rc = check_kept(kept_up);
    return rc != Q4_OK ? rc : q4_launch_silu_mul_act8_bwd(dout, type, kept_gate, kept_up, dgate, dup, (long)n, (hipStream_t)stream);
}

extern "C" int q4_token_logps(const void* logits, int type, long long sb, long long st, int B, int S, int V, const long long* labels, float* logps,
                              float* stats, void* stream) {
    if (!logps || !stats) return Q4_ERR_NULL_POINTER;
    const int rc = check_logits(logits, type, sb, st, B, S, V, labels);
    if (rc != Q4_OK) return rc;
    if (misaligned(logps, 4) || misaligned(stats, 8)) return Q4_ERR_MISALIGNED;
    return q4_launch_token_logps({logits, (long)sb, (long)st, B, S, V}, type, labels, logps, nullptr, stats, (hipStream_t)stream);
}

extern "C" int q4_token_logps_bwd(const void* logits, int type, long long sb, long long st, int B, int S, int V, const long long* labels, const float* stats,
                                  const float* coef, int per, const float* factor, void* dlogits, void* stream) {
    if (!stats || !coef || !dlogits) return Q4_ERR_NULL_POINTER;
    const int rc = check_logits(logits, type, sb, st, B, S, V, labels);
    if (rc != Q4_OK) return rc;
    if (per < 1 || ((long long)B * S) % per != 0) return Q4_ERR_BAD_SHAPE;
    if (misaligned(stats, 8) || misaligned(coef, 4) || (factor && misaligned(factor, 4)) || misaligned(dlogits)) return Q4_ERR_MISALIGNED;
    return q4_launch_token_logps_bwd({logits, (long)sb, (long)st, B, S, V}, type, labels, stats, coef, per, factor, dlogits, (hipStream_t)stream);
}

extern "C" size_t q4_preference_loss_workspace_bytes(int P, int S) {
    return P < 1 || S < 1 || 2.0 * P * S > 2147483647.0 ? 0 : 16 * ((size_t)P + (size_t)P * S);
}

extern "C" int q4_preference_loss(const void* logits, int type, long long sb, long long st, int P, int S, int V, const long long* labels, const float* ref,
                                  double beta, double smoothing, float* loss, float* rewards, float* coef, float* stats, void* workspace,
                                  size_t workspace_bytes, void* stream) {
    if (!ref || !loss || !rewards || !coef || !stats) return Q4_ERR_NULL_POINTER;
    if (P < 1 || P > (1 << 29)) return Q4_ERR_BAD_SHAPE;
    int rc = check_logits(logits, type, sb, st, 2 * P, S, V, labels);
    if (rc != Q4_OK) return rc;
    if (!(beta > 0.0) || !isfinite(beta) || !(smoothing >= 0.0) || !(smoothing <= 0.5)) return Q4_ERR_BAD_SHAPE;
    if (!workspace || workspace_bytes < q4_preference_loss_workspace_bytes(P, S)) return Q4_ERR_WORKSPACE;
    if (misaligned(ref, 4) || misaligned(loss, 4) || misaligned(rewards, 4) || misaligned(coef, 4) || misaligned(stats, 8) || misaligned(workspace, 8))
        return Q4_ERR_MISALIGNED;
    double* ratios = reinterpret_cast<double*>(workspace);
    double* logps = ratios + 2 * (size_t)P;
    rc = q4_launch_token_logps({logits, (long)sb, (long)st, 2 * P, S, V}, type, labels, nullptr, logps, stats, (hipStream_t)stream);
    return rc != Q4_OK ? rc : q4_launch_preference_pairs(logps, ref, labels, P, S, V, beta, smoothing, loss, rewards, coef, ratios, (hipStream_t)stream);
}
