// C ABI of the serving operators (declared in include/q4_gptq.h): argument validation + kernel launches.
// No torch types, no allocation, no synchronisation.
#include "q4_gptq.h"
#include "q4_kv4.hpp"

size_t q4_lora_rows_workspace(int M, int K, int R, int probs);
int q4_launch_lora_rows(const q4_lora_rows_t*, int, const void*, const int32_t*, int, int, int, int, int, void*, hipStream_t);

namespace {
inline bool misaligned(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) != 0; }

int check_cache(const q4_kv4_cache_t* c, const q4_kv4_batch_t* b) {
    if (!c || !b || !c->k_codes || !c->v_codes || !c->k_scales || !c->v_scales || !b->table || !b->lengths) return Q4_ERR_NULL_POINTER;
    if ((c->D != 64 && c->D != 128) || (c->group != 32 && c->group != 64 && c->group != 128) || c->group > c->D) return Q4_ERR_BAD_SHAPE;
    if (c->page < 16 || c->page > 1024 || c->page % 16 != 0 || c->pages < 1 || c->heads < 1 || c->heads > 4096) return Q4_ERR_BAD_SHAPE;
    // places are counted in units of 16 tokens of one head and group, in 31 bits
    if ((double)c->pages * c->heads * (c->page / 16) * (c->D / c->group) >= 2147483648.0) return Q4_ERR_BAD_SHAPE;
    if (b->width < 1 || (long long)b->width * c->page > (1ll << 26) || b->B < 1 || b->T < 1) return Q4_ERR_BAD_SHAPE;
    if (b->T > (1 << 24) || (!b->starts && b->T % b->B != 0)) return Q4_ERR_BAD_SHAPE;
    if (misaligned(c->k_codes) || misaligned(c->v_codes) || misaligned(c->k_scales) || misaligned(c->v_scales)) return Q4_ERR_MISALIGNED;
    return Q4_OK;
}

q4::Kv4Cache cache_of(const q4_kv4_cache_t* c) {
    return {reinterpret_cast<uint32_t*>(c->k_codes), reinterpret_cast<uint32_t*>(c->v_codes), reinterpret_cast<q4::half_t*>(c->k_scales),
            reinterpret_cast<q4::half_t*>(c->v_scales), c->pages, c->page, c->heads};
}
q4::Kv4Batch batch_of(const q4_kv4_batch_t* b) { return {b->table, b->lengths, b->starts, b->width, b->B, b->T}; }

bool heads_fit(const q4_kv4_cache_t* c, const q4_kv4_batch_t* b, int q_heads) {
    return q_heads >= 1 && q_heads % c->heads == 0 && q_heads <= 65536 && (double)b->T * q_heads < 2147483648.0;
}
bool launch_fits(const q4_kv4_cache_t* c, const q4_kv4_batch_t* b, int q_heads, int max_tokens, int max_length) {
    if (!heads_fit(c, b, q_heads) || max_tokens < 1 || max_length < 1) return false;
    return (double)b->B * c->heads <= 4194304.0;                           // workgroups of one block of rows each, 2^32 threads a launch
}
bool strides_fit(long long t, long long h) { return t >= 0 && h >= 0 && t < (1ll << 40) && h < (1ll << 40); }
bool vectors(const void* p, long long t, long long h) { return !misaligned(p) && t % 8 == 0 && h % 8 == 0; }
}  // namespace

extern "C" int q4_kv4_append_f16(const q4_kv4_cache_t* cache, const q4_kv4_batch_t* batch, const void* k, long long k_t, long long k_h,
                                 const void* v, long long v_t, long long v_h, const void* q, long long q_t, long long q_h, void* q_out,
                                 int q_heads, const float* rope, int rope_rows, int rot, int interleaved, void* stream) {
    const int rc = check_cache(cache, batch);
    if (rc != Q4_OK) return rc;
    if (!k || !v || (q && !q_out) || (rot && !rope)) return Q4_ERR_NULL_POINTER;
    if (q && !heads_fit(cache, batch, q_heads)) return Q4_ERR_BAD_SHAPE;
    if (rot < 0 || rot > cache->D || rot % 16 != 0 || (rot && rope_rows < 1)) return Q4_ERR_BAD_SHAPE;
    if (!strides_fit(k_t, k_h) || !strides_fit(v_t, v_h) || (q && !strides_fit(q_t, q_h))) return Q4_ERR_BAD_SHAPE;
    if ((rot && misaligned(rope)) || (q && misaligned(q_out))) return Q4_ERR_MISALIGNED;
    q4::Kv4Append a{cache_of(cache), batch_of(batch), reinterpret_cast<const q4::half_t*>(k), reinterpret_cast<const q4::half_t*>(v),
                    reinterpret_cast<const q4::half_t*>(q), reinterpret_cast<q4::half_t*>(q_out), (long)k_t, (long)k_h, (long)v_t, (long)v_h,
                    (long)q_t, (long)q_h, rope, rope_rows, rot, interleaved != 0, q ? q_heads : 0};
    const bool vec = vectors(k, k_t, k_h) && (!q || vectors(q, q_t, q_h));
    return q4_launch_kv4_append(a, cache->D, cache->group, vec, (hipStream_t)stream);
}

extern "C" int q4_kv4_read_f16(const q4_kv4_cache_t* cache, const q4_kv4_batch_t* batch, void* k, void* v, void* stream) {
    const int rc = check_cache(cache, batch);
    if (rc != Q4_OK) return rc;
    if (!k || !v) return Q4_ERR_NULL_POINTER;
    if (misaligned(k) || misaligned(v)) return Q4_ERR_MISALIGNED;
    return q4_launch_kv4_read({cache_of(cache), batch_of(batch), reinterpret_cast<q4::half_t*>(k), reinterpret_cast<q4::half_t*>(v)}, cache->D,
                              cache->group, (hipStream_t)stream);
}

extern "C" size_t q4_kv4_attention_workspace_bytes(const q4_kv4_cache_t* cache, const q4_kv4_batch_t* batch, int q_heads, int max_tokens,
                                                   int max_length) {
    if (check_cache(cache, batch) != Q4_OK || !launch_fits(cache, batch, q_heads, max_tokens, max_length)) return 0;
    return q4_kv4_attn_workspace(batch->B, cache->heads, cache->D, q_heads / cache->heads, batch->T, max_tokens, max_length);
}

extern "C" int q4_kv4_attention_f16(const q4_kv4_cache_t* cache, const q4_kv4_batch_t* batch, const void* q, long long q_t, long long q_h,
                                    int q_heads, float scale, void* out, int max_tokens, int max_length, void* workspace,
                                    size_t workspace_bytes, void* stream) {
    const int rc = check_cache(cache, batch);
    if (rc != Q4_OK) return rc;
    if (!q || !out) return Q4_ERR_NULL_POINTER;
    if (!launch_fits(cache, batch, q_heads, max_tokens, max_length) || !strides_fit(q_t, q_h)) return Q4_ERR_BAD_SHAPE;
    if (!(scale > 0.0f) || !(scale < 1e37f)) return Q4_ERR_BAD_SHAPE;       // times 8 * log2(e) it is finite
    if (!vectors(q, q_t, q_h) || misaligned(out)) return Q4_ERR_MISALIGNED;
    const size_t need = q4_kv4_attention_workspace_bytes(cache, batch, q_heads, max_tokens, max_length);
    if (need && (!workspace || workspace_bytes < need)) return Q4_ERR_WORKSPACE;
    if (need && (reinterpret_cast<uintptr_t>(workspace) & 255u) != 0) return Q4_ERR_MISALIGNED;
    q4::Kv4Attn a{cache_of(cache), batch_of(batch), reinterpret_cast<const q4::half_t*>(q), (long)q_t, (long)q_h,
                  reinterpret_cast<q4::half_t*>(out), reinterpret_cast<float*>(workspace), scale * 1.4426950408889634f, 0.f, q_heads,
                  q_heads / cache->heads, 1, 1, 0u};
    return q4_launch_kv4_attn(a, cache->D, cache->group, max_tokens, max_length, (hipStream_t)stream);
}

static bool lora_rows_shape(int count, int M, int K, int R) {
    return count >= 1 && count <= 4 && M >= 1 && K >= 32 && K % 32 == 0 && R >= 8 && R <= 64 && R % 8 == 0 && K <= (1 << 20) && M <= (1 << 24);
}

extern "C" size_t q4_lora_rows_workspace_bytes(int count, int M, int K, int R) {
    return lora_rows_shape(count, M, K, R) ? q4_lora_rows_workspace(M, K, R, count) : 0;
}

extern "C" int q4_lora_rows_f16(const q4_lora_rows_t* probs, int count, const void* x, const int32_t* index, int per, int M, int K, int R,
                                int n, void* workspace, size_t workspace_bytes, void* stream) {
    if (!probs || !x || !index) return Q4_ERR_NULL_POINTER;
    if (!lora_rows_shape(count, M, K, R) || per < 1 || n < 1) return Q4_ERR_BAD_SHAPE;
    if (misaligned(x)) return Q4_ERR_MISALIGNED;
    for (int i = 0; i < count; ++i) {
        const q4_lora_rows_t& g = probs[i];
        if (!g.a || !g.b || !g.scaling || !g.y) return Q4_ERR_NULL_POINTER;
        if (g.N < 64 || g.N % 64 != 0 || g.N > (1 << 23)) return Q4_ERR_BAD_SHAPE;
        if (((M + 31ll) / 32) * ((g.N + 255) / 256) >= (1 << 24)) return Q4_ERR_BAD_SHAPE;      /* 2^32 threads a launch */
        if (misaligned(g.a) || misaligned(g.b) || misaligned(g.y)) return Q4_ERR_MISALIGNED;
    }
    if (!workspace || workspace_bytes < q4_lora_rows_workspace_bytes(count, M, K, R)) return Q4_ERR_WORKSPACE;
    if ((reinterpret_cast<uintptr_t>(workspace) & 255u) != 0) return Q4_ERR_MISALIGNED;
    return q4_launch_lora_rows(probs, count, x, index, per, M, K, R, n, workspace, (hipStream_t)stream);
}
