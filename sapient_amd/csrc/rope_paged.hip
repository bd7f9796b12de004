// rope_paged.hip — the fused bias + RoPE + KV append into a paged cache (kernel and launch shapes: rope_kv.h).
//
// What it reads and writes is sph_rope_kv_append_tokens's, and so is what bounds it: a decode step waits on its
// chain of loads (length, table entry, then the stores), a prefill step on HBM.
#include "rope_kv.h"

extern "C" int sph_rope_kv_append_paged(const void* q, void* q_out, int64_t n_q_heads, const void* k, const void* v,
                                        int64_t n_kv_heads, int dtype, int layout, const int32_t* cu_q,
                                        const int32_t* seq_lens, const int32_t* block_table, int64_t n_seqs,
                                        int64_t max_pages, int64_t n_tokens, int64_t head_dim, float base,
                                        float pos_scale, void* kcache, void* vcache, int cache_dtype, int64_t n_pages,
                                        int64_t page_size, const void* bq, const void* bk, const void* bv,
                                        int bias_dtype, int32_t* bad_page_flag, void* stream) {
    using namespace sph;
    if (layout != SPH_ROPE_NEOX && layout != SPH_ROPE_INTERLEAVED) return SPH_EINVAL;
    if (!is_float_dtype(dtype) || !is_float_dtype(cache_dtype)) return SPH_EINVAL;
    if ((bq || bk || bv) && !is_float_dtype(bias_dtype)) return SPH_EINVAL;
    if (!(bq || bk || bv)) bias_dtype = SPH_F32;
    if (n_q_heads < 0 || n_kv_heads < 1 || n_q_heads + n_kv_heads > INT32_MAX) return SPH_EINVAL;
    if (head_dim <= 0 || head_dim % 2 != 0 || head_dim / 2 > kMaxHalf) return SPH_EINVAL;
    if (!paged_ok(seq_lens, block_table, n_seqs, max_pages, n_pages, page_size, n_kv_heads, n_tokens)) return SPH_EINVAL;
    if (cu_q == nullptr && n_tokens != n_seqs) return SPH_EINVAL;  // one row per sequence
    if (!aligned(cu_q, 4)) return SPH_EINVAL;
    if (!(pos_scale == pos_scale) || pos_scale == 0.0f) return SPH_EINVAL;
    if (n_tokens == 0 || n_seqs == 0) return SPH_OK;
    if (k == nullptr || v == nullptr || kcache == nullptr || vcache == nullptr) return SPH_EINVAL;
    if (n_q_heads > 0) {
        // A thread reads the channels that it writes, so q_out may be q itself, but may not overlap it otherwise.
        if (q == nullptr || q_out == nullptr) return SPH_EINVAL;
        const uintptr_t bytes = (uintptr_t)n_q_heads * (uintptr_t)n_tokens * (uintptr_t)head_dim * dtype_size(dtype);
        const uintptr_t a = (uintptr_t)q, b = (uintptr_t)q_out;
        if (a != b && a < b + bytes && b < a + bytes) return SPH_EINVAL;
    }
    hipStream_t s = static_cast<hipStream_t>(stream);
    return with_float_type(dtype, [&](auto t) -> int {
        using T = decltype(t);
        return with_float_type(cache_dtype, [&](auto tc) -> int {
            using TC = decltype(tc);
            RopeKvPagedArgs<T, TC> a{};
            a.q = static_cast<const T*>(q);
            a.qo = static_cast<T*>(q_out);
            a.k = static_cast<const T*>(k);
            a.v = static_cast<const T*>(v);
            a.kc = static_cast<TC*>(kcache);
            a.vc = static_cast<TC*>(vcache);
            a.bias[0] = bq;
            a.bias[1] = bk;
            a.bias[2] = bv;
            a.bias_dt = bias_dtype;
            a.nq = (int)n_q_heads;
            a.nkv = (int)n_kv_heads;
            a.seq = n_tokens;
            a.head_dim = (int)head_dim;
            a.pos_scale = pos_scale;
            a.bad = bad_page_flag;
            a.pages = paged_table(seq_lens, cu_q, block_table, n_seqs, max_pages, n_pages, page_size, n_kv_heads);
            return launch_rope_kv<true>(a, layout, base, s);
        });
    });
}
