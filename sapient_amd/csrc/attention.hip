// attention.hip — entry points of attention over the paged KV cache (kernels and their mathematics: attention.h).
#include "attention.h"

#include <math.h>

namespace sph {

int attn_args(AttnArgs& a, const void* q, void* out, int64_t n_q_heads, int64_t n_kv_heads, int dtype, const int32_t* cu_q,
              const int32_t* seq_lens, const int32_t* block_table, int64_t n_seqs, int64_t max_pages, int64_t n_rows,
              int64_t head_dim, const void* kcache, const void* vcache, int cache_dtype, int64_t n_pages,
              int64_t page_size, float scale, float softcap, int64_t window, const float* slopes,
              const int32_t* prefix_lens, int32_t* bad) {
    if (!is_float_dtype(dtype) || !is_float_dtype(cache_dtype)) return SPH_EINVAL;
    if (!paged_ok(seq_lens, block_table, n_seqs, max_pages, n_pages, page_size, n_kv_heads, n_rows)) return SPH_EINVAL;
    if (n_q_heads < 1 || n_q_heads > INT32_MAX || n_q_heads % n_kv_heads != 0) return SPH_EINVAL;
    if (head_dim <= 0 || head_dim % 8 != 0 || head_dim > 256) return SPH_EINVAL;
    if (n_rows * (n_q_heads / n_kv_heads) > INT32_MAX) return SPH_EINVAL;
    if (!isfinite(scale) || !isfinite(softcap) || softcap < 0.0f || window < 0) return SPH_EINVAL;
    if (!aligned(cu_q, 4) || !aligned(slopes, 4) || !aligned(prefix_lens, 4)) return SPH_EINVAL;
    if (!aligned(q, 16) || !aligned(out, 16) || !aligned(kcache, 16) || !aligned(vcache, 16)) return SPH_EINVAL;
    if (n_rows > 0 && n_seqs > 0 && (q == nullptr || out == nullptr || kcache == nullptr || vcache == nullptr)) return SPH_EINVAL;
    a.q = q;
    a.out = out;
    a.kc = kcache;
    a.vc = vcache;
    a.pages = paged_table(seq_lens, cu_q, block_table, n_seqs, max_pages, n_pages, page_size, n_kv_heads);
    a.slopes = slopes;
    a.prefix = prefix_lens;
    a.bad = bad;
    a.dtype = dtype;
    a.n_rows = (int)n_rows;
    a.nq = (int)n_q_heads;
    a.group = (int)(n_q_heads / n_kv_heads);
    a.head_dim = (int)head_dim;
    a.window = window > INT32_MAX ? 0 : (int)window;  // no position is that far
    a.scale = scale;
    a.cap = softcap;
    return SPH_OK;
}

namespace {

template <typename TC, bool HIGH>
int launch_tiles(const AttnArgs& a, int64_t blocks, int tiles_per_seq, hipStream_t s) {
    if (blocks * kAttnThreads > UINT32_MAX) return SPH_EINVAL;
    return with_tile_kernel<TC, HIGH>(a.head_dim, [&](auto k) {
        return launch(paged_tiles_kernel<decltype(k)>, dim3((unsigned)blocks), kAttnThreads, s, a, tiles_per_seq);
    });
}

int dispatch_tiles(const AttnArgs& a, int cache_dtype, int64_t blocks, int tiles_per_seq, hipStream_t s) {
    return with_float_type(cache_dtype, [&](auto tc) -> int {
        using TC = decltype(tc);
        if constexpr (!__is_same(TC, float)) {
            if (a.dtype == cache_dtype) return launch_tiles<TC, false>(a, blocks, tiles_per_seq, s);
        }
        return launch_tiles<TC, true>(a, blocks, tiles_per_seq, s);
    });
}

// Shares of a call's single tokens: as many blocks as the GPU holds at once, or the most units there can be.
struct SplitPlan {
    int tiles, cols, shares;
    int64_t bytes;
};
SplitPlan split_plan(int64_t nq, int64_t nkv, int64_t n_seqs, int64_t max_pages, int64_t page_size, int64_t head_dim) {
    SplitPlan p;
    const int64_t group = nq / nkv;
    const int64_t tiles = (group + 15) / 16 * nkv;
    const int64_t steps = max_pages * page_size / 64 + 1;  // the smaller of the kernels' steps
    int64_t shares = 256 * (head_dim > 128 ? 1 : 2);
    if ((__int128)n_seqs * tiles * steps < shares) shares = n_seqs * tiles * steps;
    p.tiles = (int)tiles;
    p.cols = (int)(group < 16 ? group : 16);
    p.shares = (int)shares;
    p.bytes = 2 * shares * p.cols * (head_dim + 2) * 4;
    return p;
}

template <typename TC, bool HIGH>
int launch_split(const AttnArgs& a, const SplitPlan& p, float* ws, hipStream_t s) {
    return with_tile_kernel<TC, HIGH>(a.head_dim, [&](auto k) {
        using K = decltype(k);
        const SplitArgs sp{p.tiles, p.cols, p.shares, ws};
        const int st = launch(paged_split_kernel<K>, dim3((unsigned)p.shares), kAttnThreads, s, a, sp);
        if (st != SPH_OK) return st;
        return launch(paged_join_kernel<K::kStep>, dim3((unsigned)(a.pages.n_seqs * p.tiles)), kAttnThreads, s, a, sp);
    });
}

int dispatch_split(const AttnArgs& a, int cache_dtype, const SplitPlan& p, float* ws, hipStream_t s) {
    return with_float_type(cache_dtype, [&](auto tc) -> int {
        using TC = decltype(tc);
        if constexpr (!__is_same(TC, float)) {
            if (a.dtype == cache_dtype) return launch_split<TC, false>(a, p, ws, s);
        }
        return launch_split<TC, true>(a, p, ws, s);
    });
}

}  // namespace
}  // namespace sph

extern "C" int sph_paged_attention(const void* q, void* out, int64_t n_q_heads, int64_t n_kv_heads, int dtype,
                                   const int32_t* seq_lens, const int32_t* block_table, int64_t n_seqs, int64_t max_pages,
                                   int64_t head_dim, const void* kcache, const void* vcache, int cache_dtype,
                                   int64_t n_pages, int64_t page_size, float scale, float softcap, int64_t window,
                                   const float* slopes, void* workspace, int64_t workspace_bytes, int32_t* bad_page_flag,
                                   void* stream) {
    using namespace sph;
    AttnArgs a{};
    const int st = attn_args(a, q, out, n_q_heads, n_kv_heads, dtype, nullptr, seq_lens, block_table, n_seqs, max_pages, n_seqs,
                             head_dim, kcache, vcache, cache_dtype, n_pages, page_size, scale, softcap, window, slopes,
                             nullptr, bad_page_flag);
    if (st != SPH_OK) return st;
    if (n_seqs == 0) return SPH_OK;
    const SplitPlan p = split_plan(n_q_heads, n_kv_heads, n_seqs, max_pages, page_size, head_dim);
    if (n_seqs * (int64_t)p.tiles * kAttnThreads > UINT32_MAX) return SPH_EINVAL;
    if (workspace == nullptr || !aligned(workspace, 16) || workspace_bytes < p.bytes) return SPH_EINVAL;
    return dispatch_split(a, cache_dtype, p, static_cast<float*>(workspace), static_cast<hipStream_t>(stream));
}

extern "C" int sph_paged_attention_chunk(const void* q, void* out, int64_t n_q_heads, int64_t n_kv_heads, int dtype,
                                         const int32_t* cu_q, const int32_t* seq_lens, const int32_t* block_table,
                                         int64_t n_seqs, int64_t max_pages, int64_t n_tokens, int64_t head_dim,
                                         const void* kcache, const void* vcache, int cache_dtype, int64_t n_pages,
                                         int64_t page_size, float scale, float softcap, int64_t window,
                                         const float* slopes, const int32_t* prefix_lens, void* workspace,
                                         int64_t workspace_bytes, int32_t* bad_page_flag, void* stream) {
    using namespace sph;
    AttnArgs a{};
    const int st = attn_args(a, q, out, n_q_heads, n_kv_heads, dtype, cu_q, seq_lens, block_table, n_seqs, max_pages, n_tokens,
                             head_dim, kcache, vcache, cache_dtype, n_pages, page_size, scale, softcap, window, slopes,
                             prefix_lens, bad_page_flag);
    if (st != SPH_OK) return st;
    if (n_seqs == 0 || n_tokens == 0) return SPH_OK;
    if (cu_q == nullptr) return SPH_EINVAL;
    const uintptr_t bytes = (uintptr_t)n_q_heads * (uintptr_t)n_tokens * (uintptr_t)head_dim * dtype_size(dtype);
    const uintptr_t x = (uintptr_t)q, y = (uintptr_t)out;
    if (x < y + bytes && y < x + bytes) return SPH_EINVAL;  // a row's columns are read by one block and written by another
    // Every sequence's tiles end in at most one that is not full.
    const int64_t tiles = n_tokens * a.group / 16 + n_seqs;
    return dispatch_tiles(a, cache_dtype, tiles * n_kv_heads, 1, static_cast<hipStream_t>(stream));
}

extern "C" int64_t sph_paged_attention_workspace(int64_t n_q_heads, int64_t n_kv_heads, int64_t n_seqs, int64_t max_pages,
                                                 int64_t page_size, int64_t head_dim) {
    if (n_kv_heads < 1 || n_q_heads < 1 || n_q_heads % n_kv_heads != 0 || n_seqs < 0 || max_pages < 0 || page_size < 1 ||
        head_dim < 1 || head_dim > 256)
        return SPH_EINVAL;
    return sph::split_plan(n_q_heads, n_kv_heads, n_seqs, max_pages, page_size, head_dim).bytes;
}

extern "C" int64_t sph_paged_attention_chunk_workspace(int64_t n_q_heads, int64_t n_kv_heads, int64_t n_seqs,
                                                       int64_t max_pages, int64_t page_size, int64_t n_tokens,
                                                       int64_t head_dim) {
    return 0;
}
