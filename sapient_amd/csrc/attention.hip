// attention.hip — entry points of attention over the paged KV cache (kernels and their mathematics: attention.h).
#include "attention.h"

#include <math.h>

namespace sph {
namespace {

// Sizes that every count of rows, tiles and keys stays in 32 bits for.
bool sizes_ok(int64_t nq, int64_t nkv, int64_t n_seqs, int64_t max_pages, int64_t page_size, int64_t head_dim, int64_t n_rows) {
    if (nkv < 1 || nq < 1 || nq > INT32_MAX || nkv > INT32_MAX || nq % nkv != 0) return false;
    if (head_dim <= 0 || head_dim % 8 != 0 || head_dim > 256) return false;
    if (n_seqs < 0 || n_seqs > INT32_MAX || max_pages < 0 || max_pages > INT32_MAX || page_size < 1 || page_size > INT32_MAX) return false;
    return n_rows >= 0 && n_rows <= INT32_MAX && n_rows * nq <= INT32_MAX - kPromptRows;
}

}  // namespace

int attn_args(AttnArgs& a, const void* q, void* out, int64_t n_q_heads, int64_t n_kv_heads, int dtype, const int32_t* cu_q,
              const int32_t* seq_lens, const int32_t* block_table, int64_t n_seqs, int64_t max_pages, int64_t n_rows,
              int64_t head_dim, const void* kcache, const void* vcache, int cache_dtype, int64_t n_pages,
              int64_t page_size, float scale, float softcap, int64_t window, const float* slopes,
              const int32_t* prefix_lens, int32_t* bad) {
    if (!is_float_dtype(dtype) || !is_float_dtype(cache_dtype)) return SPH_EINVAL;
    if (!paged_ok(seq_lens, block_table, n_seqs, max_pages, n_pages, page_size, n_kv_heads, n_rows)) return SPH_EINVAL;
    if (!sizes_ok(n_q_heads, n_kv_heads, n_seqs, max_pages, page_size, head_dim, n_rows)) return SPH_EINVAL;
    if (!isfinite(scale) || !isfinite(softcap) || window < 0) return SPH_EINVAL;
    if (softcap != 0.0f && !(softcap >= 1e-6f)) return SPH_EINVAL;  // scale / softcap stays finite
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

// Parts of a chunk's keys, where its tiles alone are fewer than the blocks that the GPU holds: at most 16, of 256 keys or
// more were the table full, and no more than fit the workspace. (Twice the blocks, for tiles of different lengths: nine
// sequences of five tokens over up to 12000 keys 47 -> 58 us.)
struct ChunkPlan {
    int64_t tiles;  // the most there can be, of one kv head: every sequence's end in at most one that is not full
    int splits;
    int64_t bytes;
};
ChunkPlan chunk_plan(int rows_per_tile, int64_t nq, int64_t nkv, int64_t n_seqs, int64_t max_pages, int64_t page_size,
                     int64_t n_rows, int64_t head_dim, int64_t workspace_bytes) {
    ChunkPlan p;
    p.tiles = n_rows * (nq / nkv) / rows_per_tile + (n_seqs < n_rows ? n_seqs : n_rows);
    const int64_t blocks = p.tiles * nkv, slots = 256 * (head_dim > 128 ? 1 : 2), most = max_pages * page_size / 256;
    const int64_t part = n_rows * nq * (head_dim + 2) * 4;
    int64_t s = blocks > 0 ? slots / blocks : 1;
    if (s > 16) s = 16;
    if (s > most) s = most;
    if (part > 0 && s > workspace_bytes / part) s = workspace_bytes / part;
    if (s < 1) s = 1;
    p.splits = (int)s;
    p.bytes = s > 1 ? s * part : 0;
    return p;
}

// Chunks over caches of a half type take tiles of 128 rows, over f32 ones of 16.
inline int chunk_rows(bool prompt) { return prompt ? kPromptRows : 16; }

int launch_tiles(const AttnArgs& a, unsigned blocks, const ChunkSplit& sp, hipStream_t s) {
    return with_tile_kernel<float, true>(a.head_dim, [&](auto k) {
        return launch(paged_tiles_kernel<decltype(k)>, dim3(blocks), kAttnThreads, s, a, sp);
    });
}
// Shares of a call's single tokens: as many blocks as the GPU holds at once, the most units there can be, or what fits the
// workspace. Where no
// sequence can have more than 512 keys, four block steps of most types (by its table or the window), a block takes a
// sequence's tile whole, in one launch (one sequence of 333 keys 7.4 us; split 11.2).
struct SplitPlan {
    bool whole;
    int tiles, cols, shares;
    int64_t ranges, bytes;  // of the part ranges, and of all
};
SplitPlan split_plan(int64_t nq, int64_t nkv, int64_t n_seqs, int64_t max_pages, int64_t page_size, int64_t head_dim,
                     int64_t window, int64_t workspace_bytes) {
    SplitPlan p;
    const int64_t capacity = max_pages * page_size;
    const int64_t group = nq / nkv;
    const int64_t tiles = (group + 15) / 16 * nkv;
    const int64_t steps = capacity / 64 + 1;  // the smaller of the kernels' steps
    int64_t shares = 256 * (head_dim > 128 ? 1 : 2);
    if ((__int128)n_seqs * tiles * steps < shares) shares = n_seqs * tiles * steps;
    p.tiles = (int)tiles;
    p.cols = (int)(group < 16 ? group : 16);
    p.shares = (int)shares;
    p.ranges = (n_seqs * tiles * (int64_t)sizeof(PartRange) + 15) / 16 * 16;
    const int64_t part = 2 * p.cols * (head_dim + 2) * 4;
    if (p.shares > (workspace_bytes - p.ranges) / part) p.shares = (int)((workspace_bytes - p.ranges) / part);
    p.whole = capacity <= 512 || (window > 0 && window <= 512) || workspace_bytes < p.ranges + 2 * part;
    p.bytes = p.whole ? 0 : p.ranges + p.shares * part;
    return p;
}

template <typename TC, bool HIGH>
int launch_split(const AttnArgs& a, const SplitPlan& p, char* ws, hipStream_t s) {
    return with_tile_kernel<TC, HIGH>(a.head_dim, [&](auto k) {
        using K = decltype(k);
        if (p.whole) return launch(paged_whole_kernel<K>, dim3((unsigned)(a.pages.n_seqs * p.tiles)), kAttnThreads, s, a, p.tiles);
        const SplitArgs sp{p.tiles, p.cols, p.shares, reinterpret_cast<PartRange*>(ws), reinterpret_cast<float*>(ws + p.ranges)};
        const int st = launch(paged_split_kernel<K>, dim3((unsigned)p.shares), kAttnThreads, s, a, sp);
        if (st != SPH_OK) return st;
        return launch(paged_join_kernel, dim3((unsigned)a.n_rows * (unsigned)a.nq), kAttnThreads, s, a, sp);
    });
}

int dispatch_split(const AttnArgs& a, int cache_dtype, const SplitPlan& p, char* ws, hipStream_t s) {
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
    if (n_seqs * n_q_heads * kAttnThreads > UINT32_MAX) return SPH_EINVAL;
    const SplitPlan p = split_plan(n_q_heads, n_kv_heads, n_seqs, max_pages, page_size, head_dim, a.window,
                                   workspace == nullptr ? 0 : workspace_bytes);
    if (!aligned(workspace, 16)) return SPH_EINVAL;
    return dispatch_split(a, cache_dtype, p, static_cast<char*>(workspace), static_cast<hipStream_t>(stream));
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
    const bool prompt = cache_dtype != SPH_F32;
    const ChunkPlan p = chunk_plan(chunk_rows(prompt), n_q_heads, n_kv_heads, n_seqs, max_pages, page_size, n_tokens, head_dim,
                                   workspace == nullptr ? 0 : workspace_bytes);
    if (!aligned(workspace, 16)) return SPH_EINVAL;
    const __int128 blocks = (__int128)p.tiles * n_kv_heads * p.splits;
    if (blocks * kAttnThreads > UINT32_MAX) return SPH_EINVAL;
    const ChunkSplit sp{p.splits, static_cast<float*>(workspace)};
    hipStream_t s = static_cast<hipStream_t>(stream);
    const unsigned n = (unsigned)blocks;
    int r;
    if (prompt) {
        r = launch_prompt(a, cache_dtype, n, sp, s);
    } else {
        r = launch_tiles(a, n, sp, s);
    }
    if (r != SPH_OK || p.splits == 1) return r;
    const int64_t threads = n_tokens * n_q_heads * (head_dim / 4);
    return launch(paged_chunk_join_kernel, dim3((unsigned)((threads + kAttnThreads - 1) / kAttnThreads)), kAttnThreads, s, a, sp);
}

extern "C" int64_t sph_paged_attention_workspace(int64_t n_q_heads, int64_t n_kv_heads, int64_t n_seqs, int64_t max_pages,
                                                 int64_t page_size, int64_t head_dim) {
    if (!sph::sizes_ok(n_q_heads, n_kv_heads, n_seqs, max_pages, page_size, head_dim, n_seqs)) return SPH_EINVAL;
    return sph::split_plan(n_q_heads, n_kv_heads, n_seqs, max_pages, page_size, head_dim, 0, INT64_MAX).bytes;
}

extern "C" int64_t sph_paged_attention_chunk_workspace(int64_t n_q_heads, int64_t n_kv_heads, int64_t n_seqs,
                                                       int64_t max_pages, int64_t page_size, int64_t n_tokens,
                                                       int64_t head_dim) {
    if (!sph::sizes_ok(n_q_heads, n_kv_heads, n_seqs, max_pages, page_size, head_dim, n_tokens)) return SPH_EINVAL;
    // The larger of the two tiles' plans.
    int64_t most = 0;
    for (const bool prompt : {false, true}) {
        const int64_t n = sph::chunk_plan(sph::chunk_rows(prompt), n_q_heads, n_kv_heads, n_seqs, max_pages, page_size, n_tokens,
                                          head_dim, INT64_MAX).bytes;
        if (n > most) most = n;
    }
    return most;
}
