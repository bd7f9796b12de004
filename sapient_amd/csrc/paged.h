// paged.h — the paged KV cache as its kernels see it: pools [n_pages, n_kv, page_size, head_dim] of keys and of
// values, a block table [n_seqs, max_pages] naming each sequence's pages, the sequences' lengths, and, for steps of
// several new tokens per sequence, the rows cu_q [n_seqs + 1] that hold them (token-major).
//
// Token t of sequence b is row t % page_size of page table[b, t / page_size]; its row in a pool viewed as
// [n_pages · n_kv · page_size, head_dim] is a 32-bit number (the host refuses larger pools, of 2^32 rows and more),
// so a lane holds one register per key it follows and widens to 64 bits only in the address.
// Everything in the tables comes from device memory and is checked there: an entry that names no page, or a
// position that has no entry, is a missing key (kNoRow), never an access.
#pragma once

#include "sph_common.h"

namespace sph {

constexpr uint32_t kNoRow = 0xFFFFFFFFu;
constexpr int kMaxTokens = 1 << 30;  // of a sequence: positions and steps past them stay in 32 bits

// n / d for n < 2^31 by a multiplication (page sizes are arguments; a division by one is some forty operations):
// with s = ceil(log2 d) and m = floor(2^32 (2^s - d) / d) + 1, n / d = (mulhi(m, n) + n) >> s, and for n < 2^31
// the sum stays below 2^32.
struct Divisor {
    uint32_t d, m, s;
    Divisor() = default;
    explicit Divisor(uint32_t div) : d(div), s(0) {
        while ((uint64_t(1) << s) < d) ++s;
        m = (uint32_t)((((uint64_t(1) << s) - d) << 32) / d + 1);
    }
    __device__ __forceinline__ uint32_t quotient(uint32_t n) const { return (__umulhi(m, n) + n) >> s; }
};

struct PagedTable {
    const int32_t* table;  // [n_seqs, max_pages]
    const int32_t* lens;   // [n_seqs]: tokens in the cache, the new ones included
    const int32_t* cu;     // [n_seqs + 1] or null: one new token per sequence
    int n_seqs, max_pages, n_pages, n_kv;
    Divisor page;  // by the page's tokens
    int capacity;  // tokens that a row of the table has entries for

    // Pool row of token t (kv head 0; head h's is h · page_size further), or kNoRow.
    __device__ __forceinline__ uint32_t row(int seq, uint32_t t) const {
        const uint32_t p = page.quotient(t);
        if (p >= (uint32_t)max_pages || t >= (uint32_t)kMaxTokens) return kNoRow;
        const uint32_t id = (uint32_t)table[(size_t)seq * (size_t)max_pages + p];
        return id < (uint32_t)n_pages ? id * (uint32_t)n_kv * page.d + (t - p * page.d) : kNoRow;
    }

    // The same in two parts, so that the entry can be asked for well ahead of its use: t < capacity, and no branch.
    __device__ __forceinline__ uint32_t entry(int seq, uint32_t t) const {
        return (uint32_t)table[(size_t)seq * (size_t)max_pages + page.quotient(t)];
    }
    __device__ __forceinline__ uint32_t row_in(uint32_t id, uint32_t t) const {
        return id < (uint32_t)n_pages ? id * (uint32_t)n_kv * page.d + (t - page.quotient(t) * page.d) : kNoRow;
    }

    __device__ __forceinline__ int length(int b) const { return lens[b] < 0 ? 0 : lens[b]; }

    // The rows [begin, end) of sequence b's new tokens among n_rows, whatever cu holds.
    __device__ __forceinline__ void new_rows(int b, int n_rows, int& begin, int& end) const {
        if (cu == nullptr) {
            begin = b;
            end = b + 1;
            return;
        }
        const int lo = cu[b], hi = cu[b + 1];
        begin = lo < 0 ? 0 : lo > n_rows ? n_rows : lo;
        end = hi < begin ? begin : hi > n_rows ? n_rows : hi;
    }
};

// Host: the checks that every entry point over pages shares. rows: q rows of the call.
inline bool paged_ok(const int32_t* seq_lens, const int32_t* block_table, int64_t n_seqs, int64_t max_pages, int64_t n_pages,
                     int64_t page_size, int64_t n_kv, int64_t n_rows) {
    if (n_seqs < 0 || max_pages < 0 || n_pages < 1 || page_size < 1 || n_kv < 1 || n_rows < 0) return false;
    if (n_seqs > INT32_MAX || max_pages > INT32_MAX || n_pages > INT32_MAX || page_size > INT32_MAX || n_kv > INT32_MAX ||
        n_rows > INT32_MAX)
        return false;
    if ((__int128)n_pages * n_kv * page_size >= (__int128)kNoRow) return false;
    if (n_seqs > 0 && n_rows > 0 && (seq_lens == nullptr || (block_table == nullptr && max_pages > 0))) return false;
    return aligned(seq_lens, 4) && aligned(block_table, 4);
}

inline PagedTable paged_table(const int32_t* seq_lens, const int32_t* cu_q, const int32_t* block_table, int64_t n_seqs,
                              int64_t max_pages, int64_t n_pages, int64_t page_size, int64_t n_kv) {
    PagedTable p;
    p.table = block_table;
    p.lens = seq_lens;
    p.cu = cu_q;
    p.n_seqs = (int)n_seqs;
    p.max_pages = (int)max_pages;
    p.n_pages = (int)n_pages;
    p.n_kv = (int)n_kv;
    p.page = Divisor((uint32_t)page_size);
    const int64_t capacity = max_pages * page_size;
    p.capacity = capacity < kMaxTokens ? (int)capacity : kMaxTokens;
    return p;
}

}  // namespace sph
