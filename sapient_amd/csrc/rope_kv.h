// rope_kv.h — the fused bias + RoPE + KV-cache append: its kernel, launch shape and the row
// accesses it shares with the in-place kernel (rope.hip). Included by the translation units of
// the contiguous cache (rope.hip) and of the paged one (rope_paged.hip).
#pragma once

#include <math.h>

#include <type_traits>

#include "glibc_sincosf.h"
#include "paged.h"
#include "sph_common.h"

namespace sph {
namespace {

constexpr int kThreads = 256;
constexpr int kWave = 64;
constexpr int kMaxHalf = 256;  // rotary_dim <= 512

struct DenTable {
    float v[kMaxHalf];
};

// The large-argument reduction indexes the 4/pi table per lane; staged in LDS (by each kernel, before its angles)
// the lookups stay off the vector-memory queue the row stream keeps full (measured: ~1.5 µs of 58 at the
// Llama-3-8B shape).
__constant__ InvPio4Table kInvPio4 = inv_pio4_table();

// L consecutive elements of one row held as they sit in memory (32-bit words,
// or single elements when the run is narrower than a word or ELEM asks for
// element accesses: rows only element-aligned), so that a batch of rows can be
// in flight while the previous batch is rotated and stored.
template <typename T, int L, bool ELEM = false, bool NT = true>
struct RawRun {
    static constexpr bool kWords = !ELEM && (L * (int)sizeof(T)) % 4 == 0;
    uint32_t w[kWords ? words_of<T, L>::n : 1];
    T e[kWords ? 1 : L];

    __device__ __forceinline__ void load(const T* p) {
        if constexpr (kWords) {
            load_words<T, L, NT>(p, w);
        } else {
#pragma unroll
            for (int i = 0; i < L; ++i) e[i] = p[i];
        }
    }
    __device__ __forceinline__ void to_f32(float (&v)[L]) const {
        if constexpr (kWords) {
            words_to_f32<T, L>(w, v);
        } else {
#pragma unroll
            for (int i = 0; i < L; ++i) v[i] = widen(e[i]);
        }
    }
};

template <typename T, int L, bool ELEM = false, bool NT = true>
__device__ __forceinline__ void store_run(T* p, const float (&v)[L]) {
    if constexpr (!ELEM && (L * (int)sizeof(T)) % 4 == 0) {
        store_f32<T, L, NT>(p, v);
    } else {
#pragma unroll
        for (int i = 0; i < L; ++i) p[i] = narrow<T>(v[i]);
    }
}

// Everything a fused launch reads, by value (den, where the angles are evaluated, by lane).
template <typename T, typename TC>
struct RopeKvArgs {
    using Q = T;
    using Cache = TC;
    static constexpr bool kPaged = false;
    const T* q;
    T* qo;
    const T* k;
    const T* v;
    TC* kc;
    TC* vc;
    const int32_t* pos;
    const void* bias[3];  // of q, k, v; each may be null
    int bias_dt;
    int nq, nkv;
    int64_t seq, max_seq;
    int head_dim, half;
    int lanes, toks, heads;  // lanes per row; a block's tokens, and its heads per pass
    uint32_t by_lanes, by_toks, by_heads;  // 2^16 over each, rounded up (see quotient)
    int h_first;                           // the launch's first head and token
    int64_t s_first;
    float pos_scale;
    int32_t* bad;
    const float* ang;
    bool ang_by_pos;
    DenTable den;
};

// The same for a paged cache: seq counts the rows of all sequences' new tokens, read and (q) written token-major; pos,
// max_seq and the supplied angles are not used.
template <typename T, typename TC>
struct RopeKvPagedArgs : RopeKvArgs<T, TC> {
    static constexpr bool kPaged = true;
    PagedTable pages;
};

constexpr int kMaxBlockAngles = 256;  // a block's tokens times pairs

// n / d for n < 256 and d <= 256, from 2^16 / d rounded up: exact, since the excess is below n · d / 2^16 < 1 of a
// quotient's step. An integer division by an argument is some forty operations, and a decode step's threads would
// start with three in a row (the engine's step 321 -> 310 us a token).
__host__ __device__ constexpr uint32_t reciprocal(int d) { return (0x10000u + (uint32_t)d - 1) / (uint32_t)d; }
__device__ __forceinline__ int quotient(int n, uint32_t rec) { return (int)((uint32_t)n * rec >> 16); }

// A thread's share of a row, as it sits in memory: P pairs, in two runs of P elements at i0 and
// half + i0 (NEOX) or one of 2P at 2 i0 (interleaved). In f32, f holds the runs one after the other.
template <typename T, int P, bool INTERLEAVED, bool NT>
struct PairRuns {
    static constexpr int R = INTERLEAVED ? 1 : 2, L = INTERLEAVED ? 2 * P : P;
    RawRun<T, L, false, NT> run[R];
    __device__ __forceinline__ static int at(int r, int i0, int half) { return INTERLEAVED ? 2 * i0 : i0 + r * half; }
    __device__ __forceinline__ void load(const T* row, int i0, int half) {
#pragma unroll
        for (int r = 0; r < R; ++r) run[r].load(row + at(r, i0, half));
    }
    __device__ __forceinline__ void to_f32(float (&f)[2 * P]) const {
#pragma unroll
        for (int r = 0; r < R; ++r) {
            float t[L];
            run[r].to_f32(t);
#pragma unroll
            for (int j = 0; j < L; ++j) f[r * L + j] = t[j];
        }
    }
    template <typename TR>
    __device__ __forceinline__ static void store(TR* row, int i0, int half, const float (&f)[2 * P]) {
#pragma unroll
        for (int r = 0; r < R; ++r) {
            float t[L];
#pragma unroll
            for (int j = 0; j < L; ++j) t[j] = f[r * L + j];
            store_run<TR, L, false, NT>(row + at(r, i0, half), t);
        }
    }
};

// N consecutive bias values (of any float type) as they sit in memory, halves in the first N / 2 words, so that
// their loads join the rows' in flight. The first N / 2 words are loaded alike for either width: were they loaded
// in a branch per type, each load would wait for the one before it. The launch checked the alignment.
template <int N>
struct BiasRun {
    static_assert(N % 2 == 0, "whole words of halves");
    uint32_t w[2][N / 2];
    __device__ __forceinline__ void load(const void* p, size_t at, bool f32) {
        const float* q = reinterpret_cast<const float*>(static_cast<const char*>(p) + (at << (f32 ? 2 : 1)));
        load_words<float, N / 2>(q, w[0]);
        if (f32) load_words<float, N / 2>(q + N / 2, w[1]);
    }
    __device__ __forceinline__ void to_f32(int dt, float (&b)[N]) const {
        if (dt == SPH_F32) {
#pragma unroll
            for (int i = 0; i < N; ++i) b[i] = __uint_as_float(w[i / (N / 2)][i % (N / 2)]);
        } else if (dt == SPH_F16) {
            words_to_f32<f16, N>(w[0], b);
        } else {
            words_to_f32<bf16, N>(w[0], b);
        }
    }
};

// A thread's P supplied angles, (cos, sin) pairs at 8-byte alignment.
template <int P>
__device__ __forceinline__ void load_angles(const float* p, float (&ag)[2 * P]) {
    load_run_f32<float, 2 * P, false>(p, 2 * P, ag);
}

// Fused decode step: heads [0, nq) are q rows, rotated and written to qo
// heads-major; heads [nq, nq + nkv) rotate the k row and write it, plus the v
// row, to cache row (h, positions[s]). batch = 1 and rotary_dim = head_dim, so
// a thread's P pairs and the pairs of its lane neighbours cover every channel
// of the row. TM: q, k and v are read token-major [seq, heads, head_dim] (the
// projections' layout) instead of heads-major; without TM, qo == q (in place).
// A block covers a few tokens by U passes of a few heads. Its angles (tokens x
// pairs, at most one per thread) are evaluated once, into LDS, while the rows'
// loads are in flight, and shared by all its heads: glibc's sincos in double
// arithmetic is the long pole of a launch that would otherwise wait on memory
// once. Threads take the angles pair-major, so a wave's are of one size and
// only waves of low pairs run the large-argument reduction.
//
// A paged cache (Args::kPaged) differs in where a token's position and its cache
// row come from. Row s belongs to the sequence b with cu[b] <= s < cu[b + 1]
// (b = s where there is one token each). Up to 64 sequences a wave's lanes hold
// one's cu[b + 1] and length each (requested ahead of the rows, so that waiting
// for them does not wait for those), count the entries at or below the block's
// first row, and walk on to their own rows' by exchanges between lanes, with no
// further load (a prefill step of 6 prompts, 8513 tokens of 32 + 8 x 128 f16:
// 44.8 -> 41.1 us, 35 for one contiguous cache); more sequences are counted by the block. The position is
// lens[b] - (cu[b + 1] - s); the table's entry is requested as soon as it is
// known and arrives behind the angles.
//
// The body is a file of its own, included by both kernels, with the argument struct as each kernel's own parameter `a`: in a
// function its reference had arguments asked for late, and its copy went to scratch memory, angles' denominators and all.
template <typename T, typename TC, int P, bool INTERLEAVED, bool TM, int U, bool BIAS, bool NT>
__global__ __launch_bounds__(kThreads) void rope_kv_kernel(RopeKvArgs<T, TC> a) {
    using Args = RopeKvArgs<T, TC>;
#include "rope_kv_body.h"
}
template <typename T, typename TC, int P, bool INTERLEAVED, int U, bool BIAS, bool NT>
__global__ __launch_bounds__(kThreads) void rope_kv_paged_kernel(RopeKvPagedArgs<T, TC> a) {
    using Args = RopeKvPagedArgs<T, TC>;
    constexpr bool TM = true;
#include "rope_kv_body.h"
}

// Denominators powf(base, 2i / rotary_dim) from the host libm, the call the reference makes.
inline void fill_dens(DenTable& den, int half, int rotary_dim, float base) {
    for (int i = 0; i < kMaxHalf; ++i)
        den.v[i] = i < half ? powf(base, 2.0f * (float)i / (float)rotary_dim) : 1.0f;
}

// Launch shape, from the lanes that the rows need (one row per thread and pass):
//  - small (up to 2^14: decode steps): blocks of one wave, so that the rows spread over the CUs, each with the
//    angles of one token (two heads a block 2.96 us, four 3.14, one 3.00 at one token of 14 + 2 heads x 64; with
//    the angles supplied, 24 such layers in the engine's replayed step: 304-313 us a token, four 317-323, one 305-314);
//  - up to 2^18: at most 64 angles a block, so that only some waves evaluate them, and from 2^16 on two rows
//    per thread (512 tokens of 14 + 2 x 64 f32 4.1 us with 256 angles, 3.8 with 64; 333 of 32 + 8 x 128 bf16
//    4.4 with one row, 4.0 with two; 64 tokens of 64 heads x 80 f16 4.4 with one, 4.8 with two);
//  - larger: 256 angles, two rows (2048 tokens of 32 + 8 x 128 f16 10.9 us, with 64 angles 11.6).
template <int P, bool IL, bool TM, typename A>
int launch_rope_kv_p(A& a, hipStream_t stream) {
    using T = typename A::Q;
    using TC = typename A::Cache;
    const int heads = a.nq + a.nkv;
    a.lanes = a.half / P;
    const int64_t lanes = a.seq * heads * a.lanes;
    const bool small = lanes <= 1 << 14 && a.half <= 64;
    const int threads = small ? kWave : kThreads;
    const int rows = threads / a.lanes;  // of a block per pass: toks x heads
    a.toks = (lanes < 1 << 18 ? 64 : kMaxBlockAngles) / a.half;
    if (a.toks < 1) a.toks = 1;
    if (a.toks > rows) a.toks = rows;
    if (a.toks > a.seq) a.toks = (int)a.seq;
    a.heads = rows / a.toks;
    if (small && a.heads > 2) a.heads = 2;
    if (a.heads > heads) {
        a.heads = heads;
        // Few heads: more tokens, so that the block's threads have rows (16384 tokens of 1 + 1 heads x 64: f16 13.7 ->
        // 6.2 us, f32 7.0 -> 5.6).
        if (!small) {
            int t = rows / heads;
            if (t > kMaxBlockAngles / a.half) t = kMaxBlockAngles / a.half;
            if (t > a.seq) t = (int)a.seq;
            if (t > a.toks) a.toks = t;
        }
    }
    a.by_lanes = reciprocal(a.lanes);
    a.by_toks = reciprocal(a.toks);
    a.by_heads = reciprocal(a.heads);
    const bool two = lanes >= 1 << 16;
    const bool bias = a.bias[0] != nullptr || a.bias[1] != nullptr || a.bias[2] != nullptr;
    const int tile = (two ? 2 : 1) * a.heads;  // heads per block
    // Large launches pass the caches by: 8192 tokens of 32 + 8 x 128 f16 39.7 us cached, 35.1 non-temporal, but
    // 333 tokens bf16 4.0 against 4.4 (kCachedBytes).
    const int64_t row = (int64_t)a.head_dim * (TM ? 2 : 1) * (int64_t)sizeof(T);
    const bool nt = two && a.seq * (a.nq * row + 2 * a.nkv * (int64_t)a.head_dim * (int64_t)(sizeof(T) + sizeof(TC))) >=
                               kCachedBytes;
    // A launch: fewer than 2^32 work-items in x, at most 65535 blocks in y.
    constexpr int64_t kMaxY = 65535;
    const int64_t most = UINT32_MAX / threads * (int64_t)a.toks;
    for (int64_t h0 = 0; h0 < heads; h0 += kMaxY * tile) {
        a.h_first = (int)h0;
        const int64_t tiles = (heads - h0 + tile - 1) / tile;
        for (a.s_first = 0; a.s_first < a.seq; a.s_first += most) {
            const int64_t toks = a.seq - a.s_first < most ? a.seq - a.s_first : most;
            const dim3 grid((unsigned)((toks + a.toks - 1) / a.toks), (unsigned)(tiles < kMaxY ? tiles : kMaxY));
            auto go = [&](auto u, auto b, auto n) {
                if constexpr (A::kPaged)
                    return launch(rope_kv_paged_kernel<T, TC, P, IL, decltype(u)::value, decltype(b)::value, decltype(n)::value>,
                                  grid, threads, stream, a);
                else
                    return launch(rope_kv_kernel<T, TC, P, IL, TM, decltype(u)::value, decltype(b)::value, decltype(n)::value>,
                                  grid, threads, stream, a);
            };
            using std::false_type;
            using std::true_type;
            const std::integral_constant<int, 1> one;
            const std::integral_constant<int, 2> pair;
            const int st = !two ? (bias ? go(one, true_type{}, false_type{}) : go(one, false_type{}, false_type{}))
                           : nt ? (bias ? go(pair, true_type{}, true_type{}) : go(pair, false_type{}, true_type{}))
                                : (bias ? go(pair, true_type{}, false_type{}) : go(pair, false_type{}, false_type{}));
            if (st != SPH_OK) return st;
        }
    }
    return SPH_OK;
}

// P: pairs per thread, the widest whose accesses of q/k/v (type T) and of the
// caches (type TC) stay within 16 bytes and aligned.
template <bool TM, typename A>
int launch_rope_kv(A& a, int layout, float base, hipStream_t stream) {
    using T = typename A::Q;
    using TC = typename A::Cache;
    a.half = a.head_dim / 2;
    // Supplied angles leave the denominators unused: no libm calls per launch.
    if (a.ang == nullptr) fill_dens(a.den, a.half, a.head_dim, base);
    const bool il = layout == SPH_ROPE_INTERLEAVED;
    const size_t sb = dtype_size(a.bias_dt);
    auto ok = [&](int P) {
        const int run = il ? 2 * P : P;  // contiguous elements per access
        if (a.half % P != 0 || a.head_dim % run != 0) return false;
        if (run * sizeof(T) > 16 || run * sizeof(TC) > 16) return false;
        if ((run * sizeof(T)) % 4 != 0 || (run * sizeof(TC)) % 4 != 0) return false;
        const size_t at = run * sizeof(T) < 16 ? run * sizeof(T) : 16;
        const size_t ac = run * sizeof(TC) < 16 ? run * sizeof(TC) : 16;
        const size_t ab = run * sb < 16 ? run * sb : 16;  // bias runs may span two 16-byte loads
        return aligned(a.q, at) && aligned(a.qo, at) && aligned(a.k, at) && aligned(a.v, at) && aligned(a.kc, ac) &&
               aligned(a.vc, ac) && aligned(a.bias[0], ab) && aligned(a.bias[1], ab) && aligned(a.bias[2], ab);
    };
    constexpr int V = vec16<T>::n < vec16<TC>::n ? vec16<T>::n : vec16<TC>::n;
    // A decode step (a few tokens) leaves most lanes of its blocks idle and its
    // time is one dependent chain — position load, the thread's sin/cos, store —
    // so it takes the narrowest runs that stay word-sized.
    const bool few = a.seq <= 4;
    if (!il) {
        if (few && ok(V / 2)) return launch_rope_kv_p<V / 2, false, TM>(a, stream);
        if (ok(V)) return launch_rope_kv_p<V, false, TM>(a, stream);
        if (ok(V / 2)) return launch_rope_kv_p<V / 2, false, TM>(a, stream);
        if constexpr (V / 4 >= 2) {
            if (ok(V / 4)) return launch_rope_kv_p<V / 4, false, TM>(a, stream);
        }
    } else {
        if constexpr (V / 4 >= 1) {
            if (few && ok(V / 4)) return launch_rope_kv_p<V / 4, true, TM>(a, stream);
        }
        if (ok(V / 2)) return launch_rope_kv_p<V / 2, true, TM>(a, stream);
        if constexpr (V / 4 >= 1) {
            if (ok(V / 4)) return launch_rope_kv_p<V / 4, true, TM>(a, stream);
        }
    }
    return SPH_EINVAL;  // head_dim or alignment the vector paths do not cover
}

}  // namespace
}  // namespace sph
