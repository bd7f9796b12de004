// attention.h — softmax attention over the paged KV cache: arguments, and the kernels of 16-column tiles that serve
// single tokens, and chunks over f32 caches (attention.hip; chunks over half caches: attention_prompt.hip).
//
// Mathematics. For the rows (columns of a tile) that share a kv head, with s the capped and biased score in units
// of log2 (scores times log2 e, so that a weight is one v_exp_f32):
//   m = max s;  p = 2^(s - m);  l = sum p;  out = (sum p v) / l
// in one pass over the keys: m is a running reference, raised (and l and the sums scaled by 2^(m_old - m_new))
// only when a score passes it by 2^8, which keeps every p below 2^8 and spares most tiles the exchange between
// lanes that a maximum needs. Parts of a key range (waves, workgroups) are joined by their (m, l, sums).
//
// Layout. Scores are computed transposed, S^T = K Q^T, so that lane (j = lane % 16, g = lane / 16) of a 16 x 16
// matrix instruction holds column j's scores of tokens 4g .. 4g + 3, and keeps them as the second product's
// operand O^T = V^T P^T without any exchange: the order of a product's inner dimension is free as long as both
// operands share it, so V's rows are taken in the order in which the lanes hold P. A column's m and l live in
// its own lanes. K and V go from memory to the operand registers with no stop in LDS: K as rows (lane j: token
// j, 8 channels), V as rows too (lane j: channels E j .. E j + E - 1 of its tokens, E = DP / 16) and turned in
// registers, one v_perm_b32 per two values, which leaves each lane with adjacent output channels.
//
// What bounds it: memory. Up to 16 rows share a key's bytes, some 20 matrix and 100 vector instructions a wave per 16
// KB of them (32 keys of 128 halves), a quarter of what a CU could do while they arrive. One step's V and the next
// one's K are in flight in each of 8 waves a CU. 64 sequences of 1 to 8192 keys, 32 + 8 heads x 128 bf16, 818 MB: 153
// us (5.4 TB/s; a large copy runs at 6.2); one of 131071 keys, 537 MB: 100 us. Short batches wait for a chain of loads
// (length, entry, K and V), 0.7 to 1 us each: one sequence of 333 keys 6.4 us.
#pragma once

#include "paged.h"
#include "sph_common.h"

namespace sph {

typedef _Float16 h8 __attribute__((ext_vector_type(8)));
typedef __bf16 b8 __attribute__((ext_vector_type(8)));
typedef float f32x16 __attribute__((ext_vector_type(16)));

struct AttnArgs {
    const void* q;
    void* out;
    const void* kc;
    const void* vc;
    PagedTable pages;
    const float* slopes;
    const int32_t* prefix;
    int32_t* bad;
    int dtype;  // of q and out
    int n_rows, nq, group, head_dim;
    int window;  // 0: all keys
    float scale, cap;
};

// Parts that a chunk's keys are taken in, and where they go.
struct ChunkSplit {
    int splits;
    float* part;  // [splits][n_rows · nq][head_dim] sums, then [splits][n_rows · nq][2] m and l
};

namespace {

constexpr int kWave = 64;
constexpr int kAttnWaves = 4;
constexpr int kAttnThreads = kWave * kAttnWaves;
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kSlack = 8.0f;  // how far (log2) a score may pass the running reference
constexpr float kNegInf = -__builtin_inff();

__device__ __forceinline__ float exp2_hw(float x) { return __builtin_amdgcn_exp2f(x); }

// What is done to a product q·k where it is more than a scale: the cap, and the slope's distance; the score in log2
// units. The cap is cap tanh(x / cap) = cap - 2 cap / (e^(2 x / cap) + 1), its exp and reciprocal the hardware's where the
// output is half precision (absolute error some 2^-23 of the cap, under a rounding of the weights), the library's tanh
// where it is f32.
template <bool ACCURATE>
struct ScoreForm {
    float unit, grow, cap, slope;
    // unit: what a product is multiplied by for a score in its own units
    __device__ __forceinline__ ScoreForm(const AttnArgs& a, float unit_, int head) : unit(unit_ * kLog2e) {
        cap = a.cap * kLog2e;
        grow = a.cap == 0.0f ? 0.0f : ACCURATE ? unit_ / a.cap : 2.0f * kLog2e * unit_ / a.cap;
        slope = a.slopes != nullptr ? a.slopes[head] * -kLog2e : 0.0f;
    }
    // s[i]: the products of keys at distances dist - at(i)
    template <int N, typename At>
    __device__ __forceinline__ void apply(const AttnArgs& a, float (&s)[N], float dist, At at) const {
        if (a.cap != 0.0f) {
#pragma unroll
            for (int i = 0; i < N; ++i) {
                if constexpr (ACCURATE) s[i] = cap * tanhf(s[i] * grow);
                else s[i] = __builtin_fmaf(-2.0f * cap, __builtin_amdgcn_rcpf(exp2_hw(s[i] * grow) + 1.0f), cap);
            }
        } else {
#pragma unroll
            for (int i = 0; i < N; ++i) s[i] *= unit;
        }
        if (a.slopes != nullptr) {
#pragma unroll
            for (int i = 0; i < N; ++i) s[i] = __builtin_fmaf(slope, fabsf(dist - (float)at(i)), s[i]);
        }
    }
};

template <typename TC>
__device__ __forceinline__ f32x4 mma(u32x4 a, u32x4 b, f32x4 c) {
    if constexpr (__is_same(TC, f16))
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(h8, a), __builtin_bit_cast(h8, b), c, 0, 0, 0);
    else
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(b8, a), __builtin_bit_cast(b8, b), c, 0, 0, 0);
}

template <typename TC>
__device__ __forceinline__ uint32_t narrow2(float a, float b) {
    if constexpr (__is_same(TC, f16)) return narrow2_f16(a, b);
    else return narrow2_bf16(a, b);
}
template <typename TC>
__device__ __forceinline__ float widen_half(uint32_t w, int i) {
    return widen(TC{(uint16_t)(w >> (16 * i))});
}

// f[s] = the E channels from d0 + s · step of a row of type dt (at element `at`), zeros from channel D on. One branch on the
// type with all loads of it in flight together: asked for one by one, each in a branch of its own, they were waited for
// one by one (16 us of a chunk's 19).
template <int KS, int E>
__device__ __forceinline__ void load_row_f32(const void* p, int dt, size_t at, int d0, int step, int D, float (&f)[KS][E]) {
#pragma unroll
    for (int s = 0; s < KS; ++s)
#pragma unroll
        for (int e = 0; e < E; ++e) f[s][e] = 0.0f;
    if (dt == SPH_F32) {
#pragma unroll
        for (int s = 0; s < KS; ++s)
            if (d0 + s * step < D) load_f32<float, E>(static_cast<const float*>(p) + at + d0 + s * step, f[s]);
    } else {
        uint32_t w[KS][E / 2];
#pragma unroll
        for (int s = 0; s < KS; ++s) {
#pragma unroll
            for (int i = 0; i < E / 2; ++i) w[s][i] = 0u;
            if (d0 + s * step < D) load_words<f16, E>(static_cast<const f16*>(p) + at + d0 + s * step, w[s]);
        }
#pragma unroll
        for (int s = 0; s < KS; ++s) {
            if (dt == SPH_F16) words_to_f32<f16, E>(w[s], f[s]);
            else words_to_f32<bf16, E>(w[s], f[s]);
        }
    }
}
__device__ __forceinline__ void store4_from_f32(void* p, int dt, size_t i, f32x4 v) {
    if (dt == SPH_F32) {
        *reinterpret_cast<f32x4*>(static_cast<float*>(p) + i) = v;
    } else {
        const u32x2 w = dt == SPH_F16 ? u32x2{narrow2_f16(v[0], v[1]), narrow2_f16(v[2], v[3])}
                                      : u32x2{narrow2_bf16(v[0], v[1]), narrow2_bf16(v[2], v[3])};
        *reinterpret_cast<u32x2*>(static_cast<uint16_t*>(p) + i) = w;
    }
}

// Which sequence the unit pick(total) falls to, where sequence b has count(b) units, counted by the block's NT threads:
// true, with the sequence and the unit's number within it, or false where there is no such unit (negative, or past the
// last). Every thread calls it.
struct Located {
    int64_t wave_sum[kAttnThreads / kWave];
    int64_t within;
    int seq;
};
template <int NT, typename F, typename P>
__device__ __forceinline__ bool locate_unit(int n_seqs, P pick, F count, Located& sm, int& seq, int64_t& within,
                                            int64_t& total) {
    const int tid = threadIdx.x, lane = tid % kWave;
    const int each = (n_seqs + NT - 1) / NT, b0 = tid * each, b1 = b0 + each < n_seqs ? b0 + each : n_seqs;
    int64_t own = 0;
    for (int b = b0; b < b1; ++b) own += count(b);
    int64_t upto = own;
#pragma unroll
    for (int d = 1; d < kWave; d <<= 1) {
        const int64_t o = __shfl_up(upto, d);
        if (lane >= d) upto += o;
    }
    if (lane == kWave - 1) sm.wave_sum[tid / kWave] = upto;
    __syncthreads();
    int64_t before = upto - own;
    total = 0;
#pragma unroll
    for (int w = 0; w < NT / kWave; ++w) {
        if (w < tid / kWave) before += sm.wave_sum[w];
        total += sm.wave_sum[w];
    }
    const int64_t u = pick(total);
    if (u >= before && u < before + own) {
        int b = b0;
        for (int64_t n; u >= before + (n = count(b)); ++b) before += n;
        sm.seq = b;
        sm.within = u - before;
    }
    __syncthreads();
    if (u < 0 || u >= total) return false;
    seq = sm.seq;
    within = sm.within;
    return true;
}

// Of the keys t0 .. t0 + 63, those in `there` that a row at position pos sees, as bits.
__device__ __forceinline__ uint64_t visible(uint64_t there, int t0, int pos, int prefix, int window) {
    auto below = [](int n) { return n >= 64 ? ~uint64_t(0) : n <= 0 ? uint64_t(0) : (uint64_t(1) << n) - 1; };
    uint64_t see = below(pos - t0 + 1) | below(prefix - t0);
    if (window > 0) see &= ~below(pos - window + 1 - t0);
    return pos < 0 ? 0 : see & there;
}

// Pieces of the cache's type TC that q and the weights are written as, high one first. With one piece the weights'
// rounding would add to an output of that type as much again as the output's own.
template <typename TC, bool HIGH>
struct Pieces {
    // q: exact (f16 and bf16 into one another, f32 into bf16) or within 2^-22 (f32 into f16); weights for f32 outputs
    static constexpr int q = !HIGH ? 1 : __is_same(TC, bf16) ? 3 : 2;
    static constexpr int high = __is_same(TC, bf16) ? 3 : 2;
};
// The channels f of a row, of which the largest is `most`, as pieces of TC; brought to [1, 2) by a power of two before, so
// that no piece leaves the type's range. Returns the power.
template <typename TC, int NQ, int KS>
__device__ __forceinline__ int split_row(const float (&f)[KS][8], float most, u32x4 (&q)[NQ][KS]) {
    const int ex = most > 0.0f && most < __builtin_inff() ? ilogbf(most) : 0;
#pragma unroll
    for (int s = 0; s < KS; ++s)
#pragma unroll
        for (int e = 0; e < 8; e += 2) {
            float x = ldexpf(f[s][e], -ex), y = ldexpf(f[s][e + 1], -ex);
#pragma unroll
            for (int p = 0; p < NQ; ++p) {
                const uint32_t w = narrow2<TC>(x, y);
                q[p][s][e / 2] = w;
                x -= widen_half<TC>(w, 0);
                y -= widen_half<TC>(w, 1);
            }
        }
    return ex;
}

// A tile's 16 columns: the rows (token i of the sequence's new ones, head h · group + c) with number i · group + c in
// [first, first + 16) of `rows`, for kv head h.
struct Tile {
    int seq, h, first, rows, row0;  // row0: the sequence's first row
    int pos0;                       // position of the sequence's first new token
};

// Whether a word of V (an f32, or two values of a half type) holds what is not finite. In a step of keys that only some of
// a tile's rows see, such a value would reach the others as 0 · inf: there it is cleared, and its key's score made NaN in
// the rows that see the key.
template <typename TC>
__device__ __forceinline__ bool not_finite(uint32_t w) {
    if constexpr (sizeof(TC) == 4) return (w & 0x7F800000u) == 0x7F800000u;
    constexpr uint32_t ones = __is_same(TC, f16) ? 0x7C007C00u : 0x7F807F80u, one = __is_same(TC, f16) ? 0x04000400u : 0x00800080u;
    return (((w & ones) + one) & 0x80008000u) != 0u;
}

// HIGH: q is f32, or the cache's type is another one than q's. LOW: both the same half type.
template <typename TC, int DP, bool EXACT, bool HIGH>
struct TileKernel {
    static constexpr int kDP = DP;
    static constexpr bool kF32 = sizeof(TC) == 4;
    static constexpr int ST = kF32 ? 16 : 32;              // tokens of a wave's step
    static constexpr int kStep = ST * kAttnWaves;          // and of the block's
    static constexpr int kBlocksPerCu = DP > 128 ? 1 : 2;  // by registers
    static constexpr int E = DP / 16;                      // channels of V per lane
    static constexpr int KB = ST / 16;                     // 16-token blocks
    static constexpr int KS = kF32 ? DP / 16 : DP / 32;    // 16-byte pieces of a K row per lane
    static constexpr int VT = ST / 4;                      // tokens of V per lane
    static constexpr int VW = E * (int)sizeof(TC) / 4;     // words of V per token and lane
    static constexpr int NQ = kF32 ? 1 : Pieces<TC, HIGH>::q;
    static constexpr int NP = kF32 ? 1 : HIGH ? Pieces<TC, HIGH>::high : 2;  // (two are free here: memory is waited for)
    // An f16 weight below 2^-14 loses bits: the reference is taken 2^7 lower, so that weights run up to 2^15.
    static constexpr float kLift = __is_same(TC, f16) ? 7.0f : 0.0f;
    static constexpr int kPasses = DP > 128 ? DP / 128 : 1;  // of the join over waves, 128 channels each
    static constexpr int kJoin = DP / kPasses, kJoinRow = kJoin + 4;

    struct Shared {
        float m[kAttnWaves][16], l[kAttnWaves][16];
        float acc[kAttnWaves][16][kJoinRow];  // rows padded: 16-byte writes of 8 neighbouring columns hit all banks
        Located located;
    };

    using KRegs = u32x4[KB][KS];
    using VRegs = uint32_t[VT][VW];

    // One column's state in its lanes.
    float m, l;
    f32x4 acc[E];

    // The keys [lo, hi) of the tile, over the block's four waves; then store(column, channel, m, l, sums of 4 channels)
    // for every column of the tile, by the block's threads.
    // MIXED: the tile's columns may see different keys.
    template <bool MIXED, typename Store>
    __device__ __forceinline__ void attend(const AttnArgs& a, Shared& sm, const Tile& t, uint32_t lo, uint32_t hi, Store store) {
        const int tid = threadIdx.x, wave = tid / kWave, lane = tid % kWave, j = lane % 16, g = lane / 16;
        const int D = EXACT ? DP : a.head_dim;
        const int n_cols = t.rows - t.first < 16 ? t.rows - t.first : 16;
        const int col = t.first + (j < n_cols ? j : n_cols - 1), tok = col / a.group, head = t.h * a.group + (col - tok * a.group);
        const int pos = t.pos0 + tok;
        const int pos_first = t.pos0 + t.first / a.group, pos_last = t.pos0 + (t.first + n_cols - 1) / a.group;
        const int prefix = a.prefix != nullptr ? a.prefix[t.seq] : 0;

        // q, as the B operand: column j, channels of this lane's k slots.
        float unit = a.scale;
        const size_t q_at = ((size_t)(t.row0 + tok) * (size_t)a.nq + (size_t)head) * (size_t)D;
        u32x4 q[NQ][KS];
        if constexpr (!HIGH && !kF32) {
#pragma unroll
            for (int s = 0; s < KS; ++s) {
                const int d = 32 * s + 8 * g;
                q[0][s] = u32x4{0, 0, 0, 0};
                if (EXACT || d < D) q[0][s] = *reinterpret_cast<const u32x4*>(static_cast<const TC*>(a.q) + q_at + d);
            }
        } else if constexpr (kF32) {
            float f[KS][4];
            load_row_f32(a.q, a.dtype, q_at, 4 * g, 16, D, f);
#pragma unroll
            for (int s = 0; s < KS; ++s)
#pragma unroll
                for (int e = 0; e < 4; ++e) q[0][s][e] = __float_as_uint(f[s][e]);
        } else {
            float f[KS][8], most = 0.0f;
            load_row_f32(a.q, a.dtype, q_at, 8 * g, 32, D, f);
#pragma unroll
            for (int s = 0; s < KS; ++s)
#pragma unroll
                for (int e = 0; e < 8; ++e) most = fmaxf(most, fabsf(f[s][e]));
            most = fmaxf(most, __shfl_xor(most, 16));
            most = fmaxf(most, __shfl_xor(most, 32));
            unit = ldexpf(unit, split_row<TC>(f, most, q));
        }

        const ScoreForm<HIGH || kF32> form(a, unit, head);

        const TC *kc = static_cast<const TC*>(a.kc), *vc = static_cast<const TC*>(a.vc);
        const uint32_t head_rows = (uint32_t)t.h * a.pages.page.d;
        // The table's entry for the step's token that this lane follows, asked for two steps ahead (waiting for it where
        // its rows' loads are made would wait for all loads before it), and the token's pool row, kNoRow past
        // hi and where there is no page.
        auto entry_at = [&](uint32_t t0) {
            const uint32_t k = t0 + (uint32_t)(lane % ST);
            return a.pages.entry(t.seq, k < hi ? k : hi - 1);
        };
        auto row_at = [&](uint32_t t0, uint32_t id) -> uint32_t {
            const uint32_t k = t0 + (uint32_t)(lane % ST);
            const uint32_t r = a.pages.row_in(id, k < hi ? k : hi - 1);
            if (k >= lo && k < hi && r == kNoRow && a.bad != nullptr) *a.bad = 1;
            return k < hi && r != kNoRow ? r + head_rows : kNoRow;
        };
        // Where 16 neighbouring keys share a page, lanes find their rows from the block's first by an addition, not by an
        // exchange through LDS.
        const bool by_16 = a.pages.page.d % 16 == 0;
        auto pool_row = [&](uint32_t rows, int block, int i) -> uint32_t {  // of the step's key 16 block + i
            uint32_t r;
            if (by_16) {
                r = __builtin_amdgcn_readlane(rows, 16 * block);
                return (r == kNoRow ? 0u : r) + (uint32_t)i;
            }
            r = __shfl(rows, 16 * block + i);
            return r == kNoRow ? 0u : r;
        };
        // Row 0 stands in for a missing one: there to be read, and masked or cleared.
        auto load_k = [&](uint32_t rows, KRegs& k) {
#pragma unroll
            for (int b = 0; b < KB; ++b) {
                const TC* p = kc + (size_t)pool_row(rows, b, j) * (size_t)D;
#pragma unroll
                for (int s = 0; s < KS; ++s) {
                    const int d = kF32 ? 16 * s + 4 * g : 32 * s + 8 * g;
                    k[b][s] = u32x4{0, 0, 0, 0};
                    if (EXACT || d < D) k[b][s] = *reinterpret_cast<const u32x4*>(p + d);
                }
            }
        };
        auto load_v = [&](uint32_t rows, VRegs& v) {
#pragma unroll
            for (int e = 0; e < VT; ++e) {
                const TC* p = vc + (size_t)pool_row(rows, e / 4, 4 * g + e % 4) * (size_t)D + E * j;
                constexpr int B = VW >= 4 ? 4 : 2;  // words per access
#pragma unroll
                for (int c = 0; c < VW / B; ++c) {
                    const int d = c * (B * 4 / (int)sizeof(TC));
                    if (EXACT || E * j + d < D) {
                        if constexpr (B == 4) {
                            const u32x4 w = *reinterpret_cast<const u32x4*>(p + d);
#pragma unroll
                            for (int i = 0; i < 4; ++i) v[e][4 * c + i] = w[i];
                        } else {
                            const u32x2 w = *reinterpret_cast<const u32x2*>(p + d);
                            v[e][0] = w[0];
                            v[e][1] = w[1];
                        }
                    } else {
#pragma unroll
                        for (int i = 0; i < B; ++i) v[e][B * c + i] = 0u;
                    }
                }
            }
        };

        m = kNegInf;
        l = 0.0f;
#pragma unroll
        for (int n = 0; n < E; ++n) acc[n] = f32x4{0, 0, 0, 0};

        KRegs k;
        VRegs v;
        uint32_t t0 = (lo & ~(uint32_t)(ST - 1)) + (uint32_t)(wave * ST);
        uint32_t rows = kNoRow, id_next = 0;
        if (t0 < hi) {
            const uint32_t id = entry_at(t0);
            id_next = entry_at(t0 + kStep);
            rows = row_at(t0, id);
            load_k(rows, k);
        }
        for (; t0 < hi; t0 += kStep) {
            const uint32_t rows_next = row_at(t0 + kStep, id_next);
            id_next = entry_at(t0 + 2 * kStep);
            load_v(rows, v);
            KRegs k_next;
            load_k(rows_next, k_next);  // (Past the end too: loads in a branch would all be waited for where any is.)

            f32x4 s[KB];
#pragma unroll
            for (int b = 0; b < KB; ++b) {
                s[b] = f32x4{0, 0, 0, 0};
#pragma unroll
                for (int c = 0; c < KS; ++c) {
                    if constexpr (kF32) {
#pragma unroll
                        for (int e = 0; e < 4; ++e)
                            s[b] = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(k[b][c][e]),
                                                                        __uint_as_float(q[0][c][e]), s[b], 0, 0, 0);
                    } else {
#pragma unroll
                        for (int p = NQ - 1; p >= 0; --p) s[b] = mma<TC>(k[b][c], q[p][c], s[b]);
                    }
                }
            }

            // Scores in log2 units, and the mask where the step is not all visible to all columns.
            const uint32_t there = (uint32_t)__ballot(rows != kNoRow && t0 + (uint32_t)(lane % ST) >= lo) & (uint32_t)((uint64_t(1) << ST) - 1);
            const bool whole = there == (uint32_t)((uint64_t(1) << ST) - 1);
            const uint32_t last = t0 + ST - 1;
            const bool seen = whole && pos_first >= 0 && ((int)last <= pos_first || (int)last < prefix) &&
                              (a.window == 0 || pos_last - (int)t0 < a.window);
            {
                float x[4 * KB];
#pragma unroll
                for (int i = 0; i < 4 * KB; ++i) x[i] = s[i / 4][i % 4];
                form.apply(a, x, (float)(pos - (int)t0 - 4 * g), [](int i) { return 16 * (i / 4) + i % 4; });
#pragma unroll
                for (int i = 0; i < 4 * KB; ++i) s[i / 4][i % 4] = x[i];
            }
            if (!whole) {  // what lies in a row that is no key of the sequence may be anything, and 0 · inf is not 0
#pragma unroll
                for (int e = 0; e < VT; ++e)
                    if (!((there >> (16 * (e / 4) + 4 * g + e % 4)) & 1)) {
#pragma unroll
                        for (int w = 0; w < VW; ++w) v[e][w] = 0u;
                    }
            }

            if (!seen) {
                const uint32_t see = (uint32_t)visible(there, (int)t0, pos, prefix, a.window) >> (4 * g);
#pragma unroll
                for (int b = 0; b < KB; ++b)
#pragma unroll
                    for (int r = 0; r < 4; ++r) s[b][r] = see & (1u << (16 * b + r)) ? s[b][r] : kNegInf;
                if constexpr (MIXED) {
                    uint32_t odd = 0;  // this lane's keys with a value that is not finite, as bits of see
#pragma unroll
                    for (int e = 0; e < VT; ++e) {
                        bool any = false;
#pragma unroll
                        for (int w = 0; w < VW; ++w) {
                            const bool x = not_finite<TC>(v[e][w]);
                            any |= x;
                            v[e][w] = x ? 0u : v[e][w];
                        }
                        if ((__ballot(any) >> (16 * g)) & 0xFFFF) odd |= 1u << (16 * (e / 4) + e % 4);
                    }
#pragma unroll
                    for (int b = 0; b < KB; ++b)
#pragma unroll
                        for (int r = 0; r < 4; ++r) s[b][r] = see & odd & (1u << (16 * b + r)) ? __builtin_nanf("") : s[b][r];
                }
            }
            float top = s[0][0];
#pragma unroll
            for (int b = 0; b < KB; ++b)
#pragma unroll
                for (int r = 0; r < 4; ++r) top = fmaxf(top, s[b][r]);
            if (__any(top > m + (kLift + kSlack))) {
                top = fmaxf(top, __shfl_xor(top, 16));
                top = fmaxf(top, __shfl_xor(top, 32));
                const float m_new = fmaxf(m, top - kLift);
                const float f = m_new == kNegInf ? 1.0f : exp2_hw(m - m_new);
                m = m_new;
                l *= f;
#pragma unroll
                for (int n = 0; n < E; ++n) acc[n] *= f;
            }
            const float ref = m == kNegInf ? 0.0f : m;
#pragma unroll
            for (int b = 0; b < KB; ++b)
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    s[b][r] = exp2_hw(s[b][r] - ref);
                    l += s[b][r];
                }

            if constexpr (kF32) {
#pragma unroll
                for (int r = 0; r < 4; ++r)
#pragma unroll
                    for (int n = 0; n < E; ++n)
                        acc[n] = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(v[r][n]), s[0][r], acc[n], 0, 0, 0);
            } else {
                u32x4 p[NP];
#pragma unroll
                for (int i = 0; i < 4; ++i) {  // k slots 2i, 2i + 1 of this lane
                    float x = s[i / 2][2 * (i % 2)], y = s[i / 2][2 * (i % 2) + 1];
#pragma unroll
                    for (int c = 0; c < NP; ++c) {
                        const uint32_t w = narrow2<TC>(x, y);
                        p[c][i] = w;
                        x -= widen_half<TC>(w, 0);
                        y -= widen_half<TC>(w, 1);
                    }
                }
#pragma unroll
                for (int n = 0; n < E; ++n) {
                    u32x4 w;
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        w[i] = __builtin_amdgcn_perm(v[2 * i + 1][n / 2], v[2 * i][n / 2], n % 2 ? 0x07060302u : 0x05040100u);
#pragma unroll
                    for (int c = NP - 1; c >= 0; --c) acc[n] = mma<TC>(w, p[c], acc[n]);
                }
            }
            rows = rows_next;
#pragma unroll
            for (int b = 0; b < KB; ++b)
#pragma unroll
                for (int c = 0; c < KS; ++c) k[b][c] = k_next[b][c];
        }

        // The four waves' parts. Lane (j, g) holds column j, channels E (4g + r) + n in acc[n][r].
        l += __shfl_xor(l, 16);
        l += __shfl_xor(l, 32);
        __syncthreads();  // the block's last tile has been read
        if (g == 0) {
            sm.m[wave][j] = m;
            sm.l[wave][j] = l;
        }
        constexpr int EP = E < 8 ? E : 8;  // channels of a lane's run in a pass
#pragma unroll
        for (int pass = 0; pass < kPasses; ++pass) {
            if (pass > 0) __syncthreads();
            if (j < n_cols) {
#pragma unroll
                for (int r = 0; r < 4; ++r)
#pragma unroll
                    for (int n = 0; n < EP; n += 4)
                        *reinterpret_cast<f32x4*>(&sm.acc[wave][j][EP * (4 * g + r) + n]) =
                            f32x4{acc[8 * pass + n][r], acc[8 * pass + n + 1][r], acc[8 * pass + n + 2][r], acc[8 * pass + n + 3][r]};
            }
            __syncthreads();
            constexpr int kLanes = kJoin / 4;  // threads of a column
            for (int c = tid / kLanes; c < n_cols; c += kAttnThreads / kLanes) {
                const int x = 4 * (tid % kLanes);
                const int d = kPasses == 1 ? x : 16 * (x / 8) + 8 * pass + x % 8;
                float top = kNegInf;
#pragma unroll
                for (int w = 0; w < kAttnWaves; ++w) top = fmaxf(top, sm.m[w][c]);
                float total = 0.0f;
                f32x4 sum = {0, 0, 0, 0};
#pragma unroll
                for (int w = 0; w < kAttnWaves; ++w) {
                    const float f = sm.m[w][c] == kNegInf ? 0.0f : exp2_hw(sm.m[w][c] - top);
                    const f32x4 part = *reinterpret_cast<const f32x4*>(&sm.acc[w][c][x]);
                    total = __builtin_fmaf(sm.l[w][c], f, total);
#pragma unroll
                    for (int i = 0; i < 4; ++i) sum[i] = __builtin_fmaf(part[i], f, sum[i]);
                }
                if (EXACT || d < D) store(c, d, top, total, sum);
            }
        }
    }
};

// ─────────────────────────────── chunks ───────────────────────────────
// A chunk call's blocks take (sequence, tile of rows, kv head), and, where these are fewer than the GPU holds, equal
// parts of the tile's keys, which paged_chunk_join_kernel sums. Which sequences the tiles belong to follows from cu_q
// on the device: the grid has the most tiles there can be.
struct ChunkPart {
    int split;
    uint32_t lo, hi;      // the keys
    uint32_t start, end;  // their steps, aligned
};

__device__ __forceinline__ void chunk_part_sum(const AttnArgs& a, const ChunkSplit& sp, int split, size_t q_row, int d, f32x4 sum) {
    const size_t row = (size_t)split * (size_t)a.n_rows * (size_t)a.nq + q_row;
    *reinterpret_cast<f32x4*>(sp.part + row * (size_t)a.head_dim + d) = sum;
}
__device__ __forceinline__ void chunk_part_ml(const AttnArgs& a, const ChunkSplit& sp, int split, size_t q_row, float m, float l) {
    const size_t all = (size_t)a.n_rows * (size_t)a.nq, row = (size_t)split * all + q_row;
    float* ml = sp.part + (size_t)sp.splits * all * (size_t)a.head_dim + 2 * row;
    ml[0] = m;
    ml[1] = l;
}

// The block's tile of ROWS rows and its part of the keys, in steps of KEYS; false where there is none. kv heads vary
// fastest, so that with 8 of them each XCD keeps one's keys in its L2; of a sequence's tiles the last, with the most
// keys, come first.
template <int ROWS, int KEYS>
__device__ __forceinline__ bool chunk_tile(const AttnArgs& a, const ChunkSplit& sp, Located& sm, Tile& t, ChunkPart& part) {
    const int n_kv = a.pages.n_kv;
    uint32_t block = blockIdx.x;
    t.h = (int)(block % (uint32_t)n_kv);
    block /= (uint32_t)n_kv;
    part.split = (int)(block % (uint32_t)sp.splits);
    block /= (uint32_t)sp.splits;
    auto tiles = [&](int b) -> int64_t {
        int lo, hi;
        a.pages.new_rows(b, a.n_rows, lo, hi);
        return ((int64_t)(hi - lo) * a.group + ROWS - 1) / ROWS;
    };
    int64_t total, tile;
    if (!locate_unit<kAttnThreads>(a.pages.n_seqs, [&](int64_t n) { return n - 1 - (int64_t)block; }, tiles, sm, t.seq, tile, total))
        return false;
    int begin, end;
    a.pages.new_rows(t.seq, a.n_rows, begin, end);
    t.row0 = begin;
    t.rows = (end - begin) * a.group;
    t.first = ROWS * (int)tile;
    const int len = a.pages.length(t.seq), keys = len < a.pages.capacity ? len : a.pages.capacity;
    t.pos0 = len - (end - begin);
    if ((t.pos0 < 0 || keys < len) && threadIdx.x == 0 && a.bad != nullptr) *a.bad = 1;

    // The keys that any of the tile's rows may see.
    const int last_col = t.first + ROWS - 1 < t.rows ? t.first + ROWS - 1 : t.rows - 1;
    const int pos_first = t.pos0 + t.first / a.group, pos_last = t.pos0 + last_col / a.group;
    const int prefix = a.prefix != nullptr ? a.prefix[t.seq] : 0;
    int to = pos_last + 1 > prefix ? pos_last + 1 : prefix;
    if (to > keys) to = keys;
    if (pos_last < 0) to = 0;
    const int from = a.window > 0 && pos_first - a.window + 1 > 0 ? pos_first - a.window + 1 : 0;
    part.hi = (uint32_t)to;
    part.lo = from < to ? (uint32_t)from : part.hi;
    const uint32_t start = part.lo & ~(uint32_t)(KEYS - 1), steps = (part.hi - start + KEYS - 1) / KEYS;
    const uint32_t each = (steps + sp.splits - 1) / sp.splits;
    part.start = start + KEYS * each * part.split;
    part.end = start + KEYS * (each * (part.split + 1) < steps ? each * (part.split + 1) : steps);
    if (part.start > part.end) part.start = part.end;
    return true;
}

template <typename K>
__global__ __launch_bounds__(kAttnThreads, K::kBlocksPerCu) void paged_tiles_kernel(AttnArgs a, ChunkSplit sp) {
    __shared__ typename K::Shared sm;
    Tile t;
    ChunkPart part;
    if (!chunk_tile<16, K::kStep>(a, sp, sm.located, t, part)) return;
    const uint32_t lo = part.lo > part.start ? part.lo : part.start, hi = part.hi < part.end ? part.hi : part.end;
    auto row_of = [&](int c) {
        const int col = t.first + c, tok = col / a.group;
        return (size_t)(t.row0 + tok) * (size_t)a.nq + (size_t)(t.h * a.group + (col - tok * a.group));
    };
    K k;
    if (sp.splits == 1) {
        k.template attend<true>(a, sm, t, lo, hi, [&](int c, int d, float, float l, f32x4 sum) {
            const float f = l == 0.0f ? 0.0f : 1.0f / l;
#pragma unroll
            for (int i = 0; i < 4; ++i) sum[i] = l == 0.0f ? 0.0f : sum[i] * f;
            store4_from_f32(a.out, a.dtype, row_of(c) * (size_t)a.head_dim + d, sum);
        });
    } else {
        k.template attend<true>(a, sm, t, lo, hi, [&](int c, int d, float m, float l, f32x4 sum) {
            chunk_part_sum(a, sp, part.split, row_of(c), d, sum);
            if (d == 0) chunk_part_ml(a, sp, part.split, row_of(c), m, l);
        });
    }
}

// 4 channels of a row a thread. Rows that are no tokens have no parts: cu_q's last entry says where they begin.
__global__ __launch_bounds__(kAttnThreads) void paged_chunk_join_kernel(AttnArgs a, ChunkSplit sp) {
    const size_t all = (size_t)a.n_rows * (size_t)a.nq;
    const uint32_t lanes = (uint32_t)a.head_dim / 4;
    const size_t i = (size_t)blockIdx.x * kAttnThreads + threadIdx.x, q_row = i / lanes;
    const int x = 4 * (int)(i - q_row * lanes);
    if (q_row >= all) return;
    const int64_t row = (int64_t)(q_row / (size_t)a.nq);
    if (row < a.pages.cu[0] || row >= a.pages.cu[a.pages.n_seqs]) return;
    const float* ml = sp.part + (size_t)sp.splits * all * (size_t)a.head_dim + 2 * q_row;
    float top = kNegInf, l = 0.0f;
    f32x4 sum = {0, 0, 0, 0};
    // In groups of eight, whose loads are in flight together.
    constexpr int kAhead = 8;
    for (int s0 = 0; s0 < sp.splits; s0 += kAhead) {
        float m_[kAhead], l_[kAhead];
        f32x4 p_[kAhead];
#pragma unroll
        for (int k = 0; k < kAhead; ++k) {
            const size_t s = s0 + k < sp.splits ? s0 + k : s0;
            m_[k] = ml[2 * s * all];
            l_[k] = ml[2 * s * all + 1];
            p_[k] = *reinterpret_cast<const f32x4*>(sp.part + (s * all + q_row) * (size_t)a.head_dim + x);
            if (s0 + k >= sp.splits) m_[k] = kNegInf;
        }
        float most = top;
#pragma unroll
        for (int k = 0; k < kAhead; ++k) most = fmaxf(most, m_[k]);
        const float ref = most == kNegInf ? 0.0f : most, f = exp2_hw(top - ref);
        l *= f;
#pragma unroll
        for (int c = 0; c < 4; ++c) sum[c] *= f;
#pragma unroll
        for (int k = 0; k < kAhead; ++k) {
            const float w = exp2_hw(m_[k] - ref);
            l = __builtin_fmaf(l_[k], w, l);
#pragma unroll
            for (int c = 0; c < 4; ++c) sum[c] = __builtin_fmaf(p_[k][c], w, sum[c]);
        }
        top = most;
    }
    const float f = l == 0.0f ? 0.0f : 1.0f / l;
#pragma unroll
    for (int c = 0; c < 4; ++c) sum[c] = l == 0.0f ? 0.0f : sum[c] * f;
    store4_from_f32(a.out, a.dtype, q_row * (size_t)a.head_dim + x, sum);
}

// ───────────────────────── single tokens, split ─────────────────────────
// Few sequences of many keys, and batches of mixed lengths, leave CUs idle where a block takes a whole (sequence,
// kv head): 131071 keys of 8 kv heads would run on 8 of 256 CUs. So the keys of all sequences are cut into units
// of one block step, in the order sequence, tile of columns, step, and as many blocks as the GPU holds at once take
// equal shares of them, each a run of neighbouring units: a few pieces of (sequence, tile) ranges, of which only the first
// and the last can be part of one that other blocks share. Those go to the workspace, and paged_join_kernel sums
// them in a fixed order. The shares follow the lengths on the device: nothing is read back, a captured call
// serves any lengths.
struct PartRange {
    int first, count;  // slot of a tile's first part, and its parts; 0 where one share held the tile
};
struct SplitArgs {
    int tiles_per_seq;  // of 16 columns: (kv head, tile of its group)
    int cols;           // of the widest tile
    int shares;         // blocks
    PartRange* ranges;  // [n_seqs · tiles_per_seq]
    float* part;        // [2 · shares][cols][head_dim] sums, then [2 · shares][cols][2] m and l
};

// The key range of single token b, as steps from the aligned start.
template <int STEP>
struct SplitRange {
    int len;
    uint32_t lo, hi, start, steps;
    __device__ __forceinline__ SplitRange(const AttnArgs& a, int b) {
        len = a.pages.length(b);
        hi = (uint32_t)(len < a.pages.capacity ? len : a.pages.capacity);
        lo = a.window > 0 && len > a.window ? (uint32_t)(len - a.window) : 0u;
        if (lo > hi) lo = hi;
        start = lo & ~31u;
        steps = (hi - start + STEP - 1) / STEP;
        if (steps == 0) steps = 1;  // a row without keys is one unit: its zeros
    }
};

// `shares` of `total` units, none of them empty. A double's quotient, cut, is the integers': their own distance from the
// next integer, at least 1 / divisor, is more than its rounding while units stay below 2^43. (Integer divisions of 64
// bits are some hundred operations each, in a row at every block's start.)
__device__ __forceinline__ int64_t share_count(int64_t total, int shares) { return total < shares ? total : shares; }
__device__ __forceinline__ int64_t share_start(int64_t share, int64_t total, int64_t shares) {
    return (int64_t)((double)(share * total) / (double)shares);
}
// The share that unit u is in: the largest with share_start <= u.
__device__ __forceinline__ int64_t share_of(int64_t u, int64_t total, int64_t shares) {
    return (int64_t)((double)((u + 1) * shares - 1) / (double)total);
}

template <typename K>
__global__ __launch_bounds__(kAttnThreads, K::kBlocksPerCu) void paged_split_kernel(AttnArgs a, SplitArgs sp) {
    __shared__ typename K::Shared sm;
    const int share = blockIdx.x;
    int seq;
    int64_t within, total;
    auto units = [&](int b) -> int64_t { return (int64_t)SplitRange<K::kStep>(a, b).steps * sp.tiles_per_seq; };
    auto first = [&](int64_t n) { return share_start(share, n, share_count(n, sp.shares)); };
    if (!locate_unit<kAttnThreads>(a.pages.n_seqs, first, units, sm.located, seq, within, total)) return;
    const int64_t begin = first(total), end = share_start(share + 1, total, share_count(total, sp.shares));
    const int tiles_per_head = sp.tiles_per_seq / a.pages.n_kv;
    for (int64_t u = begin; u < end; ++seq, within = 0) {
        const SplitRange<K::kStep> r(a, seq);
        if (r.len > a.pages.capacity && a.bad != nullptr && threadIdx.x == 0) *a.bad = 1;
        for (; u < end && within < (int64_t)r.steps * sp.tiles_per_seq;) {
            const int tile = (int)((double)within / (double)r.steps);
            const uint32_t step = (uint32_t)(within - (int64_t)tile * r.steps);
            uint32_t n = r.steps - step;
            if ((int64_t)n > end - u) n = (uint32_t)(end - u);
            Tile t;
            t.seq = t.row0 = seq;
            t.h = tile / tiles_per_head;
            t.first = 16 * (tile - t.h * tiles_per_head);
            t.rows = a.group;
            t.pos0 = r.len - 1;
            uint32_t lo = r.start + step * K::kStep, hi = lo + n * K::kStep;
            if (lo < r.lo) lo = r.lo;
            if (hi > r.hi) hi = r.hi;
            if (step == 0 && threadIdx.x == 0) {  // the share that begins a tile names its parts
                const int64_t last = share_of(u + r.steps - 1, total, share_count(total, sp.shares));
                sp.ranges[(size_t)seq * (size_t)sp.tiles_per_seq + tile] =
                    PartRange{2 * share + (u == begin ? 0 : 1), n == r.steps ? 0 : (int)(last - share) + 1};
            }
            K k;
            if (n == r.steps) {
                k.template attend<false>(a, sm, t, lo, hi, [&](int c, int d, float, float l, f32x4 sum) {
                    const float f = l == 0.0f ? 0.0f : 1.0f / l;
#pragma unroll
                    for (int i = 0; i < 4; ++i) sum[i] = l == 0.0f ? 0.0f : sum[i] * f;
                    const size_t row = (size_t)seq * (size_t)a.nq + (size_t)(t.h * a.group + t.first + c);
                    store4_from_f32(a.out, a.dtype, row * (size_t)a.head_dim + d, sum);
                });
            } else {
                const size_t slot = 2 * (size_t)share + (u == begin ? 0 : 1);
                k.template attend<false>(a, sm, t, lo, hi, [&](int c, int d, float m, float l, f32x4 sum) {
                    const size_t row = slot * (size_t)sp.cols + (size_t)c;
                    *reinterpret_cast<f32x4*>(sp.part + row * (size_t)a.head_dim + d) = sum;
                    if (d == 0) {
                        float* ml = sp.part + 2 * (size_t)sp.shares * (size_t)sp.cols * (size_t)a.head_dim + 2 * row;
                        ml[0] = m;
                        ml[1] = l;
                    }
                });
            }
            u += n;
            within += n;
        }
    }
}

// One block per (sequence, tile), where the table holds too few keys for a split to gain what its second launch costs.
template <typename K>
__global__ __launch_bounds__(kAttnThreads, K::kBlocksPerCu) void paged_whole_kernel(AttnArgs a, int tiles_per_seq) {
    __shared__ typename K::Shared sm;
    const int seq = blockIdx.x / tiles_per_seq, tile = blockIdx.x - seq * tiles_per_seq;
    const int tiles_per_head = tiles_per_seq / a.pages.n_kv;
    const SplitRange<K::kStep> r(a, seq);
    if (r.len > a.pages.capacity && a.bad != nullptr && threadIdx.x == 0) *a.bad = 1;
    Tile t;
    t.seq = t.row0 = seq;
    t.h = tile / tiles_per_head;
    t.first = 16 * (tile - t.h * tiles_per_head);
    t.rows = a.group;
    t.pos0 = r.len - 1;
    K k;
    k.template attend<false>(a, sm, t, r.lo, r.hi, [&](int c, int d, float, float l, f32x4 sum) {
        const float f = l == 0.0f ? 0.0f : 1.0f / l;
#pragma unroll
        for (int i = 0; i < 4; ++i) sum[i] = l == 0.0f ? 0.0f : sum[i] * f;
        const size_t row = (size_t)seq * (size_t)a.nq + (size_t)(t.h * a.group + t.first + c);
        store4_from_f32(a.out, a.dtype, row * (size_t)a.head_dim + d, sum);
    });
}

// One block per (sequence, query head): nothing where one share held its tile, else the sum of its parts, 4 channels a
// thread and the parts over as many threads as that leaves.
__global__ __launch_bounds__(kAttnThreads) void paged_join_kernel(AttnArgs a, SplitArgs sp) {
    __shared__ f32x4 sums[kAttnThreads];
    __shared__ float totals[kAttnThreads], tops[kAttnThreads];
    const uint32_t q_row = blockIdx.x, tid = threadIdx.x;
    const uint32_t seq = q_row / (uint32_t)a.nq, head = q_row - seq * (uint32_t)a.nq;
    const uint32_t h = head / (uint32_t)a.group, in_group = head - h * (uint32_t)a.group;
    const uint32_t tiles_per_head = (uint32_t)(sp.tiles_per_seq / a.pages.n_kv);
    const PartRange range = sp.ranges[(size_t)seq * (size_t)sp.tiles_per_seq + h * tiles_per_head + in_group / 16];
    if (range.count == 0) return;
    const uint32_t c = in_group % 16, lanes = (uint32_t)a.head_dim / 4, ways = kAttnThreads / lanes, way = tid / lanes;
    const uint32_t x = 4 * (tid - way * lanes);
    // Part i of a tile is its first share's slot, then the first slots of the shares after it.
    auto row_of = [&](int i) { return (size_t)(i == 0 ? range.first : (range.first & ~1) + 2 * i) * (size_t)sp.cols + c; };
    const float* ml = sp.part + 2 * (size_t)sp.shares * (size_t)sp.cols * (size_t)a.head_dim;
    float top = kNegInf, l = 0.0f;
    f32x4 sum = {0, 0, 0, 0};
    if (way < ways) {
        // In groups of four, whose loads are in flight together.
        for (int i0 = (int)way; i0 < range.count; i0 += 4 * (int)ways) {
            float m4[4], l4[4];
            f32x4 s4[4];
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const int i = i0 + k * (int)ways;
                const size_t row = row_of(i < range.count ? i : i0);
                m4[k] = ml[2 * row];
                l4[k] = ml[2 * row + 1];
                s4[k] = *reinterpret_cast<const f32x4*>(sp.part + row * (size_t)a.head_dim + x);
                if (i >= range.count) m4[k] = kNegInf;
            }
            const float t4 = fmaxf(fmaxf(fmaxf(m4[0], m4[1]), fmaxf(m4[2], m4[3])), top);
            const float ref = t4 == kNegInf ? 0.0f : t4, f = exp2_hw(top - ref);
            l *= f;
#pragma unroll
            for (int y = 0; y < 4; ++y) sum[y] *= f;
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const float w = exp2_hw(m4[k] - ref);
                l = __builtin_fmaf(l4[k], w, l);
#pragma unroll
                for (int y = 0; y < 4; ++y) sum[y] = __builtin_fmaf(s4[k][y], w, sum[y]);
            }
            top = t4;
        }
    }
    sums[tid] = sum;
    totals[tid] = l;
    tops[tid] = top;
    __syncthreads();
    if (way != 0) return;
    for (uint32_t w = 0; w < ways; ++w) top = fmaxf(top, tops[w * lanes + tid]);
    l = 0.0f;
    sum = f32x4{0, 0, 0, 0};
    for (uint32_t w = 0; w < ways; ++w) {
        const uint32_t i = w * lanes + tid;
        const float f = tops[i] == kNegInf ? 0.0f : exp2_hw(tops[i] - top);
        l = __builtin_fmaf(totals[i], f, l);
#pragma unroll
        for (int y = 0; y < 4; ++y) sum[y] = __builtin_fmaf(sums[i][y], f, sum[y]);
    }
    const float f = l == 0.0f ? 0.0f : 1.0f / l;
#pragma unroll
    for (int i = 0; i < 4; ++i) sum[i] = l == 0.0f ? 0.0f : sum[i] * f;
    store4_from_f32(a.out, a.dtype, (size_t)q_row * (size_t)a.head_dim + x, sum);
}

// The kernel of a cache type, the narrowest that holds head_dim.
template <typename TC, bool HIGH, typename F>
int with_tile_kernel(int head_dim, F&& f) {
    if (head_dim == 64) return f(TileKernel<TC, 64, true, HIGH>{});
    if (head_dim == 128) return f(TileKernel<TC, 128, true, HIGH>{});
    if (head_dim == 256) return f(TileKernel<TC, 256, true, HIGH>{});
    if (head_dim < 64) return f(TileKernel<TC, 64, false, HIGH>{});
    if (head_dim < 128) return f(TileKernel<TC, 128, false, HIGH>{});
    return f(TileKernel<TC, 256, false, HIGH>{});
}

}  // namespace

// Chunks over caches of a half type (attention_prompt.hip).
constexpr int kPromptRows = 128;
int launch_prompt(const AttnArgs& a, int cache_dtype, unsigned blocks, const ChunkSplit& sp, hipStream_t s) __attribute__((visibility("hidden")));

// The checks of both entry points; fills `a`.
int attn_args(AttnArgs& a, const void* q, void* out, int64_t n_q_heads, int64_t n_kv_heads, int dtype, const int32_t* cu_q,
              const int32_t* seq_lens, const int32_t* block_table, int64_t n_seqs, int64_t max_pages, int64_t n_rows,
              int64_t head_dim, const void* kcache, const void* vcache, int cache_dtype, int64_t n_pages,
              int64_t page_size, float scale, float softcap, int64_t window, const float* slopes,
              const int32_t* prefix_lens, int32_t* bad) __attribute__((visibility("hidden")));

}  // namespace sph
