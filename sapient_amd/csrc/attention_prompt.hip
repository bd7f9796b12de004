// attention_prompt.hip — the kernel of chunks over caches of a half type: 128 rows a block (mathematics and
// the argument block: attention.h).
//
// Four waves of 32 columns (rows of q: tokens and the query heads of one kv head, so that a block reads its keys once
// for the whole group) share steps of 64 keys through LDS, on 32x32x16 matrix instructions. Scores are transposed
// (S^T = K Q^T) as in the 16-column kernel: lane (j = lane % 32, h = lane / 32) holds column j's scores of tokens 8b +
// 4h + 0..3, which is the order in which it feeds them back as the second operand, so weights never leave their lane.
// K and V lie in LDS as they come, rows of DP channels in 16-byte pieces, piece c of row r at c ^ swap(r), so that what a
// read touches at once (a piece of 8 and of 16 neighbouring rows of K; of V, 32 bytes of 4 neighbouring rows, and 64) lies
// in different banks. They go there straight from
// memory (16 bytes a lane; a wave's lanes fill 1 KB in a row, so the swap is in which piece a lane asks for), into the
// other of two buffers while a step is computed: no registers hold them, no instruction moves them. V is read
// transposed (ds_read_b64_tr_b16: of 4 rows by 16 channels, a channel's 4 values to a lane). One barrier a step.
//
// What bounds it: per step and wave 32 products of 32 cycles and some 240 vector instructions (of which 32 exponentials),
// and the two waves of a SIMD hardly overlap them: matrix cores busy 41 % of the time, vector units 46 %. Ragged prompts of
// 10033 tokens, 32 + 8 heads x 128 bf16: 331 to 345 us by machine, 880 TFLOP/s of the products that the masks leave (a
// library product of 8192^3 1340). By step: K and V through registers 423, straight to LDS 368, reads ahead 358, swapped
// pieces 331; raised wave priority around the products, and scalar addresses, gained nothing.
#include "attention.h"

namespace sph {
namespace {

constexpr int kPromptKeys = 64;

template <typename TC>
__device__ __forceinline__ f32x16 mma32(u32x4 a, u32x4 b, f32x16 c) {
    if constexpr (__is_same(TC, f16))
        return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(h8, a), __builtin_bit_cast(h8, b), c, 0, 0, 0);
    else
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(b8, a), __builtin_bit_cast(b8, b), c, 0, 0, 0);
}

typedef short s4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) s4 lds_s4;

// 16 bytes a lane from `from` to LDS at `to` (the wave's, its lanes in a row).
__device__ __forceinline__ void to_lds(const void* from, void* to) {
    __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)from, (__attribute__((address_space(3))) void*)to,
                                     16, 0, 0);
}

// The order of the N operands just written, READS reads each, and their PRODUCTS products each: the reads run six operands
// ahead. Left alone, the scheduler reads for one product at a time and waits out LDS's latency before each.
template <int N, int READS, int PRODUCTS>
__device__ __forceinline__ void ahead_of_products() {
    constexpr int kAhead = 6, kMatrix = 0x008, kRead = 0x100;
    __builtin_amdgcn_sched_group_barrier(kRead, kAhead * READS, 0);
#pragma unroll
    for (int i = 0; i < N - kAhead; ++i) {
        __builtin_amdgcn_sched_group_barrier(kMatrix, PRODUCTS, 0);
        __builtin_amdgcn_sched_group_barrier(kRead, READS, 0);
    }
    __builtin_amdgcn_sched_group_barrier(kMatrix, kAhead * PRODUCTS, 0);
}

template <int CH>
__device__ __forceinline__ constexpr int swap_k(int row) { return CH == 8 ? (row ^ (row >> 3 & 1)) & 7 : row & 15; }
template <int CH>
__device__ __forceinline__ constexpr int swap_v(int row) { return CH == 8 ? 2 * (row & 3) : 2 * (row & 3) ^ 8 * (row & 1); }

template <typename TC, int DP>
struct PromptShared {
    alignas(16) uint16_t k[2][kPromptKeys * DP];
    alignas(16) uint16_t v[2][kPromptKeys * DP];
    uint64_t odd[2][kAttnWaves];  // the keys of each buffer whose V had a value that is not finite (of edge steps), by finder
    Located located;
};

// EXACT: head_dim is DP. HIGH: q is f32, or another half type than the cache; its pieces take the registers of a second
// block a CU where rows are wider than 64.
constexpr int prompt_blocks(int DP, bool HIGH) { return DP > 128 || (HIGH && DP > 64) ? 1 : 2; }
template <typename TC, int DP, bool EXACT, bool HIGH>
__global__ __launch_bounds__(kAttnThreads, prompt_blocks(DP, HIGH)) void paged_prompt_kernel(AttnArgs a, ChunkSplit sp) {
    __shared__ PromptShared<TC, DP> sm;
    constexpr int KS = DP / 16;                    // k steps of a score
    constexpr int DB = DP / 32;                    // blocks of channels
    constexpr int CH = DP / 8;                     // 16-byte pieces of a row
    constexpr int PL = kPromptKeys * CH / kAttnThreads;  // pieces of K, and of V, per thread and step
    constexpr int NQ = Pieces<TC, HIGH>::q, NP = HIGH ? Pieces<TC, HIGH>::high : 1;
    constexpr float kLift = __is_same(TC, f16) ? 7.0f : 0.0f;
    const int tid = threadIdx.x, wave = tid / kWave, lane = tid % kWave, j = lane % 32, h = lane / 32;
    const int D = EXACT ? DP : a.head_dim;

    Tile t;
    ChunkPart part;
    if (!chunk_tile<kPromptRows, kPromptKeys>(a, sp, sm.located, t, part)) return;
    const uint32_t lo = part.lo, hi = part.hi;

    // This lane's column, and the positions of the wave's.
    const int wave_first = t.first + 32 * wave;
    const int n_cols = t.rows - wave_first < 32 ? t.rows - wave_first : 32;  // may be 0 and less
    const int col = wave_first + j < t.rows ? wave_first + j : t.rows - 1;
    const int tok = col / a.group, head = t.h * a.group + (col - tok * a.group), pos = t.pos0 + tok;
    const int pos_first = t.pos0 + wave_first / a.group;
    const int pos_last = t.pos0 + (wave_first + (n_cols > 0 ? n_cols : 1) - 1) / a.group;
    const int prefix = a.prefix != nullptr ? a.prefix[t.seq] : 0;
    const size_t q_row = (size_t)(t.row0 + tok) * (size_t)a.nq + (size_t)head;

    u32x4 q[NQ][KS];
    float scale = a.scale;
    if constexpr (!HIGH) {
#pragma unroll
        for (int s = 0; s < KS; ++s) {
            const int d = 16 * s + 8 * h;
            q[0][s] = u32x4{0, 0, 0, 0};
            if (EXACT || d < D) q[0][s] = *reinterpret_cast<const u32x4*>(static_cast<const TC*>(a.q) + q_row * (size_t)D + d);
        }
    } else {
        float f[KS][8], most = 0.0f;
        load_row_f32(a.q, a.dtype, q_row * (size_t)D, 8 * h, 16, D, f);
#pragma unroll
        for (int s = 0; s < KS; ++s)
#pragma unroll
            for (int e = 0; e < 8; ++e) most = fmaxf(most, fabsf(f[s][e]));
        most = fmaxf(most, __shfl_xor(most, 32));
        scale = ldexpf(scale, split_row<TC>(f, most, q));
    }
    const ScoreForm<HIGH> form(a, scale, head);

    const TC *kc = static_cast<const TC*>(a.kc), *vc = static_cast<const TC*>(a.vc);
    const uint32_t head_rows = (uint32_t)t.h * a.pages.page.d;
    // The table's entry for key t0 + lane, asked for two steps ahead, and the key's pool row.
    auto entry_at = [&](uint32_t t0) { return a.pages.entry(t.seq, t0 + (uint32_t)lane < hi ? t0 + (uint32_t)lane : hi - 1); };
    auto row_at = [&](uint32_t t0, uint32_t id) -> uint32_t {
        const uint32_t k = t0 + (uint32_t)lane;
        const uint32_t r = a.pages.row_in(id, k < hi ? k : hi - 1);
        if (k >= lo && k < hi && r == kNoRow && a.bad != nullptr) *a.bad = 1;
        return k < hi && r != kNoRow ? r + head_rows : kNoRow;
    };
    auto is_key = [&](uint32_t t0, uint32_t rows) { return __ballot(rows != kNoRow && t0 + (uint32_t)lane >= lo); };
    const bool by_16 = a.pages.page.d % 16 == 0;  // 16 neighbouring keys share a page
    const int wave_u = __builtin_amdgcn_readfirstlane(wave);
    // The row of the step's key 16 block + i; rows of lanes in one block follow its first.
    auto pool_row = [&](uint32_t rows, int block, int i) -> uint32_t {
        uint32_t r;
        if (by_16) {
            r = __builtin_amdgcn_readlane(rows, 16 * block);
            return (r == kNoRow ? 0u : r) + (uint32_t)i;
        }
        r = __shfl(rows, 16 * block + i);
        return r == kNoRow ? 0u : r;
    };
    // A step's rows of K and V on their way to LDS. Row 0 stands in for a missing one: its scores are masked, and as V it
    // is cleared when it has arrived, since 0 · inf is not 0. Channels past D are not asked for; they are zeros from
    // the start.
    auto load_step = [&](uint32_t rows, int buf) {
#pragma unroll
        for (int i = 0; i < PL; ++i) {
            const int piece = i * kAttnThreads + tid, row = piece / CH, c = piece % CH;
            const int dk = 8 * (c ^ swap_k<CH>(row)), dv = 8 * (c ^ swap_v<CH>(row));
            const int block = (i * kAttnThreads + wave_u * kWave) / CH / 16;  // the wave's rows lie in one
            const size_t at = (size_t)pool_row(rows, block, row % 16) * (size_t)D;
            const int to = 8 * (i * kAttnThreads + wave_u * kWave);
            if (EXACT || dk < D) to_lds(kc + at + dk, &sm.k[buf][to]);
            if (EXACT || dv < D) to_lds(vc + at + dv, &sm.v[buf][to]);
        }
    };
    // Whether all the block's rows see all of the step's keys.
    const int block_first = t.pos0 + t.first / a.group;
    const int block_last = t.pos0 + ((t.first + kPromptRows < t.rows ? t.first + kPromptRows : t.rows) - 1) / a.group;
    auto all_see = [&](uint64_t there, int t0) {
        const int last = t0 + kPromptKeys - 1;
        return there == ~uint64_t(0) && block_first >= 0 && (last <= block_first || last < prefix) &&
               (a.window == 0 || block_last - t0 < a.window);
    };
    auto arrive = [&](uint64_t there, uint32_t t0, int buf) {
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        uint64_t odd = 0;
        if (!all_see(there, (int)t0)) {
#pragma unroll 1
            for (int i = 0; i < PL; ++i) {
                const int piece = i * kAttnThreads + tid;
                u32x4* p = reinterpret_cast<u32x4*>(&sm.v[buf][8 * piece]);
                const u32x4 w = *p;
                const bool key = (there >> (piece / CH)) & 1;
                if (!key || not_finite<TC>(w[0]) || not_finite<TC>(w[1]) || not_finite<TC>(w[2]) || not_finite<TC>(w[3])) {
                    *p = u32x4{0, 0, 0, 0};
                    if (key) odd |= uint64_t(1) << (piece / CH);
                }
            }
            if (__any(odd != 0)) {
#pragma unroll
                for (int d = 1; d < kWave; d <<= 1) odd |= __shfl_xor(odd, d);
            }
        }
        if (lane == 0) sm.odd[buf][wave] = odd;
    };
    if constexpr (!EXACT) {
        for (int i = tid; i < 2 * kPromptKeys * CH; i += kAttnThreads) {
            reinterpret_cast<u32x4*>(sm.k)[i] = u32x4{0, 0, 0, 0};
            reinterpret_cast<u32x4*>(sm.v)[i] = u32x4{0, 0, 0, 0};
        }
        __syncthreads();
    }
    const int v_row = 4 * h + lane % 16 / 4, v_chunk = 2 * (lane / 16 % 2) + lane % 4 / 2;
    auto read_v = [&](int buf, int d, int i) {  // channels 32 d + j, slots of keys 16 i
        u32x4 x;
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            const uint16_t* p = &sm.v[buf][(16 * i + 8 * e + v_row) * DP + 8 * ((4 * d + v_chunk) ^ swap_v<CH>(v_row)) + 4 * (lane % 2)];
            const u32x2 w = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4*)p));
            x[2 * e] = w[0];
            x[2 * e + 1] = w[1];
        }
        return x;
    };

    float m = kNegInf, l = 0.0f;
    f32x16 acc[DB];
#pragma unroll
    for (int d = 0; d < DB; ++d)
#pragma unroll
        for (int r = 0; r < 16; ++r) acc[d][r] = 0.0f;

    const bool plain = a.cap == 0.0f && a.slopes == nullptr && a.scale > 0.0f;
    const float unit = plain ? scale * kLog2e : 1.0f;  // scores to log2 units, where nothing has to be done to them

    uint32_t t0 = part.start;
    const uint32_t end = part.end;  // steps [start, end) of 64 keys
    uint32_t rows = kNoRow, id_next = 0;
    if (t0 < end) {
        const uint32_t id = entry_at(t0);
        id_next = entry_at(t0 + kPromptKeys);
        rows = row_at(t0, id);
        load_step(rows, 0);
        arrive(is_key(t0, rows), t0, 0);
    }
    __syncthreads();
    for (int buf = 0; t0 < end; t0 += kPromptKeys, buf ^= 1) {
        const bool more = t0 + kPromptKeys < end;
        const uint32_t rows_next = row_at(t0 + kPromptKeys, id_next);
        id_next = entry_at(t0 + 2 * kPromptKeys);
        if (more) load_step(rows_next, buf ^ 1);

        const uint64_t there = is_key(t0, rows);
        const int last = (int)t0 + kPromptKeys - 1;
        const bool none = n_cols <= 0 || (pos_last < (int)t0 && prefix <= (int)t0) ||
                          (a.window > 0 && pos_first - last >= a.window);
        if (!none) {
            f32x16 s[2];
#pragma unroll
            for (int b = 0; b < 2; ++b)
#pragma unroll
                for (int r = 0; r < 16; ++r) s[b][r] = 0.0f;
            // (Two chains of products side by side: each waits for its own last one.)
#pragma unroll
            for (int c = 0; c < KS; ++c)
#pragma unroll
                for (int b = 0; b < 2; ++b) {
                    const int row = 32 * b + j;
                    const u32x4 k = *reinterpret_cast<const u32x4*>(&sm.k[buf][row * DP + 8 * ((2 * c + h) ^ swap_k<CH>(j))]);
#pragma unroll
                    for (int p = NQ - 1; p >= 0; --p) s[b] = mma32<TC>(k, q[p][c], s[b]);
                }
            ahead_of_products<2 * KS, 1, NQ>();
            const bool seen = all_see(there, (int)t0);
            if (!plain) {
#pragma unroll
                for (int b = 0; b < 2; ++b) {
                    float x[16];
#pragma unroll
                    for (int r = 0; r < 16; ++r) x[r] = s[b][r];
                    form.apply(a, x, (float)(pos - (int)t0 - 32 * b - 4 * h), [](int r) { return 8 * (r / 4) + r % 4; });
#pragma unroll
                    for (int r = 0; r < 16; ++r) s[b][r] = x[r];
                }
            }
            if (!seen) {
                const uint64_t see = visible(there, (int)t0, pos, prefix, a.window) >> (4 * h);
#pragma unroll
                for (int b = 0; b < 2; ++b)
#pragma unroll
                    for (int r = 0; r < 16; ++r)
                        s[b][r] = (uint32_t)(see >> (32 * b)) & (1u << (8 * (r / 4) + r % 4)) ? s[b][r] : kNegInf;
                const uint64_t odd = (sm.odd[buf][0] | sm.odd[buf][1] | sm.odd[buf][2] | sm.odd[buf][3]) >> (4 * h) & see;
                if (__any(odd != 0)) {
#pragma unroll
                    for (int b = 0; b < 2; ++b)
#pragma unroll
                        for (int r = 0; r < 16; ++r)
                            s[b][r] = (uint32_t)(odd >> (32 * b)) & (1u << (8 * (r / 4) + r % 4)) ? __builtin_nanf("") : s[b][r];
                }
            }
            float top = s[0][0];
#pragma unroll
            for (int b = 0; b < 2; ++b)
#pragma unroll
                for (int r = 0; r < 16; ++r) top = fmaxf(top, s[b][r]);
            top *= unit;
            if (__any(top > m + (kLift + kSlack))) {
                top = fmaxf(top, __shfl_xor(top, 32));
                const float m_new = fmaxf(m, top - kLift);
                const float f = m_new == kNegInf ? 1.0f : exp2_hw(m - m_new);
                m = m_new;
                l *= f;
#pragma unroll
                for (int d = 0; d < DB; ++d)
#pragma unroll
                    for (int r = 0; r < 16; ++r) acc[d][r] *= f;
            }
            const float ref = m == kNegInf ? 0.0f : m;
            u32x4 p[NP][4];
#pragma unroll
            for (int b = 0; b < 2; ++b)
#pragma unroll
                for (int r = 0; r < 16; r += 2) {
                    float x = exp2_hw(__builtin_fmaf(s[b][r], unit, -ref)), y = exp2_hw(__builtin_fmaf(s[b][r + 1], unit, -ref));
                    l += x + y;
#pragma unroll
                    for (int c = 0; c < NP; ++c) {
                        const uint32_t w = narrow2<TC>(x, y);
                        p[c][2 * b + r / 8][r % 8 / 2] = w;
                        if (c + 1 < NP) {
                            x -= widen_half<TC>(w, 0);
                            y -= widen_half<TC>(w, 1);
                        }
                    }
                }
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int d = 0; d < DB; ++d) {
                    const u32x4 v = read_v(buf, d, i);
#pragma unroll
                    for (int c = NP - 1; c >= 0; --c) acc[d] = mma32<TC>(v, p[c][i], acc[d]);
                }
            ahead_of_products<4 * DB, 2, NP>();
        }
        if (more) arrive(is_key(t0 + kPromptKeys, rows_next), t0 + kPromptKeys, buf ^ 1);
        rows = rows_next;
        __syncthreads();
    }

    l += __shfl_xor(l, 32);
    if (j >= n_cols) return;
    if (sp.splits == 1) {
        const float f = l == 0.0f ? 0.0f : 1.0f / l;
#pragma unroll
        for (int d = 0; d < DB; ++d)
#pragma unroll
            for (int r = 0; r < 16; r += 4) {
                const int ch = 32 * d + 2 * r + 4 * h;
                f32x4 o;
#pragma unroll
                for (int i = 0; i < 4; ++i) o[i] = l == 0.0f ? 0.0f : acc[d][r + i] * f;
                if (EXACT || ch < D) store4_from_f32(a.out, a.dtype, q_row * (size_t)D + ch, o);
            }
    } else {
#pragma unroll
        for (int d = 0; d < DB; ++d)
#pragma unroll
            for (int r = 0; r < 16; r += 4) {
                const int ch = 32 * d + 2 * r + 4 * h;
                if (EXACT || ch < D) chunk_part_sum(a, sp, part.split, q_row, ch, f32x4{acc[d][r], acc[d][r + 1], acc[d][r + 2], acc[d][r + 3]});
            }
        if (h == 0) chunk_part_ml(a, sp, part.split, q_row, m, l);
    }
}

template <typename TC, bool HIGH>
int launch_prompt_of(const AttnArgs& a, unsigned blocks, const ChunkSplit& sp, hipStream_t s) {
    auto go = [&](auto kernel) { return launch(kernel, dim3(blocks), kAttnThreads, s, a, sp); };
    switch (a.head_dim) {
    case 64: return go(paged_prompt_kernel<TC, 64, true, HIGH>);
    case 128: return go(paged_prompt_kernel<TC, 128, true, HIGH>);
    case 256: return go(paged_prompt_kernel<TC, 256, true, HIGH>);
    default:
        return a.head_dim < 64    ? go(paged_prompt_kernel<TC, 64, false, HIGH>)
               : a.head_dim < 128 ? go(paged_prompt_kernel<TC, 128, false, HIGH>)
                                  : go(paged_prompt_kernel<TC, 256, false, HIGH>);
    }
}

}  // namespace

int launch_prompt(const AttnArgs& a, int cache_dtype, unsigned blocks, const ChunkSplit& sp, hipStream_t s) {
    auto of = [&](auto tc) {
        using TC = decltype(tc);
        return a.dtype == cache_dtype ? launch_prompt_of<TC, false>(a, blocks, sp, s) : launch_prompt_of<TC, true>(a, blocks, sp, s);
    };
    return cache_dtype == SPH_F16 ? of(f16{}) : of(bf16{});
}

}  // namespace sph
