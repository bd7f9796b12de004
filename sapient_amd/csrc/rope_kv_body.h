// rope_kv_body.h — the body of the fused step's kernels (rope_kv.h): Args a, its types T and TC, and P, INTERLEAVED, TM, U,
// BIAS and NT are the including kernel's.
    __shared__ uint32_t inv_pio4[24];
    __shared__ float cs_s[kMaxBlockAngles], sn_s[kMaxBlockAngles];
    // All arguments are asked for here: left to the branches that use them, their scalar loads form a chain of cache
    // misses, which a decode step waits for longer than for its rows (the engine's step, 24 launches of this: 334 ->
    // 321 us a token).
    asm volatile("" ::"s"(a.q), "s"(a.qo), "s"(a.k), "s"(a.v), "s"(a.kc), "s"(a.vc), "s"(a.pos), "s"(a.bias[0]),
                 "s"(a.bias[1]), "s"(a.bias[2]), "s"(a.bias_dt), "s"(a.nq), "s"(a.nkv), "s"(a.seq), "s"(a.max_seq),
                 "s"(a.head_dim), "s"(a.half), "s"(a.lanes), "s"(a.toks), "s"(a.heads), "s"(a.h_first), "s"(a.s_first),
                 "s"(a.pos_scale), "s"(a.bad), "s"(a.ang), "s"((int)a.ang_by_pos), "s"(a.by_lanes), "s"(a.by_toks), "s"(a.by_heads));
    const int tid = threadIdx.x;
    const int rho = quotient(tid, a.by_lanes), lit = tid - rho * a.lanes;
    // Neighbouring rows in memory: heads (TM), else tokens.
    const int major = quotient(rho, TM ? a.by_heads : a.by_toks), minor = rho - major * (TM ? a.heads : a.toks);
    const int tl = TM ? major : minor, hl = TM ? minor : major;
    const int64_t s0 = a.s_first + (int64_t)blockIdx.x * a.toks, s = s0 + tl;
    const bool active = rho < a.toks * a.heads && s < a.seq;
    const int h0 = a.h_first + (int)blockIdx.y * a.heads * U + hl, H = a.nq + a.nkv;
    const int i0 = lit * P;
    using Runs = PairRuns<T, P, INTERLEAVED, NT>;

    const bool eval = a.ang == nullptr, per_token = !eval && !a.ang_by_pos;
    constexpr bool kOwn = P == 1;  // a thread's one angle: no exchange (3 tokens of 14 + 2 x 64: 2.87 -> 2.66 us)
    // Clamped, not predicated: a load in a branch is waited for at its end where its value is converted there.
    auto pos_at = [&](int64_t t) { return a.pos[t < a.seq ? t : a.seq - 1]; };
    int32_t ps = 0, cu_word = INT32_MAX, len_word = 0, cu_first = 0;
    if constexpr (!Args::kPaged) {
        ps = pos_at(s);
    } else if (a.pages.cu != nullptr) {
        const int n = a.pages.n_seqs, i = n <= kWave ? tid % kWave : tid, at = i < n ? i : n - 1;
        cu_word = a.pages.cu[1 + at];
        len_word = a.pages.lens[at];
        cu_first = a.pages.cu[0];
    } else {
        ps = a.pages.lens[s < a.seq ? s : a.seq - 1] - 1;
    }
    // Angle number tid of the block.
    const int pair = eval && !kOwn ? quotient(tid, a.by_toks) : 0, tk = tid - pair * a.toks;
    const bool has_angle = eval && !kOwn && pair < a.half;
    int32_t apos = ps;
    if constexpr (!kOwn && !Args::kPaged) apos = pos_at(s0 + tk);
    if constexpr (!kOwn && Args::kPaged) {
        if (a.pages.cu == nullptr) apos = a.pages.lens[s0 + tk < a.seq ? s0 + tk : a.seq - 1] - 1;
    }
    uint32_t tab_word = 0;
    float den = 1.0f;
    if (eval) {
        tab_word = kInvPio4.w[tid < 24 ? tid : 0];
        den = a.den.v[kOwn ? i0 : pair < a.half ? pair : 0];
    }

    // Row (head h, token s) of a [heads, seq, hd] (or, TM, [seq, heads, hd]) tensor.
    auto row_of = [&](const T* base, int heads, int h) {
        return base + (TM ? (size_t)s * (size_t)heads + (size_t)h : (size_t)h * (size_t)a.seq + (size_t)s) *
                          (size_t)a.head_dim;
    };
    // Everything the rows need is requested before anything is waited for: the position, the angles where the
    // caller supplies them per token, the rows and the biases of their channels.
    float ag[2 * P];
    if (per_token && active) load_angles<P>(a.ang + 2 * ((size_t)s * (size_t)a.half + (size_t)i0), ag);
    Runs x[U], w[U];  // the q or k row, and the v row
    using BiasRuns = BiasRun<Runs::L>[BIAS ? U : 1][Runs::R];
    BiasRuns xb, wb;
    auto load_bias = [&](const void* p, int h, BiasRun<Runs::L>(&b)[Runs::R]) {
        if (p == nullptr) return;
#pragma unroll
        for (int r = 0; r < Runs::R; ++r)
            b[r].load(p, (size_t)h * (size_t)a.head_dim + (size_t)Runs::at(r, i0, a.half), a.bias_dt == SPH_F32);
    };
#pragma unroll
    for (int u = 0; u < U; ++u) {
        const int h = h0 + u * a.heads;
        if (active && h < H) {
            const bool is_q = h < a.nq;
            const int hi = is_q ? h : h - a.nq;
            x[u].load(is_q ? row_of(a.q, a.nq, hi) : row_of(a.k, a.nkv, hi), i0, a.half);
            if (!is_q) w[u].load(row_of(a.v, a.nkv, hi), i0, a.half);
            if constexpr (BIAS) {
                load_bias(is_q ? a.bias[0] : a.bias[1], hi, xb[u]);
                if (!is_q) load_bias(a.bias[2], hi, wb[u]);
            }
        }
    }

    int seq_of = (int)s;              // this row's sequence; n_seqs: none
    uint32_t crow0 = kNoRow;          // its row in the pools (kv head 0)
    if constexpr (Args::kPaged) {
        if (a.pages.cu != nullptr) {
            __shared__ int counted[kThreads / kWave];
            const int n = a.pages.n_seqs;
            if (n <= kWave) {
                const int first = __popcll(__ballot(tid % kWave < n && cu_word <= s0));
                auto locate = [&](int64_t t, int& b) {  // by all lanes of the wave
                    b = first;
                    int32_t next;
                    for (;;) {
                        next = __shfl(cu_word, b);
                        const bool on = t < a.seq && b < n && next <= t;
                        if (!__any(on)) break;
                        b += on;
                    }
                    const int64_t p = (int64_t)__shfl(len_word, b) - (next - t);
                    if (t >= a.seq || t < cu_first) b = n;
                    return b >= n || p < 0 ? -1 : (int)p;
                };
                ps = locate(s, seq_of);
                if constexpr (!kOwn) {
                    int b;
                    apos = locate(s0 + tk, b);
                }
            } else {
                int below = 0;  // cu entries at or below the block's first row
                for (int i = tid; i < n; i += blockDim.x) {
                    if (i >= (int)blockDim.x) cu_word = a.pages.cu[1 + i];
                    below += cu_word <= s0;
                }
#pragma unroll
                for (int m = 32; m > 0; m >>= 1) below += __shfl_xor(below, m);
                if (tid % kWave == 0) counted[tid / kWave] = below;
                __syncthreads();
                int first = 0;
                for (int w = 0; w < (int)blockDim.x / kWave; ++w) first += counted[w];
                auto locate = [&](int64_t t, int& b) {  // the sequence and the position of row t
                    b = first;
                    while (b < n && a.pages.cu[1 + b] <= t) ++b;
                    if (b >= n || t >= a.seq || a.pages.cu[b] > t) {
                        b = n;
                        return -1;
                    }
                    const int64_t p = a.pages.lens[b] - (a.pages.cu[b + 1] - t);
                    return p < 0 ? -1 : (int)p;
                };
                ps = locate(s, seq_of);
                if constexpr (!kOwn) {
                    int b;
                    apos = locate(s0 + tk, b);
                }
            }
        }
        if (active && ps >= 0) crow0 = a.pages.row(seq_of, (uint32_t)ps);
        if (active && lit == 0 && a.bad != nullptr) {
            // A sequence shorter than its new tokens; one of length 0 with its one row is padding.
            const bool short_seq = ps < 0 && seq_of < a.pages.n_seqs && (a.pages.cu != nullptr || ps < -1);
            if (short_seq || (ps >= 0 && crow0 == kNoRow)) *a.bad = 1;
        }
    }

    float cs[P], sn[P];
    if (eval) {
        if (tid < 24) inv_pio4[tid] = tab_word;
        __syncthreads();
        if (has_angle) {
            const float freq = ((float)apos / a.pos_scale) / den;
            glibc_sincosf_tab(freq, inv_pio4, &sn_s[tk * a.half + pair], &cs_s[tk * a.half + pair]);
        }
        if constexpr (!kOwn) __syncthreads();
        if (!active) return;
        if constexpr (kOwn) glibc_sincosf_tab(((float)ps / a.pos_scale) / den, inv_pio4, &sn[0], &cs[0]);
#pragma unroll
        for (int j = 0; j < (kOwn ? 0 : P); ++j) {
            cs[j] = cs_s[tl * a.half + i0 + j];
            sn[j] = sn_s[tl * a.half + i0 + j];
        }
    } else {
        // Angles supplied as (cos, sin) per (token, pair), or per position in a
        // table of max_seq rows. A position outside the table reads row 0 and drops it: q is
        // rotated by angle 0 (cos 1, sin 0), the caches are left alone and the flag set.
        if (!active) return;
        const bool in_table = per_token || (ps >= 0 && (int64_t)ps < a.max_seq);
        if (!per_token) load_angles<P>(a.ang + 2 * ((size_t)(in_table ? ps : 0) * (size_t)a.half + (size_t)i0), ag);
#pragma unroll
        for (int j = 0; j < P; ++j) {
            cs[j] = in_table ? ag[2 * j] : 1.0f;
            sn[j] = in_table ? ag[2 * j + 1] : 0.0f;
        }
    }
    bool pos_ok;
    if constexpr (Args::kPaged) {
        if (ps < 0) return;  // no token: its rows stay as they are
        pos_ok = crow0 != kNoRow;
    } else {
        pos_ok = ps >= 0 && (int64_t)ps < a.max_seq;
        if (!pos_ok && a.bad != nullptr && lit == 0) *a.bad = 1;
    }

    // Row values with the bias of their channels added (y + b in f32, then
    // stored in the activation type before RoPE reads it: round through T).
    auto values = [&](const Runs& raw, int which, const BiasRun<Runs::L>(&b)[Runs::R], float (&f)[2 * P]) {
        raw.to_f32(f);
        if (BIAS && a.bias[which] != nullptr) {
#pragma unroll
            for (int r = 0; r < Runs::R; ++r) {
                float t[Runs::L];
                b[r].to_f32(a.bias_dt, t);
#pragma unroll
                for (int j = 0; j < Runs::L; ++j) f[r * Runs::L + j] = widen(narrow<T>(f[r * Runs::L + j] + t[j]));
            }
        }
    };
    auto rotate = [&](float (&f)[2 * P]) {
#pragma unroll
        for (int j = 0; j < P; ++j) {
            const int A = INTERLEAVED ? 2 * j : j, B = INTERLEAVED ? 2 * j + 1 : P + j;
            const float xa = f[A], xb = f[B];
            f[A] = xa * cs[j] - xb * sn[j];
            f[B] = xb * cs[j] + xa * sn[j];
        }
    };
#pragma unroll
    for (int u = 0; u < U; ++u) {
        const int h = h0 + u * a.heads;
        if (h >= H) return;
        float f[2 * P];
        if (h < a.nq) {
            values(x[u], 0, xb[BIAS ? u : 0], f);
            rotate(f);
            const size_t qrow = Args::kPaged ? (size_t)s * (size_t)a.nq + (size_t)h : (size_t)h * (size_t)a.seq + (size_t)s;
            Runs::store(a.qo + qrow * (size_t)a.head_dim, i0, a.half, f);
        } else if (pos_ok) {
            const int hk = h - a.nq;
            size_t crow;
            if constexpr (Args::kPaged) crow = ((size_t)crow0 + (size_t)hk * a.pages.page.d) * (size_t)a.head_dim;
            else crow = ((size_t)hk * (size_t)a.max_seq + (size_t)ps) * (size_t)a.head_dim;
            values(x[u], 1, xb[BIAS ? u : 0], f);
            rotate(f);
            // The unfused sequence stores rotated k in the activation type
            // before converting it to the cache type: round through T first.
            if constexpr (!std::is_same<T, float>::value) {
#pragma unroll
                for (int j = 0; j < 2 * P; ++j) f[j] = widen(narrow<T>(f[j]));
            }
            Runs::store(a.kc + crow, i0, a.half, f);
            values(w[u], 2, wb[BIAS ? u : 0], f);
            Runs::store(a.vc + crow, i0, a.half, f);  // v: the same channels, moved unrotated
        }
    }
