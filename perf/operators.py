"""Serving with a paged key-value cache, as measurable cases: appending a step's keys and values to the pages with RoPE
on the way, attention of one new token per sequence over the pages, and attention of prompt chunks over them.

A case is a dict of plain values; ``prepare`` makes what a serving program holds before the call, ``run`` is one pass
(plain torch in f32, or with ``own`` the calls of ``sapient_amd.ops``), ``exact`` the same results in 64 bits.

Common to all: sequence b has ``seq_lens[b]`` tokens in the cache, the new ones included; token t of it is row t % page of
page ``block_table[b, t // page]`` of the pools [pages, kv_heads, page, head_dim]. The new tokens are rows
cu_q[b] .. cu_q[b + 1] of q (one row per sequence where there is no cu_q), the last of them at position seq_lens[b] - 1.

  append  q, k [rows, heads, head_dim] plus biases rotated by their positions' angles, the angle in f32 by the reference's
          definition (pos / base^(2i/d)); k and v plus bias to the pages.
  decode  softmax attention of one row per sequence: s = scale q.k, capped (cap tanh(s / cap)), less slope * distance, over
          the last ``window`` keys (0: all); no keys: zeros.
  chunk   the same for ragged prompts: a row sees its own sequence's keys up to its position, and all below prefix_lens[b].
"""
import numpy as np
import torch

own = False

DTYPE = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
THETA = {64: 1e6, 80: 1e4, 128: 5e5, 256: 1e4}

# (heads, kv_heads, head_dim): decoder shapes of this repository's benchmark and tests, and generic ones (several query
# heads over one of 256; more query heads per key head than a matrix tile has columns)
SHAPES = [(14, 2, 64), (32, 8, 128), (32, 8, 64), (28, 4, 128), (32, 32, 80), (8, 1, 256), (24, 1, 128)]


def _case(kind, shape, seqs, length, dtype, cache=None, page=16, **more):
    """length: the longest sequence's tokens; new: the most new tokens of a sequence; ragged: sequences of different
    lengths; pad: sequences without a token at the end of the batch."""
    c = dict(kind=kind, heads=shape[0], kv_heads=shape[1], head_dim=shape[2], seqs=seqs, length=length, new=1, ragged=seqs > 1,
             pad=0, mix=1, page=page, dtype=dtype, cache=cache or dtype)
    c.update(dict(biases=False, interleaved=False) if kind == "append" else dict(cap=0.0, window=0, slopes=False))
    if kind == "chunk":
        c["prefix"] = 0
    c.update(more)
    return c


def listed():
    return [
        # A decode step of one user of a 0.5B decoder (f32 activations, f16 cache, biases): the smallest append.
        dict(name="append_one", **_case("append", (14, 2, 64), 1, 1000, "f32", "f16", biases=True)),
        # A decode step of a batch of 61 in a graph for 64: three rows of padding.
        dict(name="append_batch", **_case("append", (32, 8, 128), 64, 4000, "bf16", pad=3)),
        # A prefill step: ragged prompts, 8000 tokens and more in all, GGUF rows (interleaved pairs).
        dict(name="append_prompts", **_case("append", (32, 8, 128), 6, 2400, "f16", page=64, new=2400, interleaved=True)),
        # One user, a short conversation, 0.5B decoder: the smallest attention, where launches and latency are the time.
        dict(name="decode_one", **_case("decode", (14, 2, 64), 1, 333, "f32", "f16")),
        # A served batch of an 8B decoder at mixed lengths, padded to 64.
        dict(name="decode_batch", **_case("decode", (32, 8, 128), 64, 8192, "bf16", pad=3)),
        # One user with a long document: few rows, a long axis.
        dict(name="decode_long", **_case("decode", (32, 8, 128), 1, 131071, "f16", page=64)),
        # A capped, windowed layer of wide heads.
        dict(name="decode_window", **_case("decode", (8, 1, 256), 40, 6000, "bf16", page=32, cap=50.0, window=4096)),
        # One key head per query head, f32 throughout, distance bias, pages of an odd size.
        dict(name="decode_f32", **_case("decode", (32, 32, 80), 5, 1500, "f32", page=20, slopes=True)),
        # The engine's prefill chunk: 512 tokens after 512, f32 activations, f16 cache.
        dict(name="chunk_engine", **_case("chunk", (14, 2, 64), 1, 1024, "f32", "f16", new=512)),
        # Ragged prompts of an 8B decoder: the largest.
        dict(name="chunk_prompts", **_case("chunk", (32, 8, 128), 4, 4096, "bf16", new=4096)),
        # A few drafted tokens of each sequence checked against long contexts.
        dict(name="chunk_few", **_case("chunk", (28, 4, 128), 9, 12000, "f16", page=32, new=5)),
        # An image's tokens as a prefix that sees itself whole, then text, in a capped layer with a window.
        dict(name="chunk_prefix", **_case("chunk", (32, 32, 80), 2, 1111, "f16", new=1111, cap=30.0, window=777, prefix=256)),
    ]


def _log(rng, lo, hi):
    """A whole number from lo to hi, even over the logarithm."""
    return min(hi, max(lo, int(round(lo * (hi / lo) ** rng.random()))))


def draw(rng):
    kind = rng.choice(["append", "decode", "decode", "chunk", "chunk"])
    shape = rng.choice(SHAPES)
    dtype = rng.choice(["f16", "bf16", "f16", "bf16", "f32"])
    cache = rng.choice(["f16", "bf16", "f32"]) if dtype == "f32" else dtype
    page = rng.choice([16, 16, 32, 64, 128, 24, 1 + rng.randrange(60)])
    heads, kv, hd = shape
    seqs = _log(rng, 1, 200 if kind != "chunk" else 12)
    pad = rng.choice([0, 0, 1 + rng.randrange(4)]) if kind != "chunk" else 0
    mix = rng.randrange(1 << 20)
    if kind == "append":
        new = rng.choice([1, _log(rng, 2, 4096)])
        if new > 1:
            seqs, pad = min(seqs, 10), 0
        # at most the largest prefill step's rows, and pools of at most a few GB
        length = max(new, _log(rng, new, max(new + 1, min(8192, (1 << 28) // (seqs * kv * hd)))))
        new = min(new, max(1, 8192 // seqs))
        return _case(kind, shape, seqs, length, dtype, cache, page, new=new, pad=pad, mix=mix, biases=rng.random() < 0.4,
                     interleaved=rng.random() < 0.4)
    cap = rng.choice([0.0, 0.0, 30.0, 50.0])
    slopes = rng.random() < 0.25
    if kind == "decode":
        # at most 2^27 values of keys, half as much again as the longest document's
        most = max(1, (1 << 27) // (seqs * kv * hd * (2 if cache == "f32" else 1)))
        length = _log(rng, 1, min(131072, most))
        return _case(kind, shape, seqs + pad, length, dtype, cache, page, pad=pad, mix=mix, cap=cap, slopes=slopes,
                     window=rng.choice([0, 0, _log(rng, 1, 4096)]))
    new = _log(rng, 1, 4096)
    # at most half of the largest case's products
    length = _log(rng, new, max(new + 1, min(16384, (1 << 29) // (seqs * heads * new * (2 if dtype == "f32" else 1)))))
    while seqs * heads * new * length * hd > 1 << 36:
        new, length = (new + 1) // 2, (length + 1) // 2
    return _case(kind, shape, seqs, length, dtype, cache, page, new=new, mix=mix, cap=cap, slopes=slopes,
                 window=rng.choice([0, 0, _log(rng, 1, 4096)]), prefix=rng.choice([0, 0, _log(rng, 1, length)]))


# ───────────────────────────── inputs ─────────────────────────────
def _lens(c):
    """Tokens in the cache and new tokens of each sequence: the first is the longest, the others (ragged) even over the
    logarithm between a sixteenth of it and itself; those of the padding 0."""
    r = np.random.RandomState(c["mix"])
    n = c["seqs"]
    length = np.full(n, c["length"], dtype=np.int64)
    if c["ragged"]:
        length[1:] = np.maximum(1, (c["length"] * 16.0 ** -r.rand(n - 1)).astype(np.int64))
    new = np.minimum(length, np.maximum(1, np.ceil(c["new"] * length / c["length"]).astype(np.int64)))
    if c["pad"]:
        length[n - c["pad"]:] = new[n - c["pad"]:] = 0
    return length, new


def prepare(case, seed):
    c, dev = case, torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(seed)

    def randn(*shape, dtype=torch.float32):
        return torch.randn(shape, generator=g, device=dev).to(dtype)

    Hq, Hk, D, ps, dt, ct = c["heads"], c["kv_heads"], c["head_dim"], c["page"], DTYPE[c["dtype"]], DTYPE[c["cache"]]
    length, new = _lens(c)
    chunk = c["kind"] == "chunk" or c["new"] > 1
    rows = int(new.sum()) if chunk else c["seqs"]
    need = -(-length // ps)
    width, pages = int(need.max()) + 2, int(need.sum()) + 3
    # The pool's pages in the order in which an allocator that has served for a while hands them out; entries of the
    # table past a sequence's own are left at page 0.
    order = torch.randperm(pages, generator=g, device=dev).to(torch.int32)
    first = np.cumsum(need) - need
    at = np.arange(width)[None, :]
    used = torch.from_numpy(at < need[:, None]).to(dev)
    index = torch.from_numpy(np.minimum(first[:, None] + at, pages - 1)).to(dev)
    table = torch.where(used, order[index], torch.zeros_like(order[index]))
    s = {"c": c, "table": table.contiguous(), "max_len": int(length.max()), "max_new": int(new.max()), "rows": rows,
         "lens": torch.from_numpy(length.astype(np.int32)).to(dev), "chunk": chunk,
         "kc": randn(pages, Hk, ps, D, dtype=ct), "vc": randn(pages, Hk, ps, D, dtype=ct), "q": randn(rows, Hq, D, dtype=dt)}
    if chunk:
        s["cu"] = torch.from_numpy(np.concatenate([[0], np.cumsum(new)]).astype(np.int32)).to(dev)
    # The sequence of each row and its position.
    seq = np.repeat(np.arange(c["seqs"]), new) if chunk else np.arange(c["seqs"])
    start = np.cumsum(new) - new if chunk else np.arange(c["seqs"])
    pos = length[seq] - (new[seq] if chunk else 1) + np.arange(rows) - start[seq]
    s["seq"], s["pos"] = torch.from_numpy(seq).to(dev), torch.from_numpy(pos).to(dev)
    s["slot"] = torch.from_numpy(np.arange(rows) - start[seq]).to(dev)
    s["real"] = torch.from_numpy(np.flatnonzero(pos >= 0)).to(dev)  # all but the padding's
    if c["kind"] == "append":
        s["k"], s["v"] = randn(rows, Hk, D, dtype=dt), randn(rows, Hk, D, dtype=dt)
        s["b"] = [randn(n * D) * 0.1 for n in (Hq, Hk, Hk)] if c["biases"] else [None] * 3
        s["out"] = torch.zeros_like(s["q"])
    else:
        s["slopes"] = 2.0 ** (-8.0 / Hq * (torch.arange(Hq, device=dev) + 1.0)) if c["slopes"] else None
        # Scratch memory that a serving program keeps for its calls.
        s["workspace"] = torch.zeros(1 << 26, dtype=torch.uint8, device=dev)
        if c.get("prefix"):
            s["prefix"] = torch.from_numpy(np.minimum(length, c["prefix"]).astype(np.int32)).to(dev)
    return s


# ───────────────────────────── one pass ─────────────────────────────
def run(s):
    c = s["c"]
    if own:
        import sapient_amd.ops as ops
        if c["kind"] == "append":
            bq, bk, bv = s["b"]
            q = ops.rope_kv_append_paged(s["q"], s["k"], s["v"], s["lens"], s["table"], THETA[c["head_dim"]], s["kc"], s["vc"],
                                         cu_q=s.get("cu"), interleaved=c["interleaved"], bq=bq, bk=bk, bv=bv, out=s["out"])
            return {"q": q, "kc": s["kc"], "vc": s["vc"]}
        if c["kind"] == "decode":
            return ops.paged_attention(s["q"], s["kc"], s["vc"], s["lens"], s["table"], softcap=c["cap"], window=c["window"],
                                       slopes=s["slopes"], workspace=s["workspace"])
        return ops.paged_attention_chunk(s["q"], s["kc"], s["vc"], s["lens"], s["table"], s["cu"], softcap=c["cap"],
                                         window=c["window"], slopes=s["slopes"], prefix_lens=s.get("prefix"),
                                         workspace=s["workspace"])
    return _plain_append(s) if c["kind"] == "append" else _plain_attention(s)


def _plain_append(s):
    c, D, ps = s["c"], s["c"]["head_dim"], s["c"]["page"]
    real = s["real"]
    pos, seq = s["pos"][real], s["seq"][real]
    den = (THETA[D] ** (torch.arange(0, D, 2, device=pos.device).float() / D).double()).float()
    ang = (pos.float()[:, None] / den).double()
    cs, sn = ang.cos().float()[:, None, :], ang.sin().float()[:, None, :]
    bq, bk, bv = (0.0 if b is None else b.view(-1, D) for b in s["b"])

    def rotate(x):
        y = torch.empty_like(x)
        a, b = (slice(0, D, 2), slice(1, D, 2)) if c["interleaved"] else (slice(0, D // 2), slice(D // 2, D))
        y[..., a] = x[..., a] * cs - x[..., b] * sn
        y[..., b] = x[..., b] * cs + x[..., a] * sn
        return y

    s["out"][real] = rotate(s["q"][real].float() + bq).to(s["out"].dtype)
    page, row = s["table"][seq, pos // ps].long(), pos % ps
    s["kc"][page, :, row] = rotate(s["k"][real].float() + bk).to(s["kc"].dtype)
    s["vc"][page, :, row] = (s["v"][real].float() + bv).to(s["vc"].dtype)
    return {"q": s["out"], "kc": s["kc"], "vc": s["vc"]}


def _plain_attention(s):
    c = s["c"]
    Hq, Hk, D, ps, B, N = c["heads"], c["kv_heads"], c["head_dim"], c["page"], c["seqs"], s["max_new"] if s["chunk"] else 1
    dev = s["q"].device
    P = max(1, -(-s["max_len"] // ps))
    table = s["table"][:, :P].long()
    k, v = (t[table].transpose(1, 2).reshape(B, Hk, P * ps, D).float() for t in (s["kc"], s["vc"]))
    q = torch.zeros(B, N, Hq, D, device=dev)
    q[s["seq"], s["slot"]] = s["q"].float()
    q = q.view(B, N, Hk, Hq // Hk, D).permute(0, 2, 3, 1, 4).reshape(B, Hk, (Hq // Hk) * N, D)
    x = torch.matmul(q, k.transpose(2, 3).contiguous()) * D ** -0.5
    if c["cap"]:
        x = c["cap"] * torch.tanh(x / c["cap"])
    qpos = torch.full((B, N), -1, dtype=torch.int64, device=dev)
    qpos[s["seq"], s["slot"]] = s["pos"]
    kpos = torch.arange(P * ps, device=dev)
    dist = qpos[:, :, None] - kpos
    x = x.view(B, Hk, Hq // Hk, N, P * ps)
    if s["slopes"] is not None:
        x = x - s["slopes"].view(1, Hk, Hq // Hk, 1, 1) * dist.abs()[:, None, None].float()
    see = dist >= 0
    if s.get("prefix") is not None:
        see = see | (kpos < s["prefix"][:, None, None])
    if c["window"]:
        see = see & (dist < c["window"])
    see = (see & (kpos < s["lens"][:, None, None]) & (qpos >= 0)[:, :, None])[:, None, None]
    x = x.masked_fill(~see, float("-inf"))
    m = x.amax(-1, keepdim=True)
    x = torch.exp(x - torch.where(m == float("-inf"), torch.zeros_like(m), m))
    total = x.sum(-1, keepdim=True)
    x = x / torch.where(total == 0, torch.ones_like(total), total)
    y = torch.matmul(x.view(B, Hk, (Hq // Hk) * N, P * ps), v).view(B, Hq, N, D).transpose(1, 2)
    return y[s["seq"], s["slot"]].to(s["q"].dtype)


# ───────────────────────────── bytes and operations ─────────────────────────────
def work(case):
    c = case
    e, ec = (4 if c[n] == "f32" else 2 for n in ("dtype", "cache"))
    Hq, Hk, D = c["heads"], c["kv_heads"], c["head_dim"]
    length, new = _lens(c)
    rows = int(new.sum())
    table = 4 * int((-(-length // c["page"])).sum()) + 4 * c["seqs"]
    if c["kind"] == "append":
        return {"bytes": rows * (2 * Hq * D * e + 2 * Hk * D * (e + ec) + 8) + c["biases"] * 4 * (Hq + 2 * Hk) * D,
                "flops": 4 * rows * (Hq + Hk) * D}
    pairs, keys = 0, 0
    for L, n in zip(length.tolist(), new.tolist()):
        pos = np.arange(L - n, L)
        hi = np.maximum(pos + 1, min(L, c.get("prefix", 0)))
        lo = np.maximum(0, pos + 1 - c["window"]) if c["window"] else np.zeros_like(pos)
        pairs += int((hi - lo).sum())
        keys += int(hi.max() - lo.min()) if n else 0
    return {"bytes": 2 * keys * Hk * D * ec + 2 * rows * Hq * D * e + table, "flops": 4 * pairs * Hq * D}


# ───────────────────────────── the same in 64 bits ─────────────────────────────
def exact(case, seed):
    s, c = prepare(case, seed), case
    Hq, Hk, D, ps = c["heads"], c["kv_heads"], c["head_dim"], c["page"]
    length, new = _lens(c)
    row = 0
    if c["kind"] == "append":
        den = np.power(np.float32(THETA[D]), np.arange(0, D, 2, dtype=np.float32) / np.float32(D), dtype=np.float32)
        q, kc, vc = s["out"].double(), s["kc"].double(), s["vc"].double()
        bq, bk, bv = (torch.zeros((), device=q.device) if b is None else b.view(-1, D).double() for b in s["b"])
        for b in range(c["seqs"]):
            n, L = int(new[b]), int(length[b])
            pos = torch.arange(L - n, L, device=q.device)
            turn = (pos.float()[:, None] / torch.from_numpy(den).to(q.device)).double()
            turn = torch.polar(torch.ones_like(turn), turn)[:, None, :]

            def spin(x):  # pairs as complex numbers times e^(i angle)
                if c["interleaved"]:
                    z = torch.view_as_complex(x.reshape(*x.shape[:-1], D // 2, 2).contiguous()) * turn
                    return torch.view_as_real(z).reshape(x.shape)
                z = torch.complex(x[..., :D // 2].contiguous(), x[..., D // 2:].contiguous()) * turn
                return torch.cat([z.real, z.imag], -1)

            q[row:row + n] = spin(s["q"][row:row + n].double() + bq)
            page, at = s["table"][b, pos // ps].long(), pos % ps
            kc[page, :, at] = spin(s["k"][row:row + n].double() + bk)
            vc[page, :, at] = s["v"][row:row + n].double() + bv
            row += n if s["chunk"] else 1
        return {"q": q, "kc": kc, "vc": vc}
    out = torch.zeros(s["rows"], Hq, D, dtype=torch.float64, device=s["q"].device)
    for b in range(c["seqs"]):
        n, L = int(new[b]), int(length[b])
        if n:
            pos, key = (torch.arange(a, L, device=out.device) for a in (L - n, 0))
            at = s["table"][b, key // ps].long(), key % ps
            k, v = (t[at[0], :, at[1]].double().repeat_interleave(Hq // Hk, 1) for t in (s["kc"], s["vc"]))
            far = pos[:, None] - key[None, :]
            hidden = (far < 0) & (key >= (int(s["prefix"][b]) if "prefix" in s else 0))[None, :]
            if c["window"]:
                hidden |= far >= c["window"]
            for h in range(Hq):
                x = (s["q"][row:row + n, h].double() @ k[:, h].T.contiguous()) / D ** 0.5
                x = torch.tanh(x / c["cap"]) * c["cap"] if c["cap"] else x
                x = x - float(s["slopes"][h]) * far.abs() if s["slopes"] is not None else x
                out[row:row + n, h] = torch.softmax(x.masked_fill(hidden, -float("inf")), -1) @ v[:, h].contiguous()
        row += n if s["chunk"] else 1
    return out
