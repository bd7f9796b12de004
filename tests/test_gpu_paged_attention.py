"""GPU: attention over the paged KV cache, single tokens and ragged chunks, against the definition in 64 bits."""
import numpy as np
import pytest
import torch

import sapient_amd.ops as ops
from paged_reference import Batch, HALF_STEP, check

pytestmark = pytest.mark.gpu
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
TYPES = [(F16, F16), (BF16, BF16), (F32, F32), (F32, F16), (F32, BF16), (F16, BF16), (BF16, F16), (F16, F32), (BF16, F32)]
SHAPES = [(14, 2, 64), (32, 8, 128), (5, 5, 80), (8, 1, 256), (40, 2, 8), (6, 3, 200)]
NAME = {F32: "f32", F16: "f16", BF16: "bf16"}
# Half of a step of what weights are rounded to before the product with v: single tokens use two pieces of the
# cache's type; chunks of one half type one.
ids = lambda v: "-".join(NAME[t] for t in v) if isinstance(v, tuple) and v and v[0] in NAME else str(v)


def weights(dtype, cache, chunk):
    if cache == F32:
        return 0.0
    if chunk and dtype == cache:
        return 2 * HALF_STEP[cache]
    # two pieces (three where q is another type and pieces have 8 bits); f32 into f16 pieces of q: 2^-22 of a score
    return 2 * HALF_STEP[cache] ** 2 + 2.0 ** -19


def say(*a):
    print("case", *a, flush=True)


@pytest.mark.parametrize("types", TYPES, ids=ids)
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_single_tokens(dev, types, shape):
    dt, ct = types
    c = Batch(*shape, lens=[1, 333, 0, 16, 129, 2, 31, 64], dtype=dt, cache=ct, seed=1)
    say("single", types, shape)
    check(ops.paged_attention(*c.to(dev)), c, "single", weights(dt, ct, False))


@pytest.mark.parametrize("types", TYPES, ids=ids)
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_chunks(dev, types, shape):
    dt, ct = types
    c = Batch(*shape, lens=[1, 200, 45, 33, 7], new=[1, 70, 45, 3, 0], dtype=dt, cache=ct, seed=2, extra_rows=3)
    say("chunk", types, shape)
    t = c.to(dev)
    out = torch.full_like(t[0], 7.0)
    assert ops.paged_attention_chunk(*t, out=out) is out
    check(out, c, "chunk", weights(dt, ct, True))
    assert (out[c.cu[-1]:] == 7.0).all(), "rows past the last sequence are left as they were"


@pytest.mark.parametrize("page", [1, 3, 16, 20, 48, 64, 500])
@pytest.mark.parametrize("chunk", [False, True])
def test_page_sizes(dev, page, chunk):
    for seed, n in enumerate((1, 15, 17, 100, 333)):
        c = Batch(8, 2, 128, lens=[n, 40, n + 1], new=[min(n, 19), 1, n + 1] if chunk else None, page=page, seed=seed)
        say("pages", page, chunk, n)
        f = ops.paged_attention_chunk if chunk else ops.paged_attention
        check(f(*c.to(dev)), c, f"page {page}", weights(F16, F16, chunk))


MODS = [dict(softcap=2.0), dict(window=1), dict(window=50), dict(softcap=30.0, window=33), dict(slopes=True),
        dict(slopes=True, softcap=5.0, window=100), dict(scale=0.5), dict(scale=0.0)]


@pytest.mark.parametrize("mods", MODS, ids=str)
@pytest.mark.parametrize("types", [(F16, F16), (BF16, BF16), (F32, F32), (F32, BF16)], ids=ids)
@pytest.mark.parametrize("chunk", [False, True])
def test_score_forms(dev, mods, types, chunk):
    dt, ct = types
    for shape in ((14, 2, 64), (8, 2, 128)):
        c = Batch(*shape, lens=[300, 1, 77], new=[150, 1, 77] if chunk else None, dtype=dt, cache=ct, seed=5, q_std=2.0)
        m = dict(mods)
        if m.get("slopes"):
            m["slopes"] = 2.0 ** (-8.0 / c.heads * (torch.arange(c.heads) + 1.0))
        say("scores", mods, types, chunk, shape)
        dm = {k: v.to(dev) if isinstance(v, torch.Tensor) else v for k, v in m.items()}
        f = ops.paged_attention_chunk if chunk else ops.paged_attention
        check(f(*c.to(dev), **dm), c, str(mods), weights(dt, ct, chunk), **m)


@pytest.mark.parametrize("types", [(F16, F16), (BF16, BF16), (F32, F16)], ids=ids)
@pytest.mark.parametrize("window", [0, 60])
def test_prefix(dev, types, window):
    dt, ct = types
    c = Batch(6, 2, 64, lens=[300, 90, 10, 5], new=[200, 90, 4, 5], dtype=dt, cache=ct, seed=6)
    prefix = [170, 1000, 3, 0]
    say("prefix", types, window)
    got = ops.paged_attention_chunk(*c.to(dev), window=window, prefix_lens=torch.tensor(prefix, dtype=torch.int32, device=dev))
    check(got, c, "prefix", weights(dt, ct, True), window=window, prefix=prefix)


def test_a_used_workspace_leaves_nothing(dev):
    """What an earlier call, or anything, left in the workspace does not reach a result."""
    for lens in ([333], [1, 333, 0, 16, 129], [700, 3, 650] * 5):
        c = Batch(14, 2, 64, lens=lens, seed=7)
        n = ops.paged_attention_workspace(14, 2, len(lens), c.table.shape[1], 16, 64)
        for size in (n, n // 3, n // 40, 0):  # with less of it the keys are split less
            ws = torch.full((size // 4 + 4,), float("nan"), device=dev).view(torch.uint8)[:size]
            say("workspace", lens[:5], size)
            check(ops.paged_attention(*c.to(dev), workspace=ws), c, "workspace", weights(F16, F16, False))
    for lens, new in (([700], [9]), ([1300, 40, 600], [33, 40, 1])):
        c = Batch(14, 2, 64, lens=lens, new=new, seed=8)
        n = ops.paged_attention_workspace(14, 2, len(lens), c.table.shape[1], 16, 64, n_tokens=c.q.shape[0])
        assert n > 0
        for size in (n, n // 2, 0):
            ws = torch.full((size // 4 + 4,), float("nan"), device=dev).view(torch.uint8)[:size]
            say("workspace, chunk", lens, size)
            check(ops.paged_attention_chunk(*c.to(dev), workspace=ws), c, "workspace", weights(F16, F16, True))


def test_many_sequences(dev):
    """More sequences than a block has threads, of lengths on both sides of a step."""
    for n, chunk in ((300, False), (1030, False), (300, True)):
        lens = [(7 * i) % 135 for i in range(n)]
        new = [min(x, i % 4) for i, x in enumerate(lens)] if chunk else None
        c = Batch(4, 2, 64, lens=lens, new=new, seed=n)
        say("many", n, chunk)
        f = ops.paged_attention_chunk if chunk else ops.paged_attention
        check(f(*c.to(dev)), c, f"{n} sequences", weights(F16, F16, chunk))


@pytest.mark.parametrize("types", [(F16, F16), (BF16, BF16), (F32, F32), (F32, F16)], ids=ids)
def test_long_sequences(dev, types):
    """Lengths that are split into parts, with and without a chunk's own splits."""
    dt, ct = types
    for lens, new in (([3000, 5, 1500], None), ([4097], None), ([3000, 70], [3, 70]), ([2500], [1])):
        c = Batch(8, 2, 64, lens=lens, new=new, dtype=dt, cache=ct, seed=11)
        say("long", types, lens, new)
        f = ops.paged_attention_chunk if new else ops.paged_attention
        check(f(*c.to(dev)), c, f"{lens}", weights(dt, ct, bool(new)))


@pytest.mark.parametrize("types", [(F16, F16), (F32, F32), (F32, BF16)], ids=ids)
@pytest.mark.parametrize("chunk", [False, True])
def test_missing_pages_take_no_part(dev, types, chunk):
    dt, ct = types
    new = [20, 1, 33, 5] if chunk else None
    f = ops.paged_attention_chunk if chunk else ops.paged_attention
    for entry in (-1, 10 ** 6, 2 ** 31 - 1, -2 ** 31):
        c = Batch(8, 2, 64, lens=[100, 40, 33, 5], new=new, dtype=dt, cache=ct, seed=13)
        flag = torch.zeros(1, dtype=torch.int32, device=dev)
        check(f(*c.to(dev), bad_page_flag=flag), c, "whole", weights(dt, ct, chunk))
        assert int(flag) == 0
        c.table[0, 2] = c.table[1, 0] = c.table[3, 0] = entry  # the last sequence keeps no key at all
        say("missing", types, chunk, entry)
        got = f(*c.to(dev), bad_page_flag=flag)
        check(got, c, "missing", weights(dt, ct, chunk))
        assert int(flag) == 1 and not got[c.cu[3]:c.cu[4]].any(), "rows without keys are zeros"
        check(f(*c.to(dev)), c, "no flag", weights(dt, ct, chunk))
    # a length that the table has no entries for
    c = Batch(8, 2, 64, lens=[100, 40], new=new and [3, 2], dtype=dt, cache=ct, seed=14)
    c.table = c.table[:, :4].contiguous()
    flag.zero_()
    check(f(*c.to(dev), bad_page_flag=flag), c, "narrow table", weights(dt, ct, chunk))
    assert int(flag) == 1


def test_sequences_shorter_than_their_new_rows(dev):
    for dt, ct in ((F16, F16), (F32, F32)):
        c = Batch(8, 2, 64, lens=[40, 10], new=[5, 10], dtype=dt, cache=ct, seed=15)
        c.lens[1] = 6
        c.seq_lens[1] = 6
        flag = torch.zeros(1, dtype=torch.int32, device=dev)
        say("short", dt)
        got = ops.paged_attention_chunk(*c.to(dev), bad_page_flag=flag)
        check(got, c, "short", weights(dt, ct, True))
        assert int(flag) == 1 and not got[5:9].any(), "rows without a position are zeros"


@pytest.mark.parametrize("cu", [[0, 0, 0], [5, 9, 9], [0, 9, 3], [-4, 2, 50], [9, 4, 0], [7, 7, 7]], ids=str)
def test_any_cu_q_stays_in_bounds(dev, cu):
    """Rows outside every sequence are left as they were; nothing outside q and out is touched, whatever cu_q holds."""
    for dt, ct in ((F16, F16), (F32, F32)):
        c = Batch(8, 2, 64, lens=[40, 30], new=[4, 5], dtype=dt, cache=ct, seed=16)
        t = c.to(dev)
        guard = torch.full((t[0].shape[0] + 8, 8, 64), 7.0, dtype=dt, device=dev)
        out = guard[4:-4]
        say("cu", cu, dt)
        ops.paged_attention_chunk(*t[:5], torch.tensor(cu, dtype=torch.int32, device=dev), out=out)
        assert (guard[:4] == 7).all() and (guard[-4:] == 7).all()
        inside = torch.zeros(out.shape[0], dtype=torch.bool)
        for a, b in zip(cu, cu[1:]):
            inside[max(a, 0):max(0, min(b, out.shape[0]))] = True
        if cu == sorted(cu):
            assert (out.cpu()[~inside] == 7).all()


def test_extreme_scores(dev):
    """Large scores, one key far above the rest, scores of both signs past f16's range, and q of every size."""
    for dt, ct in ((F16, F16), (BF16, BF16), (F32, F32), (F32, F16), (F32, BF16)):
        for chunk in (False, True):
            f = ops.paged_attention_chunk if chunk else ops.paged_attention
            for q_std in (1e-6, 30.0, 2000.0):
                c = Batch(4, 2, 64, lens=[130, 70], new=[70, 9] if chunk else None, dtype=dt, cache=ct, seed=17, q_std=q_std)
                say("extreme", dt, ct, chunk, q_std)
                # at 2000 a score's own rounding is several units: the largest key wins but for near ties
                got, scale = f(*c.to(dev), scale=0.125), 0.125
                if q_std < 1000:
                    check(got, c, f"q std {q_std}", weights(dt, ct, chunk), scale=scale)
                assert torch.isfinite(got.float()).all()
            check(f(*c.to(dev), scale=-0.01), c, "negative scale", weights(dt, ct, chunk), scale=-0.01)


def test_infinite_keys_and_values(dev):
    """A key whose score is minus infinity weighs nothing; what is not finite in a key or value reaches the rows that see it."""
    for dt, ct in ((F16, F16), (F32, F32), (F32, F16)):
        c = Batch(2, 1, 64, lens=[100], dtype=dt, cache=ct, seed=18)
        p, r = int(c.table[0, 2]), 5
        c.q[0] = c.q[0].abs() + 0.1
        c.kc[p, 0, r] = -60000.0  # far below every other score
        say("low", dt, ct)
        check(ops.paged_attention(*c.to(dev)), c, "low", weights(dt, ct, False))
        c.vc[p, 0, r + 1, 7] = float("inf")
        got = ops.paged_attention(*c.to(dev)).float().cpu()
        # Infinite or NaN: a weight is the sum of two or three pieces of the cache's type, whose lower ones are zero or of
        # either sign, and inf + 0 inf and inf - inf are NaN.
        assert not torch.isfinite(got[0, :, 7]).any()
        assert torch.isfinite(got[0, :, :7]).all() and torch.isfinite(got[0, :, 8:]).all()
        c.kc[p, 0, r + 2, 3] = float("nan")
        assert torch.isnan(ops.paged_attention(*c.to(dev)).float()).all()


def test_pools_past_32_bit_offsets(dev):
    """Pages whose bytes lie past 4 GiB (and elements past 2^31) of the pools."""
    pages, page, kv, D = 70000, 64, 4, 128  # 4.3 GiB and 2.3 * 2^30 elements each
    kc, vc = (torch.empty(pages, kv, page, D, dtype=F16, device=dev) for _ in range(2))
    assert kc.numel() > 1 << 31
    for new in (None, [40, 3]):
        c = Batch(8, kv, D, lens=[150, 70], new=new, page=page, seed=19)
        t = c.to(dev)
        far = torch.tensor([pages - 1 - i for i in range(c.kc.shape[0])], device=dev)
        kc[far], vc[far] = t[1], t[2]
        table = torch.where(t[4] >= 0, far[t[4].clamp(min=0).long()].int(), t[4])
        say("far pages", new)
        f = ops.paged_attention_chunk if new else ops.paged_attention
        check(f(t[0], kc, vc, t[3], table, *t[5:]), c, "far", weights(F16, F16, bool(new)))
    s = torch.randn(3, kv, D, device=dev).half()
    last = torch.tensor([[pages - 1], [pages - 2], [pages - 3]], dtype=torch.int32, device=dev)
    ops.rope_kv_append_paged(torch.zeros(3, 8, D, device=dev).half(), s, s, torch.tensor([64, 1, 2], dtype=torch.int32, device=dev),
                             last, 1e4, kc, vc)
    assert torch.equal(vc[pages - 1, :, 63], s[0]) and torch.equal(vc[pages - 2, :, 0], s[1]) and torch.equal(vc[pages - 3, :, 1], s[2])


def test_out_may_be_q_for_single_tokens(dev):
    for lens in ([333, 20], [5000, 7]):
        c = Batch(40, 2, 64, lens=lens, seed=20)
        t = c.to(dev)
        say("in place", lens)
        assert ops.paged_attention(*t, out=t[0]) is t[0]
        check(t[0], c, "in place", weights(F16, F16, False))


def test_another_stream_and_repeated_calls_agree(dev):
    c = Batch(32, 8, 128, lens=[700, 1300, 5, 90], dtype=BF16, seed=21)
    d = Batch(32, 8, 128, lens=[700, 130], new=[70, 130], dtype=BF16, seed=22)
    want = ops.paged_attention(*c.to(dev)), ops.paged_attention_chunk(*d.to(dev))
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        tc, td = c.to(dev), d.to(dev)
        for again in range(3):
            got = ops.paged_attention(*tc), ops.paged_attention_chunk(*td)
            s.synchronize()
            assert all(torch.equal(g, w) for g, w in zip(got, want)), "the same bits every time"


def test_refuses_what_does_not_fit(dev):
    c = Batch(8, 2, 64, lens=[40, 30], new=[4, 5])
    q, kc, vc, lens, table, cu = c.to(dev)
    one = q[:2].contiguous()
    ok = ops.paged_attention(one, kc, vc, lens, table)
    for bad in (lambda: ops.paged_attention(q, kc, vc, lens, table),              # rows are not the sequences
                lambda: ops.paged_attention(one, kc, vc[:-1], lens, table),
                lambda: ops.paged_attention(one, kc, vc.float(), lens, table),
                lambda: ops.paged_attention(one, kc[0], vc[0], lens, table),
                lambda: ops.paged_attention(one, kc, vc, lens.long(), table),
                lambda: ops.paged_attention(one, kc, vc, lens, table[:1]),
                lambda: ops.paged_attention(one, kc, vc, lens, table.t()),
                lambda: ops.paged_attention(one, kc, vc, lens, table, slopes=lens.float()),
                lambda: ops.paged_attention(one, kc, vc, lens, table, out=torch.empty_like(q)),
                lambda: ops.paged_attention(one.transpose(0, 1), kc, vc, lens, table),
                lambda: ops.paged_attention(one, kc, vc, lens, table, workspace=one),
                lambda: ops.paged_attention_chunk(q, kc, vc, lens, table, cu[:-1]),
                lambda: ops.paged_attention_chunk(q, kc, vc, lens, table, cu, prefix_lens=cu),
                lambda: ops.rope_kv_append_paged(q, q, q, lens, table, 1e4, kc, vc, cu_q=cu)):
        with pytest.raises(ValueError):
            bad()
    for bad in (lambda: ops.paged_attention(one, kc, vc, lens, table, softcap=-1.0),
                lambda: ops.paged_attention(one, kc, vc, lens, table, window=-1),
                lambda: ops.paged_attention(one, kc, vc, lens, table, scale=float("inf")),
                lambda: ops.paged_attention_chunk(q, kc, vc, lens, table, cu, out=q)):
        with pytest.raises(ops._lib.SapientHipError):
            bad()
    with pytest.raises(TypeError):
        ops.paged_attention_chunk(q, kc, vc, lens, table, None)
    assert torch.equal(ok, ops.paged_attention(one, kc, vc, lens, table))


@pytest.mark.parametrize("types", TYPES, ids=ids)
def test_values_that_are_not_finite_stay_in_rows_that_see_them(dev, types):
    """A value that is not finite leaves the rows that see its key not finite, in its channel at least, and no other row."""
    dt, ct = types
    for new, window in ((60, 0), (90, 20), (3, 0), (90, 0)):
        c = Batch(4, 2, 64, lens=[90, 40], new=[new, 40], dtype=dt, cache=ct, seed=23)
        at = 60
        p, r = int(c.table[0, at // 16]), at % 16
        clean = ops.paged_attention_chunk(*c.to(dev), window=window).float().cpu()
        for bad in (float("nan"), float("inf"), -float("inf")):
            c.vc[p, 1, r, 5] = bad
            say("not finite", types, new, window, bad)
            got = ops.paged_attention_chunk(*c.to(dev), window=window).float().cpu()
            sees = torch.zeros(got.shape[:2], dtype=torch.bool)
            for i in range(new):
                pos = 90 - new + i
                sees[i, 2:] = pos >= at and (not window or pos - at < window)  # heads 2 and 3 read kv head 1
            assert not torch.isfinite(got[sees][:, 5]).any()
            assert torch.equal(got[~sees], clean[~sees])


@pytest.mark.parametrize("seed", range(24))
def test_random_batches(dev, seed):
    """Any mix of heads, head_dim, types, pages, lengths, masks and score forms."""
    r = np.random.default_rng(seed)
    kv = int(r.integers(1, 6))
    heads, D = kv * int(r.choice([1, 2, 3, 7, 16, 20])), 8 * int(r.integers(1, 33))
    dt, ct = TYPES[int(r.integers(len(TYPES)))]
    chunk = bool(r.integers(2))
    lens = [int(x) for x in r.integers(0, 260, int(r.integers(1, 6)))]
    if r.integers(4) == 0:
        lens[0] = int(r.integers(600, 1500))
    new = [int(min(n, x)) for n, x in zip(lens, r.integers(0, 150, len(lens)))] if chunk else None
    if chunk and not sum(new):
        new[0] = lens[0] = max(1, lens[0])
    c = Batch(heads, kv, D, lens, new, dt, ct, page=int(r.choice([1, 5, 16, 32, 40, 64, 256])), seed=seed, extra_rows=2 * chunk)
    m = {}
    if r.integers(3) == 0:
        m["softcap"] = float(r.choice([1.0, 20.0]))
    if r.integers(3) == 0:
        m["window"] = int(r.integers(1, 300))
    if r.integers(3) == 0:
        m["slopes"] = torch.from_numpy(r.uniform(0, 0.5, heads).astype(np.float32))
    kw = {k: v.to(dev) if isinstance(v, torch.Tensor) else v for k, v in m.items()}
    if chunk and r.integers(2):
        m["prefix"] = [int(x) for x in r.integers(0, 300, len(lens))]
        kw["prefix_lens"] = torch.tensor(m["prefix"], dtype=torch.int32, device=dev)
    say("random", seed, heads, kv, D, NAME[dt], NAME[ct], c.page, lens, new, {k: v for k, v in m.items() if k != "slopes"})
    f = ops.paged_attention_chunk if chunk else ops.paged_attention
    check(f(*c.to(dev), **kw), c, f"seed {seed}", weights(dt, ct, chunk), **m)
