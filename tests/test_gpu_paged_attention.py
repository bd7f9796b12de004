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
