"""CPU: what the calls over a paged cache refuse, on the host and before any launch."""
import pytest
import torch

import sapient_amd
import sapient_amd.ops as ops
from sapient_amd import _lib
from test_cpu_launches import launches  # noqa: F401  (a fixture)

F32, F16, BF16, Q8 = _lib.F32, _lib.F16, _lib.BF16, _lib.Q8_0
A = 1 << 20  # 16-byte aligned addresses that are never read
NAN, INF = float("nan"), float("inf")


@pytest.fixture(scope="module")
def L():
    if not sapient_amd.LIB_PATH.exists():
        from sapient_amd import build
        build.build()
    return _lib.lib()


ATT = dict(q=A, out=2 * A, nq=8, nkv=2, dtype=F16, lens=A, table=A, seqs=3, max_pages=4, hd=64, kc=A, vc=A, cache=F16,
           pages=9, page=16, scale=1.0, cap=0.0, window=0, slopes=None, ws=None, wsn=0, flag=None, stream=None)
CHUNK = dict(q=A, out=2 * A, nq=8, nkv=2, dtype=F16, cu=A, lens=A, table=A, seqs=3, max_pages=4, rows=10, hd=64, kc=A, vc=A,
             cache=F16, pages=9, page=16, scale=1.0, cap=0.0, window=0, slopes=None, prefix=None, ws=None, wsn=0, flag=None,
             stream=None)
ROPE = dict(q=A, out=2 * A, nq=8, k=A, v=A, nkv=2, dtype=F16, layout=0, cu=A, lens=A, table=A, seqs=3, max_pages=4, rows=10,
            hd=64, base=1e4, pos_scale=1.0, kc=A, vc=A, cache=F16, pages=9, page=16, bq=None, bk=None, bv=None, bd=F32,
            flag=None, stream=None)
SHARED = [dict(dtype=Q8), dict(cache=Q8), dict(nq=-1), dict(nkv=0), dict(hd=0), dict(hd=-8), dict(seqs=-1),
          dict(max_pages=-1), dict(pages=0), dict(pages=-1), dict(page=0), dict(page=-16), dict(lens=None), dict(table=None),
          dict(lens=A + 2), dict(table=A + 1), dict(kc=None), dict(vc=None), dict(q=None), dict(out=None),
          dict(pages=1 << 31), dict(page=1 << 31), dict(seqs=1 << 31), dict(max_pages=1 << 31),
          dict(pages=1 << 20, page=1 << 11), dict(pages=1 << 27)]
ATTENTION = [dict(nq=0), dict(nq=7), dict(hd=20), dict(hd=264), dict(scale=NAN), dict(scale=INF), dict(cap=-1.0), dict(cap=NAN),
             dict(cap=INF), dict(cap=1e-7), dict(window=-1), dict(q=A + 8), dict(out=A + 2), dict(kc=A + 8), dict(vc=A + 8), dict(slopes=A + 2)]


def call(L, name, base, **change):
    return getattr(L, name)(*{**base, **change}.values())


@pytest.mark.parametrize("change", SHARED + ATTENTION, ids=str)
def test_paged_attention_refuses(L, change):
    assert call(L, "sph_paged_attention", ATT, **change) == _lib.EINVAL


@pytest.mark.parametrize("change", SHARED + ATTENTION + [dict(cu=None), dict(cu=A + 2), dict(rows=-1), dict(rows=1 << 31),
                                                         dict(prefix=A + 1), dict(out=A), dict(out=A + 16),
                                                         dict(rows=1 << 30, nq=1 << 10)], ids=str)
def test_paged_attention_chunk_refuses(L, change):
    assert call(L, "sph_paged_attention_chunk", CHUNK, **change) == _lib.EINVAL


@pytest.mark.parametrize("change", SHARED + [dict(layout=2), dict(hd=63), dict(hd=514), dict(pos_scale=0.0),
                                             dict(pos_scale=NAN), dict(k=None), dict(v=None), dict(cu=None), dict(cu=A + 2),
                                             dict(rows=-1), dict(rows=1 << 31), dict(out=A + 64), dict(bq=A, bd=Q8),
                                             dict(kc=A + 2), dict(q=A + 2)], ids=str)
def test_rope_kv_append_paged_refuses(L, change):
    assert call(L, "sph_rope_kv_append_paged", ROPE, **change) == _lib.EINVAL


def test_empty_calls_are_ok(L):
    assert call(L, "sph_paged_attention", ATT, seqs=0, q=None, out=None, lens=None, table=None) == _lib.OK
    assert call(L, "sph_paged_attention_chunk", CHUNK, seqs=0, rows=0, q=None, out=None) == _lib.OK
    assert call(L, "sph_paged_attention_chunk", CHUNK, rows=0, q=None, out=None) == _lib.OK
    assert call(L, "sph_rope_kv_append_paged", ROPE, rows=0, q=None, out=None, k=None, v=None) == _lib.OK
    assert call(L, "sph_rope_kv_append_paged", ROPE, rows=0, seqs=0, cu=None) == _lib.OK


X3, X4, I1, I2 = torch.zeros(2, 4, 8), torch.zeros(3, 2, 16, 8), torch.zeros(2, dtype=torch.int32), torch.zeros(2, 3, dtype=torch.int32)
CALLS = {
    "rope_kv_append_paged": lambda t: ops.rope_kv_append_paged(t, t, t, I1, I2, 1e4, X4, X4, cu_q=I1, bq=t, out=t),
    "paged_attention": lambda t: ops.paged_attention(t, X4, X4, I1, I2, scale=1.0, softcap=2.0, window=3, slopes=t, out=t, workspace=t),
    "paged_attention_chunk": lambda t: ops.paged_attention_chunk(t, X4, X4, I1, I2, I1, prefix_lens=I1, out=t, bad_page_flag=I1),
}


@pytest.mark.parametrize("name", CALLS)
def test_refuses_host_tensors_and_other_objects(name):
    with pytest.raises(ValueError, match="must be a device tensor"):
        CALLS[name](X3)
    with pytest.raises(TypeError, match="must be a torch.Tensor"):
        CALLS[name](object())


def test_workspace_sizes(L):
    assert ops.paged_attention_workspace(32, 8, 64, 512, 16, 128) > 0
    assert ops.paged_attention_workspace(32, 8, 64, 32, 16, 128) == 0       # tables of 512 keys are not split
    assert ops.paged_attention_workspace(32, 8, 1, 512, 16, 128, n_tokens=8192) == 0  # enough tiles
    assert ops.paged_attention_workspace(32, 8, 1, 512, 16, 128, n_tokens=8) > 0
    for bad in ((7, 2, 1, 1, 16, 64), (8, 2, 1 << 31, 1, 16, 64), (8, 2, 1, 1 << 62, 16, 64), (8, 2, 1, 1, 1 << 62, 64),
                (8, 2, 1, 1, 16, 20), (1 << 62, 2, 1, 1, 16, 64)):
        for n in (None, 5, 1 << 62):
            with pytest.raises(_lib.SapientHipError):
                ops.paged_attention_workspace(*bad, n_tokens=n)


@pytest.mark.parametrize("dtype", [F32, F16])
@pytest.mark.parametrize("hd", [8, 64, 128, 200])
def test_launches_at_any_batch(launches, dtype, hd):  # noqa: F811
    """Within HIP's limits, one launch or two, at the smallest and the largest batches and tables."""
    calls = []
    for seqs in (1, 64, 65536):
        for max_pages in (0, 1, 32, 1 << 20):
            a = dict(ATT, dtype=dtype, cache=dtype, hd=hd, seqs=seqs, max_pages=max_pages, ws=A, wsn=1 << 30)
            calls += [("sph_paged_attention", *a.values()), ("sph_paged_attention", *{**a, "ws": None, "wsn": 0}.values())]
            c = dict(CHUNK, dtype=dtype, cache=dtype, hd=hd, seqs=seqs, max_pages=max_pages, rows=seqs * 3, out=1 << 44, ws=A, wsn=1 << 30)
            calls += [("sph_paged_attention_chunk", *c.values()), ("sph_paged_attention_chunk", *{**c, "ws": None, "wsn": 0}.values())]
            r = dict(ROPE, dtype=dtype, cache=dtype, hd=hd, seqs=seqs, max_pages=max_pages, rows=seqs * 3, out=1 << 44)
            calls.append(("sph_rope_kv_append_paged", *r.values()))
    for call, (st, ls) in zip(calls, launches(*calls)):
        assert st == 0 and 1 <= len(ls) <= 2, (call, st, ls)
