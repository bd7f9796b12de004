"""CPU: what the calls over a paged cache refuse, on the host and before any launch."""
import pytest

import sapient_amd
from sapient_amd import _lib

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
             dict(cap=INF), dict(window=-1), dict(q=A + 8), dict(out=A + 2), dict(kc=A + 8), dict(vc=A + 8), dict(slopes=A + 2)]


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
