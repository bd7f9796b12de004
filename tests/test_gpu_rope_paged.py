"""GPU: the fused bias + RoPE + append into a paged cache, against sph_rope_kv_append_tokens on each sequence alone, bit
for bit; what is no token, and pages that are none, change nothing."""
import pytest
import torch

import sapient_amd.ops as ops

pytestmark = pytest.mark.gpu
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
NAME = {F32: "f32", F16: "f16", BF16: "bf16"}


def bits(t):
    return t.view(torch.int32 if t.dtype == F32 else torch.int16)


class Step:
    """A batch's step: pools of random old rows, a shuffled table, q, k, v for the new tokens."""

    def __init__(self, dev, heads, kv, D, lens, new, dtype, cache, page, seed=0, biases=None, extra=0):
        g = torch.Generator(device=dev).manual_seed(seed)
        r = lambda *s: torch.randn(*s, generator=g, device=dev)
        self.lens, self.new, self.page, self.shape = lens, new, page, (heads, kv, D)
        need = [-(-n // page) for n in lens]
        pages = sum(need) + 3
        order = torch.randperm(pages, generator=g, device=dev).tolist()
        table = torch.full((len(lens), max(need + [0]) + 2), -7, dtype=torch.int32)
        for b, n in enumerate(need):
            for i in range(n):
                table[b, i] = order.pop()
        self.table, self.host_table = table.to(dev), table
        self.seq_lens = torch.tensor(lens, dtype=torch.int32, device=dev)
        n = new or [1] * len(lens)
        cu = [0]
        for x in n:
            cu.append(cu[-1] + x)
        self.cu, self.starts = (torch.tensor(cu, dtype=torch.int32, device=dev) if new else None), cu
        T = cu[-1] + extra
        self.q, self.k, self.v = r(T, heads, D).to(dtype), r(T, kv, D).to(dtype), r(T, kv, D).to(dtype)
        self.kc, self.vc = r(pages, kv, page, D).to(cache), r(pages, kv, page, D).to(cache)
        self.b = [r(h * D).to(biases) for h in (heads, kv, kv)] if biases else [None] * 3
        self.flag = torch.zeros(1, dtype=torch.int32, device=dev)

    def run(self, base=1e4, out=None, **kw):
        kc, vc = self.kc.clone(), self.vc.clone()
        bq, bk, bv = self.b
        out = ops.rope_kv_append_paged(self.q, self.k, self.v, self.seq_lens, self.table, base, kc, vc, cu_q=self.cu,
                                       bad_page_flag=self.flag, bq=bq, bk=bk, bv=bv,
                                       out=torch.full_like(self.q, 7.0) if out is None else out, **kw)
        return out, kc, vc

    def want(self, base=1e4, **kw):
        """The same by one contiguous cache per sequence."""
        kc, vc, out = self.kc.clone(), self.vc.clone(), torch.full_like(self.q, 7.0)
        heads, kv, D = self.shape
        bq, bk, bv = self.b
        for b, L in enumerate(self.lens):
            rows = slice(self.starts[b], self.starts[b + 1])
            n = rows.stop - rows.start
            if L < n or n == 0:
                continue
            one = [torch.zeros(kv, L, D, dtype=kc.dtype, device=kc.device) for _ in range(2)]
            pos = torch.arange(L - n, L, dtype=torch.int32, device=kc.device)
            q = ops.rope_kv_append_tokens(self.q[rows].contiguous(), self.k[rows].contiguous(), self.v[rows].contiguous(),
                                          pos, base, *one, bq=bq, bk=bk, bv=bv, **kw)
            out[rows] = q.transpose(0, 1)
            for i, p in enumerate(range(L - n, L)):
                page = int(self.host_table[b, p // self.page]) if p // self.page < self.host_table.shape[1] else -1
                if 0 <= page < kc.shape[0]:
                    kc[page, :, p % self.page], vc[page, :, p % self.page] = one[0][:, p], one[1][:, p]
        return out, kc, vc

    def check(self, what, **kw):
        print("case", what, flush=True)
        got, want = self.run(**kw), self.want(**kw)
        for name, g, w in zip(("q", "kcache", "vcache"), got, want):
            assert torch.equal(bits(g), bits(w)), f"{what}: {name}"


TYPES = [(a, b) for a in (F32, F16, BF16) for b in (F32, F16, BF16)]


@pytest.mark.parametrize("types", TYPES, ids=lambda t: "-".join(NAME[x] for x in t))
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("biases", [None, F32, F16])
def test_types_and_layouts(dev, types, interleaved, biases):
    for shape in ((14, 2, 64), (3, 3, 80), (32, 8, 128)):
        s = Step(dev, *shape, lens=[5, 1, 70, 0, 17], new=None, dtype=types[0], cache=types[1], page=16, biases=biases)
        s.check(f"single {shape}", interleaved=interleaved, base=5e5)
        s = Step(dev, *shape, lens=[9, 1, 70, 33], new=[9, 1, 40, 0], dtype=types[0], cache=types[1], page=16,
                 biases=biases, extra=5)
        s.check(f"chunk {shape}", interleaved=interleaved, base=5e5, pos_scale=2.0)
        assert int(s.flag) == 0


@pytest.mark.parametrize("page", [1, 7, 16, 20, 64, 1000])
def test_pages_and_batches(dev, page):
    for lens, new in (([333], [333]), ([700, 2, 5], [600, 2, 1]), ([1] * 300, None), ([40] * 300, [3] * 300), ([0] * 4, None),
                      ([0, 0, 8], [0, 0, 8]), ([300] * 9, [100] * 9)):
        s = Step(dev, 8, 2, 64, lens, new, BF16, BF16, page)
        s.check(f"page {page} lens {lens[:3]} new {None if new is None else new[:3]}")
        assert int(s.flag) == 0


def test_far_positions_and_in_place(dev):
    lens = [70001, 131072, 300000]
    s = Step(dev, 4, 1, 128, lens, [3, 1, 2], F16, F16, 4096)
    s.check("far", base=1e6)
    q = s.q.clone()
    s.q, keep = q, s.q
    want = s.want()[0]
    got, _, _ = s.run(out=q)
    assert got is q and torch.equal(bits(q), bits(want))
    s.q = keep


@pytest.mark.parametrize("new", [None, [1, 3, 2, 5]])
def test_bad_pages_write_nothing_and_raise_the_flag(dev, new):
    for entry in (-1, 10 ** 6, 2 ** 31 - 1, -2 ** 31):
        s = Step(dev, 8, 2, 64, [40, 33, 64, 5], new, F16, F16, 16)
        s.host_table[1, 2] = s.table[1, 2] = entry
        s.check(f"entry {entry}")
        assert int(s.flag) == 1
    # positions that the table has no entry for, and sequences shorter than their new tokens
    s = Step(dev, 8, 2, 64, [40, 33, 64, 5], new, F16, F16, 16)
    s.table, s.host_table = s.table[:, :3].contiguous(), s.host_table[:, :3].contiguous()
    s.check("table too narrow")
    assert int(s.flag) == 1
    if new:
        s = Step(dev, 8, 2, 64, [40, 33, 64, 5], new, F16, F16, 16)
        s.lens[3] = 4
        s.seq_lens[3] = 4
        got, kc, vc = s.run()
        assert int(s.flag) == 1
        # four of the five rows have a position; the first has none and stays
        assert (got[s.starts[3]] == 7).all() and not (got[s.starts[3] + 1:] == 7).all()


@pytest.mark.parametrize("cu", [[0, 0, 0], [5, 9, 9], [0, 9, 3], [-4, 2, 50], [9, 4, 0], [7, 7, 7]], ids=str)
@pytest.mark.parametrize("many", [False, True])
def test_any_cu_q_stays_in_bounds(dev, cu, many):
    """Nothing outside q_out and the pools is touched, whatever cu_q holds, and rows outside every sequence stay."""
    lens = [40, 30] + [0] * (100 if many else 0)
    s = Step(dev, 8, 2, 64, lens, [4, 5] + [0] * (len(lens) - 2), F16, F16, 16)
    cu = cu + [cu[-1]] * (len(lens) - 2)
    s.cu = torch.tensor(cu, dtype=torch.int32, device=dev)
    guard = torch.full((s.q.shape[0] + 8, 8, 64), 7.0, dtype=F16, device=dev)
    print("case", cu[:4], many, flush=True)
    got, kc, vc = s.run(out=guard[4:-4])
    assert (guard[:4] == 7).all() and (guard[-4:] == 7).all()
    if cu == sorted(cu):
        inside = torch.zeros(got.shape[0], dtype=torch.bool)
        for a, b in zip(cu, cu[1:]):
            inside[max(a, 0):max(0, min(b, got.shape[0]))] = True
        assert (got.cpu()[~inside] == 7).all()
