"""A paged KV cache built for a test, and softmax attention over it in 64 bits on the host, written from the operator's
definition, with a bound on how far f32 arithmetic and the output's rounding may be off."""
import numpy as np
import torch

HALF_STEP = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}


class Batch:
    """Random pools, a shuffled block table, and q rows for sequences of `lens` tokens, `new` of them new (None: one
    each). What no key of a sequence lies in (the rest of its last page, pages of nobody) is filled with `stale`."""

    def __init__(self, heads, kv_heads, D, lens, new=None, dtype=torch.float16, cache=None, page=16, seed=0, stale=float("nan"),
                 q_std=1.0, extra_rows=0):
        g = torch.Generator().manual_seed(seed)
        cache = cache or dtype
        self.lens, self.page, self.D, self.heads, self.kv_heads = list(lens), page, D, heads, kv_heads
        self.new = [1] * len(lens) if new is None else list(new)
        need = [-(-n // page) for n in lens]
        pages = sum(need) + 2
        order = torch.randperm(pages, generator=g).tolist()
        width = max(need + [1]) + 1
        table = torch.full((len(lens), width), -1, dtype=torch.int32)  # entries past a sequence's pages are never read
        self.kc, self.vc = (torch.full((pages, kv_heads, page, D), stale).to(cache) for _ in range(2))
        for b, n in enumerate(lens):
            for i in range(need[b]):
                p = order.pop()
                table[b, i] = p
                m = min(page, n - i * page)
                self.kc[p, :, :m] = torch.randn(kv_heads, m, D, generator=g).to(cache)
                self.vc[p, :, :m] = torch.randn(kv_heads, m, D, generator=g).to(cache)
        self.table, self.chunk = table, new is not None
        self.cu = np.concatenate([[0], np.cumsum(self.new)]).astype(np.int32)
        rows = int(self.cu[-1]) + extra_rows
        self.q = (torch.randn(rows, heads, D, generator=g) * q_std).to(dtype)
        self.seq_lens = torch.tensor(self.lens, dtype=torch.int32)

    def to(self, dev):
        """(q, kcache, vcache, seq_lens, block_table) on the device, and cu_q after them for chunks."""
        t = [self.q, self.kc, self.vc, self.seq_lens, self.table]
        if self.chunk:
            t.append(torch.from_numpy(self.cu))
        return [x.to(dev) for x in t]

    def keys(self, b, h):
        """k and v [len, D] of kv head h of sequence b, in 64 bits; zeros and False where there is no page."""
        n, ps = self.lens[b], self.page
        k, v, there = np.zeros((n, self.D)), np.zeros((n, self.D)), np.zeros(n, bool)
        for t in range(n):
            if t // ps < self.table.shape[1] and 0 <= int(self.table[b, t // ps]) < self.kc.shape[0]:
                p = int(self.table[b, t // ps])
                k[t], v[t] = self.kc[p, h, t % ps].double().numpy(), self.vc[p, h, t % ps].double().numpy()
                there[t] = True
        return k, v, there


def attention(c, scale=None, softcap=0.0, window=0, slopes=None, prefix=None, weight_step=None):
    """(out, tolerance) [rows, heads, D] in 64 bits; rows that are no tokens are NaN. weight_step: half a step of the
    type that weights are rounded to before the product with v, relative (None: f32's)."""
    scale = c.D ** -0.5 if scale is None else scale
    out = np.full(c.q.shape, np.nan)
    tol = np.zeros(c.q.shape)
    u = 2.0 ** -24
    half = HALF_STEP[c.q.dtype]
    G = c.heads // c.kv_heads
    q = c.q.double().numpy()
    for b, n in enumerate(c.new):
        L = c.lens[b]
        pos = np.arange(L - n, L)
        p = np.arange(L)
        see = (p[None, :] <= pos[:, None]) | (p[None, :] < (0 if prefix is None else prefix[b]))
        if window:
            see &= pos[:, None] - p[None, :] < window
        see &= (pos >= 0)[:, None]
        rows = slice(int(c.cu[b]), int(c.cu[b]) + n)
        for h in range(c.kv_heads):
            k, v, there = c.keys(b, h)
            s_all = see & there[None, :]
            for hq in range(h * G, (h + 1) * G):
                x = q[rows, hq]
                with np.errstate(all="ignore"):
                    s = scale * (x @ k.T)
                    size = abs(scale) * (np.abs(x) @ np.abs(k).T)
                    if softcap:
                        s = softcap * np.tanh(s / softcap)
                    if slopes is not None:
                        s = s - float(slopes[hq]) * np.abs(pos[:, None] - p[None, :])
                    s = np.where(s_all, s, -np.inf)
                    m = s.max(axis=1, keepdims=True, initial=-np.inf)
                    w = np.where(s_all, np.exp(s - np.where(np.isinf(m), 0.0, m)), 0.0)
                    total = w.sum(axis=1, keepdims=True)
                    w = np.divide(w, total, out=np.zeros_like(w), where=total > 0)
                    out[rows, hq] = w @ v
                    # A score: D products and sums in f32 (and its terms' own roundings, each at the size of what it
                    # rounds: the cap's quotient, tanh and product, the slope's distance and difference, the change
                    # to log2 and the difference from the maximum), so |ds| <= u ((D + 4) size + 12 |s|max + 4 cap);
                    # a weight e^s then is off by ds, its exp2 by 2u, and so is the sum of all weights; the sums over n
                    # keys by n u each, the joins of parts by a few u; the weight's rounding by weight_step.
                    size = np.where(s_all, size, 0).max(axis=1, keepdims=True, initial=0)
                    smax = np.where(s_all, np.abs(s), 0).max(axis=1, keepdims=True, initial=0)
                    ds = u * ((c.D + 4) * size + 12 * smax + 4 * softcap)
                    rel = 2 * ds + 2 * (L + 16) * u + (weight_step or 0.0)
                    tol[rows, hq] = rel * (w @ np.abs(v)) + half * np.abs(out[rows, hq]) + 1e-30
    # f16 results below 2^-14 are rounded to multiples of 2^-24
    return out, tol + (2.0 ** -25 if c.q.dtype == torch.float16 else 0.0)


def check(got, c, what, weight_step=None, **mods):
    want, tol = attention(c, weight_step=weight_step, **mods)
    got = got.double().cpu().numpy()
    real = ~np.isnan(want)
    bad = real & ~(np.abs(got - want) <= tol)
    assert not bad.any(), (f"{what}: {int(bad.sum())} of {int(real.sum())} beyond the bound, first at "
                           f"{tuple(int(i) for i in np.argwhere(bad)[0])}, worst {np.nanmax(np.where(real, np.abs(got - want) / tol, 0)):.2f}x")
