"""GPU: a batch served with the paged cache as a program would: ragged prompts appended and attended in chunks, then
single tokens, eagerly and as one captured graph replayed while lengths and pages change; every step's attention against
the definition in 64 bits over all keys so far, and the cached step's values against the contiguous cache's."""
import numpy as np
import pytest
import torch

import sapient_amd.ops as ops

pytestmark = pytest.mark.gpu
HEADS, KV, D, PAGE, BASE = 8, 2, 64, 16, 1e4


def reference(q, ks, vs, first):
    """Attention of rows q [n, heads, D] at positions first.. over keys ks / vs [len, kv, D], causal, in 64 bits."""
    out = np.zeros(q.shape)
    tol = np.zeros(q.shape)
    for i in range(q.shape[0]):
        for h in range(HEADS):
            k, v = ks[:first + i + 1, h * KV // HEADS], vs[:first + i + 1, h * KV // HEADS]
            s = k @ q[i, h] * D ** -0.5
            w = np.exp(s - s.max())
            w /= w.sum()
            out[i, h] = w @ v
            # the weights' f16 pieces (one in chunks) and f32 sums, relative to the weighted sizes, and the output's rounding
            tol[i, h] = (2.0 ** -11 + 2.0 ** -15) * (w @ np.abs(v)) + 2.0 ** -11 * np.abs(out[i, h]) + 2.0 ** -24
    return out, tol


class Server:
    def __init__(self, dev, prompts, steps):
        g = torch.Generator().manual_seed(3)
        self.dev, self.lens, B = dev, [0] * len(prompts), len(prompts)
        self.r = lambda *s: torch.randn(*s, generator=g).half().to(dev)
        width = -(-(max(prompts) + steps + 1) // PAGE)
        pages = B * width
        order = torch.randperm(pages, generator=g).view(B, width).int()
        self.table = order.to(dev)
        self.kc, self.vc = (torch.full((pages, KV, PAGE, D), float("nan"), dtype=torch.float16, device=dev) for _ in range(2))
        self.one = [[torch.zeros(KV, width * PAGE, D, dtype=torch.float16, device=dev) for _ in range(2)] for _ in prompts]
        self.seq_lens = torch.zeros(B, dtype=torch.int32, device=dev)
        self.ws = torch.empty(ops.paged_attention_workspace(HEADS, KV, B, width, PAGE, D), dtype=torch.uint8, device=dev)

    def check(self, q, k, v, out, turned, new):
        """After a step of `new` tokens each: the rotated rows, the caches and the attention."""
        at = 0
        for b, n in enumerate(new):
            L = self.lens[b] = self.lens[b] + n
            rows = slice(at, at + n)
            at += n
            if n == 0:
                continue
            pos = torch.arange(L - n, L, dtype=torch.int32, device=self.dev)
            want = ops.rope_kv_append_tokens(q[rows].contiguous(), k[rows].contiguous(), v[rows].contiguous(), pos, BASE, *self.one[b])
            assert torch.equal(turned[rows], want.transpose(0, 1)), "rotated q"
            ks, vs = (c[:, :L].transpose(0, 1).double().cpu().numpy() for c in self.one[b])
            ref, tol = reference(turned[rows].double().cpu().numpy(), ks, vs, L - n)
            got = out[rows].double().cpu().numpy()
            assert (np.abs(got - ref) <= tol).all(), f"attention of sequence {b} at {L}: {np.nanmax(np.abs(got - ref) / tol):.2f}x"

    def chunk(self, new):
        T = sum(new)
        q, k, v = self.r(T, HEADS, D), self.r(T, KV, D), self.r(T, KV, D)
        cu = torch.tensor(np.concatenate([[0], np.cumsum(new)]), dtype=torch.int32, device=self.dev)
        self.seq_lens += torch.tensor(new, dtype=torch.int32, device=self.dev)
        turned = ops.rope_kv_append_paged(q, k, v, self.seq_lens, self.table, BASE, self.kc, self.vc, cu_q=cu)
        out = ops.paged_attention_chunk(turned, self.kc, self.vc, self.seq_lens, self.table, cu)
        self.check(q, k, v, out, turned, new)


def test_prompts_then_single_tokens_eager_and_in_a_graph(dev):
    prompts = [37, 5, 130, 16, 1]
    s = Server(dev, prompts, 12)
    print("case prompts", flush=True)
    s.chunk(prompts)
    print("case second chunks, one sequence without", flush=True)
    s.chunk([3, 0, 1, 2, 1])
    B = len(prompts)
    q, k, v = (torch.zeros(B, h, D, dtype=torch.float16, device=dev) for h in (HEADS, KV, KV))
    turned, out = torch.empty_like(q), torch.empty_like(q)

    def step():
        ops.rope_kv_append_paged(q, k, v, s.seq_lens, s.table, BASE, s.kc, s.vc, out=turned)
        ops.paged_attention(turned, s.kc, s.vc, s.seq_lens, s.table, out=out, workspace=s.ws)

    def fill():
        for t in (q, k, v):
            t.copy_(s.r(*t.shape))
        s.seq_lens += 1

    fill()
    step()
    print("case eager step", flush=True)
    s.check(q, k, v, out, turned, [1] * B)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graphs = []
    for n in range(2):  # two graphs share the workspace
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            step()
        graphs.append(graph)
    for n in range(6):
        fill()
        torch.cuda.synchronize()
        graphs[n % 2].replay()
        torch.cuda.synchronize()
        print("case replay", n, flush=True)
        s.check(q, k, v, out, turned, [1] * B)


def test_a_finished_sequence_is_padding(dev):
    """Length 0 in a batch: no cache row changes, its output row is zeros, and the others are as without it."""
    s = Server(dev, [40, 20, 9], 2)
    s.chunk([40, 20, 9])
    q, k, v = s.r(3, HEADS, D), s.r(3, KV, D), s.r(3, KV, D)
    s.seq_lens += 1
    s.seq_lens[1] = 0
    before = s.kc.clone()
    turned = ops.rope_kv_append_paged(q, k, v, s.seq_lens, s.table, BASE, s.kc, s.vc, out=torch.full_like(q, 7.0))
    out = ops.paged_attention(turned, s.kc, s.vc, s.seq_lens, s.table)
    assert (turned[1] == 7).all() and not out[1].any()
    changed = (s.kc.view(torch.int16) != before.view(torch.int16)).any(-1).any(1).nonzero()
    assert sorted(map(tuple, changed.tolist())) == sorted([(int(s.table[0, 40 // PAGE]), 40 % PAGE), (int(s.table[2, 9 // PAGE]), 9 % PAGE)])
    pick = torch.tensor([0, 2], device=dev)
    alone = ops.paged_attention(turned[pick].contiguous(), s.kc, s.vc, s.seq_lens[pick].contiguous(), s.table[pick].contiguous())
    assert torch.allclose(out[pick].float(), alone.float(), rtol=2 ** -10, atol=1e-6)


def test_threads_on_their_own_streams_and_captured_without_a_workspace(dev):
    """Calls from several host threads at once, each with its own stream and scratch, and a captured call that allocates its
    scratch itself: the same bits as one after the other."""
    import threading
    servers = [Server(dev, [900 + 7 * i, 5, 130], 2) for i in range(3)]
    queries = []
    for s in servers:
        for t in (s.kc, s.vc):
            t.normal_()
        s.seq_lens += torch.tensor([900, 5, 130], dtype=torch.int32, device=dev)
        queries.append(s.r(3, HEADS, D))
    call = lambda s, q: ops.paged_attention(q, s.kc, s.vc, s.seq_lens, s.table)
    want = [call(s, q) for s, q in zip(servers, queries)]
    torch.cuda.synchronize()
    got, errors = [None] * 3, []

    def work(i):
        try:
            st = torch.cuda.Stream()
            with torch.cuda.stream(st):
                for _ in range(20):
                    got[i] = call(servers[i], queries[i])
            st.synchronize()
        except Exception as e:  # reported below
            errors.append(repr(e))

    print("case threads", flush=True)
    threads = [threading.Thread(target=work, args=(i,)) for i in range(3)]
    for t in threads:
        t.start()
    for t in threads:
        t.join(timeout=60)
    assert not errors and all(torch.equal(g, w) for g, w in zip(got, want)), errors
    graph, out = torch.cuda.CUDAGraph(), torch.empty_like(want[0])
    with torch.cuda.graph(graph):
        ops.paged_attention(queries[0], servers[0].kc, servers[0].vc, servers[0].seq_lens, servers[0].table, out=out)
    for n in range(3):
        out.zero_()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        print("case replay", n, flush=True)
        assert torch.equal(out, want[0])
