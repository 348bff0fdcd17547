"""The serving operators in captured graphs: a graph keeps its scratch to itself, whatever
is called, captured or allocated after it."""
import math

import pytest
import torch

pytestmark = [pytest.mark.gpu,
              pytest.mark.skipif(not torch.cuda.is_available(), reason="needs a CUDA device")]


class Work:
    """One call of every operator on tensors of its own, sized by M and the slots in use."""

    def __init__(self, M, n, seed):
        from aria_b200.paged import PagedKV
        g = torch.Generator(device="cuda").manual_seed(seed)
        H, dh, ps = 2, 64, 16
        per = n // ps + 2
        k, v = (torch.randn(M * per, ps, H, dh, generator=g, device="cuda").half() for _ in range(2))
        table = torch.arange(M * per, dtype=torch.int32, device="cuda").view(M, per)
        self.kv = PagedKV(k, v, table, torch.full((M,), n, dtype=torch.int32, device="cuda"))
        self.q = torch.randn(M, 4, dh, generator=g, device="cuda").half()
        self.w = torch.rand(M, H, per * ps, generator=g, device="cuda")
        self.pos = torch.arange(per * ps, dtype=torch.int32, device="cuda").expand(M, H, per * ps).contiguous()
        self.x = torch.randn(1, n, H, dh, generator=g, device="cuda").half()
        self.lse = torch.full((1, H, n), math.log(n), device="cuda")
        self.logits = torch.randn(M, 30000, generator=g, device="cuda")
        self.keep = 2 * n // 3
        self.lens_out = torch.zeros(M, dtype=torch.int32, device="cuda")
        self.outs = [torch.empty_like(self.q), torch.empty_like(self.w), torch.empty(1, H, n, device="cuda"),
                     torch.empty_like(self.w), torch.empty_like(self.pos), torch.empty_like(self.logits),
                     torch.empty(M, dtype=torch.int32, device="cuda")]

    def __call__(self):
        from aria_b200.logits import adjust
        from aria_b200.paged import attention_paged, evict, prompt_weights
        o = self.outs
        attention_paged(self.q, self.kv, out=o[0], weights=self.w, weights_out=o[1])
        prompt_weights(self.x, self.x, self.lse, out=o[2])
        # (no row that is read is written and the inputs stay: from the second call on nothing changes)
        evict(self.kv, self.w, self.pos, self.kv.lens, self.keep, weights_out=o[3],
              slot_pos_out=o[4], lens_out=self.lens_out)
        adjust(self.logits, out=o[5], token=o[6])

    def expected(self):
        self()
        self()
        torch.cuda.synchronize()
        return [o.clone() for o in self.outs]

    def clear(self):
        for o in self.outs:
            o.zero_()

    def check(self, want):
        torch.cuda.synchronize()
        for i, (a, b) in enumerate(zip(self.outs, want)):
            if i in (1, 3, 4):  # slots past the lengths are not written
                n = int(self.kv.lens[0])
                a, b = a[..., :n], b[..., :n]
            assert torch.equal(a, b), i


def _capture(work, stream):
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        work()
    return graph


def test_a_larger_call_after_the_capture():
    """What a later, larger call allocates, and everything allocated after it, is not what the
    graph writes; what the graph needs is still there."""
    small, large = Work(2, 700, 1), Work(24, 5000, 2)
    want = small.expected()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        small()  # this stream's scratch exists, at the small size
    s.synchronize()
    graph = _capture(small, s)
    with torch.cuda.stream(s):
        large()
        fills = [torch.full((size,), 7, dtype=torch.uint8, device="cuda") for size in (256, 4096, 1 << 16, 1 << 20, 1 << 21, 1 << 23)
                 for _ in range(24)]
    s.synchronize()
    for _ in range(3):
        small.clear()
        torch.cuda.synchronize()
        with torch.cuda.stream(s):
            graph.replay()
        small.check(want)
    assert all(bool((f == 7).all()) for f in fills)
    del graph


def test_first_use_inside_captures_replayed_in_reverse_order():
    """No call before the captures; then the second graph runs before the first, and eager calls on
    the captured stream between them."""
    a, b, c = Work(3, 1500, 3), Work(5, 900, 4), Work(4, 1100, 5)
    s = torch.cuda.Stream()
    ga, gb = _capture(a, s), _capture(b, s)
    wants = {}
    for w in (a, b, c):
        wants[w] = w.expected()
    for order in ((gb, ga), (ga, gb), (gb, gb, ga)):
        for w in (a, b, c):
            w.clear()
        torch.cuda.synchronize()
        with torch.cuda.stream(s):
            for g in order:
                g.replay()
                c()
        for w in (a, b, c):
            w.check(wants[w])
    del ga, gb


def test_a_replay_beside_eager_calls_on_the_captured_stream():
    """A graph replayed on another stream than the one it was captured on, while that one is busy
    with eager calls of the same operators."""
    a, c = Work(3, 3000, 6), Work(4, 2600, 7)
    want_a, want_c = a.expected(), c.expected()
    s, t = torch.cuda.Stream(), torch.cuda.Stream()
    with torch.cuda.stream(s):
        a()
        c()
    s.synchronize()
    graph = _capture(a, s)
    for _ in range(10):
        a.clear()
        c.clear()
        torch.cuda.synchronize()
        for _ in range(5):
            with torch.cuda.stream(t):
                graph.replay()
            with torch.cuda.stream(s):
                c()
        a.check(want_a)
        c.check(want_c)
    del graph


def test_several_calls_in_one_graph_grow_their_scratch():
    a, b = Work(2, 300, 8), Work(9, 2500, 9)
    want_a, want_b = a.expected(), b.expected()
    s = torch.cuda.Stream()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=s):
        a()
        b()
        a()
    for _ in range(2):
        a.clear()
        b.clear()
        graph.replay()
        a.check(want_a)
        b.check(want_b)
    del graph
