"""The serving operators at the sizes of a server: many long rows evicted from at once, tables far
wider than the lengths in use, rows that are part of a wider matrix."""
import numpy as np
import pytest
import torch

pytestmark = [pytest.mark.gpu,
              pytest.mark.skipif(not torch.cuda.is_available(), reason="needs a CUDA device")]


def _rows(lens, Hkv, dh, ps, width, seed):
    """Pages scattered over a pool by a table of `width` pages per sequence (-1 past the last used)."""
    g = torch.Generator().manual_seed(seed)
    M, need = len(lens), [-(-n // ps) for n in lens]
    total = sum(need) + 1
    perm = torch.randperm(total, generator=g).to(torch.int32)
    table, at = torch.full((M, width), -1, dtype=torch.int32), 0
    for m, c in enumerate(need):
        table[m, :c] = perm[at:at + c]
        at += c
    k, v = (torch.randn(total, ps, Hkv, dh, device="cuda").half() for _ in range(2))
    return k, v, table.cuda(), torch.tensor(lens, dtype=torch.int32, device="cuda")


def _reference(k, v, table, lens, w, pos, nxt, keep, recent, sinks):
    """The definition, a sequence's heads at a time: a stable sort by (always kept, weight)."""
    ek, ev, ew, ep = k.clone(), v.clone(), w.clone(), pos.clone()
    ps, H = k.shape[1], k.shape[2]
    heads = torch.arange(H, device=k.device)
    for m, n in enumerate(lens):
        if n <= keep:
            continue
        safe = (pos[m, :, :n] >= int(nxt[m]) - recent) | (pos[m, :, :n] < sinks)
        key = torch.where(safe, float("inf"), w[m, :, :n].double())
        order = key.sort(dim=1, descending=True, stable=True)[1]
        kept = torch.zeros(H, n, dtype=torch.bool, device=k.device).scatter_(1, order[:, :keep], True)
        ew[m, :, keep:n], ep[m, :, keep:n] = 0.0, -1
        tab = table[m].long()
        for h in heads.tolist():
            to, frm = torch.nonzero(~kept[h, :keep]).view(-1), torch.nonzero(kept[h, keep:]).view(-1) + keep
            ew[m, h, to], ep[m, h, to] = w[m, h, frm], pos[m, h, frm]
            for new, old in ((ek, k), (ev, v)):
                new[tab[to // ps], to % ps, h] = old[tab[frm // ps], frm % ps, h]
    return ek, ev, ew, ep


@pytest.mark.parametrize("M,Hkv,top,keep,dh,ps", [(40, 14, 3000, 1000, 64, 32), (6, 2, 9000, 4000, 64, 16),
                                                  (100, 3, 2500, 2400, 32, 24), (20, 8, 4200, 2000, 128, 64),
                                                  (300, 1, 1200, 100, 256, 16)])
def test_evict_many_long_rows(M, Hkv, top, keep, dh, ps):
    """More rows than SMs and fewer, every row long: weights, positions and both caches, bit for bit."""
    from aria_b200.paged import PagedKV, evict
    g = torch.Generator().manual_seed(M)
    lens = torch.randint(keep // 2, top + 1, (M,), generator=g).tolist()
    lens[0], lens[1] = top, keep
    k, v, table, n = _rows(lens, Hkv, dh, ps, -(-top // ps), M)
    cap = table.shape[1] * ps
    w = torch.exp(2 * torch.randn(M, Hkv, cap, device="cuda"))
    w[:, :, ::7] = w[:, :, 3:4]  # ties
    pos = torch.stack([torch.randperm(cap, generator=g) for _ in range(M)]).to(torch.int32).cuda()
    pos = pos.view(M, 1, cap).expand(M, Hkv, cap).contiguous()
    nxt = torch.full((M,), cap, dtype=torch.int32, device="cuda")
    ek, ev, ew, ep = _reference(k, v, table, lens, w, pos, nxt, keep, keep // 8, 4)
    out = evict(PagedKV(k, v, table, n), w, pos, nxt, keep, recent=keep // 8, sinks=4)
    assert torch.equal(out, n.clamp(max=keep))
    assert torch.equal(w, ew) and torch.equal(pos, ep)
    assert torch.equal(k, ek) and torch.equal(v, ev)


@pytest.mark.parametrize("lens,keep", [([2049, 2049, 700, 2050], 2048), ([300, 0, 17, 256], 256), ([5000, 4100], 300)])
def test_a_table_far_wider_than_the_lengths(lens, keep):
    """A table for 65536 slots and one that just holds the lengths: the same attention, weights and
    eviction, bit for bit."""
    from aria_b200.paged import PagedKV, attention_paged, evict
    Hkv, dh, ps, M = 3, 64, 16, len(lens)
    narrow = -(-(max(lens) + 1) // ps)
    k0, v0, table, n = _rows([x + 1 for x in lens], Hkv, dh, ps, narrow, 5)
    n -= 1
    q = torch.randn(M, 2 * Hkv, dh, device="cuda").half()
    kn, vn = (torch.randn(M, Hkv, dh, device="cuda").half() for _ in range(2))
    w0 = torch.rand(M, Hkv, 65536, device="cuda")
    p0 = torch.arange(65536, dtype=torch.int32, device="cuda").expand(M, Hkv, 65536).contiguous()
    got = []
    for width in (narrow, 65536 // ps):
        wide = torch.full((M, width), -1, dtype=torch.int32, device="cuda")
        wide[:, :narrow] = table
        cap = width * ps
        k, v, w, p = k0.clone(), v0.clone(), w0[..., :cap].contiguous(), p0[..., :cap].contiguous()
        kv = PagedKV(k, v, wide, n.clone())
        out, lse = attention_paged(q, kv, k_new=kn, v_new=vn, want_lse=True, weights=w, slot_pos=p,
                                   positions=n + 9)
        kv.lens.add_(1)
        new = evict(kv, w, p, kv.lens + 9, keep, recent=10, sinks=2)
        got.append([out, lse, new, k, v, w[..., :narrow * ps], p[..., :narrow * ps]])
        assert torch.equal(w[..., narrow * ps:], w0[..., narrow * ps:cap])
        assert torch.equal(p[..., narrow * ps:], p0[..., narrow * ps:cap])
    for a, b in zip(*got):
        assert torch.equal(a, b)


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("V,pad", [(1003, 5), (5001, 7), (20001, 1), (40000, 8)])
def test_what_lies_between_the_rows_is_not_touched(V, pad, dtype):
    """Logits that are columns of a wider matrix, adjusted in place and into another: the columns past V,
    before the call and after it."""
    from aria_b200.logits import adjust, allowed_mask
    M = 5
    hist = torch.randint(0, V, (M, 40), dtype=torch.int32, device="cuda")
    n = torch.full((M,), 40, dtype=torch.int32, device="cuda")
    r = torch.full((M,), 1.5, device="cuda")
    mask = allowed_mask(torch.rand(1, V, device="cuda") < 0.5)
    for in_place in (True, False):
        wide, other = (torch.randn(M, V + pad, device="cuda").to(dtype) for _ in range(2))
        before, other_before = wide.clone(), other.clone()
        out = wide[:, :V] if in_place else other[:, :V]
        adjust(wide[:, :V], out=out, history=hist, history_lens=n, repetition=r, allowed=mask, want_token=True)
        ref, _ = adjust(before[:, :V].contiguous(), history=hist, history_lens=n, repetition=r, allowed=mask)
        assert torch.equal(out, ref)
        assert torch.equal(wide[:, V:], before[:, V:]) and torch.equal(other[:, V:], other_before[:, V:])
        assert in_place or torch.equal(wide, before)


def test_captured_sizes_of_a_server():
    """One graph per batch size, smallest first, replayed in any order: each gives what eager calls give."""
    from aria_b200.paged import PagedKV, attention_paged
    s, cases = torch.cuda.Stream(), []
    for M in (1, 4, 16, 64):
        k, v, table, n = _rows([100 + 13 * m for m in range(M)], 2, 64, 16, 80, M)
        kv = PagedKV(k, v, table, n)
        q, w = torch.randn(M, 4, 64, device="cuda").half(), torch.rand(M, 2, 80 * 16, device="cuda")
        out, w_out = torch.empty_like(q), torch.zeros_like(w)

        def run(q=q, kv=kv, out=out, w=w, w_out=w_out):
            attention_paged(q, kv, out=out, weights=w, weights_out=w_out)

        run()
        torch.cuda.synchronize()
        want = out.clone(), w_out.clone()
        with torch.cuda.stream(s):
            run()
        s.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=s):
            run()
        cases.append((graph, out, w_out, want, run))  # (run holds the inputs that the graph reads)
    for i in np.random.default_rng(0).permutation(np.repeat(np.arange(4), 5)):
        graph, out, w_out, want, _ = cases[i]
        out.zero_()
        w_out.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want[0]) and torch.equal(w_out, want[1])
    del cases, graph
