"""The paged KV cache on the GPU -- attention of one new token, prompt weights and
eviction -- against plain 64-bit restatements (oracle/paged_np.py).

Tolerances, from the kernels' arithmetic.  Scores: products of 16-bit values are exact
in f32, summed in f32; with |q.k| terms adding up to at most ~100 before scaling the
sum is within 64 * 2^-24 * 100 of exact, i.e. a relative error of p below 1e-4 * scale *
log2(e) < 2e-5 at dh >= 64 (dh = 32: fewer terms); 2^x to 2^-22.  Hence p and the
weights' terms are right to 3e-5, lse to 3e-5, and an output to 3e-5 max|v| (|v| < 6)
plus its one rounding: 2^-11 |out| (f16) or 2^-8 |out| (bf16: 2^-9, twice for the
comparison's own boundary).  Moved rows, positions and lengths are exact."""
import math

import numpy as np
import pytest
import torch

from oracle import paged_np

pytestmark = [pytest.mark.gpu,
              pytest.mark.skipif(not torch.cuda.is_available(), reason="needs a CUDA device")]

REL_P = 3e-5
DT = {"f16": torch.float16, "bf16": torch.bfloat16}
ROUND = {"f16": 2.0 ** -11, "bf16": 2.0 ** -8}


def _f64(t):
    return t.detach().float().cpu().numpy().astype(np.float64)


class Cache:
    """Random pages with NaN in every row that no slot uses, scattered by a random table."""

    def __init__(self, lens, Hkv, dh, ps, width, dtype="f16", head_major=False, seed=0, extra=2):
        from aria_b200.paged import PagedKV
        g = torch.Generator().manual_seed(seed)
        M = len(lens)
        total = M * width + extra
        shape = (total, Hkv, ps, dh) if head_major else (total, ps, Hkv, dh)
        k = torch.full(shape, float("nan"), dtype=DT[dtype], device="cuda")
        v = torch.full(shape, float("nan"), dtype=DT[dtype], device="cuda")
        if head_major:
            k, v = k.transpose(1, 2), v.transpose(1, 2)
        perm = torch.randperm(total, generator=g)[:M * width].view(M, width).to(torch.int32)
        # entries past a sequence's last page point outside the pool
        self.table_cpu = perm.clone()
        for m, n in enumerate(lens):
            used = -(-(n + 1) // ps)
            self.table_cpu[m, used:] = torch.tensor([-1, total, 2**31 - 1, -2**31])[
                torch.arange(max(0, width - used)) % 4].to(torch.int32)
        self.M, self.Hkv, self.dh, self.ps, self.width = M, Hkv, dh, ps, width
        self.k, self.v = k, v
        self.rows_k, self.rows_v = [], []
        for m, n in enumerate(lens):
            rk = torch.randn(n, Hkv, dh, generator=g).to(DT[dtype])
            rv = torch.randn(n, Hkv, dh, generator=g).to(DT[dtype])
            self.rows_k.append(rk)
            self.rows_v.append(rv)
            if n:
                j = torch.arange(n)
                page = self.table_cpu[m, j // ps].long().cuda()
                off = (j % ps).cuda()
                k[page, off] = rk.cuda()
                v[page, off] = rv.cuda()
        self.table = self.table_cpu.cuda()
        self.lens = torch.tensor(lens, dtype=torch.int32, device="cuda")
        self.kv = PagedKV(k, v, self.table, self.lens)
        self.slots = ps * width

    def row(self, which, m, j):
        return which[int(self.table_cpu[m, j // self.ps]), j % self.ps]


def _check_attention(lens, Hkv, G, dh, ps, width, dtype="f16", append=False, weights=False, head_major=False, seed=0,
                     strided=True):
    from aria_b200.paged import attention_paged
    c = Cache(lens, Hkv, dh, ps, width, dtype, head_major, seed)
    g = torch.Generator().manual_seed(seed + 1)
    M, Hq = c.M, Hkv * G
    row = torch.randn(M, (Hq + 2 * Hkv) * dh + (16 if strided else 0), generator=g).to(DT[dtype]).cuda()
    q = row[:, :Hq * dh].view(M, Hq, dh)
    kn = row[:, Hq * dh:(Hq + Hkv) * dh].view(M, Hkv, dh)
    vn = row[:, (Hq + Hkv) * dh:(Hq + 2 * Hkv) * dh].view(M, Hkv, dh)
    kw, cap = {}, c.slots + 3
    if append:
        kw = dict(k_new=kn, v_new=vn)
    if weights:
        w = torch.rand(M, Hkv, cap, generator=g).cuda()
        w0 = w.clone()
        kw["weights"] = w
        if append:
            sp = torch.full((M, Hkv, cap), -7, dtype=torch.int32, device="cuda")
            kw["slot_pos"], kw["positions"] = sp, torch.arange(M, dtype=torch.int32, device="cuda") + 100
    k0 = c.k.clone()
    out, lse = attention_paged(q, c.kv, want_lse=True, **kw)
    torch.cuda.synchronize()
    got, gl = _f64(out), lse.cpu().numpy()
    for m, n in enumerate(lens):
        keys, vals = c.rows_k[m], c.rows_v[m]
        room = not append or n < c.slots
        if append and room:
            keys = torch.cat([keys, kn[m].cpu().view(1, Hkv, dh)])
            vals = torch.cat([vals, vn[m].cpu().view(1, Hkv, dh)])
            assert torch.equal(c.row(c.k, m, n), kn[m]) and torch.equal(c.row(c.v, m, n), vn[m])
        if not room:
            keys, vals = keys[:0], vals[:0]
        ro, rl, rp = paged_np.attend(_f64(q[m]), _f64(keys), _f64(vals), 1.0 / math.sqrt(dh))
        assert np.all(np.abs(got[m] - ro) <= ROUND[dtype] * np.abs(ro) + REL_P * 6), (m, n, np.abs(got[m] - ro).max())
        if len(keys) == 0:
            assert np.all(gl[m] == -np.inf) and np.all(got[m] == 0)
        else:
            assert np.all(np.abs(gl[m] - rl) <= REL_P), (m, np.abs(gl[m] - rl).max())
        if weights:
            nn = len(keys)
            ref = rp.reshape(Hkv, G, nn).sum(1)
            old = min(nn, n)
            ref[:, :old] += _f64(w0[m, :, :old])
            assert np.all(np.abs(_f64(w[m, :, :nn]) - ref) <= REL_P * ref + 1e-6)
            assert torch.equal(w[m, :, max(nn, old):], w0[m, :, max(nn, old):])
            if append:
                assert bool((sp[m, :, n:n + 1] == 100 + m).all()) if room else bool((sp[m] == -7).all())
                assert bool((sp[m, :, :n] == -7).all()) and bool((sp[m, :, n + 1:] == -7).all())
    if not append:
        assert torch.equal(torch.nan_to_num(c.k, 9.0), torch.nan_to_num(k0, 9.0))


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("dh", [32, 64, 128, 256])
@pytest.mark.parametrize("G", [1, 5, 8, 9, 20])
def test_attention_shapes(dh, G, dtype):
    """Every head size, group sizes around the 8 and 16 rows of an MMA, ragged lengths
    around the 16-slot tile and the page, one sequence empty."""
    _check_attention([0, 1, 15, 16, 17, 33, 100, 257], 2, G, dh, 16, 17, dtype, append=G % 2 == 1, weights=G > 4,
                     seed=dh + G)


@pytest.mark.parametrize("ps", [1, 3, 8, 24, 100])
@pytest.mark.parametrize("head_major", [False, True])
def test_attention_pages(ps, head_major):
    """Pages that end inside a tile, of one slot and of odd sizes, both orders of heads
    and slots."""
    _check_attention([5, 99, 0, 31], 3, 2, 64, ps, -(-100 // ps), append=True, weights=True, head_major=head_major,
                     seed=ps)


def test_attention_split_and_joined():
    """Few sequences, long: every pair is shared by many CTAs; and many short pairs next to
    a long one, whose shares begin and end inside pairs."""
    _check_attention([5000], 1, 4, 64, 16, 313, append=True, weights=True, seed=1)
    _check_attention([3001, 2], 3, 1, 128, 64, 47, "bf16", seed=2)
    _check_attention([1, 0, 4000, 2, 3, 0, 0, 1, 700] * 4, 4, 1, 64, 32, 126, append=True, seed=3)


def test_attention_many_sequences():
    """More sequences than threads of a block (their tiles are summed in rounds)."""
    _check_attention([(7 * i) % 23 for i in range(300)], 2, 1, 32, 8, 3, append=True, weights=True, seed=4)


def test_attention_full_table_and_bad_lens():
    """No room for a new token: nothing written, zeros and -inf.  Lengths past the table are
    cut to it, negative ones are empty."""
    from aria_b200.paged import attention_paged
    _check_attention([32, 31, 33 - 1], 2, 1, 64, 16, 2, append=True, weights=True, seed=5)
    c = Cache([32, 32], 2, 64, 16, 2, seed=6)
    q = torch.randn(2, 2, 64, device="cuda").half()
    ref, rl = attention_paged(q, c.kv, want_lse=True)
    c.lens.copy_(torch.tensor([1000, -5]))
    out, lse = attention_paged(q, c.kv, want_lse=True)
    assert torch.equal(out[0], ref[0]) and torch.equal(lse[0], rl[0])
    assert bool((out[1] == 0).all()) and bool((lse[1] == -math.inf).all())


def test_attention_absent_pages():
    """Pages outside the pool inside a sequence: their slots take no part; with all of them
    absent the row is empty."""
    from aria_b200.paged import attention_paged
    c = Cache([60, 40], 2, 64, 16, 4, seed=7)
    c.table[0, 1] = -1
    c.table[0, 3] = 10**9
    c.table[1] = -3
    q = torch.randn(2, 4, 64, device="cuda").half()
    w = torch.zeros(2, 2, 64, device="cuda")
    out, lse = attention_paged(q, c.kv, want_lse=True, weights=w)
    present = (np.arange(60) // 16 % 2) == 0
    ro, rl, rp = paged_np.attend(_f64(q[0]), _f64(c.rows_k[0]), _f64(c.rows_v[0]), 0.125, present)
    assert np.all(np.abs(_f64(out[0]) - ro) <= ROUND["f16"] * np.abs(ro) + REL_P * 6)
    assert np.all(np.abs(lse[0].cpu().numpy() - rl) <= REL_P)
    assert np.all(np.abs(_f64(w[0, :, :60]) - rp.reshape(2, 2, 60).sum(1)) <= REL_P)
    assert bool((out[1] == 0).all()) and bool((lse[1] == -math.inf).all()) and bool((w[1] == 0).all())


def test_attention_extreme_scores():
    """One key that takes everything, and scores far apart (+-1e4 and more): no overflow."""
    from aria_b200.paged import attention_paged
    c = Cache([200], 1, 64, 16, 13, seed=8)
    q = torch.full((1, 1, 64), 100.0, device="cuda").half()
    out, lse = attention_paged(q, c.kv, want_lse=True, scale=10.0)
    ro, rl, _ = paged_np.attend(_f64(q[0]), _f64(c.rows_k[0]), _f64(c.rows_v[0]), 10.0)
    # scores of ~1e4: f32 spacing 1e-3, so p of the winner is right to about that
    assert np.all(np.abs(_f64(out[0]) - ro) <= 2e-2) and np.all(np.abs(lse[0].cpu().numpy() - rl) <= 1e-6 * np.abs(rl) + 2e-2)


def test_attention_repeats_bit_for_bit_and_leaves_workspace_ready():
    """Joins add in a fixed order: the same call gives the same bits, also after calls of
    other shapes on the same workspace."""
    from aria_b200.paged import attention_paged
    a, b = Cache([3000, 17], 2, 64, 16, 188, seed=9), Cache([40] * 40, 4, 128, 8, 5, seed=10)
    qa, qb = torch.randn(2, 2, 64, device="cuda").half(), torch.randn(40, 8, 128, device="cuda").half()
    ra, rb = attention_paged(qa, a.kv)[0].clone(), attention_paged(qb, b.kv)[0].clone()
    for _ in range(20):
        assert torch.equal(attention_paged(qa, a.kv)[0], ra)
        assert torch.equal(attention_paged(qb, b.kv)[0], rb)


def test_attention_on_another_stream():
    from aria_b200.paged import attention_paged
    c = Cache([500, 20], 2, 64, 16, 32, seed=11)
    q = torch.randn(2, 2, 64, device="cuda").half()
    ref = attention_paged(q, c.kv)[0]
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        q2 = q * 1.0
        out = attention_paged(q2, c.kv)[0]
    s.synchronize()
    assert torch.equal(out, ref)


def test_attention_in_a_graph():
    """Captured once, replayed with advanced lengths."""
    from aria_b200.paged import attention_paged
    c = Cache([100, 7], 2, 64, 16, 10, seed=12)
    for m in range(2):  # pages for the slots to come
        c.table[m] = torch.arange(10, dtype=torch.int32, device="cuda") + 10 * m
    c.k.zero_()
    c.v.zero_()
    q, kn, vn = (torch.randn(2, 2, 64, device="cuda").half() for _ in range(3))
    out = torch.empty_like(q)
    lens0 = c.lens.clone()
    attention_paged(q, c.kv, k_new=kn, v_new=vn, out=out)
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        attention_paged(q, c.kv, k_new=kn, v_new=vn, out=out)
    s.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=s):
        attention_paged(q, c.kv, k_new=kn, v_new=vn, out=out)
        c.lens.add_(1)
    want = []
    c.lens.copy_(lens0)
    for _ in range(3):
        graph.replay()
        want.append(out.clone())
    c.lens.copy_(lens0)
    c.k.zero_()
    c.v.zero_()
    for i in range(3):
        attention_paged(q, c.kv, k_new=kn, v_new=vn, out=out)
        assert torch.equal(out, want[i])
        c.lens.add_(1)
    del graph


def test_attention_past_32_bits():
    """A pool of more than 2^31 elements and 2^32 bytes: only the last pages are used."""
    from aria_b200.paged import PagedKV, attention_paged
    ps, H, dh = 64, 8, 128
    pages = (2**31) // (ps * H * dh) + 9
    k = torch.empty(pages, ps, H, dh, dtype=torch.float16, device="cuda")
    v = torch.empty_like(k)
    n = 150
    table = torch.tensor([[pages - 1, 0, pages - 3]], dtype=torch.int32, device="cuda")
    rk, rv = (torch.randn(n, H, dh, device="cuda").half() for _ in range(2))
    j = torch.arange(n, device="cuda")
    k[table[0, j // ps].long(), j % ps] = rk
    v[table[0, j // ps].long(), j % ps] = rv
    kv = PagedKV(k, v, table, torch.tensor([n], dtype=torch.int32, device="cuda"))
    q = torch.randn(1, H, dh, device="cuda").half()
    kn, vn = (torch.randn(1, H, dh, device="cuda").half() for _ in range(2))
    out, lse = attention_paged(q, kv, k_new=kn, v_new=vn, want_lse=True)
    ro, rl, _ = paged_np.attend(_f64(q[0]), _f64(torch.cat([rk, kn])), _f64(torch.cat([rv, vn])), 1 / math.sqrt(dh))
    assert np.all(np.abs(_f64(out[0]) - ro) <= ROUND["f16"] * np.abs(ro) + REL_P * 6)
    assert np.all(np.abs(lse[0].cpu().numpy() - rl) <= REL_P)
    assert torch.equal(k[pages - 3, n - 2 * ps], kn[0])


def test_contiguous_cache_equals_the_decode_attention():
    """PagedKV.contiguous over a [M][max_seq][d] cache gives what aria_attention_decode gives
    (both right to an f16 rounding)."""
    from aria_b200._lib import call
    from aria_b200.paged import PagedKV, attention_paged
    M, max_seq, heads, dh = 3, 96, 14, 64
    d = heads * dh
    kc, vc = (torch.randn(M, max_seq, d, device="cuda").half() for _ in range(2))
    qkv = torch.randn(M, 3 * d, device="cuda").half()
    pos = torch.tensor([0, 50, 95], dtype=torch.int32, device="cuda")
    k2, v2 = kc.clone(), vc.clone()
    ref = torch.empty(M, d, dtype=torch.float16, device="cuda")
    call("aria_attention_decode", qkv.data_ptr(), M, d, heads, kc.data_ptr(), vc.data_ptr(), max_seq, pos.data_ptr(),
         ref.data_ptr(), torch.cuda.current_stream().cuda_stream)
    x = qkv.view(M, 3, heads, dh)
    out, _ = attention_paged(x[:, 0], PagedKV.contiguous(k2, v2, heads, pos), k_new=x[:, 1], v_new=x[:, 2])
    assert torch.equal(k2, kc) and torch.equal(v2, vc)
    assert np.abs(_f64(out.view(M, d)) - _f64(ref)).max() <= 4e-3


# ------------------------------------------------------------------ prompt weights
@pytest.mark.parametrize("B,T,Hkv,G,dh,dtype,first", [
    (1, 1, 1, 1, 64, "f16", 0), (2, 7, 2, 1, 64, "bf16", 3), (1, 127, 1, 2, 128, "f16", 0),
    (1, 128, 2, 1, 64, "f16", 127), (2, 129, 1, 3, 128, "bf16", 128), (1, 300, 3, 1, 64, "f16", 0),
    (3, 260, 2, 2, 64, "f16", 131), (1, 700, 1, 1, 128, "f16", 0), (1, 50, 1, 1, 64, "f16", 50),
    (1, 40, 1, 1, 64, "f16", 1000), (1, 1000, 1, 4, 64, "f16", 0), (2, 900, 1, 5, 128, "bf16", 200)])
def test_prompt_weights(B, T, Hkv, G, dh, dtype, first):
    """Lengths around the 128-position block, first queries inside, at and past the end, groups,
    both types, a packed (strided) and a dense layout; slots past T untouched.  Sums of up to
    T G terms in f32 add T G / 4 * 2^-24 to the terms' own error."""
    from aria_b200 import _lib
    from aria_b200.paged import prompt_weights
    g = torch.Generator().manual_seed(T + dh)
    Hq = Hkv * G
    row = torch.randn(B, T, (Hq + 2 * Hkv) * dh, generator=g).to(DT[dtype]).cuda()
    q = row[..., :Hq * dh].unflatten(2, (Hq, dh))
    k = row[..., Hq * dh:(Hq + Hkv) * dh].unflatten(2, (Hkv, dh))
    if B == 1:
        q, k = q.contiguous(), k.contiguous()
    scale = 1.0 / math.sqrt(dh)
    refs = [paged_np.prompt_weights(_f64(q[b]), _f64(k[b]), scale, first) for b in range(B)]
    lse = torch.from_numpy(np.stack([r[1] for r in refs])).float().cuda()
    out = torch.full((B, Hkv, T + 5), 3.0, device="cuda")
    got = prompt_weights(q, k, lse, out=out, first_query=first)
    torch.cuda.synchronize()
    assert got is out and bool((out[..., T:] == 3.0).all())
    for b in range(B):
        ref = refs[b][0]
        tol = (REL_P + T * G / 4 * 2.0 ** -24 + 2e-6) * ref + 1e-6
        assert np.all(np.abs(_f64(out[b, :, :T]) - ref) <= tol), np.abs(_f64(out[b, :, :T]) - ref).max()
    assert _lib.lib().aria_q4_take_device_error() == 0


def test_prompt_weights_rows_that_must_not_count():
    """NaN in queries before first_query and in positions after T of a longer buffer, and a row
    whose lse is -inf: none reaches the sums."""
    from aria_b200.paged import prompt_weights
    T, first = 200, 40
    x = torch.randn(1, 256, 2, 64, device="cuda").half()
    x[:, T:] = float("nan")
    q, k = x[:, :T, :1].clone(), x[:, :T, 1:]
    _, rows = paged_np.prompt_weights(_f64(q[0]), _f64(k[0]), 0.125)
    rows[0, 77] = -np.inf
    ref, _ = paged_np.prompt_weights(_f64(q[0]), _f64(k[0]), 0.125, first, rows)
    q[:, :first] = float("nan")
    lse = torch.from_numpy(rows)[None].float().cuda()
    lse[:, :, :first] = float("nan")
    got = _f64(prompt_weights(q, k, lse, first_query=first)[0])
    assert np.all(np.abs(got - ref) <= 5e-5 * ref + 1e-6)


def test_prompt_weights_of_rows_that_saw_nothing():
    """Every lse -inf: exactly zero, at both head sizes (their exponentials differ)."""
    from aria_b200.paged import prompt_weights
    for dh in (64, 128):
        q, k = (torch.randn(1, 300, 2, dh, device="cuda").half() for _ in range(2))
        lse = torch.full((1, 2, 300), -math.inf, device="cuda")
        assert bool((prompt_weights(q, k, lse) == 0).all())
        lse[0, 1, 299] = 0.0  # one query counts: exp(scale q.k) of it alone
        w = prompt_weights(q, k, lse)
        ref = np.exp(_f64(k[0, :, 1]) @ _f64(q[0, 299, 1]) / math.sqrt(dh))
        assert bool((w[0, 0] == 0).all()) and np.all(np.abs(_f64(w[0, 1]) - ref) <= 5e-5 * ref + 1e-6)


def test_prompt_weights_follow_the_prefill_attention():
    """With the lse of the prompt attention itself, every query's weights add up to 1."""
    from aria_b200.attention import attention_prefill
    from aria_b200.paged import prompt_weights
    B, T, heads, dh = 2, 300, 14, 64
    qkv = torch.randn(B * T, 3 * heads * dh, device="cuda").half()
    _, lse = attention_prefill(qkv, B, T, heads, want_lse=True)
    x = qkv.view(B, T, 3, heads, dh)
    w = prompt_weights(x[:, :, 0], x[:, :, 1], lse)
    # the attention's lse is right to 2e-3 at most (its own test), typically 1e-5
    assert torch.allclose(w.sum(2), torch.full((B, heads), float(T), device="cuda"), rtol=2e-3)


# ------------------------------------------------------------------ eviction
def _check_evict(lens, Hkv, dh, ps, width, keep, recent, sinks, dtype="f16", head_major=False, in_place=True, seed=0,
                 make_w=None):
    from aria_b200.paged import evict
    c = Cache(lens, Hkv, dh, ps, width, dtype, head_major, seed)
    g = torch.Generator().manual_seed(seed + 2)
    M, cap = c.M, c.slots + 1
    w = torch.exp(2 * torch.randn(M, Hkv, cap, generator=g))
    if make_w is not None:
        w = make_w(w)
    pos = torch.full((M, Hkv, cap), -9, dtype=torch.int32)
    nxt = torch.tensor([n + 50 for n in lens], dtype=torch.int32)
    for m, n in enumerate(lens):
        for h in range(Hkv):  # positions in any order, with gaps
            pos[m, h, :n] = torch.randperm(n + 50, generator=g)[:n].to(torch.int32)
    k0, v0 = c.k.clone(), c.v.clone()
    wd, pd = w.cuda(), pos.cuda()
    kw = {}
    wo, po = wd, pd
    if not in_place:
        wo, po = torch.full_like(wd, 5.0), torch.full_like(pd, 5)
        kw = dict(weights_out=wo, slot_pos_out=po)
    lens_out = evict(c.kv, wd, pd, nxt.cuda(), keep, recent=recent, sinks=sinks, **kw)
    torch.cuda.synchronize()
    assert lens_out.tolist() == [min(n, keep) for n in lens]
    if not in_place:
        assert torch.equal(torch.nan_to_num(wd, 7.0), torch.nan_to_num(w.cuda(), 7.0)) and torch.equal(pd, pos.cuda())
    ek, ev = k0.clone(), v0.clone()
    wr, pr = (w.clone(), pos.clone()) if in_place else (torch.full_like(w, 5.0), torch.full_like(pos, 5))
    for m, n in enumerate(lens):
        for h in range(Hkv):
            moves, nw, npos = paged_np.evict_row(w[m, h, :n].numpy(), pos[m, h, :n].numpy(), int(nxt[m]), keep, recent,
                                                 sinks)
            wr[m, h, :n], pr[m, h, :n] = torch.from_numpy(nw), torch.from_numpy(npos)
            for f, t in moves:
                pf, pt = int(c.table_cpu[m, f // ps]), int(c.table_cpu[m, t // ps])
                ek[pt, t % ps, h], ev[pt, t % ps, h] = k0[pf, f % ps, h], v0[pf, f % ps, h]
    assert torch.equal(po.cpu(), pr)
    assert torch.equal(torch.nan_to_num(wo.cpu(), 7.0), torch.nan_to_num(wr, 7.0))
    assert torch.equal(torch.nan_to_num(c.k, 7.0), torch.nan_to_num(ek, 7.0))
    assert torch.equal(torch.nan_to_num(c.v, 7.0), torch.nan_to_num(ev, 7.0))


@pytest.mark.parametrize("dh,dtype", [(32, "f16"), (64, "bf16"), (128, "f16"), (256, "f16")])
@pytest.mark.parametrize("keep,recent,sinks", [(1, 0, 0), (1, 1, 0), (16, 4, 2), (50, 0, 4), (99, 30, 0), (100, 0, 0)])
def test_evict(dh, dtype, keep, recent, sinks):
    _check_evict([100, 0, 1, keep, keep + 1, 77], 2, dh, 16, 7, keep, recent, sinks, dtype, in_place=dh != 128,
                 seed=dh + keep)


@pytest.mark.parametrize("ps,head_major", [(1, False), (5, True), (64, True)])
def test_evict_pages(ps, head_major):
    _check_evict([200, 150], 3, 64, ps, -(-200 // ps), 60, 20, 3, head_major=head_major, seed=ps)


def test_evict_one_of_many_and_clusters():
    """Long rows of few heads: eight CTAs share a row; one slot given up, and most of them."""
    _check_evict([9001], 1, 32, 64, 141, 9000, 500, 4, seed=3)
    _check_evict([9000, 8191], 1, 32, 64, 141, 1000, 100, 4, in_place=False, seed=4)


def test_evict_rows_longer_than_shared_memory():
    """Past 8 x 40960 slots the keys are read again at every pass instead of kept."""
    from aria_b200.paged import PagedKV, evict
    n, keep, dh, ps = 8 * 40 * 1024 + 77, 1000, 32, 256
    width = -(-n // ps)
    k = torch.randn(width, ps, 1, dh, device="cuda").half()
    v = torch.randn(width, ps, 1, dh, device="cuda").half()
    table = torch.arange(width, dtype=torch.int32, device="cuda").view(1, -1)
    kv = PagedKV(k, v, table, torch.tensor([n], dtype=torch.int32, device="cuda"))
    w = torch.rand(1, 1, width * ps, device="cuda")
    pos = torch.arange(width * ps, dtype=torch.int32, device="cuda").view(1, 1, -1)
    flat, w0 = k.view(-1, dh).clone(), w.cpu()
    nxt = torch.tensor([n], dtype=torch.int32, device="cuda")
    evict(kv, w, pos, nxt, keep, recent=3, sinks=2)
    moves, nw, npos = paged_np.evict_row(w0[0, 0, :n].numpy(), np.arange(n), n, keep, 3, 2)
    assert torch.equal(w[0, 0, :n].cpu(), torch.from_numpy(nw))
    assert np.array_equal(pos[0, 0, :n].cpu().numpy(), npos)
    want = flat.clone()
    f, t = (torch.tensor(x, device="cuda") for x in zip(*moves))
    want[t] = flat[f]
    assert torch.equal(k.view(-1, dh), want)


@pytest.mark.parametrize("kind", ["equal", "special", "zeros", "negative"])
def test_evict_ties_and_special_weights(kind):
    """Ties go to the lowest slot; NaN is the lowest weight; +-0 are equal; infinities and
    negative sums keep their order; more safe positions than the row needs."""
    def make(w):
        if kind == "equal":
            return (w * 2).round().clamp(max=3)
        if kind == "special":
            w.view(-1)[::5] = float("nan")
            w.view(-1)[1::7] = float("inf")
            w.view(-1)[2::11] = -float("inf")
            return w
        if kind == "zeros":
            w[:] = 0.0
            w.view(-1)[::2] = -0.0
            return w
        return -w
    _check_evict([130, 64, 300], 2, 64, 16, 19, 40, 10, 2, seed=20, make_w=make)


def test_evict_absent_pages_and_stream():
    """A row whose page is absent keeps its place in the ranking; nothing is read or written
    through it.  On another stream than the tensors' own."""
    from aria_b200.paged import evict
    c = Cache([64], 1, 64, 16, 4, seed=30)
    c.table[0, 0] = -1
    k0 = c.k.clone()
    w = torch.arange(64, dtype=torch.float32, device="cuda").view(1, 1, 64)
    pos = torch.arange(64, dtype=torch.int32, device="cuda").view(1, 1, 64)
    nxt = torch.tensor([64], dtype=torch.int32, device="cuda")
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        evict(c.kv, w, pos, nxt, 32)
    s.synchronize()
    assert w[0, 0, :32].tolist() == list(range(32, 64)) and pos[0, 0, :32].tolist() == list(range(32, 64))
    for j in range(16, 32):  # slots of the one page below keep that is there
        assert torch.equal(c.row(c.k, 0, j), c.row(k0, 0, j + 32))


# ------------------------------------------------------------------ refusals
def test_python_refusals():
    from aria_b200.paged import PagedKV, attention_paged, evict, prompt_weights
    from aria_b200._lib import AriaQ4Error
    c = Cache([5], 2, 64, 16, 2, seed=40)
    q = torch.randn(1, 4, 64, device="cuda").half()
    with pytest.raises(ValueError):
        attention_paged(q[:, :3], c.kv)                    # heads not a multiple of kv_heads
    with pytest.raises(TypeError):
        attention_paged(q.bfloat16(), c.kv)
    with pytest.raises(ValueError):
        attention_paged(q, c.kv, k_new=q[:, :2])           # k_new without v_new
    with pytest.raises(ValueError):
        attention_paged(q, c.kv, slot_pos=torch.zeros(1, 2, 32, dtype=torch.int32, device="cuda"))
    with pytest.raises(AriaQ4Error):
        attention_paged(q, c.kv, weights=torch.zeros(1, 2, 31, device="cuda"))  # shorter than the table
    odd = torch.randn(1, 4, 65, device="cuda").half()[..., :64]
    with pytest.raises(AriaQ4Error):
        attention_paged(odd, c.kv)                         # strides not multiples of 8
    with pytest.raises(TypeError):
        PagedKV(c.k.float(), c.v.float(), c.table, c.lens)
    with pytest.raises(ValueError):
        PagedKV(c.k, c.v[:1], c.table, c.lens)
    k48 = torch.zeros(2, 16, 2, 48, device="cuda").half()
    with pytest.raises(AriaQ4Error):
        attention_paged(torch.zeros(1, 2, 48, device="cuda").half(), PagedKV(k48, k48.clone(), c.table, c.lens))
    w, p = torch.zeros(1, 2, 32, device="cuda"), torch.zeros(1, 2, 32, dtype=torch.int32, device="cuda")
    nxt = torch.tensor([5], dtype=torch.int32, device="cuda")
    for bad in (dict(keep=0), dict(keep=4, recent=3, sinks=2), dict(keep=4, recent=-1)):
        with pytest.raises(AriaQ4Error):
            evict(c.kv, w, p, nxt, **bad)
    with pytest.raises(ValueError):
        evict(c.kv, w, p, nxt, 4, lens_out=c.lens)
    x = torch.zeros(1, 8, 1, 32, device="cuda").half()
    with pytest.raises(AriaQ4Error):
        prompt_weights(x, x, torch.zeros(1, 1, 8, device="cuda"))  # head size 32
    with pytest.raises(ValueError):
        prompt_weights(x, x, torch.zeros(1, 1, 7, device="cuda"))


# ------------------------------------------------------------------ the two ways from Python
class _NoFast:
    def __getattr__(self, name):
        return lambda *a: None


def test_short_and_long_way_agree(monkeypatch):
    """Every operator through the C++ binding (ctypes forbidden once the workspaces exist) and
    through ctypes alone: the same bits."""
    from aria_b200 import logits as lg
    from aria_b200 import paged
    g = torch.Generator(device="cuda").manual_seed(1)
    c = Cache([100, 37, 0], 2, 64, 16, 8, seed=50)
    q, kn, vn = (torch.randn(3, n, 64, generator=g, device="cuda").half() for n in (4, 2, 2))
    w0 = torch.rand(3, 2, 130, generator=g, device="cuda")
    p0 = torch.arange(130, dtype=torch.int32, device="cuda").expand(3, 2, 130).contiguous()
    pos = c.lens + 9
    x = torch.randn(1, 50, 2, 64, generator=g, device="cuda").half()
    lse = torch.randn(1, 2, 50, generator=g, device="cuda") + 5
    lo = torch.randn(3, 1000, generator=g, device="cuda")
    hist = torch.randint(0, 1000, (3, 20), generator=g, device="cuda", dtype=torch.int32)
    n = torch.tensor([20, 3, 0], dtype=torch.int32, device="cuda")
    r = torch.full((3,), 1.3, device="cuda")
    bt, bv = hist[:, :4].contiguous(), torch.randn(3, 4, generator=g, device="cuda")
    mask = lg.allowed_mask(torch.rand(1, 1000, generator=g, device="cuda") < 0.5)

    def everything():
        w, p, out_w = w0.clone(), p0.clone(), torch.zeros(1, 2, 50, device="cuda")
        k, v = c.k.clone(), c.v.clone()
        kv = paged.PagedKV(k, v, c.table, c.lens)
        res = list(paged.attention_paged(q, kv, k_new=kn, v_new=vn, want_lse=True, weights=w, slot_pos=p, positions=pos))
        res += paged.attention_paged(q, kv, scale=0.3, out=torch.empty_like(q))[:1]
        res += [paged.prompt_weights(x, x, lse, out=out_w, first_query=3),
                paged.evict(kv, w, p, pos, 40, recent=5, sinks=2), w, p, k.nan_to_num(), v.nan_to_num()]
        res += lg.adjust(lo, history=hist, history_lens=n, prompt_lens=n // 2, repetition=r, frequency=r, presence=r,
                         bias_tokens=bt, bias_values=bv, allowed=mask, want_token=True)
        res += lg.adjust(lo, out=torch.empty_like(lo))[:1]
        torch.cuda.synchronize()
        return res

    everything()  # the workspaces exist from here on

    def forbidden(*a):
        raise AssertionError("the long way was taken")

    with monkeypatch.context() as m:
        m.setattr(paged, "call", forbidden)
        m.setattr(lg, "call", forbidden)
        short = everything()
    with monkeypatch.context() as m:
        m.setattr(paged, "fastcall", lambda: _NoFast())
        m.setattr(lg, "fastcall", lambda: _NoFast())
        long = everything()
    assert len(short) == len(long)
    for a, b in zip(short, long):
        assert torch.equal(a, b)
