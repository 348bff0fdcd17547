"""The paged attention on values that a model should not produce but may: NaN, infinities, and
scores far apart.  Every case is compared with the 64-bit restatement at lengths that take
each way through the kernel: one CTA per pair (short, few), joined states (long), pairs
that one warp finishes (short, many)."""
import math

import numpy as np
import pytest
import torch

from oracle import paged_np

pytestmark = [pytest.mark.gpu,
              pytest.mark.skipif(not torch.cuda.is_available(), reason="needs a CUDA device")]

# of p, lse and weights: as derived in test_gpu_paged.py
REL_P = 3e-5
ROUND = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
WAYS = [(40, 1), (500, 1), (5000, 1), (40, 300), (700, 40)]


def _f64(t):
    return t.detach().float().cpu().numpy().astype(np.float64)


def _cache(n, M, H, dh, dtype, seed):
    """M sequences of n slots in pages of 16, in order."""
    from aria_b200.paged import PagedKV
    g = torch.Generator(device="cuda").manual_seed(seed)
    per = -(-n // 16)
    k, v = (torch.randn(M * per, 16, H, dh, generator=g, device="cuda").to(dtype) for _ in range(2))
    table = torch.arange(M * per, dtype=torch.int32, device="cuda").view(M, per)
    kv = PagedKV(k, v, table, torch.full((M,), n, dtype=torch.int32, device="cuda"))
    q = torch.randn(M, 2 * H, dh, generator=g, device="cuda").to(dtype)
    return kv, q, k.view(M, per * 16, H, dh)[:, :n], v.view(M, per * 16, H, dh)[:, :n]


@pytest.mark.parametrize("n,M", WAYS)
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("what", ["q nan", "key nan", "key inf", "key -inf", "keys -inf", "value nan", "value inf"])
def test_nan_and_infinities_reach_the_outputs(what, dtype, n, M):
    from aria_b200.paged import attention_paged
    H, dh, m, at = 2, 64, M // 2, n // 3
    kv, q, k, v = _cache(n, M, H, dh, dtype, n + M)
    q[m, :, 5] = torch.tensor([0.5, -0.5, 0.5, 0.5])  # (the sign that an infinite key component meets)
    if what == "q nan":
        q[m, 1, 7] = float("nan")
    elif what == "key nan":
        k[m, at, 0, 7] = float("nan")
    elif what in ("key inf", "key -inf"):
        k[m, at, 0, 5] = float(what[4:])
    elif what == "keys -inf":  # nothing left for head 0, everything +inf for head 1
        k[m, :, 0, 5] = -float("inf")
    elif what == "value nan":
        v[m, at, 0, 9] = float("nan")
    else:
        v[m, at, 0, 9] = float("inf")
    w = torch.zeros(M, H, kv.slots, device="cuda")
    out, lse = attention_paged(q, kv, want_lse=True, weights=w)
    for i in {0, m, M - 1}:
        with np.errstate(invalid="ignore"):
            ro, rl, rp = paged_np.attend(_f64(q[i]), _f64(k[i]), _f64(v[i]), 1 / math.sqrt(dh))
        rw = rp.reshape(H, 2, n).sum(1)
        o, l, ww = _f64(out[i]), _f64(lse[i]), _f64(w[i, :, :n])
        if i == m and what == "keys -inf":  # as an empty row; the weights are head 1's
            assert np.all(o[0] == 0) and l[0] == -np.inf
            ro[0], rl[0] = 0, -np.inf
        if i == m and what.startswith("value"):  # one component of the group's two heads
            assert not np.isfinite(o[:2, 9]).any()
            o[:2, 9], ro[:2, 9] = 0, 0
        assert np.array_equal(np.isnan(o), np.isnan(ro)), (what, i)
        assert np.array_equal(np.isnan(l), np.isnan(rl)) and np.array_equal(np.isnan(ww), np.isnan(rw))
        bad = np.isnan(ro)
        assert np.all((np.abs(o - ro) <= ROUND[dtype] * np.abs(ro) + REL_P * 6)[~bad])
        bad = np.isnan(rl) | np.isinf(rl)
        assert np.array_equal(l[np.isinf(rl)], rl[np.isinf(rl)]) and np.all((np.abs(l - rl) <= REL_P)[~bad])
        bad = np.isnan(rw)
        assert np.all((np.abs(ww - rw) <= REL_P * rw + 1e-6)[~bad])


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("lead", [10.0, 17.0, 17.5, 20.0, 24.0])
def test_many_small_weights_beside_one_that_leads(lead, dtype):
    """One slot (an attention sink) leads by `lead` over 32749 others; its value is 0, theirs 1: the
    output is the others' share alone.  More pairs than warps, so that each pair is one warp's.
    Weights are right to 3e-5 of themselves or (f16) 2^-40 of the largest; the output is rounded
    once, to at best 2^-25 (f16)."""
    from aria_b200.paged import PagedKV, attention_paged
    M, H, dh, n, ps = 64, 20, 32, 32750, 50
    k, v = torch.zeros(n // ps, ps, H, dh, dtype=dtype, device="cuda"), torch.ones(n // ps, ps, H, dh, dtype=dtype,
                                                                                  device="cuda")
    k[0, 5, :, 0] = lead
    v[0, 5] = 0
    table = torch.arange(n // ps, dtype=torch.int32, device="cuda").expand(M, -1).contiguous()  # one cache for all
    q = torch.zeros(M, H, dh, dtype=dtype, device="cuda")
    q[:, :, 0] = 1
    kv = PagedKV(k, v, table, torch.full((M,), n, dtype=torch.int32, device="cuda"))
    out, _ = attention_paged(q, kv, scale=1.0)
    share = (n - 1) * math.exp(-lead) / (1 + (n - 1) * math.exp(-lead))
    tol = (ROUND[dtype] + 3e-5) * share + (n * 2.0 ** -40 + 2.0 ** -25 if dtype is torch.float16 else 0)
    assert np.abs(_f64(out) - share).max() <= tol


def test_large_values_with_many_equal_weights():
    """The largest f16 value in every slot: scaled weights times it, summed over 40000 slots."""
    from aria_b200.paged import PagedKV, attention_paged
    n, H, dh = 40000, 2, 64
    k, v = (torch.full((n // 16, 16, H, dh), x, dtype=torch.float16, device="cuda") for x in (0.0, 65504.0))
    table = torch.arange(n // 16, dtype=torch.int32, device="cuda").view(1, -1)
    kv = PagedKV(k, v, table, torch.tensor([n], dtype=torch.int32, device="cuda"))
    out, _ = attention_paged(torch.ones(1, H, dh, dtype=torch.float16, device="cuda"), kv)
    assert bool((out == 65504.0).all())


@pytest.mark.parametrize("lead", [0.0, 10.0, 17.0, 17.5, 20.0])
@pytest.mark.parametrize("at", [5, 20000])
def test_log_sum_exp_of_many_small_weights_beside_one_that_leads(at, lead):
    """The sum of 32749 weights of exp(-lead) and one of 1, in one warp's running sum; lse is right
    to 3e-5 as everywhere, whatever comes first."""
    from aria_b200.paged import PagedKV, attention_paged
    M, H, dh, n, ps = 64, 20, 32, 32750, 50
    k, v = (torch.zeros(n // ps, ps, H, dh, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    k[at // ps, at % ps, :, 0] = lead
    table = torch.arange(n // ps, dtype=torch.int32, device="cuda").expand(M, -1).contiguous()
    q = torch.zeros(M, H, dh, dtype=torch.bfloat16, device="cuda")
    q[:, :, 0] = 1
    kv = PagedKV(k, v, table, torch.full((M,), n, dtype=torch.int32, device="cuda"))
    _, lse = attention_paged(q, kv, scale=1.0, want_lse=True)
    assert np.abs(_f64(lse) - lead - math.log1p((n - 1) * math.exp(-lead))).max() <= REL_P


@pytest.mark.parametrize("ps,dh", [(16, 64), (48, 64), (16, 128), (24, 64), (5, 128), (7, 256)])
@pytest.mark.parametrize("n", [0, 95, 96, 111, 240, 700])
def test_a_new_token_whose_page_is_absent(n, ps, dh):
    """Its slot is absent like any other: not stored, no part in the attention, weight 0, its position
    listed.  A second sequence, whose page is there, is not affected."""
    from aria_b200.paged import PagedKV, attention_paged
    H, M = 2, 2
    g = torch.Generator(device="cuda").manual_seed(n + ps)
    per = n // ps + 2
    k, v = (torch.randn(M * per, ps, H, dh, generator=g, device="cuda").half() for _ in range(2))
    table = torch.arange(M * per, dtype=torch.int32, device="cuda").view(M, per)
    table[0, n // ps] = -1
    kv = PagedKV(k, v, table, torch.full((M,), n, dtype=torch.int32, device="cuda"))
    q = torch.randn(M, H, dh, generator=g, device="cuda").half()
    kn, vn = (torch.randn(M, H, dh, generator=g, device="cuda").half() for _ in range(2))
    w = torch.rand(M, H, kv.slots, generator=g, device="cuda")
    pos = torch.full((M, H, kv.slots), -7, dtype=torch.int32, device="cuda")
    k0, v0, w0 = k.clone(), v.clone(), w.clone()
    out, lse = attention_paged(q, kv, k_new=kn, v_new=vn, want_lse=True, weights=w, slot_pos=pos,
                               positions=torch.tensor([50, 51], dtype=torch.int32, device="cuda"))
    torch.cuda.synchronize()
    at = 1 * per + n // ps
    assert torch.equal(k[at, n % ps], kn[1]) and torch.equal(v[at, n % ps], vn[1])
    k[at, n % ps], v[at, n % ps] = k0[at, n % ps], v0[at, n % ps]
    assert torch.equal(k, k0) and torch.equal(v, v0)
    for m in range(M):
        keys, vals = (torch.cat([x.view(M, per * ps, H, dh)[m, :n], new[m:m + 1]]) for x, new in ((k0, kn), (v0, vn)))
        present = np.ones(n + 1, dtype=bool)
        if m == 0:
            present[n // ps * ps:] = False
        ro, rl, rp = paged_np.attend(_f64(q[m]), _f64(keys), _f64(vals), dh ** -0.5, present)
        assert np.all(np.abs(_f64(out[m]) - ro) <= ROUND[torch.float16] * np.abs(ro) + REL_P * 6), m
        l = _f64(lse[m])
        assert np.array_equal(np.isinf(l), np.isinf(rl)) and np.all(np.abs(l - rl)[~np.isinf(rl)] <= REL_P)
        want = rp.copy()
        want[:, :n] += _f64(w0[m, :, :n])
        assert np.all(np.abs(_f64(w[m, :, :n + 1]) - want) <= REL_P * want + 1e-6)
        assert m == 1 or bool((w[0, :, n] == 0).all())
        assert bool((pos[m, :, n] == 50 + m).all()) and bool((pos[m, :, :n] == -7).all())
