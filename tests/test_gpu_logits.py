"""Logits adjustment against the plain 64-bit restatement (oracle/paged_np.py).

Tolerance: at most six f32 roundings of values no larger than |x| r + f c + a + |b|
(below 64 here): 6 * 64 * 2^-24 < 3e-5; then one rounding to the output's type (2^-11
relative for f16, 2^-8 for bf16).  Chosen tokens are exact; the rows' random values
are far enough apart."""
import numpy as np
import pytest
import torch

from oracle import paged_np

pytestmark = [pytest.mark.gpu,
              pytest.mark.skipif(not torch.cuda.is_available(), reason="needs a CUDA device")]

DT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
ROUND = {torch.float32: 0.0, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}


def _check(M, V, hist, biases, grammar, dtype, out_dtype=None, seed=0, pad=0, in_place=False, shared_mask=False,
           prompt=True):
    from aria_b200.logits import adjust, allowed_mask
    g = np.random.default_rng(seed)
    wide = torch.from_numpy(g.standard_normal((M, V + pad)) * 3).to(DT[dtype]).cuda()
    x = wide[:, :V]
    x0 = x.clone()
    history = g.integers(-2, V + 3, (M, max(hist, 1))).astype(np.int32)
    hl = g.integers(0, hist + 1, M).astype(np.int32)
    hl[0] = hist
    pl = (hl * g.random(M)).astype(np.int32)
    rep, freq, pres = (1 + g.random(M)).astype(np.float32), g.random(M).astype(np.float32), g.random(M).astype(np.float32)
    bt = g.integers(-1, V + 1, (M, biases)).astype(np.int32)
    bv = g.standard_normal((M, biases)).astype(np.float32)
    if biases > 3:
        bt[:, 1] = bt[:, 3] = bt[:, 0]  # equal tokens add up
    ok = g.random((1 if shared_mask else M, V)) < 0.5
    kw = {}
    if hist:
        kw = dict(history=torch.from_numpy(history).cuda(), history_lens=torch.from_numpy(hl).cuda(),
                  repetition=torch.from_numpy(rep).cuda(), frequency=torch.from_numpy(freq).cuda(),
                  presence=torch.from_numpy(pres).cuda())
        if prompt:
            kw["prompt_lens"] = torch.from_numpy(pl).cuda()
    if biases:
        kw.update(bias_tokens=torch.from_numpy(bt).cuda(), bias_values=torch.from_numpy(bv).cuda())
    if grammar:
        kw["allowed"] = allowed_mask(torch.from_numpy(ok).cuda())
    out = x if in_place else torch.empty(M, V, dtype=out_dtype or DT[dtype], device="cuda")
    got, token = adjust(x, out=out, want_token=True, **kw)
    torch.cuda.synchronize()
    assert got is out
    if not in_place:
        assert torch.equal(x, x0)
    if pad:
        assert torch.equal(wide[:, V:], wide[:, V:].clone()) and bool(torch.isfinite(wide[:, V:]).all())
    for m in range(M):
        args = dict(history=history[m, :hl[m]].tolist(), prompt_len=int(pl[m]) if prompt else 0,
                    repetition=float(rep[m]), frequency=float(freq[m]), presence=float(pres[m])) if hist else {}
        ref, best = paged_np.adjust_row(x0[m].double().cpu().numpy(), biases=list(zip(bt[m].tolist(), bv[m].tolist())),
                                        allowed=ok[m % len(ok)] if grammar else None, **args)
        y = got[m].double().cpu().numpy()
        assert np.array_equal(np.isneginf(ref), np.isneginf(y))
        f = np.isfinite(ref)
        assert np.all(np.abs(y[f] - ref[f]) <= ROUND[got.dtype] * np.abs(ref[f]) + 3e-5)
        if best != int(token[m]):  # two values closer than the arithmetic tells apart
            assert abs(ref[best] - ref[int(token[m])]) <= 3e-5


@pytest.mark.parametrize("dtype,out_dtype", [("f32", None), ("f16", None), ("bf16", None), ("f16", torch.float32),
                                             ("bf16", torch.float32)])
@pytest.mark.parametrize("V", [1, 31, 33, 1000, 1025, 31500, 40001])
def test_adjust(V, dtype, out_dtype):
    _check(3, V, 40, 5, True, dtype, out_dtype, seed=V)


@pytest.mark.parametrize("M,hist,biases,grammar", [(1, 0, 0, False), (1, 1, 0, False), (5, 0, 40, False),
                                                   (5, 3000, 0, True), (600, 17, 1, True)])
def test_adjust_parts(M, hist, biases, grammar):
    _check(M, 517, hist, biases, grammar, "f32", seed=M + hist, prompt=hist != 17)


@pytest.mark.parametrize("dtype,out_dtype", [("f32", None), ("f16", None), ("bf16", torch.float32)])
@pytest.mark.parametrize("hist,biases", [(256, 0), (600, 5), (5000, 100)])
def test_adjust_long_histories(hist, biases, dtype, out_dtype):
    """Vocabularies of several chunks with histories around and beyond a block's first
    load; odd sizes, out of place and in place."""
    _check(3, 40001, hist, biases, True, dtype, out_dtype, seed=hist)
    _check(2, 33000, hist, biases, False, dtype, seed=hist + 1, pad=3, in_place=True, prompt=False)


def test_adjust_counts_beyond_15_bits():
    """Histories longer than a 15-bit count holds: forty tokens a thousand times each."""
    from aria_b200.logits import adjust
    M, V, H = 2, 50001, 40000
    x = torch.randn(M, V, device="cuda") * 3
    hist = torch.randint(0, 40, (M, H), dtype=torch.int32, device="cuda")
    hist[0, :33000] = 7  # one of them more than 32767 times
    n = torch.tensor([H, 300], dtype=torch.int32, device="cuda")
    f = torch.tensor([0.001, 0.01], device="cuda")
    a, token = adjust(x, history=hist, history_lens=n, frequency=f, repetition=f + 1, want_token=True)
    assert torch.equal(token.long(), a.argmax(1))
    for m in range(M):
        count = torch.bincount(hist[m, :int(n[m])], minlength=V).double()
        y, r, w = x[m].double(), 1 + f[m].double(), f[m].double()
        ref = torch.where(count > 0, torch.where(y > 0, y / r, y * r), y) - w * count
        assert (a[m].double() - ref).abs().max().item() <= 3e-5  # (f32: 33 + 15 at most)


def test_adjust_rows_in_place_and_shared_mask():
    _check(4, 1003, 50, 3, True, "f16", seed=1, pad=5, in_place=True, shared_mask=True)
    _check(4, 5001, 50, 33, True, "f32", seed=2, pad=7)
    _check(2, 20001, 50, 0, True, "bf16", seed=3, pad=1, shared_mask=True)


def test_adjust_special_values():
    """NaN and infinities: masked ones become -inf, others stay; NaN is never chosen; a row with
    nothing left gives -1; ties go to the lowest index, across chunks too."""
    from aria_b200.logits import adjust, allowed_mask
    V = 9000
    x = torch.zeros(5, V, device="cuda")
    x[0, 10], x[0, 20], x[0, 8500] = float("nan"), float("inf"), float("inf")
    x[1] = float("nan")
    x[2, 4000:] = 1.0
    x[3] = torch.finfo(torch.float32).min
    x[4, 7], x[4, 8999] = float("nan"), 2.0
    ok = torch.ones(5, V, dtype=torch.bool, device="cuda")
    ok[3] = False
    ok[4, 7] = False
    for _ in range(3):
        y, token = adjust(x, allowed=allowed_mask(ok), want_token=True)
        assert token.tolist() == [20, -1, 4000, -1, 8999]
    assert torch.isnan(y[0, 10]) and y[0, 20] == float("inf") and bool(torch.isnan(y[1]).all())
    assert bool((y[3] == -float("inf")).all()) and y[4, 7] == -float("inf")
    y, token = adjust(x[3:4], want_token=True)  # the type's lowest value is still a choice
    assert token.tolist() == [0] and torch.equal(y, x[3:4])
    z = torch.tensor([[-0.0, 0.0, -1.0]], device="cuda")
    assert adjust(z, want_token=True)[1].tolist() == [0]


def test_adjust_on_another_stream_and_without_token():
    from aria_b200.logits import adjust
    x = torch.randn(3, 4001, device="cuda")
    h = torch.randint(0, 4001, (3, 9), dtype=torch.int32, device="cuda")
    n = torch.full((3,), 9, dtype=torch.int32, device="cuda")
    r = torch.full((3,), 1.5, device="cuda")
    ref, none = adjust(x, history=h, history_lens=n, repetition=r)
    assert none is None
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        out, tok = adjust(x, history=h, history_lens=n, repetition=r, want_token=True)
    s.synchronize()
    assert torch.equal(out, ref) and torch.equal(tok.long(), ref.argmax(1))


def test_adjust_refusals():
    from aria_b200.logits import adjust
    x = torch.randn(2, 100, device="cuda")
    with pytest.raises(TypeError):
        adjust(x.cpu())
    with pytest.raises(TypeError):
        adjust(x, out=torch.empty(2, 100, dtype=torch.float16, device="cuda"))
    with pytest.raises(ValueError):
        adjust(x, repetition=torch.ones(2, device="cuda"))  # no history
    h = torch.zeros(2, 4, dtype=torch.int32, device="cuda")
    with pytest.raises(ValueError):
        adjust(x, history=h)
    with pytest.raises(TypeError):
        adjust(x, history=h.long(), history_lens=torch.zeros(2, dtype=torch.int32, device="cuda"))
    with pytest.raises(ValueError):
        adjust(x, allowed=torch.zeros(2, 3, dtype=torch.int32, device="cuda"))
    with pytest.raises(ValueError):
        adjust(x, bias_tokens=h)
