"""Prompt weights on values that a model should not produce but may, against the 64-bit
restatement.  Tolerance: as derived in test_gpu_paged.py (terms right to 3e-5)."""
import numpy as np
import pytest
import torch

from oracle import paged_np

pytestmark = [pytest.mark.gpu,
              pytest.mark.skipif(not torch.cuda.is_available(), reason="needs a CUDA device")]


def _f64(t):
    return t.detach().float().cpu().numpy().astype(np.float64)


@pytest.mark.parametrize("dh", [64, 128])
@pytest.mark.parametrize("residue", range(16))
def test_a_nan_query_makes_the_weights_of_its_keys_nan(residue, dh):
    """At every position of 16 queries (their exponentials are computed in two ways), in a block that
    the mask cuts and in ones that it does not: NaN for keys up to the query, sound past it."""
    from aria_b200.paged import prompt_weights
    g = torch.Generator(device="cuda").manual_seed(residue)
    T, t = 600, 416 + residue
    q, k = (torch.randn(1, T, 1, dh, generator=g, device="cuda").half() for _ in range(2))
    _, rows = paged_np.prompt_weights(_f64(q[0]), _f64(k[0]), dh ** -0.5)
    ref, _ = paged_np.prompt_weights(_f64(q[0]), _f64(k[0]), dh ** -0.5, t + 1, rows)
    q[0, t, 0, 3] = float("nan")
    got = _f64(prompt_weights(q, k, torch.from_numpy(rows)[None].float().cuda())[0, 0])
    assert np.isnan(got[:t + 1]).all()
    assert np.all(np.abs(got[t + 1:] - ref[0, t + 1:]) <= 5e-5 * ref[0, t + 1:] + 1e-6)


@pytest.mark.parametrize("dh", [64, 128])
@pytest.mark.parametrize("value", ["nan", "inf", "-inf"])
def test_rows_that_saw_nothing_give_nothing_whatever_they_hold(value, dh):
    """Queries with lse -inf whose rows hold NaN or infinities, in several blocks, among sound ones."""
    from aria_b200.paged import prompt_weights
    g = torch.Generator(device="cuda").manual_seed(dh)
    T, hidden = 700, [0, 1, 130, 131, 255, 400, 402, 403, 699]
    q, k = (torch.randn(1, T, 2, dh, generator=g, device="cuda").half() for _ in range(2))
    _, rows = paged_np.prompt_weights(_f64(q[0]), _f64(k[0]), dh ** -0.5)
    rows[1, hidden] = -np.inf
    ref, _ = paged_np.prompt_weights(_f64(q[0]), _f64(k[0]), dh ** -0.5, 0, rows)
    q[0, hidden, 1, 11] = float(value)
    got = _f64(prompt_weights(q, k, torch.from_numpy(rows)[None].float().cuda())[0])
    assert np.all(np.abs(got - ref) <= 5e-5 * ref + 1e-6)


@pytest.mark.parametrize("dh", [64, 128])
@pytest.mark.parametrize("residue", range(16))
def test_terms_past_the_range_of_f32_are_infinite(residue, dh):
    """An lse far below the scores, at every position of 16 queries: exp(100) is no f32."""
    from aria_b200.paged import prompt_weights
    T, t = 400, 256 + residue
    q, k = (torch.zeros(1, T, 1, dh, device="cuda").half() for _ in range(2))
    lse = torch.full((1, 1, T), 100.0, device="cuda")
    lse[0, 0, t] = -100.0
    got = prompt_weights(q, k, lse)[0, 0]
    assert bool(torch.isinf(got[:t + 1]).all()) and bool((got[t + 1:] < 1e-40).all())
    lse[0, 0, t] = -80.0  # exp(80) is one
    got = prompt_weights(q, k, lse)[0, 0, :t + 1].double().cpu().numpy()
    assert np.all(np.abs(got / np.exp(80.0) - 1) <= 3e-5)
