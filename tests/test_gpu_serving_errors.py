"""What the Python entry points make of the library's statuses: the C functions are replaced by
ones that count their calls and answer with a status, launching nothing."""
import ctypes

import pytest
import torch

pytestmark = [pytest.mark.gpu,
              pytest.mark.skipif(not torch.cuda.is_available(), reason="needs a CUDA device")]

NAMES = ("aria_attention_paged", "aria_prompt_weights", "aria_cache_evict", "aria_logits_adjust")


@pytest.fixture
def answered(monkeypatch):
    """answered(status): binds functions that answer with it; returns the calls that were made, the
    short way ("fast") and the long one (by name)."""
    from aria_b200 import _lib, logits, paged
    fast, keep = _lib.fastcall(), []

    def set_to(status):
        calls = []
        addresses = []
        for name in NAMES:
            kind = ctypes.CFUNCTYPE(ctypes.c_int, *_lib.SIGNATURES[name][1])
            f = kind(lambda *a: calls.append("fast") or status)
            keep.append(f)
            addresses.append(ctypes.cast(f, ctypes.c_void_p).value)
        fast.bind(*addresses, _lib.check)
        for module in (paged, logits):
            monkeypatch.setattr(module, "call", lambda name, *a: calls.append(name))
        return calls

    yield set_to
    fast.bind(*(ctypes.cast(getattr(_lib.lib(), n), ctypes.c_void_p).value for n in NAMES), _lib.check)


def _operators():
    from aria_b200.logits import adjust
    from aria_b200.paged import PagedKV, attention_paged, evict, prompt_weights
    k, v = (torch.zeros(4, 16, 2, 64, device="cuda").half() for _ in range(2))
    kv = PagedKV(k, v, torch.arange(4, dtype=torch.int32, device="cuda").view(1, 4),
                 torch.tensor([50], dtype=torch.int32, device="cuda"))
    q = torch.zeros(1, 2, 64, device="cuda").half()
    w, p = torch.zeros(1, 2, 64, device="cuda"), torch.zeros(1, 2, 64, dtype=torch.int32, device="cuda")
    x, lse, out = torch.zeros(1, 8, 2, 64, device="cuda").half(), torch.zeros(1, 2, 8, device="cuda"), torch.zeros(
        1, 2, 8, device="cuda")
    return {"aria_attention_paged": lambda: attention_paged(q, kv, weights=w),
            "aria_prompt_weights": lambda: prompt_weights(x, x, lse, out=out),
            "aria_cache_evict": lambda: evict(kv, w, p, kv.lens + 1, 32),
            "aria_logits_adjust": lambda: adjust(torch.zeros(2, 100, device="cuda"), want_token=True)}


@pytest.mark.parametrize("name", NAMES)
def test_a_cuda_error_raises_and_nothing_is_made_twice(answered, name):
    from aria_b200._lib import ECUDA, AriaQ4Error
    run = _operators()[name]
    calls = answered(ECUDA)
    with pytest.raises(AriaQ4Error, match=name) as e:
        run()
    assert e.value.status == ECUDA and calls == ["fast"]


@pytest.mark.parametrize("name", NAMES)
def test_a_refusal_goes_the_long_way(answered, name):
    from aria_b200._lib import EALIGN, ESIZE, OK
    run = _operators()[name]
    for status in (ESIZE, EALIGN):
        calls = answered(status)
        run()
        assert calls == ["fast", name]
    calls = answered(OK)
    run()
    assert calls == ["fast"]


@pytest.mark.parametrize("n", [2**31, 2**32 + 5, -2**31 - 1, 2**40 + 20])
def test_counts_past_32_bits_are_refused(n):
    """Refused, not cut to what the lower 32 bits say."""
    from aria_b200.paged import PagedKV, evict, prompt_weights
    k, v = (torch.zeros(4, 16, 2, 64, device="cuda").half() for _ in range(2))
    kv = PagedKV(k, v, torch.arange(4, dtype=torch.int32, device="cuda").view(1, 4),
                 torch.tensor([50], dtype=torch.int32, device="cuda"))
    w, p = torch.rand(1, 2, 64, device="cuda"), torch.arange(64, dtype=torch.int32, device="cuda").expand(
        1, 2, 64).contiguous()
    w0 = w.clone()
    for kw in (dict(keep=n), dict(keep=40, recent=n), dict(keep=40, sinks=n)):
        with pytest.raises(ValueError):
            evict(kv, w, p, kv.lens + 1, **kw)
    assert torch.equal(w, w0)
    x, lse = torch.zeros(1, 8, 2, 64, device="cuda").half(), torch.zeros(1, 2, 8, device="cuda")
    for out in (None, torch.zeros(1, 2, 8, device="cuda")):
        with pytest.raises(ValueError):
            prompt_weights(x, x, lse, out=out, first_query=n)


def test_counters_left_behind_are_cleared_with_the_scratch():
    """Counters as an expired wait would leave them (set by hand): the sums of a cut call are wrong
    until the scratch is cleared, and right after."""
    from aria_b200 import paged
    g = torch.Generator(device="cuda").manual_seed(0)
    q, k = (torch.randn(1, 4096, 1, 64, generator=g, device="cuda").half() for _ in range(2))
    lse = torch.full((1, 1, 4096), 9.0, device="cuda")
    want = paged.prompt_weights(q, k, lse).clone()
    held = [w for (kind, _, _), w in paged._WORKSPACES.items() if kind == "prompt"]
    assert any(w[1] > 64 * 512 for w in held)  # the call is cut: it joins parts
    for w in held:
        w[2][:4096].view(torch.int32).fill_(1)
        w[2][4096:].zero_()  # (the parts of the call before this one)
    bad = paged.prompt_weights(q, k, lse).clone()
    paged.clear_workspaces()
    assert not paged._WORKSPACES
    assert torch.equal(paged.prompt_weights(q, k, lse), want) and not torch.equal(bad, want)
