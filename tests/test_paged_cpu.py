"""The paged-cache and logits entry points without a GPU: their refusals (every check
comes before any CUDA call), their workspace sizes, and the 64-bit restatements that the
GPU tests compare with, checked against one another and by hand."""
import ctypes

import numpy as np
import pytest

from oracle import paged_np

OK, EINVAL, EUNSUPPORTED, EALIGN, ECUDA, ENODEVICE, ESIZE = range(7)
P = ctypes.c_void_p


@pytest.fixture(scope="module")
def lib():
    from aria_b200 import _lib
    return _lib.lib()


def _kv(**kw):
    from aria_b200._lib import PagedKVStruct
    d = dict(k_pages=256, v_pages=256, page_stride=16 * 2 * 64, slot_stride=128, head_stride=64, num_pages=8,
             page_size=16, kv_heads=2, head_dim=64, dtype=1, block_table=256, table_stride=4, max_pages=4, lens=256)
    d.update(kw)
    return PagedKVStruct(**d)


def _attend(lib, kv, M=1, heads=4, q=256, q_row=256, q_head=64, kn=None, vn=None, n_row=128, n_head=64, scale=0.125,
            out=256, lse=None, wi=None, wo=None, cap=64, sp=None, pos=None, ws=256, ws_bytes=1 << 30):
    return lib.aria_attention_paged(ctypes.byref(kv) if kv is not None else None, M, heads, P(q), q_row, q_head,
                                    P(kn), P(vn), n_row, n_head, scale, P(out), 256, 64, P(lse), P(wi), P(wo), cap,
                                    P(sp), P(pos), P(ws), ws_bytes, None)


def test_attention_refusals(lib):
    assert _attend(lib, None) == EINVAL
    assert _attend(lib, _kv(), M=-1) == EINVAL
    assert _attend(lib, _kv(), heads=3) == EINVAL
    assert _attend(lib, _kv(head_dim=48)) == EUNSUPPORTED
    assert _attend(lib, _kv(dtype=0)) == EINVAL
    assert _attend(lib, _kv(page_size=0)) == EINVAL
    assert _attend(lib, _kv(table_stride=3)) == EINVAL
    assert _attend(lib, _kv(), M=5000) == EUNSUPPORTED
    assert _attend(lib, _kv(max_pages=1 << 30, table_stride=1 << 30)) == ESIZE
    assert _attend(lib, _kv(slot_stride=129)) == EALIGN
    assert _attend(lib, _kv(k_pages=264)) == EALIGN
    assert _attend(lib, _kv(lens=None)) == EINVAL
    assert _attend(lib, _kv(), q=None) == EINVAL
    assert _attend(lib, _kv(), q=258) == EALIGN
    assert _attend(lib, _kv(), q_row=4) == EALIGN
    assert _attend(lib, _kv(), kn=256) == EINVAL
    assert _attend(lib, _kv(), kn=256, vn=264) == EALIGN
    assert _attend(lib, _kv(), scale=float("nan")) == EINVAL
    assert _attend(lib, _kv(), wi=256) == EINVAL
    assert _attend(lib, _kv(), wi=256, wo=256, cap=63) == ESIZE
    assert _attend(lib, _kv(), wi=256, wo=256, sp=256, pos=256) == EINVAL  # slot_pos without a new token
    assert _attend(lib, _kv(), ws=None) == EINVAL
    assert _attend(lib, _kv(), ws=257) == EALIGN
    assert _attend(lib, _kv(), M=0) == OK
    assert _attend(lib, _kv()) in (ECUDA, ENODEVICE)  # every check passed: no device here


def test_workspaces(lib):
    size = lib.aria_attention_paged_workspace_bytes
    plain, with_w = (size(ctypes.byref(_kv()), 3, 4, w) for w in (0, 1))
    assert plain > 0 and with_w >= plain + 3 * 4 * 64 * 4
    assert size(ctypes.byref(_kv()), 3, 5, 0) == 0 and size(None, 3, 4, 0) == 0
    ev = lib.aria_cache_evict_workspace_bytes
    assert ev(ctypes.byref(_kv()), 3, 64) == 0          # nothing can be given up
    assert ev(ctypes.byref(_kv()), 3, 63) == 3 * 2 * (2 + 1) * 4
    assert ev(ctypes.byref(_kv()), 3, 10) == 3 * 2 * (2 * 10 + 1) * 4
    assert lib.aria_logits_workspace_bytes(7) == 7 * 12 and lib.aria_logits_workspace_bytes(0) == 0


def test_evict_refusals(lib):
    def call(kv=None, M=1, wi=256, wo=256, pi=256, po=256, cap=64, nxt=256, keep=32, recent=0, sinks=0, ws=256,
             nb=1 << 20, lens_out=None):
        kv = _kv() if kv is None else kv
        return lib.aria_cache_evict(ctypes.byref(kv), M, P(wi), P(wo), P(pi), P(po), cap, P(nxt), keep, recent,
                                    sinks, P(lens_out), P(ws), nb, None)
    assert call(keep=0) == EINVAL and call(recent=-1) == EINVAL and call(recent=30, sinks=3) == EINVAL
    assert call(cap=63) == ESIZE and call(nb=8) == ESIZE and call(ws=None) == EINVAL and call(ws=264) == EALIGN
    assert call(lens_out=256) == EINVAL  # the lengths themselves
    assert call(wi=None) == EINVAL and call(nxt=None) == EINVAL and call(kv=_kv(head_dim=80)) == EUNSUPPORTED
    assert call(M=0) == OK and call() in (ECUDA, ENODEVICE)


def test_prompt_refusals(lib):
    def call(q=256, k=256, s=64, dtype=1, B=1, T=8, heads=2, kvh=1, dh=64, lse=256, scale=0.1, first=0, w=256, ws=None):
        return lib.aria_prompt_weights(P(q), s, s, s, P(k), s, s, s, dtype, B, T, heads, kvh, dh, P(lse), scale, first,
                                       P(w), 8, 8, P(ws), 0, None)
    assert call(dh=32) == EUNSUPPORTED and call(dtype=0) == EINVAL and call(kvh=3) == EINVAL
    assert call(first=-1) == EINVAL and call(T=-1) == EINVAL and call(q=None) == EINVAL and call(lse=None) == EINVAL
    assert call(q=264) == EALIGN and call(s=60) == EALIGN and call(s=0) == EINVAL and call(s=1 << 40) == ESIZE
    assert call(ws=264) == EALIGN
    size = lib.aria_prompt_weights_workspace_bytes
    assert size(1, 8, 2, 1, 0) == 0 and size(64, 4096, 14, 14, 0) == 0 and size(1, 8192, 1, 1, 0) > 64 * 512
    assert call(T=0) == OK and call(B=0) == OK and call() in (ECUDA, ENODEVICE)


def test_logits_refusals(lib):
    from aria_b200._lib import LogitRulesStruct

    def call(r=None, x=256, dtype=0, row=100, M=2, V=100, out=512, odt=0, orow=100, tok=None, ws=None, nb=0):
        r = LogitRulesStruct() if r is None else r
        return lib.aria_logits_adjust(ctypes.byref(r), P(x), dtype, row, M, V, P(out), odt, orow, P(tok), P(ws), nb,
                                      None)
    assert call(V=0) == EINVAL and call(M=-1) == EINVAL and call(M=70000) == EINVAL and call(dtype=2) == EINVAL
    assert call(odt=1) == EINVAL and call(dtype=1, odt=30) == EINVAL and call(x=None) == EINVAL
    assert call(out=256, orow=104) == EINVAL and call(out=256, dtype=1, odt=0) == EINVAL  # in place, another layout
    assert call(tok=256) == EINVAL and call(tok=256, ws=256, nb=8) == ESIZE and call(tok=256, ws=264, nb=99) == EALIGN
    assert call(LogitRulesStruct(history=256, history_cap=4)) == EINVAL
    assert call(LogitRulesStruct(bias_tokens=256, biases=1)) == EINVAL
    assert call(M=0) == OK and call() in (ECUDA, ENODEVICE)


def test_restated_attention_by_hand():
    q = np.zeros((2, 4))
    k, v = np.zeros((3, 1, 4)), np.arange(12.0).reshape(3, 1, 4)
    out, lse, p = paged_np.attend(q, k, v, 1.0)
    assert np.allclose(out, v.mean(0)) and np.allclose(lse, np.log(3)) and np.allclose(p, 1 / 3)
    out, lse, p = paged_np.attend(q, k, v, 1.0, [False, True, False])
    assert np.allclose(out, v[1]) and np.allclose(lse, 0) and np.allclose(p, [0, 1, 0])
    out, lse, _ = paged_np.attend(q, k[:0], v[:0], 1.0)
    assert np.all(out == 0) and np.all(lse == -np.inf)


def test_restated_prompt_weights_equal_the_attention_row_by_row():
    g = np.random.default_rng(0)
    q, k = g.standard_normal((9, 4, 8)), g.standard_normal((9, 2, 8))
    w, lse = paged_np.prompt_weights(q, k, 0.3, 2)
    ref = np.zeros((2, 9))
    for t in range(2, 9):
        _, l, p = paged_np.attend(q[t], k[:t + 1], k[:t + 1], 0.3)
        assert np.allclose(l, lse[:, t])
        ref[:, :t + 1] += p.reshape(2, 2, -1).sum(1)
    assert np.allclose(w, ref) and np.isclose(w.sum(), 7 * 4)


def test_restated_eviction_by_hand():
    nan = float("nan")
    moves, w, pos = paged_np.evict_row([1, 5, 2, nan, 3, 5], [0, 1, 2, 3, 4, 5], 6, 3, 1, 1)
    # position 0 (sink) and 5 (newest) stay, then slot 1; slot 5 moves to slot 2
    assert moves == [(5, 2)] and w.tolist() == [1, 5, 5, 0, 0, 0] and pos.tolist() == [0, 1, 5, -1, -1, -1]
    moves, w, _ = paged_np.evict_row([2, 2, 2, 2], [9, 8, 7, 6], 100, 2, 0, 0)
    assert moves == [] and w.tolist() == [2, 2, 0, 0]


def test_restated_adjustment_by_hand():
    x, best = paged_np.adjust_row([2.0, -2.0, 1.0, 0.5, 9.0], [0, 1, 2, 2], 1, 2.0, 0.25, 1.0, [(3, 4.0)],
                                  [True, True, True, True, False])
    assert np.allclose(x[:4], [1.0, -4.0 - 1.25, 0.5 - 1.5, 4.5]) and x[4] == -np.inf and best == 3
    assert paged_np.adjust_row([1.0], allowed=[False])[1] == -1


def test_allowed_mask_words():
    import torch
    from aria_b200.logits import allowed_mask
    ok = torch.zeros(2, 70, dtype=torch.bool)
    ok[0, 31] = ok[0, 32] = ok[1, 69] = ok[1, 0] = True
    w = allowed_mask(ok)
    assert w.dtype == torch.int32 and w.shape == (2, 3)
    assert w[0].tolist() == [-2**31, 1, 0] and w[1].tolist() == [1, 0, 32]


def test_pointers_that_split_an_element_are_refused(lib):
    """Every kernel reads whole elements: a pointer between two of them never reaches a launch."""
    from aria_b200._lib import LogitRulesStruct

    def logits(r=None, x=256, dtype=0, out=512, odt=0, tok=None):
        r = LogitRulesStruct() if r is None else r
        return lib.aria_logits_adjust(ctypes.byref(r), P(x), dtype, 100, 2, 100, P(out), odt, 100, P(tok), P(256), 99,
                                      None)
    assert logits(x=258) == EALIGN and logits(out=514) == EALIGN and logits(x=257, dtype=1, odt=1) == EALIGN
    assert logits(dtype=1, out=514, odt=0) == EALIGN and logits(tok=258) == EALIGN
    assert logits(x=258, dtype=1, out=518, odt=1) in (ECUDA, ENODEVICE)
    for name in ("history", "history_lens", "prompt_lens", "repetition", "frequency", "presence", "bias_tokens",
                 "bias_values", "allowed"):
        r = dict(history=256, history_lens=256, history_cap=4, history_row=4, bias_tokens=256, bias_values=256, biases=1)
        assert logits(LogitRulesStruct(**{**r, name: 258})) == EALIGN, name
    assert _attend(lib, _kv(lens=258)) == EALIGN and _attend(lib, _kv(block_table=258)) == EALIGN
    assert _attend(lib, _kv(), out=257) == EALIGN and _attend(lib, _kv(), lse=258) == EALIGN
    assert _attend(lib, _kv(), wi=258, wo=256) == EALIGN and _attend(lib, _kv(), wi=256, wo=258) == EALIGN
    new = dict(wi=256, wo=256, kn=256, vn=256)
    assert _attend(lib, _kv(), sp=258, pos=256, **new) == EALIGN
    assert _attend(lib, _kv(), sp=256, pos=258, **new) == EALIGN

    def evict(**kw):
        a = {**dict(wi=256, wo=256, pi=256, po=256, nxt=256, lo=None), **kw}
        return lib.aria_cache_evict(ctypes.byref(_kv()), 1, P(a["wi"]), P(a["wo"]), P(a["pi"]), P(a["po"]), 64,
                                    P(a["nxt"]), 32, 0, 0, P(a["lo"]), P(256), 1 << 20, None)
    for name in ("wi", "wo", "pi", "po", "nxt", "lo"):
        assert evict(**{name: 258}) == EALIGN, name

    def prompt(lse=256, w=256):
        return lib.aria_prompt_weights(P(256), 64, 64, 64, P(256), 64, 64, 64, 1, 1, 8, 2, 1, 64, P(lse), 0.1, 0, P(w),
                                       8, 8, None, 0, None)
    assert prompt(lse=258) == EALIGN and prompt(w=258) == EALIGN and prompt() in (ECUDA, ENODEVICE)


def test_sizes_past_31_bits_are_refused(lib):
    """Sizes near 2^31, where the kernels' block counts and steps would wrap."""
    from aria_b200._lib import LogitRulesStruct
    top = 2**31 - 1

    def prompt(B, T, kvh=1, heads=None):
        return lib.aria_prompt_weights(P(256), 64, 64, 64, P(256), 64, 64, 64, 1, B, T, heads or kvh, kvh, 64, P(256),
                                       0.1, 0, P(256), 8, 8, None, 0, None)
    for T in (top, top - 126, 2**28 + 1):
        assert prompt(1, T) == ESIZE and lib.aria_prompt_weights_workspace_bytes(1, T, 1, 1, 0) == 0
    assert prompt(2**16, 2**13) == ESIZE and prompt(1, 2**20, heads=2**18 + 1) == ESIZE
    assert prompt(1, 2**28 - 128) in (ECUDA, ENODEVICE)

    def logits(V=100, **kw):
        r = LogitRulesStruct(**kw)
        return lib.aria_logits_adjust(ctypes.byref(r), P(256), 1, 8, 1, V, P(256), 1, 8, None, None, 0, None)
    assert logits(V=top) == ESIZE and logits(V=2**31 - 2**17) in (ECUDA, ENODEVICE)
    assert logits(history=256, history_lens=256, history_cap=top) == ESIZE
    assert logits(bias_tokens=256, bias_values=256, biases=top) == ESIZE
