"""Host-side logic of the serving operators' Python entry points, without a GPU: CUDA's
answers (device, stream, capture) and the library are replaced."""
import pytest
import torch

from aria_b200 import paged


@pytest.fixture
def scratch(monkeypatch):
    """Scratch on the CPU; `state` says whether a capture is under way, and which."""
    state = {"id": 0}
    empty = torch.empty
    monkeypatch.setattr(paged, "_WORKSPACES", {})
    monkeypatch.setattr(paged, "_GRAPH_WORKSPACES", {})
    monkeypatch.setattr(paged, "_capturing", lambda: state["id"] != 0)
    monkeypatch.setattr(paged, "_capture_id", lambda stream: state["id"])
    monkeypatch.setattr(torch, "empty", lambda n, dtype, device: empty(n, dtype=dtype).fill_(9))
    return state


def test_graphs_and_eager_calls_share_no_scratch(scratch):
    def get(n, stream=5):
        return paged._workspace("attn", n, 0, stream)

    eager = get(50000)
    counters = paged._lib.lib().aria_paged_workspace_counter_bytes()
    assert get(500) is eager and bool((eager[2][:counters] == 0).all()) and bool((eager[2][counters:] == 9).all())
    scratch["id"] = 11
    assert paged._held("attn", 0, 5) is paged._NO_WORKSPACE
    first = get(1000)
    assert first[0] != eager[0] and get(700)[0] == first[0] and bool((first[2] == 0).all())
    assert get(1000, stream=6)[0] != first[0]  # branches of one capture run side by side
    larger = get(3000)
    assert larger[0] != first[0] and larger[1] >= 3000
    scratch["id"] = 12                     # another graph on the same stream
    assert paged._held("attn", 0, 5) is paged._NO_WORKSPACE
    assert get(1000)[0] not in (first[0], larger[0], eager[0])
    assert list(paged._GRAPH_WORKSPACES) == [("attn", 0, 5)]  # an earlier graph's are not held on to
    scratch["id"] = 0
    assert get(1000) is eager


def test_scratch_that_is_all_counters_is_cleared_to_its_end(scratch):
    """The least allocation serves larger calls than the one that made it."""
    small = paged._workspace("logits", 12, 0, 5, "all")
    assert paged._workspace("logits", 200, 0, 5, "all") is small and bool((small[2] == 0).all())


def test_capture_id_refuses_nothing_to_write():
    from aria_b200 import _lib
    assert _lib.lib().aria_stream_capture_id(None, None) == _lib.EINVAL
    assert _lib.lib().aria_paged_workspace_counter_bytes() >= 4 * 2 * 148 * 4


class _OnDevice1:
    """A tensor of cuda:1, as far as the entry points look before they call the library."""
    is_cuda, shape = True, (1, 1, 1, 64)

    def get_device(self):
        return 1


def test_calls_are_made_with_the_tensors_device_current(monkeypatch):
    """cuda:0 is current, the tensors are on cuda:1: every call is made, with every argument it was
    given, while cuda:1 is current, and cuda:0 is current again afterwards."""
    import contextlib
    import types

    from aria_b200 import logits
    state = {"device": 0, "calls": []}

    @contextlib.contextmanager
    def device(i):
        before, state["device"] = state["device"], i
        yield
        state["device"] = before

    class Fast:
        def __getattr__(self, name):
            def record(*args):
                if state["device"] != 1:  # as the binding itself: tensors of another device take the long way
                    return None
                state["calls"].append((name, state["device"], args))
                return "made"
            return record

    monkeypatch.setattr(torch.cuda, "device", device)
    for module in (paged, logits):
        monkeypatch.setattr(module, "_current_device", lambda: state["device"])
        monkeypatch.setattr(module, "_stream", lambda i: 100 + i)
        monkeypatch.setattr(module, "_held", lambda kind, dev, stream: (0, 0, None))
        monkeypatch.setattr(module, "fastcall", Fast)
    kv = types.SimpleNamespace(_ref=1, M=1, kv_heads=1, head_dim=64, index=1, _scale=0.1, _lens_ptr=2)
    t = _OnDevice1()
    args = [object() for _ in range(12)]
    for current in (0, 1):
        state.update(device=current, calls=[])
        assert paged.attention_paged(args[0], kv, k_new=args[1], v_new=args[2], scale=0.5, out=args[3], want_lse=True,
                                     weights=args[4], weights_out=args[5], slot_pos=args[6],
                                     positions=args[7]) == "made"
        assert paged.prompt_weights(t, args[0], args[1], out=args[2], scale=0.5, first_query=7) is args[2]
        assert paged.evict(kv, args[0], args[1], args[2], 9, recent=3, sinks=2, weights_out=args[3], slot_pos_out=args[4],
                           lens_out=args[5]) is args[5]
        assert logits.adjust(t, out=args[0], history=args[1], history_lens=args[2], prompt_lens=args[3],
                             repetition=args[4], frequency=args[5], presence=args[6], bias_tokens=args[7],
                             bias_values=args[8], allowed=args[9], want_token=True, token=args[10]) == "made"
        assert [(n, d) for n, d, _ in state["calls"]] == [("attention", 1), ("prompt", 1), ("evict", 1), ("logits", 1)]
        assert state["device"] == current
        attention, prompt, evict, adjust = (c[2] for c in state["calls"])
        assert attention == (1, 1, 1, 64, 1, 0.5, 0, 0, 101, True, *args[:8])
        assert prompt == (t, args[0], args[1], args[2], 0.5, 7, 0, 0, 101)
        assert evict == (1, 1, 1, 1, 2, 9, 3, 2, 0, 0, 101, *args[:6])
        assert adjust == (0, 0, 101, True, t, *args[:11])
