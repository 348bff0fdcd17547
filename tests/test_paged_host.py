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
