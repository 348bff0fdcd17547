"""What the build needs, and what the Python entry points do without the C++ binding."""
import os
import subprocess
import sys

import pytest

from aria_b200 import _lib, build


def test_without_torch_the_library_is_built_all_the_same(monkeypatch, capsys):
    monkeypatch.setattr(_lib, "fastcall_key", lambda: None)
    assert build.build() == build.LIB and os.path.exists(build.LIB)
    assert "_fastcall" in capsys.readouterr().err


def test_without_torch_headers_the_library_is_built_all_the_same(monkeypatch):
    import torch.utils.cpp_extension as ext
    monkeypatch.setattr(ext, "include_paths", lambda *a: ["/nonexistent"])
    monkeypatch.setattr(_lib, "fastcall_key", lambda: "another")
    assert build.build() == build.LIB


def test_the_binding_is_rebuilt_for_another_torch(monkeypatch):
    assert build.build_fastcall() == build.FASTCALL
    made = []

    def run(cmd, **kw):
        made.append(cmd)
        return subprocess.CompletedProcess(cmd, 1, "", "not run")

    monkeypatch.setattr(subprocess, "run", run)
    assert build.build_fastcall() == build.FASTCALL and not made  # fresh: nothing is run
    monkeypatch.setattr(_lib, "fastcall_key", lambda: "cpython-399 torch 99.0")
    with pytest.raises(RuntimeError, match="not run"):
        build.build_fastcall()
    assert len(made) == 1 and any("torch 99.0" in a for a in made[0])


@pytest.mark.parametrize("how", ["absent", "of another torch"])
def test_without_the_binding_every_call_goes_the_long_way(monkeypatch, how):
    import types
    monkeypatch.setattr(_lib, "_FAST", None)
    other = None if how == "absent" else types.SimpleNamespace(key="cpython-312 torch 0.1", bind=None)
    monkeypatch.setitem(sys.modules, "aria_b200._fastcall", other)
    monkeypatch.delattr(sys.modules["aria_b200"], "_fastcall", raising=False)
    if other is not None:
        monkeypatch.setattr(sys.modules["aria_b200"], "_fastcall", other, raising=False)
    fast = _lib.fastcall()
    assert fast.attention(1, 2) is None and fast.prompt() is None and fast.evict() is None and fast.logits() is None


def test_the_binding_that_was_built_is_the_one_that_is_used():
    assert build.build_fastcall() == build.FASTCALL
    fast = _lib.fastcall()
    assert fast.__name__ == "aria_b200._fastcall" and fast.key == _lib.fastcall_key()
