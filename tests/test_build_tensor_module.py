"""When the module that reads torch tensors is built beside the library."""

import importlib.util

import pytest

from loopspec_b200 import build as b


@pytest.fixture
def calls(monkeypatch, tmp_path):
    """build() with the compilers replaced: what it starts, in order."""
    started = []
    monkeypatch.setattr(b, "FACTS_OUT", str(tmp_path / "_tensor_facts.so"))
    monkeypatch.setattr(b, "OBJ_DIR", str(tmp_path))
    monkeypatch.setattr(b, "build_engine", lambda force, verbose: started.append("library") or "library")
    monkeypatch.setattr(b, "_nvcc", lambda: "/usr/local/cuda/bin/nvcc")

    class Done:
        returncode = 0

        def __init__(self, cmd, **_):
            started.append("module")
            self.out = cmd[cmd.index("-o") + 1]

        def communicate(self):
            open(self.out, "w").close()
            return "", None

    monkeypatch.setattr(b.subprocess, "Popen", Done)
    return started


def test_the_library_is_built_without_torch(calls, monkeypatch):
    import builtins
    find, real = importlib.util.find_spec, builtins.__import__

    def no_torch(name, *args, **kw):
        if name.split(".")[0] == "torch":
            raise ImportError("no torch")
        return real(name, *args, **kw)

    monkeypatch.setattr(importlib.util, "find_spec", lambda name, *a: None if name == "torch" else find(name, *a))
    monkeypatch.setattr(builtins, "__import__", no_torch)
    assert b.build() == "library" and calls == ["library"]


def test_both_are_built_with_torch_and_the_module_once(calls):
    assert b.build() == "library" and calls == ["module", "library"]
    b.build()
    assert calls == ["module", "library", "library"]
    b.build(force=True)
    assert calls[3:] == ["module", "library"]
