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


def test_the_module_is_built_again_for_another_torch_or_python(calls, monkeypatch):
    b.build()
    for made_for in ("another torch", "another python"):
        monkeypatch.setattr(b, "facts_made_for", lambda root, made_for=made_for: made_for)
        del calls[:]
        b.build()
        assert calls == ["module", "library"]
        b.build()
        assert calls == ["module", "library", "library"]


def test_a_module_made_for_another_torch_is_refused(monkeypatch):
    import sys
    import types

    from loopspec_b200 import _lib
    monkeypatch.setattr(_lib, "_FACTS", None)
    for made_for in (("1.0.0", *sys.version_info[:2]), ("1.0.0", 3, 1)):
        old = types.ModuleType("loopspec_b200._tensor_facts")
        old.facts = old.pointers = None
        old.made_for = made_for
        monkeypatch.setitem(sys.modules, "loopspec_b200._tensor_facts", old)
        monkeypatch.setattr(sys.modules["loopspec_b200"], "_tensor_facts", old, raising=False)
        with pytest.raises(ImportError, match="made for"):
            _lib.tensor_facts()


def test_the_built_module_is_made_for_this_torch():
    from loopspec_b200 import _lib
    b.build()
    facts, pointers = _lib.tensor_facts()
    assert callable(facts) and callable(pointers)
