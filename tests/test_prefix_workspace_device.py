"""The workspace is sized for the tensors' GPU, whichever is current: its need depends on the number of SMs."""

from contextlib import contextmanager
from types import SimpleNamespace

import pytest
import torch

from loopspec_b200 import _lib, prefix_attention, shared_prefix


@pytest.fixture
def current(monkeypatch):
    """The current device, as the code under test sets it: [index]."""
    now = [0]

    @contextmanager
    def device(d):
        before, now[0] = now[0], d if isinstance(d, int) else torch.device(d).index
        try:
            yield
        finally:
            now[0] = before

    monkeypatch.setattr(torch.cuda, "device", device)
    return now


class Sized(Exception):
    pass


def test_a_call_without_a_workspace(current, monkeypatch):
    def sized(*_, **__):
        raise Sized(current[0])

    def facts(t):
        return (256, 1, _lib.BF16 if t.dtype is torch.bfloat16 else _lib.I32, *t.shape, *t.stride())

    monkeypatch.setattr(_lib, "_FACTS", (facts, lambda *a: (256,) * ((len(a) - 2) // 2)))
    monkeypatch.setattr(prefix_attention, "workspace_bytes", sized)
    pool, ints = torch.zeros(32, 2, 64, dtype=torch.bfloat16), torch.zeros(4, dtype=torch.int32)
    q = torch.zeros(3, 4, 64, dtype=torch.bfloat16)
    with pytest.raises(Sized) as at:
        prefix_attention.prefix_attention(q, pool, pool, ints, 16, ints[:3, None], ints[:3], ints, page_size=16, max_new=1,
                                          out=torch.empty_like(q))
    assert at.value.args == (1,) and current == [0]


def test_a_batch(current, monkeypatch):
    def sized(*_, **__):
        raise Sized(current[0])

    monkeypatch.setattr(shared_prefix, "workspace_bytes", sized)
    monkeypatch.setattr(shared_prefix, "qk_norm_rope", lambda *a, **kw: None)
    pool = SimpleNamespace(shape=(32, 2, 64), device=torch.device("cuda", 1))
    batch = object.__new__(shared_prefix.PrefixBatch)
    vars(batch).update(n_tokens=3, k=[pool], v=[pool], rope=None, status=None, n_heads=4, prefix_len=0, max_new=1,
                       max_len=16, lens=torch.zeros(3), map=SimpleNamespace(positions=[0] * 3, slots=[0] * 3))
    with pytest.raises(Sized) as at:
        batch.attend(0, None, None, None)
    assert at.value.args == (1,) and current == [0]
