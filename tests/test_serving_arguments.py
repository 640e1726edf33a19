"""What the Python side of the shared-prefix operators reads from tensors, and what it refuses."""

import pytest
import torch

from loopspec_b200 import _lib
from loopspec_b200.prefix_attention import prefix_attention, workspace_bytes
from loopspec_b200.qk_norm import qk_norm_rope, rope_table
from loopspec_b200.slots import SlotMap, build_slots
from loopspec_b200.status import DeviceStatus


@pytest.fixture(scope="module")
def facts():
    from loopspec_b200.build import build
    build()
    return _lib.tensor_facts()


def test_tensor_facts_refuse(facts):
    read, pointers = facts
    host = torch.zeros(4, dtype=torch.int32)
    assert read(host) is None and pointers(0, _lib.I32, host, 4) is None
    assert pointers(0, _lib.I32, None, 4) == (0,)
    assert pointers(0, _lib.I32) == ()
    for call in (lambda: read(3), lambda: pointers(0, _lib.I32, 3, 1), lambda: pointers(0, _lib.I32, host),
                 lambda: pointers(0), lambda: pointers("0", _lib.I32, host, 4), lambda: pointers(0, _lib.I32, host, "4"),
                 lambda: pointers(0, _lib.I32, *([None, 1] * 17))):
        with pytest.raises(TypeError):
            call()


@pytest.mark.gpu
def test_tensor_facts(facts):
    read, pointers = facts
    for code, dtype in ((_lib.BF16, torch.bfloat16), (_lib.F16, torch.float16), (_lib.F32, torch.float32),
                        (_lib.I32, torch.int32), (_lib.BYTE, torch.uint8), (-1, torch.int64)):
        t = torch.zeros(5, 6, dtype=dtype, device="cuda")
        assert read(t) == (t.data_ptr(), t.get_device(), code, 5, 6, 6, 1)
        part = t[1:4, ::2]
        assert read(part) == (part.data_ptr(), t.get_device(), code, 3, 3, 6, 2)
        if code >= 0:
            assert pointers(t.get_device(), code, t, 30, None, 0, t[2], 6, t, -1) == (
                t.data_ptr(), 0, t[2].data_ptr(), t.data_ptr())
            assert pointers(t.get_device(), code, t, 29) is None
            assert pointers(t.get_device(), code, part, 9) is None
            assert pointers(t.get_device(), (code + 1) % 5, t, 30) is None
            assert pointers(t.get_device() + 1, code, t, 30) is None
    assert read(torch.zeros((), device="cuda"))[2:] == (_lib.F32,)


def ints(*shape):
    return torch.zeros(*shape, dtype=torch.int32, device="cuda")


def half(*shape):
    return torch.zeros(*shape, dtype=torch.bfloat16, device="cuda")


def every_change(good, bad, call):
    """call(**good) passes; with any one argument changed it raises ValueError."""
    call(**good)
    torch.cuda.synchronize()
    for name, values in bad.items():
        for value in values:
            with pytest.raises(ValueError):
                call(**dict(good, **{name: value}))


@pytest.mark.gpu
def test_slot_arguments(facts):
    out = SlotMap(3, 8)
    good = dict(lens=ints(3), delta=ints(3), block_table=ints(3, 4), free_blocks=ints(9), free_count=ints(1),
                page_size=16, n_blocks=9, out=out, status=DeviceStatus())
    bad = dict(lens=[ints(3).cpu(), ints(4), ints(3).long(), ints(6)[::2]], delta=[ints(2), ints(3).float()],
               block_table=[ints(4), ints(3, 4).cpu(), ints(4, 3).t(), ints(3, 4).long()],
               free_blocks=[ints(9).cpu(), ints(18)[::2]], free_count=[ints(2), ints(1).long()], out=[SlotMap(4, 8)])
    every_change(good, bad, lambda **a: build_slots(**a))


@pytest.mark.gpu
def test_qk_norm_arguments(facts):
    good = dict(qkv=half(5, 8 * 64), q_weight=half(64), k_weight=half(64), rope=rope_table(10, 64), positions=ints(5),
                k_pool=half(16, 2, 64), v_pool=half(16, 2, 64), slots=ints(5), out=half(5, 4, 64),
                status=DeviceStatus())
    bad = dict(qkv=[half(5, 8 * 64).cpu(), half(5, 4 * 64), half(5, 8 * 64 + 8), half(8 * 64, 5).t(), half(5, 8, 64),
                    half(5, 8 * 64).long()],
               q_weight=[half(63), half(64).float(), half(128)[::2], half(64).cpu()],
               rope=[rope_table(10, 64).half(), rope_table(10, 64).cpu(), rope_table(10, 64)[:, :, ::2],
                     rope_table(10, 64).view(5, 4, 32)],
               positions=[ints(4), ints(5).long(), ints(5).cpu()], slots=[ints(6), ints(10)[::2]],
               k_pool=[half(16, 2, 64).cpu(), half(16, 2, 64).half(), half(8, 2, 64), half(16, 128), half(2, 16, 64).transpose(0, 1)],
               out=[half(5, 4, 64).float(), half(4, 4, 64), half(5, 64, 4).transpose(1, 2), half(5, 4, 64).cpu()])
    every_change(good, bad, lambda **a: qk_norm_rope(**a))
    with pytest.raises(ValueError):
        qk_norm_rope(**dict(good, qkv=half(17, 8 * 64), positions=ints(17), slots=None, out=None))


@pytest.mark.gpu
def test_prefix_attention_arguments(facts):
    need = workspace_bytes(3, 4, 2, 64, n_requests=3, prefix_len=40, max_new=1, max_len=32)
    good = dict(q=half(3, 4, 64), k_pool=half(96, 2, 64), v_pool=half(96, 2, 64), prefix_table=ints(3), prefix_len=40,
                block_table=ints(3, 2), lens=ints(3) + 1, token_start=torch.arange(4, dtype=torch.int32, device="cuda"),
                page_size=16, max_new=1, out=half(3, 4, 64), status=DeviceStatus(),
                workspace=torch.empty(need, dtype=torch.uint8, device="cuda"))
    bad = dict(q=[half(3, 4, 64).cpu(), half(3, 4, 32), half(3, 256), half(3, 64, 4).transpose(1, 2)],
               k_pool=[half(96, 2, 64).float(), half(95, 2, 64)], prefix_table=[None, ints(2), ints(3).long(), ints(6)[::2]],
               block_table=[ints(3, 2).cpu(), ints(2, 3).t(), ints(6)], lens=[ints(2), ints(3).long()],
               token_start=[ints(3), ints(4).cpu()], max_len=[33], out=[half(3, 4, 64).float(), half(2, 4, 64)],
               workspace=[torch.empty(need, dtype=torch.uint8), torch.empty(need // 4 + 1, device="cuda")])
    every_change(good, bad, lambda **a: prefix_attention(**a))
