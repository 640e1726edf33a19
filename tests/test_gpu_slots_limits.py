"""Slot maps at the edges of their ranges."""

import pytest
import torch

pytestmark = pytest.mark.gpu


def test_token_buffers_of_2_31_entries():
    """The loop over the token buffers passes the last entry without running past 32 bits."""
    from loopspec_b200.slots import SlotMap, build_slots
    from loopspec_b200.status import DeviceStatus
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    most = 2 ** 31 - 1
    status = DeviceStatus("cuda")
    out = SlotMap(1, most)
    build_slots(i32([0]), i32([3]), i32([[5]]), i32([0]), i32([0]), page_size=4, n_blocks=8, out=out, status=status)
    with pytest.raises(Exception, match="free blocks"):
        status.check()                 # no block is free: every entry says so
    build_slots(i32([1]), i32([3]), i32([[5]]), i32([0]), i32([0]), page_size=4, n_blocks=8, out=out, status=status)
    status.check()
    assert out.slots[:3].tolist() == [21, 22, 23] and out.positions[:3].tolist() == [1, 2, 3]
    for buffer, rest in ((out.slots, -1), (out.positions, 0), (out.requests, -1)):
        for part in buffer[3:].split(1 << 28):
            assert bool((part == rest).all())
