"""Slot maps at the edges of their ranges."""

import os
import subprocess
import sys

import pytest
import torch

pytestmark = pytest.mark.gpu

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

ONE_CALL = """
import sys
import torch
from loopspec_b200.slots import SlotMap, build_slots
n = int(sys.argv[1])
i32 = dict(dtype=torch.int32, device="cuda")
lens, count = torch.zeros(n, **i32), torch.tensor([n], **i32)
table, stack = torch.full((n, 1), -1, **i32), torch.arange(n - 1, -1, -1, **i32)
m = build_slots(lens, torch.ones(n, **i32), table, stack, count, page_size=4, n_blocks=n, out=SlotMap(n, n))
assert m.slots.tolist() == [4 * i for i in range(n)] and m.free_count.tolist() == [0]
"""


@pytest.mark.parametrize("n", [1, 3988, 3989, 4073, 4074, 4095, 4096, 16384])
def test_any_number_of_requests_in_a_process_that_made_no_call_before(n):
    """Around 48 KB of shared memory, which a kernel gets only if it is asked for: the first call of a process."""
    run = subprocess.run([sys.executable, "-c", ONE_CALL, str(n)], cwd=ROOT, capture_output=True, text=True, timeout=300)
    assert run.returncode == 0, run.stderr[-2000:]


@pytest.mark.parametrize("table,lens,delta", [
    ([[99, 1]], [2], [-2]),            # released: both blocks go back
    ([[0, -4]], [2], [-1]),            # cut back: one does
    ([[0, 3]], [2], [-1]),             # the first block that is not there
])
def test_a_bad_block_that_is_given_back_is_reported(table, lens, delta):
    from loopspec_b200 import _lib
    from loopspec_b200.slots import SlotMap, build_slots
    from loopspec_b200.status import DeviceStatus
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    for bad in (True, False):
        tab = i32(table if bad else [[0, 1]])
        status = DeviceStatus("cuda")
        build_slots(i32(lens), i32(delta), tab, i32([2, -1, -1]), i32([1]), page_size=1, n_blocks=3, out=SlotMap(1, 4),
                    status=status)
        if not bad:
            status.check()
            continue
        with pytest.raises(_lib.EngineError) as err:
            status.check()
        assert err.value.code == _lib.LS_EDEVICE


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
