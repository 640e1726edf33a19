"""Where a status word may be: kernels write to its address, so the host refuses any other place."""

import pytest
import torch

from loopspec_b200.status import DeviceStatus, enqueue


@pytest.mark.parametrize("device", ["cpu", "meta", torch.device("cpu")])
def test_a_status_word_off_the_gpu_is_refused(device):
    with pytest.raises(ValueError):
        DeviceStatus(device)


def test_a_status_word_of_another_gpu_is_refused_before_the_call():
    status = object.__new__(DeviceStatus)
    status.gpu, status.ptr = 0, 256

    def never(*_):
        raise AssertionError("called")

    with pytest.raises(ValueError):
        enqueue(never, never, (), (), 1, status, 0)


@pytest.mark.gpu
def test_the_status_word_knows_its_gpu():
    assert DeviceStatus().gpu == DeviceStatus("cuda:0").gpu == 0
