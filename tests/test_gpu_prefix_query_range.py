"""fp32 queries on an f16 cache: magnitudes far from 1, in either direction, and rows of very different size in one
call. Bound: that of test_gpu_prefix_attention.py, whose score error is relative to sum |q_i k_i|."""

import pytest
import torch

from test_gpu_prefix_attention import call, make, near

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("cache", ["f16", "bf16"])
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("q_size,k_size,scale", [(1e-4, 1e3, 0.1), (1e-9, 6e3, 1e5), (2e5, 1e-2, 2e-3), (1e30, 1.0, 1e-30)])
@pytest.mark.parametrize("counts,lens,prefix,nh,nkv", [([1, 2], [40, 60], 90, 4, 2), ([1] * 30, [4] * 30, 700, 2, 2),
                                                       ([130, 140], [130, 140], 0, 64, 32)])
def test_query_magnitudes(counts, lens, prefix, nh, nkv, q_size, k_size, scale, hd, cache):
    c = list(make(counts, lens, prefix, 16, nh, nkv, hd, "f32", cache, seed=hd, spread=1.0))
    c[0] *= q_size
    c[1] = (c[1].float().clamp(-5, 5) * k_size).to(c[1].dtype)
    if nkv == 32:                                # the restatement takes its time: one kv head's rows do
        c[0] = c[0][:, :2].repeat(1, 32, 1)
        c[1], c[2] = c[1][:, :1].repeat(1, 32, 1), c[2][:, :1].repeat(1, 32, 1)
        out = call(tuple(c), 16, scale=scale)
        assert torch.equal(out.view(-1, 32, 2, hd), out[:, :2].view(-1, 1, 2, hd).expand(-1, 32, -1, -1))
        c[0], c[1], c[2] = c[0][:, :2], c[1][:, :1], c[2][:, :1]
        near(out[:, :2], tuple(c), 16, "f32", cache, scale=scale)
    else:
        near(call(tuple(c), 16, scale=scale), tuple(c), 16, "f32", cache, scale=scale)


@pytest.mark.parametrize("cache", ["f16", "bf16"])
@pytest.mark.parametrize("counts,lens,prefix,nh,nkv", [([1, 2], [40, 60], 90, 4, 2), ([1] * 30, [4] * 30, 700, 2, 2)])
def test_rows_of_different_size(counts, lens, prefix, nh, nkv, cache):
    """Rows of 0, of 1e-3 and of 1e6 beside ordinary ones; a large element beside small ones in one row."""
    c = list(make(counts, lens, prefix, 16, nh, nkv, 64, "f32", cache, seed=1, spread=1.0))
    T = c[0].shape[0]
    size = torch.tensor([0.0, 1.0, 1e-3, 1e6])[torch.arange(T * nh) % 4].view(T, nh, 1)
    c[0] = c[0] * size
    c[0][:, :, 7] = 300.0 * size[:, :, 0]
    c[1][:, :, 7] = c[1][:, :, 7] * 2.0 ** -6
    near(call(tuple(c), 16, scale=1e-2), tuple(c), 16, "f32", cache, scale=1e-2)
