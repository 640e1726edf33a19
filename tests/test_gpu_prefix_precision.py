"""fp32 queries behind long prefixes: the error must not grow with the number of positions.

Bound, on the 2-norm of the error over that of the result, derived for any
length: a product of a key tile takes at most 24 additions on the tensor cores
(three terms of eight steps), each off by at most 2^-23 of the running sum,
2^-24 on average; the tiles' products, sums of weights and key ranges join with
rounding to nearest, whose errors are of either sign (below 2^-22 in all). The
scores, 24 additions as well, have a root mean square of 2.5 here, and their
error is that of the weights. So 24 * 2^-24 * (1 + 2.5) + 2^-22 = 5.2e-6.
"""

import pytest
import torch

from test_gpu_prefix_attention import call, make
from test_gpu_prefix_not_finite import reference

pytestmark = pytest.mark.gpu

BOUND = 24 * 2.0 ** -24 * 3.5 + 2.0 ** -22


@pytest.mark.parametrize("cache", ["bf16", "f16"])
@pytest.mark.parametrize("counts,prefix,nh,nkv,hd", [
    ([1, 2], 8192, 4, 4, 128),                  # the stream kernel
    ([1] * 40, 32768, 32, 8, 128),              # the shared prefix, several key ranges
    ([200] * 4, 8192, 16, 16, 128),             # prompts, whole results
    ([100] * 20, 16384, 32, 8, 64),
    ([3] * 30, 16384, 32, 32, 64),
    ([300, 1, 90], 700, 28, 4, 128),
])
def test_the_error_does_not_grow_with_the_prefix(counts, prefix, nh, nkv, hd, cache):
    lens = [n + 37 * i % 90 for i, n in enumerate(counts)]
    c = make(counts, lens, prefix, 16, nh, nkv, hd, "f32", cache, seed=hd)
    ref, _, _ = reference(list(c), 16)
    error = float((call(c, 16).double() - ref).norm() / ref.norm())
    assert error <= BOUND, error


@pytest.mark.parametrize("kind", ["bf16", "f16"])
@pytest.mark.parametrize("hd", [64, 128])
def test_weights_add_up_to_one(kind, hd):
    """Where all values are 1 the output is 1, whatever 16-bit weights are rounded to: numerator and sum share it. One
    key has nearly all the weight here, 2^6.1 to 2^7.9 of the reference, the score of a key 16 before it, so nothing averages out."""
    rows = 64
    c = list(make([1] * rows, [40] * rows, 0, 16, 4, 2, hd, kind, kind, seed=3))
    q, k, table = c[0], c[1], c[5]
    q[:] = 0
    q[:, :, 0] = hd ** 0.5
    for i in range(rows):
        slots = table[i].long().repeat_interleave(16) * 16 + torch.arange(16).repeat(table.shape[1])
        k[slots[:40]] = 0
        k[slots[:40], :, 0] = -30.0
        k[slots[4], :, 0] = 0.0
        k[slots[20], :, 0] = (6.1 + 1.8 * i / rows) * 0.6931
    c[2][:] = 1
    assert bool((call(c, 16) == 1).all())
