"""Token ranges and lengths of the prefix attention that are out of their bounds, or very large."""

import pytest
import torch

from test_gpu_prefix_attention import call, make

pytestmark = pytest.mark.gpu


def test_padding_of_more_than_32_bits_of_elements():
    """A prompt of 130 tokens and 2^27 rows of padding: 2^31 pieces of four elements to clear, and one token's more."""
    from loopspec_b200.prefix_attention import prefix_attention
    nh, hd, page = 16, 64, 16
    c = make([130], [130], 0, page, nh, 1, hd, "bf16", "bf16", seed=4)
    q, k, v, prefix_table, prefix, table, lens, start = c
    n = (1 << 27) // nh + 130 + 1
    big = torch.zeros(n, nh, hd, dtype=torch.bfloat16, device="cuda")
    big[:130] = q.cuda()
    out = torch.full_like(big, 7)
    prefix_attention(big, k.cuda(), v.cuda(), None, 0, table.cuda(), lens.cuda(), start.cuda(), page_size=page, max_new=130,
                     out=out)
    assert not bool((out[:130] == 7).all(-1).any())
    for part in out[130:].split(1 << 20):
        assert not bool(part.any())
