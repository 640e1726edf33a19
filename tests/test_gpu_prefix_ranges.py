"""Token ranges and lengths of the prefix attention that are out of their bounds, or very large."""

import pytest
import torch

from test_gpu_prefix_attention import call, make

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("entry,value", [(40, -5), (40, 10 ** 6), (39, 10 ** 6), (39, -1)])
@pytest.mark.parametrize("prefix", [0, 300])
def test_a_token_range_out_of_bounds_among_prompts_leaves_valid_requests_whole(prefix, entry, value):
    """Whichever CTAs run last: tokens that a valid request holds are its own, all others get zeros."""
    from loopspec_b200 import _lib
    from loopspec_b200.status import DeviceStatus
    c = make([130] * 40, [200] * 40, prefix, 16, 32, 32, 64, "bf16", "bf16", seed=2, pad=6)
    good = call(c, 16)
    start = c[7].clone()
    start[entry] = value
    status = DeviceStatus("cuda")
    out = call((*c[:7], start), 16, max_new=130, status=status)
    with pytest.raises(_lib.EngineError) as err:
        status.check()
    assert err.value.code == _lib.LS_EDEVICE
    held = torch.zeros(out.shape[0], dtype=torch.bool, device="cuda")
    for a, b in zip(start[:-1].tolist(), start[1:].tolist()):
        if 0 <= a <= b <= out.shape[0] and b - a <= 130:
            held[a:b] = True
    assert int(held.sum()) >= 38 * 130
    assert torch.equal(out[held], good[held])
    assert not bool(out[~held].any())


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
