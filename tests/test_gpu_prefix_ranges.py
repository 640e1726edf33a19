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


@pytest.mark.parametrize("counts,nh", [([1, 1], 4), ([1] * 30, 2)])
@pytest.mark.parametrize("fault", ["max_new 0", "max_len 0", "both 0"])
def test_bounds_of_zero_are_bounds(counts, nh, fault):
    """No kernel of the requests' own positions runs then; tokens or lengths past the bound are told all the same."""
    from loopspec_b200 import _lib
    from loopspec_b200.status import DeviceStatus
    c = make(counts, [3] * len(counts), 50, 16, nh, 2, 64, "bf16", "bf16", seed=2)
    bounds = dict(max_new=0 if fault != "max_len 0" else 1, max_len=0 if fault != "max_new 0" else 16)
    status = DeviceStatus("cuda")
    out = call(c, 16, status=status, **bounds)
    assert not bool(out.any())
    with pytest.raises(_lib.EngineError) as err:
        status.check()
    assert err.value.code == _lib.LS_EDEVICE
    # and within the bounds nothing is told
    ok = make([0 if bounds["max_new"] == 0 else n for n in counts], [0 if bounds["max_len"] == 0 else 3] * len(counts), 50,
              16, nh, 2, 64, "bf16", "bf16", seed=2, pad=2)
    call(ok, 16, status=status, **bounds)
    status.check()


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
