"""Shared-prefix attention (ls_prefix_attention) against a float64 restatement, token by token.

Tolerance, derived per case. With A the largest sum |q_i k_i| * scale and V the
largest |v| that any token sees, L the positions seen and u the unit roundoff
(2^-8 bf16, 2^-11 f16):
  a score is off by at most d = A * (hd/8 + 4) * 2^-23: fp32 accumulation of
  16-term products, the scaling, and what the split of an fp32 q leaves;
  a weight by the factor e^(2 d) and 2^-20 (exp2, rescaling, what the split of
  P leaves), and u more where P is rounded to 16 bits;
  an output by the sum over L/8 accumulations, 2^-23 of the running sum each.
So |error| <= V * (2 (2 d + 2^-20 + p) + (L/8 + 64) * 2^-23) with p = u or 0,
and half a unit of the output's own type.
"""

import pytest
import torch

from serving_reference import prefix_attention_reference

pytestmark = pytest.mark.gpu

TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
UNIT = {"bf16": 2.0 ** -8, "f16": 2.0 ** -11, "f32": 2.0 ** -24}


def make(counts, lens, prefix, page, nh, nkv, hd, kind, cache, seed=0, spread=2.5, fill=None, pad=0):
    """CPU tensors of a call; slots that no request sees hold `fill`."""
    g = torch.Generator().manual_seed(seed)
    R = len(lens)
    width = max(1, max(-(-n // page) for n in lens))
    n_prefix = -(-prefix // page)
    n_blocks = n_prefix + R * width + 2
    order = torch.randperm(n_blocks, generator=g).to(torch.int32)
    prefix_table = order[:n_prefix].clone()
    table = torch.full((R, width), -5, dtype=torch.int32)
    at = n_prefix
    for i, n in enumerate(lens):
        b = -(-n // page)
        table[i, :b] = order[at:at + b]
        at += b
    k, v = torch.randn(2, n_blocks * page, nkv, hd, generator=g).to(TYPES[cache])
    if fill is not None:
        seen = torch.zeros(n_blocks * page, dtype=torch.bool)
        for tab, n in [(prefix_table, prefix)] + [(table[i], n) for i, n in enumerate(lens)]:
            pos = torch.arange(n)
            seen[tab.long()[pos // page] * page + pos % page] = True
        k[~seen] = fill
        v[~seen] = fill
    start = [0]
    for c in counts:
        start.append(start[-1] + c)
    q = (spread * torch.randn(start[-1] + pad, nh, hd, generator=g)).to(TYPES[kind])
    i32 = lambda x: torch.tensor(x, dtype=torch.int32)  # noqa: E731
    return q, k, v, prefix_table, prefix, table, i32(lens), i32(start)


def call(c, page, max_new=None, **kw):
    from loopspec_b200.prefix_attention import prefix_attention
    q, k, v, prefix_table, prefix, table, lens, start = c
    if max_new is None:
        max_new = int((start[1:] - start[:-1]).max()) if len(lens) else 0
    return prefix_attention(q.cuda(), k.cuda(), v.cuda(), prefix_table.cuda(), prefix, table.cuda(), lens.cuda(),
                            start.cuda(), page_size=page, max_new=max_new, **kw)


def near(out, c, page, kind, cache, scale=None):
    q, k, v, prefix_table, prefix, table, lens, start = c
    hd = q.shape[2]
    ref, A, V = prefix_attention_reference(q, k, v, prefix_table, prefix, table, lens, start, page,
                                           hd ** -0.5 if scale is None else scale)
    L = prefix + int(lens.max())
    d = A * (hd / 8 + 4) * 2.0 ** -23
    p = 0.0 if kind == "f32" else UNIT[cache]
    bound = V * (2 * (2 * d + 2.0 ** -20 + p) + (L / 8 + 64) * 2.0 ** -23) + UNIT[kind] * ref.abs() + 2.0 ** -24
    err = (out.double().cpu() - ref).abs()
    assert bool((err <= bound).all()), float((err / bound).max())
    return float((err / bound).max())


ALL = [("bf16", "bf16"), ("f16", "f16"), ("f32", "bf16"), ("f32", "f16")]


@pytest.mark.parametrize("kind,cache", ALL)
@pytest.mark.parametrize("nh,nkv,hd", [(4, 4, 64), (4, 1, 64), (2, 2, 128), (32, 8, 64), (28, 4, 128), (9, 3, 64),
                                       (20, 1, 128)])
def test_decode_batch(nh, nkv, hd, kind, cache):
    c = make([1] * 5, [1, 2, 33, 64, 100], 301, 16, nh, nkv, hd, kind, cache, seed=nh)
    near(call(c, 16), c, 16, kind, cache)


@pytest.mark.parametrize("kind,cache", ALL)
@pytest.mark.parametrize("page", [1, 2, 16, 64, 1024])
@pytest.mark.parametrize("prefix", [0, 1, 15, 64, 65, 700])
def test_pages_and_prefix_lengths(page, prefix, kind, cache):
    c = make([2, 0, 1, 3], [2, 17, 1, 90], prefix, page, 4, 2, 64, kind, cache, seed=page + prefix)
    near(call(c, page), c, page, kind, cache)


@pytest.mark.parametrize("kind,cache", ALL)
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("counts,lens", [([70, 0, 129], [70, 0, 140]), ([1, 200], [513, 200]), ([33], [33]),
                                         ([16, 5, 17, 64], [16, 300, 17, 65])])
def test_many_new_tokens_are_causal(counts, lens, hd, kind, cache):
    c = make(counts, lens, 130, 16, 6, 2, hd, kind, cache, seed=sum(counts))
    near(call(c, 16), c, 16, kind, cache)


@pytest.mark.parametrize("kind,cache", ALL)
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("requests,prefix,nh,nkv", [(40, 1500, 16, 16), (70, 900, 8, 2), (150, 640, 4, 1),
                                                    (300, 257, 2, 1)])
def test_many_rows_share_the_prefix(requests, prefix, nh, nkv, hd, kind, cache):
    c = make([1] * requests, [1 + 5 * i % 37 for i in range(requests)], prefix, 16, nh, nkv, hd, kind, cache,
             seed=requests)
    near(call(c, 16), c, 16, kind, cache)


@pytest.mark.parametrize("kind,cache", ALL)
def test_long_prefix_and_sharp_scores(kind, cache):
    """Scores with a spread of about 20: the running maximum moves, weights span the whole range."""
    c = make([1, 2], [40, 300], 6000, 1, 2, 1, 128, kind, cache, seed=9, spread=20.0)
    near(call(c, 1), c, 1, kind, cache)


@pytest.mark.parametrize("kind,cache", ALL)
@pytest.mark.parametrize("direction", [1, -1])
def test_maximum_that_climbs_or_falls(kind, cache, direction):
    """Scores that rise (or fall) by ~0.1 a position along the prefix."""
    c = list(make([1, 1], [3, 3], 1000, 16, 2, 2, 64, kind, cache, seed=3, spread=1.0))
    q, k, table = c[0], c[1], c[3]
    q[:] = 1.0
    pos = torch.arange(1000)
    ramp = (direction * 0.1 * pos / 8.0)[:, None, None].expand(1000, 2, 64)
    k[table.long()[pos // 16] * 16 + pos % 16] = ramp.to(k.dtype)
    near(call(tuple(c), 16), tuple(c), 16, kind, cache)


@pytest.mark.parametrize("kind,cache", ALL)
@pytest.mark.parametrize("fill", [float("nan"), float("inf"), -3.0e38])
def test_slots_that_nobody_sees_do_not_matter(kind, cache, fill):
    """NaN, infinities and the types' lowest values past a length, in a page's tail and in free blocks."""
    for counts, lens, nh in (([1, 3, 0, 2], [1, 77, 5, 30], 4), ([40, 0, 90], [40, 3, 100], 8)):
        c = make(counts, lens, 83, 32, nh, 2, 64, kind, cache, seed=5, fill=fill)
        near(call(c, 32), c, 32, kind, cache)


@pytest.mark.parametrize("kind,cache", ALL)
@pytest.mark.parametrize("counts,lens,nh", [([4, 2], [9, 40], 4), ([60, 90], [60, 100], 8)])
def test_a_later_token_that_is_not_finite_leaves_the_earlier_ones_alone(kind, cache, counts, lens, nh):
    c = make(counts, lens, 50, 16, nh, 2, 64, kind, cache, seed=6)
    want = call(c, 16)
    q, k, v, _, _, table, ln, start = c
    spoiled = [(0, lens[0] - 1), (1, lens[1] - 1)]
    for i, pos in spoiled:
        slot = int(table[i, pos // 16]) * 16 + pos % 16
        k[slot] = float("nan")
        v[slot] = float("inf") if i else float("nan")
    got = call(c, 16)
    keep = torch.ones(q.shape[0], dtype=torch.bool)
    keep[[int(start[1]) - 1, int(start[2]) - 1]] = False
    ref_ok = torch.isfinite(got.float()).flatten(1).all(1).cpu()
    assert bool(ref_ok[keep].all()) and not bool(ref_ok[~keep].any())
    near(torch.where(keep[:, None, None].cuda(), got, want), make(counts, lens, 50, 16, nh, 2, 64, kind, cache, seed=6),
         16, kind, cache)


def test_tokens_that_see_nothing_and_padding_get_zeros():
    from loopspec_b200.status import DeviceStatus
    status = DeviceStatus("cuda")
    # request 0: 3 new tokens but 1 position, so its first two see nothing; 2 tokens of padding
    c = make([3, 1, 0], [1, 4, 7], 0, 16, 4, 2, 64, "bf16", "bf16", seed=8, pad=2)
    out = call(c, 16, status=status)
    near(out, c, 16, "bf16", "bf16")
    assert not bool(out[[0, 1, 4, 5]].any()) and bool(out[2].any()) and bool(out[3].any())
    # no tokens at all
    e = make([0, 0], [5, 0], 20, 16, 4, 2, 64, "bf16", "bf16")
    assert call(e, 16, max_new=1, status=status).shape == (0, 4, 64)
    # neither prefix nor own positions
    z = make([1, 1], [0, 0], 0, 16, 4, 2, 64, "f32", "bf16")
    assert not bool(call(z, 16, status=status).any())
    status.check()


@pytest.mark.parametrize("kind,cache", ALL)
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("counts,lens,prefix,nh,nkv", [
    ([64], [64], 300, 2, 1),                      # one tile of 128 rows
    ([64, 64], [64, 190], 0, 4, 2),               # no prefix
    ([200], [200], 9000, 2, 1),                   # few rows, long prefix: several key ranges
    ([300, 1, 40], [300, 1, 129], 513, 9, 3),     # requests of one and of several tiles
    ([130, 140], [128, 100], 0, 4, 4),            # more new tokens than positions: the first see nothing
    ([256, 257], [256, 513], 127, 1, 1),
    ([200], [1500], 200, 8, 2),                   # own positions in several key ranges
])
def test_prompts_behind_a_prefix(counts, lens, prefix, nh, nkv, hd, kind, cache):
    c = make(counts, lens, prefix, 16, nh, nkv, hd, kind, cache, seed=sum(counts) + prefix, pad=3, fill=float("nan"))
    out = call(c, 16)
    near(out, c, 16, kind, cache)
    assert not bool(out[-3:].any())


@pytest.mark.parametrize("kind,cache", ALL)
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("requests,nh,nkv", [(20, 32, 32), (40, 128, 32)])
def test_many_key_tiles_in_one_unit(requests, nh, nkv, hd, kind, cache):
    """Enough kv heads that a unit walks many key tiles: every stage of its ring is used several times."""
    prefix = 2600 if requests == 20 else 1400
    c = make([1] * requests, [1 + i % 3 for i in range(requests)], prefix, 16, nh, nkv, hd, kind, cache, seed=hd)
    near(call(c, 16), c, 16, kind, cache)


@pytest.mark.parametrize("kind,cache", [("bf16", "bf16"), ("f16", "f16")])
def test_nan_in_the_prefix_reaches_every_row_and_only_its_dimensions(kind, cache):
    """A NaN key spoils all rows of its kv head; an infinite value only its own dimension."""
    for counts, lens, nh in (([1] * 30, [4] * 30, 2), ([1, 1], [4, 4], 2), ([100, 120], [100, 120], 4)):
        c = make(counts, lens, 700, 16, nh, 2, 64, kind, cache, seed=12)
        k, v, table = c[1], c[2], c[3]
        slots = table.long().repeat_interleave(16) * 16 + torch.arange(16).repeat(len(table))
        for pos in (3, 130, 255, 699):
            bad = (c[0], k.clone(), v.clone(), *c[3:])
            bad[1][slots[pos], 1] = float("nan")
            bad[2][slots[pos], 0, 5] = float("inf")
            out = call(bad, 16).float()
            G = nh // 2
            assert bool(torch.isnan(out[:, G:]).all())
            assert bool(torch.isinf(out[:, :G, 5]).all())
            rest = torch.ones(64, dtype=torch.bool)
            rest[5] = False
            assert bool(torch.isfinite(out[:, :G][..., rest.cuda()]).all())


@pytest.mark.parametrize("kind,cache", [("bf16", "bf16"), ("f32", "f16")])
def test_strides_scale_and_bounds(kind, cache):
    """q inside packed rows, pools interleaved, a wide table, generous bounds, another scale."""
    from loopspec_b200.prefix_attention import prefix_attention
    nh, nkv, hd, page = 6, 3, 128, 8
    c = make([2, 1, 5], [9, 30, 44], 77, page, nh, nkv, hd, kind, cache, seed=11)
    q, k, v, prefix_table, prefix, table, lens, start = c
    packed = torch.randn(q.shape[0], nh * hd + 192).to(TYPES[kind])
    packed[:, 64:64 + nh * hd] = q.flatten(1)
    packed = packed.cuda()
    both = torch.stack([k, v], 1).cuda()
    wide = torch.full((3, table.shape[1] + 20), -1, dtype=torch.int32)
    wide[:, :table.shape[1]] = table
    wide = wide.cuda()
    whole = torch.zeros(q.shape[0], nh * hd + 64, dtype=TYPES[kind], device="cuda")
    out = whole[:, :nh * hd].unflatten(1, (nh, hd))
    got = prefix_attention(packed[:, 64:64 + nh * hd].unflatten(1, (nh, hd)), both[:, 0], both[:, 1], prefix_table.cuda(),
                           prefix, wide, lens.cuda(), start.cuda(), page_size=page, max_new=100,
                           max_len=(table.shape[1] + 15) * page, scale=0.17, out=out)
    assert got.data_ptr() == whole.data_ptr()
    near(got, c, page, kind, cache, scale=0.17)
    assert not bool(whole[:, nh * hd:].any())


def test_same_inputs_same_bits():
    for counts, lens, nh, nkv in (([1] * 20, [50] * 20, 16, 4), ([100, 60], [100, 90], 8, 2)):
        c = make(counts, lens, 2000, 16, nh, nkv, 128, "bf16", "bf16", seed=1)
        first = call(c, 16)
        for _ in range(5):
            assert torch.equal(call(c, 16), first)


@pytest.mark.parametrize("fault", ["length", "tokens", "start", "block", "prefix block"])
def test_what_only_the_gpu_sees_is_skipped_and_reported(fault):
    from loopspec_b200 import _lib
    from loopspec_b200.status import DeviceStatus
    c = make([1, 2, 1], [5, 20, 9], 40, 16, 4, 2, 64, "bf16", "bf16", seed=2)
    good = call(c, 16)
    q, k, v, prefix_table, prefix, table, lens, start = c
    max_new = 2
    if fault == "length":
        lens[1] = 2000
    if fault == "tokens":
        max_new = 1
    if fault == "start":
        start[1:3] = torch.tensor([9, 1])
    if fault == "block":
        table[1, 0] = 1 << 20
    if fault == "prefix block":
        prefix_table[0] = -1
    status = DeviceStatus("cuda")
    out = call(c, 16, max_new=max_new, status=status)
    with pytest.raises(_lib.EngineError) as err:
        status.check()
    assert err.value.code == _lib.LS_EDEVICE
    if fault in ("length", "tokens", "block"):
        assert torch.equal(out[[0, 3]], good[[0, 3]])       # the other requests are whole
    if fault in ("length", "tokens"):
        assert not bool(out[1:3].any())


def test_a_bad_request_among_prompts_gets_zeros():
    from loopspec_b200 import _lib
    from loopspec_b200.status import DeviceStatus
    c = make([150, 200, 170], [150, 260, 170], 300, 16, 4, 4, 64, "bf16", "bf16", seed=2)
    good = call(c, 16)
    c[6][1] = 5000
    status = DeviceStatus("cuda")
    out = call(c, 16, status=status)
    with pytest.raises(_lib.EngineError):
        status.check()
    assert torch.equal(out[:150], good[:150]) and torch.equal(out[350:], good[350:])
    assert not bool(out[150:350].any())


def test_slots_past_32_bit_offsets():
    """The last slots of pools of more than 2^31 elements."""
    nkv, hd, page = 8, 128, 16
    n_slots = (2 ** 31 // (nkv * hd) // page + 3) * page
    pools = torch.zeros(2, n_slots, nkv, hd, dtype=torch.bfloat16, device="cuda")
    c = make([1, 2], [20, 9], 50, page, 8, 8, hd, "bf16", "bf16", seed=4)
    q, k, v, prefix_table, prefix, table, lens, start = c
    shift = n_slots // page - k.shape[0] // page
    pools[0, -k.shape[0]:] = k.cuda()
    pools[1, -k.shape[0]:] = v.cuda()
    from loopspec_b200.prefix_attention import prefix_attention
    got = prefix_attention(q.cuda(), pools[0], pools[1], (prefix_table + shift).cuda(), prefix,
                           torch.where(table >= 0, table + shift, table).cuda(), lens.cuda(), start.cuda(),
                           page_size=page, max_new=2)
    near(got, c, page, "bf16", "bf16")


def test_side_stream_and_graph():
    """Enqueued on a side stream behind its inputs, and captured: the replay sees new contents."""
    from loopspec_b200.prefix_attention import prefix_attention, workspace_bytes
    from loopspec_b200.status import DeviceStatus
    page = 16
    a = make([1, 2, 0], [5, 20, 9], 300, page, 8, 2, 64, "bf16", "bf16", seed=2)
    b = make([1, 2, 0], [5, 20, 9], 300, page, 8, 2, 64, "bf16", "bf16", seed=3)
    status = DeviceStatus("cuda")
    dev = [t.cuda() if torch.is_tensor(t) else t for t in a]
    new = [t.cuda() if torch.is_tensor(t) else t for t in b]
    out = torch.empty_like(dev[0])
    need = workspace_bytes(3, 8, 2, 64, n_requests=3, prefix_len=300, max_new=2, max_len=32)
    ws = torch.empty(need, dtype=torch.uint8, device="cuda")
    side = torch.cuda.Stream()
    torch.cuda.synchronize()

    def run(stream=None):
        prefix_attention(*dev[:3], dev[3], 300, dev[5], dev[6], dev[7], page_size=page, max_new=2, out=out,
                         workspace=ws, status=status, stream=stream)

    run(side.cuda_stream)
    side.synchronize()
    near(out, a, page, "bf16", "bf16")
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        run()
    for x, y in zip(dev, new):
        if torch.is_tensor(x):
            x.copy_(y)
    out.zero_()
    graph.replay()
    near(out, b, page, "bf16", "bf16")
    status.check()
