"""Per-head norm, rotation and K/V write (ls_qk_norm_rope) against a float64 restatement.

Tolerance, derived: the kernel computes in fp32 and rounds once. The norm's
sum of hd <= 128 squares adds at most 8 + log2 roundings of 2^-24 on a lane's
16 products and the shuffle tree (< 24 in all, halved by the square root),
rsqrtf 2^-22, three products, and the rotation two products and a sum of
values below sqrt(2) times the pair: under 32 * 2^-24 of the pair's length.
Output types add half a unit in the last place: 2^-8 (bf16) or 2^-11 (f16) of
the value, and f16's smallest step 2^-24.
"""

import pytest
import torch

from serving_reference import qk_norm_reference

pytestmark = pytest.mark.gpu

TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
UNIT = {"bf16": 2.0 ** -8, "f16": 2.0 ** -11, "f32": 2.0 ** -24}


def near(out, ref, kind, big):
    err = (out.double().cpu() - ref).abs()
    bound = 32 * 2.0 ** -24 * big + UNIT[kind] * (ref.abs() + 32 * 2.0 ** -24 * big) + 2.0 ** -25
    assert bool((err <= bound).all()), float((err / bound).max())


def inputs(T, nh, nkv, hd, kind, cache, rot, seed=0, limit=300, extra=0):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(T, (nh + 2 * nkv) * hd + extra, generator=g) * 3
    qw, kw = (1 + 0.3 * torch.randn(2, hd, generator=g)).to(torch.bfloat16)
    rope = torch.randn(limit, 2, rot // 2, generator=g)
    rope = rope / rope.norm(dim=1, keepdim=True)
    pos = torch.randint(0, limit, (T,), generator=g, dtype=torch.int32)
    slots = torch.randperm(T + 9, generator=g)[:T].to(torch.int32)
    return x.to(TYPES[kind]), qw, kw, rope, pos, slots


@pytest.mark.parametrize("T,nh,nkv,hd", [(1, 4, 4, 64), (1, 2, 2, 128), (7, 4, 1, 64), (67, 32, 8, 64), (5, 16, 16, 128),
                                         (33, 28, 4, 128), (1000, 9, 3, 128), (3, 1, 1, 64), (300, 71, 71, 64)])
@pytest.mark.parametrize("kind,cache", [("bf16", "bf16"), ("f16", "f16"), ("f32", "bf16"), ("f32", "f16")])
@pytest.mark.parametrize("interleaved", [False, True])
def test_matches_the_formula(T, nh, nkv, hd, kind, cache, interleaved):
    from loopspec_b200.qk_norm import qk_norm_rope
    rot = hd if (T + nh) % 2 else hd // 2 if (T + nh) % 4 else 16
    x, qw, kw, rope, pos, slots = inputs(T, nh, nkv, hd, kind, cache, rot, seed=T + nh)
    q_ref, k_ref, v_ref = qk_norm_reference(x, qw, kw, rope, pos, nh, nkv, hd, 1e-5, interleaved)
    pools = torch.full((2, T + 9, nkv, hd), 7.0, dtype=TYPES[cache], device="cuda")
    q = qk_norm_rope(x.cuda(), qw.cuda(), kw.cuda(), rope.cuda(), pos.cuda(), pools[0], pools[1], slots.cuda(), eps=1e-5,
                     interleaved=interleaved)
    big = max(float(q_ref.abs().max()), float(k_ref.abs().max())) * 1.5
    near(q, q_ref, kind, big)
    at = slots.long()
    near(pools[0].cpu()[at], k_ref, cache, big)
    assert torch.equal(pools[1].cpu()[at], v_ref.to(TYPES[cache]) if kind != "f32" else v_ref.float().to(TYPES[cache]))
    rest = torch.ones(T + 9, dtype=torch.bool)
    rest[at] = False
    assert bool((pools[:, rest.cuda()] == 7).all())      # no other slot is touched


def test_strided_rows_in_place_and_weight_types():
    """qkv inside wider rows, q written over its own input, pools inside one interleaved allocation."""
    from loopspec_b200.qk_norm import qk_norm_rope
    T, nh, nkv, hd = 19, 6, 2, 128
    x, qw, kw, rope, pos, slots = inputs(T, nh, nkv, hd, "bf16", "bf16", hd, seed=2, extra=64)
    qkv = x[:, :(nh + 2 * nkv) * hd]
    q_ref, k_ref, v_ref = qk_norm_reference(qkv.contiguous(), qw, kw, rope, pos, nh, nkv, hd, 1e-6, False)
    big = max(float(q_ref.abs().max()), float(k_ref.abs().max())) * 1.5
    for weight in (torch.bfloat16, torch.float32):
        wide = x.cuda()
        both = torch.zeros(T + 9, 2, nkv, hd, dtype=torch.bfloat16, device="cuda")
        view = wide[:, :(nh + 2 * nkv) * hd]
        out = view[:, :nh * hd].unflatten(1, (nh, hd))
        q = qk_norm_rope(view, qw.cuda().to(weight), kw.cuda().to(weight), rope.cuda(), pos.cuda(), both[:, 0], both[:, 1],
                         slots.cuda(), out=out)
        assert q.data_ptr() == wide.data_ptr()
        near(q, q_ref, "bf16", big)
        near(both[:, 0].cpu()[slots.long()], k_ref, "bf16", big)
        assert torch.equal(both[:, 1].cpu()[slots.long()].double(), v_ref)
        assert torch.equal(wide[:, nh * hd:].cpu(), x[:, nh * hd:])


def test_padding_no_slots_and_empty():
    from loopspec_b200.qk_norm import qk_norm_rope
    from loopspec_b200.status import DeviceStatus
    T, nh, nkv, hd = 6, 4, 2, 64
    x, qw, kw, rope, pos, _ = inputs(T, nh, nkv, hd, "f16", "f16", hd)
    q_ref, k_ref, _ = qk_norm_reference(x, qw, kw, rope, pos, nh, nkv, hd, 1e-6, False)
    status = DeviceStatus("cuda")
    args = [t.cuda() for t in (x, qw, kw, rope, pos)]
    pools = torch.full((2, T, nkv, hd), 7.0, dtype=torch.float16, device="cuda")
    qk_norm_rope(*args, pools[0], pools[1], status=status)          # row t without slots
    near(pools[0], k_ref, "f16", 20.0)
    pools.fill_(7)
    slots = torch.tensor([-1, 3, -1, 0, -1, -1], dtype=torch.int32, device="cuda")
    q = qk_norm_rope(*args, pools[0], pools[1], slots, status=status)
    near(q, q_ref, "f16", 20.0)
    near(pools[0][[3, 0]], k_ref[[1, 3]], "f16", 20.0)
    assert bool((pools[:, [1, 2, 4, 5]] == 7).all())
    empty = qk_norm_rope(args[0][:0], *args[1:4], args[4][:0], pools[0], pools[1], slots[:0], status=status)
    assert empty.shape == (0, nh, hd)
    status.check()


def test_bad_positions_and_slots_are_reported():
    from loopspec_b200 import _lib
    from loopspec_b200.qk_norm import qk_norm_rope
    from loopspec_b200.status import DeviceStatus
    T, nh, nkv, hd = 3, 2, 1, 64
    x, qw, kw, rope, pos, _ = inputs(T, nh, nkv, hd, "bf16", "bf16", hd, limit=10)
    status = DeviceStatus("cuda")
    for bad_pos, bad_slot in ((10, 1), (-1, 1), (2, 5), (2, -2)):
        pools = torch.full((2, 5, nkv, hd), 7.0, dtype=torch.bfloat16, device="cuda")
        p = torch.tensor([1, bad_pos, 3], dtype=torch.int32, device="cuda")
        s = torch.tensor([0, bad_slot, 4], dtype=torch.int32, device="cuda")
        qk_norm_rope(x.cuda(), qw.cuda(), kw.cuda(), rope.cuda(), p, pools[0], pools[1], s, status=status)
        with pytest.raises(_lib.EngineError):
            status.check()
        assert bool((pools[:, 1:4] == 7).all()) and not bool((pools[0, 0] == 7).any())


def test_values_that_are_not_finite_stay_in_their_head():
    from loopspec_b200.qk_norm import qk_norm_rope
    T, nh, nkv, hd = 2, 4, 2, 64
    x, qw, kw, rope, pos, slots = inputs(T, nh, nkv, hd, "f32", "bf16", 32)
    y = x.clone()
    y[0, 70] = float("inf")                     # head 1 of token 0
    pools = torch.zeros(4, T + 9, nkv, hd, dtype=torch.bfloat16, device="cuda")
    a = [t.cuda() for t in (qw, kw, rope, pos)]
    q1 = qk_norm_rope(x.cuda(), *a, pools[0], pools[1], slots.cuda())
    q2 = qk_norm_rope(y.cuda(), *a, pools[2], pools[3], slots.cuda())
    keep = torch.ones(T, nh, dtype=torch.bool)
    keep[0, 1] = False
    assert torch.equal(q1[keep.cuda()], q2[keep.cuda()])
    assert torch.equal(pools[0], pools[2]) and torch.equal(pools[1], pools[3])


def test_runs_on_the_given_stream():
    """On a side stream, ordered after work of that stream alone."""
    from loopspec_b200.qk_norm import qk_norm_rope
    T, nh, nkv, hd = 40, 8, 2, 128
    x, qw, kw, rope, pos, slots = inputs(T, nh, nkv, hd, "bf16", "bf16", hd)
    a = [t.cuda() for t in (qw, kw, rope, pos)]
    pools = torch.zeros(4, T + 9, nkv, hd, dtype=torch.bfloat16, device="cuda")
    want = qk_norm_rope(x.cuda(), *a, pools[0], pools[1], slots.cuda())
    side = torch.cuda.Stream()
    src = torch.zeros_like(x, device="cuda")
    xd, sd = x.cuda(), slots.cuda()
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        torch.cuda._sleep(20_000_000)
        src.copy_(xd)
    q = qk_norm_rope(src, *a, pools[2], pools[3], sd, stream=side.cuda_stream)
    side.synchronize()
    assert torch.equal(q, want) and torch.equal(pools[0], pools[2]) and torch.equal(pools[1], pools[3])
