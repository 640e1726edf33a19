"""Block tables and slot maps (ls_build_slots) against a list-by-list restatement: whole numbers, all equal."""

import random

import pytest
import torch

from serving_reference import slots_reference

pytestmark = pytest.mark.gpu


def make(n, page, width, seed, low=-40, high=40, full=False):
    rng = random.Random(seed)
    cap = width * page
    lens = [rng.choice([0, 1, page - 1, page, page + 1, rng.randint(0, cap), cap]) for _ in range(n)]
    lens = [max(0, min(cap, x)) for x in lens]
    delta = [max(-x, min(cap - x, rng.choice([0, 1, -1, -x, cap - x if full else 1, rng.randint(low, high)])))
             for x in lens]
    used = sum(-(-x // page) for x in lens)
    spare = sum(max(0, -(-(x + d) // page) - -(-x // page)) for x, d in zip(lens, delta))
    n_blocks = used + spare + 5
    ids = list(range(n_blocks))
    rng.shuffle(ids)
    table, at = [], 0
    for x in lens:
        b = -(-x // page)
        table.append(ids[at:at + b] + [-7] * (width - b))
        at += b
    free = ids[at:]
    return lens, delta, table, free + [-9] * (n_blocks - len(free)), len(free), n_blocks


def call(lens, delta, table, stack, count, n_blocks, page, max_tokens, base=0, pad=0, inplace=False, status=None):
    from loopspec_b200.slots import SlotMap, build_slots
    dev = "cuda"
    t = lambda x: torch.tensor(x, dtype=torch.int32, device=dev)  # noqa: E731
    tab = torch.full((len(lens), len(table[0]) + pad), -3, dtype=torch.int32, device=dev)
    tab[:, :len(table[0])] = t(table)
    tab = tab[:, :len(table[0])]
    ln, cnt, st = t(lens), t([count]), t(stack)
    out = SlotMap(len(lens), max_tokens, dev, lens=ln if inplace else None, free_count=cnt if inplace else None)
    m = build_slots(ln, t(delta), tab, st, cnt, page_size=page, n_blocks=n_blocks, base=base, out=out, status=status)
    torch.cuda.synchronize()
    return m, tab, st


@pytest.mark.parametrize("n,page,width", [(1, 1, 3), (2, 16, 4), (33, 1, 90), (100, 64, 7), (513, 16, 9),
                                          (1500, 8, 6), (5000, 4, 3)])
@pytest.mark.parametrize("inplace", [False, True])
def test_slot_maps(n, page, width, inplace):
    lens, delta, table, stack, count, n_blocks = make(n, page, width, seed=n + page, full=page * width < 400)
    tokens, start, new, tab_ref, stack_ref, height = slots_reference(lens, delta, table, stack, count, page)
    room = len(tokens) + 37
    m, tab, st = call(lens, delta, table, stack, count, n_blocks, page, room, base=11, pad=n % 3, inplace=inplace)
    assert m.token_start.tolist() == start
    assert m.lens.tolist() == new and m.free_count.tolist() == [height]
    assert m.slots.tolist() == [s for s, _, _ in tokens] + [-1] * 37
    assert m.positions.tolist() == [p + 11 for _, p, _ in tokens] + [0] * 37
    assert m.requests.tolist() == [r for _, _, r in tokens] + [-1] * 37
    assert tab.tolist() == tab_ref
    assert st.tolist() == stack_ref


def test_long_prompts_spread_over_the_cluster():
    page, width, n = 32, 300, 9
    lens = [0, 5, 32, 31, 0, 100, 64, 7, 0]
    delta = [9000, 0, -32, 4097, 1, -3, 8000, 2500, 0]
    used = [-(-x // page) for x in lens]
    ids = list(range(2000))
    random.Random(4).shuffle(ids)
    table, at = [], 0
    for b in used:
        table.append(ids[at:at + b] + [-1] * (width - b))
        at += b
    free = ids[at:]
    stack = free + [-1] * (2000 - len(free))
    tokens, start, new, tab_ref, stack_ref, height = slots_reference(lens, delta, table, stack, len(free), page)
    m, tab, st = call(lens, delta, table, stack, len(free), 2000, page, len(tokens))
    assert m.token_start.tolist() == start and m.lens.tolist() == new and m.free_count.tolist() == [height]
    assert m.slots.tolist() == [s for s, _, _ in tokens]
    assert m.requests.tolist() == [r for _, _, r in tokens]
    assert tab.tolist() == tab_ref and st.tolist() == stack_ref


def test_every_position_of_every_request_has_its_own_slot():
    """Many steps in place: growth, rollback and release never share a slot."""
    from loopspec_b200.slots import SlotMap, build_slots
    from loopspec_b200.status import DeviceStatus
    rng = random.Random(1)
    n, page, width, n_blocks = 40, 4, 16, 400
    dev = "cuda"
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=dev)  # noqa: E731
    lens, count = i32([0] * n), i32([n_blocks])
    table = torch.full((n, width), -1, dtype=torch.int32, device=dev)
    stack = torch.arange(n_blocks, dtype=torch.int32, device=dev)
    status = DeviceStatus(dev)
    out = SlotMap(n, n * width * page, dev, lens=lens, free_count=count)
    held = [0] * n
    for _ in range(60):
        delta = [rng.choice([1, 1, 5, -held[i], -min(held[i], 3), 0]) for i in range(n)]
        delta = [min(d, width * page - held[i]) for i, d in enumerate(delta)]
        build_slots(lens, i32(delta), table, stack, count, page_size=page, n_blocks=n_blocks, out=out, status=status)
        held = [h + d for h, d in zip(held, delta)]
        used = [b for i, r in enumerate(table.tolist()) for b in r[:-(-held[i] // page)]]
        left = stack.tolist()[:int(count)]
        assert lens.tolist() == held
        assert sorted(used + left) == list(range(n_blocks))
    status.check()


@pytest.mark.parametrize("fault", ["blocks", "tokens", "negative", "past the table", "count"])
def test_nothing_changes_when_the_step_cannot_be_done(fault):
    from loopspec_b200 import _lib
    from loopspec_b200.status import DeviceStatus
    page, width = 4, 5
    lens, delta, room, count = [3, 8, 0, 5], [6, 0, 3, -2], 64, 3
    if fault == "blocks":
        count = 2              # growth takes 2 + 1, rollback gives back 1: 3 fit, one fewer does not
        delta[3] = 0
    if fault == "tokens":
        room = 8
    if fault == "negative":
        delta[2] = -1
    if fault == "past the table":
        delta[1] = page * width - 8 + 1
    if fault == "count":
        count = -1
    table = [[0, -1, -1, -1, -1], [1, 2, -1, -1, -1], [-1] * 5, [3, 4, -1, -1, -1]]
    stack = [5, 6, 7, 8, 9, 10, 11, 12]
    status = DeviceStatus("cuda")
    m, tab, st = call(lens, delta, table, stack, count, 13, page, room, status=status)
    with pytest.raises(_lib.EngineError) as err:
        status.check()
    assert err.value.code == (_lib.LS_ECAPACITY if fault in ("blocks", "tokens") else _lib.LS_EDEVICE)
    status.check()             # cleared
    assert m.lens.tolist() == lens and m.free_count.tolist() == [count]
    assert tab.tolist() == table and st.tolist() == stack
    assert m.token_start.tolist() == [0] * 5
    assert set(m.slots.tolist()) == {-1} and set(m.requests.tolist()) == {-1} and set(m.positions.tolist()) == {0}
    with pytest.raises(_lib.EngineError):      # without a status word the call itself raises
        call(lens, delta, table, stack, count, 13, page, room)


def test_a_bad_block_is_reported_and_gets_no_slot():
    from loopspec_b200 import _lib
    from loopspec_b200.status import DeviceStatus
    status = DeviceStatus("cuda")
    m, _, _ = call([1, 1], [1, 1], [[99], [1]], [2], 1, 3, 4, 2, status=status)
    assert m.slots.tolist() == [-1, 5]
    with pytest.raises(_lib.EngineError):
        status.check()
