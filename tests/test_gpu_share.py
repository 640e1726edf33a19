"""PrefixBatch.share: what becomes of the request's blocks, and what it refuses."""

import pytest
import torch

pytestmark = pytest.mark.gpu

PAGE, N_BLOCKS = 4, 40


def batch_of(lens):
    from loopspec_b200.shared_prefix import PrefixBatch
    batch = PrefixBatch(1, 2, 1, 64, n_blocks=N_BLOCKS, page_size=PAGE, max_requests=len(lens), max_len=64, max_tokens=256,
                        max_positions=300)
    batch.begin(torch.tensor(lens, dtype=torch.int32, device="cuda"), sum(lens), max(lens))
    batch.check()
    return batch


def blocks(batch):
    """(the prefix's, the requests', the free) blocks."""
    own = [b for row, n in zip(batch.table.tolist(), batch.lens.tolist()) for b in row[:-(-n // PAGE)]]
    shared = [] if batch.prefix_table is None else batch.prefix_table.tolist()
    return shared, own, batch.free_blocks.tolist()[:int(batch.free_count)]


@pytest.mark.parametrize("held,length", [(33, 33), (33, 32), (33, 29), (33, 10), (33, 1), (64, 4)])
def test_every_block_is_the_prefixs_or_free(held, length):
    batch = batch_of([0, held, 0])
    first = batch.table[1, :-(-length // PAGE)].tolist()
    batch.share(1, length)
    batch.check()
    shared, own, free = blocks(batch)
    assert shared == first and own == [] and batch.lens.tolist() == [0, 0, 0] and batch.prefix_len == length
    assert sorted(shared + free) == list(range(N_BLOCKS))
    batch.begin(torch.tensor([5, 1, 64], dtype=torch.int32, device="cuda"), 70, 64)
    batch.check()
    assert sorted(sum(blocks(batch), [])) == list(range(N_BLOCKS))
    assert batch.map.positions[:2].tolist() == [length, length + 1]


@pytest.mark.parametrize("request_, length", [(1, 34), (1, 0), (1, -3), (0, 1), (3, 5), (-1, 5)])
def test_a_length_that_the_request_does_not_hold_is_refused(request_, length):
    batch = batch_of([0, 33, 0])
    before = blocks(batch)
    with pytest.raises(ValueError):
        batch.share(request_, length)
    assert blocks(batch) == before and batch.prefix_len == 0


def test_other_requests_with_positions_are_refused():
    """Their keys were rotated for positions that count from 0; behind the prefix they would count from its end."""
    batch = batch_of([7, 33, 0])
    before = blocks(batch)
    with pytest.raises(ValueError):
        batch.share(1, 33)
    assert blocks(batch) == before and batch.prefix_len == 0
    batch.begin(torch.tensor([-7, 0, 0], dtype=torch.int32, device="cuda"), 0, 0)
    batch.share(1, 33)
    with pytest.raises(ValueError):          # one prefix a batch
        batch.share(2, 1)
    batch.check()
