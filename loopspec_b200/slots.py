"""Block tables and slot maps from request lengths, on the GPU (ls_build_slots).

A request's tokens live in blocks of `page_size` slots; row i of `block_table`
lists its blocks. `build_slots` applies one step's changes to every request:
`delta[i]` > 0 appends tokens (new blocks are popped from the free stack),
`delta[i]` < 0 cuts the request back (blocks no longer needed are pushed), so
admission, decoding, rollback of rejected drafts and release are one call and
the host never learns a length.
"""

from __future__ import annotations

import torch

from . import _lib
from .status import enqueue

_pack = _lib.packer(_lib.SlotsArgs)


class SlotMap:
    """The outputs of `build_slots`, kept between calls.

    slots, positions, requests  int32 [max_tokens]: of new token k; -1, 0, -1 past the last
    token_start                 int32 [n_requests + 1]: first new token of each request
    lens, free_count            int32 [n_requests], [1]: updated; pass the call's own
                                tensors here to update them in place
    """

    def __init__(self, n_requests, max_tokens, device="cuda", lens=None, free_count=None):
        n, t = n_requests, max_tokens
        whole = torch.empty(3 * t + 2 * n + 2, dtype=torch.int32, device=device)
        self.slots, self.positions, self.requests = whole[:t], whole[t:2 * t], whole[2 * t:3 * t]
        self.token_start = whole[3 * t:3 * t + n + 1]
        self.lens = whole[3 * t + n + 1:-1] if lens is None else lens
        self.free_count = whole[-1:] if free_count is None else free_count


def build_slots(lens, delta, block_table, free_blocks, free_count, *, page_size, n_blocks, out, base=0,
                status=None, stream=None):
    """Apply one step's length changes; returns `out`, a `SlotMap`.

    lens, delta    int32 [n_requests]
    block_table    int32 [n_requests, width] (rows may be strided), updated
    free_blocks    int32 [capacity], the stack; free_count int32 [1], its height
    base           position of a request's first own token (the shared prefix's length)
    All or nothing: on a bad length, too few free blocks or more new tokens
    than out.slots holds, nothing changes and the status says why.
    """
    facts, pointers = _lib.tensor_facts()
    table = facts(block_table)
    if not (table and len(table) == 7 and table[2] == _lib.I32 and table[6] == 1):
        raise ValueError("slot maps: block_table must be an int32 CUDA tensor [n_requests, width] with contiguous rows")
    table_ptr, gpu, _, n, width, row, _ = table
    most = out.slots.numel()
    ptrs = pointers(gpu, _lib.I32, lens, n, delta, n, free_blocks, -1, free_count, 1, out.slots, most, out.positions,
                    most, out.requests, most, out.token_start, n + 1, out.lens, n, out.free_count, 1)
    if ptrs is None:
        raise ValueError("slot maps: lens, delta, free_blocks, free_count and out must be int32 contiguous CUDA tensors "
                         "that describe the block table's requests")
    before = (*ptrs[:2], table_ptr, row if n > 1 else width, *ptrs[2:])
    after = (n, width, free_blocks.numel(), n_blocks, page_size, base, most)
    enqueue(_lib.lib().ls_build_slots, _pack, before, after, gpu, status, stream)
    return out
