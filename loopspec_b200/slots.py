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
_i32 = torch.int32


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
    for t in (lens, delta, free_blocks, free_count, out.lens, out.free_count):
        if not (t.dtype is _i32 and t.is_cuda and t.is_contiguous()):
            raise ValueError("slot maps: int32 contiguous CUDA tensors expected")
    n, width = block_table.shape
    row = block_table.stride()
    if not (block_table.dtype is _i32 and block_table.is_cuda and row[1] == 1):
        raise ValueError("slot maps: block_table must be an int32 CUDA tensor with contiguous rows")
    if not (lens.numel() == n == delta.numel() == out.lens.numel() and out.token_start.numel() == n + 1
            and free_count.numel() == 1 == out.free_count.numel()):
        raise ValueError("slot maps: lens, delta, block_table and out must describe the same requests")
    before = (lens.data_ptr(), delta.data_ptr(), block_table.data_ptr(), row[0] if n > 1 else width,
              free_blocks.data_ptr(), free_count.data_ptr(), out.slots.data_ptr(), out.positions.data_ptr(),
              out.requests.data_ptr(), out.token_start.data_ptr(), out.lens.data_ptr(), out.free_count.data_ptr())
    after = (n, width, free_blocks.numel(), n_blocks, page_size, base, out.slots.numel())
    enqueue(_lib.lib().ls_build_slots, _pack, before, after, lens.device, status, stream)
    return out
