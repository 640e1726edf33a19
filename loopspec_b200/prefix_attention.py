"""Attention of a batch whose requests share a long prefix (ls_prefix_attention).

Every token attends to the whole shared prefix and, causally, to its request's
own positions. The prefix's K/V are read once for the batch; the requests' own
positions are read through their block tables, as `slots.build_slots` fills
them. With page_size 1 a block table is a timeline's row of slots, as in
`attention.decode_attention`.
"""

from __future__ import annotations

import torch

from . import _lib
from .qk_norm import FLOATS, check_pools
from .status import enqueue, on_stream

_pack = _lib.packer(_lib.PrefixAttentionArgs)


def workspace_bytes(n_tokens, n_heads, n_kv_heads, head_dim, *, n_requests, prefix_len, max_new, max_len):
    """Bytes of device scratch of one call on the current device: a function of the sizes and of its number of SMs."""
    need = int(_lib.lib().ls_prefix_attention_workspace_bytes(n_tokens, n_requests, n_heads, n_kv_heads, head_dim,
                                                              prefix_len, max_new, max_len))
    if need == 0:
        _lib.check(_lib.LS_EINVAL)
    return need


def prefix_attention(q, k_pool, v_pool, prefix_table, prefix_len, block_table, lens, token_start, *, page_size,
                     max_new, max_len=None, scale=None, out=None, workspace=None, status=None, stream=None):
    """out [T, n_heads, head_dim] of q's type.

    With 16-bit q the softmax weights are rounded to its type for the second product (errors against 64 bits, relative
    to the result: bf16 0.0022, f16 0.00027); with fp32 q they are not, and errors are below 2e-6. Infinities and NaN
    that a token sees give what the formula gives.

    q            [T, n_heads, head_dim], of the pools' type or fp32; token rows may be strided
    k_pool, v_pool   [n_slots, n_kv_heads, head_dim], bf16 or f16, n_slots a multiple of page_size
    prefix_table int32 [>= ceil(prefix_len / page_size)] blocks of the prefix (None if prefix_len is 0)
    block_table  int32 [n_requests, width], rows may be strided
    lens         int32 [n_requests] own positions of each request, its new tokens included
    out          not overlapping q
    token_start  int32 [n_requests + 1]; tokens past the last entry are padding and get zeros
    max_new      bound on a request's new tokens; max_len on lens (default: the table's width)
    workspace    uint8 CUDA tensor of workspace_bytes(...) bytes, kept by the caller or made here;
                 calls that share one must be on one stream
    """
    facts, pointers = _lib.tensor_facts()
    k_ptr, v_ptr, gpu, cache, n_slots, n_kv, hd, slot_stride = check_pools(k_pool, v_pool, "prefix attention")
    x = facts(q)
    if not (x and len(x) == 9 and x[1] == gpu and x[2] in FLOATS and x[5] == hd and x[8] == 1 and x[7] == hd):
        raise ValueError("prefix attention: q must be a CUDA tensor [T, n_heads, head_dim] with contiguous rows")
    x_ptr, _, code, n, nh, _, row = x[:7]
    table = facts(block_table)
    if not (table and len(table) == 7 and table[1] == gpu and table[2] == _lib.I32
            and (table[4] <= 1 or table[6] == 1)):
        raise ValueError("prefix attention: block_table must be an int32 CUDA tensor with contiguous rows")
    table_ptr, _, _, n_req, blocks, columns, _ = table
    ptrs = pointers(gpu, _lib.I32, lens, n_req, token_start, n_req + 1)
    if ptrs is None:
        raise ValueError("prefix attention: lens [n_requests] and token_start [n_requests + 1] must be int32 "
                         "contiguous CUDA tensors")
    if max_len is None:
        max_len = blocks * page_size
    if not (page_size >= 1 and max_len <= blocks * page_size):
        raise ValueError("prefix attention: max_len exceeds the block table")
    shared = (0,)
    if prefix_len:
        shared = pointers(gpu, _lib.I32, prefix_table, -1)
        if not (shared and prefix_table is not None and prefix_table.numel() * page_size >= prefix_len > 0):
            raise ValueError("prefix attention: prefix_table must be an int32 contiguous CUDA tensor that covers "
                             "prefix_len")
    if scale is None:
        scale = hd ** -0.5
    if out is None or workspace is None:
        with torch.cuda.device(gpu), on_stream(q.device, stream):
            if out is None:
                out = torch.empty(n, nh, hd, dtype=q.dtype, device=q.device)
            if workspace is None:
                need = workspace_bytes(n, nh, n_kv, hd, n_requests=n_req, prefix_len=prefix_len, max_new=max_new,
                                       max_len=max_len)
                workspace = torch.empty(need, dtype=torch.uint8, device=q.device)
    to = facts(out)
    if not (to and to[1:6] == x[1:6] and to[8] == 1 and to[7] == hd):
        raise ValueError("prefix attention: out must be a CUDA tensor of q's shape and type with contiguous rows")
    scratch = pointers(gpu, _lib.BYTE, workspace, -1)
    if scratch is None:
        raise ValueError("prefix attention: workspace must be a contiguous uint8 CUDA tensor")
    before = (x_ptr, row if n > 1 else nh * hd, k_ptr, v_ptr, slot_stride, *shared, table_ptr,
              columns if n_req > 1 else blocks, *ptrs, to[0], to[6] if n > 1 else nh * hd, *scratch,
              workspace.numel())
    after = (code, cache, n, n_req, nh, n_kv, hd, prefix_len, max_new, max_len, page_size, n_slots, scale)
    enqueue(_lib.lib().ls_prefix_attention, _pack, before, after, gpu, status, stream)
    return out
