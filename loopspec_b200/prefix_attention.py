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
from .qk_norm import TYPE_CODES, check_pools
from .status import enqueue, on_stream

_pack = _lib.packer(_lib.PrefixAttentionArgs)
_i32 = torch.int32


def workspace_bytes(n_tokens, n_heads, n_kv_heads, head_dim, *, n_requests, prefix_len, max_new, max_len):
    """Bytes of device scratch of one call (a function of the sizes alone)."""
    need = int(_lib.lib().ls_prefix_attention_workspace_bytes(n_tokens, n_requests, n_heads, n_kv_heads, head_dim,
                                                              prefix_len, max_new, max_len))
    if need == 0:
        _lib.check(_lib.LS_EINVAL)
    return need


def prefix_attention(q, k_pool, v_pool, prefix_table, prefix_len, block_table, lens, token_start, *, page_size,
                     max_new, max_len=None, scale=None, out=None, workspace=None, status=None, stream=None):
    """out [T, n_heads, head_dim] of q's type.

    q            [T, n_heads, head_dim], of the pools' type or fp32; token rows may be strided
    k_pool, v_pool   [n_slots, n_kv_heads, head_dim], bf16 or f16, n_slots a multiple of page_size
    prefix_table int32 [>= ceil(prefix_len / page_size)] blocks of the prefix (None if prefix_len is 0)
    block_table  int32 [n_requests, width], rows may be strided
    lens         int32 [n_requests] own positions of each request, its new tokens included
    token_start  int32 [n_requests + 1]; tokens past the last entry are padding and get zeros
    max_new      bound on a request's new tokens; max_len on lens (default: the table's width)
    workspace    uint8 CUDA tensor of workspace_bytes(...) bytes, kept by the caller or made here;
                 calls that share one must be on one stream
    """
    n_slots, n_kv, hd, slot_stride = check_pools(k_pool, v_pool, "prefix attention")
    shape, row, dtype = q.shape, q.stride(), q.dtype
    n, nh, width = shape
    if not (width == hd and q.is_cuda and row[2] == 1 and row[1] == hd and dtype in TYPE_CODES):
        raise ValueError("prefix attention: q must be a CUDA tensor [T, n_heads, head_dim] with contiguous rows")
    n_req, blocks = block_table.shape
    columns = block_table.stride()
    if not (block_table.dtype is _i32 and block_table.is_cuda and (blocks <= 1 or columns[1] == 1)):
        raise ValueError("prefix attention: block_table must be an int32 CUDA tensor with contiguous rows")
    if not (lens.dtype is _i32 and token_start.dtype is _i32 and lens.is_cuda and token_start.is_cuda
            and lens.is_contiguous() and token_start.is_contiguous() and lens.numel() == n_req
            and token_start.numel() == n_req + 1):
        raise ValueError("prefix attention: lens [n_requests] and token_start [n_requests + 1] must be int32 "
                         "contiguous CUDA tensors")
    if max_len is None:
        max_len = blocks * page_size
    if not (page_size >= 1 and max_len <= blocks * page_size):
        raise ValueError("prefix attention: max_len exceeds the block table")
    if prefix_len and not (prefix_table is not None and prefix_table.dtype is _i32 and prefix_table.is_cuda
                           and prefix_table.is_contiguous() and prefix_table.numel() * page_size >= prefix_len > 0):
        raise ValueError("prefix attention: prefix_table must be an int32 contiguous CUDA tensor that covers prefix_len")
    if scale is None:
        scale = hd ** -0.5
    if out is None or workspace is None:
        with on_stream(q.device, stream):
            if out is None:
                out = torch.empty(n, nh, hd, dtype=dtype, device=q.device)
            if workspace is None:
                need = workspace_bytes(n, nh, n_kv, hd, n_requests=n_req, prefix_len=prefix_len, max_new=max_new,
                                       max_len=max_len)
                workspace = torch.empty(need, dtype=torch.uint8, device=q.device)
    to = out.stride()
    if not (out.shape == shape and out.dtype is dtype and out.is_cuda and to[2] == 1 and to[1] == hd):
        raise ValueError("prefix attention: out must be a CUDA tensor of q's shape and type with contiguous rows")
    before = (q.data_ptr(), row[0] if n > 1 else nh * hd, k_pool.data_ptr(), v_pool.data_ptr(), slot_stride,
              prefix_table.data_ptr() if prefix_len else 0, block_table.data_ptr(),
              columns[0] if n_req > 1 else blocks, lens.data_ptr(), token_start.data_ptr(),
              out.data_ptr(), to[0] if n > 1 else nh * hd, workspace.data_ptr(), workspace.numel())
    after = (TYPE_CODES[dtype], TYPE_CODES[k_pool.dtype], n, n_req, nh, n_kv, hd, prefix_len, max_new, max_len,
             page_size, n_slots, scale)
    enqueue(_lib.lib().ls_prefix_attention, _pack, before, after, q.device, status, stream)
    return out
