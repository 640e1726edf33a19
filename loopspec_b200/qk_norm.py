"""Per-head norm of q and k, position rotation and K/V cache write in one pass
(ls_qk_norm_rope)."""

from __future__ import annotations

import torch

from . import _lib
from .status import enqueue, on_stream

_pack = _lib.packer(_lib.QkNormArgs)
_i32, _f32 = torch.int32, torch.float32
TYPE_CODES = {torch.bfloat16: 0, torch.float16: 1, torch.float32: 2}    # LS_BF16, LS_F16, LS_F32


def check_pools(k_pool, v_pool, what):
    """(n_slots, n_kv_heads, head_dim, slot stride) of a pair of K/V pools."""
    shape, stride = k_pool.shape, k_pool.stride()
    if not (len(shape) == 3 and v_pool.shape == shape and v_pool.dtype is k_pool.dtype and v_pool.stride() == stride
            and stride[2] == 1 and stride[1] == shape[2] and k_pool.is_cuda and v_pool.is_cuda
            and k_pool.dtype in TYPE_CODES):
        raise ValueError(f"{what}: k_pool and v_pool must be CUDA tensors [n_slots, n_kv_heads, head_dim] of one type "
                         "and layout, with contiguous slots")
    n_slots, n_kv, hd = shape
    return n_slots, n_kv, hd, stride[0] if n_slots > 1 else n_kv * hd


def rope_table(max_positions, rot, theta=10000.0, device="cuda"):
    """fp32 [max_positions, 2, rot / 2]: cos and sin of position * theta^(-2i/rot),
    computed in 64 bits so that long positions keep their angle."""
    inv = theta ** (-torch.arange(0, rot, 2, dtype=torch.float64, device=device) / rot)
    angle = torch.arange(max_positions, dtype=torch.float64, device=device)[:, None] * inv
    return torch.stack([angle.cos(), angle.sin()], 1).to(torch.float32)


def qk_norm_rope(qkv, q_weight, k_weight, rope, positions, k_pool, v_pool, slots=None, *, eps=1e-6,
                 interleaved=False, out=None, status=None, stream=None):
    """Norm and rotate q and k of each token, write k and v to their cache slots, return q.

    qkv        [T, (n_heads + 2 n_kv_heads) * head_dim], bf16 / f16 / fp32, rows may be strided
    q_weight, k_weight   [head_dim], one type of bf16 / f16 / fp32
    rope       fp32 [max_positions, 2, rot / 2] (see rope_table); rot <= head_dim is rotated
    positions  int32 [T]; slots int32 [T], -1 for padding, or None for row t of the pools
    k_pool, v_pool       [n_slots, n_kv_heads, head_dim], bf16 or f16
    out        q's destination [T, n_heads, head_dim] of qkv's type (may be the q part of qkv)
    """
    n_slots, n_kv, hd, slot_stride = check_pools(k_pool, v_pool, "qk norm")
    n, width = qkv.shape
    nh = width // hd - 2 * n_kv
    row, dtype = qkv.stride(), qkv.dtype
    if not (width % hd == 0 and nh > 0 and qkv.is_cuda and row[1] == 1 and dtype in TYPE_CODES):
        raise ValueError("qk norm: qkv must be a CUDA tensor whose contiguous rows hold q, k and v heads")
    if not (q_weight.numel() == hd == k_weight.numel() and q_weight.dtype is k_weight.dtype
            and q_weight.dtype in TYPE_CODES and q_weight.is_cuda and k_weight.is_cuda
            and q_weight.is_contiguous() and k_weight.is_contiguous()):
        raise ValueError("qk norm: q_weight and k_weight must be contiguous CUDA tensors [head_dim] of one type")
    limit, two, half = rope.shape
    if not (two == 2 and rope.dtype is _f32 and rope.is_cuda and rope.is_contiguous()):
        raise ValueError("qk norm: rope must be a contiguous fp32 CUDA tensor [max_positions, 2, rot / 2]")
    for t in (positions, slots):
        if t is not None and not (t.dtype is _i32 and t.is_cuda and t.is_contiguous() and t.numel() == n):
            raise ValueError("qk norm: positions and slots must be int32 contiguous CUDA tensors, one entry a token")
    if slots is None and n > n_slots:
        raise ValueError("qk norm: without slots the pools need a row for each token")
    if out is None:
        with on_stream(qkv.device, stream):
            out = torch.empty(n, nh, hd, dtype=dtype, device=qkv.device)
    to = out.stride()
    if not (out.shape == (n, nh, hd) and out.dtype is dtype and out.is_cuda and to[2] == 1 and to[1] == hd):
        raise ValueError("qk norm: out must be a CUDA tensor [T, n_heads, head_dim] of qkv's type with contiguous rows")
    before = (qkv.data_ptr(), row[0] if n > 1 else width, q_weight.data_ptr(), k_weight.data_ptr(), rope.data_ptr(),
              positions.data_ptr(), 0 if slots is None else slots.data_ptr(), k_pool.data_ptr(),
              v_pool.data_ptr(), slot_stride, out.data_ptr(), to[0] if n > 1 else nh * hd)
    after = (TYPE_CODES[dtype], TYPE_CODES[q_weight.dtype], TYPE_CODES[k_pool.dtype], n, nh, n_kv, hd, limit, 2 * half,
             int(interleaved), n_slots, eps)
    enqueue(_lib.lib().ls_qk_norm_rope, _pack, before, after, qkv.device, status, stream)
    return out
