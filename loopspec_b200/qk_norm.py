"""Per-head norm of q and k, position rotation and K/V cache write in one pass
(ls_qk_norm_rope)."""

from __future__ import annotations

import torch

from . import _lib
from .status import enqueue, on_stream

_pack = _lib.packer(_lib.QkNormArgs)
TYPE_CODES = {torch.bfloat16: _lib.BF16, torch.float16: _lib.F16, torch.float32: _lib.F32}
FLOATS = (_lib.BF16, _lib.F16, _lib.F32)


def check_pools(k_pool, v_pool, what):
    """(k pointer, v pointer, GPU, type code, n_slots, n_kv_heads, head_dim, slot stride) of a pair of K/V pools."""
    facts, _ = _lib.tensor_facts()
    k, v = facts(k_pool), facts(v_pool)
    if not (k and v and len(k) == 9 and k[1:] == v[1:] and k[2] in FLOATS and k[8] == 1 and k[7] == k[5] > 0):
        raise ValueError(f"{what}: k_pool and v_pool must be CUDA tensors [n_slots, n_kv_heads, head_dim] of one type "
                         "and layout, with contiguous slots")
    k_ptr, gpu, code, n_slots, n_kv, hd, stride = k[:7]
    return k_ptr, v[0], gpu, code, n_slots, n_kv, hd, stride if n_slots > 1 else n_kv * hd


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
    facts, pointers = _lib.tensor_facts()
    k_ptr, v_ptr, gpu, cache, n_slots, n_kv, hd, slot_stride = check_pools(k_pool, v_pool, "qk norm")
    x = facts(qkv)
    if not (x and len(x) == 7 and x[1] == gpu and x[2] in FLOATS and x[6] == 1 and x[4] % hd == 0
            and x[4] // hd > 2 * n_kv):
        raise ValueError("qk norm: qkv must be a CUDA tensor whose contiguous rows hold q, k and v heads")
    x_ptr, _, code, n, width, row, _ = x
    nh = width // hd - 2 * n_kv
    weight_code = TYPE_CODES.get(q_weight.dtype, -1)
    weights = pointers(gpu, weight_code, q_weight, hd, k_weight, hd) if weight_code >= 0 else None
    if weights is None:
        raise ValueError("qk norm: q_weight and k_weight must be contiguous CUDA tensors [head_dim] of one type")
    limit, two, half = rope.shape
    table = pointers(gpu, _lib.F32, rope, -1)
    if table is None or two != 2:
        raise ValueError("qk norm: rope must be a contiguous fp32 CUDA tensor [max_positions, 2, rot / 2]")
    where = pointers(gpu, _lib.I32, positions, n, slots, n)
    if where is None:
        raise ValueError("qk norm: positions and slots must be int32 contiguous CUDA tensors, one entry a token")
    if slots is None and n > n_slots:
        raise ValueError("qk norm: without slots the pools need a row for each token")
    if out is None:
        with on_stream(qkv.device, stream):
            out = torch.empty(n, nh, hd, dtype=qkv.dtype, device=qkv.device)
    to = facts(out)
    if not (to and to[1:6] == (gpu, code, n, nh, hd) and to[8] == 1 and to[7] == hd):
        raise ValueError("qk norm: out must be a CUDA tensor [T, n_heads, head_dim] of qkv's type with contiguous rows")
    before = (x_ptr, row if n > 1 else width, *weights, *table, *where, k_ptr, v_ptr, slot_stride, to[0],
              to[6] if n > 1 else nh * hd)
    after = (code, weight_code, cache, n, nh, n_kv, hd, limit, 2 * half, int(interleaved), n_slots, eps)
    enqueue(_lib.lib().ls_qk_norm_rope, _pack, before, after, gpu, status, stream)
    return out
