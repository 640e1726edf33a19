"""Per-head norm of q and k, position rotation and K/V cache write in one pass
(ls_qk_norm_rope)."""

from __future__ import annotations

from . import _lib
from .status import enqueue, require

_pack = _lib.packer(_lib.QkNormArgs)


def _types():
    import torch
    return {torch.bfloat16: 0, torch.float16: 1, torch.float32: 2}


_TYPES = None


def type_code(dtype, what):
    """LS_BF16 / LS_F16 / LS_F32 of a torch dtype."""
    global _TYPES
    if _TYPES is None:
        _TYPES = _types()
    code = _TYPES.get(dtype)
    require(code is not None, f"{what}: bf16, f16 or fp32 expected, got {dtype}")
    return code


def check_pools(k_pool, v_pool, what):
    """(n_slots, n_kv_heads, head_dim, slot stride) of a pair of K/V pools."""
    n_slots, n_kv, hd = k_pool.shape
    stride = k_pool.stride()
    require(v_pool.shape == k_pool.shape and v_pool.dtype is k_pool.dtype and v_pool.stride() == stride
            and stride[2] == 1 and stride[1] == hd and k_pool.is_cuda and v_pool.is_cuda,
            f"{what}: k_pool and v_pool must be CUDA tensors [n_slots, n_kv_heads, head_dim] of one type and "
            "layout, with contiguous slots")
    return n_slots, n_kv, hd, stride[0] if n_slots > 1 else n_kv * hd


def rope_table(max_positions, rot, theta=10000.0, device="cuda"):
    """fp32 [max_positions, 2, rot / 2]: cos and sin of position * theta^(-2i/rot),
    computed in 64 bits so that long positions keep their angle."""
    import torch
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
    import torch
    n_slots, n_kv, hd, slot_stride = check_pools(k_pool, v_pool, "qk norm")
    n, width = qkv.shape
    require(width % hd == 0 and width // hd > 2 * n_kv, "qk norm: qkv rows must hold q, k and v heads")
    nh = width // hd - 2 * n_kv
    row = qkv.stride()
    require(qkv.is_cuda and row[1] == 1, "qk norm: qkv must be a CUDA tensor with contiguous rows")
    require(q_weight.shape == k_weight.shape == (hd,) and q_weight.dtype is k_weight.dtype
            and q_weight.is_cuda and k_weight.is_cuda and q_weight.is_contiguous() and k_weight.is_contiguous(),
            "qk norm: q_weight and k_weight must be contiguous CUDA tensors [head_dim] of one type")
    require(rope.dim() == 3 and rope.shape[1] == 2 and rope.dtype is torch.float32 and rope.is_cuda
            and rope.is_contiguous(), "qk norm: rope must be a contiguous fp32 CUDA tensor [max_positions, 2, rot / 2]")
    for t in (positions, slots):
        require(t is None or (t.dtype is torch.int32 and t.is_cuda and t.is_contiguous() and t.numel() == n),
                "qk norm: positions and slots must be int32 contiguous CUDA tensors, one entry a token")
    require(slots is not None or n <= n_slots, "qk norm: without slots the pools need a row for each token")
    if out is None:
        if stream is None:
            out = torch.empty(n, nh, hd, dtype=qkv.dtype, device=qkv.device)
        else:
            with torch.cuda.stream(torch.cuda.ExternalStream(stream, qkv.device)):
                out = torch.empty(n, nh, hd, dtype=qkv.dtype, device=qkv.device)
    to = out.stride()
    require(out.shape == (n, nh, hd) and out.dtype is qkv.dtype and out.is_cuda and to[2] == 1 and to[1] == hd,
            "qk norm: out must be a CUDA tensor [T, n_heads, head_dim] of qkv's type with contiguous rows")
    before = (qkv.data_ptr(), row[0] if n > 1 else width, q_weight.data_ptr(), k_weight.data_ptr(), rope.data_ptr(),
              positions.data_ptr(), 0 if slots is None else slots.data_ptr(), k_pool.data_ptr(),
              v_pool.data_ptr(), slot_stride, out.data_ptr(), to[0] if n > 1 else nh * hd)
    after = (type_code(qkv.dtype, "qk norm"), type_code(q_weight.dtype, "qk norm"),
             type_code(k_pool.dtype, "qk norm"), n, nh, n_kv, hd, rope.shape[0], 2 * rope.shape[2],
             int(interleaved), n_slots, eps)
    enqueue(_lib.lib().ls_qk_norm_rope, _pack, before, after, qkv.device, status, stream)
    return out
