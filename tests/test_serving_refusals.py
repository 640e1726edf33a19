"""What the shared-prefix operators refuse on the host, through the C ABI, before any GPU work."""

import pytest

from loopspec_b200 import _lib


@pytest.fixture(scope="module")
def lib():
    from loopspec_b200.build import build
    build()
    return _lib.lib()


def refused(lib, call, args_type, good, **change):
    fields = dict(good, **change)
    pack = _lib.packer(args_type)
    code = call(pack(*(fields[name] for name, _ in args_type._fields_)), None)
    assert code == _lib.LS_EINVAL
    return lib.ls_last_error(None).decode()


SLOTS = dict(lens=256, delta=256, block_table=256, table_stride=8, free_blocks=256, free_count=256, slots=256,
             positions=256, requests=256, token_start=256, lens_out=256, free_count_out=256, status=256,
             n_requests=4, table_width=8, free_capacity=16, n_blocks=16, page_size=16, base=0, max_tokens=32)


@pytest.mark.parametrize("change", [
    dict(lens=0), dict(status=0), dict(slots=0), dict(n_requests=0), dict(n_requests=16385), dict(table_width=0),
    dict(table_stride=7), dict(free_capacity=-1), dict(n_blocks=0), dict(page_size=0), dict(page_size=24),
    dict(page_size=2048), dict(base=-1), dict(base=2 ** 31 - 5), dict(max_tokens=-1), dict(n_blocks=2 ** 28),
    dict(table_width=2 ** 30, table_stride=2 ** 30)])
def test_slot_maps(lib, change):
    assert "slot maps" in refused(lib, lib.ls_build_slots, _lib.SlotsArgs, SLOTS, **change)


QK = dict(qkv=256, qkv_stride=512, q_weight=256, k_weight=256, rope=256, positions=256, slots=0, k_pool=256, v_pool=256,
          slot_stride=128, q_out=256, q_out_stride=256, status=256, qkv_type=0, weight_type=0, cache_type=0, n_tokens=3,
          n_heads=4, n_kv_heads=2, head_dim=64, max_positions=10, rot=64, interleaved=0, n_slots=8, eps=1e-6)


@pytest.mark.parametrize("change", [
    dict(qkv=0), dict(status=0), dict(positions=0), dict(n_tokens=-1), dict(n_heads=0), dict(n_kv_heads=0),
    dict(head_dim=96), dict(rot=8), dict(rot=24), dict(rot=80), dict(qkv_type=3), dict(qkv_type=1),
    dict(cache_type=2), dict(weight_type=-1), dict(max_positions=0), dict(n_slots=0), dict(qkv_stride=504),
    dict(qkv_stride=515), dict(slot_stride=64), dict(q_out_stride=248), dict(qkv=264), dict(k_pool=258),
    dict(q_out_stride=257)])
def test_qk_norm(lib, change):
    assert "qk norm" in refused(lib, lib.ls_qk_norm_rope, _lib.QkNormArgs, QK, **change)


ATTN = dict(q=256, q_stride=512, k_pool=256, v_pool=256, slot_stride=256, prefix_table=256, block_table=256,
            table_stride=8, lens=256, token_start=256, out=256, out_stride=512, workspace=256, workspace_bytes=1 << 40,
            status=256, q_type=0, cache_type=0, n_tokens=3, n_requests=2, n_heads=8, n_kv_heads=4, head_dim=64,
            prefix_len=100, max_new=2, max_len=128, page_size=16, n_slots=512, scale=0.125)


@pytest.mark.parametrize("change", [
    dict(q=0), dict(status=0), dict(workspace=0), dict(prefix_table=0), dict(block_table=0), dict(lens=0),
    dict(n_tokens=-1), dict(n_requests=0), dict(n_heads=6), dict(n_kv_heads=0), dict(head_dim=96), dict(prefix_len=-1),
    dict(max_new=-1), dict(max_len=-1), dict(max_len=129), dict(page_size=12), dict(page_size=0), dict(n_slots=0),
    dict(q_type=1), dict(cache_type=2), dict(q_type=5), dict(q_stride=504), dict(q_stride=516), dict(out_stride=500),
    dict(slot_stride=128), dict(slot_stride=260), dict(q=264), dict(v_pool=260), dict(scale=float("inf")),
    dict(scale=float("nan")), dict(n_tokens=2 ** 30)])
def test_prefix_attention(lib, change):
    assert "prefix attention" in refused(lib, lib.ls_prefix_attention, _lib.PrefixAttentionArgs, ATTN, **change)


def test_null_structs(lib):
    for call in (lib.ls_build_slots, lib.ls_qk_norm_rope, lib.ls_prefix_attention):
        assert call(None, None) == _lib.LS_EINVAL
    assert lib.ls_check_status(None, None) == _lib.LS_EINVAL
    assert lib.ls_prefix_attention_workspace_bytes(4, 2, 6, 4, 64, 10, 1, 10) == 0    # 6 heads on 4


def test_python_entry_points_refuse_before_the_library():
    import torch
    from loopspec_b200.prefix_attention import prefix_attention
    from loopspec_b200.qk_norm import qk_norm_rope
    from loopspec_b200.slots import SlotMap, build_slots
    x = torch.zeros(4, 2, 64, dtype=torch.bfloat16)
    i = torch.zeros(3, dtype=torch.int32)
    with pytest.raises(ValueError):     # CPU tensors
        prefix_attention(x, x, x, i, 1, i[:2, None], i[:2], i, page_size=1, max_new=1)
    with pytest.raises(ValueError):
        qk_norm_rope(torch.zeros(4, 512, dtype=torch.bfloat16), x[0, 0], x[0, 0], torch.zeros(9, 2, 32), i, x, x)
    with pytest.raises(ValueError):
        build_slots(i, i, i[:, None], i, i[:1], page_size=1, n_blocks=3, out=SlotMap(3, 4, "cpu"))


def test_rope_table_keeps_long_positions():
    import math

    import torch
    from loopspec_b200.qk_norm import rope_table
    t = rope_table(100001, 64, 10000.0, device="cpu")
    assert t.shape == (100001, 2, 32) and t.dtype is torch.float32
    for i in (0, 1, 31):
        angle = 100000 * 10000.0 ** (-2 * i / 64)
        assert abs(float(t[100000, 0, i]) - math.cos(angle)) < 2e-7
        assert abs(float(t[100000, 1, i]) - math.sin(angle)) < 2e-7
