"""What flash_attn_tree_with_kvcache refuses, on the C entry point (no GPU) and in Python."""
import pytest
import torch

import fa_b200_capi as capi
import flash_attn_npu_3 as fa


def params():
    t = capi.TreeParams()
    p = t.fwd
    p.dtype, p.b, p.sq, p.sk, p.hq, p.hkv, p.d, p.dv, p.scale = 1, 2, 8, 256, 8, 2, 64, 64, 0.125
    for x in (p.q, p.k, p.v, p.o):
        x.ptr, x.stride_b, x.stride_s, x.stride_h = 0x1000, 4096, 512, 64
    p.seqused_k, p.kv_entries, p.block_table, p.page_size, p.block_table_stride = 0x1000, 16, 0x1000, 64, 4
    p.window_left, p.window_right = -1, -1
    t.parents, t.parents_stride_b, t.axes = 0x1000, 8, 1
    return t


@pytest.mark.parametrize("change,code,word", [
    (lambda t: setattr(t.fwd, "dtype", 5), 2, b"fp16"),
    (lambda t: setattr(t.fwd, "hq", 7), 3, b"divisible"),
    (lambda t: setattr(t.fwd, "sq", 257), 5, b"256"),
    (lambda t: setattr(t.fwd, "d", 60), 3, b"head dimension"),
    (lambda t: setattr(t.fwd, "dv", 128), 3, b"head dimension"),
    (lambda t: setattr(t.fwd, "seqused_k", None), 1, b"cache_seqlens"),
    (lambda t: setattr(t, "parents", None), 1, b"tree_parents"),
    (lambda t: setattr(t.fwd, "kv_entries", 0), 3, b"pages"),
    (lambda t: setattr(t.fwd, "page_size", 0), 3, b"page_size"),
    (lambda t: setattr(t.fwd, "cache_batch_idx", 0x1000), 5, b"cache_batch_idx"),
    (lambda t: setattr(t.fwd, "alibi_slopes", 0x1000), 5, b"alibi"),
    (lambda t: setattr(t.fwd, "num_splits", -1), 3, b"num_splits"),
    (lambda t: setattr(t.fwd, "rotary_cos", 0x1000), 1, b"rotary"),
    (lambda t: setattr(t.fwd.k_new, "ptr", 0x1000), 1, b"together"),
    (lambda t: setattr(t.fwd.q, "ptr", 0x1008), 4, b"aligned"),
    (lambda t: setattr(t.fwd.k, "stride_s", 513), 4, b"strides"),
    (lambda t: setattr(t.fwd, "softcap", -1.0), 3, b"softcap"),
    (lambda t: None, 6, b"workspace"),
])
def test_c_entry_point(change, code, word):
    t = params()
    change(t)
    assert capi.lib.fa_tree_fwd_kvcache(t) == code and word in capi.lib.fa_last_error()


def test_c_entry_point_nothing_to_do():
    assert capi.lib.fa_tree_fwd_kvcache(None) == 1
    for field in ("b", "sq"):
        t = params()
        setattr(t.fwd, field, 0)
        assert capi.lib.fa_tree_fwd_kvcache(t) == 0 and capi.lib.fa_tree_workspace_bytes(t) == 0
    assert capi.lib.fa_tree_workspace_bytes(params()) >= 2 * 8 * (4 + 4) + 2 * 8 * 8 * 64 * 2


def test_cpu_tensors_are_refused():
    z = torch.zeros(1, 2, 4, 64, dtype=torch.bfloat16)
    i = torch.zeros(1, 2, dtype=torch.int32)
    with pytest.raises(RuntimeError, match="CUDA"):
        fa.flash_attn_tree_with_kvcache(z, z, z, z, z, i, cache_seqlens=i[:, 0])


@pytest.mark.gpu
@pytest.mark.parametrize("change,word", [
    (dict(tree_parents=torch.zeros(2, 6)), "int32"),
    (dict(tree_parents=torch.zeros(2, 5, dtype=torch.int32)), "shape"),
    (dict(cache_seqlens=torch.zeros(3, dtype=torch.int32)), "shape"),
    (dict(cache_seqlens=None), "int32"),
    (dict(window_size=(4, 4)), "window"),
    (dict(v=None), "together"),
    (dict(k=torch.zeros(2, 6, 4, 64, dtype=torch.bfloat16)), "shape"),
    (dict(q=torch.zeros(2, 6, 4, 64, dtype=torch.float16)), "dtype"),
    (dict(q=torch.zeros(2, 6, 4, 64)), "FP16"),
    (dict(q=torch.zeros(2, 6, 3, 64, dtype=torch.bfloat16)), "divide"),
    (dict(cache_batch_idx=torch.zeros(2, dtype=torch.int32)), "paged"),
    (dict(rotary_positions=torch.zeros(2, 6, dtype=torch.int32)), "rotary_cos"),
    (dict(rotary_cos=torch.zeros(9, 32), rotary_sin=torch.zeros(9, 16)), "rotary"),
    (dict(rotary_cos=torch.zeros(9, 40), rotary_sin=torch.zeros(9, 40)), "rotary_dim"),
    (dict(rotary_cos=torch.zeros(9, 32), rotary_sin=torch.zeros(9, 32), rotary_sections=[16, 17]), "sum"),
    (dict(rotary_cos=torch.zeros(9, 32), rotary_sin=torch.zeros(9, 32), rotary_sections=[16, 16],
          rotary_positions=torch.zeros(3, 2, 6, dtype=torch.int32)), "positions"),
    (dict(rotary_cos=torch.zeros(9, 32), rotary_sin=torch.zeros(9, 32), rotary_sections=[7, 7, 6, 6, 6]), "axes"),
    (dict(softcap=-1.0), "softcap"),
    (dict(num_splits=-1), "num_splits"),
])
def test_python_refusals(change, word):
    bf = dict(dtype=torch.bfloat16, device="cuda")
    a = dict(q=torch.zeros(2, 6, 4, 64, **bf), k_cache=torch.zeros(4, 64, 2, 64, **bf), v_cache=torch.zeros(4, 64, 2, 64, **bf),
             k=torch.zeros(2, 6, 2, 64, **bf), v=torch.zeros(2, 6, 2, 64, **bf),
             tree_parents=torch.full((2, 6), -1, dtype=torch.int32, device="cuda"),
             cache_seqlens=torch.zeros(2, dtype=torch.int32, device="cuda"),
             page_table=torch.zeros(2, 2, dtype=torch.int32, device="cuda"))
    a.update({k: (x.cuda() if isinstance(x, torch.Tensor) else x) for k, x in change.items()})
    with pytest.raises(RuntimeError, match=word):
        fa.flash_attn_tree_with_kvcache(**a)
