"""Decoding from a cache, the part that needs no GPU: refusals of the Python calls and of the C ABI, and the arithmetic of the
block tables' own model (which the GPU tests hold the kernel to)."""
import numpy as np
import pytest
import torch

from paged_model import block_tables_model, release_model
from sys1_b200 import _lib, device, paged, qwen35


def _i(*shape):
    return torch.zeros(shape, dtype=torch.int32)


def _b(*shape):
    return torch.zeros(shape, dtype=torch.bfloat16)


def test_python_calls_refuse_cpu_tensors():
    with pytest.raises(ValueError, match="CUDA"):
        paged.block_tables(_i(2), _i(2, 4), _i(8), _i(1), 16)
    with pytest.raises(ValueError, match="CUDA"):
        paged.release_blocks(_i(2), _i(2), _i(2, 4), _i(8), _i(1), 16)
    with pytest.raises(ValueError, match="CUDA"):
        paged.cache_write(_b(3, 2, 64), _b(3, 2, 64), _b(4, 16, 2, 64), _b(4, 16, 2, 64), _i(3))
    with pytest.raises(ValueError, match="CUDA"):
        paged.attention_paged(_b(2, 4, 64), _b(4, 16, 2, 64), _b(4, 16, 2, 64), _i(2, 4), _i(2))
    with pytest.raises(ValueError, match="CUDA"):
        qwen35.gated_delta_rule_step(_b(2, 384), _b(384, 4), _i(2), _b(2, 1), _b(2, 1), torch.zeros(1), torch.zeros(1), _b(2, 128), _b(128), 1e-6,
                                     _b(2, 4, 384), torch.zeros(2, 1, 128, 128), 1)
    cfg = type("Cfg", (), dict(linear_num_key_heads=1, linear_num_value_heads=1, num_hidden_layers=0, head_dim=64))()
    with pytest.raises(ValueError, match="GPU"):
        paged.PagedCache(cfg, rows=1, num_pages=1, dev="cpu")
    with pytest.raises(ValueError, match="power of two"):
        paged.PagedCache(cfg, rows=1, num_pages=1, page_size=24)


@pytest.mark.parametrize("bad,match", [(dict(rows=8193), "8192"), (dict(page_size=1 << 17), "65536"), (dict(num_pages=1 << 26), "2.31"),
                                       (dict(max_length=(1 << 30) + 1), "2.30"), (dict(head_dim=96), "96")])
def test_the_cache_refuses_what_its_kernels_do(bad, match):
    """Before anything is allocated: a step that the kernels refuse would leave the rows' lengths a token ahead of their keys."""
    cfg = type("Cfg", (), dict(linear_num_key_heads=1, linear_num_value_heads=1, num_hidden_layers=0, head_dim=bad.pop("head_dim", 64)))()
    with pytest.raises(ValueError, match=match):
        paged.PagedCache(cfg, **{**dict(rows=1, num_pages=1), **bad}, dev="cpu")


def test_c_calls_refuse_a_null_context():
    lib = _lib.load_library()
    n = None
    assert lib.s1_block_tables(n, n, n, 1, 16, n, 0, n, n, n, 1, 1, n, n, n, n, 1) == _lib.S1_EINVAL
    assert lib.s1_release_blocks(n, n, 1, 16, n, n, 1, 1, n, 0, n) == _lib.S1_EINVAL
    assert lib.s1_cache_write(n, n, 0, 0, n, 0, 0, n, 0, 1, 64, n, 0.0, n, n, n, 0, 0, 0, n, n, 1, 16, 64, 64, 64) == _lib.S1_EINVAL
    assert lib.s1_attention_paged(n, n, 0, 0, n, n, 1, 16, 0, 0, 0, n, 0, 0, n, 1, 1, 1, 64, 1.0, n, 0, 0, n, 0, n, 0) == _lib.S1_EINVAL
    assert lib.s1_gated_delta_rule_step(n, n, 0, n, n, n, n, 0, n, n, n, 0, n, 0.0, n, 1, n, n, 1, 1, 1, n, 0) == _lib.S1_EINVAL
    assert lib.s1_gated_delta_rule_prefill(n, n, 0, n, n, n, n, 0, n, n, n, 0, n, 0.0, n, 1, 1, 1, 1, n, 0, n, 0, n, n, 1, n, n) == _lib.S1_EINVAL


@pytest.mark.skipif(torch.cuda.is_available(), reason="says what happens without a GPU")
@pytest.mark.parametrize("ordinal", [None, 0])
def test_a_context_without_a_gpu_says_so(ordinal):
    with pytest.raises(Exception) as plain:
        torch.cuda.init()
    with pytest.raises(type(plain.value)) as e:
        device.load(ordinal)
    assert str(e.value) == str(plain.value)


def test_the_binding_refuses_what_is_no_argument():
    """Before any of it is read: another number of arguments, things that are no tensors, no numbers, or integers that the C ABI would cut off."""
    b = _lib.load_binding()
    for call, n in ((b.block_tables, 10), (b.cache_write, 13), (b.attention_paged, 10), (b.gated_delta_rule_step, 16)):
        for m in (0, n - 1, n + 1):
            with pytest.raises(TypeError, match=f"{n} arguments"):
                call(*[None] * m)
        with pytest.raises(ValueError, match="must be a tensor"):
            call(*[None] * n)
    for page, error in ((1 << 32, ValueError), (1 << 70, OverflowError), (1.5, TypeError), (None, TypeError)):
        with pytest.raises(error):
            paged.block_tables(_i(2), _i(2, 4), _i(8), _i(1), page)
    with pytest.raises(ValueError, match="max_tokens is needed"):
        paged.block_tables(_i(2), _i(2, 4), _i(8), _i(1), 16, added=_i(2))
    with pytest.raises(ValueError, match="must not be negative"):
        paged.block_tables(_i(2), _i(2, 4), _i(8), _i(1), 16, max_tokens=-1)
    with pytest.raises(ValueError, match="v must be a tensor"):
        paged.cache_write(_b(3, 2, 64), [1], _b(4, 16, 2, 64), _b(4, 16, 2, 64), _i(3))


def test_workspace_sizes():
    assert paged.attention_paged_workspace(96) == 0
    assert 0 < paged.attention_paged_workspace(64) < paged.attention_paged_workspace(128) < paged.attention_paged_workspace(256)


def test_model_of_the_block_tables():
    tables = np.full((4, 3), -1, np.int32)
    tables[1, 0] = 7
    r = block_tables_model([0, 3, -1, 0], [5, 2, 9, 0], 4, [5, 6, 9, 8], 4, tables, 8)
    assert r["lengths"] == [5, 5, -1, 0] and r["cu_seqlens"] == [0, 5, 7, 7, 7] and r["left"] == 1 and not r["refused"]
    assert r["tables"].tolist() == [[8, 9, -1], [7, 6, -1], [-1, -1, -1], [-1, -1, -1]]
    assert r["positions"] == [0, 1, 2, 3, 4, 3, 4, 0] and r["slots"] == [32, 33, 34, 35, 36, 31, 24, -1]
    # one page is left for two rows that need one each: the second gets nothing, and a third that needs none is served
    tables = np.array([[2, -1], [3, -1], [4, -1]], np.int32)
    r = block_tables_model([4, 4, 1], None, 4, [0, 1], 1, tables, 3)
    assert r["refused"] == [1] and r["lengths"] == [5, 4, 2] and r["slots"] == [0, -1, 17] and r["positions"] == [4, 0, 1] and r["left"] == 0


def test_model_of_the_release():
    tables = np.array([[3, 4], [5, 6]], np.int32)
    free, count, lengths, refused = release_model([1, 0], [6, 8], tables, [9, -1, -1], 1, 4)
    assert free == [9, 3, 4] and count == 3 and lengths == [-1, 8] and not refused
    assert release_model([1, 1], [6, 8], tables, [9, -1, -1], 1, 4)[3] == [1]
