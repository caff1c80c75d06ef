"""What the serving operators refuse without a GPU: host tensors in Python, and bad
arguments at the C entry points (they return before anything is launched)."""
import ctypes

import pytest
import torch

import megakernel_b200 as mk
from megakernel_b200 import _lib

INVALID, MISALIGNED = 1, 716  # cudaErrorInvalidValue, cudaErrorMisalignedAddress
A = 1 << 20  # an aligned address that no refused call touches


def attn(**kw):
    a = _lib.AttnArgs(dtype=0, heads=4, kv_heads=2, head_dim=128, tokens=8, batch=2, q_len=4, q=A, out=A, k=A, v=A,
                      kv_lens=A, block_table=A, table_stride=4, table_width=4, pages=9, page_size=16, scale=0.1)
    a.q_stride[:] = a.out_stride[:] = [512, 128]
    a.k_stride[:] = a.v_stride[:] = [4096, 2048, 128]
    for k, v in kw.items():
        if isinstance(v, list):
            getattr(a, k)[:] = v
        else:
            setattr(a, k, v)
    return ctypes.byref(a)


def append(**kw):
    a = _lib.AppendArgs(dtype=0, source_dtype=0, heads=4, kv_heads=2, head_dim=128, tokens=8, batch=2, q_len=4, qkv=A,
                        eps=1e-6, cos_table=A, sin_table=A, rope_fp32=1, rope_rows=64, q_out=A, k_cache=A, v_cache=A,
                        kv_lens=A, block_table=A, table_stride=4, table_width=4, pages=9, page_size=16)
    a.qkv_stride[:] = [1024, 128]
    a.k_stride[:] = a.v_stride[:] = [4096, 2048, 128]
    for k, v in kw.items():
        if isinstance(v, list):
            getattr(a, k)[:] = v
        else:
            setattr(a, k, v)
    return ctypes.byref(a)


@pytest.mark.parametrize("kw", [dict(dtype=2), dict(dtype=-1), dict(heads=3), dict(kv_heads=0), dict(head_dim=96),
                                dict(tokens=-1), dict(tokens=9), dict(batch=0), dict(q_len=0), dict(scale=0.0),
                                dict(scale=-1.0), dict(scale=float("inf")), dict(scale=float("nan")), dict(q=None),
                                dict(out=None), dict(k=None), dict(v=None)])
def test_attention_entry_points_refuse(kw):
    lib = _lib.load()
    assert lib.mkb_paged_attention(attn(**kw), None) == INVALID
    assert lib.mkb_prompt_attention(attn(**kw), None) == INVALID


@pytest.mark.parametrize("kw", [dict(page_size=8), dict(page_size=24), dict(page_size=0), dict(kv_lens=None),
                                dict(block_table=None), dict(pages=-1), dict(table_width=-1)])
def test_paged_entry_points_refuse(kw):
    assert _lib.load().mkb_paged_attention(attn(**kw), None) == INVALID
    assert _lib.load().mkb_paged_append(append(**kw), None) == INVALID


@pytest.mark.parametrize("kw", [dict(q=A + 2), dict(k=A + 8), dict(out=A + 4), dict(workspace=A + 8),
                                dict(q_stride=[512, 100]), dict(k_stride=[4096, 2048, -128]), dict(v_stride=[4, 8, 8]),
                                dict(out_stride=[1, 128])])
def test_misaligned_operands_are_refused(kw):
    assert _lib.load().mkb_paged_attention(attn(**kw), None) == MISALIGNED


@pytest.mark.parametrize("kw,code", [(dict(dtype=2), INVALID), (dict(source_dtype=3), INVALID), (dict(heads=0), INVALID),
                                     (dict(head_dim=32), INVALID), (dict(qkv=None), INVALID), (dict(tokens=7), INVALID),
                                     (dict(cos_table=None), INVALID), (dict(qkv=A + 8), MISALIGNED),
                                     (dict(k_out=A + 2), MISALIGNED), (dict(qkv_stride=[1024, 4]), MISALIGNED)])
def test_append_entry_point_refuses(kw, code):
    assert _lib.load().mkb_paged_append(append(**kw), None) == code


def test_nothing_to_do_is_no_error():
    lib = _lib.load()
    assert lib.mkb_paged_attention(attn(tokens=0, batch=0), None) == 0
    assert lib.mkb_prompt_attention(attn(tokens=0, batch=0), None) == 0
    assert lib.mkb_paged_append(append(tokens=0, batch=0), None) == 0
    assert lib.mkb_attn_workspace_bytes(attn()) > 0


def test_host_tensors_are_refused():
    x = torch.zeros((4, 2, 128), dtype=torch.bfloat16)
    cache = torch.zeros((3, 2, 16, 128), dtype=torch.bfloat16)
    n = torch.zeros(4, dtype=torch.int32)
    table = torch.zeros((4, 1), dtype=torch.int32)
    with pytest.raises(ValueError, match="CUDA"):
        mk.prompt_attention(x, x, x, n)
    with pytest.raises(ValueError, match="CUDA"):
        mk.paged_attention(x, cache, cache, table, n)
    with pytest.raises(ValueError, match="CUDA"):
        mk.paged_append(x, cache, cache, table, n, x, x)
