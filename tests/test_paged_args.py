"""What the paged operators refuse, through the C ABI: every check runs before a GPU is touched."""
from __future__ import annotations

import ctypes

import pytest
import torch

from gpu_mesh_b200 import _lib, kernels

BASE = 1 << 20  # a fake device address: no call here gets as far as using it


def pool(**kw):
    D = kw.get("head_dim", 64)
    f = dict(k=BASE, v=2 * BASE, k_scale=None, v_scale=None, k_page_stride=2 * 16 * D, k_head_stride=16 * D,
             k_token_stride=D, v_page_stride=2 * 16 * D, v_head_stride=16 * D, v_token_stride=D, k_scale_stride=0,
             v_scale_stride=0, num_pages=8, page_size=16, num_kv_heads=2, head_dim=D, cache_dtype=_lib.MG_DTYPE_BF16)
    f.update(kw)
    return _lib.PagedPool(**f)


def batch(**kw):
    f = dict(page_table=BASE, q_start=BASE, kv_len=BASE, table_stride=4, batch=2, tokens=3, max_pages=4, max_new=2)
    f.update(kw)
    return _lib.PagedBatch(**f)


def append(p, b, dtype=_lib.MG_DTYPE_BF16, qkv=BASE, ld=8 * 64, nq=4, cos=None, sin=None, max_pos=0, qn=None, eps=1e-6,
           out=BASE, ldq=4 * 64):
    args = _lib.PagedAppendArgs(qkv, None, cos, sin, qn, None, out, ld, ldq, dtype, nq, max_pos, eps)
    return _lib.lib().mg_paged_append(p, b, args, None)


def attend(p, b, dtype=_lib.MG_DTYPE_BF16, q=BASE, qs=(256, 64), nq=4, scale=0.125, out=BASE, os=(256, 64), ws=BASE,
           nbytes=1 << 40):
    args = _lib.PagedAttentionArgs(q, out, ws, nbytes, *qs, *os, dtype, nq, scale)
    return _lib.lib().mg_paged_attention(p, b, args, None)


SHARED = [
    (dict(), dict(), dict(dtype=7), "dtype"),
    (dict(cache_dtype=_lib.MG_DTYPE_F32), dict(), dict(), "activation dtype or e4m3"),
    (dict(k=None), dict(), dict(), "null pages"),
    (dict(page_size=24), dict(), dict(), "page_size"),
    (dict(page_size=256), dict(), dict(), "page_size"),
    (dict(head_dim=96), dict(), dict(), "head_dim"),
    (dict(num_pages=0), dict(), dict(), "num_pages"),
    (dict(num_kv_heads=0), dict(), dict(), "num_kv_heads"),
    (dict(), dict(), dict(nq=3), "num_q_heads"),
    (dict(), dict(), dict(nq=34), "num_q_heads"),
    (dict(), dict(), dict(nq=0), "num_q_heads"),
    (dict(cache_dtype=_lib.MG_DTYPE_E4M3), dict(), dict(), "k_scale"),
    (dict(cache_dtype=_lib.MG_DTYPE_E4M3, k_scale=BASE, v_scale=BASE, k_scale_stride=1, v_scale_stride=2), dict(), dict(),
     "scale rows"),
    (dict(k_token_stride=32), dict(), dict(), "strides"),
    (dict(v_head_stride=1028), dict(), dict(), "strides"),
    (dict(k_page_stride=0), dict(), dict(), "strides"),
    (dict(v=BASE + 8), dict(), dict(), "16-byte"),
    (dict(), dict(batch=-1), dict(), "negative"),
    (dict(), dict(max_new=-1), dict(), "negative"),
    (dict(), dict(batch=2049), dict(), "2048"),
    (dict(), dict(tokens=1 << 26), dict(), "2^26"),
    (dict(), dict(q_start=None), dict(), "null"),
    (dict(), dict(max_pages=0), dict(), "columns"),
    (dict(), dict(max_pages=1 << 28, table_stride=1 << 28), dict(), "columns"),
    (dict(page_size=128), dict(max_pages=(1 << 23) + 1, table_stride=1 << 24), dict(), "2^30"),
    (dict(num_kv_heads=40000, page_size=16), dict(), dict(nq=80000), "65535"),
    (dict(), dict(table_stride=3), dict(), "table_stride"),
]


@pytest.mark.parametrize("p,b,kw,message", SHARED, ids=[f"{i}-{c[3]}" for i, c in enumerate(SHARED)])
@pytest.mark.parametrize("call", [append, attend])
def test_shared_refusals(call, p, b, kw, message):
    assert call(pool(**p), batch(**b), **kw) == _lib.MG_EINVAL
    assert message in _lib.last_error()


@pytest.mark.parametrize("kw,message", [
    (dict(qkv=None), "null"), (dict(out=None), "null"), (dict(ld=8 * 64 - 8), "rows"), (dict(ld=8 * 64 + 4), "rows"),
    (dict(ldq=4 * 64 - 8), "rows"), (dict(qkv=BASE + 2), "16-byte"), (dict(cos=BASE), "together"),
    (dict(cos=BASE, sin=BASE), "empty"), (dict(cos=BASE + 4, sin=BASE, max_pos=4), "16-byte"),
    (dict(qn=BASE, eps=0.0), "eps"),
])
def test_append_refusals(kw, message):
    assert append(pool(), batch(), **kw) == _lib.MG_EINVAL
    assert message in _lib.last_error()


@pytest.mark.parametrize("kw,message", [
    (dict(q=None), "null"), (dict(out=None), "null"), (dict(qs=(256, 32)), "strides"), (dict(os=(260, 64)), "strides"),
    (dict(q=BASE + 8), "16-byte"), (dict(scale=0.0), "scale"), (dict(scale=float("inf")), "scale"),
    (dict(scale=float("nan")), "scale"),
])
def test_attention_refusals(kw, message):
    assert attend(pool(), batch(), **kw) == _lib.MG_EINVAL
    assert message in _lib.last_error()


def test_null_structures_and_empty_batches():
    lib = _lib.lib()
    null_pool, null_batch = ctypes.POINTER(_lib.PagedPool)(), ctypes.POINTER(_lib.PagedBatch)()
    assert attend(null_pool, batch()) == _lib.MG_EINVAL
    assert append(pool(), null_batch) == _lib.MG_EINVAL
    assert lib.mg_paged_attention_workspace(null_pool, null_batch, 1, 4) == 0
    assert lib.mg_paged_append(pool(), batch(), None, None) == _lib.MG_EINVAL
    assert lib.mg_paged_attention(pool(), batch(), None, None) == _lib.MG_EINVAL
    for b in (batch(batch=0), batch(tokens=0)):  # nothing to do, and nothing touched
        assert append(pool(), b) == _lib.MG_OK
        assert attend(pool(), b) == _lib.MG_OK


def test_python_refuses_host_tensors():
    x = torch.zeros(1, 8 * 64, dtype=torch.bfloat16)
    pages = torch.zeros(2, 2, 16, 64, dtype=torch.bfloat16)
    ints = torch.zeros(1, 1, dtype=torch.int32)
    with pytest.raises(ValueError, match="CUDA"):
        kernels.paged_append(x, pages, pages, ints, ints[0], ints[0], num_q_heads=4)
    with pytest.raises(ValueError, match="CUDA"):
        kernels.paged_attention(x.view(1, 8, 64), pages, pages, ints, ints[0], ints[0])
