"""Direct access to single operators: the stage's linear layer
(``mg_linear``), and the paged KV cache (``mg_paged_append``,
``mg_paged_attention``).

The stage runs the linear layer inside ``mg_stage_forward``; exposing it
lets callers and tests drive one GEMM path at a time: the weight-streaming
GEMV (<= 32 rows), the tcgen05 GEMM (more rows, bf16) and the SIMT kernel
(fp32).

The paged operators serve callers that keep the keys and values of many
requests in one pool of pages, with a ragged batch per step (prompt chunks
beside single tokens)::

    q = paged_append(qkv, k_pages, v_pages, page_table, q_start, kv_len, num_q_heads=32,
                     cos=cos, sin=sin, k_scale=k_scale, v_scale=v_scale)
    out = paged_attention(q, k_pages, v_pages, page_table, q_start, kv_len,
                          k_scale=k_scale, v_scale=v_scale)

* ``k_pages`` / ``v_pages``: ``[pages, kv heads, page size, head_dim]`` in the activation dtype or
  ``torch.float8_e4m3fn``.  Any strides that are multiples of 16 bytes with ``head_dim`` contiguous: a layer of a
  larger pool, one half of an interleaved one, or a transposed ``[pages, page size, heads, head_dim]``.
* ``k_scale`` / ``v_scale``: fp32 ``[pages, kv heads]``, e4m3 pages only: the power of two that a page's codes
  are multiples of, kept by ``paged_append``.
* ``page_table``: int32 ``[sequences, columns]``; ``q_start``: int32 ``[sequences + 1]``, the token rows of each
  sequence; ``kv_len``: int32 ``[sequences]``, cached tokens with the new ones.  The kernels read them on the
  device: a captured call follows their contents.
* ``max_new``: a host bound on the new tokens of one sequence (default: all rows).  A step of single tokens
  should pass 1: it chooses the kernels.

The current stream runs the work, and nothing waits for it: what only the device can see (a page id outside the
pool, a length outside the table) leaves that sequence out and is raised by ``paged_check_device``.
"""
from __future__ import annotations

import math

import torch

from gpu_mesh_b200 import _lib

EPILOGUES = {"store": 0, "resid": 1, "swiglu": 2}
_DT = {torch.float32: _lib.MG_DTYPE_F32, torch.bfloat16: _lib.MG_DTYPE_BF16}


def linear(x: torch.Tensor, w: torch.Tensor, *, epilogue: str = "store",
           residual: torch.Tensor | None = None, out: torch.Tensor | None = None) -> torch.Tensor:
    """epilogue(x @ w.T) on the device; ``swiglu`` takes w = [gate; up]."""
    if x.dtype not in _DT or w.dtype != x.dtype or x.device.type != "cuda":
        raise ValueError("linear needs CUDA fp32 or bf16 tensors of one dtype")
    if x.stride(-1) != 1 or w.stride(-1) != 1 or not w.is_contiguous():
        raise ValueError("x rows and w must be contiguous")
    M, K = x.shape
    N = w.shape[0] // 2 if epilogue == "swiglu" else w.shape[0]
    if w.shape[1] != K:
        raise ValueError("x and w disagree on K")
    if out is None:
        out = torch.empty(M, N, dtype=x.dtype, device=x.device)
    code = EPILOGUES[epilogue]
    lib = _lib.lib()
    n_scr = lib.mg_linear_scratch(_DT[x.dtype], M, N, K, code)
    scratch = torch.empty(max(int(n_scr), 1), dtype=torch.float32, device=x.device)
    r = residual if residual is not None else None
    with torch.cuda.device(x.device):  # the kernel runs on x's GPU, on its current stream
        _lib.check(lib.mg_linear(
            _DT[x.dtype], x.data_ptr(), x.stride(0), w.data_ptr(), M, N, K, code,
            None if r is None else r.data_ptr(), 0 if r is None else r.stride(0),
            out.data_ptr(), out.stride(0), scratch.data_ptr(), scratch.numel(),
            torch.cuda.current_stream(x.device).cuda_stream,
        ))
    return out


_PAGED_DT = {torch.float32: _lib.MG_DTYPE_F32, torch.bfloat16: _lib.MG_DTYPE_BF16,
             torch.float8_e4m3fn: _lib.MG_DTYPE_E4M3}


def _index(name: str, t: torch.Tensor, device: torch.device, ndim: int, dtype: torch.dtype = torch.int32) -> None:
    if t.dtype != dtype or t.ndim != ndim or t.device != device:
        raise ValueError(f"{name} must be a {ndim}-D {dtype} tensor on {device}")
    if t.shape[-1] > 1 and t.stride(-1) != 1:
        raise ValueError(f"{name} rows must be contiguous")


def _paged(x, k_pages, v_pages, page_table, q_start, kv_len, k_scale, v_scale, max_new):
    """The C structures of a pool and a batch, checked against the activations ``x``."""
    dev = x.device
    if x.dtype not in _DT or dev.type != "cuda":
        raise ValueError("the paged operators need CUDA fp32 or bf16 activations")
    if k_pages.ndim != 4 or k_pages.shape != v_pages.shape or k_pages.dtype != v_pages.dtype:
        raise ValueError("k_pages and v_pages must be [pages, kv heads, page size, head_dim] of one dtype")
    if k_pages.device != dev or v_pages.device != dev:
        raise ValueError("the pages must be on the activations' device")
    if k_pages.dtype != x.dtype and k_pages.dtype != torch.float8_e4m3fn:
        raise ValueError("the pages must hold the activation dtype or torch.float8_e4m3fn")
    if k_pages.stride(3) != 1 or v_pages.stride(3) != 1:
        raise ValueError("head_dim must be contiguous in the pages")
    pages, nkv, ps, D = k_pages.shape
    scales = (None, None, 0, 0)
    if k_pages.dtype == torch.float8_e4m3fn:
        for s in (k_scale, v_scale):
            if s is None or s.dtype != torch.float32 or s.device != dev or s.shape != (pages, nkv) or \
                    (nkv > 1 and s.stride(1) != 1):
                raise ValueError("e4m3 pages need fp32 k_scale and v_scale [pages, kv heads] on their device")
        scales = (k_scale.data_ptr(), v_scale.data_ptr(), max(k_scale.stride(0), nkv), max(v_scale.stride(0), nkv))
        if pages > 1 and (k_scale.stride(0) < nkv or v_scale.stride(0) < nkv):
            raise ValueError("scale rows of two pages must not overlap")
    elif k_scale is not None or v_scale is not None:
        raise ValueError("only e4m3 pages have scales")
    _index("page_table", page_table, dev, 2)
    _index("q_start", q_start, dev, 1)
    _index("kv_len", kv_len, dev, 1)
    B = kv_len.shape[0]
    if page_table.shape[0] != B or q_start.shape[0] != B + 1:
        raise ValueError("page_table, q_start and kv_len disagree on the number of sequences")
    if max_new is None:
        max_new = x.shape[0]
    elif max_new < 0:
        raise ValueError("max_new must not be negative")
    pool = _lib.PagedPool(
        k_pages.data_ptr(), v_pages.data_ptr(), scales[0], scales[1],
        _stride(k_pages, 0), _stride(k_pages, 1), _stride(k_pages, 2),
        _stride(v_pages, 0), _stride(v_pages, 1), _stride(v_pages, 2), scales[2], scales[3],
        pages, ps, nkv, D, _PAGED_DT[k_pages.dtype])
    batch = _lib.PagedBatch(page_table.data_ptr(), q_start.data_ptr(), kv_len.data_ptr(), page_table.stride(0),
                            B, x.shape[0], page_table.shape[1], min(max_new, x.shape[0]))
    return pool, batch


def _stride(t: torch.Tensor, dim: int) -> int:
    """The stride of a dimension; of one element, whose stride means nothing, the one that a dense tensor has."""
    return t.stride(dim) if t.shape[dim] > 1 else max(1, math.prod(t.shape[dim + 1:]))


def paged_append(qkv: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor, page_table: torch.Tensor,
                 q_start: torch.Tensor, kv_len: torch.Tensor, *, num_q_heads: int, max_new: int | None = None,
                 cos: torch.Tensor | None = None, sin: torch.Tensor | None = None,
                 positions: torch.Tensor | None = None, q_norm: torch.Tensor | None = None,
                 k_norm: torch.Tensor | None = None, eps: float = 1e-6, k_scale: torch.Tensor | None = None,
                 v_scale: torch.Tensor | None = None, out: torch.Tensor | None = None) -> torch.Tensor:
    """Append the new tokens' keys and values to their pages; returns the queries ``[T, num_q_heads, head_dim]``.

    ``qkv`` is ``[T, (num_q_heads + 2 kv heads) * head_dim]``: each row's query heads, then key, then value heads
    (the fused projection).  Queries and keys pass the per-head RMSNorm (``q_norm`` / ``k_norm`` ``[head_dim]``,
    either may be None) and the rotary embedding (``cos`` / ``sin`` fp32 ``[positions, head_dim / 2]``, None for
    none) at ``positions`` (int64 ``[T]``) or at the token's place in its sequence, in fp32 with one rounding.
    Rows behind ``q_start[-1]`` are left as they are in ``out``.  No two sequences of a call may append to one
    page: a page that sequences share is full, or copied first.
    """
    pool, batch = _paged(qkv, k_pages, v_pages, page_table, q_start, kv_len, k_scale, v_scale, max_new)
    dev, nkv, D = qkv.device, pool.num_kv_heads, pool.head_dim
    if qkv.ndim != 2 or num_q_heads < 1 or qkv.shape[1] != (num_q_heads + 2 * nkv) * D:
        raise ValueError("qkv must be [T, (num_q_heads + 2 kv heads) * head_dim]")
    if qkv.stride(1) != 1:
        raise ValueError("qkv rows must be contiguous")
    if (cos is None) != (sin is None):
        raise ValueError("cos and sin come together")
    for name, t in (("cos", cos), ("sin", sin)):
        if t is not None and (t.dtype != torch.float32 or t.device != dev or t.ndim != 2 or t.shape[1] != D // 2
                              or t.shape != cos.shape or not t.is_contiguous()):
            raise ValueError(f"{name} must be a contiguous fp32 [positions, head_dim / 2] table on {dev}")
    for name, t in (("q_norm", q_norm), ("k_norm", k_norm)):
        if t is not None and (t.dtype != qkv.dtype or t.device != dev or t.shape != (D,) or not t.is_contiguous()):
            raise ValueError(f"{name} must be a contiguous [head_dim] tensor in the activation dtype")
    T = qkv.shape[0]
    if positions is not None:
        _index("positions", positions, dev, 1, torch.int64)
        if positions.shape[0] != T:
            raise ValueError("positions must have one entry per token row")
    if out is None:
        out = torch.empty(T, num_q_heads, D, dtype=qkv.dtype, device=dev)
    elif out.shape != (T, num_q_heads, D) or out.dtype != qkv.dtype or out.device != dev or \
            out.stride(2) != 1 or (num_q_heads > 1 and out.stride(1) != D):
        raise ValueError("out must be [T, num_q_heads, head_dim] with contiguous token rows")
    with torch.cuda.device(dev):
        _lib.check(_lib.lib().mg_paged_append(
            pool, batch, _DT[qkv.dtype], qkv.data_ptr(), _stride(qkv, 0), num_q_heads,
            None if positions is None else positions.data_ptr(), None if cos is None else cos.data_ptr(),
            None if sin is None else sin.data_ptr(), 0 if cos is None else cos.shape[0],
            None if q_norm is None else q_norm.data_ptr(), None if k_norm is None else k_norm.data_ptr(),
            eps, out.data_ptr(), _stride(out, 0), torch.cuda.current_stream(dev).cuda_stream))
    return out


def paged_attention(q: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor, page_table: torch.Tensor,
                    q_start: torch.Tensor, kv_len: torch.Tensor, *, max_new: int | None = None,
                    scale: float | None = None, k_scale: torch.Tensor | None = None,
                    v_scale: torch.Tensor | None = None, out: torch.Tensor | None = None) -> torch.Tensor:
    """Causal attention of the new tokens' queries ``[T, query heads, head_dim]`` over their sequences' pages.

    The s-th of a sequence's n new tokens sees its cached tokens j <= kv_len - n + s (a row that sees none gives
    0); ``scale`` defaults to head_dim ** -0.5.  Returns ``out`` (``[T, query heads, head_dim]``, not overlapping
    ``q``); rows behind ``q_start[-1]`` are left as they are in it.  The scratch is the call's own.
    """
    if q.ndim != 3 or q.stride(2) != 1:
        raise ValueError("q must be [T, query heads, head_dim] with head_dim contiguous")
    pool, batch = _paged(q, k_pages, v_pages, page_table, q_start, kv_len, k_scale, v_scale, max_new)
    dev, nq = q.device, q.shape[1]
    if q.shape[2] != pool.head_dim:
        raise ValueError("q and the pages disagree on head_dim")
    if out is None:
        out = torch.empty(q.shape, dtype=q.dtype, device=dev)
    elif out.shape != q.shape or out.dtype != q.dtype or out.device != dev or out.stride(2) != 1:
        raise ValueError("out must have q's shape and dtype, with head_dim contiguous")
    lib, dt = _lib.lib(), _DT[q.dtype]
    with torch.cuda.device(dev):
        need = lib.mg_paged_attention_workspace(pool, batch, dt, nq)
        ws = torch.empty(need, dtype=torch.uint8, device=dev) if need else None
        _lib.check(lib.mg_paged_attention(
            pool, batch, dt, q.data_ptr(), _stride(q, 0), _stride(q, 1), nq,
            pool.head_dim ** -0.5 if scale is None else scale, out.data_ptr(), _stride(out, 0), _stride(out, 1),
            None if ws is None else ws.data_ptr(), need, torch.cuda.current_stream(dev).cuda_stream))
    return out


def paged_check_device(device: torch.device | str | int | None = None) -> None:
    """Wait for the current stream and raise what the paged calls on ``device`` met since the last check."""
    with torch.cuda.device(device):
        _lib.check(_lib.lib().mg_paged_check_device(torch.cuda.current_stream().cuda_stream))
