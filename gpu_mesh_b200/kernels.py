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

Page sizes 16, 32, 64 and 128, head sizes 8, 16, 32, 64 and 128, up to 16 query heads per KV head, 2048 sequences
and 2^26 - 1 token rows per call.  bf16 with head sizes 64 and 128 runs attention on the tensor cores.

The current stream runs the work, and nothing waits for it (a call can be captured once one has run on its device
outside a capture).  What only the device can see is raised by ``paged_check_device``: a length or rows outside the
table, the bound or the batch, which leave that sequence out, and a page id outside the pool, which leaves out that
page: nothing is stored for its tokens, and attention takes its keys and values as zeros, so that the rows of that
sequence are written but mean nothing.  Other sequences are not disturbed.
"""
from __future__ import annotations

import contextlib

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


def _refuse(x, k_pages, v_pages, page_table, q_start, kv_len, k_scale, v_scale) -> None:
    """Raise for what ``_paged`` found wrong; return where it was only the stride of a dimension of one element."""
    dev = x.device
    if x.dtype not in _DT or dev.type != "cuda":
        raise ValueError("the paged operators need CUDA fp32 or bf16 activations")
    if k_pages.ndim != 4 or k_pages.shape != v_pages.shape or k_pages.dtype != v_pages.dtype:
        raise ValueError("k_pages and v_pages must be [pages, kv heads, page size, head_dim] of one dtype")
    if k_pages.device != dev or v_pages.device != dev:
        raise ValueError("the pages must be on the activations' device")
    if k_pages.dtype != x.dtype and k_pages.dtype != torch.float8_e4m3fn:
        raise ValueError("the pages must hold the activation dtype or torch.float8_e4m3fn")
    if k_pages.shape[3] > 1 and (k_pages.stride(3) != 1 or v_pages.stride(3) != 1):
        raise ValueError("head_dim must be contiguous in the pages")
    if k_pages.dtype == torch.float8_e4m3fn:
        for s in (k_scale, v_scale):
            if s is None or s.dtype != torch.float32 or s.device != dev or s.shape != k_pages.shape[:2] or \
                    (s.shape[1] > 1 and s.stride(1) != 1):
                raise ValueError("e4m3 pages need fp32 k_scale and v_scale [pages, kv heads] on their device")
    elif k_scale is not None or v_scale is not None:
        raise ValueError("only e4m3 pages have scales")
    for name, t, ndim in (("page_table", page_table, 2), ("q_start", q_start, 1), ("kv_len", kv_len, 1)):
        if t.dtype != torch.int32 or t.ndim != ndim or t.device != dev:
            raise ValueError(f"{name} must be a {ndim}-D torch.int32 tensor on {dev}")
        if t.shape[-1] > 1 and t.stride(-1) != 1:
            raise ValueError(f"{name} rows must be contiguous")
    if page_table.shape[0] != kv_len.shape[0] or q_start.shape[0] != kv_len.shape[0] + 1:
        raise ValueError("page_table, q_start and kv_len disagree on the number of sequences")


def _paged(x, T, k_pages, v_pages, page_table, q_start, kv_len, k_scale, v_scale, max_new):
    """The C structures of a pool and a batch as bytes, checked against the ``T`` rows of activations ``x``.

    Decode steps call this twice per layer, so each tensor property is read once and by its cheapest accessor, and
    the checks are one expression; ``_refuse`` then names what it found."""
    index, kd, shape = x.get_device(), k_pages.dtype, k_pages.shape
    ks, vs, ts, table = k_pages.stride(), v_pages.stride(), page_table.stride(), page_table.shape
    e4m3, i32, B = kd is torch.float8_e4m3fn, torch.int32, kv_len.numel()
    if not (index >= 0 and x.dtype in _DT and len(shape) == 4 and v_pages.shape == shape and v_pages.dtype is kd
            and (e4m3 or kd is x.dtype) and k_pages.get_device() == index and v_pages.get_device() == index
            and ks[3] == 1 and vs[3] == 1
            and page_table.dtype is i32 and q_start.dtype is i32 and kv_len.dtype is i32
            and page_table.get_device() == index and q_start.get_device() == index and kv_len.get_device() == index
            and len(table) == 2 and table[0] == B and ts[1] == 1 and q_start.ndim == 1 and kv_len.ndim == 1
            and q_start.numel() == B + 1 and q_start.is_contiguous() and kv_len.is_contiguous()):
        _refuse(x, k_pages, v_pages, page_table, q_start, kv_len, k_scale, v_scale)
    pages, nkv, ps, D = shape
    kp = vp = kr = vr = 0
    if e4m3:
        good = k_scale is not None and v_scale is not None
        if good:
            rows, kst, vst = shape[:2], k_scale.stride(), v_scale.stride()
            good = (k_scale.dtype is torch.float32 and v_scale.dtype is torch.float32 and k_scale.shape == rows
                    and v_scale.shape == rows and kst[1] == 1 and vst[1] == 1
                    and k_scale.get_device() == index and v_scale.get_device() == index)
        if not good:
            _refuse(x, k_pages, v_pages, page_table, q_start, kv_len, k_scale, v_scale)
        kp, vp, kr, vr = k_scale.data_ptr(), v_scale.data_ptr(), kst[0], vst[0]
    elif k_scale is not None or v_scale is not None:
        _refuse(x, k_pages, v_pages, page_table, q_start, kv_len, k_scale, v_scale)
    if max_new is None or max_new > T:
        max_new = T
    elif max_new < 0:
        raise ValueError("max_new must not be negative")
    return _lib.PAGED_POOL.pack(k_pages.data_ptr(), v_pages.data_ptr(), kp, vp, ks[0], ks[1], ks[2], vs[0], vs[1], vs[2],
                                kr, vr, pages, ps, nkv, D, _PAGED_DT[kd]), \
        _lib.PAGED_BATCH.pack(page_table.data_ptr(), q_start.data_ptr(), kv_len.data_ptr(), ts[0], B, T, table[1], max_new)


_HERE = contextlib.nullcontext()


def _current(index: int):
    """Makes device ``index`` current, at no cost where it is already."""
    return _HERE if torch.cuda.current_device() == index else torch.cuda.device(index)


# The current stream's handle, without the Stream object that torch.cuda.current_stream builds.
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (
    lambda index: torch.cuda.current_stream(index).cuda_stream)


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
    if qkv.ndim != 2:
        raise ValueError("qkv must be [T, (num_q_heads + 2 kv heads) * head_dim]")
    (T, width), (ld, inner) = qkv.shape, qkv.stride()
    pool, batch = _paged(qkv, T, k_pages, v_pages, page_table, q_start, kv_len, k_scale, v_scale, max_new)
    dev, (_, nkv, _, D) = qkv.device, k_pages.shape
    if num_q_heads < 1 or width != (num_q_heads + 2 * nkv) * D:
        raise ValueError("qkv must be [T, (num_q_heads + 2 kv heads) * head_dim]")
    if inner != 1 and width > 1:
        raise ValueError("qkv rows must be contiguous")
    c = sn = qn = kn = pos = max_pos = 0
    if cos is not None or sin is not None:
        if cos is None or sin is None:
            raise ValueError("cos and sin come together")
        max_pos = cos.shape[0]
        table = (max_pos, D // 2)
        if not (cos.dtype is torch.float32 and sin.dtype is torch.float32 and cos.shape == table and sin.shape == table
                and cos.device == dev and sin.device == dev and cos.is_contiguous() and sin.is_contiguous()):
            raise ValueError(f"cos and sin must be contiguous fp32 [positions, head_dim / 2] tables on {dev}")
        c, sn = cos.data_ptr(), sin.data_ptr()
    if q_norm is not None or k_norm is not None:
        if not 0.0 < eps < 3.4e38:
            raise ValueError("eps must be positive")
        for name, t in (("q_norm", q_norm), ("k_norm", k_norm)):
            if t is not None and (t.dtype is not qkv.dtype or t.device != dev or t.shape != (D,) or not t.is_contiguous()):
                raise ValueError(f"{name} must be a contiguous [head_dim] tensor in the activation dtype")
        qn = 0 if q_norm is None else q_norm.data_ptr()
        kn = 0 if k_norm is None else k_norm.data_ptr()
    if positions is not None:
        if positions.dtype is not torch.int64 or positions.shape != (T,) or positions.device != dev or \
                (T > 1 and positions.stride(0) != 1):
            raise ValueError("positions must be contiguous int64 with one entry per token row")
        pos = positions.data_ptr()
    ldq = num_q_heads * D
    if out is None:
        out = qkv.new_empty((T, num_q_heads, D))
    elif out.shape != (T, num_q_heads, D) or out.dtype != qkv.dtype or out.device != dev or \
            out.stride(2) != 1 or (num_q_heads > 1 and out.stride(1) != D):
        raise ValueError("out must be [T, num_q_heads, head_dim] with contiguous token rows")
    else:
        ldq = out.stride(0)
    index = dev.index
    args = _lib.PAGED_APPEND_ARGS.pack(qkv.data_ptr(), pos, c, sn, qn, kn, out.data_ptr(), ld, ldq, _DT[qkv.dtype],
                                       num_q_heads, max_pos, eps)
    with _current(index):
        _lib.check(_lib.lib().mg_paged_append(pool, batch, args, _raw_stream(index)))
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
    strides = q.stride()
    if len(strides) != 3 or strides[2] != 1:
        raise ValueError("q must be [T, query heads, head_dim] with head_dim contiguous")
    T, nq, D = q.shape
    pool, batch = _paged(q, T, k_pages, v_pages, page_table, q_start, kv_len, k_scale, v_scale, max_new)
    if k_pages.shape[3] != D:
        raise ValueError("q and the pages disagree on head_dim")
    if out is None:
        out = torch.empty_like(q)
    elif out.shape != q.shape or out.dtype != q.dtype or out.device != q.device or out.stride(2) != 1:
        raise ValueError("out must have q's shape and dtype, with head_dim contiguous")
    if scale is None:
        scale = D ** -0.5
    elif not 0.0 < scale < 3.4e38:
        raise ValueError("scale must be positive and finite")
    lib, dt, index = _lib.lib(), _DT[q.dtype], q.get_device()
    (ql, qh, _), (ol, oh, _) = strides, out.stride()
    with _current(index):
        need, ws = lib.mg_paged_attention_workspace(pool, batch, dt, nq), 0
        if need:
            scratch = q.new_empty(need, dtype=torch.uint8)
            ws = scratch.data_ptr()
        args = _lib.PAGED_ATTENTION_ARGS.pack(q.data_ptr(), out.data_ptr(), ws, need, ql, qh, ol, oh, dt, nq, scale)
        _lib.check(lib.mg_paged_attention(pool, batch, args, _raw_stream(index)))
    return out


def paged_check_device(device: torch.device | str | int | None = None) -> None:
    """Wait for the current stream and raise what the paged calls on ``device`` met since the last check."""
    with torch.cuda.device(device):
        _lib.check(_lib.lib().mg_paged_check_device(torch.cuda.current_stream().cuda_stream))
