"""A paged KV cache and its two operators in 64 bits on the CPU, token by token, for the tests.

``Pool`` keeps what every page holds as the values that the store rounds (e4m3: codes and exponents, moved as the
operator documents), ``append`` and ``attend`` follow the formulas.  Nothing here uses the package.
"""
from __future__ import annotations

import math

import torch

E4M3 = torch.float8_e4m3fn
HALF = {torch.bfloat16: 2.0**-8, torch.float32: 2.0**-24}  # half a step, relative
F32 = 2.0**-24


def spans(q_start, kv_len):
    """(first row, new tokens, past) of every sequence."""
    return [(a, b - a, n - (b - a)) for a, b, n in zip(q_start, q_start[1:], kv_len)]


def least_exp(amax: float) -> int:
    if amax <= 0:
        return -100
    e = math.frexp(amax / 448.0)[1] - 1
    while 448.0 * 2.0**e < amax:
        e += 1
    while 448.0 * 2.0 ** (e - 1) >= amax:
        e -= 1
    return min(max(e, -100), 100)


def rotate(x, w, cos, sin, eps):
    """x [heads, D] in 64 bits: norm, rotation; and the magnitudes |x1 c| + |x2 s| that its error scales with."""
    if w is not None:
        x = x / (x.square().mean(-1, keepdim=True) + eps).sqrt() * w.double()
    if cos is None:
        return x, x.abs()
    h = x.shape[-1] // 2
    lo, hi, c, s = x[..., :h], x[..., h:], cos.double(), sin.double()
    y = torch.cat((lo * c - hi * s, hi * c + lo * s), -1)
    return y, torch.cat(((lo * c).abs() + (hi * s).abs(), (hi * c).abs() + (lo * s).abs()), -1)


def dense(pages, scale, table_row, length):
    """[heads, length, D] in 64 bits of one sequence."""
    ps = pages.shape[2]
    ids = table_row[: -(-length // ps)].long()
    x = pages.float()[ids].double() if pages.dtype == E4M3 else pages[ids].double()
    if scale is not None:
        x = x * scale[ids].double()[:, :, None, None]
    return x.transpose(0, 1).reshape(pages.shape[1], -1, pages.shape[3])[:, :length]


def attend(q, k, v, past, scale):
    """One sequence: q [n, nq, D], k / v [nkv, L, D] (64 bits) -> out, and per output the sum of p|v| and, over its
    visible keys, the largest scale·Σ|q||k| and the largest scale·max|q|·Σ|k|."""
    n, nq, D = q.shape
    nkv, L = k.shape[0], k.shape[1]
    kk, vv = k.repeat_interleave(nq // nkv, 0), v.repeat_interleave(nq // nkv, 0)
    s = torch.einsum("nhd,hld->hnl", q, kk) * scale
    mag = torch.einsum("nhd,hld->hnl", q.abs(), kk.abs()) * scale
    most = q.abs().amax(-1).transpose(0, 1)[..., None] * kk.abs().sum(-1)[:, None] * scale  # [nq, n, L]
    seen = torch.arange(L)[None] <= past + torch.arange(n)[:, None]
    s = s.masked_fill(~seen, -math.inf)
    mag = mag.masked_fill(~seen, 0.0)
    most = most.masked_fill(~seen, 0.0)
    p = torch.exp(s - s.amax(-1, keepdim=True).clamp(min=-1e300)) if L else s
    p = p / p.sum(-1, keepdim=True).clamp(min=1e-300)
    vs = torch.where(torch.arange(L)[None, :, None] < past + n, vv, 0.0) if L else vv
    out = torch.einsum("hnl,hld->nhd", p, vs)
    weight = torch.einsum("hnl,hld->nhd", p, vs.abs())
    top = torch.stack([(m.amax(-1) if L else torch.zeros(nq, n, dtype=torch.float64)).transpose(0, 1) for m in (mag, most)])
    return out, weight, top


def attention_tolerance(out, weight, top, D, L, dtype, p_step, codes=False):
    """|error| of an attention row computed from fp32 scores, with P rounded to `p_step` relative (0: kept in fp32).

    A score is D products added in fp32, scaled: off by at most (D + 4)·2^-24·Σ|q||k|·scale, and its exponential by as
    much relatively plus 4 steps of the exponential itself; numerator and denominator each carry that, the sums over L
    keys add L + 8 roundings (of positive terms: relative), and the result is rounded to its type.

    `codes`: bf16 queries over e4m3 pages, whose elements may be taken as the sum of two e4m3 numbers of a row scaled
    to [128, 256) by a power of two.  The first is off by at most half a step, 2^-5 of a power of two 2^p <= |q|; the
    remainder is a multiple of q's last bit, 2^(p - 7), and at most 2^(p - 4): four bits, exact unless that last bit
    lies below e4m3's least step 2^-9, where it is off by at most 2^-10, that is 2^-17 of the row's largest (>= 128).
    Its products with the key add up to at most 2^-17·max|q|·Σ|k|·scale."""
    rel = 2 * ((D + 4) * F32 * top[0] + 4 * F32 + (2.0**-17 * top[1] if codes else 0.0)) + 2 * (L + 8) * F32
    return HALF[dtype] * out.abs() + (rel[..., None] + p_step) * 1.01 * weight + 1e-30


def append(qkv, pools, table, q_start, kv_len, nq, *, cos=None, sin=None, positions=None, q_norm=None, k_norm=None,
           eps=1e-6):
    """The operator on CPU pools {"k": (pages, scale), "v": ...}: returns q in 64 bits with its error magnitudes, and
    per pool what a page must now hold: {(page, head, offset): (values, magnitudes)} of the new tokens, {(page, head):
    exponent}, and {(page, head): (old tokens, shift)} of the pages whose codes move."""
    nkv, ps, D = pools["k"][0].shape[1:]
    x = qkv.double().view(-1, nq + 2 * nkv, D)
    q, qm = torch.zeros(len(x), nq, D, dtype=torch.float64), torch.zeros(len(x), nq, D, dtype=torch.float64)
    new = {"k": {}, "v": {}}
    for b, (t0, n, past) in enumerate(spans(q_start, kv_len)):
        for s in range(n):
            t, j = t0 + s, past + s
            p = j if positions is None else int(positions[t])
            c, sn = (None, None) if cos is None else (cos[p], sin[p])
            q[t], qm[t] = rotate(x[t, :nq], q_norm, c, sn, eps)
            page = int(table[b][j // ps])
            ky, km = rotate(x[t, nq:nq + nkv], k_norm, c, sn, eps)
            for h in range(nkv):
                new["k"][page, h, j % ps] = (ky[h], km[h])
                new["v"][page, h, j % ps] = (x[t, nq + nkv + h], torch.zeros(D, dtype=torch.float64))
    exps, moves = {"k": {}, "v": {}}, {"k": {}, "v": {}}
    for key, (pages, scale) in pools.items():
        if scale is None:
            continue
        for b, (t0, n, past) in enumerate(spans(q_start, kv_len)):
            for i in range(past // ps, -(-(past + n) // ps)) if n else ():
                page, held = int(table[b][i]), max(0, past - i * ps)
                for h in range(nkv):
                    vals = [new[key][page, h, o][0] for o in range(ps) if (page, h, o) in new[key]]
                    a = torch.stack(vals)
                    e = least_exp(float(torch.where(a.isfinite(), a.abs(), 0.0).max()))
                    if held:
                        old = math.frexp(float(scale[page, h]))[1] - 1
                        if e > old:
                            moves[key][page, h] = (held, old - e)
                        e = max(e, old)
                    exps[key][page, h] = e
    return q, qm, new, exps, moves
