"""The paged KV cache at its edges: calls right behind one another, and what the tolerances of the ordinary cases do
not reach.  Reference, tolerances and pools as in ``test_gpu_paged``."""
from __future__ import annotations

import pytest
import torch

from gpu_mesh_b200 import kernels
from tests import paged_ref as R
from tests.test_gpu_paged import BF16, DEV, E4M3, P_STEP, Cache, check_append, dev32, starts, tables

pytestmark = pytest.mark.gpu


def key_scales(c, scale, b, length):
    """[heads, length] in 64 bits: the scale of each cached token's page."""
    return scale[c.table[b][torch.arange(length) // c.ps].long()].double().T


def half_floor(q, k, v, vscale, past, scale, offset):
    """What weights in half lose besides their relative rounding, where the queries are bf16 and the pages e4m3.

    Key j's code is weighed by P_j = 2^(s_j + e_j - m + offset) with 2^e its page's scale and m at most the largest
    s + e of the row (offset: 14 for up to 16 query rows per KV head, else 7).  A half is a multiple of 2^-24, so P_j
    is off by at most 2^-25 where that exceeds its relative rounding, and the output, sum(P code) / (2^offset
    sum(2^(s - m))), by at most 2^(-25 - offset) sum|code| 2^m / sum(2^s).  As 2^m / sum(2^s) is at most the largest
    p_j 2^(e_j) of the row with p its softmax, that is 2^(-25 - offset) sum|code| max(p 2^e), over the keys it sees."""
    n, nq, _ = q.shape
    G, L = nq // k.shape[0], k.shape[1]
    s = torch.einsum("nhd,hld->hnl", q, k.repeat_interleave(G, 0)) * scale
    seen = torch.arange(L)[None] <= past + torch.arange(n)[:, None]
    p = torch.softmax(s.masked_fill(~seen, -torch.inf), -1).nan_to_num(0.0)
    most = (p * vscale.repeat_interleave(G, 0)[:, None]).amax(-1)  # [nq, n]
    codes = torch.einsum("nl,hld->hnd", seen.double(), (v.abs() / vscale[..., None]).nan_to_num(0.0, 0.0, 0.0))
    return 2.0**(-25 - offset) * (codes.repeat_interleave(G, 0) * most[..., None]).transpose(0, 1)


@pytest.mark.parametrize("nkv", [1, 2])
@pytest.mark.parametrize("n", [1, 4, 9])
def test_attention_directly_behind_an_append(nkv, n):
    """Steps whose values grow, so that every append changes scales (of several pages to a memory sector) and codes,
    with the attention that reads them enqueued behind it and the host looking only afterwards."""
    nq, D, ps, steps = 4 * nkv, 64, 16, 6
    past = [(11 * i) % 37 for i in range(60)]
    c = Cache([p + steps * n for p in past], nkv, ps, D, BF16, E4M3)
    c.fill(past, spread=6)
    cos, sin = (t.to(DEV) for t in tables(D))
    table = c.table.to(DEV)
    new = [n] * len(past)
    q_start = dev32(starts(new))
    g = torch.Generator().manual_seed(n)
    for i in range(steps):
        lens = [p + (i + 1) * n for p in past]
        qkv = torch.randn(sum(new), (nq + 2 * nkv) * D, generator=g) * 2.0**(i - 2)
        qkv[:, :nq * D] *= 2.0**(-2 * i)  # the scores stay of one size
        qkv = qkv.to(BF16)
        x, kv_len = qkv.to(DEV), dev32(lens)
        before = c.host()
        torch.cuda.synchronize()
        q = kernels.paged_append(x, c.k, c.v, table, q_start, kv_len, num_q_heads=nq, max_new=n, cos=cos, sin=sin, **c.scales())
        out = kernels.paged_attention(q, c.k, c.v, table, q_start, kv_len, max_new=n, **c.scales())
        kernels.paged_check_device()
        pools = c.host()
        check_append(c, before, pools, q, R.append(qkv, before, c.table, starts(new), lens, nq, cos=cos.cpu(), sin=sin.cpu()),
                     BF16, D)
        for b, (t0, _, gone) in enumerate(R.spans(starts(new), lens)):
            k, v = (R.dense(*pools[key], c.table[b], lens[b]) for key in ("k", "v"))
            ref, weight, top = R.attend(q[t0:t0 + n].cpu().double(), k, v, gone, D**-0.5)
            tol = R.attention_tolerance(ref, weight, top, D, lens[b], BF16, P_STEP[BF16], True)
            tol += half_floor(q[t0:t0 + n].cpu().double(), k, v, key_scales(c, pools["v"][1], b, lens[b]), gone, D**-0.5,
                              14 if n * nq // nkv <= 16 else 7)
            assert ((out[t0:t0 + n].cpu().double() - ref).abs() <= tol).all(), (i, b)
