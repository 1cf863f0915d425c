"""The paged KV cache at its edges: calls right behind one another, and what the tolerances of the ordinary cases do
not reach.  Reference, tolerances and pools as in ``test_gpu_paged``."""
from __future__ import annotations

import threading

import pytest
import torch

from gpu_mesh_b200 import _lib, kernels
from tests import paged_ref as R
from tests.test_gpu_paged import BF16, DEV, E4M3, F32, P_STEP, Cache, check_append, dev32, starts, tables

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


def workspace_and_call(c, q, out, q_start, kv_len, max_new, between):
    """``kernels.paged_attention`` by the C ABI, with ``between()`` between the workspace's query and the call."""
    lib, table = _lib.lib(), c.table.to(DEV)
    ks, vs, e4m3 = c.k.stride(), c.v.stride(), c.cache == E4M3
    dt = {BF16: _lib.MG_DTYPE_BF16, F32: _lib.MG_DTYPE_F32}[c.dtype]
    pool = _lib.PagedPool(c.k.data_ptr(), c.v.data_ptr(), c.ks.data_ptr() if e4m3 else None, c.vs.data_ptr() if e4m3 else None,
                          *ks[:3], *vs[:3], c.ks.stride(0) if e4m3 else 0, c.vs.stride(0) if e4m3 else 0, c.pages, c.ps, c.nkv,
                          c.D, _lib.MG_DTYPE_E4M3 if e4m3 else dt)
    batch = _lib.PagedBatch(table.data_ptr(), q_start.data_ptr(), kv_len.data_ptr(), table.stride(0), len(c.table), len(q),
                            table.shape[1], max_new)
    need = lib.mg_paged_attention_workspace(pool, batch, dt, q.shape[1])
    ws = torch.empty(need, dtype=torch.uint8, device=DEV)
    between()
    args = _lib.PagedAttentionArgs(q.data_ptr(), out.data_ptr(), ws.data_ptr(), need, *q.stride()[:2], *out.stride()[:2], dt,
                                   q.shape[1], c.D**-0.5)
    _lib.check(lib.mg_paged_attention(pool, batch, args, torch.cuda.current_stream().cuda_stream))
    return need


@pytest.mark.parametrize("dtype,cache", [(BF16, BF16), (BF16, E4M3), (F32, F32)])
def test_workspace_does_not_follow_reserved_sms(dtype, cache):
    """SMs that are reserved, or given back, between the query of the workspace and the call."""
    lens, new = [3000, 1, 777, 200], [1, 1, 1, 90]
    c = Cache(lens, 2, 16, 64, dtype, cache)
    c.fill(lens)
    q = torch.randn(sum(new), 8, 64, generator=torch.Generator().manual_seed(1)).to(dtype).to(DEV)
    reserve = lambda n: _lib.check(_lib.lib().mg_reserve_sms(0, n))  # noqa: E731
    rows = {n: (q[:sum(n)], dev32(starts(n)), dev32(lens), max(n)) for n in ((1, 1, 1, 1), tuple(new))}
    pools, good, sizes = c.host(), {}, {}
    for n in rows:
        good[n] = []
        for b, (t0, m, past) in enumerate(R.spans(starts(n), lens)):
            x = q[t0:t0 + m].cpu().double()
            k, v = (R.dense(*pools[key], c.table[b], lens[b]) for key in ("k", "v"))
            ref, weight, top = R.attend(x, k, v, past, 64**-0.5)
            tol = R.attention_tolerance(ref, weight, top, 64, lens[b], dtype, P_STEP[dtype], cache == E4M3)
            if cache == E4M3:
                tol += half_floor(x, k, v, key_scales(c, pools["v"][1], b, lens[b]), past, 64**-0.5, 14 if 4 * m <= 16 else 7)
            good[n].append((ref, tol))

    def check(out, n):
        ref, tol = (torch.cat(x) for x in zip(*good[n]))
        assert ((out.cpu().double() - ref).abs() <= tol).all()

    try:
        for n, (x, s, m, most) in rows.items():
            sizes[n] = set()
            for before, after in ((0, 0), (70, 0), (0, 70), (70, 16)):
                reserve(before)
                out = torch.empty_like(x)
                sizes[n].add(workspace_and_call(c, x, out, s, m, most, lambda: reserve(after)))
                check(out, n)
        assert all(len(s) == 1 for s in sizes.values())
        # The wrapper, with another thread that changes the reservation all the time.
        stop = threading.Event()

        def toggle():
            i = 0
            while not stop.is_set():
                reserve((0, 70, 5)[i % 3])
                i += 1

        t = threading.Thread(target=toggle)
        t.start()
        try:
            got = [(n, kernels.paged_attention(x, c.k, c.v, c.table.to(DEV), s, m, max_new=most, **c.scales()))
                   for _ in range(100) for n, (x, s, m, most) in rows.items()]
        finally:
            stop.set()
            t.join()
        for n, out in got:
            check(out, n)
    finally:
        reserve(0)
    kernels.paged_check_device()


def fill_exponents(c, b, exps, g, zero=-100):
    """Sequence b's pages: random keys of one size, values whose pages have the scale 2^e (`zero`: a page of zeros)."""
    for i, e in enumerate(exps):
        p = int(c.table[b, i])
        k = torch.randn(c.nkv, c.ps, c.D, generator=g)
        ek = torch.tensor([float(R.least_exp(float(k[h].abs().max()))) for h in range(c.nkv)])
        c.ks[p] = torch.exp2(ek).to(DEV)
        c.k.view(torch.uint8)[p] = (k * torch.exp2(-ek)[:, None, None]).to(E4M3).view(torch.uint8).to(DEV)
        x = torch.zeros(c.nkv, c.ps, c.D) if e == zero else torch.randn(c.nkv, c.ps, c.D, generator=g)
        x *= 448.0 / x.abs().amax((1, 2), keepdim=True).clamp(min=1.0)
        c.vs[p] = 2.0**e
        c.v.view(torch.uint8)[p] = x.to(E4M3).view(torch.uint8).to(DEV)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("n", [1, 4, 40])
@pytest.mark.parametrize("big", [0, 8, 9, 30, 34, 41, 60, 100])
def test_softmax_sum_over_pages_of_all_scales(dtype, n, big):
    """Pages of zeros (scale 2^-100), of tiny and of huge values in one sequence, in every order, next to one another
    and so far apart that the run's parts are joined: a key weighs the same in the softmax whatever its values."""
    D, nkv, nq, ps = (64, 2, 8, 16) if n == 4 else (128, 1, 4, 32)
    g = torch.Generator().manual_seed(big + n)
    low = -100
    orders = [[low, big], [big, low], [low, big, -30, 0], [big] + [low] * 40, [low] * 40 + [big], [low] * 60 + [big] * 60,
              ([low] * 7 + [big] + [-8] * 5) * 9, [-30, low, big, low] * 3, [low] * 3]
    lens = [max(ps * len(o) - 5 * (i % 2), 1) for i, o in enumerate(orders)]
    c = Cache(lens, nkv, ps, D, dtype, E4M3, seed=big)
    for b, o in enumerate(orders):
        fill_exponents(c, b, o, g)
    for amp in (1e-3, 1.0):  # equal scores, ordinary ones
        new = [min(n, L) for L in lens]
        q = (torch.randn(sum(new), nq, D, generator=g) * amp).to(dtype)
        out = kernels.paged_attention(q.to(DEV), c.k, c.v, c.table.to(DEV), dev32(starts(new)), dev32(lens), max_new=n, **c.scales())
        kernels.paged_check_device()
        pools = c.host()
        for b, (t0, m, past) in enumerate(R.spans(starts(new), lens)):
            x = q[t0:t0 + m].double()
            k, v = (R.dense(*pools[key], c.table[b], lens[b]) for key in ("k", "v"))
            ref, weight, top = R.attend(x, k, v, past, D**-0.5)
            tol = R.attention_tolerance(ref, weight, top, D, lens[b], dtype, P_STEP[dtype], dtype == BF16)
            if dtype == BF16:
                tol += half_floor(x, k, v, key_scales(c, pools["v"][1], b, lens[b]), past, D**-0.5, 14 if 4 * m <= 16 else 7)
            err = (out[t0:t0 + m].cpu().double() - ref).abs()
            assert (err <= tol).all(), (b, amp, float((err / tol).max()))


@pytest.mark.parametrize("dtype,cache", [(BF16, BF16), (F32, F32)])
@pytest.mark.parametrize("D", [64, 128])
def test_keys_of_no_weight_before_broken_tokens(dtype, cache, D):
    """Infinite first keys whose scores are -inf (weight 0), while values of later tokens are NaN or infinite: the rows
    before those come out as if the first keys were not there."""
    new, lens = [4, 60, 3, 200, 1], [700, 90, 5000, 3000, 40]
    c = Cache(lens, 2, 16, D, dtype, cache, seed=D)
    c.fill(lens)
    g = torch.Generator().manual_seed(D)
    q = torch.randn(sum(new), 8, D, generator=g)
    q[..., 5] = q[..., 5].abs() + 0.1
    q = q.to(dtype)
    none = 3  # first keys without weight, fewer than any row sees
    for b, (n, L) in enumerate(zip(new, lens)):
        for j in range(none):
            c.k[int(c.table[b, 0]), :, j, 5] = -torch.inf
        if n > 1:
            p, o = int(c.table[b, (L - 1) // 16]), (L - 1) % 16
            c.v[p, 0, o, 3] = torch.nan
            c.v[p, 1, o, ::7] = torch.inf
    out = kernels.paged_attention(q.to(DEV), c.k, c.v, c.table.to(DEV), dev32(starts(new)), dev32(lens), **c.scales())
    kernels.paged_check_device()
    pools = c.host()
    for b, (t0, n, past) in enumerate(R.spans(starts(new), lens)):
        k, v = (R.dense(*pools[key], c.table[b], lens[b])[:, none:] for key in ("k", "v"))
        for s in range(n):
            seen = past + s + 1 - none
            ref, weight, top = R.attend(q[t0 + s:t0 + s + 1].double(), k[:, :seen], v[:, :seen], seen - 1, D**-0.5)
            tol = R.attention_tolerance(ref, weight, top, D, lens[b], dtype, P_STEP[dtype])
            x = out[t0 + s].cpu().double()
            fine = ref[0].isfinite()
            assert torch.equal(x.isnan(), ref[0].isnan()) and torch.equal(x.isinf(), ref[0].isinf()), (b, s)
            assert ((x - ref[0]).abs()[fine] <= tol[0][fine]).all(), (b, s)


@pytest.mark.parametrize("dtype,cache,D", [(F32, F32, 64), (F32, E4M3, 128), (BF16, BF16, 32), (BF16, E4M3, 16),
                                           (BF16, BF16, 64), (BF16, E4M3, 64), (BF16, BF16, 128), (BF16, E4M3, 128)])
@pytest.mark.parametrize("n", [1, 3, 40])
def test_broken_values_of_keys_without_weight(dtype, cache, D, n):
    """A NaN or an infinity in a value that a row sees reaches it however little its key weighs (0 times either is
    NaN), also where the key's part of the context holds no other weight."""
    lens, ps = [2500, 70], 16
    new = [n, n]
    c = Cache(lens, 2, ps, D, dtype, cache, seed=n)
    c.fill(lens, spread=0)
    q = torch.zeros(sum(new), 4, D, dtype=dtype)
    q[..., 0] = 64.0 * D**0.5
    for b, L in enumerate(lens):  # scores 64 times the first dim: 16 for the keys that count, -16 for the first tokens
        for j in range(L):
            at = (int(c.table[b, j // ps]), slice(None), j % ps)
            low = j < min(40, L - n)
            if cache == E4M3:
                c.k.view(torch.uint8)[at] = 0
                c.k.view(torch.uint8)[at[0], :, at[2], 0] = 0x48 | (0x80 if low else 0)  # 4.0
            else:
                c.k[at] = 0.0
                c.k[at[0], :, at[2], 0] = -4.0 if low else 4.0
        if cache == E4M3:
            c.ks[c.table[b][: -(-L // ps)].long().to(DEV)] = 1.0
        for h, d, x in ((0, 1, torch.nan), (1, 2, torch.inf)):
            if cache == E4M3:
                c.v.view(torch.uint8)[int(c.table[b, 0]), h, 7, d] = 0x7F
            else:
                c.v[int(c.table[b, 0]), h, 7, d] = x
    out = kernels.paged_attention(q.to(DEV), c.k, c.v, c.table.to(DEV), dev32(starts(new)), dev32(lens), **c.scales())
    kernels.paged_check_device()
    broken = torch.zeros(out.shape, dtype=torch.bool)
    broken[:, :2, 1] = True
    broken[:, 2:, 2] = True
    assert torch.equal(out.cpu().isfinite(), ~broken)


@pytest.mark.parametrize("dtype,cache", [(BF16, BF16), (BF16, E4M3), (F32, F32)])
@pytest.mark.parametrize("limit", [None, 4])
def test_bad_metadata_disturbs_no_other_sequence(dtype, cache, limit):
    """Lengths, row ranges and page ids that do not fit: the other sequences' rows, pages and scales come out as ever,
    and nothing is stored for what was left out.  A page id outside the pool leaves out its page alone."""
    few = limit is not None
    lens, new = [40, 20, 33, 10, 300], [2, 1, 4 if few else 33, 2, 3 if few else 50]
    nq, nkv, D, ps = 8, 2, 64, 16
    g = torch.Generator().manual_seed(3)
    q = torch.randn(sum(new), nq, D, generator=g).to(dtype)
    qkv = torch.randn(sum(new), (nq + 2 * nkv) * D, generator=g).to(dtype).to(DEV)

    def cache_of():
        c = Cache(lens, nkv, ps, D, dtype, cache)
        c.fill(lens)  # the attention's own tokens; the append writes over them
        return c

    def run_append(q_start, n, table, wrong):
        c = cache_of()
        out = torch.full((sum(new), nq, D), 7.0, dtype=dtype, device=DEV)
        kernels.paged_append(qkv, c.k, c.v, table.to(DEV), dev32(q_start), dev32(n), num_q_heads=nq, max_new=limit, out=out,
                             **c.scales())
        if wrong:
            with pytest.raises(_lib.DeviceRangeError, match="page id, length"):
                kernels.paged_check_device()
        kernels.paged_check_device()
        return c, out

    bits = lambda t: t.cpu().contiguous().view(torch.int8)  # noqa: E731
    c = cache_of()
    cap = c.cols * ps
    good, good_q = run_append(starts(new), lens, c.table, False)
    at = starts(new)
    cases = [(at, [40, cap + 1, 33, 10, 300], 1, None), (at, [40, -1, 33, 10, 300], 1, None),
             (at[:4] + [2000] + at[5:], lens, 3, None)]  # (sequence 4 then begins at 2000 too: left out as well)
    cases += [(at, lens, b, wrong) for b in (0, 4) for wrong in (-1, c.pages, 2**31 - 1, -(2**31))]
    pools = c.host()
    for q_start, n, b, wrong in cases:
        table, last = c.table.clone(), (lens[b] - 1) // ps
        if wrong is not None:
            table[b, last] = wrong
        bad = [i for i in range(len(lens)) if i == b or (q_start[i] != at[i])]
        out = torch.full_like(q, 7.0).to(DEV)
        kernels.paged_attention(q.to(DEV), c.k, c.v, table.to(DEV), dev32(q_start), dev32(n), max_new=limit, out=out, **c.scales())
        with pytest.raises(_lib.DeviceRangeError, match="page id, length"):
            kernels.paged_check_device()
        after, after_q = run_append(q_start, n, table, True)
        skipped = torch.zeros(c.pages, dtype=torch.bool)
        for i, (t0, m, past) in enumerate(R.spans(at, lens)):
            rows = slice(t0, t0 + m)
            if i in bad:
                if wrong is None:
                    assert (out[rows] == 7.0).all() and (after_q[rows] == 7.0).all()
                    skipped[c.table[i][past // ps: (lens[i] - 1) // ps + 1].long()] = True
                else:
                    assert torch.equal(after_q[rows], good_q[rows])
                    skipped[int(c.table[i, last])] = True
                continue
            assert torch.equal(after_q[rows], good_q[rows])
            k, v = (R.dense(*pools[key], c.table[i], lens[i]) for key in ("k", "v"))
            ref, weight, top = R.attend(q[rows].double(), k, v, past, D**-0.5)
            tol = R.attention_tolerance(ref, weight, top, D, lens[i], dtype, P_STEP[dtype], cache == E4M3 and dtype == BF16)
            if cache == E4M3:
                tol += half_floor(q[rows].double(), k, v, key_scales(c, pools["v"][1], i, lens[i]), past, D**-0.5,
                                  14 if 4 * m <= 16 else 7)
            assert ((out[rows].cpu().double() - ref).abs() <= tol).all(), (b, wrong, i)
        for x, y, start in ((after.k, good.k, c.k), (after.v, good.v, c.v), (after.ks, good.ks, c.ks), (after.vs, good.vs, c.vs)):
            if x is not None:
                assert torch.equal(bits(x[(~skipped).to(DEV)]), bits(y[(~skipped).to(DEV)]))
                assert torch.equal(bits(x[skipped.to(DEV)]), bits(start[skipped.to(DEV)]))


@pytest.mark.parametrize("cache", [BF16, E4M3])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("n", [1, 2, 4])
def test_precision_with_few_query_rows(cache, D, n):
    """Up to 16 query rows per KV head the queries stay exact and the weights are a bf16 and its remainder (each off by
    half a step: 2^-16 together) or a half (2^-11).  Neighbouring keys are nearly alike and their values of opposite
    sign, so that outputs are small beside sum(p|v|) and the output's own rounding hides nothing: weights rounded to
    bf16 alone would not pass."""
    nq, nkv, ps = 8, 2, 16
    lens, g = [24, 40, 12, 300, 64, 1000], torch.Generator().manual_seed(D + n)
    c = Cache(lens, nkv, ps, D, BF16, cache, seed=n)
    for b, L in enumerate(lens):
        k, v = (torch.randn(nkv, L, D, generator=g).clamp(-6, 6) for _ in range(2))
        k[:, 1::2] = k[:, ::2] + 0.02 * torch.randn(nkv, L // 2, D, generator=g)
        v[:, 1::2] = -v[:, ::2]
        for x, pages, scale in ((k, c.k, c.ks), (v, c.v, c.vs)):
            for i in range(-(-L // ps)):
                p, y = int(c.table[b, i]), x[:, i * ps:(i + 1) * ps]
                if cache == E4M3:
                    scale[p] = 2.0**-6
                    pages.view(torch.uint8)[p, :, :y.shape[1]] = (y * 64.0).to(E4M3).view(torch.uint8).to(DEV)
                else:
                    pages[p, :, :y.shape[1]] = y.to(BF16).to(DEV)
    new = [n] * len(lens)
    q = (torch.randn(sum(new), nq, D, generator=g) * torch.tensor([0.3, 1.0, 3.0, 0.3] * 2)[:nq, None]).to(BF16)
    out = kernels.paged_attention(q.to(DEV), c.k, c.v, c.table.to(DEV), dev32(starts(new)), dev32(lens), max_new=n, **c.scales())
    kernels.paged_check_device()
    pools, coarse = c.host(), 0
    for b, (t0, _, past) in enumerate(R.spans(starts(new), lens)):
        x = q[t0:t0 + n].double()
        k, v = (R.dense(*pools[key], c.table[b], lens[b]) for key in ("k", "v"))
        ref, weight, top = R.attend(x, k, v, past, D**-0.5)
        tol = R.attention_tolerance(ref, weight, top, D, lens[b], BF16, 2.0**-16 if cache == BF16 else 2.0**-11)
        if cache == E4M3:
            # The exponent carries V's -6 and 14 beside the score: two roundings of it more, in every weight and the sum.
            tol += half_floor(x, k, v, key_scales(c, pools["v"][1], b, lens[b]), past, D**-0.5, 14) + 4 * R.F32 * 20 * weight
        assert ((out[t0:t0 + n].cpu().double() - ref).abs() <= tol).all(), (b, lens[b])
        s = torch.einsum("nhd,hld->hnl", x, k.repeat_interleave(nq // nkv, 0)) * D**-0.5
        s = s.masked_fill(torch.arange(lens[b])[None] > past + torch.arange(n)[:, None], -torch.inf)
        p = torch.exp(s - s.amax(-1, keepdim=True))
        rough = torch.einsum("hnl,hld->nhd", p.to(BF16).double() / p.sum(-1, keepdim=True), v.repeat_interleave(nq // nkv, 0))
        coarse += int(((rough - ref).abs() > tol).sum())
    assert coarse > 0  # the tolerance tells a coarser P apart
