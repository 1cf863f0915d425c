"""The paged KV cache on the GPU against a 64-bit token-by-token reference: append and attention.

Tolerances count the roundings of each path and are set before a run (``paged_ref.attention_tolerance``; for the
append see ``check_append``)."""
from __future__ import annotations

import math

import pytest
import torch

from gpu_mesh_b200 import _lib, kernels
from tests import paged_ref as R

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda", 0)
BF16, F32, E4M3 = torch.bfloat16, torch.float32, torch.float8_e4m3fn
P_STEP = {BF16: 2.0**-8, F32: 0.0}  # the coarsest rounding of P of any kernel of a type


def tables(D, n=4096, theta=10000.0):
    inv = theta ** (-torch.arange(0, D, 2, dtype=torch.float64) / D)
    a = torch.arange(n, dtype=torch.float64)[:, None] * inv
    return a.cos().float(), a.sin().float()


class Cache:
    """A pool on the GPU with junk in every byte that no sequence has written, and its page tables."""

    def __init__(self, lens, nkv, ps, D, dtype, cache, *, seed=0, spare=3, layout="dense", poison=True):
        self.g = torch.Generator().manual_seed(seed)
        self.nkv, self.ps, self.D, self.dtype, self.cache = nkv, ps, D, dtype, cache
        need = [-(-n // ps) for n in lens]
        self.pages = sum(need) + spare
        self.cols = max(need + [1]) + 1
        perm = torch.randperm(self.pages, generator=self.g).to(torch.int32)
        self.table = torch.full((len(lens), self.cols), -7, dtype=torch.int32)
        at = 0
        for b, n in enumerate(need):
            self.table[b, :n] = perm[at:at + n]
            at += n
        shape = (self.pages, nkv, ps, D)
        junk = float("nan") if poison else 0.0
        if layout == "dense":
            k, v = torch.full(shape, junk), torch.full(shape, junk)
            k, v = k.to(cache).to(DEV), v.to(cache).to(DEV)
        elif layout == "interleaved":  # [pages, 2, heads, page, D]
            both = torch.full((self.pages, 2, nkv, ps, D), junk).to(cache).to(DEV)
            k, v = both[:, 0], both[:, 1]
        elif layout == "tokens":  # [pages, page, heads, D]
            k, v = (torch.full((self.pages, ps, nkv, D), junk).to(cache).to(DEV).transpose(1, 2) for _ in range(2))
        else:  # one layer of [layers, pages, ...], K and V with different strides
            k = torch.full((3, *shape), junk).to(cache).to(DEV)[1]
            v = torch.full((self.pages, 3, nkv, ps, D), junk).to(cache).to(DEV)[:, 2]
        self.k, self.v = k, v
        self.ks = self.vs = None
        if cache == E4M3:
            self.ks = torch.full((self.pages, nkv), float("nan"), device=DEV)
            self.vs = torch.full((self.pages, nkv + 3), float("nan"), device=DEV)[:, :nkv]

    def fill(self, lens, spread=2):
        """Every sequence's first `lens` tokens: random keys and values, heads and pages of different sizes."""
        for pages, scale in ((self.k, self.ks), (self.v, self.vs)):
            for b, n in enumerate(lens):
                for i in range(-(-n // self.ps)):
                    p, m = int(self.table[b, i]), min(self.ps, n - i * self.ps)
                    x = torch.randn(self.nkv, m, self.D, generator=self.g)
                    x *= 2.0 ** torch.randint(-spread, spread + 1, (self.nkv, 1, 1), generator=self.g)
                    if scale is not None:
                        e = torch.tensor([R.least_exp(float(x[h].abs().max())) for h in range(self.nkv)])
                        scale[p] = torch.exp2(e.float()).to(DEV)
                        codes = (x * torch.exp2(-e.float())[:, None, None]).to(E4M3)
                        pages.view(torch.uint8)[p, :, :m] = codes.view(torch.uint8).to(DEV)
                    else:
                        pages[p, :, :m] = x.to(self.dtype).to(DEV)

    def host(self):
        return {"k": (self.k.cpu(), None if self.ks is None else self.ks.cpu()),
                "v": (self.v.cpu(), None if self.vs is None else self.vs.cpu())}

    def scales(self):
        return {"k_scale": self.ks, "v_scale": self.vs}


def starts(new):
    return [0] + torch.tensor(new).cumsum(0).tolist() if new else [0]


def dev32(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


def check_append(c, before, after, q, ref, dtype, D):
    """q and native pages: one rounding of an fp32 result whose own error is at most (D + 16) fp32 steps of
    |x1 c| + |x2 s| (the norm's sum of D squares, its root, quotient and products, the rotation's two products and
    sum).  Codes: half a step of e4m3 (2^-4 relative, 2^-10 of the scale below the normal range) more.  Moved codes:
    exact, but for codes that reach the subnormals (half of their step).  Scales: exact, unless the largest magnitude
    lies within its fp32 error of a border."""
    rq, qm, new, exps, moves = ref
    slack = (D + 16) * R.F32
    err = (q.double().cpu() - rq).abs()
    assert (err <= R.HALF[dtype] * rq.abs() + slack * qm + 1e-30).all(), float(err.max())
    for key in ("k", "v"):
        pages, scale = after[key]
        old_pages, old_scale = before[key]
        touched = torch.zeros(pages.shape[:3], dtype=torch.bool)
        values = pages.float().double() if pages.dtype == E4M3 else pages.double()
        for (p, h, o), (x, m) in new[key].items():
            touched[p, h, o] = True
            got = values[p, h, o]
            if scale is None:
                tol = R.HALF[dtype] * x.abs() + slack * m + 1e-30
            else:
                s = float(scale[p, h])
                got = got * s
                x = torch.where(x.abs() > 448.0 * s * (1 + slack), x.sign() * 448.0 * s, x)  # saturates
                tol = 2.0**-4 * x.abs() * (1 + 2.0**-10) + 2.0**-10 * s + slack * m
            assert torch.equal(got.isnan(), x.isnan())
            assert ((got - x).abs()[~x.isnan()] <= tol[~x.isnan()]).all(), (key, p, h, o)
        if scale is None:
            assert torch.equal(pages[~touched].view(torch.int8), old_pages[~touched].view(torch.int8))
            continue
        for (p, h), e in exps[key].items():
            assert float(scale[p, h]) == 2.0**e, (key, p, h, float(scale[p, h]), e)
        for (p, h), (held, shift) in moves[key].items():
            touched[p, h, :held] = True
            want = old_pages[p, h, :held].float().double() * 2.0**shift
            assert ((values[p, h, :held] - want).abs() <= 2.0**-10).all()
            normal = want.abs() >= 2.0**-6
            assert torch.equal(values[p, h, :held][normal], want[normal])
        assert torch.equal(pages.view(torch.uint8)[~touched], old_pages.view(torch.uint8)[~touched])
        rest = torch.ones_like(scale, dtype=torch.bool)
        for p, h in exps[key]:
            rest[p, h] = False
        assert torch.equal(scale[rest].view(torch.int32), old_scale[rest].view(torch.int32))


def run_append(c, new, lens, nq, *, norm=False, rope=True, positions=None, seed=1, scale_x=1.0, qkv=None, extra=0,
               max_new=None):
    g = torch.Generator().manual_seed(seed)
    width = (nq + 2 * c.nkv) * c.D
    T = sum(new) + extra
    if qkv is None:
        qkv = (torch.randn(T, width, generator=g) * scale_x).to(c.dtype)
    cos, sin = tables(c.D) if rope else (None, None)
    w = [(1 + 0.3 * torch.randn(c.D, generator=g)).to(c.dtype) if norm else None for _ in range(2)]
    before = c.host()
    ref = R.append(qkv[:sum(new)], before, c.table, starts(new), lens, nq, cos=cos, sin=sin, positions=positions,
                   q_norm=w[0], k_norm=w[1], eps=1e-6)
    out = torch.full((T, nq, c.D), 7.0, dtype=c.dtype, device=DEV)
    to = lambda t: None if t is None else t.to(DEV)  # noqa: E731
    got = kernels.paged_append(
        qkv.to(DEV), c.k, c.v, c.table.to(DEV), dev32(starts(new)), dev32(lens), num_q_heads=nq, max_new=max_new,
        cos=to(cos), sin=to(sin), positions=to(positions), q_norm=to(w[0]), k_norm=to(w[1]), out=out, **c.scales())
    assert got is out
    kernels.paged_check_device()
    assert (out[sum(new):] == 7.0).all()
    check_append(c, before, c.host(), out[:sum(new)], ref, c.dtype, c.D)


SHAPES = [(8, 2, 1, 16), (16, 6, 2, 16), (32, 4, 4, 32), (64, 8, 1, 16), (64, 14, 2, 64), (128, 8, 2, 128),
          (128, 5, 5, 32), (128, 32, 8, 64)]  # D, query heads, KV heads, page


@pytest.mark.parametrize("D,nq,nkv,ps", SHAPES)
@pytest.mark.parametrize("dtype,cache", [(BF16, BF16), (BF16, E4M3), (F32, F32), (F32, E4M3)])
@pytest.mark.parametrize("norm", [False, True])
def test_append(D, nq, nkv, ps, dtype, cache, norm):
    new = [1, 0, ps, 3, 2 * ps + 5, 1, 1, 7]
    past = [0, 5, 0, ps - 2, ps + 3, ps - 1, ps, 2 * ps - 3]
    lens = [p + n for p, n in zip(past, new)]
    c = Cache(lens, nkv, ps, D, dtype, cache, seed=D + nq)
    c.fill(past)
    run_append(c, new, lens, nq, norm=norm, extra=2)


@pytest.mark.parametrize("dtype,cache", [(BF16, BF16), (BF16, E4M3), (F32, F32), (F32, E4M3)])
@pytest.mark.parametrize("limit", [1, 8, None])
def test_append_few_tokens(dtype, cache, limit):
    """Single tokens and up to eight: the host's bound chooses the kernel, the results are the same."""
    new = [1, 1, 0, 1, 1] if limit == 1 else [8, 1, 3, 0, 5, 8]
    past = [15, 0, 3, 16, 40, 11][:len(new)]
    lens = [p + n for p, n in zip(past, new)]
    c = Cache(lens, 8, 16, 128, dtype, cache)
    c.fill(past, spread=9)  # some pages hold far smaller values: their scales grow
    run_append(c, new, lens, 8, max_new=limit, norm=True)


def test_append_grows_scales_token_by_token():
    """Twenty calls of one token, each larger than the last: every call moves the page's codes."""
    c = Cache([32, 20], 2, 32, 64, BF16, E4M3)
    for i in range(20):
        run_append(c, [1, 1], [i + 1, i + 1], 4, seed=i, scale_x=2.0 ** (i - 10))


def test_append_special_values():
    """Zeros, infinities, NaN, the largest and smallest values: scales follow the finite ones."""
    new, lens = [4, 2], [4, 20]
    for dtype in (BF16, F32):
        for big in (1.0, torch.finfo(dtype).max, 2.0**-120):
            c = Cache(lens, 2, 16, 32, dtype, E4M3)
            c.fill([0, 18])
            g = torch.Generator().manual_seed(3)
            qkv = (torch.rand(6, 6 * 32, generator=g) * big).to(dtype)
            qkv[0, 64:] = 0.0                       # a token of zeros
            qkv[1, 2 * 32 + 5] = math.inf           # key, value: infinities and NaN
            qkv[2, 4 * 32 + 9] = -math.inf
            qkv[3, 5 * 32 + 1] = math.nan
            run_append(c, new, lens, 2, rope=False, qkv=qkv)


def test_append_positions():
    """Explicit positions: far ones, repeated ones, one clamped and reported."""
    new, lens = [5, 1], [25, 3]
    c = Cache(lens, 2, 16, 64, BF16, BF16)
    c.fill([20, 2])
    run_append(c, new, lens, 4, positions=torch.tensor([4095, 0, 17, 17, 1000, 3]))
    cos, sin = (t.to(DEV) for t in tables(64, 8))
    qkv = torch.randn(6, 8 * 64, device=DEV).to(BF16)
    args = (c.k, c.v, c.table.to(DEV), dev32([0, 5, 6]), dev32(lens))
    a = kernels.paged_append(qkv, *args, num_q_heads=4, cos=cos, sin=sin,
                             positions=torch.tensor([0, 8, 7, -1, 3, 7], device=DEV))
    with pytest.raises(_lib.DeviceRangeError, match="position"):
        kernels.paged_check_device()
    b = kernels.paged_append(qkv, *args, num_q_heads=4, cos=cos, sin=sin,
                             positions=torch.tensor([0, 7, 7, 0, 3, 7], device=DEV))
    kernels.paged_check_device()
    assert torch.equal(a, b)


@pytest.mark.parametrize("layout", ["interleaved", "tokens", "layers"])
@pytest.mark.parametrize("cache", [BF16, E4M3])
def test_append_layouts(layout, cache):
    new, lens = [3, 40, 1], [30, 40, 17]
    c = Cache(lens, 4, 32, 64, BF16, cache, layout=layout)
    c.fill([27, 0, 16])
    run_append(c, new, lens, 8)


def attend(c, new, lens, nq, *, dtype=None, scale=None, seed=5, amp=1.0, extra=0, max_new=None, check=True):
    dtype = c.dtype if dtype is None else dtype
    g = torch.Generator().manual_seed(seed)
    T = sum(new) + extra
    q = (torch.randn(T, nq, c.D, generator=g) * amp).to(dtype)
    out = torch.full((T, nq, c.D), 7.0, dtype=dtype, device=DEV)
    got = kernels.paged_attention(q.to(DEV), c.k, c.v, c.table.to(DEV), dev32(starts(new)), dev32(lens),
                                  max_new=max_new, scale=scale, out=out, **c.scales())
    assert got is out
    kernels.paged_check_device()
    assert (out[sum(new):] == 7.0).all()
    if not check:
        return out
    pools = c.host()
    for b, (t0, n, past) in enumerate(R.spans(starts(new), lens)):
        if not n:
            continue
        k, v = (R.dense(*pools[key], c.table[b], lens[b]) for key in ("k", "v"))
        ref, weight, top = R.attend(q[t0:t0 + n].double(), k, v, past, c.D ** -0.5 if scale is None else scale)
        tol = R.attention_tolerance(ref, weight, top, c.D, max(1, lens[b]), dtype, P_STEP[dtype],
                                    c.cache == E4M3 and dtype == BF16)
        err = (out[t0:t0 + n].cpu().double() - ref).abs()
        assert (err <= tol).all(), (b, n, lens[b], float((err / tol).max()))
    return out


RAGGED = [
    ([1, 1, 1, 1, 1, 1], [1, 2, 15, 16, 17, 300]),       # single tokens
    ([1, 0, 3, 1, 2, 4], [1, 9, 3, 129, 257, 700]),      # a few together, one sequence with none
    ([40, 1, 0, 129, 7, 64], [40, 5, 0, 400, 7, 65]),    # prompts and chunks beside single tokens
]


@pytest.mark.parametrize("D,nq,nkv,ps", SHAPES)
@pytest.mark.parametrize("dtype,cache", [(BF16, BF16), (BF16, E4M3), (F32, F32), (F32, E4M3)])
@pytest.mark.parametrize("case", range(len(RAGGED)))
def test_attention(D, nq, nkv, ps, dtype, cache, case):
    new, lens = RAGGED[case]
    c = Cache(lens, nkv, ps, D, dtype, cache, seed=D + nq + case)
    c.fill(lens)
    attend(c, new, lens, nq, extra=3, max_new=max(new))


@pytest.mark.parametrize("dtype,cache", [(BF16, BF16), (BF16, E4M3), (F32, F32), (F32, E4M3)])
@pytest.mark.parametrize("G", [1, 2, 3, 5, 7, 8, 9, 16])
def test_attention_groups(dtype, cache, G):
    new, lens = [1, 2, 1, 33], [200, 131, 16, 90]
    for D in (64, 128):
        c = Cache(lens, 2, 32, D, dtype, cache, seed=G)
        c.fill(lens)
        attend(c, new, lens, 2 * G)
        attend(c, [1, 1, 1, 1], lens, 2 * G, max_new=1)


@pytest.mark.parametrize("cache", [BF16, E4M3])
@pytest.mark.parametrize("D", [64, 128])
def test_attention_long_and_many(cache, D):
    """Sequences of several thousand tokens beside short ones; more sequences than SMs."""
    lens = [5000, 1, 3001, 128, 4097]
    c = Cache(lens, 4, 64, D, BF16, cache)
    c.fill(lens)
    attend(c, [1] * 5, lens, 16, max_new=1)
    attend(c, [3, 1, 200, 2, 4], lens, 16)
    lens = [(37 * i) % 211 + 1 for i in range(300)]
    c = Cache(lens, 2, 16, D, BF16, cache)
    c.fill(lens)
    attend(c, [1] * 300, lens, 8, max_new=1)
    attend(c, [min(n, 1 + i % 5) for i, n in enumerate(lens)], lens, 8)


@pytest.mark.parametrize("dtype,cache", [(BF16, BF16), (BF16, E4M3), (F32, F32), (F32, E4M3)])
def test_attention_rows_without_keys(dtype, cache):
    """More new tokens than cached ones: the first rows see nothing and give 0."""
    for new, lens in (([1, 1], [0, 0]), ([3, 1, 5], [2, 0, 5]), ([40, 64], [10, 0])):
        c = Cache(lens, 2, 16, 64, dtype, cache)
        c.fill(lens)
        out = attend(c, new, lens, 8)
        for t0, n, past in R.spans(starts(new), lens):
            assert (out[t0:t0 + min(n, max(0, -past))] == 0).all()


@pytest.mark.parametrize("dtype,cache", [(BF16, BF16), (BF16, E4M3), (F32, E4M3)])
@pytest.mark.parametrize("n", [1, 3, 40])
def test_attention_sharp_and_flat(dtype, cache, n):
    """Large scores (one key takes all), nearly equal ones, and pages whose sizes differ by 2^24."""
    lens = [333, 64, 150]
    for amp, scale in ((30.0, None), (1e-3, None), (1.0, 3.0)):
        c = Cache(lens, 2, 32, 128, dtype, cache)
        c.fill(lens, spread=2)
        attend(c, [n] * 3, lens, 8, amp=amp, scale=scale)
    c = Cache(lens, 2, 32, 64, dtype, cache)
    c.fill(lens, spread=12)
    attend(c, [n] * 3, lens, 8, amp=2.0**-10)


@pytest.mark.parametrize("layout", ["interleaved", "tokens", "layers"])
@pytest.mark.parametrize("cache", [BF16, E4M3])
def test_attention_layouts(layout, cache):
    lens = [100, 33, 260]
    for D in (32, 64, 128):
        c = Cache(lens, 4, 32, D, BF16, cache, layout=layout)
        c.fill(lens)
        attend(c, [1, 1, 1], lens, 8, max_new=1)
        attend(c, [50, 2, 140], lens, 8)


@pytest.mark.parametrize("dtype,cache", [(BF16, BF16), (BF16, E4M3), (F32, E4M3)])
def test_attention_strided_queries(dtype, cache):
    """Queries and outputs inside wider rows, heads in front of tokens, and of one head."""
    lens, new = [50, 7], [2, 7]
    c = Cache(lens, 2, 16, 64, dtype, cache)
    c.fill(lens)
    plain = attend(c, new, lens, 4)
    g = torch.Generator().manual_seed(5)
    q = torch.randn(9, 4, 64, generator=g).to(dtype).to(DEV)
    for make in (lambda: torch.zeros(9, 12, 64, dtype=dtype, device=DEV)[:, 5:9],
                 lambda: torch.zeros(4, 9, 64, dtype=dtype, device=DEV).transpose(0, 1),
                 lambda: torch.zeros(9, 4, 128, dtype=dtype, device=DEV)[..., :64]):
        qs, out = make(), make()
        qs.copy_(q)
        kernels.paged_attention(qs, c.k, c.v, c.table.to(DEV), dev32(starts(new)), dev32(lens), out=out, **c.scales())
        assert torch.equal(out, plain)


@pytest.mark.parametrize("cache", [BF16, E4M3])
def test_bad_metadata_is_left_out_and_reported(cache):
    """Lengths, row ranges and page ids that do not fit: those sequences are left out, the others are not disturbed."""
    lens, new = [40, 20, 33, 10], [2, 1, 33, 2]
    c = Cache(lens, 2, 16, 64, BF16, cache)
    c.fill([p - n for p, n in zip(lens, new)])
    q = torch.randn(38, 8, 64, device=DEV).to(BF16)
    qkv = torch.randn(38, 12 * 64, device=DEV).to(BF16)
    c2 = Cache(lens, 2, 16, 64, BF16, cache)
    cap = c.cols * 16
    bad = [
        (starts(new), [40, cap + 1, 33, 10], c.table, 1, None),     # longer than the table
        (starts(new), [40, -1, 33, 10], c.table, 1, None),          # negative length
        (starts(new), lens, c.table, 2, 32),                        # more new tokens than the bound
        ([0, 2, 3, 36, 2000], lens, c.table, 3, None),              # rows outside the batch
        ([0, 2, 3, 36, 30], lens, c.table, 3, None),                # rows that run backwards
    ]
    for q_start, n, table, b, limit in bad:
        out = torch.full_like(q, 7.0)
        kernels.paged_attention(q, c.k, c.v, table.to(DEV), dev32(q_start), dev32(n), out=out, max_new=limit, **c.scales())
        with pytest.raises(_lib.DeviceRangeError, match="page id, length"):
            kernels.paged_check_device()
        kernels.paged_check_device()  # cleared
        lo, hi = starts(new)[b], starts(new)[b + 1]
        assert (out[lo:hi] == 7.0).all()
        before = c.host()
        kernels.paged_append(qkv, c.k, c.v, table.to(DEV), dev32(q_start), dev32(n), num_q_heads=8, max_new=limit, **c.scales())
        with pytest.raises(_lib.DeviceRangeError):
            kernels.paged_check_device()
        after = c.host()
        pages = [int(p) for p in table[b] if p >= 0]
        for key in ("k", "v"):
            assert torch.equal(before[key][0][pages].view(torch.int8), after[key][0][pages].view(torch.int8))
    for wrong in (-1, c.pages, 2**31 - 1, -(2**31)):
        table = c.table.clone()
        table[0, 2] = wrong  # the page that sequence 0 appends to
        kernels.paged_append(qkv, c.k, c.v, table.to(DEV), dev32(starts(new)), dev32(lens), num_q_heads=8, **c.scales())
        with pytest.raises(_lib.DeviceRangeError):
            kernels.paged_check_device()
        kernels.paged_attention(q, c.k, c.v, table.to(DEV), dev32(starts(new)), dev32(lens), **c.scales())
        with pytest.raises(_lib.DeviceRangeError):
            kernels.paged_check_device()
    del c2


def test_python_refusals():
    c = Cache([20], 2, 16, 64, BF16, E4M3)
    q, qkv = torch.zeros(1, 8, 64, dtype=BF16, device=DEV), torch.zeros(1, 12 * 64, dtype=BF16, device=DEV)
    t, s, n = c.table.to(DEV), dev32([0, 1]), dev32([20])

    def att(q=q, k=c.k, v=c.v, t=t, s=s, n=n, ks=c.ks, vs=c.vs, **kw):
        kernels.paged_attention(q, k, v, t, s, n, k_scale=ks, v_scale=vs, **kw)

    def app(x=qkv, k=c.k, v=c.v, t=t, s=s, n=n, ks=c.ks, vs=c.vs, nq=8, **kw):
        kernels.paged_append(x, k, v, t, s, n, num_q_heads=nq, k_scale=ks, v_scale=vs, **kw)

    for call in (att, app):
        for kw, message in [
            (dict(k=c.k.float().to(BF16)), "one dtype"), (dict(v=c.v[:, :1]), "one dtype"),
            (dict(ks=None), "k_scale"), (dict(vs=c.vs.double()), "k_scale"), (dict(ks=c.ks[:1]), "k_scale"),
            (dict(t=t.long()), "page_table"), (dict(t=t.repeat(2, 1)), "disagree"), (dict(n=n.cpu()), "kv_len"),
            (dict(s=dev32([0])), "disagree"), (dict(s=dev32([[0, 1]])), "q_start"), (dict(max_new=-1), "max_new"),
            (dict(t=t.repeat(1, 4)[:, ::2]), "contiguous"),
        ]:
            with pytest.raises(ValueError, match=message):
                call(**kw)
    native = c.k.float().to(BF16)
    with pytest.raises(ValueError, match="only e4m3"):
        att(k=native, v=native)
    with pytest.raises(ValueError, match="activation dtype"):
        att(k=native.float(), v=native.float(), ks=None, vs=None)
    with pytest.raises(ValueError, match="head_dim"):
        att(q=q[..., :32])
    with pytest.raises(ValueError, match="head_dim contiguous"):
        att(q=q.transpose(1, 2))
    with pytest.raises(ValueError, match="num_q_heads"):
        att(q=q[:, :3])
    with pytest.raises(ValueError, match="out"):
        att(out=q.float())
    with pytest.raises(ValueError, match="scale"):
        att(scale=-1.0)
    with pytest.raises(ValueError, match="16-byte"):
        att(q=torch.zeros(8 * 64 + 4, dtype=BF16, device=DEV)[4:].view(1, 8, 64))
    cos = torch.zeros(4, 32, device=DEV)
    for kw, message in [
        (dict(nq=7), "num_q_heads"), (dict(cos=cos), "together"), (dict(cos=cos.double(), sin=cos), "cos"),
        (dict(cos=cos, sin=cos[:3]), "sin"), (dict(q_norm=torch.ones(64, device=DEV)), "q_norm"),
        (dict(k_norm=torch.ones(32, dtype=BF16, device=DEV)), "k_norm"), (dict(out=q[:, :7]), "out"),
        (dict(positions=torch.zeros(2, dtype=torch.int64, device=DEV)), "positions"),
        (dict(positions=dev32([0])), "positions"), (dict(x=qkv.expand(2, -1)), "rows"),
    ]:
        with pytest.raises(ValueError, match=message):
            app(**kw)


def test_strides_of_single_elements_do_not_matter():
    """One row, one head, one page: their strides may hold anything."""
    for cache in (BF16, E4M3):
        c = Cache([9], 1, 16, 64, BF16, cache, spare=0)
        c.fill([8])
        qkv = torch.randn(1, 3 * 64, device=DEV).to(BF16)
        want = kernels.paged_append(qkv, c.k, c.v, c.table.to(DEV), dev32([0, 1]), dev32([9]), num_q_heads=1, **c.scales())
        odd = lambda t, dims: t.as_strided(t.shape, [s if n > 1 else 3 for n, s in zip(t.shape, t.stride())][:dims])  # noqa: E731
        k, v = odd(c.k, 4), odd(c.v, 4)
        sc = {} if c.ks is None else {"k_scale": odd(c.ks, 2), "v_scale": odd(c.vs, 2)}
        args = (odd(c.table[:, :1].contiguous().to(DEV), 2), dev32([0, 1]), dev32([9, 0])[::2])
        got = kernels.paged_append(odd(qkv, 2), k, v, *args, num_q_heads=1, **sc)
        assert torch.equal(got, want)
        a = kernels.paged_attention(want, c.k, c.v, c.table.to(DEV), dev32([0, 1]), dev32([9]), **c.scales())
        b = kernels.paged_attention(odd(want, 3), k, v, *args, **sc)
        assert torch.equal(a, b)
    kernels.paged_check_device()


def test_empty_calls():
    c = Cache([20], 2, 16, 64, BF16, E4M3)
    t = c.table.to(DEV)
    assert kernels.paged_attention(torch.zeros(0, 8, 64, dtype=BF16, device=DEV), c.k, c.v, t, dev32([0, 0]), dev32([20]),
                                   **c.scales()).shape == (0, 8, 64)
    assert kernels.paged_append(torch.zeros(0, 12 * 64, dtype=BF16, device=DEV), c.k, c.v, t[:0], dev32([0]), dev32([]),
                                num_q_heads=8, **c.scales()).shape == (0, 8, 64)
    q = torch.zeros(3, 8, 64, dtype=BF16, device=DEV)
    out = torch.full_like(q, 7.0)
    kernels.paged_attention(q, c.k, c.v, t[:0], dev32([0]), dev32([]), out=out, **c.scales())
    kernels.paged_attention(q, c.k, c.v, t, dev32([0, 0]), dev32([20]), out=out, max_new=0, **c.scales())
    kernels.paged_check_device()
    assert (out == 7.0).all()


@pytest.mark.parametrize("cache", [BF16, E4M3])
def test_serving_run(cache):
    """Requests as they are served: prompts, chunks and single tokens of several requests over shared calls, one of
    them admitted later, against each request's own dense attention over what the cache holds."""
    nq, nkv, D, ps = 8, 2, 128, 16
    total = [75, 40, 130]
    c = Cache(total, nkv, ps, D, BF16, cache)
    cos, sin = (t.to(DEV) for t in tables(D))
    have = [0, 0, 0]
    steps = [[30, 5, 0], [1, 20, 64], [1, 1, 1], [8, 1, 1], [1, 1, 50]]
    g = torch.Generator().manual_seed(9)
    for i, new in enumerate(steps):
        have = [h + n for h, n in zip(have, new)]
        qkv = torch.randn(sum(new), (nq + 2 * nkv) * D, generator=g).to(BF16)
        args = (c.table.to(DEV), dev32(starts(new)), dev32(have))
        before = c.host()
        q = kernels.paged_append(qkv.to(DEV), c.k, c.v, *args, num_q_heads=nq, cos=cos, sin=sin, max_new=max(new), **c.scales())
        check_append(c, before, c.host(), q, R.append(qkv, before, c.table, starts(new), have, nq, cos=cos.cpu(),
                                                      sin=sin.cpu()), BF16, D)
        out = kernels.paged_attention(q, c.k, c.v, *args, max_new=max(new), **c.scales())
        kernels.paged_check_device()
        pools = c.host()
        for b, (t0, n, past) in enumerate(R.spans(starts(new), have)):
            if not n:
                continue
            k, v = (R.dense(*pools[key], c.table[b], have[b]) for key in ("k", "v"))
            ref, weight, top = R.attend(q[t0:t0 + n].cpu().double(), k, v, past, D ** -0.5)
            tol = R.attention_tolerance(ref, weight, top, D, have[b], BF16, P_STEP[BF16], cache == E4M3)
            assert ((out[t0:t0 + n].cpu().double() - ref).abs() <= tol).all(), (i, b)


@pytest.mark.parametrize("dtype,cache", [(BF16, BF16), (BF16, E4M3), (F32, F32)])
def test_graph_replays_follow_the_device(dtype, cache):
    """One captured step (append, attention) replayed as the sequences grow, against the same calls made directly;
    two graphs that are replayed at once on two streams keep their scratch apart."""
    nq, nkv, D, ps = 8, 2, 64, 16
    total = [70, 50, 300]
    c, d = Cache(total, nkv, ps, D, dtype, cache), Cache(total, nkv, ps, D, dtype, cache)
    past = [60, 47, 290]
    for x in (c, d):
        x.g.manual_seed(4)
        x.fill(past)
    cos, sin = (t.to(DEV) for t in tables(D))
    table, q_start, kv_len = c.table.to(DEV), dev32(starts([1, 1, 1])), dev32([1, 1, 1])
    qkv = torch.zeros(3, (nq + 2 * nkv) * D, dtype=dtype, device=DEV)

    def step(x, table=table, kv_len=kv_len):
        q = kernels.paged_append(qkv, x.k, x.v, table, q_start, kv_len, num_q_heads=nq, max_new=1, cos=cos, sin=sin, **x.scales())
        return kernels.paged_attention(q, x.k, x.v, table, q_start, kv_len, max_new=1, **x.scales())

    spare = Cache(total, nkv, ps, D, dtype, cache)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(spare)
    torch.cuda.current_stream().wait_stream(side)
    graphs, outs = [], []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(step(c))
        graphs.append(graph)
    for i in range(1, 4):
        kv_len.copy_(dev32([p + i for p in past]))
        qkv.copy_(torch.randn(qkv.shape, generator=torch.Generator().manual_seed(i)).to(dtype))
        want = step(d, d.table.to(DEV))
        graphs[i % 2].replay()
        assert torch.equal(outs[i % 2], want)
    kernels.paged_check_device()
    # Both graphs at once: the appends write the same values, the attention is read-only.
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    for _ in range(20):
        for graph, stream in zip(graphs, streams):
            with torch.cuda.stream(stream):
                graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(outs[0], want) and torch.equal(outs[1], want)


def test_same_results_every_time():
    """Splits, joins and orders do not depend on timing."""
    lens = [2000, 17, 900, 450]
    for cache in (BF16, E4M3):
        c = Cache(lens, 2, 16, 128, BF16, cache)
        c.fill(lens)
        for new in ([1, 1, 1, 1], [3, 2, 1, 4], [300, 17, 2, 90]):
            first = attend(c, new, lens, 8, check=False)
            for _ in range(10):
                assert torch.equal(first, attend(c, new, lens, 8, check=False))


@pytest.mark.parametrize("dtype,cache", [(BF16, E4M3), (BF16, BF16), (F32, F32)])
def test_pool_past_32_bits(dtype, cache):
    """A pool of more than 2^31 elements (2^32 bytes where the type is wider): pages at its end."""
    D, ps, nkv = 128, 128, 8
    per_page = ps * nkv * D
    pages = (1 << 31) // per_page + 40
    k = torch.zeros(pages, nkv, ps, D, dtype=cache, device=DEV)
    c = Cache([300, 130], nkv, ps, D, dtype, cache, spare=0)
    small_k, small_v = c.k, c.v
    c.fill([290, 130])
    shift = pages - c.pages
    ids = torch.arange(c.pages, device=DEV) + shift
    byte = k.view(torch.uint8)
    byte[ids] = small_k.view(torch.uint8)
    v = torch.zeros_like(k)
    v.view(torch.uint8)[ids] = small_v.view(torch.uint8)
    c.k, c.v = k[shift:], v[shift:]
    sc = {}
    if cache == E4M3:
        for key, s in (("k_scale", c.ks), ("v_scale", c.vs)):
            sc[key] = torch.ones(pages, nkv, device=DEV)
            sc[key][shift:] = s
    table = (c.table.clamp(min=0) + shift).to(DEV)
    new, lens = [10, 0], [300, 130]
    qkv = torch.randn(10, (8 + 16) * D, generator=torch.Generator().manual_seed(1)).to(dtype).to(DEV)
    args = (dev32(starts(new)), dev32(lens))
    for limit in (10, 1):
        n = new if limit == 10 else [1, 1]
        a = (dev32(starts(n)), dev32(lens))
        q = torch.randn(sum(n), 8, D, generator=torch.Generator().manual_seed(2)).to(dtype).to(DEV)
        if limit == 10:
            q1 = kernels.paged_append(qkv, k, v, table, *args, num_q_heads=8, **sc)
            q2 = kernels.paged_append(qkv, small_k, small_v, c.table.to(DEV), *args, num_q_heads=8, **c.scales())
            assert torch.equal(q1, q2)
            assert torch.equal(byte[ids], small_k.view(torch.uint8))
        big = kernels.paged_attention(q, k, v, table, *a, max_new=limit, **sc)
        small = kernels.paged_attention(q, small_k, small_v, c.table.to(DEV), *a, max_new=limit, **c.scales())
        assert torch.equal(big, small)
    kernels.paged_check_device()


@pytest.mark.parametrize("dtype,cache", [(BF16, BF16), (BF16, E4M3), (F32, F32), (F32, E4M3)])
@pytest.mark.parametrize("case", range(4))
def test_attention_broken_tokens(dtype, cache, case):
    """Infinities and NaN in keys or values reach the rows that see them, none before: not those of the same block of
    keys, of the same tile, or of other sequences in the same page's row of the pool."""
    new, lens = [([4, 2, 1], [700, 40, 300]), ([3, 4, 1, 2], [5000, 4000, 17, 2]), ([60, 9, 150], [60, 33, 420]),
                 ([200, 130], [3001, 1500])][case]
    D, nq, nkv, ps = (64, 4, 2, 32) if case % 2 else (128, 8, 2, 64)
    c = Cache(lens, nkv, ps, D, dtype, cache, seed=case)
    c.fill(lens)
    q = torch.randn(sum(new), nq, D, generator=torch.Generator().manual_seed(case)).to(dtype)
    code = cache == E4M3

    def put(pages, b, j, h, d, x):
        at = (int(c.table[b, j // ps]), h, j % ps)
        if code:
            pages.view(torch.uint8)[at][d] = 0x7F  # the only special value of the type
        else:
            pages[at][d] = x

    for b, (n, L) in enumerate(zip(new, lens)):
        if n < 2:
            continue
        put(c.v, b, L - 1, 0, 3, math.nan)                # seen by the last token alone
        put(c.v, b, L - n // 2 - 1, 1, slice(0, D, 7), math.inf)
        put(c.k, b, L - 1, 1, 5, math.nan)
    got = torch.full_like(q, 7.0).to(DEV)
    kernels.paged_attention(q.to(DEV), c.k, c.v, c.table.to(DEV), dev32(starts(new)), dev32(lens), out=got, **c.scales())
    kernels.paged_check_device()
    pools, got = c.host(), got.cpu().double()
    for b, (t0, n, past) in enumerate(R.spans(starts(new), lens)):
        k, v = (R.dense(*pools[key], c.table[b], lens[b]) for key in ("k", "v"))
        for i in range(n):
            see = past + i + 1
            ref, weight, top = R.attend(q[t0 + i:t0 + i + 1].double(), k[:, :see], v[:, :see], past + i, D**-0.5)
            tol = R.attention_tolerance(ref, weight, top, D, see, dtype, P_STEP[dtype], code and dtype == BF16)
            x, ref, tol = got[t0 + i], ref[0], tol[0]
            assert torch.equal(x.isnan(), ref.isnan()), (b, i)
            assert torch.equal(x.isinf(), ref.isinf()) and torch.equal(x[x.isinf()], ref[ref.isinf()]), (b, i)
            fine = ref.isfinite()
            assert ((x - ref).abs()[fine] <= tol[fine]).all(), (b, i)


@pytest.mark.parametrize("dtype,cache", [(BF16, BF16), (BF16, E4M3), (F32, F32), (F32, E4M3)])
def test_attention_broken_queries(dtype, cache):
    """An infinity or a NaN in a query row reaches that row alone, also where the keys are cut into parts."""
    new, lens = [1, 4, 70, 1], [6000, 300, 2500, 9]
    c = Cache(lens, 2, 32, 64, dtype, cache, seed=9)
    c.fill(lens)
    q = torch.randn(sum(new), 6, 64, generator=torch.Generator().manual_seed(2)).to(dtype).to(DEV)
    bad = torch.zeros(q.shape[:2], dtype=torch.bool, device=DEV)
    args = (c.k, c.v, c.table.to(DEV), dev32(starts(new)), dev32(lens))
    plain = kernels.paged_attention(q, *args, **c.scales())
    for t, h, x in ((0, 1, math.nan), (0, 4, math.inf), (2, 0, -math.inf), (20, 5, math.nan), (60, 2, math.inf)):
        q[t, h, 7] = x
        bad[t, h] = True
    got = kernels.paged_attention(q, *args, **c.scales())
    kernels.paged_check_device()
    assert got[bad].isnan().all()
    assert torch.equal(got[~bad], plain[~bad])


@pytest.mark.parametrize("dtype,cache", [(BF16, BF16), (BF16, E4M3), (F32, E4M3)])
@pytest.mark.parametrize("rows", [400, 800, 1400])
def test_append_many_rows(dtype, cache, rows):
    """Hundreds of rows of forty sequences: fewer warps per token, and a sequence that is not among the first 32."""
    g = torch.Generator().manual_seed(rows)
    new = (torch.rand(40, generator=g) ** 3 * rows / 20).long().tolist()
    new[37] += rows - sum(new)
    past = torch.randint(0, 70, (40,), generator=g).tolist()
    lens = [p + n for p, n in zip(past, new)]
    for D, nq, nkv, ps in ((64, 3, 1, 16), (128, 4, 2, 64)):
        c = Cache(lens, nkv, ps, D, dtype, cache, seed=rows)
        c.fill(past, spread=6)
        run_append(c, new, lens, nq, norm=True, extra=5)


@pytest.mark.parametrize("cache", [BF16, E4M3])
def test_most_sequences(cache):
    """The most sequences of a call, single tokens and a few with more; one more is refused."""
    g = torch.Generator().manual_seed(8)
    new, lens = [1] * 2048, torch.randint(1, 50, (2048,), generator=g).tolist()
    for i, n in ((5, 30), (1200, 2), (2047, 40)):
        new[i], lens[i] = n, max(n, lens[i])
    c = Cache(lens, 1, 16, 64, BF16, cache)
    c.fill([a - b for a, b in zip(lens, new)])
    run_append(c, new, lens, 2)
    attend(c, new, lens, 4)
    attend(c, [1] * 2048, lens, 2, max_new=1)
    with pytest.raises(ValueError, match="2048"):
        kernels.paged_attention(torch.zeros(1, 2, 64, dtype=BF16, device=DEV), c.k, c.v, torch.zeros(2049, 1, dtype=torch.int32, device=DEV),
                                dev32([0] * 2050), dev32([0] * 2049), **c.scales())


@pytest.mark.parametrize("dtype,cache", [(BF16, BF16), (F32, F32)])
def test_padded_batch(dtype, cache):
    """A batch padded to a captured size: rows of no sequence, sequences without rows or tokens, a wide table."""
    lens = [300, 45, 0, 0]
    c = Cache(lens, 2, 16, 64, dtype, cache)
    c.cols += 500
    c.table = torch.cat((c.table, torch.full((4, 500), -1, dtype=torch.int32)), 1)
    c.fill(lens)
    attend(c, [1, 1, 0, 0], lens, 4, extra=4094, max_new=1)
    attend(c, [1, 3, 0, 0], lens, 4, extra=600, max_new=8)
    run_append(c, [1, 1, 0, 0], lens, 4, extra=2000, max_new=1)


@pytest.mark.parametrize("dtype,cache", [(BF16, BF16), (BF16, E4M3), (F32, E4M3)])
@pytest.mark.parametrize("D,nkv,ps", [(8, 2, 16), (64, 3, 32), (128, 8, 16)])
def test_append_two_to_four_tokens(dtype, cache, D, nkv, ps):
    """A few tokens per sequence that cross a page's end, into pages whose scales grow."""
    new = [4, 1, 3, 0, 2, 4]
    past = [ps - 1, 0, ps - 3, 5, ps, 2 * ps - 2]
    lens = [p + n for p, n in zip(past, new)]
    c = Cache(lens, nkv, ps, D, dtype, cache, seed=D)
    c.fill(past, spread=9)
    run_append(c, new, lens, 2 * nkv, max_new=4, norm=True, extra=1)


@pytest.mark.parametrize("dtype,cache", [(BF16, E4M3), (BF16, BF16), (F32, F32)])
def test_captured_chunks_follow_the_device(dtype, cache):
    """A captured batch of chunks and single tokens, replayed with other ranges, lengths and pages."""
    lens = [700, 300, 64, 2000]
    c = Cache(lens, 2, 16, 128, dtype, cache, seed=3)
    c.fill(lens)
    q = torch.randn(300, 8, 128, generator=torch.Generator().manual_seed(6)).to(dtype).to(DEV)
    table, q_start, kv_len = c.table.to(DEV), dev32([0, 1, 2, 3, 4]), dev32([1, 1, 1, 1])
    out = torch.full_like(q, 7.0)
    graph = torch.cuda.CUDAGraph()
    kernels.paged_attention(q, c.k, c.v, table, q_start, kv_len, max_new=200, **c.scales())
    with torch.cuda.graph(graph):
        kernels.paged_attention(q, c.k, c.v, table, q_start, kv_len, max_new=200, out=out, **c.scales())
    for new, long, order in (([200, 1, 30, 9], lens, [0, 1, 2, 3]), ([1, 1, 1, 1], [5, 300, 64, 1999], [0, 1, 2, 3]),
                             ([0, 150, 0, 150], [2000, 700, 300, 150], [3, 0, 1, 3])):
        table.copy_(c.table[order])
        q_start.copy_(dev32(starts(new)))
        kv_len.copy_(dev32(long))
        out.fill_(7.0)
        graph.replay()
        kernels.paged_check_device()
        want = kernels.paged_attention(q, c.k, c.v, table, q_start, kv_len, max_new=200, out=torch.full_like(q, 7.0), **c.scales())
        assert torch.equal(out, want) and (out[sum(new):] == 7.0).all()
        t0, n = starts(new)[1], new[1]  # against the plain form: one sequence of them
        k, v = (R.dense(*c.host()[key], c.table[order[1]], long[1]) for key in ("k", "v"))
        ref, weight, top = R.attend(q[t0:t0 + n].cpu().double(), k, v, long[1] - n, 128**-0.5)
        tol = R.attention_tolerance(ref, weight, top, 128, long[1], dtype, P_STEP[dtype], cache == E4M3 and dtype == BF16)
        assert ((out[t0:t0 + n].cpu().double() - ref).abs() <= tol).all()


@pytest.mark.parametrize("dtype,cache", [(BF16, E4M3), (BF16, BF16), (F32, E4M3)])
def test_two_streams_at_once(dtype, cache):
    """Appends and attention of two pools on two streams that run side by side."""
    work, streams = [], [torch.cuda.Stream(), torch.cuda.Stream()]
    for seed, (new, lens) in enumerate((([1, 90, 3], [900, 400, 33]), ([2, 1, 140], [50, 1500, 140]))):
        c = Cache(lens, 2, 32, 64, dtype, cache, seed=seed)
        c.fill([b - a for a, b in zip(new, lens)])
        qkv = torch.randn(sum(new), 8 * 64, generator=torch.Generator().manual_seed(seed)).to(dtype).to(DEV)
        args = (c.k, c.v, c.table.to(DEV), dev32(starts(new)), dev32(lens))
        first = kernels.paged_append(qkv, *args, num_q_heads=4, **c.scales())  # the pages hold the tokens from here on
        work.append((c, qkv, args, first, kernels.paged_attention(first, *args, **c.scales())))
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(10):
        for i, (c, qkv, args, first, _) in enumerate(work):
            with torch.cuda.stream(streams[i]):
                got[i].append((kernels.paged_append(qkv, *args, num_q_heads=4, **c.scales()),
                               kernels.paged_attention(first, *args, **c.scales())))
    torch.cuda.synchronize()
    kernels.paged_check_device()
    for i, (_, _, _, first, want) in enumerate(work):
        assert all(torch.equal(q, first) and torch.equal(out, want) for q, out in got[i])
