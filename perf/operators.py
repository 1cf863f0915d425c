"""Cases for the paged KV cache: append (norm, rotation, store) and attention.

Two operators of a serving step on a cache of pages that requests share:

* ``append``: QK-norm and rotary positions of a ragged batch's fused q/k/v rows, keys and values into
  their pages (activation type, or e4m3 with a power-of-two scale per page and head);
* ``attention``: every new token's query heads against its sequence's pages.

A case names the batch (``B`` sequences, ``n_lo..n_hi`` new tokens each, ``l_lo..l_hi`` cached tokens after
the append), the heads and the types.
"""
from __future__ import annotations

import math

import torch

own = False

E4M3 = torch.float8_e4m3fn
E4M3_MAX = 448.0
MIN_EXP = -100
DTYPES = {"bf16": torch.bfloat16, "f32": torch.float32}


def _case(name, op, B, n, length, heads, page, dtype, cache, norm=False):
    return {"name": name, "op": op, "B": B, "n_lo": n[0], "n_hi": n[1], "l_lo": length[0], "l_hi": length[1],
            "nq": heads[0], "nkv": heads[1], "D": heads[2], "page": page, "dtype": dtype, "cache": cache, "norm": norm}


LLAMA_8B = (32, 8, 128)
TINYLLAMA = (32, 4, 64)
QWEN3_4B = (32, 8, 128)


def listed():
    return [
        # One request alone, its next token: the launch is all there is.
        _case("append_one", "append", 1, (1, 1), (130, 130), LLAMA_8B, 64, "bf16", "native"),
        # The benchmark's decode batch (32 rows near 1 K positions), 8-bit pages, Qwen3's QK-norm.
        _case("append_decode_e4m3", "append", 32, (1, 1), (900, 1100), QWEN3_4B, 64, "bf16", "e4m3", True),
        # A prefill micro-batch of the benchmark (8 x 1024 prompt tokens) into 8-bit pages.
        _case("append_prefill_e4m3", "append", 8, (1024, 1024), (1024, 1024), LLAMA_8B, 64, "bf16", "e4m3"),
        # Prompt chunks of odd lengths beside single tokens, fp32 stage with TinyLlama's heads.
        _case("append_ragged_f32", "append", 24, (1, 333), (350, 1500), TINYLLAMA, 16, "f32", "native"),
        # One request alone, its next token, a short context.
        _case("decode_one", "attention", 1, (1, 1), (130, 130), LLAMA_8B, 64, "bf16", "e4m3"),
        # The benchmark's decode batch over 8-bit pages, and over bf16 pages.
        _case("decode_batch_e4m3", "attention", 32, (1, 1), (900, 1100), LLAMA_8B, 64, "bf16", "e4m3"),
        _case("decode_batch_bf16", "attention", 32, (1, 1), (900, 1100), LLAMA_8B, 64, "bf16", "native"),
        # The benchmark's long-context stage: 64 rows at 8 K.
        _case("decode_long_e4m3", "attention", 64, (1, 1), (7900, 8192), LLAMA_8B, 128, "bf16", "e4m3"),
        # Speculative tokens verified together, small pages, very different lengths.
        _case("verify_e4m3", "attention", 16, (2, 4), (17, 5000), LLAMA_8B, 16, "bf16", "e4m3"),
        # Prompt chunks appended to long contexts of 8-bit pages.
        _case("chunk_e4m3", "attention", 4, (700, 1024), (5000, 8192), LLAMA_8B, 64, "bf16", "e4m3"),
        # Prompts from their first token, bf16 pages, TinyLlama's heads, odd lengths.
        _case("prefill_bf16", "attention", 8, (801, 1024), (801, 1024), TINYLLAMA, 32, "bf16", "native"),
        # An fp32 stage's decode step.
        _case("decode_f32", "attention", 8, (1, 1), (1, 2047), TINYLLAMA, 16, "f32", "native"),
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))))


def draw(rng):
    op = rng.choice(["append", "attention", "attention"])
    dtype = rng.choice(["bf16", "bf16", "bf16", "f32"])
    cache = rng.choice(["e4m3", "native"])
    D = rng.choice([64, 128])
    nkv = rng.choice([1, 2, 4, 8])
    G = rng.choice([1, 2, 3, 4, 5, 7, 8])
    page = rng.choice([16, 32, 64, 128])
    B = _log_int(rng, 1, 64)
    n_hi = 1 if rng.random() < 0.5 else _log_int(rng, 2, 1024)
    if op == "attention":
        l_hi = _log_int(rng, 1, 8192 if dtype == "bf16" else 2048)
        if dtype == "f32":
            n_hi = min(n_hi, 64)
        # no dearer than the largest listed ones: cached tokens, score products and their fp32 scores
        B = max(1, min(B, (64 * 8192 * 8) // (l_hi * nkv), int(2.5e11 / (4.0 * min(n_hi, l_hi) * l_hi * nkv * G * D)) or 1))
    else:
        l_hi = _log_int(rng, 1, 2048)
        B = max(1, min(B, 8192 // max(1, min(n_hi, l_hi))))
    n_hi = min(n_hi, l_hi)
    n_lo = rng.randint(1, n_hi)
    l_lo = rng.randint(max(1, min(n_hi, l_hi)), l_hi)
    c = _case("", op, B, (n_lo, n_hi), (l_lo, l_hi), (nkv * G, nkv, D), page, dtype, cache, rng.random() < 0.5)
    del c["name"]
    return c


def _lengths(case):
    """New and cached tokens of every sequence: spread over the case's ranges, the same for every seed."""
    B = case["B"]
    new, cached = [], []
    for b in range(B):
        u = (b * 0.6180339887498949 + 0.35) % 1.0
        v = (b * 0.7548776662466927 + 0.8) % 1.0
        n = case["n_lo"] + int(u * (case["n_hi"] - case["n_lo"] + 1))
        new.append(n)
        cached.append(max(n, case["l_lo"] + int(v * (case["l_hi"] - case["l_lo"] + 1))))
    return new, cached


def _quantise(x, exp):
    return (x * torch.exp2(-exp.float())).clamp(-E4M3_MAX, E4M3_MAX).to(E4M3)


def _exponent(amax):
    """The least e with amax <= 448 * 2^e, at least MIN_EXP."""
    m, e = torch.frexp(amax)  # amax = m * 2^e, 0.5 <= m < 1; 448 = 0.875 * 2^9
    e = e - 9 + (m > 0.875).to(e.dtype)
    return torch.where(amax > 0, e, torch.full_like(e, MIN_EXP)).clamp(min=MIN_EXP)


def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(seed)
    dt = DTYPES[case["dtype"]]
    nq, nkv, D, ps, B = case["nq"], case["nkv"], case["D"], case["page"], case["B"]
    new, cached = _lengths(case)
    need = [-(-c // ps) for c in cached]
    pages = sum(need) + 4
    # A pool that has been in use: pages of a sequence lie anywhere, table entries past its end are -1.
    table = torch.full((B, max(need) + 2), -1, dtype=torch.int32)
    perm = torch.randperm(pages, generator=torch.Generator().manual_seed(seed)).to(torch.int32)
    at = 0
    for b in range(B):
        table[b, : need[b]] = perm[at : at + need[b]]
        at += need[b]
    s = {
        "case": case, "max_new": max(new), "page_table": table.to(dev),
        "q_start": torch.tensor([0] + new, dtype=torch.int32).cumsum(0).to(torch.int32).to(dev),
        "kv_len": torch.tensor(cached, dtype=torch.int32, device=dev),
        "k_scale": None, "v_scale": None,
    }
    T = sum(new)
    for key in ("k", "v"):
        # Heads differ in size by a few powers of two, as keys and values of trained models do.
        x = torch.randn(pages, nkv, ps, D, generator=g, device=dev)
        x *= torch.exp2(torch.rand(1, nkv, 1, 1, generator=g, device=dev) * (2.0 if key == "k" else 6.0) - 1.0)
        if case["cache"] == "e4m3":
            e = _exponent(x.abs().amax((2, 3)))
            s[key + "_pages"] = _quantise(x, e[:, :, None, None])
            s[key + "_scale"] = torch.exp2(e.float())
        else:
            s[key + "_pages"] = x.to(dt)
        del x
    if case["op"] == "append":
        s["qkv"] = torch.randn(T, (nq + 2 * nkv) * D, generator=g, device=dev).mul_(1.7).to(dt)
        inv = 500000.0 ** (-torch.arange(0, D, 2, device=dev, dtype=torch.float64) / D)
        angle = torch.arange(8192, device=dev, dtype=torch.float64)[:, None] * inv
        s["cos"], s["sin"] = angle.cos().float(), angle.sin().float()
        s["q_norm"] = s["k_norm"] = None
        if case["norm"]:
            s["q_norm"] = (1.0 + 0.2 * torch.randn(D, generator=g, device=dev)).to(dt)
            s["k_norm"] = (1.0 + 0.2 * torch.randn(D, generator=g, device=dev)).to(dt)
    else:
        s["q"] = torch.randn(T, nq, D, generator=g, device=dev).mul_(1.2).to(dt)
    return s


def run(s):
    if own:
        from gpu_mesh_b200 import kernels

        if s["case"]["op"] == "append":
            q = kernels.paged_append(
                s["qkv"], s["k_pages"], s["v_pages"], s["page_table"], s["q_start"], s["kv_len"],
                num_q_heads=s["case"]["nq"], max_new=s["max_new"], cos=s["cos"], sin=s["sin"],
                q_norm=s["q_norm"], k_norm=s["k_norm"], eps=1e-6, k_scale=s["k_scale"], v_scale=s["v_scale"])
            return _appended(s, q)
        return kernels.paged_attention(
            s["q"], s["k_pages"], s["v_pages"], s["page_table"], s["q_start"], s["kv_len"],
            max_new=s["max_new"], k_scale=s["k_scale"], v_scale=s["v_scale"])
    if s["case"]["op"] == "append":
        return _appended(s, _append(s))
    return _attention(s)


def _appended(s, q):
    out = {"q": q, "k_pages": s["k_pages"], "v_pages": s["v_pages"]}
    if s["k_scale"] is not None:
        out["k_scale"], out["v_scale"] = s["k_scale"], s["v_scale"]
    return out


# ---- plain forms -------------------------------------------------------------------------------------


def _rows(s):
    """Sequence and cache position of every token row."""
    T = (s["qkv"] if "qkv" in s else s["q"]).shape[0]
    start = s["q_start"].long()
    t = torch.arange(T, device=start.device)
    b = torch.searchsorted(start[1:].contiguous(), t, right=True)
    past = s["kv_len"].long() - (start[1:] - start[:-1])
    return b, past[b] + t - start[:-1][b], past


def _rotate(x, w, cos, sin):
    x = x.float()
    if w is not None:
        x = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + 1e-6) * w.float()
    lo, hi = x.chunk(2, -1)
    return torch.cat((lo * cos - hi * sin, hi * cos + lo * sin), -1)


def _append(s):
    c = s["case"]
    nq, nkv, D, ps = c["nq"], c["nkv"], c["D"], c["page"]
    b, j, past = _rows(s)
    cos, sin = s["cos"][j][:, None], s["sin"][j][:, None]
    q, k, v = s["qkv"].view(-1, nq + 2 * nkv, D).split((nq, nkv, nkv), 1)
    q = _rotate(q, s["q_norm"], cos, sin).to(s["qkv"].dtype)
    page = s["page_table"][b, j // ps].long()
    _store(s["k_pages"], s["k_scale"], _rotate(k, s["k_norm"], cos, sin), page, j % ps, s, past)
    _store(s["v_pages"], s["v_scale"], v.float(), page, j % ps, s, past)
    return q


def _store(pages, scale, x, page, off, s, past):
    if scale is None:
        pages[page, :, off] = x.to(pages.dtype)
        return
    ps = pages.shape[2]
    bits = pages.view(torch.uint8)
    amax = torch.where(x.isfinite(), x.abs(), 0.0).amax(-1)
    new = torch.zeros_like(scale).scatter_reduce_(0, page[:, None].expand_as(amax), amax, "amax")
    need = _exponent(new)
    old = torch.frexp(scale)[1] - 1
    touched = torch.zeros(len(scale), dtype=torch.bool, device=scale.device).index_fill_(0, page, True)
    # The page that a sequence's first new token goes to, where it holds earlier tokens already.
    first = s["page_table"].gather(1, (past[:, None] // ps).clamp(max=s["page_table"].shape[1] - 1))[:, 0].long()
    part = past % ps
    kept = torch.zeros_like(touched).index_put_((first.clamp(min=0),), (part > 0) & (first >= 0), accumulate=True) & touched
    exp = torch.where(kept[:, None], torch.maximum(old, need), need)
    exp = torch.where(touched[:, None], exp, old)
    f = first.clamp(min=0)
    held = pages[f].float() * torch.exp2((old - exp)[f].float())[:, :, None, None]
    valid = (torch.arange(ps, device=part.device) < part[:, None])[:, None, :, None] & kept[f][:, None, None, None]
    bits[f] = torch.where(valid, held.to(E4M3).view(torch.uint8), bits[f])
    bits[page, :, off] = _quantise(x, exp[page][:, :, None]).view(torch.uint8)
    scale.copy_(torch.where(touched[:, None], torch.exp2(exp.float()), scale))


def _dense(pages, scale, table):
    """Keys or values of every sequence as fp32 [B, nkv, table columns * page, D]."""
    x = pages.view(torch.uint8)[table].view(pages.dtype) if scale is not None else pages[table]
    x = x.float()
    if scale is not None:
        x = x * scale[table][..., None, None]
    B, n, nkv, ps, D = x.shape
    return x.permute(0, 2, 1, 3, 4).reshape(B, nkv, n * ps, D)


def _attention(s):
    q = s["q"]
    T, nq, D = q.shape
    nkv, N = s["k_pages"].shape[1], s["max_new"]
    G = nq // nkv
    b, j, past = _rows(s)
    table = s["page_table"].long().clamp(min=0)
    k, v = _dense(s["k_pages"], s["k_scale"], table), _dense(s["v_pages"], s["v_scale"], table)
    B, L = k.shape[0], k.shape[2]
    key = torch.arange(L, device=q.device)
    v = v.masked_fill((key >= s["kv_len"].long()[:, None])[:, None, :, None], 0.0)
    at = torch.arange(T, device=q.device) - s["q_start"].long()[b]
    padded = torch.zeros(B, N, nkv, G, D, device=q.device)
    padded[b, at] = q.float().view(T, nkv, G, D)
    score = padded.permute(0, 2, 1, 3, 4).reshape(B, nkv, N * G, D) @ k.transpose(2, 3) * (1.0 / math.sqrt(D))
    seen = key <= (past[:, None] + torch.arange(N, device=q.device))[:, :, None]  # [B, N, L]
    score = score.view(B, nkv, N, G, L).masked_fill(~seen[:, None, :, None], -math.inf)
    p = torch.exp(score - score.amax(-1, keepdim=True).clamp(min=-3e38))
    p = p / p.sum(-1, keepdim=True).clamp(min=1e-38)
    out = (p.view(B, nkv, N * G, L) @ v).view(B, nkv, N, G, D)
    return out.permute(0, 2, 1, 3, 4)[b, at].reshape(T, nq, D).to(q.dtype)


# ---- work and 64-bit values --------------------------------------------------------------------------


def work(case):
    new, cached = _lengths(case)
    nq, nkv, D = case["nq"], case["nkv"], case["D"]
    e = 2 if case["dtype"] == "bf16" else 4
    c = 1 if case["cache"] == "e4m3" else e
    T = sum(new)
    if case["op"] == "append":
        tables = T * D * 4 if not case["n_hi"] == 1 else min(T, case["l_hi"]) * D * 4
        scales = 0 if c == e else 2 * 4 * nkv * sum(-(-n // case["page"]) for n in new)
        return {"bytes": T * (2 * nq + 2 * nkv) * D * e + T * 2 * nkv * D * c + tables + scales,
                "flops": T * (nq + 2 * nkv) * D * (7 if case["norm"] else 3)}
    seen = sum(n * (l - n) + n * (n + 1) / 2 for n, l in zip(new, cached))
    scales = 0 if case["cache"] != "e4m3" else 2 * 4 * nkv * sum(-(-l // case["page"]) for l in cached)
    return {"bytes": 2 * T * nq * D * e + 2 * sum(cached) * nkv * D * c + scales, "flops": 4.0 * nq * D * seen}


def exact(case, seed):
    s = prepare(case, seed)
    new, cached = _lengths(case)
    nq, nkv, D, ps = case["nq"], case["nkv"], case["D"], case["page"]
    table = s["page_table"].cpu().long()
    if case["op"] == "attention":
        out = torch.empty(sum(new), nq, D, dtype=torch.float64, device="cuda")
        t = 0
        for b, (n, L) in enumerate(zip(new, cached)):
            ids = table[b, : -(-L // ps)].cuda()
            held = []
            for key in ("k", "v"):
                x = s[key + "_pages"].view(torch.uint8)[ids].view(E4M3).double() if case["cache"] == "e4m3" else s[key + "_pages"][ids].double()
                if case["cache"] == "e4m3":
                    x = x * s[key + "_scale"][ids].double()[:, :, None, None]
                held.append(x.transpose(0, 1).reshape(nkv, -1, D)[:, :L])
            bar = torch.ones(n, L, dtype=torch.bool, device="cuda").triu(L - n + 1)
            for h in range(nq):
                g = h // (nq // nkv)
                w = (s["q"][t : t + n, h].double() @ held[0][g].T / math.sqrt(D)).masked_fill(bar, -math.inf)
                out[t : t + n, h] = torch.softmax(w, -1) @ held[1][g]
            t += n
        return out
    x = s["qkv"].double().view(-1, nq + 2 * nkv, D)
    place = [(b, L - n + i) for b, (n, L) in enumerate(zip(new, cached)) for i in range(n)]
    j = torch.tensor([p for _, p in place], device="cuda")
    turn = torch.complex(s["cos"][j].double(), s["sin"][j].double())[:, None]

    def turned(y, w):
        if w is not None:
            y = y / (y.square().mean(-1, keepdim=True) + 1e-6).sqrt() * w.double()
        z = torch.complex(y[..., : D // 2], y[..., D // 2 :]) * turn
        return torch.cat((z.real, z.imag), -1)

    out = {"q": turned(x[:, :nq], s["q_norm"])}
    page = torch.tensor([int(table[b, p // ps]) for b, p in place])
    for key, y in (("k", turned(x[:, nq : nq + nkv], s["k_norm"])), ("v", x[:, nq + nkv :])):
        pool = s[key + "_pages"].double()
        if case["cache"] != "e4m3":
            pool[page.cuda(), :, j % ps] = y
            out[key + "_pages"] = pool
            continue
        # What a page is worth in units of its scale, before the rounding to 8 bits.
        step = s[key + "_scale"].double()
        amax = torch.zeros(len(step), nkv, dtype=torch.float64, device="cuda")
        amax.index_reduce_(0, page.cuda(), y.abs().amax(-1), "amax")
        e = (torch.log2(amax / E4M3_MAX).round() - 1).clamp(min=MIN_EXP)
        for _ in range(2):  # the least step that reaches amax, by exact comparisons
            e += E4M3_MAX * torch.exp2(e) < amax
        want = torch.exp2(e)
        grown = step.clone()
        for b, (n, L) in enumerate(zip(new, cached)):
            for i in range((L - n) // ps, -(-L // ps)):
                held, p = max(0, L - n - i * ps), int(table[b, i])
                grown[p] = torch.maximum(step[p], want[p]) if held else want[p]
                pool[p, :, :held] *= (step[p] / grown[p])[:, None, None]
        pool[page.cuda(), :, j % ps] = y / grown[page.cuda()][:, :, None]
        out[key + "_pages"], out[key + "_scale"] = pool, grown
    return out
