"""The serving attention operators whose speed is measured: one call each.

Four operators that a program serving a model with full-length attention runs next to
the hybrid block stack: per-head norms with the position rotation, appending to a paged
key-value cache, attention of one new token over that cache, and attention over packed
prompts.  Head layouts are those of ``hybrid_llm_amd.config`` (C1: 4 heads x 64; C5: 16
query heads x 64) and generic grouped ones.

``listed()`` names the cases, ``draw(rng)`` gives more of the same ranges; a case is a
dict of plain values.  ``prepare`` makes what a program holds before the call, ``run`` is
one call (the plain form, or the package's kernels where ``own`` is true), ``exact`` the
same in 64 bits.
"""
from __future__ import annotations

import math

import torch

own = False

DEV = "cuda"
BF16 = torch.bfloat16
FP8 = torch.float8_e4m3fn
FP8_MAX = 448.0
EPS = 1e-6

# (query heads, key-value heads, head width): C1's, C5's with grouped keys, generic ones
HEADS = ((4, 4, 64), (16, 4, 64), (8, 8, 64), (16, 2, 128), (32, 8, 128))


def listed():
    return [
        # one token of one chat: q and k of a single row, far into its context
        {"name": "qk_one_token", "family": "qk", "tokens": 1, "hq": 16, "hkv": 4, "hd": 64,
         "rot": 64, "interleaved": False, "norm": True, "far": True},
        # one prompt of odd length, interleaved pairs, half of each head rotated
        {"name": "qk_prompt_1003", "family": "qk", "tokens": 1003, "hq": 16, "hkv": 2, "hd": 128,
         "rot": 64, "interleaved": True, "norm": True, "far": False},
        # 16384 tokens of packed prompts
        {"name": "qk_prompt_16384", "family": "qk", "tokens": 16384, "hq": 32, "hkv": 8,
         "hd": 128, "rot": 128, "interleaved": False, "norm": True, "far": False},
        # the new token of 64 sequences: q, k and v in one call, bf16 pages of 16 tokens
        {"name": "append_step_64", "family": "append", "step": True, "seqs": 64, "tokens": 64,
         "hq": 32, "hkv": 8, "hd": 128, "page": 16, "fp8": False, "norm": True, "with_q": True},
        # four prompts, 8191 tokens in all, into 8-bit pages of 64 tokens
        {"name": "append_prompts_8191", "family": "append", "step": False, "seqs": 4,
         "tokens": 8191, "hq": 16, "hkv": 2, "hd": 128, "page": 64, "fp8": True, "norm": False,
         "with_q": False},
        # one chat's next token, about a thousand tokens in
        {"name": "decode_chat", "family": "decode", "seqs": 1, "longest": 1023, "even": True,
         "hq": 16, "hkv": 4, "hd": 64, "page": 16, "fp8": False, "window": 0, "cap": 0.0,
         "slopes": False},
        # a batch of 64 sequences of any length up to 4096, capped scores
        {"name": "decode_ragged_64", "family": "decode", "seqs": 64, "longest": 4096,
         "even": False, "hq": 32, "hkv": 8, "hd": 128, "page": 16, "fp8": False, "window": 0,
         "cap": 50.0, "slopes": False},
        # four sequences of 131072 tokens, 8-bit cache: long documents
        {"name": "decode_long_4", "family": "decode", "seqs": 4, "longest": 131072, "even": True,
         "hq": 32, "hkv": 8, "hd": 128, "page": 64, "fp8": True, "window": 0, "cap": 0.0,
         "slopes": False},
        # one short prompt with a two-way prefix and capped scores, C1's heads
        {"name": "prefill_prefix_777", "family": "prefill", "docs": 1, "tokens": 777, "hq": 4,
         "hkv": 4, "hd": 64, "window": 0, "cap": 30.0, "slopes": False, "prefix": True},
        # 37 prompts of ragged lengths in one call, windowed, with a distance bias
        {"name": "prefill_packed_8192", "family": "prefill", "docs": 37, "tokens": 8192,
         "hq": 16, "hkv": 4, "hd": 64, "window": 512, "cap": 0.0, "slopes": True,
         "prefix": False},
        # one long document
        {"name": "prefill_long_16384", "family": "prefill", "docs": 1, "tokens": 16384, "hq": 16,
         "hkv": 2, "hd": 128, "window": 0, "cap": 0.0, "slopes": False, "prefix": False},
    ]


def _log(rng, lo, hi):
    """A whole number of [lo, hi], spread over the logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    family = rng.choice(("qk", "append", "decode", "decode", "prefill", "prefill"))
    hq, hkv, hd = rng.choice(HEADS)
    c = {"family": family, "hq": hq, "hkv": hkv, "hd": hd}
    if family == "qk":
        c.update(tokens=_log(rng, 1, 16384), rot=rng.choice((hd, hd, hd // 2)),
                 interleaved=rng.random() < 0.4, norm=rng.random() < 0.7,
                 far=rng.random() < 0.3)
    elif family == "append":
        step = rng.random() < 0.5
        seqs = _log(rng, 1, 128) if step else rng.randint(1, 8)
        c.update(step=step, seqs=seqs, tokens=seqs if step else _log(rng, seqs, 8191),
                 page=rng.choice((16, 64, 128)), fp8=rng.random() < 0.4,
                 norm=rng.random() < 0.6, with_q=step or rng.random() < 0.4)
    elif family == "decode":
        seqs = _log(rng, 1, 64)
        c.update(seqs=seqs, longest=_log(rng, 1, 262144 // seqs), even=rng.random() < 0.4,
                 page=rng.choice((16, 32, 64, 256)), fp8=rng.random() < 0.4,
                 window=rng.choice((0, 0, 0, 512)), cap=rng.choice((0.0, 0.0, 50.0)),
                 slopes=rng.random() < 0.25)
    else:
        tokens = _log(rng, 1, 8192)
        c.update(tokens=tokens, docs=min(tokens, _log(rng, 1, 64)),
                 window=rng.choice((0, 0, 128, 512)), cap=rng.choice((0.0, 0.0, 30.0)),
                 slopes=rng.random() < 0.25, prefix=rng.random() < 0.3)
    return c


# ----------------------------------------------------------------------- inputs
def _cuts(total, parts, g):
    """`parts` lengths of at least 1 that sum to `total`, as their running sums from 0."""
    inner = torch.randperm(total - 1, generator=g)[:parts - 1].sort().values + 1
    return torch.cat([torch.zeros(1, dtype=torch.long), inner, torch.tensor([total])])


def _heads_slopes(hq):
    """One slope per head: a geometric series from 2^(-8/hq) to 2^-8."""
    return [2.0 ** (-8.0 * (h + 1) / hq) for h in range(hq)]


def prepare(c, seed):
    """Inputs, cache and page tables of one case, made from the seed."""
    g = torch.Generator(device=DEV).manual_seed(int(seed))
    host = torch.Generator().manual_seed(int(seed) + 1)
    f, hq, hkv, hd = c["family"], c["hq"], c["hkv"], c["hd"]

    def randn(*shape, std=1.0, mean=0.0):
        return torch.empty(shape, device=DEV).normal_(mean, std, generator=g)

    def stored(t, scale):
        return (t / scale).clamp(-FP8_MAX, FP8_MAX).to(FP8) if c["fp8"] else t.to(BF16)

    s = {"case": c}
    if f in ("qk", "append", "prefill"):
        # rows of one fused projection: q | k | v side by side
        row = randn(c["tokens"], (hq + 2 * hkv) * hd).to(BF16)
        q, k, v = row.split([hq * hd, hkv * hd, hkv * hd], dim=1)
        s.update(q=q.view(-1, hq, hd), k=k.view(-1, hkv, hd), v=v.view(-1, hkv, hd))
    if f in ("qk", "append"):
        rot = c.get("rot", hd)
        s["inv_freq"] = (10000.0 ** (-torch.arange(0, rot, 2, dtype=torch.float64) / rot)
                         ).float().to(DEV)
        for n in ("q_norm", "k_norm"):
            s[n] = randn(hd, std=0.1, mean=1.0) if c["norm"] else None
    if f == "qk":
        first = int(torch.randint(200000, 1000000, (1,), generator=host)) if c["far"] else 0
        s["positions"] = torch.arange(first, first + c["tokens"], dtype=torch.int32, device=DEV)
    elif f in ("append", "decode"):
        B, P = c["seqs"], c["page"]
        if f == "decode":
            if c["even"]:  # all near the longest, the first one at it
                low = max(1, c["longest"] - c["longest"] // 16)
            else:
                low = 1
            lens = torch.randint(low, c["longest"] + 1, (B,), generator=host)
            lens[0] = c["longest"]
        elif c["step"]:
            lens = torch.randint(1, 513, (B,), generator=host)
        else:
            cu = _cuts(c["tokens"], B, host)
            lens = cu[1:] - cu[:-1]
        # as many pages as any lengths of the case can fill, handed out in random order
        if f == "append" and not c["step"]:
            width, pages = (c["tokens"] + P - 1) // P, c["tokens"] // P + B + 3
        else:
            width = ((c["longest"] if f == "decode" else 512) + P - 1) // P
            pages = B * width + 3
        used = (lens + P - 1) // P
        table = torch.zeros(B, width, dtype=torch.long)
        table[torch.arange(width) < used[:, None]] = torch.randperm(
            pages, generator=host)[:int(used.sum())]
        s.update(page_table=table.to(torch.int32).to(DEV), k_scale=1.0, v_scale=1.0)
        if c["fp8"]:
            s.update(k_scale=0.021, v_scale=0.017)
        if f == "decode":
            s["lengths"] = lens.to(torch.int32).to(DEV)
            s["q"] = randn(B, hq, hd).to(BF16)
            s["slopes"] = (torch.tensor(_heads_slopes(hq), device=DEV) if c["slopes"] else None)
        elif c["step"]:
            s.update(positions=(lens - 1).to(torch.int32).to(DEV), rows=None)
        else:
            rows = torch.repeat_interleave(torch.arange(B), lens)
            s["positions"] = (torch.arange(c["tokens"]) - cu[:-1][rows]).to(torch.int32).to(DEV)
            s["rows"] = rows.to(torch.int32).to(DEV)
        shape = (pages, hkv, P, hd)
        s["k_cache"] = stored(randn(*shape), s["k_scale"])
        s["v_cache"] = stored(randn(*shape), s["v_scale"])
    else:
        cu = _cuts(c["tokens"], c["docs"], host)
        lens = cu[1:] - cu[:-1]
        s["cu_seqlens"] = cu.to(torch.int32).to(DEV)
        s["slopes"] = torch.tensor(_heads_slopes(hq), device=DEV) if c["slopes"] else None
        s["prefix"] = (lens // 4).to(torch.int32).to(DEV) if c["prefix"] else None
    return s


# ----------------------------------------------------------------------- plain forms
def _norm_rope(x, weight, positions, inv_freq, interleaved):
    """x [N, H, hd] in 32 bits: RMSNorm over hd (where weight is given), rotated pairs."""
    x = x.float()
    if weight is not None:
        x = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS) * weight
    angle = positions.double()[:, None] * inv_freq.double()
    cos, sin = angle.cos().float()[:, None], angle.sin().float()[:, None]
    half = inv_freq.numel()
    turned, rest = x[..., :2 * half], x[..., 2 * half:]
    if interleaved:
        a, b = turned[..., 0::2], turned[..., 1::2]
        turned = torch.stack((a * cos - b * sin, b * cos + a * sin), -1).flatten(-2)
    else:
        a, b = turned[..., :half], turned[..., half:]
        turned = torch.cat((a * cos - b * sin, b * cos + a * sin), -1)
    return torch.cat((turned, rest), -1)


def _put(cache, page, slot, x, scale):
    """x [N, H, hd] in 32 bits into cache[page, :, slot]."""
    if cache.dtype == FP8:
        x = (x / scale).clamp(-FP8_MAX, FP8_MAX).to(FP8).view(torch.uint8)
        cache.view(torch.uint8)[page, :, slot] = x
    else:
        cache[page, :, slot] = x.to(BF16)


def _gather(cache, table, scale):
    """The pages of each sequence in order: [B, H, tokens, hd] in 32 bits."""
    codes = cache.view(torch.uint8)[table] if cache.dtype == FP8 else cache[table]
    x = codes.view(cache.dtype).float() if cache.dtype == FP8 else codes.float()
    B, n, H, P, hd = x.shape
    return x.permute(0, 2, 1, 3, 4).reshape(B, H, n * P, hd) * scale


def _softmax_product(scores, seen, v, cap, bias):
    """softmax over the seen scores, times v; zeros where nothing is seen."""
    if cap:
        scores = torch.tanh(scores / cap) * cap
    if bias is not None:
        scores = scores - bias
    scores = scores.masked_fill_(~seen, -math.inf)
    top = scores.amax(-1, keepdim=True).clamp_min(torch.finfo(scores.dtype).min)
    p = scores.sub_(top).exp_()
    return torch.matmul(p, v) / p.sum(-1, keepdim=True).clamp_min(1e-30)


def _plain_decode(s):
    c = s["case"]
    B, hq, hkv, hd = c["seqs"], c["hq"], c["hkv"], c["hd"]
    table = s["page_table"].long()
    k = _gather(s["k_cache"], table, s["k_scale"])
    v = _gather(s["v_cache"], table, s["v_scale"])
    n = k.shape[2]
    j = torch.arange(n, device=DEV)
    last = s["lengths"].long()[:, None] - 1
    seen = j <= last
    if c["window"]:
        seen &= j > last - c["window"]
    # positions past a length hold whatever the page held: not part of the sum
    v = v.masked_fill(~seen[:, None, :, None], 0.0)
    scores = torch.matmul(s["q"].float().view(B, hkv, hq // hkv, hd) * hd ** -0.5,
                          k.transpose(-1, -2).contiguous())
    bias = None
    if s["slopes"] is not None:
        bias = s["slopes"].view(1, hkv, -1, 1) * (last - j).float()[:, None, None, :]
    out = _softmax_product(scores, seen[:, None, None, :], v, c["cap"], bias)
    return out.reshape(B, hq, hd).to(BF16)


def _seen_in_prompts(c, s):
    """[N, N]: whether query i (row) sees key j."""
    cu = s["cu_seqlens"].long()
    i = torch.arange(c["tokens"], device=DEV)
    doc = torch.searchsorted(cu, i, right=True) - 1
    end = i + 1
    if s["prefix"] is not None:
        end = torch.maximum(end, torch.minimum(cu[doc] + s["prefix"].long()[doc], cu[doc + 1]))
    first = cu[doc]
    if c["window"]:
        first = torch.maximum(first, i - c["window"] + 1)
    return (i >= first[:, None]) & (i < end[:, None])


def _plain_prefill(s):
    c = s["case"]
    N, hq, hkv, hd = c["tokens"], c["hq"], c["hkv"], c["hd"]
    q = s["q"].float().transpose(0, 1).contiguous() * hd ** -0.5
    k = s["k"].float().permute(1, 2, 0).repeat_interleave(hq // hkv, 0)
    v = s["v"].float().transpose(0, 1).repeat_interleave(hq // hkv, 0)
    bias = None
    if s["slopes"] is not None:
        i = torch.arange(N, device=DEV, dtype=torch.float32)
        bias = s["slopes"][:, None, None] * (i[:, None] - i).abs()
    out = _softmax_product(torch.matmul(q, k), _seen_in_prompts(c, s), v, c["cap"], bias)
    return out.transpose(0, 1).to(BF16)


def _plain(s):
    c = s["case"]
    f = c["family"]
    if f == "qk":
        return {n: _norm_rope(s[n], s[n + "_norm"], s["positions"], s["inv_freq"],
                              c["interleaved"]).to(BF16) for n in ("q", "k")}
    if f == "append":
        pos = s["positions"].long()
        rows = s["rows"].long() if s["rows"] is not None else torch.arange(len(pos), device=DEV)
        page, slot = s["page_table"].long()[rows, pos // c["page"]], pos % c["page"]
        k = _norm_rope(s["k"], s["k_norm"], pos, s["inv_freq"], False)
        _put(s["k_cache"], page, slot, k, s["k_scale"])
        _put(s["v_cache"], page, slot, s["v"].float(), s["v_scale"])
        out = {"k_cache": s["k_cache"], "v_cache": s["v_cache"]}
        if c["with_q"]:
            out["q"] = _norm_rope(s["q"], s["q_norm"], pos, s["inv_freq"], False).to(BF16)
        return out
    return _plain_decode(s) if f == "decode" else _plain_prefill(s)


def _own(s):
    from hybrid_llm_amd import ops
    c = s["case"]
    f = c["family"]
    if f == "qk":
        q, k = ops.qk_norm_rope(s["q"], s["k"], s["positions"], s["inv_freq"],
                                q_norm=s["q_norm"], k_norm=s["k_norm"], eps=EPS,
                                interleaved=c["interleaved"])
        return {"q": q, "k": k}
    if f == "append":
        with_q = {"q": s["q"], "q_norm": s["q_norm"]} if c["with_q"] else {}
        q = ops.paged_kv_append(s["k"], s["v"], s["k_cache"], s["v_cache"], s["page_table"],
                                s["positions"], rows=s["rows"], inv_freq=s["inv_freq"],
                                k_norm=s["k_norm"], eps=EPS, k_scale=s["k_scale"],
                                v_scale=s["v_scale"], **with_q)
        out = {"k_cache": s["k_cache"], "v_cache": s["v_cache"]}
        if c["with_q"]:
            out["q"] = q
        return out
    if f == "decode":
        return ops.paged_attn_decode(s["q"], s["k_cache"], s["v_cache"], s["page_table"],
                                     s["lengths"], window=c["window"], softcap=c["cap"],
                                     slopes=s["slopes"], k_scale=s["k_scale"],
                                     v_scale=s["v_scale"])
    return ops.packed_attn_prefill(s["q"], s["k"], s["v"], s["cu_seqlens"], window=c["window"],
                                   softcap=c["cap"], slopes=s["slopes"], prefix=s["prefix"])


def run(s):
    return _own(s) if own else _plain(s)


# ----------------------------------------------------------------------- necessary work
def _case_lengths(c):
    """Total visible keys of a decode case: exact where lengths are even, else expected."""
    longest = c["longest"]
    mean = longest - longest // 32 if c["even"] else (longest + 1) / 2
    rest = min(mean, c["window"]) if c["window"] else mean
    return (min(longest, c["window"]) if c["window"] else longest) + (c["seqs"] - 1) * rest


def _pairs(n, window):
    w = min(window, n) if window else n
    return w * (w + 1) / 2 + (n - w) * w


def work(c):
    f, hq, hkv, hd = c["family"], c["hq"], c["hkv"], c["hd"]
    if f == "qk":
        elems = c["tokens"] * (hq + hkv) * hd
        return {"bytes": 4 * elems + 4 * c["tokens"], "flops": 8 * elems}
    if f == "append":
        kv = c["tokens"] * hkv * hd
        q = c["tokens"] * hq * hd if c["with_q"] else 0
        return {"bytes": 2 * kv * (3 if c["fp8"] else 4) + 4 * q + 8 * c["tokens"],
                "flops": 8 * (kv + q)}
    if f == "decode":
        keys = _case_lengths(c)
        return {"bytes": 2 * keys * hkv * hd * (1 if c["fp8"] else 2) + 4 * c["seqs"] * hq * hd,
                "flops": 4 * keys * hq * hd}
    n = c["tokens"] / c["docs"]
    pairs = c["docs"] * _pairs(n, c["window"])
    if c["prefix"]:  # the upper triangle of the first quarter of each prompt
        p = n / 4
        pairs += c["docs"] * (p * (p - 1) / 2)
    return {"bytes": 2 * c["tokens"] * hd * (2 * hq + 2 * hkv), "flops": 4 * pairs * hq * hd}


# ----------------------------------------------------------------------- 64-bit results
def _exact_rope(x, weight, positions, inv_freq, interleaved):
    """Each pair as a complex number times e^(i angle)."""
    x = x.double()
    if weight is not None:
        x = x / (x.pow(2).sum(-1, keepdim=True) / x.shape[-1] + EPS).sqrt() * weight.double()
    angle = torch.outer(positions.double(), inv_freq.double())[:, None]
    turn = torch.polar(torch.ones_like(angle), angle)
    R = 2 * inv_freq.numel()
    head = x[..., :R].clone()
    if interleaved:
        z = torch.view_as_complex(head.view(*head.shape[:-1], R // 2, 2)) * turn
        head = torch.view_as_real(z).flatten(-2)
    else:
        z = torch.complex(head[..., :R // 2].contiguous(), head[..., R // 2:].contiguous()) * turn
        head = torch.cat((z.real, z.imag), -1)
    return torch.cat((head, x[..., R:]), -1)


def _exact_rows(q, k, v, first, end, at, scale, cap, slope):
    """softmax attention of the queries q [n, hd] over k, v [m, hd], key j seen where
    first <= j < end; `at`: the queries' own key indices."""
    z = q @ k.t() * scale
    if cap:
        z = cap * torch.tanh(z / cap)
    j = torch.arange(k.shape[0], device=DEV)
    if slope is not None:
        z = z - slope * (at[:, None] - j).abs().double()
    z = torch.where((j >= first[:, None]) & (j < end[:, None]), z, -math.inf)
    return torch.softmax(z, -1) @ v


def exact(c, seed):
    s = prepare(c, seed)
    f, hq, hkv, hd = c["family"], c["hq"], c["hkv"], c["hd"]
    if f == "qk":
        return {n: _exact_rope(s[n], s[n + "_norm"], s["positions"], s["inv_freq"],
                               c["interleaved"]) for n in ("q", "k")}
    group, scale = hq // hkv, hd ** -0.5
    if f == "append":
        pos = s["positions"].long()
        rows = s["rows"].long() if s["rows"] is not None else torch.arange(len(pos), device=DEV)
        new = {"k": _exact_rope(s["k"], s["k_norm"], pos, s["inv_freq"], False),
               "v": s["v"].double()}
        out = {}
        for n in ("k", "v"):
            cache = s[n + "_cache"].float().double()
            x = new[n] / s[n + "_scale"] if c["fp8"] else new[n]
            cache[s["page_table"].long()[rows, pos // c["page"]], :, pos % c["page"]] = x
            out[n + "_cache"] = cache
        if c["with_q"]:
            out["q"] = _exact_rope(s["q"], s["q_norm"], pos, s["inv_freq"], False)
        return out
    slopes = s["slopes"].double() if s["slopes"] is not None else [None] * hq
    if f == "decode":
        out = torch.empty(c["seqs"], hq, hd, dtype=torch.float64, device=DEV)
        for b, n in enumerate(s["lengths"].tolist()):
            pages = s["page_table"][b, :(n + c["page"] - 1) // c["page"]].long()
            k, v = (s[x + "_cache"].view(torch.uint8)[pages].view(s[x + "_cache"].dtype).float()
                    .double().transpose(0, 1).reshape(hkv, -1, hd)[:, :n] * s[x + "_scale"]
                    for x in ("k", "v"))
            at = torch.tensor([n - 1], device=DEV)
            first = torch.tensor([max(0, n - c["window"]) if c["window"] else 0], device=DEV)
            for h in range(hq):
                out[b, h] = _exact_rows(s["q"][b, h:h + 1].double(), k[h // group], v[h // group],
                                        first, at + 1, at, scale, c["cap"], slopes[h])[0]
        return out
    cu = s["cu_seqlens"].tolist()
    out = torch.empty(c["tokens"], hq, hd, dtype=torch.float64, device=DEV)
    for d, (a, b) in enumerate(zip(cu, cu[1:])):
        n = b - a
        at = torch.arange(n, device=DEV)
        first = (at - c["window"] + 1).clamp_min(0) if c["window"] else torch.zeros_like(at)
        end = at + 1
        if s["prefix"] is not None:
            end = end.clamp_min(min(n, int(s["prefix"][d])))
        for h in range(hq):
            k, v = s["k"][a:b, h // group].double(), s["v"][a:b, h // group].double()
            for i in range(0, n, 4096):
                m = slice(i, min(n, i + 4096))
                out[a + m.start:a + m.stop, h] = _exact_rows(
                    s["q"][a + m.start:a + m.stop, h].double(), k, v, first[m], end[m], at[m],
                    scale, c["cap"], slopes[h])
    return out
