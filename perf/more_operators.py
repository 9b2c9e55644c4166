"""Serving operators around a paged cache held in 4 bits whose speed is measured: one pass each.

The step of a program that serves a model with drafted tokens: pages handed out for the new
tokens of a batch, their keys and values stored in 4 bits (and read back), attention of one
or several new tokens per sequence over that cache, and the verification of drafted tokens
against the target's probabilities.  Head layouts are those of ``hybrid_llm_amd.config``
(C1: 4 heads x 64; C5: 16 query heads x 64) and generic grouped ones; the vocabularies are
C1's 32000 and generic ones.

The 4-bit format is the microscaling one of 32-value blocks: each value a 4-bit float (sign,
2 exponent bits, 1 mantissa bit: 0, 0.5, 1, 1.5, 2, 3, 4, 6), each block of 32 dims of one
row a power of two 2^(byte - 127) (byte 255: a block that holds a NaN or an infinity).

``listed()`` names the cases, ``draw(rng)`` gives more of the same ranges; a case is a
dict of plain values.  ``prepare`` makes what a program holds before the call, ``run`` is
one pass (the plain form, or the package's kernels where ``own`` is true), ``exact`` the
same from the definition in 64 bits.
"""
from __future__ import annotations

import math

import torch

own = False

DEV = "cuda"
BF16 = torch.bfloat16
FP4 = torch.float4_e2m1fn_x2
E8M0 = torch.float8_e8m0fnu
EPS = 1e-6
TEMPERATURE = 0.8

# (query heads, key-value heads, head width): C1's, C5's with grouped keys, generic ones
HEADS = ((4, 4, 64), (16, 4, 64), (8, 8, 64), (16, 2, 128), (32, 8, 128))


def listed():
    return [
        # one step of 64 chats: a token each, a few finished chats replaced by new ones
        {"name": "plan_step_64", "family": "plan", "seqs": 64, "tokens": 64, "page": 16,
         "new": False, "tight": False},
        # 127 new prompts, 262139 tokens in all, more than the free pages can hold
        {"name": "plan_prompts_262139", "family": "plan", "seqs": 127, "tokens": 262139,
         "page": 16, "new": True, "tight": True},
        # one chat's next token
        {"name": "append_one_token", "family": "append", "step": True, "seqs": 1, "drafts": 0,
         "tokens": 1, "hq": 16, "hkv": 4, "hd": 64, "page": 16, "norm": True, "with_q": True,
         "interleaved": False},
        # 64 sequences with three drafted tokens each: q, k and v in one call
        {"name": "append_drafts_64", "family": "append", "step": True, "seqs": 64, "drafts": 3,
         "tokens": 256, "hq": 32, "hkv": 8, "hd": 128, "page": 16, "norm": True, "with_q": True,
         "interleaved": False},
        # four prompts, 8191 tokens in all
        {"name": "append_prompts_8191", "family": "append", "step": False, "seqs": 4, "drafts": 0,
         "tokens": 8191, "hq": 16, "hkv": 2, "hd": 128, "page": 64, "norm": False,
         "with_q": False, "interleaved": True},
        # one chat's next token, about a thousand tokens in
        {"name": "attn_chat", "family": "attn", "seqs": 1, "drafts": 0, "longest": 1023,
         "even": True, "hq": 16, "hkv": 4, "hd": 64, "page": 16, "window": 0, "cap": 0.0,
         "slopes": False},
        # 64 sequences of any length up to 4096 with three drafted tokens each, capped scores
        {"name": "attn_drafts_64", "family": "attn", "seqs": 64, "drafts": 3, "longest": 4096,
         "even": False, "hq": 32, "hkv": 8, "hd": 128, "page": 16, "window": 0, "cap": 50.0,
         "slopes": False},
        # 16 sequences with seven drafted tokens each, windowed, with a distance bias
        {"name": "attn_window_16", "family": "attn", "seqs": 16, "drafts": 7, "longest": 16384,
         "even": True, "hq": 16, "hkv": 4, "hd": 64, "page": 32, "window": 4096, "cap": 0.0,
         "slopes": True},
        # four sequences of 131072 tokens: long documents
        {"name": "attn_long_4", "family": "attn", "seqs": 4, "drafts": 0, "longest": 131072,
         "even": True, "hq": 32, "hkv": 8, "hd": 128, "page": 64, "window": 0, "cap": 0.0,
         "slopes": False},
        # four drafted tokens of one chat, C1's vocabulary
        {"name": "verify_chat", "family": "verify", "seqs": 1, "drafts": 4, "vocab": 32000,
         "greedy": False, "probs": True},
        # greedy verification of 64 sequences' drafts, C1's vocabulary
        {"name": "verify_greedy_64", "family": "verify", "seqs": 64, "drafts": 3, "vocab": 32000,
         "greedy": True, "probs": False},
        # four drafted tokens each of 64 sequences, a large vocabulary
        {"name": "verify_batch_64", "family": "verify", "seqs": 64, "drafts": 4,
         "vocab": 128256, "greedy": False, "probs": True},
    ]


def _log(rng, lo, hi):
    """A whole number of [lo, hi], spread over the logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    family = rng.choice(("plan", "append", "attn", "attn", "verify"))
    hq, hkv, hd = rng.choice(HEADS)
    heads = {"hq": hq, "hkv": hkv, "hd": hd}
    c = {"family": family}
    if family == "plan":
        new = rng.random() < 0.5
        seqs = _log(rng, 1, 512)
        c.update(seqs=seqs, tokens=_log(rng, seqs, 262139) if new else seqs * rng.randint(1, 8),
                 page=rng.choice((16, 32, 64, 256)), new=new, tight=rng.random() < 0.3)
    elif family == "append":
        step = rng.random() < 0.5
        seqs = _log(rng, 1, 128) if step else rng.randint(1, 8)
        drafts = rng.randint(0, 7) if step else 0
        c.update(step=step, seqs=seqs, drafts=drafts,
                 tokens=seqs * (drafts + 1) if step else _log(rng, seqs, 8191),
                 page=rng.choice((16, 64, 128)), norm=rng.random() < 0.6,
                 with_q=step or rng.random() < 0.4, interleaved=rng.random() < 0.3, **heads)
    elif family == "attn":
        seqs, drafts = _log(rng, 1, 64), rng.choice((0, 0, rng.randint(1, 7)))
        c.update(seqs=seqs, drafts=drafts, longest=_log(rng, drafts + 1, 262144 // seqs),
                 even=rng.random() < 0.4, page=rng.choice((16, 32, 64, 256)),
                 window=rng.choice((0, 0, 0, 512)), cap=rng.choice((0.0, 0.0, 50.0)),
                 slopes=rng.random() < 0.25, **heads)
    else:
        seqs, drafts = _log(rng, 1, 64), rng.randint(1, 8)
        most = min(128256, 64 * 5 * 128256 // (seqs * (drafts + 1)))
        c.update(seqs=seqs, drafts=drafts, vocab=_log(rng, 1000, most),
                 greedy=rng.random() < 0.25, probs=rng.random() < 0.7)
    return c


# ----------------------------------------------------------------------- inputs
def _cuts(total, parts, g):
    """`parts` lengths of at least 1 that sum to `total`, as their running sums from 0."""
    inner = torch.randperm(total - 1, generator=g)[:parts - 1].sort().values + 1
    return torch.cat([torch.zeros(1, dtype=torch.long), inner, torch.tensor([total])])


def _heads_slopes(hq):
    """One slope per head: a geometric series from 2^(-8/hq) to 2^-8."""
    return [2.0 ** (-8.0 * (h + 1) / hq) for h in range(hq)]


def _up(n, m):
    return (n + m - 1) // m


def prepare(c, seed):
    """Inputs, cache and page tables of one case, made from the seed."""
    g = torch.Generator(device=DEV).manual_seed(int(seed))
    host = torch.Generator().manual_seed(int(seed) + 1)
    f, B = c["family"], c["seqs"]

    def randn(*shape, std=1.0, mean=0.0):
        return torch.empty(shape, device=DEV).normal_(mean, std, generator=g)

    def i32(t):
        return t.to(torch.int32).to(DEV)

    s = {"case": c}
    if f == "plan":
        P, N = c["page"], c["tokens"]
        lens, base = torch.randint(1, 2049, (B,), generator=host), N // B
        new = base + (torch.arange(B) < N % B).long()
        over = (torch.rand(B, generator=host) < 1 / 16).long()
        if c["new"]:  # every sequence is a new prompt, of up to 2 N / B tokens, for a finished one
            more = torch.randint(0, base, (B // 2,), generator=host)
            new[:2 * (B // 2)] += torch.stack((more, -more), 1).flatten()
            over[:] = 1
        held = _up(lens, P)
        width = _up(max(2048, 2 * base + 1) if c["new"] else 2048 + base, P)
        need = _up(torch.where(over > 0, new, lens + new), P).clamp_min(held * (over == 0))
        spare = int(need.sum()) - int(held.sum())  # beside what the finished ones give back
        spare = max(3, spare - int(need.sum()) // 4) if c["tight"] else max(3, spare + 7)
        used = int(held.sum())
        ids = torch.randperm(used + spare, generator=host)
        table = torch.full((B, width), -1, dtype=torch.long)
        table[torch.arange(width) < held[:, None]] = ids[:used]
        free = torch.full((2 * B * width,), -1, dtype=torch.long)
        free[:spare] = ids[used:]
        s.update(lengths=i32(lens), new_tokens=i32(new), page_table=i32(table), held=i32(held),
                 free_pages=i32(free), n_free=i32(torch.tensor([spare])), reset=i32(over),
                 capacity=64 * _up(N, 64))
        return s
    if f == "verify":
        K, V = c["drafts"], c["vocab"]
        s["logits"] = randn(B, K + 1, V, std=2.5)
        # a smaller model's opinion of the same rows, and tokens drawn from it
        drafts = s["logits"][:, :K] + randn(B, K, V)
        noise = torch.rand(B, K, V, generator=g, device=DEV).clamp_min(1e-20).log().neg().log()
        if c["greedy"]:
            s["draft_tokens"] = drafts.argmax(-1).int()
        else:
            s["draft_tokens"] = (drafts / TEMPERATURE - noise).argmax(-1).int()
        s["draft_probs"] = torch.softmax(drafts / TEMPERATURE, -1) if c["probs"] else None
        s["u"] = torch.rand(B, K + 1, generator=g, device=DEV)
        s["counts"] = i32(torch.randint(K // 2, K + 1, (B,), generator=host))
        s["temperature"] = 0.0 if c["greedy"] else TEMPERATURE
        return s
    hq, hkv, hd, P, T = c["hq"], c["hkv"], c["hd"], c["page"], c["drafts"] + 1
    if f == "append":
        N = c["tokens"]
        # rows of one fused projection: q | k | v side by side
        row = randn(N, (hq + 2 * hkv) * hd).to(BF16)
        q, k, v = row.split([hq * hd, hkv * hd, hkv * hd], dim=1)
        s.update(q=q.view(-1, hq, hd), k=k.view(-1, hkv, hd), v=v.view(-1, hkv, hd))
        s["inv_freq"] = (10000.0 ** (-torch.arange(0, hd, 2, dtype=torch.float64) / hd)
                         ).float().to(DEV)
        for n in ("q_norm", "k_norm"):
            s[n] = randn(hd, std=0.1, mean=1.0) if c["norm"] else None
        if c["step"]:
            lens = torch.randint(T, 513, (B,), generator=host)
            new = torch.full((B,), T)
        else:
            cu = _cuts(N, B, host)
            lens = new = cu[1:] - cu[:-1]
        rows = torch.repeat_interleave(torch.arange(B), new)
        at = torch.arange(N) - (new.cumsum(0) - new)[rows]
        s.update(positions=i32((lens - new)[rows] + at), rows=i32(rows))
    else:
        low = max(T, c["longest"] - c["longest"] // 16) if c["even"] else T
        lens = torch.randint(low, c["longest"] + 1, (B,), generator=host)
        lens[0] = c["longest"]
        s["lengths"] = i32(lens)
        s["q"] = randn(B, T, hq, hd).to(BF16)
        s["slopes"] = torch.tensor(_heads_slopes(hq), device=DEV) if c["slopes"] else None
    # as many pages as any lengths of the case can fill, handed out in random order
    if f == "append" and not c["step"]:
        width, pages = _up(c["tokens"], P), c["tokens"] // P + B + 3
    else:
        width = _up(c["longest"] if f == "attn" else 512, P)
        pages = B * width + 3
    used = _up(lens, P)
    table = torch.zeros(B, width, dtype=torch.long)
    table[torch.arange(width) < used[:, None]] = torch.randperm(
        pages, generator=host)[:int(used.sum())]
    s["page_table"] = i32(table)
    for n in ("k", "v"):
        codes, scales = _stored(randn(pages, hkv, P, hd))
        s[n + "_cache"], s[n + "_scales"] = codes.view(FP4), scales.view(E8M0)
    return s


# ----------------------------------------------------------------------- plain forms
def _stored(x):
    """x [..., hd] in 32 bits as (codes [..., hd / 2], block scales [..., hd / 32]) bytes."""
    x = x.clamp(-1.5 * 2.0 ** 127, 1.5 * 2.0 ** 127).unflatten(-1, (-1, 32))
    most = x.abs().amax(-1, keepdim=True)
    m, e = torch.frexp(most)
    # the largest value lies at 7 steps of the scale or below: 6 after rounding
    e = torch.where(most > 0, e - 3 + (m > 0.875), -126).clamp_min(-126)
    y = torch.ldexp(x.abs(), -e)
    code = ((y > 0.25).to(torch.uint8) + (y >= 0.75) + (y > 1.25) + (y >= 1.75) + (y > 2.5)
            + (y >= 3.5) + (y > 5))
    code = (code | torch.signbit(x).to(torch.uint8) << 3).flatten(-2)
    lost = ~torch.isfinite(x.sum(-1))
    return (code[..., 0::2] | code[..., 1::2] << 4,
            torch.where(lost, 255, e.squeeze(-1) + 127).to(torch.uint8))


def _values(codes, scales):
    """What codes and scales (as bytes) stand for, in 32 bits."""
    table = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6, -0.0, -0.5, -1, -1.5, -2, -3, -4, -6],
                         device=DEV)
    x = torch.stack((table[(codes & 15).int()], table[(codes >> 4).int()]), -1).flatten(-2)
    return (x.unflatten(-1, (-1, 32)) * scales.view(E8M0).float()[..., None]).flatten(-2)


def _norm_rope(x, weight, positions, inv_freq, interleaved):
    """x [N, H, hd] in 32 bits: RMSNorm over hd (where weight is given), rotated pairs."""
    x = x.float()
    if weight is not None:
        x = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS) * weight
    angle = positions.double()[:, None] * inv_freq.double()
    cos, sin = angle.cos().float()[:, None], angle.sin().float()[:, None]
    if interleaved:
        a, b = x[..., 0::2], x[..., 1::2]
        return torch.stack((a * cos - b * sin, b * cos + a * sin), -1).flatten(-2)
    a, b = x.chunk(2, -1)
    return torch.cat((a * cos - b * sin, b * cos + a * sin), -1)


def _plain_plan(s):
    table, held, free = s["page_table"], s["held"].long(), s["free_pages"]
    over, P = s["reset"] != 0, s["case"]["page"]
    B, width = table.shape
    N, n0 = s["capacity"], s["n_free"].long()
    # pages of the sequences that start over go on top of the stack
    back = held * over
    at = n0 + back.cumsum(0)[:, None] - back[:, None] + torch.arange(width, device=DEV)
    gone = torch.arange(width, device=DEV) < back[:, None]
    stack = torch.cat((free, free.new_zeros(1)))
    stack.scatter_(0, torch.where(gone, at, len(free)).flatten(), table.flatten())
    n1, held = n0 + back.sum(), held - back
    lens = torch.where(over, 0, s["lengths"].long())
    new = s["new_tokens"].long()
    cu = torch.cat((n0 * 0, new.cumsum(0)))
    fits = (lens + new <= width * P) & (cu[1:] <= N)
    need = torch.where(fits & (new > 0), _up(lens + new, P) - held, 0).clamp_min(0)
    upto = need.cumsum(0)
    given = fits & ((need == 0) | (upto <= n1))
    got = need * given
    # the sequences' new pages come off the top, in their order
    i = torch.arange(width, device=DEV) - held[:, None]
    fresh = (i >= 0) & (i < got[:, None])
    at = torch.where(fresh, n1 - 1 - (upto - need)[:, None] - i, 0)
    table.copy_(torch.where(fresh, stack[at], table))
    s["free_pages"].copy_(stack[:-1])
    s["held"].copy_(held + got)
    s["n_free"].copy_(n1 - got.sum())
    j = torch.arange(N, device=DEV)
    rows = torch.searchsorted(cu, j, right=True) - 1
    inside = j < cu[-1]
    b = rows.clamp_max(B - 1)
    return {"cu_seqlens": cu.clamp_max(N).int(), "rows": torch.where(inside, rows, -1).int(),
            "positions": torch.where(inside & given[b], lens[b] + j - cu[b], -1).int(),
            "lengths": (lens + new * given).int(), "page_table": table, "held": s["held"],
            "free_pages": s["free_pages"], "n_free": s["n_free"]}


def _plain_append(s):
    c = s["case"]
    pos, rows = s["positions"].long(), s["rows"].long()
    page, slot = s["page_table"].long()[rows, pos // c["page"]], pos % c["page"]
    k = _norm_rope(s["k"], s["k_norm"], pos, s["inv_freq"], c["interleaved"])
    out = {}
    for n, x in (("k", k), ("v", s["v"].float())):
        codes, scales = _stored(x)
        cache, steps = s[n + "_cache"].view(torch.uint8), s[n + "_scales"].view(torch.uint8)
        cache[page, :, slot] = codes
        steps[page, :, slot] = scales
        out[n] = _values(cache[page, :, slot], steps[page, :, slot]).to(BF16)
    if c["with_q"]:
        out["q"] = _norm_rope(s["q"], s["q_norm"], pos, s["inv_freq"], c["interleaved"]).to(BF16)
    return out


def _gather(s, n):
    """The pages of each sequence in order: [B, H, tokens, hd] in 32 bits."""
    table = s["page_table"].long()
    x = _values(s[n + "_cache"].view(torch.uint8)[table], s[n + "_scales"].view(torch.uint8)[table])
    B, pages, H, P, hd = x.shape
    return x.permute(0, 2, 1, 3, 4).reshape(B, H, pages * P, hd)


def _plain_attn(s):
    c = s["case"]
    B, T, hq, hkv, hd = c["seqs"], c["drafts"] + 1, c["hq"], c["hkv"], c["hd"]
    k, v = _gather(s, "k"), _gather(s, "v")
    j = torch.arange(k.shape[2], device=DEV)
    # token t of a sequence stands at position length - T + t
    at = s["lengths"].long()[:, None, None] - T + torch.arange(T, device=DEV)[:, None]
    seen = j <= at
    if c["window"]:
        seen &= j > at - c["window"]
    # positions past a length hold whatever the page held: not part of the sum
    v = v.masked_fill(~seen.any(1)[:, None, :, None], 0.0)
    q = s["q"].float().view(B, T, hkv, hq // hkv, hd).permute(0, 2, 3, 1, 4)
    q = q.reshape(B, hkv, -1, hd) * hd ** -0.5
    z = torch.matmul(q, k.transpose(-1, -2).contiguous()).view(B, hkv, hq // hkv, T, -1)
    if c["cap"]:
        z = torch.tanh(z / c["cap"]) * c["cap"]
    if s["slopes"] is not None:
        z = z - s["slopes"].view(1, hkv, -1, 1, 1) * (at - j).float()[:, None, None]
    z = z.masked_fill_(~seen[:, None, None], -math.inf)
    p = z.sub_(z.amax(-1, keepdim=True).clamp_min(torch.finfo(z.dtype).min)).exp_()
    o = torch.matmul(p.view(B, hkv, -1, p.shape[-1]), v).view(B, hkv, hq // hkv, T, hd)
    o = o / p.sum(-1, keepdim=True).clamp_min(1e-30)
    return o.permute(0, 3, 1, 2, 4).reshape(B, T, hq, hd).to(BF16)


def _plain_verify(s):
    x, drafts, u = s["logits"], s["draft_tokens"].long(), s["u"].double()
    B, K = drafts.shape
    V = x.shape[-1]
    t, ids = torch.arange(K, device=DEV), torch.arange(V, device=DEV)
    there = t < s["counts"][:, None]
    top = x.amax(-1, keepdim=True)
    if s["temperature"] <= 0:
        best = torch.where(x == top, ids, V).amin(-1)
        accepted = ((drafts == best[:, :K]) & there).long().cumprod(1).sum(1)
        fresh = best.gather(1, accepted[:, None])
    else:
        # in 64 bits: the draw looks for a border among as many as V of them
        e = ((x.double() - top.double()) / s["temperature"]).exp_()
        p = e / e.sum(-1, keepdim=True)
        pd = p[:, :K].gather(2, drafts[..., None])[..., 0]
        qd = 1.0
        if s["draft_probs"] is not None:
            qd = s["draft_probs"].gather(2, drafts[..., None])[..., 0].double()
        accepted = ((u[:, :K] * qd < pd) & there).long().cumprod(1).sum(1)
        b, last = torch.arange(B, device=DEV), accepted.clamp_max(K - 1)
        if s["draft_probs"] is not None:
            less = s["draft_probs"][b, last].double()
        else:
            less = (ids == drafts[b, last][:, None]).double()
        pa = p[b, accepted]
        rest = (pa - less * (accepted < s["counts"])[:, None]).clamp_min(0)
        rest = torch.where(rest.sum(-1, keepdim=True) > 0, rest, pa)
        run_up = rest.cumsum(-1)
        fresh = (run_up <= u[:, K:] * run_up[:, -1:]).sum(-1)
        fresh = torch.minimum(fresh, torch.where(rest > 0, ids, 0).amax(-1))[:, None]
    t = torch.arange(K + 1, device=DEV)
    tokens = torch.where(t < accepted[:, None], torch.nn.functional.pad(drafts, (0, 1)),
                         torch.where(t == accepted[:, None], fresh, -1))
    return {"tokens": tokens.int(), "accepted": accepted.int()}


_PLAIN = {"plan": _plain_plan, "append": _plain_append, "attn": _plain_attn,
          "verify": _plain_verify}


def _own(s):
    from hybrid_llm_amd import ops
    c = s["case"]
    if c["family"] == "plan":
        cu, rows, positions, lengths = ops.paged_plan(
            s["lengths"], s["new_tokens"], s["page_table"], s["held"], s["free_pages"],
            s["n_free"], c["page"], s["capacity"], reset=s["reset"])
        return {"cu_seqlens": cu, "rows": rows, "positions": positions, "lengths": lengths,
                "page_table": s["page_table"], "held": s["held"],
                "free_pages": s["free_pages"], "n_free": s["n_free"]}
    if c["family"] == "verify":
        tokens, accepted = ops.verify_drafts(
            s["logits"], s["draft_tokens"], s["u"], temperature=s["temperature"],
            draft_probs=s["draft_probs"], counts=s["counts"])
        return {"tokens": tokens, "accepted": accepted}
    cache = (s["k_cache"], s["v_cache"], s["k_scales"], s["v_scales"], s["page_table"])
    if c["family"] == "attn":
        return ops.paged_attn_mx4(s["q"], *cache, s["lengths"], window=c["window"],
                                  softcap=c["cap"], slopes=s["slopes"])
    with_q = {"q": s["q"], "q_norm": s["q_norm"]} if c["with_q"] else {}
    q = ops.paged_kv_append_mx4(s["k"], s["v"], *cache, s["positions"], rows=s["rows"],
                                inv_freq=s["inv_freq"], k_norm=s["k_norm"], eps=EPS,
                                interleaved=c["interleaved"], **with_q)
    k, v = ops.paged_kv_read_mx4(*cache, s["positions"], rows=s["rows"])
    return {"k": k, "v": v, "q": q} if c["with_q"] else {"k": k, "v": v}


def run(s):
    return _own(s) if own else _PLAIN[s["case"]["family"]](s)


# ----------------------------------------------------------------------- necessary work
def _mean_keys(c, n):
    """Keys of a sequence of length n that any of its new tokens sees."""
    return min(n, c["window"] + c["drafts"]) if c["window"] else n


def work(c):
    f, B = c["family"], c["seqs"]
    if f == "plan":
        # the sequences' numbers, a page id in and out for each that changes hands, and the
        # tokens' two; finished sequences hold up to 2048 tokens, 1024 on average
        pages = _up(c["tokens"], c["page"]) if c["new"] else B // 16 + 1
        back = B * (1024 // c["page"]) // (1 if c["new"] else 16)
        return {"bytes": 28 * B + 8 * (pages + back) + 8 * c["tokens"], "flops": 0}
    if f == "verify":
        K, V = c["drafts"], c["vocab"]
        rows = B * (K + 1)
        # every target row, and the draft row that a rejected token's draw subtracts
        return {"bytes": 4 * V * (rows + (B if c["probs"] and not c["greedy"] else 0)),
                "flops": rows * V * (1 if c["greedy"] else 4)}
    hq, hkv, hd = c["hq"], c["hkv"], c["hd"]
    if f == "append":
        kv, q = 2 * c["tokens"] * hkv * hd, c["tokens"] * hq * hd if c["with_q"] else 0
        # bf16 in, 17 / 32 of a byte a value stored and read back, bf16 out
        return {"bytes": kv * (4 + 17 / 16) + 4 * q + 8 * c["tokens"], "flops": 10 * (kv + q)}
    longest, T = c["longest"], c["drafts"] + 1
    mean = longest - longest // 32 if c["even"] else (longest + T) / 2
    keys = _mean_keys(c, longest) + (B - 1) * _mean_keys(c, mean)
    return {"bytes": 2 * keys * hkv * hd * 17 / 32 + 4 * B * T * hq * hd,
            "flops": 4 * keys * T * hq * hd}


# ----------------------------------------------------------------------- 64-bit results
def _exact_rope(x, weight, positions, inv_freq, interleaved):
    """Each pair as a complex number times e^(i angle)."""
    x = x.double()
    if weight is not None:
        x = x / (x.pow(2).sum(-1, keepdim=True) / x.shape[-1] + EPS).sqrt() * weight.double()
    angle = torch.outer(positions.double(), inv_freq.double())[:, None]
    turn = torch.polar(torch.ones_like(angle), angle)
    if interleaved:
        z = torch.view_as_complex(x.unflatten(-1, (-1, 2)).contiguous()) * turn
        return torch.view_as_real(z).flatten(-2)
    half = x.shape[-1] // 2
    z = torch.complex(x[..., :half].contiguous(), x[..., half:].contiguous()) * turn
    return torch.cat((z.real, z.imag), -1)


def _exact_rounded(x):
    """The stored value nearest to x [N, H, hd], ties to the even code."""
    blocks = x.view(*x.shape[:-1], -1, 32)
    # the smallest power of two, 2^-126 or more, of which 7 cover the block's largest value
    power = torch.log2(blocks.abs().amax(-1, keepdim=True).clamp_min(2.0 ** -126) / 7).ceil()
    step = torch.exp2(power.clamp_min(-126))
    grid = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6], dtype=torch.float64, device=DEV)
    y = (blocks / step).abs()
    up = torch.searchsorted(grid, y.contiguous()).clamp(1, 7)
    low, high = grid[up - 1], grid[up]
    higher = (y - low > high - y) | ((y - low == high - y) & (up % 2 == 0))
    return (torch.where(higher, high, low) * step * blocks.sign()).view_as(x)


def _exact_pages(s, n, pages):
    """Pages [n pages] of a cache as [Hkv, tokens, hd] in 64 bits."""
    w = s[n + "_cache"].view(torch.uint8)[pages].long()
    code = torch.stack((w % 16, w // 16), -1).flatten(-2)
    e, m = code // 2 % 4, code % 2
    x = torch.where(e == 0, m / 2, (1 + m / 2) * 2.0 ** (e - 1)).double() * (1 - 2 * (code // 8))
    step = torch.exp2(s[n + "_scales"].view(torch.uint8)[pages].double() - 127)
    x = x * step.repeat_interleave(32, -1)
    return x.transpose(0, 1).flatten(1, 2)


def _exact_plan(s):
    lens, new, held, over = (s[n].tolist() for n in ("lengths", "new_tokens", "held", "reset"))
    table, free, P, N = s["page_table"].tolist(), s["free_pages"].tolist(), s["case"]["page"], \
        s["capacity"]
    top = int(s["n_free"])
    for b, h in enumerate(held):
        if over[b]:
            free[top:top + h] = table[b][:h]
            top, held[b], lens[b] = top + h, 0, 0
    cu, rows, positions, asked, room = [0], [-1] * N, [-1] * N, 0, top
    for b, n in enumerate(new):
        first, end = cu[-1], cu[-1] + n
        rows[first:end] = [b] * (min(end, N) - first)
        cu.append(end)
        if lens[b] + n > len(table[b]) * P or end > N:
            continue
        need = max(0, _up(lens[b] + n, P) - held[b]) if n else 0
        asked += need
        if need and asked > room:
            continue
        for _ in range(need):
            top -= 1
            table[b][held[b]] = free[top]
            held[b] += 1
        positions[first:end] = range(lens[b], lens[b] + n)
        lens[b] += n
    def i32(v):
        return torch.tensor(v, dtype=torch.int32)
    return {"cu_seqlens": i32([min(n, N) for n in cu]), "rows": i32(rows[:N]),
            "positions": i32(positions), "lengths": i32(lens), "page_table": i32(table),
            "held": i32(held), "free_pages": i32(free), "n_free": i32([top])}


def _exact_verify(s):
    u, counts, drafts = s["u"].tolist(), s["counts"].tolist(), s["draft_tokens"].tolist()
    tokens, accepted = [], []
    for b, ids in enumerate(drafts):
        K, out = len(ids), []
        for t in range(K + 1):
            row = s["logits"][b, t].double()
            if s["temperature"] <= 0:
                first = int((row == row.max()).nonzero()[0])
                out.append(first)
                if t == K or t >= counts[b] or ids[t] != first:
                    break
                continue
            p = torch.softmax(row / s["temperature"], 0)
            there = t < counts[b]
            q = torch.zeros_like(p)
            if there and s["draft_probs"] is not None:
                q = s["draft_probs"][b, t].double()
            elif there:
                q[ids[t]] = 1
            if there and u[b][t] * float(q[ids[t]]) < float(p[ids[t]]):
                out.append(ids[t])
                continue
            rest = torch.where(p > q, p - q, 0)
            rest = rest if float(rest.sum()) > 0 else p
            c = rest.cumsum(0)
            at = int(torch.searchsorted(c, float(c[-1]) * u[b][K], right=True))
            out.append(min(at, int(rest.nonzero()[-1])))
            break
        accepted.append(len(out) - 1)
        tokens.append(out + [-1] * (K + 1 - len(out)))
    return {"tokens": torch.tensor(tokens, dtype=torch.int32),
            "accepted": torch.tensor(accepted, dtype=torch.int32)}


def exact(c, seed):
    s = prepare(c, seed)
    f = c["family"]
    if f == "plan":
        return _exact_plan(s)
    if f == "verify":
        return _exact_verify(s)
    hq, hkv, hd = c["hq"], c["hkv"], c["hd"]
    if f == "append":
        pos = s["positions"]
        out = {"k": _exact_rounded(_exact_rope(s["k"], s["k_norm"], pos, s["inv_freq"],
                                               c["interleaved"])),
               "v": _exact_rounded(s["v"].double())}
        if c["with_q"]:
            out["q"] = _exact_rope(s["q"], s["q_norm"], pos, s["inv_freq"], c["interleaved"])
        return out
    B, T, P = c["seqs"], c["drafts"] + 1, c["page"]
    out = torch.empty(B, T, hq, hd, dtype=torch.float64, device=DEV)
    for b, n in enumerate(s["lengths"].tolist()):
        pages = s["page_table"][b, :_up(n, P)].long()
        k, v = (_exact_pages(s, x, pages)[:, :n] for x in ("k", "v"))
        for t in range(T):
            end = n - T + t + 1
            first = max(0, end - c["window"]) if c["window"] else 0
            far = torch.arange(end - first - 1, -1, -1, dtype=torch.float64, device=DEV)
            for h in range(hq):
                z = k[h * hkv // hq, first:end] @ s["q"][b, t, h].double() / math.sqrt(hd)
                if c["cap"]:
                    z = c["cap"] * torch.tanh(z / c["cap"])
                if s["slopes"] is not None:
                    z = z - s["slopes"][h].double() * far
                out[b, t, h] = torch.softmax(z, 0) @ v[h * hkv // hq, first:end]
    return out
