"""Attention over packed prompts against the 64-bit oracle, and the serving operators in
one run: prompts, append, then steps over the cache.

Tolerance (the bound of tests/test_gpu_paged.py): weights rounded to bf16 under the sum
of the rounded ones, 2^-8 of sum_j w_j |v_j - out|; scores in fp32 over hd <= 128 terms
of sum |q_d k_d| scale < 2^5, 2^-11 and the sum's as much again, 2^-10 of the same; one
store to bf16, 2^-8 of the value.
"""
import math

import pytest
import torch

from oracle import paged as ref

pytestmark = pytest.mark.gpu

BF16 = torch.bfloat16
HALF_BF16 = 2.0 ** -8


def _ops():
    from hybrid_llm_amd import ops
    return ops


def _ok(got, want, spread):
    tol = HALF_BF16 * want.abs() + (HALF_BF16 + 2.0 ** -10) * spread * (1 + HALF_BF16) + 1e-30
    err = (got.double() - want).abs()
    assert bool((err <= tol).all()), float((err / tol).nan_to_num(1e9).max())


def _inputs(N, Hq, Hkv, hd, seed):
    g = torch.Generator().manual_seed(seed)
    row = torch.randn(N, (Hq + 2 * Hkv) * hd, generator=g).to(BF16)
    return g, [t.view(N, -1, hd) for t in row.split([Hq * hd, Hkv * hd, Hkv * hd], 1)]


def _both(q, k, v, cu, **kw):
    dev = {n: t.cuda() if torch.is_tensor(t) else t for n, t in kw.items()}
    row = torch.cat([t.flatten(1) for t in (q, k, v)], 1).cuda()  # one fused projection
    qd, kd, vd = (t.view(t.shape[0], -1, q.shape[2])
                  for t in row.split([q[0].numel(), k[0].numel(), v[0].numel()], 1))
    got = _ops().packed_attn_prefill(qd, kd, vd, cu.cuda(), **dev)
    want, spread = ref.packed_prefill(q, k, v, cu, **kw)
    return got.cpu(), want, spread


def _cu(lens):
    return torch.tensor([0] + lens, dtype=torch.int32).cumsum(0).to(torch.int32)


DOCS = [
    [1], [2], [31], [32], [33], [127, 1, 1], [64, 64, 64], [200], [0, 5, 0, 0, 130, 1, 0, 65],
    [1] * 150, [300, 17],
]


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("lens", DOCS, ids=str)
def test_documents(lens, hd):
    _, (q, k, v) = _inputs(sum(lens), 4, 2, hd, len(lens) + hd)
    _ok(*_both(q, k, v, _cu(lens)))


@pytest.mark.parametrize("Hq,Hkv,hd", [(1, 1, 64), (3, 3, 128), (7, 1, 64), (16, 2, 64),
                                       (20, 5, 128)])
def test_head_layouts(Hq, Hkv, hd):
    _, (q, k, v) = _inputs(141, Hq, Hkv, hd, Hq)
    _ok(*_both(q, k, v, _cu([100, 41])))


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("kw", [
    {"window": 1}, {"window": 32}, {"window": 45}, {"window": 1000}, {"softcap": 2.0},
    {"softcap": 50.0}, {"slopes": True}, {"prefix": [40, 500, 0, 3]}, {"prefix": [0, -9, 64, 65]},
    {"window": 20, "prefix": [90, 64, 1, 30]}, {"scale": 0.0},
    {"window": 70, "softcap": 4.0, "slopes": True, "prefix": [10, 70, 0, 200], "scale": 0.2},
], ids=str)
def test_options(kw, hd):
    g, (q, k, v) = _inputs(391, 4, 1, hd, 7)
    kw = dict(kw)
    if kw.pop("slopes", False):
        kw["slopes"] = torch.rand(4, generator=g) * 0.5
    if "prefix" in kw:
        kw["prefix"] = torch.tensor(kw["prefix"], dtype=torch.int32)
    _ok(*_both(q, k, v, _cu([97, 200, 1, 93]), **kw))


@pytest.mark.parametrize("hd", [64, 128])
def test_longer_prompt(hd):
    _, (q, k, v) = _inputs(1500, 2, 1, hd, 3)
    _ok(*_both(q * 2, k, v, _cu([1400, 100])))


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("kw", [{}, {"softcap": 10.0}, {"slopes": True, "window": 150},
                                {"prefix": [100, 0, 150, 9, 400, 1]}], ids=str)
def test_many_heads(kw, hd):
    """Enough rows and heads for workgroups of 64 rows (fewer give 32-row ones)."""
    g, (q, k, v) = _inputs(640, 64, 2, hd, 4)
    kw = dict(kw)
    if kw.pop("slopes", False):
        kw["slopes"] = torch.rand(64, generator=g) * 0.1
    if "prefix" in kw:
        kw["prefix"] = torch.tensor(kw["prefix"], dtype=torch.int32)
    _ok(*_both(q, k, v, _cu([130, 1, 200, 0, 290, 19]), **kw))


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("kw", [
    {}, {"softcap": 10.0}, {"slopes": True}, {"slopes": True, "window": 150},
    {"prefix": [100, 0, 150, 9, 400]}, {"window": 33},
    {"slopes": True, "softcap": 8.0, "prefix": [3, 1, 650, 0, 7]}], ids=str)
def test_rows_and_heads_for_whole_workgroups(kw, hd):
    """Over two 128-row workgroups a compute unit, each wave takes its rows alone; rows
    past the last document are left."""
    g, (q, k, v) = _inputs(1170, 64, 2, hd, 14)
    kw = dict(kw)
    if kw.pop("slopes", False):
        kw["slopes"] = torch.rand(64, generator=g) * 0.1
    if "prefix" in kw:
        kw["prefix"] = torch.tensor(kw["prefix"], dtype=torch.int32)
    cu = _cu([130, 1, 700, 0, 290])
    dev = {n: t.cuda() if torch.is_tensor(t) else t for n, t in kw.items()}
    out = torch.full((1170, 64, hd), 9.0, dtype=BF16, device="cuda")
    _ops().packed_attn_prefill(q.cuda(), k.cuda(), v.cuda(), cu.cuda(), out=out, **dev)
    heads = [0, 31, 32, 63]
    if "slopes" in kw:
        kw["slopes"] = kw["slopes"][heads]
    want, spread = ref.packed_prefill(q[:1121, heads], k[:1121], v[:1121], cu, **kw)
    _ok(out[:1121, heads].cpu(), want, spread)
    assert (out[1121:] == 9.0).all()


@pytest.mark.parametrize("heads", [8, 256])
@pytest.mark.parametrize("kw", [{}, {"softcap": 20.0}, {"prefix": [40, 0]}], ids=str)
def test_largest_slopes(kw, heads):
    """Past 1024 they count as 1024: one key is left, the nearest or the farthest one."""
    _, (q, k, v) = _inputs(300, heads, 2, 64, 15)
    top = torch.finfo(torch.float32).max
    slopes = torch.tensor([top, -top, 1e7, -1e7, 2048.0, -2000.0, 500.0, -0.25])
    kw = {n: torch.tensor(x, dtype=torch.int32) if n == "prefix" else x for n, x in kw.items()}
    cu = _cu([290, 10])
    got = _ops().packed_attn_prefill(
        q.cuda(), k.cuda(), v.cuda(), cu.cuda(), slopes=slopes.repeat(heads // 8).cuda(),
        **{n: t.cuda() if torch.is_tensor(t) else t for n, t in kw.items()}).cpu()
    at = list(range(4)) + list(range(heads - 4, heads))  # four heads of either key-value head
    want, spread = ref.packed_prefill(q[:, at], k, v, cu, slopes=slopes.clamp(-1024, 1024), **kw)
    _ok(got[:, at], want, spread)


def test_more_documents_than_fit_the_table():
    """Over 511 documents the bounds are bisected in memory."""
    _, (q, k, v) = _inputs(900, 2, 1, 64, 5)
    _ok(*_both(q, k, v, _cu([1] * 300 + [0] * 20 + [2] * 300)))


def test_rows_of_no_document_are_left():
    _, (q, k, v) = _inputs(200, 4, 2, 64, 5)
    for t in (q, k, v):  # what they hold reaches nobody
        t[:10] = math.nan
        t[150:] = math.inf
    cu = torch.tensor([10, 60, 60, 150], dtype=torch.int32)
    out = torch.full((200, 4, 64), 9.0, dtype=BF16, device="cuda")
    got = _ops().packed_attn_prefill(q.cuda(), k.cuda(), v.cuda(), cu.cuda(), out=out).cpu()
    want, spread = ref.packed_prefill(q, k, v, cu)
    assert (got[:10] == 9.0).all() and (got[150:] == 9.0).all()
    _ok(got[10:150], want[10:150], spread[10:150])


@pytest.mark.parametrize("heads", [2, 128])
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
def test_values_that_are_not_finite_reach_only_rows_that_see_them(bad, hd, heads):
    """In v: the dims of rows that see the key; in k: every dim of such rows (a NaN score);
    windowed, prefixed and other documents' rows do not."""
    lens = [70, 90, 40]
    prefix = torch.tensor([0, 30, 0], dtype=torch.int32)
    _, (q, k, v) = _inputs(200, heads, 1, hd, 6)
    v[40, 0, 5] = bad
    v[120, 0, hd - 1] = bad
    v[120, 0, 7] = -bad
    k[165] = math.nan
    cu = _cu(lens)
    kw = {"window": 25, "prefix": prefix}
    got, _, _ = _both(q, k, v, cu, **kw)
    i, j = torch.arange(200)[:, None], torch.arange(200)
    doc = torch.bucketize(torch.arange(200), cu[1:].long(), right=True)
    sees = (doc[:, None] == doc) & ((j <= i) | (j < (cu.long()[doc] + prefix[doc])[:, None]))
    sees &= i - j < 25
    clean_v, clean_k = v.clone(), k.clone()
    for r, d in ((40, 5), (120, hd - 1), (120, 7)):
        clean_v[r, 0, d] = 0
    clean_k[165] = 0
    want, spread = ref.packed_prefill(q, clean_k, clean_v, cu, **kw)
    hit = torch.zeros(200, heads, hd, dtype=torch.bool)
    for r, d, x in ((40, 5, bad), (120, hd - 1, bad), (120, 7, -bad)):
        rows = sees[:, r]
        hit[rows, :, d] = True
        cell = got[rows][..., d].float()
        assert cell.isnan().all() if x != x else (cell == x).all()
    rows = sees[:, 165]
    assert got[rows].isnan().all()
    hit[rows] = True
    _ok(torch.where(hit, want.to(BF16), got), want, spread)


@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
def test_values_that_are_not_finite_in_whole_workgroups(bad):
    test_values_that_are_not_finite_reach_only_rows_that_see_them(bad, 64, 300)


@pytest.mark.parametrize("heads", [1, 8, 128, 180])
def test_infinite_scores_stay_with_their_rows(heads):
    """A key of infinities makes the rows that see it NaN, in every split of the keys; rows
    before it are those of the finite keys."""
    _, (q, k, v) = _inputs(300, heads, 1, 64, 16)
    k[250] = math.inf
    got = _ops().packed_attn_prefill(q.cuda(), k.cuda(), v.cuda(), _cu([300]).cuda()).cpu()
    want, spread = ref.packed_prefill(q[:250], k[:250], v[:250], _cu([250]))
    _ok(got[:250], want, spread)
    assert got[250:].isnan().all()


def test_one_visible_key_is_returned_exactly():
    _, (q, k, v) = _inputs(77, 6, 3, 128, 8)
    got = _ops().packed_attn_prefill(q.cuda(), k.cuda(), v.cuda(), _cu([50, 27]).cuda(), window=1)
    assert torch.equal(got.cpu(), v.repeat_interleave(2, 1))


def test_nothing_to_do():
    _, (q, k, v) = _inputs(9, 2, 2, 64, 1)
    out = torch.full((9, 2, 64), 3.0, dtype=BF16, device="cuda")
    zero = torch.zeros(1, dtype=torch.int32, device="cuda")
    _ops().packed_attn_prefill(q.cuda(), k.cuda(), v.cuda(), zero, out=out)
    _ops().packed_attn_prefill(q.cuda(), k.cuda(), v.cuda(),
                               torch.zeros(4, dtype=torch.int32).cuda(), out=out)
    assert (out == 3.0).all()
    e = q[:0].cuda()
    assert _ops().packed_attn_prefill(e, e, e, zero).shape == (0, 2, 64)


def test_matches_the_banded_kernel():
    """One document under a window of equal heads is banded attention."""
    _, (q, k, v) = _inputs(700, 4, 4, 64, 2)
    q, k, v = (t.contiguous().cuda() for t in (q, k, v))
    a = _ops().packed_attn_prefill(q, k, v, _cu([700]).cuda(), window=128)
    b = _ops().banded_attn_prefill(q[None], k[None], v[None], 128)[0]
    assert (a.float() - b.float()).abs().max() <= 2 * HALF_BF16 * b.float().abs().max()


def test_last_row_equals_the_cached_step():
    """A prompt's last row equals a step over its cache, to both calls' rounding."""
    ops = _ops()
    g, (q, k, v) = _inputs(333, 8, 2, 128, 9)
    q, k, v = (t.cuda() for t in (q, k, v))
    kw = {"window": 200, "softcap": 20.0, "slopes": (torch.rand(8, generator=g) * 0.1).cuda()}
    rows = ops.packed_attn_prefill(q, k, v, _cu([333]).cuda(), **kw)
    table = torch.randperm(21, generator=g).view(1, 21).to(torch.int32).cuda()
    kc = torch.zeros(21, 2, 16, 128, dtype=BF16, device="cuda")
    vc = torch.zeros_like(kc)
    pos = torch.arange(333, dtype=torch.int32, device="cuda")
    ops.paged_kv_append(k, v, kc, vc, table, pos, rows=torch.zeros_like(pos))
    step = ops.paged_attn_decode(q[332:], kc, vc, table, pos[-1:] + 1, **kw)
    want, spread = ref.packed_prefill(q.cpu(), k.cpu(), v.cpu(), _cu([333]),
                                      **{n: t.cpu() if torch.is_tensor(t) else t
                                         for n, t in kw.items()})
    _ok(rows[332:].cpu(), want[332:], spread[332:])
    _ok(step.cpu(), want[332:], spread[332:])


@pytest.mark.parametrize("fp8", [False, True])
def test_prompts_then_steps(fp8):
    """A batch as it is served: rotated, normed prompts into the cache and through packed
    attention, then steps of append and paged attention, each against 64-bit attention over
    the rows that the cache holds."""
    ops = _ops()
    g = torch.Generator().manual_seed(21)
    B, Hq, Hkv, hd, page, steps = 3, 8, 2, 64, 16, 4
    lens = [40, 1, 77]
    N, width = sum(lens), 6
    f = (10000.0 ** (-torch.arange(0, hd, 2, dtype=torch.float64) / hd)).float().cuda()
    qw, kw = (torch.rand(hd, generator=g).cuda() + 0.5 for _ in range(2))
    table = torch.randperm(B * width, generator=g).view(B, width).to(torch.int32).cuda()
    dt, ks, vs = (torch.float8_e4m3fn, 0.02, 0.02) if fp8 else (BF16, 1.0, 1.0)
    kc = torch.zeros(B * width, Hkv, page, hd, device="cuda").to(dt)
    vc = torch.zeros_like(kc)
    common = dict(inv_freq=f, k_norm=kw, q_norm=qw, k_scale=ks, v_scale=vs)

    def project(n):
        row = torch.randn(n, (Hq + 2 * Hkv) * hd, generator=g).to(BF16).cuda()
        return (t.view(n, -1, hd) for t in row.split([Hq * hd, Hkv * hd, Hkv * hd], 1))

    rows = torch.repeat_interleave(torch.arange(B), torch.tensor(lens))
    pos = torch.cat([torch.arange(n) for n in lens]).to(torch.int32).cuda()
    q, k, v = project(N)
    qr = ops.paged_kv_append(k, v, kc, vc, table, pos, rows=rows.to(torch.int32).cuda(), q=q,
                             **common)
    q2, k2 = ops.qk_norm_rope(q, k, pos, f, q_norm=qw, k_norm=kw)
    assert torch.equal(q2, qr)
    out = ops.packed_attn_prefill(qr, k2, v, _cu(lens).cuda())
    want, spread = ref.packed_prefill(qr.cpu(), k2.cpu(), v.cpu(), _cu(lens))
    _ok(out.cpu(), want, spread)
    for t in range(steps):
        at = torch.tensor(lens, dtype=torch.int32).cuda() + t
        q, k, v = project(B)
        qr = ops.paged_kv_append(k, v, kc, vc, table, at, q=q, **common)
        out = ops.paged_attn_decode(qr, kc, vc, table, at + 1, k_scale=ks, v_scale=vs)
        want, spread = ref.paged_decode(qr.cpu(), kc.cpu(), vc.cpu(), table.cpu(), at.cpu() + 1,
                                        k_scale=ks, v_scale=vs)
        _ok(out.cpu(), want, spread)


def test_captured_and_replayed():
    """Captured once, replayed on new rows and documents, equal to the eager call."""
    ops = _ops()
    g = torch.Generator(device="cuda").manual_seed(3)
    row = torch.zeros(300, 8 * 64, dtype=BF16, device="cuda")
    cu = torch.tensor([0, 100, 300], dtype=torch.int32, device="cuda")

    def call():
        q, k, v = (t.view(300, -1, 64) for t in row.split([256, 128, 128], 1))
        return ops.packed_attn_prefill(q, k, v, cu, softcap=30.0)

    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        call()
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = call()
    for ends in ([0, 100, 300], [0, 1, 300], [0, 300, 300]):
        row.copy_(torch.randn(row.shape, device="cuda", generator=g).to(BF16))
        cu.copy_(torch.tensor(ends, dtype=torch.int32))
        graph.replay()
        want = call()
        torch.cuda.synchronize()
        assert torch.equal(out, want)
