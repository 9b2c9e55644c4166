"""Rotated rows, the paged cache and its one-token attention against 64-bit oracles.

Tolerances are sums of what the kernels round.  A store to bf16 is off by at most
2^-8 of the value (half of torch.finfo(bfloat16).eps), to e4m3 by 2^-4 of a normal
value and 2^-10 below (half the subnormal step 2^-9).

norm_rope: the fp32 path before the store: the sum of squares of hd <= 128 values in
a tree of at most 12 additions and its root, weight and two products, 2^-20 of the
value together; the angle's fraction of a turn in fp32, 2^-25 turns or 2^-22 of a
radian, and sincospi within 2^-22.  Under 2^-19 of the row's largest value.

attention: weights w_j are rounded to bf16 at the worst (2^-8 each) and divided by their
sum, so the result moves by at most 2^-8 sum_j w_j |v_j - out|.  Scores in
fp32: the products of hd <= 128 terms, sum |q_d k_d| scale <= 2^5 on these inputs, off
by 2^-24 * 132 * 2^5 < 2^-11; exp2 and the cap add under 2^-16.  A score's error e moves a
weight by e, twice that with the sum's: 2^-10 of the same spread.  Then one store.
"""
import math

import pytest
import torch

from oracle import paged as ref

pytestmark = pytest.mark.gpu

BF16, FP8 = torch.bfloat16, torch.float8_e4m3fn
HALF_BF16, HALF_E4M3, SUB_E4M3 = 2.0 ** -8, 2.0 ** -4, 2.0 ** -10


def _ops():
    from hybrid_llm_amd import ops
    return ops


def _inv_freq(rot):
    return (10000.0 ** (-torch.arange(0, rot, 2, dtype=torch.float64) / max(rot, 1))).float()


def _rope_ok(got, want):
    want = want.double()
    tol = HALF_BF16 * want.abs() + 2.0 ** -19 * want.abs().amax(-1, keepdim=True)
    err = (got.double() - want).abs()
    assert bool((err <= tol).all()), float((err / tol.clamp_min(1e-30)).max())


def _attn_ok(got, want, spread):
    tol = HALF_BF16 * want.abs() + (HALF_BF16 + 2.0 ** -10) * spread * (1 + HALF_BF16) + 1e-30
    err = (got.double() - want).abs()
    assert bool((err <= tol).all()), float((err / tol).max())


# ----------------------------------------------------------------- norms and rotation
@pytest.mark.parametrize("N,Hq,Hkv,hd,rot,interleaved,normed", [
    (1, 16, 4, 64, 64, False, True),
    (3, 5, 1, 128, 128, True, True),
    (37, 16, 2, 128, 64, False, False),
    (129, 7, 7, 64, 24, True, True),
    (1003, 32, 8, 128, 128, False, True),
    (64, 4, 4, 64, 0, False, True),
    (5, 1, 1, 64, 8, False, False),
    (2000, 12, 3, 64, 40, False, True),
])
def test_qk_norm_rope(N, Hq, Hkv, hd, rot, interleaved, normed):
    g = torch.Generator().manual_seed(N + hd)
    row = torch.randn(N, (Hq + 2 * Hkv) * hd, generator=g).to(BF16)
    pos = torch.randint(0, 2 ** 20, (N,), generator=g, dtype=torch.int32)
    pos[0] = 2 ** 31 - 1
    f = _inv_freq(rot) if rot else None
    w = [torch.randn(hd, generator=g) + 1 if normed else None for _ in range(2)]
    d = row.cuda()
    q, k = d[:, :Hq * hd].view(N, Hq, hd), d[:, Hq * hd:(Hq + Hkv) * hd].view(N, Hkv, hd)
    dev = [None if t is None else t.cuda() for t in (f, *w)]
    qo, ko = _ops().qk_norm_rope(q, k, pos.cuda(), dev[0], q_norm=dev[1], k_norm=dev[2],
                                 interleaved=interleaved)
    for got, x, wt in ((qo, q, w[0]), (ko, k, w[1])):
        assert got.is_contiguous()
        _rope_ok(got.cpu(), ref.norm_rope(x.cpu(), pos, f, wt, 1e-6, interleaved))
    # in place on the projection's own rows: the same bits, the values untouched
    before = d.clone()
    _ops().qk_norm_rope(q, k, pos.cuda(), dev[0], q_norm=dev[1], k_norm=dev[2],
                        interleaved=interleaved, q_out=q, k_out=k)
    assert torch.equal(q, qo) and torch.equal(k, ko)
    assert torch.equal(d[:, (Hq + Hkv) * hd:], before[:, (Hq + Hkv) * hd:])


def test_norm_of_extreme_rows():
    """Zero rows stay zero (eps), rows at bf16's ends neither overflow where the 64-bit
    result is finite nor lose their sign; NaN stays in its own row."""
    x = torch.zeros(4, 2, 64)
    x[1] = 2.0 ** -60
    x[2] = torch.linspace(-1e15, 1e15, 64)
    x[3, 0] = math.nan
    x[3, 1] = 1.0
    x = x.to(BF16)
    pos = torch.tensor([0, 1, 2, 3], dtype=torch.int32)
    f, w = _inv_freq(64), torch.ones(64)
    qo, ko = _ops().qk_norm_rope(x.cuda(), x.cuda(), pos.cuda(), f.cuda(), q_norm=w.cuda())
    want = ref.norm_rope(x, pos, f, w)
    _rope_ok(qo[:3].cpu(), want[:3])
    assert qo[3, 0].isnan().all()
    _rope_ok(qo[3, 1:].cpu(), want[3, 1:])
    _rope_ok(ko[:3].cpu(), ref.norm_rope(x, pos, f)[:3])


def test_padding_rows_are_left():
    q = torch.randn(6, 4, 64).to(BF16).cuda()
    pos = torch.tensor([3, -1, 0, -7, 2, -2 ** 31], dtype=torch.int32).cuda()
    qo = torch.full_like(q, 7.0)
    ko = torch.full_like(q, 7.0)
    _ops().qk_norm_rope(q, q, pos, _inv_freq(64).cuda(), q_out=qo, k_out=ko)
    for o in (qo, ko):
        assert (o[[1, 3, 5]] == 7.0).all()
        assert not (o[[0, 2, 4]] == 7.0).all()


# ----------------------------------------------------------------- append
def _table(B, width, pages, g, rows_used=None):
    return torch.randperm(pages, generator=g)[:B * width].view(B, width).to(torch.int32)


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("N,Hq,Hkv,hd,page,with_q", [
    (1, 16, 4, 64, 16, True),
    (5, 8, 8, 64, 64, False),
    (61, 32, 8, 128, 16, True),
    (300, 6, 2, 128, 256, True),
    (2049, 3, 3, 64, 32, False),
])
def test_paged_kv_append(N, Hq, Hkv, hd, page, with_q, fp8):
    g = torch.Generator().manual_seed(N + page)
    B = 4
    lens = torch.tensor([N - N // 2 - N // 3, N // 3, 0, N // 2])
    rows = torch.repeat_interleave(torch.arange(B), lens).to(torch.int32)
    start = torch.tensor([0, 3, 9, 17])
    pos = torch.cat([torch.arange(int(n)) + int(s) for n, s in zip(lens, start)]).to(torch.int32)
    order = torch.randperm(N, generator=g)
    rows, pos = rows[order].contiguous(), pos[order].contiguous()
    width = int((lens + start).max() + page - 1) // page
    pages = B * width + 2
    table = _table(B, width, pages, g)
    row = torch.randn(N, (Hq + 2 * Hkv) * hd, generator=g).to(BF16)
    q, k, v = (t.view(N, -1, hd) for t in row.split([Hq * hd, Hkv * hd, Hkv * hd], 1))
    cache = torch.randn(2, pages, Hkv, page, hd, generator=g).to(FP8 if fp8 else BF16)
    ks, vs = (0.013, 0.25) if fp8 else (1.0, 1.0)
    f, kw, qw = _inv_freq(hd), torch.randn(hd, generator=g) + 1, torch.randn(hd, generator=g)
    dev = row.cuda()
    dq, dk, dv = (t.view(N, -1, hd) for t in dev.split([Hq * hd, Hkv * hd, Hkv * hd], 1))
    dc = cache.cuda()
    more = {"q": dq, "q_norm": qw.cuda()} if with_q else {}
    qo = _ops().paged_kv_append(dk, dv, dc[0], dc[1], table.cuda(), pos.cuda(), rows=rows.cuda(),
                                inv_freq=f.cuda(), k_norm=kw.cuda(), k_scale=ks, v_scale=vs,
                                **more)
    if with_q:
        _rope_ok(qo.cpu(), ref.norm_rope(q, pos, f, qw))
    else:
        assert qo is None
    kr = ref.norm_rope(k, pos, f, kw) / ks
    got = dc.cpu()
    written = torch.zeros(pages, page, dtype=torch.bool)
    for n, at in enumerate(ref.slots(table, rows, pos, page, pages)):
        pg, sl = at
        written[pg, sl] = True
        if fp8:
            for c, want in ((0, kr[n]), (1, v[n].double() / vs)):
                want = want.clamp(-ref.E4M3_MAX, ref.E4M3_MAX)
                err = (got[c][pg, :, sl].float().double() - want).abs()
                tol = (HALF_E4M3 * want.abs() + SUB_E4M3
                       + 2.0 ** -19 * want.abs().amax(-1, keepdim=True))
                assert bool((err <= tol).all())
        else:
            _rope_ok(got[0][pg, :, sl], kr[n])
            assert torch.equal(got[1][pg, :, sl], v[n])
    keep = ~written[:, None, :, None].expand(pages, Hkv, page, hd)
    for c in range(2):  # every other slot holds the bits that it held
        assert torch.equal(got[c].view(torch.uint8 if fp8 else torch.int16)[keep],
                           cache[c].view(torch.uint8 if fp8 else torch.int16)[keep])


def test_append_step_equals_qk_norm_rope():
    """rows None: token n belongs to page-table row n; the same bits as the unpaged call."""
    g = torch.Generator().manual_seed(5)
    B, Hq, Hkv, hd, page = 7, 8, 2, 64, 16
    row = torch.randn(B, (Hq + 2 * Hkv) * hd, generator=g).to(BF16).cuda()
    q, k, v = (t.view(B, -1, hd) for t in row.split([Hq * hd, Hkv * hd, Hkv * hd], 1))
    pos = torch.tensor([0, 1, 15, 16, 31, 47, 33], dtype=torch.int32).cuda()
    table = _table(B, 3, 3 * B, g).cuda()
    f, w = _inv_freq(32).cuda(), torch.randn(hd, generator=g).cuda()
    cache = torch.zeros(2, 3 * B, Hkv, page, hd, dtype=BF16, device="cuda")
    qo = _ops().paged_kv_append(k, v, cache[0], cache[1], table, pos, inv_freq=f, k_norm=w, q=q,
                                interleaved=True)
    q2, k2 = _ops().qk_norm_rope(q, k, pos, f, k_norm=w, interleaved=True)
    assert torch.equal(qo, q2)
    at = (table[torch.arange(B, device="cuda"), pos.long() // page].long(), pos.long() % page)
    assert torch.equal(cache[0][at[0], :, at[1]], k2)
    assert torch.equal(cache[1][at[0], :, at[1]], v)


@pytest.mark.parametrize("fp8", [False, True])
def test_tokens_without_a_slot_are_not_stored(fp8):
    dt = FP8 if fp8 else BF16
    k = torch.ones(8, 2, 64, dtype=BF16, device="cuda")
    table = torch.tensor([[0, 9, -1], [2, 1, 7]], dtype=torch.int32).cuda()
    # negative, past the table, page past the cache, page -1, rows outside; the last two stored
    pos = torch.tensor([-1, 48, 16, 40, 0, 0, 3, 20], dtype=torch.int32).cuda()
    rows = torch.tensor([0, 0, 0, 0, 2, -1, 0, 1], dtype=torch.int32).cuda()
    kc = torch.zeros(3, 2, 16, 64, dtype=dt, device="cuda")
    vc = torch.zeros_like(kc)
    q = torch.ones(8, 1, 64, dtype=BF16, device="cuda")
    qo = _ops().paged_kv_append(k, k, kc, vc, table, pos, rows=rows, q=q,
                                q_out=torch.full_like(q, 5.0))
    want = torch.zeros(3, 2, 16, 64)
    want[0, :, 3] = 1
    want[1, :, 4] = 1
    assert torch.equal(kc.float().cpu(), want) and torch.equal(vc.float().cpu(), want)
    assert (qo[0] == 5.0).all() and (qo[1:] == 1.0).all()


def test_e4m3_saturates_and_keeps_nan():
    x = torch.zeros(1, 1, 64)
    x[0, 0, :8] = torch.tensor([1e4, -1e4, math.inf, -math.inf, math.nan, 448.0, 460.0, 2e-3])
    x = x.to(BF16).cuda()
    kc = torch.zeros(1, 1, 16, 64, dtype=FP8, device="cuda")
    vc = torch.zeros_like(kc)
    zero = torch.zeros(1, dtype=torch.int32, device="cuda")
    _ops().paged_kv_append(x, x, kc, vc, zero.view(1, 1), zero, k_scale=1.0, v_scale=1.0)
    for c in (kc, vc):
        got = c[0, 0, 0, :8].float().cpu()
        assert got[:4].tolist() == [448.0, -448.0, 448.0, -448.0]
        assert math.isnan(got[4]) and got[5:7].tolist() == [448.0, 448.0]
        assert abs(got[7] - 2e-3) <= 2.0 ** -10


# ----------------------------------------------------------------- one-token attention
def _decode_case(B, Hq, Hkv, hd, page, lens, fp8, g, std=1.0):
    width = max(1, (max(lens) + page - 1) // page)
    pages = B * width + 2
    table = _table(B, width, pages, g)
    ks, vs = (0.02, 0.03) if fp8 else (1.0, 1.0)

    def cache(scale):
        x = torch.randn(pages, Hkv, page, hd, generator=g)
        return (x / scale).clamp(-448, 448).to(FP8) if fp8 else x.to(BF16)

    q = (torch.randn(B, Hq, hd, generator=g) * std).to(BF16)
    return q, cache(ks), cache(vs), table, torch.tensor(lens, dtype=torch.int32), ks, vs


def _decode_both(q, kc, vc, table, lens, ks, vs, **kw):
    dev = {n: t.cuda() if torch.is_tensor(t) else t for n, t in kw.items()}
    got = _ops().paged_attn_decode(q.cuda(), kc.cuda(), vc.cuda(), table.cuda(), lens.cuda(),
                                   k_scale=ks, v_scale=vs, **dev)
    want, spread = ref.paged_decode(q, kc, vc, table, lens, k_scale=ks, v_scale=vs, **kw)
    return got, want, spread


EDGES = [0, 1, 2, 15, 16, 17, 31, 32, 33, 63, 64, 65, 127, 128, 129, 255, 257]


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("Hq,Hkv,hd,page", [
    (4, 4, 64, 16), (16, 4, 64, 32), (8, 1, 128, 64), (7, 7, 128, 16), (40, 2, 64, 256),
    (32, 8, 128, 128), (17, 1, 128, 16),
])
def test_decode_edges(Hq, Hkv, hd, page, fp8):
    g = torch.Generator().manual_seed(Hq + hd)
    case = _decode_case(len(EDGES), Hq, Hkv, hd, page, EDGES, fp8, g)
    got, want, spread = _decode_both(*case)
    _attn_ok(got.cpu(), want, spread)
    assert (got[0] == 0).all()


@pytest.mark.parametrize("lens,page", [([1], 16), ([16], 16), ([100], 128), ([77, 3, 0], 64),
                                       ([0, 0], 16), ([512, 480, 1, 33], 16), ([1024, 1], 32),
                                       ([1025, 1000], 16)])
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("fp8", [False, True])
def test_decode_short_tables(lens, page, hd, fp8):
    """Around the table lengths up to which a workgroup takes a whole head (no second
    launch): 512 tokens for bf16 of 128 dims, else 1024."""
    g = torch.Generator().manual_seed(sum(lens) + hd)
    got, want, spread = _decode_both(*_decode_case(len(lens), 8, 2, hd, page, lens, fp8, g))
    _attn_ok(got.cpu(), want, spread)


@pytest.mark.parametrize("hd,fp8,n", [(64, False, 2048), (128, True, 2048), (64, True, 2064)])
def test_decode_many_heads_of_short_tables(hd, fp8, n):
    """128 heads and more: whole heads up to 2048 tokens."""
    g = torch.Generator().manual_seed(n + hd)
    lens = [n] + [(97 * i) % n for i in range(31)]
    case = _decode_case(32, 4, 4, hd, 16, lens, fp8, g)
    got, want, spread = _decode_both(*case, window=70)
    _attn_ok(got.cpu(), want, spread)


@pytest.mark.parametrize("lens", [[300], [5000, 40]])
def test_visible_infinities(lens):
    """A value of +inf, -inf or NaN that a query sees is what its dim becomes."""
    g = torch.Generator().manual_seed(17)
    q, kc, vc, table, n, ks, vs = _decode_case(len(lens), 8, 2, 64, 16, lens, False, g)
    want, spread = ref.paged_decode(q, kc, vc, table, n)
    for t, d, bad in ((7, 3, math.inf), (0, 5, -math.inf), (22, 6, math.nan), (8, 9, math.inf),
                      (9, 9, -math.inf)):
        vc[int(table[0, t // 16]), :, t % 16, d] = bad
    got = _ops().paged_attn_decode(q.cuda(), kc.cuda(), vc.cuda(), table.cuda(), n.cuda()).cpu()
    assert (got[0, :, 3] == math.inf).all() and (got[0, :, 5] == -math.inf).all()
    assert got[0, :, 6].isnan().all() and got[0, :, 9].isnan().all()
    for d in (3, 5, 6, 9):
        got[0, :, d] = want[0, :, d].to(BF16)
    _attn_ok(got, want, spread)


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("kw", [
    {"window": 1}, {"window": 33}, {"window": 200}, {"softcap": 2.0}, {"softcap": 50.0},
    {"slopes": True}, {"window": 100, "softcap": 5.0, "slopes": True, "scale": 0.3},
])
def test_decode_options(kw, hd, fp8):
    g = torch.Generator().manual_seed(11)
    kw = dict(kw)
    if kw.pop("slopes", False):
        kw["slopes"] = torch.rand(12, generator=g) * 0.5
    case = _decode_case(5, 12, 4, hd, 16, [700, 1, 0, 130, 300], fp8, g)
    got, want, spread = _decode_both(*case, **kw)
    _attn_ok(got.cpu(), want, spread)


@pytest.mark.parametrize("lens", [[300, 17], [5000, 40]])
def test_decode_largest_slopes(lens):
    """Past 1024 they count as 1024: one key is left, the nearest or the farthest one."""
    g = torch.Generator().manual_seed(18)
    case = _decode_case(2, 8, 2, 64, 16, lens, False, g)
    top = torch.finfo(torch.float32).max
    slopes = torch.tensor([top, -top, 1e7, -1e7, 2048.0, -2000.0, 500.0, -0.25])
    got, _, _ = _decode_both(*case, slopes=slopes)
    want, spread = ref.paged_decode(*case[:5], slopes=slopes.clamp(-1024, 1024))
    _attn_ok(got.cpu(), want, spread)


@pytest.mark.parametrize("B,lens", [
    (1, [20000]),                            # one sequence over many runs
    (3, [9000, 5, 6100]),                    # runs that end in one head and start in the next
    (130, [(37 * i) % 300 for i in range(130)]),  # more sequences than lanes
    (70, [0] * 30 + [500] + [0] * 38 + [260]),    # long stretches with nothing
])
def test_decode_split_and_join(B, lens):
    g = torch.Generator().manual_seed(B)
    got, want, spread = _decode_both(*_decode_case(B, 4, 2, 64, 64, lens, False, g, std=2.0))
    _attn_ok(got.cpu(), want, spread)


def test_one_visible_key_is_returned_exactly():
    g = torch.Generator().manual_seed(2)
    q, kc, vc, table, lens, ks, vs = _decode_case(2, 8, 2, 128, 16, [1, 150], False, g)
    got = _ops().paged_attn_decode(q.cuda(), kc.cuda(), vc.cuda(), table.cuda(), lens.cuda(),
                                   window=1)
    for b, n in enumerate([1, 150]):
        v = vc[int(table[b, (n - 1) // 16]), :, (n - 1) % 16]
        assert torch.equal(got[b].cpu(), v.repeat_interleave(4, 0))


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("poison", [math.nan, math.inf, 3.0e38])
def test_what_is_not_visible_has_no_effect(poison, fp8):
    """Slots past the length, before the window, of unnamed pages and of other pages."""
    if fp8 and poison == poison:
        poison = 448.0  # e4m3's largest
    g = torch.Generator().manual_seed(8)
    q, kc, vc, table, lens, ks, vs = _decode_case(4, 8, 2, 64, 16, [37, 200, 5, 160], fp8, g)
    table[1, 4] = -1
    table[1, 7] = kc.shape[0]
    table[3, 0] = 2 ** 31 - 1
    want, spread = ref.paged_decode(q, kc, vc, table, lens, window=120, k_scale=ks, v_scale=vs)
    seen = torch.zeros(kc.shape[0], 16, dtype=torch.bool)
    for b, n in enumerate(lens.tolist()):
        for t in range(max(0, n - 120), n):
            pg = int(table[b, t // 16])
            if 0 <= pg < kc.shape[0]:
                seen[pg, t % 16] = True
    hidden = ~seen[:, None, :, None].expand_as(kc)
    for c in (kc, vc):
        f = c.float()
        f[hidden] = poison
        c.copy_(f.to(c.dtype))
    got = _ops().paged_attn_decode(q.cuda(), kc.cuda(), vc.cuda(), table.cuda(), lens.cuda(),
                                   window=120, k_scale=ks, v_scale=vs)
    _attn_ok(got.cpu(), want, spread)


def test_no_named_page_gives_zeros():
    g = torch.Generator().manual_seed(9)
    q, kc, vc, table, lens, ks, vs = _decode_case(3, 4, 2, 64, 16, [300, 20, 129], False, g)
    table.fill_(-1)
    got = _ops().paged_attn_decode(q.cuda(), kc.cuda(), vc.cuda(), table.cuda(), lens.cuda())
    assert (got == 0).all()
    empty = kc[:0].cuda()
    got = _ops().paged_attn_decode(q.cuda(), empty, empty, table.cuda(), lens.cuda())
    assert (got == 0).all()


def test_lengths_outside_the_table():
    """Below 0 as 0, past the table's pages as the table's tokens."""
    g = torch.Generator().manual_seed(3)
    q, kc, vc, table, lens, ks, vs = _decode_case(3, 4, 4, 64, 16, [144, 144, 144], False, g)
    lens = torch.tensor([-5, 2 ** 31 - 1, 144], dtype=torch.int32)
    got, want, spread = _decode_both(q, kc, vc, table, lens, ks, vs)
    _attn_ok(got.cpu(), want, spread)
    assert (got[0] == 0).all()


def test_a_table_of_no_pages():
    q = torch.ones(3, 4, 64, dtype=BF16, device="cuda")
    c = torch.ones(2, 2, 16, 64, dtype=BF16, device="cuda")
    table = torch.zeros(3, 0, dtype=torch.int32, device="cuda")
    lens = torch.full((3,), 9, dtype=torch.int32, device="cuda")
    assert (_ops().paged_attn_decode(q, c, c, table, lens) == 0).all()
    pos = torch.zeros(3, dtype=torch.int32, device="cuda")
    before = c.clone()
    _ops().paged_kv_append(q[:, :2], q[:, :2], c, torch.zeros_like(c), table, pos)
    assert torch.equal(c, before)


def test_keys_and_values_in_one_cache():
    """One tensor as both caches is an ordinary read."""
    g = torch.Generator().manual_seed(14)
    q, kc, _, table, lens, ks, vs = _decode_case(2, 8, 1, 64, 16, [200, 31], False, g)
    one = kc.cuda()
    got = _ops().paged_attn_decode(q.cuda(), one, one, table.cuda(), lens.cuda())
    want, spread = ref.paged_decode(q, kc, kc, table, lens)
    _attn_ok(got.cpu(), want, spread)


@pytest.mark.parametrize("cap", [0.01, 1024.0])
def test_smallest_and_largest_cap(cap):
    """The cap's own error is 2^-23 of it: a score of the largest is off by 2^-13."""
    g = torch.Generator().manual_seed(15)
    got, want, spread = _decode_both(*_decode_case(2, 4, 2, 64, 16, [150, 40], False, g),
                                     softcap=cap)
    _attn_ok(got.cpu(), want, spread)


def test_strided_queries_and_given_buffers():
    g = torch.Generator().manual_seed(4)
    q, kc, vc, table, lens, ks, vs = _decode_case(6, 8, 2, 64, 32, [300, 7, 64, 190, 0, 222],
                                                  False, g)
    wide = torch.zeros(6, 12 * 64, dtype=BF16, device="cuda")
    wide[:, 128:128 + 512] = q.cuda().view(6, 512)
    qv = wide[:, 128:128 + 512].view(6, 8, 64)
    out = torch.empty(6, 8, 64, dtype=BF16, device="cuda")
    from hybrid_llm_amd import _lib
    n = _lib.load().llmy_paged_attn_workspace_bytes(6, 8, 2, 64, table.shape[1], 32, 0)
    ws = torch.full((n,), 255, dtype=torch.uint8, device="cuda")  # NaNs
    got = _ops().paged_attn_decode(qv, kc.cuda(), vc.cuda(), table.cuda(), lens.cuda(), out=out,
                                   workspace=ws)
    assert got is out
    want, spread = ref.paged_decode(q, kc, vc, table, lens)
    _attn_ok(got.cpu(), want, spread)


def test_large_scores():
    """Scores of thousands, of both signs: the maximum carries the exponents."""
    g = torch.Generator().manual_seed(6)
    q, kc, vc, table, lens, ks, vs = _decode_case(2, 4, 2, 64, 16, [500, 140], False, g)
    got, want, spread = _decode_both(q, kc, vc, table, lens, ks, vs, scale=64.0)
    # a score is off by at most 2^-24 (hd terms, scaling and the subtraction) of the sum of
    # its terms' magnitudes, under 64 * max|q| max|k| hd; a weight by e^(2 e) - 1
    total = 64.0 * 64 * float(q.abs().max()) * float(kc.abs().max())
    e = 2.0 ** -24 * (64 + 12) * total
    tol = (HALF_BF16 * want.abs() + (HALF_BF16 + math.expm1(2 * e)) * spread * (1 + HALF_BF16)
           + 1e-30)
    err = (got.cpu().double() - want).abs()
    assert bool((err <= tol).all()), float((err / tol).max())


def test_offsets_past_32_bits():
    """A cache of more than 2^32 bytes and 2^31 elements, its last pages in use."""
    pages = 2 ** 31 // (2 * 256 * 128) + 40
    kc = torch.empty(pages, 2, 256, 128, dtype=BF16, device="cuda")
    vc = torch.empty_like(kc)
    g = torch.Generator().manual_seed(1)
    table = torch.tensor([[pages - 1, 0], [pages - 3, pages - 2]], dtype=torch.int32)
    small = torch.randn(4, 2, 2, 256, 128, generator=g).to(BF16)
    for i, p in enumerate(table.view(-1).tolist()):
        kc[p].copy_(small[i, 0])
        vc[p].copy_(small[i, 1])
    q = torch.randn(2, 8, 128, generator=g).to(BF16)
    lens = torch.tensor([300, 511], dtype=torch.int32)
    # position 511 of sequence 1 and 300 of sequence 0 by an append
    new = torch.randn(2, 2, 2, 128, generator=g).to(BF16)
    _ops().paged_kv_append(new[0].cuda(), new[1].cuda(), kc, vc, table.cuda(), lens.cuda())
    small_table = torch.tensor([[0, 1], [2, 3]], dtype=torch.int32)
    for b, n in enumerate(lens.tolist()):
        small[2 * b + n // 256, 0][:, n % 256] = new[0, b]
        small[2 * b + n // 256, 1][:, n % 256] = new[1, b]
    got = _ops().paged_attn_decode(q.cuda(), kc, vc, table.cuda(), (lens + 1).cuda())
    want, spread = ref.paged_decode(q, small[:, 0], small[:, 1], small_table, lens + 1)
    _attn_ok(got.cpu(), want, spread)


def test_steps_in_a_captured_graph():
    """Append and attention captured as one step, replayed with new rows, positions and
    lengths: each replay equals the eager calls, with eager work in between."""
    ops = _ops()
    g = torch.Generator(device="cuda").manual_seed(3)
    B, Hq, Hkv, hd, page, width = 5, 8, 2, 64, 16, 20
    table = torch.randperm(B * width, device="cuda", generator=g).view(B, width).to(torch.int32)
    kc = torch.randn(B * width, Hkv, page, hd, device="cuda", generator=g).to(BF16)
    vc = torch.randn(B * width, Hkv, page, hd, device="cuda", generator=g).to(BF16)
    f = _inv_freq(hd).cuda()
    row = torch.zeros(B, (Hq + 2 * Hkv) * hd, dtype=BF16, device="cuda")
    pos = torch.zeros(B, dtype=torch.int32, device="cuda")

    def step(k_cache, v_cache):
        q, k, v = (t.view(B, -1, hd) for t in row.split([Hq * hd, Hkv * hd, Hkv * hd], 1))
        q = ops.paged_kv_append(k, v, k_cache, v_cache, table, pos, inv_freq=f, q=q)
        return ops.paged_attn_decode(q, k_cache, v_cache, table, pos + 1)

    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        step(kc.clone(), vc.clone())
    side.synchronize()
    gk, gv = kc.clone(), vc.clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(gk, gv)
    gk.copy_(kc)
    gv.copy_(vc)
    for i in range(4):
        row.copy_(torch.randn(row.shape, device="cuda", generator=g).to(BF16))
        pos.copy_(torch.tensor([i, 15 + i, 100 + i, 319 - i, 200], dtype=torch.int32))
        graph.replay()
        want = step(kc, vc)
        torch.cuda.synchronize()
        assert torch.equal(out, want) and torch.equal(gk, kc) and torch.equal(gv, vc)


def test_results_repeat_bit_for_bit():
    g = torch.Generator().manual_seed(12)
    q, kc, vc, table, lens, ks, vs = _decode_case(9, 16, 2, 128, 16, [1000 + 97 * i for i in range(9)],
                                                  False, g)
    args = [t.cuda() for t in (q, kc, vc, table, lens)]
    first = _ops().paged_attn_decode(*args)
    for _ in range(3):
        assert torch.equal(first, _ops().paged_attn_decode(*args))


def test_another_stream():
    """The call runs on the current stream, after what that stream holds."""
    g = torch.Generator().manual_seed(13)
    q, kc, vc, table, lens, ks, vs = _decode_case(2, 4, 2, 64, 16, [300, 40], False, g)
    want, spread = ref.paged_decode(q, kc, vc, table, lens)
    qd, kd, vd, td, ld = (t.cuda() for t in (q, kc, vc, table, lens))
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        late = torch.zeros_like(qd)
        torch.cuda._sleep(2_000_000)
        late.copy_(qd)
        got = _ops().paged_attn_decode(late, kd, vd, td, ld)
    s.synchronize()
    _attn_ok(got.cpu(), want, spread)


def test_two_streams_at_once():
    """Calls that overlap, each with a workspace of its own, do not disturb each other."""
    g = torch.Generator().manual_seed(18)
    cases = [_decode_case(3, 8, 2, 128, 16, [4000, 700 + i, 90], False, g) for i in range(2)]
    dev = [[t.cuda() for t in c[:5]] for c in cases]
    alone = [_ops().paged_attn_decode(*d) for d in dev]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in dev]
    got = [[], []]
    for _ in range(10):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(_ops().paged_attn_decode(*dev[i]))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(o, alone[i]) for o in got[i])


def test_row_offsets_past_32_bits():
    """Rows 2^21 elements apart, the last one past 2^31."""
    wide = torch.empty(1100, 2 ** 21, dtype=BF16, device="cuda")
    g = torch.Generator().manual_seed(19)
    small = torch.randn(1100, 6 * 64, generator=g).to(BF16)
    wide[:, 64:64 + 6 * 64] = small.cuda()
    q = wide[:, 64:64 + 256].view(1100, 4, 64)
    k = wide[:, 320:320 + 128].view(1100, 2, 64)
    pos = torch.arange(1100, dtype=torch.int32)
    f = _inv_freq(64)
    qo, ko = _ops().qk_norm_rope(q, k, pos.cuda(), f.cuda())
    _rope_ok(qo.cpu(), ref.norm_rope(small[:, :256].view(1100, 4, 64), pos, f))
    _rope_ok(ko.cpu(), ref.norm_rope(small[:, 256:].view(1100, 2, 64), pos, f))
    cu = torch.tensor([0, 1040, 1100], dtype=torch.int32)
    got = _ops().packed_attn_prefill(q, k, k, cu.cuda()).cpu()
    want, spread = ref.packed_prefill(small[1040:, :256].view(60, 4, 64),
                                      small[1040:, 256:].view(60, 2, 64),
                                      small[1040:, 256:].view(60, 2, 64),
                                      torch.tensor([0, 60], dtype=torch.int32))
    _attn_ok(got[1040:], want, spread)


def test_a_later_piece_of_a_prompt():
    """Rows appended behind a cached prefix, each as a sequence of its own over the same
    pages, are causal attention of the whole prompt's tail."""
    g = torch.Generator().manual_seed(20)
    n, tail, Hq, Hkv, hd, page = 150, 37, 8, 2, 64, 16
    q, k, v = (torch.randn(n, h, hd, generator=g).to(BF16) for h in (Hq, Hkv, Hkv))
    table = torch.randperm(12, generator=g)[:10].view(1, 10).to(torch.int32).cuda()
    kc = torch.zeros(12, Hkv, page, hd, dtype=BF16, device="cuda")
    vc = torch.zeros_like(kc)
    pos = torch.arange(n, dtype=torch.int32).cuda()
    zero = torch.zeros_like(pos)
    for a, b in ((0, n - tail), (n - tail, n)):
        _ops().paged_kv_append(k[a:b].cuda(), v[a:b].cuda(), kc, vc, table, pos[a:b],
                               rows=zero[a:b])
    got = _ops().paged_attn_decode(q[n - tail:].cuda(), kc, vc, table.repeat(tail, 1),
                                   pos[n - tail:] + 1)
    want, spread = ref.packed_prefill(q, k, v, torch.tensor([0, n], dtype=torch.int32))
    _attn_ok(got.cpu(), want[n - tail:], spread[n - tail:])
