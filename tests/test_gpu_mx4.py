"""The 4-bit paged cache and its attention against 64-bit oracles.

Tolerances.  Values are stored from bf16 rows by powers of two, which round nothing: codes
and scales equal the oracle's.  Normed and rotated keys reach the quantiser in fp32, off by
2^-19 of the row's largest value (12 additions of squares, a root, two products: 2^-20; the
angle 2^-22 of a radian, sine and cosine 2^-22), so a stored one lies between what the
oracle's value less that and plus that round to.

Attention: the cache's values are exact in bf16.  Weights keep 16 bits (two bf16: off by
2^-16 of each), which moves the result by 2^-16 sum_j w_j |v_j - out|.  Scores in fp32, with
sum |q_d k_d| scale <= 2^5 on these inputs: products of hd <= 128 terms off by 2^-24 * 132 *
2^5 < 2^-11; exp2 and the cap under 2^-16: a score's error e moves a weight by e, twice that
with the sum's: 2^-10 of the same spread.  Then one store, 2^-8 of the value.
"""
import math

import pytest
import torch

from oracle import mx4 as ref
from oracle import paged

pytestmark = pytest.mark.gpu

BF16 = torch.bfloat16
FP4, E8M0 = torch.float4_e2m1fn_x2, torch.float8_e8m0fnu


def _ops():
    from hybrid_llm_amd import ops
    return ops


def _inv_freq(rot):
    return (10000.0 ** (-torch.arange(0, rot, 2, dtype=torch.float64) / max(rot, 1))).float()


def _table(B, width, pages, g):
    return torch.randperm(pages, generator=g)[:B * width].view(B, width).to(torch.int32)


def _cache(pages, Hkv, page, hd, g, spread=3, junk=False):
    """A cache of random codes and scales around 1: (device tensors, fp64 keys, values)."""
    made, vals = [], []
    for _ in range(2):
        codes = torch.randint(0, 16, (pages, Hkv, page, hd), generator=g)
        scales = torch.randint(127 - spread, 128, (pages, Hkv, page, hd // 32), generator=g)
        made.append(ref.pack(codes, scales))
        vals.append(ref.values(codes, scales))
    (kc, ks), (vc, vs) = made
    dev = (kc.cuda().view(FP4), vc.cuda().view(FP4), ks.cuda().view(E8M0), vs.cuda().view(E8M0))
    return dev, vals[0], vals[1]


def _attn_ok(got, want, spread, more=0.0):
    want = want.reshape(got.shape)
    tol = 2.0 ** -8 * want.abs() + (2.0 ** -16 + 2.0 ** -10 + more) * spread.reshape(got.shape) \
        * (1 + 2.0 ** -8) + 1e-30
    err = (got.double() - want).abs()
    assert bool((err <= tol).all()), float((err / tol).max())


# ----------------------------------------------------------------- append and read
@pytest.mark.parametrize("N,Hq,Hkv,hd,rot,interleaved,normed,page", [
    (1, 16, 4, 64, 64, False, True, 16),
    (3, 0, 1, 128, 128, True, True, 32),
    (37, 6, 2, 128, 64, False, False, 64),
    (70, 7, 7, 64, 24, True, True, 16),
    (130, 0, 3, 128, 40, False, True, 128),
    (300, 32, 8, 128, 128, False, True, 256),
    (64, 4, 4, 64, 0, False, True, 16),
    (1700, 24, 8, 64, 64, False, True, 16),     # four iterations a wave
    (1003, 40, 13, 128, 8, False, False, 16),
])
def test_append_and_read(N, Hq, Hkv, hd, rot, interleaved, normed, page):
    g = torch.Generator().manual_seed(N + hd)
    row = (torch.randn(N, (Hq + 2 * Hkv) * hd, generator=g) * 3).to(BF16)
    row[0, -hd:] = 0
    width = 5
    B = -(-N // (width * page)) + 2
    pages = B * width + 3
    table = _table(B, width, pages, g)
    slot = torch.randperm(B * width * page, generator=g)[:N]
    rows, pos = (slot // (width * page)).int(), (slot % (width * page)).int()
    f = _inv_freq(rot) if rot else None
    w = [torch.randn(hd, generator=g) + 1 if normed else None for _ in range(2)]
    d = row.cuda()
    q, k, v = (t.view(N, -1, hd) for t in d.split([Hq * hd, Hkv * hd, Hkv * hd], 1))
    fd, wq, wk, td, pd, rd = (None if t is None else t.cuda() for t in (f, *w, table, pos, rows))
    cache = _ops().mx4_cache(pages, Hkv, page, hd)
    before = [t.view(torch.uint8).random_(0, 200).clone().cpu() for t in cache]
    with_q = {"q": q, "q_norm": wq} if Hq else {}
    got_q = _ops().paged_kv_append_mx4(k, v, *cache, td, pd, rows=rd, inv_freq=fd, k_norm=wk,
                                       interleaved=interleaved, **with_q)
    if Hq:  # as without a cache, to the bit
        want_q, _ = _ops().qk_norm_rope(q, k, pd, fd, q_norm=wq, interleaved=interleaved)
        assert torch.equal(got_q, want_q)
    ids = table[rows.long(), pos.long() // page].long()
    at = pos.long() % page
    kc, vc, ks, vs = (t.view(torch.uint8).cpu() for t in cache)
    # values: codes and scales of the definition
    want, want_s = ref.pack(*ref.stored(v.cpu()))
    assert torch.equal(vs[ids, :, at], want_s)
    assert torch.equal(vc[ids, :, at], want)
    # keys: between the roundings of what the fp32 path may give
    x = paged.norm_rope(k.cpu(), pos, f, w[1], 1e-6, interleaved)
    off = 2.0 ** -19 * x.abs().amax(-1, keepdim=True) if normed or rot else 0 * x[..., :1]
    codes, bytes_ = ref.unpack(kc[ids, :, at], ks[ids, :, at])
    low = ref.stored((x.abs() - off).clamp_min(0))[1]
    high = ref.stored(x.abs() + off)[1]
    assert bool(((low <= bytes_) & (bytes_ <= high)).all())
    step = torch.exp2(bytes_.double() - 127).repeat_interleave(32, -1)
    val = ref.values(codes, bytes_)
    lo, hi = (ref.values(ref.round_to(x + s * off, step), torch.full_like(bytes_, 127)) * step
              for s in (-1, 1))
    assert bool(((lo <= val) & (val <= hi)).all())
    # every other slot as it was
    mine = torch.zeros(pages, page, dtype=torch.bool)
    mine[ids, at] = True
    for t, b in zip((kc, vc, ks, vs), before):
        assert torch.equal(t.transpose(1, 2)[~mine], b.transpose(1, 2)[~mine])
    # read back: exactly the stored values
    rk, rv = _ops().paged_kv_read_mx4(*cache, td, pd, rows=rd)
    assert rk.dtype is BF16 and torch.equal(rk.cpu().double(), val)
    assert torch.equal(rv.cpu().double(), ref.values(*ref.unpack(vc[ids, :, at], vs[ids, :, at])))


def _put(row, page=16):
    """Rows [N, hd] stored as values: (codes, bytes) and what is read back."""
    N, hd = row.shape
    cache = _ops().mx4_cache(-(-N // page), 1, page, hd)
    x = row.to(BF16).cuda().view(N, 1, hd)
    table = torch.arange(-(-N // page), dtype=torch.int32).view(1, -1).cuda()
    pos, rows = torch.arange(N, dtype=torch.int32).cuda(), torch.zeros(N, dtype=torch.int32).cuda()
    _ops().paged_kv_append_mx4(x, x, *cache, table, pos, rows=rows)
    k, v = _ops().paged_kv_read_mx4(*cache, table, pos, rows=rows)
    assert torch.equal(k.view(torch.int16), v.view(torch.int16))
    for a, b in ((cache[0], cache[1]), (cache[2], cache[3])):
        assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))
    codes, scales = (t.view(torch.uint8)[:, 0].flatten(0, 1)[:N].cpu() for t in (cache[1], cache[3]))
    return codes, scales, v[:, 0].cpu()


def test_ties_borders_and_ends():
    """Every border between codes and both sides of it, scales at their border and their ends,
    zeros of both signs."""
    ties = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 7.0])
    near = torch.cat([ties, ties * (1 - 2.0 ** -8), ties * (1 + 2.0 ** -7)])
    rows = []
    for e in (-126, -120, -20, 0, 1, 30, 120, 125):
        for top in (4.0, 6.0, 7.0, 7.03125):
            x = torch.zeros(64, dtype=torch.float64)
            x[:24] = near.to(BF16).double().clamp(max=top)
            x[24] = top
            x[32:56] = -x[:24]
            x[57] = -top
            rows.append(x * 2.0 ** e)
    rows.append(torch.zeros(64, dtype=torch.float64))
    rows.append(torch.full((64,), -0.0, dtype=torch.float64))
    rows.append(torch.full((64,), 2.0 ** -133, dtype=torch.float64))      # bf16's smallest
    rows.append(torch.full((64,), float(torch.finfo(BF16).max), dtype=torch.float64))
    x = torch.stack(rows).clamp(-float(torch.finfo(BF16).max), float(torch.finfo(BF16).max)).to(BF16)
    codes, scales, back = _put(x)
    want, want_s = ref.pack(*ref.stored(x))
    assert torch.equal(scales, want_s)
    assert torch.equal(codes, want)
    assert torch.equal(back.double(), ref.values(*ref.stored(x)))
    assert int(scales.max()) == 252 and bool(torch.isfinite(back).all())


@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
def test_a_block_that_is_not_finite(bad):
    x = torch.randn(5, 128)
    x[1, 40] = bad
    x[3, 127] = bad
    codes, scales, back = _put(x)
    lost = torch.zeros(5, 4, dtype=torch.bool)
    lost[1, 1] = lost[3, 3] = True
    assert torch.equal(scales == 255, lost)
    assert torch.equal(back.isnan(), lost.repeat_interleave(32, 1))
    keep = ~lost.repeat_interleave(32, 1)
    assert torch.equal(back.double()[keep], ref.values(*ref.stored(x.to(BF16)))[keep])


def test_tokens_without_a_slot():
    ops = _ops()
    cache = ops.mx4_cache(4, 2, 16, 64)
    table = torch.tensor([[0, 9], [-1, 2]], dtype=torch.int32).cuda()
    rows = torch.tensor([0, 0, 1, 1, 5, -1, 0, 1], dtype=torch.int32).cuda()
    pos = torch.tensor([3, 16, 0, 31, 0, 0, -1, 32], dtype=torch.int32).cuda()
    x = torch.randn(8, 2, 64).to(BF16).cuda()
    ops.paged_kv_append_mx4(x, x, *cache, table, pos, rows=rows)
    stored = (cache[1].view(torch.uint8) != 0).any(-1).any(1).cpu()
    assert stored.nonzero().tolist() == [[0, 3], [2, 15]]
    k, v = ops.paged_kv_read_mx4(*cache, table, pos, rows=rows)
    assert [bool(t.any()) for t in k] == [True, False, False, True, False, False, False, False]
    assert torch.equal(k, v)


# ----------------------------------------------------------------- attention
@pytest.mark.parametrize("B,T,Hq,Hkv,hd,page,lens,window,cap,slopes", [
    (1, 1, 1, 1, 64, 16, [1], 0, 0.0, False),
    (1, 1, 16, 4, 64, 16, [1023], 0, 0.0, False),
    (3, 1, 8, 2, 128, 32, [0, 17, 500], 0, 30.0, True),
    (4, 4, 8, 2, 128, 16, [4, 2, 300, 33], 0, 0.0, False),
    (2, 5, 16, 4, 64, 64, [77, 641], 100, 0.0, True),       # 20 columns: two tiles a wave
    (3, 8, 10, 1, 64, 128, [9, 128, 400], 0, 50.0, False),  # 80 columns
    (2, 3, 40, 2, 128, 16, [200, 65], 33, 0.0, False),
    (2, 16, 4, 4, 128, 16, [16, 161], 0, 0.0, True),
    (2, 64, 2, 1, 64, 16, [64, 100], 7, 0.0, False),
    (5, 2, 32, 8, 128, 256, [257, 1, 256, 3, 511], 0, 0.0, False),
    # long tables: runs over the flat list, joined
    (1, 1, 4, 4, 64, 16, [9000], 0, 0.0, False),
    (3, 4, 16, 4, 64, 64, [5000, 4, 4097], 0, 20.0, True),
    (2, 2, 32, 2, 128, 32, [6001, 3333], 0, 0.0, False),
    (7, 1, 8, 1, 128, 64, [8192, 1, 0, 4000, 31, 32, 8191], 0, 0.0, False),
    (2, 7, 16, 4, 64, 32, [7000, 6], 1000, 0.0, True),
    (2, 1, 8, 8, 128, 256, [3100, 9216], 513, 0.0, False),
])
def test_attention(B, T, Hq, Hkv, hd, page, lens, window, cap, slopes):
    g = torch.Generator().manual_seed(sum(lens) + hd + T)
    width = -(-max(max(lens), 1) // page) + (1 if len(lens) > 2 else 0)
    pages = B * width + 2
    table = _table(B, width, pages, g)
    dev, k, v = _cache(pages, Hkv, page, hd, g)
    q = torch.randn(B, T, Hq, hd, generator=g).to(BF16)
    s = torch.rand(Hq, generator=g) * 0.1 if slopes else None
    lengths = torch.tensor(lens, dtype=torch.int32)
    got = _ops().paged_attn_mx4(q.cuda(), *dev, table.cuda(), lengths.cuda(), window=window,
                                softcap=cap, slopes=None if s is None else s.cuda())
    want, spread = ref.attend(q, k, v, table, lengths, window=window, softcap=cap, slopes=s)
    assert got.shape == q.shape
    _attn_ok(got.cpu(), want, spread)
    if T == 1:
        one = _ops().paged_attn_mx4(q[:, 0].cuda(), *dev, table.cuda(), lengths.cuda(),
                                    window=window, softcap=cap,
                                    slopes=None if s is None else s.cuda())
        assert one.shape == (B, Hq, hd) and torch.equal(one, got[:, 0])


def test_strided_queries_and_scale():
    g = torch.Generator().manual_seed(3)
    B, T, Hq, Hkv, hd, page = 3, 4, 8, 2, 64, 16
    table = _table(B, 6, 20, g)
    dev, k, v = _cache(20, Hkv, page, hd, g)
    wide = torch.randn(B, T + 1, (Hq + 3) * hd, generator=g).to(BF16)
    d = wide.cuda()
    q = d[:, 1:, hd:(Hq + 1) * hd].unflatten(-1, (Hq, hd))
    assert not q.is_contiguous()
    lengths = torch.tensor([50, 96, 7], dtype=torch.int32)
    got = _ops().paged_attn_mx4(q, *dev, table.cuda(), lengths.cuda(), scale=0.05)
    want, spread = ref.attend(q.cpu(), k, v, table, lengths, scale=0.05)
    _attn_ok(got.cpu(), want, spread)
    # one token's heads laid out last to first in memory, by head and token swapped
    q = d[:, :4, :8 * hd].unflatten(-1, (8, hd)).transpose(1, 2)[:, :, :].contiguous().transpose(1, 2)
    got = _ops().paged_attn_mx4(q, *dev, table.cuda(), lengths.cuda())
    want, spread = ref.attend(q.cpu(), k, v, table, lengths)
    _attn_ok(got.cpu(), want, spread)


@pytest.mark.parametrize("hd,T,width", [(64, 1, 8), (128, 4, 8), (64, 6, 300), (128, 1, 300)])
def test_unseen_slots_hold_anything(hd, T, width):
    """NaN scales in slots past the length, before the window, in pages that nothing names."""
    g = torch.Generator().manual_seed(hd + width)
    B, Hq, Hkv, page, window = 3, 8, 2, 16, 60
    pages = B * width + 4
    table = _table(B, width, pages, g)
    n = width * page
    lengths = torch.tensor([n - 13, n // 2 + 5, 40], dtype=torch.int32)
    dev, k, v = _cache(pages, Hkv, page, hd, g)
    table[1, int(lengths[1]) // page - 2] = -1
    table[0, 3] = pages + 7
    dirty = [t.view(torch.uint8).clone() for t in dev]
    seen = torch.zeros(pages, page, dtype=torch.bool)
    for b in range(B):
        for p in range(max(0, int(lengths[b]) - (T - 1) - window), int(lengths[b])):
            i = int(table[b, p // page])
            if 0 <= i < pages:
                seen[i, p % page] = True
    for t in dirty[:2]:
        t.transpose(1, 2)[~seen.cuda()] = 0x77
    for t in dirty[2:]:
        t.transpose(1, 2)[~seen.cuda()] = 255
    dirty = [t.view(o.dtype) for t, o in zip(dirty, dev)]
    q = torch.randn(B, T, Hq, hd, generator=g).to(BF16)
    got = _ops().paged_attn_mx4(q.cuda(), *dirty, table.cuda(), lengths.cuda(), window=window)
    want, spread = ref.attend(q, k, v, table, lengths, window=window)
    _attn_ok(got.cpu(), want, spread)


@pytest.mark.parametrize("hd,width", [(64, 4), (128, 4), (64, 300), (128, 300)])
@pytest.mark.parametrize("byte", [253, 255])
def test_a_seen_block_that_is_nan(hd, width, byte):
    """A value's NaN block: its dims of the tokens that see it, whatever its weight; a later
    token's block does not reach an earlier token.  A key's: the rows that see it."""
    g = torch.Generator().manual_seed(hd)
    T, Hq, Hkv, page = 4, 4, 2, 16
    table = _table(1, width, width + 2, g)
    n = width * page - 5
    lengths = torch.tensor([n], dtype=torch.int32)
    dev, k, v = _cache(width + 2, Hkv, page, hd, g)
    q = torch.randn(1, T, Hq, hd, generator=g).to(BF16)
    clean = _ops().paged_attn_mx4(q.cuda(), *dev, table.cuda(), lengths.cuda()).cpu()
    at = n - 2  # tokens 2 and 3 see it
    vs = dev[3].view(torch.uint8).clone()
    vs[int(table[0, at // page]), 1, at % page, 1] = byte
    got = _ops().paged_attn_mx4(q.cuda(), *dev[:3], vs.view(E8M0), table.cuda(),
                                lengths.cuda()).cpu()
    lost = torch.zeros(1, T, Hq, hd, dtype=torch.bool)
    lost[0, 2:, 2:, 32:64] = True
    assert torch.equal(got.isnan(), lost)
    assert torch.equal(got[~lost], clean[~lost])
    # far back, under a weight that vanishes
    vs = dev[3].view(torch.uint8).clone()
    vs[int(table[0, 0]), 0, 2, 0] = byte
    slopes = torch.full((Hq,), 1000.0)
    got = _ops().paged_attn_mx4(q.cuda(), *dev[:3], vs.view(E8M0), table.cuda(), lengths.cuda(),
                                slopes=slopes.cuda()).cpu()
    lost.zero_()
    lost[0, :, :2, :32] = True
    assert torch.equal(got.isnan(), lost)
    if byte == 255:
        ks = dev[2].view(torch.uint8).clone()
        ks[int(table[0, at // page]), 1, at % page, 0] = byte
        got = _ops().paged_attn_mx4(q.cuda(), *dev[:2], ks.view(E8M0), dev[3], table.cuda(),
                                    lengths.cuda()).cpu()
        assert got[0, 2:, 2:].isnan().all() and torch.equal(got[0, :2], clean[0, :2])
        assert torch.equal(got[0, :, :2], clean[0, :, :2])


@pytest.mark.parametrize("big", [100.0, 1e4, 1e30])
@pytest.mark.parametrize("width", [4, 200])
def test_large_scores(big, width):
    """Keys apart by far more than a weight spans: the largest score's value alone."""
    g = torch.Generator().manual_seed(int(math.log10(big)))
    table = _table(1, width, width, g)
    n = width * 16
    dev, k, v = _cache(width, 1, 16, 64, g)
    q = torch.zeros(1, 1, 2, 64)
    q[..., 5] = big
    q[0, 0, 1] *= -1
    q = q.to(BF16)
    lengths = torch.tensor([n], dtype=torch.int32)
    got = _ops().paged_attn_mx4(q.cuda(), *dev, table.cuda(), lengths.cuda(), scale=1.0).cpu()
    want, spread = ref.attend(q, k, v, table, lengths, scale=1.0)
    # scores are single products, exact; their difference is off by 2^-24 of the larger
    _attn_ok(got, want, spread, more=0.0 if big > 1e3 else 2 * 2.0 ** -23 * 6 * big)


def test_rows_that_are_nan():
    g = torch.Generator().manual_seed(1)
    dev, k, v = _cache(4, 1, 16, 64, g)
    table = torch.arange(4, dtype=torch.int32).view(1, 4).cuda()
    q = torch.randn(1, 2, 2, 64).to(BF16)
    q[0, 0, 1, 3] = math.nan
    q[0, 1, 0, 9] = math.inf
    got = _ops().paged_attn_mx4(q.cuda(), *dev, table, torch.tensor([60], dtype=torch.int32).cuda())
    assert got[0, 0, 1].isnan().all() and got[0, 1, 0].isnan().all()
    assert torch.isfinite(got[0, 0, 0]).all() and torch.isfinite(got[0, 1, 1]).all()


def test_empty_calls():
    ops = _ops()
    dev, _, _ = _cache(2, 2, 16, 64, torch.Generator().manual_seed(0))
    i32 = dict(dtype=torch.int32, device="cuda")
    q = torch.randn(3, 2, 4, 64, device="cuda").to(BF16)
    lengths = torch.tensor([0, -4, 9], **i32)
    out = ops.paged_attn_mx4(q, *dev, torch.full((3, 1), 5, **i32), lengths)  # no page is named
    assert not out.any()
    out = ops.paged_attn_mx4(q, *dev, torch.zeros(3, 0, **i32), lengths)
    assert not out.any()
    none = ops.mx4_cache(0, 2, 16, 64)
    out = ops.paged_attn_mx4(q, *none, torch.zeros(3, 1, **i32), lengths)
    assert not out.any()
    assert ops.paged_attn_mx4(q[:0], *dev, torch.zeros(0, 1, **i32), lengths[:0]).shape == (0, 2, 4, 64)
    x = torch.empty(0, 2, 64, device="cuda", dtype=BF16)
    ops.paged_kv_append_mx4(x, x, *dev, torch.zeros(1, 1, **i32), torch.zeros(0, **i32))
    k, _ = ops.paged_kv_read_mx4(*dev, torch.zeros(1, 1, **i32), torch.zeros(0, **i32))
    assert k.shape == (0, 2, 64)


def test_repeats_are_equal_to_the_bit():
    """Attention over long tables, captured and replayed beside eager calls of other lengths."""
    ops = _ops()
    g = torch.Generator().manual_seed(4)
    B, T, Hq, Hkv, hd, page, width = 4, 3, 8, 2, 128, 64, 80
    table = _table(B, width, B * width, g).cuda()
    dev, _, _ = _cache(B * width, Hkv, page, hd, g)
    q = torch.randn(B, T, Hq, hd, generator=g).to(BF16).cuda()
    lengths = torch.tensor([5000, 70, 3, 4100], dtype=torch.int32).cuda()
    first = ops.paged_attn_mx4(q, *dev, table, lengths)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = ops.paged_attn_mx4(q, *dev, table, lengths)
    for n in (5000, 1200, 64, 5000):
        lengths[0] = n
        want = ops.paged_attn_mx4(q, *dev, table, lengths)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want)
    assert torch.equal(want, first)


# -------------------------------------------- every form, long caches, other streams
@pytest.mark.parametrize("B,T,Hq,Hkv,hd,page,longest,window", [
    (40, 1, 8, 8, 128, 16, 90, 0),        # more head tiles than CUs, short tables: four waves each
    (36, 3, 16, 8, 128, 32, 700, 50),
    (70, 1, 8, 4, 64, 16, 500, 0),
    (70, 5, 16, 4, 64, 64, 500, 0),       # two column tiles
    (64, 2, 4, 4, 64, 32, 4000, 0),       # long ones: a CU's waves each
    (34, 1, 8, 8, 128, 64, 5000, 0),      # as many tiles, long tables: runs
    (3, 64, 4, 1, 64, 16, 4500, 0),       # 256 columns in runs
    (2, 33, 6, 2, 128, 128, 6000, 2 ** 31 - 1),
    (300, 2, 2, 1, 64, 16, 2500, 90),     # a window that only some of them pass
])
def test_attention_of_many(B, T, Hq, Hkv, hd, page, longest, window):
    """Lengths from nothing to the longest, some below T: their first tokens see nothing."""
    g = torch.Generator().manual_seed(B + T + longest)
    width = -(-longest // page)
    pages = min(B * width, 600)
    table = torch.randint(0, pages, (B, width), generator=g).int()  # pages may be shared
    dev, k, v = _cache(pages, Hkv, page, hd, g)
    q = torch.randn(B, T, Hq, hd, generator=g).to(BF16)
    lengths = torch.randint(0, longest + 1, (B,), generator=g).int()
    lengths[:2] = torch.tensor([longest, T // 2])
    got = _ops().paged_attn_mx4(q.cuda(), *dev, table.cuda(), lengths.cuda(), window=window).cpu()
    some = [0, 1, B // 2, B - 1] if B > 4 else list(range(B))
    want, spread = ref.attend(q[some], k, v, table[some], lengths[some], window=window)
    _attn_ok(got[some], want, spread)
    if T > 1:
        assert not got[1, :T - T // 2].any()  # tokens before the text
    # and each alone: another split of the work, the same within both calls' errors
    for b in (B // 2, B - 2):
        one = _ops().paged_attn_mx4(q[b:b + 1].cuda(), *dev, table[b:b + 1].cuda().contiguous(),
                                    lengths[b:b + 1].cuda(), window=window).cpu()
        both = 2.0 ** -7 * got[b].double().abs() + 2 * (2.0 ** -16 + 2.0 ** -10) * 12 + 1e-30
        assert bool(((one[0].double() - got[b].double()).abs() <= both).all())


def test_nothing_to_see_over_long_tables():
    ops = _ops()
    i32 = dict(dtype=torch.int32, device="cuda")
    q = torch.randn(3, 2, 4, 64, device="cuda").to(BF16)
    dev, _, _ = _cache(2, 2, 16, 64, torch.Generator().manual_seed(0))
    lengths = torch.tensor([0, -4, 9000], **i32)
    empty = torch.zeros(3, 900, **i32)
    assert not ops.paged_attn_mx4(q, *ops.mx4_cache(0, 2, 16, 64), empty, lengths).any()
    assert not ops.paged_attn_mx4(q, *dev, empty - 1, lengths).any()
    assert not ops.paged_attn_mx4(q, *dev, empty, lengths * 0).any()


@pytest.mark.parametrize("hd,width", [(128, 3), (128, 200), (64, 200)])
def test_a_cache_past_32_bit_offsets(hd, width):
    """Codes of k and of v past 4 GiB each: pages at both ends and around 2^31 and 2^32."""
    ops, g = _ops(), torch.Generator().manual_seed(width)
    Hkv, page, Hq, T = 8, 256, 8, 2
    per = Hkv * page * hd // 2
    pages = 2 ** 32 // per + 40
    cache = tuple(torch.empty(s, dtype=torch.uint8, device="cuda").view(t) for s, t in (
        ((pages, Hkv, page, hd // 2), FP4), ((pages, Hkv, page, hd // 2), FP4),
        ((pages, Hkv, page, hd // 32), E8M0), ((pages, Hkv, page, hd // 32), E8M0)))
    B = 2
    at = 2 ** 31 // per
    ids = torch.tensor([pages - 1, 0, 2 ** 32 // per, 2 ** 32 // per - 1, at, at - 1])
    n = 3 * page
    lengths = torch.tensor([n - 1, n - 40], dtype=torch.int32)
    table = torch.full((B, width), -1, dtype=torch.int32)
    table[:, :3] = ids.view(B, 3).int()
    x = [torch.randn(B * n, Hkv, hd, generator=g).to(BF16) for _ in range(2)]
    pos = torch.arange(n).repeat(B).int()
    rows = torch.arange(B).repeat_interleave(n).int()
    td = table.cuda()
    ops.paged_kv_append_mx4(x[0].cuda(), x[1].cuda(), *cache, td, pos.cuda(), rows=rows.cuda())
    vals = [ref.values(*ref.stored(t)) for t in x]
    for got, want in zip(ops.paged_kv_read_mx4(*cache, td, pos.cuda(), rows=rows.cuda()), vals):
        assert torch.equal(got.cpu().double(), want)
    # the oracle's cache: the six pages alone
    k, v = (t.view(B * 3, page, Hkv, hd).transpose(1, 2) for t in vals)
    q = torch.randn(B, T, Hq, hd, generator=g).to(BF16)
    got = ops.paged_attn_mx4(q.cuda(), *cache, td, lengths.cuda())
    want, spread = ref.attend(q, k, v, torch.arange(6).view(B, 3).int(), lengths)
    _attn_ok(got.cpu(), want, spread)


def test_on_other_streams_and_two_at_once():
    """Calls that overlap on two streams, over one cache, each with its own workspace."""
    ops, g = _ops(), torch.Generator().manual_seed(8)
    Hq, Hkv, hd, page = 8, 2, 64, 32
    dev, k, v = _cache(300, Hkv, page, hd, g)
    sets = []
    for B, T, width in ((3, 2, 250), (5, 4, 200)):
        table = torch.randint(0, 300, (B, width), generator=g).int()
        q = torch.randn(B, T, Hq, hd, generator=g).to(BF16)
        lengths = torch.randint(T, width * page + 1, (B,), generator=g).int()
        sets.append((q, table, lengths))
    given = [[t.cuda() for t in s] for s in sets]
    want = [ops.paged_attn_mx4(q, *dev, t, n).cpu() for q, t, n in given]
    for (q, table, lengths), w in zip(sets, want):
        exact, spread = ref.attend(q, k, v, table, lengths)
        _attn_ok(w, exact, spread)
    streams = [torch.cuda.Stream() for _ in sets]
    torch.cuda.synchronize()
    for _ in range(4):
        got = []
        for (q, t, n), s in zip(given, streams):
            with torch.cuda.stream(s):
                got.append(ops.paged_attn_mx4(q, *dev, t, n))
        torch.cuda.synchronize()
        for a, w in zip(got, want):
            assert torch.equal(a.cpu(), w)
