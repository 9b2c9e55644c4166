"""Every code under every scale byte: what a 4-bit cache that another program has filled may hold."""
import math

import pytest
import torch

from oracle import mx4 as ref

pytestmark = pytest.mark.gpu

BF16 = torch.bfloat16
FP4, E8M0 = torch.float4_e2m1fn_x2, torch.float8_e8m0fnu


def _ops():
    from hybrid_llm_amd import ops
    return ops


def _device(codes, scales):
    c, s = ref.pack(codes, scales)
    return c.cuda().view(FP4), s.cuda().view(E8M0)


@pytest.mark.parametrize("hd", [64, 128])
def test_read(hd):
    """Exact in bf16, subnormals at the bottom; past its end infinity; byte 255 NaN throughout."""
    token = torch.arange(256)
    blocks = hd // 32
    scales = [(token[:, None] * (2 * i + 1) + 64 * torch.arange(blocks)) % 256 for i in (0, 1)]
    codes = [((torch.arange(hd) + i) % 16).expand(256, hd) for i in (0, 5)]
    made = [_device(c.view(1, 1, 256, hd), s.view(1, 1, 256, -1)) for c, s in zip(codes, scales)]
    table = torch.zeros(1, 1, dtype=torch.int32).cuda()
    got = _ops().paged_kv_read_mx4(made[0][0], made[1][0], made[0][1], made[1][1], table,
                                   token.int().cuda(), rows=torch.zeros_like(token).int().cuda())
    for g, c, s in zip(got, codes, scales):
        want = ref.values(c, s).to(BF16)
        g = g[:, 0].cpu()
        assert torch.equal(g.isnan(), want.isnan())
        assert int(want.isnan().sum()) == 32 * blocks
        assert bool(want.isinf().any()) and bool((want.abs().double() == 2.0 ** -128).any())
        keep = ~want.isnan()
        assert torch.equal(g.view(torch.int16)[keep], want.view(torch.int16)[keep])


@pytest.mark.parametrize("hd,T,width", [(64, 1, 4), (128, 4, 4), (64, 8, 300), (128, 1, 300)])
def test_attention_under_byte_0(hd, T, width):
    """Keys and values of which one block in two stands for code x 2^-127, bf16's subnormals among
    them; the queries are 2^125 there, so that the scores depend on those keys.

    Scores: products are exact, their sums off by 2^-24 (hd + 4) of the largest sum |q_d k_d|, the rest
    of a score's way to its weight by 2^-16; a score's error e moves a weight by e, twice that with the
    sum's; the weights' 16 bits are 2^-16 more.  The store: 2^-8 of a normal value, 2^-134 of a
    subnormal one; what products and sums under 2^-126 lose is 2^-150 each of a few thousand."""
    g = torch.Generator().manual_seed(hd + T)
    Hq, Hkv, page = 4, 2, 16
    pages = width + 3
    made, vals = [], []
    for _ in range(2):
        codes = torch.randint(0, 16, (pages, Hkv, page, hd), generator=g)
        scales = torch.randint(125, 128, (pages, Hkv, page, hd // 32), generator=g)
        scales[..., 0::2] = 0
        made.append(_device(codes, scales))
        vals.append(ref.values(codes, scales))
    q = torch.randn(1, T, Hq, hd, generator=g).clamp(-3, 3)
    low = torch.arange(hd) // 32 % 2 == 0
    q = torch.where(low, torch.sign(q) * 2.0 ** 125, q).to(BF16)
    table = torch.randperm(pages, generator=g)[:width].view(1, width).int()
    lengths = torch.tensor([width * page - 3], dtype=torch.int32)
    got = _ops().paged_attn_mx4(q.cuda(), made[0][0], made[1][0], made[0][1], made[1][1],
                                table.cuda(), lengths.cuda(), scale=0.25).cpu()
    want, spread = ref.attend(q, *vals, table, lengths, scale=0.25)
    assert 0 < float(want[..., low].abs().max()) < 2.0 ** -124
    most = max(float((q[0, t, h].double().abs() * vals[0][:, h // 2].abs()).sum(-1).max())
               for t in range(T) for h in range(Hq))
    by = 2 * (2.0 ** -24 * (hd + 4) * most * 0.25 + 2.0 ** -16) + 2.0 ** -16
    assert by < 2.0 ** -9
    tol = 2.0 ** -8 * want.abs() + by * spread * (1 + 2.0 ** -8) + 2.0 ** -133
    err = (got.double() - want).abs()
    assert bool((err <= tol).all()), float((err / tol).max())
    # the subnormal keys count: without them the weights are others
    flat = [vals[0] * ~low, vals[1]]
    other, _ = ref.attend(q, *flat, table, lengths, scale=0.25)
    assert bool(((got.double() - other).abs() > tol).any())
