"""Short texts in a table for long ones, as a server with a fixed table has them: runs of many small head
tiles.  Entries past a text name anything, pages that do not exist among them.

Tolerances.  Values are exact in bf16; weights keep 16 bits, 2^-16 of the spread sum_j w_j |v_j - out|.
Scores in fp32: sum |q_d k_d| scale <= 2^5 on these inputs, off by 2^-24 x 132 x 2^5 < 2^-11, which
moves weights by twice that with their sum: 2^-10 of the spread.  The store: 2^-8 of the value."""
import pytest
import torch

from oracle import mx4 as ref

pytestmark = pytest.mark.gpu

BF16 = torch.bfloat16
FP4, E8M0 = torch.float4_e2m1fn_x2, torch.float8_e8m0fnu


@pytest.mark.parametrize("B,T,Hq,Hkv,hd,page,longest,window", [
    (1, 1, 16, 4, 64, 16, 1023, 0),
    (1, 1, 4, 4, 128, 256, 1, 0),
    (64, 1, 32, 8, 128, 16, 100, 0),
    (16, 4, 16, 4, 64, 32, 70, 0),
    (300, 2, 8, 1, 64, 16, 3, 0),            # tiles of one step, some of none
    (130, 8, 16, 4, 64, 64, 33, 5000),       # two column tiles, a window that is wider still
    (7, 3, 40, 2, 128, 16, 65, 0),           # 60 columns in two head tiles
    (1000, 1, 4, 4, 64, 128, 64, 0),
])
def test_short_texts(B, T, Hq, Hkv, hd, page, longest, window):
    from hybrid_llm_amd import ops
    g = torch.Generator().manual_seed(B + T + longest)
    used, width = -(-longest // page), 131072 // page
    pages = min(B * used, 500)
    made, vals = [], []
    for _ in range(2):
        codes = torch.randint(0, 16, (pages, Hkv, page, hd), generator=g)
        scales = torch.randint(124, 128, (pages, Hkv, page, hd // 32), generator=g)
        c, s = ref.pack(codes, scales)
        made.append((c.cuda().view(FP4), s.cuda().view(E8M0)))
        vals.append(ref.values(codes, scales))
    lengths = torch.randint(0, longest + 1, (B,), generator=g).int()
    lengths[B // 2] = longest
    table = torch.randint(-pages, 3 * pages, (B, width), generator=g).int()
    table[:, :used] = torch.randint(0, pages, (B, used), generator=g).int()
    q = torch.randn(B, T, Hq, hd, generator=g).to(BF16)
    cache = (made[0][0], made[1][0], made[0][1], made[1][1])
    got = ops.paged_attn_mx4(q.cuda(), *cache, table.cuda(), lengths.cuda(), window=window).cpu()
    some = sorted({0, B // 3, B // 2, B - 1}) if B > 20 else list(range(B))
    want, spread = ref.attend(q[some], *vals, table[some], lengths[some], window=window)
    tol = 2.0 ** -8 * want.abs() + (2.0 ** -16 + 2.0 ** -10) * spread * (1 + 2.0 ** -8) + 1e-30
    err = (got[some].double() - want).abs()
    assert bool((err <= tol).all()), float((err / tol).max())
    # all of them: as in a table of their own width, within both calls' errors; zeros where none is seen
    narrow = ops.paged_attn_mx4(q.cuda(), *cache, table[:, :used].contiguous().cuda(), lengths.cuda(),
                                window=window).cpu().double()
    both = 2.0 ** -7 * narrow.abs() + 2 * (2.0 ** -16 + 2.0 ** -10) * 12 + 1e-30
    assert bool(((got.double() - narrow).abs() <= both).all())
    unseen = (lengths[:, None] - T + torch.arange(T)) < 0
    assert not got[unseen].any()
