"""Infinite and NaN values that a row sees under a weight below fp32's range: the row's dim is
that value, as in 64 bits, whatever waves or runs the keys are cut into.  Tolerance of the
other dims: that of tests/test_gpu_paged.py and tests/test_gpu_packed_attention.py."""
import math

import pytest
import torch

from oracle import paged as ref
from test_gpu_packed_attention import _cu, _inputs, _ok
from test_gpu_paged import _attn_ok, _decode_case, _ops

pytestmark = pytest.mark.gpu

# dims and what they hold at the far key
BAD = {3: math.inf, 5: -math.inf, 11: math.nan}


def _aside(got, want, ok, rows):
    """The dims of BAD in `rows` are what they should be; then out of the comparison."""
    got, want = got.clone(), want.clone()
    for d, x in BAD.items():
        cell = got[rows][..., d].float()
        assert bool(cell.isnan().all() if x != x else (cell == x).all()), (d, cell)
        got[..., d] = 0
        want[..., d] = 0
    ok(got, want)


@pytest.mark.parametrize("longest", [100, 5000])
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("far", [0, 40, 76])
@pytest.mark.parametrize("by", [-160.0, 100.0])
def test_a_step_over_a_value_without_weight(by, far, hd, longest):
    """The far key's score is 160 below the others, or the last one's 100 above (and the far key's
    60 below the rest)."""
    g = torch.Generator().manual_seed(hd + far)
    q, kc, vc, table, lens, ks, vs = _decode_case(2, 8, 2, hd, 16, [78, longest], False, g, std=0.5)
    q[..., 0] = 1.0
    kc[..., 0] = 0

    def at(c, t):
        return c[int(table[0, t // 16]), :, t % 16]

    at(kc, far)[:, 0] = -160.0 if by < 0 else -60.0
    if by > 0:
        at(kc, 77)[:, 0] = by
    want, spread = ref.paged_decode(q, kc, vc, table, lens, scale=1.0)
    for d, x in BAD.items():
        at(vc, far)[:, d] = x
    exact, _ = ref.paged_decode(q, kc, vc, table, lens, scale=1.0)
    assert exact[0, :, 3].eq(math.inf).all() and exact[0, :, 5].eq(-math.inf).all()
    got = _ops().paged_attn_decode(q.cuda(), kc.cuda(), vc.cuda(), table.cuda(), lens.cuda(),
                                   scale=1.0).cpu()
    spread = spread.clone()
    spread[..., list(BAD)] = 0
    _aside(got[:1], want[:1], lambda a, b: _attn_ok(a, b, spread[:1]), slice(None))
    _attn_ok(got[1:], want[1:], ref.paged_decode(q, kc, vc, table, lens, scale=1.0)[1][1:])


@pytest.mark.parametrize("heads", [8, 128, 180])
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("far", [0, 40, 200])
@pytest.mark.parametrize("kw", [{}, {"softcap": 200.0}], ids=str)
def test_a_prompt_over_a_value_without_weight(kw, far, hd, heads):
    """Rows well behind the far key take it in sub-tiles that all their rows see."""
    _, (q, k, v) = _inputs(300, heads, 1, hd, 23)
    q, k = q / 2, k / 2
    q[..., 0] = 1.0
    k[..., 0] = 0
    k[far, :, 0] = -160.0
    cu = _cu([300])
    some = [0, heads // 2, heads - 1]
    want, spread = ref.packed_prefill(q[:, some], k, v, cu, scale=1.0, **kw)
    for d, x in BAD.items():
        v[far, :, d] = x
    got = _ops().packed_attn_prefill(q.cuda(), k.cuda(), v.cuda(), cu.cuda(), scale=1.0,
                                     **kw).cpu()[:, some]
    _ok(got[:far], want[:far], spread[:far]) if far else None
    spread = spread.clone()
    spread[..., list(BAD)] = 0
    _aside(got[far:], want[far:], lambda a, b: _ok(a, b, spread[far:]), slice(None))


@pytest.mark.parametrize("longest", [100, 5000])
@pytest.mark.parametrize("hd", [64, 128])
def test_an_8_bit_nan_without_weight(hd, longest):
    g = torch.Generator().manual_seed(hd)
    q, kc, vc, table, lens, ks, vs = _decode_case(2, 8, 2, hd, 16, [78, longest], True, g)
    q[..., 0] = 8.0
    k, v = kc.float(), vc.float()
    k[..., 0] = 0
    k[int(table[0, 2]), :, 8, 0] = -448.0
    kc = k.to(kc.dtype)
    want, spread = ref.paged_decode(q, kc, vc, table, lens, scale=2.0, k_scale=ks, v_scale=vs)
    v[int(table[0, 2]), :, 8, 11] = math.nan
    got = _ops().paged_attn_decode(q.cuda(), kc.cuda(), v.to(vc.dtype).cuda(), table.cuda(),
                                   lens.cuda(), scale=2.0, k_scale=ks, v_scale=vs).cpu()
    assert got[0, :, 11].isnan().all()
    got[0, :, 11] = 0
    want[0, :, 11] = spread[0, :, 11] = 0
    _attn_ok(got, want, spread)
