"""Infinite and NaN values that a row sees under a weight below fp32's range: the row's dim is
that value, as in 64 bits, whatever waves or runs the keys are cut into.  Tolerance of the
other dims: that of tests/test_gpu_packed_attention.py."""
import math

import pytest
import torch

from oracle import paged as ref
from test_gpu_packed_attention import _cu, _inputs, _ok, _ops

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
