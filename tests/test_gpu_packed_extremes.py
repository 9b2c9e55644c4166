"""Scores that are not finite, and finite ones of any size, in attention over packed prompts.

Heads 8, 128 and 180 at 300 rows have four, two and one waves along the keys.
Tolerance: that of tests/test_gpu_packed_attention.py (its bound on scores is not used where
they are exact or tie, as said at the test).
"""
import math

import pytest
import torch

from oracle import paged as ref
from test_gpu_packed_attention import BF16, _cu, _inputs, _ok, _ops

pytestmark = pytest.mark.gpu

HEADS = [8, 128, 180]


def _prompt(q, k, v, cu, **kw):
    return _ops().packed_attn_prefill(q.cuda(), k.cuda(), v.cuda(), cu.cuda(), **kw).cpu()


# ------------------------------------------------------------------ NaN
@pytest.mark.parametrize("heads", HEADS)
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("kw", [{}, {"softcap": 20.0}, {"slopes": 0.01},
                                {"softcap": 20.0, "slopes": 0.01}], ids=str)
def test_a_nan_key_alone_in_its_sub_tile(kw, hd, heads):
    """A document's first key, on the last row of 32: every row of it sees a NaN score."""
    _, (q, k, v) = _inputs(300, heads, 1, hd, 16)
    kw = dict(kw)
    if "slopes" in kw:
        kw["slopes"] = torch.full((heads,), kw["slopes"])
    cu = _cu([31, 269])
    k[31, 0, 3] = math.nan
    dev = {n: t.cuda() if torch.is_tensor(t) else t for n, t in kw.items()}
    got = _prompt(q, k, v, cu, **dev)
    assert got[31:].isnan().all()
    some = [0, heads // 2, heads - 1]
    if "slopes" in kw:
        kw["slopes"] = kw["slopes"][some]
    want, spread = ref.packed_prefill(q[:31, some], k[:31], v[:31], _cu([31]), **kw)
    _ok(got[:31, some], want, spread)


@pytest.mark.parametrize("heads", HEADS)
def test_a_nan_key_that_a_window_begins_on(heads):
    """Rows 95 to 119 see key 95, the last of them nothing else of its sub-tile."""
    _, (q, k, v) = _inputs(300, heads, 1, 64, 17)
    k[95, 0, 3] = math.nan
    got = _prompt(q, k, v, _cu([300]), window=25)
    assert got[95:120].isnan().all()
    some = [0, heads // 2, heads - 1]
    k[95] = 0
    want, spread = ref.packed_prefill(q[:, some], k, v, _cu([300]), window=25)
    _ok(got[:95, some], want[:95], spread[:95])
    _ok(got[120:, some], want[120:], spread[120:])


# ------------------------------------------------------------------ a cap and infinite scores
@pytest.mark.parametrize("heads", HEADS)
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("cap", [0.5, 30.0, 1000.0])
@pytest.mark.parametrize("keys", [(0, 300), (0, 70), (40, 41), (64, 200)], ids=str)
def test_capped_scores_of_minus_infinity(keys, cap, hd, heads):
    """They are -cap: alone they weigh alike, beside others e^-cap.  Capped scores are off by
    2^-23 of the cap and 2^-11, a weight by e^(2 of that) - 1."""
    _, (q, k, v) = _inputs(300, heads, 1, hd, 18)
    q[..., 0] = q[..., 0].abs() + 0.125
    k[keys[0]:keys[1], :, 0] = -math.inf
    cu = _cu([250, 50])
    got = _prompt(q, k, v, cu, softcap=cap)
    some = [0, heads // 2, heads - 1]
    want, spread = ref.packed_prefill(q[:, some], k, v, cu, softcap=cap)
    assert bool(want.isfinite().all())
    # the oracle's own capped -inf scores weigh alike exactly, and so do the kernel's
    _ok(got[:, some], want, spread)
