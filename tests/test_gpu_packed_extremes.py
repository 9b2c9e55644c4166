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


# ------------------------------------------------------------------ large finite scores
def _ternary(N, heads, hd, seed):
    """q and k of 20 entries +-1 each, the rest 0, so that products are whole numbers to
    20; each document's first row opposes its key."""
    g = torch.Generator().manual_seed(seed)

    def signs(n, h):
        x = torch.zeros(n, h, hd)
        x[..., :20] = (torch.randint(0, 2, (n, h, 20), generator=g) * 2 - 1).float()
        return x.to(BF16)

    q, k = signs(N, heads), signs(N, 1)
    for row in (0, 200):
        q[row] = -k[row]
    return q, k, torch.randn(N, 1, hd, generator=g).to(BF16)


@pytest.mark.parametrize("heads", HEADS)
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("exponent", [18, 25, 29, 34, 60, 100, 122])
@pytest.mark.parametrize("biased", [False, True])
def test_finite_scores_of_any_size(biased, exponent, hd, heads):
    """Scores are n 2^exponent for whole n up to 20, exact in fp32 before the factor log2(e),
    whose rounding moves equal ones alike and unequal ones by 2^-22 of 20 2^exponent at most,
    less than a 10000th of what lies between them: the rows' largest score, and its ties,
    have all the weight, in any arithmetic.  -20 2^122 log2(e) is the largest that fp32 holds
    of these.  The bias of slope 0 changes nothing."""
    q, k, v = _ternary(300, heads, hd, exponent + hd)
    cu = _cu([200, 100])
    kw = {"slopes": torch.zeros(heads).cuda()} if biased else {}
    got = _prompt(q, k, v, cu, scale=2.0 ** exponent, **kw)
    some = [0, heads // 2, heads - 1]
    want, spread = ref.packed_prefill(q[:, some], k, v, cu, scale=2.0 ** exponent)
    _ok(got[:, some], want, spread)


@pytest.mark.parametrize("heads", HEADS)
@pytest.mark.parametrize("exponent", [20, 34, 100])
def test_large_scores_under_a_bias_stay_averages(heads, exponent):
    """A bias far below the scores' own rounding: which of the tied keys wins is open, but every
    output is an average of its row's visible values (to the weights' rounding, 2^-8, and
    the store's)."""
    q, k, v = _ternary(300, heads, 64, exponent)
    got = _prompt(q, k, v, _cu([200, 100]), scale=2.0 ** exponent,
                  slopes=torch.full((heads,), 0.3).cuda()).double()
    top = v.double().abs()
    for a, e in ((0, 200), (200, 300)):
        most = top[a:e].cummax(0).values
        assert bool((got[a:e].abs() <= most * (1 + 2.0 ** -8) ** 3).all())


@pytest.mark.parametrize("heads", HEADS)
def test_large_and_ordinary_rows_in_one_workgroup(heads):
    """One row's scores past 2^34 leave its neighbours' as they are."""
    _, (q, k, v) = _inputs(300, heads, 1, 64, 19)
    want, spread = ref.packed_prefill(q[:, :1], k, v, _cu([300]))
    q[100] = q[100] * 2.0 ** 40
    got = _prompt(q, k, v, _cu([300]))
    rows = [i for i in range(300) if i != 100]
    _ok(got[rows][:, :1], want[rows], spread[rows])
    assert bool((got[100].double().abs() <= v[:101].double().abs().amax(0) * (1 + 2.0 ** -6)).all())
