"""NaN scores in one-token attention: a query or a visible key with a NaN makes its rows NaN,
whatever waves or runs its head is cut into; other heads and sequences keep their
results.  Tolerance: that of tests/test_gpu_paged.py."""
import math

import pytest
import torch

from oracle import paged as ref
from test_gpu_paged import _attn_ok, _decode_case, _ops

pytestmark = pytest.mark.gpu

# a table short enough for a workgroup a head, and one that is cut into runs
TABLES = [100, 5000]


def _step(q, kc, vc, table, lens, ks, vs, **kw):
    return _ops().paged_attn_decode(q.cuda(), kc.cuda(), vc.cuda(), table.cuda(), lens.cuda(),
                                    k_scale=ks, v_scale=vs, **kw).cpu()


def _poison(kc, table, b, pos, page, head):
    """One NaN in the key of position pos of sequence b."""
    x = kc.float()
    x[int(table[b, pos // page]), head, pos % page, 9] = math.nan
    return x.to(kc.dtype)


@pytest.mark.parametrize("longest", TABLES)
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("fp8", [False, True])
def test_a_nan_query(fp8, hd, longest):
    g = torch.Generator().manual_seed(hd + longest)
    case = _decode_case(3, 8, 2, hd, 16, [longest, 33, 1], fp8, g)
    want, spread = ref.paged_decode(*case[:5], k_scale=case[5], v_scale=case[6])
    q = case[0].clone()
    q[0, 3, 5] = q[1, 6, 0] = q[2, 0, hd - 1] = math.nan
    got = _step(q, *case[1:])
    for b, h in ((0, 3), (1, 6), (2, 0)):
        assert got[b, h].isnan().all()
        got[b, h] = want[b, h].to(got.dtype)
    _attn_ok(got, want, spread)


@pytest.mark.parametrize("longest", TABLES)
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("window,first", [(0, 0), (69, 31)])
def test_a_nan_key_alone_in_its_step(window, first, fp8, hd, longest):
    """The only visible key of its 32-key step: the newest of 33, or the first of a window."""
    g = torch.Generator().manual_seed(hd + window)
    n, at = (100, 31) if window else (33, 32)
    case = _decode_case(3, 8, 2, hd, 16, [n, longest, n], fp8, g)
    want, spread = ref.paged_decode(*case[:5], window=window, k_scale=case[5], v_scale=case[6])
    kc = _poison(case[1], case[3], 0, at, 16, 1)
    got = _step(case[0], kc, *case[2:], window=window)
    assert got[0, 4:].isnan().all()
    got[0, 4:] = want[0, 4:].to(got.dtype)
    _attn_ok(got, want, spread)


@pytest.mark.parametrize("heads", [8, 1024])
@pytest.mark.parametrize("pos", [0, 40, 4000, 4999])
def test_a_nan_key_beside_far_larger_scores(pos, heads):
    """Scores of thousands: the NaN's run has no weight beside the others, but it is NaN."""
    g = torch.Generator().manual_seed(pos + 1)
    case = _decode_case(2, heads, 2, 64, 16, [5000, 40], False, g)
    kc = _poison(case[1], case[3], 0, pos, 16, 0)
    got = _step(case[0], kc, *case[2:], scale=64.0)
    assert got[0, :heads // 2].isnan().all()
    assert not got[0, heads // 2:].isnan().any() and not got[1].isnan().any()


@pytest.mark.parametrize("longest", TABLES)
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("keys", ["all", "but the last", "a whole step"])
def test_scores_of_minus_infinity(keys, hd, longest):
    """Beside a finite score they have no weight; alone their softmax is 0 / 0, as in a prompt's
    rows, where a sequence without a visible key gives zeros."""
    g = torch.Generator().manual_seed(hd + longest)
    q, kc, vc, table, lens, ks, vs = _decode_case(4, 8, 2, hd, 16, [77, longest, 0, 90], False, g)
    table[3] = -1
    q[..., 0] = q[..., 0].abs() + 0.125
    for t in range(77):
        if keys == "all" or keys == "but the last" and t < 76 or keys == "a whole step" and t < 32:
            kc[int(table[0, t // 16]), 1, t % 16, 0] = -math.inf
    want, spread = ref.paged_decode(q, kc, vc, table, lens)
    got = _step(q, kc, vc, table, lens, ks, vs)
    assert bool(want[0, 4:].isnan().all()) == (keys == "all")
    assert bool((got[2:] == 0).all())
    if keys == "all":
        assert got[0, 4:].isnan().all()
        prompt = _ops().packed_attn_prefill(
            q[:1].cuda(), kc[int(table[0, 0]), :, :1].transpose(0, 1).cuda(),
            torch.ones(1, 2, hd, dtype=q.dtype).cuda(),
            torch.tensor([0, 1], dtype=torch.int32).cuda()).cpu()
        assert prompt[0, 4:].isnan().all() and not prompt[0, :4].isnan().any()
        got[0, 4:] = 0
        want[0, 4:] = spread[0, 4:] = 0
    _attn_ok(got, want, spread)
