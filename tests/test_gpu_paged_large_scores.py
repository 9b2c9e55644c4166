"""Finite scores of any size in one-token attention.  Tolerance: that of
tests/test_gpu_paged.py; the scores here are exact or tie, as said at the test."""
import pytest
import torch

from oracle import paged as ref
from test_gpu_paged import _attn_ok, _decode_case, _ops

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("lens", [[300, 1, 33], [5000, 1, 40]])
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("exponent", [18, 34, 100, 122])
def test_finite_scores_of_any_size(exponent, fp8, hd, lens):
    """q and k of 20 entries +-1 each, scale 2^exponent: scores n 2^exponent for whole n up to
    20, of which the largest and its ties have all the weight."""
    g = torch.Generator().manual_seed(exponent + hd)
    q, kc, vc, table, n, _, vs = _decode_case(3, 8, 2, hd, 16, lens, fp8, g)

    def signs(t):
        x = torch.zeros(t.shape)
        x[..., :20] = (torch.randint(0, 2, (*t.shape[:-1], 20), generator=g) * 2 - 1).float()
        return x.to(t.dtype)

    q, kc = signs(q), signs(kc)
    q[1] = -kc[int(table[1, 0]), :, 0].to(q.dtype).repeat_interleave(4, 0)
    got = _ops().paged_attn_decode(q.cuda(), kc.cuda(), vc.cuda(), table.cuda(), n.cuda(),
                                   scale=2.0 ** exponent, v_scale=vs)
    want, spread = ref.paged_decode(q, kc, vc, table, n, scale=2.0 ** exponent, v_scale=vs)
    _attn_ok(got.cpu(), want, spread)


def test_values_under_the_smallest_scale():
    """130055 values of 448 under the smallest scale: their mean keeps its bits."""
    n, page = 130055, 256
    width = (n + page - 1) // page
    q = torch.zeros(1, 1, 64, dtype=torch.bfloat16, device="cuda")
    kc = torch.zeros(width, 1, page, 64, device="cuda").to(torch.float8_e4m3fn)
    vc = torch.full((width, 1, page, 64), 448.0, device="cuda").to(torch.float8_e4m3fn)
    table = torch.arange(width, dtype=torch.int32, device="cuda").view(1, -1)
    lens = torch.tensor([n], dtype=torch.int32, device="cuda")
    got = _ops().paged_attn_decode(q, kc, vc, table, lens, v_scale=2.0 ** -100).double()
    want = 448.0 * 2.0 ** -100
    assert bool(((got - want).abs() <= 2.0 ** -8 * want).all())
