"""Per-head norms of rows of any magnitude."""
import math

import pytest
import torch

from oracle import paged as ref
from test_gpu_paged import BF16, _inv_freq, _ops, _rope_ok

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("N,heads,hd", [(6, 2, 64), (37, 5, 128), (1100, 60, 64)])
@pytest.mark.parametrize("eps", [0.0, 1e-30, 1e-6])
def test_norm_over_the_whole_range(eps, N, heads, hd):
    """Rows of any magnitude, ordinary ones among them: 2^-19 of a row's largest value, as
    derived in tests/test_gpu_paged.py, where squares in fp32 would overflow or vanish."""
    g = torch.Generator().manual_seed(N + hd)
    size = [2.0 ** e for e in (0, 64, 100, 125, -20, -50, -64, -80, -110, 30, 60, 1)]
    x = torch.randn(N, heads, hd, generator=g).clamp(-3, 3)
    row = torch.arange(N * heads).view(N, heads) * 7 % 12
    x = (x * torch.tensor(size)[row][..., None]).to(BF16)
    x[0, 0] = (torch.linspace(-1, 1, hd) * 3.38e38).to(BF16)
    x[0, 1, :] = 0
    x[0, 1, 3] = 2.0 ** 127
    if eps:
        x[1, 0] = 0
    pos = torch.randint(0, 5000, (N,), generator=g, dtype=torch.int32)
    f, w = _inv_freq(hd), torch.rand(hd, generator=g) + 0.5
    qo, ko = _ops().qk_norm_rope(x.cuda(), x[:, :1].contiguous().cuda(), pos.cuda(), f.cuda(),
                                 q_norm=w.cuda(), k_norm=w.cuda(), eps=eps)
    want = ref.norm_rope(x, pos, f, w, eps)
    assert bool(want.isfinite().all())
    _rope_ok(qo.cpu(), want)
    _rope_ok(ko.cpu(), want[:, :1])


def test_norm_of_infinite_rows():
    """x / inf: 0 for the finite ones of the row, NaN for infinities, without a rotation."""
    x = torch.ones(2, 3, 64)
    x[0, 0, 5] = math.inf
    x[0, 1, 6] = -math.inf
    x[1, 2, 7] = math.nan
    x = x.to(BF16)
    pos = torch.zeros(2, dtype=torch.int32)
    w = torch.ones(64)
    qo, _ = _ops().qk_norm_rope(x.cuda(), x.cuda(), pos.cuda(), q_norm=w.cuda())
    want = ref.norm_rope(x, pos, None, w)
    assert torch.equal(qo.cpu().isnan(), want.isnan())
    assert torch.equal(qo.cpu().double().nan_to_num(9.0)[0, :2], want.nan_to_num(9.0)[0, :2])
