"""Every bf16 value through the append to a paged cache."""
import pytest
import torch

from test_gpu_paged import BF16, FP8, _ops

pytestmark = pytest.mark.gpu


def _all_bf16():
    """[1024, 1, 64]: every 16-bit pattern."""
    bits = torch.arange(65536, dtype=torch.int32).to(torch.int16)
    return bits.view(BF16).view(1024, 1, 64)


def _append_all(dtype, **kw):
    x = _all_bf16().cuda()
    kc = torch.zeros(64, 1, 16, 64, device="cuda").to(dtype)
    vc = torch.zeros_like(kc)
    table = torch.arange(64, dtype=torch.int32, device="cuda").view(1, 64)
    pos = torch.arange(1024, dtype=torch.int32, device="cuda")
    _ops().paged_kv_append(x, x, kc, vc, table, pos, rows=torch.zeros_like(pos), **kw)
    return kc.cpu().view(1024, 1, 64), vc.cpu().view(1024, 1, 64)


@pytest.mark.parametrize("scale", [0.3, 7 / 64, 13 / 64, 0.875, 0.021, 3.0, 60.0, 1.0, 1e30,
                                   1e-30, 2.0 ** -100, 7 * 2.0 ** -102])
def test_e4m3_codes_of_every_value(scale):
    """x / scale in fp32, saturated, to nearest even: the same codes as on the CPU."""
    x = _all_bf16()
    want = (x.float() / torch.tensor(scale, dtype=torch.float32)).clamp(-448, 448).to(FP8)
    bad = x.isnan()
    for got in _append_all(FP8, k_scale=scale, v_scale=scale):
        assert bool(got.float().isnan()[bad].all()) and not bool(got.float().isnan()[~bad].any())
        assert torch.equal(got.view(torch.uint8)[~bad], want.view(torch.uint8)[~bad])


def test_bf16_cache_holds_every_value():
    x = _all_bf16()
    bad = x.isnan()
    for got in _append_all(BF16):
        assert torch.equal(got.isnan(), bad)
        assert torch.equal(got.view(torch.int16)[~bad], x.view(torch.int16)[~bad])
