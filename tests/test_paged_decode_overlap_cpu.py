"""Overlaps of what one-token attention writes with what its other workgroups read are refused
on the host (no GPU needed)."""
import pytest

from conftest import gpu_available
from test_paged_refusals_cpu import INVALID, _call

Q, KC, VC, OUT, WS = 1 << 23, 1 << 24, 1 << 26, 1 << 25, 1 << 28
CACHE = 120 * 4 * 16 * 64 * 2    # bytes
DECODE = dict(q=Q, q_row=512, q_head=64, kc=KC, vc=VC, kind=0, ks=1.0, vs=1.0,
              table=1 << 16, lens=1 << 16, slopes=None, out=OUT, ws=WS, ws_bytes=1 << 26, B=4,
              Hq=8, Hkv=4, hd=64, width=90, page=16, pages=120, window=0, scale=0.125, cap=0.0,
              stream=None)


def _workspace(lib):
    return lib.llmy_paged_attn_workspace_bytes(4, 8, 4, 64, 90, 16, 0)


@pytest.mark.parametrize("change", [
    {"out": KC}, {"out": KC + CACHE - 16}, {"out": VC}, {"out": VC - 4 * 8 * 64 * 2 + 16},
    {"ws": KC}, {"ws": KC + CACHE - 16}, {"ws": VC + 1024}, {"ws": OUT}, {"ws": OUT + 1024},
    {"ws": Q}, {"ws": Q + 2 * (3 * 512 + 504)}, {"out": WS}, {"q": WS + 4096},
    {"kind": 1, "out": KC + CACHE // 2 - 16},
], ids=str)
def test_decode_refuses_overlaps(lib, change):
    assert _workspace(lib) > 4096
    assert _call(lib.llmy_paged_attn_decode, DECODE, **change) == INVALID


def test_a_workspace_that_ends_in_an_operand(lib):
    for at in (KC, VC, OUT, Q):
        ws = at - _workspace(lib) // 16 * 16 + 16
        assert _call(lib.llmy_paged_attn_decode, DECODE, ws=ws) == INVALID


@pytest.mark.skipif(gpu_available(), reason="addresses that name no memory")
@pytest.mark.parametrize("change", [
    {}, {"vc": KC}, {"out": KC + CACHE}, {"ws": KC + CACHE}, {"out": VC - 4 * 8 * 64 * 2},
    {"ws": OUT + 4 * 8 * 64 * 2}, {"kind": 1, "out": KC + CACHE // 2},
    {"width": 9, "ws": KC}, {"width": 9, "ws": None, "ws_bytes": 0},   # short tables take none
], ids=str)
def test_decode_takes_what_lies_apart(lib, change):
    """Such a call ends at the launch here, for want of a device."""
    assert _call(lib.llmy_paged_attn_decode, DECODE, **change) not in (0, INVALID)
