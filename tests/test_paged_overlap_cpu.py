"""Overlaps of what the rotation and append entry points write with what other waves read are
refused on the host; rows that merely interleave are not (no GPU needed)."""
import pytest

from conftest import gpu_available
from test_paged_refusals_cpu import INVALID, _call

ROW = (8 + 2 * 4) * 64           # elements of one fused row: 8 query heads, 4 + 4 of k and v
BASE = 1 << 24                   # bytes
OUT, OUT2 = 1 << 26, 1 << 27     # far from it

ROPE = dict(q=BASE, q_row=ROW, q_head=64, k=BASE + 2 * 512, k_row=ROW, k_head=64, pos=1 << 20,
            freq=1 << 20, half=32, qn=1 << 20, kn=1 << 20, eps=1e-6, inter=0, qo=OUT, qo_row=512,
            qo_head=64, ko=OUT2, ko_row=256, ko_head=64, N=5, Hq=8, Hkv=4, hd=64, stream=None)
APPEND = dict(k=BASE + 2 * 512, k_row=ROW, k_head=64, v=BASE + 2 * 768, v_row=ROW, v_head=64,
              kc=1 << 22, vc=1 << 23, kind=0, ks=1.0, vs=1.0, table=1 << 20, rows=None,
              pos=1 << 20, freq=1 << 20, half=32, kn=1 << 20, eps=1e-6, inter=0, q=BASE,
              q_row=ROW, q_head=64, qn=1 << 20, qo=OUT, qo_row=512, qo_head=64, N=5, Hq=8,
              Hkv=4, hd=64, B=5, width=3, page=16, pages=12, stream=None)
IN_PLACE = dict(qo=BASE, qo_row=ROW)
K_IN_PLACE = dict(ko=BASE + 2 * 512, ko_row=ROW)
CACHE = 12 * 4 * 16 * 64 * 2     # bytes of a bf16 cache


@pytest.mark.parametrize("change", [
    {"ko": OUT},                                         # the outputs on each other
    {"ko": OUT + 2 * (4 * 512 + 448)},                   # the last of q_out's blocks
    {"qo": BASE + 2 * 512, "qo_row": ROW},               # q_out over k and v
    {"qo": BASE + 2 * 64, "qo_row": ROW},                # one head beside its own rows
    {"qo": BASE + 2 * ROW, "qo_row": ROW},               # one token beside them
    {"qo": BASE + 2 * 4, "qo_row": ROW},                 # a few elements beside them
    {"qo": BASE, "qo_row": 512},                         # on its rows at another pitch
    {"qo": BASE, "qo_row": ROW, "qo_head": 128},         # or another head stride
    {"ko": BASE, "ko_row": ROW},                         # k_out over q
    {"ko": BASE + 2 * (512 + 64), "ko_row": ROW},        # one head beside its own rows
    {**IN_PLACE, "ko": BASE + 2 * 448, "ko_row": ROW},   # over the last query head
    {"ko_row": 64},                                      # (n, h + 1) and (n + 1, h) on one row
    {"qo_row": 64}, {"qo_row": 256}, {"qo_row": 448}, {"qo_row": 0},
    {"qo_row": 1 << 62},                                 # past any memory
], ids=str)
def test_norm_rope_refuses_overlaps(lib, change):
    assert _call(lib.llmy_qk_norm_rope_bf16, ROPE, **change) == INVALID


@pytest.mark.parametrize("change", [
    {"qo": BASE + 2 * 512, "qo_row": ROW},               # q_out over k
    {"qo": BASE + 2 * 768, "qo_row": ROW},               # over v
    {"qo": BASE + 2 * 64, "qo_row": ROW}, {"qo": BASE, "qo_row": 512}, {"qo_row": 64},
    {"qo": 1 << 22}, {"qo": (1 << 22) + CACHE - 8}, {"qo": (1 << 22) - 5 * 512 * 2 + 8},
    {"qo": 1 << 23}, {"qo": (1 << 23) + CACHE - 8},
], ids=str)
def test_append_refuses_overlaps(lib, change):
    assert _call(lib.llmy_paged_kv_append, APPEND, **change) == INVALID


# A call that passes the checks ends at the launch here, for want of a device.
no_gpu = pytest.mark.skipif(gpu_available(), reason="addresses that name no memory")

HEAD_MAJOR = dict(q_row=64, q_head=5 * 64, k=BASE + 2 * 8 * 5 * 64, k_row=64, k_head=5 * 64)
PER_HEAD = dict(Hq=4, Hkv=4, q_row=4 * 192, q_head=192, k=BASE + 2 * 64, k_row=4 * 192, k_head=192)


@no_gpu
@pytest.mark.parametrize("change", [
    {}, IN_PLACE, K_IN_PLACE, {**IN_PLACE, **K_IN_PLACE},
    {"ko": OUT + 2 * 5 * 512},                                        # right behind q_out
    {"qo": OUT, "qo_row": ROW, "ko": OUT + 2 * 512, "ko_row": ROW},   # one new fused row
    {"qo": BASE + 2 * ROW * 5, "qo_row": ROW},                        # right behind the input
    {**HEAD_MAJOR, "qo": BASE, "qo_row": 64, "qo_head": 5 * 64, "ko": HEAD_MAJOR["k"],
     "ko_row": 64, "ko_head": 5 * 64},
    {**PER_HEAD, "qo": BASE, "qo_row": 4 * 192, "qo_head": 192, "ko": BASE + 2 * 64,
     "ko_row": 4 * 192, "ko_head": 192},
    {"N": 1, "qo_row": 0, "ko_row": 0}, {"N": 1, "qo_row": 1 << 62},
    {"q_row": 0, "k_row": 0},                                         # one row for every token
], ids=str)
def test_norm_rope_takes_rows_that_lie_apart(lib, change):
    assert _call(lib.llmy_qk_norm_rope_bf16, ROPE, **change) not in (0, INVALID)


@no_gpu
@pytest.mark.parametrize("change", [
    {}, IN_PLACE, {"qo": (1 << 22) + CACHE}, {"qo": (1 << 22) - 5 * 512 * 2},
    {"kind": 1, "qo": (1 << 22) + CACHE // 2}, {"Hq": 0, "q": None, "qo": None, "qn": None},
], ids=str)
def test_append_takes_rows_that_lie_apart(lib, change):
    assert _call(lib.llmy_paged_kv_append, APPEND, **change) not in (0, INVALID)
