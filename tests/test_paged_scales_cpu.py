"""Scales that fp32 does not carry through the kernels are refused on the host (no GPU
needed)."""
import math

import pytest

from test_paged_refusals_cpu import APPEND, DECODE, INVALID, PACKED, _call


@pytest.mark.parametrize("name", ["ks", "vs"])
@pytest.mark.parametrize("scale", [2.0 ** -149, 1e-39, 2.0 ** -127, 2.0 ** -101, 2.0 ** 101, 3e38])
def test_cache_scales_outside_the_range(lib, name, scale):
    """Among them those whose reciprocal is infinite: a stored 0 would become NaN."""
    change = {"kind": 1, "vc": 1 << 23, name: scale}
    assert _call(lib.llmy_paged_kv_append, APPEND, **change) == INVALID
    assert _call(lib.llmy_paged_attn_decode, DECODE, kind=1, **{name: scale}) == INVALID


@pytest.mark.parametrize("scale", [2.4e38, 3.4e38])
def test_score_scales_that_overflow_in_log2_units(lib, scale):
    assert scale * math.log2(math.e) > 3.4028235e38
    assert _call(lib.llmy_paged_attn_decode, DECODE, scale=scale) == INVALID
    assert _call(lib.llmy_packed_attn_prefill_bf16, PACKED, scale=scale) == INVALID
    # the scale that counts is the one beside the cache's
    assert _call(lib.llmy_paged_attn_decode, DECODE, kind=1, scale=scale / 4, ks=4.0) == INVALID


@pytest.mark.parametrize("scale", [2.0 ** -100, 1e-30, 1.0, 2.0 ** 100])
def test_the_ends_of_the_range_pass(lib, scale):
    """Seen by a call of no tokens and one of no sequences, whose scales are looked at."""
    assert _call(lib.llmy_paged_kv_append, APPEND, kind=1, ks=scale, vs=scale, N=0) == 0
    assert _call(lib.llmy_paged_attn_decode, DECODE, kind=1, ks=scale, vs=scale, B=0) == 0
