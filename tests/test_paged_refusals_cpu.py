"""Refusals of the paged-cache and rotation entry points, decided on the host before any
launch (no GPU needed), and their no-op sizes."""
import math

import pytest

FAKE = 0x10000  # non-null, 256-byte aligned; never dereferenced (validation fails first)
INVALID = 1

ROPE = dict(q=FAKE, q_row=512, q_head=64, k=FAKE, k_row=256, k_head=64, pos=FAKE, freq=FAKE,
            half=32, qn=FAKE, kn=FAKE, eps=1e-6, inter=0, qo=FAKE, qo_row=512, qo_head=64, ko=FAKE,
            ko_row=256, ko_head=64, N=4, Hq=8, Hkv=4, hd=64, stream=None)
APPEND = dict(k=FAKE, k_row=256, k_head=64, v=FAKE, v_row=256, v_head=64, kc=1 << 22, vc=1 << 23, kind=0,
              ks=1.0, vs=1.0, table=FAKE, rows=None, pos=FAKE, freq=FAKE, half=32, kn=FAKE,
              eps=1e-6, inter=0, q=FAKE, q_row=512, q_head=64, qn=FAKE, qo=FAKE, qo_row=512,
              qo_head=64, N=4, Hq=8, Hkv=4, hd=64, B=4, width=3, page=16, pages=12, stream=None)
DECODE = dict(q=1 << 20, q_row=512, q_head=64, kc=FAKE, vc=FAKE, kind=0, ks=1.0, vs=1.0, table=FAKE,
              lens=FAKE, slopes=None, out=FAKE, ws=FAKE, ws_bytes=1 << 30, B=4, Hq=8, Hkv=4,
              hd=64, width=90, page=16, pages=12, window=0, scale=0.125, cap=0.0, stream=None)

PACKED = dict(q=1 << 19, q_row=512, q_head=64, k=1 << 20, k_row=256, k_head=64, v=1 << 21, v_row=256,
              v_head=64, cu=FAKE, prefix=None, slopes=None, out=1 << 22, N=100, docs=3, Hq=8,
              Hkv=4, hd=64, window=0, scale=0.125, cap=0.0, stream=None)


def _call(fn, base, **change):
    return fn(*{**base, **change}.values())


@pytest.mark.parametrize("change", [
    {"hd": 96}, {"hd": 32}, {"Hq": 0}, {"Hkv": 0}, {"Hq": 1025}, {"N": -1}, {"half": 3},
    {"half": 36}, {"half": -4}, {"freq": None}, {"q": None}, {"k": None}, {"pos": None},
    {"qo": None}, {"ko": None}, {"q": FAKE + 2}, {"q_row": 510}, {"k_head": 66}, {"qn": FAKE + 8},
    {"eps": -1e-6}, {"q_head": 32}, {"qo_row": 32}, {"qo_head": 0}, {"q_row": -512},
])
def test_norm_rope_refuses(lib, change):
    assert _call(lib.llmy_qk_norm_rope_bf16, ROPE, **change) == INVALID


def test_norm_rope_of_no_rows(lib):
    assert _call(lib.llmy_qk_norm_rope_bf16, ROPE, N=0, q=None, k=None, pos=None) == 0


@pytest.mark.parametrize("change", [
    {"hd": 100}, {"Hkv": 0}, {"Hq": -1}, {"N": -1}, {"page": 15}, {"page": 8}, {"page": 512},
    {"page": 0}, {"page": 48}, {"pages": -1}, {"width": -1}, {"B": -1}, {"kind": 2}, {"ks": 0.5},
    {"kind": 1, "ks": 0.0}, {"kind": 1, "vs": -1.0}, {"kind": 1, "ks": math.inf},
    {"kind": 1, "vs": math.nan}, {"k": None}, {"v": None}, {"kc": None}, {"vc": (1 << 23) + 8},
    {"vc": 1 << 22}, {"vc": (1 << 22) + 12 * 4 * 16 * 64 * 2 - 16}, {"eps": -1.0}, {"eps": math.nan},
    {"kind": 1, "vc": (1 << 22) + 12 * 4 * 16 * 64 - 16},
    {"table": None}, {"pos": None}, {"q": None}, {"qo": None}, {"qo_row": 8}, {"half": 2},
    {"v_row": 258}, {"kn": FAKE + 4},
])
def test_append_refuses(lib, change):
    assert _call(lib.llmy_paged_kv_append, APPEND, **change) == INVALID


def test_append_of_no_tokens(lib):
    assert _call(lib.llmy_paged_kv_append, APPEND, N=0, k=None, kc=None, table=None) == 0


@pytest.mark.parametrize("change", [
    {"hd": 96}, {"Hq": 6}, {"Hkv": 0}, {"Hq": 0}, {"B": -1}, {"page": 17}, {"width": -1},
    {"pages": -1}, {"window": -1}, {"cap": -1.0}, {"cap": math.nan}, {"kind": 5}, {"vs": 2.0},
    {"kind": 1, "ks": math.nan}, {"q": None}, {"out": None}, {"lens": None}, {"table": None},
    {"kc": None}, {"scale": -0.1}, {"scale": math.nan}, {"vc": FAKE + 4}, {"q": (1 << 20) + 8}, {"cap": 1025.0}, {"cap": 1e-39, "scale": 1e3},
    {"scale": math.inf}, {"out": 1 << 20}, {"out": (1 << 20) + 4 * 1024 - 16}, {"q_row": 516}, {"q_head": 68},
    {"out": FAKE + 8}, {"ws": None}, {"ws": FAKE + 8}, {"ws_bytes": 64},
    {"width": 1 << 27, "page": 16},
])
def test_decode_refuses(lib, change):
    assert _call(lib.llmy_paged_attn_decode, DECODE, **change) == INVALID


def test_decode_of_no_sequences(lib):
    assert _call(lib.llmy_paged_attn_decode, DECODE, B=0, q=None, ws=None) == 0


@pytest.mark.parametrize("change", [
    {"hd": 80}, {"Hq": 6}, {"Hkv": 0}, {"Hq": 2048}, {"N": -1}, {"N": 1 << 30}, {"docs": -1},
    {"window": -1}, {"scale": -1.0}, {"scale": math.nan}, {"cap": -0.5}, {"cap": 2e3}, {"cap": math.nan}, {"q": None}, {"k": None},
    {"v": None}, {"out": None}, {"cu": None}, {"q": (1 << 19) + 8}, {"out": 1 << 19}, {"out": (1 << 22) + 8},
    {"k_row": 260}, {"v_head": 4}, {"q_row": -512}, {"k_row": 1 << 22},
    {"out": 1 << 20}, {"out": (1 << 20) + 99 * 512 + 496}, {"out": (1 << 21) - 16},
])
def test_prefill_refuses(lib, change):
    assert _call(lib.llmy_packed_attn_prefill_bf16, PACKED, **change) == INVALID


def test_prefill_of_nothing(lib):
    assert _call(lib.llmy_packed_attn_prefill_bf16, PACKED, N=0, q=None) == 0
    assert _call(lib.llmy_packed_attn_prefill_bf16, PACKED, docs=0, cu=None) == 0


def test_workspace_sizes(lib):
    ws = lib.llmy_paged_attn_workspace_bytes
    assert ws(4, 8, 4, 64, 64, 16, 0) == 0         # 1024 tokens: a workgroup a head
    assert ws(4, 8, 4, 128, 32, 16, 0) == 0        # 512
    assert ws(4, 8, 4, 128, 33, 16, 0) > 0
    assert ws(4, 8, 4, 64, 65, 16, 0) > 0
    assert ws(4, 8, 3, 64, 9, 16, 0) == -1
    assert ws(4, 8, 4, 64, 9, 20, 0) == -1
    # the length does not change it, a sequence takes one word
    assert ws(1, 8, 4, 64, 900, 16, 0) == ws(1, 8, 4, 64, 65, 16, 0)
    assert ws(400, 8, 4, 64, 900, 16, 0) == ws(1, 8, 4, 64, 65, 16, 0) + 399 * 4


def test_wrappers_refuse_before_the_library():
    import torch
    from hybrid_llm_amd import ops
    b = torch.bfloat16
    q, k = torch.zeros(4, 8, 64, dtype=b), torch.zeros(4, 4, 64, dtype=b)
    pos, freq = torch.zeros(4, dtype=torch.int32), torch.zeros(32)
    cache = torch.zeros(12, 4, 16, 64, dtype=b)
    table = torch.zeros(4, 3, dtype=torch.int32)
    for bad in (dict(k_cache=cache.float()), dict(v_cache=cache[:, :2]), dict(positions=pos.long()),
                dict(k=k.float()), dict(page_table=table.long()), dict(page_table=table[0]),
                dict(page_table=table[:3]), dict(q_norm=freq), dict(rows=pos[:3]),
                dict(inv_freq=freq.double()), dict(k_cache=cache.transpose(0, 1)),
                dict(v=k[..., ::2])):
        args = {**dict(k=k, v=k, k_cache=cache, v_cache=cache, page_table=table, positions=pos),
                **bad}
        with pytest.raises(ValueError):
            ops.paged_kv_append(**args)
    for bad in (dict(q=q.half()), dict(lengths=pos[:2]), dict(lengths=pos.long()),
                dict(page_table=table[:2]), dict(slopes=torch.zeros(4)), dict(out=q.float()),
                dict(v_cache=cache.to(torch.float8_e4m3fn))):
        args = {**dict(q=q, k_cache=cache, v_cache=cache, page_table=table, lengths=pos), **bad}
        with pytest.raises(ValueError):
            ops.paged_attn_decode(**args)
    cu = torch.tensor([0, 4], dtype=torch.int32)
    for bad in (dict(q=q.half()), dict(v=k[:3]), dict(cu_seqlens=cu.long()), dict(cu_seqlens=cu[:0]),
                dict(prefix=pos), dict(slopes=freq), dict(out=q.transpose(0, 1)),
                dict(k=k[..., :32])):
        args = {**dict(q=q, k=k, v=k, cu_seqlens=cu), **bad}
        with pytest.raises(ValueError):
            ops.packed_attn_prefill(**args)
