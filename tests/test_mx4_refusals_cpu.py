"""The 4-bit cache, page planning and draft verification: calls refused before any launch, and
calls of nothing, which need no GPU."""
import pytest
import torch

from hybrid_llm_amd import ops

INVALID = 1
P = 0x10000       # non-null, aligned, never dereferenced
FAR = 0x10000000  # so far apart that no range meets another


def at(i):
    return P + i * FAR


def append(lib, **over):
    a = dict(k=at(0), k_row=256, k_head=128, v=at(1), v_row=256, v_head=128, kc=at(2), vc=at(3),
             ks=at(4), vs=at(5), table=at(6), rows=None, pos=at(7), inv=at(8), half=64, kn=None,
             eps=1e-6, il=0, q=None, q_row=0, q_head=0, qn=None, qo=None, qo_row=0, qo_head=0, N=3,
             Hq=0, Hkv=2, hd=128, B=3, width=4, page=16, pages=12, stream=None)
    assert set(over) <= set(a)
    return lib.llmy_paged_kv_append_mx4(*{**a, **over}.values())


@pytest.mark.parametrize("over", [
    {"k": None}, {"v": None}, {"kc": None}, {"vc": None}, {"ks": None}, {"vs": None},
    {"table": None}, {"pos": None}, {"inv": None}, {"half": 62}, {"half": 68}, {"hd": 96},
    {"page": 24}, {"page": 8}, {"page": 512}, {"N": -1}, {"Hkv": 0}, {"eps": -1.0},
    {"eps": float("nan")}, {"kc": at(2) + 8}, {"vc": at(3) + 4}, {"ks": at(4) + 2},
    {"vs": at(5) + 1}, {"k": at(0) + 2}, {"k_row": 255}, {"kn": at(9) + 4}, {"pages": -1},
    {"width": -1}, {"B": -1}, {"Hq": 4}, {"Hkv": 1025},
    # the parts of the cache on each other, or on rows
    {"vc": at(2)}, {"ks": at(2) + 64}, {"vs": at(4) + 4}, {"kc": at(0)}, {"vs": at(1) + 512},
    # queries written over the cache, or read from where it is written
    {"Hq": 2, "q": at(10), "q_row": 256, "q_head": 128, "qo": at(4), "qo_row": 256, "qo_head": 128},
    {"Hq": 2, "q": at(3), "q_row": 256, "q_head": 128, "qo": at(10), "qo_row": 256, "qo_head": 128},
    {"Hq": 2, "q": at(10), "q_row": 256, "q_head": 128, "qo": at(0), "qo_row": 256, "qo_head": 128},
])
def test_append_refuses(lib, over):
    assert append(lib, **over) == INVALID


def test_append_of_nothing(lib):
    assert append(lib, N=0) == 0


def read(lib, **over):
    a = dict(kc=at(0), vc=at(1), ks=at(2), vs=at(3), table=at(4), rows=None, pos=at(5), k=at(6),
             v=at(7), N=3, Hkv=2, hd=64, B=3, width=4, page=16, pages=12, stream=None)
    assert set(over) <= set(a)
    return lib.llmy_paged_kv_read_mx4(*{**a, **over}.values())


@pytest.mark.parametrize("over", [
    {"kc": None}, {"vs": None}, {"table": None}, {"pos": None}, {"k": None}, {"v": None},
    {"k": at(6) + 8}, {"v": at(6)}, {"v": at(6) + 512}, {"k": at(0)}, {"v": at(3) + 16},
    {"hd": 32}, {"page": 0}, {"N": -1}, {"Hkv": 0}, {"pages": -1}, {"vs": at(3) + 1},
])
def test_read_refuses(lib, over):
    assert read(lib, **over) == INVALID


def test_read_of_nothing(lib):
    assert read(lib, N=0) == 0


def attn(lib, **over):
    a = dict(q=at(0), q_seq=512, q_row=256, q_head=64, kc=at(1), vc=at(2), ks=at(3), vs=at(4),
             table=at(5), lengths=at(6), slopes=None, out=at(7), ws=at(8), wsb=1 << 30, B=2, T=2,
             Hq=4, Hkv=2, hd=64, width=4, page=16, pages=12, window=0, scale=0.125, cap=0.0,
             stream=None)
    assert set(over) <= set(a)
    return lib.llmy_paged_attn_mx4(*{**a, **over}.values())


@pytest.mark.parametrize("over", [
    {"q": None}, {"kc": None}, {"ks": None}, {"vs": None}, {"table": None}, {"lengths": None},
    {"out": None}, {"T": 0}, {"T": 65}, {"Hq": 5}, {"Hq": 0}, {"Hq": 2048, "Hkv": 1024},
    {"hd": 80}, {"page": 48}, {"window": -1}, {"scale": -1.0}, {"scale": float("inf")},
    {"scale": float("nan")}, {"cap": 2048.0}, {"cap": -1.0}, {"q": at(0) + 8}, {"q_seq": 4},
    {"q_row": -256}, {"q_head": 2}, {"out": at(7) + 2}, {"pages": -1}, {"B": -1},
    {"kc": at(1) + 4}, {"ks": at(3) + 1},
    {"out": at(0)}, {"out": at(0) + 1024}, {"out": at(1)}, {"out": at(4) + 16},
    {"q_seq": 1 << 60},
    # a long table needs its workspace, apart from all else
    {"width": 1024, "ws": None}, {"width": 1024, "wsb": 64}, {"width": 1024, "ws": at(8) + 4},
    {"width": 1024, "ws": at(7)}, {"width": 1024, "ws": at(2)}, {"width": 1024, "ws": at(0)},
    {"width": 1 << 27},
])
def test_attention_refuses(lib, over):
    assert attn(lib, **over) == INVALID


def test_attention_of_nothing_and_its_workspace(lib):
    assert attn(lib, B=0) == 0
    size = lib.llmy_paged_attn_mx4_workspace_bytes
    assert size(2, 1, 4, 2, 64, 4, 16, 0) == 0           # short: none
    assert size(2, 1, 4, 2, 64, 1024, 16, 0) > 0
    assert size(2, 1, 4, 2, 64, 1024, 16, 64) == 0    # short by its window
    assert size(2, 1, 4, 3, 64, 4, 16, 0) == -1
    assert size(2, 0, 4, 2, 64, 4, 16, 0) == -1
    assert size(2, 1, 4, 2, 64, 4, 16, -1) == -1


def plan(lib, **over):
    a = dict(lengths=at(0), new=at(1), reset=None, table=at(2), held=at(3), free=at(4),
             n_free=at(5), cu=at(6), rows=at(7), pos=at(8), out=at(9), ws=None, wsb=0, B=4, width=8,
             page=16, free_capacity=64, capacity=100, stream=None)
    assert set(over) <= set(a)
    return lib.llmy_paged_plan(*{**a, **over}.values())


@pytest.mark.parametrize("over", [
    {"lengths": None}, {"new": None}, {"table": None}, {"held": None}, {"free": None},
    {"n_free": None}, {"cu": None}, {"rows": None}, {"pos": None}, {"out": None}, {"B": -1},
    {"B": 4097}, {"width": -1}, {"width": 1 << 27}, {"page": 20}, {"free_capacity": -1},
    {"capacity": -1}, {"capacity": 5000}, {"capacity": 5000, "ws": at(10), "wsb": 8},
    {"held": at(0)}, {"out": at(1)}, {"pos": at(7) + 396}, {"free": at(2) + 4}, {"reset": at(3)},
    {"n_free": at(4) + 252}, {"cu": at(9) + 12},
])
def test_plan_refuses(lib, over):
    assert plan(lib, **over) == INVALID


def verify(lib, **over):
    a = dict(logits=at(0), drafts=at(1), probs=None, counts=None, u=at(2), T=1.0, tokens=at(3),
             accepted=at(4), ws=at(5), wsb=1 << 20, B=2, K=3, V=1000, stream=None)
    assert set(over) <= set(a)
    return lib.llmy_verify_drafts_f32(*{**a, **over}.values())


@pytest.mark.parametrize("over", [
    {"logits": None}, {"drafts": None}, {"u": None}, {"tokens": None}, {"accepted": None},
    {"ws": None}, {"ws": at(5) + 4}, {"wsb": 16}, {"K": 0}, {"K": 64}, {"V": 0},
    {"V": (1 << 30) + 1}, {"B": -1}, {"T": float("nan")}, {"T": float("inf")},
    {"tokens": at(1)}, {"accepted": at(3) + 4}, {"tokens": at(0) + 4000}, {"accepted": at(2)},
    {"ws": at(0)}, {"probs": at(6), "accepted": at(6) + 23996}, {"counts": at(4)},
])
def test_verify_refuses(lib, over):
    assert verify(lib, **over) == INVALID


def test_verify_of_nothing_and_its_workspace(lib):
    assert verify(lib, B=0) == 0
    assert lib.llmy_verify_drafts_workspace_bytes(2, 3, 1000) == 16 * (2 * 4 + 2) + 2 * 32
    assert lib.llmy_verify_drafts_workspace_bytes(2, 64, 1000) == -1


def test_wrappers_name_what_is_wrong():
    cache = ops.mx4_cache(4, 2, 16, 64, device="cpu")
    assert [tuple(t.shape) for t in cache] == [(4, 2, 16, 32)] * 2 + [(4, 2, 16, 2)] * 2
    i32 = torch.zeros(3, dtype=torch.int32)
    row = torch.zeros(3, 2, 64, dtype=torch.bfloat16)
    table = torch.zeros(3, 4, dtype=torch.int32)
    with pytest.raises(ValueError, match="k must be"):  # on the CPU
        ops.paged_kv_append_mx4(row, row, *cache, table, i32)
    with pytest.raises(ValueError, match="4-bit cache"):
        ops.paged_kv_read_mx4(*cache, table, i32)
    with pytest.raises(ValueError, match="q must be"):
        ops.paged_attn_mx4(row, *cache, table, i32)
    with pytest.raises(ValueError, match="page_table"):
        ops.paged_plan(i32, i32, i32, i32, i32, i32, 16, 4)
    with pytest.raises(ValueError, match="logits must be"):
        ops.verify_drafts(torch.zeros(2, 3, 10), torch.zeros(2, 3, dtype=torch.int32))
