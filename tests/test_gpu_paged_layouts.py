"""Rows written in place of their inputs in layouts that interleave q, k and v: the bits of the
call with outputs of its own, and nothing else touched."""
import pytest
import torch

from test_gpu_paged import BF16, _inv_freq, _ops

pytestmark = pytest.mark.gpu

N, H, HD = 37, 5, 64


def _views(layout, x):
    """q, k, v [N, H, HD] of one buffer [3 N H HD]."""
    if layout == "fused rows":
        return [x.view(N, 3, H, HD)[:, i] for i in range(3)]
    if layout == "a head's q, k, v together":
        return [x.view(N, H, 3, HD)[:, :, i] for i in range(3)]
    if layout == "a head's tokens together":
        return [x.view(3, H, N, HD)[i].transpose(0, 1) for i in range(3)]
    return [x.view(H, N, 3, HD)[:, :, i].transpose(0, 1) for i in range(3)]


@pytest.mark.parametrize("layout", ["fused rows", "a head's q, k, v together",
                                    "a head's tokens together", "heads of tokens of q, k, v"])
def test_in_place(layout):
    g = torch.Generator().manual_seed(1)
    x = torch.randn(3 * N * H * HD, generator=g).to(BF16).cuda()
    pos = torch.randint(0, 1000, (N,), generator=g, dtype=torch.int32).cuda()
    f, w = _inv_freq(HD).cuda(), (torch.rand(HD, generator=g) + 0.5).cuda()
    q, k, v = _views(layout, x)
    want_q, want_k = _ops().qk_norm_rope(q, k, pos, f, q_norm=w, k_norm=w)
    y = x.clone()
    q, k, _ = _views(layout, y)
    _ops().qk_norm_rope(q, k, pos, f, q_norm=w, k_norm=w, q_out=q, k_out=k)
    assert torch.equal(q, want_q) and torch.equal(k, want_k)
    assert torch.equal(_views(layout, y)[2], v)
    z = x.clone()
    q, k, v = _views(layout, z)
    table = torch.randperm(N, generator=g).view(1, N).to(torch.int32).cuda()
    kc = torch.zeros(N, H, 16, HD, dtype=BF16, device="cuda")
    vc = torch.zeros_like(kc)
    at = torch.arange(N, dtype=torch.int32, device="cuda")
    got = _ops().paged_kv_append(k, v, kc, vc, table, at, rows=torch.zeros_like(at), inv_freq=f,
                                 q=q, q_norm=w, q_out=q)
    assert got is q
    want_q, want_k = _ops().qk_norm_rope(_views(layout, x)[0], k, at, f, q_norm=w)
    assert torch.equal(q, want_q)
    assert torch.equal(k, _views(layout, x)[1]) and torch.equal(v, _views(layout, x)[2])
    page, slot = table[0, at.long() // 16].long(), at.long() % 16
    assert torch.equal(kc[page, :, slot], want_k) and torch.equal(vc[page, :, slot], v)


def test_overlaps_raise():
    from hybrid_llm_amd._lib import LlmyError
    x = torch.ones(N + 1, 3 * H * HD, dtype=BF16, device="cuda")
    q, k = x[:N, :H * HD].view(N, H, HD), x[:N, H * HD:2 * H * HD].view(N, H, HD)
    pos = torch.zeros(N, dtype=torch.int32, device="cuda")
    below = x[1:, :H * HD].view(N, H, HD)
    for out in ({"q_out": k}, {"q_out": below}, {"k_out": q}, {"q_out": q, "k_out": q}):
        with pytest.raises(LlmyError):
            _ops().qk_norm_rope(q, k, pos, _inv_freq(HD).cuda(), **out)
    assert bool((x == 1).all())
