"""Keys of a 4-bit cache after their norm and rotation: codes and scale bytes equal to the 64-bit
oracle's, also where a value lies so near to a border between two codes that one in 32 bits would
often fall on its other side.

What is left out: values within 2^-38 of their row's largest of a border.  Both sides are off by less:
a row's sum of squares (bf16 squares, exact, in 64 bits), its root, quotient and two products by
2^-48; an angle at a position p < 2^12 by 2 x 2^-53 p on the oracle's side (one product, one
argument) and 3 x 2^-53 p on the kernel's (a product with the frequency, one with 1 / 2 pi and that
number's own rounding): together 5 x 2^-41 of a pair, whose length is at most sqrt(2) of the largest:
2^-38.1; the parts under 2^-48 fit beside it."""
import pytest
import torch

from oracle import mx4 as ref
from oracle import paged

pytestmark = pytest.mark.gpu

BF16 = torch.bfloat16
OFF = 2.0 ** -38
BORDERS = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0], dtype=torch.float64)


def _ops():
    from hybrid_llm_amd import ops
    return ops


def _inv_freq(rot):
    return (10000.0 ** (-torch.arange(0, rot, 2, dtype=torch.float64) / rot)).float()


def _store(k, pos, inv_freq, weight, eps, interleaved):
    """(codes [N, H, hd / 2], bytes [N, H, hd / 32]) of keys k [N, H, hd] as the cache holds them."""
    N, H, hd = k.shape
    page = 16
    pages = -(-N // page)
    cache = _ops().mx4_cache(pages * 4096 // page if N == 1 else pages, H, page, hd)
    d = k.cuda()
    rows = torch.arange(N) // page  # a token its own slot, whatever its position
    width = 4096 // page
    table = torch.full((pages, width), -1, dtype=torch.int32)
    if N == 1:
        table[0] = torch.arange(width)
        ids, at = pos.long() // page, pos.long() % page
    else:
        ids, at = rows, pos.long() % page
        table[rows, pos.long() // page] = rows.int()
    fd, wd = (None if t is None else t.cuda() for t in (inv_freq, weight))
    _ops().paged_kv_append_mx4(d, d, *cache, table.cuda(), pos.int().cuda(), rows=rows.int().cuda(),
                               inv_freq=fd, k_norm=wd, eps=eps, interleaved=interleaved)
    return [t.view(torch.uint8).cpu()[ids, :, at] for t in (cache[0], cache[2])]


def _near(x, scales):
    """Which values of x [..., hd] a change by OFF of their row's largest can move to another code,
    by a border of codes or of their block's scale."""
    off = OFF * x.abs().amax(-1, keepdim=True)
    step = torch.exp2(scales.double() - 127).repeat_interleave(32, -1)
    near = (ref.round_to(x - off, step) != ref.round_to(x + off, step)) & (x.abs() > off)
    most = x.unflatten(-1, (-1, 32)).abs().amax(-1)
    turn = ref.steps((most - off).clamp_min(0)) != ref.steps(most + off)
    return near | turn.repeat_interleave(32, -1)


def _same(got, x, most_left_out):
    """Stored codes and bytes against the values x (fp64)."""
    codes, scales = ref.unpack(*got)
    want, want_s = ref.stored(x)
    left = _near(x, want_s)
    assert int(left.sum()) <= most_left_out, int(left.sum())
    assert torch.equal(scales.repeat_interleave(32, -1)[~left],
                       want_s.repeat_interleave(32, -1)[~left])
    wrong = (codes != want) & ~left
    assert not bool(wrong.any()), int(wrong.sum())


def _fp32(k, pos, inv_freq, weight, eps, interleaved):
    """The same keys formed in 32 bits but for their angles."""
    y = k.float()
    y = y * torch.rsqrt(y.square().mean(-1, keepdim=True) + eps) * weight
    half = inv_freq.numel()
    t = pos.double()[:, None, None] * inv_freq.double()
    c, s = t.cos().float(), t.sin().float()
    out = y.clone()
    a, b = (slice(0, 2 * half, 2), slice(1, 2 * half, 2)) if interleaved else (
        slice(0, half), slice(half, 2 * half))
    out[..., a] = y[..., a] * c - y[..., b] * s
    out[..., b] = y[..., b] * c + y[..., a] * s
    return out


def _beside_borders(hd, inv_freq, interleaved, seed):
    """A key, its position and norm weights whose normed and rotated values lie within 2^-22 of
    borders: the rotation undone, divided by the normed row and rounded to 32 bits."""
    g = torch.Generator().manual_seed(seed)
    x = ((0.5 + torch.rand(1, 1, hd, generator=g)) * 2.0 ** (seed % 5 - 2)).to(BF16)
    pos = torch.randint(1, 4096, (1,), generator=g)
    aim = BORDERS[torch.randint(0, 7, (hd,), generator=g)]
    aim[::32] = 6.0 if seed % 2 else 7.0  # a block's largest: no border, or the scale's
    aim = aim * torch.where(torch.rand(hd, generator=g) < 0.5, -1.0, 1.0)
    back = paged.norm_rope(aim.view(1, 1, hd), -pos, inv_freq, None, 0.0, interleaved)
    unit = paged.norm_rope(x, pos, None, torch.ones(hd), 0.0)
    return x, pos, (back / unit).view(hd).float()


@pytest.mark.parametrize("hd,rot,interleaved", [(64, 64, False), (128, 128, False), (64, 64, True),
                                                (128, 64, True), (128, 72, False)])
def test_beside_borders(hd, rot, interleaved):
    f = _inv_freq(rot)
    flips = 0
    for seed in range(24):
        x, pos, w = _beside_borders(hd, f, interleaved, seed)
        y = paged.norm_rope(x, pos, f, w, 0.0, interleaved)
        _same(_store(x, pos, f, w, 0.0, interleaved), y, 2)
        flips += int((ref.stored(_fp32(x, pos, f, w, 0.0, interleaved))[0] != ref.stored(y)[0]).sum())
    assert flips > 100, flips  # 32 bits do not do here


@pytest.mark.parametrize("N,H,hd,rot,interleaved", [(4096, 4, 128, 128, False), (4096, 8, 64, 48, True)])
def test_many(N, H, hd, rot, interleaved):
    """Two million keys; one within OFF of a border is expected once in thousands of such calls."""
    g = torch.Generator().manual_seed(N + hd)
    k = (torch.randn(N, H, hd, generator=g) * 3).to(BF16)
    w = 1 + 0.1 * torch.randn(hd, generator=g)
    pos = torch.arange(N) % 16 + 16 * torch.randint(0, 256, (N,), generator=g)
    f = _inv_freq(rot)
    codes, scales = _store(k, pos, f, w, 1e-6, interleaved)
    eps = float(torch.tensor(1e-6))  # as the call holds it
    for n in range(0, N, 512):
        x = paged.norm_rope(k[n:n + 512], pos[n:n + 512], f, w, eps, interleaved)
        _same((codes[n:n + 512], scales[n:n + 512]), x, 0)


def test_weights_alone_and_rotation_alone():
    """Without a rotation, and without a norm."""
    g = torch.Generator().manual_seed(5)
    k = (torch.randn(64, 3, 128, generator=g) * 3).to(BF16)
    pos = 1 + torch.arange(64)  # (at 0 a key is not turned, and may lie on a border)
    w, f = 1 + 0.1 * torch.randn(128, generator=g), _inv_freq(128)
    eps = float(torch.tensor(1e-6))
    _same(_store(k, pos, None, w, 1e-6, False), paged.norm_rope(k, pos, None, w, eps), 0)
    _same(_store(k, pos, f, None, 1e-6, False), paged.norm_rope(k, pos, f), 0)
    flat = (k.float().abs() + 0.5).to(BF16)[:1, :1]  # eps 0, weights onto borders
    aim = BORDERS[torch.randint(0, 7, (128,), generator=g)]
    aim[::32] = 6.0
    w = (aim / paged.norm_rope(flat, pos[:1], None, torch.ones(128), 0.0).view(128)).float()
    _same(_store(flat, pos[:1], None, w, 0.0, False), paged.norm_rope(flat, pos[:1], None, w, 0.0), 2)
