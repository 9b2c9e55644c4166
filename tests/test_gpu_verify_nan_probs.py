"""Draft distributions with a NaN here and there: such an entry counts as 0, its draft is not kept.

Tokens equal the 64-bit oracle's; both sides sum in 64 bits, off by 2^-52 V of a row's whole at
most, and no decision of these inputs lies within 2^-28 of its border."""
import math

import pytest
import torch

from oracle import drafts as ref

pytestmark = pytest.mark.gpu
NEAR = 2.0 ** -28


def _run(logits, ids, u, q):
    from hybrid_llm_amd import ops
    tokens, accepted = ops.verify_drafts(logits.cuda(), ids.cuda(), u.cuda(), temperature=1.0,
                                         draft_probs=q.cuda())
    return tokens.cpu(), accepted.cpu()


# few sequences: decisions, sums and draw in one launch; many: in three
@pytest.mark.parametrize("B,V", [(1, 5000), (3, 1001), (40, 40000)])
def test_the_id_that_the_draw_takes(B, V):
    """Nearly all of the target's weight at an id whose draft probability is NaN, and a little at one
    that the drafts do not have."""
    g = torch.Generator().manual_seed(V)
    K = 2
    logits = torch.randn(B, K + 1, V, generator=g)
    q = torch.softmax(torch.randn(B, K, V, generator=g), -1)
    at = torch.randint(0, V, (B,), generator=g)
    ids, other = ((at[:, None] + 1 + torch.arange(K)) % V).int(), (at + V // 2) % V
    b = torch.arange(B)
    logits[b, 0, at], logits[b, 0, other] = 30.0, 25.0
    q[b, 0, at], q[b, 0, other] = math.nan, 0.0
    u = 0.1 + 0.8 * torch.rand(B, K + 1, generator=g)
    q[b, 0, ids[:, 0].long()] = 0.5  # far above the target's: put away
    tokens, accepted = _run(logits, ids, u, q)
    assert not accepted.any() and torch.equal(tokens[:, 0].long(), at)


@pytest.mark.parametrize("B,K,V,seed", [(1, 4, 32000, 0), (5, 3, 777, 1), (48, 4, 30001, 2)])
def test_a_few_of_many(B, K, V, seed):
    """One entry in ten, and every third draft's own."""
    g = torch.Generator().manual_seed(seed)
    logits = torch.randn(B, K + 1, V, generator=g) * 2.5
    q = torch.softmax(logits[:, :K] + torch.randn(B, K, V, generator=g), -1)
    ids = torch.multinomial(q.view(-1, V), 1, generator=g).view(B, K).int()
    u = torch.rand(B, K + 1, generator=g)
    bad = torch.rand(B, K, V, generator=g) < 0.1
    own = torch.arange(B * K).view(B, K) % 3 == 2
    bad.scatter_(2, ids[..., None].long(), own[..., None])
    q[bad] = math.nan
    want, kept, margin = ref.verify(logits, ids, u, 1.0, q)
    assert float(margin.min()) > NEAR
    tokens, accepted = _run(logits, ids, u, q)
    assert torch.equal(accepted, kept) and torch.equal(tokens, want)
    assert bool((accepted <= 2).all()) or B == 1
