"""The serving step with drafted tokens as the documents give it, run on the CPU with the oracles in
the operators' place: what it makes of each sequence's length and last token."""
import types
from pathlib import Path

import torch

from oracle import drafts as ref

B, K, V, Hq, Hkv, hd, page, pages = 6, 3, 50, 4, 2, 64, 16, 64
T = K + 1


def _example():
    """The one block of python in the documents that plans, verifies and goes on."""
    found = [part.split("```")[0] for f in sorted(Path(__file__).resolve().parents[1].glob("*.md"))
             for part in f.read_text().split("```python\n")[1:]]
    found = [b for b in found if "ops.paged_plan(" in b and "ops.verify_drafts(" in b]
    assert len(found) == 1
    return found[0]


def test_lengths_and_tokens_after_a_step():
    i32 = dict(dtype=torch.int32)
    names = ("an ordinary one", "reset", "refused", "reset and refused", "at a page's end", "reset")
    lengths = torch.tensor([20, 100, 40, 30, 32, 0], **i32)
    held = torch.tensor([2, 7, 3, 2, 2, 0], **i32)
    finished = torch.tensor([0, 1, 0, 1, 0, 1], **i32)
    new_tokens = torch.tensor([T, T, T, 300, T, T], **i32)  # (300: more than its row of the table)
    table = torch.arange(B * 8, **i32).view(B, 8)
    free_pages = torch.full((200,), -1, **i32)
    n_free = torch.tensor([0], **i32)
    kept = torch.tensor([2, 1, 3, 0, 3, 2], **i32)
    found = torch.arange(B * T, **i32).view(B, T)
    last = -1 - torch.arange(B, **i32)
    before, was = lengths.clone(), last.clone()

    def paged_plan(lengths, new_tokens, page_table, held, free_pages, n_free, page, tokens, reset=None):
        given = (lengths, new_tokens, page_table, held, free_pages, n_free)
        r = ref.plan(*(t.numpy() for t in given), page, 700, reset.numpy())
        return [torch.from_numpy(r[n]).int()
                for n in ("cu_seqlens", "rows", "positions", "lengths")]

    ops = types.SimpleNamespace(
        mx4_cache=lambda *a: (None,) * 4, paged_plan=paged_plan,
        paged_kv_append_mx4=lambda k, v, *a, q=None, **kw: q,
        paged_attn_mx4=lambda q, *a, **kw: q, verify_drafts=lambda *a, **kw: (found, kept))
    space = dict(ops=ops, torch=torch, pages=pages, Hkv=Hkv, Hq=Hq, page=page, hd=hd, B=B, T=T, K=K,
                 lengths=lengths, new_tokens=new_tokens, page_table=table, held=held,
                 free_pages=free_pages, n_free=n_free, finished=finished, inv_freq=None, wk=None,
                 wq=None, k=None, v=None, q=torch.zeros(B * T, Hq, hd), logits=None, drafts=None,
                 u=None, draft_probs=None, last=last)
    want_plan = paged_plan(lengths, new_tokens, table, held, free_pages, n_free, page, 0, finished)[3]
    served = want_plan > torch.where(finished != 0, 0, lengths)
    assert served.tolist() == [True, True, True, False, True, True], names
    # once as it is, once with more new tokens than its row takes for the third
    for refuse in (False, True):
        lengths.copy_(before)
        last.copy_(was)
        new_tokens[2] = 300 if refuse else T
        exec(_example(), space)
        # the same buffers, which a captured step reads again
        assert space["lengths"] is lengths
        want = [20 + 3, 0 + 2, 40 if refuse else 40 + 4, 0, 32 + 4, 0 + 3]
        assert lengths.tolist() == want, dict(zip(names, zip(lengths.tolist(), want)))
        told = [0 * T + 2, 1 * T + 1, -3 if refuse else 2 * T + 3, -4, 4 * T + 3, 5 * T + 2]
        assert last.tolist() == told
