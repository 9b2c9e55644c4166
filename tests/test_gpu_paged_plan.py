"""Pages and slots for new tokens: whole numbers, equal to the sequential oracle's."""
import numpy as np
import pytest
import torch

from oracle import drafts as ref

pytestmark = pytest.mark.gpu

NAMES = ("cu_seqlens", "rows", "positions", "lengths", "page_table", "held", "free_pages", "n_free")


def _ops():
    from hybrid_llm_amd import ops
    return ops


def _case(B, width, page, seed, free=None, top=64, most_new=40, over=0.3, capacity=None):
    """Sequences with some tokens, on disjoint pages, the others free."""
    r = np.random.RandomState(seed)
    lens = r.randint(0, width * page + 1, B) if B else np.zeros(0, int)
    held = -(-lens // page)
    new = r.randint(0, most_new + 1, B)
    ids = r.permutation(int(held.sum()) + top)
    table = np.full((B, width), -7)
    at = 0
    for b in range(B):
        table[b, :held[b]] = ids[at:at + held[b]]
        at += held[b]
    stack = np.full(len(ids) if free is None else free, -3)
    stack[:top] = ids[at:at + top]
    return dict(lengths=lens, new_tokens=new, page_table=table, held=held, free_pages=stack,
                n_free=np.array([top]), page=page,
                tokens=int(new.sum()) + 5 if capacity is None else capacity,
                reset=(r.rand(B) < over).astype(int))


def _run(c):
    i32 = {n: torch.tensor(np.asarray(v), dtype=torch.int32).cuda() for n, v in c.items()
           if n not in ("page", "tokens") and v is not None}
    got = _ops().paged_plan(i32["lengths"], i32["new_tokens"], i32["page_table"], i32["held"],
                            i32["free_pages"], i32["n_free"], c["page"], c["tokens"],
                            reset=i32.get("reset"))
    got = dict(zip(NAMES, (*got, i32["page_table"], i32["held"], i32["free_pages"], i32["n_free"])))
    return {n: t.cpu().numpy() for n, t in got.items()}


def _same(c):
    want, got = ref.plan(**c), _run(c)
    for n in NAMES:
        assert np.array_equal(got[n], want[n]), (n, got[n], want[n])
    return got


@pytest.mark.parametrize("B,width,page,seed,kw", [
    (1, 4, 16, 0, {}), (3, 8, 16, 1, {}), (64, 20, 32, 2, {}), (64, 20, 32, 3, {"top": 7}),
    (65, 6, 64, 4, {"over": 1.0}), (130, 9, 128, 5, {"over": 0.0}), (1024, 4, 256, 6, {}),
    (1025, 5, 16, 7, {"top": 900}), (4096, 3, 16, 8, {"top": 2000}), (3000, 3, 16, 9, {"most_new": 0}),
    (5, 600, 16, 10, {"most_new": 5000, "over": 0.6, "top": 1000}),
    (37, 300, 16, 11, {"most_new": 4000, "over": 0.9, "top": 600}),
    (4096, 4, 16, 12, {"most_new": 50, "top": 5000}),
    (9, 40, 16, 13, {"capacity": 60}), (9, 400, 16, 14, {"capacity": 5000, "most_new": 2000}),
    (20, 10, 16, 15, {"free": 70}),        # a stack too small for what comes back
    (20, 10, 16, 16, {"top": 0}), (4, 0, 16, 17, {"top": 3}),
    (16, 64, 16, 18, {"capacity": 0}), (2, 20000, 16, 19, {"most_new": 200000, "top": 30000}),
])
def test_plan(B, width, page, seed, kw):
    _same(_case(B, width, page, seed, **kw))


def test_no_sequences():
    got = _same(dict(lengths=[], new_tokens=[], page_table=np.zeros((0, 4), int), held=[],
                     free_pages=[3, 4], n_free=[2], page=16, tokens=3, reset=None))
    assert got["cu_seqlens"].tolist() == [0] and got["rows"].tolist() == [-1] * 3


def test_numbers_out_of_range():
    """Negative counts are 0, more held than a row has is the row, a stack is no higher than it
    is; lengths near 2^31 do not wrap."""
    c = _case(6, 5, 16, 0)
    c.update(lengths=[-5, 3, 2 ** 31 - 1, 10, 80, 70], new_tokens=[4, -2, 2 ** 31 - 1, 9, 1, 10],
             held=[-1, 1, 5, 900, 5, 5], n_free=[10 ** 6], reset=[0, 0, 0, 1, 0, 0])
    _same(c)
    c.update(n_free=[-3], new_tokens=[4, -2, 7, 2 ** 31 - 1, 2 ** 31 - 1, 10])
    _same(c)


def test_pages_stay_whole_over_many_steps():
    """200 steps of arrivals, growth, cut-backs and resets: at every step each page is held by
    one sequence or free, once."""
    r = np.random.RandomState(0)
    B, width, page, pages = 24, 12, 16, 150
    dev = dict(dtype=torch.int32, device="cuda")
    table, held = torch.full((B, width), -1, **dev), torch.zeros(B, **dev)
    free, n_free = torch.arange(pages, **dev), torch.tensor([pages], **dev)
    lengths = torch.zeros(B, **dev)
    for step in range(200):
        new = torch.tensor(r.randint(0, 20, B) * (r.rand(B) < 0.7), **dev)
        over = torch.tensor(r.rand(B) < 0.1, **dev)
        _, rows, pos, lengths = _ops().paged_plan(lengths, new, table, held, free, n_free, page, 512,
                                                  reset=over)
        t, h, n = table.cpu().numpy(), held.cpu().numpy(), int(n_free)
        owned = np.concatenate([t[b, :h[b]] for b in range(B)] + [free.cpu().numpy()[:n]])
        assert np.array_equal(np.sort(owned), np.arange(pages)), step
        ln = lengths.cpu().numpy()
        assert (ln <= h * page).all()
        kept = pos.cpu().numpy() >= 0
        assert (pos.cpu().numpy()[kept] < ln[rows.cpu().numpy()[kept]]).all()
        # drafts that were not kept: shorter, the pages stay
        lengths = torch.clamp(lengths - torch.tensor(r.randint(0, 4, B), **dev), min=0)


def test_captured_and_replayed():
    ops = _ops()
    c = _case(40, 30, 16, 3, top=500)
    t = {n: torch.tensor(np.asarray(v), dtype=torch.int32).cuda() for n, v in c.items()
         if n not in ("page", "tokens")}
    for tokens in (c["tokens"], 6000):   # one launch, and two
        c["tokens"] = tokens
        keep = {n: x.clone() for n, x in t.items()}
        args = [t[n] for n in ("lengths", "new_tokens", "page_table", "held", "free_pages", "n_free")]
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = ops.paged_plan(*args, c["page"], tokens, reset=t["reset"])
        for i in range(3):
            for n, x in keep.items():
                t[n].copy_(x)
            t["new_tokens"].add_(i)
            now = {**c, "new_tokens": t["new_tokens"].cpu().numpy()}
            graph.replay()
            torch.cuda.synchronize()
            want = ref.plan(**now)
            got = (*out, t["page_table"], t["held"], t["free_pages"], t["n_free"])
            for n, x in zip(NAMES, got):
                assert np.array_equal(x.cpu().numpy(), want[n]), (tokens, i, n)
        for n, x in keep.items():
            t[n].copy_(x)
