"""Verification of drafted tokens against the 64-bit oracle: whole numbers, equal.

The kernels decide in 64 bits too, by sums in another order: off by 2^-52 * V of a row's whole
at most, 2^-30 at V = 2^20.  A decision nearer to its border than 2^-28 would be left out of the
comparison; the oracle's margin says that none of these inputs has one."""
import math

import pytest
import torch

from oracle import drafts as ref

pytestmark = pytest.mark.gpu
NEAR = 2.0 ** -28


def _ops():
    from hybrid_llm_amd import ops
    return ops


def _case(B, K, V, seed, temperature=0.8, probs=True, std=2.5, counts=True):
    g = torch.Generator().manual_seed(seed)
    logits = torch.randn(B, K + 1, V, generator=g) * std
    near = logits[:, :K] + torch.randn(B, K, V, generator=g)
    q = torch.softmax(near / max(temperature, 0.5), -1)
    ids = torch.multinomial(q.view(-1, V), 1, generator=g).view(B, K).int()
    n = torch.randint(0, K + 1, (B,), generator=g).int() if counts else None
    u = torch.rand(B, K + 1, generator=g)
    return logits, ids, u, temperature, (q if probs else None), n


def _run(case):
    logits, ids, u, temperature, q, n = case
    dev = [None if t is None else t.cuda() for t in (logits, ids, u, q, n)]
    tokens, accepted = _ops().verify_drafts(dev[0], dev[1], dev[2], temperature=temperature,
                                            draft_probs=dev[3], counts=dev[4])
    return tokens.cpu(), accepted.cpu()


def _same(case):
    want, kept, margin = ref.verify(*case)
    assert float(margin.min()) > NEAR
    tokens, accepted = _run(case)
    assert torch.equal(accepted, kept), (accepted, kept)
    assert torch.equal(tokens, want), (tokens, want)
    return tokens, accepted


@pytest.mark.parametrize("B,K,V,seed,kw", [
    (1, 1, 1, 0, {}), (2, 3, 2, 1, {}), (5, 4, 1000, 2, {}), (64, 3, 4099, 3, {}),
    (7, 8, 32000, 4, {}), (3, 2, 128256, 5, {}), (16, 5, 4096, 6, {"temperature": 0.0}),
    (9, 63, 257, 7, {"std": 6.0}), (64, 4, 8191, 8, {"probs": False}),
    (33, 6, 12289, 9, {"temperature": 1.5, "counts": False}),
    (40, 4, 5000, 10, {"temperature": 0.05}), (8, 3, 32000, 11, {"temperature": 0.0, "probs": False}),
    (30, 2, 600, 12, {"std": 0.0}), (2, 3, 300001, 13, {}),
])
def test_verify(B, K, V, seed, kw):
    tokens, accepted = _same(_case(B, K, V, seed, **kw))
    assert tokens.shape == (B, K + 1) and accepted.shape == (B,)


def test_all_kept_and_none_kept():
    B, K, V = 6, 4, 9000
    logits, ids, u, t, q, _ = _case(B, K, V, 0, counts=False)
    same = torch.softmax(logits[:, :K].double() / t, -1).float()
    # the target's own distribution, a touch lower so that rounding rejects none
    tokens, accepted = _same((logits, ids, u, t, same * (1 - 2.0 ** -20), None))
    assert (accepted == K).all()
    ids = logits[:, :K].argmin(-1).int()
    tokens, accepted = _same((logits, ids, u.clamp_min(0.5), t, None, None))
    assert (accepted == 0).all() and (tokens[:, 1:] == -1).all() and (tokens[:, 0] >= 0).all()


def test_uniforms_at_their_ends():
    """u 0 takes the first id with weight; one at 1 or past it, or NaN, the last."""
    logits = torch.full((4, 2, 5000), -math.inf)
    logits[..., 17], logits[..., 4100], logits[..., 4999] = 1.0, 2.0, 0.5
    ids = torch.full((4, 1), 3, dtype=torch.int32)
    u = torch.tensor([[0.5, 0.0], [0.5, 1.0], [0.5, 7.0], [0.5, math.nan]])
    tokens, accepted = _run((logits, ids, u, 1.0, None, None))
    assert accepted.tolist() == [0] * 4
    assert tokens[:, 0].tolist() == [17, 4999, 4999, 4999]


def test_drafts_outside_the_vocabulary_and_counts_out_of_range():
    logits, ids, u, t, q, _ = _case(6, 3, 700, 5)
    ids[0, 0], ids[1, 0], ids[2, 1] = -1, 700, 2 ** 31 - 1
    n = torch.tensor([3, 3, 3, -4, 9, 2], dtype=torch.int32)
    for probs in (q, None):
        tokens, accepted = _same((logits, ids, u, t, probs, n))
        assert accepted[0] == 0 and accepted[1] == 0 and accepted[2] <= 1 and accepted[3] == 0
        assert (tokens.gather(1, accepted[:, None].long()) >= 0).all()


@pytest.mark.parametrize("what", ["nan", "inf", "all -inf", "one"])
def test_rows_without_a_finite_largest_logit(what):
    V = 4500
    logits = torch.randn(4, 3, V, generator=torch.Generator().manual_seed(0))
    sure = {"nan": 4400, "inf": 77, "all -inf": 0, "one": 4499}[what]
    if what == "nan":
        logits[:, :, 4400] = math.nan
        logits[:, :, 10] = math.inf
    elif what == "inf":
        logits[:, :, [77, 78, 4444]] = math.inf
    else:
        logits[:] = -math.inf
        if what == "one":
            logits[..., sure] = 3.0
    ids = torch.tensor([[sure, sure], [sure, 5], [5, sure], [sure, -1]], dtype=torch.int32)
    u = torch.rand(4, 3, generator=torch.Generator().manual_seed(1)) * 0.9 + 0.05
    for t in (1.0, 0.0):
        tokens, accepted = _run((logits, ids, u, t, None, None))
        assert accepted.tolist() == [2, 1, 0, 1]
        assert tokens.tolist() == [[sure] * 3, [sure, sure, -1], [sure, -1, -1], [sure, sure, -1]]


def test_ties_go_to_the_lowest_id():
    logits = torch.zeros(2, 2, 10000)
    logits[:, :, [9000, 500, 8191]] = 4.0
    ids = torch.tensor([[500], [8191]], dtype=torch.int32)
    tokens, accepted = _run((logits, ids, torch.rand(2, 2), 0.0, None, None))
    assert accepted.tolist() == [1, 0] and tokens.tolist() == [[500, 500], [500, -1]]


def test_draft_distributions_that_leave_nothing_or_are_wrong():
    """q above p everywhere: a draw from p; NaN in q rejects the draft and takes nothing off."""
    logits, ids, u, t, q, _ = _case(3, 2, 5000, 8, counts=False)
    u[:, :2] = 0.999
    _, accepted = _same((logits, ids, u, t, torch.full_like(q, 2.0), None))
    assert (accepted == 0).all()
    want, kept, _ = ref.verify(logits, torch.full_like(ids, -1), u, t, torch.zeros_like(q), None)
    tokens, accepted = _run((logits, ids, u, t, torch.full_like(q, math.nan), None))
    assert torch.equal(tokens, want) and torch.equal(accepted, kept)


def test_the_tokens_are_distributed_as_the_target():
    """Over 40000 independent draws, the first token's frequencies are the target's softmax:
    each within 5 standard deviations of a binomial (one in 1.7 million each, 12 of them)."""
    N, V = 40000, 12
    g = torch.Generator().manual_seed(0)
    row, near = torch.randn(V, generator=g), torch.randn(V, generator=g)
    q = torch.softmax(near, -1)
    ids = torch.multinomial(q.expand(N, V), 1, generator=g).int()
    u = torch.rand(N, 2, generator=g)
    tokens, _ = _run((row.expand(N, 2, V).contiguous(), ids, u, 1.0,
                      q.expand(N, 1, V).contiguous(), None))
    p = torch.softmax(row.double(), -1)
    freq = torch.bincount(tokens[:, 0].long(), minlength=V).double() / N
    assert bool(((freq - p).abs() <= 5 * (p * (1 - p) / N).sqrt()).all())


def test_captured_and_replayed():
    ops = _ops()
    cases = [_case(4, 3, 9000, s) for s in range(3)]
    dev = [None if t is None or isinstance(t, float) else t.cuda() for t in cases[0]]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = ops.verify_drafts(dev[0], dev[1], dev[2], temperature=0.8, draft_probs=dev[4],
                                counts=dev[5])
    for c in cases + cases[:1]:
        for d, t in zip(dev, c):
            if d is not None:
                d.copy_(t)
        graph.replay()
        torch.cuda.synchronize()
        want, kept, margin = ref.verify(*c)
        assert float(margin.min()) > NEAR
        assert torch.equal(out[0].cpu(), want) and torch.equal(out[1].cpu(), kept)


@pytest.mark.parametrize("B,K,V,seed,kw", [
    # several chunks a workgroup of the first kernel, the last of them short; 16 ids a thread
    (72, 7, 36000, 20, {}), (65, 5, 57345, 21, {"probs": False}),
    (90, 5, 45055, 22, {"temperature": 0.0, "probs": False}),
])
def test_many_rows(B, K, V, seed, kw):
    _same(_case(B, K, V, seed, **kw))


def test_many_rows_without_a_finite_largest_logit():
    """Rows of several chunks a workgroup: -inf at first, throughout, infinities and NaN late."""
    B, K, V = 66, 7, 33000
    case = list(_case(B, K, V, 30, probs=False, counts=False))
    x = case[0]
    x[0::5, :, :20000] = -math.inf
    x[1::5, 2] = -math.inf
    x[2::5, 1, [20, 32999]] = math.inf
    x[3::5, 0, 29000] = math.nan
    x[3::5, 0, 100] = math.inf
    case[1] = x[:, :K].nan_to_num(nan=9e9, posinf=8e9, neginf=-9e9).argmax(-1).int()  # often kept
    case[2] = case[2] * 0.5
    tokens, accepted = _same(tuple(case))
    assert 0 < int(accepted.float().mean() * 10) and int(accepted.min()) < K
    case[3] = 0.0
    _same(tuple(case))


@pytest.mark.parametrize("temperature", [1e-9, 1e-16, 1e-20, 1e-30, 1e-300, 5e-324])
@pytest.mark.parametrize("scale", [1.0, 1e30])
def test_temperatures_near_zero(temperature, scale):
    """Only a row's largest logits have any weight, however far their quotients reach."""
    B, K, V = 5, 3, 9001
    logits, ids, u, _, q, n = _case(B, K, V, 3, counts=False)
    logits *= scale
    logits[1, :, [7, 8888]] = 50.0 * scale  # two that are largest
    ids[1] = 7
    ids[2] = logits[2, :K].argmax(-1).int()
    u[1, :K], u[1, K] = 0.25, 0.75
    _, accepted = _same((logits, ids, u, temperature, None, None))
    assert accepted[1] == K and accepted[2] == K
    _same((logits, ids, u, temperature, q, None))


def test_on_another_stream_and_two_at_once():
    ops = _ops()
    cases = [_case(20, 4, 30000, 40), _case(70, 3, 9000, 41)]
    dev = [[None if t is None or isinstance(t, float) else t.cuda() for t in c] for c in cases]
    streams = [torch.cuda.Stream() for _ in cases]
    torch.cuda.synchronize()
    for _ in range(3):
        got = []
        for d, c, s in zip(dev, cases, streams):
            with torch.cuda.stream(s):
                got.append(ops.verify_drafts(d[0], d[1], d[2], temperature=c[3], draft_probs=d[4],
                                             counts=d[5]))
        torch.cuda.synchronize()
        for g, c in zip(got, cases):
            want, kept, margin = ref.verify(*c)
            assert float(margin.min()) > NEAR
            assert torch.equal(g[0].cpu(), want) and torch.equal(g[1].cpu(), kept)


def test_few_rows_and_many_replayed_in_one_graph():
    """Calls of every form, back to back in one graph, replayed over inputs that change: what a call
    counts on the GPU starts anew each time."""
    ops = _ops()
    sizes = [(1, 4, 32000), (4, 2, 32000), (8, 2, 32000), (1, 63, 9000), (2, 3, 60000), (70, 3, 17000)]
    sets = [[_case(*n, 50 + i + 10 * r) for i, n in enumerate(sizes)] for r in range(3)]
    dev = [[None if t is None or isinstance(t, float) else t.cuda() for t in c] for c in sets[0]]

    def calls():
        return [ops.verify_drafts(d[0], d[1], d[2], temperature=0.8, draft_probs=d[4], counts=d[5])
                for d in dev]

    calls()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = calls()
    for r in (0, 1, 2, 0, 0):
        for d, c in zip(dev, sets[r]):
            for a, b in zip(d, c):
                if a is not None:
                    a.copy_(b)
        graph.replay()
        torch.cuda.synchronize()
        eager = calls()
        for c, got, now in zip(sets[r], out, eager):
            want, kept, margin = ref.verify(*c)
            assert float(margin.min()) > NEAR
            for tokens, accepted in (got, now):
                assert torch.equal(tokens.cpu(), want) and torch.equal(accepted.cpu(), kept)
