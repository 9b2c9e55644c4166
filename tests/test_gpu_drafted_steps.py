"""A serving loop with drafted tokens over the 4-bit cache: pages planned, keys and values stored,
attention of a token and its drafts, their verification, lengths cut back to what was kept.

One layer stands for the target: a token's row gives q, k and v, the attention's output times a
matrix the logits.  Each step is checked against the oracles on the step's own inputs, and at the end the
cache against the tokens that each sequence has kept."""
import pytest
import torch

from oracle import drafts as plan_ref
from oracle import mx4 as ref

pytestmark = pytest.mark.gpu

B, K, V, Hq, Hkv, hd, page, width, pages = 6, 3, 997, 8, 2, 64, 16, 12, 40
T = K + 1


def _ops():
    from hybrid_llm_amd import ops
    return ops


class Loop:
    """A server's state: the cache, its pages, each sequence's length and last token."""

    def __init__(self, seed=0):
        g = torch.Generator().manual_seed(seed)
        i32 = dict(dtype=torch.int32, device="cuda")
        self.rows = torch.randn(V, (Hq + 2 * Hkv) * hd, generator=g).to(torch.bfloat16).cuda()
        self.out = (torch.randn(Hq * hd, V, generator=g) / 6).cuda()
        self.norm = (1 + 0.1 * torch.randn(hd, generator=g)).cuda()
        self.inv_freq = (10000.0 ** (-torch.arange(0, hd, 2) / hd)).cuda()
        self.cache = _ops().mx4_cache(pages, Hkv, page, hd)
        self.table = torch.full((B, width), -1, **i32)
        self.held, self.lengths = torch.zeros(B, **i32), torch.zeros(B, **i32)
        self.free, self.n_free = torch.arange(pages, **i32), torch.tensor([pages], **i32)
        self.last = torch.randint(0, V, (B,), generator=g).int().cuda()
        self.new, self.reset = torch.full((B,), T, **i32), torch.zeros(B, **i32)
        self.u = torch.zeros(B, T, device="cuda")
        self.drafts = torch.zeros(B, K, **i32)
        self.probs = torch.zeros(B, K, V, device="cuda")

    def tensors(self):
        return [t for v in vars(self).values() for t in (v if isinstance(v, tuple) else (v,))]

    def draw(self, g):
        """The next step's drafts, their distributions, the uniforms: from a smaller model."""
        q = torch.softmax(torch.randn(B, K, V, generator=g) * 3, -1)
        self.probs.copy_(q)
        self.drafts.copy_(torch.multinomial(q.view(-1, V), 1, generator=g).view(B, K))
        self.u.copy_(torch.rand(B, T, generator=g) * 0.999)

    def qkv(self, tokens):
        row = self.rows[tokens.long()]
        return [t.view(-1, n, hd) for t, n in
                zip(row.split([Hq * hd, Hkv * hd, Hkv * hd], 1), (Hq, Hkv, Hkv))]

    def step(self):
        """One step of every sequence; what the checks look at."""
        ops = _ops()
        before = self.lengths * (self.reset == 0)
        _, rows, pos, lengths = ops.paged_plan(self.lengths, self.new, self.table, self.held,
                                               self.free, self.n_free, page, B * T,
                                               reset=self.reset)
        tokens = torch.cat((self.last[:, None], self.drafts), 1)
        q, k, v = self.qkv(tokens.flatten())
        q = ops.paged_kv_append_mx4(k, v, *self.cache, self.table, pos, rows=rows,
                                    inv_freq=self.inv_freq, k_norm=self.norm, q=q,
                                    q_norm=self.norm).view(B, T, Hq, hd)
        o = ops.paged_attn_mx4(q, *self.cache, self.table, lengths)
        logits = o.flatten(0, 1).flatten(1).float() @ self.out
        logits = logits.view(B, T, V)
        found, kept = ops.verify_drafts(logits, self.drafts, self.u, draft_probs=self.probs)
        served = lengths > before  # a sequence without pages waits
        self.lengths.copy_(torch.where(served, before + kept + 1, before))
        nxt = found.gather(1, kept[:, None].long())[:, 0]
        self.last.copy_(torch.where(served, nxt, self.last))
        return dict(tokens=tokens, q=q, o=o, logits=logits, found=found, kept=kept,
                    served=served, planned=lengths, rows=rows, pos=pos, before=before)


def test_steps_against_the_oracles():
    s, g = Loop(), torch.Generator().manual_seed(1)
    texts = [[] for _ in range(B)]  # the tokens whose keys each sequence's cache holds
    kept_any = 0
    for step in range(12):
        s.draw(g)
        s.reset.zero_()
        if step in (5, 9):  # a chat ends, another takes its row
            s.reset[step % B] = 1
            texts[step % B] = []
        names = ("lengths", "new", "table", "held", "free", "n_free")
        state = [getattr(s, n).cpu().numpy() for n in names]
        want = plan_ref.plan(*state, page, B * T, s.reset.cpu().numpy())
        r = s.step()
        for n, t in (("rows", r["rows"]), ("positions", r["pos"]), ("lengths", r["planned"]),
                     ("page_table", s.table), ("held", s.held), ("n_free", s.n_free)):
            assert (t.cpu().numpy() == want[n]).all(), (step, n)
        # attention over what the cache holds now
        kc, vc, ks, vs = (t.cpu() for t in s.cache)
        k, v = ref.values(*ref.unpack(kc, ks)), ref.values(*ref.unpack(vc, vs))
        out, spread = ref.attend(r["q"].cpu(), k, v, s.table.cpu(), r["planned"].cpu())
        # |q| and |k| are norms of 64 dims, sum |q_d k_d| / 8 <= 2^4: scores off by less than
        # 2^-11, weights by 2^-10 and 2^-16 of the spread; the store by 2^-8 of the value
        ok = r["served"].cpu()
        tol = 2.0 ** -8 * out.abs() + 2.0 ** -9 * spread + 1e-30
        assert bool(((r["o"].cpu().double() - out).abs() <= tol)[ok].all())
        # the verdicts on the step's own logits; no decision within 2^-28 of its border
        found, kept, margin = plan_ref.verify(r["logits"].cpu(), s.drafts.cpu(), s.u.cpu(), 1.0,
                                              s.probs.cpu())
        sure = margin > 2.0 ** -28
        assert bool(sure.all())
        assert torch.equal(r["found"].cpu(), found) and torch.equal(r["kept"].cpu(), kept)
        for b in range(B):
            if ok[b]:
                texts[b] += r["tokens"][b, :int(kept[b]) + 1].tolist()
        kept_any += int(kept.sum())
        assert s.lengths.tolist() == [len(t) for t in texts]
    assert kept_any > 0
    # the cache: as if each sequence's kept tokens had been stored at once
    for b, text in enumerate(texts):
        n = len(text)
        pos = torch.arange(n, dtype=torch.int32).cuda()
        fresh = _ops().mx4_cache(width, Hkv, page, hd)
        table = torch.arange(width, dtype=torch.int32).view(1, -1).cuda()
        _, k, v = s.qkv(torch.tensor(text).cuda())
        zero = torch.zeros(n, dtype=torch.int32).cuda()
        _ops().paged_kv_append_mx4(k, v, *fresh, table, pos, rows=zero, inv_freq=s.inv_freq,
                                   k_norm=s.norm)
        want = _ops().paged_kv_read_mx4(*fresh, table, pos, rows=zero)
        got = _ops().paged_kv_read_mx4(*s.cache, s.table[b:b + 1].contiguous(), pos, rows=zero)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_a_captured_step_replays():
    """The same steps eagerly and as one captured graph, with eager work between the replays."""
    one, two = Loop(3), Loop(3)
    warm = Loop(4)
    warm.draw(torch.Generator().manual_seed(0))
    warm.step()
    for loop in (one, two):
        loop.draw(torch.Generator().manual_seed(9))
    keep = [t.clone() for t in two.tensors()]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = two.step()
    for t, k in zip(two.tensors(), keep):
        t.copy_(k)
    for step in range(5):
        for loop in (one, two):
            loop.draw(torch.Generator().manual_seed(20 + step))
            loop.reset.zero_()
            loop.reset[step] = step == 3
        want = one.step()
        graph.replay()
        torch.cuda.synchronize()
        for n in want:
            assert torch.equal(got[n], want[n]), (step, n)
        for a, b in zip(one.tensors(), two.tensors()):
            same = [t.view(torch.uint8) if t.element_size() == 1 else t for t in (a, b)]
            assert torch.equal(*same), step
