"""A serving loop with too few pages and drafts of different numbers: sequences wait for pages that a
finished one gives back, and each step's new tokens are packed by their own number.

A sequence with n new tokens has them in the last n of the attention's T places, which stand at the end
of its text, and in the first n rows of the verification, which counts from the front.  Each step is
checked against the oracles on the step's own inputs, for the sequences that it served."""
import pytest
import torch

from oracle import drafts as plan_ref
from oracle import mx4 as ref

pytestmark = pytest.mark.gpu

B, K, V, Hq, Hkv, hd, page, width, pages = 6, 3, 500, 8, 2, 64, 16, 6, 9
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
        self.inv_freq = (10000.0 ** (-torch.arange(0, hd, 2) / hd)).cuda()
        self.cache = _ops().mx4_cache(pages, Hkv, page, hd)
        self.table = torch.full((B, width), -1, **i32)
        self.held, self.lengths = torch.zeros(B, **i32), torch.zeros(B, **i32)
        self.free, self.n_free = torch.arange(pages, **i32), torch.tensor([pages], **i32)
        self.last = torch.randint(0, V, (B,), generator=g).int().cuda()
        self.counts, self.reset = torch.zeros(B, **i32), torch.zeros(B, **i32)
        self.u = torch.zeros(B, T, device="cuda")
        self.drafts = torch.zeros(B, K, **i32)
        self.probs = torch.zeros(B, K, V, device="cuda")

    def tensors(self):
        return [t for v in vars(self).values() for t in (v if isinstance(v, tuple) else (v,))]

    def draw(self, g):
        """The next step's drafts, 0 to K a sequence, and the uniforms."""
        q = torch.softmax(torch.randn(B, K, V, generator=g) * 3, -1)
        self.probs.copy_(q)
        self.drafts.copy_(torch.multinomial(q.view(-1, V), 1, generator=g).view(B, K))
        self.counts.copy_(torch.randint(0, K + 1, (B,), generator=g))
        self.u.copy_(torch.rand(B, T, generator=g) * 0.999)

    def step(self):
        ops = _ops()
        new = self.counts + 1
        cu, rows, pos, planned = ops.paged_plan(self.lengths, new, self.table, self.held, self.free,
                                                self.n_free, page, B * T, reset=self.reset)
        at = torch.arange(T, device="cuda")
        tokens = torch.cat((self.last[:, None], self.drafts), 1)
        b = rows.clamp(min=0).long()
        nth = torch.arange(B * T, device="cuda") - cu[b]
        flat = tokens[b, nth.clamp(0, T - 1).long()]  # (behind the last token: any)
        row = self.rows[flat.long()]
        q, k, v = (t.view(-1, n, hd) for t, n in
                   zip(row.split([Hq * hd, Hkv * hd, Hkv * hd], 1), (Hq, Hkv, Hkv)))
        q = ops.paged_kv_append_mx4(k, v, *self.cache, self.table, pos, rows=rows,
                                    inv_freq=self.inv_freq, q=q)
        late = (cu[:-1, None] + at - (T - new[:, None])).clamp(0, B * T - 1).long()
        q = q[late]                                  # [B, T, Hq, hd], aligned to the text's end
        o = ops.paged_attn_mx4(q, *self.cache, self.table, planned)
        logits = o.flatten(0, 1).flatten(1).float() @ self.out
        early = (at + T - new[:, None]).clamp(max=T - 1).long()
        logits = logits.view(B, T, V).gather(1, early[..., None].expand(B, T, V)).contiguous()
        found, kept = ops.verify_drafts(logits, self.drafts, self.u, draft_probs=self.probs,
                                        counts=self.counts)
        start = torch.where(self.reset != 0, 0, self.lengths)
        served = planned > start
        self.lengths.copy_(torch.where(served, start + kept + 1, start))
        nxt = found.gather(1, kept[:, None].long())[:, 0]
        self.last.copy_(torch.where(served, nxt, self.last))
        return dict(tokens=tokens, q=q, o=o, logits=logits, found=found, kept=kept, served=served,
                    planned=planned, rows=rows, pos=pos)


def _resets(step, lengths, waiting):
    """The longest sequence ends in a step after which another waits, every third time."""
    over = torch.zeros(B, dtype=torch.int32)
    if waiting and step % 3 == 2:
        over[int(torch.tensor(lengths).argmax())] = 1
    return over


def test_waiting_sequences_are_served_later():
    s, g = Loop(), torch.Generator().manual_seed(1)
    texts, waiting = [[] for _ in range(B)], set()
    refused = resumed = kept_any = 0
    for step in range(60):
        s.draw(g)
        s.reset.copy_(_resets(step, s.lengths.tolist(), waiting))
        for b in s.reset.nonzero().flatten().tolist():
            texts[b] = []
        new, last = s.counts + 1, s.last.clone()
        state = [t.cpu().numpy() for t in (s.lengths, new, s.table, s.held, s.free, s.n_free)]
        want = plan_ref.plan(*state, page, B * T, s.reset.cpu().numpy())
        r = s.step()
        for n, t in (("rows", r["rows"]), ("positions", r["pos"]), ("lengths", r["planned"]),
                     ("page_table", s.table), ("held", s.held), ("n_free", s.n_free)):
            assert (t.cpu().numpy() == want[n]).all(), (step, n)
        ok, new = r["served"].cpu(), new.cpu()
        # the attention's places that hold a token, over what the cache holds now
        kc, vc, ks, vs = (t.cpu() for t in s.cache)
        k, v = ref.values(*ref.unpack(kc, ks)), ref.values(*ref.unpack(vc, vs))
        out, spread = ref.attend(r["q"].cpu(), k, v, s.table.cpu(), r["planned"].cpu())
        # sum |q_d k_d| / 8 <= 2^5 for these rows (unnormed, 64 dims of about 1): scores off by less
        # than 2^-24 x 68 x 2^5 < 2^-12, weights by 2^-11 and 2^-16 of the spread; the store 2^-8
        tol = 2.0 ** -8 * out.abs() + 2.0 ** -9 * spread + 1e-30
        there = ok[:, None] & (torch.arange(T) >= T - new[:, None])
        assert bool(((r["o"].cpu().double() - out).abs() <= tol)[there].all())
        found, kept, margin = plan_ref.verify(r["logits"].cpu()[ok], s.drafts.cpu()[ok], s.u.cpu()[ok],
                                              1.0, s.probs.cpu()[ok], s.counts.cpu()[ok])
        assert bool((margin > 2.0 ** -28).all())
        assert torch.equal(r["found"].cpu()[ok], found) and torch.equal(r["kept"].cpu()[ok], kept)
        kept_any += int(kept.sum())
        for b in range(B):
            if ok[b]:
                texts[b] += r["tokens"][b, :int(r["kept"][b]) + 1].tolist()
                resumed += b in waiting
                waiting.discard(b)
            else:
                refused += 1
                waiting.add(b)
                assert int(s.last[b]) == int(last[b])
        assert s.lengths.tolist() == [len(t) for t in texts]
    assert refused > 20 and resumed > 3 and kept_any > 10, (refused, resumed, kept_any)
    # the cache: as if each sequence's kept tokens had been stored at once
    for b, text in enumerate(texts):
        n = len(text)
        if n == 0:
            continue
        pos = torch.arange(n, dtype=torch.int32).cuda()
        fresh = _ops().mx4_cache(width, Hkv, page, hd)
        table = torch.arange(width, dtype=torch.int32).view(1, -1).cuda()
        row = s.rows[torch.tensor(text).cuda()]
        _, k, v = (t.view(-1, m, hd) for t, m in
                   zip(row.split([Hq * hd, Hkv * hd, Hkv * hd], 1), (Hq, Hkv, Hkv)))
        zero = torch.zeros(n, dtype=torch.int32).cuda()
        _ops().paged_kv_append_mx4(k, v, *fresh, table, pos, rows=zero, inv_freq=s.inv_freq)
        want = _ops().paged_kv_read_mx4(*fresh, table, pos, rows=zero)
        got = _ops().paged_kv_read_mx4(*s.cache, s.table[b:b + 1].contiguous(), pos, rows=zero)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_captured_while_sequences_wait():
    """Eager steps and replays of one captured step leave the same state, refusals among them."""
    one, two, warm = Loop(3), Loop(3), Loop(4)
    for loop in (one, two, warm):
        loop.draw(torch.Generator().manual_seed(9))
    warm.step()
    keep = [t.clone() for t in two.tensors()]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = two.step()
    for t, k in zip(two.tensors(), keep):
        t.copy_(k)
    waiting, refused = False, 0
    for step in range(30):
        over = _resets(step, one.lengths.tolist(), waiting)
        for loop in (one, two):
            loop.draw(torch.Generator().manual_seed(20 + step))
            loop.reset.copy_(over)
        want = one.step()
        graph.replay()
        torch.cuda.synchronize()
        ok = want["served"]
        for n in ("planned", "rows", "pos", "served"):
            assert torch.equal(got[n], want[n]), (step, n)
        for n in ("found", "kept"):
            assert torch.equal(got[n][ok], want[n][ok]), (step, n)
        for a, b in zip(one.tensors(), two.tensors()):
            same = [t.view(torch.uint8) if t.element_size() == 1 else t for t in (a, b)]
            assert torch.equal(*same), step
        waiting = not bool(ok.all())
        refused += int((~ok).sum())
    assert refused > 5
