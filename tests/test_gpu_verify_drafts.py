"""Drafted tokens against the model's filtered distributions: the plain rule in 64 bits (q4_cases.verify)."""
import numpy as np
import pytest

import q4_cases as q4

pytestmark = pytest.mark.gpu

CANDIDATES = 1024


@pytest.fixture(scope="module")
def be():
    from zeninfer_b200 import Backend
    return Backend()


class Check:
    def __init__(self, be, logits, tokens, uniforms, *, q=None, temperature=1.0, top_k=0, top_p=1.0, gap=0):
        """q: [drafts, vocab] probabilities, at most CANDIDATES of a row not zero, or None."""
        import torch
        from zeninfer_b200.backend import DraftCheck
        self.torch, self.be = torch, be
        drafts, vocab = len(tokens), logits.shape[1]
        dev = lambda a: torch.from_numpy(np.ascontiguousarray(a)).cuda()   # noqa: E731
        t = self.t = dict(logits=dev(np.concatenate([logits, np.full((drafts + 1, gap), 1e30, np.float32)], 1)), tokens=dev(np.array(list(tokens) + [0], np.int64)), uniforms=dev(np.array(uniforms, np.float64)),
                          out=torch.full((drafts + 1,), 77, dtype=torch.int64, device="cuda"), accepted=torch.full((1,), 77, dtype=torch.int32, device="cuda"),
                          probs=torch.full((max(drafts, 1),), 77.0, dtype=torch.float64, device="cuda"))
        if q is not None:
            ids, probs, count = np.full((drafts, CANDIDATES), -1, np.int32), np.full((drafts, CANDIDATES), np.nan), np.zeros(drafts, np.int32)
            for i, row in enumerate(q):
                at = np.flatnonzero(row)
                ids[i, :at.size], probs[i, :at.size], count[i] = at, row[at], at.size
            t.update(q_ids=dev(ids), q_probs=dev(probs), q_count=dev(count))
        p = lambda n: t[n].data_ptr() if n in t else None   # noqa: E731
        self.c = DraftCheck(logits=p("logits"), logits_ld=vocab + gap, vocab=vocab, drafts=drafts, tokens=p("tokens"), q_ids=p("q_ids"), q_probs=p("q_probs"), q_count=p("q_count"),
                            uniforms=p("uniforms"), temperature=temperature, top_k=top_k, top_p=top_p, out=p("out"), accepted=p("accepted"), probs=p("probs"))
        self.room = torch.full((be.verify_drafts_workspace_bytes(self.c),), 0xCD, dtype=torch.uint8, device="cuda")
        self.c.workspace, self.c.workspace_bytes = self.room.data_ptr(), self.room.numel()
        torch.cuda.synchronize()

    def run(self):
        st = self.torch.cuda.Stream()
        self.be.dev_verify_drafts(self.c, st.cuda_stream)
        self.be.dev_check(st.cuda_stream)
        return self.t["out"].cpu().numpy(), int(self.t["accepted"][0]), self.t["probs"].cpu().numpy()[:self.c.drafts]


def agree(be, logits, tokens, uniforms, q=None, **how):
    out, accepted, probs = Check(be, logits, tokens, uniforms, q=q, **how).run()
    args = dict(temperature=1.0, top_k=0, top_p=1.0, **{})
    args.update({n: v for n, v in how.items() if n in args})
    r_out, r_accepted, r_probs = q4.verify(logits, list(tokens), q, uniforms, **args)
    # both sides add up to 2^17 terms of 53 bits: 2^-40 covers their order, and exp's last bits
    assert np.abs(probs - r_probs).max(initial=0) <= 2.0 ** -40
    assert accepted == r_accepted and np.array_equal(out, r_out)
    return accepted


def model_rows(rng, drafts, vocab):
    logits = rng.standard_normal((drafts + 1, vocab)).astype(np.float32) * np.float32(2)
    for row in logits:
        row[rng.integers(0, vocab, 12)] += rng.uniform(2, 9, 12).astype(np.float32)
    return logits


def draft_rows(rng, logits, drafts, kept, temperature):
    q = np.zeros((drafts, logits.shape[1]))
    for i in range(drafts):
        row = logits[i] + rng.standard_normal(logits.shape[1]).astype(np.float32) * np.float32(0.5)
        q[i] = q4.distribution(row, temperature or 1.0, min(kept, logits.shape[1]), 1.0)
    return q


@pytest.mark.parametrize("drafts,vocab", [(0, 50), (1, 1), (1, 2), (1, 33), (2, 1000), (4, 8191), (8, 32000), (3, 128256), (33, 777), (64, 501), (2, 200003), (1, 262144)])
@pytest.mark.parametrize("filters", [(1.0, 0, 1.0), (0.0, 0, 1.0), (0.7, 40, 1.0), (1.3, 0, 0.9), (0.8, 50, 0.8), (1.0, 5000, 0.99), (1.0, 1, 0.5), (5.0, 0, 1e-6)], ids=str)
@pytest.mark.parametrize("listed", [False, True])
def test_against_the_plain_rule(be, drafts, vocab, filters, listed):
    temperature, top_k, top_p = filters
    rng = np.random.default_rng(drafts * 1000 + vocab)
    logits = model_rows(rng, drafts, vocab)
    q = draft_rows(rng, logits, drafts, 200, temperature) if listed else None
    for trial in range(2):
        if listed:
            tokens = [int(rng.choice(vocab, p=row)) for row in q]
        else:
            tokens = [int(row.argmax()) if rng.random() < 0.85 else int(rng.integers(vocab)) for row in logits[:drafts]]
        agree(be, logits, tokens, rng.random(drafts + 1), q, temperature=temperature, top_k=top_k, top_p=top_p, gap=3 * trial)


def test_every_number_of_accepted_drafts_happens(be):
    rng = np.random.default_rng(0)
    logits = model_rows(rng, 4, 500)
    seen = {agree(be, logits, [int(r.argmax()) for r in logits[:4]], rng.random(5)) for _ in range(40)}
    assert seen == {0, 1, 2, 3, 4}


def test_ties_are_cut_in_order_of_id(be):
    rng = np.random.default_rng(1)
    logits = rng.choice(np.array([0.0, -0.0, 1.0, 2.0], np.float32), (4, 3000))
    for top_k in (1, 7, 800, 1600, 2999, 3000, 4000):
        for top_p in (1.0, 0.5, 0.05):
            agree(be, logits, [int(rng.integers(3000)) for _ in range(3)], rng.random(4), top_k=top_k, top_p=top_p)
    flat = np.zeros((2, 20000), np.float32)
    for top_p in (1.0, 0.3):
        for u in (0.0, 0.1, 0.999999):
            agree(be, flat, [5], [0.9, u], top_p=top_p)


def test_logits_that_are_not_finite_never_win(be):
    rng = np.random.default_rng(2)
    logits = model_rows(rng, 3, 2000)
    logits[:, ::7] = np.nan
    logits[:, 1::7] = np.inf
    logits[:, 2::7] = -np.inf
    agree(be, logits, [7, 8, 3], rng.random(4))                       # a NaN, an infinity: not accepted
    agree(be, logits, [int(np.nanargmax(np.where(np.isfinite(r), r, -1e9))) for r in logits[:3]], [0.0, 0.0, 0.0, 0.5], top_k=20, top_p=0.9)
    empty = logits.copy()
    empty[1] = np.nan
    out, accepted, probs = Check(be, empty, [int(np.nanargmax(np.where(np.isfinite(empty[0]), empty[0], -1e9))), 4, 4], [0.0, 0.0, 0.0, 0.5]).run()
    assert accepted == 1 and list(out[1:]) == [-1, -1, -1] and probs[1] == 0.0
    extreme = np.zeros((2, 64), np.float32)
    extreme[0, 9], extreme[0, 10] = 3e38, -3e38
    agree(be, extreme, [9], [0.99, 0.5])
    agree(be, extreme, [10], [0.0, 0.5], temperature=1e-30)


def test_what_is_left_when_the_draft_was_certain_or_equal(be):
    rng = np.random.default_rng(3)
    logits = model_rows(rng, 1, 300)
    p = q4.distribution(logits[0], 1.0, 0, 1.0)
    # q equal to p: never rejected, and a list that takes more than there is leaves p itself to draw from
    agree(be, logits, [int(p.argmax())], [0.999999, 0.3], p[None])
    agree(be, logits, [int(p.argmin())], [0.999999, 0.3], np.minimum(1.0, p[None] * 4))
    one = np.full((2, 300), -50.0, np.float32)
    one[0, 17] = 1000.0
    agree(be, one, [17], [0.5, 0.5])                 # accepted: it has all of p
    agree(be, one, [18], [0.0, 0.0])                 # 0 < 0 is false: rejected, and the draw is the one token there is
    agree(be, logits, [3], [0.0, 0.0])               # u = 0 reaches the first id with a share


def test_a_draft_outside_the_vocabulary(be):
    from zeninfer_b200 import BackendError
    rng = np.random.default_rng(4)
    logits = model_rows(rng, 2, 100)
    for bad in (-1, 100, 2 ** 40):
        c = Check(be, logits, [int(logits[0].argmax()), bad], [0.0, 0.0, 0.4])
        with pytest.raises(BackendError, match="token"):
            c.run()
        out, accepted, _ = q4.verify(logits, [int(logits[0].argmax()), bad], None, [0.0, 0.0, 0.4], 1.0, 0, 1.0)
        assert int(c.t["accepted"][0]) == accepted == 1 and np.array_equal(c.t["out"].cpu().numpy(), out)


def test_lists_with_entries_outside_the_vocabulary_and_counts_outside_the_list(be):
    rng = np.random.default_rng(5)
    logits = model_rows(rng, 1, 100)
    q = draft_rows(rng, logits, 1, 50, 1.0)
    c = Check(be, logits, [int(q[0].argmax())], [0.2, 0.7], q=q)
    first = c.run()
    c.t["q_ids"][0, 50:52] = c.torch.tensor([-5, 100], dtype=c.torch.int32)
    c.t["q_probs"][0, 50:52] = 0.5
    c.t["q_count"][0] = 52
    c.torch.cuda.synchronize()
    assert all(np.array_equal(a, b) for a, b in zip(first, c.run()))
    c.t["q_ids"][0, 50:] = -1
    c.t["q_count"][0] = 5000
    c.torch.cuda.synchronize()
    assert all(np.array_equal(a, b) for a, b in zip(first, c.run()))
    c.t["q_count"][0] = -3                          # none: nothing is taken off, and a draft of no probability is accepted where p has any
    c.torch.cuda.synchronize()
    assert c.run()[1] == 1


def test_captured_and_at_once(be):
    import torch
    rng = np.random.default_rng(6)
    one, two = (Check(be, model_rows(rng, 4, 32000), [int(t) for t in rng.integers(0, 32000, 4)], rng.random(5), top_p=0.9) for _ in range(2))
    eager = [c.run() for c in (one, two)]
    streams, graphs = [torch.cuda.Stream() for _ in range(2)], []
    for c, s in zip((one, two), streams):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            be.dev_verify_drafts(c.c, s.cuda_stream)
        graphs.append((g, s))
    for c in (one, two):
        c.t["out"].fill_(-7)
        c.room.fill_(0xFF)
    torch.cuda.synchronize()
    for _ in range(10):
        for g, s in graphs:
            with torch.cuda.stream(s):
                g.replay()
    torch.cuda.synchronize()
    for c, (out, accepted, probs) in zip((one, two), eager):
        assert np.array_equal(c.t["out"].cpu().numpy(), out) and int(c.t["accepted"][0]) == accepted and np.array_equal(c.t["probs"].cpu().numpy(), probs)


def test_the_samplers_kept_list_is_a_drafts_distribution(be):
    """A draft drawn by dev_sample, and its kept list handed over as it is."""
    import torch
    rng = np.random.default_rng(7)
    logits = model_rows(rng, 1, 32000)
    drafted = logits[0] + rng.standard_normal(32000).astype(np.float32) * np.float32(0.3)
    d = torch.from_numpy(drafted).cuda()
    pick, st = torch.zeros(1, dtype=torch.int64, device="cuda"), torch.cuda.Stream()
    c = Check(be, logits, [0], [0.4, 0.6], q=np.eye(1, 32000), temperature=0.9, top_k=100, top_p=0.95)
    torch.cuda.synchronize()
    be.dev_sample(d.data_ptr(), 32000, 0.9, 100, 0.95, 0.33, c.t["tokens"].data_ptr(), st.cuda_stream, d_kept_ids=c.t["q_ids"].data_ptr(), d_kept_probs=c.t["q_probs"].data_ptr(),
                  d_kept_count=c.t["q_count"].data_ptr())
    be.dev_verify_drafts(c.c, st.cuda_stream)
    be.dev_check(st.cuda_stream)
    token = int(c.t["tokens"][0])
    q = q4.distribution(drafted, 0.9, 100, 0.95)[None]
    out, accepted, probs = q4.verify(logits, [token], q, [0.4, 0.6], 0.9, 100, 0.95)
    assert int(c.t["accepted"][0]) == accepted and np.array_equal(c.t["out"].cpu().numpy(), out) and abs(float(c.t["probs"][0]) - probs[0]) <= 2.0 ** -40


def test_a_goal_between_two_roundings_of_a_sum_is_reached_in_one_place(be):
    """A row of 16 entries lies in four runs of four.  The sum up to the second run's end may be rounded once, as a multiply-add, or twice; the uniform number is chosen so that the first
    of these has not reached the goal and the second has.  Either neighbour of that place is a right answer, and what the workspace held is none."""
    from fractions import Fraction
    rng = np.random.default_rng(8)
    found = 0
    while found < 48:
        at = -rng.uniform(0.1, 3.0, 3).astype(np.float32)
        shares = [3 * np.exp(float(x)) for x in at] + [3.0]
        ahead, whole = shares[0], ((shares[0] + shares[1]) + shares[2]) + shares[3]
        twice = ahead + shares[1]
        exact = Fraction(ahead) + 3 * Fraction(float(np.exp(float(at[1]))))
        once = float(exact)                                # a Fraction is rounded to the nearest
        u = float(Fraction(twice) / Fraction(whole))
        u = u if Fraction(u) * Fraction(whole) <= Fraction(twice) else float(np.nextafter(u, 0.0))
        if not once < twice or Fraction(u) * Fraction(whole) <= Fraction(once):
            continue
        found += 1
        row = np.full((1, 16), -np.inf, np.float32)
        for r, x in enumerate([*at, np.float32(0.0)]):
            row[0, 4 * r:4 * r + 3] = x
        out, accepted, _ = Check(be, row, [], [u]).run()
        assert accepted == 0 and out[0] in (6, 8), (found, out)


def test_the_draw_is_not_limited_to_the_samplers_candidates(be):
    """Of 4000 equal logits dev_sample considers the first 1024; a checked block's draw takes any, and the same ones where top_k says so."""
    import torch
    flat, pick, st = np.zeros((1, 4000), np.float32), torch.zeros(1, dtype=torch.int64, device="cuda"), torch.cuda.Stream()
    for top_k in (0, 2000, 1024, 7):
        c = Check(be, flat, [], [0.9999], top_k=top_k)
        out, _, _ = c.run()
        be.dev_sample(c.t["logits"].data_ptr(), 4000, 1.0, top_k, 1.0, 0.9999, pick.data_ptr(), st.cuda_stream)
        be.dev_check(st.cuda_stream)
        n = top_k or 4000
        assert out[0] == int(np.ceil(0.9999 * n)) - 1 and int(pick) == int(np.ceil(0.9999 * min(n, CANDIDATES))) - 1


@pytest.mark.parametrize("n,top_p,kept", [(6, 0.5, 3), (10, 0.5, 5), (12, 0.25, 3), (12, 0.75, 9), (20, 0.75, 15), (28, 0.25, 7), (1000, 0.5, 500), (1000, 0.125, 125), (3000, 0.75, 2250), (49, 0.5, 25)])
def test_equal_entries_that_reach_the_share_exactly(be, n, top_p, kept):
    """`kept` of n equal entries have top_p of the mass (the last case: reach it): the shortest run that reaches it has so many.  Alone, and with entries far below that have no mass."""
    for vocab in (n, 3 * n, 9000):
        row = np.full((2, vocab), -1e4, np.float32)
        at = np.sort(np.random.default_rng(n).choice(vocab, n, replace=False))
        row[:, at] = 1.25
        for draft, u in ((kept - 1, 0.5), (kept, 0.5), (0, 0.999999)):      # the last that stays, the first that goes
            out, accepted, probs = Check(be, row, [int(at[draft])], [0.0, u], top_p=top_p).run()
            assert accepted == (draft < kept) and abs(probs[0] - (1.0 / kept if draft < kept else 0.0)) <= 2.0 ** -50
            assert out[accepted] == at[int(np.ceil(u * kept)) - 1]
