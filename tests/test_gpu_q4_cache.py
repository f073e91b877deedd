"""Attention over the 4-bit cache and eviction from it, against plain implementations in 64 bits (q4_cases.py)."""
import numpy as np
import pytest

import q4_cases as q4

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def be():
    from zeninfer_b200 import Backend
    return Backend()


class Setup:
    """A cache with `filled` slots of a made-up sequence and junk behind them, and `tokens` new rows."""

    def __init__(self, be, tokens, filled, heads, kv_heads, dim, *, slots=None, weights=False, pairs=None, adjacent=True, scale=0.0, q_gap=0, kv_gap=0, seed=0, spread=1.0):
        import torch
        from zeninfer_b200.backend import Q4Attention, Q4Cache
        self.torch, self.be = torch, be
        self.tokens, self.filled, self.heads, self.kv_heads, self.dim = tokens, filled, heads, kv_heads, dim
        self.slots = slots or q4.round_up(filled + tokens, 32)
        self.scale = scale or float(np.float32(1) / np.sqrt(np.float32(dim)))
        rng = np.random.default_rng(seed)
        self.adjacent, self.pairs = adjacent, dim // 2 if pairs is None else pairs
        self.rotated_from = 5
        angle = rng.uniform(0, 2 * np.pi, (self.rotated_from + tokens + 3, max(self.pairs, 1)))
        self.cos, self.sin = np.cos(angle).astype(np.float32), np.sin(angle).astype(np.float32)
        normal = lambda *shape: rng.standard_normal(shape, dtype=np.float32)   # noqa: E731
        self.q, self.k, self.v = normal(tokens, heads, dim) * np.float32(spread), normal(tokens, kv_heads, dim), normal(tokens, kv_heads, dim)
        self.old = {s: q4.quantise(normal(kv_heads, self.slots, dim)) for s in "kv"}
        dev = lambda a: torch.from_numpy(np.ascontiguousarray(a)).cuda()   # noqa: E731
        t = self.t = {}
        for s in "kv":
            d, c = self.old[s]
            d = d.copy()
            d[:, filled:] = np.nan                       # nothing of the slots behind may reach a result
            t[s + "_codes"], t[s + "_scales"] = dev(q4.pack(c)), dev(d)
        self.before = {n: x.clone() for n, x in t.items()}
        wide = lambda a, gap: np.concatenate([a.reshape(tokens, -1), np.full((tokens, gap), np.nan, np.float32)], 1)   # noqa: E731
        t["q"], t["k"], t["v"] = dev(wide(self.q, q_gap)), dev(wide(self.k, kv_gap)), dev(wide(self.v, kv_gap))
        t["cos"], t["sin"] = dev(self.cos), dev(self.sin)
        t["at"] = torch.tensor([self.rotated_from, filled], dtype=torch.int32, device="cuda")
        t["out"] = torch.full((tokens, heads * dim), 7.0, device="cuda")
        t["k_held"], t["v_held"] = torch.zeros((tokens, kv_heads * dim), device="cuda"), torch.zeros((tokens, kv_heads * dim), device="cuda")
        self.weight_in = rng.random((kv_heads, self.slots)).astype(np.float32) if weights else None
        if weights:
            t["weight_in"], t["weight_out"] = dev(self.weight_in), torch.full((kv_heads, self.slots), -3.0, device="cuda")
        p = lambda n: t[n].data_ptr() if n in t else None   # noqa: E731
        self.cache = Q4Cache.of(t["k_codes"], t["k_scales"], t["v_codes"], t["v_scales"], kv_heads=kv_heads, head_dim=dim, slots=self.slots)
        self.a = Q4Attention(cache=self.cache, heads=heads, scale=scale, cos_t=p("cos"), sin_t=p("sin"), pairs=self.pairs, positions=self.cos.shape[0], adjacent=int(adjacent),
                             position=t["at"].data_ptr(), filled=t["at"][1:].data_ptr(), q_ld=heads * dim + q_gap if q_gap else 0, kv_ld=kv_heads * dim + kv_gap if kv_gap else 0,
                             weight_in=p("weight_in"), weight_out=p("weight_out"), k_held=p("k_held"), v_held=p("v_held"))
        self.room = torch.full((be.q4_attention_workspace_bytes(self.a, tokens),), 0xAB, dtype=torch.uint8, device="cuda")
        self.a.workspace, self.a.workspace_bytes = self.room.data_ptr(), self.room.numel()
        torch.cuda.synchronize()

    def enqueue(self, stream):
        self.be.dev_q4_attention(self.a, self.t["q"].data_ptr(), self.t["k"].data_ptr(), self.t["v"].data_ptr(), self.tokens, self.t["out"].data_ptr(), stream)

    def run(self):
        s = self.torch.cuda.Stream()
        self.enqueue(s.cuda_stream)
        self.be.dev_check(s.cuda_stream)
        return self

    def expected(self):
        rows = slice(self.rotated_from, self.rotated_from + self.tokens)
        turn = (lambda x: q4.rotate(x, self.cos[rows], self.sin[rows], self.adjacent)) if self.pairs else (lambda x: x)
        q, k_new = turn(self.q), turn(self.k)
        self.new = {"k": q4.quantise(k_new), "v": q4.quantise(self.v)}
        whole = {}
        for s in "kv":
            d, c = self.old[s]
            nd, nc = self.new[s]
            old = q4.values(q4.pack(c), d)[:, :self.filled]
            whole[s] = np.concatenate([old, (nc.reshape(*nd.shape, 32).astype(np.float64) - 8).transpose(1, 0, 2, 3).reshape(self.kv_heads, self.tokens, self.dim) *
                                       nd.astype(np.float64).repeat(32, -1).transpose(1, 0, 2)], 1)
        out, received = q4.attention(q, whole["k"], whole["v"], self.filled, self.scale)
        if self.weight_in is not None:
            received[:, :self.filled] += self.weight_in[:, :self.filled]
        # a score is off by at most `away`: q enters as 22 bits (2^-22 of its largest value), products are added in fp32 within tensor-core steps that may cut
        # (2^-23 each, some twenty one after the other), the scaled sum is rounded a few times: 2^-19 of sum |q| |k| covers them.  A weight is then off by 2 away + 2^-20 of
        # itself, and a row's output by that much of the largest value, and 2^-19 of it for the sums over slots.
        sizes = np.abs(q).max(-1).max() * np.abs(whole["k"]).sum(-1).max() * abs(self.scale)
        self.away = 2.0 ** -19 * sizes
        self.tolerance = np.abs(whole["v"]).max() * (2 * self.away + 2.0 ** -19)
        return out, received

    def check(self):
        out, received = self.expected()
        got = self.t["out"].cpu().numpy().astype(np.float64).reshape(out.shape)
        assert np.abs(got - out).max() <= self.tolerance
        # what the limit above does not see: the error as a whole is that of fp32 arithmetic
        assert np.linalg.norm(got - out) <= 8e-6 * np.linalg.norm(out)
        self.check_append()
        if self.weight_in is not None:
            w, n = self.t["weight_out"].cpu().numpy(), self.filled + self.tokens
            assert np.abs(w[:, :n] - received).max() <= (2 * self.away + 2.0 ** -19) * received.max()
            assert (w[:, n:] == -3.0).all()
        return got

    def check_append(self):
        f, n = self.filled, self.filled + self.tokens
        for s in "kv":
            d, c = self.new[s]
            got_c, got_d = q4.unpack(self.t[s + "_codes"].cpu().numpy()), self.t[s + "_scales"].cpu().numpy()
            before_c, before_d = q4.unpack(self.before[s + "_codes"].cpu().numpy()), self.before[s + "_scales"].cpu().numpy()
            assert np.array_equal(got_c[:, f:n], c.transpose(1, 0, 2)) and np.array_equal(got_d[:, f:n].view(np.uint16), d.transpose(1, 0, 2).view(np.uint16))
            for keep in (slice(0, f), slice(n, None)):
                assert np.array_equal(got_c[:, keep], before_c[:, keep]) and np.array_equal(got_d[:, keep].view(np.uint16), before_d[:, keep].view(np.uint16))
            h = self.t[s + "_held"].cpu().numpy().reshape(c.shape)
            assert np.array_equal(h, ((c.reshape(*d.shape, 32).astype(np.float32) - 8) * d.astype(np.float32)[..., None]).reshape(c.shape), equal_nan=True)


# tokens, filled, heads, kv_heads, dim
SHAPES = [(1, 0, 4, 2, 64), (1, 1, 1, 1, 32), (1, 15, 4, 4, 128), (1, 16, 4, 1, 128), (1, 31, 8, 2, 96), (1, 63, 32, 8, 128), (1, 1000, 32, 8, 128), (1, 2047, 7, 1, 64), (1, 700, 28, 4, 128),
          (1, 333, 16, 2, 256), (1, 257, 5, 5, 160), (1, 129, 24, 2, 192), (1, 97, 3, 1, 224), (1, 9001, 4, 2, 128),
          (2, 0, 4, 2, 64), (2, 5, 8, 1, 128), (3, 30, 4, 4, 32), (5, 4003, 32, 8, 128), (7, 60, 12, 4, 96), (8, 31, 16, 4, 256), (9, 33, 7, 1, 64), (16, 100, 32, 8, 128), (17, 16, 6, 2, 64),
          (40, 4001, 16, 8, 128), (35, 3333, 34, 34, 64), (130, 2500, 10, 10, 128),
          (33, 0, 4, 2, 64), (64, 64, 8, 2, 128), (77, 200, 16, 16, 64), (128, 0, 32, 8, 128), (129, 1, 12, 4, 96), (200, 55, 8, 1, 256), (512, 300, 8, 2, 128)]


@pytest.mark.parametrize("shape", SHAPES, ids=str)
@pytest.mark.parametrize("weights", [False, True])
def test_attention(be, shape, weights):
    Setup(be, *shape, weights=weights, seed=sum(shape)).run().check()


@pytest.mark.parametrize("tokens", [1, 6, 40])
def test_strides_rotations_and_scales(be, tokens):
    Setup(be, tokens, 70, 8, 2, 128, q_gap=5, kv_gap=3, weights=True).run().check()
    Setup(be, tokens, 70, 8, 2, 128, adjacent=False).run().check()
    Setup(be, tokens, 70, 8, 2, 128, adjacent=False, pairs=20).run().check()
    Setup(be, tokens, 70, 8, 2, 128, adjacent=True, pairs=7, scale=0.3).run().check()
    Setup(be, tokens, 70, 8, 2, 64, pairs=0, scale=-0.2).run().check()
    Setup(be, tokens, 70, 8, 2, 64, slots=4096, weights=True).run().check()
    Setup(be, tokens, 500, 8, 2, 128, spread=12.0).run().check()      # a few slots have nearly all of the weight


def test_no_row_depends_on_earlier_calls_or_on_the_workspace(be):
    s = Setup(be, 4, 300, 8, 2, 128, weights=True).run()
    first = s.check().copy()
    for fill in (0, 0xFF):
        s.room.fill_(fill)
        s.run()
        assert np.array_equal(s.check(), first)


def test_weights_in_place(be):
    s = Setup(be, 3, 40, 4, 2, 64, weights=True)
    s.a.weight_out = s.a.weight_in
    s.run()
    _, received = s.expected()
    got = s.t["weight_in"].cpu().numpy()
    assert np.abs(got[:, :43] - received).max() <= (2 * s.away + 2.0 ** -19) * received.max()
    assert np.array_equal(got[:, 43:], s.weight_in[:, 43:])


@pytest.mark.parametrize("tokens", [1, 5, 40])
def test_a_captured_call_serves_every_step(be, tokens):
    """Captured once, replayed while position and filled advance: each replay gives what an eager call gives at that place."""
    import torch
    s = Setup(be, tokens, 20, 8, 2, 128, slots=256, weights=True)
    s.a.weight_out = s.a.weight_in
    eager = Setup(be, tokens, 20, 8, 2, 128, slots=256, weights=True)
    eager.a.weight_out = eager.a.weight_in
    st = torch.cuda.Stream()
    s.enqueue(st.cuda_stream)                       # kernels' attributes are set by a first call
    torch.cuda.synchronize()
    for n in ("k_codes", "v_codes", "k_scales", "v_scales"):
        s.t[n].copy_(s.before[n])
    s.t["weight_in"].copy_(eager.t["weight_in"])
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=st):
        s.enqueue(st.cuda_stream)
    for step in range(4):
        rows = torch.randn_like(s.t["k"])
        for one in (s, eager):
            one.t["k"].copy_(rows)
            one.t["at"].copy_(torch.tensor([min(step, 3), 20 + step * tokens], dtype=torch.int32))
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        eager.run()
        assert torch.equal(s.t["out"], eager.t["out"]) and torch.equal(s.t["weight_in"], eager.t["weight_in"]) and torch.equal(s.t["k_codes"], eager.t["k_codes"])
    be.dev_check(st.cuda_stream)


def test_two_calls_at_once(be):
    """Two sequences on two streams, each with its own workspace."""
    import torch
    a, b = Setup(be, 1, 3000, 32, 8, 128, weights=True, seed=1), Setup(be, 6, 2500, 32, 8, 128, weights=True, seed=2)
    sa, sb = torch.cuda.Stream(), torch.cuda.Stream()
    for _ in range(20):
        a.enqueue(sa.cuda_stream)
        b.enqueue(sb.cuda_stream)
    be.dev_check(sa.cuda_stream)
    be.dev_check(sb.cuda_stream)
    a.check()
    b.check()


def test_two_blocks_at_once(be):
    import torch
    a, b = Setup(be, 100, 1900, 16, 8, 128, weights=True, seed=3), Setup(be, 150, 900, 16, 16, 64, weights=True, seed=4)
    sa, sb = torch.cuda.Stream(), torch.cuda.Stream()
    for _ in range(10):
        a.enqueue(sa.cuda_stream)
        b.enqueue(sb.cuda_stream)
    be.dev_check(sa.cuda_stream)
    be.dev_check(sb.cuda_stream)
    a.check()
    b.check()


@pytest.mark.parametrize("shape", [(1, 9, 4, 2, 64), (1, 1500, 32, 8, 128), (1, 9000, 16, 8, 64), (3, 700, 32, 8, 128), (6, 600, 12, 4, 96), (30, 900, 8, 2, 128), (64, 2100, 16, 16, 64)], ids=str)
def test_the_error_is_that_of_32_bits(be, shape):
    """The error of all outputs together.  Scores are about 1 and pass some twelve sums, each off by 2^-24 of them; so are weights, and twice as many roundings follow: 2^-24 * 24 is
    below 2^-19.  Codes that entered the sums with their offset on were at 2^-18."""
    s = Setup(be, *shape, weights=True, seed=11 + sum(shape)).run()
    got, (out, received) = s.check(), s.expected()
    assert np.linalg.norm(got - out) <= 2.0 ** -19 * np.linalg.norm(out)
    w = s.t["weight_out"].cpu().numpy()[:, :received.shape[1]]
    assert np.linalg.norm(w - received) <= 2.0 ** -19 * np.linalg.norm(received)


@pytest.mark.parametrize("tokens,dim", [(1, 64), (5, 128), (40, 128), (40, 64)])
def test_rows_that_begin_anywhere(be, tokens, dim):
    """Inputs and outputs four bytes behind an aligned place: the same bits."""
    import torch
    s = Setup(be, tokens, 70, 8, 2, dim).run()
    first = s.check().copy()
    moved = {n: torch.cat([torch.zeros(1, device="cuda"), s.t[n].flatten()])[1:] for n in ("q", "k", "v", "out", "k_held", "v_held", "cos", "sin")}
    for n, x in moved.items():
        assert x.data_ptr() % 16 == 4
        if n not in ("q", "k", "v", "out"):
            setattr(s.a, {"cos": "cos_t", "sin": "sin_t"}.get(n, n), x.data_ptr())
    moved["out"].fill_(5.0)
    moved["k_held"].fill_(5.0)
    st = torch.cuda.Stream()
    torch.cuda.synchronize()
    be.dev_q4_attention(s.a, moved["q"].data_ptr(), moved["k"].data_ptr(), moved["v"].data_ptr(), tokens, moved["out"].data_ptr(), st.cuda_stream)
    be.dev_check(st.cuda_stream)
    assert np.array_equal(moved["out"].cpu().numpy().reshape(first.shape), first)
    assert torch.equal(moved["k_held"], s.t["k_held"].flatten()) and torch.equal(moved["v_held"], s.t["v_held"].flatten())


@pytest.mark.parametrize("tokens,filled,position", [(1, 64, 5), (3, 62, 5), (1, -1, 5), (2, 10, 9), (1, 10, -1), (40, 30, 0), (1, 2 ** 31 - 1, 0)])
def test_places_outside_the_cache_or_the_tables_write_nothing(be, tokens, filled, position):
    import torch
    from zeninfer_b200 import BackendError
    s = Setup(be, tokens, 10, 4, 2, 64, slots=64, weights=True)
    s.a.positions = 10
    s.t["at"].copy_(torch.tensor([position, filled], dtype=torch.int32))
    torch.cuda.synchronize()
    with pytest.raises(BackendError, match="position"):
        s.run()
    assert (s.t["out"] == 7.0).all() and (s.t["weight_out"] == -3.0).all() and (s.t["k_held"] == 0).all()
    for n, x in s.before.items():
        assert torch.equal(x.view(torch.uint8), s.t[n].view(torch.uint8))
    be.dev_check(0)


@pytest.mark.parametrize("tokens", [2, 40])
def test_a_value_that_is_not_finite_reaches_the_rows_that_see_it_only(be, tokens):
    from zeninfer_b200 import BackendError
    s = Setup(be, tokens, 50, 8, 2, 64, weights=False)
    s.v[1, 0, 3] = np.inf                        # token 1, kv head 0: seen by tokens 1 .. of query heads 0 .. 3
    s.t["v"].copy_(s.torch.from_numpy(s.v.reshape(tokens, -1)))
    s.torch.cuda.synchronize()
    s.run()                                      # the scores are finite
    out, _ = s.expected()
    got = s.t["out"].cpu().numpy().reshape(out.shape)
    assert np.isnan(got[1:, :4, :32]).all() and np.isfinite(got[:1]).all() and np.isfinite(got[:, 4:]).all() and np.isfinite(got[1:, :4, 32:]).all()
    fine = np.isfinite(got)
    assert np.abs(got[fine] - out[fine]).max() <= 2.0 ** -12
    s.check_append()
    s = Setup(be, tokens, 50, 8, 2, 64)
    s.t["q"][1, 64 * 5 + 2] = float("nan")       # token 1, head 5
    s.torch.cuda.synchronize()
    with pytest.raises(BackendError, match="non-finite"):
        s.run()
    got = s.t["out"].cpu().numpy().reshape(tokens, 8, 64)
    assert np.isnan(got[1, 5]).all() and np.isfinite(np.delete(got.reshape(tokens * 8, 64), 8 + 5, 0)).all()


def test_the_quantiser_at_its_borders(be):
    """Values on and beside the borders between two codes, zeros, subnormal and saturated scales, ties for the largest, values that are not finite."""
    rng = np.random.default_rng(9)
    s = Setup(be, 64, 0, 2, 2, 64, pairs=0)
    x = rng.standard_normal((64, 2, 64)).astype(np.float32)
    for t in range(40):
        d = np.float32(np.float16(rng.uniform(-1, 1) * 2.0 ** rng.integers(-12, 8)))
        border = ((rng.integers(0, 16, (2, 64)) - 8.5) * d).astype(np.float32)
        x[t] = np.nextafter(border, rng.choice([-np.inf, np.inf], border.shape).astype(np.float32)) if t % 3 else border
        x[t, :, ::32] = d * np.float32(-8)
    x[40] = 0
    x[41] = 1e-9
    x[42] = rng.standard_normal((2, 64)) * 1e-7
    x[43] = rng.standard_normal((2, 64)) * 1e6
    x[44] = 3e38
    x[45, :, :] = np.where(rng.random((2, 64)) < 0.5, 2.0, -2.0)
    x[46, 0, 5] = np.nan
    x[47, 1, 40] = -np.inf
    x[48] = -0.0
    x[49] = 2.0 ** -25 * 8
    x[50] = np.nextafter(np.float32(2.0 ** -25 * 8), np.float32(1))
    s.v = x
    s.t["v"].copy_(s.torch.from_numpy(x.reshape(64, -1)))
    s.torch.cuda.synchronize()
    s.run()
    s.expected()
    s.check_append()


# ---- eviction --------------------------------------------------------------------------------------------------------------

class Evict:
    def __init__(self, be, filled, kv_heads, dim, *, slots=None, room=None, weight=None, seed=0):
        import torch
        from zeninfer_b200.backend import Q4Cache
        self.torch, self.be, self.filled, self.kv_heads, self.dim = torch, be, filled, kv_heads, dim
        self.slots = slots or max(32, q4.round_up(filled, 32))
        rng = np.random.default_rng(seed)
        self.weight = rng.lognormal(0, 2, (kv_heads, self.slots)).astype(np.float32) if weight is None else weight

        def made(n, fill):
            codes = lambda: torch.from_numpy(rng.integers(0, 256, Q4Cache.codes_shape(kv_heads, dim, n), dtype=np.uint8) if fill else np.full(Q4Cache.codes_shape(kv_heads, dim, n), 0x5A, np.uint8)).cuda()   # noqa: E731
            scales = lambda: torch.from_numpy(rng.random(Q4Cache.scales_shape(kv_heads, dim, n)).astype(np.float16) if fill else np.full(Q4Cache.scales_shape(kv_heads, dim, n), 9, np.float16)).cuda()   # noqa: E731
            t = dict(k_codes=codes(), k_scales=scales(), v_codes=codes(), v_scales=scales())
            return t, Q4Cache.of(**t, kv_heads=kv_heads, head_dim=dim, slots=n)
        self.t, self.cache = made(self.slots, True)
        self.t["weight"] = torch.from_numpy(self.weight).cuda()
        self.room = room or self.slots
        self.to, self.to_cache = made(self.room, False)
        self.to["weight"] = torch.full((kv_heads, self.room), -5.0, device="cuda")
        self.d_filled = torch.tensor([filled], dtype=torch.int32, device="cuda")
        self.ws = torch.full((be.q4_cache_evict_workspace_bytes(self.cache),), 0xEE, dtype=torch.uint8, device="cuda")
        torch.cuda.synchronize()

    def run(self, keep, first, last, in_place=False, stream=None):
        torch = self.torch
        to, cache = (self.t, self.cache) if in_place else (self.to, self.to_cache)
        before_from, before_to = ({n: x.clone() for n, x in t.items()} for t in (self.t, to))
        kept = torch.full((self.kv_heads, keep), -9, dtype=torch.int32, device="cuda")
        st = torch.cuda.Stream()
        torch.cuda.synchronize()
        self.be.dev_q4_cache_evict(self.cache, self.t["weight"].data_ptr(), self.d_filled.data_ptr(), cache, to["weight"].data_ptr(), keep, first, last, self.ws.data_ptr(), self.ws.numel(),
                                   st.cuda_stream, d_kept=kept.data_ptr())
        self.be.dev_check(st.cuda_stream)
        ref = q4.kept_slots(self.weight, self.filled, keep, first, last)
        n = ref.shape[1]
        kept = kept.cpu().numpy()
        assert np.array_equal(kept[:, :n], ref) and (kept[:, n:] == -9).all()
        by_slot = lambda t, name: t[name].transpose(2, 3).reshape(self.kv_heads, -1, self.dim // 32, 16) if name.endswith("codes") else t[name]   # noqa: E731
        for name in ("k_codes", "v_codes", "k_scales", "v_scales", "weight"):
            got, src, old = by_slot(to, name).cpu().numpy(), by_slot(before_from, name).cpu().numpy(), by_slot(before_to, name).cpu().numpy()
            got, src, old = (a.view(np.uint8 if a.dtype == np.uint8 else np.uint16 if a.dtype == np.float16 else np.uint32) for a in (got, src, old))
            for h in range(self.kv_heads):
                assert np.array_equal(got[h, :n], src[h, ref[h]]), name
            assert np.array_equal(got[:, n:], old[:, n:]), name
        if not in_place:
            for n_, x in before_from.items():
                assert torch.equal(x.view(torch.uint8), self.t[n_].view(torch.uint8))


@pytest.mark.parametrize("filled,keep,first,last,kv_heads,dim", [
    (1, 1, 0, 0, 1, 32), (2, 1, 0, 0, 2, 64), (2, 1, 1, 0, 1, 64), (2, 1, 0, 1, 1, 64), (33, 32, 4, 8, 2, 128), (100, 64, 64, 0, 2, 96), (100, 64, 0, 64, 2, 96), (100, 64, 10, 54, 3, 256), (100, 99, 4, 32, 2, 128),
    (1100, 1024, 4, 64, 8, 128), (5000, 37, 1, 2, 2, 160), (9999, 5000, 0, 0, 1, 64), (20000, 8192, 4, 512, 2, 128), (64, 64, 4, 8, 2, 64), (10, 64, 4, 8, 2, 64), (0, 32, 4, 8, 2, 64)])
@pytest.mark.parametrize("in_place", [False, True])
def test_eviction(be, filled, keep, first, last, kv_heads, dim, in_place):
    Evict(be, filled, kv_heads, dim, slots=q4.round_up(max(filled, keep), 32), seed=filled).run(keep, first, last, in_place)


@pytest.mark.parametrize("in_place", [False, True])
def test_eviction_of_equal_and_strange_weights(be, in_place):
    rng = np.random.default_rng(3)
    n = 3000
    some = rng.choice(np.array([0.0, -0.0, 1.0, 1.0, 2.0, np.inf, -np.inf, np.nan, -1.0, 1e-42, -1e-42], np.float32), (4, 3008))
    some[3] = 1.0
    for keep in (1, 500, 1500, 2999):
        Evict(be, n, 4, 64, slots=3008, weight=some).run(keep, 0, 0, in_place)
    Evict(be, n, 4, 64, slots=3008, weight=some).run(700, 300, 300, in_place)


def test_eviction_into_a_smaller_cache_and_outside_it(be):
    from zeninfer_b200 import BackendError
    Evict(be, 1000, 2, 128, room=96).run(70, 4, 8)
    e = Evict(be, 1000, 2, 128)
    e.d_filled.fill_(1025)
    with pytest.raises(BackendError, match="position"):
        e.be.dev_q4_cache_evict(e.cache, e.t["weight"].data_ptr(), e.d_filled.data_ptr(), e.to_cache, e.to["weight"].data_ptr(), 10, 0, 0, e.ws.data_ptr(), e.ws.numel(), 1)
        e.be.dev_check(1)
    assert (e.to["k_codes"] == 0x5A).all() and (e.to["weight"] == -5.0).all()


def test_a_sequence_with_evictions(be):
    """Steps, an eviction by the weights they received, more steps: each is the plain attention over the slots that stayed."""
    import torch
    s = Setup(be, 1, 60, 8, 2, 64, slots=64, weights=True, seed=5)
    s.a.weight_out = s.a.weight_in
    st = torch.cuda.Stream()
    ws = torch.zeros(be.q4_cache_evict_workspace_bytes(s.cache), dtype=torch.uint8, device="cuda")
    filled = 60
    for step in range(12):
        if filled == 64:
            before = s.t["weight_in"].cpu().numpy()
            kept = torch.zeros((2, 48), dtype=torch.int32, device="cuda")
            be.dev_q4_cache_evict(s.cache, s.a.weight_in, s.a.filled, s.cache, s.a.weight_out, 48, 4, 16, ws.data_ptr(), ws.numel(), st.cuda_stream, d_kept=kept.data_ptr())
            be.dev_advance_position(s.a.filled, 48 - 64, st.cuda_stream)
            st.synchronize()
            assert np.array_equal(kept.cpu().numpy(), q4.kept_slots(before, 64, 48, 4, 16))
            filled = 48
        k_old, v_old = (q4.values(s.t[n + "_codes"].cpu().numpy(), s.t[n + "_scales"].cpu().numpy())[:, :filled] for n in "kv")
        w_old = s.t["weight_in"].cpu().numpy()[:, :filled]
        s.enqueue(st.cuda_stream)
        be.dev_advance_position(s.a.filled, 1, st.cuda_stream)
        be.dev_check(st.cuda_stream)
        rows = slice(s.rotated_from, s.rotated_from + 1)
        q, k_new = q4.rotate(s.q, s.cos[rows], s.sin[rows], True), q4.rotate(s.k, s.cos[rows], s.sin[rows], True)
        k, v = np.concatenate([k_old, q4.held(k_new).transpose(1, 0, 2)], 1), np.concatenate([v_old, q4.held(s.v).transpose(1, 0, 2)], 1)
        out, received = q4.attention(q, k, v, filled, s.scale)
        received[:, :filled] += w_old
        got = s.t["out"].cpu().numpy().reshape(out.shape)
        assert np.linalg.norm(got - out) <= 8e-6 * np.linalg.norm(out)
        assert np.abs(s.t["weight_in"].cpu().numpy()[:, :filled + 1] - received).max() <= 1e-5 * received.max()
        filled += 1


@pytest.mark.parametrize("shape", [(1, 70, 8, 2, 64), (1, 9001, 4, 2, 128), (6, 70, 8, 2, 128), (9, 31, 8, 2, 96), (40, 70, 8, 2, 64), (40, 0, 8, 2, 128), (40, 4001, 16, 8, 128), (64, 40, 8, 2, 96)], ids=str)
@pytest.mark.parametrize("keys", [0.0, 2.0 ** -14, 1.0])
def test_rows_of_zeros_and_scales_that_leave_nothing_of_a_score(be, shape, keys):
    """A row whose scores are zero, or too small to be told from it, is the mean of what it sees, whatever the keys' sizes are: its products' factor may be less than the smallest
    normal number, and what is masked must stay masked after it."""
    import torch
    tokens, filled, heads, kv_heads, dim = shape
    for zeros, scale, weights in ((slice(None), 0.0, True), (slice(0, None, 3), 0.0, True), (slice(0, None, 2), 1e-3, False), (slice(0, 0), 1e-9, True), (slice(0, 0), -1e-38, False),
                                  (slice(0, None, 2), 1e-45, True)):
        s = Setup(be, *shape, weights=weights, scale=scale, seed=sum(shape))
        s.q.reshape(tokens * heads, dim)[zeros] = 0
        s.k *= np.float32(keys)
        d, c = s.old["k"]
        s.old["k"] = ((d.astype(np.float32) * np.float32(keys)).astype(np.float16), c)
        s.t["q"].copy_(torch.from_numpy(s.q.reshape(tokens, -1)))
        s.t["k"].copy_(torch.from_numpy(s.k.reshape(tokens, -1)))
        s.t["k_scales"][:, :filled] = torch.from_numpy(s.old["k"][0][:, :filled]).cuda()
        s.before["k_scales"] = s.t["k_scales"].clone()
        s.torch.cuda.synchronize()
        s.run().check()


@pytest.mark.parametrize("tokens,stay,filled,heads,kv_heads,dim", [(2, 1, 30, 8, 2, 64), (5, 3, 700, 32, 8, 128), (9, 4, 70, 8, 2, 96), (40, 1, 300, 8, 2, 128), (64, 40, 2000, 16, 16, 64)])
def test_the_weights_of_the_tokens_that_stay(be, tokens, stay, filled, heads, kv_heads, dim):
    """A block writes its weights beside the old ones; called again with its first tokens it leaves what those alone give, and the same slots, whichever kernels take the two."""
    import torch
    s = Setup(be, tokens, filled, heads, kv_heads, dim, weights=True, seed=tokens).run()
    s.check()
    slots = {n: s.t[n].clone() for n in s.before}
    rows = s.t["out"][:stay].clone()
    s.tokens, s.q, s.k, s.v = stay, s.q[:stay], s.k[:stay], s.v[:stay]
    s.t["weight_out"].fill_(-3.0)
    room = torch.full((be.q4_attention_workspace_bytes(s.a, stay),), 0xAB, dtype=torch.uint8, device="cuda")
    s.a.workspace, s.a.workspace_bytes = room.data_ptr(), room.numel()
    torch.cuda.synchronize()
    s.run()
    assert all(torch.equal(x.view(torch.uint8), s.t[n].view(torch.uint8)) for n, x in slots.items())
    out, received = s.expected()
    w, n = s.t["weight_out"].cpu().numpy(), filled + stay
    assert np.abs(w[:, :n] - received).max() <= (2 * s.away + 2.0 ** -19) * received.max() and (w[:, n:] == -3.0).all()
    assert float((s.t["out"][:stay] - rows).abs().max()) <= 2 * s.tolerance
