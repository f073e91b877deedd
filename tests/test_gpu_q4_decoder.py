"""LlamaDecoder with its keys and values in 4 bits, with slots dropped by the attention they received, and with drafted tokens: what a user calls, against the model in 64 bits.

A key or value near a border between two codes may take either, for the products that make it are within 5e-5 of their sums.  So the plain model attends to the codes that the decoder
holds, after it has seen that they are roundings of its own values and that older ones stayed where its own weights say.  What is left is the
products' difference: logits are compared within 1e-3 of their largest, the bar of the other generation tests, and every test shows on the plain model that what it is about (the
four bits, the drops) is worth many times that."""
import numpy as np
import pytest

import q4_cases as q4
from q4_llama import PlainLlama
from zeninfer_b200.backend import ACT_FP32
from zeninfer_b200.llama import LlamaConfig, LlamaDecoder, synthetic_tensors

pytestmark = pytest.mark.gpu
SEED, STD = 11, 0.08
BAR = 1e-3


def config(dim: int) -> LlamaConfig:
    return LlamaConfig(embedding=256, layers=2, heads=512 // dim, kv_heads=2, head_dim=dim, ffn=512, vocab=700, rope_base=10000.0, context=256)


@pytest.fixture(scope="module")
def be():
    from zeninfer_b200 import Backend
    return Backend()


def decoder(be, cfg, **kwargs):
    return LlamaDecoder(be, cfg, synthetic_tensors(cfg, SEED, STD), act_mode=ACT_FP32, **kwargs)


def near(got, want):
    return float(np.abs(got - want).max() / np.abs(want).max())


class Watched:
    """Repeats on the plain model what a decoder is asked: prefill and step, with the place they happen at."""

    def __init__(self, dec, plain):
        self.dec, self.plain, self.last, self.worst, self.calls = dec, plain, None, 0.0, []
        self.prefill, self.step = dec.prefill, dec.step
        dec.prefill, dec.step = self._prefill, self._step

    def cache(self, layer):
        b = {n: t[layer].cpu().numpy() for n, t in self.dec.sequence.buffers.items()}
        return tuple(q4.values(b[x + "_codes"], b[x + "_scales"])[:, :self.dec.held] for x in "kv")

    def follow(self, tokens, place):
        self.dec.stream.synchronize()
        self.last = self.plain.block(tokens, place, self.cache)
        self.calls.append(len(tokens))

    def _prefill(self, d_tokens, count):
        place = self.dec.place
        self.prefill(d_tokens, count)
        self.follow(d_tokens[:count].cpu().tolist(), place)

    def _step(self, want_token):
        self.dec.stream.synchronize()
        token, place = int(self.dec.token.item()), self.dec.place
        self.step(want_token)
        self.follow([token], place)
        if want_token:
            self.see(self.dec.last_logits()[None])

    def see(self, logits):
        self.worst = max(self.worst, near(logits, self.last[-len(logits):]))


@pytest.mark.parametrize("dim", [32, 64, 128])
@pytest.mark.parametrize("graphs", [False, True])
def test_a_cache_in_four_bits(be, dim, graphs):
    cfg = config(dim)
    tokens = np.random.default_rng(dim).integers(0, cfg.vocab, 90).tolist()
    dec = decoder(be, cfg, kv="q4")
    try:
        if graphs:
            dec.capture()
        assert dec.slots == 256 and dec.sequence.nbytes() == cfg.layers * 2 * cfg.kv_width * 256 * 9 // 16
        for _ in range(2):                        # the second sequence finds the first one's slots
            seen, exact = Watched(dec, PlainLlama(cfg, SEED, STD, 256)), PlainLlama(cfg, SEED, STD, 256, quantised=False)
            dec.reset()
            at = 0
            for n in (1, 1, 40, 17, 3, 28):       # steps and blocks
                seen.see(dec.feed(tokens[at:at + n], [n - 1]))
                at += n
            dec.prefill, dec.step = seen.prefill, seen.step
            assert seen.calls == [1, 1, 40, 17, 1, 1, 1, 28] and seen.worst <= BAR
            assert near(exact.block(tokens, 0)[-1:], seen.last[-1:]) > 10 * BAR
            assert dec.held == dec.place == 90
    finally:
        dec.close()


@pytest.mark.parametrize("dim,slots,keep,first,last", [(64, 96, 48, 4, 8), (128, 64, None, 2, None), (32, 96, 80, 0, 0), (64, 64, 33, 4, 29)])
def test_slots_are_dropped_by_the_attention_they_received(be, dim, slots, keep, first, last):
    cfg = config(dim)
    prompt = np.random.default_rng(slots + dim).integers(0, cfg.vocab, 130).tolist()
    dec = decoder(be, cfg, kv="q4", kv_slots=slots, kv_keep=keep, kv_keep_first=first, kv_keep_last=last)
    try:
        dec.capture()
        for _ in range(2):
            dec.reset()
            plain, never = PlainLlama(cfg, SEED, STD, slots, dec.keep, dec.keep_first, dec.keep_last), PlainLlama(cfg, SEED, STD, 256)
            seen = Watched(dec, plain)
            got = dec.generate(prompt, 40, on_token=lambda t: None)
            dec.prefill, dec.step = seen.prefill, seen.step
            assert seen.worst <= BAR and plain.drops >= 2
            whole = never.block(prompt + got[:-1], 0)
            assert near(seen.last[-1:], whole[-1:]) > 10 * BAR
            assert dec.pos.item() == dec.place == 169 and dec.filled.item() == dec.held <= slots
        again = dec.generate(prompt, 40)          # without a callback steps are launched ahead
        assert again == got
    finally:
        dec.close()


@pytest.mark.parametrize("options", [{}, dict(kv="q4"), dict(kv="q4", kv_slots=96, kv_keep=64)], ids=str)
@pytest.mark.parametrize("drafts", [1, 5, 16])
def test_drafted_tokens_are_those_of_the_model(be, options, drafts):
    cfg = config(64)
    prompt = np.random.default_rng(drafts).integers(0, cfg.vocab, 50).tolist()
    dec = decoder(be, cfg, **options)
    try:
        dec.capture()
        greedy = dec.generate(prompt, 60)
        # drafts of all kinds: right ones, wrong ones at every place, none
        rng = np.random.default_rng(3)

        def propose(context, n):
            done = len(context) - len(prompt)
            assert context[:len(prompt)] == prompt
            right = greedy[done:done + int(rng.integers(0, n + 1))]
            wrong = int(rng.integers(0, len(right) + 1))
            return [t if i != wrong else (t + 1) % cfg.vocab for i, t in enumerate(right)]

        if not options:
            assert dec.generate_drafted(prompt, 60, drafts, propose) == greedy
            assert dec.generate_drafted(prompt, 60, drafts, lambda c, n: []) == greedy
            assert dec.generate_drafted(prompt, 1, drafts) == greedy[:1] and dec.generate_drafted(prompt, 0, drafts) == []
            return
        plain = PlainLlama(cfg, SEED, STD, dec.slots, dec.keep, 4, dec.keep_last if dec.keep else 0)
        seen, block = Watched(dec, plain), dec.forward_block

        def forward_block(tokens, start, tail):
            answer = block(tokens, start, tail)
            seen.see(answer.cpu().numpy())
            return answer

        dec.forward_block = forward_block
        got = dec.generate_drafted(prompt, 60, drafts, propose)
        assert len(got) == 60 and seen.worst <= BAR and max(seen.calls[4:]) > 1
        assert plain.drops >= (dec.keep is not None)
    finally:
        dec.close()


def test_sampled_drafts_follow_the_seed_and_the_filters(be):
    cfg = config(64)
    prompt = list(range(30)) + list(range(20))
    dec = decoder(be, cfg)
    try:
        one = dec.generate_drafted(prompt, 40, 4, temperature=0.9, top_k=20, top_p=0.9, seed=5)
        assert dec.generate_drafted(prompt, 40, 4, temperature=0.9, top_k=20, top_p=0.9, seed=5) == one
        assert dec.generate_drafted(prompt, 40, 4, temperature=0.9, top_k=20, top_p=0.9, seed=6) != one
        assert dec.generate_drafted(prompt, 40, 4, temperature=0.9, top_k=1, seed=7) == dec.generate(prompt, 40)
        # every token is among the twenty likeliest of the plain model's row, give or take the bar
        plain = PlainLlama(cfg, SEED, STD, 256, quantised=False)
        rows = plain.block(prompt + one[:-1], 0)[len(prompt) - 1:]
        for row, t in zip(rows, one):
            assert row[t] >= np.sort(row)[-20] - 2 * BAR * np.abs(row).max()
    finally:
        dec.close()


def test_refusals_of_the_decoder(be):
    cfg = config(64)
    for bad in (dict(kv="q5"), dict(kv_slots=64), dict(kv_keep=4), dict(kv="q4", kv_keep=4), dict(kv="q4", kv_slots=64, kv_keep=60), dict(kv="q4", kv_slots=64, kv_keep=0),
                dict(kv="q4", kv_slots=64, kv_keep=32, kv_keep_first=30, kv_keep_last=3)):
        with pytest.raises(ValueError):
            decoder(be, cfg, **bad)
    dec = decoder(be, cfg, kv="q4", kv_slots=64, kv_keep=32)
    try:
        dec.feed(list(range(60)))
        dec.forward_block([1, 2, 3], 58, 1)       # back two
        with pytest.raises(ValueError):
            dec.forward_block([1], 62, 1)         # a gap
        dec.feed(list(range(20)))                 # drops: what was before is there in part only
        with pytest.raises(ValueError):
            dec.forward_block([1], 20, 1)
        for bad in (dict(drafts=0), dict(drafts=65), dict(max_new=500)):
            with pytest.raises(ValueError):
                dec.generate_drafted([1, 2], **{**dict(max_new=4, drafts=2), **bad})
        with pytest.raises(ValueError):
            dec.generate_drafted([1, 2], 4, 2, propose=lambda c, n: [cfg.vocab])
    finally:
        dec.close()


def test_the_command(be, tmp_path, capsys):
    import os
    import sys
    sys.path.insert(0, os.path.join(os.path.dirname(__file__), "golden"))
    from make_llama_golden import write_gguf
    from zeninfer_b200.__main__ import main
    cfg = LlamaConfig(embedding=256, layers=2, heads=4, kv_heads=2, head_dim=64, ffn=512, vocab=700, rope_base=10000.0, context=256)
    path = str(tmp_path / "m.gguf")
    write_gguf(path, cfg, synthetic_tensors(cfg, SEED, STD))
    ids = {}
    for extra in ("", "--kv q4", "--kv q4 --draft 3", "--draft 3", "--kv q4 --kv-slots 64 --kv-keep 32 --draft 4"):
        assert main(["generate", "--model", path, "--prompt-ids", ",".join(map(str, range(40))), "--max-new", "30"] + extra.split()) == 0
        ids[extra] = [int(t) for t in capsys.readouterr().out.strip().split("\n")[-1].split(",")]
        assert len(ids[extra]) == 30


@pytest.mark.parametrize("kv", [{}, dict(kv="q4")], ids=str)
@pytest.mark.parametrize("drafts", [3, 12])
def test_drafts_are_checked_in_the_arithmetic_of_the_steps(be, monkeypatch, kv, drafts):
    """A decoder as the registry loads it takes its prompt with 32-bit activations and its steps with int8 ones.  generate() draws from the steps' logits, so drafted tokens are
    checked against blocks in the steps' mode; the prompt, and a caller's own forward_block, keep the prompt's."""
    from zeninfer_b200.backend import ACT_INT8
    cfg = config(64)
    dec = LlamaDecoder(be, cfg, synthetic_tensors(cfg, SEED, STD), act_mode=ACT_INT8, prompt_act_mode=ACT_FP32, **kv)
    product, modes = be.dev_gemm_q8_0, []

    def recorded(*args, act_mode=ACT_INT8, **more):
        modes.append(act_mode)
        return product(*args, act_mode=act_mode, **more)

    monkeypatch.setattr(be, "dev_gemm_q8_0", recorded)
    try:
        dec.capture()
        prompt = np.random.default_rng(5).integers(0, cfg.vocab, 40).tolist()
        assert len(dec.generate_drafted(prompt[:5], 20, drafts, lambda c, n: [1] * n)) == 20       # the first blocks of the decoder, in buffers that serve both modes
        assert set(modes) == {ACT_INT8}
        del modes[:]
        greedy = dec.generate(prompt, 40)
        assert set(modes) == {ACT_FP32}
        of_prompt = len(modes)
        del modes[:]
        assert len(dec.generate_drafted(prompt, 40, drafts, lambda c, n: greedy[len(c) - 40:][:n])) == 40
        assert set(modes[:of_prompt]) == {ACT_FP32} and set(modes[of_prompt:]) == {ACT_INT8}
        del modes[:]
        dec.forward_block(greedy[:9], 40, 9)
        assert set(modes) == {ACT_FP32}
    finally:
        dec.close()


@pytest.mark.parametrize("drafts", [2, 5, 16])
def test_drafted_tokens_drop_slots_where_steps_do(be, drafts):
    """Slots are dropped when a step finds none free, as in generate(), and never for a block whose tokens may be taken back."""
    cfg = config(64)
    dec = decoder(be, cfg, kv="q4", kv_slots=96, kv_keep=64)
    try:
        dec.capture()
        prompt = np.random.default_rng(17).integers(0, cfg.vocab, 50).tolist()
        drop, places = be.dev_q4_cache_evict, []

        def dropped(*args, **more):
            places.append((dec.place, dec.held))
            return drop(*args, **more)

        be.dev_q4_cache_evict = dropped
        try:
            greedy = dec.generate(prompt, 120, on_token=lambda t: None)
            steps = places[:]
            del places[:]
            asked = []

            def propose(context, n):
                done = len(context) - len(prompt)
                asked.append(n)
                right = greedy[done:done + n]
                wrong = done % 7                       # right ones, and wrong ones at every place
                return [t if i != wrong else (t + 1) % cfg.vocab for i, t in enumerate(right)]

            assert len(dec.generate_drafted(prompt, 120, drafts, propose)) == 120
        finally:
            del be.dev_q4_cache_evict
        assert len(steps) == 3 * cfg.layers and set(places) == set(steps) and len(places) == len(steps)
        assert all(held == dec.slots for _, held in places) and 1 <= min(asked) < max(asked) == drafts
    finally:
        dec.close()


def test_what_rejected_drafts_gave_stays_counted(be):
    """Every token gives each query head's weight of 1 to the slots it sees.  With right drafts, or none, the slots have what the tokens of the sequence gave; rejected ones add to the slots that
    were there before them."""
    cfg = config(64)
    dec = decoder(be, cfg, kv="q4", kv_slots=192, kv_keep=128)
    try:
        prompt = np.random.default_rng(19).integers(0, cfg.vocab, 40).tolist()
        greedy = dec.generate(prompt, 60)

        def given(propose):
            assert len(dec.generate_drafted(prompt, 60, 4, propose)) == 60
            dec.stream.synchronize()
            sums = dec.weight[:, :, :dec.held].sum(-1).cpu().numpy() / (cfg.heads // cfg.kv_heads)
            return sums, dec.held

        right = lambda c, n: greedy[len(c) - 40:][:n]                                # noqa: E731
        wrong = lambda c, n: [(t + 1) % cfg.vocab for t in greedy[len(c) - 40:][:n]]   # noqa: E731
        for propose, more in ((lambda c, n: [], False), (right, False), (wrong, True)):
            sums, held = given(propose)
            assert held == 99
            if more:
                assert (sums > held + 1).all()
            else:
                assert (np.abs(sums - held) <= 1e-3 * held).all()
    finally:
        dec.close()


@pytest.mark.parametrize("options", [{}, dict(kv="q4")], ids=str)
def test_drafts_by_look_up_are_those_of_look_up(be, options):
    """Without a function of the caller's the context is looked up in an index that grows with it: the same drafts, and the same tokens."""
    cfg = config(64)
    dec = decoder(be, cfg, **options)
    try:
        prompt = (list(range(40)) * 2)[:70]
        blocks = {}
        block = dec.forward_block
        for name, propose in (("index", None), ("scan", dec.look_up)):
            asked = blocks[name] = []
            dec.forward_block = lambda tokens, start, tail: (asked.append(tokens), block(tokens, start, tail))[1]
            asked.append(dec.generate_drafted(prompt, 60, 4, propose, temperature=0.8, top_k=3, seed=4))
        assert blocks["index"] == blocks["scan"] and len(blocks["index"]) > 2
    finally:
        dec.close()


@pytest.mark.parametrize("slots", [0, -1, -64])
def test_no_slots_are_refused(be, slots):
    for keep in (None, 4):
        with pytest.raises(ValueError, match="kv_slots"):
            decoder(be, config(64), kv="q4", kv_slots=slots, kv_keep=keep)
