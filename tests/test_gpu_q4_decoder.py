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


@pytest.mark.parametrize("options", [{}, dict(kv="q4"), dict(kv="q4", kv_slots=96, kv_keep=64)], ids=str)
@pytest.mark.parametrize("drafts", [1, 4, 13])
@pytest.mark.parametrize("mode", ["int8", "fp32"])
def test_a_drafted_token_is_the_pick_of_the_row_before_it(be, options, drafts, mode):
    """Every token that comes back is the first of the largest logits of the row that the decoder formed for its place: a draft kept or dropped wrongly is another."""
    from zeninfer_b200.backend import ACT_INT8
    cfg = config(64)
    dec = LlamaDecoder(be, cfg, synthetic_tensors(cfg, SEED, STD), act_mode=ACT_INT8 if mode == "int8" else ACT_FP32, prompt_act_mode=ACT_FP32, **options)
    try:
        dec.capture()
        prompt = np.random.default_rng(drafts + 20).integers(0, cfg.vocab, 50).tolist()
        greedy, rng, rows, lengths = dec.generate(prompt, 70), np.random.default_rng(1), {}, []
        feed, block, step = dec.feed_prompt, dec.forward_block, dec.step

        def feed_prompt(*args):
            feed(*args)
            rows[len(prompt) - 1] = dec.last_logits()

        def forward_block(tokens, start, tail):
            answer = block(tokens, start, tail)
            dec.stream.synchronize()
            rows.update(enumerate(answer.cpu().numpy(), start))
            lengths.append(tail)
            return answer

        def one_step(want_token):
            dec.stream.synchronize()
            place = int(dec.pos.item())
            step(want_token)
            rows[place] = dec.last_logits()

        def propose(context, n):
            done = len(context) - len(prompt)
            right = greedy[done:done + int(rng.integers(0, n + 1))]
            return [t if rng.random() < 0.8 else int(rng.integers(cfg.vocab)) for t in right]

        dec.feed_prompt, dec.forward_block, dec.step = feed_prompt, forward_block, one_step
        got = dec.generate_drafted(prompt, 70, drafts, propose)
        assert got == [int(rows[len(prompt) - 1 + i].argmax()) for i in range(70)]
        assert max(lengths) > 1 and len(lengths) < 70
    finally:
        dec.close()


def test_the_command_prints_what_the_decoder_gives(be, tmp_path, capsys, monkeypatch):
    import os
    import sys
    sys.path.insert(0, os.path.join(os.path.dirname(__file__), "golden"))
    from make_llama_golden import write_gguf
    from zeninfer_b200 import registry
    from zeninfer_b200.__main__ import main
    cfg = LlamaConfig(embedding=256, layers=2, heads=4, kv_heads=2, head_dim=64, ffn=512, vocab=700, rope_base=10000.0, context=256)
    path, prompt = str(tmp_path / "m.gguf"), list(range(20)) * 2
    write_gguf(path, cfg, synthetic_tensors(cfg, SEED, STD))
    made = []
    init = LlamaDecoder.__init__
    monkeypatch.setattr(LlamaDecoder, "__init__", lambda self, *a, **k: (made.append(self), init(self, *a, **k))[1])
    for extra, options, drafts in (("", {}, 0), ("--draft 3", {}, 3), ("--kv q4", dict(kv="q4"), 0), ("--kv q4 --draft 3", dict(kv="q4"), 3),
                                   ("--kv q4 --kv-slots 64 --kv-keep 32 --draft 4", dict(kv="q4", kv_slots=64, kv_keep=32), 4),
                                   ("--kv q4 --kv-slots 96 --temperature 0.8 --top-k 20 --top-p 0.9 --seed 3", dict(kv="q4", kv_slots=96), 0)):
        assert main(["generate", "--model", path, "--prompt-ids", ",".join(map(str, prompt)), "--max-new", "50"] + extra.split()) == 0
        ids = [int(t) for t in capsys.readouterr().out.strip().split("\n")[-1].split(",")]
        dec = registry.load_model(be, path, **options)
        try:
            assert made[-2].q4 == dec.q4 == bool(options)
            if options:
                assert (made[-2].slots, made[-2].keep) == (dec.slots, dec.keep) == (options.get("kv_slots", 256), options.get("kv_keep", 72 if "kv_slots" in options else None))
            sampling = dict(temperature=0.8, top_k=20, top_p=0.9, seed=3) if "temperature" in extra else {}
            assert ids == (dec.generate_drafted(prompt, 50, drafts) if drafts else dec.generate(prompt, 50, **sampling))
        finally:
            dec.close()
        made.clear()


def test_a_rank_holds_its_own_heads(be):
    """A sharded decoder's cache has this rank's heads: step by step the same attention, slots and weights as those heads of a decoder that has all.  (One rank after the other: nothing is exchanged
    in this part.)"""
    cfg = config(64)
    options = dict(kv="q4", kv_slots=64, kv_keep=40)
    whole = decoder(be, cfg, **options)
    ranks = [decoder(be, cfg, rank=r, world=2, gather="nccl", **options) for r in range(2)]
    try:
        half = lambda t, r: t[r * (t.shape[0] // 2):(r + 1) * (t.shape[0] // 2)]   # noqa: E731
        rng = np.random.default_rng(2)
        for step in range(70):
            import torch
            for n in ("q", "k", "v"):
                getattr(whole, n).copy_(torch.from_numpy(rng.standard_normal(getattr(whole, n).shape[0]).astype(np.float32)))
                for r, dec in enumerate(ranks):
                    getattr(dec, n).copy_(half(getattr(whole, n), r))
            torch.cuda.synchronize()
            for dec in (whole, *ranks):
                dec._make_room(1)
                st = dec.stream.cuda_stream
                be.dev_q4_attention(dec.q4_calls[1], dec.q.data_ptr(), dec.k.data_ptr(), dec.v.data_ptr(), 1, dec.att_mine.data_ptr(), st)
                be.dev_advance_position(dec.pos.data_ptr(), 1, st)
                be.dev_advance_position(dec.filled.data_ptr(), 1, st)
                be.dev_check(st)
            for r, dec in enumerate(ranks):
                assert torch.equal(dec.att_mine, half(whole.att, r)) and int(dec.filled) == int(whole.filled) == dec.held
        for r, dec in enumerate(ranks):
            assert dec.q4_calls[1].cache.kv_heads == 1 and dec.q4_calls[1].heads == cfg.heads // 2 and dec.floor == whole.floor == 40
            for n in ("k_codes", "v_codes", "weight"):
                assert torch.equal(dec.sequence.buffers[n][1], half(whole.sequence.buffers[n][1], r))
    finally:
        for dec in (whole, *ranks):
            dec.close()


def test_a_look_up_of_a_subclass_is_asked(be):
    cfg, asked = config(64), []

    class Own(LlamaDecoder):
        def look_up(self, context, drafts):
            asked.append((len(context), drafts))
            return context[:drafts]

    dec = Own(be, cfg, synthetic_tensors(cfg, SEED, STD), act_mode=ACT_FP32)
    try:
        assert len(dec.generate_drafted(list(range(20)), 12, 3)) == 12
        assert asked[0] == (21, 3) and all(1 <= n <= 3 for _, n in asked)
    finally:
        dec.close()
