"""The 4-bit cache and the check of drafted tokens without a GPU: sizes, refusals, and the plain implementations the GPU tests compare with."""
import ctypes as C

import numpy as np
import pytest

from zeninfer_b200 import backend, blocks, build

import q4_cases as q4
from zeninfer_b200.backend import DraftCheck, Q4Attention, Q4Cache


@pytest.fixture(scope="module")
def lib():
    library = backend.load_library(build.build())
    yield library
    library.zen_cuda_shutdown()      # forgets that no device was found, so that the next one to ask is told why


def cache(**changes):
    c = dict(k_codes=0x1000000, v_codes=0x2000000, k_scales=0x3000000, v_scales=0x4000000, kv_heads=2, head_dim=64, slots=96)
    return Q4Cache(**{**c, **changes})


def attention(c=None, **changes):
    a = dict(cache=c or cache(), heads=4, scale=0.0, cos_t=0x5000000, sin_t=0x5100000, pairs=32, positions=128, adjacent=1, position=0x5200000, filled=0x5200010,
             workspace=0x6000000, workspace_bytes=1 << 40)
    return Q4Attention(**{**a, **changes})


def refused(lib, value):
    assert value == 0
    return lib.zen_cuda_last_error().decode()


BAD_CACHES = [dict(k_codes=0), dict(v_scales=0), dict(k_codes=0x1000008), dict(kv_heads=0), dict(head_dim=0), dict(head_dim=48), dict(head_dim=288), dict(slots=0), dict(slots=40)]


@pytest.mark.parametrize("bad", BAD_CACHES)
def test_a_cache_that_is_none_is_refused(lib, bad):
    assert lib.zen_cuda_q4_attention_workspace_bytes(attention(cache(**bad)), 1) == 0
    assert "bad arguments" in refused(lib, lib.zen_cuda_dev_q4_attention(attention(cache(**bad)), 16, 16, 16, 1, 16, None))
    assert lib.zen_cuda_q4_cache_evict_workspace_bytes(cache(**bad)) == 0
    assert "bad arguments" in refused(lib, lib.zen_cuda_dev_q4_cache_evict(cache(**bad), 16, 16, cache(), 16, 1, 0, 0, None, 16, 1 << 40, None))


@pytest.mark.parametrize("bad,tokens,why", [
    (dict(), 0, "tokens"), (dict(), 97, "tokens"), (dict(heads=0), 1, "heads"), (dict(heads=3), 1, "heads"), (dict(filled=0), 1, "rows"), (dict(q_ld=255), 1, "rows"),
    (dict(kv_ld=127), 1, "rows"), (dict(scale=float("nan")), 1, "rows"), (dict(pairs=33), 1, "rotation"), (dict(cos_t=0), 1, "rotation"), (dict(position=0), 1, "rotation"),
    (dict(positions=0), 1, "rotation"), (dict(weight_in=0x7000000), 1, "together"), (dict(weight_out=0x7000000), 1, "together"), (dict(workspace=0), 1, "workspace"),
    (dict(workspace=0x6000004), 1, "workspace"), (dict(workspace_bytes=16), 1, "workspace")])
def test_attention_refusals(lib, bad, tokens, why):
    assert why in refused(lib, lib.zen_cuda_dev_q4_attention(attention(**bad), 16, 16, 16, tokens, 16, None))


@pytest.mark.parametrize("missing", range(4))
def test_attention_refuses_missing_rows(lib, missing):
    rows = [16, 16, 16, 16]
    rows[missing] = None
    assert "rows" in refused(lib, lib.zen_cuda_dev_q4_attention(attention(), rows[0], rows[1], rows[2], 1, rows[3], None))


def test_eviction_refusals(lib):
    other = cache(k_codes=0x11000000, v_codes=0x12000000, k_scales=0x13000000, v_scales=0x14000000)
    call = lambda source=None, to=None, weight=0x8000000, filled=0x9000000, weight_to=0xa000000, keep=8, first=2, last=2, room=1 << 20: (   # noqa: E731
        lib.zen_cuda_dev_q4_cache_evict(source or cache(), weight, filled, to or other, weight_to, keep, first, last, None, 0xb000000, room, None))
    for bad in (dict(weight=None), dict(weight_to=None), dict(filled=None), dict(keep=0), dict(keep=97), dict(first=9), dict(first=5, last=4), dict(last=2 ** 64 - 1, first=2)):
        assert "bad arguments" in refused(lib, call(**bad))
    assert "workspace" in refused(lib, call(room=2 * 96 * 4 - 1))
    assert "bad arguments" in refused(lib, call(to=cache(kv_heads=1)))
    # the same codes under other weights, a cache that begins inside the other, weights inside a cache
    assert "neither the same nor apart" in refused(lib, call(to=cache()))
    assert "neither the same nor apart" in refused(lib, call(to=cache(k_codes=0x1000010, v_codes=0x12000000, k_scales=0x13000000, v_scales=0x14000000)))
    assert "neither the same nor apart" in refused(lib, call(weight_to=0x1000100))


def test_verify_refusals(lib):
    good = dict(logits=16, logits_ld=100, vocab=100, drafts=2, tokens=16, uniforms=16, temperature=1.0, top_k=0, top_p=1.0, out=16, accepted=16, workspace=16, workspace_bytes=1 << 20)
    assert lib.zen_cuda_verify_drafts_workspace_bytes(DraftCheck(**good)) > 0
    for bad in (dict(vocab=0), dict(vocab=262145, logits_ld=262145), dict(drafts=65)):
        assert lib.zen_cuda_verify_drafts_workspace_bytes(DraftCheck(**{**good, **bad})) == 0
        assert "bad arguments" in refused(lib, lib.zen_cuda_dev_verify_drafts(DraftCheck(**{**good, **bad}), None))
    for bad in (dict(logits=0), dict(logits_ld=99), dict(tokens=0), dict(uniforms=0), dict(out=0), dict(accepted=0), dict(q_ids=16), dict(q_ids=16, q_probs=16), dict(q_count=16)):
        assert "bad arguments" in refused(lib, lib.zen_cuda_dev_verify_drafts(DraftCheck(**{**good, **bad}), None))
    for bad in (dict(temperature=-0.1), dict(temperature=float("nan")), dict(temperature=float("inf")), dict(top_p=float("nan"))):
        assert "temperature" in refused(lib, lib.zen_cuda_dev_verify_drafts(DraftCheck(**{**good, **bad}), None))
    for bad in (dict(workspace=0), dict(workspace=8), dict(workspace_bytes=16)):
        assert "workspace" in refused(lib, lib.zen_cuda_dev_verify_drafts(DraftCheck(**{**good, **bad}), None))


def test_structures_have_the_headers_size(tmp_path):
    import os
    import subprocess
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    src = tmp_path / "t.c"
    src.write_text('#include <stdio.h>\n#include "zen_cuda.h"\nint main(void){printf("%zu %zu %zu", sizeof(zen_cuda_q4_cache), sizeof(zen_cuda_q4_attention), sizeof(zen_cuda_draft_check));return 0;}\n')
    subprocess.run(["gcc", "-std=c99", "-I", os.path.join(root, "include"), str(src), "-o", str(tmp_path / "t")], check=True)
    sizes = [int(n) for n in subprocess.run([str(tmp_path / "t")], check=True, capture_output=True).stdout.split()]
    assert sizes == [C.sizeof(Q4Cache), C.sizeof(Q4Attention), C.sizeof(DraftCheck)]


# ---- the plain implementations ----
def test_the_quantiser_is_that_of_q4_0_blocks_up_to_the_choice_at_borders():
    x = np.random.default_rng(0).standard_normal((40, 256)).astype(np.float32)
    d, c = q4.quantise(x)
    b = blocks.quantize_q4_0(x).reshape(40, 8, 18)
    assert np.array_equal(b[..., :2].copy().view(np.float16)[..., 0], d)
    theirs = np.concatenate([b[..., 2:] & 15, b[..., 2:] >> 4], -1).reshape(40, 256)
    assert (np.abs(theirs.astype(int) - c) <= 1).all() and (theirs != c).mean() < 2e-3      # x / d by the rounded scale, not by the one before rounding


def test_an_error_of_the_quantiser_is_at_most_half_a_step_within_the_codes_range():
    x = (np.random.default_rng(1).standard_normal((64, 64)) * 10.0 ** np.random.default_rng(2).uniform(-3, 3, (64, 1))).astype(np.float32)
    d, c = q4.quantise(x)
    step = np.abs(d.astype(np.float64)).repeat(32, -1)
    # 15 is 7 steps up: a value of the other sign than the largest may be 8 steps away, and f16 rounds d by 2^-11
    assert (np.abs(q4.held(x) - x) <= np.where((c == 15) | (c == 0), 1.0 + 2.0 ** -7, 0.5) * step + 1e-30).all()


def test_packing_is_the_documented_layout():
    codes = np.random.default_rng(3).integers(0, 16, (2, 24, 64), dtype=np.uint8)
    data = q4.pack(codes)
    assert data.shape == Q4Cache.codes_shape(2, 64, 24)
    for h, s, e in ((0, 0, 0), (1, 9, 17), (0, 23, 63), (1, 8, 33)):
        byte = data[h, s // 8, e // 32, s % 8, e % 16]
        assert (byte >> 4 if e % 32 >= 16 else byte & 15) == codes[h, s, e]
    assert np.array_equal(q4.unpack(data), codes)


def test_the_drawn_tokens_are_distributed_as_the_model_says():
    # the rule's point: whatever the draft's distribution, accepted or replaced, the token is distributed as p
    rng = np.random.default_rng(4)
    logits = rng.standard_normal((2, 6)).astype(np.float32)
    q = np.array([[0.5, 0.1, 0.2, 0.0, 0.2, 0.0]])
    p = q4.distribution(logits[0], 1.0, 0, 1.0)
    n = 20000
    seen = np.zeros(6)
    drafts = rng.choice(6, n, p=q[0])
    u = rng.random((n, 2))
    for t, uu in zip(drafts, u):
        seen[q4.verify(logits, [t], q, uu, 1.0, 0, 1.0)[0][0]] += 1
    assert np.abs(seen / n - p).max() < 5 * np.sqrt(0.25 / n)


# ---- the decoder's side that needs no device ----
def test_drafts_are_looked_up_at_the_last_place_that_reads_alike():
    from zeninfer_b200.llama import LlamaDecoder
    look = LlamaDecoder.look_up
    assert look(LlamaDecoder, [1, 2, 3, 9, 1, 2, 3], 2) == [9, 1]
    assert look(LlamaDecoder, [5, 2, 3, 7, 1, 2, 3, 8, 4, 2, 3], 3) == [8, 4, 2]      # two tokens alike, and the later place
    assert look(LlamaDecoder, [4, 4], 5) == [4] and look(LlamaDecoder, [1, 2, 3], 4) == [] and look(LlamaDecoder, [1], 4) == []


@pytest.mark.parametrize("argv", ["--kv-slots 64", "--kv-keep 8", "--kv q5", "--draft 65", "--draft -1"])
def test_the_command_refuses(argv, capsys):
    from zeninfer_b200.__main__ import main
    with pytest.raises(SystemExit) as e:
        main(["generate", "--model", "x", "--prompt-ids", "1"] + argv.split())
    assert e.value.code == 2


def test_options_of_other_models_are_refused(tmp_path):
    import json
    from zeninfer_b200 import registry
    (tmp_path / "config.json").write_text(json.dumps({"architecture": "Kipirax"}))
    with pytest.raises(ValueError, match="kv"):
        registry.load_model(None, str(tmp_path), kv="q4")


def test_the_plain_model_with_a_cache_reads_blocks_as_it_reads_tokens():
    from q4_llama import PlainLlama
    from zeninfer_b200.llama import LlamaConfig
    cfg = LlamaConfig(embedding=64, layers=2, heads=2, kv_heads=1, head_dim=32, ffn=64, vocab=50, rope_base=10000.0, context=32)
    a, b = PlainLlama(cfg, 1, 0.1, 32), PlainLlama(cfg, 1, 0.1, 32)
    tokens = [3, 1, 4, 1, 5, 9, 2, 6]
    whole = a.block(tokens, 0)
    rows = [b.block([t], i)[0] for i, t in enumerate(tokens)]
    assert np.abs(whole - rows).max() <= 1e-9 * np.abs(whole).max()
    assert np.abs(b.block(tokens[5:], 5) - whole[5:]).max() <= 1e-9 * np.abs(whole).max()       # taken back and read again


def test_an_index_of_the_context_drafts_what_looking_it_up_does():
    from zeninfer_b200.llama import ContextIndex, LlamaDecoder
    rng = np.random.default_rng(6)
    for vocab, longest in ((2, 3), (4, 3), (30, 3), (5, 1)):
        tokens, decoder = rng.integers(0, vocab, 300).tolist(), type("Decoder", (LlamaDecoder,), dict(LOOKUP=longest))
        index, at = ContextIndex(tokens[:1], longest), 1
        while at < len(tokens):
            for drafts in (1, 4):
                assert index.look_up(drafts) == LlamaDecoder.look_up(decoder, tokens[:at], drafts)
            n = int(rng.integers(1, 6))
            index.extend(tokens[at:at + n])
            at += n


def test_a_draft_from_the_index_reads_the_contexts_end_only():
    from zeninfer_b200.llama import ContextIndex

    class Counted(list):
        read = 0

        def __getitem__(self, at):
            part = list.__getitem__(self, at)
            Counted.read += len(part) if isinstance(at, slice) else 1
            return part

    index = ContextIndex([], 3)
    index.tokens = Counted()
    index.extend(range(20000))
    Counted.read = 0
    for t in range(50):
        index.extend([t % 7])
        index.look_up(4)
    assert Counted.read <= 50 * (6 + 6 + 4)      # three runs to remember, three to look for, a draft


def test_tensors_that_the_device_cannot_read_make_no_cache():
    import torch
    tensors = lambda device: [torch.empty(shape(2, 64, 32), dtype=dtype, device=device)   # noqa: E731
                              for shape, dtype in ((Q4Cache.codes_shape, torch.uint8), (Q4Cache.scales_shape, torch.float16)) * 2]
    for device in ("cpu", "meta"):
        with pytest.raises(ValueError, match=device):
            Q4Cache.of(*tensors(device), kv_heads=2, head_dim=64, slots=32)
    with pytest.raises(ValueError, match="v_codes does not hold"):
        Q4Cache.of(*tensors("cpu")[:2], torch.empty(7, dtype=torch.uint8), torch.empty(7, dtype=torch.float16), kv_heads=2, head_dim=64, slots=32)


def test_a_call_whose_last_launch_does_not_fit_a_grid_is_refused_before_the_first(lib):
    """Many rows of heads of 96 with weights: 256 slots a CTA along a grid's second axis."""
    bytes_of = lambda slots, tokens, **more: lib.zen_cuda_q4_attention_workspace_bytes(attention(cache(head_dim=96, slots=slots), pairs=48, **more), tokens)   # noqa: E731
    weights = dict(weight_in=0x7000000, weight_out=0x7000000)
    most = 65535 * 256
    assert bytes_of(most, 40, **weights) > 0 and bytes_of(most + 32, 40, **weights) == 0
    assert bytes_of(most + 32, 40) > 0 and bytes_of(most + 32, 16, **weights) > 0        # no weights, or few rows
    big = attention(cache(head_dim=96, slots=most + 32), pairs=48, **weights)
    assert "bad arguments" in refused(lib, lib.zen_cuda_dev_q4_attention(big, 16, 16, 16, 40, 16, None))
