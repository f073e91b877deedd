"""A dense Llama-style model in 64 bits whose keys and values go through the 4-bit cache, for the tests of the decoder that holds them so."""
from __future__ import annotations

import numpy as np

import q4_cases as q4
from zeninfer_b200 import blocks
from zeninfer_b200.llama import LlamaConfig, rope_tables, synthetic_tensors


class PlainLlama:
    """block(tokens, position): their logits [tokens, vocab].  With keep, slots are dropped as LlamaDecoder documents; quantised False: the cache is exact; position behind
    the last one: tokens are taken back.

    cache(layer) -> keys and values [kv_heads, slots in use, head_dim] after the block, as a decoder holds them: they are then what the model attends to, once it is seen that the
    new ones are roundings of the model's own, and the older ones those that were there, less the dropped ones."""

    def __init__(self, cfg: LlamaConfig, seed: int, weight_std: float, slots: int, keep: int | None = None, first: int = 4, last: int = 0, quantised: bool = True) -> None:
        self.cfg, self.slots, self.keep, self.first, self.last, self.quantised = cfg, slots, keep, first, last, quantised
        self.t = {}
        for name, a, is_matrix in synthetic_tensors(cfg, seed, weight_std):
            columns = cfg.q_width if name.endswith("attn_output.weight") else cfg.ffn if name.endswith("ffn_down.weight") else cfg.embedding
            self.t[name] = blocks.dequantize(blocks.Q8_0, a, a.shape[0], columns).astype(np.float64) if is_matrix else a.astype(np.float64)
        self.cos, self.sin = (x.astype(np.float32) for x in rope_tables(cfg, cfg.context))
        empty = lambda: np.zeros((cfg.kv_heads, 0, cfg.head_dim))
        self.k, self.v = [empty() for _ in range(cfg.layers)], [empty() for _ in range(cfg.layers)]
        self.w = [np.zeros((cfg.kv_heads, 0)) for _ in range(cfg.layers)]
        self.place = self.drops = 0

    def norm(self, x, name):
        return x / np.sqrt((x * x).mean(-1, keepdims=True) + self.cfg.rms_eps) * self.t[name]

    @staticmethod
    def rounded(x: np.ndarray, held: np.ndarray) -> None:
        """held is x [tokens, heads, D] on a grid of sixteen steps of a 32nd-block's scale: off by half a step, by one where the grid ends one short, and 1 % of
        a step for x itself, whose products are within 5e-5 of the largest value, 8 steps."""
        b, h = x.reshape(*x.shape[:-1], -1, 32).astype(np.float64), held.reshape(*x.shape[:-1], -1, 32)
        step = np.abs(b).max(-1, keepdims=True) / 8 * (1 + 2.0 ** -10)
        off = np.abs(b - h)
        assert (off <= 1.01 * step).all() and ((off <= 0.51 * step) | (np.abs(h) >= 6.98 * step / (1 + 2.0 ** -9))).all()

    def block(self, tokens: list[int], position: int, cache=None) -> np.ndarray:
        cfg, n = self.cfg, len(tokens)
        back = self.place - position
        held = self.k[0].shape[1] - back
        for layer in range(cfg.layers):
            self.k[layer], self.v[layer], self.w[layer] = self.k[layer][:, :held], self.v[layer][:, :held], self.w[layer][:, :held]
        if held + n > self.slots:
            for layer in range(cfg.layers):
                stay = q4.kept_slots(self.w[layer], held, self.keep, self.first, self.last)
                pick = lambda a: np.stack([a[h, stay[h]] for h in range(cfg.kv_heads)])
                self.k[layer], self.v[layer], self.w[layer] = pick(self.k[layer]), pick(self.v[layer]), pick(self.w[layer])
            held = self.k[0].shape[1]
            self.drops += 1
        self.place = position + n
        rows = slice(position, position + n)
        x = self.t["token_embd.weight"][tokens]
        hold = q4.held if self.quantised else lambda a: a.astype(np.float64)
        for layer in range(cfg.layers):
            g = lambda name: self.t[f"blk.{layer}.{name}.weight"]
            y = self.norm(x, f"blk.{layer}.attn_norm.weight")
            project = lambda name, heads: (y @ g(name).T).astype(np.float32).reshape(n, heads, cfg.head_dim)
            q = q4.rotate(project("attn_q", cfg.heads), self.cos[rows], self.sin[rows], True)
            k = q4.rotate(project("attn_k", cfg.kv_heads), self.cos[rows], self.sin[rows], True)
            v = project("attn_v", cfg.kv_heads)
            if cache is None:
                self.k[layer] = np.concatenate([self.k[layer], hold(k).transpose(1, 0, 2)], 1)
                self.v[layer] = np.concatenate([self.v[layer], hold(v).transpose(1, 0, 2)], 1)
            else:
                before, (self.k[layer], self.v[layer]) = (self.k[layer], self.v[layer]), cache(layer)
                for old, now, new in zip(before, (self.k[layer], self.v[layer]), (k, v)):
                    assert now.shape[1] == held + n and np.array_equal(now[:, :held], old)
                    self.rounded(new, now[:, held:].transpose(1, 0, 2))
            out, received = q4.attention(q, self.k[layer], self.v[layer], held, cfg.head_dim ** -0.5)
            received[:, :held] += self.w[layer]
            self.w[layer] = received
            x = x + out.reshape(n, -1) @ g("attn_output").T
            y = self.norm(x, f"blk.{layer}.ffn_norm.weight")
            gate = y @ g("ffn_gate").T
            x = x + (gate / (1 + np.exp(-gate)) * (y @ g("ffn_up").T)) @ g("ffn_down").T
        return self.norm(x, "output_norm.weight") @ self.t["output.weight"].T
