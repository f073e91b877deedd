"""Operators of decoding over a small cache and of drafted tokens, as cases that can be timed and compared.

Three operators, each in a plain form (elementary torch operations) and as a user of this package calls it:

  attention  new tokens of a sequence against a cache held in 4 bits: rotation of q and k, the new keys and values quantised and
             appended, grouped-query attention over everything cached, and the attention weight each slot received added up
             (zen_cuda_dev_q4_attention).  One token is a decode step, a few are a block of drafted tokens to verify, many a prompt.
  evict      the slots of a cache that received the least attention weight are dropped, per key/value head; the first and the last
             slots stay, what is kept closes up in its order (zen_cuda_dev_q4_cache_evict).
  verify     drafted tokens against the target model's filtered distributions, with given uniform numbers: how many are accepted,
             and the token that follows them (zen_cuda_dev_verify_drafts).

The cache's form is that of Q4_0 blocks: 32 consecutive values of a head share an f16 scale d and have codes 0 .. 15, value = d (code - 8).
Codes [kv_heads][slots / 8][head_dim / 32][8][16 bytes], byte i of 16 holding values i (low) and i + 16 (high) of the block; scales
[kv_heads][slots][head_dim / 32].
"""
import math

import numpy as np
import torch

own = False

DEV = "cuda"
CANDIDATES = 1024        # entries of a draft's kept list, as the sampler leaves it


# ---- the cases ---------------------------------------------------------------------------------------------------------

def _attention(tokens, filled, heads, kv_heads, dim, weights, **more):
    return dict(kind="attention", tokens=tokens, filled=filled, heads=heads, kv_heads=kv_heads, dim=dim, weights=weights, **more)


def _evict(filled, keep, first, last, kv_heads, dim, **more):
    return dict(kind="evict", filled=filled, keep=keep, first=first, last=last, kv_heads=kv_heads, dim=dim, **more)


def _verify(drafts, vocab, listed_q, temperature, top_k, top_p, **more):
    return dict(kind="verify", drafts=drafts, vocab=vocab, listed_q=listed_q, temperature=temperature, top_k=top_k, top_p=top_p, **more)


def listed():
    return [
        # the first tokens of an answer by a small model: latency
        _attention(1, 19, 4, 2, 64, False, name="step of a small model"),
        # a token of an 8B model in an ordinary conversation, with the weights an eviction will ask for
        _attention(1, 1000, 32, 8, 128, True, name="step, 1000 slots"),
        # a token behind a long document
        _attention(1, 65501, 32, 8, 128, False, name="step, 65501 slots"),
        # a block of drafted tokens and the one before them
        _attention(5, 4003, 32, 8, 128, False, name="5 tokens, 4003 slots"),
        # a prompt's first block, and a later one of a long prompt whose weights are kept
        _attention(512, 0, 32, 8, 128, False, name="512 tokens from the start"),
        _attention(512, 7680, 32, 8, 128, True, name="512 tokens, 7680 slots"),
        # a ragged prompt of a model without grouped heads
        _attention(333, 77, 16, 16, 64, True, name="333 tokens, heads of 64"),
        # a conversation's cache brought back to its budget, and a long prompt's to a small one
        _evict(1100, 1024, 4, 64, 8, 128, name="evict 76 of 1100"),
        _evict(65501, 8192, 4, 512, 8, 128, name="evict 57309 of 65501"),
        # two tokens looked up in the prompt, accepted by a small vocabulary's distribution
        _verify(2, 32000, False, 1.0, 0, 1.0, name="verify 2 of 32000"),
        # eight tokens of a draft model, nucleus sampling
        _verify(8, 128256, True, 0.8, 0, 0.95, name="verify 8 of 128256, top-p"),
        # four looked-up tokens, the usual filters
        _verify(4, 128256, False, 0.7, 40, 0.9, name="verify 4 of 128256, top-k"),
    ]


def _spread(rng, low, high):
    """A size from low to high, even over its logarithm."""
    return min(max(int(round(math.exp(rng.uniform(math.log(low), math.log(high))))), low), high)


def draw(rng):
    kind = rng.choice(("step", "step", "block", "prompt", "evict", "verify"))
    heads, kv_heads, dim = rng.choice(((4, 2, 64), (32, 8, 128), (16, 16, 64), (12, 4, 96), (8, 1, 128), (16, 4, 256), (28, 4, 128)))
    if kind == "step":
        return _attention(1, _spread(rng, 2, 65500), heads, kv_heads, dim, rng.random() < 0.5)
    if kind == "block":
        return _attention(rng.randint(2, 17), _spread(rng, 2, 20000), heads, kv_heads, dim, rng.random() < 0.3)
    if kind == "prompt":
        tokens = _spread(rng, 18, 512)
        return _attention(tokens, rng.choice((0, _spread(rng, 1, 4000))), heads, kv_heads, dim, rng.random() < 0.5)
    if kind == "evict":
        filled = _spread(rng, 64, 65000)
        keep = max(1, int(filled * rng.uniform(0.05, 0.99)))
        return _evict(filled, keep, min(4, keep // 4), keep // rng.choice((2, 8, 32)), kv_heads, dim)
    return _verify(rng.randint(1, 8), rng.choice((512, 16384, 32000, 50257, 128256)), rng.random() < 0.5, rng.choice((0.0, 0.6, 1.0, 1.3)),
                   rng.choice((0, 0, 5, 40, 2000)), rng.choice((1.0, 0.95, 0.8)))


# ---- inputs ------------------------------------------------------------------------------------------------------------

class State:
    """What a user's program has in hand, and (own) the call's handle, made at its first use."""

    def __init__(self, **fields):
        self.handle = None
        self.__dict__.update(fields)


def _round_up(n, m):
    return (n + m - 1) // m * m


def _generator(seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed * 7919 + 17)
    return g


def _scale_and_codes(x):
    """x [..., 32] fp32 -> the block's f16 scale [..., 1] and codes [..., 32]: d = (the first value of largest magnitude) / -8 to f16
    (at most 65504 in magnitude), the code nearest to x / d + 8, halves upwards, within 0 .. 15.  In 64 bits: x / d is next to a border."""
    size = x.abs()
    at = torch.where(size == size.amax(-1, keepdim=True), torch.arange(32, device=x.device), 32).amin(-1, keepdim=True)
    d = (torch.gather(x, -1, at) / -8.0).clamp(-65504.0, 65504.0).to(torch.float16)
    ratio = x.double() / torch.where(d == 0, torch.ones_like(d), d).double()
    codes = torch.where(d == 0, torch.full_like(ratio, 8.0), torch.floor(ratio + 8.5).clamp(0.0, 15.0))
    return d, codes


def _pack(codes):
    """codes [kv_heads, slots, blocks, 32] -> bytes [kv_heads, slots / 8, blocks, 8, 16]."""
    c = codes.to(torch.uint8)
    h, s, b, _ = c.shape
    return (c[..., :16] | (c[..., 16:] << 4)).view(h, s // 8, 8, b, 16).transpose(2, 3).contiguous()


def _made_cache(g, kv_heads, slots, dim, outliers):
    """A cache as a model leaves it: normal values, some channels of the keys several times larger than the others."""
    blocks = dim // 32
    channel = torch.ones((kv_heads, 1, dim), device=DEV)
    if outliers:
        channel += 5.0 * (torch.rand((kv_heads, 1, dim), generator=g, device=DEV) < 0.05)
    codes = torch.empty((kv_heads, slots // 8, blocks, 8, 16), dtype=torch.uint8, device=DEV)
    scales = torch.empty((kv_heads, slots, blocks), dtype=torch.float16, device=DEV)
    for head in range(kv_heads):      # a head at a time: the values are eight times the cache
        x = torch.randn((1, slots, dim), generator=g, device=DEV) * channel[head:head + 1]
        d, c = _scale_and_codes(x.view(1, slots, blocks, 32))
        codes[head:head + 1] = _pack(c)
        scales[head:head + 1] = d[..., 0]
    return codes, scales


def _cache(g, kv_heads, slots, dim):
    k, v = _made_cache(g, kv_heads, slots, dim, True), _made_cache(g, kv_heads, slots, dim, False)
    return dict(k_codes=k[0], k_scales=k[1], v_codes=v[0], v_scales=v[1], kv_heads=kv_heads, dim=dim, slots=slots)


def _prepare_attention(case, g):
    tokens, filled, heads, kv_heads, dim = (case[n] for n in ("tokens", "filled", "heads", "kv_heads", "dim"))
    slots = _round_up(filled + tokens, 32)
    row = lambda n: torch.randn((tokens, n * dim), generator=g, device=DEV)   # noqa: E731
    position = filled + 13          # a cache that has been evicted from holds fewer slots than the sequence has had positions
    angle = (torch.arange(position + tokens, device=DEV, dtype=torch.float64)[:, None] *
             500000.0 ** (-torch.arange(dim // 2, device=DEV, dtype=torch.float64) * 2.0 / dim)[None, :])
    cells = torch.rand((kv_heads, slots), generator=g, device=DEV) * 0.3 if case["weights"] else None
    return State(case=case, cache=_cache(g, kv_heads, slots, dim), q=row(heads) * 1.5, k=row(kv_heads), v=row(kv_heads), cos=angle.cos().float(), sin=angle.sin().float(),
                 position=torch.tensor([position], dtype=torch.int32, device=DEV), filled=torch.tensor([filled], dtype=torch.int32, device=DEV),
                 weight_in=cells, weight_out=None if cells is None else torch.zeros_like(cells), out=torch.zeros((tokens, heads * dim), device=DEV),
                 k_held=torch.zeros((tokens, kv_heads * dim), device=DEV), v_held=torch.zeros((tokens, kv_heads * dim), device=DEV))


def _prepare_evict(case, g):
    kv_heads, dim, filled, keep = (case[n] for n in ("kv_heads", "dim", "filled", "keep"))
    slots, room = _round_up(filled, 32), _round_up(keep, 32)
    blocks = dim // 32

    def cache(n, full):
        made = dict(kv_heads=kv_heads, dim=dim, slots=n)
        for side in "kv":
            shape = (kv_heads, n // 8, blocks, 8, 16)
            made[side + "_codes"] = torch.randint(0, 256, shape, generator=g, device=DEV, dtype=torch.uint8) if full else torch.zeros(shape, device=DEV, dtype=torch.uint8)
            made[side + "_scales"] = (torch.rand((kv_heads, n, blocks), generator=g, device=DEV) * 0.3 if full else torch.zeros((kv_heads, n, blocks), device=DEV)).half()
        return made
    # most slots received little, a few nearly everything; equal weights happen
    weight = torch.exp(2.0 * torch.randn((kv_heads, slots), generator=g, device=DEV)) * 1e-2
    weight = torch.where(torch.rand((kv_heads, slots), generator=g, device=DEV) < 0.05, torch.full_like(weight, 1e-3), weight)
    return State(case=case, cache=cache(slots, True), to=cache(room, False), weight=weight, weight_to=torch.zeros((kv_heads, room), device=DEV),
                 kept=torch.zeros((kv_heads, keep), dtype=torch.int32, device=DEV), filled=torch.tensor([filled], dtype=torch.int32, device=DEV))


def _prepare_verify(case, g):
    drafts, vocab, temperature = case["drafts"], case["vocab"], case["temperature"]
    logits = torch.randn((drafts + 1, vocab), generator=g, device=DEV) * 2.0
    likely = torch.randint(0, vocab, (drafts + 1, 24), generator=g, device=DEV)
    logits.scatter_add_(1, likely, 4.0 + 8.0 * torch.rand((drafts + 1, 24), generator=g, device=DEV))
    uniforms = torch.rand((drafts + 1,), generator=g, device=DEV, dtype=torch.float64)
    q_ids = q_probs = q_count = None
    if case["listed_q"]:
        # a draft model that mostly agrees, its distribution cut to its most likely tokens, as the sampler's kept list
        kept = min(CANDIDATES, vocab // 2)
        drafted = logits[:drafts] + 0.5 * torch.randn((drafts, vocab), generator=g, device=DEV)
        ids = drafted.topk(kept, dim=1).indices.sort(1).values
        q_ids = torch.zeros((drafts, CANDIDATES), dtype=torch.int32, device=DEV)
        q_probs = torch.zeros((drafts, CANDIDATES), dtype=torch.float64, device=DEV)
        q_ids[:, :kept] = ids.int()
        q_probs[:, :kept] = torch.softmax(drafted.gather(1, ids).double() / (temperature or 1.0), 1)
        q_count = torch.full((drafts,), kept, dtype=torch.int32, device=DEV)
        tokens = ids.gather(1, torch.multinomial(q_probs[:, :kept].float(), 1, generator=g))[:, 0]
    else:
        tokens = torch.where(torch.rand((drafts,), generator=g, device=DEV) < 0.8, logits[:drafts].argmax(1), torch.randint(0, vocab, (drafts,), generator=g, device=DEV))
    return State(case=case, logits=logits, tokens=tokens.contiguous(), uniforms=uniforms, q_ids=q_ids, q_probs=q_probs, q_count=q_count,
                 out=torch.zeros((drafts + 1,), dtype=torch.int64, device=DEV), accepted=torch.zeros((1,), dtype=torch.int32, device=DEV),
                 probs=torch.zeros((drafts,), dtype=torch.float64, device=DEV))


def prepare(case, seed):
    return {"attention": _prepare_attention, "evict": _prepare_evict, "verify": _prepare_verify}[case["kind"]](case, _generator(seed))


# ---- the plain forms ---------------------------------------------------------------------------------------------------

def _values(codes, scales, n):
    """The first n slots' values [kv_heads, n, dim] in fp32."""
    h, _, blocks, _, _ = codes.shape
    c = codes[:, :_round_up(n, 8) // 8].transpose(2, 3)
    c = torch.cat((c & 15, c >> 4), -1).reshape(h, -1, blocks, 32)[:, :n]
    return ((c.float() - 8.0) * scales[:, :n, :, None].float()).view(h, n, blocks * 32)


def _turned(x, cos, sin):
    """Adjacent pairs of x [tokens, heads, dim] turned, every product and sum rounded on its own."""
    a, b = x[..., 0::2], x[..., 1::2]
    c, s = cos[:, None, :], sin[:, None, :]
    return torch.stack((a * c - b * s, a * s + b * c), -1).flatten(-2)


def _plain_append(codes, scales, held, x, filled):
    """x [tokens, kv_heads, dim] into slots filled .. of the cache; `held`: what the cache now holds of it."""
    tokens, kv_heads, dim = x.shape
    d, c = _scale_and_codes(x.view(tokens, kv_heads, dim // 32, 32))
    packed = c.to(torch.uint8)
    packed = (packed[..., :16] | (packed[..., 16:] << 4)).transpose(0, 1)           # [kv_heads, tokens, blocks, 16]
    slot = filled + torch.arange(tokens, device=x.device)
    codes[:, slot // 8, :, slot % 8] = packed.transpose(0, 1)
    scales[:, slot] = d[..., 0].transpose(0, 1)
    held.copy_(((c.float() - 8.0) * d.float()).reshape(tokens, -1))


def _plain_attention(s):
    case, cache = s.case, s.cache
    tokens, filled, heads, kv_heads, dim = (case[n] for n in ("tokens", "filled", "heads", "kv_heads", "dim"))
    total, group = filled + tokens, heads // kv_heads
    rows = s.position.long() + torch.arange(tokens, device=DEV)
    cos, sin = s.cos[rows], s.sin[rows]
    q = _turned(s.q.view(tokens, heads, dim), cos, sin)
    _plain_append(cache["k_codes"], cache["k_scales"], s.k_held, _turned(s.k.view(tokens, kv_heads, dim), cos, sin), filled)
    _plain_append(cache["v_codes"], cache["v_scales"], s.v_held, s.v.view(tokens, kv_heads, dim), filled)
    k, v = _values(cache["k_codes"], cache["k_scales"], total), _values(cache["v_codes"], cache["v_scales"], total)
    q = q.view(tokens, kv_heads, group, dim).permute(1, 2, 0, 3).reshape(kv_heads, group * tokens, dim)
    scores = (q @ k.transpose(1, 2)).view(kv_heads, group, tokens, total) * (1.0 / math.sqrt(dim))
    if tokens > 1:
        slot, token = torch.arange(total, device=DEV), torch.arange(tokens, device=DEV)
        scores = scores.masked_fill(slot[None, :] > filled + token[:, None], -math.inf)
    p = torch.exp(scores - scores.amax(-1, keepdim=True))
    p = p / p.sum(-1, keepdim=True)
    s.out.copy_((p.view(kv_heads, group * tokens, total) @ v).view(kv_heads, group, tokens, dim).permute(2, 0, 1, 3).reshape(tokens, heads * dim))
    if s.weight_in is not None:
        received = p.sum((1, 2))
        received[:, :filled] += s.weight_in[:, :filled]
        s.weight_out[:, :total] = received
    return _attention_outputs(s)


def _attention_outputs(s):
    """The rows, the new tokens as the cache now holds them, and the weights."""
    return [s.out, s.k_held, s.v_held] + ([s.weight_out] if s.weight_out is not None else [])


def _evict_outputs(s):
    return [s.kept, s.weight_to, s.to["k_codes"], s.to["k_scales"], s.to["v_codes"], s.to["v_scales"]]


def _plain_evict(s):
    case, cache, to = s.case, s.cache, s.to
    filled, keep, first, last = (case[n] for n in ("filled", "keep", "first", "last"))
    rank = s.weight[:, :filled].clone()
    rank[:, :first] = math.inf
    rank[:, filled - last:] = math.inf
    order = torch.sort(rank, dim=1, descending=True, stable=True).indices[:, :keep]      # equal weights: the lowest slots
    kept = order.sort(1).values                                                          # [kv_heads, keep]
    s.kept.copy_(kept)
    s.weight_to[:, :keep] = s.weight.gather(1, kept)
    head = torch.arange(case["kv_heads"], device=DEV)[:, None]
    slot = torch.arange(keep, device=DEV)
    for side in "kv":
        to[side + "_codes"][head, slot[None] // 8, :, slot[None] % 8] = cache[side + "_codes"][head, kept // 8, :, kept % 8]
        to[side + "_scales"][:, :keep] = cache[side + "_scales"][head, kept]
    return _evict_outputs(s)


def _filtered(logits, temperature, top_k, top_p):
    """The distributions [rows, vocab] in 64 bits, in order of id: the top_k most likely, of them the shortest run that reaches top_p."""
    if temperature == 0.0:
        temperature, top_k, top_p = 1.0, 1, 1.0
    value, order = torch.sort(logits.double() + 0.0, dim=1, descending=True, stable=True)
    e = torch.exp((value - value[:, :1]) / temperature)
    if top_k:
        e[:, top_k:] = 0.0
    if 0.0 < top_p < 1.0:
        share = torch.cumsum(e, 1) / e.sum(1, keepdim=True)
        e[:, 1:] = torch.where(share[:, :-1] < top_p, e[:, 1:], torch.zeros_like(e[:, 1:]))
    e = e / e.sum(1, keepdim=True)
    return torch.zeros_like(e).scatter_(1, order, e)


def _plain_verify(s):
    case = s.case
    drafts, vocab = case["drafts"], case["vocab"]
    temperature = float(np.float32(case["temperature"]))
    p = _filtered(s.logits, temperature, case["top_k"], float(np.float32(case["top_p"])))
    q = torch.zeros((drafts + 1, vocab), dtype=torch.float64, device=DEV)      # nothing is taken off behind the last draft
    if s.q_ids is not None:
        listed_entry = torch.arange(CANDIDATES, device=DEV)[None, :] < s.q_count[:, None]
        q[:drafts].scatter_add_(1, s.q_ids.long(), torch.where(listed_entry, s.q_probs, torch.zeros_like(s.q_probs)))
    else:
        q[:drafts].scatter_(1, s.tokens[:, None], 1.0)
    s.probs.copy_(p[:drafts].gather(1, s.tokens[:, None])[:, 0])
    fits = s.uniforms[:drafts] * q[:drafts].gather(1, s.tokens[:, None])[:, 0] < s.probs
    accepted = torch.cumprod(fits.long(), 0).sum().view(1)
    row = p.index_select(0, accepted)[0]
    rest = (row - q.index_select(0, accepted)[0]).clamp_min(0.0)
    rest = torch.where(rest.sum() > 0.0, rest, row)
    reached = torch.cumsum(rest, 0)
    drawn = ((reached >= s.uniforms[drafts] * reached[-1]) & (rest > 0.0)).long().argmax()
    place = torch.arange(drafts + 1, device=DEV)
    tokens = torch.cat((s.tokens, s.tokens.new_full((1,), -1)))
    s.out.copy_(torch.where(place < accepted, tokens, torch.where(place == accepted, drawn, torch.full_like(tokens, -1))))
    s.accepted.copy_(accepted)
    return [s.out, s.accepted, s.probs]


# ---- the framework's calls -----------------------------------------------------------------------------------------------

_BACKEND = []


def _backend():
    if not _BACKEND:
        from zeninfer_b200 import Backend
        _BACKEND.append(Backend())
    return _BACKEND[0]


def _stream():
    return torch.cuda.current_stream().cuda_stream or 1      # 1: the legacy default stream, which 0 does not name in this package


def _own_cache(c):
    from zeninfer_b200.backend import Q4Cache
    return Q4Cache.of(c["k_codes"], c["k_scales"], c["v_codes"], c["v_scales"], kv_heads=c["kv_heads"], head_dim=c["dim"], slots=c["slots"])


def _own_attention(s):
    be = _backend()
    if s.handle is None:
        from zeninfer_b200.backend import Q4Attention
        ptr = lambda t: None if t is None else t.data_ptr()   # noqa: E731
        a = Q4Attention(cache=_own_cache(s.cache), heads=s.case["heads"], cos_t=ptr(s.cos), sin_t=ptr(s.sin), pairs=s.cos.shape[1], positions=s.cos.shape[0], adjacent=1,
                        position=ptr(s.position), filled=ptr(s.filled), weight_in=ptr(s.weight_in), weight_out=ptr(s.weight_out), k_held=ptr(s.k_held), v_held=ptr(s.v_held))
        room = torch.zeros(be.q4_attention_workspace_bytes(a, s.case["tokens"]), dtype=torch.uint8, device=DEV)
        a.workspace, a.workspace_bytes = ptr(room), room.numel()
        s.handle = (a, room)
    be.dev_q4_attention(s.handle[0], s.q.data_ptr(), s.k.data_ptr(), s.v.data_ptr(), s.case["tokens"], s.out.data_ptr(), _stream())
    return _attention_outputs(s)


def _own_evict(s):
    be = _backend()
    if s.handle is None:
        caches = _own_cache(s.cache), _own_cache(s.to)
        s.handle = (*caches, torch.zeros(be.q4_cache_evict_workspace_bytes(caches[0]), dtype=torch.uint8, device=DEV))
    case, (source, to, room) = s.case, s.handle
    be.dev_q4_cache_evict(source, s.weight.data_ptr(), s.filled.data_ptr(), to, s.weight_to.data_ptr(), case["keep"], case["first"], case["last"], room.data_ptr(), room.numel(), _stream(),
                          d_kept=s.kept.data_ptr())
    return _evict_outputs(s)


def _own_verify(s):
    be = _backend()
    if s.handle is None:
        from zeninfer_b200.backend import DraftCheck
        ptr = lambda t: None if t is None else t.data_ptr()   # noqa: E731
        c = s.case
        s.handle = DraftCheck(logits=ptr(s.logits), logits_ld=c["vocab"], vocab=c["vocab"], drafts=c["drafts"], tokens=ptr(s.tokens), q_ids=ptr(s.q_ids), q_probs=ptr(s.q_probs),
                              q_count=ptr(s.q_count), uniforms=ptr(s.uniforms), temperature=c["temperature"], top_k=c["top_k"], top_p=c["top_p"], out=ptr(s.out), accepted=ptr(s.accepted),
                              probs=ptr(s.probs))
        room = torch.zeros(be.verify_drafts_workspace_bytes(s.handle), dtype=torch.uint8, device=DEV)
        s.handle.workspace, s.handle.workspace_bytes, s.room = ptr(room), room.numel(), room
    be.dev_verify_drafts(s.handle, _stream())
    return [s.out, s.accepted, s.probs]


def run(state):
    kind = state.case["kind"]
    if own:
        return {"attention": _own_attention, "evict": _own_evict, "verify": _own_verify}[kind](state)
    return {"attention": _plain_attention, "evict": _plain_evict, "verify": _plain_verify}[kind](state)


# ---- what a pass cannot do without -----------------------------------------------------------------------------------------

def work(case):
    if case["kind"] == "attention":
        tokens, filled, heads, kv_heads, dim = (case[n] for n in ("tokens", "filled", "heads", "kv_heads", "dim"))
        slot = kv_heads * 2 * (dim // 2 + dim // 16)                       # codes and scales of a slot, keys and values
        rows = tokens * 4 * (2 * heads * dim + 4 * kv_heads * dim)         # q and out, k, v and what is held of them
        weights = 4 * kv_heads * (2 * filled + tokens) if case["weights"] else 0
        seen = tokens * filled + tokens * (tokens + 1) // 2
        return {"bytes": (filled + 2 * tokens) * slot + rows + weights, "flops": 4 * heads * dim * seen}
    if case["kind"] == "evict":
        kv_heads, dim, filled, keep = (case[n] for n in ("kv_heads", "dim", "filled", "keep"))
        slot = 2 * (dim // 2 + dim // 16)
        return {"bytes": kv_heads * (4 * filled + 2 * keep * slot + keep * (4 + 4)), "flops": 0}
    drafts, vocab = case["drafts"], case["vocab"]
    lists = drafts * CANDIDATES * 12 if case["listed_q"] else 0
    return {"bytes": 4 * (drafts + 1) * vocab + lists + 32 * (drafts + 1), "flops": (drafts + 1) * vocab}


# ---- the definition in 64 bits ---------------------------------------------------------------------------------------------

def _exact_rows(x, cos=None, sin=None):
    """numpy [tokens, heads, dim] -> the values a 4-bit cache holds of it, in 64 bits, rotated first where tables are given (in 32 bits,
    as the definition has it: a code is chosen for the rounded key)."""
    if cos is not None:
        turned = np.empty_like(x)
        turned[..., 0::2] = x[..., 0::2] * cos[:, None] - x[..., 1::2] * sin[:, None]
        turned[..., 1::2] = x[..., 0::2] * sin[:, None] + x[..., 1::2] * cos[:, None]
        x = turned
    blocks = x.reshape(*x.shape[:-1], -1, 32).astype(np.float64)
    top = np.take_along_axis(blocks, np.abs(blocks).argmax(-1)[..., None], -1)          # numpy: the first of the largest
    d = np.clip(top / -8.0, -65504.0, 65504.0).astype(np.float32).astype(np.float16).astype(np.float64)
    with np.errstate(divide="ignore", invalid="ignore"):
        code = np.where(d == 0.0, 8.0, np.clip(np.floor(blocks / d + 8.5), 0.0, 15.0))
    return x, ((code - 8.0) * d).reshape(x.shape)


def _exact_verify(case, seed):
    s = prepare(case, seed)
    logits, tokens = s.logits.cpu().numpy().astype(np.float64), s.tokens.cpu().numpy()
    top_p, found = float(np.float32(case["top_p"])), []
    for row, token in zip(logits, tokens):
        order = np.lexsort((np.arange(row.size), -row))          # by value, then by id
        if case["temperature"] == 0.0:
            found.append(float(order[0] == token))
            continue
        order = order[:case["top_k"] or row.size]
        mass = np.exp((row[order] - row[order[0]]) / float(np.float32(case["temperature"]))).astype(np.longdouble)
        mass /= mass.sum()
        if 0.0 < top_p < 1.0:
            run_length = int(np.searchsorted(np.cumsum(mass), top_p)) + 1
            order, mass = order[:run_length], mass[:run_length] / mass[:run_length].sum()
        found.append(float(mass[order == token].sum()))
    return [None, None, torch.tensor(found, dtype=torch.float64)]


def exact(case, seed):
    if case["kind"] == "evict":
        return None                                       # whole numbers and bytes that are moved
    if case["kind"] == "verify":
        return _exact_verify(case, seed)
    s = prepare(case, seed)
    tokens, filled, heads, kv_heads, dim = (case[n] for n in ("tokens", "filled", "heads", "kv_heads", "dim"))
    first = int(s.position[0])
    cos, sin = s.cos[first:first + tokens].cpu().numpy(), s.sin[first:first + tokens].cpu().numpy()
    q, _ = _exact_rows(s.q.cpu().numpy().reshape(tokens, heads, dim), cos, sin)
    k_new = _exact_rows(s.k.cpu().numpy().reshape(tokens, kv_heads, dim), cos, sin)[1]
    v_new = _exact_rows(s.v.cpu().numpy().reshape(tokens, kv_heads, dim))[1]
    out = torch.empty((tokens, heads, dim), dtype=torch.float64, device=DEV)
    weights = None if s.weight_in is None else torch.zeros(s.weight_in.shape, dtype=torch.float64, device=DEV)
    per, future = heads // kv_heads, torch.arange(filled + tokens, device=DEV)[None, :] > filled + torch.arange(tokens, device=DEV)[:, None]
    for h in range(kv_heads):
        def whole(side, new):
            low = s.cache[side + "_codes"][h].permute(0, 2, 1, 3).reshape(-1, dim // 32, 16)[:filled]
            nibbles = torch.stack((low % 16, low // 16), 2).reshape(filled, dim // 32, 32).double() - 8.0
            old = (nibbles * s.cache[side + "_scales"][h, :filled].double()[..., None]).reshape(filled, dim)
            return torch.cat((old, torch.from_numpy(np.ascontiguousarray(new[:, h])).to(DEV)))
        keys, values = whole("k", k_new), whole("v", v_new)
        for j in range(h * per, (h + 1) * per):
            score = torch.from_numpy(np.ascontiguousarray(q[:, j])).to(DEV).double() @ keys.T / math.sqrt(dim)
            p = torch.softmax(score.masked_fill(future, -math.inf), 1)
            out[:, j] = p @ values
            if weights is not None:
                weights[h, :filled + tokens] += p.sum(0)
        if weights is not None:
            weights[h, :filled] += s.weight_in[h, :filled].double()
    flat = lambda a: torch.from_numpy(np.ascontiguousarray(a.reshape(tokens, -1)))   # noqa: E731
    return [out.reshape(tokens, -1), flat(k_new), flat(v_new)] + ([weights] if weights is not None else [])
