"""From a token's projections to the tokens that a draft's check gives out, as timed cases.

  turn     norms of the query and key heads and their rotation in one pass, positions of one axis (text) or three
           (time, height and width of images and video)
  fill     the same where the keys and the values go straight into a cache held in 4 bits, and a read of the rows
           that were written
  attend   attention over that cache: single tokens, drafted tokens to be checked, prompts; a window, scores that are
           capped by a tanh
  verify   drafted tokens against the target's distribution (temperature, top-k, top-p, min-p) from given uniform
           numbers, and the token that follows the accepted ones

Head layouts and vocabularies are those of the benchmark's configurations (32 heads over 8, 16 over 8; 128256 and
151936 words) and generic ones. Activations are N(0, 1); logits N(0, 3) with a few words well ahead of the others.

The cache: blocks of 32 neighbouring values of a token and head share a power of two, 2^(byte - 127); a value is a sign
and one of 0, 1/2, 1, 3/2, 2, 3, 4, 6 times that. Powers written are 2^-96 and above. A byte holds two neighbours, the first in its low half.
  keys    [pages, kv_heads, page, dim / 2], their powers [pages, kv_heads, page, dim / 32]
  values  [pages, kv_heads, page / 4, 16, 4, dim / 32]: four tokens, a sixteenth of the head of each together;
          their powers [pages, kv_heads, dim / 32, page]
"""
from __future__ import annotations

import math
import random

import torch

own = False

DEV = "cuda:0"
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZES = {"f32": 4, "f16": 2, "bf16": 2}
# query heads, key / value heads, values per head
HEADS = {"32x8x128": (32, 8, 128), "16x8x128": (16, 8, 128), "32x4x128": (32, 4, 128), "12x12x64": (12, 12, 64),
         "12x4x64": (12, 4, 64), "8x1x256": (8, 1, 256), "8x4x256": (8, 4, 256)}
VOCABULARIES = (32000, 50257, 128256, 151936, 262144)
LADDER = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)
POWERS = tuple(2.0 ** (b - 127) for b in range(255))


# ------------------------------------------------------------------------------------------ cases
def listed():
    return [
        # one chat user's next token between the projection and the cache
        {"name": "turn-1-f32", "kind": "turn", "rows": 1, "heads": "16x8x128", "type": "f32", "norm": True, "share": 1.0,
         "neighbours": False, "axes": "text", "far": 40000, "mix": 1},
        # a prompt with images: three axes that alternate from pair to pair
        {"name": "turn-4096-images-bf16", "kind": "turn", "rows": 4096, "heads": "32x8x128", "type": "bf16", "norm": True, "share": 1.0,
         "neighbours": False, "axes": "alternating", "far": 3000, "mix": 2},
        # a decode step of 64 sequences: rotated queries, keys and values into the cache
        {"name": "fill-64-f32", "kind": "fill", "rows": 64, "mode": "single", "page": 16, "heads": "16x8x128", "type": "f32", "norm": True,
         "share": 1.0, "neighbours": False, "axes": "text", "far": 8000, "mix": 3},
        # a prefill chunk, no head norms, pairs of neighbours
        {"name": "fill-2048-bf16", "kind": "fill", "rows": 2048, "mode": "chunk", "page": 32, "heads": "32x8x128", "type": "bf16", "norm": False,
         "share": 1.0, "neighbours": True, "axes": "text", "far": 100000, "mix": 4},
        # the smallest attention call: one sequence, a short context
        {"name": "attend-1x517", "kind": "attend", "mode": "even", "seqs": 1, "past": 516, "fresh": 1, "page": 16, "mix": 5,
         "heads": "16x8x128", "type": "f32", "window": 0, "cap": 0.0},
        # a full decode batch over ragged contexts
        {"name": "attend-64x8192", "kind": "attend", "mode": "ragged", "seqs": 64, "past": 8192, "fresh": 1, "page": 16, "mix": 6,
         "heads": "32x8x128", "type": "f32", "window": 0, "cap": 0.0},
        # one user with a long document
        {"name": "attend-1x131072-f16", "kind": "attend", "mode": "even", "seqs": 1, "past": 131071, "fresh": 1, "page": 64, "mix": 7,
         "heads": "32x8x128", "type": "f16", "window": 0, "cap": 0.0},
        # sixteen sequences' drafts of four tokens, capped scores
        {"name": "attend-16x5-capped-bf16", "kind": "attend", "mode": "even", "seqs": 16, "past": 4000, "fresh": 5, "page": 32, "mix": 8,
         "heads": "8x4x256", "type": "bf16", "window": 0, "cap": 50.0},
        # a prompt's prefill
        {"name": "attend-prefill-2048-bf16", "kind": "attend", "mode": "even", "seqs": 1, "past": 0, "fresh": 2048, "page": 16, "mix": 9,
         "heads": "32x8x128", "type": "bf16", "window": 0, "cap": 0.0},
        # four drafted tokens of one chat user
        {"name": "verify-1x5-151936", "kind": "verify", "mode": "even", "seqs": 1, "drafts": 4, "vocab": 151936, "type": "f32", "draft": "f32",
         "how": "chat", "mix": 10},
        # a batch of users who each ask for something else
        {"name": "verify-64x5-128256", "kind": "verify", "mode": "even", "seqs": 64, "drafts": 4, "vocab": 128256, "type": "f32", "draft": "bf16",
         "how": "all", "mix": 11},
        # drafts from a look-up, which are certain, against the model's own distribution
        {"name": "verify-32x8-certain-bf16", "kind": "verify", "mode": "ragged", "seqs": 32, "drafts": 8, "vocab": 151936, "type": "bf16",
         "draft": "certain", "how": "plain", "mix": 12},
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["turn", "turn", "fill", "fill", "attend", "attend", "attend", "verify", "verify"])
    mix = rng.randrange(1 << 20)
    if kind == "verify":
        return {"kind": kind, "mode": rng.choice(["even", "ragged"]), "seqs": _log_int(rng, 1, 48), "drafts": rng.randint(1, 6),
                "vocab": rng.choice(VOCABULARIES[:4] + (_log_int(rng, 1000, 151936),)), "type": rng.choice(["f32", "f32", "f16", "bf16"]),
                "draft": rng.choice(["f32", "f16", "bf16", "certain"]), "how": rng.choice(["chat", "all", "plain", "nucleus"]), "mix": mix}
    heads, dtype = rng.choice(sorted(HEADS)), rng.choice(["f32", "f32", "f16", "bf16"])
    if kind in ("turn", "fill"):
        case = {"kind": kind, "rows": _log_int(rng, 1, 2000), "heads": heads, "type": dtype, "norm": rng.random() < 0.6,
                "share": rng.choice([1.0, 1.0, 0.5]), "neighbours": rng.random() < 0.4, "axes": rng.choice(["text", "text", "sections", "alternating"]),
                "far": _log_int(rng, 100, 1 << 20), "mix": mix}
        if kind == "fill":
            case.update({"mode": rng.choice(["single", "chunk"]), "page": rng.choice([16, 16, 32, 64, 128])})
        return case
    page, window, cap = rng.choice([16, 16, 32, 64, 128]), rng.choice([0, 0, 0, _log_int(rng, 100, 4000)]), rng.choice([0.0, 0.0, 30.0, 50.0])
    if rng.random() < 0.5:     # decode, and a few tokens a sequence as a draft model's check brings them
        seqs = _log_int(rng, 1, 64)
        past = _log_int(rng, 1, 8192 * 16 // max(seqs, 16))
        return {"kind": kind, "mode": rng.choice(["even", "ragged"]), "seqs": seqs, "past": past, "fresh": rng.choice([1, 1, 1, rng.randint(2, 6)]),
                "page": page, "mix": mix, "heads": heads, "type": dtype, "window": window, "cap": cap}
    return {"kind": kind, "mode": rng.choice(["even", "ragged", "mixed"]), "seqs": rng.randint(1, 4), "past": _log_int(rng, 1, 2000),
            "fresh": _log_int(rng, 7, 900), "page": page, "mix": mix, "heads": heads, "type": dtype, "window": window, "cap": cap}


def _lengths(case):
    """Tokens that each sequence has in the cache, and tokens that it brings."""
    rng, seqs, past, fresh = random.Random(case["mix"]), case["seqs"], case["past"], case["fresh"]
    if case["mode"] == "even":
        return [past] * seqs, [fresh] * seqs
    if case["mode"] == "mixed":
        return [rng.randint(past // 2, past) for _ in range(seqs)], [fresh if i == 0 else 1 for i in range(seqs)]
    return [rng.randint(0 if fresh > 1 else 1, past) for _ in range(seqs)], [rng.randint(1, fresh) for _ in range(seqs)]


def _drafts(case):
    """Rows of each sequence: its drafted tokens and the one behind them."""
    rng = random.Random(case["mix"])
    return [1 + (case["drafts"] if case["mode"] == "even" else rng.randint(0, case["drafts"])) for _ in range(case["seqs"])]


# ------------------------------------------------------------------------------------------ inputs
def _int32(values):
    return torch.tensor(values, dtype=torch.int32, device=DEV)


def _prepare_turn(case, gen):
    heads, kv_heads, dim = HEADS[case["heads"]]
    rows, dtype = case["rows"], TYPES[case["type"]]
    # rows of a fused projection: queries, keys and values of a token side by side
    x = torch.randn((rows, heads + 2 * kv_heads, dim), device=DEV, generator=gen).to(dtype)
    pairs = int(dim * case["share"]) // 2
    state = {"case": case, "q": x[:, :heads], "k": x[:, heads:heads + kv_heads], "v": x[:, heads + kv_heads:]}
    state["frequencies"] = (1e6 ** (-torch.arange(pairs, dtype=torch.float64) / pairs)).float().to(DEV)
    first = torch.randint(0, case["far"], (1,), device=DEV, generator=gen)
    row = torch.arange(rows, device=DEV)
    if case["axes"] == "text":
        state["axis"] = None
        state["positions"] = ((first + row) if case.get("mode") != "single" else torch.randint(0, case["far"], (rows,), device=DEV, generator=gen)).int()
    else:
        # frames of 32 x 32 patches
        state["positions"] = torch.stack([first + row // 1024, first + row // 32 % 32, first + row % 32]).int()
        pair = torch.arange(pairs, device=DEV)
        state["axis"] = (pair % 3 if case["axes"] == "alternating" else pair * 3 // pairs).to(torch.uint8)
    for name in ("q_weight", "k_weight"):
        state[name] = torch.rand(dim, device=DEV, generator=gen) + 0.5 if case["norm"] else None
    if case["kind"] == "fill":
        page = case["page"]
        if case["mode"] == "single":     # each row in a page of its own
            pages = rows + 8
            slots = torch.randperm(pages, device=DEV, generator=gen)[:rows] * page + torch.randint(0, page, (rows,), device=DEV, generator=gen)
        else:
            pages, start = -(-rows // page) + 9, case["mix"] % page
            ids = torch.randperm(pages, device=DEV, generator=gen)
            slots = ids[(start + row) // page] * page + (start + row) % page
        state["pages"], state["slots"] = pages, slots
        _cache(state, gen, kv_heads, dim, page)
    return state


def _codes(gen, *shape):
    """Bytes of two codes each, as values that are normally distributed have them where the largest of 32 is about 4.5 units."""
    x = torch.empty(1 << 15, device=DEV).normal_(0.0, 2.2, generator=gen)
    table = _nearest(x.double())
    table = table[0::2] | table[1::2] << 4
    return table[torch.randint(0, table.numel(), shape, device=DEV, generator=gen, dtype=torch.int32)]


def _cache(state, gen, kv_heads, dim, page):
    pages = state["pages"]
    state["cache_k"] = _codes(gen, pages, kv_heads, page, dim // 2)
    state["cache_v"] = _codes(gen, pages, kv_heads, page // 4, 16, 4, dim // 32)
    state["k_powers"] = torch.randint(125, 127, (pages, kv_heads, page, dim // 32), device=DEV, generator=gen, dtype=torch.uint8)
    state["v_powers"] = torch.randint(125, 127, (pages, kv_heads, dim // 32, page), device=DEV, generator=gen, dtype=torch.uint8)


def _prepare_attend(case, gen):
    past, fresh = _lengths(case)
    page, seqs = case["page"], case["seqs"]
    want = [-(-(p + f) // page) for p, f in zip(past, fresh)]
    pages = sum(want) + 8
    ids = torch.randperm(pages, generator=gen, device=DEV).to(torch.int32)
    stride = max(want) + 1
    table = torch.full((seqs, stride), -1, dtype=torch.int32, device=DEV)
    cols, held = torch.arange(stride, device=DEV)[None], torch.tensor(want, device=DEV)[:, None]
    inside = cols < held
    table[inside] = ids[(torch.cumsum(held, 0) - held + cols)[inside]]
    starts = [0]
    for f in fresh:
        starts.append(starts[-1] + f)
    heads, kv_heads, dim = HEADS[case["heads"]]
    state = {"case": case, "table": table, "pages": pages, "starts": _int32(starts), "lens": _int32([p + f for p, f in zip(past, fresh)]),
             "max_fresh": max(fresh), "max_len": max(p + f for p, f in zip(past, fresh))}
    _cache(state, gen, kv_heads, dim, page)
    state["q"] = torch.randn((starts[-1], heads, dim), device=DEV, generator=gen).to(TYPES[case["type"]])
    state["out"] = torch.empty_like(state["q"])
    return state


def _prepare_verify(case, seed, gen):
    lengths, vocab = _drafts(case), case["vocab"]
    starts = [0]
    for n in lengths:
        starts.append(starts[-1] + n)
    rows = starts[-1]
    logits = torch.randn((rows, vocab), device=DEV, generator=gen) * 3.0
    ahead = torch.randint(0, vocab, (rows, 12), device=DEV, generator=gen)
    logits.scatter_(1, ahead, 12.0 + 2.0 * torch.rand((rows, 12), device=DEV, generator=gen))
    rng = random.Random(case["mix"] * 1000003 + seed)
    ask = {"chat": lambda: (0.7, 50, 0.9, 0.0), "plain": lambda: (1.0, 0, 1.0, 0.0), "nucleus": lambda: (1.0, 0, 0.95, 0.0),
           "all": lambda: rng.choice([(0.0, 0, 1.0, 0.0), (0.7, 40, 0.95, 0.05), (1.0, 0, 0.92, 0.0), (1.3, 0, 1.0, 0.02),
                                      (0.9, 1000, 1.0, 0.0), (1.0, 0, 1.0, 0.0), (2.0, 5, 0.5, 0.3)])}[case["how"]]
    rules = [r for n in lengths for r in [ask()] * n]     # a sequence's rows go by one request
    temperature, top_k, top_p, min_p = zip(*rules)
    f32 = lambda v: torch.tensor(v, dtype=torch.float32, device=DEV)  # noqa: E731
    state = {"case": case, "starts": _int32(starts), "temperature": f32(temperature), "top_k": _int32(top_k), "top_p": f32(top_p),
             "min_p": f32(min_p), "uniform": torch.rand(rows, device=DEV, generator=gen), "draw": torch.rand(len(lengths), device=DEV, generator=gen)}
    # the draft's view of the same text, a little off, at the request's temperature
    t = state["temperature"].clamp(min=0.1)[:, None]
    off = torch.softmax((logits + torch.randn((rows, vocab), device=DEV, generator=gen) * 0.5) / t, -1)
    if case["draft"] == "certain":
        state["draft"] = None
        state["drafted"] = off.argmax(-1).int()
    else:
        state["draft"] = off.to(TYPES[case["draft"]])
        state["drafted"] = torch.multinomial(off, 1, generator=gen)[:, 0].int()
    state["logits"] = logits.to(TYPES[case["type"]])
    return state


def prepare(case, seed):
    gen = torch.Generator(device=DEV)
    gen.manual_seed(seed)
    if case["kind"] == "verify":
        return _prepare_verify(case, seed, gen)
    return _prepare_attend(case, gen) if case["kind"] == "attend" else _prepare_turn(case, gen)


# ------------------------------------------------------------------------------------------ the plain forms
def _turned(x, weight, s, dtype):
    """Heads [rows, heads, dim], normed and rotated, in `dtype`."""
    case, pairs = s["case"], s["frequencies"].numel()
    x = x.to(dtype)
    if weight is not None:
        x = x / torch.sqrt((x * x).mean(-1, keepdim=True) + 1e-6) * weight.to(dtype)
    at = s["positions"].double()
    at = at[:, None] if s["axis"] is None else at[s["axis"].long()].T
    angle = (at * s["frequencies"].double())[:, None]
    cos, sin = torch.cos(angle).to(dtype), torch.sin(angle).to(dtype)
    if case["neighbours"]:
        a, b = x[..., 0:2 * pairs:2], x[..., 1:2 * pairs:2]
        turned = torch.stack([a * cos - b * sin, a * sin + b * cos], -1).flatten(-2)
    else:
        a, b = x[..., :pairs], x[..., pairs:2 * pairs]
        turned = torch.cat([a * cos - b * sin, a * sin + b * cos], -1)
    return torch.cat([turned, x[..., 2 * pairs:]], -1)


def _turn_plain(s):
    return {"q": _turned(s["q"], s["q_weight"], s, torch.float32).to(s["q"].dtype),
            "k": _turned(s["k"], s["k_weight"], s, torch.float32).to(s["k"].dtype)}


def _nearest(x):
    """Codes of values in units of their block's power: the nearest, halves to the even code; the sign in bit 3."""
    m = x.abs()
    code = (m > 0.25).int() + (m >= 0.75) + (m > 1.25) + (m >= 1.75) + (m > 2.5) + (m >= 3.5) + (m > 5.0)
    return (code + 8 * (x < 0)).to(torch.uint8)


def _held(x):
    """Rows [rows, heads, dim] as the cache's values, in 64 bits: borders of codes and powers are not to be missed."""
    blocks = x.double().unflatten(-1, (-1, 32))
    part, power = torch.frexp(blocks.abs().amax(-1, keepdim=True))
    power = torch.where(part == 0, -96, power - 3 + (part >= 0.875).int()).clamp(-96, 125)
    power = torch.tensor(POWERS, dtype=torch.float64, device=DEV)[power.long() + 127]
    ladder = torch.tensor(LADDER + tuple(-v for v in LADDER), dtype=torch.float64, device=DEV)
    return (ladder[_nearest(blocks / power).long()] * power).flatten(-2)


def _fill_plain(s):
    q = _turned(s["q"], s["q_weight"], s, torch.float32)
    k = _turned(s["k"], s["k_weight"], s, torch.float64)
    return {"q": q.to(s["q"].dtype), "k": _held(k).to(s["q"].dtype), "v": _held(s["v"]).to(s["q"].dtype)}


def _values(codes, powers, dtype=torch.float32):
    """Bytes [..., dim / 2] and powers [..., dim / 32] as values [..., dim]."""
    ladder = torch.tensor(LADDER + tuple(-v for v in LADDER), dtype=dtype, device=DEV)
    both = torch.stack([codes & 15, codes >> 4], -1).flatten(-2)
    power = torch.tensor(POWERS, dtype=dtype, device=DEV)[powers.int()]
    return (ladder[both.int()].unflatten(-1, (-1, 32)) * power[..., None]).flatten(-2)


def _by_token(v):
    """Values' bytes [..., page / 4, 16, 4, n] as [..., page, 16 n]."""
    return v.transpose(-3, -2).flatten(-4, -3).flatten(-2)


def _attend_plain(s):
    case = s["case"]
    heads, kv_heads, dim = HEADS[case["heads"]]
    page, most, window, cap = case["page"], s["max_fresh"], case["window"], case["cap"]
    q, starts, lens = s["q"], s["starts"].long(), s["lens"].long()
    seqs, group = lens.numel(), heads // kv_heads
    entries = s["table"][:, :-(-s["max_len"] // page)].long().clamp(min=0)
    ctx = entries.shape[1] * page

    def values(codes, powers):
        return _values(codes, powers).permute(0, 2, 1, 3, 4).reshape(seqs, kv_heads, ctx, dim)

    row = torch.arange(most, device=DEV)[None]
    n = (starts[1:] - starts[:-1])[:, None]
    token = (starts[:-1, None] + row).clamp(max=q.shape[0] - 1)
    rows = q.float()[token].reshape(seqs, most, kv_heads, group, dim).permute(0, 2, 3, 1, 4).reshape(seqs, kv_heads, group * most, dim)
    keys = values(s["cache_k"][entries], s["k_powers"][entries])
    scores = torch.matmul(rows, keys.transpose(-1, -2).contiguous()) / math.sqrt(dim)
    if cap:
        scores = cap * torch.tanh(scores / cap)
    at, pos = torch.arange(ctx, device=DEV)[None, None], (lens[:, None] - n + row)[..., None]
    seen = at <= pos
    if window:
        seen = seen & (at > pos - window)
    scores = scores.reshape(seqs, kv_heads, group, most, ctx).masked_fill(~seen[:, None, None], -math.inf)
    p = torch.exp(scores - scores.amax(-1, keepdim=True))
    p = p / p.sum(-1, keepdim=True)
    out = torch.matmul(p.reshape(seqs, kv_heads, group * most, ctx), values(_by_token(s["cache_v"][entries]), s["v_powers"][entries].transpose(-1, -2)))
    out = out.reshape(seqs, kv_heads, group, most, dim).permute(0, 3, 1, 2, 4).reshape(seqs, most, heads, dim)
    # each row of the batch from its place in the padded rectangle
    place = torch.arange(q.shape[0], device=DEV)
    seq = torch.searchsorted(starts[1:], place, right=True)
    return out[seq, place - starts[seq]].to(q.dtype)


def _target(s):
    """The target's distribution of every row, in 64 bits: a sum over a vocabulary decides between neighbours."""
    logits = s["logits"].double()
    ordered, order = torch.sort(logits, dim=-1, descending=True, stable=True)
    temperature = s["temperature"].double()[:, None]
    greedy = temperature <= 0
    weight = torch.exp((ordered - ordered[:, :1]) / torch.where(greedy, 1.0, temperature))
    total = torch.cumsum(weight, -1)
    at = torch.arange(logits.shape[1], device=DEV)[None]
    k = s["top_k"].long()[:, None]
    n1 = torch.where(k > 0, k.clamp(max=logits.shape[1]), logits.shape[1])
    top_p = s["top_p"].double()[:, None]
    reach = ((total < top_p * total.gather(-1, n1 - 1)) & (at < n1)).sum(-1, keepdim=True) + 1
    n2 = torch.where(top_p < 1, torch.minimum(reach, n1), n1)
    n3 = (weight >= s["min_p"].double()[:, None]).sum(-1, keepdim=True).clamp(min=1)
    n = torch.where(greedy, 1, torch.minimum(n2, n3))
    p = torch.where(at < n, weight, 0.0) / total.gather(-1, n - 1)
    return torch.zeros_like(p).scatter_(-1, order, p)


def _verify_plain(s):
    p, starts, drafted = _target(s), s["starts"].long(), s["drafted"].long()
    rows, seqs = drafted.numel(), starts.numel() - 1
    row = torch.arange(rows, device=DEV)
    seq = torch.searchsorted(starts[1:], row, right=True)
    at, n = row - starts[seq], starts[1:] - starts[:-1]
    of_target = p.gather(-1, drafted[:, None])[:, 0]
    of_draft = torch.ones_like(of_target) if s["draft"] is None else s["draft"].gather(-1, drafted[:, None])[:, 0].double()
    refused = (at < n[seq] - 1) & ~(s["uniform"].double() * of_draft < of_target)
    accepted = (n - 1).scatter_reduce(0, seq, torch.where(refused, at, rows), "amin")
    last = starts[:-1] + accepted
    some = (accepted < n - 1)[:, None]
    if s["draft"] is None:
        taken = torch.zeros((seqs, p.shape[1]), dtype=torch.float64, device=DEV).scatter_(-1, drafted[last][:, None], 1.0)
    else:
        taken = s["draft"][last].double()
    left = (p[last] - torch.where(some, taken, 0.0)).clamp(min=0)
    left = torch.where(left.sum(-1, keepdim=True) > 0, left, p[last])
    sums = torch.cumsum(left, -1)
    word = (sums <= s["draw"].double()[:, None] * sums[:, -1:]).sum(-1)
    word = torch.minimum(word, (sums < sums[:, -1:]).sum(-1))
    tokens = torch.where(at < accepted[seq], drafted, torch.where(at == accepted[seq], word[seq], -1))
    probs = torch.where(tokens >= 0, p.gather(-1, tokens.clamp(min=0)[:, None])[:, 0], 0.0)
    return {"tokens": tokens.int(), "accepted": accepted.int(), "probs": probs.float()}


# ------------------------------------------------------------------------------------------ the library's calls
def _handle(s):
    """The cache's handle, which a program keeps."""
    if "handle" not in s:
        from loken_amd import kv
        s["handle"] = kv.KvCacheMxfp4(s["cache_k"], s["cache_v"], s["k_powers"], s["v_powers"])
    return s["handle"]


def _rotary(s):
    """A model's rotation, which a program keeps."""
    if "rotary" not in s:
        from loken_amd import rotary
        s["rotary"] = rotary.Rotary(s["frequencies"], axis=s["axis"], neighbours=s["case"]["neighbours"])
    return s["rotary"]


def _turn_own(s):
    from loken_amd import rotary
    q, k = rotary.rotate(s["q"], s["k"], s["positions"], _rotary(s), q_weight=s["q_weight"], k_weight=s["k_weight"], eps=1e-6)
    return {"q": q, "k": k}


def _fill_own(s):
    from loken_amd import kv, rotary
    q = rotary.rotate_into(_handle(s), s["q"], s["k"], s["v"], s["positions"], s["slots"], _rotary(s), q_weight=s["q_weight"], k_weight=s["k_weight"],
                           eps=1e-6)
    k, v = kv.kv_read(_handle(s), s["slots"], dtype=s["q"].dtype)
    return {"q": q, "k": k, "v": v}


def _attend_own(s):
    from loken_amd import kv
    return kv.kv_attention(s["q"], _handle(s), s["table"], s["lens"], s["starts"], max_fresh=s["max_fresh"], max_len=s["max_len"],
                           window=s["case"]["window"], softcap=s["case"]["cap"], out=s["out"])


def _verify_own(s):
    from loken_amd import sampling
    tokens, accepted, probs = sampling.verify(s["logits"], s["drafted"], s["starts"], s["uniform"], s["draw"], s["temperature"], s["top_k"],
                                              s["top_p"], s["min_p"], draft=s["draft"])
    return {"tokens": tokens, "accepted": accepted, "probs": probs}


def run(state):
    kind = state["case"]["kind"]
    if own:
        return {"turn": _turn_own, "fill": _fill_own, "attend": _attend_own, "verify": _verify_own}[kind](state)
    return {"turn": _turn_plain, "fill": _fill_plain, "attend": _attend_plain, "verify": _verify_plain}[kind](state)


# ------------------------------------------------------------------------------------------ in 64 bits, from the definitions
def exact(case, seed):
    s = prepare(case, seed)
    return {"turn": _turn_exact, "fill": _fill_exact, "attend": _attend_exact, "verify": _verify_exact}[case["kind"]](s)


def _turned_exact(x, weight, s):
    x = x.double()
    if weight is not None:
        x = x * weight.double() * (x.pow(2).sum(-1, keepdim=True) / x.shape[-1] + 1e-6).pow(-0.5)
    freq, out = s["frequencies"].tolist(), x.clone()
    n = len(freq)
    for i in range(n):
        pos = s["positions"] if s["axis"] is None else s["positions"][int(s["axis"][i])]
        turn = torch.polar(torch.ones(pos.numel(), dtype=torch.float64, device=DEV), pos.double() * freq[i])[:, None]
        one, two = (2 * i, 2 * i + 1) if s["case"]["neighbours"] else (i, i + n)
        z = torch.complex(x[:, :, one], x[:, :, two]) * turn
        out[:, :, one], out[:, :, two] = z.real, z.imag
    return out


def _turn_exact(s):
    return {"q": _turned_exact(s["q"], s["q_weight"], s), "k": _turned_exact(s["k"], s["k_weight"], s)}


def _held_exact(x):
    x = x.double()
    for b in range(0, x.shape[-1], 32):
        block = x[..., b:b + 32]
        peak = block.abs().amax(-1, keepdim=True)
        unit = torch.full_like(peak, 2.0 ** -96)
        while bool((peak >= 7 * unit).any()):
            unit = torch.where(peak >= 7 * unit, 2 * unit, unit)
        steps = torch.tensor(LADDER, dtype=torch.float64, device=DEV)
        far = (block.abs()[..., None] / unit[..., None] - steps).abs()
        best = far.amin(-1, keepdim=True)
        even = torch.tensor([0, 9, 1, 9, 2, 9, 3, 9], device=DEV)     # of two that are as near, the even code
        pick = torch.where(far == best, torch.where(even < 9, 0, 1), 2).argmin(-1)
        x[..., b:b + 32] = torch.sign(block) * steps[pick] * unit
    return x


def _fill_exact(s):
    return {"q": _turned_exact(s["q"], s["q_weight"], s), "k": _held_exact(_turned_exact(s["k"], s["k_weight"], s)), "v": _held_exact(s["v"])}


def _attend_exact(s):
    case = s["case"]
    heads, kv_heads, dim = HEADS[case["heads"]]
    page, window = case["page"], case["window"]
    lens, starts = s["lens"].tolist(), s["starts"].tolist()
    out = torch.zeros((starts[-1], heads, dim), dtype=torch.float64, device=DEV)
    for i, length in enumerate(lens):
        ids = s["table"][i, :-(-length // page)].long()
        sides = []
        for codes, powers in ((s["cache_k"][ids], s["k_powers"][ids]), (_by_token(s["cache_v"][ids]), s["v_powers"][ids].transpose(-1, -2))):
            sides.append(_values(codes, powers, torch.float64).permute(0, 2, 1, 3).reshape(-1, kv_heads, dim)[:length])
        a, b = starts[i], starts[i + 1]
        pos = torch.arange(length - (b - a), length, device=DEV)[:, None]
        at = torch.arange(length, device=DEV)[None]
        hidden = (at > pos) | ((at <= pos - window) if window else (at < 0))
        for h in range(heads):
            kh, vh = sides[0][:, h // (heads // kv_heads)], sides[1][:, h // (heads // kv_heads)]
            z = (s["q"][a:b, h].double() @ kh.T.contiguous()) / math.sqrt(dim)
            if case["cap"]:
                z = torch.tanh(z / case["cap"]) * case["cap"]
            out[a:b, h] = torch.softmax(z.masked_fill(hidden, -math.inf), -1) @ vh.contiguous()
    return out


def _verify_exact(s):
    starts, drafted = s["starts"].tolist(), s["drafted"].tolist()
    rules = list(zip(*(s[name].tolist() for name in ("temperature", "top_k", "top_p", "min_p"))))
    tokens, accepted, probs = [], [], []

    def distribution(r):
        x = s["logits"][r].double()
        temperature, top_k, top_p, min_p = rules[r]
        order = torch.argsort(x, descending=True, stable=True)
        w = torch.exp((x[order] - x[order[0]]) / temperature) if temperature > 0 else torch.ones(1, dtype=torch.float64, device=DEV)
        kept = w[:top_k] if top_k > 0 else w
        if top_p < 1:
            sums = torch.cumsum(kept, 0)
            kept = kept[:int((sums < top_p * sums[-1]).sum()) + 1]
        kept = kept[:max(1, int((w >= min_p).sum()))]
        p = torch.zeros_like(x)
        p[order[:kept.numel()]] = kept / kept.sum()
        return p

    for i in range(len(starts) - 1):
        here = 0
        for r in range(starts[i], starts[i + 1]):
            p = distribution(r)
            left = p
            if r < starts[i + 1] - 1:
                word = drafted[r]
                of_draft = 1.0 if s["draft"] is None else float(s["draft"][r, word])
                if float(s["uniform"][r]) * of_draft < float(p[word]):
                    tokens.append(word)
                    probs.append(float(p[word]))
                    here += 1
                    continue
                if s["draft"] is None:
                    left = p.clone()
                    left[word] = 0
                else:
                    left = (p - s["draft"][r].double()).clamp(min=0)
                left = left if float(left.sum()) > 0 else p
            sums = torch.cumsum(left, 0)
            word = min(int((sums <= float(s["draw"][i]) * sums[-1]).sum()), int((sums < sums[-1]).sum()))
            tokens.append(word)
            probs.append(float(p[word]))
            break
        accepted.append(here)
        tokens += [-1] * (starts[i + 1] - len(tokens))
        probs += [0.0] * (starts[i + 1] - len(probs))
    return {"tokens": torch.tensor(tokens, dtype=torch.int32), "accepted": torch.tensor(accepted, dtype=torch.int32),
            "probs": torch.tensor(probs, dtype=torch.float64)}


# ------------------------------------------------------------------------------------------ what a pass needs
def work(case):
    if case["kind"] == "verify":
        rows, seqs, vocab = sum(_drafts(case)), case["seqs"], case["vocab"]
        draft = 0 if case["draft"] == "certain" else SIZES[case["draft"]]
        # the logits of every row, and the draft's distribution where a sequence ends
        return {"bytes": float(vocab) * (rows * SIZES[case["type"]] + seqs * draft) + 36.0 * rows, "flops": 4.0 * rows * vocab}
    heads, kv_heads, dim = HEADS[case["heads"]]
    size = SIZES[case["type"]]
    if case["kind"] in ("turn", "fill"):
        turned = case["rows"] * (heads + kv_heads) * dim
        held = 2 * case["rows"] * kv_heads * dim
        if case["kind"] == "turn":
            return {"bytes": 2.0 * turned * size, "flops": 8.0 * turned}
        # queries in and out; keys and values in, written and read back as 4.25 bits each, and out as values
        return {"bytes": 2.0 * case["rows"] * heads * dim * size + held * (2.0 * size + 2 * 0.53125), "flops": 8.0 * turned + 8.0 * held}
    past, fresh = _lengths(case)
    tokens, window = sum(fresh), case["window"] or 1 << 40
    cached = sum(min(p + f, f - 1 + window) for p, f in zip(past, fresh))
    pairs = sum(sum(min(p + j + 1, window) for j in range(f)) for p, f in zip(past, fresh))
    return {"bytes": 2.0 * kv_heads * cached * dim * 0.53125 + 2.0 * tokens * heads * dim * size, "flops": 4.0 * heads * dim * pairs}
