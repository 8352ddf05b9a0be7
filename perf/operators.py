"""The steps of a served decode step around the quantized linears, as timed cases.

  plan     block tables and slot maps of a batch from its request lengths: which pages of the cache each sequence
           gets, where each new token's keys and values go, and where each sequence's rows start
  store    the new tokens' keys and values into a cache held in 8 bits with a scale for each page of tokens and
           head, and a read of the pages that were touched
  attend   attention of the new tokens over that cache: single tokens of many sequences, one long sequence,
           prefill chunks, and batches that mix them
  sample   the next token of each sequence from its logits: temperature, top-k, top-p, min-p and a given
           uniform number

Head layouts and vocabularies are those of the benchmark's configurations (32 heads over 8, 16 over 8; 128256 and
151936 words) and generic ones. Activations are N(0, 1); logits N(0, 3) with a few words well ahead of the others.

The cache: page p of head h holds `page` tokens. Keys [pages, kv_heads, page, dim]; values in runs of sixteen
tokens, [pages, kv_heads, page / 16, dim, 16]; scales [pages, kv_heads]. A value is code * scale.
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
HEADS = {"32x8x128": (32, 8, 128), "16x8x128": (16, 8, 128), "32x4x128": (32, 4, 128), "16x16x64": (16, 16, 64),
         "12x4x64": (12, 4, 64), "8x1x256": (8, 1, 256), "8x4x256": (8, 4, 256)}
VOCABULARIES = (32000, 50257, 128256, 151936, 262144)


# ------------------------------------------------------------------------------------------ cases
def listed():
    return [
        # the step's plan for 64 sequences that each got one token, as every decode step makes it
        {"name": "plan-64-decode", "kind": "plan", "mode": "even", "seqs": 64, "past": 4096, "fresh": 1, "page": 16, "mix": 1},
        # the same where 512 requests come in with ragged prompts (some sharing a cached start)
        {"name": "plan-512-prompts", "kind": "plan", "mode": "ragged", "seqs": 512, "past": 1000, "fresh": 700, "page": 16, "mix": 2},
        # one decode step's keys and values of 64 sequences
        {"name": "store-64-decode", "kind": "store", "mode": "ragged", "seqs": 64, "past": 2000, "fresh": 1, "page": 16, "mix": 3,
         "heads": "16x8x128", "type": "f32"},
        # a prefill chunk of five ragged prompts
        {"name": "store-prompts-bf16", "kind": "store", "mode": "ragged", "seqs": 5, "past": 300, "fresh": 1800, "page": 32, "mix": 4,
         "heads": "32x8x128", "type": "bf16"},
        # the smallest attention call: one sequence, a short context
        {"name": "attend-1x517", "kind": "attend", "mode": "even", "seqs": 1, "past": 516, "fresh": 1, "page": 16, "mix": 5,
         "heads": "16x8x128", "type": "f32", "window": 0},
        # a full decode batch over ragged contexts
        {"name": "attend-64x8192", "kind": "attend", "mode": "ragged", "seqs": 64, "past": 8192, "fresh": 1, "page": 16, "mix": 6,
         "heads": "32x8x128", "type": "f32", "window": 0},
        # one user with a long document
        {"name": "attend-1x131072-f16", "kind": "attend", "mode": "even", "seqs": 1, "past": 131071, "fresh": 1, "page": 64, "mix": 7,
         "heads": "32x8x128", "type": "f16", "window": 0},
        # a prompt's prefill
        {"name": "attend-prefill-2048-bf16", "kind": "attend", "mode": "even", "seqs": 1, "past": 0, "fresh": 2048, "page": 16, "mix": 8,
         "heads": "32x8x128", "type": "bf16", "window": 0},
        # chunked prefill beside decode: one sequence brings 700 tokens, eleven bring one
        {"name": "attend-mixed-700", "kind": "attend", "mode": "mixed", "seqs": 12, "past": 3000, "fresh": 700, "page": 16, "mix": 9,
         "heads": "32x4x128", "type": "f32", "window": 0},
        # one user's next token, as chat programs sample
        {"name": "sample-1x151936", "kind": "sample", "rows": 1, "vocab": 151936, "type": "f32", "how": "chat", "mix": 10},
        # a batch of users who each ask for something else
        {"name": "sample-64x128256", "kind": "sample", "rows": 64, "vocab": 128256, "type": "f32", "how": "all", "mix": 11},
        # many samples of one prompt at the model's own distribution
        {"name": "sample-256x151936-bf16", "kind": "sample", "rows": 256, "vocab": 151936, "type": "bf16", "how": "plain", "mix": 12},
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["plan", "store", "attend", "attend", "attend", "sample", "sample"])
    mix = rng.randrange(1 << 20)
    if kind == "plan":
        return {"kind": kind, "mode": rng.choice(["even", "ragged", "mixed"]), "seqs": _log_int(rng, 1, 512), "past": _log_int(rng, 1, 8192),
                "fresh": rng.choice([1, _log_int(rng, 1, 700)]), "page": rng.choice([16, 32, 64, 128]), "mix": mix}
    if kind == "sample":
        return {"kind": kind, "rows": _log_int(rng, 1, 128), "vocab": rng.choice(VOCABULARIES + (_log_int(rng, 1000, 262144),)),
                "type": rng.choice(["f32", "f32", "f16", "bf16"]), "how": rng.choice(["chat", "all", "plain", "nucleus"]), "mix": mix}
    heads, page, dtype = rng.choice(sorted(HEADS)), rng.choice([16, 16, 32, 64, 128]), rng.choice(["f32", "f32", "f16", "bf16"])
    if kind == "store":
        return {"kind": kind, "mode": rng.choice(["even", "ragged", "mixed"]), "seqs": _log_int(rng, 1, 16), "past": _log_int(rng, 1, 3000),
                "fresh": rng.choice([1, _log_int(rng, 1, 900)]), "page": page, "mix": mix, "heads": heads, "type": dtype}
    window = rng.choice([0, 0, 0, _log_int(rng, 100, 4000)])
    if rng.random() < 0.5:     # decode, and a few tokens a sequence as a draft model's check brings them
        seqs = _log_int(rng, 1, 64)
        past = _log_int(rng, 1, 8192 * 16 // max(seqs, 16))
        return {"kind": kind, "mode": rng.choice(["even", "ragged"]), "seqs": seqs, "past": past, "fresh": rng.choice([1, 1, 1, rng.randint(2, 6)]),
                "page": page, "mix": mix, "heads": heads, "type": dtype, "window": window}
    return {"kind": kind, "mode": rng.choice(["even", "ragged", "mixed"]), "seqs": rng.randint(1, 4), "past": _log_int(rng, 1, 2000),
            "fresh": _log_int(rng, 7, 900), "page": page, "mix": mix, "heads": heads, "type": dtype, "window": window}


def _lengths(case):
    """Tokens that each sequence has in the cache, and tokens that it brings."""
    rng, seqs, past, fresh = random.Random(case["mix"]), case["seqs"], case["past"], case["fresh"]
    if case["mode"] == "even":
        return [past] * seqs, [fresh] * seqs
    if case["mode"] == "mixed":
        return [rng.randint(past // 2, past) for _ in range(seqs)], [fresh if i == 0 else 1 for i in range(seqs)]
    return [rng.randint(0 if fresh > 1 else 1, past) for _ in range(seqs)], [rng.randint(1, fresh) for _ in range(seqs)]


# ------------------------------------------------------------------------------------------ inputs
def _int32(values):
    return torch.tensor(values, dtype=torch.int32, device=DEV)


def _prepare_plan(case, gen):
    past, fresh = _lengths(case)
    page, seqs = case["page"], case["seqs"]
    have = [-(-p // page) for p in past]
    want = [-(-(p + f) // page) for p, f in zip(past, fresh)]
    pages = sum(want) + 64
    ids = torch.randperm(pages, generator=gen, device=DEV).to(torch.int32)
    stride = max(want) + 3
    table = torch.full((seqs, stride), -1, dtype=torch.int32, device=DEV)
    cols = torch.arange(stride, device=DEV)[None]
    held = torch.tensor(have, device=DEV)[:, None]
    first = torch.cumsum(held, 0) - held
    inside = cols < held
    table[inside] = ids[(first + cols)[inside]]
    # a batch padded to a multiple of 64 rows, as a program that replays recorded steps has it
    rows = -(-sum(fresh) // 64) * 64
    return {"case": case, "past": _int32(past), "fresh": _int32(fresh), "table": table, "free": ids[sum(have):].contiguous(),
            "taken": torch.zeros(1, dtype=torch.int32, device=DEV), "rows": rows, "pages": pages}


def _where(case, gen):
    """A batch's tables as torch makes them: the plan that `store` and `attend` are given."""
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
    seq = torch.repeat_interleave(torch.arange(seqs, device=DEV), torch.tensor(fresh, device=DEV))
    at = torch.arange(starts[-1], device=DEV) - torch.tensor(starts, device=DEV)[seq] + torch.tensor(past, device=DEV)[seq]
    slots = table[seq, at // page].long() * page + at % page
    return {"case": case, "table": table, "pages": pages, "slots": slots, "starts": _int32(starts),
            "lens": _int32([p + f for p, f in zip(past, fresh)]), "max_fresh": max(fresh), "max_len": max(p + f for p, f in zip(past, fresh)),
            "tokens": starts[-1]}


def _codes(gen, *shape):
    """Codes of normal values whose largest in a page is about 3.5 deviations."""
    return torch.empty(shape, dtype=torch.float16, device=DEV).normal_(0.0, 36.0, generator=gen).clamp_(-127, 127).round_().to(torch.int8)


def _cache(state, gen, kv_heads, dim, page):
    pages = state["pages"]
    state["k"] = _codes(gen, pages, kv_heads, page, dim)
    state["v"] = _codes(gen, pages, kv_heads, page // 16, dim, 16)
    for name in ("k_scales", "v_scales"):
        state[name] = torch.rand((pages, kv_heads), device=DEV, generator=gen) * 0.01 + 0.02
    return state


def prepare(case, seed):
    gen = torch.Generator(device=DEV)
    gen.manual_seed(seed)
    if case["kind"] == "plan":
        return _prepare_plan(case, gen)
    if case["kind"] == "sample":
        return _prepare_sample(case, seed, gen)
    heads, kv_heads, dim = HEADS[case["heads"]]
    state, dtype = _cache(_where(case, gen), gen, kv_heads, dim, case["page"]), TYPES[case["type"]]
    if case["kind"] == "store":
        # rows of a fused projection: queries, keys and values of a token side by side
        rows = torch.randn((state["tokens"], heads + 2 * kv_heads, dim), device=DEV, generator=gen).to(dtype)
        state["new_k"], state["new_v"] = rows[:, heads:heads + kv_heads], rows[:, heads + kv_heads:]
        touched = torch.unique(state["slots"] // case["page"])
        state["read"] = (touched[:, None] * case["page"] + torch.arange(case["page"], device=DEV)).reshape(-1)
        return state
    state["q"] = torch.randn((state["tokens"], heads, dim), device=DEV, generator=gen).to(dtype)
    state["out"] = torch.empty_like(state["q"])
    return state


def _prepare_sample(case, seed, gen):
    rows, vocab = case["rows"], case["vocab"]
    logits = torch.randn((rows, vocab), device=DEV, generator=gen) * 3.0
    ahead = torch.randint(0, vocab, (rows, 12), device=DEV, generator=gen)
    logits.scatter_(1, ahead, 12.0 + 2.0 * torch.rand((rows, 12), device=DEV, generator=gen))
    rng = random.Random(case["mix"] * 1000003 + seed)
    ask = {"chat": lambda: (0.7, 50, 0.9, 0.0), "plain": lambda: (1.0, 0, 1.0, 0.0), "nucleus": lambda: (1.0, 0, 0.95, 0.0),
           "all": lambda: rng.choice([(0.0, 0, 1.0, 0.0), (0.7, 40, 0.95, 0.05), (1.0, 0, 0.92, 0.0), (1.3, 0, 1.0, 0.02),
                                      (0.9, 1000, 1.0, 0.0), (1.0, 0, 1.0, 0.0), (2.0, 5, 0.5, 0.3)])}[case["how"]]
    temperature, top_k, top_p, min_p = zip(*(ask() for _ in range(rows)))
    f32 = lambda v: torch.tensor(v, dtype=torch.float32, device=DEV)  # noqa: E731
    return {"case": case, "logits": logits.to(TYPES[case["type"]]), "temperature": f32(temperature), "top_k": _int32(top_k),
            "top_p": f32(top_p), "min_p": f32(min_p), "uniform": torch.rand(rows, device=DEV, generator=gen)}


# ------------------------------------------------------------------------------------------ the plain forms
def _plan_plain(s):
    page, rows, table, free = s["case"]["page"], s["rows"], s["table"], s["free"]
    past, fresh, taken = s["past"].long(), s["fresh"].long(), s["taken"].long()
    total = past + fresh
    have, want = (past + page - 1) // page, (total + page - 1) // page
    need = want - have
    first = taken + torch.cumsum(need, 0) - need
    cols = torch.arange(table.shape[1], device=DEV)[None]
    place = first[:, None] + cols - have[:, None]
    got = torch.where(place < free.numel(), free[place.clamp(0, free.numel() - 1)], -1)
    table = torch.where((cols >= have[:, None]) & (cols < want[:, None]), got, table)
    starts = torch.cat([torch.zeros_like(taken), torch.cumsum(fresh, 0)])
    row = torch.arange(rows, device=DEV)
    seq = torch.searchsorted(starts[1:], row, right=True).clamp(max=past.numel() - 1)
    live = row < starts[-1]
    at = torch.where(live, past[seq] + row - starts[seq], 0)
    entry = table[seq, at // page].long()
    slots = torch.where(live & (entry >= 0), entry * page + at % page, -1)
    return {"table": table, "lens": total.int(), "starts": starts.int(), "slots": slots, "positions": at.int(),
            "taken": (taken + need.sum()).int()}


def _away(x):
    """The nearest whole number, halves away from zero."""
    whole = torch.trunc(x)
    return whole + torch.where((x - whole).abs() >= 0.5, torch.sign(x), torch.zeros_like(x))


def _store_side(codes, scales, new, slots, touched, page):
    """One side's codes [pages, heads, page, dim] and scales with the new rows in them."""
    at, off = slots // page, slots % page
    peak = new.abs().amax(-1)
    most = torch.zeros_like(scales).scatter_reduce_(0, at[:, None].expand_as(peak), peak, "amax")
    least = torch.full((scales.shape[0],), page, device=DEV, dtype=torch.int64).scatter_reduce_(0, at, off, "amin")
    kept = torch.where(least[:, None] > 0, scales, torch.zeros_like(scales))
    d = torch.maximum(kept, most / torch.full_like(most, 127.0))     # f32, correctly rounded
    scale = torch.where((least < page)[:, None], d, scales)
    # the quotients stand next to the border of two codes now and then: 64 bits
    ratio = codes[touched].double() * kept[touched].double()[:, :, None, None] / scale[touched].double()[:, :, None, None]
    codes = codes.index_put((touched,), _away(torch.nan_to_num(ratio, nan=0.0)).to(torch.int8))
    code = _away(torch.nan_to_num(new.double() / scale[at].double()[:, :, None], nan=0.0)).to(torch.int8)
    return codes.index_put((at[:, None], torch.arange(scales.shape[1], device=DEV)[None], off[:, None]), code), scale


def _by_token(v):
    """Values [pages, heads, page / 16, dim, 16] as [pages, heads, page, dim]."""
    return v.permute(0, 1, 2, 4, 3).reshape(v.shape[0], v.shape[1], v.shape[2] * 16, v.shape[3])


def _store_plain(s):
    page, out = s["case"]["page"], {}
    touched = s["read"][::page] // page
    for side, codes in (("k", s["k"]), ("v", _by_token(s["v"]))):
        new = s["new_" + side]
        codes, scales = _store_side(codes, s[side + "_scales"], new.float(), s["slots"], touched, page)
        at = s["read"] // page
        out[side] = (codes[at, :, s["read"] % page].float() * scales[at][:, :, None]).to(new.dtype)
        out[side + "_scales"] = scales
    return out


def _attend_plain(s):
    case = s["case"]
    heads, kv_heads, dim = HEADS[case["heads"]]
    page, most, window = case["page"], s["max_fresh"], case["window"]
    q, starts, lens = s["q"], s["starts"].long(), s["lens"].long()
    seqs, group = lens.numel(), heads // kv_heads
    entries = s["table"][:, :-(-s["max_len"] // page)].long().clamp(min=0)
    ctx = entries.shape[1] * page

    def values(codes, scales):
        x = codes[entries].float() * scales[entries][..., None, None]          # [seqs, entries, kv_heads, page, dim]
        return x.permute(0, 2, 1, 3, 4).reshape(seqs, kv_heads, ctx, dim)

    row = torch.arange(most, device=DEV)[None]
    n = (starts[1:] - starts[:-1])[:, None]
    live = row < n
    token = (starts[:-1, None] + row).clamp(max=q.shape[0] - 1)
    rows = q.float()[token].reshape(seqs, most, kv_heads, group, dim).permute(0, 2, 3, 1, 4).reshape(seqs, kv_heads, group * most, dim)
    scores = torch.matmul(rows, values(s["k"], s["k_scales"]).transpose(-1, -2).contiguous()) / math.sqrt(dim)
    at, pos = torch.arange(ctx, device=DEV)[None, None], (lens[:, None] - n + row)[..., None]
    seen = at <= pos
    if window:
        seen = seen & (at > pos - window)
    scores = scores.reshape(seqs, kv_heads, group, most, ctx).masked_fill(~seen[:, None, None], -math.inf)
    p = torch.exp(scores - scores.amax(-1, keepdim=True))
    p = p / p.sum(-1, keepdim=True)
    out = torch.matmul(p.reshape(seqs, kv_heads, group * most, ctx), values(_by_token(s["v"]), s["v_scales"]))
    out = out.reshape(seqs, kv_heads, group, most, dim).permute(0, 3, 1, 2, 4).reshape(seqs, most, heads, dim)
    # each row of the batch from its place in the padded rectangle
    place = torch.arange(q.shape[0], device=DEV)
    seq = torch.searchsorted(starts[1:], place, right=True)
    return out[seq, place - starts[seq]].to(q.dtype)


def _sample_plain(s):
    # 64 bits: a sum over a vocabulary decides between neighbours that differ by a share of 1e-6 and less
    logits = s["logits"].double()
    valid = logits > -math.inf
    logits = torch.where(valid, logits, -math.inf)
    ordered, order = torch.sort(logits, dim=-1, descending=True, stable=True)
    temperature = s["temperature"].double()[:, None]
    greedy = temperature <= 0
    weight = torch.exp((ordered - ordered[:, :1]) / torch.where(greedy, 1.0, temperature))
    total = torch.cumsum(weight, -1)
    count = valid.sum(-1, keepdim=True)
    at = torch.arange(logits.shape[1], device=DEV)[None]
    k = s["top_k"].long()[:, None]
    n1 = torch.where(k > 0, torch.minimum(k, count), count)
    top_p = s["top_p"].double()[:, None]
    reach = ((total < top_p * total.gather(-1, n1 - 1)) & (at < n1)).sum(-1, keepdim=True) + 1
    n2 = torch.where(top_p < 1, torch.minimum(reach, n1), n1)
    n3 = ((weight >= s["min_p"].double()[:, None]) & (at < count)).sum(-1, keepdim=True).clamp(min=1)
    n = torch.where(greedy, 1, torch.minimum(n2, n3))
    mass = total.gather(-1, n - 1)
    pick = ((total <= s["uniform"].double()[:, None] * mass) & (at < n)).sum(-1, keepdim=True)
    pick = torch.minimum(pick, n - 1)
    return {"tokens": order.gather(-1, pick)[:, 0].int(), "probs": (weight.gather(-1, pick) / mass)[:, 0].float()}


# ------------------------------------------------------------------------------------------ the library's calls
def _handle(s):
    """The cache's handle, which a program keeps."""
    if "handle" not in s:
        from loken_amd import kv
        s["handle"] = kv.KvCacheQ8(s["k"], s["v"], s["k_scales"], s["v_scales"])
    return s["handle"]


def _plan_own(s):
    from loken_amd import kv
    if "plan" not in s:
        s["plan"] = kv.KvPlan(s["case"]["seqs"], s["rows"], s["table"].device)
    p = kv.kv_plan(s["past"], s["fresh"], s["table"], s["free"], s["case"]["page"], s["plan"], taken=s["taken"])
    return {"table": s["table"], "lens": p.lens, "starts": p.starts, "slots": p.slots, "positions": p.positions, "taken": p.taken}


def _store_own(s):
    from loken_amd import kv
    cache = _handle(s)
    kv.kv_write(cache, s["new_k"], s["new_v"], s["slots"])
    k, v = kv.kv_read(cache, s["read"], dtype=s["new_k"].dtype)
    return {"k": k, "k_scales": s["k_scales"], "v": v, "v_scales": s["v_scales"]}


def _attend_own(s):
    from loken_amd import kv
    return kv.kv_attention(s["q"], _handle(s), s["table"], s["lens"], s["starts"], max_fresh=s["max_fresh"], max_len=s["max_len"],
                           window=s["case"]["window"], out=s["out"])


def _sample_own(s):
    from loken_amd import sampling
    tokens, probs = sampling.sample(s["logits"], s["uniform"], s["temperature"], s["top_k"], s["top_p"], s["min_p"])
    return {"tokens": tokens, "probs": probs}


def run(state):
    kind = state["case"]["kind"]
    if own:
        return {"plan": _plan_own, "store": _store_own, "attend": _attend_own, "sample": _sample_own}[kind](state)
    return {"plan": _plan_plain, "store": _store_plain, "attend": _attend_plain, "sample": _sample_plain}[kind](state)


# ------------------------------------------------------------------------------------------ in 64 bits, from the definitions
def exact(case, seed):
    s = prepare(case, seed)
    return {"plan": _plan_exact, "store": _store_exact, "attend": _attend_exact, "sample": _sample_exact}[case["kind"]](s)


def _plan_exact(s):
    page, table, free = s["case"]["page"], s["table"].cpu(), s["free"].tolist()
    past, fresh, taken = s["past"].tolist(), s["fresh"].tolist(), int(s["taken"])
    slots, positions, starts = [], [], [0]
    for i, (p, f) in enumerate(zip(past, fresh)):
        for col in range(-(-p // page), -(-(p + f) // page)):
            table[i, col] = free[taken] if taken < len(free) else -1
            taken += 1
        for pos in range(p, p + f):
            entry = int(table[i, pos // page])
            slots.append(entry * page + pos % page if entry >= 0 else -1)
            positions.append(pos)
        starts.append(starts[-1] + f)
    pad = s["rows"] - len(slots)
    i32 = torch.int32
    return {"table": table, "lens": torch.tensor([p + f for p, f in zip(past, fresh)], dtype=i32), "starts": torch.tensor(starts, dtype=i32),
            "slots": torch.tensor(slots + [-1] * pad), "positions": torch.tensor(positions + [0] * pad, dtype=i32),
            "taken": torch.tensor([taken], dtype=i32)}


def _store_exact(s):
    page, out = s["case"]["page"], {}
    slots = s["slots"].cpu()
    for side in ("k", "v"):
        scales = s[side + "_scales"].cpu()
        codes = s[side].cpu().double()
        if side == "v":
            codes = codes.transpose(-1, -2).flatten(2, 3)
        new = s["new_" + side].cpu().double()
        for p in torch.unique(slots // page).tolist():
            mine = (slots // page == p).nonzero()[:, 0]
            places = slots[mine] % page
            old = torch.zeros_like(scales[p]) if bool((places == 0).any()) else scales[p]
            # the scale is a 32-bit number: the larger of the old one and a 127th of the largest new value
            scale = torch.maximum(old, (new[mine].abs().amax((0, 2)) / 127.0).float())
            part = codes[p] * old.double()[:, None, None] / scale.double()[:, None, None]
            part[:, places] = (new[mine] / scale.double()[None, :, None]).transpose(0, 1)
            codes[p] = torch.sign(part) * torch.floor(part.abs() + 0.5)
            scales[p] = scale
        read = s["read"].cpu()
        out[side] = codes[read // page, :, read % page] * scales.double()[read // page][:, :, None]
        out[side + "_scales"] = scales.double()
    return out


def _attend_exact(s):
    case = s["case"]
    heads, kv_heads, dim = HEADS[case["heads"]]
    page, window = case["page"], case["window"]
    lens, starts = s["lens"].tolist(), s["starts"].tolist()
    out = torch.zeros((s["tokens"], heads, dim), dtype=torch.float64, device=DEV)
    for i, length in enumerate(lens):
        ids = s["table"][i, :-(-length // page)].long()
        k = (s["k"][ids].double() * s["k_scales"][ids].double()[:, :, None, None]).permute(0, 2, 1, 3).reshape(-1, kv_heads, dim)[:length]
        v = (s["v"][ids].double() * s["v_scales"][ids].double()[:, :, None, None, None]).permute(0, 2, 4, 1, 3).reshape(-1, kv_heads, dim)[:length]
        a, b = starts[i], starts[i + 1]
        pos = torch.arange(length - (b - a), length, device=DEV)[:, None]
        at = torch.arange(length, device=DEV)[None]
        hidden = (at > pos) | ((at <= pos - window) if window else (at < 0))
        for h in range(heads):
            kh, vh = k[:, h // (heads // kv_heads)], v[:, h // (heads // kv_heads)]
            z = (s["q"][a:b, h].double() @ kh.T.contiguous()) / math.sqrt(dim)
            out[a:b, h] = torch.softmax(z.masked_fill(hidden, -math.inf), -1) @ vh.contiguous()
    return out


def _sample_exact(s):
    tokens, probs = [], []
    ask = zip(*(s[name].tolist() for name in ("temperature", "top_k", "top_p", "min_p", "uniform")))
    for row, (temperature, top_k, top_p, min_p, uniform) in zip(s["logits"], ask):
        x = row.double()
        order = torch.argsort(x, descending=True, stable=True)
        order = order[x[order] > -math.inf]
        if temperature <= 0:
            tokens.append(int(order[0]))
            probs.append(1.0)
            continue
        w = torch.exp((x[order] - x[order[0]]) / temperature)
        kept = w[:top_k] if top_k > 0 else w
        if top_p < 1:
            sums = torch.cumsum(kept, 0)
            kept = kept[:int((sums < top_p * sums[-1]).sum()) + 1]
        kept = kept[:max(1, int((w >= min_p).sum()))]
        sums = torch.cumsum(kept, 0)
        i = min(int((sums <= uniform * sums[-1]).sum()), kept.numel() - 1)
        tokens.append(int(order[i]))
        probs.append(float(kept[i] / sums[-1]))
    return {"tokens": torch.tensor(tokens, dtype=torch.int32), "probs": torch.tensor(probs, dtype=torch.float64)}


# ------------------------------------------------------------------------------------------ what a pass needs
def work(case):
    if case["kind"] == "sample":
        n = case["rows"] * case["vocab"]
        return {"bytes": n * SIZES[case["type"]] + 28.0 * case["rows"], "flops": 4.0 * n}
    past, fresh = _lengths(case)
    tokens, page = sum(fresh), case["page"]
    if case["kind"] == "plan":
        new_pages = sum(-(-(p + f) // page) - -(-p // page) for p, f in zip(past, fresh))
        return {"bytes": 16.0 * case["seqs"] + 8.0 * new_pages + 12.0 * (-(-tokens // 64) * 64), "flops": 4.0 * tokens}
    heads, kv_heads, dim = HEADS[case["heads"]]
    size = SIZES[case["type"]]
    if case["kind"] == "store":
        touched = sum(-(-(p + f) // page) - p // page for p, f in zip(past, fresh)) * page
        # the new rows in, their pages written, and read back as values
        return {"bytes": 2.0 * kv_heads * dim * (tokens * size + touched * (2 + size)), "flops": 2.0 * kv_heads * dim * (4 * tokens + touched)}
    window = case["window"] or 1 << 40
    cached = sum(min(p + f, f - 1 + window) for p, f in zip(past, fresh))
    pairs = sum(sum(min(p + j + 1, window) for j in range(f)) for p, f in zip(past, fresh))
    return {"bytes": 2.0 * kv_heads * cached * (dim + 4.0 / page) + 2.0 * tokens * heads * dim * size, "flops": 4.0 * heads * dim * pairs}
