"""A served step with drafted tokens over the 4-bit cache, operator after operator as a decode loop uses them between its quantized linears:
eagerly against the definitions, and recorded."""
import json
from types import SimpleNamespace

import numpy as np
import pytest

torch = pytest.importorskip("torch")

import mxfp4_reference as ref
import serving_reference as served
from loken_amd import kv, lib, ops, rotary, sampling, synth, workloads
from test_gpu_graph_scratch import record
from test_gpu_kv_attention import i32
from test_gpu_mxfp4_cache import check_cache, dev

pytestmark = pytest.mark.gpu

HEADS, KV_HEADS, DIM, PAGE, PAGES, VOCAB, SEQS, MOST, DRAFTS, CAP = 4, 2, 64, 16, 60, 1003, 3, 128, 3, 30.0
HIDDEN = HEADS * DIM


def linear(weights, x, ns):
    """The mat-vec launch takes up to eight rows."""
    parts = [ops.mmvq_fused(lib.TYPE_Q8_0, weights, x[i:i + 8], ns) for i in range(0, len(x), 8)]
    return [torch.cat(of_one) for of_one in zip(*parts)]


class Loop:
    """Sequences of a small layer with quantized linears: x -> q, k, v -> norms, rotation, cache -> attention -> logits -> the check of the
    drafts, whose number of accepted ones says how far each sequence has come."""

    def __init__(self, seed):
        g = np.random.default_rng(seed)
        sizes = (HIDDEN, KV_HEADS * DIM, KV_HEADS * DIM, VOCAB)
        self.weights = [dev(synth.weight(lib.TYPE_Q8_0, n, HIDDEN, seed=seed, stream=i)) for i, n in enumerate(sizes)]
        self.words = dev(g.normal(size=(VOCAB, HIDDEN)).astype(np.float32))
        self.cache = kv.KvCacheMxfp4.empty(PAGES, KV_HEADS, DIM, PAGE)
        self.frequencies = (10000.0 ** (-np.arange(DIM // 2) / (DIM // 2))).astype(np.float32)
        self.rotary = rotary.Rotary(dev(self.frequencies))
        self.norm = g.uniform(0.5, 1.5, (2, DIM)).astype(np.float32)
        self.q_weight, self.k_weight = dev(self.norm[0]), dev(self.norm[1])
        self.free = g.permutation(PAGES).astype(np.int32)
        self.free_pages, self.table, self.past, self.taken = i32(self.free), i32(np.full((SEQS, MOST // PAGE), -1)), i32([0] * SEQS), i32([0])
        self.draws, self.u = g.random((40, SEQS)).astype(np.float32), g.random((40, SEQS * (DRAFTS + 1))).astype(np.float32)
        self.draw, self.uniform = torch.empty(SEQS, device="cuda"), torch.empty(SEQS * (DRAFTS + 1), device="cuda")
        rows = SEQS * (DRAFTS + 1)
        self.rules = [np.full(rows, 0.9, np.float32), np.tile([0, 40, 7, 0], SEQS).astype(np.int32), np.full(rows, 0.95, np.float32)]
        self.rules_there = [dev(r) for r in self.rules]

    def step(self, x, drafted, share, fresh, plan):
        kv.kv_plan(self.past, fresh, self.table, self.free_pages, PAGE, plan, self.taken)
        q, k, v = linear(self.weights[:3], x, [HIDDEN, KV_HEADS * DIM, KV_HEADS * DIM])
        q, k, v = q.view(-1, HEADS, DIM), k.unflatten(1, (KV_HEADS, DIM)), v.unflatten(1, (KV_HEADS, DIM))
        turned = rotary.rotate_into(self.cache, q, k, v, plan.positions, plan.slots, self.rotary, q_weight=self.q_weight, k_weight=self.k_weight)
        out = kv.kv_attention(turned, self.cache, self.table, plan.lens, plan.starts, max_fresh=DRAFTS + 1, max_len=MOST, softcap=CAP)
        logits = linear(self.weights[3:], out.view(-1, HIDDEN), [VOCAB])[0]
        tokens, accepted, probs = sampling.verify(logits, drafted, plan.starts, self.uniform, self.draw, *self.rules_there, draft=share)
        return q, k, v, turned, out, logits, tokens, accepted, probs

    def after(self, plan, accepted):
        """What was drafted behind the accepted tokens is forgotten: the next step writes over it."""
        self.past.add_(accepted + 1)
        self.taken.copy_(plan.taken)


def bring_drafts(loop, words, x, drafted, share, fresh, plan):
    """Drafts from the layer itself, at a higher temperature, one after the other: a step over what is there so far gives the next one's
    distribution, and the steps after it write over its rows. Its largest word, or in every third sequence another, is drafted."""
    first = torch.arange(SEQS, device="cuda") * (DRAFTS + 1)
    drafted.zero_()
    share.fill_(1.0 / VOCAB)
    x.copy_(loop.words[words.repeat_interleave(DRAFTS + 1).long()])
    for j in range(DRAFTS):
        logits = loop.step(x, drafted, share, fresh, plan)[5][first + j]
        share[first + j] = torch.softmax(logits / 1.5, -1)
        word = logits.argmax(-1)
        word[j % SEQS] = (word[j % SEQS] + 1) % VOCAB
        drafted[first + j] = word.int()
        x[first + j + 1] = loop.words[word]


def test_a_loop_of_drafted_steps():
    loop, g = Loop(3), np.random.default_rng(4)
    want, table = ref.Cache(PAGES, KV_HEADS, PAGE, DIM), np.full((SEQS, MOST // PAGE), -1, np.int32)
    past, taken, rows = np.zeros(SEQS, np.int32), 0, SEQS * (DRAFTS + 1)
    words, fresh, some = dev(np.array([5, 77, 900])), i32([DRAFTS + 1] * SEQS), 0
    x, drafted, share = torch.empty((rows, HIDDEN), device="cuda"), i32([0] * rows), torch.empty((rows, VOCAB), device="cuda")
    for n in range(12):
        plan = kv.KvPlan(SEQS, rows)
        bring_drafts(loop, words, x, drafted, share, fresh, plan)
        loop.draw.copy_(dev(loop.draws[n]))
        loop.uniform.copy_(dev(loop.u[n]))
        q, k, v, turned, out, logits, tokens, accepted, probs = loop.step(x, drafted, share, fresh, plan)
        table, lens, starts, slots, positions, taken = served.plan(past, [DRAFTS + 1] * SEQS, table, loop.free, PAGE, rows, taken)
        for got, w in zip((loop.table, plan.lens, plan.starts, plan.slots, plan.positions, plan.taken), (table, lens, starts, slots, positions, [taken])):
            assert np.array_equal(got.cpu().numpy(), w), n
        kn, vn = k.double().cpu().numpy(), v.double().cpu().numpy()
        want.write(ref.rope(kn, positions, loop.frequencies, None, loop.norm[1]), vn, slots)
        check_cache(loop.cache, want)
        exact_q = ref.rope(q.double().cpu().numpy(), positions, loop.frequencies, None, loop.norm[0])
        size = np.sqrt((exact_q ** 2).max(-1, keepdims=True)) * np.sqrt(2)
        assert (np.abs(turned.double().cpu().numpy() - exact_q) <= 16 * 2.0 ** -24 * size).all(), n      # as for any rows
        exact, reach, most = ref.attention(turned.cpu().numpy(), want, table, lens, starts, DIM ** -0.5, 0, CAP, np.zeros(out.shape))
        score = (3 * DIM + 6) * 2.0 ** -24 * reach + CAP * 2.0 ** -22
        bound = most * (2 * score + 4 * 2.0 ** -22 + 2 * lens.max() * 2.0 ** -24 + 2.0 ** -24)
        assert (np.abs(out.double().cpu().numpy() - exact) <= bound[..., None] + 2.0 ** -24 * np.abs(exact)).all(), n
        chosen, how_many, p = ref.verify(logits.double().cpu().numpy(), drafted.cpu().numpy(), starts, loop.u[n], loop.draws[n], *loop.rules,
                                         draft=share.double().cpu().numpy())
        assert np.array_equal(tokens.cpu().numpy(), chosen) and np.array_equal(accepted.cpu().numpy(), how_many)
        assert np.allclose(probs.double().cpu().numpy(), p, rtol=2.0 ** -24 + 1e-9, atol=1e-11)
        loop.after(plan, accepted)
        past = past + how_many.astype(np.int32) + 1
        some += int(how_many.sum())
        words = dev(chosen[starts[:-1] + how_many])
    assert past.max() > PAGE and 0 < some < 12 * SEQS * DRAFTS and np.array_equal(loop.past.cpu().numpy(), past)


def test_a_recorded_step_is_the_eager_one():
    """Replays with the loop's own eager work (lengths, the next rows and drafts) and a synchronization between them."""
    eager, other = Loop(5), Loop(5)
    rows = SEQS * (DRAFTS + 1)
    fresh, plans = i32([DRAFTS + 1] * SEQS), [kv.KvPlan(SEQS, rows) for _ in "ab"]
    x, drafted, share = torch.empty((rows, HIDDEN), device="cuda"), i32([0] * rows), torch.empty((rows, VOCAB), device="cuda")
    words, first = dev(np.array([5, 77, 900])), torch.arange(SEQS, device="cuda") * (DRAFTS + 1)

    def bring(n):
        bring_drafts(eager, words, x, drafted, share, fresh, plans[0])
        for loop in (eager, other):
            loop.draw.copy_(dev(loop.draws[n]))
            loop.uniform.copy_(dev(loop.u[n]))

    bring(0)
    for loop, plan in zip((eager, other), plans):
        accepted = loop.step(x, drafted, share, fresh, plan)[7]
        loop.after(plan, accepted)
    torch.cuda.synchronize()
    graph, got = record(lambda: other.step(x, drafted, share, fresh, plans[1]), torch.cuda.Stream())
    for n in range(1, 9):
        bring(n)
        want = eager.step(x, drafted, share, fresh, plans[0])
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(want, got):
            assert torch.equal(a, b), n
        for a, b in zip((*eager.cache._tensors, eager.table), (*other.cache._tensors, other.table)):
            assert torch.equal(a, b), n
        words = want[6][first + want[7]]
        eager.after(plans[0], want[7])
        other.after(plans[1], got[7])


@pytest.mark.parametrize("batch,context,drafts", [(1, 64, 0), (6, 100, 2)])
def test_the_measured_step_over_the_4_bit_cache(batch, context, drafts, capsys):
    """bench.py's step: its line, and a layer's attention and the check at its end over what it left."""
    made = []

    class Kept(workloads.BetweenMxfp4):
        def __init__(self, *a):
            super().__init__(*a)
            made.append(self)

        def attention_items(self, q, k, v, out, s):
            wide = self.kv_heads * workloads.HEAD_DIM   # (of rows as wide as the queries')
            self.rows_of = (q, k[:, :wide], v[:, :wide], out.view(self.rows, self.heads, workloads.HEAD_DIM))
            return super().attention_items(q, k, v, out, s)

    args = SimpleNamespace(batch=batch, context=context, kv_cache="mxfp4", drafts=drafts, mid_rows="auto", acts="f32", steps=1, warmup=1, gpus=1)
    before, workloads.BetweenMxfp4 = workloads.BetweenMxfp4, Kept
    try:
        assert workloads.decode_1p7b(args, torch.device("cuda", 0)) == 0
    finally:
        workloads.BetweenMxfp4 = before
    line = json.loads(capsys.readouterr().out.strip().splitlines()[-1])
    between = made[0]
    assert "4 bits" in line["config"]["workload"] and line["config"]["cache_bytes_per_step"] == 28 * between.bytes_read()
    q, k, v, out = between.rows_of
    heads = lambda x: x.unflatten(1, (-1, workloads.HEAD_DIM))  # noqa: E731
    p, turning = between.plan, rotary.Rotary(between.frequencies)
    turned, turned_k = rotary.rotate(heads(q), heads(k), p.positions, turning, q_weight=between.norms[0], k_weight=between.norms[1])
    there = kv.kv_read(between.caches[-1], p.slots)
    for got, rows in zip(there, (turned_k, heads(v))):      # (a key's code may be the border's other one: 64 bits there, 32 here)
        want = torch.tensor(ref.values(*ref.quantize(rows.double().cpu().numpy())))
        assert (got.double().cpu() != want).double().mean() < 1e-3
    exact = kv.kv_attention(turned, between.caches[-1], between.table, p.lens, p.starts, max_fresh=drafts + 1, max_len=context + drafts + 1)
    assert torch.allclose(out, exact, rtol=1e-4, atol=1e-4)
    if drafts:
        assert ((between.accepted >= 0) & (between.accepted <= drafts)).all()
        first = p.starts[:-1].long() + between.accepted
        assert (between.tokens[first] >= 0).all() and (between.probs[first] > 0).all()


def test_two_streams_at_once():
    """Cut contexts, prompts and checks of drafts whose workspaces are their stream's, in turn on two streams."""
    from test_gpu_mxfp4_attention import Batch
    from test_gpu_verify import Drafts
    calls = []
    for seed, lens, fresh, heads in ((1, [9000, 40], [1, 1], (8, 2)), (2, [600, 900, 70], [90, 300, 2], (4, 4)), (3, [5000], [4], (4, 1))):
        b = Batch(lens, fresh, *heads, 128, 16, "bf16", seed=seed)
        at = b.q.cuda(), b.cache(), i32(b.table), i32(b.lens), i32(b.starts)
        calls.append(lambda at=at, fresh=fresh, lens=lens: kv.kv_attention(*at, max_fresh=max(fresh), max_len=max(lens)))
        d = Drafts([5, 1, 3], 20011, seed=seed)
        given = dict(logits=d.logits.cuda(), drafted=dev(d.drafted), starts=dev(d.starts), uniform=dev(d.uniform), draw=dev(d.draw), temperature=dev(d.temperature),
                     top_k=dev(d.top_k), top_p=dev(d.top_p), min_p=dev(d.min_p), draft=d.draft.cuda())
        calls.append(lambda given=given: torch.cat([t.double() for t in sampling.verify(**given)]))
    want = [call() for call in calls]
    torch.cuda.synchronize()
    sides, got = [torch.cuda.Stream(), torch.cuda.Stream()], []
    for turn in range(3):
        for i in range(len(calls)):
            for j, side in enumerate(sides):
                with torch.cuda.stream(side):
                    at = (i + j * (turn + 1)) % len(calls)
                    got.append((at, calls[at]()))
    torch.cuda.synchronize()
    for at, out in got:
        assert torch.equal(out, want[at])


def test_pages_of_refused_drafts_go_back_to_the_list():
    """A recorded step and what follows its check, recorded too and without a look at the device: the pages that refused drafts alone had are the
    next ones to be given, so that a loop in a cache of as many pages as its tokens need comes through."""
    loop = Loop(6)
    rows, pages = SEQS * (DRAFTS + 1), SEQS * (MOST // PAGE)
    free = torch.cat([loop.free_pages[:pages], i32([-1])])      # one place behind the list, for what is not given back
    loop.free_pages = free[:pages]
    fresh, plan = i32([DRAFTS + 1] * SEQS), kv.KvPlan(SEQS, rows)
    x, drafted, share = torch.empty((rows, HIDDEN), device="cuda"), i32([0] * rows), torch.empty((rows, VOCAB), device="cuda")
    cols, words = torch.arange(MOST // PAGE, device="cuda"), dev(np.array([5, 77, 900]))
    first = torch.arange(SEQS, device="cuda") * (DRAFTS + 1)

    def give_back(accepted):
        loop.past.add_(accepted + 1)
        back = (cols >= ((loop.past + PAGE - 1) // PAGE)[:, None]) & (cols < ((plan.lens + PAGE - 1) // PAGE)[:, None])
        up_to = back.flatten().long().cumsum(0)
        loop.taken.copy_(plan.taken - up_to[-1])
        place = torch.where(back.flatten(), loop.taken + up_to - 1, pages)
        free.scatter_(0, place, loop.table.flatten())

    def step():
        out = loop.step(x, drafted, share, fresh, plan)
        give_back(out[7])
        return out

    def bring(n):
        x.copy_(loop.words[words.repeat_interleave(DRAFTS + 1).long()])
        share.fill_(1.0 / VOCAB)
        drafted.copy_(dev(np.random.default_rng(n).integers(0, VOCAB, rows).astype(np.int32)))
        loop.draw.copy_(dev(loop.draws[n]))
        loop.uniform.copy_(dev(loop.u[n]))

    bring(0)
    step()
    torch.cuda.synchronize()
    graph, got = record(step, torch.cuda.Stream())
    refused = 0
    for n in range(1, 40):
        past, table, list_before, taken = (t.cpu().numpy().copy() for t in (loop.past, loop.table, free, loop.taken))
        bring(n)
        graph.replay()
        torch.cuda.synchronize()
        want, lens, *_ , after = served.plan(past, [DRAFTS + 1] * SEQS, table, list_before[:pages], PAGE, rows, int(taken[0]))
        assert np.array_equal(loop.table.cpu().numpy(), want), n
        past = past + got[7].cpu().numpy() + 1
        assert np.array_equal(loop.past.cpu().numpy(), past), n
        held = [int(e) for i in range(SEQS) for e in want[i, :-(-int(past[i]) // PAGE)]]
        left = free[int(loop.taken):pages].tolist()
        assert sorted(held + left) == sorted(loop.free[:pages].tolist()), n      # each page once
        refused += after - int(loop.taken)
        words = got[6][first + got[7]]
    assert refused > 3 and past.max() > PAGE
