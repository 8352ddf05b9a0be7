"""A served step's operators one after the other, as a decode loop uses them between its quantized linears: eagerly, recorded,
on streams of their own, and where the tensors are larger than 32-bit offsets."""
import json
from types import SimpleNamespace

import numpy as np
import pytest

torch = pytest.importorskip("torch")

import serving_reference as ref
from loken_amd import kv, lib, ops, sampling, synth, workloads
from test_gpu_graph_scratch import check_replays, record
from test_gpu_kv_attention import Batch, i32
from test_gpu_kv_cache import check_cache

pytestmark = pytest.mark.gpu

HEADS, KV_HEADS, DIM, PAGE, PAGES, VOCAB, SEQS, MOST = 4, 2, 64, 16, 12, 1003, 3, 64
HIDDEN = HEADS * DIM


def dev(a):
    return torch.tensor(np.ascontiguousarray(a), device="cuda")


class Loop:
    """Sequences of a small layer with quantized linears: x -> q, k, v -> cache -> attention -> logits -> the next x."""

    def __init__(self, seed):
        g = np.random.default_rng(seed)
        self.weights = [dev(synth.weight(lib.TYPE_Q8_0, n, HIDDEN, seed=seed, stream=i)) for i, n in enumerate((HIDDEN, KV_HEADS * DIM, KV_HEADS * DIM, VOCAB))]
        self.words = dev(g.normal(size=(VOCAB, HIDDEN)).astype(np.float32))
        self.cache = kv.KvCacheQ8.empty(PAGES, KV_HEADS, DIM, PAGE)
        self.free = g.permutation(PAGES).astype(np.int32)
        self.state(np.zeros(SEQS, np.int32), np.full((SEQS, MOST // PAGE), -1, np.int32))
        self.rules = [dev(a) for a in (np.full(SEQS, 0.9, np.float32), np.array([0, 40, 7], np.int32), np.array([0.9, 1.0, 0.95], np.float32))]
        self.drawn = dev(g.random((64, SEQS)).astype(np.float32))
        self.u = torch.empty(SEQS, device="cuda")

    def state(self, past, table):
        self.past, self.table, self.taken = i32(past), i32(table), i32([0])
        self.free_pages = i32(self.free)

    def step(self, x, fresh, plan, last):
        """`last`: the row of each sequence that has its last token."""
        kv.kv_plan(self.past, fresh, self.table, self.free_pages, PAGE, plan, self.taken)
        q, k, v = ops.mmvq_fused(lib.TYPE_Q8_0, self.weights[:3], x, [w for w in (HIDDEN, KV_HEADS * DIM, KV_HEADS * DIM)])
        q, k, v = q.view(-1, HEADS, DIM), k.unflatten(1, (KV_HEADS, DIM)), v.unflatten(1, (KV_HEADS, DIM))
        kv.kv_write(self.cache, k, v, plan.slots)
        out = kv.kv_attention(q, self.cache, self.table, plan.lens, plan.starts, max_fresh=4, max_len=MOST)
        logits = ops.mmvq_fused(lib.TYPE_Q8_0, self.weights[3:], out[last].view(-1, HIDDEN), [VOCAB])[0]
        tokens, probs = sampling.sample(logits, self.u, *self.rules)
        return q, k, v, out, logits, tokens, probs

    def after(self, plan):
        self.past.copy_(plan.lens)
        self.taken.copy_(plan.taken)


def test_a_loop_of_steps():
    loop = Loop(3)
    want, table, past, taken = ref.Cache(PAGES, KV_HEADS, PAGE, DIM), np.full((SEQS, MOST // PAGE), -1, np.int32), np.zeros(SEQS, np.int32), 0
    x = loop.words[torch.arange(8, device="cuda")].clone()
    rules = [r.cpu().numpy() for r in loop.rules]
    for n in range(20):
        fresh = np.array([4, 1, 3] if n == 0 else [1, 1, 1], np.int32)
        rows, last = int(fresh.sum()), np.cumsum(fresh) - 1
        plan = kv.KvPlan(SEQS, rows)
        loop.u.copy_(loop.drawn[n])
        q, k, v, out, logits, tokens, probs = loop.step(x[:rows], i32(fresh), plan, torch.tensor(last, device="cuda"))
        table, lens, starts, slots, positions, taken = ref.plan(past, fresh, table, loop.free, PAGE, rows, taken)
        for got, w in zip((loop.table, plan.lens, plan.starts, plan.slots, plan.positions, plan.taken), (table, lens, starts, slots, positions, [taken])):
            assert np.array_equal(got.cpu().numpy(), w), n
        want.write(k.cpu().numpy(), v.cpu().numpy(), slots)
        check_cache(loop.cache, want)
        rk, rv = kv.kv_read(loop.cache, plan.slots)
        for side, got in (("k", rk), ("v", rv)):
            values = np.stack([want.values(side, s // PAGE)[:, s % PAGE] for s in slots])
            assert np.allclose(got.cpu().numpy(), values, rtol=2.0 ** -23, atol=0)
        qn = q.cpu().numpy()
        exact, reach, most = ref.attention(qn, want, table, lens, starts, DIM ** -0.5, 0, np.zeros(qn.shape))
        # (as for any f32 query: its values to 2^-22, weights to 2^-17 of the largest value, the output's rounding)
        bound = most * (2 * reach * 2.0 ** -22 + 2.0 ** -17 + 2.0 ** -20)
        assert (np.abs(out.double().cpu().numpy() - exact) <= bound[..., None] + 2.0 ** -24 * np.abs(exact)).all(), n
        chosen, share = ref.sample(logits.cpu().numpy(), loop.u.cpu().numpy(), *rules)
        assert np.array_equal(tokens.cpu().numpy(), chosen) and np.allclose(probs.cpu().numpy(), share, rtol=2.0 ** -24 + 1e-9, atol=1e-12)
        loop.after(plan)
        past = lens
        x = loop.words[tokens.long()]
    assert past.max() > PAGE


def test_a_recorded_step_is_the_eager_one():
    """Replays with the loop's own eager work (lengths, the next rows) and a synchronization between them."""
    eager, other = Loop(5), Loop(5)
    one, rows, last = i32([1, 1, 1]), torch.arange(8, device="cuda"), torch.arange(SEQS, device="cuda")
    plans, x = [kv.KvPlan(SEQS, SEQS) for _ in "ab"], torch.empty((SEQS, HIDDEN), device="cuda")
    for loop in (eager, other):
        prompt = kv.KvPlan(SEQS, 8)
        loop.u.copy_(loop.drawn[0])
        tokens = loop.step(loop.words[rows], i32([4, 1, 3]), prompt, torch.tensor([3, 4, 7], device="cuda"))[5]
        loop.after(prompt)
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    graph, got = record(lambda: other.step(x, one, plans[1], last), side)
    for n in range(1, 30):
        here = eager.words[tokens.long()]
        for loop in (eager, other):
            loop.u.copy_(loop.drawn[n])
        x.copy_(here)
        want = eager.step(here, one, plans[0], last)
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(want, got):
            assert torch.equal(a, b), n
        for a, b in zip((eager.cache.k, eager.cache.v, eager.cache.k_scales, eager.cache.v_scales, eager.table, plans[0].slots),
                        (other.cache.k, other.cache.v, other.cache.k_scales, other.cache.v_scales, other.table, plans[1].slots)):
            assert torch.equal(a, b), n
        eager.after(plans[0])
        other.after(plans[1])
        tokens = want[5]


ATTENTION = {"a context in parts": ([9000], [1], "f32", 8, 2), "contexts in pieces": ([4000, 1, 2700, 3000, 9, 5000, 4100, 3900], [1] * 8, "f16", 16, 16),
             "a chunk in parts": ([3000], [40], "bf16", 8, 2), "a chunk beside single rows": ([2500, 2400, 70], [33, 1, 1], "f32", 8, 2)}


@pytest.mark.parametrize("what", sorted(ATTENTION))
def test_recorded_attention_beside_other_calls(what):
    """Graphs and eager calls on streams that nothing orders, in the library's scratch memory."""
    lens, fresh, dtype, heads, kv_heads = ATTENTION[what]

    def call(seed):
        b = Batch(lens, fresh, heads, kv_heads, 64, 32, dtype, seed=seed)
        at = (b.q.cuda(), b.cache(), i32(b.table), i32(b.lens), i32(b.starts))
        return lambda: kv.kv_attention(*at, max_fresh=max(fresh), max_len=max(lens))

    check_replays([call(seed) for seed in (1, 2, 3)], torch.cuda.Stream())


@pytest.mark.parametrize("rows,vocab", [(1, 151936), (40, 32000)])
def test_recorded_sampling_beside_other_calls(rows, vocab):
    def call(seed):
        g = torch.Generator(device="cuda").manual_seed(seed)
        logits, u = torch.randn((rows, vocab), device="cuda", generator=g) * 3, torch.rand(rows, device="cuda", generator=g)
        t, p = torch.full_like(u, 0.9), torch.full_like(u, 0.95)
        return lambda: torch.cat([w.view(torch.int32) for w in sampling.sample(logits, u, t, top_p=p)])

    check_replays([call(seed) for seed in (4, 5, 6)], torch.cuda.Stream())


def test_a_recording_that_no_call_came_before_is_refused():
    """Scratch is not allocated while a graph is recorded: a call that needs some and finds none says so, and the next works."""
    b = Batch([9000], [1], 8, 2, 64, 32, "f32", seed=8)
    at = (b.q.cuda(), b.cache(), i32(b.table), i32(b.lens), i32(b.starts))
    x, u = torch.randn((2, 32000), device="cuda"), torch.rand(2, device="cuda")
    calls = [lambda: kv.kv_attention(*at, max_fresh=1, max_len=9000), lambda: sampling.sample(x, u, u)]
    torch.cuda.synchronize()
    lib.load().loken_stream_scratch_release()
    for call in calls:
        side, graph, refused = torch.cuda.Stream(), torch.cuda.CUDAGraph(), []
        with torch.cuda.stream(side):
            with torch.cuda.graph(graph, stream=side):
                try:
                    call()
                except lib.LokenError as err:
                    refused.append(str(err))
        assert refused and "LK_ERR_NOMEM" in refused[0]
        call()
    b.check()


def test_calls_on_a_stream_of_their_own():
    """Nothing of a call goes to another stream than the current one."""
    b = Batch([3000, 700, 5], [1, 30, 5], 8, 2, 128, 16, "f16", seed=9)
    x, u = torch.randn((5, 50000), device="cuda"), torch.rand(5, device="cuda")
    want, drawn = b.check(), sampling.sample(x, u, u)
    side, q, cache = torch.cuda.Stream(), b.q.cuda(), b.cache()
    table, lens, starts = i32(b.table), i32(b.lens), i32(b.starts)
    late, wait = torch.zeros_like(q), torch.empty(1 << 28, device="cuda")
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        for _ in range(4):
            wait.fill_(1.0)          # what the calls' input waits for, on their stream alone
        late.copy_(q)
        out = kv.kv_attention(late, cache, table, lens, starts, max_fresh=30, max_len=3000)
        tokens, probs = sampling.sample(x, u, u)
    side.synchronize()
    assert torch.equal(out, want) and torch.equal(tokens, drawn[0]) and torch.equal(probs, drawn[1])


def test_rows_behind_2_to_the_31_values():
    stride, vocab = (1 << 30) + 8, 5003
    wide = torch.empty(2 * stride + 8192, dtype=torch.bfloat16, device="cuda")
    near = (torch.randn((3, vocab), device="cuda") * 3).to(torch.bfloat16)
    far = wide.as_strided((3, vocab), (stride, 1))
    far.copy_(near)
    u = torch.rand(3, device="cuda")
    for a, b in zip(sampling.sample(near, u, u + 0.5), sampling.sample(far, u, u + 0.5)):
        assert torch.equal(a, b)
    for fresh in (3, 20):   # the kernel of a few rows and the one of many
        b = Batch([200], [fresh], 4, 1, 64, 16, "bf16", seed=10)
        q, at = b.q.cuda(), (b.cache(), i32(b.table), i32(b.lens), i32(b.starts))
        across = 2 * stride // (fresh - 1) // 8 * 8
        q_far = wide.as_strided(q.shape, (across, 64, 1))
        q_far.copy_(q)
        want = kv.kv_attention(q, *at, max_fresh=fresh, max_len=200)
        assert torch.equal(kv.kv_attention(q_far, *at, max_fresh=fresh, max_len=200), want)
        kv.kv_attention(q, *at, max_fresh=fresh, max_len=200, out=q_far)
        assert torch.equal(q_far, want)


@pytest.mark.parametrize("batch,context", [(1, 64), (5, 100)])
def test_the_measured_step_with_a_context(batch, context, capsys):
    """The command's plan of launches: every sequence gets a word, and its new row is in the cache."""
    made = []

    class Kept(workloads.Between):
        def __init__(self, *args):
            super().__init__(*args)
            made.append(self)

    args = SimpleNamespace(batch=batch, context=context, mid_rows="auto", acts="f32", steps=1, warmup=1, gpus=1)
    before = workloads.Between
    workloads.Between = Kept
    try:
        assert workloads.decode_1p7b(args, torch.device("cuda", 0)) == 0
    finally:
        workloads.Between = before
    step, result = made[0], json.loads(capsys.readouterr().out)
    assert result["config"]["cache_bytes_per_step"] == 28 * 2 * batch * (context + 1) * 1024
    assert ((step.tokens >= 0) & (step.tokens < 151936)).all() and (step.probs > 0).all()
    assert (step.plan.lens == context + 1).all() and (step.plan.slots >= 0).all() and len(step.caches) == 28
    assert (step.table[:, :context // 64 + 1] >= 0).all()
    k, v = kv.kv_read(step.caches[0], step.plan.slots)
    assert torch.isfinite(k).all() and (k.abs().amax((1, 2)) > 0).all() and (v.abs().amax((1, 2)) > 0).all()
