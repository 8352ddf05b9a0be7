"""The check of drafted tokens against its definition in 64 bits: accepted numbers and tokens equal, probabilities to their rounding."""
import numpy as np
import pytest

torch = pytest.importorskip("torch")

import mxfp4_reference as ref
from loken_amd import sampling
from test_gpu_graph_scratch import check_replays

pytestmark = pytest.mark.gpu

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
RULES = [(1.0, 0, 1.0, 0.0), (0.7, 50, 0.9, 0.0), (0.0, 0, 1.0, 0.0), (0.7, 40, 0.95, 0.05), (1.0, 0, 0.92, 0.0), (1.3, 0, 1.0, 0.02), (0.9, 1000, 1.0, 0.0),
         (2.0, 5, 0.5, 0.3), (1.0, 3000, 0.99, 0.0)]


def dev(a, dtype=None):
    t = torch.tensor(np.ascontiguousarray(a))
    return (t if dtype is None else t.to(dtype)).cuda()


class Drafts:
    """Sequences' drafts from a view of the target's logits that is a little off."""

    def __init__(self, lengths, vocab, dtype="f32", draft="f32", rules=RULES, seed=0, pad=0, off=0.5):
        g = np.random.default_rng(seed)
        self.starts = np.concatenate([[0], np.cumsum(lengths)]).astype(np.int32)
        rows = self.rows = int(self.starts[-1]) + pad
        x = g.normal(size=(rows, vocab)) * 3
        x[np.arange(rows)[:, None], g.integers(0, vocab, (rows, 5))] += 8
        self.logits = torch.tensor(x, dtype=torch.float32).to(TYPES[dtype])
        ask = [rules[g.integers(len(rules))] for _ in lengths]
        ask = [a for a, n in zip(ask, lengths) for _ in range(n)] + [(1.0, 0, 1.0, 0.0)] * pad
        self.temperature, self.top_k, self.top_p, self.min_p = (np.array([a[i] for a in ask], np.int32 if i == 1 else np.float32) for i in range(4))
        seen = x + g.normal(size=x.shape) * off
        q = np.exp((seen - seen.max(-1, keepdims=True)) / np.maximum(self.temperature, 0.2)[:, None])
        q /= q.sum(-1, keepdims=True)
        if draft:
            self.drafted = np.array([g.choice(vocab, p=row) for row in q] or [], np.int32)
            self.draft = torch.tensor(q, dtype=torch.float32).to(TYPES[draft])
        else:
            self.drafted, self.draft = q.argmax(-1).astype(np.int32) if rows else np.zeros(0, np.int32), None
        self.uniform, self.draw = g.random(rows).astype(np.float32), g.random(len(lengths)).astype(np.float32)

    def call(self, **change):
        a = dict(logits=self.logits.cuda(), drafted=dev(self.drafted), starts=dev(self.starts), uniform=dev(self.uniform), draw=dev(self.draw),
                 temperature=dev(self.temperature), top_k=dev(self.top_k), top_p=dev(self.top_p), min_p=dev(self.min_p),
                 draft=None if self.draft is None else self.draft.cuda())
        a.update(change)
        return sampling.verify(**a)

    def want(self):
        return ref.verify(self.logits.double().numpy(), self.drafted, self.starts, self.uniform, self.draw, self.temperature, self.top_k, self.top_p,
                          self.min_p, None if self.draft is None else self.draft.double().numpy())

    def check(self, **change):
        got, want = self.call(**change), self.want()
        assert np.array_equal(got[1].cpu().numpy(), want[1])
        assert np.array_equal(got[0].cpu().numpy(), want[0])
        # weights to 2e-13 and a step of 2^-42 each, rounded to f32: half a step
        assert np.allclose(got[2].double().cpu().numpy(), want[2], rtol=2.0 ** -24 + 1e-9, atol=1e-11)
        return got


@pytest.mark.parametrize("dtype", sorted(TYPES))
@pytest.mark.parametrize("draft", ["f32", "f16", "bf16", None])
@pytest.mark.parametrize("vocab", [7, 1003, 4096, 20011])
def test_drafts(vocab, draft, dtype):
    Drafts([5, 1, 2, 9, 5, 3, 1, 4], vocab, dtype, draft, seed=vocab).check()


@pytest.mark.parametrize("rule", RULES)
def test_each_rule(rule):
    for draft in ("f32", None):
        Drafts([4] * 6, 5003, "f32", draft, [rule], seed=int(rule[0] * 10) + rule[1]).check()


def test_many_drafts_of_a_sequence():
    """More than a wave has lanes, all of them good, the last one not, and one in the middle."""
    d = Drafts([150, 70, 3], 257, "f32", "f32", [(1.0, 0, 1.0, 0.0)], seed=3, off=0.0)
    d.uniform[:] = 0
    got = d.check()
    assert got[1].tolist() == [149, 69, 2]
    d.uniform[[148, 150 + 66]] = 0.999
    d.draft[148], d.draft[150 + 66] = 1, 1
    got = d.check()
    assert got[1].tolist() == [148, 66, 2]


def test_every_word_equal():
    """Ties everywhere, more equal words than are sorted at once, and rules that cut within them."""
    d = Drafts([3] * 4, 9000, "f32", "f32", [(1.0, 0, 1.0, 0.0)], seed=5)
    d.logits[:] = 1.5
    d.top_k[:] = np.repeat([0, 7, 5000, 0], 3)
    d.top_p[:] = np.repeat([1.0, 1.0, 0.5, 0.3], 3).astype(np.float32)
    d.draft[:] = 1 / 9000
    d.drafted[:] = np.repeat([8999, 3, 2400, 2600], 3)
    d.uniform[:] = 0.7
    d.check()


def test_nothing_is_left():
    """A draft's share that is nowhere below the target's, refused: the next token is drawn from the target's as it is; and the same for certain."""
    d = Drafts([2, 2, 2], 3001, "f32", "f32", [(1.0, 0, 1.0, 0.0), (1.0, 9, 1.0, 0.0)], seed=6)
    d.draft[:] = 1.0
    d.uniform[:] = 0.9999
    got = d.check()
    assert got[1].tolist() == [0, 0, 0] and (got[0][[0, 2, 4]] >= 0).all()
    d.draft, d.temperature[:] = None, 0.0        # one word is all there is: drafted for certain it is accepted, another is refused
    d.drafted[:] = d.logits.argmax(-1).numpy()
    assert d.check()[1].tolist() == [1, 1, 1]
    d.drafted[:] = (d.drafted + 1) % 3001
    assert d.check()[1].tolist() == [0, 0, 0]


def test_rows_with_few_words_or_none():
    d = Drafts([3] * 6, 2050, "f32", "f32", [(1.0, 0, 1.0, 0.0), (0.8, 40, 0.9, 0.01), (0.0, 0, 1.0, 0.0)], seed=7)
    inf = float("inf")
    d.logits[0:3] = -inf                        # no words
    d.logits[3:6] = -inf
    d.logits[3:6, 77] = 3.0                     # one
    d.drafted[3:6] = 77
    d.logits[6, ::2] = float("nan")
    d.logits[9, [5, 900]] = inf                 # two infinite ones: half each
    d.drafted[9], d.uniform[9], d.draft[9] = 900, 0.3, 0.0
    d.draft[9, 900] = 1.0
    d.logits[12:15] = -inf
    d.logits[12:15, 3:6] = -4.0
    d.uniform[3:6] = 0.2
    got = d.check()
    assert got[0][:3].tolist() == [-1, -1, -1] and got[1][0] == 0


@pytest.mark.parametrize("share", [-1.0, -1e30, float("-inf"), float("inf"), float("nan")])
def test_shares_that_are_none_leave_the_calls_rows_in_bounds(share):
    """What a draft that is no distribution gives is not defined, but it is a word or none, and other sequences' are theirs."""
    d = Drafts([3, 4, 2], 5003, "f32", "f32", [(1.0, 0, 1.0, 0.0), (1.0, 9, 1.0, 0.0)], seed=6)
    d.uniform[3:6] = 1.0 - 2.0 ** -24
    want = d.call()
    d.draft[3:6, 1::2] = share
    tokens, accepted, _ = d.call()
    assert 0 <= int(accepted[1]) <= 3 and (tokens >= -1).all() and (tokens < 5003).all()
    assert torch.equal(tokens[[0, 1, 2, 7, 8]], want[0][[0, 1, 2, 7, 8]]) and torch.equal(accepted[[0, 2]], want[1][[0, 2]])


def test_words_outside_the_vocabulary_are_refused():
    for draft in ("f32", None):
        d = Drafts([3, 3, 3], 1000, "f32", draft, seed=8)
        d.drafted[0], d.drafted[4], d.uniform[3] = -1, 1000, 0.0
        d.drafted[[2, 5, 8]] = [1 << 30, -(1 << 31), 5]      # last rows': not looked at
        got = d.check()
        assert got[1][0] == 0 and got[1][1] <= 1


@pytest.mark.parametrize("draft", ["f32", None])
def test_empty_sequences_and_rows_of_none(draft):
    d = Drafts([0, 3, 0, 1, 0], 1000, "f32", draft, seed=9, pad=5)
    got = d.check()
    assert (got[0][4:] == -1).all() and (got[2][4:] == 0).all()
    none = Drafts([], 100, "f32", draft, pad=2)
    got = none.call()
    assert got[0].tolist() == [-1, -1] and got[1].numel() == 0
    empty = Drafts([0, 0], 100, "f32", draft)
    assert empty.call()[1].tolist() == [0, 0]


def test_rules_may_be_left_out():
    d = Drafts([4, 4], 3000, "f32", "bf16", [(0.8, 0, 1.0, 0.0)], seed=10)
    whole = d.check()
    for a, b in zip(whole, d.call(top_k=None, top_p=None, min_p=None)):
        assert torch.equal(a, b)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_a_large_vocabulary_in_pieces(dtype):
    Drafts([5, 3], 151936, dtype, "bf16", seed=11).check()
    Drafts([1], 262144, dtype, None, [(1.0, 0, 0.95, 0.0)], seed=12).check()


def test_rows_of_wider_tensors():
    d = Drafts([3, 2], 501, "f16", "f16", seed=13)
    want = d.check()
    wide = torch.full((d.rows, 777), 50.0, dtype=torch.float16, device="cuda")
    wide[:, 3:504] = d.logits.cuda()
    shares = torch.full((d.rows, 600), 1.0, dtype=torch.float16, device="cuda")
    shares[:, 7:508] = d.draft.cuda()
    for a, b in zip(want, d.call(logits=wide[:, 3:504], draft=shares[:, 7:508])):
        assert torch.equal(a, b)


def test_accepted_as_often_as_the_target_says():
    """The tokens that come out are the target's: 4000 first tokens of a small vocabulary, drafted from another distribution."""
    g = np.random.default_rng(14)
    n, vocab = 4000, 6
    p, q = np.array([0.4, 0.05, 0.2, 0.1, 0.2, 0.05]), np.array([0.1, 0.3, 0.2, 0.3, 0.05, 0.05])
    d = Drafts([2] * 8, vocab, seed=14)
    rows = 2 * n
    logits, draft = np.tile(np.log(p), (rows, 1)).astype(np.float32), np.tile(q, (rows, 1)).astype(np.float32)
    one = np.ones(rows, np.float32)
    tokens = sampling.verify(dev(logits), dev(g.choice(vocab, rows, p=q).astype(np.int32)), dev(2 * np.arange(n + 1, dtype=np.int32)),
                             dev(g.random(rows).astype(np.float32)), dev(g.random(n).astype(np.float32)), dev(one), draft=dev(draft))[0]
    share = np.bincount(tokens.cpu().numpy()[0::2], minlength=vocab) / n
    # five deviations of a share of n draws
    assert (np.abs(share - p) <= 5 * np.sqrt(p * (1 - p) / n)).all()


@pytest.mark.parametrize("draft", ["f32", None])
def test_recorded_beside_other_calls(draft):
    def call(seed):
        d = Drafts([5, 1, 3], 30011, "f32", draft, seed=seed)
        at = dict(logits=d.logits.cuda(), drafted=dev(d.drafted), starts=dev(d.starts), uniform=dev(d.uniform), draw=dev(d.draw),
                  temperature=dev(d.temperature), top_k=dev(d.top_k), top_p=dev(d.top_p), min_p=dev(d.min_p),
                  draft=None if draft is None else d.draft.cuda())
        return lambda: torch.cat([t.double() for t in sampling.verify(**at)])

    check_replays([call(seed) for seed in (1, 2, 3)], torch.cuda.Stream())


FLOORS = [(1.0, 0, 1.0, 1.0), (1.0, 0, 1.0, 2.0), (0.7, 0, 0.9, 2.0), (0.9, 20, 1.0, 1.5), (1.1, 20, 0.95, 1.0), (1.0, 3000, 0.99, 3.0), (0.0, 0, 1.0, 2.0)]


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("draft", ["f32", None])
@pytest.mark.parametrize("rule", FLOORS)
def test_the_first_word_always_stays(rule, draft, dtype):
    """min_p of 1 and above leaves the first word (of 1: and those that are equal to it), which is then all of the distribution."""
    d = Drafts([4, 1, 3, 5], 30011, dtype, draft, [rule], seed=21)
    d.logits[5, [7, 20000, 30010]] = 40.0     # equal ones
    got = d.check()
    first = d.starts[:-1] + got[1].cpu().numpy()
    assert (got[0].cpu().numpy()[first] >= 0).all() and (got[2].cpu().numpy()[first] > 0).all()


@pytest.mark.parametrize("dtype", sorted(TYPES))
@pytest.mark.parametrize("draft", ["f32", None])
def test_many_rows_in_several_pieces(draft, dtype):
    """Rows enough for pieces of sixteen words a thread, the last of them a part of one, every rule, and largest words that are equal across pieces."""
    lengths = np.random.default_rng(30).integers(1, 6, 100)
    d = Drafts(list(lengths), 16411, dtype, draft, RULES + FLOORS, seed=31)
    assert d.rows * 3 >= 512
    d.logits[::3, [17, 4100, 8200, 16410]] = 30.0
    d.logits[1::9, 16408:] = 31.0
    d.check()


@pytest.mark.parametrize("vocab", [1 << 20, (1 << 20) - 3, 300007])
@pytest.mark.parametrize("draft", ["bf16", None])
@pytest.mark.parametrize("rule", [(1.0, 0, 1.0, 0.0), (0.8, 50, 1.0, 0.0), (0.8, 20, 0.9, 0.0), (1.0, 0, 0.95, 0.0)])
def test_the_largest_vocabularies(rule, draft, vocab):
    for lengths in ([1], [2, 1]):
        d = Drafts(lengths, vocab, "f32", draft, [rule], seed=33)
        d.uniform[0] = 0.9999
        for draw in (1e-6, 0.5, 1 - 1e-6):
            d.draw[:] = draw
            d.check()


@pytest.mark.parametrize("dtype", sorted(TYPES))
def test_words_whose_weight_rounds_to_none_are_not_drawn(dtype):
    """As in sampling: 2^-44.7 of the largest word's weight is none, also where no rule cuts and the draw is 0."""
    d = Drafts([1, 1, 2, 2], 5003, dtype, None, [(1.0, 0, 1.0, 0.0)], seed=40)
    d.logits[:] = -100.0
    d.logits[:, 0], d.logits[:, 4900] = -31.0, 0.0
    d.draw[:], d.uniform[:] = 0.0, 0.5
    d.drafted[:] = 0                       # refused: its weight is none
    tokens, accepted, probs = d.call()
    first = torch.tensor(d.starts[:-1], device="cuda").long()
    assert accepted.tolist() == [0, 0, 0, 0] and (tokens[first] == 4900).all() and (probs[first] == 1).all()
