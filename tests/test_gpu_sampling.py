"""The next token of each row against its definition in 64 bits: tokens equal, probabilities to 32 bits."""
import numpy as np
import pytest

torch = pytest.importorskip("torch")

import serving_reference as ref
from loken_amd import sampling

pytestmark = pytest.mark.gpu

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def check(logits, uniform, temperature, top_k=None, top_p=None, min_p=None, device_logits=None):
    rows = logits.shape[0]
    full = lambda v, d: None if v is None else np.broadcast_to(np.asarray(v, d), rows).copy()  # noqa: E731
    u, t, k, p, m = full(uniform, np.float32), full(temperature, np.float32), full(top_k, np.int32), full(top_p, np.float32), full(min_p, np.float32)
    dev = lambda a: None if a is None else torch.tensor(a, device="cuda")  # noqa: E731
    tokens, probs = sampling.sample(logits.cuda() if device_logits is None else device_logits, dev(u), dev(t), dev(k), dev(p), dev(m))
    want, share = ref.sample(logits.float().numpy(), u, t, k, p, m)
    assert np.array_equal(tokens.cpu().numpy(), want)
    # a weight to 1e-10 and 2^-43 of the first, the sum likewise, rounded to 32 bits
    assert np.allclose(probs.cpu().numpy(), share, rtol=2.0 ** -24 + 1e-9, atol=1e-12)
    return tokens


def normal(rows, vocab, seed, dtype=torch.float32, spread=3.0):
    return torch.tensor(np.random.default_rng(seed).normal(size=(rows, vocab)) * spread, dtype=torch.float32).to(dtype)


def uniforms(rows, seed):
    return np.random.default_rng(seed + 99).random(rows).astype(np.float32)


RULES = [dict(), dict(top_k=1), dict(top_k=50), dict(top_k=5000), dict(top_p=0.9), dict(top_p=0.999), dict(min_p=0.05), dict(top_k=40, top_p=0.95, min_p=0.02),
         dict(top_p=0.0), dict(min_p=1.0), dict(top_k=10 ** 6, top_p=1.0, min_p=0.0), dict(top_p=0.5, min_p=2.0)]


@pytest.mark.parametrize("rules", RULES, ids=str)
@pytest.mark.parametrize("dtype", sorted(TYPES))
@pytest.mark.parametrize("rows,vocab", [(1, 32000), (3, 151936), (70, 5003)])
def test_rules(rows, vocab, dtype, rules):
    check(normal(rows, vocab, vocab, TYPES[dtype]), uniforms(rows, vocab), 0.8, **rules)


@pytest.mark.parametrize("vocab", [1, 2, 3, 63, 64, 65, 511, 512, 513, 2047, 2048, 2049, 4097])
def test_small_and_odd_vocabularies(vocab):
    check(normal(9, vocab, vocab), uniforms(9, vocab), 1.0, top_k=[0, 1, 2, 5, 40, 0, 0, 3, 7], top_p=[1, 1, 1, 0.9, 0.5, 0.3, 1, 0.7, 0.99])


@pytest.mark.parametrize("temperature", [1e-30, 1e-3, 0.1, 1.0, 7.0, 100.0, 1e30, float("inf")])
@pytest.mark.parametrize("rules", [dict(), dict(top_k=300), dict(top_p=0.6), dict(min_p=0.5)], ids=str)
def test_temperatures(temperature, rules):
    check(normal(4, 40000, 5), uniforms(4, 5), temperature, **rules)


@pytest.mark.parametrize("temperature", [0.0, -1.0, float("nan")])
def test_the_first_word_without_a_temperature(temperature):
    x = normal(4, 3001, 6)
    x[1, 7] = x[1, 2000] = 50.0          # equal ones: the lower number
    x[2, :] = 1.0
    assert check(x, 0.99, temperature, top_k=5).tolist()[1:3] == [7, 0]


@pytest.mark.parametrize("dtype", sorted(TYPES))
@pytest.mark.parametrize("rules", [dict(), dict(top_k=7), dict(top_k=3000), dict(top_p=0.37), dict(min_p=0.5)], ids=str)
def test_equal_words_stand_in_their_order(rules, dtype):
    """Rows of equal words, of a few values, and of values around both zeros; more of one kind than are sorted at once."""
    rows = torch.zeros(5, 10007)
    rows[1] = -2.5
    rows[2] = torch.tensor(np.random.default_rng(1).integers(0, 3, 10007).astype(np.float32))
    rows[3, ::2] = -0.0
    rows[4] = torch.tensor(np.random.default_rng(2).integers(-2, 2, 10007).astype(np.float32))
    for u in (0.0, 0.25, 0.7, 0.99999994):
        check(rows.to(TYPES[dtype]), u, 1.0, **rules)


@pytest.mark.parametrize("low", [float("-inf"), -3.4028234663852886e38, -1e9, -65504.0, -1e4])
@pytest.mark.parametrize("rules", [dict(), dict(top_k=60), dict(top_p=0.8), dict(top_k=20000)], ids=str)
def test_masked_words(low, rules):
    """Most of a vocabulary is masked, by any of the values that programs mask with."""
    x = normal(6, 30000, 8)
    keep = np.random.default_rng(3).random((6, 30000)) < 0.002
    keep[:, 17] = True
    x = torch.where(torch.tensor(keep), x, torch.tensor(low))
    x[5] = torch.where(torch.arange(30000) == 12345, x[5], torch.tensor(low))   # masked as well: a row of equal words, or of none
    check(x, uniforms(6, 8), 1.2, **rules)
    one = torch.full((1, 30000), low)
    one[0, 12345] = -3.0
    assert check(one, 0.99, 1.2, **rules).tolist() == [12345]


def test_rows_without_words_and_words_that_are_none():
    x = normal(5, 4000, 9)
    x[0] = float("-inf")
    x[1] = float("nan")
    x[2, ::3] = float("nan")
    x[3, 100] = x[3, 3000] = x[3, 3500] = float("inf")
    x[4, 1:] = float("-inf")
    for rules in (dict(), dict(top_k=2), dict(top_p=0.5)):
        tokens = check(x, 0.6, 1.0, **rules)
        assert tokens[:2].tolist() == [-1, -1] and int(tokens[4]) == 0 and int(tokens[3]) in (100, 3000, 3500)
    check(x, 0.6, 0.0)


@pytest.mark.parametrize("rules", [dict(), dict(top_k=100), dict(top_p=0.9)], ids=str)
def test_values_far_apart(rules):
    """A step of the histogram that holds nearly all words; words that lie 1e-6 apart; falling powers of two."""
    x = normal(4, 20000, 10, spread=1e-3)
    x[0, 5] = 30.0
    x[1] *= 1e-3
    x[2] = -torch.tensor(2.0 ** (np.arange(20000) % 40 - 30), dtype=torch.float32)
    x[3] = 1e6 + torch.arange(20000) / 16.0
    for u in (0.0, 0.5, 0.999):
        check(x, u, [40.0, 1.0, 0.01, 900.0], **rules)


@pytest.mark.parametrize("u", [0.0, 0.5, 0.99999994, 1.0, 2.0, -1.0, float("nan")])
def test_the_ends_of_the_uniform_number(u):
    x = normal(3, 1000, 11)
    inside = min(max(np.nan_to_num(u, nan=0.0), 0.0), 0.99999994)
    dev = lambda v: torch.full((3,), v, device="cuda")  # noqa: E731
    got = sampling.sample(x.cuda(), dev(u), dev(1.0), torch.full((3,), 20, dtype=torch.int32, device="cuda"))
    want = sampling.sample(x.cuda(), dev(inside), dev(1.0), torch.full((3,), 20, dtype=torch.int32, device="cuda"))
    assert torch.equal(got[0], want[0])
    check(x, inside, 1.0, top_k=20)


def test_rows_that_are_parts_of_wider_ones():
    wide = normal(7, 9000, 12)
    for a, b in ((0, 8191), (1, 8192), (3, 4003)):
        check(wide[:, a:b].contiguous(), uniforms(7, 12), 0.9, top_p=0.9, device_logits=wide.cuda()[:, a:b])


def test_many_rows_and_the_largest_vocabulary():
    check(normal(600, 777, 13), uniforms(600, 13), 1.0, top_k=50, top_p=0.9)
    check(normal(2, sampling.MAX_VOCAB, 14), uniforms(2, 14), 1.0)
    assert sampling.sample(torch.zeros((0, 10), device="cuda"), *(torch.zeros(0, device="cuda"),) * 2)[0].numel() == 0


def test_what_is_drawn_follows_the_probabilities():
    """Uniform numbers that step through [0, 1): each word comes up as often as its share says, to one step."""
    n = 4000
    x = normal(1, 50, 15, spread=1.5)
    u = torch.arange(n, device="cuda", dtype=torch.float32) / n
    tokens, _ = sampling.sample(x.cuda().expand(n, 50).contiguous(), u, torch.ones(n, device="cuda"))
    share = torch.softmax(x[0].double(), 0).numpy()
    counts = np.bincount(tokens.cpu().numpy(), minlength=50)
    assert (np.abs(counts / n - share) <= 1.0 / n + 1e-6).all()


def test_the_same_call_gives_the_same_bits():
    x = normal(5, 151936, 16, torch.bfloat16).cuda()
    u, t = torch.tensor(uniforms(5, 16), device="cuda"), torch.ones(5, device="cuda")
    first = sampling.sample(x, u, t)
    for _ in range(5):
        again = sampling.sample(x, u, t)
        assert torch.equal(first[0], again[0]) and torch.equal(first[1], again[1])


@pytest.mark.parametrize("top_k", [200, 255, 256, 257, 300, 511, 512, 513, 777, 1000, 1023, 1024, 1025, 2047])
@pytest.mark.parametrize("coarse", [0, 64, 4, 1])
def test_lists_of_every_length(top_k, coarse):
    """Words sorted by counting, by their steps, and (many of a value) by exchanges; the draw anywhere among them."""
    x = normal(6, 50000, top_k + coarse)
    x = x if not coarse else (x * coarse).round() / coarse
    check(x, [0.0, 0.3, 0.9, 0.999, 0.99999, 0.5], 3.0, top_k=top_k, top_p=[1, 1, 1, 1, 0.99, 0.7])


@pytest.mark.parametrize("top_p", [0.5, 0.9, 0.95, 0.99, 0.9999])
@pytest.mark.parametrize("spread", [0.01, 0.3, 1.0])
def test_a_nucleus_that_ends_with_the_last_words(spread, top_p):
    """Rows of a few words, whose smallest one is the end of the histogram, alone and among masked ones; draws all over [0, 1)."""
    g = np.random.default_rng(int(spread * 100))
    for words in (2, 3, 4, 8, 16):
        x = normal(33, words, words, spread=spread)
        u = ((np.arange(33) + g.random(33)) / 33).astype(np.float32)
        check(x, u, 1.0, top_p=top_p)
        masked = torch.full((33, 5003), float("-inf"))
        masked[:, torch.tensor(np.sort(g.choice(5003, words, replace=False)))] = x
        check(masked, u, 1.0, top_p=top_p)
        check(masked, u, 1.0, top_p=top_p, top_k=10 ** 6, min_p=1e-6)
    check(normal(9, 3001, 2, spread=spread), ((np.arange(9) + 0.5) / 9).astype(np.float32), 1.0, top_p=top_p)


@pytest.mark.parametrize("temperature", [1e-14, 1e-15, 1e-16, 1e-17, 3e-18, 1e-18, 1e-19, 1e-20, 1e-22, 1e-24, 1e-38, 1e-44])
@pytest.mark.parametrize("rules", [dict(), dict(top_k=3), dict(top_k=2000), dict(top_p=0.6), dict(min_p=0.5)], ids=str)
def test_temperatures_far_below_the_logits(temperature, rules):
    """Only words equal to the largest are left, each with a weight of one: alone, and as one of a few or of thousands."""
    x = normal(8, 5003, 17)
    for r, n in enumerate((1, 2, 3, 7, 300, 2500, 1, 2)):
        at = np.random.default_rng(r).choice(5003, n, replace=False)
        x[r, torch.tensor(at)] = [11.37, 12.5, 14.0, 9.1, 15.999, 8.3, 1e5, 65504.0][r]
    for u in (0.0, 0.37, 0.99999994):
        check(x, u, temperature, **rules)


@pytest.mark.parametrize("size", [1e8, 1e12, 1e16, 1e17, 1e18, 1e20, 1e22, 1e26, 1e29, 3e38])
@pytest.mark.parametrize("sign", [1, -1])
@pytest.mark.parametrize("rules", [dict(), dict(top_k=3), dict(top_p=0.6), dict(min_p=0.5)], ids=str)
def test_logits_far_from_zero(size, sign, rules):
    """Rows of large logits: equal ones, neighbours in their type, and words far behind them."""
    g = np.random.default_rng(18)
    top = np.float32(sign * size)
    x = np.full((6, 4001), -np.inf, np.float32)
    near = [top]
    for _ in range(6):
        near.append(np.nextafter(near[-1], np.float32(-np.inf)))
    for r in range(6):
        x[r] = np.array(near)[g.integers(0, 1 + r, 4001)]
        x[r, g.random(4001) < 0.9] = [-np.inf, np.float32(-3.4e38), near[-1], -np.inf, -np.inf, near[2]][r]
        x[r, 17] = top
    if sign > 0:
        x[0, ::7] = 0.5
    for temperature in (1.0, float(near[0]) - float(near[1])):
        for u in (0.0, 0.37, 0.99999994):
            check(torch.tensor(x), u, temperature, **rules)
