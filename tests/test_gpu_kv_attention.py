"""Attention over the paged 8-bit cache against its definition in 64 bits over the same codes."""
import numpy as np
import pytest

torch = pytest.importorskip("torch")

import serving_reference as ref
from loken_amd import kv

pytestmark = pytest.mark.gpu

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def i32(v):
    return torch.tensor(np.asarray(v, np.int32), device="cuda")


class Batch:
    """A cache of random codes, tables of scattered pages, and queries."""

    def __init__(self, lens, fresh, heads, kv_heads, dim, page, dtype, seed=0, spare=2, pad=0):
        g = np.random.default_rng(seed)
        want = [-(-n // page) for n in lens]
        pages = sum(want) + spare
        self.want = ref.Cache(pages, kv_heads, page, dim)
        for s in "kv":
            self.want.codes[s] = g.integers(-127, 128, (pages, kv_heads, page, dim))
            self.want.scales[s] = (g.uniform(0.2, 1.0, (pages, kv_heads)) * 0.02).astype(np.float32)
        ids = g.permutation(pages)
        cols = max(want + [1]) + 1
        self.table = np.full((len(lens), cols), -1, np.int32)
        n = 0
        for i, w in enumerate(want):
            self.table[i, :w] = ids[n:n + w]
            n += w
        self.lens, self.starts = np.array(lens, np.int32), np.concatenate([[0], np.cumsum(fresh)]).astype(np.int32)
        self.rows = int(self.starts[-1]) + pad
        self.q = torch.tensor(g.normal(size=(self.rows, heads, dim)), dtype=torch.float32).to(TYPES[dtype])
        self.dtype, self.page, self.dim, self.heads = dtype, page, dim, heads
        self.fresh = fresh

    def cache(self):
        c = self.want
        pages, heads, page, dim = c.codes["k"].shape
        v = c.codes["v"].reshape(pages, heads, page // 16, 16, dim).transpose(0, 1, 2, 4, 3)
        t = lambda a, d: torch.tensor(np.ascontiguousarray(a), dtype=d, device="cuda")  # noqa: E731
        return kv.KvCacheQ8(t(c.codes["k"], torch.int8), t(v, torch.int8), t(c.scales["k"], torch.float32), t(c.scales["v"], torch.float32))

    def check(self, scale=None, window=0, max_fresh=None, max_len=None, q=None, cache=None):
        q = self.q.cuda() if q is None else q
        out = torch.full((self.rows, self.heads, self.dim), 7.0, dtype=q.dtype, device="cuda")
        kv.kv_attention(q, cache or self.cache(), i32(self.table), i32(self.lens), i32(self.starts), scale=scale, window=window, out=out,
                        max_fresh=max([*self.fresh, 0]) if max_fresh is None else max_fresh, max_len=max([*self.lens, 0]) if max_len is None else max_len)
        scale = 1.0 / np.sqrt(self.dim) if scale is None else scale
        want, reach, most = ref.attention(q.float().cpu().numpy(), self.want, self.table, self.lens, self.starts, scale, window, np.full(out.shape, 7.0))
        got = out.double().cpu().numpy()
        # What may be lost. A query value is held to 2^-22 (f32) or 2^-15 (16-bit types) of the row's largest, half of that by
        # rounding: the scores are off by up to reach * that and shift a weighted mean of values by up to twice as much of the
        # largest. f32 sums of scores lose some units of 2^-24 of the score's parts, as little. The weights are held to
        # 2^-22 or 2^-15 of the largest of 64 positions, or to 2^-11 each: 64 * 2^-23, 64 * 2^-16 = 2^-10 of the largest value at most.
        # Then the output's rounding, half a step.
        fine = self.dtype == "f32"
        bound = most * (2 * reach * 2.0 ** (-22 if fine else -15) + 2.0 ** (-17 if fine else -10) + 2.0 ** -20)
        step = 2.0 ** -24 if fine else torch.finfo(q.dtype).eps / 2
        assert np.isfinite(got).all()
        off = np.abs(got - want) - step * np.abs(want) - bound[..., None]
        assert (off <= 0).all(), (off.max(), np.abs(got - want).max())
        return out


HEADS = [(4, 1, 128), (2, 2, 64), (8, 1, 256), (6, 2, 64), (16, 8, 128), (5, 1, 64), (20, 1, 128), (32, 4, 128)]


@pytest.mark.parametrize("dtype", sorted(TYPES))
@pytest.mark.parametrize("heads,kv_heads,dim", HEADS)
def test_single_tokens(heads, kv_heads, dim, dtype):
    Batch([1, 15, 16, 17, 63, 64, 65, 200, 777], [1] * 9, heads, kv_heads, dim, 16, dtype, seed=heads).check()


@pytest.mark.parametrize("dtype", sorted(TYPES))
@pytest.mark.parametrize("page", [16, 32, 64, 128, 256])
def test_pages_of_every_size(page, dtype):
    Batch([1, page - 1, page, page + 1, 3 * page + 7], [1, 1, 2, 1, 5], 4, 2, 128, page, dtype, seed=page).check()


@pytest.mark.parametrize("dtype", sorted(TYPES))
@pytest.mark.parametrize("heads,kv_heads,dim", [(4, 1, 128), (2, 2, 64), (3, 1, 256), (8, 2, 64)])
@pytest.mark.parametrize("lens,fresh", [([40], [40]), ([1], [1]), ([129], [129]), ([300], [37]), ([70, 3, 200], [64, 3, 33]), ([333, 90], [1, 90])])
def test_prompts_and_chunks(heads, kv_heads, dim, lens, fresh, dtype):
    Batch(lens, fresh, heads, kv_heads, dim, 16, dtype, seed=dim + len(lens)).check()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("n", [2, 3, 4, 5, 8, 9, 16, 17, 33])
def test_a_few_tokens_a_sequence(n, dtype):
    Batch([n, 100, 64 + n], [n, n, n], 4, 2, 128, 16, dtype, seed=n).check()


@pytest.mark.parametrize("dtype", ["f32", "f16"])
@pytest.mark.parametrize("window", [1, 2, 16, 17, 63, 64, 100, 1000, 0x7FFFFFFF])
def test_windows(window, dtype):
    Batch([1, 70, 500, 260], [1, 1, 3, 90], 4, 2, 64, 16, dtype, seed=window & 255).check(window=window)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("hint", [(0, 0), (1, 1), (1, 100000), (5000, 1), (5000, 100000)])
def test_sizes_given_are_hints(hint, dtype):
    """The caller's idea of the most rows and tokens of a sequence chooses launches, not results."""
    Batch([700, 90, 260, 0, 2500], [1, 4, 150, 0, 2], 8, 2, 128, 16, dtype, seed=5, pad=6).check(max_fresh=hint[0], max_len=hint[1])


@pytest.mark.parametrize("dtype", sorted(TYPES))
def test_rows_behind_the_last_sequence_and_empty_sequences(dtype):
    b = Batch([0, 50, 7, 0, 90], [0, 1, 0, 0, 1], 4, 1, 64, 16, dtype, seed=3, pad=9)
    out = b.check()
    assert (out[2:] == 7).all()


@pytest.mark.parametrize("dtype", sorted(TYPES))
@pytest.mark.parametrize("fresh", [1, 40])
def test_rows_that_see_nothing_are_zeros(fresh, dtype):
    """Pages that are absent, a sequence without tokens that brings rows, and more rows than tokens."""
    b = Batch([90, 200, 64, 5], [fresh] * 4, 4, 1, 128, 16, dtype, seed=8)
    b.table[0] = -1
    b.table[1, 3:6] = [-1, 10 ** 6, -(1 << 31)]
    b.lens[2] = 0
    out = b.check()
    assert (out[:fresh] == 0).all() and (out[2 * fresh:3 * fresh] == 0).all()
    if fresh > 5:
        assert (out[3 * fresh:4 * fresh - 5] == 0).all()


@pytest.mark.parametrize("dtype", ["f32", "f16"])
@pytest.mark.parametrize("fresh", [1, 50])
def test_lengths_past_the_end_of_the_table(fresh, dtype):
    """Positions whose column the table does not have are absent."""
    b = Batch([300, 80], [fresh, fresh], 2, 1, 64, 16, dtype, seed=2)
    b.table = np.ascontiguousarray(b.table[:, :9])
    b.check()


def test_starts_past_the_batch_are_cut():
    """A plan of more rows than the batch holds: those that it holds are computed, nothing is written behind it."""
    b = Batch([40, 60], [10, 20], 2, 1, 64, 16, "f32", seed=12)
    guard = torch.full((40, 2, 64), 9.0, device="cuda")
    kv.kv_attention(b.q[:17].cuda().contiguous(), b.cache(), i32(b.table), i32(b.lens), i32(b.starts), max_fresh=20, max_len=60, out=guard[:17])
    assert (guard[17:] == 9).all()
    # the seven rows that are left of the second sequence are few enough for another kernel: held to the definition, not to its bits
    b.q, b.rows = b.q[:17], 17
    assert torch.equal(b.check(max_fresh=20, max_len=60), guard[:17])


@pytest.mark.parametrize("dtype", sorted(TYPES))
@pytest.mark.parametrize("fresh", [1, 70])
def test_strided_queries_and_outputs(fresh, dtype):
    b = Batch([130, 75], [fresh, 2], 4, 2, 64, 16, dtype, seed=6)
    want = b.check()
    wide = torch.zeros((b.rows, 9, 64), dtype=TYPES[dtype], device="cuda")
    wide[:, 3:7] = b.q.cuda()
    target = torch.full((b.rows, 11, 64), 3.0, dtype=TYPES[dtype], device="cuda")
    table = torch.full((2, 20), 1, dtype=torch.int32, device="cuda")
    table[:, :b.table.shape[1]] = i32(b.table)
    kv.kv_attention(wide[:, 3:7], b.cache(), table[:, :b.table.shape[1]], i32(b.lens), i32(b.starts), max_fresh=max(fresh, 2), max_len=130, out=target[:, 5:9])
    assert torch.equal(target[:, 5:9], want) and (target[:, :5] == 3).all() and (target[:, 9:] == 3).all()


@pytest.mark.parametrize("dtype", sorted(TYPES))
@pytest.mark.parametrize("fresh", [1, 40])
@pytest.mark.parametrize("what", ["a peak", "flat", "zero values", "scales far apart", "large queries", "small queries"])
def test_distributions(what, fresh, dtype):
    b = Batch([400, 33], [fresh, 1], 4, 2, 64, 16, dtype, seed=20)
    scale = None
    if what == "a peak":
        scale = 2.0            # one position takes nearly all
    elif what == "flat":
        b.q *= 0
    elif what == "zero values":
        b.want.codes["v"] *= 0
        b.want.scales["v"][::2] = 0
    elif what == "scales far apart":
        b.want.scales["v"] *= np.float32(10.0) ** np.random.default_rng(0).integers(-5, 6, b.want.scales["v"].shape).astype(np.float32)
        b.want.scales["k"][1::3] *= np.float32(1e-4)
        b.want.scales["k"][2::3] = 0
    elif what == "large queries":
        b.q *= 2000.0
        scale = 1e-5
    else:
        b.q = (b.q.float() * 1e-4).to(b.q.dtype)
        scale = 300.0
    b.check(scale=scale)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("power", [-120, -60, 60, 100])
def test_queries_of_any_size(power, dtype):
    """Types with eight bits of exponent: the scale makes up for the queries' size."""
    b = Batch([150, 90], [1, 40], 2, 1, 64, 16, dtype, seed=21)
    b.q = (b.q.double() * 2.0 ** power).to(b.q.dtype)
    b.check(scale=0.125 * 2.0 ** -power)


@pytest.mark.parametrize("dtype", sorted(TYPES))
@pytest.mark.parametrize("fresh", [1, 40])
def test_query_values_that_are_not_finite(fresh, dtype):
    b = Batch([100, 60], [fresh, 1], 4, 2, 64, 16, dtype, seed=22)
    want = b.check()
    q = b.q.cuda()
    q[0, 1, 3], q[fresh - 1, 2, 60], q[fresh, 0, 0] = float("nan"), float("inf"), float("-inf")
    out = kv.kv_attention(q, b.cache(), i32(b.table), i32(b.lens), i32(b.starts), max_fresh=fresh, max_len=100)
    bad = torch.zeros(out.shape[:2], dtype=torch.bool, device="cuda")
    bad[0, 1] = bad[fresh - 1, 2] = bad[fresh, 0] = True
    assert torch.isnan(out[bad]).all() and torch.equal(out[~bad], want[~bad])


@pytest.mark.parametrize("dtype,heads,kv_heads,length,fresh", [("f32", 4, 1, 33000, 1), ("f16", 2, 1, 70001, 1), ("bf16", 4, 2, 20000, 3), ("f32", 2, 1, 9000, 40),
                                                             ("bf16", 2, 1, 9000, 150)])
def test_long_contexts_are_split_and_joined(dtype, heads, kv_heads, length, fresh):
    Batch([length, 40], [fresh, 1], heads, kv_heads, 64, 64, dtype, seed=length & 1023).check()


def test_pages_behind_2_to_the_31_bytes():
    pages = (1 << 31) // (16 * 64) + 9
    small = Batch([100, 30], [1, 9], 2, 1, 64, 16, "f32", seed=30, spare=0)
    cache = small.cache()
    big = kv.KvCacheQ8(torch.zeros((pages, 1, 16, 64), dtype=torch.int8, device="cuda"), torch.zeros((pages, 1, 1, 64, 16), dtype=torch.int8, device="cuda"),
                       torch.zeros((pages, 1), device="cuda"), torch.zeros((pages, 1), device="cuda"))
    for name in ("k", "v", "k_scales", "v_scales"):
        getattr(big, name)[pages - 9:] = getattr(cache, name)
    table = np.where(small.table >= 0, small.table + pages - 9, -1)
    args = (i32(small.lens), i32(small.starts))
    assert torch.equal(kv.kv_attention(small.q.cuda(), big, i32(table), *args, max_fresh=9, max_len=100),
                       kv.kv_attention(small.q.cuda(), cache, i32(small.table), *args, max_fresh=9, max_len=100))


def test_a_row_does_not_depend_on_its_companions():
    """The same sequence alone and in a batch, with equal sizes given: the same bits."""
    b = Batch([500, 60, 900], [1, 1, 1], 8, 2, 128, 16, "f32", seed=31)
    whole = b.check(max_len=900)
    for i in range(3):
        one = kv.kv_attention(b.q[i:i + 1].cuda(), b.cache(), i32(b.table[i:i + 1]), i32(b.lens[i:i + 1]), i32([0, 1]), max_fresh=1, max_len=900)
        assert (one[0] - whole[i]).abs().max() <= 2e-5 * whole[i].abs().max()   # split over other workgroups: the parts join in another order
    assert torch.equal(whole, b.check(max_len=900))


@pytest.mark.parametrize("dtype", sorted(TYPES))
@pytest.mark.parametrize("what", ["ragged", "one long", "window", "more rows than said", "beside a prompt"])
def test_many_contexts_are_cut_into_equal_pieces(what, dtype):
    """Enough sequences for pieces that hold several of them, ends of them, and sequences without rows or tokens."""
    g = np.random.default_rng(40)
    lens = [0, 1, 64, 65, 0] + [int(v) for v in g.integers(1, 5000, 36)] + [0, 3]
    fresh = [0] + [1] * 42
    fresh[4], fresh[11], fresh[20], fresh[42] = 1, 0, 2, 0
    if what == "one long":
        lens = [100] * 42 + [40000]
    if what == "more rows than said":
        fresh[7], fresh[30] = 9, 40
    if what == "beside a prompt":
        fresh[9] = 70
    b = Batch(lens, fresh, 2, 1, 64, 16, dtype, seed=41, pad=3)
    out = b.check(window=700 if what == "window" else 0, max_fresh=2 if what != "beside a prompt" else 70, max_len=9000)
    assert (out[-3:] == 7).all()


@pytest.mark.parametrize("dtype", sorted(TYPES))
@pytest.mark.parametrize("seqs,longest", [(70, 150), (130, 40), (200, 300)])
def test_long_and_short_sequences_of_a_batch(seqs, longest, dtype):
    """Row tiles of a few sequences among many that have none, in more than one look's worth of sequences; hints too small as well."""
    g = np.random.default_rng(seqs)
    fresh = [int(g.integers(0, longest)) if i % 9 == 4 else int(g.integers(0, 3)) for i in range(seqs)]
    fresh[-1] = longest
    b = Batch([f + int(g.integers(0, 30)) for f in fresh], fresh, 4, 2, 64, 16, dtype, seed=seqs, pad=3)
    assert (b.check()[-3:] == 7).all()
    b.check(max_fresh=17, max_len=5)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("fresh", [1, 30])
def test_queries_whose_scale_alone_would_overflow(fresh, dtype):
    """Scores of ordinary size from queries at the end of the type's range and keys at the beginning of it."""
    b = Batch([200], [fresh], 4, 2, 64, 16, dtype, seed=31)
    g = np.random.default_rng(31)
    shape = b.want.scales["k"].shape
    b.want.codes["k"] = g.integers(-3, 4, b.want.codes["k"].shape)
    b.want.scales["k"] = g.uniform(1.2e-38, 2e-38, shape).astype(np.float32)
    b.q = (b.q.float() * 7e37).clamp(-3e38, 3e38)
    b.q[..., 5] = 3e38
    b.q = b.q.to(TYPES[dtype])
    b.check(scale=1.3)


@pytest.mark.parametrize("dtype", sorted(TYPES))
@pytest.mark.parametrize("hint", [1, 40])
def test_first_rows_far_outside_the_batch(hint, dtype):
    """Rows that a sequence claims are those of the batch at most, whatever `starts` holds: one that ends before it starts has none,
    even where the difference passes 32 bits; one whose positions are all below zero sees nothing."""
    b = Batch([300, 200, 100], [0, 0, 0], 4, 2, 64, 16, dtype, pad=40)
    out = torch.full((b.rows, b.heads, b.dim), 7.0, dtype=TYPES[dtype], device="cuda")
    for starts, want in (([2000000000, -2000000000, -2147483648, -2147483648], 7.0), ([2147483647, -2147483648, 2147483647, -2147483648], 0.0),
                         ([2147483647, -5, -2147483648, 0], 7.0)):
        out.fill_(7.0)
        kv.kv_attention(b.q.cuda(), b.cache(), i32(b.table), i32(b.lens), i32(starts), max_fresh=hint, max_len=300, out=out)
        assert (out == want).all()


@pytest.mark.parametrize("dtype", sorted(TYPES))
@pytest.mark.parametrize("fresh", [1, 40])
@pytest.mark.parametrize("largest", ["first", "last", "in the middle"])
@pytest.mark.parametrize("ratio", [-20, -36, -39, -40, -41, -44, -60, -100, -120, -126])
def test_value_scales_of_any_ratio(ratio, largest, fresh, dtype):
    """One page of large values among pages of values that do not show beside them: their weights count all the same."""
    b = Batch([300], [fresh], 4, 2, 64, 16, dtype, seed=50)
    b.want.scales["v"][:] = np.float32(2.0 ** ratio)
    b.want.scales["v"][b.table[0, {"first": 0, "last": 16, "in the middle": 9}[largest]]] = 1.0
    for scale in (0.125, 1.5):
        b.check(scale=scale)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("fresh", [1, 40])
def test_value_scales_at_both_ends_of_what_a_page_may_have(fresh, dtype):
    b = Batch([300], [fresh], 4, 2, 64, 16, dtype, seed=51)
    b.want.scales["v"][:] = np.float32(2.0 ** -126)
    b.want.scales["v"][b.table[0, ::5]] = np.float32(2.0 ** 14)
    b.check()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("fresh,length", [(1, 300), (40, 300), (1, 9000), (40, 9000)])
@pytest.mark.parametrize("power", [-126, -120, -110, -100])
def test_values_near_the_smallest(power, fresh, length, dtype):
    """Pages whose scales are the smallest that a page may have, alike: outputs keep the bits that their type has there."""
    b = Batch([length], [fresh], 2, 1, 64, 16, dtype, seed=52)
    b.want.scales["v"] = (b.want.scales["v"].astype(np.float64) * 50 * 2.0 ** power).clip(2.0 ** -126).astype(np.float32)
    out = torch.zeros((b.rows, b.heads, b.dim), dtype=TYPES[dtype], device="cuda")
    kv.kv_attention(b.q.cuda(), b.cache(), i32(b.table), i32(b.lens), i32(b.starts), max_fresh=fresh, max_len=length, out=out)
    want, reach, most = ref.attention(b.q.float().numpy(), b.want, b.table, b.lens, b.starts, b.dim ** -0.5, 0, np.zeros(out.shape))
    fine = dtype == "f32"
    bound = most * (2 * reach * 2.0 ** (-22 if fine else -15) + 2.0 ** (-17 if fine else -10) + 2.0 ** -20)
    step = 2.0 ** -24 if fine else torch.finfo(TYPES[dtype]).eps / 2
    least = 2.0 ** -150 if fine else 2.0 ** -134   # half of the type's smallest step, which a rounding below the normal numbers goes by
    off = np.abs(out.double().cpu().numpy() - want) - step * np.abs(want) - bound[..., None] - least
    assert (off <= 0).all(), off.max() / most.max()


@pytest.mark.parametrize("dtype,ratio", [(d, r) for d in sorted(TYPES) for r in (-8, -12, -20, -40, -100) if d != "f16" or r >= -12])   # (f16: normal numbers)
@pytest.mark.parametrize("length,fresh,window,hidden", [(300, 1, 70, (12, 13)), (300, 3, 70, (12, 13)), (300, 1, 33, (0, 16)), (290, 4, 0, (18,)), (290, 4, 20, (16, 18)),
                                                        (2000, 1, 300, (104, 105))])
def test_pages_that_a_row_does_not_see_do_not_cost_it_bits(length, fresh, window, hidden, dtype, ratio):
    """Large values behind a window's border, or of the sequence's later rows: what is lost of a row goes by the values that it sees."""
    b = Batch([length], [fresh], 4, 2, 64, 16, dtype, seed=53)
    b.want.scales["v"] *= np.float32(2.0 ** ratio)
    b.want.scales["v"][b.table[0, list(hidden)]] = 1.0
    b.check(window=window)


@pytest.mark.parametrize("dtype,ratio", [(d, r) for d in sorted(TYPES) for r in (-4, -8, -12, -16, -20, -28, -40, -60) if d != "f16" or r >= -12])   # (f16: normal numbers)
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("length,fresh,window,hidden", [(300, 40, 0, (18,)), (300, 40, 0, (17,)), (400, 40, 70, (16, 17, 18)), (400, 40, 70, (18, 19)), (400, 100, 0, (20, 21, 22, 23, 24)),
                                                        (3000, 33, 500, (156, 157, 186)), (3000, 300, 0, (170, 186))])
def test_pages_that_a_row_of_a_prompt_does_not_see_do_not_cost_it_bits(length, fresh, window, hidden, dim, dtype, ratio):
    b = Batch([length], [fresh], 2, 1, dim, 16, dtype, seed=54)
    b.want.scales["v"] *= np.float32(2.0 ** ratio)
    b.want.scales["v"][b.table[0, list(hidden)]] = 1.0
    b.check(window=window)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("fresh", [1, 40])
def test_value_scales_that_grow_again_and_again(fresh, dtype):
    """Each page's values a multiple of the ones before: every step's sums are put to another size, up to what f32 holds."""
    for step in (0.5, 3.0, 12.0):
        b = Batch([500], [fresh], 4, 2, 64, 16, dtype, seed=55)
        n = int((b.table[0] >= 0).sum())
        powers = np.minimum(-120 + step * np.arange(n), 90)
        b.want.scales["v"][b.table[0, :n]] = (2.0 ** powers)[:, None].astype(np.float32)
        b.check()
        b.want.scales["v"][b.table[0, :n]] = (2.0 ** powers[::-1])[:, None].astype(np.float32)
        b.check()
