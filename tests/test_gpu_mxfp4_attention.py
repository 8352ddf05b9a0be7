"""Attention over the paged 4-bit cache against its definition in 64 bits over the same codes."""
import numpy as np
import pytest

torch = pytest.importorskip("torch")

import mxfp4_reference as ref
from loken_amd import kv
from test_gpu_graph_scratch import check_replays
from test_gpu_mxfp4_cache import TYPES, dev, handle

pytestmark = pytest.mark.gpu


def i32(v):
    return torch.tensor(np.asarray(v, np.int32), device="cuda")


class Batch:
    """A cache of random codes, tables of scattered pages, and queries."""

    def __init__(self, lens, fresh, heads, kv_heads, dim, page, dtype, seed=0, spare=2, pad=0, powers=(124, 128)):
        g = np.random.default_rng(seed)
        want = [-(-n // page) for n in lens]
        pages = sum(want) + spare
        self.want = ref.Cache(pages, kv_heads, page, dim, seed=seed, powers=powers)
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
        self.dtype, self.page, self.dim, self.heads, self.fresh = dtype, page, dim, heads, fresh

    def cache(self):
        return handle(self.want)

    def check(self, scale=None, window=0, cap=0.0, max_fresh=None, max_len=None, q=None, cache=None):
        q = self.q.cuda() if q is None else q
        out = torch.full((self.rows, self.heads, self.dim), 7.0, dtype=q.dtype, device="cuda")
        kv.kv_attention(q, cache or self.cache(), i32(self.table), i32(self.lens), i32(self.starts), scale=scale, window=window, softcap=cap, out=out,
                        max_fresh=max([*self.fresh, 0]) if max_fresh is None else max_fresh, max_len=max([*self.lens, 0]) if max_len is None else max_len)
        scale = 1.0 / np.sqrt(self.dim) if scale is None else scale
        want, reach, most = ref.attention(q.float().cpu().numpy(), self.want, self.table, self.lens, self.starts, scale, window, cap, np.full(out.shape, 7.0))
        got = out.double().cpu().numpy()
        # What may be lost. A score is a sum of dim products of up to three pieces, exact ones, in f32: 3 dim half steps of 2^-24 of the sum of
        # their sizes (`reach`) at the very most; its factor, log2(e) and the difference to the maximum 6 more. A cap adds its tanh's 2^-22. A score that is
        # off by e shifts a weighted mean of values by up to 2 e of the largest. The power of two and the sums of weights and of values: 2^-22 each, and
        # a half step an addition in the sums, of which there are as many as positions, relative to sums of weights. Weights are held to
        # 24 bits (f32), 16 or 8: to half a step of 2^-24, 2^-16 or 2^-8. Then the output's rounding, half a step.
        fine = self.dtype == "f32"
        score = (3 * self.dim + 6) * 2.0 ** -24 * reach + (cap * 2.0 ** -22 if cap else 0.0)
        length = max([*self.lens, 1])
        bound = most * (2 * score + 4 * 2.0 ** -22 + 2 * length * 2.0 ** -24 + (2.0 ** -24 if fine else 2.0 ** -9 if self.dtype == "bf16" else 2.0 ** -17))
        step = 2.0 ** -24 if fine else torch.finfo(q.dtype).eps / 2
        assert np.isfinite(got).all()
        off = np.abs(got - want) - step * np.abs(want) - bound[..., None]
        assert (off <= 0).all(), (off.max(), np.abs(got - want).max())
        return out


HEADS = [(4, 1, 128), (2, 2, 64), (8, 1, 256), (6, 2, 64), (16, 8, 128), (5, 1, 64), (20, 1, 128), (32, 4, 128), (4, 4, 256)]


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


@pytest.mark.parametrize("fresh", [1, 20])
def test_pages_behind_32_bit_offsets(fresh):
    """The same pages of a small cache and of one whose codes pass 2^32 bytes: the same rows, bit for bit."""
    b = Batch([700, 300], [fresh, fresh], 4, 2, 256, 256, "bf16", seed=3)
    small = b.cache()
    at = b.q.cuda(), i32(b.lens), i32(b.starts)
    want = kv.kv_attention(at[0], small, i32(b.table), *at[1:], max_fresh=fresh, max_len=700)
    pages = (1 << 32) // (2 * 256 * 128) + small.pages
    large = kv.KvCacheMxfp4.empty(pages, 2, 256, 256)
    to = torch.arange(pages - small.pages, pages, device="cuda")
    to[0] = 1
    for into, of in zip((large.k, large.v, large.k_powers, large.v_powers), (small.k, small.v, small.k_powers, small.v_powers)):
        into[to] = of
    assert large.k[int(to[1]):].data_ptr() - large.k.data_ptr() >= 1 << 32
    table = np.where(b.table >= 0, to.cpu().numpy()[np.maximum(b.table, 0)], -1).astype(np.int32)
    got = kv.kv_attention(at[0], large, i32(table), *at[1:], max_fresh=fresh, max_len=700)
    assert torch.equal(got, want)


@pytest.mark.parametrize("dtype", ["f32", "f16"])
@pytest.mark.parametrize("window", [1, 2, 16, 17, 63, 64, 100, 1000, 0x7FFFFFFF])
def test_windows(window, dtype):
    Batch([1, 70, 500, 260], [1, 1, 3, 90], 4, 2, 64, 16, dtype, seed=window & 255).check(window=window)


@pytest.mark.parametrize("dtype", sorted(TYPES))
@pytest.mark.parametrize("cap,scale", [(50.0, None), (30.0, 0.5), (1.0, 3.0), (1e-3, 1.0), (1e6, None)])
def test_capped_scores(cap, scale, dtype):
    Batch([1, 70, 500, 260], [1, 4, 3, 90], 4, 2, 128, 16, dtype, seed=int(cap) & 255).check(cap=cap, scale=scale)


@pytest.mark.parametrize("dtype", sorted(TYPES))
@pytest.mark.parametrize("fresh", [1, 40])
@pytest.mark.parametrize("cap", [1e4, 1e9])
def test_a_cap_far_above_the_scores(cap, fresh, dtype):
    """cap tanh(s / cap) is s but for s^3 / (3 cap^2): what is asked of the scores as they are, of scores up to 30."""
    b = Batch([300, 77], [fresh, fresh], 4, 2, 64, 16, dtype, seed=11)
    plain = b.check().double()
    at = b.q.cuda(), b.cache(), i32(b.table), i32(b.lens), i32(b.starts)
    got = kv.kv_attention(*at, max_fresh=fresh, max_len=300, softcap=cap).double()
    want, reach, most = ref.attention(b.q.double().numpy(), b.want, b.table, b.lens, b.starts, 0.125, 0, 0.0, np.zeros(b.q.shape))
    assert reach.max() < 600
    # the bound of the scores as they are for either, and 8 half steps of a score more for the cap's product, series and product; s^3 / (3 cap^2) of a
    # score of 30 is below 1e-4 at 1e4
    fine, length = dtype == "f32", 300
    score = (3 * 64 + 6 + 8) * 2.0 ** -24 * reach + 30.0 ** 3 / (3 * cap ** 2)
    bound = most * (2 * score + 4 * 2.0 ** -22 + 2 * length * 2.0 ** -24 + (2.0 ** -24 if fine else 2.0 ** -9 if dtype == "bf16" else 2.0 ** -17))
    step = 2.0 ** -24 if fine else torch.finfo(TYPES[dtype]).eps / 2
    for out in (plain, got):
        off = np.abs(out.cpu().numpy() - want) - step * np.abs(want) - bound[..., None]
        assert (off <= 0).all(), off.max()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("hint", [(0, 0), (1, 1), (1, 100000), (5000, 1), (5000, 100000)])
def test_sizes_given_are_hints(hint, dtype):
    """The caller's idea of the most rows and tokens of a sequence chooses launches, not results."""
    Batch([700, 90, 260, 0, 2500], [1, 4, 150, 0, 2], 8, 2, 128, 16, dtype, seed=5, pad=6).check(max_fresh=hint[0], max_len=hint[1])


@pytest.mark.parametrize("dtype", sorted(TYPES))
def test_rows_behind_the_last_sequence_and_empty_sequences(dtype):
    out = Batch([0, 50, 7, 0, 90], [0, 1, 0, 0, 1], 4, 1, 64, 16, dtype, seed=3, pad=9).check()
    assert (out[2:] == 7).all()


@pytest.mark.parametrize("dtype", sorted(TYPES))
@pytest.mark.parametrize("lens,fresh", [([4000], [1]), ([9000, 130, 5000], [1, 1, 1]), ([4000, 1, 2700, 900, 9, 5000, 4100, 3900], [1] * 8), ([3000, 2500], [5, 6])])
def test_long_contexts(lens, fresh, dtype):
    """Parts of a context, and pieces of a batch's."""
    Batch(lens, fresh, 8, 4, 64, 32, dtype, seed=sum(lens) & 255).check()


@pytest.mark.parametrize("dtype", sorted(TYPES))
@pytest.mark.parametrize("heads,kv_heads,dim,fresh,window", [(8, 4, 128, [1] * 8, 0), (4, 4, 256, [1, 1, 3, 0, 1, 2, 1, 1], 0), (16, 4, 64, [1, 1, 2, 1, 0, 1, 2, 1], 1500), (4, 4, 64, [1, 1, 1, 60, 1, 1, 1, 1], 0)])
def test_pieces_of_a_batch(heads, kv_heads, dim, fresh, window, dtype):
    """A table that is wide enough for long contexts, by which the batch is cut into pieces of equal lengths, and sequences that begin and end in them."""
    b = Batch([4000, 1, 2700, 900, 9, 700, 4100, 130], fresh, heads, kv_heads, dim, 16, dtype, seed=7, pad=2)
    b.table = np.concatenate([b.table, np.full((8, 4000 - b.table.shape[1]), -1, np.int32)], 1)
    b.check(max_len=64000, window=window)


@pytest.mark.parametrize("dtype", sorted(TYPES))
@pytest.mark.parametrize("fresh", [1, 3, 70])
def test_absent_pages(fresh, dtype):
    b = Batch([200, 100, 700], [fresh] * 3, 4, 2, 128, 16, dtype, seed=fresh)
    b.table[0, :-1] = -1                       # a sequence that sees nothing
    b.table[1, 2] = len(b.want.codes["k"])     # a page past the cache
    b.table[2, [0, 5, 6, 7, 8, 20]] = [-1, -7, -1, 1 << 30, -1, -1]
    out = b.check()
    assert (out[:fresh] == 0).all()


@pytest.mark.parametrize("dtype", sorted(TYPES))
@pytest.mark.parametrize("fresh,window", [(1, 0), (1, 40), (5, 40), (90, 0), (90, 30)])
def test_what_no_row_sees_may_hold_anything(fresh, window, dtype):
    """Tokens behind a sequence's last one, pages in front of a window and other sequences' pages: powers that are no number, the largest ones."""
    b = Batch([100, 205], [fresh] * 2, 4, 2, 128, 32, dtype, seed=fresh)
    clean = b.cache()
    seen = np.zeros((len(b.want.codes["k"]), 32), bool)
    for i, n in enumerate(b.lens):
        for at in range(max(0, int(n) - fresh - window + 1) if window else 0, int(n)):
            seen[b.table[i, at // 32], at % 32] = True
    want = b.check(window=window, cache=clean)
    for bad in (255, 254):
        for s in "kv":
            b.want.powers[s][~seen[:, None].repeat(2, 1)] = bad
            b.want.codes[s][~seen[:, None].repeat(2, 1)] = 15
        out = torch.full_like(want, 7.0)
        kv.kv_attention(b.q.cuda(), b.cache(), i32(b.table), i32(b.lens), i32(b.starts), window=window, out=out, max_fresh=fresh, max_len=205)
        assert torch.equal(out, want)


@pytest.mark.parametrize("dtype", sorted(TYPES))
@pytest.mark.parametrize("fresh", [1, 40])
def test_rows_that_are_no_numbers(fresh, dtype):
    b = Batch([100, 300], [fresh] * 2, 4, 2, 64, 16, dtype, seed=1)
    q = b.q.cuda()
    want = b.check()
    q[0, 1, 3], q[fresh, 2, 60], q[fresh, 0, 0] = float("nan"), float("inf"), float("-inf")
    out = torch.full_like(want, 7.0)
    kv.kv_attention(q, b.cache(), i32(b.table), i32(b.lens), i32(b.starts), out=out, max_fresh=fresh, max_len=300)
    for r, h in ((0, 1), (fresh, 2), (fresh, 0)):
        assert torch.isnan(out[r, h]).all()
        out[r, h] = want[r, h]
    assert torch.equal(out, want)


def test_every_bit_of_an_f32_query_counts():
    """Two scores that differ by the last bit of a query's value, at a scale that makes it one."""
    c = ref.Cache(1, 1, 16, 64)
    c.codes["k"][0, 0, 0, :2], c.codes["k"][0, 0, 1, :2] = [2, 10], [10, 2]      # (1, -1) and (-1, 1)
    c.powers["k"][:], c.powers["v"][:] = 127, 127
    c.codes["v"][0, 0, 0], c.codes["v"][0, 0, 1] = 2, 10
    q = torch.zeros((1, 1, 64), device="cuda")
    q[0, 0, 0], q[0, 0, 1] = 1 + 2.0 ** -23, 1
    out = kv.kv_attention(q, handle(c), i32([[0]]), i32([2]), i32([0, 1]), max_fresh=1, max_len=2, scale=2.0 ** 22)
    want = np.tanh(0.5)     # weights e^(1/2) and e^(-1/2)
    assert np.abs(out.double().cpu().numpy() - want).max() <= 2.0 ** -21


@pytest.mark.parametrize("dtype", sorted(TYPES))
@pytest.mark.parametrize("fresh", [1, 50])
@pytest.mark.parametrize("powers", [(31, 32), (60, 61), (100, 140)])
def test_powers_far_from_one(powers, fresh, dtype):
    """Small values lose nothing, and large ones beside them are weighed as they are. (Scores by a scale that keeps them near one.)"""
    b = Batch([130, 70], [fresh] * 2, 4, 2, 64, 16, dtype, seed=powers[0], powers=powers)
    if powers == (100, 140):
        b.want.powers["k"][:] = 126
        scale = None
    else:
        scale = 2.0 ** (127 - powers[0] - 4)
    if dtype == "f16":      # (its own values go no lower than 2^-24)
        b.want.powers["v"][:] = 128
    b.check(scale=scale)


def test_strided_rows_and_outputs():
    b = Batch([70, 300, 41], [1, 4, 40], 6, 2, 64, 16, "bf16", seed=4)
    wide = torch.full((b.rows, 11, 64), 3.0, dtype=torch.bfloat16, device="cuda")
    wide[:, 1:7] = b.q.cuda()
    out = torch.full((b.rows, 9, 64), 5.0, dtype=torch.bfloat16, device="cuda")
    kv.kv_attention(wide[:, 1:7], b.cache(), i32(b.table), i32(b.lens), i32(b.starts), out=out[:, 2:8], max_fresh=40, max_len=300)
    assert torch.equal(out[:, 2:8], b.check()) and (out[:, :2] == 5).all() and (out[:, 8:] == 5).all()


ATTENTION = {"a context in parts": ([9000], [1], "f32", 8, 2), "contexts in pieces": ([4000, 1, 2700, 3000, 9, 5000, 4100, 3900], [1] * 8, "f16", 16, 16),
             "a chunk in parts": ([3000], [40], "bf16", 8, 2), "a chunk beside single rows": ([2500, 2400, 70], [33, 1, 1], "f32", 8, 2)}


@pytest.mark.parametrize("what", sorted(ATTENTION))
def test_recorded_attention_beside_other_calls(what):
    """Graphs and eager calls on streams that nothing orders, in the library's scratch memory."""
    lens, fresh, dtype, heads, kv_heads = ATTENTION[what]

    def call(seed):
        b = Batch(lens, fresh, heads, kv_heads, 64, 32, dtype, seed=seed)
        at = (b.q.cuda(), b.cache(), i32(b.table), i32(b.lens), i32(b.starts))
        return lambda: kv.kv_attention(*at, max_fresh=max(fresh), max_len=max(lens), softcap=30.0)

    check_replays([call(seed) for seed in (1, 2, 3)], torch.cuda.Stream())


@pytest.mark.parametrize("dtype", sorted(TYPES))
@pytest.mark.parametrize("fresh", [1, 5, 50])
@pytest.mark.parametrize("page,cols", [(16, 1), (16, 9), (16, 7), (16, 18), (32, 3), (32, 5)])
def test_lengths_past_the_end_of_the_table(page, cols, fresh, dtype):
    """Positions whose column the table does not have are absent: of a sequence that ends inside the step in which the table does, of one that ends far
    behind it, and of one that ends before."""
    limit = page * cols
    lens = [max(limit - 3, fresh), max(limit + 1, fresh), max(limit | 63, fresh), limit + 300]
    b = Batch(lens, [fresh] * 4, 4, 2, 64, page, dtype, seed=cols)
    b.table = np.ascontiguousarray(b.table[:, :cols])
    b.check()
    b.check(window=90)


@pytest.mark.parametrize("dtype", sorted(TYPES))
@pytest.mark.parametrize("heads,kv_heads,dim,fresh", [(8, 4, 128, 1), (4, 4, 256, 2), (16, 4, 64, 9)])
def test_long_lengths_past_the_end_of_the_table(heads, kv_heads, dim, fresh, dtype):
    """The same of contexts in parts and of a batch in pieces."""
    for lens in ([4000, 300, 2700, 900, 1500, 700, 4100, 130], [9000]):
        b = Batch(lens, [fresh] * len(lens), heads, kv_heads, dim, 16, dtype, seed=dim)
        b.table = np.ascontiguousarray(b.table[:, :157])
        b.check()
        b.check(max_len=64000)


def test_starts_past_the_batch_are_cut():
    """A plan of more rows than the batch holds: those that it holds are computed, nothing is written behind it."""
    b = Batch([40, 60], [10, 20], 2, 1, 64, 16, "f32", seed=12)
    guard = torch.full((40, 2, 64), 9.0, device="cuda")
    kv.kv_attention(b.q[:17].cuda().contiguous(), b.cache(), i32(b.table), i32(b.lens), i32(b.starts), max_fresh=20, max_len=60, out=guard[:17])
    assert (guard[17:] == 9).all()
    b.q, b.rows = b.q[:17], 17
    assert torch.equal(b.check(max_fresh=20, max_len=60), guard[:17])


@pytest.mark.parametrize("dtype", sorted(TYPES))
@pytest.mark.parametrize("hint", [1, 40])
def test_first_rows_far_outside_the_batch(hint, dtype):
    """Rows that a sequence claims are those of the batch at most, whatever `starts` holds."""
    b = Batch([300, 200, 100], [0, 0, 0], 4, 2, 64, 16, dtype, pad=40)
    out = torch.full((b.rows, b.heads, b.dim), 7.0, dtype=TYPES[dtype], device="cuda")
    for starts, want in (([2000000000, -2000000000, -2147483648, -2147483648], 7.0), ([2147483647, -2147483648, 2147483647, -2147483648], 0.0),
                         ([2147483647, -5, -2147483648, 0], 7.0)):
        out.fill_(7.0)
        kv.kv_attention(b.q.cuda(), b.cache(), i32(b.table), i32(b.lens), i32(starts), max_fresh=hint, max_len=300, out=out)
        assert (out == want).all()


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


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("fresh", [1, 30])
def test_queries_whose_scale_alone_would_overflow(fresh, dtype):
    """Scores of ordinary size from queries at the end of the type's range and the smallest keys."""
    b = Batch([200], [fresh], 4, 2, 64, 16, dtype, seed=31, powers=(31, 34))
    b.want.powers["v"][:] = 127
    b.q = (b.q.float() * 7e37).clamp(-3e38, 3e38)
    b.q[..., 5] = 3e38
    b.q = b.q.to(TYPES[dtype])
    b.check(scale=2.0 ** -33)


@pytest.mark.parametrize("fresh", [1, 6, 40])
def test_the_largest_f32_queries(fresh):
    """Values within a bf16's half step of f32's end, which round to infinity as one."""
    b = Batch([200], [fresh], 4, 2, 64, 16, "f32", seed=31, powers=(31, 32))
    b.want.powers["v"][:] = 127
    most = float(np.finfo(np.float32).max)
    b.q[..., 5], b.q[..., 9] = most, -most * (1 - 2.0 ** -10)
    b.check(scale=2.0 ** -33)


def two_positions(fresh, heads, dtype, seed):
    """Sequences whose rows see a position 0 of score 0 and value 1, a position 1 of score -d (a row and head's own) and value -1, and others of
    weight 0: an output is tanh(d / 2), the difference of two weights that are nearly equal."""
    g = np.random.default_rng(seed)
    c = ref.Cache(6, 1, 16, 64)
    c.powers["k"][:], c.powers["v"][:] = 127, 127
    c.codes["k"][:, 0, :, 1], c.powers["k"][..., 0] = 15, 136   # -6 * 2^9
    c.codes["k"][0, 0, 0], c.codes["k"][0, 0, 1] = 0, 0
    c.codes["k"][0, 0, 1, 0], c.powers["k"][0, 0, 1] = 10, 127   # -1
    c.codes["v"][:] = 7
    c.codes["v"][0, 0, 0], c.codes["v"][0, 0, 1] = 2, 10
    q = torch.zeros((fresh, heads, 64), dtype=TYPES[dtype])
    q[:, :, 0] = torch.tensor(2.0 ** g.uniform(-9, -6, (fresh, heads))).to(TYPES[dtype])
    q[:, :, 1] = 1
    return c, q


@pytest.mark.parametrize("dtype", sorted(TYPES))
@pytest.mark.parametrize("fresh,heads", [(1, 1), (1, 4), (3, 1), (2, 4), (6, 1), (5, 3), (4, 4), (40, 1), (30, 5)])
def test_the_weights_bits(fresh, heads, dtype):
    """Weights are held to 24 bits in f32, to 16 in f16 and bf16: what is left of a difference of two says so."""
    for seed in range(4):
        c, q = two_positions(fresh, heads, dtype, seed)
        length = 2 + fresh
        out = kv.kv_attention(q.cuda(), handle(c), i32([range(6)]), i32([length]), i32([0, fresh]), max_fresh=fresh, max_len=length, scale=1.0)
        want = np.tanh(q[:, :, :1].double().numpy() / 2)
        # The weights 1 and w = e^-d: w's power of two and its argument are off by 2^-22, the weight as it goes into the product by half a step of its pieces,
        # 2^-24 (three) or 2^-16 (two), each halved by 1 / (1 + w). Sums, quotient: 2^-22 of the result. Then the result's rounding.
        pieces = 3 if dtype == "f32" else 2
        step = 2.0 ** -24 if dtype == "f32" else torch.finfo(TYPES[dtype]).eps / 2
        bound = 0.5 * (2.0 ** -22 + 2.0 ** (-8 * pieces)) + (step + 2.0 ** -22) * np.abs(want)
        off = np.abs(out.double().cpu().numpy() - want)
        assert (off <= bound).all(), (off.max(), bound.max())


@pytest.mark.parametrize("fresh,heads", [(1, 1), (2, 2), (6, 1), (4, 4), (40, 1)])
@pytest.mark.parametrize("dtype,bit", [("f32", 23), ("f16", 10), ("bf16", 7)])
def test_every_bit_of_a_query_counts(dtype, bit, fresh, heads):
    """Two scores that differ by the last bit of a query's value, at a scale that makes it one half either way; others of weight 0."""
    c = ref.Cache(4, 1, 16, 64)
    c.powers["k"][:], c.powers["v"][:] = 127, 127
    c.codes["k"][:, 0, :, 2] = 15
    c.codes["k"][0, 0, :2, 2] = 0
    c.codes["k"][0, 0, 0, :2], c.codes["k"][0, 0, 1, :2] = [2, 10], [10, 2]      # (1, -1) and (-1, 1)
    c.codes["v"][0, 0, 0], c.codes["v"][0, 0, 1] = 2, 10
    q = torch.zeros((fresh, heads, 64))
    q[..., 0], q[..., 1], q[..., 2] = 1 + 2.0 ** -bit, 1, 1
    out = kv.kv_attention(q.to(TYPES[dtype]).cuda(), handle(c), i32([range(4)]), i32([2 + fresh]), i32([0, fresh]), max_fresh=fresh, max_len=2 + fresh,
                          scale=2.0 ** (bit - 1))
    want = np.tanh(0.5)     # weights e^(1/2) and e^(-1/2)
    # (a weight of e^-1 in two pieces is off by 2^-16 of itself, which the quotient makes 2 / (1 + e^-1)^2 = 1.07 of; the result's rounding)
    step = 2.0 ** -21 if dtype == "f32" else 2.0 ** -16 + torch.finfo(TYPES[dtype]).eps / 2 * want
    assert np.abs(out.double().cpu().numpy() - want).max() <= step
    assert out.shape == (fresh, heads, 64)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("fresh", [1, 6, 40])
@pytest.mark.parametrize("scale", [0.125, 4.0])
def test_values_near_the_end_of_f32(scale, fresh, dtype):
    """130 positions of up to 6 * 2^110, in scores of any order: 2^8 times all of them is a number still."""
    b = Batch([130, 70], [fresh] * 2, 4, 2, 64, 16, dtype, seed=60)
    b.want.powers["v"][:] = 110 + 127
    b.check(scale=scale)


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
    b = Batch(lens, fresh, 16, 16, 64, 16, dtype, seed=41, pad=3)
    b.table = np.concatenate([b.table, np.full((43, 4100 - b.table.shape[1]), -1, np.int32)], 1)     # (room for contexts that are worth pieces)
    out = b.check(window=700 if what == "window" else 0, max_fresh=2 if what != "beside a prompt" else 70, max_len=64000)
    assert (out[-3:] == 7).all()


@pytest.mark.parametrize("dtype", sorted(TYPES))
def test_a_row_does_not_depend_on_its_companions(dtype):
    """The same sequence alone and in a batch, and the same call again: the same bits, but for contexts that are cut elsewhere."""
    b = Batch([500, 60, 900], [1, 1, 1], 8, 2, 128, 16, dtype, seed=31)
    whole = b.check(max_len=900)
    for i in range(3):
        one = kv.kv_attention(b.q[i:i + 1].cuda(), b.cache(), i32(b.table[i:i + 1]), i32(b.lens[i:i + 1]), i32([0, 1]), max_fresh=1, max_len=900)
        assert (one[0].float() - whole[i].float()).abs().max() <= (2e-5 if dtype == "f32" else 2 * torch.finfo(TYPES[dtype]).eps) * whole[i].float().abs().max()
    assert torch.equal(whole, b.check(max_len=900))
