"""The plan of pages and slots and the paged 8-bit cache against their definitions in 64 bits: whole numbers and codes equal."""
import numpy as np
import pytest

torch = pytest.importorskip("torch")

import serving_reference as ref
from loken_amd import kv, lib

pytestmark = pytest.mark.gpu


def i32(v):
    return torch.tensor(np.asarray(v, np.int32), device="cuda")


def i64(v):
    return torch.tensor(np.asarray(v, np.int64), device="cuda")


# ------------------------------------------------------------------------------------------ the plan
def check_plan(past, fresh, page, rows, cols, free, taken=0, stride=None):
    seqs = len(past)
    table = np.full((seqs, cols), -1, np.int32)
    nxt = 1000
    for i, p in enumerate(past):
        for c in range(min(-(-max(p, 0) // page), cols)):
            table[i, c], nxt = nxt, nxt + 3
    whole = torch.full((seqs, stride or cols), -7, dtype=torch.int32, device="cuda")
    whole[:, :cols] = i32(table)
    plan = kv.KvPlan(seqs, rows)
    for t in (plan.lens, plan.starts, plan.slots, plan.positions, plan.taken):
        t.fill_(-99)
    kv.kv_plan(i32(past), i32(fresh), whole[:, :cols], i32(free), page, plan, taken=i32([taken]) if taken else None)
    want = ref.plan(past, fresh, table, free, page, rows, taken)
    for got, w in zip((whole[:, :cols], plan.lens, plan.starts, plan.slots, plan.positions), want):
        assert np.array_equal(got.cpu().numpy(), w)
    assert int(plan.taken) == want[5]
    assert (whole[:, cols:] == -7).all()


@pytest.mark.parametrize("page", [16, 32, 64, 128, 256])
@pytest.mark.parametrize("seqs,most_past,most_fresh", [(1, 0, 1), (1, 5000, 1), (7, 100, 40), (64, 300, 1), (300, 60, 90), (1025, 40, 3)])
def test_plan_of_ragged_batches(page, seqs, most_past, most_fresh):
    g = np.random.default_rng(seqs * page)
    past, fresh = g.integers(0, most_past + 1, seqs), g.integers(0, most_fresh + 1, seqs)
    rows, cols = int(fresh.sum()) + 13, (most_past + most_fresh) // page + 2
    check_plan(past, fresh, page, rows, cols, g.permutation(seqs * cols + 9), taken=int(g.integers(0, 9)), stride=cols + 5)


@pytest.mark.parametrize("what", ["no sequences", "no rows", "nothing new", "list runs out", "no list", "row of the table ends", "more rows than the batch holds",
                                  "lengths below zero", "on the border of a page"])
def test_plan_at_its_edges(what):
    free = np.arange(50, 90)
    if what == "no sequences":
        plan = kv.KvPlan(0, 5)
        kv.kv_plan(i32([]), i32([]), torch.empty((0, 4), dtype=torch.int32, device="cuda"), i32(free), 16, plan, taken=i32([4]))
        assert plan.starts.tolist() == [0] and plan.slots.tolist() == [-1] * 5 and plan.positions.tolist() == [0] * 5 and int(plan.taken) == 4
    else:
        check_plan(*{"no rows": ([3, 20], [1, 2], 16, 0, 4, free), "nothing new": ([3, 0, 20], [0, 0, 0], 16, 4, 4, free),
                     "list runs out": ([0, 30, 5], [40, 50, 60], 16, 160, 8, free[:5]), "no list": ([0, 30], [4, 5], 16, 12, 4, free[:0]),
                     "row of the table ends": ([10, 60], [100, 100], 16, 210, 5, free), "more rows than the batch holds": ([0, 9], [30, 30], 16, 35, 6, free),
                     "lengths below zero": ([-5, 7, 3], [4, -2, 2], 16, 8, 3, free), "on the border of a page": ([16, 15, 17, 32], [16, 1, 15, 0], 16, 33, 4, free)}[what])


def test_the_largest_plan():
    seqs = kv.PLAN_SEQS
    g = np.random.default_rng(3)
    past, fresh = g.integers(0, 40, seqs), g.integers(0, 4, seqs)
    check_plan(past, fresh, 16, int(fresh.sum()) + 70, 4, g.permutation(seqs))


@pytest.mark.parametrize("seqs,most_fresh", [(3, 5), (700, 4)])
def test_plan_of_arrays_side_by_side(seqs, most_fresh):
    """All arrays of a plan in one allocation, each starting where another ends; and past and taken from the plan before."""
    g = np.random.default_rng(seqs)
    past, fresh, cols = g.integers(0, 60, seqs), g.integers(0, most_fresh + 1, seqs), 6
    rows, free = int(fresh.sum()) + 7, g.permutation(seqs * 9)
    sizes = dict(slots=2 * rows, past=seqs, lens=seqs, fresh=seqs, taken=1, out=1, free=len(free), table=seqs * cols, starts=seqs + 1, positions=rows)
    whole, at = torch.full((sum(sizes.values()),), -99, dtype=torch.int32, device="cuda"), {}
    for name, n in sizes.items():
        first = sum(v.numel() for v in at.values())
        at[name] = whole[first:first + n]
    table = np.full((seqs, cols), -1, np.int32)
    for i, p in enumerate(past):
        table[i, :-(-p // 16)] = np.arange(-(-p // 16)) + 10 * i
    for name, v in (("past", past), ("fresh", fresh), ("free", free), ("table", table.reshape(-1)), ("taken", [2])):
        at[name].copy_(i32(v))
    L = lib.load()

    def plan(a):
        lib.check("lk_kv_plan", L.lk_kv_plan(a["past"].data_ptr(), a["fresh"].data_ptr(), seqs, 16, a["free"].data_ptr(), len(free), a["taken"].data_ptr(),
                                             a["table"].data_ptr(), cols, cols, a["lens"].data_ptr(), a["starts"].data_ptr(), a["slots"].data_ptr(),
                                             a["positions"].data_ptr(), rows, a["out"].data_ptr(), torch.cuda.current_stream().cuda_stream))

    taken, lens = 2, past
    other = {n: torch.empty_like(v) for n, v in at.items()}
    for step in range(4):   # what was written is read by the next one, which writes the other arrays
        a, b = (at, other) if step % 2 == 0 else (other, at)
        plan(a)
        table, lens, starts, slots, positions, taken = ref.plan(lens, fresh, table, free, 16, rows, taken)
        for name, want in (("table", table.reshape(-1)), ("lens", lens), ("starts", starts), ("positions", positions), ("out", [taken])):
            assert np.array_equal(a[name].cpu().numpy(), want), (step, name)
        assert np.array_equal(a["slots"].view(torch.int64).cpu().numpy(), slots)
        for name, v in (("past", a["lens"]), ("taken", a["out"]), ("fresh", a["fresh"]), ("free", a["free"]), ("table", a["table"])):
            b[name].copy_(v)


# ------------------------------------------------------------------------------------------ the cache
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def check_cache(cache, want):
    v = cache.v.cpu().numpy().transpose(0, 1, 2, 4, 3).reshape(want.codes["v"].shape)
    assert np.array_equal(cache.k_scales.cpu().numpy(), want.scales["k"])
    assert np.array_equal(cache.v_scales.cpu().numpy(), want.scales["v"])
    assert np.array_equal(cache.k.cpu().numpy(), want.codes["k"])
    assert np.array_equal(v, want.codes["v"])


def both(pages, heads, page, dim):
    return kv.KvCacheQ8.empty(pages, heads, dim, page), ref.Cache(pages, heads, page, dim)


def rows_of(g, tokens, heads, dim, dtype, spread=1.0):
    x = torch.tensor(g.normal(size=(tokens, heads, dim)) * spread, dtype=torch.float32).to(dtype)
    return x


def write(cache, want, k, v, slots):
    kv.kv_write(cache, k.cuda(), v.cuda(), i64(slots))
    want.write(k.float().numpy(), v.float().numpy(), np.asarray(slots))


@pytest.mark.parametrize("dtype", sorted(TYPES))
@pytest.mark.parametrize("page,dim,heads", [(16, 128, 2), (32, 64, 3), (64, 256, 1), (128, 128, 2), (256, 64, 1)])
def test_steps_of_several_sequences(page, dim, heads, dtype):
    """Prompts that end inside pages, then tokens one by one whose values grow: a page's scale grows and its codes go with it."""
    g = np.random.default_rng(page + dim)
    cache, want = both(12, heads, page, dim)
    tables = [[3, 7, 1], [0, 11, 5], [9, 2, 4]]
    lens = [0, 0, 0]
    for step, fresh in enumerate(([page + 5, 1, 2 * page], [1, 1, 1], [2, 0, 1], [1, 3, 1], [1, 1, page - 1 - 2])):
        slots = []
        for i, f in enumerate(fresh):
            slots += [tables[i][at // page] * page + at % page for at in range(lens[i], lens[i] + f)]
            lens[i] += f
        write(cache, want, rows_of(g, len(slots), heads, dim, TYPES[dtype], 1.0 + step), rows_of(g, len(slots), heads, dim, TYPES[dtype], 3.0 - step / 2), slots)
        check_cache(cache, want)


@pytest.mark.parametrize("what", ["absent", "past the cache", "a slot twice", "falling order", "over what was there", "many rows", "one page many times"])
def test_slots_of_all_kinds(what):
    g = np.random.default_rng(7)
    cache, want = both(40, 2, 16, 64)
    write(cache, want, rows_of(g, 48, 2, 64, torch.float32), rows_of(g, 48, 2, 64, torch.float32), range(48))
    slots = {"absent": [-1, 48, -1, 49, -5, 80, -1], "past the cache": [640, 100, 641, 1 << 40], "a slot twice": [21, 21, 22, 22, 22],
             "falling order": [47, 46, 45, 44, 70, 69, 68], "over what was there": [18, 19, 20, 33], "many rows": list(range(64, 640)),
             "one page many times": [40 + (i * 5) % 8 for i in range(150)]}[what]
    write(cache, want, rows_of(g, len(slots), 2, 64, torch.float32, 2.0), rows_of(g, len(slots), 2, 64, torch.float32, 0.5), slots)
    check_cache(cache, want)


def test_values_at_the_border_of_two_codes():
    """Quotients that are whole numbers and a half exactly, and their neighbours in 32 bits on either side."""
    cache, want = both(2, 1, 16, 64)
    s = np.float32(0.3)
    half = (np.arange(64) - 32 + 0.5) * np.float64(s)
    x = np.stack([half.astype(np.float32), np.nextafter(half.astype(np.float32), np.float32(np.inf)), np.nextafter(half.astype(np.float32), np.float32(-np.inf))])[:, None]
    x = np.concatenate([x, np.full((1, 1, 64), np.float32(127 * np.float64(s)))])
    exact = ((np.arange(64) - 32 + 0.5) * 0.25).astype(np.float32)
    y = np.concatenate([np.stack([exact, np.nextafter(exact, np.float32(9)), np.nextafter(exact, np.float32(-9))])[:, None], np.full((1, 1, 64), np.float32(31.75))])
    write(cache, want, torch.tensor(x), torch.tensor(y), range(4))
    check_cache(cache, want)
    assert (cache.k_scales[0, 0] != 0) and float(cache.v_scales[0, 0]) == 0.25
    # the scale doubles: odd codes stand at a half exactly
    write(cache, want, torch.tensor(x[3:]) * 2, torch.full((1, 1, 64), 63.5), [4])
    check_cache(cache, want)


@pytest.mark.parametrize("bad", [float("inf"), float("-inf"), float("nan")])
@pytest.mark.parametrize("zeros", [False, True])
def test_values_that_are_not_finite(bad, zeros):
    g = np.random.default_rng(9)
    cache, want = both(2, 1, 16, 64)
    k = rows_of(g, 3, 1, 64, torch.float32) * (0 if zeros else 1)
    k[1, 0, 5] = bad
    write(cache, want, k, rows_of(g, 3, 1, 64, torch.float32), [0, 1, 2])
    check_cache(cache, want)
    k2, v2 = kv.kv_read(cache, i64([0, 1, 2]))
    assert torch.isfinite(k2).all() and torch.isfinite(v2).all()


@pytest.mark.parametrize("size", [0.0, 1e-45, 1e-40, 1.4e-36, 1e-30, 1e37, 3.4e38])
def test_small_and_large_values(size):
    g = np.random.default_rng(4)
    cache, want = both(2, 1, 16, 64)
    x = torch.tensor(np.clip(g.normal(size=(5, 1, 64)), -1, 1) * size, dtype=torch.float32)
    write(cache, want, x, -x, range(5))
    check_cache(cache, want)


@pytest.mark.parametrize("dtype", sorted(TYPES))
def test_rows_that_are_parts_of_wider_ones_and_reads(dtype):
    g = np.random.default_rng(11)
    t = TYPES[dtype]
    cache, want = both(9, 2, 32, 128)
    wide = rows_of(g, 50, 9, 128, t).cuda()
    k, v = wide[:, 4:6], wide[:, 7:]
    slots = np.concatenate([np.arange(96, 140), [7, -1, 9, 10, 11, 300]])
    kv.kv_write(cache, k, v, i64(slots))
    want.write(k.float().cpu().numpy(), v.float().cpu().numpy(), np.where(slots >= 288, -1, slots))
    check_cache(cache, want)
    asked = np.concatenate([slots, [-3, 287, 288, 1 << 50], np.arange(90, 150)])
    gk, gv = kv.kv_read(cache, i64(asked), dtype=t)
    for side, got in (("k", gk), ("v", gv)):
        for i, s in enumerate(asked):
            row = want.values(side, s // 32)[:, s % 32] if 0 <= s < 288 else np.zeros((2, 128))
            # a product of 8 and 24 bits, rounded to 32 bits and then to the type
            assert np.allclose(got[i].double().cpu().numpy(), row, rtol=torch.finfo(t).eps / 2 + 2.0 ** -24, atol=0)
            assert torch.equal(got[i].cpu(), torch.tensor(row.astype(np.float32)).to(t)) or t == torch.float32


def test_no_rows():
    cache = kv.KvCacheQ8.empty(2, 1, 64)
    empty = torch.empty((0, 1, 64), device="cuda")
    kv.kv_write(cache, empty, empty, i64([]))
    assert kv.kv_read(cache, i64([]))[0].shape == (0, 1, 64)
    assert not cache.k.any()


def test_the_plan_s_slots_are_where_rows_go():
    """A page number that the free list holds but the cache does not is nobody's: the row is skipped."""
    g = np.random.default_rng(2)
    cache, want = both(4, 1, 16, 64)
    table = torch.full((2, 3), -1, dtype=torch.int32, device="cuda")
    plan = kv.kv_plan(i32([0, 0]), i32([20, 3]), table, i32([2, 77, 0]), 16, kv.KvPlan(2, 32))
    k = rows_of(g, 32, 1, 64, torch.float32)
    write(cache, want, k, k, np.where(plan.slots.cpu().numpy() >= 64, -1, plan.slots.cpu().numpy()))
    check_cache(cache, want)
    again = kv.KvCacheQ8.empty(4, 1, 64)
    kv.kv_write(again, k.cuda(), k.cuda(), plan.slots)
    assert torch.equal(again.k, cache.k) and torch.equal(again.v, cache.v)


def test_pages_behind_2_to_the_31_bytes():
    """Codes whose offset takes more than 32 bits."""
    pages = (1 << 31) // (16 * 64) + 5
    k = torch.zeros((pages, 1, 16, 64), dtype=torch.int8, device="cuda")
    v = torch.zeros((pages, 1, 1, 64, 16), dtype=torch.int8, device="cuda")
    cache = kv.KvCacheQ8(k, v, torch.zeros((pages, 1), device="cuda"), torch.zeros((pages, 1), device="cuda"))
    slots = (pages - 2) * 16 + np.arange(20)
    x = rows_of(np.random.default_rng(1), 20, 1, 64, torch.float32)
    kv.kv_write(cache, x.cuda(), x.cuda(), i64(slots))
    gk, gv = kv.kv_read(cache, i64(slots))
    assert torch.equal(gk, gv) and (gk.cpu() - x).abs().max() <= x.abs().max() / 127 / 2 * 1.001
    assert not k[:pages - 2].any() and not k[pages - 1, 0, 4:].any()


def test_calls_go_to_where_the_tensors_are():
    """A tensor of the cache that has been given other memory: rows go there, and come from there."""
    g = np.random.default_rng(5)
    cache, want = both(4, 2, 16, 64)
    old = [getattr(cache, n).data for n in ("k", "v", "k_scales", "v_scales")]   # (their memory stays)
    write(cache, want, rows_of(g, 20, 2, 64, torch.float32), rows_of(g, 20, 2, 64, torch.float32), range(20))
    before = [t.clone() for t in old]
    for n in ("k", "v", "k_scales", "v_scales"):
        getattr(cache, n).data = getattr(cache, n).clone()
    write(cache, want, rows_of(g, 9, 2, 64, torch.float32), rows_of(g, 9, 2, 64, torch.float32), range(20, 29))
    check_cache(cache, want)
    assert all(torch.equal(a, b) for a, b in zip(old, before))
    gk, gv = kv.kv_read(cache, i64(range(16, 29)))
    for side, got in (("k", gk), ("v", gv)):
        assert np.allclose(got.cpu().numpy(), want.values(side, 1)[:, :13].transpose(1, 0, 2), rtol=2.0 ** -23, atol=0)


@pytest.mark.parametrize("behind", [1, 63, 64, 200, 4000])
def test_rows_behind_the_last_sequence_are_not_a_run_s(behind):
    """A batch padded as a plan pads it, with anything in its rows behind the last: the same cache, and no more than a few times the time
    (66 times with 4000 were each of them taken as a row of the run)."""
    g = np.random.default_rng(behind)
    (cache, want), (exact, _) = both(9, 2, 64, 64), both(9, 2, 64, 64)
    n = 64 + 50 + 9
    slots = np.concatenate([np.arange(64, 128), np.arange(200, 250), np.arange(320, 329)])
    padded = np.concatenate([slots, np.full(behind, -1)])
    k, v = (torch.cat([rows_of(g, n, 2, 64, torch.float32), torch.full((behind, 2, 64), bad)]) for bad in (float("nan"), 1e30))
    for _ in range(2):
        write(cache, want, k, v, padded)
        kv.kv_write(exact, k[:n].cuda(), v[:n].cuda(), i64(slots))
    check_cache(cache, want)
    assert torch.equal(cache.k, exact.k) and torch.equal(cache.v, exact.v)
    if behind < 4000:
        return

    def time_of(rows, cache):
        args = k[:rows].cuda(), v[:rows].cuda(), i64(padded[:rows])
        took = []
        for _ in range(8):
            begin, end = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
            begin.record()
            for _ in range(20):
                kv.kv_write(cache, *args)
            end.record()
            end.synchronize()
            took.append(begin.elapsed_time(end))
        return min(took)

    assert time_of(n + behind, cache) < 12 * time_of(n, exact)
