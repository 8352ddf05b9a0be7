"""The 4-bit cache's rows, and head norms with rotation before it, against their definitions in 64 bits: codes and powers equal."""
import numpy as np
import pytest

torch = pytest.importorskip("torch")

import mxfp4_reference as ref
from loken_amd import kv, rotary
from test_gpu_graph_scratch import record

pytestmark = pytest.mark.gpu

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def dev(a, dtype=None):
    return torch.tensor(np.ascontiguousarray(a), device="cuda") if dtype is None else torch.tensor(np.ascontiguousarray(a)).to(dtype).cuda()


def handle(want):
    return kv.KvCacheMxfp4(*(dev(t) for t in want.tensors()))


def check_cache(cache, want):
    for got, w, name in zip((cache.k, cache.v, cache.k_powers, cache.v_powers), want.tensors(), ("k", "v", "k_powers", "v_powers")):
        assert np.array_equal(got.cpu().numpy(), w), name


def rows_of(dtype, g, *shape, scale=1.0):
    return torch.tensor(g.normal(size=shape) * scale, dtype=torch.float32).to(TYPES[dtype])


# ------------------------------------------------------------------------------------------ rows that are there already
@pytest.mark.parametrize("dtype", sorted(TYPES))
@pytest.mark.parametrize("kv_heads,dim,page,tokens", [(1, 64, 16, 1), (3, 64, 32, 37), (2, 128, 16, 65), (8, 128, 64, 5), (1, 256, 256, 300), (5, 256, 16, 2)])
def test_write_and_read(kv_heads, dim, page, tokens, dtype):
    g = np.random.default_rng(dim + tokens)
    pages = -(-tokens // page) + 3
    want = ref.Cache(pages, kv_heads, page, dim, seed=tokens)
    cache = handle(want)
    slots = g.permutation(pages * page)[:tokens]     # scattered, in any order
    slots[::7] = -1
    slots[tokens // 2] = pages * page + 3
    wide = rows_of(dtype, g, tokens, 2 * kv_heads + 1, dim)
    k, v = wide[:, :kv_heads], wide[:, kv_heads:2 * kv_heads]
    d = wide.cuda()
    kv.kv_write(cache, d[:, :kv_heads], d[:, kv_heads:2 * kv_heads], dev(slots))
    want.write(k.double().numpy(), v.double().numpy(), slots)
    check_cache(cache, want)
    for out in sorted(TYPES):
        got = kv.kv_read(cache, dev(slots), dtype=TYPES[out])
        for side, t in zip("kv", got):
            for i, s in enumerate(slots):
                if not 0 <= s < pages * page:
                    assert (t[i] == 0).all()
                    continue
                exact = torch.tensor(want.values(side, s // page)[:, s % page]).to(TYPES[out])
                assert torch.equal(t[i].cpu(), exact)


def test_values_at_the_borders():
    """Halves, the largest, zeros of either sign, infinities, no numbers, and powers at both ends."""
    unit = np.array([0, 0.25, 0.26, 0.5, 0.75, 0.74, 1, 1.25, 1.26, 1.5, 1.75, 1.74, 2, 2.5, 2.51, 3, 3.5, 3.49, 4, 5, 5.01, 6, 6.99, -0.0, -0.25, -0.75,
                     -2.5, -3.5, -5, -6, 0.1, -0.1])
    rows = []
    for e in (0, -3, 20, -90, -96, -97, 120):
        rows.append(unit * 2.0 ** e)
    rows.append(np.where(unit == 6.99, 7.0, unit))                    # the next power
    rows.append(np.zeros(32))
    rows.append(np.where(np.arange(32) == 3, np.inf, np.where(np.arange(32) == 9, -np.inf, np.where(np.arange(32) == 20, np.nan, unit))))
    rows.append(np.full(32, np.nan))
    rows.append(np.full(32, -np.inf))
    rows.append(np.where(np.arange(32) % 2, 3.4e38, -3.4e38))
    rows.append(np.full(32, 1e-45))
    rows.append(unit * 2.0 ** -99)
    x = np.stack(rows).astype(np.float32)
    x = np.concatenate([x, x[:(-len(x)) % 2]])
    x = x.reshape(-1, 1, 64)
    want = ref.Cache(2, 1, 16, 64)
    cache, slots = kv.KvCacheMxfp4.empty(2, 1, 64), np.arange(len(x)) + 5
    kv.kv_write(cache, dev(x), dev(-x), dev(slots))
    want.write(x, -x, slots)
    check_cache(cache, want)


def test_any_power_is_read():
    want = ref.Cache(16, 1, 16, 64)
    want.codes["k"][:] = (np.arange(64) % 16)[None, None, None]
    want.powers["k"][:] = np.arange(512).reshape(16, 1, 16, 2) % 256
    want.codes["v"][:], want.powers["v"][:] = want.codes["k"][..., ::-1], want.powers["k"][:, :, ::-1]
    cache, slots = handle(want), np.arange(256)
    for side, got in zip("kv", kv.kv_read(cache, dev(slots))):
        exact = np.stack([want.values(side, s // 16)[:, s % 16] for s in slots])
        assert np.array_equal(got.cpu().numpy(), exact.astype(np.float32), equal_nan=True)


# ------------------------------------------------------------------------------------------ norms and rotation
def turned(g, rows, heads, kv_heads, dim, dtype, pairs, axes, far=1 << 20):
    x = rows_of(dtype, g, rows, heads + 2 * kv_heads, dim)
    freq = (10000.0 ** (-np.arange(pairs) / max(pairs, 1))).astype(np.float32)
    pos = g.integers(0, far, (axes, rows)).astype(np.int32)
    axis = g.integers(0, axes, pairs).astype(np.uint8) if axes > 1 else None
    return x, freq, pos, axis


CASES = [(1, 1, 1, 64, 32, 1, False), (3, 5, 1, 64, 16, 1, True), (2, 16, 8, 128, 64, 1, False), (7, 6, 2, 128, 64, 3, False), (5, 32, 4, 128, 32, 2, True),
         (130, 8, 4, 256, 128, 4, False), (2, 3, 3, 256, 4, 1, False), (1100, 4, 2, 64, 32, 3, True), (4, 4, 2, 128, 0, 1, False)]


@pytest.mark.parametrize("dtype", sorted(TYPES))
@pytest.mark.parametrize("norm", [True, False])
@pytest.mark.parametrize("rows,heads,kv_heads,dim,pairs,axes,neighbours", CASES)
def test_rotation(rows, heads, kv_heads, dim, pairs, axes, neighbours, norm, dtype):
    g = np.random.default_rng(rows + dim)
    x, freq, pos, axis = turned(g, rows, heads, kv_heads, dim, dtype, pairs, axes)
    w = [g.uniform(0.5, 2, dim).astype(np.float32) if norm else None for _ in "qk"]
    r = rotary.Rotary(dev(freq), axis=None if axis is None else dev(axis), neighbours=neighbours, factor=1.25)
    d = x.cuda()
    q, k = d[:, :heads], d[:, heads:heads + kv_heads]
    weights = [None if a is None else dev(a) for a in w]
    position = dev(pos) if axes > 1 else dev(pos[0])
    got = rotary.rotate(q, k, position, r, q_weight=weights[0], k_weight=weights[1], eps=1e-5)
    xn = x.double().numpy()
    for t, side, weight in zip(got, (xn[:, :heads], xn[:, heads:heads + kv_heads]), w):
        exact = ref.rope(side, pos, freq, axis, weight, 1e-5, neighbours, 1.25)
        # f32 throughout, in half steps of 2^-24: a norm's sum, mean, root and quotient 8 of them (a sum of 2^n squares: n + 3 additions with errors that
        # are shares of the sum, halved by the root), its two products 2, cosine and sine, the factor in them, two products and the sum 5: of the pair's size
        size = np.sqrt((exact ** 2).reshape(rows, -1, dim).max(-1, keepdims=True)) * np.sqrt(2)
        step = 0.0 if dtype == "f32" else torch.finfo(TYPES[dtype]).eps / 2
        off = np.abs(t.double().cpu().numpy() - exact) - step * np.abs(exact) - (2.0 ** -25 if dtype == "f16" else 0)
        assert (off <= 16 * 2.0 ** -24 * size).all(), off.max()
    # in place
    same = d.clone()
    rotary.rotate(same[:, :heads], same[:, heads:heads + kv_heads], position, r, q_weight=weights[0], k_weight=weights[1], eps=1e-5,
                  q_out=same[:, :heads], k_out=same[:, heads:heads + kv_heads])
    assert torch.equal(same[:, :heads], got[0]) and torch.equal(same[:, heads:heads + kv_heads], got[1])
    assert torch.equal(same[:, heads + kv_heads:], d[:, heads + kv_heads:])


def test_far_positions():
    """The angle of a position past 2^30 is made in 64 bits."""
    pos = np.array([0, 1, -1, (1 << 31) - 1, -(1 << 31), 1 << 24, (1 << 24) + 1], np.int32)
    freq = np.array([1.0, 0.1, 0.3, 1e-6], np.float32)
    x = np.zeros((len(pos), 1, 64), np.float32)
    x[:, :, :4] = 1
    r = rotary.Rotary(dev(freq))
    got = rotary.rotate(dev(x), dev(x), dev(pos), r)[0]
    assert np.abs(got.double().cpu().numpy() - ref.rope(x, pos, freq)).max() <= 2.0 ** -23


@pytest.mark.parametrize("dtype", sorted(TYPES))
@pytest.mark.parametrize("dim,neighbours", [(64, False), (128, True), (256, False)])
def test_what_is_not_rotated_passes_as_it_is(dim, neighbours, dtype):
    """Infinities, no numbers and zeros of either sign behind the rotated pairs: each leaves what is beside it alone."""
    g = np.random.default_rng(dim)
    x = rows_of(dtype, g, 3, 2, dim)
    past = x[:, :, dim // 2:]
    past[:, :, ::7], past[:, :, 1::11], past[:, :, 2::13], past[:, :, 3::17] = float("inf"), float("-inf"), float("nan"), -0.0
    r = rotary.Rotary(dev(np.linspace(0.1, 1, dim // 4).astype(np.float32)), neighbours=neighbours)
    d, pos = x.cuda(), dev(np.array([3, 0, 9], np.int32))
    for got in rotary.rotate(d, d, pos, r):
        bits = torch.int32 if dtype == "f32" else torch.int16
        number = ~past.isnan()
        assert torch.equal(got[:, :, dim // 2:].cpu().view(bits)[number], past.contiguous().view(bits)[number])
        assert got[:, :, dim // 2:].isnan().cpu().equal(~number)
    want = ref.Cache(2, 2, 16, dim, seed=1)
    cache, slots = handle(want), np.array([0, 17, 5])
    rotary.rotate_into(cache, d, d, d, pos, dev(slots), r)
    xn = x.double().numpy()
    keys = np.concatenate([ref.rope(xn[:, :, :dim // 2], pos.cpu().numpy()[None], np.linspace(0.1, 1, dim // 4).astype(np.float32), neighbours=neighbours), xn[:, :, dim // 2:]], -1)
    want.write(keys, xn, slots)
    check_cache(cache, want)


@pytest.mark.parametrize("dtype", sorted(TYPES))
@pytest.mark.parametrize("norm", [True, False])
@pytest.mark.parametrize("rows,heads,kv_heads,dim,pairs,axes,neighbours", CASES)
def test_rotation_into_the_cache(rows, heads, kv_heads, dim, pairs, axes, neighbours, norm, dtype):
    g = np.random.default_rng(rows + dim + 1)
    page = 16 if rows < 100 else 64
    x, freq, pos, axis = turned(g, rows, heads, kv_heads, dim, dtype, pairs, axes)
    w = [g.uniform(0.5, 2, dim).astype(np.float32) if norm else None for _ in "qk"]
    r = rotary.Rotary(dev(freq), axis=None if axis is None else dev(axis), neighbours=neighbours)
    weights = [None if a is None else dev(a) for a in w]
    pages = -(-rows // page) + 2
    want = ref.Cache(pages, kv_heads, page, dim, seed=rows)
    cache, slots = handle(want), g.permutation(pages * page)[:rows]
    if rows > 1:
        slots[rows // 2] = -1
    d = x.cuda()
    position = dev(pos) if axes > 1 else dev(pos[0])
    q, k, v = d[:, :heads], d[:, heads:heads + kv_heads], d[:, heads + kv_heads:]
    got = rotary.rotate_into(cache, q, k, v, position, dev(slots), r, q_weight=weights[0], k_weight=weights[1])
    plain = rotary.rotate(q, k, position, r, q_weight=weights[0], k_weight=weights[1])[0]
    # the queries are those of the call without a cache but for the last places of angles that were kept in 64 bits
    assert torch.allclose(got.double(), plain.double(), rtol=2 * torch.finfo(TYPES[dtype]).eps, atol=2.0 ** -20)
    xn = x.double().numpy()
    want.write(ref.rope(xn[:, heads:heads + kv_heads], pos, freq, axis, w[1], 1e-6, neighbours), xn[:, heads + kv_heads:], slots)
    check_cache(cache, want)


@pytest.mark.parametrize("dtype", sorted(TYPES))
@pytest.mark.parametrize("rows,heads,kv_heads,dim,pairs,axes,neighbours", [(2051, 3, 1, 64, 32, 1, False), (4097, 1, 1, 128, 32, 3, True), (2222, 2, 3, 256, 128, 2, False)])
def test_many_rows_into_the_cache(rows, heads, kv_heads, dim, pairs, axes, neighbours, dtype):
    test_rotation_into_the_cache(rows, heads, kv_heads, dim, pairs, axes, neighbours, True, dtype)


def test_recorded_rows_go_where_the_slots_say():
    """Replays with other rows, positions and slots, and eager work between them."""
    g = np.random.default_rng(8)
    rows, heads, kv_heads, dim = 6, 4, 2, 64
    x, pos = torch.empty((rows, heads + 2 * kv_heads, dim), device="cuda"), torch.zeros(rows, dtype=torch.int32, device="cuda")
    slots = torch.full((rows,), -1, dtype=torch.int64, device="cuda")
    freq = (10000.0 ** (-np.arange(32) / 32)).astype(np.float32)
    r, weight = rotary.Rotary(dev(freq)), dev(np.linspace(0.5, 1.5, dim).astype(np.float32))
    want, cache = ref.Cache(4, kv_heads, 16, dim), kv.KvCacheMxfp4.empty(4, kv_heads, dim)

    def call(into):
        q = rotary.rotate_into(into, x[:, :heads], x[:, heads:heads + kv_heads], x[:, heads + kv_heads:], pos, slots, r, q_weight=weight, k_weight=weight)
        return (q, *kv.kv_read(into, slots))

    x.zero_()
    graph, got = record(lambda: call(cache), torch.cuda.Stream())
    for n in range(4):
        rows_now = rows_of("f32", g, rows, heads + 2 * kv_heads, dim)
        at, to = g.integers(0, 5000, rows).astype(np.int32), g.permutation(64)[:rows]
        x.copy_(rows_now)
        pos.copy_(dev(at))
        slots.copy_(dev(to))
        graph.replay()
        torch.cuda.synchronize()
        xn = rows_now.double().numpy()
        want.write(ref.rope(xn[:, heads:heads + kv_heads], at, freq, None, weight.cpu().numpy()), xn[:, heads + kv_heads:], to)
        check_cache(cache, want)
        other = kv.KvCacheMxfp4.empty(4, kv_heads, dim)
        for a, b in zip(got, call(other)):
            assert torch.equal(a, b), n


def test_rows_behind_32_bit_offsets():
    """Codes past 2^31 bytes from their tensor's start, rows past 2^31 values from theirs."""
    pages, kv_heads, dim, page = (1 << 31) // (256 * 64) + 3, 2, 128, 128
    cache = kv.KvCacheMxfp4.empty(pages, kv_heads, dim, page)
    assert cache.k.numel() > 1 << 31
    stride = (1 << 31) // 2 + 64
    wide = torch.zeros((3, stride), dtype=torch.bfloat16, device="cuda")
    g = np.random.default_rng(2)
    x = rows_of("bf16", g, 3, 2 * kv_heads, dim)
    wide[:, :2 * kv_heads * dim] = x.reshape(3, -1).cuda()
    rows = wide[:, :2 * kv_heads * dim].unflatten(1, (2 * kv_heads, dim))
    slots = np.array([(pages - 1) * page + 127, 5, (pages - 2) * page], np.int64)
    kv.kv_write(cache, rows[:, :kv_heads], rows[:, kv_heads:], dev(slots))
    codes = ref.quantize(x.double().numpy())
    for got, part in zip(kv.kv_read(cache, dev(slots)), (slice(0, kv_heads), slice(kv_heads, None))):
        assert np.array_equal(got.cpu().numpy(), ref.values(codes[0][:, part], codes[1][:, part]).astype(np.float32))


@pytest.mark.parametrize("pairs", [0, 16])
def test_the_largest_numbers_of_f32_are_numbers(pairs):
    """They count for a block's power, as rows that are there already and as keys on their way from the norms."""
    most = np.finfo(np.float32).max
    x = np.zeros((3, 3, 64), np.float32)
    x[0, :, 40], x[1, :, 41], x[2, :, 63] = most, -most, np.nextafter(most, np.float32(0))
    x[:, :, 32] = 1e30
    r = rotary.Rotary(dev(np.ones(pairs, np.float32)))
    slots, d = np.array([3, 17, 30]), dev(x)
    want = ref.Cache(2, 1, 16, 64)
    want.write(x[:, 1:2], x[:, 2:], slots)
    for into in ("write", "rotate"):
        cache = kv.KvCacheMxfp4.empty(2, 1, 64)
        if into == "write":
            kv.kv_write(cache, d[:, 1:2], d[:, 2:], dev(slots))
        else:
            rotary.rotate_into(cache, d[:, :1], d[:, 1:2], d[:, 2:], dev(np.array([1, 2, 3], np.int32)), dev(slots), r)
        check_cache(cache, want)
