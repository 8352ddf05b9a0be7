"""What the cache, the attention and the sampling refuse, before anything touches a device: statuses of the C ABI on
addresses that are never read, and the host layer's checks of its tensors."""
import math

import pytest

torch = pytest.importorskip("torch")

from loken_amd import kv, lib, sampling

P = 4096   # an address; nothing behind it is touched


def plan_args(**change):
    a = dict(past=P, fresh=P, seqs=2, page=16, free=P, n_free=4, taken=None, table=P, stride=8, cols=8, lens=P, starts=P, slots=P, positions=P,
             rows=10, out=P, stream=None)
    a.update(change)
    return list(a.values())


@pytest.mark.parametrize("change,status", [
    (dict(seqs=-1), lib.LK_ERR_ARG), (dict(rows=-1), lib.LK_ERR_ARG), (dict(n_free=-1), lib.LK_ERR_ARG), (dict(page=8), lib.LK_ERR_ARG),
    (dict(page=48), lib.LK_ERR_ARG), (dict(page=512), lib.LK_ERR_ARG), (dict(page=0), lib.LK_ERR_ARG), (dict(stride=7), lib.LK_ERR_ARG),
    (dict(cols=-1), lib.LK_ERR_ARG), (dict(past=None), lib.LK_ERR_ARG), (dict(fresh=None), lib.LK_ERR_ARG), (dict(table=None), lib.LK_ERR_ARG),
    (dict(lens=None), lib.LK_ERR_ARG), (dict(starts=None), lib.LK_ERR_ARG), (dict(slots=None), lib.LK_ERR_ARG), (dict(slots=P + 4), lib.LK_ERR_ARG),
    (dict(positions=None), lib.LK_ERR_ARG), (dict(free=None), lib.LK_ERR_ARG), (dict(out=None), lib.LK_ERR_ARG), (dict(taken=P, out=P), lib.LK_ERR_ARG),
    (dict(seqs=8193), lib.LK_ERR_SIZE)])
def test_plan(change, status):
    assert lib.load().lk_kv_plan(*plan_args(**change)) == status


def write_args(**change):
    a = dict(k=P, v=P, type=0, ks=1024, vs=1024, slots=P, tokens=3, heads=8, dim=128, page=16, pages=4, kc=P, vc=P, ksc=P, vsc=P, stream=None)
    a.update(change)
    return list(a.values())


POOL = [(dict(dim=96), lib.LK_ERR_ARG), (dict(dim=512), lib.LK_ERR_ARG), (dict(page=24), lib.LK_ERR_ARG), (dict(pages=0), lib.LK_ERR_ARG),
        (dict(kc=None), lib.LK_ERR_ARG), (dict(vc=None), lib.LK_ERR_ARG), (dict(ksc=None), lib.LK_ERR_ARG), (dict(vsc=None), lib.LK_ERR_ARG),
        (dict(kc=P + 8), lib.LK_ERR_ARG), (dict(vc=P + 1), lib.LK_ERR_ARG), (dict(ksc=P + 2), lib.LK_ERR_ARG), (dict(type=2), lib.LK_ERR_TYPE),
        (dict(type=8), lib.LK_ERR_TYPE)]


@pytest.mark.parametrize("change,status", POOL + [
    (dict(heads=0), lib.LK_ERR_ARG), (dict(tokens=-1), lib.LK_ERR_ARG), (dict(ks=1023), lib.LK_ERR_ARG), (dict(vs=0), lib.LK_ERR_ARG), (dict(k=None), lib.LK_ERR_ARG),
    (dict(v=None), lib.LK_ERR_ARG), (dict(k=P + 2), lib.LK_ERR_ARG), (dict(type=30, v=P + 1), lib.LK_ERR_ARG), (dict(slots=None), lib.LK_ERR_ARG),
    (dict(slots=P + 4), lib.LK_ERR_ARG), (dict(tokens=0), lib.LK_OK)])
def test_write(change, status):
    assert lib.load().lk_kv_write_q8(*write_args(**change)) == status


def read_args(**change):
    a = dict(slots=P, tokens=3, heads=8, dim=128, page=16, pages=4, kc=P, vc=P, ksc=P, vsc=P, k=P, v=P, type=0, stream=None)
    a.update(change)
    return list(a.values())


@pytest.mark.parametrize("change,status", POOL + [
    (dict(slots=None), lib.LK_ERR_ARG), (dict(k=None), lib.LK_ERR_ARG), (dict(v=P + 2), lib.LK_ERR_ARG), (dict(tokens=-1), lib.LK_ERR_ARG),
    (dict(tokens=0), lib.LK_OK)])
def test_read(change, status):
    assert lib.load().lk_kv_read_q8(*read_args(**change)) == status


def attention_args(**change):
    a = dict(q=P, type=0, qs=4096, out=P, outs=4096, kc=P, vc=P, ksc=P, vsc=P, pages=4, page=16, table=P, stride=8, cols=8, lens=P, starts=P, seqs=2,
             rows=3, fresh=1, len=100, heads=32, kv=8, dim=128, scale=0.1, window=0, stream=None)
    a.update(change)
    return list(a.values())


@pytest.mark.parametrize("change,status", POOL + [
    (dict(heads=0), lib.LK_ERR_ARG), (dict(heads=12), lib.LK_ERR_ARG), (dict(kv=0), lib.LK_ERR_ARG), (dict(qs=4095), lib.LK_ERR_ARG),
    (dict(outs=128), lib.LK_ERR_ARG), (dict(scale=0.0), lib.LK_ERR_ARG), (dict(scale=-1.0), lib.LK_ERR_ARG), (dict(scale=math.nan), lib.LK_ERR_ARG),
    (dict(scale=math.inf), lib.LK_ERR_ARG), (dict(window=-1), lib.LK_ERR_ARG), (dict(fresh=-1), lib.LK_ERR_ARG), (dict(len=-1), lib.LK_ERR_ARG),
    (dict(rows=-1), lib.LK_ERR_ARG), (dict(seqs=-1), lib.LK_ERR_ARG), (dict(stride=4), lib.LK_ERR_ARG), (dict(q=None), lib.LK_ERR_ARG),
    (dict(out=P + 2), lib.LK_ERR_ARG), (dict(lens=None), lib.LK_ERR_ARG), (dict(starts=None), lib.LK_ERR_ARG), (dict(table=None), lib.LK_ERR_ARG),
    (dict(cols=1 << 27, stride=1 << 27), lib.LK_ERR_SIZE), (dict(rows=1 << 30), lib.LK_ERR_SIZE), (dict(rows=0), lib.LK_OK), (dict(seqs=0), lib.LK_OK)])
def test_attention(change, status):
    assert lib.load().lk_kv_attention_q8(*attention_args(**change)) == status


def sample_args(**change):
    a = dict(logits=P, type=0, stride=1000, rows=2, vocab=1000, uniform=P, temperature=P, k=None, p=None, m=None, tokens=P, probs=None, stream=None)
    a.update(change)
    return list(a.values())


@pytest.mark.parametrize("change,status", [
    (dict(type=8), lib.LK_ERR_TYPE), (dict(rows=-1), lib.LK_ERR_ARG), (dict(rows=65536), lib.LK_ERR_ARG), (dict(vocab=0), lib.LK_ERR_ARG), (dict(stride=999), lib.LK_ERR_ARG),
    (dict(vocab=(1 << 20) + 1, stride=1 << 21), lib.LK_ERR_SIZE), (dict(logits=None), lib.LK_ERR_ARG), (dict(logits=P + 2), lib.LK_ERR_ARG),
    (dict(uniform=None), lib.LK_ERR_ARG), (dict(temperature=None), lib.LK_ERR_ARG), (dict(tokens=None), lib.LK_ERR_ARG), (dict(rows=0), lib.LK_OK)])
def test_sample(change, status):
    assert lib.load().lk_sample(*sample_args(**change)) == status


def cpu_cache(page=16, dim=64):
    return kv.KvCacheQ8.empty(3, 2, dim, page, device="cpu")


def test_the_cache_checks_its_tensors():
    c = cpu_cache()
    with pytest.raises(ValueError):
        kv.KvCacheQ8.empty(3, 2, 80, 16, device="cpu")
    with pytest.raises(ValueError):
        kv.KvCacheQ8.empty(3, 2, 64, 20, device="cpu")
    with pytest.raises(ValueError):
        kv.KvCacheQ8(c.k, c.k, c.k_scales, c.v_scales)
    with pytest.raises(ValueError):
        kv.KvCacheQ8(c.k, c.v, c.k_scales, c.v_scales.double())
    with pytest.raises(ValueError):
        kv.KvCacheQ8(c.k.transpose(0, 1).contiguous().transpose(0, 1), c.v, c.k_scales, c.v_scales)
    with pytest.raises(ValueError):
        kv.KvCacheQ8(torch.zeros(3 * 2 * 16 * 64 + 8, dtype=torch.int8)[8:].view(3, 2, 16, 64), c.v, c.k_scales, c.v_scales)


def test_tensors_of_another_place_or_shape_are_refused():
    c = cpu_cache()
    rows, slots = torch.zeros(4, 2, 64), torch.zeros(4, dtype=torch.int64)
    for call in (lambda: kv.kv_write(c, rows, rows, slots),                            # not on a device
                 lambda: kv.kv_write(c, rows, rows.half(), slots),
                 lambda: kv.kv_write(c, rows[:, :1], rows[:, :1], slots),
                 lambda: kv.kv_write(c, rows, rows, slots.int()),
                 lambda: kv.kv_write(c, rows, rows, slots[:3]),
                 lambda: kv.kv_write(c, rows.transpose(0, 1), rows.transpose(0, 1), slots[:2]),
                 lambda: kv.kv_read(c, slots),
                 lambda: kv.kv_read(c, slots, dtype=torch.float64)):
        with pytest.raises(ValueError):
            call()
    i32 = lambda *v: torch.tensor(v, dtype=torch.int32)  # noqa: E731
    table, q = torch.zeros(1, 4, dtype=torch.int32), torch.zeros(2, 4, 64)
    good = dict(max_fresh=2, max_len=9)
    for args, more in (((q, c, table, i32(9), i32(0, 2)), good), ((q[:, :3], c, table, i32(9), i32(0, 2)), good), ((q, c, table, i32(9), i32(0)), good),
                       ((q, c, table.long(), i32(9), i32(0, 2)), good), ((q, c, table, i32(9), i32(0, 2)), dict(good, scale=-1.0)),
                       ((q, c, table, i32(9), i32(0, 2)), dict(good, out=q.half())), ((q, c, table, i32(9), i32(0, 2)), dict(good, window=-1)),
                       ((q, c, table[:0], i32(9), i32(0, 2)), good)):
        with pytest.raises(ValueError):
            kv.kv_attention(*args, **more)
    plan = kv.KvPlan(1, 8, device="cpu")
    for args, more in (((i32(1), i32(1), table, i32(1), 16, plan), {}), ((i32(1, 2), i32(1), table, i32(1), 16, plan), {}),
                       ((i32(1), i32(1), table, i32(1), 20, plan), {}), ((i32(1), i32(1), table, i32(1), 16, kv.KvPlan(2, 8, device="cpu")), {}),
                       ((i32(1), i32(1), table, i32(1), 16, plan), dict(taken=plan.taken)), ((i32(1).long(), i32(1), table, i32(1), 16, plan), {})):
        with pytest.raises(ValueError):
            kv.kv_plan(*args, **more)
    logits, u = torch.zeros(2, 10), torch.zeros(2)
    for args in ((logits, u, u), (logits.double(), u, u), (logits, u[:1], u), (logits, u, u, u), (logits[:, ::2], u, u), (logits[:1].expand(2, 10), u, u)):
        with pytest.raises(ValueError):
            sampling.sample(*args)


# arrays of a plan of 100 sequences and 700 rows, far from each other
APART = dict(past=1 << 20, fresh=2 << 20, seqs=100, page=16, free=3 << 20, n_free=50, taken=4 << 20, table=5 << 20, stride=12, cols=8, lens=6 << 20,
             starts=7 << 20, slots=8 << 20, positions=9 << 20, rows=700, out=10 << 20)
# bytes of each: the table's last row ends with its columns
SIZES = dict(past=400, fresh=400, free=200, taken=4, table=4 * (99 * 12 + 8), lens=400, starts=404, slots=5600, positions=2800, out=4)


@pytest.mark.parametrize("written", ["table", "lens", "starts", "slots", "positions", "out"])
@pytest.mark.parametrize("other", sorted(SIZES))
def test_a_plan_does_not_write_what_it_reads(written, other):
    """The first and the last byte's word in common are enough; slots stand on eight bytes."""
    if other == written:
        return
    word = 8 if written == "slots" else 4
    for at in (APART[other], APART[other] + (SIZES[other] - 4) // word * word, APART[other] - SIZES[written] + word):
        assert lib.load().lk_kv_plan(*plan_args(**{**APART, written: at})) == lib.LK_ERR_ARG, at


def test_lengths_of_the_plan_itself_are_refused():
    i32 = lambda *v: torch.tensor(v, dtype=torch.int32)  # noqa: E731
    plan = kv.KvPlan(2, 8, device="cpu")
    with pytest.raises(ValueError, match="plan's own"):
        kv.kv_plan(plan.lens, i32(1, 1), torch.zeros(2, 4, dtype=torch.int32), i32(1), 16, plan)


@pytest.mark.parametrize("name", ["k", "v", "k_scales", "v_scales"])
def test_the_tensors_of_a_cache_are_not_assigned_anew(name):
    """Without checks of the new ones, and with calls that go on with the old ones' memory."""
    c = cpu_cache()
    with pytest.raises(AttributeError):
        setattr(c, name, getattr(c, name).clone())
