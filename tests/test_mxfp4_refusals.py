"""What the 4-bit cache, the rotation, attention over the cache and the check of drafted tokens refuse, before anything touches a device:
statuses of the C ABI on addresses that are never read, and the host layer's checks of its tensors."""
import math

import pytest

torch = pytest.importorskip("torch")

from loken_amd import kv, lib, rotary, sampling

P = 4096   # an address; nothing behind it is touched
ARG, TYPE, SIZE, OK = lib.LK_ERR_ARG, lib.LK_ERR_TYPE, lib.LK_ERR_SIZE, lib.LK_OK


def call(name, base, change):
    a = dict(base)
    a.update(change)
    return getattr(lib.load(), name)(*a.values())


POOL = [(dict(dim=96), ARG), (dict(dim=512), ARG), (dict(page=24), ARG), (dict(page=8), ARG), (dict(page=512), ARG), (dict(pages=0), ARG), (dict(kc=None), ARG),
        (dict(vc=None), ARG), (dict(kp=None), ARG), (dict(vp=None), ARG), (dict(kc=P + 8), ARG), (dict(vc=P + 1), ARG), (dict(kp=P + 4), ARG), (dict(vp=P + 2), ARG),
        (dict(type=2), TYPE), (dict(type=39), TYPE)]
WRITE = dict(k=P, v=P, type=0, ks=1024, vs=1024, slots=P, tokens=3, heads=8, dim=128, page=16, pages=4, kc=P, vc=P, kp=P, vp=P, stream=None)


@pytest.mark.parametrize("change,status", POOL + [
    (dict(heads=0), ARG), (dict(tokens=-1), ARG), (dict(ks=1023), ARG), (dict(vs=0), ARG), (dict(k=None), ARG), (dict(v=None), ARG), (dict(k=P + 2), ARG),
    (dict(type=30, v=P + 1), ARG), (dict(slots=None), ARG), (dict(slots=P + 4), ARG), (dict(tokens=0), OK)])
def test_write(change, status):
    assert call("lk_kv_write_mxfp4", WRITE, change) == status


READ = dict(slots=P, tokens=3, heads=8, dim=128, page=16, pages=4, kc=P, vc=P, kp=P, vp=P, k=P, v=P, type=0, stream=None)


@pytest.mark.parametrize("change,status", POOL + [(dict(slots=None), ARG), (dict(k=None), ARG), (dict(v=P + 2), ARG), (dict(tokens=-1), ARG), (dict(tokens=0), OK)])
def test_read(change, status):
    assert call("lk_kv_read_mxfp4", READ, change) == status


TURN = dict(q=P, k=P, type=0, qs=4096, ks=1024, qo=P, ko=P, qos=4096, kos=1024, rows=3, heads=32, kv=8, dim=128, qw=None, kw=None, eps=1e-6, pos=P, across=3,
            axes=1, freq=P, axis=None, pairs=64, neighbours=0, factor=1.0, stream=None)
TURNS = [(dict(type=2), TYPE), (dict(dim=96), ARG), (dict(rows=-1), ARG), (dict(heads=0), ARG), (dict(kv=0), ARG), (dict(heads=65536), ARG), (dict(pairs=68), ARG),
         (dict(pairs=62), ARG), (dict(pairs=-4), ARG), (dict(axes=0), ARG), (dict(axes=5), ARG), (dict(across=2), ARG), (dict(eps=-1.0), ARG),
         (dict(eps=math.nan), ARG), (dict(eps=math.inf), ARG), (dict(factor=math.nan), ARG), (dict(factor=math.inf), ARG), (dict(q=None), ARG), (dict(k=None), ARG),
         (dict(qo=None), ARG), (dict(pos=None), ARG), (dict(freq=None), ARG), (dict(qs=4095), ARG), (dict(ks=1000), ARG), (dict(qos=0), ARG), (dict(q=P + 2), ARG),
         (dict(type=1, k=P + 1), ARG), (dict(qo=P + 1), ARG), (dict(rows=0, across=0), OK)]


@pytest.mark.parametrize("change,status", TURNS + [(dict(ko=None), ARG), (dict(kos=1023), ARG), (dict(ko=P + 2), ARG)])
def test_rotation(change, status):
    assert call("lk_qk_norm_rope", TURN, change) == status


FILL = dict(q=P, k=P, v=P, type=0, qs=4096, ks=1024, vs=1024, qo=P, qos=4096, slots=P, rows=3, heads=32, kv=8, dim=128, qw=None, kw=None, eps=1e-6, pos=P,
            across=3, axes=1, freq=P, axis=None, pairs=64, neighbours=0, factor=1.0, page=16, pages=4, kc=P, vc=P, kp=P, vp=P, stream=None)


@pytest.mark.parametrize("change,status", TURNS + POOL + [(dict(v=None), ARG), (dict(vs=1023), ARG), (dict(v=P + 2), ARG), (dict(slots=None), ARG), (dict(slots=P + 4), ARG)])
def test_rotation_into_the_cache(change, status):
    assert call("lk_qk_norm_rope_kv_mxfp4", FILL, change) == status


ATTEND = dict(q=P, type=0, qs=4096, out=P, outs=4096, kc=P, vc=P, kp=P, vp=P, pages=4, page=16, table=P, stride=8, cols=8, lens=P, starts=P, seqs=2, rows=3,
              fresh=1, len=100, heads=32, kv=8, dim=128, scale=0.1, window=0, cap=0.0, stream=None)


@pytest.mark.parametrize("change,status", POOL + [
    (dict(heads=0), ARG), (dict(heads=12), ARG), (dict(kv=0), ARG), (dict(qs=4095), ARG), (dict(outs=128), ARG), (dict(scale=0.0), ARG), (dict(scale=-1.0), ARG),
    (dict(scale=math.nan), ARG), (dict(scale=math.inf), ARG), (dict(cap=-1.0), ARG), (dict(cap=math.nan), ARG), (dict(cap=math.inf), ARG), (dict(window=-1), ARG),
    (dict(fresh=-1), ARG), (dict(len=-1), ARG), (dict(rows=-1), ARG), (dict(seqs=-1), ARG), (dict(stride=4), ARG), (dict(q=None), ARG), (dict(out=P + 2), ARG),
    (dict(lens=None), ARG), (dict(starts=None), ARG), (dict(table=None), ARG), (dict(cols=1 << 27, stride=1 << 27), SIZE), (dict(rows=1 << 30), SIZE),
    (dict(rows=0), OK), (dict(seqs=0), OK)])
def test_attention(change, status):
    assert call("lk_kv_attention_mxfp4", ATTEND, change) == status


@pytest.mark.parametrize("cap", [2.0 ** -65, 2.0 ** 65, 1e-40, 3e38])
def test_caps_that_leave_no_scores(cap):
    assert call("lk_kv_attention_mxfp4", ATTEND, dict(cap=cap)) == ARG
    with pytest.raises(ValueError, match="softcap"):
        kv.kv_attention(torch.zeros((2, 6, 64)), cache(), torch.zeros((1, 4), dtype=torch.int32), torch.tensor([5], dtype=torch.int32), torch.tensor([0, 2], dtype=torch.int32),
                        max_fresh=2, max_len=5, softcap=cap)


JUDGE = dict(logits=P, type=0, stride=1000, rows=5, vocab=1000, drafted=P, starts=P, seqs=2, draft=P, draft_type=0, draft_stride=1000, uniform=P, draw=P,
             temperature=P, top_k=None, top_p=None, min_p=None, tokens=P, accepted=P, probs=P, stream=None)


@pytest.mark.parametrize("change,status", [
    (dict(type=2), TYPE), (dict(draft_type=2), TYPE), (dict(rows=-1), ARG), (dict(rows=65536), ARG), (dict(seqs=-1), ARG), (dict(seqs=65536), ARG), (dict(vocab=0), ARG),
    (dict(stride=999), ARG), (dict(draft_stride=999), ARG), (dict(vocab=(1 << 20) + 1, stride=1 << 21, draft_stride=1 << 21), SIZE), (dict(logits=None), ARG),
    (dict(drafted=None), ARG), (dict(starts=None), ARG), (dict(uniform=None), ARG), (dict(draw=None), ARG), (dict(temperature=None), ARG), (dict(tokens=None), ARG),
    (dict(accepted=None), ARG), (dict(logits=P + 2), ARG), (dict(draft=P + 2), ARG), (dict(rows=0), OK), (dict(seqs=0), OK)])
def test_verification(change, status):
    assert call("lk_verify", JUDGE, change) == status


# ------------------------------------------------------------------------------------------ the host layer
def cache(**change):
    a = dict(k=torch.zeros((2, 3, 16, 32), dtype=torch.uint8), v=torch.zeros((2, 3, 4, 16, 4, 2), dtype=torch.uint8),
             k_powers=torch.zeros((2, 3, 16, 2), dtype=torch.uint8), v_powers=torch.zeros((2, 3, 2, 16), dtype=torch.uint8))
    a.update(change)
    return kv.KvCacheMxfp4(**a)


def test_caches():
    c = cache()
    assert (c.pages, c.kv_heads, c.page_tokens, c.head_dim) == (2, 3, 16, 64)
    for bad in (dict(k=torch.zeros((2, 3, 16, 32), dtype=torch.int8)), dict(k=torch.zeros((2, 3, 8, 32), dtype=torch.uint8)),
                dict(k=torch.zeros((2, 3, 16, 48), dtype=torch.uint8)), dict(v=torch.zeros((2, 3, 16, 32), dtype=torch.uint8)),
                dict(k_powers=torch.zeros((2, 3, 2, 16), dtype=torch.uint8)), dict(v_powers=torch.zeros((2, 3, 16, 2), dtype=torch.uint8)),
                dict(k=torch.zeros((2, 3, 16, 64), dtype=torch.uint8)[..., ::2]), dict(k=torch.zeros(2 * 3 * 16 * 32 + 1, dtype=torch.uint8)[1:].view(2, 3, 16, 32))):
        with pytest.raises(ValueError):
            cache(**bad)
    for bad in ((2, 3, 96, 16), (2, 3, 64, 24)):
        with pytest.raises(ValueError):
            kv.KvCacheMxfp4.empty(*bad, device="cpu")
    with pytest.raises(AttributeError):
        c.k = torch.zeros(1)


def test_rotaries():
    f = torch.ones(32)
    rotary.Rotary(f, axis=torch.zeros(32, dtype=torch.uint8))
    for bad in (dict(frequencies=f.double()), dict(frequencies=torch.ones(30)), dict(frequencies=torch.ones(132)), dict(frequencies=f[::2]),
                dict(frequencies=f, axis=torch.zeros(31, dtype=torch.uint8)), dict(frequencies=f, axis=torch.zeros(32, dtype=torch.int32)),
                dict(frequencies=f, factor=math.inf)):
        with pytest.raises(ValueError):
            rotary.Rotary(**bad)


def test_rotation_arguments():
    r = rotary.Rotary(torch.ones(32))
    good = dict(q=torch.zeros((4, 6, 64)), k=torch.zeros((4, 3, 64)), positions=torch.zeros(4, dtype=torch.int32), rotary=r)
    for bad in (dict(q=torch.zeros((4, 6, 60))), dict(q=torch.zeros((4, 384))), dict(k=torch.zeros((5, 3, 64))), dict(k=torch.zeros((4, 3, 64), dtype=torch.float16)),
                dict(k=torch.zeros((4, 3, 128))), dict(q=torch.zeros((4, 6, 64), dtype=torch.float64)), dict(q=torch.zeros((4, 6, 128))[..., ::2]),
                dict(positions=torch.zeros(4, dtype=torch.int64)), dict(positions=torch.zeros(3, dtype=torch.int32)), dict(positions=torch.zeros((5, 4), dtype=torch.int32)),
                dict(positions=torch.zeros((4, 2), dtype=torch.int32).T[:, ::1]), dict(q_weight=torch.ones(32)), dict(k_weight=torch.ones(64, dtype=torch.float16)),
                dict(eps=-1.0), dict(rotary=rotary.Rotary(torch.ones(64))), dict(q_out=torch.zeros((4, 6, 64), dtype=torch.float16)), dict(k_out=torch.zeros((4, 2, 64))),
                {}):
        with pytest.raises(ValueError):     # (the last: not on a device)
            rotary.rotate(**{**good, **bad})
    into = dict(good, cache=cache(), v=torch.zeros((4, 3, 64)), slots=torch.zeros(4, dtype=torch.int64))
    for bad in (dict(cache=kv.KvCacheQ8.empty(2, 3, 64, device="cpu")), dict(v=torch.zeros((3, 3, 64))), dict(v=torch.zeros((4, 3, 64), dtype=torch.float16)),
                dict(slots=torch.zeros(4, dtype=torch.int32)), dict(slots=torch.zeros(5, dtype=torch.int64)), dict(k=torch.zeros((4, 2, 64))), {}):
        with pytest.raises(ValueError):
            rotary.rotate_into(**{**into, **bad})


def test_attention_arguments():
    i32 = lambda *v: torch.tensor(v, dtype=torch.int32)  # noqa: E731
    good = dict(q=torch.zeros((2, 6, 64)), cache=cache(), table=torch.zeros((1, 4), dtype=torch.int32), lens=i32(5), starts=i32(0, 2), max_fresh=2, max_len=5)
    for bad in (dict(softcap=-1.0), dict(softcap=math.nan), dict(softcap=math.inf), dict(cache=kv.KvCacheQ8.empty(2, 3, 64, device="cpu"), softcap=30.0),
                dict(q=torch.zeros((2, 5, 64))), dict(q=torch.zeros((2, 6, 128))), {}):
        with pytest.raises(ValueError):
            kv.kv_attention(**{**good, **bad})


def test_verification_arguments():
    i32, n = (lambda *v: torch.tensor(v, dtype=torch.int32)), torch.zeros(3)
    good = dict(logits=torch.zeros((3, 50)), drafted=i32(1, 2, 3), starts=i32(0, 3), uniform=n, draw=torch.zeros(1), temperature=torch.ones(3))
    for bad in (dict(logits=torch.zeros((3, 50), dtype=torch.float64)), dict(logits=torch.zeros(150)), dict(logits=torch.zeros((3, 100))[:, ::2]),
                dict(drafted=i32(1, 2)), dict(drafted=torch.zeros(3, dtype=torch.int64)), dict(starts=torch.zeros(0, dtype=torch.int32)),
                dict(starts=torch.zeros(2, dtype=torch.int64)), dict(uniform=torch.zeros(2)), dict(draw=torch.zeros(2)), dict(temperature=torch.ones(3).double()),
                dict(top_k=torch.ones(3)), dict(top_p=torch.ones(2)), dict(min_p=torch.ones(3).half()), dict(draft=torch.zeros((3, 49))),
                dict(draft=torch.zeros((3, 50), dtype=torch.int32)), dict(draft=torch.zeros((50, 3)).T), {}):
        with pytest.raises(ValueError):
            sampling.verify(**{**good, **bad})


def test_rotation_by_several_axes_needs_to_know_which():
    """Positions of several axes and a rotation that does not say which of them turns a pair: all would go by the first."""
    several = torch.zeros((3, 4), dtype=torch.int32)
    good = dict(q=torch.zeros((4, 6, 64)), k=torch.zeros((4, 3, 64)), positions=several, rotary=rotary.Rotary(torch.ones(32)))
    into = dict(good, cache=cache(), v=torch.zeros((4, 3, 64)), slots=torch.zeros(4, dtype=torch.int64))
    for call_of, given in ((rotary.rotate, good), (rotary.rotate_into, into)):
        with pytest.raises(ValueError, match="axis"):
            call_of(**given)
        with pytest.raises(ValueError, match="device"):     # one axis, or a rotation that says
            call_of(**dict(given, positions=several[:1]))
        with pytest.raises(ValueError, match="device"):
            call_of(**dict(given, rotary=rotary.Rotary(torch.ones(32), axis=torch.zeros(32, dtype=torch.uint8))))


@pytest.mark.parametrize("change", [dict(scale=3e38), dict(scale=1e-40), dict(scale=2.0 ** 127 * 1.01), dict(scale=2.0 ** 70, cap=2.0 ** -64),
                                    dict(scale=2.0 ** -70, cap=2.0 ** 64), dict(scale=1e-37, cap=1e3)])
def test_scales_past_what_a_factor_of_f32_holds(change):
    """A score's factor, scale * log2 e or scale / cap, has to be a normal number: an infinite one leaves no number of a product of 0."""
    assert call("lk_kv_attention_mxfp4", ATTEND, change) == ARG
    with pytest.raises(ValueError, match="scale"):
        kv.kv_attention(torch.zeros((2, 6, 64)), cache(), torch.zeros((1, 4), dtype=torch.int32), torch.tensor([5], dtype=torch.int32),
                        torch.tensor([0, 2], dtype=torch.int32), max_fresh=2, max_len=5, scale=change["scale"], softcap=change.get("cap", 0.0))


@pytest.mark.parametrize("change", [dict(scale=2.0 ** 127), dict(scale=2.0 ** -126), dict(scale=2.0 ** 60, cap=2.0 ** -64), dict(scale=2.0 ** -60, cap=2.0 ** 64)])
def test_scales_at_both_ends(change):
    assert call("lk_kv_attention_mxfp4", ATTEND, dict(change, rows=0)) == OK
