"""Calls of the paged cache that its documentation allows or refuses, at their borders."""
import pytest
import torch

from candle_b200 import capi
from candle_b200.kv_cache import PagedKvCache
from test_gpu_kv_cache import _make

pytestmark = pytest.mark.gpu


def _faulted(cache, text):
    with pytest.raises(capi.CandleQError, match=text):
        cache.check()


def test_slots_beyond_32_bits_are_out_of_range(cuda_dev):
    """Whole numbers of any type: none becomes another slot on its way to the device's int32."""
    cache = _make(8, 16, 1, 64, 4, 64, torch.float32)
    cache.reserve([0], 5)
    for dtype, values in ((torch.int64, (1 << 32, -(1 << 32), (1 << 32) + 2, 1 << 62, 4, -1)), (torch.uint32, ((1 << 32) - 4, 1 << 31)), (torch.int16, (-1, 300)),
                          (torch.uint8, (200,))):
        for v in values:
            for device in ("cpu", "cuda"):
                cache.free(torch.tensor([v], dtype=dtype, device=device))
                _faulted(cache, "out of range")
    assert cache.lens.tolist() == [5, 0, 0, 0]
    for dtype in (torch.int64, torch.int32, torch.uint32, torch.int16, torch.uint16, torch.int8, torch.uint8):
        cache.reserve(torch.tensor([3, 1], dtype=dtype, device="cuda"), 1)
    cache.check()
    assert cache.lens.tolist() == [5, 7, 0, 7]


def test_lists_of_other_than_whole_numbers_are_refused(cuda_dev):
    cache = _make(8, 16, 1, 64, 4, 64, torch.float32)
    for slots in ([0.7], [0.0], [0, "1"], [None]):
        with pytest.raises(capi.CandleQError, match="whole numbers"):
            cache.reserve(slots, 1)
    with pytest.raises(capi.CandleQError, match="whole numbers"):
        cache.attention_plan(2, 1, groups=[1.5, 1])
    assert cache.lens.tolist() == [0, 0, 0, 0]


KINDS = {"slot": "out of range", "twice": "named twice", "long": "position", "rotary": "position", "shared": "shared page", "table": "not there"}


@pytest.mark.parametrize("kind", list(KINDS))
@pytest.mark.parametrize("where", [0, 2])
@pytest.mark.parametrize("batch,t,page,hkv,hq", [(3, 1, 16, 1, 1), (3, 40, 16, 3, 5), (3, 3000, 64, 4, 4), (3, 3000, 16, 1, 2), (300, 1, 16, 2, 2), (600, 2, 16, 1, 1)])
def test_a_faulted_append_does_nothing(cuda_dev, kind, where, batch, t, page, hkv, hq):
    """One slot of many cannot be stored, the first or the last: nothing is stored, no query given, whoever finds it; a second call does nothing either; the state is as it was, and
    once the fault is taken the call without that slot does all.  From one check to one a thread, several a thread (144 and 300 of them), and more than a CTA makes itself (567, 1200)."""
    if kind == "rotary" and where == 0:
        pytest.skip("the tables end for the longest sequence")
    per = -(-(t + 40) // page)
    cache = _make((batch + 1) * per + 2, page, hkv, 64, batch + 2, per * page, torch.bfloat16)
    g = torch.Generator(device="cuda").manual_seed(batch + t)
    every = torch.arange(batch, dtype=torch.int32, device="cuda")
    bad = 0 if where == 0 else batch - 1
    cache.reserve(every, t)
    cache.reserve([bad], 20)                    # the longest
    slots, rotary = every.clone(), (torch.ones((t + 20, 32), device="cuda"), torch.zeros((t + 20, 32), device="cuda"))
    if kind == "slot":
        slots[bad] = batch + 2
    elif kind == "twice":
        slots[bad] = 1
    elif kind == "long":
        slots[bad] = batch + 1                  # an empty one
    elif kind == "rotary":
        rotary = tuple(x[:-1].contiguous() for x in rotary)
    elif kind == "shared":                      # in the middle of a prompt, else the page of the row
        cache.refs[cache.tables[bad, (int(cache.lens[bad]) - 1 - t // 2) // page].long()] += 1
    else:
        cache.tables[bad, (int(cache.lens[bad]) - 1 - t // 2) // page] = cache.pages
    q, k, v = (torch.randn((batch, t, h, 64), device="cuda", generator=g).to(torch.bfloat16) for h in (hq, hkv, hkv))
    was = cache.k.clone(), cache.v.clone(), cache.state[16:].clone()
    for _ in range(2):
        assert float(cache.append(0, slots, k, v, q=q, rotary=rotary).abs().max()) == 0.0
        good = every[:1] if bad else every[1:2]
        assert float(cache.append(0, good, k[:1], v[:1], q=q[:1]).abs().max()) == 0.0
        cache.reserve(good, 0 if t > 1 else 1)
        assert torch.equal(cache.k, was[0]) and torch.equal(cache.v, was[1]) and torch.equal(cache.state[16:], was[2])
        _faulted(cache, KINDS[kind])
    rest = torch.cat([every[:bad], every[bad + 1:]])
    pick = rest.long()
    assert torch.equal(cache.append(0, rest, k[pick], v[pick], q=q[pick], rotary=rotary), q[pick])
    cache.check()
    for i in rest.tolist()[:3] + rest.tolist()[-3:]:
        at = torch.arange(int(cache.lens[i]) - t, int(cache.lens[i]), device="cuda")
        ids = cache.tables[i].long()[at // page]
        assert torch.equal(cache.k[0][ids, :, at % page], k[i]) and torch.equal(cache.v[0][ids, :, at % page], v[i])


@pytest.mark.parametrize("dtype,pages", [(torch.bfloat16, 34000), (torch.float32, 17100)])
def test_pools_beyond_32_bits(cuda_dev, dtype, pages):
    """Pages whose elements, or bytes, are numbered beyond 2^32: stored, forked, moved and read there as in a small pool."""
    shape = (1, pages, 8, 128, 128)
    torch.cuda.empty_cache()
    big = PagedKvCache(1, pages, 128, 8, 128, 6, 1024, dtype=dtype, pools=tuple(torch.empty(shape, dtype=dtype, device="cuda") for _ in range(2)))
    small = PagedKvCache(1, 48, 128, 8, 128, 6, 1024, dtype=dtype)
    big.refs[:pages - 40] = 1                   # taken by others
    assert (pages - 40) * 8 * 128 * 128 * big.k.element_size() > 1 << 32
    g = torch.Generator(device="cuda").manual_seed(3)
    q, k, v = (torch.randn((1, 700, h, 128), device="cuda", generator=g).to(dtype) for h in (32, 8, 8))
    step_q = torch.randn((5, 1, 32, 128), device="cuda", generator=g).to(dtype)
    outs = []
    for c in (big, small):
        c.reserve([0], 700)
        c.append(0, [0], k, v)
        c.fork([0] * 4, [1, 2, 3, 4])
        c.reserve([0, 1, 2, 3, 4], 1)
        c.append(0, [0, 1, 2, 3, 4], k[0, :5, None], v[0, :5, None])
        plan = c.attention_plan(5, 32)
        plan.update([0, 1, 2, 3, 4])
        outs.append([c.attention(0, step_q, plan)])
        c.copy([2], [5])
        c.free([1, 2])
        if c is big:
            c.refs[:30] = 0                     # room at the front, the others' pages stay
        c.compact()
        plan.update([0, 3, 4, 5, 5])
        outs[-1].append(c.attention(0, step_q, plan))
        c.check()
    assert int(big.tables.max()) < pages - 40 + 30 and int(big.tables[0, 0]) < 30
    for a, b in zip(*outs):
        assert torch.equal(a, b) and bool(torch.isfinite(a).all())
