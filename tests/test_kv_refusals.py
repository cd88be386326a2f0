"""What the paged cache, its attention and the token log probabilities refuse, checked before anything is launched (no GPU needed)."""
import ctypes as C

import pytest
import torch

from candle_b200 import capi
from candle_b200.kv_cache import PagedKvCache
from candle_b200.logprobs import token_logprobs

FAKE = 1 << 12      # an aligned address that is never read


def _cache(**over):
    f = dict(k=FAKE, v=FAKE, state=FAKE, layers=2, pages=8, kv_heads=2, page_size=16, head_dim=64, max_seqs=4, max_pages=4, elem=capi.F32)
    f.update(over)
    return capi.KvCache(**f)


def _refused(lib, status, text, fn, *args):
    lib.cq_clear_status()
    fn(*args)
    try:
        assert lib.cq_last_status() == status, lib.cq_last_message()
        assert text in lib.cq_last_message().decode()
    finally:
        lib.cq_clear_status()


@pytest.mark.parametrize("status,text,over", [
    (1, "null pointer", dict(k=0)), (1, "null pointer", dict(state=0)), (1, "positive", dict(pages=0)), (1, "positive", dict(layers=-1)),
    (1, "element type", dict(elem=3)), (1, "aligned", dict(v=FAKE + 8)), (2, "page_size", dict(page_size=24)), (2, "head_dim", dict(head_dim=96)),
    (2, "slots", dict(max_seqs=65537)), (2, "rows in a layer", dict(pages=1 << 28)),
])
def test_cache_descriptions(lib, status, text, over):
    c = _cache(**over)
    for fn, args in ((lib.cq_kv_reset, (None,)), (lib.cq_kv_reserve, (FAKE, 1, 1, None)), (lib.cq_kv_fork, (FAKE, FAKE, 1, 0, None)),
                     (lib.cq_kv_free, (FAKE, 1, None)), (lib.cq_kv_compact, (None,))):
        _refused(lib, status, text, fn, C.byref(c), *args)
    assert lib.cq_kv_take_fault(C.byref(c), None) == -1
    lib.cq_clear_status()


def test_lists_and_counts(lib):
    c = C.byref(_cache())
    _refused(lib, 1, "null list", lib.cq_kv_reserve, c, None, 1, 1, None)
    _refused(lib, 1, "more slots", lib.cq_kv_free, c, FAKE, 5, None)
    _refused(lib, 1, "null list", lib.cq_kv_fork, c, FAKE, None, 1, 0, None)
    _refused(lib, 1, "negative", lib.cq_kv_reserve, c, FAKE, 1, -1, None)
    assert lib.cq_kv_state_ints(0, 1, 1) == 0 and lib.cq_kv_state_ints(8, 4, 4) > 8 + 4 + 16


def test_append_arguments(lib):
    c = C.byref(_cache())

    def call(layer=0, q=FAKE, k=FAKE, v=FAKE, elem=capi.F32, hq=4, qs=256, ks=128, vs=128, cos=FAKE, sin=FAKE, max_pos=64, out=FAKE * 2, t=1):
        lib.cq_kv_append(c, layer, FAKE, 1, t, q, k, v, elem, hq, qs, ks, vs, cos, sin, max_pos, 0, out, None)

    for text, kw in (("layer", dict(layer=2)), ("null", dict(k=None)), ("null", dict(out=None)), ("null", dict(sin=None)), ("null", dict(t=0)),
                     ("element type", dict(elem=5)), ("aligned", dict(qs=258)), ("aligned", dict(ks=64)), ("aligned", dict(v=FAKE + 4)),
                     ("same type", dict(out=FAKE, elem=capi.F16))):
        _refused(lib, 1, text, lambda: call(**kw))


@pytest.mark.parametrize("status,text,over", [
    (1, "positive", dict(batch=0)), (1, "multiple", dict(heads=3)), (1, "group", dict(groups=5)), (1, "group", dict(groups=0)),
    (2, "4096", dict(batch=2000, queries=3)), (2, "32 query heads", dict(heads=66)),
])
def test_plan_shapes(lib, status, text, over):
    f = dict(batch=4, queries=1, heads=4, groups=1)
    f.update(over)
    _refused(lib, status, text, lib.cq_prefix_plan_shape, C.byref(_cache()), C.byref(capi.PrefixPlan(**f)), None, None)


def test_plan_groups_and_memory(lib):
    cache, plan = C.byref(_cache()), capi.PrefixPlan(batch=4, queries=1, heads=4, groups=2)
    sizes = (C.c_int * 2)(1, 2)
    _refused(lib, 1, "add up", lib.cq_prefix_plan_shape, cache, C.byref(plan), C.addressof(sizes), None)
    sizes[1] = 3
    shapes = (C.c_int * 8)()
    assert lib.cq_prefix_plan_shape(cache, C.byref(plan), C.addressof(sizes), C.addressof(shapes)) == 0
    assert list(shapes) == [0, 2, 0, 1, 1, 6, 2, 1] and plan.n_ints > 0 and plan.n_floats > 0
    _refused(lib, 1, "memory is missing", lib.cq_prefix_plan_update, cache, C.byref(plan), FAKE, None)
    plan.ints = plan.scratch = FAKE
    _refused(lib, 1, "null slots", lib.cq_prefix_plan_update, cache, C.byref(plan), None, None)
    for q, stride, scale in ((None, 256, 1.0), (FAKE, 255, 1.0), (FAKE, 258, 1.0), (FAKE, 256, 0.0), (FAKE, 256, float("nan")), (FAKE, 256, float("inf"))):
        _refused(lib, 1, "prefix_attention", lib.cq_prefix_attention, cache, 0, C.byref(plan), q, stride, FAKE, scale, None)
    _refused(lib, 1, "prefix_attention", lib.cq_prefix_attention, cache, 2, C.byref(plan), FAKE, 256, FAKE, 1.0, None)
    plan.n_floats += 1
    _refused(lib, 1, "not one", lib.cq_prefix_attention, cache, 0, C.byref(plan), FAKE, 256, FAKE, 1.0, None)


def test_logprobs_arguments(lib):
    size = lib.cq_token_logprobs_scratch_bytes
    assert size(1, 10, 11) == 0 and size(1, 100, 33) == 0 and size(0, 10, 1) == 0 and size(1, 10, 10) > 0

    def call(logits=FAKE, elem=capi.F32, rows=1, vocab=100, tokens=FAKE, top=2, logprob=FAKE, best=FAKE, scratch=FAKE, stride=100):
        lib.cq_token_logprobs(logits, elem, stride, rows, vocab, tokens, top, logprob, FAKE, best, FAKE, scratch, None)

    for text, kw in (("null", dict(logits=None)), ("null", dict(tokens=None)), ("null", dict(best=None)), ("misaligned", dict(logits=FAKE + 2)),
                     ("element type", dict(elem=7)), ("misaligned", dict(scratch=FAKE + 8)), ("top", dict(top=33)), ("positive", dict(rows=0)),
                     ("top", dict(vocab=1))):
        _refused(lib, 1, text, lambda: call(**kw))


def test_python_refuses_the_cpu():
    with pytest.raises(capi.CandleQError, match="no CPU path"):
        PagedKvCache(1, 4, 16, 1, 64, 1, 16, device="cpu")
    with pytest.raises(capi.CandleQError, match="no CPU path"):
        token_logprobs(torch.zeros(2, 8))
