"""The paged KV cache on the GPU: page operations against a restatement in numpy, exactly; the store of keys and values and the shared-prefix attention against
64-bit formulas.

Tolerances.  u is half a step of a type relative to the value (f32 2^-24, f16 2^-11, bf16 2^-8).  A rotated value is a product and a fused product-sum in f32 and
one rounding to the type: within 2 * 2^-24 * (|x0| + |x1|) + u |y|.  Attention: a score is a sum of D products, its error at most (D + 4) 2^-24 sum |q k| scale,
the same for all that follows (exp2 2 ulp, sums of n weights): relative to the weights' own size e = 2 (D + 4) 2^-24 max(sum |q k|) scale + (n + 64) 2^-24; 16-bit types also
round each weight, by u, in the product and in its sum alike.  Weights w (1 + d), |d| <= e + u, move sum w v / sum w by at most (e + u) * 2 max |v|, and the
result is rounded once: 2 (e + u) max |v| / (1 - e - u) + u max |v|."""
import math

import numpy as np
import pytest
import torch

from candle_b200 import capi
from candle_b200.kv_cache import PagedKvCache

pytestmark = pytest.mark.gpu
U = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
TYPES = [torch.float32, torch.float16, torch.bfloat16]


class Mirror:
    """The bookkeeping of the header's description, in numpy, with a copy of the pools."""

    def __init__(self, cache):
        self.page, self.cap = cache.page_size, cache.max_len
        self.refs, self.lens, self.tables = np.zeros(cache.pages, int), np.zeros(cache.max_seqs, int), np.full(tuple(cache.tables.shape), -1)
        self.k, self.v = cache.k.clone(), cache.v.clone()

    def n(self, length):
        return -(-length // self.page)

    def take(self, count):
        free = np.flatnonzero(self.refs == 0)
        return list(free[:count]) if len(free) >= count else None

    def reserve(self, slots, tokens):
        need = [self.n(self.lens[s] + tokens) - self.n(self.lens[s]) for s in slots]
        if any(self.lens[s] + tokens > self.cap for s in slots):
            return False
        got = self.take(sum(need))
        if got is None:
            return False
        for s, c in zip(slots, need):
            have = self.n(self.lens[s])
            for j in range(c):
                p = got.pop(0)
                self.tables[s, have + j], self.refs[p] = p, 1
            self.lens[s] += tokens
        return True

    def fork(self, src, dst, deep=False):
        if any(self.lens[d] for d in dst) or set(src) & set(dst) or len(set(dst)) < len(dst):
            return False
        full = [0 if deep else self.lens[s] // self.page for s in src]
        got = self.take(sum(self.n(self.lens[s]) - f for s, f in zip(src, full)))
        if got is None:
            return False
        for s, d, f in zip(src, dst, full):
            for j in range(self.n(self.lens[s])):
                p = self.tables[s, j]
                if j < f:
                    self.tables[d, j] = p
                    self.refs[p] += 1
                else:
                    to, rows = got.pop(0), min(self.page, self.lens[s] - j * self.page)
                    self.tables[d, j], self.refs[to] = to, 1
                    for pool in (self.k, self.v):
                        pool[:, to, :, :rows] = pool[:, p, :, :rows]
            self.lens[d] = self.lens[s]
        return True

    def free(self, slots):
        for s in slots:
            for p in self.tables[s][self.tables[s] >= 0]:
                self.refs[p] -= 1
            self.tables[s], self.lens[s] = -1, 0

    def compact(self):
        live = int((self.refs > 0).sum())
        holes = [p for p in range(live) if self.refs[p] == 0]
        movers = [p for p in range(live, len(self.refs)) if self.refs[p] > 0]
        for a, b in zip(movers, holes):
            for pool in (self.k, self.v):
                pool[:, b] = pool[:, a]
            self.refs[b], self.refs[a] = self.refs[a], 0
            self.tables[self.tables == a] = b

    def same(self, cache):
        assert np.array_equal(cache.refs.cpu().numpy(), self.refs)
        assert np.array_equal(cache.lens.cpu().numpy(), self.lens)
        assert np.array_equal(cache.tables.cpu().numpy(), self.tables)
        assert torch.equal(cache.k, self.k) and torch.equal(cache.v, self.v)


def _make(pages, page, hkv, dim, seqs, max_len, dtype, layers=1, seed=0):
    c = PagedKvCache(layers, pages, page, hkv, dim, seqs, max_len, dtype=dtype)
    g = torch.Generator(device="cuda").manual_seed(seed)
    c.k.normal_(generator=g)
    c.v.normal_(generator=g)
    return c


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("page,dim,layers,hkv", [(16, 64, 3, 2), (32, 128, 1, 1), (64, 64, 2, 3), (128, 128, 2, 2)])
def test_page_operations_against_numpy(cuda_dev, dtype, page, dim, layers, hkv):
    rng = np.random.default_rng(page + dim)
    cache = _make(48, page, hkv, dim, 12, 6 * page, dtype, layers)
    m = Mirror(cache)
    done = 0
    for step in range(60):
        op = rng.choice(["reserve", "fork", "copy", "free", "compact"], p=[0.35, 0.25, 0.1, 0.2, 0.1])
        busy, empty = [s for s in range(12) if m.lens[s]], [s for s in range(12) if not m.lens[s]]
        if op == "reserve":
            slots = [int(s) for s in rng.permutation(12)[:rng.integers(1, 5)]]
            tokens = int(rng.integers(0, 2 * page + 2))
            ok = m.reserve(slots, tokens)
            cache.reserve(slots, tokens)
        elif op in ("fork", "copy"):
            if not busy or not empty:
                continue
            dst = [int(s) for s in rng.permutation(empty)[:rng.integers(1, 4)]]
            src = [int(rng.choice(busy)) for _ in dst]
            ok = m.fork(src, dst, op == "copy")
            (cache.fork if op == "fork" else cache.copy)(src, dst)
        elif op == "free":
            slots = [int(s) for s in rng.permutation(12)[:rng.integers(1, 3)]]      # empty ones among them
            ok = True
            m.free(slots)
            cache.free(slots)
        else:
            ok = True
            m.compact()
            cache.compact()
        if ok:
            cache.check()
            done += 1
        else:
            with pytest.raises(capi.CandleQError):
                cache.check()
        m.same(cache)
    assert done > 30


@pytest.mark.parametrize("pages", [5000, 4097])
def test_many_pages_and_slots(cuda_dev, pages):
    """More pages than one pass of the bookkeeping covers, more slots than it has threads."""
    cache = _make(pages, 16, 1, 64, 1500, 64, torch.float16)
    m = Mirror(cache)
    order = np.random.default_rng(1).permutation(1500)
    for slots, tokens in ((order.tolist(), 17), (order[:1100].tolist(), 16)):
        ok = m.reserve(slots, tokens)           # 3000 pages, then 1100: three more than the smaller pool has left
        cache.reserve(torch.tensor(slots, device="cuda"), tokens)
        assert ok == (tokens == 17 or pages == 5000)
        if not ok:
            _faulted(cache, "out of pages")
        m.same(cache)
    gone = order[100:1400].tolist()
    m.free(gone), cache.free(gone)
    m.compact(), cache.compact()
    m.same(cache)
    dst = sorted(gone)[:1200]
    src = [int(order[i % 100]) for i in range(1200)]
    assert m.fork(src, dst)
    cache.fork(src, dst)
    cache.check()
    m.same(cache)


def _faulted(cache, text):
    with pytest.raises(capi.CandleQError, match=text):
        cache.check()
    cache.check()


def test_faults_change_nothing(cuda_dev):
    cache = _make(6, 16, 2, 64, 4, 64, torch.float32)
    cache.reserve([0, 2], 20)
    m = Mirror(cache)
    assert m.reserve([0, 2], 20)
    t = lambda *s: torch.tensor(s, dtype=torch.int32, device="cuda")
    for text, call in (("out of range", lambda: cache.reserve(t(0, 4), 1)), ("out of range", lambda: cache.free(t(-1))),
                       ("named twice", lambda: cache.reserve(t(1, 1), 1)), ("named twice", lambda: cache.free(t(0, 2, 0))),
                       ("named twice", lambda: cache.fork(t(0, 0), t(1, 1))), ("source and destination", lambda: cache.fork(t(0, 1), t(1, 3))),
                       ("not empty", lambda: cache.fork(t(0), t(2))), ("out of pages", lambda: cache.reserve(t(1, 3), 32)),
                       ("out of pages", lambda: cache.copy(t(0, 2), t(1, 3))), ("longer than its table", lambda: cache.reserve(t(0), 45))):
        call()
        cache.reserve([1], 1)               # and so do the calls after it, until the fault is taken
        cache.free([0])
        cache.compact()
        _faulted(cache, text)
        m.same(cache)
    with pytest.raises(capi.CandleQError, match="slots are 0"):
        cache.free([4])
    with pytest.raises(capi.CandleQError, match="one destination"):
        cache.fork([0], [1, 3])
    with pytest.raises(capi.CandleQError, match="tokens"):
        cache.reserve([0], -1)


# ---- keys and values ----
def _rotate64(x, cos, sin, neox):
    x = x.double()
    half = x.shape[-1] // 2
    first = torch.arange(half, device=x.device) if neox else 2 * torch.arange(half, device=x.device)
    second = first + (half if neox else 1)
    y = torch.empty_like(x)
    y[..., first] = x[..., first] * cos - x[..., second] * sin
    y[..., second] = x[..., first] * sin + x[..., second] * cos
    size = torch.empty_like(x)
    size[..., first] = size[..., second] = x[..., first].abs() + x[..., second].abs()
    return y, size


@pytest.mark.parametrize("inp,dtype", [(a, b) for a in TYPES for b in TYPES])
@pytest.mark.parametrize("neox", [False, True])
@pytest.mark.parametrize("batch,t,hq,hkv,dim,page", [(1, 1, 1, 1, 64, 16), (5, 1, 6, 2, 128, 32), (3, 19, 4, 4, 64, 16), (1, 130, 3, 1, 128, 64)])
def test_append(cuda_dev, inp, dtype, neox, batch, t, hq, hkv, dim, page):
    g = torch.Generator(device="cuda").manual_seed(batch * 100 + t)
    cache = _make(64, page, hkv, dim, batch + 2, 300, dtype, layers=2, seed=3)
    slots = list(range(batch, 0, -1))
    for i, s in enumerate(slots):
        cache.reserve([s], 7 * i)
    cache.reserve(slots, t)
    before = cache.k.clone(), cache.v.clone()
    wide = torch.randn((batch * t, (hq + 2 * hkv) * dim + 8), device="cuda", generator=g).to(inp)      # q, k, v as columns of one product
    q = wide[:, :hq * dim].unflatten(1, (hq, dim)).unflatten(0, (batch, t))
    k = wide[:, hq * dim:(hq + hkv) * dim].unflatten(1, (hkv, dim)).unflatten(0, (batch, t))
    v = wide[:, (hq + hkv) * dim:(hq + 2 * hkv) * dim].unflatten(1, (hkv, dim)).unflatten(0, (batch, t))
    ang = torch.rand((300, dim // 2), device="cuda", generator=g) * 6.28
    cos, sin = ang.cos(), ang.sin()
    q_out = cache.append(1, slots, k, v, q=q, rotary=(cos, sin), neox=neox)
    cache.check()
    assert q_out.dtype == dtype and torch.equal(cache.k[0], before[0][0]) and torch.equal(cache.v[0], before[1][0])
    ref_k, ref_v = before[0][1].clone().double(), before[1][1].clone().double()
    written = torch.zeros(cache.k[1].shape, dtype=torch.bool, device="cuda")
    size_k = torch.zeros_like(ref_k)
    for b, s in enumerate(slots):
        pos = torch.arange(int(cache.lens[s]) - t, int(cache.lens[s]), device="cuda")
        ids = cache.tables[s].long()[pos // page]
        c, n = cos[pos].double()[:, None], sin[pos].double()[:, None]
        y, size = _rotate64(k[b], c, n, neox)
        ref_k[ids, :, pos % page], size_k[ids, :, pos % page] = y, size
        ref_v[ids, :, pos % page] = v[b].to(dtype).double()
        written[ids, :, pos % page] = True
        y, size = _rotate64(q[b], c, n, neox)
        assert bool(((q_out[b].double() - y).abs() <= 2 * 2.0 ** -24 * size + U[dtype] * y.abs() * (1 + 2.0 ** -20) + 2.0 ** -25).all())
    assert bool(((cache.k[1].double() - ref_k).abs() <= 2 * 2.0 ** -24 * size_k + U[dtype] * ref_k.abs() * (1 + 2.0 ** -20) + 2.0 ** -25)[written].all())
    assert torch.equal(cache.v[1].double(), ref_v) and torch.equal(cache.k[1][~written], before[0][1][~written])
    # without rotation, without q: the values themselves
    assert cache.append(0, slots, k, v) is None
    for b, s in enumerate(slots):
        pos = torch.arange(int(cache.lens[s]) - t, int(cache.lens[s]), device="cuda")
        ids = cache.tables[s].long()[pos // page]
        assert torch.equal(cache.k[0][ids, :, pos % page], k[b].to(dtype)) and torch.equal(cache.v[0][ids, :, pos % page], v[b].to(dtype))


def test_append_has_the_bits_of_the_contiguous_store(lib, cuda_dev):
    """f32, interleaved pairs: cq_rope_store_kv_f32 on a cache of one block per sequence."""
    B, T, Hq, Hkv, D, Tmax, pos0 = 2, 5, 4, 2, 128, 64, 20
    q, k, v = (torch.randn(B, T, h, D, device="cuda") for h in (Hq, Hkv, Hkv))
    ang = torch.rand(Tmax, D // 2, device="cuda") * 6.28
    cos, sin = ang.cos(), ang.sin()
    kc, vc = torch.zeros(B, Hkv, Tmax, D, device="cuda"), torch.zeros(B, Hkv, Tmax, D, device="cuda")
    q2, k2, pos = q.clone(), k.clone(), torch.tensor([pos0], dtype=torch.int32, device="cuda")
    lib.cq_rope_store_kv_f32(q2.data_ptr(), k2.data_ptr(), v.data_ptr(), cos.data_ptr(), sin.data_ptr(), pos.data_ptr(), kc.data_ptr(), vc.data_ptr(), B, T, Hq,
                             Hkv, D, Tmax, Hq * D, Hkv * D, Hkv * D, torch.cuda.current_stream().cuda_stream)
    capi.check("rope")
    cache = PagedKvCache(1, 8, 32, Hkv, D, B, Tmax)
    cache.reserve([0, 1], pos0 + T)
    got = cache.append(0, [0, 1], k, v, q=q, rotary=(cos, sin))
    cache.check()
    assert torch.equal(got, q2)
    for b in range(B):
        rows = cache.k[0][cache.tables[b].long()].permute(1, 0, 2, 3).flatten(1, 2), cache.v[0][cache.tables[b].long()].permute(1, 0, 2, 3).flatten(1, 2)
        assert torch.equal(rows[0][:, pos0:pos0 + T], kc[b, :, pos0:pos0 + T]) and torch.equal(rows[1][:, pos0:pos0 + T], vc[b, :, pos0:pos0 + T])


def test_append_faults(cuda_dev):
    cache = _make(8, 16, 1, 64, 4, 64, torch.float32)
    cache.reserve([0, 1], 10)
    row = lambda b, t: torch.ones((b, t, 1, 64), device="cuda")
    was = cache.k.clone()
    t = lambda *s: torch.tensor(s, dtype=torch.int32, device="cuda")
    tables = torch.ones((10, 32), device="cuda")
    for text, slots, n, rotary in (("out of range", t(4), 1, None), ("named twice", t(0, 0), 1, None), ("position", t(0), 11, None), ("position", t(2), 1, None),
                                   ("position", t(1), 1, (tables[:9].contiguous(), tables[:9].contiguous()))):
        q = cache.append(0, slots, row(len(slots), n), row(len(slots), n), q=row(len(slots), n), rotary=rotary)
        if text != "named twice":
            assert float(q[0, 0].abs().sum()) == 0.0
        again = cache.append(0, [0], row(1, 1), row(1, 1), q=row(1, 1))       # until the fault is taken: nothing stored, no query
        assert float(again.abs().sum()) == 0.0
        _faulted(cache, text)
        if text == "out of range":
            assert torch.equal(cache.k, was)
        cache.k.copy_(was)
    for bad in (dict(layer=1), dict(k=row(1, 1)[..., :32]), dict(v=row(1, 2)), dict(q=row(1, 1).half()), dict(rotary=(tables.double(), tables.double()))):
        kw = dict(layer=0, k=row(1, 1), v=row(1, 1), q=None, rotary=None)
        kw.update(bad)
        with pytest.raises(capi.CandleQError):
            cache.append(kw["layer"], [0], kw["k"], kw["v"], q=kw["q"], rotary=kw["rotary"])


# ---- attention ----
def _fill(cache, slot, n, g, layer=0):
    if n:
        cache.reserve([slot], n)
        kv = [torch.randn((1, n, cache.kv_heads, cache.head_dim), device="cuda", generator=g) for _ in range(2)]
        cache.append(layer, [slot], kv[0].to(cache.dtype), kv[1].to(cache.dtype))


def _attention64(cache, layer, q, slots, scale):
    """(out, tolerance) by the formula, sequence by sequence."""
    b, t, hq, d = q.shape
    per, page = hq // cache.kv_heads, cache.page_size
    out = torch.zeros(q.shape, dtype=torch.float64, device="cuda")
    worst = vmax = 0.0
    longest = 1
    lens = cache.lens.tolist()
    for i, s in enumerate(slots):
        n = lens[s]
        if n == 0:
            continue
        ids = cache.tables[s, :-(-n // page)].long()
        k = cache.k[layer][ids].permute(1, 0, 2, 3).flatten(1, 2)[:, :n].double().repeat_interleave(per, 0)
        v = cache.v[layer][ids].permute(1, 0, 2, 3).flatten(1, 2)[:, :n].double().repeat_interleave(per, 0)
        qi = q[i].double().permute(1, 0, 2)
        sc = torch.matmul(qi, k.transpose(1, 2)) * scale
        last = n - t + torch.arange(t, device="cuda")
        hidden = torch.arange(n, device="cuda")[None] > last[:, None]
        p = torch.softmax(sc.masked_fill(hidden[None], -math.inf), dim=-1)
        p = torch.where(last[None, :, None] >= 0, p, 0.0)
        out[i] = torch.matmul(p, v).permute(1, 0, 2)
        worst = max(worst, float(torch.matmul(qi.abs(), k.abs().transpose(1, 2)).max()) * scale)
        vmax, longest = max(vmax, float(v.abs().max())), max(longest, n)
    u = U[cache.dtype]
    e = 2 * (d + 4) * 2.0 ** -24 * worst + (longest + 64) * 2.0 ** -24 + (u if cache.dtype != torch.float32 else 0.0)
    return out, 2 * e * vmax / (1 - e) + u * vmax


def _batch(dtype, page, dim, hkv, prompts, own, seed=0, extra=0):
    """Slots of one group after another: prompts[g] tokens, then own[g][i] more for each of its sequences (None: an empty slot)."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    seqs = sum(len(o) for o in own) + len(prompts)
    longest = max(p + max([x or 0 for x in o]) for p, o in zip(prompts, own)) + extra
    per = -(-longest // page)
    cache = PagedKvCache(2, seqs * per, page, hkv, dim, seqs, longest, dtype=dtype)
    cache.k.fill_(float("nan"))                 # what no sequence has written
    cache.v.fill_(float("inf"))
    slots, at = [], len(prompts)
    for j, (p, o) in enumerate(zip(prompts, own)):
        _fill(cache, j, p, g)
        for x in o:
            if x is not None:
                if p:
                    cache.fork([j], [at])
                _fill(cache, at, x, g)
            slots.append(at)
            at += 1
    cache.check()
    return cache, slots, g


CASES = [
    # prompts, own tokens
    ([0], [[1]]), ([0], [[1, 2, 3]]), ([16], [[0]]), ([130], [[1, 40, 7]]), ([64], [[0, 0, 64, 65]]), ([300, 17], [[5, 200, 1], [1, 1]]),
    ([128], [[1, None, 3, None]]), ([257], [[130] * 9 + [1]]), ([33, 0, 500], [[3], [9, 9], [2, 600, 3, 4]]),
]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("page,dim,hkv,per", [(16, 64, 2, 4), (32, 128, 1, 1), (64, 128, 2, 5), (128, 64, 1, 32), (16, 128, 1, 8)])
@pytest.mark.parametrize("case", range(len(CASES)))
def test_attention_against_the_formula(cuda_dev, dtype, page, dim, hkv, per, case):
    prompts, own = CASES[case]
    cache, slots, g = _batch(dtype, page, dim, hkv, prompts, own, seed=case)
    q = torch.randn((len(slots), 1, hkv * per, dim), device="cuda", generator=g).to(dtype)
    ref, tol = _attention64(cache, 0, q, slots, dim ** -0.5)
    for groups in ([len(o) for o in own], None, [1] * len(slots)):      # as they are, all as one (they share nothing, or less), none
        plan = cache.attention_plan(len(slots), hkv * per, groups=groups)
        plan.update(slots)
        got = cache.attention(0, q, plan)
        cache.check()
        assert got.dtype == dtype and bool(((got.double() - ref).abs() <= tol).all()), float((got.double() - ref).abs().max()) / tol
        again = cache.attention(0, q, plan)
        assert torch.equal(got, again)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("queries", [2, 5, 9])
def test_attention_of_several_queries(cuda_dev, dtype, queries):
    """Each query sees the positions up to its own; keys and values of later ones may be anything."""
    cache, slots, g = _batch(dtype, 16, 64, 2, [100, 7], [[queries, 40, queries + 1], [queries - 1, 90]], seed=queries)
    q = torch.randn((5, queries, 6, 64), device="cuda", generator=g).to(dtype)
    ref, tol = _attention64(cache, 0, q, slots, 0.2)
    plan = cache.attention_plan(5, 6, queries=queries, groups=[3, 2])
    plan.update(slots)
    got = cache.attention(0, q, plan, scale=0.2)
    assert bool(((got.double() - ref).abs() <= tol).all())
    # the last position of every sequence made unusable: only the last query may notice
    for s in slots:
        n = int(cache.lens[s]) - 1
        page = int(cache.tables[s, n // 16])
        cache.k[0, page, :, n % 16] = float("nan")
        cache.v[0, page, :, n % 16] = float("inf")
    bad = cache.attention(0, q, plan, scale=0.2)
    cache.check()
    assert torch.equal(bad[:, :-1], got[:, :-1]) and not bool(torch.isfinite(bad[:, -1]).any())


def test_attention_with_fewer_positions_than_queries(cuda_dev):
    cache, slots, g = _batch(torch.float32, 16, 64, 1, [40], [[0, 3, None]], seed=1)
    cache.free([slots[0]])
    _fill(cache, slots[0], 2, g)                # two positions, four queries: the first two see nothing
    q = torch.randn((3, 4, 2, 64), device="cuda", generator=g)
    plan = cache.attention_plan(3, 2, queries=4)
    plan.update(slots)
    got = cache.attention(0, q, plan)
    cache.check()
    ref, tol = _attention64(cache, 0, q, slots, 0.125)
    assert bool(((got.double() - ref).abs() <= tol).all()) and float(got[0, :2].abs().max()) == 0.0 and float(got[2].abs().max()) == 0.0


def test_attention_finds_the_shared_pages_itself(cuda_dev):
    """Tables that agree, differ in the middle, or name the same slot twice: sharing only ever saves reads."""
    cache, slots, g = _batch(torch.bfloat16, 16, 128, 2, [200], [[5, 6, 7]], seed=5)
    q = torch.randn((4, 1, 8, 128), device="cuda", generator=g).to(torch.bfloat16)
    cache.free([slots[2]])
    cache.copy([slots[0]], [slots[2]])          # the same tokens in pages of its own
    use = [slots[0], slots[1], slots[2], slots[0]]
    plan = cache.attention_plan(4, 8)
    plan.update(use)
    got = cache.attention(0, q, plan)
    ref, tol = _attention64(cache, 0, q, use, 128 ** -0.5)
    assert bool(((got.double() - ref).abs() <= tol).all())
    # a page number out of range is a fault, and nothing is read there
    cache.tables[slots[1], 3] = cache.pages + 5
    plan.update(use)
    cache.attention(0, q, plan)
    _faulted(cache, "page")
    plan.update(torch.tensor([0, 1, 2, 99], dtype=torch.int32, device="cuda"))
    cache.attention(0, q, plan)
    _faulted(cache, "slot")


@pytest.mark.parametrize("dtype", TYPES)
def test_attention_of_scores_that_are_not_finite(cuda_dev, dtype):
    """NaN and infinite scores give what the formula gives; a key of -inf scores alone among others has no weight."""
    cache, slots, g = _batch(dtype, 16, 64, 1, [48], [[4, 4, 4]], seed=2)
    q = torch.rand((3, 1, 1, 64), device="cuda", generator=g).to(dtype) + 0.5
    at = lambda s, n: (0, int(cache.tables[s, n // 16]), 0, n % 16)
    cache.k[at(slots[0], 50)] = float("-inf")
    cache.k[at(slots[1], 50)] = float("inf")
    cache.k[at(slots[2], 51)] = float("nan")
    plan = cache.attention_plan(3, 1)
    plan.update(slots)
    got = cache.attention(0, q, plan)
    assert bool(torch.isfinite(got[0]).all()) and bool(torch.isnan(got[1]).all()) and bool(torch.isnan(got[2]).all())
    ref = _attention64(cache, 0, q, slots, 0.125)[0][0]
    assert bool(((got[0].double() - ref).abs() <= 4 * (U[dtype] + 2.0 ** -16) * float(cache.v[0][cache.tables[slots[0], :3].long()].abs().max())).all())


def test_attention_arguments(cuda_dev):
    cache = _make(8, 16, 2, 64, 4, 64, torch.float32)
    cache.reserve([0, 1], 10)
    plan = cache.attention_plan(2, 4)
    q = torch.zeros((2, 1, 4, 64), device="cuda")
    with pytest.raises(capi.CandleQError, match="no slots yet"):
        cache.attention(0, q, plan)
    plan.update([0, 1])
    for bad in (q[:1], q[..., :32], q.half(), q[:, :, :2]):
        with pytest.raises(capi.CandleQError):
            cache.attention(0, bad, plan)
    with pytest.raises(capi.CandleQError):
        cache.attention(0, q, plan, scale=0.0)
    with pytest.raises(capi.CandleQError, match="another cache"):
        _make(8, 16, 2, 64, 4, 64, torch.float32).attention(0, q, plan)
    with pytest.raises(capi.CandleQError, match="add up"):
        cache.attention_plan(3, 4, groups=[1, 1])
    with pytest.raises(capi.CandleQError, match="2 slots"):
        plan3 = cache.attention_plan(3, 4)
        plan3.update([0, 1])


def test_strided_queries_layers_and_streams(cuda_dev):
    cache, slots, g = _batch(torch.float16, 32, 128, 2, [150], [[9, 30]], seed=8)
    cache.k[1], cache.v[1] = cache.v[0], cache.k[0]         # another layer
    wide = torch.randn((2, 8 * 128 + 64), device="cuda", generator=g).half()
    q = wide[:, :8 * 128].unflatten(1, (8, 128)).unsqueeze(1)
    plan = cache.attention_plan(2, 8)
    plan.update(slots)
    a = cache.attention(0, q, plan)
    assert torch.equal(a, cache.attention(0, q.contiguous(), plan))
    odd = torch.empty(2 * 8 * 128 + 1, dtype=torch.float16, device="cuda")[1:].view(2, 1, 8, 128)       # off the 16-byte grid
    odd.copy_(q)
    assert torch.equal(a, cache.attention(0, odd, plan))
    swapped = q.transpose(1, 2).contiguous().transpose(1, 2)
    assert torch.equal(a, cache.attention(0, swapped, plan))
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        plan.update(slots)
        b = cache.attention(0, q, plan)
    side.synchronize()
    assert torch.equal(a, b)


def test_a_step_in_a_graph(cuda_dev):
    """reserve, append, plan and attention of a decode step, captured once and replayed while the sequences grow into new pages."""
    dtype = torch.bfloat16
    cache, slots, g = _batch(dtype, 16, 64, 2, [70], [[1, 9, 14]], seed=4, extra=40)
    s = torch.tensor(slots, dtype=torch.int32, device="cuda")
    q, k, v = (torch.zeros((3, 1, h, 64), dtype=dtype, device="cuda") for h in (4, 2, 2))
    plan = cache.attention_plan(3, 4)

    def step():
        cache.reserve(s, 1)
        qr = cache.append(0, s, k, v, q=q)
        plan.update(s)
        return cache.attention(0, qr, plan)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
        side.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            out = step()
    torch.cuda.synchronize()
    for i in range(20):
        for x in (q, k, v):
            x.normal_(generator=g)
        graph.replay()
        ref, tol = _attention64(cache, 0, q, slots, 0.125)
        assert bool(((out.double() - ref).abs() <= tol).all())
    cache.check()
    assert int(cache.lens[slots[0]]) == 70 + 1 + 21


def test_a_sequence_can_come_and_go(cuda_dev):
    """A pool used to its last page: fork, grow, free, compact, and the contexts that stay are the same."""
    dtype = torch.float32
    cache, slots, g = _batch(dtype, 16, 64, 1, [90], [[3, 20, 31, 8]], seed=6)
    q = torch.randn((4, 1, 2, 64), device="cuda", generator=g)
    plan = cache.attention_plan(4, 2)
    plan.update(slots)
    was = cache.attention(0, q, plan)
    cache.free([slots[1]])
    cache.free([0])
    cache.compact()
    cache.check()
    live = int((cache.refs > 0).sum())
    assert bool((cache.refs[:live] > 0).all()) and bool((cache.refs[live:] == 0).all())
    plan.update(slots)
    now = cache.attention(0, q, plan)
    keep = [0, 2, 3]
    assert torch.equal(now[keep], was[keep]) and float(now[1].abs().max()) == 0.0


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("dim", [64, 128])
def test_infinite_values_and_plain_numbers(cuda_dev, dtype, dim):
    """Queries, keys and values of few significant bits (1, 0.5, infinities): an infinity comes out as the formula has it, also where the other factor leaves
    nothing behind its first bits."""
    cache, slots, g = _batch(dtype, 16, dim, 1, [40], [[3, 3]], seed=3)
    ids = cache.tables[slots[0], :3].long()
    cache.k[0][cache.tables[slots, :3].long()] = 1.0
    cache.v[0][cache.tables[slots, :3].long()] = 0.5
    at = lambda s, n: (0, int(cache.tables[s, n // 16]), 0, n % 16)
    cache.k[at(slots[0], 41)] = -math.inf            # this sequence's own key: a score of -inf, no weight
    cache.v[at(slots[1], 42) + (5,)] = math.inf      # one value of the other's
    q = torch.full((2, 1, 2, dim), 0.5, dtype=dtype, device="cuda")
    plan = cache.attention_plan(2, 2)
    plan.update(slots)
    got = cache.attention(0, q, plan)
    want = torch.full_like(got, 0.5)
    want[1, :, :, 5] = math.inf
    assert torch.equal(got, want)


@pytest.mark.parametrize("dim", [64, 128])
def test_the_largest_numbers_and_any_nan_in_f32(cuda_dev, dim):
    """Numbers that would round to infinity when split, where their products are finite, and a NaN with nothing but its last bit set."""
    cache, slots, g = _batch(torch.float32, 16, dim, 1, [40], [[3, 3]], seed=3)
    rows = cache.tables[slots, :3].long()
    big = torch.finfo(torch.float32).max
    cache.k[0][rows] = 1.0
    cache.k[0, :, :, :, 4] = 0.0
    cache.v[0][rows] = 0.5
    at = lambda s, n: (0, int(cache.tables[s, n // 16]), 0, n % 16)
    cache.k[at(slots[0], 7) + (2,)] = -big           # a shared key, times 0 of the query
    cache.k[at(slots[0], 41) + (2,)] = big           # an own one
    cache.v[at(slots[0], 9) + (3,)] = big            # a shared value
    cache.v[at(slots[0], 42) + (6,)] = -big
    cache.v.view(torch.int32)[at(slots[1], 42) + (5,)] = 0x7F800001
    q = torch.full((2, 1, 2, dim), 0.5, device="cuda")
    q[..., 2] = 0.0
    q[..., 4] = big
    plan = cache.attention_plan(2, 2)
    plan.update(slots)
    got = cache.attention(0, q, plan)
    want = torch.full_like(got, 0.5)
    want[:, :, :, 3] = big / 43
    want[0, :, :, 6] = -big / 43
    want[1, :, :, 5] = math.nan
    # 43 equal weights: the sums' and the quotient's roundings, and the other values' part of 43 * 0.5 / big.
    torch.testing.assert_close(got, want, rtol=50 * 2.0 ** -24, atol=0, equal_nan=True)


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("prompt", [40, 700])
def test_the_largest_values_of_bf16(cuda_dev, dim, prompt):
    """Sums of many values that are nearly the largest number: no weight passes 1 by a rounding, and no sum of them overflows where the mean does not."""
    cache, slots, g = _batch(torch.bfloat16, 16, dim, 1, [prompt], [[3] * 9], seed=3)
    rows = cache.tables[slots].long().clamp(min=0)
    big = torch.finfo(torch.bfloat16).max
    cache.k[0][rows] = 1.0
    cache.v[0][rows] = big
    q = torch.full((9, 1, 4, dim), 0.3, dtype=torch.bfloat16, device="cuda")
    plan = cache.attention_plan(9, 4)
    plan.update(slots)
    got = cache.attention(0, q, plan).double()
    # equal weights: what is left are the roundings of the sums (f32) and of the result (2^-8)
    assert bool(((got - big).abs() <= (2.0 ** -8 + 1e-4) * big).all())


def test_append_leaves_shared_pages_alone(cuda_dev):
    """More tokens than the slot has reserved since its fork would reach into pages that the other one reads."""
    cache = _make(8, 16, 1, 64, 4, 64, torch.float32)
    row = lambda b, t: torch.ones((b, t, 1, 64), device="cuda")
    cache.reserve([0], 20)
    cache.append(0, [0], row(1, 20), row(1, 20))
    cache.fork([0], [1])
    cache.reserve([1], 2)
    was = cache.k.clone()
    cache.append(0, [1], 2 * row(1, 6), row(1, 6))          # positions 16 .. 21: pages of its own
    cache.check()
    assert float(cache.k[0, int(cache.tables[1, 1]), 0, :6].min()) == 2.0 and torch.equal(cache.k[:, cache.tables[0, :2].long()], was[:, cache.tables[0, :2].long()])
    cache.append(0, [1], 3 * row(1, 7), row(1, 7))
    assert torch.equal(cache.k[:, cache.tables[0, :2].long()], was[:, cache.tables[0, :2].long()])
    _faulted(cache, "shared page")
    cache.free([0])
    cache.append(0, [1], 3 * row(1, 7), row(1, 7))          # now it is alone
    cache.check()
    assert float(cache.k[0, int(cache.tables[1, 0]), 0, 15, 0]) == 3.0


def test_empty_lists_change_nothing(cuda_dev):
    cache = _make(8, 16, 1, 64, 4, 64, torch.float32)
    cache.reserve([0], 20)
    was = cache.state.clone()
    cache.reserve([], 3), cache.free([]), cache.fork([], []), cache.copy([], []), cache.reserve([0], 0)
    cache.check()
    assert torch.equal(cache.state, was)
    with pytest.raises(capi.CandleQError, match="5 slots"):
        cache.reserve([0, 1, 2, 3, 0], 1)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("seqs,queries,hkv,per,dim,prompt,own", [(20, 4, 2, 16, 64, 70, 9), (130, 1, 1, 32, 128, 150, 5), (1, 1, 1, 1, 64, 0, 20000), (3, 1, 1, 2, 128, 9000, 40),
                                                                 (1, 1, 8, 4, 128, 0, 4000)])
def test_attention_of_many_and_few_rows(cuda_dev, dtype, seqs, queries, hkv, per, dim, prompt, own):
    """From rows with one or two segments each to one row with more than a thousand: the joins by one, two and eight warps a row, the last in several rounds."""
    cache, slots, g = _batch(dtype, 64, dim, hkv, [prompt], [[own] * seqs], seed=seqs, extra=1)
    q = torch.randn((seqs, queries, hkv * per, dim), device="cuda", generator=g).to(dtype)
    ref, tol = _attention64(cache, 0, q, slots, dim ** -0.5)
    plan = cache.attention_plan(seqs, hkv * per, queries=queries)
    plan.update(slots)
    got = cache.attention(0, q, plan)
    cache.check()
    assert bool(((got.double() - ref).abs() <= tol).all()), float((got.double() - ref).abs().max()) / tol
    assert torch.equal(got, cache.attention(0, q, plan))


@pytest.mark.parametrize("dtype", TYPES)
def test_two_plans_on_two_streams(cuda_dev, dtype):
    """Two batches over one cache at once, eager and from two graphs: each has its own plan, the cache is only read."""
    cache, slots, g = _batch(dtype, 16, 64, 2, [300, 40], [[20, 30, 40], [7, 9]], seed=4)
    parts = [torch.tensor(slots[:3], dtype=torch.int32, device="cuda"), torch.tensor(slots[3:], dtype=torch.int32, device="cuda")]
    qs = [torch.randn((len(p), 1, 8, 64), device="cuda", generator=g).to(dtype) for p in parts]
    plans = [cache.attention_plan(len(p), 8) for p in parts]
    streams = [torch.cuda.Stream() for _ in parts]

    def step(i):
        plans[i].update(parts[i])
        return cache.attention(0, qs[i], plans[i])

    want = [step(i).clone() for i in range(2)]
    torch.cuda.synchronize()
    graphs, outs = [], []
    for i in range(2):
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[i], stream=streams[i]):
            outs.append(step(i))
    for _ in range(5):
        for i in range(2):
            with torch.cuda.stream(streams[i]):
                graphs[i].replay()
    torch.cuda.synchronize()
    assert torch.equal(outs[0], want[0]) and torch.equal(outs[1], want[1])
    for _ in range(5):
        for i in range(2):
            with torch.cuda.stream(streams[i]):
                outs[i] = step(i)
    torch.cuda.synchronize()
    assert torch.equal(outs[0], want[0]) and torch.equal(outs[1], want[1])
    cache.check()
