"""Attention over pages where its kernels have much to do: CTAs with many tiles of the shared items and more than one item, scores that rise along the context,
contexts of a thousand segments.

Values are one-hot by blocks of 16 positions, so that an output is the weight of some of the blocks: nothing cancels, and a lost or doubled block shows in an output of its own size.

Tolerance, for each output by itself.  With weights w (1 + d), |d| <= e, the quotient sum w v / sum w moves by at most 2 e / (1 - e) sum p |v|; the result is rounded once, u |out|.
e has
  the score's error: f32 products of three tf32 ones drop l l', 2^-22 of |a b|, and cut both l's by a bit, 2^-23 each; f16 and bf16 products are exact; the sums over d are cut,
    (d / 8 + 8) 2^-23 of sum |q k|; scale, log2 e and the difference from the maximum are rounded, 4 * 2^-24 of the largest |score|, and 2^-22 is ex2's own;
  the weight's rounding to 16 bits, u, in the product and in the sum alike;
  sums of weights: a step for every 16 keys of the longest context and 64 for lanes, warps and the join, 2^-23 each.
f16 weights below its normal numbers have an absolute error instead: half a step of 2^-24, of weights that are 2^7 times what the formula says: 2^-32 of the largest, for each key;
and f16 results below 2^-14 half a step of 2^-24 as well, 2^-25."""
import math

import pytest
import torch

from test_gpu_kv_cache import TYPES, U, _batch

pytestmark = pytest.mark.gpu


def _one_hot_values(cache, layer=0):
    """Every written block of 16 rows has ones in one dim, another one for each of its neighbours in the pool."""
    pages, heads, page, d = cache.v[layer].shape
    block = torch.arange(pages * page // 16, device="cuda").view(pages, 1, page // 16, 1) + 7 * torch.arange(heads, device="cuda").view(1, heads, 1, 1)
    hot = torch.nn.functional.one_hot((block % d).squeeze(-1).repeat_interleave(16, -1), d)
    written = torch.isfinite(cache.v[layer])
    cache.v[layer] = torch.where(written, hot.to(cache.dtype), cache.v[layer])


def _exact(cache, layer, q, slots, scale):
    """(out, tolerance), both [batch, queries, heads, dim] in 64 bits."""
    b, t, hq, d = q.shape
    per, page = hq // cache.kv_heads, cache.page_size
    out, size = torch.zeros(q.shape, dtype=torch.float64, device="cuda"), torch.zeros(q.shape, dtype=torch.float64, device="cuda")
    lens = cache.lens.tolist()
    terms = score = 0.0
    for i, s in enumerate(slots):
        n = lens[s]
        if n == 0:
            continue
        ids = cache.tables[s, :-(-n // page)].long()
        k = cache.k[layer][ids].permute(1, 0, 2, 3).flatten(1, 2)[:, :n].double()
        v = cache.v[layer][ids].permute(1, 0, 2, 3).flatten(1, 2)[:, :n].double()
        qi = q[i].double().permute(1, 0, 2).reshape(cache.kv_heads, per * t, d)
        sc = torch.matmul(qi, k.transpose(1, 2)) * scale
        last = n - t + torch.arange(t, device="cuda").repeat(per)
        hidden = torch.arange(n, device="cuda")[None] > last[:, None]
        p = torch.softmax(sc.masked_fill(hidden[None], -math.inf), dim=-1)
        p = torch.where(last[None, :, None] >= 0, p, 0.0)
        back = lambda x: x.view(cache.kv_heads, per, t, d).permute(2, 0, 1, 3).reshape(t, hq, d)
        out[i], size[i] = back(torch.matmul(p, v)), back(torch.matmul(p, v.abs()))
        finite = torch.where(torch.isfinite(k), k.abs(), 0.0)
        terms = max(terms, float(torch.matmul(qi.abs(), finite.transpose(1, 2)).max()) * scale)
        score = max(score, float(sc[torch.isfinite(sc)].abs().max()) if bool(torch.isfinite(sc).any()) else 0.0)
    u, f32, n = U[cache.dtype], cache.dtype == torch.float32, max(lens)
    e = terms * ((2.0 ** -21 if f32 else 0.0) + (d / 8 + 8) * 2.0 ** -23) + score * 4 * 2.0 ** -24 + 2.0 ** -22 + (0.0 if f32 else u) + (n / 16 + 64) * 2.0 ** -23
    tol = 2 * e / (1 - e) * size + u * out.abs()
    return out, tol + (n * 2.0 ** -32 * float(size.max()) * 2 + 2.0 ** -25 if cache.dtype == torch.float16 else 0.0)


def _check(cache, q, slots, groups, scale):
    ref, tol = _exact(cache, 0, q, slots, scale)
    plan = cache.attention_plan(len(slots), q.shape[2], queries=q.shape[1], groups=groups)
    plan.update(slots)
    got = cache.attention(0, q, plan, scale=scale)
    cache.check()
    off = (got.double() - ref).abs()
    assert bool((off <= tol).all()), f"{int((off > tol).sum())} of {off.numel()}, worst {float((off / tol.clamp_min(1e-300)).max()):.3g} times the tolerance"
    assert torch.equal(got, cache.attention(0, q, plan, scale=scale))
    return got


LONG = [
    # sequences and shared tokens of each group, KV heads, query heads a KV head, dim, page.  Units of the shared line, by 148 CTAs:
    ([40], [8000], 8, 4, 128, 128),              # 504: four a CTA, both halves (160 rows), every item by 16 CTAs
    ([70], [8192], 8, 4, 64, 16),                # 1024: seven, two row tiles (280 rows), the second with one half
    ([30, 40], [4111, 5003], 8, 4, 128, 16),     # 576: a CTA goes from one half of an item to the next item with two
    ([12, 9, 33], [130, 6000, 9000], 4, 8, 64, 128),     # items of 2, 47 and 71 units, one of two row tiles
    ([3], [40000], 8, 1, 128, 64),               # 2504: seventeen, three rows
]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("case", range(len(LONG)))
def test_many_tiles_a_cta(cuda_dev, dtype, case):
    sizes, prompts, hkv, per, dim, page = LONG[case]
    own = [[(37 * i + 11 * j) % 150 for i in range(n)] for j, n in enumerate(sizes)]
    cache, slots, g = _batch(dtype, page, dim, hkv, prompts, own, seed=case)
    _one_hot_values(cache)
    q = torch.randn((len(slots), 1, hkv * per, dim), device="cuda", generator=g).to(dtype)
    _check(cache, q, slots, sizes, dim ** -0.5)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("dim,page", [(64, 128), (128, 16)])
def test_many_tiles_of_several_queries(cuda_dev, dtype, dim, page):
    cache, slots, g = _batch(dtype, page, dim, 4, [6000], [[3 + (29 * i) % 170 for i in range(24)]], seed=dim)
    _one_hot_values(cache)
    q = torch.randn((24, 3, 16, dim), device="cuda", generator=g).to(dtype)
    _check(cache, q, slots, None, dim ** -0.5)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("dim,page,seqs,prompt,own", [(64, 16, 40, 8000, 40), (128, 128, 40, 8000, 40), (64, 64, 60, 0, 2500), (128, 32, 60, 0, 2500), (128, 16, 1, 0, 5000)])
def test_scores_that_rise(cuda_dev, dtype, dim, page, seqs, prompt, own):
    """By 10 in powers of two from each 32 keys to the next, four times, and back: within any 128 keys of a segment the maximum has to follow three times, and sums and
    outputs with it.  The last 32 of 128 keys have nearly all the weight."""
    cache, slots, g = _batch(dtype, page, dim, 4, [prompt], [[own] * seqs], seed=dim + page)
    q = 0.2 * torch.randn((seqs, 1, 16, dim), device="cuda", generator=g)
    q[..., 0] = 2.0
    step = 10 * math.log(2.0) / (2.0 * dim ** -0.5)
    for s in [0] + slots:
        n = int(cache.lens[s])
        at = torch.arange(n, device="cuda")
        ids = cache.tables[s].long()[at // page]
        cache.k[0][ids, :, at % page, 0] = (step * (at // 32 % 4)).to(dtype)[:, None]
    _one_hot_values(cache)
    _check(cache, q.to(dtype), slots, None, dim ** -0.5)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("seqs,heads,prompt,own", [(1, 1, 0, 20000), (3, 2, 9000, 40), (1, 32, 0, 4000), (130, 32, 150, 5)])
def test_no_block_is_lost(cuda_dev, dtype, seqs, heads, prompt, own):
    """From one row of more than a thousand segments to thousands of one or two."""
    cache, slots, g = _batch(dtype, 64, 128, 1, [prompt], [[own] * seqs], seed=seqs)
    _one_hot_values(cache)
    q = torch.randn((seqs, 1, heads, 128), device="cuda", generator=g).to(dtype)
    _check(cache, q, slots, None, 128 ** -0.5)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("seqs,heads", [(1, 1), (50, 32), (100, 32)])
def test_segments_of_nothing_but_minus_infinity(cuda_dev, dtype, seqs, heads):
    """A long context whose first third has scores of -inf, so that whole segments have no weight, and so has the first of the join's rounds or of its warps' shares (eight,
    two and one of them a row).  Others have one key.  Nothing but -inf: NaN, as the formula gives."""
    cache, slots, g = _batch(dtype, 64, 64, 1, [0], [[1] * (seqs - 1) + [20000]], seed=seqs)
    _one_hot_values(cache)
    q = torch.rand((seqs, 1, heads, 64), device="cuda", generator=g).to(dtype) + 0.5
    ids = cache.tables[slots[-1]].long()
    cache.k[0][ids[:105]] = -math.inf               # 6720 keys
    _check(cache, q, slots, None, 0.125)
    cache.k[0][ids] = -math.inf
    plan = cache.attention_plan(seqs, heads)
    plan.update(slots)
    got = cache.attention(0, q, plan)
    assert bool(torch.isnan(got[-1]).all()) and bool(torch.isfinite(got[:-1]).all())


@pytest.mark.parametrize("below", [20.5, 24.5])
@pytest.mark.parametrize("prompt,own,seqs", [(9000, 20, 40), (0, 9000, 3)])
def test_one_key_over_many_small_ones_in_f16(cuda_dev, prompt, own, seqs, below):
    """One key has nearly all the weight, and each of thousands of others 2^-20.5 or 2^-24.5 of it, less than f16's normal numbers: together they are what is left."""
    cache, slots, g = _batch(torch.float16, 64, 64, 1, [prompt], [[own] * seqs], seed=5)
    q = torch.zeros((seqs, 1, 4, 64), dtype=torch.float16, device="cuda")
    q[..., 0] = 1.0
    written = torch.isfinite(cache.k[0])
    cache.k[0] = torch.where(written, -below * math.log(2.0), cache.k[0].float()).half()
    cache.v[0] = torch.where(written, 1.0, cache.v[0].float()).half()
    for s in [0] if prompt else slots:
        cache.k[0, int(cache.tables[s, 3]), 0, 11] = 0.0
        cache.v[0, int(cache.tables[s, 3]), 0, 11] = 0.0
    got = _check(cache, q, slots, None, 1.0)
    assert float(got.min()) > 0.0


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("prompt,own", [(9000, 30), (0, 9000)])
def test_the_largest_values_of_f16(cuda_dev, dim, prompt, own):
    """All weights at the top of their range and all values the largest number: the sums stay finite and so does their quotient."""
    cache, slots, g = _batch(torch.float16, 16, dim, 1, [prompt], [[own] * 9], seed=3)
    q = torch.full((9, 1, 4, dim), 0.5, dtype=torch.float16, device="cuda")
    big = torch.finfo(torch.float16).max
    for s in [0] + slots:           # scores that rise by 7.5 in powers of two once: not enough for the maximum to follow
        n = int(cache.lens[s])
        at = torch.arange(n, device="cuda")
        ids = cache.tables[s].long()[at // 16]
        cache.k[0][ids, :, at % 16] = ((at // 128 % 2) * (7.5 * math.log(2.0) / (0.5 * dim ** 0.5))).half()[:, None, None]
        cache.v[0][ids, :, at % 16] = big
    got = _check(cache, q, slots, None, dim ** -0.5)
    assert float(got.min()) == big
