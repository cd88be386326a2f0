"""Serving several continuations of one prompt, as cases that can be timed and whose outputs can be compared.

Four kinds of work, each as a decoder's program calls it:

* ``attention`` - ``PagedKvCache.attention``: the decode attention of a batch whose sequences share the pages of a long prompt;
* ``fork`` / ``compact`` - ``PagedKvCache.fork`` and ``.compact``: sequences that go on from another one, and live pages moved to
  the front of the pool, over all layers of a model;
* ``append`` - ``PagedKvCache.append``: rotary embedding at each sequence's own position, keys and values stored into pages;
* ``logprobs`` - ``token_logprobs``: log probabilities of given tokens, the entropy of their distribution, the best alternatives.

``own`` false: the same in elementary tensor operations.  Caches hold normal keys and values with a spread between channels; the
pages of a sequence lie anywhere in the pool, as they do after some hours of service.
"""
from __future__ import annotations

import math

import torch

own = False

_DEVICE = "cuda:0"
_ELEM = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def listed():
    return [
        # --- attention of one decode step.  The decoder harness's own cache type and prompt length, eight continuations: the
        # smallest call, where launches count
        dict(name="attention_f32_b8_p512", kind="attention", elem="f32", heads=32, kv_heads=8, dim=128, page=64, groups=1, batch=8,
             queries=1, prompt=512, own_min=1, own_max=16),
        # 64 samples of one prompt of 8191 tokens (the last page of it is each sample's own), up to 1024 tokens further on
        dict(name="attention_bf16_b64_p8191", kind="attention", elem="bf16", heads=32, kv_heads=8, dim=128, page=64, groups=1,
             batch=64, queries=1, prompt=8191, own_min=1, own_max=1024),
        # four drafted tokens per sequence checked at once, small pages, more query heads per KV head
        dict(name="attention_f16_b32_q4_p2000", kind="attention", elem="f16", heads=64, kv_heads=8, dim=128, page=16, groups=1,
             batch=32, queries=4, prompt=2000, own_min=8, own_max=200),
        # four prompts with eight samples each, heads of 64, f32 cache
        dict(name="attention_f32_d64_4x8_p1500", kind="attention", elem="f32", heads=32, kv_heads=4, dim=64, page=32, groups=4,
             batch=32, queries=1, prompt=1500, own_min=1, own_max=400),
        # a batch of 128 over one long document: the largest
        dict(name="attention_bf16_b128_p32768", kind="attention", elem="bf16", heads=32, kv_heads=8, dim=128, page=128, groups=1,
             batch=128, queries=1, prompt=32768, own_min=1, own_max=1024),
        # --- pages.  63 continuations of a prompt that ends inside a page, 32 layers
        dict(name="fork_bf16_l32_1to63", kind="fork", elem="bf16", layers=32, kv_heads=8, dim=128, page=64, prompt=1000, children=63),
        # a pool after many sequences have ended: 64 of 160 live pages move to the front, 32 layers
        dict(name="compact_bf16_l32_m64", kind="compact", elem="bf16", layers=32, kv_heads=8, dim=128, page=64, pages=320, live=160,
             moves=64),
        # --- new keys and values.  One token of 64 sequences of different lengths: a decode step of one layer
        dict(name="append_bf16_b64_t1", kind="append", elem="bf16", inp="f32", heads=32, kv_heads=8, dim=128, page=64, batch=64,
             tokens=1, own_max=1024, neox=False),
        # a prompt of 2047 tokens, f32 cache
        dict(name="append_f32_b1_t2047", kind="append", elem="f32", inp="f32", heads=32, kv_heads=8, dim=128, page=64, batch=1,
             tokens=2047, own_max=100, neox=False),
        # --- log probabilities.  The token of one sequence with 20 alternatives: one row, where latency counts
        dict(name="logprobs_f32_r1_top20", kind="logprobs", elem="f32", rows=1, vocab=128256, top=20),
        # a step of 64 samples in 16 bits
        dict(name="logprobs_bf16_r64_top5", kind="logprobs", elem="bf16", rows=64, vocab=151936, top=5),
        # a whole text of 1024 tokens scored at once
        dict(name="logprobs_f32_r1024_top1", kind="logprobs", elem="f32", rows=1024, vocab=128256, top=1),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choices(["attention", "fork", "compact", "append", "logprobs"], [6, 1, 1, 1, 2])[0]
    elem = rng.choice(["f32", "f16", "bf16"])
    if kind == "attention":
        dim, page, kv = rng.choice([64, 128]), rng.choice([16, 32, 64, 128]), rng.choice([1, 2, 4, 8])
        per_kv = rng.choice([1, 2, 3, 4, 5, 8, 16])
        batch = _log_int(rng, 1, 128)
        groups = rng.choice([1, 1, 2, 3, 8])
        groups = min(groups, batch)
        queries = rng.choice([1, 1, 1, 2, 3, 5])
        own_max = _log_int(rng, queries + 1, 1500)
        prompt = _log_int(rng, 1, 32768 if elem != "f32" else 8192)
        while batch * queries * kv * per_kv * (prompt + own_max) > 120e6 or groups * prompt > 200000:
            prompt = prompt // 2 + 1
            own_max = max(queries + 1, own_max // 2)
        return dict(kind=kind, elem=elem, heads=kv * per_kv, kv_heads=kv, dim=dim, page=page, groups=groups, batch=batch,
                    queries=queries, prompt=prompt, own_min=queries, own_max=own_max)
    if kind == "fork":
        layers, page = _log_int(rng, 1, 32), rng.choice([16, 32, 64, 128])
        return dict(kind=kind, elem=elem, layers=layers, kv_heads=rng.choice([1, 2, 4, 8]), dim=rng.choice([64, 128]), page=page,
                    prompt=_log_int(rng, 2, 1500), children=_log_int(rng, 1, 31))
    if kind == "compact":
        pages = _log_int(rng, 8, 300)
        live = max(2, int(pages * rng.uniform(0.2, 0.7)))
        return dict(kind=kind, elem=elem, layers=_log_int(rng, 1, 16), kv_heads=rng.choice([1, 2, 4, 8]), dim=rng.choice([64, 128]),
                    page=rng.choice([16, 32, 64, 128]), pages=pages, live=live, moves=rng.randint(1, min(live, pages - live)))
    if kind == "append":
        kv = rng.choice([1, 2, 4, 8])
        batch = _log_int(rng, 1, 128)
        return dict(kind=kind, elem=elem, inp=rng.choice(["f32", elem]), heads=kv * rng.choice([1, 2, 4, 7]), kv_heads=kv,
                    dim=rng.choice([64, 128]), page=rng.choice([16, 32, 64, 128]), batch=batch,
                    tokens=max(1, min(_log_int(rng, 1, 2048), 4096 // batch)), own_max=_log_int(rng, 1, 1024), neox=rng.random() < 0.5)
    vocab = _log_int(rng, 1000, 160000)
    rows = _log_int(rng, 1, 1024)
    return dict(kind=kind, elem=elem, rows=max(1, min(rows, 1024 * 128256 // vocab)), vocab=vocab, top=rng.choice([0, 1, 3, 5, 8, 20, 32]))


def _gen(seed):
    g = torch.Generator(device=_DEVICE)
    g.manual_seed(seed)
    return g


def _spread(lo, hi, n):
    """n whole numbers from lo to hi, evenly spread."""
    return [lo + (hi - lo) * i // max(n - 1, 1) for i in range(n)]


def _group_sizes(case):
    b, g = case["batch"], case["groups"]
    return [b * (i + 1) // g - b * i // g for i in range(g)]


def _pool(case, layers, pages, gen):
    shape = (layers, pages, case["kv_heads"], case["page"], case["dim"])
    spread = torch.exp(0.5 * torch.randn(case["dim"], device=_DEVICE, generator=gen))
    k, v = torch.empty(shape, dtype=_ELEM[case["elem"]], device=_DEVICE), torch.empty(shape, dtype=_ELEM[case["elem"]], device=_DEVICE)
    for layer in range(layers):
        k[layer] = (torch.randn(shape[1:], device=_DEVICE, generator=gen) * spread).to(k.dtype)
        v[layer] = torch.randn(shape[1:], device=_DEVICE, generator=gen).to(v.dtype)
    return k, v


def _cache(case, k, v, refs, lens, tables):
    """What the program keeps: a cache object on the framework's side, its four parts as tensors on the other."""
    if not own:
        return dict(k=k, v=v, refs=refs, lens=lens, tables=tables)
    from candle_b200.kv_cache import PagedKvCache
    cache = PagedKvCache(k.shape[0], k.shape[1], case["page"], case["kv_heads"], case["dim"], tables.shape[0],
                         tables.shape[1] * case["page"], dtype=k.dtype, device=_DEVICE, pools=(k, v))
    cache.refs.copy_(refs)
    cache.lens.copy_(lens)
    cache.tables.copy_(tables)
    return cache


def _shared_pages(case):
    return case["prompt"] // case["page"]


def _lens(case):
    """Context lengths, queries included: the prompt and each sequence's own tokens."""
    return [case["prompt"] + t for t in _spread(case["own_min"], case["own_max"], case["batch"])]


def _prepare_attention(case, gen):
    page, batch, shared = case["page"], case["batch"], _shared_pages(case)
    order = torch.randperm(batch, device=_DEVICE, generator=gen).cpu().tolist()
    spread = _lens(case)
    lens = [spread[i] for i in order]
    need = [-(-n // page) for n in lens]
    sizes = _group_sizes(case)
    pages = shared * len(sizes) + sum(n - shared for n in need) + 3
    ids = torch.randperm(pages, device=_DEVICE, generator=gen).to(torch.int32).cpu()
    tables = torch.full((batch, max(need)), -1, dtype=torch.int32)
    refs = torch.zeros(pages, dtype=torch.int32)
    at = b = 0
    for size in sizes:
        prefix, at = ids[at:at + shared], at + shared
        for _ in range(size):
            mine = need[b] - shared
            tables[b, :need[b]] = torch.cat([prefix, ids[at:at + mine]])
            refs[tables[b, :need[b]].long()] += 1
            at, b = at + mine, b + 1
    k, v = _pool(case, 1, pages, gen)
    q = torch.randn((batch, case["queries"], case["heads"], case["dim"]), device=_DEVICE, generator=gen).to(k.dtype)
    lens_t = torch.tensor(lens, dtype=torch.int32, device=_DEVICE)
    st = dict(kind="attention", case=case, q=q, slots=torch.arange(batch, dtype=torch.int32, device=_DEVICE),
              cache=_cache(case, k, v, refs.to(_DEVICE), lens_t, tables.to(_DEVICE)))
    if own:
        st["plan"] = st["cache"].attention_plan(batch, case["heads"], queries=case["queries"], groups=sizes)
    return st


def _prepare_fork(case, gen):
    page, n = case["page"], case["children"]
    used = -(-case["prompt"] // page)
    pages = used + n + 5
    ids = torch.randperm(pages, device=_DEVICE, generator=gen).to(torch.int32)
    tables = torch.full((n + 1, used + 1), -1, dtype=torch.int32, device=_DEVICE)
    tables[0, :used] = ids[:used]
    refs = torch.zeros(pages, dtype=torch.int32, device=_DEVICE)
    refs[ids[:used].long()] = 1
    lens = torch.zeros(n + 1, dtype=torch.int32, device=_DEVICE)
    lens[0] = case["prompt"]
    k, v = _pool(case, case["layers"], pages, gen)
    saved = [refs.clone(), lens.clone(), tables.clone()]
    st = dict(kind="fork", case=case, cache=_cache(case, k, v, refs, lens, tables), saved=saved)
    st["src"] = torch.zeros(n, dtype=torch.int32, device=_DEVICE)
    st["dst"] = torch.arange(1, n + 1, dtype=torch.int32, device=_DEVICE)
    return st


def _prepare_compact(case, gen):
    pages, live, moves, page = case["pages"], case["live"], case["moves"], case["page"]
    low = torch.randperm(live, device=_DEVICE, generator=gen)[:live - moves]
    high = live + torch.randperm(pages - live, device=_DEVICE, generator=gen)[:moves]
    ids = torch.cat([low, high])[torch.randperm(live, device=_DEVICE, generator=gen)].to(torch.int32)
    width = min(8, live)
    seqs = -(-live // width)
    tables = torch.full((seqs * width,), -1, dtype=torch.int32, device=_DEVICE)
    tables[:live] = ids
    tables = tables.view(seqs, width)
    lens = ((tables >= 0).sum(1) * page - torch.arange(seqs, device=_DEVICE) % page).to(torch.int32)
    refs = torch.zeros(pages, dtype=torch.int32, device=_DEVICE)
    refs[ids.long()] = 1
    k, v = _pool(case, case["layers"], pages, gen)
    saved = [refs.clone(), lens.clone(), tables.clone()]
    return dict(kind="compact", case=case, cache=_cache(case, k, v, refs, lens, tables), saved=saved)


def _prepare_append(case, gen):
    page, batch, t = case["page"], case["batch"], case["tokens"]
    order = torch.randperm(batch, device=_DEVICE, generator=gen).cpu().tolist()
    spread = _spread(0, case["own_max"], batch)
    lens = [spread[i] + t for i in order]
    need = [-(-n // page) for n in lens]
    pages = sum(need) + 2
    ids = torch.randperm(pages, device=_DEVICE, generator=gen).to(torch.int32).cpu()
    tables = torch.full((batch, max(need)), -1, dtype=torch.int32)
    refs = torch.zeros(pages, dtype=torch.int32)
    at = 0
    for b in range(batch):
        tables[b, :need[b]] = ids[at:at + need[b]]
        at += need[b]
    refs[ids[:at].long()] = 1
    k, v = _pool(case, 1, pages, gen)
    inp, d = _ELEM[case["inp"]], case["dim"]
    row = lambda heads: torch.randn((batch, t, heads, d), device=_DEVICE, generator=gen).to(inp)
    inv = 1.0 / (500000.0 ** (torch.arange(0, d, 2, device=_DEVICE, dtype=torch.float32) / d))
    ang = torch.arange(max(lens), device=_DEVICE, dtype=torch.float32)[:, None] * inv[None, :]
    return dict(kind="append", case=case, cache=_cache(case, k, v, refs.to(_DEVICE), torch.tensor(lens, dtype=torch.int32, device=_DEVICE),
                                                       tables.to(_DEVICE)),
                slots=torch.arange(batch, dtype=torch.int32, device=_DEVICE), q=row(case["heads"]), k=row(case["kv_heads"]),
                v=row(case["kv_heads"]), cos=ang.cos(), sin=ang.sin())


def _prepare_logprobs(case, gen):
    rows, vocab = case["rows"], case["vocab"]
    logits = torch.empty((rows, vocab), dtype=_ELEM[case["elem"]], device=_DEVICE)
    for r in range(0, rows, 128):
        n = min(128, rows - r)
        logits[r:r + n] = (3.0 * torch.randn((n, vocab), device=_DEVICE, generator=gen)).to(logits.dtype)
    # a model is sure of many of its tokens
    best = torch.randint(0, vocab, (rows,), device=_DEVICE, generator=gen)
    at = torch.arange(rows, device=_DEVICE)
    logits[at, best] = (10.0 + 8.0 * torch.rand(rows, device=_DEVICE, generator=gen)).to(logits.dtype)
    other = torch.randint(0, vocab, (rows,), device=_DEVICE, generator=gen)
    tokens = torch.where(torch.rand(rows, device=_DEVICE, generator=gen) < 0.7, best, other)
    return dict(kind="logprobs", case=case, logits=logits, tokens=tokens)


_PREPARE = {"attention": _prepare_attention, "fork": _prepare_fork, "compact": _prepare_compact, "append": _prepare_append,
            "logprobs": _prepare_logprobs}


def prepare(case, seed):
    return _PREPARE[case["kind"]](case, _gen(seed))


# ---- the framework's calls ---------------------------------------------------------------------------------------------
def _restore(cache, saved):
    for mine, was in zip((cache.refs, cache.lens, cache.tables), saved):
        mine.copy_(was)


def _run_own(st):
    kind = st["kind"]
    if kind == "attention":
        st["plan"].update(st["slots"])
        return st["cache"].attention(0, st["q"], st["plan"])
    if kind == "append":
        cache = st["cache"]
        q = cache.append(0, st["slots"], st["k"], st["v"], q=st["q"], rotary=(st["cos"], st["sin"]), neox=st["case"]["neox"])
        return dict(q=q, k=cache.k, v=cache.v)
    if kind == "logprobs":
        from candle_b200.logprobs import token_logprobs
        got = token_logprobs(st["logits"], st["tokens"], top=st["case"]["top"])
        return [got.logprob, got.entropy, got.top_logprobs, got.top_ids]
    cache = st["cache"]
    _restore(cache, st["saved"])
    if kind == "fork":
        cache.fork(st["src"], st["dst"])
    else:
        cache.compact()
    return dict(k=cache.k, v=cache.v, refs=cache.refs, lens=cache.lens, tables=cache.tables)


# ---- the plain forms ---------------------------------------------------------------------------------------------------
def _rows_of(pool, ids):
    """[tokens, kv_heads, dim] of the pages `ids` in 32 bits."""
    return pool.index_select(0, ids).float().permute(0, 2, 1, 3).flatten(0, 1)


def _plain_attention(st):
    """Scores against the shared pages as one product for all sequences of a group, against the own ones padded to the longest."""
    case, c = st["case"], st["cache"]
    page, t, hkv, d = case["page"], case["queries"], case["kv_heads"], case["dim"]
    g = case["heads"] // hkv
    k_pool, v_pool, shared = c["k"][0], c["v"][0], _shared_pages(case)
    scale = 1.0 / math.sqrt(d)
    outs, b0 = [], 0
    for size in _group_sizes(case):
        tables, lens = c["tables"][b0:b0 + size], c["lens"][b0:b0 + size]
        q = st["q"][b0:b0 + size].float().view(size, t, hkv, g, d)
        parts = []
        if shared:
            kp = _rows_of(k_pool, tables[0, :shared])                       # [P, hkv, d]
            vp = _rows_of(v_pool, tables[0, :shared])
            parts.append(torch.matmul(q.permute(2, 0, 1, 3, 4).reshape(hkv, size * t * g, d), kp.permute(1, 2, 0))
                         .view(hkv, size, t * g, -1))
        width = tables.shape[1] - shared
        if width:
            own_ids = tables[:, shared:].clamp_min(0).flatten()
            ko = k_pool.index_select(0, own_ids).float().view(size, width, hkv, page, d).permute(2, 0, 1, 3, 4).reshape(hkv, size, width * page, d)
            vo = v_pool.index_select(0, own_ids).float().view(size, width, hkv, page, d).permute(2, 0, 1, 3, 4).reshape(hkv, size, width * page, d)
            s = torch.matmul(q.permute(2, 0, 1, 3, 4).reshape(hkv, size, t * g, d), ko.transpose(-1, -2))
            last = lens.view(-1, 1) - t + torch.arange(t, device=q.device)                  # [size, t]: last key of a query
            seen = shared * page + torch.arange(width * page, device=q.device) <= last.unsqueeze(-1)
            parts.append(s.view(hkv, size, t, g, -1).masked_fill(~seen[None, :, :, None, :], -math.inf).view(hkv, size, t * g, -1))
        s = torch.cat(parts, dim=-1) * scale
        s -= s.amax(dim=-1, keepdim=True)
        s.exp_()
        total = s.sum(dim=-1, keepdim=True)
        o = 0.0
        if shared:
            o = torch.matmul(s[..., :shared * page].reshape(hkv, size * t * g, -1), vp.permute(1, 0, 2)).view(hkv, size, t * g, d)
        if width:
            o = o + torch.matmul(s[..., shared * page:], vo)
        o = (o / total).view(hkv, size, t, g, d).permute(1, 2, 0, 3, 4).reshape(size, t, hkv * g, d)
        outs.append(o.to(st["q"].dtype))
        b0 += size
    return torch.cat(outs)


def _plain_fork(st):
    case, c = st["case"], st["cache"]
    for mine, was in zip((c["refs"], c["lens"], c["tables"]), st["saved"]):
        mine.copy_(was)
    n, full, part = case["children"], case["prompt"] // case["page"], case["prompt"] % case["page"]
    src, dst = st["src"].long(), st["dst"].long()
    rows = c["tables"].index_select(0, src)
    c["refs"].index_add_(0, rows[:, :full].flatten().long(), torch.ones(n * full, dtype=torch.int32, device=rows.device))
    if part:
        fresh = torch.argsort((c["refs"] != 0).to(torch.int8), stable=True)[:n]         # the lowest free pages
        last = rows[:, full].long()
        for pool in (c["k"], c["v"]):
            pool[:, fresh, :, :part] = pool[:, last, :, :part]
        c["refs"].index_fill_(0, fresh, 1)
        rows[:, full] = fresh.to(torch.int32)
    c["tables"].index_copy_(0, dst, rows)
    c["lens"].index_copy_(0, dst, c["lens"].index_select(0, src))
    return dict(k=c["k"], v=c["v"], refs=c["refs"], lens=c["lens"], tables=c["tables"])


def _plain_compact(st):
    c = st["cache"]
    for mine, was in zip((c["refs"], c["lens"], c["tables"]), st["saved"]):
        mine.copy_(was)
    live = c["refs"] > 0
    ids = torch.arange(live.numel(), device=live.device)
    front = ids < live.sum()
    src, dst = ids[live & ~front], ids[front & ~live]
    for pool in (c["k"], c["v"]):
        pool[:, dst] = pool[:, src]
    c["refs"][dst] = c["refs"][src]
    c["refs"][src] = 0
    to = ids.to(torch.int32)
    to[src] = dst.to(torch.int32)
    c["tables"].copy_(torch.where(c["tables"] >= 0, to[c["tables"].clamp_min(0).long()], c["tables"]))
    return dict(k=c["k"], v=c["v"], refs=c["refs"], lens=c["lens"], tables=c["tables"])


def _rotate(x, cos, sin, neox):
    """x [batch, tokens, heads, dim]; cos / sin [batch, tokens, 1, dim / 2]."""
    if neox:
        a, b = x.chunk(2, dim=-1)
        return torch.cat([a * cos - b * sin, a * sin + b * cos], dim=-1)
    a, b = x[..., 0::2], x[..., 1::2]
    return torch.stack([a * cos - b * sin, a * sin + b * cos], dim=-1).flatten(-2)


def _plain_append(st):
    case, c = st["case"], st["cache"]
    t, page = case["tokens"], case["page"]
    pos = c["lens"].long().view(-1, 1) - t + torch.arange(t, device=c["lens"].device)             # [batch, t]
    cos, sin = st["cos"][pos].unsqueeze(2), st["sin"][pos].unsqueeze(2)
    ids = c["tables"].long().gather(1, pos // page)
    c["k"][0][ids, :, pos % page] = _rotate(st["k"].float(), cos, sin, case["neox"]).to(c["k"].dtype)
    c["v"][0][ids, :, pos % page] = st["v"].to(c["v"].dtype)
    return dict(q=_rotate(st["q"].float(), cos, sin, case["neox"]).to(c["k"].dtype), k=c["k"], v=c["v"])


def _plain_logprobs(st):
    x, top, outs = st["logits"], st["case"]["top"], []
    vocab = x.shape[1]
    lowest = 0xffffffff - torch.arange(vocab, device=x.device)
    for r in range(0, x.shape[0], 256):                 # a part of the rows at a time, for the memory of the copies
        v = x[r:r + 256].float()
        v_max = v.amax(dim=-1, keepdim=True)
        z = v - v_max
        e = z.exp()
        total = e.sum(dim=-1, keepdim=True)
        log_total = total.log()
        entropy = (log_total - (e * z).sum(dim=-1, keepdim=True) / total).squeeze(-1)
        logprob = (z.gather(1, st["tokens"][r:r + 256].unsqueeze(1)) - log_total).squeeze(-1)
        # whole numbers in the order of the values, the lower index the greater among equals
        bits = v.view(torch.int32).to(torch.int64)
        key = torch.where(bits < 0, -(bits & 0x7fffffff), bits) * (1 << 32) + lowest
        best = key.topk(top, dim=-1).indices
        outs.append((logprob, entropy, z.gather(1, best) - log_total, best))
    return [torch.cat(part) for part in zip(*outs)]


_PLAIN = {"attention": _plain_attention, "fork": _plain_fork, "compact": _plain_compact, "append": _plain_append, "logprobs": _plain_logprobs}


def run(state):
    return _run_own(state) if own else _PLAIN[state["kind"]](state)


# ---- the definitions in 64 bits ----------------------------------------------------------------------------------------
def exact(case, seed):
    global own
    if case["kind"] in ("fork", "compact"):
        return None                                     # pages and whole numbers, nothing computed
    was, own = own, False
    try:
        st = prepare(case, seed)
    finally:
        own = was
    return {"attention": _exact_attention, "append": _exact_append, "logprobs": _exact_logprobs}[case["kind"]](st)


def _exact_attention(st):
    case, c = st["case"], st["cache"]
    t, hkv, page = case["queries"], case["kv_heads"], case["page"]
    g = case["heads"] // hkv
    out = torch.zeros(st["q"].shape, dtype=torch.float64, device=_DEVICE)
    for b, n in enumerate(c["lens"].tolist()):
        ids = c["tables"][b, :-(-n // page)].long()
        for h in range(hkv):
            keys, vals = c["k"][0][ids, h].reshape(-1, case["dim"])[:n].double(), c["v"][0][ids, h].reshape(-1, case["dim"])[:n].double()
            s = torch.einsum("tgd,nd->tgn", st["q"][b, :, h * g:(h + 1) * g].double(), keys) / math.sqrt(case["dim"])
            hidden = torch.arange(n, device=_DEVICE)[None, :] > n - t + torch.arange(t, device=_DEVICE)[:, None]
            p = torch.softmax(s.masked_fill(hidden[:, None, :], -math.inf), dim=-1)
            out[b, :, h * g:(h + 1) * g] = torch.einsum("tgn,nd->tgd", p, vals)
    return out


def _exact_append(st):
    case, c = st["case"], st["cache"]
    t, page, half = case["tokens"], case["page"], case["dim"] // 2
    first = torch.arange(half, device=_DEVICE) if case["neox"] else 2 * torch.arange(half, device=_DEVICE)
    second = first + (half if case["neox"] else 1)
    k, v, q = c["k"].double(), c["v"].double(), torch.empty(st["q"].shape, dtype=torch.float64, device=_DEVICE)

    def turned(x, p):           # x [t, heads, dim], p [t]
        co, si = st["cos"][p].double()[:, None], st["sin"][p].double()[:, None]
        y = torch.empty(x.shape, dtype=torch.float64, device=_DEVICE)
        y[..., first] = x[..., first].double() * co - x[..., second].double() * si
        y[..., second] = x[..., first].double() * si + x[..., second].double() * co
        return y

    for b, n in enumerate(c["lens"].tolist()):
        p = torch.arange(n - t, n, device=_DEVICE)
        ids = c["tables"][b].long()[p // page]
        q[b] = turned(st["q"][b], p)
        k[0][ids, :, p % page] = turned(st["k"][b], p)
        v[0][ids, :, p % page] = st["v"][b].double()
    return dict(q=q, k=k, v=v)


def _exact_logprobs(st):
    rows, top = st["logits"].shape[0], st["case"]["top"]
    logprob, entropy = (torch.empty(rows, dtype=torch.float64, device=_DEVICE) for _ in range(2))
    alternatives = torch.empty((rows, top), dtype=torch.float64, device=_DEVICE)
    for r in range(0, rows, 64):
        lp = torch.log_softmax(st["logits"][r:r + 64].double(), dim=-1)
        logprob[r:r + 64] = lp.gather(1, st["tokens"][r:r + 64, None])[:, 0]
        entropy[r:r + 64] = -(lp.exp() * lp).sum(dim=-1)
        alternatives[r:r + 64] = lp.topk(top, dim=-1).values
    return [logprob, entropy, alternatives, None]


# ---- what a pass cannot do without ---------------------------------------------------------------------------------------
def work(case):
    kind, es = case["kind"], _ELEM[case["elem"]].itemsize
    if kind == "logprobs":
        r, v, k = case["rows"], case["vocab"], case["top"]
        return {"bytes": r * v * es + r * (8 + 8 + 12 * k), "flops": 6 * r * v}
    token = case["kv_heads"] * case["dim"] * es * 2             # a key and a value of one layer, all heads
    if kind == "attention":
        b, t, hq, d = case["batch"], case["queries"], case["heads"], case["dim"]
        shared, lens = _shared_pages(case) * case["page"], _lens(case)
        keys = sum(n - t + 1 + i for n in lens for i in range(t))
        return {"bytes": (case["groups"] * shared + sum(n - shared for n in lens)) * token + 2 * b * t * hq * d * es, "flops": 4 * d * hq * keys}
    if kind == "fork":
        part, pages = case["prompt"] % case["page"], -(-case["prompt"] // case["page"])
        return {"bytes": case["layers"] * token * part * (1 + case["children"]) + 8 * case["children"] * pages, "flops": 0}
    if kind == "compact":
        return {"bytes": 2 * case["layers"] * token * case["page"] * case["moves"] + 8 * (case["pages"] + case["live"]), "flops": 0}
    rows, ins = case["batch"] * case["tokens"], _ELEM[case["inp"]].itemsize
    values = rows * case["dim"] * (case["heads"] + 2 * case["kv_heads"])
    return {"bytes": values * (ins + es) + rows * case["dim"] * 4, "flops": 3 * values}
