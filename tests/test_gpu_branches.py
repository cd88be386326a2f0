"""LlamaShapedDecoder.branches: prompt, log probabilities, fork, paged store and shared-prefix attention together, as a program uses them."""
import pytest
import torch

from candle_b200.decoder import DecoderConfig, LlamaShapedDecoder
from candle_b200.logprobs import token_logprobs
from test_gpu_kv_cache import _attention64

pytestmark = pytest.mark.gpu


def _model(dtype, **over):
    cfg = DecoderConfig.tiny()
    for k, v in over.items():
        setattr(cfg, k, v)
    m = LlamaShapedDecoder(cfg, "cuda:0", batch=1, seed=5)
    m.use_pages(64, page_size=16, max_seqs=12, dtype=dtype)
    return m


def _prompt(m, n):
    return torch.randint(0, m.cfg.vocab, (1, n), device="cuda", generator=torch.Generator(device="cuda").manual_seed(n))


@pytest.mark.parametrize("n_tokens", [1, 37, 64, 70])
def test_the_prompt_has_the_bits_of_forward(cuda_dev, n_tokens):
    m = _model(torch.float32)
    prompt = _prompt(m, n_tokens)
    m.fuse_quantize = m.fuse_rope = False
    m.forward(prompt)
    want = m.last_logits.clone()
    m.kv.reset(), m.reset()
    assert torch.equal(m._prompt_pages(prompt), want)
    ids = m.kv.tables[0, :-(-n_tokens // 16)].long()
    for li, L in enumerate(m.layers):
        for pool, flat in ((m.kv.k, L.k_cache), (m.kv.v, L.v_cache)):
            assert torch.equal(pool[li][ids].permute(1, 0, 2, 3).flatten(1, 2)[:, :n_tokens], flat[0, :, :n_tokens])


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("n_tokens,n,steps", [(37, 5, 4), (64, 12, 3), (1, 2, 2), (20, 1, 3), (8, 4, 1)])
def test_branches(cuda_dev, dtype, n_tokens, n, steps):
    """Every step from its own inputs: the attention of both layers against the 64-bit formula over the pages, tokens and numbers against the logits."""
    m = _model(dtype)
    prompt = _prompt(m, n_tokens)
    record, checked = [], 0
    real = m.forward_pages

    def watched(tokens, slots, plan):
        nonlocal checked
        m.tap = {}
        logits = real(tokens, slots, plan)
        for li in range(m.cfg.layers):
            ref, tol = _attention64(m.kv, li, m.tap[f"{li}.q_rot"], slots.tolist(), m.cfg.head_dim ** -0.5)
            assert bool(((m.tap[f"{li}.att"].double() - ref).abs() <= tol).all())
            checked += 1
        m.tap = None
        assert m.kv.lens[:n].tolist() == [n_tokens + len(record) + 1] * n
        record.append(logits.clone())
        return logits

    m.forward_pages = watched
    got = m.branches(prompt, n, steps)
    assert checked == m.cfg.layers * (steps - 1) and got.tokens.shape == got.logprobs.shape == got.entropy.shape == (n, steps)
    m.kv.reset(), m.reset()
    first = token_logprobs(m._prompt_pages(prompt), top=n)
    assert torch.equal(got.tokens[:, 0], first.top_ids[0]) and torch.equal(got.logprobs[:, 0], first.top_logprobs[0])
    assert torch.equal(got.entropy[:, 0], first.entropy.expand(n)) and len(set(got.tokens[:, 0].tolist())) == n
    for i, logits in enumerate(record):
        assert torch.equal(got.tokens[:, i + 1], logits.argmax(-1))
        lp = torch.log_softmax(logits.double(), -1)
        assert bool((got.logprobs[:, i + 1].double() - lp.max(-1).values).abs().max() <= 2.0 ** -23 * 230)
    del m.forward_pages
    again = m.branches(prompt, n, steps)
    for a, b in zip(got, again):
        assert torch.equal(a, b)
    assert int(m.kv.lens.sum()) >= 0 and bool((m.kv.refs == 0).all())


def test_branches_share_the_prompt(cuda_dev):
    m = _model(torch.float32)
    seen = []
    real = m.forward_pages
    m.forward_pages = lambda t, s, p: (seen.append(int((m.kv.refs > 0).sum())), real(t, s, p))[1]
    m.branches(_prompt(m, 50), 8, 2)            # three full pages shared, the fourth copied for each
    assert seen == [3 + 8]


def test_refusals(cuda_dev):
    m = LlamaShapedDecoder(DecoderConfig.tiny(), "cuda:0")
    p = _prompt(m, 5)
    with pytest.raises(ValueError, match="use_pages"):
        m.branches(p, 2, 2)
    m.use_pages(4, page_size=16, max_seqs=3)
    for args in ((p, 4, 2), (p, 0, 2), (p, 2, 0), (p.repeat(2, 1), 2, 2), (p[:, :0], 2, 2), (p, 2, m.cfg.max_pos)):
        with pytest.raises(ValueError):
            m.branches(*args)
    with pytest.raises(Exception, match="out of pages"):
        m.branches(_prompt(m, 40), 3, 2)        # three pages, and one more for each of two forks


def test_logits_that_are_no_distribution(cuda_dev, monkeypatch):
    """A NaN among the logits (the quantized products make none of their own: their activations' blocks drop it): tokens of -1 that are not looked up, NaN for
    their numbers, the cache empty as ever."""
    m = _model(torch.float32)
    real = m._logits

    def with_nan(*args):
        logits = real(*args)
        logits[:, 7] = float("nan")
        return logits

    monkeypatch.setattr(m, "_logits", with_nan)
    got = m.branches(_prompt(m, 20), 3, 4)
    assert bool((got.tokens == -1).all()) and bool(got.logprobs.isnan().all()) and bool(got.entropy.isnan().all())
    assert int(m.kv.lens.sum()) == 0 and int(m.kv.refs.sum()) == 0


def test_a_plan_of_another_shape_is_refused(cuda_dev):
    m = _model(torch.float32)
    slots = torch.arange(2, dtype=torch.int32, device="cuda")
    tokens = torch.zeros((2, 1), dtype=torch.int64, device="cuda")
    for plan in (m.kv.attention_plan(3, m.hq_l), m.kv.attention_plan(2, m.hq_l, queries=2), m.kv.attention_plan(2, 2 * m.hq_l)):
        with pytest.raises(ValueError):
            m.forward_pages(tokens, slots, plan)
    assert int(m.kv.lens.sum()) == 0
