"""token_logprobs against log-softmax in 64 bits.

Tolerance: the logits are exact in both, x - M is rounded once (2^-24 |x - M|), an exp2 of a rounded product is within (2 + |x - M|) 2^-23, a sum of n positive
terms in a tree of 32 + 8 + 3 + parts levels within 64 * 2^-24 of itself, a log adds 2 ulp: |log p - exact| <= 2^-23 (|log p| + 200), where 200 covers terms
with |x - M| <= 100 (smaller ones weigh nothing).  The entropy's second sum has the same errors on terms that add up to at most its own size plus one: 2^-23 * 400 (1 + H)."""
import pytest
import torch

from candle_b200 import capi
from candle_b200.logprobs import token_logprobs

pytestmark = pytest.mark.gpu


def _check(x, tokens, top):
    got = token_logprobs(x, tokens, top)
    lp = torch.log_softmax(x.double(), dim=-1)
    lp = torch.where(lp < -3.4028235677973366e38, -torch.inf, lp)           # beyond the results' type, halfway to the next value: -inf there
    ent = -(torch.where(lp == -torch.inf, 0.0, lp.exp() * lp)).sum(-1)
    tol = 2.0 ** -23
    want = lp.gather(1, tokens[:, None])[:, 0]
    same = (got.logprob.double() == want) | ((got.logprob.double() - want).abs() <= tol * (want.abs() + 200))
    assert bool(same.all())
    assert bool(((got.entropy.double() - ent).abs() <= tol * 400 * (1 + ent)).all())
    order = torch.sort(x.float() + 0.0, dim=-1, descending=True, stable=True).indices[:, :top]
    assert torch.equal(got.top_ids, order)
    best = lp.gather(1, order)
    assert bool(((got.top_logprobs.double() == best) | ((got.top_logprobs.double() - best).abs() <= tol * (best.abs() + 200))).all())


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("rows,vocab", [(1, 1), (3, 2), (2, 33), (5, 1000), (2, 8183), (3, 8184), (1, 8193), (4, 32000), (7, 50257), (2, 128256)])
def test_against_log_softmax(cuda_dev, dtype, rows, vocab):
    g = torch.Generator(device="cuda").manual_seed(vocab)
    x = (torch.randn((rows, vocab), device="cuda", generator=g) * 4).to(dtype)
    x[0, vocab // 2] = 30.0
    tokens = torch.randint(0, vocab, (rows,), device="cuda", generator=g)
    for top in {0, min(1, vocab), min(5, vocab), min(32, vocab)}:
        _check(x, tokens, top)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("vocab", [700, 20000])
def test_ties_and_masked_logits(cuda_dev, dtype, vocab):
    g = torch.Generator(device="cuda").manual_seed(3)
    x = torch.randint(-2, 3, (6, vocab), device="cuda", generator=g).to(dtype)          # thousands of equal ones
    x[0] = 0.0
    x[0, ::2] = -0.0                                                                     # equal as well
    x[1] = -torch.inf
    x[1, vocab - 1] = 3.0                                                                # one token alone: probability 1, entropy 0
    x[2, 10:] = -torch.inf                                                               # fewer tokens than alternatives
    x[3] = torch.finfo(dtype).min
    x[4] = torch.finfo(dtype).min
    x[4, 17] = torch.finfo(dtype).max
    tokens = torch.tensor([5, vocab - 1, 11, 3, 17, 0], device="cuda")
    _check(x, tokens, 32)
    got = token_logprobs(x, tokens, 2)
    assert float(got.logprob[1]) == 0.0 and float(got.entropy[1]) == 0.0 and float(got.logprob[2]) == -float("inf")


@pytest.mark.parametrize("rows", [1, 70])
def test_where_the_best_lie(cuda_dev, rows):
    """Together, at the row's ends, one in each part of it, ascending, with everything else masked: the search must not depend on it."""
    vocab, g = 150000, torch.Generator(device="cuda").manual_seed(rows)
    at = torch.arange(vocab, device="cuda")
    for values in (torch.where((at >= 5000) & (at < 5040), 1.0 + at / vocab, -torch.inf), torch.where(at % 4000 == 17, at / vocab, -3.0),
                   at / vocab, -at / vocab, torch.where(at % 1024 < 20, 2.0, torch.where(at > vocab - 9, 3.0, 0.0)), torch.where(at < 31, 1.0, -torch.inf)):
        x = values.float().repeat(rows, 1)
        _check(x, torch.randint(0, vocab, (rows,), device="cuda", generator=g), 32)


def test_rows_without_a_distribution(cuda_dev):
    x = torch.randn((5, 9000), device="cuda")
    good = token_logprobs(x, torch.zeros(5, dtype=torch.int64, device="cuda"), 4)
    x[0, 8999], x[1, 4], x[2] = float("nan"), float("inf"), -float("inf")
    x[3] = float("nan")
    got = token_logprobs(x, torch.zeros(5, dtype=torch.int64, device="cuda"), 4)
    assert bool(torch.isnan(got.logprob[:4]).all()) and bool(torch.isnan(got.entropy[:4]).all()) and bool(torch.isnan(got.top_logprobs[:4]).all())
    assert bool((got.top_ids[:4] == -1).all())
    for a, b in zip(got, good):
        assert torch.equal(a[4], b[4])


def test_tokens_and_shapes(cuda_dev):
    g = torch.Generator(device="cuda").manual_seed(9)
    x = torch.randn((2, 3, 5000), device="cuda", generator=g)
    tokens = torch.tensor([[4999, -1, 5000], [0, -100, 7]], device="cuda")
    got = token_logprobs(x, tokens, 3)
    ref = torch.log_softmax(x.double(), -1)
    assert got.logprob.shape == (2, 3) and got.top_ids.shape == (2, 3, 3)
    assert float(got.logprob[0, 1]) == 0.0 and float(got.logprob[1, 1]) == 0.0 and bool(torch.isnan(got.logprob[0, 2]))
    assert abs(float(got.logprob[0, 0]) - float(ref[0, 0, 4999])) < 1e-5
    one = token_logprobs(x[0, 0], tokens[0, 0])
    assert one.logprob.shape == () and torch.equal(one.logprob, got.logprob[0, 0]) and one.top_ids.shape == (0,)
    none = token_logprobs(x[:, :0], tokens[:, :0], 2)
    assert none.logprob.shape == (2, 0) and none.top_ids.shape == (2, 0, 2)
    assert token_logprobs(x, top=1).logprob is None
    for bad in (dict(tokens=tokens[:1]), dict(tokens=tokens.float()), dict(top=33), dict(top=-1)):
        with pytest.raises(capi.CandleQError):
            token_logprobs(x, bad.get("tokens", tokens), bad.get("top", 0))
    with pytest.raises(capi.CandleQError):
        token_logprobs(x.double())


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
def test_rows_off_the_grid(cuda_dev, dtype):
    """Rows at odd distances and odd addresses, whose neighbours hold what would change every number."""
    buf = torch.full((6 * 9001 + 16,), float("nan"), dtype=dtype, device="cuda")
    for off in (0, 1, 3, 7):
        x = torch.as_strided(buf, (5, 8997), (9001, 1), off)
        x.normal_()
        want = token_logprobs(x.contiguous(), torch.arange(5, device="cuda"), 7)
        got = token_logprobs(x, torch.arange(5, device="cuda"), 7)
        assert torch.equal(got.top_ids, want.top_ids)
        for a, b in zip(got[:3], want[:3]):             # another division into parts: another order of the sums
            assert bool(((a - b).abs() <= 2.0 ** -22 * (b.abs() + 200)).all())
        buf.fill_(float("nan"))
    assert torch.equal(token_logprobs(x.zero_().t().contiguous().t(), top=2).top_ids, torch.tensor([[0, 1]] * 5, device="cuda"))


def test_captured_and_on_another_stream(cuda_dev):
    x = torch.randn((3, 30000), device="cuda")
    tokens = torch.tensor([1, 2, 3], device="cuda")
    want = token_logprobs(x, tokens, 5)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        token_logprobs(x, tokens, 5)
        side.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            got = token_logprobs(x, tokens, 5)
    for _ in range(3):
        graph.replay()
    torch.cuda.synchronize()
    for a, b in zip(got, want):
        assert torch.equal(a, b)
