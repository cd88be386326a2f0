"""token_logprobs where the logits are numbered beyond 32 bits; tolerance as in test_gpu_logprobs.py."""
import pytest
import torch

from candle_b200.logprobs import token_logprobs

pytestmark = pytest.mark.gpu


def test_rows_beyond_32_bits(cuda_dev):
    """18,000 rows of 128256 in 16 bits: 2.3 billion logits, the last rows as by themselves."""
    x = torch.empty((18000, 128256), dtype=torch.bfloat16, device="cuda")
    x[-3:].normal_(generator=torch.Generator(device="cuda").manual_seed(1))
    x[:-3] = 0.0
    tokens = torch.arange(18000, device="cuda")
    got = token_logprobs(x, tokens, 3)
    lp = torch.log_softmax(x[-3:].double(), -1)
    assert torch.equal(got.top_ids[-3:], torch.sort(x[-3:].float(), dim=-1, descending=True, stable=True).indices[:, :3])
    assert bool(((got.logprob[-3:].double() - lp.gather(1, tokens[-3:, None])[:, 0]).abs() <= 2.0 ** -23 * 230).all())
    assert bool((got.top_ids[:-3] == torch.arange(3, device="cuda")).all())
