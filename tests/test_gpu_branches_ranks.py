"""LlamaShapedDecoder.branches at two tensor-parallel ranks, both on one device: one host thread each, of which one runs at a time, from gather to gather; the gather joins
the slices that both have left.  Nothing on the device waits for the other rank."""
import threading

import pytest
import torch

import candle_b200.decoder as decoder
from candle_b200.decoder import DecoderConfig, LlamaShapedDecoder
from test_gpu_kv_cache import _attention64

pytestmark = pytest.mark.gpu


class _Lockstep:
    """`run(work)` calls work(rank) for each rank in turn; `gather(rank)` is that rank's gather."""

    def __init__(self, world):
        self.world, self.turn, self.parts, self.cv, self.failed = world, 0, [None] * world, threading.Condition(), None

    def _yield(self, rank, done=False):
        with self.cv:
            self.turn = (rank + 1) % self.world
            self.cv.notify_all()
            if not done:
                assert self.cv.wait_for(lambda: self.turn == rank or self.failed, timeout=60)
                if self.failed:
                    raise RuntimeError("another rank has failed")

    def gather(self, rank):
        def call(local):
            self.parts[rank] = local.clone()
            self._yield(rank)                       # back here when the others have left theirs
            full = torch.cat(self.parts, dim=1)
            self._yield(rank)                       # and when they have read these
            return full
        return call

    def run(self, work):
        out = [None] * self.world

        def one(rank):
            try:
                with self.cv:
                    assert self.cv.wait_for(lambda: self.turn == rank or self.failed, timeout=60)
                out[rank] = work(rank)
                self._yield(rank, done=True)
            except BaseException as e:
                with self.cv:
                    self.failed = self.failed or e
                    self.cv.notify_all()

        threads = [threading.Thread(target=one, args=(r,)) for r in range(self.world)]
        for t in threads:
            t.start()
        for t in threads:
            t.join()
        if self.failed:
            raise self.failed
        return out


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("n_tokens,n,steps", [(37, 5, 4), (64, 12, 3), (1, 2, 2)])
def test_branches_of_two_ranks(cuda_dev, monkeypatch, dtype, n_tokens, n, steps):
    """The first tokens, from the prompt's kernels, are those of one rank to the last bit; each rank's attention is that of its heads; both ranks come to the same."""
    cfg = DecoderConfig.tiny()
    prompt = torch.randint(0, cfg.vocab, (1, n_tokens), device="cuda", generator=torch.Generator(device="cuda").manual_seed(n_tokens))
    single = LlamaShapedDecoder(cfg, "cuda:0", batch=1, seed=5)
    single.use_pages(64, page_size=16, max_seqs=12, dtype=dtype)
    want = single.branches(prompt, n, steps)

    steps_of = _Lockstep(2)
    monkeypatch.setattr(decoder, "make_gatherer", lambda group, world, device: None)
    monkeypatch.setattr(torch.distributed, "barrier", lambda group=None: None)
    ranks = []
    for r in range(2):
        m = LlamaShapedDecoder(cfg, "cuda:0", rank=r, world=2, batch=1, seed=5)
        m.gather = steps_of.gather(r)
        m.use_pages(64, page_size=16, max_seqs=12, dtype=dtype)
        assert (m.hq_l, m.hkv_l) == (cfg.n_heads // 2, cfg.n_kv_heads // 2)
        ranks.append(m)
    checked = []

    def work(r):
        m = ranks[r]
        real = m.forward_pages

        def watched(tokens, slots, plan):
            m.tap = {}
            logits = real(tokens, slots, plan)
            for li in range(cfg.layers):
                ref, tol = _attention64(m.kv, li, m.tap[f"{li}.q_rot"], slots.tolist(), cfg.head_dim ** -0.5)
                assert bool(((m.tap[f"{li}.att"].double() - ref).abs() <= tol).all())
                checked.append(r)
            m.tap = None
            return logits

        m.forward_pages = watched
        return m.branches(prompt, n, steps)

    got = steps_of.run(work)
    for a, b in zip(*got):
        assert torch.equal(a, b)
    for a, b in zip(got[0], want):
        assert a.shape == b.shape and torch.equal(a[:, 0], b[:, 0])
    assert checked.count(0) == checked.count(1) == cfg.layers * (steps - 1)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_the_cache_is_left_empty(cuda_dev, dtype):
    """Also where there were too few pages, found at the end."""
    m = LlamaShapedDecoder(DecoderConfig.tiny(), "cuda:0", batch=1, seed=5)
    kv = m.use_pages(4, page_size=16, max_seqs=3, dtype=dtype)
    prompt = torch.zeros((1, 20), dtype=torch.int64, device="cuda")
    m.branches(prompt, 3, 2)
    assert not bool(kv.lens.any()) and not bool(kv.refs.any()) and bool((kv.tables == -1).all())
    with pytest.raises(Exception, match="out of pages"):
        m.branches(prompt, 3, 20)
    assert not bool(kv.lens.any()) and not bool(kv.refs.any()) and bool((kv.tables == -1).all())
    kv.check()
    m.branches(prompt, 3, 2)
