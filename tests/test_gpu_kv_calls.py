"""Calls of the paged cache that its documentation allows or refuses, at their borders."""
import pytest
import torch

from candle_b200 import capi
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
