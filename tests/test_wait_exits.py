"""Waits that give up must not leave the rest of a CTA behind at a barrier: read from the source, since a kernel that hangs is not run."""
import os
import re

from candle_b200 import build


def test_roles_have_no_barrier_without_a_limit():
    """The warps of the tcgen05 attention give up one by one, each at any of its waits.  So inside a role they meet at mbarriers, whose waits are limited; the barriers
    without a limit come behind the roles, and every warp gets there."""
    text = re.sub(r"//[^\n]*", "", open(os.path.join(build.CSRC, "prefix_attn_mma.cu")).read())
    kernel = text.index("prefix_mma_kernel(const cq_kv_cache")
    roles, body = text[text.index("__device__ bool softmax_part"):kernel], text[kernel:text.index("bool encode(")]
    unlimited = r"bar\.sync|barrier\.(?!cluster)|__syncthreads|cq_mbar_wait\b"
    assert not re.search(unlimited, roles)
    assert re.search(unlimited, body) and not re.search(r"\breturn\b", body)
