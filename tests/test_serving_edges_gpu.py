"""Calls at the edges of what the operators around the decode take."""
import math

import pytest
import torch

import mx_flash_attn_kernel_opt__b200 as pgqa
from tests import test_cross_gpu

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kv", ["bf16", "e4m3"])
@pytest.mark.parametrize("new,lens,Hq,Hkv", [
    ([40, 0, 3, 150], [700, 30, 0, 129], 8, 2),        # whole items, rows without keys among them
    ([2], [37000], 8, 1), ([70, 3, 500], [9000, 20000, 700], 4, 1)])   # items cut between CTAs
def test_cross_out_at_every_multiple_of_16_bytes(new, lens, Hq, Hkv, kv, cuda_device):
    """`out` may begin anywhere that its 16-byte pieces allow: inside a buffer of other tensors,
    where it is a multiple of 16 bytes but not of 32.  The rest of the buffer stays."""
    dev = cuda_device
    q, k, v, bt, lens, cu = test_cross_gpu.make(new, lens, Hq, Hkv, 16, seed=len(new), kv=kv)
    a = [x.to(dev) for x in (q, k, v, bt, lens)]
    want, lse = pgqa.cross_attention(*a, cu_seqlens_q=cu.to(dev), return_lse=True)
    one = torch.ones(Hkv) if kv == "e4m3" else None
    test_cross_gpu.check(want, lse, test_cross_gpu.reference(q, k, v, bt, lens, cu, 1 / math.sqrt(128), dev, one, one))
    n = q.numel()
    for first in (8, 16, 24, 32, 40):
        flat = torch.full((n + 64,), 7.0, dtype=torch.bfloat16, device=dev)
        out = flat[first:first + n].view(q.shape)
        assert out.data_ptr() % 32 == (16 if first % 16 else 0)
        assert pgqa.cross_attention(*a, cu_seqlens_q=cu.to(dev), out=out) is out
        assert torch.equal(out, want)
        assert (flat[:first] == 7).all() and (flat[first + n:] == 7).all()
    pgqa.check_device_error()
