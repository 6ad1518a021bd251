"""Calls at the edges of what the operators around the decode take."""
import math

import pytest
import torch

import mx_flash_attn_kernel_opt__b200 as pgqa
from mx_flash_attn_kernel_opt__b200 import PgqaError
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


@pytest.mark.parametrize("kv", ["bf16", "e4m3"])
@pytest.mark.parametrize("new,lens", [([5, 3], [800, 600]), ([40] + [0] * 70, [300] * 71), ([0] * 33 + [9], [64] * 34),
                                      ([600, 900], [3000, 1111])])
def test_cross_slice_longer_than_its_items_ends(new, lens, kv, cuda_device, monkeypatch):
    """Every role's walk over the items ends behind the last sequence, whatever the length of
    the slice that it was given: the call reports it, and its outputs and the next call are right."""
    q, k, v, bt, lens, cu = test_cross_gpu.make(new, lens, 8, 2, 16, seed=60, kv=kv)
    a = [x.to(cuda_device) for x in (q, k, v, bt, lens)]
    cu = cu.to(cuda_device)
    want = pgqa.cross_attention(*a, cu_seqlens_q=cu)
    pgqa.check_device_error()
    monkeypatch.setenv("PGQA_DEBUG_LONG_SLICE", "1")
    monkeypatch.setenv("PGQA_WAIT_LIMIT_NS", "3000000")
    out = pgqa.cross_attention(*a, cu_seqlens_q=cu)
    with pytest.raises(PgqaError) as e:
        pgqa.check_device_error()
    assert e.value.status == 10
    assert torch.equal(out, want)
    monkeypatch.delenv("PGQA_DEBUG_LONG_SLICE")
    monkeypatch.delenv("PGQA_WAIT_LIMIT_NS")
    assert torch.equal(pgqa.cross_attention(*a, cu_seqlens_q=cu), want)
    pgqa.check_device_error()
