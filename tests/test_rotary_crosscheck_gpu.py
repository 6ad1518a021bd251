"""The rotary arguments of flash_attn_with_kvcache against flash-attn itself, where that library
runs on this GPU (it is called, never inspected).  Its paged mode wants pages of 256 tokens."""
import pytest
import torch

import mx_flash_attn_kernel_opt__b200 as pgqa
from tests import _paged
from tests.test_parity_gpu import ATOL, RTOL
from tests.test_rope_gpu import tables

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("Sq,S,causal,interleaved,R", [(1, 1, False, True, 128), (4, 4, True, False, 128),
                                                       (4, 4, False, False, 64), (3, 3, True, True, 32)])
def test_matches_flash_attn(Sq, S, causal, interleaved, R, cuda_device):
    try:
        from flash_attn import flash_attn_with_kvcache as fa
    except Exception as e:  # pragma: no cover - depends on the image
        pytest.skip(f"flash_attn unavailable: {e}")
    g = torch.Generator().manual_seed(R + Sq)
    lens, Hq, Hkv, P = [0, 7, 255, 600], 16, 4, 256
    bt, pages = _paged.table([n + S for n in lens], P, g)
    bt[bt == 2 ** 30] = 0
    dev = cuda_device
    k, v = (_paged.pool(pages, P, Hkv, g).to(dev) for _ in range(2))
    q = torch.randn(len(lens), Sq, Hq, 128, generator=g).to(torch.bfloat16).to(dev)
    kn, vn = (torch.randn(len(lens), S, Hkv, 128, generator=g).to(torch.bfloat16).to(dev) for _ in range(2))
    cos, sin = (x.to(dev) for x in tables(1024, R, torch.bfloat16))
    args = dict(rotary_cos=cos, rotary_sin=sin, cache_seqlens=torch.tensor(lens, dtype=torch.int32, device=dev),
                block_table=bt.to(dev), causal=causal, rotary_interleaved=interleaved)
    kf, vf = k.clone(), v.clone()
    try:
        ref = fa(q, kf, vf, k=kn, v=vn, **args)
        torch.cuda.synchronize()
    except RuntimeError as e:  # no kernel image for this GPU
        pytest.skip(f"flash_attn_with_kvcache did not run here: {e}")
    out = pgqa.flash_attn_with_kvcache(q, k, v, k=kn, v=vn, **args)
    torch.cuda.synchronize()
    assert torch.equal(v, vf)
    # each side rounds the turned keys once
    assert ((k.float() - kf.float()).abs() <= 2.0 ** -7 * kf.float().abs() + 1e-6).all()
    assert torch.allclose(out.float(), ref.float(), atol=ATOL, rtol=RTOL)
