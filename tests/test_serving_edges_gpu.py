"""Calls at the edges of what the operators around the decode take."""
import math
import os
import subprocess
import sys

import pytest
import torch

import mx_flash_attn_kernel_opt__b200 as pgqa
from mx_flash_attn_kernel_opt__b200 import PgqaError
from tests import _paged, test_cross_gpu, test_evict_gpu, test_rope_gpu, test_weights_gpu

pytestmark = pytest.mark.gpu

REPO = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

ONE_BATCH = """
import sys, torch
import mx_flash_attn_kernel_opt__b200 as pgqa
B, Sq = int(sys.argv[1]), int(sys.argv[2])
z = lambda *s, dtype=torch.float32: torch.zeros(*s, dtype=dtype, device="cuda")
lens = z(B, dtype=torch.int32)
lens[-1] = 5
w = z(1, 1, 16)
q, k = z(B, Sq, 1, 128, dtype=torch.bfloat16), z(1, 16, 1, 128, dtype=torch.bfloat16)
pgqa.accumulate_weights(q, k, z(B, 1, dtype=torch.int32), lens, z(B, 1, Sq), w)
pgqa.check_device_error()
# scores of 0 and a log-sum-exp of 0: each row adds exp(0)
assert torch.equal(w.flatten().cpu(), torch.tensor([float(Sq)] * 5 + [0.0] * 11)), w
"""


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
    monkeypatch.setenv("PGQA_DEBUG_STUCK_BARRIER", "-1")
    monkeypatch.setenv("PGQA_WAIT_LIMIT_NS", "3000000")
    out = pgqa.cross_attention(*a, cu_seqlens_q=cu)
    with pytest.raises(PgqaError) as e:
        pgqa.check_device_error()
    assert e.value.status == 10
    assert torch.equal(out, want)
    monkeypatch.delenv("PGQA_DEBUG_STUCK_BARRIER")
    monkeypatch.delenv("PGQA_WAIT_LIMIT_NS")
    assert torch.equal(pgqa.cross_attention(*a, cu_seqlens_q=cu), want)
    pgqa.check_device_error()


@pytest.mark.parametrize("Sq", [1, 5])
def test_chains_without_a_stop_between_the_calls(Sq, both_kernels, cuda_device):
    """rope -> decode -> weights -> evict -> decode and append at the lengths that the eviction
    wrote, step after step: calls queued without a wait equal calls that wait for each other."""
    dev, P, Hq, Hkv, B, keep = cuda_device, 16, 32, 4, 6, 900
    g = torch.Generator().manual_seed(70)
    cap = 1024
    bt, pages = _paged.table([cap] * B, P, g)
    k, v = (_paged.pool(pages, P, Hkv, g) for _ in range(2))
    cos, sin = (x.to(dev) for x in test_rope_gpu.tables(2048, 128))
    bt = bt.to(dev)
    xs = [torch.randn(B, Sq, Hq + 2 * Hkv, 128, generator=g).to(torch.bfloat16).to(dev) for _ in range(6)]
    first = torch.tensor([880, 10, 899, 0, 600, 890], dtype=torch.int32, device=dev)
    more = torch.randn(2, B, 3, Hkv, 128, generator=g).to(torch.bfloat16).to(dev)

    def run(wait):
        stop = torch.cuda.synchronize if wait else (lambda: None)
        kd, vd, w, lens, got = k.to(dev), v.to(dev), torch.zeros(pages, Hkv, P, device=dev), first.clone(), []
        torch.cuda.synchronize()
        for x in xs:
            q = pgqa.rope_append_kv(x[:, :, :Hq], x[:, :, Hq:Hq + Hkv], x[:, :, Hq + Hkv:], kd, vd, bt, lens, cos, sin,
                                    weights=w)
            stop()
            full = lens + Sq
            out, lse = pgqa.decode(q, kd, vd, bt, full, causal=True, return_lse=True)
            stop()
            pgqa.accumulate_weights(q, kd, bt, full, lse, w, causal=True)
            stop()
            kept, lens = pgqa.evict_kv(kd, vd, w, bt, full, keep, sinks=4, recent=64)
            stop()
            again = pgqa.decode(q, kd, vd, bt, lens, causal=True)
            stop()
            pgqa.append_kv(more[0], more[1], kd, vd, bt, lens)
            stop()
            got += [q, out, lse, kept, lens, again]
        torch.cuda.synchronize()
        return got + [kd, vd, w]

    want = run(True)
    for _ in range(4):
        for a, b in zip(run(False), want):
            assert torch.equal(a, b)
    pgqa.check_device_error()


@pytest.mark.parametrize("B,Sq", [(12279, 1), (12284, 1), (12287, 8), (3575, 16), (3580, 16), (3583, 9)])
def test_weights_of_a_batch_whose_table_ends_near_48_kb(B, Sq, cuda_device):
    """The kernel's shared memory, its few static bytes included, lies around the size up to
    which a launch needs no raised limit.  In a fresh process: no larger call has raised it."""
    r = subprocess.run([sys.executable, "-c", ONE_BATCH, str(B), str(Sq)], cwd=REPO, capture_output=True, text=True,
                       timeout=300)
    assert r.returncode == 0, r.stderr[-2000:]


TWO_THREADS = """
import threading, torch
import mx_flash_attn_kernel_opt__b200 as pgqa
torch.cuda.init()
z = lambda *s, dtype=torch.float32: torch.zeros(*s, dtype=dtype, device="cuda")
bad = []
def calls(B):
    try:
        k, w = z(1, 16, 1, 128, dtype=torch.bfloat16), z(1, 1, 16)
        a = (z(B, 1, 128, dtype=torch.bfloat16), k, z(B, 1, dtype=torch.int32), z(B, dtype=torch.int32), z(B, 1, 1), w)
        go.wait()
        for _ in range(50):
            pgqa.accumulate_weights(*a)
    except Exception as e:
        bad.append((B, repr(e)))
go = threading.Barrier(4)
ts = [threading.Thread(target=calls, args=(B,)) for B in (13000, 28000, 100, 20000)]
[t.start() for t in ts]
[t.join() for t in ts]
pgqa.check_device_error()
assert not bad, bad
"""


def test_weights_of_small_and_large_batches_from_several_threads(cuda_device):
    for _ in range(3):
        r = subprocess.run([sys.executable, "-c", TWO_THREADS], cwd=REPO, capture_output=True, text=True, timeout=300)
        assert r.returncode == 0, r.stderr[-2000:]


def test_one_check_clears_the_errors_of_every_entry_point(cuda_device):
    """A decode in the library's own workspace and a rotary append both go wrong: one check
    reports, and the next one finds nothing."""
    c = test_rope_gpu.Case([5, 20], [2, 2], seed=1, rows=64).to(cuda_device)
    c.d["pos"][0, 3] = 64
    c.call()
    z = lambda *s, dtype=torch.bfloat16: torch.zeros(*s, dtype=dtype, device=cuda_device)  # noqa: E731
    k, bt = z(2, 16, 2, 128), torch.tensor([[0], [1]], dtype=torch.int32, device=cuda_device)
    lens = torch.tensor([3, 17], dtype=torch.int32, device=cuda_device)      # 17 tokens in one page of 16
    pgqa.run_kernel_cabi(z(2, 8, 128), k, k, z(2, 8, 128), lens, bt, 2, 16, 1, 8, 2, 128, 16, 2, 0)
    torch.cuda.synchronize()
    with pytest.raises(PgqaError) as e:
        pgqa.check_device_error()
    assert e.value.status in (10, 12)
    pgqa.check_device_error()


def odd_strides(x):
    """The same elements with strides of 7 for every dimension of size 1."""
    return x.as_strided(x.shape, [7 if n == 1 else s for n, s in zip(x.shape, x.stride())])


@pytest.mark.parametrize("lens,new,Hq,Hkv,packed", [
    ([5], [3], 8, 2, False), ([5, 9, 2], [1, 1, 1], 8, 2, False), ([4], [1], 1, 1, False), ([3], [4], 1, 1, False),
    ([7], [1], 4, 1, True)])
def test_strides_of_dimensions_of_size_one(lens, new, Hq, Hkv, packed, cuda_device):
    """torch gives such a dimension any stride, and no address depends on it."""
    c = test_rope_gpu.Case(lens, new, Hq=Hq, Hkv=Hkv, packed=packed, seed=len(lens) + Hq).to(cuda_device)
    x = c.d["qkv"]
    cu = None
    pos = c.d["pos"]
    q, k, v = c.split(x)
    if packed:
        cu = torch.tensor([0, sum(new)], dtype=torch.int32, device=cuda_device)
    else:
        q, k, v = (t.unflatten(0, (len(new), new[0])) for t in (q, k, v))
        pos = pos.unflatten(1, (len(new), new[0]))
    q, k, v = (odd_strides(t) for t in (q, k, v))
    out = pgqa.rope_append_kv(q, k, v, c.d["kc"], c.d["vc"], c.d["bt"], c.d["lens"], c.d["cos"], c.d["sin"],
                              positions=pos, axes=c.axes, cu_seqlens=cu, weights=c.d["w"])
    pgqa.check_device_error()
    c.check(out)


def test_empty_batches(cuda_device):
    """A step in which no sequence is left: every operator returns outputs of no rows."""
    z = lambda *s, dtype=torch.float32: torch.zeros(*s, dtype=dtype, device=cuda_device)  # noqa: E731
    bf, i32 = torch.bfloat16, torch.int32
    k, v = z(4, 16, 2, 128, dtype=bf), z(4, 16, 2, 128, dtype=bf)
    w, bt, lens, t = z(4, 2, 16) + 3, z(0, 2, dtype=i32), z(0, dtype=i32), z(8, 64)
    q, kn = z(0, 8, 128, dtype=bf), z(0, 2, 128, dtype=bf)
    assert pgqa.rope_append_kv(q, kn, kn, k, v, bt, lens, t, t, weights=w).shape == (0, 8, 128)
    assert pgqa.accumulate_weights(q, k, bt, lens, z(0, 8, 1), w) is w
    kept, new = pgqa.evict_kv(k, v, w, bt, lens, 5)
    assert kept.shape == (0, 2, 5) and kept.dtype == i32 and new.shape == (0,) and new.dtype == i32
    assert pgqa.cross_attention(z(0, 3, 8, 128, dtype=bf), k, v, bt, lens).shape == (0, 3, 8, 128)
    assert (w == 3).all()
    with pytest.raises(PgqaError):
        pgqa.evict_kv(k, v, w, bt, lens, 0)
    with pytest.raises(PgqaError):
        pgqa.accumulate_weights(q, k, bt, lens, z(0, 7, 1), w)
    pgqa.check_device_error()


@pytest.mark.parametrize("Hq,Sq", [(8, 1), (8, 5)])
@pytest.mark.parametrize("up", [2.0 ** 118, 2.0 ** -116])
def test_weights_of_very_large_and_very_small_queries(up, Hq, Sq, cuda_device):
    """q times 2^n and the scale of K times 2^-n: the same scores, so the same weights and bounds."""
    q, k, bt, lens, lse, w, scale, ks = test_weights_gpu.make([33, 7], Hq, 2, 16, Sq, "e4m3", seed=50 + Sq)
    big = (q.float() * up).to(torch.bfloat16)
    assert big.isfinite().all() and (up < 1 or torch.equal(big.float() / up, q.float()))
    test_weights_gpu.run_and_check((big, k, bt, lens, lse, w, scale, ks / up), False, cuda_device)


@pytest.mark.parametrize("Hq,Sq", [(8, 1), (8, 5)])
def test_weights_of_queries_with_elements_far_below_the_largest(Hq, Sq, cuda_device):
    """Each row's elements span 2^40: those far below the largest keep fewer bits in f16.  What
    that may move a score, 2^-25 of the scaled row against 2^14 at the least, 2^-39 of the largest
    element for each product, is far inside the bound, which counts 2^-16 of the products' sum."""
    q, k, bt, lens, lse, w, scale, ks = test_weights_gpu.make([33, 7], Hq, 2, 16, Sq, "e4m3", seed=60 + Sq)
    g = torch.Generator().manual_seed(61)
    small = (q.float() * 2.0 ** -torch.randint(0, 41, q.shape, generator=g).float()).to(torch.bfloat16)
    test_weights_gpu.run_and_check((small, k, bt, lens, lse, w, scale, ks), False, cuda_device)


@pytest.mark.parametrize("interleaved,table", [(False, "fp32"), (True, "bf16")])
def test_packed_prompts_into_e4m3_pages(interleaved, table, cuda_device):
    c = test_rope_gpu.Case([0, 7, 31, 2], [5, 0, 40, 1], R=64, kv="e4m3", axes="turn", packed=True,
                           interleaved=interleaved, table=table, seed=80).to(cuda_device)
    c.check(c.call())
    pgqa.check_device_error()


def evict_cluster(pairs, capacity):
    """CTAs per (sequence, KV head), by the rule in csrc/pgqa_evict.cu."""
    places, n = 2 * torch.cuda.get_device_properties(0).multi_processor_count, 2
    while n < 8 and pairs * 2 * n <= places and capacity // (2 * n) >= 1024:
        n *= 2
    return n


@pytest.mark.parametrize("lens,Hkv,keep,sinks,recent,cluster", [
    ([4200, 4100, 60, 0, 30], 8, 1500, 4, 64, 4), ([4097, 4096], 1, 4095, 0, 0, 4), ([2300] * 2, 2, 700, 1, 2, 2),
    ([9000, 100], 2, 2100, 0, 300, 8)])
@pytest.mark.parametrize("kv,apart", [("bf16", False), ("e4m3", True)])
def test_evict_in_clusters_of_each_size(lens, Hkv, keep, sinks, recent, cluster, kv, apart, cuda_device):
    case = test_evict_gpu.make(lens, Hkv, 16, kv, seed=90 + cluster)
    assert evict_cluster(len(lens) * Hkv, 16 * case[3].shape[1]) == cluster
    test_evict_gpu.run_and_check(case, keep, sinks, recent, cuda_device, apart=apart)


@pytest.mark.parametrize("kv", ["bf16", "e4m3"])
def test_pools_of_more_than_2_31_elements(kv, cuda_device):
    """The same calls on the last pages of a large pool and on a small one: equal results, and
    no byte of the large pool changes anywhere else."""
    dev, P, Hq, Hkv, S = cuda_device, 16, 16, 8, 3
    g = torch.Generator().manual_seed(100)
    lens = [70, 1, 200]
    bt, pages = _paged.table([n + S for n in lens], P, g)
    more = 140000                       # pages of 16 x 8 x 128 elements
    assert more * P * Hkv * 128 > 2 ** 31
    k, v = (_paged.pool(pages, P, Hkv, g, kv) for _ in range(2))
    w0 = torch.rand(pages, Hkv, P, generator=g) * 0.01
    cos, sin = (x.to(dev) for x in test_rope_gpu.tables(512, 128))
    x = torch.randn(len(lens), S, Hq + 2 * Hkv, 128, generator=g).to(torch.bfloat16).to(dev)
    before = torch.tensor(lens, dtype=torch.int32, device=dev)
    after = before + S
    scale = dict(k_scale=0.7, v_scale=0.9) if kv == "e4m3" else {}
    ks = {n: s for n, s in scale.items() if n == "k_scale"}

    def run(kd, vd, w, table):
        q = pgqa.rope_append_kv(x[:, :, :Hq], x[:, :, Hq:Hq + Hkv], x[:, :, Hq + Hkv:], kd, vd, table, before, cos,
                                sin, weights=w, **scale)
        out, lse = pgqa.cross_attention(q, kd, vd, table, after, return_lse=True, **scale)
        pgqa.accumulate_weights(q, kd, table, after, lse, w, **ks)
        kept, new = pgqa.evict_kv(kd, vd, w, table, after, 50, sinks=2, recent=5)
        pgqa.check_device_error()
        return q, out, lse, kept, new

    small = [t.to(dev) for t in (k, v, w0)]
    want = run(*small, bt.to(dev))
    large = []
    for t in (k, v, w0):
        big = torch.zeros(more + pages, *t.shape[1:], dtype=t.dtype, device=dev)
        big.view(torch.uint8)[more:] = t.view(torch.uint8).to(dev)
        large.append(big)
    used = bt != 2 ** 30
    got = run(*large, torch.where(used, bt + more, bt).to(dev))
    for a, b in zip(got, want):
        assert torch.equal(a, b)
    for a, b in zip(large, small):
        assert torch.equal(_paged.raw(a[more:]), _paged.raw(b))
        assert not a[:more].view(torch.uint8).any()


def test_refused_rotary_calls_leave_the_cache(cuda_device):
    """flash_attn_with_kvcache with rotary inputs: whatever it refuses, it refuses before the new
    tokens enter the cache, as it does without them."""
    dev = cuda_device
    g = torch.Generator().manual_seed(110)
    B, S, Hq, Hkv, P = 2, 3, 8, 2, 16
    bt, pages = _paged.table([20 + S, 5 + S], P, g)
    k, v = (_paged.pool(pages, P, Hkv, g).to(dev) for _ in range(2))
    before = _paged.raw(k), _paged.raw(v)
    cos, sin = (x.to(dev) for x in test_rope_gpu.tables(64, 128))
    bt, lens = bt.to(dev), torch.tensor([20, 5], dtype=torch.int32, device=dev)
    z = lambda *s: torch.randn(*s, generator=g).to(torch.bfloat16).to(dev)  # noqa: E731
    q, kn = z(B, S, Hq, 128), z(B, S, Hkv, 128)
    for error, kw in (
            (PgqaError, dict(k=z(B, Hkv, 128), v=z(B, Hkv, 128))),              # no dimension of tokens
            (PgqaError, dict(k=z(B, Hkv, 128), v=z(B, Hkv, 128), causal=True)),
            (TypeError, dict(q=z(B, 5, Hq, 128).half())), (TypeError, dict(q=z(B, S, Hq, 128).half(), causal=True)),
            (PgqaError, dict(q=z(B, S, 7, 128))), (PgqaError, dict(q=z(B, 5, 7, 128))),
            (PgqaError, dict(q=z(3, 5, Hq, 128))), (PgqaError, dict(softmax_scale=0.0)),
            (PgqaError, dict(softmax_scale=float("nan"), causal=True)), (PgqaError, dict(softmax_scale=-1.0, q=z(B, 1, Hq, 128)))):
        a = dict(q=q, k=kn, v=kn, rotary_cos=cos, rotary_sin=sin, cache_seqlens=lens, block_table=bt)
        a.update(kw)
        with pytest.raises(error):
            pgqa.flash_attn_with_kvcache(a.pop("q"), k, v, **a)
        torch.cuda.synchronize()
        assert torch.equal(_paged.raw(k), before[0]) and torch.equal(_paged.raw(v), before[1]), kw
    pgqa.check_device_error()
    # and what it takes still enters
    pgqa.flash_attn_with_kvcache(q, k, v, k=kn, v=kn, rotary_cos=cos, rotary_sin=sin, cache_seqlens=lens, block_table=bt)
    assert not torch.equal(_paged.raw(k), before[0]) and not torch.equal(_paged.raw(v), before[1])
    pgqa.check_device_error()
