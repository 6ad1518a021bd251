"""evict_kv: indices, moved rows and moved weights equal the restatement's exactly."""
import pytest
import torch

import mx_flash_attn_kernel_opt__b200 as pgqa
from mx_flash_attn_kernel_opt__b200 import PgqaError
from oracle import evict_ref
from tests import _paged

pytestmark = pytest.mark.gpu


def make(lens, Hkv, P, kv="bf16", seed=0, ties=True):
    g = torch.Generator().manual_seed(seed)
    bt, pages = _paged.table(lens, P, g)
    k, v = (_paged.pool(pages, P, Hkv, g, kv) for _ in range(2))
    w = torch.randn(pages, Hkv, P, generator=g).exp()
    if ties:  # many equal weights, zeros of both signs among them
        w = torch.where(torch.rand(w.shape, generator=g) < 0.5, (w * 2).round() / 2, w)
        w = torch.where(torch.rand(w.shape, generator=g) < 0.1, -0.0, w)
    return k, v, w, bt, torch.tensor(lens, dtype=torch.int32)


def run_and_check(case, keep, sinks, recent, dev, apart=False):
    k, v, w, bt, lens = case
    out = torch.full_like(w, 5.0) if apart else None
    ref = evict_ref(k, v, w, bt, lens, keep, sinks, recent, out)
    kd, vd, wd = k.to(dev), v.to(dev), w.to(dev)
    od = out.to(dev) if apart else None
    kept, new = pgqa.evict_kv(kd, vd, wd, bt.to(dev), lens.to(dev), keep, sinks=sinks, recent=recent,
                              weights_out=od)
    pgqa.check_device_error()
    assert torch.equal(new.cpu(), ref[1])
    assert torch.equal(kept.cpu(), ref[0])
    for got, want in ((kd, ref[2]), (vd, ref[3]), (od if apart else wd, ref[4])):
        assert torch.equal(_paged.raw(got), _paged.raw(want))
    if apart:
        assert torch.equal(_paged.raw(wd), _paged.raw(w))


@pytest.mark.parametrize("kv", ["bf16", "e4m3"])
@pytest.mark.parametrize("P,Hkv", [(16, 8), (64, 3), (48, 1)])
@pytest.mark.parametrize("keep,sinks,recent", [(32, 4, 8), (1, 0, 0), (1, 1, 0), (1, 0, 1), (40, 0, 40),
                                               (17, 17, 0), (33, 16, 17), (50, 0, 0), (63, 1, 5)])
def test_matches_the_restatement(kv, P, Hkv, keep, sinks, recent, cuda_device):
    run_and_check(make([0, 1, keep, keep + 1, 64, 150], Hkv, P, kv, seed=keep + P), keep, sinks, recent,
                  cuda_device, apart=keep % 2 == 0)


@pytest.mark.parametrize("L,keep", [(5000, 4999), (5000, 700), (9000, 4500), (4097, 4096)])
def test_long_sequences(L, keep, cuda_device):
    run_and_check(make([L, 10], 2, 16, seed=L), keep, 4, min(64, keep // 2), cuda_device)


def test_pairs_cut_by_clusters_and_pairs_left_alone(cuda_device):
    """Few pairs with a large capacity: several CTAs select for one pair, some of them without
    a candidate, and short sequences beside long ones."""
    run_and_check(make([20000, 3, 8000, 1025], 1, 32, seed=20), 1024, 4, 300, cuda_device)
    run_and_check(make([17000], 1, 16, "e4m3", seed=21), 16000, 0, 1, cuda_device)
    k, v, w, bt, lens = make([33000, 40], 1, 16, seed=22)
    w[:] = 1.0  # ties across the CTAs
    run_and_check((k, v, w, bt, lens), 20000, 1, 2, cuda_device)
    run_and_check((k, v, w, bt, lens), 37, 30, 7, cuda_device)


def test_more_kept_than_places_looked_up_at_a_time(cuda_device):
    """More than 2048 kept rows, by a pair of CTAs and by more, in place and apart."""
    for pairs, P in ((90, 16), (1, 64)):
        case = make([5300] + [0] * (pairs - 1), 4 if pairs > 1 else 1, P, "e4m3", seed=30 + pairs)
        run_and_check(case, 5000, 7, 100, cuda_device)
        run_and_check(case, 2600, 0, 2600, cuda_device, apart=True)


def test_longer_than_shared_memory_holds(cuda_device):
    """More candidates than the select keeps in shared memory: keys are re-read."""
    g = torch.Generator().manual_seed(1)
    L, keep = 60000, 300
    case = list(make([L], 1, 256, seed=2))
    case[2] = torch.randn(case[2].shape, generator=g).exp()
    run_and_check(tuple(case), keep, 4, 100, cuda_device)


def test_equal_weights_keep_the_lowest_indices(cuda_device):
    for fill in (0.0, 1.0, -0.0, float("inf"), float("-inf")):
        k, v, w, bt, lens = make([3000], 1, 16, seed=3)
        w[:] = fill
        run_and_check((k, v, w, bt, lens), 1000, 3, 5, cuda_device)


def test_nan_and_infinite_weights(cuda_device):
    k, v, w, bt, lens = make([200, 90], 2, 16, seed=4)
    g = torch.Generator().manual_seed(5)
    for val, share in ((float("nan"), 0.05), (float("inf"), 0.05), (float("-inf"), 0.2)):
        w = torch.where(torch.rand(w.shape, generator=g) < share, val, w)
    run_and_check((k, v, w, bt, lens), 40, 2, 3, cuda_device)


def test_negative_and_tiny_weights(cuda_device):
    k, v, w, bt, lens = make([500], 2, 16, seed=6, ties=False)
    g = torch.Generator().manual_seed(7)
    w = torch.randn(w.shape, generator=g) * 1e-42  # subnormal, both signs
    run_and_check((k, v, w, bt, lens), 100, 0, 0, cuda_device)


def test_many_pairs_and_few(cuda_device):
    run_and_check(make([70] * 60, 8, 16, seed=8), 64, 4, 16, cuda_device)   # one column range
    run_and_check(make([70], 1, 16, seed=9), 64, 4, 16, cuda_device)        # most column ranges
    run_and_check(make([70], 1, 16, "e4m3", seed=9), 64, 4, 16, cuda_device)


def test_cut_again_and_again(cuda_device):
    """A cache held at its budget: append one token, evict one, many times over."""
    dev = cuda_device
    L, keep, steps = 33, 32, 12
    k, v, w, bt, _ = make([L, L], 2, 16, seed=10)
    kd, vd, wd, btd = (x.to(dev) for x in (k, v, w, bt))
    lens = torch.tensor([L, L], dtype=torch.int32)
    g = torch.Generator().manual_seed(11)
    for _ in range(steps):
        _, _, k, v, w = evict_ref(k, v, w, bt, lens, keep, 2, 8)
        _, new = pgqa.evict_kv(kd, vd, wd, btd, lens.to(dev), keep, sinks=2, recent=8)
        assert new.tolist() == [keep, keep]
        row = torch.randn(2, 2, 128, generator=g).to(torch.bfloat16)
        for b in range(2):
            pg, sl = int(bt[b, keep // 16]), keep % 16
            for x, xd in ((k, kd), (v, vd)):
                x[pg, sl] = row[b]
                xd[pg, sl] = row[b].to(dev)
            val = torch.rand(2, generator=g)
            w[pg, :, sl] = val
            wd[pg, :, sl] = val.to(dev)
    assert torch.equal(_paged.raw(kd), _paged.raw(k)) and torch.equal(_paged.raw(vd), _paged.raw(v))
    assert torch.equal(wd.cpu(), w)


def test_graph_and_other_stream(cuda_device):
    dev = cuda_device
    case = make([100, 40, 64], 2, 16, seed=12)
    ref = evict_ref(*case, 48, 4, 8)
    k, v, w, bt, lens = (x.to(dev) for x in case)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        kept, new = pgqa.evict_kv(k, v, w, bt, lens, 48, sinks=4, recent=8)
    s.synchronize()
    assert torch.equal(kept.cpu(), ref[0]) and torch.equal(_paged.raw(k), _paged.raw(ref[2]))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        kept, new = pgqa.evict_kv(k, v, w, bt, lens, 48, sinks=4, recent=8)
    for x, y in zip((k, v, w), case):
        x.copy_(y)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(kept.cpu(), ref[0]) and torch.equal(new.cpu(), ref[1])
    for got, want in ((k, ref[2]), (v, ref[3]), (w, ref[4])):
        assert torch.equal(_paged.raw(got), _paged.raw(want))


def test_bad_pages_and_lengths_are_reported(cuda_device):
    dev = cuda_device
    for what, status in (("page", 9), ("len", 10), ("neg", 10)):
        k, v, w, bt, lens = make([60, 60], 2, 16, seed=13)
        if what == "page":
            bt[1, 2] = 10 ** 6
        elif what == "len":
            bt[bt == 2 ** 30] = 0
            lens[1] = 16 * bt.shape[1] + 7
        else:
            lens[1] = -5
        _, new = pgqa.evict_kv(k.to(dev), v.to(dev), w.to(dev), bt.to(dev), lens.to(dev), 20)
        with pytest.raises(PgqaError) as e:
            pgqa.check_device_error()
        assert e.value.status == status, what
        assert new.tolist() == ([20, 0] if what == "neg" else [20, 20])
