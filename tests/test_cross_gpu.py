"""cross_attention against a plain 64-bit computation.

Bounds: each weight is rounded to bf16 (2^-8 relative at most) and weighted sums are
rounded to bf16 once more (2^-8); fp32 scores are within d = scale * sum|q k| * 128 * 2^-23 (a
sum of 128 exact products, even if truncated), which moves a weight and the normaliser by
d relative each.  For rows of random values the roundings of the weights are independent, so
the error's norm stays below 2^-8 of the result's for each of the two."""
import math

import pytest
import torch

import mx_flash_attn_kernel_opt__b200 as pgqa
from mx_flash_attn_kernel_opt__b200 import PgqaError
from tests import _paged

pytestmark = pytest.mark.gpu


def make(new, lens, Hq, Hkv, P, seed=0, std=1.0, kv="bf16"):
    g = torch.Generator().manual_seed(seed)
    bt, pages = _paged.table(lens, P, g)
    k, v = (_paged.poison_unused(_paged.pool(pages, P, Hkv, g, kv, std), lens, bt, P) for _ in range(2))
    q = torch.randn(sum(new), Hq, 128, generator=g).to(torch.bfloat16)
    return q, k, v, bt, torch.tensor(lens, dtype=torch.int32), \
        torch.tensor([sum(new[:b]) for b in range(len(new) + 1)], dtype=torch.int32)


def reference(q, k, v, bt, lens, cu, scale, dev, ks=None, vs=None):
    """64 bits, on the device: out, lse [Hq, T], sum of |weight * v|, score bound."""
    T, Hq, _ = q.shape
    Hkv, P = k.shape[2], k.shape[1]
    out = torch.zeros(T, Hq, 128, dtype=torch.float64, device=dev)
    mag = torch.zeros_like(out)
    lse = torch.full((Hq, T), -math.inf, dtype=torch.float64, device=dev)
    d = torch.zeros(Hq, T, dtype=torch.float64, device=dev)
    kd, vd, qd = k.to(dev).float(), v.to(dev).float(), q.to(dev).double()
    if ks is not None:
        kd = kd.double() * ks.to(dev).double().view(1, 1, Hkv, 1)
        vd = vd.double() * vs.to(dev).double().view(1, 1, Hkv, 1)
    for b, L in enumerate(lens.tolist()):
        x0, x1 = int(cu[b]), int(cu[b + 1])
        if not L or x0 == x1:
            continue
        t = torch.arange(L)
        pg, sl = bt[b, t // P].long().to(dev), (t % P).to(dev)
        K, V = kd[pg, sl].double().repeat_interleave(Hq // Hkv, 1), vd[pg, sl].double().repeat_interleave(Hq // Hkv, 1)
        x = torch.einsum("xhd,thd->hxt", qd[x0:x1], K) * scale
        p = torch.softmax(x, -1)
        out[x0:x1] = torch.einsum("hxt,thd->xhd", p, V)
        mag[x0:x1] = torch.einsum("hxt,thd->xhd", p, V.abs())
        lse[:, x0:x1] = torch.logsumexp(x, -1)
        d[:, x0:x1] = torch.einsum("xhd,thd->hxt", qd[x0:x1].abs(), K.abs()).amax(-1) * scale * 128 * 2.0 ** -23
    return out, lse, mag, d


def check(out, lse, ref, random_rows=True):
    want, wl, mag, d = ref
    got = out.double()
    dd = d.t().unsqueeze(-1)
    tol = 2.0 ** -8 * want.abs() + (2.0 ** -8 + 2 * dd + 2.0 ** -20) * mag * (1 + 2.0 ** -7)
    over = (got - want).abs() - tol
    assert not over.isnan().any() and (over <= 0).all(), f"over the bound by {over.max().item():.3e}"
    if random_rows and want.numel():
        assert (got - want).norm() <= 2.0 ** -7 * want.norm()
    if lse is not None:
        fin = wl > -math.inf
        assert torch.equal(lse > -math.inf, fin)
        err = (lse.double()[fin] - wl[fin]).abs()
        assert (err <= d[fin] + 2.0 ** -20 + wl[fin].abs() * 2.0 ** -22).all()


def run_and_check(case, dev, scale=None, **kw):
    q, k, v, bt, lens, cu = case
    out, lse = pgqa.cross_attention(q.to(dev), k.to(dev), v.to(dev), bt.to(dev), lens.to(dev),
                                    cu_seqlens_q=cu.to(dev), scale=scale, return_lse=True)
    pgqa.check_device_error()
    check(out, lse, reference(q, k, v, bt, lens, cu, scale or 1 / math.sqrt(128), dev), **kw)
    return out, lse


@pytest.mark.parametrize("L", [0, 1, 15, 16, 17, 64, 100, 127, 128, 129, 256, 300])
def test_one_tile(L, cuda_device):
    run_and_check(make([32], [L], 4, 1, 16, seed=L), cuda_device)


@pytest.mark.parametrize("n", [1, 2, 31, 32, 33, 63, 64, 65, 130])
def test_numbers_of_query_tokens(n, cuda_device):
    run_and_check(make([n], [200], 8, 2, 16, seed=n), cuda_device)


@pytest.mark.parametrize("Hq,Hkv,P", [(32, 8, 16), (28, 4, 64), (16, 16, 48), (64, 1, 32), (6, 2, 256),
                                      (10, 2, 128), (128, 1, 16), (100, 1, 80)])
def test_ragged_batches(Hq, Hkv, P, cuda_device):
    run_and_check(make([40, 0, 1, 150, 7, 300, 0], [700, 30, 0, 129, 1300, 256, 5], Hq, Hkv, P, seed=Hq + P), cuda_device)


def test_many_sequences(cuda_device):
    g = torch.Generator().manual_seed(1)
    new = torch.randint(0, 9, (150,), generator=g).tolist()
    lens = torch.randint(0, 200, (150,), generator=g).tolist()
    run_and_check(make(new, lens, 8, 4, 16, seed=2), cuda_device)


def test_few_sequences_with_tokens_among_many(cuda_device):
    """Long runs of sequences without prompt tokens between those with some, and keys of 0."""
    new, lens = [0] * 333, [30 + i % 50 for i in range(333)]
    for at, n, L in ((0, 5, 100), (31, 3, 0), (32, 70, 300), (95, 1, 16), (96, 2, 129), (200, 40, 513), (332, 9, 77)):
        new[at], lens[at] = n, L
    run_and_check(make(new, lens, 8, 2, 16, seed=40), cuda_device)
    new[332] = 0
    run_and_check(make(new, lens, 4, 4, 16, seed=41), cuda_device)


def test_more_items_than_sms_and_long_keys(cuda_device):
    run_and_check(make([600, 900], [3000, 1111], 32, 8, 16, seed=3), cuda_device)


@pytest.mark.parametrize("lens", [[8192, 3000], [8192, 0], [513, 7000]])
def test_few_tokens_over_long_keys(lens, cuda_device):
    """Few items: the keys are cut into ranges and joined."""
    run_and_check(make([3, 9], lens, 8, 2, 16, seed=4), cuda_device)


@pytest.mark.parametrize("new,lens,Hq,Hkv", [
    ([1], [100000], 2, 1),                 # one item over every SM
    ([2], [37000], 8, 1), ([1, 1], [50000, 100], 4, 2), ([70, 3, 500], [9000, 20000, 700], 4, 1),
    ([33] * 40, [300 + 97 * i for i in range(40)], 8, 2), ([200], [18944], 4, 1), ([260, 5], [129, 40000], 6, 2)])
def test_items_cut_between_ctas(new, lens, Hq, Hkv, cuda_device):
    run_and_check(make(new, lens, Hq, Hkv, 16, seed=sum(lens)), cuda_device)


def test_growing_scores_move_the_maximum(cuda_device):
    """Keys that grow along the sequence: the running maximum moves in every tile."""
    case = list(make([100], [1500], 4, 1, 16, seed=5))
    q, k, v, bt, lens, cu = case
    for t in range(1500):
        k[bt[0, t // 16].long(), t % 16] *= 1 + t / 100
    run_and_check((q, k, v, bt, lens, cu), cuda_device, random_rows=False)
    run_and_check((q, k, v, bt, lens, cu), cuda_device, scale=1.7, random_rows=False)
    run_and_check((q * 0, k, v, bt, lens, cu), cuda_device)


def test_padded_form_and_strided_q(cuda_device):
    dev = cuda_device
    q, k, v, bt, lens, cu = make([50, 50, 50], [300, 5, 0], 8, 2, 16, seed=6)
    wide = torch.zeros(150, 20, 128, dtype=torch.bfloat16, device=dev)
    wide[:, 3:11] = q.to(dev)
    view = wide[:, 3:11]
    a = [x.to(dev) for x in (k, v, bt, lens)]
    out, lse = pgqa.cross_attention(view.unflatten(0, (3, 50)), *a, return_lse=True)
    packed, plse = pgqa.cross_attention(view, *a, cu_seqlens_q=cu.to(dev), return_lse=True)
    assert out.shape == (3, 50, 8, 128) and lse.shape == (3, 8, 50) and plse.shape == (8, 150)
    assert torch.equal(out.reshape(150, 8, 128), packed)
    assert torch.equal(lse.permute(1, 0, 2).reshape(8, 150), plse)
    check(packed, plse, reference(q, k, v, bt, lens, cu, 1 / math.sqrt(128), dev))
    one = pgqa.cross_attention(view[::50].unsqueeze(1), *a)
    first = pgqa.cross_attention(view[::50], *a, cu_seqlens_q=torch.arange(4, dtype=torch.int32, device=dev))
    assert torch.equal(one[:, 0], first)


def test_agrees_with_the_decode(cuda_device):
    """The decode's non-causal form on the same pages: within the two roundings of each."""
    dev = cuda_device
    q, k, v, bt, lens, cu = make([6, 6], [700, 90], 16, 4, 16, seed=7)
    a = [x.to(dev) for x in (k, v, bt, lens)]
    q4 = q.to(dev).unflatten(0, (2, 6))
    out, lse = pgqa.cross_attention(q4, *a, return_lse=True)
    dout, dlse = pgqa.decode(q4, *a, return_lse=True)
    ref = reference(q, k, v, bt, lens, cu, 1 / math.sqrt(128), dev)
    for o, l in ((out, lse), (dout, dlse)):
        check(o.reshape(12, 16, 128), l.permute(1, 0, 2).reshape(16, 12), ref)


def test_minus_infinity_and_nan_stay_in_their_rows(cuda_device):
    dev = cuda_device
    q, k, v, bt, lens, cu = make([40], [200], 2, 1, 16, seed=8)
    q[:, 0, 0] = q[:, 0, 0].abs() + 0.1
    q[:, 1, 0] = 0
    k[bt[0, 4].long(), 2, 0, 0] = -math.inf       # head 0: weight 0; head 1: 0 * inf
    out, lse = pgqa.cross_attention(q.to(dev), k.to(dev), v.to(dev), bt.to(dev), lens.to(dev),
                                    cu_seqlens_q=cu.to(dev), return_lse=True)
    assert out[:, 0].isfinite().all() and lse[0].isfinite().all()
    assert out[:, 1].isnan().all()
    q[5, 0, 3] = float("nan")
    out = pgqa.cross_attention(q.to(dev), k.to(dev), v.to(dev), bt.to(dev), lens.to(dev), cu_seqlens_q=cu.to(dev))
    assert out[5, 0].isnan().all() and out[6:, 0].isfinite().all() and out[:5, 0].isfinite().all()
    # every score of a row -inf: no weight anywhere
    k[..., 0] = -math.inf
    out, lse = pgqa.cross_attention(q[6:8].to(dev), k.to(dev), torch.nan_to_num(v).to(dev), bt.to(dev), lens.to(dev),
                                    cu_seqlens_q=torch.tensor([0, 2], dtype=torch.int32, device=dev), return_lse=True)
    assert (out[:, 0] == 0).all() and (lse[0] == -math.inf).all()


@pytest.mark.parametrize("L", [300, 8192])
def test_rows_behind_the_last_sequence_stay(L, cuda_device):
    dev = cuda_device
    q, k, v, bt, lens, _ = make([20], [L], 4, 1, 16, seed=9)
    out = torch.full(q.shape, 7.0, dtype=torch.bfloat16, device=dev)
    cu = torch.tensor([3, 12], dtype=torch.int32, device=dev)
    pgqa.cross_attention(q.to(dev), k.to(dev), v.to(dev), bt.to(dev), lens.to(dev), cu_seqlens_q=cu, out=out)
    assert (out[:3] == 7).all() and (out[12:] == 7).all() and not (out[3:12] == 7).any()


def test_empty_calls(cuda_device):
    dev = cuda_device
    q, k, v, bt, lens, cu = make([0, 0], [30, 0], 4, 2, 16, seed=10)
    out, lse = pgqa.cross_attention(q.to(dev), k.to(dev), v.to(dev), bt.to(dev), lens.to(dev),
                                    cu_seqlens_q=cu.to(dev), return_lse=True)
    assert out.shape == (0, 4, 128) and lse.shape == (4, 0)


def test_two_streams_and_graphs(cuda_device):
    dev = cuda_device
    cases = [make([5, 3], [8000, 600], 8, 2, 16, seed=11 + i) for i in range(2)]
    args = [[x.to(dev) for x in c] for c in cases]
    alone = [pgqa.cross_attention(*a[:5], cu_seqlens_q=a[5]) for a in args]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in args]
    for _ in range(5):
        outs = []
        for s, a in zip(streams, args):
            with torch.cuda.stream(s):
                outs.append(pgqa.cross_attention(*a[:5], cu_seqlens_q=a[5]))
        torch.cuda.synchronize()
        assert all(torch.equal(o, r) for o, r in zip(outs, alone))
    graphs, outs = [], []
    for a in args:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(pgqa.cross_attention(*a[:5], cu_seqlens_q=a[5]))
        graphs.append(g)
    for s, g in zip(streams, graphs):
        with torch.cuda.stream(s):
            g.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(o, r) for o, r in zip(outs, alone))


def test_bad_pages_and_lengths_are_reported(cuda_device):
    dev = cuda_device
    for what, status in (("page", 9), ("len", 10), ("neg", 10), ("cu", 10)):
        q, k, v, bt, lens, cu = make([10, 10], [60, 60], 4, 2, 16, seed=13)
        k, v = (torch.nan_to_num(x.float()).to(torch.bfloat16) for x in (k, v))
        if what == "page":
            bt[1, 1] = -7
        elif what == "len":
            bt[bt == 2 ** 30] = 0
            lens[1] = 16 * bt.shape[1] + 1
        elif what == "neg":
            lens[0] = -1
        else:
            cu[2] = 21
        pgqa.cross_attention(q.to(dev), k.to(dev), v.to(dev), bt.to(dev), lens.to(dev), cu_seqlens_q=cu.to(dev))
        with pytest.raises(PgqaError) as e:
            pgqa.check_device_error()
        assert e.value.status == status, what
        pgqa.check_device_error()


def test_an_expired_wait_is_reported_and_leaves_the_context_usable(cuda_device, monkeypatch):
    """A load that waits for 16 bytes that are never sent: every role gives up at its (short)
    limit, the call ends and the next one is right."""
    case = make([70, 9], [900, 333], 8, 2, 16, seed=30)
    args = [x.to(cuda_device) for x in case]
    monkeypatch.setenv("PGQA_DEBUG_STUCK_BARRIER", "1")
    monkeypatch.setenv("PGQA_WAIT_LIMIT_NS", "3000000")
    pgqa.cross_attention(*args[:5], cu_seqlens_q=args[5])
    with pytest.raises(PgqaError) as e:
        pgqa.check_device_error()
    assert e.value.status == 8
    monkeypatch.delenv("PGQA_DEBUG_STUCK_BARRIER")
    monkeypatch.delenv("PGQA_WAIT_LIMIT_NS")
    run_and_check(case, cuda_device)


@pytest.mark.parametrize("Hq,Hkv,P", [(32, 8, 16), (28, 4, 64), (6, 2, 256), (16, 16, 48)])
def test_e4m3_pages(Hq, Hkv, P, cuda_device):
    """e4m3 K and V are exact in bf16 and their scales multiply in fp32: the bounds of bf16
    pages, with one more fp32 rounding of the score's factor (2^-23 of the largest score)."""
    dev = cuda_device
    for new, lens in (([40, 0, 1, 150, 7, 300, 0], [700, 30, 0, 129, 1300, 256, 5]), ([2], [20000]),
                      ([65, 64, 1], [1, 16, 17]), ([33] * 12, [64 * i + 1 for i in range(12)])):
        q, k, v, bt, lens, cu = make(new, lens, Hq, Hkv, P, seed=Hq + len(new), std=4.0, kv="e4m3")
        g = torch.Generator().manual_seed(1)
        ks, vs = (torch.rand(Hkv, generator=g) * 0.2 + 0.15 for _ in range(2))
        a = [x.to(dev) for x in (q, k, v, bt, lens)]
        out, lse = pgqa.cross_attention(*a, cu_seqlens_q=cu.to(dev), k_scale=ks.to(dev), v_scale=vs.to(dev),
                                        return_lse=True)
        pgqa.check_device_error()
        check(out, lse, reference(q, k, v, bt, lens, cu, 1 / math.sqrt(128), dev, ks, vs))
    plain = pgqa.cross_attention(*a, cu_seqlens_q=cu.to(dev))
    one = torch.ones(Hkv)
    check(plain, None, reference(q, k, v, bt, lens, cu, 1 / math.sqrt(128), dev, one, one))
    # a scale of zero gives every key the same weight, one below zero turns the scores around
    ks = torch.tensor([0.0, -0.2] * (Hkv // 2))
    out, lse = pgqa.cross_attention(*a, cu_seqlens_q=cu.to(dev), k_scale=ks.to(dev), v_scale=-0.3, return_lse=True)
    check(out, lse, reference(q, k, v, bt, lens, cu, 1 / math.sqrt(128), dev, ks, torch.full((Hkv,), -0.3)))
    with pytest.raises(ValueError):
        pgqa.cross_attention(a[0], a[1].to(torch.bfloat16), a[2].to(torch.bfloat16), *a[3:], cu_seqlens_q=cu.to(dev),
                             k_scale=1.0)


def test_e4m3_every_value(cuda_device):
    """One key: the output is its V, exactly, for all 256 codes (a NaN stays one and stays in
    its place); a NaN in K makes its row's result NaN."""
    dev = cuda_device
    codes = torch.arange(256, dtype=torch.uint8).view(torch.float8_e4m3fn).view(2, 1, 1, 128)
    k = torch.zeros(2, 16, 2, 128).to(torch.float8_e4m3fn)
    v = torch.full((2, 16, 2, 128), float("nan")).to(torch.float8_e4m3fn)
    v.view(torch.uint8)[:, :1] = codes.view(torch.uint8)
    bt = torch.tensor([[0], [1], [0]], dtype=torch.int32)
    lens = torch.ones(3, dtype=torch.int32)
    k.view(torch.uint8)[1, 0, 1, 77] = 0x7F
    q = torch.randn(6, 4, 128).to(torch.bfloat16)
    out = pgqa.cross_attention(*[x.to(dev) for x in (q.view(3, 2, 4, 128), k, v, bt, lens)]).cpu()
    want = codes.float().view(2, 128)
    for b, page in enumerate((0, 1, 0)):
        w = want[page].expand(2, 2, 128)
        assert torch.equal(torch.nan_to_num(out[b, :, :2].float(), 1e9), torch.nan_to_num(w, 1e9))
        assert out[b, :, 2:].isnan().all() if page else torch.equal(
            torch.nan_to_num(out[b, :, 2:].float(), 1e9), torch.nan_to_num(w, 1e9))


def test_e4m3_expired_wait(cuda_device, monkeypatch):
    case = make([70, 9], [900, 333], 8, 2, 16, seed=30, kv="e4m3")
    args = [x.to(cuda_device) for x in case]
    want = pgqa.cross_attention(*args[:5], cu_seqlens_q=args[5])
    monkeypatch.setenv("PGQA_DEBUG_STUCK_BARRIER", "1")
    monkeypatch.setenv("PGQA_WAIT_LIMIT_NS", "3000000")
    pgqa.cross_attention(*args[:5], cu_seqlens_q=args[5])
    with pytest.raises(PgqaError) as e:
        pgqa.check_device_error()
    assert e.value.status == 8
    monkeypatch.delenv("PGQA_DEBUG_STUCK_BARRIER")
    monkeypatch.delenv("PGQA_WAIT_LIMIT_NS")
    assert torch.equal(pgqa.cross_attention(*args[:5], cu_seqlens_q=args[5]), want)
