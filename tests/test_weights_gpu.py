"""accumulate_weights against the 64-bit restatement, within the bound that fp32 scores,
exponents and sums allow (derived in oracle/serving.py)."""
import math

import pytest
import torch

import mx_flash_attn_kernel_opt__b200 as pgqa
from mx_flash_attn_kernel_opt__b200 import PgqaError
from oracle import weights_ref
from tests import _paged

pytestmark = pytest.mark.gpu


def make(lens, Hq, Hkv, P, Sq=1, kv="bf16", causal=False, seed=0, one_token=False):
    g = torch.Generator().manual_seed(seed)
    bt, pages = _paged.table(lens, P, g)
    k = _paged.poison_unused(_paged.pool(pages, P, Hkv, g, kv, 2.0 if kv == "e4m3" else 1.0), lens, bt, P)
    q = torch.randn(len(lens), Sq, Hq, 128, generator=g).to(torch.bfloat16)
    ks = torch.rand(Hkv, generator=g) * 0.4 + 0.3 if kv == "e4m3" else None
    w = torch.rand(pages, Hkv, P, generator=g) * 0.01
    lens_t = torch.tensor(lens, dtype=torch.int32)
    scale = 1 / math.sqrt(128)
    # the decode's log-sum-exp, in 64 bits
    lse = torch.full((len(lens), Hq, Sq), -math.inf)
    kd = k.float().double() * (ks.double().view(1, 1, Hkv, 1) if ks is not None else 1.0)
    for b, L in enumerate(lens):
        if not L:
            continue
        rows = kd[bt[b, [t // P for t in range(L)]].long(), [t % P for t in range(L)]]
        for i in range(Sq):
            m = max(0, L - Sq + 1 + i) if causal else L
            if m:
                x = torch.einsum("thd,hgd->hgt", rows[:m], q[b, i].double().view(Hkv, Hq // Hkv, 128)) * scale
                lse[b, :, i] = torch.logsumexp(x, -1).flatten().float()
    if one_token:
        q = q[:, 0]
    return q, k, bt, lens_t, lse, w, scale, ks


def run_and_check(args, causal, dev):
    q, k, bt, lens, lse, w, scale, ks = args
    ref, bound = weights_ref(q, k, bt, lens, lse, w, scale, causal, ks)
    wd = w.to(dev)
    out = pgqa.accumulate_weights(q.to(dev), k.to(dev), bt.to(dev), lens.to(dev), lse.to(dev), wd,
                                  causal=causal, k_scale=None if ks is None else ks.to(dev))
    assert out is wd
    pgqa.check_device_error()
    got = wd.cpu().double()
    untouched = bound == 0
    assert torch.equal(got[untouched], w.double()[untouched])
    over = (got - ref).abs() - bound
    assert not over.isnan().any() and (over <= 0).all(), f"over the bound by {over.max().item():.3e}"


@pytest.mark.parametrize("kv", ["bf16", "e4m3"])
@pytest.mark.parametrize("Hq,Hkv,P,Sq", [(32, 8, 16, 1), (28, 4, 64, 1), (4, 2, 48, 3), (16, 1, 32, 1),
                                         (8, 2, 16, 4), (12, 1, 16, 3), (2, 2, 16, 40), (20, 2, 32, 5)])
@pytest.mark.parametrize("causal", [False, True])
def test_matches_the_restatement(kv, Hq, Hkv, P, Sq, causal, cuda_device):
    run_and_check(make([0, 1, 2, 17, 45, 64], Hq, Hkv, P, Sq, kv, causal, seed=Hq + P + Sq), causal, cuda_device)


def test_one_token_form_and_long_sequence(cuda_device):
    run_and_check(make([700, 3], 4, 1, 16, one_token=True, seed=1), False, cuda_device)


def test_many_sequences(cuda_device):
    g = torch.Generator().manual_seed(3)
    lens = torch.randint(0, 6, (700,), generator=g).tolist()
    run_and_check(make(lens, 2, 1, 16, seed=4), False, cuda_device)


def test_follows_a_decode(cuda_device):
    """With the decode's own log-sum-exp every row gives one unit of weight per head."""
    q, k, bt, lens, _, w, _, _ = make([33, 0, 200, 1], 16, 4, 16, Sq=2, seed=5)
    dev = cuda_device
    k = torch.nan_to_num(k.float()).to(torch.bfloat16)
    qd, kd, btd, ld = q.to(dev), k.to(dev), bt.to(dev), lens.to(dev)
    _, lse = pgqa.decode(qd, kd, kd, btd, ld, causal=True, return_lse=True)
    wd = torch.zeros_like(w, device=dev)
    pgqa.accumulate_weights(qd, kd, btd, ld, lse, wd, causal=True)
    for b, L in enumerate(lens.tolist()):
        pg = torch.tensor([int(bt[b, t // 16]) for t in range(L)], dtype=torch.long)
        sl = torch.arange(L) % 16
        got = wd.cpu()[pg, :, sl].sum(0) if L else torch.zeros(4)
        # 4 heads x 2 tokens, of which the first token of a one-token sequence sees nothing
        want = 0 if L == 0 else 4.0 * (1 if L == 1 else 2)
        assert torch.allclose(got, torch.full((4,), float(want)), atol=1e-4)


def test_infinite_scores_and_masked_nan(cuda_device):
    """-inf scores weigh 0 and do not disturb the padding rows of a tile; NaN in masked slots
    stays out (the pools of `make` hold NaN in every unused slot)."""
    q, k, bt, lens, lse, w, scale, _ = make([20], 1, 1, 16, seed=6)
    dev = cuda_device
    k[bt[0, 0].long(), 3] = 0
    k[bt[0, 0].long(), 3, 0, 0] = -math.inf
    q[..., 0] = q[..., 0].abs() + 0.1
    wd = torch.zeros_like(w, device=dev)
    pgqa.accumulate_weights(q.to(dev), k.to(dev), bt.to(dev), lens.to(dev), lse.to(dev), wd)
    row = torch.stack([wd.cpu()[bt[0, t // 16].long(), 0, t % 16] for t in range(20)])
    assert row[3] == 0 and row.isfinite().all() and (row[:3] > 0).all()


def test_shared_page_gets_both_sums(cuda_device):
    q, k, bt, lens, lse, w, scale, _ = make([16, 16], 4, 1, 16, seed=7)
    bt[1, 0] = bt[0, 0]
    ref, bound = weights_ref(q, k, bt, lens, lse, w, scale)
    dev = cuda_device
    wd = w.to(dev)
    pgqa.accumulate_weights(q.to(dev), k.to(dev), bt.to(dev), lens.to(dev), lse.to(dev), wd)
    assert ((wd.cpu().double() - ref).abs() <= bound).all()


def test_repeats_bit_for_bit_and_in_a_graph(cuda_device):
    q, k, bt, lens, lse, w, _, _ = make([300, 77], 8, 2, 16, Sq=2, seed=8)
    dev = cuda_device
    a = [x.to(dev) for x in (q, k, bt, lens, lse)]
    w1, w2 = w.to(dev), w.to(dev)
    pgqa.accumulate_weights(*a, w1)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        pgqa.accumulate_weights(*a, w2)
    w2.copy_(w)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(w1, w2)


def test_bad_pages_and_lengths_are_reported(cuda_device):
    dev = cuda_device
    for what, status in (("page", 9), ("len", 10), ("neg", 10)):
        q, k, bt, lens, lse, w, _, _ = make([40, 40], 4, 2, 16, seed=9)
        k = torch.nan_to_num(k.float()).to(torch.bfloat16)
        if what == "page":
            bt[1, 1] = -1
        elif what == "len":
            bt[bt == 2 ** 30] = 0
            lens[1] = 16 * bt.shape[1] + 1
        else:
            lens[0] = -1
        wd = w.to(dev)
        pgqa.accumulate_weights(q.to(dev), k.to(dev), bt.to(dev), lens.to(dev), lse.to(dev), wd)
        with pytest.raises(PgqaError) as e:
            pgqa.check_device_error()
        assert e.value.status == status, what


@pytest.mark.parametrize("kv", ["bf16", "e4m3"])
def test_more_rows_than_one_turn_takes(kv, cuda_device):
    """g * Sq of 66 and of 35: several turns over a warp's chunks, the last one partly empty."""
    run_and_check(make([50, 3, 0], 22, 2, 16, 6, kv, True, seed=20), True, cuda_device)
    run_and_check(make([90], 5, 1, 32, 7, kv, False, seed=21), False, cuda_device)


@pytest.mark.parametrize("kv", ["bf16", "e4m3"])
@pytest.mark.parametrize("Hq,Sq", [(16, 4), (32, 4), (4, 8)])
@pytest.mark.parametrize("causal", [False, True])
def test_whole_groups_of_rows_over_long_sequences(kv, Hq, Sq, causal, cuda_device):
    """32, 64 and 16 rows per KV head without a padding row: chunks that every row sees, the
    causal border and the ragged end are in one call."""
    run_and_check(make([700, 33, 257, 16], Hq, 2, 16, Sq, kv, causal, seed=30 + Hq), causal, cuda_device)


@pytest.mark.parametrize("kv", ["bf16", "e4m3"])
def test_one_row_that_saw_nothing_among_many(kv, cuda_device):
    """A log-sum-exp of -inf in a whole group of rows: that row adds nothing, the others theirs."""
    q, k, bt, lens, lse, w, scale, ks = make([320, 40], 16, 2, 16, 4, kv, False, seed=41)
    lse[0, 5, 2] = -math.inf
    ref, bound = weights_ref(q, k, bt, lens, lse, w, scale, False, ks)
    dev = cuda_device
    wd = w.to(dev)
    pgqa.accumulate_weights(q.to(dev), k.to(dev), bt.to(dev), lens.to(dev), lse.to(dev), wd, scale=scale,
                            k_scale=None if ks is None else ks.to(dev))
    assert ((wd.cpu().double() - ref).abs() <= bound).all()
