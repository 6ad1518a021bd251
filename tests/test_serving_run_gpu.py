"""The operators around the decode together, as a server uses them: prompts of text and image
tokens enter the cache, attend over an encoder's states, and a decode loop turns, appends,
attends, keeps the attention weights and holds the cache at a budget.  Every step is compared
with 64-bit restatements of the same steps on the CPU."""
import math

import pytest
import torch

import mx_flash_attn_kernel_opt__b200 as pgqa
from oracle import evict_ref, paged_decode_ref, rope_ref, weights_ref
from tests import _paged
from tests.test_cross_gpu import check as check_cross, reference as cross_reference
from tests.test_parity_gpu import assert_parity
from tests.test_rope_gpu import tables

pytestmark = pytest.mark.gpu

Hq, Hkv, P, KEEP, SINKS, RECENT = 8, 2, 16, 24, 2, 6


def test_prompts_decode_and_eviction(cuda_device):
    dev = cuda_device
    g = torch.Generator().manual_seed(0)
    new = [30, 9, 41]
    B, T, scale = len(new), sum(new), 1 / math.sqrt(128)
    lens = torch.zeros(B, dtype=torch.int32)
    bt, pages = _paged.table([64] * B, P, g)
    k = torch.zeros(pages, P, Hkv, 128, dtype=torch.bfloat16)
    v, w = torch.zeros_like(k), torch.full((pages, Hkv, P), 9.0)   # what an earlier user of the pages left
    cos, sin = tables(2048, 128)
    axes = [i % 3 for i in range(64)]
    cu = torch.tensor([0, 30, 39, 80], dtype=torch.int32)
    pos = torch.randint(0, 500, (3, T), generator=g, dtype=torch.int32)
    qkv = torch.randn(T, Hq + 2 * Hkv, 128, generator=g).to(torch.bfloat16)

    d = {n: x.to(dev) for n, x in dict(k=k, v=v, w=w, bt=bt, cos=cos, sin=sin).items()}
    x = qkv.to(dev)
    q = pgqa.rope_append_kv(x[:, :Hq], x[:, Hq:Hq + Hkv], x[:, Hq + Hkv:], d["k"], d["v"], d["bt"], lens.to(dev),
                            d["cos"], d["sin"], positions=pos.to(dev), axes=axes, cu_seqlens=cu.to(dev), weights=d["w"])
    rows = pos.long()[torch.tensor(axes)].t()
    want = rope_ref(qkv[:, :Hq], cos, sin, rows)
    assert ((q.cpu().double() - want).abs() <= 2.0 ** -8 * want.abs() + 2.0 ** -20 * want.abs().max()).all()

    # the prompt's tokens over an encoder's states of other lengths, none for the second prompt
    enc_lens = torch.tensor([197, 0, 333], dtype=torch.int32)
    ebt, epages = _paged.table(enc_lens.tolist(), 64, g)
    ek, ev = (_paged.pool(epages, 64, Hkv, g) for _ in range(2))
    out, lse = pgqa.cross_attention(q, ek.to(dev), ev.to(dev), ebt.to(dev), enc_lens.to(dev), cu_seqlens_q=cu.to(dev),
                                    return_lse=True)
    check_cross(out, lse, cross_reference(q.cpu(), ek, ev, ebt, enc_lens, cu, scale, dev))

    # the CPU's state from here on is what the device wrote, step by step
    k, v, w = d["k"].cpu(), d["v"].cpu(), d["w"].cpu()
    for b in range(B):
        for t in range(new[b]):
            assert (w[bt[b, t // P], :, t % P] == 0).all()
    lens = torch.tensor(new, dtype=torch.int32)
    for step in range(6):
        qkv = torch.randn(B, Hq + 2 * Hkv, 128, generator=g).to(torch.bfloat16)
        pos = torch.randint(0, 2048, (3, B), generator=g, dtype=torch.int32)
        x = qkv.to(dev)
        q = pgqa.rope_append_kv(x[:, :Hq], x[:, Hq:Hq + Hkv], x[:, Hq + Hkv:], d["k"], d["v"], d["bt"], lens.to(dev),
                                d["cos"], d["sin"], positions=pos.to(dev), axes=axes, weights=d["w"])
        k, v, w = d["k"].cpu(), d["v"].cpu(), d["w"].cpu()
        lens = lens + 1
        out, lse = pgqa.decode(q, d["k"], d["v"], d["bt"], lens.to(dev), return_lse=True)
        ref, rlse = paged_decode_ref(q.cpu(), k, v, bt, lens, return_lse=True)
        assert_parity(out, ref, edge=True, what=f"step {step}")
        assert torch.allclose(lse.cpu(), rlse, atol=1e-3, rtol=1e-3)
        pgqa.accumulate_weights(q, d["k"], d["bt"], lens.to(dev), lse, d["w"])
        wref, bound = weights_ref(q.cpu(), k, bt, lens, lse.cpu(), w, scale)
        assert ((d["w"].cpu().double() - wref).abs() <= bound).all()
        w = d["w"].cpu()
        kept, new_lens = pgqa.evict_kv(d["k"], d["v"], d["w"], d["bt"], lens.to(dev), KEEP, sinks=SINKS, recent=RECENT)
        rk, rl, k, v, w = evict_ref(k, v, w, bt, lens, KEEP, SINKS, RECENT)
        assert torch.equal(kept.cpu(), rk) and torch.equal(new_lens.cpu(), rl)
        assert torch.equal(_paged.raw(d["k"]), _paged.raw(k)) and torch.equal(d["w"].cpu(), w)
        lens = rl
    assert lens.tolist() == [24, 15, 24]
    pgqa.check_device_error()


def test_decode_loop_in_one_graph(cuda_device):
    """One captured step (turn and append, decode, weights, eviction) replayed with new inputs
    equals the eager calls bit for bit."""
    dev = cuda_device
    g = torch.Generator().manual_seed(1)
    B, L = 2, 25
    bt, pages = _paged.table([32] * B, P, g)
    k, v = (_paged.pool(pages, P, Hkv, g) for _ in range(2))
    cos, sin = (x.to(dev) for x in tables(64, 64))
    btd, lens = bt.to(dev), torch.full((B,), L - 1, dtype=torch.int32, device=dev)
    after = lens + 1
    pos = torch.arange(B, dtype=torch.int32, device=dev)
    inputs = [torch.randn(B, Hq + 2 * Hkv, 128, generator=g).to(torch.bfloat16).to(dev) for _ in range(4)]

    def step(x, kd, vd, wd):
        q = pgqa.rope_append_kv(x[:, :Hq], x[:, Hq:Hq + Hkv], x[:, Hq + Hkv:], kd, vd, btd, lens, cos, sin,
                                positions=pos, weights=wd)
        out, lse = pgqa.decode(q, kd, vd, btd, after, return_lse=True)
        pgqa.accumulate_weights(q, kd, btd, after, lse, wd)
        kept, _ = pgqa.evict_kv(kd, vd, wd, btd, after, L - 1, sinks=1, recent=4)
        return out, kept

    def state():
        return k.to(dev), v.to(dev), torch.zeros(pages, Hkv, P, device=dev)

    eager = state()
    want = [step(x, *eager) for x in inputs]
    graphed, x = state(), inputs[0].clone()
    fresh = state()
    step(x, *graphed)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step(x, *graphed)
    for a, b in zip(graphed, fresh):
        a.copy_(b)
    for i, new in enumerate(inputs):
        x.copy_(new)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(got[0], want[i][0]) and torch.equal(got[1], want[i][1])
    for a, b in zip(graphed, eager):
        assert torch.equal(a, b)


def test_flash_attn_rotary_arguments(cuda_device):
    """flash_attn_with_kvcache turns and appends with rotary_cos / rotary_sin as flash-attn does:
    k at cache_seqlens + s; q there too if causal, at cache_seqlens for every token if not."""
    dev = cuda_device
    g = torch.Generator().manual_seed(2)
    lens = [5, 0, 30]
    for causal, Sq, S, interleaved, R in ((True, 3, 3, True, 128), (False, 3, 3, False, 64), (True, 2, 4, False, 128),
                                          (False, 1, 1, True, 32)):
        B = len(lens)
        bt, pages = _paged.table([n + S for n in lens], P, g)
        k, v = (_paged.pool(pages, P, Hkv, g) for _ in range(2))
        cos, sin = tables(64, R, torch.bfloat16)
        q = torch.randn(B, Sq, Hq, 128, generator=g).to(torch.bfloat16)
        kn, vn = (torch.randn(B, S, Hkv, 128, generator=g).to(torch.bfloat16) for _ in range(2))
        seq = torch.tensor(lens, dtype=torch.int32)
        kd, vd = k.to(dev), v.to(dev)
        out = pgqa.flash_attn_with_kvcache(q.to(dev), kd, vd, k=kn.to(dev), v=vn.to(dev), rotary_cos=cos.to(dev),
                                           rotary_sin=sin.to(dev), cache_seqlens=seq.to(dev), block_table=bt.to(dev),
                                           causal=causal, rotary_interleaved=interleaved)
        at = lambda n, step: (seq.long()[:, None] + torch.arange(n) * step).reshape(-1, 1).expand(-1, R // 2)  # noqa: E731
        # q at the end-aligned places of a causal call: the tables' row is cache_seqlens + i
        qt = rope_ref(q.reshape(-1, Hq, 128), cos, sin, at(Sq, 1 if causal else 0), interleaved)
        kt = rope_ref(kn.reshape(-1, Hkv, 128), cos, sin, at(S, 1), interleaved).to(torch.bfloat16).reshape(kn.shape)
        got_k, got_v = kd.cpu(), vd.cpu()
        for b, n in enumerate(lens):
            for s in range(S):
                pg, sl = int(bt[b, (n + s) // P]), (n + s) % P
                assert ((got_k[pg, sl].double() - kt[b, s].double()).abs()
                        <= 2.0 ** -7 * kt[b, s].double().abs() + 1e-6).all()   # the two roundings of one value
                assert torch.equal(got_v[pg, sl], vn[b, s])
        ref = paged_decode_ref(qt.to(torch.bfloat16).reshape(q.shape), got_k, got_v, bt, seq + S, causal=causal)
        assert_parity(out, ref, edge=True, what=f"causal={causal} Sq={Sq} S={S}")
    pgqa.check_device_error()


def test_captured_with_scalar_scales(cuda_device):
    """e4m3 pages with one number as the scale of all heads: the calls can be captured, and the
    replay equals the eager calls."""
    dev = cuda_device
    g = torch.Generator().manual_seed(3)
    lens = [20, 33]
    bt, pages = _paged.table([n + 1 for n in lens], P, g)
    pools = [_paged.pool(pages, P, Hkv, g, "e4m3").to(dev) for _ in range(2)]
    cos, sin = (x.to(dev) for x in tables(64, 128))
    btd, before = bt.to(dev), torch.tensor(lens, dtype=torch.int32, device=dev)
    after = before + 1
    x = torch.randn(2, Hq + 2 * Hkv, 128, generator=g).to(torch.bfloat16).to(dev)

    def step(k, v, w):
        q = pgqa.rope_append_kv(x[:, :Hq], x[:, Hq:Hq + Hkv], x[:, Hq + Hkv:], k, v, btd, before, cos, sin, weights=w,
                                k_scale=0.5, v_scale=0.25)
        out, lse = pgqa.cross_attention(q.unsqueeze(1), k, v, btd, after, k_scale=0.5, v_scale=0.25, return_lse=True)
        pgqa.accumulate_weights(q, k, btd, after, lse, w, k_scale=0.5)
        return out

    eager = [p.clone() for p in pools] + [torch.zeros(pages, Hkv, P, device=dev)]
    want = step(*eager)
    # one query token per sequence: the weights that each KV head's tokens received sum up to its rows
    w = eager[2].cpu()
    sums = torch.stack([w[bt[b, :-(-(n + 1) // P)].long()].sum((0, 2)) for b, n in enumerate(lens)])
    assert torch.allclose(sums, torch.full_like(sums, Hq / Hkv), rtol=1e-4)
    state = [p.clone() for p in pools] + [torch.zeros(pages, Hkv, P, device=dev)]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step(*state)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(got, want) and torch.equal(state[2], eager[2])
    assert all(torch.equal(_paged.raw(a), _paged.raw(b)) for a, b in zip(state, eager))
    pgqa.check_device_error()
