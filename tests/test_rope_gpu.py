"""rope_append_kv against the 64-bit restatement: rotation within one rounding, cache rows and
weight entries at the right places and nothing else touched."""
import pytest
import torch

import mx_flash_attn_kernel_opt__b200 as pgqa
from mx_flash_attn_kernel_opt__b200 import PgqaError
from oracle import rope_ref
from tests import _paged

pytestmark = pytest.mark.gpu


def tables(rows, R, dtype=torch.float32):
    inv = 1e4 ** (-torch.arange(0, R, 2, dtype=torch.float64) / R)
    ang = torch.arange(rows, dtype=torch.float64)[:, None] * inv
    return ang.cos().to(dtype), ang.sin().to(dtype)


def assert_turned(got, ref, x, scale=None):
    """got: bf16, or e4m3 standing for value * scale.  Half a step of the type (bf16 2^-8
    relative; e4m3 2^-4, or 2^-10 of the scale below its smallest normal), plus fp32's error
    on two products and a sum: 3 * 2^-24 of their magnitudes, at most 2 |x|max each."""
    got, ref = got.cpu().float().double(), ref.double()
    arith = 6 * 2.0 ** -24 * x.abs().double().amax(-1, keepdim=True)
    if scale is None:
        tol = 2.0 ** -8 * ref.abs() + 2 * arith
    else:
        s = scale.cpu().double().view(1, -1, 1)
        got, ref = got * s, ref.clamp(-448 * s, 448 * s)
        tol = torch.maximum(2.0 ** -4 * ref.abs(), 2.0 ** -10 * s) * (1 + 2.0 ** -20) + 2 * arith
    over = (got - ref).abs() - tol
    assert not over.isnan().any()
    assert (over <= 0).all(), f"over the bound by {over.max().item():.3e}"


class Case:
    def __init__(self, lens, new, Hq=8, Hkv=2, P=16, R=128, kv="bf16", axes="one", packed=False,
                 interleaved=False, table="fp32", seed=0, clear=True, rows=4096):
        g = torch.Generator().manual_seed(seed)
        self.lens, self.new, self.P, self.R, self.kv = lens, new, P, R, kv
        self.bt, self.pages = _paged.table([a + b for a, b in zip(lens, new)], P, g)
        T = sum(new)
        self.T, self.Hq, self.Hkv = T, Hq, Hkv
        # slices of one projection
        self.qkv = torch.randn(T, Hq + 2 * Hkv + 1, 128, generator=g).to(torch.bfloat16)
        self.kc, self.vc = (_paged.pool(self.pages, P, Hkv, g, kv) for _ in range(2))
        self.cos, self.sin = tables(rows, R, torch.float32 if table == "fp32" else torch.bfloat16)
        n = R // 2
        self.naxes = 1 if axes == "one" else 3
        self.axes = {"one": [0] * n, "runs": [3 * i // n for i in range(n)],
                     "turn": [i % 3 for i in range(n)]}[axes]
        self.pos = torch.randint(0, rows, (self.naxes, T), generator=g, dtype=torch.int32)
        self.ks = (torch.rand(Hkv, generator=g) * 0.02 + 0.002) if kv == "e4m3" else None
        self.vs = (torch.rand(Hkv, generator=g) * 0.02 + 0.002) if kv == "e4m3" else None
        self.w = torch.rand(self.pages, Hkv, P, generator=g) if clear else None
        self.packed, self.interleaved = packed, interleaved

    def split(self, x):
        return x[:, :self.Hq], x[:, self.Hq:self.Hq + self.Hkv], \
            x[:, self.Hq + self.Hkv:self.Hq + 2 * self.Hkv]

    def to(self, dev):
        self.d = {n: (None if getattr(self, n) is None else getattr(self, n).to(dev)) for n in
                  ("qkv", "bt", "kc", "vc", "cos", "sin", "pos", "ks", "vs", "w")}
        self.d["lens"] = torch.tensor(self.lens, dtype=torch.int32, device=dev)
        return self

    def call(self, positions=True, **kw):
        d = self.d
        q, k, v = self.split(d["qkv"])
        cu = None
        pos = d["pos"]
        if self.packed:
            cu = torch.tensor([sum(self.new[:b]) for b in range(len(self.new) + 1)],
                              dtype=torch.int32, device=q.device)
        else:
            B, S = len(self.new), self.new[0]
            q, k, v = (x.unflatten(0, (B, S)) for x in (q, k, v))
            pos = pos.unflatten(1, (B, S))
        args = dict(positions=pos if positions else None, axes=self.axes if positions else None,
                    interleaved=self.interleaved, cu_seqlens=cu, weights=d["w"], k_scale=d["ks"],
                    v_scale=d["vs"])
        args.update(kw)
        return pgqa.rope_append_kv(q, k, v, d["kc"], d["vc"], d["bt"], d["lens"], d["cos"],
                                   d["sin"], **args)

    def places(self):
        return [(b, self.lens[b] + s) for b in range(len(self.new)) for s in range(self.new[b])]

    def check(self, out, positions=True):
        q, k, v = self.split(self.qkv)
        if positions:
            rows = self.pos.long()[torch.tensor(self.axes)].t()
        else:
            rows = torch.tensor([[t] * (self.R // 2) for _, t in self.places()])
        turn = lambda x: rope_ref(x, self.cos, self.sin, rows, self.interleaved)  # noqa: E731
        if self.T:
            assert_turned(out.reshape(self.T, self.Hq, 128), turn(q), q.float())
        kc, vc = self.d["kc"].cpu(), self.d["vc"].cpu()
        at = [(int(self.bt[b, t // self.P]), t % self.P) for b, t in self.places()]
        if self.T:
            pg, sl = (torch.tensor(x) for x in zip(*at))
            gk, gv = kc.float()[pg, sl], vc.float()[pg, sl]
            assert_turned(gk, turn(k), k.float(), self.ks)
            if self.kv == "bf16":
                assert torch.equal(gv, v.float())
            else:
                assert_turned(gv, v.double(), v.float(), self.vs)
            # every other slot is as it was
            for got, was in ((kc, self.kc), (vc, self.vc)):
                g8, w8 = got.view(torch.uint8).clone(), was.view(torch.uint8)
                g8[pg, sl] = w8[pg, sl]
                assert torch.equal(g8, w8)
            if self.w is not None:
                w = self.w.clone()
                w[pg, :, sl] = 0
                assert torch.equal(self.d["w"].cpu(), w)
        else:
            assert torch.equal(_paged.raw(kc), _paged.raw(self.kc))


@pytest.mark.parametrize("kv", ["bf16", "e4m3"])
@pytest.mark.parametrize("R,axes,interleaved,table", [
    (128, "one", False, "fp32"), (128, "turn", False, "fp32"), (128, "runs", True, "bf16"),
    (64, "turn", True, "fp32"), (48, "runs", False, "bf16"), (16, "one", True, "fp32"),
    (96, "one", False, "bf16"), (112, "runs", False, "fp32")])
def test_turns_and_appends(kv, R, axes, interleaved, table, cuda_device):
    c = Case([0, 5, 31, 16], [3] * 4, R=R, axes=axes, interleaved=interleaved, table=table, kv=kv,
             seed=R).to(cuda_device)
    c.check(c.call())
    pgqa.check_device_error()


@pytest.mark.parametrize("Hq,Hkv,P", [(32, 8, 16), (28, 4, 64), (5, 1, 48), (16, 16, 32)])
@pytest.mark.parametrize("new", [[1], [7, 0, 1, 30, 0], [0, 0, 2], [0], [65, 3]])
def test_packed_sequences(Hq, Hkv, P, new, cuda_device):
    lens = [(13 * i) % 40 for i in range(len(new))]
    c = Case(lens, new, Hq=Hq, Hkv=Hkv, P=P, packed=True, axes="turn", seed=P + len(new)).to(cuda_device)
    c.check(c.call())
    pgqa.check_device_error()


def test_many_packed_sequences(cuda_device):
    g = torch.Generator().manual_seed(5)
    new = torch.randint(0, 4, (1100,), generator=g).tolist()
    c = Case([1] * 1100, new, Hq=2, Hkv=1, R=16, packed=True, seed=6).to(cuda_device)
    c.check(c.call())


def test_own_places_are_the_positions(cuda_device):
    c = Case([0, 9, 40], [4] * 3, seed=2, clear=False).to(cuda_device)
    c.check(c.call(positions=False), positions=False)


def test_one_token_per_sequence_and_strided_table_free_q(cuda_device):
    c = Case([3, 17], [1, 1], seed=3).to(cuda_device)
    q, k, v = c.split(c.d["qkv"])
    pos = c.d["pos"][0].contiguous()
    out = pgqa.rope_append_kv(q, k, v, c.d["kc"], c.d["vc"], c.d["bt"], c.d["lens"], c.d["cos"],
                              c.d["sin"], positions=pos, weights=c.d["w"])
    assert out.shape == q.shape and out.is_contiguous()
    c.check(out)


def test_batch_strides_of_a_padded_buffer(cuda_device):
    """q, k, v as the first tokens of every sequence of a longer padded projection."""
    c = Case([2, 30, 7], [2] * 3, seed=4).to(cuda_device)
    wide = torch.zeros(3, 5, *c.qkv.shape[1:], dtype=torch.bfloat16, device=cuda_device)
    wide[:, :2] = c.d["qkv"].unflatten(0, (3, 2))
    part = wide[:, :2]
    q, k, v = part[:, :, :8], part[:, :, 8:10], part[:, :, 10:12]
    assert not q.is_contiguous()
    out = pgqa.rope_append_kv(q, k, v, c.d["kc"], c.d["vc"], c.d["bt"], c.d["lens"], c.d["cos"],
                              c.d["sin"], positions=c.d["pos"].unflatten(1, (3, 2)), axes=c.axes,
                              weights=c.d["w"])
    c.check(out)


def test_append_without_q_and_rows_behind_the_last_sequence(cuda_device):
    c = Case([4, 4], [2, 3], packed=True, seed=8).to(cuda_device)
    q, k, v = c.split(c.d["qkv"])
    # two more tokens than cu_seqlens covers: their rows of q_out stay as they are
    cu = torch.tensor([0, 2, 3], dtype=torch.int32, device=cuda_device)
    q_out = torch.full(q.shape, 7.0, dtype=torch.bfloat16, device=cuda_device)
    c.call(cu_seqlens=cu, q_out=q_out)
    assert (q_out[3:] == 7).all() and not (q_out[:3] == 7).all()
    fresh = Case([4, 4], [2, 3], packed=True, seed=8).to(cuda_device)
    cu = torch.tensor([0, 2, 5], dtype=torch.int32, device=cuda_device)
    q, k, v = fresh.split(fresh.d["qkv"])
    assert pgqa.rope_append_kv(None, k, v, fresh.d["kc"], fresh.d["vc"], fresh.d["bt"], fresh.d["lens"],
                               fresh.d["cos"], fresh.d["sin"], positions=fresh.d["pos"], axes=fresh.axes,
                               cu_seqlens=cu, weights=fresh.d["w"]) is None
    full = Case([4, 4], [2, 3], packed=True, seed=8).to(cuda_device)
    full.call()
    assert torch.equal(_paged.raw(fresh.d["kc"]), _paged.raw(full.d["kc"]))
    assert torch.equal(_paged.raw(fresh.d["vc"]), _paged.raw(full.d["vc"]))


def test_e4m3_saturates_and_keeps_nan(cuda_device):
    c = Case([0], [2], kv="e4m3", seed=9, Hq=1, Hkv=1, R=16).to(cuda_device)
    c.d["qkv"][:] = 1000.0
    c.d["qkv"][1, 2, 100] = float("nan")
    c.d["ks"][:] = 1.0
    c.d["vs"][:] = 2.0
    c.call()
    pg = int(c.bt[0, 0])
    k, v = c.d["kc"].cpu().float()[pg], c.d["vc"].cpu().float()[pg]
    assert (k[:2, 0, 16:] == 448).all() and (v[0, 0] == 448).all()
    assert v[1, 0, 100].isnan() and (v[1, 0, :100] == 448).all()


def test_bad_positions_pages_and_lengths_are_reported(cuda_device):
    for what, status in (("pos", 12), ("neg", 12), ("page", 9), ("len", 10), ("neglen", 10)):
        c = Case([5, 20], [2, 2], seed=11, rows=64).to(cuda_device)
        if what == "pos":
            c.d["pos"][0, 3] = 64
        elif what == "neg":
            c.d["pos"][0, 3] = -1
        elif what == "page":
            c.d["bt"][1, 1] = c.pages
        elif what == "len":
            c.d["lens"][1] = 16 * c.bt.shape[1]
        else:
            c.d["lens"][1] = -3
        q_out = torch.full((2, 2, 8, 128), 7.0, dtype=torch.bfloat16, device=cuda_device)
        c.call(q_out=q_out)
        with pytest.raises(PgqaError) as e:
            pgqa.check_device_error()
        assert e.value.status == status, what
        assert (q_out[1, 1] == 7).all()          # nothing of the bad token is written
        assert not (q_out[0] == 7).all()
        pgqa.check_device_error()                # cleared


def test_other_stream_and_graph(cuda_device):
    c = Case([1, 2], [3, 3], seed=12).to(cuda_device)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        out = c.call()
    s.synchronize()
    c.check(out)
    kc0, vc0, w0 = c.kc.to(cuda_device), c.vc.to(cuda_device), c.w.to(cuda_device)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = c.call()
    for _ in range(2):
        c.d["kc"].copy_(kc0); c.d["vc"].copy_(vc0); c.d["w"].copy_(w0); out.zero_()
        graph.replay()
        torch.cuda.synchronize()
        c.check(out)
