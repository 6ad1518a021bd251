"""Cases of the operators around the paged decode, in a plain form and through the package.

Four operators of a serving step over a paged key-value cache:

  rope    rotary positions on one or several axes, and the append of the rotated keys and
          the values to the pages (bf16 or e4m3)
  weights the attention weight that each cached token receives, added to its slot
  evict   the least used tokens of each KV head leave the cache, the kept ones close up
  cross   attention of packed prompt tokens over encoder states held in pages

Layouts: q [B, Sq, Hq, 128] or packed [T, Hq, 128] with cu_seqlens [B + 1]; pools
[pages, P, Hkv, 128]; weights [pages, Hkv, P] fp32; block_table [B, width] int32; seq_lens
[B] int32.  With `own` false every operator is computed from elementary torch operations in
32 bits; with `own` true by the package's entry points.
"""
import math
import random

import torch

own = False

D = 128
FP8 = torch.float8_e4m3fn


# ---------------------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------------------

def listed():
    return [
        # one decode step of a small batch: launch latency
        dict(name="rope-step", op="rope", B=4, S=1, packed=False, Hq=32, Hkv=8, P=16, lo=900, hi=1024,
             R=128, axes="one", interleaved=False, table="fp32", kv="bf16", clear=False, ls=1),
        # one decode step of a large batch with e4m3 pages, three axes dealt out in turn
        dict(name="rope-step-e4m3", op="rope", B=256, S=1, packed=False, Hq=32, Hkv=8, P=16, lo=16, hi=256,
             R=128, axes="turn", interleaved=False, table="fp32", kv="e4m3", clear=True, ls=2),
        # prompts of text and images, packed, three axes in runs, half of each head turned
        dict(name="rope-prompts", op="rope", B=9, S=2047, packed=True, Hq=28, Hkv=4, P=64, lo=0, hi=40,
             R=64, axes="runs", interleaved=True, table="bf16", kv="bf16", clear=True, ls=3),
        # weights after a step of a small batch: latency
        dict(name="weights-step", op="weights", B=4, Sq=1, causal=False, Hq=32, Hkv=8, P=16, lo=1024, hi=1024,
             kv="bf16", ls=4),
        # after a step of a large ragged batch
        dict(name="weights-batch", op="weights", B=256, Sq=1, causal=False, Hq=32, Hkv=8, P=16, lo=128, hi=2048,
             kv="bf16", ls=5),
        # the last four tokens of long prompts in e4m3 pages vote, g = 8
        dict(name="weights-window-e4m3", op="weights", B=2, Sq=4, causal=True, Hq=64, Hkv=8, P=16, lo=32768,
             hi=32768, kv="e4m3", ls=6),
        # every step evicts one token per head
        dict(name="evict-step", op="evict", B=16, Hkv=8, P=16, lo=1025, hi=1025, keep=1024, sinks=4, recent=256,
             kv="bf16", ls=7),
        # a ragged batch is cut to a budget once its prompts are in
        dict(name="evict-batch", op="evict", B=64, Hkv=4, P=64, lo=64, hi=8192, keep=2048, sinks=4, recent=255,
             kv="bf16", ls=8),
        # two long prompts in e4m3 pages are cut to a quarter
        dict(name="evict-long-e4m3", op="evict", B=2, Hkv=8, P=16, lo=32000, hi=32768, keep=8192, sinks=16,
             recent=1024, kv="e4m3", ls=9),
        # a few prompt tokens over one image's states: latency
        dict(name="cross-few", op="cross", B=2, Hq=32, Hkv=8, P=16, qlo=5, qhi=16, lo=1024, hi=1024, ls=10),
        # ragged prompts over images of several sizes, g = 7
        dict(name="cross-ragged", op="cross", B=8, Hq=28, Hkv=4, P=64, qlo=17, qhi=1024, lo=197, hi=4097, ls=11),
        # long prompts over a video's states
        dict(name="cross-long", op="cross", B=2, Hq=32, Hkv=8, P=16, qlo=4096, qhi=4096, lo=8192, hi=8192, ls=12),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["rope", "weights", "evict", "cross"])
    Hq, Hkv = rng.choice([(32, 8), (64, 8), (28, 4), (16, 16), (8, 1)])
    c = dict(op=op, Hq=Hq, Hkv=Hkv, P=rng.choice([16, 32, 48, 64, 256]), ls=rng.randrange(1 << 20))
    kv = rng.choice(["bf16", "e4m3"])
    if op == "rope":
        tokens = _log_int(rng, 1, 16384)
        c.update(B=min(tokens, _log_int(rng, 1, 256)), R=16 * rng.randint(1, 8),
                 axes=rng.choice(["one", "runs", "turn"]), interleaved=rng.random() < 0.5,
                 table=rng.choice(["fp32", "bf16"]), kv=kv, clear=rng.random() < 0.5, packed=rng.random() < 0.5)
        c["S"] = max(1, tokens // c["B"])
        c["lo"] = 0
        c["hi"] = _log_int(rng, 16, 300)
    elif op == "weights":
        total = _log_int(rng, 64, 1 << 18)           # tokens over all sequences
        c.update(B=min(max(1, total // 16), _log_int(rng, 1, 256)), Sq=rng.choice([1, 1, 1, 2, 3, 4, 8]), kv=kv)
        c["causal"] = rng.random() < 0.5
        c["hi"] = max(2, total // c["B"])
        c["lo"] = rng.randint(1, c["hi"])
    elif op == "evict":
        total = _log_int(rng, 256, 1 << 17)
        c.update(B=min(max(1, total // 128), _log_int(rng, 1, 64)), kv=kv)
        c["hi"] = max(16, total // c["B"])
        c["lo"] = rng.randint(0, c["hi"])
        c["keep"] = rng.randint(4, c["hi"])
        c["sinks"] = rng.randint(0, min(16, c["keep"] // 4))
        c["recent"] = rng.randint(0, c["keep"] // 2)
        c.pop("Hq")
    else:
        c.update(B=_log_int(rng, 1, 16))
        c["qhi"] = max(1, _log_int(rng, 1, 4096) // c["B"])
        c["qlo"] = rng.randint(0, c["qhi"])
        c["hi"] = _log_int(rng, 16, 8192)
        c["lo"] = rng.randint(0, c["hi"])
    return c


def _lens(case, lo, hi, salt):
    """Lengths of the case's sequences: part of the case, the same for every seed."""
    r = random.Random(case["ls"] * 64 + salt)
    return [r.randint(lo, hi) for _ in range(case["B"])]


def _new_lens(case):
    """New tokens of each sequence of a rope case."""
    if not case["packed"]:
        return [case["S"]] * case["B"]
    r = random.Random(case["ls"] * 64 + 2)
    return [r.randint(0, 2 * case["S"]) for _ in range(case["B"])]


def _axis_of_pair(case):
    """Which position axis turns each pair of a head: the first for all, three in runs, or three in turn."""
    n = case["R"] // 2
    if case["axes"] == "one":
        return [0] * n
    if case["axes"] == "runs":
        return [min(2, 3 * i // n) for i in range(n)]
    return [i % 3 for i in range(n)]


# ---------------------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------------------

def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed * 7919 + 17)
    return g


def _table(lens, P, extra_pages, g):
    """A pool's pages dealt out to the sequences in random order; the pool's page count."""
    need = [-(-n // P) for n in lens]
    width = max(1, max(need))
    pages = max(1, sum(need) + extra_pages)
    ids = torch.randperm(pages, generator=g, device="cuda").to(torch.int32)
    bt = torch.zeros(len(lens), width, dtype=torch.int32, device="cuda")
    flat = torch.arange(width, device="cuda").unsqueeze(0).expand(len(lens), width)
    n = torch.tensor(need, device="cuda").unsqueeze(1)
    start = torch.tensor([sum(need[:b]) for b in range(len(lens))], device="cuda").unsqueeze(1)
    return torch.where(flat < n, ids[(start + flat).clamp(max=pages - 1)], bt), pages


def _pool(shape, kv, g, std=1.0):
    if kv == "bf16":
        return torch.randn(shape, generator=g, device="cuda", dtype=torch.bfloat16).mul_(std)
    return torch.randn(shape, generator=g, device="cuda", dtype=torch.float16).mul_(std).to(FP8)


def _i32(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def prepare(case, seed):
    return {"rope": _prepare_rope, "weights": _prepare_weights, "evict": _prepare_evict,
            "cross": _prepare_cross}[case["op"]](case, _gen(seed))


def _prepare_rope(case, g):
    B, Hq, Hkv, P, R = case["B"], case["Hq"], case["Hkv"], case["P"], case["R"]
    old, new = _lens(case, case["lo"], case["hi"], 1), _new_lens(case)
    bt, pages = _table([a + b for a, b in zip(old, new)], P, 2, g)
    T = sum(new)
    # the projection's output, of which q, k and v are slices
    qkv = torch.randn(T, Hq + 2 * Hkv, D, generator=g, device="cuda", dtype=torch.bfloat16)
    naxes = 1 if case["axes"] == "one" else 3
    rows = 32768
    inv = 1e6 ** (-torch.arange(0, R, 2, device="cuda", dtype=torch.float64) / R)
    ang = torch.arange(rows, device="cuda", dtype=torch.float64).unsqueeze(1) * inv
    dt = torch.float32 if case["table"] == "fp32" else torch.bfloat16
    first = torch.randint(0, rows - 8192, (naxes, 1), generator=g, device="cuda")
    pos = (first + torch.randint(0, 8192, (naxes, T), generator=g, device="cuda")).to(torch.int32)
    state = dict(op="rope", q=qkv[:, :Hq], k=qkv[:, Hq:Hq + Hkv], v=qkv[:, Hq + Hkv:], bt=bt, lens=_i32(old),
                 cos=ang.cos().to(dt), sin=ang.sin().to(dt), pos=pos, axes=_axis_of_pair(case),
                 interleaved=case["interleaved"], cu=None, kc=_pool((pages, P, Hkv, D), case["kv"], g),
                 vc=_pool((pages, P, Hkv, D), case["kv"], g), w=None, ks=None, vs=None)
    state["axes_gpu"] = torch.tensor(state["axes"], device="cuda")
    if case["kv"] == "e4m3":
        state["ks"] = torch.rand(Hkv, generator=g, device="cuda") * 0.02 + 0.01
        state["vs"] = torch.rand(Hkv, generator=g, device="cuda") * 0.02 + 0.01
    if case["clear"]:
        state["w"] = torch.rand(pages, Hkv, P, generator=g, device="cuda")
    if case["packed"]:
        state["cu"] = _i32([sum(new[:b]) for b in range(B + 1)])
    else:
        S = case["S"]
        for n in ("q", "k", "v"):
            state[n] = state[n].unflatten(0, (B, S))
        state["pos"] = state["pos"].unflatten(1, (B, S))
    return state


def _padded(pool, bt, width_tokens):
    """Every sequence's tokens in order, [B, tokens, Hkv, D], with whatever the table's unused entries point at behind them."""
    P = pool.shape[1]
    n = max(1, -(-width_tokens // P))
    return pool[bt[:, :n].long()].flatten(1, 2)


def _prepare_weights(case, g):
    B, Hq, Hkv, P, Sq = case["B"], case["Hq"], case["Hkv"], case["P"], case["Sq"]
    lens = _lens(case, case["lo"], case["hi"], 1)
    bt, pages = _table(lens, P, 2, g)
    e4m3 = case["kv"] == "e4m3"
    state = dict(op="weights", kc=_pool((pages, P, Hkv, D), case["kv"], g, 4.0 if e4m3 else 1.0), bt=bt,
                 lens=_i32(lens), most=max(lens), causal=case["causal"], ks=None,
                 q=torch.randn(B, Sq, Hq, D, generator=g, device="cuda", dtype=torch.bfloat16),
                 # what earlier steps left: of the size of one row's mean weight
                 w=torch.rand(pages, Hkv, P, generator=g, device="cuda") / max(lens))
    if e4m3:
        state["ks"] = torch.rand(Hkv, generator=g, device="cuda") * 0.1 + 0.2
    state["lse"] = torch.logsumexp(_scores(state, slice(0, B)), -1).unflatten(2, (Sq, Hq // Hkv)).permute(
        0, 1, 3, 2).reshape(B, Hq, Sq).contiguous()
    return state


def _prepare_evict(case, g):
    Hkv, P = case["Hkv"], case["P"]
    lens = _lens(case, case["lo"], case["hi"], 1)
    bt, pages = _table(lens, P, 2, g)
    # sums of attention weights: a long tail, and newer tokens that nobody has looked at yet (ties at zero)
    w = torch.empty(pages, Hkv, P, device="cuda").log_normal_(-6.0, 2.0, generator=g)
    w = torch.where(torch.rand(pages, Hkv, P, generator=g, device="cuda") < 0.05, 0.0, w)
    return dict(op="evict", kc=_pool((pages, P, Hkv, D), case["kv"], g), vc=_pool((pages, P, Hkv, D), case["kv"], g),
                w=w, w_out=torch.zeros_like(w), bt=bt, lens=_i32(lens), most=max(lens), keep=case["keep"],
                sinks=case["sinks"], recent=case["recent"])


def _prepare_cross(case, g):
    Hq, Hkv, P = case["Hq"], case["Hkv"], case["P"]
    lens, new = _lens(case, case["lo"], case["hi"], 1), _lens(case, case["qlo"], case["qhi"], 2)
    bt, pages = _table(lens, P, 2, g)
    T = sum(new)
    return dict(op="cross", kc=_pool((pages, P, Hkv, D), "bf16", g), vc=_pool((pages, P, Hkv, D), "bf16", g), bt=bt,
                lens=_i32(lens), most=max(lens), new=max(new), cu=_i32([sum(new[:b]) for b in range(len(new) + 1)]),
                q=torch.randn(T, Hq, D, generator=g, device="cuda", dtype=torch.bfloat16))


# ---------------------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------------------

def run(s):
    if own:
        return _own(s)
    return {"rope": _plain_rope, "weights": _plain_weights, "evict": _plain_evict, "cross": _plain_cross}[s["op"]](s)


def _own(s):
    import mx_flash_attn_kernel_opt__b200 as pgqa
    if s["op"] == "rope":
        q = pgqa.rope_append_kv(s["q"], s["k"], s["v"], s["kc"], s["vc"], s["bt"], s["lens"], s["cos"], s["sin"],
                                positions=s["pos"], axes=s["axes"], interleaved=s["interleaved"], cu_seqlens=s["cu"],
                                weights=s["w"], k_scale=s["ks"], v_scale=s["vs"])
        return [q, s["kc"], s["vc"]] + ([s["w"]] if s["w"] is not None else [])
    if s["op"] == "weights":
        return pgqa.accumulate_weights(s["q"], s["kc"], s["bt"], s["lens"], s["lse"], s["w"], causal=s["causal"],
                                       k_scale=s["ks"])
    if s["op"] == "evict":
        kept, lens = pgqa.evict_kv(s["kc"], s["vc"], s["w"], s["bt"], s["lens"], s["keep"], sinks=s["sinks"],
                                   recent=s["recent"], weights_out=s["w_out"])
        return [kept, lens, s["kc"], s["vc"], s["w_out"]]
    return list(pgqa.cross_attention(s["q"], s["kc"], s["vc"], s["bt"], s["lens"], cu_seqlens_q=s["cu"],
                                     return_lse=True))


def _turn(x, c, s, R, interleaved):
    """The first R elements of each head turned, pair by pair."""
    t = x[..., :R]
    if interleaved:
        a, b = t[..., 0::2], t[..., 1::2]
        y = torch.stack([a * c - b * s, b * c + a * s], -1).flatten(-2)
    else:
        a, b = t[..., :R // 2], t[..., R // 2:]
        y = torch.cat([a * c - b * s, b * c + a * s], -1)
    return torch.cat([y, x[..., R:]], -1)


def _plain_rope(s):
    B, P = s["bt"].shape[0], s["kc"].shape[1]
    R = 2 * s["cos"].shape[1]
    lead = s["q"].shape[:-2]
    T = s["pos"].shape[1:].numel()
    flat = lambda x: x.reshape(T, *x.shape[len(lead):])  # noqa: E731
    if s["cu"] is not None:
        token = torch.arange(T, device="cuda", dtype=torch.int32)
        b = torch.searchsorted(s["cu"], token, right=True) - 1
        t = token - s["cu"][b] + s["lens"][b]
    else:
        b = torch.arange(B, device="cuda").unsqueeze(1).expand(lead).reshape(T)
        t = (s["lens"].unsqueeze(1) + torch.arange(lead[1], device="cuda")).reshape(T)
    page, slot = s["bt"][b, (t // P).long()].long(), (t % P).long()
    at = s["pos"].flatten(1)[s["axes_gpu"]].long().t()                       # [T, R / 2]
    pair = torch.arange(R // 2, device="cuda")
    c, n = s["cos"][at, pair].float().unsqueeze(1), s["sin"][at, pair].float().unsqueeze(1)
    q = _turn(flat(s["q"]).float(), c, n, R, s["interleaved"]).to(torch.bfloat16).reshape(s["q"].shape)
    k, v = _turn(flat(s["k"]).float(), c, n, R, s["interleaved"]), flat(s["v"])
    if s["ks"] is not None:
        k = (k / s["ks"][:, None]).clamp(-448, 448)
        v = (v.float() / s["vs"][:, None]).clamp(-448, 448)
        # bytes: index_put_ is not defined on 8-bit floats
        s["kc"].view(torch.uint8)[page, slot] = k.to(FP8).view(torch.uint8)
        s["vc"].view(torch.uint8)[page, slot] = v.to(FP8).view(torch.uint8)
    else:
        s["kc"][page, slot] = k.to(torch.bfloat16)
        s["vc"][page, slot] = v
    out = [q, s["kc"], s["vc"]]
    if s["w"] is not None:
        s["w"][page, :, slot] = 0.0
        out.append(s["w"])
    return out


def _scores(s, seqs):
    """scale * q.k of sequences `seqs`, [B, Hkv, Sq * g, tokens], -inf where a row does not see the token."""
    q, lens = s["q"][seqs], s["lens"][seqs]
    B, Sq, Hq, _ = q.shape
    Hkv = s["kc"].shape[2]
    k = _padded(s["kc"], s["bt"][seqs], s["most"]).to(torch.float32).permute(0, 2, 3, 1)      # [B, Hkv, D, tokens]
    if s["ks"] is not None:
        k = k * s["ks"][:, None, None]
    qf = q.float().unflatten(2, (Hkv, Hq // Hkv)).permute(0, 2, 1, 3, 4).flatten(2, 3)        # [B, Hkv, Sq * g, D]
    x = torch.matmul(qf, k) / math.sqrt(D)
    t = torch.arange(x.shape[-1], device="cuda")
    last = lens[:, None].expand(B, Sq)
    if s["causal"]:
        last = last - Sq + 1 + torch.arange(Sq, device="cuda")
    sees = t < last.repeat_interleave(Hq // Hkv, 1)[:, :, None]                              # [B, Sq * g, tokens]
    return x.masked_fill(~sees[:, None], -math.inf)


def _plain_weights(s):
    B, Sq, Hq, _ = s["q"].shape
    Hkv, P = s["kc"].shape[2], s["kc"].shape[1]
    lse = s["lse"].unflatten(1, (Hkv, Hq // Hkv)).transpose(2, 3).flatten(2, 3).unsqueeze(-1)
    # a row that sees nothing has a log-sum-exp of -inf and no weight to give
    w = torch.exp(_scores(s, slice(0, B)) - lse.masked_fill(lse == -math.inf, 0.0)).sum(2)    # [B, Hkv, tokens]
    t = torch.arange(w.shape[-1], device="cuda")
    b, t = torch.nonzero(t < s["lens"][:, None], as_tuple=True)
    page = s["bt"][b, t // P].long()
    s["w"][page, :, t % P] += w[b, :, t]
    return s["w"]


def _plain_evict(s):
    lens, keep, sinks, recent = s["lens"].long(), s["keep"], s["sinks"], s["recent"]
    B, Hkv, P = lens.shape[0], s["w"].shape[1], s["w"].shape[2]
    w = s["w"][s["bt"].long()].transpose(1, 2).flatten(2)                                     # [B, Hkv, tokens]
    t = torch.arange(w.shape[-1], device="cuda")
    middle = (t >= sinks) & (t < (lens - recent)[:, None])
    order = torch.sort(torch.where(middle[:, None], w, -1.0), dim=-1, descending=True, stable=True).indices
    n = min(keep - sinks - recent, w.shape[-1])
    j = torch.arange(keep, device="cuda")
    ends = torch.cat([torch.arange(sinks, device="cuda").expand(B, sinks),
                      (lens - recent)[:, None] + torch.arange(recent, device="cuda")], 1)
    cut = torch.cat([ends[:, None].expand(B, Hkv, sinks + recent), order[..., :n]], -1).sort(-1).values
    if cut.shape[-1] < keep:
        cut = torch.cat([cut, cut.new_zeros(B, Hkv, keep - cut.shape[-1])], -1)
    short = (lens <= keep)[:, None, None]
    kept = torch.where(short, torch.where(j < lens[:, None], j, -1)[:, None], cut)
    b, h, j = torch.nonzero(kept >= 0, as_tuple=True)
    src, P64 = kept[b, h, j], s["bt"].long()
    here, there = (P64[b, src // P], src % P), (P64[b, j // P], j % P)
    for pool in (s["kc"], s["vc"]):
        raw = pool.view(torch.uint8) if pool.dtype == FP8 else pool
        raw[there[0], there[1], h] = raw[here[0], here[1], h]
    s["w_out"][there[0], h, there[1]] = s["w"][here[0], h, here[1]]
    return [kept.to(torch.int32), lens.clamp(max=keep).to(torch.int32), s["kc"], s["vc"], s["w_out"]]


def _plain_cross(s):
    T, Hq, _ = s["q"].shape
    Hkv, B, Sq = s["kc"].shape[2], s["bt"].shape[0], s["new"]
    token = torch.arange(T, device="cuda", dtype=torch.int32)
    b = torch.searchsorted(s["cu"], token, right=True) - 1
    i = (token - s["cu"][b]).long()
    q = torch.zeros(B, Sq, Hq, D, device="cuda")
    q[b, i] = s["q"].float()
    q = q.unflatten(2, (Hkv, Hq // Hkv)).permute(0, 2, 3, 1, 4).flatten(2, 3)                 # [B, Hkv, g * Sq, D]
    k, v = (_padded(s[n], s["bt"], s["most"]).float().transpose(1, 2) for n in ("kc", "vc"))  # [B, Hkv, tokens, D]
    hidden = torch.arange(k.shape[2], device="cuda") >= s["lens"][:, None]
    v = v.masked_fill(hidden[:, None, :, None], 0.0)
    x = torch.matmul(q, k.transpose(2, 3)).div_(math.sqrt(D)).masked_fill_(hidden[:, None, None], -math.inf)
    top = x.amax(-1, keepdim=True)
    top = top.masked_fill(top == -math.inf, 0.0)                                             # no key: all weights 0
    x = x.sub_(top).exp_()
    total = x.sum(-1, keepdim=True)
    out = torch.matmul(x, v) / total.masked_fill(total == 0.0, 1.0)
    lse = (top + total.log()).squeeze(-1)
    back = lambda y: y.unflatten(2, (Hq // Hkv, Sq)).flatten(1, 2).transpose(1, 2)[b, i]      # noqa: E731
    return [back(out).to(torch.bfloat16), back(lse).t().contiguous()]


# ---------------------------------------------------------------------------------------
# work and exact values
# ---------------------------------------------------------------------------------------

def _pages_read(lens, P):
    return 4 * sum(-(-n // P) for n in lens) + 4 * len(lens)


def work(case):
    Hkv, P = case["Hkv"], case["P"]
    size = 1 if case.get("kv") == "e4m3" else 2
    lens = _lens(case, case["lo"], case["hi"], 1)
    if case["op"] == "rope":
        T, R = sum(_new_lens(case)), case["R"]
        heads = case["Hq"] + 2 * Hkv
        entry = 4 if case["table"] == "fp32" else 2
        b = T * (heads * D * 2 + case["Hq"] * D * 2 + 2 * Hkv * D * size + (Hkv * 4 if case["clear"] else 0))
        b += T * 4 * (1 if case["axes"] == "one" else 3) + min(T, 8192) * R * entry
        return {"bytes": b, "flops": 3 * T * R * (case["Hq"] + Hkv)}
    if case["op"] == "weights":
        n, Hq, Sq = sum(lens), case["Hq"], case["Sq"]
        b = n * Hkv * (D * size + 8) + case["B"] * Sq * Hq * (D * 2 + 4) + _pages_read(lens, P)
        return {"bytes": b, "flops": 2 * n * Hq * Sq * D}
    if case["op"] == "evict":
        b = _pages_read(lens, P)
        keep, fixed = case["keep"], case["sinks"] + case["recent"]
        for n in lens:
            b += Hkv * min(n, keep) * (4 + 4 + 4)                       # kept's entry, its weight read and written
            if n > keep:
                gone = n - keep
                still = case["sinks"] + (n - fixed - gone) / (gone + 1)  # rows before the first that goes, on average
                b += Hkv * ((n - fixed) * 4 + (keep - still) * 2 * 2 * D * size)
        return {"bytes": b, "flops": 0}
    new = _lens(case, case["qlo"], case["qhi"], 2)
    pairs = sum(a * b for a, b in zip(lens, new))
    b = sum(lens) * Hkv * D * 4 + sum(new) * case["Hq"] * (D * 4 + 4) + _pages_read(lens, P)
    return {"bytes": b, "flops": 4 * pairs * case["Hq"] * D}


def _rows64(pool, bt, b, n, h, scale=None):
    """Head h's first n rows of sequence b, in 64 bits."""
    P = pool.shape[1]
    x = pool[bt[b, :max(1, -(-n // P))].long(), :, h].to(torch.float32).double().flatten(0, 1)[:n]
    return x if scale is None else x * scale[h].double()


def exact(case, seed):
    s = prepare(case, seed)
    B, Hkv, P = case["B"], case["Hkv"], case["P"]
    lens, bt = s["lens"].tolist(), s["bt"]
    if case["op"] == "rope":
        new = _new_lens(case)
        T, R = sum(new), case["R"]
        i = torch.arange(R // 2, device="cuda")
        row = s["pos"].reshape(-1, T).long()[torch.tensor(s["axes"], device="cuda")].t()
        z = torch.complex(s["cos"].double()[row, i], s["sin"].double()[row, i])[:, None]

        def spin(x):
            y = x.reshape(T, -1, D).double().clone()
            xs, ys = (slice(0, R, 2), slice(1, R, 2)) if s["interleaved"] else (slice(0, R // 2), slice(R // 2, R))
            w = torch.complex(y[..., xs], y[..., ys]) * z
            y[..., xs], y[..., ys] = w.real, w.imag
            return y

        at = torch.tensor([n + j for n, m in zip(lens, new) for j in range(m)], device="cuda")
        seq = torch.tensor([b for b, m in enumerate(new) for _ in range(m)], device="cuda")
        page = bt[seq, at // P].long()
        out = [spin(s["q"]).reshape(s["q"].shape)]
        for pool, x, f in ((s["kc"], spin(s["k"]), s["ks"]), (s["vc"], s["v"].reshape(T, Hkv, D).double(), s["vs"])):
            y = pool.to(torch.float32).double()
            y[page, at % P] = x if f is None else x / f.double()[:, None]
            out.append(y)
        if s["w"] is not None:
            y = s["w"].double()
            y[page, :, at % P] = 0.0
            out.append(y)
        return out
    if case["op"] == "weights":
        if B * Hkv > 2100:
            return None
        Sq, Hq = case["Sq"], case["Hq"]
        g, y = Hq // Hkv, s["w"].double()
        for b in range(B):
            n = lens[b]
            t = torch.arange(n, device="cuda")
            page = bt[b, t // P].long()
            for h in range(Hkv):
                k = _rows64(s["kc"], bt, b, n, h, s["ks"])
                for i in range(Sq):
                    m = max(0, n - Sq + 1 + i) if case["causal"] else n
                    x = k[:m] @ s["q"][b, i, h * g:(h + 1) * g].double().t() / math.sqrt(D)
                    y[page[:m], h, t[:m] % P] += torch.exp(x - s["lse"][b, h * g:(h + 1) * g, i].double()).sum(1)
        return y
    if case["op"] == "evict":
        keep, sinks, recent = case["keep"], case["sinks"], case["recent"]
        kept = torch.full((B, Hkv, keep), -1, dtype=torch.int32)
        kc, vc, w_out = s["kc"].cpu(), s["vc"].cpu(), s["w_out"].double().cpu()
        tab, w = bt.cpu().long(), s["w"].cpu()
        old = [x.clone() for x in (kc, vc)]
        for b in range(B):
            n = lens[b]
            t = torch.arange(n)
            for h in range(Hkv):
                row = w[tab[b, t // P], h, t % P].double()
                if n > keep:
                    mid = row[sinks:n - recent]
                    # highest first, the lowest index first among equals
                    best = sorted(range(len(mid)), key=mid.neg().tolist().__getitem__)[:keep - sinks - recent]
                    stay = list(range(sinks)) + sorted(sinks + i for i in best) + list(range(n - recent, n))
                else:
                    stay = list(range(n))
                a = torch.tensor(stay, dtype=torch.long)
                j = torch.arange(len(stay))
                kept[b, h, :len(stay)] = a.to(torch.int32)
                for pool, was in zip((kc, vc), old):
                    raw, src = (pool.view(torch.uint8), was.view(torch.uint8)) if pool.dtype == FP8 else (pool, was)
                    raw[tab[b, j // P], j % P, h] = src[tab[b, a // P], a % P, h]
                w_out[tab[b, j // P], h, j % P] = row[a]
        return [kept, torch.tensor([min(n, keep) for n in lens], dtype=torch.int32), kc, vc, w_out]
    Hq, new = case["Hq"], _lens(case, case["qlo"], case["qhi"], 2)
    g, out = Hq // Hkv, torch.zeros(s["q"].shape, device="cuda", dtype=torch.float64)
    lse = torch.full((Hq, s["q"].shape[0]), -math.inf, device="cuda", dtype=torch.float64)
    first = 0
    for b in range(B):
        rows = slice(first, first + new[b])
        first += new[b]
        if not lens[b] or not new[b]:
            continue
        for h in range(Hkv):
            k, v = (_rows64(s[p], bt, b, lens[b], h) for p in ("kc", "vc"))
            for a in range(h * g, (h + 1) * g):
                x = s["q"][rows, a].double() @ k.t() / math.sqrt(D)
                lse[a, rows] = torch.logsumexp(x, 1)
                out[rows, a] = torch.softmax(x, 1) @ v
    return [out, lse]
