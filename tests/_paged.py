"""Small paged caches for the tests of the operators around the decode."""
import torch

FP8 = torch.float8_e4m3fn


def table(lens, P, gen, spare=3, width=None):
    """Pages dealt out in random order; unused table entries name pages out of range (they
    must never be read).  Returns (block_table [B, width], num_pages)."""
    need = [-(-n // P) for n in lens]
    pages = sum(need) + spare
    ids = torch.randperm(pages, generator=gen).to(torch.int32)
    width = width or max(1, max(need) + 1)
    bt = torch.full((len(lens), width), 2 ** 30, dtype=torch.int32)
    at = 0
    for b, n in enumerate(need):
        bt[b, :n] = ids[at:at + n]
        at += n
    return bt, pages


def pool(pages, P, Hkv, gen, kv="bf16", std=1.0):
    x = torch.randn(pages, P, Hkv, 128, generator=gen) * std
    return x.to(torch.bfloat16) if kv == "bf16" else x.clamp(-448, 448).to(FP8)


def raw(x):
    """The bytes of a tensor, on the CPU (NaN patterns compare equal to themselves)."""
    return x.detach().cpu().contiguous().view(torch.uint8)


def poison_unused(x, lens, bt, P, value=float("nan")):
    """Sets every token slot past the sequences' lengths (and every unused page) to `value`."""
    keep = torch.zeros(x.shape[0], P, dtype=torch.bool)
    for b, n in enumerate(lens):
        for t in range(n):
            keep[bt[b, t // P], t % P] = True
    y = x.float()
    y[~keep] = value
    return y.to(x.dtype)
