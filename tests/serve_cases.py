"""Inputs of the serving tests: caches, tables and probabilities from a seed, on the CPU."""
import torch

from fpa import PagedCache

STORE = {"f16": torch.float16, "f32": torch.float32, "e4m3": torch.float8_e4m3fn}


def tables(lengths, width, pages, g):
    """(B, width) int32: each sequence's pages in random order, -1 behind them."""
    ids = torch.randperm(pages, generator=g).to(torch.int32)
    t = torch.full((len(lengths), width), -1, dtype=torch.int32)
    at = 0
    for b, n in enumerate(lengths):
        k = -(-n // 64)
        t[b, :k] = ids[at:at + k]
        at += k
    assert at <= pages
    return t


def poison(c):
    """Fills a cache with what must never be read: NaN, infinities and large exponents."""
    if c.dtype == torch.float8_e4m3fn:
        c.k.view(torch.uint8).fill_(0x7f)
        c.v.view(torch.uint8).fill_(0xff)
        c.k_exp.fill_(60)
        c.v_exp.fill_(60)
    else:
        c.k.fill_(float("nan"))
        c.v.fill_(float("inf"))
        c.v[:, :, ::2] = float("nan")
    c.phi.fill_(float("-inf"))
    c.psi.fill_(float("nan"))
    c.phi_min.fill_(float("-inf"))


def rows(B, H, N, D, dtype, g, phi_scale=0.3):
    """k, v (B, H, N, D) as views of a projection's output, phi a walk and psi near it."""
    x = torch.randn(B, N, 2, H, D, generator=g).to(dtype)
    k, v = x.permute(2, 0, 3, 1, 4)
    phi = phi_scale * torch.randn(B, H, N, generator=g).cumsum(-1)
    return k, v, phi, phi + 0.5 * torch.randn(B, H, N, generator=g)


def filled(B, H, D, lengths, store, q, seed, prefix=0, width=None, device="cpu", impl=None):
    """A poisoned cache with B sequences of `lengths` (and a shared prefix) appended; everything else it takes.

    Returns (cache, table, lengths, prefix pages or None, q of N = 16 rows, beta)."""
    g = torch.Generator().manual_seed(seed)
    every = list(lengths) + ([prefix] if prefix else [])
    need = sum(-(-n // 64) for n in every)
    width = width or max(1, max(-(-n // 64) for n in every))
    cache = PagedCache(need + 2, H, D, STORE[store], device=device)
    poison(cache)
    table = tables(every, max(width, -(-prefix // 64)), need + 2, g)
    dt = STORE[q]
    k, v, phi, psi = (t.to(device) for t in rows(len(every), H, max(1, max(every)), D, dt, g))
    dev_table = table.to(device)
    count = torch.tensor(every, dtype=torch.int32, device=device)
    cache.append(k, v, phi, psi, dev_table, torch.zeros_like(count), count, impl=impl)
    x = torch.randn(B, 16, 3, H, D, generator=g).to(dt)
    beta = torch.rand(H, generator=g) + 0.5
    pre = dev_table[B, :-(-prefix // 64)].contiguous() if prefix else None
    return cache, dev_table[:B, :width].contiguous(), count[:B].contiguous(), pre, x.permute(2, 0, 3, 1, 4)[0].to(device), beta.to(device)


def probabilities(B, N, V, dtype, seed, draft=True, sharp=2.0):
    """target, draft (or None), tokens drawn from it, accept_u, sample_u."""
    g = torch.Generator().manual_seed(seed)
    z = sharp * torch.randn(B, N + 1, V, generator=g)
    near = torch.softmax(z[:, :N] + 0.7 * torch.randn(B, N, V, generator=g), -1)
    tokens = torch.multinomial(near.reshape(B * N, V), 1, generator=g).view(B, N) if N else torch.zeros(B, 0, dtype=torch.int64)
    return (torch.softmax(z, -1).to(dtype), near.to(dtype) if draft else None, tokens,
            torch.rand(B, N, generator=g), torch.rand(B, generator=g))
