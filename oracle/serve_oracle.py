"""Float64 oracle of the serving operators, by loops over sequences, heads and positions (test infrastructure only).

Values are read from a cache's buffers one position at a time, so nothing here shares an indexing expression with the
package.  Probabilities and sums are Python floats or float64 tensors on the CPU.
"""
import math

import torch

PAGE = 64


def e4m3_values():
    """The 127 non-negative e4m3 numbers by code."""
    out = []
    for code in range(127):
        e, m = divmod(code, 8)
        out.append(m / 512.0 if e == 0 else (1 + m / 8.0) * 2.0 ** (e - 7))
    return torch.tensor(out, dtype=torch.float64)


def nearest_e4m3(x):
    """float64 values rounded to the nearest e4m3 number (ties to the even code), saturating; NaN stays."""
    v = e4m3_values()
    a = x.abs().clamp(max=448.0)
    hi = torch.searchsorted(v, a.contiguous()).clamp(max=126)
    lo = (hi - 1).clamp(min=0)
    up, down = v[hi] - a, a - v[lo]
    pick = torch.where((up < down) | ((up == down) & (hi % 2 == 0)), hi, lo)
    return torch.where(x.isnan(), x, torch.copysign(v[pick], x))


def row_exponent(row):
    """Exponent of one row: the least e in [-60, 60] with max |row| <= 448 * 2^e; -60 for zeros."""
    top = max((abs(float(x)) for x in row if not math.isnan(float(x))), default=0.0)
    for e in range(-60, 60):
        if top <= 448.0 * 2.0 ** e:
            return e
    return 60


def quantised(x):
    """(values that the rows of x (..., D) stand for in 8 bits, exponents)."""
    rows = x.double().reshape(-1, x.shape[-1])
    exps = torch.tensor([row_exponent(r) for r in rows.tolist()], dtype=torch.float64).unsqueeze(1)
    vals = nearest_e4m3(rows * 2.0 ** -exps) * 2.0 ** exps
    return vals.view(x.shape), exps.view(x.shape[:-1]).to(torch.int8)


def position(cache, page, slot, h):
    """k, v (D,), phi, psi of one position in float64 (CPU copies of the buffers in `cache`, a dict)."""
    k, v = cache["k"][page, h, slot].double(), cache["v"][page, h, :, slot].double()
    if cache["k_exp"] is not None:
        k, v = k * 2.0 ** int(cache["k_exp"][page, h, slot]), v * 2.0 ** int(cache["v_exp"][page, h, slot])
    return k, v, float(cache["phi"][page, h, slot]), float(cache["psi"][page, h, slot])


def buffers(c):
    """CPU copies of a PagedCache's buffers."""
    names = ("k", "v", "phi", "psi", "phi_min", "k_exp", "v_exp")
    return {n: None if getattr(c, n) is None else getattr(c, n).detach().cpu().clone() for n in names}


def sequence(cache, table_row, n, h):
    rows = [position(cache, int(table_row[s // PAGE]), s % PAGE, h) for s in range(n)]
    if not rows:
        return None
    return (torch.stack([r[0] for r in rows]), torch.stack([r[1] for r in rows]),
            torch.tensor([r[2] for r in rows], dtype=torch.float64), torch.tensor([r[3] for r in rows], dtype=torch.float64))


def attend_row(q, k, v, phi, psi, beta, t):
    """o (D,) of one query at position t against keys 0 .. t."""
    low = math.inf
    bias = torch.zeros(t + 1, dtype=torch.float64)
    for s in range(t, -1, -1):
        bias[s] = float(beta) * min(0.0, low - float(psi[s]))
        low = min(low, float(phi[s]))
    logits = (k[:t + 1] @ q.double()) / math.sqrt(q.shape[-1]) + bias
    p = torch.exp(logits - logits.max())
    p = p / p.sum()
    seen = v[:t + 1]
    return (p.unsqueeze(1) * seen).sum(0)


def attention(q, cache, beta, table, lengths, prefix=None, prefix_length=0):
    """o (B, H, N, D) float64; q, beta, table, lengths on the CPU, cache as buffers() gives it."""
    B, H, N, D = q.shape
    o = torch.zeros(B, H, N, D, dtype=torch.float64)
    for h in range(H):
        pre = sequence(cache, prefix, prefix_length, h) if prefix_length else None
        for b in range(B):
            L = int(lengths[b])
            own = sequence(cache, table[b], L, h)
            if own is None:
                continue
            k, v, phi, psi = own if pre is None else [torch.cat(x) for x in zip(pre, own)]
            for i in range(N):
                t = L - N + i
                if t >= 0:
                    o[b, h, i] = attend_row(q[b, h, i], k, v, phi, psi, beta[h], prefix_length + t)
    return o


def verify(target, draft, tokens, accept_u, sample_u):
    """(accepted, out) as lists, one sequence after the other, in Python floats (fp64)."""
    B, N = tokens.shape
    V = target.shape[2]
    accepted, out = [], []
    for b in range(B):
        n, ended = 0, False
        while n < N:
            x = int(tokens[b, n])
            if not 0 <= x < V:
                ended = True
                break
            qx = 1.0 if draft is None else float(draft[b, n, x])
            if not float(accept_u[b, n]) * qx < float(target[b, n, x]):
                break
            n += 1
        p = target[b, n].double().tolist()
        w = [max(x, 0.0) for x in p]
        if n < N and not ended:
            x = int(tokens[b, n])
            d = [0.0] * V if draft is None else draft[b, n].double().tolist()
            less = [max(a - c, 0.0) for a, c in zip(p, d)]
            if draft is None:
                less[x] = 0.0
            if math.fsum(less) > 0:
                w = less
        total = math.fsum(w)
        token = -1
        if 0 < total < math.inf:
            goal, run = float(sample_u[b]) * total, 0.0
            for v, x in enumerate(w):
                run += x
                if x > 0:
                    token = v
                    if run > goal:
                        break
        accepted.append(n)
        out.append([int(tokens[b, i]) for i in range(n)] + [token] + [-1] * (N - n))
    return torch.tensor(accepted), torch.tensor(out)
