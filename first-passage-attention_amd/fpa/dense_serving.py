"""PyTorch path of the serving operators: ``impl="reference"`` of ``cache.py`` and ``drafts.py``.

Any device, float32 inside (float64 for the drafts), (B, H, N, T) tensors materialised.  The same results as the
kernels' up to rounding, the same codes for 8-bit caches, and the same tokens.
"""
import math

import torch

PAGE = 64
EXP_MIN, EXP_MAX = -60, 60
_INF = math.inf


def quantise(x):
    """(e4m3 codes, int8 exponents) of rows x (..., D) float32: exponent clamp(ceil(log2(max |x| / 448)), -60, 60), -60
    for zeros; codes rounded to nearest even, saturating; NaN stays."""
    top = torch.where(x.isnan(), 0.0, x.abs()).amax(-1)
    m, e = torch.frexp(top)  # top = m 2^e; 448 = 0.875 * 2^9
    e = torch.where(m > 0.875, e - 8, e - 9)
    e = torch.where(top.isinf(), EXP_MAX, torch.where(top > 0, e, EXP_MIN)).clamp(EXP_MIN, EXP_MAX)
    scaled = torch.ldexp(x, -e.unsqueeze(-1))
    return scaled.clamp(-448.0, 448.0).to(torch.float8_e4m3fn), e.to(torch.int8)


def _places(cache, table, start, n):
    """(page, slot, named) of positions start[b] + i, (B, n); page 0 where the table names none."""
    pos = start.long().unsqueeze(1) + torch.arange(n, device=table.device)
    P = table.shape[1]
    named = (start >= 0).unsqueeze(1) & (pos < P * PAGE)
    pos = pos.clamp(0, P * PAGE - 1)
    page = table.gather(1, pos // PAGE).long()
    named &= (page >= 0) & (page < cache.pages)
    return torch.where(named, page, 0), pos % PAGE, named


def append(c, k, v, phi, psi, table, start, counts):
    B, H, N, D = k.shape
    i = torch.arange(N, device=k.device)
    page, slot, named = _places(c, table, start, N)
    n = torch.full_like(start, N) if counts is None else counts.clamp(max=N)
    b, j = (named & (i < n.unsqueeze(1))).nonzero(as_tuple=True)
    page, slot = page[b, j], slot[b, j]
    kr, vr = k[b, :, j], v[b, :, j]  # (M, H, D)
    if c.k_exp is not None:
        (kr, ke), (vr, ve) = quantise(kr.float()), quantise(vr.float())
        c.k_exp[page, :, slot], c.v_exp[page, :, slot] = ke, ve
        c.k.view(torch.uint8)[page, :, slot] = kr.view(torch.uint8)
        c.v.view(torch.uint8)[page, :, :, slot] = vr.view(torch.uint8)
    else:
        c.k[page, :, slot], c.v[page, :, :, slot] = kr, vr
    c.phi[page, :, slot], c.psi[page, :, slot] = phi[b, :, j].float(), psi[b, :, j].float()
    # phi_min of the written pages: over the positions up to the last one written
    top = torch.full((c.pages,), -1, dtype=torch.long, device=k.device).scatter_reduce(0, page, slot, "amax")
    some = (top >= 0).nonzero(as_tuple=True)[0]
    held = torch.where(torch.arange(PAGE, device=k.device) <= top[some].view(-1, 1, 1), c.phi[some], _INF)
    c.phi_min[some] = held.amin(-1)


def _rows(c, page, slot):
    """k, v (B, n, H, D) and phi, psi (B, n, H) float32 at (page, slot) (B, n)."""
    k, v = c.k.float()[page, :, slot], c.v.float()[page, :, :, slot]
    if c.k_exp is not None:
        k = torch.ldexp(k, c.k_exp[page, :, slot].to(torch.int32).unsqueeze(-1))
        v = torch.ldexp(v, c.v_exp[page, :, slot].to(torch.int32).unsqueeze(-1))
    return k, v, c.phi[page, :, slot], c.psi[page, :, slot]


def read(c, table, start, n, counts, dtype):
    page, slot, named = _places(c, table, start, n)
    m = torch.full_like(start, n) if counts is None else counts
    there = (torch.arange(n, device=table.device) < m.unsqueeze(1)).unsqueeze(-1)
    k, v, phi, psi = _rows(c, page, slot)

    def only(x):
        t = there if x.dim() == 3 else there.unsqueeze(-1)
        ok = named.view(*named.shape, *[1] * (x.dim() - 2))
        return torch.where(t, torch.where(ok, x, math.nan), 0.0).transpose(1, 2)
    k, v, phi, psi = (only(x) for x in (k, v, phi, psi))
    return k.to(dtype).contiguous(), v.to(dtype).contiguous(), phi.contiguous(), psi.contiguous()


def attention(q, c, beta, table, lengths, prefix=None, prefix_length=0):
    B, H, N, D = q.shape
    dev, P = q.device, prefix_length
    cap = table.shape[1] * PAGE
    L = lengths.long().clamp(0, cap)
    pos = torch.arange(cap, device=dev)
    page, slot, named = _places(c, table, torch.zeros_like(lengths), cap)
    k, v, phi, psi = (x.transpose(1, 2) for x in _rows(c, page, slot))  # (B, H, T, ..)
    used = pos < L.unsqueeze(1)
    lost = (lengths > cap) | (used & ~named).any(1)  # a page that is needed and not there
    t = L.unsqueeze(1) - N + torch.arange(N, device=dev)  # (B, N)
    if P:
        zero = torch.zeros(1, dtype=torch.int32, device=dev)
        pp, ps, pn = _places(c, prefix.unsqueeze(0), zero, P)
        pre = [x.transpose(1, 2).expand(B, *x.transpose(1, 2).shape[1:]) for x in _rows(c, pp, ps)]
        k, v, phi, psi = (torch.cat((a, b), 2) for a, b in zip(pre, (k, v, phi, psi)))
        lost = lost | ~pn.all()
    s = torch.arange(P + cap, device=dev) - P  # own position; the prefix before 0
    there = ((s <= t.unsqueeze(-1)) & (t >= 0).unsqueeze(-1))[:, None]  # (B, 1, N, P + T)
    # min of phi over the later positions up to t
    low = torch.where(there, phi.float().unsqueeze(2), _INF).flip(-1).cummin(-1).values.flip(-1)
    low = torch.cat((low[..., 1:], torch.full_like(low[..., :1], _INF)), -1)
    bias = beta.view(1, H, 1, 1) * (low - psi.unsqueeze(2)).clamp(max=0.0)
    logits = q.float() @ k.transpose(-1, -2).contiguous() * D ** -0.5 + bias
    logits = torch.where(there, logits, -_INF)
    top = logits.amax(-1, keepdim=True)
    p = torch.where(there, torch.exp(logits - torch.where(top == -_INF, 0.0, top)), 0.0)
    # what a row does not see is not multiplied: values that are not finite go to the rows that see them
    fine = v.isfinite()
    o = p @ torch.where(fine, v, 0.0).contiguous()
    if not bool(fine.all()):
        for b, h, at in (~fine).any(-1).nonzero().tolist():
            sees = there[b, 0, :, at]
            rest = torch.where(fine[b, h, at], 0.0, v[b, h, at])
            o[b, h] = torch.where(sees.unsqueeze(-1) & ~fine[b, h, at], o[b, h] + p[b, h, :, at:at + 1] * rest, o[b, h])
    total = p.sum(-1, keepdim=True)
    o = torch.where(there.any(-1, keepdim=True), o / total, 0.0)
    return torch.where(lost.view(B, 1, 1, 1), math.nan, o).to(q.dtype)


def verify(target, draft, tokens, accept_u, sample_u):
    B, N = tokens.shape
    V, dev = target.shape[2], target.device
    named = (tokens >= 0) & (tokens < V)
    at = torch.where(named, tokens, 0).unsqueeze(2)
    px = target[:, :N].gather(2, at).squeeze(2).double()
    qx = torch.ones_like(px) if draft is None else draft.gather(2, at).squeeze(2).double()
    n = (named & (accept_u.double() * qx < px)).long().cumprod(1).sum(1)
    b = torch.arange(B, device=dev)
    full = target[b, n].double().clamp(min=0.0)
    w = full
    if N:
        j = n.clamp(max=N - 1)
        if draft is None:
            less = torch.zeros_like(full).scatter_(1, at[b, j], _INF)
        else:
            less = draft[b, j].double()
        w = torch.where(((n < N) & named[b, j]).unsqueeze(1), (target[b, n].double() - less).clamp(min=0.0), full)
    total = w.sum(1, keepdim=True)
    w = torch.where((total > 0) & total.isfinite(), w, full)
    c = w.cumsum(1)
    total = c[:, -1:]
    over = (c > sample_u.double().unsqueeze(1) * total) & (w > 0)
    last = torch.where(w > 0, torch.arange(V, device=dev), -1).amax(1)  # sums that round below their target
    token = torch.where(over.any(1), over.to(torch.uint8).argmax(1), last)
    token = torch.where((total > 0).squeeze(1) & total.isfinite().squeeze(1), token, -1)
    i = torch.arange(N + 1, device=dev)
    kept = torch.cat((tokens, torch.full_like(n, -1).unsqueeze(1)), 1)
    return n, torch.where(i < n.unsqueeze(1), kept, torch.where(i == n.unsqueeze(1), token.unsqueeze(1), -1))
