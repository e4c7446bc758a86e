"""The serving operators on the HIP kernels: argument structs, outputs and scratch (the binding of ``cache.py`` and
``drafts.py``).  Everything is enqueued on torch's current stream of the cache's device, with no host sync."""
import functools

import torch

from . import _lib
from ._hip import counters, device_guard, workspace

_CODES = {torch.float16: _lib.FPA_F16, torch.float32: _lib.FPA_F32, torch.float8_e4m3fn: _lib.FPA_E4M3}


def _pages(c):
    if c._packed is None:
        c._packed = _lib.PAGES_PACK.pack(
            c.pages, c.n_heads, c.d_head, _CODES[c.dtype],
            *(t.data_ptr() if t is not None else 0 for t in (c.k, c.v, c.phi, c.psi, c.phi_min, c.k_exp, c.v_exp)))
    return c._packed


def _unit(t):
    """t with unit stride along its last axis (length one aside, where the stride means nothing)."""
    return t if t.stride(-1) == 1 else t.contiguous()


def rows(t):
    """(t, its strides): t itself when the kernels can read its rows in 16-byte pieces, else a fresh copy (also of a contiguous
    tensor whose first element is not aligned)."""
    s, ce = t.stride(), 8 if t.dtype is torch.float16 else 4
    if not (s[3] == 1 and t.data_ptr() % 16 == 0 and s[0] % ce == 0 and s[1] % ce == 0 and s[2] % ce == 0
            and 0 <= s[2] * 64 * t.element_size() < 2 ** 31):
        t = t.clone(memory_format=torch.contiguous_format)
        s = t.stride()
    return t, s


def _ptr(t):
    return 0 if t is None else t.data_ptr()


def append(c, k, v, phi, psi, table, start, counts):
    (k, ks), (v, vs) = rows(k), rows(v)
    phi = phi if phi.dtype is torch.float32 else phi.float()
    psi = psi if psi.dtype is torch.float32 else psi.float()
    table, start = _unit(table), start.contiguous()
    counts = None if counts is None else counts.contiguous()
    shape, dev = k.shape, c.device
    a = _lib.FpaAppendArgs.from_buffer_copy(_lib.APPEND_PACK.pack(
        _pages(c), shape[0], shape[2], table.shape[1], _CODES[k.dtype],
        k.data_ptr(), *ks, v.data_ptr(), *vs, phi.data_ptr(), *phi.stride(), psi.data_ptr(), *psi.stride(),
        table.data_ptr(), table.stride(0), start.data_ptr(), _ptr(counts)))
    with device_guard(dev):
        _lib.check(_lib.lib().fpa_cache_append(a, _lib.stream_of(dev)))


def read(c, table, start, n, counts, dtype):
    B, H, D, dev = table.shape[0], c.n_heads, c.d_head, c.device
    table, start, counts = _unit(table), start.contiguous(), None if counts is None else counts.contiguous()
    with device_guard(dev):
        kv = torch.empty((2, B, H, n, D), dtype=dtype, device=dev)
        pp = torch.empty((2, B, H, n), dtype=torch.float32, device=dev)
        at, half, ap, hp = kv.data_ptr(), B * H * n * D * kv.element_size(), pp.data_ptr(), B * H * n * 4
        a = _lib.FpaReadArgs.from_buffer_copy(_lib.READ_PACK.pack(
            _pages(c), B, n, table.shape[1], _CODES[dtype], at, at + half, ap, ap + hp,
            table.data_ptr(), table.stride(0), start.data_ptr(), _ptr(counts)))
        _lib.check(_lib.lib().fpa_cache_read(a, _lib.stream_of(dev)))
    return *kv.unbind(0), *pp.unbind(0)


@functools.lru_cache(maxsize=1024)
def _attend_scratch(B, H, N, D, P, prefix_length, dtype, store):
    """(workspace bytes, counters) of a call of this shape."""
    L = _lib.lib()
    return (L.fpa_attend_workspace_bytes(B, H, N, D, P, prefix_length, _CODES[dtype], _CODES[store]), L.fpa_attend_counts(B, H, N))


def attend(q, c, beta, table, lengths, prefix, prefix_length):
    B, H, N, D = q.shape
    dev, dtype = q.device, q.dtype
    (q, qs), beta, table, lengths = rows(q), beta.contiguous(), _unit(table), lengths.contiguous()
    prefix = None if prefix is None or prefix_length == 0 else prefix.contiguous()
    P = table.shape[1]
    nws, ncounts = _attend_scratch(B, H, N, D, P, prefix_length, dtype, c.dtype)
    os = (N * H * D, D, H * D, 1)  # (B, N, H, D) in memory
    with device_guard(dev):
        o = torch.empty_strided((B, H, N, D), os, dtype=dtype, device=dev)
        # held until the launch: a captured graph's pool would give the memory of one that is gone to the next
        ws, counts = workspace(dev, nws) if nws else None, counters(dev, ncounts)
        a = _lib.FpaAttendArgs.from_buffer_copy(_lib.ATTEND_PACK.pack(
            _pages(c), B, N, P, _CODES[dtype], q.data_ptr(), *qs, o.data_ptr(), *os, beta.data_ptr(),
            table.data_ptr(), table.stride(0), lengths.data_ptr(), _ptr(prefix), prefix_length,
            _ptr(ws), counts.data_ptr()))
        _lib.check(_lib.lib().fpa_attend(a, _lib.stream_of(dev)))
    return o


@functools.lru_cache(maxsize=1024)
def _verify_ws_bytes(B, V):
    return _lib.lib().fpa_verify_workspace_bytes(B, V)


def verify(target, draft, tokens, accept_u, sample_u):
    (B, N), V, dev = tokens.shape, target.shape[2], target.device
    target, draft = _unit(target), None if draft is None else _unit(draft)
    tokens, accept_u, sample_u = _unit(tokens), _unit(accept_u), sample_u.contiguous()
    ts, ds = target.stride(), (0, 0) if draft is None else draft.stride()
    with device_guard(dev):
        both = torch.empty(B * (N + 2), dtype=torch.int64, device=dev)  # both results in one allocation
        at = both.data_ptr()
        ws, counts = workspace(dev, _verify_ws_bytes(B, V)), counters(dev, B)  # held until the launch, as above
        a = _lib.FpaVerifyArgs.from_buffer_copy(_lib.VERIFY_PACK.pack(
            B, N, V, _CODES[target.dtype], target.data_ptr(), ts[0], ts[1], _ptr(draft), ds[0], ds[1],
            tokens.data_ptr(), tokens.stride(0), accept_u.data_ptr(), accept_u.stride(0), sample_u.data_ptr(), at, at + 8 * B,
            ws.data_ptr(), counts.data_ptr()))
        _lib.check(_lib.lib().fpa_verify(a, _lib.stream_of(dev)))
    return both[:B], both[B:].view(B, N + 1)
