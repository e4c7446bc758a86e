"""The serving operators on the HIP kernels: argument structs, outputs and scratch (the binding of ``cache.py`` and
``drafts.py``).  Everything is enqueued on torch's current stream of the cache's device, with no host sync."""
import functools

import torch

from . import _lib
from ._hip import _rows_ok, counters, device_guard, workspace

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
    """t itself when the kernels can read its rows in 16-byte pieces, else a fresh copy (also of a contiguous tensor whose
    first element is not aligned)."""
    return t if _rows_ok(t) else t.clone(memory_format=torch.contiguous_format)


def _ptr(t):
    return 0 if t is None else t.data_ptr()


def append(c, k, v, phi, psi, table, start, counts):
    k, v, phi, psi, table = rows(k), rows(v), phi.float(), psi.float(), _unit(table)
    start, counts = start.contiguous(), None if counts is None else counts.contiguous()
    a = _lib.FpaAppendArgs.from_buffer_copy(_lib.APPEND_PACK.pack(
        _pages(c), k.shape[0], k.shape[2], table.shape[1], _CODES[k.dtype],
        k.data_ptr(), *k.stride(), v.data_ptr(), *v.stride(), phi.data_ptr(), *phi.stride(), psi.data_ptr(), *psi.stride(),
        table.data_ptr(), table.stride(0), start.data_ptr(), _ptr(counts)))
    with device_guard(c.device):
        _lib.check(_lib.lib().fpa_cache_append(a, _lib.stream_of(c.device)))


def read(c, table, start, n, counts, dtype):
    B, H, D, dev = table.shape[0], c.n_heads, c.d_head, c.device
    table, start, counts = _unit(table), start.contiguous(), None if counts is None else counts.contiguous()
    with device_guard(dev):
        k, v = torch.empty((2, B, H, n, D), dtype=dtype, device=dev).unbind(0)
        phi, psi = torch.empty((2, B, H, n), dtype=torch.float32, device=dev).unbind(0)
        a = _lib.FpaReadArgs.from_buffer_copy(_lib.READ_PACK.pack(
            _pages(c), B, n, table.shape[1], _CODES[dtype], k.data_ptr(), v.data_ptr(), phi.data_ptr(), psi.data_ptr(),
            table.data_ptr(), table.stride(0), start.data_ptr(), _ptr(counts)))
        _lib.check(_lib.lib().fpa_cache_read(a, _lib.stream_of(dev)))
    return k, v, phi, psi


@functools.lru_cache(maxsize=256)
def _attend_scratch(B, H, N, D, P, prefix_length, dtype, store):
    """(workspace bytes, counters) of a call of this shape."""
    L = _lib.lib()
    return L.fpa_attend_workspace_bytes(B, H, N, D, P, prefix_length, dtype, store), L.fpa_attend_counts(B, H, N)


def attend(q, c, beta, table, lengths, prefix, prefix_length):
    B, H, N, D = q.shape
    dev = q.device
    q, beta, table, lengths = rows(q), beta.contiguous(), _unit(table), lengths.contiguous()
    prefix = None if prefix is None or prefix_length == 0 else prefix.contiguous()
    P = table.shape[1]
    with device_guard(dev):
        o = torch.empty((B, N, H, D), dtype=q.dtype, device=dev).transpose(1, 2)
        nws, ncounts = _attend_scratch(B, H, N, D, P, prefix_length, _CODES[q.dtype], _CODES[c.dtype])
        ws = workspace(dev, nws) if nws else None
        a = _lib.FpaAttendArgs.from_buffer_copy(_lib.ATTEND_PACK.pack(
            _pages(c), B, N, P, _CODES[q.dtype], q.data_ptr(), *q.stride(), o.data_ptr(), *o.stride(), beta.data_ptr(),
            table.data_ptr(), table.stride(0), lengths.data_ptr(), _ptr(prefix), prefix_length, _ptr(ws),
            counters(dev, ncounts).data_ptr()))
        _lib.check(_lib.lib().fpa_attend(a, _lib.stream_of(dev)))
    return o


@functools.lru_cache(maxsize=256)
def _verify_ws_bytes(B, V):
    return _lib.lib().fpa_verify_workspace_bytes(B, V)


def verify(target, draft, tokens, accept_u, sample_u):
    (B, N), V, dev = tokens.shape, target.shape[2], target.device
    target, draft = _unit(target), None if draft is None else _unit(draft)
    tokens, accept_u, sample_u = _unit(tokens), _unit(accept_u), sample_u.contiguous()
    with device_guard(dev):
        out = torch.empty(B * (N + 2), dtype=torch.int64, device=dev)  # both results in one allocation
        accepted, out = out[:B], out[B:].view(B, N + 1)
        ws = workspace(dev, _verify_ws_bytes(B, V))
        a = _lib.FpaVerifyArgs.from_buffer_copy(_lib.VERIFY_PACK.pack(
            B, N, V, _CODES[target.dtype], target.data_ptr(), *target.stride()[:2],
            _ptr(draft), *(draft.stride()[:2] if draft is not None else (0, 0)), tokens.data_ptr(), tokens.stride(0),
            accept_u.data_ptr(), accept_u.stride(0), sample_u.data_ptr(), accepted.data_ptr(), out.data_ptr(),
            ws.data_ptr()))
        _lib.check(_lib.lib().fpa_verify(a, _lib.stream_of(dev)))
    return accepted, out
