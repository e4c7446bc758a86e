"""The serving operators on the CPU: impl="reference" against the float64 oracle, and every refusal (also of the C ABI,
which validates before any launch)."""
import copy
import ctypes
import os
import shutil
import subprocess

import pytest
import torch

import fpa
from fpa import PagedCache, _lib, cached_attention, shared_prefix_attention, verify_drafts
from oracle import serve_oracle as S
from serve_cases import STORE, filled, probabilities, rows, tables

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
# The dense path computes in fp32: a relative error of at most about (D + T) rounding steps of 2^-24 a sum, for the few
# hundred terms here below 1e-4 / 4; fp16 outputs add half a step, 2^-11, of the value.
TOL = {"f32": 2.5e-5, "f16": 2.5e-5 + 2.0 ** -11}


def close(a, b, tol):
    assert a.shape == b.shape
    assert torch.isfinite(a).all()
    assert (a.double() - b).norm() <= tol * b.norm() + 1e-30, ((a.double() - b).norm() / b.norm()).item()


@pytest.mark.parametrize("dtype", ["f16", "f32"])
@pytest.mark.parametrize("D", [16, 64])
def test_quantised_rows(dtype, D):
    """Codes, exponents and values against a search over all e4m3 numbers: ordinary rows, zeros, subnormals, ties, huge values,
    infinities and NaN."""
    g = torch.Generator().manual_seed(1)
    k, v, phi, psi = rows(1, 2, 70, D, STORE[dtype], g)
    k, v = k.contiguous(), v.contiguous()
    k[0, 0, 0] = 0.0
    k[0, 0, 1] = 448.0
    k[0, 0, 2] = 449.0
    k[0, 0, 3] = 6e-8
    k[0, 0, 4] = torch.arange(D) * 0.0625 + 17.0  # ties between codes
    k[0, 1, 5, 0] = float("nan")
    k[0, 1, 6, 1] = float("inf")
    k[0, 1, 7, 2] = float("-inf")
    if dtype == "f32":
        v[0, 0, 0] = 1e30
        v[0, 0, 1] = 1e-30
        v[0, 0, 2] = 1e-45
    c = PagedCache(3, 2, D, torch.float8_e4m3fn)
    table = torch.tensor([[2, 0]], dtype=torch.int32)
    start = torch.tensor([11], dtype=torch.int32)
    c.append(k, v, phi, psi, table, start)
    back = c.read(table, start, 70, dtype=torch.float32)
    for x, y, exp in ((k, back[0], c.k_exp), (v, back[1], c.v_exp)):
        want, e = S.quantised(x)
        assert torch.equal(torch.nan_to_num(y.double(), nan=7.0), torch.nan_to_num(want, nan=7.0))
        held = torch.cat((exp[2], exp[0]), -1)[:, 11:81]
        assert torch.equal(held, e[0])
    assert torch.equal(back[2], phi) and torch.equal(back[3], psi)


@pytest.mark.parametrize("store,q", [("f16", "f16"), ("f32", "f32"), ("e4m3", "f16"), ("e4m3", "f32")])
@pytest.mark.parametrize("N", [1, 5, 16])
def test_reference_attention(store, q, N):
    cache, table, lengths, _, x, beta = filled(4, 2, 16, [130, 64, 1, 0], store, q, 3)
    o = cached_attention(x[:, :, :N], cache, beta, table, lengths)
    want = S.attention(x[:, :, :N], S.buffers(cache), beta, table, lengths)
    close(o, want, TOL[q])
    assert (o[3] == 0).all()


@pytest.mark.parametrize("P", [1, 64, 100])
@pytest.mark.parametrize("N", [1, 3])
def test_reference_prefix(P, N):
    cache, table, lengths, pre, x, beta = filled(3, 2, 16, [70, 2, 0], "f32", "f32", 4, prefix=P)
    o = shared_prefix_attention(x[:, :, :N], cache, beta, pre, P, table, lengths)
    close(o, S.attention(x[:, :, :N], S.buffers(cache), beta, table, lengths, pre, P), TOL["f32"])
    assert (o[2] == 0).all()


def test_prefix_of_no_positions_is_cached_attention():
    cache, table, lengths, pre, x, beta = filled(2, 2, 16, [70, 20], "f32", "f32", 5, prefix=10)
    a = shared_prefix_attention(x, cache, beta, pre, 0, table, lengths)
    assert torch.equal(a, cached_attention(x, cache, beta, table, lengths))


def test_cached_rows_are_the_rows_of_the_whole_attention():
    """Position by position, the cache gives first_passage_attention's rows."""
    B, H, T, D = 2, 2, 90, 16
    g = torch.Generator().manual_seed(6)
    k, v, phi, psi = rows(B, H, T, D, torch.float32, g)
    q = torch.randn(B, H, T, D, generator=g)
    beta = torch.rand(H, generator=g) + 0.5
    want = fpa.first_passage_attention(q, k, v, phi, psi, beta, impl="reference")
    c = PagedCache(2 * B, H, D, torch.float32)
    table = torch.arange(2 * B, dtype=torch.int32).view(B, 2)
    at = 0
    for n in (30, 1, 1, 16, 20, 22):
        start = torch.full((B,), at, dtype=torch.int32)
        c.append(*(x[:, :, at:at + n] for x in (k, v, phi, psi)), table, start)
        o = cached_attention(q[:, :, at:at + n], c, beta, table, start + n)
        assert torch.allclose(o, want[:, :, at:at + n], rtol=0, atol=1e-5)
        at += n


@pytest.mark.parametrize("draft", [True, False])
@pytest.mark.parametrize("N,V", [(1, 1), (4, 300), (0, 50), (7, 33)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
def test_reference_verify(draft, N, V, dtype):
    t, d, x, u, r = probabilities(20, N, V, dtype, N + V, draft)
    if N > 2:
        x[3, 1], x[4, 0], x[5, 2] = -1, V, 2 ** 40
        t[6, 0] = 0.0
        if draft:
            t[7, 0] = d[7, 0]
            u[7, 0] = 1 - 2 ** -24
    a, out = verify_drafts(t, d, x, u, r)
    ea, eout = S.verify(t, d, x, u, r)
    assert torch.equal(a, ea) and torch.equal(out, eout)


def test_verify_keeps_the_target_distribution():
    """Over many random numbers the first token is distributed as the target's row (6 sigma)."""
    M, V = 60000, 5
    g = torch.Generator().manual_seed(9)
    p, d = torch.tensor([.5, .2, .1, .15, .05]), torch.tensor([.1, .2, .4, .05, .25])
    x = torch.multinomial(d, M, replacement=True, generator=g).view(M, 1)
    _, out = verify_drafts(p.expand(M, 2, V), d.expand(M, 1, V), x, torch.rand(M, 1, generator=g), torch.rand(M, generator=g))
    share = torch.bincount(out[:, 0], minlength=V) / M
    assert ((share - p).abs() <= 6 * (p * (1 - p) / M).sqrt()).all()


def test_a_missing_page_is_nan_and_touches_nothing():
    cache, table, lengths, _, x, beta = filled(3, 2, 16, [130, 64, 70], "f32", "f32", 7)
    whole = cached_attention(x[:, :, :2], cache, beta, table, lengths)
    for wrong in (-1, cache.pages, 2 ** 31 - 1, -2 ** 31):
        t = table.clone()
        t[0, 1] = wrong
        o = cached_attention(x[:, :, :2], cache, beta, t, lengths)
        assert o[0].isnan().all() and torch.equal(o[1:], whole[1:])
        before = S.buffers(cache)
        k, v, phi, psi = rows(3, 2, 1, 16, torch.float32, torch.Generator().manual_seed(1))
        cache.append(k, v, phi, psi, t, torch.tensor([64, 2 ** 31 - 1, -5], dtype=torch.int32))
        after = S.buffers(cache)
        for n in before:
            assert before[n] is None or torch.equal(torch.nan_to_num(before[n], nan=3.0), torch.nan_to_num(after[n], nan=3.0)), n
        back = cache.read(t, torch.tensor([64, 2 ** 31 - 1, -5], dtype=torch.int32), 1)
        assert all(b.isnan().all() for b in back)
    o = cached_attention(x[:, :, :2], cache, beta, table, torch.tensor([130, 64, 64 * table.shape[1] + 1], dtype=torch.int32))
    assert o[2].isnan().all() and torch.equal(o[:2], whole[:2])


def args():
    c = PagedCache(4, 2, 16, torch.float32)
    g = torch.Generator().manual_seed(0)
    k, v, phi, psi = rows(1, 2, 3, 16, torch.float32, g)
    return c, k, v, phi, psi, torch.tensor([[0, 1]], dtype=torch.int32), torch.tensor([5], dtype=torch.int32)


def test_refusals_of_the_cache():
    c, k, v, phi, psi, table, start = args()
    bad = [
        lambda: PagedCache(0, 2, 16), lambda: PagedCache(1, 2, 24), lambda: PagedCache(1, 2, 8),
        lambda: PagedCache(1, 2, 16, torch.bfloat16),
        lambda: PagedCache.from_buffers(c.k, c.k, c.phi, c.psi, c.phi_min),
        lambda: PagedCache.from_buffers(c.k, c.v, c.phi.double(), c.psi, c.phi_min),
        lambda: PagedCache.from_buffers(c.k, c.v, c.phi, c.psi, c.phi_min[:, :1]),
        lambda: PagedCache.from_buffers(c.k, c.v, c.phi, c.psi, c.phi_min, c.phi, c.phi),
        lambda: PagedCache.from_buffers(c.k.transpose(0, 1), c.v.transpose(0, 1), c.phi, c.psi, c.phi_min),
        lambda: c.append(k[:, :1], v[:, :1], phi, psi, table, start),
        lambda: c.append(k.half(), v.half(), phi, psi, table, start),
        lambda: c.append(k, v.half(), phi, psi, table, start),
        lambda: c.append(k.double(), v.double(), phi, psi, table, start),
        lambda: c.append(k, v, phi[..., :2], psi, table, start),
        lambda: c.append(k, v, phi, psi, table.long(), start),
        lambda: c.append(k, v, phi, psi, table[0], start),
        lambda: c.append(k, v, phi, psi, table, start.long()),
        lambda: c.append(k, v, phi, psi, table, start, start.float()),
        lambda: c.append(k[:, :, :0], v[:, :, :0], phi[..., :0], psi[..., :0], table, start),
        lambda: c.append(k.clone().requires_grad_(), v, phi, psi, table, start),
        lambda: c.append(k, v, phi, psi, table, start, impl="other"),
        lambda: c.read(table, start, 0), lambda: c.read(table, start, 2, dtype=torch.float16),
        lambda: c.read(table, start[:0], 2),
    ]
    for i, f in enumerate(bad):
        with pytest.raises(ValueError):
            f()
            pytest.fail(f"call {i} was not refused")
    with pytest.raises(RuntimeError):
        c.append(k, v, phi, psi, table, start, impl="hip")


def test_buffers_stay_and_copies_have_their_own():
    """The argument block of a cache is kept with it: its buffers cannot be exchanged, and a copy starts without the block."""
    c = fpa.PagedCache(2, 1, 16)
    with pytest.raises(AttributeError, match="from_buffers"):
        c.k = torch.zeros_like(c.k)
    c._packed = b"addresses of the buffers"
    d = copy.deepcopy(c)
    assert d._packed is None and d.k.data_ptr() != c.k.data_ptr() and torch.equal(d.phi_min, c.phi_min)
    d.name = "further attributes are the caller's"


def test_refusals_of_the_attention():
    c, k, v, phi, psi, table, start = args()
    beta = torch.ones(2)
    bad = [
        lambda: cached_attention(k[0], c, beta, table, start), lambda: cached_attention(k[:, :1], c, beta, table, start),
        lambda: cached_attention(k[..., :8], c, beta, table, start), lambda: cached_attention(k.half(), c, beta, table, start),
        lambda: cached_attention(k[:, :, :0], c, beta, table, start), lambda: cached_attention(k[:0], c, beta, table[:0], start[:0]),
        lambda: cached_attention(k, c, torch.ones(3), table, start), lambda: cached_attention(k, c, beta, table, start.long()),
        lambda: cached_attention(k, c, beta, table[:, :0], start), lambda: cached_attention(k, c, beta.requires_grad_(), table, start),
        lambda: shared_prefix_attention(k, c, 1.0, table, 3, table, start),
        lambda: shared_prefix_attention(k, c, 1.0, table[0].long(), 3, table, start),
        lambda: shared_prefix_attention(k, c, 1.0, table[0], 129, table, start),
        lambda: shared_prefix_attention(k, c, 1.0, table[0], -1, table, start),
    ]
    for i, f in enumerate(bad):
        with pytest.raises(ValueError):
            f()
            pytest.fail(f"call {i} was not refused")
    with torch.no_grad():
        cached_attention(k, c, torch.ones(2).requires_grad_(), table, start)


def test_refusals_of_the_drafts():
    t, d, x, u, r = probabilities(2, 3, 10, torch.float32, 0)
    bad = [
        lambda: verify_drafts(t[:, :3], d, x, u, r), lambda: verify_drafts(t, d[:, :2], x, u, r),
        lambda: verify_drafts(t, d.half(), x, u, r), lambda: verify_drafts(t.double(), d.double(), x, u, r),
        lambda: verify_drafts(t, d, x.int(), u, r), lambda: verify_drafts(t, d, x, u[:, :2], r),
        lambda: verify_drafts(t, d, x, u.double(), r), lambda: verify_drafts(t, d, x, u, r[:1]),
        lambda: verify_drafts(t[..., :0], d[..., :0], x, u, r), lambda: verify_drafts(t[:0], d[:0], x[:0], u[:0], r[:0]),
        lambda: verify_drafts(t.requires_grad_(), d, x, u, r),
    ]
    for i, f in enumerate(bad):
        with pytest.raises(ValueError):
            f()
            pytest.fail(f"call {i} was not refused")


def test_serving_structs_match_the_header(tmp_path):
    cc = shutil.which("gcc") or shutil.which("cc")
    if cc is None:
        pytest.skip("no C compiler")
    lines, names = [], ("FpaPages", "FpaAppendArgs", "FpaReadArgs", "FpaAttendArgs", "FpaVerifyArgs")
    for n in names:
        lines.append(f'printf("{n} sizeof %zu\\n", sizeof({n}));')
        lines += [f'printf("{n} {f} %zu\\n", offsetof({n}, {f}));' for f, _ in getattr(_lib, n)._fields_]
    src = tmp_path / "layout.c"
    src.write_text('#include <stdio.h>\n#include <stddef.h>\n#include "fpa.h"\nint main(void){\n' + "\n".join(lines) + "\nreturn 0;}\n")
    subprocess.run([cc, "-I", os.path.join(ROOT, "include"), str(src), "-o", str(tmp_path / "layout")], check=True)
    for line in subprocess.run([str(tmp_path / "layout")], check=True, capture_output=True, text=True).stdout.split("\n"):
        if line:
            n, f, val = line.split()
            cls = getattr(_lib, n)
            assert (ctypes.sizeof(cls) if f == "sizeof" else getattr(cls, f).offset) == int(val), (n, f)


def attend_args(**over):
    """FpaAttendArgs that pass every check but the one under test (addresses are never dereferenced: each call is
    refused before a launch)."""
    a = _lib.FpaAttendArgs()
    a.cache.pages, a.cache.H, a.cache.D, a.cache.store = 4, 2, 16, _lib.FPA_F32
    for n in ("k", "v", "phi", "psi", "phi_min"):
        setattr(a.cache, n, 256)
    a.B, a.N, a.P, a.dtype = 1, 1, 2, _lib.FPA_F32
    a.q, a.o, a.beta, a.table, a.lengths = 256, 256, 256, 256, 256
    a.sq, a.so = (ctypes.c_int64 * 4)(32, 16, 16, 1), (ctypes.c_int64 * 4)(32, 16, 16, 1)
    for n, v in over.items():
        if n.startswith("cache_"):
            setattr(a.cache, n[6:], v)
        else:
            setattr(a, n, (ctypes.c_int64 * 4)(*v) if n in ("sq", "so") else v)
    return a


@pytest.mark.parametrize("over,code,msg", [
    (dict(cache_pages=0), 1, "at least one page"), (dict(cache_D=24), 1, "power of two"), (dict(cache_D=512), 2, "not built"),
    (dict(cache_store=7), 1, "fp16, fp32 or e4m3"), (dict(cache_k=None), 1, "NULL"), (dict(cache_v=8), 1, "16-byte aligned"),
    (dict(cache_store=2), 1, "NULL"), (dict(cache_pages=2 ** 31), 2, "2^31"), (dict(cache_H=65536), 2, "65535"),
    (dict(dtype=0), 1, "cache's type"), (dict(dtype=2), 1, "fp16 or fp32"), (dict(B=0), 1, "at least 1"), (dict(N=0), 1, "at least 1"),
    (dict(P=0), 1, "at least 1"), (dict(P=131073), 2, "pages"), (dict(B=65536), 2, "65535"), (dict(table=None), 1, "table"),
    (dict(lengths=None), 1, "lengths"), (dict(q=None), 1, "q is NULL"), (dict(q=264), 1, "aligned"),
    (dict(sq=(32, 16, 16, 2)), 1, "contiguous"), (dict(o=None), 1, "non-NULL"), (dict(beta=None), 1, "non-NULL"),
    (dict(prefix_length=-1), 1, "prefix_length"), (dict(prefix_length=2 ** 24), 1, "prefix_length"),
    (dict(prefix_length=5), 1, "prefix is NULL"), (dict(prefix_length=5, prefix=256), 1, "workspace"),
    (dict(P=1000), 1, "workspace"), (dict(P=1000, workspace=128), 1, "workspace"), (dict(P=1000, workspace=256), 1, "counts"),
])
def test_attend_c_abi_validation(over, code, msg):
    L = _lib.lib()
    assert L.fpa_attend(attend_args(**over), None) == code
    assert msg in L.fpa_last_error().decode()


def test_serving_c_abi_null_and_sizes():
    L = _lib.lib()
    for f in (L.fpa_cache_append, L.fpa_cache_read, L.fpa_attend, L.fpa_verify):
        assert f(None, None) == _lib.FPA_ERR_INVALID
    a = _lib.FpaVerifyArgs()
    assert L.fpa_verify(a, None) == _lib.FPA_ERR_INVALID
    a.B, a.N, a.V = 1, 1, 10
    assert L.fpa_verify(a, None) == _lib.FPA_ERR_INVALID and "non-NULL" in L.fpa_last_error().decode()
    a.V = 2 ** 31
    assert L.fpa_verify(a, None) == _lib.FPA_ERR_UNSUPPORTED
    assert L.fpa_attend_workspace_bytes(1, 2, 1, 64, 1, 0, 0, 0) == 0
    n = L.fpa_attend_workspace_bytes(1, 2, 1, 64, 100, 0, 0, 0)
    assert n > 0 and n % 256 == 0
    assert tables([1], 1, 1, torch.Generator().manual_seed(0)).tolist() == [[0]]
