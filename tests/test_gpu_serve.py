"""The serving operators' kernels on the GPU against float64 and, where values are exact, against the PyTorch path bit for bit."""
import math

import pytest
import torch

import fpa
from fpa import PagedCache, cached_attention, shared_prefix_attention, verify_drafts
from oracle import serve_oracle as S
from serve_cases import STORE, filled, poison, probabilities, rows, tables

pytestmark = pytest.mark.gpu
DEV = "cuda"

# A row's error, as a share of sum_s p_s |v_s| (at most the largest |v_s|).
# fp32: the logits here are below 64 in base 2, so the three roundings of one are at most 3 * 64 * 2^-25 = 5.7e-6, times ln 2 in
# its weight, twice (weight and sum); the products' sums of up to 256 and 3000 terms, accumulated 4 or 16 at a time, add well under 1.5e-5.
# fp16: the same, and two half steps of 2^-11: of a weight and of the result.
TOL = {"f32": 2.5e-5, "f16": 2.5e-5 + 2 * 2.0 ** -11}


@pytest.fixture(autouse=True)
def need_gpu(request):
    if not torch.cuda.is_available():
        pytest.skip("needs a GPU")
    print(f"[serve] {request.node.name}", flush=True)


def want64(q, c, beta, table, lengths, prefix=None, P=0):
    """(o, largest |v| a sequence sees) in float64 on the CPU, by the definition on values read one page at a time."""
    buf = {n: None if x is None else x for n, x in S.buffers(c).items()}
    q, beta = q.detach().cpu().double(), beta.cpu().double()
    B, H, N, D = q.shape
    o, vmax = torch.zeros(B, H, N, D, dtype=torch.float64), torch.ones(B, dtype=torch.float64)

    def seq(pages, n):
        k = torch.cat([buf["k"][int(p)].double() * (1 if buf["k_exp"] is None else 2.0 ** buf["k_exp"][int(p)].double().unsqueeze(-1))
                       for p in pages], 1)[:, :n]
        v = torch.cat([buf["v"][int(p)].double().transpose(-1, -2) *
                       (1 if buf["v_exp"] is None else 2.0 ** buf["v_exp"][int(p)].double().unsqueeze(-1)) for p in pages], 1)[:, :n]
        return [k, v] + [torch.cat([buf[x][int(p)].double() for p in pages], 1)[:, :n] for x in ("phi", "psi")]
    pre = seq(prefix.cpu(), P) if P else None
    for b in range(B):
        L = int(lengths[b])
        if L == 0:
            continue
        own = seq(table[b, :-(-L // 64)].cpu(), L)
        k, v, phi, psi = own if pre is None else [torch.cat(x, 1) for x in zip(pre, own)]
        vmax[b] = max(vmax[b], v.norm(dim=-1).max())
        for i in range(max(0, N - L), N):
            n = P + L - N + i + 1
            low = torch.cat((phi[:, 1:n], torch.full((H, 1), math.inf)), 1).flip(1).cummin(1).values.flip(1)
            z = (k[:, :n] * q[b, :, i].unsqueeze(1)).sum(-1) * D ** -0.5 + beta.unsqueeze(1) * (low - psi[:, :n]).clamp(max=0.0)
            o[b, :, i] = (torch.softmax(z, -1).unsqueeze(-1) * v[:, :n]).sum(1)
    return o, vmax


def held(o, want, vmax, tol):
    o = o.detach().cpu().double()
    assert o.shape == want.shape and torch.isfinite(o).all()
    off = ((o - want).norm(dim=-1) / vmax.view(-1, 1, 1)).max().item()
    assert off <= tol, off


def same_buffers(a, b):
    for n, x in S.buffers(a).items():
        y = S.buffers(b)[n]
        if x is None:
            continue
        if n in ("k", "v") and x.element_size() == 1:
            x, y = x.view(torch.uint8), y.view(torch.uint8)
        elif x.is_floating_point():
            x, y = (t.contiguous().view(torch.int16 if t.element_size() == 2 else torch.int32) for t in (x, y))
        assert torch.equal(x, y), n


MOVES = [("f16", "f16"), ("f32", "f32"), ("e4m3", "f16"), ("e4m3", "f32")]


@pytest.mark.parametrize("store,q", MOVES)
@pytest.mark.parametrize("D", [16, 32, 64, 128, 256])
def test_append_and_read(store, q, D):
    """Appends that begin and end anywhere in a page, ragged, in several steps, on poisoned pages: every buffer, and what is read back,
    bit for bit that of the PyTorch path (codes are one rounding, the rest is copied)."""
    g = torch.Generator().manual_seed(D)
    B, H = 4, 3
    here, there = PagedCache(17, H, D, STORE[store], DEV), PagedCache(17, H, D, STORE[store])
    poison(here)
    poison(there)
    table = tables([200, 64, 130, 1], 6, 17, g)
    start = torch.tensor([0, 5, 63, 0], dtype=torch.int32)
    for n, counts in ((70, [70, 1, 60, 0]), (1, [1, 1, 1, 1]), (64, [64, 40, 3, -2]), (2, None)):
        k, v, phi, psi = rows(B, H, n, D, STORE[q], g)
        k = k.clone()
        k[0, 0, 0] = 0.0
        k[1, 1, 0, 3] = float("inf")
        c = None if counts is None else torch.tensor(counts, dtype=torch.int32)
        there.append(k, v, phi, psi, table, start, c)
        dev = [x.to(DEV) for x in (k, v, phi, psi, table, start)]
        here.append(*dev, None if c is None else c.to(DEV))
        same_buffers(here, there)
        for dt in {STORE[q], *((torch.float16, torch.float32) if store == "e4m3" else ())}:
            back = here.read(dev[4], dev[5], n, None if c is None else c.to(DEV), dtype=dt)
            for x, y in zip(back, there.read(table, start, n, c, dtype=dt)):
                assert torch.equal(torch.nan_to_num(x.cpu(), nan=5.0), torch.nan_to_num(y, nan=5.0))
        start = start + (n if c is None else c.clamp(min=0))


def test_quantise_every_kind_of_value():
    """All fp16 numbers, then fp32 ones of every exponent, ties and neighbours of ties, in rows with a known maximum."""
    allh = torch.arange(65536, dtype=torch.int32).to(torch.int16).view(torch.float16)
    f32 = torch.cat([torch.ldexp(torch.tensor([1.0, 1.0625, 1.1875, 1.0624999, 1.0625001, 1.9999999, 1.75, 1.7500001]), torch.tensor(float(e)))
                     for e in range(-149, 128)])
    f32 = torch.cat([f32, -f32, torch.tensor([0.0, -0.0, math.inf, -math.inf, math.nan] + [1.0] * 59)])
    f32 = f32[:f32.numel() // 64 * 64]
    for x, dt in ((allh, torch.float16), (f32, torch.float32)):
        x = x.view(1, 1, -1, 64).contiguous()
        n = x.shape[2]
        zero = torch.zeros(1, 1, n)
        cs = [PagedCache(-(-n // 64), 1, 64, torch.float8_e4m3fn, d) for d in (DEV, "cpu")]
        for c, d in zip(cs, (DEV, "cpu")):
            c.append(x.to(d), x.flip(-1).to(d), zero.to(d), zero.to(d), torch.arange(c.pages, dtype=torch.int32, device=d).view(1, -1),
                     torch.zeros(1, dtype=torch.int32, device=d))
        same = S.buffers(cs[0]), S.buffers(cs[1])
        for name in ("k_exp", "v_exp"):
            assert torch.equal(same[0][name], same[1][name])
        for name in ("k", "v"):
            a, b = (torch.nan_to_num(s[name].float(), nan=1000.0) for s in same)
            assert torch.equal(a, b)


@pytest.mark.parametrize("store,q", MOVES)
@pytest.mark.parametrize("D", [16, 32, 64, 128, 256])
def test_attention(store, q, D):
    """Every type and head size, ragged lengths around page borders, one to seventeen rows."""
    lengths = [200, 64, 65, 63, 1, 0, 129, 7]
    cache, table, L, _, x, beta = filled(8, 2, D, lengths, store, q, D, device=DEV)
    for N in (1, 2, 3, 4, 5, 16):
        o = cached_attention(x[:, :, :N], cache, beta, table, L)
        held(o, *want64(x[:, :, :N], cache, beta, table, L), TOL[q])
        assert (o[5] == 0).all()


@pytest.mark.parametrize("store,q", MOVES)
def test_attention_of_many_rows(store, q):
    """More rows than a tile holds, the last tile ragged, some before the sequence's first position."""
    cache, table, L, _, x, beta = filled(3, 2, 64, [150, 64, 20], store, q, 2, device=DEV)
    x = torch.cat([x, x.flip(2), x * 0.5], 2)[:, :, :43]
    held(cached_attention(x, cache, beta, table, L), *want64(x, cache, beta, table, L), TOL[q])


@pytest.mark.parametrize("store,q,D", [("f16", "f16", 64), ("f32", "f32", 32), ("e4m3", "f16", 128)])
@pytest.mark.parametrize("N", [1, 3, 6])
def test_long_sequences_in_parts(store, q, D, N):
    """Sequences cut into parts, next to short and empty ones, with a table wider than any needs."""
    cache, table, L, _, x, beta = filled(3, 2, D, [2900, 0, 130], store, q, N, width=60, device=DEV)
    a = cached_attention(x[:, :, :N], cache, beta, table, L)
    held(a, *want64(x[:, :, :N], cache, beta, table, L), TOL[q])
    assert torch.equal(a, cached_attention(x[:, :, :N], cache, beta, table, L))


@pytest.mark.parametrize("store,q", [("f16", "f16"), ("e4m3", "f32")])
@pytest.mark.parametrize("prefix", [0, 70])
def test_many_short_sequences(store, q, prefix):
    """So many that a wave takes each by itself; with odd sizes, so that the last workgroup is not full."""
    g = torch.Generator().manual_seed(11)
    B = 61
    lengths = [0, 1, 256, 64] + torch.randint(0, 257, (B - 4,), generator=g).tolist()
    cache, table, L, pre, x, beta = filled(B, 9, 32, lengths, store, q, 1, prefix=prefix, device=DEV)
    for N in (1, 3):
        if prefix:
            o = shared_prefix_attention(x[:, :, :N], cache, beta, pre, prefix, table, L)
        else:
            o = cached_attention(x[:, :, :N], cache, beta, table, L)
        held(o, *want64(x[:, :, :N], cache, beta, table, L, pre, prefix), TOL[q])
        t = table.clone()
        t[2, 3] = -1
        bad = shared_prefix_attention(x[:, :, :N], cache, beta, pre, prefix, t, L) if prefix else cached_attention(x[:, :, :N], cache, beta, t, L)
        assert bad[2].isnan().all() and torch.equal(bad[:2], o[:2]) and torch.equal(bad[3:], o[3:])


@pytest.mark.parametrize("store,q,D", [("e4m3", "f16", 16), ("e4m3", "f32", 16), ("f16", "f16", 16), ("f32", "f32", 128)])
def test_very_long_sequences(store, q, D):
    """Small pages, of which a part holds more than of others (D = 16), and parts of 48 pages; one long sequence, and one among
    short ones in a table that is far too wide."""
    cache, table, L, _, x, beta = filled(3, 2, D, [16500, 40, 9000], store, q, D, width=400, device=DEV)
    for b in (slice(0, 1), slice(0, 3)):
        for N in (1, 2):
            o = cached_attention(x[b, :, :N], cache, beta, table[b], L[b])
            held(o, *want64(x[b, :, :N], cache, beta, table[b], L[b]), 4 * TOL[q])  # sums over 16500 positions


@pytest.mark.parametrize("store,q", MOVES)
@pytest.mark.parametrize("P", [1, 64, 100, 777])
def test_prefix(store, q, P):
    """Prefixes that end inside and at the end of a page, sequences of every kind behind them."""
    cache, table, L, pre, x, beta = filled(5, 2, 64, [70, 2, 0, 128, 64], store, q, P, prefix=P, device=DEV)
    for N in (1, 4):
        o = shared_prefix_attention(x[:, :, :N], cache, beta, pre, P, table, L)
        held(o, *want64(x[:, :, :N], cache, beta, table, L, pre, P), TOL[q])
        assert (o[2] == 0).all()
        assert torch.equal(o, shared_prefix_attention(x[:, :, :N], cache, beta, pre, P, table, L))


@pytest.mark.parametrize("D", [16, 32, 128, 256])
def test_prefix_head_sizes_and_many_rows(D):
    cache, table, L, pre, x, beta = filled(9, 1, D, [33, 64, 65, 1, 300, 2, 16, 17, 90], "f16", "f16", D, prefix=200, device=DEV)
    for N in (3, 16):
        o = shared_prefix_attention(x[:, :, :N], cache, beta, pre, 200, table, L)
        held(o, *want64(x[:, :, :N], cache, beta, table, L, pre, 200), TOL["f16"])


@pytest.mark.parametrize("store,q", MOVES)
@pytest.mark.parametrize("D", [16, 32, 64, 128, 256])
def test_prefix_of_every_kernel(store, q, D):
    """Every type and head size with tiles of 16 and of 32 rows, own rows in both forms, and own pages in several parts."""
    for B, lengths in ((3, [70, 2, 1800]), (9, [33, 64, 65, 1, 300, 0, 16, 1700, 90])):
        cache, table, L, pre, x, beta = filled(B, 2, D, lengths, store, q, D, prefix=200, device=DEV)
        for N in (1, 5):
            o = shared_prefix_attention(x[:, :, :N], cache, beta, pre, 200, table, L)
            held(o, *want64(x[:, :, :N], cache, beta, table, L, pre, 200), TOL[q])


@pytest.mark.parametrize("N", [20, 43])
def test_prefix_with_more_rows_than_a_tile(N):
    cache, table, L, pre, x, beta = filled(3, 2, 64, [130, 1700, 25], "f16", "f16", N, prefix=130, device=DEV)
    x = torch.cat([x, x.flip(2), x * 0.5], 2)[:, :, :N]
    for b in (slice(0, 1), slice(0, 3)):
        o = shared_prefix_attention(x[b], cache, beta, pre, 130, table[b], L[b])
        held(o, *want64(x[b], cache, beta, table[b], L[b], pre, 130), TOL["f16"])


@pytest.mark.parametrize("store,q", MOVES)
@pytest.mark.parametrize("D", [16, 64, 128, 256])
def test_waves_alone_of_every_kernel(store, q, D):
    g = torch.Generator().manual_seed(D)
    lengths = torch.randint(0, 257, (48,), generator=g).tolist()
    cache, table, L, pre, x, beta = filled(48, 16, D, lengths, store, q, 1, prefix=64, device=DEV)
    for N in (1, 2):
        held(cached_attention(x[:, :, :N], cache, beta, table, L), *want64(x[:, :, :N], cache, beta, table, L), TOL[q])
    o = shared_prefix_attention(x[:, :, :2], cache, beta, pre, 64, table, L)
    held(o, *want64(x[:, :, :2], cache, beta, table, L, pre, 64), TOL[q])


def test_prefix_equals_its_copy_in_every_table():
    """The prefix in front of each sequence's own pages (a whole number of pages) through cached_attention."""
    P = 192
    cache, table, L, pre, x, beta = filled(4, 3, 64, [70, 2, 128, 9], "f16", "f16", 1, prefix=P, device=DEV)
    a = shared_prefix_attention(x[:, :, :2], cache, beta, pre, P, table, L)
    b = cached_attention(x[:, :, :2], cache, beta, torch.cat((pre.expand(4, -1), table), 1), L + P)
    assert (a.double() - b.double()).abs().max() <= 2 * TOL["f16"] * 4.0 * 8  # |v| <= 4 sqrt(D)


@pytest.mark.parametrize("store,q", MOVES)
@pytest.mark.parametrize("N", [4, 5])
def test_values_that_some_rows_must_not_see(store, q, N):
    """Infinities and NaN in k, v and psi of a later drafted position leave the rows before it alone; v's reach the rows that
    see them."""
    at = 66  # of 68 positions the last five rows stand at 63 .. 67
    cache, table, L, _, x, beta = filled(2, 2, 32, [68, 68], store, q, 8, device=DEV)
    x = x[:, :, :N]
    whole = cached_attention(x, cache, beta, table, L)
    page, slot = int(table[0, at // 64]), at % 64
    bad = 0x7f if store == "e4m3" else math.inf
    (cache.v.view(torch.uint8) if store == "e4m3" else cache.v)[page, :, 3, slot] = bad
    o = cached_attention(x, cache, beta, table, L)
    assert torch.equal(o[:, :, :N - 2], whole[:, :, :N - 2]) and torch.equal(o[1], whole[1])
    assert not torch.isfinite(o[0, :, N - 2:, 3]).any()
    others = [d for d in range(32) if d != 3]
    assert torch.equal(o[0][..., others], whole[0][..., others])
    (cache.k.view(torch.uint8) if store == "e4m3" else cache.k)[page, :, slot] = 0x7f if store == "e4m3" else math.nan
    cache.psi[page, :, slot] = math.nan
    cache.phi[page, :, slot] = -math.inf
    o = cached_attention(x, cache, beta, table, L)
    assert torch.equal(o[:, :, :N - 2], whole[:, :, :N - 2]) and torch.equal(o[1], whole[1])


def test_extreme_scales():
    """Rows of K and V at very different scales in 8 bits: the weights fill fp16's range whatever the powers are."""
    g = torch.Generator().manual_seed(3)
    B, H, T, D = 1, 2, 300, 64
    k, v, phi, psi = rows(B, H, T, D, torch.float32, g)
    v = v * torch.ldexp(torch.ones(()), torch.randint(-30, 10, (B, H, T, 1), generator=g).float())
    v[:, 1] *= 2.0 ** -40
    k[:, :, 7] = 0.0
    v[:, :, 9] = 0.0
    c = PagedCache(5, H, D, torch.float8_e4m3fn, DEV)
    table, zero = torch.arange(5, dtype=torch.int32, device=DEV).view(1, 5), torch.zeros(1, dtype=torch.int32, device=DEV)
    c.append(*(x.to(DEV) for x in (k, v, phi, psi)), table, zero)
    q = torch.randn(1, H, 2, D, generator=g)
    L = zero + T
    beta = torch.tensor([0.5, 0.0], device=DEV)
    want, _ = want64(q, c, beta, table, L)
    o = cached_attention(q.to(DEV), c, beta, table, L).cpu().double()
    assert ((o - want).norm(dim=-1) <= 4 * TOL["f32"] * want.norm(dim=-1)).all()
    h = q[:, :1].half()
    both = torch.cat((h, h), 1)
    want, _ = want64(both, c, beta, table, L)
    o = cached_attention(both.to(DEV), c, beta, table, L).cpu().double()
    # one weight's rounding against the largest weighted row: the same 2^-11 as without scales
    assert ((o - want)[:, 0].norm(dim=-1) <= 4 * TOL["f16"] * want[:, 0].norm(dim=-1)).all()


def test_steep_and_flat_bias():
    """beta of both signs and zero, phi with infinities (a key that nothing separates from the query and one that everything does)."""
    cache, table, L, _, x, _ = filled(2, 3, 64, [200, 100], "f32", "f32", 12, device=DEV)
    beta = torch.tensor([0.0, 2.5, -0.01], device=DEV)
    held(cached_attention(x[:, :, :3], cache, beta, table, L), *want64(x[:, :, :3], cache, beta, table, L), TOL["f32"])
    cache.phi[int(table[0, 1]), 1, 5] = -math.inf
    cache.phi_min[int(table[0, 1]), 1] = -math.inf
    cache.phi[int(table[1, 0]), 2, 9] = math.inf
    held(cached_attention(x[:, :, :3], cache, beta[1], table, L), *want64(x[:, :, :3], cache, beta[1].expand(3), table, L), TOL["f32"])


@pytest.mark.parametrize("prefix", [0, 100])
def test_missing_pages(prefix):
    cache, table, L, pre, x, beta = filled(3, 2, 32, [400, 64, 70], "f16", "f16", 7, prefix=prefix, device=DEV)

    def run(t, n, pages=None):
        if prefix:
            return shared_prefix_attention(x[:, :, :2], cache, beta, pre if pages is None else pages, prefix, t, n)
        return cached_attention(x[:, :, :2], cache, beta, t, n)
    whole = run(table, L)
    for wrong in (-1, cache.pages, 2 ** 31 - 1, -2 ** 31):
        for at in (0, 3, 6):
            t = table.clone()
            t[0, at] = wrong
            o = run(t, L)
            assert o[0].isnan().all() and torch.equal(o[1:], whole[1:])
        if prefix:
            p = pre.clone()
            p[1] = wrong
            assert run(table, L, p).isnan().all()
    too_long = L.clone()
    too_long[2] = 64 * table.shape[1] + 1
    assert run(table, too_long)[2].isnan().all() and torch.equal(run(table, too_long)[:2], whole[:2])
    short = L.clone()
    short[1] = -7
    assert (run(table, short)[1] == 0).all()


def test_appends_to_missing_places():
    cache, table, L, _, x, beta = filled(3, 2, 16, [130, 64, 70], "e4m3", "f16", 7, device=DEV)
    before = S.buffers(cache)
    t = table.clone()
    t[0, 1] = cache.pages
    start = torch.tensor([64, 2 ** 31 - 1, -5], dtype=torch.int32, device=DEV)
    k, v, phi, psi = (a.to(DEV) for a in rows(3, 2, 3, 16, torch.float16, torch.Generator().manual_seed(1)))
    cache.append(k, v, phi, psi, t, start)
    after = S.buffers(cache)
    for n in before:
        a, b = ((z.view(torch.uint8) if z.element_size() == 1 else torch.nan_to_num(z, nan=3.0)) for z in (before[n], after[n]))
        assert torch.equal(a, b), n
    assert all(b.isnan().all() for b in cache.read(t, start, 3))


def test_rollback_and_append_again():
    """Drafts that were rejected are overwritten: phi_min of the page follows, so that the next pages' queries see the new values."""
    g = torch.Generator().manual_seed(4)
    c = PagedCache(4, 2, 32, torch.float32, DEV)
    table = torch.tensor([[2, 0, 3]], dtype=torch.int32, device=DEV)
    k, v, phi, psi = (a.to(DEV) for a in rows(1, 2, 190, 32, torch.float32, g))

    def put(a, b, low=0.0):
        c.append(k[:, :, a:b], v[:, :, a:b], phi[..., a:b] + low, psi[..., a:b], table, torch.tensor([a], dtype=torch.int32, device=DEV))
    put(0, 60)
    put(60, 70, low=-100.0)  # drafts, rejected from position 61 on
    put(61, 64)
    put(64, 190)
    phi[..., 60] -= 100.0
    x = torch.randn(1, 2, 3, 32, generator=g).to(DEV)
    L, beta = torch.tensor([190], dtype=torch.int32, device=DEV), torch.ones(2, device=DEV)
    assert torch.equal(c.read(table, torch.zeros_like(L), 190)[2], phi)
    held(cached_attention(x, c, beta, table, L), *want64(x, c, beta, table, L), TOL["f32"])


def test_offsets_beyond_32_bits():
    """Pages whose rows lie more than 2^32 elements into the pool."""
    D, pages = 256, 270000  # 64 * 256 * 270000 = 4.4e9 elements of k and of v
    if torch.cuda.mem_get_info()[0] < 40e9:
        pytest.skip("needs 40 GB of free memory")
    c = PagedCache.from_buffers(torch.empty(pages, 1, 64, D, dtype=torch.float16, device=DEV),
                                torch.empty(pages, 1, D, 64, dtype=torch.float16, device=DEV),
                                *(torch.empty(pages, 1, 64, device=DEV) for _ in range(2)), torch.empty(pages, 1, device=DEV))
    table = torch.tensor([[pages - 1, 1, pages - 2]], dtype=torch.int32, device=DEV)
    g = torch.Generator().manual_seed(0)
    k, v, phi, psi = (a.to(DEV) for a in rows(1, 1, 150, D, torch.float16, g))
    zero = torch.zeros(1, dtype=torch.int32, device=DEV)
    c.append(k, v, phi, psi, table, zero)
    assert torch.equal(c.read(table, zero, 150)[1], v)
    few = PagedCache(3, 1, D, torch.float16, DEV)
    order = torch.tensor([[2, 0, 1]], dtype=torch.int32, device=DEV)
    few.append(k, v, phi, psi, order, zero)
    x, beta = torch.randn(1, 1, 2, D, generator=g).half().to(DEV), torch.ones(1, device=DEV)
    assert torch.equal(cached_attention(x, c, beta, table, zero + 150), cached_attention(x, few, beta, order, zero + 150))


def test_strides_orders_and_scalars():
    """Layouts that a caller may hold: transposed tables, expanded and sliced vectors, unaligned rows, a scalar beta."""
    cache, table, L, _, x, beta = filled(4, 2, 64, [130, 64, 5, 200], "f16", "f16", 2, device=DEV)
    x = x[:, :, :3]
    whole = cached_attention(x, cache, 0.7, table, L)
    wide = torch.full((table.shape[1] + 3, 9), -9, dtype=torch.int32, device=DEV)
    wide[1:1 + table.shape[1], 2:6] = table.t()
    vec = torch.full((9,), -9, dtype=torch.int32, device=DEV)
    vec[1::2] = L
    odd = torch.empty(x.numel() + 1, dtype=x.dtype, device=DEV)[1:].view(x.shape).copy_(x)
    assert odd.data_ptr() % 16 != 0
    for q in (x.contiguous(), odd, x.transpose(0, 1).contiguous().transpose(0, 1), x.repeat_interleave(2, -1)[..., ::2]):
        assert torch.equal(cached_attention(q, cache, torch.full((1,), 0.7, device=DEV), wide[1:1 + table.shape[1], 2:6].t(), vec[1::2]), whole)
    one = cached_attention(x[:1].expand(4, -1, -1, -1), cache, 0.7, table[:1].expand(4, -1), L[:1].expand(4))
    assert torch.equal(one, whole[:1].expand(4, -1, -1, -1))


VERIFY = [(1, 4, 32000, "f32", True), (5, 1, 1, "f32", True), (7, 3, 1000, "f16", True), (9, 8, 65537, "f32", False), (3, 0, 50, "f32", True),
          (64, 5, 999, "f32", True), (2, 70, 130, "f16", False)]


@pytest.mark.parametrize("B,N,V,dtype,draft", VERIFY)
def test_verify(B, N, V, dtype, draft):
    """Counts and tokens equal the float64 oracle's, with rows that end early, that hold nothing, and that equal their draft's."""
    t, d, x, u, r = probabilities(B, N, V, STORE[dtype], B + V, draft)
    if N >= 2 and B >= 7:
        x[1, 1], x[2, 0] = -1, V
        t[3, 0] = 0.0
        if draft:
            t[4, 0] = d[4, 0]
            u[4, 0] = 1 - 2 ** -24
        t[5] = math.nan
        r[6], u[6] = 0.0, 0.0
    a, out = verify_drafts(*(None if z is None else z.to(DEV) for z in (t, d, x, u, r)))
    ea, eout = verify_drafts(t, d, x, u, r, impl="reference")
    assert torch.equal(a.cpu(), ea) and torch.equal(out.cpu(), eout)
    if B * V <= 10000 and B < 7:
        oa, oo = S.verify(t, d, x, u, r)
        assert torch.equal(ea, oa) and torch.equal(eout, oo)


def test_verify_strided():
    t, d, x, u, r = (z.to(DEV) for z in probabilities(6, 4, 500, torch.float32, 3))
    a, out = verify_drafts(t, d, x, u, r)
    big = torch.full((6, 9, 700), math.nan, device=DEV)
    big[:, 2:7, 100:600] = t
    b2, out2 = verify_drafts(big[:, 2:7, 100:600], d.transpose(1, 2).contiguous().transpose(1, 2), x.t().contiguous().t(),
                             torch.stack((u, u), -1)[..., 0], torch.stack((r, r), -1)[..., 1])
    assert torch.equal(a, b2) and torch.equal(out, out2)


def test_another_stream():
    cache, table, L, pre, x, beta = filled(4, 2, 64, [1030, 64, 5, 200], "e4m3", "f16", 2, prefix=500, device=DEV)
    want = shared_prefix_attention(x, cache, beta, pre, 500, table, L)
    torch.cuda.synchronize()
    side = [torch.cuda.Stream() for _ in range(2)]
    got = []
    for _ in range(3):
        for s in side:
            with torch.cuda.stream(s):
                got.append(shared_prefix_attention(x, cache, beta, pre, 500, table, L))
    torch.cuda.synchronize()
    assert all(torch.equal(o, want) for o in got)


def test_captured_step_replays():
    """Append, read, both attentions and the verification captured in two graphs that share a pool, replayed in turn with eager work and
    new inputs in between: every replay equals the eager result."""
    B, H, D = 3, 2, 64
    cache, table, L, pre, x, beta = filled(B, H, D, [1030, 64, 205], "e4m3", "f16", 2, prefix=300, device=DEV)
    g = torch.Generator().manual_seed(5)
    k, v, phi, psi = (a.to(DEV) for a in rows(B, H, 2, D, torch.float16, g))
    k, v = k.contiguous(), v.contiguous()
    t, d, tok, u, r = (z.to(DEV) for z in probabilities(B, 3, 777, torch.float32, 1))
    x = x[:, :, :2].contiguous()

    def step():
        cache.append(k, v, phi, psi, table, L - 2)
        return (*cache.read(table, L - 2, 2), cached_attention(x, cache, beta, table, L),
                shared_prefix_attention(x, cache, beta, pre, 300, table, L), *verify_drafts(t, d, tok, u, r))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graphs, outs = [], []
    pool = None
    for _ in range(2):
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr, pool=pool):
            outs.append(step())
        pool = pool or gr.pool()
        graphs.append(gr)
    for turn in range(3):
        k.copy_(torch.randn(k.shape, generator=g))
        v.copy_(torch.randn(v.shape, generator=g))
        x.copy_(torch.randn(x.shape, generator=g))
        r.copy_(torch.rand(r.shape, generator=g))
        for gr, out in zip(graphs, outs):
            gr.replay()
            torch.cuda.synchronize()
            kept = [o.clone() for o in out]
            for a, b in zip(kept, step()):
                assert torch.equal(a, b)


def test_whole_decoding_equals_training_attention():
    """A sequence appended and attended to in steps of different sizes gives the rows of first_passage_attention."""
    B, H, T, D = 2, 3, 150, 64
    g = torch.Generator().manual_seed(6)
    k, v, phi, psi = (a.to(DEV) for a in rows(B, H, T, D, torch.float32, g))
    q, beta = torch.randn(B, H, T, D, generator=g).to(DEV), (torch.rand(H, generator=g) + 0.5).to(DEV)
    want = fpa.first_passage_attention(q, k, v, phi, psi, beta, impl="hip")
    c = PagedCache(3 * B, H, D, torch.float32, DEV)
    table, at = torch.arange(3 * B, dtype=torch.int32, device=DEV).view(B, 3), 0
    for n in (50, 1, 1, 16, 20, 40, 22):
        start = torch.full((B,), at, dtype=torch.int32, device=DEV)
        c.append(*(z[:, :, at:at + n] for z in (k, v, phi, psi)), table, start)
        o = cached_attention(q[:, :, at:at + n], c, beta, table, start + n)
        assert (o - want[:, :, at:at + n]).abs().max() <= 2 * TOL["f32"] * 4 * 8  # two sides, |v| <= 4 sqrt(D)
        at += n
