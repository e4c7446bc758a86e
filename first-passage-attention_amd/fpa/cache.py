"""The paged cache of a model that answers, and First Passage Attention against it.

``PagedCache`` holds k, v, phi and psi of past positions on pages of 64; ``append`` writes new positions (in 8 bits
if the cache is of that type) and ``read`` gives them back.  ``cached_attention`` is FPA of a sequence's last few
positions against its pages, ``shared_prefix_attention`` the same for sequences that continue one prefix, which is
read once for all of them.  None has a counterpart in the reference, which trains only.

A *table* (B, P) int32 names each sequence's pages in order, and *lengths* (B,) int32 counts its positions; entries
behind the last page are not read.  Both stay on the device, so no call waits for it.  What only the device knows is
not checked on the host: a page that the pool does not have, or a position behind the table, is never touched;
appends to it are dropped, and what is read from it, like every attention row that would need it, is NaN.

``impl`` is "hip" (the gfx950 kernels), "reference" (PyTorch, any device) or None for "hip" on GPU tensors and
"reference" otherwise, as in ``first_passage_attention``.  These operators have no gradient: they refuse tensors
that need one, outside ``torch.no_grad()``.
"""
import torch

from . import dense_serving as dense

PAGE = 64
STORES = (torch.float16, torch.float32, torch.float8_e4m3fn)
_HIP_NAMES = ("hip", "triton")


def _refuse_grad(*tensors):
    for t in tensors:
        if t.requires_grad and torch.is_grad_enabled():
            raise ValueError("the serving operators have no gradient: call them under torch.no_grad()")


def _hip():
    """The binding of the kernels; importing it loads libfpa.so and raises if it is missing."""
    global _BINDING
    if _BINDING is None:
        from . import _serve
        _BINDING = _serve
    return _BINDING


_BINDING = None


def pick_impl(impl, t):
    if impl is None:
        return "hip" if t.is_cuda else "reference"
    if impl == "reference":
        return impl
    if impl not in _HIP_NAMES:
        raise ValueError(f"unknown implementation {impl!r}")
    if not t.is_cuda:
        raise RuntimeError("impl='hip' needs tensors on a ROCm GPU")
    return "hip"


_FIXED = frozenset(("k", "v", "phi", "psi", "phi_min", "k_exp", "v_exp", "pages", "n_heads", "d_head", "dtype", "device"))


class PagedCache:
    """Pages of 64 positions for the heads of one attention layer.

    dtype: torch.float16, torch.float32, or torch.float8_e4m3fn for 8-bit codes with one power of two for each
    row of k and of v (k_exp, v_exp).  A code times its power is what the row stands for everywhere.

    Buffers (all contiguous): k (pages, H, 64, D); v (pages, H, D, 64), transposed; phi, psi (pages, H, 64) and phi_min
    (pages, H), the minimum of phi over the page's positions up to the last one appended; float32.
    """

    def __init__(self, pages, n_heads, d_head, dtype=torch.float16, device=None):
        if pages < 1 or n_heads < 1:
            raise ValueError("a cache has at least one page and one head")
        shape = (pages, n_heads)
        exps = [torch.zeros(*shape, PAGE, dtype=torch.int8, device=device) for _ in range(2)] if dtype == STORES[2] else [None] * 2
        z = torch.zeros(2, *shape, PAGE * d_head, dtype=torch.uint8 if dtype == STORES[2] else dtype, device=device).view(dtype)
        self._set(z[0].view(*shape, PAGE, d_head), z[1].view(*shape, d_head, PAGE),
                  torch.zeros(*shape, PAGE, device=device), torch.zeros(*shape, PAGE, device=device),
                  torch.full(shape, float("inf"), device=device), *exps)

    @classmethod
    def from_buffers(cls, k, v, phi, psi, phi_min, k_exp=None, v_exp=None):
        """A cache on existing buffers, which it shares."""
        c = cls.__new__(cls)
        c._set(k, v, phi, psi, phi_min, k_exp, v_exp)
        return c

    def _set(self, k, v, phi, psi, phi_min, k_exp, v_exp):
        if k.dim() != 4 or k.shape[2] != PAGE or v.shape != (*k.shape[:2], k.shape[3], PAGE):
            raise ValueError("k must be (pages, H, 64, D) and v (pages, H, D, 64)")
        if k.dtype not in STORES or v.dtype != k.dtype:
            raise ValueError("a cache holds fp16, fp32 or float8_e4m3fn")
        n, H, _, D = k.shape
        if D < 16 or D & (D - 1):
            raise ValueError("the head dimension must be a power of two >= 16")
        eight = k.dtype == STORES[2]
        if eight != (k_exp is not None) or eight != (v_exp is not None):
            raise ValueError("k_exp and v_exp belong to float8_e4m3fn caches, and to those alone")
        want = [(phi, (n, H, PAGE), torch.float32), (psi, (n, H, PAGE), torch.float32), (phi_min, (n, H), torch.float32)]
        if eight:
            want += [(k_exp, (n, H, PAGE), torch.int8), (v_exp, (n, H, PAGE), torch.int8)]
        for t, shape, dt in want:
            if t.shape != shape or t.dtype != dt:
                raise ValueError("phi and psi must be (pages, H, 64) and phi_min (pages, H), float32; k_exp and v_exp "
                                 "(pages, H, 64), int8")
        for t in (k, v, *(t for t, _, _ in want)):
            if not t.is_contiguous() or t.device != k.device or t.data_ptr() % 16:
                raise ValueError("a cache's buffers must be contiguous, 16-byte aligned and on one device")
        self.k, self.v, self.phi, self.psi, self.phi_min, self.k_exp, self.v_exp = k, v, phi, psi, phi_min, k_exp, v_exp
        self.pages, self.n_heads, self.d_head = n, H, D
        self.dtype, self.device = k.dtype, k.device
        self._packed = None  # the kernels' argument block, with the buffers' addresses

    def __setattr__(self, name, value):
        if name in _FIXED and name in self.__dict__:
            raise AttributeError(f"a cache keeps its {name}: PagedCache.from_buffers makes one of other buffers")
        super().__setattr__(name, value)

    def __getstate__(self):  # of copies, whose buffers may be others
        return {**self.__dict__, "_packed": None}

    def _check(self, B, table, dtype, start, name, counts=None):
        if dtype is not self.dtype:
            if dtype not in (torch.float16, torch.float32):
                raise ValueError("the tensors must be fp16 or fp32")
            if self.dtype is not torch.float8_e4m3fn:
                raise ValueError(f"a cache of {self.dtype} takes and gives tensors of that type")
        elif dtype is torch.float8_e4m3fn:
            raise ValueError("the tensors must be fp16 or fp32")
        dev = self.device
        if table.dtype is not torch.int32 or table.dim() != 2 or table.shape[0] != B or table.shape[1] < 1 or table.device != dev:
            raise ValueError("table must be (B, P) int32 with P >= 1, on the cache's device")
        if start.dtype is not torch.int32 or start.shape != (B,) or start.device != dev:
            raise ValueError(f"{name} must be (B,) int32, on the cache's device")
        if counts is not None and (counts.dtype is not torch.int32 or counts.shape != (B,) or counts.device != dev):
            raise ValueError("counts must be (B,) int32, on the cache's device")

    def append(self, k, v, phi, psi, table, start, counts=None, impl=None):
        """Writes k, v (B, H, N, D), phi, psi (B, H, N) to positions start[b] + i, for i < counts[b] (all N without
        counts).  Positions that a call writes must not share a page between two of its sequences.  Earlier positions of a
        page stay; phi_min becomes that of the positions up to the last one written."""
        if k.dim() != 4 or k.shape[1] != self.n_heads or k.shape[3] != self.d_head or v.shape != k.shape or v.dtype != k.dtype:
            raise ValueError(f"k and v must be (B, {self.n_heads}, N, {self.d_head}) of one type")
        B, H, N, _ = k.shape
        if B < 1 or N < 1:
            raise ValueError("k and v must hold at least one sequence and one position")
        if phi.shape != (B, H, N) or psi.shape != (B, H, N):
            raise ValueError("phi and psi must have shape (B, H, N)")
        self._check(B, table, k.dtype, start, "start", counts)
        dev = self.device
        if k.device != dev or v.device != dev or phi.device != dev or psi.device != dev:
            raise ValueError(f"k, v, phi and psi must be on the cache's device, {dev}")
        _refuse_grad(k, v, phi, psi)
        if pick_impl(impl, self.k) == "reference":
            return dense.append(self, k, v, phi, psi, table, start, counts)
        _hip().append(self, k, v, phi, psi, table, start, counts)

    def read(self, table, start, n, counts=None, dtype=None, impl=None):
        """k, v (B, H, n, D) and phi, psi (B, H, n) of positions start[b] + i; zero for i >= counts[b].  dtype: of k and v,
        the cache's own, or fp16 (the default) or fp32 for a cache of 8 bits."""
        B = table.shape[0]
        dtype = dtype or (torch.float16 if self.dtype == STORES[2] else self.dtype)
        if n < 1 or B < 1:
            raise ValueError("at least one sequence and one position are read")
        self._check(B, table, dtype, start, "start", counts)
        if pick_impl(impl, self.k) == "reference":
            return dense.read(self, table, start, n, counts, dtype)
        return _hip().read(self, table, start, n, counts, dtype)


def _check_attention(q, cache, beta, table, lengths):
    """Validation of both attention entry points; returns beta as (H,) float32."""
    shape = q.shape
    H = cache.n_heads
    if len(shape) != 4 or shape[1] != H or shape[3] != cache.d_head or shape[0] < 1 or shape[2] < 1:
        raise ValueError(f"q must be (B, {H}, N, {cache.d_head}) with B, N >= 1")
    cache._check(shape[0], table, q.dtype, lengths, "lengths")
    if not torch.is_tensor(beta):
        beta = torch.tensor(float(beta), device=q.device)
    if beta.shape != (H,):
        beta = beta.reshape(-1)
        if beta.numel() == 1:
            beta = beta.expand(H)
        if beta.shape != (H,):
            raise ValueError("beta must have shape (H,) or a single value")
    if q.device != cache.device or beta.device != cache.device:
        raise ValueError(f"q and beta must be on the cache's device, {cache.device}")
    _refuse_grad(q, beta)
    return beta if beta.dtype is torch.float32 else beta.float()


def cached_attention(q, cache, beta, table, lengths, impl=None):
    """o (B, H, N, D) of the last N positions of B sequences against their pages.

    lengths[b] counts all of a sequence's positions, its N new ones, already appended, among them: query i stands at
    t = lengths[b] - N + i and attends to positions s <= t with the bias beta * min(0, min_{s<u<=t} phi_u - psi_s).
    Rows with t < 0 (a sequence shorter than N, an unused slot of the batch) are zero.  Made for few new positions at a
    time, up to 16 or so; any number is computed, 16 rows together.  The memory of o is in (B, N, H, D) order.
    """
    beta = _check_attention(q, cache, beta, table, lengths)
    if pick_impl(impl, q) == "reference":
        return dense.attention(q, cache, beta, table, lengths)
    return _hip().attend(q, cache, beta, table, lengths, None, 0)


def shared_prefix_attention(q, cache, beta, prefix, prefix_length, table, lengths, impl=None):
    """cached_attention for sequences that all continue one prefix: its prefix_length positions stand on the pages
    prefix (n,) int32 of the cache, once, and come before position 0 of every sequence.  table and lengths are those of
    the sequences' own positions.  The rows of all sequences are computed together against the prefix."""
    beta = _check_attention(q, cache, beta, table, lengths)
    prefix_length = int(prefix_length)
    if prefix.dim() != 1 or prefix.dtype != torch.int32 or prefix.device != cache.device:
        raise ValueError("prefix must be a vector of int32 page numbers, on the cache's device")
    if not 0 <= prefix_length <= PAGE * prefix.shape[0]:
        raise ValueError(f"prefix_length must be between 0 and the {PAGE * prefix.shape[0]} positions of its pages")
    if pick_impl(impl, q) == "reference":
        return dense.attention(q, cache, beta, table, lengths, prefix, prefix_length)
    return _hip().attend(q, cache, beta, table, lengths, prefix, prefix_length)
