"""A paged key-value cache whose page tables can be a graph search's answer.

What a language model needs next to the search that finds its passages: the
cache that holds their keys and values in pages, and the operators that write
and read it.  ``Graph.search`` returns int32 [nq, k] ids, -1 where unfilled;
a cache that keeps passage i in page i takes them as they are
(:meth:`PagedCache.adopt`), and the attention skips the pages that are not
there.

* :class:`Rotary` -- rotary positions (half and interleaved pairs, part of a
  head, scaled for long contexts) and their gradient.
* :class:`PagedCache` -- extending, forking, freeing, adopting, compacting and
  copying pages; appending new (rotated) keys and values; the attention of one
  new token of each row.

Tensors are checked and passed on by a small CPython module
(csrc/paged_torch.cc); the kernels are those of libjasper_b200.so
(``jb_rotary``, ``jb_kv_append``, ``jb_pages_*``, ``jb_paged_attention`` in
include/jasper_b200.h).  Calls are asynchronous on torch's current stream of
the cache's device and read nothing back: a row or page that does not fit sets
a bit of the cache's status word, which :meth:`PagedCache.check` reads.  After
a first call they can be captured into CUDA graphs.  The cache is for
inference: a backward pass that reaches the results of append() or attend()
raises, and none goes into the keys and values that it holds.  No reference
counterpart.
"""
from __future__ import annotations

import ctypes as C
import decimal
import math

import torch
from torch.autograd import forward_ad

from . import _lib

__all__ = ["Rotary", "PagedCache"]

_DTYPES = {torch.float16: 0, torch.bfloat16: 1, torch.float32: 2}

_PI = decimal.Decimal("3.14159265358979323846264338327950288419716939937510582097494459")
_DIGITS = decimal.Context(prec=40)  # of frequencies, on their way to 64-bit fixed point

EXHAUSTED, BAD_ROW, BAD_TOKEN = 1, 2, 4
_STATUS = {
    EXHAUSTED: "no free page was left for a row that needed one",
    BAD_ROW: "a row is out of range, named twice, too long for the table or not empty",
    BAD_TOKEN: "a token's place or a page's number is out of range",
}


class Rotary:
    """Rotary positions of heads of ``head_dim`` elements.

    The first ``rot_dim`` elements (default: all) turn by position * theta_i,
    theta_i = base ** (-2 i / rot_dim) for pair i; ``layout`` "half" pairs
    elements i and i + rot_dim / 2, "interleaved" 2 i and 2 i + 1.

    ``scaling`` stretches a model that was trained on ``trained_length``
    tokens by ``factor``: "linear" divides every theta; "ntk" raises the base
    so that the slowest pair slows by the factor and the fastest not at all;
    "yarn" (Peng et al. 2023) divides the thetas of pairs that turn less than
    ``beta_slow`` times over the trained length, keeps those of pairs that
    turn more than ``beta_fast`` times, blends between, and multiplies the
    rotated elements by 0.1 ln(factor) + 1.

    Thetas are kept as 64-bit fixed-point fractions of a turn, rounded once to
    their last unit, so angles are reduced exactly and are off by at most
    2^-65 of a turn a position: no more than a float32 angle's own rounding for
    positions up to 2^39, and known for every int32 or int64.
    """

    def __init__(self, head_dim: int, rot_dim: int | None = None, *, base: float = 10000.0,
                 layout: str = "half", scaling: str | None = None, factor: float = 1.0,
                 trained_length: int = 0, beta_fast: float = 32.0, beta_slow: float = 1.0,
                 device: torch.device | str = "cuda"):
        rot_dim = head_dim if rot_dim is None else rot_dim
        if rot_dim % 2 or not 0 < rot_dim <= head_dim:
            raise ValueError(f"rot_dim must be even, 2 to head_dim ({head_dim}), got {rot_dim}")
        if layout not in ("half", "interleaved"):
            raise ValueError(f"layout must be 'half' or 'interleaved', got {layout!r}")
        if scaling not in (None, "linear", "ntk", "yarn"):
            raise ValueError(f"scaling must be None, 'linear', 'ntk' or 'yarn', got {scaling!r}")
        if not base > 1:
            raise ValueError(f"base must be above 1, got {base}")
        if scaling is not None and not factor > 0:
            raise ValueError(f"factor must be positive, got {factor}")
        if scaling == "ntk" and rot_dim <= 2:
            raise ValueError("scaling 'ntk' needs rot_dim > 2")
        if scaling == "yarn" and trained_length <= 0:
            raise ValueError("scaling 'yarn' needs trained_length")
        self.head_dim, self.rot_dim, self.layout = head_dim, rot_dim, layout
        self.scale = 1.0
        with decimal.localcontext(_DIGITS):
            wide, by = decimal.Decimal(float(base)), decimal.Decimal(float(factor))
            if scaling == "ntk":
                wide *= by ** (decimal.Decimal(rot_dim) / (rot_dim - 2))
            step, theta = wide ** (decimal.Decimal(-2) / rot_dim), [decimal.Decimal(1)]
            for _ in range(rot_dim // 2 - 1):
                theta.append(theta[-1] * step)
            if scaling == "linear":
                theta = [t / by for t in theta]
            elif scaling == "yarn":
                def pair_of(turns):  # the pair that turns so often over the trained length
                    return rot_dim * math.log(trained_length / (turns * 2 * math.pi)) / (2 * math.log(base))
                low = max(math.floor(pair_of(beta_fast)), 0)
                high = min(math.ceil(pair_of(beta_slow)), rot_dim - 1)
                ramp = max(decimal.Decimal(high - low), decimal.Decimal("0.001"))
                slow = [min(1, max(0, (i - low) / ramp)) for i in range(len(theta))]
                theta = [t / by * s + t * (1 - s) for t, s in zip(theta, slow)]
                self.scale = 0.1 * math.log(factor) + 1.0
            radian = 2 ** 64 / (2 * _PI)
            turns = [int((t * radian).to_integral_value()) % 2 ** 64 for t in theta]
        self.theta = [float(t) for t in theta]
        self._freq = torch.tensor([t - 2 ** 64 if t >= 2 ** 63 else t for t in turns],
                                  dtype=torch.int64).to(device)
        self.device = self._freq.device
        self._args = (self._freq, head_dim, rot_dim, self.scale, layout == "interleaved")

    def apply(self, x: torch.Tensor, positions: torch.Tensor,
              out: torch.Tensor | None = None) -> torch.Tensor:
        """``x`` [tokens, heads, head_dim] or [batch, tokens, heads, head_dim]
        (float16, bfloat16 or float32; any strides with contiguous heads)
        turned by ``positions`` (int32 or int64, [tokens] or [batch, tokens]).
        ``out`` may be ``x``.  Differentiable in ``x``, any number of times and
        in forward mode too, unless ``out`` (which must not require a gradient)
        is given."""
        return self._turn(x, positions, out, False)

    __call__ = apply

    def grad(self, dy: torch.Tensor, positions: torch.Tensor,
             out: torch.Tensor | None = None) -> torch.Tensor:
        """The gradient with respect to apply()'s ``x``, given its output's;
        differentiable in ``dy`` as apply() is in ``x``."""
        return self._turn(dy, positions, out, True)

    def _turn(self, x, positions, out, inverse):
        if out is None and (x.requires_grad and torch.is_grad_enabled()
                            or forward_ad.unpack_dual(x).tangent is not None):
            return _Turn.apply(x, positions, self, inverse)
        return _lib.paged_module().rotary(x, positions, out, inverse, *self._args)


class _Turn(torch.autograd.Function):
    """A turn is linear in x, and its transpose is the turn backwards: each is
    the other's gradient, and its own forward derivative."""

    @staticmethod
    def forward(x, positions, rotary, inverse):
        return _lib.paged_module().rotary(x, positions, None, inverse, *rotary._args)

    @staticmethod
    def setup_context(ctx, inputs, output):
        _, positions, ctx.rotary, ctx.inverse = inputs
        ctx.save_for_backward(positions)
        ctx.save_for_forward(positions)

    @staticmethod
    def backward(ctx, dy):
        return ctx.rotary._turn(dy, ctx.saved_tensors[0], None, not ctx.inverse), None, None, None

    @staticmethod
    def jvp(ctx, dx, *_):
        return ctx.rotary._turn(dx, ctx.saved_tensors[0], None, ctx.inverse)


class PagedCache:
    """Keys and values of many rows (conversations) in a pool of pages.

    ``k``, ``v``: float16 or bfloat16 [layers, pages, page_size, kv_heads,
    head_dim], at equal strides with contiguous heads (``allocate`` makes
    them).  ``table`` int32 [rows, max_pages]: a row's pages, -1 for none;
    ``lengths`` int32 [rows]; ``refs`` int32 [pages]: how many rows hold a
    page (0: free).  The tensors stay the caller's: the cache changes them in
    place, and a program may read or write them between calls.  ``marks`` int32
    [rows] (made here if not given) is what the calls note of a row: negative
    while its last extend() was refused, so that append() does not write over
    its last token; the other bits where adopt() ended inside a page; 0 for a
    row whose length and pages the program sets itself.
    """

    def __init__(self, k: torch.Tensor, v: torch.Tensor, table: torch.Tensor, lengths: torch.Tensor,
                 refs: torch.Tensor, status: torch.Tensor | None = None, marks: torch.Tensor | None = None):
        if not k.is_cuda:
            raise ValueError("k must be a CUDA tensor")
        device = k.device
        if k.ndim != 5 or v.shape != k.shape:
            raise ValueError("k and v must be [layers, pages, page_size, kv_heads, head_dim] alike, got "
                             f"{list(k.shape)} and {list(v.shape)}")
        if k.dtype not in (torch.float16, torch.bfloat16) or v.dtype != k.dtype:
            raise ValueError(f"k and v must be float16 or bfloat16 alike, got {k.dtype} and {v.dtype}")
        if v.stride() != k.stride() or k.stride(4) != 1:
            raise ValueError("k and v must have equal strides and contiguous heads")
        n_pages = k.size(1)
        if table.ndim != 2 or (table.size(1) > 1 and table.stride(1) != 1):
            raise ValueError("table must be [rows, max_pages] with contiguous rows")
        if lengths.shape != (table.size(0),) or not lengths.is_contiguous():
            raise ValueError(f"lengths must be a contiguous [{table.size(0)}]")
        if refs.shape != (n_pages,) or not refs.is_contiguous():
            raise ValueError(f"refs must be a contiguous [{n_pages}]")
        if status is None:
            status = torch.zeros(1, dtype=torch.int32, device=device)
        elif status.numel() != 1:
            raise ValueError(f"status must have one element, got {status.numel()}")
        if marks is None:
            marks = torch.zeros(table.size(0), dtype=torch.int32, device=device)
        elif marks.shape != (table.size(0),) or not marks.is_contiguous():
            raise ValueError(f"marks must be a contiguous [{table.size(0)}]")
        for t, name in ((table, "table"), (lengths, "lengths"), (refs, "refs"), (status, "status"),
                        (marks, "marks")):
            if t.dtype != torch.int32:
                raise ValueError(f"{name} must be int32, got {t.dtype}")
        for t, name in ((v, "v"), (table, "table"), (lengths, "lengths"), (refs, "refs"),
                        (status, "status"), (marks, "marks")):
            if t.device != device:
                raise ValueError(f"{name} must be on {device}, got {t.device}")
        self.k, self.v, self.table, self.lengths, self.refs, self.status = k, v, table, lengths, refs, status
        self.marks = marks
        self.device, self.dtype = device, k.dtype
        self.n_layers, self.n_pages, self.page_size, self.n_kv_heads, self.head_dim = k.shape
        self.n_rows, self.max_pages = table.shape
        self._c = _lib.PageCache(
            k.data_ptr(), v.data_ptr(), table.data_ptr(), lengths.data_ptr(), refs.data_ptr(),
            status.data_ptr(), marks.data_ptr(), *k.stride()[:4], table.stride(0), *k.shape, *table.shape,
            _DTYPES[k.dtype], device.index)
        self._ref = C.addressof(self._c)
        self._native = _lib.paged_module()

    @classmethod
    def allocate(cls, n_layers: int, n_pages: int, page_size: int, n_kv_heads: int, head_dim: int,
                 n_rows: int, max_pages: int, dtype: torch.dtype = torch.float16,
                 layout: str = "token", device: torch.device | str = "cuda") -> "PagedCache":
        """An empty cache.  ``layout`` "token" keeps a page's tokens one after
        the other, "head" a page's heads (each with its tokens together)."""
        if layout == "token":
            shape = (n_layers, n_pages, page_size, n_kv_heads, head_dim)
        elif layout == "head":
            shape = (n_layers, n_pages, n_kv_heads, page_size, head_dim)
        else:
            raise ValueError(f"layout must be 'token' or 'head', got {layout!r}")
        k, v = (torch.zeros(shape, dtype=dtype, device=device) for _ in range(2))
        if layout == "head":
            k, v = k.transpose(2, 3), v.transpose(2, 3)
        table = torch.full((n_rows, max_pages), -1, dtype=torch.int32, device=device)
        lengths = torch.zeros(n_rows, dtype=torch.int32, device=device)
        refs = torch.zeros(n_pages, dtype=torch.int32, device=device)
        return cls(k, v, table, lengths, refs)

    # ── pages ──────────────────────────────────────────────────────────
    def extend(self, rows: torch.Tensor, tokens: torch.Tensor) -> None:
        """Room for ``tokens[i]`` more tokens in row ``rows[i]``: pages where
        its last one is full (the lowest free ones), and a length that counts
        them.  Rows are served in order; from the first that finds too few
        free pages on, rows that need pages stay as they were, and append()
        leaves their last token alone until they are extended."""
        self._native.extend(self._ref, rows, tokens)

    def fork(self, parents: torch.Tensor, children: torch.Tensor) -> None:
        """Makes the empty rows ``children`` copies of ``parents``: whole pages
        are shared, a part-filled page is copied, so that each goes on alone."""
        self._native.fork(self._ref, parents, children)

    def free(self, rows: torch.Tensor) -> None:
        """Empties rows; pages that no row holds any more are free."""
        self._native.free(self._ref, rows)

    def adopt(self, rows: torch.Tensor, pages: torch.Tensor, lengths: torch.Tensor | None = None) -> None:
        """Makes the empty rows ``rows`` further holders of ``pages`` (int32
        [len(rows), m]; -1: not there), whole or, with ``lengths``, the first
        lengths[i] tokens of them: a search's ids become rows to attend to.  A
        row that ends so inside a page shares it with holders who may still
        fill it: what follows in that page is not the row's, append() does not
        write it and attend() does not read it.  To go on behind such a row
        fork() it, which copies the tokens that it has there."""
        self._native.adopt(self._ref, rows, pages, lengths)

    def compact(self) -> torch.Tensor:
        """Moves the live pages to the lowest numbers.  Returns int32 [pages]:
        each page's new number, -1 for one that was free."""
        return self._native.compact(self._ref)

    def copy_pages(self, src: torch.Tensor, dst: torch.Tensor) -> None:
        """Copies keys and values of pages ``src`` to pages ``dst``, in every
        layer (no page twice in ``dst``, none in both)."""
        self._native.copy_pages(self._ref, src, dst)

    # ── tokens ─────────────────────────────────────────────────────────
    def append(self, layer: int, k: torch.Tensor, v: torch.Tensor, rows: torch.Tensor,
               index: torch.Tensor | None = None, *, q: torch.Tensor | None = None,
               rotary: Rotary | None = None, positions: torch.Tensor | None = None,
               q_out: torch.Tensor | None = None) -> torch.Tensor | None:
        """Writes keys and values [tokens, kv_heads, head_dim] as tokens
        ``index`` (default: each row's last) of rows ``rows`` (extend() made
        the room; a token of a row that it refused, or in the rest of a page
        that the row was adopted into, is not written).  With ``rotary``, keys are turned by ``positions`` (default:
        the index) on the way, and so is ``q`` [tokens, heads, head_dim], which
        is returned (in ``q_out`` if given, which may be ``q``)."""
        r = (None, 0, 0, 1.0, False) if rotary is None else rotary._args
        return self._native.append(self._ref, layer, k, v, rows, index, q, positions, q_out, *r)

    def attend(self, layer: int, q: torch.Tensor, rows: torch.Tensor | None = None, *,
               scale: float | None = None, window: int = 0, mask: torch.Tensor | None = None,
               return_lse: bool = False, out: torch.Tensor | None = None):
        """Attention of one new token of each row: ``q`` [n, heads, head_dim]
        (heads a multiple of the cache's) over the tokens of rows ``rows``
        (default: the first n).  ``scale`` defaults to head_dim ** -0.5;
        ``window`` > 0 keeps a row's last tokens only; ``mask`` (bool [n,
        width], True: attended to) covers the first width tokens.  Returns [n,
        heads, head_dim], zeros where nothing is attended to; with
        ``return_lse`` also float32 [n, heads], log sum exp of the scores
        (-inf there)."""
        return self._native.attend(self._ref, layer, q, rows, scale, window, mask, return_lse, out)

    def check(self) -> None:
        """Waits for the current stream, and raises what the calls on it since
        the last check() could not do."""
        bits = int(self.status.item())
        if bits:
            self.status.zero_()
            raise _lib.JasperError(_lib.JB_ERR_RUNTIME,
                                   "; ".join(m for b, m in _STATUS.items() if bits & b))

    def __repr__(self) -> str:
        return (f"PagedCache(n_layers={self.n_layers}, n_pages={self.n_pages}, "
                f"page_size={self.page_size}, n_kv_heads={self.n_kv_heads}, head_dim={self.head_dim}, "
                f"n_rows={self.n_rows}, max_pages={self.max_pages}, dtype={self.dtype})")
