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

The kernels are those of libjasper_b200.so (``jb_rotary``, ``jb_kv_append``,
``jb_pages_*``, ``jb_paged_attention`` in include/jasper_b200.h).  Calls are
asynchronous on torch's current stream of the cache's device and read nothing
back: a row or page that does not fit sets a bit of the cache's status word,
which :meth:`PagedCache.check` reads.  No reference counterpart.
"""
from __future__ import annotations

import ctypes as C
import math

import torch

from . import _lib

__all__ = ["Rotary", "PagedCache"]

_DTYPES = {torch.float16: 0, torch.bfloat16: 1, torch.float32: 2}

EXHAUSTED, BAD_ROW, BAD_TOKEN = 1, 2, 4
_STATUS = {
    EXHAUSTED: "no free page was left for a row that needed one",
    BAD_ROW: "a row is out of range, named twice, too long for the table or not empty",
    BAD_TOKEN: "a token's place or a page's number is out of range",
}


def _stream(device: torch.device) -> int:
    return torch.cuda.current_stream(device).cuda_stream


def _heads(t: torch.Tensor, name: str, heads: int | None, dim: int, dtype: torch.dtype,
           device: torch.device) -> torch.Tensor:
    """[tokens, heads, dim] with dim contiguous, on the device."""
    if t.ndim != 3 or t.size(2) != dim or (heads is not None and t.size(1) != heads):
        raise ValueError(f"{name} must be [n, {'heads' if heads is None else heads}, {dim}], "
                         f"got {list(t.shape)}")
    if t.dtype != dtype:
        raise ValueError(f"{name} must be {dtype}, got {t.dtype}")
    if t.device != device:
        raise ValueError(f"{name} must be on {device}, got {t.device}")
    return t if t.stride(2) == 1 or dim == 1 else t.contiguous()


def _ints(t: torch.Tensor, name: str, n: int | None, device: torch.device) -> torch.Tensor:
    if t.dtype != torch.int32 or t.device != device or t.ndim != 1:
        raise ValueError(f"{name} must be a 1D int32 tensor on {device}, got {t.ndim}D {t.dtype} "
                         f"on {t.device}")
    if n is not None and t.size(0) != n:
        raise ValueError(f"{name} must have {n} entries, got {t.size(0)}")
    return t if t.stride(0) == 1 or t.size(0) <= 1 else t.contiguous()


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

    Thetas are kept as 64-bit fixed-point fractions of a turn, so angles are
    reduced exactly: positions may be any int32 or int64.
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
        if scaling is not None and not factor > 0:
            raise ValueError(f"factor must be positive, got {factor}")
        if scaling == "ntk" and rot_dim <= 2:
            raise ValueError("scaling 'ntk' needs rot_dim > 2")
        if scaling == "yarn" and trained_length <= 0:
            raise ValueError("scaling 'yarn' needs trained_length")
        self.head_dim, self.rot_dim, self.layout = head_dim, rot_dim, layout
        self.scale = 1.0
        if scaling == "ntk":
            base = base * factor ** (rot_dim / (rot_dim - 2))
        theta = [base ** (-2.0 * i / rot_dim) for i in range(rot_dim // 2)]
        if scaling == "linear":
            theta = [t / factor for t in theta]
        elif scaling == "yarn":
            def pair_of(turns):  # the pair that turns so often over the trained length
                return rot_dim * math.log(trained_length / (turns * 2 * math.pi)) / (2 * math.log(base))
            low = max(math.floor(pair_of(beta_fast)), 0)
            high = min(math.ceil(pair_of(beta_slow)), rot_dim - 1)
            slow = [min(1.0, max(0.0, (i - low) / max(high - low, 0.001))) for i in range(len(theta))]
            theta = [t / factor * s + t * (1 - s) for t, s in zip(theta, slow)]
            self.scale = 0.1 * math.log(factor) + 1.0
        self.theta = theta
        turns = [round(t / (2 * math.pi) * 2.0 ** 64) % 2 ** 64 for t in theta]
        self._freq = torch.tensor([t - 2 ** 64 if t >= 2 ** 63 else t for t in turns],
                                  dtype=torch.int64).to(device)
        self.device = self._freq.device

    def apply(self, x: torch.Tensor, positions: torch.Tensor,
              out: torch.Tensor | None = None) -> torch.Tensor:
        """``x`` [tokens, heads, head_dim] or [batch, tokens, heads, head_dim]
        (float16, bfloat16 or float32; any strides with contiguous heads)
        turned by ``positions`` (int32 or int64, [tokens] or [batch, tokens]).
        ``out`` may be ``x``.  Differentiable in ``x`` unless ``out`` is given."""
        if out is None and x.requires_grad and torch.is_grad_enabled():
            return _Turn.apply(x, positions, self)
        return self._turn(x, positions, out, False)

    __call__ = apply

    def grad(self, dy: torch.Tensor, positions: torch.Tensor,
             out: torch.Tensor | None = None) -> torch.Tensor:
        """The gradient with respect to apply()'s ``x``, given its output's."""
        return self._turn(dy, positions, out, True)

    def _turn(self, x, positions, out, inverse):
        if out is None:
            out = torch.empty(x.shape, dtype=x.dtype, device=x.device)
        elif out.shape != x.shape or out.dtype != x.dtype or out.device != x.device:
            raise ValueError("out must have x's shape, type and device")
        if x.ndim == 4:
            if out.stride(0) != out.size(1) * out.stride(1) and out.size(0) > 1:
                raise ValueError("out's batch and tokens must be one run of tokens")
            positions = positions.expand(x.shape[:2]).reshape(-1)
            self._turn(x.flatten(0, 1), positions, out.flatten(0, 1), inverse)
            return out
        if x.dtype not in _DTYPES:
            raise ValueError(f"Unsupported tensor dtype: {x.dtype}")
        x = _heads(x, "x", None, self.head_dim, x.dtype, self.device)
        if out.stride(2) != 1:
            raise ValueError("out's heads must be contiguous")
        n = x.size(0)
        p64 = positions.dtype == torch.int64
        if not p64 and positions.dtype != torch.int32:
            raise ValueError(f"positions must be int32 or int64, got {positions.dtype}")
        if positions.shape != (n,) or positions.device != self.device:
            raise ValueError(f"positions must be [{n}] on {self.device}")
        positions = positions.contiguous()
        args = (x.data_ptr(), x.stride(0), x.stride(1), out.data_ptr(), out.stride(0), out.stride(1),
                _DTYPES[x.dtype], n, x.size(1), self.head_dim, self.rot_dim, positions.data_ptr(), p64,
                self._freq.data_ptr(), self.scale, self.layout == "interleaved", inverse,
                _stream(self.device))
        if torch.cuda.current_device() == self.device.index:
            _lib.call("jb_rotary", *args)
        else:
            with torch.cuda.device(self.device):
                _lib.call("jb_rotary", *args)
        return out


class _Turn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, positions, rotary):
        ctx.rotary = rotary
        ctx.save_for_backward(positions)
        return rotary._turn(x, positions, None, False)

    @staticmethod
    def backward(ctx, dy):
        return ctx.rotary._turn(dy, ctx.saved_tensors[0], None, True), None, None


class PagedCache:
    """Keys and values of many rows (conversations) in a pool of pages.

    ``k``, ``v``: float16 or bfloat16 [layers, pages, page_size, kv_heads,
    head_dim], at equal strides with contiguous heads (``allocate`` makes
    them).  ``table`` int32 [rows, max_pages]: a row's pages, -1 for none;
    ``lengths`` int32 [rows]; ``refs`` int32 [pages]: how many rows hold a
    page (0: free).  The tensors stay the caller's: the cache changes them in
    place, and a program may read or write them between calls.
    """

    def __init__(self, k: torch.Tensor, v: torch.Tensor, table: torch.Tensor, lengths: torch.Tensor,
                 refs: torch.Tensor, status: torch.Tensor | None = None):
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
        for t, name in ((table, "table"), (lengths, "lengths"), (refs, "refs"), (status, "status")):
            if t.dtype != torch.int32:
                raise ValueError(f"{name} must be int32, got {t.dtype}")
        for t, name in ((v, "v"), (table, "table"), (lengths, "lengths"), (refs, "refs"),
                        (status, "status")):
            if t.device != device:
                raise ValueError(f"{name} must be on {device}, got {t.device}")
        self.k, self.v, self.table, self.lengths, self.refs, self.status = k, v, table, lengths, refs, status
        self.device, self.dtype = device, k.dtype
        self.n_layers, self.n_pages, self.page_size, self.n_kv_heads, self.head_dim = k.shape
        self.n_rows, self.max_pages = table.shape
        self._c = _lib.PageCache(
            k.data_ptr(), v.data_ptr(), table.data_ptr(), lengths.data_ptr(), refs.data_ptr(),
            status.data_ptr(), *k.stride()[:4], table.stride(0), *k.shape, *table.shape,
            _DTYPES[k.dtype], device.index)
        self._ref = C.addressof(self._c)

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
        free pages on, rows that need pages stay as they were."""
        rows = _ints(rows, "rows", None, self.device)
        tokens = _ints(tokens, "tokens", rows.size(0), self.device)
        _lib.call("jb_pages_extend", self._ref, rows.data_ptr(), tokens.data_ptr(), rows.size(0),
                  _stream(self.device))

    def fork(self, parents: torch.Tensor, children: torch.Tensor) -> None:
        """Makes the empty rows ``children`` copies of ``parents``: whole pages
        are shared, a part-filled page is copied, so that each goes on alone."""
        parents = _ints(parents, "parents", None, self.device)
        children = _ints(children, "children", parents.size(0), self.device)
        _lib.call("jb_pages_fork", self._ref, parents.data_ptr(), children.data_ptr(),
                  parents.size(0), _stream(self.device))

    def free(self, rows: torch.Tensor) -> None:
        """Empties rows; pages that no row holds any more are free."""
        rows = _ints(rows, "rows", None, self.device)
        _lib.call("jb_pages_free", self._ref, rows.data_ptr(), rows.size(0), _stream(self.device))

    def adopt(self, rows: torch.Tensor, pages: torch.Tensor, lengths: torch.Tensor | None = None) -> None:
        """Makes the empty rows ``rows`` further holders of ``pages`` (int32
        [len(rows), m]; -1: not there), whole or, with ``lengths``, the first
        lengths[i] tokens of them: a search's ids become rows to attend to."""
        rows = _ints(rows, "rows", None, self.device)
        if pages.dtype != torch.int32 or pages.ndim != 2 or pages.device != self.device:
            raise ValueError(f"pages must be a 2D int32 tensor on {self.device}")
        if pages.size(0) != rows.size(0):
            raise ValueError(f"pages must have {rows.size(0)} rows, got {pages.size(0)}")
        if pages.size(1) > 1 and pages.stride(1) != 1:
            pages = pages.contiguous()
        if lengths is not None:
            lengths = _ints(lengths, "lengths", rows.size(0), self.device)
        _lib.call("jb_pages_adopt", self._ref, rows.data_ptr(), pages.data_ptr(), pages.stride(0),
                  pages.size(1), None if lengths is None else lengths.data_ptr(), rows.size(0),
                  _stream(self.device))

    def compact(self) -> torch.Tensor:
        """Moves the live pages to the lowest numbers.  Returns int32 [pages]:
        each page's new number, -1 for one that was free."""
        remap = torch.empty(self.n_pages, dtype=torch.int32, device=self.device)
        _lib.call("jb_pages_compact", self._ref, remap.data_ptr(), _stream(self.device))
        return remap

    def copy_pages(self, src: torch.Tensor, dst: torch.Tensor) -> None:
        """Copies keys and values of pages ``src`` to pages ``dst``, in every
        layer (no page twice in ``dst``, none in both)."""
        src = _ints(src, "src", None, self.device)
        dst = _ints(dst, "dst", src.size(0), self.device)
        _lib.call("jb_pages_copy", self._ref, src.data_ptr(), dst.data_ptr(), src.size(0),
                  _stream(self.device))

    # ── tokens ─────────────────────────────────────────────────────────
    def append(self, layer: int, k: torch.Tensor, v: torch.Tensor, rows: torch.Tensor,
               index: torch.Tensor | None = None, *, q: torch.Tensor | None = None,
               rotary: Rotary | None = None, positions: torch.Tensor | None = None,
               q_out: torch.Tensor | None = None) -> torch.Tensor | None:
        """Writes keys and values [tokens, kv_heads, head_dim] as tokens
        ``index`` (default: each row's last) of rows ``rows`` (extend() made
        the room).  With ``rotary``, keys are turned by ``positions`` (default:
        the index) on the way, and so is ``q`` [tokens, heads, head_dim], which
        is returned (in ``q_out`` if given, which may be ``q``)."""
        dev, dim = self.device, self.head_dim
        k = _heads(k, "k", self.n_kv_heads, dim, self.dtype, dev)
        v = _heads(v, "v", self.n_kv_heads, dim, self.dtype, dev)
        n = k.size(0)
        if v.size(0) != n:
            raise ValueError(f"v must have {n} tokens, got {v.size(0)}")
        rows = _ints(rows, "rows", n, dev)
        if index is not None:
            index = _ints(index, "index", n, dev)
        if q is None:
            q_args = (None, 0, 0, None, 0, 0, 0)
        else:
            if rotary is None:
                raise ValueError("q is only taken to be rotated: pass rotary")
            q = _heads(q, "q", None, dim, self.dtype, dev)
            if q.size(0) != n:
                raise ValueError(f"q must have {n} tokens, got {q.size(0)}")
            if q_out is None:
                q_out = torch.empty(q.shape, dtype=q.dtype, device=dev)
            elif q_out.shape != q.shape or q_out.dtype != q.dtype or q_out.device != dev or q_out.stride(2) != 1:
                raise ValueError("q_out must have q's shape, type and device, and contiguous heads")
            q_args = (q.data_ptr(), q.stride(0), q.stride(1), q_out.data_ptr(), q_out.stride(0),
                      q_out.stride(1), q.size(1))
        p64 = False
        if positions is not None:
            p64 = positions.dtype == torch.int64
            if (not p64 and positions.dtype != torch.int32) or positions.shape != (n,) or positions.device != dev:
                raise ValueError(f"positions must be int32 or int64 [{n}] on {dev}")
            positions = positions.contiguous()
        if rotary is None:
            r_args = (None, 0, 1.0, 0)
        elif rotary.head_dim != dim or rotary.device != dev:
            raise ValueError(f"rotary must be for heads of {dim} on {dev}")
        else:
            r_args = (rotary._freq.data_ptr(), rotary.rot_dim, rotary.scale, rotary.layout == "interleaved")
        _lib.call("jb_kv_append", self._ref, layer, n, *q_args, k.data_ptr(), k.stride(0), k.stride(1),
                  v.data_ptr(), v.stride(0), v.stride(1), rows.data_ptr(),
                  None if index is None else index.data_ptr(),
                  None if positions is None else positions.data_ptr(), p64, *r_args, _stream(dev))
        return q_out if q is not None else None

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
        dev = self.device
        q = _heads(q, "q", None, self.head_dim, self.dtype, dev)
        n, heads, dim = q.shape
        if heads % self.n_kv_heads:
            raise ValueError(f"q's heads ({heads}) must be a multiple of the cache's ({self.n_kv_heads})")
        if q.stride(0) % 8 or q.stride(1) % 8 or q.data_ptr() % 16:
            q = q.contiguous()
            if q.data_ptr() % 16:
                q = q.clone()
        if rows is not None:
            rows = _ints(rows, "rows", n, dev)
        elif n > self.n_rows:
            raise ValueError(f"q has {n} rows, the cache {self.n_rows}")
        if window < 0:
            raise ValueError(f"window must not be negative, got {window}")
        if mask is None:
            m_args = (None, 0, 0)
        else:
            if mask.dtype != torch.bool or mask.ndim != 2 or mask.size(0) != n or mask.device != dev:
                raise ValueError(f"mask must be bool [{n}, width] on {dev}")
            if mask.size(1) > 1 and mask.stride(1) != 1:
                mask = mask.contiguous()
            m_args = (mask.data_ptr(), mask.stride(0), mask.size(1))
        if out is None:
            out = torch.empty((n, heads, dim), dtype=q.dtype, device=dev)
        elif out.shape != q.shape or out.dtype != q.dtype or out.device != dev or out.stride(2) != 1:
            raise ValueError("out must have q's shape, type and device, and contiguous heads")
        lse = torch.empty((n, heads), dtype=torch.float32, device=dev) if return_lse else None
        _lib.call("jb_paged_attention", self._ref, layer, q.data_ptr(), q.stride(0), q.stride(1),
                  out.data_ptr(), out.stride(0), out.stride(1), n, heads,
                  None if rows is None else rows.data_ptr(), *m_args, window,
                  dim ** -0.5 if scale is None else scale, None if lse is None else lse.data_ptr(),
                  _stream(dev))
        return (out, lse) if return_lse else out

    def check(self) -> None:
        """Waits for the cache's stream, and raises what the calls since the
        last check() could not do."""
        bits = int(self.status.item())
        if bits:
            self.status.zero_()
            raise _lib.JasperError(_lib.JB_ERR_RUNTIME,
                                   "; ".join(m for b, m in _STATUS.items() if bits & b))

    def __repr__(self) -> str:
        return (f"PagedCache(n_layers={self.n_layers}, n_pages={self.n_pages}, "
                f"page_size={self.page_size}, n_kv_heads={self.n_kv_heads}, head_dim={self.head_dim}, "
                f"n_rows={self.n_rows}, max_pages={self.max_pages}, dtype={self.dtype})")
