"""Refusals of the paged cache's C entry points that come before any CUDA
call: no GPU is needed."""
import ctypes as C

import pytest

from jasper_b200 import _lib


def cache(**kw):
    """A cache whose pointers are never followed: every call here is refused."""
    f = dict(k=4096, v=4096, table=4096, lengths=4096, refs=4096, status=4096, layer_stride=2048, page_stride=1024,
             token_stride=64, head_stride=32, table_stride=4, n_layers=2, n_pages=8, page_size=16, n_kv_heads=2,
             head_dim=32, n_rows=3, max_pages=4, dtype=0, device=0)
    return C.byref(_lib.PageCache(**{**f, **kw}))


def test_a_rows_last_token_needs_marks():
    with pytest.raises(ValueError, match="marks"):
        _lib.call("jb_kv_append", cache(), 0, 1, None, 0, 0, None, 0, 0, 0, 4096, 0, 0, 4096, 0, 0, 4096, None, None,
                  0, None, 0, 1.0, 0, None)


def test_adopting_part_of_a_page_needs_marks():
    with pytest.raises(ValueError, match="marks"):
        _lib.call("jb_pages_adopt", cache(), 4096, 4096, 4, 4, 4096, 1, None)
