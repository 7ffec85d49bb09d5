"""What of the paged cache needs no GPU: rotary frequencies, and the C entry
points' refusals, which come before any CUDA call."""
import ctypes as C
import math

import pytest
import torch

from jasper_b200 import _lib, paged


def test_frequencies_are_turns_in_fixed_point():
    r = paged.Rotary(128, 64, base=500_000.0, device="cpu")
    assert len(r.theta) == 32 and r.theta[0] == 1.0
    for theta, f in zip(r.theta, r._freq.tolist()):
        # a float64's last bits (its own, pi's and the quotient's), and half a unit of 2^-64 of a turn
        assert abs(f / 2.0 ** 64 * 2 * math.pi - theta) <= theta * 2.0 ** -50 + math.pi * 2.0 ** -64


def test_scaled_frequencies():
    plain = paged.Rotary(64, device="cpu").theta
    linear = paged.Rotary(64, scaling="linear", factor=4.0, device="cpu")
    assert linear.theta == [t / 4.0 for t in plain] and linear.scale == 1.0
    ntk = paged.Rotary(64, scaling="ntk", factor=4.0, device="cpu").theta
    assert ntk[0] == plain[0] and abs(ntk[-1] * 4.0 / plain[-1] - 1) < 1e-12
    yarn = paged.Rotary(64, scaling="yarn", factor=4.0, trained_length=4096, device="cpu")
    assert abs(yarn.scale - (0.1 * math.log(4.0) + 1)) < 1e-15
    ratio = [p / y for p, y in zip(plain, yarn.theta)]
    assert ratio[0] == 1.0 and abs(ratio[-1] - 4.0) < 1e-12 and ratio == sorted(ratio)
    for p, y in zip(plain, ratio):  # pairs that turn over 32 times keep their theta, those under once are divided
        turns = 4096 * p / (2 * math.pi)
        assert y == 1.0 if turns > 64 else abs(y - 4.0) < 1e-12 if turns < 0.5 else 1.0 <= y <= 4.0


@pytest.mark.parametrize("kw", [{"rot_dim": 3}, {"rot_dim": 0}, {"rot_dim": 66}, {"layout": "pairs"},
                                {"scaling": "other"}, {"scaling": "linear", "factor": 0.0},
                                {"scaling": "ntk", "factor": 2.0, "rot_dim": 2}, {"scaling": "yarn", "factor": 2.0},
                                {"base": 1.0}, {"base": -3.0}])
def test_rotary_refusals(kw):
    with pytest.raises(ValueError):
        paged.Rotary(64, device="cpu", **kw)


def test_a_cache_lives_on_a_gpu():
    k = torch.zeros(1, 2, 4, 1, 8, dtype=torch.float16)
    t = torch.zeros(2, dtype=torch.int32)
    with pytest.raises(ValueError, match="CUDA"):
        paged.PagedCache(k, k, torch.zeros(2, 2, dtype=torch.int32), t, t)


def cache(**kw):
    """A cache whose pointers are never followed: every call here is refused."""
    f = dict(k=4096, v=4096, table=4096, lengths=4096, refs=4096, status=4096, layer_stride=2048, page_stride=1024,
             token_stride=64, head_stride=32, table_stride=4, n_layers=2, n_pages=8, page_size=16, n_kv_heads=2,
             head_dim=32, n_rows=3, max_pages=4, dtype=0, device=0)
    return C.byref(_lib.PageCache(**{**f, **kw}))


@pytest.mark.parametrize("kw,message", [
    ({"dtype": 2}, "dtype"), ({"dtype": -1}, "dtype"), ({"head_dim": 12}, "head_dim"), ({"head_dim": 0}, "head_dim"),
    ({"head_dim": 264}, "head_dim"), ({"page_size": 0}, "page_size"), ({"n_kv_heads": 0}, "n_kv_heads"),
    ({"n_pages": 2 ** 30}, "n_pages"), ({"table": None}, "null"), ({"status": None}, "null"), ({"k": None}, "null"),
    ({"k": 4104}, "aligned"), ({"token_stride": 36}, "strides"), ({"page_stride": 1}, "strides"),
    ({"table_stride": 3}, "table_stride"), ({"max_pages": 2 ** 31}, "max_pages")])
def test_refused_caches(kw, message):
    calls = [("jb_pages_extend", 4096, 4096, 1, None), ("jb_pages_fork", 4096, 4096, 1, None),
             ("jb_pages_free", 4096, 1, None), ("jb_pages_adopt", 4096, 4096, 1, 1, None, 1, None),
             ("jb_pages_compact", 4096, None), ("jb_pages_copy", 4096, 4096, 1, None),
             ("jb_kv_append", 0, 1, None, 0, 0, None, 0, 0, 0, 4096, 0, 0, 4096, 0, 0, 4096, None, None, 0, None, 0,
              1.0, 0, None),
             ("jb_paged_attention", 0, 4096, 64, 32, 4096, 64, 32, 1, 2, None, None, 0, 0, 0, 1.0, None, None)]
    for name, *args in calls:
        with pytest.raises(ValueError, match=message):
            _lib.call(name, cache(**kw), *args)
        with pytest.raises(ValueError, match="null"):
            _lib.call(name, None, *args)


def test_refused_arguments():
    at = dict(layer=0, q=4096, qr=64, qh=32, out=4096, orow=64, oh=32, n=1, heads=2, rows=None, mask=None, ms=0, mw=0,
              window=0, scale=1.0, lse=None, stream=None)
    for kw, message in (({"layer": 2}, "layer"), ({"heads": 3}, "multiple"), ({"q": None}, "null"),
                        ({"out": None}, "null"), ({"q": 4100}, "16"), ({"qr": 65}, "16"), ({"oh": 36}, "16"),
                        ({"scale": math.nan}, "scale"), ({"n": 2 ** 30}, "rows")):
        with pytest.raises(ValueError, match=message):
            _lib.call("jb_paged_attention", cache(), *{**at, **kw}.values())
    with pytest.raises(ValueError, match="2\\^31"):
        _lib.call("jb_paged_attention", cache(max_pages=2 ** 28, table_stride=2 ** 28), *at.values())
    ro = dict(x=4096, xt=64, xh=32, y=4096, yt=64, yh=32, dtype=0, n=1, heads=2, dim=32, rot=32, pos=4096, p64=0,
              freq=4096, scale=1.0, inter=0, inverse=0, stream=None)
    for kw, message in (({"dtype": 3}, "dtype"), ({"rot": 33}, "rot_dim"), ({"rot": 34}, "rot_dim"),
                        ({"dim": 0}, "head_dim"), ({"freq": None}, "null"), ({"pos": None}, "null")):
        with pytest.raises(ValueError, match=message):
            _lib.call("jb_rotary", *{**ro, **kw}.values())
    for name in ("jb_pages_fork", "jb_pages_copy"):
        with pytest.raises(ValueError, match="too many pages"):
            _lib.call(name, cache(n_layers=2 ** 20), 4096, 4096, 1025, None)
        with pytest.raises(ValueError, match="too large"):
            _lib.call(name, cache(page_size=2 ** 20, n_kv_heads=65536), 4096, 4096, 1, None)
    with pytest.raises(ValueError, match="more pages"):
        _lib.call("jb_pages_adopt", cache(), 4096, 4096, 5, 5, None, 1, None)


def test_nothing_to_do_is_no_error():
    _lib.call("jb_pages_free", cache(), None, 0, None)
    _lib.call("jb_pages_extend", cache(), None, None, 0, None)
    _lib.call("jb_rotary", None, 0, 0, None, 0, 0, 0, 0, 2, 32, 32, None, 0, None, 1.0, 0, 0, None)
