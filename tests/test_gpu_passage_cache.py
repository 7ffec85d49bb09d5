"""The example that answers from retrieved passages: search, cache and
operators together."""
import importlib.util
from pathlib import Path

import pytest
import torch

pytestmark = pytest.mark.gpu


def test_search_cache_and_attention_together(cuda):
    path = Path(__file__).resolve().parents[1] / "examples" / "passage_cache.py"
    spec = importlib.util.spec_from_file_location("passage_cache", path)
    example = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(example)
    n, requests = 3000, 9
    r = example.run(n_passages=n, n_requests=requests, tokens=10, k=6, layers=2, heads=8, kv_heads=2, page_size=16,
                    verbose=False)
    ids = r["ids"]
    assert ids.shape == (requests, 6) and ids.dtype == torch.int32
    assert ((ids >= -1) & (ids < n)).all()
    for row in ids.tolist():
        found = [i for i in row if i >= 0]
        assert found and len(set(found)) == len(found)
    # a fork reads exactly what its parent reads
    assert torch.equal(r["same"][:requests], r["same"][requests:])
    assert not torch.equal(r["states"][:requests], r["states"][requests:])
    assert torch.isfinite(r["states"].float()).all()
    # freeing the others and moving pages changes nothing for those who stay
    assert torch.equal(r["before"], r["after"])
    cache = r["cache"]
    held = (cache.table >= 0).sum(1)
    assert held[0] == n and (held[2:1 + requests] == 0).all() and (held[2 + requests:] == 0).all()
    assert cache.refs.sum() == held.sum()
    assert r["free"] == cache.n_pages - int((cache.refs > 0).sum())
    live = int((cache.refs > 0).sum())
    assert (cache.refs[:live] > 0).all()
