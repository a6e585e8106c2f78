"""The transformer operators where a value that a row does not use could reach it, and where a score or a scale leaves
the ordinary range, against 64-bit references (transformer_ref.py)."""
import math

import pytest
import torch

import transformer_ref as ref
from test_transformer_ops_gpu import TYPES, Cache, attend_cache, cross, done, gen, randn

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("p", [1, 2])
@pytest.mark.parametrize("queries,keys", [(1, 200), (140, 200), (140, 4000), (300, 130)])
@pytest.mark.parametrize("d", [64, 128])
def test_cross_attention_rows_of_nan(cuda, dav2lib, queries, keys, d, p):
    """A query with a NaN, all of whose scores are NaN, gives NaN; the rows beside it are as without it."""
    g = gen(queries + keys)
    q, k, v = (randn(g, 2, n, 2, d, dtype=TYPES[p]) for n in (queries, keys, keys))
    out = torch.empty(2, queries, 2, d, device="cuda")
    want, bound = ref.cross_attention(q, k, v, [keys, keys], 0.125, p, 0)
    for row in {0, queries // 2, queries - 1}:
        hurt = q.clone()
        hurt[1, row, 1, 3] = math.nan
        cross(dav2lib, hurt, k, v, None, 0.125, out)
        done(dav2lib)
        assert out[1, row, 1].isnan().all()
        keep = torch.ones_like(out, dtype=torch.bool)
        keep[1, row, 1] = False
        assert ref.outside(out[keep], want[keep], bound[keep]) <= 1


@pytest.mark.parametrize("p", [1, 2])
@pytest.mark.parametrize("queries,length", [(1, 200), (140, 200), (140, 4000)])
@pytest.mark.parametrize("d", [64, 128])
def test_cache_attention_rows_of_nan(cuda, dav2lib, queries, length, d, p):
    g = gen(queries + length)
    c = Cache(g, [length], 2, d, 32)
    q = randn(g, queries, 2, d, dtype=TYPES[p])
    out = torch.empty(queries, 2, d, device="cuda")
    want, bound = ref.cache_attention(q, c.k, c.ks, c.v, c.vs, c.table, [length], [0, queries], 0.125, True, 0)
    hurt = q.clone()
    hurt[queries - 1, 1, 3] = math.nan
    attend_cache(dav2lib, c, hurt, [length], [0, queries], True, out, 0.125)
    assert out[-1, 1].isnan().all()
    keep = torch.ones_like(out, dtype=torch.bool)
    keep[-1, 1] = False
    assert ref.outside(out[keep], want[keep], bound[keep]) <= 1
