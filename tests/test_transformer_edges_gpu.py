"""The transformer operators where a value that a row does not use could reach it, and where a score or a scale leaves
the ordinary range, against 64-bit references (transformer_ref.py)."""
import math

import pytest
import torch

import transformer_ref as ref
from test_transformer_ops_gpu import TYPES, Cache, attend_cache, cross, done, gen, ints, randn

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


@pytest.mark.parametrize("up", [20, 40, 110])
@pytest.mark.parametrize("queries,length,page", [(2, 161, 16), (2, 2945, 64), (100, 161, 16), (100, 3009, 64), (300, 385, 128)])
@pytest.mark.parametrize("d", [64, 128])
def test_cache_attention_large_values_behind_the_mask(cuda, dav2lib, queries, length, page, d, up):
    """The last token's page has V scales 2^up times the others': rows that do not see it are as without it."""
    g = gen(32)
    c = Cache(g, [length], 2, d, page)
    begin = [0, queries]
    q = randn(g, queries, 4, d, dtype=torch.bfloat16)
    seen = max(0, (length - 1) // page * page - length + queries)  # rows that see earlier pages only
    assert seen
    want, bound = ref.cache_attention(q, c.k, c.ks, c.v, c.vs, c.table, [length], begin, 0.125, True, 0)
    c.vs[c.table[0][(length - 1) // page]] *= 2.0 ** up
    out = torch.empty(queries, 4, d, device="cuda")
    attend_cache(dav2lib, c, q, [length], begin, True, out, 0.125)
    assert ref.outside(out[:seen], want[:seen], bound[:seen]) <= 1
    want, bound = ref.cache_attention(q, c.k, c.ks, c.v, c.vs, c.table, [length], begin, 0.125, True, 0)
    assert ref.outside(out[seen:], want[seen:], bound[seen:]) <= 1


@pytest.mark.parametrize("where", [0, 4, 9])
@pytest.mark.parametrize("queries", [2, 100])
@pytest.mark.parametrize("d", [64, 128])
def test_cache_attention_large_values_without_weight(cuda, dav2lib, queries, d, where):
    """A page of keys 400 and more below the others in score, with V scales 2^60 times theirs: as without it."""
    g = gen(33)
    c = Cache(g, [160], 2, d, 16)
    c.k[..., 5] = 0
    q = randn(g, queries, 4, d, dtype=torch.float16)
    q[..., 5] = 16.0
    hot = c.table[0][where]
    pages = [p for p in c.table[0] if p != hot]
    want, bound = ref.cache_attention(q, c.k, c.ks, c.v, c.vs, [pages], [144], [0, queries], 0.125, False, 0)
    # its scores are 0.125 * 16 * -127 * 2 = -508; the others', of normal q and |k| <= 3.5, are some units from 0
    c.k[hot] = 0
    c.k[hot, :, :, 5] = -127
    c.ks[hot] = 2.0
    c.vs[hot] *= 2.0 ** 60
    out = torch.empty(queries, 4, d, device="cuda")
    attend_cache(dav2lib, c, q, [160], [0, queries], False, out, 0.125)
    assert ref.outside(out, want, bound) <= 1


@pytest.mark.parametrize("queries", [1, 140])
@pytest.mark.parametrize("d", [64, 128])
def test_cache_attention_infinite_queries(cuda, dav2lib, queries, d):
    """A query with -inf beside values above f16's range: keys that it scores -inf are left out (zeros if there is no
    other), one of inf makes the row NaN."""
    g = gen(35)
    c = Cache(g, [150], 2, d, 32)
    c.k[..., 5], c.k[..., 6] = 1, 1
    q = randn(g, queries, 2, d, dtype=torch.bfloat16)
    want, bound = ref.cache_attention(q, c.k, c.ks, c.v, c.vs, c.table, [150], [0, queries], 0.125, False, 0)
    hurt = q.clone()
    hurt[0, 1, 5], hurt[0, 1, 6] = -math.inf, 1e30
    keep = torch.ones(queries, 2, d, dtype=torch.bool, device="cuda")
    keep[0, 1] = False
    out = torch.empty(queries, 2, d, device="cuda")
    attend_cache(dav2lib, c, hurt, [150], [0, queries], False, out, 0.125)
    assert (out[0, 1] == 0).all()
    assert ref.outside(out[keep], want[keep], bound[keep]) <= 1
    hurt[0, 1, 5], hurt[0, 1, 6] = math.inf, -1e30
    attend_cache(dav2lib, c, hurt, [150], [0, queries], False, out, 0.125)
    assert out[0, 1].isnan().all()
    assert ref.outside(out[keep], want[keep], bound[keep]) <= 1


@pytest.mark.parametrize("low", [-math.inf, -1e4])
@pytest.mark.parametrize("queries", [1, 140])
@pytest.mark.parametrize("d", [64, 128])
def test_cross_attention_keys_without_weight(cuda, dav2lib, queries, d, low):
    """Keys whose score is -inf, or 1250 and more below the others, weigh nothing, however large their values: as
    without them."""
    g = gen(31)
    q, k, v = (randn(g, 1, n, 2, d, dtype=torch.bfloat16) for n in (queries, 150, 150))
    q[..., 5], k[..., 5] = 1.0, 0.0
    gone = list(range(0, 150, 7))
    k[:, gone, :, 5], v[:, gone] = low, 3e38
    out = torch.empty(1, queries, 2, d, device="cuda")
    cross(dav2lib, q, k, v, None, 0.125, out)
    done(dav2lib)
    rest = [i for i in range(150) if i not in gone]
    want, bound = ref.cross_attention(q, k[:, rest], v[:, rest], [len(rest)], 0.125, 1, 0)
    assert ref.outside(out, want, bound) <= 1


@pytest.mark.parametrize("queries", [1, 140])
@pytest.mark.parametrize("d", [64, 128])
def test_attention_scale_zero_of_large_products(cuda, dav2lib, queries, d):
    """scale 0 weighs all keys alike, however large q . k is, as long as it is finite."""
    g = gen(34)
    q, k, v = (randn(g, 1, n, 2, d, dtype=torch.bfloat16) for n in (queries, 150, 150))
    q, k = q * 2.0 ** 60, k * 2.0 ** 60
    out = torch.empty(1, queries, 2, d, device="cuda")
    want, bound = ref.cross_attention(q * 0, k * 0, v, [150], 0.0, 1, 0)
    for scale in (0.0, -0.0, 1e-44):
        cross(dav2lib, q, k, v, None, scale, out)
        done(dav2lib)
        assert ref.outside(out, want, bound) <= 1
    for low in (math.inf, -math.inf):  # 0 times an infinite product is NaN
        hurt = k.clone()
        hurt[0, 7, 1, 5] = low
        cross(dav2lib, q, hurt, v, None, 0.0, out)
        done(dav2lib)
        assert out[:, :, 1].isnan().all() and ref.outside(out[:, :, 0], want[:, :, 0], bound[:, :, 0]) <= 1
        cross(dav2lib, q, hurt, v, ints([7]), 0.0, out)
        done(dav2lib)
        short, within = ref.cross_attention(q * 0, k * 0, v, [7], 0.0, 1, 0)
        assert ref.outside(out, short, within) <= 1
    c = Cache(g, [150], 2, d, 16)
    want, bound = ref.cache_attention(q[0] * 0, c.k, c.ks, c.v, c.vs, c.table, [150], [0, queries], 0.0, False, 0)
    c.ks *= 2.0 ** 50
    attend_cache(dav2lib, c, q[0], [150], [0, queries], False, out[0], 0.0)
    assert ref.outside(out[0], want, bound) <= 1


@pytest.mark.parametrize("p,po", [(1, 0), (2, 2)])
@pytest.mark.parametrize("batch,queries,keys,hq,hkv,d", [
    (3, 1, 70, 4, 2, 64), (2, 5, 130, 4, 4, 128), (3, 140, 200, 4, 2, 64), (2, 300, 1000, 8, 2, 128), (3, 70, 90, 6, 2, 72)])
def test_cross_attention_sequence_first(cuda, dav2lib, batch, queries, keys, hq, hkv, d, p, po):
    """q, k, v and the output as [tokens][batch][heads][dim]: batch strides below the token strides."""
    g = gen(36)
    q, k, v = (randn(g, n, batch, h, d, dtype=TYPES[p]).transpose(0, 1) for n, h in ((queries, hq), (keys, hkv), (keys, hkv)))
    held = torch.full((queries + 1, batch, hq, d), 5.0, dtype=TYPES[po], device="cuda")
    out, lengths = held[:queries].transpose(0, 1), [keys - 7 * b for b in range(batch)]
    cross(dav2lib, q, k, v, ints(lengths), 0.125, out)
    done(dav2lib)
    want, bound = ref.cross_attention(q, k, v, lengths, 0.125, p, po)
    assert ref.outside(out, want, bound) <= 1
    assert (held[queries:] == 5.0).all()
