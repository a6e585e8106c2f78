"""The transformer operators where a value that a row does not use could reach it, and where a score or a scale leaves
the ordinary range, against 64-bit references (transformer_ref.py)."""
import math

import pytest
import torch

import transformer_ref as ref
from test_transformer_ops_gpu import TYPES, Cache, attend_cache, check_cache, cross, done, gen, ints, randn

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


# -------------------------------------------- the tiles kernel (more than 32 rows to a key head) over difficult caches
@pytest.mark.parametrize("queries,causal", [(20, False), (200, True)])
@pytest.mark.parametrize("d,page", [(64, 16), (128, 32), (80, 128)])
def test_cache_attention_scales_far_apart_many_rows(cuda, dav2lib, queries, causal, d, page):
    """V scales from 1e-6 to 1e3 between pages, K scales 0 in some; an all-zero query."""
    g = gen(37)
    c = Cache(g, [900], 2, d, page)
    c.vs *= 10.0 ** torch.randint(-6, 4, c.vs.shape, generator=g, device="cuda")
    c.ks[::3] = 0.0
    q = randn(g, queries, 4, d, dtype=torch.bfloat16)
    q[1] = 0
    out = torch.empty(queries, 4, d, device="cuda")
    attend_cache(dav2lib, c, q, [900], [0, queries], causal, out, 0.125)
    want, bound = ref.cache_attention(q, c.k, c.ks, c.v, c.vs, c.table, [900], [0, queries], 0.125, causal, 0)
    assert ref.outside(out, want, bound) <= 1


@pytest.mark.parametrize("queries", [1, 20, 200])
@pytest.mark.parametrize("d,page", [(64, 16), (128, 32), (128, 64), (96, 128)])
@pytest.mark.parametrize("missing", [[0], [1], [3], [0, 2], [3, 0, 1, 2]])
def test_cache_attention_leaves_out_bad_pages_anywhere(cuda, dav2lib, queries, d, page, missing):
    """Keys of pages that the cache does not have, at the beginning, within and at the end of a sequence, are left out
    and the device error word says so; the neighbour is as always. The kernels check each index before it becomes an
    address."""
    g = gen(38)
    c = Cache(g, [4 * page, 100], 2, d, page)
    q = randn(g, 2 * queries, 4, d, dtype=torch.float16)
    out = torch.empty(2 * queries, 4, d, device="cuda")
    begin = [0, queries, 2 * queries]
    rest = [[x for i, x in enumerate(c.table[0][:4]) if i not in missing], c.table[1]]
    for i, at in enumerate(missing):
        c.table_d[0, at] = -1 - i if i % 2 else c.pages + i
    attend_cache(dav2lib, c, q, [4 * page, 100], begin, False, out, 0.1, expect=3)
    want, bound = ref.cache_attention(q, c.k, c.ks, c.v, c.vs, rest, [page * len(rest[0]), 100], begin, 0.1, False, 0)
    assert ref.outside(out, want, bound) <= 1


@pytest.mark.parametrize("d", [64, 128])
def test_cache_attention_beyond_32_bit_offsets_many_rows(cuda, dav2lib, d):
    """Codes that lie more than 2^32 bytes into the cache, more than 32 rows to a key head."""
    g = gen(39)
    heads, page = 8, 128
    pages = 33000 * 128 // d  # 4.3 GB for K and as much for V
    c = Cache(g, [0], heads, d, page)
    c.k, c.v = (torch.empty((pages, heads, page, d), dtype=torch.int8, device="cuda") for _ in "kv")
    c.ks, c.vs = (torch.ones((pages, heads), device="cuda") for _ in "kv")
    c.pages, c.table = pages, [[pages - 1, 0, pages - 2]]
    c.table_d = ints(c.table)
    small = []
    for codes, scales in ((c.k, c.ks), (c.v, c.vs)):
        for at in c.table[0]:
            codes[at] = torch.randint(-127, 128, (heads, page, d), generator=g, device="cuda", dtype=torch.int8)
            scales[at] = (0.5 + torch.rand(heads, generator=g, device="cuda") * 3) / 127
        at = torch.tensor(c.table[0], device="cuda")
        small += [codes[at], scales[at]]
    q = randn(g, 40, heads, d, dtype=torch.bfloat16)
    out = torch.empty(40, heads, d, device="cuda")
    attend_cache(dav2lib, c, q, [300], [0, 40], True, out, 0.09)
    want, bound = ref.cache_attention(q, *small, [[0, 1, 2]], [300], [0, 40], 0.09, True, 0)
    assert ref.outside(out, want, bound) <= 1


@pytest.mark.parametrize("hq,hkv,d,counts,lengths", [
    (4, 4, 64, [1] * 30 + [300], [200 + 17 * i for i in range(30)] + [900]),          # mean 11 rows: the rows kernel
    (8, 2, 128, [1] * 10 + [400] + [1] * 10, [90 * i for i in range(10)] + [1000] + [31 * i + 1 for i in range(10)])])
@pytest.mark.parametrize("causal", [True, False])
def test_cache_attention_chunk_among_single_tokens(cuda, dav2lib, hq, hkv, d, counts, lengths, causal):
    """One kernel serves a whole call, chosen by the mean: a long chunk beside single tokens is right in either."""
    check_cache(dav2lib, 32, d, hq, hkv, lengths, counts, causal, 2, 0, seed=40)


@pytest.mark.parametrize("hq,hkv,d,length", [(48, 1, 128, 8192), (48, 1, 64, 900), (71, 1, 64, 20003), (128, 2, 128, 1025)])
def test_cache_attention_many_heads_to_a_key_head(cuda, dav2lib, hq, hkv, d, length):
    check_cache(dav2lib, 64, d, hq, hkv, [length], [1], True, 1, 1, seed=41)


@pytest.mark.parametrize("before", [1, 5])
@pytest.mark.parametrize("hq,hkv,d,counts,lengths", [(8, 8, 128, [1], [5000]), (4, 4, 64, [2, 0, 1], [70, 9, 300]),
                                                     (4, 1, 64, [60, 30], [2000, 30]), (2, 2, 128, [300], [4000])])
def test_cache_attention_rows_before_the_first_sequence(cuda, dav2lib, hq, hkv, d, counts, lengths, before):
    """Offsets that begin behind row 0 (a part of a longer batch): the rows before stay as they were."""
    g = gen(42)
    c = Cache(g, lengths, hkv, d, 16)
    begin = [before + sum(counts[:i]) for i in range(len(counts) + 1)]
    q = randn(g, begin[-1], hq, d, dtype=torch.float16)
    q[:before] = math.nan
    out = torch.full((begin[-1], hq, d), 5.0, device="cuda")
    attend_cache(dav2lib, c, q, lengths, begin, True, out, 0.125)
    want, bound = ref.cache_attention(q, c.k, c.ks, c.v, c.vs, c.table, lengths, begin, 0.125, True, 0)
    assert (out[:before] == 5.0).all()
    assert ref.outside(out[before:], want[before:], bound[before:]) <= 1
    cached = [lengths[i] - counts[i] for i in range(len(counts))] if all(a >= b for a, b in zip(lengths, counts)) else [0] * len(counts)
    k = randn(g, begin[-1], hkv, d)
    wk = ref.append(c.k, c.ks, k, c.table, cached, begin)
    wv = ref.append(c.v, c.vs, k, c.table, cached, begin)
    c.append(dav2lib, k, k, cached, begin)
    assert torch.equal(c.k, wk[0]) and torch.equal(c.ks, wk[1]) and torch.equal(c.v, wv[0]) and torch.equal(c.vs, wv[1])


@pytest.mark.parametrize("begin", [[0, 200, 80], [0, -1, 80], [90, 95, 99], [0, 80, 1 << 30], [0, 40, 39]])
def test_cache_attention_leaves_out_bad_offsets(cuda, dav2lib, begin):
    """Offsets out of range or falling set the device error word, and nothing outside the output is touched. The
    kernels check each offset before it becomes an address."""
    g = gen(43)
    c = Cache(g, [300, 200], 2, 64, 16)
    q = randn(g, 80, 2, 64, dtype=torch.float16)
    held = torch.full((80 + 200, 2, 64), 5.0, device="cuda")
    attend_cache(dav2lib, c, q, [300, 200], begin, True, held[100: 180], 0.125, expect=3)
    assert (held[:100] == 5.0).all() and (held[180:] == 5.0).all()


@pytest.mark.parametrize("queries", [1, 100])
def test_cross_attention_cuts_lengths(cuda, dav2lib, queries):
    """Key lengths above the keys, or negative, are cut and set the device error word."""
    g = gen(44)
    q, k, v = (randn(g, 3, n, 2, 64, dtype=torch.float16) for n in (queries, 150, 150))
    out = torch.empty(3, queries, 2, 64, device="cuda")
    for lengths, real in (([151, 20, 1], [150, 20, 1]), ([150, -7, 3], [150, 0, 3]), ([2 ** 31 - 1, -2 ** 31, 150], [150, 0, 150])):
        cross(dav2lib, q, k, v, ints(lengths), 0.125, out)
        done(dav2lib, 3)
        want, bound = ref.cross_attention(q, k, v, real, 0.125, 2, 0)
        assert ref.outside(out, want, bound) <= 1


@pytest.mark.parametrize("queries", [1, 100])
def test_cross_attention_beyond_32_bit_offsets(cuda, dav2lib, queries):
    """Batches that lie more than 2^32 bytes apart, in all four operands."""
    g = gen(45)
    far = (1 << 31) + 64
    store = torch.empty(far + (1 << 20), dtype=torch.float16, device="cuda")

    def place(n, at):
        t = store.as_strided((2, n, 2, 64), (far, 128, 64, 1), at)
        t.copy_(randn(g, 2, n, 2, 64))
        return t

    q, k, v, out = place(queries, 0), place(150, 1 << 16), place(150, 1 << 17), place(queries, 1 << 18)
    cross(dav2lib, q, k, v, ints([150, 77]), 0.125, out)
    done(dav2lib)
    want, bound = ref.cross_attention(q, k, v, [150, 77], 0.125, 2, 2)
    assert ref.outside(out, want, bound) <= 1


def test_large_calls_at_once(cuda, dav2lib):
    """Calls of the tiles kernel on two streams, each with more units than SMs, take over their own units alone: the
    results of lone calls."""
    g = gen(46)
    q, k, v = (randn(g, 8, n, 16, 64, dtype=torch.bfloat16) for n in (700, 600, 600))
    lengths = [ints([600 - 70 * i for i in range(8)]), ints([60 * i for i in range(8)])]
    out = [[torch.empty_like(q) for _ in range(3)] for _ in range(2)]
    streams = [torch.cuda.Stream() for _ in range(2)]
    need = dav2lib.dav2cuda_cross_attention_16_workspace_size(8, 700, 600, 16, 16, 64)
    space = [torch.empty(max(16, need), dtype=torch.uint8, device="cuda") for _ in range(2)]
    for a in range(2):
        cross(dav2lib, q, k, v, lengths[a], 0.125, out[a][0], space[a])
        done(dav2lib)
    for _ in range(4):
        for a in range(2):
            for i in (1, 2):
                with torch.cuda.stream(streams[a]):
                    cross(dav2lib, q, k, v, lengths[a], 0.125, out[a][i], space[a])
    done(dav2lib)
    for a in range(2):
        assert torch.equal(out[a][0], out[a][1]) and torch.equal(out[a][0], out[a][2])
