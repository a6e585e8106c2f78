"""The transformer operators on the GPU against 64-bit references (transformer_ref.py, whose bounds count the kernels'
roundings): norm and rotary positions of q and k, the 8-bit key/value cache, its attention, cross attention, and a
decoder's steps through all of them. The cache's codes and scales are held to equality."""
import math

import pytest
import torch

import transformer_ref as ref

pytestmark = pytest.mark.gpu

TYPES = ref.TYPES


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def randn(g, *shape, dtype=torch.float32):
    return torch.randn(shape, generator=g, device="cuda").to(dtype)


def ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def ptr(t):
    return None if t is None else t.data_ptr()


def ok(lib, rc):
    assert rc == 0, lib.dav2cuda_last_error()


def done(lib, code=0):
    torch.cuda.synchronize()
    assert lib.dav2cuda_device_error() == code


def stream():
    return torch.cuda.current_stream().cuda_stream


# ------------------------------------------------------------ norm and rotary
def rope(lib, q, k, qo, ko, w, f, pos, rotary, axes, norm, layout, rotary_scale=1.0, eps=1e-6):
    """q, k, qo, ko: [tokens, heads, d] views whose heads are contiguous, or None."""
    some = q if q is not None else k
    p = {v: n for n, v in TYPES.items()}
    st = lambda x: 0 if x is None else x.stride(0)  # noqa: E731
    ok(lib, lib.dav2cuda_qk_norm_rope(
        ptr(qo), ptr(ko), ptr(q), ptr(k), ptr(w[0]), ptr(w[1]), ptr(w[2]), ptr(w[3]), ptr(f), ptr(pos), some.shape[0],
        0 if q is None else q.shape[1], 0 if k is None else k.shape[1], some.shape[2], rotary, axes, st(qo), st(ko),
        st(q), st(k), norm, eps, layout, rotary_scale, p[some.dtype], p[(qo if qo is not None else ko).dtype], stream()))


def check_rope(lib, tokens, hq, hk, d, rotary, axes, layout, norm, pin, pout, seed=0, pad=0, reach=5000,
               weights="all", rotary_scale=1.0, in_place=False):
    g = gen(seed)
    row = (hq + 2 * hk) * d + pad
    qkv = randn(g, tokens, row, dtype=TYPES[pin]) * 2 + 0.25
    view = lambda t, at, h: t[:, at: at + h * d].unflatten(1, (h, d)) if h else None  # noqa: E731
    q, k = view(qkv, 0, hq), view(qkv, hq * d, hk)
    w = [1 + 0.3 * randn(g, d), 0.2 * randn(g, d), 1 - 0.3 * randn(g, d), 0.2 * randn(g, d)]
    if weights == "none":
        w = [None] * 4
    elif weights == "no bias":
        w[1] = w[3] = None
    f = (10000.0 ** (-torch.arange(rotary // 2 // axes, device="cuda").double() / max(1, rotary // 2 // axes)))
    f = f.float().repeat(axes) if rotary else None
    pos = torch.randint(-reach, reach, (tokens, axes), generator=g, device="cuda", dtype=torch.int32)
    want = [ref.norm_rope(x, w[2 * i], w[2 * i + 1], f, pos, rotary, axes, layout, norm, 1e-6, rotary_scale)
            for i, x in enumerate((q, k)) if x is not None]
    out = qkv if in_place else torch.full((tokens, row), 7.0, dtype=TYPES[pout], device="cuda")
    before = out.clone()
    qo, ko = view(out, 0, hq), view(out, hq * d, hk)
    rope(lib, q, k, qo, ko, w, f, pos, rotary, axes, norm, layout, rotary_scale)
    done(lib)
    for got, (y, size) in zip([x for x in (qo, ko) if x is not None], want):
        worst = ref.outside(got, y, ref.norm_rope_bound(y, size, pout))
        assert worst <= 1, worst
    assert torch.equal(out[:, (hq + hk) * d:], before[:, (hq + hk) * d:])  # v and the padding stay


@pytest.mark.parametrize("pin,pout", [(0, 0), (0, 1), (0, 2), (1, 1), (2, 2)])
@pytest.mark.parametrize("norm", [0, 1, 2])
@pytest.mark.parametrize("layout", [0, 1, 2])
def test_qk_norm_rope_types(cuda, dav2lib, pin, pout, norm, layout):
    check_rope(dav2lib, 37, 6, 2, 64, 64, 2, layout, norm, pin, pout, seed=norm)


@pytest.mark.parametrize("tokens,hq,hk,d,rotary,axes,layout,pad", [
    (1, 1, 1, 2, 2, 1, 0, 0), (1, 32, 8, 128, 128, 1, 0, 0), (3, 5, 0, 80, 40, 2, 2, 0), (5, 0, 3, 96, 48, 1, 1, 0),
    (2, 3, 1, 256, 256, 1, 0, 0), (7, 3, 2, 72, 66, 3, 0, 0), (7, 3, 2, 72, 66, 3, 2, 0), (9, 2, 2, 254, 250, 1, 1, 0),
    (11, 4, 4, 64, 0, 1, 0, 0), (13, 16, 16, 64, 32, 1, 0, 3), (2500, 4, 2, 128, 64, 1, 1, 8), (1370, 3, 3, 64, 64, 2, 0, 1),
    (2, 300, 100, 16, 16, 1, 0, 0)])
@pytest.mark.parametrize("norm", [0, 2])
def test_qk_norm_rope_shapes(cuda, dav2lib, tokens, hq, hk, d, rotary, axes, layout, pad, norm):
    """Single tokens, odd heads, head sizes that are no power of two, partial rotation, unaligned rows."""
    check_rope(dav2lib, tokens, hq, hk, d, rotary, axes, layout, norm, 1, 1, seed=tokens + d, pad=pad)


@pytest.mark.parametrize("weights", ["none", "no bias"])
@pytest.mark.parametrize("norm", [1, 2])
def test_qk_norm_rope_without_weights(cuda, dav2lib, weights, norm):
    check_rope(dav2lib, 20, 4, 4, 64, 64, 1, 0, norm, 0, 2, weights=weights)


@pytest.mark.parametrize("layout", [0, 1])
@pytest.mark.parametrize("tokens", [5, 3000])
def test_qk_norm_rope_in_place_and_far(cuda, dav2lib, layout, tokens):
    """In place on the packed rows; positions up to +-2^31 - 1, where f32 angles would be noise; scaled rotation."""
    check_rope(dav2lib, tokens, 4, 2, 128, 64, 1, layout, 1, 2, 2, reach=2 ** 31 - 1, rotary_scale=1.3, in_place=True)


def test_rope_without_positions_counts_tokens(cuda, dav2lib):
    g = gen(1)
    x = randn(g, 50, 2, 64, dtype=torch.float16)
    f = torch.linspace(1, 0.01, 32, device="cuda")
    a, b = torch.empty_like(x), torch.empty_like(x)
    rope(dav2lib, x, None, a, None, [None] * 4, f, None, 64, 1, 0, 0)
    rope(dav2lib, x, None, b, None, [None] * 4, f, ints(list(range(50)))[:, None], 64, 1, 0, 0)
    done(dav2lib)
    assert torch.equal(a, b)


# ---------------------------------------------------------------------- cache
class Cache:
    """A paged cache for sequences of given capacities, pages shuffled, unused table places -1."""

    def __init__(self, g, capacity, heads, d, page, spare=2):
        need = [-(-c // page) for c in capacity]
        self.pages, self.page, self.heads, self.d = sum(need) + spare, page, heads, d
        order = torch.randperm(self.pages, generator=g, device="cuda").tolist()
        width = max(need + [1])
        self.table, at = [], 0
        for n in need:
            self.table.append(order[at: at + n] + [-1] * (width - n))
            at += n
        self.table_d = ints(self.table)
        shape = (self.pages, heads, page, d)
        self.k, self.v = (torch.randint(-128, 128, shape, generator=g, device="cuda", dtype=torch.int8) for _ in "kv")
        self.ks, self.vs = ((0.5 + torch.rand(shape[:2], generator=g, device="cuda") * 3) / 127 for _ in "kv")

    def append(self, lib, k, v, cached, begin, expect=0):
        p = {t: n for n, t in TYPES.items()}[k.dtype]
        held, rows = ints(cached), ints(begin)  # named: a temporary's memory would be handed to the next one
        ok(lib, lib.dav2cuda_kv_cache_append_s8(
            ptr(self.k), ptr(self.ks), ptr(self.v), ptr(self.vs), ptr(k), ptr(v), ptr(self.table_d), ptr(held),
            ptr(rows), len(cached), k.shape[0], self.heads, self.d, self.pages, self.page,
            self.table_d.shape[1], k.stride(0), v.stride(0), p, stream()))
        done(lib, expect)


@pytest.mark.parametrize("p", [0, 1, 2])
@pytest.mark.parametrize("page,d,heads,cached,counts", [
    (16, 64, 2, [0], [1]), (16, 128, 3, [15, 16, 0, 5], [1, 1, 0, 27]), (32, 96, 1, [31, 3], [33, 29]),
    (64, 16, 2, [0, 64, 100], [64, 1, 200]), (128, 128, 2, [127, 1, 0], [1, 126, 385]), (16, 80, 5, [7] * 9, [1] * 9)])
def test_append(cuda, dav2lib, p, page, d, heads, cached, counts):
    """Codes, scales and everything around them equal the definition's; scales that grow requantize their page."""
    g = gen(page + d)
    c = Cache(g, [a + b for a, b in zip(cached, counts)], heads, d, page)
    begin = [sum(counts[:i]) for i in range(len(counts) + 1)]
    both = randn(g, begin[-1] + 3, 2 * heads * d + 16, dtype=TYPES[p])  # rows behind the last sequence are not read
    both[0] *= 3
    both[begin[-1]:] = math.nan
    k = both[:, : heads * d].unflatten(1, (heads, d))
    v = both[:, heads * d + 16:].unflatten(1, (heads, d))
    wk = ref.append(c.k, c.ks, k, c.table, cached, begin)
    wv = ref.append(c.v, c.vs, v, c.table, cached, begin)
    c.append(dav2lib, k, v, cached, begin)
    for got, want in ((c.k, wk[0]), (c.ks, wk[1]), (c.v, wv[0]), (c.vs, wv[1])):
        assert torch.equal(got, want)


def test_append_special_values(cuda, dav2lib):
    """Zeros, tiny values, infinities and NaN; half-way quotients; an old scale that covers the new rows."""
    g = gen(3)
    c = Cache(g, [16, 40, 24], 1, 16, 16)
    c.ks[c.table[2][0]] = 100.0
    k = randn(g, 16 + 30 + 20, 1, 16)
    k[:16] = 0
    k[20, 0, 3], k[21, 0, 4], k[22, 0, 5] = math.inf, -math.inf, math.nan
    k[40, 0] = torch.arange(16, device="cuda") / 2
    k[40, 0, 0] = 127.0
    k[50:] *= 1e-9
    v = k.flip(0).contiguous()
    cached, begin = [0, 10, 4], [0, 16, 46, 66]
    wk, wv = (ref.append(a, b, x, c.table, cached, begin) for a, b, x in ((c.k, c.ks, k), (c.v, c.vs, v)))
    c.append(dav2lib, k, v, cached, begin)
    assert torch.equal(c.k, wk[0]) and torch.equal(c.ks, wk[1])
    assert torch.equal(c.v, wv[0]) and torch.equal(c.vs, wv[1])
    assert torch.isfinite(c.ks).all() and c.ks.min() >= 1e-8


def test_append_leaves_out_what_is_out_of_range(cuda, dav2lib):
    """A page that is not in the cache and a table that is too short: those rows are left out, the others stored, and
    the device error word says so. The kernel checks each index before it becomes an address."""
    g = gen(4)
    c = Cache(g, [16, 16, 32], 2, 32, 16)
    k, v = randn(g, 50, 2, 32), randn(g, 50, 2, 32)
    want = ref.append(c.k, c.ks, k[:10], c.table, [0], [0, 10])
    c.table_d[1, 0] = c.pages
    before = c.k.clone()
    c.append(dav2lib, k, v, [0, 0, 30], [0, 10, 14, 50], expect=3)  # 30 + 36 tokens: more than two pages
    first, last = c.table[0][0], c.table[2][1]
    assert torch.equal(c.k[first], want[0][first]) and torch.equal(c.ks[first], want[1][first])
    assert not torch.equal(c.k[last], before[last])
    untouched = [i for i in range(c.pages) if i not in (first, last)]
    assert torch.equal(c.k[untouched], before[untouched])
    c.append(dav2lib, k, v, [0, -1, 0], [0, 10, 9, 60], expect=3)


def attend_cache(lib, c, q, lengths, begin, causal, out, scale, longest=None, workspace=None, expect=0):
    p = {t: n for n, t in TYPES.items()}
    longest = max(lengths) if longest is None else longest
    lengths_d, begin_d = ints(lengths), ints(begin)
    args = (len(lengths), q.shape[0], longest, q.shape[1], c.heads, c.d)
    if workspace is None:
        workspace = torch.full((max(16, lib.dav2cuda_attention_cache_s8_workspace_size(*args)),), 255, dtype=torch.uint8, device="cuda")
    ok(lib, lib.dav2cuda_attention_cache_s8(
        ptr(out), ptr(q), ptr(c.k), ptr(c.ks), ptr(c.v), ptr(c.vs), ptr(c.table_d), ptr(lengths_d), ptr(begin_d),
        *args, c.pages, c.page, c.table_d.shape[1], q.stride(0), out.stride(0), scale, int(causal), p[q.dtype],
        p[out.dtype], ptr(workspace), workspace.numel(), stream()))
    done(lib, expect)


def check_cache(lib, page, d, hq, hkv, lengths, counts, causal, p, po, seed=0, extra=2, spread=1.0):
    g = gen(seed)
    c = Cache(g, lengths, hkv, d, page)
    begin = [sum(counts[:i]) for i in range(len(counts) + 1)]
    rows = randn(g, begin[-1] + extra, hq * d + 24, dtype=TYPES[p]) * spread
    q = rows[:, 16: 16 + hq * d].unflatten(1, (hq, d))
    q[begin[-1]:] = math.nan
    out = torch.full((begin[-1] + extra, hq * d + 8), 5.0, dtype=TYPES[po], device="cuda")
    o = out[:, : hq * d].unflatten(1, (hq, d))
    attend_cache(lib, c, q, lengths, begin, causal, o, 1 / math.sqrt(d))
    want, bound = ref.cache_attention(q, c.k, c.ks, c.v, c.vs, c.table, lengths, begin, 1 / math.sqrt(d), causal, po)
    n = begin[-1]
    worst = ref.outside(o[:n], want[:n], bound[:n])
    assert worst <= 1, worst
    assert (out[n:] == 5.0).all() and (out[:, hq * d:] == 5.0).all()


@pytest.mark.parametrize("p,po", [(1, 1), (1, 0), (2, 2), (2, 0)])
@pytest.mark.parametrize("page,d,hq,hkv,lengths,counts,causal", [
    (16, 64, 4, 4, [1], [1], True), (16, 64, 4, 4, [0, 17, 0], [1, 1, 2], True), (32, 128, 8, 2, [33, 500, 64], [1, 1, 1], True),
    (64, 128, 32, 8, [3000, 1, 777], [1, 1, 1], True), (128, 96, 6, 2, [129, 128], [3, 5], True),
    (16, 16, 3, 1, [50, 49], [7, 0], False), (64, 80, 10, 2, [300], [9], True), (32, 112, 16, 1, [257], [1], False),
    (16, 48, 2, 2, [40, 3], [40, 5], True), (64, 128, 16, 2, [700, 90], [70, 90], True), (64, 64, 12, 4, [1370], [200], False),
    (128, 128, 8, 8, [5000], [1], True), (16, 32, 40, 2, [64, 2100, 31], [1, 2, 3], True)])
def test_cache_attention(cuda, dav2lib, page, d, hq, hkv, lengths, counts, causal, p, po):
    """One token to long lengths, empty sequences and caches shorter than their queries (rows that see nothing), shared
    heads from one to twenty, head sizes between the tiles, splits of the keys, rows of no sequence."""
    check_cache(dav2lib, page, d, hq, hkv, lengths, counts, causal, p, po, seed=d + hq)


@pytest.mark.parametrize("p", [1, 2])
@pytest.mark.parametrize("spread", [1e-4, 30.0])
def test_cache_attention_sharp_and_flat(cuda, dav2lib, p, spread):
    """Scores that are all alike and scores that leave one key; queries far from 1 in their type."""
    check_cache(dav2lib, 64, 128, 8, 2, [2000, 100], [1, 1], True, p, 0, spread=spread)


def test_cache_attention_scales_far_apart(cuda, dav2lib):
    """V scales from 1e-6 to 1e3 between pages, K scales 0 in some; an all-zero query."""
    g = gen(9)
    c = Cache(g, [900], 2, 64, 16)
    c.vs *= 10.0 ** torch.randint(-6, 4, c.vs.shape, generator=g, device="cuda")
    c.ks[::3] = 0.0
    q = randn(g, 3, 4, 64, dtype=torch.bfloat16)
    q[1] = 0
    out = torch.empty(3, 4, 64, device="cuda")
    attend_cache(dav2lib, c, q, [900], [0, 3], False, out, 0.125)
    want, bound = ref.cache_attention(q, c.k, c.ks, c.v, c.vs, c.table, [900], [0, 3], 0.125, False, 0)
    assert ref.outside(out, want, bound) <= 1


def test_cache_attention_leaves_out_bad_pages(cuda, dav2lib):
    """Keys of a page that the cache does not have are left out, a length above max_length is cut, and the device
    error word says so. The kernel checks each index before it becomes an address."""
    g = gen(5)
    c = Cache(g, [64, 64], 2, 64, 16)
    q = randn(g, 2, 4, 64, dtype=torch.float16)
    out = torch.empty(2, 4, 64, device="cuda")
    good = c.table
    c.table_d[0, 3] = c.pages + 5  # the last 16 of sequence 0's keys
    attend_cache(dav2lib, c, q, [64, 64], [0, 1, 2], False, out, 0.1, expect=3)
    want, bound = ref.cache_attention(q, c.k, c.ks, c.v, c.vs, good, [48, 64], [0, 1, 2], 0.1, False, 0)
    assert ref.outside(out, want, bound) <= 1
    attend_cache(dav2lib, c, q, [48, 70], [0, 1, 2], False, out, 0.1, longest=64, expect=3)
    assert ref.outside(out, want, bound) <= 1
    attend_cache(dav2lib, c, q, [48, -3], [0, 1, 2], False, out, 0.1, longest=64, expect=3)
    assert (out[1] == 0).all()
    attend_cache(dav2lib, c, q, [48, 64], [0, 5, 2], False, out, 0.1, longest=64, expect=3)


def test_cache_beyond_32_bit_offsets(cuda, dav2lib):
    """Codes that lie more than 2^32 bytes into the cache: append to the last pages and attend to them."""
    g = gen(6)
    heads, d, page, pages = 8, 128, 128, 33000  # 4.3 GB for K and as much for V
    c = Cache(g, [0], heads, d, page)
    c.k, c.v = (torch.empty((pages, heads, page, d), dtype=torch.int8, device="cuda") for _ in "kv")
    c.ks, c.vs = (torch.ones((pages, heads), device="cuda") for _ in "kv")
    c.pages, c.table = pages, [[pages - 1, 0, pages - 2]]
    c.table_d = ints(c.table)
    k, v = randn(g, 300, heads, d, dtype=torch.bfloat16), randn(g, 300, heads, d, dtype=torch.bfloat16)
    c.append(dav2lib, k, v, [0], [0, 300])
    at = torch.tensor(c.table[0], device="cuda")
    small = [torch.zeros((3, heads, page, d), dtype=torch.int8, device="cuda"), torch.ones((3, heads), device="cuda")]
    wk, wv = (ref.append(*small, x, [[0, 1, 2]], [0], [0, 300]) for x in (k, v))
    flat = lambda x: x.transpose(1, 2).flatten(0, 1)[:300]  # noqa: E731
    assert torch.equal(flat(c.k[at]), flat(wk[0])) and torch.equal(flat(c.v[at]), flat(wv[0]))
    q = randn(g, 4, heads, d, dtype=torch.bfloat16)
    out = torch.empty(4, heads, d, device="cuda")
    attend_cache(dav2lib, c, q, [300], [0, 4], True, out, 0.09)
    want, bound = ref.cache_attention(q, *wk, *wv, [[0, 1, 2]], [300], [0, 4], 0.09, True, 0)
    assert ref.outside(out, want, bound) <= 1


# ---------------------------------------------------------------------- cross
def cross(lib, q, k, v, lengths, scale, out, workspace=None):
    p = {t: n for n, t in TYPES.items()}
    b, n, hq, d = q.shape
    args = (b, n, k.shape[1], hq, k.shape[2], d)
    if workspace is None:
        workspace = torch.full((max(16, lib.dav2cuda_cross_attention_16_workspace_size(*args)),), 255, dtype=torch.uint8, device="cuda")
    ok(lib, lib.dav2cuda_cross_attention_16(
        ptr(out), ptr(q), ptr(k), ptr(v), ptr(lengths), *args, q.stride(0), q.stride(1), k.stride(0), k.stride(1),
        v.stride(0), v.stride(1), out.stride(0), out.stride(1), scale, p[q.dtype], p[out.dtype], ptr(workspace),
        workspace.numel(), stream()))


def check_cross(lib, batch, queries, keys, hq, hkv, d, lengths, p, po, seed=0, spread=1.0):
    g = gen(seed)
    q = randn(g, batch, queries, hq, d, dtype=TYPES[p]) * spread
    kv = randn(g, batch, max(keys, 1), 2, hkv, d, dtype=TYPES[p])[:, :keys]
    k, v = kv[:, :, 0], kv[:, :, 1]
    real = lengths or [keys] * batch
    clean = kv.clone()
    for b, n in enumerate(real):  # what masked places hold must not matter
        kv[b, n:] = math.nan
        kv[b, n: n + 1, :, :, ::2] = math.inf
        kv[b, n + 1: n + 3] = torch.finfo(TYPES[p]).min
    out = torch.full((batch, queries + 1, hq * d + 8), 5.0, dtype=TYPES[po], device="cuda")
    o = out[:, :queries, : hq * d].unflatten(2, (hq, d))
    lengths_d = ints(lengths) if lengths else None
    cross(lib, q, k, v, lengths_d, 1 / math.sqrt(d), o)
    done(lib)
    want, bound = ref.cross_attention(q, clean[:, :, 0], clean[:, :, 1], real, 1 / math.sqrt(d), p, po)
    worst = ref.outside(o, want, bound)
    assert worst <= 1, worst
    assert (out[:, queries:] == 5.0).all() and (out[..., hq * d:] == 5.0).all()


@pytest.mark.parametrize("p,po", [(1, 1), (1, 0), (2, 2), (2, 0)])
@pytest.mark.parametrize("batch,queries,keys,hq,hkv,d,lengths", [
    (1, 1, 1, 1, 1, 8, None), (2, 1, 33, 4, 4, 64, [33, 0]), (3, 1, 1370, 16, 16, 64, [1370, 7, 900]),
    (1, 1, 4001, 32, 8, 128, None), (2, 5, 100, 6, 2, 80, [1, 100]), (2, 129, 65, 2, 1, 64, [64, 65]),
    (1, 300, 700, 4, 4, 128, [513]), (2, 257, 1000, 8, 2, 128, [1000, 128]), (1, 128, 128, 3, 3, 64, None),
    (2, 200, 0, 2, 2, 64, None), (2, 200, 190, 2, 2, 72, [0, 190]), (1, 1370, 1370, 6, 6, 64, None),
    (3, 130, 260, 12, 4, 96, [260, 3, 129]), (1, 640, 2000, 2, 2, 40, [1999]), (2, 40, 500, 16, 2, 128, [500, 449])])
def test_cross_attention(cuda, dav2lib, batch, queries, keys, hq, hkv, d, lengths, p, po):
    check_cross(dav2lib, batch, queries, keys, hq, hkv, d, lengths, p, po, seed=keys + d)


@pytest.mark.parametrize("queries", [1, 200])
@pytest.mark.parametrize("spread", [1e-4, 30.0])
def test_cross_attention_sharp_and_flat(cuda, dav2lib, queries, spread):
    check_cross(dav2lib, 2, queries, 900, 4, 2, 64, [900, 600], 1, 0, spread=spread)


@pytest.mark.parametrize("scale", [0.0, -0.2])
@pytest.mark.parametrize("queries", [1, 300])
def test_attention_scale_zero_and_negative(cuda, dav2lib, scale, queries):
    g = gen(15)
    q, k, v = (randn(g, 2, n, 4, 64, dtype=torch.float16) for n in (queries, 333, 333))
    out, lengths = torch.empty(2, queries, 4, 64, device="cuda"), ints([333, 190])
    cross(dav2lib, q, k, v, lengths, scale, out)
    done(dav2lib)
    want, bound = ref.cross_attention(q, k, v, [333, 190], scale, 2, 0)
    assert ref.outside(out, want, bound) <= 1
    c = Cache(g, [333, 500], 2, 64, 32)
    q = q.flatten(0, 1)
    out = torch.empty(2 * queries, 4, 64, device="cuda")
    attend_cache(dav2lib, c, q, [333, 500], [0, queries, 2 * queries], True, out, scale)
    want, bound = ref.cache_attention(q, c.k, c.ks, c.v, c.vs, c.table, [333, 500], [0, queries, 2 * queries], scale, True, 0)
    assert ref.outside(out, want, bound) <= 1


@pytest.mark.parametrize("p", [1, 2])
@pytest.mark.parametrize("hq,hkv,d", [(16, 16, 64), (8, 2, 128), (12, 4, 64), (6, 2, 128)])
def test_cross_attention_more_units_than_sms(cuda, dav2lib, hq, hkv, d, p):
    """Several units of work to an SM, some without keys, some of one row tile; groups that divide a tile and groups
    that do not."""
    batch = 40
    lengths = [(i * 53) % 334 if i % 5 else 0 for i in range(batch)]
    check_cross(dav2lib, batch, 300, 333, hq, hkv, d, lengths, p, p, seed=hq)


@pytest.mark.parametrize("hq,hkv,d,page,causal", [(8, 8, 64, 16, True), (16, 4, 128, 128, True), (12, 4, 96, 64, False)])
def test_cache_attention_more_units_than_sms(cuda, dav2lib, hq, hkv, d, page, causal):
    n = 45
    counts = [(i * 17) % 160 for i in range(n)]
    lengths = [max(0, c + (i * 31) % 300 - 20) if i % 6 else 0 for i, c in enumerate(counts)]
    check_cache(dav2lib, page, d, hq, hkv, lengths, counts, causal, 2, 2, seed=n)


@pytest.mark.parametrize("queries", [2, 260])
def test_cross_attention_shared_states_and_queries(cuda, dav2lib, queries):
    """Batch strides of 0: one encoder's states for every batch entry, one set of queries for several encoders."""
    g = gen(16)
    q, k, v = (randn(g, 3, n, h, 64, dtype=torch.bfloat16) for n, h in ((queries, 4), (150, 2), (150, 2)))
    out, lengths = torch.empty(3, queries, 4, 64, device="cuda"), ints([150, 20, 0])
    for qq, kk, vv in ((q, k[:1].expand(3, -1, -1, -1), v[1:2].expand(3, -1, -1, -1)),
                       (q[:1].expand(3, -1, -1, -1), k, v)):
        cross(dav2lib, qq, kk, vv, lengths, 0.125, out)
        done(dav2lib)
        want, bound = ref.cross_attention(qq, kk, vv, [150, 20, 0], 0.125, 1, 0)
        assert ref.outside(out, want, bound) <= 1


@pytest.mark.parametrize("queries", [1, 140])
@pytest.mark.parametrize("d", [64, 128])
def test_cross_attention_nan_stays_where_it_is(cuda, dav2lib, queries, d):
    """A NaN that a row sees makes that row NaN, and no other."""
    g = gen(17)
    q, k, v = (randn(g, 2, n, 2, d, dtype=torch.float16) for n in (queries, 200, 200))
    for key in range(0, 130, 13):
        kk = k.clone()
        kk[1, key, 1, 5] = math.nan
        out = torch.empty(2, queries, 2, d, device="cuda")
        cross(dav2lib, q, kk, v, None, 0.125, out)
        done(dav2lib)
        assert out[1, :, 1].isnan().all()
        want, bound = ref.cross_attention(q, k, v, [200, 200], 0.125, 2, 0)
        keep = torch.ones_like(out, dtype=torch.bool)
        keep[1, :, 1] = False
        assert ref.outside(out[keep], want[keep], bound[keep]) <= 1


@pytest.mark.parametrize("queries", [1, 140])
@pytest.mark.parametrize("d", [64, 128])
def test_cross_attention_infinite_scores(cuda, dav2lib, queries, d):
    """A score of inf makes the row NaN, as inf - inf does in the formula; one of -inf leaves its key out."""
    g = gen(18)
    q, k, v = (randn(g, 1, n, 2, d, dtype=torch.bfloat16) for n in (queries, 150, 150))
    for key in range(0, 150, 7):
        kk = k.clone()
        kk[0, key, 1, 5] = math.inf
        out = torch.empty(1, queries, 2, d, device="cuda")
        cross(dav2lib, q, kk, v, None, 0.125, out)
        done(dav2lib)
        lost = torch.zeros(1, queries, 2, dtype=torch.bool, device="cuda")
        lost[0, :, 1] = ~(q[0, :, 1, 5] < 0)
        assert out[lost].isnan().all()
        want, bound = ref.cross_attention(q, k, v, [150], 0.125, 1, 0)
        rest = [i for i in range(150) if i != key]
        without = ref.cross_attention(q[:, :, 1:], k[:, rest, 1:], v[:, rest, 1:], [149], 0.125, 1, 0)
        want[:, :, 1:], bound[:, :, 1:] = without
        assert ref.outside(out[~lost], want[~lost], bound[~lost]) <= 1


@pytest.mark.parametrize("queries", [1, 140])
@pytest.mark.parametrize("d", [64, 128])
def test_cache_attention_infinite_scores(cuda, dav2lib, queries, d):
    g = gen(19)
    q = randn(g, queries, 2, d, dtype=torch.float16)
    hot = q.clone()
    hot[0, 1, 5] = math.inf
    for key in range(0, 150, 7):
        c = Cache(gen(20), [150], 2, d, 32)
        c.k[..., 5] = -1
        c.k[c.table[0][key // 32], 1, key % 32, 5] = 1
        out = torch.empty(queries, 2, d, device="cuda")
        attend_cache(dav2lib, c, hot, [150], [0, queries], False, out, 0.125)
        assert out[0, 1].isnan().all()
        want, bound = ref.cache_attention(q, c.k, c.ks, c.v, c.vs, c.table, [150], [0, queries], 0.125, False, 0)
        keep = torch.ones_like(out, dtype=torch.bool)
        keep[0, 1] = False
        assert ref.outside(out[keep], want[keep], bound[keep]) <= 1


def test_attention_in_captured_graphs(cuda, dav2lib):
    """Large calls captured into two graphs that share a workspace, replayed in turn on a side stream with new inputs."""
    g = gen(18)
    c = Cache(g, [900, 300, 0], 2, 128, 32)
    lengths, counts = [900, 300, 0], [200, 100, 40]
    begin = [0, 200, 300, 340]
    lengths_d, begin_d = ints(lengths), ints(begin)
    q = randn(g, 340, 8, 128, dtype=torch.float16)
    x, k, v = randn(g, 2, 700, 4, 64, dtype=torch.float16), randn(g, 2, 800, 4, 64, dtype=torch.float16), randn(g, 2, 800, 4, 64, dtype=torch.float16)
    o1, o2 = torch.empty(340, 8, 128, device="cuda"), torch.empty(2, 700, 4, 64, device="cuda")
    args = (3, 340, 900, 8, 2, 128)
    size = max(16, dav2lib.dav2cuda_attention_cache_s8_workspace_size(*args),
               dav2lib.dav2cuda_cross_attention_16_workspace_size(2, 700, 800, 4, 4, 64))
    ws = torch.empty(size, dtype=torch.uint8, device="cuda")

    def first():
        ok(dav2lib, dav2lib.dav2cuda_attention_cache_s8(
            ptr(o1), ptr(q), ptr(c.k), ptr(c.ks), ptr(c.v), ptr(c.vs), ptr(c.table_d), ptr(lengths_d), ptr(begin_d), *args,
            c.pages, c.page, c.table_d.shape[1], 1024, 1024, 0.1, 1, 2, 0, ptr(ws), size, stream()))

    def second():
        cross(dav2lib, x, k, v, None, 0.125, o2, ws)

    side, graphs = torch.cuda.Stream(), []
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        for call in (first, second):
            call()  # sets the kernels up
            torch.cuda.synchronize()
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=side):
                call()
            graphs.append(graph)
        for _ in range(3):
            q.copy_(randn(g, 340, 8, 128, dtype=torch.float16))
            x.copy_(randn(g, 2, 700, 4, 64, dtype=torch.float16))
            for graph in graphs:
                graph.replay()
            side.synchronize()
            want, bound = ref.cache_attention(q, c.k, c.ks, c.v, c.vs, c.table, lengths, begin, 0.1, True, 0)
            assert ref.outside(o1, want, bound) <= 1
            want, bound = ref.cross_attention(x, k, v, [800, 800], 0.125, 2, 0)
            assert ref.outside(o2, want, bound) <= 1
    done(dav2lib)


def test_cross_attention_rows_in_any_order(cuda, dav2lib):
    """Batch and token strides of slices, q as a part of packed rows, k and v from different tensors."""
    g = gen(2)
    q = randn(g, 3, 50, 3, 4, 64, dtype=torch.float16)[:, ::2, 1]
    k = randn(g, 4, 90, 2, 64, dtype=torch.float16)[1:]
    v = randn(g, 3, 100, 4, 2, 64, dtype=torch.float16)[:, 5:95, 2]
    out = torch.empty(3, 25, 4, 64, dtype=torch.float16, device="cuda")
    cross(dav2lib, q, k, v, None, 0.125, out)
    done(dav2lib)
    want, bound = ref.cross_attention(q, k, v, [90] * 3, 0.125, 2, 2)
    assert ref.outside(out, want, bound) <= 1


# ------------------------------------------------------------------- together
class Decoder:
    """One layer of a streaming decoder through the C ABI: qkv linear (f16 operands), head norms and rotary positions,
    cache append, attention over the cache, cross attention to an encoder's states; and the same in 64 bits from the
    values that each stage was given."""

    D, HQ, HKV, HD, PAGE = 256, 8, 2, 64, 16

    def __init__(self, lib, sequences, capacity):
        self.lib, g = lib, gen(11)
        self.cache = Cache(g, [capacity] * sequences, self.HKV, self.HD, self.PAGE)
        rows = (self.HQ + 2 * self.HKV) * self.HD
        self.w, self.b = randn(g, rows, self.D) / 16, randn(g, rows) / 8
        self.qw, self.kw = 1 + 0.1 * randn(g, self.HD), 1 + 0.1 * randn(g, self.HD)
        self.f = torch.linspace(1, 0.001, self.HD // 2, device="cuda")
        self.states = randn(g, sequences, 77, 2, self.HKV, self.HD, dtype=torch.bfloat16)
        self.state_lengths = ints([77 - 9 * i for i in range(sequences)])
        self.n = sequences

    def buffers(self, tokens):
        t = lambda *s, dtype=torch.bfloat16: torch.empty(s, dtype=dtype, device="cuda")  # noqa: E731
        lib, c = self.lib, self.cache
        ws = [lib.dav2cuda_linear_half_workspace_size(tokens, self.D, self.w.shape[0]),
              lib.dav2cuda_attention_cache_s8_workspace_size(self.n, tokens, c.page * c.table_d.shape[1], self.HQ, self.HKV, self.HD),
              lib.dav2cuda_cross_attention_16_workspace_size(self.n, tokens // self.n, 77, self.HQ, self.HKV, self.HD)]
        return dict(qkv=t(tokens, self.w.shape[0], dtype=torch.float32), q=t(tokens, self.HQ, self.HD), k=t(tokens, self.HKV, self.HD),
                    o=t(tokens, self.HQ, self.HD, dtype=torch.float32), x=t(tokens, self.HQ, self.HD),
                    ws=[t(max(16, n), dtype=torch.uint8) for n in ws])

    def step(self, x, positions, cached, lengths, begin, b):
        """x f32 [tokens, D], device arrays; queues the layer on the current stream."""
        lib, c, n = self.lib, self.cache, x.shape[0]
        hq, hkv, hd, st = self.HQ, self.HKV, self.HD, stream()
        row = self.w.shape[0]
        ok(lib, lib.dav2cuda_linear_half(ptr(b["qkv"]), ptr(x), ptr(self.w), ptr(self.b), n, self.D, row, 0, 2,
                                         ptr(b["ws"][0]), b["ws"][0].numel(), st))
        at = ptr(b["qkv"])
        ok(lib, lib.dav2cuda_qk_norm_rope(ptr(b["q"]), ptr(b["k"]), at, at + hq * hd * 4, ptr(self.qw), None, ptr(self.kw),
                                          None, ptr(self.f), ptr(positions), n, hq, hkv, hd, hd, 1, hq * hd, hkv * hd, row,
                                          row, 1, 1e-6, 0, 1.0, 0, 1, st))
        # K as bf16 from the norm; V as f32 from the linear: two appends would store each twice, so V goes to bf16 too
        b["v"] = b["qkv"][:, (hq + hkv) * hd:].to(torch.bfloat16)
        ok(lib, lib.dav2cuda_kv_cache_append_s8(ptr(c.k), ptr(c.ks), ptr(c.v), ptr(c.vs), ptr(b["k"]), ptr(b["v"]), ptr(c.table_d),
                                                ptr(cached), ptr(begin), self.n, n, hkv, hd, c.pages, c.page,
                                                c.table_d.shape[1], hkv * hd, hkv * hd, 1, st))
        ok(lib, lib.dav2cuda_attention_cache_s8(ptr(b["o"]), ptr(b["q"]), ptr(c.k), ptr(c.ks), ptr(c.v), ptr(c.vs), ptr(c.table_d),
                                                ptr(lengths), ptr(begin), self.n, n, c.page * c.table_d.shape[1], hq, hkv, hd,
                                                c.pages, c.page, c.table_d.shape[1], hq * hd, hq * hd, 0.125, 1, 1, 0,
                                                ptr(b["ws"][1]), b["ws"][1].numel(), st))
        s = self.states
        ok(lib, lib.dav2cuda_cross_attention_16(ptr(b["x"]), ptr(b["q"]), ptr(s), ptr(s) + hkv * hd * 2, ptr(self.state_lengths), self.n,
                                                n // self.n, 77, hq, hkv, hd, n // self.n * hq * hd, hq * hd, s.stride(0), s.stride(1),
                                                s.stride(0), s.stride(1), n // self.n * hq * hd, hq * hd, 0.125, 1, 1,
                                                ptr(b["ws"][2]), b["ws"][2].numel(), st))

    def check(self, x, positions, before, cached, lengths, begin, b):
        """Each stage against 64 bits on the values it was given."""
        c, n = self.cache, x.shape[0]
        hq, hkv, hd = self.HQ, self.HKV, self.HD
        want = x.double() @ self.w.double().T + self.b.double()
        # f16 operands: two roundings of 2^-11 on each of 256 products
        size = x.double().abs() @ self.w.double().abs().T + self.b.double().abs()
        assert ref.outside(b["qkv"], want, 2 ** -10 * size + 256 * 2.0 ** -23 * size) <= 1
        for at, h, w, got in ((0, hq, self.qw, b["q"]), (hq * hd, hkv, self.kw, b["k"])):
            y, size = ref.norm_rope(b["qkv"][:, at: at + h * hd].unflatten(1, (h, hd)), w, None, self.f, positions, hd, 1, 0, 1, 1e-6, 1.0)
            assert ref.outside(got, y, ref.norm_rope_bound(y, size, 1)) <= 1
        v = b["v"].unflatten(1, (hkv, hd))
        for (codes, scales), rows, now in ((before[:2], b["k"], (c.k, c.ks)), (before[2:], v, (c.v, c.vs))):
            a, s = ref.append(codes, scales, rows, c.table, cached, begin)
            assert torch.equal(now[0], a) and torch.equal(now[1], s)
        o, bound = ref.cache_attention(b["q"], c.k, c.ks, c.v, c.vs, c.table, lengths, begin, 0.125, True, 0)
        assert ref.outside(b["o"], o, bound) <= 1
        o, bound = ref.cross_attention(b["q"].unflatten(0, (self.n, -1)), self.states[:, :, 0], self.states[:, :, 1],
                                       self.state_lengths.tolist(), 0.125, 1, 1)
        assert ref.outside(b["x"].unflatten(0, (self.n, -1)), o, bound) <= 1

    def state(self):
        c = self.cache
        return [t.clone() for t in (c.k, c.ks, c.v, c.vs)]


def test_decoder_steps(cuda, dav2lib):
    """A prompt of 19 tokens for each of 3 streams, then single tokens, the latter as a captured graph that is replayed
    on another stream with new inputs and lengths in its device arrays."""
    n, g = 3, gen(12)
    dec = Decoder(dav2lib, n, 64)
    held = [0] * n

    def inputs(each):
        return (randn(g, n * each, dec.D), ints([[h + i] for h in held for i in range(each)]), ints(held),
                ints([h + each for h in held]), ints([each * i for i in range(n + 1)]))

    for each in (19, 1):
        x, pos, cached, lengths, begin = inputs(each)
        b, before = dec.buffers(n * each), dec.state()
        dec.step(x, pos, cached, lengths, begin, b)
        done(dav2lib)
        dec.check(x, pos, before, cached.tolist(), lengths.tolist(), begin.tolist(), b)
        held = [h + each for h in held]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    x, pos, cached, lengths, begin = inputs(1)
    graph, b = torch.cuda.CUDAGraph(), dec.buffers(n)
    with torch.cuda.stream(side):
        torch.cuda.synchronize()
        with torch.cuda.graph(graph, stream=side):
            dec.step(x, pos, cached, lengths, begin, b)
        for _ in range(15):
            new = inputs(1)
            for old, t in zip((x, pos, cached, lengths, begin), new):
                old.copy_(t)
            before = dec.state()
            graph.replay()
            side.synchronize()
            dec.check(x, pos, before, cached.tolist(), lengths.tolist(), begin.tolist(), b)
            held = [h + 1 for h in held]
    done(dav2lib)


def test_two_calls_at_once(cuda, dav2lib):
    """Two streams with a workspace each, and one workspace used by two calls in turn: the results of lone calls."""
    g = gen(13)
    c = Cache(g, [6000, 3500], 2, 64, 32)
    q = [randn(g, 2, 8, 64, dtype=torch.bfloat16) for _ in range(2)]
    lone, both, turn = ([torch.empty(2, 8, 64, dtype=torch.bfloat16, device="cuda") for _ in range(2)] for _ in range(3))
    for a in range(2):
        attend_cache(dav2lib, c, q[a], [6000, 3500], [0, 1, 2], True, lone[a], 0.125)
    args = (2, 2, 6000, 8, 2, 64)
    size = max(16, dav2lib.dav2cuda_attention_cache_s8_workspace_size(*args))
    ws = [torch.empty(size, dtype=torch.uint8, device="cuda") for _ in range(2)]
    lengths, begin = ints([6000, 3500]), ints([0, 1, 2])
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()

    def start(a, out, w, st):
        ok(dav2lib, dav2lib.dav2cuda_attention_cache_s8(
            ptr(out), ptr(q[a]), ptr(c.k), ptr(c.ks), ptr(c.v), ptr(c.vs), ptr(c.table_d), ptr(lengths), ptr(begin), *args,
            c.pages, c.page, c.table_d.shape[1], 512, 512, 0.125, 1, 1, 1, ptr(w), size, st))

    for _ in range(10):
        for a in range(2):
            start(a, both[a], ws[a], streams[a].cuda_stream)
    torch.cuda.synchronize()
    for _ in range(3):
        for a in range(2):
            start(a, turn[a], ws[0], stream())
    done(dav2lib)
    for a in range(2):
        assert torch.equal(lone[a], both[a]) and torch.equal(lone[a], turn[a])


def test_frequencies_to_rotation(cuda, dav2lib):
    """Frequencies of a stretched context, computed by the host entry, through the rotation."""
    import ctypes

    import numpy as np

    f, s = np.zeros(32, np.float32), ctypes.c_float()
    ok(dav2lib, dav2lib.dav2cuda_rope_frequencies(f.ctypes.data, ctypes.addressof(s), 64, 1, 10000.0, 3, 16.0, 4096.0))
    g = gen(14)
    x = randn(g, 9, 2, 64)
    pos = ints([[i * 8000] for i in range(9)])
    out, fd = torch.empty_like(x), torch.from_numpy(f).cuda()
    rope(dav2lib, x, None, out, None, [None] * 4, fd, pos, 64, 1, 0, 0, s.value)
    done(dav2lib)
    y, size = ref.norm_rope(x, None, None, fd, pos, 64, 1, 0, 0, 0, s.value)
    assert ref.outside(out, y, ref.norm_rope_bound(y, size, 0)) <= 1


