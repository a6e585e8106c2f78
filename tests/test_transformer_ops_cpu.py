"""The transformer operators without a GPU: frequencies (host arithmetic), and the refusals, which answer before any
launch (null or host pointers only: nothing can be touched)."""
import ctypes
import math

import numpy as np
import pytest
import torch

import transformer_ref as ref


def frequencies(lib, rotary, axes, base, scaling, factor=1.0, trained=1.0):
    f, s = np.zeros(max(1, rotary // 2), np.float32), ctypes.c_float()
    rc = lib.dav2cuda_rope_frequencies(f.ctypes.data, ctypes.addressof(s), rotary, axes, base, scaling, factor, trained)
    return rc, f, s.value


@pytest.mark.parametrize("rotary,axes", [(64, 1), (128, 1), (64, 2), (2, 1), (96, 3)])
def test_frequencies(dav2lib, rotary, axes):
    n = rotary // 2 // axes
    plain = 10000.0 ** (-np.arange(n) / n)
    rc, f, s = frequencies(dav2lib, rotary, axes, 10000.0, 0)
    assert rc == 0 and s == 1.0
    # one rounding to f32, and pow's last bits
    assert np.abs(f.reshape(axes, n) / plain - 1).max() < 2 ** -23
    rc, f, s = frequencies(dav2lib, rotary, axes, 10000.0, 1, 4.0)
    assert rc == 0 and s == 1.0 and np.abs(f.reshape(axes, n) / (plain / 4) - 1).max() < 2 ** -23
    rc, f, s = frequencies(dav2lib, rotary, axes, 10000.0, 2, 4.0)
    assert rc == 0 and f[0] == 1.0
    if n > 1:
        assert abs(f[n - 1] / (plain[-1] / 4) - 1) < 2 ** -23 and np.all(np.diff(f[:n]) < 0)
    rc, f, s = frequencies(dav2lib, rotary, axes, 10000.0, 3, 8.0, 4096.0)
    turns = 4096 * plain / (2 * math.pi)
    keep = np.clip((turns - 1) / 31, 0, 1)
    assert rc == 0 and abs(s - (0.1 * math.log(8) + 1)) < 1e-6
    assert np.abs(f.reshape(axes, n) / (plain * keep + plain / 8 * (1 - keep)) - 1).max() < 2 ** -23


def test_frequencies_refusals(dav2lib):
    for args in [(63, 1, 1e4, 0), (64, 3, 1e4, 0), (0, 1, 1e4, 0), (64, 0, 1e4, 0), (64, 1, 1.0, 0), (64, 1, 1e4, 4),
                 (64, 1, math.nan, 0), (64, 1, 1e4, 1, 0.5), (64, 1, 1e4, 2, math.inf), (64, 1, 1e4, 3, 2.0, 0.0),
                 (512, 1, 1e4, 0)]:
        assert frequencies(dav2lib, *args)[0] == 1, args
    assert dav2lib.dav2cuda_rope_frequencies(None, None, 64, 1, 1e4, 0, 1.0, 1.0) == 1


A = 1 << 20  # an aligned address that nothing reads


def rope_args(**change):
    a = dict(q_out=A, k_out=A, q=A, k=A, qw=None, qb=None, kw=None, kb=None, f=A, pos=A, tokens=2, hq=4, hk=2, d=64,
             rotary=64, axes=1, qos=256, kos=128, qs=256, ks=128, norm=0, eps=1e-6, layout=0, scale=1.0, pin=1, pout=1)
    a.update(change)
    return list(a.values()) + [None]


@pytest.mark.parametrize("change,words", [
    (dict(d=63), b"head_dim"), (dict(d=0), b"head_dim"), (dict(d=258, rotary=64), b"head_dim"),
    (dict(rotary=66), b"rotary_dim"), (dict(rotary=63), b"rotary_dim"), (dict(axes=0), b"rotary_dim"),
    (dict(axes=3), b"rotary_dim"), (dict(norm=3), b"unknown norm"), (dict(layout=3), b"unknown norm"),
    (dict(norm=1, eps=-1.0), b"epsilon"), (dict(norm=1, eps=math.nan), b"epsilon"), (dict(scale=math.inf), b"scale"),
    (dict(pin=1, pout=2), b"type"), (dict(pin=1, pout=0), b"type"), (dict(pin=3, pout=3), b"type"),
    (dict(hq=0, hk=0), b"heads"), (dict(hq=65000, hk=65000), b"heads"), (dict(qs=255), b"stride"),
    (dict(kos=100), b"stride"), (dict(q=None), b"null"), (dict(k_out=None), b"null"), (dict(f=None), b"null"),
    (dict(axes=2, pos=None), b"positions")])
def test_qk_norm_rope_refusals(dav2lib, change, words):
    assert dav2lib.dav2cuda_qk_norm_rope(*rope_args(**change)) == 1
    assert words in dav2lib.dav2cuda_last_error()


def append_args(**change):
    a = dict(kc=A, ks=A, vc=A, vs=A, k=A, v=A, table=A, cached=A, begin=A, sequences=2, tokens=3, heads=2, d=64,
             pages=8, page=16, stride=4, k_stride=128, v_stride=128, precision=1)
    a.update(change)
    return list(a.values()) + [None]


@pytest.mark.parametrize("change,words", [
    (dict(precision=3), b"precision"), (dict(d=72), b"head_dim"), (dict(d=144), b"head_dim"), (dict(d=0), b"head_dim"),
    (dict(page=8), b"page_tokens"), (dict(page=48), b"page_tokens"), (dict(page=256), b"page_tokens"),
    (dict(heads=0), b"invalid"), (dict(pages=0), b"invalid"), (dict(stride=0), b"invalid"),
    (dict(tokens=1 << 31), b"too many"), (dict(sequences=1 << 30), b"too many"), (dict(k_stride=127), b"stride"),
    (dict(v_stride=64), b"stride"), (dict(kc=None), b"null"), (dict(vs=None), b"null"), (dict(begin=None), b"null"),
    (dict(k=A + 8), b"aligned"), (dict(vc=A + 4), b"aligned"), (dict(k_stride=130), b"aligned")])
def test_append_refusals(dav2lib, change, words):
    assert dav2lib.dav2cuda_kv_cache_append_s8(*append_args(**change)) == 1
    assert words in dav2lib.dav2cuda_last_error()


def cache_args(**change):
    a = dict(out=A, q=A, kc=A, ks=A, vc=A, vs=A, table=A, lengths=A, begin=A, sequences=2, queries=2, longest=64, hq=8,
             hkv=2, d=64, pages=8, page=16, stride=4, q_stride=512, out_stride=512, scale=0.125, causal=1, precision=1,
             out_precision=1, workspace=A, bytes=1 << 30)
    a.update(change)
    return list(a.values()) + [None]


@pytest.mark.parametrize("change,words", [
    (dict(precision=0), b"bf16 or f16"), (dict(precision=3), b"bf16 or f16"), (dict(out_precision=2), b"output"),
    (dict(hq=9), b"multiple"), (dict(hkv=0), b"multiple"), (dict(d=40), b"head_dim"), (dict(d=256), b"head_dim"),
    (dict(page=24), b"page_tokens"), (dict(longest=65), b"page table"), (dict(pages=0), b"page table"),
    (dict(scale=math.nan), b"scale"), (dict(queries=1 << 30), b"too many"), (dict(q_stride=504), b"stride"),
    (dict(out_stride=64), b"stride"), (dict(q=None), b"null"), (dict(table=None), b"null"), (dict(q=A + 2), b"aligned"),
    (dict(out_stride=516), b"aligned"),
    (dict(longest=1 << 16, stride=1 << 12, bytes=1000), b"workspace"),
    (dict(longest=1 << 16, stride=1 << 12, workspace=None), b"workspace")])
def test_cache_attention_refusals(dav2lib, change, words):
    assert dav2lib.dav2cuda_attention_cache_s8(*cache_args(**change)) == 1
    assert words in dav2lib.dav2cuda_last_error()


def cross_args(**change):
    a = dict(out=A, q=A, k=A, v=A, lengths=None, batch=2, queries=3, keys=1 << 14, hq=8, hkv=2, d=64, qb=1536, qs=512,
             kb=1 << 22, ks=256, vb=1 << 22, vs=256, ob=1536, os=512, scale=0.125, precision=2, out_precision=2,
             workspace=A, bytes=1 << 30)
    a.update(change)
    return list(a.values()) + [None]


@pytest.mark.parametrize("change,words", [
    (dict(precision=0), b"bf16 or f16"), (dict(out_precision=1), b"output"), (dict(hq=7), b"multiple"),
    (dict(hkv=0), b"multiple"), (dict(d=60), b"head_dim"), (dict(d=136), b"head_dim"), (dict(scale=math.inf), b"scale"),
    (dict(queries=1 << 30), b"too many"), (dict(keys=1 << 31), b"too many"), (dict(qs=511), b"stride"),
    (dict(os=256), b"stride"), (dict(vs=64), b"stride"), (dict(ob=1000), b"overlap"), (dict(q=None), b"null"),
    (dict(v=None), b"null"), (dict(k=A + 8), b"aligned"), (dict(ks=260), b"aligned"), (dict(vb=4), b"aligned"),
    (dict(bytes=100), b"workspace"), (dict(workspace=None), b"workspace")])
def test_cross_attention_refusals(dav2lib, change, words):
    assert dav2lib.dav2cuda_cross_attention_16(*cross_args(**change)) == 1
    assert words in dav2lib.dav2cuda_last_error()


def test_nothing_to_do(dav2lib):
    """Calls without tokens succeed and launch nothing."""
    before = dav2lib.dav2cuda_launch_count(0)
    assert dav2lib.dav2cuda_qk_norm_rope(*rope_args(tokens=0, q=None, k=None, q_out=None, k_out=None)) == 0
    assert dav2lib.dav2cuda_kv_cache_append_s8(*append_args(tokens=0, k=None, v=None)) == 0
    assert dav2lib.dav2cuda_kv_cache_append_s8(*append_args(sequences=0)) == 0
    assert dav2lib.dav2cuda_attention_cache_s8(*cache_args(queries=0, q=None)) == 0
    assert dav2lib.dav2cuda_cross_attention_16(*cross_args(queries=0, q=None)) == 0
    assert dav2lib.dav2cuda_cross_attention_16(*cross_args(batch=0, q=None)) == 0
    assert dav2lib.dav2cuda_launch_count(0) == before


def test_workspace_sizes(dav2lib):
    f = dav2lib.dav2cuda_attention_cache_s8_workspace_size
    assert f(1, 1, 100, 32, 8, 128) == 0  # too short to be split
    assert f(1, 1, 200000, 32, 8, 128) >= 2 * 32 * (128 * 4 + 8)
    assert f(0, 1, 100, 32, 8, 128) == 0 and f(1, 1, 100, 32, 0, 128) == 0 and f(1, 1, 100, 30, 8, 128) == 0
    g = dav2lib.dav2cuda_cross_attention_16_workspace_size
    assert g(16, 1370, 1370, 16, 16, 64) == 0 and g(1, 1, 20000, 8, 8, 64) > 0


def test_reference_append_matches_the_int8_rows_rule():
    """A fresh page of one head holds the codes and scale of the oracle's row quantizer over the same values."""
    import oracle

    x = torch.from_numpy(np.random.default_rng(0).standard_normal((16, 1, 32)).astype(np.float32))
    codes, scales = ref.append(torch.zeros(1, 1, 16, 32, dtype=torch.int8), torch.zeros(1, 1), x, [[0]], [0], [0, 16])
    packed, scale = oracle.quantize_rows_s8(x.numpy().reshape(1, -1), 1, 512)
    assert np.array_equal(codes.numpy().reshape(-1), np.asarray(packed).view(np.int8).reshape(-1))
    assert scales[0, 0] == np.asarray(scale).reshape(-1)[0]


@pytest.mark.parametrize("change", [dict(ob=512, os=1016), dict(ob=504, os=4096), dict(ob=1528, os=512),
                                    dict(batch=3, ob=512, os=1528)])
def test_cross_attention_outputs_that_overlap(dav2lib, change):
    """Rows of 512 values: neither a batch after the other nor the batches of a token side by side."""
    assert dav2lib.dav2cuda_cross_attention_16(*cross_args(**change)) == 1
    assert b"overlap" in dav2lib.dav2cuda_last_error()


@pytest.mark.parametrize("grow", [1.0, 1.1])
def test_reference_append_token_by_token(grow):
    """A page filled by several calls: its scale is that of one call, its codes need not be. A value is off by half a
    step of the scale that it was stored with and of each larger one since (and f32's roundings: a code times the
    ratio, 127 at most, and the ratio itself, 2^-23 * 127 of a step each time)."""
    g = torch.Generator().manual_seed(0)
    x = torch.randn(64, 1, 64, generator=g) * grow ** torch.arange(64.0)[:, None, None]
    codes, scales = torch.zeros(1, 1, 64, 64, dtype=torch.int8), torch.zeros(1, 1)
    off = torch.zeros(64, dtype=torch.float64)
    growths = 0
    for t in range(64):
        before = float(scales)
        codes, scales = ref.append(codes, scales, x[t: t + 1], [[0]], [t], [0, 1])
        now = float(scales)
        step = 0.5 + 127 * 2.0 ** -23
        off[t] = now * step
        if t and now > before:
            off[:t] += now * step
            growths += 1
    error = (codes[0, 0].double() * float(scales) - x[:, 0].double()).abs().amax(-1)
    assert growths >= 2 and (error <= off).all()
    once, scale = ref.append(torch.zeros_like(codes), torch.zeros(1, 1), x, [[0]], [0], [0, 64])
    assert torch.equal(scale, scales) and not torch.equal(once, codes)
    assert ((once[0, 0].double() * float(scale) - x[:, 0].double()).abs() <= float(scale) * step).all()


def test_workspace_of_the_longest_keys(dav2lib):
    """Keys whose pass would outlast the kernels' bounded waits are split, also where there are rows for all SMs: no
    part is longer than 2^26 keys."""
    g, f = dav2lib.dav2cuda_cross_attention_16_workspace_size, dav2lib.dav2cuda_attention_cache_s8_workspace_size
    rows = 148 * 256 * 4
    for keys in (1 << 20, 1 << 26):
        assert g(1, rows, keys, 1, 1, 64) == 0 and f(1, rows, keys, 1, 1, 128) == 0
    for keys in ((1 << 26) + 1, 190_000_000, 0x7FFFFF00):
        parts = -(-keys // (1 << 26))
        assert g(1, rows, keys, 1, 1, 64) >= rows * parts * (64 * 4 + 8)
        assert f(1, rows, keys, 1, 1, 128) >= rows * parts * (128 * 4 + 8)
