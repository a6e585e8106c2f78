"""Measured cases of the transformer operators: queries and keys with norm and rotary positions, the 8-bit key/value
cache with its attention, and cross attention.

``run`` computes an operator in elementary torch operations, or, where ``own`` is set, through the C ABI of
libdav2_b200.so (include/dav2cuda.h). ``exact`` gives the same results from the definitions in 64 bits.
"""
import math
import sys
from pathlib import Path

import torch

own = False

TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
PRECISION = {"f32": 0, "bf16": 1, "f16": 2}  # the C ABI's numbers of the types


# ----------------------------------------------------------------- the cases
def listed():
    return [
        # a decoder's step for three streams: latency
        dict(name="qk_step", op="rope", tokens=3, q_heads=32, k_heads=8, head_dim=128, rotary=128, axes=1, layout=0,
             norm=1, input="bf16", output="bf16", reach=8192),
        # the f32 qkv rows of 8 images at 518 x 518, normed per head, positions on the patch grid, f16 out for attention
        dict(name="qk_images", op="rope", tokens=10960, q_heads=16, k_heads=16, head_dim=64, rotary=64, axes=2,
             layout=0, norm=2, input="f32", output="f16", reach=37),
        # a long prompt far from the origin, half of the head rotated in interleaved pairs
        dict(name="qk_long", op="rope", tokens=32768, q_heads=32, k_heads=8, head_dim=128, rotary=64, axes=1,
             layout=1, norm=0, input="bf16", output="bf16", reach=1000000),
        # one new token for each of 64 streams into partly filled pages
        dict(name="append_step", op="append", sequences=64, tokens=64, heads=8, head_dim=128, page=16, type="bf16"),
        # prompts of different lengths
        dict(name="append_prompts", op="append", sequences=5, tokens=20011, heads=8, head_dim=128, page=64,
             type="f16"),
        # one stream with one image in its cache: latency
        dict(name="cache_one", op="cache", sequences=1, queries=1, length=1370, q_heads=16, kv_heads=16, head_dim=64,
             page=32, causal=True, type="f16"),
        # a serving batch, one token each, lengths up to 8192
        dict(name="cache_batch", op="cache", sequences=48, queries=48, length=8192, q_heads=32, kv_heads=8,
             head_dim=128, page=64, causal=True, type="bf16"),
        # one very long stream
        dict(name="cache_long", op="cache", sequences=1, queries=1, length=200003, q_heads=32, kv_heads=8,
             head_dim=128, page=64, causal=True, type="bf16"),
        # new chunks of tokens on top of what is cached
        dict(name="cache_extend", op="cache", sequences=6, queries=700, length=6000, q_heads=32, kv_heads=8,
             head_dim=128, page=64, causal=True, type="f16"),
        # one query token for each of 16 streams over an encoder's image tokens, padded to the longest
        dict(name="cross_step", op="cross", batch=16, queries=1, keys=1370, q_heads=16, kv_heads=16, head_dim=64,
             ragged=True, type="f16"),
        # every token of one view against another view, 8 pairs of images at 518 x 518
        dict(name="cross_views", op="cross", batch=8, queries=1370, keys=1370, q_heads=16, kv_heads=16, head_dim=64,
             ragged=False, type="bf16"),
        # 518 x 518 tokens against 1036 x 1036 tokens, shared key heads, padded batch
        dict(name="cross_large", op="cross", batch=4, queries=1370, keys=5477, q_heads=16, kv_heads=4, head_dim=128,
             ragged=True, type="bf16"),
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(("rope", "append", "cache", "cross"))
    if op == "rope":
        d = rng.choice((64, 80, 96, 128))
        q_heads = rng.choice((8, 12, 16, 24, 32))
        axes = rng.choice((1, 1, 2))
        rotary = rng.choice((d, d, d // 2)) // (2 * axes) * (2 * axes)
        given = rng.choice(("f32", "bf16", "f16"))
        return dict(op=op, tokens=_log(rng, 1, 32768 if given != "f32" else 12000), q_heads=q_heads,
                    k_heads=rng.choice((q_heads, q_heads // 4)), head_dim=d, rotary=rotary, axes=axes,
                    layout=rng.choice((0, 1, 2)), norm=rng.choice((0, 1, 2)), input=given,
                    output=given if given != "f32" else rng.choice(("f32", "bf16", "f16")),
                    reach=_log(rng, 40, 1000000))
    if op == "append":
        tokens = _log(rng, 1, 20000)
        return dict(op=op, sequences=min(tokens, _log(rng, 1, 64)), tokens=tokens, heads=rng.choice((4, 8, 16)) // (2 if tokens > 9000 else 1),
                    head_dim=rng.choice((64, 96, 128)), page=rng.choice((16, 32, 64, 128)),
                    type=rng.choice(("f32", "bf16", "f16")))
    if op == "cache":
        kv = rng.choice((4, 8))
        group = rng.choice((1, 2, 4, 6, 8))
        d = rng.choice((64, 96, 128))
        sequences = _log(rng, 1, 48)
        queries = sequences * (1 if rng.random() < 0.6 else _log(rng, 2, max(2, 500 // sequences)))
        most = min(200000, 390000 // sequences, 20000000 // (queries * kv * group) if queries > sequences else 200000)
        return dict(op=op, sequences=sequences, queries=queries, length=_log(rng, 5, most), q_heads=kv * group,
                    kv_heads=kv, head_dim=d, page=rng.choice((16, 32, 64, 128)), causal=rng.random() < 0.8,
                    type=rng.choice(("bf16", "f16")))
    kv = rng.choice((4, 8))
    group = rng.choice((1, 2, 4))
    batch = _log(rng, 1, 16)
    queries = 1 if rng.random() < 0.3 else _log(rng, 2, 1500)
    keys = _log(rng, 3, 5500)
    while batch * queries * keys * kv * group > 400000000:
        batch = max(1, batch // 2)
        keys = max(3, keys * 2 // 3)
    return dict(op=op, batch=batch, queries=queries, keys=keys, q_heads=kv * group, kv_heads=kv,
                head_dim=rng.choice((64, 80, 128)), ragged=rng.random() < 0.5, type=rng.choice(("bf16", "f16")))


def _lengths(c):
    """Tokens in the cache and new queries of each sequence, the same for every seed (ragged, the first the longest)."""
    n, most = c["sequences"], c["length"]
    lengths = [max(1, most - (most * 3 // 4) * ((i * 37) % 64) // 64) for i in range(n)]
    counts = _share(c["queries"], n)
    if c["causal"]:
        lengths = [max(a, b) for a, b in zip(lengths, counts)]
    return lengths, counts


def _share(total, parts):
    """`total` in `parts` uneven parts of at least one."""
    weights = [1 + (i * 29) % 7 for i in range(parts)]
    rest = total - parts
    got = [1 + rest * w // sum(weights) for w in weights]
    got[0] += total - sum(got)
    return got


def _cached(c):
    """Tokens that each sequence holds before an append: partly filled pages, some fresh ones."""
    return [(i * 11) % c["page"] for i in range(c["sequences"])]


def _key_lengths(c):
    if not c["ragged"]:
        return [c["keys"]] * c["batch"]
    return [max(1, c["keys"] - (c["keys"] // 2) * ((i * 5) % 8) // 8) for i in range(c["batch"])]


def work(case):
    c = case
    if c["op"] == "rope":
        n = c["tokens"] * (c["q_heads"] + c["k_heads"]) * c["head_dim"]
        size = TYPES[c["input"]].itemsize + TYPES[c["output"]].itemsize
        return {"bytes": n * size, "flops": n * (4 + (6 if c["norm"] else 0))}
    if c["op"] == "append":
        n = 2 * c["tokens"] * c["heads"] * c["head_dim"]
        return {"bytes": n * (TYPES[c["type"]].itemsize + 1), "flops": 4 * n}
    if c["op"] == "cache":
        lengths, counts = _lengths(c)
        row = c["head_dim"] * c["q_heads"]
        seen = sum(b * a - (b * (b - 1) // 2 if c["causal"] else 0) for a, b in zip(lengths, counts))
        return {"bytes": 2 * sum(lengths) * c["kv_heads"] * c["head_dim"] + 4 * c["queries"] * row, "flops": 4 * seen * row}
    lengths = _key_lengths(c)
    row = c["head_dim"] * c["q_heads"]
    return {"bytes": 4 * sum(lengths) * c["kv_heads"] * c["head_dim"] + 4 * c["batch"] * c["queries"] * row,
            "flops": 4 * c["queries"] * sum(lengths) * row}


# ------------------------------------------------------------------- inputs
def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _begins(counts):
    got = [0]
    for n in counts:
        got.append(got[-1] + n)
    return got


def prepare(case, seed):
    c = dict(case)
    g = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*shape, dtype=torch.float32):
        return torch.randn(shape, generator=g, device="cuda", dtype=torch.float32).to(dtype)

    s = {"case": c}
    if c["op"] == "rope":
        d, rotary, axes = c["head_dim"], c["rotary"], c["axes"]
        row = (c["q_heads"] + 2 * c["k_heads"]) * d
        s["qkv"] = normal(c["tokens"], row, dtype=TYPES[c["input"]])  # q | k | v of one linear layer
        for n in ("q", "k"):
            s[n + "_weight"] = 1 + 0.2 * normal(d)
            s[n + "_bias"] = 0.1 * normal(d)
        pairs = rotary // 2 // axes
        one = 10000.0 ** (-torch.arange(pairs, dtype=torch.float64, device="cuda") / pairs)
        s["frequencies"] = one.repeat(axes).to(torch.float32)
        s["positions"] = torch.randint(0, c["reach"], (c["tokens"], axes), generator=g, device="cuda", dtype=torch.int32)
        s["q_out"] = torch.empty((c["tokens"], c["q_heads"], d), dtype=TYPES[c["output"]], device="cuda")
        s["k_out"] = torch.empty((c["tokens"], c["k_heads"], d), dtype=TYPES[c["output"]], device="cuda")
    elif c["op"] == "append":
        h, d, page = c["heads"], c["head_dim"], c["page"]
        counts, held = _share(c["tokens"], c["sequences"]), _cached(c)
        need = [-(-(a + b) // page) for a, b in zip(held, counts)]
        s["table"] = _table(need, g)
        s["pages"] = pages = sum(need)
        for n in ("k", "v"):
            s[n] = normal(c["tokens"], h, d, dtype=TYPES[c["type"]])
            s[n + "_codes"] = torch.randint(-127, 128, (pages, h, page, d), generator=g, device="cuda", dtype=torch.int8)
            s[n + "_scales"] = (2.0 + normal(pages, h).abs()) / 127
            s[n + "_values"] = torch.empty((pages, h, page, d), dtype=TYPES[c["type"]], device="cuda")
        s["cached"], s["begin"] = _ints(held), _ints(_begins(counts))
    elif c["op"] == "cache":
        h, d, page = c["kv_heads"], c["head_dim"], c["page"]
        lengths, counts = _lengths(c)
        need = [-(-a // page) for a in lengths]
        s["table"] = _table(need, g)
        s["pages"] = pages = sum(need)
        s["longest"], s["most"] = max(lengths), max(counts)
        for n in ("k", "v"):
            s[n + "_codes"] = (normal(pages, h, page, d, dtype=torch.float16) * 40).clamp_(-127, 127).round_().to(torch.int8)
            s[n + "_scales"] = (3.0 + normal(pages, h).abs()) / 127
        s["q"] = normal(c["queries"], c["q_heads"], d, dtype=TYPES[c["type"]])
        s["lengths"], s["begin"] = _ints(lengths), _ints(_begins(counts))
        s["out"] = torch.empty_like(s["q"])
    else:
        d, t = c["head_dim"], TYPES[c["type"]]
        s["q"] = normal(c["batch"], c["queries"], c["q_heads"], d, dtype=t)
        kv = normal(c["batch"], c["keys"], 2, c["kv_heads"], d, dtype=t)  # k | v of one linear layer
        s["k"], s["v"] = kv[:, :, 0], kv[:, :, 1]
        s["key_lengths"] = _ints(_key_lengths(c))
        s["out"] = torch.empty_like(s["q"])
    return s


def _table(need, g):
    """A page table of shuffled pages; places past a sequence's pages hold -1."""
    order = torch.randperm(sum(need), generator=g, device="cuda").to(torch.int32)
    table = torch.full((len(need), max(need)), -1, dtype=torch.int32, device="cuda")
    row = torch.repeat_interleave(torch.arange(len(need)), torch.tensor(need)).cuda()
    first = torch.tensor(_begins(need)[:-1]).cuda()
    table[row, torch.arange(sum(need), device="cuda") - first[row]] = order
    return table


def run(state):
    return {"rope": _rope, "append": _append, "cache": _cache, "cross": _cross}[state["case"]["op"]](state)


# ----------------------------------------------------- the framework's calls
def _library():
    at = str(Path(__file__).resolve().parent.parent / "depth-anything-v2_b200")
    if at not in sys.path:
        sys.path.insert(0, at)
    import dav2_b200

    return dav2_b200


_lib = None


def _call(name, *args):
    global _lib
    if _lib is None:
        _lib = _library().load()
    rc = getattr(_lib, name)(*args, torch.cuda.current_stream().cuda_stream)
    if rc != 0:
        raise RuntimeError(name + ": " + _lib.dav2cuda_last_error().decode())


def _workspace(s, name, *args):
    """The workspace that a program keeps beside its plan."""
    global _lib
    if "workspace" not in s:
        if _lib is None:
            _lib = _library().load()
        s["workspace"] = torch.empty(max(1, getattr(_lib, name)(*args)), dtype=torch.uint8, device="cuda")
    return s["workspace"].data_ptr(), s["workspace"].numel()


# ------------------------------------------------------ norm and positions
def _rope(s):
    c = s["case"]
    d, hq, hk, row = c["head_dim"], c["q_heads"], c["k_heads"], s["qkv"].shape[1]
    if own:
        at, size = s["qkv"].data_ptr(), s["qkv"].element_size()
        _call("dav2cuda_qk_norm_rope", s["q_out"].data_ptr(), s["k_out"].data_ptr(), at, at + hq * d * size,
              s["q_weight"].data_ptr(), s["q_bias"].data_ptr(), s["k_weight"].data_ptr(), s["k_bias"].data_ptr(),
              s["frequencies"].data_ptr(), s["positions"].data_ptr(), c["tokens"], hq, hk, d, c["rotary"], c["axes"],
              hq * d, hk * d, row, row, c["norm"], 1e-6, c["layout"], 1.0, PRECISION[c["input"]],
              PRECISION[c["output"]])
        return s["q_out"], s["k_out"]
    x = s["qkv"][:, : (hq + hk) * d].float().unflatten(1, (hq + hk, d))
    if c["norm"]:
        if c["norm"] == 2:
            x = x - x.mean(-1, keepdim=True)
        x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + 1e-6)
        weight = torch.cat((s["q_weight"].expand(hq, d), s["k_weight"].expand(hk, d)))
        bias = torch.cat((s["q_bias"].expand(hq, d), s["k_bias"].expand(hk, d)))
        x = x * weight + bias
    pairs = c["rotary"] // 2
    axis = torch.arange(pairs, device="cuda") // (pairs // c["axes"])
    angle = s["positions"].double()[:, axis] * s["frequencies"].double()
    cos, sin = angle.cos().float()[:, None], angle.sin().float()[:, None]
    first, second = _pair_places(c, "cuda")
    u, v = x[..., first], x[..., second]
    y = x.clone()
    y[..., first] = u * cos - v * sin
    y[..., second] = v * cos + u * sin
    y = y.to(TYPES[c["output"]])
    return y[:, :hq].contiguous(), y[:, hq:].contiguous()


def _pair_places(c, device):
    """Where the first and the second value of each pair lie in the head."""
    i = torch.arange(c["rotary"] // 2, device=device)
    if c["layout"] == 1:
        return 2 * i, 2 * i + 1
    if c["layout"] == 0:
        return i, i + c["rotary"] // 2
    part = c["rotary"] // c["axes"]
    first = i // (part // 2) * part + i % (part // 2)
    return first, first + part // 2


# ------------------------------------------------------------------- append
def _append(s):
    c = s["case"]
    h, d, page = c["heads"], c["head_dim"], c["page"]
    if own:
        _call("dav2cuda_kv_cache_append_s8", s["k_codes"].data_ptr(), s["k_scales"].data_ptr(),
              s["v_codes"].data_ptr(), s["v_scales"].data_ptr(), s["k"].data_ptr(), s["v"].data_ptr(),
              s["table"].data_ptr(), s["cached"].data_ptr(), s["begin"].data_ptr(), c["sequences"], c["tokens"], h, d,
              s["pages"], page, s["table"].shape[1], h * d, h * d, PRECISION[c["type"]])
    else:
        token = torch.arange(c["tokens"], device="cuda", dtype=torch.int32)
        seq = torch.searchsorted(s["begin"][1:], token, right=True)
        at = s["cached"][seq] + token - s["begin"][seq]
        where, slot = s["table"][seq, (at // page).long()].long(), (at % page).long()
        last = (s["cached"] // page).long()
        held = torch.zeros(s["pages"], dtype=torch.int32, device="cuda")  # tokens of before in each page
        row = torch.arange(c["sequences"], device="cuda")
        held[s["table"][row, last.clamp(max=s["table"].shape[1] - 1)].long()] = s["cached"] % page
        for n in ("k", "v"):
            x, codes, scales = s[n].float(), s[n + "_codes"], s[n + "_scales"]
            limit = torch.full((), 127.0, device="cuda")  # a tensor: a number would be multiplied by its reciprocal
            most = torch.zeros_like(scales).scatter_reduce(0, where[:, None].expand(-1, h), x.abs().amax(-1), "amax")
            need = (most / limit).clamp(min=1e-8)
            grows = (held[:, None] == 0) | (need > scales)
            new = torch.where(grows, need, scales)
            ratio = torch.where(grows & (held[:, None] > 0), scales / new, torch.ones_like(new))
            kept = (codes.float() * ratio[..., None, None]).round().to(torch.int8)
            old = torch.arange(page, device="cuda") < held[:, None]
            codes.copy_(torch.where(old[:, None, :, None], kept, codes))
            scales.copy_(new)
            codes[where, :, slot] = (x / new[where][..., None]).clamp(-127, 127).round().to(torch.int8)
    for n in ("k", "v"):
        torch.mul(s[n + "_codes"], s[n + "_scales"][..., None, None], out=s[n + "_values"])
    return s["k_values"], s["v_values"], s["k_scales"], s["v_scales"]


# -------------------------------------------------------- attention, cached
def _cache(s):
    c = s["case"]
    hq, h, d, page = c["q_heads"], c["kv_heads"], c["head_dim"], c["page"]
    scale = 1 / math.sqrt(d)
    if own:
        space = _workspace(s, "dav2cuda_attention_cache_s8_workspace_size", c["sequences"], c["queries"], s["longest"],
                           hq, h, d)
        kind = PRECISION[c["type"]]
        _call("dav2cuda_attention_cache_s8", s["out"].data_ptr(), s["q"].data_ptr(), s["k_codes"].data_ptr(),
              s["k_scales"].data_ptr(), s["v_codes"].data_ptr(), s["v_scales"].data_ptr(), s["table"].data_ptr(),
              s["lengths"].data_ptr(), s["begin"].data_ptr(), c["sequences"], c["queries"], s["longest"], hq, h, d,
              s["pages"], page, s["table"].shape[1], hq * d, hq * d, scale, int(c["causal"]), kind, kind, *space)
        return s["out"]
    n, t = c["sequences"], s["table"].clamp(min=0).long()

    def dense(codes, scales):  # [sequences, heads, tokens, d]
        x = codes[t].float() * scales[t][..., None, None]
        return x.transpose(1, 2).flatten(2, 3)[:, :, : s["longest"]]

    k, v = dense(s["k_codes"], s["k_scales"]), dense(s["v_codes"], s["v_scales"])
    i = torch.arange(s["most"], device="cuda")
    counts = s["begin"].diff()
    rows = (s["begin"][:-1, None] + i).clamp(max=c["queries"] - 1).long()
    q = s["q"].float()[rows].unflatten(2, (h, hq // h)).permute(0, 2, 3, 1, 4)  # [n, h, group, most, d]
    scores = q.flatten(2, 3) @ k.transpose(-1, -2) * scale
    scores = scores.unflatten(2, (hq // h, s["most"]))
    reach = s["lengths"][:, None].expand(n, s["most"])
    if c["causal"]:
        reach = reach - counts[:, None] + i + 1
    seen = torch.arange(s["longest"], device="cuda") < reach[..., None]
    o = _softmax(scores, seen[:, None, None]).flatten(2, 3) @ v
    o = o.unflatten(2, (hq // h, s["most"])).permute(0, 3, 1, 2, 4).flatten(2, 3)
    return o[i < counts[:, None]].to(s["q"].dtype)


def _softmax(scores, seen):
    """Over the last axis, where `seen`; rows that see nothing are zero."""
    scores = scores.masked_fill(~seen, -math.inf)
    top = scores.amax(-1, keepdim=True)
    p = (scores - top.masked_fill(top == -math.inf, 0)).exp()
    return p / p.sum(-1, keepdim=True).clamp(min=1e-30)


# --------------------------------------------------------- attention, cross
def _cross(s):
    c = s["case"]
    hq, h, d, keys = c["q_heads"], c["kv_heads"], c["head_dim"], c["keys"]
    scale = 1 / math.sqrt(d)
    q, k, v = s["q"], s["k"], s["v"]
    if own:
        space = _workspace(s, "dav2cuda_cross_attention_16_workspace_size", c["batch"], c["queries"], keys, hq, h, d)
        kind = PRECISION[c["type"]]
        _call("dav2cuda_cross_attention_16", s["out"].data_ptr(), q.data_ptr(), k.data_ptr(), v.data_ptr(),
              s["key_lengths"].data_ptr(), c["batch"], c["queries"], keys, hq, h, d, q.stride(0), q.stride(1),
              k.stride(0), k.stride(1), v.stride(0), v.stride(1), s["out"].stride(0), s["out"].stride(1), scale, kind,
              kind, *space)
        return s["out"]
    q = q.float().unflatten(2, (h, hq // h)).permute(0, 2, 3, 1, 4).flatten(2, 3)  # [batch, h, group * queries, d]
    seen = torch.arange(keys, device="cuda") < s["key_lengths"][:, None, None, None]
    p = _softmax(q @ k.float().permute(0, 2, 3, 1) * scale, seen)
    o = p @ v.float().transpose(1, 2)
    return o.unflatten(2, (hq // h, c["queries"])).permute(0, 3, 1, 2, 4).flatten(2, 3).to(s["q"].dtype)


# ------------------------------------------------- the definitions in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    return {"rope": _exact_rope, "append": _exact_append, "cache": _exact_cache, "cross": _exact_cross}[case["op"]](s)


def _exact_rope(s):
    c = s["case"]
    d, hq = c["head_dim"], c["q_heads"]
    cycles = s["positions"].double()
    per = c["rotary"] // 2 // c["axes"]
    first, second = (p.tolist() for p in _pair_places(c, "cpu"))
    outs = []
    for name, begin, heads in (("q", 0, hq), ("k", hq * d, c["k_heads"])):
        x = s["qkv"][:, begin: begin + heads * d].double().view(-1, heads, d)
        if c["norm"] == 1:
            x = x / (x.pow(2).mean(-1, keepdim=True) + 1e-6).sqrt()
        elif c["norm"] == 2:
            x = (x - x.mean(-1, keepdim=True)) / (x.var(-1, unbiased=False, keepdim=True) + 1e-6).sqrt()
        if c["norm"]:
            x = x * s[name + "_weight"].double() + s[name + "_bias"].double()
        y = x.clone()
        for i in range(c["rotary"] // 2):
            turn = torch.polar(torch.ones((), dtype=torch.float64, device="cuda"),
                               cycles[:, i // per] * s["frequencies"][i].double())
            z = torch.complex(x[..., first[i]], x[..., second[i]]) * turn[:, None]
            y[..., first[i]], y[..., second[i]] = z.real, z.imag
        outs.append(y)
    return tuple(outs)


def _exact_append(s):
    """Scales and quotients are defined in 32 bits, as the codes of the int8 linears are: a quotient or product is the
    exact one rounded once."""
    c = s["case"]
    page, once = c["page"], lambda x: x.float().double()
    table, held, begin = s["table"].tolist(), s["cached"].tolist(), s["begin"].tolist()
    out = []
    for n in ("k", "v"):
        codes, scales, x = s[n + "_codes"].double(), s[n + "_scales"].double(), s[n].double()
        for i in range(c["sequences"]):
            at, row = held[i], begin[i]
            while row < begin[i + 1]:
                p, slot = table[i][at // page], at % page
                count = min(page - slot, begin[i + 1] - row)
                new = x[row: row + count].transpose(0, 1)  # [heads, count, d]
                need = once(new.abs().amax((1, 2)) / 127).clamp(min=float(torch.tensor(1e-8)))
                if slot:
                    grown = need > scales[p]
                    need = torch.where(grown, need, scales[p])
                    ratio = once(scales[p] / need)[:, None, None]
                    codes[p, :, :slot] = torch.where(grown[:, None, None], once(codes[p, :, :slot] * ratio).round(),
                                                     codes[p, :, :slot])
                scales[p] = need
                codes[p, :, slot: slot + count] = once(new / need[:, None, None]).clamp(-127, 127).round()
                at, row = at + count, row + count
        out.append((codes * scales[..., None, None], scales))
    return out[0][0], out[1][0], out[0][1], out[1][1]


def _attend(q, k, v, scale, reach):
    """q [heads, n, d] over k, v [heads, tokens, d] in 64 bits; row r sees the first reach[r] tokens."""
    score = torch.einsum("hnd,htd->hnt", q, k) * scale
    score[:, torch.arange(k.shape[1], device="cuda")[None] >= reach[:, None]] = -math.inf
    o = torch.einsum("hnt,htd->hnd", torch.softmax(score, -1), v)
    o[:, reach <= 0] = 0
    return o


def _exact_cache(s):
    c = s["case"]
    group, page = c["q_heads"] // c["kv_heads"], c["page"]
    lengths, begin, rows = s["lengths"].tolist(), s["begin"].tolist(), []
    for i in range(c["sequences"]):
        n, length = begin[i + 1] - begin[i], lengths[i]
        pages = s["table"][i, : -(-length // page)].long()
        k, v = ((s[x + "_codes"][pages].double() * s[x + "_scales"][pages].double()[..., None, None])
                .transpose(0, 1).flatten(1, 2)[:, :length] for x in ("k", "v"))
        reach = torch.full((n,), length, device="cuda")
        if c["causal"]:
            reach = reach - n + 1 + torch.arange(n, device="cuda")
        q = s["q"][begin[i]: begin[i + 1]].double().transpose(0, 1)
        o = [_attend(q[a * group: (a + 1) * group], k[a: a + 1].expand(group, -1, -1),
                     v[a: a + 1].expand(group, -1, -1), 1 / math.sqrt(c["head_dim"]), reach) for a in range(c["kv_heads"])]
        rows.append(torch.cat(o).transpose(0, 1))
    return torch.cat(rows)


def _exact_cross(s):
    c = s["case"]
    group = c["q_heads"] // c["kv_heads"]
    out = torch.empty(s["q"].shape, dtype=torch.float64, device="cuda")
    for i, length in enumerate(_key_lengths(c)):
        for a in range(c["kv_heads"]):
            heads = slice(a * group, (a + 1) * group)
            k, v = (s[x][i, :length, a].double()[None].expand(group, -1, -1) for x in ("k", "v"))
            reach = torch.full((c["queries"],), length, device="cuda")
            out[i, :, heads] = _attend(s["q"][i, :, heads].double().transpose(0, 1), k, v,
                                       1 / math.sqrt(c["head_dim"]), reach).transpose(0, 1)
    return out
