"""Plain 64-bit references of the transformer operators, on the CPU or the GPU (torch, no library attention), and the
bounds that the kernels' roundings allow. U[t] is half a step of type t: the largest relative error of one rounding."""
import math

import torch

TYPES = {0: torch.float32, 1: torch.bfloat16, 2: torch.float16}
U = {p: torch.finfo(t).eps / 2 for p, t in TYPES.items()}


def pair_places(rotary, axes, layout):
    i = torch.arange(rotary // 2)
    if layout == 1:
        return 2 * i, 2 * i + 1
    if layout == 0:
        return i, i + rotary // 2
    half = rotary // axes // 2
    first = i // half * 2 * half + i % half
    return first, first + half


def norm_rope(x, weight, bias, frequencies, positions, rotary, axes, layout, norm, eps, rotary_scale):
    """x [tokens, heads, d] (any type) -> (y in 64 bits, scale of the values that the roundings are relative to)."""
    x = x.double()
    size = x.abs().amax(-1, keepdim=True)
    if norm:
        if norm == 2:
            x = x - x.mean(-1, keepdim=True)
        r = 1 / (x.square().mean(-1, keepdim=True) + eps).sqrt()
        x, size = x * r, size * r
        if weight is not None:
            x, size = x * weight.double(), size * weight.double().abs().max()
        if bias is not None:
            x, size = x + bias.double(), size + bias.double().abs().max()
    y = x.clone()
    if rotary:
        per = rotary // 2 // axes
        axis = (torch.arange(rotary // 2) // per).to(x.device)
        a = (positions.double()[:, axis] * frequencies.double())[:, None]
        first, second = (p.to(x.device) for p in pair_places(rotary, axes, layout))
        u, v = x[..., first], x[..., second]
        y[..., first] = rotary_scale * (u * a.cos() - v * a.sin())
        y[..., second] = rotary_scale * (v * a.cos() + u * a.sin())
    return y, size * max(1.0, abs(rotary_scale))


def norm_rope_bound(y, size, precision):
    """Half a step of the output, and f32 arithmetic relative to the row's largest value: the sum of up to 256 squares
    in a lane's chain of 16 (8 for unaligned heads) and 5 lane steps is within 22 roundings, half of that in the root;
    mean, product, weight and bias 4 + 22 / 2 more; sine and cosine 2 units each and the angle's rounding pi / 2, on
    two terms: 11 + 15 + 8 < 40."""
    return U[precision] * y.abs() + 40 * 2.0 ** -24 * size


def append(codes, scales, x, table, cached, begin):
    """codes [pages, heads, P, d], scales [pages, heads], x [tokens, heads, d]: new copies. Scale, quotient and ratio
    are defined in 32 bits: exact quotients rounded once (a 53-bit quotient of 24-bit numbers rounds like the exact one)."""
    codes, scales, page = codes.clone(), scales.clone(), codes.shape[2]
    f32 = lambda v: v.float().double()  # noqa: E731
    for s in range(len(cached)):
        at, row = cached[s], begin[s]
        while row < begin[s + 1]:
            p, slot = table[s][at // page], at % page
            n = min(page - slot, begin[s + 1] - row)
            new = x[row: row + n].double().transpose(0, 1).nan_to_num(nan=0.0, posinf=math.inf, neginf=-math.inf)
            most = torch.where(new.isinf(), 0.0, new.abs()).amax((1, 2))
            need = f32(most / 127).clamp(min=float(torch.tensor(1e-8)))
            old = scales[p].double()
            if slot:
                grows = need > old
                need = torch.where(grows, need, old)
                ratio = f32(old / need)[:, None, None]
                kept = f32(codes[p, :, :slot].double() * ratio).round()
                codes[p, :, :slot] = torch.where(grows[:, None, None], kept, codes[p, :, :slot].double()).to(torch.int8)
            scales[p] = need.float()
            codes[p, :, slot: slot + n] = f32(new / need[:, None, None]).clamp(-127, 127).round().to(torch.int8)
            at, row = at + n, row + n
    return codes, scales


def attend(q, k, v, scale, reach, p_unit, out_precision):
    """q [n, heads, d], k, v [tokens, heads, d] in 64 bits (heads alike), reach [n]: (o [n, heads, d], bound).

    Bound: p is rounded once (p_unit) and, held times 2^7 in f16, to no finer than 2^-32; a score is off by at most the
    f32 sum's d roundings of sum |q||k|, which changes p by that relative amount, above and below the bar; an
    exponential is off by 2^-22 (ex2.approx) or 2.7e-6 < 2^-18.4 (the polynomial), and the maximum's and the merges'
    factors by a few 2^-22: together below 2^-18; the result is rounded once."""
    n, d = q.shape[0], q.shape[2]
    score = torch.einsum("nhd,thd->hnt", q, k) * scale
    size = torch.einsum("nhd,thd->hnt", q.abs(), k.abs()).amax() * abs(scale) if k.shape[0] else torch.zeros(())
    seen = torch.arange(k.shape[0], device=q.device) < reach[:, None]
    score = score.masked_fill(~seen, -math.inf)
    p = torch.softmax(score, -1).nan_to_num(nan=0.0)
    o = torch.einsum("hnt,thd->nhd", p, v)
    spread = torch.einsum("hnt,thd->nhd", p, v.abs())
    least = 2.0 ** -32 * k.shape[0] * (v.abs().amax() if k.shape[0] else 0)
    bound = (p_unit + 2 * (d + 8) * 2.0 ** -23 * float(size) + 2.0 ** -18) * spread + U[out_precision] * o.abs() + least
    return o, bound


def dense(codes, scales, pages, length, group):
    """The cache's values of one sequence, [length, heads * group, d] in 64 bits."""
    x = codes[pages].double() * scales[pages].double()[..., None, None]
    return x.transpose(0, 1).flatten(1, 2)[:, :length].transpose(0, 1).repeat_interleave(group, 1)


def cache_attention(q, kc, ks, vc, vs, table, lengths, begin, scale, causal, out_precision):
    """q [queries, heads, d]: (o, bound) for the rows of the sequences, zeros elsewhere."""
    group, page = q.shape[1] // kc.shape[1], kc.shape[2]
    o, bound = torch.zeros(q.shape, dtype=torch.float64, device=q.device), torch.zeros(q.shape, dtype=torch.float64, device=q.device)
    for s in range(len(lengths)):
        n, length = begin[s + 1] - begin[s], lengths[s]
        if not n:
            continue
        pages = torch.tensor(table[s][: -(-length // page)], dtype=torch.long, device=q.device)
        reach = torch.full((n,), length, device=q.device)
        if causal:
            reach = reach - n + 1 + torch.arange(n, device=q.device)
        k, v = dense(kc, ks, pages, length, group), dense(vc, vs, pages, length, group)
        rows = slice(begin[s], begin[s + 1])
        o[rows], bound[rows] = attend(q[rows].double(), k, v, scale, reach, U[2], out_precision)
    return o, bound


def cross_attention(q, k, v, lengths, scale, precision, out_precision):
    """q [batch, queries, heads, d], k, v [batch, keys, kv_heads, d]."""
    group = q.shape[2] // k.shape[2]
    o, bound = [], []
    for b in range(q.shape[0]):
        n = lengths[b]
        kk, vv = (x[b, :n].double().repeat_interleave(group, 1) for x in (k, v))
        reach = torch.full((q.shape[1],), n, device=q.device)
        a, c = attend(q[b].double(), kk, vv, scale, reach, U[precision], out_precision)
        o.append(a), bound.append(c)
    return torch.stack(o), torch.stack(bound)


def outside(got, want, bound):
    """The largest error in units of its bound (NaN counts as infinite)."""
    off = (got.double() - want).abs() / bound.clamp(min=1e-300)
    off = torch.where((got.double() == want), torch.zeros_like(off), off)
    return float(off.nan_to_num(nan=math.inf).max()) if off.numel() else 0.0
