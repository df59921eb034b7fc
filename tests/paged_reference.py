"""Plain 64-bit forms of the page pool operators, and pools to run them on."""
from __future__ import annotations

import math

import torch


def make_pool(cq, dev, fmt, pages, hkv, d, page, seed, dtype=torch.bfloat16, scale=1.0):
    """A pool with a quantized row in every place (through the dense append), as (k_side, v_side)."""
    g = torch.Generator().manual_seed(seed)
    sides = []
    for value in (False, True):
        s = cq.CacheSide.empty(fmt, value, pages, hkv, d, page, dev)
        x = (torch.randn(pages, hkv, page, d, generator=g) * scale).to(dtype)
        cq.quant_append(s, x.to(dev), 0)
        sides.append(s)
    return sides


def make_table(kv, page, pages, dev, seed, spare=1):
    """Shuffled page ids for sequences of kv[b] tokens; entries past a sequence's pages are -1."""
    need = [-(-n // page) for n in kv]
    order = torch.randperm(pages, generator=torch.Generator().manual_seed(seed)).tolist()
    t = torch.full((len(kv), max(max(need), 1) + spare), -1, dtype=torch.int32)
    at = 0
    for b, n in enumerate(need):
        t[b, :n] = torch.tensor(order[at:at + n], dtype=torch.int32)
        at += n
    assert at <= pages
    return t.to(dev)


def prefix(lens, dev, first=0):
    c = [first]
    for n in lens:
        c.append(c[-1] + n)
    return torch.tensor(c, dtype=torch.int32, device=dev)


def ints(v, dev):
    return torch.tensor(v, dtype=torch.int32, device=dev)


def page_rows(values, table, b, n):
    """values (pages, heads, page, d) -> the first n positions (n, heads, d) of sequence b and the mask
    of those that lie in a page of the pool."""
    pages, heads, page, d = values.shape
    p = torch.arange(n)
    ids = table[b].long().cpu()[p // page]
    ok = (ids >= 0) & (ids < pages)
    return values[ids.clamp(0, pages - 1), :, p % page], ok


def attention64(q, kvals, vvals, table, cu, kv, scale, wl=-1, wr=0, softcap=0.0, alibi=None,
                max_q=None):
    """q (total, hq, d); kvals / vvals (pages, hkv, page, d), all on the CPU. Returns the f64 output,
    the weighted mean of |v| (what a relative error of the weights scales with), and the rows that a
    call writes."""
    total, hq, d = q.shape
    hkv = kvals.shape[1]
    out = torch.zeros(total, hq, d, dtype=torch.float64)
    mag, wrote = torch.zeros_like(out), torch.zeros(total, dtype=torch.bool)
    cu = cu.tolist()
    for b, lk in enumerate(kv):
        first, lq = cu[b], cu[b + 1] - cu[b]
        for i in range(min(lq, max_q) if max_q is not None else lq):
            wrote[first + i] = True
            pos = i + lk - lq
            lo = max(pos - wl, 0) if wl >= 0 else 0
            hi = min(pos + wr + 1, lk) if wr >= 0 else lk
            if hi <= lo:
                continue
            k, ok = page_rows(kvals, table, b, hi)
            v, _ = page_rows(vvals, table, b, hi)
            ok[:lo] = False
            if not ok.any():
                continue
            key = torch.arange(hi)[ok]
            k, v = k[ok].double(), v[ok].double()
            for h in range(hq):
                x = k[:, h * hkv // hq] @ q[first + i, h].double() * scale
                if softcap > 0:
                    x = softcap * torch.tanh(x / softcap)
                if alibi is not None:
                    a = alibi[b, h] if alibi.dim() == 2 else alibi[h]
                    x = x - a.double() * (pos - key).abs().double()
                w = torch.softmax(x, 0)
                out[first + i, h] = w @ v[:, h * hkv // hq]
                mag[first + i, h] = w @ v[:, h * hkv // hq].abs()
    return out, mag, wrote


def score_spread(q, kvals, scale):
    """Largest sum of |q_i k_i| scale of a call's queries and keys (.., .., .., d): the size of a score's
    terms."""
    return (q.double().abs().flatten(0, 1) @ kvals.double().abs().amax((0, 1, 2))).max().item() * scale


def assert_attention(got, want, mag, dtype, fmt4=False, chunk=False, spread=0.0):
    """|got - want| within the roundings of the call; mag the weighted mean of |v|.

    The output to its dtype: half a step, 2^-8 (bf16) or 2^-11 (f16) of a value that the other errors
    have moved. Decode kernel: the weights as bf16 hi + lo parts (2^-16), or one bf16 part for bf16 calls
    over 4-bit pools (2^-8). Chunk kernel, in the dtype's half step h: the weights (h), the values (h),
    the keys and the scaled queries (h each, of the terms of a score: these move a weight, and the sum of
    weights, by 2 x 2 h times at most the sum of |q_i k_i| scale, `spread`, if every term erred its worst
    way; independent errors stay below a quarter of that, and the largest sum over all keys and queries is
    taken). f32 sums, exponentials and scores below 32: 2^-13."""
    half = torch.finfo(dtype).eps / 2
    w = 2.0 ** -13
    if chunk:
        w += 2 * half + half * spread
    else:
        w += 2.0 ** -8 if fmt4 and dtype == torch.bfloat16 else 2.0 ** -16
    tol = half * want.abs() + (w * (1 + half)) * mag + torch.finfo(dtype).tiny
    err = (got.double().cpu() - want).abs()
    assert bool((err <= tol).all()), f"{(err / tol).max().item():.3f} of the bound, {err.max().item():.3e}"


def assert_call(out, q, kvals, vvals, table, cu, kv, scale, dtype, fmt4, **kw):
    """A whole call against f64, its sequences of few columns (the decode kernel's) and of many (the chunk
    kernel's) each within their bound; the rows that it does not write hold 77."""
    want, mag, wrote = attention64(q, kvals, vvals, table, cu, kv, scale, **kw)
    assert bool((out[~wrote] == 77.0).all())
    group, d = q.shape[1] // kvals.shape[1], q.shape[2]
    many = torch.zeros_like(wrote)
    for a, b in zip(cu.tolist(), cu.tolist()[1:]):
        many[a:b] = (b - a) * group > (64 if d > 128 else 48)
    for rows, chunk in ((wrote & ~many, False), (wrote & many, True)):
        if rows.any():
            used = [page_rows(kvals, table, b, n) for b, n in enumerate(kv) if n]
            used = torch.cat([r[ok] for r, ok in used])  # (tokens, heads, d)
            spread = score_spread(q[rows], used[:, :, None], scale) if chunk else 0.0
            assert_attention(out[rows], want[rows], mag[rows], dtype, fmt4, chunk, spread)


def rope64(x, cos, sin, rope_pos, axes, kind):
    """x (total, heads, d) rotated in f64 (not rounded)."""
    half = x.shape[-1] // 2
    rows = rope_pos.long()[torch.tensor(list(axes))]
    j = torch.arange(half)[:, None]
    c, s = (t.double()[rows, j].t()[:, None] for t in (cos, sin))
    f = x.double()
    if kind == 1:
        a, b = f[..., :half], f[..., half:]
        return torch.cat((a * c - b * s, a * s + b * c), -1)
    a, b = f[..., 0::2], f[..., 1::2]
    return torch.stack((a * c - b * s, a * s + b * c), -1).flatten(-2)


def rope32(x, cos, sin, rope_pos, axes, kind):
    """The same with f32 products rounded before the sum, rounded to x's dtype."""
    half = x.shape[-1] // 2
    rows = rope_pos.long()[torch.tensor(list(axes))]
    j = torch.arange(half)[:, None]
    c, s = (t.float()[rows, j].t()[:, None] for t in (cos, sin))
    f = x.float()
    if kind == 1:
        a, b = f[..., :half], f[..., half:]
        y = torch.cat((a * c - b * s, a * s + b * c), -1)
    else:
        a, b = f[..., 0::2], f[..., 1::2]
        y = torch.stack((a * c - b * s, a * s + b * c), -1).flatten(-2)
    return y.to(x.dtype)


def angle_tables(rows, d, dtype):
    ang = torch.arange(rows, dtype=torch.float64)[:, None] * 10000.0 ** (
        -torch.arange(d // 2, dtype=torch.float64) * 2 / d)
    return ang.cos().to(dtype), ang.sin().to(dtype)


def scale_of(d):
    return 1.0 / math.sqrt(d)
