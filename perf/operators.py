"""The measured workloads of the paged cache operators: attention over a page pool, appends into it
(with and without rotary positions of several axes), and the read-back of its rows.

A page pool is a key side and a value side of the quantized cache whose planes are (page, kv head)
and whose capacity is the page size. Sequences are packed: row i of a token tensor belongs to the
sequence b with cu[b] <= i < cu[b + 1] and sits at position positions[b] + i - cu[b] of it, in page
table[b][position // page].

With `own` false run() computes the operators from elementary torch operations on the documented
pool layout; with `own` true it makes the calls of the library.
"""
import math
import os
import sys

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
_cq = None


def _lib():
    global _cq
    if _cq is None:
        sys.path.insert(0, os.path.join(os.getcwd(), "candle-rocm-vulkan_amd"))
        import cqkv
        _cq = cqkv
    return _cq


# --------------------------------------------------------------------------------------------
# the cases. Lengths are texts: "5,1*3" is [5, 1, 1, 1]
# --------------------------------------------------------------------------------------------
def _ints(text):
    out = []
    for part in text.split(","):
        v, _, n = part.partition("*")
        out += [int(v)] * (int(n) if n else 1)
    return out


def _text(values):
    return ",".join(str(v) for v in values)


def _spread(n, lo, hi):
    """n lengths between lo and hi in a fixed, uneven order."""
    return [lo + (i * 7919 * 613 + 271 * i * i) % (hi - lo + 1) for i in range(n)]


def listed():
    return [
        # the next token of one short conversation: launches and host calls are the time
        dict(name="attn_one_token_d64", kind="attn", fmt="fp8", dtype="bf16", hq=8, hkv=8, d=64,
             page=32, new="1", kv="512", window=-1, softcap=0.0),
        # a server's decode step: a full batch of different lengths, FP8 pool
        dict(name="attn_step_fp8_batch64", kind="attn", fmt="fp8", dtype="bf16", hq=32, hkv=8,
             d=128, page=64, new="1*64", kv=_text(_spread(64, 100, 8192)), window=-1, softcap=0.0),
        # long documents in a 4-bit pool, few sequences: the keys of one are split over the chip
        dict(name="attn_step_mxfp4_128k", kind="attn", fmt="mxfp4", dtype="bf16", hq=64, hkv=8,
             d=128, page=128, new="1*4", kv="131072,130001,65537,99991", window=-1, softcap=0.0),
        # speculative decoding: the drafted tokens of a batch scored in one pass
        dict(name="attn_draft_f16", kind="attn", fmt="fp8", dtype="f16", hq=32, hkv=8, d=128,
             page=32, new="5*16", kv=_text(_spread(16, 300, 8192)), window=-1, softcap=0.0),
        # one chunk of a long prompt against everything before it
        dict(name="attn_chunk_fp8_16k", kind="attn", fmt="fp8", dtype="bf16", hq=32, hkv=8, d=128,
             page=64, new="512", kv="16384", window=-1, softcap=0.0),
        # continuous batching: a prompt's chunk next to the single tokens of running sequences
        dict(name="attn_mixed_mxfp8", kind="attn", fmt="mxfp8", dtype="bf16", hq=32, hkv=8, d=128,
             page=64, new="1*11,1023,1*12", kv=_text(_spread(11, 500, 8192) + [7001] +
                                                     _spread(12, 300, 6000)),
             window=-1, softcap=0.0),
        # the new token of every running sequence written to its page, then read back
        dict(name="append_step_fp8", kind="append", fmt="fp8", dtype="bf16", hq=32, hkv=8, d=128,
             page=64, new="1*64", kv=_text(_spread(64, 100, 8192)), out="bf16"),
        # prompts quantized into a 4-bit pool, three of them behind a cached prefix
        dict(name="append_prompts_mxfp4", kind="append", fmt="mxfp4", dtype="bf16", hq=32, hkv=8,
             d=128, page=64, new="4096,1777,300,2019", kv="4096,2048,1333,2050", out="bf16"),
        # a decode step of a multimodal model: q and k rotated on three axes, k and v written
        dict(name="rope_step_mxfp8", kind="rope", fmt="mxfp8", dtype="f16", hq=16, hkv=16, d=64,
             page=32, new="1*32", kv=_text(_spread(32, 40, 4096)), axes="8,12,12", layout=1,
             out="f16"),
        # prompts with an image in them: text positions, then a grid of rows and columns
        dict(name="rope_prompt_image_fp8", kind="rope", fmt="fp8", dtype="bf16", hq=32, hkv=8,
             d=128, page=64, new="6000,333", kv="6000,901", axes="16,24,24", layout=1, out="bf16"),
        # the cached rows of a short prefix as plain values
        dict(name="read_short_mxfp8", kind="read", fmt="mxfp8", dtype="f16", hq=8, hkv=8, d=64,
             page=32, new="300", kv="300", out="f16"),
        # long sequences read back, one from the middle of its pages on
        dict(name="read_long_fp8", kind="read", fmt="fp8", dtype="bf16", hq=32, hkv=8, d=128,
             page=64, new="32768,16001", kv="32768,20000", out="bf16"),
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _draw_one(rng):
    hq, hkv = rng.choice([(8, 8), (32, 8), (32, 8), (64, 8), (12, 4), (16, 16), (32, 2), (7, 1)])
    kind = rng.choice(["attn", "attn", "attn", "append", "rope", "read"])
    c = dict(kind=kind, fmt=rng.choice(["fp8", "fp8", "mxfp8", "mxfp4"]),
             dtype=rng.choice(["bf16", "bf16", "f16"]), hq=hq, hkv=hkv,
             d=rng.choice([64, 96, 128, 128, 128, 256]), page=rng.choice([32, 64, 64, 128, 256]))
    form = rng.choice(["step", "step", "few", "chunk", "mixed"])
    batch = 1 if form == "chunk" and rng.random() < 0.5 else _log_int(rng, 1, 64)
    top = _log_int(rng, 64, 65536)
    kv = [_log_int(rng, max(1, top // 20), top) for _ in range(batch)]
    if form == "step":
        new = [1] * batch
    elif form == "few":
        n = rng.randint(2, 8)
        new = [min(n, l) for l in kv]
    else:
        n = _log_int(rng, 16, 2048)
        new = [min(l, max(1, n - rng.randint(0, n // 2))) for l in kv]
        if form == "mixed":
            new = [l if rng.random() < 0.2 else 1 for l in new]
    c.update(new=_text(new), kv=_text(kv))
    if kind == "attn":
        c.update(window=rng.choice([-1, -1, -1, 1023]), softcap=rng.choice([0.0, 0.0, 0.0, 30.0]))
    else:
        c["out"] = rng.choice(["bf16", "f16", "f32"]) if kind == "read" else c["dtype"]
    if kind == "rope":
        half = c["d"] // 2
        n = rng.choice([1, 2, 3])
        cut = sorted(rng.sample(range(1, half), n - 1))
        c.update(axes=_text(b - a for a, b in zip([0] + cut, cut + [half])),
                 layout=rng.choice([1, 2]))
    return c


def draw(rng):
    """A case of the ranges above that costs no more than the largest listed one."""
    tops = {k: [work(c) for c in listed() if c["kind"] == k] for k in ("attn", "append", "rope", "read")}
    while True:
        c = _draw_one(rng)
        w, top = work(c), tops[c["kind"]]
        if w["bytes"] > max(t["bytes"] for t in top) or w["flops"] > max(t["flops"] for t in top):
            continue
        # rows in the pool, and scores of one sequence in the plain form
        if sum(_ints(c["kv"])) * c["hkv"] * c["d"] > 1 << 29:
            continue
        if max(n * l for n, l in zip(_ints(c["new"]), _ints(c["kv"]))) * c["hq"] > 1 << 28:
            continue
        return c


# --------------------------------------------------------------------------------------------
# pool layout: codes (page, head, row, D) of keys; (page, head, row / 8, D, 8) of values; 4-bit
# codes two to a byte, low nibble first, along the last of these dims; scales an f32 per row (FP8)
# or a byte per 32 elements of a row (MX). D is the plane row: 64, 128 or 256, the head dim padded.
# --------------------------------------------------------------------------------------------
def _plane(d):
    return 64 if d <= 64 else 128 if d <= 128 else 256


def _row_bytes(fmt, d):
    """Bytes of one row that carry information."""
    return d + 4 if fmt == "fp8" else d + d // 32 if fmt == "mxfp8" else d // 2 + d // 32


def _store_codes(codes, value_side, fmt):
    """Codes (pages, heads, rows, D) uint8 -> the bytes of the pool's codes planes."""
    p, h, r, d = codes.shape
    if value_side:
        codes = codes.view(p, h, r // 8, 8, d).transpose(3, 4)
    if fmt == "mxfp4":
        codes = codes[..., 0::2] | (codes[..., 1::2] << 4)
    return codes.contiguous().view(-1)


def _load_codes(flat, pages, heads, rows, d, value_side, fmt, ids):
    """The codes (ids, heads, rows, D) uint8 of the pages `ids`."""
    last = 8 if value_side else d
    if fmt == "mxfp4":
        last //= 2
    shape = (pages, heads, rows // 8, d, last) if value_side else (pages, heads, rows, last)
    c = flat.view(shape)[ids]
    if fmt == "mxfp4":
        c = torch.stack((c & 15, c >> 4), -1).flatten(-2)
    if value_side:
        c = c.transpose(3, 4).reshape(len(ids), heads, rows, d)
    return c


_E2M1 = [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0]


def _code_values(codes, fmt):
    if fmt == "mxfp4":
        lut = torch.tensor(_E2M1 + [-v for v in _E2M1], device=codes.device)
        return lut[codes.long()]
    return codes.view(torch.float8_e4m3fn).float()


def _scale_values(sc, fmt):
    """Row scales (.., 1) f32 or block scales (.., D / 32) f32."""
    if fmt == "fp8":
        return sc.view(torch.float32)
    return torch.where(sc == 0, torch.zeros((), device=sc.device),
                       torch.ldexp(torch.ones((), device=sc.device), sc.int() - 127))


def _read_pages(state, value_side, ids):
    """The rows of pages `ids` in 32 bits: (ids, heads, rows, d)."""
    c = state["case"]
    fmt, h, r, d = c["fmt"], c["hkv"], c["page"], _plane(c["d"])
    codes, scales = state["v" if value_side else "k"]
    v = _code_values(_load_codes(codes, state["pages"], h, r, d, value_side, fmt, ids), fmt)
    s = _scale_values(scales.view(state["pages"], h, r, -1)[ids], fmt)
    if fmt != "fp8":
        s = s.repeat_interleave(32, -1)
    return (v * s)[..., :c["d"]]


def _encode(x, fmt):
    """x (.., d) f32 -> codes (.., d) uint8, scale bytes (.., 4 or d / 32)."""
    if fmt == "fp8":
        amax = x.abs().amax(-1, keepdim=True)
        s = torch.where(amax > 0, amax / 448.0, torch.ones_like(amax))
        return (x / s).to(torch.float8_e4m3fn).view(torch.uint8), s.contiguous().view(torch.uint8)
    b = x.unflatten(-1, (-1, 32))
    amax = b.abs().amax(-1, keepdim=True)
    e = torch.frexp(amax).exponent - 1 - (8 if fmt == "mxfp8" else 2)
    sc = torch.where(amax > 0, (e + 127).clamp(0, 254), torch.zeros_like(e))
    y = torch.where(sc > 0, torch.ldexp(b, -e), torch.zeros_like(b)).flatten(-2)
    if fmt == "mxfp8":
        codes = y.clamp(-448.0, 448.0).to(torch.float8_e4m3fn).view(torch.uint8)
    else:
        a = y.abs()
        codes = ((a > 0.25).to(torch.uint8) + (a >= 0.75) + (a > 1.25) + (a >= 1.75) + (a > 2.5)
                 + (a >= 3.5) + (a > 5.0)).to(torch.uint8)
        codes = codes | (torch.signbit(y).to(torch.uint8) << 3)
    codes = torch.where(sc.expand(b.shape).flatten(-2) > 0, codes, torch.zeros_like(codes))
    return codes, sc.squeeze(-1).to(torch.uint8)


# --------------------------------------------------------------------------------------------
# inputs
# --------------------------------------------------------------------------------------------
def _values(gen, shape, dtype, outliers=False):
    """N(0, 1); with `outliers` 1 % of the (head, dim) channels eight times larger."""
    x = torch.randn(shape, generator=gen, device="cuda")
    if outliers:
        m = torch.rand(shape[-2:], generator=gen, device="cuda") < 0.01
        x = torch.where(m, x * 8.0, x)
    return x.to(dtype)


def _fill_pool(gen, pages, c, value_side):
    """Quantized rows in every page: (codes bytes, scales bytes)."""
    d, dp, h, r, fmt = c["d"], _plane(c["d"]), c["hkv"], c["page"], c["fmt"]
    chan = torch.rand((h, 1, d), generator=gen, device="cuda") < 0.01
    cb, sb = [], []
    step = max(1, (1 << 26) // (h * r * dp))
    for p0 in range(0, pages, step):
        x = torch.randn((min(step, pages - p0), h, r, d), generator=gen, device="cuda")
        x = torch.where(chan, x * 8.0, x).to(DTYPES[c["dtype"]]).float()
        codes, sc = _encode(torch.nn.functional.pad(x, (0, dp - d)), fmt)
        cb.append(_store_codes(codes, value_side, fmt))
        sb.append(sc.reshape(-1))
    return torch.cat(cb), torch.cat(sb)


def _grid_positions(lens, starts, gen):
    """Rotary positions (3, total): the first third of a prompt text, then an image of rows and
    columns of patches, then text again; the third axis of a token follows the columns."""
    out = []
    for n, s in zip(lens, starts):
        p = torch.arange(n).expand(3, n).clone()
        if n >= 16:
            a, w = n // 3, int(math.sqrt(n // 3))
            m = w * (n // 3 // w)
            i = torch.arange(m)
            p[0, a:a + m] = a
            p[1, a:a + m] = a + i // w
            p[2, a:a + m] = a + i % w
            p[:, a + m:] = a + w + torch.arange(n - a - m)
        out.append(p + s)
    return torch.cat(out, 1).to(torch.int32)


def prepare(case, seed):
    c = case
    gen = torch.Generator(device="cuda").manual_seed(seed)
    new, kv = _ints(c["new"]), _ints(c["kv"])
    batch, total, dt = len(new), sum(new), DTYPES[c["dtype"]]
    need = [-(-l // c["page"]) for l in kv]
    pages = sum(need) + 3  # a few free pages
    order = torch.randperm(pages, generator=torch.Generator().manual_seed(seed)).tolist()
    table = torch.full((batch, max(need)), -1, dtype=torch.int32)
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = torch.tensor(order[at:at + n], dtype=torch.int32)
        at += n
    cu = [0]
    for n in new:
        cu.append(cu[-1] + n)
    dev = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")
    s = dict(case=c, new=new, kv=kv, pages=pages, table=table.cuda(), cu=dev(cu),
             kv_lens=dev(kv), positions=dev([l - n for l, n in zip(kv, new)]), total=total)
    s["k"], s["v"] = _fill_pool(gen, pages, c, False), _fill_pool(gen, pages, c, True)
    if c["kind"] == "attn":
        s["q"] = _values(gen, (total, c["hq"], c["d"]), dt) * 1.5
    elif c["kind"] != "read":
        # the projection output of the packed tokens: q, k and v beside each other in a row
        hs = (c["hq"] if c["kind"] == "rope" else 0) + 2 * c["hkv"]
        qkv = _values(gen, (total, hs, c["d"]), dt, True)
        s["qkv"] = qkv
        s["kx"], s["vx"] = qkv[:, -2 * c["hkv"]:-c["hkv"]], qkv[:, -c["hkv"]:]
        if c["kind"] == "rope":
            s["q"] = qkv[:, :c["hq"]]
            sections = _ints(c["axes"])
            s["axes"] = [a for a, n in enumerate(sections) for _ in range(n)]
            pos = _grid_positions(new, [l - n for l, n in zip(kv, new)], gen)[:len(sections)]
            s["rope_pos"] = pos.contiguous().cuda()
            freq = 1e6 ** (-torch.arange(c["d"] // 2, dtype=torch.float64) * 2 / c["d"])
            ang = torch.arange(int(pos.max()) + 1, dtype=torch.float64)[:, None] * freq
            s["cos"], s["sin"] = ang.cos().to(dt).cuda(), ang.sin().to(dt).cuda()
    if own:
        cq = _lib()
        fmt = cq.FORMAT_NAMES[c["fmt"]]
        for side in ("k", "v"):
            s[side + "_side"] = cq.CacheSide(fmt, side == "v", pages, c["hkv"], c["d"], c["page"],
                                             *s[side])
    return s


# --------------------------------------------------------------------------------------------
# one pass
# --------------------------------------------------------------------------------------------
def run(state):
    return _run_own(state) if own else _run_plain(state)


def _run_own(s):
    cq, c = _lib(), s["case"]
    ks, vs = s["k_side"], s["v_side"]
    if c["kind"] == "attn":
        return cq.paged_attention(s["q"], ks, vs, s["table"], s["cu"], s["kv_lens"], max(s["new"]),
                                  max(s["kv"]), 1.0 / math.sqrt(c["d"]), True,
                                  window_left=c["window"], softcap=c["softcap"])
    read = lambda side: cq.paged_dequantize(side, s["table"], s["cu"], s["positions"], s["total"],
                                            dtype=DTYPES[c["out"]])
    if c["kind"] == "append":
        cq.paged_append(ks, vs, s["kx"], s["vx"], s["table"], s["cu"], s["positions"])
        return read(ks), read(vs)
    if c["kind"] == "rope":
        q = cq.paged_rope_append(ks, vs, s["q"], s["kx"], s["vx"], s["cos"], s["sin"],
                                 s["rope_pos"], s["axes"], s["table"], s["cu"], s["positions"],
                                 kind=c["layout"])
        return q, read(ks), read(vs)
    return read(ks), read(vs)


def _slots(s):
    """Page id and row in it of every packed token."""
    c, page, row = s["case"], [], []
    for b, (n, l) in enumerate(zip(s["new"], s["kv"])):
        p = torch.arange(l - n, l, device="cuda")
        page.append(s["table"][b][p // c["page"]])
        row.append(p % c["page"])
    return torch.cat(page).long(), torch.cat(row)


def _plain_write(s, x, value_side, page, row):
    """Quantizes x (total, heads, d) f32 into rows (page, row) of the pool."""
    c = s["case"]
    fmt, h, r, dp = c["fmt"], c["hkv"], c["page"], _plane(c["d"])
    codes, sc = _encode(torch.nn.functional.pad(x, (0, dp - c["d"])), fmt)
    flat, scales = s["v" if value_side else "k"]
    ids, at = torch.unique(page, return_inverse=True)
    whole = _load_codes(flat, s["pages"], h, r, dp, value_side, fmt, ids).contiguous()
    whole[at, :, row] = codes
    flat.view(s["pages"], -1)[ids] = _store_codes(whole, value_side, fmt).view(len(ids), -1)
    scales.view(s["pages"], h, r, -1)[page, :, row] = sc


def _plain_read(s, value_side, page, row):
    ids, at = torch.unique(page, return_inverse=True)
    return _read_pages(s, value_side, ids)[at, :, row].to(DTYPES[s["case"]["out"]])


def _plain_rope(s, x):
    """x (total, heads, d) rotated in 32 bits, rounded to its dtype."""
    c = s["case"]
    half = c["d"] // 2
    axis = torch.tensor(s["axes"], device="cuda")
    rows = s["rope_pos"].long()[axis]  # (d / 2, total)
    pair = torch.arange(half, device="cuda")[:, None]
    cos, sin = (t.float()[rows, pair].t()[:, None] for t in (s["cos"], s["sin"]))
    f = x.float()
    if c["layout"] == 1:
        x0, x1 = f[..., :half], f[..., half:]
        y = torch.cat((x0 * cos - x1 * sin, x0 * sin + x1 * cos), -1)
    else:
        x0, x1 = f[..., 0::2], f[..., 1::2]
        y = torch.stack((x0 * cos - x1 * sin, x0 * sin + x1 * cos), -1).flatten(-2)
    return y.to(x.dtype)


def _plain_attention(s):
    c = s["case"]
    hq, hkv, d, g = c["hq"], c["hkv"], c["d"], c["hq"] // c["hkv"]
    out = torch.zeros_like(s["q"])
    row = 0
    for b, (n, l) in enumerate(zip(s["new"], s["kv"])):
        first = max(0, l - n - c["window"]) // c["page"] if c["window"] >= 0 else 0
        ids = s["table"][b, first:-(-l // c["page"])].long()
        k, v = (_read_pages(s, side, ids).transpose(0, 1).reshape(hkv, -1, d)[:, :l - first * c["page"]]
                for side in (False, True))
        q = s["q"][row:row + n].float().view(n, hkv, g, d).permute(1, 2, 0, 3).reshape(hkv, g * n, d)
        x = torch.matmul(q, k.transpose(1, 2).contiguous()) * (1.0 / math.sqrt(d))
        if c["softcap"] > 0:
            x = torch.tanh(x / c["softcap"]) * c["softcap"]
        pos = torch.arange(l - n, l, device="cuda").repeat(g)[:, None]
        key = torch.arange(first * c["page"], l, device="cuda")[None]
        hide = key > pos
        if c["window"] >= 0:
            hide = hide | (key < pos - c["window"])
        x = x.masked_fill(hide, -math.inf)
        p = torch.exp(x - x.amax(-1, keepdim=True))
        o = torch.matmul(p, v) / p.sum(-1, keepdim=True)
        out[row:row + n] = o.view(hkv, g, n, d).permute(2, 0, 1, 3).reshape(n, hq, d).to(out.dtype)
        row += n
    return out


def _run_plain(s):
    c = s["case"]
    if c["kind"] == "attn":
        return _plain_attention(s)
    page, row = _slots(s)
    read = lambda side: _plain_read(s, side, page, row)
    if c["kind"] == "read":
        return read(False), read(True)
    if c["kind"] == "append":
        _plain_write(s, s["kx"].float(), False, page, row)
        _plain_write(s, s["vx"].float(), True, page, row)
        return read(False), read(True)
    q, k = _plain_rope(s, s["q"]), _plain_rope(s, s["kx"])
    _plain_write(s, k.float(), False, page, row)
    _plain_write(s, s["vx"].float(), True, page, row)
    return q, read(False), read(True)


# --------------------------------------------------------------------------------------------
# what a pass cannot do without
# --------------------------------------------------------------------------------------------
def work(case):
    c = case
    new, kv = _ints(c["new"]), _ints(c["kv"])
    total, rb, esz = sum(new), _row_bytes(c["fmt"], c["d"]), 2
    head = total * c["d"] * esz
    if c["kind"] == "attn":
        seen = pairs = 0
        for n, l in zip(new, kv):
            w = c["window"] if c["window"] >= 0 else l
            seen += l - max(0, l - n - w)
            pairs += sum(min(p, w) + 1 for p in range(l - n, l))
        return {"bytes": 2 * seen * c["hkv"] * rb + 2 * head * c["hq"],
                "flops": 4 * c["d"] * c["hq"] * pairs}
    out = total * c["d"] * c["hkv"] * (4 if c["out"] == "f32" else 2)
    read = 2 * (total * c["hkv"] * rb + out)
    flops = 2 * total * c["hkv"] * c["d"]
    if c["kind"] == "read":
        return {"bytes": read, "flops": flops}
    write = 2 * (head * c["hkv"] + total * c["hkv"] * rb)
    flops += 6 * total * c["hkv"] * c["d"]
    if c["kind"] == "rope":
        write += 2 * head * c["hq"] + total * (c["d"] * esz + 4 * len(_ints(c["axes"])))
        flops += 3 * total * (c["hq"] + c["hkv"]) * c["d"]
    return {"bytes": read + write, "flops": flops}


# --------------------------------------------------------------------------------------------
# the definitions in 64 bits
# --------------------------------------------------------------------------------------------
def _e4m3_table():
    t = []
    for b in range(128):
        e, m = b >> 3, b & 7
        t.append(m * 2.0 ** -9 if e == 0 else math.nan if b == 127 else (8 + m) * 2.0 ** (e - 10))
    return torch.tensor(t + [-v for v in t], dtype=torch.float64, device="cuda")


def _exact_rows(s, value_side, page, row):
    """The values (tokens, heads, d) that the pool's bytes stand for, from their addresses."""
    c = s["case"]
    fmt, h, r, d, dp = c["fmt"], c["hkv"], c["page"], c["d"], _plane(c["d"])
    codes, scales = s["v" if value_side else "k"]
    page, row = page[:, None, None].long(), row[:, None, None].long()
    head = torch.arange(h, device="cuda")[None, :, None]
    j = torch.arange(d, device="cuda")[None, None]
    plane = page * h + head
    unit = plane * r * dp + (row // 8 * dp * 8 + j * 8 + row % 8 if value_side else row * dp + j)
    if fmt == "mxfp4":
        nib = (codes[unit // 2].int() >> (4 * (unit % 2)).int()) & 15
        mag = torch.tensor(_E2M1, dtype=torch.float64, device="cuda")
        val = mag[(nib & 7).long()] * (1 - 2 * (nib >> 3)).double()
    else:
        val = _e4m3_table()[codes[unit].long()]
    if fmt == "fp8":
        return val * scales.view(torch.float32).double()[plane * r + row]
    e = scales[(plane * r + row) * (dp // 32) + j // 32].double()
    return val * torch.where(e > 0, torch.exp2(e - 127.0), torch.zeros_like(e))


def _nearest(y, table):
    """The entry of `table` (non-negative values in order) nearest |y|, ties to the even index."""
    a = y.abs().contiguous()
    i = torch.searchsorted(table, a).clamp(1, len(table) - 1)
    lo, hi = table[i - 1], table[i]
    up = (a - lo > hi - a) | ((a - lo == hi - a) & (i % 2 == 0))
    return torch.where(up, hi, lo) * torch.where(torch.signbit(y), -1.0, 1.0)


def _exact_quant(x, fmt):
    """Quantized and dequantized x (.., d) f64."""
    if fmt == "fp8":
        amax = x.abs().amax(-1, keepdim=True)
        # the scale is stored in 32 bits and the code is that of the 32-bit quotient, by definition:
        # with 8-bit significands many quotients by the unrounded scale lie on a tie
        s = torch.where(amax > 0, amax / 448.0, torch.ones_like(amax)).float().double()
        return _nearest((x / s).float().double(), _e4m3_table()[:127].contiguous()) * s
    b = x.unflatten(-1, (-1, 32))
    amax = b.abs().amax(-1, keepdim=True)
    s = torch.exp2(torch.floor(torch.log2(amax.clamp_min(1e-300))) - (8 if fmt == "mxfp8" else 2))
    t = _e4m3_table()[:127].contiguous() if fmt == "mxfp8" else \
        torch.tensor(_E2M1, dtype=torch.float64, device="cuda")
    y = _nearest(b / s, t) * s
    return torch.where(amax > 0, y, torch.zeros_like(y)).flatten(-2)


def _exact_rope(s, x):
    c = s["case"]
    half = c["d"] // 2
    y = x.double().clone()
    for j in range(half):
        r = s["rope_pos"][s["axes"][j]].long()
        cos, sin = s["cos"][r, j].double()[:, None], s["sin"][r, j].double()[:, None]
        a, b = (j, j + half) if c["layout"] == 1 else (2 * j, 2 * j + 1)
        x0, x1 = x[..., a].double(), x[..., b].double()
        y[..., a], y[..., b] = x0 * cos - x1 * sin, x0 * sin + x1 * cos
    return y


def _exact_attention(s):
    c = s["case"]
    g = c["hq"] // c["hkv"]
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    row = 0
    for b, (n, l) in enumerate(zip(s["new"], s["kv"])):
        lo = max(0, l - n - c["window"]) if c["window"] >= 0 else 0
        p = torch.arange(lo, l, device="cuda")
        page = s["table"][b][p // c["page"]]
        k, v = (_exact_rows(s, side, page, p % c["page"]) for side in (False, True))
        pos = torch.arange(l - n, l, device="cuda")[:, None]
        see = p[None] <= pos
        if c["window"] >= 0:
            see &= p[None] >= pos - c["window"]
        for h in range(c["hq"]):
            x = s["q"][row:row + n, h].double() @ k[:, h // g].T / math.sqrt(c["d"])
            if c["softcap"] > 0:
                x = c["softcap"] * torch.tanh(x / c["softcap"])
            w = torch.softmax(x.masked_fill(~see, -math.inf), -1)
            out[row:row + n, h] = w @ v[:, h // g]
        row += n
    return out


def exact(case, seed):
    global own
    was, own = own, False
    try:
        s = prepare(case, seed)
    finally:
        own = was
    c = case
    if c["kind"] == "attn":
        return _exact_attention(s)
    if c["kind"] == "read":
        page, row = _slots(s)
        return _exact_rows(s, False, page, row), _exact_rows(s, True, page, row)
    v = _exact_quant(s["vx"].double(), c["fmt"])
    if c["kind"] == "append":
        return _exact_quant(s["kx"].double(), c["fmt"]), v
    # the rotated keys are rows of the dtype, which are then quantized
    k = _exact_rope(s, s["kx"]).to(DTYPES[c["dtype"]]).double()
    return _exact_rope(s, s["q"]), _exact_quant(k, c["fmt"]), v
