"""Page pools on the GPU: the codes of appends against the dense appends (bit for bit), rotary axes
against f32 torch (bit for bit) and f64, the read-back against the dense read-back, attention against
f64 over the pool's values."""
import pytest
import torch

from tests import paged_reference as R

pytestmark = pytest.mark.gpu

FP8, MXFP8, MXFP4 = 5, 4, 2
DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}


def view_of_page(cq, side, page_id):
    """One page of a pool as a dense side of batch 1 over the same memory."""
    cb, sb = side.codes.numel() // side.batch, side.scales.numel() // side.batch
    return cq.CacheSide(side.fmt, side.is_value, 1, side.kv_heads, side.head_dim, side.capacity,
                        side.codes[page_id * cb:(page_id + 1) * cb],
                        side.scales[page_id * sb:(page_id + 1) * sb])


def copy_side(cq, s):
    return cq.CacheSide(s.fmt, s.is_value, s.batch, s.kv_heads, s.head_dim, s.capacity,
                        s.codes.clone(), s.scales.clone())


def dense_append(cq, side, x, table, cu, starts):
    """The packed rows through the dense append, page by page."""
    cu = cu.tolist()
    for b, s in enumerate(starts):
        p, end = s, s + cu[b + 1] - cu[b]
        while p < end and s >= 0:
            n = min(end - p, side.capacity - p % side.capacity)
            slot = p // side.capacity
            page = int(table[b, slot]) if slot < table.shape[1] else -1
            if 0 <= page < side.batch:
                rows = x[cu[b] + p - s:cu[b] + p - s + n].transpose(0, 1)[None].contiguous()
                cq.quant_append(view_of_page(cq, side, page), rows, p % side.capacity)
            p += n


def random_bytes(t, seed):
    g = torch.Generator().manual_seed(seed)
    t.copy_(torch.randint(0, 256, (t.numel(),), generator=g, dtype=torch.uint8))


def empty_pool(cq, dev, fmt, pages, hkv, d, page):
    sides = [cq.CacheSide.empty(fmt, v, pages, hkv, d, page, dev) for v in (False, True)]
    for i, s in enumerate(sides):
        random_bytes(s.codes, 7 + i)
        random_bytes(s.scales, 9 + i)
    return sides


def assert_same_pool(a, b, hkv, d):
    """Bytes equal; the plane rows past the head dim are zero codes in both."""
    assert torch.equal(a.codes, b.codes)
    assert torch.equal(a.scales, b.scales)


APPENDS = [
    # fmt, d, hkv, page, dtype, row counts, first positions
    (FP8, 128, 8, 64, "bf16", [1, 1, 1], [0, 63, 64]),
    (FP8, 128, 2, 32, "bf16", [5, 0, 33, 100], [3, 10, 31, 0]),
    (FP8, 64, 3, 32, "f16", [17, 1, 64], [0, 7, 40]),
    (FP8, 256, 2, 64, "bf16", [9, 70], [60, 1]),
    (FP8, 96, 5, 64, "bf16", [70, 3], [10, 62]),
    (FP8, 80, 2, 32, "f32", [40], [5]),
    (FP8, 5, 1, 32, "f16", [33, 2], [1, 0]),
    (FP8, 256, 1, 128, "f32", [3], [126]),
    (MXFP8, 128, 8, 64, "bf16", [1, 200], [5, 0]),
    (MXFP8, 64, 16, 32, "f16", [31, 1], [1, 8]),
    (MXFP8, 256, 3, 32, "bf16", [40], [30]),
    (MXFP8, 96, 1, 64, "f32", [11], [0]),
    (MXFP4, 128, 8, 64, "bf16", [1, 1, 130], [0, 9, 3]),
    (MXFP4, 64, 5, 32, "f16", [7, 8, 9], [0, 8, 15]),
    (MXFP4, 256, 2, 256, "bf16", [300], [100]),
    (MXFP4, 32, 2, 32, "bf16", [20], [13]),
]


@pytest.mark.parametrize("fmt,d,hkv,page,dtype,lens,starts", APPENDS)
def test_append_codes(cq, dev, fmt, d, hkv, page, dtype, lens, starts):
    pages = sum(-(-(s + n) // page) for s, n in zip(starts, lens)) + 2
    k, v = empty_pool(cq, dev, fmt, pages, hkv, d, page)
    k2, v2 = copy_side(cq, k), copy_side(cq, v)
    table = R.make_table([s + n for s, n in zip(starts, lens)], page, pages, dev, 1)
    cu = R.prefix(lens, dev)
    g = torch.Generator().manual_seed(3)
    x = torch.randn(sum(lens), 2 * hkv + 1, d, generator=g)
    x[:, 1] *= 40
    if sum(lens) > 4:
        x[2] = 0
    x = x.to(DTYPES[dtype]).to(dev)
    kx, vx = x[:, :hkv], x[:, hkv:2 * hkv]  # strided rows
    cq.paged_append(k, v, kx, vx, table, cu, R.ints(starts, dev))
    dense_append(cq, k2, kx, table, cu, starts)
    dense_append(cq, v2, vx, table, cu, starts)
    assert_same_pool(k, k2, hkv, d)
    assert_same_pool(v, v2, hkv, d)


@pytest.mark.parametrize("fmt", [FP8, MXFP8, MXFP4])
def test_append_special_values(cq, dev, fmt):
    """NaN, infinities, zeros, subnormals and the largest values: the dense append's codes."""
    hkv, d, page = 2, 128, 32
    k, v = empty_pool(cq, dev, fmt, 4, hkv, d, page)
    k2, v2 = copy_side(cq, k), copy_side(cq, v)
    x = torch.randn(40, 2 * hkv, d, generator=torch.Generator().manual_seed(1))
    x[0, :, 3] = float("nan")
    x[1, :, 70] = float("inf")
    x[2, :, 5] = -float("inf")
    x[3] = -0.0
    x[4] = 1e-39
    x[5] *= 1e-36
    x[6, :, 9] = 3e38
    x[7] = 1.0
    x = x.to(torch.bfloat16).to(dev)
    table, cu = R.make_table([40], page, 4, dev, 1), R.prefix([40], dev)
    cq.paged_append(k, v, x[:, :hkv], x[:, hkv:], table, cu, R.ints([0], dev))
    dense_append(cq, k2, x[:, :hkv], table, cu, [0])
    dense_append(cq, v2, x[:, hkv:], table, cu, [0])
    assert_same_pool(k, k2, hkv, d)
    assert_same_pool(v, v2, hkv, d)


@pytest.mark.parametrize("fmt", [FP8, MXFP4])
def test_append_misaligned_rows(cq, dev, fmt):
    """Rows off 16-byte boundaries take the element path: the same codes."""
    hkv, d, page = 3, 64, 32
    k, v = empty_pool(cq, dev, fmt, 4, hkv, d, page)
    k2, v2 = copy_side(cq, k), copy_side(cq, v)
    flat = torch.randn(1 + 50 * hkv * 67 * 2, generator=torch.Generator().manual_seed(1)).to(torch.bfloat16).to(dev)
    x = flat[1:].view(50, 2 * hkv, 67)[..., :d]
    table, cu = R.make_table([50], page, 4, dev, 1), R.prefix([50], dev)
    cq.paged_append(k, v, x[:, :hkv], x[:, hkv:], table, cu, R.ints([0], dev))
    dense_append(cq, k2, x[:, :hkv], table, cu, [0])
    dense_append(cq, v2, x[:, hkv:], table, cu, [0])
    assert_same_pool(k, k2, hkv, d)
    assert_same_pool(v, v2, hkv, d)


def test_append_holes_and_ends(cq, dev):
    """Pages outside the pool, positions past the table, negative first positions and rows outside
    every sequence leave the pool alone."""
    hkv, d, page, pages = 2, 64, 32, 5
    k, v = empty_pool(cq, dev, FP8, pages, hkv, d, page)
    k2, v2 = copy_side(cq, k), copy_side(cq, v)
    table = torch.tensor([[0, -1, 1], [pages, 2, -2 ** 31], [3, 4, 2 ** 31 - 1]], dtype=torch.int32, device=dev)
    starts, lens = [0, 10, -1], [130, 70, 9]  # the first runs past the table's three pages
    cu = R.prefix(lens, dev, first=4)
    x = torch.randn(4 + sum(lens) + 6, 2 * hkv, d, generator=torch.Generator().manual_seed(1)).to(torch.bfloat16).to(dev)
    cq.paged_append(k, v, x[:, :hkv], x[:, hkv:], table, cu, R.ints(starts, dev))
    dense_append(cq, k2, x[:, :hkv], table, cu, starts)
    dense_append(cq, v2, x[:, hkv:], table, cu, starts)
    assert_same_pool(k, k2, hkv, d)
    assert_same_pool(v, v2, hkv, d)
    got = cq.paged_dequantize(k, table, cu, R.ints(starts, dev), x.shape[0], out=torch.full(
        (x.shape[0], hkv, d), 7.0, device=dev))
    vals = cq.dequantize(k, page).cpu()
    want = torch.full((x.shape[0], hkv, d), 7.0)
    want[4:134] = 0
    want[134:204] = 0
    for i in range(130):
        p = i
        if p // page < 3 and p // page != 1:
            want[4 + i] = vals[int(table[0, p // page]), :, p % page]
    for i in range(70):
        p = 10 + i
        if p // page == 1:
            want[134 + i] = vals[2, :, p % page]
    assert torch.equal(got.cpu(), want)


@pytest.mark.parametrize("batch", [1, 64, 65, 200])
def test_append_many_sequences(cq, dev, batch):
    """The tile search over more sequences than a wavefront has lanes, some of them empty."""
    hkv, d, page = 1, 64, 32
    lens = [(i * 7) % 5 for i in range(batch)]
    starts = [(i * 13) % 40 for i in range(batch)]
    lens[0] = 3
    kv = [s + n for s, n in zip(starts, lens)]
    pages = sum(-(-n // page) for n in kv) + 1
    k, v = empty_pool(cq, dev, FP8, pages, hkv, d, page)
    k2, v2 = copy_side(cq, k), copy_side(cq, v)
    table, cu = R.make_table(kv, page, pages, dev, 2), R.prefix(lens, dev)
    x = torch.randn(sum(lens), 2, d, generator=torch.Generator().manual_seed(1)).to(torch.bfloat16).to(dev)
    cq.paged_append(k, v, x[:, :1], x[:, 1:], table, cu, R.ints(starts, dev))
    dense_append(cq, k2, x[:, :1], table, cu, starts)
    dense_append(cq, v2, x[:, 1:], table, cu, starts)
    assert_same_pool(k, k2, hkv, d)
    assert_same_pool(v, v2, hkv, d)


ROPES = [
    # fmt, d, hq, hkv, dtype, kind, sections
    (FP8, 128, 8, 2, "bf16", 1, (16, 24, 24)),
    (FP8, 128, 5, 5, "f16", 2, (16, 24, 24)),
    (FP8, 128, 8, 1, "bf16", 1, (13, 30, 21)),  # sections that end inside a table chunk
    (MXFP8, 64, 4, 4, "f16", 1, (8, 12, 12)),
    (MXFP8, 256, 3, 1, "bf16", 1, (40, 44, 44)),
    (MXFP4, 96, 4, 2, "bf16", 1, (16, 16, 8, 8)),
    (MXFP4, 128, 4, 2, "bf16", 2, (5, 59)),
    (FP8, 80, 2, 2, "bf16", 1, (40,)),
    (FP8, 6, 2, 1, "f16", 1, (1, 2)),
    (FP8, 64, 2, 2, "f32", 1, (10, 11, 11)),
    (FP8, 64, 2, 2, "f32", 2, (32,)),
    (FP8, 36, 2, 1, "bf16", 1, (9, 9)),
]


@pytest.mark.parametrize("fmt,d,hq,hkv,dtype,kind,sections", ROPES)
def test_rope_axes(cq, dev, fmt, d, hq, hkv, dtype, kind, sections):
    page, lens, starts = 32, [1, 37, 20], [31, 5, 0]
    kv = [s + n for s, n in zip(starts, lens)]
    pages = sum(-(-n // page) for n in kv) + 1
    k, v = empty_pool(cq, dev, fmt, pages, hkv, d, page)
    k2, v2 = copy_side(cq, k), copy_side(cq, v)
    table, cu = R.make_table(kv, page, pages, dev, 4), R.prefix(lens, dev)
    total, dt = sum(lens), DTYPES[dtype]
    g = torch.Generator().manual_seed(5)
    x = torch.randn(total, hq + 2 * hkv, d, generator=g).to(dt)
    cos, sin = R.angle_tables(50, d, dt)
    rp = torch.randint(0, 50, (len(sections), total), generator=g, dtype=torch.int32)
    axes = cq.rope_sections(sections)
    xd = x.to(dev)
    q, kx, vx = xd[:, :hq], xd[:, hq:hq + hkv], xd[:, hq + hkv:]
    got = cq.paged_rope_append(k, v, q, kx, vx, cos.to(dev), sin.to(dev), rp.to(dev), axes, table, cu,
                               R.ints(starts, dev), kind=kind)
    want = R.rope32(x[:, :hq], cos, sin, rp, axes, kind)
    assert torch.equal(got.cpu(), want)
    # against f64: two products and a sum of f32, each within 2^-24 of at most sqrt(2) |x|, and the
    # rounding to the dtype (half a step, and none for f32 beyond those)
    exact = R.rope64(x[:, :hq], cos, sin, rp, axes, kind)
    half = torch.finfo(dt).eps / 2
    err = (got.cpu().double() - exact).abs()
    assert bool((err <= half * exact.abs() * (1 + 2 ** -20) + 4 * 2.0 ** -24 * x[:, :hq].double().abs().max()).all())
    rot = R.rope32(x[:, hq:hq + hkv], cos, sin, rp, axes, kind).to(dev)
    dense_append(cq, k2, rot, table, cu, starts)
    dense_append(cq, v2, vx, table, cu, starts)
    assert_same_pool(k, k2, hkv, d)
    assert_same_pool(v, v2, hkv, d)


@pytest.mark.parametrize("kind", [1, 2])
def test_rope_one_axis_is_the_dense_rope_append(cq, dev, kind):
    b, hq, hkv, d, t, page = 2, 8, 2, 128, 40, 32
    g = torch.Generator().manual_seed(2)
    q, kx, vx = (torch.randn(b, h, t, d, generator=g).to(torch.bfloat16).to(dev) for h in (hq, hkv, hkv))
    cos, sin = (x.to(dev) for x in R.angle_tables(100, d, torch.bfloat16))
    cache = cq.TurboKvCache(cq.FP8, cq.FP8, b, hkv, d, 64, device=dev)
    want = cq.rope_quant_append(cache.k, cache.v, q, kx, vx, cos, sin, kind=kind, position=3)
    k, v = empty_pool(cq, dev, cq.FP8, 5, hkv, d, page)
    table, cu = R.make_table([t + 3] * b, page, 5, dev, 4), R.prefix([t] * b, dev)
    rp = torch.cat([torch.arange(3, 3 + t)] * b).to(torch.int32)[None].to(dev)
    pack = lambda x: x.transpose(1, 2).reshape(b * t, -1, d)
    got = cq.paged_rope_append(k, v, pack(q), pack(kx), pack(vx), cos, sin, rp, [0] * (d // 2), table,
                               cu, R.ints([3] * b, dev), kind=kind)
    assert torch.equal(got, pack(want))
    for pool, dense in ((k, cache.k), (v, cache.v)):
        got = cq.paged_dequantize(pool, table, cu, R.ints([3] * b, dev), b * t)
        assert torch.equal(got, pack(cq.dequantize(dense, t, position=3)))


@pytest.mark.parametrize("fmt", [FP8, MXFP8, MXFP4])
@pytest.mark.parametrize("kind", [1, 2])
def test_rope_special_values(cq, dev, fmt, kind):
    """Infinities, zeros, subnormals and the largest values through the rotation: the codes are those of
    the rotated rows."""
    hq, hkv, d, page, n = 1, 2, 128, 32, 45
    k, v = empty_pool(cq, dev, fmt, 2, hkv, d, page)
    k2, v2 = copy_side(cq, k), copy_side(cq, v)
    x = torch.randn(n, hq + 2 * hkv, d, generator=torch.Generator().manual_seed(1))
    x[1, :, 70] = float("inf")
    x[2, :, 5] = -float("inf")
    x[3] = -0.0
    x[4] = 1e-39
    x[5] *= 1e-36
    x[6, :, 9] = 3e38
    x[13, 2, 3] = float("inf")
    x[20] = 0.0
    x = x.to(torch.bfloat16)
    cos, sin = R.angle_tables(60, d, torch.bfloat16)
    rp = torch.randint(1, 60, (2, n), generator=torch.Generator().manual_seed(2), dtype=torch.int32)
    axes = cq.rope_sections((24, 40))
    table, cu = R.make_table([n + 3], page, 2, dev, 1), R.prefix([n], dev)
    xd = x.to(dev)
    got = cq.paged_rope_append(k, v, xd[:, :hq], xd[:, hq:hq + hkv], xd[:, hq + hkv:], cos.to(dev),
                               sin.to(dev), rp.to(dev), axes, table, cu, R.ints([3], dev), kind=kind)
    assert torch.equal(got.cpu(), R.rope32(x[:, :hq], cos, sin, rp, axes, kind))
    rot = R.rope32(x[:, hq:hq + hkv], cos, sin, rp, axes, kind)
    assert not bool(rot.isnan().any())
    dense_append(cq, k2, rot.to(dev), table, cu, [3])
    dense_append(cq, v2, xd[:, hq + hkv:], table, cu, [3])
    assert_same_pool(k, k2, hkv, d)
    assert_same_pool(v, v2, hkv, d)


@pytest.mark.parametrize("fmt,d,hq,hkv,dtype", [(FP8, 256, 14, 2, "bf16"), (MXFP4, 128, 17, 3, "f16"), (MXFP8, 64, 33, 9, "bf16")])
def test_rope_long_call(cq, dev, fmt, d, hq, hkv, dtype):
    """Calls so long that a wavefront takes two head groups (of k, of q, of both): holes keep their
    queries, rows with an angle outside the tables are left out, an infinity in a key."""
    page, lens, starts = 64, [5000, 1, 2000], [3, 900, 0]
    kv = [s + n for s, n in zip(starts, lens)]
    pages = sum(-(-n // page) for n in kv)
    k, v = empty_pool(cq, dev, fmt, pages, hkv, d, page)
    k2, v2 = copy_side(cq, k), copy_side(cq, v)
    table, cu = R.make_table(kv, page, pages, dev, 4), R.prefix(lens, dev)
    table[0, 7] = -1
    total, dt = sum(lens), DTYPES[dtype]
    g = torch.Generator().manual_seed(5)
    x = torch.randn(total, hq + 2 * hkv, d, generator=g).to(dt)
    x[77, hq, 3] = float("inf")
    cos, sin = R.angle_tables(50, d, dt)
    rp = torch.randint(1, 50, (2, total), generator=g, dtype=torch.int32)
    axes = cq.rope_sections((16, d // 2 - 16))
    rp[1, 1234] = 50
    xd = x.to(dev)
    out = torch.full((total, hq, d), 5.0, dtype=dt, device=dev)
    cq.paged_rope_append(k, v, xd[:, :hq], xd[:, hq:hq + hkv], xd[:, hq + hkv:], cos.to(dev), sin.to(dev),
                         rp.to(dev), axes, table, cu, R.ints(starts, dev), q_out=out)
    rp[1, 1234] = 49
    want = R.rope32(x[:, :hq], cos, sin, rp, axes, 1)
    want[1234] = 5.0
    assert torch.equal(out.cpu(), want)
    rot = R.rope32(x[:, hq:hq + hkv], cos, sin, rp, axes, 1).to(dev)
    # (the dense appends of the packed rows in front of and behind the one left out)
    for a, b, first in ((0, 1234, 3), (1235, 5000, 3 + 1235)):
        dense_append(cq, k2, rot[a:b], table, R.prefix([b - a], dev), [first])
        dense_append(cq, v2, xd[a:b, hq + hkv:], table, R.prefix([b - a], dev), [first])
    dense_append(cq, k2, rot[5000:], table[1:], R.prefix(lens[1:], dev), starts[1:])
    dense_append(cq, v2, xd[5000:, hq + hkv:], table[1:], R.prefix(lens[1:], dev), starts[1:])
    assert_same_pool(k, k2, hkv, d)
    assert_same_pool(v, v2, hkv, d)


def test_rope_positions_outside_the_tables(cq, dev):
    """A row with one angle outside the tables: q_out, k and v left as they were."""
    hq, hkv, d, page, n = 2, 1, 64, 32, 20
    k, v = empty_pool(cq, dev, FP8, 2, hkv, d, page)
    k2, v2 = copy_side(cq, k), copy_side(cq, v)
    g = torch.Generator().manual_seed(2)
    x = torch.randn(n, hq + 2 * hkv, d, generator=g).to(torch.bfloat16)
    cos, sin = R.angle_tables(30, d, torch.bfloat16)
    rp = torch.randint(0, 30, (2, n), generator=g, dtype=torch.int32)
    rp[0, 3], rp[1, 9], rp[0, 10], rp[1, 19] = 30, -1, 2 ** 31 - 1, -2 ** 31
    out = torch.full((n, hq, d), 5.0, dtype=torch.bfloat16, device=dev)
    table, cu = R.make_table([n], page, 2, dev, 1), R.prefix([n], dev)
    axes = [0] * 16 + [1] * 16
    xd = x.to(dev)
    cq.paged_rope_append(k, v, xd[:, :hq], xd[:, hq:hq + 1], xd[:, hq + 1:], cos.to(dev), sin.to(dev),
                         rp.to(dev), axes, table, cu, R.ints([0], dev), q_out=out)
    ok = ((rp >= 0) & (rp < 30)).all(0)
    safe = rp.clamp(0, 29)
    want = torch.where(ok[:, None, None], R.rope32(x[:, :hq], cos, sin, safe, axes, 1).float(), 5.0)
    assert torch.equal(out.cpu().float(), want)
    rot = R.rope32(x[:, hq:hq + 1], cos, sin, safe, axes, 1).to(dev)
    for i in range(n):
        if ok[i]:
            dense_append(cq, k2, rot[i:i + 1], table, R.prefix([1], dev), [i])
            dense_append(cq, v2, xd[i:i + 1, hq + 1:], table, R.prefix([1], dev), [i])
    assert_same_pool(k, k2, hkv, d)
    assert_same_pool(v, v2, hkv, d)


@pytest.mark.parametrize("fmt", [FP8, MXFP8, MXFP4])
@pytest.mark.parametrize("d,dtype", [(64, "f16"), (96, "bf16"), (128, "bf16"), (128, "f32"), (256, "f16")])
def test_read_back(cq, dev, fmt, d, dtype):
    hkv, page, lens, starts = 3, 64, [1, 130, 7, 0, 64], [63, 0, 100, 3, 64]
    kv = [s + n for s, n in zip(starts, lens)]
    pages = sum(-(-n // page) for n in kv) + 1
    sides = R.make_pool(cq, dev, fmt, pages, hkv, d, page, 3)
    table, cu = R.make_table(kv, page, pages, dev, 6), R.prefix(lens, dev)
    for side in sides:
        vals = cq.dequantize(side, page, dtype=DTYPES[dtype]).cpu()
        got = cq.paged_dequantize(side, table, cu, R.ints(starts, dev), sum(lens), dtype=DTYPES[dtype])
        at = 0
        for b, (s, n) in enumerate(zip(starts, lens)):
            rows, ok = R.page_rows(vals, table, b, s + n)
            assert ok.all() and torch.equal(got[at:at + n].cpu(), rows[s:])
            at += n


def test_read_back_into_strided_rows(cq, dev):
    side, _ = R.make_pool(cq, dev, FP8, 4, 2, 80, 32, 3)
    table, cu = R.make_table([100], 32, 4, dev, 6), R.prefix([100], dev)
    buf = torch.full((100, 3, 83), 9.0, dtype=torch.float16, device=dev)
    cq.paged_dequantize(side, table, cu, R.ints([0], dev), 100, out=buf[:, 1:, 1:81])
    want, _ = R.page_rows(cq.dequantize(side, 32, dtype=torch.float16).cpu(), table, 0, 100)
    assert torch.equal(buf[:, 1:, 1:81].cpu(), want)
    buf[:, 1:, 1:81] = 9.0
    assert bool((buf == 9.0).all())


# ---------------------------------------------------------------------------------------------
# attention
# ---------------------------------------------------------------------------------------------
ATTN = [
    # fmt, d, hq, hkv, page, dtype, new, kv
    (FP8, 128, 8, 2, 64, "bf16", [1], [1]),
    (FP8, 128, 8, 8, 32, "bf16", [1, 1, 1], [31, 32, 33]),
    (FP8, 64, 4, 4, 32, "f16", [1, 2, 1], [700, 2, 65]),
    (FP8, 128, 32, 2, 64, "f16", [1, 1], [300, 1000]),
    (FP8, 128, 12, 4, 64, "bf16", [5, 5, 3], [5, 900, 77]),
    (FP8, 256, 4, 2, 64, "bf16", [1, 7], [333, 70]),
    (FP8, 96, 6, 3, 64, "f16", [1, 4], [200, 100]),
    (FP8, 80, 2, 1, 32, "bf16", [3], [100]),
    (FP8, 7, 2, 1, 32, "bf16", [3], [40]),
    (FP8, 128, 7, 1, 128, "bf16", [9, 1], [200, 500]),
    (FP8, 128, 4, 1, 32, "bf16", [70, 1, 33], [200, 61, 33]),
    (MXFP8, 128, 8, 2, 64, "bf16", [1, 1], [1500, 40]),
    (MXFP8, 128, 8, 2, 64, "f16", [4, 1], [150, 40]),
    (MXFP8, 64, 2, 2, 32, "bf16", [1, 20], [90, 50]),
    (MXFP8, 256, 2, 1, 32, "f16", [2], [130]),
    (MXFP8, 64, 8, 2, 32, "f16", [40, 3], [100, 90]),
    (MXFP4, 128, 8, 2, 64, "bf16", [1, 1], [1500, 40]),
    (MXFP4, 128, 8, 2, 32, "f16", [4, 1], [150, 40]),
    (MXFP4, 64, 4, 2, 32, "bf16", [1, 20], [90, 50]),
    (MXFP4, 256, 2, 1, 32, "bf16", [2], [130]),
    (MXFP4, 96, 2, 2, 256, "f16", [1, 17], [130, 60]),
    (MXFP4, 128, 8, 1, 64, "bf16", [40, 3], [100, 90]),
]


# many (query, head) columns per kv head: the chunk kernel, alone and next to short sequences
CHUNKS = [
    (FP8, 128, 8, 2, 64, "bf16", [64], [64]),
    (FP8, 128, 8, 2, 32, "bf16", [65, 1, 17, 2], [300, 1000, 17, 33]),
    (FP8, 128, 8, 1, 64, "f16", [33, 100], [700, 100]),
    (FP8, 128, 32, 2, 32, "bf16", [37], [1500]),
    (FP8, 64, 4, 4, 32, "bf16", [70, 129, 300], [71, 500, 300]),
    (FP8, 64, 8, 1, 64, "f16", [9, 40], [900, 41]),
    (FP8, 256, 4, 2, 64, "bf16", [70, 9, 3], [333, 70, 10]),
    (FP8, 96, 6, 3, 64, "f16", [90, 4], [200, 100]),
    (FP8, 80, 2, 1, 32, "bf16", [150], [151]),
    (FP8, 6, 2, 1, 32, "f16", [100], [133]),
    (MXFP8, 128, 8, 2, 64, "bf16", [100, 1], [1500, 40]),
    (MXFP8, 128, 7, 1, 32, "f16", [64, 1], [150, 40]),
    (MXFP8, 64, 2, 2, 32, "bf16", [290], [300]),
    (MXFP8, 256, 2, 1, 32, "f16", [50], [130]),
    (MXFP8, 96, 3, 1, 64, "bf16", [55], [130]),
    (MXFP4, 128, 8, 2, 64, "bf16", [100, 1], [1500, 40]),
    (MXFP4, 128, 8, 2, 32, "f16", [40, 1], [150, 40]),
    (MXFP4, 64, 4, 2, 32, "bf16", [100, 200], [100, 250]),
    (MXFP4, 256, 2, 1, 256, "bf16", [50], [130]),
    (MXFP4, 32, 8, 2, 32, "f16", [100], [600]),
]


def run_attention(cq, dev, fmt, d, hq, hkv, page, dtype, new, kv, seed=1, qscale=1.0, extra=0, **kw):
    pages = sum(-(-n // page) for n in kv) + 1
    sides = R.make_pool(cq, dev, fmt, pages, hkv, d, page, seed)
    table, cu = R.make_table(kv, page, pages, dev, seed), R.prefix(new, dev, first=extra)
    g = torch.Generator().manual_seed(seed + 1)
    q = (torch.randn(sum(new) + 2 * extra, hq, d, generator=g) * qscale).to(DTYPES[dtype])
    out = torch.full(q.shape, 77.0, dtype=q.dtype, device=dev)
    alibi = kw.pop("alibi", None)
    causal = kw.pop("causal", True)
    cq.paged_attention(q.to(dev), *sides, table, cu, R.ints(kv, dev), max(new), max(kv), R.scale_of(d),
                       causal, alibi_slopes=None if alibi is None else alibi.to(dev), out=out, **kw)
    vals = [cq.dequantize(s, page).cpu() for s in sides]
    wr = 0 if causal else kw.get("window_right", -1)
    R.assert_call(out.cpu(), q, *vals, table.cpu(), cu, kv, R.scale_of(d), DTYPES[dtype], fmt == MXFP4,
                  wl=kw.get("window_left", -1), wr=wr, softcap=kw.get("softcap", 0.0), alibi=alibi)


@pytest.mark.parametrize("fmt,d,hq,hkv,page,dtype,new,kv", ATTN)
def test_attention(cq, dev, fmt, d, hq, hkv, page, dtype, new, kv):
    run_attention(cq, dev, fmt, d, hq, hkv, page, dtype, new, kv)


@pytest.mark.parametrize("fmt,d,hq,hkv,page,dtype,new,kv", CHUNKS)
def test_attention_chunks(cq, dev, fmt, d, hq, hkv, page, dtype, new, kv):
    run_attention(cq, dev, fmt, d, hq, hkv, page, dtype, new, kv)


@pytest.mark.parametrize("fmt", [FP8, MXFP8, MXFP4])
@pytest.mark.parametrize("kw", [
    dict(window_left=40), dict(causal=False), dict(causal=False, window_left=10, window_right=5),
    dict(softcap=2.0), dict(window_left=0), dict(window_left=100, softcap=5.0)])
def test_attention_masks_and_terms(cq, dev, fmt, kw):
    run_attention(cq, dev, fmt, 128, 8, 2, 32, "bf16", [1, 6, 30, 90], [400, 77, 130, 333], **dict(kw))


@pytest.mark.parametrize("d", [64, 256])
@pytest.mark.parametrize("kw", [dict(window_left=40), dict(causal=False), dict(softcap=2.0)])
def test_attention_chunk_masks_other_head_dims(cq, dev, d, kw):
    run_attention(cq, dev, FP8, d, 4, 2, 32, "f16", [70, 100], [400, 130], **dict(kw))


@pytest.mark.parametrize("rows", [1, 2])
def test_attention_alibi(cq, dev, rows):
    slopes = torch.rand(*((2, 8) if rows == 2 else (8,)), generator=torch.Generator().manual_seed(1)) * 0.05
    run_attention(cq, dev, FP8, 128, 8, 2, 32, "bf16", [1, 60], [300, 177], alibi=slopes)


@pytest.mark.parametrize("fmt", [FP8, MXFP4])
def test_attention_peaked(cq, dev, fmt):
    """Large scores: a few keys take all the weight, and the running maximum moves often."""
    run_attention(cq, dev, fmt, 64, 4, 2, 32, "f16", [1, 6, 80], [300, 77, 300], qscale=4.0)


def test_attention_rows_outside_sequences(cq, dev):
    run_attention(cq, dev, FP8, 64, 4, 2, 32, "bf16", [1, 6, 0, 2, 80], [900, 77, 5, 2, 400], extra=3)


def test_attention_long_split(cq, dev):
    """Keys of one sequence split over the chip, next to short sequences in one split."""
    run_attention(cq, dev, FP8, 128, 4, 1, 64, "bf16", [1, 1, 2, 20], [5000, 3, 2500, 4000])


PIECES = [
    # fmt, d, hq, hkv, page, dtype, new, kv: planes that are cut into pieces, few and many of them, in calls of
    # more than 64 sequences, with empty ones, of 1 to 4 column blocks, next to chunks
    (FP8, 64, 4, 2, 32, "bf16", [1] * 70, [3000] + [1, 33, 64] * 22 + [0, 2000, 1100]),
    (MXFP4, 64, 2, 2, 32, "f16", [1] * 60 + [0] * 10 + [2] * 75, [40] * 69 + [1500, 1100, 7000] + [3] * 73),
    (MXFP8, 128, 4, 1, 64, "bf16", [9, 1, 16, 5], [5000, 1025, 1500, 5]),
    (FP8, 128, 7, 1, 64, "f16", [9, 7, 1], [4000, 1300, 2100]),
    (MXFP4, 128, 64, 8, 128, "bf16", [1, 1], [9000, 2000]),
    (FP8, 256, 4, 2, 64, "bf16", [20, 1, 32], [3000, 1500, 1100]),
    (MXFP8, 256, 2, 1, 32, "f16", [3, 0], [2500, 100]),
    (FP8, 128, 8, 2, 64, "bf16", [100, 1, 9, 0, 40], [3000, 5000, 2500, 7, 1200]),
    (FP8, 96, 3, 1, 64, "f16", [1, 6], [2500, 3300]),
]


@pytest.mark.parametrize("fmt,d,hq,hkv,page,dtype,new,kv", PIECES)
def test_attention_pieces(cq, dev, fmt, d, hq, hkv, page, dtype, new, kv):
    run_attention(cq, dev, fmt, d, hq, hkv, page, dtype, new, kv)


@pytest.mark.parametrize("kw", [dict(window_left=1500), dict(causal=False, window_left=1300, window_right=40),
                                dict(softcap=2.0)])
def test_attention_pieces_masks(cq, dev, kw):
    run_attention(cq, dev, MXFP8, 128, 8, 2, 64, "bf16", [1, 9, 1], [4000, 2500, 30], **kw)


@pytest.mark.parametrize("new,kv", [([1, 9, 30], [40, 2000, 20]), ([100, 30], [300, 20])])
def test_attention_widest_windows(cq, dev, new, kv):
    """Windows of the largest 32-bit values (also of queries in front of the first key) are no windows."""
    most = 2 ** 31 - 1
    run_attention(cq, dev, FP8, 64, 4, 2, 32, "bf16", new, kv, causal=False, window_left=most, window_right=most)
    run_attention(cq, dev, FP8, 64, 4, 2, 32, "bf16", new, kv, window_left=most)


def test_attention_workspace_of_another_device_or_alignment(cq, dev):
    sides = R.make_pool(cq, dev, FP8, 80, 2, 128, 32, 1)
    table, cu = R.make_table([2500], 32, 80, dev, 1), R.prefix([1], dev)
    q = torch.zeros(1, 8, 128, dtype=torch.bfloat16, device=dev)
    args = (q, *sides, table, cu, R.ints([2500], dev), 1, 2500, 0.1, True)
    n = cq.paged_attention_workspace_bytes(sides[0], 1, 1, 8, 1, 2500)
    for ws in (torch.zeros(n, dtype=torch.uint8), torch.zeros(n + 1, dtype=torch.uint8, device=dev)[1:],
               torch.zeros(2 * n, dtype=torch.uint8, device=dev)[::2]):
        with pytest.raises(cq.CqkvError):
            cq.paged_attention(*args, workspace=ws)


def test_attention_shared_pages(cq, dev):
    """Two sequences over the same pages, and one that holds a page twice."""
    sides = R.make_pool(cq, dev, FP8, 3, 2, 64, 32, 1)
    table = torch.tensor([[2, 0], [2, 0], [1, 1]], dtype=torch.int32, device=dev)
    cu, kv = R.prefix([1, 1, 1], dev), [50, 50, 64]
    q = torch.randn(3, 4, 64, generator=torch.Generator().manual_seed(1)).to(torch.bfloat16)
    q[1] = q[0]
    out = cq.paged_attention(q.to(dev), *sides, table, cu, R.ints(kv, dev), 1, 64, 0.125, True)
    want, mag, _ = R.attention64(q, *[cq.dequantize(s, 32).cpu() for s in sides], table.cpu(), cu, kv, 0.125)
    R.assert_attention(out, want, mag, torch.bfloat16)
    assert torch.equal(out[0], out[1])


def test_attention_holes(cq, dev):
    """Keys in pages outside the pool are masked; a sequence of holes alone gives zeros."""
    sides = R.make_pool(cq, dev, FP8, 4, 2, 64, 32, 1)
    table = torch.tensor([[2, -1, 0, 4], [-1, 4, -7, 2 ** 31 - 1]], dtype=torch.int32, device=dev)
    cu, kv = R.prefix([2, 3], dev), [110, 128]
    q = torch.randn(5, 4, 64, generator=torch.Generator().manual_seed(1)).to(torch.bfloat16)
    out = cq.paged_attention(q.to(dev), *sides, table, cu, R.ints(kv, dev), 3, 128, 0.125, True)
    want, mag, _ = R.attention64(q, *[cq.dequantize(s, 32).cpu() for s in sides], table.cpu(), cu, kv, 0.125)
    R.assert_attention(out, want, mag, torch.bfloat16)
    assert bool((out[2:] == 0).all())
    # the same holes under a chunk
    cu, n = R.prefix([50, 60], dev), 110
    q = torch.randn(n, 4, 64, generator=torch.Generator().manual_seed(1)).to(torch.bfloat16)
    out = cq.paged_attention(q.to(dev), *sides, table, cu, R.ints(kv, dev), 60, 128, 0.125, True)
    vals = [cq.dequantize(s, 32).cpu() for s in sides]
    want, mag, _ = R.attention64(q, *vals, table.cpu(), cu, kv, 0.125)
    R.assert_attention(out, want, mag, torch.bfloat16, False, True, R.score_spread(q, vals[0], 0.125))
    assert bool((out[50:] == 0).all())


def test_attention_lengths_are_clamped(cq, dev):
    """kv_lens past max_seqlen_k and past the table, negative lengths, queries past max_seqlen_q."""
    sides = R.make_pool(cq, dev, FP8, 6, 2, 64, 32, 1)
    table = torch.tensor([[2, 1], [0, 3], [4, 5]], dtype=torch.int32, device=dev)
    cu = R.prefix([2, 4, 1], dev)
    q = torch.randn(7, 4, 64, generator=torch.Generator().manual_seed(1)).to(torch.bfloat16)
    out = torch.full(q.shape, 77.0, dtype=q.dtype, device=dev)
    cq.paged_attention(q.to(dev), *sides, table, cu, R.ints([1000, 50, -3], dev), 3, 60, 0.125, True, out=out)
    want, mag, wrote = R.attention64(q, *[cq.dequantize(s, 32).cpu() for s in sides], table.cpu(), cu,
                                     [60, 50, 0], 0.125, max_q=3)
    assert bool((out[~wrote.to(dev)] == 77.0).all()) and not wrote[5]
    R.assert_attention(out[wrote.to(dev)], want[wrote], mag[wrote], torch.bfloat16)
    assert bool((out[6] == 0).all())


def poison(cq, dev, side, value, page, table, b, positions):
    """Rows of `value` at `positions` of sequence b, through the dense append; "some": ones with a NaN in
    every fourth element (an MX block of nothing but NaN has no maximum and is stored as zeros)."""
    for p in positions:
        one = view_of_page(cq, side, int(table[b, p // page]))
        row = torch.ones(1, side.kv_heads, 1, side.head_dim)
        if value == "some":
            row[..., ::4] = float("nan")
        else:
            row[:] = value
        cq.quant_append(one, row.to(torch.bfloat16).to(dev), p % page)


@pytest.mark.parametrize("fmt", [FP8, MXFP8, MXFP4])
@pytest.mark.parametrize("value", [float("nan"), float("inf"), 3e38, "some"])
@pytest.mark.parametrize("new", [1, 9, 40, 100])
def test_attention_keys_out_of_sight(cq, dev, fmt, value, new):
    """Rows that a query does not see (behind it, before its window, past the length) may hold NaN,
    infinities or the largest values: they never reach its output."""
    d, hq, hkv, page, kv, wl = 64, 4, 2, 32, 180, 70
    sides = R.make_pool(cq, dev, fmt, 6, hkv, d, page, 1)
    table, cu = R.make_table([192], page, 6, dev, 1), R.prefix([new], dev)
    q = torch.randn(new, hq, d, generator=torch.Generator().manual_seed(1)).to(torch.bfloat16)
    args = (table, cu, R.ints([kv], dev), new, kv, 0.125, True)
    clean = cq.paged_attention(q.to(dev), *sides, *args, window_left=wl)
    first = kv - new - wl  # the first query's first key
    bad = [first - 1, first - 5, kv, kv + 1, 191] + ([kv - 1] if new > 1 else [])
    for s in sides:
        poison(cq, dev, s, value, page, table, 0, bad)
    out = cq.paged_attention(q.to(dev), *sides, *args, window_left=wl)
    rows = new - 1 if new > 1 else 1  # only the last query sees the row at kv - 1
    assert torch.equal(out[:rows], clean[:rows])
    # the last query sees the row at kv - 1: NaN where it is stored as NaN (a product of a query with rows
    # of 3e38 is outside f32, so those are not looked at)
    if new > 1 and (value == "some" or value != value):
        stored, _ = R.page_rows(cq.dequantize(sides[0], page).cpu(), table.cpu(), 0, kv)
        assert bool(out[new - 1].isnan().all()) == bool(stored[kv - 1].isnan().any())
        assert not (fmt == FP8 and value != value) or bool(out[new - 1].isnan().all())


@pytest.mark.parametrize("fmt", [FP8, MXFP8])
def test_attention_visible_nan(cq, dev, fmt):
    """A NaN key or value that is seen makes the row NaN, a NaN query its own rows."""
    sides = R.make_pool(cq, dev, fmt, 4, 2, 64, 32, 1)
    table, cu = R.make_table([100], 32, 4, dev, 1), R.prefix([3], dev)
    q = torch.randn(3, 4, 64, generator=torch.Generator().manual_seed(1)).to(torch.bfloat16)
    q[1, 2] = float("nan")
    call = lambda: cq.paged_attention(q.to(dev), *sides, table, cu, R.ints([100], dev), 3, 100, 0.125, True)
    out = call()
    assert bool(out[1, 2].isnan().all())
    assert bool(out[0].isfinite().all() and out[2].isfinite().all() and out[1, [0, 1, 3]].isfinite().all())
    poison(cq, dev, sides[1], "some", 32, table, 0, [50])
    out = call()
    assert bool(out[..., ::4].isnan().all() and out[0, :, 1::4].isfinite().all())
    poison(cq, dev, sides[0], "some", 32, table, 0, [99])  # the last query's own key
    out = call()
    assert bool(out[2].isnan().all() and out[0, :, 1::4].isfinite().all())


def test_attention_arguments_from_another_stream(cq, dev):
    sides = R.make_pool(cq, dev, FP8, 40, 2, 128, 32, 1)
    table, cu = R.make_table([1200], 32, 40, dev, 1), R.prefix([1], dev)
    q = torch.randn(1, 8, 128, generator=torch.Generator().manual_seed(1)).to(torch.bfloat16).to(dev)
    args = (table, cu, R.ints([1200], dev), 1, 1200, 0.1, True)
    want = cq.paged_attention(q, *sides, *args)
    torch.cuda.synchronize()
    st = torch.cuda.Stream()
    with torch.cuda.stream(st):
        got = cq.paged_attention(q, *sides, *args)
    st.synchronize()
    assert torch.equal(got, want)


def test_attention_library_workspace_and_given_one(cq, dev):
    sides = R.make_pool(cq, dev, FP8, 80, 2, 128, 32, 1)
    table, cu = R.make_table([2500], 32, 80, dev, 1), R.prefix([1], dev)
    q = torch.randn(1, 8, 128, generator=torch.Generator().manual_seed(1)).to(torch.bfloat16).to(dev)
    n = cq.paged_attention_workspace_bytes(sides[0], 1, 1, 8, 1, 2500)
    assert n > 0
    ws = torch.full((n + 256,), 0xff, dtype=torch.uint8, device=dev)
    args = (table, cu, R.ints([2500], dev), 1, 2500, 0.1, True)
    want = cq.paged_attention(q, *sides, *args)
    assert torch.equal(cq.paged_attention(q, *sides, *args, workspace=ws[:n]), want)
    assert bool((ws[n:] == 0xff).all())
    with pytest.raises(cq.CqkvError):
        cq.paged_attention(q, *sides, *args, workspace=ws[:n - 1])


# ---------------------------------------------------------------------------------------------
# the operators together
# ---------------------------------------------------------------------------------------------
@pytest.mark.parametrize("fmt", [FP8, MXFP8, MXFP4])
def test_serving_steps(cq, dev, fmt):
    """Prompts in chunks, drafted tokens, single tokens and a rollback over one pool, q and k rotated
    on three axes: every step's output against f64 attention over the rows appended so far."""
    hq, hkv, d, page, pages = 4, 2, 64, 32, 12
    k, v = empty_pool(cq, dev, fmt, pages, hkv, d, page)
    table = torch.randperm(pages, generator=torch.Generator().manual_seed(1)).to(torch.int32).view(2, 6).to(dev)
    cos, sin = R.angle_tables(400, d, torch.bfloat16)
    axes = cq.rope_sections((8, 12, 12))
    g = torch.Generator().manual_seed(2)
    lens = [0, 0]
    for step, new in enumerate([[50, 7], [33, 1], [4, 4], [1, 1], [1, 0], [70, 1]]):
        if step == 3:
            lens = [lens[0] - 2, lens[1]]  # two drafted tokens are rejected
        total = sum(new)
        x = torch.randn(total, hq + 2 * hkv, d, generator=g).to(torch.bfloat16)
        rp = torch.cat([torch.stack([torch.arange(l, l + n) + a for a in range(3)]) for l, n in zip(lens, new)],
                       1).to(torch.int32)
        cu, starts = R.prefix(new, dev), R.ints(lens, dev)
        xd = x.to(dev)
        q = cq.paged_rope_append(k, v, xd[:, :hq], xd[:, hq:hq + hkv], xd[:, hq + hkv:], cos.to(dev),
                                 sin.to(dev), rp.to(dev), axes, table, cu, starts)
        lens = [l + n for l, n in zip(lens, new)]
        out = cq.paged_attention(q, k, v, table, cu, R.ints(lens, dev), max(new), max(lens), 0.125, True)
        vals = [cq.dequantize(s, page).cpu() for s in (k, v)]
        R.assert_call(out.cpu(), q.cpu(), *vals, table.cpu(), cu, lens, 0.125, torch.bfloat16, fmt == MXFP4)


def test_captured_step(cq, dev):
    """A decode step in a graph (append, then attention), replayed with new tokens, lengths, pages and
    eager work between the replays."""
    hq, hkv, d, page, pages, b = 8, 2, 128, 32, 80, 3
    k, v = R.make_pool(cq, dev, FP8, pages, hkv, d, page, 1)
    ke, ve = copy_side(cq, k), copy_side(cq, v)
    table = torch.randperm(pages, generator=torch.Generator().manual_seed(1))[:75].to(torch.int32).view(b, 25).to(dev)
    lens = R.ints([700, 31, 5], dev)
    pos = lens - 1
    cu = R.prefix([1] * b, dev)
    x = torch.zeros(b, hq + 2 * hkv, d, dtype=torch.bfloat16, device=dev)
    out = torch.zeros(b, hq, d, dtype=torch.bfloat16, device=dev)
    ws = torch.empty(max(1, cq.paged_attention_workspace_bytes(k, b, b, hq, 1, 800)), dtype=torch.uint8, device=dev)

    def step(k, v, out):
        cq.paged_append(k, v, x[:, hq:hq + hkv], x[:, hq + hkv:], table, cu, pos)
        cq.paged_attention(x[:, :hq], k, v, table, cu, lens, 1, 800, 0.1, True, out=out, workspace=ws)

    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        step(ke, ve, out)
    torch.cuda.current_stream().wait_stream(st)
    ke.codes.copy_(k.codes), ke.scales.copy_(k.scales), ve.codes.copy_(v.codes), ve.scales.copy_(v.scales)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step(k, v, out)
    g = torch.Generator().manual_seed(2)
    for i in range(4):
        x.copy_(torch.randn(x.shape, generator=g).to(torch.bfloat16))
        graph.replay()
        got = out.clone()
        eager = torch.zeros_like(out)
        step(ke, ve, eager)
        torch.cuda.synchronize()
        assert torch.equal(got, eager)
        assert torch.equal(k.codes, ke.codes) and torch.equal(v.scales, ve.scales)
        lens += 1
        pos += 1
        table.copy_(table.roll(1, 0) if i == 1 else table)


def test_captured_steps_share_a_workspace(cq, dev):
    """Two graphs of one workspace (a decode step of cut planes and a chunk with single tokens beside it),
    replayed in turn while lengths grow and shrink past every cut, with eager calls in between."""
    hq, hkv, d, page, pages, b, top = 8, 2, 128, 64, 140, 3, 3000
    k, v = R.make_pool(cq, dev, MXFP8, pages, hkv, d, page, 1)
    table = torch.randperm(pages, generator=torch.Generator().manual_seed(1)).to(torch.int32)
    table = torch.cat([table, table[:1]]).view(b, 47).to(dev)
    lens = R.ints([1, 1, 1], dev)
    x = torch.randn(202, hq, d, generator=torch.Generator().manual_seed(2)).to(torch.bfloat16).to(dev)
    cus = [R.prefix([1] * b, dev), R.prefix([1, 200, 1], dev)]
    most = [1, 200]
    need = [cq.paged_attention_workspace_bytes(k, b, t, hq, m, top) for t, m in ((b, 1), (202, 200))]
    assert min(need) > 0
    ws = torch.full((max(need),), 0xff, dtype=torch.uint8, device=dev)
    outs = [torch.zeros(t, hq, d, dtype=torch.bfloat16, device=dev) for t in (b, 202)]

    def step(i, out, ws):
        return cq.paged_attention(x[:out.shape[0]], k, v, table, cus[i], lens, most[i], top, 0.1, True, out=out,
                                  workspace=ws)

    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        for i in range(2):
            step(i, outs[i], ws)
    torch.cuda.current_stream().wait_stream(st)
    graphs = []
    for i in range(2):
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[i]):
            step(i, outs[i], ws)
    for n in ([2900, 1500, 3], [1, 0, 2], [3000, 2999, 2998], [70, 205, 1100], [40, 3000, 1]):
        lens.copy_(R.ints(n, dev))
        for i in (0, 1, 0):
            outs[i].fill_(7.0)
            graphs[i].replay()
            eager = step(i, torch.full_like(outs[i], 7.0), None)
            torch.cuda.synchronize()
            assert torch.equal(outs[i], eager)
            assert bool(eager.isfinite().all())


def test_two_calls_at_once(cq, dev):
    """Calls on two streams over one pool, each with the library's own workspace."""
    sides = R.make_pool(cq, dev, FP8, 160, 2, 128, 32, 1)
    g = torch.Generator().manual_seed(1)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    args, wants = [], []
    for i, n in enumerate((5000, 3100)):
        table, cu = R.make_table([n], 32, 160, dev, i), R.prefix([1], dev)
        q = torch.randn(1, 8, 128, generator=g).to(torch.bfloat16).to(dev)
        args.append((q, *sides, table, cu, R.ints([n], dev), 1, 5000, 0.1, True))
        wants.append(cq.paged_attention(*args[i]))
    torch.cuda.synchronize()
    gots = [[], []]
    for _ in range(5):
        for i, st in enumerate(streams):
            with torch.cuda.stream(st):
                gots[i].append(cq.paged_attention(*args[i]))
    torch.cuda.synchronize()
    for i in range(2):
        for got in gots[i]:
            assert torch.equal(got, wants[i])
