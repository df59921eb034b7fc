"""Refusals of the page pool entry points (host checks before any launch): no GPU is needed."""
import ctypes

import pytest

BAD = 0x1000  # a non-null, 16-byte aligned pointer that is never followed


def side(cq, value=False, fmt=5, d=128, hkv=2, page=64, codes=BAD, scales=BAD, rotation=0, seed=0):
    return cq.Side(fmt, int(value), d, hkv, page, rotation, 0, 0, seed, codes, scales, None, None)


def pages(cq, batch=2, max_pages=4, n_pages=9, table=BAD, stride=4, cu=BAD):
    return cq.Pages(table, stride, cu, batch, max_pages, n_pages, 0)


def i64(*v):
    return (ctypes.c_int64 * len(v))(*v)


def append(cq, k=None, v=None, p=None, total=3, dtype=0, x=BAD, pos=BAD):
    k, v, p = k or side(cq), v or side(cq, True), p or pages(cq)
    return cq.lib().cqkv_paged_append(ctypes.byref(k), ctypes.byref(v), ctypes.byref(p), pos, x,
                                      i64(256, 128), x, i64(256, 128), dtype, total, None)


def rope(cq, k=None, v=None, p=None, total=3, dtype=0, hq=4, rows=10, kind=1, axes=3, stride=3,
         pair=None, q=BAD):
    k, v, p = k or side(cq), v or side(cq, True), p or pages(cq)
    pair = bytes(64) if pair is None else pair
    s = i64(256, 128)
    return cq.lib().cqkv_paged_rope_append(
        ctypes.byref(k), ctypes.byref(v), ctypes.byref(p), BAD, q, s, BAD, s, BAD, s, dtype, total, hq,
        BAD, BAD, rows, kind, axes, BAD, stride, pair, BAD, s, None)


def read(cq, s=None, p=None, total=3, dtype=0, out=BAD):
    s, p = s or side(cq), p or pages(cq)
    return cq.lib().cqkv_paged_dequantize(ctypes.byref(s), ctypes.byref(p), BAD, total, out, dtype,
                                          i64(256, 128), None)


def attend(cq, k=None, v=None, p=None, total=3, dtype=0, hq=4, max_q=2, max_kv=100, softcap=0.0,
           alibi=None, alibi_bs=0, q=BAD, ws=None, ws_bytes=0):
    k, v, p = k or side(cq), v or side(cq, True), p or pages(cq)
    return cq.lib().cqkv_paged_attention(
        q, i64(512, 128), dtype, ctypes.byref(k), ctypes.byref(v), ctypes.byref(p), BAD, total, hq,
        max_q, max_kv, 0.1, -1, 0, softcap, alibi, alibi_bs, BAD, i64(512, 128), ws, ws_bytes, None)


POOL_FAULTS = {
    "NVFP4 pool": lambda cq: dict(k=side(cq, fmt=3), v=side(cq, True, fmt=3)),
    "TurboQuant pool": lambda cq: dict(k=side(cq, fmt=0), v=side(cq, True, fmt=0)),
    "rotated keys": lambda cq: dict(k=side(cq, rotation=2)),
    "formats differ": lambda cq: dict(v=side(cq, True, fmt=4)),
    "head dims differ": lambda cq: dict(v=side(cq, True, d=64)),
    "heads differ": lambda cq: dict(v=side(cq, True, hkv=1)),
    "page sizes differ": lambda cq: dict(v=side(cq, True, page=32)),
    "page of 96 tokens": lambda cq: dict(k=side(cq, page=96), v=side(cq, True, page=96)),
    "page of 16 tokens": lambda cq: dict(k=side(cq, page=16), v=side(cq, True, page=16)),
    "two key sides": lambda cq: dict(v=side(cq)),
    "two value sides": lambda cq: dict(k=side(cq, True)),
    "head dim 257": lambda cq: dict(k=side(cq, d=257), v=side(cq, True, d=257)),
    "codes off a 16-byte boundary": lambda cq: dict(k=side(cq, codes=BAD + 8)),
    "scales off a 16-byte boundary": lambda cq: dict(v=side(cq, True, scales=BAD + 4)),
    "negative batch": lambda cq: dict(p=pages(cq, batch=-1)),
    "negative pages": lambda cq: dict(p=pages(cq, n_pages=-1)),
    "negative table width": lambda cq: dict(p=pages(cq, max_pages=-1)),
    "table rows overlap": lambda cq: dict(p=pages(cq, stride=3)),
    "null table": lambda cq: dict(p=pages(cq, table=None)),
    "null prefix sums": lambda cq: dict(p=pages(cq, cu=None)),
    "sequences above 2^30 tokens": lambda cq: dict(p=pages(cq, max_pages=1 << 25, stride=1 << 25)),
    "negative rows": lambda cq: dict(total=-1),
}


@pytest.mark.parametrize("call", [append, rope, attend])
@pytest.mark.parametrize("fault", POOL_FAULTS)
def test_pool_faults_are_refused(cq, call, fault):
    assert call(cq, **POOL_FAULTS[fault](cq)) == cq.ERR_ARG
    assert cq.lib().cqkv_last_error().decode().startswith("cqkv_paged_")


@pytest.mark.parametrize("fault", ["NVFP4 pool", "rotated keys", "page of 96 tokens", "null table",
                                   "codes off a 16-byte boundary", "negative rows"])
def test_read_back_faults_are_refused(cq, fault):
    kw = POOL_FAULTS[fault](cq)
    if "k" in kw:
        kw = dict(s=kw["k"])
    assert read(cq, **kw) == cq.ERR_ARG


@pytest.mark.parametrize("call,kw", [
    (append, dict(dtype=3)), (append, dict(x=None)), (append, dict(pos=None)),
    (append, dict(total=(1 << 28) + 1)),
    (rope, dict(dtype=-1)), (rope, dict(hq=0)), (rope, dict(rows=0)), (rope, dict(kind=0)),
    (rope, dict(axes=0)), (rope, dict(axes=5)), (rope, dict(pair=bytes([3] * 64))),
    (rope, dict(stride=2)), (rope, dict(q=None)),
    (read, dict(dtype=3)), (read, dict(out=None)),
    (attend, dict(dtype=2)), (attend, dict(hq=3)), (attend, dict(hq=0)), (attend, dict(max_q=-1)),
    (attend, dict(max_kv=-1)), (attend, dict(softcap=float("inf"))), (attend, dict(softcap=-1.0)),
    (attend, dict(alibi=BAD, alibi_bs=3)), (attend, dict(q=None)),
    (attend, dict(max_q=1 << 24, hq=8)),
])
def test_call_faults_are_refused(cq, call, kw):
    assert call(cq, **kw) == cq.ERR_ARG


def test_odd_head_dims_have_no_rotary_pairs(cq):
    assert rope(cq, k=side(cq, d=5), v=side(cq, True, d=5)) == cq.ERR_ARG


def test_small_workspace_is_refused(cq):
    k = side(cq)
    need = cq.lib().cqkv_paged_attention_workspace_bytes(ctypes.byref(k), 1, 1, 4, 1, 4096, -1, 0)
    assert need > 0
    p = pages(cq, batch=1, max_pages=64, stride=64)
    assert attend(cq, p=p, total=1, max_q=1, max_kv=4096, ws=BAD, ws_bytes=need - 1) == cq.ERR_WORKSPACE


def test_misaligned_workspace_is_refused(cq):
    need = cq.lib().cqkv_paged_attention_workspace_bytes(ctypes.byref(side(cq)), 1, 1, 4, 1, 4096, -1, 0)
    p = pages(cq, batch=1, max_pages=64, stride=64)
    assert attend(cq, p=p, total=1, max_q=1, max_kv=4096, ws=BAD + 8, ws_bytes=need + 8) == cq.ERR_ARG


@pytest.mark.parametrize("call", [append, rope, read, attend])
def test_nothing_to_do(cq, call):
    """No rows, or no sequences: the arguments are checked, nothing is launched."""
    assert call(cq, total=0) == cq.OK
    assert call(cq, p=pages(cq, batch=0, table=None, cu=None)) == cq.OK


def test_front_end_refuses_cpu_pools(cq):
    import torch
    s = cq.CacheSide.empty(cq.FP8, False, 2, 2, 64, 32, "cpu")
    v = cq.CacheSide.empty(cq.FP8, True, 2, 2, 64, 32, "cpu")
    x = torch.zeros(1, 2, 64, dtype=torch.bfloat16)
    t, cu, one = torch.zeros(1, 1, dtype=torch.int32), torch.tensor([0, 1], dtype=torch.int32), \
        torch.zeros(1, dtype=torch.int32)
    for f in (lambda: cq.paged_append(s, v, x, x, t, cu, one),
              lambda: cq.paged_dequantize(s, t, cu, one, 1),
              lambda: cq.paged_attention(x, s, v, t, cu, one, 1, 1, 0.1, True)):
        with pytest.raises(cq.CqkvError):
            f()


def test_rope_sections(cq):
    assert list(cq.rope_sections((2, 1, 3))) == [0, 0, 1, 2, 2, 2]
