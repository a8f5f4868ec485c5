"""The entry points of generation without a GPU: what they refuse, and that a call they accept asks for a device."""
import ctypes as C

import pytest
import torch

from pequegrad_b200 import _lib as L
from pequegrad_b200 import kernels as K

ES = {L.F16: 2, L.BF16: 2, L.F32: 4, L.I8: 1, L.I32: 4, L.F64: 8}


def t(shape, dtype=L.F16, strides=None, ptr=4096):
    if strides is None:
        strides, acc = [], 1
        for s in reversed(shape):
            strides.insert(0, acc)
            acc *= s
    return L.pack_tensor(ptr, dtype, shape, [s * ES[dtype] for s in strides])


def i32(*shape, **kw):
    return t(shape, L.I32, **kw)


CACHE = (9, 4, 32, 64)
BASE = dict(k=t((5, 4, 64)), v=t((5, 4, 64)), kc=t(CACHE), vc=t(CACHE), ks=None, vs=None, start=i32(4), ctx=i32(3), table=i32(3, 7))
INT8 = dict(kc=t(CACHE, L.I8), vc=t(CACHE, L.I8), ks=t(CACHE[:3], L.F32), vs=t(CACHE[:3], L.F32))

needs_no_device = pytest.mark.skipif(torch.cuda.is_available(), reason="the accepted call would run")


def write(**kw):
    a = {**BASE, **kw}
    return L.lib().pgb_kv_write(a["k"], a["v"], a["kc"], a["vc"], a["ks"], a["vs"], a["start"], a["ctx"], a["table"], None)


def read(**kw):
    a = {**BASE, **kw}
    return L.lib().pgb_kv_read(a["kc"], a["vc"], a["ks"], a["vs"], a["start"], a["table"], a["k"], a["v"], None)


def attend(scale=0.125, **kw):
    a = {**BASE, "q": t((5, 8, 64)), "out": t((5, 8, 64)), **kw}
    return L.lib().pgb_paged_attention(a["q"], a["kc"], a["vc"], a["ks"], a["vs"], a["start"], a["ctx"], a["table"], scale, a["out"], None)


def refused(status, code, text):
    msg = L.lib().pgb_last_error()
    assert status == code and text in msg, (status, msg)


def test_packed_descriptors_are_the_structures_bytes():
    for shape, strides in [((), ()), ((3,), (4,)), ((2, 3, 4, 64), (1 << 40, 512, 128, 2)), ((1,) * 8, (16,) * 8)]:
        assert L.pack_tensor(1 << 45, L.BF16, shape, strides) == bytes(L.make_tensor(1 << 45, L.BF16, shape, strides))
    assert C.sizeof(L.PgbTensor) == len(L.pack_tensor(0, 0, (), ()))
    with pytest.raises(ValueError):
        L.pack_tensor(0, 0, (1,) * 9, (1,) * 9)


@needs_no_device
def test_accepted_calls_ask_for_a_device():
    for st in (write(), read(), attend(), write(**INT8), read(**INT8), attend(**INT8), read(**INT8, k=t((5, 4, 64), L.F32), v=t((5, 4, 64), L.F32)),
               write(kc=t(CACHE, strides=(32 * 256, 64, 256, 1)), vc=t(CACHE)), attend(q=t((0, 8, 64)), out=t((0, 8, 64)))):
        refused(st, L.ERR_CUDA, b"no CPU fallback")
    with pytest.raises(RuntimeError, match="CUDA tensors"):
        K.kv_write(*[torch.zeros(1)] * 7)
    with pytest.raises(RuntimeError, match="CUDA tensors"):
        K.logits_process(torch.zeros(2, 8))


@pytest.mark.parametrize("call", [write, read, attend])
def test_caches_and_plans_that_are_refused(call):
    bad, no = L.ERR_INVALID_ARG, L.ERR_UNSUPPORTED
    refused(call(kc=None), bad, b"null cache")
    refused(call(kc=t((9, 4, 32))), bad, b"a cache is [pages")
    refused(call(vc=t((9, 4, 16, 64))), bad, b"differ in shape")
    refused(call(vc=t(CACHE, L.BF16)), bad, b"differ in dtype")
    refused(call(kc=t(CACHE, L.F32), vc=t(CACHE, L.F32)), no, b"not implemented for a cache of float32")
    refused(call(ks=INT8["ks"], vs=INT8["vs"]), bad, b"only an int8 cache has scales")
    refused(call(kc=INT8["kc"], vc=INT8["vc"]), bad, b"needs k_scale and v_scale")
    refused(call(**{**INT8, "vs": None}), bad, b"needs k_scale and v_scale")
    refused(call(**{**INT8, "ks": t((9, 4, 16), L.F32)}), bad, b"the scales must be")
    refused(call(**{**INT8, "ks": t(CACHE[:3], L.F16)}), bad, b"the scales must be")
    refused(call(**{**INT8, "ks": t(CACHE[:3], L.F32, strides=(128, 1, 4))}), no, b"contiguous and 16-byte")
    for D in (32, 80, 96, 256):
        refused(call(kc=t((9, 4, 32, D)), vc=t((9, 4, 32, D))), no, b"head dims of 64 and 128")
    for P in (1, 8, 24, 48, 256):
        refused(call(kc=t((9, 4, P, 64)), vc=t((9, 4, P, 64))), no, b"page size")
    refused(call(kc=t(CACHE, ptr=4104)), no, b"16-byte aligned")
    refused(call(kc=t(CACHE, strides=(32 * 260, 65, 260, 1))), no, b"multiples of 16 bytes")
    refused(call(vc=t(CACHE, strides=(8192, 2048, 1, 32))), bad, b"must be contiguous")
    refused(call(kc=t(CACHE, ptr=0)), bad, b"null cache")
    refused(call(start=None), bad, b"null plan")
    refused(call(table=None), bad, b"null plan")
    refused(call(table=t((3, 7), L.F32)), bad, b"must be int32")
    refused(call(start=i32(4, 1)), bad, b"row offsets")
    refused(call(start=i32(0)), bad, b"row offsets")
    refused(call(start=i32(4, strides=(2,))), bad, b"row offsets")
    refused(call(table=i32(4, 7)), bad, b"page table must be")
    refused(call(table=i32(3, 7, strides=(1, 3))), bad, b"must be contiguous")
    refused(call(start=i32(4, ptr=4098)), bad, b"4-byte aligned")
    if call is not read:
        refused(call(ctx=None), bad, b"null plan")
        refused(call(ctx=i32(4)), bad, b"the lengths must be")
        refused(call(ctx=t((3,), L.F32)), bad, b"must be int32")


def test_rows_that_are_refused():
    bad, no = L.ERR_INVALID_ARG, L.ERR_UNSUPPORTED
    for call in (write, read):
        refused(call(k=t((5, 2, 64))), bad, b"with the heads and head dim of the cache")
        refused(call(k=t((5, 4, 128))), bad, b"with the heads and head dim of the cache")
        refused(call(v=t((6, 4, 64))), bad, b"differ in rows")
        refused(call(k=t((5, 4, 64), strides=(256, 1, 4))), bad, b"must be contiguous")
        refused(call(k=t((5, 4, 64), ptr=4100)), no, b"16-byte aligned")
        refused(call(v=t((5, 4, 64), strides=(260, 64, 1))), no, b"multiples of 16 bytes")
        refused(call(k=t((5, 4, 64), L.BF16), v=t((5, 4, 64), L.BF16)), bad, b"dtype")
        refused(call(k=None), bad, b"")
    refused(write(k=t((5, 4, 64), L.F32), v=t((5, 4, 64), L.F32)), bad, b"float16")
    refused(write(kc=t(CACHE, strides=(8192, 0, 64, 1))), bad, b"overlaps itself")
    refused(read(k=t((5, 4, 64), strides=(0, 64, 1))), bad, b"overlaps itself")
    refused(read(**INT8, k=t((5, 4, 64), L.I8), v=t((5, 4, 64), L.I8)), bad, b"is read as")
    refused(attend(q=t((5, 6, 64)), out=t((5, 6, 64))), bad, b"a multiple of the cache's")
    refused(attend(q=t((5, 8, 64), L.F32)), no, b"paged_attention not implemented for float32")
    refused(attend(out=t((5, 8, 64), L.BF16)), bad, b"one dtype")
    refused(attend(q=t((5, 8, 64), L.BF16), out=t((5, 8, 64), L.BF16)), bad, b"one dtype")
    refused(attend(out=t((6, 8, 64))), bad, b"differ in rows")
    refused(attend(out=t((5, 8, 64), strides=(0, 64, 1))), bad, b"overlaps itself")
    refused(attend(q=t((5, 8, 64), ptr=4098)), no, b"16-byte aligned")
    refused(attend(q=None), bad, b"null")
    for s in (0.0, -1.0, float("nan"), float("inf")):
        refused(attend(scale=s), bad, b"positive and finite")


def logits(**kw):
    a = dict(x=t((3, 100)), history=None, total=None, prompt=None, rep=None, freq=None, pres=None, ids=None, bias=None, mask=None, out=t((3, 100)))
    a.update(kw)
    return L.lib().pgb_logits_process(*[a[n] for n in ("x", "history", "total", "prompt", "rep", "freq", "pres", "ids", "bias", "mask", "out")], None)


@needs_no_device
def test_accepted_logit_calls_ask_for_a_device():
    for kw in (dict(), dict(mask=i32(3, 4)), dict(history=i32(3, 9), total=i32(3), rep=t((3,), L.F32)), dict(ids=i32(3, 2), bias=t((3, 2), L.F32))):
        refused(logits(**kw), L.ERR_CUDA, b"no CPU fallback")


def test_logit_calls_that_are_refused():
    bad, no = L.ERR_INVALID_ARG, L.ERR_UNSUPPORTED
    f32 = lambda *s: t(s, L.F32)  # noqa: E731
    refused(logits(x=None), bad, b"null tensor")
    refused(logits(x=t((3, 100), L.F64), out=t((3, 100), L.F64)), no, b"not implemented for float64")
    refused(logits(out=t((3, 101))), bad, b"one dtype")
    refused(logits(out=t((3, 100), L.F32)), bad, b"one dtype")
    refused(logits(x=t((300,))), bad, b"one dtype")
    refused(logits(x=t((3, 100), strides=(1, 3))), bad, b"must be contiguous")
    refused(logits(out=t((3, 100), strides=(50, 1))), bad, b"overlaps itself")
    refused(logits(x=t((70000, 8)), out=t((70000, 8))), no, b"too many rows")
    for kw in (dict(total=i32(3)), dict(prompt=i32(3)), dict(rep=f32(3)), dict(freq=f32(3)), dict(pres=f32(3))):
        refused(logits(**kw), bad, b"need a history")
    h = dict(history=i32(3, 9))
    refused(logits(history=i32(2, 9)), bad, b"history must be")
    refused(logits(history=f32(3, 9)), bad, b"history must be")
    refused(logits(history=i32(3, 9, strides=(1, 3))), bad, b"history must be")
    refused(logits(**h, total=i32(2)), bad, b"lengths must be")
    refused(logits(**h, total=i32(3, strides=(2,))), bad, b"lengths must be")
    refused(logits(**h, rep=i32(3)), bad, b"penalties must be")
    refused(logits(**h, freq=f32(3, 1)), bad, b"penalties must be")
    refused(logits(ids=i32(3, 2)), bad, b"come together")
    refused(logits(ids=i32(3, 2), bias=f32(3, 3)), bad, b"[rows, entries]")
    refused(logits(ids=f32(3, 2), bias=f32(3, 2)), bad, b"[rows, entries]")
    refused(logits(mask=i32(3, 3)), bad, b"a bit for each")
    refused(logits(mask=f32(3, 4)), bad, b"a bit for each")


# ---- which sequence holds which page ------------------------------------------------------------------------------------

def cache(pages, page_size=16, dtype=torch.float16):
    from pequegrad_b200.kvcache import PagedKVCache
    return PagedKVCache(2, 3, 64, pages, page_size, dtype, device="cpu")


def test_plans_of_a_cache():
    c = cache(8)
    a, b = c.open(), c.open()
    p = c.extend([a, b], [20, 16])
    assert p.rows == 36 and p.longest == 20
    assert p.q_start.tolist() == [0, 20, 36] and p.ctx_len.tolist() == [20, 16] and p.last.tolist() == [19, 35]
    assert p.positions.tolist() == list(range(20)) + list(range(16))
    assert p.page_table.shape == (2, 2) and p.page_table[1, 1] == -1
    first = p.page_table[0].tolist()
    used = set(first) | {int(p.page_table[1, 0])}
    assert len(used) == 3 and c.free_pages() == 5
    p = c.extend([b, a], [1, 1])  # in any order; b enters a new page, a does not
    assert p.ctx_len.tolist() == [17, 21] and p.positions.tolist() == [16, 20] and p.last.tolist() == [0, 1]
    assert p.page_table[1].tolist() == first and c.free_pages() == 4
    assert not set(p.page_table[0].tolist()) & set(first)
    c.close(b)
    assert c.free_pages() == 6 and c.length(a) == 21
    p = c.extend([a], [0])
    assert p.rows == 0 and p.q_start.tolist() == [0, 0] and p.ctx_len.tolist() == [21]
    assert c.extend([], []).page_table.shape == (0, 0)


def test_a_cache_that_is_full_changes_nothing():
    c = cache(3)
    a, b = c.open(), c.open()
    c.extend([a], [33])
    with pytest.raises(RuntimeError, match="1 pages are needed and 0 are free"):
        c.extend([a, b], [1, 1])
    assert c.length(a) == 33 and c.length(b) == 0 and c.free_pages() == 0
    c.extend([a], [15])
    with pytest.raises(ValueError, match="each sequence once"):
        c.extend([a, a], [1, 1])
    with pytest.raises(ValueError, match="each sequence once"):
        c.extend([a], [-1])
    with pytest.raises(KeyError):
        c.close(99)
    c.close(a)
    with pytest.raises(KeyError):
        c.extend([a], [1])


def test_an_int8_cache_has_scales_and_a_16_bit_cache_has_none():
    assert cache(4).k_scale is None
    c = cache(4, 32, torch.int8)
    assert c.k.shape == (2, 4, 3, 32, 64) and c.v_scale.shape == (2, 4, 3, 32) and c.v_scale.dtype == torch.float32
