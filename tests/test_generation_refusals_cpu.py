"""Calls of generation that a C caller can make and that must not reach the device: null data, extents below zero."""
from pequegrad_b200 import _lib as L
from test_generation_cpu import CACHE, attend, i32, logits, read, refused, t, write

bad = L.ERR_INVALID_ARG


def test_null_data_of_logits_and_their_operands():
    f32 = lambda *s: t(s, L.F32, ptr=0)  # noqa: E731
    refused(logits(x=t((3, 100), ptr=0)), bad, b"null tensor")
    refused(logits(out=t((3, 100), ptr=0)), bad, b"null tensor")
    h = dict(history=i32(3, 9))
    refused(logits(history=i32(3, 9, ptr=0)), bad, b"history must be")
    refused(logits(**h, total=i32(3, ptr=0)), bad, b"lengths must be")
    refused(logits(**h, prompt=i32(3, ptr=0)), bad, b"lengths must be")
    for name in ("rep", "freq", "pres"):
        refused(logits(**h, **{name: f32(3)}), bad, b"penalties must be")
    refused(logits(ids=i32(3, 2, ptr=0), bias=t((3, 2), L.F32)), bad, b"[rows, entries]")
    refused(logits(ids=i32(3, 2), bias=f32(3, 2)), bad, b"[rows, entries]")
    refused(logits(mask=i32(3, 4, ptr=0)), bad, b"a bit for each")


def test_extents_below_zero():
    s = (256, 64, 1)
    refused(write(k=t((-5, 4, 64), strides=s), v=t((-5, 4, 64), strides=s)), bad, b"negative number of rows")
    refused(read(k=t((-5, 4, 64), strides=s), v=t((-5, 4, 64), strides=s)), bad, b"negative number of rows")
    refused(attend(q=t((-5, 8, 64), strides=(512, 64, 1)), out=t((-5, 8, 64), strides=(512, 64, 1))), bad, b"negative number of rows")
    for call in (write, read, attend):
        refused(call(table=i32(3, -7, strides=(7, 1))), bad, b"page table must be")
        refused(call(kc=t((-9, *CACHE[1:]), strides=(8192, 2048, 64, 1)), vc=t((-9, *CACHE[1:]), strides=(8192, 2048, 64, 1))), L.ERR_UNSUPPORTED, b"bad number of pages")
    refused(logits(x=t((-3, 100), strides=(100, 1)), out=t((-3, 100), strides=(100, 1))), bad, b"negative rows")
    refused(logits(x=t((3, -100), strides=(100, 1)), out=t((3, -100), strides=(100, 1))), bad, b"negative rows")
    refused(logits(history=i32(3, -9, strides=(9, 1))), bad, b"history must be")
    refused(logits(ids=i32(3, -2, strides=(2, 1)), bias=t((3, -2), L.F32, strides=(2, 1))), bad, b"[rows, entries]")
