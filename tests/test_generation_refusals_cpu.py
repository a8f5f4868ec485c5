"""Calls of generation that a C caller can make and that must not reach the device: null data."""
from pequegrad_b200 import _lib as L
from test_generation_cpu import i32, logits, refused, t

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
