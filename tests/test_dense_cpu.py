"""What needs no device: the refusals of the norm, quantizer, product and log-probability entry
points. Every refused call fails before it touches its context, so a block of zeroed memory stands
for one."""
import ctypes as C

import pytest

from objeta_amd import DenseBackend, _lib

INVALID = 5
A, B, D, E, F, G, H = (0x10000000 * i for i in range(1, 8))  # addresses far apart; never read


@pytest.fixture
def lib():
    return _lib.load()


@pytest.fixture
def ctx():
    return (C.c_uint64 * 1024)()


def refused(lib, status, text):
    rec = _lib.Error()
    lib.objeta_hip_last_error(C.byref(rec))
    assert status == INVALID, (status, rec.source_message)
    assert text.encode() in rec.source_message, rec.source_message


def call_norm(lib, ctx, **kw):
    a = dict(n=4, hidden=256, dtype=0, x=A, xs=256, wt=0, w=B, offset=0.0, eps=1e-6, rt=0, r=D, rs=256, ro=E, ros=256, ot=0, o=F,
             os=256, codes=1, q=G, qs=256, s=H)
    a.update(kw)
    return lib.objeta_hip_rms_norm_device(C.cast(ctx, C.c_void_p), None, *a.values())


@pytest.mark.parametrize("kw,text", [
    ({"hidden": 0}, "hidden"), ({"hidden": 32769}, "hidden"), ({"dtype": 3}, "dtype"), ({"wt": 9}, "dtype"), ({"rt": 3}, "residual dtype"),
    ({"ot": -1}, "out dtype"), ({"codes": 3}, "unknown codes"), ({"codes": -1}, "unknown codes"), ({"codes": 2, "hidden": 200}, "multiple of 128"),
    ({"eps": -1e-9}, "eps"), ({"eps": float("nan")}, "eps"), ({"eps": float("inf")}, "eps"), ({"offset": float("nan")}, "offset"),
    ({"n": 1 << 31}, "too many tokens"), ({"o": None, "ro": None, "codes": 0}, "no output"), ({"x": None}, "x is NULL"),
    ({"w": None}, "weight is NULL"), ({"x": A + 2}, "not aligned"), ({"xs": 255}, "stride"), ({"rs": 255}, "stride"),
    ({"os": 255}, "stride"), ({"qs": 255}, "stride"), ({"xs": 1 << 31}, "stride"), ({"q": None}, "codes is NULL"),
    ({"s": None}, "scales is NULL"), ({"s": H + 2}, "not aligned"), ({"ro": D + 4}, "residual out overlaps"),
    ({"ro": D, "ros": 512}, "residual out overlaps"), ({"ro": A}, "residual out overlaps"), ({"ro": B + 16}, "residual out overlaps"),
    ({"o": D}, "out overlaps"), ({"o": E}, "out overlaps"), ({"o": A, "ot": 1}, "out overlaps"), ({"o": A + 4}, "out overlaps"),
    ({"q": A}, "codes overlaps"), ({"q": F + 3}, "codes overlaps"), ({"s": G + 4}, "scales overlaps"), ({"s": B}, "scales overlaps"),
])
def test_rms_norm_refuses(lib, ctx, kw, text):
    refused(lib, call_norm(lib, ctx, **kw), text)


def call_quantize(lib, ctx, **kw):
    a = dict(n=4, cols=256, dtype=0, x=A, xs=256, q=B, qs=256, s=D)
    a.update(kw)
    return lib.objeta_hip_quantize_rows_i8_device(C.cast(ctx, C.c_void_p), None, *a.values())


@pytest.mark.parametrize("kw,text", [
    ({"cols": 0}, "cols"), ({"cols": 65537}, "cols"), ({"dtype": 5}, "dtype"), ({"n": 1 << 31}, "too many rows"), ({"x": None}, "x is NULL"),
    ({"q": None}, "codes is NULL"), ({"s": None}, "scales is NULL"), ({"x": A + 1, "dtype": 1}, "not aligned"), ({"xs": 200}, "stride"),
    ({"qs": 200}, "stride"), ({"q": A + 256}, "codes overlaps"), ({"s": A + 1024}, "scales overlaps"), ({"s": B + 4}, "scales overlaps"),
])
def test_quantize_rows_refuses(lib, ctx, kw, text):
    refused(lib, call_quantize(lib, ctx, **kw), text)


def call_product(lib, ctx, **kw):
    a = dict(n=4, rows=64, cols=256, a=A, as_=256, sa=B, w=D, ws=256, sw=E, bias=F, ot=0, o=G, os=64)
    a.update(kw)
    return lib.objeta_hip_i8_product_device(C.cast(ctx, C.c_void_p), None, *a.values())


@pytest.mark.parametrize("kw,text", [
    ({"cols": 0}, "cols"), ({"cols": 131072}, "cols"), ({"rows": 1 << 24}, "too many rows"), ({"n": 1 << 20}, "too many tokens"),
    ({"ot": 4}, "dtype"), ({"a": None}, "a is NULL"), ({"w": None}, "w is NULL"), ({"sa": None}, "a scales is NULL"),
    ({"sw": None}, "w scales is NULL"), ({"o": None}, "out is NULL"), ({"sa": B + 1}, "not aligned"), ({"bias": F + 2}, "not aligned"),
    ({"o": G + 2}, "not aligned"), ({"as_": 255}, "stride"), ({"ws": 255}, "stride"), ({"os": 63}, "stride"), ({"o": A}, "out overlaps"),
    ({"o": D + 64}, "out overlaps"), ({"o": B}, "out overlaps"), ({"o": E + 4}, "out overlaps"), ({"o": F + 8}, "out overlaps"),
])
def test_product_refuses(lib, ctx, kw, text):
    refused(lib, call_product(lib, ctx, **kw), text)


def call_log_probs(lib, ctx, **kw):
    a = dict(n=4, vocab=1000, dtype=0, x=A, stride=1000, scale=1.0, tokens=B, given=2, lp=D, lse=E, entropy=F, top=3, ids=G, tops=H)
    a.update(kw)
    return lib.objeta_hip_log_probs_device(C.cast(ctx, C.c_void_p), None, *a.values())


@pytest.mark.parametrize("kw,text", [
    ({"vocab": 0}, "vocab"), ({"vocab": (1 << 31) - 1}, "vocab"), ({"dtype": 7}, "dtype"), ({"scale": 0.0}, "scale"), ({"scale": -1.0}, "scale"),
    ({"scale": float("nan")}, "scale"), ({"scale": float("inf")}, "scale"), ({"given": 1025}, "given"), ({"given": 0}, "come together"),
    ({"tokens": None}, "come together"), ({"lp": None}, "come together"), ({"top": 33}, "n_top"), ({"top": 3, "vocab": 2}, "n_top"),
    ({"ids": None}, "top ids"), ({"top": 0}, "n_top 0"), ({"n": 1 << 31}, "too many rows"), ({"x": None}, "logits is NULL"),
    ({"x": A + 2}, "not aligned"), ({"stride": 999}, "stride"), ({"lp": D + 1}, "not aligned"), ({"lse": E + 2}, "not aligned"),
    ({"lse": A + 400}, "overlaps"), ({"entropy": E + 4}, "overlaps"), ({"lp": B}, "overlaps"), ({"ids": H}, "overlaps"),
    ({"tokens": None, "given": 0, "lp": None, "lse": None, "entropy": None, "top": 0, "ids": None, "tops": None}, "no output"),
])
def test_log_probs_refuses(lib, ctx, kw, text):
    refused(lib, call_log_probs(lib, ctx, **kw), text)


def test_calls_with_nothing_to_do_succeed(lib, ctx):
    assert call_norm(lib, ctx, n=0) == 0 and call_quantize(lib, ctx, n=0) == 0
    assert call_product(lib, ctx, n=0) == 0 and call_product(lib, ctx, rows=0, os=0) == 0 and call_log_probs(lib, ctx, n=0) == 0


def test_a_null_context_is_refused(lib):
    refused(lib, call_norm(lib, None), "context is NULL")
    refused(lib, call_product(lib, None), "context is NULL")
    refused(lib, call_log_probs(lib, None), "context is NULL")
    refused(lib, call_quantize(lib, None), "context is NULL")


def test_names_are_refused(lib):
    class Stub:
        L, ctx = lib, None
    d = DenseBackend(Stub())
    with pytest.raises(ValueError):
        d.rms_norm_device(1, 8, "f64", A, B, d_out=D)
    with pytest.raises(ValueError):
        d.rms_norm_device(1, 8, "f32", A, B, codes="int4", d_codes=D, d_scales=E)
    with pytest.raises(ValueError):
        d.log_probs_device(1, 8, "i8", A, d_lse=B)
