"""What needs no device: the rotary plan against its formulas, and the refusals of the
attention entry points. Every refused call fails before it touches its context, so a block
of zeroed memory stands for one."""
import ctypes as C

import numpy as np
import pytest

from attn_reference import frequencies
from objeta_amd import HipError, KvCache, Rope, _lib
from objeta_amd._lib import KvCacheDesc, RopePlan

INVALID, UNSUPPORTED = 5, 6


@pytest.mark.parametrize("scaling,kw", [("none", {}), ("linear", {"factor": 8.0}), ("ntk", {"factor": 4.0}),
                                        ("yarn", {"factor": 32.0, "original": 4096}),
                                        ("yarn", {"factor": 4.0, "original": 32768, "fast": 16.0, "slow": 2.0})])
@pytest.mark.parametrize("rotary,theta", [(2, 10000.0), (64, 10000.0), (128, 1e6), (250, 500000.0)])
def test_turns_follow_the_formulas(rotary, theta, scaling, kw):
    names = {"original": "original_context", "fast": "beta_fast", "slow": "beta_slow"}
    r = Rope(rotary, theta=theta, scaling=scaling, **{names.get(k, k): v for k, v in kw.items()})
    want = frequencies(rotary, theta, scaling, **kw) / (2 * np.pi)
    got = r.turns().astype(np.longdouble) / np.longdouble(2) ** 64
    # half a unit of the 64-bit fraction, and the doubles' powers and logarithms: their arguments'
    # roundings times at most ln theta (14), about 50 half steps of 2^-53
    assert np.all(np.abs(got - want) <= 2.0 ** -65 + 1e-14 * want)
    assert r.plan.amplitude == np.float32(0.1 * np.log(kw["factor"]) + 1 if scaling == "yarn" else 1)


def test_a_given_amplitude_is_taken():
    assert Rope(64, scaling="yarn", factor=4.0, amplitude=1.25).plan.amplitude == np.float32(1.25)
    assert Rope(64, amplitude=0.5).plan.amplitude == np.float32(0.5)


@pytest.mark.parametrize("kw", [{"rotary_dim": 0}, {"rotary_dim": 3}, {"rotary_dim": 258}, {"rotary_dim": 64, "theta": 0.0},
                                {"rotary_dim": 64, "theta": float("nan")}, {"rotary_dim": 64, "scaling": "linear", "factor": 0.0},
                                {"rotary_dim": 64, "scaling": "yarn", "factor": 0.5},
                                {"rotary_dim": 64, "scaling": "yarn", "factor": 2.0, "original_context": 0},
                                {"rotary_dim": 64, "scaling": "yarn", "factor": 2.0, "beta_fast": 1.0, "beta_slow": 1.0},
                                {"rotary_dim": 64, "scaling": "ntk", "factor": float("inf")},
                                {"rotary_dim": 64, "amplitude": -1.0}])
def test_rope_refuses(kw):
    with pytest.raises(HipError) as e:
        Rope(**kw)
    assert e.value.kind == "InvalidInput"


@pytest.mark.parametrize("kw", [{"layout": "pairs"}, {"scaling": "dynamic"}, {"amplitude": 0.0}])
def test_rope_refuses_names(kw):
    with pytest.raises(ValueError):
        Rope(64, **kw)


@pytest.fixture
def lib():
    return _lib.load()


@pytest.fixture
def ctx():
    return (C.c_uint64 * 1024)()


def addr(x):
    return C.cast(x, C.c_void_p)


A, B, D, E, F = (0x10000000 * i for i in range(1, 6))  # addresses far apart; never read


def plan(rotary=64, layout=1):
    p = RopePlan()
    p.rotary_dim, p.layout, p.amplitude = rotary, layout, 1.0
    return p


def refused(lib, status, want, text=""):
    rec = _lib.Error()
    lib.objeta_hip_last_error(C.byref(rec))
    assert status == want, (status, rec.source_message)
    assert text.encode() in rec.source_message, rec.source_message


def call_rope(lib, ctx, **kw):
    a = dict(rope=plan(), pos=F, n=4, dim=64, dtype=0, out=0, q=A, qs=512, qo=B, qos=512, nq=8, k=D, ks=128, ko=E, kos=128,
             nk=2)
    a.update(kw)
    return lib.objeta_hip_rope_device(addr(ctx), None, C.byref(a["rope"]) if a["rope"] else None, a["pos"], a["n"], a["dim"],
                                      a["dtype"], a["out"], a["q"], a["qs"], a["qo"], a["qos"], a["nq"], a["k"], a["ks"],
                                      a["ko"], a["kos"], a["nk"])


@pytest.mark.parametrize("kw,text", [
    ({"rope": None}, "rope is NULL"), ({"rope": plan(128)}, "exceeds head_dim"), ({"rope": plan(64, 7)}, "layout"),
    ({"rope": plan(0)}, "rotary_dim"), ({"rope": plan(63)}, "rotary_dim"), ({"dim": 260}, "head_dim"), ({"dim": 60}, "head_dim"),
    ({"dim": 264}, "head_dim"), ({"dtype": 3}, "dtype"), ({"out": 8}, "dtype"), ({"nq": 0}, "n_q_heads"), ({"pos": None}, "positions"),
    ({"q": None}, "q is NULL"), ({"qo": None}, "q_out is NULL"), ({"ko": None}, "k_out is NULL"), ({"q": A + 2}, "not aligned"),
    ({"qs": 511}, "stride"), ({"kos": 127}, "stride"), ({"n": 1 << 31}, "too many tokens"),
    ({"qo": A + 4}, "overlaps its input"), ({"qo": A, "qos": 1024}, "overlaps its input"), ({"qo": A, "out": 2}, "overlaps its input"),
    ({"qo": D}, "overlaps another"), ({"ko": B}, "overlaps another"), ({"ko": A + 64}, "overlaps another"),
])
def test_rope_device_refuses(lib, ctx, kw, text):
    refused(lib, call_rope(lib, ctx, **kw), INVALID, text)


def test_calls_with_nothing_to_do_succeed(lib, ctx):
    assert call_rope(lib, ctx, n=0) == 0
    assert call_prompt(lib, ctx, n=0) == 0 and call_prompt(lib, ctx, seqs=0) == 0
    assert call_cached(lib, ctx, rows=0) == 0 and call_cached(lib, ctx, batch=0) == 0
    assert call_append(lib, ctx, rows=0) == 0
    c = cache()
    assert lib.objeta_hip_kv_free_device(addr(ctx), None, C.byref(c), None, 0) == 0


def test_in_place_and_packed_columns_are_no_overlap(lib, ctx):
    """In place, and q, k and their outputs as columns of one packed buffer: these pass the checks
    and fail only for want of a device (a driver error)."""
    if lib.objeta_hip_device_count(C.byref(C.c_int32())) == 0:
        pytest.skip("a device is here: the call would run on made-up addresses")
    for kw in ({"qo": A, "ko": D}, {"q": A, "qs": 1280, "qo": A, "qos": 1280, "k": A + 2048, "ks": 1280, "ko": A + 2048, "kos": 1280}):
        refused(lib, call_rope(lib, ctx, **kw), 1)


def call_prompt(lib, ctx, **kw):
    a = dict(dtype=2, q=A, qs=512, nq=8, k=B, ks=128, v=D, vs=128, nk=2, dim=64, n=4, cu=F, seqs=1, scale=0.125, out=E, os=512,
             lse=None)
    a.update(kw)
    return lib.objeta_hip_attn_prompt_device(addr(ctx), None, a["dtype"], a["q"], a["qs"], a["nq"], a["k"], a["ks"], a["v"],
                                             a["vs"], a["nk"], a["dim"], a["n"], a["cu"], a["seqs"], 1, a["scale"], a["out"],
                                             a["os"], a["lse"])


@pytest.mark.parametrize("kw,text", [
    ({"dtype": 4}, "dtype"), ({"dim": 12}, "head_dim"), ({"dim": 512}, "head_dim"), ({"nq": 7}, "multiple of n_kv_heads"),
    ({"nk": 0}, "multiple"), ({"nq": 0}, "multiple"), ({"n": 1 << 29}, "2^31"), ({"n": 1 << 40}, "2^31"), ({"scale": 0.0}, "scale"),
    ({"scale": -1.0}, "scale"), ({"scale": float("nan")}, "scale"), ({"scale": float("inf")}, "scale"), ({"cu": None}, "cu_seqlens"),
    ({"q": None}, "q is NULL"), ({"v": None}, "v is NULL"), ({"out": None}, "out is NULL"), ({"k": B + 8}, "16-byte"),
    ({"vs": 132}, "16-byte"), ({"qs": 504}, "stride"), ({"out": A}, "overlaps"), ({"out": D}, "overlaps"), ({"lse": E}, "overlaps"),
    ({"lse": A}, "overlaps"), ({"lse": F + 2}, "lse"),
])
def test_prompt_refuses(lib, ctx, kw, text):
    refused(lib, call_prompt(lib, ctx, **kw), INVALID, text)


def test_prompt_refuses_most_rows(lib, ctx):
    """A key's index and a tile's keys add up in 32 bits: some room is left below 2^31."""
    refused(lib, call_prompt(lib, ctx, n=0x7FFF0000 // 8 + 1), INVALID, "2^31")
    refused(lib, call_cached(lib, ctx, cache(max_pages=0x7FFF0000 // 16 + 1)), INVALID, "too large")


@pytest.mark.parametrize("kw", [{"ks": (1 << 23) + 8, "n": 2}, {"vs": 1 << 24, "n": 2}])
def test_prompt_refuses_wide_rows(lib, ctx, kw):
    """Rows of keys and values no further apart than 2^23 elements."""
    far = dict(q=1 << 45, k=1 << 46, v=3 << 45, out=1 << 47)
    refused(lib, call_prompt(lib, ctx, **far, **kw), INVALID, "strides must not exceed")


def cache(**kw):
    a = dict(k=0x7000000000, v=0x7100000000, page_table=0x7200000000, seq_lens=0x7200100000, ref_counts=0x7200200000, dtype=2,
             n_layers=2, n_pages=64, n_kv_heads=2, page_size=16, head_dim=64, n_seqs=4, max_pages=16)
    a.update(kw)
    return KvCacheDesc(**a)


def call_append(lib, ctx, c=None, **kw):
    a = dict(layer=0, seqs=F, cu=F + 4096, batch=1, rows=4, dtype=0, k=A, ks=128, v=B, vs=128, rope=plan(), pos=F + 8192, q=D,
             qs=512, nq=8, qt=0, qo=E, qos=512)
    a.update(kw)
    c = c or cache()
    return lib.objeta_hip_kv_append_device(addr(ctx), None, C.byref(c), a["layer"], a["seqs"], a["cu"], a["batch"], a["rows"],
                                           a["dtype"], a["k"], a["ks"], a["v"], a["vs"], C.byref(a["rope"]) if a["rope"] else None,
                                           a["pos"], a["q"], a["qs"], a["nq"], a["qt"], a["qo"], a["qos"])


def call_cached(lib, ctx, c=None, **kw):
    a = dict(layer=0, seqs=F, cu=F + 4096, batch=1, rows=4, mr=4, ml=100, dtype=2, q=A, qs=512, nq=8, tree=None, scale=0.125,
             out=B, os=512, lse=None)
    a.update(kw)
    c = c or cache()
    return lib.objeta_hip_attn_cached_device(addr(ctx), None, C.byref(c), a["layer"], a["seqs"], a["cu"], a["batch"], a["rows"],
                                             a["mr"], a["ml"], a["dtype"], a["q"], a["qs"], a["nq"], a["tree"], a["scale"],
                                             a["out"], a["os"], a["lse"])


BAD_CACHES = [({"k": None}, "NULL"), ({"page_table": None}, "NULL"), ({"dtype": 8}, "dtype"), ({"n_layers": 0}, "no layers"),
              ({"page_size": 4}, "page_size"), ({"page_size": 24}, "page_size"), ({"page_size": 512}, "page_size"),
              ({"head_dim": 4}, "head_dim"), ({"head_dim": 320}, "head_dim"), ({"v": 0x7100000008}, "16-byte"),
              ({"n_pages": 1 << 31}, "too large"), ({"max_pages": 1 << 28}, "too large"), ({"n_layers": 60000, "n_pages": 1 << 30}, "too large")]


@pytest.mark.parametrize("kw,text", BAD_CACHES)
def test_every_cache_call_checks_the_cache(lib, ctx, kw, text):
    c = cache(**kw)
    refused(lib, call_append(lib, ctx, c), INVALID, text)
    refused(lib, call_cached(lib, ctx, c), INVALID, text)
    refused(lib, lib.objeta_hip_kv_extend_device(addr(ctx), None, C.byref(c), F, F, 1), INVALID, text)
    refused(lib, lib.objeta_hip_kv_fork_device(addr(ctx), None, C.byref(c), F, F, 1), INVALID, text)
    refused(lib, lib.objeta_hip_kv_compact_device(addr(ctx), None, C.byref(c), F, F, F, F, 1, 4), INVALID, text)
    refused(lib, lib.objeta_hip_kv_free_device(addr(ctx), None, C.byref(c), F, 1), INVALID, text)


@pytest.mark.parametrize("kw,text", [
    ({"layer": 2}, "layer 2 out of bounds"), ({"rope": plan(128)}, "exceeds"), ({"dtype": 5}, "dtype"), ({"qt": 5}, "dtype"),
    ({"seqs": None}, "sequences"), ({"cu": None}, "cu_rows"), ({"pos": None}, "positions"), ({"k": None}, "k is NULL"),
    ({"vs": 120}, "stride"), ({"q": None}, "q is NULL"), ({"qo": D, "qt": 2}, "overlaps its input"), ({"qo": A}, "overlaps another"),
    ({"k": 0x7000000000}, "overlaps"), ({"v": 0x7100000100}, "overlaps"), ({"qo": 0x7000000000}, "overlaps"), ({"nq": 70000}, "n_q_heads"),
    ({"rows": 1 << 31}, "too many"),
])
def test_append_refuses(lib, ctx, kw, text):
    refused(lib, call_append(lib, ctx, **kw), INVALID, text)


@pytest.mark.parametrize("kw", [{"nq": 0}, {"nq": 0, "q": None}, {"nq": 0, "qo": None}, {"nq": 0, "rows": 0}])
def test_append_refuses_queries_without_heads(lib, ctx, kw):
    """Queries that would be left as they are without a word: their count was forgotten."""
    refused(lib, call_append(lib, ctx, **kw), INVALID, "without n_q_heads")


@pytest.mark.parametrize("kw,text", [
    ({"layer": 2}, "out of bounds"), ({"dtype": 9}, "dtype"), ({"nq": 3}, "multiple"), ({"scale": 0.0}, "scale"), ({"batch": 65536}, "65535"),
    ({"seqs": None}, "sequences"), ({"mr": 0}, "max_rows"), ({"ml": 0}, "max_len"), ({"q": A + 4}, "16-byte"), ({"os": 508}, "stride"),
    ({"out": A}, "overlaps"), ({"out": 0x7000000000}, "overlaps"), ({"lse": B}, "overlaps"), ({"tree": F + 4}, "tree"),
])
def test_cached_refuses(lib, ctx, kw, text):
    refused(lib, call_cached(lib, ctx, **kw), INVALID, text)


def test_cached_refuses_mixed_types(lib, ctx):
    refused(lib, call_cached(lib, ctx, dtype=1), UNSUPPORTED, "float or of the cache's type")
    refused(lib, call_cached(lib, ctx, cache(dtype=0), dtype=2), UNSUPPORTED, "float or of the cache's type")


def test_page_operations_refuse(lib, ctx):
    c = cache()
    refused(lib, lib.objeta_hip_kv_extend_device(addr(ctx), None, C.byref(c), F, F, 1025), INVALID, "at most 1024")
    refused(lib, lib.objeta_hip_kv_extend_device(addr(ctx), None, C.byref(c), None, F, 1), INVALID, "NULL")
    refused(lib, lib.objeta_hip_kv_fork_device(addr(ctx), None, C.byref(c), F, None, 1), INVALID, "NULL")
    refused(lib, lib.objeta_hip_kv_free_device(addr(ctx), None, C.byref(c), None, 1), INVALID, "NULL")
    refused(lib, lib.objeta_hip_kv_compact_device(addr(ctx), None, C.byref(c), F, F, None, F, 1, 4), INVALID, "NULL")
    refused(lib, lib.objeta_hip_kv_compact_device(addr(ctx), None, C.byref(c), F, F, F, F, 1, 65), INVALID, "max_keep")
    refused(lib, lib.objeta_hip_kv_free_device(addr(ctx), None, None, F, 1), INVALID, "cache is NULL")
    for fn in (lib.objeta_hip_kv_extend_device, lib.objeta_hip_kv_fork_device):
        refused(lib, fn(None, None, C.byref(c), F, F, 1), INVALID, "context is NULL")


def test_python_names_are_checked():
    with pytest.raises(ValueError):
        KvCache(type("B", (), {"L": None})(), 1, 1, 1, 8, 8, 1, 1, dtype="f64")
