"""Calls on the caches of a batch that the library refuses, or has nothing to do for: both are
settled on the host before anything is launched, so they run without a GPU."""
import ctypes

import pytest

import uaii_amd
from uaii_amd import KV_F16, KV_F32, KV_Q8, ScoreOptions

I64 = ctypes.c_int64
A = 1 << 20  # addresses that are never followed
REFUSED = -1


def at(p):
    return None if p is None else ctypes.c_void_p(p)


def test_cache_bytes():
    L = uaii_amd.lib()
    assert L.uaii_hip_kv_cache_bytes(KV_F32, 8, 100, 64) == 8 * 100 * 64 * 4
    assert L.uaii_hip_kv_cache_bytes(KV_F16, 8, 100, 64) == 8 * 100 * 64 * 2
    assert L.uaii_hip_kv_cache_bytes(KV_Q8, 8, 100, 64) == 8 * 100 * 68
    assert L.uaii_hip_kv_cache_bytes(KV_Q8, 1, 7, 16) == 144  # 140 bytes, to the next 16
    for bad in [(3, 8, 100, 64), (-1, 8, 100, 64), (KV_Q8, 0, 100, 64), (KV_Q8, 8, 0, 64), (KV_Q8, 8, 100, 0), (KV_Q8, 8, 100, 72),
                (KV_Q8, 8, 100, 272), (KV_Q8, 8, (1 << 30) + 1, 64), (KV_Q8, 65536, 100, 64)]:
        assert L.uaii_hip_kv_cache_bytes(*bad) == -1, bad


ROWS = dict(k=A, v=2 * A, ld=512, kc=4 * A, vc=5 * A, t=KV_Q8, n=2, rows=3, kv=8, hd=64, seq=100, p0=0, past=6 * A)


def rows_call(append, **kw):
    a = {**ROWS, **kw}
    L = uaii_amd.lib()
    place = [a["t"], I64(a["n"]), I64(a["rows"]), a["kv"], a["hd"], I64(a["seq"]), I64(a["p0"]), at(a["past"])]
    if append:
        return L.uaii_hip_kv_append_batch(at(a["k"]), at(a["v"]), I64(a["ld"]), at(a["kc"]), at(a["vc"]), *place, None)
    return L.uaii_hip_kv_read(at(a["kc"]), *place, at(a["k"]), I64(a["ld"]), None)


@pytest.mark.parametrize("append", [True, False])
@pytest.mark.parametrize("bad", [dict(k=None), dict(kc=None), dict(kc=4 * A + 8), dict(k=A + 2), dict(past=6 * A + 2), dict(t=3),
                                 dict(t=-1), dict(n=-1), dict(rows=-1), dict(kv=0), dict(hd=24), dict(hd=0), dict(hd=512), dict(seq=0),
                                 dict(seq=(1 << 30) + 1), dict(ld=511), dict(p0=-1), dict(p0=101), dict(past=None, p0=98),
                                 dict(rows=1 << 32), dict(n=1 << 31), dict(n=1 << 16, rows=1 << 13)], ids=str)
def test_rows_refused(append, bad):
    assert rows_call(append, **bad) == REFUSED


@pytest.mark.parametrize("append", [True, False])
def test_no_rows(append):
    assert rows_call(append, n=0) == 0
    assert rows_call(append, rows=0) == 0
    assert rows_call(append, rows=0, k=None, v=None, kc=None, vc=None) == 0


def test_append_needs_v():
    assert rows_call(True, v=None) == REFUSED and rows_call(True, vc=None) == REFUSED and rows_call(True, vc=5 * A + 4) == REFUSED


ATTN = dict(q=A, ldq=2048, n=2, kc=4 * A, vc=5 * A, t=KV_F16, seq=100, lens=6 * A, kp=7 * A, vp=8 * A, pre_seq=50, prefix=50, heads=32, kv=8,
            hd=64, opt={}, out=16 * A, ldo=2048, p0=10, bidir=0, first=9 * A)


def attn_call(batch, **kw):
    a = {**ATTN, **kw}
    L = uaii_amd.lib()
    o = a["opt"] if not isinstance(a["opt"], dict) else ScoreOptions(**a["opt"])
    tail = [a["heads"], a["kv"], a["hd"], None if o is None else ctypes.byref(o), at(a["out"]), I64(a["ldo"]), None]
    head = [at(a["q"]), I64(a["ldq"]), I64(a["n"]), at(a["kc"]), at(a["vc"]), a["t"], I64(a["seq"])]
    if batch:
        return L.uaii_hip_attention_batch(*head, at(a["lens"]), at(a["kp"]), at(a["vp"]), I64(a["pre_seq"]), I64(a["prefix"]), *tail)
    return L.uaii_hip_attention_prompt(*head, I64(a["p0"]), I64(a["bidir"]), at(a["first"]), *tail)


def short_options():
    o = ScoreOptions()
    o.struct_size -= 4
    return o


@pytest.mark.parametrize("batch", [True, False])
@pytest.mark.parametrize("bad", [dict(q=None), dict(out=None), dict(kc=None), dict(vc=None), dict(kc=4 * A + 8), dict(vc=5 * A + 2), dict(q=A + 1),
                                 dict(out=16 * A + 2), dict(ldq=2047), dict(ldo=2047), dict(n=-1), dict(n=1 << 31), dict(t=5), dict(seq=0),
                                 dict(seq=(1 << 30) + 1), dict(heads=0), dict(heads=33), dict(heads=65536 * 8), dict(kv=0), dict(hd=65), dict(hd=0),
                                 dict(hd=288), dict(out=A), dict(out=A + 4 * 2047), dict(out=A - 4 * 2048), dict(opt=dict(softcap=-1.0)),
                                 dict(opt=dict(softcap=float("nan"))), dict(opt=dict(softcap=float("inf"))), dict(opt=dict(scale=float("inf"))),
                                 dict(opt=dict(window=-1)), dict(opt=dict(slopes=ctypes.c_void_p(A + 2))), dict(opt=short_options())],
                         ids=lambda d: str(d) if not any(isinstance(v, ScoreOptions) for v in d.values()) else "short options")
def test_attention_refused(batch, bad):
    assert attn_call(batch, **bad) == REFUSED


@pytest.mark.parametrize("bad", [dict(lens=None), dict(lens=6 * A + 1), dict(prefix=-1), dict(kp=None), dict(vp=None), dict(kp=7 * A + 8),
                                 dict(prefix=51), dict(prefix=(1 << 30) - 99, pre_seq=1 << 30), dict(pre_seq=(1 << 30) + 1)], ids=str)
def test_batch_refused(bad):
    assert attn_call(True, **bad) == REFUSED


@pytest.mark.parametrize("bad", [dict(p0=-1), dict(p0=99), dict(p0=101), dict(n=91), dict(bidir=-1), dict(bidir=13), dict(first=9 * A + 2)], ids=str)
def test_prompt_refused(bad):
    assert attn_call(False, **bad) == REFUSED


@pytest.mark.parametrize("batch", [True, False])
def test_no_queries(batch):
    assert attn_call(batch, n=0, q=None, out=None, lens=None, first=None, prefix=0) == 0


def test_options_init():
    o = ScoreOptions(scale=3.0, softcap=2.0, window=9)
    uaii_amd.lib().uaii_hip_score_options_init(ctypes.byref(o))
    assert (o.struct_size, o.scale, o.softcap, o.slopes, o.window) == (ctypes.sizeof(ScoreOptions), 0.0, 0.0, None, 0)


@pytest.mark.parametrize("batch", [True, False])
def test_softcap_has_an_end(batch):
    assert attn_call(batch, opt=dict(softcap=1.01e20)) == REFUSED


@pytest.mark.parametrize("batch", [True, False])
@pytest.mark.parametrize("bad", [dict(out=A + 4 * 2047, ldq=4096, ldo=4096), dict(out=A + 4 * 2049, ldq=4096, ldo=4096),
                                 dict(out=A + 4 * 2048, ldq=4096, ldo=4097), dict(out=A + 4 * 4096, ldq=4096, ldo=4096)], ids=str)
def test_rows_that_meet(batch, bad):
    """Rows of one pitch may lie between each other, if none touches another; with two pitches the ranges count."""
    assert attn_call(batch, **bad) == REFUSED
