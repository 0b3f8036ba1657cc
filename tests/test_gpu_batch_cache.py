"""Caches of a batch: rows written and read back, and attention over them.

Every result is held against the operator's definition in 64 bits. Tolerances of the
attentions are worked out for each output value from the inputs (see `attend`); what the
caches hold is compared exactly."""
import ctypes
import math
import threading

import numpy as np
import pytest
import torch

import uaii_amd
from uaii_amd import KV_F16, KV_F32, KV_Q8, ScoreOptions, check_hip

pytestmark = pytest.mark.gpu

I64 = ctypes.c_int64
TYPES = [KV_F32, KV_F16, KV_Q8]
NAMES = {KV_F32: "f32", KV_F16: "f16", KV_Q8: "q8"}
BEHIND = 0xAB  # what lies where nothing may be written


def ptr(t):
    return None if t is None else ctypes.c_void_p(t.data_ptr())


def seq_bytes(t, kv, seq, hd):
    n = uaii_amd.lib().uaii_hip_kv_cache_bytes(t, kv, seq, hd)
    assert n > 0
    return n


# ---- the definition ---------------------------------------------------------------------


def quantised(x):
    """Bytes and scales of 8-bit rows (numpy, the last axis a row)."""
    x = x.astype(np.float64)
    with np.errstate(all="ignore"):
        top = np.abs(x).max(-1)
        d = (top / 127.0).astype(np.float32)
        d = np.minimum(d, np.nextafter(np.float32(np.finfo(np.float32).max / 127.0), np.float32(0)))  # 127 d stays finite
        q = np.clip(np.rint(np.where(d[..., None] > 0, x / d[..., None].astype(np.float64), 0.0)), -127, 127)
    bad = ~np.isfinite(x).all(-1)
    d[bad] = np.nan
    q[bad] = 0
    return (q + 128).astype(np.uint8), d


def pack(x, t):
    """[n, kv, seq, hd] f32 (numpy) as the bytes of a batch's cache, and the values it holds in 64 bits."""
    n, kv, seq, hd = x.shape
    if t == KV_F32:
        return torch.from_numpy(x.view(np.uint8).reshape(n, -1).copy()).cuda(), x.astype(np.float64)
    if t == KV_F16:
        h = x.astype(np.float16)
        return torch.from_numpy(h.view(np.uint8).reshape(n, -1).copy()).cuda(), h.astype(np.float64)
    q, d = quantised(x)
    out = np.full((n, seq_bytes(t, kv, seq, hd)), BEHIND, dtype=np.uint8)
    out[:, : kv * seq * hd] = q.reshape(n, -1)
    out[:, kv * seq * hd : kv * seq * (hd + 4)] = d.reshape(n, -1).view(np.uint8)
    return torch.from_numpy(out).cuda(), (q.astype(np.float64) - 128) * d.astype(np.float64)[..., None]


def attend(q, k, v, at, pos, lo, hi, scale, cap, slope):
    """One head's rows q [r, hd] over k, v [n, hd] at positions `at`; row i is at pos[i] and sees
    lo[i] <= position < hi[i]. The result and what the library's may differ from it by.

    The bound, with u = 2^-24: q and the probabilities enter as pairs of f16 numbers (off by
    4 u relative, both together 8 u), products and sums in f32 of hd terms are off by at most
    (hd + 4) u of the sum of magnitudes, softcap and bias add a few u of their size, and the
    exponential a few u. An error e of a score is one of e relative in its probability, and of
    2 e in a normalised one. Sums over the keys: at most (n + 8) u, of which blocked sums keep
    under 64 u for any n."""
    q, k, v = q.astype(np.float64), k.astype(np.float64), v.astype(np.float64)
    u = 2.0 ** -24
    out, tol = np.zeros_like(q), np.zeros_like(q)
    for i in range(q.shape[0]):
        seen = (at >= lo[i]) & (at < hi[i])
        if not seen.any():
            continue
        kk, vv = k[seen], v[seen]
        s = scale * (kk @ q[i])
        e = abs(scale) * (np.abs(kk) @ np.abs(q[i])) * (q.shape[1] + 12) * u
        if cap:
            s = cap * np.tanh(s / cap)
            e = np.minimum(e, 2 * cap) + 8 * u * cap
        bias = slope * np.abs(pos[i] - at[seen])
        s = s - bias
        e = e + 2 * u * bias + 4 * u * np.abs(s)
        p = np.exp(s - s.max())
        p /= p.sum()
        e = 2 * e.max() + 80 * u
        out[i] = p @ vv
        tol[i] = e * (p @ np.abs(vv)) + 2.0 ** -36 * np.abs(vv).max()
    return out, tol


def close(got, want, tol):
    off = np.abs(got.astype(np.float64) - want)
    assert np.isfinite(got).all()
    worst = float((off / np.maximum(tol, 1e-300)).max()) if off.size else 0.0
    assert worst <= 1.0, "off by %.3g of the bound" % worst


def rows(rng, *shape):
    return rng.standard_normal(shape).astype(np.float32)


def options(cap=0.0, slopes=None, window=0, scale=0.0):
    return ScoreOptions(scale=scale, softcap=cap, slopes=ptr(slopes), window=window)


# ---- writing and reading back ---------------------------------------------------------------


@pytest.mark.parametrize("hd", [16, 32, 48, 64, 80, 112, 128, 192, 256])
@pytest.mark.parametrize("t", TYPES, ids=NAMES.get)
def test_rows_written_and_read(hip, t, hd):
    """Odd counts, padded rows, lengths of their own, rows outside the cache; nothing else moves."""
    rng = np.random.default_rng(hd)
    n, m, kv, seq, ld = 3, 5, 3, 37, 3 * hd + 7
    past = np.array([0, seq - 2, -1], dtype=np.int32)  # at the start, over the end, before the start
    k, v = rows(rng, n * m, ld) * 3, rows(rng, n * m, ld)
    size = seq_bytes(t, kv, seq, hd)
    kc, vc = (torch.full((n * size + 64,), BEHIND, dtype=torch.uint8, device="cuda") for _ in range(2))
    dk, dv, dp = (torch.from_numpy(x).cuda() for x in (k, v, past))
    place = [t, I64(n), I64(m), kv, hd, I64(seq), I64(0), ptr(dp)]
    check_hip(hip.uaii_hip_kv_append_batch(ptr(dk), ptr(dv), I64(ld), ptr(kc), ptr(vc), *place, None))
    for x, cache in ((k, kc), (v, vc)):
        want = np.full(n * size + 64, BEHIND, dtype=np.uint8)
        held = np.zeros((n * m, kv, hd))
        there = np.zeros(n * m, dtype=bool)
        x3 = x[:, : kv * hd].reshape(n * m, kv, hd)
        q, d = quantised(x3)
        for s in range(n):
            mine = want[s * size : (s + 1) * size]
            for i in range(m):
                at, r = int(past[s]) + i, s * m + i
                if not 0 <= at < seq:
                    continue
                there[r] = True
                for h in range(kv):
                    row = h * seq + at
                    if t == KV_Q8:
                        mine[row * hd : (row + 1) * hd] = q[r, h]
                        mine[kv * seq * hd + 4 * row : kv * seq * hd + 4 * row + 4] = d[r, h : h + 1].view(np.uint8)
                        held[r, h] = ((q[r, h].astype(np.float32) - 128) * d[r, h]).astype(np.float64)
                    else:
                        val = x3[r, h].astype(np.float16 if t == KV_F16 else np.float32)
                        e = val.dtype.itemsize
                        mine[row * hd * e : (row + 1) * hd * e] = val.view(np.uint8)
                        held[r, h] = val
        assert np.array_equal(cache.cpu().numpy(), want)
        back = torch.full((n * m, ld), -7.0, device="cuda")
        check_hip(hip.uaii_hip_kv_read(ptr(cache), *place, ptr(back), I64(ld), None))
        back = back.cpu().numpy()
        assert np.array_equal(back[:, kv * hd :], np.full((n * m, ld - kv * hd), -7.0, np.float32))
        got = back[:, : kv * hd].reshape(n * m, kv, hd)
        assert np.array_equal(got[there], held[there].astype(np.float32))
        assert (got[~there] == -7.0).all()


def test_8_bit_rounding(hip):
    """Ties, zeros, the ends of f32 and rows that are not finite, against exact quotients."""
    hd, kv, seq = 64, 1, 64
    rng = np.random.default_rng(5)
    x = rows(rng, seq, hd)
    x[0] = 0.0
    x[1] = np.linspace(-127, 127, hd)
    x[2, :] = np.arange(hd) + 0.5  # scale 1: ties everywhere
    x[2, 0] = 127.0
    x[3] = -x[2]
    x[4] *= np.float32(1e-44)
    x[5] *= np.float32(3e-39)
    x[6] *= np.float32(2.0 ** -100)
    x[7] = rows(rng, hd) * np.float32(5e37)
    x[8, 3] = np.inf
    x[9, 5] = np.nan
    x[10] = np.float32(1e-45)
    x[11, :] = np.float32(3.4028235e38)
    x[12] = np.float32(0.1) * (np.arange(hd) - 31)
    x[13] = (np.arange(hd) - 31.5) * np.float32(2.0 ** -30)
    x[13, 0] = 127 * 2.0 ** -30
    q, d = quantised(x)
    cache = [torch.zeros(seq_bytes(KV_Q8, kv, seq, hd), dtype=torch.uint8, device="cuda") for _ in range(2)]
    dx = torch.from_numpy(x).cuda()
    check_hip(hip.uaii_hip_kv_append_batch(ptr(dx), ptr(dx), I64(hd), ptr(cache[0]), ptr(cache[1]), KV_Q8, I64(1), I64(seq), kv, hd,
                                           I64(seq), I64(0), None, None))
    for c in cache:
        got = c.cpu().numpy()
        assert np.array_equal(got[seq * hd : seq * hd + 4 * seq].view(np.float32), d, equal_nan=True)
        assert np.array_equal(got[: seq * hd].reshape(seq, hd), q)
    back = torch.zeros(seq, hd, device="cuda")
    check_hip(hip.uaii_hip_kv_read(ptr(cache[0]), KV_Q8, I64(1), I64(seq), kv, hd, I64(seq), I64(0), None, ptr(back), I64(hd), None))
    back = back.cpu().numpy()
    assert np.isnan(back[8]).all() and np.isnan(back[9]).all() and (back[0] == 0).all()
    fine = [i for i in range(seq) if i not in (8, 9) and d[i] >= 2.0 ** -126]
    assert (np.abs(back[fine] - x[fine].astype(np.float64)) <= d[fine, None].astype(np.float64) * 0.5001).all()


@pytest.mark.parametrize("hd", [16, 80, 256])
def test_8_bit_rounding_of_many(hip, hd):
    """Rows of all sizes, a third of them on halves of a step, a third a last place beside one."""
    rng = np.random.default_rng(hd)
    n = 600_000 // hd
    x = rows(rng, n, hd)
    half = (rng.integers(-253, 254, (n, hd)) * 0.5).astype(np.float32)
    half[:, 0] = 127.0
    x[n // 3 :] = half[n // 3 :]
    beside = np.nextafter(half, np.where(rng.random((n, hd)) < 0.5, -np.inf, np.inf).astype(np.float32))
    beside[:, 0] = 127.0
    x[2 * n // 3 :] = beside[2 * n // 3 :]
    with np.errstate(over="ignore", under="ignore"):
        x *= (2.0 ** rng.uniform(-149, 121, (n, 1))).astype(np.float32)
        x[::2] *= np.float32(1.0 / 3.0)
    assert np.isfinite(x).all()
    q, d = quantised(x)
    caches = [torch.zeros(seq_bytes(KV_Q8, 1, n, hd), dtype=torch.uint8, device="cuda") for _ in range(2)]
    dx = torch.from_numpy(x).cuda()
    check_hip(hip.uaii_hip_kv_append_batch(ptr(dx), ptr(dx), I64(hd), ptr(caches[0]), ptr(caches[1]), KV_Q8, I64(1), I64(n), 1, hd, I64(n),
                                           I64(0), None, None))
    for c in caches:
        got = c.cpu().numpy()
        assert np.array_equal(got[n * hd : n * (hd + 4)].view(np.float32), d)
        assert np.array_equal(got[: n * hd].reshape(n, hd), q)


# ---- attention of a batch --------------------------------------------------------------------


def run_batch(hip, rng, t, heads, kv, hd, lens, seq, prefix=0, cap=0.0, slopes=False, window=0, scale=0.0, ldq=None, stream=None,
              spread=1.0):
    """One call on random inputs; places that no query sees hold NaN. (result, want, bound)."""
    n, g = len(lens), heads // kv
    ldq = ldq or heads * hd
    pre_seq = prefix + 5
    q = rows(rng, n, ldq) * np.float32(spread)
    k, v = rows(rng, n, kv, seq, hd), rows(rng, n, kv, seq, hd)
    kp, vp = rows(rng, 1, kv, pre_seq, hd), rows(rng, 1, kv, pre_seq, hd)
    used = [min(max(x, 0), seq) for x in lens]
    for s, x in enumerate(used):
        k[s, :, x:] = v[s, :, x:] = np.nan
        if window:
            k[s, :, : max(0, x - window)] = v[s, :, : max(0, x - window)] = np.nan
    kp[:, :, prefix:] = vp[:, :, prefix:] = np.nan
    if window:
        hidden = max(0, prefix + min(used) - window)
        kp[:, :, :hidden] = vp[:, :, :hidden] = np.nan
    (kc, kx), (vc, vx), (kpc, kpx), (vpc, vpx) = (pack(x, t) for x in (k, v, kp, vp))
    slope = np.array([2.0 ** (-8 * (i + 1) / heads) for i in range(heads)], dtype=np.float32) if slopes else np.zeros(heads, np.float32)
    ds = torch.from_numpy(slope).cuda()
    opt = options(cap, ds if slopes else None, window, scale)
    dq, dn = torch.from_numpy(q).cuda(), torch.tensor(lens, dtype=torch.int32, device="cuda")
    out = torch.full((n + 2, heads * hd + 3), -7.0, device="cuda")
    keep = (kc, vc, kpc, vpc, dq, dn, ds)

    def call(stream=stream):
        check_hip(hip.uaii_hip_attention_batch(
            ptr(dq), I64(ldq), I64(n), ptr(kc), ptr(vc), t, I64(seq), ptr(dn), ptr(kpc) if prefix else None, ptr(vpc) if prefix else None,
            I64(pre_seq), I64(prefix), heads, kv, hd, ctypes.byref(opt), ptr(out), I64(heads * hd + 3), stream))
        return out, keep

    want, tol = np.zeros((n, heads, hd)), np.zeros((n, heads, hd))
    sc = float(np.float32(scale)) if scale else float(np.float32(1.0 / math.sqrt(hd)))
    for s, x in enumerate(used):
        at = np.arange(prefix + x)
        pos = np.array([prefix + x - 1])
        lo = pos - window + 1 if window else np.array([0])
        for h in range(heads):
            j = h // g
            kk = np.concatenate([kpx[0, j, :prefix], kx[s, j, :x]])
            vv = np.concatenate([vpx[0, j, :prefix], vx[s, j, :x]])
            if not len(at):
                continue
            want[s, h], tol[s, h] = (y[0] for y in attend(q[s : s + 1, h * hd : (h + 1) * hd], kk, vv, at, pos, lo, pos + 1, sc, cap, float(slope[h])))
    return call, want.reshape(n, -1), tol.reshape(n, -1)


def check_batch(hip, *a, **kw):
    call, want, tol = run_batch(hip, *a, **kw)
    out, keep = call()
    torch.cuda.synchronize()
    out = out.cpu().numpy()
    n = want.shape[0]
    close(out[:n, : want.shape[1]], want, tol)
    assert (out[n:] == -7.0).all() and (out[:, want.shape[1] :] == -7.0).all()


SHAPES = [(8, 8, 64), (32, 8, 64), (8, 2, 128), (14, 2, 32), (6, 2, 80), (20, 4, 112), (4, 1, 256), (40, 2, 48), (8, 1, 16), (64, 2, 128)]


@pytest.mark.parametrize("shape", SHAPES, ids=str)
@pytest.mark.parametrize("t", TYPES, ids=NAMES.get)
def test_batch_shapes(hip, t, shape):
    check_batch(hip, np.random.default_rng(1), t, *shape, lens=[1, 150, 0, 31, 64, 33], seq=150)


@pytest.mark.parametrize("t", TYPES, ids=NAMES.get)
@pytest.mark.parametrize("lens,seq", [([0], 1), ([1], 1), ([2], 3), ([16], 16), ([17], 40), ([127], 127), ([128], 128), ([129], 200),
                                      ([-5, 300, 7], 260), ([0, 0, 0], 9), ([1000, 3, 0, 77, 513, 511, 512, 1], 1000)], ids=str)
def test_batch_lengths(hip, t, lens, seq):
    """Nothing, one, the tiles' borders, lengths that the caches do not have."""
    check_batch(hip, np.random.default_rng(2), t, 8, 2, 64, lens=lens, seq=seq)


@pytest.mark.parametrize("t", TYPES, ids=NAMES.get)
@pytest.mark.parametrize("prefix", [1, 63, 64, 300, 1111])
@pytest.mark.parametrize("shape", [(8, 2, 64), (32, 8, 128), (5, 1, 80), (4, 2, 256)], ids=str)
def test_batch_prefix(hip, t, prefix, shape):
    check_batch(hip, np.random.default_rng(3), t, *shape, lens=[5, 0, 200, 1, 33], seq=200, prefix=prefix)


# (shape, sequences, prefix): too much for each sequence to read the prefix by itself, with few
# and many query rows, a last row tile of one row, prefixes of whole tiles and not
SHARED = [((8, 2, 64), 50, 2100), ((32, 8, 128), 20, 1300), ((5, 1, 80), 70, 3000), ((4, 2, 256), 40, 2600), ((14, 2, 32), 36, 2816),
          ((8, 8, 64), 3, 8500), ((8, 8, 128), 33, 800), ((4, 1, 256), 65, 3100), ((20, 4, 112), 13, 4001)]


@pytest.mark.parametrize("t", TYPES, ids=NAMES.get)
@pytest.mark.parametrize("shape,n,prefix", SHARED, ids=str)
def test_batch_shared_prefix(hip, t, shape, n, prefix):
    assert n * prefix * shape[1] > 192 << 10
    check_batch(hip, np.random.default_rng(3), t, *shape, lens=[(7 * i) % 45 for i in range(n)], seq=45, prefix=prefix)


@pytest.mark.parametrize("t", TYPES, ids=NAMES.get)
@pytest.mark.parametrize("shape,n,prefix", SHARED[:2] + SHARED[3:4], ids=str)
@pytest.mark.parametrize("opt", [dict(cap=30.0), dict(slopes=True), dict(window=20), dict(window=700), dict(window=1000, cap=4.0, slopes=True, spread=4.0)],
                         ids=str)
def test_batch_shared_prefix_options(hip, t, shape, n, prefix, opt):
    """A window may hide all of the prefix from some sequences, a part of it from others."""
    check_batch(hip, np.random.default_rng(5), t, *shape, lens=[(7 * i) % 45 for i in range(n)], seq=45, prefix=prefix, **opt)


@pytest.mark.parametrize("t,shape,n,prefix", [
    (KV_F32, (16, 4, 64), 165, 128), (KV_F32, (64, 8, 64), 139, 287), (KV_F32, (32, 4, 128), 163, 128), (KV_F32, (8, 8, 256), 95, 128),
    (KV_F16, (8, 8, 64), 119, 128), (KV_Q8, (8, 8, 64), 119, 128), (KV_F16, (64, 8, 64), 133, 160), (KV_Q8, (4, 4, 64), 150, 133),
    (KV_F16, (64, 8, 64), 154, 302), (KV_Q8, (64, 8, 64), 154, 302), (KV_F16, (4, 4, 128), 142, 128), (KV_F16, (64, 8, 128), 144, 360),
    (KV_Q8, (64, 8, 128), 144, 360), (KV_F16, (8, 8, 256), 78, 128), (KV_Q8, (8, 8, 256), 78, 128)], ids=str)
def test_batch_shared_prefix_of_many(hip, t, shape, n, prefix):
    """One, two and four row waves, with and without splits."""
    check_batch(hip, np.random.default_rng(33), t, *shape, lens=[(7 * i) % 20 for i in range(n)], seq=45, prefix=prefix)


@pytest.mark.parametrize("t,shape,n,prefix", [
    (KV_F32, (64, 8, 64), 161, 157), (KV_F32, (8, 8, 64), 9, 2781), (KV_F32, (64, 8, 256), 181, 139), (KV_F32, (8, 8, 256), 146, 172),
    (KV_F16, (16, 8, 64), 202, 128), (KV_Q8, (2, 2, 64), 162, 619), (KV_F16, (64, 8, 64), 190, 140), (KV_Q8, (8, 8, 64), 178, 151),
    (KV_Q8, (32, 8, 128), 247, 128), (KV_F16, (1, 1, 128), 84, 2403), (KV_F16, (64, 8, 256), 155, 164), (KV_Q8, (8, 8, 256), 123, 204)], ids=str)
def test_batch_prefix_read_once_for_many(hip, t, shape, n, prefix):
    """The same, beyond what the sequences' own blocks would read of the prefix."""
    assert n * shape[1] * prefix > 192 << 10
    check_batch(hip, np.random.default_rng(41), t, *shape, lens=[(7 * i) % 12 for i in range(n)], seq=45, prefix=prefix)


@pytest.mark.parametrize("t", TYPES, ids=NAMES.get)
@pytest.mark.parametrize("heads,window", [(8, 20), (8, 100), (40, 45)])
def test_batch_shared_prefix_window(hip, t, heads, window):
    """The same for many sequences and a narrow window; more query heads than a block has rows."""
    check_batch(hip, np.random.default_rng(31), t, heads, 4, 32, lens=[(7 * i) % 45 for i in range(300)], seq=45, prefix=500, window=window,
                slopes=True)


@pytest.mark.parametrize("t", TYPES, ids=NAMES.get)
@pytest.mark.parametrize("window", [60, 97, 128, 129, 161, 200])
def test_batch_prefix_in_a_window(hip, t, window):
    """Windows that begin anywhere in a prefix read with the sequences' own keys."""
    check_batch(hip, np.random.default_rng(32), t, 4, 2, 64, lens=[0, 1, 31, 32, 33, 96, 160, 160], seq=160, prefix=75, window=window)


@pytest.mark.parametrize("t", TYPES, ids=NAMES.get)
@pytest.mark.parametrize("prefix", [0, 200])
@pytest.mark.parametrize("opt", [dict(cap=30.0), dict(cap=0.5), dict(slopes=True), dict(window=1), dict(window=50), dict(window=150),
                                 dict(window=1 << 40), dict(scale=0.3), dict(scale=-0.1),
                                 dict(cap=5.0, slopes=True, window=170, scale=0.2, spread=4.0)], ids=str)
def test_batch_options(hip, t, prefix, opt):
    check_batch(hip, np.random.default_rng(4), t, 12, 4, 64, lens=[140, 3, 0, 77], seq=140, prefix=prefix, ldq=12 * 64 + 5, **opt)


@pytest.mark.parametrize("t", TYPES, ids=NAMES.get)
@pytest.mark.parametrize("n", [40, 300])
def test_batch_of_many(hip, t, n):
    """More sequences than a block has threads, most of them short."""
    lens = [(i * 37) % 60 for i in range(n)]
    lens[n // 2] = 700
    check_batch(hip, np.random.default_rng(6), t, 8, 4, 32, lens=lens, seq=700, prefix=90)


@pytest.mark.parametrize("t", TYPES, ids=NAMES.get)
@pytest.mark.parametrize("heads,window,prefix", [(8, 0, 0), (8, 60, 0), (40, 0, 0), (8, 0, 40)])
def test_batch_of_many_short(hip, t, heads, window, prefix):
    """At most 128 keys for each of many sequences, and sequences with none."""
    check_batch(hip, np.random.default_rng(37), t, heads, 8, 64, lens=[(i * 31) % 61 * (i % 5 != 2) for i in range(300)],
                seq=300 if window else 60, window=window, prefix=prefix)


@pytest.mark.parametrize("t", TYPES, ids=NAMES.get)
@pytest.mark.parametrize("shape,n", [((8, 8, 64), 40), ((8, 4, 64), 90), ((8, 4, 128), 64), ((4, 4, 256), 65)], ids=str)
@pytest.mark.parametrize("opt", [dict(), dict(prefix=300), dict(prefix=50, window=1300), dict(window=1200, cap=20.0, slopes=True)], ids=str)
def test_batch_in_shares(hip, t, shape, n, opt):
    """More units than blocks: heads cut anywhere, sequences with none between them."""
    lens = [[0, 30, 1500, 129, 700, 1, 1501][i % 7] if i % 3 else 40 + i for i in range(n)]
    check_batch(hip, np.random.default_rng(38), t, *shape, lens=lens, seq=1500, **opt)


@pytest.mark.parametrize("t", TYPES, ids=NAMES.get)
@pytest.mark.parametrize("shape,n,seq", [((8, 2, 64), 3, 512), ((8, 8, 128), 17, 1024), ((8, 8, 128), 17, 1025), ((2, 1, 256), 5, 512), ((40, 4, 64), 33, 900)],
                         ids=str)
def test_batch_short_capacity(hip, t, shape, n, seq):
    """A block a head up to a capacity, a block a unit behind it."""
    lens = [[seq, 0, 1, 128, 129, 257, seq - 1, seq // 2][i % 8] for i in range(n)]
    check_batch(hip, np.random.default_rng(39), t, *shape, lens=lens, seq=seq)
    check_batch(hip, np.random.default_rng(39), t, *shape, lens=lens, seq=seq, prefix=33, window=seq - 40)


@pytest.mark.parametrize("t", TYPES, ids=NAMES.get)
def test_batch_peaked(hip, t):
    """Scores that one key rules, found late, and keys of unlike size."""
    check_batch(hip, np.random.default_rng(7), t, 8, 2, 64, lens=[900, 333], seq=900, prefix=400, spread=20.0)


def test_batch_values_of_unlike_size(hip):
    """8-bit rows whose scales span ten powers of ten, zero rows among them."""
    rng = np.random.default_rng(8)
    heads, kv, hd, seq = 8, 2, 64, 400
    k, v, q = rows(rng, 1, kv, seq, hd), rows(rng, 1, kv, seq, hd), rows(rng, 1, heads * hd)
    v *= (10.0 ** rng.uniform(-6, 4, (1, kv, seq, 1))).astype(np.float32)
    v[:, :, ::7] = 0.0
    k[:, :, ::5] = 0.0
    (kc, kx), (vc, vx) = pack(k, KV_Q8), pack(v, KV_Q8)
    dq, dn = torch.from_numpy(q).cuda(), torch.tensor([seq], dtype=torch.int32, device="cuda")
    out = torch.zeros(1, heads * hd, device="cuda")
    check_hip(hip.uaii_hip_attention_batch(ptr(dq), I64(heads * hd), I64(1), ptr(kc), ptr(vc), KV_Q8, I64(seq), ptr(dn), None, None,
                                           I64(0), I64(0), heads, kv, hd, None, ptr(out), I64(heads * hd), None))
    got, at = out.cpu().numpy(), np.arange(seq)
    for h in range(heads):
        w, tol = attend(q[:, h * hd : (h + 1) * hd], kx[0, h // 4], vx[0, h // 4], at, np.array([seq - 1]), np.array([0]), np.array([seq]),
                        float(np.float32(1 / 8)), 0.0, 0.0)
        close(got[:, h * hd : (h + 1) * hd], w, tol)


@pytest.mark.parametrize("t", TYPES, ids=NAMES.get)
@pytest.mark.parametrize("prefix", [0, 70])
def test_batch_value_not_finite(hip, t, prefix):
    """A NaN that one sequence sees is that sequence's alone."""
    rng = np.random.default_rng(9)
    heads, kv, hd, seq, lens = 4, 2, 64, 100, [100, 60, 30]
    k, v, q = rows(rng, 3, kv, seq, hd), rows(rng, 3, kv, seq, hd), rows(rng, 3, heads * hd)
    v[1, 0, 20, 7] = np.nan
    kp, vp = rows(rng, 1, kv, max(prefix, 1), hd), rows(rng, 1, kv, max(prefix, 1), hd)
    (kc, _), (vc, _), (kpc, _), (vpc, _) = (pack(x, t) for x in (k, v, kp, vp))
    dq, dn = torch.from_numpy(q).cuda(), torch.tensor(lens, dtype=torch.int32, device="cuda")
    out = torch.zeros(3, heads, hd, device="cuda")
    check_hip(hip.uaii_hip_attention_batch(ptr(dq), I64(heads * hd), I64(3), ptr(kc), ptr(vc), t, I64(seq), ptr(dn), ptr(kpc), ptr(vpc),
                                           I64(max(prefix, 1)), I64(prefix), heads, kv, hd, None, ptr(out), I64(heads * hd), None))
    got = out.cpu().numpy()
    assert np.isnan(got[1, :2, 7]).all()
    assert np.isfinite(got[0]).all() and np.isfinite(got[2]).all() and np.isfinite(got[1, 2:]).all()


@pytest.mark.parametrize("t", TYPES, ids=NAMES.get)
@pytest.mark.parametrize("cap", [1e-38, 1e-20, 1e20])
def test_extreme_softcap(hip, t, cap):
    """A cap that makes all scores alike, those of a query of zeros too, and one that changes none."""
    rng = np.random.default_rng(10)
    heads, kv, hd, seq = 4, 2, 64, 70
    k, v, q = rows(rng, 1, kv, seq, hd), rows(rng, 1, kv, seq, hd), rows(rng, 2, heads * hd)
    q[1] = 0.0
    (kc, kx), (vc, vx) = pack(k, t), pack(v, t)
    twice = lambda c: torch.cat([c, c])  # noqa: E731
    dq, dn, opt = torch.from_numpy(q).cuda(), torch.tensor([seq, seq - 1], dtype=torch.int32, device="cuda"), options(cap)
    kc2, vc2, out = twice(kc), twice(vc), torch.zeros(2, 2, heads * hd, device="cuda")
    check_hip(hip.uaii_hip_attention_batch(ptr(dq), I64(heads * hd), I64(2), ptr(kc2), ptr(vc2), t, I64(seq), ptr(dn), None, None, I64(0),
                                           I64(0), heads, kv, hd, ctypes.byref(opt), ptr(out[0]), I64(heads * hd), None))
    check_hip(hip.uaii_hip_attention_prompt(ptr(dq), I64(heads * hd), I64(2), ptr(kc), ptr(vc), t, I64(seq), I64(seq - 2), I64(0), None, heads,
                                            kv, hd, ctypes.byref(opt), ptr(out[1]), I64(heads * hd), None))
    got, at, none = out.cpu().numpy(), np.arange(seq), np.zeros(2)
    for h in range(heads):
        for call, hi in ((0, [seq, seq - 1]), (1, [seq - 1, seq])):
            w, tol = attend(q[:, h * hd : (h + 1) * hd], kx[0, h // 2], vx[0, h // 2], at, none, none, np.array(hi), 0.125, float(np.float32(cap)), 0.0)
            if cap == 1e20:  # its 8 u of a cap, in the bound, are 8 u of the scores here: cap tanh(s / cap) is s
                w, tol = attend(q[:, h * hd : (h + 1) * hd], kx[0, h // 2], vx[0, h // 2], at, none, none, np.array(hi), 0.125, 0.0, 0.0)
                tol = 2 * tol
            close(got[call][:, h * hd : (h + 1) * hd], w, tol)


@pytest.mark.parametrize("batch", [False, True])
def test_rows_between_each_other(hip, batch):
    """q and out as columns of one buffer."""
    rng = np.random.default_rng(11)
    heads, kv, hd, seq, n = 4, 2, 64, 50, 3
    k, v, q = rows(rng, n, kv, seq, hd), rows(rng, n, kv, seq, hd), rows(rng, n, heads * hd)
    (kc, kx), (vc, vx) = pack(k, KV_F16), pack(v, KV_F16)
    width = heads * hd
    both = torch.full((n, 2 * width + 4), -7.0, device="cuda")
    both[:, :width] = torch.from_numpy(q).cuda()
    lens, out, ld = torch.tensor([50, 7, 20], dtype=torch.int32, device="cuda"), both[:, width:], I64(2 * width + 4)
    if batch:
        check_hip(hip.uaii_hip_attention_batch(ptr(both), ld, I64(n), ptr(kc), ptr(vc), KV_F16, I64(seq), ptr(lens), None, None, I64(0), I64(0),
                                               heads, kv, hd, None, ptr(out), ld, None))
    else:
        check_hip(hip.uaii_hip_attention_prompt(ptr(both), ld, I64(n), ptr(kc), ptr(vc), KV_F16, I64(seq), I64(6), I64(0), None, heads, kv, hd,
                                                None, ptr(out), ld, None))
    got, at, none = both.cpu().numpy(), np.arange(seq), np.zeros(1)
    assert np.array_equal(got[:, :width], q) and (got[:, 2 * width :] == -7.0).all()
    for s in range(n):
        for h in range(heads):
            c, hi = (s, int(lens[s])) if batch else (0, 7 + s)
            w, tol = attend(q[s : s + 1, h * hd : (h + 1) * hd], kx[c, h // 2], vx[c, h // 2], at, none, none, np.array([hi]), 0.125, 0.0, 0.0)
            close(got[s : s + 1, width + h * hd : width + (h + 1) * hd], w, tol)


# ---- attention of prompt rows ----------------------------------------------------------------


def check_prompt(hip, rng, t, heads, kv, hd, m, p0, bidir=0, first=None, cap=0.0, slopes=False, window=0, scale=0.0, room=9, poison=None,
                 spread=1.0, which=None, stream=None, sync=True):
    """One call on random inputs; keys behind the last query hold NaN, and those of `poison`."""
    g, seq, ldq = heads // kv, p0 + m + room, heads * hd + 5
    q = rows(rng, m, ldq) * np.float32(spread)
    k, v = rows(rng, 1, kv, seq, hd), rows(rng, 1, kv, seq, hd)
    k[:, :, p0 + m :] = v[:, :, p0 + m :] = np.nan
    if poison is not None:
        k[:, :, poison] = v[:, :, poison] = np.nan
    (kc, kx), (vc, vx) = pack(k, t), pack(v, t)
    slope = np.array([2.0 ** (-8 * (i + 1) / heads) for i in range(heads)], dtype=np.float32) if slopes else np.zeros(heads, np.float32)
    ds, dq = torch.from_numpy(slope).cuda(), torch.from_numpy(q).cuda()
    df = None if first is None else torch.tensor(first, dtype=torch.int32, device="cuda")
    out = torch.full((m + 2, heads * hd + 3), -7.0, device="cuda")
    opt = options(cap, ds if slopes else None, window, scale)
    check_hip(hip.uaii_hip_attention_prompt(ptr(dq), I64(ldq), I64(m), ptr(kc), ptr(vc), t, I64(seq), I64(p0), I64(bidir), ptr(df), heads,
                                            kv, hd, ctypes.byref(opt), ptr(out), I64(heads * hd + 3), stream))
    torch.cuda.synchronize()
    out = out.cpu().numpy()
    assert (out[m:] == -7.0).all() and (out[:, heads * hd :] == -7.0).all()
    sc = float(np.float32(scale)) if scale else float(np.float32(1.0 / math.sqrt(hd)))
    at, pos = np.arange(p0 + m), p0 + np.arange(m)
    hi = np.maximum(pos + 1, bidir)
    lo = np.zeros(m, dtype=int) if first is None else np.maximum(0, np.array(first, dtype=np.int64))
    if window:
        lo = np.maximum(lo, pos - window + 1)
    pick = np.arange(m) if which is None else np.array(which)
    for h in range(heads):
        w, tol = attend(q[pick, h * hd : (h + 1) * hd], kx[0, h // g, : p0 + m], vx[0, h // g, : p0 + m], at, pos[pick], lo[pick], hi[pick],
                        sc, cap, float(slope[h]))
        close(out[pick, h * hd : (h + 1) * hd], w, tol)


@pytest.mark.parametrize("shape", SHAPES, ids=str)
@pytest.mark.parametrize("t", TYPES, ids=NAMES.get)
def test_prompt_shapes(hip, t, shape):
    check_prompt(hip, np.random.default_rng(11), t, *shape, m=45, p0=70)


@pytest.mark.parametrize("t", TYPES, ids=NAMES.get)
@pytest.mark.parametrize("m,p0", [(1, 0), (1, 5), (2, 0), (3, 130), (16, 0), (17, 64), (64, 63), (65, 0), (128, 1), (200, 333), (5, 2000)])
def test_prompt_lengths(hip, t, m, p0):
    check_prompt(hip, np.random.default_rng(12), t, 8, 2, 64, m=m, p0=p0)


@pytest.mark.parametrize("t", TYPES, ids=NAMES.get)
@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("opt", [dict(cap=30.0), dict(slopes=True), dict(window=1), dict(window=37), dict(window=100), dict(bidir=1),
                                 dict(bidir=190), dict(bidir=129, window=90), dict(scale=0.3, cap=2.0, slopes=True, window=140, spread=3.0)],
                         ids=str)
def test_prompt_options(hip, t, hd, opt):
    check_prompt(hip, np.random.default_rng(13), t, 4, 2, hd, m=150, p0=40, **opt)


@pytest.mark.parametrize("t", TYPES, ids=NAMES.get)
@pytest.mark.parametrize("hd", [64, 128])
def test_prompt_documents(hip, t, hd):
    """Packed documents, rows that see nothing, a negative first key; one document's keys are NaN
    and only its own queries, which see nothing either, could meet them."""
    m, p0 = 210, 20
    first = [-3] * 60 + [p0 + 60] * 50 + [1 << 30] * 40 + [p0 + 150] * 60
    first[-1] = p0 + m
    check_prompt(hip, np.random.default_rng(14), t, 8, 2, hd, m=m, p0=p0, first=first, poison=slice(p0 + 110, p0 + 150))
    check_prompt(hip, np.random.default_rng(15), t, 8, 2, hd, m=m, p0=p0, first=first, poison=slice(p0 + 110, p0 + 150), bidir=p0 + 70, window=99)


@pytest.mark.parametrize("t", TYPES, ids=NAMES.get)
def test_prompt_row_meets_nan(hip, t):
    """Values that are not finite reach the queries that see them and no others."""
    rng = np.random.default_rng(16)
    heads, kv, hd, m = 4, 2, 64, 100
    k, v, q = rows(rng, 1, kv, m, hd), rows(rng, 1, kv, m, hd), rows(rng, m, heads * hd)
    v[0, 0, 50, 3] = np.nan
    v[0, 1, 70, 9] = np.inf
    k[0, 1, 90] = np.nan
    (kc, _), (vc, _) = pack(k, t), pack(v, t)
    dq, out = torch.from_numpy(q).cuda(), torch.zeros(m, heads, hd, device="cuda")
    check_hip(hip.uaii_hip_attention_prompt(ptr(dq), I64(heads * hd), I64(m), ptr(kc), ptr(vc), t, I64(m), I64(0), I64(0), None, heads, kv, hd,
                                            None, ptr(out), I64(heads * hd), None))
    got = out.cpu().numpy()
    assert np.isfinite(got[:50, :2]).all() and np.isfinite(got[:70, 2:]).all()
    assert not np.isfinite(got[50:, :2, 3]).any() and not np.isfinite(got[70:, 2:, 9]).any() and np.isnan(got[90:, 2:]).all()


@pytest.mark.parametrize("t", TYPES, ids=NAMES.get)
@pytest.mark.parametrize("shape", [(32, 8, 128), (8, 8, 64)], ids=str)
def test_prompt_long(hip, t, shape):
    """Blocks of every kind of a longer prompt; some rows are checked."""
    check_prompt(hip, np.random.default_rng(17), t, *shape, m=1100, p0=500, window=700, which=[0, 1, 199, 200, 201, 555, 1023, 1024, 1099])
    check_prompt(hip, np.random.default_rng(18), t, *shape, m=40, p0=6000, which=[0, 7, 39])


# (shape, rows, position of the first): one, two and four row waves, with and without splits
KINDS = [((32, 8, 64), 346, 325), ((8, 4, 64), 1351, 20), ((1, 1, 128), 1, 281), ((16, 4, 128), 680, 777), ((8, 8, 128), 1500, 0),
         ((32, 8, 128), 1700, 3), ((1, 1, 256), 1, 264), ((4, 2, 256), 359, 110), ((4, 4, 256), 387, 144), ((16, 8, 256), 900, 0)]


@pytest.mark.parametrize("t", TYPES, ids=NAMES.get)
@pytest.mark.parametrize("shape,m,p0", KINDS, ids=str)
def test_prompt_kinds(hip, t, shape, m, p0):
    which = sorted({0, m // 3, m // 2, max(m - 40, 0), m - 1} | set(range(31, m, 97)))
    check_prompt(hip, np.random.default_rng(34), t, *shape, m=m, p0=p0, which=which)
    check_prompt(hip, np.random.default_rng(35), t, *shape, m=m, p0=p0, which=which[::2], cap=8.0, slopes=True, window=max(m // 2, 3),
                 bidir=p0 + m // 4, first=[max(0, p0 + i - 300 + 150 * (i % 3)) for i in range(m)], spread=3.0)


@pytest.mark.parametrize("t", TYPES, ids=NAMES.get)
@pytest.mark.parametrize("shape,m", [((8, 8, 128), 1500), ((32, 8, 64), 700), ((16, 8, 256), 900)], ids=str)
def test_prompt_documents_of_many(hip, t, shape, m):
    """Documents whose values are not finite, next to others, in blocks of four row waves."""
    ends = [0, m // 5, m // 5 + 130, m // 2, m // 2 + 1, m]
    first = np.concatenate([np.full(b - a, a) for a, b in zip(ends, ends[1:])])
    bad = slice(ends[1], ends[2])
    first[bad] = 1 << 30
    which = [i for i in range(0, m, 53)] + [ends[1] - 1, ends[1], ends[2] - 1, ends[2], ends[3] - 1, ends[3], ends[4], m - 1]
    check_prompt(hip, np.random.default_rng(36), t, *shape, m=m, p0=0, first=first.tolist(), poison=bad, which=sorted(set(which)))


def test_prompt_scale_not_finite(hip):
    """An 8-bit row with a scale of infinity reaches the queries that see it and no others."""
    rng = np.random.default_rng(19)
    heads, kv, hd, m = 4, 2, 64, 100
    (kc, _), (vc, _) = (pack(rows(rng, 1, kv, m, hd), KV_Q8) for _ in range(2))
    scales = vc[0, kv * m * hd : kv * m * (hd + 4)].view(torch.float32)
    scales[50] = math.inf
    dq, out = torch.from_numpy(rows(rng, m, heads * hd)).cuda(), torch.zeros(m, heads, hd, device="cuda")
    check_hip(hip.uaii_hip_attention_prompt(ptr(dq), I64(heads * hd), I64(m), ptr(kc), ptr(vc), KV_Q8, I64(m), I64(0), I64(0), None, heads, kv,
                                            hd, None, ptr(out), I64(heads * hd), None))
    got = out.cpu().numpy()
    assert np.isfinite(got[:50]).all() and np.isfinite(got[:, 2:]).all() and not np.isfinite(got[50:, :2]).any()


# ---- the largest offsets, streams, graphs, and all of it together --------------------------------


@pytest.mark.parametrize("t,seq", [(KV_F32, 1 << 21), (KV_F16, 1 << 22), (KV_Q8, 1 << 23)], ids=["f32", "f16", "q8"])
def test_offsets_past_32_bits(hip, t, seq):
    """Two heads' caches of a GiB each, six sequences' worth of bytes: equal scores, so that the
    result is the mean of values that stand at the far end."""
    kv, hd, n = 2, 128, 3
    size = seq_bytes(t, kv, seq, hd)
    assert size * n > 1 << 32
    kc, vc = (torch.zeros(n * size, dtype=torch.uint8, device="cuda") for _ in range(2))
    if t == KV_Q8:  # bytes of zero with a scale of zero are zeros
        assert int(kc[0]) == 0
    m = 1000
    ones = torch.ones(n * m, kv * hd, device="cuda") * torch.arange(1, n + 1, device="cuda").repeat_interleave(m).view(-1, 1)
    lens = torch.tensor([seq - m, seq - m, seq - m], dtype=torch.int32, device="cuda")
    zero = torch.zeros_like(ones)
    place = [t, I64(n), I64(m), kv, hd, I64(seq), I64(0), ptr(lens)]
    check_hip(hip.uaii_hip_kv_append_batch(ptr(zero), ptr(ones), I64(kv * hd), ptr(kc), ptr(vc), *place, None))
    back = torch.zeros_like(ones)
    check_hip(hip.uaii_hip_kv_read(ptr(vc), *place, ptr(back), I64(kv * hd), None))
    assert torch.equal(back, ones)
    q, out = torch.randn(n, 4 * hd, device="cuda"), torch.zeros(n, 4 * hd, device="cuda")
    full = torch.full((n,), seq, dtype=torch.int32, device="cuda")
    check_hip(hip.uaii_hip_attention_batch(ptr(q), I64(4 * hd), I64(n), ptr(kc), ptr(vc), t, I64(seq), ptr(full), None, None, I64(0), I64(0),
                                           4, kv, hd, None, ptr(out), I64(4 * hd), None))
    want = torch.arange(1, n + 1, device="cuda").double().view(-1, 1) * m / seq
    assert float(((out.double() - want) / want).abs().max()) < 2.0 ** -17  # 64 u of the sums, and to spare
    # the last sequence's cache as a prefix, and under a prompt's rows in its window
    last = ctypes.c_void_p(kc.data_ptr() + (n - 1) * size), ctypes.c_void_p(vc.data_ptr() + (n - 1) * size)
    short = torch.zeros(n * seq_bytes(t, kv, 16, hd), dtype=torch.uint8, device="cuda")
    none = torch.zeros(n, dtype=torch.int32, device="cuda")
    check_hip(hip.uaii_hip_attention_batch(ptr(q), I64(4 * hd), I64(n), ptr(short), ptr(short), t, I64(16), ptr(none), *last, I64(seq), I64(seq),
                                           4, kv, hd, None, ptr(out), I64(4 * hd), None))
    assert float((out.double() / (n * m / seq) - 1).abs().max()) < 2.0 ** -17
    opt = options(window=2 * m)
    check_hip(hip.uaii_hip_attention_prompt(ptr(q), I64(4 * hd), I64(n), *last, t, I64(seq), I64(seq - n), I64(0), None, 4, kv, hd,
                                            ctypes.byref(opt), ptr(out), I64(4 * hd), None))
    seen = torch.tensor([m - 2, m - 1, m], device="cuda").double().view(-1, 1) * n / (2 * m)
    assert float((out.double() / seen - 1).abs().max()) < 2.0 ** -17


def test_streams(hip):
    """Calls on six streams and the null stream at once give the bits of the same calls alone."""
    made = [run_batch(hip, np.random.default_rng(20 + i), [KV_Q8, KV_F16][i % 2], 8, 2, 64, lens=[700 + i, 3, 50], seq=800, prefix=64 * i)
            for i in range(7)]
    want, outs = [], []
    for call, _, _ in made:
        out, _ = call(None)
        torch.cuda.synchronize()
        want.append(out.clone())
        outs.append(out.fill_(-7.0))
    streams = [torch.cuda.Stream() for _ in range(6)]
    torch.cuda.synchronize()
    for _ in range(4):
        for i, (call, _, _) in enumerate(made):
            call(ctypes.c_void_p(streams[i].cuda_stream) if i < 6 else None)
    torch.cuda.synchronize()
    for out, w in zip(outs, want):
        assert torch.equal(out, w)


def test_serving_run(hip):
    """A prompt's rows into a cache, its attention, then steps of a batch that shares it: each step's
    rows are appended where the last ended, and attended; on a stream, eagerly and as one graph whose
    lengths move between replays."""
    rng = np.random.default_rng(30)
    heads, kv, hd, m, n, seq, steps = 8, 2, 64, 130, 3, 40, 5
    g, t, width = heads // kv, KV_Q8, kv * hd
    pk, pv, pq = rows(rng, m, width), rows(rng, m, width), rows(rng, m, heads * hd)
    sk, sv, sq = rows(rng, steps, n, width), rows(rng, steps, n, width), rows(rng, steps, n, heads * hd)
    stream = torch.cuda.Stream()
    raw = ctypes.c_void_p(stream.cuda_stream)
    dev = lambda x: torch.from_numpy(x).cuda()  # noqa: E731
    new = lambda c, s: torch.zeros(c * seq_bytes(t, kv, s, hd), dtype=torch.uint8, device="cuda")  # noqa: E731
    kpc, vpc = new(1, m), new(1, m)
    dpk, dpv, dpq, pout = dev(pk), dev(pv), dev(pq), torch.zeros(m, heads * hd, device="cuda")
    torch.cuda.synchronize()
    check_hip(hip.uaii_hip_kv_append_batch(ptr(dpk), ptr(dpv), I64(width), ptr(kpc), ptr(vpc), t, I64(1), I64(m), kv, hd, I64(m), I64(0), None, raw))
    check_hip(hip.uaii_hip_attention_prompt(ptr(dpq), I64(heads * hd), I64(m), ptr(kpc), ptr(vpc), t, I64(m), I64(0), I64(0), None, heads, kv, hd,
                                            None, ptr(pout), I64(heads * hd), raw))
    stream.synchronize()
    _, kx = pack(pk.reshape(1, m, kv, hd).transpose(0, 2, 1, 3), t)
    _, vx = pack(pv.reshape(1, m, kv, hd).transpose(0, 2, 1, 3), t)
    sc = float(np.float32(1 / math.sqrt(hd)))
    at = np.arange(m)
    for h in range(heads):
        w, tol = attend(pq[:, h * hd : (h + 1) * hd], kx[0, h // g], vx[0, h // g], at, at, np.zeros(m), at + 1, sc, 0.0, 0.0)
        close(pout.cpu().numpy()[:, h * hd : (h + 1) * hd], w, tol)

    start = torch.tensor([0, 4, 30], dtype=torch.int32, device="cuda")  # sequences that are at different places
    kin, vin, qin = dev(sk[0]), dev(sv[0]), dev(sq[0])

    def made():
        return {"kc": new(n, seq), "vc": new(n, seq), "past": start.clone(), "lens": start + 1, "out": torch.zeros(n, heads * hd, device="cuda")}

    def step(state, s):
        check_hip(hip.uaii_hip_kv_append_batch(ptr(kin), ptr(vin), I64(width), ptr(state["kc"]), ptr(state["vc"]), t, I64(n), I64(1), kv, hd,
                                               I64(seq), I64(0), ptr(state["past"]), s))
        check_hip(hip.uaii_hip_attention_batch(ptr(qin), I64(heads * hd), I64(n), ptr(state["kc"]), ptr(state["vc"]), t, I64(seq),
                                               ptr(state["lens"]), ptr(kpc), ptr(vpc), I64(m), I64(m), heads, kv, hd, None,
                                               ptr(state["out"]), I64(heads * hd), s))

    eager, graphed = made(), made()
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=torch.cuda.Stream()):
        step(graphed, ctypes.c_void_p(torch.cuda.current_stream().cuda_stream))
    torch.cuda.synchronize()
    empty = np.zeros((n, seq, kv, hd), np.float32)
    ks, vs = empty.copy(), empty.copy()
    first = [0, 4, 30]
    for i in range(steps):
        kin.copy_(dev(sk[i])), vin.copy_(dev(sv[i])), qin.copy_(dev(sq[i]))
        torch.cuda.synchronize()
        step(eager, raw)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(eager["out"], graphed["out"])
        assert torch.equal(eager["kc"], graphed["kc"]) and torch.equal(eager["vc"], graphed["vc"])
        for s in range(n):
            ks[s, first[s] + i], vs[s, first[s] + i] = sk[i, s].reshape(kv, hd), sv[i, s].reshape(kv, hd)
        _, k1 = pack(ks.transpose(0, 2, 1, 3).copy(), t)
        _, v1 = pack(vs.transpose(0, 2, 1, 3).copy(), t)
        got = eager["out"].cpu().numpy()
        for s in range(n):
            held = first[s] + i + 1
            at = np.arange(m + held)
            for h in range(heads):
                kk, vv = (np.concatenate([a[0, h // g], b[s, h // g, :held]]) for a, b in ((kx, k1), (vx, v1)))
                w, tol = attend(sq[i, s : s + 1, h * hd : (h + 1) * hd], kk, vv, at, at[-1:], np.array([0]), at[-1:] + 1, sc, 0.0, 0.0)
                close(got[s : s + 1, h * hd : (h + 1) * hd], w, tol)
        for state in (eager, graphed):
            state["past"] += 1
            state["lens"] += 1
        torch.cuda.synchronize()


@pytest.mark.parametrize("t", TYPES, ids=NAMES.get)
def test_graph_of_large_calls(hip, t):
    """Units in shares, a shared prefix and split prompt rows in one graph, replayed with other lengths
    and queries between eager calls: the same bits as those."""
    rng = np.random.default_rng(40)
    heads, kv, hd, n, seq, prefix, m = 8, 4, 64, 70, 1100, 900, 30
    width = heads * hd
    new = lambda *shape: torch.randn(*shape, device="cuda", generator=gen)  # noqa: E731
    gen = torch.Generator(device="cuda").manual_seed(7)
    size, psize = seq_bytes(t, kv, seq, hd), seq_bytes(t, kv, prefix, hd)
    kc, vc = (torch.zeros(n * size, dtype=torch.uint8, device="cuda") for _ in range(2))
    kp, vp = (torch.zeros(psize, dtype=torch.uint8, device="cuda") for _ in range(2))
    for k, v, s, count, to in ((kc, vc, seq, n, seq), (kp, vp, prefix, 1, prefix)):
        a, b = new(count * to, kv * hd), new(count * to, kv * hd)
        check_hip(hip.uaii_hip_kv_append_batch(ptr(a), ptr(b), I64(kv * hd), ptr(k), ptr(v), t, I64(count), I64(to), kv, hd, I64(s), I64(0),
                                               None, None))
        torch.cuda.synchronize()
    q, lens = new(n, width), torch.zeros(n, dtype=torch.int32, device="cuda")
    outs = [[torch.zeros(n, width, device="cuda"), torch.zeros(n, width, device="cuda"), torch.zeros(m, width, device="cuda")] for _ in range(2)]

    def calls(to, stream):
        for out, pre in ((to[0], 0), (to[1], prefix)):
            check_hip(hip.uaii_hip_attention_batch(ptr(q), I64(width), I64(n), ptr(kc), ptr(vc), t, I64(seq), ptr(lens), ptr(kp), ptr(vp),
                                                   I64(prefix), I64(pre), heads, kv, hd, None, ptr(out), I64(width), stream))
        check_hip(hip.uaii_hip_attention_prompt(ptr(q), I64(width), I64(m), ptr(kc), ptr(vc), t, I64(seq), I64(seq - m), I64(0), None, heads, kv,
                                                hd, None, ptr(to[2]), I64(width), stream))

    calls(outs[0], None)
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=torch.cuda.Stream()):
        calls(outs[1], ctypes.c_void_p(torch.cuda.current_stream().cuda_stream))
    torch.cuda.synchronize()
    for i in range(4):
        lens.copy_(torch.from_numpy(rng.integers(0, [5, seq, 1, seq][i] + 1, n).astype(np.int32)))
        q.copy_(new(n, width))
        for o in outs[0] + outs[1]:
            o.fill_(-7.0)
        torch.cuda.synchronize()
        calls(outs[0], None)
        graph.replay()
        calls(outs[0], None)
        torch.cuda.synchronize()
        for a, b in zip(*outs):
            assert torch.equal(a, b) and torch.isfinite(a).all()
    assert float(outs[0][1].abs().max()) > 0


def test_threads(hip):
    """Calls from four threads, each on a stream of its own, give the bits of the same calls alone."""
    made = [run_batch(hip, np.random.default_rng(50 + i), TYPES[i % 3], 8, 2, 64, lens=[(97 * j) % 400 for j in range(30)], seq=400, prefix=[0, 700][i % 2])
            for i in range(4)]
    want, outs = [], []
    for call, _, _ in made:
        out, _ = call(None)
        torch.cuda.synchronize()
        want.append(out.clone())
        outs.append(out.fill_(-7.0))
    streams = [torch.cuda.Stream() for _ in made]
    torch.cuda.synchronize()
    failed = []

    def work(i):
        try:
            for _ in range(20):
                made[i][0](ctypes.c_void_p(streams[i].cuda_stream))
        except Exception as e:  # noqa: BLE001
            failed.append(e)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(len(made))]
    for th in threads:
        th.start()
    for th in threads:
        th.join()
    torch.cuda.synchronize()
    assert not failed
    for out, w in zip(outs, want):
        assert torch.equal(out, w)
