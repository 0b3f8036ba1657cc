"""Operators of the caches that serve a batch: their plain forms and the library's calls.

  kv        K and V rows written into the caches of a batch and read back (f32, f16 or
            8-bit caches);
  batch     attention of one query per sequence over the sequence's own keys, and over a
            prefix that all sequences share;
  prompt    attention of a run of prompt positions, causal or with a prefix that every
            query sees, over one document or several packed ones.

Scores may be capped by a tanh, biased by the distance of query and key, and cut to a
window. Queries and outputs are f32. A cache is head-major, [n_kv_heads][max_seq][head_dim];
an 8-bit one holds the bytes q + 128 there and one f32 scale for each head's row behind
them ([n_kv_heads][max_seq]), a row's values being q * scale with scale = max |x| / 127.
A batch's caches lie one behind the other.
"""
from __future__ import annotations

import ctypes
import math
import sys
from pathlib import Path

import torch

own = False

KV_TYPE = {"f32": 0, "f16": 1, "q8": 2}


# ---- the cases ---------------------------------------------------------------------------


def listed():
    return [
        # a decode step of a small model for a few users: the call and the launch
        {"name": "kv_step_q8", "kind": "kv", "type": "q8", "seqs": 8, "rows": 1, "kv": 8, "hd": 64, "past": 500},
        # a long document's rows of one layer of the 8B shape
        {"name": "kv_prompt_q8", "kind": "kv", "type": "q8", "seqs": 1, "rows": 4001, "kv": 8, "hd": 128, "past": 0},
        # chunks of several prompts at once into f16 caches, heads of an odd width
        {"name": "kv_chunks_f16", "kind": "kv", "type": "f16", "seqs": 6, "rows": 500, "kv": 4, "hd": 80, "past": 300},
        # one user's first tokens on a small model
        {"name": "batch_one_q8", "kind": "batch", "type": "q8", "seqs": 1, "heads": 8, "kv": 8, "hd": 64, "keys": 37,
         "ragged": False, "idle": 0, "prefix": 0, "cap": 0.0, "slopes": False, "window": 0},
        # a full batch of long chats on the 8B shape
        {"name": "batch_chats_q8", "kind": "batch", "type": "q8", "seqs": 32, "heads": 32, "kv": 8, "hd": 128, "keys": 8000,
         "ragged": True, "idle": 1, "prefix": 0, "cap": 0.0, "slopes": False, "window": 0},
        # a local layer of a model with wide heads, capped scores and a window
        {"name": "batch_window_f16", "kind": "batch", "type": "f16", "seqs": 12, "heads": 16, "kv": 8, "hd": 256, "keys": 5003,
         "ragged": True, "idle": 0, "prefix": 0, "cap": 50.0, "slopes": False, "window": 1024},
        # many users of one long system prompt
        {"name": "prefix_users_f16", "kind": "batch", "type": "f16", "seqs": 48, "heads": 32, "kv": 8, "hd": 128, "keys": 400,
         "ragged": True, "idle": 2, "prefix": 6000, "cap": 0.0, "slopes": False, "window": 0},
        # a few answers drawn for one very long question, distances in the scores
        {"name": "prefix_answers_q8", "kind": "batch", "type": "q8", "seqs": 5, "heads": 20, "kv": 4, "hd": 64, "keys": 90,
         "ragged": True, "idle": 0, "prefix": 30011, "cap": 0.0, "slopes": True, "window": 0},
        # a chat turn of a few words on a 1B layer with the f32 cache, distances in the scores
        {"name": "prompt_words_f32", "kind": "prompt", "type": "f32", "m": 33, "p0": 777, "heads": 32, "kv": 8, "hd": 64,
         "cap": 0.0, "slopes": True, "window": 0, "bidir": 0, "docs": 1, "pad": 0},
        # the second chunk of a long prompt, capped scores, a window, the 8-bit cache
        {"name": "prompt_window_q8", "kind": "prompt", "type": "q8", "m": 1003, "p0": 2048, "heads": 32, "kv": 8, "hd": 128,
         "cap": 30.0, "slopes": False, "window": 1500, "bidir": 0, "docs": 1, "pad": 0},
        # packed documents with padding behind them
        {"name": "prompt_docs_f16", "kind": "prompt", "type": "f16", "m": 4096, "p0": 0, "heads": 32, "kv": 8, "hd": 128,
         "cap": 0.0, "slopes": False, "window": 0, "bidir": 0, "docs": 3, "pad": 50},
        # a picture's positions that see each other, then text
        {"name": "prompt_prefix_f16", "kind": "prompt", "type": "f16", "m": 1300, "p0": 0, "heads": 8, "kv": 1, "hd": 256,
         "cap": 0.0, "slopes": False, "window": 0, "bidir": 1024, "docs": 1, "pad": 0},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


HEADS = [(8, 8), (32, 8), (32, 32), (14, 2), (20, 4), (64, 8), (8, 1)]


def draw(rng):
    kind = rng.choice(["kv", "batch", "batch", "batch", "prompt", "prompt"])
    kv_type = rng.choice(["q8", "q8", "f16", "f16", "f32"])
    heads, kv = rng.choice(HEADS)
    hd = rng.choice([32, 64, 64, 80, 112, 128, 128, 256])
    if kind == "kv":
        seqs = _log(rng, 1, 64)
        rows = 1 if rng.random() < 0.4 else _log(rng, 1, max(2, min(4000, 4e6 / (seqs * kv * hd))))
        return {"kind": kind, "type": kv_type, "seqs": seqs, "rows": rows, "kv": kv, "hd": hd, "past": rng.choice([0, _log(rng, 1, 800)])}
    c = {"kind": kind, "type": kv_type, "heads": heads, "kv": kv, "hd": hd, "cap": rng.choice([0.0, 0.0, 30.0, 50.0]),
         "slopes": rng.random() < 0.25, "window": 0 if rng.random() < 0.7 else _log(rng, 1, 3000)}
    wide = kv * hd * {"f32": 4, "f16": 2, "q8": 1}[kv_type] * 2  # bytes of one position's keys and values
    if kind == "batch":
        seqs = _log(rng, 1, 64)
        c |= {"seqs": seqs, "keys": _log(rng, 1, max(2, min(12000, 2.5e8 / (seqs * wide)))), "ragged": rng.random() < 0.7,
              "idle": rng.choice([0, 0, 1]),
              "prefix": 0 if rng.random() < 0.5 else _log(rng, 1, min(30000, 2e8 / wide, 2.5e9 / (seqs * heads * hd)))}
        return c
    p0 = rng.choice([0, _log(rng, 1, 4000)])
    pairs = 5e10 / (4 * heads * hd)
    m = _log(rng, 1, max(2, min(2500, (math.sqrt(p0 * p0 + 4 * pairs) - p0) / 2)))
    c |= {"m": m, "p0": p0, "bidir": 0 if rng.random() < 0.7 else rng.randint(1, p0 + m), "docs": rng.choice([1, 1, 3, 6]),
          "pad": rng.choice([0, 0, min(m - 1, 20)])}
    return c


def _spread(i):
    """Numbers in [0, 1) that fill it evenly."""
    return (0.35 + i * 0.6180339887498949) % 1.0


def _lengths(case):
    """Keys that each sequence of a batch holds itself; idle places at its end hold none."""
    n, keys, busy = case["seqs"], case["keys"], max(1, case["seqs"] - case["idle"])
    return [0 if i >= busy else max(1, round(keys * (0.1 + 0.9 * _spread(i)))) if case["ragged"] else keys for i in range(n)]


def _first_keys(case):
    """First key that each row of a prompt may see: its document's, or one behind all for padding."""
    m, p0 = case["m"], case["p0"]
    starts = [0] + [p0 + int(m * _spread(i)) for i in range(case["docs"] - 1)]
    return [max(s for s in starts if s <= p0 + i) if i < m - case["pad"] else p0 + m for i in range(m)]


# ---- inputs ---------------------------------------------------------------------------------


def _gen(seed, stream):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed * 64 + stream)
    return g


def _rows(seed, stream, *shape, outliers=False):
    """Rows as a layer makes them: N(0, 1), for keys with a few channels of larger size."""
    x = torch.randn(*shape, generator=_gen(seed, stream), device="cuda")
    if outliers:
        x *= torch.randn(shape[-1], generator=_gen(seed, stream + 1), device="cuda").mul_(0.4).exp_()
    return x


def _quantise(x):
    """8-bit rows of the last axis and their scales; quotients in 64 bits, next to a border of two steps."""
    d = (x.abs().amax(-1).double() / torch.full((), 127.0, dtype=torch.float64, device=x.device)).float()
    q = x.double() / d.double().unsqueeze(-1)
    q = torch.where(d.unsqueeze(-1) > 0, q, torch.zeros_like(q)).round_().clamp_(-127, 127)
    return q.add_(128).to(torch.uint8), d


def _pack(x, kv_type):
    """A batch's cache [n, kv, max_seq, hd] as the bytes [n, bytes of a sequence]."""
    n = x.shape[0]
    if kv_type != "q8":
        x = x if kv_type == "f32" else x.half()
        return x.contiguous().view(torch.uint8).reshape(n, -1)
    q, d = _quantise(x)
    side = d.reshape(n, -1).contiguous().view(torch.uint8)
    out = torch.zeros(n, _seq_bytes(kv_type, x.shape[1], x.shape[2], x.shape[3]), dtype=torch.uint8, device=x.device)
    out[:, :q[0].numel()] = q.reshape(n, -1)
    out[:, q[0].numel():q[0].numel() + side.shape[1]] = side
    return out


def _unpack(cache, kv_type, kv, max_seq, hd):
    """The values of a batch's cache, [n, kv, max_seq, hd] in f32."""
    n, count = cache.shape[0], kv * max_seq * hd
    if kv_type == "q8":
        d = cache[:, count:count + 4 * kv * max_seq].contiguous().view(torch.float32).reshape(n, kv, max_seq, 1)
        return (cache[:, :count].reshape(n, kv, max_seq, hd).float() - 128) * d
    x = cache.view(torch.float16 if kv_type == "f16" else torch.float32)
    return x.reshape(n, kv, max_seq, hd).float()


def _seq_bytes(kv_type, kv, max_seq, hd):
    """Bytes of one sequence's K (or V)."""
    if kv_type == "q8":
        return (kv * max_seq * (hd + 4) + 15) // 16 * 16
    return kv * max_seq * hd * (2 if kv_type == "f16" else 4)


def _room(keys):
    return max(256, (keys + 255) // 256 * 256)


def _kv_inputs(case, seed):
    n, rows, kv, hd = case["seqs"], case["rows"], case["kv"], case["hd"]
    past = [round(case["past"] * _spread(i)) for i in range(n)]
    k = _rows(seed, 1, n * rows, kv * hd, outliers=True)
    v = _rows(seed, 3, n * rows, kv * hd)
    return k, v, past, _room(case["past"] + rows)


def _slopes(case):
    h = case["heads"]
    return torch.tensor([2.0 ** (-8.0 * (i + 1) / h) for i in range(h)], device="cuda") if case["slopes"] else None


def _batch_inputs(case, seed):
    n, heads, kv, hd, prefix = (case[x] for x in ("seqs", "heads", "kv", "hd", "prefix"))
    max_seq, pre_seq = _room(case["keys"]), _room(prefix)
    t = {"q": _rows(seed, 1, n, heads * hd).mul_(1.5), "lens": _lengths(case), "max_seq": max_seq, "pre_seq": pre_seq}
    t["k"] = _rows(seed, 2, n, kv, max_seq, hd, outliers=True)
    t["v"] = _rows(seed, 4, n, kv, max_seq, hd)
    if prefix:
        t["kp"] = _rows(seed, 5, 1, kv, pre_seq, hd, outliers=True)
        t["vp"] = _rows(seed, 7, 1, kv, pre_seq, hd)
    return t


def _prompt_inputs(case, seed):
    max_seq = _room(case["p0"] + case["m"])
    t = {"q": _rows(seed, 1, case["m"], case["heads"] * case["hd"]).mul_(1.5), "max_seq": max_seq, "first": _first_keys(case)}
    t["k"] = _rows(seed, 2, 1, case["kv"], max_seq, case["hd"], outliers=True)
    t["v"] = _rows(seed, 4, 1, case["kv"], max_seq, case["hd"])
    return t


def prepare(case, seed):
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    if case["kind"] == "kv":
        k, v, past, max_seq = _kv_inputs(case, seed)
        empty = torch.zeros(case["seqs"], _seq_bytes(case["type"], case["kv"], max_seq, case["hd"]), dtype=torch.uint8, device="cuda")
        return {"case": case, "k": k, "v": v, "past": i32(past), "max_seq": max_seq, "kc": empty, "vc": empty.clone(),
                "k_back": torch.empty_like(k), "v_back": torch.empty_like(v)}
    t = (_batch_inputs if case["kind"] == "batch" else _prompt_inputs)(case, seed)
    s = {"case": case, "q": t["q"], "max_seq": t["max_seq"], "slopes": _slopes(case), "out": torch.empty_like(t["q"])}
    s["kc"], s["vc"] = _pack(t["k"], case["type"]), _pack(t["v"], case["type"])
    if case["kind"] == "prompt":
        packed = case["docs"] > 1 or case["pad"] > 0
        return s | {"first": i32(t["first"]) if packed else None}
    s |= {"lens": i32(t["lens"]), "pre_seq": t["pre_seq"]}
    if case["prefix"]:
        s["kp"], s["vp"] = _pack(t["kp"], case["type"]), _pack(t["vp"], case["type"])
    return s


# ---- the plain forms --------------------------------------------------------------------------


def _scores(dot, case, slopes, distance):
    """Scores of query heads [..., kv, G, (rows,) keys] from the scaled products."""
    if case["cap"]:
        dot = case["cap"] * torch.tanh(dot / case["cap"])
    return dot if slopes is None else dot - slopes * distance


def _weights(s, seen):
    """Softmax over the last axis of what is seen, and zeros in rows that see nothing."""
    s = torch.where(seen, s, torch.full_like(s, -math.inf))
    top = s.amax(-1, keepdim=True)
    e = torch.exp(s - torch.where(top > -math.inf, top, torch.zeros_like(top)))
    total = e.sum(-1, keepdim=True)
    return e / torch.where(total > 0, total, torch.ones_like(total))


def _plain_batch(st):
    case, n, kv, hd, pre = st["case"], st["case"]["seqs"], st["case"]["kv"], st["case"]["hd"], st["case"]["prefix"]
    g = case["heads"] // kv
    q = st["q"].view(n, kv, g, hd) * (1.0 / math.sqrt(hd))
    k, v = (_unpack(st[x], case["type"], kv, st["max_seq"], hd) for x in ("kc", "vc"))
    dot = q @ k.transpose(-1, -2).contiguous()
    lens = st["lens"].view(n, 1, 1, 1)
    own_at = torch.arange(st["max_seq"], device=q.device)
    seen = (own_at < lens).expand(n, 1, 1, -1)
    at = own_at + pre
    if pre:
        kp, vp = (_unpack(st[x], case["type"], kv, st["pre_seq"], hd)[0, :, :pre] for x in ("kp", "vp"))
        qp = q.transpose(0, 1).reshape(kv, n * g, hd)
        dp = (qp @ kp.transpose(-1, -2).contiguous()).view(kv, n, g, pre).transpose(0, 1)
        dot = torch.cat([dp, dot], -1)
        seen = torch.cat([torch.ones(n, 1, 1, pre, dtype=torch.bool, device=q.device), seen], -1)
        at = torch.cat([torch.arange(pre, device=q.device), at])
    back = (pre + lens - 1) - at
    if case["window"]:
        seen = seen & (back < case["window"])
    slopes = None if st["slopes"] is None else st["slopes"].view(1, kv, g, 1)
    p = _weights(_scores(dot, case, slopes, back.abs().float()), seen)
    out = p[..., pre:].contiguous() @ v
    if pre:
        pp = p[..., :pre].transpose(0, 1).reshape(kv, n * g, pre)
        out = out + (pp @ vp.contiguous()).view(kv, n, g, hd).transpose(0, 1)
    return out.reshape(n, -1)


def _plain_prompt(st):
    case, m, p0, kv, hd = st["case"], st["case"]["m"], st["case"]["p0"], st["case"]["kv"], st["case"]["hd"]
    g, keys = case["heads"] // kv, p0 + m
    q = (st["q"].view(m, kv, g, hd) * (1.0 / math.sqrt(hd))).permute(1, 2, 0, 3).reshape(kv, g * m, hd)
    k, v = (_unpack(st[x], case["type"], kv, st["max_seq"], hd)[0, :, :keys] for x in ("kc", "vc"))
    dot = (q @ k.transpose(-1, -2).contiguous()).view(kv, g, m, keys)
    at = torch.arange(keys, device=q.device)
    pos = torch.arange(p0, keys, device=q.device).view(m, 1)
    seen = (at <= pos) | (at < case["bidir"])
    if case["window"]:
        seen = seen & (at > pos - case["window"])
    if st["first"] is not None:
        seen = seen & (at >= st["first"].view(m, 1))
    slopes = None if st["slopes"] is None else st["slopes"].view(kv, g, 1, 1)
    p = _weights(_scores(dot, case, slopes, (pos - at).abs().float()), seen)
    out = p.view(kv, g * m, keys) @ v.contiguous()
    return out.view(kv, g, m, hd).permute(2, 0, 1, 3).reshape(m, -1)


def _plain_kv(st):
    case, n, rows, kv, hd = st["case"], st["case"]["seqs"], st["case"]["rows"], st["case"]["kv"], st["case"]["hd"]
    # places [seqs, kv, rows] of the written rows, counted in rows of a sequence's cache
    at = st["past"].long().view(n, 1, 1) + torch.arange(rows, device=st["k"].device)
    at = (at + torch.arange(kv, device=st["k"].device).view(1, kv, 1) * st["max_seq"]).reshape(n, kv * rows, 1)
    return {"k": _plain_write_read(st["k"], st["kc"], at, case, st["max_seq"]),
            "v": _plain_write_read(st["v"], st["vc"], at, case, st["max_seq"])}


def _plain_write_read(x, cache, at, case, max_seq):
    n, rows, kv, hd, kv_type = case["seqs"], case["rows"], case["kv"], case["hd"], case["type"]
    x = x.view(n, rows, kv, hd).transpose(1, 2).reshape(n, kv * rows, hd)
    count, index = kv * max_seq * hd, at.expand(n, kv * rows, hd)
    if kv_type == "q8":
        q, d = _quantise(x)
        values = cache[:, :count].view(n, kv * max_seq, hd)
        scales = cache[:, count:count + 4 * kv * max_seq].view(torch.float32)
        values.scatter_(1, index, q)
        scales.scatter_(1, at[:, :, 0], d)
        back = (values.gather(1, index).float() - 128) * scales.gather(1, at[:, :, 0]).unsqueeze(-1)
    else:
        dtype = torch.float16 if kv_type == "f16" else torch.float32
        values = cache.view(dtype).view(n, kv * max_seq, hd)
        values.scatter_(1, index, x.to(dtype))
        back = values.gather(1, index).float()
    return back.view(n, kv, rows, hd).transpose(1, 2).reshape(n * rows, kv * hd)


# ---- the library's calls ------------------------------------------------------------------------

_ready = []


def _library():
    if not _ready:
        sys.path.insert(0, str(Path(__file__).resolve().parent.parent / "universal-ai-inference_amd"))
        import uaii_amd
        uaii_amd.check_hip(uaii_amd.lib().uaii_hip_init(torch.cuda.current_device()), "init")
        _ready.append(uaii_amd)
    return _ready[0]


def _p(t):
    return None if t is None else ctypes.c_void_p(t.data_ptr())


def _call(st):
    """The pass's calls: (function, arguments) each, made once a state as a program keeps them."""
    uaii = _library()
    L, c, i64 = uaii.lib(), st["case"], ctypes.c_int64
    kv_type, stream = KV_TYPE[c["type"]], None
    if c["kind"] == "kv":
        width = c["kv"] * c["hd"]
        place = [kv_type, i64(c["seqs"]), i64(c["rows"]), c["kv"], c["hd"], i64(st["max_seq"]), i64(0), _p(st["past"])]
        return [(L.uaii_hip_kv_append_batch, [_p(st["k"]), _p(st["v"]), i64(width), _p(st["kc"]), _p(st["vc"]), *place, stream]),
                (L.uaii_hip_kv_read, [_p(st["kc"]), *place, _p(st["k_back"]), i64(width), stream]),
                (L.uaii_hip_kv_read, [_p(st["vc"]), *place, _p(st["v_back"]), i64(width), stream])], {"k": st["k_back"], "v": st["v_back"]}
    width = c["heads"] * c["hd"]
    opts = uaii.ScoreOptions(softcap=c["cap"], slopes=_p(st["slopes"]), window=c["window"])
    shape = [c["heads"], c["kv"], c["hd"], ctypes.byref(opts)]
    caches = [_p(st["kc"]), _p(st["vc"]), kv_type, i64(st["max_seq"])]
    if c["kind"] == "batch":
        pre = [_p(st.get("kp")), _p(st.get("vp")), i64(st["pre_seq"]), i64(c["prefix"])]
        call = L.uaii_hip_attention_batch, [_p(st["q"]), i64(width), i64(c["seqs"]), *caches, _p(st["lens"]), *pre, *shape,
                                            _p(st["out"]), i64(width), stream]
    else:
        call = L.uaii_hip_attention_prompt, [_p(st["q"]), i64(width), i64(c["m"]), *caches, i64(c["p0"]), i64(c["bidir"]),
                                             _p(st["first"]), *shape, _p(st["out"]), i64(width), stream]
    return [call], st["out"]


def run(state):
    if not own:
        return {"kv": _plain_kv, "batch": _plain_batch, "prompt": _plain_prompt}[state["case"]["kind"]](state)
    if "calls" not in state:
        state["calls"], state["result"] = _call(state)
    for call, args in state["calls"]:
        rc = call(*args)
        if rc:
            _library().check_hip(rc, "run")
    return state["result"]


# ---- what a pass cannot do without -------------------------------------------------------------


def work(case):
    width = case["kv"] * case["hd"]
    at = width * {"f32": 4, "f16": 2, "q8": 1}[case["type"]] + (4 * case["kv"] if case["type"] == "q8" else 0)  # of a cached row
    if case["kind"] == "kv":
        n = case["seqs"] * case["rows"]
        return {"bytes": 2 * n * (8 * width + at), "flops": 4 * n * width}  # rows in and back, and into the cache
    lo_hi = []
    if case["kind"] == "batch":
        rows, pre = case["seqs"], case["prefix"]
        lo_hi = [(max(0, pre + n - case["window"]) if case["window"] else 0, pre + n) for n in _lengths(case)]
        keys = max(0, pre - min(lo for lo, _ in lo_hi)) + sum(hi - max(lo, pre) for lo, hi in lo_hi)
    else:
        rows = case["m"]
        for i, first in enumerate(_first_keys(case)):
            pos = case["p0"] + i
            lo = max(first, pos - case["window"] + 1 if case["window"] else 0)
            lo_hi.append((lo, max(lo, pos + 1, case["bidir"])))
        full = [(lo, hi) for lo, hi in lo_hi if hi > lo]
        keys = max(hi for _, hi in full) - min(lo for lo, _ in full)
    pairs = sum(hi - lo for lo, hi in lo_hi)
    return {"bytes": 2 * keys * at + 8 * rows * case["heads"] * case["hd"], "flops": 4 * pairs * case["heads"] * case["hd"]}


# ---- the same in 64 bits -----------------------------------------------------------------------


def _exact_values(x, kv_type):
    """What a cache of the type holds of the rows x, in 64 bits."""
    if kv_type == "f32":
        return x.double()
    if kv_type == "f16":
        return x.half().double()
    x = x.double()
    scale = (x.abs().max(-1, keepdim=True).values / torch.tensor(127.0, dtype=torch.float64, device=x.device)).float().double()
    steps = torch.round(x / scale)  # ties to even; the rows of these cases are not all zero
    return steps * scale


def _exact_head(q, k, v, lo, hi, pos, at, case, slope):
    """Rows q of one head over k, v at positions `at`; row i sees the positions lo[i] .. hi[i] - 1."""
    s = (q @ k.T.contiguous()) / math.sqrt(case["hd"])
    if case["cap"]:
        s = torch.tanh(s / case["cap"]) * case["cap"]
    if slope is not None:
        s = s - slope * (pos[:, None] - at[None, :]).abs()
    hidden = (at[None, :] < lo[:, None]) | (at[None, :] >= hi[:, None])
    p = torch.softmax(s.masked_fill_(hidden, -math.inf), -1)
    return p.nan_to_num_(0.0) @ v  # a row that sees nothing


def exact(case, seed):
    kv_type, kv, hd = case["type"], case["kv"], case["hd"]
    if case["kind"] == "kv":
        k, v, _, _ = _kv_inputs(case, seed)
        return {"k": _exact_values(k.view(-1, kv, hd), kv_type).reshape(k.shape), "v": _exact_values(v.view(-1, kv, hd), kv_type).reshape(v.shape)}
    t = (_batch_inputs if case["kind"] == "batch" else _prompt_inputs)(case, seed)
    heads, slopes, window = case["heads"], _slopes(case), case["window"]
    q = t["q"].double().view(-1, heads, hd)
    out = torch.zeros_like(q)
    far = 1 << 40
    if case["kind"] == "prompt":
        keys = case["p0"] + case["m"]
        at = torch.arange(keys, device="cuda", dtype=torch.float64)
        pos = at[case["p0"]:]
        lo = torch.tensor(t["first"], device="cuda", dtype=torch.float64)
        lo = torch.maximum(lo, pos - (window or far) + 1)
        hi = (pos + 1).clamp(min=case["bidir"])
        for h in range(heads):
            j = h // (heads // kv)
            k, v = (_exact_values(t[x][0, j, :keys], kv_type) for x in ("k", "v"))
            out[:, h] = _exact_head(q[:, h], k, v, lo, hi, pos, at, case, None if slopes is None else slopes[h].double())
        return out.reshape(t["q"].shape)
    pre = case["prefix"]
    for j in range(kv):
        shared = [_exact_values(t[x][0, j, :pre], kv_type) for x in ("kp", "vp")] if pre else None
        for i, n in enumerate(t["lens"]):
            if pre + n == 0:
                continue
            k, v = (_exact_values(t[x][i, j, :n], kv_type) for x in ("k", "v"))
            if pre:
                k, v = torch.cat([shared[0], k]), torch.cat([shared[1], v])
            at = torch.arange(pre + n, device="cuda", dtype=torch.float64)
            pos = at[-1:]
            lo, hi = (pos - (window or far) + 1), pos + 1
            for h in range(j * (heads // kv), (j + 1) * (heads // kv)):
                out[i, h] = _exact_head(q[i:i + 1, h], k, v, lo, hi, pos, at, case, None if slopes is None else slopes[h].double())[0]
    return out.reshape(t["q"].shape)
