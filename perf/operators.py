"""Operators of a serving step whose keys and values live in pages, as cases that can be timed and checked.

  append   CtxDecode.paged_append_dev: the rows of new tokens (per-head RMSNorm,
           rotation by position) into the pages of their streams, queries rotated
           on the way
  attn     CtxDecode.paged_attn_dev: one query token a stream over its pages
  rows     CtxDecode.w8a8_rows_dev: residual addition, norm, int8 activations with
           a scale a row, int8 matrix product, bias / activation / residual

`run` computes them in plain torch, or, where `own` is true, through the
library; `exact` restates them in 64 bits.

The library's calls queue on a stream of their own, which neither waits for
torch's streams nor makes them wait: `prepare` ends when its inputs are there,
and what `run` returns is there once the device has been waited for
(`torch.cuda.synchronize()`, or the context's `synchronize()`).
"""
import math
import os

import torch

own = False

_open = {}


def _package():
    """The library's host module (its directory name is no identifier), the program's one device and op context."""
    if not _open:
        import importlib.util
        import sys
        root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
        spec = importlib.util.spec_from_file_location(
            "xdna_engine", os.path.join(root, "xdna-engine_amd", "xdna_engine.py"))
        xe = importlib.util.module_from_spec(spec)
        sys.modules["xdna_engine"] = xe
        spec.loader.exec_module(xe)
        dev = xe.Device(0)
        _open.update(xe=xe, dev=dev, ctx=xe.CtxDecode(dev))
    return _open["xe"], _open["ctx"]


# ---------------------------------------------------------------------------
# the cases
# ---------------------------------------------------------------------------

def _append(name, streams, rows, first, hq, hkv, hd, page, norm, rope):
    """`rows` new tokens of `streams` streams: one each, or ragged prompts; positions start below `first`."""
    return {"name": name, "kind": "append", "streams": streams, "rows": rows, "first": first, "hq": hq, "hkv": hkv,
            "hd": hd, "page": page, "norm": norm, "rope": rope}


def _attn(name, streams, ctx, spread, hq, hkv, hd, page, window):
    """Lengths of `streams` streams: "full" (all ctx), "late" (ctx / 2 .. ctx), "mixed" (0 .. ctx, a few idle ones)."""
    return {"name": name, "kind": "attn", "streams": streams, "ctx": ctx, "spread": spread, "hq": hq, "hkv": hkv,
            "hd": hd, "page": page, "window": window}


def _rows(name, batch, m, k, norm, add, act, res):
    return {"name": name, "kind": "rows", "batch": batch, "m": m, "k": k, "norm": norm, "add": add, "act": act,
            "res": res}


def listed():
    return [
        # one user's next token in Gemma-3-1B: the smallest call, latency
        _append("append_b1_gqa4x256", 1, 1, 4000, 4, 1, 256, 16, True, True),
        # the next token of 64 users, grouped heads
        _append("append_b64_gqa8x128", 64, 64, 3000, 8, 2, 128, 32, False, True),
        # prompts of different lengths taken in together, Gemma-3-1B's heads
        _append("append_prompts_gqa4x256", 23, 8111, 1, 4, 1, 256, 64, True, True),
        # one short stream (Whisper's self attention): latency
        _attn("attn_b1_448_mha12x64", 1, 448, "full", 12, 12, 64, 16, 0),
        # one very long stream
        _attn("attn_b1_32768_gqa4x256", 1, 32768, "full", 4, 1, 256, 64, 0),
        # many users of Gemma-3-1B in the middle of their answers
        _attn("attn_b64_4096_gqa4x256", 64, 4096, "late", 4, 1, 256, 16, 0),
        # a sliding window over long streams, the pages before it given back
        _attn("attn_b32_window1024_gqa8x128", 32, 16384, "late", 8, 2, 128, 32, 1024),
        # a large server: lengths of every size, idle slots among them
        _attn("attn_b150_mixed8192_gqa16x128", 150, 8192, "mixed", 16, 2, 128, 16, 0),
        # one token through Gemma-3-1B's gate and up projections
        _rows("rows_b1_13824x1152_geglu", 1, 13824, 1152, "rms1p", True, "geglu", False),
        # 64 streams through a square layer, its output onto the residual
        _rows("rows_b64_4096x4096_res", 64, 4096, 4096, "none", False, "none", True),
        # a ragged batch of prompt rows through a down projection
        _rows("rows_b200_4096x14336_res", 200, 4096, 14336, "none", False, "none", True),
        # the widest batch through the largest layer
        _rows("rows_b512_14336x4096_silu", 512, 14336, 4096, "rms", True, "silu", False),
    ]


def _log(rng, lo, hi):
    """A whole number from lo to hi, uniform in its logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


HEADS = [(12, 12, 64), (4, 1, 256), (8, 2, 128), (16, 2, 128), (6, 2, 64), (7, 1, 128)]


def _drawn(case):
    del case["name"]
    return case


def draw(rng):
    kind = rng.choice(["append", "attn", "attn", "rows", "rows"])
    page = rng.choice([16, 32, 64, 128, 256])
    if kind == "append":
        hq, hkv, hd = rng.choice(HEADS)
        streams = _log(rng, 1, 256)
        rows = streams if rng.random() < 0.5 else max(streams, _log(rng, 16, 8111))
        return _drawn(_append("", streams, rows, _log(rng, 1, 4000), hq, hkv, hd, page, rng.random() < 0.5,
                              rng.random() < 0.75))
    if kind == "attn":
        hq, hkv, hd = rng.choice(HEADS)
        streams = _log(rng, 1, 192)
        room = (1 << 28) // (streams * hkv * hd)  # keys a stream, so that the keys of all take at most 512 MB
        ctx = _log(rng, 1, min(65536, room))
        return _drawn(_attn("", streams, ctx, rng.choice(["full", "late", "mixed"]) if streams > 1 else "full", hq, hkv,
                            hd, page, rng.choice([0, 0, 0, _log(rng, 1, 4096)])))
    m = 2 * _log(rng, 125, 8192)
    k = 16 * _log(rng, 16, min(896, (14336 * 4096) // (16 * m)))
    act = rng.choice(["none", "relu", "gelu", "silu", "geglu"])
    return _drawn(_rows("", _log(rng, 1, 512), m, k, rng.choice(["none", "ln", "rms", "rms1p"]), rng.random() < 0.5, act,
                        rng.random() < 0.5))


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------

class _Ptr:
    """A torch tensor as the device buffer the op layer takes."""

    def __init__(self, t):
        self.t, self.ptr = t, t.data_ptr()


def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(1000003 * seed + 29)
    return g


def _normal(g, *shape):
    return torch.randn(*shape, generator=g, device="cuda")


def _pages(g, case, streams, room):
    """K and V pages with the rows of earlier tokens, and a page table of scattered pages for `room` positions a stream."""
    hkv, hd, page = case["hkv"], case["hd"], case["page"]
    per = -(-room // page)
    n = streams * per
    k = torch.randn(n, hkv, page, hd, generator=g, device="cuda", dtype=torch.bfloat16)
    v = torch.randn(n, hkv, page, hd, generator=g, device="cuda", dtype=torch.bfloat16)
    table = torch.randperm(n, generator=g, device="cuda").to(torch.int32).view(streams, per).contiguous()
    return k, v, table


def _prepare_append(case, seed):
    g = _gen(seed)
    streams, rows, hq, hkv, hd = (case[f] for f in ("streams", "rows", "hq", "hkv", "hd"))
    cpu = torch.Generator().manual_seed(1000003 * seed + 31)
    counts = torch.ones(streams, dtype=torch.int64)
    if rows > streams:  # ragged: the rest spread unevenly, the same lengths from every seed
        w = torch.rand(streams, generator=torch.Generator().manual_seed(rows)) ** 2 + 0.02
        counts += ((rows - streams) * w / w.sum()).long()
        counts[streams // 2] += rows - int(counts.sum())
    first = torch.randint(0, case["first"], (streams,), generator=cpu)
    room = case["first"] + int(counts.max())
    start = torch.cat([torch.zeros(1, dtype=torch.int64), counts.cumsum(0)])
    k, v, table = _pages(g, case, streams, room)
    x = _normal(g, rows, (hq + 2 * hkv) * hd)  # one fused projection's output: q | k | v
    at = torch.arange(room, dtype=torch.float64)[:, None] * 1e6 ** (-torch.arange(hd // 2, dtype=torch.float64) / (hd // 2))
    return {"kind": "append", "case": case, "x": x, "kp": k, "vp": v, "table": table,
            "pos": first.to(torch.int32).cuda(), "start": start.to(torch.int32).cuda() if rows > streams else None,
            "qn": 0.1 * _normal(g, hd) if case["norm"] else None, "kn": 0.1 * _normal(g, hd) if case["norm"] else None,
            "cos": at.cos().float().cuda() if case["rope"] else None,
            "sin": at.sin().float().cuda() if case["rope"] else None,
            "q_out": torch.empty(rows, hq * hd, device="cuda"), "eps": 1e-6}


def _prepare_attn(case, seed):
    g = _gen(seed)
    streams, ctx, hq, hd = (case[f] for f in ("streams", "ctx", "hq", "hd"))
    k, v, table = _pages(g, case, streams, ctx)
    lo = {"full": ctx, "late": (ctx + 1) // 2, "mixed": 1}[case["spread"]]
    lens = torch.randint(lo, ctx + 1, (streams,), generator=g, device="cuda")
    lens[0] = ctx
    if case["spread"] == "mixed":
        lens[5::9] = 0  # idle slots of the batch
    if case["window"]:  # pages wholly before the window are no longer the stream's
        last = (torch.arange(table.shape[1], device="cuda") + 1) * case["page"] - 1
        table[last[None] < (lens - case["window"])[:, None]] = -1
    return {"kind": "attn", "case": case, "q": _normal(g, streams, hq, hd), "kp": k, "vp": v, "table": table,
            "lens": lens.to(torch.int32), "out": torch.empty(streams, hq, hd, device="cuda"), "scale": hd ** -0.5}


def _prepare_rows(case, seed):
    g = _gen(seed)
    batch, m, k, norm = (case[f] for f in ("batch", "m", "k", "norm"))
    w = _normal(g, m, k) * 0.02
    scale = w.abs().amax(1) / 127.0
    w = (w / scale[:, None]).round_().clamp_(-127, 127).to(torch.int8)
    big = torch.rand(k, generator=g, device="cuda") < 0.004  # a few channels of a residual stream are far larger
    x = torch.where(big, 30.0, 1.0) * _normal(g, batch, k)
    out = m // 2 if case["act"] == "geglu" else m
    return {"kind": "rows", "case": case, "w": w, "scale": scale, "bias": 0.02 * _normal(g, m), "x": x,
            "add": _normal(g, batch, k) if case["add"] else None,
            "sum": torch.empty(batch, k, device="cuda") if case["add"] else None,
            "gamma": 1.0 + 0.1 * _normal(g, k) if norm != "none" else None,
            "beta": 0.1 * _normal(g, k) if norm == "ln" else None, "eps": 1e-6,
            "res": _normal(g, batch, out) if case["res"] else None, "y": torch.empty(batch, out, device="cuda")}


def _paged(xe, st):
    return xe.PagedKV(_Ptr(st["kp"]), _Ptr(st["vp"]), _Ptr(st["table"]), *st["kp"].shape, *st["table"].shape)


def _handles(st):
    """What a program makes once: the cache's description, the arguments' struct, the registered weight."""
    xe, ctx = _package()
    case = st["case"]
    p = {n: _Ptr(t) for n, t in st.items() if isinstance(t, torch.Tensor)}
    if st["kind"] == "append":
        ld, qw, kw = st["x"].shape[1], case["hq"] * case["hd"], case["hkv"] * case["hd"]
        st["kv"] = _paged(xe, st)
        st["args"] = xe.PagedRows(case["rows"], case["hq"], q=p["x"].ptr, k=p["x"].ptr + 4 * qw,
                                  v=p["x"].ptr + 4 * (qw + kw), ldq=ld, ldkv=ld, q_out=p["q_out"].ptr, ldqo=qw,
                                  pos=p["pos"].ptr, start=p["start"].ptr if "start" in p else None,
                                  q_norm=p["qn"].ptr if "qn" in p else None, k_norm=p["kn"].ptr if "kn" in p else None,
                                  eps=st["eps"], cos=p["cos"].ptr if "cos" in p else None,
                                  sin=p["sin"].ptr if "sin" in p else None,
                                  rope_len=st["cos"].shape[0] if "cos" in p else 0)
    elif st["kind"] == "attn":
        st["kv"] = _paged(xe, st)
        st["p"] = p
    else:
        w = ctx.register_weight_view(xe.XE_I8, case["m"], case["k"], p["w"].ptr, p["scale"].ptr, None, p["bias"].ptr)
        if case["norm"] != "none":
            gamma = st["gamma"].cpu().numpy()
            make = {"ln": lambda: xe.Norm.Ln(gamma, st["beta"].cpu().numpy(), st["eps"]),
                    "rms": lambda: xe.Norm.Rms(gamma, st["eps"]), "rms1p": lambda: xe.Norm.Rms1p(gamma, st["eps"])}
            ctx.set_norm(w, make[case["norm"]]())
        st["weight"] = w
        act = {"none": xe.XE_ACT_NONE, "relu": xe.XE_ACT_RELU, "gelu": xe.XE_ACT_GELU, "silu": xe.XE_ACT_SILU,
               "geglu": xe.XE_ACT_GEGLU}[case["act"]]
        st["args"] = xe.W8a8Rows(case["batch"], p["x"].ptr, p["y"].ptr, act=act,
                                 **{n: p[n].ptr for n in ("add", "sum", "res") if n in p})
    return st


def prepare(case, seed):
    st = {"append": _prepare_append, "attn": _prepare_attn, "rows": _prepare_rows}[case["kind"]](case, seed)
    if not own:
        return st
    st = _handles(st)
    torch.cuda.synchronize()  # the library's stream does not wait for torch's
    return st


# ---------------------------------------------------------------------------
# plain forms, and the library's calls
# ---------------------------------------------------------------------------

def _turn(x, w, eps, cos, sin):
    """Heads [n, h, hd]: RMSNorm (1 + w) over a head, then dimension j rotated with j + hd / 2."""
    if w is not None:
        x = x / torch.sqrt((x * x).mean(-1, keepdim=True) + eps) * (1.0 + w)
    if cos is not None:
        a, b = x.chunk(2, -1)
        x = torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
    return x


def _run_append(st):
    case = st["case"]
    n, hq, hkv, hd, page = (case[f] for f in ("rows", "hq", "hkv", "hd", "page"))
    if own:
        _open["ctx"].paged_append_dev(st["kv"], st["args"])
        return [st["q_out"], st["kp"], st["vp"]]
    row = torch.arange(n, device="cuda")
    stream, pos = row, st["pos"].long()
    if st["start"] is not None:
        start = st["start"].long()
        stream = (row[:, None] >= start[None, 1:]).sum(1)
        pos = pos[stream] + row - start[stream]
    q, k, v = st["x"].split([hq * hd, hkv * hd, hkv * hd], 1)
    cos, sin = (None if st[t] is None else st[t][pos][:, None] for t in ("cos", "sin"))
    q = _turn(q.reshape(n, hq, hd), st["qn"], st["eps"], cos, sin)
    k = _turn(k.reshape(n, hkv, hd), st["kn"], st["eps"], cos, sin)
    at = st["table"][stream, pos // page].long()
    st["kp"][at, :, pos % page] = k.bfloat16()
    st["vp"][at, :, pos % page] = v.reshape(n, hkv, hd).bfloat16()
    return [q.reshape(n, hq * hd), st["kp"], st["vp"]]


def _run_attn(st):
    case = st["case"]
    hq, hkv, hd = case["hq"], case["hkv"], case["hd"]
    if own:
        p = st["p"]
        _open["ctx"].paged_attn_dev(st["kv"], p["q"], p["lens"], hq, st["scale"], p["out"], window=case["window"])
        return st["out"]
    b, per = st["table"].shape
    room = per * case["page"]
    at = st["table"].long()
    pos = torch.arange(room, device="cuda")
    lens = st["lens"].long()[:, None]
    on = (pos < lens) & (at >= 0).repeat_interleave(case["page"], 1)
    if case["window"]:
        on = on & (pos >= lens - case["window"])
    at = at.clamp_min(0)
    on = on[:, None, :, None]
    keys = torch.where(on, st["kp"][at].transpose(1, 2).reshape(b, hkv, room, hd).float(), 0.0)
    values = torch.where(on, st["vp"][at].transpose(1, 2).reshape(b, hkv, room, hd).float(), 0.0)
    q = st["q"].view(b, hkv, hq // hkv, hd).transpose(2, 3).contiguous()
    s = torch.where(on, torch.matmul(keys, q) * st["scale"], -math.inf)  # [b, hkv, room, group]
    top = s.amax(2, keepdim=True)
    p = torch.exp(s - torch.where(top > -math.inf, top, 0.0))
    total = p.sum(2, keepdim=True)
    p = (p / torch.where(total > 0, total, 1.0)).transpose(2, 3).contiguous()
    return torch.matmul(p, values).reshape(b, hq, hd)


def _codes(h):
    """int8 codes of rows and their scales: max|row| / 127, half away from zero."""
    amax = h.abs().amax(1, keepdim=True)
    s = torch.where(amax > 0, amax / 127.0, 1.0).float().double()
    r = h / s
    return torch.sign(r) * torch.floor(r.abs() + 0.5), s


def _run_rows(st):
    case = st["case"]
    if own:
        _open["ctx"].w8a8_rows_dev(st["weight"], st["args"])
        return [st["y"]] if st["sum"] is None else [st["y"], st["sum"]]
    t = st["x"] if st["add"] is None else st["x"] + st["add"]
    h = t.double()  # a code next to a border between two needs more than 32 bits
    if case["norm"] == "ln":
        h = h - h.mean(1, keepdim=True)
    if case["norm"] != "none":
        h = h / torch.sqrt((h * h).mean(1, keepdim=True) + st["eps"])
        h = h * ((1.0 if case["norm"] == "rms1p" else 0.0) + st["gamma"].double())
    if case["norm"] == "ln":
        h = h + st["beta"].double()
    q, s = _codes(h)
    y = torch.matmul(q.float(), st["w"].float().t().contiguous())
    y = y * s.float() * st["scale"] + st["bias"]
    if case["act"] == "relu":
        y = torch.where(y > 0, y, 0.0)
    elif case["act"] == "gelu":
        y = 0.5 * y * (1.0 + torch.erf(y * math.sqrt(0.5)))
    elif case["act"] == "silu":
        y = y / (1.0 + torch.exp(-y))
    elif case["act"] == "geglu":
        gate, up = y[:, 0::2], y[:, 1::2]
        y = 0.5 * gate * (1.0 + torch.tanh(math.sqrt(2.0 / math.pi) * (gate + 0.044715 * gate * gate * gate))) * up
    if st["res"] is not None:
        y = y + st["res"]
    return [y] if st["add"] is None else [y, t]


def run(state):
    return {"append": _run_append, "attn": _run_attn, "rows": _run_rows}[state["kind"]](state)


# ---------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------

def _keys_read(case):
    """Keys of all streams that a pass attends to, on average over seeds."""
    ctx, n = case["ctx"], case["streams"]
    window = case["window"] or ctx
    lo = {"full": ctx, "late": (ctx + 1) // 2, "mixed": 1}[case["spread"]]
    w = min(window, ctx)
    # mean of min(len, window) over len = lo .. ctx
    short = max(0, min(ctx, w) - lo + 1)
    total = (lo + min(ctx, w)) * short / 2 if short else 0.0
    mean = (total + (ctx - lo + 1 - short) * w) / (ctx - lo + 1)
    idle = len(range(5, n, 9)) if case["spread"] == "mixed" else 0
    return w + (n - 1 - idle) * mean


def work(case):
    if case["kind"] == "append":
        n, hq, hkv, hd = (case[f] for f in ("rows", "hq", "hkv", "hd"))
        tables = 8 * case["streams"] + 4 * n * (hd if case["rope"] else 0)
        return {"bytes": n * hd * (8 * hq + 12 * hkv) + tables, "flops": 10 * n * hd * (hq + hkv)}
    if case["kind"] == "attn":
        keys, hq, hkv, hd = _keys_read(case), case["hq"], case["hkv"], case["hd"]
        return {"bytes": 4 * keys * hkv * hd + 4 * keys / case["page"] + case["streams"] * (8 * hq * hd + 4),
                "flops": 4 * keys * hq * hd}
    b, m, k = case["batch"], case["m"], case["k"]
    out = m // 2 if case["act"] == "geglu" else m
    rows = 4 * b * k * (3 if case["add"] else 1) + 4 * b * out * (2 if case["res"] else 1)
    return {"bytes": m * k + 8 * m + (4 * k if case["norm"] != "none" else 0) + rows, "flops": 2 * b * m * k}


# ---------------------------------------------------------------------------
# the definitions in 64 bits
# ---------------------------------------------------------------------------

def _exact_append(case, seed):
    st = _prepare_append(case, seed)
    hq, hkv, hd, page = (case[f] for f in ("hq", "hkv", "hd", "page"))
    x = st["x"].double()
    start = list(range(case["streams"] + 1)) if st["start"] is None else st["start"].tolist()
    first = st["pos"].tolist()
    half = hd // 2
    swap = torch.cat([torch.arange(half, hd), torch.arange(half)]).cuda()
    sign = torch.where(torch.arange(hd) < half, -1.0, 1.0).double().cuda()

    def heads(cols, count, w, at):
        h = cols.reshape(-1, count, hd)
        if w is not None:
            h = h * torch.rsqrt(h.square().sum(-1, keepdim=True) / hd + st["eps"]) * (w.double() + 1.0)
        if st["cos"] is not None:
            c, s = (torch.cat([t[at], t[at]], 1).double()[:, None] for t in (st["cos"], st["sin"]))
            h = h * c + sign * h[..., swap] * s
        return h

    kp, vp, q = st["kp"].double(), st["vp"].double(), []
    for i, a in enumerate(first):
        rows = x[start[i]:start[i + 1]]
        at = torch.arange(a, a + rows.shape[0], device="cuda")
        q.append(heads(rows[:, :hq * hd], hq, st["qn"], at).reshape(-1, hq * hd))
        pages, slot = st["table"][i].long()[at // page], at % page
        kp[pages, :, slot] = heads(rows[:, hq * hd:(hq + hkv) * hd], hkv, st["kn"], at)
        vp[pages, :, slot] = rows[:, (hq + hkv) * hd:].reshape(-1, hkv, hd)
    return [torch.cat(q), kp, vp]


def _exact_attn(case, seed):
    st = _prepare_attn(case, seed)
    hq, hkv, hd = case["hq"], case["hkv"], case["hd"]
    out = torch.zeros(case["streams"], hq, hd, dtype=torch.float64, device="cuda")
    for i, n in enumerate(st["lens"].tolist()):
        lo = max(0, n - case["window"]) if case["window"] else 0
        if n <= lo:
            continue
        pos = torch.arange(lo, n, device="cuda")
        pages = st["table"][i].long()[pos // case["page"]]
        k = st["kp"][pages, :, pos % case["page"]].double()  # [keys, hkv, hd]
        v = st["vp"][pages, :, pos % case["page"]].double()
        for h in range(hq):
            g = h * hkv // hq
            s = (k[:, g] @ st["q"][i, h].double()) * st["scale"]
            out[i, h] = torch.softmax(s, 0) @ v[:, g]
    return out


def _exact_rows(case, seed):
    st = _prepare_rows(case, seed)
    h = st["x"].clone()
    if st["add"] is not None:
        h += st["add"]
    total, h = h.double(), h.double()
    k = case["k"]
    if case["norm"] == "ln":
        h = torch.nn.functional.layer_norm(h, (k,), st["gamma"].double(), st["beta"].double(), st["eps"])
    elif case["norm"] != "none":
        weight = st["gamma"].double() + (1.0 if case["norm"] == "rms1p" else 0.0)
        h = h * torch.rsqrt(h.square().sum(1, keepdim=True) / k + st["eps"]) * weight
    s = h.abs().max(1).values / 127.0
    s[s == 0] = 1.0
    s = s.float().double()  # held in 32 bits
    q = h / s[:, None]
    q = torch.where(q < 0, torch.ceil(q - 0.5), torch.floor(q + 0.5))
    z = (q @ st["w"].double().t()) * s[:, None] * st["scale"].double() + st["bias"].double()
    f = torch.nn.functional
    if case["act"] == "geglu":
        z = z.view(case["batch"], -1, 2)
        z = f.gelu(z[..., 0], approximate="tanh") * z[..., 1]
    elif case["act"] != "none":
        z = {"relu": f.relu, "gelu": f.gelu, "silu": f.silu}[case["act"]](z)
    if st["res"] is not None:
        z = z + st["res"].double()
    return [z] if st["add"] is None else [z, total]


def exact(case, seed):
    return {"append": _exact_append, "attn": _exact_attn, "rows": _exact_rows}[case["kind"]](case, seed)
