"""The operators of a long-context speculative round, as they are measured: the heads' norms and
rotation, the 4-bit K/V cache's append, the attention that reads it, and the sampled verification
of drafted tokens.

`own` false: the same results from elementary torch operations (float32, float64 for angles, long
sums and probabilities next to a border), on the same inputs. `own` true: the calls of a program
that uses qwen35 (include/q35.h).

The 4-bit format: 32 consecutive dims of a head at one slot share one scale byte b (2^(b - 127));
a code is sign << 3 | index into (0, 0.5, 1, 1.5, 2, 3, 4, 6), two codes a byte, the lower dim in
the low nibble; the scale is the smallest power of two whose largest code, 6, covers the group.
"""
import functools
import math
import sys
from pathlib import Path

import numpy as np
import torch

own = False

DEV = "cuda"
THETA, EPS = 1e7, 1e-6
VOCAB = 248320
GRID = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


# ------------------------------------------------------------------------------ the cases
def _heads(lanes, rows, pos, q, kv, dim, rot):
    return {"lanes": lanes, "rows": rows, "pos": pos, "q_heads": q, "kv_heads": kv, "dim": dim, "rot": rot}


def _attn(lanes, rows, ctx, q, kv, dim, window, sinks, ragged):
    return {"lanes": lanes, "rows": rows, "ctx": ctx, "q_heads": q, "kv_heads": kv, "dim": dim, "window": window,
            "sinks": sinks, "ragged": ragged}


def listed():
    return [
        # A layer's heads before any cache: one request's step far into a long conversation; a whole
        # prompt.
        {"name": "norm_rope_1", "kind": "heads", **_heads(1, 1, 32000, 8, 2, 256, 64)},
        {"name": "norm_rope_4096", "kind": "heads", **_heads(1, 4096, 0, 8, 2, 256, 64)},
        # The same with the append in 4 bits: a step of the headline batch; a prompt wave that ends
        # on an odd slot, of a layer with the whole head rotated.
        {"name": "append_256", "kind": "append", **_heads(256, 1, 4096, 8, 2, 256, 64)},
        {"name": "append_1999", "kind": "append", **_heads(1, 1999, 2048, 32, 8, 128, 128)},
        # Attention over the cache: one long conversation's step; the headline batch; a server's
        # conversations of many lengths under a window with 4 sinks; a speculative round's 3 rows a
        # lane; the prompt that fills a cache.
        {"name": "attn_1x32768", "kind": "attn", **_attn(1, 1, 32768, 8, 2, 256, 0, 0, False)},
        {"name": "attn_256x4096", "kind": "attn", **_attn(256, 1, 4096, 8, 2, 256, 0, 0, False)},
        {"name": "attn_64x8192_window", "kind": "attn", **_attn(64, 1, 8192, 32, 4, 128, 1024, 4, True)},
        {"name": "attn_verify_128x2000", "kind": "attn", **_attn(128, 3, 2000, 8, 2, 256, 0, 0, True)},
        {"name": "attn_prompt_4096", "kind": "attn", **_attn(1, 4096, 4096, 8, 2, 256, 0, 0, False)},
        # Sampled verification: one request with greedy drafts (a draft is certain of itself); a few
        # requests with the drafter's own probabilities over a small odd vocabulary in bfloat16; the
        # headline batch.
        {"name": "verify_1", "kind": "verify", "lanes": 1, "drafts": 2, "vocab": VOCAB, "probs": False, "bf16": False},
        {"name": "verify_17_odd", "kind": "verify", "lanes": 17, "drafts": 4, "vocab": 32003, "probs": True,
         "bf16": True},
        {"name": "verify_256", "kind": "verify", "lanes": 256, "drafts": 2, "vocab": VOCAB, "probs": False,
         "bf16": False},
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


LAYOUTS = [(8, 2, 256), (8, 2, 256), (32, 8, 128), (32, 4, 128), (16, 16, 64), (14, 2, 64), (5, 1, 128), (48, 3, 256)]


def draw(rng):
    kind = rng.choice(["heads", "append", "attn", "attn", "attn", "prompt", "verify"])
    q, kv, dim = rng.choice(LAYOUTS)
    if kind in ("heads", "append"):
        lanes = _log_int(rng, 1, 256)
        rot = rng.choice([dim, dim // 2, dim // 4])
        return {"kind": kind, **_heads(lanes, _log_int(rng, 1, max(1, 4096 // lanes)), _log_int(rng, 1, 131072 if
                                       kind == "heads" else 4096), q, kv, dim, rot)}
    if kind == "attn":
        lanes = _log_int(rng, 1, 256)
        rows = rng.choice([1, 1, 1, 2, 3, 5])
        most = max(16, min(32768, (1 << 29) // (lanes * kv * dim)))
        window = rng.choice([0, 0, 1, _log_int(rng, 16, 4096)])
        sinks = rng.choice([0, 4, _log_int(rng, 1, 64)]) if window else 0
        return {"kind": "attn", **_attn(lanes, rows, _log_int(rng, rows, most), q, kv, dim, window, sinks,
                                        rng.random() < 0.5)}
    if kind == "prompt":
        ctx = _log_int(rng, 64, 4096 if q * dim <= 4096 else 2048)
        rows = ctx if rng.random() < 0.5 else _log_int(rng, 17, ctx)
        window = rng.choice([0, _log_int(rng, 16, 2048)])
        return {"kind": "attn", **_attn(1, rows, ctx, q, kv, dim, window, rng.choice([0, 4]) if window else 0, False)}
    drafts = rng.randint(1, 4)
    vocab = rng.choice([VOCAB, 32003, 151_936, 50257])
    lanes = _log_int(rng, 1, max(1, min(256, 190_000_000 // ((2 * drafts + 1) * vocab))))
    return {"kind": kind, "lanes": lanes, "drafts": drafts, "vocab": vocab, "probs": rng.random() < 0.5,
            "bf16": rng.random() < 0.5}


# ------------------------------------------------------------------------------ inputs
def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(int(seed))


def _bf16(g, *shape, scale=1.0):
    return (torch.randn(*shape, generator=g, device=DEV) * scale).to(torch.bfloat16)


def _lane_pos(case):
    """Position of each lane's first row: all the same, or spread evenly from an eighth of it up."""
    n = case["lanes"]
    last = case["pos"] if "pos" in case else case["ctx"] - case["rows"]
    if not case.get("ragged"):
        return np.full(n, last, np.int32)
    return np.array([last - (i * (last - last // 8)) // n for i in range(n)], np.int32)


def _two(e):
    """2^e in float32, for whole numbers e."""
    return (e.int() + 127 << 23).view(torch.float32)


def _cache_rows(g, *shape):
    """Codes and scale bytes of N(0, 1) rows [..., dim], as a filled cache holds them."""
    x = torch.randn(*shape, generator=g, device=DEV).view(*shape[:-1], shape[-1] // 32, 32)
    e = torch.frexp(x.abs().amax(-1, keepdim=True) / 6.0)
    e = e.exponent - (e.mantissa == 0.5).int()              # smallest e with amax <= 6 * 2^e
    mag = x.abs() * _two(-e)
    code = torch.zeros_like(mag, dtype=torch.uint8)
    for mid, tie_up in ((0.25, False), (0.75, True), (1.25, False), (1.75, True), (2.5, False), (3.5, True), (5.0, False)):
        code += (mag >= mid) if tie_up else (mag > mid)
    code |= (x < 0).to(torch.uint8) << 3
    code = code.view(*shape[:-1], shape[-1] // 2, 2)
    return code[..., 0] | code[..., 1] << 4, (e[..., 0] + 127).to(torch.uint8)


@functools.lru_cache(maxsize=None)
def engine():
    pkg = str(Path(__file__).resolve().parents[1] / "qwen3.5-0.8b_amd")
    if pkg not in sys.path:
        sys.path.insert(0, pkg)
    from qwen35 import Engine
    torch.zeros(1, device=DEV)        # torch's runtime first: it makes the buffers
    return Engine(max_rows=2048, max_ctx=33024, seed=None)


def _inputs(case, seed):
    """What the call reads, from the seed alone."""
    g, kind, n = _gen(seed), case["kind"], case["lanes"]
    s = {"case": case}
    if kind in ("heads", "append"):
        q, kv, d, R = case["q_heads"], case["kv_heads"], case["dim"], n * case["rows"]
        # a projection's rows: (q | gate) per q head, then k, then v
        s["proj"] = _bf16(g, R, (2 * q + 2 * kv) * d)
        s["qn"], s["kn"] = _bf16(g, d, scale=0.1), _bf16(g, d, scale=0.1)
        s["pos"] = _lane_pos(case)
    elif kind == "attn":
        q, kv, d, R = case["q_heads"], case["kv_heads"], case["dim"], n * case["rows"]
        s["kc"], s["ks"] = _cache_rows(g, n, kv, case["ctx"], d)
        s["vc"], s["vs"] = _cache_rows(g, n, kv, case["ctx"], d)
        s["q"], s["gate"] = _bf16(g, R, q, d), _bf16(g, R, q, d)
        s["pos"] = np.random.default_rng(seed).permutation(_lane_pos(case)).astype(np.int32)
    else:
        k, v = case["drafts"], case["vocab"]
        t = torch.bfloat16 if case["bf16"] else torch.float32
        s["temp"] = 0.8
        lg = torch.randn(n, k + 1, v, generator=g, device=DEV) * 2.0
        hot = torch.randint(0, v, (n, k + 1, 12), generator=g, device=DEV)
        lg.scatter_add_(2, hot, 8.0 + 3.0 * torch.randn(n, k + 1, 12, generator=g, device=DEV))
        s["logits"] = lg.to(torch.bfloat16).to(t)     # a bf16 head's logits
        dl = lg[:, :k] + 0.7 * torch.randn(n, k, v, generator=g, device=DEV)
        if case["probs"]:
            s["dlogits"] = dl.to(torch.bfloat16).to(t)
            gum = -torch.log(-torch.log(torch.rand(n, k, v, generator=g, device=DEV).clamp_(1e-20, 1 - 1e-7)))
            s["drafts"] = (s["dlogits"].float() / s["temp"] + gum).argmax(-1).int()
        else:
            s["dlogits"] = None
            s["drafts"] = dl.argmax(-1).int()
        # a lane in five has fewer drafts: -1 ends them
        short = torch.rand(n, k, generator=g, device=DEV) < 0.2 / k
        s["drafts"][short.cumsum(1) > 0] = -1
        s["u"] = torch.rand(n, k + 1, generator=g, device=DEV)
    return s


def prepare(case, seed):
    s, kind, n = _inputs(case, seed), case["kind"], case["lanes"]
    if own:
        s["eng"] = engine()
        from qwen35 import KvCache4
        s["lanes"] = np.arange(n, dtype=np.int32)
        bf16 = functools.partial(torch.empty, dtype=torch.bfloat16, device=DEV)
        if kind in ("heads", "append"):
            q, kv, d, R = case["q_heads"], case["kv_heads"], case["dim"], n * case["rows"]
            s["qo"], s["ko"], s["vo"] = bf16(R, q, d), bf16(R, kv, d), bf16(R, kv, d)
            if kind == "append":
                s["cache"] = KvCache4(s["eng"], n, int(s["pos"].max()) + case["rows"], kv_heads=kv, head_dim=d)
                s["cache"].set_len(s["lanes"], s["pos"])      # the earlier slots are held already
        elif kind == "attn":
            kv, d, c = case["kv_heads"], case["dim"], case["ctx"]
            s["out"] = bf16(n * case["rows"], case["q_heads"], d)
            s["cache"] = KvCache4(s["eng"], n, c, kv_heads=kv, head_dim=d)
            torch.cuda.synchronize()
            s["cache"].write(0, 0, n, 0, c, *[s[k].data_ptr() for k in ("kc", "ks", "vc", "vs")])
            s["eng"].sync()
            for k in ("kc", "ks", "vc", "vs"):
                del s[k]
        else:
            s["acc"] = torch.empty(n, dtype=torch.int32, device=DEV)
            s["tok"] = torch.empty(n, case["drafts"] + 1, dtype=torch.int32, device=DEV)
        torch.cuda.synchronize()          # the engine's stream reads what torch's stream has made
    return s


# ------------------------------------------------------------------------------ the plain forms
def _rows_pos(s):
    at = torch.from_numpy(s["pos"].astype(np.int64)).to(DEV, non_blocking=True)
    return at[:, None] + torch.arange(s["case"]["rows"], device=DEV)


def _split(s):
    """The projection's rows as q [R][q][d], k [R][kv][d], v [R][kv][d]."""
    c = s["case"]
    q, kv, d = c["q_heads"], c["kv_heads"], c["dim"]
    x = s["proj"]
    R = x.shape[0]
    return (x[:, :2 * q * d].view(R, q, 2 * d)[..., :d], x[:, 2 * q * d:(2 * q + kv) * d].view(R, kv, d),
            x[:, (2 * q + kv) * d:].view(R, kv, d))


def _norm_rope(x, w, at, rot):
    """Rows [R][h][d] in float32: the head's RMS norm with weight 1 + w, dims [0, rot) rotated in
    pairs (i, i + rot / 2) by at * theta^(-2 i / rot); sums of squares and angles in float64."""
    xf = x.float()
    rs = (1.0 / (xf.double().square().mean(-1, keepdim=True) + EPS).sqrt()).float()
    y = xf * rs * (1.0 + w.float())
    half = rot // 2
    ang = at.reshape(-1, 1, 1).double() * THETA ** (torch.arange(half, dtype=torch.float64, device=DEV) * (-2.0 / rot))
    c, n = ang.cos().float(), ang.sin().float()
    a, b = y[..., :half], y[..., half:rot]
    return torch.cat([a * c - b * n, b * c + a * n, y[..., rot:]], -1)


def _through_4_bits(x):
    """float32 rows [..., d] -> the values their codes stand for."""
    g = x.reshape(*x.shape[:-1], -1, 32)
    top = g.abs().amax(-1, keepdim=True)
    m, e = torch.frexp(top)                                 # top = m 2^e, m in [0.5, 1)
    e = torch.where(m > 0.75, e - 2, e - 3)                 # top <= 6 * 2^e
    y = g * _two(-e)
    mag = y.abs()
    step = torch.where(mag < 2, 0.5, torch.where(mag < 4, 1.0, 2.0))
    return (torch.round(y / step) * step * _two(e)).view_as(x)   # ties to the even code


@functools.lru_cache(maxsize=None)
def _pairs():
    one = torch.tensor(GRID + tuple(-v for v in GRID), device=DEV)
    b = torch.arange(256, device=DEV)
    return torch.stack([one[b & 15], one[b >> 4]], -1)      # a byte's two values


def _values(codes, scales):
    x = _pairs()[codes.int()].view(*scales.shape, 32)
    return (x * _two(scales.int() - 127)[..., None]).flatten(-2)


def _plain_attn(s):
    c = s["case"]
    n, T, hq, kv, d = c["lanes"], c["rows"], c["q_heads"], c["kv_heads"], c["dim"]
    K, V = _values(s["kc"], s["ks"]), _values(s["vc"], s["vs"])              # [n][kv][ctx][d]
    q = s["q"].float().view(n, T, kv, hq // kv, d).permute(0, 2, 3, 1, 4).reshape(n, kv, -1, d)
    at = _rows_pos(s)[:, :, None]                                            # [n][T][1]
    slot = torch.arange(c["ctx"], device=DEV)
    see = slot <= at
    if c["window"]:
        see &= (slot > at - c["window"]) | (slot < c["sinks"])
    sc = torch.matmul(q, K.transpose(-1, -2)).view(n, kv, hq // kv, T, -1) * d ** -0.5
    sc = sc.masked_fill_(~see[:, None, None], -math.inf)
    p = torch.exp_(sc - sc.amax(-1, keepdim=True))
    o = torch.matmul(p.view(n, kv, -1, c["ctx"]), V).view(n, kv, hq // kv, T, d) / p.sum(-1, keepdim=True)
    o = o.permute(0, 3, 1, 2, 4).reshape(n * T, hq, d)
    return (o * torch.sigmoid(s["gate"].float())).to(torch.bfloat16)


def _probs(logits, temp):
    x = logits.double() / temp
    e = torch.exp(x - x.amax(-1, keepdim=True))
    return e / e.sum(-1, keepdim=True)


def _plain_verify(s):
    n, k = s["case"]["lanes"], s["case"]["drafts"]
    p = _probs(s["logits"], s["temp"])
    d, u = s["drafts"].long(), s["u"].double()
    real, di = d >= 0, d.clamp(min=0)[..., None]
    pd = p[:, :k].gather(2, di)[..., 0]
    if s["dlogits"] is not None:
        q = _probs(s["dlogits"], s["temp"])
        qd = q.gather(2, di)[..., 0]
    else:
        qd = torch.ones_like(pd)
    a = (real & (u[:, :k] * qd < pd)).long().cumprod(1).sum(1)               # accepted drafts
    lane, at = torch.arange(n, device=DEV), a.clamp(max=k - 1)
    refused = (a < k) & real[lane, at]
    w = p[lane, a]
    if s["dlogits"] is not None:
        rest = (w - q[lane, at]).clamp_(min=0)
    else:
        rest = w.scatter(1, di[lane, at], 0.0)
    c = torch.where((refused & (rest.sum(1) > 0))[:, None], rest, w).cumsum(1)
    tok = (c > u[:, k:] * c[:, -1:]).int().argmax(1)
    col = torch.arange(k + 1, device=DEV)
    out = torch.where(col < a[:, None], torch.nn.functional.pad(d, (0, 1)), -1)
    return {"accepted": a.int(), "tokens": torch.where(col == a[:, None], tok[:, None], out).int()}


# ------------------------------------------------------------------------------ one pass
def _view(t, heads, off=0, head=None):
    """Rows of heads in a buffer: address, elements from row to row, elements from head to head."""
    return t.data_ptr() + 2 * off, t.stride(0), head or t.shape[-1]


def run(s):
    c = s["case"]
    kind = c["kind"]
    if not own:
        if kind == "attn":
            return _plain_attn(s)
        if kind == "verify":
            return _plain_verify(s)
        q, k, v = _split(s)
        at = _rows_pos(s)
        q, k = _norm_rope(q, s["qn"], at, c["rot"]).to(torch.bfloat16), _norm_rope(k, s["kn"], at, c["rot"])
        if kind == "heads":
            return {"q": q, "k": k.to(torch.bfloat16)}
        return {"q": q, "k": _through_4_bits(k).to(torch.bfloat16), "v": _through_4_bits(v.float()).to(torch.bfloat16)}
    eng = s["eng"]
    if kind in ("heads", "append"):
        q, kv, d, x = c["q_heads"], c["kv_heads"], c["dim"], s["proj"]
        rows = {"q": _view(x, q, 0, 2 * d), "k": _view(x, kv, 2 * q * d, d), "q_norm": s["qn"].data_ptr(),
                "k_norm": s["kn"].data_ptr(), "q_out": _view(s["qo"], q), "k_out": _view(s["ko"], kv)}
        if kind == "heads":
            eng.op_qk_norm_rope(s["pos"], c["rows"], q, kv, d, rot_dim=c["rot"], theta=THETA, eps=EPS, **rows)
            return {"q": s["qo"], "k": s["ko"]}
        eng.op_kv4_append(s["cache"], 0, s["lanes"], s["pos"], c["rows"], q, rot_dim=c["rot"], theta=THETA, eps=EPS,
                          v=_view(x, kv, (2 * q + kv) * d, d), v_out=_view(s["vo"], kv), **rows)
        return {"q": s["qo"], "k": s["ko"], "v": s["vo"]}
    if kind == "attn":
        h = c["q_heads"]
        eng.op_attn_kv4(s["cache"], 0, s["lanes"], s["pos"], c["rows"], h, _view(s["q"], h), _view(s["out"], h),
                        window=c["window"], sinks=c["sinks"], gate=_view(s["gate"], h))
        return s["out"]
    dl = s["dlogits"]
    eng.op_draft_verify(c["lanes"], c["drafts"], c["vocab"], s["logits"].data_ptr(), s["drafts"].data_ptr(),
                        s["u"].data_ptr(), s["acc"].data_ptr(), s["tok"].data_ptr(), temperature=s["temp"],
                        draft_logits=dl.data_ptr() if dl is not None else 0, bf16=c["bf16"])
    return {"accepted": s["acc"], "tokens": s["tok"]}


# ------------------------------------------------------------------------------ floors
def _visible(case):
    """Slots a lane's rows see together, and (row, slot) pairs, over all lanes."""
    slots = pairs = 0
    for p in _lane_pos(case).astype(np.int64):
        at = p + np.arange(case["rows"])
        if case["window"]:
            low = np.maximum(at - case["window"] + 1, 0)
            sink = np.minimum(case["sinks"], low)
            pairs += int((at - low + 1 + sink).sum())
            slots += int(at[-1] - low[0] + 1 + sink[0])
        else:
            pairs += int((at + 1).sum())
            slots += int(at[-1] + 1)
    return slots, pairs


def work(case):
    """Bytes and operations of one pass: inputs read once, outputs written once."""
    kind, n = case["kind"], case["lanes"]
    if kind in ("heads", "append"):
        q, kv, d, R = case["q_heads"], case["kv_heads"], case["dim"], n * case["rows"]
        b = R * d * (2 * q + 2 * kv) * 2 + 4 * d
        if kind == "append":      # v in, the values that k's and v's codes stand for, the codes and scales
            b += R * d * kv * (2 + 2 + 2 * (0.5 + 1 / 32))
        return {"bytes": b, "flops": R * d * (q + kv) * 8}
    if kind == "attn":
        slots, pairs = _visible(case)
        hq, d = case["q_heads"], case["dim"]
        return {"bytes": slots * case["kv_heads"] * (d + d // 16) + n * case["rows"] * hq * d * 6,
                "flops": 4 * pairs * hq * d}
    rows = n * (case["drafts"] + 1) + (n * case["drafts"] if case["probs"] else 0)
    return {"bytes": rows * case["vocab"] * (2 if case["bf16"] else 4), "flops": rows * case["vocab"] * 4}


# ------------------------------------------------------------------------------ the same in 64 bits
def exact(case, seed):
    kind = case["kind"]
    if kind == "verify":
        return None                       # whole numbers
    s = _inputs(case, seed)
    T, n = case["rows"], case["lanes"]
    at = np.concatenate([p + np.arange(T) for p in s["pos"].astype(np.int64)])
    if kind in ("heads", "append"):
        q, k, v = (t.double() for t in _split(s))
        rot = case["rot"]
        th = torch.from_numpy(at[:, None] * np.exp(np.arange(rot // 2) * (-2.0 / rot) * math.log(THETA))).to(DEV)

        def turned(x, w):
            x = x / torch.sqrt((x * x).sum(-1, keepdim=True) / x.shape[-1] + EPS) * (w.double() + 1)
            z = torch.complex(x[..., :rot // 2], x[..., rot // 2:rot]) * torch.polar(torch.ones_like(th), th)[:, None]
            return torch.cat([z.real, z.imag, x[..., rot:]], -1)

        def four(x):
            g = x.unflatten(-1, (-1, 32))
            e = torch.ceil(torch.log2(g.abs().amax(-1, keepdim=True) / 6) - 1e-12)
            grid = torch.tensor(GRID, dtype=torch.float64, device=DEV)
            m = g.abs() * torch.exp2(-e)
            hi = torch.searchsorted(grid, m.contiguous()).clamp(1, 7)
            lo = hi - 1
            far = (grid[hi] - m) - (m - grid[lo])                # > 0: the lower one is nearer
            pick = torch.where((far > 0) | ((far == 0) & (lo % 2 == 0)), lo, hi)
            return (torch.sign(g) * grid[pick] * torch.exp2(e)).flatten(-2)

        out = {"q": turned(q, s["qn"]), "k": turned(k, s["kn"])}
        return out if kind == "heads" else {"q": out["q"], "k": four(out["k"]), "v": four(v)}
    hq, kv, d = case["q_heads"], case["kv_heads"], case["dim"]
    if n * kv > 4096 or case["ctx"] * T * hq > 1 << 30:
        return None
    grid = np.array(GRID)
    lut = torch.from_numpy(np.concatenate([grid, -grid])).to(DEV)
    out = torch.empty(n * T, hq, d, dtype=torch.float64, device=DEV)

    def stored(codes, scales):
        lo, hi = codes.long() & 15, codes.long() >> 4
        x = torch.stack([lut[lo], lut[hi]], -1).flatten(-2)
        return x * torch.exp2(scales.double() - 127).repeat_interleave(32, -1)

    for i in range(n):
        end = int(s["pos"][i]) + T
        rows = torch.from_numpy(at[i * T:(i + 1) * T]).to(DEV)[:, None]
        j = torch.arange(end, device=DEV)[None]
        hide = j > rows
        if case["window"]:
            hide = hide | ((j <= rows - case["window"]) & (j >= case["sinks"]))
        for h in range(kv):
            K, V = stored(s["kc"][i, h, :end], s["ks"][i, h, :end]), stored(s["vc"][i, h, :end], s["vs"][i, h, :end])
            for a in range(h * hq // kv, (h + 1) * hq // kv):
                w = (s["q"][i * T:(i + 1) * T, a].double() @ K.T / math.sqrt(d)).masked_fill_(hide, -math.inf).softmax(-1)
                out[i * T:(i + 1) * T, a] = w @ V
    return out / (1 + torch.exp(-s["gate"].double()))
