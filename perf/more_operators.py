"""The operators of many answers to one prompt, as they are measured: the heads' norms and rotation by
positions on several axes (a prompt with images), with and without the 4-bit K/V cache's append; the
attention of a batch that shares a long prefix, held and read once for all; and the log probabilities of
the tokens that were answered, with their ranks, the entropy and the most likely alternatives.

`own` false: the same results from elementary torch operations (float32; float64 for angles and long
sums), on the same inputs. `own` true: the calls of a program that uses qwen35 (include/q35.h).

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
def _heads(seqs, rows, pos, q, kv, dim, rot, axes, dealt):
    return {"seqs": seqs, "rows": rows, "pos": pos, "q_heads": q, "kv_heads": kv, "dim": dim, "rot": rot, "axes": axes,
            "dealt": dealt}


def _shared(groups, each, rows, prefix, tail, q, kv, dim, ragged, gate):
    return {"groups": groups, "each": each, "rows": rows, "prefix": prefix, "tail": tail, "q_heads": q, "kv_heads": kv,
            "dim": dim, "ragged": ragged, "gate": gate}


def _logprobs(rows, vocab, top, bf16, temp, masked):
    return {"rows": rows, "vocab": vocab, "top": top, "bf16": bf16, "temp": temp, "masked": masked}


def listed():
    return [
        # A layer's heads: one answer's step behind a long prompt with images; a prompt of images and
        # text, its pairs dealt to time, height and width in turn.
        {"name": "axes_rope_1", "kind": "rope", **_heads(1, 1, 32000, 8, 2, 256, 64, 3, True)},
        {"name": "axes_rope_4096", "kind": "rope", **_heads(1, 4096, 0, 8, 2, 256, 64, 3, True)},
        # The same with the append, at slots that are not the positions: a step of the headline batch;
        # a prompt of odd length of a layer whose whole head is rotated, its pairs in sections.
        {"name": "axes_append_256", "kind": "append", **_heads(256, 1, 4096, 8, 2, 256, 64, 3, True)},
        {"name": "axes_append_1999", "kind": "append", **_heads(1, 1999, 2048, 32, 8, 128, 128, 3, False)},
        # Attention of answers to shared prompts: four answers to one short question; the headline batch over
        # one prompt; eight prompts with 32 answers each of many lengths; a speculative round's 3 rows an answer;
        # the headline batch over one long document.
        {"name": "shared_4x1999", "kind": "shared", **_shared(1, 4, 1, 1999, 65, 8, 2, 256, False, True)},
        {"name": "shared_256x4096", "kind": "shared", **_shared(1, 256, 1, 4096, 256, 8, 2, 256, True, True)},
        {"name": "shared_8x32x8192", "kind": "shared", **_shared(8, 32, 1, 8192, 512, 32, 4, 128, True, False)},
        {"name": "shared_verify_64x2000", "kind": "shared", **_shared(1, 64, 3, 2000, 300, 8, 2, 256, True, True)},
        {"name": "shared_256x32768", "kind": "shared", **_shared(1, 256, 1, 32768, 128, 8, 2, 256, False, True)},
        # Log probabilities: one step of one answer with its 20 alternatives; a step of the headline batch with 5;
        # a scored prompt's rows of a bfloat16 head over an odd vocabulary, a quarter of which a grammar bars.
        {"name": "logprobs_1", "kind": "logprobs", **_logprobs(1, VOCAB, 20, False, 1.0, False)},
        {"name": "logprobs_256", "kind": "logprobs", **_logprobs(256, VOCAB, 5, False, 1.0, False)},
        {"name": "logprobs_1999_odd", "kind": "logprobs", **_logprobs(1999, 32003, 20, True, 0.7, True)},
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


LAYOUTS = [(8, 2, 256), (8, 2, 256), (32, 8, 128), (32, 4, 128), (16, 16, 64), (14, 2, 64), (5, 1, 128), (48, 3, 256)]


def draw(rng):
    kind = rng.choice(["rope", "append", "shared", "shared", "shared", "logprobs", "logprobs"])
    q, kv, dim = rng.choice(LAYOUTS)
    if kind in ("rope", "append"):
        seqs = _log_int(rng, 1, 256)
        rot = rng.choice([dim, dim // 2, dim // 4])
        return {"kind": kind, **_heads(seqs, _log_int(rng, 1, max(1, 4096 // seqs)), _log_int(rng, 1, 131072 if
                                       kind == "rope" else 4096), q, kv, dim, rot, rng.choice([1, 2, 3, 3, 4]),
                                       rng.random() < 0.5)}
    if kind == "shared":
        groups = rng.choice([1, 1, 1, 2, 3, _log_int(rng, 1, 16)])
        each = _log_int(rng, 1, 256 // groups)
        rows = rng.choice([1, 1, 1, 2, 3, 5])
        most = max(64, min(32768, (1 << 34) // (groups * each * rows * q * dim), (1 << 28) // (groups * kv * dim)))
        tail = _log_int(rng, rows, max(rows, min(1024, (1 << 27) // (groups * each * kv * dim))))
        return {"kind": kind, **_shared(groups, each, rows, _log_int(rng, 1, most), tail, q, kv, dim, rng.random() < 0.5,
                                        rng.random() < 0.5)}
    vocab = rng.choice([VOCAB, 32003, 151_936, 50257, _log_int(rng, 128, VOCAB)])
    return {"kind": kind, **_logprobs(_log_int(rng, 1, max(1, min(4096, 64_000_000 // vocab))), vocab, rng.choice([0, 1, 5, 20, 32]),
                                      rng.random() < 0.5, rng.choice([1.0, 1.0, 0.7, 1.3]), rng.random() < 0.3)}


# ------------------------------------------------------------------------------ inputs
def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(int(seed))


def _bf16(g, *shape, scale=1.0):
    return (torch.randn(*shape, generator=g, device=DEV) * scale).to(torch.bfloat16)


def _axis_of_pair(case):
    """The axis of each pair of dims: dealt out in turn, or in sections."""
    pairs, axes = case["rot"] // 2, case["axes"]
    if case["dealt"]:
        return np.arange(pairs) % axes
    return np.arange(pairs) * axes // pairs


def _positions(case, seed):
    """Positions [seqs * rows][axes]: runs of text, the same on every axis, and images, whose rows and columns count
    from the position where the image begins; the text goes on behind the largest of them."""
    rng = np.random.default_rng(seed)
    axes, out = case["axes"], []
    for _ in range(case["seqs"]):
        at, left = case["pos"] + int(rng.integers(0, 64)), case["rows"]
        while left > 0:
            text = min(left, int(rng.integers(1, 200)))
            out.append(np.repeat(at + np.arange(text), axes).reshape(text, axes))
            at, left = at + text, left - text
            h, w = int(rng.integers(4, 33)), int(rng.integers(4, 33))
            cells = min(left, h * w)
            if cells:
                i = np.arange(cells)
                grid = np.stack([np.zeros_like(i), i // w, i % w, i // w], 1)[:, :axes]
                out.append(at + grid)
                at, left = at + max(h, w), left - cells
    return np.concatenate(out).astype(np.int32)


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


def _spread(n, last, ragged):
    """n numbers: all `last`, or spread evenly from an eighth of it up."""
    i = np.arange(n)
    return (last - (i * (last - last // 8) // n if ragged else 0 * i)).astype(np.int32)


def _inputs(case, seed):
    """What the call reads, from the seed alone."""
    g, kind = _gen(seed), case["kind"]
    s = {"case": case}
    if kind in ("rope", "append"):
        q, kv, d, R = case["q_heads"], case["kv_heads"], case["dim"], case["seqs"] * case["rows"]
        # a projection's rows: (q | gate) per q head, then k, then v
        s["proj"] = _bf16(g, R, (2 * q + 2 * kv) * d)
        s["qn"], s["kn"] = _bf16(g, d, scale=0.1), _bf16(g, d, scale=0.1)
        s["at"] = torch.from_numpy(_positions(case, seed)).to(DEV)
    elif kind == "shared":
        G, n, T = case["groups"], case["groups"] * case["each"], case["rows"]
        q, kv, d = case["q_heads"], case["kv_heads"], case["dim"]
        s["pk"], s["pks"] = _cache_rows(g, G, kv, case["prefix"], d)
        s["pv"], s["pvs"] = _cache_rows(g, G, kv, case["prefix"], d)
        s["tk"], s["tks"] = _cache_rows(g, n, kv, case["tail"], d)
        s["tv"], s["tvs"] = _cache_rows(g, n, kv, case["tail"], d)
        s["q"] = _bf16(g, n * T, q, d)
        s["gate"] = _bf16(g, n * T, q, d) if case["gate"] else None
        rng = np.random.default_rng(seed)
        s["plen"] = _spread(G, case["prefix"], case["ragged"] and G > 1)
        # the last row's slot of each answer: T - 1 or more
        s["pos"] = rng.permutation(np.maximum(_spread(n, case["tail"], case["ragged"]), T) - T).astype(np.int32)
    else:
        n, v = case["rows"], case["vocab"]
        lg = torch.randn(n, v, generator=g, device=DEV) * 2.0
        if case["masked"]:            # the words that a grammar bars
            lg.masked_fill_(torch.rand(v, generator=g, device=DEV) < 0.25, -math.inf)
        hot = torch.randint(0, v, (n, 40), generator=g, device=DEV)
        lg.scatter_reduce_(1, hot, 8.0 + 3.0 * torch.randn(n, 40, generator=g, device=DEV), "amax")
        lg = lg.to(torch.bfloat16)                    # a bf16 head's logits
        s["logits"] = lg if case["bf16"] else lg.float()
        s["targets"] = hot[:, 0].int().contiguous()   # what was answered
    return s


def prepare(case, seed):
    s, kind = _inputs(case, seed), case["kind"]
    if own:
        s["eng"] = engine()
        from qwen35 import KvCache4
        bf16 = functools.partial(torch.empty, dtype=torch.bfloat16, device=DEV)
        if kind in ("rope", "append"):
            q, kv, d, n, T = case["q_heads"], case["kv_heads"], case["dim"], case["seqs"], case["rows"]
            s["qo"], s["ko"], s["vo"] = bf16(n * T, q, d), bf16(n * T, kv, d), bf16(n * T, kv, d)
            s["axis"] = _axis_of_pair(case).astype(np.uint8)
            if kind == "append":
                s["cache"] = KvCache4(s["eng"], n, 16 + T, kv_heads=kv, head_dim=d)
                s["slots"] = np.full(n, 16, np.int32)             # behind 16 slots that are held already
                s["cache"].set_len(None, s["slots"])
        elif kind == "shared":
            G, n = case["groups"], case["groups"] * case["each"]
            kv, d = case["kv_heads"], case["dim"]
            s["out"] = bf16(n * case["rows"], case["q_heads"], d)
            s["lanes"] = np.arange(n, dtype=np.int32)
            s["plane"] = (s["lanes"] // case["each"]).astype(np.int32)
            s["plens"] = s["plen"][s["plane"]]
            s["prefix"] = KvCache4(s["eng"], G, case["prefix"], kv_heads=kv, head_dim=d)
            s["cache"] = KvCache4(s["eng"], n, case["tail"], kv_heads=kv, head_dim=d)
            torch.cuda.synchronize()
            s["prefix"].write(0, 0, G, 0, case["prefix"], *[s[k].data_ptr() for k in ("pk", "pks", "pv", "pvs")])
            s["cache"].write(0, 0, n, 0, case["tail"], *[s[k].data_ptr() for k in ("tk", "tks", "tv", "tvs")])
            s["eng"].sync()
            for k in ("pk", "pks", "pv", "pvs", "tk", "tks", "tv", "tvs"):
                del s[k]
        else:
            n, k = case["rows"], case["top"]
            f32, i32 = (functools.partial(torch.empty, dtype=t, device=DEV) for t in (torch.float32, torch.int32))
            s["lp"], s["ent"], s["rank"], s["ids"], s["tlp"] = f32(n), f32(n), i32(n), i32(n, k), f32(n, k)
        torch.cuda.synchronize()          # the engine's stream reads what torch's stream has made
    return s


# ------------------------------------------------------------------------------ the plain forms
def _split(s):
    """The projection's rows as q [R][q][d], k [R][kv][d], v [R][kv][d]."""
    c = s["case"]
    q, kv, d = c["q_heads"], c["kv_heads"], c["dim"]
    x = s["proj"]
    R = x.shape[0]
    return (x[:, :2 * q * d].view(R, q, 2 * d)[..., :d], x[:, 2 * q * d:(2 * q + kv) * d].view(R, kv, d),
            x[:, (2 * q + kv) * d:].view(R, kv, d))


def _angles(s):
    """cos and sin [R][1][rot / 2]: pair i turns by the position on its axis times theta^(-2 i / rot)."""
    c = s["case"]
    rate = THETA ** (torch.arange(c["rot"] // 2, dtype=torch.float64, device=DEV) * (-2.0 / c["rot"]))
    at = s["at"][:, torch.from_numpy(_axis_of_pair(c)).to(DEV, non_blocking=True)].double()
    ang = (at * rate)[:, None]
    return ang.cos().float(), ang.sin().float()


def _norm_rope(x, w, cos, sin, rot):
    """Rows [R][h][d] in float32: the head's RMS norm with weight 1 + w, dims [0, rot) rotated in
    pairs (i, i + rot / 2); sums of squares in float64."""
    xf = x.float()
    rs = (1.0 / (xf.double().square().mean(-1, keepdim=True) + EPS).sqrt()).float()
    y = xf * rs * (1.0 + w.float())
    half = rot // 2
    a, b = y[..., :half], y[..., half:rot]
    return torch.cat([a * cos - b * sin, b * cos + a * sin, y[..., rot:]], -1)


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


def _plain_shared(s):
    c = s["case"]
    G, each, T, hq, kv, d = c["groups"], c["each"], c["rows"], c["q_heads"], c["kv_heads"], c["dim"]
    n, grp = G * each, hq // kv
    q = s["q"].float().view(n, T, kv, grp, d).permute(0, 2, 3, 1, 4)                  # [n][kv][grp][T][d]
    # over the prefixes, the answers of a prompt as rows of one product
    pq = q.reshape(G, each, kv, grp * T, d).transpose(1, 2).reshape(G, kv, each * grp * T, d)
    ps = torch.matmul(pq, _values(s["pk"], s["pks"]).transpose(-1, -2)) * d ** -0.5   # [G][kv][rows][prefix]
    held = torch.arange(c["prefix"], device=DEV) < torch.from_numpy(s["plen"]).to(DEV, non_blocking=True)[:, None]
    ps.masked_fill_(~held[:, None, None], -math.inf)
    # over each answer's own slots
    ts = torch.matmul(q.reshape(n, kv, grp * T, d), _values(s["tk"], s["tks"]).transpose(-1, -2)) * d ** -0.5
    at = torch.from_numpy(s["pos"]).to(DEV, non_blocking=True)[:, None] + torch.arange(T, device=DEV)
    see = torch.arange(c["tail"], device=DEV) <= at[..., None]                        # [n][T][tail]
    ts = ts.view(n, kv, grp, T, -1).masked_fill_(~see[:, None, None], -math.inf).view(G, each, kv, grp * T, -1)
    ts = ts.transpose(1, 2).reshape(G, kv, each * grp * T, -1)
    top = torch.maximum(ps.amax(-1, keepdim=True), ts.amax(-1, keepdim=True))
    pw, tw = torch.exp_(ps - top), torch.exp_(ts - top)
    total = pw.sum(-1, keepdim=True) + tw.sum(-1, keepdim=True)
    o = torch.matmul(pw, _values(s["pv"], s["pvs"]))
    tw = tw.view(G, kv, each, grp * T, -1).transpose(1, 2).reshape(n, kv, grp * T, -1)
    to = torch.matmul(tw, _values(s["tv"], s["tvs"])).view(G, each, kv, grp * T, d).transpose(1, 2)
    o = (o + to.reshape(G, kv, each * grp * T, d)) / total
    o = o.view(G, kv, each, grp, T, d).permute(0, 2, 4, 1, 3, 5).reshape(n * T, hq, d)
    if s["gate"] is not None:
        o = o * torch.sigmoid(s["gate"].float())
    return o.to(torch.bfloat16)


def _plain_logprobs(s):
    c, lg, k = s["case"], s["logits"], s["case"]["top"]
    x = lg.float()
    top = x.amax(-1, keepdim=True)
    z = (x - top) * (1.0 / c["temp"])
    w = torch.exp(z)
    total = w.sum(-1, keepdim=True, dtype=torch.float64)
    log_total = total.log()
    ent = log_total + (w * z.clamp_(min=-200.0)).sum(-1, keepdim=True, dtype=torch.float64) / -total
    t = s["targets"].long()[:, None]
    xt, ids = x.gather(1, t), torch.arange(c["vocab"], device=DEV)
    rank = ((x > xt) | ((x == xt) & (ids < t))).sum(-1)
    # one whole number per id whose order is the logits', the lower id first among equals
    bits = (x + 0.0).view(torch.int32)
    key = (bits ^ ((bits >> 31) & 0x7fffffff)).long() << 32 | (0xffffffff - ids)
    best = 0xffffffff - (torch.topk(key, k, dim=-1).values & 0xffffffff)
    top_lp = (x.gather(1, best) - top).double() / c["temp"] - log_total
    lp = (xt - top).double() / c["temp"] - log_total
    return {"logprobs": lp[:, 0].float(), "entropy": ent[:, 0].float(), "ranks": rank.int(), "top_ids": best.int(),
            "top_logprobs": top_lp.float()}


# ------------------------------------------------------------------------------ one pass
def _view(t, heads, off=0, head=None):
    """Rows of heads in a buffer: address, elements from row to row, elements from head to head."""
    return t.data_ptr() + 2 * off, t.stride(0), head or t.shape[-1]


def run(s):
    c = s["case"]
    kind = c["kind"]
    if not own:
        if kind == "shared":
            return _plain_shared(s)
        if kind == "logprobs":
            return _plain_logprobs(s)
        q, k, v = _split(s)
        turn = _angles(s)
        q, k = _norm_rope(q, s["qn"], *turn, c["rot"]).to(torch.bfloat16), _norm_rope(k, s["kn"], *turn, c["rot"])
        if kind == "rope":
            return {"q": q, "k": k.to(torch.bfloat16)}
        return {"q": q, "k": _through_4_bits(k).to(torch.bfloat16), "v": _through_4_bits(v.float()).to(torch.bfloat16)}
    eng = s["eng"]
    if kind in ("rope", "append"):
        q, kv, d, x = c["q_heads"], c["kv_heads"], c["dim"], s["proj"]
        rows = {"q": _view(x, q, 0, 2 * d), "k": _view(x, kv, 2 * q * d, d), "q_norm": s["qn"].data_ptr(),
                "k_norm": s["kn"].data_ptr(), "q_out": _view(s["qo"], q), "k_out": _view(s["ko"], kv),
                "rot_dim": c["rot"], "theta": THETA, "eps": EPS}
        at = (s["at"].data_ptr(), s["at"].stride(0), s["at"].stride(1))
        if kind == "rope":
            eng.op_qk_norm_rope_axes(at, s["axis"], c["seqs"] * c["rows"], q, kv, d, **rows)
            return {"q": s["qo"], "k": s["ko"]}
        eng.op_kv4_append_axes(s["cache"], 0, None, s["slots"], c["rows"], q, at, s["axis"],
                               v=_view(x, kv, (2 * q + kv) * d, d), v_out=_view(s["vo"], kv), **rows)
        return {"q": s["qo"], "k": s["ko"], "v": s["vo"]}
    if kind == "shared":
        h = c["q_heads"]
        eng.op_attn_kv4_shared(s["prefix"], s["cache"], 0, s["plane"], s["plens"], s["lanes"], s["pos"], c["rows"], h,
                               _view(s["q"], h), _view(s["out"], h), gate=_view(s["gate"], h) if c["gate"] else None)
        return s["out"]
    eng.op_token_logprobs(c["rows"], c["vocab"], s["logits"].data_ptr(), targets=s["targets"].data_ptr(),
                          logprobs=s["lp"].data_ptr(), ranks=s["rank"].data_ptr(), entropy=s["ent"].data_ptr(), top=c["top"],
                          top_ids=s["ids"].data_ptr(), top_logprobs=s["tlp"].data_ptr(), temperature=c["temp"],
                          bf16=c["bf16"])
    return {"logprobs": s["lp"], "entropy": s["ent"], "ranks": s["rank"], "top_ids": s["ids"], "top_logprobs": s["tlp"]}


# ------------------------------------------------------------------------------ floors
def work(case):
    """Bytes and operations of one pass: inputs read once, outputs written once."""
    kind = case["kind"]
    if kind in ("rope", "append"):
        q, kv, d, R = case["q_heads"], case["kv_heads"], case["dim"], case["seqs"] * case["rows"]
        b = R * d * (2 * q + 2 * kv) * 2 + 4 * d + R * case["axes"] * 4
        if kind == "append":      # v in, the values that k's and v's codes stand for, the codes and scales
            b += R * d * kv * (2 + 2 + 2 * (0.5 + 1 / 32))
        return {"bytes": b, "flops": R * d * (q + kv) * 8}
    if kind == "shared":
        G, n, T, hq, d = case["groups"], case["groups"] * case["each"], case["rows"], case["q_heads"], case["dim"]
        plen = _spread(G, case["prefix"], case["ragged"] and G > 1).astype(np.int64)
        end = np.maximum(_spread(n, case["tail"], case["ragged"]), T).astype(np.int64)
        pairs = int(plen.sum()) * case["each"] * T + int(end.sum()) * T - n * T * (T - 1) // 2
        return {"bytes": int(plen.sum() + end.sum()) * case["kv_heads"] * (d + d // 16) + n * T * hq * d * (6 if case["gate"] else 4),
                "flops": 4 * pairs * hq * d}
    n = case["rows"]
    return {"bytes": n * case["vocab"] * (2 if case["bf16"] else 4) + n * (16 + 8 * case["top"]),
            "flops": n * case["vocab"] * 6}


# ------------------------------------------------------------------------------ the same in 64 bits
def exact(case, seed):
    kind = case["kind"]
    s = _inputs(case, seed)
    if kind == "logprobs":
        n, k = case["rows"], case["top"]
        t = s["targets"].long()
        lp, ent = (torch.empty(n, dtype=torch.float64, device=DEV) for _ in range(2))
        tlp = torch.empty(n, k, dtype=torch.float64, device=DEV)
        for i in range(0, n, 256):
            x = torch.log_softmax(s["logits"][i:i + 256].double() / case["temp"], -1)
            lp[i:i + 256] = x[torch.arange(x.shape[0], device=DEV), t[i:i + 256]]
            ent[i:i + 256] = torch.special.entr(x.exp()).sum(-1)
            tlp[i:i + 256] = x.sort(-1, descending=True).values[:, :k]
        return {"logprobs": lp, "entropy": ent, "ranks": None, "top_ids": None, "top_logprobs": tlp}
    if kind in ("rope", "append"):
        q, k, v = (t.double() for t in _split(s))
        rot = case["rot"]
        axis = _axis_of_pair(case)
        at = s["at"].cpu().numpy().astype(np.float64)
        th = torch.from_numpy(at[:, axis] * np.exp(np.arange(rot // 2) * (-2.0 / rot) * math.log(THETA))).to(DEV)

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
        return out if kind == "rope" else {"q": out["q"], "k": four(out["k"]), "v": four(v)}
    G, each, T, hq, kv, d = (case[k] for k in ("groups", "each", "rows", "q_heads", "kv_heads", "dim"))
    n, grp = G * each, hq // kv
    if n * kv > 4096:
        return None
    grid = np.array(GRID)
    lut = torch.from_numpy(np.concatenate([grid, -grid])).to(DEV)

    def stored(codes, scales):
        lo, hi = codes.long() & 15, codes.long() >> 4
        x = torch.stack([lut[lo], lut[hi]], -1).flatten(-2)
        return x * torch.exp2(scales.double() - 127).repeat_interleave(32, -1)

    out = torch.empty(n * T, hq, d, dtype=torch.float64, device=DEV)
    for j in range(G):
        P = int(s["plen"][j])
        for h in range(kv):
            pk, pv = stored(s["pk"][j, h, :P], s["pks"][j, h, :P]), stored(s["pv"][j, h, :P], s["pvs"][j, h, :P])
            for i in range(j * each, (j + 1) * each):
                end = int(s["pos"][i]) + T
                K = torch.cat([pk, stored(s["tk"][i, h, :end], s["tks"][i, h, :end])])
                V = torch.cat([pv, stored(s["tv"][i, h, :end], s["tvs"][i, h, :end])])
                rows = s["q"][i * T:(i + 1) * T, h * grp:(h + 1) * grp].double()              # [T][grp][d]
                last = P + end - T + torch.arange(T, device=DEV)
                hide = torch.arange(P + end, device=DEV) > last[:, None]
                w = torch.matmul(rows, K.T).div_(math.sqrt(d)).masked_fill_(hide[:, None], -math.inf).softmax(-1)
                out[i * T:(i + 1) * T, h * grp:(h + 1) * grp] = torch.matmul(w, V)
    return out / (1 + torch.exp(-s["gate"].double())) if case["gate"] else out
