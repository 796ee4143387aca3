"""The 4-bit cache's operators against float64 (tests/kv4_ref.py), at the layouts, lengths, windows and
values where they can go wrong, and a layer's rounds through them in a row.

Tolerances. Norm and rotation: the float32 steps (root, product, weight, cosine, two products, a sum) are
eight roundings of 2^-24 on |a| + |b| of the rotated pair, then bf16's 2^-8 of the result. Codes: a code is
a nearest one to a value known to those eight roundings, the scale byte the rule's unless the group's
largest magnitude lies that near a border. Attention: kv4_ref.attention_bound."""
import numpy as np
import pytest

import kv4_ref as ref

pytestmark = pytest.mark.gpu

SLACK = 8 * 2.0 ** -24


@pytest.fixture(scope="module")
def eng():
    from qwen35 import Engine
    e = Engine(max_rows=64, max_ctx=40000, seed=None)
    yield e
    e.close()


class Dev:
    """Host arrays on the device and back."""

    def __init__(self):
        import torch
        self.t = torch

    def up(self, a):
        a = np.ascontiguousarray(a)
        t = self.t.from_numpy(a.view({2: np.int16, 4: np.int32, 1: np.uint8}[a.dtype.itemsize])).cuda()
        return t

    def bits(self, t):
        return t.cpu().numpy().view(np.uint16)


def bf16_randn(rng, *shape, scale=1.0):
    return ref.bf16_bits(rng.standard_normal(shape) * scale)


def read_cache(eng, c, layer, lane0, n, slot0, m):
    import torch
    kc, ks = (torch.zeros(n, c.kv_heads, m, c.head_dim // w, dtype=torch.uint8, device="cuda") for w in (2, 32))
    vc, vs = torch.zeros_like(kc), torch.zeros_like(ks)
    torch.cuda.synchronize()
    c.read(layer, lane0, n, slot0, m, *[x.data_ptr() for x in (kc, ks, vc, vs)])
    eng.sync()
    return [x.cpu().numpy() for x in (kc, ks, vc, vs)]


class Heads:
    """Projection rows (q | gate) x hq, k x kv, v x kv, with `pad` spare elements a row."""

    def __init__(self, rng, R, hq, kv, d, pad=0):
        self.hq, self.kv, self.d, self.R = hq, kv, d, R
        self.width = (2 * hq + 2 * kv) * d + pad
        self.x = bf16_randn(rng, R, self.width)
        self.qn, self.kn = bf16_randn(rng, d, scale=0.1), bf16_randn(rng, d, scale=0.1)

    def parts(self):
        x, d = ref.val(self.x), self.d
        a, b = 2 * self.hq * d, (2 * self.hq + self.kv) * d
        return (x[:, :a].reshape(self.R, self.hq, 2 * d)[..., :d], x[:, a:b].reshape(self.R, self.kv, d),
                x[:, b:b + self.kv * d].reshape(self.R, self.kv, d))

    def views(self, p):
        w, d = self.width, self.d
        return {"q": (p, w, 2 * d), "k": (p + 2 * (2 * self.hq) * d, w, d)}, (p + 2 * (2 * self.hq + self.kv) * d, w, d)


def check_norm_rope(bits, x, w, pos, rot, theta, eps):
    want, size = ref.norm_rope(x, ref.val(w), pos, rot, theta, eps)
    assert np.all(np.abs(ref.val(bits) - want) <= 2.0 ** -8 * np.abs(want) + SLACK * size + 1e-37)
    return want


@pytest.mark.parametrize("hq,kv,d,rot", [(8, 2, 256, 64), (8, 2, 256, 256), (5, 1, 128, 128), (3, 3, 128, 0), (14, 2, 64, 64),
                                         (1, 7, 64, 6), (2, 1, 256, 2), (4, 2, 128, 100)])
@pytest.mark.parametrize("n,T", [(1, 1), (3, 5), (300, 1)])
def test_norm_rope(eng, hq, kv, d, rot, n, T):
    import torch
    print(f"norm_rope {hq} {kv} {d} {rot} {n}x{T}", flush=True)
    rng, D = np.random.default_rng(hq * d + rot + n), Dev()
    h = Heads(rng, n * T, hq, kv, d, pad=8)
    h.x[0, :d] = 0                                # a head of zeros
    if n * T > 1:
        h.x[1, :d] = ref.bf16_bits(rng.standard_normal(d) * 1e-18)
        h.x[1, 2 * d:3 * d] = ref.bf16_bits(rng.standard_normal(d) * 1e18)
    pos = rng.integers(0, 200000, n).astype(np.int32)
    pos[0] = 0
    x, qn, kn = D.up(h.x), D.up(h.qn), D.up(h.kn)
    qo = torch.zeros(n * T, hq + 1, d, dtype=torch.int16, device="cuda")
    ko = torch.zeros(kv, n * T, d, dtype=torch.int16, device="cuda")         # heads outside, rows inside
    torch.cuda.synchronize()
    v, _ = h.views(x.data_ptr())
    eng.op_qk_norm_rope(pos, T, hq, kv, d, rot_dim=rot, theta=1e6, eps=1e-6, q_norm=qn.data_ptr(), k_norm=kn.data_ptr(),
                        q_out=(qo.data_ptr(), (hq + 1) * d, d), k_out=(ko.data_ptr(), d, n * T * d), **v)
    eng.sync()
    at = (pos[:, None] + np.arange(T)).reshape(-1).astype(np.float64)
    q, k, _ = h.parts()
    got = D.bits(qo)
    check_norm_rope(got[:, :hq], q, h.qn, at, rot, 1e6, 1e-6)
    check_norm_rope(D.bits(ko).transpose(1, 0, 2), k, h.kn, at, rot, 1e6, 1e-6)
    assert not got[:, hq].any()                   # what lies between the rows' heads stays
    # in place gives the same bits, and k alone leaves q out
    eng.op_qk_norm_rope(pos, T, hq, kv, d, rot_dim=rot, theta=1e6, eps=1e-6, q_norm=qn.data_ptr(), k_norm=kn.data_ptr(),
                        q_out=v["q"], k_out=v["k"], **v)
    eng.sync()
    y = D.bits(x)
    assert np.array_equal(y[:, :2 * hq * d].reshape(n * T, hq, 2, d)[:, :, 0], got[:, :hq])
    assert np.array_equal(y[:, 2 * hq * d:(2 * hq + kv) * d].reshape(n * T, kv, d), D.bits(ko).transpose(1, 0, 2))
    assert np.array_equal(y[:, (2 * hq + kv) * d:], h.x[:, (2 * hq + kv) * d:])


def check_codes(x, codes, scales, slack):
    """Codes and scale bytes of rows x [..][d] known within slack."""
    amax = np.abs(x).reshape(*x.shape[:-1], -1, 32).max(-1)
    lo, hi = ref.scale_byte(amax * (1 - slack)), ref.scale_byte(amax * (1 + slack))
    assert np.all((scales >= lo) & (scales <= hi))
    assert np.all(ref.nearest_ok(x, codes, scales, slack))


@pytest.mark.parametrize("hq,kv,d,rot", [(8, 2, 256, 64), (5, 1, 128, 128), (4, 4, 64, 32)])
@pytest.mark.parametrize("n,T,pos0", [(1, 1, 0), (4, 3, 30), (2, 70, 17), (270, 1, 5)])
def test_append(eng, hq, kv, d, rot, n, T, pos0):
    import torch
    from qwen35 import KvCache4
    print(f"append {hq} {kv} {d} {rot} {n}x{T}@{pos0}", flush=True)
    rng, D = np.random.default_rng(n * T + d), Dev()
    cap = pos0 + n + T + 2
    c = KvCache4(eng, n + 1, cap, layers=2, kv_heads=kv, head_dim=d)
    lanes = rng.permutation(n + 1)[:n].astype(np.int32)
    pos = (pos0 + np.arange(n) % 7).astype(np.int32)
    c.set_len(None, np.full(n + 1, cap, np.int32))
    before = read_cache(eng, c, 1, 0, n + 1, 0, cap)
    c.set_len(lanes, pos)
    h = Heads(rng, n * T, hq, kv, d)
    _, _, vv = h.parts()
    x, qn, kn = D.up(h.x), D.up(h.qn), D.up(h.kn)
    qo, ko, vo = (torch.zeros(n * T, m, d, dtype=torch.int16, device="cuda") for m in (hq, kv, kv))
    torch.cuda.synchronize()
    v, vview = h.views(x.data_ptr())
    args = dict(rot_dim=rot, theta=1e7, eps=1e-6, q_norm=qn.data_ptr(), k_norm=kn.data_ptr(), v=vview, **v)
    eng.op_kv4_append(c, 1, lanes, pos, T, hq, q_out=(qo.data_ptr(), hq * d, d), k_out=(ko.data_ptr(), kv * d, d),
                      v_out=(vo.data_ptr(), kv * d, d), **args)
    eng.sync()
    assert [c.length(1, l) for l in lanes] == list(pos + T) and [c.length(0, l) for l in lanes] == list(pos)
    q, k, vx = h.parts()
    at = (pos[:, None] + np.arange(T)).reshape(-1).astype(np.float64)
    check_norm_rope(D.bits(qo), q, h.qn, at, rot, 1e7, 1e-6)
    want, size = ref.norm_rope(k, ref.val(h.kn), at, rot, 1e7, 1e-6)
    c.set_len(None, np.full(n + 1, cap, np.int32))
    kc, ks, vc, vs = read_cache(eng, c, 1, 0, n + 1, 0, cap)
    rows = lambda a: np.concatenate([a[l, :, p:p + T].transpose(1, 0, 2) for l, p in zip(lanes, pos)])  # noqa: E731
    # a rotated value's error is relative to its pair, so the borders' slack is widened there
    wide = SLACK * np.maximum(size / np.maximum(np.abs(want), 1e-30), 1)
    amax = np.abs(want).reshape(*want.shape[:-1], -1, 32).max(-1)
    gw = (SLACK * size).reshape(*want.shape[:-1], -1, 32).max(-1)
    assert np.all((rows(ks) >= ref.scale_byte(amax - gw)) & (rows(ks) <= ref.scale_byte(amax + gw)))
    assert np.all(ref.nearest_ok(want, rows(kc), rows(ks), wide))
    check_codes(vx, rows(vc), rows(vs), 0.0)
    assert np.array_equal(ref.val(D.bits(ko)), ref.values(rows(kc), rows(ks)))
    assert np.array_equal(ref.val(D.bits(vo)), ref.values(rows(vc), rows(vs)))
    # every other slot, lane and layer as it was
    after, now = (kc, ks, vc, vs), read_cache(eng, c, 0, 0, n + 1, 0, cap)
    for a, b, z in zip(after, before, now):
        a = a.copy()
        for l, p in zip(lanes, pos):
            a[l, :, p:p + T] = b[l, :, p:p + T]
        assert np.array_equal(a, b) and not z.any()
    c.close()


def test_append_special_values(eng):
    """Groups of zeros, of tiny and of huge values, on the code borders, and with an infinity or a NaN."""
    import torch
    from qwen35 import KvCache4
    D, d = Dev(), 128
    v = np.zeros((8, 1, d))
    v[1] = 2.0 ** -130
    v[2] = 3e38
    mids = np.array([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 6.0])
    v[3] = np.tile(np.concatenate([mids, -mids]), d // 16)
    v[4] = v[3] * 2.0 ** -118
    v[5], v[5, 0, 40] = 1.0, np.inf
    v[6], v[6, 0, 127] = 1.0, np.nan
    v[7] = np.tile(np.array([6.03125, -1.0, 0.1, 5.9]), d // 4)
    x = np.zeros((8, 3 * d), np.uint16)
    x[:, 2 * d:] = ref.bf16_bits(v[:, 0])
    x[:, :d] = 0x3F80
    c = KvCache4(eng, 1, 64, kv_heads=1, head_dim=d)
    t, w = D.up(x), D.up(np.zeros(d, np.uint16))
    ko, vo = (torch.zeros(8, d, dtype=torch.int16, device="cuda") for _ in range(2))
    torch.cuda.synchronize()
    p = t.data_ptr()
    eng.op_kv4_append(c, 0, [0], [0], 8, 1, rot_dim=0, theta=1.0, eps=0.0, q_norm=w.data_ptr(), k_norm=w.data_ptr(),
                      k=(p, 3 * d, d), v=(p + 4 * d, 3 * d, d), k_out=(ko.data_ptr(), d, d), v_out=(vo.data_ptr(), d, d))
    eng.sync()
    kc, ks, vc, vs = read_cache(eng, c, 0, 0, 1, 0, 8)
    got, b = ref.values(vc[0, 0], vs[0, 0]), vs[0, 0]
    assert np.all(ref.val(D.bits(ko)) == 1.0)
    assert np.all(got[0] == 0) and np.all(b[0] == 8) and np.all(got[1] == 0) and np.all(b[1] == 8)
    assert np.all(b[2] == 252) and np.all(got[2] == 6 * 2.0 ** 125)
    even = np.array([0, 1, 1, 2, 2, 4, 4, 6.0])
    assert np.all(b[3] == 127) and np.array_equal(got[3], np.tile(np.concatenate([even, -even]), d // 16))
    assert np.all(b[4] == 9) and np.array_equal(got[4], got[3] * 2.0 ** -118)
    assert np.all(b[5] == [125, 255, 125, 125]) and np.all(np.isnan(got[5, 32:64])) and np.all(got[5, 64:] == 1)
    assert np.all(b[6] == [125, 125, 125, 255]) and np.all(np.isnan(got[6, 96:])) and np.all(got[6, :96] == 1)
    assert np.all(b[7] == 128)
    check_codes(ref.val(ref.bf16_bits(v[7])), vc[0, 0, 7:8], vs[0, 0, 7:8], 0.0)
    out = ref.val(D.bits(vo))
    assert np.array_equal(np.isnan(out), np.isnan(got)) and np.array_equal(out[~np.isnan(got)], got[~np.isnan(got)])
    c.close()


class Filled:
    """A cache of one layer whose lanes hold `cap` random slots, with their values on the host."""

    def __init__(self, eng, rng, lanes, cap, kv, d, nan=()):
        import torch
        from qwen35 import KvCache4
        self.c = KvCache4(eng, lanes, cap, kv_heads=kv, head_dim=d)
        codes = lambda: rng.integers(0, 256, (lanes, kv, cap, d // 2)).astype(np.uint8)          # noqa: E731
        scales = lambda: rng.integers(124, 127, (lanes, kv, cap, d // 32)).astype(np.uint8)      # noqa: E731
        kc, ks, vc, vs = codes(), scales(), codes(), scales()
        for what, lane, head, slot, blk in nan:
            (ks if what == "k" else vs)[lane, head, slot, blk] = 255
        t = [torch.from_numpy(a).cuda() for a in (kc, ks, vc, vs)]
        torch.cuda.synchronize()
        self.c.write(0, 0, lanes, 0, cap, *[x.data_ptr() for x in t])
        eng.sync()
        back = read_cache(eng, self.c, 0, 0, lanes, 0, cap)
        assert all(np.array_equal(a, b) for a, b in zip(back, (kc, ks, vc, vs)))
        self.K, self.V = ref.values(kc, ks), ref.values(vc, vs)


def run_attention(eng, f, lanes, pos, T, hq, rng, window=0, sinks=0, gated=False, scale=None, spread=0):
    """One call on random q; returns (bits of out, q, gate), and checks the elements between the rows."""
    import torch
    D, n, d = Dev(), len(pos), f.c.head_dim
    qb, gb = bf16_randn(rng, n * T, hq, d), bf16_randn(rng, n * T, hq, d)
    q, g = D.up(qb), D.up(gb)
    out = torch.full((n * T + 1, hq, d + spread), 0x1234, dtype=torch.int16, device="cuda")
    torch.cuda.synchronize()
    eng.op_attn_kv4(f.c, 0, lanes, pos, T, hq, (q.data_ptr(), hq * d, d), (out.data_ptr(), hq * (d + spread), d + spread),
                    scale=scale, window=window, sinks=sinks, gate=(g.data_ptr(), hq * d, d) if gated else None)
    eng.sync()
    o = D.bits(out)
    assert np.all(o[n * T:] == 0x1234) and np.all(o[:, :, d:] == 0x1234)
    return o[:n * T, :, :d], ref.val(qb), ref.val(gb) if gated else None


def check_attention(f, lanes, pos, T, got, q, gate, window=0, sinks=0, scale=None):
    d = f.c.head_dim
    sc = d ** -0.5 if scale is None else scale
    for i, (l, p) in enumerate(zip(lanes, pos)):
        r = slice(i * T, (i + 1) * T)
        out, pv, big = ref.attention(q[r], f.K[l], f.V[l], p, window, sinks, sc)
        want, e = ref.attention_bound(out, pv, big, p + T, d, None if gate is None else gate[r])
        g = ref.val(got[r])
        assert np.array_equal(np.isnan(g), np.isnan(want)), f"NaN places of sequence {i}"
        bad = ~np.isnan(want) & ~(np.abs(g - want) <= e)
        assert not bad.any(), (i, int(bad.sum()), float(np.nanmax(np.abs(g - want) / e)))


LAYOUTS = [(8, 2, 256), (32, 8, 128), (14, 2, 64), (5, 1, 128), (6, 6, 64), (48, 3, 256), (40, 1, 128)]


@pytest.mark.parametrize("hq,kv,d", LAYOUTS)
@pytest.mark.parametrize("T", [1, 2, 5, 19])
def test_attention(eng, hq, kv, d, T):
    """Lanes of every length around a tile's ends, some twice, in another order than they lie."""
    rng = np.random.default_rng(hq + d + T)
    f = Filled(eng, rng, 5, 300, kv, d)
    pos = np.array([0, 1, 15, 16, 30, 31, 32, 33, 63, 64, 100, 127, 255, 300 - T], np.int32)
    lanes = rng.integers(0, 5, pos.size).astype(np.int32)
    for gated, window, sinks in [(False, 0, 0), (True, 0, 0), (False, 1, 0), (True, 33, 0), (False, 40, 3), (True, 64, 70),
                                 (False, 1000, 4), (False, 5, 1000)]:
        print(f"attention {hq} {kv} {d} T={T} gated={gated} window={window} sinks={sinks}", flush=True)
        got, q, g = run_attention(eng, f, lanes, pos, T, hq, rng, window, sinks, gated, spread=8)
        check_attention(f, lanes, pos, T, got, q, g, window, sinks)
    f.c.close()


@pytest.mark.parametrize("hq,kv,d", [(8, 2, 256), (32, 4, 128), (4, 4, 64)])
def test_attention_long(eng, hq, kv, d):
    """One lane whose tiles are split over many blocks, in several lengths, alone and beside a short one."""
    rng = np.random.default_rng(d)
    f = Filled(eng, rng, 2, 9001, kv, d)
    for lanes, pos, T, window, sinks in [([0], [9000], 1, 0, 0), ([1, 0], [3, 8998], 3, 0, 0), ([0], [9000], 1, 5000, 40),
                                         ([0, 0, 1], [4095, 4096, 8191], 1, 0, 0), ([1], [8989], 12, 2048, 4)]:
        print(f"attention long {hq} {kv} {d} {lanes} {pos} {T} {window} {sinks}", flush=True)
        got, q, g = run_attention(eng, f, lanes, pos, T, hq, rng, window, sinks, True)
        check_attention(f, lanes, pos, T, got, q, g, window, sinks)
    f.c.close()


@pytest.mark.parametrize("hq,kv,d,ctx,T", [(8, 2, 256, 200, 200), (8, 2, 256, 333, 97), (32, 8, 128, 257, 130), (6, 2, 64, 400, 311),
                                           (5, 1, 128, 129, 65)])
def test_attention_prompt(eng, hq, kv, d, ctx, T):
    """Prompt rows, from the cache's start and behind earlier slots, with and without a window."""
    rng = np.random.default_rng(ctx + T)
    f = Filled(eng, rng, 2, ctx, kv, d)
    for window, sinks, gated in [(0, 0, True), (50, 4, False), (1, 0, False), (ctx, 0, False)]:
        print(f"attention prompt {hq} {kv} {d} {ctx} {T} {window} {sinks}", flush=True)
        lanes, pos = [1, 0], [ctx - T, max(0, ctx - T - 3)]
        got, q, g = run_attention(eng, f, lanes, pos, T, hq, rng, window, sinks, gated)
        check_attention(f, lanes, pos, T, got, q, g, window, sinks)
    f.c.close()


def test_attention_many_lanes(eng):
    """More sequences than one launch takes."""
    rng = np.random.default_rng(5)
    f = Filled(eng, rng, 300, 70, 1, 64)
    lanes, pos = rng.permutation(300).astype(np.int32), rng.integers(0, 69, 300).astype(np.int32)
    got, q, g = run_attention(eng, f, lanes, pos, 2, 3, rng, 16, 2, True)
    check_attention(f, lanes, pos, 2, got, q, g, 16, 2)
    f.c.close()


@pytest.mark.parametrize("hq,kv,d", [(8, 2, 256), (4, 1, 128), (2, 2, 64)])
@pytest.mark.parametrize("T", [1, 3, 40])
def test_attention_nan_slots(eng, hq, kv, d, T):
    """A NaN group of K or V reaches the rows that see its slot, and in V its dims only; masked ones
    (later rows' slots, outside the window, behind the length, behind the capacity's last row) nobody."""
    rng = np.random.default_rng(d + T)
    nan = [("v", 0, 0, 70, 0), ("v", 0, kv - 1, 75, d // 32 - 1), ("v", 1, 0, 3, 1), ("k", 2, 0, 60, 0), ("k", 2, kv - 1, 90, 1),
           ("v", 3, 0, 99, 1), ("k", 3, 0, 98, 0), ("v", 3, 0, 20, 0), ("v", 0, 0, 0, 1)]
    f = Filled(eng, rng, 4, 100, kv, d, nan)
    lanes = np.array([0, 1, 2, 3, 0, 1, 2, 3], np.int32)
    pos = np.array([58, 40, 55, 55, 100 - T, 0, 10, 100 - T], np.int32)
    for window, sinks in [(0, 0), (12, 0), (20, 4), (8, 1)]:
        print(f"attention nan {hq} {kv} {d} T={T} {window} {sinks}", flush=True)
        got, q, g = run_attention(eng, f, lanes, pos, T, hq, rng, window, sinks)
        # the reference, NaN groups taken by who sees them
        for i, (l, p) in enumerate(zip(lanes, pos)):
            for t in range(T):
                j = np.arange(p + t + 1)
                if window:
                    j = j[(j > p + t - window) | (j < sinks)]
                for h in range(hq):
                    k, v = f.K[l][h // (hq // kv)][j], f.V[l][h // (hq // kv)][j]
                    o = ref.val(got[i * T + t, h])
                    if np.isnan(k).any():
                        assert np.isnan(o).all(), (i, t, h)
                        continue
                    assert np.array_equal(np.isnan(o), np.isnan(v).any(0)), (i, t, h)
                    out, pv, big = ref.attention(q[i * T + t:i * T + t + 1, h:h + 1], k[None], v[None], len(j) - 1, 0, 0,
                                                 d ** -0.5)
                    want, e = ref.attention_bound(out, pv, big, p + T, d)
                    ok = ~np.isnan(o)
                    assert np.all(np.abs(o - want[0, 0])[ok] <= e[0, 0][ok]), (i, t, h)
    f.c.close()


def test_attention_extreme_scores(eng):
    """Scores far apart and far from zero: one slot takes all the weight; a scale of 0 and a negative one."""
    rng = np.random.default_rng(11)
    f = Filled(eng, rng, 1, 500, 2, 128)
    for scale in (300.0, 0.0, -2.0, 1e-30):
        got, q, g = run_attention(eng, f, [0], [497], 3, 4, rng, scale=scale)
        check_attention(f, [0], [497], 3, got, q, g, scale=scale)
    f.c.close()


def test_attention_row_is_its_own(eng):
    """A row's bits do not depend on which other sequences the call names (their splits stay the same
    here: one split each), nor on the call being repeated."""
    rng = np.random.default_rng(12)
    f = Filled(eng, rng, 300, 64, 2, 256)
    lanes, pos = np.arange(300, dtype=np.int32), rng.integers(0, 64, 300).astype(np.int32)
    a = run_attention(eng, f, lanes, pos, 1, 8, np.random.default_rng(1))[0]
    b = run_attention(eng, f, lanes, pos, 1, 8, np.random.default_rng(1))[0]
    assert np.array_equal(a, b)
    f.c.close()


def test_write_any_bytes(eng):
    """Codes are stored as they are, scale bytes up to 252 too and larger ones as 255; attention over
    the largest and the smallest scales behind the rows that see none of them stays finite."""
    import torch
    from qwen35 import KvCache4
    rng = np.random.default_rng(14)
    c = KvCache4(eng, 1, 300, kv_heads=1, head_dim=64)
    kc, vc = (rng.integers(0, 256, (1, 1, 300, 32)).astype(np.uint8) for _ in range(2))
    ks, vs = (np.full((1, 1, 300, 2), 126, np.uint8) for _ in range(2))
    ks[0, 0, 40:296, 0], vs[0, 0, 40:296, 1] = np.arange(256), np.arange(256)[::-1]
    t = [torch.from_numpy(a).cuda() for a in (kc, ks, vc, vs)]
    torch.cuda.synchronize()
    c.write(0, 0, 1, 0, 300, *[x.data_ptr() for x in t])
    eng.sync()
    back = read_cache(eng, c, 0, 0, 1, 0, 300)
    ks[ks > 252], vs[vs > 252] = 255, 255
    assert all(np.array_equal(a, b) for a, b in zip(back, (kc, ks, vc, vs)))
    f = Filled.__new__(Filled)
    f.c, f.K, f.V = c, ref.values(kc, ks), ref.values(vc, vs)
    for pos, T, window in [([37], 3, 0), ([298], 2, 3), ([36], 4, 7)]:
        got, q, g = run_attention(eng, f, [0], pos, T, 4, rng, window)
        check_attention(f, [0], pos, T, got, q, g, window)
        assert np.isfinite(ref.val(got)).all()
    c.close()


def test_cache_reuse_and_two_caches(eng):
    """set_len starts a lane over on old contents; two caches of other shapes share the engine's
    workspace in one stream; a closed engine's cache can still be closed."""
    from qwen35 import Engine, KvCache4
    rng = np.random.default_rng(13)
    f = Filled(eng, rng, 2, 5000, 2, 256, [("v", 0, 0, 40, 0), ("k", 0, 1, 4000, 0)])
    h = Filled(eng, rng, 3, 3000, 4, 64)
    for cache, lanes, pos, hq in [(f, [0, 1], [30, 4999], 8), (h, [2, 0], [2999, 10], 4), (f, [1], [4096], 8)]:
        got, q, g = run_attention(eng, cache, lanes, pos, 1, hq, rng)
        check_attention(cache, lanes, pos, 1, got, q, g)
    f.c.close()
    h.c.close()
    e2 = Engine(max_rows=16, max_ctx=64, seed=None)
    c = KvCache4(e2, 1, 64)
    e2.close()
    c.close()


@pytest.mark.parametrize("hq,kv,d,rot,window,sinks", [(8, 2, 256, 64, 0, 0), (8, 2, 256, 64, 24, 4), (12, 3, 128, 128, 40, 0),
                                                      (4, 4, 64, 32, 16, 2)])
def test_rounds_of_a_layer(eng, hq, kv, d, rot, window, sinks):
    """Speculative rounds of one layer as a server runs them, nothing waited for within a round: prompts of several
    lengths, then rounds of 3 rows a lane -- heads and append from the projection's rows where they lie,
    attention with the rows' own gate, verification of drafts -- and the rejected rows dropped, so that
    the next round's append lies on them. Every round's output against float64 on the cache read back."""
    import torch
    from qwen35 import KvCache4
    rng, D, n, k, V = np.random.default_rng(d + window), Dev(), 4, 2, 5003
    c = KvCache4(eng, n, 200, layers=2, kv_heads=kv, head_dim=d)
    lens = np.array([1, 31, 64, 90], np.int32)
    layer = 1

    def layer_call(lanes, pos, T):
        R = len(lanes) * T
        h = Heads(rng, R, hq, kv, d)
        x, qn, kn = D.up(h.x), D.up(h.qn), D.up(h.kn)
        q, out = (torch.zeros(R, hq, d, dtype=torch.int16, device="cuda") for _ in range(2))
        torch.cuda.synchronize()
        p = x.data_ptr()
        v, vv = h.views(p)
        eng.op_kv4_append(c, layer, lanes, pos, T, hq, rot_dim=rot, theta=1e7, eps=1e-6, q_norm=qn.data_ptr(),
                          k_norm=kn.data_ptr(), v=vv, q_out=(q.data_ptr(), hq * d, d), **v)
        eng.op_attn_kv4(c, layer, lanes, pos, T, hq, (q.data_ptr(), hq * d, d), (out.data_ptr(), hq * d, d), window=window,
                        sinks=sinks, gate=(p + 2 * d, h.width, 2 * d))
        return h, x, qn, kn, q, out

    def check(lanes, pos, T, h, q, out):
        gate = ref.val(h.x)[:, :2 * hq * d].reshape(-1, hq, 2 * d)[..., d:]
        for i, (l, p) in enumerate(zip(lanes, pos)):
            kc, ks, vc, vs = read_cache(eng, c, layer, l, 1, 0, p + T)
            K, Vv = ref.values(kc, ks)[0], ref.values(vc, vs)[0]
            r = slice(i * T, (i + 1) * T)
            o, pv, big = ref.attention(ref.val(D.bits(q)[r]), K, Vv, p, window, sinks, d ** -0.5)
            want, e = ref.attention_bound(o, pv, big, p + T, d, gate[r])
            assert np.all(np.abs(ref.val(D.bits(out)[r]) - want) <= e), (l, p)

    for l in range(n):                       # prompts, a lane at a time
        call = layer_call([l], [0], int(lens[l]))
        eng.sync()
        check([l], [0], int(lens[l]), call[0], call[4], call[5])
    taken = set()
    for r in range(4):
        print(f"rounds {hq} {kv} {d} {window} {sinks}: round {r} at {lens.tolist()}", flush=True)
        lanes = rng.permutation(n).astype(np.int32)
        pos = lens[lanes]
        call = layer_call(lanes, pos, k + 1)
        lg = torch.from_numpy(rng.standard_normal((n, k + 1, V)).astype(np.float32)).cuda()
        lg[:, :, 7] = 9.0                    # about half of the probability
        dr = torch.where(torch.from_numpy(rng.random((n, k)) < 0.6).cuda(), 7, 8).int()
        u = torch.from_numpy(rng.random((n, k + 1)).astype(np.float32)).cuda()
        acc, tok = torch.zeros(n, dtype=torch.int32, device="cuda"), torch.zeros(n, k + 1, dtype=torch.int32, device="cuda")
        torch.cuda.synchronize()
        eng.op_draft_verify(n, k, V, lg.data_ptr(), dr.data_ptr(), u.data_ptr(), acc.data_ptr(), tok.data_ptr())
        eng.sync()
        check(lanes, pos, k + 1, call[0], call[4], call[5])
        a = acc.cpu().numpy()
        for i in range(n):
            aa, w, border, near = ref.verify(lg[i].double().cpu().numpy(), dr[i].cpu().numpy(), u[i].double().cpu().numpy(), 1.0)
            assert near > 1e-9 and a[i] == aa and ref.token_ok(int(tok[i, aa]), w, border)
        lens[lanes] = pos + a + 1
        c.set_len(lanes, lens[lanes])
        taken |= set(a.tolist())
        assert [c.length(layer, l) for l in range(n)] == lens.tolist() and c.length(0, 1) == int(lens[1])
    assert len(taken) > 1                    # some rounds dropped rows, some fewer
    c.close()


@pytest.mark.parametrize("hq,kv,d,T", [(8, 2, 64, 1100), (8, 2, 256, 1024), (9, 3, 128, 1300), (32, 4, 64, 700)])
def test_attention_long_prompt(eng, hq, kv, d, T):
    """One prompt of more row tiles than CUs, up to two a CU and more: rows from all over it, and none left out."""
    rng = np.random.default_rng(T)
    f = Filled(eng, rng, 1, T + 37, kv, d)
    for window, sinks in [(0, 0), (100, 5)]:
        print(f"attention long prompt {hq} {kv} {d} {T} {window} {sinks}", flush=True)
        got, q, g = run_attention(eng, f, [0], [37], T, hq, rng, window, sinks, True)
        assert not (got == 0x1234).all(-1).any()
        for t in np.unique(np.r_[0, 1, T - 1, np.arange(31, T, 97), rng.integers(0, T, 12)]):
            check_attention(f, [0], [37 + t], 1, got[t:t + 1], q[t:t + 1], g[t:t + 1], window, sinks)
    f.c.close()
