"""The 4-bit cache's operators at values, sizes and slots where a wrong step shows: infinities and the ends of the
float32 range, scores far from zero, rows that hang on single slots of a long context, several rows of heads in a
block, calls larger than one launch takes. References and tolerances are those of tests/test_gpu_kv4.py."""
import numpy as np
import pytest

import kv4_ref as ref
import test_gpu_kv4 as base
from test_gpu_kv4 import Dev, Filled, check_attention, read_cache, run_attention

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def eng():
    from qwen35 import Engine
    e = Engine(max_rows=64, max_ctx=40000, seed=None)
    yield e
    e.close()


# ------------------------------------------------------------------------------ norms and append
class Plain:
    """q, k, v rows of one kv head and `hq` q heads, dense, for heads of given values."""

    def __init__(self, x, hq, d):
        import torch
        D, R = Dev(), x.shape[0]
        assert x.shape == (R, hq + 2, d)
        self.x, self.hq, self.d, self.R = ref.bf16_bits(x), hq, d, R          # [R][hq + 2][d]: q heads, k, v
        self.w = ref.bf16_bits(np.random.default_rng(d).standard_normal(d) * 0.1)
        self.dx, self.dw = D.up(self.x), D.up(self.w)
        self.q = torch.zeros(R, hq, d, dtype=torch.int16, device="cuda")
        self.k, self.v = (torch.zeros(R, 1, d, dtype=torch.int16, device="cuda") for _ in range(2))
        torch.cuda.synchronize()

    def args(self, rot, eps):
        p, ld, d, w = self.dx.data_ptr(), (self.hq + 2) * self.d, self.d, self.dw.data_ptr()
        return dict(rot_dim=rot, theta=1e6, eps=eps, q_norm=w, k_norm=w, q=(p, ld, d), k=(p + 2 * self.hq * d, ld, d),
                    q_out=(self.q.data_ptr(), self.hq * d, d), k_out=(self.k.data_ptr(), d, d))

    def want(self, rot, eps, pos):
        with np.errstate(invalid="ignore", divide="ignore"):
            return ref.norm_rope(ref.val(self.x)[:, :self.hq + 1], ref.val(self.w), pos, rot, 1e6, eps)


def same(bits, want, size):
    """NaN where the formula has NaN, and elsewhere the tolerance of the finite cases."""
    got = ref.val(bits)
    assert np.array_equal(np.isnan(got), np.isnan(want))
    ok = ~np.isnan(want)
    assert np.all(np.abs(got - want)[ok] <= (2.0 ** -8 * np.abs(want) + base.SLACK * size + 1e-37)[ok])


@pytest.mark.parametrize("d,rot", [(256, 64), (128, 128), (64, 0), (128, 100)])
def test_norm_rope_infinities(eng, d, rot):
    """An infinity makes its own element NaN (inf * 0), and its partner in the rotation; the head's other
    elements become 0. A NaN makes the whole head NaN."""
    print(f"norm_rope infinities {d} {rot}", flush=True)
    rng = np.random.default_rng(d + rot)
    x = rng.standard_normal((6, 5, d))
    x[0, 0, d - 1] = np.inf
    x[1, 1, 3] = -np.inf
    x[2, 3, 40], x[2, 3, 41] = np.inf, -np.inf
    x[3, 2, 5] = np.nan
    x[4, :, ::7] = np.inf
    p = Plain(x, 3, d)
    pos = np.arange(6) + 1000
    eng.op_qk_norm_rope([1000], 6, 3, 1, d, **p.args(rot, 1e-6))
    eng.sync()
    want, size = p.want(rot, 1e-6, pos.astype(np.float64))
    D = Dev()
    same(D.bits(p.q), want[:, :3], size[:, :3])
    same(D.bits(p.k), want[:, 3:], size[:, 3:])
    assert np.isnan(want).any() and (want[4] == 0).any()


def test_append_infinity_in_k(eng):
    """Only the groups of k that hold a NaN after the norm are marked; the head's other groups are zeros."""
    from qwen35 import KvCache4
    d = 128
    x = np.random.default_rng(2).standard_normal((3, 4, d))
    x[1, 2, 70] = np.inf
    p = Plain(x, 2, d)
    c = KvCache4(eng, 1, 8, kv_heads=1, head_dim=d)
    args = p.args(0, 1e-6)
    args.update(v=(p.dx.data_ptr() + 2 * 3 * d, 4 * d, d), v_out=(p.v.data_ptr(), d, d))
    eng.op_kv4_append(c, 0, [0], [0], 3, 2, **args)
    eng.sync()
    kc, ks, vc, vs = read_cache(eng, c, 0, 0, 1, 0, 3)
    assert list(ks[0, 0, 1]) == [8, 8, 255, 8] and np.all(ks[0, 0, [0, 2]] < 200)
    got = ref.values(kc[0, 0], ks[0, 0])
    assert np.isnan(got[1, 64:96]).all() and np.all(np.delete(got[1], range(64, 96)) == 0)
    assert np.isfinite(ref.values(vc, vs)).all()
    c.close()


@pytest.mark.parametrize("d,rot", [(256, 64), (64, 6)])
def test_norm_rope_tiny_and_huge_heads(eng, d, rot):
    """eps 0: heads of subnormal numbers, whose 1 / root is past float32, have the norm of any other head; so have
    heads near bf16's largest number."""
    print(f"norm_rope tiny and huge {d} {rot}", flush=True)
    rng = np.random.default_rng(d)
    x = rng.standard_normal((6, 4, d))
    x[0] *= 2.0 ** -128
    x[1] *= 2.0 ** -131
    x[2] = 0
    x[2, :, 17] = 2.0 ** -133
    x[3] = np.clip(x[3], -1.5, 1.5) * 2.0 ** 127
    x[4, :, ::2] *= 2.0 ** -130
    p = Plain(x, 2, d)
    eng.op_qk_norm_rope([77], 6, 2, 1, d, **p.args(rot, 0.0))
    eng.sync()
    want, size = p.want(rot, 0.0, 77.0 + np.arange(6))
    assert np.isfinite(want).all() and np.abs(want[:3]).max() > 1
    D = Dev()
    same(D.bits(p.q), want[:, :2], size[:, :2])
    same(D.bits(p.k), want[:, 2:], size[:, 2:])


@pytest.mark.parametrize("hq,kv,d,rot", [(5, 1, 128, 128), (3, 3, 128, 100), (14, 2, 64, 64), (8, 2, 256, 256), (2, 1, 256, 2)])
@pytest.mark.parametrize("n,T", [(1, 1025), (205, 5), (1, 4099), (17, 241), (300, 15)])
def test_norm_rope_rows_in_blocks(eng, hq, kv, d, rot, n, T):
    """Two rows a block from 1024 rows on, four from 4096: waves that take heads of two rows, a short last block, the
    whole table of angles, blocks over the border of two sequences."""
    base.test_norm_rope(eng, hq, kv, d, rot, n, T)


@pytest.mark.parametrize("hq,kv,d,rot", [(5, 1, 128, 128), (3, 3, 64, 6), (8, 2, 256, 256)])
@pytest.mark.parametrize("n,T,pos0", [(1, 1025, 7), (41, 25, 3), (1, 4099, 30), (17, 241, 17)])
def test_append_rows_in_blocks(eng, hq, kv, d, rot, n, T, pos0):
    base.test_append(eng, hq, kv, d, rot, n, T, pos0)


# ------------------------------------------------------------------------------ attention
def filled(eng, kc, ks, vc, vs):
    """A cache of one layer with these codes and scale bytes [lanes][kv][cap][..], and its values."""
    import torch
    from qwen35 import KvCache4
    lanes, kv, cap, half = kc.shape
    f = Filled.__new__(Filled)
    f.c = KvCache4(eng, lanes, cap, kv_heads=kv, head_dim=2 * half)
    t = [torch.from_numpy(a).cuda() for a in (kc, ks, vc, vs)]
    torch.cuda.synchronize()
    f.c.write(0, 0, lanes, 0, cap, *[x.data_ptr() for x in t])
    eng.sync()
    f.K, f.V = ref.values(kc, ks), ref.values(vc, vs)
    return f


def random_rows(rng, lanes, kv, cap, d):
    a = [rng.integers(0, 256, (lanes, kv, cap, d // 2)).astype(np.uint8) for _ in range(2)]
    b = [rng.integers(124, 127, (lanes, kv, cap, d // 32)).astype(np.uint8) for _ in range(2)]
    return a[0], b[0], a[1], b[1]


@pytest.mark.parametrize("hq,kv,d,T,cap", [(4, 2, 128, 3, 500), (8, 2, 256, 1, 9000), (4, 1, 64, 20, 300)])
def test_attention_scores_past_their_spacing(eng, hq, kv, d, T, cap):
    """Scores so far from zero that float32 numbers lie further apart than 2^8 there: the largest one takes all the
    weight, the row is its V exactly, and no row is NaN. Every row's largest score leads by more than
    float32 sums of its products can be off."""
    rng = np.random.default_rng(cap)
    f = Filled(eng, rng, 1, cap, kv, d)
    for scale in (3e8, -4e9, 1e12, 1e30):
        print(f"attention far scores {hq} {kv} {d} {T} {cap} {scale}", flush=True)
        got, q, _ = run_attention(eng, f, [0], [cap - T], T, hq, rng, scale=scale)
        g, sure = ref.val(got), 0
        assert np.isfinite(g).all()
        for t in range(T):
            for h in range(hq):
                k, v = f.K[0][h // (hq // kv)][:cap - T + t + 1], f.V[0][h // (hq // kv)]
                s = k @ q[t, h] * np.sign(scale)
                off = (d + 4) * 2.0 ** -24 * (np.abs(k) @ np.abs(q[t, h])).max()
                a = np.argsort(s)
                if s[a[-1]] - s[a[-2]] > 4 * off and (s[a[-1]] - s[a[-2]]) * abs(scale) > 200:
                    sure += 1
                    assert np.array_equal(g[t, h], v[a[-1]]), (t, h)
        assert sure >= T * hq // 2
    f.c.close()


@pytest.mark.parametrize("hq,kv,d,T,cap", [(4, 2, 128, 1, 500), (8, 2, 256, 1, 9000), (4, 1, 64, 20, 300)])
def test_attention_largest_values(eng, hq, kv, d, T, cap):
    """V at the largest numbers the format has: the sums before the division stay finite. A weight under 2^-126 is 0, and
    the largest one is at least 2^-28 here, so each slot may lose 2^-98 of the largest V beyond attention_bound (at V
    of 2^127 that is no longer under its 1e-30)."""
    rng = np.random.default_rng(cap + 1)
    kc, ks, vc, vs = random_rows(rng, 1, kv, cap, d)
    vs[:], vc[:, :, :, : d // 4] = 252, 0x77
    f = filled(eng, kc, ks, vc, vs)
    for scale in (None, 1e-30, 5.0):
        got, q, _ = run_attention(eng, f, [0], [cap - T], T, hq, rng, scale=scale)
        g = ref.val(got)
        out, pv, big = ref.attention(q, f.K[0], f.V[0], cap - T, 0, 0, d ** -0.5 if scale is None else scale)
        want, e = ref.attention_bound(out, pv, big, cap, d)
        assert np.isfinite(g).all() and np.all(np.abs(g - want) <= e + cap * 2.0 ** -98 * 6 * 2.0 ** 125)
        assert (g[..., : d // 2] > 2.5e38).all()
    f.c.close()


@pytest.mark.parametrize("T", [1, 20])
def test_attention_scale_of_zero_and_next_to_it(eng, T):
    """Products near 10^38 times a scale of 0 or of a subnormal number: even weights, and those of the formula."""
    import torch
    rng, D, d, cap, hq = np.random.default_rng(18), Dev(), 128, 300, 4
    f = Filled(eng, rng, 1, cap, 2, d)
    qb = base.bf16_randn(rng, T, hq, d, scale=2e36)
    q, out = D.up(qb), torch.zeros(T, hq, d, dtype=torch.int16, device="cuda")
    torch.cuda.synchronize()
    for scale in (0.0, 3e-38, 1e-39, -1e-39, 2e-41):
        eng.op_attn_kv4(f.c, 0, [0], [cap - T], T, hq, (q.data_ptr(), hq * d, d), (out.data_ptr(), hq * d, d), scale=scale)
        eng.sync()
        check_attention(f, [0], [cap - T], T, D.bits(out), ref.val(qb), None, scale=float(np.float32(scale)))
    f.c.close()


def test_attention_smallest_scales(eng):
    """Scale bytes 0 to 8 with every pair of codes, written by the caller: a row that sees one slot gives its V exactly,
    down to 2^-128; as K they give scores next to 0."""
    rng, kv, d = np.random.default_rng(9), 2, 256
    kc, ks, vc, vs = random_rows(rng, 1, kv, 9, d)
    vs[0] = np.arange(9)[None, :, None]
    vc[0] = np.arange(256).reshape(kv, 1, 128)
    f = filled(eng, kc, ks, vc, vs)
    got, q, g = run_attention(eng, f, [0], [0], 9, kv, rng, window=1)
    assert np.array_equal(ref.val(got), f.V[0].transpose(1, 0, 2))
    ks[0] = np.arange(9)[None, :, None]
    f2 = filled(eng, kc, ks, *random_rows(rng, 1, kv, 9, d)[2:])
    got, q, g = run_attention(eng, f2, [0], [8], 1, kv, rng)
    check_attention(f2, [0], [8], 1, got, q, g)
    f.c.close()
    f2.c.close()


class Pairs:
    """A cache in which the slots of each pair hold the same K and other V, in every lane and head: a query along that K,
    steep enough, takes half of each, so a row's answer shows a slot that is left out, counted twice or
    seen wrongly."""

    def __init__(self, eng, rng, lanes, cap, kv, d, pairs):
        kc, ks, vc, vs = random_rows(rng, lanes, kv, cap, d)
        for a, b in pairs:
            kc[:, :, b], ks[:, :, b] = kc[:, :, a], ks[:, :, a]
        self.f, self.pairs, self.d = filled(eng, kc, ks, vc, vs), pairs, d

    def run(self, eng, lanes, pos, T, hq, probe, window=0, sinks=0):
        """probe [n][T][hq]: the pair each row's head asks for."""
        import torch
        D, d, n, kv, K = Dev(), self.d, len(lanes), self.f.c.kv_heads, self.f.K
        first = np.array([p[0] for p in self.pairs])[probe]
        q = ref.bf16_bits(K[np.array(lanes)[:, None, None], (np.arange(hq) // (hq // kv))[None, None], first])
        x, out = D.up(q.reshape(n * T, hq, d)), torch.zeros(n * T, hq, d, dtype=torch.int16, device="cuda")
        torch.cuda.synchronize()
        scale = 4 * d ** -0.5
        eng.op_attn_kv4(self.f.c, 0, lanes, pos, T, hq, (x.data_ptr(), hq * d, d), (out.data_ptr(), hq * d, d), scale=scale,
                        window=window, sinks=sinks)
        eng.sync()
        got, told = D.bits(out).reshape(n, T, hq, d), 0
        for i, (l, p) in enumerate(zip(lanes, pos)):
            r = ref.val(q[i])
            o, pv, big = ref.attention(r, K[l], self.f.V[l], p, window, sinks, scale)
            want, e = ref.attention_bound(o, pv, big, p + T, d)
            assert np.all(np.abs(ref.val(got[i]) - want) <= e), (l, p)
            # the reference itself, with the first slot of the last row's pairs left out and counted twice
            for h in range(hq):
                a, b = self.pairs[probe[i, T - 1, h]]
                seen = lambda s: s <= p + T - 1 and (not window or s > p + T - 1 - window or s < sinks)  # noqa: E731
                if seen(a) and seen(b):
                    v = self.f.V[l][h // (hq // kv)]
                    for wa in (0.0, 2.0):
                        assert np.any(np.abs((wa * v[a] + v[b]) / (wa + 1) - want[T - 1, h]) > e[T - 1, h])
                    told += 1
        return told


def tile_pairs(rng, tiles, cap):
    """Every tile's first, last or another slot, paired with one of the tile half the length away."""
    at = np.array([min(cap - 1, 32 * t + int(rng.choice([0, 31, rng.integers(1, 31)]))) for t in range(tiles)])
    return [(int(at[i]), int(at[i + tiles // 2])) for i in range(tiles // 2)]


@pytest.mark.parametrize("hq,kv,d", [(8, 2, 256), (4, 1, 128), (6, 2, 64)])
def test_every_tile_of_a_long_context(eng, hq, kv, d):
    """One lane of 9001 slots over up to 128 blocks (attn_kv4_join), a slot of each of its 282 tiles asked for."""
    rng = np.random.default_rng(d + 1)
    P = Pairs(eng, rng, 1, 9001, kv, d, tile_pairs(rng, 282, 9001))
    told = 0
    for i in range(0, 141, hq):
        print(f"tiles {hq} {kv} {d}: pairs from {i}", flush=True)
        told += P.run(eng, [0], [9000], 1, hq, np.minimum(i + np.arange(hq), 140)[None, None])
    assert told >= 141
    P.f.c.close()


@pytest.mark.parametrize("hq,kv,d,T,lanes,cap", [(8, 2, 256, 1, 16, 2000), (8, 2, 256, 3, 4, 1100), (8, 2, 128, 9, 2, 1500),
                                                 (8, 2, 128, 9, 2, 3000), (6, 1, 64, 12, 1, 5000), (8, 2, 256, 12, 1, 5000)])
def test_tiles_of_split_rows(eng, hq, kv, d, T, lanes, cap):
    """Ragged lanes of a few splits each (attn_kv4_join_few), and rows of 16 and 32 in more (attn_kv4_join)."""
    rng = np.random.default_rng(cap + T)
    tiles = (cap - T) // 32 - 1
    P = Pairs(eng, rng, lanes, cap, kv, d, tile_pairs(rng, tiles, cap))
    pos = np.array([cap - T - 37 * i for i in range(lanes)], np.int32)
    for r in range(2):
        print(f"split rows {hq} {kv} {d} {T} {lanes} {cap}: {r}", flush=True)
        probe = rng.integers(0, len(P.pairs), (lanes, T, hq))
        assert P.run(eng, np.arange(lanes), pos, T, hq, probe) > 0
    P.f.c.close()


@pytest.mark.parametrize("hq,kv,d,T", [(8, 2, 256, 1), (8, 1, 128, 1), (4, 2, 64, 40)])
def test_slots_at_the_ends_of_a_window(eng, hq, kv, d, T):
    """The last sink and the slot behind it, the window's first slot and the one before it, the row's own and the
    next: each paired with a slot inside, in windows that end in and between tiles, over many splits and few."""
    rng = np.random.default_rng(d + T)
    cap, inside = 9001, 8900
    for window, sinks in [(5000, 40), (4992, 32), (2049, 1), (300, 64), (4000, 0)]:
        p = cap - 1 - T
        low = p - window + 1
        ends = {0, sinks - 1, sinks, low - 1, low, low + T - 1, low + T, p, p + T - 1, p + T}
        ends = [s for s in sorted(ends) if 0 <= s < cap]
        pairs = [(s, inside + i) for i, s in enumerate(ends)]
        P = Pairs(eng, rng, 1, cap, kv, d, pairs)
        print(f"window ends {hq} {kv} {d} {T}: {window} {sinks}", flush=True)
        for i in range(0, len(pairs), hq):
            probe = np.broadcast_to(np.minimum(i + np.arange(hq), len(pairs) - 1), (1, T, hq))
            P.run(eng, [0], [p], T, hq, probe, window, sinks)
        P.f.c.close()


def test_a_rows_bits_do_not_depend_on_the_others(eng):
    """Lanes whose rows stay in one split give the same bits in another order, among fewer lanes, beside other rows and
    on the other side of a launch's 256 sequences."""
    import torch
    rng, D, n, hq, d = np.random.default_rng(15), Dev(), 300, 8, 256
    f = Filled(eng, rng, n, 64, 2, d)
    pos, qb = rng.integers(0, 62, n).astype(np.int32), base.bf16_randn(rng, n, 2, hq, d)

    def call(lanes):
        q = D.up(qb[lanes].reshape(-1, hq, d))
        out = torch.zeros_like(q)
        torch.cuda.synchronize()
        eng.op_attn_kv4(f.c, 0, lanes, pos[lanes], 2, hq, (q.data_ptr(), hq * d, d), (out.data_ptr(), hq * d, d))
        eng.sync()
        return D.bits(out).reshape(len(lanes), 2, hq, d)

    whole = call(np.arange(n))
    for lanes in (rng.permutation(n), rng.permutation(n)[:280], np.array([299]), np.array([7, 250, 7])):
        assert np.array_equal(call(lanes), whole[lanes])
    f.c.close()


# ------------------------------------------------------------------------------ calls and their sizes
def test_calls_after_a_refused_allocation(eng):
    """A cache that no memory holds is refused, and the next call does not report that error again."""
    from qwen35 import EngineError, KvCache4
    with pytest.raises(EngineError):
        KvCache4(eng, 65535, 40000, layers=64, kv_heads=1024, head_dim=256)
    p = Plain(np.ones((1, 3, 64)), 1, 64)
    eng.op_qk_norm_rope([0], 1, 1, 1, 64, **p.args(0, 0.0))
    eng.sync()
    assert Dev().bits(p.q).any()


def test_attention_of_many_rows(eng):
    """2^27 rows of heads in one call (17 GB of output), more than a launch was once allowed: under a window of one slot
    every row is its own slot's V."""
    import torch
    n, T, hq, d = 256, 8192, 64, 64
    rng = np.random.default_rng(3)
    f = filled(eng, *random_rows(rng, 1, 1, T, d))
    q = Dev().up(base.bf16_randn(rng, d))
    out = torch.empty(n * T, hq, d, dtype=torch.bfloat16, device="cuda")
    v = torch.from_numpy(f.V[0][0]).to("cuda", torch.bfloat16)
    torch.cuda.synchronize()
    eng.op_attn_kv4(f.c, 0, [0] * n, [0] * n, T, hq, (q.data_ptr(), 0, 0), (out.data_ptr(), hq * d, d), window=1)
    eng.sync()
    out = out.view(n, T, hq, d)
    for i in range(n):
        assert torch.equal(out[i], v[:, None].expand(T, hq, d)), i
    f.c.close()
    del out
    torch.cuda.empty_cache()


def test_cache_copies_past_one_launch(eng):
    """Rows in and out of a 36 GB cache in one call: 2^32 threads' work, more than a launch can have."""
    import torch
    from qwen35 import KvCache4
    lanes, kv, cap, d = 16, 1024, 32768, 64
    c = KvCache4(eng, lanes, cap, kv_heads=kv, head_dim=d)
    codes = torch.empty(lanes, kv, cap, d // 2, dtype=torch.uint8, device="cuda")
    codes.view(torch.int64).random_()
    scales = torch.randint(8, 250, (lanes, kv, cap, d // 32), dtype=torch.uint8, device="cuda")
    torch.cuda.synchronize()
    c.write(0, 0, lanes, 0, cap, codes.data_ptr(), scales.data_ptr(), codes.data_ptr(), scales.data_ptr())
    got = [torch.empty_like(x) for x in (codes, scales)]
    torch.cuda.synchronize()
    c.read(0, 0, lanes, 0, cap, got[0].data_ptr(), got[1].data_ptr(), got[0].data_ptr(), got[1].data_ptr())
    eng.sync()
    for i in range(lanes):
        assert torch.equal(got[0][i], codes[i]) and torch.equal(got[1][i], scales[i]), i
    # K and V of a few slots apart from each other, in every lane
    k, v = (torch.empty(1, kv, 40, d // 2, dtype=torch.uint8, device="cuda") for _ in range(2))
    ks, vs = (torch.empty(1, kv, 40, d // 32, dtype=torch.uint8, device="cuda") for _ in range(2))
    for i in (0, 7, 8, 15):
        for s in (0, cap - 40):
            torch.cuda.synchronize()
            c.read(0, i, 1, s, 40, k.data_ptr(), ks.data_ptr(), v.data_ptr(), vs.data_ptr())
            eng.sync()
            assert torch.equal(k[0], codes[i, :, s:s + 40]) and torch.equal(v, k)
            assert torch.equal(ks[0], scales[i, :, s:s + 40]) and torch.equal(vs, ks)
    c.close()
    del codes, scales, got
    torch.cuda.empty_cache()


def test_norm_rope_of_many_rows(eng):
    """2^26 rows in one call, in two launches (8.6 GB of output): one input row, without a rotation."""
    import torch
    n, T, d = 2, 2 ** 25, 64
    rng, D = np.random.default_rng(4), Dev()
    k, w = D.up(base.bf16_randn(rng, d)), D.up(base.bf16_randn(rng, d, scale=0.1))
    out = torch.zeros(n, T, d, dtype=torch.int16, device="cuda")
    one = torch.zeros(1, d, dtype=torch.int16, device="cuda")
    torch.cuda.synchronize()
    args = dict(rot_dim=0, theta=1.0, eps=1e-6, q_norm=0, k_norm=w.data_ptr(), k=(k.data_ptr(), 0, 0))
    eng.op_qk_norm_rope([0], 1, 0, 1, d, k_out=(one.data_ptr(), d, d), **args)
    eng.op_qk_norm_rope([0, 0], T, 0, 1, d, k_out=(out.data_ptr(), d, d), **args)
    eng.sync()
    assert one.any() and all(torch.equal(out[i], one.expand(T, d)) for i in range(n))
    del out
    torch.cuda.empty_cache()


def test_lanes_past_32_bit_offsets(eng):
    """Append, attention and read at the end of a lane, 6.8 GB into the cache."""
    import torch
    from qwen35 import KvCache4
    rng, D, kv, d, cap, T = np.random.default_rng(16), Dev(), 1024, 64, 32768, 3
    c = KvCache4(eng, 3, cap, kv_heads=kv, head_dim=d)
    pos = cap - T
    c.set_len([2], [pos])
    x = base.bf16_randn(rng, T, 3 * kv, d)                   # q, k, v
    w = D.up(np.zeros(d, np.uint16))
    t, q = D.up(x), torch.zeros(T, kv, d, dtype=torch.int16, device="cuda")
    out = torch.zeros_like(q)
    torch.cuda.synchronize()
    p, ld = t.data_ptr(), 3 * kv * d
    eng.op_kv4_append(c, 0, [2], [pos], T, kv, rot_dim=0, theta=1.0, eps=1e-6, q_norm=w.data_ptr(), k_norm=w.data_ptr(),
                      q=(p, ld, d), k=(p + 2 * kv * d, ld, d), v=(p + 4 * kv * d, ld, d), q_out=(q.data_ptr(), kv * d, d))
    eng.op_attn_kv4(c, 0, [2], [pos], T, kv, (q.data_ptr(), kv * d, d), (out.data_ptr(), kv * d, d), window=2)
    eng.sync()
    kc, ks, vc, vs = read_cache(eng, c, 0, 2, 1, pos, T)
    base.check_codes(ref.val(x[:, 2 * kv:]).transpose(1, 0, 2), vc[0], vs[0], 0.0)
    K, V = ref.values(kc, ks)[0], ref.values(vc, vs)[0]
    o, pv, big = ref.attention(ref.val(D.bits(q)), K, V, 0, 2, 0, d ** -0.5)
    want, e = ref.attention_bound(o, pv, big, cap, d)
    g = ref.val(D.bits(out))
    assert np.all(np.abs(g - want)[1:] <= e[1:])             # (row 0 sees the slot before the appended ones, too)
    c.close()


def test_the_most_lanes_and_the_largest_windows(eng):
    """A cache of 65,535 lanes, all of them in one append and one attention, the last lane first; windows and sinks of
    2^31 - 1 see what no window sees."""
    import torch
    from qwen35 import KvCache4
    rng, D, n, d, big = np.random.default_rng(17), Dev(), 65535, 64, 2 ** 31 - 1
    c = KvCache4(eng, n, 3, kv_heads=1, head_dim=d)
    lanes, pos = np.arange(n, dtype=np.int32)[::-1].copy(), np.zeros(n, np.int32)
    x = base.bf16_randn(rng, n, 3, d)                        # q, k, v
    w = D.up(np.zeros(d, np.uint16))
    t, q, out = D.up(x), *(torch.zeros(n, d, dtype=torch.int16, device="cuda") for _ in range(2))
    torch.cuda.synchronize()
    p = t.data_ptr()
    eng.op_kv4_append(c, 0, lanes, pos, 1, 1, rot_dim=0, theta=1.0, eps=1e-6, q_norm=w.data_ptr(), k_norm=w.data_ptr(),
                      q=(p, 3 * d, d), k=(p + 2 * d, 3 * d, d), v=(p + 4 * d, 3 * d, d), q_out=(q.data_ptr(), d, d))
    eng.op_attn_kv4(c, 0, lanes, pos, 1, 1, (q.data_ptr(), d, d), (out.data_ptr(), d, d))
    eng.sync()
    kc, ks, vc, vs = read_cache(eng, c, 0, 0, n, 0, 1)
    base.check_codes(ref.val(x[:, 2]), vc[lanes, 0, 0], vs[lanes, 0, 0], 0.0)
    assert np.array_equal(ref.val(D.bits(out)), ref.values(vc, vs)[lanes, 0, 0])      # one slot: its V
    c.close()
    f = Filled(eng, rng, 1, 400, 2, 128)
    for window, sinks in [(big, 0), (big, big), (3, big)]:
        got, q, g = run_attention(eng, f, [0], [380], 20, 4, rng, window, sinks)
        check_attention(f, [0], [380], 20, got, q, g)
    f.c.close()
