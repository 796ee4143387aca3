"""Attention of answers that share prompts over the 4-bit cache, against float64 (tests/kv4_ref.py) on the slots that a row
sees: its prompt's, then its own up to its position. Tolerance: kv4_ref.attention_bound, its 2^-8 for the weights and
2^-24 a sum as for one list of slots; the join's factors are two float32 roundings of 2^-24 more, within its 64."""
import numpy as np
import pytest

import kv4_ref as ref
from test_gpu_kv4 import Dev, Filled, bf16_randn

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def eng():
    from qwen35 import Engine
    e = Engine(max_rows=64, max_ctx=40000, seed=None)
    yield e
    e.close()


def run(eng, pre, own, plane, plen, lanes, pos, T, hq, rng, gated=False, scale=None, spread=0):
    import torch
    D, n, d = Dev(), len(pos), own.c.head_dim
    qb, gb = bf16_randn(rng, n * T, hq, d), bf16_randn(rng, n * T, hq, d)
    q, g = D.up(qb), D.up(gb)
    out = torch.full((n * T + 1, hq, d + spread), 0x1234, dtype=torch.int16, device="cuda")
    torch.cuda.synchronize()
    eng.op_attn_kv4_shared(pre.c, own.c, 0, plane, plen, lanes, pos, T, hq, (q.data_ptr(), hq * d, d),
                           (out.data_ptr(), hq * (d + spread), d + spread), scale=scale,
                           gate=(g.data_ptr(), hq * d, d) if gated else None)
    eng.sync()
    o = D.bits(out)
    assert np.all(o[n * T:] == 0x1234) and np.all(o[:, :, d:] == 0x1234)
    return o[:n * T, :, :d], ref.val(qb), ref.val(gb) if gated else None


def seen(pre, own, pl, pn, l, end):
    """K and V of a sequence: its prompt's slots, then its own."""
    if pl < 0 or pn == 0:
        return own.K[l][:, :end], own.V[l][:, :end]
    return (np.concatenate([pre.K[pl][:, :pn], own.K[l][:, :end]], 1), np.concatenate([pre.V[pl][:, :pn], own.V[l][:, :end]], 1))


def check(pre, own, plane, plen, lanes, pos, T, got, q, gate, scale=None, pick=None):
    d = own.c.head_dim
    sc = d ** -0.5 if scale is None else scale
    for i in range(len(pos)) if pick is None else pick:
        r = slice(i * T, (i + 1) * T)
        K, V = seen(pre, own, plane[i], plen[i], lanes[i], pos[i] + T)
        out, pv, big = ref.attention(q[r], K, V, K.shape[1] - T, 0, 0, sc)
        want, e = ref.attention_bound(out, pv, big, K.shape[1], d, None if gate is None else gate[r])
        g = ref.val(got[r])
        assert np.array_equal(np.isnan(g), np.isnan(want)), f"NaN places of sequence {i}"
        bad = ~np.isnan(want) & ~(np.abs(g - want) <= e)
        assert not bad.any(), (i, int(bad.sum()), float(np.nanmax(np.abs(g - want) / e)))


LAYOUTS = [(8, 2, 256), (32, 8, 128), (14, 2, 64), (5, 1, 128), (6, 6, 64), (48, 3, 256), (40, 1, 128)]


@pytest.mark.parametrize("hq,kv,d", LAYOUTS)
@pytest.mark.parametrize("T", [1, 2, 5, 19])
def test_groups(eng, hq, kv, d, T):
    """Prompts of every length around a tile's ends, with one to many answers each, answers without one, in mixed order."""
    rng = np.random.default_rng(hq + d + T)
    pre, own = Filled(eng, rng, 6, 300, kv, d), Filled(eng, rng, 9, 100, kv, d)
    plane = np.array([0, 1, 1, 2, -1, 2, 2, 3, 0, 4, 5, 1, 2, 2, 1], np.int32)
    plen = np.array([300, 31, 31, 64, 7, 64, 63, 1, 300, 0, 33, 32, 64, 64, 31], np.int32)
    lanes = rng.integers(0, 9, plane.size).astype(np.int32)
    pos = rng.integers(0, 101 - T, plane.size).astype(np.int32)
    pos[:4] = [0, 100 - T, 31, 32]
    for gated in (False, True):
        print(f"shared {hq} {kv} {d} T={T} gated={gated}", flush=True)
        got, q, g = run(eng, pre, own, plane, plen, lanes, pos, T, hq, rng, gated, spread=8)
        check(pre, own, plane, plen, lanes, pos, T, got, q, g)
    pre.c.close()
    own.c.close()


@pytest.mark.parametrize("hq,kv,d", [(8, 2, 256), (32, 8, 128), (14, 2, 64), (5, 1, 128), (48, 3, 256)])
@pytest.mark.parametrize("T", [1, 5])
def test_long_groups(eng, hq, kv, d, T):
    """The same with prompts long enough to be read in parts for many answers, some beside short ones and none."""
    rng = np.random.default_rng(hq + d + T)
    pre, own = Filled(eng, rng, 4, 4300, kv, d), Filled(eng, rng, 9, 100, kv, d)
    plane = np.array([0, 1, 1, 2, -1, 2, 2, 3, 0, 3, 3, 1, 2, 2, 1], np.int32)
    plen = np.array([4300, 4031, 4031, 4064, 7, 4064, 4063, 1, 4300, 33, 0, 4032, 4064, 4064, 4031], np.int32)
    lanes = rng.integers(0, 9, plane.size).astype(np.int32)
    pos = rng.integers(0, 101 - T, plane.size).astype(np.int32)
    pos[:4] = [0, 100 - T, 31, 32]
    for gated in (False, True):
        print(f"shared long groups {hq} {kv} {d} T={T} gated={gated}", flush=True)
        got, q, g = run(eng, pre, own, plane, plen, lanes, pos, T, hq, rng, gated, spread=8)
        check(pre, own, plane, plen, lanes, pos, T, got, q, g, pick=None if not gated else [0, 3, 4, 7, 10])
    pre.c.close()
    own.c.close()


@pytest.mark.parametrize("hq,kv,d,n,P,T", [(8, 2, 256, 64, 3000, 1), (8, 2, 256, 2, 9000, 1), (32, 4, 128, 40, 2500, 1),
                                           (4, 4, 64, 100, 1500, 3), (8, 2, 256, 20, 1111, 3), (48, 3, 256, 9, 700, 5)])
def test_long_prompt(eng, hq, kv, d, n, P, T):
    """One prompt whose tiles are split over many blocks, and answers of unlike lengths, a long one among them."""
    rng = np.random.default_rng(P + d)
    pre, own = Filled(eng, rng, 1, P, kv, d), Filled(eng, rng, n, 1300, kv, d)
    plane, plen = np.zeros(n, np.int32), np.full(n, P, np.int32)
    lanes, pos = rng.permutation(n).astype(np.int32), rng.integers(0, 200, n).astype(np.int32)
    pos[n // 2] = 1300 - T
    print(f"shared long {hq} {kv} {d} {n} {P} {T}", flush=True)
    got, q, g = run(eng, pre, own, plane, plen, lanes, pos, T, hq, rng, True)
    assert not (got == 0x1234).all(-1).any()
    check(pre, own, plane, plen, lanes, pos, T, got, q, g, pick=np.unique(np.r_[0, n // 2, n - 1, rng.integers(0, n, 6)]))
    pre.c.close()
    own.c.close()


def test_no_prompt_is_the_attention(eng):
    """Without prompts: the attention of single lanes, both within the bound of the same float64 result (the lists are
    split among waves in other ways, so last bits may differ)."""
    import torch
    rng = np.random.default_rng(2)
    own = Filled(eng, rng, 7, 200, 2, 256)
    lanes, pos = np.arange(7, dtype=np.int32), rng.integers(0, 200, 7).astype(np.int32)
    none, len5 = np.full(7, -1, np.int32), np.full(7, 5, np.int32)
    got, q, g = run(eng, own, own, none, len5, lanes, pos, 1, 8, np.random.default_rng(1))
    check(own, own, none, len5, lanes, pos, 1, got, q, g)
    qd = Dev().up(ref.bf16_bits(q))
    out = torch.zeros(7, 8, 256, dtype=torch.int16, device="cuda")
    torch.cuda.synchronize()
    eng.op_attn_kv4(own.c, 0, lanes, pos, 1, 8, (qd.data_ptr(), 2048, 256), (out.data_ptr(), 2048, 256))
    eng.sync()
    check(own, own, none, len5, lanes, pos, 1, out.cpu().numpy().view(np.uint16), q, g)
    own.c.close()


@pytest.mark.parametrize("hq,kv,d", [(8, 2, 256), (4, 1, 128), (6, 6, 64)])
@pytest.mark.parametrize("T", [4, 5, 17, 40])
def test_no_prompt_many_rows(eng, hq, kv, d, T):
    """Launches without any prompt, of fewer and more rows a kv head than one tile has."""
    rng = np.random.default_rng(T + d)
    own = Filled(eng, rng, 3, 300, kv, d)
    lanes, pos = np.array([2, 0, 1], np.int32), np.array([300 - T, 0, 100], np.int32)
    none = np.full(3, -1, np.int32)
    got, q, g = run(eng, own, own, none, none + 1, lanes, pos, T, hq, rng, True)
    check(own, own, none, none + 1, lanes, pos, T, got, q, g)
    own.c.close()


def test_many(eng):
    """More sequences and prompts than a launch takes, and more rows than the partial results have room for."""
    rng = np.random.default_rng(5)
    pre, own = Filled(eng, rng, 90, 40, 1, 64), Filled(eng, rng, 300, 50, 1, 64)
    n = 600
    plane = rng.integers(-1, 90, n).astype(np.int32)
    plen = np.where(rng.random(n) < 0.5, 40, rng.integers(0, 41, n)).astype(np.int32)
    lanes, pos = rng.integers(0, 300, n).astype(np.int32), rng.integers(0, 49, n).astype(np.int32)
    got, q, g = run(eng, pre, own, plane, plen, lanes, pos, 2, 3, rng, True)
    check(pre, own, plane, plen, lanes, pos, 2, got, q, g)
    pre.c.close()
    own.c.close()
    pre, own = Filled(eng, rng, 2, 70, 2, 256), Filled(eng, rng, 3, 420, 2, 256)
    # 3 sequences x 400 rows x 64 heads: 76,800 rows of 260 floats, twice, in 32,768
    plane, plen = np.array([0, 1, 0], np.int32), np.array([70, 33, 70], np.int32)
    lanes, pos = np.array([2, 0, 1], np.int32), np.array([20, 0, 5], np.int32)
    print("shared: many rows", flush=True)
    got, q, g = run(eng, pre, own, plane, plen, lanes, pos, 400, 64, rng)
    assert not (got == 0x1234).all(-1).any()
    for i in range(3):
        for t in np.r_[0, 1, 255, 256, 257, 399, rng.integers(0, 400, 5)]:
            K, V = seen(pre, own, plane[i], plen[i], lanes[i], pos[i] + t + 1)
            r = slice(i * 400 + t, i * 400 + t + 1)
            out, pv, big = ref.attention(q[r], K, V, K.shape[1] - 1, 0, 0, 1 / 16)
            want, e = ref.attention_bound(out, pv, big, K.shape[1], 256)
            assert np.all(np.abs(ref.val(got[r]) - want) <= e), (i, t)
    pre.c.close()
    own.c.close()


@pytest.mark.parametrize("hq,kv,d", [(8, 2, 256), (4, 1, 128), (2, 2, 64)])
@pytest.mark.parametrize("T,far", [(1, 0), (3, 0), (40, 0), (1, 6000), (3, 6000), (9, 6016)])
def test_nan_slots(eng, hq, kv, d, T, far):
    """A NaN group of a prompt's K or V reaches the answers that name it with that length, in V its dims only; one behind
    the prefix's length, or in an answer's later slots, nobody. In prompts of up to 100 slots, and of 6000 more."""
    rng = np.random.default_rng(d + T)
    pre = Filled(eng, rng, 3, far + 100, kv, d, [("v", 0, 0, far + 70, 0), ("v", 0, kv - 1, far + 75, d // 32 - 1),
                                                     ("k", 1, 0, far + 60, 0), ("v", 2, 0, far + 99, 1)])
    own = Filled(eng, rng, 4, 60, kv, d, [("v", 0, 0, 59, 0), ("k", 1, 0, 45, 1), ("v", 2, kv - 1, 41, 1)])
    plane = np.array([0, 0, 1, 1, 2, 2, 0, -1], np.int32)
    plen = np.array([70, 76, 60, 61, 99, 100, 76, -far], np.int32) + far
    lanes = np.array([0, 0, 1, 2, 2, 3, 3, 1], np.int32)
    pos = np.array([60 - T, 0, 5, 10, 41 if T < 3 else 20, 3, 60 - T, 2], np.int32)
    got, q, _ = run(eng, pre, own, plane, plen, lanes, pos, T, hq, rng)
    for i in range(8):
        for t in range(T):
            K, V = seen(pre, own, plane[i], plen[i], lanes[i], pos[i] + t + 1)
            for h in range(hq):
                k, v = K[h // (hq // kv)], V[h // (hq // kv)]
                o = ref.val(got[i * T + t, h])
                if np.isnan(k).any():
                    assert np.isnan(o).all(), (i, t, h)
                    continue
                assert np.array_equal(np.isnan(o), np.isnan(v).any(0)), (i, t, h)
                out, pv, big = ref.attention(q[i * T + t:i * T + t + 1, h:h + 1], k[None], v[None], K.shape[1] - 1, 0, 0, d ** -0.5)
                want, e = ref.attention_bound(out, pv, big, K.shape[1], d)
                ok = ~np.isnan(o)
                assert np.all(np.abs(o - want[0, 0])[ok] <= e[0, 0][ok]), (i, t, h)
    pre.c.close()
    own.c.close()


def test_extreme_scores(eng):
    """Scores far apart and far from zero, scales of 0 and below: one part of a row may take all the weight."""
    rng = np.random.default_rng(11)
    pre, own = Filled(eng, rng, 1, 700, 2, 128), Filled(eng, rng, 5, 90, 2, 128)
    plane, plen = np.zeros(5, np.int32), np.full(5, 700, np.int32)
    lanes, pos = np.arange(5, dtype=np.int32), np.array([0, 10, 31, 64, 86], np.int32)
    for scale in (300.0, 0.0, -2.0, 1e-30, 3e7):
        print(f"shared scale {scale}", flush=True)
        got, q, g = run(eng, pre, own, plane, plen, lanes, pos, 3, 4, rng, scale=scale)
        check(pre, own, plane, plen, lanes, pos, 3, got, q, g, scale=scale)
    pre.c.close()
    own.c.close()


def test_one_cache_for_both(eng):
    """Prompts in some lanes of a cache, answers in others; the same call gives the same bits."""
    rng = np.random.default_rng(13)
    f = Filled(eng, rng, 6, 333, 2, 256)
    plane, plen = np.array([4, 4, 5, 5], np.int32), np.array([333, 333, 100, 100], np.int32)
    lanes, pos = np.array([0, 1, 2, 4], np.int32), np.array([3, 50, 200, 331], np.int32)
    a = run(eng, f, f, plane, plen, lanes, pos, 2, 8, np.random.default_rng(1), True)
    b = run(eng, f, f, plane, plen, lanes, pos, 2, 8, np.random.default_rng(1), True)
    assert np.array_equal(a[0], b[0])
    check(f, f, plane, plen, lanes, pos, 2, *a)
    f.c.close()
