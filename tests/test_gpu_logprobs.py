"""Token log probabilities (q35_op_token_logprobs) against float64, at the vocabularies, alignments, masks and orders where
they can go wrong.

Tolerances, in units of e = 2^-24. z = (x - m) c is off by three roundings, 3 e |z|, so a term w = 2^z by 3 e |z| ln 2
and the instruction's 2 e, and a float32 sum of 32 terms by eights by its 3 + 3 roundings, 6 e; the sums end in float64.
The term of the maximum itself, 1, is exact; it lies in one such sum of a wave, whose 6 roundings may then be e
each, unless the wave's S is under 2, where that sum is made without it: 6 e at S - 1 >= 1, so 6 e (S - 1) at most.
With gap = sum w |z| ln 2 / S and r rescalings of a wave (one a tile at most, each another 2 e), log S is off by
(14 + 3 gap + 2 r) e (S - 1) / S.
The entropy log S + gap adds gap's own error: up to 64 terms of a lane in float32, (64 + 8 + 2 r) e gap + 3 e gap2,
gap2 = sum w z^2 / S, and log S's relative one. Each result is rounded once, e |result|. Ranks and ids are exact."""
import numpy as np
import pytest

import kv4_ref as ref

pytestmark = pytest.mark.gpu

E = 2.0 ** -24


@pytest.fixture(scope="module")
def eng():
    from qwen35 import Engine
    e = Engine(max_rows=8, max_ctx=64, seed=None)
    yield e
    e.close()


def call(eng, x, targets, top, bf16=False, temperature=1.0, pad=0, shift=0, skip=()):
    """x [rows][vocab] float32 (of bf16's values where bf16); rows lie pad elements apart, shift elements behind a
    16-byte border. Returns the outputs, whose neighbours must stay."""
    import torch
    n, v = x.shape
    ld = v + pad
    t = torch.full((n * ld + 16,), 1e30, dtype=torch.bfloat16 if bf16 else torch.float32, device="cuda")
    rows = t[shift:shift + n * ld].view(n, ld)
    rows[:, :v] = torch.from_numpy(x).cuda().to(t.dtype)
    tg = torch.from_numpy(np.asarray(targets, np.int32)).cuda()
    out = {"logprobs": (n,), "ranks": (n,), "entropy": (n,), "top_ids": (n, top), "top_logprobs": (n, top)}
    out = {k: torch.full((int(np.prod(s)) + 2,), 77, dtype=torch.float32 if k in ("logprobs", "entropy", "top_logprobs") else
                         torch.int32, device="cuda") for k, s in out.items()}
    torch.cuda.synchronize()
    ptr = {k: (0 if k in skip else o[1:].data_ptr()) for k, o in out.items()}
    eng.op_token_logprobs(n, v, rows.data_ptr(), targets=tg.data_ptr(), top=top, temperature=temperature, bf16=bf16, ld=ld, **ptr)
    eng.sync()
    got = {}
    for k, o in out.items():
        a = o.cpu().numpy()
        assert a[0] == 77 and a[-1] == 77 and (k not in skip or (a == 77).all())
        got[k] = a[1:-1].reshape(n, top) if k.startswith("top") else a[1:-1]
    return got


def near(got, want, e):
    """got = want within e and one rounding to float32, in which what is past its largest number is an infinity."""
    with np.errstate(over="ignore", invalid="ignore"):
        r = np.asarray(want).astype(np.float32)
        return np.where(np.isfinite(r), np.abs(got - want) <= e + E * np.abs(want) + 1e-45, got == r)


def check(got, x, targets, top, temperature=1.0, skip=()):
    n, v = x.shape
    tiles = v // 2048 + 2
    for i in range(n):
        row, t = x[i].astype(np.float64), int(targets[i])
        if not ref.dist(row):
            assert np.isnan(got["logprobs"][i]) and got["ranks"][i] == -1 and np.isnan(got["entropy"][i]), i
            assert (got["top_ids"][i] == -1).all() and np.isnan(got["top_logprobs"][i]).all(), i
            continue
        with np.errstate(over="ignore"):
            z = (row - row.max()) / temperature
        w = np.exp(z)
        s = w.sum()
        zz = np.where(w > 0, z, 0)
        gap, gap2 = (w * -zz).sum() / s, (w * zz * zz).sum() / s
        lse = np.log1p(w[np.arange(v) != row.argmax()].sum())
        e_lse = (14 + 3 * gap + 2 * tiles) * E * (1 - 1 / s) + 1e-15
        e_ent = (72 + 2 * tiles) * E * gap + 3 * E * gap2 + e_lse * (1 + gap)
        order = np.lexsort((np.arange(v), -row))
        if 0 <= t < v:
            with np.errstate(over="ignore"):
                lp = z[t] - lse
            if "logprobs" not in skip:
                assert near(got["logprobs"][i], lp, e_lse), (i, got["logprobs"][i], lp)
            if "ranks" not in skip:
                assert got["ranks"][i] == int(np.flatnonzero(order == t)[0]), i
        else:
            assert np.isnan(got["logprobs"][i]) and got["ranks"][i] == -1, i
        if "entropy" not in skip:
            ent = lse + gap
            assert abs(got["entropy"][i] - ent) <= e_ent + E * ent + 1e-45, (i, got["entropy"][i], ent, e_ent)
        ids = order[:top]
        if "top_ids" not in skip:
            assert np.array_equal(got["top_ids"][i], ids), (i, got["top_ids"][i], ids)
        if "top_logprobs" not in skip:
            assert np.all(near(got["top_logprobs"][i], z[ids] - lse, e_lse)), i


def values(rng, n, v, bf16, scale=3.0):
    x = (rng.standard_normal((n, v)) * scale).astype(np.float32)
    return ref.val(ref.bf16_bits(x)).astype(np.float32) if bf16 else x


@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("v", [1, 2, 7, 15, 16, 17, 40, 63, 64, 129, 1000, 2048, 2049, 4103, 16384, 32003])
def test_vocabularies(eng, v, bf16):
    """Every vocabulary from one word on, rows at every alignment, few and many rows, all numbers of alternatives."""
    rng = np.random.default_rng(v + bf16)
    for n, top, pad, shift, temp in [(1, 0, 0, 0, 1.0), (1, 32, 0, 3, 1.0), (5, 5, 1, 0, 0.7), (9, 1, 3, 1, 1.3), (300, 20, 0, 7, 1.0),
                                     (2050, 3, 5, 2, 2.0)]:
        top = min(top, v)
        if n * v > 20_000_000:
            n = 600
        print(f"logprobs v={v} bf16={bf16} n={n} top={top} pad={pad} shift={shift}", flush=True)
        x = values(rng, n, v, bf16)
        t = rng.integers(0, v, n)
        t[rng.random(n) < 0.1] = -1
        t[0] = x[0].argmax() if n > 3 else v - 1
        pick = np.unique(np.r_[np.arange(min(n, 12)), rng.integers(0, n, 20), n - 1])
        got = call(eng, x, t, top, bf16, temp, pad, shift)
        check({k: a[pick] for k, a in got.items()}, x[pick], t[pick], top, temp)


@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("n", [1, 3, 40])
def test_large_vocabulary(eng, n, bf16):
    rng = np.random.default_rng(n)
    v = 248320
    x = values(rng, n, v, bf16)
    x[:, rng.integers(0, v, 30)] += 8
    x = ref.val(ref.bf16_bits(x)).astype(np.float32) if bf16 else x
    t = rng.integers(0, v, n)
    for top, temp in [(20, 1.0), (32, 0.6)]:
        print(f"logprobs large n={n} bf16={bf16} top={top}", flush=True)
        got = call(eng, x, t, top, bf16, temp)
        check(got, x, t, top, temp)


ORDERS = {
    "equal": lambda rng, v: np.zeros(v),
    "few values": lambda rng, v: rng.integers(0, 3, v),
    "rising": lambda rng, v: np.linspace(-20, 20, v),
    "falling": lambda rng, v: np.linspace(20, -20, v),
    "steps": lambda rng, v: np.arange(v) // 100,
    "masked": lambda rng, v: np.where(rng.random(v) < 0.9, -np.inf, rng.standard_normal(v)),
    "one left": lambda rng, v: np.where(np.arange(v) == v // 3, 4.0, -np.inf),
    "five left": lambda rng, v: np.where(np.arange(v) % (v // 5) == 1, rng.standard_normal(v), -np.inf),
    "lowest masks": lambda rng, v: np.where(rng.random(v) < 0.5, -3.3895e38, rng.standard_normal(v)),
    "all lowest": lambda rng, v: np.full(v, -3.3895e38),
    "far apart": lambda rng, v: rng.standard_normal(v) * 1e37,
    "certain": lambda rng, v: np.where(np.arange(v) == v - 1, 30.0, rng.standard_normal(v)),
    "certain, first": lambda rng, v: np.where(np.arange(v) == 0, 14.0, rng.standard_normal(v) - 2),
    "zeros of both signs": lambda rng, v: np.where(rng.random(v) < 0.5, 0.0, -0.0),
    "subnormal": lambda rng, v: rng.integers(-5, 6, v) * 1.5e-45,
    "head and tail": lambda rng, v: np.where((np.arange(v) < 3) | (np.arange(v) > v - 4), 5.0, rng.standard_normal(v)),
    "last of a tie": lambda rng, v: np.where(np.arange(v) >= v - 40, 9.0, -np.arange(v) / v),
}


@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("order", list(ORDERS))
def test_orders_and_masks(eng, order, bf16):
    """Ties (the lower id first), masks of -inf and of the type's lowest value, rows in order, all but certain rows."""
    rng = np.random.default_rng(7)
    for v, n, shift in [(67, 2, 1), (2500, 2, 5), (40001, 3, 3), (40001, 900, 0)]:
        x = np.stack([ORDERS[order](rng, v) for _ in range(2)]).astype(np.float32)
        x = ref.val(ref.bf16_bits(x)).astype(np.float32) if bf16 else x
        x = np.ascontiguousarray(np.resize(x, (n, v)))
        t = rng.integers(0, v, n)
        t[0] = np.flatnonzero(x[0] == x[0].max())[-1]
        t[1] = x[1].argmin()
        for top, temp in [(20, 1.0), (32, 0.001), (1, 5.0)]:
            print(f"logprobs {order} bf16={bf16} v={v} n={n} top={top}", flush=True)
            got = call(eng, x, t, top, bf16, temp, shift=shift)
            pick = np.arange(min(n, 3))
            check({k: a[pick] for k, a in got.items()}, x[pick], t[pick], top, temp)


@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("order", list(ORDERS))
def test_orders_in_a_wide_block(eng, order, bf16):
    """The same in rows that a block of 16 or 8 waves has to itself, and of lengths that leave some of its waves without a tile."""
    rng = np.random.default_rng(8)
    for v, n, shift in [(40001, 30, 3), (10300, 6, 1), (40001, 300, 0), (70003, 257, 5)]:
        x = np.stack([ORDERS[order](rng, v) for _ in range(3)]).astype(np.float32)
        x = ref.val(ref.bf16_bits(x)).astype(np.float32) if bf16 else x
        x = np.ascontiguousarray(np.resize(x, (n, v)))
        t = rng.integers(0, v, n)
        t[0] = np.flatnonzero(x[0] == x[0].max())[-1]
        t[1] = x[1].argmin()
        for top, temp in [(20, 1.0), (32, 0.01), (0, 3.0)]:
            print(f"logprobs {order} bf16={bf16} v={v} n={n} top={top}", flush=True)
            got = call(eng, x, t, top, bf16, temp, shift=shift)
            pick = np.array([0, 1, 2, n - 1])
            check({k: a[pick] for k, a in got.items()}, x[pick], t[pick], top, temp)


@pytest.mark.parametrize("bf16", [False, True])
def test_rows_without_a_distribution(eng, bf16):
    """A NaN, a +inf or nothing but -inf anywhere in a row: NaN and -1 there, the rows beside it untouched."""
    rng = np.random.default_rng(3)
    for v in (5, 300, 20011):
        x = values(rng, 40, v, bf16)
        for i, at in enumerate([0, 1, 2, v // 2, v - 2, v - 1]):
            x[2 * i + 1, at] = np.nan
            x[2 * i + 13, at] = np.inf
        x[27] = -np.inf
        x[29] = np.nan
        x[31], x[31, 0] = -np.inf, np.nan
        x[33] = np.inf
        t = rng.integers(0, v, 40)
        t[36], t[37], t[38] = v, 2 ** 31 - 1, -2 ** 31
        top = min(v, 20)
        got = call(eng, x, t, top, bf16)
        check(got, x, t, top)


def test_outputs_left_out(eng):
    """Any output may be NULL; the others are what they are with all of them."""
    rng = np.random.default_rng(4)
    x, t = values(rng, 6, 5003, False), rng.integers(0, 5003, 6)
    full = call(eng, x, t, 7)
    for skip in [("logprobs",), ("ranks",), ("entropy",), ("top_ids",), ("top_logprobs",), ("top_ids", "top_logprobs"),
                 ("logprobs", "ranks", "entropy"), tuple(full)]:
        got = call(eng, x, t, 7, skip=skip)
        for k in full:
            if k not in skip:
                assert np.array_equal(got[k], full[k]), (skip, k)
    import torch
    xs, ent = torch.from_numpy(x).cuda(), torch.zeros(6, device="cuda")
    torch.cuda.synchronize()
    eng.op_token_logprobs(6, 5003, xs.data_ptr(), entropy=ent.data_ptr())        # no targets
    eng.sync()
    assert np.array_equal(ent.cpu().numpy(), full["entropy"])


def test_row_is_its_own(eng):
    """The same call gives the same bits; a row's ids and ranks do not depend on the rows beside it."""
    rng = np.random.default_rng(5)
    x, t = values(rng, 33, 60001, True), rng.integers(0, 60001, 33)
    a, b = call(eng, x, t, 20, True), call(eng, x, t, 20, True)
    one = call(eng, x[32:], t[32:], 20, True)
    assert all(np.array_equal(a[k], b[k]) for k in a)
    assert np.array_equal(a["top_ids"][32:], one["top_ids"]) and a["ranks"][32] == one["ranks"][0]


@pytest.mark.parametrize("bf16", [False, True])
def test_many_rows_and_far_ones(eng, bf16):
    """More rows than a launch takes, and rows more than 2^32 bytes apart."""
    import torch
    rng = np.random.default_rng(6)
    x = values(rng, 20000, 33, bf16)
    t = rng.integers(-1, 34, 20000)
    pick = np.r_[0, 8191, 8192, 16383, 16384, 19999, rng.integers(0, 20000, 30)]
    got = call(eng, x, t, 4, bf16)
    check({k: v[pick] for k, v in got.items()}, x[pick], t[pick], 4)
    v, ld = 70001, 2 ** 31 + 5
    far = torch.zeros(2 * ld + v, dtype=torch.bfloat16 if bf16 else torch.float32, device="cuda")
    x, t = values(rng, 3, v, bf16), rng.integers(0, v, 3)
    for i in range(3):
        far[i * ld:i * ld + v] = torch.from_numpy(x[i]).cuda().to(far.dtype)
    tg = torch.from_numpy(t.astype(np.int32)).cuda()
    out = {k: torch.zeros(3, *s, dtype=d, device="cuda") for k, s, d in
           [("logprobs", (), torch.float32), ("ranks", (), torch.int32), ("entropy", (), torch.float32), ("top_ids", (9,), torch.int32),
            ("top_logprobs", (9,), torch.float32)]}
    torch.cuda.synchronize()
    eng.op_token_logprobs(3, v, far.data_ptr(), targets=tg.data_ptr(), top=9, bf16=bf16, ld=ld, **{k: o.data_ptr() for k, o in out.items()})
    eng.sync()
    check({k: o.cpu().numpy() for k, o in out.items()}, x, t, 9)
    del far
    torch.cuda.empty_cache()
