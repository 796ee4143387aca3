"""Sampled draft verification (q35_op_draft_verify) against float64 (tests/kv4_ref.py): accepted counts equal,
the token the one whose running sum holds the border (1e-12 of the total for the two sides' order of
summing), over vocabularies around the chunk and vector sizes, types, strides, temperatures, ragged drafts
and rows without a distribution."""
import numpy as np
import pytest

import kv4_ref as ref

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def eng():
    from qwen35 import Engine
    e = Engine(max_rows=2048, max_ctx=64, seed=None)
    yield e
    e.close()


def run(eng, logits, drafts, u, temperature, dlogits=None, bf16=False, pad=0, dpad=0, shift=0):
    """Host arrays [n][k + 1][v], [n][k], [n][k + 1] -> (accepted, tokens); rows `pad` elements apart, the first one
    `shift` elements into its buffer. The spare elements hold NaN."""
    import torch
    n, k = drafts.shape
    t = torch.bfloat16 if bf16 else torch.float32

    def up(a, p):
        v = a.shape[-1]
        b = torch.full((shift + a.shape[0] * a.shape[1] * (v + p),), float("nan"), dtype=t, device="cuda")
        b[shift:].view(-1, v + p)[:, :v] = torch.from_numpy(a.reshape(-1, v)).to("cuda").to(t)
        return b

    lg, dl = up(logits, pad), up(dlogits, dpad) if dlogits is not None else None
    d, uu = torch.from_numpy(drafts.astype(np.int32)).cuda(), torch.from_numpy(u.astype(np.float32)).cuda()
    acc = torch.full((n + 1,), -7, dtype=torch.int32, device="cuda")
    tok = torch.full((n + 1, k + 1), -7, dtype=torch.int32, device="cuda")
    torch.cuda.synchronize()
    es, v = (2 if bf16 else 4), logits.shape[-1]
    eng.op_draft_verify(n, k, v, lg.data_ptr() + shift * es, d.data_ptr(), uu.data_ptr(), acc.data_ptr(), tok.data_ptr(),
                        temperature=temperature, draft_logits=dl.data_ptr() + shift * es if dl is not None else 0, bf16=bf16,
                        ld=v + pad, draft_ld=v + dpad)
    eng.sync()
    assert (acc[n:] == -7).all() and (tok[n:] == -7).all()
    return acc[:n].cpu().numpy(), tok[:n].cpu().numpy()


def check(logits, drafts, u, temperature, got, dlogits=None):
    acc, tok = got
    n, k = drafts.shape
    u = u.astype(np.float32).astype(np.float64)
    kinds = set()
    for i in range(n):
        a, w, r, near = ref.verify(logits[i], drafts[i], u[i], temperature, None if dlogits is None else dlogits[i])
        assert near > 1e-9, "the random numbers fall on a border: another seed"
        assert acc[i] == a, (i, acc[i], a)
        assert list(tok[i, :a]) == list(drafts[i, :a]) and np.all(tok[i, a + 1:] == -1), (i, tok[i])
        assert ref.token_ok(int(tok[i, a]), w, r), (i, tok[i, a])
        kinds.add((a, w is None))
    return kinds


def make(rng, n, k, v, probs, bf16, peak=6.0):
    lg = rng.standard_normal((n, k + 1, v)) * 1.5
    hot = rng.integers(0, v, (n, k + 1, 3))
    np.put_along_axis(lg, hot, peak, 2)
    dl = lg[:, :k] + 0.6 * rng.standard_normal((n, k, v))
    f = (lambda x: ref.val(ref.bf16_bits(x))) if bf16 else (lambda x: x.astype(np.float32).astype(np.float64))
    lg, dl = f(lg), f(dl)
    gum = -np.log(-np.log(rng.random((n, k, v))))
    drafts = (dl / 0.8 + gum).argmax(-1) if probs else dl.argmax(-1)
    drafts[rng.random((n, k)) < 0.1] = -1
    return lg, (dl if probs else None), drafts.astype(np.int32), rng.random((n, k + 1)).astype(np.float32)


@pytest.mark.parametrize("v", [1, 2, 7, 8, 9, 2047, 2048, 2049, 8191, 8193, 32003, 248320])
@pytest.mark.parametrize("probs", [False, True])
@pytest.mark.parametrize("bf16", [False, True])
def test_verify(eng, v, probs, bf16):
    n, k = (3, 2) if v > 100000 else (9, 3)
    print(f"verify v={v} probs={probs} bf16={bf16}", flush=True)
    rng = np.random.default_rng(v + 2 * probs + bf16)
    lg, dl, d, u = make(rng, n, k, v, probs, bf16)
    check(lg, d, u, 0.8, run(eng, lg, d, u, 0.8, dl, bf16), dl)
    # rows on odd elements
    check(lg, d, u, 1.7, run(eng, lg, d, u, 1.7, dl, bf16, pad=3, dpad=1, shift=1), dl)


@pytest.mark.parametrize("n,k,v", [(1, 1, 5000), (1, 8, 70001), (200, 8, 300), (680, 2, 1000), (64, 4, 50257)])
@pytest.mark.parametrize("probs", [False, True])
def test_verify_shapes(eng, n, k, v, probs):
    """Few rows in small chunks, many rows in large ones, the most drafts."""
    rng = np.random.default_rng(n + k)
    lg, dl, d, u = make(rng, n, k, v, probs, True)
    kinds = check(lg, d, u, 0.8, run(eng, lg, d, u, 0.8, dl, True), dl)
    if n > 100 and probs:      # (a certain drafter's k = 8 are all kept about once in 10^4 lanes)
        assert {a for a, _ in kinds} == set(range(k + 1))      # every count of accepted drafts occurs


@pytest.mark.parametrize("v", [1 << 20, 5])
def test_verify_greedy(eng, v):
    """Temperature 0: argmax with ties to the lowest id; drafts of every kind."""
    rng = np.random.default_rng(v)
    lg = np.round(rng.standard_normal((4, 3, v)) * 2) / 2
    top = lg.argmax(-1)
    d = top[:, :2].astype(np.int32).copy()
    d[1, 1] = (d[1, 1] + 1) % v
    d[2, 0] = -1
    d[3, 1] = v
    u = rng.random((4, 3))
    acc, tok = run(eng, lg, d, u, 0.0)
    assert list(acc) == [2, 1, 0, 1]
    assert [int(tok[i, a]) for i, a in enumerate(acc)] == [int(top[i, a]) for i, a in enumerate(acc)]
    assert list(tok[0, :2]) == list(d[0]) and np.all(tok[2, 1:] == -1)
    # the drafter's logits are not looked at
    again = run(eng, lg, d, u, 0.0, np.full((4, 2, v), np.nan))
    assert np.array_equal(again[0], acc) and np.array_equal(again[1], tok)


@pytest.mark.parametrize("probs", [False, True])
@pytest.mark.parametrize("temperature", [0.0, 1.0])
def test_verify_rows_without_a_distribution(eng, probs, temperature):
    v, inf, nan = 9000, np.inf, np.nan
    rng = np.random.default_rng(3)
    lg = rng.standard_normal((8, 3, v)).astype(np.float32).astype(np.float64)
    dl = rng.standard_normal((8, 2, v)).astype(np.float32).astype(np.float64)
    if not probs:
        dl = None
    d = lg[:, :2].argmax(-1).astype(np.int32)
    u = np.zeros((8, 3))
    u[:, 2] = rng.random(8)
    lg[0, 0, 8999] = nan                 # a NaN in the first row
    lg[1, 1, 5] = inf                    # an infinity in the second
    lg[2, 2] = -inf                      # nothing left in the last
    lg[3, 0, :] = -inf                   # one id left
    lg[3, 0, 77] = -4.0
    d[3, 0] = 77
    lg[4, 0, d[4, 0] + 1:] = -inf        # half the vocabulary masked; the draft the last id left
    d[5, 0] = v + 3                      # no such id
    if probs:
        dl[6, 1, 3] = nan                # a draft row without one
        dl[7, 0] = -inf
    got = run(eng, lg, d, u, temperature, dl)
    check(lg, d, u, temperature, got, dl)
    assert got[0][0] == 0 and got[1][0, 0] == -1 and got[0][3] >= 1


def test_verify_borders(eng):
    """u = 0 keeps any draft the target can give and draws the first possible id; u just under 1 the last
    one; a certain target leaves nothing for the rest; equal distributions accept every draft."""
    v = 4100
    one = np.nextafter(np.float32(1), np.float32(0))
    lg = np.full((4, 2, v), -np.inf)
    lg[:, :, 1000:3000] = 0.0
    lg[3] = -np.inf
    lg[3, :, 2048] = 3.0
    d = np.array([[1500], [999], [2000], [2048]], np.int32)
    u = np.array([[0, 0], [0, 0], [one, one], [one, one]], np.float32)
    acc, tok = run(eng, lg, d, u, 1.0)
    assert list(acc) == [1, 0, 0, 1] and list(tok[0]) == [1500, 1000] and tok[1, 0] == 1000 and tok[2, 0] == 2999
    assert list(tok[3]) == [2048, 2048]
    acc, tok = run(eng, lg, d, u, 1.0, lg[:, :1])
    assert list(acc) == [1, 0, 1, 1]     # q = p: u q < p for every draft the target can give
    assert tok[1, 0] == 1000             # p - q leaves nothing: p itself


def test_verify_keeps_the_targets_distribution(eng):
    """Over 20,000 lanes with a poor drafter, the first emitted id has the target's probabilities: each count
    within 5 standard deviations."""
    rng = np.random.default_rng(21)
    v, n = 6, 680
    p = np.log(np.array([0.05, 0.3, 0.1, 0.25, 0.2, 0.1]))
    q = np.log(np.array([0.4, 0.1, 0.1, 0.1, 0.1, 0.2]))
    seen = np.zeros(v)
    for _ in range(30):
        d = rng.choice(v, (n, 2), p=np.exp(q)).astype(np.int32)
        u = rng.random((n, 3)).astype(np.float32)
        _, tok = run(eng, np.broadcast_to(p, (n, 3, v)).copy(), d, u, 1.0, np.broadcast_to(q, (n, 2, v)).copy())
        seen += np.bincount(tok[:, 0], minlength=v)
    N = seen.sum()
    P = np.exp(p)
    assert np.all(np.abs(seen - N * P) <= 5 * np.sqrt(N * P * (1 - P))), seen / N
