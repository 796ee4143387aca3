"""A sampled round (q35_mtp_verify_sample) in which one lane's logits have no distribution: that lane emits nothing and
keeps its state, the others finish their round, and later rounds of all of them are plain steps' bit for
bit. A NaN in a lane's K cache makes its logits NaN. The model is the peaked one of tests/test_gpu_mtp_sample.py."""
import numpy as np
import pytest

import kv4_ref as ref
from test_gpu_mtp_sample import A, B, D, lanes_of, same_state

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def eng():
    from qwen35 import Engine
    e = Engine(max_rows=64, max_ctx=512, seed=0)
    emb = "model.language_model.embed_tokens.weight"
    E = e.read_tensor(emb, 248320 * 1024).reshape(248320, 1024)
    E[A, D], E[B, D] = 0x3F80, 0xBF80
    e.load_tensor(emb, E.reshape(-1))
    w = np.full(1024, 0xBF80, np.uint16)              # 1 + w = 0
    w[D] = 0x41C0                                     # 24
    e.load_tensor("model.language_model.norm.weight", w)
    yield e
    e.close()


@pytest.mark.parametrize("then", ["round", "step"])
def test_one_lane_without_a_distribution(eng, then):
    from qwen35 import State
    n, T, sick = 4, 1.5, 1
    rng = np.random.default_rng(6)
    spec, plain, look = State(eng, n, 256, mtp_k=2, mtp_cap=64), State(eng, n, 256), State(eng, n, 256)
    cur = lanes_of(eng, spec, n)
    assert lanes_of(eng, plain, n) == cur
    P = spec.prefix_len(sick)
    good = spec.read(sick, "k", P)
    for r in range(3):
        print(f"mtp sample lanes: round {r}", flush=True)
        bad = r == 1
        drafts = rng.choice([A, B], (n, 2)).astype(np.int32)
        u = rng.random((n, 3)).astype(np.float32)
        if bad:
            P = spec.prefix_len(sick)
            good = spec.read(sick, "k", P)
            k = good.copy()
            k[0, :, 0, :] = 0x7FC0
            spec.write(sick, "k", k, P)
        rows = np.zeros((n, 3, 248320))
        for i in range(n):
            plain.copy_lane(i, look, i)
        for j, toks in enumerate([np.array(cur), drafts[:, 0], drafts[:, 1]]):
            rows[:, j] = look.decode_step(toks, logits=True)[1]
        stats = np.zeros(4, np.int64)
        em = spec.mtp_verify_sample(cur, drafts, u, T, stats=stats)
        if bad:
            assert em[sick] == [] and spec.prefix_len(sick) == P
            spec.write(sick, "k", good, P)
            if then == "step":               # what the round left behind the lane's prefix stays out of a plain step
                x, y = (s.decode_step([cur[sick]], [sick], logits=True) for s in (spec, plain))
                assert np.array_equal(x[1], y[1])
                cur[sick] = int(x[0][0])
        assert stats[0] == 2 * (n - bad) and stats[2] == n - bad and stats[3] == 3 * (n - bad)
        for i in range(n):
            if bad and i == sick:
                continue
            a, w, border, near = ref.verify(rows[i], drafts[i], u[i].astype(np.float64), T)
            assert near > 1e-9 and len(em[i]) == a + 1 and list(em[i][:a]) == list(drafts[i][:a])
            assert ref.token_ok(int(em[i][a]), w, border), (r, i, em[i])
            for t in [cur[i]] + [int(x) for x in em[i][:-1]]:
                plain.decode_step([t], [i])
            cur[i] = int(em[i][-1])
        same_state(spec, plain, n)
    for s in (spec, plain, look):
        s.close()


def test_temperature_zero_takes_such_rows_as_the_greedy_round_does(eng):
    from qwen35 import State
    a, b = State(eng, 2, 256, mtp_k=2, mtp_cap=64), State(eng, 2, 256, mtp_k=2, mtp_cap=64)
    cur = lanes_of(eng, a, 2)
    assert lanes_of(eng, b, 2) == cur
    for s in (a, b):
        P = s.prefix_len(0)
        k = s.read(0, "k", P)
        k[0, :, 0, :] = 0x7FC0
        s.write(0, "k", k, P)
    drafts = np.array([[A, B], [B, A]], np.int32)
    ea = a.mtp_verify(cur, drafts)
    eb = b.mtp_verify_sample(cur, drafts, np.full((2, 3), 0.5), 0.0)
    assert [list(x) for x in ea] == [list(x) for x in eb]
    assert [a.prefix_len(i) for i in range(2)] == [b.prefix_len(i) for i in range(2)]
    a.close()
    b.close()
