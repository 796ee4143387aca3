"""Sampled speculative rounds (q35_mtp_verify_sample) at 6 lanes. Norms and two embedding rows are reshaped as
in the accepting-draft tests, milder: the two tokens' logits are +-6.25 x_d (a flat target: drafts are all but
never kept) or +-25 x_d (the two hold most of the probability: drafts of either are often kept). Checked: the emitted tokens are the float64 rule's (tests/kv4_ref.py)
on the logits that plain decode steps give for the same tokens; the state after each round is that of
plain steps over what was kept, bit for bit; temperature 0 is q35_mtp_verify; the stop cut; refusals."""
import numpy as np
import pytest

import kv4_ref as ref

pytestmark = pytest.mark.gpu

A, B, D = 248046, 1000, 7


@pytest.fixture(scope="module", params=[0x3E80, 0x3F80], ids=["flat", "peaked"])      # bf16 0.25, 1.0
def eng(request):
    from qwen35 import Engine
    e = Engine(max_rows=64, max_ctx=512, seed=0)
    e.peaked = request.param == 0x3F80
    emb = "model.language_model.embed_tokens.weight"
    E = e.read_tensor(emb, 248320 * 1024).reshape(248320, 1024)
    E[A, D], E[B, D] = request.param, request.param | 0x8000
    e.load_tensor(emb, E.reshape(-1))
    w = np.full(1024, 0xBF80, np.uint16)              # 1 + w = 0
    w[D] = 0x41C0                                     # 24
    e.load_tensor("model.language_model.norm.weight", w)
    yield e
    e.close()


def lanes_of(eng, st, n):
    from oracle.weights import lane_prompt_ids
    return [int(st.prefill(i, lane_prompt_ids(50 + i, 0, 6 + 5 * i))) for i in range(n)]


def same_state(a, b, n):
    for i in range(n):
        P = a.prefix_len(i)
        assert P == b.prefix_len(i)
        for which in ("S", "win"):
            assert np.array_equal(a.read(i, which), b.read(i, which)), (i, which)
        for which in ("k", "v"):
            assert np.array_equal(a.read(i, which, P), b.read(i, which, P)), (i, which)


def test_sampled_rounds_match_plain_steps(eng):
    from qwen35 import State
    n, T = 6, 1.5
    rng = np.random.default_rng(4)
    spec, plain, look = State(eng, n, 256, mtp_k=2, mtp_cap=64), State(eng, n, 256), State(eng, n, 256)
    cur = lanes_of(eng, spec, n)
    assert lanes_of(eng, plain, n) == cur
    kept, stats = set(), np.zeros(4, np.int64)
    for r in range(5):
        print(f"mtp sample: round {r}", flush=True)
        drafts = rng.choice([A, B, 5], (n, 2), p=[0.45, 0.45, 0.1]).astype(np.int32)
        u = rng.random((n, 3)).astype(np.float32)
        rows = np.zeros((n, 3, 248320))
        for i in range(n):
            plain.copy_lane(i, look, i)
        for j, toks in enumerate([np.array(cur), drafts[:, 0], drafts[:, 1]]):
            rows[:, j] = look.decode_step(toks, logits=True)[1]
        em = spec.mtp_verify_sample(cur, drafts, u, T, stats=stats)
        for i in range(n):
            a, w, border, near = ref.verify(rows[i], drafts[i], u[i].astype(np.float64), T)
            assert near > 1e-9
            assert len(em[i]) == a + 1 and list(em[i][:a]) == list(drafts[i][:a]), (r, i)
            assert ref.token_ok(int(em[i][a]), w, border), (r, i, em[i])
            kept.add(a)
            for t in [cur[i]] + [int(x) for x in em[i][:-1]]:
                plain.decode_step([t], [i])
            cur[i] = int(em[i][-1])
        same_state(spec, plain, n)
    assert kept >= {0, 1} or not eng.peaked        # (both drafts kept: the stop cut's test, with u = 0)
    assert stats[0] == 5 * n * 2 and stats[2] == 5 * n
    for s in (spec, plain, look):
        s.close()


def test_temperature_zero_is_the_greedy_round(eng):
    from qwen35 import State
    n = 6
    rng = np.random.default_rng(5)
    a, b = State(eng, n, 256, mtp_k=2, mtp_cap=64), State(eng, n, 256, mtp_k=2, mtp_cap=64)
    cur = lanes_of(eng, a, n)
    assert lanes_of(eng, b, n) == cur
    for r in range(3):
        print(f"mtp sample greedy: round {r}", flush=True)
        drafts = rng.choice([A, B], (n, 2)).astype(np.int32)
        ea = a.mtp_verify(cur, drafts, stop=A)
        eb = b.mtp_verify_sample(cur, drafts, rng.random((n, 3)), 0.0, stop=A)
        assert [list(x) for x in ea] == [list(x) for x in eb]
        cur = [int(x[-1]) for x in ea]
    same_state(a, b, n)
    a.close()
    b.close()


def test_stop_cut_and_refusals(eng):
    from qwen35 import EngineError, State
    st = State(eng, 2, 256, mtp_k=2, mtp_cap=64)
    cur = lanes_of(eng, st, 2)
    p0 = st.prefix_len(0)
    drafts, u = np.array([[A, B], [B, A]], np.int32), np.zeros((2, 3), np.float32)     # u = 0 keeps every draft
    em = st.mtp_verify_sample(cur, drafts, u, 1.0, stop=A)
    assert list(em[0]) == [A] and list(em[1]) == [B, A] and st.prefix_len(0) == p0 + 1
    before = [st.prefix_len(i) for i in range(2)]
    for kw in (dict(temperature=-1.0), dict(temperature=float("nan")), dict(temperature=1e-5), dict(u=np.full((2, 3), 1.0)),
               dict(u=np.full((2, 3), np.nan)), dict(drafts=[[A, -1], [B, A]]), dict(drafts=[[A, 248320], [B, A]]),
               dict(lanes=[0, 0]), dict(lanes=[0, 2])):
        args = dict(drafts=drafts, u=u, temperature=1.0)
        args.update(kw)
        with pytest.raises(EngineError):
            st.mtp_verify_sample(cur, args["drafts"], args["u"], args["temperature"], lanes=args.get("lanes"))
    assert [st.prefix_len(i) for i in range(2)] == before
    st.close()
