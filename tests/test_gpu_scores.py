"""Log probabilities on the model's own rows (q35_prefill_logprobs, q35_decode_step_logprobs): against float64 on the logits that
q35_prefill_all and q35_decode_step hand out, with the tolerances of test_gpu_logprobs.py; ids and states as theirs."""
import numpy as np
import pytest

from test_gpu_logprobs import check

pytestmark = pytest.mark.gpu


def fields(s, rows=slice(None)):
    return {k: v[rows] for k, v in s._asdict().items()}


@pytest.mark.parametrize("max_rows,n,top,temperature", [(8, 1, 0, 1.0), (16, 40, 3, 1.0), (64, 150, 32, 0.7), (512, 400, 5, 2.0)])
def test_prompt(max_rows, n, top, temperature):
    """Prompts of one wave, of several, and of waves whose rows take two lm_head launches."""
    from oracle.weights import lane_prompt_ids
    from qwen35 import Engine, State, VOCAB
    print(f"prompt scores {max_rows} {n} {top}", flush=True)
    ids = lane_prompt_ids(5, 0, n)
    e = Engine(max_rows=max_rows, max_ctx=512, seed=0)
    try:
        sa, sb, sc = State(e, 2, 500), State(e, 2, 500), State(e, 2, 500)
        want, _, lg = sa.prefill_all(1, ids, logits=True)
        got, s = sb.prefill_logprobs(1, ids, top=top, temperature=temperature)
        nxt = np.r_[ids[1:], -1]
        assert np.array_equal(got, want)
        check(fields(s), lg, nxt, top, temperature)
        other = np.random.default_rng(n).integers(-2, VOCAB + 2, n)
        got, s2 = sc.prefill_logprobs(1, ids, targets=other, top=top, temperature=temperature)
        check(fields(s2), lg, other, top, temperature)
        assert np.array_equal(got, want)
        assert np.array_equal(s.entropy, s2.entropy) and np.array_equal(s.top_ids, s2.top_ids)
        for w in ("S", "win"):
            assert np.array_equal(sa.read(1, w), sb.read(1, w))
        ta, tb = sa.decode_step([want[-1]], [1]), sb.decode_step([want[-1]], [1])
        assert np.array_equal(ta, tb)
    finally:
        e.close()


@pytest.mark.parametrize("graph", [0, 1])
@pytest.mark.parametrize("n", [1, 3, 40])
def test_steps(n, graph):
    """Steps with and without scores in turn, captured ones replayed, another number of lanes between: the ids and logits of
    a state that takes plain steps."""
    from oracle.weights import lane_prompt_ids
    from qwen35 import Engine, State
    print(f"step scores {n} graph={graph}", flush=True)
    e = Engine(max_rows=64, max_ctx=128, seed=0)
    e.set_option("graph", graph)
    rng = np.random.default_rng(n)
    try:
        sa, sb = State(e, n + 1, 100), State(e, n + 1, 100)
        lanes = rng.permutation(n + 1)[:n]
        tok = []
        for l in lanes:
            p = lane_prompt_ids(9, int(l), 5)
            tok.append(sa.prefill(int(l), p))
            assert sb.prefill(int(l), p) == tok[-1]
        tok = np.array(tok, np.int32)
        for step in range(6):
            k = n if step != 3 else max(1, n // 2)
            want, lg = sa.decode_step(tok[:k], lanes[:k], logits=True)
            if step == 1:
                got = sb.decode_step(tok[:k], lanes[:k])
            else:
                targets = None if step % 2 else rng.integers(0, 1000, k)
                got, s = sb.decode_step_logprobs(tok[:k], lanes[:k], targets=targets, top=4, temperature=1.0 + step / 4)
                check(fields(s), lg, want if targets is None else targets, 4, 1.0 + step / 4)
                if targets is None:
                    assert (s.ranks == 0).all()
            assert np.array_equal(got, want)
            tok[:k] = want
        assert all(np.array_equal(sa.read(int(l), "S"), sb.read(int(l), "S")) for l in lanes)
    finally:
        e.close()


def test_refusals():
    """A refused call leaves the state; the arrays that are not wanted stay away."""
    import ctypes as C
    from qwen35 import Engine, EngineError, State, load_library
    from qwen35.engine import _LOGPROBS, _p
    e = Engine(max_rows=8, max_ctx=64, seed=0)
    try:
        s = State(e, 1, 40)
        y = s.prefill(0, [5, 6, 7])
        before = s.read(0, "S")
        for text, kw in [("temperature", dict(temperature=0.0)), ("top is", dict(top=33)), ("top is", dict(top=-1)),
                         ("temperature", dict(temperature=float("nan")))]:
            with pytest.raises(EngineError, match=text):
                s.prefill_logprobs(0, [1, 2], **kw)
            with pytest.raises(EngineError, match=text):
                s.decode_step_logprobs([y], **kw)
        for bad in ([1], [1, 2, 3]):
            with pytest.raises(ValueError):
                s.prefill_logprobs(0, [1, 2], targets=bad)
        with pytest.raises(EngineError, match="capacity"):
            s.prefill_logprobs(0, [1] * 38)
        with pytest.raises(EngineError, match="token out of range"):
            s.decode_step_logprobs([-1])
        L, ids, out, ent = load_library(), np.array([1, 2], np.int32), np.zeros(2, np.int32), np.zeros(2, np.float32)
        own = _LOGPROBS.pack(64, 0, 0, 0, 1.0, 0, 0, 0, ent.ctypes.data, 0, 0)
        for rc in (L.q35_prefill_logprobs(e.h, s.h, 0, _p(ids), 2, _p(out), None), L.q35_decode_step_logprobs(e.h, s.h, None, 1, _p(ids), _p(out), None),
                   L.q35_prefill_logprobs(e.h, s.h, 0, _p(ids), 2, _p(out), own), L.q35_decode_step_logprobs(e.h, s.h, None, 1, _p(ids), _p(out), own)):
            assert rc == -1
        assert s.prefix_len(0) == 3 and np.array_equal(s.read(0, "S"), before)
        d = _LOGPROBS.pack(0, 0, 0, 0, 1.0, 7, 0, 0, ent.ctypes.data, 0, 0)
        assert L.q35_prefill_logprobs(e.h, s.h, 0, _p(ids), 2, _p(out), d) == 0 and (ent > 0).all()
    finally:
        e.close()
