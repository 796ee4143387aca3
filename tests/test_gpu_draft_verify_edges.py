"""Sampled draft verification at the ends of what its arguments allow: the largest vocabulary in the most chunks, the
least and the largest temperatures, logits near float32's largest. References and checks of
tests/test_gpu_draft_verify.py."""
import numpy as np
import pytest

from test_gpu_draft_verify import check, make, run

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def eng():
    from qwen35 import Engine
    e = Engine(max_rows=64, max_ctx=64, seed=None)
    yield e
    e.close()


@pytest.mark.parametrize("n,k", [(1, 1), (1, 2), (3, 8)])
@pytest.mark.parametrize("probs", [False, True])
@pytest.mark.parametrize("bf16", [False, True])
def test_largest_vocabulary(eng, n, k, probs, bf16):
    v = 1 << 20
    print(f"verify 2^20 {n} {k} {probs} {bf16}", flush=True)
    rng = np.random.default_rng(n + k + 2 * probs + bf16)
    lg, dl, d, u = make(rng, n, k, v, probs, bf16, peak=14.0)
    check(lg, d, u, 0.8, run(eng, lg, d, u, 0.8, dl, bf16), dl)
    d[0, 0] = v - 1                            # the last id, refused or kept
    check(lg, d, u, 1.2, run(eng, lg, d, u, 1.2, dl, bf16), dl)


@pytest.mark.parametrize("probs", [False, True])
@pytest.mark.parametrize("temperature,size", [(0.001, 1.0), (0.001, 1e-3), (0.001, 1e37), (1e300, 1.0), (1e300, 1e37), (1e37, 1e37),
                                              (3.0, 1e37), (0.8, 1e-40)])
def test_temperatures_and_sizes(eng, probs, temperature, size):
    n, k, v = 7, 2, 9001
    print(f"verify temperature {temperature} size {size} probs {probs}", flush=True)
    rng = np.random.default_rng(int(probs))
    lg = (rng.standard_normal((n, k + 1, v)) * size).astype(np.float32).astype(np.float64)
    dl = (rng.standard_normal((n, k, v)) * size).astype(np.float32).astype(np.float64) if probs else None
    lg[1, :, 4000:] = -np.inf
    d = lg[:, :k].argmax(-1).astype(np.int32)
    d[2:4] = rng.integers(0, v, (2, k))
    u = rng.random((n, k + 1)).astype(np.float32)
    check(lg, d, u, temperature, run(eng, lg, d, u, temperature, dl), dl)
