"""Heads at positions on some of the four axes only (test_gpu_kv4_axes.py has maps with all up to the largest), against
float64 with its tolerances."""
import numpy as np
import pytest

from test_gpu_kv4 import Dev, Heads
from test_gpu_kv4_axes import close, turned

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def eng():
    from qwen35 import Engine
    e = Engine(max_rows=64, max_ctx=1000, seed=None)
    yield e
    e.close()


@pytest.mark.parametrize("hq,kv,d,rot", [(8, 2, 256, 64), (5, 1, 128, 128), (4, 4, 64, 6)])
@pytest.mark.parametrize("named", [[1], [3], [0, 3], [1, 2], [2, 3], [0, 2, 3]])
@pytest.mark.parametrize("R", [1, 1500])
def test_axes_left_out(eng, hq, kv, d, rot, named, R):
    """Positions [axis][row], those on the axes that no pair has of a value that would show."""
    import torch
    print(f"named axes {named} {hq} {kv} {d} {rot} {R}", flush=True)
    rng, D = np.random.default_rng(sum(named) + d + R), Dev()
    h = Heads(rng, R, hq, kv, d)
    axis = bytes(named[i % len(named)] for i in range(rot // 2))
    names = sorted(set(axis))
    where = np.full((R, 4), 12345, np.int32)
    where[:, names] = rng.integers(-500, 100000, (R, len(names)))
    room = D.up(np.ascontiguousarray(where.T))
    x, qn, kn = D.up(h.x), D.up(h.qn), D.up(h.kn)
    qo, ko = (torch.zeros(R, m, d, dtype=torch.int16, device="cuda") for m in (hq, kv))
    torch.cuda.synchronize()
    v, _ = h.views(x.data_ptr())
    eng.op_qk_norm_rope_axes((room.data_ptr(), 1, R), axis, R, hq, kv, d, rot_dim=rot, theta=1e6, eps=1e-6, q_norm=qn.data_ptr(),
                             k_norm=kn.data_ptr(), q_out=(qo.data_ptr(), hq * d, d), k_out=(ko.data_ptr(), kv * d, d), **v)
    eng.sync()
    q, k, _ = h.parts()
    close(D.bits(qo), *turned(q, h.qn, where, axis, rot, 1e6, 1e-6))
    close(D.bits(ko), *turned(k, h.kn, where, axis, rot, 1e6, 1e-6))
