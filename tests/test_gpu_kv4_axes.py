"""Heads at positions on several axes, with and without the append at slots apart from them, against float64
(tests/kv4_ref.py). Tolerances as in test_gpu_kv4.py: eight float32 roundings on a rotated pair, then bf16's."""
import numpy as np
import pytest

import kv4_ref as ref
from test_gpu_kv4 import SLACK, Dev, Heads, check_codes, read_cache

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def eng():
    from qwen35 import Engine
    e = Engine(max_rows=64, max_ctx=40000, seed=None)
    yield e
    e.close()


def turned(x, w, at, axis, rot, theta, eps):
    """x [rows][heads][d], at [rows][axes] -> (result, size) as ref.norm_rope gives them for one axis."""
    y, size = ref.norm_rope(x, ref.val(w), np.zeros(len(x)), 0, theta, eps)
    half = rot // 2
    if rot:
        ang = at[:, list(axis)].astype(np.float64)[:, None, :] * theta ** (-2.0 * np.arange(half) / rot)
        c, s = np.cos(ang), np.sin(ang)
        a, b = y[..., :half].copy(), y[..., half:rot].copy()
        y[..., :half], y[..., half:rot] = a * c - b * s, b * c + a * s
        size = size.copy()
        size[..., :half] = size[..., half:rot] = np.abs(a) + np.abs(b)
    return y, size


def close(bits, want, size):
    assert np.all(np.abs(ref.val(bits) - want) <= 2.0 ** -8 * np.abs(want) + SLACK * size + 1e-37)


AXES = [(8, 2, 256, 64, 3, True), (8, 2, 256, 256, 4, False), (5, 1, 128, 128, 2, True), (14, 2, 64, 64, 3, False),
        (1, 7, 64, 6, 3, True), (2, 1, 256, 2, 1, True), (4, 2, 128, 100, 3, True), (3, 3, 128, 0, 1, True)]


def a_map(rot, axes, dealt):
    from qwen35 import pair_axes
    pairs = rot // 2
    return pair_axes([pairs // axes + (a < pairs % axes) for a in range(axes)], dealt)


@pytest.mark.parametrize("hq,kv,d,rot,axes,dealt", AXES)
@pytest.mark.parametrize("R", [1, 3, 300, 1500, 4099])
def test_norm_rope_axes(eng, hq, kv, d, rot, axes, dealt, R):
    """Positions of any int32, as [rows][axes] and as [axes][rows] with spare elements; one position for all rows."""
    import torch
    print(f"axes {hq} {kv} {d} {rot} {axes} {R}", flush=True)
    rng, D = np.random.default_rng(hq * d + rot + R), Dev()
    h = Heads(rng, R, hq, kv, d, pad=8)
    axis = a_map(rot, axes, dealt)
    at = rng.integers(0, 200000, (R, axes)).astype(np.int32)
    at[0] = [0, -1, 2 ** 31 - 1, -2 ** 31][:axes]
    x, qn, kn = D.up(h.x), D.up(h.qn), D.up(h.kn)
    q, k, _ = h.parts()
    same = np.broadcast_to(at[R // 2], (R, axes))
    for layout, pos in [("rows", at), ("axes", at), ("one", same)]:
        if layout == "rows":
            t, step = D.up(np.pad(at, ((0, 0), (0, 2)))), (axes + 2, 1)
        elif layout == "axes":
            t, step = D.up(np.pad(at.T, ((0, 0), (0, 5)))), (1, R + 5)
        else:
            t, step = D.up(at[R // 2]), (0, 1)
        qo, ko = (torch.zeros(R, m, d, dtype=torch.int16, device="cuda") for m in (hq, kv))
        torch.cuda.synchronize()
        v, _ = h.views(x.data_ptr())
        eng.op_qk_norm_rope_axes((t.data_ptr(), *step), axis, R, hq, kv, d, rot_dim=rot, theta=1e6, eps=1e-6, q_norm=qn.data_ptr(),
                                 k_norm=kn.data_ptr(), q_out=(qo.data_ptr(), hq * d, d), k_out=(ko.data_ptr(), kv * d, d), **v)
        eng.sync()
        close(D.bits(qo), *turned(q, h.qn, pos, axis, rot, 1e6, 1e-6))
        close(D.bits(ko), *turned(k, h.kn, pos, axis, rot, 1e6, 1e-6))


@pytest.mark.parametrize("hq,kv,d,rot", [(8, 2, 256, 64), (5, 1, 128, 128), (4, 4, 64, 6)])
@pytest.mark.parametrize("n,T", [(1, 1), (5, 3), (270, 2), (1, 2100)])
def test_one_axis_is_the_rope(eng, hq, kv, d, rot, n, T):
    """With one axis and the sequences' positions: the same bits as q35_op_qk_norm_rope."""
    import torch
    rng, D = np.random.default_rng(n * T + d), Dev()
    h = Heads(rng, n * T, hq, kv, d)
    pos = rng.integers(0, 100000, n).astype(np.int32)
    at = D.up((pos[:, None] + np.arange(T, dtype=np.int32)).reshape(-1).astype(np.int32))
    x, qn, kn = D.up(h.x), D.up(h.qn), D.up(h.kn)
    out = [[torch.zeros(n * T, m, d, dtype=torch.int16, device="cuda") for m in (hq, kv)] for _ in range(2)]
    torch.cuda.synchronize()
    v, _ = h.views(x.data_ptr())
    args = dict(rot_dim=rot, theta=1e7, eps=1e-6, q_norm=qn.data_ptr(), k_norm=kn.data_ptr(), **v)
    views = [dict(q_out=(a.data_ptr(), hq * d, d), k_out=(b.data_ptr(), kv * d, d)) for a, b in out]
    eng.op_qk_norm_rope(pos, T, hq, kv, d, **args, **views[0])
    eng.op_qk_norm_rope_axes((at.data_ptr(), 1, 0), bytes(rot // 2), n * T, hq, kv, d, **args, **views[1])
    eng.sync()
    assert all(torch.equal(a, b) for a, b in zip(*out))


@pytest.mark.parametrize("hq,kv,d,rot,axes,dealt", [(8, 2, 256, 64, 3, True), (5, 1, 128, 128, 3, False), (4, 4, 64, 32, 2, True)])
@pytest.mark.parametrize("n,T,slot0", [(1, 1, 0), (4, 3, 30), (2, 70, 17), (270, 1, 5), (3, 1, 64)])
def test_append_axes(eng, hq, kv, d, rot, axes, dealt, n, T, slot0):
    """Rows at slots of their own; every other slot, lane and layer stays."""
    import torch
    from qwen35 import KvCache4
    print(f"append axes {hq} {kv} {d} {rot} {n}x{T}@{slot0}", flush=True)
    rng, D = np.random.default_rng(n * T + d), Dev()
    cap = slot0 + n + T + 2
    c = KvCache4(eng, n + 1, cap, layers=2, kv_heads=kv, head_dim=d)
    lanes = rng.permutation(n + 1)[:n].astype(np.int32)
    slots = (slot0 + np.arange(n) % 7).astype(np.int32)
    c.set_len(None, np.full(n + 1, cap, np.int32))
    before = read_cache(eng, c, 1, 0, n + 1, 0, cap)
    c.set_len(lanes, slots)
    h = Heads(rng, n * T, hq, kv, d)
    axis = a_map(rot, axes, dealt)
    at = rng.integers(0, 90000, (n * T, axes)).astype(np.int32)
    x, qn, kn, t = D.up(h.x), D.up(h.qn), D.up(h.kn), D.up(at)
    qo, ko, vo = (torch.zeros(n * T, m, d, dtype=torch.int16, device="cuda") for m in (hq, kv, kv))
    torch.cuda.synchronize()
    v, vview = h.views(x.data_ptr())
    eng.op_kv4_append_axes(c, 1, lanes, slots, T, hq, (t.data_ptr(), axes, 1), axis, rot_dim=rot, theta=1e7, eps=1e-6,
                           q_norm=qn.data_ptr(), k_norm=kn.data_ptr(), v=vview, q_out=(qo.data_ptr(), hq * d, d),
                           k_out=(ko.data_ptr(), kv * d, d), v_out=(vo.data_ptr(), kv * d, d), **v)
    eng.sync()
    assert [c.length(1, l) for l in lanes] == list(slots + T) and [c.length(0, l) for l in lanes] == list(slots)
    q, k, vx = h.parts()
    close(D.bits(qo), *turned(q, h.qn, at, axis, rot, 1e7, 1e-6))
    want, size = turned(k, h.kn, at, axis, rot, 1e7, 1e-6)
    c.set_len(None, np.full(n + 1, cap, np.int32))
    kc, ks, vc, vs = read_cache(eng, c, 1, 0, n + 1, 0, cap)
    rows = lambda a: np.concatenate([a[l, :, p:p + T].transpose(1, 0, 2) for l, p in zip(lanes, slots)])  # noqa: E731
    wide = SLACK * np.maximum(size / np.maximum(np.abs(want), 1e-30), 1)
    amax = np.abs(want).reshape(*want.shape[:-1], -1, 32).max(-1)
    gw = (SLACK * size).reshape(*want.shape[:-1], -1, 32).max(-1)
    assert np.all((rows(ks) >= ref.scale_byte(amax - gw)) & (rows(ks) <= ref.scale_byte(amax + gw)))
    assert np.all(ref.nearest_ok(want, rows(kc), rows(ks), wide))
    check_codes(vx, rows(vc), rows(vs), 0.0)
    assert np.array_equal(ref.val(D.bits(ko)), ref.values(rows(kc), rows(ks)))
    assert np.array_equal(ref.val(D.bits(vo)), ref.values(rows(vc), rows(vs)))
    for a, b in zip((kc, ks, vc, vs), before):
        a = a.copy()
        for l, p in zip(lanes, slots):
            a[l, :, p:p + T] = b[l, :, p:p + T]
        assert np.array_equal(a, b)
    assert not any(z.any() for z in read_cache(eng, c, 0, 0, n + 1, 0, cap))
    c.close()


def test_positions_far_apart(eng):
    """Rows' and axes' positions more than 2^32 bytes apart."""
    import torch
    rng, D = np.random.default_rng(8), Dev()
    h = Heads(rng, 3, 4, 2, 128)
    axis, step = a_map(64, 2, True), 2 ** 30 + 3
    at = rng.integers(-1000, 100000, (3, 2)).astype(np.int32)
    x, qn, kn = D.up(h.x), D.up(h.qn), D.up(h.kn)
    for rows, axes in ((step, 1), (1, step)):
        t = torch.zeros(2 * step + 8, dtype=torch.int32, device="cuda")
        for r in range(3):
            for a in range(2):
                t[r * rows + a * axes] = int(at[r, a])
        qo, ko = (torch.zeros(3, m, 128, dtype=torch.int16, device="cuda") for m in (4, 2))
        torch.cuda.synchronize()
        v, _ = h.views(x.data_ptr())
        eng.op_qk_norm_rope_axes((t.data_ptr(), rows, axes), axis, 3, 4, 2, 128, rot_dim=64, theta=1e6, eps=1e-6, q_norm=qn.data_ptr(),
                                 k_norm=kn.data_ptr(), q_out=(qo.data_ptr(), 512, 128), k_out=(ko.data_ptr(), 256, 128), **v)
        eng.sync()
        q, k, _ = h.parts()
        close(D.bits(qo), *turned(q, h.qn, at, axis, 64, 1e6, 1e-6))
        close(D.bits(ko), *turned(k, h.kn, at, axis, 64, 1e6, 1e-6))
        del t
    torch.cuda.empty_cache()
