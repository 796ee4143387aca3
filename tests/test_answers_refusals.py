"""Argument checks of the operators of answers that share prompts, on the CPU: their host source built against a stub that
counts launches. A refused call has its status and text, launches nothing and leaves the lanes' lengths; the call beside it
that is allowed goes through, in the launches and with the prompts that it should have."""
import ctypes as C
import shutil
import subprocess
from pathlib import Path

import numpy as np
import pytest

from test_kv4_refusals import ARG, CAP, REPO, STATE, Bed, heads

NAMES = ("q35_op_qk_norm_rope_axes", "q35_op_kv4_append_axes", "q35_op_attn_kv4_shared", "q35_op_token_logprobs")


@pytest.fixture(scope="module")
def lib(tmp_path_factory):
    cxx = shutil.which("g++") or "/opt/rocm/llvm/bin/clang++"
    so, src = tmp_path_factory.mktemp("answers") / "libanswershost.so", REPO / "qwen3.5-0.8b_amd" / "csrc"
    subprocess.run([cxx, "-std=c++17", "-O1", "-shared", "-fPIC", "-Bsymbolic", "-D__HIP_PLATFORM_AMD__=1", "-I/opt/rocm/include",
                    "-I", str(src), "-I", str(REPO / "include"), str(Path(__file__).parent / "answers_host_stub.cpp"),
                    str(src / "q35_kv4.cpp"), str(src / "q35_answers.cpp"), "-o", str(so)], check=True, capture_output=True)
    from qwen35 import engine
    L = C.CDLL(str(so))
    for name in tuple("q35_kv4_" + n for n in ("alloc", "free", "set_len", "len")) + NAMES:
        f = getattr(L, name)
        f.argtypes, f.restype = engine._SIGS[name]
    L.stub_engine.restype = C.c_void_p
    L.stub_launches.argtypes = [C.c_void_p]
    L.stub_rows.restype = C.c_longlong
    L.stub_room.argtypes = [C.c_longlong]
    L.stub_shared.argtypes = [C.c_void_p]
    L.q35_last_error.restype = C.c_char_p
    return L


@pytest.fixture
def bed(lib):
    return Bed(lib)


def at(pos=1 << 12, row=3, axis=1):
    from qwen35.engine import _VIEW
    return _VIEW.pack(pos, row, axis)


def test_rope_axes(bed):
    L, far = bed.L, 1 << 16

    def call(rows=5, kv=2, d=64, where=at(), axis=bytes(16), **kw):
        h = heads(**{**dict(v=(0, 0, 0), k_out=(5 << 16, 128, 64)), **kw})
        return L.q35_op_qk_norm_rope_axes(bed.e, h, kv, d, where, axis, rows)

    assert call() == 0 and L.stub_rows() == 5
    n = L.stub_launches(bed.e)
    for text, kw in [("null argument", dict(where=None)), ("null positions", dict(where=at(0))), ("null positions", dict(axis=None)),
                     ("misaligned positions", dict(where=at((1 << 12) + 2))), ("negative stride", dict(where=at(row=-1))),
                     ("negative stride", dict(where=at(axis=-1))), ("axis is 0", dict(axis=bytes([0] * 15 + [4]))),
                     ("axis is 0", dict(axis=bytes([255] * 16))), ("row count", dict(rows=0)), ("row count", dict(rows=-1)),
                     ("row count", dict(rows=4 * (2 ** 24 - 1) + 1)), ("head_dim", dict(d=96)), ("head count", dict(kv=0)),
                     ("rot_dim", dict(rot_dim=66)), ("rot_dim", dict(rot_dim=5)), ("theta", dict(theta=0.0)),
                     ("no norm", dict(v=(far, 512, 64))), ("overlap", dict(k_out=(far, 64, 64))), ("null norm", dict(k_norm=None))]:
        bed.refused(ARG, call(**kw), text)
    assert L.stub_launches(bed.e) == n
    # the neighbours: no rotation needs no positions; every pair's axis arrives
    assert call(rot_dim=0, where=at(0), axis=None) == 0 and L.stub_axes() == 0
    axis = bytes(np.random.default_rng(0).integers(0, 4, 128).astype(np.uint8))
    assert call(kv=1, d=256, rot_dim=256, axis=axis, q=(far, 2048, 256), q_out=(2 * far, 1024, 256), k_out=(3 * far, 256, 256)) == 0
    assert bytes(L.stub_axis(i) for i in range(128)) == axis and L.stub_axes() == max(axis) + 1
    assert call(rows=4 * (2 ** 24 - 1), k_out=(far, 128, 64)) == 0


def test_append_axes(bed):
    def call(lanes, slots, T=1, layer=0, where=at(), axis=bytes(16), **kw):
        la, p = np.array(lanes, np.int32), np.array(slots, np.int32)
        return bed.L.q35_op_kv4_append_axes(bed.e, bed.c, layer, la.ctypes.data, p.ctypes.data, p.size, T, heads(**kw), where, axis)

    assert call([0, 2], [0, 0], T=5) == 0 and bed.lengths() == [5, 0, 5]
    n = bed.L.stub_launches(bed.e)
    for code, text, args, kw in [
            (ARG, "twice", ([1, 1], [0, 0]), {}), (ARG, "lane out of range", ([3], [0]), {}), (STATE, "gap", ([1], [1]), {}),
            (CAP, "capacity", ([0], [4]), {"T": 97}), (CAP, "capacity", ([0], [-1]), {}), (ARG, "layer", ([0], [4]), {"layer": 2}),
            (ARG, "null positions", ([0], [4]), {"where": at(0)}), (ARG, "null positions", ([0], [4]), {"axis": None}),
            (ARG, "null argument", ([0], [4]), {"where": None}), (ARG, "axis is 0", ([0], [4]), {"axis": bytes([9] * 16)}),
            (ARG, "k: null", ([0], [4]), {"k": (0, 512, 64)}), (ARG, "v: null", ([0], [4]), {"v": (0, 512, 64)}),
            (ARG, "k: the pointer", ([0], [4]), {"k": ((1 << 16) + 8, 512, 64)})]:
        bed.refused(code, call(*args, **kw), text)
    assert bed.L.stub_launches(bed.e) == n and bed.lengths() == [5, 0, 5]
    assert call([0], [5], T=95) == 0 and bed.lengths() == [100, 0, 5]
    assert call([0], [3]) == 0 and bed.lengths() == [4, 0, 5]
    bed.L.stub_rows()
    # a launch has 256 sequences: the positions move on with the rows
    big = C.c_void_p()
    assert bed.L.q35_kv4_alloc(bed.e, 1, 300, 64, 2, 64, C.byref(big)) == 0
    z, before = np.zeros(300, np.int32), bed.L.stub_launches(bed.e)
    assert bed.L.q35_op_kv4_append_axes(bed.e, big, 0, None, z.ctypes.data, 300, 2, heads(k_out=(0, 0, 0)), at(), bytes(16)) == 0
    assert bed.L.stub_launches(bed.e) - before == 2 and bed.L.stub_rows() == 600
    assert bed.L.q35_kv4_free(bed.e, big) == 0


class Shared(Bed):
    """The bed's cache and a prompts' cache of 2 layers x 4 lanes x 50 slots, 2 heads of 64."""

    def __init__(self, lib):
        super().__init__(lib)
        self.p = C.c_void_p()
        assert lib.q35_kv4_alloc(self.e, 2, 4, 50, 2, 64, C.byref(self.p)) == 0
        n = np.array([50, 20, 0, 7], np.int32)
        assert lib.q35_kv4_set_len(self.e, self.p, None, n.ctypes.data, 4) == 0
        assert self.set_len([0, 1, 2], [100, 10, 5]) == 0

    def call(self, plane, plen, lanes, pos, T=1, layer=0, hq=4, q=(1 << 16, 256, 64), out=(1 << 20, 256, 64), gate=None,
             scale=0.125, prefix=None, cache=None):
        from qwen35.engine import _VIEW
        a = [None if x is None else np.array(x, np.int32) for x in (plane, plen, lanes, pos)]
        ptr = [None if x is None else x.ctypes.data for x in a]
        return self.L.q35_op_attn_kv4_shared(self.e, prefix or self.p, cache or self.c, layer, *ptr, len(pos), T, hq,
                                             q and _VIEW.pack(*q), gate and _VIEW.pack(*gate), scale, out and _VIEW.pack(*out))


def test_shared(lib):
    s = Shared(lib)
    L = s.L
    assert s.call([0, 1], [50, 3], [0, 1], [99, 9]) == 0 and s.call([-1, -9], [7, 0], [0, 1], [0, 0]) == 0
    n = L.stub_launches(s.e)
    assert n == 2
    other, foreign, e2 = C.c_void_p(), C.c_void_p(), C.c_void_p(L.stub_engine())
    assert L.q35_kv4_alloc(s.e, 2, 4, 50, 2, 128, C.byref(other)) == 0 and L.q35_kv4_alloc(e2, 2, 4, 50, 2, 64, C.byref(foreign)) == 0
    thin = C.c_void_p()
    assert L.q35_kv4_alloc(s.e, 1, 4, 50, 2, 64, C.byref(thin)) == 0
    ok = ([0], [50], [0], [99])
    for code, text, args, kw in [
            (STATE, "prefix slots", ([0], [51], [0], [0]), {}), (STATE, "prefix slots", ([2], [1], [0], [0]), {}),
            (ARG, "prefix lane out of range", ([4], [1], [0], [0]), {}), (ARG, "negative prefix", ([0], [-1], [0], [0]), {}),
            (ARG, "negative prefix", ([-1], [-1], [0], [0]), {}),
            (STATE, "does not hold", ([0], [5], [1], [10]), {}), (STATE, "does not hold", ([0], [5], [1], [9]), {"T": 2}),
            (CAP, "capacity", ([0], [5], [0], [-1]), {}), (CAP, "capacity", ([0], [5], [0], [100]), {}),
            (ARG, "lane out of range", ([0], [5], [3], [0]), {}), (ARG, "row count", ([0], [5], [0], [0]), {"T": 0}),
            (ARG, "layer", ok, {"layer": 2}), (ARG, "layer", ok, {"layer": -1}), (ARG, "q_heads", ok, {"hq": 3}),
            (ARG, "q_heads", ok, {"hq": 0}), (ARG, "q_heads", ok, {"hq": 1026}), (ARG, "scale", ok, {"scale": float("nan")}),
            (ARG, "scale", ok, {"scale": 3e38}), (ARG, "null argument", ok, {"q": None}), (ARG, "null argument", ok, {"out": None}),
            (ARG, "null argument", (None, [5], [0], [0]), {}), (ARG, "null argument", ([0], None, [0], [0]), {}),
            (ARG, "q: null", ok, {"q": (0, 256, 64)}), (ARG, "q: the pointer", ok, {"q": ((1 << 16) + 2, 256, 64)}),
            (ARG, "gate: the pointer", ok, {"gate": (1 << 16, 100, 64)}), (ARG, "out: rows or heads", ok, {"out": (1 << 20, 256, 32)}),
            (ARG, "heads differ", ok, {"prefix": other}), (ARG, "another engine", ok, {"prefix": foreign}),
            (ARG, "another engine", ok, {"cache": foreign}), (ARG, "layer out of range", ok, {"prefix": thin, "layer": 1}),
            (ARG, "its own prefix", ([0], [5], [0], [9]), {"prefix": s.c}), (ARG, "its own prefix", ([1], [5], [1], [9]), {"prefix": s.c})]:
        s.refused(code, s.call(*args, **kw), text)
    assert L.stub_launches(s.e) == n
    assert s.call([0], [5], [1], [9], prefix=s.c) == 0 and s.call([1], [0], [1], [9], prefix=s.c) == 0
    assert s.call(*ok, gate=(0, 0, 0)) == 0 and s.call(*ok, scale=0.0, hq=1024, q=(1 << 16, 0, 0), out=(1 << 20, 65536, 64)) == 0
    assert s.call([0, 0], [50, 50], None, [0, 0], layer=1) == 0


def last(lib, most=300):
    a = np.zeros(3 + 4 * most, np.int32)
    lib.stub_shared(a.ctypes.data)
    return a[:3].tolist(), a[3:3 + 4 * a[0]].reshape(-1, 4)


def test_shared_prompts_are_sorted(lib):
    """Sequences of one lane and length share a prompt wherever they stand; those without one come last."""
    s = Shared(lib)
    assert s.call([1, 0, -1, 1, 3, 0, 1, 2], [20, 50, 3, 20, 7, 49, 19, 0], [0] * 8, [7, 6, 5, 4, 3, 2, 1, 0]) == 0
    (n, groups, T), rows = last(lib)
    assert (n, groups, T) == (8, 6, 1)
    assert rows.tolist() == [[5, 0, 49, 2], [1, 0, 50, 6], [6, 1, 19, 1], [0, 1, 20, 7], [3, 1, 20, 4], [4, 3, 7, 3], [2, -1, 0, 5],
                             [7, -1, 0, 0]]


def test_shared_in_launches(lib):
    """256 neighbouring sequences, 64 prompts and the partial results' room bound a launch; every row is in one."""
    s, big, pre = Shared(lib), C.c_void_p(), C.c_void_p()
    assert lib.q35_kv4_alloc(s.e, 1, 100, 64, 2, 64, C.byref(pre)) == 0 and lib.q35_kv4_alloc(s.e, 1, 2, 4096, 2, 64, C.byref(big)) == 0
    a, b = np.full(100, 64, np.int32), np.full(2, 4096, np.int32)
    assert lib.q35_kv4_set_len(s.e, pre, None, a.ctypes.data, 100) == 0 and lib.q35_kv4_set_len(s.e, big, None, b.ctypes.data, 2) == 0

    def launches(n, T, hq, groups=1):
        before = lib.stub_launches(s.e)
        lib.stub_rows()
        g = [i % groups for i in range(n)]
        assert s.call(g, [64] * n, [0] * n, [0] * n, T=T, hq=hq, prefix=pre, cache=big, out=(1 << 20, 64 * hq, 64)) == 0
        assert lib.stub_rows() == n * T
        return lib.stub_launches(s.e) - before

    assert launches(256, 1, 8) == 1 and launches(257, 1, 8) == 2 and launches(1000, 1, 8) == 4
    assert launches(128, 1, 8, 64) == 1 and launches(130, 1, 8, 65) == 2 and launches(256, 1, 8, 100) == 2
    # room for 2064 tiles of 16 rows, 1032 a kv head: T / 4 of each sequence (4 rows a query row), and as much of its prompt's
    assert launches(256, 8, 8) == 1 and launches(256, 9, 8) == 2 and launches(128, 16, 8, 64) == 1 and launches(128, 17, 8, 64) == 2
    assert launches(1, 2064, 8) == 1 and launches(1, 2065, 8) == 2 and launches(3, 4096, 8) == 6
    assert launches(1, 4096, 1024) == 256      # 512 query heads each: 16 rows of T in 512 tiles
    lib.stub_room(68)
    assert launches(5, 3, 1024) == 15
    lib.stub_room(0)


def test_logprobs(bed):
    from qwen35.engine import _LOGPROBS
    base = dict(logits=1 << 16, ld=100, dtype=0, targets=1 << 12, temperature=1.0, top=5, logprobs=1 << 12, ranks=1 << 12,
                entropy=1 << 12, top_ids=1 << 12, top_logprobs=1 << 12)

    def call(rows=3, vocab=100, **kw):
        return bed.L.q35_op_token_logprobs(bed.e, _LOGPROBS.pack(*{**base, **kw}.values()), rows, vocab)

    assert call() == 0
    n = bed.L.stub_launches(bed.e)
    for text, kw in [("null argument", dict(logits=0)), ("row count", dict(rows=0)), ("row count", dict(rows=-3)), ("vocab", dict(vocab=0)),
                     ("vocab", dict(vocab=(1 << 20) + 1, ld=1 << 21)), ("row stride", dict(ld=99)), ("dtype", dict(dtype=2)),
                     ("misaligned", dict(logits=(1 << 16) + 2)), ("misaligned", dict(logits=(1 << 16) + 1, dtype=1)),
                     ("temperature", dict(temperature=0.0)), ("temperature", dict(temperature=-1.0)),
                     ("temperature", dict(temperature=float("nan"))), ("temperature", dict(temperature=float("inf"))),
                     ("top is", dict(top=33)), ("top is", dict(top=-1)), ("top is", dict(top=4, vocab=3)), ("need targets", dict(targets=0))]:
        bed.refused(ARG, call(**kw), text)
    bed.refused(ARG, bed.L.q35_op_token_logprobs(bed.e, None, 1, 5), "null argument")
    assert bed.L.stub_launches(bed.e) == n
    assert call(targets=0, logprobs=0, ranks=0) == 0 and call(top=32) == 0 and call(vocab=1, top=1) == 0
    assert call(logits=(1 << 16) + 2, dtype=1) == 0 and call(logits=(1 << 16) + 4) == 0 and call(vocab=1 << 20, ld=1 << 20) == 0
    assert call(temperature=0.001) == 0 and call(temperature=1000.0) == 0 and call(rows=2 ** 31 - 1) == 0


def test_pair_axes():
    from qwen35 import pair_axes
    from qwen35.engine import _axis
    assert pair_axes([2, 1, 3]) == bytes([0, 0, 1, 2, 2, 2]) and pair_axes([2, 1, 3], True) == bytes([0, 1, 2, 0, 2, 2])
    assert pair_axes([11, 11, 10], True)[-2:] == bytes([0, 1]) and pair_axes([]) == b"" and pair_axes([0, 2]) == bytes([1, 1])
    assert _axis(np.array([0, 1], np.int64), 4) == _axis([0, 1], 4) == _axis(np.array([0, 1], np.uint8), 5) == bytes([0, 1])
    for bad in ([0], [0, 1, 2]):
        with pytest.raises(ValueError, match="pairs"):
            _axis(bad, 4)
    with pytest.raises(ValueError):
        _axis([0, 256], 4)
