"""Argument checks of the 4-bit cache's entry points and of the draft verification, on the CPU: the host
source (q35_kv4.cpp) built against tests/kv4_host_stub.cpp, which counts launches instead of making
them. A refused call has its status and text, launches nothing and leaves the lanes' lengths; the
call beside it that is allowed goes through."""
import ctypes as C
import shutil
import subprocess
from pathlib import Path

import numpy as np
import pytest

REPO = Path(__file__).resolve().parents[1]
ARG, CAP, STATE = -1, -2, -4


@pytest.fixture(scope="module")
def lib(tmp_path_factory):
    cxx = shutil.which("g++") or "/opt/rocm/llvm/bin/clang++"
    so = tmp_path_factory.mktemp("kv4") / "libkv4host.so"
    subprocess.run([cxx, "-std=c++17", "-O1", "-shared", "-fPIC", "-Bsymbolic", "-D__HIP_PLATFORM_AMD__=1", "-I/opt/rocm/include",
                    "-I", str(REPO / "qwen3.5-0.8b_amd" / "csrc"), "-I", str(REPO / "include"),
                    str(REPO / "tests" / "kv4_host_stub.cpp"),
                    str(REPO / "qwen3.5-0.8b_amd" / "csrc" / "q35_kv4.cpp"), "-o", str(so)], check=True,
                   capture_output=True)
    from qwen35 import engine
    L = C.CDLL(str(so))
    for name in ("alloc", "free", "set_len", "len", "write", "read"):
        f = getattr(L, "q35_kv4_" + name)
        f.argtypes, f.restype = engine._SIGS["q35_kv4_" + name]
    for name in ("q35_op_qk_norm_rope", "q35_op_kv4_append", "q35_op_attn_kv4", "q35_op_draft_verify"):
        f = getattr(L, name)
        f.argtypes, f.restype = engine._SIGS[name]
    L.stub_engine.restype = C.c_void_p
    L.stub_launches.argtypes = [C.c_void_p]
    L.q35_last_error.restype = C.c_char_p
    return L


class Bed:
    """A stub engine with a cache of 2 layers x 3 lanes x 100 slots, 2 heads of 64."""

    def __init__(self, lib):
        self.L, self.e, self.c = lib, C.c_void_p(lib.stub_engine()), C.c_void_p()
        assert lib.q35_kv4_alloc(self.e, 2, 3, 100, 2, 64, C.byref(self.c)) == 0

    def lengths(self, layer=0):
        out, v = [], C.c_int32()
        for l in range(3):
            assert self.L.q35_kv4_len(self.e, self.c, layer, l, C.byref(v)) == 0
            out.append(v.value)
        return out

    def set_len(self, lanes, lens):
        a, b = (np.array(x, np.int32) for x in (lanes, lens))
        return self.L.q35_kv4_set_len(self.e, self.c, a.ctypes.data, b.ctypes.data, a.size)

    def refused(self, code, rc, text):
        said = self.L.q35_last_error().decode()
        assert rc == code, (rc, said)
        assert text in said, said


@pytest.fixture
def bed(lib):
    return Bed(lib)


def heads(**kw):
    from qwen35.engine import _HEADS
    h = dict(q_heads=4, rot_dim=32, theta=1e7, eps=1e-6, q_norm=4096, k_norm=4096)
    v = dict(q=(1 << 16, 512, 64), k=(2 << 16, 512, 64), v=(3 << 16, 512, 64), q_out=(4 << 16, 256, 64), k_out=(0, 0, 0),
             v_out=(0, 0, 0))
    for n, x in kw.items():
        (v if n in v else h)[n] = x
    return _HEADS.pack(*[x or 0 for x in h.values()], *[y for x in v.values() for y in x])


def append(bed, lanes, pos, T=1, layer=0, **kw):
    la, p, h = np.array(lanes, np.int32), np.array(pos, np.int32), heads(**kw)
    return bed.L.q35_op_kv4_append(bed.e, bed.c, layer, la.ctypes.data, p.ctypes.data, p.size, T, h)


def test_append(bed):
    assert append(bed, [0, 2], [0, 0], T=5) == 0
    assert bed.lengths() == [5, 0, 5] and bed.lengths(1) == [0, 0, 0]
    assert append(bed, [0], [3]) == 0 and bed.lengths() == [4, 0, 5]      # the rows behind it are dropped
    n = bed.L.stub_launches(bed.e)
    assert n == 2
    far = 1 << 16
    for code, text, args, kw in [
            (ARG, "twice", ([1, 1], [0, 0]), {}), (ARG, "lane out of range", ([3], [0]), {}),
            (ARG, "lane out of range", ([-1], [0]), {}), (STATE, "gap", ([1], [1]), {}), (CAP, "capacity", ([0], [-1]), {}),
            (CAP, "capacity", ([0], [4]), {"T": 97}), (CAP, "capacity", ([0], [0]), {"T": 2 ** 31 - 1}),
            (CAP, "capacity", ([0], [2 ** 31 - 1]), {}), (ARG, "row count", ([0], [4]), {"T": 0}),
            (ARG, "layer", ([0], [4]), {"layer": 2}), (ARG, "layer", ([0], [4]), {"layer": -1}),
            (ARG, "rot_dim", ([0], [4]), {"rot_dim": 33}), (ARG, "rot_dim", ([0], [4]), {"rot_dim": 66}),
            (ARG, "rot_dim", ([0], [4]), {"rot_dim": -2}), (ARG, "theta", ([0], [4]), {"theta": 0.0}),
            (ARG, "theta", ([0], [4]), {"theta": float("nan")}), (ARG, "eps", ([0], [4]), {"eps": -1.0}),
            (ARG, "eps", ([0], [4]), {"eps": float("inf")}), (ARG, "norm", ([0], [4]), {"k_norm": None}),
            (ARG, "norm", ([0], [4]), {"q_norm": None}), (ARG, "aligned", ([0], [4]), {"k_norm": 4100}),
            (ARG, "k: null", ([0], [4]), {"k": (0, 512, 64)}), (ARG, "v: null", ([0], [4]), {"v": (0, 512, 64)}),
            (ARG, "k: the pointer", ([0], [4]), {"k": (far + 8, 512, 64)}),
            (ARG, "v: the pointer", ([0], [4]), {"v": (far, 516, 64)}),
            (ARG, "q: the pointer", ([0], [4]), {"q": (far, 512, 60)}),
            (ARG, "negative", ([0], [4]), {"q": (far, -512, 64)}), (ARG, "go together", ([0], [4]), {"q_out": (0, 0, 0)}),
            (ARG, "go together", ([0], [4]), {"q": (0, 0, 0)}), (ARG, "head count", ([0], [4]), {"q_heads": 1025}),
            (ARG, "without q_heads", ([0], [4]), {"q_heads": 0}),
            (ARG, "q_out: rows or heads overlap", ([0], [4]), {"T": 2, "q_out": (far, 128, 64)}),
            (ARG, "q_out: rows or heads overlap", ([0], [4]), {"q_out": (far, 512, 56)}),
            (ARG, "k_out: rows or heads overlap", ([0], [4]), {"T": 2, "k_out": (far, 0, 64)})]:
        bed.refused(code, append(bed, *args, **kw), text)
    assert bed.L.stub_launches(bed.e) == n and bed.lengths() == [4, 0, 5]
    # the neighbours of the refused calls
    assert append(bed, [0], [4], T=96, rot_dim=0, theta=0.0) == 0 and bed.lengths()[0] == 100
    assert append(bed, [1], [0], q=(0, 0, 0), q_out=(0, 0, 0), q_heads=0, q_norm=None) == 0
    assert append(bed, [2], [5], T=2, q_out=(far, 64, 128)) == 0       # heads outside, rows inside


def test_sequences_past_one_launch(lib):
    e, c = C.c_void_p(lib.stub_engine()), C.c_void_p()
    assert lib.q35_kv4_alloc(e, 1, 600, 8, 1, 64, C.byref(c)) == 0
    p, h = np.zeros(600, np.int32), heads()
    assert lib.q35_op_kv4_append(e, c, 0, None, p.ctypes.data, 600, 2, h) == 0
    assert lib.stub_launches(e) == 3
    assert lib.q35_kv4_free(e, c) == 0


def test_norm_rope(bed):
    p = np.array([0, 2 ** 31 - 4], np.int32)
    none = dict(v=(0, 0, 0), k_out=(5 << 16, 128, 64))

    def call(T=1, kv=2, dim=64, n=2, **kw):
        h = heads(**{**none, **kw})
        return bed.L.q35_op_qk_norm_rope(bed.e, h, kv, dim, p.ctypes.data, n, T)

    assert call() == 0 and call(T=3) == 0
    bed.refused(ARG, call(T=4), "position out of range")
    bed.refused(ARG, call(dim=96), "head_dim")
    bed.refused(ARG, call(kv=0), "head count")
    bed.refused(ARG, call(n=0), "sequence")
    bed.refused(ARG, call(v=(3 << 16, 512, 64)), "v has no norm")
    bed.refused(ARG, call(k_out=(0, 0, 0)), "k_out: null")
    bed.refused(ARG, call(T=2 ** 30), "row count")
    assert bed.L.q35_op_qk_norm_rope(None, None, 2, 64, None, 1, 1) == ARG


def test_attention(bed):
    from qwen35.engine import _VIEW
    assert bed.set_len([0, 1, 2], [10, 0, 100]) == 0
    q0, out0 = (1 << 16, 512, 64), (2 << 16, 256, 64)

    def call(lanes, pos, T=1, layer=0, hq=4, q=q0, out=out0, gate=None, scale=0.125, window=0, sinks=0):
        la, p = np.array(lanes, np.int32), np.array(pos, np.int32)
        return bed.L.q35_op_attn_kv4(bed.e, bed.c, layer, la.ctypes.data, p.ctypes.data, p.size, T, hq, _VIEW.pack(*q),
                                     _VIEW.pack(*gate) if gate else None, scale, window, sinks, _VIEW.pack(*out))

    assert call([0, 0, 2], [9, 0, 99]) == 0                  # a lane may occur twice
    assert call([0], [7], T=3, window=1, sinks=5) == 0
    n = bed.L.stub_launches(bed.e)
    for code, text, args, kw in [
            (STATE, "does not hold", ([0], [10]), {}), (STATE, "does not hold", ([0], [8]), {"T": 3}),
            (STATE, "does not hold", ([1], [0]), {}), (CAP, "capacity", ([2], [100]), {}), (CAP, "capacity", ([2], [-1]), {}),
            (ARG, "lane out of range", ([3], [0]), {}), (ARG, "multiple", ([0], [0]), {"hq": 3}),
            (ARG, "multiple", ([0], [0]), {"hq": 0}), (ARG, "negative", ([0], [0]), {"window": -1}),
            (ARG, "sinks go with", ([0], [0]), {"sinks": 4}), (ARG, "negative", ([0], [0]), {"window": 4, "sinks": -4}),
            (ARG, "scale", ([0], [0]), {"scale": float("inf")}), (ARG, "q: null", ([0], [0]), {"q": (0, 512, 64)}),
            (ARG, "out: null", ([0], [0]), {"out": (0, 512, 64)}), (ARG, "gate: the pointer", ([0], [0]), {"gate": (8, 512, 64)}),
            (ARG, "out: rows or heads overlap", ([0], [0]), {"T": 2, "out": (1 << 16, 64, 64)}),
            (ARG, "layer", ([0], [0]), {"layer": 2})]:
        bed.refused(code, call(*args, **kw), text)
    assert bed.L.stub_launches(bed.e) == n
    other = C.c_void_p(bed.L.stub_engine())
    assert bed.L.q35_op_attn_kv4(other, bed.c, 0, None, np.zeros(1, np.int32).ctypes.data, 1, 1, 4, _VIEW.pack(*q0), None,
                                 1.0, 0, 0, _VIEW.pack(*out0)) == ARG


def test_cache_shapes_lengths_copies(bed):
    c = C.c_void_p()
    for args, code in [((0, 1, 8, 1, 64), ARG), ((1, 0, 8, 1, 64), ARG), ((1, 1, 0, 1, 64), ARG), ((1, 1, 8, 0, 64), ARG),
                       ((1, 1, 8, 1, 80), ARG), ((1, 65536, 8, 1, 64), ARG), ((1, 1, 4097, 1, 64), CAP)]:
        assert bed.L.q35_kv4_alloc(bed.e, *args, C.byref(c)) == code, args
    assert bed.L.q35_kv4_alloc(None, 1, 1, 8, 1, 64, C.byref(c)) == ARG
    bed.refused(CAP, bed.set_len([0, 1], [5, 101]), "capacity")
    bed.refused(CAP, bed.set_len([0], [-1]), "capacity")
    bed.refused(ARG, bed.set_len([0, 3], [5, 5]), "lane out of range")
    assert bed.lengths() == [0, 0, 0]                        # none of them took part
    assert bed.set_len([1], [40]) == 0 and bed.lengths(0) == bed.lengths(1) == [0, 40, 0]

    def copy(name, lane0, n, slot0, m, layer=0, ptrs=(16, 16, 16, 16)):
        return getattr(bed.L, name)(bed.e, bed.c, layer, lane0, n, slot0, m, *ptrs)

    assert copy("q35_kv4_write", 0, 3, 0, 30) == 0 and bed.lengths() == [30, 40, 30]
    assert copy("q35_kv4_write", 1, 1, 40, 60, layer=1) == 0 and bed.lengths(1) == [0, 100, 0]
    assert copy("q35_kv4_read", 0, 3, 10, 20) == 0
    for code, args, kw in [(STATE, ("q35_kv4_write", 0, 3, 31, 1), {}), (STATE, ("q35_kv4_read", 0, 3, 11, 20), {}),
                           (CAP, ("q35_kv4_write", 1, 1, 40, 61), {}), (CAP, ("q35_kv4_write", 1, 1, -1, 2), {}),
                           (CAP, ("q35_kv4_read", 1, 1, 0, 0), {}), (ARG, ("q35_kv4_read", 2, 2, 0, 1), {}),
                           (ARG, ("q35_kv4_read", -1, 1, 0, 1), {}), (ARG, ("q35_kv4_read", 0, 1, 0, 1), {"layer": 2}),
                           (ARG, ("q35_kv4_read", 0, 1, 0, 1), {"ptrs": (16, 0, 16, 16)})]:
        assert copy(*args, **kw) == code, (args, kw)
    assert bed.lengths() == [30, 40, 30]
    assert bed.L.q35_kv4_free(C.c_void_p(bed.L.stub_engine()), bed.c) == ARG
    assert bed.L.q35_kv4_free(None, bed.c) == 0              # its engine gone
    assert bed.L.q35_kv4_free(bed.e, None) == 0


def test_verify(bed):
    from qwen35.engine import _DRAFTS

    def call(n=4, k=2, vocab=100, acc=16, tok=16, **kw):
        d = dict(logits=16, ld=100, draft_logits=0, draft_ld=100, dtype=0, drafts=16, u=16, temperature=1.0)
        d.update(kw)
        return bed.L.q35_op_draft_verify(bed.e, _DRAFTS.pack(*[x or 0 for x in d.values()]), n, k, vocab, acc, tok)

    assert call() == 0 and call(n=21) == 0 and call(temperature=0.0) == 0 and call(draft_logits=16, dtype=1) == 0
    n = bed.L.stub_launches(bed.e)
    for code, text, kw in [
            (CAP, "max_rows", {"n": 22}), (CAP, "max_rows", {"n": 2 ** 31 - 1}), (CAP, "max_rows", {"n": 0}),
            (ARG, "drafts per lane", {"k": 0}), (ARG, "drafts per lane", {"k": 9, "n": 1}), (ARG, "vocab", {"vocab": 0}),
            (ARG, "vocab", {"vocab": (1 << 20) + 1, "ld": 1 << 21}), (ARG, "stride", {"ld": 99}),
            (ARG, "stride", {"draft_logits": 16, "draft_ld": 99}), (ARG, "dtype", {"dtype": 2}),
            (ARG, "misaligned", {"logits": 18}), (ARG, "misaligned", {"logits": 17, "dtype": 1}),
            (ARG, "misaligned", {"draft_logits": 18}), (ARG, "temperature", {"temperature": -1.0}),
            (ARG, "temperature", {"temperature": float("nan")}), (ARG, "temperature", {"temperature": 1e-4}),
            (ARG, "null", {"logits": None}), (ARG, "null", {"drafts": None}), (ARG, "null", {"u": None}),
            (ARG, "null", {"acc": None}), (ARG, "null", {"tok": None})]:
        bed.refused(code, call(**kw), text)
    assert bed.L.stub_launches(bed.e) == n


def test_lane_and_position_counts_must_match():
    from qwen35.engine import _i32, _lp
    with pytest.raises(ValueError):
        _lp(_i32([0, 1]), _i32([0]))


def test_attention_numbers_past_their_types(lib):
    """Rows past 2^31 in all, and a scale that overflows where the kernel takes it to base 2."""
    from qwen35.engine import _VIEW
    e, c = C.c_void_p(lib.stub_engine()), C.c_void_p()
    assert lib.q35_kv4_alloc(e, 1, 1, 4096, 1, 64, C.byref(c)) == 0
    full = np.array([4096], np.int32)
    assert lib.q35_kv4_set_len(e, c, None, full.ctypes.data, 1) == 0
    z = np.zeros(1 << 20, np.int32)

    def call(n, T, scale):
        return lib.q35_op_attn_kv4(e, c, 0, z.ctypes.data, z.ctypes.data, n, T, 1, _VIEW.pack(1 << 16, 64, 64), None, scale, 0, 0,
                                   _VIEW.pack(1 << 17, 64, 64))

    assert call(1 << 20, 4096, 1.0) == ARG and "row count" in lib.q35_last_error().decode()
    assert call(1 << 19, 4096, 1.0) == ARG
    assert call(1, 4096, 3e38) == ARG and "scale" in lib.q35_last_error().decode()
    assert lib.stub_launches(e) == 0
    assert call(1, 4096, 2e38) == 0 and lib.stub_launches(e) == 1
    assert lib.q35_kv4_free(e, c) == 0
