"""Arguments of the answers' operators that the Python side looks over itself, and the positions that a map of axes has read, on
the CPU."""
import ctypes as C
import shutil
import subprocess
from pathlib import Path

import numpy as np
import pytest

from test_answers_refusals import at
from test_kv4_refusals import REPO, Bed, heads


@pytest.mark.parametrize("dealt", [False, True])
@pytest.mark.parametrize("sections", [[-1], [2, -1, 3], [0, -5]])
@pytest.mark.timeout(20)
def test_pair_axes_of_negative_sections(sections, dealt):
    from qwen35 import pair_axes
    with pytest.raises(ValueError, match="negative"):
        pair_axes(sections, dealt)


@pytest.mark.parametrize("axis", [0, 1, 32, np.int64(32), np.uint8(7)])
@pytest.mark.parametrize("rot_dim", [0, 2, 64])
def test_one_number_is_no_list_of_axes(axis, rot_dim):
    """bytes(32) is 32 zero bytes: every pair on axis 0."""
    from qwen35.engine import _axis
    with pytest.raises(ValueError, match="pairs"):
        _axis(axis, rot_dim)


@pytest.mark.parametrize("lanes", [[], [0], [0, 1, 2], np.zeros(7, np.int32)])
def test_scored_step_with_other_lanes_than_tokens(lanes):
    """The library reads a lane for each token: of a shorter list it would read what lies behind it."""
    from types import SimpleNamespace
    from qwen35 import State
    s = object.__new__(State)
    s.eng, s.h = SimpleNamespace(h=None), None
    with pytest.raises(ValueError, match="lanes"):
        s.decode_step_logprobs([5, 6], lanes)


@pytest.fixture(scope="module")
def stub(tmp_path_factory):
    cxx = shutil.which("g++") or "/opt/rocm/llvm/bin/clang++"
    so, src = tmp_path_factory.mktemp("axes") / "libaxeshost.so", REPO / "qwen3.5-0.8b_amd" / "csrc"
    subprocess.run([cxx, "-std=c++17", "-O1", "-shared", "-fPIC", "-Bsymbolic", "-D__HIP_PLATFORM_AMD__=1", "-I/opt/rocm/include",
                    "-I", str(src), "-I", str(REPO / "include"), str(Path(__file__).parent / "answers_axes_stub.cpp"),
                    str(src / "q35_kv4.cpp"), str(src / "q35_answers.cpp"), "-o", str(so)], check=True, capture_output=True)
    from qwen35 import engine
    L = C.CDLL(str(so))
    for name in ("q35_kv4_alloc", "q35_op_qk_norm_rope_axes"):
        f = getattr(L, name)
        f.argtypes, f.restype = engine._SIGS[name]
    L.stub_engine.restype, L.stub_axis_at.restype = C.c_void_p, C.c_longlong
    return L


@pytest.mark.parametrize("named", [[0], [1], [3], [0, 1], [0, 3], [1, 2], [2, 3], [0, 2, 3], [1, 3], [0, 1, 2, 3]])
@pytest.mark.parametrize("step", [0, 1, 4096, 2 ** 31 + 3])
def test_positions_of_other_axes_are_not_read(stub, named, step):
    """A caller need not have positions on axes that no pair has: what is read up to the largest is a named one's."""
    axis = bytes(named[i % len(named)] for i in range(16))
    h = heads(v=(0, 0, 0), k_out=(5 << 16, 128, 64))
    assert stub.q35_op_qk_norm_rope_axes(Bed(stub).e, h, 2, 64, at(axis=step), axis, 5) == 0
    assert stub.stub_axes() == max(named) + 1
    for a in range(max(named) + 1):
        assert stub.stub_axis_at(a) in ([a * step] if a in named else [b * step for b in named])
