"""Calls of the 4-bit cache's entry points that are more than one launch can have: HIP counts a launch's threads in
32 bits, 2^24 - 1 blocks of 256. On the CPU, with the host source and the stub of tests/test_kv4_refusals.py."""
import ctypes as C

import numpy as np

from test_kv4_refusals import ARG, heads, lib  # noqa: F401


def test_attention_of_many_rows(lib):  # noqa: F811
    from qwen35.engine import _VIEW
    e, c = C.c_void_p(lib.stub_engine()), C.c_void_p()
    assert lib.q35_kv4_alloc(e, 1, 1, 4096, 1, 64, C.byref(c)) == 0
    full, z = np.array([4096], np.int32), np.zeros(300, np.int32)
    assert lib.q35_kv4_set_len(e, c, None, full.ctypes.data, 1) == 0

    def call(n, T, hq):
        before = lib.stub_launches(e)
        assert lib.q35_op_attn_kv4(e, c, 0, z.ctypes.data, z.ctypes.data, n, T, hq, _VIEW.pack(1 << 16, 0, 0), None, 1.0, 0, 0,
                                   _VIEW.pack(1 << 17, 64 * hq, 64)) == 0
        return lib.stub_launches(e) - before

    assert call(256, 4096, 64) == 1 and call(300, 4096, 64) == 2          # 2^13 blocks a sequence
    assert call(256, 4096, 1024) == 3                                     # 2^17: 127 sequences a launch
    assert call(1, 4096, 1024) == 1
    assert lib.q35_kv4_free(e, c) == 0


def test_heads_of_many_rows(lib):  # noqa: F811
    e, z = C.c_void_p(lib.stub_engine()), np.zeros(300, np.int32)
    h = heads(q=(0, 0, 0), q_out=(0, 0, 0), q_norm=None, v=(0, 0, 0), k=(1 << 16, 0, 64), k_out=(1 << 17, 128, 64))
    most = 4 * (2 ** 24 - 1)                       # rows of a launch

    def call(n, T):
        before = lib.stub_launches(e)
        rc = lib.q35_op_qk_norm_rope(e, h, 2, 64, z.ctypes.data, n, T)
        return rc or lib.stub_launches(e) - before

    assert call(300, 1000) == 2 and call(1, most) == 1 and call(2, most // 2) == 1
    assert call(2, most // 2 + 1) == 2 and call(256, 2 ** 22) == 18            # 15 sequences a launch
    assert call(1, most + 1) == ARG and b"row count" in lib.q35_last_error()
