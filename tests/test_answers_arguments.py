"""Arguments of the answers' operators that the Python side looks over itself, on the CPU."""
import numpy as np
import pytest


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
