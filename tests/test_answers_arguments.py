"""Arguments of the answers' operators that the Python side looks over itself, on the CPU."""
import pytest


@pytest.mark.parametrize("dealt", [False, True])
@pytest.mark.parametrize("sections", [[-1], [2, -1, 3], [0, -5]])
@pytest.mark.timeout(20)
def test_pair_axes_of_negative_sections(sections, dealt):
    from qwen35 import pair_axes
    with pytest.raises(ValueError, match="negative"):
        pair_axes(sections, dealt)
