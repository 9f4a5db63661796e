"""What the dense layer and the optimiser ask of their callers, without a GPU."""
import pytest

from compressgnn_b200 import _lib


@pytest.mark.parametrize("dtype, packed", [(0, 6), (2, 2), (3, 2)])
def test_a_weight_gradient_of_one_split_has_no_copy_in_the_scratch(dtype, packed):
    """There are more tiles than multiprocessors: a split writes the gradient itself, and the scratch holds the weight's image (six bytes
    an element in fp32) and a sum for each column."""
    room = _lib.lib().cgnn_linear_backward_scratch_bytes(dtype, 4000, 4096, 4096)
    assert packed * 4096 * 4096 <= room <= packed * 4096 * 4096 + (1 << 16)
