"""What a host copy of e4m3 weights is made from: bytes and their blocks' scales. Nothing here needs a GPU."""
import numpy as np
import pytest

import telmo_amd


@pytest.mark.parametrize("values", [np.ones((200, 300), np.float32), np.ones((200, 300), np.int8), np.ones((200, 300), np.int64),
                                    np.ones((200, 300)), np.ones(200 * 300, np.uint8), np.ones((200, 300, 1), np.uint8), [[1.5, 2.5]]])
def test_values_are_bytes(values):
    """Numbers are not codes: 1.0 is 0x38. They were converted to whole numbers without a word."""
    with pytest.raises(TypeError):
        telmo_amd.E4m3Weights.from_parts(None, values, np.ones((2, 3), np.float32))


@pytest.mark.parametrize("shape", [(3, 2), (2, 2), (2, 4), (6,), (1, 3), ()])
def test_scales_are_one_for_each_block(shape):
    with pytest.raises(ValueError):
        telmo_amd.E4m3Weights.from_parts(None, np.zeros((200, 300), np.uint8), np.ones(shape, np.float32))
