"""The product in eight bits where its tiles take it, on an MI355X, against the definition in 64 bits: many rows, outputs of
16 bits."""
import pytest

from test_gpu_e4m3_product import run

pytestmark = pytest.mark.gpu


def test_wide_tiles_past_the_last_scales(tk):
    """Tiles of 256 x 256 whose second half has no outputs and no scales: 1100 outputs are nine blocks of 128."""
    run(tk, 13100, 272, 1100, "bf16", "bf16")
