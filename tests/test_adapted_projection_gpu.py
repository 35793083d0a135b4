"""The norm, a quantized product, adapters and the router with groups together, forward and back (examples/adapted_projection.py)."""
import os
import sys

import pytest

sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples"))

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("tokens,hidden,outputs,rank,adapters", [(384, 1024, 1536, 16, 6), (1, 512, 256, 8, 1), (1300, 256, 384, 32, 9), (37, 1040, 208, 24, 4)])
def test_layer(gpu, tokens, hidden, outputs, rank, adapters):
    """Against 32-bit torch from the library's own 8-bit values and choices.  What is off: results and the norm that the adapters
    read are rounded to bf16 (2^-8 of a value, a step and half of one on the way back: below 2^-6 of the largest), weights of the
    router and the sums in 32 bits."""
    import adapted_projection
    difference, layer = adapted_projection.run(tokens, hidden, outputs, rank, adapters)
    for name in ("sum", "y", "dx", "dgamma"):
        assert difference[name] < 2.0 ** -6, (name, difference)
    assert difference["w"] < 2.0 ** -18
