"""The example layer: trained through the softmax differential gradients, served from the 4-bit cache."""
import os
import sys

import pytest

pytestmark = pytest.mark.gpu


def test_layer_trains_and_serves():
    sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples"))
    import differential_layer
    losses, drift, lengths, expected = differential_layer.main(steps=15, decode_steps=40)
    assert losses[-1] < 0.9 * losses[0], losses
    # a code's step is 1 / 7 of its group's largest element, an error of about a tenth of a key or value, averaged
    # over the tokens a query attends to and, for the first requests, over few of them
    assert 0.0 < drift < 0.15, drift
    assert lengths == expected
