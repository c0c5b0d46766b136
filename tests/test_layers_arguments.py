"""CPU tests of the learned layers' arguments that Python checks."""
import pytest

import af2cuda


def test_needs_that_name_no_gradient():
    """Refused before anything else is looked at."""
    dense, gated = af2cuda.encode_dense_backward_tensors, af2cuda.encode_gated_transition_backward_tensors
    for need in (["dx"], ("x", "weights"), "w", ["x", "bias"], [None]):
        with pytest.raises(af2cuda.RangeError, match="need names"):
            dense(None, None, None, None, need=need)
    for need in (["weight"], "gate", ["x", "outputweight"], {"gateWeight": 1, "bias": 2}):
        with pytest.raises(af2cuda.RangeError, match="need names"):
            gated(None, None, None, None, saved=None, need=need)
