"""The kernel's input gradient with few columns in many dimensions."""
import pytest

import test_features_gpu as base

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("leaf", ["rbf", "m12", "m32", "m52", "rq"])
@pytest.mark.parametrize("ard", [False, True])
@pytest.mark.parametrize("n,d,t", [(200, 33, 1), (300, 33, 4), (300, 64, 1), (150, 64, 4), (257, 64, 3),
                                   (260, 33, 17), (130, 64, 20), (300, 48, 19), (300, 32, 2), (300, 32, 18)])
def test_input_gradient_of_many_dimensions(gpb_lib, leaf, n, d, t, ard):
    """Up to 4 columns, alone or left over from chunks of 16, in 32 to 64 dimensions."""
    base.test_input_gradient_formula(gpb_lib, leaf, n, d, t, ard)
