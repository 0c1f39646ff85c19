"""The gradient of a layer norm's bias without a weight: what the Python layer refuses, without a GPU."""
import pytest

import dpnp_amd.tensor as dpt
from tests.test_row_operators_cpu import fake


def test_refusals():
    x, stat = fake((4, 8)), fake((4,))
    with pytest.raises(ValueError, match="need weight"):
        dpt.layer_norm_grad(x, x, stat, stat, out=(x, fake((8,)), fake((8,))))
    with pytest.raises(ValueError, match="shape"):
        dpt.layer_norm_grad(x, x, stat, stat, out=(x, None, fake((9,))))
    with pytest.raises(ValueError, match="type"):
        dpt.layer_norm_grad(x, x, stat, stat, out=(x, None, fake((8,), "f8")))
    with pytest.raises(ValueError, match="type"):
        dpt.layer_norm_grad(fake((4, 8), "f8"), fake((4, 8), "f8"), stat, stat, out=(fake((4, 8), "f8"), None, fake((8,))))
    with pytest.raises(TypeError, match="usm_ndarray"):
        dpt.layer_norm_grad(x, x, stat, stat, out=(x, None, [0.0] * 8))
