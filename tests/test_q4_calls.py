"""The Python layer of the 4-bit operators without a GPU."""
import pytest
import torch


@pytest.mark.parametrize("shape,rows", [((0,), 1), ((3, 0), 3), ((2, 3, 0), 6), ((2, 0, 3, 0), 0), ((2, 3, 5), 6), ((5,), 1), ((0, 4, 8), 0)])
def test_rows_of_any_shape(shape, rows):
    """(..., n) as rows, with no columns too: the gradient of a product with a matrix that has no rows."""
    from ultraquant_b200 import q4
    assert tuple(q4._rows(torch.ones(shape)).shape) == (rows, shape[-1])
