"""Calls of the 4-bit operators at their edges."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def q4():
    from ultraquant_b200 import q4 as m
    return m


@pytest.fixture(autouse=True)
def no_device_errors():
    yield
    q4().check_errors()


# ---- nothing to do ---------------------------------------------------------------------------------------------

@pytest.mark.parametrize("shape", [(64,), (3, 64), (2, 3, 64), (2, 0, 3, 64), (0, 64)])
def test_gradients_of_a_matrix_without_rows(shape):
    m = q4()
    none = m.enc_q4(torch.zeros(0, 64), 32)
    x = torch.ones(shape, device="cuda", dtype=torch.bfloat16, requires_grad=True)
    s = none.group_scales().requires_grad_()
    y = m.linear(x, none, s)
    assert y.shape == (*shape[:-1], 0)
    dx, dc = torch.autograd.grad(y, (x, s), torch.ones_like(y))
    assert torch.equal(dx, torch.zeros_like(x)) and dc.shape == (0, 2)
