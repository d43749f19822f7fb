"""pipeline.quant_q4_device and its layer: the reported error is that of the reconstruction over the matrix's own columns,
the result does not go by the unit of the imatrix, and the weights' device is the one that is launched on.  Bounds are
counted as in test_gpu_q4.py."""
import contextlib

import numpy as np
import pytest
import torch

import oracle
from oracle import uq_q4 as O4

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
HALF = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
TINY = {torch.bfloat16: 2.0 ** -133, torch.float16: 2.0 ** -25}
DT = {"bf16": torch.bfloat16, "fp16": torch.float16}


def make(rows, n0, seed):
    rng = np.random.RandomState(seed)
    W = torch.from_numpy(rng.standard_t(4, size=(rows, n0)) * 0.02).cuda()
    return W, torch.from_numpy(np.exp(rng.standard_normal(n0))).cuda()


def restated(W, H, group):
    """sH, codes, E4M3 bytes and the quantized rotated matrix, in numpy from the definition."""
    sH = torch.maximum(H, H.max() * 1e-3).sqrt().cpu().numpy()
    A = W.cpu().numpy() * sH
    codes, e, s = O4.encode(oracle.rht_rows(A), group)
    return sH, A, codes, e, O4.decode(codes, e, s, group)


WIDTHS = [(40, 300, 32), (24, 14336, 256), (64, 96, 128), (130, 1024, 64), (16, 11008, 32), (9, 2560, 64), (7, 33, 64)]


@pytest.mark.parametrize("rows,n0,group", WIDTHS)
def test_error_sums_are_those_of_the_reconstruction(rows, n0, group):
    """err = [sum (A - Ah)^2, sum A^2] over the n0 columns, as of the other recipes: what the rotated error puts into the
    padding reaches no output."""
    from ultraquant_b200 import pipeline
    W, H = make(rows, n0, n0)
    layer = pipeline.quant_q4_device(W, H, group)
    sH, A, codes, e, Xq = restated(W, H, group)
    assert np.array_equal(layer.w.codes.cpu().numpy(), codes) and np.array_equal(layer.w.scales.view(torch.uint8).cpu().numpy(), e)
    Ah = oracle.irht_rows(Xq, n0)
    want = ((A - Ah) ** 2).sum() / (A ** 2).sum()
    assert abs(layer.wnmse - want) <= 1e-12
    assert abs(layer.err[1].item() / (A ** 2).sum() - 1) <= 1e-12
    # What() is Ah / sH, both in float32: times sH off by at most 2^-23 of Ah's size
    d = A - layer.What().double().cpu().numpy() * sH
    slack = 4 * U * np.linalg.norm(Ah) * (np.linalg.norm(A - Ah) + U * np.linalg.norm(Ah)) / (A ** 2).sum()
    assert abs((d ** 2).sum() / (A ** 2).sum() - layer.wnmse) <= slack + 1e-12


def test_error_of_an_empty_matrix_is_zero():
    from ultraquant_b200 import pipeline
    layer = pipeline.quant_q4_device(torch.zeros(0, 96, device="cuda"), torch.ones(96, device="cuda"), 32)
    assert torch.equal(layer.err, torch.zeros(2, dtype=torch.float64, device="cuda")) and layer.What().shape == (0, 96)
    assert layer(torch.zeros(3, 96, device="cuda", dtype=torch.bfloat16)).shape == (3, 0)


def check_layer(layer, W, H, x, dy, group):
    """y, its gradient and What() against the recipe in 64 bits."""
    dt = x.dtype
    sHn, A, codes, e, Xq = restated(W, H, group)
    assert np.array_equal(layer.w.codes.cpu().numpy(), codes) and np.array_equal(layer.w.scales.view(torch.uint8).cpu().numpy(), e)
    n0, n, sH, Q = W.shape[1], Xq.shape[1], torch.from_numpy(sHn).cuda(), torch.from_numpy(Xq).cuda()
    Wh = oracle.irht_rows(Xq, n0) / sHn
    assert np.abs(layer.What().double().cpu().numpy() - Wh).max() <= 2.0 ** -23 * np.abs(Wh).max()
    x = x.detach().requires_grad_()
    y = layer(x)
    (dx,) = torch.autograd.grad(y, x, dy)
    # rotated activations: a float32 transform (log2 n + 6 roundings of values of at most the row's length), one rounding to
    # dt; a subnormal one is half a step of the type at the size that the layer gives them
    xr = torch.from_numpy(oracle.rht_rows((x.detach().double() / sH).cpu().numpy())).cuda()
    unit = (layer.rotate(x.detach()).double().norm() / xr.norm()).item()
    dxr = HALF[dt] * xr.abs() + (np.log2(n) + 6) * 2 * U * xr.norm(dim=1, keepdim=True) + TINY[dt] / unit
    bound = dxr @ Q.abs().T + 2 * (n + 2) * U * ((xr.abs() + dxr) @ Q.abs().T)
    exact = xr @ Q.T
    off = (y.detach().double() - exact).abs()
    assert (off <= bound * (1 + HALF[dt]) + HALF[dt] * exact.abs() + TINY[dt]).all(), (off / exact.abs().mean()).max()
    g = dy.double() @ Q
    dg = HALF[dt] * g.abs() + 2 * (W.shape[0] + 2) * U * (dy.double().abs() @ Q.abs()) + TINY[dt] * unit
    back = torch.from_numpy(oracle.irht_rows(g.cpu().numpy(), n0)).cuda() / sH
    tol = (dg.norm(dim=1, keepdim=True) + (np.log2(n) + 6) * 2 * U * g.norm(dim=1, keepdim=True)) / sH
    assert ((dx.double() - back).abs() <= tol * 1.001 + HALF[dt] * (back.abs() + tol) + TINY[dt]).all()
    return y.detach(), dx


def acts(T, n, dt, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randn(T, n, generator=g, device="cuda").to(dt)


@pytest.mark.parametrize("dt", ["bf16", "fp16"])
@pytest.mark.parametrize("rows,n0,group,T", [(40, 300, 32, 5), (24, 14336, 256, 3), (64, 96, 128, 33), (130, 1024, 64, 40)])
def test_layer_values_and_gradient(rows, n0, group, T, dt):
    from ultraquant_b200 import pipeline
    W, H = make(rows, n0, n0)
    layer = pipeline.quant_q4_device(W, H, group)
    check_layer(layer, W, H, acts(T, n0, DT[dt], 1), acts(T, rows, DT[dt], 2), group)


@pytest.mark.parametrize("dt", ["bf16", "fp16"])
@pytest.mark.parametrize("n0", [256, 300])
def test_layer_does_not_go_by_the_unit_of_the_imatrix(n0, dt):
    """The whitening and its inverse cancel: a factor on H changes nothing.  By a power of 4 the bits stay the same."""
    from ultraquant_b200 import pipeline
    W, H = make(48, n0, 7)
    x, dy = acts(9, n0, DT[dt], 3), acts(9, 48, DT[dt], 4)
    base = pipeline.quant_q4_device(W, H, 32)
    y0, dx0 = check_layer(base, W, H, x, dy, 32)
    for unit in (4.0 ** -100, 4.0 ** -17, 4.0 ** -3, 4.0 ** 9, 4.0 ** 40, 4.0 ** 100):
        layer = pipeline.quant_q4_device(W, H * unit, 32)
        y = layer(x.clone().requires_grad_())
        assert torch.equal(y.detach(), y0), unit
        xg = x.clone().requires_grad_()
        assert torch.equal(torch.autograd.grad(layer(xg), xg, dy)[0], dx0), unit
        assert torch.equal(layer.What(), base.What()) and layer.wnmse == base.wnmse
        assert torch.equal(layer.err, base.err * unit)
    for unit in (1e-60, 1e-10, 3e-4, 7.0, 1e12, 1e60):
        check_layer(pipeline.quant_q4_device(W, H * unit, 32), W, H * unit, x, dy, 32)


def test_layer_launches_with_the_weights_device_current(monkeypatch):
    """With another device current each launch is made inside torch.cuda.device(the weights' device): seen from a device
    number that is said to be another one."""
    from ultraquant_b200 import _lib, pipeline
    real = torch.cuda.device
    inside = []

    class Spy(real):
        def __enter__(self):
            inside.append(self.idx)
            return super().__enter__()

        def __exit__(self, *a):
            inside.pop()
            return super().__exit__(*a)

    lib, met = _lib.load(), set()

    class Watched:
        def __getattr__(self, name):
            fn = getattr(lib, name)
            if name in ("uq_fwht", "uq_rht_rows", "uq_irht_rows", "uq_wnmse_sums", "uq_device_errors"):
                def call(*a):
                    met.add(name)
                    assert inside and inside[-1] == 0, f"{name} outside the weights' device"
                    return fn(*a)
                return call
            return fn

    W, H = make(8, 96, 1)
    x = acts(3, 96, torch.bfloat16, 1).requires_grad_()
    with contextlib.ExitStack() as stack:
        m = stack.enter_context(pytest.MonkeyPatch.context())
        m.setattr(torch.cuda, "current_device", lambda: inside[-1] if inside else 1)
        m.setattr(torch.cuda, "device", Spy)
        m.setattr(_lib, "load", lambda *a: Watched())
        layer = pipeline.quant_q4_device(W, H, 32)
        y = layer(x)
        layer.rotate(x.detach())
        layer.What()
        torch.autograd.grad(y, x, torch.ones_like(y))
    assert met == {"uq_fwht", "uq_rht_rows", "uq_irht_rows", "uq_wnmse_sums", "uq_device_errors"}
