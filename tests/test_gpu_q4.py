"""4-bit weight operators on the GPU, each against its formula in 64 bits.

Tolerances are counted: products of bfloat16 / float16 activations with e q are exact, a float32 sum of n terms is off by
at most n roundings of 2^-24 of the sum of sizes (taken twice: a matrix instruction may cut instead of round), and the
result rounds by half a step of its type."""
import numpy as np
import pytest
import torch

from oracle import uq_q4 as O4

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
HALF = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: U}
TINY = {torch.bfloat16: 2.0 ** -133, torch.float16: 2.0 ** -25, torch.float32: 2.0 ** -149}     # half a subnormal step
DT = {"bf16": torch.bfloat16, "fp16": torch.float16}


def q4():
    from ultraquant_b200 import q4 as m
    return m


@pytest.fixture(autouse=True)
def no_device_errors():
    """No test leaves a wait that gave up, or another error that it did not ask for."""
    yield
    q4().check_errors()


def make(shape, group, seed, s=None):
    """Q4 of random codes and signed scales, and its parts in float64."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    *lead, N, K = shape
    codes = torch.randint(0, 256, (*lead, N, K // 2), generator=g, device="cuda").to(torch.uint8)
    e = torch.randn(*lead, N, K // group, generator=g, device="cuda") * 3
    e = e.to(torch.float8_e4m3fn)
    sc = torch.rand(tuple(lead), generator=g, device="cuda") * 0.01 + 0.01 if s is None else torch.full(tuple(lead), s, device="cuda")
    w = q4().Q4(codes, e, sc)
    q = torch.from_numpy(O4.unpack(codes.cpu().numpy())).double().cuda()
    c = e.double() * sc.double().reshape(*lead, 1, 1)
    return w, q, c, q * c.repeat_interleave(group, -1)


def close(got, exact, size, n, dt=None):
    """|got - exact| <= 2 n U size + half a step of the result."""
    dt = dt or got.dtype
    got, exact, size = got.double(), exact.double(), size.double()
    tol = 2 * (n + 2) * U * size + HALF[dt] * (exact.abs() + 2 * (n + 2) * U * size) + TINY[dt]
    off = (got - exact).abs()
    worst = (off - tol).max().item() if off.numel() else -1.0
    assert not torch.isnan(got).any() or torch.isnan(exact).any()
    assert worst <= 0, f"off by {off.max().item():.3g}, {worst:.3g} more than allowed"


def acts(T, n, dt, seed):
    g = torch.Generator(device="cuda").manual_seed(1000 + seed)
    return torch.randn(T, n, generator=g, device="cuda").to(dt)


# ---- codec -----------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("dtype", [torch.float32, torch.float64, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("N,K,group", [(1, 32, 32), (7, 256, 256), (33, 96, 32), (300, 1024, 64), (5, 4096 + 128, 128)])
def test_encode_is_the_restated_one(dtype, N, K, group):
    g = torch.Generator().manual_seed(N * K)
    W = torch.randn(N, K, generator=g, dtype=torch.float64) * torch.exp(2 * torch.randn(N, 1, generator=g, dtype=torch.float64))
    W[0, : group // 2] = 0
    if N > 5:
        W[1] = 0
        W[2] = torch.round(W[2] * 2) / 2                    # ties between steps and between sizes
        W[3] = -W[3].abs()
        W[4] *= 1e-4                                        # scales below the smallest E4M3
    W = W.to(dtype)
    w = q4().enc_q4(W.cuda(), group)
    codes, e, s = O4.encode(W.float().numpy() if dtype != torch.float64 else W.numpy(), group)
    assert w.scale.item() == s
    assert np.array_equal(w.scales.view(torch.uint8).cpu().numpy(), e)
    assert np.array_equal(w.codes.cpu().numpy(), codes)
    d = q4().deq_q4(w)
    ref = O4.decode(codes, e, s, group)
    assert np.array_equal(d.double().cpu().numpy(), ref)
    for dt in (torch.bfloat16, torch.float16):
        assert torch.equal(q4().deq_q4(w, dt), torch.from_numpy(ref).float().cuda().to(dt))


def test_encode_ties_borders_and_extremes():
    rows = []
    base = np.zeros(32, np.float32)
    for v in (1e-45, 1e-39, 2.0 ** -126, 2.0 ** -100, 1.0, 448.0, 3e38):
        r = base.copy()
        r[5], r[9] = v, -v                                  # the first of the largest decides the sign
        rows.append(r)
    r = np.linspace(-8, 8, 33, dtype=np.float32)[:32]       # every half step
    rows += [r, np.nextafter(r, np.float32(100)), np.nextafter(r, np.float32(-100)), r * np.float32(1.0625)]
    W = np.stack(rows)
    for sub in (W, W[:6], W[:2], W[7:], W[1:2]):
        w = q4().enc_q4(sub, 32)
        codes, e, s = O4.encode(sub, 32)
        assert w.scale.item() == s and np.array_equal(w.scales.view(torch.uint8).cpu().numpy(), e)
        assert np.array_equal(w.codes.cpu().numpy(), codes)


def test_encode_experts_each_with_its_scale_and_non_finite_groups():
    g = torch.Generator().manual_seed(3)
    W = torch.randn(3, 11, 128, generator=g) * torch.tensor([1.0, 1e-3, 50.0])[:, None, None]
    W[1, 2, 40] = float("nan")
    W[2, 5, 127] = -float("inf")
    w = q4().enc_q4(W, 32)
    for i in range(3):
        codes, e, s = O4.encode(W[i].numpy(), 32)
        assert w.scale[i].item() == s
        assert np.array_equal(w.scales[i].view(torch.uint8).cpu().numpy(), e)
        assert np.array_equal(w.codes[i].cpu().numpy(), codes)
    d = q4().deq_q4(w)
    assert torch.isnan(d[1, 2, 32:64]).all() and torch.isnan(d[2, 5, 96:]).all() and int(torch.isnan(d).sum()) == 64
    empty = q4().enc_q4(torch.zeros(0, 64), 32)
    assert empty.shape == (0, 64) and q4().deq_q4(empty).shape == (0, 64)


def test_round_scales():
    w, q, c, _ = make((2, 40, 256), 64, 5)
    g = torch.Generator(device="cuda").manual_seed(8)
    t = torch.randn(2, 40, 4, generator=g, device="cuda") * torch.tensor([1.0, 1e-5], device="cuda")[:, None, None]
    t[0, 0, 0], t[0, 1, 1], t[1, 0, 0], t[1, 3, 3] = 0.0, 1e-30, float("inf"), -1e-40
    r = q4().round_scales(w, t)
    assert r.codes.data_ptr() == w.codes.data_ptr()
    for i in range(2):
        e, s = O4.round_scales(t[i].cpu().numpy())
        assert r.scale[i].item() == s and np.array_equal(r.scales[i].view(torch.uint8).cpu().numpy(), e)
    # scales in the stored form (a power of two times E4M3) are a fixed point
    fine = torch.where(torch.isfinite(r.group_scales()), r.group_scales(), 0.0)
    assert torch.equal(q4().round_scales(w, fine).group_scales(), fine)


# ---- products --------------------------------------------------------------------------------------------------

SIZES = [(1, 1, 32, 32), (1, 130, 64, 64), (2, 5, 96, 32), (3, 257, 1024, 128), (7, 64, 4128, 32), (8, 300, 512, 256), (9, 129, 288, 32),
         (16, 1000, 320, 64), (17, 8, 2048, 256), (31, 384, 160, 32), (33, 77, 96, 32), (64, 128, 256, 128), (65, 250, 1056, 32),
         (129, 136, 640, 64), (256, 256, 256, 256), (300, 520, 544, 32), (515, 1100, 1280, 256), (1, 4096, 14336, 32), (5, 1024, 28672, 256)]


@pytest.mark.parametrize("dt", ["bf16", "fp16"])
@pytest.mark.parametrize("T,N,K,group", SIZES)
def test_linear_values(T, N, K, group, dt):
    w, q, c, wd = make((N, K), group, T + N + K)
    x = acts(T, K, DT[dt], T)
    y = q4().linear(x, w)
    assert y.shape == (T, N) and y.dtype == DT[dt]
    xd = x.double()
    close(y, xd @ wd.T, xd.abs() @ wd.abs().T, K)
    assert torch.equal(y, q4().linear(x, w))                # the same bits again


@pytest.mark.parametrize("dt", ["bf16", "fp16"])
@pytest.mark.parametrize("T,N,K", [(1, 4096, 14336), (8, 2048, 16384), (12, 1024, 8192), (40, 2048, 8192), (300, 1024, 8192)])
def test_linear_from_a_cold_cache(T, N, K, dt):
    """Copies that come late and out of step, through rings that are filled several times: always the same bits."""
    w, q, c, wd = make((N, K), 32, K)
    x = acts(T, K, DT[dt], T)
    dy = acts(T, N, DT[dt], T)
    flush = torch.empty(256 << 20, dtype=torch.uint8, device="cuda")
    first = None
    for i in range(60):
        flush.fill_(i)
        y = q4().linear(x, w)
        if first is None:
            first = y
            close(y, x.double() @ wd.T, x.double().abs() @ wd.abs().T, K)
        assert torch.equal(y, first), i
    xg, s = x.clone().requires_grad_(), w.group_scales().requires_grad_()
    ref = None
    for i in range(20):
        y = q4().linear(xg, w, s)
        flush.fill_(i)
        got = torch.autograd.grad(y, (xg, s), dy)
        ref = ref or got
        assert torch.equal(got[0], ref[0]) and torch.equal(got[1], ref[1]), i


@pytest.mark.parametrize("dt", ["bf16", "fp16"])
@pytest.mark.parametrize("T,N,K,group", [(1, 140, 608, 32), (2, 200, 320, 64), (4, 33, 192, 32), (6, 150, 384, 128), (8, 129, 32, 32),
                                         (8, 260, 8224, 32), (10, 40, 1120, 32), (15, 131, 448, 64), (24, 100, 4160, 32), (32, 600, 8480, 32)])
def test_linear_few_rows_at_the_end_of_a_chunk(T, N, K, group, dt):
    """Few rows, the last chunk of 256 values cut off at each place a group can end; a NaN scale there stays in its row."""
    w, q, c, wd = make((N, K), group, T * K)
    x = acts(T, K, DT[dt], K)
    xd = x.double()
    close(q4().linear(x, w), xd @ wd.T, xd.abs() @ wd.abs().T, K)
    bad = w.scales.view(torch.uint8).clone()
    bad[N // 2, -1] = 0x7F
    y = q4().linear(x, q4().Q4(w.codes, bad.view(torch.float8_e4m3fn), w.scale))
    rest = [n for n in range(N) if n != N // 2]
    assert torch.isnan(y[:, N // 2]).all() and torch.equal(y[:, rest], q4().linear(x, w)[:, rest])


@pytest.mark.parametrize("dt", ["bf16", "fp16"])
@pytest.mark.parametrize("T,N,K,group", [(2100, 2500, 4096, 32), (2090, 4100, 2560, 64), (700, 1030, 9472, 128)])
def test_linear_whose_last_tiles_are_split(T, N, K, group, dt):
    """More tiles than run at a time, the rest of them in parts along the contraction (of y or of dx)."""
    w, q, c, wd = make((N, K), group, T)
    x = acts(T, K, DT[dt], N).requires_grad_()
    dy = acts(T, N, DT[dt], K)
    y = q4().linear(x, w)
    xd, d = x.detach().double(), dy.double()
    close(y.detach(), xd @ wd.T, xd.abs() @ wd.abs().T, K)
    (dx,) = torch.autograd.grad(y, x, dy)
    close(dx, d @ wd, d.abs() @ wd.abs(), N)
    y2 = q4().linear(x, w)
    assert torch.equal(y, y2) and torch.equal(dx, torch.autograd.grad(y2, x, dy)[0])


def test_offsets_beyond_32_bits():
    """Codes, activations and results of more than 2^31 elements: the last rows are right."""
    m = q4()
    g = torch.Generator(device="cuda").manual_seed(5)
    E, N, K, group, last = 3, 24576, 65536, 256, 48              # 2.4 GB of codes
    codes = torch.randint(0, 256, (E, N, K // 2), generator=g, device="cuda", dtype=torch.uint8)
    e = (torch.randn(E, N, K // group, generator=g, device="cuda") * 3).to(torch.float8_e4m3fn)
    w = m.Q4(codes, e, torch.full((E,), 0.015625, device="cuda"))
    tail = m.Q4(codes[2, -last:].clone(), e[2, -last:].clone(), w.scale[2:].reshape(()))
    wt, q = m.deq_q4(tail).double(), torch.from_numpy(O4.unpack(tail.codes.cpu().numpy())).double().cuda()
    for T in (4, 100):
        off = torch.tensor([0, 1, 1, T], dtype=torch.int32, device="cuda")
        x = acts(T, K, torch.bfloat16, T).requires_grad_()
        s = w.group_scales().requires_grad_()
        y = m.grouped_linear(x, off, w, s)
        xd = x.detach()[1:].double()
        close(y.detach()[1:, -last:], xd @ wt.T, xd.abs() @ wt.abs().T, K)
        dy = torch.zeros(T, N, device="cuda", dtype=torch.bfloat16)
        dy[:, -last:] = acts(T, last, torch.bfloat16, 7)
        dx, dc = torch.autograd.grad(y, (x, s), dy)
        d = dy[1:, -last:].double()
        close(dx[1:], d @ wt, d.abs() @ wt.abs(), N)
        close(dc[2, -last:], ((d.T @ xd) * q).view(last, -1, group).sum(-1), ((d.abs().T @ xd.abs()) * q.abs()).view(last, -1, group).sum(-1), T + group)
        del x, s, y, dy, dx, dc
    # the last rows of a table, and a result of more than 2^31 elements
    table = m.Q4(codes.view(E * N, K // 2), e.view(E * N, K // group), w.scale[0].reshape(()))
    tok = torch.full((33000,), E * N - last, dtype=torch.int64, device="cuda")
    tok[-last:] = torch.arange(E * N - last, E * N, device="cuda")
    assert torch.equal(m.embedding(tok, table)[-last:], m.deq_q4(tail, torch.bfloat16))
    del codes, e, w, table
    # many rows of x
    T, N, K = 70001, 64, 32768
    w, q, c, wd = make((N, K), 256, 9)
    x = torch.randn(T, K, generator=g, device="cuda", dtype=torch.bfloat16).requires_grad_()
    y = m.linear(x, w)
    dy = acts(T, N, torch.bfloat16, 3)
    (dx,) = torch.autograd.grad(y, x, dy)
    xd, d = x.detach()[-200:].double(), dy[-200:].double()
    close(y[-200:], xd @ wd.T, xd.abs() @ wd.abs().T, K)
    close(dx[-200:], d @ wd, d.abs() @ wd.abs(), N)


@pytest.mark.parametrize("dt", ["bf16", "fp16"])
@pytest.mark.parametrize("T,N,K,group", SIZES)
def test_linear_gradients(T, N, K, group, dt):
    w, q, c, wd = make((N, K), group, T * N + K)
    x = acts(T, K, DT[dt], T).requires_grad_()
    dy = acts(T, N, DT[dt], T + 1)
    scales = w.group_scales().requires_grad_()
    y = q4().linear(x, w, scales)
    assert torch.equal(y.detach(), q4().linear(x.detach(), w))
    dx, dc = torch.autograd.grad(y, (x, scales), dy)
    d, xd = dy.double(), x.detach().double()
    close(dx, d @ wd, d.abs() @ wd.abs(), N)
    full = ((d.T @ xd) * q).view(N, -1, group).sum(-1)
    size = ((d.abs().T @ xd.abs()) * q.abs()).view(N, -1, group).sum(-1)
    close(dc, full, size, T + group)
    again = torch.autograd.grad(q4().linear(x, w, scales), (x, scales), dy)
    assert torch.equal(dx, again[0]) and torch.equal(dc, again[1])


def test_linear_gradient_against_differences():
    # y is linear in x and in c: sum(dy (y(c + d) - y(c))) = sum(dc d), in float64 from the gradients' own values
    w, q, c, wd = make((48, 128), 32, 2)
    x = acts(20, 128, torch.bfloat16, 4).requires_grad_()
    dy = acts(20, 48, torch.bfloat16, 5)
    scales = w.group_scales().requires_grad_()
    dx, dc = torch.autograd.grad(q4().linear(x, w, scales), (x, scales), dy)
    g = torch.Generator(device="cuda").manual_seed(1)
    step_c = torch.randn(c.shape, generator=g, device="cuda", dtype=torch.float64)
    step_x = torch.randn(x.shape, generator=g, device="cuda", dtype=torch.float64)
    f = lambda xx, cc: (dy.double() * (xx @ (q * cc.repeat_interleave(32, -1)).T)).sum()
    xd = x.detach().double()
    size = ((dy.double().abs().T @ xd.abs()) * q.abs()).view(48, -1, 32).sum(-1)
    tol_c = ((2 * 56 * U + U) * size * step_c.abs()).sum().item()
    assert abs((f(xd, c + step_c) - f(xd, c)).item() - (dc.double() * step_c).sum().item()) <= tol_c + 1e-9
    tol_x = ((HALF[torch.bfloat16] + 2 * 52 * U) * (dy.double().abs() @ wd.abs()) * step_x.abs()).sum().item()
    assert abs((f(xd + step_x, c) - f(xd, c)).item() - (dx.double() * step_x).sum().item()) <= tol_x + 1e-9


def test_only_the_gradient_that_is_wanted():
    w, *_ = make((64, 64), 32, 1)
    x = acts(5, 64, torch.bfloat16, 1).requires_grad_()
    q4().linear(x, w).sum().backward()
    assert x.grad is not None
    s = w.group_scales().requires_grad_()
    q4().linear(x.detach(), w, s).sum().backward()           # dy is an expanded tensor of ones
    ones = torch.ones(5, 64, device="cuda", dtype=torch.bfloat16)
    y = q4().linear(x.detach(), w, s)
    assert torch.equal(s.grad, torch.autograd.grad(y, s, ones)[0])
    with torch.no_grad():
        assert not q4().linear(x, w, s).requires_grad


@pytest.mark.parametrize("T", [3, 40])
def test_linear_strides_shapes_and_alignment(T):
    w, q, c, wd = make((72, 160), 32, 9)
    big = acts(2 * T, 400, torch.bfloat16, 2)
    ref = lambda x: (x.double() @ wd.T, x.double().abs() @ wd.abs().T)
    for x in (big[:T, :160], big[:T, 8:168], big[:T, 3:163], big[::2, 16:176], big[:T, :320:2], big[:T, :160].t().contiguous().t(),
              big[:1, 240:].expand(T, 160)):
        assert x.shape == (T, 160)
        y = q4().linear(x, w)
        close(y, *ref(x), 160)
    x = acts(T * 6, 160, torch.float16, 3).view(T, 2, 3, 160)
    y = q4().linear(x, w)
    assert y.shape == (T, 2, 3, 72)
    close(y.view(-1, 72), *ref(x.reshape(-1, 160)), 160)
    one = q4().linear(x[0, 0, 0], w)
    assert one.shape == (72,)
    # gradients come back in x's shape through a strided, misaligned input and gradient
    xs = big[:T, 3:163].detach().requires_grad_()
    dy = acts(T, 90, torch.bfloat16, 7)[:, 5:77]
    (dx,) = torch.autograd.grad(q4().linear(xs, w), xs, dy)
    close(dx, dy.double() @ wd, dy.double().abs() @ wd.abs(), 72)


def test_linear_empty_and_zero():
    w, *_ = make((48, 64), 32, 1)
    x = torch.zeros(0, 64, device="cuda", dtype=torch.bfloat16, requires_grad=True)
    s = w.group_scales().requires_grad_()
    y = q4().linear(x, w, s)
    assert y.shape == (0, 48)
    dx, dc = torch.autograd.grad(y, (x, s), torch.zeros_like(y))
    assert dx.shape == (0, 64) and torch.equal(dc, torch.zeros_like(dc))
    none = q4().enc_q4(torch.zeros(0, 64), 32)
    assert q4().linear(acts(3, 64, torch.bfloat16, 1), none).shape == (3, 0)
    zero = q4().enc_q4(torch.zeros(40, 64), 32)
    assert torch.equal(q4().linear(acts(3, 64, torch.bfloat16, 1), zero), torch.zeros(3, 40, device="cuda", dtype=torch.bfloat16))


@pytest.mark.parametrize("T", [4, 50])
def test_non_finite_values_stay_in_their_row(T):
    w, q, c, wd = make((140, 256), 64, 3)
    x = acts(T, 256, torch.bfloat16, 1)
    clean = q4().linear(x, w)
    x2 = x.clone()
    x2[1, 7], x2[2, 200] = float("nan"), float("inf")
    y = q4().linear(x2, w)
    keep = [t for t in range(T) if t not in (1, 2)]
    assert torch.equal(y[keep], clean[keep]) and torch.isnan(y[1]).all() and not torch.isfinite(y[2]).any()
    # a weight group of NaN spoils its output column, in the gradient its columns of x
    W = torch.randn(140, 256, generator=torch.Generator().manual_seed(1))
    W[5, 70] = float("nan")
    wn = q4().enc_q4(W, 64)
    y = q4().linear(x, wn)
    assert torch.isnan(y[:, 5]).all() and int(torch.isnan(y).sum()) == T
    xg = x.clone().requires_grad_()
    (dx,) = torch.autograd.grad(q4().linear(xg, wn), xg, acts(T, 140, torch.bfloat16, 2))
    bad = torch.isnan(dx).any(0)
    assert bad[64:128].all() and int(bad.sum()) == 64


@pytest.mark.parametrize("T", [2, 33])
def test_large_and_small_scales(T):
    # s far from 1: sums beyond the activations' type before s
    for s, dt in ((2.0 ** -60, torch.bfloat16), (2.0 ** 60, torch.bfloat16), (2.0 ** -14, torch.float16)):
        w, q, c, wd = make((66, 128), 32, 4, s=s)
        x = acts(T, 128, dt, 1)
        close(q4().linear(x, w), x.double() @ wd.T, x.double().abs() @ wd.abs().T, 128)
    # the extremes of E4M3
    codes = torch.full((16, 32), 0x0F, dtype=torch.uint8, device="cuda")
    e = torch.tensor([[448.0], [2.0 ** -9], [-448.0], [-(2.0 ** -9)]] * 4, device="cuda").repeat(1, 2).to(torch.float8_e4m3fn)
    w = q4().Q4(codes, e, torch.tensor(2.0 ** -8, device="cuda"))
    wd = torch.from_numpy(O4.decode(codes.cpu().numpy(), e.view(torch.uint8).cpu().numpy(), 2.0 ** -8, 32)).cuda()
    for dt in (torch.bfloat16, torch.float16):
        x = acts(T, 64, dt, 2)
        close(q4().linear(x, w), x.double() @ wd.T, x.double().abs() @ wd.abs().T, 64)
        xg = x.clone().requires_grad_()
        dy = acts(T, 16, dt, 3)
        (dx,) = torch.autograd.grad(q4().linear(xg, w), xg, dy)
        close(dx, dy.double() @ wd, dy.double().abs() @ wd.abs(), 16)


# ---- experts ---------------------------------------------------------------------------------------------------

RAGGED = [([5], 5, 40, 64, 32), ([0, 3, 0, 1], 4, 130, 96, 32), ([1, 1, 1, 1, 1, 1, 1], 7, 64, 256, 64), ([17, 0, 200, 3, 64], 284, 300, 320, 32),
          ([0, 0, 0], 4, 64, 64, 32), ([129, 128, 127, 1, 0, 255], 640, 136, 512, 256), ([2] * 40, 80, 257, 160, 32), ([600, 0, 5], 620, 1030, 288, 32)]


def experts(counts, first=0):
    return torch.tensor([first + sum(counts[:i]) for i in range(len(counts) + 1)], dtype=torch.int32, device="cuda")


@pytest.mark.parametrize("dt", ["bf16", "fp16"])
@pytest.mark.parametrize("counts,T,N,K,group", RAGGED)
@pytest.mark.parametrize("first", [0, 2])
def test_grouped_values_and_gradients(counts, T, N, K, group, dt, first):
    T = T + first
    E = len(counts)
    w, q, c, wd = make((E, N, K), group, T + N)
    off = experts(counts, first)
    x = acts(T, K, DT[dt], T).requires_grad_()
    dy = acts(T, N, DT[dt], T + 1)
    with torch.no_grad():
        x[:first] = float("nan")                            # rows of nobody
        dy[:first] = float("nan")
        if first + sum(counts) < T:
            x[first + sum(counts):] = float("inf")
            dy[first + sum(counts):] = float("nan")
    scales = w.group_scales().requires_grad_()
    y = q4().grouped_linear(x, off, w, scales)
    dx, dc = torch.autograd.grad(y, (x, scales), dy)
    at = off.tolist()
    for i in range(E):
        a, b = at[i], at[i + 1]
        d, xd = dy[a:b].double(), x.detach()[a:b].double()
        close(y[a:b], xd @ wd[i].T, xd.abs() @ wd[i].abs().T, K)
        close(dx[a:b], d @ wd[i], d.abs() @ wd[i].abs(), N)
        full = ((d.T @ xd) * q[i]).view(N, -1, group).sum(-1)
        size = ((d.abs().T @ xd.abs()) * q[i].abs()).view(N, -1, group).sum(-1)
        close(dc[i], full, size, (b - a) + group)
    rest = torch.ones(T, dtype=torch.bool)
    rest[at[0]:at[-1]] = False
    assert not y[rest.cuda()].any() and not dx[rest.cuda()].any()
    q4().check_errors()


def test_grouped_out_keeps_the_rows_of_nobody():
    w, q, c, wd = make((3, 72, 64), 32, 1)
    x = acts(50, 64, torch.bfloat16, 1)
    off = torch.tensor([4, 20, 20, 45], dtype=torch.int32, device="cuda")
    full = q4().grouped_linear(x, off, w)
    buf = torch.full((50, 100), 7.0, device="cuda", dtype=torch.bfloat16)
    r = q4().grouped_linear(x, off, w, out=buf[:, :72])
    assert r.data_ptr() == buf.data_ptr()
    assert torch.equal(buf[4:45, :72], full[4:45])
    buf[4:45, :72] = 7.0
    assert (buf == 7.0).all()


def test_grouped_takes_falling_and_far_offsets_in_order_and_reports_them():
    w, q, c, wd = make((4, 40, 64), 32, 1)
    x = acts(30, 64, torch.bfloat16, 1)
    for bad, fixed in (([0, 10, 5, 20, 30], [0, 10, 10, 20, 30]), ([0, 10, 20, 90, 95], [0, 10, 20, 30, 30]),
                       ([-5, 10, 20, 25, 30], [0, 10, 20, 25, 30]), ([0, 2**31 - 1, 3, -2**31, 30], [0, 30, 30, 30, 30])):
        y = q4().grouped_linear(x, torch.tensor(bad, dtype=torch.int32, device="cuda"), w)
        with pytest.raises(ValueError, match="offsets"):
            q4().check_errors()
        assert torch.equal(y, q4().grouped_linear(x, torch.tensor(fixed, dtype=torch.int32, device="cuda"), w))
        q4().check_errors()


def test_no_expert_and_many_experts():
    none = q4().Q4(torch.empty(0, 40, 32, dtype=torch.uint8, device="cuda"), torch.empty(0, 40, 2, device="cuda").to(torch.float8_e4m3fn),
                   torch.empty(0, device="cuda"))
    x = acts(5, 64, torch.bfloat16, 1).requires_grad_()
    s = none.group_scales().requires_grad_()
    torch.full((5, 40), 3.0, device="cuda", dtype=torch.bfloat16)            # memory that the result may get, not zero
    y = q4().grouped_linear(x, torch.zeros(1, dtype=torch.int32, device="cuda"), none, s)
    dx, dc = torch.autograd.grad(y, (x, s), torch.ones_like(y))
    assert torch.equal(y, torch.zeros_like(y)) and torch.equal(dx, torch.zeros_like(dx)) and dc.shape == (0, 40, 2)
    # more experts than a warp looks at a time, single rows and gaps between them
    E, N, K = 131, 24, 64
    w, q, c, wd = make((E, N, K), 32, 7)
    counts = [(i * 7) % 3 for i in range(E)]
    off = experts(counts)
    T = sum(counts)
    x = acts(T, K, torch.bfloat16, 3).requires_grad_()
    s = w.group_scales().requires_grad_()
    dy = acts(T, N, torch.bfloat16, 4)
    y = q4().grouped_linear(x, off, w, s)
    dx, dc = torch.autograd.grad(y, (x, s), dy)
    which = torch.repeat_interleave(torch.arange(E), torch.tensor(counts)).cuda()
    xd, d, we = x.detach().double(), dy.double(), wd[which]
    close(y, torch.einsum("tk,tnk->tn", xd, we), torch.einsum("tk,tnk->tn", xd.abs(), we.abs()), K)
    close(dx, torch.einsum("tn,tnk->tk", d, we), torch.einsum("tn,tnk->tk", d.abs(), we.abs()), N)
    outer = torch.zeros(E, N, K, dtype=torch.float64, device="cuda").index_add_(0, which, d[:, :, None] * xd[:, None])
    size = torch.zeros(E, N, K, dtype=torch.float64, device="cuda").index_add_(0, which, d.abs()[:, :, None] * xd.abs()[:, None])
    close(dc, (outer * q).view(E, N, 2, 32).sum(-1), (size * q.abs()).view(E, N, 2, 32).sum(-1), 2 + 32)
    # the same rows in one run, many to the kernels for many rows
    big = q4().Q4(w.codes[:3].contiguous(), w.scales[:3].contiguous(), w.scale[:3].contiguous())
    x2 = acts(900, K, torch.bfloat16, 5)
    y2 = q4().grouped_linear(x2, torch.tensor([0, 0, 900, 900], dtype=torch.int32, device="cuda"), big)
    close(y2, x2.double() @ wd[1].T, x2.double().abs() @ wd[1].abs().T, K)


def test_one_expert_is_linear():
    for T in (3, 70):
        w, *_ = make((1, 200, 320), 64, 2)
        x = acts(T, 320, torch.bfloat16, 2)
        one = q4().Q4(w.codes[0], w.scales[0], w.scale[0])
        d = (q4().grouped_linear(x, experts([T]), w).double() - q4().linear(x, one).double()).abs()
        size = x.double().abs() @ q4().deq_q4(one).double().abs().T
        assert (d <= 4 * 322 * U * size + 2 * HALF[torch.bfloat16] * (x.double() @ q4().deq_q4(one).double().T).abs() + 2 * HALF[torch.bfloat16] * 4 * 322 * U * size).all()


# ---- lookup ----------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("T,V,K,group", [(1, 1, 32, 32), (3, 1000, 4096, 32), (70, 17, 96, 32), (500, 300, 2048 + 256, 256), (33, 40, 320, 64)])
def test_embedding_values(T, V, K, group, dtype):
    w, q, c, wd = make((V, K), group, T + V)
    g = torch.Generator(device="cuda").manual_seed(T)
    tok = torch.randint(0, V, (T,), generator=g, device="cuda")
    for alpha in (1.0, 0.37):
        y = q4().embedding(tok, w, alpha, dtype=dtype)
        exact = alpha * wd[tok]
        # float32 factor alpha s e (two roundings; alpha itself is one more), its product with q, the result
        off = (y.double() - exact).abs()
        assert (off <= exact.abs() * (4 * U + HALF[dtype] * (1 + 4 * U)) + TINY[dtype]).all()
    assert torch.equal(q4().embedding(tok.int().view(1, T, 1), w, dtype=dtype)[0, :, 0], q4().embedding(tok, w, dtype=dtype))


def embed_case(T, V, K, group, dt, tok, alpha, seed):
    w, q, c, wd = make((V, K), group, seed)
    d = acts(T, K, dt, seed)
    s = w.group_scales().requires_grad_()
    y = q4().embedding(tok, w, alpha, s, dtype=dt)
    (dc,) = torch.autograd.grad(y, s, d)
    ok = (tok >= 0) & (tok < V)
    t, dd = tok[ok].long(), d[ok].double()
    sums = lambda v: torch.zeros(V, K // group, dtype=torch.float64, device="cuda").index_add_(0, t, v.view(len(t), K // group, group).sum(-1))
    count = torch.bincount(t, minlength=V).double()[:, None] if len(t) else torch.zeros(V, 1, dtype=torch.float64, device="cuda")
    exact, size = alpha * sums(q[t] * dd), abs(alpha) * sums((q[t] * dd).abs())
    off = (dc.double() - exact).abs()
    assert (off <= (count + group + 4) * U * size).all()
    (again,) = torch.autograd.grad(q4().embedding(tok, w, alpha, s, dtype=dt), s, d)
    assert torch.equal(dc, again)
    return dc


@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("T,V,K,group", [(1, 1, 32, 32), (31, 5, 64, 64), (32, 40, 4096, 32), (33, 2, 96, 32), (1000, 300, 2048 + 256, 256),
                                         (5000, 100000, 128, 128), (1500, 700, 320, 64)])
def test_embedding_gradient(T, V, K, group, dt):
    g = torch.Generator(device="cuda").manual_seed(T + V)
    tok = (torch.rand(T, generator=g, device="cuda") ** 3 * V).long()
    embed_case(T, V, K, group, dt, tok, 1.5, T)
    embed_case(T, V, K, group, dt, tok.int(), -0.3, T + 1)


def test_embedding_gradient_of_one_token_and_of_runs():
    for T in (32, 64, 97, 3000):                             # one token through many pieces
        embed_case(T, 50, 64, 32, torch.bfloat16, torch.full((T,), 7, device="cuda"), 1.0, T)
    tok = torch.arange(64, device="cuda").repeat_interleave(32)         # runs that end where pieces end
    embed_case(2048, 64, 64, 32, torch.bfloat16, tok, 1.0, 1)
    embed_case(2048, 64, 64, 32, torch.bfloat16, tok.roll(16), 1.0, 2)
    embed_case(70000, 3, 32, 32, torch.bfloat16, torch.arange(70000, device="cuda") % 3, 1.0, 3)      # several tiles a chunk


def test_embedding_tokens_outside_the_table():
    w, q, c, wd = make((20, 64), 32, 1)
    tok = torch.tensor([3, -1, 20, 19, 2**40, 3], device="cuda")
    y = q4().embedding(tok, w)
    assert torch.isnan(y[[1, 2, 4]]).all() and torch.isfinite(y[[0, 3, 5]]).all()
    with pytest.raises(ValueError, match="token"):
        q4().check_errors()
    q4().check_errors()
    embed_case(6, 20, 64, 32, torch.float32, tok, 1.0, 4)
    with pytest.raises(ValueError, match="token"):
        q4().check_errors()
    embed_case(40, 20, 64, 32, torch.float32, torch.full((40,), -7, device="cuda"), 1.0, 5)
    with pytest.raises(ValueError):
        q4().check_errors()
    none = torch.zeros(0, dtype=torch.long, device="cuda")
    assert q4().embedding(none, w).shape == (0, 64)
    s = w.group_scales().requires_grad_()
    (dc,) = torch.autograd.grad(q4().embedding(none, w, 1.0, s), s, torch.zeros(0, 64, device="cuda", dtype=torch.bfloat16))
    assert torch.equal(dc, torch.zeros_like(dc))


# ---- refusals --------------------------------------------------------------------------------------------------

def test_refusals():
    m = q4()
    w, *_ = make((40, 64), 32, 1)
    e3, *_ = make((2, 40, 64), 32, 1)
    x = acts(4, 64, torch.bfloat16, 1)
    off = torch.tensor([0, 2, 4], dtype=torch.int32, device="cuda")
    with pytest.raises(TypeError):
        m.linear(x.float(), w)
    with pytest.raises(ValueError):
        m.linear(x[:, :32], w)
    with pytest.raises(ValueError):
        m.linear(x.cpu(), w)
    with pytest.raises(ValueError):
        m.linear(x, e3)
    with pytest.raises(ValueError):
        m.linear(x, w, torch.ones(40, 3, device="cuda"))
    with pytest.raises(ValueError):
        m.grouped_linear(x, off, w)
    with pytest.raises(ValueError):
        m.grouped_linear(x, off.long(), e3)
    with pytest.raises(ValueError):
        m.grouped_linear(x, off[:2], e3)
    with pytest.raises(ValueError):
        m.grouped_linear(x, off.cpu(), e3)
    with pytest.raises(ValueError):
        m.grouped_linear(x[None], off, e3)
    with pytest.raises(ValueError):
        m.grouped_linear(x, off, e3, out=torch.empty(4, 39, device="cuda", dtype=torch.bfloat16))
    with pytest.raises(ValueError):
        m.grouped_linear(x.clone().requires_grad_(), off, e3, out=torch.empty(4, 40, device="cuda", dtype=torch.bfloat16))
    with pytest.raises(TypeError):
        m.embedding(torch.zeros(3, device="cuda"), w)
    with pytest.raises(ValueError):
        m.embedding(torch.zeros(3, dtype=torch.long), w)
    with pytest.raises(ValueError):
        m.embedding(torch.zeros(3, dtype=torch.long, device="cuda"), e3)
    with pytest.raises(TypeError):
        m.embedding(torch.zeros(3, dtype=torch.long, device="cuda"), w, dtype=torch.float64)
    with pytest.raises(ValueError):
        m.enc_q4(torch.zeros(4, 48), 32)
    with pytest.raises(ValueError):
        m.enc_q4(torch.zeros(4, 64), 16)
    with pytest.raises(ValueError):
        m.enc_q4(torch.zeros(64), 32)
    with pytest.raises(ValueError, match="16-byte"):
        m.Q4(torch.zeros(4 * 32 + 8, dtype=torch.uint8, device="cuda")[8:].view(4, 32), w.scales[:4], w.scale)
    with pytest.raises(ValueError, match="contiguous"):
        m.Q4(w.codes[::2], w.scales[::2], w.scale)


# ---- together --------------------------------------------------------------------------------------------------

def test_first_calls_of_a_thread():
    """A thread that has made no CUDA call yet, as autograd's is at its first backward."""
    import threading
    w, q, c, wd = make((256, 512), 32, 1)
    x = acts(300, 512, torch.bfloat16, 1)
    dy = acts(300, 256, torch.bfloat16, 2)
    lib = __import__("ultraquant_b200._lib", fromlist=["load"]).load()
    st = torch.cuda.current_stream().cuda_stream
    out, dx = torch.empty(300, 256, device="cuda", dtype=torch.bfloat16), torch.empty(300, 512, device="cuda", dtype=torch.bfloat16)
    dc = torch.empty(256, 16, device="cuda")
    ptr = (w.codes.data_ptr(), w.scales.data_ptr(), w.scale.data_ptr())
    ws = torch.empty(64 << 20, dtype=torch.uint8, device="cuda")
    tail = (ws.data_ptr(), ws.numel(), st)
    calls = [lambda: lib.uq_q4_linear(x.data_ptr(), 2, 300, 512, *ptr, 1, 256, 512, 32, None, out.data_ptr(), 256, 0, *tail),
             lambda: lib.uq_q4_linear_dx(dy.data_ptr(), 2, 300, 256, *ptr, 1, 256, 512, 32, None, dx.data_ptr(), 512, 0, *tail),
             lambda: lib.uq_q4_linear_dscale(dy.data_ptr(), x.data_ptr(), 2, 300, 256, 512, ptr[0], 1, 256, 512, 32, None, dc.data_ptr(), *tail)]
    for call in calls:
        got = []
        t = threading.Thread(target=lambda: got.append((call(), lib.uq_last_error())))
        t.start()
        t.join()
        assert got[0][0] == 0, got
    close(out, x.double() @ wd.T, x.double().abs() @ wd.abs().T, 512)
    close(dx, dy.double() @ wd, dy.double().abs() @ wd.abs(), 256)


def test_streams_and_captured_graphs():
    m = q4()
    w, *_ = make((520, 1024), 32, 1)
    e, *_ = make((6, 264, 512), 32, 2)
    tab, *_ = make((900, 1024), 32, 3)
    off = experts([3, 0, 20, 9, 1, 7])

    def step(tok, dy):
        x = m.embedding(tok, tab)
        h = m.linear(x, w)[:, :512]
        y = m.grouped_linear(h, off, e)
        s = tab.group_scales().requires_grad_()
        (dc,) = torch.autograd.grad(m.embedding(tok, tab, 1.0, s), s, dy)
        return y, dc

    g = torch.Generator(device="cuda").manual_seed(1)
    toks = [torch.randint(0, 900, (40,), generator=g, device="cuda") for _ in range(3)]
    dys = [acts(40, 1024, torch.bfloat16, i) for i in range(3)]
    want = [step(t, d) for t, d in zip(toks, dys)]
    torch.cuda.synchronize()
    # two side streams at once
    streams = [torch.cuda.Stream() for _ in range(3)]
    got = []
    for s, t, d in zip(streams, toks, dys):
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            for _ in range(5):
                r = step(t, d)
            got.append(r)
    torch.cuda.synchronize()
    for a, b in zip(got, want):
        assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    # two graphs, replayed in turn and with new contents of their inputs
    graphs = []
    for i in range(2):
        t, d = toks[i].clone(), dys[i].clone()
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            step(t, d)
        torch.cuda.current_stream().wait_stream(s)
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            out = step(t, d)
        graphs.append((gr, t, d, out))
    for i in (0, 1, 2):
        for gr, t, d, out in graphs:
            t.copy_(toks[i])
            d.copy_(dys[i])
            gr.replay()
        torch.cuda.synchronize()
        for gr, t, d, out in graphs:
            assert torch.equal(out[0], want[i][0]) and torch.equal(out[1], want[i][1])


@pytest.mark.parametrize("dt", ["bf16", "fp16"])
@pytest.mark.parametrize("rows,n0,T,group", [(40, 300, 5, 32), (130, 1024, 40, 64), (24, 14336, 3, 256), (64, 96, 33, 128)])
def test_recipe_layer(rows, n0, T, group, dt):
    """pipeline.quant_q4_device: the layer is What x without What, and its error sums are those of What."""
    from ultraquant_b200 import pipeline
    rng = np.random.RandomState(n0)
    W = torch.from_numpy(rng.standard_t(4, size=(rows, n0)) * 0.02).cuda()
    H = torch.from_numpy(np.exp(rng.standard_normal(n0))).cuda()
    layer = pipeline.quant_q4_device(W, H, group)
    What = layer.What()
    n = layer.signs.numel()
    sH = torch.maximum(H, H.max() * 1e-3).sqrt()
    # the codes are the restated encoder's of the rotated matrix
    import oracle
    X = oracle.rht_rows((W * sH).cpu().numpy())
    codes, e, s = O4.encode(X, group)
    assert np.array_equal(layer.w.codes.cpu().numpy(), codes) and np.array_equal(layer.w.scales.view(torch.uint8).cpu().numpy(), e)
    Xq = O4.decode(codes, e, s, group)
    assert abs(layer.wnmse - ((X - Xq) ** 2).sum() / (X ** 2).sum()) <= 1e-12
    ref = oracle.irht_rows(Xq, n0) / sH.cpu().numpy()
    assert np.abs(What.double().cpu().numpy() - ref).max() <= 2.0 ** -23 * np.abs(ref).max() + 1e-30      # float32 of a float64 value
    x = acts(T, n0, DT[dt], 1).requires_grad_()
    y = layer(x)
    # rotated activations: float32 transform (log2 n + 3 roundings of values of at most the row's length), one rounding to dt
    xr = torch.from_numpy(oracle.rht_rows((x.detach().double() / sH).cpu().numpy())).cuda()
    norm = xr.norm(dim=1, keepdim=True)
    dxr = HALF[DT[dt]] * xr.abs() + (np.log2(n) + 6) * 2 * U * norm + TINY[DT[dt]]
    Q = torch.from_numpy(Xq).cuda()
    exact = xr @ Q.T
    bound = dxr @ Q.abs().T + 2 * (n + 2) * U * ((xr.abs() + dxr) @ Q.abs().T)
    off = (y.detach().double() - exact).abs()
    assert (off <= bound * (1 + HALF[DT[dt]]) + HALF[DT[dt]] * exact.abs() + TINY[DT[dt]]).all()
    # gradient with respect to x: through the product's dx (rounded to dt) and the transform back
    dy = acts(T, rows, DT[dt], 2)
    (dx,) = torch.autograd.grad(y, x, dy)
    g = dy.double() @ Q
    dg = HALF[DT[dt]] * g.abs() + 2 * (rows + 2) * U * (dy.double().abs() @ Q.abs()) + TINY[DT[dt]]
    back = torch.from_numpy(oracle.irht_rows(g.cpu().numpy(), n0)).cuda() / sH
    tol = ((dg.norm(dim=1, keepdim=True) + (np.log2(n) + 6) * 2 * U * g.norm(dim=1, keepdim=True)) / sH.float().double())
    assert ((dx.double() - back).abs() <= tol * 1.001 + HALF[DT[dt]] * (back.abs() + tol) + TINY[DT[dt]]).all()
    with pytest.raises(ValueError):
        layer(x[:, :-1])
    with pytest.raises(TypeError):
        layer(x.float())


def test_a_model_of_them():
    """Lookup, rotated projection, experts and head as a model runs them: a prompt and then single tokens give the same
    results within counted rounding, and a tuning step on all group scales goes through every operator's gradient."""
    from ultraquant_b200 import pipeline
    m = q4()
    V, d, f, E = 300, 256, 384, 4
    rng = np.random.RandomState(5)
    weights = lambda *s: torch.from_numpy(rng.standard_normal(s) / np.sqrt(s[-1])).cuda()
    table = m.enc_q4(weights(V, d), 32)
    up = pipeline.quant_q4_device(weights(f, d), torch.from_numpy(np.exp(rng.standard_normal(d))).cuda(), 64)
    ex = m.enc_q4(weights(E, d, f), 128)
    head = m.enc_q4(weights(V, d), 64)
    tok = torch.from_numpy(rng.randint(0, V, 37)).cuda()
    which = torch.from_numpy(rng.randint(0, E - 1, 37)).cuda()          # the last expert gets nothing
    order = torch.argsort(which, stable=True)
    off = torch.cat([torch.zeros(1, dtype=torch.long, device="cuda"), torch.bincount(which, minlength=E).cumsum(0)]).int()

    def run(tok, order, off, p=(None, None, None, None)):
        h = m.embedding(tok, table, 4.0, p[0])
        u = up(h, p[1])
        y = m.grouped_linear(u[order], off, ex, p[2])
        back = torch.empty_like(y).index_copy(0, order, y) + h
        return h, u, back, m.linear(back, head, p[3])

    h, u, back, logits = run(tok, order, off)
    # one token at a time: the same products through the kernels for few rows
    H = HALF[torch.bfloat16]
    for t in (0, 20, 36):
        one = torch.zeros(1, dtype=torch.long, device="cuda")
        o1 = torch.where(torch.arange(E + 1, device="cuda") > which[t], 1, 0).int()
        h1, u1, b1, l1 = run(tok[t : t + 1], one, o1)
        assert torch.equal(h1[0], h[t])
        # each stage: twice its own rounding, and what the stage before may differ by times the sizes of its weights
        du = 2 * H * u[t].double().abs() * 1.01 + 1e-5
        assert ((u1[0].double() - u[t].double()).abs() <= du).all()
        we = m.deq_q4(ex)[which[t]].double().abs()
        db = we @ du + 4 * H * (back[t].double().abs() + h[t].double().abs()) * 1.01 + 1e-5
        assert ((b1[0].double() - back[t].double()).abs() <= db).all()
        dl = m.deq_q4(head).double().abs() @ db + 2 * H * logits[t].double().abs() * 1.01 + 1e-5
        assert ((l1[0].double() - logits[t].double()).abs() <= dl).all()
    # the tuning step: gradients of the whole equal those of the pieces, called one by one
    p = [w.group_scales().requires_grad_() for w in (table, up.w, ex, head)]
    g = acts(37, V, torch.bfloat16, 3)
    h, u, back, logits = run(tok, order, off, p)
    grads = torch.autograd.grad(logits, p, g, retain_graph=True)
    gb, gh = torch.autograd.grad(logits, (back, p[3]), g, retain_graph=True)
    assert torch.equal(gh, grads[3])
    gu, ge = torch.autograd.grad(back, (u, p[2]), gb, retain_graph=True)
    assert torch.equal(ge, grads[2])
    ghh, gup = torch.autograd.grad(u, (h, p[1]), gu, retain_graph=True)
    assert torch.equal(gup, grads[1])
    (gt,) = torch.autograd.grad(h, p[0], ghh + gb)
    assert torch.equal(gt, grads[0])
    # the new scales are stored and used
    with torch.no_grad():
        new = m.round_scales(head, p[3] - 0.1 * grads[3] * p[3].abs().mean() / grads[3].abs().mean())
    assert not torch.equal(m.linear(back, new), logits)
    assert torch.equal(new.codes, head.codes)
