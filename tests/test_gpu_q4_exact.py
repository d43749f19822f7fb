"""Products with 4-bit weights on whole numbers: every sum is exact in float32 in whatever order it is formed, so the
result is the 64-bit value rounded once, bit for bit.  A group, chunk or part of a long contraction that is lost, taken
twice or read from another stage shows, which a tolerance that grows with the length does not see.

Codes are any; group scales +-1 or +-2, activations and gradients -1, 0 or 1, the matrix's scale a power of two.  Sums of
products are at most 16 K (16 N for dx) and 8 group T for the gradient of a group scale: below 2^24 at every size here."""
import numpy as np
import pytest
import torch

from oracle import uq_q4 as O4

pytestmark = pytest.mark.gpu

DT = {"bf16": torch.bfloat16, "fp16": torch.float16}
MOST = 2 ** 24


def q4():
    from ultraquant_b200 import q4 as m
    return m


@pytest.fixture(autouse=True)
def no_device_errors():
    yield
    q4().check_errors()


def whole(shape, group, seed):
    """Q4, q in float64 and the weights over the matrix's scale (2^-3) in float64."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    *lead, N, K = shape
    codes = torch.randint(0, 256, (*lead, N, K // 2), generator=g, device="cuda").to(torch.uint8)
    e = (1.0 + torch.randint(0, 2, (*lead, N, K // group), generator=g, device="cuda")) * (
        1.0 - 2.0 * torch.randint(0, 2, (*lead, N, K // group), generator=g, device="cuda"))
    w = q4().Q4(codes, e.to(torch.float8_e4m3fn), torch.full(tuple(lead), 0.125, device="cuda"))
    q = torch.from_numpy(O4.unpack(codes.cpu().numpy()).astype(np.float32)).cuda().double()
    return w, q, q * e.double().repeat_interleave(group, -1)


def signs(T, n, dt, seed):
    g = torch.Generator(device="cuda").manual_seed(7000 + seed)
    return (torch.randint(0, 3, (T, n), generator=g, device="cuda") - 1).to(dt)


def once(v, dt):
    """Whole numbers below 2^24 over 8, rounded once."""
    assert v.numel() == 0 or v.abs().max().item() < MOST
    return (v * 0.125).float().to(dt)


def scales_gradient(dy, x, q, group):
    N = q.shape[0]
    return ((dy.double().T @ x.double()) * q).view(N, -1, group).sum(-1).float()


LONG = [(1, 300, 14336, 32), (1, 4096, 14336, 32), (2, 130, 65536, 256), (5, 1024, 28672, 256), (7, 14331, 4128, 32), (8, 2048, 16384, 32),
        (12, 1024, 8192, 64), (15, 77, 32768, 128), (16, 600, 28672, 32), (24, 100, 4160, 32), (32, 600, 8480, 32), (33, 257, 16416, 32),
        (40, 2048, 8192, 32), (64, 300, 65536, 128), (100, 520, 28672, 64), (129, 136, 640, 64), (200, 4096, 4096, 32), (300, 1024, 8192, 32),
        (515, 1100, 1280, 256), (700, 1030, 9472, 128), (2090, 4100, 2560, 64), (2100, 2500, 4096, 32), (3001, 300, 16384, 128)]


@pytest.mark.parametrize("dt", ["bf16", "fp16"])
@pytest.mark.parametrize("T,N,K,group", LONG)
def test_linear_and_gradients_are_exact(T, N, K, group, dt):
    w, q, ws = whole((N, K), group, T + N + K)
    assert 16 * max(K, N) < MOST and 8 * group * T < MOST
    x = signs(T, K, DT[dt], T).requires_grad_()
    dy = signs(T, N, DT[dt], N)
    s = w.group_scales().requires_grad_()
    want = once(x.detach().double() @ ws.T, DT[dt]), once(dy.double() @ ws, DT[dt]), scales_gradient(dy, x.detach(), q, group)
    flush = torch.empty(256 << 20, dtype=torch.uint8, device="cuda")
    for i in range(3):                                       # the last from a cold cache
        y = q4().linear(x, w, s)
        got = y.detach(), *torch.autograd.grad(y, (x, s), dy)
        for a, b in zip(got, want):
            assert a.dtype == b.dtype and torch.equal(a, b), f"{int((a != b).sum())} of {a.numel()} values"
        flush.fill_(i)


def runs(counts, first=0):
    return torch.tensor([first + sum(counts[:i]) for i in range(len(counts) + 1)], dtype=torch.int32, device="cuda")


# even and skewed loads: few experts with most of the rows, alone or among many idle ones
LOADS = [([17, 0, 200, 3, 64], 300, 1056, 32), ([0] * 30 + [256] + [0] * 20 + [256, 256] + [0] * 10 + [255], 264, 2048, 64), ([0] * 63 + [1000], 130, 4096, 32),
         ([900] + [1] * 40, 260, 1312, 32), ([3] * 64, 513, 4096, 128), ([40, 25, 70, 100, 33, 64, 65, 17], 300, 8192, 256), ([600, 0, 5], 1030, 16384, 128)]


@pytest.mark.parametrize("dt", ["bf16", "fp16"])
@pytest.mark.parametrize("counts,N,K,group", LOADS)
def test_experts_and_gradients_are_exact(counts, N, K, group, dt):
    E, T = len(counts), sum(counts) + 3
    w, q, ws = whole((E, N, K), group, T + N)
    off = runs(counts, 1)
    x = signs(T, K, DT[dt], T).requires_grad_()
    dy = signs(T, N, DT[dt], N)
    s = w.group_scales().requires_grad_()
    assert 16 * max(K, N) < MOST and 8 * group * max(counts) < MOST
    y = q4().grouped_linear(x, off, w, s)
    dx, dc = torch.autograd.grad(y, (x, s), dy)
    at = off.tolist()
    for i in range(E):
        a, b = at[i], at[i + 1]
        assert torch.equal(y.detach()[a:b], once(x.detach()[a:b].double() @ ws[i].T, DT[dt])), i
        assert torch.equal(dx[a:b], once(dy[a:b].double() @ ws[i], DT[dt])), i
        assert torch.equal(dc[i], scales_gradient(dy[a:b], x.detach()[a:b], q[i], group)), i
    for r in (y, dx):
        assert not r[: at[0]].any() and not r[at[-1]:].any()


def test_offsets_beyond_32_bits_are_exact():
    """More than 2^31 codes and long rows: the last matrix's results whole, not its last rows alone."""
    m = q4()
    g = torch.Generator(device="cuda").manual_seed(6)
    E, N, K, group = 3, 24576, 65536, 256                    # 2.4 GB of codes
    codes = torch.randint(0, 256, (E, N, K // 2), generator=g, device="cuda", dtype=torch.uint8)
    e = (1.0 + torch.randint(0, 2, (E, N, K // group), generator=g, device="cuda")).to(torch.float8_e4m3fn)
    w = m.Q4(codes, e, torch.full((E,), 0.125, device="cuda"))
    last = m.Q4(codes[2], e[2], w.scale[2])
    for T in (4, 100):
        off = torch.tensor([0, 1, 1, T], dtype=torch.int32, device="cuda")
        x = signs(T, K, torch.bfloat16, T).requires_grad_()
        dy = signs(T, N, torch.bfloat16, T)
        s = w.group_scales().requires_grad_()
        y = m.grouped_linear(x, off, w, s)
        dx, dc = torch.autograd.grad(y, (x, s), dy)
        sums, dsums = torch.empty(T - 1, N, dtype=torch.float64, device="cuda"), torch.zeros(T - 1, K, dtype=torch.float64, device="cuda")
        xd, d = x.detach()[1:].double(), dy[1:].double()
        for n in range(0, N, 4096):
            part = m.Q4(codes[2, n : n + 4096], e[2, n : n + 4096], torch.ones((), device="cuda"))
            wd = m.deq_q4(part).double()                     # e q, whole numbers
            sums[:, n : n + 4096] = xd @ wd.T
            dsums += d[:, n : n + 4096] @ wd
            qd = wd / part.scales.double().repeat_interleave(group, -1)
            assert torch.equal(dc[2, n : n + 4096], scales_gradient(dy[1:, n : n + 4096], x.detach()[1:], qd, group))
        assert torch.equal(y.detach()[1:], once(sums, torch.bfloat16)) and torch.equal(dx[1:], once(dsums, torch.bfloat16))
        # one matrix of it through the entry without offsets
        assert torch.equal(m.linear(x.detach()[1:], last), y.detach()[1:])
        del x, dy, s, y, dx, dc


@pytest.mark.parametrize("dt", ["bf16"])
@pytest.mark.parametrize("T", [3, 20, 150])
def test_small_and_large_activations_scale(T, dt):
    """A power of two on the activations is one on the result while both stay normal numbers."""
    w, *_ = whole((300, 4128), 32, 5)
    x = signs(T, 4128, DT[dt], 2)
    y = q4().linear(x, w)
    for k in (-90, -30, 30, 90):
        f = torch.tensor(2.0 ** k, device="cuda")
        assert torch.equal(q4().linear((x.float() * f).to(DT[dt]), w).float(), y.float() * f), k
