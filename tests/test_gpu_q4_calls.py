"""Calls of the 4-bit operators at their edges."""
import numpy as np
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


def constant(shape, q, e, s, group=32):
    *lead, N, K = shape
    codes = torch.full((*lead, N, K // 2), (q + 8) * 17, dtype=torch.uint8, device="cuda")
    return q4().Q4(codes, torch.full((*lead, N, K // group), e, device="cuda").to(torch.float8_e4m3fn), torch.full(tuple(lead), s, device="cuda"))


# ---- sums before the scale -------------------------------------------------------------------------------------

@pytest.mark.parametrize("T,N,K", [(1, 300, 8192), (12, 140, 8192), (30, 140, 64), (40, 2048, 8192), (300, 256, 8192), (515, 264, 320)])
def test_sum_before_the_scale_may_pass_the_largest_float(T, N, K):
    """y = s sum e q x is a bfloat16 although sum e q x is beyond float32 (weights and results of ordinary proportion)."""
    s, x0 = 2.0 ** -24, 2.0 ** 111
    w = constant((N, K), 7, 448.0, s)
    x = torch.full((T, K), x0, device="cuda", dtype=torch.bfloat16).requires_grad_()
    y = q4().linear(x, w)
    (dx,) = torch.autograd.grad(y, x, torch.full_like(y, x0))
    assert float(K) * 3136 * x0 > 3.5e38
    # exact sums of equal terms: multiples of 3136 = 49 * 2^6 below 49 * 2^13 terms, so only the result rounds
    assert torch.equal(y, torch.full_like(y, K * 3136 * x0 * s)) and torch.equal(dx, torch.full_like(dx, N * 3136 * x0 * s))


def test_sum_before_the_scale_may_pass_the_largest_float_with_experts():
    w = constant((5, 136, 1024), -8, 448.0, 2.0 ** -30)
    for counts in ([1, 0, 3, 2, 1], [40, 0, 70, 2, 300]):
        T = sum(counts)
        off = torch.tensor(np.concatenate([[0], np.cumsum(counts)]), dtype=torch.int32, device="cuda")
        x = torch.full((T, 1024), 2.0 ** 112, device="cuda", dtype=torch.bfloat16).requires_grad_()
        y = q4().grouped_linear(x, off, w)
        (dx,) = torch.autograd.grad(y, x, torch.full_like(y, 2.0 ** 112))
        assert torch.equal(y, torch.full_like(y, -1024 * 3584 * 2.0 ** 82)) and torch.equal(dx, torch.full_like(dx, -136 * 3584 * 2.0 ** 82))


@pytest.mark.parametrize("T", [2, 40])
def test_scales_from_the_smallest_to_the_largest(T):
    """s from 2^-126 to 2^120: the result neither overflows nor is lost where it is an ordinary number."""
    for k in (-126, -117, -60, -1, 0, 1, 60, 112, 113, 114, 120):
        w = constant((72, 128), 3, 1.0, 2.0 ** k)
        x = torch.full((T, 128), 2.0 ** -max(min(k, 100), -100), device="cuda", dtype=torch.bfloat16)
        assert torch.equal(q4().linear(x, w), torch.full((T, 72), 384 * 2.0 ** (k - max(min(k, 100), -100)), device="cuda", dtype=torch.bfloat16)), k


# ---- outputs that are given ------------------------------------------------------------------------------------

def experts(seed=0, N=64, K=64):
    g = torch.Generator().manual_seed(seed)
    return q4().enc_q4(torch.randn(3, N, K, generator=g), 32), torch.tensor([0, 300, 301, 700], dtype=torch.int32, device="cuda")


def rows(T, n, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randn(T, n, generator=g, device="cuda").bfloat16()


def test_out_that_overlaps_what_is_read_is_refused():
    m = q4()
    w, off = experts()
    x = rows(700, 64, 1)
    want = m.grouped_linear(x, off, w)
    kept = x.clone()
    for out in (x, torch.as_strided(x, (700, 64), (64, 1), 0)):
        with pytest.raises(ValueError, match="overlap"):
            m.grouped_linear(x, off, w, out=out)
    buf = torch.zeros(701 * 64, device="cuda", dtype=torch.bfloat16)
    a, b = buf[: 700 * 64].view(700, 64), buf[64:].view(700, 64)
    with pytest.raises(ValueError, match="overlap"):
        m.grouped_linear(a, off, w, out=b)
    wide = torch.zeros(700, 160, device="cuda", dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="overlap"):
        m.grouped_linear(wide[:, :64], off, w, out=wide[:, 63:127])
    with pytest.raises(ValueError, match="overlap"):
        m.grouped_linear(wide[:, 96:160], off, w, out=wide[:, 40:104])
    assert torch.equal(x, kept) and not wide.any() and not buf.any()
    # offsets and weights are read as well
    raw = torch.empty(700 * 64 * 2, dtype=torch.uint8, device="cuda")
    inside = raw[: 4 * 4].view(torch.int32)
    inside.copy_(off)
    with pytest.raises(ValueError, match="overlap"):
        m.grouped_linear(x, inside, w, out=raw.view(torch.bfloat16).view(700, 64))
    assert torch.equal(inside, off) and torch.equal(m.grouped_linear(x, off, w), want)


def test_out_beside_what_is_read_is_taken():
    """Parts of one buffer that share no element: before, behind, and columns of the same rows."""
    m = q4()
    w, off = experts()
    x = rows(700, 64, 2)
    want = m.grouped_linear(x, off, w)
    buf = torch.zeros(1400 * 64, device="cuda", dtype=torch.bfloat16)
    a, b = buf[: 700 * 64].view(700, 64), buf[700 * 64 :].view(700, 64)
    for i, o in ((a, b), (b, a)):
        i.copy_(x)
        assert torch.equal(m.grouped_linear(i, off, w, out=o), want)
    wide = torch.zeros(700, 128, device="cuda", dtype=torch.bfloat16)
    for i, o in ((wide[:, :64], wide[:, 64:]), (wide[:, 64:], wide[:, :64])):
        i.copy_(x)
        assert torch.equal(m.grouped_linear(i, off, w, out=o), want)
    half = torch.zeros(1400, 64, device="cuda", dtype=torch.bfloat16)     # every other row
    half[::2] = x
    assert torch.equal(m.grouped_linear(half[::2], off, w, out=half[1::2]), want) and torch.equal(half[::2], x)


def test_out_that_a_backward_pass_needs_is_noticed():
    m = q4()
    w, off = experts()
    v = m.enc_q4(torch.randn(40, 64, generator=torch.Generator().manual_seed(3)), 32)
    s = v.group_scales().requires_grad_()
    buf = rows(700, 64, 3)
    y = m.linear(buf, v, s)                                  # keeps buf for the gradient of s
    m.grouped_linear(rows(700, 64, 4), off, w, out=buf)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        torch.autograd.grad(y.sum(), s)


def test_out_that_wants_a_gradient_is_refused():
    m = q4()
    w, off = experts()
    out = torch.zeros(700, 64, device="cuda", dtype=torch.bfloat16, requires_grad=True)
    with pytest.raises(ValueError, match="gradient"):
        m.grouped_linear(rows(700, 64, 5), off, w, out=out)
    with torch.no_grad():
        assert m.grouped_linear(rows(700, 64, 5), off, w, out=out) is out


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


# ---- what check_errors tells -----------------------------------------------------------------------------------

def test_every_error_is_named_once():
    m = q4()
    w, off = experts()
    table = m.enc_q4(torch.randn(20, 64, generator=torch.Generator().manual_seed(1)), 32)
    bad = torch.tensor([0, 400, 301, 700], dtype=torch.int32, device="cuda")
    m.embedding(torch.tensor([25], device="cuda"), table)
    m.grouped_linear(rows(700, 64, 1), bad, w)
    with pytest.raises(ValueError) as e:
        m.check_errors()
    assert "token" in str(e.value) and "offsets" in str(e.value)
    m.check_errors()


def test_a_wait_that_gives_up_is_reported():
    """The products' bounded wait on a barrier that nothing arrives at, with a limit of 50 ms: it ends, and the report
    raises once, together with what else was met."""
    from ultraquant_b200 import _lib
    m, lib = q4(), _lib.load()
    st = torch.cuda.current_stream().cuda_stream
    assert lib.uq_q4_wait_selftest(st) == _lib.UQ_OK
    with pytest.raises(_lib.UQError, match="timed out"):
        m.check_errors()
    m.check_errors()
    table = m.enc_q4(torch.randn(20, 64, generator=torch.Generator().manual_seed(1)), 32)
    assert lib.uq_q4_wait_selftest(st) == _lib.UQ_OK
    m.embedding(torch.tensor([-1], device="cuda"), table)
    with pytest.raises(_lib.UQError, match="timed out.*token"):
        m.check_errors()
    m.check_errors()


def test_errors_are_read_on_their_own_stream():
    """A side stream's check neither waits for another stream's work nor loses what that one meets later."""
    m = q4()
    table = m.enc_q4(torch.randn(20, 64, generator=torch.Generator().manual_seed(1)), 32)
    tok = torch.tensor([99], device="cuda")
    m.embedding(tok, table)                                  # loads what is launched below
    with pytest.raises(ValueError, match="token"):
        m.check_errors()
    a, b = torch.cuda.Stream(), torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(a):
        torch.cuda._sleep(200_000_000)                       # some 0.1 s
        m.embedding(tok, table)
    with torch.cuda.stream(b):
        m.check_errors()
        assert not a.query(), "the check waited for another stream"
    with torch.cuda.stream(a), pytest.raises(ValueError, match="token"):
        m.check_errors()


def test_profile_case_reports_a_product_that_gave_up(monkeypatch):
    from ultraquant_b200 import _lib, profile_case
    lib = _lib.load()
    st = torch.cuda.current_stream().cuda_stream
    real = profile_case.build_case

    def build(args, lib_, stream):
        run, units, unit = real(args, lib_, stream)

        def with_wait():
            run()
            _lib.check(lib.uq_q4_wait_selftest(st), "selftest")
        return with_wait, units, unit

    monkeypatch.setattr(profile_case, "build_case", build)
    with pytest.raises(_lib.UQError, match="timed out"):
        profile_case.measure("q4few", rows=2, n=256, n0=128, iters=1)


# ---- a frequent token ------------------------------------------------------------------------------------------

@pytest.mark.parametrize("T,dt", [(1 << 20, torch.bfloat16), ((1 << 20) + 17, torch.float32)])
def test_gradient_of_a_token_that_is_everywhere(T, dt):
    """A padding token's gradient: T rows of odd whole numbers, whose sum passes 2^24 early.  Pieces of 32 rows are exact in
    float32 and their sum is the 64-bit one rounded once, with no error that grows with T."""
    m = q4()
    w = constant((5, 64), 1, 1.0, 1.0)
    w.codes.fill_(0x88)                                      # q = 0 but for the first element of each group
    w.codes[:, 0] = 0x89
    w.codes[:, 16] = 0x89
    g = torch.Generator(device="cuda").manual_seed(T)
    d = torch.zeros(T, 64, device="cuda", dtype=dt)
    d[:, 0] = (torch.randint(0, 64, (T,), generator=g, device="cuda") * 2 + 65).to(dt)
    d[:, 32] = (torch.randint(0, 64, (T,), generator=g, device="cuda") * 2 + 1).to(dt)
    s = w.group_scales().requires_grad_()
    tok = torch.full((T,), 3, device="cuda")
    tok[5], tok[T // 2] = 1, 4
    for alpha in (1.0, -0.3):
        (dc,) = torch.autograd.grad(m.embedding(tok, w, alpha, s, dtype=dt), s, d)
        here = tok == 3
        want = torch.stack([d[here, 0].double().sum(), d[here, 32].double().sum()]) * torch.tensor(alpha, dtype=torch.float32, device="cuda").double()
        assert want.abs().max() > 2 ** 24
        assert torch.equal(dc[3], want.float()), (dc[3].double() / want - 1).tolist()
        assert torch.equal(dc[1], (d[5, [0, 32]].double() * torch.tensor(alpha, dtype=torch.float32).item()).float())


def test_gradient_of_a_frequent_token_keeps_infinities():
    m = q4()
    w = constant((5, 64), 1, 1.0, 1.0)
    s = w.group_scales().requires_grad_()
    d = torch.ones(500, 64, device="cuda", dtype=torch.bfloat16)
    d[7, 0], d[300, 40] = float("inf"), float("nan")
    (dc,) = torch.autograd.grad(m.embedding(torch.full((500,), 2, device="cuda"), w, 1.0, s), s, d)
    assert dc[2, 0].item() == float("inf") and torch.isnan(dc[2, 1]) and not dc[[0, 1, 3, 4]].any()
