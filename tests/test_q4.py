"""4-bit weights without a GPU: the restated form, and what the Python layer and the C ABI refuse."""
import numpy as np
import pytest
import torch

from oracle import uq_q4 as O4


def test_pack_round_trip_and_place_of_each_element():
    q = np.arange(-8, 8).reshape(1, 16)
    b = O4.pack(q)
    assert np.array_equal(O4.unpack(b), q)
    # u = 0 .. 7: bytes hold (0, 2), (4, 6), (1, 3), (5, 7) as low | high << 4
    assert b[0, :4].tolist() == [0x20, 0x64, 0x31, 0x75]


def test_e4m3_values_are_torchs():
    c = np.arange(256, dtype=np.uint8)
    t = torch.from_numpy(c.copy()).view(torch.float8_e4m3fn).double().numpy()
    assert np.array_equal(O4.e4m3_values(c), t, equal_nan=True)


def test_e4m3_rounding_is_torchs_away_from_zero():
    rng = np.random.RandomState(0)
    mid = (O4.E4M3[1:] + O4.E4M3[:-1]) / 2                    # ties
    v = np.concatenate([rng.uniform(-448, 448, 2000), 2.0 ** rng.uniform(-9, 8, 2000), mid[1:], -mid[1:]])
    t = torch.from_numpy(v).float()
    v = t.double().numpy()
    assert np.array_equal(O4.e4m3_round(v), t.to(torch.float8_e4m3fn).view(torch.uint8).numpy())
    assert O4.e4m3_round(np.array([0.0, 1e-9, -1e-9, 2.0 ** -10])).tolist() == [0, 1, 129, 1]


@pytest.mark.parametrize("group", [32, 64, 128, 256])
def test_encode_restated(group):
    rng = np.random.RandomState(group)
    W = rng.standard_normal((9, 512)).astype(np.float32) * np.exp(rng.standard_normal((9, 1)))
    W[3, :group] = 0
    codes, e, s = O4.encode(W, group)
    w = O4.decode(codes, e, s, group)
    c = np.repeat(np.abs(O4.e4m3_values(e)) * float(s), group, 1)
    # half a step, and the clipped end: a value of the other sign as large as the largest is -8 against 7 steps,
    # whose step is off by an E4M3 rounding (1 in 16)
    assert np.all(np.abs(w - W) <= c * (0.5 + 1 + 8 / 16) + 1e-30)
    assert np.all(w[3, :group] == 0)
    top = np.abs(W).max()
    assert top <= 3584 * float(s) < 2 * 3584 * float(s) and top > 3584 * float(s) / 2


def test_python_layer_refuses_what_is_not_built():
    from ultraquant_b200 import q4
    codes, e, s = torch.zeros(4, 32, dtype=torch.uint8), torch.zeros(4, 2).to(torch.float8_e4m3fn), torch.ones(())
    with pytest.raises(ValueError, match="CUDA"):
        q4.Q4(codes, e, s)
    with pytest.raises(TypeError):
        q4.Q4(codes.int(), e, s)
    with pytest.raises(TypeError):
        q4.Q4(codes, e.float(), s)
    with pytest.raises(ValueError, match="shapes"):
        q4.Q4(codes, e[:3], s)
    with pytest.raises(ValueError, match="shapes"):
        q4.Q4(codes, e, torch.ones(2))
    with pytest.raises(ValueError, match="groups"):
        q4.Q4(codes, torch.zeros(4, 4).to(torch.float8_e4m3fn), s)      # groups of 16
    with pytest.raises(ValueError, match="groups"):
        q4.Q4(codes, torch.zeros(4, 3).to(torch.float8_e4m3fn), s)
    with pytest.raises(TypeError, match="dtype"):
        q4.enc_q4(torch.zeros(4, 64, dtype=torch.int32))


def test_c_abi_refuses(tmp_path):
    from ultraquant_b200 import _lib
    lib = _lib.load()
    bad, err = _lib.UQ_ERR_INVALID, lambda: lib.uq_last_error().decode()
    p = 1 << 20      # never followed: every call below is refused before a launch
    assert lib.uq_q4_encode(p, 0, 1, 4, 48, 48, 32, p, p, p, p, 1 << 20, None) == bad and "whole groups" in err()
    assert lib.uq_q4_encode(p, 0, 1, 4, 64, 63, 32, p, p, p, p, 1 << 20, None) == bad
    assert lib.uq_q4_encode(p, 0, 1, 4, 64, 64, 48, p, p, p, p, 1 << 20, None) == bad
    assert lib.uq_q4_encode(p, 9, 1, 4, 64, 64, 32, p, p, p, p, 1 << 20, None) == bad and "dtype" in err()
    assert lib.uq_q4_encode(None, 0, 1, 4, 64, 64, 32, p, p, p, p, 1 << 20, None) == bad and "null" in err()
    assert lib.uq_q4_encode(p, 0, 1, 4, 64, 64, 32, p + 4, p, p, p, 1 << 20, None) == bad and "aligned" in err()
    assert lib.uq_q4_encode(p, 0, 1, 4, 64, 64, 32, p, p, p, None, 0, None) == _lib.UQ_ERR_WORKSPACE and "workspace" in err()
    assert lib.uq_q4_encode(p, 0, 65536, 4, 64, 64, 32, p, p, p, p, 1 << 30, None) == bad
    assert lib.uq_q4_decode(p, p, p, 1, 4, 64, 32, p, 1, None) == bad and "dtype" in err()
    assert lib.uq_q4_round_scales(p, -1, 4, p, p, None) == bad
    lin = lambda f, dt=2, T=4, ldx=64, mats=1, N=8, K=64, g=32, off=None, x=p, c=p, ld2=64: f(
        x, dt, T, ldx, c, p, p, mats, N, K, g, off, p, ld2, 1, None, 0, None)
    for f in (lib.uq_q4_linear, lib.uq_q4_linear_dx):
        assert lin(f, dt=0) == bad and "dtype" in err()
        assert lin(f, K=48) == bad and lin(f, g=16) == bad and lin(f, T=-1) == bad and lin(f, T=1 << 31) == bad
        assert lin(f, mats=2) == bad                         # several matrices need offsets
        assert lin(f, x=None) == bad and "null" in err()
        assert lin(f, x=p + 8) == bad and "aligned" in err()
        assert lin(f, c=p + 8) == bad
        assert lin(f, ldx=60) == bad and lin(f, ldx=4) == bad
        assert lin(f, ld2=4) == bad
        assert lin(f, T=0) == 0
    ds = lambda dt=2, T=4, ldy=8, ldx=64, mats=1, N=8, K=64, g=32, off=None, dc=p: lib.uq_q4_linear_dscale(
        p, p, dt, T, ldy, ldx, p, mats, N, K, g, off, dc, None, 0, None)
    assert ds(dt=0) == bad and ds(K=48) == bad and ds(mats=3) == bad and ds(dc=None) == bad
    assert ds(ldy=12) == bad and ds(ldx=56) == bad and ds(ldx=60) == bad
    em = lambda T=2, V=8, K=64, g=32, dt=2, out=p, c=p: lib.uq_q4_embed(p, 1, T, c, p, p, V, K, g, 1.0, out, dt, None)
    assert em(T=-1) == bad and em(K=40) == bad and em(dt=1) == bad and em(out=None) == bad and em(c=p + 2) == bad and em(T=0) == 0
    eb = lambda T=2, V=8, K=64, g=32, dt=2, ld=64, ws=None, n=0: lib.uq_q4_embed_dscale(p, 1, T, p, dt, ld, p, V, K, g, 1.0, p, ws, n, None)
    assert eb(T=-1) == bad and eb(T=1 << 30) == bad and eb(K=40) == bad and eb(dt=1) == bad and eb(ld=60) == bad and eb(ld=32) == bad
    assert eb() == _lib.UQ_ERR_WORKSPACE and "workspace" in err()


def test_c_abi_refuses_scales_off_their_boundary():
    from ultraquant_b200 import _lib
    lib = _lib.load()
    p = 1 << 20      # never followed
    for f in (lib.uq_q4_linear, lib.uq_q4_linear_dx):
        for off in (1, 2, 8):
            rc = f(p, 2, 4, 64, p, p + off, p, 1, 8, 64, 32, None, p, 64, 1, None, 0, None)
            assert rc == _lib.UQ_ERR_INVALID and "scales" in lib.uq_last_error().decode()


def test_workspace_sizes_grow_with_the_call():
    from ultraquant_b200 import _lib
    lib = _lib.load()
    f = lib.uq_q4_embed_dscale_workspace_bytes
    assert f(0, 100, 64, 32) == 0
    a, b = f(1000, 1000, 4096, 32), f(100000, 1000, 4096, 32)
    assert 16 * 1000 < a < b
