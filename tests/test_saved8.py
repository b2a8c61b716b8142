"""CPU: the 8-bit format's oracle, and the refusals of the training operators that use it (no GPU is touched)."""
import ctypes

import numpy as np
import pytest
import torch

from oracle import saved8 as O


@pytest.fixture(scope="module")
def lib():
    from spurfies_amd import _lib, build

    build.build(verbose=False)
    return _lib.lib()


def test_format_is_off_by_at_most_half_a_step():
    rng = np.random.default_rng(0)
    x = np.float32(rng.standard_normal((64, 75)) * np.exp(rng.uniform(-30, 30, (64, 1)))).astype(np.float64)
    codes, steps = O.pack(x)
    step = np.repeat(2.0 ** (steps.astype(float) - 127), 32, axis=1)[:, :75]
    assert (np.abs(O.restore(codes, steps, 75) - x) <= step / 2).all()
    top = np.abs(np.pad(x, ((0, 0), (0, 21))).reshape(64, 3, 32)).max(axis=2)
    s = 2.0 ** (steps.astype(float) - 127)
    assert (np.round(top / s) <= 127).all() and (np.round(top / (s / 2)) > 127).all()          # the least step that holds the largest
    assert (codes[:, 75:] == 0).all()


def test_format_of_zeros_signs_and_values_that_are_not_finite():
    x = np.zeros((4, 33))
    x[1, :5] = [1.0, -1.0, 1e-30, -1e-30, -0.0]
    x[2, 3], x[3, 32] = np.inf, np.nan
    codes, steps = O.pack(x)
    v = O.restore(codes, steps, 33)
    assert (v[0] == 0).all() and np.signbit(v[0]).all()                  # zero is not greater than zero
    assert list(np.signbit(v[1, :5])) == [False, True, False, True, True]
    assert np.isnan(v[2, :32]).all() and v[2, 32] == 0 and (v[3, :32] == 0).all() and np.isnan(v[3, 32])


def test_library_refuses_bad_arguments(lib):
    p, q = ctypes.c_void_p(4096), ctypes.c_void_p(4096 + 8)                # never dereferenced: every call is refused on the host
    err = lambda: lib.spf_last_error().decode()  # noqa: E731
    assert lib.spf_saved8_pack(p, 7, 32, 4, 32, p, p, None) == -22 and "type" in err()
    assert lib.spf_saved8_pack(p, 0, 32, -1, 32, p, p, None) == -22 and "negative" in err()
    assert lib.spf_saved8_pack(p, 0, 32, 4, 32, None, p, None) == -22 and "null" in err()
    assert lib.spf_saved8_pack(p, 0, 32, 4, 32, q, p, None) == -22 and "misaligned" in err()
    assert lib.spf_saved8_pack(p, 0, 1 << 20, 1 << 27, 1 << 20, p, p, None) == -22 and "blocks" in err()
    assert lib.spf_saved8_restore(p, p, 4, 32, p, 0, 31, None) == -22 and "stride" in err()
    assert lib.spf_act8_forward(p, 0, 32, 4, 32, 9, 1.0, p, 32, None, None, None, None, None) == -22 and "activation" in err()
    assert lib.spf_act8_forward(p, 0, 32, 4, 32, 0, -0.1, p, 32, None, None, None, None, None) == -22 and "slope" in err()
    assert lib.spf_act8_forward(p, 0, 32, 4, 32, 1, 0.0, p, 32, None, None, None, None, None) == -22 and "beta" in err()
    assert lib.spf_act8_forward(p, 0, 32, 4, 32, 2, 0.0, p, 32, p, None, None, None, None) == -22 and "null" in err()
    assert lib.spf_act8_backward(p, 0, 32, 4, 32, 2, 0.0, None, None, p, 32, None) == -22 and "null" in err()
    ln = lambda **k: lib.spf_layer_norm_forward(p, k.get("type", 0), 32, k.get("rows", 4), 32, p, p, 0, k.get("eps", 1e-5), p, k.get("ldy", 32), p, k.get("rstd", p), None, None,  # noqa: E731
                                                None, None, None)
    assert ln(type=3) == -22 and "type" in err()
    assert ln(eps=-1.0) == -22 and "eps" in err()
    assert ln(eps=float("nan")) == -22 and "eps" in err()
    assert ln(ldy=31) == -22 and "stride" in err()
    assert ln(rstd=None) == -22 and "null" in err()
    assert ln(rows=1 << 31) == -22 and "2^31" in err()
    back = lambda x, c, ws: lib.spf_layer_norm_backward(p, 0, 32, 4, 32, x, 32, c, c, p, p, p, 0, p, 32, p, p, 0, ws, None)  # noqa: E731
    assert back(None, None, p) == -22 and "one of" in err()
    assert back(p, p, p) == -22 and "one of" in err()
    assert back(p, None, None) == -22 and "workspace" in err()
    assert lib.spf_wgrad8(p, 0, 32, p, p, 4, 32, 32, p, None, 5, 0, p, None) == -22 and "type" in err()
    assert lib.spf_wgrad8_workspace_floats(1 << 16, 32, 32, 0, 0) > 0 and lib.spf_wgrad8_workspace_floats(4, 32, 32, 0, 0) == 0
    assert lib.spf_wgrad8(p, 0, 32, p, p, 1 << 16, 32, 32, p, None, 0, 0, None, None) == -22 and "null" in err()
    assert lib.spf_wgrad8(p, 0, 32, q, p, 4, 32, 32, p, None, 0, 0, p, None) == -22 and "misaligned" in err()
    assert lib.spf_wgrad8(p, 0, 32, p, p, 4, 1 << 21, 32, p, None, 0, 0, p, None) == -22 and "2^20" in err()


def test_nothing_to_do_is_not_an_error(lib):
    for rows, cols in ((0, 32), (4, 0)):
        assert lib.spf_saved8_pack(None, 0, cols, rows, cols, None, None, None) == 0
        assert lib.spf_saved8_restore(None, None, rows, cols, None, 0, cols, None) == 0
        assert lib.spf_layer_norm_forward(None, 0, cols, rows, cols, None, None, 0, 1e-5, None, cols, None, None, None, None, None, None, None) == 0
        assert lib.spf_layer_norm_workspace_floats(rows, cols) == 0 and lib.spf_wgrad8_workspace_floats(rows, 8, cols, 0, 1) == 0
        assert lib.spf_wgrad8(None, 0, 8, None, None, rows, 8, cols, None, None, 0, 0, None, None) == 0


def test_python_refuses_bad_arguments():
    from spurfies_amd import ops

    x = torch.zeros(4, 32)
    for call in (lambda: ops.checkpoint8(x), lambda: ops.act8(x, "silu"), lambda: ops.layer_norm(x), lambda: ops.linear8(x, torch.zeros(8, 32))):
        with pytest.raises(ValueError, match="GPU"):
            call()
    u8 = lambda *s: torch.zeros(*s, dtype=torch.uint8)  # noqa: E731
    for codes, steps, cols in ((u8(4, 32), u8(4, 2), 32), (u8(4, 33), u8(4, 2), 33), (u8(4, 64), u8(3, 2), 64), (torch.zeros(4, 32), u8(4, 1), 32)):
        with pytest.raises(ValueError, match="uint8"):
            ops.Checkpoint8(codes, steps, cols)
    with pytest.raises(ValueError, match="contiguous"):
        ops.Checkpoint8(u8(4, 64)[:, :32], u8(4, 1), 32)
    with pytest.raises(ValueError, match="shape"):
        ops.Checkpoint8(u8(4, 32), u8(4, 1), 32, shape=(3, 32))
    with pytest.raises(ValueError, match="float32"):
        ops.Checkpoint8(u8(4, 32), u8(4, 1), 32, torch.float64)
    ck = ops.Checkpoint8(u8(4, 64), u8(4, 2), 40, shape=(2, 2, 40))
    assert ck.rows == 4 and ck.nbytes == 4 * 66
    with pytest.raises(ValueError, match="GPU"):
        ck.restore()


def test_library_refuses_one_place_for_both_parameter_gradients(lib):
    p = ctypes.c_void_p(4096)                                              # never dereferenced
    assert lib.spf_layer_norm_backward(p, 0, 32, 4, 32, p, 32, None, None, p, p, p, 0, None, 32, p, p, 1, p, None) == -22 and "one address" in lib.spf_last_error().decode()


def test_bias_gradient_by_itself_refuses_bad_arguments(lib):
    p, q = ctypes.c_void_p(4096), ctypes.c_void_p(4096 + 2)                # never dereferenced: every call is refused on the host
    err = lambda: lib.spf_last_error().decode()  # noqa: E731
    sums = lambda g=p, type=0, ld=32, rows=4, n=32, k=32, db=p, wtype=0, ws=p: lib.spf_wgrad8_bias(g, type, ld, rows, n, k, db, wtype, 0, ws, None)  # noqa: E731
    for call, why in ((lambda: sums(type=3), "type"), (lambda: sums(wtype=-1), "type"), (lambda: sums(rows=-1), "negative"), (lambda: sums(n=1 << 21), "2^20"),
                      (lambda: sums(g=None), "null"), (lambda: sums(db=None), "null"), (lambda: sums(ws=None), "null"), (lambda: sums(ld=-1), "stride"), (lambda: sums(g=q), "misaligned"),
                      (lambda: sums(db=q), "misaligned")):
        assert call() == -22 and why in err()
    for rows, n in ((0, 32), (4, 0)):
        assert sums(g=None, rows=rows, n=n, db=None, ws=None) == 0 and lib.spf_wgrad8_bias_workspace_floats(rows, n, 32, 0) == 0
    for rows, n, k in ((1, 1, 1), (70001, 256, 64), (9, 9001, 64), (1 << 30, 1 << 10, 1 << 10)):
        w = lib.spf_wgrad8_bias_workspace_floats(rows, n, k, 1)
        assert w % n == 0 and w >= n and (k + 1) * w == lib.spf_wgrad8_workspace_floats(rows, n, k, 1, 1)


def test_tile_query(lib):
    """The plan as tests see it: by sizes and type alone, nothing for what is refused."""
    assert lib.spf_wgrad8_tile(8192, 4096, 4096, 1) == 256 and lib.spf_wgrad8_tile(1, 1, 1, 0) == 64
    assert {lib.spf_wgrad8_tile(m, n, k, t) for m in (40, 4000, 400000) for n in (7, 100, 256, 2000) for k in (7, 100, 256, 2000) for t in (0, 1, 2)} == {64, 128, 256}
    assert lib.spf_wgrad8_tile(0, 8, 8, 0) == lib.spf_wgrad8_tile(8, 8, 8, 7) == lib.spf_wgrad8_tile(8, 1 << 21, 8, 0) == 0
