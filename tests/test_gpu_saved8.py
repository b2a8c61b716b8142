"""The training operators with 8-bit saved activations (ops.checkpoint8, act8, layer_norm, wgrad8, linear8) against their definitions in 64 bits.

Tolerances.  u = 2^-24 is half a unit in the last place of a 32-bit result, h(type) = finfo.eps / 2 that of the result's type.  A result is held to
h |result| + K u M, M the sum of the magnitudes that were added up and K the number of roundings on the way, which is said where it is used."""
import numpy as np
import pytest
import torch

from oracle import saved8 as O

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
TYPES = [torch.float32, torch.bfloat16, torch.float16]
KINDS = [("leaky_relu", 0.01), ("leaky_relu", 0.0), ("softplus", 100.0), ("silu", None), ("gelu", None)]


def half(dtype):
    return torch.finfo(dtype).eps / 2


def tiny(dtype):
    """the spacing of the type's smallest numbers"""
    return torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps


def f64(t):
    return t.detach().double().cpu().numpy()


def randn(shape, dtype, seed, scale=1.0, shift=0.0, pad=0):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(*shape[:-1], shape[-1] + pad, generator=g) * scale + shift
    return x.to(dtype).cuda()[..., :shape[-1]]


def close(got, want, tol, what):
    got = f64(got) if torch.is_tensor(got) else got
    assert got.shape == want.shape, (what, got.shape, want.shape)
    bad = ~(np.abs(got - want) <= tol)
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.size} off, worst {np.nanmax(np.abs(got - want) / np.maximum(tol, 1e-300)):.3g} times the tolerance"


# ---- the format -------------------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,cols,pad", [(1, 1, 0), (3, 7, 0), (5, 31, 2), (4, 32, 0), (7, 33, 0), (129, 104, 0), (2, 515, 9), (65, 256, 8), (1, 4099, 0)])
def test_checkpoint_is_the_format_byte_for_byte(dtype, rows, cols, pad):
    from spurfies_amd import ops

    x = randn((rows, cols), dtype, rows * 1000 + cols, pad=pad)
    x = x * torch.exp(torch.linspace(-9, 9, rows, device="cuda"))[:, None].to(dtype) if not pad else x
    ck = ops.checkpoint8(x)
    codes, steps = O.pack(f64(x))
    assert np.array_equal(ck.codes.cpu().numpy(), codes) and np.array_equal(ck.steps.cpu().numpy(), steps)
    assert ck.shape == (rows, cols) and ck.dtype == dtype
    back = ck.restore()
    assert back.dtype == dtype and np.array_equal(f64(back), np.clip(O.restore(codes, steps, cols), -float(torch.finfo(dtype).max), float(torch.finfo(dtype).max)))
    assert np.array_equal(f64(ck.restore(torch.float32)), np.float32(O.restore(codes, steps, cols)).astype(np.float64))


@pytest.mark.parametrize("dtype", TYPES)
def test_checkpoint_of_special_values(dtype):
    from spurfies_amd import ops

    big, small = float(torch.finfo(dtype).max), float(torch.finfo(dtype).smallest_normal)
    rows = [[0.0] * 64, [-0.0] * 64, [big] * 64, [-big, 1.0] * 32, [small] * 64, [small / 4, -small / 4] * 32, [1.0, -1.0, 1e-30, -1e-30] * 16,
            [127.0, 126.5, 0.5, 1.5, 2.5, -0.5, -1.5, 63.5] * 8, [127.5, 1.0, -1.0, 0.0] * 16, [127.4, 1.0, -1.0, 0.0] * 16,
            [float("inf")] + [1.0] * 63, [1.0] * 40 + [float("nan")] + [2.0] * 23, [float("-inf")] * 32 + [3.0] * 32]
    x = torch.tensor(rows).to(dtype).cuda()
    ck = ops.checkpoint8(x)
    codes, steps = O.pack(f64(x))
    assert np.array_equal(ck.steps.cpu().numpy(), steps)
    fine = np.repeat(steps != 255, 32, axis=1)
    assert np.array_equal(ck.codes.cpu().numpy()[fine], codes[fine])
    want = O.restore(codes, steps, 64)
    with np.errstate(invalid="ignore"):
        want = np.clip(want, -65504, 65504) if dtype == torch.float16 else want
    got = f64(ck.restore())
    assert np.array_equal(np.isnan(got), np.isnan(want)) and np.array_equal(got[~np.isnan(want)], want[~np.isnan(want)])
    assert np.array_equal(np.signbit(got[fine]), np.signbit(want[fine]))


def test_checkpoint_of_shapes_strides_and_nothing():
    from spurfies_amd import ops

    x = randn((3, 5, 40), torch.float32, 1)
    assert torch.equal(ops.checkpoint8(x).restore(), ops.checkpoint8(x.reshape(15, 40)).restore().view(3, 5, 40))
    t = x.transpose(0, 2)                                              # the last dimension is not the dense one
    assert torch.equal(ops.checkpoint8(t).restore(), ops.checkpoint8(t.contiguous()).restore())
    e = x[0, :1].expand(7, 40)                                         # a row stride of zero
    assert torch.equal(ops.checkpoint8(e).restore(), ops.checkpoint8(e.contiguous()).restore())
    one = x[0, 0]
    assert torch.equal(ops.checkpoint8(one).restore(), ops.checkpoint8(one[None]).restore()[0])
    off = torch.randn(4 * 33 + 3, device="cuda")[3:].view(4, 33)       # rows that start between 16-byte boundaries
    assert torch.equal(ops.checkpoint8(off).restore(), ops.checkpoint8(off.clone()).restore())
    for shape in ((0, 40), (4, 0), (2, 0, 40), (0,)):
        ck = ops.checkpoint8(torch.empty(shape, device="cuda"))
        assert ck.restore().shape == shape


def test_offsets_beyond_32_bits():
    """Rows more than 2^31 elements apart: bf16, 2.2 * 10^9 elements, of which three rows are touched."""
    from spurfies_amd import ops

    far = 1_100_000_000
    base = torch.empty(2 * far + 515, dtype=torch.bfloat16, device="cuda")
    x = base.as_strided((3, 515), (far, 1))
    x.copy_(randn((3, 515), torch.bfloat16, 4))
    small = x.clone()
    w, b = randn((515,), torch.float32, 5), randn((515,), torch.float32, 6)
    assert torch.equal(ops.checkpoint8(x).codes, ops.checkpoint8(small).codes)
    assert torch.equal(ops.layer_norm(x, w, b), ops.layer_norm(small, w, b))
    assert torch.equal(ops.act8(x, "gelu"), ops.act8(small, "gelu"))
    ck = ops.checkpoint8(small[:, :100])
    assert all(torch.equal(p, q) for p, q in zip(ops.wgrad8(x, ck), ops.wgrad8(small, ck)))


def test_more_than_2_31_elements():
    """70000 x 32768 bf16 in one piece: the last rows come out as they do alone."""
    from spurfies_amd import ops

    x = torch.full((70000, 32768), 0.5, dtype=torch.bfloat16, device="cuda")
    tail = randn((3, 32768), torch.bfloat16, 1)
    x[-3:] = tail
    ck = ops.checkpoint8(x)
    small = ops.checkpoint8(tail)
    assert torch.equal(ck.codes[-3:], small.codes) and torch.equal(ck.steps[-3:], small.steps)
    assert torch.equal(ck.restore()[-3:], small.restore())
    del ck
    assert torch.equal(ops.act8(x, "silu")[-3:], ops.act8(tail, "silu"))
    assert torch.equal(ops.layer_norm(x)[-3:], ops.layer_norm(tail))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_rows_between_vector_boundaries(dtype):
    """Views that start at any element, with odd row strides: the same bits as their copies."""
    from spurfies_amd import ops

    base = randn((40, 1031), dtype, 1)
    w, b = randn((515,), dtype, 2), randn((515,), dtype, 3)
    for off in (1, 2, 3, 5):
        x, g = base[:, off:off + 515], base[:, 515 - off:1030 - off]
        xs = [x.detach().requires_grad_(True), x.detach().clone().requires_grad_(True)]
        got = []
        for v, h in zip(xs, (g, g.clone())):
            y = ops.layer_norm(v, w, b, saved8=True)
            z = ops.act8(v, "gelu")
            got.append((y.detach(), z.detach(), torch.autograd.grad(y, v, h)[0], torch.autograd.grad(z, v, h)[0]) + tuple(ops.wgrad8(h, ops.checkpoint8(v))))
        assert all(torch.equal(p, q) for p, q in zip(*got)), off


# ---- activations ------------------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("kind,param", KINDS)
@pytest.mark.parametrize("shape,pad", [((1, 1), 0), ((5, 31), 0), ((128, 256), 0), ((33, 104), 8), ((3, 2, 515), 5)])
def test_act8_forward_and_backward(dtype, kind, param, shape, pad):
    from spurfies_amd import ops

    p = 0.0 if param is None else param
    x = randn(shape, dtype, 3, scale=0.05 if kind == "softplus" else 2.0, pad=pad).requires_grad_(True)
    g = randn(shape, dtype, 4, pad=pad)
    y, ck = ops.act8(x, kind, param=param, out8=True)
    dx, = torch.autograd.grad(y, x, g)
    cols = shape[-1]
    X, G = f64(x).reshape(-1, cols), f64(g).reshape(-1, cols)
    z = np.abs(p * X) if kind == "softplus" else np.abs(X)
    # K: exp / log1p / erf within 4 u, a quotient or product each u; the exponential's argument is rounded once, which counts |argument| u
    want = O.act(kind, X, p)
    scale = {"leaky_relu": np.abs(want), "softplus": np.abs(want) + np.log1p(np.exp(-z)) / max(p, 1e-30), "silu": np.abs(want), "gelu": np.abs(X)}[kind]
    close(f64(y).reshape(-1, cols), want, half(dtype) * np.abs(want) + 16 * U * scale * (1 + z) + tiny(dtype), "y")
    assert torch.equal(ck.codes, ops.checkpoint8(y).codes) and torch.equal(ck.steps, ops.checkpoint8(y).steps) and ck.shape == tuple(shape)
    saved = f64(y).reshape(-1, cols) if kind == "leaky_relu" else X
    R = O.restore(*O.pack(saved), cols)
    slope = O.act_slope(kind, R, p)
    zr = np.abs(p * R) if kind == "softplus" else np.abs(R)
    want = G * slope
    # the slope's terms are at most 1 + |x|; the same counting
    close(f64(dx).reshape(-1, cols), want, half(dtype) * np.abs(want) + (4 if kind == "leaky_relu" else 16) * U * np.abs(G) * (1 + zr) ** 2 + tiny(dtype), "dx")
    if kind == "leaky_relu":      # the sign survives: the slope is the exact input's
        exact = G * np.where(X > 0, 1.0, p)
        close(f64(dx).reshape(-1, cols), exact, half(dtype) * np.abs(exact) + 2 * U * np.abs(exact) + tiny(dtype), "dx by the exact sign")


@pytest.mark.parametrize("kind,param", [("softplus", 100.0), ("silu", None), ("gelu", None)])
def test_act8_slope_against_differences(kind, param):
    """dx / dy at the restored input against central differences of the 64-bit function: h = 1e-5 leaves h^2 / 6 |f'''| (softplus: f''' <= beta^2 / 10 there)."""
    from spurfies_amd import ops

    p = 0.0 if param is None else param
    x = randn((16, 96), torch.float32, 8, scale=0.03 if kind == "softplus" else 2.0).requires_grad_(True)
    y = ops.act8(x, kind, param=param)
    dx, = torch.autograd.grad(y, x, torch.ones_like(y))
    r = O.restore(*O.pack(f64(x)), 96)
    h = 1e-5 / max(1.0, p)
    diff = (O.act(kind, r + h, p) - O.act(kind, r - h, p)) / (2 * h)
    # h^2 f''' < 1e-10 for each, the quotient of doubles 2^-52 |f| / h < 2^-52 * 10 / 1e-7, and dx's own roundings (16 (1 + |z|)^2 u as above)
    z = np.abs(p * r) if kind == "softplus" else np.abs(r)
    close(dx, diff, 1e-8 + 16 * U * (1 + z) ** 2, "slope")


def test_act8_values_that_are_not_finite_and_extremes():
    from spurfies_amd import ops

    inf, nan = float("inf"), float("nan")
    x = torch.tensor([[inf] + [1.0] * 31, [-inf] + [1.0] * 31, [nan] + [1.0] * 31, [1e30] * 32, [-1e30] * 32, [0.0] * 32], device="cuda", requires_grad=True)
    for kind, first in (("leaky_relu", (inf, -inf)), ("softplus", (inf, 0.0)), ("silu", (inf, nan)), ("gelu", (inf, nan))):
        y = ops.act8(x, kind)
        dx, = torch.autograd.grad(y, x, torch.ones_like(y))
        y = y.detach()
        assert float(y[0, 0]) == first[0] and (float(y[1, 0]) == first[1] or (first[1] != first[1] and torch.isnan(y[1, 0])))
        assert torch.isnan(y[2, 0]) and torch.isfinite(y[:3, 1:]).all() and torch.isfinite(y[3:]).all()
        bad = torch.isnan(dx).all(dim=1).tolist()
        # a block whose saved form is not finite has no slope (softplus(-inf) = 0 and the like change y, not the saved x; leaky_relu saves y)
        assert bad == [True, True, True, False, False, False], (kind, bad)
        assert torch.isfinite(dx[3:]).all()
    assert torch.equal(torch.autograd.grad(ops.act8(x[5:], "leaky_relu", 0.25), x, torch.ones(1, 32, device="cuda"))[0][5], torch.full((32,), 0.25, device="cuda"))


# ---- layer norm -------------------------------------------------------------------------------------------------------------------------
NORM_SHAPES = [(1, 1), (3, 2), (37, 17), (9, 32), (70, 45), (33, 100), (21, 256), (5, 257), (19, 515), (6, 1024), (5, 1500), (4, 2048), (5, 3001), (3, 4099), (3, 8192), (2, 9000), (2, 16385)]


def norm_tolerances(X, G, W, B, R, mean, rstd, dtype, wdtype, rows):
    """K: a thread adds up to 16 columns (cols / 4096 where rows are read again), a row's threads meet in 10 steps, five more roundings follow."""
    cols = X.shape[1]
    K = 32 + cols / 2048
    dmean = K * U * np.abs(X).mean(axis=1, keepdims=True)                       # of the mean
    # rstd: the squares' sum has relative error K u + that of the differences; half of it survives the square root
    dev = X - mean
    drel = K * U + 2 * (dmean + U * np.abs(dev)) * np.abs(dev).mean(axis=1, keepdims=True) * rstd ** 2 + 4 * U
    n = dev * rstd
    dn = (dmean + U * np.abs(dev)) * rstd + np.abs(n) * drel
    y = n * W + B
    ty = half(dtype) * np.abs(y) + dn * np.abs(W) + 3 * U * (np.abs(n * W) + np.abs(B)) + tiny(dtype)
    nr = (R - mean) * rstd
    dnr = (dmean + U * np.abs(R - mean)) * rstd + np.abs(nr) * drel
    t = G * W
    m = lambda v: v.mean(axis=1, keepdims=True)  # noqa: E731
    dx, dw, db = O.layer_norm_backward(G, R, W, mean, rstd)
    td = half(dtype) * np.abs(dx) + tiny(dtype) + np.abs(dx) * drel + rstd * (
        K * U * (np.abs(t) + m(np.abs(t)) + np.abs(nr) * m(np.abs(t * nr))) + dnr * np.abs(m(t * nr)) + np.abs(nr) * m(np.abs(t) * dnr))
    # the column sums: a workgroup's rows one after the other, then its lines, 16 apart, then 16 more
    L = 40 + rows / 16
    tw = half(wdtype) * np.abs(dw) + L * U * np.abs(G * nr).sum(axis=0) + (np.abs(G) * dnr).sum(axis=0) + tiny(wdtype)
    tb = half(wdtype) * np.abs(db) + L * U * np.abs(G).sum(axis=0) + tiny(wdtype)
    return y, ty, dx, td, dw, tw, db, tb


@pytest.mark.parametrize("dtype,wdtype", [(torch.float32, torch.float32), (torch.bfloat16, torch.bfloat16), (torch.bfloat16, torch.float32), (torch.float16, torch.float16),
                                          (torch.float16, torch.float32)])
@pytest.mark.parametrize("saved8", [False, True])
@pytest.mark.parametrize("rows,cols", NORM_SHAPES)
def test_layer_norm(dtype, wdtype, saved8, rows, cols):
    from spurfies_amd import ops

    pad = (cols % 3) * 3
    x = randn((rows, cols), dtype, cols, scale=1.5, shift=0.7, pad=pad).requires_grad_(True)
    w, b = randn((cols,), wdtype, 1, scale=0.3, shift=1.0).requires_grad_(True), randn((cols,), wdtype, 2).requires_grad_(True)
    g = randn((rows, cols), dtype, 3, pad=pad)
    y, ck = ops.layer_norm(x, w, b, eps=1e-5, saved8=saved8, out8=True)
    dx, dw, db = torch.autograd.grad(y, (x, w, b), g)
    assert y.dtype == dtype and dx.dtype == dtype and dw.dtype == wdtype and db.dtype == wdtype
    X, G, W, B = f64(x), f64(g), f64(w), f64(b)
    mean, rstd = O.statistics(X, 1e-5)
    R = O.restore(*O.pack(X), cols) if saved8 else X
    Y, ty, DX, td, DW, tw, DB, tb = norm_tolerances(X, G, W, B, R, mean, rstd, dtype, wdtype, rows)
    close(y, Y, ty, "y")
    close(dx, DX, td, "dx")
    close(dw, DW, tw, "dw")
    close(db, DB, tb, "db")
    same = ops.checkpoint8(y)
    assert torch.equal(ck.codes, same.codes) and torch.equal(ck.steps, same.steps)
    assert torch.equal(y, ops.layer_norm(x.detach(), w, b))                       # with nothing saved


@pytest.mark.parametrize("saved8", [False, True])
def test_layer_norm_of_many_rows(saved8):
    """More rows than workgroups: each walks over several, and adds their columns up."""
    from spurfies_amd import ops

    rows, cols = 9001, 136
    x = randn((rows, cols), torch.float32, 1, shift=-2.0).requires_grad_(True)
    w, b = randn((cols,), torch.float32, 2, shift=1.0).requires_grad_(True), randn((cols,), torch.float32, 3).requires_grad_(True)
    g = randn((rows, cols), torch.float32, 4)
    y = ops.layer_norm(x, w, b, saved8=saved8)
    got = torch.autograd.grad(y, (x, w, b), g)
    again = torch.autograd.grad(ops.layer_norm(x, w, b, saved8=saved8), (x, w, b), g)
    assert all(torch.equal(p, q) for p, q in zip(got, again))                     # the same bits
    X, G = f64(x), f64(g)
    mean, rstd = O.statistics(X, 1e-5)
    R = O.restore(*O.pack(X), cols) if saved8 else X
    Y, ty, DX, td, DW, tw, DB, tb = norm_tolerances(X, G, f64(w), f64(b), R, mean, rstd, torch.float32, torch.float32, rows)
    close(y, Y, ty, "y")
    for a, want, tol, what in zip(got, (DX, DW, DB), (td, tw, tb), ("dx", "dw", "db")):
        close(a, want, tol, what)


def test_layer_norm_gradient_against_differences():
    """The input's and the weight's gradient against central differences of the 64-bit forward: 64 columns, h = 1e-4 leaves h^2 times third derivatives
    (below 30 for rows of unit variance: < 3e-7) and the quotient of doubles; the kernel's own error is below 1e-5 here (K u M, M < 50)."""
    from spurfies_amd import ops

    x = randn((3, 64), torch.float32, 5).requires_grad_(True)
    w, b = randn((64,), torch.float32, 6, shift=1.0).requires_grad_(True), randn((64,), torch.float32, 7).requires_grad_(True)
    g = randn((3, 64), torch.float32, 8)
    dx, dw, db = torch.autograd.grad(ops.layer_norm(x, w, b), (x, w, b), g)
    X, W, B, G, h = f64(x), f64(w), f64(b), f64(g), 1e-4
    loss = lambda X, W, B: (O.layer_norm(X, W, B, 1e-5) * G).sum()  # noqa: E731
    for got, at in ((dx, 0), (dw, 1), (db, 2)):
        args = [X, W, B]
        diff = np.zeros_like(args[at])
        for i in np.ndindex(diff.shape):
            p, q = args[at].copy(), args[at].copy()
            p[i] += h
            q[i] -= h
            diff[i] = (loss(*[p if j == at else v for j, v in enumerate(args)]) - loss(*[q if j == at else v for j, v in enumerate(args)])) / (2 * h)
        close(got, diff, 2e-5, ("dx", "dw", "db")[at])


@pytest.mark.parametrize("make", [lambda x: x[0, 0], lambda x: x, lambda x: x.transpose(0, 2), lambda x: x[:, ::2], lambda x: x[:, :1].expand(4, 7, 40), lambda x: x[:0]])
def test_shapes_and_strides_of_rows(make):
    """One dimension, three, a transposed last one, skipped rows, broadcast rows, none: as the dense copy, gradients included."""
    from spurfies_amd import ops

    x = make(randn((4, 6, 40), torch.float32, 1)).detach()
    cols = x.shape[-1]
    w, b = randn((cols,), torch.float32, 2).requires_grad_(True), randn((cols,), torch.float32, 3).requires_grad_(True)
    m = randn((24, cols), torch.float32, 4).requires_grad_(True)
    g, h = randn(tuple(x.shape), torch.float32, 5), randn(tuple(x.shape[:-1]) + (24,), torch.float32, 6)
    got = []
    for v in (x, x.reshape(-1, cols).clone()):
        v = v.requires_grad_(True)
        for saved8 in (False, True):
            y = ops.layer_norm(v, w, b, saved8=saved8)
            got.append([y] + list(torch.autograd.grad(y, (v, w, b), g.view(y.shape))))
        y = ops.act8(v, "gelu")
        got.append([y] + list(torch.autograd.grad(y, v, g.view(y.shape))))
        y = ops.linear8(v, m)
        dx, dm = torch.autograd.grad(y, (v, m), h.view(y.shape))
        got.append([dm])
        assert dx.shape == v.shape and y.shape == v.shape[:-1] + (24,)
    for p, q in zip(got[:4], got[4:]):
        assert all(torch.equal(i.reshape(j.shape), j) for i, j in zip(p, q))


def test_layer_norm_without_parameters_and_partial_gradients():
    from spurfies_amd import ops

    x = randn((6, 100), torch.float32, 1).requires_grad_(True)
    w, b, g = randn((100,), torch.float32, 2).requires_grad_(True), randn((100,), torch.float32, 3).requires_grad_(True), randn((6, 100), torch.float32, 4)
    ones, zeros = torch.ones(100, device="cuda"), torch.zeros(100, device="cuda")
    assert torch.equal(ops.layer_norm(x), ops.layer_norm(x, ones, zeros)) and torch.equal(ops.layer_norm(x, w), ops.layer_norm(x, w, zeros))
    assert torch.equal(ops.layer_norm(x, None, b), ops.layer_norm(x, ones, b))
    full = torch.autograd.grad(ops.layer_norm(x, w, b), (x, w, b), g)
    assert torch.equal(torch.autograd.grad(ops.layer_norm(x, w.detach(), b.detach()), x, g)[0], full[0])
    assert torch.equal(torch.autograd.grad(ops.layer_norm(x.detach(), w, b.detach()), w, g)[0], full[1])
    assert torch.equal(torch.autograd.grad(ops.layer_norm(x.detach(), w.detach(), b), b, g)[0], full[2])
    assert torch.equal(torch.autograd.grad(ops.layer_norm(x), x, g)[0], torch.autograd.grad(ops.layer_norm(x, ones, zeros), x, g)[0])
    with torch.no_grad():
        assert not ops.layer_norm(x, w, b).requires_grad
    s = ops.layer_norm(x, w, b).sum()                                   # a gradient that is one broadcast number
    assert torch.equal(torch.autograd.grad(s, w)[0], torch.autograd.grad(ops.layer_norm(x, w, b), w, torch.ones_like(g))[0])


@pytest.mark.parametrize("cols", [40, 700, 5000, 20000])
def test_layer_norm_rows_that_are_not_finite_stay_alone(cols):
    from spurfies_amd import ops

    x = randn((5, cols), torch.float32, 1)
    x[1, 3], x[3, cols - 1] = float("nan"), float("inf")
    x[4] = 2.5                                                            # no variance
    y = ops.layer_norm(x, eps=1e-5)
    assert torch.isnan(y[1]).all() and torch.isnan(y[3]).all() and (y[4] == 0).all()
    assert torch.equal(y[[0, 2]], ops.layer_norm(x[[0, 2]].contiguous(), eps=1e-5))


def test_layer_norm_far_from_zero():
    """Rows with a mean of 1000 times their deviation: the mean is taken out before the squares, so the variance keeps its digits."""
    from spurfies_amd import ops

    x = randn((7, 300), torch.float32, 1, shift=1000.0)
    X = f64(x)
    mean, rstd = O.statistics(X, 0.0)
    y = ops.layer_norm(x, eps=0.0)
    # the mean's error (K u 1000) moves every element alike; relative to the deviation of one: 32 * 6e-8 * 1000 = 2e-3, and its square in the variance
    close(y, (X - mean) * rstd, 32 * U * 1000 * rstd + 1e-4, "y")


def test_nothing_is_written_behind_a_row():
    """Through the library itself: outputs of a wider row stride, whose gaps keep their values."""
    from spurfies_amd import _lib

    l, s = _lib.lib(), _lib.stream_ptr()
    for cols in (1, 33, 515, 2049, 17000):
        x = randn((3, cols), torch.float32, cols)
        out = torch.full((3, cols + 7), -9.0, device="cuda")
        mean, rstd = torch.empty(3, device="cuda"), torch.empty(3, device="cuda")
        gap = torch.full((3, 7), -9.0, device="cuda")
        _lib.check(l.spf_layer_norm_forward(_lib.ptr(x), 0, cols, 3, cols, None, None, 0, 1e-5, _lib.ptr(out), cols + 7, _lib.ptr(mean), _lib.ptr(rstd), None, None, None, None, s))
        assert torch.equal(out[:, cols:], gap)
        out.fill_(-9.0)
        _lib.check(l.spf_layer_norm_backward(_lib.ptr(x), 0, cols, 3, cols, _lib.ptr(x), cols, None, None, _lib.ptr(mean), _lib.ptr(rstd), None, 0, _lib.ptr(out), cols + 7, None,
                                             None, 0, None, s))
        assert torch.equal(out[:, cols:], gap)
        out.fill_(-9.0)
        _lib.check(l.spf_act8_forward(_lib.ptr(x), 0, cols, 3, cols, 2, 0.0, _lib.ptr(out), cols + 7, None, None, None, None, s))
        assert torch.equal(out[:, cols:], gap)


# ---- weight gradients -------------------------------------------------------------------------------------------------------------------
WGRAD_SHAPES = [(1, 1, 1), (1, 8, 33), (3, 64, 64), (17, 65, 31), (63, 5, 200), (64, 130, 129), (65, 256, 256), (100, 257, 300), (1237, 131, 515), (513, 40, 1000),
                (4100, 300, 140), (700, 512, 40)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,n,k", WGRAD_SHAPES)
def test_wgrad8(dtype, rows, n, k):
    from spurfies_amd import ops

    a, g = randn((rows, k), dtype, 1), randn((rows, n), dtype, 2, pad=3)
    ck = ops.checkpoint8(a)
    dw, db = ops.wgrad8(g, ck)
    A, G = O.restore(*O.pack(f64(a)), k), f64(g)
    # products are exact; a chain has at most one (truncating: 2 u) rounding for each of the up to three pieces of a row, and 64 more where splits meet
    L = 2 * (3 * rows + 64)
    close(dw, G.T @ A, L * U * (np.abs(G).T @ np.abs(A)), "dw")
    close(db, G.sum(axis=0), (rows + 64) * U * np.abs(G).sum(axis=0), "db")
    # typical errors grow with the root of the chain: hold the whole to that too (a lost piece of a gradient would be 2^-9 or 2^-16 of it)
    err = np.linalg.norm(f64(dw) - G.T @ A) / max(np.linalg.norm(G.T @ A), 1e-30)
    assert err < 2 * U * 8 * np.sqrt(3 * rows + 64), err


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,n,k", [(66001, 256, 130), (66001, 256, 256), (7400, 520, 515), (3300, 1030, 800), (100003, 257, 511), (20011, 127, 129), (9000, 1001, 97),
                                      (2500, 2049, 1030)])
def test_wgrad8_of_large_layers(dtype, rows, n, k):
    """The wide tiles, with and without split rows and with ragged edges; the restored input is the kernels' own (tested byte for byte above)."""
    from spurfies_amd import ops

    a, g = randn((rows, k), dtype, 1), randn((rows, n), dtype, 2)
    ck = ops.checkpoint8(a)
    dw, db = ops.wgrad8(g, ck)
    A, G = f64(ck.restore(torch.float32)), f64(g)
    want = G.T @ A
    # 2 u sqrt(chain) of sqrt(rows) times the factors' sizes (1 each): the spread of a sum of independent roundings, held to eight of it
    close(dw, want, 8 * 2 * U * np.sqrt(3 * rows) * np.sqrt(rows) * 2, "dw")
    close(db, G.sum(axis=0), 8 * U * np.sqrt(rows) * np.sqrt(rows) * 2, "db")
    assert np.linalg.norm(f64(dw) - want) < 2 * U * 8 * np.sqrt(3 * rows + 64) * np.linalg.norm(want)
    assert all(torch.equal(p, q) for p, q in zip((dw, db), ops.wgrad8(g, ck)))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,n,k", [(1, 3, 5), (64, 70, 96), (97, 256, 256), (130, 300, 131), (900, 64, 64), (800, 2050, 2050)])
def test_wgrad8_is_exact_for_whole_numbers(dtype, rows, n, k):
    """Inputs with as many digits as their type has and sums that fit 24 bits: nothing may round, so every piece of every gradient has to arrive."""
    from spurfies_amd import ops

    rng = np.random.default_rng(rows)
    bits = {torch.float32: 23, torch.float16: 11, torch.bfloat16: 8}[dtype]
    if dtype == torch.float32:
        # full 23-bit numbers in one row of each column, elsewhere zero: a column's sum is one product with a = +-1
        G = np.zeros((rows, n))
        G[rng.integers(0, rows, n), np.arange(n)] = rng.integers(2 ** 22, 2 ** 23, n) * rng.choice([-1, 1], n)
        A = rng.choice([-1.0, 1.0], (rows, k))
    else:
        G = rng.integers(-(2 ** bits) + 1, 2 ** bits, (rows, n)).astype(float)
        A = rng.integers(-7, 8, (rows, k)).astype(float)                    # 900 * 2048 * 7 < 2^24
    a, g = torch.tensor(A, device="cuda").to(dtype), torch.tensor(G, device="cuda").to(dtype)
    assert np.array_equal(f64(a), A) and np.array_equal(f64(g), G)
    dw, db = ops.wgrad8(g, ops.checkpoint8(a))
    assert np.array_equal(f64(dw), G.T @ A) and np.array_equal(f64(db), G.sum(axis=0))


def test_wgrad8_places_every_row_and_column():
    """One non-zero element of g and one of a at a time, over tile, stage and block borders."""
    from spurfies_amd import ops

    rows, n, k = 131, 260, 290
    for m in (0, 7, 8, 15, 16, 31, 32, 63, 64, 130):
        for i, j in ((0, 0), (31, 32), (32, 31), (127, 128), (128, 127), (255, 256), (256, 255), (259, 289), (5, 7), (40, 9)):
            a, g = torch.zeros(rows, k, device="cuda"), torch.zeros(rows, n, device="cuda")
            a[m, j], g[m, i] = 0.75, 3.0
            dw, db = ops.wgrad8(g, ops.checkpoint8(a))
            want = torch.zeros(n, k, device="cuda")
            want[i, j] = 2.25
            assert torch.equal(dw, want) and float(db[i]) == 3.0 and float(db.sum()) == 3.0, (m, i, j)


@pytest.mark.parametrize("wdtype", TYPES)
def test_wgrad8_adds_into_given_tensors(wdtype):
    from spurfies_amd import ops

    a, g = randn((300, 70), torch.float32, 1), randn((300, 50), torch.float32, 2)
    ck = ops.checkpoint8(a)
    dw, db = ops.wgrad8(g, ck)
    w0, b0 = randn((50, 70), wdtype, 3), randn((50,), wdtype, 4)
    w, b = w0.clone(), b0.clone()
    r = ops.wgrad8(g, ck, out=w, dbias=b)
    assert r[0] is w and r[1] is b
    assert torch.equal(w, (w0.float() + dw).to(wdtype)) and torch.equal(b, (b0.float() + db).to(wdtype))
    w = w0.clone()
    assert ops.wgrad8(g, ck, out=w)[1] is None and torch.equal(w, (w0.float() + dw).to(wdtype))
    assert ops.wgrad8(g, ck, bias=False)[1] is None and torch.equal(ops.wgrad8(g, ck, bias=False)[0], dw)


def test_wgrad8_strides_shapes_and_nothing():
    from spurfies_amd import ops

    a, g = randn((6, 10, 70), torch.float32, 1), randn((6, 10, 50), torch.float32, 2)
    dw, db = ops.wgrad8(g, ops.checkpoint8(a))
    flat = ops.wgrad8(g.reshape(60, 50), ops.checkpoint8(a.reshape(60, 70)))
    assert torch.equal(dw, flat[0]) and torch.equal(db, flat[1])
    e = g[0, :1].expand(60, 50)
    assert all(torch.equal(p, q) for p, q in zip(ops.wgrad8(e, ops.checkpoint8(a)), ops.wgrad8(e.contiguous(), ops.checkpoint8(a))))
    t = randn((50, 60), torch.float32, 3).t()
    assert all(torch.equal(p, q) for p, q in zip(ops.wgrad8(t, ops.checkpoint8(a)), ops.wgrad8(t.contiguous(), ops.checkpoint8(a))))
    dw, db = ops.wgrad8(torch.empty(0, 50, device="cuda"), ops.checkpoint8(torch.empty(0, 70, device="cuda")))
    assert dw.shape == (50, 70) and not dw.any() and not db.any()
    dw, db = ops.wgrad8(torch.empty(4, 0, device="cuda"), ops.checkpoint8(torch.empty(4, 70, device="cuda")))
    assert dw.shape == (0, 70) and db.shape == (0,)


def test_wgrad8_values_that_are_not_finite_are_loud():
    from spurfies_amd import ops

    a, g = randn((40, 70), torch.float32, 1), randn((40, 50), torch.float32, 2)
    ok = ops.wgrad8(g, ops.checkpoint8(a))[0]
    bad = a.clone()
    bad[7, 33] = float("inf")
    dw, db = ops.wgrad8(g, ops.checkpoint8(bad))
    assert torch.isnan(dw[:, 32:64]).all() and torch.equal(dw[:, :32], ok[:, :32]) and torch.equal(dw[:, 64:], ok[:, 64:]) and torch.isfinite(db).all()
    for v in (float("nan"), float("inf"), float("-inf")):
        h = g.clone()
        h[5, 9] = v
        dw, db = ops.wgrad8(h, ops.checkpoint8(a))
        assert not torch.isfinite(dw[9]).any() and not torch.isfinite(db[9]) and torch.isfinite(dw[:9]).all() and torch.isfinite(dw[10:]).all()


# ---- together ---------------------------------------------------------------------------------------------------------------------------
def block(x, p, kind):
    """A residual MLP block every saved tensor of which is in 8 bits."""
    from spurfies_amd import ops

    y, y8 = ops.layer_norm(x, p["g"], p["b"], saved8=True, out8=True)
    h = ops.linear8(y, p["w1"], p["b1"], saved=y8)
    a, a8 = ops.act8(h, kind, out8=True)
    return x + ops.linear8(a, p["w2"], p["b2"], saved=a8), (y, h, a)


def block_params(width, hidden, dtype):
    mk = lambda shape, s, scale, shift=0.0: randn(shape, dtype, s, scale=scale, shift=shift).requires_grad_(True)  # noqa: E731
    return {"g": mk((width,), 1, 0.2, 1.0), "b": mk((width,), 2, 0.2), "w1": mk((hidden, width), 3, width ** -0.5), "b1": mk((hidden,), 4, 0.1),
            "w2": mk((width, hidden), 5, hidden ** -0.5), "b2": mk((width,), 6, 0.1)}


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("kind", ["leaky_relu", "gelu"])
def test_block_gradients(dtype, kind):
    """Each gradient of a block against the 64-bit formulas, fed with the block's own forward values (so that no code of a saved activation can round the
    other way); the products in between are the library's, whose 16-bit results count their rounding."""
    rows, width, hidden = 210, 72, 160
    x = randn((rows, width), dtype, 9).requires_grad_(True)
    p = block_params(width, hidden, dtype)
    out, (y, h, a) = block(x, p, kind)
    g = randn((rows, width), dtype, 10)
    names = list(p)
    grads = dict(zip(["x"] + names, torch.autograd.grad(out, [x] + [p[k] for k in names], g)))
    q = lambda v: O.restore(*O.pack(v), v.shape[1])  # noqa: E731
    X, Y, H, A, G = (f64(t) for t in (x, y, h, a, g))
    P = {k: f64(v) for k, v in p.items()}
    want = {"b2": G.sum(0), "w2": G.T @ q(A)}
    dA = G @ P["w2"]
    dH = dA * O.act_slope(kind, q(A if kind == "leaky_relu" else H), 0.01)
    want["b1"], want["w1"] = dH.sum(0), dH.T @ q(Y)
    dY = dH @ P["w1"]
    mean, rstd = O.statistics(X, 1e-5)
    dX, want["g"], want["b"] = O.layer_norm_backward(dY, q(X), P["g"], mean, rstd)
    want["x"] = dX + G
    # in norm: every stage multiplies by operators of norm about one and rounds once in `dtype` (three stages, then the sum; h each) or keeps 32 bits with
    # chains of at most 210 terms
    for k, v in want.items():
        err = np.linalg.norm(f64(grads[k]) - v) / np.linalg.norm(v)
        assert err < 6 * half(dtype) + 256 * U, (k, err)


def test_block_trains_in_captured_steps():
    """One whole training pass of the block as a captured graph: replays on new inputs give the eager pass' bits, with eager work in between; a second graph of
    the same shapes replayed between them shares nothing with the first."""
    rows, width, hidden = 300, 64, 96
    p = {k: v.detach().requires_grad_(True) for k, v in block_params(width, hidden, torch.float32).items()}

    def grads(x, g):
        out, _ = block(x, p, "leaky_relu")
        return (out.detach(),) + torch.autograd.grad(out, [p[k] for k in p], g)

    xs = [randn((rows, width), torch.float32, 20 + i) for i in range(4)]
    gs = [randn((rows, width), torch.float32, 30 + i) for i in range(4)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for i in range(2):
            grads(xs[0], gs[0])
    torch.cuda.current_stream().wait_stream(side)
    graphs = []
    for _ in range(2):
        x, g = xs[0].clone(), gs[0].clone()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            res = grads(x, g)
        graphs.append((graph, x, g, res))
    for i in range(4):
        want = [grads(xs[(i + j) % 4], gs[(i + j) % 4]) for j in range(2)]
        for j, (graph, x, g, _) in enumerate(graphs):
            x.copy_(xs[(i + j) % 4])
            g.copy_(gs[(i + j) % 4])
        for graph, *_ in graphs:
            graph.replay()
        torch.cuda.synchronize()
        for (_, _, _, res), w in zip(graphs, want):
            assert all(torch.equal(a, b) for a, b in zip(res, w)), i


def test_operators_on_two_streams_at_once():
    """Workspaces belong to a call: passes of two streams that overlap give what they give alone."""
    rows, width, hidden = 4000, 256, 256
    p = block_params(width, hidden, torch.float32)
    x = [randn((rows, width), torch.float32, 40 + i) for i in range(2)]
    g = [randn((rows, width), torch.float32, 50 + i) for i in range(2)]

    def grads(i):
        out, _ = block(x[i], p, "gelu")
        return torch.autograd.grad(out, [p[k] for k in p], g[i])

    want = [grads(0), grads(1)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = [[], []]
    for _ in range(3):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(grads(i))
    torch.cuda.synchronize()
    for i in range(2):
        for r in got[i]:
            assert all(torch.equal(a, b) for a, b in zip(r, want[i]))


def test_gradients_go_into_their_sinks():
    """Parameters with gradient sinks (sync-free steps): the backward passes add to .grad and hand autograd nothing."""
    from spurfies_amd import ops

    p = block_params(64, 96, torch.float32)
    x, g = randn((50, 64), torch.float32, 1), randn((50, 64), torch.float32, 2)
    want = torch.autograd.grad(block(x, p, "silu")[0], list(p.values()), g)
    for v in p.values():
        v.grad = torch.full_like(v, 0.5)
    ops.set_grad_sinks(p.values())
    try:
        block(x, p, "silu")[0].backward(g)
    finally:
        ops.set_grad_sinks(p.values(), on=False)
    for (k, v), w in zip(p.items(), want):
        assert torch.equal(v.grad, 0.5 + w), k


def test_linear8_under_autocast_and_with_frozen_parameters():
    from spurfies_amd import ops

    x, w, b = randn((60, 96), torch.float32, 1).requires_grad_(True), randn((40, 96), torch.float32, 2).requires_grad_(True), randn((40,), torch.float32, 3).requires_grad_(True)
    g = randn((60, 40), torch.float32, 4)
    want = torch.autograd.grad(ops.linear8(x, w, b), (x, w, b), g)
    with torch.autocast("cuda", dtype=torch.bfloat16):
        y = ops.linear8(x, w, b)
    assert y.dtype == torch.float32 and all(torch.equal(p, q) for p, q in zip(torch.autograd.grad(y, (x, w, b), g), want))
    assert torch.equal(torch.autograd.grad(ops.linear8(x, w.detach(), b.detach()), x, g)[0], want[0])
    assert torch.equal(torch.autograd.grad(ops.linear8(x.detach(), w, b.detach()), w, g)[0], want[1])
    assert torch.equal(torch.autograd.grad(ops.linear8(x.detach(), w.detach(), b), b, g)[0], want[2])
    assert torch.equal(torch.autograd.grad(ops.linear8(x.view(3, 20, 96), w), w, g.view(3, 20, 40))[0], want[1])


def test_saved8_keeps_a_quarter_and_forgets_the_input():
    """What a block keeps between its passes: one byte an element of every layer's input (and 1 / 32), not four; the inputs may be overwritten."""
    from spurfies_amd import ops

    x, g = randn((512, 256), torch.float32, 1), randn((512, 256), torch.float32, 2)
    w = randn((256, 256), torch.float32, 3, scale=0.06).requires_grad_(True)
    gamma = torch.ones(256, device="cuda", requires_grad=True)
    want = torch.autograd.grad(ops.linear8(ops.act8(ops.layer_norm(x, gamma, saved8=True), "gelu"), w), (gamma, w), g)
    x2 = x.clone()
    n = ops.layer_norm(x2, gamma, saved8=True)
    a = ops.act8(n, "gelu")
    out = ops.linear8(a, w)
    with torch.no_grad():
        for t in (x2, n, a):
            t.fill_(float("nan"))
    got = torch.autograd.grad(out, (gamma, w), g)
    assert all(torch.equal(p, q) for p, q in zip(got, want))


def test_gpu_refusals():
    from spurfies_amd import ops

    x = torch.zeros(4, 32, device="cuda")
    with pytest.raises(ValueError, match="float32"):
        ops.layer_norm(x.double())
    with pytest.raises(ValueError, match="shape"):
        ops.layer_norm(x, torch.ones(31, device="cuda"))
    with pytest.raises(ValueError, match="type"):
        ops.layer_norm(x, torch.ones(32, device="cuda", dtype=torch.bfloat16))
    with pytest.raises(ValueError, match="type"):
        ops.layer_norm(x.bfloat16(), torch.ones(32, device="cuda"), torch.ones(32, device="cuda", dtype=torch.bfloat16))
    with pytest.raises(ValueError, match="GPU"):
        ops.layer_norm(x, torch.ones(32))
    with pytest.raises(ValueError, match="eps"):
        ops.layer_norm(x, eps=-1e-5)
    with pytest.raises(ValueError, match="dimension"):
        ops.layer_norm(torch.zeros((), device="cuda"))
    with pytest.raises(ValueError, match="none of"):
        ops.act8(x, "tanh")
    with pytest.raises(ValueError, match="no parameter"):
        ops.act8(x, "silu", 1.0)
    with pytest.raises(ValueError, match="slope"):
        ops.act8(x, "leaky_relu", -0.1)
    with pytest.raises(ValueError, match="beta"):
        ops.act8(x, "softplus", 0.0)
    ck = ops.checkpoint8(x)
    with pytest.raises(ValueError, match="rows"):
        ops.wgrad8(torch.zeros(5, 8, device="cuda"), ck)
    with pytest.raises(ValueError, match="Checkpoint8"):
        ops.wgrad8(x, x)
    with pytest.raises(ValueError, match="without out"):
        ops.wgrad8(x, ck, dbias=torch.zeros(32, device="cuda"))
    with pytest.raises(ValueError, match="contiguous"):
        ops.wgrad8(x, ck, out=torch.zeros(32, 33, device="cuda")[:, :32])
    with pytest.raises(ValueError, match="no columns"):
        ops.wgrad8(x, ops.checkpoint8(torch.zeros(4, 0, device="cuda")))
    with pytest.raises(ValueError, match="share one type"):
        ops.linear8(x, torch.zeros(8, 32, device="cuda", dtype=torch.float16))
    with pytest.raises(ValueError, match="Checkpoint8 of x"):
        ops.linear8(x, torch.zeros(8, 32, device="cuda"), saved=ops.checkpoint8(torch.zeros(5, 32, device="cuda")))
    with pytest.raises(ValueError, match="Checkpoint8 of x"):
        ops.linear8(x, torch.zeros(8, 32, device="cuda"), saved=x)
    with pytest.raises(ValueError, match="devices"):
        ops.linear8(x, torch.zeros(8, 32))
    x.requires_grad_(True)
    w = torch.zeros(8, 32, device="cuda")
    for y in (ops.act8(x, "silu"), ops.layer_norm(x), ops.linear8(x, w)):
        with pytest.raises(RuntimeError, match="not differentiable"):
            torch.autograd.grad(y.sum(), x, create_graph=True)
