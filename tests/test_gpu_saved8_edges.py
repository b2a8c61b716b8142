"""The training operators with 8-bit saved activations at the edges of what their documentation allows: far arguments, values that are not finite, autocast,
shared parameters, sizes beyond a launch's limits, and shapes that reach every form of the kernels.  Tolerances count roundings: u = 2^-24, half(type) = finfo.eps / 2."""
import numpy as np
import pytest
import torch

from oracle import saved8 as O

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
TYPES = [torch.float32, torch.bfloat16, torch.float16]


def half(dtype):
    return torch.finfo(dtype).eps / 2


def tiny(dtype):
    """the spacing of the type's smallest numbers"""
    return torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps


def f64(t):
    return t.detach().double().cpu().numpy()


def randn(shape, dtype, seed, scale=1.0, shift=0.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(*shape, generator=g) * scale + shift).to(dtype).cuda()


def close(got, want, tol, what):
    got = f64(got) if torch.is_tensor(got) else got
    assert got.shape == want.shape, (what, got.shape, want.shape)
    bad = ~(np.abs(got - want) <= tol)
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.size} off, worst {np.nanmax(np.abs(got - want) / np.maximum(tol, 1e-300)):.3g} times the tolerance"


# ---- activations far from zero ----------------------------------------------------------------------------------------------------------
def passes(x, kind, param):
    """y, dx for a gradient of ones, and the 64-bit values of x and of its restored 8-bit form"""
    from spurfies_amd import ops

    x = x.requires_grad_(True)
    y = ops.act8(x, kind, param=param)
    dx, = torch.autograd.grad(y, x, torch.ones_like(y))
    return y, dx, f64(x), O.restore(*O.pack(f64(x)), x.shape[1])


@pytest.mark.parametrize("dtype", TYPES)
def test_silu_is_exact_to_its_last_digits_wherever_it_lies(dtype):
    """Relative to the result.  e^-|x| has the hardware's 2 u and up to 5 u around it; 1 + it, its inverse and three products another 7 (fp32: K = 14); 16-bit results
    take the exponential of a rounded product, 1.3 |x| u more.  The hardware's 2^t has nothing below the smallest normal number: 2^-126 of it, times x."""
    x = torch.linspace(-100.0, 20.0, 64 * 96).view(64, 96).to(dtype).cuda()
    y, dx, X, R = passes(x, "silu", None)
    k = lambda z: 14 + (0 if dtype == torch.float32 else 2 * np.abs(z))  # noqa: E731
    with np.errstate(over="ignore"):
        s, o = 1 / (1 + np.exp(-X)), 1 / (1 + np.exp(X))
        close(y, X * s, (half(dtype) + k(X) * U) * np.abs(X * s) + np.abs(X) * 2.0 ** -126 + tiny(dtype), "y")
        s, o = 1 / (1 + np.exp(-R)), 1 / (1 + np.exp(R))
    # the slope's two terms, s and s x (1 - s)
    close(dx, s * (1 + R * o), half(dtype) * np.abs(s * (1 + R * o)) + 2 * k(R) * U * s * (1 + np.abs(R) * o) + (1 + np.abs(R)) * 2.0 ** -126 + tiny(dtype), "dx")


@pytest.mark.parametrize("dtype", TYPES)
def test_softplus_is_exact_to_its_last_digits_wherever_it_lies(dtype):
    """As SiLU, with z = beta x: its rounding counts |z| u unless it is carried along (fp32); the logarithm adds 4 u, 1 / beta and the sum 3."""
    beta = 100.0
    x = torch.linspace(-0.85, 0.3, 64 * 96).view(64, 96).to(dtype).cuda()
    y, dx, X, R = passes(x, "softplus", beta)
    k = lambda z: 21 + (0 if dtype == torch.float32 else 3 * np.abs(z))  # noqa: E731
    want = np.logaddexp(0.0, beta * X) / beta
    close(y, want, (half(dtype) + k(beta * X) * U) * want + 2.0 ** -126 + tiny(dtype), "y")
    want = 1 / (1 + np.exp(-beta * R))
    close(dx, want, (half(dtype) + k(beta * R) * U) * want + 2.0 ** -126 + tiny(dtype), "dx")


@pytest.mark.parametrize("dtype", TYPES)
def test_softplus_of_values_whose_product_with_beta_overflows(dtype):
    """beta x beyond fp32's range: y is x, and nothing on the other side."""
    from spurfies_amd import ops

    big = float(torch.finfo(dtype).max)
    x = torch.tensor([[big, -big, big / 2, 1.0] * 8]).to(dtype).cuda()
    y = ops.act8(x, "softplus", param=1e38)
    assert torch.equal(y, x.clamp(min=0))


@pytest.mark.parametrize("dtype", TYPES)
def test_gelu_is_exact_to_its_last_digits_wherever_it_lies(dtype):
    """Relative to the result, also in the far negative tail.  fp32: the approximation of the tail is off by 0.4 u, the exponential beside it by 7, eight steps of the
    polynomial, an inverse and three products by another 12 (K = 20).  16-bit results: an approximation within 15 u, an exponential off by x^2 / 2 * 1.3 u."""
    x = torch.linspace(-12.5, 6.0, 64 * 96).view(64, 96).to(dtype).cuda()
    y, dx, X, R = passes(x, "gelu", None)
    from scipy.special import erfc

    k = lambda z: 20 + (0 if dtype == torch.float32 else 15 + z * z)  # noqa: E731
    cdf = lambda z: 0.5 * erfc(-z / np.sqrt(2))  # noqa: E731
    close(y, X * cdf(X), (half(dtype) + k(X) * U) * np.abs(X * cdf(X)) + np.abs(X) * 2.0 ** -126 + tiny(dtype), "y")
    bell = R * np.exp(-R * R / 2) / np.sqrt(2 * np.pi)
    close(dx, cdf(R) + bell, half(dtype) * np.abs(cdf(R) + bell) + k(R) * U * (cdf(R) + np.abs(bell)) + (1 + np.abs(R)) * 2.0 ** -126 + tiny(dtype), "dx")


def test_gelu_in_32_bits_is_as_exact_as_its_formula():
    """Near zero, where the inputs are: 0.5 x (1 + erf(x / sqrt 2)) in fp32 has the roundings of the product, erf (2 u), the sum and two more; a cdf of a half to within
    1.5 u of one, i.e. 3 u of the result, and one for the last product."""
    x = randn((512, 256), torch.float32, 5, scale=0.3)
    y, _, X, _ = passes(x, "gelu", None)
    from scipy.special import erfc

    want = X * 0.5 * erfc(-X / np.sqrt(2))
    assert np.linalg.norm(f64(y) - want) < 1.0 * U * np.linalg.norm(want)          # (independent roundings: their root mean square)
    close(y, want, 5 * U * np.abs(want) + tiny(torch.float32), "y")


@pytest.mark.parametrize("dtype", TYPES)
def test_bytes_of_blocks_that_are_not_finite(dtype):
    """The sign bit says "not greater than zero" there as well: a NaN, of either sign, is not."""
    from spurfies_amd import ops

    nan, inf = float("nan"), float("inf")
    x = torch.tensor([[nan, 1.0, -1.0, 0.0] * 16, [inf, -inf, 2.0, -2.0] * 16, [1.0] * 40 + [nan] * 24]).to(dtype).cuda()
    x[2, 50:] = -x[2, 50:]
    ck = ops.checkpoint8(x)
    codes, steps = O.pack(f64(x))
    assert np.array_equal(ck.steps.cpu().numpy(), steps) and np.array_equal(ck.codes.cpu().numpy(), codes)
    # LayerNorm's and the activations' 8-bit forms are written by the same code
    for form in (ops.layer_norm(x, out8=True), ops.act8(x, "leaky_relu", out8=True)):
        assert torch.equal(form[1].codes, ops.checkpoint8(form[0]).codes)
        assert np.array_equal(form[1].codes.cpu().numpy(), O.pack(f64(form[0]))[0])


# ---- linear8 ----------------------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_linear8_keeps_its_type_where_the_backward_pass_runs_under_autocast(dtype):
    from spurfies_amd import ops

    x, w, b = randn((60, 96), dtype, 1).requires_grad_(True), randn((40, 96), dtype, 2).requires_grad_(True), randn((40,), dtype, 3).requires_grad_(True)
    g = randn((60, 40), dtype, 4)
    want = torch.autograd.grad(ops.linear8(x, w, b), (x, w, b), g)
    for other in (torch.bfloat16, torch.float16):
        with torch.autocast("cuda", dtype=other):
            got = torch.autograd.grad(ops.linear8(x, w, b), (x, w, b), g)
        assert all(p.dtype == dtype and torch.equal(p, q) for p, q in zip(got, want))


# ---- sizes beyond a launch's 2^32 work-items --------------------------------------------------------------------------------------------
def _room(gigabytes):
    torch.cuda.empty_cache()
    if torch.cuda.mem_get_info()[0] < gigabytes * 1e9:
        pytest.skip(f"needs {gigabytes} GB of GPU memory")


def test_wgrad8_adds_into_more_than_2_31_outputs():
    from spurfies_amd import ops

    _room(24)
    n, k = 1 << 18, 8200
    g = randn((3, n), torch.bfloat16, 1)
    ck = ops.checkpoint8(randn((3, k), torch.bfloat16, 2))
    out, db = torch.ones(n, k, dtype=torch.bfloat16, device="cuda"), torch.zeros(n, dtype=torch.bfloat16, device="cuda")
    ops.wgrad8(g, ck, out=out, dbias=db)
    for rows in (slice(0, 300), slice(n // 2, n // 2 + 300), slice(n - 300, n)):
        part, dpart = torch.ones(300, k, dtype=torch.bfloat16, device="cuda"), torch.zeros(300, dtype=torch.bfloat16, device="cuda")
        ops.wgrad8(g[:, rows].contiguous(), ck, out=part, dbias=dpart)
        assert torch.equal(out[rows], part) and torch.equal(db[rows], dpart)
    del out, part
    torch.cuda.empty_cache()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_layer_norm_of_many_wide_rows(dtype):
    """The widest form's rows come out as they do in small batches."""
    from spurfies_amd import ops

    rows, cols = 16384 + 37, 16385
    x = randn((64, cols), dtype, 1)
    big = x.repeat(-(-rows // 64), 1)[:rows]
    w, b = randn((cols,), dtype, 2), randn((cols,), dtype, 3)
    big.requires_grad_(True)
    y = ops.layer_norm(big, w, b)
    dx, = torch.autograd.grad(y, big, big.detach())
    x.requires_grad_(True)
    y0 = ops.layer_norm(x, w, b)
    d0, = torch.autograd.grad(y0, x, x.detach())
    for i in range(0, rows, 64):
        n = min(64, rows - i)
        assert torch.equal(y[i:i + n], y0[:n]) and torch.equal(dx[i:i + n], d0[:n]), i


def test_layer_norm_of_more_than_2_22_wide_rows():
    """Through the library, with broadcast inputs: 2^22 rows of 1024 threads each are 2^32 threads."""
    from spurfies_amd import _lib

    rows, cols = (1 << 22) + 3, 8200
    _room(80)
    l, s = _lib.lib(), _lib.stream_ptr()
    x, g = randn((1, cols), torch.bfloat16, 1), randn((1, cols), torch.bfloat16, 2)
    mean, rstd = torch.full((rows,), 0.25, device="cuda"), torch.full((rows,), 1.5, device="cuda")
    dx, one = torch.zeros(rows, cols, dtype=torch.bfloat16, device="cuda"), torch.empty(1, cols, dtype=torch.bfloat16, device="cuda")
    for out, n in ((dx, rows), (one, 1)):
        _lib.check(l.spf_layer_norm_backward(_lib.ptr(g), 1, 0, n, cols, _lib.ptr(x), 0, None, None, _lib.ptr(mean), _lib.ptr(rstd), None, 1, _lib.ptr(out), cols, None, None, 0,
                                             None, s))
    for i in (0, 1, 1 << 20, (1 << 22) - 1, 1 << 22, rows - 1):
        assert torch.equal(dx[i], one[0]), i
    del dx
    torch.cuda.empty_cache()


def test_layer_norm_parameter_gradients_of_more_than_2_28_columns():
    """Each column's sum, the last ones' too: 64 columns a workgroup of 1024 threads are a launch's 2^32 threads at 2^28."""
    from spurfies_amd import _lib

    cols = (1 << 28) + 1000
    _room(12)
    l, s = _lib.lib(), _lib.stream_ptr()
    x, g = torch.randint(-3, 4, (cols,), device="cuda").float()[None], torch.randint(-3, 4, (cols,), device="cuda").float()[None]
    mean, rstd = torch.full((1,), 1.0, device="cuda"), torch.full((1,), 0.5, device="cuda")
    dw, db = torch.full((cols,), 9.0, device="cuda"), torch.full((cols,), 9.0, device="cuda")
    ws = torch.empty(l.spf_layer_norm_workspace_floats(1, cols), device="cuda")
    _lib.check(l.spf_layer_norm_backward(_lib.ptr(g), 0, cols, 1, cols, _lib.ptr(x), cols, None, None, _lib.ptr(mean), _lib.ptr(rstd), None, 0, None, cols, _lib.ptr(dw), _lib.ptr(db), 0,
                                         _lib.ptr(ws), s))
    assert torch.equal(db, g[0]) and torch.equal(dw, (g * ((x - 1) * 0.5))[0])               # small whole numbers and halves: nothing rounds
    del ws
    torch.cuda.empty_cache()


# ---- gradients into shared or partial places --------------------------------------------------------------------------------------------
def test_one_parameter_as_weight_and_bias_with_a_sink():
    """The same tensor twice: both gradients arrive in its .grad."""
    from spurfies_amd import ops

    x, g = randn((500, 96), torch.float32, 1), randn((500, 96), torch.float32, 2)
    p = randn((96,), torch.float32, 3).requires_grad_(True)
    q, r = p.detach().clone().requires_grad_(True), p.detach().clone().requires_grad_(True)
    dq, dr = torch.autograd.grad(ops.layer_norm(x, q, r), (q, r), g)
    p.grad = torch.full_like(p, 0.5)
    ops.set_grad_sinks([p])
    try:
        ops.layer_norm(x, p, p).backward(g)
    finally:
        ops.set_grad_sinks([p], on=False)
    # 0.5, dw and db added in one order or another: two roundings of sums no larger than their magnitudes'
    want = 0.5 + f64(dq) + f64(dr)
    close(p.grad, want, 3 * U * (0.5 + np.abs(f64(dq)) + np.abs(f64(dr))), "grad")


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,n", [(1, 1), (7, 3), (1000, 40), (33, 515), (70001, 256), (9, 9001)])
def test_linear8_with_only_the_bias_to_train(dtype, rows, n):
    """A column sum: nothing of the input is packed or kept, and no weight gradient is formed."""
    from spurfies_amd import ops

    x, w = randn((rows, 64), dtype, 1), randn((n, 64), dtype, 2, scale=0.1)
    b = randn((n,), dtype, 3).requires_grad_(True)
    g = randn((rows, n + 5), dtype, 4)[:, :n]
    y = ops.linear8(x, w, b)
    assert all(t is None or t.dtype != torch.uint8 for t in y.grad_fn.saved_tensors)
    db, = torch.autograd.grad(y, b, g, retain_graph=True)
    G = f64(g)
    # a chain of at most one addition a row, 64 where splits meet, and the last rounding
    tol = half(dtype) * np.abs(G.sum(0)) + (rows + 64) * U * np.abs(G).sum(0) + tiny(dtype)
    assert db.dtype == dtype
    close(db, G.sum(0), tol, "db")
    # independent roundings: a thread's chain of at most 128 rows, the splits and their sum each leave a few u of the root of the rows
    assert np.linalg.norm(f64(db) - G.sum(0)) < (half(dtype) + 8 * U) * np.linalg.norm(G.sum(0)) + 8 * U * np.sqrt(rows) * np.sqrt(n) + tiny(dtype)
    # the same bits as beside a weight gradient
    v = w.detach().clone().requires_grad_(True)
    assert torch.equal(db, torch.autograd.grad(ops.linear8(x, v, b), (v, b), g)[1])
    b.grad = torch.full_like(b, 2.0)
    ops.set_grad_sinks([b])
    try:
        z = ops.linear8(x, w, b)
        z.backward(g)
    finally:
        ops.set_grad_sinks([b], on=False)
    close(b.grad, 2.0 + G.sum(0), half(dtype) * np.abs(2.0 + G.sum(0)) + (rows + 66) * U * (2 + np.abs(G).sum(0)) + tiny(dtype), "sink")


def test_linear8_with_only_the_bias_to_train_in_a_captured_step():
    from spurfies_amd import ops

    x, w = randn((5000, 64), torch.float32, 1), randn((300, 64), torch.float32, 2)
    b = randn((300,), torch.float32, 3).requires_grad_(True)
    gs = [randn((5000, 300), torch.float32, 10 + i) for i in range(3)]
    want = [torch.autograd.grad(ops.linear8(x, w, b), b, h)[0] for h in gs]
    c, g = b.detach().clone().requires_grad_(True), gs[0].clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        torch.autograd.grad(ops.linear8(x, w, c), c, g)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        db, = torch.autograd.grad(ops.linear8(x, w, c), c, g)
    for h, d in zip(gs, want):
        g.copy_(h)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(db, d)
        torch.randn(1000, device="cuda").sum().item()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,n,k", [(300000, 256, 256), (8192, 1024, 1024), (4100, 300, 140), (40, 7, 64), (1000, 2000, 2000)])
def test_bias_gradient_by_itself_in_every_plan(dtype, rows, n, k):
    """Wide, middle and narrow tiles, split rows and not: the bits of the call that forms the weight gradient as well."""
    from spurfies_amd import ops

    g = randn((rows, n), dtype, 1)
    want = ops.wgrad8(g, ops.checkpoint8(randn((rows, k), dtype, 2)))[1]
    db = torch.empty_like(want)
    ops._wgrad8_bias_into(g, n, k, db, False)
    assert torch.equal(db, want)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,n", [(33, 40), (40, 5), (64, 260), (70001, 128)])
def test_wgrad8_bias_gradient_of_infinities(dtype, rows, n):
    """db is the column's sum: an infinity stays one, in whichever row it is; both signs together, or a NaN, give NaN.  The weight gradient is not finite there."""
    from spurfies_amd import ops

    inf, nan = float("inf"), float("nan")
    ck = ops.checkpoint8(randn((rows, 70), dtype, 1))
    for m in (0, 5, 31, 32, rows - 2, rows - 1):
        g = randn((rows, n), dtype, 2)
        g[m, 0], g[m, 1], g[m, 2], g[m - 1, 2], g[m, n - 1] = inf, -inf, inf, -inf, nan
        dw, db = ops.wgrad8(g, ck)
        db = f64(db)
        assert db[0] == inf and db[1] == -inf and np.isnan(db[2]) and np.isnan(db[n - 1]) and np.isfinite(db[3:n - 1]).all(), m
        assert not torch.isfinite(dw[[0, 1, 2, n - 1]]).any() and torch.isfinite(dw[3:n - 1]).all()


# ---- every form of the kernels ----------------------------------------------------------------------------------------------------------
def tile(rows, n, k, dtype):
    from spurfies_amd import _lib, ops

    return _lib.lib().spf_wgrad8_tile(rows, n, k, ops._TYPES[dtype])


# split rows and not, tiles that the layer does not fill: a last piece of one and of seven columns, rows that do not fill a stage
WIDE = [(389017, 256, 256), (5000, 2049, 2051), (5003, 2055, 2050), (1900, 4091, 4085)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,n,k", WIDE)
def test_wgrad8_with_the_widest_tiles(dtype, rows, n, k):
    from spurfies_amd import ops

    assert tile(rows, n, k, dtype) == 256
    a, g = randn((rows, k), dtype, 1), randn((rows, n), dtype, 2)
    ck = ops.checkpoint8(a)
    dw, db = ops.wgrad8(g, ck)
    A, G = ck.restore(torch.float32).double(), g.double()
    want, sums = f64(G.t() @ A), f64(G.sum(0))
    # independent roundings of a chain of three piece products a row (each up to 2 u of sums of about the root of the rows), held to eight times their spread
    close(dw, want, 8 * 2 * U * np.sqrt(3 * rows) * np.sqrt(rows) * 2, "dw")
    close(db, sums, 8 * U * rows * 2, "db")
    assert np.linalg.norm(f64(dw) - want) < 2 * U * 8 * np.sqrt(3 * rows + 64) * np.linalg.norm(want)
    assert all(torch.equal(p, q) for p, q in zip((dw, db), ops.wgrad8(g, ck)))
    out, dbias = torch.ones_like(dw), torch.ones_like(db)
    ops.wgrad8(g, ck, out=out, dbias=dbias)
    assert torch.equal(out, 1 + dw) and torch.equal(dbias, 1 + db)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,n,k", [(5000, 2049, 2051), (1900, 4091, 4085)])
def test_wgrad8_with_the_widest_tiles_is_exact_for_whole_numbers(dtype, rows, n, k):
    """Sums within 24 bits do not round: every piece of every element has to arrive in its place."""
    from spurfies_amd import ops

    assert tile(rows, n, k, dtype) == 256
    gen = torch.Generator(device="cuda").manual_seed(rows)
    ints = lambda low, high, *shape: torch.randint(low, high, shape, generator=gen, device="cuda").double()  # noqa: E731
    A = ints(0, 2, rows, k) * 2 - 1
    if dtype == torch.float32:
        G = torch.zeros(rows, n, dtype=torch.float64, device="cuda")       # one number of 23 bits a column
        G[torch.randint(0, rows, (n,), generator=gen, device="cuda"), torch.arange(n, device="cuda")] = ints(2 ** 22, 2 ** 23, n)
    else:
        bits = 8 if dtype == torch.bfloat16 else 11                        # 5000 * 2047 < 2^24
        G = ints(1 - 2 ** bits, 2 ** bits, rows, n)
    a, g = A.to(dtype), G.to(dtype)
    assert torch.equal(a.double(), A) and torch.equal(g.double(), G)
    dw, db = ops.wgrad8(g, ops.checkpoint8(a))
    assert torch.equal(dw.double(), G.t() @ A) and torch.equal(db.double(), G.sum(0))


@pytest.mark.parametrize("saved8", [False, True])
@pytest.mark.parametrize("dtype,rows,cols", [(torch.float32, 2003, 1030), (torch.float32, 2003, 4099), (torch.float32, 2003, 8192), (torch.bfloat16, 4001, 1500), (torch.bfloat16, 4001, 4096),
                                             (torch.float16, 2003, 8191), (torch.float32, 150, 9001), (torch.bfloat16, 150, 9001), (torch.bfloat16, 150, 17003)])
def test_layer_norm_of_many_rows_of_several_waves(dtype, rows, cols, saved8):
    """Workgroups that walk over rows whose threads meet in LDS, and the column sums of rows that are read again: each row as it comes out alone, the columns as in 64 bits."""
    from spurfies_amd import ops

    x = randn((rows, cols), dtype, cols, scale=1.5, shift=0.7).requires_grad_(True)
    w, b = randn((cols,), dtype, 1, scale=0.3, shift=1.0).requires_grad_(True), randn((cols,), dtype, 2).requires_grad_(True)
    g = randn((rows, cols), dtype, 3)
    y, ck = ops.layer_norm(x, w, b, saved8=saved8, out8=True)
    dx, dw, db = torch.autograd.grad(y, (x, w, b), g, retain_graph=True)
    assert all(torch.equal(p, q) for p, q in zip((dx, dw, db), torch.autograd.grad(y, (x, w, b), g)))
    assert torch.equal(ck.codes, ops.checkpoint8(y).codes) and torch.equal(ck.steps, ops.checkpoint8(y).steps)
    for i in range(0, rows, 50):                                            # (a batch of 50 rows has a workgroup for each)
        v = x[i:i + 50].detach().requires_grad_(True)
        z = ops.layer_norm(v, w.detach(), b.detach(), saved8=saved8)
        assert torch.equal(z, y[i:i + 50]) and torch.equal(torch.autograd.grad(z, v, g[i:i + 50])[0], dx[i:i + 50]), i
    X, G = x.detach().double(), g.double()
    R = ops.checkpoint8(x).restore(torch.float32).double() if saved8 else X
    mean = X.mean(1, keepdim=True)
    rstd = 1 / torch.sqrt(((X - mean) ** 2).mean(1, keepdim=True) + 1e-5)
    n = (R - mean) * rstd
    # the mean and the deviation from chains of K roundings, n from those; the columns from chains of at most rows / 16 + 64
    K, L = 32 + cols / 2048, 64 + rows / 16
    dmean = K * U * X.abs().mean(1, keepdim=True)
    dn = (dmean + U * (R - mean).abs()) * rstd + n.abs() * (K * U + 2 * (dmean + U * (X - mean).abs().mean(1, keepdim=True)) * rstd + 4 * U)
    for got, want, size, what in ((dw, (G * n).sum(0), L * U * (G * n).abs().sum(0) + (G.abs() * dn).sum(0), "dw"), (db, G.sum(0), L * U * G.abs().sum(0), "db")):
        close(got, f64(want), half(dtype) * np.abs(f64(want)) + f64(size) + tiny(dtype), what)
