"""CPU: how the training operators with 8-bit saved activations stand in autograd — forward mode, gradients that nobody asked for, autocast.  The kernels do
not run: the library's calls are replaced by nothing, or not reached."""
import pytest
import torch
import torch.autograd.forward_ad as fwAD

from spurfies_amd import _lib, ops


@pytest.fixture
def no_kernels(monkeypatch):
    """Tensors on the CPU pass as the GPU's, and the library's calls are only written down."""
    calls = []
    monkeypatch.setattr(ops, "_type_of", lambda t, who: ops._TYPES[t.dtype])
    monkeypatch.setattr(_lib, "call", lambda name, device, *args: calls.append((name,) + args))
    return calls


@pytest.mark.parametrize("grad", [True, False])
def test_forward_mode_derivatives_are_refused(no_kernels, grad):
    """A dual tensor needs no gradient and has a data pointer: without a refusal its tangent would be dropped."""
    x, w, b = torch.randn(4, 32), torch.randn(32), torch.randn(32)
    with fwAD.dual_level(), torch.set_grad_enabled(grad):
        d, dw = fwAD.make_dual(x, torch.ones_like(x)), fwAD.make_dual(w, torch.ones_like(w))
        for call in (lambda: ops.act8(d, "silu"), lambda: ops.act8(d, "gelu", out8=True), lambda: ops.layer_norm(d, w, b), lambda: ops.layer_norm(x, dw, b),
                     lambda: ops.layer_norm(x, w, dw, saved8=True)):
            with pytest.raises(RuntimeError, match="forward-mode"):
                call()
        assert not no_kernels
        ops.layer_norm(x, w, b)                                              # plain tensors pass
        ops.act8(x, "silu")
        assert len(no_kernels) == 2
        # linear8 without a graph is the library's product, which has the derivative
        m = torch.randn(8, 32)
        assert torch.equal(fwAD.unpack_dual(ops.linear8(d, m)).tangent, torch.ones_like(x) @ m.t())
        if grad:
            with pytest.raises(RuntimeError):
                ops.linear8(d, m.requires_grad_(True))


@pytest.mark.parametrize("function", ["_Act8", "_LayerNorm"])
def test_no_gradients_are_made_for_the_8_bit_forms(no_kernels, monkeypatch, function):
    """With out8 a layer's codes and steps are outputs without a gradient: autograd must not fill zeros of their size for the backward pass."""
    seen = []
    original = getattr(ops, function)

    class Spy(original):
        @staticmethod
        def backward(ctx, *grads):
            seen.append(grads)
            return original.backward(ctx, *grads)

    monkeypatch.setattr(ops, function, Spy)
    x = torch.randn(4, 64, requires_grad=True)
    y, ck = ops.act8(x, "gelu", out8=True) if function == "_Act8" else ops.layer_norm(x, out8=True)
    torch.autograd.grad(y, x, torch.ones_like(y))
    assert len(seen) == 1 and seen[0][0] is not None and seen[0][1:] == (None, None)


def test_linear8_backward_keeps_its_type_under_autocast():
    """The engine carries the caller's autocast state into the backward pass (here the CPU's, with frozen parameters: no kernel is reached)."""
    x, w, g = torch.randn(5, 64, requires_grad=True), torch.randn(8, 64), torch.randn(5, 8)
    y = ops._Linear8.apply(x, w, None, None, None)
    with torch.autocast("cpu", dtype=torch.bfloat16):
        dx, = torch.autograd.grad(y, x, g)
    assert dx.dtype == torch.float32 and torch.equal(dx, g @ w)


def test_linear8_with_only_the_bias_to_train_saves_nothing_of_the_input(no_kernels):
    x, w, b = torch.randn(5, 64), torch.randn(8, 64), torch.randn(8, requires_grad=True)
    y = ops.linear8(x, w, b)
    assert not no_kernels and all(t is None or t.dtype != torch.uint8 for t in y.grad_fn.saved_tensors)
    y.backward(torch.ones_like(y))
    assert [c[0] for c in no_kernels] == ["spf_wgrad8_bias"]


def test_wgrad8_refuses_results_that_share_memory(no_kernels):
    ck = ops.Checkpoint8(torch.zeros(4, 32, dtype=torch.uint8), torch.ones(4, 1, dtype=torch.uint8), 1)
    out = torch.zeros(8, 1)
    with pytest.raises(ValueError, match="share"):
        ops.wgrad8(torch.zeros(4, 8), ck, out=out, dbias=out.view(8))
    assert not no_kernels


def test_wgrad8_marks_what_it_adds_into_as_changed(no_kernels):
    """A graph that saved the tensor before has to notice."""
    ck = ops.Checkpoint8(torch.zeros(4, 32, dtype=torch.uint8), torch.ones(4, 1, dtype=torch.uint8), 32)
    out, db, t = torch.zeros(8, 32), torch.zeros(8), torch.ones(8, 32, requires_grad=True)
    y = (out * t).sum() + (db * t[:, 0]).sum()
    before = out._version, db._version
    ops.wgrad8(torch.zeros(4, 8), ck, out=out, dbias=db)
    assert out._version > before[0] and db._version > before[1]
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward()


def test_rows_of_lazily_negated_tensors():
    """torch's imaginary part of a conjugate is a view whose memory holds the other sign."""
    x = torch.randn(4, 32)
    z = torch.complex(x, -x).conj()
    for t in (z.imag, torch._neg_view(x), torch._neg_view(x)[:, :1], torch._neg_view(x)[0]):
        assert t.is_neg()
        m, ld = ops._rows_of(t, "test")
        assert not m.is_neg() and torch.equal(m, t.reshape(-1, t.shape[-1]).clone())
        assert torch.equal(torch.as_strided(m, m.shape, (ld, 1), m.storage_offset()), m)


def test_lazily_negated_parameters_and_results_are_refused(no_kernels):
    x, w, ck = torch.randn(4, 32), torch.randn(32), ops.Checkpoint8(torch.zeros(4, 32, dtype=torch.uint8), torch.ones(4, 1, dtype=torch.uint8), 32)
    with pytest.raises(ValueError, match="negated"):
        ops.layer_norm(x, torch._neg_view(w))
    with pytest.raises(ValueError, match="negated"):
        ops.wgrad8(x, ck, out=torch._neg_view(torch.zeros(32, 32)))
    assert not no_kernels


def test_parameters_beyond_the_kernels_32_bits_are_wrong_arguments(no_kernels):
    x = torch.randn(4, 32)
    for call in (lambda: ops.act8(x, "softplus", 1e-60), lambda: ops.act8(x, "softplus", 1e60), lambda: ops.act8(x, "leaky_relu", 1e60), lambda: ops.layer_norm(x, eps=1e60)):
        with pytest.raises(ValueError):
            call()
    assert not no_kernels
    ops.layer_norm(x, eps=torch.tensor(1e-5))
    ops.act8(x, "leaky_relu", 1)
    assert len(no_kernels) == 2
