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


def test_linear8_backward_keeps_its_type_under_autocast():
    """The engine carries the caller's autocast state into the backward pass (here the CPU's, with frozen parameters: no kernel is reached)."""
    x, w, g = torch.randn(5, 64, requires_grad=True), torch.randn(8, 64), torch.randn(5, 8)
    y = ops._Linear8.apply(x, w, None, None, None)
    with torch.autocast("cpu", dtype=torch.bfloat16):
        dx, = torch.autograd.grad(y, x, g)
    assert dx.dtype == torch.float32 and torch.equal(dx, g @ w)
