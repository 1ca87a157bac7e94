"""What the lean training operators' autograd functions hand to the library, and their plans, without a GPU: the library's
calls are recorded in place of being made."""
import pytest
import torch

from reversability_b200 import _lib, functional as fn, functions as fx


@pytest.fixture
def recorded(monkeypatch):
    """Calls of the library as (name, arguments); CPU tensors stand for device tensors."""
    calls = []
    monkeypatch.setattr(fn, "require_cuda", lambda *t, **k: None)
    monkeypatch.setattr(fn, "_on_current_device", lambda *t: None)
    monkeypatch.setattr(_lib, "stream_ptr", lambda device=None: 0)
    monkeypatch.setattr(_lib, "call", lambda name, *args: calls.append((name, args)))
    return calls


@pytest.mark.parametrize("shape,cut,dtype", [((40, 768), 256, torch.bfloat16), ((5, 6, 96), 32, torch.float32)])
def test_layer_norm_backward_takes_the_stride_of_the_tensor_it_gets(recorded, shape, cut, dtype):
    """Hooks on saved tensors (offloading ones, say) hand rows back side by side where the forward's were further apart."""
    x = torch.randn(*shape).to(dtype)[..., :cut].requires_grad_()
    w = torch.ones(cut).requires_grad_()
    assert fn.even_rows(x)[3] == shape[-1]  # read where it lies
    with torch.autograd.graph.saved_tensors_hooks(lambda t: t.detach(),
                                                  lambda t: t.clone(memory_format=torch.contiguous_format)):
        y = fx.layer_norm(x, w)
    assert recorded[-1][0] == "rk_layernorm_fwd" and recorded[-1][1][2] == shape[-1]
    y.backward(torch.zeros_like(y))
    name, args = recorded[-1]
    assert name == "rk_layernorm_bwd"
    rows = x.numel() // cut
    assert args[2] == cut and args[8] == cut and args[10] == cut and args[15:17] == (rows, cut)


def test_layer_norm_backward_refuses_saved_tensors_of_other_sizes(recorded):
    """Hooks that return something else than they were given are an error, not a read behind an array's end."""
    x = torch.randn(8, 16, requires_grad=True)
    with torch.autograd.graph.saved_tensors_hooks(lambda t: t.detach(), lambda t: t[:1]):
        y = fx.layer_norm(x, torch.ones(16))
    with pytest.raises(ValueError):
        y.backward(torch.zeros_like(y))
    assert recorded[-1][0] == "rk_layernorm_fwd"
