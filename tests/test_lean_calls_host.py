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


def test_head_loss_workspace_holds_what_the_call_writes():
    """dz of a piece and the gathered rows; sums of dx only with dx; tiles of dW only with dW, and not the whole of it."""
    lib, MB, NO_DX, NO_DW = _lib.lib(), 1 << 20, 2, 4
    for M, V, K in ((256, 128256, 8192), (1024, 151936, 4096), (4096, 131072, 4096), (14848, 50257, 256), (32768, 50257, 1024)):
        both, no_dx, no_dw, none = (lib.rk_linear_ce_bwd_workspace(M, V, K, f) for f in (0, NO_DX, NO_DW, NO_DX | NO_DW))
        rows, tiles = -(-M // 256) * 256, -(-V // 256)
        dz = min(512 * MB, rows * tiles * 512)
        gathered = rows * K * 2
        assert none <= dz + gathered + rows * 8 + MB
        assert 0 < both - no_dx == no_dw - none <= 16 * rows * K * 4  # whole slices of dx
        assert (both - no_dx) % (rows * K * 4) == 0
        assert 0 < both - no_dw == no_dx - none <= 128 * MB or (both - no_dw) % (256 * K * 4) == 0 and both - no_dw <= 512 * MB
        assert lib.rk_linear_ce_bwd_workspace(M, V, K, 1) == both + V * K * 2 + -V * K * 2 % 1024
    assert lib.rk_linear_ce_bwd_workspace(256, 128256, 8192, 0) < 256 * MB  # where dW itself takes 2 GB


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_head_loss_backward_refuses_what_the_forward_did_not_keep(recorded, dtype):
    """kept, weight and gradient of other sizes would be read behind their ends."""
    x, w, up = torch.zeros(6, 8, dtype=dtype), torch.zeros(11, 8, dtype=dtype), torch.ones(())
    kept = torch.zeros(6, dtype=torch.int64) if dtype == torch.float32 else torch.zeros(4 + 4 * 6, dtype=torch.int32)
    for bad, match in ((lambda: fn.linear_ce_bwd(x, w, kept[:-1], up), "kept"),
                       (lambda: fn.linear_ce_bwd(x, w, kept.float(), up), "kept"),
                       (lambda: fn.linear_ce_bwd(x[:5], w, kept, up), "kept"),
                       (lambda: fn.linear_ce_bwd(x, w[:, :4], kept, up), "weight"),
                       (lambda: fn.linear_ce_bwd(x, w.double(), kept, up), "share a type"),
                       (lambda: fn.linear_ce_bwd(x, w, kept, up, "max"), "reduction"),
                       (lambda: fn.linear_ce_bwd(x, w, kept, up, "none"), "one a row"),
                       (lambda: fn.linear_ce_bwd(x, w, kept, torch.ones(6)), "one number")):
        with pytest.raises(ValueError, match=match):
            bad()
    assert not recorded
    if dtype != torch.float32:
        fn.linear_ce_bwd(x, w, kept, up)
        assert recorded[-1][0] == "rk_linear_ce_bwd"
