"""Host-side behaviour of layer norm, dropout and the head loss in pieces: refusals of CPU tensors and of invalid C
arguments, before any CUDA call."""
import pytest
import torch

from reversability_b200 import _lib, functions as fx, optimized


def test_cpu_tensors_are_refused():
    x, w, y = torch.zeros(3, 8), torch.zeros(5, 8), torch.zeros(3, dtype=torch.int64)
    for call in (lambda: fx.layer_norm(x), lambda: fx.layer_norm(x, torch.ones(8)), lambda: fx.dropout(x, 0.1, 0),
                 lambda: fx.dropout(x.requires_grad_(), 0.1, 0, training=False), lambda: fx.linear_cross_entropy(x, w, y),
                 lambda: optimized.head_pieces_backward(x, w, y, 1, torch.float32)):
        with pytest.raises(ValueError, match="CUDA"):
            call()


def test_layer_norm_entries_reject_bad_arguments():
    lib = _lib.lib()

    def fwd(x=64, xd=1, ldx=8, pd=0, y=64, yd=1, ldy=8, stats=None, rows=2, width=8):
        return lib.rk_layernorm_fwd(x, xd, ldx, None, None, pd, y, yd, ldy, stats, rows, width, 1e-5, None)
    assert fwd(rows=0, x=None, y=None) == 0
    assert fwd(x=None) == 1 and fwd(ldx=7) == 1 and fwd(ldy=7) == 1 and fwd(rows=-1) == 1 and fwd(width=0) == 1
    assert fwd(xd=1, yd=2) == 3 and fwd(xd=9) == 3 and fwd(pd=5) == 3
    assert fwd(width=16385, ldx=16385, ldy=16385) == 5
    assert fwd(stats=68) == 2
    assert fwd(y=66) == 2 and fwd(ldy=9) == 2 and fwd(x=65) == 2  # rows that are not equally far from a boundary

    def bwd(stats=64, dy=64, lddy=8, dx=64, lddx=8, dw=64, ws=64, size=1 << 30, rows=2):
        return lib.rk_layernorm_bwd(64, 1, 8, None, 0, stats, dy, 1, lddy, dx, lddx, dw, None, ws, size, rows, 8, None)
    assert bwd(stats=None) == 1 and bwd(dy=None) == 1 and bwd(lddx=7) == 1 and bwd(stats=68) == 2
    assert bwd(ws=None) == 6 and bwd(size=lib.rk_layernorm_bwd_workspace(2, 8) - 1) == 6
    assert bwd(dy=66) == 2 and bwd(lddx=9) == 2
    assert bwd(dx=None, dw=None) == 0  # nothing is wanted
    assert lib.rk_layernorm_bwd_workspace(0, 8) == 0
    for rows, width in ((1, 1), (100000, 1024), (100000, 1020), (5, 16384)):
        assert lib.rk_layernorm_bwd_workspace(rows, width) >= 8 * width


def test_dropout_entry_rejects_bad_arguments():
    lib = _lib.lib()

    def drop(x=64, xd=1, res=None, y=64, yd=1, n=8, p=0.5, seed_dev=None):
        return lib.rk_dropout(x, xd, res, y, yd, n, p, 1, seed_dev, 0, None)
    assert drop(n=0, x=None, y=None) == 0
    assert drop(x=None) == 1 and drop(n=-1) == 1 and drop(p=-0.1) == 1 and drop(p=1.1) == 1 and drop(p=float("nan")) == 1
    assert drop(xd=1, yd=2) == 3 and drop(xd=0, yd=1, res=64) == 3 and drop(xd=7) == 3
    assert drop(seed_dev=68) == 2


def test_head_loss_entries_reject_bad_arguments():
    lib = _lib.lib()
    kept, need, back = lib.rk_linear_ce_kept(9), lib.rk_linear_ce_fwd_workspace(9, 300, 40, 0), lib.rk_linear_ce_bwd_workspace(9, 300, 40, 0)
    assert kept >= 9 * 16 and need > 0 and back > 9 * 600
    assert lib.rk_linear_ce_fwd_workspace(9, 300, 40, 1) >= need + 300 * 80
    assert lib.rk_linear_ce_bwd_workspace(9, 300, 40, 1) >= back + 300 * 80

    def fwd(x=64, ldh=40, w=64, ldw=40, y=64, M=9, V=300, K=40, dtype=1, red=2, loss=64, kept=64, ws=256, size=need):
        return lib.rk_linear_ce_fwd(x, ldh, w, ldw, y, -100, M, V, K, dtype, red, loss, kept, ws, size, None)
    assert fwd(dtype=0) == 3 and fwd(dtype=5) == 3
    assert fwd(x=None) == 1 and fwd(w=None) == 1 and fwd(y=None) == 1 and fwd(loss=None) == 1 and fwd(kept=None) == 1
    assert fwd(ldh=39) == 1 and fwd(ldw=39) == 1 and fwd(V=0) == 1 and fwd(K=0) == 1 and fwd(M=-1) == 1 and fwd(red=3) == 1
    assert fwd(M=1 << 26) == 1 and fwd(V=1 << 30) == 1
    assert fwd(kept=68) == 2 and fwd(x=65) == 2 and fwd(w=65) == 2 and fwd(ws=64) == 2
    assert fwd(ws=None) == 6 and fwd(size=need - 1) == 6 and fwd(w=66) == 6  # a weight that has to be copied needs more

    def bwd(grad=64, dx=64, lddx=40, dxd=1, dw=64, lddw=40, dwd=1, red=2, ws=256, size=back):
        return lib.rk_linear_ce_bwd(64, 40, 64, 40, 64, 9, 300, 40, 1, red, grad, dx, lddx, dxd, dw, lddw, dwd, ws, size, None)
    assert bwd(grad=None) == 1 and bwd(lddx=39) == 1 and bwd(lddw=39) == 1 and bwd(red=-1) == 1
    assert bwd(dxd=4) == 3 and bwd(dwd=4) == 3
    assert bwd(ws=None) == 6 and bwd(size=back - 1) == 6 and bwd(ws=128) == 2
    assert bwd(dx=None, dw=None) == 0  # nothing is wanted


def test_head_loss_workspace_is_bounded():
    """dz of a piece takes 512 MB at most, whatever the vocabulary, unless one 256-column tile needs more."""
    lib = _lib.lib()
    for M, V, K in ((14848, 50257, 256), (32768, 50257, 1024), (32768, 1 << 20, 64), (4096, 131072, 4096)):
        rows = -(-M // 256) * 256
        other = 16 * rows * (K + 4) * 4 + 16 * (1 << 29) // (2 * rows) * (K + 4) * 4  # fp32 slices of both gradients
        assert lib.rk_linear_ce_bwd_workspace(M, V, K, 0) < (1 << 29) + other + rows * (2 * K + 64)
    assert lib.rk_linear_ce_bwd_workspace(1 << 22, 1000, 8, 0) >= (1 << 22) * 512
