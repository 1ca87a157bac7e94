"""Layer norm, dropout and the head loss in the calls around them: saved-tensor hooks, forward-mode derivatives, labels and
gradients that are not numbers to count with, several pieces of the vocabulary."""
import pytest
import torch
from test_norm_dropout_gpu import _check as _check_norm  # with the tolerances derived there
from test_linear_ce_gpu import E, HALF_ULP, _check as _check_head, _inputs  # the same
from torch.autograd import forward_ad

from reversability_b200 import ModelConfig, ReversibleLM, _lib, alignment, functional as fn, functions as fx, optimized, optimized_v3

pytestmark = pytest.mark.gpu
DEV = "cuda"
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("rows,width,pitch", [(300, 256, 768), (37, 1000, 1024), (9, 20, 24)])
def test_layer_norm_of_spaced_rows_offloaded_to_the_host(rows, width, pitch, dtype):
    """What is saved comes back from the host with rows side by side: the same gradients as without the detour."""
    g = torch.Generator(device=DEV).manual_seed(0)
    x = torch.randn(rows, pitch, generator=g, device=DEV).to(dtype)[:, :width].requires_grad_()
    w = torch.randn(width, generator=g, device=DEV).requires_grad_()
    b = torch.randn(width, generator=g, device=DEV).requires_grad_()
    dy = torch.randn(rows, width, generator=g, device=DEV).to(dtype)
    y = fx.layer_norm(x, w, b)
    want = torch.autograd.grad(y, (x, w, b), dy)
    with torch.autograd.graph.save_on_cpu():
        z = fx.layer_norm(x, w, b)
    got = torch.autograd.grad(z, (x, w, b), dy)
    assert torch.equal(y, z) and all(torch.equal(s, t) for s, t in zip(got, want))


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_head_loss_and_dropout_offloaded_to_the_host(dtype):
    """The same for the other two: wide hidden rows, a transposed weight, a seed on the device."""
    x = torch.randn(70, 96, device=DEV).to(dtype)[:, :64].requires_grad_()
    w = torch.randn(64, 500, device=DEV).to(dtype).t().requires_grad_()
    y = torch.randint(0, 500, (70,), device=DEV)
    seed = torch.tensor(3, device=DEV)

    def step():
        loss = fx.linear_cross_entropy(fx.dropout(x, 0.3, seed), w, y)
        return loss
    want = torch.autograd.grad(step(), (x, w))
    with torch.autograd.graph.save_on_cpu():
        loss = step()
    assert all(torch.equal(s, t) for s, t in zip(torch.autograd.grad(loss, (x, w)), want))
    assert fn is not None and _lib.device_status() == 0


def test_forward_mode_derivatives_are_refused():
    """A tangent is not dropped without a word, with gradients recorded or not, whichever input carries it."""
    x, w, y = torch.randn(4, 16, device=DEV), torch.ones(16, device=DEV), torch.randint(0, 9, (4,), device=DEV)
    head, b16 = torch.randn(9, 16, device=DEV), x.to(BF16)
    for calls, like in (((lambda t: fx.layer_norm(t, w), lambda t: fx.dropout(t, 0.5, 3), lambda t: fx.dropout(x, 0.5, 3, residual=t),
                          lambda t: fx.linear_cross_entropy(t, head, y)), x),
                        ((lambda t: fx.linear_cross_entropy(t, head.to(BF16), y),), b16),
                        ((lambda t: fx.layer_norm(x, t), lambda t: fx.layer_norm(x, w, t)), w),
                        ((lambda t: fx.linear_cross_entropy(x, t, y),), head)):
        for call in calls:
            for mode in (torch.enable_grad, torch.no_grad):
                with forward_ad.dual_level(), mode():
                    call(like)  # without a tangent: as ever
                    with pytest.raises(RuntimeError, match="forward"):
                        call(forward_ad.make_dual(like, torch.ones_like(like)))


def test_forward_mode_derivatives_of_token_losses_are_refused():
    """The same for the losses on token log-probabilities: a tangent on the logits or on a constant."""
    z, y, ref = torch.randn(4, 6, 20, device=DEV), torch.randint(0, 20, (4, 6), device=DEV), torch.randn(4, 6, device=DEV)
    for call, like, match in ((lambda t: alignment.token_logprobs(t, y), z, "forward"),
                              (lambda t: alignment.policy_loss(t, y, ref, ref), z, "forward"),
                              (lambda t: alignment.policy_loss(z, y, ref, t), ref, "constant"),
                              (lambda t: alignment.preference_loss(t, y, ref), z, "forward"),
                              (lambda t: alignment.preference_loss(z, y, t), ref, "constant")):
        with forward_ad.dual_level(), torch.no_grad():
            call(like)
            with pytest.raises((RuntimeError, ValueError), match=match):
                call(forward_ad.make_dual(like, torch.ones_like(like)))


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("ignore,bad", [(-100, (100, -3)), (7, (-100, 1 << 40)), (-1, (-100, -2))])
def test_labels_outside_the_vocabulary_set_the_status(dtype, ignore, bad):
    """In every type, whichever number is the ignored one; the ignored one alone sets nothing."""
    x = torch.randn(200, 16, device=DEV).to(dtype).requires_grad_()
    w = torch.randn(100, 16, device=DEV).to(dtype).requires_grad_()
    y = torch.randint(0, 100, (200,), device=DEV)
    y[3] = y[60] = ignore
    wrong = y.clone()
    wrong[9], wrong[150] = bad
    y[9] = y[150] = ignore
    assert _lib.device_status() == 0
    want = fx.linear_cross_entropy(x, w, y, ignore_index=ignore)
    assert _lib.device_status() == 0
    got = fx.linear_cross_entropy(x, w, wrong, ignore_index=ignore)
    assert _lib.device_status() == 4  # RK_DEV_CE_LABEL
    assert torch.equal(got, want)
    for a, b in zip(torch.autograd.grad(got, (x, w)), torch.autograd.grad(want, (x, w))):
        assert torch.equal(a, b)
    assert _lib.device_status() == 0


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
def test_ignored_rows_have_zero_gradients_under_an_infinite_weight(dtype):
    x = torch.randn(70, 32, device=DEV).to(dtype).requires_grad_()
    w = torch.randn(90, 32, device=DEV).to(dtype)
    w[5, 0], w[6, 1] = float("inf"), -float("inf")
    y = torch.randint(10, 90, (70,), device=DEV)
    y[::3] = -100
    dx, = torch.autograd.grad(fx.linear_cross_entropy(x, w, y), x)
    assert not dx[::3].any()


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("reduction", ["none", "sum", "mean"])
@pytest.mark.parametrize("K", [32, 27])
def test_no_row_counts_under_a_gradient_that_is_no_number(dtype, reduction, K):
    """Zeros, as there is nothing to multiply (a weight gradient stored at once, and one from slices)."""
    x, w = torch.randn(300, K, device=DEV).to(dtype).requires_grad_(), torch.randn(90, K, device=DEV).to(dtype).requires_grad_()
    y = torch.full((300,), -100, device=DEV)
    for bad in (float("inf"), float("nan")):
        loss = fx.linear_cross_entropy(x, w, y, reduction=reduction)
        assert not any(t.any() for t in torch.autograd.grad(loss, (x, w), torch.full_like(loss, bad)))


def test_an_infinite_gradient_of_one_row_leaves_the_others():
    """fp16, a gradient a row: the common scale is that of the finite ones, so theirs do not overflow beside an infinite one."""
    x, w = torch.randn(40, 32, device=DEV).to(F16).requires_grad_(), torch.randn(50, 32, device=DEV).to(F16).requires_grad_()
    y = torch.randint(0, 50, (40,), device=DEV)
    g = torch.full((40,), 300.0, device=DEV)
    want, = torch.autograd.grad(fx.linear_cross_entropy(x, w, y, reduction="none"), x, g)
    for bad in (float("inf"), float("nan")):
        g[7] = bad
        dx, = torch.autograd.grad(fx.linear_cross_entropy(x, w, y, reduction="none"), x, g)
        rest = torch.arange(40, device=DEV) != 7
        assert torch.equal(dx[rest], want[rest]) and not torch.isfinite(dx[7]).any()


@pytest.mark.parametrize("rows,width,ld,at", [(3, 1, 1, 0), (3, 1, 1, 5), (4, 1, 9, 7), (5, 3, 3, 2), (7, 2, 5, 1), (2, 5, 6, 3),
                                              (9, 7, 7, 6), (1, 3, 3, 4), (40, 6, 8, 1), (700, 4, 7, 3), (700, 9, 9, 5)])
@pytest.mark.parametrize("xt,yt", [(F32, F32), (F32, BF16), (BF16, BF16), (BF16, F32), (F16, F32)])
def test_layer_norm_entries_on_narrow_rows_at_any_address(rows, width, ld, at, xt, yt):
    """Rows shorter than a vector, closer together than one, starting anywhere: the entries against 64 bits, and what lies
    around the arrays untouched."""
    g = torch.Generator(device=DEV).manual_seed(rows + width)

    def array(dtype, fill=float("nan")):
        store = torch.full((at + rows * ld + 40,), fill, device=DEV, dtype=dtype)
        return store, store[at:at + rows * ld].view(rows, ld)[:, :width]
    (_, x), (_, dy) = array(xt), array(yt)
    x.copy_(torch.randn(rows, width, generator=g, device=DEV)), dy.copy_(torch.randn(rows, width, generator=g, device=DEV))
    (ys, y), (dxs, dx) = array(yt, -7.0), array(xt, -7.0)
    w = torch.randn(width, generator=g, device=DEV)
    b, dw, db = torch.randn(width, generator=g, device=DEV), torch.empty(width, device=DEV), torch.empty(width, device=DEV)
    stats = torch.empty(rows, 2, device=DEV)
    n_ws = _lib.lib().rk_layernorm_bwd_workspace(rows, width)
    ws = torch.empty(n_ws // 4, device=DEV)
    xc, yc, s = _lib.code(xt), _lib.code(yt), _lib.stream_ptr()
    _lib.call("rk_layernorm_fwd", x.data_ptr(), xc, ld, w.data_ptr(), b.data_ptr(), 0, y.data_ptr(), yc, ld, stats.data_ptr(),
              rows, width, 1e-3, s)
    _lib.call("rk_layernorm_bwd", x.data_ptr(), xc, ld, w.data_ptr(), 0, stats.data_ptr(), dy.data_ptr(), yc, ld,
              dx.data_ptr(), ld, dw.data_ptr(), db.data_ptr(), ws.data_ptr(), n_ws, rows, width, s)
    _check_norm(x, w, b, 1e-3, y, dy, dx, dw, db)
    for store, part in ((ys, y), (dxs, dx)):
        part.fill_(-7.0)
        assert (store == -7.0).all()


@pytest.mark.parametrize("M,V,K", [(300, 9000, 8200), (40, 5000, 16384), (700, 20011, 2056), (90, 6001, 8197), (300, 9000, 8196), (6, 1, 1),
                                   (6, 1, 5), (6, 300, 33), (6, 257, 12)])
@pytest.mark.parametrize("dtype", [BF16, F16])
def test_weight_gradients_staged_a_step_at_a_time(M, V, K, dtype):
    """A weight gradient in the other 16-bit type, or of a width whose rows TMA cannot write, leaves through a buffer of some
    of its tiles; one in the operands' type or fp32 at once: all are the fp32 one, rounded. And each gradient alone, in a
    workspace without the other's part."""
    g = torch.Generator(device=DEV).manual_seed(K)
    w = (torch.randn(V, K, generator=g, device=DEV) * (2 / K ** 0.5)).to(dtype)
    y = torch.randint(0, V, (M,), generator=g, device=DEV)
    x = (torch.randn(M, K, generator=g, device=DEV) + w[y].float()).to(dtype)
    y[::5] = -100
    _, kept = fn.linear_ce_fwd(x, w, y)
    up = torch.tensor(64.0, device=DEV)
    dx, dw = fn.linear_ce_bwd(x, w, kept, up)
    dx32, dw32 = fn.linear_ce_bwd(x, w, kept, up, dx_dtype=F32, dw_dtype=F32)
    assert torch.equal(dw32.to(dtype), dw) and torch.equal(dx32.to(dtype), dx)
    other = F16 if dtype == BF16 else BF16
    assert torch.equal(fn.linear_ce_bwd(x, w, kept, up, dw_dtype=other)[1], dw32.to(other))
    assert torch.equal(fn.linear_ce_bwd(x, w, kept, up, want_dx=False, dw_dtype=F32)[1], dw32)
    assert torch.equal(fn.linear_ce_bwd(x, w, kept, up, want_dw=False, dx_dtype=F32)[0], dx32)
    X, live = x.double(), y >= 0
    some = torch.randint(0, V, (97,), generator=g, device=DEV)
    some[0], some[1] = 0, V - 1
    z = torch.cat([X @ w[s:s + 2000].double().T for s in range(0, V, 2000)], 1)
    p = (torch.softmax(z, 1) - torch.nn.functional.one_hot(y.clamp(min=0), V)) * live[:, None] * (64 / live.sum())
    part = p[:, some]
    want = part.T @ X
    # as in test_linear_ce_gpu: logits off by (K / 16 + 16) 2e sum|x w|, terms rounded to 16 bits one by one, fp32 sums
    e, h = 2.0 ** -24, {BF16: 2.0 ** -8, F16: 2.0 ** -11}[dtype]
    q = 2 * (K / 16 + 16) * 2 * e * (X.abs() @ w.double().abs().amax(0)) + 4e-6
    soft = part + torch.nn.functional.one_hot(y.clamp(min=0), V)[:, some] * live[:, None] * (64 / live.sum())
    tol = 7 * h * (part.square().T @ X.square()).sqrt() + (soft * q[:, None]).T @ X.abs() + \
        (M / 16 + 64) * 2 * e * (part.abs().T @ X.abs()) + 2.0 ** -38 * 64 * X.abs().sum(0)
    assert ((dw32[some].double() - want).abs() <= tol + 1e-12).all()
    assert _lib.device_status() == 0


@pytest.mark.parametrize("M,V,K", [(16500, 48500, 24), (16500, 49500, 264), (120000, 5000, 40)])
@pytest.mark.parametrize("dtype", [BF16, F16])
def test_several_pieces_of_the_vocabulary(M, V, K, dtype):
    """Three pieces and more, the last one shorter and ending inside a tile, over many row tiles with ignored rows: both
    gradients against 64 bits, a chunk of rows at a time, with the tolerances of test_linear_ce_gpu."""
    Mp = -(-M // 256) * 256
    assert _lib.lib().rk_linear_ce_bwd_workspace(M, V, K, 6) < Mp * -(-V // 256) * 512 / 2  # dz of less than half of the tiles
    x, w, y = _inputs(M, V, K, dtype)
    rows = fx.linear_cross_entropy(x, w, y, reduction="none")
    up = torch.rand(M, device=DEV, generator=torch.Generator(device=DEV).manual_seed(2)) - 0.5
    dx, dw = torch.autograd.grad(rows, (x, w), up)
    W, h = w.detach().double(), HALF_ULP[dtype]
    sums = [torch.zeros(V, K, device=DEV, dtype=torch.float64) for _ in range(4)]
    live = y >= 0
    assert not rows[~live].any() and not dx[~live].any()
    top = up[live].abs().max().double()
    for s in range(0, M, 3000):
        n = torch.arange(s, min(s + 3000, M), device=DEV)
        n = n[live[n]]
        X, t, u = x.detach()[n].double(), y[n][:, None], up[n].double()[:, None]
        z = X @ W.T
        size = (X.abs() @ W.abs().T).amax(1)
        dz = ((K / 16 + 16) * 2 * E * size)[:, None]
        want = torch.logsumexp(z, 1) - z.gather(1, t)[:, 0]
        assert ((rows[n].double() - want).abs() <= 2 * dz[:, 0] + 4e-6 + 4 * E * z.abs().amax(1)).all()
        p = torch.softmax(z, 1)
        err = p * (2 * dz + 4e-6) * u.abs()
        d = p.scatter_add(1, t, torch.full_like(p[:, :1], -1.0)) * u
        err += 2 * E * d.abs() + 2.0 ** -38 * top
        want = d @ W
        tol = 7 * h * (d.square() @ W.square()).sqrt() + err @ W.abs() + (V / 16 + 64) * 2 * E * (d.abs() @ W.abs()) + h * want.abs()
        assert ((dx[n].double() - want).abs() <= tol + 3e-8).all()
        for total, part in zip(sums, (d.T @ X, d.square().T @ X.square(), err.T @ X.abs(), d.abs().T @ X.abs())):
            total += part
    want, square, flat, total = sums
    tol = 7 * h * square.sqrt() + flat + (M / 16 + 64) * 2 * E * total + h * want.abs()
    assert ((dw.double() - want).abs() <= tol + 3e-8).all()
    again = torch.autograd.grad(fx.linear_cross_entropy(x, w, y, reduction="none"), (x, w), up)
    assert torch.equal(again[0], dx) and torch.equal(again[1], dw)
    assert _lib.device_status() == 0


@pytest.mark.parametrize("compute", [BF16, F16])
def test_pieces_backward_under_a_loss_scaler(compute):
    """fp32 gradients of fp32 hidden states with the scaler's factor in them, from operands of 16 bits."""
    x, w, y = _inputs(900, 1100, 72, F32)
    scaler = torch.amp.GradScaler("cuda", init_scale=2.0 ** 16)
    total, dx, dw = optimized.head_pieces_backward(x.detach(), w, y, 640, compute, scaler)
    lx, lw = x.detach().to(compute), w.detach().to(compute)
    rows = fx.linear_cross_entropy(lx, lw, y, reduction="none")
    assert dx.dtype == dw.dtype == F32 and abs(total.double() - rows.double().sum()) <= E * total.abs()
    _check_head(lx, lw, y, torch.full((900,), 1 / 640, device=DEV), rows, dx, dw, 2.0 ** 16)


@pytest.mark.parametrize("call", [optimized.chunked_backward, optimized_v3.cached_head_backward])
def test_pieces_as_a_loss_backend_in_fp16_with_a_scaler(call):
    """The explicit training step under a loss scaler: 'pieces' against the chunked softmax head, whose logits are fp16
    (|z| < 2: off by 2^-11 each) and whose hidden gradients are, once more, an eighth of what bf16 may differ by."""
    ids = torch.randint(0, 997, (4, 64), device=DEV, generator=torch.Generator(device=DEV).manual_seed(0))
    labels = ids.roll(-1, 1).clone()
    labels[:, -1], labels[0, :40] = -100, -100
    grads = {}
    for backend in ("cuda", "pieces"):
        torch.manual_seed(3)
        model = ReversibleLM(ModelConfig(vocab_size=997, max_sequence_length=64, n_layers=2, n_heads=4, d_model=128, d_ff=256),
                             "midpoint").to(DEV)
        scaler = torch.amp.GradScaler("cuda", init_scale=2.0 ** 12)
        loss = call(model, ids, labels, 200, 96, scaler=scaler, precision="fp16", loss_backend=backend)
        grads[backend] = [loss] + [p.grad for p in model.parameters()]
    for a, b in zip(grads["cuda"], grads["pieces"]):
        assert torch.isfinite(b).all() and (a - b).norm() <= 2.0 ** -9 * a.norm()


def _philox(counter, key):
    """Philox 4x32, 10 rounds, in Python's whole numbers."""
    c, k = list(counter), list(key)
    for _ in range(10):
        a, b = c[0] * 0xD2511F53, c[2] * 0xCD9E8D57
        c = [b >> 32 ^ c[1] ^ k[0], b & 0xFFFFFFFF, a >> 32 ^ c[3] ^ k[1], a & 0xFFFFFFFF]
        k = [(k[0] + 0x9E3779B9) & 0xFFFFFFFF, (k[1] + 0xBB67AE85) & 0xFFFFFFFF]
    return c


def test_the_generator_at_its_known_answers():
    """The published vectors, of all-zero and all-one counters and keys and of digits of pi, pin the restatement; the masks
    pin the kernel to it under the keys of the second and third."""
    ones = 0xFFFFFFFF
    assert _philox([0] * 4, [0] * 2) == [0x6627E8D5, 0xE169C58D, 0xBC57AC4C, 0x9B00DBD8]
    assert _philox([ones] * 4, [ones] * 2) == [0x408F276D, 0x41C83B0E, 0xA20BC7C6, 0x6D5451FD]
    pi = [0x243F6A88, 0x85A308D3, 0x13198A2E, 0x03707344], [0xA4093822, 0x299F31D0]
    assert _philox(*pi) == [0xD16CFE09, 0x94FDCCEB, 0x5001E420, 0x24126EA1]
    x = torch.ones(8, device=DEV)
    for offset, key in (([ones, ones], [ones, ones]), (pi[0][2:], pi[1])):
        words = [v for block in range(2) for v in _philox([block, 0, *offset], key)]
        seed, at = key[0] + (key[1] << 32), offset[0] + (offset[1] << 32)
        for i, word in enumerate(words):
            assert [bool(fx.dropout(x, b / 2 ** 32, seed, offset=at)[i]) for b in (word, word + 1)] == [True, False]


def test_dropout_past_the_lower_half_of_the_block_number():
    """More than 2^34 elements: from there on the block number's upper 32 bits count."""
    torch.cuda.empty_cache()
    n = (1 << 34) + 4099
    x = torch.ones(n, device=DEV, dtype=BF16)
    y = fx.dropout(x, 0.5, 21, offset=2)
    del x
    for first, last in (((1 << 34) - 4096, (1 << 34) + 4096), ((1 << 34) + 4096, n)):  # whole tiles on both sides, the rest
        words = [v for b in range(first // 4, (last + 3) // 4) for v in _philox([b & 0xFFFFFFFF, b >> 32, 2, 0], [21, 0])]
        assert torch.equal(y[first:last] != 0, torch.tensor(words[:last - first], device=DEV) >= 1 << 31)
    del y
    torch.cuda.empty_cache()
