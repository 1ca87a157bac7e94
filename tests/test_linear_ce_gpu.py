"""The head loss in pieces of the vocabulary (functions.linear_cross_entropy) against its definition in 64 bits, on the
same inputs, and the three operators of the lean training step together.

Tolerances, derived from the arithmetic (e = 2^-24). A logit is a sum of K exact products in fp32, added sixteen at a
time with at most one ulp lost a step: off by dz = (K / 16 + 16) 2e sum|x w|. A log-sum-exp is off by the largest dz and
2e-6 (exponentials within 2^-22, a blocked sum), a softmax term p by p q with q = 2 dz + 4e-6. The terms dlogits =
(p - [label]) g are rounded to 16 bits, each by at most h |dlogit| (h: half an ulp); the sums over vocabulary or rows of
those independent roundings exceed 7 h sqrt(sum (dlogit v)^2) with a probability below 1e-10 each (Hoeffding). The sums
themselves are fp32, 16 terms a step and pieces added: off by (n / 16 + 64) 2e sum|dlogit v| at most; a gradient is rounded
once, by half an ulp of its type."""
import pytest
import torch

from reversability_b200 import ModelConfig, ReversibleLM, _lib, functional as fn, functions as fx, optimized, optimized_v3
from reversability_b200.reversible import forward_pair, inverse_pair

pytestmark = pytest.mark.gpu
DEV = "cuda"
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
HALF_ULP = {F32: 2.0 ** -24, BF16: 2.0 ** -8, F16: 2.0 ** -11}
SMALLEST = {F32: 1e-36, BF16: 1e-36, F16: 3e-8}
E = 2.0 ** -24
# (rows, vocabulary, width): one of each, tile and k-block edges, several pieces, a slice of every reduction
SHAPES = [(1, 1, 1), (1, 2, 8), (3, 7, 5), (5, 300, 33), (130, 1000, 64), (257, 4099, 72), (600, 513, 256), (1000, 2000, 328),
          (64, 50257, 256), (300, 257, 1024), (2500, 1500, 96), (40, 700, 2056), (5000, 300, 40),
          (256, 256, 64), (512, 512, 128), (257, 257, 65), (9000, 600, 520), (3, 20000, 24), (32, 900, 40),
          (33, 900, 40), (300000, 64, 16), (20, 300, 8200)]


def _inputs(M, V, K, dtype, seed=0, ignored=0.3):
    g = torch.Generator(device=DEV).manual_seed(seed)
    w = (torch.randn(V, K, generator=g, device=DEV) * (2 / K ** 0.5)).to(dtype)
    y = torch.randint(0, V, (M,), generator=g, device=DEV)
    x = (torch.randn(M, K, generator=g, device=DEV) + w[y].float()).to(dtype)
    drop = torch.rand(M, generator=g, device=DEV) < ignored
    drop[0] = False
    return x.requires_grad_(), w.requires_grad_(), torch.where(drop, -100, y)


def _check(x, w, y, up, loss_rows, dx, dw, scale=1.0):
    """loss per row, and gradients of sum up_r loss_r (up: one number a row)."""
    M, K = x.shape
    V = w.shape[0]
    X, W, up = x.detach().double(), w.detach().double(), up.double()
    valid = (y >= 0) & (y < V)
    X = torch.where(valid[:, None], X, 0.0)
    t = y.clamp(0, V - 1)[:, None]
    z = X @ W.T
    size = (X.abs() @ W.abs().T).amax(1)
    dz = (K / 16 + 16) * 2 * E * size
    want = torch.where(valid, torch.logsumexp(z, 1) - z.gather(1, t)[:, 0], 0.0)
    tol = torch.where(valid, 2 * dz + 4e-6 + 4 * E * z.abs().amax(1), 0.0)
    assert ((loss_rows.double() - want).abs() <= tol).all()
    p = torch.softmax(z, 1)
    q = (2 * dz + 4e-6)[:, None]
    d = p.clone()
    d.scatter_add_(1, t, torch.full_like(d[:, :1], -1.0))
    up = torch.where(valid, up, 0.0)[:, None]
    d, err = d * up, p * q * up.abs() + 2 * E * (d * up).abs() + torch.where(valid, 2.0 ** -38, 0.0)[:, None] * up.abs().max()
    h = HALF_ULP[x.dtype]
    for got, want, square, flat, total, n in (
            (dx, d @ W, d.square() @ W.square(), err @ W.abs(), d.abs() @ W.abs(), V),
            (dw, d.T @ X, d.square().T @ X.square(), err.T @ X.abs(), d.abs().T @ X.abs(), M)):
        if got is not None:
            tol = 7 * h * square.sqrt() + flat + (n / 16 + 64) * 2 * E * total + HALF_ULP[got.dtype] * want.abs()
            assert ((got.double() / scale - want).abs() <= tol + SMALLEST[got.dtype] / scale).all()


@pytest.mark.parametrize("M,V,K", SHAPES)
@pytest.mark.parametrize("dtype", [BF16, F16])
def test_one_loss_a_row(M, V, K, dtype):
    x, w, y = _inputs(M, V, K, dtype)
    rows = fx.linear_cross_entropy(x, w, y, reduction="none")
    assert rows.shape == y.shape and rows.dtype == F32
    g = torch.randn(M, device=DEV, generator=torch.Generator(device=DEV).manual_seed(1)) * 0.3
    dx, dw = torch.autograd.grad(rows, (x, w), g)
    assert dx.dtype == dw.dtype == dtype
    _check(x, w, y, g, rows, dx, dw)
    assert torch.equal(fx.linear_cross_entropy(x.detach(), w.detach(), y, reduction="none"), rows)


@pytest.mark.parametrize("M,V,K", [(5, 300, 33), (600, 513, 256), (257, 4099, 72), (2500, 1500, 96)])
@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("reduction", ["sum", "mean"])
def test_one_loss_for_all(M, V, K, dtype, reduction):
    x, w, y = _inputs(M, V, K, dtype)
    rows = fx.linear_cross_entropy(x.detach(), w.detach(), y, reduction="none")
    n = (y >= 0).sum()
    loss = fx.linear_cross_entropy(x, w, y, reduction=reduction)
    want = rows.double().sum() / (n if reduction == "mean" else 1)
    assert loss.dtype == F32 and loss.shape == () and abs(loss.double() - want) <= E * abs(want)
    scale = 1024.0 if dtype == F16 else 1.0  # a loss scaler's
    dx, dw = torch.autograd.grad(loss * scale, (x, w))
    up = torch.ones(M, device=DEV) / (n if reduction == "mean" else 1)
    _check(x, w, y, up, rows, dx, dw, scale)


def test_a_large_mean_in_fp16_does_not_underflow():
    """Gradients of the size of fp16's smallest numbers, from terms far below them."""
    x, w, y = _inputs(6000, 2000, 64, F16, ignored=0.0)
    loss = fx.linear_cross_entropy(x, w, y)
    dx, dw = torch.autograd.grad(loss, (x, w))
    rows = fx.linear_cross_entropy(x.detach(), w.detach(), y, reduction="none")
    _check(x, w, y, torch.full((6000,), 1 / 6000, device=DEV), rows, dx, dw)
    assert (dw != 0).float().mean() > 0.5


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
def test_ignored_rows_are_not_read(dtype):
    x, w, y = _inputs(700, 900, 48, dtype, ignored=0.6)
    with torch.no_grad():
        x[y < 0] = float("nan")
    rows = fx.linear_cross_entropy(x, w, y, reduction="none")
    dx, dw = torch.autograd.grad(rows.sum(), (x, w))
    assert torch.isfinite(rows).all() and torch.isfinite(dx).all() and torch.isfinite(dw).all()
    assert not rows[y < 0].any() and not dx[y < 0].any()
    live = y >= 0  # the same as without them
    x2 = x.detach()[live].requires_grad_()
    rows2 = fx.linear_cross_entropy(x2, w, y[live], reduction="none")
    dx2, dw2 = torch.autograd.grad(rows2.sum(), (x2, w))
    if dtype != F32:
        assert torch.equal(rows[live], rows2) and torch.equal(dx[live], dx2)
        _check(x, w, y, torch.ones(700, device=DEV), rows, dx, dw)
    else:
        assert torch.allclose(rows[live], rows2, atol=1e-5) and torch.allclose(dw, dw2, atol=1e-4)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("reduction", ["none", "sum", "mean"])
def test_no_row_counts_and_no_row_at_all(dtype, reduction):
    for M in (0, 3, 300):
        x, w, _ = _inputs(300, 40, 24, dtype)
        x = x.detach()[:M].requires_grad_()
        y = torch.full((M,), -100, device=DEV)
        loss = fx.linear_cross_entropy(x, w, y, reduction=reduction)
        assert not loss.any() and loss.shape == ((M,) if reduction == "none" else ())
        dx, dw = torch.autograd.grad(loss.sum(), (x, w))
        assert dx.shape == x.shape and not dx.any() and not dw.any()


def test_labels_outside_the_vocabulary_count_as_ignored():
    x, w, y = _inputs(200, 100, 16, BF16)
    bad = y.clone()
    bad[7], bad[9] = 100, -3
    ref = y.clone()
    ref[7] = ref[9] = -100
    assert _lib.device_status() == 0
    got = fx.linear_cross_entropy(x, w, bad)
    assert _lib.device_status() == 4  # RK_DEV_CE_LABEL
    assert torch.equal(got, fx.linear_cross_entropy(x, w, ref)) and _lib.device_status() == 0
    # any number may be the one that is ignored
    got = fx.linear_cross_entropy(x, w, torch.where(y < 0, 5, y), ignore_index=5)
    assert torch.equal(got, fx.linear_cross_entropy(x, w, torch.where(y == 5, -100, y)))


@pytest.mark.parametrize("dtype", [BF16, F16])
def test_layouts(dtype):
    """Hidden states in wider rows, at odd addresses, transposed or with more dimensions; weights at odd addresses."""
    x, w, y = _inputs(60, 500, 40, dtype)
    want = fx.linear_cross_entropy(x, w, y, reduction="none")
    g = torch.autograd.grad(want.sum(), (x, w))
    wide = torch.zeros(60, 57, device=DEV, dtype=dtype)
    wide[:, 3:43] = x.detach()
    shifted = torch.zeros(500 * 40 + 1, device=DEV, dtype=dtype)[1:].view(500, 40)
    shifted.copy_(w.detach())
    odd = torch.zeros(500, 43, device=DEV, dtype=dtype)
    odd[:, :40] = w.detach()
    for a, b, shape in ((wide[:, 3:43], shifted, (60,)), (x.detach().t().contiguous().t(), odd[:, :40], (60,)),
                        (x.detach().view(4, 15, 40), w.detach().t().contiguous().t(), (4, 15))):
        a, b = a.requires_grad_(), b.requires_grad_()
        rows = fx.linear_cross_entropy(a, b, y.view(shape), reduction="none")
        assert rows.shape == shape and torch.equal(rows.view(-1), want)
        dx, dw = torch.autograd.grad(rows.sum(), (a, b))
        assert dx.shape == a.shape and torch.equal(dx.reshape(60, 40), g[0]) and torch.equal(dw, g[1])


def test_each_gradient_alone_and_twice():
    x, w, y = _inputs(500, 1200, 72, BF16)
    rows = fx.linear_cross_entropy(x, w, y, reduction="none")
    a = torch.rand(500, device=DEV)
    first = torch.autograd.grad(rows, (x, w), a, retain_graph=True)
    second = torch.autograd.grad(rows, (x, w), 2 * a)
    assert all(torch.equal(s, 2 * f) for f, s in zip(first, second))  # a power of two: the same digits, and no state kept
    dx, = torch.autograd.grad(fx.linear_cross_entropy(x, w.detach(), y, reduction="none"), x, a)
    dw, = torch.autograd.grad(fx.linear_cross_entropy(x.detach(), w, y, reduction="none"), w, a)
    assert torch.equal(dx, first[0]) and torch.equal(dw, first[1])
    huge = torch.autograd.grad(fx.linear_cross_entropy(x, w, y, reduction="none"), (x, w), a * 2.0 ** 90)
    assert all(torch.equal(t, f * 2.0 ** 90) for t, f in zip(huge, first))


def test_gradient_against_differences():
    x, w, y = _inputs(6, 11, 8, BF16)
    up = torch.randn(6, device=DEV)
    dx, dw = torch.autograd.grad(fx.linear_cross_entropy(x, w, y, reduction="none"), (x, w), up)

    def value(x, w):
        z = x @ w.T
        valid = y >= 0
        return ((torch.logsumexp(z, 1) - z.gather(1, y.clamp(min=0)[:, None])[:, 0]) * valid * up.double()).sum()
    base = [x.detach().double(), w.detach().double()]
    step = 1e-6
    for i, got in enumerate((dx, dw)):
        for k in range(got.numel()):
            moved = []
            for sign in (1, -1):
                args = [t.clone() for t in base]
                args[i].view(-1)[k] += sign * step
                moved.append(value(*args))
            # 16-bit terms: 11 (or 6) roundings of at most 2^-8 |up p v| and the result's own
            assert abs((moved[0] - moved[1]) / (2 * step) - got.view(-1)[k]) < 0.06


def test_a_weight_past_32_bits():
    """More than 2^31 weight elements: losses and gradients where the last rows are labels."""
    V, K = 4_200_001, 520
    w = torch.empty(V, K, device=DEV, dtype=BF16).normal_(std=0.02).requires_grad_()
    y = torch.tensor([V - 1, 5, V - 2], device=DEV)
    x = torch.randn(3, K, device=DEV).to(BF16).requires_grad_()
    rows = fx.linear_cross_entropy(x, w, y, reduction="none")
    dx, dw = torch.autograd.grad(rows.sum(), (x, w))
    X = x.detach().double()
    z = torch.cat([X @ w.detach()[s:s + 300_000].double().T for s in range(0, V, 300_000)], 1)
    lse = torch.logsumexp(z, 1)
    assert (rows.double() - (lse - z.gather(1, y[:, None])[:, 0])).abs().max() < 1e-4
    for s in (0, 4_129_800, V - 1000):  # 2^31 elements lie before row 4129777
        p = torch.exp(z[:, s:s + 1000] - lse[:, None])
        for r in range(3):
            if s <= y[r] < s + 1000:
                p[r, y[r] - s] -= 1
        want = p.T @ X
        # three terms rounded to 16 bits, and the result
        tol = 2.0 ** -8 * (p.T.abs() @ X.abs()) + 2.0 ** -8 * want.abs() + 1e-12
        assert ((dw[s:s + 1000].double() - want).abs() <= tol).all()
    # dx is the mean of 4 million small rows less one row: that row, within what the others can add
    assert ((dx.double() + w.detach()[y].double()).abs() < 0.02).all()


def test_large_logits():
    """Spread of hundreds: most softmax terms vanish, the running reference moves."""
    x, w, y = _inputs(300, 3000, 64, BF16)
    x = (x.detach() * 40).requires_grad_()
    rows = fx.linear_cross_entropy(x, w, y, reduction="none")
    dx, dw = torch.autograd.grad(rows.sum(), (x, w))
    _check(x, w, y, torch.ones(300, device=DEV), rows, dx, dw)


@pytest.mark.parametrize("rows", [3, 300, 512])
@pytest.mark.parametrize("dtype", [BF16, F16, F32])
def test_an_entry_of_minus_infinity(dtype, rows):
    """An entry whose logits are -inf is as one whose exponentials underflow, also where rows of zeros pad a tile."""
    x, w, y = _inputs(rows, 600, 64, dtype)
    x = x.detach()
    x[:, 0] = 1 + x[:, 0].abs()
    y = torch.where(y == 5, 6, y)
    got = []
    for entry in (-float("inf"), -30000.0):
        v = w.detach().clone()
        v[5] = 0
        v[5, 0] = entry
        v.requires_grad_()
        loss = fx.linear_cross_entropy(x, v, y)
        got.append((loss.detach(), torch.autograd.grad(loss, v)[0]))
    assert torch.isfinite(got[0][1]).all()
    assert torch.equal(got[0][0], got[1][0]) and torch.equal(got[0][1], got[1][1])


def test_results_are_the_same_bits_every_run():
    x, w, y = _inputs(3000, 5000, 264, BF16)
    runs = []
    for _ in range(3):
        loss = fx.linear_cross_entropy(x, w, y)
        runs.append((loss, *torch.autograd.grad(loss, (x, w))))
    for r in runs[1:]:
        assert all(torch.equal(s, t) for s, t in zip(r, runs[0]))
    assert _lib.device_status() == 0


@pytest.mark.parametrize("reduction", ["none", "sum", "mean"])
def test_fp32(reduction):
    M, V, K = 70, 333, 48
    x, w, y = _inputs(M, V, K, F32)
    up = torch.rand(M, device=DEV) if reduction == "none" else torch.ones((), device=DEV)
    got = fx.linear_cross_entropy(x, w, y, reduction=reduction)
    grads = torch.autograd.grad(got, (x, w), up)
    X, W = x.detach().double().requires_grad_(), w.detach().double().requires_grad_()
    want = torch.nn.functional.cross_entropy(X @ W.T, y, reduction=reduction)
    # K and V terms a sum in fp32, in order: below 400 e of sums of magnitudes below 50
    assert torch.allclose(got.double(), want, atol=400 * E * 50)
    for a, b in zip(grads, torch.autograd.grad(want, (X, W), up.double())):
        assert torch.allclose(a.double(), b, atol=400 * E * 50)


def test_fp32_in_pieces_of_the_rows(monkeypatch):
    x, w, y = _inputs(70, 333, 48, F32)
    whole = fx.linear_cross_entropy(x, w, y)
    grads = torch.autograd.grad(whole, (x, w))
    monkeypatch.setattr(fn, "_PIECE_BYTES", 333 * 4 * 16)
    parts = fx.linear_cross_entropy(x, w, y)
    assert torch.equal(parts, whole)
    for a, b in zip(torch.autograd.grad(parts, (x, w)), grads):
        assert torch.allclose(a, b, rtol=0, atol=70 * 2 * E)


def test_autocast_casts_both():
    x, w, y = _inputs(50, 120, 32, F32)
    with torch.autocast("cuda", dtype=BF16):
        loss = fx.linear_cross_entropy(x, w, y)
    dx, dw = torch.autograd.grad(loss, (x, w))
    assert dx.dtype == dw.dtype == F32
    assert torch.equal(loss, fx.linear_cross_entropy(x.detach().to(BF16), w.detach().to(BF16), y))


def test_refusals():
    x, w, y = _inputs(6, 11, 8, BF16)
    for bad, match in ((lambda: fx.linear_cross_entropy(x, w, y, reduction="max"), "reduction"),
                       (lambda: fx.linear_cross_entropy(x, w[:, :4], y), "weight"),
                       (lambda: fx.linear_cross_entropy(x, w.float(), y), "share a type"),
                       (lambda: fx.linear_cross_entropy(x.double(), w.double(), y), "share a type"),
                       (lambda: fx.linear_cross_entropy(x, w, y[:3]), "labels"),
                       (lambda: fx.linear_cross_entropy(x, w, y.int()), "labels"),
                       (lambda: fx.linear_cross_entropy(x, w[:0], y), "non-empty"),
                       (lambda: fx.linear_cross_entropy(x, w, y.cpu()), "CUDA")):
        with pytest.raises(ValueError, match=match):
            bad()


def test_two_streams_and_two_graphs_at_once():
    """Calls of different sizes in flight together, then two captured steps replayed in turn: each as if alone."""
    cases = [_inputs(700, 1500, 64, BF16, 1), _inputs(300, 4000, 136, BF16, 2)]

    def step(x, w, y):
        loss = fx.linear_cross_entropy(x, w, y)
        return (loss.detach(), *torch.autograd.grad(loss, (x, w)))
    want = [step(*c) for c in cases]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in cases]
    got = [[], []]
    for _ in range(5):
        for k, c in enumerate(cases):
            with torch.cuda.stream(streams[k]):
                got[k].append(step(*c))
    torch.cuda.synchronize()
    for k in range(2):
        assert all(torch.equal(s, t) for r in got[k] for s, t in zip(r, want[k]))
    graphs, outs = [], []
    for x, w, y in cases:
        leaves = (x.detach().clone().requires_grad_(), w.detach().clone().requires_grad_())  # no eager graph holds them
        with torch.cuda.stream(streams[0]):
            step(*leaves, y)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(step(*leaves, y))
        graphs.append((graph, leaves, y))
    for _ in range(3):
        for graph, _, _ in graphs:
            graph.replay()
    torch.cuda.synchronize()
    for k in range(2):
        assert all(torch.equal(s, t) for s, t in zip(outs[k], want[k]))
    assert _lib.device_status() == 0


def test_captured_and_replayed():
    x, w, y = _inputs(300, 700, 64, BF16)
    x, w = x.detach(), w.detach()
    leaf_x, leaf_w = x.clone().requires_grad_(), w.clone().requires_grad_()
    labels = y.clone()
    out = [torch.empty((), device=DEV), torch.empty_like(x), torch.empty_like(w)]

    def step():
        loss = fx.linear_cross_entropy(leaf_x, leaf_w, labels)
        for o, t in zip(out, (loss.detach(), *torch.autograd.grad(loss, (leaf_x, leaf_w)))):
            o.copy_(t)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for seed, ignored in ((1, 0.0), (2, 0.9), (3, 0.5)):  # the number of rows that count is read on the device
        a, b, c = _inputs(300, 700, 64, BF16, seed, ignored)
        with torch.no_grad():
            leaf_x.copy_(a), leaf_w.copy_(b)
        labels.copy_(c)
        graph.replay()
        loss = fx.linear_cross_entropy(a, b, c)
        want = (loss, *torch.autograd.grad(loss, (a, b)))
        assert all(torch.equal(s, t) for s, t in zip(out, want))
    assert _lib.device_status() == 0


@pytest.mark.parametrize("precision", ["bf16", "fp32"])
@pytest.mark.parametrize("call", [optimized.chunked_backward, optimized_v3.cached_head_backward])
def test_pieces_as_a_loss_backend(precision, call):
    """The reversible model's explicit training step: 'pieces' against the chunked softmax head."""
    ids = torch.randint(0, 997, (4, 64), device=DEV, generator=torch.Generator(device=DEV).manual_seed(0))
    labels = ids.roll(-1, 1).clone()
    labels[:, -1] = -100
    labels[0, :40] = -100
    grads = {}
    for backend in ("cuda", "pieces"):
        torch.manual_seed(3)
        model = ReversibleLM(ModelConfig(vocab_size=997, max_sequence_length=64, n_layers=2, n_heads=4, d_model=128, d_ff=256),
                             "midpoint").to(DEV)
        loss = call(model, ids, labels, 200, 96, precision=precision, loss_backend=backend)
        grads[backend] = [loss] + [p.grad for p in model.parameters()]
    # bf16: logits rounded to bf16 (|z| < 2: 2^-8 each) in the softmax head, hidden gradients rounded to bf16
    tol = 2.0 ** -6 if precision == "bf16" else 1e-4
    for a, b in zip(grads["cuda"], grads["pieces"]):
        assert (a - b).norm() <= tol * a.norm()


class _Block(torch.nn.Module):
    """A block with layer norms and dropout whose masks are a function of (seed, place): a force that can be replayed."""

    def __init__(self, d, place):
        super().__init__()
        self.norms = torch.nn.ModuleList(torch.nn.LayerNorm(d) for _ in range(2))
        self.lin = torch.nn.ModuleList(torch.nn.Linear(d, d) for _ in range(2))
        self.place, self.seed = place, 0
        self.attn_norm = lambda x: fx.layer_norm(x, self.norms[0].weight, self.norms[0].bias)
        self.mlp_norm = lambda x: fx.layer_norm(x, self.norms[1].weight, self.norms[1].bias)
        self.attn = lambda x: self._branch(0, x)
        self.mlp = lambda x: self._branch(1, x)

    def _branch(self, i, x):
        y = torch.tanh(fx.linear(x, self.lin[i].weight, self.lin[i].bias))
        return fx.dropout(y, 0.2, self.seed, offset=2 * self.place + i)


@pytest.mark.parametrize("method", ["midpoint", "euler"])
def test_a_lean_step_of_all_three(method):
    """Blocks of layer norm and dropout, inverted by replaying the masks, under the head loss in pieces: states come
    back, and the gradients are those of the same step with stored masks and logits."""
    torch.manual_seed(0)
    d, V = 96, 613
    blocks = torch.nn.ModuleList(_Block(d, i) for i in range(3)).to(DEV)
    emb = torch.nn.Parameter(torch.randn(V, d, device=DEV) * 0.3)
    ids = torch.randint(0, V, (2, 50), device=DEV)
    labels = ids.roll(-1, 1)
    for b in blocks:
        b.seed = 1234
    x = emb[ids]
    p, q = x, x
    states = [(p, q)]
    for b in blocks:
        p, q = forward_pair(b, p, q, method, 0.25)
        states.append((p, q))
    with torch.no_grad():
        rp, rq = p, q
        for b, (wp, wq) in zip(reversed(blocks), reversed(states[:-1])):
            rp, rq = inverse_pair(b, rp, rq, method, 0.25)
            # sums and differences of the same fp32 terms of size below 16, six roundings a layer
            assert (rp - wp).abs().max() < 1e-4 and (rq - wq).abs().max() < 1e-4
    loss = fx.linear_cross_entropy(fx.layer_norm(q if method == "midpoint" else p), emb, labels)
    grads = torch.autograd.grad(loss, [emb, *blocks.parameters()])

    def plain(i, x, n, lin, place):
        y = torch.tanh(torch.nn.functional.linear(x, lin.weight, lin.bias))
        mask = fx.dropout(torch.ones_like(y), 0.2, 1234, offset=2 * place + i).detach()
        return y * mask
    p, q = emb[ids], emb[ids]
    for k, b in enumerate(blocks):
        norm = lambda i, x: torch.nn.functional.layer_norm(x, (d,), b.norms[i].weight, b.norms[i].bias)  # noqa: E731, B023
        A = lambda x: plain(0, norm(0, x), None, b.lin[0], k)  # noqa: E731, B023
        Mlp = lambda x: plain(1, norm(1, x), None, b.lin[1], k)  # noqa: E731, B023
        if method == "midpoint":
            a = A(q)
            p, q = q, p + 2 * 0.25 * (a + Mlp(q + a))
        else:
            nq = q + A(p)
            p, q = p + Mlp(nq), nq
    logits = torch.nn.functional.layer_norm(q if method == "midpoint" else p, (d,)) @ emb.T
    want = torch.nn.functional.cross_entropy(logits.view(-1, V), labels.view(-1))
    # fp32 both: sums of up to 613 terms, a dozen layers of them
    assert abs(loss - want) < 1e-4
    for a, b in zip(grads, torch.autograd.grad(want, [emb, *blocks.parameters()])):
        assert (a - b).norm() <= 1e-3 * b.norm() + 1e-7
