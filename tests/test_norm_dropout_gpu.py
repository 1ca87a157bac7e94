"""Layer norm and counter-based dropout (functions.py) against their definitions in 64 bits, on the same inputs.

Tolerances, derived from the arithmetic (e = 2^-24, half an ulp of fp32). A row's sum is formed from chains of at most
32 elements, five lane steps and five warp steps, so it is off by at most 42 e times the sum of magnitudes; with the
division, the difference x - mean and the product with 1/sigma a normalised value n is off by at most
dn = 45 e (mean|x| / sigma) + 50 e |n|. The other bounds follow from dn below. A result is then rounded once, by half
an ulp of its type."""
import pytest
import torch

from reversability_b200 import _lib, functional as fn, functions as fx, kernels_v3

pytestmark = pytest.mark.gpu
DEV = "cuda"
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
HALF_ULP = {F32: 2.0 ** -24, BF16: 2.0 ** -8, F16: 2.0 ** -11}
SMALLEST = {F32: 1e-36, BF16: 1e-36, F16: 3e-8}
E = 2.0 ** -24
# (rows, width): one element, warp, vector and CTA edges, more rows than the backward has CTAs, the widest
SHAPES = [(1, 1), (3, 2), (5, 7), (9, 8), (17, 31), (33, 256), (70, 257), (10, 1000), (6, 1024), (5, 1025), (3, 4097),
          (3, 8192), (2, 16384), (5000, 333), (7000, 64), (1500, 768), (700, 1536),
          (100, 1017), (100, 1019), (1400, 1501), (310, 5003), (160, 8191), (150, 10007),
          (3, 16377), (300, 8185)]


def _rows(rows, width, dtype, layout="plain", seed=0, shift=0.5):
    """plain; wide: rows further apart than they are wide; odd: an odd distance and an odd address."""
    g = torch.Generator(device=DEV).manual_seed(seed)
    if layout == "plain":
        x = torch.empty(rows, width, device=DEV, dtype=dtype)
    elif layout == "wide":
        x = torch.empty(rows, (width + 39) // 16 * 16, device=DEV, dtype=dtype)[:, :width]
    else:
        pitch = width + 2 + width % 2 + 1
        x = torch.empty(rows * pitch + 1, device=DEV, dtype=dtype)[1:].view(rows, pitch)[:, :width]
    x.copy_(torch.randn(rows, width, generator=g, device=DEV) + shift)
    return x


def _check(x, w, b, eps, y, g, dx, dw, db):
    X, width = x.detach().double(), x.shape[-1]
    mean = X.mean(-1, keepdim=True)
    sigma = ((X - mean).square().mean(-1, keepdim=True) + eps).sqrt()
    n = (X - mean) / sigma
    W = torch.ones(width, device=DEV, dtype=torch.float64) if w is None else w.detach().double()
    want = n * W + (0 if b is None else b.detach().double())
    dn = 45 * E * X.abs().mean(-1, keepdim=True) / sigma + 50 * E * n.abs()
    tol = dn * W.abs() + 2 * E * (want.abs() + (n * W).abs()) + HALF_ULP[y.dtype] * want.abs() + SMALLEST[y.dtype]
    assert ((y.double() - want).abs() <= tol).all()
    if g is None:
        return
    G = g.detach().double()
    t = G * W
    m1, m2 = t.mean(-1, keepdim=True), (t * n).mean(-1, keepdim=True)
    dm1 = 45 * E * t.abs().mean(-1, keepdim=True)
    dm2 = 45 * E * (t * n).abs().mean(-1, keepdim=True) + (t.abs() * dn).mean(-1, keepdim=True)
    want = (t - m1 - n * m2) / sigma
    tol = (dm1 + n.abs() * dm2 + dn * m2.abs() + 4 * E * (t.abs() + m1.abs() + (n * m2).abs())) / sigma
    tol = tol + 50 * E * want.abs() + HALF_ULP[dx.dtype] * want.abs() + SMALLEST[dx.dtype]
    assert ((dx.double() - want).abs() <= tol).all()
    chain = x.shape[0] / 148 + 8 + 64  # a warp's rows, the warps, the partial rows
    for got, terms, extra in ((dw, G * n, G.abs() * dn), (db, G, None)):
        if got is not None:
            want = terms.sum(0)
            tol = chain * E * terms.abs().sum(0) + HALF_ULP[got.dtype] * want.abs() + SMALLEST[got.dtype]
            tol = tol if extra is None else tol + extra.sum(0)
            assert ((got.double() - want).abs() <= tol).all()


def _params(width, dtype, seed=5):
    g = torch.Generator(device=DEV).manual_seed(seed)
    return ((1 + 0.2 * torch.randn(width, generator=g, device=DEV)).to(dtype).requires_grad_(),
            (0.2 * torch.randn(width, generator=g, device=DEV)).to(dtype).requires_grad_())


@pytest.mark.parametrize("rows,width", SHAPES)
@pytest.mark.parametrize("dtype,out", [(F32, F32), (F32, BF16), (F32, F16), (BF16, BF16), (BF16, F32), (F16, F16), (F16, F32)])
def test_layer_norm_matches_its_definition(rows, width, dtype, out):
    x = _rows(rows, width, dtype).requires_grad_()
    w, b = _params(width, F32)
    y = fx.layer_norm(x, w, b, out_dtype=out)
    g = _rows(rows, width, out, seed=1, shift=0.1)
    _check(x, w, b, 1e-5, y, g, *torch.autograd.grad(y, (x, w, b), g))
    assert torch.equal(fx.layer_norm(x.detach(), w.detach(), b.detach(), out_dtype=out), y)


@pytest.mark.parametrize("layout", ["wide", "odd"])
@pytest.mark.parametrize("rows,width", [(5, 7), (33, 256), (70, 257), (10, 1000), (5, 1025), (3, 4097), (3, 8192)])
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
def test_layer_norm_of_strided_and_unaligned_rows(layout, rows, width, dtype):
    x, g = _rows(rows, width, dtype, layout).requires_grad_(), _rows(rows, width, dtype, layout, seed=1)
    w, b = _params(width + 1, dtype)
    w, b = w.detach()[1:].requires_grad_(), b.detach()[1:].requires_grad_()  # off any 16-byte boundary
    y = fx.layer_norm(x, w, b, 1e-3)
    _check(x, w, b, 1e-3, y, g, *torch.autograd.grad(y, (x, w, b), g))


@pytest.mark.parametrize("rows,width", [(4099, k) for k in (248, 257, 505, 512, 513, 999, 1024, 1031, 1536, 2041, 2048, 2055)] +
                         [(1301, k) for k in (2553, 2560, 2561, 3401, 4096, 5105, 5120, 5127, 8192, 8199)])
@pytest.mark.parametrize("dtype,out", [(F32, F32), (BF16, BF16), (F32, F16), (F16, F32)])
def test_layer_norm_gradients_of_many_rows_at_the_borders_of_rows_threads(rows, width, dtype, out):
    x = _rows(rows, width, dtype).requires_grad_()
    w, b = _params(width, F32)
    y = fx.layer_norm(x, w, b, out_dtype=out)
    g = _rows(rows, width, out, seed=1, shift=0.1)
    grads = torch.autograd.grad(y, (x, w, b), g, retain_graph=True)
    _check(x, w, b, 1e-5, y, g, *grads)
    for one, again in zip(grads, torch.autograd.grad(y, (x, w, b), g)):
        assert torch.equal(one, again)


@pytest.mark.parametrize("which", ["none", "weight", "bias"])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_layer_norm_without_parameters(which, dtype):
    x, g = _rows(40, 320, dtype).requires_grad_(), _rows(40, 320, dtype, seed=1)
    w, b = _params(320, dtype)
    w, b = (w if which == "weight" else None), (b if which == "bias" else None)
    y = fx.layer_norm(x, w, b)
    grads = list(torch.autograd.grad(y, [t for t in (x, w, b) if t is not None], g))
    _check(x, w, b, 1e-5, y, g, grads[0], grads[1] if w is not None else None, grads[1] if b is not None else None)
    if w is not None:  # the weight's gradient alone
        y = fx.layer_norm(x.detach(), w)
        assert torch.equal(torch.autograd.grad(y, w, g)[0], grads[1])


def test_layer_norm_keeps_digits_of_rows_far_from_zero():
    x = (_rows(64, 512, F32) * 1e-2 + 1e3).requires_grad_()
    w, b = _params(512, F32)
    y = fx.layer_norm(x, w, b)
    g = _rows(64, 512, F32, seed=1)
    _check(x, w, b, 1e-5, y, g, *torch.autograd.grad(y, (x, w, b), g))


@pytest.mark.parametrize("width", [256, 3001])
def test_layer_norm_keeps_bad_rows_to_themselves(width):
    x, g = _rows(24, width, BF16), _rows(24, width, BF16, seed=1)
    x[3], x[5, 7], x[20] = float("inf"), float("nan"), 2.0
    x.requires_grad_()
    w, b = _params(width, F32)
    y = fx.layer_norm(x, w, b)
    dx, = torch.autograd.grad(y, x, g)
    bad = torch.zeros(24, dtype=torch.bool, device=DEV)
    bad[3] = bad[5] = True
    assert torch.isnan(y[bad]).all() and torch.isnan(dx[bad]).any(1).all()
    assert torch.isfinite(y[~bad]).all() and torch.isfinite(dx[~bad]).all()
    assert torch.equal(y[20], b.detach().to(BF16))  # a constant row


def test_layer_norm_shapes_expanded_and_empty():
    w, b = _params(96, F32)
    x = torch.randn(2, 1, 96, device=DEV).expand(2, 5, 96).requires_grad_()
    y = fx.layer_norm(x, w, b)
    assert y.shape == x.shape
    y.sum().backward()  # an expanded gradient, too
    assert torch.allclose(b.grad, torch.full_like(b.grad, 10.0))
    y = fx.layer_norm(torch.randn(3, 4, 192, device=DEV)[..., ::2], w, b)  # no unit stride
    assert y.shape == (3, 4, 96)
    z = torch.empty(0, 96, device=DEV, requires_grad=True)
    y = fx.layer_norm(z, w, b)
    dx, dw, db = torch.autograd.grad(y, (z, w, b), torch.empty_like(y))
    assert dx.shape == (0, 96) and not dw.any() and not db.any()
    assert fx.layer_norm(torch.randn(96, device=DEV), w, b).shape == (96,)


def test_layer_norm_gradients_are_the_same_bits_every_run():
    x, g = _rows(4001, 512, BF16).requires_grad_(), _rows(4001, 512, BF16, seed=1)
    w, b = _params(512, F32)
    runs = [torch.autograd.grad(fx.layer_norm(x, w, b), (x, w, b), g) for _ in range(3)]
    for r in runs[1:]:
        assert all(torch.equal(s, t) for s, t in zip(r, runs[0]))


def test_layer_norm_on_two_streams_at_once():
    inputs = [(_rows(3000, 640, BF16, seed=k).requires_grad_(), _rows(3000, 640, BF16, seed=9 + k)) for k in range(2)]
    w, b = _params(640, F32)
    want = [torch.autograd.grad(fx.layer_norm(x, w, b), (x, w, b), g) for x, g in inputs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = [[], []]
    for _ in range(10):
        for k, (x, g) in enumerate(inputs):
            with torch.cuda.stream(streams[k]):
                got[k].append(torch.autograd.grad(fx.layer_norm(x, w, b), (x, w, b), g))
    torch.cuda.synchronize()
    for k in range(2):
        for r in got[k]:
            assert all(torch.equal(s, t) for s, t in zip(r, want[k]))


def test_layer_norm_gradient_against_differences():
    x = torch.randn(3, 10, device=DEV, dtype=torch.float64)
    w, b = 1 + 0.1 * torch.randn(10, device=DEV, dtype=torch.float64), torch.randn(10, device=DEV, dtype=torch.float64)
    g = torch.randn(3, 10, device=DEV, dtype=torch.float64)

    def value(x, w, b):
        return (torch.nn.functional.layer_norm(x, (10,), w, b) * g).sum()
    leaves = [t.float().requires_grad_() for t in (x, w, b)]
    grads = torch.autograd.grad(fx.layer_norm(*leaves), leaves, g.float())
    h = 1e-5
    for i, t in enumerate((x, w, b)):
        for k in range(t.numel()):
            moved = []
            for sign in (1, -1):
                args = [u.clone() for u in (x, w, b)]
                args[i].view(-1)[k] += sign * h
                moved.append(value(*args))
            # the differences are off by h^2 times a third derivative (below 1e3), the gradient by fp32
            assert abs((moved[0] - moved[1]) / (2 * h) - grads[i].view(-1)[k]) < 1e-5 + 1e-7


def test_layer_norm_refusals():
    x, w = torch.randn(4, 8, device=DEV), torch.ones(8, device=DEV)
    for bad, match in ((lambda: fx.layer_norm(x, torch.ones(7, device=DEV)), "width"),
                       (lambda: fx.layer_norm(x, w.to(BF16)), "fp32 or the input"),
                       (lambda: fx.layer_norm(x.to(BF16), w, w.to(BF16)), "share a type"),
                       (lambda: fx.layer_norm(x.to(BF16), w, out_dtype=F16), "16-bit inputs"),
                       (lambda: fx.layer_norm(x.double(), None), "not supported"),
                       (lambda: fx.layer_norm(torch.empty(3, 0, device=DEV)), "non-empty"),
                       (lambda: fx.layer_norm(x, w.cpu()), "CUDA")):
        with pytest.raises(ValueError, match=match):
            bad()
    for width in (16385, 16383):  # the second reaches over more than 16384 elements between boundaries
        with pytest.raises(RuntimeError, match="rk_layernorm_fwd"):
            fx.layer_norm(torch.randn(2, width, device=DEV, dtype=BF16))


def test_enable_layernorm_routes_modules():
    torch.manual_seed(0)
    m = torch.nn.Sequential(torch.nn.LayerNorm(48), torch.nn.Linear(48, 48), torch.nn.LayerNorm((6, 8), eps=1e-3)).to(DEV)
    x = torch.randn(5, 48, device=DEV)
    want = m[2](m[1](m[0](x)).view(5, 6, 8))
    kernels_v3.enable_layernorm(m)
    before = _lib.launch_count()
    got = m[2](m[1](m[0](x)).view(5, 6, 8))
    assert _lib.launch_count() == before + 2
    assert torch.allclose(got, want, atol=2e-5)  # torch's own error and this one's, each 45 e |x| / sigma and less
    with pytest.raises(ValueError, match="trailing"):
        m[2](x)


# ---------------------------------------------------------------- dropout
def _words(n, seed, offset):
    """Words 0 .. n-1 in Python's whole numbers (Philox 4x32, 10 rounds)."""
    out = []
    for block in range((n + 3) // 4):
        c = [block & 0xFFFFFFFF, block >> 32, offset & 0xFFFFFFFF, offset >> 32]
        k = [seed & 0xFFFFFFFF, seed >> 32 & 0xFFFFFFFF]
        for _ in range(10):
            a, b = c[0] * 0xD2511F53, c[2] * 0xCD9E8D57
            c = [b >> 32 ^ c[1] ^ k[0], b & 0xFFFFFFFF, a >> 32 ^ c[3] ^ k[1], a & 0xFFFFFFFF]
            k = [(k[0] + 0x9E3779B9) & 0xFFFFFFFF, (k[1] + 0xBB67AE85) & 0xFFFFFFFF]
        out += c
    return out[:n]


def test_words_are_those_of_the_published_generator():
    """The known answers that come with the paper, for all-zero and all-one counters and keys."""
    assert _words(4, 0, 0) == [0x6627E8D5, 0xE169C58D, 0xBC57AC4C, 0x9B00DBD8]
    # kept exactly where the word is at least round(p 2^32): a border between two words shows it
    x = torch.ones(4, device=DEV)
    for i, word in enumerate(_words(4, 0, 0)):
        kept = [bool(fx.dropout(x, b / 2 ** 32, 0)[i]) for b in (word, word + 1)]
        assert kept == [True, False]


@pytest.mark.parametrize("n", [1, 3, 4, 5, 255, 2048, 4099])
@pytest.mark.parametrize("dtype,res", [(F32, None), (BF16, None), (F16, None), (F32, F32), (BF16, BF16), (BF16, F32),
                                       (F16, F16), (F16, F32)])
def test_dropout_matches_its_definition(n, dtype, res):
    seed, offset, p = 0x123456789ABCDEF0 + n, (7 << 33) + 5, 0.3
    kept = torch.tensor(_words(n, seed, offset), device=DEV) >= round(p * 2 ** 32)
    g = torch.Generator(device=DEV).manual_seed(n)
    x = torch.randn(n, generator=g, device=DEV).to(dtype).requires_grad_()
    r = torch.randn(n, generator=g, device=DEV).to(res).requires_grad_() if res else None
    y = fx.dropout(x, p, seed, offset=offset, residual=r)
    scaled = torch.where(kept, x.detach().double() / (1 - p), 0.0)
    want = scaled + (r.detach().double() if res else 0)
    # the factor, the product and the sum are off by half an ulp of fp32 each
    tol = 3 * E * (scaled.abs() + want.abs()) + HALF_ULP[y.dtype] * want.abs() + SMALLEST[y.dtype]
    assert y.dtype == (res or dtype) and ((y.double() - want).abs() <= tol).all()
    dy = torch.randn(n, generator=g, device=DEV).to(y.dtype)
    grads = torch.autograd.grad(y, (x, r) if res else (x,), dy)
    want = torch.where(kept, dy.double() / (1 - p), 0.0)
    tol = 2 * E * want.abs() + HALF_ULP[dtype] * want.abs() + SMALLEST[dtype]
    assert grads[0].dtype == dtype and ((grads[0].double() - want).abs() <= tol).all()
    if res:
        assert torch.equal(grads[1], dy)


def test_dropout_mask_does_not_depend_on_type_layout_or_alignment():
    x = torch.ones(37, 50, device=DEV)
    want = fx.dropout(x, 0.4, 11, offset=3) != 0
    store = torch.ones(37 * 50 + 1, device=DEV)
    for other in (x.to(BF16), x.to(F16), store[1:].view(37, 50), x.to(BF16).t().contiguous().t(),
                  torch.ones(37, 64, device=DEV, dtype=F16)[:, :50], torch.ones(1, 1, device=DEV).expand(37, 50)):
        assert torch.equal(fx.dropout(other, 0.4, 11, offset=3) != 0, want)
    assert not torch.equal(fx.dropout(x, 0.4, 11, offset=4) != 0, want)
    assert not torch.equal(fx.dropout(x, 0.4, 12, offset=3) != 0, want)


def test_dropout_share_and_independence():
    """8 million elements: the share kept within five standard deviations, and so the products of neighbours'."""
    n = 1 << 23
    for p in (0.1, 0.5):
        kept = (fx.dropout(torch.ones(n, device=DEV, dtype=BF16), p, 1234, offset=9) != 0).double()
        assert abs(kept.mean().item() - (1 - p)) < 5 * (p * (1 - p) / n) ** 0.5
        for lag in (1, 4, 8, 2048):
            pair = ((kept[lag:] - (1 - p)) * (kept[:-lag] - (1 - p))).mean().item()
            assert abs(pair) < 5 * p * (1 - p) / n ** 0.5


def test_dropout_edges_of_p():
    x = torch.randn(1000, device=DEV)
    r = torch.randn(1000, device=DEV)
    assert torch.equal(fx.dropout(x, 0.0, 1), x)
    assert torch.equal(fx.dropout(x, 0.5, 1, training=False), x)
    assert torch.equal(fx.dropout(x, 1e-12, 1), x)  # rounds to no word
    assert not fx.dropout(x, 1.0, 1).any()
    assert torch.equal(fx.dropout(x, 1.0, 1, residual=r), r)
    assert fx.dropout(torch.empty(0, 3, device=DEV), 0.5, 1).shape == (0, 3)


def test_dropped_values_do_not_spread():
    words = torch.tensor(_words(64, 3, 0), device=DEV)
    x = torch.where(words >= round(0.5 * 2 ** 32), 1.0, float("nan")).to(BF16).requires_grad_()
    y = fx.dropout(x, 0.5, 3)
    assert torch.isfinite(y).all() and torch.isfinite(torch.autograd.grad(y, x, x.detach())[0]).all()


def test_dropout_seed_on_the_device_and_replays():
    x = torch.randn(4096, device=DEV)
    seed = torch.tensor(-5, device=DEV)
    assert torch.equal(fx.dropout(x, 0.2, seed), fx.dropout(x, 0.2, -5))
    assert torch.equal(fx.dropout(x, 0.2, seed), fx.dropout(x, 0.2, 2 ** 64 - 5))
    out, dx = torch.empty_like(x), torch.empty_like(x)
    leaf = x.clone().requires_grad_()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())

    def step():
        y = fx.dropout(leaf, 0.2, seed, offset=1)
        out.copy_(y.detach())
        dx.copy_(torch.autograd.grad(y, leaf, leaf.detach())[0])
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for number in (7, 8):
        seed.fill_(number)
        graph.replay()
        want = fx.dropout(x, 0.2, number, offset=1)
        assert torch.equal(out, want) and torch.equal(dx, want)
    y = fx.dropout(leaf, 0.2, seed)
    seed.add_(1)  # the mask of the forward is gone: autograd says so
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()


def test_dropout_past_32_bits():
    """More than 2^32 elements: the last ones have the words of their own positions."""
    n = (1 << 32) + 4099
    x = torch.ones(n, device=DEV, dtype=BF16)
    y = fx.dropout(x, 0.5, 21, offset=2)
    first = (n - 3001) // 4 * 4
    tail = []
    for block in range(first // 4, (n + 3) // 4):
        c, k = [block & 0xFFFFFFFF, block >> 32, 2, 0], [21, 0]
        for _ in range(10):
            a, b = c[0] * 0xD2511F53, c[2] * 0xCD9E8D57
            c = [b >> 32 ^ c[1] ^ k[0], b & 0xFFFFFFFF, a >> 32 ^ c[3] ^ k[1], a & 0xFFFFFFFF]
            k = [(k[0] + 0x9E3779B9) & 0xFFFFFFFF, (k[1] + 0xBB67AE85) & 0xFFFFFFFF]
        tail += c
    want = torch.tensor(tail[:n - first], device=DEV) >= 1 << 31
    assert torch.equal(y[first:] != 0, want)


def test_dropout_refusals():
    x = torch.randn(4, 8, device=DEV)
    for bad, match in ((lambda: fx.dropout(x, 1.5, 0), "probability"), (lambda: fx.dropout(x, float("nan"), 0), "probability"),
                       (lambda: fx.dropout(x, 0.5, 2 ** 64), "seed"), (lambda: fx.dropout(x, 0.5, 0, offset=-1), "offset"),
                       (lambda: fx.dropout(x, 0.5, torch.zeros(2, dtype=torch.int64, device=DEV)), "seed"),
                       (lambda: fx.dropout(x, 0.5, torch.zeros(1, device=DEV)), "seed"),
                       (lambda: fx.dropout(x, 0.5, torch.tensor(3)), "device"),
                       (lambda: fx.dropout(x, 0.5, 0, residual=x[:2]), "shape"),
                       (lambda: fx.dropout(x, 0.5, 0, residual=x.to(BF16)), "type"),
                       (lambda: fx.dropout(x.double(), 0.5, 0), "not supported")):
        with pytest.raises(ValueError, match=match):
            bad()


def test_kernels_run_on_the_stream_that_is_current():
    """Both directions on a side stream behind a long copy: results are those of the copied values."""
    big = torch.randn(1 << 26, device=DEV)
    src = torch.randn(512, 512, device=DEV)
    x, g = torch.zeros_like(src), torch.randn(512, 512, device=DEV)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        for _ in range(4):
            big.mul_(1.0)
        x.copy_(src)
        leaf = x.requires_grad_()
        y = fx.layer_norm(fx.dropout(leaf, 0.1, 5))
        dx, = torch.autograd.grad(y, leaf, g)
    side.synchronize()
    leaf = src.clone().requires_grad_()
    y2 = fx.layer_norm(fx.dropout(leaf, 0.1, 5))
    assert torch.equal(y, y2) and torch.equal(dx, torch.autograd.grad(y2, leaf, g)[0])
    assert fn is not None and _lib.device_status() == 0


def test_second_derivatives_are_refused():
    x = torch.randn(4, 16, device=DEV, requires_grad=True)
    w = torch.ones(16, device=DEV, requires_grad=True)
    for y in (fx.layer_norm(x, w), fx.dropout(x, 0.5, 3)):
        dx, = torch.autograd.grad(y.square().sum(), x, create_graph=True)
        with pytest.raises(RuntimeError, match="once_differentiable"):
            dx.sum().backward()


def test_layer_norm_past_32_bits():
    """More than 2^31 elements: the last rows are those of a short call, and the column sums those of equal rows."""
    rows, width = (1 << 21) + 5, 1024
    x = torch.zeros(rows, width, device=DEV, dtype=BF16)
    x[-3:] = _rows(3, width, BF16)
    g = torch.zeros_like(x)
    g[-3:] = _rows(3, width, BF16, seed=1)
    w, b = _params(width, F32)
    x.requires_grad_()
    y = fx.layer_norm(x, w, b)
    dx, dw, db = torch.autograd.grad(y, (x, w, b), g)
    short = x.detach()[-3:].clone().requires_grad_()
    ys = fx.layer_norm(short, w, b)
    sx, sw, sb = torch.autograd.grad(ys, (short, w, b), g[-3:])
    assert torch.equal(y[-3:], ys) and torch.equal(dx[-3:], sx) and not dx[:-3].any()
    # three terms a column, added in another order: two roundings of half an ulp each way
    assert torch.allclose(dw, sw, rtol=0, atol=4 * E * float(sw.abs().max()) * 3) and torch.allclose(db, sb, rtol=0, atol=4 * E * 30)
