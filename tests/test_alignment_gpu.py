"""Token log-probabilities, clipped policy loss and paired preference loss
(alignment.py) against their definitions in 64 bits, on the same inputs.

Tolerances, derived from the arithmetic: a log-probability is
(z - m) - ln S with z, m rounded to fp32 (relative 2^-24 each, so absolute
2^-22 max|z|) and ln S within 2e-6 (exponentials within 2^-22 relative, a
blocked fp32 sum). A probability then carries a relative error of 2e-5 as long
as |ln p| < 60, and smaller ones round to nothing. A gradient is rounded once:
half an ulp of its type on top of that."""
import math

import pytest
import torch

from reversability_b200 import _lib, alignment, functional as fn

pytestmark = pytest.mark.gpu
DEV = "cuda"
DTYPES = [torch.float32, torch.bfloat16, torch.float16]
HALF_ULP = {torch.float32: 0.0, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
SMALLEST = {torch.float32: 1e-36, torch.bfloat16: 1e-36, torch.float16: 6e-8}
# (rows, vocabulary): single elements, warp and vector edges, the decoder's vocabulary, a large odd one
SHAPES = [(1, 1), (3, 2), (5, 7), (64, 31), (70, 101), (9, 255), (300, 1000), (33, 4097), (17, 8209), (6, 50257), (3, 131075)]


def _logits(rows, vocab, dtype, layout="plain", seed=0, scale=2.0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    if layout == "plain":
        x = torch.empty(rows, vocab, device=DEV, dtype=dtype)
    elif layout == "padded":  # rows start on 128 bytes
        x = torch.empty(rows, (vocab + 63) // 64 * 64, device=DEV, dtype=dtype)[:, :vocab]
    else:  # "shifted": an odd row stride and a base that is no multiple of 16 bytes
        width = vocab + 3 + vocab % 2
        x = torch.empty(rows * width + 1, device=DEV, dtype=dtype)[1:].view(rows, width)[:, 1:1 + vocab]
    x.copy_(torch.randn(rows, vocab, generator=g, device=DEV) * scale)
    return x


def _labels(rows, vocab, seed=0, ignored=0.3):
    g = torch.Generator(device=DEV).manual_seed(100 + seed)
    y = torch.randint(0, vocab, (rows,), generator=g, device=DEV)
    drop = torch.rand(rows, generator=g, device=DEV) < ignored
    drop[0] = False
    y[drop] = -100
    return y


def _rows64(x, y, temperature=1.0):
    """fp64 (logp of all columns, lp at the label, entropy, valid) by torch's own log_softmax."""
    logp = torch.log_softmax(x.double() / temperature, -1)
    valid = y >= 0
    lp = logp.gather(-1, y.clamp(min=0)[..., None])[..., 0] * valid
    p = logp.exp()
    h = -torch.where(p > 0, p * logp, torch.zeros_like(p)).sum(-1) * valid
    return logp, lp, h, valid


def _lp_tol(x, temperature=1.0):
    live = x.double().abs()
    live = torch.where(live > 1e3, torch.zeros_like(live), live)  # masked columns do not count
    return 2e-6 + 2.0 ** -22 * float(live.max()) / temperature


def _check_grad(d, x, y, temperature, g_lp, g_h=None):
    """d against g_lp ([j = y] - p) - g_h p (ln p + H), over the temperature, in 64 bits."""
    logp, _, h, valid = _rows64(x, y, temperature)
    p = logp.exp()
    g = (torch.as_tensor(g_lp, device=DEV).double() * valid)[:, None]
    want = -g * p
    want.scatter_add_(1, y.clamp(min=0)[:, None], g)
    size = g.abs() * p
    size.scatter_add_(1, y.clamp(min=0)[:, None], g.abs() * p.gather(1, y.clamp(min=0)[:, None]))
    if g_h is not None:
        gh = (torch.as_tensor(g_h, device=DEV).double() * valid)[:, None]
        want = want - gh * torch.where(p > 0, p * (logp + h[:, None]), torch.zeros_like(p))
        size = size + gh.abs() * torch.where(p > 0, p * (logp.abs() + h[:, None] + 1), torch.zeros_like(p))
    want, size = want / temperature, size / temperature
    # the label's entry is g (1 - p): its error is that of p and fp32's own rounding of g
    tol = HALF_ULP[d.dtype] * want.abs() + 2e-5 * size + 2.0 ** -22 * want.abs() + SMALLEST[d.dtype]
    over = ((d.double() - want).abs() - tol).max()
    assert float(over) <= 0, f"gradient off by {float(over):.3e} more than its tolerance"
    assert not d[~valid].any(), "ignored rows must have zero gradients"


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("layout", ["plain", "padded", "shifted"])
@pytest.mark.parametrize("shape", SHAPES)
def test_token_logprobs_forward_and_backward(shape, layout, dtype):
    rows, vocab = shape
    for temperature in (1.0, 0.7):
        x = _logits(rows, vocab, dtype, layout, seed=rows).requires_grad_()
        y = _labels(rows, vocab)
        _, lp64, h64, _ = _rows64(x.detach(), y, temperature)
        lp, h = alignment.token_logprobs(x, y, temperature=temperature, entropy=True)
        assert lp.dtype == h.dtype == torch.float32 and lp.requires_grad and h.requires_grad
        tol = _lp_tol(x.detach(), temperature)
        assert float((lp.detach().double() - lp64).abs().max()) <= tol
        # the entropy is a mean of log-probabilities
        assert float((h.detach().double() - h64).abs().max()) <= tol + 1e-5 * float(h64.max().clamp(min=1e-3))
        g = torch.Generator(device=DEV).manual_seed(7)
        a = torch.randn(rows, generator=g, device=DEV)
        b = torch.randn(rows, generator=g, device=DEV)
        d, = torch.autograd.grad([lp, h], x, [a, b], retain_graph=True)
        _check_grad(d, x.detach(), y, temperature, a, b)
        d, = torch.autograd.grad(lp, x, a)
        _check_grad(d, x.detach(), y, temperature, a)
    assert _lib.device_status() == 0


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("vocab", [5, 130, 3000, 50257])
def test_masked_columns_infinities_and_nan(vocab, dtype):
    """Columns at -inf or at the type's lowest value have probability 0 and no gradient; a NaN stays in its row, and
    in an ignored row it is not read; +inf gives NaN as log_softmax does; large logits lose nothing to their size."""
    rows = 8
    x = _logits(rows, vocab, dtype, seed=3)
    y = torch.randint(0, vocab // 2, (rows,), device=DEV, generator=torch.Generator(device=DEV).manual_seed(1))
    half = vocab // 2 + 1
    x[0, half:] = -math.inf
    x[1, half:] = torch.finfo(dtype).min
    x[2, vocab - 1] = math.nan
    x[3] = math.nan
    y[3] = -100
    x[4, 0] = math.inf
    x[5] = torch.finfo(dtype).min  # a row with nothing but masks of the lowest value: uniform
    x[6] = -math.inf               # a row with nothing at all: NaN, as log_softmax gives
    if dtype != torch.float16:
        x[7] += 4096.0
    x.requires_grad_()
    lp, h = alignment.token_logprobs(x, y, entropy=True)
    d, = torch.autograd.grad([lp, h], x, [torch.ones_like(lp), torch.full_like(h, 0.5)])
    ok = torch.tensor([0, 1, 3, 5, 7], device=DEV)
    _, lp64, h64, _ = _rows64(x.detach()[ok], y[ok])
    lp64[2] = h64[2] = 0.0  # the ignored row
    assert float((lp.detach()[ok].double() - lp64).abs().max()) <= 2e-6 + 2.0 ** -22 * (4200 if dtype != torch.float16 else 20)
    assert float((h.detach()[ok].double() - h64).abs().max()) <= 2e-4
    for r in (2, 4, 6):
        assert math.isnan(float(lp.detach()[r])) and bool(d[r].isnan().any())
    assert not d[3].any() and not d[0, half:].any() and not d[1, half:].any()
    assert bool(d[ok].isfinite().all())
    live = torch.tensor([0, 1, 5], device=DEV)
    _check_grad(d[live], x.detach()[live], y[live], 1.0, torch.ones(3, device=DEV), torch.full((3,), 0.5, device=DEV))


def test_label_out_of_range_sets_the_status_bit_and_is_ignored():
    x = _logits(4, 33, torch.float32).requires_grad_()
    y = torch.tensor([3, 33, -5, 0], device=DEV)
    lp = alignment.token_logprobs(x, y)
    assert _lib.device_status() == 1 << 2
    d, = torch.autograd.grad(lp.sum(), x)
    assert not d[1].any() and not d[2].any() and bool(d[0].any())
    assert float(lp[1].detach()) == float(lp[2].detach()) == 0.0
    old = torch.zeros(4, device=DEV)
    alignment.policy_loss_and_grad(x, y, old, torch.ones(4, device=DEV))
    assert _lib.device_status() == 1 << 2
    _lib.device_status()


def test_all_rows_ignored_and_no_rows():
    x = _logits(6, 77, torch.bfloat16)
    y = torch.full((6,), -100, device=DEV)
    z = torch.zeros(6, device=DEV)
    r, d = alignment.policy_loss_and_grad(x, y, z, z + 1, ref_logprobs=z, kl_coef=0.1, entropy_coef=0.1)
    assert float(r.loss) == 0.0 and float(r.clip_fraction) == 0.0
    assert not d.any() and not r.logprobs.any() and not r.kl.any() and not r.entropy.any()
    e = torch.zeros(0, device=DEV)
    none = torch.zeros(0, dtype=torch.int64, device=DEV)
    r, d = alignment.policy_loss_and_grad(x[:0], none, e, e)
    assert float(r.loss) == 0.0 and d.shape == (0, 77)
    assert alignment.token_logprobs(x[:0], none).shape == (0,)
    r, d = alignment.preference_loss_and_grad(torch.zeros(2, 0, 9, device=DEV), torch.zeros(2, 0, dtype=torch.int64, device=DEV), None)
    assert abs(float(r.loss) - math.log(2)) < 1e-6 and d.shape == (2, 0, 9)
    # pairs without a labelled token: gap 0, no gradient
    y = torch.full((2, 3), -100, device=DEV)
    r, d = alignment.preference_loss_and_grad(x.view(2, 3, 77), y, None, average=True)
    assert abs(float(r.loss) - math.log(2)) < 1e-6 and not d.any() and not r.rewards.any()


# ---------------------------------------------------------------- policy loss
def _policy64(x, y, old, adv, ref, w, lo, hi, ckl, cent, temperature, denom, gscale):
    z = x.double().requires_grad_()
    logp = torch.log_softmax(z / temperature, -1)
    valid = y >= 0
    lp = logp.gather(1, y.clamp(min=0)[:, None])[:, 0]
    p = logp.exp()
    h = -(torch.where(p > 0, p * logp, torch.zeros_like(p))).sum(1)
    ratio = (lp - old.double()).exp()
    free, held = ratio * adv.double(), ratio.clamp(1 - lo, 1 + hi) * adv.double()
    clipped = held < free
    each = -torch.where(clipped, held, free) - cent * h
    kl = torch.zeros_like(lp)
    if ref is not None:
        kl = (ref.double() - lp).exp() - 1 - (ref.double() - lp)
        each = each + ckl * kl
    ww = (torch.ones_like(lp) if w is None else w.double()) * valid
    total = ww.sum() if denom is None else denom.double()
    loss = (torch.where(valid, each, torch.zeros_like(each)) * ww).sum() / total
    lp.retain_grad()
    d, g_lp = torch.autograd.grad(loss * gscale, [z, lp])
    return loss.detach(), lp.detach() * valid, kl.detach() * valid, h.detach() * valid, (clipped * ww).sum() / total, d, g_lp


def _policy_inputs(rows, vocab, dtype, layout, seed=0):
    x = _logits(rows, vocab, dtype, layout, seed)
    y = _labels(rows, vocab, seed)
    g = torch.Generator(device=DEV).manual_seed(seed + 9)
    lp = _rows64(x, y)[1].float()
    step = torch.linspace(-0.65, 0.65, rows, device=DEV)  # log ratios on both sides of both clip edges, none on one
    old = lp - step
    ref = lp + 0.3 * torch.randn(rows, generator=g, device=DEV)
    adv = torch.randn(rows, generator=g, device=DEV)
    adv[rows // 2] = 0.0
    w = torch.rand(rows, generator=g, device=DEV) + 0.5
    return x, y, old, adv, ref, w


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("layout", ["plain", "padded", "shifted"])
@pytest.mark.parametrize("shape", [(2, 3), (70, 101), (300, 1000), (33, 4097), (14, 50257), (3, 131075)])
def test_policy_loss_both_forms(shape, layout, dtype):
    rows, vocab = shape
    x, y, old, adv, ref, w = _policy_inputs(rows, vocab, dtype, layout)
    gscale = 1024.0 if dtype == torch.float16 else 1.0
    for bonus, ckl, weights, temperature, given in ((0.0, 0.0, None, 1.0, False), (0.02, 0.1, w, 1.0, True),
                                                    (0.0, 0.1, None, 1.3, False)):
        denom = torch.full((), 3.0, device=DEV) if given else None
        want = _policy64(x, y, old, adv, ref, weights, 0.2, 0.28, ckl, bonus, temperature, denom, gscale)
        kw = dict(ref_logprobs=ref, weights=weights, clip_low=0.2, clip_high=0.28, kl_coef=ckl, entropy_coef=bonus,
                  temperature=temperature, denominator=denom)
        r, d = alignment.policy_loss_and_grad(x, y, old, adv, grad_scale=gscale, **kw)
        xg = x.detach().requires_grad_()
        r2 = alignment.policy_loss(xg, y, old, adv, **kw)
        d2, = torch.autograd.grad(r2.loss * gscale, xg)
        tol = _lp_tol(x, temperature)
        size = float(adv.abs().max()) * 2 + 1
        for got in (r, r2):
            # a token's loss moves by about (|A| r + c) times the log-probability's error
            assert abs(float(got.loss.detach()) - float(want[0])) <= 2 * size * tol * (rows / 3 if given else 1) + 1e-6
            assert float((got.logprobs.double() - want[1]).abs().max()) <= tol
            assert float((got.kl.double() - want[2]).abs().max()) <= 4 * tol
            assert abs(float(got.clip_fraction) - float(want[4])) <= 1e-6 * (rows if given else 1)
            if bonus:
                assert float((got.entropy.double() - want[3]).abs().max()) <= tol + 1e-5 * float(want[3].max())
            else:
                assert got.entropy is None
        ww = (y >= 0) if weights is None else w * (y >= 0)
        total = float(ww.double().sum()) if denom is None else 3.0
        g_h = -bonus * ww.double() * gscale / total if bonus else None
        for got in (d, d2):
            # the factor of a row (w/D)(A r + ...) is within 1e-5 of itself, beside the gradient's own tolerance
            logp = _rows64(x, y, temperature)[0]
            p = logp.exp()
            err = (got.double() - want[5]).abs()
            g = want[6].abs()[:, None]
            hot = torch.zeros_like(p).scatter_(1, y.clamp(min=0)[:, None], 1.0)
            span = (g + (w.double() * gscale / total * (1 + adv.double().abs()))[:, None] * 2) * (p + hot)
            if g_h is not None:
                span = span + g_h.abs()[:, None] * torch.where(p > 0, p * (logp.abs() + 12), torch.zeros_like(p))
            lim = HALF_ULP[dtype] * want[5].abs() + 4e-5 * span / temperature + SMALLEST[dtype]
            assert float((err - lim).max()) <= 0
            assert not got[y < 0].any()
    assert _lib.device_status() == 0


def test_policy_loss_per_sequence_advantages_and_shapes():
    B, T, V = 3, 5, 211
    x, y, old, adv, ref, w = _policy_inputs(B * T, V, torch.float32, "plain")
    per_seq = torch.tensor([0.5, -1.5, 2.0], device=DEV)
    a, da = alignment.policy_loss_and_grad(x.view(B, T, V), y.view(B, T), old.view(B, T), per_seq)
    b, db = alignment.policy_loss_and_grad(x, y, old, per_seq.repeat_interleave(T))
    assert a.logprobs.shape == (B, T) and da.shape == (B, T, V) and a.kl is None and a.entropy is None
    assert torch.equal(a.loss, b.loss) and torch.equal(da.view_as(db), db)
    r = alignment.policy_loss(x.view(B, T, V), y.view(B, T), old.view(B, T), per_seq, entropy=True)
    assert torch.equal(r.logprobs, a.logprobs) and r.entropy.shape == (B, T)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("vocab", [9, 1000, 50257])
def test_gradients_over_the_logits_in_place(vocab, dtype):
    """out=logits: the same bits as a separate gradient, whatever the row alignment."""
    rows = 37
    for layout in ("plain", "padded", "shifted"):
        x, y, old, adv, ref, w = _policy_inputs(rows, vocab, dtype, layout)
        _, d = alignment.policy_loss_and_grad(x, y, old, adv, entropy_coef=0.01)
        buf = _logits(rows, vocab, dtype, layout)
        assert torch.equal(buf, x)
        _, d2 = alignment.policy_loss_and_grad(buf, y, old, adv, entropy_coef=0.01, out=buf)
        assert d2.data_ptr() == buf.data_ptr() and torch.equal(d, buf)
        other = torch.full((rows, vocab + 5), 7.0, device=DEV, dtype=dtype)  # another stride than the logits'
        alignment.policy_loss_and_grad(x, y, old, adv, entropy_coef=0.01, out=other[:, 3:3 + vocab])
        assert torch.equal(other[:, 3:3 + vocab], d)
        assert bool((other[:, :3] == 7.0).all()) and bool((other[:, 3 + vocab:] == 7.0).all())
        pairs = x[:36].view(2, 18, vocab)
        _, d = alignment.preference_loss_and_grad(pairs, y[:36].view(2, 18), None)
        buf = _logits(rows, vocab, dtype, layout)
        alignment.preference_loss_and_grad(buf[:36].view(2, 18, vocab), y[:36].view(2, 18), None,
                                           out=buf[:36].view(2, 18, vocab))
        assert torch.equal(buf[:36].view_as(d), d) and torch.equal(buf[36:], x[36:])


def test_policy_gradient_agrees_with_differences():
    """Central differences of the loss along a random sign vector, step e: the loss is fp32 (2^-23 |L| / e) and its
    third derivative of order one (e^2 / 6)."""
    rows, vocab, e = 24, 301, 5e-3
    x, y, old, adv, ref, w = _policy_inputs(rows, vocab, torch.float32, "plain")
    kw = dict(ref_logprobs=ref, kl_coef=0.1, entropy_coef=0.05, weights=w)
    u = torch.randint(0, 2, x.shape, device=DEV, generator=torch.Generator(device=DEV).manual_seed(5)).float() * 2 - 1
    _, d = alignment.policy_loss_and_grad(x, y, old, adv, **kw)
    up, down = (float(alignment.policy_loss_and_grad(x + s * e * u, y, old, adv, **kw)[0].loss) for s in (1, -1))
    assert abs((up - down) / (2 * e) - float((d.double() * u).sum())) <= 3e-4


# ---------------------------------------------------------------- preference loss
def _preference64(x, y, ref, kind, beta, smoothing, average, temperature=1.0):
    z = x.double().requires_grad_()
    logp = torch.log_softmax(z / temperature, -1)
    valid = y >= 0
    lp = logp.gather(2, y.clamp(min=0)[..., None])[..., 0] * valid
    gap = ((lp - (0 if ref is None else ref.double())) * valid).sum(1)
    if average:
        gap = gap / valid.sum(1).clamp(min=1)
    n = x.shape[0] // 2
    diff = gap[:n] - gap[n:]
    u = beta * diff
    if kind == "sigmoid":
        ls = torch.nn.functional.logsigmoid
        loss = -((1 - smoothing) * ls(u) + smoothing * ls(-u)).mean()
    elif kind == "hinge":
        loss = torch.relu(1 - u).mean()
    else:
        loss = (diff - 1 / (2 * beta)).square().mean()
    d, g_lp = torch.autograd.grad(loss, [z, lp])
    return loss.detach(), beta * gap.detach(), lp.detach(), d, g_lp * valid


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("kind,beta,smoothing,average", [("sigmoid", 0.1, 0.0, False), ("sigmoid", 0.5, 0.2, True),
                                                         ("hinge", 0.05, 0.0, False), ("squared", 0.1, 0.0, True),
                                                         ("squared", 0.3, 0.0, False)])
@pytest.mark.parametrize("shape", [(1, 1, 5), (3, 7, 101), (2, 33, 1000), (5, 130, 515), (1, 9, 50257)])
def test_preference_loss_both_forms(shape, kind, beta, smoothing, average, dtype):
    pairs, length, vocab = shape
    rows = 2 * pairs * length
    x = _logits(rows, vocab, dtype, "padded" if length % 2 else "plain").view(2 * pairs, length, vocab)
    y = _labels(rows, vocab, ignored=0.4).view(2 * pairs, length)
    if pairs > 2:
        y[1] = -100  # a chosen sequence without a token
    g = torch.Generator(device=DEV).manual_seed(4)
    ref = _rows64(x, y)[1].float() + 0.3 * torch.randn(y.shape, generator=g, device=DEV)
    ref = torch.where(y >= 0, ref, torch.full_like(ref, math.nan))  # not read where there is no label
    clean = torch.nan_to_num(ref)
    want = _preference64(x, y, clean, kind, beta, smoothing, average)
    kw = dict(kind=kind, beta=beta, label_smoothing=smoothing, average=average)
    r, d = alignment.preference_loss_and_grad(x, y, ref, **kw)
    xg = x.detach().requires_grad_()
    r2 = alignment.preference_loss(xg, y, ref, **kw)
    d2, = torch.autograd.grad(r2.loss * 3.0, xg)
    tol = _lp_tol(x)
    # a gap sums at most `length` log-probabilities whose errors are independent or share a sign
    gap_tol = (1 if average else length) * tol
    slope = 2 * (float((want[1][:pairs] - want[1][pairs:]).abs().max()) / beta + 1 / (2 * beta)) if kind == "squared" else beta
    for got, scale in ((r, 1.0), (r2, 1.0)):
        assert float((got.logprobs.double() - want[2]).abs().max()) <= tol
        assert float((got.rewards.double() - want[1]).abs().max()) <= beta * gap_tol + 1e-6
        assert abs(float(got.loss.detach()) - float(want[0])) <= slope * 2 * gap_tol + 2.0 ** -22 * abs(float(want[0])) + 1e-7
    for got, scale in ((d, 1.0), (d2, 3.0)):
        # the row factors are those of 64 bits up to the slope's change over the gaps' error
        p = _rows64(x, y)[0].exp()
        hot = torch.zeros_like(p).scatter_(2, y.clamp(min=0)[..., None], 1.0)
        per = want[4].abs()[..., None] * scale
        bend = {"sigmoid": beta * beta / 4, "hinge": 0.0, "squared": 2.0}[kind] * 2 * gap_tol / pairs * scale
        lim = HALF_ULP[dtype] * want[3].abs() * scale + (3e-5 * per + bend) * (p + hot) + SMALLEST[dtype]
        assert float(((got.double() - want[3] * scale).abs() - lim).max()) <= 0
        assert not got[y < 0].any()
    assert _lib.device_status() == 0


def test_preference_gradient_agrees_with_differences():
    x = _logits(4 * 6, 53, torch.float32).view(4, 6, 53)
    y = _labels(24, 53).view(4, 6)
    u = torch.randint(0, 2, x.shape, device=DEV, generator=torch.Generator(device=DEV).manual_seed(5)).float() * 2 - 1
    for kind in ("sigmoid", "squared"):
        _, d = alignment.preference_loss_and_grad(x, y, None, kind=kind, beta=0.5)
        e = 5e-3
        up, down = (float(alignment.preference_loss_and_grad(x + s * e * u, y, None, kind=kind, beta=0.5)[0].loss) for s in (1, -1))
        slope = float((d.double() * u).sum())
        # fp32 loss: 2^-23 L / e; the gaps are sums of a dozen terms of size up to 8 with third derivatives of order 10
        assert abs((up - down) / (2 * e) - slope) <= 2.0 ** -22 * max(1.0, abs(up)) / e + 1e-3 * max(1.0, abs(slope))


# ---------------------------------------------------------------- how they are called
def test_other_stream_and_determinism():
    x, y, old, adv, ref, w = _policy_inputs(300, 5000, torch.bfloat16, "plain")
    a, da = alignment.policy_loss_and_grad(x, y, old, adv, ref_logprobs=ref, kl_coef=0.1)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        b, db = alignment.policy_loss_and_grad(x, y, old, adv, ref_logprobs=ref, kl_coef=0.1)
    torch.cuda.current_stream().wait_stream(s)
    assert torch.equal(a.loss, b.loss) and torch.equal(da, db) and torch.equal(a.kl, b.kl)


def test_captured_graph_replays_with_new_inputs():
    x, y, old, adv, ref, w = _policy_inputs(40, 5000, torch.bfloat16, "plain")
    alignment.policy_loss_and_grad(x, y, old, adv)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        r, d = alignment.policy_loss_and_grad(x, y, old, adv)
    x.copy_(_logits(40, 5000, torch.bfloat16, seed=8))
    graph.replay()
    r2, d2 = alignment.policy_loss_and_grad(x, y, old, adv)
    assert torch.equal(r.loss, r2.loss) and torch.equal(d, d2)


def test_offsets_beyond_32_bits():
    """Rows whose element offset passes 2^31: only the last few are labelled."""
    rows, vocab = 43000, 50257
    assert (rows - 1) * vocab > 2 ** 31
    x = torch.empty(rows, vocab, device=DEV, dtype=torch.bfloat16)
    x[-3:] = _logits(3, vocab, torch.bfloat16)
    y = torch.full((rows,), -100, device=DEV)
    y[-3:] = torch.tensor([5, 50256, 77], device=DEV)
    lp = alignment.token_logprobs(x, y)
    want = _rows64(x[-3:], y[-3:])[1]
    assert float((lp[-3:].double() - want).abs().max()) <= _lp_tol(x[-3:])
    tail = x[-3:].clone()
    r, d = alignment.policy_loss_and_grad(x, y, lp, torch.ones_like(lp), out=x)
    assert not d[:-3].any()
    _check_grad(d[-3:], tail, y[-3:], 1.0, torch.full((3,), -1 / 3, device=DEV))


def test_model_path_preference_and_policy_through_the_head():
    """backward_through_head on a reversible model: the preference loss's parameter gradients agree with autograd
    over the model's logits, in fp32."""
    import reversability_b200 as rb
    torch.manual_seed(0)
    model = rb.ReversibleLM(rb.ModelConfig(vocab_size=101, max_sequence_length=16, n_layers=2, n_heads=2, d_model=64,
                                           d_ff=128), "midpoint").to(DEV)
    g = torch.Generator(device=DEV).manual_seed(2)
    ids = torch.randint(0, 101, (4, 16), generator=g, device=DEV)
    y = torch.randint(0, 101, (4, 16), generator=g, device=DEV)
    y[:, :5] = -100
    loss = alignment.preference_loss(model(ids), y, None, beta=0.5).loss
    loss.backward()
    want = {n: p.grad.clone() for n, p in model.named_parameters()}
    model.zero_grad()
    r = alignment.backward_through_head(
        model, ids, lambda x, out: alignment.preference_loss_and_grad(x, y, None, beta=0.5, out=out), precision="fp32")
    assert abs(float(r.loss) - float(loss.detach())) <= 1e-6
    for n, p in model.named_parameters():
        assert float((p.grad - want[n]).norm()) <= 1e-5 * float(want[n].norm()), n
    assert _lib.device_status() == 0


def test_refusals():
    x = _logits(6, 40, torch.float32)
    y = torch.zeros(6, dtype=torch.int64, device=DEV)
    f = torch.zeros(6, device=DEV)
    bad = [
        lambda: alignment.token_logprobs(x, y.int()),
        lambda: alignment.token_logprobs(x, y[:5]),
        lambda: alignment.token_logprobs(x.double(), y),
        lambda: alignment.token_logprobs(x.t(), torch.zeros(40, dtype=torch.int64, device=DEV)),
        lambda: alignment.token_logprobs(x[:1].expand(6, 40), y),
        lambda: alignment.token_logprobs(x.view(2, 3, 40)[:, :2], torch.zeros(2, 2, dtype=torch.int64, device=DEV)),
        lambda: alignment.token_logprobs(x, y, temperature=0.0),
        lambda: alignment.token_logprobs(x, y.cpu()),
        lambda: alignment.policy_loss(x, y, f[:5], f),
        lambda: alignment.policy_loss(x, y, f, f[:5]),
        lambda: alignment.policy_loss(x, y, f, f, kl_coef=0.1),
        lambda: alignment.policy_loss(x, y, f, f, clip_low=-0.1),
        lambda: alignment.policy_loss(x, y, f.clone().requires_grad_(), f),
        lambda: alignment.policy_loss_and_grad(x, y, f, f, out=x.half()),
        lambda: alignment.policy_loss_and_grad(x, y, f, f, denominator=f),
        lambda: alignment.preference_loss(x, y, None),
        lambda: alignment.preference_loss(x[:3].view(3, 1, 40), y[:3].view(3, 1), None),
        lambda: alignment.preference_loss(x.view(2, 3, 40), y.view(2, 3), f),
        lambda: alignment.preference_loss(x.view(2, 3, 40), y.view(2, 3), None, kind="other"),
        lambda: alignment.preference_loss(x.view(2, 3, 40), y.view(2, 3), None, beta=0.0),
        lambda: alignment.preference_loss(x.view(2, 3, 40), y.view(2, 3), None, kind="hinge", label_smoothing=0.1),
    ]
    for k, call in enumerate(bad):
        with pytest.raises(ValueError):
            call()
            print("no refusal:", k)
    assert _lib.device_status() == 0


@pytest.mark.parametrize("shape,dtype", [((1500, 11003), torch.bfloat16), ((20011, 4301), torch.bfloat16),
                                         ((1025, 6001), torch.float32), ((1300, 61), torch.float16)])
@pytest.mark.parametrize("mask", ["blocks", "all", "none", "first"])
def test_many_rows_with_uneven_masks(shape, dtype, mask):
    """Row counts at which the rows are listed first: every labelled row is done once, every other is left at zero."""
    rows, vocab = shape
    x = _logits(rows, vocab, dtype, "padded")
    y = _labels(rows, vocab, ignored=0.0)
    if mask == "blocks":  # prompts and padding: runs of ignored rows, one label out of range
        y[(torch.arange(rows, device=DEV) % 100) < 60] = -100
        y[99] = vocab
    elif mask == "all":
        y[:] = -100
    elif mask == "first":
        y[1:] = -100
    valid = (y >= 0) & (y < vocab)
    clean = torch.where(valid, y, torch.full_like(y, -100))
    lp = alignment.token_logprobs(x, y)
    step = max(1, (1 << 27) // vocab)
    want = torch.cat([_rows64(x[s:s + step], clean[s:s + step])[1] for s in range(0, rows, step)])
    assert float((lp.double() - want).abs().max()) <= _lp_tol(x)
    assert not lp[~valid].any()
    old = torch.where(valid, lp, torch.zeros_like(lp))
    r, d = alignment.policy_loss_and_grad(x, y, old, torch.ones_like(lp), grad_scale=float(rows))
    n = max(int(valid.sum()), 1)
    assert abs(float(r.loss) + (1.0 if valid.any() else 0.0)) <= 1e-5 and not d[~valid].any()
    # the factor at the log-probabilities that the loss itself reports (they may be sums in another order than `lp`)
    g = -(r.logprobs.double() - old.double()).exp() * (float(rows) / n)
    for s in range(0, rows, step):
        _check_grad(d[s:s + step], x[s:s + step], clean[s:s + step], 1.0, g[s:s + step])
    assert torch.equal(r.logprobs, lp) or float((r.logprobs - lp).abs().max()) <= 2e-6 + _lp_tol(x)
    assert _lib.device_status() == (1 << 2 if mask == "blocks" else 0)


def test_refuses_what_overlaps_and_constants_out_of_range():
    buf = torch.randn(7, 100, device=DEV)
    x, y, f = buf[:6, :40], torch.zeros(6, dtype=torch.int64, device=DEV), torch.zeros(6, device=DEV)
    for out in (buf[:6, 1:41], buf[1:, :40], buf[:6, 39:79], buf.view(-1)[4:244].view(6, 40)):
        with pytest.raises(ValueError):
            alignment.policy_loss_and_grad(x, y, f, f, out=out)
    for kw in (dict(temperature=1e-39), dict(temperature=float("inf")), dict(ignore_index=2 ** 31),
               dict(ignore_index=-2 ** 31 - 1)):
        with pytest.raises(ValueError):
            alignment.token_logprobs(x, y, **kw)
    keep = x.clone()
    _, want = alignment.policy_loss_and_grad(x, y, f, f + 1)
    _, d = alignment.policy_loss_and_grad(x, y, f, f + 1, out=buf[:6, 50:90])  # beside the logits in the same rows
    assert torch.equal(d, want) and torch.equal(x, keep) and d.data_ptr() == buf[:6, 50:90].data_ptr()
    assert _lib.device_status() == 0


@pytest.mark.parametrize("layout", ["plain", "padded", "shifted"])
@pytest.mark.parametrize("shape,ignored", [((593, 16389), 0.3), ((1301, 25001), 0.0), ((2100, 17000), 0.97), ((600, 57343), 0.5)])
def test_many_long_fp32_rows(shape, ignored, layout):
    """Rows whose sums run beside the gradients of those before them: masks that leave few or uneven rows, masked
    columns, a row of nothing but the lowest value, the gradient over the logits and in rows of another stride."""
    rows, vocab = shape
    x = _logits(rows, vocab, torch.float32, layout, seed=5)
    y = _labels(rows, vocab, 5, ignored)
    low = torch.finfo(torch.float32).min
    x[1, vocab // 2:] = -math.inf
    x[2, vocab // 2:] = low
    x[rows - 1] = low
    y[:3] = torch.tensor([7, 11, 0], device=DEV)
    y[rows - 1] = vocab - 1
    g = torch.Generator(device=DEV).manual_seed(3)
    step = 290  # rows of one look at the 64-bit values
    lp64 = torch.cat([_rows64(x[s:s + step], y[s:s + step])[1] for s in range(0, rows, step)])
    old = (lp64 + 0.1 * torch.randn(rows, generator=g, device=DEV)).float()
    adv = torch.randn(rows, generator=g, device=DEV)
    kw = dict(clip_low=1.0, clip_high=10.0, entropy_coef=0.01, grad_scale=float(rows))
    r, d = alignment.policy_loss_and_grad(x, y, old, adv, **kw)
    valid = y >= 0
    n = int(valid.sum())
    assert float((r.logprobs.double() - lp64).abs().max()) <= _lp_tol(x)
    scale = float(rows) / n
    g_lp = -(r.logprobs.double() - old.double()).exp() * adv.double() * scale
    g_h = torch.full_like(g_lp, -0.01 * scale)
    for s in range(0, rows, step):
        _check_grad(d[s:s + step], x[s:s + step], y[s:s + step], 1.0, g_lp[s:s + step], g_h[s:s + step])
    assert not d[~valid].any()
    again, d2 = alignment.policy_loss_and_grad(x, y, old, adv, **kw)
    assert torch.equal(d, d2) and torch.equal(r.loss, again.loss)
    other = torch.full((rows, vocab + 6), 7.0, device=DEV)
    alignment.policy_loss_and_grad(x, y, old, adv, out=other[:, 3:3 + vocab], **kw)
    assert torch.equal(other[:, 3:3 + vocab], d) and bool((other[:, :3] == 7.0).all()) and bool((other[:, 3 + vocab:] == 7.0).all())
    buf = _logits(rows, vocab, torch.float32, layout)
    buf.copy_(x)
    _, d2 = alignment.policy_loss_and_grad(buf, y, old, adv, out=buf, **kw)
    assert d2.data_ptr() == buf.data_ptr() and torch.equal(buf, d)
    assert _lib.device_status() == 0


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("layout", ["plain", "shifted"])
@pytest.mark.parametrize("vocab", [61, 1003, 3001, 5003])
def test_many_short_rows(vocab, layout, dtype):
    """Row counts at which short rows are taken by a warp each, and weights and losses are summed by many CTAs."""
    rows = 5003
    x = _logits(rows, vocab, dtype, layout, seed=2)
    y = _labels(rows, vocab, 2)
    _, lp64, h64, valid = _rows64(x, y)
    g = torch.Generator(device=DEV).manual_seed(4)
    g_lp, g_h = (torch.randn(rows, generator=g, device=DEV) for _ in range(2))
    xg = x.detach().requires_grad_()
    lp, h = alignment.token_logprobs(xg, y, entropy=True)
    d, = torch.autograd.grad([lp, h], xg, [g_lp, g_h])
    assert float((lp.detach().double() - lp64).abs().max()) <= _lp_tol(x)
    _check_grad(d, x, y, 1.0, g_lp, g_h)
    assert not d[~valid].any()
    d, = torch.autograd.grad(alignment.token_logprobs(xg, y), xg, g_lp)
    _check_grad(d, x, y, 1.0, g_lp)
    w = torch.rand(rows, generator=g, device=DEV) + 0.5
    adv = torch.randn(rows, generator=g, device=DEV)
    old = (lp64 + 0.1 * torch.randn(rows, generator=g, device=DEV)).float()
    kw = dict(weights=w, clip_low=1.0, clip_high=10.0, entropy_coef=0.01)
    r, d = alignment.policy_loss_and_grad(x, y, old, adv, grad_scale=float(rows), **kw)
    r2 = alignment.policy_loss(xg, y, old, adv, **kw)
    d2, = torch.autograd.grad(r2.loss * float(rows), xg)
    ww = w.double() * valid
    terms = (lp64 - old.double()).exp() * adv.double() + 0.01 * h64
    want = -float((ww * terms).sum() / ww.sum())
    size = float((ww * terms.abs()).sum() / ww.sum())
    for got, grad in ((r, d), (r2, d2)):
        # each term is as far off as the log-probability in its exponent
        assert abs(float(got.loss.detach()) - want) <= 2 * _lp_tol(x) * (size + 1) + 1e-6
        ratio = (got.logprobs.double() - old.double()).exp()
        _check_grad(grad, x, y, 1.0, -ratio * adv.double() * ww * (rows / ww.sum()), -0.01 * ww * (rows / ww.sum()))
    assert _lib.device_status() == 0


@pytest.mark.parametrize("pairs,length", [(1, 257), (2, 1030), (3, 256)])
def test_preference_of_long_sequences(pairs, length):
    vocab = 37
    x = _logits(2 * pairs * length, vocab, torch.float32, seed=8)
    y = _labels(2 * pairs * length, vocab, 8)
    lp64 = _rows64(x, y)[1].view(2 * pairs, length)
    g = torch.Generator(device=DEV).manual_seed(5)
    ref = (lp64 + 0.05 * torch.randn(2 * pairs, length, generator=g, device=DEV)).float()
    x3, y2 = x.view(2 * pairs, length, vocab), y.view(2 * pairs, length)
    for average in (False, True):
        r, d = alignment.preference_loss_and_grad(x3, y2, ref, beta=0.2, average=average, grad_scale=float(pairs))
        valid = (y2 >= 0).double()
        n = valid.sum(1).clamp(min=1)
        per = 1 / n if average else torch.ones_like(n)
        gap = ((lp64 - ref.double()) * valid).sum(1) * per
        diff = 0.2 * (gap[:pairs] - gap[pairs:])
        want = torch.nn.functional.softplus(-diff)
        # a gap is off by its tokens' log-probabilities, which are not rounded before they are summed
        tol = _lp_tol(x) * float((n * per).max())
        assert float((r.rewards.double() - 0.2 * gap).abs().max()) <= 0.2 * tol + 1e-6
        assert abs(float(r.loss) - float(want.mean())) <= 0.4 * tol + 1e-6
        # the slope at the reported rewards
        slope = -0.2 * torch.sigmoid(r.rewards.double()[pairs:] - r.rewards.double()[:pairs])
        g_lp = torch.cat([slope, -slope])[:, None] * per[:, None] * valid
        _check_grad(d.view(-1, vocab), x, y, 1.0, g_lp.view(-1))
    assert _lib.device_status() == 0


def test_changing_what_was_returned_leaves_the_backward_alone():
    """Metrics are often reduced in place over processes before the backward; what that reads lies apart from them. The
    entropies, which the bonus's gradient is formed from, may not be changed."""
    x, y, old, adv, ref, w = _policy_inputs(12, 50, torch.float32, "plain")

    def policy(z):
        return alignment.policy_loss(z, y, old, adv, ref_logprobs=ref, kl_coef=0.1, entropy_coef=0.01)

    def preference(z):
        return alignment.preference_loss(z.view(2, 6, 50), y.view(2, 6), None)
    for make in (policy, preference):
        a, b = (x.clone().requires_grad_() for _ in range(2))
        want, = torch.autograd.grad(make(a).loss, a)
        r = make(b)
        for name, t in r._asdict().items():
            if name != "entropy" and t is not None:
                t.detach().mul_(3.0)
        got, = torch.autograd.grad(r.loss, b, retain_graph=True)
        assert torch.equal(got, want)
        loss = r.loss
        loss *= 0.5
        half, = torch.autograd.grad(loss, b)
        assert torch.equal(half, want * 0.5)
    r = policy(x.clone().requires_grad_())
    r.entropy.mul_(3.0)
    with pytest.raises(RuntimeError, match="inplace"):
        r.loss.backward()


def test_a_loss_that_saved_the_logits_notices_gradients_written_over_them():
    x, y, old, adv, ref, w = _policy_inputs(12, 50, torch.float32, "plain")
    others = torch.zeros_like(x)
    for write in (lambda z: alignment.policy_loss_and_grad(z.detach(), y, old, adv, out=z.detach()),
                  lambda z: alignment.preference_loss_and_grad(z.detach().view(2, 6, 50), y.view(2, 6), None,
                                                               out=z.detach().view(2, 6, 50))):
        for loss in (lambda z: alignment.token_logprobs(z, y).sum(), lambda z: alignment.policy_loss(z, y, old, adv).loss,
                     lambda z: alignment.preference_loss(z.view(2, 6, 50), y.view(2, 6), None).loss):
            z = x.clone().requires_grad_()
            kept = loss(z)
            write(z)
            with pytest.raises(RuntimeError, match="inplace"):
                kept.backward()
    z = x.clone().requires_grad_()
    kept = alignment.token_logprobs(z, y).sum()
    alignment.policy_loss_and_grad(z.detach(), y, old, adv, out=others)  # the logits stay as they are
    kept.backward()
    with torch.inference_mode():  # such tensors have no such count
        z = x.clone()
        alignment.policy_loss_and_grad(z, y, old, adv, out=z)


def test_out_may_name_the_same_rows_by_other_strides():
    """Dimensions of size 1 may have any stride; rows that start together and lie apart otherwise are refused."""
    full = torch.randn(2, 4, 60, device=DEV)
    y, f = torch.tensor([[3]], device=DEV), torch.zeros(1, 1, device=DEV)
    x = full[:1, :1]
    _, want = alignment.policy_loss_and_grad(x, y, f, f + 1)
    same = full.view(8, 60)[:1].view(1, 1, 60).as_strided((1, 1, 60), (60, 7, 1))
    assert same.stride() != x.stride()
    _, d = alignment.policy_loss_and_grad(x, y, f, f + 1, out=same)
    assert torch.equal(x, want) and d.data_ptr() == x.data_ptr()
    y, f = torch.zeros(1, 2, dtype=torch.int64, device=DEV), torch.zeros(1, 2, device=DEV)
    x = full.view(8, 60)[:3:2][None]
    _, want = alignment.policy_loss_and_grad(x, y, f, f + 1)
    same = full.view(8, 60).as_strided((1, 2, 60), (9999, 120, 1))
    alignment.policy_loss_and_grad(x, y, f, f + 1, out=same)
    assert torch.equal(x, want)
    with pytest.raises(ValueError, match="strides"):
        alignment.policy_loss_and_grad(x, y, f, f + 1, out=full.view(8, 60)[:2][None])


def _check_policy_rows(x, y, layout, seed, entropy_coef=0.01):
    """The policy loss with its gradient against 64 bits, again (the same bits), over the logits and in rows of another
    stride. The rows' factors are the kernel's own: an exponential (2 ulp) and six roundings, 10 * 2^-24."""
    rows, vocab = x.shape
    dtype = x.dtype
    g = torch.Generator(device=DEV).manual_seed(seed)
    step = max(1, (1 << 24) // vocab)
    lp64 = torch.cat([_rows64(x[s:s + step], y[s:s + step])[1] for s in range(0, rows, step)])
    old = (lp64 + 0.1 * torch.randn(rows, generator=g, device=DEV)).float()
    adv = torch.randn(rows, generator=g, device=DEV)
    kw = dict(clip_low=1.0, clip_high=10.0, entropy_coef=entropy_coef, grad_scale=float(rows))
    r, d = alignment.policy_loss_and_grad(x, y, old, adv, **kw)
    valid = y >= 0
    assert float((r.logprobs.double() - lp64).abs().max()) <= _lp_tol(x)
    scale = float(rows) / int(valid.sum())
    g_lp = -(r.logprobs.double() - old.double()).exp() * adv.double() * scale
    g_h = torch.full_like(g_lp, -entropy_coef * scale)
    for s in range(0, rows, step):
        logp, _, h, _ = _rows64(x[s:s + step], y[s:s + step])
        p, at = logp.exp(), y[s:s + step].clamp(min=0)[:, None]
        gl, gh = ((t[s:s + step] * valid[s:s + step])[:, None] for t in (g_lp, g_h))
        inner = torch.where(p > 0, p * (logp + h[:, None]), torch.zeros_like(p))
        want = (-gl * p - gh * inner).scatter_add_(1, at, gl)
        near = gl.abs() * p + gh.abs() * torch.where(p > 0, p * (logp.abs() + h[:, None] + 1), torch.zeros_like(p))
        near.scatter_add_(1, at, gl.abs() * p.gather(1, at))
        # as in _check_grad, and the factor's own error where it stands alone
        lim = (HALF_ULP[dtype] + 2.0 ** -22) * want.abs() + 2e-5 * near + SMALLEST[dtype]
        lim.scatter_add_(1, at, 10 * 2.0 ** -24 * gl.abs())
        assert float(((d[s:s + step].double() - want).abs() - lim).max()) <= 0
    assert not d[~valid].any()
    again, d2 = alignment.policy_loss_and_grad(x, y, old, adv, **kw)
    assert torch.equal(d, d2) and torch.equal(r.loss, again.loss)
    other = torch.full((rows, vocab + 6), 7.0, device=DEV, dtype=dtype)
    alignment.policy_loss_and_grad(x, y, old, adv, out=other[:, 3:3 + vocab], **kw)
    assert torch.equal(other[:, 3:3 + vocab], d) and bool((other[:, :3] == 7.0).all()) and bool((other[:, 3 + vocab:] == 7.0).all())
    buf = _logits(rows, vocab, dtype, layout)
    buf.copy_(x)
    _, d2 = alignment.policy_loss_and_grad(buf, y, old, adv, out=buf, **kw)
    assert d2.data_ptr() == buf.data_ptr() and torch.equal(buf, d)
    assert _lib.device_status() == 0


@pytest.mark.parametrize("layout", ["plain", "shifted"])
@pytest.mark.parametrize("rows,vocab,dtype", [(200, 131075, torch.bfloat16), (200, 131075, torch.float16), (200, 131075, torch.float32),
                                              (500, 50257, torch.float32), (400, 100003, torch.bfloat16), (310, 114689, torch.float16)])
def test_rows_longer_than_their_ring(rows, vocab, dtype, layout):
    """Rows whose first chunks pass through the ring twice, several of them a CTA: the second time while the rest of the
    row is written over. Uneven masks, masked columns, a row of nothing but the lowest value."""
    x = _logits(rows, vocab, dtype, layout, seed=6)
    y = _labels(rows, vocab, 6)
    y[150:190] = -100
    y[:4] = torch.tensor([7, 11, vocab // 3, vocab - 1], device=DEV)
    x[1, vocab // 2:] = -math.inf
    x[2, vocab // 2:] = torch.finfo(dtype).min
    x[3] = torch.finfo(dtype).min
    for bonus in (0.01, 0.0):
        _check_policy_rows(x, y, layout, 7, bonus)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("layout", ["plain", "shifted"])
@pytest.mark.parametrize("rows,vocab", [(5, 131075), (9, 50257), (2, 300007)])
def test_few_long_rows_of_the_lowest_value(rows, vocab, layout, dtype):
    """Rows that a cluster shares and forms again relative to their largest element, while the gradient goes over the logits."""
    x = _logits(rows, vocab, dtype, layout, seed=9)
    y = _labels(rows, vocab, 9, 0.0)
    for r in range(0, rows, 2):
        x[r] = torch.finfo(dtype).min
    if dtype != torch.float16:
        x[1] -= 3e7  # a finite reference beyond what x c is exact for
        x[1, vocab // 2] = x[1].max()
    _check_policy_rows(x, y, layout, 3)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("vocab", [101, 1000, 8192, 50257])
def test_losses_have_no_bias_of_the_exponential_unit(vocab, dtype):
    """Mean signed error of the log-probabilities that enter a preference loss, seen through rewards of sequences of one
    token whose reference is the 64-bit value rounded to fp32. What is taken out for the exponential unit is 8e-8: the
    mean may be no further off than that, beside 2^-26 (the rounding of log2 e) of the label's distance from the mean
    logit under p and, where exponentials are exact, 2^-24 of a logit in base 2 (the rounding of the reference)."""
    rows = 4096 if vocab < 20000 else 1024
    for spread in (0.0, 0.01, 0.1, 0.5, 1.0, 2.0, 4.0, 8.0):
        g = torch.Generator(device=DEV).manual_seed(1)
        x = (torch.randn(rows, vocab, generator=g, device=DEV) * spread + 0.37).to(dtype)
        y = torch.randint(0, vocab, (rows,), generator=g, device=DEV)
        lp, far = [], []
        for s in range(0, rows, 256):
            z = x[s:s + 256].double()
            logp = torch.log_softmax(z, -1)
            lp.append(logp.gather(1, y[s:s + 256, None])[:, 0])
            far.append((logp.exp() * z).sum(1) - z.gather(1, y[s:s + 256, None])[:, 0])
        lp, far = torch.cat(lp), torch.cat(far)
        ref = lp.float()
        r = alignment.preference_loss(x.view(rows, 1, vocab), y.view(rows, 1), ref.view(rows, 1), beta=1.0)
        mean = float((r.rewards.double() - (lp - ref.double())).mean())
        tied = 2.0 ** -24 * 0.37 * 1.4427 if spread == 0.0 else 0.0
        assert abs(mean) <= 8e-8 + 2.0 ** -26 * abs(float(far.mean())) + tied


def test_out_beside_the_logits_with_wider_rows():
    """Neighbours in memory, as an allocator hands them out, are not refused for the stride of the one behind."""
    buf = torch.randn(2000, device=DEV)
    y, f = torch.zeros(6, dtype=torch.int64, device=DEV), torch.zeros(6, device=DEV)
    narrow, wide = (lambda at: buf[at:at + 240].view(6, 40)), (lambda at: buf[at:at + 360].view(6, 60)[:, :40])
    for x, out in ((narrow(0), wide(240)), (wide(0), narrow(340)), (wide(240), narrow(0)), (narrow(340), wide(0))):
        keep = x.clone()
        _, want = alignment.policy_loss_and_grad(x, y, f, f + 1)
        _, d = alignment.policy_loss_and_grad(x, y, f, f + 1, out=out)
        assert torch.equal(d, want) and torch.equal(x, keep) and d.data_ptr() == out.data_ptr()
    for x, out in ((narrow(0), wide(239)), (wide(0), narrow(339)), (wide(239), narrow(0)), (narrow(339), wide(0))):
        with pytest.raises(ValueError, match="overlaps"):
            alignment.policy_loss_and_grad(x, y, f, f + 1, out=out)
