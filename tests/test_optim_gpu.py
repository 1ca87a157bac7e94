"""AdamW over many tensors (optim.py) against the update in 64 bits.

Tolerances, derived from the arithmetic: each of m, v and p takes a handful of
fp32 operations (2^-24 relative each) and an approximate root and quotient
(2^-21 together), so one step is within 2^-20 of the moments' and the update's
own size; errors of several steps add up. 8-bit codes are compared as codes:
they may differ by one where the unrounded code lies within 1e-3 of a half."""
import math

import pytest
import torch

from reversability_b200 import _lib, optim

pytestmark = pytest.mark.gpu
DEV = "cuda"
SIZES = [1, 3, 4, 127, 255, 256, 257, 1000, 2047, 2048, 2049, 40961, 3 * 2048 * 7 + 5]
HP = dict(lr=1e-2, betas=(0.9, 0.95), eps=1e-8, weight_decay=0.1)


def _tensors(sizes, dtype=torch.float32, seed=0, offset=0, scale=1.0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    return [(torch.randn(n + offset, generator=g, device=DEV) * scale).to(dtype)[offset:] for n in sizes]


def _params(sizes, dtype=torch.float32, offset=0):
    return [torch.nn.Parameter(t) for t in _tensors(sizes, dtype, 1, offset, 0.1)]


class Ref:
    """The update in 64 bits over a list of tensors; 8-bit moments pass through their codes after each step."""

    def __init__(self, params, bits=32, max_norm=None, lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=1e-2):
        self.p = [p.detach().double().clone() for p in params]
        self.m = [torch.zeros_like(p) for p in self.p]
        self.v = [torch.zeros_like(p) for p in self.p]
        self.bits, self.max_norm, self.t = bits, max_norm, 0
        self.lr, self.betas, self.eps, self.wd = lr, betas, eps, weight_decay

    def step(self, grads):
        self.t += 1
        b1, b2 = self.betas
        g64 = [g.double() for g in grads]
        self.norm = math.sqrt(sum(float((g * g).sum()) for g in g64))
        coef = 1.0 if self.max_norm is None else min(1.0, self.max_norm / (self.norm + 1e-6))
        for i, g in enumerate(g64):
            g = g * coef
            self.m[i] = b1 * self.m[i] + (1 - b1) * g
            self.v[i] = b2 * self.v[i] + (1 - b2) * g * g
            hat = self.m[i] / (1 - b1 ** self.t) / ((self.v[i] / (1 - b2 ** self.t)).sqrt() + self.eps)
            self.p[i] = self.p[i] * (1 - self.lr * self.wd) - self.lr * hat


def _codes64(m, v):
    """Unrounded codes and scales of 8-bit moments for fp64 moments: (code of m, code of v, scales)."""
    n = m.numel()
    pad = -n % 256
    mb = torch.nn.functional.pad(m, (0, pad)).view(-1, 256)
    rb = torch.nn.functional.pad(v.sqrt(), (0, pad)).view(-1, 256)
    ms, rs = mb.abs().amax(1), rb.amax(1)
    safe = lambda t: torch.where(t > 0, t, torch.ones_like(t))[:, None]  # noqa: E731
    cm = 127 * (mb.abs() / safe(ms)).sqrt() * mb.sign()
    cv = 255 * (rb / safe(rs)).sqrt()
    return cm.view(-1)[:n], torch.where(cv > 0, cv.clamp(min=1.0), cv).view(-1)[:n], ms, rs


def _set(params, grads):
    for p, g in zip(params, grads):
        p.grad = g


@pytest.mark.parametrize("offset", [0, 1, 2])
@pytest.mark.parametrize("max_norm", [None, 0.5])
def test_32_bit_moments_against_64_bits(max_norm, offset):
    params = _params(SIZES, offset=offset)
    opt = optim.AdamW(params, max_norm=max_norm, **HP)
    ref = Ref(params, max_norm=max_norm, **HP)
    steps = 7
    for k in range(steps):
        grads = _tensors(SIZES, seed=10 + k, offset=offset)
        _set(params, grads)
        opt.step()
        ref.step(grads)
        if max_norm is not None:
            assert abs(float(opt.grad_norm) - ref.norm) <= 1e-5 * ref.norm
    # Adam's update is at most lr / (1 - b1) a step whatever the gradient's size; the clip coefficient
    # carries the norm's 1e-6 but cancels in the update
    for p, m, v, q in zip(ref.p, ref.m, ref.v, params):
        st = opt.state[q]
        assert float((q.detach().double() - p).abs().max()) <= steps * (2.0 ** -20 * HP["lr"] * 10 + 2.0 ** -23 * float(p.abs().max()))
        assert float((st["exp_avg"].double() - m).abs().max()) <= steps * 3e-6 * float(m.abs().max())
        assert float((st["exp_avg_sq"].double() - v).abs().max()) <= steps * 3e-6 * float(v.abs().max())


def test_matches_torch_adamw_on_a_model():
    torch.manual_seed(0)
    a = torch.nn.Sequential(torch.nn.Linear(37, 300), torch.nn.GELU(), torch.nn.Linear(300, 11)).to(DEV)
    b = torch.nn.Sequential(torch.nn.Linear(37, 300), torch.nn.GELU(), torch.nn.Linear(300, 11)).to(DEV)
    b.load_state_dict(a.state_dict())
    oa = optim.AdamW(a.parameters(), max_norm=1.0, **HP)
    ob = torch.optim.AdamW(b.parameters(), **HP)
    x = torch.randn(64, 37, device=DEV)
    for k in range(5):
        grads = [torch.randn(p.shape, device=DEV, generator=torch.Generator(device=DEV).manual_seed(k)) for p in a.parameters()]
        _set(a.parameters(), [g.clone() for g in grads])
        _set(b.parameters(), [g.clone() for g in grads])
        oa.step()
        torch.nn.utils.clip_grad_norm_(b.parameters(), 1.0)
        ob.step()
        for pa, pb in zip(a.parameters(), b.parameters()):
            assert float((pa - pb).detach().abs().max()) <= 2.0 ** -18 * HP["lr"] * 10 * (k + 1) + 1e-7


@pytest.mark.parametrize("p_dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("g_dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("bits", [32, 8])
def test_parameter_and_gradient_types(bits, p_dtype, g_dtype):
    params = _params([300, 2049, 7], p_dtype)
    opt = optim.AdamW(params, state_bits=bits, **HP)
    ref = Ref(params, **HP)
    grads = _tensors([300, 2049, 7], g_dtype, seed=3)
    if p_dtype == g_dtype:
        _set(params, grads)
        opt.step()
    else:
        opt.step(grads=grads)
    ref.step(grads)
    ulp = {torch.float32: 2.0 ** -23, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}[p_dtype]
    for p, q in zip(ref.p, params):
        assert float(((q.detach().double() - p).abs() - ulp * p.abs()).max()) <= 2.0 ** -20 * HP["lr"] * 10
        assert q.dtype == p_dtype


@pytest.mark.parametrize("offset", [0, 1, 4])
def test_8_bit_moments_against_64_bits(offset):
    """Each step is compared from the framework's own codes before it, so that errors do not pile up."""
    params = _params(SIZES, offset=offset)
    opt = optim.AdamW(params, state_bits=8, max_norm=0.7, **HP)
    for k in range(4):
        grads = _tensors(SIZES, seed=20 + k, offset=offset)
        grads[5].zero_()  # a tensor whose gradient vanishes
        if k == 0:
            grads[7][10:200] = 0.0
        ref = Ref(params, max_norm=0.7, **HP)
        ref.t = k
        if k:
            ref.m, ref.v = ([t.double() for t in ts] for ts in zip(*opt.moments()))
        _set(params, grads)
        opt.step()
        ref.step(grads)
        for i, q in enumerate(params):
            st = opt.state[q]
            # coefficients and moments within 3e-6, so the update within 1e-5 of lr / (1 - b1)
            assert float((q.detach().double() - ref.p[i]).abs().max()) <= 1e-5 * HP["lr"] * 10 + 2.0 ** -23 * float(ref.p[i].abs().max())
            cm, cv, ms, rs = _codes64(ref.m[i], ref.v[i])
            assert float((st["exp_avg_scale"].double() - ms).abs().max()) <= 1e-5 * float(ms.max())
            assert float((st["exp_avg_sq_scale"].double() - rs).abs().max()) <= 1e-5 * float(rs.max())
            assert float((st["exp_avg"].double() - cm).abs().max()) <= 0.5 + 1e-3
            assert float((st["exp_avg_sq"].double() - cv).abs().max()) <= 0.5 + 1e-3
            assert bool(((st["exp_avg_sq"] > 0) == (ref.v[i] > 0)).all())
    # the decoded values: m = scale c|c| / 127^2, v = (scale c^2 / 255^2)^2, in fp32 and in bf16
    for (m, v), (mb, vb), q in zip(opt.moments(), opt.moments(dtype=torch.bfloat16), params):
        st, n = opt.state[q], q.numel()
        c, d = st["exp_avg"].double(), st["exp_avg_sq"].double()
        ms = st["exp_avg_scale"].double().repeat_interleave(256)[:n]
        rs = st["exp_avg_sq_scale"].double().repeat_interleave(256)[:n]
        want_m, want_v = ms * c * c.abs() / 127 ** 2, (rs * d * d / 255 ** 2) ** 2
        assert float((m.double() - want_m).abs().max()) <= 2.0 ** -21 * float(want_m.abs().max())
        assert float((v.double() - want_v).abs().max()) <= 2.0 ** -20 * float(want_v.max())
        assert torch.equal(mb, m.bfloat16()) and torch.equal(vb, v.bfloat16())


def test_8_bit_moments_follow_32_bits_over_many_steps():
    """600 steps on noisy gradients of very different sizes: the 8-bit second moment's root follows the 32-bit one
    within 25 % at nearly all elements, and no element's update runs away."""
    n = 4096
    a, b = torch.nn.Parameter(torch.zeros(n, device=DEV)), torch.nn.Parameter(torch.zeros(n, device=DEV))
    hp = dict(lr=1e-3, betas=(0.9, 0.99), eps=1e-8, weight_decay=0.0)
    oa, ob = optim.AdamW([a], state_bits=8, **hp), optim.AdamW([b], **hp)
    g = torch.Generator(device=DEV).manual_seed(0)
    size = torch.exp(torch.randn(n, generator=g, device=DEV))
    for _ in range(600):
        grad = torch.randn(n, generator=g, device=DEV) * size
        a.grad, b.grad = grad, grad
        oa.step()
        ob.step()
    (_, v8), = oa.moments()
    ratio = (v8 / ob.state[b]["exp_avg_sq"]).sqrt()
    assert 0.97 <= float(ratio.mean()) <= 1.03
    assert float(((ratio - 1).abs() < 0.25).float().mean()) >= 0.97
    assert float((a - b).detach().abs().max()) <= 0.1 and float(a.detach().abs().max()) <= 0.6


def test_zero_gradients_nan_and_infinity():
    for bits in (32, 8):
        p, q = _params([600, 600])
        opt = optim.AdamW([p, q], state_bits=bits, **HP)
        before = p.detach().clone()
        p.grad, q.grad = torch.zeros_like(p), torch.zeros_like(q)
        q.grad[300] = math.nan
        q.grad[5] = math.inf
        opt.step()
        # nothing but decay where the gradient is zero
        assert torch.allclose(p.detach(), before * (1 - HP["lr"] * HP["weight_decay"]), rtol=2.0 ** -22, atol=0)
        assert bool(q[300].isnan()) and bool(q[100].isfinite()) and bool(q[599].isfinite())
        if bits == 8:  # the scales of the blocks that saw them say so; the third block does not
            m, v = opt.moments()[1]
            assert not bool(m[256:512].isfinite().any() & m[300:301].isfinite().all())
            assert bool(m[512:].isfinite().all()) and bool(v[512:].isfinite().all())
    # a NaN norm shows in every parameter
    p, q = _params([600, 600])
    opt = optim.AdamW([p, q], max_norm=1.0, **HP)
    p.grad, q.grad = torch.ones_like(p), torch.full_like(q, math.nan)
    opt.step()
    assert math.isnan(float(opt.grad_norm)) and bool(p.isnan().all())


@pytest.mark.parametrize("bits", [32, 8])
def test_more_tensors_than_one_launch_groups_and_missing_gradients(bits):
    sizes = [(7 * i) % 900 + (0 if i % 13 == 5 else 1) for i in range(150)]
    sizes[5] = 0
    params = _params(sizes)
    groups = [dict(params=params[:70], state_bits=bits), dict(params=params[70:], lr=3e-2, state_bits=32)]
    opt = optim.AdamW(groups, max_norm=2.0, **HP)
    grads = _tensors(sizes, seed=4)
    _set(params, grads)
    params[3].grad = None
    params[100].grad = None
    kept = [params[3].detach().clone(), params[100].detach().clone()]
    live = [i for i in range(150) if i not in (3, 100)]
    a = Ref([params[i] for i in live if i < 70], **HP)
    b = Ref([params[i] for i in live if i >= 70], **dict(HP, lr=3e-2))
    norm = math.sqrt(sum(float(grads[i].double().square().sum()) for i in live))
    opt.step()
    for r, idx in ((a, [i for i in live if i < 70]), (b, [i for i in live if i >= 70])):
        r.step([grads[i].double() * min(1.0, 2.0 / (norm + 1e-6)) for i in idx])
        for p, i in zip(r.p, idx):
            if p.numel():
                assert float((params[i].detach().double() - p).abs().max()) <= 1e-5 * r.lr * 10 + 2.0 ** -22
    assert abs(float(opt.grad_norm) - norm) <= 1e-5 * norm
    assert torch.equal(params[3], kept[0]) and torch.equal(params[100], kept[1])
    assert len(opt.state[params[3]]) == 0


@pytest.mark.parametrize("bits", [32, 8])
def test_state_dict_round_trip(bits, tmp_path):
    params = _params([300, 2049], torch.bfloat16)
    twin = [torch.nn.Parameter(p.detach().clone()) for p in params]
    opt = optim.AdamW(params, state_bits=bits, **HP)
    for k in range(3):
        _set(params, _tensors([300, 2049], torch.bfloat16, seed=k))
        opt.step()
    torch.save(opt.state_dict(), tmp_path / "opt.pt")
    for p, q in zip(params, twin):
        q.data.copy_(p.data)
    other = optim.AdamW(twin, state_bits=bits, **dict(HP, lr=0.5))
    other.load_state_dict(torch.load(tmp_path / "opt.pt", map_location="cpu"))
    assert other.param_groups[0]["lr"] == HP["lr"]
    for p, q in zip(params, twin):
        for k, v in opt.state[p].items():
            assert other.state[q][k].dtype == v.dtype and torch.equal(other.state[q][k], v)
    grads = _tensors([300, 2049], torch.bfloat16, seed=9)
    _set(params, grads)
    _set(twin, grads)
    opt.step()
    other.step()
    for p, q in zip(params, twin):
        assert torch.equal(p, q)


def test_captured_graph_counts_steps_and_takes_a_new_learning_rate():
    params, twin = _params([300, 2049]), _params([300, 2049])
    a, b = optim.AdamW(params, max_norm=1.0, **HP), optim.AdamW(twin, max_norm=1.0, **HP)
    grads = _tensors([300, 2049], seed=2)
    _set(params, grads)
    _set(twin, grads)
    a.step()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        a.step()
    for lr in (1e-2, 1e-2, 3e-3):
        a.param_groups[0]["lr"] = lr
        a.sync_lr()
        graph.replay()
    for lr in (1e-2, 1e-2, 1e-2, 3e-3):
        b.param_groups[0]["lr"] = lr
        b.step()
    for p, q in zip(params, twin):
        assert torch.equal(p, q)
    assert float(a.param_groups[0]["scalars"][1]) == 4.0


def test_scheduler_closure_and_noncontiguous_gradient():
    p = torch.nn.Parameter(torch.ones(20, 30, device=DEV))
    q = torch.nn.Parameter(torch.ones(20, 30, device=DEV))
    opt, ref = optim.AdamW([p], **HP), optim.AdamW([q], **HP)
    sched = torch.optim.lr_scheduler.LambdaLR(opt, lambda k: 0.5 ** k)
    g = torch.randn(30, 20, device=DEV).t()
    p.grad, q.grad = g, g.contiguous()

    def closure():
        return torch.tensor(3.0)
    assert float(opt.step(closure)) == 3.0
    ref.step()
    assert torch.equal(p, q)
    sched.step()
    opt.step()
    ref.param_groups[0]["lr"] = HP["lr"] / 2
    ref.step()
    assert torch.equal(p, q)


def test_refusals():
    p = _params([10])[0]
    for kw in (dict(state_bits=16), dict(lr=-1.0), dict(betas=(1.0, 0.9)), dict(eps=-1e-8), dict(max_norm=0.0)):
        with pytest.raises(ValueError):
            optim.AdamW([p], **kw)
    with pytest.raises(ValueError, match="CUDA"):
        optim.AdamW([torch.nn.Parameter(torch.zeros(3))])
    with pytest.raises(ValueError):
        optim.AdamW([torch.nn.Parameter(torch.zeros(3, 4, device=DEV).t())])
    with pytest.raises(ValueError):
        optim.AdamW([torch.nn.Parameter(torch.zeros(3, device=DEV, dtype=torch.float64))])
    opt = optim.AdamW([p], **HP)
    with pytest.raises(ValueError):
        opt.step(grads=[torch.zeros(9, device=DEV)])
    with pytest.raises(ValueError):
        opt.step(grads=[torch.zeros(10, device=DEV, dtype=torch.float64)])
    opt8 = optim.AdamW([p], state_bits=8, **HP)
    opt8.step(grads=[torch.zeros(10, device=DEV)])
    with pytest.raises(ValueError):
        opt8.moments(out=[])
    assert _lib.device_status() == 0


@pytest.mark.parametrize("bits", [8, 32])
def test_tensors_moved_between_steps(bits):
    """Parameters and moments that get other memory between steps are found there."""
    a, b = _params([300, 5000, 7]), _params([300, 5000, 7])
    opt, ref = optim.AdamW(a, state_bits=bits, **HP), optim.AdamW(b, state_bits=bits, **HP)
    held = []  # what the tensors left must not be handed out again
    for k in range(4):
        g = _tensors([300, 5000, 7], seed=20 + k)
        opt.step(grads=g)
        ref.step(grads=[t.clone() for t in g])
        for p, q in zip(a, b):
            assert torch.equal(p, q)
        for p in a:
            for t in (p, *(t for t in opt.state[p].values() if isinstance(t, torch.Tensor))):
                held.append(t.data)
                t.data = t.data.clone()
                held[-1].zero_()
        if bits == 8:
            for (m, v), (mr, vr) in zip(opt.moments(), ref.moments()):
                assert torch.equal(m, mr) and torch.equal(v, vr)
    state = opt.state[a[1]]
    state["exp_avg_sq"] = state["exp_avg_sq"].clone()
    g = _tensors([300, 5000, 7], seed=30)
    opt.step(grads=g)
    ref.step(grads=g)
    assert all(torch.equal(p, q) for p, q in zip(a, b))


def test_refuses_tensors_that_left_the_device():
    p = _params([100])[0]
    g = torch.ones(100, device=DEV)
    opt = optim.AdamW([p], state_bits=8, **HP)
    opt.step(grads=[g])
    before = p.detach().clone()
    for name in ("exp_avg", "exp_avg_sq", "exp_avg_scale", "exp_avg_sq_scale"):
        t = opt.state[p][name]
        there = t.data
        t.data = there.cpu()
        with pytest.raises(ValueError):
            opt.step(grads=[g])
        with pytest.raises(ValueError):
            opt.moments()
        t.data = there
    there, p.data = p.data, p.data.cpu()
    for h in (g, g.cpu()):
        with pytest.raises(ValueError):
            opt.step(grads=[h])
    p.data = there
    with pytest.raises(ValueError):
        opt.step(grads=[g.cpu()])
    assert torch.equal(p, before) and float(opt.param_groups[0]["scalars"][1]) == 1.0
    opt.step(grads=[g])
    assert not torch.equal(p, before) and _lib.device_status() == 0


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("given", [False, True])
@pytest.mark.parametrize("max_norm", [None, 0.5])
def test_a_group_added_after_a_step(max_norm, given, bits):
    """Layers unfrozen during tuning: their first update is that of a new optimizer, within the clip over all groups."""
    sizes = [300, 2049, 7, 513]
    params = _params(sizes)
    opt = optim.AdamW(params[:2], max_norm=max_norm, state_bits=bits, **HP)
    old, new = Ref(params[:2], **HP), Ref(params[2:], **dict(HP, lr=3e-2))
    for k in range(2):  # within the second step the moments of 8 bits have been rounded once
        grads = _tensors(sizes, seed=40 + k)
        live = grads[:2] if k == 0 else grads
        if k == 1:
            opt.add_param_group(dict(params=params[2:], lr=3e-2))
            if bits == 8:
                old.m, old.v = ([t.double() for t in ts] for ts in zip(*opt.moments()))
        norm = math.sqrt(sum(float(g.double().square().sum()) for g in live))
        coef = 1.0 if max_norm is None else min(1.0, max_norm / (norm + 1e-6))
        if given:
            opt.step(grads=live)
        else:
            _set(params, live)
            opt.step()
        old.step([g.double() * coef for g in live[:2]])
        if k == 1:
            new.step([g.double() * coef for g in live[2:]])
        if max_norm is not None:
            assert abs(float(opt.grad_norm) - norm) <= 1e-5 * norm
    for q, p, lr in [(q, p, HP["lr"]) for q, p in zip(params, old.p)] + [(q, p, 3e-2) for q, p in zip(params[2:], new.p)]:
        # the tolerance of a step with 8-bit moments, twice
        assert float((q.detach().double() - p).abs().max()) <= 2e-5 * lr * 10 + 2.0 ** -22 * float(p.abs().max())
    if bits == 8:
        assert len(opt.moments()) == 4


@pytest.mark.parametrize("tensor_rate", [False, True])
def test_learning_rates_around_a_capture(tensor_rate):
    """A rate changed before a capture, between replays and behind them: each update takes the rate that was last copied
    to the device, a graph recorded with a rate on the device the one that is there."""
    params, twin = _params([300, 2049]), _params([300, 2049])
    a, b = optim.AdamW(params, max_norm=1.0, **HP), optim.AdamW(twin, max_norm=1.0, **HP)
    grads = _tensors([300, 2049], seed=2)
    rate = torch.tensor(5e-3, device=DEV, dtype=torch.float64) if tensor_rate else 5e-3
    taken = []

    def step():
        a.step(grads=grads)
        taken.append(float(a.param_groups[0]["lr"]))
    step()
    a.param_groups[0]["lr"] = rate
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        a.step(grads=grads)
    step()  # takes the rate that was set before the capture
    for lr in (7e-3, 2e-3):
        if tensor_rate:
            rate.fill_(lr)
        else:
            a.param_groups[0]["lr"] = lr
            a.sync_lr()
        graph.replay()
        graph.replay()
        taken += [lr, lr]
    step()
    for lr in taken:
        b.param_groups[0]["lr"] = lr
        b.step(grads=grads)
    for p, q in zip(params, twin):
        assert torch.equal(p, q)
    assert float(a.param_groups[0]["scalars"][1]) == len(taken) == 7.0


def test_a_first_step_is_not_captured():
    p, q = _params([300, 2049])
    opt = optim.AdamW([p, q], **HP)
    g = _tensors([300, 2049], seed=2)
    opt.step(grads=[g[0], None])
    with pytest.raises(RuntimeError, match="first step"):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            opt.step(grads=g)
    before = q.detach().clone()
    opt.step(grads=g)
    assert not torch.equal(q, before) and bool(q.isfinite().all())


def test_an_eager_step_with_other_gradients_between_replays():
    """The plan of an eager step leaves a captured graph its workspace: replays give the gradients' norm and write to
    nothing that was allocated since."""
    params = _params([300, 2049])
    opt = optim.AdamW(params, max_norm=1.0, **HP)
    grads = _tensors([300, 2049], seed=2)
    norm = math.sqrt(sum(float(g.double().square().sum()) for g in grads))
    opt.step(grads=grads)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        opt.step(grads=grads)
    opt.step(grads=[grads[0], None])
    opt.step(grads=[grads[0].bfloat16(), grads[1]])
    others = [torch.full((n,), 7.0, device=DEV) for n in (128, 512, 592, 600, 1184, 4096) for _ in range(20)]
    for _ in range(2):
        graph.replay()
        assert abs(float(opt.param_groups[0]["scalars"][2]) - norm) <= 1e-5 * norm
    assert all(bool((t == 7.0).all()) for t in others)
    opt.step(grads=grads)
    assert abs(float(opt.grad_norm) - norm) <= 1e-5 * norm
    assert all(bool(p.isfinite().all()) for p in params)


def test_tensors_that_come_late_or_rest_follow_torch_adamw():
    """Each tensor's bias correction goes by its own steps: against torch.optim.AdamW, whose fp32 arithmetic is as far off
    as this one's, with the default betas, over steps that leave out changing tensors."""
    sizes = [300, 2049, 7, 513, 1000]
    a, b = _params(sizes), _params(sizes)
    hp = dict(lr=1e-2, betas=(0.9, 0.999), eps=1e-8, weight_decay=0.1)
    oa, ob = optim.AdamW(a, **hp), torch.optim.AdamW(b, **hp)
    live = [(0, 1), (0, 1), (0, 1, 2), (0, 2), (3,), (0, 1, 2, 3, 4), (1, 4), (0, 1, 2, 3, 4), (0, 1, 2, 3, 4), (2, 3)]
    for k, now in enumerate(live):
        grads = _tensors(sizes, seed=60 + k)
        for i in range(5):
            a[i].grad = b[i].grad = grads[i] if i in now else None
        oa.step()
        ob.step()
        for p, q in zip(a, b):
            # as in the test beside torch's on a model; an update is at most lr / (1 - b1), and a first one 1 / (1 - b1^t)
            assert float((p - q).detach().abs().max()) <= 2.0 ** -18 * hp["lr"] * 10 * (k + 1) + 1e-7
    steps = [float(oa.state[p].get("scalars", oa.param_groups[0]["scalars"])[1]) for p in a]
    assert steps == [sum(i in now for now in live) for i in range(5)]


@pytest.mark.parametrize("bits", [32, 8])
def test_late_tensors_survive_a_round_trip(bits, tmp_path):
    sizes = [300, 2049, 7]
    params = _params(sizes)
    opt = optim.AdamW(params, state_bits=bits, max_norm=1.0, **HP)
    for k, now in enumerate([(0,), (0, 1), (1, 2), (0, 1, 2)]):
        grads = _tensors(sizes, seed=k)
        opt.step(grads=[g if i in now else None for i, g in enumerate(grads)])
    torch.save(opt.state_dict(), tmp_path / "opt.pt")
    twin = [torch.nn.Parameter(p.detach().clone()) for p in params]
    other = optim.AdamW(twin, state_bits=bits, max_norm=1.0, **HP)
    other.load_state_dict(torch.load(tmp_path / "opt.pt", map_location="cpu"))
    for k in range(2):
        grads = _tensors(sizes, seed=10 + k)
        opt.step(grads=grads)
        other.step(grads=[g.clone() for g in grads])
    assert all(torch.equal(p, q) for p, q in zip(params, twin))
    assert float(opt.grad_norm) == float(other.grad_norm)


def test_an_update_is_as_near_to_64_bits_as_the_plain_form():
    """The kernel rounds no more often than the plain fp32 form, operation by operation (products fused into sums round
    less): over many elements its error is that form's, to a tenth. The betas are exact in fp32, parameters 0, so
    that the update itself is what is rounded last."""
    n, b1, b2, lr, eps, step = 1 << 18, 0.875, 0.96875, 1e-2, 1e-8, 40
    gen = torch.Generator(device=DEV).manual_seed(3)
    g, m, v = (torch.randn(n, generator=gen, device=DEV) for _ in range(3))
    v = v.square() + 1e-3
    p = torch.nn.Parameter(torch.zeros(n, device=DEV))
    opt = optim.AdamW([p], lr=lr, betas=(b1, b2), eps=eps, weight_decay=0.0)
    opt.state[p].update(exp_avg=m.clone(), exp_avg_sq=v.clone())
    opt.set_step(step - 1)
    opt.step(grads=[g])
    a, s = lr / (1 - b1 ** step), math.sqrt(1 - b2 ** step)
    ours = opt.state[p]["exp_avg"], opt.state[p]["exp_avg_sq"], p.detach()
    mp = m + (1 - b1) * (g - m)
    vp = b2 * v + (1 - b2) * g * g
    plain = mp, vp, -a * (mp / (vp.sqrt() / s + eps))
    m64, g64, v64 = m.double(), g.double(), v.double()
    me = b1 * m64 + (1 - b1) * g64
    ve = b2 * v64 + (1 - b2) * g64 * g64
    exact = me, ve, -a * (me / (ve.sqrt() / s + eps))
    for got, other, want in zip(ours, plain, exact):
        off, its = ((t.double() - want).square().mean().sqrt() for t in (got, other))
        assert float(off) <= 1.1 * float(its) + 1e-12 * float(want.abs().max())


@pytest.mark.parametrize("bits", [32, 8])
def test_gradients_whose_squares_are_denormal(bits):
    """eps = 0 and gradients of 3e-20: the second moment is a denormal of 15 bits, so its root is within 2^-16 and the
    first update within that of lr, instead of infinite."""
    n = 512
    g = torch.full((n,), 3e-20, device=DEV)
    g[::2] = -3e-20
    p = torch.nn.Parameter(torch.zeros(n, device=DEV))
    opt = optim.AdamW([p], lr=1e-2, betas=(0.9, 0.95), eps=0.0, weight_decay=0.0, state_bits=bits)
    for k in range(3):  # the same gradient: bias-corrected moments stay g and g^2, 8-bit codes are exact at a block's largest
        opt.step(grads=[g])
        # a code's own rounding (2^-22) and what three roundings of a denormal leave
        assert float((p.detach() + (k + 1) * 1e-2 * g.sign()).abs().max()) <= (k + 1) * 1e-2 * 2.0 ** -13


@pytest.mark.parametrize("betas", [(0.9, 0.999), (0.9, 0.95), (0.8, 0.9999), (0.5, 0.3), (0.0, 0.0)])
def test_moments_take_the_betas_in_64_bits(betas):
    """One step from given moments. exp_avg_sq: its weights and their products are rounded 2^-24 four times, its sums
    twice, all terms positive; exp_avg: a difference, its product and a sum, of the size of both terms."""
    n, (b1, b2) = 1 << 16, betas
    gen = torch.Generator(device=DEV).manual_seed(4)
    g, m, v = (torch.randn(n, generator=gen, device=DEV) for _ in range(3))
    v = v.square() * 3
    v[::7] = 0.0
    p = torch.nn.Parameter(torch.zeros(n, device=DEV))
    opt = optim.AdamW([p], betas=betas, weight_decay=0.0)
    opt.state[p].update(exp_avg=m.clone(), exp_avg_sq=v.clone())
    opt.set_step(3)
    opt.step(grads=[g])
    m64, g64, v64 = m.double(), g.double(), v.double()
    me = b1 * m64 + (1 - b1) * g64
    ve = b2 * v64 + (1 - b2) * g64 * g64
    assert float(((opt.state[p]["exp_avg_sq"].double() - ve).abs() - 6 * 2.0 ** -24 * ve).max()) <= 0
    lim = 4 * 2.0 ** -24 * (m64.abs() + g64.abs())
    assert float(((opt.state[p]["exp_avg"].double() - me).abs() - lim).max()) <= 0


def test_default_betas_against_64_bits():
    """The class's own betas from the first step on: each step adds its six roundings to exp_avg_sq (which are at most
    those of the sum so far) and as many to the update, whose bias corrections are formed in 64 bits."""
    params = _params([300, 2049])
    opt, ref = optim.AdamW(params, lr=1e-2), Ref(params, lr=1e-2)
    for k in range(1, 31):
        grads = _tensors([300, 2049], seed=70 + k)
        opt.step(grads=grads)
        ref.step(grads)
        for p, m, v, q in zip(ref.p, ref.m, ref.v, params):
            st = opt.state[q]
            assert float(((st["exp_avg_sq"].double() - v).abs() - 6 * k * 2.0 ** -24 * v).max()) <= 0
            assert float((st["exp_avg"].double() - m).abs().max()) <= 4 * k * 2.0 ** -24 * 10
            # the update is at most lr |m| / sqrt(v), both corrected: here below 10 lr; p itself is rounded each step
            assert float((q.detach().double() - p).abs().max()) <= k * (2.0 ** -20 * 1e-2 * 10 + 2.0 ** -24)


def test_scales_of_8_bit_blocks_mark_nan_and_infinity():
    """A block that saw either has scales, and so decoded moments, that are not finite; its neighbours' are."""
    q = _params([1300])[0]
    opt = optim.AdamW([q], state_bits=8, **HP)
    g = _tensors([1300], seed=1)[0]
    g[5], g[300], g[1290] = math.inf, math.nan, -math.inf
    for _ in range(2):  # and it stays so
        opt.step(grads=[g])
        (m, v), = opt.moments()
        st = opt.state[q]
        for name, values in (("exp_avg_scale", m), ("exp_avg_sq_scale", v)):
            assert st[name].isfinite().tolist() == [False, False, True, True, True, False]
            for block in range(6):
                finite = values[block * 256:(block + 1) * 256].isfinite()
                assert bool(finite.all() if block in (2, 3, 4) else ~finite.any())
        g = _tensors([1300], seed=2)[0]
    assert bool(q[512:1280].isfinite().all()) and not bool(q[[5, 300, 1290]].isfinite().any())
