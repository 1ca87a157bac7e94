"""Host side of optim.AdamW on CPU tensors: the library calls are recorded
instead of launched, so what is planned, allocated and refused is seen without
a GPU."""
import weakref

import pytest
import torch

from reversability_b200 import _lib, optim


class Recorder:
    def __init__(self):
        self.calls = []
        self.capturing = False

    def __call__(self, name, *args):
        self.calls.append((name, args))

    def named(self, name):
        return [args for n, args in self.calls if n == name]

    def stepped(self):
        """The parameter addresses that the recorded steps would update."""
        return [args[0][i * 7] for args in self.named("rk_adamw_multi_step") for i in range(args[1])]


@pytest.fixture
def recorded(monkeypatch):
    """A CPU tensor's device index is -1: so is the current device here."""
    r = Recorder()
    monkeypatch.setattr(optim.fn, "require_cuda", lambda *a, **k: None)
    monkeypatch.setattr(torch.cuda, "current_device", lambda: -1)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: r.capturing)
    monkeypatch.setattr(_lib, "stream_ptr", lambda device=None: 0)
    monkeypatch.setattr(_lib, "call", r)
    return r


def _params(n, size=10):
    return [torch.nn.Parameter(torch.zeros(size)) for _ in range(n)]


def _grads(params):
    return [torch.ones_like(p) for p in params]


@pytest.mark.parametrize("given", [False, True])
@pytest.mark.parametrize("max_norm", [None, 1.0])
def test_a_group_added_after_a_step_is_updated(recorded, max_norm, given):
    params = _params(3)
    opt = optim.AdamW(params[:2], max_norm=max_norm)

    def step(which):
        if not given:
            for p, g in zip(which, _grads(which)):
                p.grad = g
        recorded.calls.clear()
        opt.step(grads=_grads(which) if given else None)
    step(params[:2])
    opt.add_param_group(dict(params=params[2:], state_bits=8))
    step(params)
    assert sorted(recorded.stepped()) == sorted(p.data_ptr() for p in params)
    assert opt.state[params[2]]["exp_avg"].dtype is torch.int8
    if max_norm:
        assert sum(args[1] for args in recorded.named("rk_adamw_multi_sumsq")) == 3


def test_parameters_put_into_a_group_by_hand(recorded):
    params = _params(4)
    opt = optim.AdamW(params[:2])
    opt.step(grads=_grads(params[:2]))
    group = opt.param_groups[0]
    group["params"].append(params[2])
    recorded.calls.clear()
    opt.step(grads=_grads(params[:3]))
    assert recorded.stepped() == [p.data_ptr() for p in params[:3]]
    group["params"][1] = params[3]
    recorded.calls.clear()
    opt.step(grads=_grads(params[:3]))
    assert recorded.stepped() == [params[i].data_ptr() for i in (0, 3, 2)]
    del opt.param_groups[0]["params"][0]
    recorded.calls.clear()
    opt.step(grads=_grads(params[:2]))
    assert recorded.stepped() == [params[i].data_ptr() for i in (3, 2)]


def test_another_state_bits_is_noticed(recorded):
    params = _params(2)
    opt = optim.AdamW([dict(params=params[:1]), dict(params=params[1:])])
    opt.step(grads=_grads(params))
    for bits in (8, 16):  # the moments are there in 32 bits; 16 there is not
        opt.param_groups[1]["state_bits"] = bits
        with pytest.raises(ValueError, match="bit"):
            opt.step(grads=_grads(params))
    opt.param_groups[1]["state_bits"] = 8
    opt.state[params[1]].clear()
    recorded.calls.clear()
    opt.step(grads=_grads(params))
    assert [args[4] for args in recorded.named("rk_adamw_multi_step")] == [32, 8]


def test_groups_that_change_places_keep_their_learning_rates(recorded):
    params = _params(2)
    opt = optim.AdamW([dict(params=params[:1], lr=1.0), dict(params=params[1:], lr=2.0)])
    opt.step(grads=_grads(params))
    opt.param_groups.reverse()
    opt.param_groups[0]["lr"], opt.param_groups[1]["lr"] = 1.0, 2.0
    opt.step(grads=_grads(params)[::-1])
    assert [float(g["scalars"][0]) for g in opt.param_groups] == [1.0, 2.0]


def test_a_number_after_a_learning_rate_tensor(recorded):
    params = _params(1)
    opt = optim.AdamW(params, lr=1.0)
    for lr in (1.0, torch.tensor(2.0), 1.0):
        opt.param_groups[0]["lr"] = lr
        opt.step(grads=_grads(params))
        assert float(opt.param_groups[0]["scalars"][0]) == float(lr)


def _used(recorded, opt, params):
    """Whether the last step was given the moments that the optimizer's state holds."""
    given = {args[0][i * 7]: (args, i) for args in recorded.named("rk_adamw_multi_step") for i in range(args[1])}
    for p in params:
        args, i = given[p.data_ptr()]
        names = ("exp_avg", "exp_avg_sq", "exp_avg_scale", "exp_avg_sq_scale")[:4 if args[4] == 8 else 2]
        assert [args[0][i * 7 + 2 + k] for k in range(len(names))] == [opt.state[p][name].data_ptr() for name in names]


@pytest.mark.parametrize("bits", [32, 8])
def test_state_that_is_replaced_or_dropped(recorded, bits):
    params, held = _params(3), []

    def step():
        recorded.calls.clear()
        opt.step(grads=_grads(params))
        _used(recorded, opt, params)
    opt = optim.AdamW(params, state_bits=bits)
    step()
    for change in (lambda: opt.state.clear(), lambda: opt.state.pop(params[1]), lambda: opt.state[params[2]].clear(),
                   lambda: opt.state.update({params[0]: {k: v.clone() for k, v in opt.state[params[0]].items()}}),
                   lambda: opt.state[params[0]].update(exp_avg_sq=opt.state[params[0]]["exp_avg_sq"].clone())):
        if bits == 8:
            opt.moments()
        held.append([dict(s) for s in opt.state.values()])  # so that nothing new lies where something was
        change()
        if bits == 8 and all(opt.state.get(p) for p in params):
            recorded.calls.clear()
            opt.moments()
            (table, n, *_), = recorded.named("rk_adamw_multi_moments")
            assert [table[i * 7 + 3] for i in range(n)] == [opt.state[p]["exp_avg_sq"].data_ptr() for p in params]
        step()
    del opt.state[params[0]]["exp_avg"]  # not a whole state
    opt.state[params[0]]["exp_avg"] = torch.zeros(9)
    with pytest.raises(ValueError, match="exp_avg"):
        step()


def test_a_capture_does_not_write_the_learning_rate(recorded):
    params = _params(1)
    opt = optim.AdamW(params, lr=1.0)
    opt.step(grads=_grads(params))
    scalars = opt.param_groups[0]["scalars"]
    opt.param_groups[0]["lr"] = 2.0
    recorded.capturing = True
    opt.step(grads=_grads(params))
    assert float(scalars[0]) == 1.0
    with pytest.raises(RuntimeError, match="captured"):
        opt.sync_lr()
    recorded.capturing = False
    opt.step(grads=_grads(params))  # nor does a capture note it as written
    assert float(scalars[0]) == 2.0
    rate = torch.tensor(3.0)  # a tensor on the parameters' device: replays read it, so it is kept
    opt.param_groups[0]["lr"] = rate
    recorded.capturing = True
    opt.step(grads=_grads(params))
    assert float(scalars[0]) == 3.0
    gone = weakref.ref(rate)
    opt.param_groups[0]["lr"] = 2.0
    del rate
    assert gone() is not None


def test_a_first_step_is_not_captured(recorded):
    params = _params(3)
    opt = optim.AdamW([dict(params=params[:2]), dict(params=params[2:])])
    g = _grads(params)
    recorded.capturing = True
    with pytest.raises(RuntimeError, match="first step"):
        opt.step(grads=[g[0], None, None])
    recorded.capturing = False
    opt.step(grads=[g[0], None, None])
    recorded.capturing = True
    opt.step(grads=[g[0], None, None])
    for grads in ([g[0], g[1], None], [g[0], None, g[2]]):
        with pytest.raises(RuntimeError, match="first step"):
            opt.step(grads=grads)
    opt.step(grads=[g[0], None, None])
    for name in ("exp_avg", "exp_avg_sq"):
        opt.state[params[2]][name] = torch.zeros(10)
    with pytest.raises(RuntimeError, match="first step"):  # its group has no count yet
        opt.step(grads=g[:1] + [None] + g[2:])
    recorded.capturing = False
    opt.step(grads=g)
    recorded.capturing = True
    opt.step(grads=g)


def test_the_workspace_of_the_norm_outlives_plans(recorded, monkeypatch):
    """What a captured graph has been given stays where it is when the plan is made anew, also a smaller or a larger one."""
    params, made, empty = _params(70), [], torch.empty

    def allocate(*args, **kwargs):
        t = empty(*args, **kwargs)
        made.append((weakref.ref(t), t.data_ptr(), t.data_ptr() + 4 * t.numel()))
        return t
    monkeypatch.setattr(torch, "empty", allocate)

    def inside(a, b):
        return any(r() is not None and first <= a and b <= end for r, first, end in made)
    opt = optim.AdamW(params, max_norm=1.0)
    g = _grads(params)
    opt.step(grads=g)
    recorded.capturing = True
    recorded.calls.clear()
    opt.step(grads=g)
    recorded.capturing = False
    at = [args[3] for args in recorded.named("rk_adamw_multi_sumsq")]
    prepare, = recorded.named("rk_adamw_multi_prepare")
    assert at[0] == prepare[0] and inside(at[0], at[0] + 4 * prepare[1])

    def some(n, dtype=torch.float32):
        return [x.to(dtype) if i < n else None for i, x in enumerate(g)]
    for grads in (some(3), some(70), some(69), some(70, torch.bfloat16), [x.bfloat16() if i % 2 else x for i, x in enumerate(g)]):
        recorded.calls.clear()
        opt.step(grads=grads)
        calls = recorded.named("rk_adamw_multi_sumsq")
        (begin, parts), = {args[:2] for args in recorded.named("rk_adamw_multi_prepare")}
        assert parts == sum(_lib.lib().rk_adamw_multi_parts(args[1]) for args in calls)  # no part that nothing has written
        ends = [args[3] + 4 * _lib.lib().rk_adamw_multi_parts(args[1]) for args in calls]
        assert [args[3] for args in calls] == [begin] + ends[:-1]
        assert inside(begin, ends[-1])
    more = _params(70)
    opt.add_param_group(dict(params=more))
    opt.step(grads=g + _grads(more))
    opt.load_state_dict(opt.state_dict())
    opt.step(grads=g + _grads(more))
    assert inside(at[0], at[0] + 4 * prepare[1])


def test_what_a_capture_has_seen_outlives_the_state(recorded):
    params = _params(2)
    opt = optim.AdamW([dict(params=params[:1]), dict(params=params[1:], state_bits=8)])
    opt.step(grads=_grads(params))
    recorded.capturing = True
    opt.step(grads=_grads(params))
    opt.moments()
    recorded.capturing = False
    seen = [weakref.ref(t) for s in opt.state.values() for t in s.values()]
    seen += [weakref.ref(group["scalars"]) for group in opt.param_groups]
    opt.load_state_dict(opt.state_dict())
    opt.step(grads=_grads(params))
    assert all(r() is not None for r in seen)


def _counts(recorded, opt):
    """Lets the recorded prepares count, as they do on the device; the counts of all parameters with moments."""
    blocks = {t.data_ptr(): t for t in [g["scalars"] for g in opt.param_groups if g["scalars"] is not None]
              + [s["scalars"] for s in opt.state.values() if "scalars" in s]}
    for args in recorded.named("rk_adamw_multi_prepare"):
        blocks[args[6]][1] += 1
    recorded.calls.clear()
    return [float(opt.state[p].get("scalars", g["scalars"])[1]) for g in opt.param_groups for p in g["params"]
            if "exp_avg" in opt.state.get(p, ())]


def test_each_tensor_counts_its_own_steps(recorded):
    params = _params(5)
    opt = optim.AdamW([dict(params=params[:4]), dict(params=params[4:])])
    want, g = [0.0] * 5, _grads(params)
    for live in ((0, 1, 4), (0, 1), (0, 1, 2), (2, 3), (0, 1, 2, 3, 4), (0, 3), (0, 1, 2, 3, 4), (4,), (0, 1, 2, 3, 4)):
        opt.step(grads=[x if i in live else None for i, x in enumerate(g)])
        want = [w + (i in live) for i, w in enumerate(want)]
        launches = len(recorded.named("rk_adamw_multi_step"))
        assert launches == len(recorded.named("rk_adamw_multi_prepare")) >= len({(i == 4, want[i]) for i in live})
        assert _counts(recorded, opt) == [w for w in want if w]
    again = optim.AdamW([dict(params=params[:4]), dict(params=params[4:])])
    again.load_state_dict(opt.state_dict())
    opt.step(grads=g)
    launches = len(recorded.named("rk_adamw_multi_step"))
    recorded.calls.clear()
    again.step(grads=g)
    assert len(recorded.named("rk_adamw_multi_step")) == launches  # who counted together still does
    assert _counts(recorded, again) == [w + 1 for w in want]
    again.set_step(7)
    again.step(grads=g)
    assert _counts(recorded, again) == [8.0] * 5
    again.param_groups[0]["lr"] = 0.5
    again.sync_lr()
    assert all(float(again.state[p].get("scalars", again.param_groups[0]["scalars"])[0]) == 0.5 for p in params[:4])


def test_tensors_that_step_together_stay_in_one_launch(recorded):
    params = _params(6)
    opt = optim.AdamW(params)
    g = _grads(params)
    opt.step(grads=g[:4] + [None, None])
    for _ in range(3):  # two frozen from here on
        recorded.calls.clear()
        opt.step(grads=[None, None] + g[2:4] + [None, None])
        assert len(recorded.named("rk_adamw_multi_step")) == 1
    recorded.calls.clear()
    opt.step(grads=g)  # three histories: the frozen, those that went on, those that are new
    assert len(recorded.named("rk_adamw_multi_step")) == 3


def test_dropped_moments_start_from_zero(recorded):
    params = _params(2)
    opt = optim.AdamW(params)
    for _ in range(3):
        opt.step(grads=_grads(params))
    assert _counts(recorded, opt) == [3.0, 3.0]
    opt.state.clear()
    opt.step(grads=_grads(params))
    assert _counts(recorded, opt) == [1.0, 1.0]
    opt.state.pop(params[1])
    opt.step(grads=_grads(params))
    assert _counts(recorded, opt) == [2.0, 1.0]
    opt.load_state_dict(opt.state_dict())
    opt.state.clear()
    opt.step(grads=_grads(params))
    assert _counts(recorded, opt) == [1.0, 1.0]
    by_hand = optim.AdamW(params)
    for p in params:
        by_hand.state[p].update(exp_avg=torch.zeros(10), exp_avg_sq=torch.zeros(10))
    by_hand.step(grads=[None, torch.ones(10)])
    assert _counts(recorded, by_hand) == [0.0, 1.0]
    fresh = optim.AdamW(params)
    fresh.set_step(40)  # before the first step: moments from elsewhere, or none yet
    fresh.step(grads=_grads(params))
    assert _counts(recorded, fresh) == [41.0, 41.0]


def test_a_capture_does_not_part_counts(recorded):
    params = _params(2)
    opt = optim.AdamW(params)
    opt.step(grads=_grads(params))
    recorded.capturing = True
    with pytest.raises(RuntimeError, match="captured"):
        opt.step(grads=[torch.ones(10), None])
    assert "scalars" not in opt.state[params[1]]


def test_the_state_of_another_optimizer_is_refused(recorded):
    params = _params(2)
    for p in params:
        p.grad = torch.ones_like(p)
    other = torch.optim.AdamW(params)
    other.step()
    opt = optim.AdamW(params, lr=0.5)
    opt.step()
    before = [dict(s) for s in opt.state.values()]
    with pytest.raises(ValueError, match="scalars, state_bits"):
        opt.load_state_dict(other.state_dict())
    assert opt.param_groups[0]["lr"] == 0.5 and all(a[k] is s[k] for a, s in zip(before, opt.state.values()) for k in a)
    opt.step()
    # the way that the refusal names
    new = optim.AdamW(params)
    for p in params:
        new.state[p].update({k: other.state[p][k].clone() for k in ("exp_avg", "exp_avg_sq")})
    new.set_step(int(other.state[params[0]]["step"]))
    recorded.calls.clear()
    new.step()
    _used(recorded, new, params)
    assert _counts(recorded, new) == [2.0, 2.0]


def test_a_graph_kept_over_a_step_notices(recorded):
    p, q, r = params = _params(3)
    opt = optim.AdamW(params)
    for _ in range(2):  # with a new plan and with the one that is there
        a, b = (p * q).sum(), (r * r).sum()
        opt.step(grads=[torch.ones(10), None, None])
        b.backward()  # what was not updated may still be used
        with pytest.raises(RuntimeError, match="inplace"):
            a.backward()


def test_grad_norm_follows_scalars_that_move(recorded):
    params = _params(2)
    opt = optim.AdamW(params, max_norm=1.0)
    opt.step(grads=[torch.ones(10), None])
    for _ in range(2):
        opt.step(grads=_grads(params))
        first = opt.state[params[0]].get("scalars", opt.param_groups[0]["scalars"])
        first[2] = 3.0
        assert float(opt.grad_norm) == 3.0
        first.data = first.data.clone()
        opt.step(grads=_grads(params))
        first[2] = 4.0
        assert float(opt.grad_norm) == 4.0
        opt.step(grads=[None, torch.ones(10)])
