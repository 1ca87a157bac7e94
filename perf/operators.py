"""Workloads of the post-training operators: token log-probabilities, the clipped
policy loss, the paired preference loss (alignment.py) and AdamW over many
tensors (optim.py).

`listed()` names the fixed cases, `draw(rng)` makes more of the same ranges,
`prepare` makes a case's inputs on the GPU, `run` does one pass in plain torch
operations (or, with `own` set, through the package), `exact` gives the same
outputs from the definitions in 64 bits and `work` the bytes and operations no
implementation can do without.
"""
import math

import torch

own = False

DEV = "cuda"
DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
SIZE = {"f32": 4, "bf16": 2, "f16": 2}
IGNORE = -100
CLIP_LOW, CLIP_HIGH = 0.2, 0.28
LOW = {"f32": torch.finfo(torch.float32).min, "bf16": torch.finfo(torch.bfloat16).min, "f16": torch.finfo(torch.float16).min}
ADAM = dict(lr=6e-4, betas=(0.9, 0.95), eps=1e-8, weight_decay=0.1)
STEPS_BEFORE = 40  # the optimizer's step count before the measured step
BLOCK = 256  # elements that share a scale in 8-bit states


def listed():
    return [
        # One sampled token is scored: the call after each generated token. Latency only.
        dict(name="logprob_one_token", op="logprob", rows=1, vocab=50257, dtype="bf16", pad=False, grad=False,
             entropy=True, temperature=1.0, masked=0.0, dead=0),
        # A reference model scores a whole microbatch of the 20.3M decoder (29 x 512 tokens): forward only.
        dict(name="logprob_score_batch", op="logprob", rows=14848, vocab=50257, dtype="bf16", pad=False, grad=False,
             entropy=False, temperature=1.0, masked=0.25, dead=0),
        # A user's own loss on log-probabilities and entropies, fp32 logits, odd sizes: forward and backward.
        dict(name="logprob_train_f32", op="logprob", rows=2047, vocab=32003, dtype="f32", pad=False, grad=True,
             entropy=True, temperature=0.7, masked=0.1, dead=3),
        # One short response is trained on (a 64-token rollout).
        dict(name="policy_short", op="policy", rows=64, vocab=50257, dtype="bf16", pad=False, entropy_coef=0.0,
             kl_coef=0.05, temperature=1.0, masked=0.0, dead=0, weights=False, group=1, api="grad"),
        # A policy step on the 20.3M decoder's microbatch, rows in the padded buffer its head writes.
        dict(name="policy_batch", op="policy", rows=14848, vocab=50257, dtype="bf16", pad=True, entropy_coef=0.0,
             kl_coef=0.05, temperature=1.0, masked=0.1, dead=0, weights=False, group=512, api="grad"),
        # A larger vocabulary in half precision with entropy bonus and token weights, through autograd.
        dict(name="policy_wide_f16", op="policy", rows=1500, vocab=131072, dtype="f16", pad=False, entropy_coef=0.01,
             kl_coef=0.02, temperature=0.9, masked=0.1, dead=72, weights=True, group=1, api="autograd"),
        # Byte- or character-level vocabulary, many short rows, fp32.
        dict(name="policy_narrow_f32", op="policy", rows=12001, vocab=1000, dtype="f32", pad=False, entropy_coef=0.01,
             kl_coef=0.05, temperature=1.0, masked=0.2, dead=0, weights=False, group=1, api="grad"),
        # One pair of short answers.
        dict(name="preference_one_pair", op="preference", pairs=1, length=64, vocab=50257, dtype="bf16", pad=False,
             kind="sigmoid", beta=0.1, smoothing=0.0, average=False, api="grad"),
        # A microbatch of pairs at the decoder's context of 512.
        dict(name="preference_batch", op="preference", pairs=14, length=512, vocab=50257, dtype="bf16", pad=False,
             kind="sigmoid", beta=0.1, smoothing=0.1, average=False, api="grad"),
        # A two-layer test model's tensors: launch and host time only.
        dict(name="adamw_tiny", op="adamw", layers=2, d=256, ff=1024, vocab=101, context=64, bits=32, pdtype="f32",
             gdtype="f32", clip=True),
        # The 20.3M decoder's 45 tensors, clipped to norm 1, 32-bit states.
        dict(name="adamw_decoder", op="adamw", layers=7, d=256, ff=1024, vocab=50257, context=512, bits=32,
             pdtype="f32", gdtype="f32", clip=True),
        # The scaled decoder (24 layers of 1024), 8-bit states.
        dict(name="adamw_scaled_8bit", op="adamw", layers=24, d=1024, ff=4096, vocab=50257, context=2048, bits=8,
             pdtype="f32", gdtype="f32", clip=False),
    ]


def _log_int(rng, low, high):
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    op = rng.choice(["logprob", "policy", "policy", "preference", "adamw"])
    if op == "adamw":
        bits = rng.choice([8, 32])
        return dict(op=op, layers=rng.randint(1, 24), d=_log_int(rng, 64, 1024 if bits == 8 else 768), ff=_log_int(rng, 100, 4096),
                    vocab=_log_int(rng, 101, 50257), context=_log_int(rng, 16, 2048), bits=bits,
                    pdtype=rng.choice(["f32", "f32", "bf16"]), gdtype=rng.choice(["f32", "bf16"]),
                    clip=rng.random() < 0.5)
    dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
    vocab = _log_int(rng, 100, 131072)
    most = int(1.4e9 / SIZE[dtype]) // vocab  # rows that keep the case below the largest listed one
    base = dict(op=op, vocab=vocab, dtype=dtype, pad=rng.random() < 0.4)
    if op == "preference":
        length = _log_int(rng, 4, 1024)
        return dict(base, pairs=_log_int(rng, 1, max(1, min(64, most // (2 * length)))), length=length,
                    kind=rng.choice(["sigmoid", "hinge", "squared"]), beta=rng.choice([0.05, 0.1, 0.5]),
                    smoothing=rng.choice([0.0, 0.1]), average=rng.random() < 0.3,
                    api=rng.choice(["grad", "autograd"]))
    base |= dict(rows=_log_int(rng, 1, max(1, min(16384, most))), temperature=rng.choice([1.0, 1.0, 0.7, 1.3]),
                 masked=rng.choice([0.0, 0.1, 0.5]), dead=rng.choice([0, 0, 1, vocab // 50]))
    if op == "logprob":
        return dict(base, grad=rng.random() < 0.5, entropy=rng.random() < 0.5)
    return dict(base, entropy_coef=rng.choice([0.0, 0.0, 0.01]), kl_coef=rng.choice([0.0, 0.05]),
                weights=rng.random() < 0.3, group=1, api=rng.choice(["grad", "autograd"]))


# ---------------------------------------------------------------- inputs
def _logits(gen, rows, vocab, dtype, pad, actions, dead):
    """Logits of a trained model: spread 2, the target token well above the rest, the last `dead` columns
    (vocabulary rows that no token uses) at the type's lowest value."""
    width = (vocab + 63) // 64 * 64 if pad else vocab
    x = torch.randn(rows, width, generator=gen, device=DEV, dtype=DTYPES[dtype]).mul_(2.0)[:, :vocab]
    if dead:
        x[:, vocab - dead:] = LOW[dtype]
    r = torch.arange(rows, device=DEV)
    bump = torch.rand(rows, generator=gen, device=DEV) * 4 + 2
    x[r, actions] = (x[r, actions].float() + bump).to(x.dtype)
    return x


def _row_logprobs(x, actions, temperature):
    """fp32 log-probabilities, a few rows at a time."""
    step = max(1, (1 << 26) // x.shape[1])
    out = []
    for s in range(0, x.shape[0], step):
        z = x[s:s + step].float() / temperature
        out.append(z.gather(1, actions[s:s + step, None])[:, 0] - torch.logsumexp(z, 1))
    return torch.cat(out)


def _off_the_kink(d):
    """Log ratios with none within 0.001 of the clip's two edges, where the loss has no single derivative."""
    for edge in (math.log(1 - CLIP_LOW), math.log(1 + CLIP_HIGH)):
        d = torch.where((d - edge).abs() < 1e-3, torch.full_like(d, edge + 2e-3), d)
    return d


def _shapes(case):
    d, ff = case["d"], case["ff"]
    block = [(d,), (3 * d, d), (d, d), (d,), (2 * ff, d), (d, ff)]
    return [(case["vocab"], d), (case["context"], d)] + block * case["layers"] + [(d,)]


def _prepare_adamw(case, gen):
    """The tensors of a decoder in one arena, as an allocator lays them out: each starts at a multiple of 256
    elements, and what lies between them is zero."""
    shapes = _shapes(case)
    sizes = [math.prod(s) for s in shapes]
    starts, at = [], 0
    for n in sizes:
        starts.append(at)
        at += -(-n // BLOCK) * BLOCK
    inside = torch.ones(at, dtype=torch.bool, device=DEV)
    for n, s in zip(sizes, starts):
        inside[s + n:s + -(-n // BLOCK) * BLOCK] = False

    def arena(dtype):
        return torch.zeros(at, dtype=dtype, device=DEV)

    def normal():
        return torch.randn(at, generator=gen, device=DEV).mul_(inside)

    p, g = arena(DTYPES[case["pdtype"]]), arena(DTYPES[case["gdtype"]])
    p.copy_(normal().mul_(0.02))
    # the gradients' size differs from block to block by a few powers of two
    level = torch.exp2(torch.randint(-3, 4, (at // BLOCK, 1), generator=gen, device=DEV).float()) * 1e-3
    g.copy_((normal().view(-1, BLOCK) * level).view(-1))
    m = (normal().view(-1, BLOCK) * level * 0.3).view(-1)
    v = ((normal().view(-1, BLOCK) * level * 0.3).square() + level.square() * 0.7).view(-1).mul_(inside)
    views = lambda t: [t[s:s + n].view(shape) for shape, n, s in zip(shapes, sizes, starts)]  # noqa: E731
    state = dict(p=p, g=g, starts=starts, sizes=sizes, inside=inside, step=torch.full((), STEPS_BEFORE, device=DEV),
                 params=[torch.nn.Parameter(t) for t in views(p)])
    for q, t in zip(state["params"], views(g)):
        if q.dtype == t.dtype:
            q.grad = t
    state["grads"] = views(g)
    if case["bits"] == 32:
        state |= dict(m=m, v=v, ms=views(m), vs=views(v))
    else:
        mb, rb = m.view(-1, BLOCK), v.view(-1, BLOCK).sqrt()
        msc, vsc = mb.abs().amax(1), rb.amax(1)
        mc = torch.round(127 * (mb.abs() / msc[:, None]).sqrt()).mul_(mb.sign()).to(torch.int8).view(-1)
        vc = torch.round(255 * (rb / vsc[:, None]).sqrt()).clamp_(min=1).mul_(inside.view(-1, BLOCK)).to(torch.uint8).view(-1)
        blocks = [(s // BLOCK, s // BLOCK + -(-n // BLOCK)) for n, s in zip(sizes, starts)]
        state |= dict(m=mc, v=vc, msc=msc, vsc=vsc, ms=views(mc), vs=views(vc),
                      mscs=[msc[a:b] for a, b in blocks], vscs=[vsc[a:b] for a, b in blocks])
    return state


def prepare(case, seed):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    if case["op"] == "adamw":
        return dict(_prepare_adamw(case, gen), case=case)
    vocab = case["vocab"]
    live = vocab - case.get("dead", 0)
    if case["op"] == "preference":
        n, t = 2 * case["pairs"], case["length"]
        labels = torch.randint(0, live, (n, t), generator=gen, device=DEV)
        x = _logits(gen, n * t, vocab, case["dtype"], case["pad"], labels.view(-1), 0)
        ref = (_row_logprobs(x, labels.view(-1), 1.0).view(n, t)
               + 0.3 * torch.randn(n, t, generator=gen, device=DEV))
        # a shared prompt in front, answers of different lengths, padding behind them
        prompt = (torch.rand(n // 2, generator=gen, device=DEV) * 0.4 * t).long().repeat(2)
        end = prompt + 1 + (torch.rand(n, generator=gen, device=DEV) * (t - prompt)).long()
        at = torch.arange(t, device=DEV)
        labels[(at < prompt[:, None]) | (at >= end[:, None])] = IGNORE
        x = x.unflatten(0, (n, t)).requires_grad_(case["api"] == "autograd")
        return dict(case=case, logits=x, labels=labels, ref=ref)
    rows = case["rows"]
    actions = torch.randint(0, live, (rows,), generator=gen, device=DEV)
    x = _logits(gen, rows, vocab, case["dtype"], case["pad"], actions, case["dead"])
    state = dict(case=case)
    if case["op"] == "policy":
        lp = _row_logprobs(x, actions, case["temperature"])
        state["old"] = lp - _off_the_kink(0.2 * torch.randn(rows, generator=gen, device=DEV))
        # a drift of 0.2 and more: nearer to zero the KL term is a difference of equal numbers
        drift = 0.4 * torch.randn(rows, generator=gen, device=DEV)
        state["ref"] = lp + drift + torch.where(drift < 0, -0.2, 0.2)
        group = case["group"]
        adv = torch.randn(rows // group, generator=gen, device=DEV)
        state["advantages"] = adv
        state["weights"] = torch.rand(rows, generator=gen, device=DEV) + 0.5 if case["weights"] else None
    else:
        state["d_logprob"] = torch.randn(rows, generator=gen, device=DEV)
        state["d_entropy"] = torch.randn(rows, generator=gen, device=DEV) * 0.1
    hide = torch.rand(rows, generator=gen, device=DEV) < case["masked"]
    hide[0] = False
    state["actions"] = torch.where(hide, torch.full_like(actions, IGNORE), actions)
    if case["op"] == "policy" and case["group"] > 1:  # [sequences, tokens], one advantage a sequence
        shape = (rows // case["group"], case["group"])
        x = x.unflatten(0, shape)
        for k in ("actions", "old", "ref"):
            state[k] = state[k].view(shape)
    state["logits"] = x.requires_grad_(case.get("grad", False) or case.get("api") == "autograd")
    return state


def _grad_scale(case):
    """fp16 gradients are taken of the loss times a power of two, as a loss scaler does."""
    return 4096.0 if case["dtype"] == "f16" else 1.0


# ---------------------------------------------------------------- plain forms
def _plain_rows(x, actions, temperature, want_entropy):
    """(valid, target, p, log p of all columns, log-probability, entropy), in 32 bits."""
    z = x.detach().float() / temperature
    z = z - z.amax(-1, keepdim=True)
    e = torch.exp(z)
    s = e.sum(-1, keepdim=True)
    logp = z - torch.log(s)
    p = e / s
    valid = actions != IGNORE
    target = torch.where(valid, actions, torch.zeros_like(actions))
    lp = torch.where(valid, logp.gather(-1, target[..., None])[..., 0], torch.zeros_like(logp[..., 0]))
    h = None
    if want_entropy:
        h = -torch.where(p > 0, p * logp, torch.zeros_like(p)).sum(-1)
        h = torch.where(valid, h, torch.zeros_like(h))
    return valid, target, p, logp, lp, h


def _plain_dlogits(x, target, p, logp, h, d_lp, d_h, temperature):
    """d_lp (1[j = target] - p_j) - d_h p_j (log p_j + h), over the temperature, rounded to the logits' type."""
    d = -p * d_lp[..., None]
    d.scatter_add_(-1, target[..., None], d_lp[..., None])
    if d_h is not None:
        d = d - torch.where(p > 0, p * (logp + h[..., None]), torch.zeros_like(p)) * d_h[..., None]
    return (d / temperature).to(x.dtype)


def _plain_logprob(s):
    c = s["case"]
    valid, target, p, logp, lp, h = _plain_rows(s["logits"], s["actions"], c["temperature"], c["entropy"])
    out = dict(logprob=lp, entropy=h)
    if c["grad"]:
        zero = torch.zeros_like(lp)
        d_h = torch.where(valid, s["d_entropy"], zero) if c["entropy"] else None
        out["dlogits"] = _plain_dlogits(s["logits"], target, p, logp, h, torch.where(valid, s["d_logprob"], zero), d_h,
                                        c["temperature"])
    return out


def _plain_policy(s):
    c = s["case"]
    bonus = c["entropy_coef"] != 0
    valid, target, p, logp, lp, h = _plain_rows(s["logits"], s["actions"], c["temperature"], bonus)
    zero = torch.zeros_like(lp)
    adv = s["advantages"]
    adv = adv[:, None].expand_as(lp) if adv.dim() < lp.dim() else adv
    ratio = torch.exp(lp - s["old"])
    held = ratio.clamp(1 - CLIP_LOW, 1 + CLIP_HIGH)
    clipped = valid & (ratio * adv > held * adv)
    drift = s["ref"] - lp
    kl = torch.where(valid, torch.expm1(drift) - drift, zero)
    each = -torch.minimum(ratio * adv, held * adv) + c["kl_coef"] * kl
    d_lp = torch.where(clipped, zero, -adv * ratio) + c["kl_coef"] * (1 - torch.exp(drift))
    if bonus:
        each = each - c["entropy_coef"] * h
    w = torch.where(valid, zero + 1 if s["weights"] is None else s["weights"], zero)
    total = w.sum().clamp(min=1e-20)
    up = w * (_grad_scale(c) / total)
    d_h = -c["entropy_coef"] * up if bonus else None
    dlogits = _plain_dlogits(s["logits"], target, p, logp, h, torch.where(valid, d_lp, zero) * up, d_h, c["temperature"])
    return dict(loss=torch.where(valid, w * each, zero).sum() / total, logprob=lp, kl=kl, entropy=h,
                clip_fraction=(w * clipped).sum() / total, dlogits=dlogits)


def _plain_preference(s):
    c = s["case"]
    valid, target, p, logp, lp, _ = _plain_rows(s["logits"], s["labels"], 1.0, False)
    zero = torch.zeros_like(lp)
    w = torch.where(valid, zero + 1, zero)
    if c["average"]:
        w = w / w.sum(-1, keepdim=True).clamp(min=1)
    gap = (torch.where(valid, lp - s["ref"], zero) * w).sum(-1)
    n = c["pairs"]
    diff = gap[:n] - gap[n:]
    u = c["beta"] * diff
    softplus = lambda t: torch.clamp(t, min=0) + torch.log1p(torch.exp(-t.abs()))  # noqa: E731
    if c["kind"] == "sigmoid":
        e = c["smoothing"]
        each = (1 - e) * softplus(-u) + e * softplus(u)
        slope = c["beta"] * (e / (1 + torch.exp(-u)) - (1 - e) / (1 + torch.exp(u)))
    elif c["kind"] == "hinge":
        each = torch.clamp(1 - u, min=0)
        slope = -c["beta"] * (u < 1).float()
    else:
        off = diff - 0.5 / c["beta"]
        each, slope = off * off, 2 * off
    slope = slope * (_grad_scale(c) / n)
    d_lp = torch.cat([slope, -slope])[:, None] * w
    dlogits = _plain_dlogits(s["logits"], target, p, logp, None, d_lp, None, 1.0)
    return dict(loss=each.mean(), rewards=c["beta"] * gap, logprob=lp, dlogits=dlogits)


def _plain_adamw(s):
    c = s["case"]
    (b1, b2), lr = ADAM["betas"], ADAM["lr"]
    s["step"] += 1
    t = s["step"].double()
    step_size = (lr / (1 - torch.pow(b1, t))).float()
    root = torch.sqrt(1 - torch.pow(b2, t)).float()
    g = s["g"].float()
    norm = None
    if c["clip"]:
        norm = torch.sqrt((g * g).sum())
        g = g * (1.0 / (norm + 1e-6)).clamp(max=1.0)
    if c["bits"] == 8:
        mc = s["m"].view(-1, BLOCK).float()
        m = (mc * mc.abs() * (s["msc"][:, None] * (1 / 127 ** 2))).view(-1)
        rc = s["v"].view(-1, BLOCK).float()
        v = (rc * rc * (s["vsc"][:, None] * (1 / 255 ** 2))).square().view(-1)
    else:
        m, v = s["m"], s["v"]
    m = m + (1 - b1) * (g - m)
    v = b2 * v + (1 - b2) * (g * g)
    r = torch.sqrt(v)
    p = s["p"].float() * (1 - lr * ADAM["weight_decay"]) - step_size * (m / (r / root + ADAM["eps"]))
    s["p"].copy_(p)
    out = dict(p=s["p"], norm=norm)
    if c["bits"] == 32:
        s["m"].copy_(m)
        s["v"].copy_(v)
        return dict(out, m=s["m"], v=s["v"])
    mb, rb = m.view(-1, BLOCK), r.view(-1, BLOCK)
    msc, vsc = mb.abs().amax(1), rb.amax(1)
    some = lambda t: torch.where(t > 0, t, torch.ones_like(t))[:, None]  # noqa: E731
    mc = torch.round(127 * torch.sqrt(mb.abs() / some(msc))) * mb.sign()
    rc = torch.maximum(torch.round(255 * torch.sqrt(rb / some(vsc))), (rb > 0).float())
    s["m"].copy_(mc.view(-1))
    s["v"].copy_(rc.view(-1))
    s["msc"].copy_(msc)
    s["vsc"].copy_(vsc)
    # the values that the codes stand for; bf16 holds what 8 bits can say of them
    m8 = (mc * mc.abs() * (msc[:, None] / 127 ** 2)).to(torch.bfloat16).view(-1)
    v8 = (rc * rc * (vsc[:, None] / 255 ** 2)).square().to(torch.bfloat16).view(-1)
    return dict(out, m=m8, v=v8)


# ---------------------------------------------------------------- the package's calls
def _own_logprob(s):
    from reversability_b200 import alignment
    c = s["case"]
    r = alignment.token_logprobs(s["logits"], s["actions"], temperature=c["temperature"], entropy=c["entropy"])
    lp, h = r if c["entropy"] else (r, None)
    out = dict(logprob=lp, entropy=h)
    if c["grad"]:
        outs, grads = ([lp, h], [s["d_logprob"], s["d_entropy"]]) if c["entropy"] else ([lp], [s["d_logprob"]])
        out["dlogits"], = torch.autograd.grad(outs, s["logits"], grads)
    return out


def _own_policy(s):
    from reversability_b200 import alignment
    c = s["case"]
    args = dict(ref_logprobs=s["ref"], weights=s["weights"], clip_low=CLIP_LOW, clip_high=CLIP_HIGH,
                kl_coef=c["kl_coef"], entropy_coef=c["entropy_coef"], temperature=c["temperature"])
    if c["api"] == "grad":
        r, d = alignment.policy_loss_and_grad(s["logits"], s["actions"], s["old"], s["advantages"],
                                              grad_scale=_grad_scale(c), **args)
    else:
        r = alignment.policy_loss(s["logits"], s["actions"], s["old"], s["advantages"], **args)
        d, = torch.autograd.grad(r.loss * _grad_scale(c) if _grad_scale(c) != 1 else r.loss, s["logits"])
    return dict(loss=r.loss, logprob=r.logprobs, kl=r.kl, entropy=r.entropy, clip_fraction=r.clip_fraction, dlogits=d)


def _own_preference(s):
    from reversability_b200 import alignment
    c = s["case"]
    args = dict(kind=c["kind"], beta=c["beta"], label_smoothing=c["smoothing"] if c["kind"] == "sigmoid" else 0.0,
                average=c["average"])
    if c["api"] == "grad":
        r, d = alignment.preference_loss_and_grad(s["logits"], s["labels"], s["ref"], grad_scale=_grad_scale(c), **args)
    else:
        r = alignment.preference_loss(s["logits"], s["labels"], s["ref"], **args)
        d, = torch.autograd.grad(r.loss * _grad_scale(c) if _grad_scale(c) != 1 else r.loss, s["logits"])
    return dict(loss=r.loss, rewards=r.rewards, logprob=r.logprobs, dlogits=d)


def _own_adamw(s):
    c = s["case"]
    if "optimizer" not in s:  # built once, as a training program does
        from reversability_b200 import optim
        opt = optim.AdamW(s["params"], state_bits=c["bits"], max_norm=1.0 if c["clip"] else None, **ADAM)
        opt.set_step(STEPS_BEFORE)
        for i, p in enumerate(s["params"]):
            opt.state[p].update(exp_avg=s["ms"][i], exp_avg_sq=s["vs"][i])
            if c["bits"] == 8:
                opt.state[p].update(exp_avg_scale=s["mscs"][i], exp_avg_sq_scale=s["vscs"][i])
        if c["bits"] == 8:
            s["m8"], s["v8"] = (torch.zeros_like(s["p"], dtype=torch.bfloat16) for _ in range(2))
            s["values"] = [tuple(t[a:a + n].view(p.shape) for t in (s["m8"], s["v8"]))
                           for a, n, p in zip(s["starts"], s["sizes"], s["params"])]
        s["optimizer"] = opt
    opt = s["optimizer"]
    opt.step(grads=None if c["pdtype"] == c["gdtype"] else s["grads"])
    out = dict(p=s["p"], norm=opt.grad_norm if c["clip"] else None)
    if c["bits"] == 32:
        return dict(out, m=s["m"], v=s["v"])
    opt.moments(out=s["values"])
    return dict(out, m=s["m8"], v=s["v8"])


def run(state):
    op = state["case"]["op"]
    if own:
        return {"logprob": _own_logprob, "policy": _own_policy, "preference": _own_preference,
                "adamw": _own_adamw}[op](state)
    return {"logprob": _plain_logprob, "policy": _plain_policy, "preference": _plain_preference,
            "adamw": _plain_adamw}[op](state)


# ---------------------------------------------------------------- 64 bits
def _exact_tokens(x, actions, temperature, step, of_rows):
    """of_rows(start, log-probabilities, entropies, valid) -> a scalar or None; its gradient by autograd, in 64 bits."""
    flat, act = x.detach().reshape(-1, x.shape[-1]), actions.reshape(-1)
    lps, hs, ds = [], [], []
    for s in range(0, flat.shape[0], step):
        z = flat[s:s + step].double().requires_grad_()
        logp = torch.log_softmax(z / temperature, -1)
        valid = act[s:s + step] >= 0
        lp = logp.gather(1, act[s:s + step].clamp(min=0)[:, None])[:, 0] * valid
        h = -(torch.exp(logp) * logp).sum(-1) * valid
        scalar = of_rows(s, lp, h, valid)
        lps.append(lp.detach())
        hs.append(h.detach())
        if scalar is not None:
            ds.append(torch.autograd.grad(scalar, z)[0])
    shape = actions.shape
    return torch.cat(lps).view(shape), torch.cat(hs).view(shape), torch.cat(ds).view(x.shape) if ds else None


def _exact_logprob(c, s, step):
    n = lambda t, a, b: t.reshape(-1)[a:a + b].double()  # noqa: E731

    def scalar(a, lp, h, valid):
        if not c["grad"]:
            return None
        r = (lp * n(s["d_logprob"], a, len(lp))).sum()
        return r + (h * n(s["d_entropy"], a, len(lp))).sum() if c["entropy"] else r
    lp, h, d = _exact_tokens(s["logits"], s["actions"], c["temperature"], step, scalar)
    out = dict(logprob=lp, entropy=h if c["entropy"] else None)
    return dict(out, dlogits=d) if c["grad"] else out


def _exact_policy(c, s, step):
    rows = s["actions"].numel()
    adv = s["advantages"].double().repeat_interleave(c["group"])
    old, ref = s["old"].reshape(-1).double(), s["ref"].reshape(-1).double()
    valid = s["actions"].reshape(-1) >= 0
    w = (torch.ones(rows, device=DEV).double() if s["weights"] is None else s["weights"].double()) * valid
    total = w.sum().clamp(min=1e-20)
    sums = dict(loss=0.0, clip=0.0)
    kls = []

    def scalar(a, lp, h, ok):
        b = a + len(lp)
        ratio = (lp - old[a:b]).exp()
        free, held = ratio * adv[a:b], ratio.clamp(1 - CLIP_LOW, 1 + CLIP_HIGH) * adv[a:b]
        kl = (ref[a:b] - lp).exp() - 1 - (ref[a:b] - lp)
        each = c["kl_coef"] * kl - torch.where(held < free, held, free) - c["entropy_coef"] * h
        part = (each * w[a:b])[ok].sum() / total
        sums["loss"] = sums["loss"] + part.detach()
        sums["clip"] = sums["clip"] + ((held < free) * w[a:b]).sum() / total
        kls.append((kl * ok).detach())
        return part * _grad_scale(c)
    lp, h, d = _exact_tokens(s["logits"], s["actions"], c["temperature"], step, scalar)
    return dict(loss=sums["loss"], logprob=lp, kl=torch.cat(kls).view(lp.shape),
                entropy=h if c["entropy_coef"] else None, clip_fraction=sums["clip"], dlogits=d)


def _exact_preference(c, s, step):
    n, labels = c["pairs"], s["labels"]
    lp, _, _ = _exact_tokens(s["logits"], labels, 1.0, step, lambda *a: None)
    valid = labels >= 0
    leaf = lp.clone().requires_grad_()
    gap = ((leaf - s["ref"].double()) * valid).sum(1)
    if c["average"]:
        gap = gap / valid.sum(1).clamp(min=1)
    u = c["beta"] * (gap[:n] - gap[n:])
    if c["kind"] == "sigmoid":
        log_sigmoid = torch.nn.functional.logsigmoid
        loss = -((1 - c["smoothing"]) * log_sigmoid(u) + c["smoothing"] * log_sigmoid(-u)).mean()
    elif c["kind"] == "hinge":
        loss = torch.relu(1 - u).mean()
    else:
        loss = (gap[:n] - gap[n:] - 1 / (2 * c["beta"])).square().mean()
    up = (torch.autograd.grad(loss, leaf)[0] * valid).reshape(-1) * _grad_scale(c)
    _, _, d = _exact_tokens(s["logits"], labels, 1.0, step, lambda a, q, h, ok: (q * up[a:a + len(q)]).sum())
    return dict(loss=loss.detach(), rewards=(c["beta"] * gap).detach(), logprob=lp, dlogits=d)


def _exact_adamw(c, s):
    b1, b2 = ADAM["betas"]
    t = STEPS_BEFORE + 1
    p, g = s["p"].double(), s["g"].double()
    norm = g.norm() if c["clip"] else None
    if c["clip"]:
        g = g * min(1.0, 1.0 / (float(norm) + 1e-6))
    if c["bits"] == 8:
        m = s["msc"].double()[:, None] * (s["m"].double() / 127).view(-1, BLOCK).square()
        m = (m * s["m"].view(-1, BLOCK).sign()).view(-1)
        v = (s["vsc"].double()[:, None] * (s["v"].double() / 255).view(-1, BLOCK).square()).square().view(-1)
    else:
        m, v = s["m"].double(), s["v"].double()
    m = b1 * m + (1 - b1) * g
    v = b2 * v + (1 - b2) * g * g
    hat = (m / (1 - b1 ** t)) / ((v / (1 - b2 ** t)).sqrt() + ADAM["eps"])
    p = p - ADAM["lr"] * ADAM["weight_decay"] * p - ADAM["lr"] * hat
    if c["bits"] == 8:
        mb, vb = m.view(-1, BLOCK), v.view(-1, BLOCK)
        mm, vm = mb.abs().amax(1, keepdim=True).clamp(min=1e-300), vb.amax(1, keepdim=True).clamp(min=1e-300)
        m = (torch.round(127 * (mb.abs() / mm).sqrt()) / 127).square().mul(mm).mul(mb.sign()).view(-1)
        code = torch.round(255 * (vb / vm).pow(0.25))
        v = (torch.where((vb > 0) & (code == 0), torch.ones_like(code), code) / 255).pow(4).mul(vm).view(-1)
    return dict(p=p, norm=norm, m=m, v=v)


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "adamw":
        return _exact_adamw(case, s)
    step = max(1, (1 << 27) // case["vocab"])
    return {"logprob": _exact_logprob, "policy": _exact_policy, "preference": _exact_preference}[case["op"]](case, s, step)


# ---------------------------------------------------------------- floors
def work(case):
    if case["op"] == "adamw":
        n = sum(math.prod(s) for s in _shapes(case))
        moments = 16 if case["bits"] == 32 else 4 + 16 / BLOCK + 4  # codes in and out, scales, the bf16 values returned
        return dict(bytes=n * (2 * SIZE[case["pdtype"]] + SIZE[case["gdtype"]] + moments), flops=20 * n)
    size, vocab = SIZE[case["dtype"]], case["vocab"]
    if case["op"] == "preference":
        rows = 2 * case["pairs"] * case["length"]
        read = 0.4 * rows  # a prompt of a fifth in the mean, then half of what is left
        return dict(bytes=(read + rows) * vocab * size + 16 * rows, flops=8 * read * vocab)
    rows = case["rows"]
    read = (1 - case["masked"]) * rows
    if case["op"] == "policy" or case["grad"]:
        return dict(bytes=(read + rows) * vocab * size + 32 * rows, flops=8 * read * vocab)
    return dict(bytes=read * vocab * size + 12 * rows, flops=4 * read * vocab)
