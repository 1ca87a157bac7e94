"""Workloads of the training operators that keep nothing they can compute again:
layer norm (two numbers a row), dropout from a counter-based generator (no mask)
and cross entropy from the hidden states in pieces of the vocabulary (no logits);
all three in functions.py.

`listed()` names the fixed cases, `draw(rng)` makes more of the same ranges,
`prepare` makes a case's inputs on the GPU, `run` does one pass in plain torch
operations (or, with `own` set, through the package), `exact` gives the same
outputs from the definitions in 64 bits and `work` the bytes and operations no
implementation can do without.
"""
import math
import random

import torch

own = False

DEV = "cuda"
DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
SIZE = {"f32": 4, "bf16": 2, "f16": 2}
IGNORE = -100
EPS = 1e-5
M32 = 0xFFFFFFFF


def listed():
    return [
        # The final norm before one generated token is scored: latency only.
        dict(name="norm_one_token", op="norm", rows=1, width=1024, dtype="bf16", out="bf16", params="f32", bias=True,
             grad=False),
        # A norm of the 20.3M decoder over a microbatch (29 x 512): fp32 residual stream in, bf16 branch out, both
        # directions.
        dict(name="norm_decoder_step", op="norm", rows=14848, width=256, dtype="f32", out="bf16", params="f32", bias=True,
             grad=True),
        # A norm of the scaled decoder (16 x 2048 tokens, width 1024) in bf16, both directions.
        dict(name="norm_scaled_step", op="norm", rows=32768, width=1024, dtype="bf16", out="bf16", params="f32", bias=True,
             grad=True),
        # fp32 throughout, an odd number of odd rows, no shift.
        dict(name="norm_odd_f32", op="norm", rows=2047, width=5001, dtype="f32", out="f32", params="f32", bias=False,
             grad=True),
        # The hidden states of one short sequence: latency only.
        dict(name="dropout_short", op="dropout", rows=64, width=256, dtype="bf16", residual=None, p=0.1, device_seed=False,
             grad=False),
        # A branch of the 20.3M decoder dropped and added to the fp32 residual stream, with the branch's gradient.
        dict(name="dropout_residual_step", op="dropout", rows=14848, width=256, dtype="bf16", residual="f32", p=0.1,
             device_seed=False, grad=True),
        # The MLP activations of the scaled decoder (width 4096), the seed on the device as a captured update keeps
        # it, both directions.
        dict(name="dropout_scaled_step", op="dropout", rows=32768, width=4096, dtype="bf16", residual=None, p=0.2,
             device_seed=True, grad=True),
        # Odd sizes in fp16, residual of the same type.
        dict(name="dropout_odd_f16", op="dropout", rows=2047, width=1001, dtype="f16", residual="f16", p=0.5,
             device_seed=False, grad=True),
        # One token is scored against the whole vocabulary of the 20.3M decoder: latency and one read of the weight.
        dict(name="head_loss_one_token", op="head", rows=1, vocab=50257, d=256, dtype="bf16", masked=0.0, reduction="sum",
             grad=False),
        # A training microbatch of the 20.3M decoder (29 x 512 tokens), loss and both gradients.
        dict(name="head_loss_decoder_step", op="head", rows=14848, vocab=50257, d=256, dtype="bf16", masked=0.0,
             reduction="mean", grad=True),
        # A training microbatch of the scaled decoder (16 x 2048 tokens, width 1024), loss and both gradients.
        dict(name="head_loss_scaled_step", op="head", rows=32768, vocab=50257, d=1024, dtype="bf16", masked=0.0,
             reduction="mean", grad=True),
        # Tuning on answers only: half of the labels masked, odd sizes, fp16 with a loss scale.
        dict(name="head_loss_masked_f16", op="head", rows=3001, vocab=32003, d=328, dtype="f16", masked=0.5,
             reduction="mean", grad=True),
    ]


def _log_int(rng, low, high):
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    op = rng.choice(["norm", "dropout", "head", "head"])
    dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
    if op == "norm":
        width = _log_int(rng, 16, 8192)
        return dict(op=op, rows=_log_int(rng, 1, max(1, min(32768, (1 << 24) // width))), width=width, dtype=dtype,
                    out=rng.choice([dtype, dtype, "bf16", "f32"]) if dtype != "f16" else rng.choice(["f16", "f32"]),
                    params=rng.choice(["f32", dtype]), bias=rng.random() < 0.7, grad=rng.random() < 0.7)
    if op == "dropout":
        width = _log_int(rng, 16, 8192)
        return dict(op=op, rows=_log_int(rng, 1, max(1, min(32768, (1 << 26) // width))), width=width, dtype=dtype,
                    residual=rng.choice([None, dtype, "f32"]), p=rng.choice([0.05, 0.1, 0.2, 0.5]),
                    device_seed=rng.random() < 0.4, grad=rng.random() < 0.7)
    dtype = rng.choice(["bf16", "bf16", "f16"])
    vocab = _log_int(rng, 100, 131072)
    d = _log_int(rng, 32, 2048)
    most = int(min(7e8 / vocab, 1e12 / (vocab * d)))  # rows that keep the case below the largest listed one
    return dict(op=op, rows=_log_int(rng, 1, max(1, min(16384, most))), vocab=vocab, d=d, dtype=dtype,
                masked=rng.choice([0.0, 0.1, 0.5]), reduction=rng.choice(["mean", "mean", "sum", "none"]),
                grad=rng.random() < 0.8)


# ---------------------------------------------------------------- inputs
def prepare(case, seed):
    gen = torch.Generator(device=DEV).manual_seed(seed)

    def normal(*shape):
        return torch.randn(*shape, generator=gen, device=DEV)

    if case["op"] == "norm":
        rows, width, grad = case["rows"], case["width"], case["grad"]
        # a residual stream: rows of different size, channels with an offset
        x = (normal(rows, width) * torch.exp(0.5 * normal(rows, 1)) + normal(width)).to(DTYPES[case["dtype"]])
        params = DTYPES[case["params"]]
        weight = (1 + 0.1 * normal(width)).to(params).requires_grad_(grad)
        bias = (0.1 * normal(width)).to(params).requires_grad_(grad) if case["bias"] else None
        dy = normal(rows, width).to(DTYPES[case["out"]]) if grad else None
        return dict(case=case, x=x.requires_grad_(grad), weight=weight, bias=bias, dy=dy)
    if case["op"] == "dropout":
        rows, width, grad = case["rows"], case["width"], case["grad"]
        rng = random.Random(seed)
        number, call = rng.getrandbits(62), rng.randrange(1 << 40)
        x = normal(rows, width).to(DTYPES[case["dtype"]])
        residual = normal(rows, width).to(DTYPES[case["residual"]]) if case["residual"] else None
        dy = normal(rows, width).to(residual.dtype if case["residual"] else x.dtype) if grad else None
        return dict(case=case, x=x.requires_grad_(grad), residual=residual, dy=dy, number=number, call=call,
                    seed=torch.tensor(number, device=DEV) if case["device_seed"] else number)
    rows, vocab, d = case["rows"], case["vocab"], case["d"]
    dtype, grad = DTYPES[case["dtype"]], case["grad"]
    # logits of a trained model: spread 2, the target token well above the rest
    weight = (normal(vocab, d) * (2 / math.sqrt(d))).to(dtype)
    labels = torch.randint(0, vocab, (rows,), generator=gen, device=DEV)
    hidden = normal(rows, d) + weight[labels].float() * (torch.rand(rows, 1, generator=gen, device=DEV) + 0.5)
    hide = torch.rand(rows, generator=gen, device=DEV) < case["masked"]
    hide[0] = False
    labels = torch.where(hide, torch.full_like(labels, IGNORE), labels)
    d_rows = normal(rows) if case["reduction"] == "none" else None
    return dict(case=case, hidden=hidden.to(dtype).requires_grad_(grad), weight=weight.requires_grad_(grad),
                labels=labels, d_rows=d_rows)


def _loss_scale(case):
    """fp16 gradients are taken of the loss times a power of two, as a loss scaler does."""
    return 4096.0 if case["dtype"] == "f16" and case["reduction"] == "mean" else 1.0


# ---------------------------------------------------------------- plain forms
def _plain_norm(s):
    x, w, b = s["x"].detach().float(), s["weight"].detach().float(), s["bias"]
    mean = x.mean(-1, keepdim=True)
    centred = x - mean
    rstd = 1 / torch.sqrt((centred * centred).mean(-1, keepdim=True) + EPS)
    xhat = centred * rstd
    y = xhat * w if b is None else xhat * w + b.detach().float()
    out = dict(y=y.to(DTYPES[s["case"]["out"]]))
    if s["dy"] is not None:
        g = s["dy"].float()
        gw = g * w
        dx = rstd * (gw - gw.mean(-1, keepdim=True) - xhat * (gw * xhat).mean(-1, keepdim=True))
        out |= dict(dx=dx.to(s["x"].dtype), dweight=(g * xhat).sum(0).to(s["weight"].dtype))
        if b is not None:
            out["dbias"] = g.sum(0).to(b.dtype)
    return out


def _mul32(a, m):
    """High and low words of the 64-bit product of 32-bit words `a` (in int64) and the constant m."""
    low, high = (a & 0xFFFF) * m, (a >> 16) * m
    return (high + (low >> 16)) >> 16, (low + ((high & 0xFFFF) << 16)) & M32


def _random_words(n, key, call, device):
    """Words 0 .. n-1 of the Philox 4x32 generator with 10 rounds (Salmon et al., SC 2011): word i is number i % 4
    of the block whose counter is (i // 4, call), both as 64 bits, under the 64-bit key."""
    block = torch.arange((n + 3) // 4, device=device)
    c0, c1 = block & M32, block >> 32
    c2, c3 = torch.full_like(block, call & M32), torch.full_like(block, call >> 32)
    k0, k1 = key & M32, key >> 32
    for _ in range(10):
        h0, l0 = _mul32(c0, 0xD2511F53)
        h1, l1 = _mul32(c2, 0xCD9E8D57)
        c0, c1, c2, c3 = h1 ^ c1 ^ k0, l1, h0 ^ c3 ^ k1, l0
        k0, k1 = (k0 + 0x9E3779B9) & M32, (k1 + 0xBB67AE85) & M32
    return torch.stack([c0, c1, c2, c3], 1).view(-1)[:n]


def _plain_dropout(s):
    c, x = s["case"], s["x"].detach()
    kept = (_random_words(x.numel(), s["number"], s["call"], x.device) >= round(c["p"] * 2 ** 32)).view(x.shape)
    zero = torch.zeros((), device=x.device)
    scale = 1 / (1 - c["p"])
    y = torch.where(kept, x.float() * scale, zero)
    if s["residual"] is not None:
        y = y + s["residual"].float()
    out = dict(y=y.to(x.dtype if s["residual"] is None else s["residual"].dtype))
    if s["dy"] is not None:
        out["dx"] = torch.where(kept, s["dy"].float() * scale, zero).to(x.dtype)
    return out


def _plain_head(s):
    c = s["case"]
    x, w, labels = s["hidden"].detach().float(), s["weight"].detach().float(), s["labels"]
    z = x @ w.T
    top = z.amax(-1, keepdim=True)
    valid = labels != IGNORE
    target = torch.where(valid, labels, torch.zeros_like(labels))[:, None]
    at = z.gather(1, target)
    e = torch.exp(z - top)
    del z
    total = e.sum(-1, keepdim=True)
    rows = torch.where(valid, (top + torch.log(total) - at)[:, 0], torch.zeros_like(top[:, 0]))
    if c["reduction"] == "none":
        loss, up = rows, s["d_rows"]
    elif c["reduction"] == "sum":
        loss, up = rows.sum(), torch.ones_like(rows)
    else:
        count = valid.sum().clamp(min=1)
        loss, up = rows.sum() / count, (_loss_scale(c) / count).expand_as(rows)
    out = dict(loss=loss)
    if c["grad"]:
        p = e.div_(total)
        p.scatter_add_(1, target, torch.full_like(at, -1.0))
        p *= torch.where(valid, up, torch.zeros_like(up))[:, None]
        out |= dict(dhidden=(p @ w).to(s["hidden"].dtype), dweight=(p.T @ x).to(s["weight"].dtype))
    return out


# ---------------------------------------------------------------- the package's calls
def _own_norm(s):
    from reversability_b200 import functions
    x, w, b = s["x"], s["weight"], s["bias"]
    y = functions.layer_norm(x, w, b, EPS, out_dtype=DTYPES[s["case"]["out"]])
    if s["dy"] is None:
        return dict(y=y)
    grads = torch.autograd.grad(y, [x, w] if b is None else [x, w, b], s["dy"])
    return dict(zip(("y", "dx", "dweight", "dbias"), (y, *grads)))


def _own_dropout(s):
    from reversability_b200 import functions
    y = functions.dropout(s["x"], s["case"]["p"], s["seed"], offset=s["call"], residual=s["residual"])
    if s["dy"] is None:
        return dict(y=y)
    dx, = torch.autograd.grad(y, s["x"], s["dy"])
    return dict(y=y, dx=dx)


def _own_head(s):
    from reversability_b200 import functions
    c = s["case"]
    loss = functions.linear_cross_entropy(s["hidden"], s["weight"], s["labels"], ignore_index=IGNORE,
                                          reduction=c["reduction"])
    if not c["grad"]:
        return dict(loss=loss)
    scaled = loss * _loss_scale(c) if _loss_scale(c) != 1 else loss
    dhidden, dweight = torch.autograd.grad(scaled, [s["hidden"], s["weight"]], s["d_rows"])
    return dict(loss=loss, dhidden=dhidden, dweight=dweight)


PLAIN = dict(norm=_plain_norm, dropout=_plain_dropout, head=_plain_head)
OWN = dict(norm=_own_norm, dropout=_own_dropout, head=_own_head)


def run(state):
    return (OWN if own else PLAIN)[state["case"]["op"]](state)


# ---------------------------------------------------------------- bytes and operations
def work(case):
    size = SIZE[case["dtype"]]
    if case["op"] == "norm":
        n, width, out = case["rows"] * case["width"], case["width"], SIZE[case["out"]]
        params = (1 + case["bias"]) * width * SIZE[case["params"]]
        moved = n * (size + out) + params
        if case["grad"]:  # x and dy in, dx out; the statistics of the rows written and read
            moved += n * (2 * size + out) + 2 * params + 16 * case["rows"]
        return dict(bytes=moved, flops=n * (8 + 14 * case["grad"]))
    if case["op"] == "dropout":
        n = case["rows"] * case["width"]
        out = SIZE[case["residual"]] if case["residual"] else size
        moved = n * (size + out * (2 if case["residual"] else 1))
        if case["grad"]:
            moved += n * (out + size)
        return dict(bytes=moved, flops=n * 2 * (1 + case["grad"]))
    rows, vocab, d = case["rows"], case["vocab"], case["d"]
    live = max(1, round(rows * (1 - case["masked"])))
    moved = (live + vocab) * d * size + rows * 8
    if case["grad"]:  # both gradients written
        moved += (rows + vocab) * d * size
    return dict(bytes=moved, flops=2 * live * vocab * d * (3 if case["grad"] else 1))


# ---------------------------------------------------------------- 64 bits
def _exact_norm(s):
    c = s["case"]
    x, w = s["x"].detach().double(), s["weight"].detach().double()
    var, mean = torch.var_mean(x, dim=1, unbiased=False, keepdim=True)
    sigma = (var + EPS).sqrt()
    y = (x - mean) / sigma * w
    if s["bias"] is not None:
        y += s["bias"].detach().double()
    out = dict(y=y)
    if c["grad"]:
        g = s["dy"].double()
        n = (x - mean) / sigma
        t = g * w
        out["dx"] = (t - (t.sum(1, keepdim=True) + n * (t * n).sum(1, keepdim=True)) / c["width"]) / sigma
        out["dweight"] = torch.einsum("rc,rc->c", g, n)
        if s["bias"] is not None:
            out["dbias"] = g.sum(0)
    return out


def _philox_block(words, key):
    """One block of four words, from whole numbers as Python has them or tensors below 2^32 held in int64."""
    a, b, c, d = words
    for r in range(10):
        x, y = (key % 2 ** 32 + r * 2654435769) % 2 ** 32, (key // 2 ** 32 + r * 3144134277) % 2 ** 32
        # 3528531795 = 53841 * 65536 + 8019 and 3449720151 = 52638 * 65536 + 36183
        ah, ch = (a * 53841 + a * 8019 // 65536) // 65536, (c * 52638 + c * 36183 // 65536) // 65536
        al = (a * 53841 % 65536 * 65536 + a * 8019) % 2 ** 32
        cl = (c * 52638 % 65536 * 65536 + c * 36183) % 2 ** 32
        a, b, c, d = ch ^ b ^ x, cl, ah ^ d ^ y, al
    return a, b, c, d


def _exact_dropout(s):
    c = s["case"]
    x = s["x"].detach().reshape(-1)
    n, call = x.numel(), s["call"]
    border = round(c["p"] * 2 ** 32)
    y, dx = torch.empty(n, dtype=torch.float64, device=x.device), torch.empty(n, dtype=torch.float64, device=x.device)
    step = 1 << 24
    for at in range(0, n, step):
        end = min(n, at + step)
        block = torch.arange(at // 4, (end + 3) // 4, device=x.device)
        words = _philox_block((block % 2 ** 32, block // 2 ** 32, torch.full_like(block, call % 2 ** 32),
                               torch.full_like(block, call // 2 ** 32)), s["number"])
        keep = (torch.stack(words, -1).flatten()[:end - at] >= border).double() / (1 - c["p"])
        y[at:end] = x[at:end].double() * keep
        if s["residual"] is not None:
            y[at:end] += s["residual"].reshape(-1)[at:end].double()
        if c["grad"]:
            dx[at:end] = s["dy"].reshape(-1)[at:end].double() * keep
    out = dict(y=y.view(s["x"].shape))
    if c["grad"]:
        out["dx"] = dx.view(s["x"].shape)
    return out


def _exact_head(s):
    c = s["case"]
    x, w, labels = s["hidden"].detach().double(), s["weight"].detach().double(), s["labels"]
    rows, vocab = x.shape[0], w.shape[0]
    loss = torch.zeros(rows, dtype=torch.float64, device=x.device)
    dx, dw = torch.zeros_like(x), torch.zeros_like(w)
    count = max(1, int((labels != IGNORE).sum()))
    for at in range(0, rows, 2048):
        live = (labels[at:at + 2048] != IGNORE).nonzero()[:, 0] + at
        if not live.numel():
            continue
        z = x[live] @ w.T
        one = torch.arange(live.numel(), device=x.device)
        lse = torch.logsumexp(z, 1)
        loss[live] = lse - z[one, labels[live]]
        if c["grad"]:
            d = torch.exp(z - lse[:, None])
            d[one, labels[live]] -= 1
            if c["reduction"] == "none":
                d *= s["d_rows"][live, None]
            dx[live] = d @ w
            dw += d.T @ x[live]
    out = dict(loss=loss if c["reduction"] == "none" else loss.sum() / (count if c["reduction"] == "mean" else 1))
    if c["grad"]:
        f = _loss_scale(c) / count if c["reduction"] == "mean" else 1.0
        out |= dict(dhidden=dx * f, dweight=dw * f)
    return out


def exact(case, seed):
    return dict(norm=_exact_norm, dropout=_exact_dropout, head=_exact_head)[case["op"]](prepare(case, seed))
