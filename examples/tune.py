"""Tunes a reversible decoder on preference pairs or on sampled rewards: the head's logits, the loss with its
gradient over them, the reversible backward and an 8-bit AdamW step, with nothing of the vocabulary in autograd.

    python examples/tune.py --mode preference --steps 30
    python examples/tune.py --mode policy --steps 30

The data are synthetic (seeded): in a preferred answer, as for a rewarded token, ids are even, in a rejected one
odd, so the margin between the two (preference) or the reward (policy) has to rise.
"""
from __future__ import annotations

import argparse
import sys
import time
from pathlib import Path

import torch

ROOT = Path(__file__).resolve().parents[1]
if str(ROOT) not in sys.path:
    sys.path.insert(0, str(ROOT))

import reversability_b200 as rb  # noqa: E402
from reversability_b200 import alignment, optim  # noqa: E402

IGNORE = -100


def make_optimizer(model, lr: float) -> optim.AdamW:
    """Matrices with 8-bit moments; norm weights, few and sensitive, with 32-bit ones and no decay."""
    matrices = [p for p in model.parameters() if p.dim() > 1]
    norms = [p for p in model.parameters() if p.dim() == 1]
    return optim.AdamW([dict(params=matrices, state_bits=8), dict(params=norms, state_bits=32, weight_decay=0.0)],
                       lr=lr, betas=(0.9, 0.95), weight_decay=0.1, max_norm=1.0)


def scores(model, ids, labels):
    """A model's log-probabilities of the labelled tokens (forward only)."""
    with torch.no_grad(), torch.autocast("cuda", dtype=torch.bfloat16):
        return alignment.token_logprobs(model(ids), labels)


def preference_batch(pairs: int, length: int, vocab: int, gen) -> tuple[torch.Tensor, torch.Tensor]:
    """(ids, labels) [2 * pairs, length], chosen sequences first: a shared prompt of a quarter, then the answer."""
    prompt = length // 4
    ids = torch.randint(0, vocab // 2, (2 * pairs, length + 1), generator=gen, device="cuda") * 2
    ids[pairs:, prompt:] += 1
    ids[pairs:, :prompt] = ids[:pairs, :prompt]
    labels = ids[:, 1:].clone()
    labels[:, :prompt] = IGNORE
    return ids[:, :-1].contiguous(), labels


def preference_step(model, reference, opt, ids, labels):
    ref = scores(reference, ids, labels)
    loss = alignment.backward_through_head(
        model, ids, lambda logits, out: alignment.preference_loss_and_grad(logits, labels, ref, beta=0.1, out=out))
    opt.step()
    opt.zero_grad()
    half = ids.shape[0] // 2
    return loss.loss, (loss.rewards[:half] - loss.rewards[half:]).mean()


@torch.no_grad()
def sample(model, ids, gen):
    """One sampled continuation token for every position (the model's own policy at each prefix)."""
    with torch.autocast("cuda", dtype=torch.bfloat16):
        logits = model(ids)
    noise = torch.rand(logits.shape, generator=gen, device="cuda").clamp_(1e-9)
    actions = (logits.float() - torch.log(-torch.log(noise))).argmax(-1)
    return actions, alignment.token_logprobs(logits, actions)


def policy_step(model, reference, opt, ids, gen, epochs: int = 2):
    actions, old = sample(model, ids, gen)
    reward = (actions % 2 == 0).float()
    advantages = (reward - reward.mean()) / (reward.std() + 1e-6)
    ref = scores(reference, ids, actions)
    for _ in range(epochs):  # the second pass meets ratios other than 1
        loss = alignment.backward_through_head(
            model, ids, lambda logits, out: alignment.policy_loss_and_grad(
                logits, actions, old, advantages, ref_logprobs=ref, kl_coef=0.02, clip_high=0.28, out=out))
        opt.step()
        opt.zero_grad()
    return loss.loss, reward.mean()


def main(argv=None) -> list[float]:
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    ap.add_argument("--mode", choices=("preference", "policy"), default="preference")
    ap.add_argument("--steps", type=int, default=30)
    ap.add_argument("--batch", type=int, default=8, help="pairs, or sequences")
    ap.add_argument("--length", type=int, default=128)
    ap.add_argument("--layers", type=int, default=7)
    ap.add_argument("--vocab", type=int, default=50257)
    ap.add_argument("--lr", type=float, default=3e-4)
    args = ap.parse_args(argv)
    torch.manual_seed(0)
    cfg = rb.ModelConfig(vocab_size=args.vocab, n_layers=args.layers, max_sequence_length=max(args.length, 512))
    model = rb.ReversibleLM(cfg, "midpoint").cuda()
    reference = rb.ReversibleLM(cfg, "midpoint").cuda().requires_grad_(False)
    reference.load_state_dict(model.state_dict())
    opt = make_optimizer(model, args.lr)
    gen = torch.Generator(device="cuda").manual_seed(1)
    values = []
    began = time.perf_counter()
    for step in range(args.steps):
        if args.mode == "preference":
            loss, value = preference_step(model, reference, opt,
                                          *preference_batch(args.batch, args.length, args.vocab, gen))
        else:
            ids = torch.randint(0, args.vocab, (args.batch, args.length), generator=gen, device="cuda")
            loss, value = policy_step(model, reference, opt, ids, gen)
        values.append(value)
        if step % 10 == 0 or step == args.steps - 1:
            print(f"step {step:3d}  loss {float(loss):.4f}  {'margin' if args.mode == 'preference' else 'reward'} "
                  f"{float(value):.4f}  grad norm {float(opt.grad_norm):.3f}")
    torch.cuda.synchronize()
    print(f"{1e3 * (time.perf_counter() - began) / args.steps:.2f} ms per step, "
          f"{torch.cuda.max_memory_allocated() / 2 ** 20:.0f} MiB at most")
    return [float(v) for v in values]


if __name__ == "__main__":
    main()
