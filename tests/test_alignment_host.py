"""Host-side behaviour of the post-training operators: refusals of CPU tensors
and of invalid C arguments, before any CUDA call."""
import ctypes

import pytest
import torch

from reversability_b200 import _lib, alignment, optim


def test_cpu_tensors_are_refused():
    x, y, f = torch.zeros(2, 3, 7), torch.zeros(2, 3, dtype=torch.int64), torch.zeros(2, 3)
    for call in (lambda: alignment.token_logprobs(x, y), lambda: alignment.policy_loss(x, y, f, f),
                 lambda: alignment.policy_loss_and_grad(x, y, f, f), lambda: alignment.preference_loss(x, y, None),
                 lambda: alignment.preference_loss_and_grad(x, y, f),
                 lambda: optim.AdamW([torch.nn.Parameter(torch.zeros(3))])):
        with pytest.raises(ValueError, match="CUDA"):
            call()


def test_c_entries_reject_bad_arguments_without_cuda_calls():
    lib = _lib.lib()
    assert lib.rk_token_logprob_fwd(None, 7, 7, None, 3, 1.0, -100, 1, None, None, None, None, 0, None) == 1
    assert lib.rk_token_logprob_fwd(None, 6, 7, None, 0, 1.0, -100, 1, None, None, None, None, 0, None) == 1  # ld < vocab
    assert lib.rk_token_logprob_fwd(None, 7, 7, None, 0, 1.0, -100, 9, None, None, None, None, 0, None) == 3
    assert lib.rk_token_logprob_fwd(None, 7, 7, None, 0, 1.0, -100, 1, None, None, None, None, 0, None) == 0  # no rows
    assert lib.rk_token_logprob_fwd(16, 7, 7, 16, 1, 1.0, -100, 1, 16, None, 12, None, 0, None) == 2  # stats alignment
    need = lib.rk_token_logprob_workspace(5000)
    assert need >= 5000 * 8 and lib.rk_token_logprob_workspace(1) == 0
    assert lib.rk_token_logprob_fwd(16, 7, 7, 16, 5000, 1.0, -100, 1, 16, None, 16, 16, need - 1, None) == 6
    assert lib.rk_token_logprob_bwd(None, 7, 7, None, 0, 1.0, -100, 1, None, 16, None, None, 1, None, None, 7,
                                    None) == 1  # entropy without its gradient
    ws = lib.rk_policy_workspace(4)

    def policy(old=16, group=1, bonus=0.0, size=ws):
        terms = _lib.POLICY_TERMS.pack(old, old, 0, 0, 0, 0, group, 0.2, 0.2, 0.0, bonus, 1.0, 1.0)
        return lib.rk_policy_loss(16, 7, 7, 16, 4, -100, 1, terms, 16, None, None, 16, None, None, None, 7, 16, size, None)
    assert policy(old=0) == 1  # no old log-probabilities
    assert policy(size=ws - 1) == 6
    assert policy(group=0) == 1
    assert policy(bonus=0.1) == 1  # a bonus needs the entropies' array
    n = lib.rk_preference_workspace(1, 4)

    def preference(kind=0, size=n):
        terms = _lib.PREFERENCE_TERMS.pack(0, 0, 0.1, 0.0, 1.0, 1.0, kind, 0)
        return lib.rk_preference_loss(16, 7, 7, 16, 1, 4, -100, 1, terms, 16, 16, 16, 16, 16, None, 7, 16, size, None)
    assert preference(kind=3) == 1  # unknown kind
    assert preference(size=n - 1) == 6
    table = (ctypes.c_uint64 * 7)(0, 0, 0, 0, 0, 0, 5)
    assert lib.rk_adamw_multi_step(table, 1, 0, 0, 32, 16, 0.9, 0.9, 1e-8, None) == 1  # null tensors
    assert lib.rk_adamw_multi_step(table, 1, 0, 0, 16, 16, 0.9, 0.9, 1e-8, None) == 3
    assert lib.rk_adamw_multi_step(table, 1, 7, 0, 32, 16, 0.9, 0.9, 1e-8, None) == 3
    assert lib.rk_adamw_multi_step(None, 0, 0, 0, 32, 16, 0.9, 0.9, 1e-8, None) == 0
    assert lib.rk_adamw_multi_sumsq(table, 1, 0, 16, None) == 1
    assert lib.rk_adamw_multi_prepare(None, 3, 1.0, 0.9, 0.9, 0.0, 16, None) == 1
    assert lib.rk_adamw_multi_moments(table, 1, 0, None) == 1


def test_workspace_sizes_grow_with_rows():
    lib = _lib.lib()
    assert lib.rk_policy_workspace(0) > 0 and lib.rk_policy_workspace(1000) >= lib.rk_policy_workspace(0) + 8000
    assert lib.rk_preference_workspace(9, 100) >= 36
    assert lib.rk_adamw_multi_parts(0) == 0 and lib.rk_adamw_multi_parts(65) == 2 * lib.rk_adamw_multi_parts(64)
