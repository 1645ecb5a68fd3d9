"""The operators of a policy with a memory (fast_mario_env_amd.memory) where digits can be lost: each bf16 result is rounded once, a
constant or a large mean costs a norm no digits, and what is not finite stays where it belongs, on every path.

A result in bf16 is the rounding of a sum kept to 2^-16 of its parts, so an element is off by at most 2^-8 of itself and (2^-16 + (T + D +
E + 16) 2^-23) of the sum of absolute values; over an env's head the error is, in norm, that of rounding the exact result, within
5 % (the few values near the middle of two neighbours that fall to the other side), and 2^-13 of the result for independent errors of
2^-16 of its parts (they grow as the result does, by squares)."""

import pytest
import torch

from fast_mario_env_amd import memory
from fast_mario_env_amd.memory import group_norm_act, head_decays, linear_attention, linear_attention_step
from test_memory import attend64, attend_inputs, norm64, norm_inputs


# ---------------------------------------------------------------- what is not finite
@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_attention_what_is_not_finite_stays_in_its_column(dtype):
    """One value of k is infinite: of dq, which meets the state row by row, only that row is."""
    T, N, H, D = 130, 1, 1, 32
    q, k, v, decay, _, state, do, ds = attend_inputs(T, N, H, D, D, dtype)
    k[5, 0, 0, 7] = float("inf")
    leaves = [t.requires_grad_() for t in (q, k, v)]
    out, end = linear_attention(*leaves, decay, None, state)
    (dq,) = torch.autograd.grad((out, end), leaves[:1], (do, ds))
    good = torch.ones(D, dtype=torch.bool, device="cuda")
    good[7] = False
    want = attend64(q.detach().float(), torch.where(torch.isinf(k), 0.0, k.detach().float()), v.detach(), decay, None, state, D ** -0.5, do, ds)[2]
    assert torch.isfinite(dq[..., good]).all() and not torch.isfinite(dq[5:, ..., 7]).any()
    assert torch.allclose(dq[..., good].double(), want[..., good], rtol=2e-2, atol=2e-2)
