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


def rounded_once(got, want, size, f32, heads, what):
    """`heads`: the dimensions of got that count an env's head; the others are its values."""
    assert got.shape == want.shape and torch.isfinite(got).all(), what
    d = got.double() - want
    off = d.abs() / (2.0 ** -8 * want.abs() + (2.0 ** -16 + f32) * size + 1e-30)
    assert off.max() <= 1, (what, off.max().item())
    rest = [i for i in range(got.dim()) if i not in heads]
    norm = lambda x: x.square().sum(rest).sqrt()   # noqa: E731
    least = norm(want.to(got.dtype).double() - want)
    if got.numel() // least.numel() >= 1024:
        assert (norm(d) <= 1.05 * least + 2.0 ** -13 * norm(want)).all(), (what, norm(d) / norm(want), least / norm(want))


def check_once(q, k, v, decay, start, state, do, ds):
    leaves = [t.detach().requires_grad_() for t in (q, k, v, state)]
    out, last = linear_attention(*leaves[:3], decay, start, leaves[3])
    with torch.no_grad():
        assert torch.equal(linear_attention(q, k, v, decay, start, state)[0], out)
    grads = torch.autograd.grad((out, last), leaves, (do, ds))
    scale = q.shape[-1] ** -0.5
    want = attend64(q, k, v, decay, start, state, scale, do, ds)
    size = attend64(q.abs(), k.abs(), v.abs(), decay, start, state.abs(), scale, do.abs(), ds.abs())
    f32 = (q.shape[0] + q.shape[-1] + v.shape[-1] + 16) * 2.0 ** -23
    for i, x, name in ((0, out.detach(), "out"), (2, grads[0], "dq"), (3, grads[1], "dk"), (4, grads[2], "dv")):
        rounded_once(x, want[i], size[i], f32, (1, 2), name)
    for i, x, name in ((1, last.detach(), "state"), (5, grads[3], "dstate")):
        assert ((x.double() - want[i]).abs() <= f32 * size[i]).all(), name


@pytest.mark.gpu
@pytest.mark.parametrize("T,N,H,D,E", [(130, 3, 2, 64, 64), (64, 4, 2, 32, 32), (200, 2, 2, 128, 128), (128, 3, 3, 40, 24), (97, 2, 2, 64, 128),
                                       (300, 5, 1, 16, 96), (1000, 1, 2, 64, 64), (513, 2, 2, 128, 32), (90, 2, 2, 33, 5)])
def test_attention_is_rounded_once(T, N, H, D, E):
    check_once(*attend_inputs(T, N, H, D, E, torch.bfloat16, seed=T, starts=0.02))


@pytest.mark.gpu
def test_attention_keeps_its_states():
    """Only the state that entered a chunk gives dq: k and v are zero, and the memory decays slowly."""
    q, k, v, _, _, state, do, ds = attend_inputs(256, 2, 2, 64, 64, torch.bfloat16)
    decay = torch.tensor([0.9999, 0.99], device="cuda")
    check_once(q, torch.zeros_like(k), torch.zeros_like(v), decay, None, state, do, ds)


@pytest.mark.gpu
@pytest.mark.parametrize("N,H,D,E", [(40, 2, 64, 64), (300, 1, 33, 7)])
def test_step_is_rounded_once(N, H, D, E):
    q, k, v, decay, start, state, _, _ = attend_inputs(1, N, H, D, E, torch.bfloat16)
    want, _ = attend64(q, k, v, decay, start, state, D ** -0.5)
    size, _ = attend64(q.abs(), k.abs(), v.abs(), decay, start, state.abs(), D ** -0.5)
    out = linear_attention_step(q[0], k[0], v[0], decay, state, start[0])
    rounded_once(out[None], want, size, (16 + D) * 2.0 ** -23, (0,), "out")


# ---------------------------------------------------------------- what is not finite
@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
def test_attention_what_is_not_finite_stays_in_its_episode_of_a_cut_sequence(bad, dtype):
    """Few long sequences go in segments (T = 1500 of two heads): a bad value in any of them shows in no other episode, forwards or back."""
    T, N, H, D = 1500, 2, 1, 32
    starts = (100, 470, 700, 1100)
    edges = (0,) + starts + (T,)
    start = torch.zeros(T, N, dtype=torch.bool, device="cuda")
    start[list(starts)] = True
    q, k, v, decay, _, state, do, ds = attend_inputs(T, N, H, D, D, dtype)
    leaves = [t.detach().requires_grad_() for t in (q, k, v)]
    out, end = linear_attention(*leaves, decay, start, state)
    clean = [out.detach(), *torch.autograd.grad((out, end), leaves, (do, ds))]
    for where in (50, 99, 100, 300, 900, 1099, 1499):
        e = max(i for i, x in enumerate(edges) if x <= where)
        mine = slice(edges[e], edges[e + 1])
        for which in range(4):
            x = [t.clone() for t in (q, k, v, do)]
            x[which][where] = bad
            leaves = [t.requires_grad_() for t in x[:3]]
            out, end = linear_attention(*leaves, decay, start, state)
            got = [out.detach(), *torch.autograd.grad((out, end), leaves, (x[3], ds))]
            for name, a, c in zip(("out", "dq", "dk", "dv"), got, clean):
                for s in (slice(0, mine.start), slice(mine.stop, T)):
                    assert torch.isfinite(a[s]).all(), (where, which, name)
                    assert torch.allclose(a[s].float(), c[s].float(), rtol=2e-2, atol=2e-2), (where, which, name)
            assert torch.isfinite(got[0][mine.start:where]).all(), (where, which)        # nor in a step before it
            if which < 3:
                assert not torch.isfinite(got[0][where]).all(), (where, which)
            assert torch.isfinite(end).all() == (which in (0, 3) or mine.stop < T), (where, which)
    (bad_ds := ds.clone()).fill_(bad)                        # a gradient that comes from behind reaches the last episode only
    leaves = [t.detach().requires_grad_() for t in (q, k, v)]
    out, end = linear_attention(*leaves, decay, start, state)
    for a, c in zip(torch.autograd.grad((out, end), leaves, (do, bad_ds)), clean[1:]):
        assert torch.allclose(a[:1100].float(), c[:1100].float(), rtol=2e-2, atol=2e-2)


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
