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


# ---------------------------------------------------------------- group norm
PATHS = [(5, 64, (9, 9), 8), (5, 512, (), 8), (4, 32, (20, 20), 4), (3, 64, (9, 9), 64), (3, 64, (9, 9), 32), (3, 64, (9, 9), 16), (5, 24, (), 1),
         (3, 96, (11, 5), 4), (4, 24, (6, 6), 4), (6, 30, (5, 4), 5), (5, 1200, (), 4), (2, 64, (130, 117), 4), (2, 2304, (2,), 3), (2, 48, (84, 84), 6),
         (2, 56, (60, 50), 2), (2, 21, (90, 70), 3)]   # samples in registers of a wave and of several, groups in a wave, slabs


@pytest.mark.gpu
@pytest.mark.parametrize("B,C,sp,groups", PATHS)
def test_norm_of_a_constant_is_the_bias(B, C, sp, groups):
    """Sums go about a value of the group, so equal values, of any size, have no deviation at all: h is 0, and dx and dweight are
    what h = 0 makes of them."""
    x, w, b, dy = norm_inputs(B, C, sp, torch.float32)
    w.requires_grad_()
    for value in (3.3, -1000.1, 3000.1, 7e-7, 3e30):
        flat = torch.full_like(x, value).requires_grad_()
        y = group_norm_act(flat, groups, w, b)
        assert torch.equal(y, b.view(1, -1, *(1,) * len(sp)).expand_as(y)), value
        dx, dw = torch.autograd.grad(y, (flat, w), dy)
        assert (dw == 0).all(), value
        d = (dy * w.detach().view(1, -1, *(1,) * len(sp))).double().reshape(B, groups, -1)
        want = (d - d.mean(-1, keepdim=True)).reshape(x.shape) / 1e-5 ** 0.5
        assert (dx.double() - want).norm() <= 2.0 ** -20 * want.norm(), value


@pytest.mark.gpu
@pytest.mark.parametrize("B,C,sp,groups", PATHS)
def test_norm_of_a_large_mean(B, C, sp, groups):
    """About a mean of 3,000 deviations: h is off by two ulp of the mean (its rounding where it is stored, and its sum's), times rstd, and by a
    few 2^-24 of itself; silu's slope is below 1.1 and changes by 0.5 at most, and dx and dw follow h by their formulas."""
    x, w, b, dy = norm_inputs(B, C, sp, torch.float32)
    x = (x + 3000.0).requires_grad_()
    w, b = w.requires_grad_(), b.requires_grad_()
    y = group_norm_act(x, groups, w, b, act="silu")
    dx, dw, db = torch.autograd.grad(y, (x, w, b), dy)
    want = norm64(x.detach(), groups, w.detach(), b.detach(), 1e-5, "silu", dy)
    x3 = x.detach().double().reshape(B, groups, -1)
    mean, r = x3.mean(-1), 1.0 / (x3.var(-1, unbiased=False) + 1e-5).sqrt()
    shift = (2 * 2.0 ** -23 * mean.abs() * r).max().item()
    few, big = 64 * 2.0 ** -24, w.detach().abs().max().item()
    assert (y.detach().double() - want[0]).abs().max() <= 1.1 * big * shift + few * (1 + want[0].abs().max())
    # dx = r (dh - mean dh - h mean(dh h)): dh changes by 0.5 w^2 |dy| shift, the last term by 3 shift of dh's size
    assert (dx.double() - want[1]).norm() <= (0.5 * big ** 2 + 3 * big + few / shift) * shift * r.max() * 1.1 * dy.double().norm()
    to_c = lambda t: t.double().abs().sum([0, *range(2, t.dim())])   # noqa: E731
    assert ((dw.double() - want[2]).abs() <= (1.1 + 0.5 * big * 6) * shift * to_c(dy) + few * 6 * to_c(dy)).all()
    assert ((db.double() - want[3]).abs() <= 0.5 * big * shift * to_c(dy) + few * to_c(dy)).all()


@pytest.mark.gpu
def test_norm_does_not_go_by_alignment():
    """The same values off a 16-byte boundary take another kernel, and give the same norm of a large mean."""
    x, w, b, _ = norm_inputs(5, 64, (9, 9), torch.float32, offset=3000.0)
    off = torch.empty(x.numel() + 1, device="cuda")[1:].view(5, 9, 9, 64).permute(0, 3, 1, 2)
    off.copy_(x)
    d = group_norm_act(x, 8, w, b).double() - group_norm_act(off, 8, w, b).double()
    assert d.abs().max() <= 4 * 2.0 ** -23 * 3000.0 * 1.6


@pytest.mark.gpu
@pytest.mark.parametrize("rows,far", [(1, 1e4), (128, 1e5)])
def test_norm_of_a_far_first_value(rows, far):
    """Samples of one slab, 512 pixels a thread, whose first pixel or border is far from the rest: it is one of few values that
    its sums go about. Runs of 16 values lose 16 roundings at most, their joining a few."""
    B, C, S = 520, 64, 16384
    g = torch.Generator(device="cuda").manual_seed(0)
    x = torch.randn(B, 128, S // 128, C, generator=g, device="cuda")
    x[:, 0, :rows] = far
    y = group_norm_act(x.permute(0, 3, 1, 2), 8)
    for i in (0, B - 1):
        want = norm64(x[i:i + 1].permute(0, 3, 1, 2), 8, None, None, 1e-5, "none")
        x3 = x[i].double().view(S, 8, 8).permute(1, 0, 2).reshape(8, -1)
        d = (y[i].double() - want[0]).reshape(8, -1)
        shift = 2 * 2.0 ** -23 * x3.mean(-1).abs() / x3.std(-1)
        # the rest, far below the standard deviation, is compared as itself: rstd's error shows on all values alike
        limit = 128 * 2.0 ** -24 * want[0].abs().reshape(8, -1) + shift[:, None] + 8 * 2.0 ** -24 * want[0].abs().reshape(8, -1).max(-1, keepdim=True).values / 64
        assert (d.abs() <= limit).all(), (d.abs() / limit).max().item()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("B,C,sp,groups", [(6, 64, (9, 9), 8), (300, 30, (), 5), (40, 24, (9, 9), 4), (50, 1024, (), 8), (2, 64, (130, 117), 4), (2, 21, (90, 70), 3)])
def test_norm_relu_gradient(B, C, sp, groups, dtype):
    """relu's gradient jumps where its argument is 0: dy is 0 wherever it is within a rounding of it."""
    x, w, b, dy = norm_inputs(B, C, sp, dtype)
    z = norm64(x, groups, w, b, 1e-5, "none")
    dy = torch.where(z.abs() < 1e-3, torch.zeros_like(dy), dy)
    x, w, b = (t.requires_grad_() for t in (x, w, b))
    grads = torch.autograd.grad(group_norm_act(x, groups, w, b, act="relu"), (x, w, b), dy)
    want = norm64(x.detach(), groups, w.detach(), b.detach(), 1e-5, "relu", dy)[1:]
    cells = x.numel() // B // groups
    for a, e in zip(grads, want):
        rel = 2.0 ** -8 if a.dtype == torch.bfloat16 else 2.0 ** -24 * (32 + 4 * cells ** 0.5) * 8
        assert (a.double() - e).norm() <= rel * e.norm() + 2.0 ** -20 * x.numel() ** 0.5


@pytest.mark.gpu
def test_norm_of_more_than_the_caches():
    """One position a sample and more than 256 MiB: x and dy are read past the caches."""
    B, C = 280000, 512
    g = torch.Generator(device="cuda").manual_seed(0)
    x, dy = (torch.randn(B, C, generator=g, device="cuda").bfloat16() for _ in range(2))
    w, b = (torch.randn(C, generator=g, device="cuda") for _ in range(2))
    x, w, b = (t.requires_grad_() for t in (x, w, b))
    y = group_norm_act(x, 8, w, b, act="silu")
    grads = torch.autograd.grad(y, (x, w, b), dy)
    dw, db = torch.zeros(C, dtype=torch.float64, device="cuda"), torch.zeros(C, dtype=torch.float64, device="cuda")
    for i in range(0, B, 40000):
        s = slice(i, i + 40000)
        want = norm64(x[s].detach(), 8, w.detach(), b.detach(), 1e-5, "silu", dy[s])
        assert (y[s].double() - want[0]).norm() <= 2.0 ** -8 * want[0].norm()
        assert (grads[0][s].double() - want[1]).norm() <= 2.0 ** -8 * want[1].norm()
        dw += want[2]
        db += want[3]
    # sums of 280,000 terms in trees of blocks: a few 2^-24 of the sum of absolute values
    assert (grads[1].double() - dw).abs().max() <= 256 * 2.0 ** -24 * B and (grads[2].double() - db).abs().max() <= 256 * 2.0 ** -24 * B


@pytest.mark.gpu
def test_step_of_odd_heads_past_the_caches():
    """States of more than 256 MiB whose rows no 16-byte access fits: a column a lane, two rows of blocks, past the caches."""
    N, D, E = 4300, 128, 127
    q, k, v, decay, start, state, _, _ = attend_inputs(1, N, 1, D, E, torch.float32, starts=0.2)
    assert state.numel() * 4 > 256 << 20
    want, last = attend64(q, k, v, decay, start, state, D ** -0.5)
    size, lsize = attend64(q.abs(), k.abs(), v.abs(), decay, start, state.abs(), D ** -0.5)
    out = linear_attention_step(q[0], k[0], v[0], decay, state, start[0])
    f32 = (16 + D) * 2.0 ** -23
    assert ((out.double() - want[0]).abs() <= f32 * size[0]).all() and ((state.double() - last).abs() <= f32 * lsize).all()


# ---------------------------------------------------------------- as a program uses them
@pytest.mark.gpu
def test_operators_run_behind_what_makes_their_inputs():
    """On a side stream whose inputs come late, behind long products: a launch on any other stream would see the old ones."""
    q, k, v, decay, start, state, do, ds = attend_inputs(300, 2, 2, 64, 64, torch.bfloat16)
    x, w, b, dy = norm_inputs(5, 24, (9, 9), torch.bfloat16)

    def work(q, k, v, state, x, S):
        leaves = [t.requires_grad_() for t in (q, k, v, state, x)]
        out, last = linear_attention(*leaves[:3], decay, start, leaves[3])
        y = group_norm_act(leaves[4], 3, w, b, act="silu")
        grads = torch.autograd.grad((out, last, y), leaves, (do, ds, dy))
        with torch.no_grad():
            one = linear_attention_step(leaves[0][0], leaves[1][0], leaves[2][0], decay, S, start[0])
        return [out.detach(), last.detach(), y.detach(), *grads, one, S]

    want = work(*(t.clone() for t in (q, k, v, state, x, state)))
    late = [torch.zeros_like(t) for t in (q, k, v, state, x, state)]
    big = torch.randn(8192, 8192, device="cuda")
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        for _ in range(4):
            big @ big
        for to, t in zip(late, (q, k, v, state, x, state)):
            to.copy_(t)
        got = work(*late)
    side.synchronize()
    assert all(torch.equal(a, c) for a, c in zip(got, want))


@pytest.mark.gpu
@pytest.mark.parametrize("sp", [(), (3,), (9, 9)])
def test_outputs_may_be_changed_in_place(sp):
    """What follows a norm may add to its result or clamp it in place, as it may with torch's own, and the gradient is the same."""
    x, w, b, dy = norm_inputs(6, 32, sp, torch.float32)
    r = torch.randn_like(x)
    leaves = [t.requires_grad_() for t in (x, w, b)]
    want = torch.autograd.grad((group_norm_act(x, 4, w, b, act="silu") * 2 + r).clamp(min=0), leaves, dy)
    y = group_norm_act(x, 4, w, b, act="silu")
    y *= 2
    y += r
    y.clamp_(min=0)
    assert all(torch.equal(a, e) for a, e in zip(torch.autograd.grad(y, leaves, dy), want))
    q, k, v, decay, start, state, do, _ = attend_inputs(7, 2, 2, 16, 16, torch.float32)
    (dq,) = torch.autograd.grad(linear_attention(q.requires_grad_(), k, v, decay, start, state)[0] * 2, q, do)
    out = linear_attention(q, k, v, decay, start, state)[0]
    out *= 2
    assert torch.equal(torch.autograd.grad(out, q, do)[0], dq)


@pytest.mark.gpu
def test_memory_net_makes_its_input_once(monkeypatch):
    """The scaled observations take one buffer: nothing that is not there yet is copied."""
    net = memory.make_memory_net()
    obs = torch.zeros(256, 4, 84, 84, dtype=torch.uint8, device="cuda")
    state, peak = net.initial_state(256), []
    net.step(obs, None, state)
    inner = memory.policy_input
    monkeypatch.setattr(memory, "policy_input", lambda o, x: peak.append(torch.cuda.max_memory_allocated() - before) or inner(o, x))
    torch.cuda.reset_peak_memory_stats()
    before = torch.cuda.memory_allocated()
    net.step(obs, None, state)
    assert peak == [obs.numel() * 2]


def test_build_needs_the_operators_last(monkeypatch):
    """Where the operators cannot be built (no C++ compiler or torch headers), the emulator and the oracle are built all the same, and
    build() says what failed."""
    import __graft_entry__ as entry
    import build_native
    import build_ops
    done = []
    monkeypatch.setattr(build_native, "build", lambda *a, **k: done.append("emulator"))
    monkeypatch.setattr(entry.subprocess, "run", lambda *a, **k: done.append("oracle"))

    def fails(*a, **k):
        raise RuntimeError("no compiler")
    monkeypatch.setattr(build_ops, "build", fails)
    with pytest.raises(RuntimeError, match="no compiler"):
        entry.build()
    assert done == ["emulator", "oracle"]


def test_rollout_takes_networks_without_memories():
    """A network's own `initial_state` does not make it one whose `act` takes memories."""
    from types import SimpleNamespace
    from fast_mario_env_amd.rollout import Rollout
    env = SimpleNamespace(n=2, dev=torch.device("cpu"), k=4)

    class Recurrent:
        def initial_state(self, batch, layers):
            raise AssertionError("not asked for")

        def act(self, obs, generator=None):
            return obs

    assert Rollout(env, Recurrent(), T=3).memory is None
    ro = Rollout(env, memory.make_memory_net(device="cpu"), T=3)
    assert ro.memory.shape == (2, 8, 64, 64) and torch.equal(ro.memory0, ro.memory)
