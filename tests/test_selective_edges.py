"""The operators of a memory that selects and of the gradients' norm where a value, a layout or a state is out of the ordinary: values that are not
finite, states that go on from a sequence to single steps, gradients that share memory or only lie between one another. Definitions and
bounds are those of test_selective.py."""
import random

import pytest
import torch

from fast_mario_env_amd.memory import (causal_conv_act, causal_conv_act_step, group_norm_act, linear_attention, linear_attention_step, make_memory_net,
                                       state_scan, state_scan_step)
from fast_mario_env_amd.rollout import _share_elements, clip_gradients, gradient_norm
from test_selective import DTYPES, check_scan, conv_inputs, scan64, scan_inputs


def same_kind(got, want, what):
    """NaN where the definition has NaN, an infinity where it has that infinity, finite elsewhere."""
    assert got.shape == want.shape, what
    assert torch.equal(torch.isnan(got), torch.isnan(want)), what
    for inf in (float("inf"), -float("inf")):
        assert torch.equal(got == inf, want == inf), (what, inf)


# ---------------------------------------------------------------- convolution
@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("act", ["none", "relu", "silu"])
@pytest.mark.parametrize("C,K", [(16, 4), (5, 4), (64, 8), (8, 1)])
def test_convolution_keeps_a_nan(C, K, act, dtype):
    """A NaN among the inputs, the weights, the biases or in the state shows in every step that sees it and in its weights' gradient, and nowhere else."""
    T, N, c = 24, 2, 3
    x, w, b, _, state, dy, _ = conv_inputs(T, N, C, K, dtype, starts=None)

    def run(x, w, b, state):
        leaves = [t.detach().requires_grad_() for t in (x, w)]
        y, _ = causal_conv_act(*leaves, b, None, state, act)
        return (y.detach(), *torch.autograd.grad(y, leaves, dy))

    clean = run(x, w, b, state)
    for name in ("x", "w", "b", "state"):
        if name == "state" and K == 1:
            continue
        a = dict(x=x.clone(), w=w.clone(), b=b.clone(), state=state.clone())
        hit = torch.zeros(T, N, C, dtype=torch.bool, device="cuda")
        if name == "x":
            a["x"][9, 1, c], hit[9:9 + K, 1, c] = float("nan"), True
        elif name == "state":
            a["state"][1, -1, c], hit[:K - 1, 1, c] = float("nan"), True
        else:
            a[name][c], hit[:, :, c] = float("nan"), True
        y, dx, dw = run(**a)
        assert torch.isnan(y[hit]).all() and torch.equal(y[~hit], clean[0][~hit]), name
        others = [i for i in range(C) if i != c]
        assert torch.equal(dx[..., others], clean[1][..., others]) and torch.equal(dw[others], clean[2][others]), name
        if name == "x":
            assert torch.isnan(dw[c]).all()
        if name != "state":
            s = state.clone()
            step = causal_conv_act_step(a["x"][9], a["w"], a["b"], s, act=act)
            assert torch.equal(torch.isnan(step), hit[9])


@pytest.mark.parametrize("device", ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)])
def test_convolution_relu_at_zero(device):
    """relu's slope is 0 where its argument is 0 (nothing but zeros, no bias), 1 where it is a NaN: on either device."""
    x, w, _, _, _, dy, _ = conv_inputs(9, 2, 8, 4, torch.float32, starts=None, device=device)
    for value, slope in ((0.0, 0.0), (float("nan"), 1.0)):
        leaf = torch.full_like(x, value).requires_grad_()
        b = torch.zeros(8, device=device, requires_grad=True)
        y, _ = causal_conv_act(leaf, w, b, act="relu")
        dx, db = torch.autograd.grad(y, (leaf, b), dy)
        assert torch.equal(y.detach().nan_to_num(5.0), torch.full_like(y, 0.0 if value == 0.0 else 5.0))
        assert torch.allclose(db, slope * dy.sum((0, 1)), atol=18 * 2.0 ** -24 * 18) and torch.isfinite(dx).all() and (dx == 0).all() == (slope == 0)


@pytest.mark.parametrize("device", ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)])
@pytest.mark.parametrize("T", [1, 2, 7])
def test_steps_go_on_from_a_sequence(T, device):
    """The state that a sequence returns is one that the steps take and update, without copies of it elsewhere; so are the network's memories."""
    x, w, b, start, state, _, _ = conv_inputs(T + 4, 3, 8, 4, torch.float32, device=device)
    a, _, _ = scan_inputs(T + 4, 3, 8, 4, 1, torch.float32, device=device)
    timed = lambda part: {n: v[part] if n in ("x", "dt", "B", "C", "z", "start") else v for n, v in a.items()}   # noqa: E731
    for given in (None, state):
        y, _ = causal_conv_act(x, w, b, start, given)
        _, s = causal_conv_act(x[:T], w, b, start[:T], given)
        for t in range(T, T + 4):
            assert torch.allclose(causal_conv_act_step(x[t], w, b, s, start[t]), y[t], atol=1e-5)
    y, _ = state_scan(**a)
    _, h = state_scan(**timed(slice(0, T)))
    for t in range(T, T + 4):
        assert torch.allclose(state_scan_step(**{**timed(t), "state": h}), y[t], atol=1e-4)
    back = lambda t: t.permute(*reversed(range(t.dim()))).contiguous().permute(*reversed(range(t.dim())))   # noqa: E731
    for n in (0, 1, T):                                      # inputs of another order in memory
        for given in (None, back):
            c = {k: back(v[:n] if k in ("x", "dt", "B", "C", "z", "start") else v) for k, v in a.items()}
            c["state"] = given and c["state"]
            q, d, m = back(torch.randn(n, 3, 2, 4, device=device)), torch.ones(2, device=device), torch.zeros(3, 2, 4, 4, device=device)
            for last in (causal_conv_act(back(x[:n]), back(w), b, None, given and given(state))[1], state_scan(**c)[1],
                         linear_attention(q, q, q, d, None, given and given(m))[1]):
                assert last.is_contiguous()
    if device == "cpu":
        net = make_memory_net(device="cpu", memory="scan")
        obs = torch.randint(0, 256, (T + 2, 3, 4, 84, 84), dtype=torch.uint8, generator=torch.Generator().manual_seed(0))
        with torch.no_grad():
            logits, _, _ = net(obs)
            _, _, memories = net(obs[:T])
            for t in range(T, T + 2):
                assert torch.allclose(net.step(obs[t], None, memories)[0], logits[t], atol=1e-5)


# ---------------------------------------------------------------- scan
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
def test_cpu_what_is_not_finite_stays_in_its_episode(bad):
    """On the CPU too: a value that is not finite shows in no step and no gradient of a step of another episode, and in no
    gradient at all where no step sees it."""
    T, N, C, S = 12, 2, 6, 3
    a, dout, ds = scan_inputs(T, N, C, S, 1, torch.float32, device="cpu")
    x, w, b, _, window, dy, dw = conv_inputs(T, N, C, 4, torch.float32, device="cpu")
    start = a["start"] = torch.zeros(T, N, dtype=torch.bool)
    start[4], start[8] = True, True

    def run(a, dout, x, window):
        leaves = {n: a[n].detach().requires_grad_() for n in ("x", "dt", "B", "C", "z")}
        y, end = state_scan(**{**a, **leaves})
        leaf = x.detach().requires_grad_()
        y2, last = causal_conv_act(leaf, w, b, start, window)
        return [y.detach(), y2.detach(), *torch.autograd.grad((y, end), list(leaves.values()), (dout, ds)), *torch.autograd.grad((y2, last), leaf, (dy, dw))]

    clean = run(a, dout, x, window)
    for where in (0, 3, 4, 7, 8, T - 1):
        hit = slice(where // 4 * 4, where // 4 * 4 + 4)
        for name in ("x", "dt", "B", "C", "z", "dout", "state"):
            b2, do, x2, st2 = dict(a), dout.clone(), x.clone(), window
            if name == "dout":
                do[where] = bad
            elif name == "state":
                if where:
                    continue
                b2["state"], st2 = torch.full_like(a["state"], bad), torch.full_like(window, bad)
            else:
                b2[name] = a[name].clone()
                b2[name][where] = x2[where] = bad
            for got, want in zip(run(b2, do, x2, st2), clean):
                for part in (slice(0, hit.start), slice(hit.stop, T)):
                    assert torch.equal(got[part], want[part]), (where, name)
    start[0] = True                                          # a state that nothing looks at: no gradient knows it
    names = ("x", "dt", "A", "B", "C", "D", "z", "dt_bias", "state")
    leaves = {n: a[n].detach().requires_grad_() for n in names}
    dirty = {**leaves, "state": torch.full_like(a["state"], bad).requires_grad_()}
    for v in (leaves, dirty):
        y, end = state_scan(**{**a, **v})
        v["grads"] = torch.autograd.grad((y, end), [v[n] for n in names], (dout, ds))
    assert all(torch.equal(p, q) for p, q in zip(leaves["grads"], dirty["grads"]))


def rising(T, N, C, S, G, dtype, D, z):
    """Inputs whose products are all positive but for z's, and decays that do not vanish: an infinity keeps its sign."""
    a, dout, ds = scan_inputs(T, N, C, S, G, dtype, starts=None, D=D, z=z)
    for n in ("x", "B", "C", "state"):
        a[n] = a[n].abs() + 0.25
    a["A"] = a["A"].clamp(min=-1.0)
    if D:
        a["D"] = a["D"].abs()
    a["start"] = torch.zeros(T, N, dtype=torch.bool, device="cuda")
    a["start"][T // 2, 0] = True
    return a, dout.abs() + 0.25, ds.abs()


def check_infinite(a, dout, ds):
    """y, the state and the gradients that do not add infinities of both signs, against the definition."""
    names = ("x", "B", "C", "z", "state")
    leaves = {n: a[n].detach().requires_grad_() for n in names if a[n] is not None}
    y, last = state_scan(**{**a, **leaves})
    got = dict(zip(leaves, torch.autograd.grad((y, last), list(leaves.values()), (dout, ds))))
    with torch.no_grad():
        again = state_scan(**a)
    want = scan64(*(a[n] for n in ("x", "dt", "A", "B", "C", "D", "z", "dt_bias", "start", "state")), dout, ds)
    for v, u in zip((y.detach(), last.detach()), again):
        assert torch.equal(v.nan_to_num(7.0), u.nan_to_num(7.0))
    same_kind(y.detach(), want[0], "y")
    same_kind(last.detach(), want[1], "state")
    for n, g in got.items():
        same_kind(g, want[2]["d" + n], "d" + n)
    h = a["state"].clone()
    for t in range(3):
        one = {n: v[t] if v is not None and n in ("x", "dt", "B", "C", "z", "start") else v for n, v in a.items()}
        same_kind(state_scan_step(**{**one, "state": h}), want[0][t], "step")


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("z", [False, True])
@pytest.mark.parametrize("T,C,S,G", [(20, 64, 16, 1), (20, 40, 4, 2), (20, 48, 64, 1), (600, 24, 8, 1), (600, 70, 24, 2)])
def test_scan_without_D_keeps_an_infinity(T, C, S, G, z, dtype):
    """An infinite x, an infinite gradient of y: what is not there adds no 0 times infinity."""
    for D in (False, True):
        for what in ("x", "dout"):
            a, dout, ds = rising(T, 2, C, S, G, dtype, D, z)
            if a["z"] is not None:
                a["z"] = a["z"].abs() + 0.25
            (a["x"] if what == "x" else dout)[2, 1, 5] = float("inf")
            check_infinite(a, dout, ds)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("T", [20, 600])
@pytest.mark.parametrize("C,S,G", [(64, 1, 1), (40, 3, 2), (65, 13, 1), (48, 20, 1), (30, 33, 3), (24, 49, 1), (8, 2, 1)])
def test_scan_of_any_number_of_states_keeps_an_infinity(C, S, G, T, dtype):
    """Numbers of states that fill no whole registers: the rest of them take no part."""
    for what in ("x", "dout", "state", "dt"):
        a, dout, ds = rising(T, 2, C, S, G, dtype, True, True)
        a["z"] = a["z"].abs() + 0.25
        if what == "state":
            a["state"][1, 5] = float("inf")
        else:
            (dout if what == "dout" else a[what])[2, 1, 5] = float("inf")
        check_infinite(a, dout, ds)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("past", [-8, 0, 8, 1])
def test_scan_of_steps_far_apart(past, dtype):
    """Steps as far apart as a chunk's places fit 32 bits, and farther: the same bits as from tensors without gaps, and within the bounds."""
    T, N, C, S = 9, 2, 64, 16
    a, dout, ds = scan_inputs(T, N, C, S, 1, dtype)
    step = 2 ** 28 // dtype.itemsize + past
    buf = torch.zeros((T - 1) * step + N * (3 * C + 2 * S), dtype=dtype, device="cuda")
    view = buf.as_strided((T, N, 3 * C + 2 * S), (step, 3 * C + 2 * S, 1))
    view.normal_(generator=torch.Generator(device="cuda").manual_seed(1))
    x, dt, z, B, Ct = view.split((C, C, C, S, S), -1)
    far = {**a, "x": x, "dt": dt, "z": z, "B": B.unsqueeze(2), "C": Ct.unsqueeze(2)}
    y, last, got = check_scan(far, dout, ds)
    y2, last2, got2 = check_scan({n: v.contiguous() for n, v in far.items()}, dout, ds)
    assert torch.equal(y, y2) and torch.equal(last, last2) and all(torch.equal(g, got2[n]) for n, g in got.items())


# ---------------------------------------------------------------- the gradients' norm
def parameters_of(*grads):
    ps = [torch.zeros_like(g, requires_grad=True) for g in grads]
    for p, g in zip(ps, grads):
        p.grad = g
    return ps


DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]


@pytest.mark.parametrize("device", DEVICES)
def test_clipping_refuses_shared_elements(device):
    """Gradients that share an element are refused before anything is scaled, on either device."""
    n = lambda *s: torch.randn(s, generator=torch.Generator().manual_seed(0)).to(device)   # noqa: E731
    flat, wide, cube = n(64), n(6, 40), n(5, 6, 8)
    for buf, parts in ((flat, (flat[:40], flat[30:])), (wide, (wide[:, :6], wide[:, 5:])), (wide, (wide, wide[2:3, 7])), (wide, (wide[:4], wide[3])),
                       (flat, (flat[::2], flat[10:20])), (flat, (flat[::2], flat[::3])), (cube, (cube[:, :3, 2:5], cube[:, 2:, 4:])), (wide, (wide.t(), wide[1:3, 39:])),
                       (flat, (flat[:1], flat[1:], flat[5]))):
        before = buf.clone()
        with pytest.raises(ValueError, match="share"):
            clip_gradients(parameters_of(*parts), 0.1)
        assert torch.equal(buf, before)
        want = torch.cat([p.flatten() for p in parts]).double().norm()      # (the norm alone changes nothing: whatever it is given)
        assert abs(gradient_norm(parameters_of(*parts)).double() - want) <= 2.0 ** -23 * want


def test_elements_shared_or_not_by_enumeration():
    """Random views of one buffer: boxes of its own grid are told exactly; where one takes every second row, what is said not to share never does."""
    rng, base = random.Random(1), torch.zeros(4, 5, 6, 7)
    for _ in range(3000):
        views, boxes = [], True
        for _ in range(2):
            v = base
            for d in range(4):
                lo = rng.randrange(v.shape[d])
                v = v.narrow(d, lo, rng.randint(1, v.shape[d] - lo))
            if rng.random() < 0.3:
                v, boxes = v[:, :, ::2], False
            if rng.random() < 0.3:
                v = v.select(rng.randrange(4), 0)
            if rng.random() < 0.3:
                v = v.transpose(0, -1)
            views.append(v)
        at = [torch.zeros(base.numel(), dtype=torch.bool) for _ in views]
        for a, v in zip(at, views):
            a.as_strided(v.shape, v.stride(), v.storage_offset()).fill_(True)
        shared, said = bool((at[0] & at[1]).any()), _share_elements(*views)
        assert said == shared or said and not boxes


@pytest.mark.parametrize("device", DEVICES)
def test_clipping_takes_views_that_lie_between_one_another(device):
    """Views of one buffer that share no element, wherever they lie: their values are scaled once, the rest of the buffer is left."""
    n = lambda *s: torch.randn(s, generator=torch.Generator().manual_seed(0)).to(device)   # noqa: E731
    def parts_of(k):
        if k < 4:
            w = n(30, 40)
            return w, ((w[:, :5], w[:, 5:]), (w[:, 20:], w[1:, :10], w[0, :4]), (w[::2], w[1::2], w[0:0]), (w.t()[3], w[:, 4:30:5], w[2:9, :3]))[k]
        if k < 6:
            c = n(4, 6, 8)
            return c, ((c[:, :3, 2:5], c[:, 3:, 4:], c[1:3, 0:2, :2]), (c[..., 0], c[..., 1:].transpose(0, 2), ))[k - 4]
        f = n(64)
        return f, ((f[::2], f[1::2]), (f[::3], f[1::3], f[2::3], f[:0]), (f[0], f[1:30], f[30:31], f[40:]))[k - 6]

    for k in range(9):
        buf, parts = parts_of(k)
        mine = torch.zeros_like(buf)
        for p in parts:                                      # (which elements of the buffer are in a part)
            mine.as_strided(p.shape, p.stride(), p.storage_offset()).add_(1.0)
        assert mine.max() == 1.0 and len(parts) > 1
        before, want = buf.double(), torch.cat([p.flatten() for p in parts]).double().norm()
        norm = clip_gradients(parameters_of(*parts), 0.5, eps=0.0)
        assert abs(norm.double() - want) <= 2.0 ** -23 * want
        after = torch.where(mine > 0, before * (0.5 / want), before)
        assert ((buf.double() - after).abs() <= 2.0 ** -22 * after.abs()).all(), k


def test_clipping_float64_on_cpu():
    """Gradients in float64 are scaled by a factor in float64: a division, a sum and a product, 2^-53 each, and the norm's own 2^-52."""
    g = torch.randn(1000, generator=torch.Generator().manual_seed(2), dtype=torch.float64)
    half = torch.randn(50, generator=torch.Generator().manual_seed(3))
    ps = parameters_of(g.clone(), half.clone())
    norm = torch.cat([g, half.double()]).norm()
    assert torch.allclose(clip_gradients(ps, 0.5).double(), norm, rtol=2.0 ** -24)
    by = 0.5 / (norm + 1e-6)
    assert ((ps[0].grad - g * by).abs() <= 2.0 ** -50 * (g * by).abs()).all()
    assert ((ps[1].grad.double() - half.double() * by).abs() <= 2.0 ** -22 * half.double().abs() * by).all()


# ---------------------------------------------------------------- what follows a call
@pytest.mark.gpu
def test_what_torch_transforms_takes_torch_operations():
    """Forward-mode tangents, vmap, functional gradients, a dispatch mode and tracing see the operations (a kernel called by address would pass them by);
    the results are the kernels'. Float32 on both sides: a few hundred roundings of 2^-24 a value."""
    import torch.autograd.forward_ad as fwd
    from torch.utils.flop_counter import FlopCounterMode
    a, dout, _ = scan_inputs(6, 3, 8, 4, 2, torch.float32)
    x, w, b, start, state, dy, _ = conv_inputs(6, 3, 8, 4, torch.float32)
    scan = lambda v: state_scan(**{**a, "x": v})[0]          # noqa: E731
    conv = lambda v: causal_conv_act(v, w, b, start, state)[0]   # noqa: E731
    step = {n: v[0] if n in ("x", "dt", "B", "C", "z", "start") else v for n, v in a.items()}
    near = lambda p, q: torch.allclose(p, q, rtol=1e-4, atol=1e-4)   # noqa: E731
    g = torch.Generator(device="cuda").manual_seed(3)
    for f, at, back in ((scan, a["x"], dout), (conv, x, dy)):
        y, u = f(at), torch.randn(at.shape, generator=g, device="cuda")
        leaf = at.clone().requires_grad_()
        (grad,) = torch.autograd.grad(f(leaf), leaf, back)
        with fwd.dual_level():
            primal, tangent = fwd.unpack_dual(f(fwd.make_dual(at, u)))
        assert near(primal, y) and tangent is not None
        assert near((tangent * back).sum() / 100, (grad * u).sum() / 100)      # (one sum of 144 products of size 1 to 10, either way)
        many = torch.stack([at, 0.5 * at, -at])
        assert near(torch.func.vmap(f)(many), torch.stack([f(v) for v in many]))
        assert near(torch.func.grad(lambda v: (f(v) * back).sum())(at), grad)
        with FlopCounterMode(display=False):
            assert near(f(at), y)
        assert near(torch.jit.trace(f, at, check_trace=False)(0.5 * at), f(0.5 * at))
    states = torch.stack([a["state"], 2 * a["state"]])
    windows = torch.stack([state, 2 * state])
    want = [[t.clone() for t in ts] for ts in (states, windows)]
    ys = [[state_scan_step(**{**step, "state": s}) for s in want[0]], [causal_conv_act_step(x[0], w, b, s, start[0]) for s in want[1]]]
    got = torch.func.vmap(lambda s: state_scan_step(**{**step, "state": s}))(states), torch.func.vmap(lambda s: causal_conv_act_step(x[0], w, b, s, start[0]))(windows)
    for y, e, s, m in zip(got, ys, (states, windows), want):
        assert near(y, torch.stack(e)) and near(s, torch.stack(m))
    old = [torch.randn(40, generator=g, device="cuda") for _ in range(3)]
    ps = parameters_of(*(o.clone() for o in old))
    with FlopCounterMode(display=False):
        norm = clip_gradients(ps, 0.5)
    assert near(norm, torch.cat(old).norm()) and all(near(p.grad, o * (0.5 / norm)) for p, o in zip(ps, old))


@pytest.mark.parametrize("device", DEVICES)
def test_group_norm_relu_at_zero(device):
    """Where relu's argument is 0 (a group without spread, no bias), its slope is 0 on either device."""
    x = torch.ones(3, 8, device=device)
    w, b = torch.ones(8, device=device, requires_grad=True), torch.zeros(8, device=device, requires_grad=True)
    y = group_norm_act(x, 2, w, b, act="relu")
    assert (y == 0).all() and all((g == 0).all() for g in torch.autograd.grad(y, (w, b), torch.ones_like(y)))


@pytest.mark.parametrize("device", DEVICES)
def test_what_torch_transforms_of_attention_and_group_norm(device):
    """The same for the operators of the memory that decays by constants, and their step."""
    import torch.autograd.forward_ad as fwd
    g = torch.Generator().manual_seed(4)
    n = lambda *s: torch.randn(s, generator=g).to(device)    # noqa: E731
    q, k, v, state = n(6, 3, 2, 8), n(6, 3, 2, 8), n(6, 3, 2, 5), n(3, 2, 8, 5)
    decay, start = torch.tensor([0.9, 0.99], device=device), torch.zeros(6, 3, dtype=torch.bool, device=device)
    start[2, 1] = True
    w, b = n(8), n(8)
    attend = lambda t: linear_attention(t, k, v, decay, start, state)[0]    # noqa: E731
    norm = lambda t: group_norm_act(t, 2, w, b, act="silu")  # noqa: E731
    near = lambda p, r: torch.allclose(p, r, rtol=1e-4, atol=1e-4)   # noqa: E731
    for f, at in ((attend, q), (norm, n(4, 8, 3))):
        y, u = f(at), n(*at.shape)
        back, leaf = n(*y.shape), at.clone().requires_grad_()
        (grad,) = torch.autograd.grad(f(leaf), leaf, back)
        with fwd.dual_level():
            primal, tangent = fwd.unpack_dual(f(fwd.make_dual(at, u)))
        assert near(primal, y) and near((tangent * back).sum() / 100, (grad * u).sum() / 100)
        many = torch.stack([at, 0.5 * at, -at])
        assert near(torch.func.vmap(f)(many), torch.stack([f(t) for t in many]))
        assert near(torch.func.grad(lambda t: (f(t) * back).sum())(at), grad)
        assert near(torch.jit.trace(f, at, check_trace=False)(0.5 * at), f(0.5 * at))
    states = torch.stack([state, 2 * state])
    want = [s.clone() for s in states]
    ys = [linear_attention_step(q[0], k[0], v[0], decay, s, start[0]) for s in want]
    got = torch.func.vmap(lambda s: linear_attention_step(q[0], k[0], v[0], decay, s, start[0]))(states)
    assert near(got, torch.stack(ys)) and near(states, torch.stack(want))
