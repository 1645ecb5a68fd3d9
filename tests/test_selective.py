"""The operators of a memory that selects (fast_mario_env_amd.memory: causal_conv_act, state_scan and their single steps) and of the gradients'
norm (fast_mario_env_amd.rollout: gradient_norm, clip_gradients), against their definitions in float64 written out here.

Tolerances, with e = 2^-24, half a step of float32. `size` is the same sum over absolute values. A sum of n rounded terms is within n e
size. A step size d = softplus(r): r is one sum, exp(-|r|) has |r| e from its argument, the series and a reciprocal a few e, and d's error is at most
r's times sigmoid / softplus <= 1: (2 |r| + 8) e, under 40 e for |r| <= 16. Its error moves a decay exp(E) by 40 e |E| exp(E) <= 15 e however
long the memory; each step's exponential and product add 3 e. silu and its slope: (|z| + 6) e. So outputs and states are within
(3 T + S + 64) e size, gradients, which go through the steps twice and sum over a group's channels, (6 T + 2 S + C / G + 160) e, those of
parameters, which sum over all steps and envs, T N e more. A bf16 result is rounded once: 2^-8 of its value on top."""
import ctypes
import os

import pytest
import torch

from fast_mario_env_amd import _native, memory
from fast_mario_env_amd.memory import causal_conv_act, causal_conv_act_step, state_scan, state_scan_step
from fast_mario_env_amd.rollout import clip_gradients, gradient_norm

E32 = 2.0 ** -24
DTYPES = [torch.float32, torch.bfloat16]


# ---------------------------------------------------------------- the definitions, in float64
def act64(p, act):
    s = torch.sigmoid(p)
    if act == "silu":
        return p * s, s * (1 + p * (1 - s))
    return (p.clamp(min=0), (p > 0).double()) if act == "relu" else (p, torch.ones_like(p))


def conv64(x, w, b, start, state, act, dy=None, dstate=None, size=False):
    """y and the state, then dx, dw, db and dstate where dy is given; size: the same over absolute values."""
    a = (lambda t: t.double().abs()) if size else (lambda t: t.double())
    (T, N, C), K = x.shape, w.shape[1]
    st = x.new_zeros(N, K - 1, C) if state is None else state
    every = torch.cat([st.transpose(0, 1), x])
    p64 = torch.zeros(T, N, C, dtype=torch.float64, device=x.device) if b is None else b.double().expand(T, N, C).clone()
    sums = p64.abs()
    alive = torch.ones(T, N, K, dtype=torch.bool, device=x.device)      # whether step t sees the input j steps before it
    for t in range(T):
        for j in range(1, K):
            alive[t, :, j] = alive[t, :, j - 1] & ~(start[t - j + 1] if start is not None and t - j + 1 >= 0 else torch.zeros(N, dtype=torch.bool, device=x.device))
    for j in range(K):
        term = torch.where(alive[:, :, j, None], every[K - 1 - j:K - 1 - j + T].double(), 0.0) * w[:, K - 1 - j].double()
        p64, sums = p64 + term, sums + term.abs()
    y, slope = act64(p64, act)
    if size:
        y = 1.1 * sums + y.abs() * (1 + p64.abs())
    last = torch.stack([torch.where((alive_after(start, T, j, N, x.device))[:, None], every[T + K - 1 - j].double(), 0.0) for j in range(K - 1, 0, -1)], 1) \
        if K > 1 else torch.zeros(N, 0, C, dtype=torch.float64, device=x.device)
    if dy is None:
        return y, last
    # slope's own error: its change with p is at most 0.5
    dp = a(dy) * (slope.abs() * (2 + p64.abs()) + 0.5 * sums if size else slope)
    d = torch.zeros(T + K - 1, N, C, dtype=torch.float64, device=x.device)
    dw = torch.zeros(C, K, dtype=torch.float64, device=x.device)
    for j in range(K):
        keep = alive[:, :, j, None]
        d[K - 1 - j:K - 1 - j + T] += torch.where(keep, dp * a(w)[:, K - 1 - j], 0.0)
        dw[:, K - 1 - j] = torch.where(keep, dp * a(every[K - 1 - j:K - 1 - j + T]), 0.0).sum((0, 1))
    if dstate is not None:
        for j in range(1, K):
            d[T + K - 1 - j] += torch.where(alive_after(start, T, j, N, x.device)[:, None], a(dstate[:, K - 1 - j]), 0.0)
    return y, last, d[K - 1:], dw, dp.sum((0, 1)), d[:K - 1].transpose(0, 1)


def alive_after(start, T, j, N, device):
    """Whether the episode after the last step holds the input j steps before its end."""
    if start is None:
        return torch.ones(N, dtype=torch.bool, device=device)
    return ~start[max(0, T - j + 1):].any(0)


def scan64(x, dt, A, B, C, D, z, bias, start, state, dout=None, dstate=None, size=False):
    """y and the state, then the gradients by name where dout is given; size: the same over absolute values (of all but the decays)."""
    a = (lambda t: t.double().abs()) if size else (lambda t: t.double())
    T, N, ch = x.shape
    rep, S = ch // B.shape[2], A.shape[1]
    wide = lambda t: a(t).repeat_interleave(rep, 1)   # noqa: E731
    raw = dt.double() + (0.0 if bias is None else bias.double())
    d = torch.where(raw > 30, raw, torch.log1p(torch.exp(raw.clamp(max=30))))
    zero = torch.zeros(N, ch, S, dtype=torch.float64, device=x.device)
    h = zero if state is None else a(state)
    cut = lambda t: torch.zeros(N, 1, 1, dtype=torch.bool, device=x.device) if start is None else start[t][:, None, None]   # noqa: E731
    before, hs, ys = [], [], []
    for t in range(T):
        before.append(torch.where(cut(t), 0.0, h))
        h = torch.where(cut(t), 0.0, torch.exp(d[t][..., None] * A.double()) * h) + (d[t] * a(x[t]))[..., None] * wide(B[t])
        y = (wide(C[t]) * h).sum(-1)
        ys.append(y if D is None else y + a(D) * a(x[t]))
        hs.append(h)
    y = torch.stack(ys) if T else torch.zeros(x.shape, dtype=torch.float64, device=x.device)
    gate = slope = None
    if z is not None:
        gate, slope = act64(z.double(), "silu")
        if size:   # the slope s + z s (1 - s) is a sum too, which crosses 0 at z = -1.28: its size is s + |z| s (1 - s), never less than its value
            s, az = torch.sigmoid(z.double()), z.double().abs()
            gate, slope = gate.abs() * (1 + az / 8), s * (1 + az * (1 - s)) * (1 + az / 8)
    out = y if z is None else y * gate
    if dout is None:
        return out, h
    g = dict(dx=torch.zeros_like(y), ddt=torch.zeros_like(y), dB=torch.zeros(B.shape, dtype=torch.float64, device=x.device))
    g["dC"], dA = torch.zeros_like(g["dB"]), torch.zeros(A.shape, dtype=torch.float64, device=x.device)
    if z is not None:
        g["dz"] = a(dout) * y * slope
    dy = a(dout) if z is None else a(dout) * gate
    Q = zero if dstate is None else a(dstate)
    group = lambda v: v.view(N, -1, rep, S).sum(2)   # noqa: E731
    for t in reversed(range(T)):
        R = Q + wide(C[t]) * dy[t][..., None]
        u = d[t] * a(x[t])
        g["dC"][t], g["dB"][t] = group(hs[t] * dy[t][..., None]), group(R * u[..., None])
        du = (R * wide(B[t])).sum(-1)
        Q = torch.where(cut(t), 0.0, R * torch.exp(d[t][..., None] * A.double()))
        q = Q * before[t]
        g["dx"][t] = du * d[t] + (0.0 if D is None else a(D) * dy[t])
        g["ddt"][t] = (du * a(x[t]) + (q * a(A)).sum(-1)) * torch.sigmoid(raw[t])
        dA += (q * d[t][..., None]).sum(0)
    g.update(dA=dA, dbias=g["ddt"].sum((0, 1)), dstate=Q)
    if D is not None:
        g["dD"] = (dy * a(x)).sum((0, 1))
    return out, h, g


# ---------------------------------------------------------------- comparisons
def near(got, want, size, rel, what):
    """Each element within rel of the sum of absolute values behind it, and one rounding of a bf16 result."""
    assert got.shape == want.shape, what
    assert torch.isfinite(got).all(), what
    bound = rel * size + 1e-30
    if got.dtype == torch.bfloat16:
        bound = bound + 2.0 ** -8 * (want.abs() + bound)
    d = (got.double() - want).abs()
    assert (d <= bound).all(), (what, (d / bound).max().item())


def conv_inputs(T, N, C, K, dtype, seed=0, starts=0.1, state=True, bias=True, device="cuda"):
    g = torch.Generator().manual_seed(seed)
    n = lambda *s: torch.randn(s, generator=g)   # noqa: E731
    x, dy, st, ds = (n(*s).to(dtype).to(device) for s in ((T, N, C), (T, N, C), (N, K - 1, C), (N, K - 1, C)))
    w, b = (n(C, K) / K ** 0.5).to(device), (0.3 * n(C)).to(device)
    start = (torch.rand(T, N, generator=g) < starts).to(device) if starts is not None else None
    return x, w, b if bias else None, start, st if state else None, dy, ds


def check_conv(x, w, b, start, state, dy, ds, act="silu"):
    K, (T, N, C) = w.shape[1], x.shape
    leaves = {n: t.detach().requires_grad_() for n, t in (("x", x), ("w", w), ("b", b), ("state", state)) if t is not None}
    y, last = causal_conv_act(leaves["x"], leaves["w"], leaves.get("b"), start, leaves.get("state"), act=act)
    assert y.dtype == last.dtype == x.dtype
    with torch.no_grad():
        again = causal_conv_act(x, w, b, start, state, act=act)
        assert torch.equal(again[0], y) and torch.equal(again[1], last)
    outs, back = ((y, last), (dy, ds)) if K > 1 else ((y,), (dy,))
    got = dict(zip(leaves, torch.autograd.grad(outs, list(leaves.values()), back, allow_unused=K == 1)))
    want, size = (conv64(x, w, b, start, state, act, dy, ds, size=z) for z in (False, True))
    few = (2 * K + 16) * E32
    near(y.detach(), want[0], size[0], few, "y")
    assert torch.equal(last.detach().double(), want[1])
    for name, i, rel in (("x", 2, 2 * few), ("w", 3, 2 * few + T * N * E32), ("b", 4, 2 * few + T * N * E32), ("state", 5, 2 * few)):
        if name in got and not (name == "state" and K == 1):
            assert got[name].dtype == leaves[name].dtype
            near(got[name], want[i], size[i], rel, name)
    return y.detach(), last.detach(), got


def scan_inputs(T, N, C, S, G, dtype, seed=0, starts=0.1, state=True, D=True, z=True, bias=True, device="cuda"):
    g = torch.Generator().manual_seed(seed)
    n = lambda *s: torch.randn(s, generator=g)   # noqa: E731
    t = lambda v: v.to(dtype).to(device)         # noqa: E731
    a = dict(x=t(n(T, N, C)), dt=t(n(T, N, C)), A=-(torch.rand(C, S, generator=g) * torch.arange(1, S + 1)).to(device), B=t(n(T, N, G, S)), C=t(n(T, N, G, S)),
             D=n(C).to(device) if D else None, z=t(n(T, N, C)) if z else None, dt_bias=(n(C) - 2.0).to(device) if bias else None,
             start=(torch.rand(T, N, generator=g) < starts).to(device) if starts is not None else None, state=n(N, C, S).to(device) if state else None)
    return a, t(n(T, N, C)), n(N, C, S).to(device)


_NAMES = dict(x="dx", dt="ddt", A="dA", B="dB", C="dC", D="dD", z="dz", dt_bias="dbias", state="dstate")


def scan_tolerances(T, N, C, S, G):
    few, grads = (3 * T + S + 64) * E32, (6 * T + 2 * S + C // G + 160) * E32
    return few, {n: grads + (T * N * E32 if n in ("A", "D", "dt_bias") else 0.0) for n in _NAMES}


def check_scan(a, dout, ds):
    T, N, C = a["x"].shape
    S, G = a["A"].shape[1], a["B"].shape[2]
    leaves = {n: a[n].detach().requires_grad_() for n in _NAMES if a[n] is not None}
    y, last = state_scan(**{**a, **leaves})
    assert y.dtype == a["x"].dtype and last.dtype == torch.float32
    with torch.no_grad():
        again = state_scan(**a)
        assert torch.equal(again[0], y) and torch.equal(again[1], last)
    got = dict(zip(leaves, torch.autograd.grad((y, last), list(leaves.values()), (dout, ds))))
    order = [a[n] for n in ("x", "dt", "A", "B", "C", "D", "z", "dt_bias", "start", "state")]
    want, size = (scan64(*order, dout, ds, size=s) for s in (False, True))
    few, rel = scan_tolerances(T, N, C, S, G)
    near(y.detach(), want[0], size[0], few, "y")
    near(last.detach(), want[1], size[1], few, "state")
    for name, g in got.items():
        assert g.dtype == leaves[name].dtype
        near(g, want[2][_NAMES[name]], size[2][_NAMES[name]], rel[name], name)
    return y.detach(), last.detach(), got


# ---------------------------------------------------------------- without a GPU
@pytest.mark.parametrize("T,N,C,K", [(1, 1, 1, 1), (7, 3, 5, 4), (2, 2, 4, 8), (20, 2, 3, 2)])
@pytest.mark.parametrize("act", ["none", "relu", "silu"])
def test_cpu_convolution_is_the_definition(T, N, C, K, act):
    check_conv(*conv_inputs(T, N, C, K, torch.float32, device="cpu"), act=act)
    check_conv(*conv_inputs(T, N, C, K, torch.float32, starts=None, state=K == 1, bias=False, device="cpu"), act=act)
    x, w, b, start, state, _, _ = conv_inputs(T, N, C, K, torch.float32, seed=1, starts=0.4, device="cpu")
    y, last = causal_conv_act(x, w, b, start, state, act)
    s = state.clone()
    for t in range(T):
        assert torch.allclose(causal_conv_act_step(x[t], w, b, s, start[t], act), y[t], atol=1e-6)
    assert torch.equal(s, last)


@pytest.mark.parametrize("T,N,C,S,G", [(1, 1, 1, 1, 1), (7, 3, 6, 5, 3), (20, 2, 8, 16, 2)])
def test_cpu_scan_is_the_recurrence(T, N, C, S, G):
    check_scan(*scan_inputs(T, N, C, S, G, torch.float32, device="cpu"))
    check_scan(*scan_inputs(T, N, C, S, G, torch.float32, starts=None, state=False, D=False, z=False, bias=False, device="cpu"))
    a, _, _ = scan_inputs(T, N, C, S, G, torch.float32, seed=1, starts=0.4, device="cpu")
    y, last = state_scan(**a)
    h = a["state"].clone()
    for t in range(T):
        step = {n: v[t] if n in ("x", "dt", "B", "C", "z", "start") else v for n, v in a.items()}
        assert torch.allclose(state_scan_step(**{**step, "state": h}), y[t], atol=1e-5)
    assert torch.allclose(h, last, atol=1e-5)


def test_oracle_gradients_are_differences():
    """conv64's and scan64's gradients against central differences in float64 (truncation h^2, rounding 2^-53 / h)."""
    g = torch.Generator().manual_seed(3)
    n = lambda *s: torch.randn(s, generator=g, dtype=torch.float64)   # noqa: E731
    T, N, C, S, G, K = 9, 2, 6, 3, 2, 4
    start = torch.rand(T, N, generator=g) < 0.3
    do, ds = n(T, N, C), n(N, C, S)
    x = dict(x=n(T, N, C), dt=n(T, N, C), A=-n(C, S).abs(), B=n(T, N, G, S), C=n(T, N, G, S), D=n(C), z=n(T, N, C), bias=n(C), state=n(N, C, S))
    run = lambda v, *back: scan64(*(v[k] for k in ("x", "dt", "A", "B", "C", "D", "z", "bias")), start, v["state"], *back)   # noqa: E731
    grads = run(x, do, ds)[2]
    names = dict(x="dx", dt="ddt", A="dA", B="dB", C="dC", D="dD", z="dz", bias="dbias", state="dstate")
    cases = [(x, lambda v: sum((p * q).sum() for p, q in zip(run(v), (do, ds))), {k: grads[names[k]] for k in x})]
    cx, cds = dict(x=n(T, N, C), w=n(C, K), b=n(C), state=n(N, K - 1, C)), n(N, K - 1, C)
    conv = lambda v, *back: conv64(v["x"], v["w"], v["b"], start, v["state"], "silu", *back)   # noqa: E731
    cases.append((cx, lambda v: sum((p * q).sum() for p, q in zip(conv(v), (do, cds))), dict(zip(("x", "w", "b", "state"), conv(cx, do, cds)[2:]))))
    for at, loss, grad in cases:
        for k, d in grad.items():
            u, h = n(*at[k].shape), 1e-5
            diff = (loss({**at, k: at[k] + h * u}) - loss({**at, k: at[k] - h * u})) / (2 * h)
            assert abs(diff - (d * u).sum()) < 1e-6 * (1 + (d * u).abs().sum()), k


def test_refusals():
    x, w, b, start, state, _, _ = conv_inputs(4, 3, 6, 4, torch.float32, device="cpu")
    ok = dict(x=x, weight=w, bias=b, start=start, state=state)
    for change in [dict(x=x.half()), dict(x=x[0]), dict(weight=w[:5]), dict(weight=torch.zeros(6, 9)), dict(weight=w[:, :0]), dict(weight=w.long()),
                   dict(bias=b[:5]), dict(start=start[:2]), dict(start=start.float()), dict(state=state.bfloat16()), dict(state=state[:, :2]), dict(act="tanh")]:
        with pytest.raises(ValueError, match="causal_conv_act"):
            causal_conv_act(**{**ok, **change})
    step = dict(x=x[0], weight=w, bias=b, start=start[0], state=state)
    for change in [dict(x=x), dict(state=None), dict(state=state.transpose(0, 1).contiguous().transpose(0, 1)), dict(x=x[0].clone().requires_grad_()),
                   dict(start=start)]:
        with pytest.raises(ValueError, match="causal_conv_act_step"):
            causal_conv_act_step(**{**step, **change})
    a, _, _ = scan_inputs(4, 3, 6, 5, 2, torch.float32, device="cpu")
    for change in [dict(x=a["x"].half()), dict(dt=a["dt"].bfloat16()), dict(z=a["z"][:2]), dict(A=a["A"][:4]), dict(A=torch.zeros(6, 65)), dict(A=a["A"].long()),
                   dict(B=a["B"][..., :4]), dict(B=a["B"].bfloat16()), dict(B=a["B"][:, :, :1]), dict(B=a["B"].repeat(1, 1, 2, 1), C=a["C"].repeat(1, 1, 2, 1)),
                   dict(D=a["D"][:2]), dict(dt_bias=a["dt_bias"][None]), dict(start=a["start"].float()), dict(state=a["state"].bfloat16()),
                   dict(state=a["state"][:2]), dict(x=a["x"][0])]:
        with pytest.raises(ValueError, match="state_scan"):
            state_scan(**{**a, **change})
    one = {n: v[0] if n in ("x", "dt", "B", "C", "z", "start") else v for n, v in a.items()}
    for change in [dict(x=a["x"]), dict(state=None), dict(state=a["state"].transpose(1, 2).contiguous().transpose(1, 2)), dict(A=a["A"].clone().requires_grad_())]:
        with pytest.raises(ValueError, match="state_scan_step"):
            state_scan_step(**{**one, **change})


def test_gradients_norm_on_cpu_and_refusals():
    g = torch.Generator().manual_seed(0)
    ps = [torch.zeros(s, requires_grad=True) for s in ((3, 4), (), (5,), (0,))]
    for p in ps[:2] + ps[3:]:
        p.grad = torch.randn(p.shape, generator=g)
    want = torch.cat([p.grad.flatten() for p in ps if p.grad is not None]).double().norm()
    old = [None if p.grad is None else p.grad.clone() for p in ps]
    assert torch.allclose(gradient_norm(ps).double(), want, rtol=1e-6) and torch.allclose(gradient_norm(ps + ps).double(), want, rtol=1e-6)
    norm = clip_gradients(iter(ps + ps), 0.5)                # (twice the same: scaled once)
    assert norm.dtype == torch.float32 and torch.allclose(norm.double(), want, rtol=1e-6)
    for p, o in zip(ps, old):
        assert o is None or torch.allclose(p.grad, o * (0.5 / want).float(), rtol=1e-6)
    small = [p.grad.clone() for p in ps if p.grad is not None]
    clip_gradients(ps, 10.0)
    assert all(torch.equal(a, b) for a, b in zip(small, (p.grad for p in ps if p.grad is not None)))
    assert gradient_norm([]) == 0 and clip_gradients(ps[2], 1.0) == 0
    for bad in (dict(max_norm=-1.0), dict(max_norm=float("nan")), dict(max_norm=1.0, eps=-1.0)):
        with pytest.raises(ValueError, match="clip_gradients"):
            clip_gradients(ps, **bad)
    p = torch.zeros(3, 4, requires_grad=True)
    p.grad = torch.ones(3, 1).expand(3, 4)
    with pytest.raises(ValueError, match="expanded"):
        clip_gradients([p], 1.0)
    p = torch.zeros(3, requires_grad=True)
    p.grad = torch.ones(3).to_sparse()
    with pytest.raises(ValueError, match="dense"):
        gradient_norm([p])


class Rows(ctypes.Structure):
    _fields_ = [("p", ctypes.c_void_p), ("st", ctypes.c_int64), ("sn", ctypes.c_int64), ("sh", ctypes.c_int64)]


class CConv(ctypes.Structure):
    _fields_ = [(n, ctypes.c_int32) for n in ("dtype", "act", "C", "K")] + [(n, ctypes.c_int64) for n in ("T", "N")] + [(n, Rows) for n in ("x", "y")] + \
               [(n, ctypes.c_void_p) for n in ("weight", "bias", "start", "state", "state_out", "work")] + [(n, Rows) for n in ("dy", "dx")] + \
               [(n, ctypes.c_void_p) for n in ("dstate_out", "dstate", "dweight", "dbias")]


class CScan(ctypes.Structure):
    _fields_ = [(n, ctypes.c_int32) for n in ("dtype", "C", "S", "G")] + [(n, ctypes.c_int64) for n in ("T", "N")] + \
               [(n, Rows) for n in ("x", "dt", "z", "Bt", "Ct", "out")] + [(n, ctypes.c_void_p) for n in ("A", "D", "dt_bias", "start", "state", "state_out", "saved", "work")] + \
               [(n, Rows) for n in ("dout", "dx", "ddt", "dz", "dB", "dC")] + [(n, ctypes.c_void_p) for n in ("dstate_out", "dstate", "dA", "dD", "ddt_bias")]


class CTensor(ctypes.Structure):
    _fields_ = [("p", ctypes.c_void_p), ("n", ctypes.c_int64), ("dtype", ctypes.c_int32), ("reserved", ctypes.c_int32)]


def test_c_entry_points_check_sizes_and_pointers():
    """Before any device: sizes; then pointers that are not the GPU's (or no GPU at all). Nothing is queued."""
    L = ctypes.CDLL(os.path.join(os.path.dirname(_native.__file__), "libmario_ops.so"))
    L.mo_last_error.restype = ctypes.c_char_p
    for f in ("mo_conv_work", "mo_scan_work", "mo_scan_saved", "mo_gradient_work"):
        getattr(L, f).restype = ctypes.c_int64
    host = (ctypes.c_float * 4096)()
    at = ctypes.addressof(host)
    row = Rows(at, 8, 8, 8)
    for bad in (dict(C=0), dict(K=0), dict(K=9), dict(dtype=2), dict(act=3), dict(T=-1), dict(N=-1), dict(C=(1 << 20) + 1), dict(N=1 << 31), dict(dweight=at)):
        c = CConv(**{**dict(dtype=0, act=2, C=8, K=4, T=2, N=2, x=row, y=row, dy=row, dx=row, weight=at), **bad})
        for f in ("mo_conv", "mo_conv_backward", "mo_conv_step"):
            assert getattr(L, f)(ctypes.byref(c), None) == -1 and L.mo_last_error(), (f, bad)
        assert L.mo_conv_work(ctypes.byref(c)) == -1
    for bad in (dict(C=0), dict(S=0), dict(S=65), dict(G=3), dict(G=0), dict(dtype=7), dict(T=-1), dict(N=1 << 31)):
        c = CScan(**{**dict(dtype=0, C=8, S=4, G=1, T=2, N=2, x=row, dt=row, Bt=row, Ct=row, out=row, A=at, state_out=at), **bad})
        for f in ("mo_scan", "mo_scan_backward", "mo_scan_step"):
            assert getattr(L, f)(ctypes.byref(c), None) == -1 and L.mo_last_error(), (f, bad)
        assert L.mo_scan_work(ctypes.byref(c), 0) == L.mo_scan_work(ctypes.byref(c), 1) == L.mo_scan_saved(ctypes.byref(c)) == -1
    for T in (0, 2):                                         # sums over no steps are made too, and need their rows
        assert L.mo_conv_work(ctypes.byref(CConv(dtype=0, act=2, C=8, K=4, T=T, N=2, x=row, y=row, dy=row, dx=row, weight=at, dweight=at, dbias=at))) >= 2 * 5 * 8 * 4
        assert L.mo_scan_work(ctypes.byref(CScan(dtype=0, C=8, S=4, G=1, T=T, N=2, x=row, dt=row, Bt=row, Ct=row, out=row, A=at, state_out=at)), 1) >= 2 * 6 * 8 * 4
    c = CConv(dtype=0, act=2, C=8, K=4, T=2, N=2, x=row, y=row, dy=row, dx=row, weight=at)       # pageable host memory
    s = CScan(dtype=0, C=8, S=4, G=1, T=2, N=2, x=row, dt=row, Bt=row, Ct=row, out=row, A=at, state_out=at)
    for f, a in (("mo_conv", c), ("mo_conv_backward", c), ("mo_conv_step", c), ("mo_scan", s), ("mo_scan_backward", s), ("mo_scan_step", s)):
        assert getattr(L, f)(ctypes.byref(a), None) == -1 and L.mo_last_error(), f
    L.mo_gradient_norm.argtypes = [ctypes.c_void_p, ctypes.c_int64, ctypes.c_int, ctypes.c_float, ctypes.c_float] + [ctypes.c_void_p] * 3
    t = CTensor(at, 8, 0, 0)
    for args in ((ctypes.addressof(t), -1, 1, 1.0, 0.0), (None, 1, 1, 1.0, 0.0), (ctypes.addressof(t), 1, 1, -1.0, 0.0), (ctypes.addressof(t), 1, 1, 1.0, 0.0)):
        assert L.mo_gradient_norm(*args, at, at, None) == -1 and L.mo_last_error()
    t.dtype = 5
    assert L.mo_gradient_norm(ctypes.addressof(t), 1, 0, 0.0, 0.0, at, at, None) == -1 and b"MO_F32" in L.mo_last_error()
    assert L.mo_gradient_work(-1) == -1 and L.mo_gradient_work(500) > 0
    assert all(hasattr(_native.ops(), f) for f in ("conv", "conv_step", "scan", "scan_step", "gradient_norm"))


# ---------------------------------------------------------------- causal convolution on the GPU
@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("T", [1, 2, 3, 15, 16, 17, 40, 100])
@pytest.mark.parametrize("C,K", [(64, 4), (8, 2), (40, 8), (5, 3), (513, 4), (1, 1), (256, 1), (24, 5), (16, 6), (7, 7)])
def test_convolution_vs_float64(T, C, K, dtype):
    check_conv(*conv_inputs(T, 3, C, K, dtype, seed=T))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("starts", [None, 0.0, 0.5, 1.0])
def test_convolution_episode_starts(starts, dtype):
    check_conv(*conv_inputs(70, 5, 32, 4, dtype, starts=starts))
    check_conv(*conv_inputs(70, 5, 32, 4, dtype, starts=starts, state=False, bias=False), act="none")
    x, w, b, start, state, dy, ds = conv_inputs(33, 4, 16, 4, dtype, starts=starts)
    z = conv64(x, w, b, start, state, "none")[0]
    assert z.abs().min() > 1e-6                              # relu's gradient jumps at zero
    check_conv(x, w, b, start, state, dy, ds, act="relu")


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("T,N,C", [(3000, 1, 16), (700, 300, 24), (5, 9000, 8), (2, 3, 8200)])
def test_convolution_long_and_many(T, N, C, dtype):
    check_conv(*conv_inputs(T, N, C, 4, dtype, starts=0.02))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
def test_convolution_takes_views(dtype):
    T, N, C, K = 20, 3, 32, 4
    _, w, b, start, state, dy, ds = conv_inputs(T, N, C, K, dtype)
    g = torch.Generator().manual_seed(9)
    n = lambda *s: torch.randn(s, generator=g).to(dtype).cuda()   # noqa: E731
    part = n(T, N, 2 * C).chunk(2, -1)[1]
    for x in (part, n(N, T, C).transpose(0, 1), n(T, N, 2 * C)[..., ::2], n(T, N, C + 1)[..., 1:], n(T, 1, C).expand(T, N, C), n(T, N, 1).expand(T, N, C),
              n(T * N * C + 1)[1:].view(T, N, C)):
        check_conv(x, w, b, start, state, dy, ds)
        check_conv(x, w.t().contiguous().t(), b, start.t().contiguous().t(), state, dy.transpose(0, 1).contiguous().transpose(0, 1), ds)
    one = n(T, 1, C).requires_grad_()
    y, last = causal_conv_act(one.expand(T, N, C), w, b, start, state)
    (got,) = torch.autograd.grad((y, last), one, (dy, ds))
    want, size = (conv64(one.detach().expand(T, N, C), w, b, start, state, "silu", dy, ds, size=s)[2].sum(1, keepdim=True) for s in (False, True))
    near(got.float(), want, size, 2.0 ** -7 if dtype == torch.bfloat16 else 2.0 ** -18, "shared")   # (a bf16 gradient an env, summed in bf16)
    half = w.bfloat16().requires_grad_()
    y, _ = causal_conv_act(part, half, b.double(), start, state)
    assert torch.equal(y.detach(), causal_conv_act(part, half.detach().float(), b, start, state)[0])
    assert torch.autograd.grad(y, half, dy)[0].dtype == torch.bfloat16
    (dw,) = torch.autograd.grad(causal_conv_act(part, w.requires_grad_(), b, start, state)[0].sum(), w)   # an expanded gradient
    want, size = (conv64(part, w.detach(), b, start, state, "silu", torch.ones_like(dy), size=s)[3] for s in (False, True))
    near(dw, want, size, (40 + T * N) * E32, "dw")


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
def test_convolution_what_is_not_finite_stays_in_its_episode(bad, dtype):
    T, N, C, K = 50, 2, 16, 4
    x, w, b, _, state, dy, ds = conv_inputs(T, N, C, K, dtype)
    start = torch.zeros(T, N, dtype=torch.bool, device="cuda")
    start[10], start[30] = True, True

    def run(x, state):
        leaf = x.detach().requires_grad_()
        y, last = causal_conv_act(leaf, w, b, start, state)
        return [y.detach(), torch.autograd.grad((y, last), leaf, (dy, ds))[0]]

    clean = run(x, state)
    for where, hit in ((-1, slice(0, 10)), (8, slice(0, 10)), (20, slice(10, 30)), (29, slice(10, 30)), (45, slice(30, T))):
        y, s = x.clone(), state.clone()
        if where < 0:
            s.fill_(bad)
        else:
            y[where] = bad
        for a, c in zip(run(y, s), clean):
            for part in (slice(0, hit.start), slice(hit.stop, T)):
                assert torch.equal(a[part], c[part]), where


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("N,C,K", [(1, 1, 1), (3, 64, 4), (700, 40, 4), (5, 33, 2), (2, 16, 8), (4, 7, 3), (66003, 64, 4), (66001, 32, 7)])
def test_convolution_step_is_the_convolution(N, C, K, dtype):
    T = 6
    x, w, b, start, state, _, _ = conv_inputs(T, N, C, K, dtype, starts=0.4)
    y, last = causal_conv_act(x, w, b, start, state)
    s = state.clone()
    s[start[0]] = float("nan")                               # what a starting env saw before is never looked at
    for t in range(T):
        assert torch.equal(causal_conv_act_step(x[t], w, b, s, start[t]), y[t])
    assert torch.equal(s, last)
    s = state.clone()
    assert torch.equal(causal_conv_act_step(torch.stack([x[0], x[1]], -1)[..., 1], w, None, s, act="none"), causal_conv_act(x[1:2], w, None, None, state, "none")[0][0])


# ---------------------------------------------------------------- state space scan on the GPU
@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("T", [1, 2, 7, 8, 9, 17, 64, 130])
@pytest.mark.parametrize("C,S,G", [(64, 16, 1), (512, 16, 1), (40, 4, 2), (200, 24, 2), (1, 1, 1), (65, 13, 1), (128, 64, 4), (30, 33, 3), (96, 8, 1), (70, 48, 1)])
def test_scan_vs_float64(T, C, S, G, dtype):
    check_scan(*scan_inputs(T, 3, C, S, G, dtype, seed=T))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("D", [False, True])
@pytest.mark.parametrize("z", [False, True])
@pytest.mark.parametrize("bias,state", [(False, True), (True, False)])
def test_scan_parts_that_are_not_there(D, z, bias, state, dtype):
    check_scan(*scan_inputs(21, 3, 72, 16, 1, dtype, D=D, z=z, bias=bias, state=state))
    check_scan(*scan_inputs(21, 3, 72, 20, 2, dtype, D=D, z=z, bias=bias, state=state))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("starts", [None, 0.0, 0.5, 1.0])
def test_scan_episode_starts(starts, dtype):
    check_scan(*scan_inputs(70, 4, 64, 16, 1, dtype, starts=starts))
    check_scan(*scan_inputs(300, 2, 32, 8, 1, dtype, starts=starts))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("T,N,C,S,G", [(1999, 2, 64, 16, 1), (4001, 1, 16, 4, 2), (600, 5, 200, 24, 2), (2048, 1, 130, 64, 1)])
def test_scan_long_and_few(T, N, C, S, G, dtype):
    """Few sequences, cut over their length; episodes that span many cuts and ones within one."""
    a, dout, ds = scan_inputs(T, N, C, S, G, dtype, starts=0.002)
    a["start"][T // 2:T // 2 + 3] = True
    check_scan(a, dout, ds)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("T,N,C,S,G", [(20, 1500, 70, 16, 1), (9, 5000, 8, 4, 2)])
def test_scan_many(T, N, C, S, G, dtype):
    check_scan(*scan_inputs(T, N, C, S, G, dtype))


@pytest.mark.gpu
@pytest.mark.parametrize("T", [12, 3000])
def test_scan_step_sizes_small_and_large(T):
    """Step sizes from 1e-6 (memories of the whole length) to over 30 (nothing is kept), decays of exactly one among them."""
    a, dout, ds = scan_inputs(T, 2, 64, 16, 1, torch.float32, starts=0.001)
    a["dt_bias"] = torch.linspace(-13.0, 14.0, 64, device="cuda")
    a["dt"] = a["dt"].clamp(-2, 2)
    a["A"][:, 0] = 0.0
    check_scan(a, dout, ds)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
def test_scan_takes_views(dtype):
    T, N, C, S, G = 20, 3, 32, 16, 2
    a, dout, ds = scan_inputs(T, N, C, S, G, dtype)
    g = torch.Generator().manual_seed(9)
    n = lambda *s: torch.randn(s, generator=g).to(dtype).cuda()   # noqa: E731
    x, z, rest = n(T, N, 3 * C + 2 * G * S).split((C, C, C + 2 * G * S), -1)
    dt, B, Ct = rest.split((C, G * S, G * S), -1)
    fused = dict(x=x, z=z, dt=dt, B=B.unflatten(-1, (G, S)), C=Ct.unflatten(-1, (G, S)))
    swapped = dict(x=n(N, T, C).transpose(0, 1), dt=n(C, T, N).permute(1, 2, 0), B=n(N, G, T, S).permute(2, 0, 1, 3), C=n(T, N, S, G).transpose(2, 3))
    shared = dict(x=n(T, 1, C).expand(T, N, C), z=n(T, N, 1).expand(T, N, C), B=n(T, N, 1, S).expand(T, N, G, S), C=n(1, N, G, S).expand(T, N, G, S))
    odd = dict(x=n(T, N, C + 1)[..., 1:], B=n(T, N, G, S + 1)[..., 1:], C=n(T * N * G * S + 1)[1:].view(T, N, G, S))
    for change in (fused, swapped, shared, odd):
        b = {**a, **change}
        check_scan(b, dout, ds)
        check_scan({**b, "A": a["A"].t().contiguous().t(), "state": a["state"].transpose(0, 1).contiguous().transpose(0, 1)},
                   dout.transpose(0, 1).contiguous().transpose(0, 1), ds.transpose(0, 2).contiguous().transpose(0, 2))
    one = n(T, N, 1, S).requires_grad_()
    y, last = state_scan(**{**a, "B": one.expand(T, N, G, S)})
    (got,) = torch.autograd.grad((y, last), one, (dout, ds))
    order = [{**a, "B": one.detach().expand(T, N, G, S)}[k] for k in ("x", "dt", "A", "B", "C", "D", "z", "dt_bias", "start", "state")]
    want, size = (scan64(*order, dout, ds, size=s)[2]["dB"].sum(2, keepdim=True) for s in (False, True))
    near(got.float(), want, size, 2.0 ** -7 if dtype == torch.bfloat16 else 2.0 ** -15, "shared")   # (a bf16 gradient a group, summed in bf16)
    half = a["A"].bfloat16().requires_grad_()
    y, _ = state_scan(**{**a, "A": half})
    assert torch.equal(y.detach(), state_scan(**{**a, "A": half.detach().float()})[0]) and torch.autograd.grad(y, half, dout)[0].dtype == torch.bfloat16


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("T", [50, 600])
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
def test_scan_what_is_not_finite_stays_in_its_episode(bad, T, dtype):
    """A value that is not finite shows in no step and no gradient of a step of another episode."""
    N, C, S = 2, 32, 16
    a, dout, ds = scan_inputs(T, N, C, S, 1, dtype)
    first, last = T // 5, 3 * T // 5
    start = a["start"] = torch.zeros(T, N, dtype=torch.bool, device="cuda")
    start[first], start[last] = True, True

    def run(a, dout):
        leaves = {n: a[n].detach().requires_grad_() for n in ("x", "dt", "B", "C", "z")}
        y, end = state_scan(**{**a, **leaves})
        return [y.detach()] + list(torch.autograd.grad((y, end), list(leaves.values()), (dout, ds)))

    clean = run(a, dout)
    for where in (0, first - 1, first, last - 1, last, T - 1):
        hit = slice(0, first) if where < first else slice(first, last) if where < last else slice(last, T)
        for name in ("x", "dt", "B", "C", "z", "dout", "state"):
            b, do = dict(a), dout
            if name == "dout":
                do = dout.clone()
                do[where] = bad
            elif name == "state":
                if where:
                    continue
                b["state"] = torch.full_like(a["state"], bad)
            else:
                b[name] = a[name].clone()
                b[name][where] = bad
            for got, want in zip(run(b, do), clean):
                for part in (slice(0, hit.start), slice(hit.stop, T)):
                    assert torch.equal(got[part], want[part]), (where, name)
            if name == "x":
                assert not torch.isfinite(run(b, do)[0][where]).any() and torch.isfinite(run(b, do)[0][hit.start:where].float()).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("T,N,C,S,G", [(20, 3, 1100, 16, 1), (17, 3, 300, 64, 1), (9, 2, 1300, 40, 2), (40, 300, 520, 4, 1), (3, 2, 9000, 16, 1)])
def test_scan_more_channels_than_a_workgroup_has(T, N, C, S, G, dtype):
    """Sums over a group's channels that several workgroups leave, and more envs than are taken at a time."""
    check_scan(*scan_inputs(T, N, C, S, G, dtype))


@pytest.mark.gpu
def test_two_graphs_and_two_streams_at_once():
    """Two captured passes, replayed in turn and on two streams at once, each against its eager result."""
    def make(seed):
        a, dout, ds = scan_inputs(200, 3, 64, 16, 1, torch.bfloat16, seed=seed)
        leaves = [a[n].requires_grad_() for n in _NAMES]

        def work():
            y, last = state_scan(**a)
            return [y.detach(), last.detach(), *torch.autograd.grad((y, last), leaves, (dout, ds))]
        return work

    works, graphs, held = [make(s) for s in (1, 2)], [], []
    want = [[t.clone() for t in w()] for w in works]
    torch.cuda.synchronize()
    for w in works:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            held.append(w())
        graphs.append(graph)
    streams = [torch.cuda.Stream() for _ in works]
    for i in range(4):
        for g, s in zip(graphs, streams):
            if i % 2:
                g.replay()
            else:
                with torch.cuda.stream(s):
                    g.replay()
        torch.cuda.synchronize()
        for h, e in zip(held, want):
            assert all(torch.equal(x, y) for x, y in zip(h, e)), i


@pytest.mark.gpu
def test_scan_empty():
    for T, N in ((0, 3), (4, 0), (0, 0)):
        a, dout, ds = scan_inputs(T, N, 8, 4, 1, torch.bfloat16)
        y, last, got = check_scan_empty(a, dout, ds)
        assert y.shape == a["x"].shape and torch.equal(last, a["state"])
        assert all(g.shape == a[n].shape for n, g in got.items()) and torch.equal(got["state"], ds)
        assert all((got[n] == 0).all() for n in ("A", "D", "dt_bias"))
        x, w, b, start, state, dy, dl = conv_inputs(T, N, 8, 4, torch.bfloat16)
        leaves = [t.requires_grad_() for t in (x, w, b, state)]
        y, last = causal_conv_act(x, w, b, start, state)
        gx, gw, gb, gs = torch.autograd.grad((y, last), leaves, (dy, dl))
        assert torch.equal(last, state) and torch.equal(gs, dl) and gx.shape == x.shape and (gw == 0).all() and (gb == 0).all()
    a, _, _ = scan_inputs(1, 0, 8, 4, 1, torch.float32)
    one = {n: v[0] if n in ("x", "dt", "B", "C", "z", "start") else v for n, v in a.items()}
    assert state_scan_step(**one).shape == (0, 8)


def check_scan_empty(a, dout, ds):
    leaves = {n: a[n].detach().requires_grad_() for n in _NAMES}
    y, last = state_scan(**{**a, **leaves})
    return y.detach(), last.detach(), dict(zip(leaves, torch.autograd.grad((y, last), list(leaves.values()), (dout, ds))))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("N,C,S,G", [(1, 1, 1, 1), (3, 64, 16, 1), (70, 512, 16, 1), (5, 40, 4, 2), (5, 200, 24, 2), (4, 65, 13, 1), (2, 128, 64, 4), (3, 30, 33, 3),
                                     (2, 24, 8, 1), (2, 7, 5, 7)])
def test_scan_step_is_the_recurrence(N, C, S, G, dtype):
    T = 6
    a, _, _ = scan_inputs(T, N, C, S, G, dtype, starts=0.4)
    order = [a[n] for n in ("x", "dt", "A", "B", "C", "D", "z", "dt_bias", "start", "state")]
    (want, last), (size, lsize) = (scan64(*order, size=s) for s in (False, True))
    h = a["state"].clone()
    h[a["start"][0]] = float("nan")                          # what a starting env remembers is never looked at
    few, _ = scan_tolerances(T, N, C, S, G)
    for t in range(T):
        step = {n: v[t] if n in ("x", "dt", "B", "C", "z", "start") else v for n, v in a.items()}
        near(state_scan_step(**{**step, "state": h}), want[t], size[t], few, "y")
    near(h, last, lsize, few, "state")
    h0 = a["state"].clone()                                  # strided inputs, nothing that may be missing
    views = {n: torch.stack([a[n][0], a[n][1]], -1)[..., 1] for n in ("x", "dt", "B", "C")}
    got = state_scan_step(**views, A=a["A"], state=h0)
    one = [a[n][1:2] for n in ("x", "dt")] + [a["A"]] + [a[n][1:2] for n in ("B", "C")] + [None, None, None, None, a["state"]]
    (want, last), (size, lsize) = (scan64(*one, size=s) for s in (False, True))
    near(got, want[0], size[0], few, "y")
    near(h0, last, lsize, few, "state")


@pytest.mark.gpu
def test_scan_gradients_are_differences():
    """Differences of the kernel's own float32 forward pass, summed in float64: cubic terms h^2, rounding 2^-24 sqrt(values) / h."""
    a, dout, ds = scan_inputs(40, 3, 64, 16, 2, torch.float32)
    leaves = {n: a[n].detach().requires_grad_() for n in _NAMES}
    y, last = state_scan(**{**a, **leaves})
    grads = dict(zip(leaves, torch.autograd.grad((y, last), list(leaves.values()), (dout, ds))))
    g = torch.Generator().manual_seed(5)
    with torch.no_grad():
        for n, grad in grads.items():
            u, h = torch.randn(a[n].shape, generator=g).cuda() * (0.1 if n == "A" else 1.0), 2.0 ** -7
            side = []
            for s in (h, -h):
                y, last = state_scan(**{**a, n: a[n] + s * u})
                side.append((y.double() * dout).sum() + (last.double() * ds).sum())
            want = (grad.double() * u).sum()
            scale = (grad.double() * u).norm()
            noise = E32 * 32 * ((y.double() * dout).norm() + (last.double() * ds).norm()) / h
            assert abs((side[0] - side[1]) / (2 * h) - want) <= noise + 8 * h * h * scale * 8, (n, (side[0] - side[1]) / (2 * h), want)


# ---------------------------------------------------------------- streams, graphs, autograd
@pytest.mark.gpu
@pytest.mark.parametrize("T,N,C", [(128, 6, 128), (1500, 1, 64), (20, 900, 96)])
def test_same_bits_and_other_streams(T, N, C):
    """The same inputs give the same bits, on another stream and beside other work too."""
    a, dout, ds = scan_inputs(T, N, C, 16, 1, torch.bfloat16)
    cv = conv_inputs(T, N, C, 4, torch.bfloat16)

    def run():
        leaves = [a[n].detach().requires_grad_() for n in _NAMES]
        y, last = state_scan(**{**a, **dict(zip(_NAMES, leaves))})
        x, w, b, s = (cv[i].detach().requires_grad_() for i in (0, 1, 2, 4))
        y2, last2 = causal_conv_act(x, w, b, cv[3], s)
        back = torch.autograd.grad((y, last), leaves, (dout, ds)) + torch.autograd.grad((y2, last2), (x, w, b, s), cv[5:])
        p = [torch.zeros_like(g, requires_grad=True) for g in back]
        for q, g in zip(p, back):
            q.grad = g.clone()
        return [y, last, y2, last2, *back, clip_gradients(p, 1.0), *(q.grad for q in p)]

    first = run()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = [run() for _ in range(3)][-1]
    again = run()
    side.synchronize()
    torch.cuda.synchronize()
    for i, (p, q, r) in enumerate(zip(first, other, again)):
        assert torch.equal(p, q) and torch.equal(p, r), i


@pytest.mark.gpu
def test_differentiable_once_and_who_saved_a_state():
    a, dout, _ = scan_inputs(5, 2, 16, 4, 1, torch.float32)
    x, w, b, start, state, dy, _ = conv_inputs(5, 2, 16, 4, torch.float32)
    x.requires_grad_()
    a["x"].requires_grad_()
    for y, leaf, g in ((state_scan(**a)[0], a["x"], dout), (causal_conv_act(x, w, b, start, state)[0], x, dy)):
        (first,) = torch.autograd.grad(y, leaf, g, create_graph=True)
        assert torch.isfinite(first).all()
        with pytest.raises(RuntimeError, match="once"):
            first.square().sum().backward()
    one = {n: v.detach()[0] if n in ("x", "dt", "B", "C", "z", "start") else v for n, v in a.items()}
    for change in (lambda: state_scan_step(**one), lambda: causal_conv_act_step(x[0].detach(), w, b, state)):
        held = torch.randn_like(a["state"], requires_grad=True), torch.randn_like(state, requires_grad=True)
        loss = (held[0] * a["state"]).sum() + (held[1] * state).sum()
        with torch.no_grad():
            change()
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            loss.backward()


@pytest.mark.gpu
def test_under_graph_capture():
    """Captured once, replayed on new inputs with eager work in between, every replay against the eager result: forward, steps, gradients by
    autograd.grad, the norm and clipping."""
    a, dout, ds = scan_inputs(300, 2, 64, 16, 1, torch.bfloat16)
    x, w, b, start, state, dy, dl = conv_inputs(300, 2, 64, 4, torch.bfloat16)
    leaves = [a[n].requires_grad_() for n in _NAMES] + [x.requires_grad_(), w.requires_grad_()]
    h, win = a["state"].detach().clone(), state.clone()
    p = torch.zeros(5000, device="cuda", requires_grad=True)
    p.grad = torch.zeros(5000, device="cuda")
    fresh = torch.zeros(5000, device="cuda")

    def work():
        y, last = state_scan(**a)
        y2, last2 = causal_conv_act(x, w, b, start, state)
        back = torch.autograd.grad((y, last, y2, last2), leaves, (dout, ds, dy, dl))
        with torch.no_grad():
            one = {n: v[0] if n in ("x", "dt", "B", "C", "z", "start") else v for n, v in a.items()}
            s1 = state_scan_step(**{**one, "state": h})
            s2 = causal_conv_act_step(x[0], w, b, win, start[0])
            p.grad.copy_(fresh)
            norm = clip_gradients([p], 0.5)
        return [y.detach(), last.detach(), y2.detach(), last2.detach(), *back, s1, s2, norm, gradient_norm([p]), p.grad, h, win]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        work()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = work()
    for i in range(4):
        g = torch.Generator(device="cuda").manual_seed(i)
        with torch.no_grad():
            for t in (a["x"], a["dt"], a["B"], a["C"], a["z"], a["state"], x, state, dout, dy, fresh):
                t.normal_(generator=g)
        h.copy_(a["state"].detach())
        win.copy_(state)
        want = [t.clone() for t in work()]
        h.copy_(a["state"].detach())
        win.copy_(state)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        for k, (got, e) in enumerate(zip(held, want)):
            assert torch.equal(got, e), (i, k)


@pytest.mark.gpu
def test_past_32_bits():
    """Steps 2^30 elements apart in one buffer: offsets past 2^31 elements and 2^32 bytes."""
    T, N, C, S = 3, 2, 64, 16
    a, dout, ds = scan_inputs(T, N, C, S, 1, torch.bfloat16)
    buf = torch.zeros(2 * 2 ** 30 + 4096, dtype=torch.bfloat16, device="cuda")
    view = buf.as_strided((T, N, 3 * C + 2 * S), (2 ** 30, 3 * C + 2 * S, 1))
    view.normal_(generator=torch.Generator(device="cuda").manual_seed(1))
    x, dt, z, B, Ct = view.split((C, C, C, S, S), -1)
    check_scan({**a, "x": x, "dt": dt, "z": z, "B": B.unsqueeze(2), "C": Ct.unsqueeze(2)}, dout, ds)
    _, w, b, start, state, dy, dl = conv_inputs(T, N, C, 4, torch.bfloat16)
    check_conv(x, w, b, start, state, dy, dl)


@pytest.mark.gpu
def test_step_past_32_bits():
    """States of over 2^32 bytes and 2^31 values; the last envs are compared."""
    N, C, S = 264000, 512, 16
    x, B = torch.randn(N, C, device="cuda").bfloat16(), torch.randn(N, 1, S, device="cuda").bfloat16()
    A = -torch.rand(C, S, device="cuda")
    state = torch.empty(N, C, S, device="cuda").normal_()
    tail = state[-3:].clone()
    y = state_scan_step(x, x, A, B, B, state)
    last3 = [x[None, -3:], x[None, -3:], A, B[None, -3:], B[None, -3:], None, None, None, None, tail]
    (want, last), (size, lsize) = (scan64(*last3, size=s) for s in (False, True))
    few, _ = scan_tolerances(1, 3, C, S, 1)
    near(y[-3:], want[0], size[0], few, "y")
    near(state[-3:], last, lsize, few, "state")


# ---------------------------------------------------------------- the gradients' norm on the GPU
def with_gradients(gs):
    ps = [torch.zeros_like(g, requires_grad=True) for g in gs]
    for p, g in zip(ps, gs):
        p.grad = g
    return ps


def check_clip(gs, max_norm=0.5, eps=1e-6):
    """The factor is rounded once and each value once: 2 e, or the bf16 rounding; the norm once."""
    ps, old = with_gradients(gs), [g.double() for g in gs]
    want = torch.sqrt(sum([g.square().sum() for g in old], torch.zeros((), dtype=torch.float64, device="cuda")))
    n = gradient_norm(ps)
    assert n.dtype == torch.float32 and n.dim() == 0 and abs(n.double() - want) <= 1.01 * E32 * want
    assert all(torch.equal(g.double(), o) for g, o in zip(gs, old))
    assert torch.equal(clip_gradients(ps, max_norm, eps=eps), n)
    by = min(1.0, max_norm / (want.item() + eps))
    for g, o in zip(gs, old):
        rel = 2.0 ** -8 if g.dtype == torch.bfloat16 else E32
        assert ((g.double() - o * by).abs() <= (rel + 1.1 * E32) * (o * by).abs() + 1e-40).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("sizes", [[1], [7], [16384], [16385], [100000, 3, 0, 1], [5000] * 300, [3_000_001], [17] * 129, [0], list(range(1, 260))])
def test_clipping_vs_float64(sizes, dtype):
    g = torch.Generator(device="cuda").manual_seed(len(sizes))
    check_clip([torch.randn(n, generator=g, device="cuda").to(dtype) for n in sizes])
    check_clip([torch.randn(n, generator=g, device="cuda").to(dtype) for n in sizes], max_norm=1e9)     # (nothing to clip)
    flat = torch.randn(sum(sizes) + 1, generator=g, device="cuda").to(dtype)
    before = flat[:1].clone()
    check_clip(list(flat[1:].split(sizes)))                  # views that begin anywhere
    assert torch.equal(flat[:1], before)


@pytest.mark.gpu
def test_clipping_layouts_and_values():
    g = torch.Generator(device="cuda").manual_seed(1)
    n = lambda *s: torch.randn(s, generator=g, device="cuda")   # noqa: E731
    wide = n(30, 40)
    edge = wide[:, 5:].clone()
    check_clip([n(8, 4, 3, 3).to(memory_format=torch.channels_last), n(5, 7).t(), wide[:, :5], n(6, 2).bfloat16(), n()])
    assert torch.equal(wide[:, 5:], edge)
    check_clip([n(1000) * 1e25, n(10)])                      # squares past float32's range
    check_clip([n(1000) * 1e-30], max_norm=1e-32, eps=0.0)
    for bad, left in ((float("nan"), torch.isnan), (float("inf"), lambda t: (t == 0) | torch.isnan(t))):
        gs = [n(100), n(50)]
        gs[1][3] = bad
        norm = clip_gradients(with_gradients(gs), 0.5)
        assert not torch.isfinite(norm) and left(gs[0]).all() and torch.isnan(gs[1][3])
    same = n(64)
    with pytest.raises(ValueError, match="share"):
        clip_gradients(with_gradients([same[:40], same[30:]]), 0.5)
    twice = with_gradients([n(64)])[0]
    want = twice.grad.double().norm()
    assert abs(clip_gradients([twice, twice], 0.1).double() - want) <= 2 * E32 * want and abs(twice.grad.double().norm() - 0.1) < 1e-5
    with pytest.raises(ValueError, match="float32 or bf16"):
        clip_gradients(with_gradients([n(4).half()]), 1.0)
    with pytest.raises(ValueError, match="one device"):
        clip_gradients(with_gradients([n(4)]) + with_gradients([torch.ones(3)]), 1.0)
    held = n(10)
    loss = (torch.randn(10, device="cuda", requires_grad=True) * held).sum()
    clip_gradients(with_gradients([held]), 1e-3)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()


@pytest.mark.gpu
def test_norm_past_32_bits():
    g = torch.ones(2 ** 32 + 12345, dtype=torch.bfloat16, device="cuda")
    n = gradient_norm(with_gradients([g]))
    want = (2 ** 32 + 12345) ** 0.5
    assert abs(n.item() - want) <= 1.01 * E32 * want
    clip_gradients(with_gradients([g]), want / 4, eps=0.0)
    assert (g[-5:] == 0.25).all() and (g[:5] == 0.25).all() and g[2 ** 31 + 3] == 0.25


# ---------------------------------------------------------------- the network that uses them
def test_scan_net_on_cpu():
    """Steps and the whole sequence agree, memories are cleared at starts, and every parameter gets a gradient."""
    T, N = 5, 3
    net = memory.make_memory_net(device="cpu", memory="scan", states=6, taps=3)
    obs = torch.randint(0, 256, (T, N, 4, 84, 84), dtype=torch.uint8, generator=torch.Generator().manual_seed(0))
    start = torch.zeros(T, N, dtype=torch.bool)
    start[0], start[3, 1] = True, True
    logits, value, last = net(obs, start)
    state = tuple(s + 7.0 for s in net.initial_state(N))     # what a first step's env remembers is not seen
    for t in range(T):
        lg, v = net.step(obs[t], start[t], state)
        assert torch.allclose(lg, logits[t], atol=1e-5) and torch.allclose(v, value[t], atol=1e-4)
    assert all(torch.allclose(a, b, atol=1e-4) for a, b in zip(state, last))
    alone, _, _ = net(obs[3:, 1:2], None, None)              # an episode from its start on
    assert torch.allclose(alone, logits[3:, 1:2], atol=1e-5)
    (logits.sum() + value.sum()).backward()
    assert all(p.grad is not None and torch.isfinite(p.grad).all() for p in net.parameters())
    want = torch.cat([p.grad.flatten() for p in net.parameters()]).double().norm()
    assert torch.allclose(clip_gradients(net.parameters(), 0.5).double(), want, rtol=1e-6)
    for bad in (dict(memory="lstm"), dict(memory="scan", states=65), dict(memory="scan", taps=0)):
        with pytest.raises(ValueError, match="make_memory_net"):
            memory.make_memory_net(device="cpu", **bad)


@pytest.mark.gpu
def test_scan_net_gradients_as_on_cpu():
    """The network's loss and gradients on the GPU (bf16 trunk and memory) against the same weights on the CPU in float32."""
    T, N = 40, 3
    g = torch.Generator().manual_seed(1)
    obs = torch.randint(0, 256, (T, N, 4, 84, 84), dtype=torch.uint8, generator=g)
    start = torch.rand(T, N, generator=g) < 0.05
    nets = [memory.make_memory_net(seed=3, device=d, memory="scan") for d in ("cpu", "cuda")]
    assert all(torch.equal(a.cpu(), b.cpu()) for a, b in zip(nets[0].parameters(), nets[1].parameters()))
    grads = []
    for net, dev in zip(nets, ("cpu", "cuda")):
        h = torch.Generator().manual_seed(2)
        state = [torch.randn(s.shape, generator=h).to(s.dtype).to(dev).requires_grad_() for s in nets[1].initial_state(N)]
        if dev == "cpu":
            state[0] = state[0].detach().float().requires_grad_()
        logits, value, last = net(obs.to(dev), start.to(dev), tuple(state))
        (torch.log_softmax(logits, -1)[..., 2].mean() + value.square().mean() + 1e-3 * last[1].square().mean()).backward()
        grads.append([p.grad.float().cpu() for p in net.parameters()] + [s.grad.float().cpu() for s in state])
    for name, a, b in zip([n for n, _ in nets[0].named_parameters()] + ["window", "state"], *grads):
        # a bf16 network of about twelve layers: each rounds by 2^-9 at most, forth and back
        assert (a - b).norm() <= 0.1 * a.norm() + 1e-6, (name, ((a - b).norm() / a.norm()).item())


@pytest.mark.gpu
def test_rollout_with_a_selective_memory_is_computed_again():
    """A rollout under the network: its stored log-probabilities and values come out again from the stored sequence, episodes
    ending inside; a second rollout goes on from the memories of the first; a training step of the example changes every parameter."""
    from build_roms import rom_path
    from fast_mario_env_amd import HipVecEnv
    from fast_mario_env_amd.rollout import Rollout
    import importlib.util
    spec = importlib.util.spec_from_file_location("memory_policy", os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples", "memory_policy.py"))
    example = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(example)
    n, T = 24, 20
    env = HipVecEnv("1-1", n, seed=0, sticky=0.25, noop_max=30, max_steps=13, maxpool=True, rom=open(rom_path("vanilla"), "rb").read())
    env.reset()
    net = memory.make_memory_net(seed=0, memory="scan")
    ro = Rollout(env, net, T=T, seed=3)
    for _ in range(2):
        before = [m.clone() for m in ro.memory]
        ro.collect()
        assert all(torch.equal(a, b) for a, b in zip(ro.memory0, before))
        with torch.no_grad():
            logits, value, last = net(*ro.sequence(torch.arange(n, device="cuda")))
        logp = torch.log_softmax(logits, -1).gather(-1, ro.act[..., None]).squeeze(-1)
        # (the convolutions of another batch size may take other kernels: bf16 either way)
        assert torch.allclose(logp, ro.logp, atol=2e-2) and torch.allclose(value, ro.val, atol=0.1, rtol=0.05)
        assert all((a.float() - b.float()).norm() <= 0.03 * a.float().norm() for a, b in zip(last, ro.memory))
        assert ro.start[1:].any()
    with torch.no_grad():                                    # a share of the envs, by index
        part, _, _ = net(*ro.sequence(torch.tensor([5, 2], device="cuda")))
    assert torch.allclose(torch.log_softmax(part, -1), torch.log_softmax(logits[:, [5, 2]], -1), atol=2e-2)
    opt = torch.optim.Adam(net.parameters(), 1e-3)
    old = [p.detach().clone() for p in net.parameters()]
    assert torch.isfinite(example.update(net, opt, ro))
    assert all(not torch.equal(a, b) for a, b in zip(old, net.parameters()))
    assert gradient_norm(net.parameters()) <= 0.5
    env.close()
