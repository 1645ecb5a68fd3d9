"""The operators of a policy with a memory (fast_mario_env_amd.memory): linear attention over rollouts and by single steps, and
group norm with an activation, against their definitions in float64 written out here.

Tolerances. float32: with a the same sums over absolute values, a result of n terms is within about n 2^-24 a of the exact
one; (T + D + E + 16) 2^-23 covers the terms, the decay's powers and the joining of chunks. bf16 results carry three roundings to 8
bits of significand: that of a masked product, that of the state that meets q (the two act on parts of one sum), and the
result's own. A rounding is off by at most 2^-8 of its value and by 2^-9 or less for most values, so three of them seldom reach 3 *
2^-9, which is asked for in norm and, element by element, of the sum of absolute values: tighter than the worst case."""

import ctypes
import os
import re
import struct

import numpy as np
import pytest
import torch

from fast_mario_env_amd import _native, memory
from fast_mario_env_amd.memory import group_norm_act, head_decays, linear_attention, linear_attention_step

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
HALF = 3 * 2.0 ** -9
DTYPES = [torch.float32, torch.bfloat16]


# ---------------------------------------------------------------- the definitions, in float64
def attend64(q, k, v, decay, start, state, scale, dout=None, dstate=None):
    """out and state, then dq, dk, dv and dstate_in where dout is given: step by step."""
    q, k, v, g = q.double(), k.double(), v.double(), decay.double()[:, None, None]
    T, N, H, D = q.shape
    S = torch.zeros(N, H, D, v.shape[-1], dtype=torch.float64, device=q.device) if state is None else state.double()
    cut = torch.zeros(T, N, 1, 1, 1, dtype=torch.bool, device=q.device) if start is None else start[..., None, None, None]
    out, dq = torch.zeros_like(v), torch.zeros_like(q)
    for t in range(T):
        S = torch.where(cut[t], 0.0, g * S) + k[t][..., :, None] * v[t][..., None, :]
        out[t] = (q[t][..., :, None] * S).sum(-2) * scale
        if dout is not None:
            dq[t] = (S * dout[t].double()[..., None, :]).sum(-1) * scale
    if dout is None:
        return out, S
    R = torch.zeros_like(S) if dstate is None else dstate.double()
    dk, dv = torch.zeros_like(k), torch.zeros_like(v)
    for t in reversed(range(T)):
        R = R + scale * q[t][..., :, None] * dout[t].double()[..., None, :]
        dk[t] = (R * v[t][..., None, :]).sum(-1)
        dv[t] = (R * k[t][..., :, None]).sum(-2)
        R = torch.where(cut[t], 0.0, g * R)
    return out, S, dq, dk, dv, R


def norm64(x, groups, w, b, eps, act, dy=None):
    """y, then dx, dw and db where dy is given; channels are dimension 1."""
    B, C = x.shape[:2]
    x3 = x.double().reshape(B, groups, -1)
    mean = x3.mean(-1, keepdim=True)
    r = 1.0 / ((x3 - mean).square().mean(-1, keepdim=True) + eps).sqrt()
    h = ((x3 - mean) * r).reshape(B, C, -1)
    w = torch.ones(C, dtype=torch.float64, device=x.device) if w is None else w.double()
    b = torch.zeros_like(w) if b is None else b.double()
    z = h * w[:, None] + b[:, None]
    s = torch.sigmoid(z)
    y = {"none": z, "relu": z.clamp(min=0), "silu": z * s}[act].reshape(x.shape)
    if dy is None:
        return y
    dz = dy.double().reshape(B, C, -1) * {"none": torch.ones_like(z), "relu": (z > 0).double(), "silu": s * (1 + z * (1 - s))}[act]
    dh = (dz * w[:, None]).reshape(B, groups, -1)
    h3 = h.reshape(B, groups, -1)
    dx = r * (dh - dh.mean(-1, keepdim=True) - h3 * (dh * h3).mean(-1, keepdim=True))
    return y, dx.reshape(x.shape), (dz * h).sum((0, 2)), dz.sum((0, 2))


# ---------------------------------------------------------------- comparisons
def near(got, want, size, rel, what):
    """In norm over everything and over each env and head with enough values to have one; and each element by the sum of
    absolute values behind it."""
    assert got.shape == want.shape and torch.isfinite(got).all(), what
    d = (got.double() - want).abs()
    assert (d <= rel * size + 1e-30).all(), (what, (d / (rel * size + 1e-30)).max().item())
    assert d.norm() <= rel * want.norm() + 1e-30, (what, (d.norm() / want.norm()).item())


def attend_inputs(T, N, H, D, E, dtype, seed=0, starts=0.1, state=True, device="cuda"):
    g = torch.Generator().manual_seed(seed)
    n = lambda *s: torch.randn(s, generator=g).to(dtype).to(device)   # noqa: E731
    q, k, v, do = n(T, N, H, D), n(T, N, H, D), n(T, N, H, E), n(T, N, H, E)
    start = (torch.rand(T, N, generator=g) < starts).to(device) if starts is not None else None
    st = torch.randn(N, H, D, E, generator=g).to(device) if state else None
    ds = torch.randn(N, H, D, E, generator=g).to(device)
    return q, k, v, head_decays(H, device), start, st, do, ds


def check_attend(q, k, v, decay, start, state, do, ds, scale=None, grads=True):
    s = q.shape[-1] ** -0.5 if scale is None else scale
    leaves = [t for t in (q, k, v, state) if t is not None]
    if grads:
        leaves = [t.detach().requires_grad_() for t in leaves]
    args = leaves[:3] + [decay, start] + (leaves[3:] or [None])
    out, last = linear_attention(*args, scale=scale)
    assert out.dtype == q.dtype and last.dtype == torch.float32
    got = [out.detach(), last.detach()]
    if grads:
        dg = torch.autograd.grad((out, last), leaves, (do, ds))
        assert all(a.dtype == b.dtype for a, b in zip(dg, leaves))
        got += list(dg)
    a = lambda t: None if t is None else t.abs()   # noqa: E731
    back = (do, ds) if grads else ()
    want = attend64(q, k, v, decay, start, state, s, *back)
    size = attend64(a(q), a(k), a(v), decay, start, a(state), abs(s), *map(a, back))
    f32 = (q.shape[0] + q.shape[-1] + v.shape[-1] + 16) * 2.0 ** -23
    for x, y, z, name in zip(got, want, size, ("out", "state", "dq", "dk", "dv", "dstate")):
        near(x, y, z, HALF if x.dtype == torch.bfloat16 else f32, name)
    return got


def norm_inputs(B, C, sp, dtype, seed=0, device="cuda", offset=0.0):
    g = torch.Generator().manual_seed(seed)
    n = lambda *s: torch.randn(s, generator=g)   # noqa: E731
    back = lambda t: t.to(dtype).to(device).movedim(-1, 1)   # noqa: E731
    x, dy = back(n(B, *sp, C) + n(C) + offset), back(n(B, *sp, C))
    return x, (1 + 0.2 * n(C)).to(device), (0.3 * n(C)).to(device), dy


def check_norm(x, groups, w, b, act, dy, eps=1e-5):
    leaves = [t.detach().requires_grad_() for t in (x, w, b) if t is not None]
    y = group_norm_act(leaves[0], groups, *leaves[1:], eps=eps, act=act)
    assert y.dtype == x.dtype and y.shape == x.shape
    with torch.no_grad():
        assert torch.equal(group_norm_act(x, groups, w, b, eps=eps, act=act), y.detach())
    got = [y.detach()] + list(torch.autograd.grad(y, leaves, dy))
    want = norm64(x, groups, w, b, eps, act, dy)
    cells = x.numel() // x.shape[0] // groups
    # h is off by 2^-24 of |x - mean| r and of |mean| r, and sums of n terms by a few 2^-24 sqrt(n) where they are joined in trees
    x3 = x.double().reshape(x.shape[0], groups, -1)
    big = 1.0 + (x3.mean(-1).abs() / (x3.var(-1, unbiased=False) + eps).sqrt()).max().item()
    f32 = 2.0 ** -24 * (32 + 4 * cells ** 0.5) * big
    for i, (a, e) in enumerate(zip(got, want)):
        assert torch.isfinite(a).all()
        rel = 2.0 ** -8 if a.dtype == torch.bfloat16 else f32   # one rounding to bf16, and the sums'
        size = e.norm() + (0 if i < 2 else f32 * x.numel() ** 0.5)
        assert (a.double() - e).norm() <= rel * size, (i, ((a.double() - e).norm() / size).item(), rel)
    return got


# ---------------------------------------------------------------- without a GPU
@pytest.mark.parametrize("T,N,H,D,E", [(1, 1, 1, 1, 1), (7, 3, 2, 5, 4), (20, 2, 3, 8, 16)])
def test_cpu_attention_is_the_recurrence(T, N, H, D, E):
    check_attend(*attend_inputs(T, N, H, D, E, torch.float32, device="cpu"))
    q, k, v, decay, start, state, _, _ = attend_inputs(T, N, H, D, E, torch.float32, seed=1, device="cpu")
    out, last = linear_attention(q, k, v, decay, start, state)
    S = state.clone()
    for t in range(T):
        assert torch.allclose(linear_attention_step(q[t], k[t], v[t], decay, S, start[t]), out[t], atol=1e-5)
    assert torch.allclose(S, last, atol=1e-5)


@pytest.mark.parametrize("act", ["none", "relu", "silu"])
def test_cpu_norm_is_the_formula(act):
    check_norm(*(lambda x, w, b, dy: (x, 3, w, b, act, dy))(*norm_inputs(4, 12, (5, 3), torch.float32, device="cpu")))
    ref = torch.nn.functional.group_norm(norm_inputs(4, 12, (5, 3), torch.float32, device="cpu")[0], 3)
    assert torch.allclose(group_norm_act(norm_inputs(4, 12, (5, 3), torch.float32, device="cpu")[0], 3), ref, atol=1e-5)


def test_oracle_gradients_are_differences():
    """attend64's gradients against central differences: the loss is linear in each of q, k, v and the state."""
    g = torch.Generator().manual_seed(3)
    n = lambda *s: torch.randn(s, generator=g, dtype=torch.float64)   # noqa: E731
    T, N, H, D, E = 9, 2, 2, 3, 4
    x = [n(T, N, H, D), n(T, N, H, D), n(T, N, H, E), n(N, H, D, E)]
    decay, start, do, ds = torch.tensor([0.9, 0.3]), torch.rand(T, N, generator=g) < 0.3, n(T, N, H, E), n(N, H, D, E)

    def loss(q, k, v, s):
        out, last = attend64(q, k, v, decay, start, s, 0.7)
        return (out * do).sum() + (last * ds).sum()

    grads = attend64(*x[:3], decay, start, x[3], 0.7, do, ds)[2:]
    for i, grad in enumerate(grads):
        u = n(*x[i].shape)
        up, down = ([t + s * u if j == i else t for j, t in enumerate(x)] for s in (1.0, -1.0))
        assert abs((loss(*up) - loss(*down)) / 2 - (grad * u).sum()) < 1e-9 * (grad * u).abs().sum()


def test_refusals():
    q, k, v, decay, start, state, _, _ = attend_inputs(4, 3, 2, 8, 6, torch.float32, device="cpu")
    bad = [dict(q=q.half(), k=k.half(), v=v.half()), dict(k=k.bfloat16()), dict(k=k[..., :4]), dict(v=v[:2]), dict(q=q[0]),
           dict(decay=decay[:1]), dict(decay=decay.double()), dict(start=start[:2]), dict(start=start.float()),
           dict(state=state.bfloat16()), dict(state=state[:, :, :4]), dict(decay=decay.clone().requires_grad_()),
           dict(q=q.expand(4, 3, 2, 8)[..., :0], k=k[..., :0])]
    for change in bad:
        with pytest.raises(ValueError, match="linear_attention"):
            linear_attention(**{**dict(q=q, k=k, v=v, decay=decay, start=start, state=state), **change})
    wide = torch.zeros(1, 1, 1, 129)
    with pytest.raises(ValueError, match="128"):
        linear_attention(wide, wide, wide, decay[:1])
    step = dict(q=q[0], k=k[0], v=v[0], decay=decay, state=state, start=start[0])
    for change in [dict(q=q), dict(state=state.transpose(0, 1).contiguous().transpose(0, 1)), dict(q=q[0].clone().requires_grad_()),
                   dict(start=start), dict(v=v[0].bfloat16())]:
        with pytest.raises(ValueError, match="linear_attention_step"):
            linear_attention_step(**{**step, **change})
    x, w, b, _ = norm_inputs(2, 12, (3, 3), torch.float32, device="cpu")
    for args, kw in [((x, 5, w, b), {}), ((x, 0, w, b), {}), ((x, 3, w), {}), ((x, 3, w[:4], b), {}), ((x.half(), 3, w, b), {}),
                     ((x, 3, w, b), dict(act="tanh")), ((x, 3, w, b), dict(eps=-1.0)), ((x, 3, w, b), dict(eps=float("nan"))),
                     ((x[0, 0, 0], 1), {}), ((x[:, :, :0], 3, w, b), {})]:
        with pytest.raises(ValueError, match="group_norm_act"):
            group_norm_act(*args, **kw)


def test_ops_library_exports_and_checks():
    """libmario_ops.so loads without a GPU, exports what include/mario_ops.h declares (all of which the torch module calls), and
    checks sizes before any device."""
    package = os.path.dirname(_native.__file__)
    names = set(re.findall(r"\b(mo_\w+)\s*\(", open(os.path.join(ROOT, "include", "mario_ops.h")).read()))
    assert len(names) >= 8
    L = ctypes.CDLL(os.path.join(package, "libmario_ops.so"))
    L.mo_last_error.restype = ctypes.c_char_p
    L.mo_attend_work.restype = ctypes.c_int64
    calls = open(os.path.join(ROOT, "fast-mario-env_amd", "csrc", "ops", "torch_ops.cpp")).read()
    for s in names:
        assert hasattr(L, s) and s in calls, s
    attend, norm = struct.Struct("=4i2qf4x" + 4 * "Qqqq" + "6Q" + 4 * "Qqqq" + "2Q"), struct.Struct("=4i2qf4x10Q")   # MoAttend, MoNorm
    a = attend.pack(1, 2, 200, 8, 1, 1, 1.0, *(0,) * 16, *(0,) * 6, *(0,) * 16, 0, 0)      # a head size of 200
    assert L.mo_attend(a, None) == -1 and b"head sizes" in L.mo_last_error()
    assert L.mo_attend_work(a, 0) == -1
    m = norm.pack(1, 0, 10, 3, 1, 1, 1e-5, *(0,) * 10)
    assert L.mo_group_norm(m, None) == -1 and b"groups" in L.mo_last_error()
    host = np.zeros(64, np.float32)
    at = host.ctypes.data
    m = norm.pack(0, 0, 8, 1, 1, 1, 1e-5, at, 0, 0, at, 0, at, 0, 0, 0, 0)
    assert L.mo_group_norm(m, None) == -1 and L.mo_last_error()   # pageable host memory (or no GPU at all)
    assert all(hasattr(_native.ops(), f) for f in ("attend", "attend_step", "group_norm_act"))


# ---------------------------------------------------------------- linear attention on the GPU
@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("T", [1, 2, 31, 32, 33, 64, 65, 130])
@pytest.mark.parametrize("D,E", [(64, 64), (32, 64), (128, 128), (40, 24), (5, 33)])
def test_attention_vs_float64(T, D, E, dtype):
    check_attend(*attend_inputs(T, 3, 2, D, E, dtype, seed=T))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("starts", [None, 0.0, 0.5, 1.0])
def test_attention_episode_starts(starts, dtype):
    check_attend(*attend_inputs(140, 4, 3, 32, 32, dtype, starts=starts))
    check_attend(*attend_inputs(70, 4, 3, 32, 32, dtype, starts=starts, state=False), scale=-0.3)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("T,N,H,D,E", [(1999, 2, 2, 64, 32), (2048, 1, 1, 128, 128), (4001, 1, 3, 16, 16), (513, 5, 2, 96, 64)])
def test_attention_long_and_few(T, N, H, D, E, dtype):
    """Few sequences, long enough to be cut over their length; episodes that span many cuts and ones within one."""
    a = list(attend_inputs(T, N, H, D, E, dtype, starts=0.002))
    a[4][T // 2:T // 2 + 3] = True
    check_attend(*a)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
def test_attention_many(dtype):
    check_attend(*attend_inputs(37, 700, 4, 32, 32, dtype))


@pytest.mark.gpu
@pytest.mark.parametrize("D,E", [(4, 4), (5, 4)])
def test_attention_more_heads_than_a_row_of_blocks(D, E):
    check_attend(*attend_inputs(2, 2 ** 22 + 37, 1, D, E, torch.float32, starts=0.3))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("T,N", [(20000, 1), (4000, 300)])
def test_attention_decays_near_one(T, N, dtype):
    """Nothing is added, so the states decay by g^T and back: a rounding of a factor and of a product a chunk (of 32 steps at
    least) and a segment, however near to one the factor is."""
    q, k, v, _, _, state, do, ds = attend_inputs(T, N, 4, 16, 16, dtype, starts=None)
    decay = torch.tensor([1 - 2.0 ** -20, 0.99999, 0.999, 1.0], device="cuda")
    state.requires_grad_()
    out, last = linear_attention(q, torch.zeros_like(k), v, decay, None, state)
    (dstate,) = torch.autograd.grad((out, last), state, (torch.zeros_like(do), ds))
    f = (decay.double() ** T)[:, None, None]
    for got, want in ((last, f * state.double()), (dstate, f * ds.double())):
        assert ((got.double() - want).abs() <= 2 * (T / 32 + 8) * 2.0 ** -24 * want.abs()).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
def test_attention_decays_zero_and_one(dtype):
    a = list(attend_inputs(150, 2, 4, 32, 32, dtype))
    a[3] = torch.tensor([0.0, 1.0, 0.5, 1e-30], device="cuda")
    check_attend(*a)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
def test_attention_takes_views(dtype):
    """A fused projection's parts, time and envs exchanged, heads shared by expansion, a last dimension that is strided, and
    pointers off a 16-byte boundary; every gradient reaches its own elements."""
    T, N, H, D = 70, 3, 2, 32
    _, _, _, decay, start, state, do, ds = attend_inputs(T, N, H, D, D, dtype)
    g = torch.Generator().manual_seed(9)
    n = lambda *s: torch.randn(s, generator=g).to(dtype).cuda()   # noqa: E731
    fused = n(T, N, 3 * H * D).view(T, N, 3, H, D).unbind(2)
    swapped = [n(N, H, T, D).permute(2, 0, 1, 3) for _ in range(3)]
    shared = [n(T, N, H, D), n(T, N, 1, D).expand(T, N, H, D), n(T, 1, H, D).expand(T, N, H, D)]
    strided = [n(T, N, H, 2 * D)[..., ::2] for _ in range(3)]
    odd = [n(T, N, H, D + 1)[..., 1:] for _ in range(3)]
    shifted = [n(T * N * H * D + 4)[4:].view(T, N, H, D) for _ in range(3)]
    for q, k, v in (fused, swapped, shared, strided, odd, shifted):
        check_attend(q, k, v, decay, start, state, do, ds)
    one = n(T, N, 1, D).requires_grad_()
    q, v = n(T, N, H, D), n(T, N, H, D)
    out, last = linear_attention(q, one.expand(T, N, H, D), v, decay, start, state)
    (got,) = torch.autograd.grad((out, last), one, (do, ds))
    want = attend64(q, one.detach().expand(T, N, H, D), v, decay, start, state, D ** -0.5, do, ds)[3].sum(2, keepdim=True)
    assert (got.double() - want).norm() <= (HALF if dtype == torch.bfloat16 else 1e-5) * 2 * want.norm()
    (got,) = torch.autograd.grad(linear_attention(q, q, v.requires_grad_(), decay, start, state)[0].sum(), v)   # an expanded gradient
    want = attend64(q, q, v.detach(), decay, start, state, D ** -0.5, torch.ones_like(v), None)[4]
    assert (got.double() - want).norm() <= (HALF if dtype == torch.bfloat16 else 1e-5) * want.norm()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
def test_attention_what_is_not_finite_stays_in_its_episode(bad, dtype):
    """A value that is not finite, anywhere in the inputs or the entering state, shows in no step and no gradient of another
    episode, nor in a step before it."""
    T, N, H, D = 150, 2, 1, 32
    for where in (0, 20, 40, 70):
        q, k, v, decay, _, state, do, ds = attend_inputs(T, N, H, D, D, dtype, seed=where)
        start = torch.zeros(T, N, dtype=torch.bool, device="cuda")
        first, last = 10, 50
        start[first], start[last] = True, True
        hit = slice(0, first) if where < first else slice(first, last) if where < last else slice(last, T)
        clean = check_attend(q, k, v, decay, start, state, do, ds)
        for which in range(4):
            x = [t.clone() for t in (q, k, v, do)]
            x[which][where] = bad
            st = state.clone()
            if where < first:
                st.fill_(bad)
            leaves = [t.requires_grad_() for t in x[:3]]
            out, end = linear_attention(*leaves, decay, start, st)
            got = [out.detach()] + list(torch.autograd.grad((out, end), leaves, (x[3], ds)))
            for name, a, c in zip(("out", "dq", "dk", "dv"), got, [clean[0]] + clean[2:5]):
                for s in (slice(0, hit.start), slice(hit.stop, T)):
                    assert torch.equal(a[s], c[s]) or torch.allclose(a[s].float(), c[s].float(), rtol=2e-2, atol=2e-2), (where, which, name)
            assert torch.isfinite(out[hit.start + (where - hit.start):hit.stop].float()).all() == (which == 3 and where >= first)
            before = out[hit.start:where]
            assert where < first or torch.isfinite(before.float()).all()


@pytest.mark.gpu
def test_attention_empty():
    for T, N in ((0, 3), (4, 0), (0, 0)):
        q, k, v, decay, start, state, do, ds = attend_inputs(T, N, 2, 16, 16, torch.bfloat16)
        leaves = [t.requires_grad_() for t in (q, k, v, state)]
        out, last = linear_attention(*leaves[:3], decay, start, leaves[3])
        assert out.shape == v.shape and torch.equal(last, state)
        grads = torch.autograd.grad((out, last), leaves, (do, ds))
        assert [g.shape for g in grads] == [t.shape for t in leaves] and torch.equal(grads[3], ds)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
def test_attention_gradients_are_differences(dtype):
    """Differences of the kernel's own forward pass: the loss is linear in each input, so they have no truncation error."""
    T, N, H, D, E = 90, 3, 2, 64, 32
    q, k, v, decay, start, state, do, ds = attend_inputs(T, N, H, D, E, torch.float32)
    x = [t.requires_grad_() for t in (q, k, v, state)]
    out, last = linear_attention(*x[:3], decay, start, x[3])
    grads = torch.autograd.grad((out, last), x, (do, ds))
    if dtype == torch.bfloat16:   # the bf16 gradients against the float32 ones of the same (rounded) inputs
        y = [t.detach().to(dtype if i < 3 else torch.float32).requires_grad_() for i, t in enumerate(x)]
        x = [t.detach().float().requires_grad_() for t in y]
        out, last = linear_attention(*x[:3], decay, start, x[3])
        do = do.to(dtype).float()
        grads = torch.autograd.grad((out, last), x, (do, ds))
        out, last = linear_attention(*y[:3], decay, start, y[3])
        for a, b in zip(torch.autograd.grad((out, last), y, (do.to(dtype), ds)), grads):
            assert (a.float() - b).norm() <= HALF * b.norm()
        return
    g = torch.Generator().manual_seed(5)
    with torch.no_grad():
        for i, grad in enumerate(grads):
            u = torch.randn(x[i].shape, generator=g).cuda()
            side = []
            for s in (1.0, -1.0):
                y = [t + s * u if j == i else t for j, t in enumerate(x)]
                out, last = linear_attention(*y[:3], decay, start, y[3])
                side.append((out.double() * do).sum() + (last.double() * ds).sum())
            want = (grad.double() * u).sum()
            assert abs((side[0] - side[1]) / 2 - want) <= 1e-5 * (grad.double() * u).norm() * 8, i


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("N,H,D,E", [(1, 1, 1, 1), (3, 2, 64, 64), (70, 8, 64, 64), (5, 3, 32, 128), (5, 2, 128, 32), (9, 1, 128, 128),
                                     (4, 2, 40, 24), (4, 2, 33, 5), (2, 3, 7, 127), (3, 1, 100, 100)])
def test_step_is_the_recurrence(N, H, D, E, dtype):
    q, k, v, decay, start, state, _, _ = attend_inputs(6, N, H, D, E, dtype, starts=0.4)
    want, last = attend64(q, k, v, decay, start, state, D ** -0.5)
    size, lsize = attend64(q.abs(), k.abs(), v.abs(), decay, start, state.abs(), D ** -0.5)
    S = state.clone()
    S[start[0]] = float("nan")                       # what a starting env remembers is never looked at
    f32 = (16 + D) * 2.0 ** -23
    for t in range(6):
        out = linear_attention_step(q[t], k[t], v[t], decay, S, start[t])
        assert out.dtype == dtype
        near(out, want[t], size[t], HALF if dtype == torch.bfloat16 else f32, "out")
    near(S, last, lsize, f32, "state")
    S0, views = state.clone(), [torch.stack([t[0], t[1]], -1)[..., 1] for t in (q, k, v)]
    out = linear_attention_step(*views, decay, S0)   # strided inputs, no starts
    want, last = attend64(q[1:2], k[1:2], v[1:2], decay, None, state, D ** -0.5)
    near(S0, last, lsize + state.abs() + 1, f32, "state")
    near(out, want[0], size[1] + 50, HALF if dtype == torch.bfloat16 else f32, "out")


@pytest.mark.gpu
def test_step_past_32_bits():
    """A state of over 2^32 bytes and 2^31 values; the last envs are compared."""
    N, H, D = 66000, 8, 64
    q = torch.randn(N, H, D, device="cuda").bfloat16()
    state = torch.empty(N, H, D, D, device="cuda").normal_()
    tail = state[-3:].clone()
    out = linear_attention_step(q, q, q, head_decays(H), state)
    want, last = attend64(q[None, -3:], q[None, -3:], q[None, -3:], head_decays(H), None, tail, D ** -0.5)
    assert torch.allclose(state[-3:].double(), last, atol=1e-4)
    assert (out[-3:].double() - want[0]).norm() <= HALF * want.norm()


@pytest.mark.gpu
def test_step_more_heads_than_a_row_of_blocks():
    N, D = 2 ** 24 + 5, 4
    q, k, v = (torch.randn(N, 1, D, device="cuda") for _ in range(3))
    state, decay = torch.randn(N, 1, D, D, device="cuda"), torch.tensor([0.5], device="cuda")
    want = 0.5 * state.double() + k.double()[..., :, None] * v.double()[..., None, :]
    out = linear_attention_step(q, k, v, decay, state)
    assert ((state.double() - want).abs() <= 2.0 ** -22 * (1 + want.abs())).all()
    assert ((out.double() - (q.double()[..., :, None] * want).sum(-2) / 2).abs() <= 2.0 ** -20 * (1 + (q[..., :, None].abs() * want.abs()).sum(-2))).all()


@pytest.mark.gpu
def test_step_tells_who_saved_its_state():
    q = torch.randn(3, 2, 8, device="cuda")
    w, state = torch.randn(3, 2, 8, 8, device="cuda", requires_grad=True), torch.randn(3, 2, 8, 8, device="cuda")
    y = (w * state).sum()
    with torch.no_grad():
        linear_attention_step(q, q, q, head_decays(2), state)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward()
    with torch.inference_mode():
        linear_attention_step(q, q, q, head_decays(2), torch.zeros(3, 2, 8, 8, device="cuda"))


@pytest.mark.gpu
def test_attention_past_32_bits():
    """Steps 2^30 elements apart in one buffer: offsets past 2^31 elements and 2^32 bytes."""
    T, N, H, D = 3, 2, 2, 64
    buf = torch.zeros(2 * 2 ** 30 + 4096, dtype=torch.bfloat16, device="cuda")
    view = buf.as_strided((T, N, H, 3 * D), (2 ** 30, H * 3 * D, 3 * D, 1))
    view.normal_(generator=torch.Generator(device="cuda").manual_seed(1))
    q, k, v = view[..., :D], view[..., D:2 * D], view[..., 2 * D:]
    _, _, _, decay, start, state, do, ds = attend_inputs(T, N, H, D, D, torch.bfloat16)
    check_attend(q, k, v, decay, start, state, do, ds)


@pytest.mark.gpu
@pytest.mark.parametrize("T,N,H,D", [(128, 6, 2, 64), (1500, 1, 2, 64)])
def test_attention_same_bits_and_other_streams(T, N, H, D):
    """The same inputs give the same bits, on another stream and beside other work too; forward and step agree."""
    q, k, v, decay, start, state, do, ds = attend_inputs(T, N, H, D, D, torch.bfloat16)

    def run():
        x = [t.detach().requires_grad_() for t in (q, k, v, state)]
        out, last = linear_attention(*x[:3], decay, start, x[3])
        return [out, last] + list(torch.autograd.grad((out, last), x, (do, ds)))

    first = run()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = [run() for _ in range(3)][-1]
    again = run()
    side.synchronize()
    torch.cuda.synchronize()
    for a, b, c in zip(first, other, again):
        assert torch.equal(a, b) and torch.equal(a, c)


@pytest.mark.gpu
def test_operators_are_differentiable_once():
    q, k, v, decay, start, state, do, ds = attend_inputs(5, 2, 2, 16, 16, torch.float32)
    x, w, b, dy = norm_inputs(3, 16, (3, 3), torch.float32)
    q, x = q.requires_grad_(), x.requires_grad_()
    for y, leaf, g in ((linear_attention(q, k, v, decay, start, state)[0], q, do), (group_norm_act(x, 2, w, b, act="silu"), x, dy)):
        (first,) = torch.autograd.grad(y, leaf, g, create_graph=True)
        assert torch.isfinite(first).all()
        with pytest.raises(RuntimeError, match="once"):
            first.square().sum().backward()


@pytest.mark.gpu
def test_operators_under_graph_capture():
    """Captured once, replayed on new inputs with eager work in between, every replay against the eager result."""
    q, k, v, decay, start, state, _, _ = attend_inputs(300, 2, 2, 64, 64, torch.bfloat16)
    x, w, b, _ = norm_inputs(5, 24, (9, 9), torch.bfloat16)
    S = state.clone()

    def work():
        out, last = linear_attention(q, k, v, decay, start, state)
        return out, last, linear_attention_step(q[0], k[0], v[0], decay, S, start[0]), group_norm_act(x, 3, w, b, act="silu")

    with torch.no_grad():
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
            for t in (q, k, v, state, x):
                t.normal_(generator=g)
            S.copy_(state)
            want = [t.clone() for t in work()]
            S.copy_(state)
            torch.cuda.synchronize()
            graph.replay()
            torch.cuda.synchronize()
            for a, e in zip(held, want):
                assert torch.equal(a, e), i


# ---------------------------------------------------------------- group norm on the GPU
@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("B,C,sp,groups", [
    (1, 8, (), 1), (3, 512, (), 8), (70, 64, (), 1), (5, 512, (), 64), (200, 24, (), 3), (7, 64, (9, 9), 8), (9, 64, (7, 7), 64),
    (4, 32, (20, 20), 4), (3, 32, (20, 20), 8), (6, 16, (3, 3), 4), (2, 48, (84, 84), 6), (2, 96, (11, 5), 4), (3, 30, (5, 4), 5),
    (2, 24, (6, 6), 2), (1, 64, (130, 117), 4), (2, 3, (41, 41), 1), (2, 1, (9, 9), 1), (3, 1024, (4, 4), 32), (2, 2304, (2,), 3),
    (300, 128, (3,), 2), (700, 24, (), 2), (40000, 30, (), 10), (50, 1024, (), 8), (9, 2304, (), 3), (5, 2040, (), 2), (300, 96, (3, 3), 16),
    (60, 12, (9, 9), 2), (5, 130, (2,), 10), (3000, 32, (9, 9), 16), (900, 32, (9, 9), 8), (20, 64, (20, 20), 32)])
def test_norm_vs_float64(B, C, sp, groups, dtype):
    x, w, b, dy = norm_inputs(B, C, sp, dtype, seed=C)
    for act in ("none", "silu"):
        check_norm(x, groups, w, b, act, dy)
    check_norm(x, groups, None, None, "silu", dy)


@pytest.mark.gpu
def test_norm_more_samples_than_a_row_of_blocks():
    x, w, b, dy = norm_inputs(2 ** 22 + 9, 6, (), torch.float32)
    check_norm(x, 2, w, b, "silu", dy)


@pytest.mark.gpu
def test_norm_relu_and_its_gradient():
    """relu's gradient jumps at zero: inputs whose arguments stay away from it by more than their rounding."""
    x, w, b, dy = norm_inputs(6, 32, (9, 9), torch.float32)
    z = norm64(x, 4, w, b, 1e-5, "none")
    assert (z.abs().min() > 1e-6)
    check_norm(x, 4, w, b, "relu", dy)


@pytest.mark.gpu
@pytest.mark.parametrize("B,C,sp", [(3, 64, (9, 9)), (2, 64, (130, 117)), (4, 24, (6, 6)), (3, 48, (5, 5)), (30, 1200, ())])
def test_norm_large_mean_and_constants(B, C, sp):
    x, w, b, dy = norm_inputs(B, C, sp, torch.float32, offset=3000.0)
    check_norm(x, 4, w, b, "silu", dy)
    flat = torch.full_like(x, 7.25)                  # no variance: everything is the bias
    y = group_norm_act(flat, 4, w, b)
    assert torch.allclose(y, b.view(1, -1, *(1,) * len(sp)).expand_as(y), atol=1e-6)
    peak = torch.randn_like(x)                       # one value far above all others, first in its group
    peak[:, 0].view(B, -1)[:, 0] = 1e4
    check_norm(peak, 4, w, b, "none", dy)


@pytest.mark.gpu
@pytest.mark.parametrize("B,C,sp", [(3, 64, (9, 9)), (40, 512, ()), (2, 64, (130, 117)), (3, 48, (5, 5)), (40, 1200, ()), (40, 48, ())])
def test_norm_what_is_not_finite_stays_in_its_group(B, C, sp):
    x, w, b, dy = norm_inputs(B, C, sp, torch.bfloat16)
    clean = group_norm_act(x, 8, w, b, act="relu")
    for bad in (float("nan"), float("inf")):
        y = x.clone()
        y[1, 0] = bad
        got = group_norm_act(y, 8, w, b, act="relu")
        same = torch.ones_like(got, dtype=torch.bool)
        same[1, :C // 8] = False
        assert torch.equal(got[same], clean[same])
        assert torch.isnan(got[1, 0]).all()


@pytest.mark.gpu
def test_norm_takes_views_and_other_types():
    x, w, b, dy = norm_inputs(4, 32, (6, 5), torch.bfloat16)
    want = group_norm_act(x, 4, w, b, act="silu")
    assert want.is_contiguous(memory_format=torch.channels_last)
    assert torch.equal(group_norm_act(x.contiguous(), 4, w, b, act="silu"), want)          # channels first
    off = torch.empty(x.numel() + 1, dtype=x.dtype, device="cuda")[1:].view(4, 6, 5, 32).permute(0, 3, 1, 2)
    off.copy_(x)                                                                           # off a 16-byte boundary
    assert torch.allclose(group_norm_act(off, 4, w, b, act="silu").float(), want.float(), atol=2e-2)
    check_norm(off, 4, w, b, "silu", dy.contiguous())
    wide = torch.zeros(4, 64, 6, 5, dtype=x.dtype, device="cuda").to(memory_format=torch.channels_last)
    wide[:, :32] = x
    assert torch.equal(group_norm_act(wide[:, :32], 4, w, b, act="silu"), want)            # channels of a wider tensor
    wb, bb = w.bfloat16().requires_grad_(), b.bfloat16().requires_grad_()
    y = group_norm_act(x, 4, wb, bb, act="silu")
    assert torch.equal(y.detach(), group_norm_act(x, 4, wb.detach().float(), bb.detach().float(), act="silu"))
    gw, gb = torch.autograd.grad(y, (wb, bb), dy)
    assert gw.dtype == gb.dtype == torch.bfloat16
    empty = x[:0].requires_grad_()
    y = group_norm_act(empty, 4, w.requires_grad_(), b)
    gx, gw = torch.autograd.grad(y, (empty, w), torch.zeros_like(y))
    assert y.shape == empty.shape and gx.shape == empty.shape and (gw == 0).all()


@pytest.mark.gpu
@pytest.mark.parametrize("B,C,sp,groups", [(2000, 64, (9, 9), 8), (20000, 512, (), 8), (2, 64, (130, 117), 4),
                                             (20000, 24, (3, 3), 4), (9000, 1024, (), 8)])
def test_norm_same_bits(B, C, sp, groups):
    x, w, b, dy = norm_inputs(B, C, sp, torch.bfloat16)
    x, w, b = (t.requires_grad_() for t in (x, w, b))
    runs = [torch.autograd.grad(group_norm_act(x, groups, w, b, act="silu"), (x, w, b), dy) for _ in range(3)]
    for r in runs[1:]:
        assert all(torch.equal(a, c) for a, c in zip(runs[0], r))


@pytest.mark.gpu
def test_norm_gradients_are_differences():
    """Directional differences of the kernel's own float32 forward pass, summed in float64."""
    x, w, b, dy = norm_inputs(3, 32, (7, 7), torch.float32)
    x, w, b = (t.requires_grad_() for t in (x, w, b))
    grads = torch.autograd.grad(group_norm_act(x, 4, w, b, act="silu"), (x, w, b), dy)
    g = torch.Generator().manual_seed(2)
    with torch.no_grad():
        for i, (t, grad) in enumerate(zip((x, w, b), grads)):
            u = torch.randn(t.shape, generator=g).cuda()
            h = 1e-2
            up, down = ([s + e * h * u if j == i else s for j, s in enumerate((x, w, b))] for e in (1, -1))
            f = lambda a: (group_norm_act(a[0], 4, a[1], a[2], act="silu").double() * dy).sum()   # noqa: E731
            d, want = (f(up) - f(down)) / (2 * h), (grad.double() * u).sum()
            # rounding 2^-24 sqrt(n) |y dy| / h, and the cubic term h^2 with a third derivative of order one
            assert abs(d - want) <= 2.0 ** -22 * dy.norm() / h + 2 * h ** 2 * (grad.double() * u).norm() * t.numel() ** 0.5, i


# ---------------------------------------------------------------- the network that uses them
def test_memory_net_on_cpu():
    """Steps and the whole sequence agree, memories are cleared at starts, and every parameter gets a gradient."""
    torch.manual_seed(0)
    T, N = 5, 3
    net = memory.make_memory_net(heads=4, device="cpu")
    obs = torch.randint(0, 256, (T, N, 4, 84, 84), dtype=torch.uint8)
    start = torch.zeros(T, N, dtype=torch.bool)
    start[0], start[3, 1] = True, True
    logits, value, last = net(obs, start)
    state = net.initial_state(N) + 7.0                       # what a first step's env remembers is not seen
    for t in range(T):
        lg, v = net.step(obs[t], start[t], state)
        assert torch.allclose(lg, logits[t], atol=1e-5) and torch.allclose(v, value[t], atol=1e-4)
    assert torch.allclose(state, last, atol=1e-4)
    alone, _, _ = net(obs[3:, 1:2], None, None)              # an episode from its start on
    assert torch.allclose(alone, logits[3:, 1:2], atol=1e-5)
    (logits.sum() + value.sum()).backward()
    assert all(p.grad is not None and torch.isfinite(p.grad).all() for p in net.parameters())
    with pytest.raises(ValueError, match="heads"):
        memory.make_memory_net(heads=3, device="cpu")


@pytest.mark.gpu
def test_memory_net_gradients_as_on_cpu():
    """The network's loss and gradients on the GPU (bf16 trunk and memory) against the same weights on the CPU in float32."""
    T, N = 70, 3
    g = torch.Generator().manual_seed(1)
    obs = torch.randint(0, 256, (T, N, 4, 84, 84), dtype=torch.uint8, generator=g)
    start = torch.rand(T, N, generator=g) < 0.05
    nets = [memory.make_memory_net(seed=3, device=d) for d in ("cpu", "cuda")]
    assert all(torch.equal(a.cpu(), b.cpu()) for a, b in zip(nets[0].parameters(), nets[1].parameters()))
    grads = []
    for net, dev in zip(nets, ("cpu", "cuda")):
        state = torch.randn(N, 8, 64, 64, generator=torch.Generator().manual_seed(2)).to(dev).requires_grad_()
        logits, value, last = net(obs.to(dev), start.to(dev), state)
        (torch.log_softmax(logits, -1)[..., 2].mean() + value.square().mean() + 1e-3 * last.square().mean()).backward()
        grads.append([p.grad.float().cpu() for p in net.parameters()] + [state.grad.cpu()])
    for name, a, b in zip([n for n, _ in nets[0].named_parameters()] + ["state"], *grads):
        # a bf16 network of about ten layers: each rounds by 2^-9 at most, forth and back
        assert (a - b).norm() <= 0.1 * a.norm() + 1e-6, (name, ((a - b).norm() / a.norm()).item())


@pytest.mark.gpu
def test_rollout_with_a_memory_is_computed_again():
    """A rollout under the network: its stored log-probabilities and values come out again from the stored sequence, episodes
    ending inside; a second rollout goes on from the memories of the first; training steps change the policy."""
    from build_roms import rom_path
    from fast_mario_env_amd import HipVecEnv
    from fast_mario_env_amd.rollout import Rollout
    import importlib.util
    spec = importlib.util.spec_from_file_location("memory_policy", os.path.join(ROOT, "examples", "memory_policy.py"))
    example = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(example)
    n, T = 24, 20
    env = HipVecEnv("1-1", n, seed=0, sticky=0.25, noop_max=30, max_steps=13, maxpool=True, rom=open(rom_path("vanilla"), "rb").read())
    env.reset()
    net = memory.make_memory_net(seed=0)
    ro = Rollout(env, net, T=T, seed=3)
    for _ in range(2):
        before = ro.memory.clone()
        ro.collect()
        assert torch.equal(ro.memory0, before)
        envs = torch.arange(n, device="cuda")
        with torch.no_grad():
            logits, value, last = net(*ro.sequence(envs))
        logp = torch.log_softmax(logits, -1).gather(-1, ro.act[..., None]).squeeze(-1)
        # (the convolutions of another batch size may take other kernels, and the memory another order of sums: bf16 either way)
        assert torch.allclose(logp, ro.logp, atol=2e-2) and torch.allclose(value, ro.val, atol=0.1, rtol=0.05)
        assert (last - ro.memory).norm() <= 0.03 * last.norm()
        assert ro.start[1:].any()
    with torch.no_grad():                                    # a share of the envs, by index
        part, _, _ = net(*ro.sequence(torch.tensor([5, 2], device="cuda")))
    assert torch.allclose(torch.log_softmax(part, -1), torch.log_softmax(logits[:, [5, 2]], -1), atol=2e-2)
    opt = torch.optim.Adam(net.parameters(), 1e-3)
    old = [p.detach().clone() for p in net.parameters()]
    assert torch.isfinite(example.update(net, opt, ro))
    assert all(not torch.equal(a, b) for a, b in zip(old, net.parameters()))
    env.close()
