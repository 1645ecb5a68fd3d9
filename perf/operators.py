"""The operators of a policy with a memory, as they are timed: through the package's public entry points, or in plain form.

kinds of case
  attend        linear_attention over a rollout (T, N): values and log-probabilities of stored steps, no gradient
  attend_train  the same with its gradients, as in a training step
  step          linear_attention_step: one new step of every env, the memories updated in place
  norm          group_norm_act of channels-last features, no gradient
  norm_train    the same with its gradients

Of one env and head with factor g, steps t of a rollout and episode starts s_t:
  S_t = (0 where s_t, else g S_{t-1}) + k_t v_t^T,   o_t = scale S_t^T q_t.
Group norm: y = act(w (x - mean) / sqrt(var + eps) + b), mean and var over a sample's pixels and a group's channels.
"""
import os
import sys

import torch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
DEV = "cuda:0"
own = False   # the package's operators instead of the plain forms

CHUNK = 64    # steps that the plain form's masked products span
P_START = 0.011   # share of steps that start an episode, as in the headline workload
TYPES = {"bf16": torch.bfloat16, "f32": torch.float32}
EPS = 1e-5


def listed():
    return [
        # a PPO rollout's 128 steps: the policy's values of a shard of the envs from the fused projection
        dict(name="attend_128x4096", kind="attend", dtype="bf16", T=128, N=4096, H=8, D=64, E=64, fused=True),
        # a handful of envs looked at over a few steps, in the float32 of a CPU-trained network
        dict(name="attend_24x40_f32", kind="attend", dtype="f32", T=24, N=40, H=4, D=32, E=32, fused=False),
        # whole recorded episodes of two envs, far longer than a rollout, with the widest heads
        dict(name="attend_16001x2", kind="attend", dtype="bf16", T=16001, N=2, H=8, D=128, E=128, fused=False),
        # one minibatch of the training epochs over the rollout
        dict(name="train_128x2048", kind="attend_train", dtype="bf16", T=128, N=2048, H=8, D=64, E=64, fused=False),
        # imitation of whole episodes at the time limit: few envs, long, ragged, values wider than keys
        dict(name="train_1999x8", kind="attend_train", dtype="bf16", T=1999, N=8, H=8, D=64, E=128, fused=False),
        # a small training run without mixed precision
        dict(name="train_97x64_f32", kind="attend_train", dtype="f32", T=97, N=64, H=8, D=64, E=64, fused=False),
        # one act of the headline's envs
        dict(name="step_32768", kind="step", dtype="bf16", N=32768, H=8, D=64, E=64),
        # one act of the class's default of 8 envs
        dict(name="step_8", kind="step", dtype="bf16", N=8, H=8, D=64, E=64),
        # after the trunk's first convolution, at a rollout's batch
        dict(name="norm_4096x32x20x20", kind="norm", dtype="bf16", B=4096, C=32, W=20, groups=4, act="relu"),
        # after its second one, in a training step
        dict(name="norm_train_4096x64x9x9", kind="norm_train", dtype="bf16", B=4096, C=64, W=9, groups=8, act="silu"),
        # the memory's own output, a group a head and one position a row, in a training step
        dict(name="norm_train_262144x512", kind="norm_train", dtype="bf16", B=262144, C=512, W=1, groups=8, act="silu"),
        # whole observations of a few envs under an odd channel count
        dict(name="norm_train_37x48x84x84_f32", kind="norm_train", dtype="f32", B=37, C=48, W=84, groups=6, act="silu"),
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(lo * (hi / lo) ** rng.random()))))


def draw(rng):
    kind = rng.choice(("attend", "attend", "attend_train", "attend_train", "step", "norm", "norm_train", "norm_train"))
    dtype = rng.choice(("bf16", "bf16", "f32"))
    if kind in ("attend", "attend_train", "step"):
        H = rng.choice((1, 2, 3, 4, 8))
        D = rng.choice((16, 32, 40, 64, 64, 96, 128))
        E = D if rng.random() < 0.7 else rng.choice((32, 64, 128))
        if kind == "step":
            return dict(kind=kind, dtype=dtype, N=_log_int(rng, 1, 8192), H=H, D=D, E=E)
        T = _log_int(rng, 1, 8192)
        N = _log_int(rng, 1, max(1, min(4096, 1 << 26 >> (T * H * (D + E)).bit_length())))
        return dict(kind=kind, dtype=dtype, T=T, N=N, H=H, D=D, E=E, fused=kind == "attend" and rng.random() < 0.5)
    C = rng.choice((16, 24, 32, 48, 64, 64, 96, 128, 256, 512))
    W = rng.choice((1, 1, 3, 7, 9, 20, 27, 41, 84))
    groups = rng.choice([g for g in (1, 2, 4, 6, 8, 16, 32) if C % g == 0 and (W > 1 or C // g >= 8)])
    B = _log_int(rng, 1, max(2, min(131072, (1 << 26) // (C * W * W))))
    # (the gradient of relu jumps at zero, where two right results of its argument may lie on either side)
    return dict(kind=kind, dtype=dtype, B=B, C=C, W=W, groups=groups,
                act=rng.choice(("none", "silu") if kind == "norm_train" else ("none", "relu", "silu")))


# ---------------------------------------------------------------- what a program has in hand before the call
def _decay(H):
    """The heads' factors: half-lives from about 22 steps to over a thousand."""
    return 1.0 - 2.0 ** -torch.linspace(5.0, 11.0, H, device=DEV, dtype=torch.float64).float()


def _inputs(case, seed):
    """The inputs by name, in an order and with values that the seed alone sets."""
    g = torch.Generator(device=DEV)
    g.manual_seed(int(seed))
    t = TYPES[case["dtype"]]

    def normal(*shape, dtype=t, by=1.0):
        return torch.randn(shape, generator=g, device=DEV, dtype=dtype if dtype == torch.float32 else torch.bfloat16).mul_(by).to(dtype)

    if case["kind"] in ("norm", "norm_train"):
        B, C, W = case["B"], case["C"], case["W"]
        x = normal(B, W, W, C) + normal(C)                      # each channel about a mean of its own
        s = dict(x=x.permute(0, 3, 1, 2) if W > 1 else x.view(B, C), w=1.0 + 0.1 * normal(C, dtype=torch.float32),
                 b=0.1 * normal(C, dtype=torch.float32))
        if case["kind"] == "norm_train":
            dy = normal(B, W, W, C)
            s["dy"] = dy.permute(0, 3, 1, 2) if W > 1 else dy.view(B, C)
        return s
    N, H, D, E = (case[k] for k in ("N", "H", "D", "E"))
    lead = (N,) if case["kind"] == "step" else (case["T"], N)
    if case.get("fused"):
        x = normal(*lead, H * (2 * D + E))
        q, k, v = (y.unflatten(-1, (H, -1)) for y in x.split((H * D, H * D, H * E), -1))
    else:
        q, k, v = normal(*lead, H, D), normal(*lead, H, D), normal(*lead, H, E)
    s = dict(q=q, k=k, v=v, decay=_decay(H), start=torch.rand(lead, generator=g, device=DEV) < P_START,
             state=normal(N, H, D, E, dtype=torch.float32, by=2.0))
    if case["kind"] == "attend_train":
        s["do"], s["dstate"] = normal(*lead, H, E), normal(N, H, D, E, dtype=torch.float32)
    return s


def prepare(case, seed):
    s = _inputs(case, seed)
    for name in {"attend_train": ("q", "k", "v", "state"), "norm_train": ("x", "w", "b")}.get(case["kind"], ()):
        s[name].requires_grad_()
    return dict(s, kind=case["kind"], groups=case.get("groups"), act=case.get("act"))


# ---------------------------------------------------------------- the plain forms
def _plain_attend(q, k, v, decay, start, state):
    """Chunks of steps: masked products inside a chunk, and the chunks' own sums mixed into what enters each of them."""
    (T, N, H, D), E, t32 = q.shape, v.shape[-1], torch.float32
    L = min(CHUNK, T)
    n = -(-T // L)

    def chunks(x):                                               # (T, N, H, d) -> (N, H, n, L, d), zeros after the end
        x = torch.cat([x.to(t32), x.new_zeros((n * L - T,) + x.shape[1:], dtype=t32)])
        return x.view(n, L, N, H, -1).permute(2, 3, 0, 1, 4)

    q, k, v = chunks(q), chunks(k), chunks(v)
    lg = decay.to(t32).log().view(H, 1, 1, 1)
    i = torch.arange(L, device=DEV)
    seg = start.to(t32).cumsum(0).t()                            # the episode of each step, 0: the state's
    seg = torch.cat([seg, seg[:, -1:].expand(N, n * L - T)], 1).view(N, 1, n, L)
    same = (seg[..., :, None] == seg[..., None, :]) & (i[:, None] >= i[None, :])
    mask = torch.where(same, ((i[:, None] - i[None, :]).clamp(min=0) * lg).exp(), 0.0)
    out = ((q @ k.transpose(-1, -2)) * mask) @ v
    ends = (torch.arange(n + 1, device=DEV) * L).clamp(max=T)     # where chunk c begins and chunk c - 1 ends
    left = (ends[1:, None] - 1 - (ends[:-1, None] + i)).clamp(min=0)
    own_sum = (k * torch.where(seg == seg[..., -1:], (left * lg[..., 0, 0].view(1, H, 1, 1)).exp(), 0.0)[..., None]).transpose(-1, -2) @ v
    every = torch.cat([state.to(t32)[:, :, None], own_sum], 2).flatten(3)
    last = torch.cat([seg.new_zeros(N, 1, 1), seg[..., -1]], 2)   # the episode that an entering state belongs to
    alive = (last[..., :, None] == last[..., None, :]) & (ends[:, None] >= ends[None, :])
    alive = alive & (torch.arange(n + 1, device=DEV)[:, None] >= torch.arange(n + 1, device=DEV))
    mix = torch.where(alive, ((ends[:, None] - ends[None, :]).clamp(min=0) * lg[..., 0]).exp(), 0.0)
    enter = (mix @ every).view(N, H, n + 1, D, E)
    reach = torch.where(seg == last[..., :-1, None], ((i + 1) * lg[..., 0]).exp(), 0.0)
    out = (out + reach[..., None] * (q @ enter[:, :, :-1])) * D ** -0.5
    return out.permute(2, 3, 0, 1, 4).reshape(n * L, N, H, E)[:T], enter[:, :, -1]


def _plain_step(q, k, v, decay, state, start):
    q, k, v = q.float(), k.float(), v.float()
    state.copy_(torch.where(start[:, None, None, None], 0.0, decay[:, None, None] * state) + k[..., :, None] * v[..., None, :])
    return (q[..., None] * state).sum(-2) * q.shape[-1] ** -0.5


def _plain_norm(x, groups, w, b, act):
    y = x.to(torch.float32).reshape(x.shape[0], groups, x.shape[1] // groups, -1)
    d = y - y.mean((2, 3), keepdim=True)
    z = d * (d.square().mean((2, 3), keepdim=True) + EPS).rsqrt()
    one = (1, -1) + (1,) * (x.dim() - 2)
    z = z.reshape(x.shape) * w.view(one) + b.view(one)
    return z.clamp(min=0.0) if act == "relu" else z / (1.0 + (-z).exp()) if act == "silu" else z


# ---------------------------------------------------------------- one pass
def _package():
    if os.path.join(ROOT, "fast-mario-env_amd") not in sys.path:
        sys.path.insert(0, os.path.join(ROOT, "fast-mario-env_amd"))
    from fast_mario_env_amd import memory
    return memory


def _attend(s):
    if own:
        return _package().linear_attention(s["q"], s["k"], s["v"], s["decay"], s["start"], s["state"])
    out, state = _plain_attend(s["q"], s["k"], s["v"], s["decay"], s["start"], s["state"])
    return out.to(s["q"].dtype), state


def _norm(s):
    if own:
        return _package().group_norm_act(s["x"], s["groups"], s["w"], s["b"], eps=EPS, act=s["act"])
    y = _plain_norm(s["x"], s["groups"], s["w"], s["b"], s["act"])
    return y.to(s["x"].dtype)


def run(s):
    kind = s["kind"]
    if kind == "step":
        if own:
            out = _package().linear_attention_step(s["q"], s["k"], s["v"], s["decay"], s["state"], s["start"])
        else:
            out = _plain_step(s["q"], s["k"], s["v"], s["decay"], s["state"], s["start"]).to(s["q"].dtype)
        return dict(out=out, state=s["state"])
    if kind in ("attend", "norm"):
        with torch.no_grad():
            if kind == "norm":
                return dict(y=_norm(s))
            out, state = _attend(s)
            return dict(out=out, state=state)
    if kind == "attend_train":
        out, state = _attend(s)
        dq, dk, dv, ds = torch.autograd.grad((out, state), (s["q"], s["k"], s["v"], s["state"]), (s["do"], s["dstate"]))
        return dict(out=out.detach(), state=state.detach(), dq=dq, dk=dk, dv=dv, ds=ds)
    y = _norm(s)
    dx, dw, db = torch.autograd.grad(y, (s["x"], s["w"], s["b"]), s["dy"])
    return dict(y=y.detach(), dx=dx, dw=dw, db=db)


# ---------------------------------------------------------------- what a pass cannot do without
def work(case):
    size = 2 if case["dtype"] == "bf16" else 4
    if case["kind"] in ("norm", "norm_train"):
        values, train = case["B"] * case["C"] * case["W"] ** 2, case["kind"] == "norm_train"
        return dict(bytes=values * size * (4 if train else 2) + case["C"] * 4 * (4 if train else 2), flops=values * (24 if train else 10))
    N, H, D, E = (case[k] for k in ("N", "H", "D", "E"))
    steps, states = case.get("T", 1) * N, N * H * D * E * 4
    if case["kind"] == "attend_train":
        # q, k, v, do in, out, dq, dk, dv out; state and dstate in, state and ds out; a state's update, its gradient's,
        # the update again going back, and the products of out, dq, dk and dv
        return dict(bytes=steps * H * (4 * D + 4 * E) * size + steps + 4 * states, flops=14 * steps * H * D * E)
    return dict(bytes=steps * H * (2 * D + 2 * E) * size + steps + 2 * states, flops=4 * steps * H * D * E)


# ---------------------------------------------------------------- from the definition, in 64 bits
def _exact_attend(s, train):
    """Step by step: forward for out and dq, backward for dk and dv."""
    f = {n: s[n].detach().double() for n in ("q", "k", "v", "state", "do", "dstate") if n in s}
    g, scale, T = s["decay"].double()[:, None, None], s["q"].shape[-1] ** -0.5, s["q"].shape[0]
    keep = (~s["start"]).double()[..., None, None, None] * g     # (T, N, H, 1, 1)
    S, out, dq = f["state"], torch.empty_like(f["v"]), torch.empty_like(f["q"])
    for t in range(T):
        S = keep[t] * S + f["k"][t][..., None] * f["v"][t][..., None, :]
        out[t] = (f["q"][t][..., None, :] @ S)[..., 0, :] * scale
        if train:
            dq[t] = (S @ f["do"][t][..., None])[..., 0] * scale
    got = dict(out=out, state=S)
    if not train:
        return got
    R, dk, dv = f["dstate"], torch.empty_like(f["k"]), torch.empty_like(f["v"])
    for t in reversed(range(T)):
        R = R + scale * f["q"][t][..., None] * f["do"][t][..., None, :]
        dk[t] = (R @ f["v"][t][..., None])[..., 0]
        dv[t] = (f["k"][t][..., None, :] @ R)[..., 0, :]
        R = keep[t] * R
    return dict(got, dq=dq, dk=dk, dv=dv, ds=R)


def _exact_norm(s, groups, act, train):
    x, w, b = (s[n].detach().double() for n in ("x", "w", "b"))
    B, C = x.shape[:2]
    rows = lambda y: y.reshape(B, C, -1).transpose(1, 2)         # noqa: E731  (B, pixels, C)
    x3 = rows(x)
    of = torch.arange(C, device=DEV) // (C // groups)
    to_group = (of[:, None] == torch.arange(groups, device=DEV)).double() * (groups / (C * x3.shape[1]))
    per = lambda y: (y.sum(1) @ to_group)[:, of][:, None]        # noqa: E731  each channel's group mean
    mean = per(x3)
    r = (per(x3 * x3) - mean * mean + EPS) ** -0.5
    h = (x3 - mean) * r
    z = h * w + b
    sig = torch.sigmoid(z)
    back = lambda y: y.transpose(1, 2).reshape(x.shape)          # noqa: E731
    got = dict(y=back(torch.relu(z) if act == "relu" else z * sig if act == "silu" else z))
    if not train:
        return got
    dz = rows(s["dy"].double())
    dz = dz * (z > 0) if act == "relu" else dz * sig * (1.0 + z * (1.0 - sig)) if act == "silu" else dz
    dh = dz * w
    dx = r * (dh - per(dh) - h * per(dh * h))
    return dict(got, dx=back(dx), dw=(dz * h).sum((0, 1)), db=dz.sum((0, 1)))


def exact(case, seed):
    s = _inputs(case, seed)
    if case["kind"] in ("norm", "norm_train"):
        return _exact_norm(s, case["groups"], case["act"], case["kind"] == "norm_train")
    if case["kind"] == "step":
        s = {n: x[None] if n in ("q", "k", "v", "start") else x for n, x in s.items()}
        got = _exact_attend(s, False)
        return dict(out=got["out"][0], state=got["state"])
    return _exact_attend(s, case["kind"] == "attend_train")
