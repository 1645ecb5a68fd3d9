"""The operators of a policy that remembers its episode, on the GPU.

The reference's policy sees four stacked frames and keeps nothing between steps (src/fast_mario_env/ppo/model.py:13-38). A
memory of fixed size per env goes on where the stack ends:

- `linear_attention`: over a stored rollout (T, N), each head's memory a matrix that decays by the head's factor each step and
  is cleared where an episode starts; with the gradients of training.
- `linear_attention_step`: one step of the same for every env, the memories updated in place: what acting needs.
- `state_scan`: the same for a memory that selects: a few states a channel whose decays and intake come from the input; with its
  gradients. `state_scan_step`: one step for every env, in place.
- `causal_conv_act`, `causal_conv_act_step`: the short convolution over the steps that goes before such a scan, and an activation.
- `group_norm_act`: group norm and an activation over channels-last features: of the memory's output (a group a head; its size
  grows with the episode) and of convolutions; with its gradients.

`make_memory_net` is an actor-critic that uses them, with either memory, and `Rollout` (rollout.py) runs it: `act` steps the memories along with the
envs, and calling the network on a stored rollout gives the same policy and values, with gradients.

Float32 or bf16 in and out, sums and states in float32. On the GPU they are HIP kernels (libmario_ops.so, include/mario_ops.h),
queued on torch's current stream. CPU tensors, and what torch traces or transforms, take torch operations.
"""
from __future__ import annotations

import math

import torch

from ._native import ops
from .rollout import N_ACTIONS, _transformed, policy_input

ACTS = {"none": 0, "relu": 1, "silu": 2}
MAX_HEAD, MAX_TAPS, MAX_STATES = 128, 8, 64
_DTYPES = (torch.float32, torch.bfloat16)


def _kernel_takes(*ts):
    """Whether a kernel called by address computes these: plain tensors on a GPU that nothing traces or transforms."""
    for t in ts:
        if type(t) not in (torch.Tensor, torch.nn.Parameter) or not t.is_cuda or t.is_neg():
            return False
    return not _transformed(*ts)


def _own(last, state):
    """A state as it is returned: one that the steps take, and not the caller's."""
    return last.clone(memory_format=torch.contiguous_format) if last is state else last.contiguous()


def head_decays(heads: int, device="cuda"):
    """Factors (heads,) whose memories last from about 22 steps (half-life) to about 1,400: 1 - 2^-5 .. 1 - 2^-11."""
    return (1.0 - 2.0 ** -torch.linspace(5.0, 11.0, heads, dtype=torch.float64)).float().to(device)


# ---------------------------------------------------------------- linear attention
def _check_attend(name, lead, q, k, v, decay, start, state):
    shape, dt, dev = q.shape, q.dtype, q.device
    H, D, E = shape[-2], shape[-1], v.shape[-1]
    if (dt not in _DTYPES or k.dtype != dt or v.dtype != dt or k.shape != shape or v.shape[:-1] != shape[:-1]
            or not (1 <= D <= MAX_HEAD and 1 <= E <= MAX_HEAD) or H < 1):
        raise ValueError(f"{name}: q and k must be ({lead}, H, D), v ({lead}, H, E), all float32 or all bf16, head sizes 1 .. {MAX_HEAD}")
    if decay.dtype != torch.float32 or decay.shape != (H,):
        raise ValueError(f"{name}: decay must be ({H},) float32")
    if decay.requires_grad:
        raise ValueError(f"{name}: decay is a constant of the heads: it has no gradient here")
    if start is not None and (start.dtype != torch.bool or start.shape != shape[:-2]):
        raise ValueError(f"{name}: start must be ({lead}) bool")
    if state is not None and (state.dtype != torch.float32 or state.shape != (shape[-3], H, D, E)):
        raise ValueError(f"{name}: state must be (N, H, D, E) = {(shape[-3], H, D, E)} float32")
    for t in (k, v, decay, start, state):
        if t is not None and t.device != dev:
            raise ValueError(f"{name}: all tensors must be on the device of q ({dev})")


def _attend_plain(q, k, v, decay, start, state, scale):
    """The recurrence step by step in torch operations, in float32."""
    S = q.new_zeros(q.shape[1:] + v.shape[-1:], dtype=torch.float32) if state is None else state
    g, out = decay[:, None, None], []
    for t in range(q.shape[0]):
        S = g * S
        if start is not None:
            S = torch.where(start[t][:, None, None, None], torch.zeros_like(S), S)
        S = S + k[t].float()[..., :, None] * v[t].float()[..., None, :]
        out.append((q[t].float()[..., :, None] * S).sum(-2) * scale)
    out = torch.stack(out).to(q.dtype) if out else v.new_empty(v.shape)
    return out, _own(S, state)


def linear_attention(q, k, v, decay, start=None, state=None, scale=None):
    """Linear attention with a decay for each head over T steps of N envs. With g = decay[h], of each env and head:

        S_t = (0 where start[t], else g S_{t-1}) + k_t v_t^T,    out_t = scale S_t^T q_t,    S_{-1} = state

    q, k (T, N, H, D) and v (T, N, H, E), all float32 or all bf16, head sizes up to 128, any strides (views of a fused
    projection are taken as they lie); decay (H,) float32 in [0, 1], a constant without gradient (`head_decays`); start (T, N)
    bool, the steps that start an episode, as `gae` takes them: nothing of an episode reaches the next one; state (N, H, D, E)
    float32 or None for zeros; scale: 1/sqrt(D) if None. Returns out (T, N, H, E) in the type of q and the state after the last
    step, float32. Differentiable once in q, k, v and state.

    Sums and states are float32, those kept for the gradient among them. With bf16 inputs what enters a matrix product from another
    one or from a state goes in as two bf16 parts (2^-16 of it is left out), so results are rounded once, at their end."""
    if q.dim() != 4 or k.dim() != 4 or v.dim() != 4:
        raise ValueError("linear_attention: q, k and v must be (T, N, H, head size)")
    _check_attend("linear_attention", "T, N", q, k, v, decay, start, state)
    scale = q.shape[-1] ** -0.5 if scale is None else float(scale)
    if not _kernel_takes(*(t for t in (q, k, v, decay, start, state) if t is not None)):
        return _attend_plain(q, k, v, decay, start, state, scale)
    return ops().attend(q, k, v, decay, start, state, scale)


def linear_attention_step(q, k, v, decay, state, start=None, scale=None):
    """One step of `linear_attention` for every env: q, k (N, H, D), v (N, H, E), start (N,) bool or None; state (N, H, D, E)
    float32, contiguous, is updated in place. Returns out (N, H, E) in the type of q. No gradient."""
    if q.dim() != 3 or k.dim() != 3 or v.dim() != 3:
        raise ValueError("linear_attention_step: q, k and v must be (N, H, head size)")
    _check_attend("linear_attention_step", "N", q, k, v, decay, start, state)
    if not state.is_contiguous():
        raise ValueError("linear_attention_step: state is updated in place and must be contiguous")
    if torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad or state.requires_grad):
        raise ValueError("linear_attention_step has no gradient: call it under torch.no_grad(), or linear_attention to train")
    scale = q.shape[-1] ** -0.5 if scale is None else float(scale)
    every = (q, k, v, decay, state) if start is None else (q, k, v, decay, state, start)
    if not _kernel_takes(*every):
        out, S = _attend_plain(q[None], k[None], v[None], decay, None if start is None else start[None], state, scale)
        state.copy_(S)
        return out[0]
    return ops().attend_step(q, k, v, decay, state, start, scale)


# ---------------------------------------------------------------- group norm and activation
def _norm_plain(x, groups, weight, bias, eps, act):
    """The same in torch operations, in float32."""
    y = x.float().reshape(x.shape[0], groups, x.shape[1] // groups, -1)
    d = y - y.mean((2, 3), keepdim=True)
    z = (d * torch.rsqrt(d.square().mean((2, 3), keepdim=True) + eps)).reshape(x.shape)
    if weight is not None:
        one = (1, -1) + (1,) * (x.dim() - 2)
        z = z * weight.float().view(one) + bias.float().view(one)
    z = torch.relu(z) if act == "relu" else z * torch.sigmoid(z) if act == "silu" else z
    return z.to(x.dtype)


def group_norm_act(x, groups, weight=None, bias=None, eps=1e-5, act="none"):
    """act(group_norm(x)): x (B, C, ...) float32 or bf16, its channels in `groups` groups of consecutive ones, each normalised
    over the group's channels and all positions of a sample (biased variance), scaled and shifted per channel by weight and
    bias (C,) (both or neither; float32, other float types are converted), then act: "none", "relu" or "silu". All in float32,
    rounded once. The result has x's type and lies channels last, as x does (`memory_format=torch.channels_last`, or (B, C));
    an x that lies otherwise is copied first. Differentiable once."""
    if x.dim() < 2 or x.dtype not in _DTYPES:
        raise ValueError("group_norm_act: x must be (B, C, ...) float32 or bf16")
    C = x.shape[1]
    if not isinstance(groups, int) or groups < 1 or C < 1 or C % groups:
        raise ValueError(f"group_norm_act: {C} channels do not fall into {groups} equal groups")
    if act not in ACTS:
        raise ValueError(f"group_norm_act: act must be one of {', '.join(ACTS)}")
    if not eps >= 0:
        raise ValueError("group_norm_act: eps must be >= 0")
    if (weight is None) != (bias is None):
        raise ValueError("group_norm_act: weight and bias go together")
    if weight is not None and any(p.shape != (C,) or not p.is_floating_point() or p.device != x.device for p in (weight, bias)):
        raise ValueError(f"group_norm_act: weight and bias must be ({C},) on the device of x ({x.device})")
    if 0 in x.shape[2:]:
        raise ValueError("group_norm_act: a sample has no positions")
    if not _kernel_takes(*((x,) if weight is None else (x, weight, bias))):
        return _norm_plain(x, groups, weight, bias, eps, act)
    return ops().group_norm_act(x, groups, weight, bias, eps, ACTS[act])


# ---------------------------------------------------------------- a memory that selects: causal convolution
def _check_conv(name, lead, x, weight, bias, start, state, act):
    C, dev = x.shape[-1], x.device
    if x.dtype not in _DTYPES or C < 1:
        raise ValueError(f"{name}: x must be ({lead}, C) float32 or bf16")
    if weight.dim() != 2 or weight.shape[0] != C or not 1 <= weight.shape[1] <= MAX_TAPS or not weight.is_floating_point():
        raise ValueError(f"{name}: weight must be (C, K) = ({C}, 1 .. {MAX_TAPS})")
    if bias is not None and (bias.shape != (C,) or not bias.is_floating_point()):
        raise ValueError(f"{name}: bias must be ({C},)")
    if start is not None and (start.dtype != torch.bool or start.shape != x.shape[:-1]):
        raise ValueError(f"{name}: start must be ({lead}) bool")
    if state is not None and (state.dtype != x.dtype or state.shape != (x.shape[-2], weight.shape[1] - 1, C)):
        raise ValueError(f"{name}: state must be (N, K - 1, C) = {(x.shape[-2], weight.shape[1] - 1, C)} in the type of x")
    if act not in ACTS:
        raise ValueError(f"{name}: act must be one of {', '.join(ACTS)}")
    for t in (weight, bias, start, state):
        if t is not None and t.device != dev:
            raise ValueError(f"{name}: all tensors must be on the device of x ({dev})")


def _conv_plain(x, weight, bias, start, state, act):
    """The window moved step by step in torch operations, in float32."""
    K = weight.shape[1]
    w = weight.float().t()
    window = x.new_zeros(x.shape[1], K - 1, x.shape[2]) if state is None else state
    out = []
    for t in range(x.shape[0]):
        if start is not None:
            window = torch.where(start[t][:, None, None], torch.zeros_like(window), window)
        every = torch.cat([window, x[t][:, None]], 1)
        p = (every.float() * w).sum(1)
        p = p if bias is None else p + bias.float()
        out.append(torch.relu(p) if act == "relu" else p * torch.sigmoid(p) if act == "silu" else p)
        window = every[:, 1:]
    out = torch.stack(out).to(x.dtype) if out else x.new_empty(x.shape)
    return out, _own(window, state)


def causal_conv_act(x, weight, bias=None, start=None, state=None, act="silu"):
    """A short convolution of each channel over the steps, then act, over T steps of N envs. With K taps:

        y_t = act(bias + sum_j weight[:, K - 1 - j] x_{t-j}),   j = 0 .. K - 1, of what the episode of step t holds

    x (T, N, C) float32 or bf16, any strides; weight (C, K), K up to 8, and bias (C,) or None float32 (other float types are converted);
    start (T, N) bool, the steps that start an episode: no tap reaches past one; state (N, K - 1, C) in the type of x, the inputs before
    the first step, oldest first, None for zeros; act "none", "relu" or "silu". Returns y (T, N, C) in the type of x and the state after
    the last step (0 for what its episode does not hold). Sums in float32, rounded once. Differentiable once in x, weight, bias and state."""
    if x.dim() != 3:
        raise ValueError("causal_conv_act: x must be (T, N, C)")
    _check_conv("causal_conv_act", "T, N", x, weight, bias, start, state, act)
    if not _kernel_takes(*(t for t in (x, weight, bias, start, state) if t is not None)):
        return _conv_plain(x, weight, bias, start, state, act)
    return ops().conv(x, weight, bias, start, state, ACTS[act])


def causal_conv_act_step(x, weight, bias, state, start=None, act="silu"):
    """One step of `causal_conv_act` for every env: x (N, C), start (N,) bool or None; state (N, K - 1, C), contiguous, moves on by the step in
    place. Returns y (N, C). No gradient."""
    if x.dim() != 2:
        raise ValueError("causal_conv_act_step: x must be (N, C)")
    _check_conv("causal_conv_act_step", "N", x, weight, bias, start, state, act)
    if state is None or not state.is_contiguous():
        raise ValueError("causal_conv_act_step: state is updated in place and must be contiguous")
    _no_gradient("causal_conv_act_step", "causal_conv_act", x, weight, bias, state)
    if not _kernel_takes(*(t for t in (x, weight, bias, start, state) if t is not None)):
        y, last = _conv_plain(x[None], weight, bias, None if start is None else start[None], state, act)
        state.copy_(last)
        return y[0]
    return ops().conv_step(x, weight, bias, state, start, ACTS[act])


def _no_gradient(name, instead, *ts):
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in ts):
        raise ValueError(f"{name} has no gradient: call it under torch.no_grad(), or {instead} to train")


# ---------------------------------------------------------------- a memory that selects: state space scan
def _check_scan(name, lead, x, dt, A, B, C, D, z, dt_bias, start, state):
    ch, dev = x.shape[-1], x.device
    if x.dtype not in _DTYPES or ch < 1 or any(t is not None and (t.dtype != x.dtype or t.shape != x.shape) for t in (dt, z)):
        raise ValueError(f"{name}: x, dt and z must be ({lead}, C), all float32 or all bf16")
    if A.dim() != 2 or A.shape[0] != ch or not 1 <= A.shape[1] <= MAX_STATES or not A.is_floating_point():
        raise ValueError(f"{name}: A must be (C, S) = ({ch}, 1 .. {MAX_STATES})")
    S = A.shape[1]
    if (B.dim() != x.dim() + 1 or B.shape != C.shape or B.shape[:-2] != x.shape[:-1] or B.shape[-1] != S or B.dtype != x.dtype
            or C.dtype != x.dtype or B.shape[-2] < 1 or ch % B.shape[-2]):
        raise ValueError(f"{name}: B and C must be ({lead}, G, {S}) in the type of x, G a divisor of {ch}")
    for n, t in (("D", D), ("dt_bias", dt_bias)):
        if t is not None and (t.shape != (ch,) or not t.is_floating_point()):
            raise ValueError(f"{name}: {n} must be ({ch},)")
    if start is not None and (start.dtype != torch.bool or start.shape != x.shape[:-1]):
        raise ValueError(f"{name}: start must be ({lead}) bool")
    if state is not None and (state.dtype != torch.float32 or state.shape != (x.shape[-2], ch, S)):
        raise ValueError(f"{name}: state must be (N, C, S) = {(x.shape[-2], ch, S)} float32")
    for t in (dt, A, B, C, D, z, dt_bias, start, state):
        if t is not None and t.device != dev:
            raise ValueError(f"{name}: all tensors must be on the device of x ({dev})")


def _scan_plain(x, dt, A, B, C, D, z, dt_bias, start, state):
    """The recurrence step by step in torch operations, in float32."""
    T, N, ch = x.shape
    h = x.new_zeros((N,) + A.shape, dtype=torch.float32) if state is None else state
    A, out = A.float(), []
    every = lambda v: v.float().unsqueeze(2).expand(N, v.shape[1], ch // v.shape[1], v.shape[2]).reshape(N, ch, v.shape[2])   # noqa: E731 (a group's channels)
    for t in range(T):
        xt, raw = x[t].float(), dt[t].float() if dt_bias is None else dt[t].float() + dt_bias.float()
        d = torch.logaddexp(raw, torch.zeros_like(raw))
        if start is not None:
            h = torch.where(start[t][:, None, None], torch.zeros_like(h), h)   # (before the product, whose gradient reads it)
        h = torch.exp(d[..., None] * A) * h + (d * xt)[..., None] * every(B[t])
        y = (every(C[t]) * h).sum(-1)
        y = y if D is None else y + D.float() * xt
        if z is not None:
            zt = z[t].float()
            y = y * (zt * torch.sigmoid(zt))
        out.append(y)
    out = torch.stack(out).to(x.dtype) if out else x.new_empty(x.shape)
    return out, _own(h, state)


def state_scan(x, dt, A, B, C, D=None, z=None, dt_bias=None, start=None, state=None):
    """A selective state space scan over T steps of N envs: what a channel's states keep and take up depends on the input. Of each env and
    channel, with d = softplus(dt + dt_bias) and B, C those of the channel's group:

        h_t = (0 where start[t], else exp(d_t A) h_{t-1}) + d_t x_t B_t,    y_t = (C_t . h_t + D x_t) silu(z_t),    h_{-1} = state

    x, dt and z (T, N, C) (z None: no factor), B and C (T, N, G, S), G a divisor of C (groups of C / G neighbouring channels), all float32 or all
    bf16, any strides; A (C, S), S up to 64, none above 0, D and dt_bias (C,) or None float32 (other float types are converted); start (T, N)
    bool: nothing of an episode reaches the next one; state (N, C, S) float32 or None for zeros. Returns y (T, N, C) in the type of x and the state
    after the last step, float32. States, step sizes, decays and sums are float32, results rounded once. Differentiable once in all but start."""
    if x.dim() != 3:
        raise ValueError("state_scan: x must be (T, N, C)")
    _check_scan("state_scan", "T, N", x, dt, A, B, C, D, z, dt_bias, start, state)
    if not _kernel_takes(*(t for t in (x, dt, A, B, C, D, z, dt_bias, start, state) if t is not None)):
        return _scan_plain(x, dt, A, B, C, D, z, dt_bias, start, state)
    return ops().scan(x, dt, A, B, C, D, z, dt_bias, start, state)


def state_scan_step(x, dt, A, B, C, state, D=None, z=None, dt_bias=None, start=None):
    """One step of `state_scan` for every env: x, dt, z (N, C), B and C (N, G, S), start (N,) bool or None; state (N, C, S) float32,
    contiguous, is updated in place. Returns y (N, C) in the type of x. No gradient."""
    if x.dim() != 2:
        raise ValueError("state_scan_step: x must be (N, C)")
    _check_scan("state_scan_step", "N", x, dt, A, B, C, D, z, dt_bias, start, state)
    if state is None or not state.is_contiguous():
        raise ValueError("state_scan_step: state is updated in place and must be contiguous")
    _no_gradient("state_scan_step", "state_scan", x, dt, A, B, C, D, z, dt_bias, state)
    if not _kernel_takes(*(t for t in (x, dt, A, B, C, D, z, dt_bias, start, state) if t is not None)):
        one = lambda t: None if t is None else t[None]   # noqa: E731
        y, last = _scan_plain(x[None], dt[None], A, B[None], C[None], D, one(z), dt_bias, one(start), state)
        state.copy_(last)
        return y[0]
    return ops().scan_step(x, dt, A, B, C, state, D, z, dt_bias, start)


# ---------------------------------------------------------------- an actor-critic with a memory
def make_memory_net(n_actions: int = N_ACTIONS, in_ch: int = 4, heads: int = 8, seed: int = 0, device="cuda", memory: str = "attention",
                    states: int = 16, taps: int = 4):
    """The Nature trunk of `make_net` with a group norm after each convolution, and between its features and the two heads a
    memory, added to the features:

    - "attention": projection to q, k and v, linear attention with `heads` decaying memories of 512 / heads, group norm a head, projection;
    - "scan": projection to x and z, causal convolution of x over `taps` steps, projection to step sizes (through 32 values), B and C, a state
      space scan with `states` states a channel, gated by z, projection.

    Random weights. On the GPU the trunk and the memory run in bf16 (the memories themselves and the heads in float32), on the CPU
    everything in float32."""
    nn, F = torch.nn, torch.nn.functional
    width, rank = 512, 32
    if memory not in ("attention", "scan"):
        raise ValueError("make_memory_net: memory must be attention or scan")
    if memory == "attention" and (heads < 1 or width % heads or width // heads > MAX_HEAD):
        raise ValueError(f"make_memory_net: heads must divide {width} into heads of at most {MAX_HEAD}")
    if memory == "scan" and not (1 <= states <= MAX_STATES and 1 <= taps <= MAX_TAPS):
        raise ValueError(f"make_memory_net: 1 .. {MAX_STATES} states and 1 .. {MAX_TAPS} taps")

    class MemoryAC(nn.Module):
        def __init__(self):
            super().__init__()
            self.convs = nn.ModuleList([nn.Conv2d(in_ch, 32, 8, 4), nn.Conv2d(32, 64, 4, 2), nn.Conv2d(64, 64, 3, 1)])
            self.norms = nn.ModuleList([nn.GroupNorm(8, c) for c in (32, 64, 64)])   # (parameters; group_norm_act computes)
            self.fc = nn.Linear(64 * 7 * 7, width)
            self._make_memory()
            self.out = nn.Linear(width, width, bias=False)
            self.pi = nn.Linear(width, n_actions)
            self.vf = nn.Linear(width, 1)
            for m in list(self.convs) + [self.fc]:
                nn.init.orthogonal_(m.weight, math.sqrt(2.0))
                nn.init.zeros_(m.bias)
            for m, gain in ((self.into, 1.0), (self.out, 1.0), (self.pi, 0.01), (self.vf, 1.0)):
                nn.init.orthogonal_(m.weight, gain)
            nn.init.zeros_(self.pi.bias)
            nn.init.zeros_(self.vf.bias)

        def _device(self):
            return self.fc.weight.device

        def _autocast(self):
            on = self.fc.weight.is_cuda
            return torch.autocast("cuda" if on else "cpu", dtype=torch.bfloat16, enabled=on)

        def _features(self, obs_u8):
            """uint8 (B, k, 84, 84) -> the projected features and what goes into the memory, (B, 512) and (B, ..)."""
            if obs_u8.is_cuda:
                x = torch.empty(obs_u8.shape, dtype=torch.bfloat16, device=obs_u8.device, memory_format=torch.channels_last)
                policy_input(obs_u8.contiguous(), x)
            else:
                x = obs_u8.float().mul_(1.0 / 255.0)
            with self._autocast():
                for c, g in zip(self.convs, self.norms):
                    x = group_norm_act(c(x), g.num_groups, g.weight, g.bias, eps=g.eps, act="silu")
                h = F.silu(self.fc(x.flatten(1)))
                return h, self.into(h)

        def _heads(self, h, y):
            with self._autocast():
                h = h + self.out(self._leave(y))
            h = h.float()
            return self.pi(h), self.vf(h).squeeze(-1)

        def forward(self, obs_u8, start=None, state=None):
            """A rollout: obs_u8 (T, N, k, 84, 84) uint8, start (T, N) bool and state, the memories before it (as `initial_state`
            makes them) -> logits (T, N, A), values (T, N), the memories after it."""
            T, N = obs_u8.shape[:2]
            h, u = self._features(obs_u8.flatten(0, 1))
            y, state = self._remember(u.unflatten(0, (T, N)), start, state)
            logits, value = self._heads(h, y.flatten(0, 1))
            return logits.unflatten(0, (T, N)), value.unflatten(0, (T, N)), state

        @torch.no_grad()
        def step(self, obs_u8, start, state):
            """One step: obs_u8 (N, k, 84, 84), start (N,) bool or None; state is updated. Logits (N, A), values (N,)."""
            h, u = self._features(obs_u8)
            return self._heads(h, self._remember_step(u, start, state))

        @torch.no_grad()
        def act(self, obs_u8, generator=None, start=None, state=None):
            """Action (Gumbel-max sample), its log-probability and the value, as NatureAC.act; state is updated."""
            logits, value = self.step(obs_u8, start, state)
            logp = F.log_softmax(logits, -1)
            u = torch.rand(logits.shape, generator=generator, device=logits.device).clamp_(1e-20, 1.0)
            a = (logp - torch.log(-torch.log(u))).argmax(-1)
            return a, logp.gather(-1, a[:, None]).squeeze(-1), value

    class AttentionAC(MemoryAC):
        def _make_memory(self):
            self.heads = heads
            self.qkv = nn.Linear(width, 3 * width, bias=False)
            self.norm = nn.GroupNorm(heads, width)
            self.register_buffer("decay", head_decays(heads, "cpu"))

        @property
        def into(self):
            return self.qkv

        def initial_state(self, n: int):
            """The memories of n envs before anything: (n, heads, D, D) float32 zeros."""
            d = width // heads
            return torch.zeros(n, heads, d, d, device=self._device())

        def _split(self, u):
            return (y.unflatten(-1, (heads, -1)) for y in u.chunk(3, -1))

        def _remember(self, u, start, state):
            out, state = linear_attention(*self._split(u), self.decay, start, state)
            return out.flatten(2), state

        def _remember_step(self, u, start, state):
            return linear_attention_step(*self._split(u), self.decay, state, start).flatten(1)

        def _leave(self, y):
            return group_norm_act(y, heads, self.norm.weight, self.norm.bias, eps=self.norm.eps, act="silu")

    class ScanAC(MemoryAC):
        def _make_memory(self):
            self.into = nn.Linear(width, 2 * width, bias=False)
            self.taps = nn.Parameter(torch.randn(width, taps) / taps ** 0.5)
            self.taps_bias = nn.Parameter(torch.zeros(width))
            self.select = nn.Linear(width, rank + 2 * states, bias=False)
            self.sizes = nn.Linear(rank, width, bias=False)
            # step sizes from 0.001 to 0.1 and decay rates 1 .. states: memories of a few steps to about a thousand
            size = torch.exp(torch.rand(width) * math.log(100.0) + math.log(0.001))
            self.size_bias = nn.Parameter(torch.log(torch.expm1(size)))
            self.log_rate = nn.Parameter(torch.log(torch.arange(1.0, states + 1.0)).repeat(width, 1))
            self.skip = nn.Parameter(torch.ones(width))

        def initial_state(self, n: int):
            """The memories of n envs before anything: zeros, the last inputs (n, taps - 1, 512) and the states (n, 512, states) float32."""
            dev = self._device()
            return (torch.zeros(n, taps - 1, width, device=dev, dtype=torch.bfloat16 if dev.type == "cuda" else torch.float32),
                    torch.zeros(n, width, states, device=dev))

        def _scan_in(self, x):
            """Of the convolved inputs (.., 512): step sizes, B and C, and what does not go by the step."""
            with self._autocast():
                small, B, C = self.select(x).split((rank, states, states), -1)
                dt = self.sizes(small)
            return dict(x=x, dt=dt, A=-torch.exp(self.log_rate), B=B.unsqueeze(-2), C=C.unsqueeze(-2), D=self.skip, dt_bias=self.size_bias)

        def _remember(self, u, start, state):
            x, z = u.chunk(2, -1)
            window, states_before = (None, None) if state is None else state
            x, window = causal_conv_act(x, self.taps, self.taps_bias, start, window)
            y, after = state_scan(**self._scan_in(x), z=z, start=start, state=states_before)
            return y, (window, after)

        def _remember_step(self, u, start, state):
            x, z = u.chunk(2, -1)
            x = causal_conv_act_step(x, self.taps, self.taps_bias, state[0], start)
            return state_scan_step(**self._scan_in(x), z=z, start=start, state=state[1])

        def _leave(self, y):
            return y

    torch.manual_seed(seed)
    net = (AttentionAC if memory == "attention" else ScanAC)().to(device)
    if torch.device(device).type == "cuda":
        net = net.to(memory_format=torch.channels_last)
    return net
