"""The operators of a policy that remembers its episode, on the GPU.

The reference's policy sees four stacked frames and keeps nothing between steps (src/fast_mario_env/ppo/model.py:13-38). A
memory of fixed size per env goes on where the stack ends:

- `linear_attention`: over a stored rollout (T, N), each head's memory a matrix that decays by the head's factor each step and
  is cleared where an episode starts; with the gradients of training.
- `linear_attention_step`: one step of the same for every env, the memories updated in place: what acting needs.
- `group_norm_act`: group norm and an activation over channels-last features: of the memory's output (a group a head; its size
  grows with the episode) and of convolutions; with its gradients.

`make_memory_net` is an actor-critic that uses them, and `Rollout` (rollout.py) runs it: `act` steps the memories along with the
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
MAX_HEAD = 128
_DTYPES = (torch.float32, torch.bfloat16)


def _kernel_takes(*ts):
    """Whether a kernel called by address computes these: plain tensors on a GPU that nothing traces or transforms."""
    for t in ts:
        if type(t) not in (torch.Tensor, torch.nn.Parameter) or not t.is_cuda or t.is_neg():
            return False
    return not _transformed(*ts)


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
    return out, S.clone() if S is state else S


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
    z = z.clamp(min=0.0) if act == "relu" else z * torch.sigmoid(z) if act == "silu" else z
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


# ---------------------------------------------------------------- an actor-critic with a memory
def make_memory_net(n_actions: int = N_ACTIONS, in_ch: int = 4, heads: int = 8, seed: int = 0, device="cuda"):
    """The Nature trunk of `make_net` with a group norm after each convolution, and between its features and the two heads a
    memory: projection to q, k and v, linear attention with `heads` decaying memories of 512 / heads, group norm a head,
    projection, added to the features. Random weights. On the GPU the trunk and the memory run in bf16 (the memories
    themselves and the heads in float32), on the CPU everything in float32."""
    nn, F = torch.nn, torch.nn.functional
    width = 512
    if heads < 1 or width % heads or width // heads > MAX_HEAD:
        raise ValueError(f"make_memory_net: heads must divide {width} into heads of at most {MAX_HEAD}")

    class MemoryAC(nn.Module):
        def __init__(self):
            super().__init__()
            self.heads = heads
            self.convs = nn.ModuleList([nn.Conv2d(in_ch, 32, 8, 4), nn.Conv2d(32, 64, 4, 2), nn.Conv2d(64, 64, 3, 1)])
            self.norms = nn.ModuleList([nn.GroupNorm(8, c) for c in (32, 64, 64)])   # (parameters; group_norm_act computes)
            self.fc = nn.Linear(64 * 7 * 7, width)
            self.qkv = nn.Linear(width, 3 * width, bias=False)
            self.norm = nn.GroupNorm(heads, width)
            self.out = nn.Linear(width, width, bias=False)
            self.pi = nn.Linear(width, n_actions)
            self.vf = nn.Linear(width, 1)
            self.register_buffer("decay", head_decays(heads, "cpu"))
            for m in list(self.convs) + [self.fc]:
                nn.init.orthogonal_(m.weight, math.sqrt(2.0))
                nn.init.zeros_(m.bias)
            for m, gain in ((self.qkv, 1.0), (self.out, 1.0), (self.pi, 0.01), (self.vf, 1.0)):
                nn.init.orthogonal_(m.weight, gain)
            nn.init.zeros_(self.pi.bias)
            nn.init.zeros_(self.vf.bias)

        def initial_state(self, n: int):
            """The memories of n envs before anything: (n, heads, D, D) float32 zeros."""
            d = width // heads
            return torch.zeros(n, heads, d, d, device=self.decay.device)

        def _autocast(self):
            on = self.decay.is_cuda
            return torch.autocast("cuda" if on else "cpu", dtype=torch.bfloat16, enabled=on)

        def _features(self, obs_u8):
            """uint8 (B, k, 84, 84) -> the projected features and q, k, v of each, (B, 512) and (B, heads, D)."""
            if obs_u8.is_cuda:
                x = torch.empty(obs_u8.shape, dtype=torch.bfloat16, device=obs_u8.device, memory_format=torch.channels_last)
                policy_input(obs_u8.contiguous(), x)
            else:
                x = obs_u8.float().mul_(1.0 / 255.0)
            with self._autocast():
                for c, g in zip(self.convs, self.norms):
                    x = group_norm_act(c(x), g.num_groups, g.weight, g.bias, eps=g.eps, act="silu")
                h = F.silu(self.fc(x.flatten(1)))
                q, k, v = (y.unflatten(-1, (heads, -1)) for y in self.qkv(h).chunk(3, -1))
            return h, q, k, v

        def _heads(self, h, memory):
            with self._autocast():
                y = group_norm_act(memory.flatten(1), heads, self.norm.weight, self.norm.bias, eps=self.norm.eps, act="silu")
                h = h + self.out(y)
            h = h.float()
            return self.pi(h), self.vf(h).squeeze(-1)

        def forward(self, obs_u8, start=None, state=None):
            """A rollout: obs_u8 (T, N, k, 84, 84) uint8, start (T, N) bool and state (N, heads, D, D), the memories before it ->
            logits (T, N, A), values (T, N), the memories after it."""
            T, N = obs_u8.shape[:2]
            h, q, k, v = self._features(obs_u8.flatten(0, 1))
            out, state = linear_attention(*(y.unflatten(0, (T, N)) for y in (q, k, v)), self.decay, start, state)
            logits, value = self._heads(h, out.flatten(0, 1))
            return logits.unflatten(0, (T, N)), value.unflatten(0, (T, N)), state

        @torch.no_grad()
        def step(self, obs_u8, start, state):
            """One step: obs_u8 (N, k, 84, 84), start (N,) bool or None; state is updated. Logits (N, A), values (N,)."""
            h, q, k, v = self._features(obs_u8)
            return self._heads(h, linear_attention_step(q, k, v, self.decay, state, start))

        @torch.no_grad()
        def act(self, obs_u8, generator=None, start=None, state=None):
            """Action (Gumbel-max sample), its log-probability and the value, as NatureAC.act; state is updated."""
            logits, value = self.step(obs_u8, start, state)
            logp = F.log_softmax(logits, -1)
            u = torch.rand(logits.shape, generator=generator, device=logits.device).clamp_(1e-20, 1.0)
            a = (logp - torch.log(-torch.log(u))).argmax(-1)
            return a, logp.gather(-1, a[:, None]).squeeze(-1), value

    torch.manual_seed(seed)
    net = MemoryAC().to(device)
    if torch.device(device).type == "cuda":
        net = net.to(memory_format=torch.channels_last)
    return net
