"""A policy with a memory, trained for a few updates: rollouts of HipVecEnv under `make_memory_net`, then PPO's clipped loss over
whole sequences of the stored rollout, minibatch by minibatch of envs.

    python examples/memory_policy.py [--rom PATH] [--envs 256] [--steps 64] [--updates 4] [--device cuda]
"""
import argparse
import os
import sys
import time

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
sys.path.insert(0, os.path.join(ROOT, "fast-mario-env_amd"))

import torch  # noqa: E402

from fast_mario_env_amd import HipVecEnv  # noqa: E402
from fast_mario_env_amd.memory import make_memory_net  # noqa: E402
from fast_mario_env_amd.rollout import Rollout  # noqa: E402


def update(net, opt, ro, minibatches=4, clip=0.2):
    """One pass over the rollout, a share of the envs at a time; the mean loss (a tensor: nothing here waits for the GPU)."""
    adv, ret = ro.advantages()
    adv = (adv - adv.mean()) / (adv.std() + 1e-8)
    total = 0.0
    for envs in torch.randperm(ro.env.n, device=adv.device).chunk(minibatches):
        logits, value, _ = net(*ro.sequence(envs))
        logp = torch.log_softmax(logits, -1).gather(-1, ro.act[:, envs, None]).squeeze(-1)
        ratio, a = (logp - ro.logp[:, envs]).exp(), adv[:, envs]
        loss = -torch.minimum(ratio * a, ratio.clamp(1 - clip, 1 + clip) * a).mean() + 0.5 * (value - ret[:, envs]).square().mean()
        opt.zero_grad(set_to_none=True)
        loss.backward()
        torch.nn.utils.clip_grad_norm_(net.parameters(), 0.5)
        opt.step()
        total = total + loss.detach()
    return total / minibatches


def main():
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    ap.add_argument("--rom", default=os.path.join(ROOT, "tests", "golden", "roms", "mini_smb_vanilla.nes"))
    ap.add_argument("--envs", type=int, default=256)
    ap.add_argument("--steps", type=int, default=64)
    ap.add_argument("--updates", type=int, default=4)
    ap.add_argument("--device", default="cuda")
    args = ap.parse_args()
    with open(args.rom, "rb") as f:
        env = HipVecEnv("1-1", args.envs, seed=0, sticky=0.25, noop_max=30, maxpool=True, rom=f.read(), device=args.device)
    env.reset()
    net = make_memory_net(device=args.device)
    opt = torch.optim.Adam(net.parameters(), 2.5e-4)
    ro = Rollout(env, net, T=args.steps)
    for i in range(args.updates):
        t0 = time.perf_counter()
        ro.collect()
        loss = float(update(net, opt, ro))
        print(f"update {i}: loss {loss:.4f}, mean reward a step {ro.rew.mean().item():.3f}, {time.perf_counter() - t0:.2f} s", flush=True)
    env.close()


if __name__ == "__main__":
    main()
