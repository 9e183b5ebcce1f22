"""A recurrent memory beside the simulator: one memory block learns, from the observations of whole rollouts, to
estimate what only the critic is given (the 32 privileged inputs of MDN_BUF_CO), and is then stepped tick by tick as a
deployed policy would.

    block_norm -> projections -> delta_rule -> projection -> block_norm (gate, residual scale) -> estimate

A rollout's arrays are used where the simulator has them, [steps][envs][...] on the GPU. Episode ends clear the memory
through `starts`; the memory's state is carried from one rollout to the next.

    python examples/memory_policy.py [--envs 512] [--horizon 64] [--rollouts 6]
"""
import argparse
import importlib
import pathlib
import sys

import torch

sys.path.insert(0, str(pathlib.Path(__file__).resolve().parents[1]))
mdn = importlib.import_module("metal-drone-nav_b200")

OBS, PRIVILEGED = 184, 32


class DeviceArray:
    """A simulator buffer for torch.as_tensor, without a copy."""

    def __init__(self, sim, name, shape, typestr):
        self.__cuda_array_interface__ = dict(shape=shape, typestr=typestr, data=(sim.buffer(name)[0], False), version=3)


def rollout_tensor(sim, name, width, typestr="<f4"):
    shape = (sim.horizon, sim.n) + ((width,) if width else ())
    return torch.as_tensor(DeviceArray(sim, name, shape, typestr), device="cuda")


class MemoryEstimator(torch.nn.Module):
    def __init__(self, dim=128, heads=4, key=32):
        super().__init__()
        self.dim, self.heads, self.key = dim, heads, key
        self.embed = torch.nn.Linear(OBS, dim)
        self.project = torch.nn.Linear(dim, 3 * heads * key + dim)     # queries, keys, values, gate
        self.rates = torch.nn.Linear(dim, 2 * heads)                    # log-decay and beta, before their functions
        self.out = torch.nn.Linear(heads * key, dim)
        self.estimate = torch.nn.Linear(dim, PRIVILEGED)
        for name in ("norm_in", "norm_branch", "norm_out"):
            self.register_parameter(name, torch.nn.Parameter(torch.ones(dim)))
        self.residual_scale = torch.nn.Parameter(torch.full((dim,), 0.5))
        torch.nn.init.constant_(self.rates.bias[:heads], -3.0)          # remember some twenty steps at first

    def inputs(self, y):
        """Everything the memory takes, as slices of one projection."""
        size = self.heads * self.key
        qkvg = self.project(y)
        q, k, v = (qkvg[..., i * size:(i + 1) * size].unflatten(-1, (self.heads, self.key)) for i in range(3))
        rates = self.rates(y)
        log_decay = -torch.nn.functional.softplus(rates[..., :self.heads])
        return q, k, v, log_decay, torch.sigmoid(rates[..., self.heads:]), qkvg[..., 3 * size:]

    def rollout(self, obs, starts, state):
        """obs [steps, envs, 184] -> estimates [steps, envs, 32] and the memory after the last step."""
        steps, envs = obs.shape[:2]
        x = self.embed(obs).reshape(steps * envs, self.dim)
        x, y = mdn.block_norm_train(x, norm_weight=self.norm_in)
        q, k, v, log_decay, beta, gate = self.inputs(y.reshape(steps, envs, self.dim))
        memory, state = mdn.delta_rule_train(q, k, v, log_decay, beta, state, starts=starts)
        branch = self.out(memory.reshape(steps * envs, -1))
        _, y = mdn.block_norm_train(x, branch, gate.reshape(steps * envs, self.dim), self.norm_branch,
                                    self.residual_scale, self.norm_out, gate_act="silu")
        return self.estimate(y).reshape(steps, envs, PRIVILEGED), state

    @torch.no_grad()
    def tick(self, obs, starts, state):
        """obs [envs, 184] -> estimates [envs, 32]; the memory is stepped in place."""
        x = self.embed(obs)
        y = mdn.block_norm(x, norm_weight=self.norm_in)[1]
        q, k, v, log_decay, beta, gate = self.inputs(y)
        memory, _ = mdn.delta_step(q, k, v, log_decay, beta, state, starts=starts)
        branch = self.out(memory.reshape(len(obs), -1))
        y = mdn.block_norm(x, branch, gate, self.norm_branch, self.residual_scale, self.norm_out, gate_act="silu")[1]
        return self.estimate(y)


def run(envs=512, horizon=64, rollouts=6, seed=3, updates=4, report=print):
    """Losses of each rollout before it is learnt from, and how far ticks are from the rollout's estimates."""
    torch.manual_seed(seed)
    device = mdn.Device(0)
    sim = mdn.Sim(device, mdn.layouts.default_config(n=envs, family=17, seed=seed), horizon)
    try:
        obs, target = rollout_tensor(sim, "obs", OBS), rollout_tensor(sim, "co", PRIVILEGED)
        ended = [rollout_tensor(sim, name, 0, "|u1") for name in ("terminated", "truncated")]
        model = MemoryEstimator().cuda()
        optimizer = torch.optim.Adam(model.parameters(), lr=2e-3)
        state = torch.zeros(envs, model.heads, model.key, model.key, device="cuda")
        last = torch.ones(envs, dtype=torch.uint8, device="cuda")  # every environment begins an episode
        losses = []
        for index in range(rollouts):
            sim.collect()
            device.finish()  # the buffers are complete before torch's stream reads them
            ends = ended[0] | ended[1]
            starts = torch.cat([last[None], ends[:-1]])
            for update in range(updates):
                estimate, after = model.rollout(obs, starts, state)
                loss = ((estimate - target) ** 2).mean()
                if update == 0:
                    losses.append(loss.item())
                optimizer.zero_grad()
                loss.backward()
                optimizer.step()
            report(f"rollout {index}: loss {losses[-1]:.4f}")
            if index + 1 < rollouts:
                state, last = after.detach(), ends[-1].clone()
        with torch.no_grad():
            whole, after = model.rollout(obs, starts, state)
        memory = state.clone()
        ticks = torch.stack([model.tick(obs[t], starts[t], memory) for t in range(horizon)])
        off = ((ticks - whole).norm() / whole.norm()).item(), ((memory - after).norm() / after.norm()).item()
        report(f"tick by tick: estimates off by {off[0]:.2g}, memory by {off[1]:.2g}")
        torch.cuda.synchronize()
        return losses, off
    finally:
        sim.close()
        device.close()


if __name__ == "__main__":
    parser = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    for name, value in (("envs", 512), ("horizon", 64), ("rollouts", 6)):
        parser.add_argument(f"--{name}", type=int, default=value)
    run(**vars(parser.parse_args()))
