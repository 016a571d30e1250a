"""A Neural Particle Automaton trained with its MLP's inputs kept in 8 bits, then rolled out in 8-bit integers.

A cloud of particles is trained to take on a colour pattern given by position: each training step rolls the
automaton out for ``--steps`` steps and propagates back through all of them.  The run is made twice, with what
the MLP keeps between forward and backward in float32 and in 8 bits (``step_euler(..., checkpoint="int8")``), and
prints the loss, the memory that a rollout holds and the time of a training step of both.  The trained model is
then stepped with its MLP as products of 8-bit integers (``int8.Int8Mlp``) beside the float32 one.

    python examples/eight_bit_rollout.py [--particles 65536] [--steps 16] [--epochs 60]
"""
import argparse
import math
import os
import sys
import time

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
import npa_amd.sphops as sphops  # noqa: E402
from npa_amd import int8, step  # noqa: E402

CHANNELS, HIDDEN = 16, 128


class Automaton(torch.nn.Module):
    """What ``step_euler`` reads of the reference's NPA module (models/npa.py:15-78), in 2D."""

    def __init__(self):
        super().__init__()
        self.spatial_dims = 2
        self.register_buffer("eps0", torch.tensor([0.1]))
        self.register_buffer("alpha", torch.tensor([0.05]))
        self.state_grad = self.density_grad = self.log_norm_grad = self.log_norm_density_grad = True
        self.stopgrad_pos, self.stopgrad_state = True, False
        width = 2 * CHANNELS + 2 * CHANNELS + 2
        self.model = torch.nn.Sequential(torch.nn.Linear(width, HIDDEN), torch.nn.ReLU(),
                                         torch.nn.Linear(HIDDEN, 2 + CHANNELS, bias=False))
        torch.nn.init.zeros_(self.model[2].weight)


def cloud(n, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    r, t = (torch.rand(1, n, device="cuda", generator=gen) for _ in range(2))
    r, t = r.sqrt(), 2 * math.pi * t
    x = torch.stack((r * t.cos(), r * t.sin()), -1)
    s = 0.1 * torch.randn(1, n, CHANNELS, device="cuda", generator=gen)
    s[..., 3:5] = x  # where a particle starts, in two of its states
    return x, s


def rollout(model, grid, x, s, steps, checkpoint=None):
    for _ in range(steps):
        x, s, _ = step.step_euler(model, x, s, grid, dt=0.5, update_prob=1.0, checkpoint=checkpoint)
    return x, s


def target(x):
    return torch.stack((torch.sin(3 * x[..., 0]), torch.cos(3 * x[..., 1]), x[..., 0] * x[..., 1]), -1)


def train(grid, n, steps, epochs, checkpoint):
    torch.manual_seed(0)
    model = Automaton().cuda()
    opt = torch.optim.Adam(model.parameters(), lr=5e-3)
    x0, s0 = cloud(n, 1)
    for epoch in range(epochs):
        torch.cuda.synchronize()
        start, held = time.perf_counter(), torch.cuda.memory_allocated()
        x, s = rollout(model, grid, x0, s0, steps, checkpoint)
        loss = (s[..., :3] - target(x)).square().mean()
        held = torch.cuda.memory_allocated() - held
        opt.zero_grad()
        loss.backward()
        torch.nn.utils.clip_grad_norm_(model.parameters(), 1.0)
        opt.step()
        torch.cuda.synchronize()
        took = time.perf_counter() - start
    print(f"checkpoint={checkpoint}: loss {loss.item():.4f}, a rollout holds {held / 2 ** 20:.0f} MiB, "
          f"a training step takes {took * 1e3:.1f} ms", flush=True)
    return model


def main():
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    ap.add_argument("--particles", type=int, default=65536)
    ap.add_argument("--steps", type=int, default=16)
    ap.add_argument("--epochs", type=int, default=60)
    a = ap.parse_args()
    eps = 0.0692 * math.sqrt(4096 / a.particles)  # about 20 neighbours a particle
    cells = 2 * math.ceil(1.2 / eps)
    grid = sphops.HashGrid(dim=2, boundary="clamped", mode="grid", grid_size=(cells, cells), eps=eps,
                           num_particles=a.particles, batch_size=1, max_particles_per_block=32)
    train(grid, a.particles, a.steps, a.epochs, None)
    model = train(grid, a.particles, a.steps, a.epochs, "int8")

    x0, s0 = cloud(a.particles, 2)
    exact = model.model
    results = []
    with torch.no_grad():
        for name, mlp in (("float32", exact), ("8-bit integers", int8.Int8Mlp(exact))):
            model.model = mlp
            for _ in range(2):  # the first sizes the neighbour lists
                torch.cuda.synchronize()
                start = time.perf_counter()
                x, s = rollout(model, grid, x0, s0, a.steps)
                torch.cuda.synchronize()
                took = time.perf_counter() - start
            results.append((s[..., :3] - target(x)).square().mean().item())
            print(f"rollout in {name}: loss on another cloud {results[-1]:.4f}, {took * 1e3 / a.steps:.2f} ms a step",
                  flush=True)


if __name__ == "__main__":
    main()
