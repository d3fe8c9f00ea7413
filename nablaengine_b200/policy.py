"""A control policy trained through the differentiable control step: a small network reads each world's state (qpos,
qvel and the last ctrl), sets the PD setpoints of the next step, and learns from the gradient of a T-step rollout's loss.
It runs the training operators together as a learner uses them: the observation and every hidden layer are normalised by
torch_ffi.layer_norm, the rollout goes through torch_ffi.step, and the gradients, which contacts can make very large,
are clipped by their global norm with torch_ffi.clip_grad_norm before the optimiser's step. A world that diverges, in
its state or in its gradient, is left out before it enters the parameters' gradients, which are sums over the worlds.

  python -m nablaengine_b200.policy [--worlds 4096] [--steps 8] [--iterations 10] [--hidden 256,128]
"""
import json

from . import synthetic

NQ, NV, NU = 36, 35, 29
OBS = NQ + NV + NU


def _finite_rows(x):
    """(B, 1): the rows whose values are all finite (their sum is; one that overflows counts as lost too)."""
    return x.sum(dim=1, keepdim=True) * 0 == 0


def make_policy(hidden=(256, 128), seed=0, device="cpu", layer_norm=None):
    """A torch module: (qpos, qvel, last ctrl) -> setpoints' change. Normalised observation, then per hidden width a
    linear layer, a layer norm and an ELU, then a linear layer to the controls (small at the start, so that the first
    rollouts stand). A state that is not finite is seen as zeros: times its gradient, zero too, it would make the
    weights' gradients NaN. layer_norm: the operator (default torch_ffi.layer_norm; tests on CPU pass their own)."""
    import torch
    if layer_norm is None:
        from .torch_ffi import layer_norm

    class Norm(torch.nn.Module):
        def __init__(self, width):
            super().__init__()
            self.weight = torch.nn.Parameter(torch.ones(width))
            self.bias = torch.nn.Parameter(torch.zeros(width))

        def forward(self, x):
            return layer_norm(x, self.weight, self.bias)

    class Policy(torch.nn.Module):
        def __init__(self):
            super().__init__()
            layers, width = [Norm(OBS)], OBS
            for h in hidden:
                layers += [torch.nn.Linear(width, h), Norm(h), torch.nn.ELU()]
                width = h
            layers.append(torch.nn.Linear(width, NU))
            with torch.no_grad():
                layers[-1].weight.mul_(0.1)
                layers[-1].bias.zero_()
            self.layers = torch.nn.Sequential(*layers)

        def forward(self, qpos, qvel, ctrl):
            x = torch.cat([qpos, qvel, ctrl], dim=1)
            return self.layers(torch.where(_finite_rows(x), x, 0.0))

    with torch.random.fork_rng(devices=[]):
        torch.manual_seed(seed)
        return Policy().to(device)


def rollout_loss(policy, inputs, steps, step_fn=None, scale=0.2, kept=None, **step_kw):
    """The mean over steps and worlds of |qvel|^2 of `steps` closed-loop control steps from the inputs' states (qpos,
    qvel, warm, ctrl, friction, com): ctrl_t = the inputs' ctrl + scale * policy(state, ctrl_(t-1)). The loss of a world
    that diverges is not finite, and so is the mean; but where a step's gradient of a world's controls is not finite,
    the backward takes zeros for it, so the parameters' gradient is that of the other worlds. kept: a list that the
    backward appends the worlds (B, 1) to whose controls' gradient was finite, one tensor a step."""
    import torch
    if step_fn is None:
        from .torch_ffi import step as step_fn

    def finite_worlds(g):
        finite = _finite_rows(g)
        if kept is not None:
            kept.append(finite)
        return torch.where(finite, g, 0.0)

    q, v, w, base = (inputs[k] for k in ("qpos", "qvel", "warm", "ctrl"))
    ctrl, loss = base, 0.0
    for _ in range(steps):
        change = policy(q, v, ctrl)
        if change.requires_grad:
            change.register_hook(finite_worlds)
        ctrl = base + scale * change
        q, v, w = step_fn(q, v, w, ctrl, inputs["friction"], inputs["com"], **step_kw)
        loss = loss + (v * v).sum() / (steps * v.shape[0])
    return loss


def train_step(policy, optimizer, inputs, steps, max_norm=1.0, clip=None, **rollout_kw):
    """One update: the rollout's loss, its gradient, the clip and the optimiser's step. Returns (loss, norm, bad): 0-d
    tensors, the gradient's global norm before the clip, and what was not finite and is left out: the worlds' steps
    whose controls' gradient was not, and any values of the parameters' gradients themselves. clip: the operator
    (default torch_ffi.clip_grad_norm)."""
    import torch
    if clip is None:
        from .torch_ffi import clip_grad_norm as clip
    optimizer.zero_grad(set_to_none=True)
    kept = []
    loss = rollout_loss(policy, inputs, steps, kept=kept, **rollout_kw)
    loss.backward()
    norm, bad = clip([p.grad for p in policy.parameters() if p.grad is not None], max_norm, nonfinite="zero")
    optimizer.step()
    return loss.detach(), norm, bad + (~torch.cat(kept)).sum() if kept else bad


def inputs_for(worlds, device="cpu"):
    """The benchmark's seeded standing states as float32 tensors."""
    import torch
    return {k: torch.from_numpy(x).to(device) for k, x in synthetic.config_states("forward", B=worlds).items()}


def main(argv=None):
    import argparse
    import torch
    from . import torch_ffi
    ap = argparse.ArgumentParser()
    ap.add_argument("--worlds", type=int, default=4096)
    ap.add_argument("--steps", type=int, default=8, help="control steps of a rollout")
    ap.add_argument("--iterations", type=int, default=10)
    ap.add_argument("--hidden", default="256,128", help="the hidden layers' widths")
    ap.add_argument("--max-norm", type=float, default=1.0)
    ap.add_argument("--lr", type=float, default=3e-4)
    a = ap.parse_args(argv)
    torch_ffi.init()
    dev = torch.device("cuda", torch.cuda.current_device())
    policy = make_policy(tuple(int(h) for h in a.hidden.split(",")), device=dev)
    optimizer = torch.optim.Adam(policy.parameters(), lr=a.lr, fused=True)
    inputs = inputs_for(a.worlds, dev)
    rows, times = [], []
    for _ in range(a.iterations):
        e0, e1 = (torch.cuda.Event(enable_timing=True) for _ in range(2))
        e0.record()
        rows.append(train_step(policy, optimizer, inputs, a.steps, a.max_norm))
        e1.record()
        times.append((e0, e1))
    torch.cuda.synchronize()
    ms = sorted(e0.elapsed_time(e1) for e0, e1 in times)
    print(json.dumps({"worlds": a.worlds, "steps": a.steps, "iterations": a.iterations,
                      "ms_per_iteration": ms[len(ms) // 2], "loss": [float(r[0]) for r in rows],
                      "grad_norm": [float(r[1]) for r in rows], "nonfinite": [int(r[2]) for r in rows]}), flush=True)


if __name__ == "__main__":
    main()
