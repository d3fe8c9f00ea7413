"""Host logic of the policy's training step (nablaengine_b200/policy.py) on CPU, the operators stood in for by their
definitions in torch and the control step by a small differentiable map."""
import torch

from nablaengine_b200 import policy


def _norm(x, weight, bias, eps=1e-5):
    d = x - x.mean(-1, keepdim=True)
    return d / (d.square().mean(-1, keepdim=True) + eps).sqrt() * weight + bias


def _step(q, v, w, ctrl, friction, com):
    u = torch.nn.functional.pad(ctrl, (6, 0))
    v1 = 0.9 * v - 0.2 * u * friction[:, None] + 0.01 * com.sum(1, keepdim=True)
    return q + 0.005 * torch.nn.functional.pad(v1, (0, 1)), v1, w


def _clip(grads, max_norm, nonfinite):
    bad = sum(int((~torch.isfinite(g)).sum()) for g in grads)
    for g in grads:
        g.copy_(torch.nan_to_num(g, nan=0.0, posinf=0.0, neginf=0.0))
    norm = torch.stack([g.norm() for g in grads]).norm()
    for g in grads:
        g.mul_(min(1.0, max_norm / (float(norm) + 1e-6)))
    return norm, torch.tensor(bad)


def test_training_lowers_the_loss_and_clips():
    net = policy.make_policy((32, 16), layer_norm=_norm)
    inputs = policy.inputs_for(12)
    opt = torch.optim.Adam(net.parameters(), lr=1e-2)
    losses = []
    for _ in range(20):
        loss, norm, bad = policy.train_step(net, opt, inputs, 3, max_norm=0.1, clip=_clip, step_fn=_step)
        total = torch.stack([p.grad.norm() for p in net.parameters()]).norm()
        assert float(total) <= 0.1 * (1 + 1e-5) and float(norm) > 0 and int(bad) == 0
        losses.append(float(loss))
    assert losses[-1] < losses[0]


def test_the_policy_is_the_seeds():
    a, b, c = (policy.make_policy((8,), seed=s, layer_norm=_norm) for s in (3, 3, 4))
    x = policy.inputs_for(2)
    args = (x["qpos"], x["qvel"], x["ctrl"])
    assert torch.equal(a(*args), b(*args)) and not torch.equal(a(*args), c(*args))
    assert a(*args).shape == (2, 29)
