"""A policy with frozen parameters, which have no gradient, trains its others."""
import torch

from nablaengine_b200 import policy

from test_policy_cpu import _clip, _norm, _step


def test_frozen_parameters_are_left_out_of_the_clip():
    net = policy.make_policy((16,), layer_norm=_norm)
    params = list(net.parameters())
    for p in params[:3]:
        p.requires_grad_(False)
    before = [p.detach().clone() for p in params]
    given = []

    def clip(grads, max_norm, nonfinite):
        given.append(len(grads))
        assert all(isinstance(g, torch.Tensor) for g in grads)
        return _clip(grads, max_norm, nonfinite)

    opt = torch.optim.SGD([p for p in params if p.requires_grad], lr=1.0)
    policy.train_step(net, opt, policy.inputs_for(4), 2, clip=clip, step_fn=_step)
    assert given == [len(params) - 3]
    assert [torch.equal(a, p.detach()) for a, p in zip(before, params)] == [k < 3 for k in range(len(params))]
