"""A world that diverges takes no other world's gradient with it: the policy's update is that of the remaining worlds."""
import pytest
import torch

from nablaengine_b200 import policy

from test_policy_cpu import _clip, _norm, _step

WORLDS, LOST = 12, 7


class _Spoiled(torch.autograd.Function):
    """The identity whose cotangent's row LOST becomes `value`."""

    @staticmethod
    def forward(ctx, x, value):
        ctx.value = value
        return x.view_as(x)

    @staticmethod
    def backward(ctx, g):
        g = g.clone()
        g[LOST, 13:15] = ctx.value
        return g, None


def _step_that_loses(where, value):
    """A control step that loses world LOST: its state, from the second step on, or its gradient alone, at every step, or
    at the last one."""
    calls = []

    def step(q, v, w, ctrl, friction, com):
        calls.append(1)
        q, v, w = _step(q, v, w, ctrl, friction, com)
        if q.shape[0] < WORLDS:
            return q, v, w
        if where == "state" and len(calls) > 1:
            q, v = q.clone(), v.clone()
            q[LOST], v[LOST] = q[LOST] * value, v[LOST] * value
        if where == "gradient" or (where == "last gradient" and len(calls) == 3):
            v = _Spoiled.apply(v, value)
        return q, v, w
    return step


def _grads(inputs, where, value):
    net = policy.make_policy((32, 16), layer_norm=_norm).double()
    inputs = {k: x.double() for k, x in inputs.items()}
    opt = torch.optim.SGD(net.parameters(), lr=1.0)
    before = [p.detach().clone() for p in net.parameters()]
    loss, norm, bad = policy.train_step(net, opt, inputs, 3, max_norm=float("inf"), clip=_clip,
                                        step_fn=_step_that_loses(where, value))
    return [b - p.detach() for b, p in zip(before, net.parameters())], norm, bad


@pytest.mark.parametrize("value", [float("nan"), float("inf")])
@pytest.mark.parametrize("where", ["state", "gradient", "last gradient"])
def test_the_update_is_the_remaining_worlds(where, value):
    """Both are sums over the worlds and steps of the same terms in 64 bits, added up in other orders: far below 1e-5 of
    the largest. The loss is a mean over all worlds, so the remaining ones' own mean counts 11/12."""
    inputs = policy.inputs_for(WORLDS)
    rest = [k for k in range(WORLDS) if k != LOST]
    got, norm, bad = _grads(inputs, where, value)
    want, _, none = _grads({k: x[rest] for k, x in inputs.items()}, where, value)
    assert int(none) == 0 and int(bad) > 0 and torch.isfinite(norm)
    for a, b in zip(got, want):
        b = b * (WORLDS - 1) / WORLDS
        assert torch.isfinite(a).all() and b.abs().max() > 0
        assert float((a - b).abs().max()) <= 1e-5 * float(b.abs().max())


def test_a_state_that_starts_non_finite():
    inputs = policy.inputs_for(WORLDS)
    rest = [k for k in range(WORLDS) if k != LOST]
    spoiled = {k: x.clone() for k, x in inputs.items()}
    spoiled["qvel"][LOST, 11] = float("nan")
    got, _, bad = _grads(spoiled, "", 0.0)
    want, _, _ = _grads({k: x[rest] for k, x in inputs.items()}, "", 0.0)
    assert int(bad) > 0
    for a, b in zip(got, want):
        b = b * (WORLDS - 1) / WORLDS
        assert float((a - b).abs().max()) <= 1e-5 * float(b.abs().max())
