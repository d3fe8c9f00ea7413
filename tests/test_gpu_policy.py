"""The policy's training step (nablaengine_b200/policy.py) through the CUDA step and the training operators: its
gradient against the same rollout with layer norm in elementary torch operations, and the clip's effect."""
import pytest

pytestmark = pytest.mark.gpu


def _norm(x, weight, bias, eps=1e-5):
    d = x - x.mean(-1, keepdim=True)
    return d * (d.square().mean(-1, keepdim=True) + eps).rsqrt() * weight + bias


def test_gradient_equals_the_plain_operators():
    """Both rollouts differ by float32 rounding alone. The step's own gradient carries a float32 error of up to 6e-4 of
    its size against 64 bits, so the two may differ by twice that per step; the bound is 1e-2 for two steps."""
    import torch
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    from nablaengine_b200 import policy
    inputs = policy.inputs_for(64, "cuda")
    grads = []
    for norm in (None, _norm):
        net = policy.make_policy((128, 64), device="cuda", layer_norm=norm)
        loss = policy.rollout_loss(net, inputs, 2)
        loss.backward()
        grads.append([p.grad for p in net.parameters()])
        assert torch.isfinite(loss)
    num = sum(float((a - b).double().square().sum()) for a, b in zip(*grads))
    den = sum(float(b.double().square().sum()) for b in grads[1])
    assert den > 0 and (num / den) ** 0.5 < 1e-2, (num / den) ** 0.5


def test_training_step_clips_and_updates():
    import torch
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    from nablaengine_b200 import policy
    inputs = policy.inputs_for(128, "cuda")
    net = policy.make_policy((64,), device="cuda")
    before = [p.detach().clone() for p in net.parameters()]
    opt = torch.optim.SGD(net.parameters(), lr=1.0)
    loss, norm, bad = policy.train_step(net, opt, inputs, 2, max_norm=1e-3)
    assert torch.isfinite(loss) and float(norm) > 1e-3 and int(bad) == 0
    moved = torch.stack([(p.detach() - b).double().norm() for p, b in zip(net.parameters(), before)]).norm()
    assert float(moved) == pytest.approx(1e-3, rel=1e-3)
