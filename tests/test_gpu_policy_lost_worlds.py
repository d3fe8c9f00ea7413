"""A world that diverges takes no other world's gradient with it, through the CUDA step and the training operators."""
import pytest

pytestmark = pytest.mark.gpu


def test_the_gradient_is_the_remaining_worlds():
    """Both rollouts of the remaining worlds differ by float32 rounding alone (the order of the sums over the worlds);
    the step's own gradient carries up to 6e-4 of its size against 64 bits, so 1e-2 of its size for two steps, as in
    test_gpu_policy.py. The loss is a mean over all worlds, so the remaining ones' own mean counts 63/64."""
    import torch
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    from nablaengine_b200 import policy
    inputs = policy.inputs_for(64, "cuda")
    rest = [k for k in range(64) if k != 41]
    spoiled = {k: x.clone() for k, x in inputs.items()}
    spoiled["qvel"][41, 8] = float("nan")

    def grads(states):
        net = policy.make_policy((128, 64), device="cuda")
        before = [p.detach().clone() for p in net.parameters()]
        opt = torch.optim.SGD(net.parameters(), lr=1.0)
        _, norm, bad = policy.train_step(net, opt, states, 2, max_norm=float("inf"))
        return [b - p.detach() for b, p in zip(before, net.parameters())], norm, bad

    got, norm, bad = grads(spoiled)
    want, _, none = grads({k: x[rest].contiguous() for k, x in inputs.items()})
    assert int(bad) > 0 and int(none) == 0 and torch.isfinite(norm) and float(norm) > 0
    num = sum(float((a - b * 63 / 64).double().square().sum()) for a, b in zip(got, want))
    den = sum(float((b * 63 / 64).double().square().sum()) for b in want)
    assert den > 0 and (num / den) ** 0.5 < 1e-2, (num / den) ** 0.5
