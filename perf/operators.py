"""The training operators around the differentiable control step, as measured cases: layer norm (forward, and backward
with the weight and bias gradients) and the global gradient norm with clipping. `own` false: the plain form in
elementary torch operations; true: the calls of nablaengine_b200.torch_ffi.

Sizes: 100 is a policy's observation of the step's state (36 qpos + 35 qvel + 29 ctrl), 4096 and 32768 the benchmark's
and the rollout's worlds per GPU, 32 the rollout's steps, 29 the controls; the layer widths are generic.
"""
import math

import torch

own = False

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
EPS, CLIP_EPS = 1e-5, 1e-6
# a policy (observation norm, then linear layers with a norm after each hidden one) of hidden widths 128, 128, and a
# policy with its critic of hidden widths 512, 256, 128
SMALL_POLICY = "100;100;128x100;128;128;128;128x128;128;128;128;29x128;29"
ACTOR_CRITIC = ("100;100;512x100;512;512;512;256x512;256;256;256;128x256;128;128;128;29x128;29;"
                "512x100;512;512;512;256x512;256;256;256;128x256;128;128;128;1x128;1")
WIDE_BLOCK = "4096x1024;4096;1024x4096;1024"


def _norm(name, op, rows, cols, dtype, affine="f32", pad=0):
    """A layer norm case: `affine` is the type of weight and bias ("" for none, "same" for x's), `pad` the columns of a
    wider buffer that x's rows skip."""
    return {"name": name, "op": op, "rows": rows, "cols": cols, "dtype": dtype, "affine": affine, "pad": pad}


def _clip(name, shapes, repeat, dtype, out, nonfinite, max_norm):
    """A clipping case: the gradients' shapes, `repeat` times over, their type, the type of the clipped copies, what is
    done with non-finite values, and the bound."""
    return {"name": name, "op": "clip", "shapes": shapes, "repeat": repeat, "dtype": dtype, "out": out,
            "nonfinite": nonfinite, "max_norm": max_norm}


def listed():
    return [
        # one robot's policy step: a hidden layer for a single world, latency alone
        _norm("forward 1x512 f32", "forward", 1, 512, "f32"),
        # the observations of the benchmark's 4096 worlds, a width that no vector length divides into warps
        _norm("forward 4096x100 f32", "forward", 4096, 100, "f32"),
        # a hidden layer over all 32 steps of 4096 worlds
        _norm("forward 131072x512 bf16", "forward", 131072, 512, "bf16"),
        # a wide layer with parameters in x's type
        _norm("forward 8192x8192 bf16", "forward", 8192, 8192, "bf16", "same"),
        # the gradients of the cases above, and an odd width
        _norm("backward 4096x100 f32", "backward", 4096, 100, "f32"),
        _norm("backward 131072x512 f32", "backward", 131072, 512, "f32"),
        _norm("backward 8192x8192 bf16", "backward", 8192, 8192, "bf16", "same"),
        _norm("backward 5000x1001 f16", "backward", 5000, 1001, "f16"),
        # the gradients of a small policy: the latency of many short tensors
        _clip("clip small policy f32", SMALL_POLICY, 1, "f32", "f32", "keep", 1.0),
        # a policy and its critic trained in bf16, the clipped gradients going to float32
        _clip("clip actor-critic bf16", ACTOR_CRITIC, 1, "bf16", "f32", "keep", 0.5),
        # the rollout's ctrl gradient over 32 steps of 32768 worlds, its non-finite values zeroed
        _clip("clip ctrl gradient f32", "32x32768x29", 1, "f32", "f32", "zero", 10.0),
        # a large model's gradients, twice the size of the second-level cache
        _clip("clip 100M bf16", WIDE_BLOCK, 12, "bf16", "bf16", "keep", 1.0),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    dtype = rng.choice(["f32", "bf16", "f16"])
    op = rng.choice(["forward", "backward", "clip", "norm"])
    if op in ("forward", "backward"):
        # (below 4 columns the input's gradient is what eps leaves of terms that cancel: nothing a sum in 32 bits holds)
        cols = _log_int(rng, 1 if op == "forward" else 4, 16384)
        rows = _log_int(rng, 1, min(262144, 60_000_000 // cols))
        affine = rng.choice(["", "f32", "same"])
        return {k: v for k, v in _norm("", op, rows, cols, dtype, affine, rng.choice([0, 0, 1, 8, 37])).items()
                if k != "name"}
    count = _log_int(rng, 1, 60)
    each = max(1, _log_int(rng, 1000, 90_000_000) // count)
    shapes = ";".join(str(max(1, int(each * rng.uniform(0.1, 1.0)))) for _ in range(count))
    # (gradients in f16 carry a loss scale, and so does their bound)
    case = _clip("", shapes, 1, dtype, rng.choice([dtype, "f32"]), rng.choice(["keep", "zero"]),
                 rng.choice([0.5, 1.0, 10.0, 1e6]) * (1024.0 if dtype == "f16" else 1.0))
    case["op"] = op
    return {k: v for k, v in case.items() if k != "name"}


def _shapes(case):
    one = [tuple(int(n) for n in s.split("x")) for s in case["shapes"].split(";")]
    return one * case["repeat"]


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)

    def randn(*shape):
        return torch.randn(shape, device="cuda", generator=gen)

    s = dict(case)
    dtype = DTYPES[case["dtype"]]
    if case["op"] in ("forward", "backward"):
        rows, cols, pad = case["rows"], case["cols"], case["pad"]
        # columns of different scale and offset, as joint angles, heights and velocities side by side have
        scale = torch.exp(randn(cols + pad) * 0.5)
        x = torch.addcmul(randn(cols + pad) * 0.5, randn(rows, cols + pad), scale).to(dtype)
        s["x"] = x[:, :cols]
        kind = dtype if case["affine"] == "same" else torch.float32
        s["weight"] = (1.0 + 0.2 * randn(cols)).to(kind) if case["affine"] else None
        s["bias"] = (0.1 * randn(cols)).to(kind) if case["affine"] else None
        if case["op"] == "backward":
            # the cotangent of a loss averaged over the rows (in f16 with a loss scale that takes the average out)
            s["g_y"] = (randn(rows, cols) * (1.0 if dtype == torch.float16 else 1.0 / rows)).to(dtype)
            d = s["x"].double()
            s["mean"] = d.mean(-1).float()
            s["rstd"] = (d.var(-1, unbiased=False) + EPS).rsqrt().float()
        return s
    # gradients of one step: each tensor with a scale of its own
    s["grads"] = [(randn(*shape) * math.exp((k % 7) - 3.0) * 0.1).to(dtype) for k, shape in enumerate(_shapes(case))]
    if case["nonfinite"] == "zero":
        for g in s["grads"][:3]:  # worlds whose gradient through the contacts overflowed
            at = torch.randint(0, g.numel(), (1 + g.numel() // 100000,), device="cuda", generator=gen)
            g.view(-1)[at] = float("inf")
            g.view(-1)[at[: 1 + at.numel() // 2]] = float("nan")
    s["outs"] = [torch.empty(g.shape, dtype=DTYPES[case["out"]], device="cuda") for g in s["grads"]]
    return s


def run(s):
    op = s["op"]
    if own:
        from nablaengine_b200 import torch_ffi
        if op == "forward":
            return torch_ffi.layer_norm_forward(s["x"], s["weight"], s["bias"], EPS)
        if op == "backward":
            return torch_ffi.layer_norm_backward(s["g_y"], s["x"], s["mean"], s["rstd"], s["weight"], s["bias"])
        if op == "norm":
            return torch_ffi.grad_norm(s["grads"], nonfinite=s["nonfinite"])
        norm, bad = torch_ffi.clip_grad_norm(s["grads"], s["max_norm"], eps=CLIP_EPS, nonfinite=s["nonfinite"],
                                             out=s["outs"])
        return norm, bad, s["outs"]
    if op == "forward":
        return _plain_forward(s["x"], s["weight"], s["bias"])
    if op == "backward":
        return _plain_backward(s["g_y"], s["x"], s["mean"], s["rstd"], s["weight"], s["bias"])
    return _plain_clip(s["grads"], s["outs"], s["max_norm"], s["nonfinite"], op == "norm")


def _plain_forward(x, weight, bias):
    f = x.float()
    mean = f.mean(-1)
    d = f - mean[:, None]
    rstd = (d.square().mean(-1) + EPS).rsqrt()
    y = d * rstd[:, None]
    if weight is not None:
        y = y * weight.float() + bias.float()
    return y.to(x.dtype), mean, rstd


def _plain_backward(g_y, x, mean, rstd, weight, bias):
    g = g_y.float()
    xh = (x.float() - mean[:, None]) * rstd[:, None]
    h = g if weight is None else g * weight.float()
    gx = (h - h.mean(-1, keepdim=True) - xh * (h * xh).mean(-1, keepdim=True)) * rstd[:, None]
    if weight is None:
        return gx.to(x.dtype), None, None
    return gx.to(x.dtype), (g * xh).sum(0).to(weight.dtype), g.sum(0).to(bias.dtype)


def _plain_clip(grads, outs, max_norm, nonfinite, norm_only):
    flat = torch.cat([g.reshape(-1) for g in grads]).float()
    finite = torch.isfinite(flat)
    bad = (~finite).sum()
    if nonfinite == "zero":
        flat = torch.where(finite, flat, torch.zeros_like(flat))
    norm = flat.square().sum().sqrt()
    if norm_only:
        return norm, bad
    flat = flat * (max_norm / (norm + CLIP_EPS)).clamp(max=1.0)
    parts = flat.split([g.numel() for g in grads])
    return norm, bad, [o.copy_(p.view(o.shape)) for o, p in zip(outs, parts)]


def work(case):
    size = {"f32": 4, "bf16": 2, "f16": 2}
    if case["op"] in ("forward", "backward"):
        rows, cols, e = case["rows"], case["cols"], size[case["dtype"]]
        par = {"": 0, "f32": 4, "same": e}[case["affine"]]
        if case["op"] == "forward":
            return {"bytes": rows * cols * 2 * e + 8 * rows + 2 * par * cols, "flops": 8 * rows * cols}
        return {"bytes": rows * cols * 3 * e + 8 * rows + 3 * par * cols, "flops": 14 * rows * cols}
    n = sum(math.prod(shape) for shape in _shapes(case))
    if case["op"] == "norm":
        return {"bytes": n * size[case["dtype"]] + 12, "flops": 2 * n}
    return {"bytes": n * (size[case["dtype"]] + size[case["out"]]) + 12, "flops": 3 * n}


def exact(case, seed):
    """The definitions in 64 bits: deviations from the row's mean over its standard deviation; the gradient as the
    cotangent with its components along the constant vector and along the normalised row taken out; the root of the
    tensors' summed squares and the gradients times the clip coefficient."""
    s = prepare(case, seed)
    if case["op"] == "forward":
        x = s["x"].double()
        n = x.shape[1]
        mean = torch.einsum("ij->i", x) / n
        x = x - mean.unsqueeze(1)
        rstd = 1.0 / torch.sqrt(torch.einsum("ij,ij->i", x, x) / n + EPS)
        y = torch.einsum("ij,i->ij", x, rstd)
        if s["weight"] is not None:
            y = torch.addcmul(s["bias"].double(), y, s["weight"].double())
        return y, mean, rstd
    if case["op"] == "backward":
        n = s["x"].shape[1]
        g, rstd = s["g_y"].double(), s["rstd"].double()
        z = torch.einsum("ij,i->ij", s["x"].double().sub_(s["mean"].double().unsqueeze(1)), rstd)
        gw = gb = None
        if s["weight"] is not None:
            gw, gb = torch.einsum("ij,ij->j", g, z), torch.einsum("ij->j", g)
            g = torch.einsum("ij,j->ij", g, s["weight"].double())
        along = torch.einsum("ij,ij->i", g, z) / n
        level = torch.einsum("ij->i", g) / n
        gx = g.sub_(level.unsqueeze(1)).sub_(z.mul_(along.unsqueeze(1)))
        return gx.mul_(rstd.unsqueeze(1)), gw, gb
    grads = [g.double().flatten() for g in s["grads"]]
    bad = sum(int((g.isnan() | g.isinf()).sum()) for g in grads)
    if case["nonfinite"] == "zero":
        grads = [torch.nan_to_num(g, nan=0.0, posinf=0.0, neginf=0.0) for g in grads]
    norm = math.sqrt(math.fsum(float(torch.dot(g, g)) for g in grads))
    told = torch.tensor(norm, dtype=torch.float64)
    if case["op"] == "norm":
        return told, bad
    c = min(1.0, case["max_norm"] / (norm + CLIP_EPS))
    return told, bad, [(g * c).view(t.shape) for g, t in zip(grads, s["grads"])]
