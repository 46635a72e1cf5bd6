"""Group norm and the pointwise product in 64 bits, on the CPU, with bounds on how far float32 sums and one rounding
to the output's type may take a result from them."""
import math

import torch

U32 = 2.0 ** -24                                       # unit roundoffs
UNIT = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
TINY = {torch.float32: 2.0 ** -149, torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -133}   # half a step of the subnormals

# Of an activation: Lipschitz constants of itself and of its derivative, and what the evaluation itself may be off: the
# exponential and reciprocal take a few units of float32 (their argument's rounding times |z| included), gelu's polynomial
# for the error function 1.5e-7 (Abramowitz and Stegun 7.1.26), times |z|.
LIPSCHITZ, LIPSCHITZ2 = 1.13, 0.8


def act(z, name):
    if name == "relu":
        return z.clamp_min(0)
    if name == "silu":
        return z * torch.sigmoid(z)
    if name == "gelu":
        return 0.5 * z * torch.special.erfc(-z / math.sqrt(2))
    return z


def slope(z, name):
    if name == "relu":
        return (z > 0).double()
    if name == "silu":
        s = torch.sigmoid(z)
        return s * (1 + z * (1 - s))
    if name == "gelu":
        return 0.5 * torch.special.erfc(-z / math.sqrt(2)) + z * torch.exp(-z * z / 2) / math.sqrt(2 * math.pi)
    return torch.ones_like(z)


def act_error(z, name):
    return 0.0 if name in (None, "relu") else 4e-7 * (z.abs() + 1)


def slope_error(z, dz_error, name):
    """How far the derivative may be off when z is off by dz_error."""
    if name is None:
        return torch.zeros_like(z)
    if name == "relu":                                  # either side of the kink
        return (z.abs() <= dz_error).double()
    return LIPSCHITZ2 * dz_error + 1e-6 * (z.abs() + 1)


def rounded(value, error, dtype):
    """Bound after rounding a value that is off by `error` to dtype."""
    return error + UNIT[dtype] * (value.abs() + error) + TINY[dtype]


def linear(x, weight, bias, residual, name, grad, dtype):
    """{output: (value, bound)}; float64 inputs on the CPU."""
    K, N, rows = x.size(1), weight.size(0), x.size(0)
    extra = [t for t in (bias, residual) if t is not None]
    z, size = x @ weight.t(), x.abs() @ weight.abs().t()
    for t in extra:
        z, size = z + t, size + t.abs()
    z_err = (K + 4) * U32 * size
    y = act(z, name)
    out = {"y": (y, rounded(y, LIPSCHITZ * z_err + act_error(z, name), dtype))}
    if grad is None:
        return out
    d = slope(z, name)
    d_err = slope_error(z, z_err, name)
    if name in ("silu", "gelu") and dtype != torch.float32:
        d_err = d_err + 2.0 ** -16                      # kept in steps of 2^-15
    dz = grad * d
    exact_err = grad.abs() * d_err + 2 * U32 * dz.abs() * (name is not None)
    dz_err = rounded(dz, exact_err, dtype) if name is not None else exact_err
    if residual is not None:
        out["residual"] = (dz, dz_err)

    def product(a, b, a_err, terms):
        v = a @ b
        return v, rounded(v, a_err @ b.abs() + (terms + 4) * U32 * (a.abs() @ b.abs()), dtype)
    out["x"] = product(dz, weight, dz_err, N)
    out["weight"] = product(dz.t(), x, dz_err.t(), rows)
    if bias is not None:
        s = dz.sum(0)
        out["bias"] = (s, rounded(s, exact_err.sum(0) + (rows + 4) * U32 * dz.abs().sum(0), dtype))
    return out


# most float32 additions in a row that a value of group norm's sums goes through (rows of one lane, lanes of a workgroup,
# workgroups of an item, with what the joining formulas add): sums of the sizes tested here go through fewer
DEPTH = 512


def group_norm(x, groups, weight, bias, residual, name, eps, grad, dtype, param_dtype):
    """{output: (value, bound)}; x [B, S, C] in float64."""
    B, S, C = x.shape
    per = C // groups
    w = torch.ones(C, dtype=torch.float64) if weight is None else weight
    b = torch.zeros(C, dtype=torch.float64) if bias is None else bias

    def split(t):
        return t.reshape(B, S, groups, per)

    def whole(t):
        return t.expand(B, S, groups, per).reshape(B, S, C)
    xs = split(x)
    mean = xs.mean((1, 3), keepdim=True)
    var = (xs - mean).square().mean((1, 3), keepdim=True)
    rstd = 1 / torch.sqrt(var + eps)
    u = whole((xs - mean) * rstd)
    # the mean: a weighted mean of partial means, each a sum; the deviations are taken around partial means
    mean_err = DEPTH * U32 * xs.abs().amax((1, 3), keepdim=True)
    u_err = whole(mean_err * rstd + ((xs - mean) * rstd).abs() * (2 * DEPTH * U32 + (mean_err * rstd).square()))
    z, size = u * w + b, (u * w).abs() + b.abs()
    if residual is not None:
        z, size = z + residual, size + residual.abs()
    z_err = u_err * w.abs() + 8 * U32 * size
    y = act(z, name)
    out = {"y": (y, rounded(y, LIPSCHITZ * z_err + act_error(z, name), dtype))}
    if grad is None:
        return out
    dz = grad * slope(z, name)
    dz_err = grad.abs() * slope_error(z, z_err, name) + 2 * U32 * dz.abs()
    if residual is not None:
        out["residual"] = (dz, rounded(dz, dz_err, dtype))
    dot_err = dz_err * u.abs() + dz.abs() * u_err
    if weight is not None:
        v = (dz * u).sum((0, 1))
        out["weight"] = (v, rounded(v, dot_err.sum((0, 1)) + DEPTH * U32 * (dz * u).abs().sum((0, 1)), param_dtype))
    if bias is not None:
        v = dz.sum((0, 1))
        out["bias"] = (v, rounded(v, dz_err.sum((0, 1)) + DEPTH * U32 * dz.abs().sum((0, 1)), param_dtype))

    def group_mean(t):
        return whole(split(t).mean((1, 3), keepdim=True))
    s1, s2 = group_mean(dz * w), group_mean(dz * w * u)
    s1_err = group_mean(dz_err * w.abs()) + DEPTH * U32 * group_mean((dz * w).abs())
    s2_err = group_mean(dot_err * w.abs()) + DEPTH * U32 * group_mean((dz * w * u).abs())
    r = whole(rstd)
    dx = r * (w * dz - s1 - u * s2)
    dx_err = r * (w.abs() * dz_err + s1_err + u.abs() * s2_err + s2.abs() * u_err)
    dx_err = dx_err + r * (w * dz).abs().add(s1.abs()).add((u * s2).abs()) * (4 * DEPTH * U32 + whole((mean_err * rstd).square()))
    out["x"] = (dx, rounded(dx, dx_err, dtype))
    return out


def check(got, expected):
    """Every output within its bound; where the definition is NaN or infinite, the same."""
    assert set(got) == set(expected), (sorted(got), sorted(expected))
    for name, (value, bound) in expected.items():
        g = got[name].detach().double().cpu().reshape(value.shape)
        fine = torch.isfinite(value)
        assert torch.equal(torch.isnan(value), torch.isnan(g)), "%s: NaN in other places" % name
        assert torch.equal(value[~fine & ~value.isnan()], g[~fine & ~value.isnan()]), "%s: other infinities" % name
        off = (g - value).abs()[fine]
        worst = (off / bound[fine]).max().item() if off.numel() else 0.0
        assert bool((off <= bound[fine]).all()), "%s: %.3g times the bound" % (name, worst)
