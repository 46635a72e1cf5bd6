"""What lies between residual blocks, blocks of 128 in 8 bits and their product in 64 bits, on the CPU, with bounds on how far float32
sums, the 8-bit matrix instructions and one rounding to the output's type may take a result from them."""
import torch

from operator_reference import DEPTH, LIPSCHITZ, U32, act, act_error, rounded

BLOCK = 128


def _moments(v, v_err, centre, eps):
    """(unit, its error bound, rstd, its relative error) of rows v that are off by at most v_err themselves."""
    C = v.size(-1)
    mean = v.mean(-1, keepdim=True) if centre else torch.zeros_like(v[..., :1])
    dev = v - mean
    rstd = 1 / torch.sqrt(dev.square().mean(-1, keepdim=True) + eps)
    # the mean is off by its own sum's roundings and by the mean of the errors; every deviation by that and its own
    off = v_err + centre * (v_err.mean(-1, keepdim=True) + DEPTH * U32 * v.abs().amax(-1, keepdim=True))
    # the mean square M of the deviations changes by at most 2 sqrt(M) rms(off) + rms(off)^2; rstd by half of that relatively, and by the
    # sum's roundings
    part = off.square().mean(-1, keepdim=True).sqrt() * rstd
    relative = part + part.square() + 2 * DEPTH * U32
    unit = dev * rstd
    assert C > 0
    return unit, off * rstd + unit.abs() * relative, rstd, relative


def _mean_pair(e, e_err, unit, unit_err, centre):
    """(mean(e), error, mean(e * unit), error)."""
    m1 = e.mean(-1, keepdim=True) * centre
    m1_err = centre * (e_err.mean(-1, keepdim=True) + DEPTH * U32 * e.abs().mean(-1, keepdim=True))
    m2 = (e * unit).mean(-1, keepdim=True)
    m2_err = (e.abs() * unit_err + e_err * (unit.abs() + unit_err)).mean(-1, keepdim=True) + DEPTH * U32 * (e * unit).abs().mean(-1, keepdim=True)
    return m1, m1_err, m2, m2_err


def _through(e, e_err, unit, unit_err, rstd, relative, centre):
    """The gradient of a row from that of its normalised form, and its error."""
    m1, m1_err, m2, m2_err = _mean_pair(e, e_err, unit, unit_err, centre)
    size = e.abs() + m1.abs() + (unit * m2).abs()
    v = rstd * (e - m1 - unit * m2)
    err = rstd * (e_err + m1_err + unit.abs() * m2_err + unit_err * (m2.abs() + m2_err) + 4 * U32 * size)
    return v, err * (1 + relative) + relative * (v.abs() + err) + 4 * U32 * v.abs()


def residual_norm(x, residual, gate, scale, after, before, kind, eps, grad_stream, grad_normed, dtype, param_dtype, gate_dtype):
    """{output: (value, bound)}: x, residual [B, S, C] in float64; gate None, [C], [B, C] or [B, S, C]; after, before None or (weight, bias),
    either of which may be None."""
    B, S, C = x.shape
    centre = float(kind == "layer")
    one, zero = torch.ones(C, dtype=torch.float64), torch.zeros(C, dtype=torch.float64)

    def pair(p):
        return (one if p[0] is None else p[0], zero if p[1] is None else p[1])
    u, u_err = x, torch.zeros_like(x)
    if after is not None:
        wa, ba = pair(after)
        p, p_err, rstd_x, rel_x = _moments(x, torch.zeros_like(x), centre, eps)
        u = p * wa + ba
        u_err = p_err * wa.abs() + 4 * U32 * ((p * wa).abs() + ba.abs())
    g = torch.ones_like(x) if gate is None else gate.expand(B, S, C) if gate.dim() == 1 else gate[:, None, :].expand(B, S, C) if gate.dim() == 2 else gate
    r = torch.zeros_like(x) if residual is None else residual
    t = scale * g * u
    s = r + t
    s_err = (scale * g).abs() * u_err + 4 * U32 * (r.abs() + t.abs())
    out = {"stream": (s, rounded(s, s_err, dtype))}
    if before is not None:
        wb, bb = pair(before)
        q, q_err, rstd_s, rel_s = _moments(s, s_err, centre, eps)
        h = q * wb + bb
        out["normed"] = (h, rounded(h, q_err * wb.abs() + 4 * U32 * ((q * wb).abs() + bb.abs()), dtype))
    if grad_stream is None:
        return out

    def total(v, err, dims, to):
        return v.sum(dims), rounded(v.sum(dims), err.sum(dims) + DEPTH * U32 * v.abs().sum(dims), to)
    ds, ds_err = grad_stream, torch.zeros_like(x)
    if before is not None:
        dh = grad_normed
        e = dh * wb
        through, through_err = _through(e, 2 * U32 * e.abs(), q, q_err, rstd_s, rel_s, centre)
        ds = ds + through
        ds_err = through_err + 4 * U32 * (grad_stream.abs() + through.abs())
        if before[0] is not None:
            out["before_weight"] = total(dh * q, dh.abs() * q_err + 2 * U32 * (dh * q).abs(), (0, 1), param_dtype)
        if before[1] is not None:
            out["before_bias"] = total(dh, torch.zeros_like(dh), (0, 1), param_dtype)
    if residual is not None:
        out["residual"] = (ds, rounded(ds, ds_err, dtype))
    if gate is not None:
        dg = scale * u * ds
        dg_err = abs(scale) * (u.abs() * ds_err + u_err * (ds.abs() + ds_err)) + 4 * U32 * dg.abs()
        out["gate"] = (dg, rounded(dg, dg_err, dtype)) if gate.dim() == 3 else total(dg, dg_err, 1 if gate.dim() == 2 else (0, 1), gate_dtype)
    du = scale * g * ds
    du_err = (scale * g).abs() * ds_err + 4 * U32 * du.abs()
    if after is not None:
        if after[0] is not None:
            out["after_weight"] = total(du * p, p.abs() * du_err + p_err * (du.abs() + du_err) + 2 * U32 * (du * p).abs(), (0, 1), param_dtype)
        if after[1] is not None:
            out["after_bias"] = total(du, du_err, (0, 1), param_dtype)
        f = du * wa
        dx, dx_err = _through(f, du_err * wa.abs() + 2 * U32 * f.abs(), p, p_err, rstd_x, rel_x, centre)
        out["x"] = (dx, rounded(dx, dx_err, dtype))
    else:
        out["x"] = (du, rounded(du, du_err, dtype))
    return out


# ---- 8 bits -----------------------------------------------------------------------------------

def _code_values():
    """The values of codes 0 to 126: 4 bits of exponent (bias 7), 3 of mantissa."""
    out = []
    for c in range(127):
        e, m = c >> 3, c & 7
        out.append((1 + m / 8) * 2.0 ** (e - 7) if e else m / 8 * 2.0 ** -6)
    return torch.tensor(out, dtype=torch.float64)


CODE_VALUES = _code_values()


def two_to(e):
    """2**e of whole numbers from -1022 on, exactly."""
    return ((e.to(torch.int64) + 1023) << 52).view(torch.float64)


def quantize(x):
    """(values in units of their block's power, padded to whole blocks; stored exponents, padded to whole words) of float64 rows on the CPU. NaN where x is not
    finite."""
    rows, K = x.shape
    blocks = -(-K // BLOCK)
    full = torch.zeros(rows, blocks * BLOCK, dtype=torch.float64)
    full[:, :K] = x
    full = full.view(rows, blocks, BLOCK)
    most = torch.where(full.isfinite(), full.abs(), torch.zeros_like(full)).amax(-1)
    e = torch.full_like(most, -126)
    for power in range(-126, 121):                                  # the least that does
        e = torch.where(most > 448 * 2.0 ** power, torch.full_like(e, power + 1), e)
    e = torch.where(most == 0, torch.zeros_like(e), e)
    units = full / two_to(e)[..., None]
    size = units.abs().nan_to_num(0.0, 0.0, 0.0).clamp_max(448.0)
    above = torch.searchsorted(CODE_VALUES, size.contiguous()).clamp_max(126)       # first code value >= size
    below = (above - 1).clamp_min(0)
    lo, hi = CODE_VALUES[below], CODE_VALUES[above]
    nearer = torch.where(hi - size < size - lo, above, below)
    nearer = torch.where(hi - size == size - lo, torch.where(above % 2 == 0, above, below), nearer)     # ties to even
    out = torch.copysign(CODE_VALUES[nearer], units)
    out = torch.where(full.isfinite(), out, torch.full_like(out, float("nan")))
    words = torch.full((rows, -(-blocks // 4) * 4), 127, dtype=torch.uint8)
    words[:, :blocks] = (e + 127).to(torch.uint8)
    return out.reshape(rows, -1), words


def dequantize(x):
    """The values on their blocks' grid, [rows, K]."""
    units, words = quantize(x)
    blocks = units.size(1) // BLOCK
    power = two_to(words[:, :blocks].to(torch.int64) - 127)
    return (units.view(x.size(0), blocks, BLOCK) * power[..., None]).reshape(x.size(0), -1)[:, :x.size(1)]


def product(x, weight, bias, residual, name, dtype):
    """{"y": (value, bound)} of rows and weights on their grids (float64)."""
    K = x.size(1)
    z, size = x @ weight.t(), x.abs() @ weight.abs().t()
    for t in (bias, residual):
        if t is not None:
            z, size = z + t, size + t.abs()
    z_err = (K + 8) * U32 * size
    if dtype != torch.float32:
        # each of 8 neighbouring products may lose what is below 2^-13 of the largest of them
        def most(v):
            pad = torch.zeros(v.size(0), -(-K // 8) * 8, dtype=torch.float64)
            pad[:, :K] = v.abs()
            return pad.view(v.size(0), -1, 8).amax(-1)
        z_err = z_err + 8 * 2.0 ** -13 * (most(x) @ most(weight).t())
    y = act(z, name)
    return {"y": (y, rounded(y, LIPSCHITZ * z_err + act_error(z, name), dtype))}
