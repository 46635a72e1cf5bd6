"""``residual_norm`` and ``ResidualNorm`` against their formulas in 64 bits (tests/block_reference.py derives the bounds), at numbers of
channels and rows where vectors, lanes and workgroups end."""
import random

import pytest
import torch

import block_reference as ref
from operator_reference import U32, check

pytestmark = pytest.mark.gpu
TYPES = [torch.float32, torch.float16, torch.bfloat16]
GATES = [None, "channel", "item", "full"]
LEAVES = ("x", "residual", "gate", "after_weight", "after_bias", "before_weight", "before_bias")


def case(B, C, spatial, dtype, kind="layer", gate=None, after=True, before=True, residual=True, params="float", float_gate=False, train=True,
         scale=0.75, eps=1e-6, seed=0, shift=0.0):
    """Host tensors, channels last: x [B, *spatial, C]."""
    gen = torch.Generator().manual_seed(seed + B + 3 * C + sum(spatial))

    def image(scale=1.0):
        return (torch.randn((B, *spatial, C), generator=gen) * scale + shift).to(dtype)
    ptype = {"none": torch.float32, "float": torch.float32, "same": dtype}[params]

    def vector(mean):
        return None if params == "none" else (torch.randn(C, generator=gen) * 0.3 + mean).to(ptype)
    gtype = torch.float32 if float_gate else dtype
    c = {"x": image(), "residual": image(1.5) if residual else None, "after": after, "before": before, "kind": kind, "scale": scale, "eps": eps, "dtype": dtype,
         "ptype": ptype, "gtype": gtype, "gate_kind": gate,
         "gate": {None: lambda: None, "channel": lambda: torch.randn(C, generator=gen).to(gtype), "item": lambda: torch.randn(B, C, generator=gen).to(gtype),
                  "full": image}[gate]()}
    for at in ("after", "before"):
        c[at + "_weight"] = vector(1.0) if c[at] else None
        c[at + "_bias"] = vector(0.0) if c[at] and kind == "layer" else None
    c["grad_stream"], c["grad_normed"] = (image(), image() if before else None) if train else (None, None)
    return c


def call(c, dev, **more):
    from box_convolution import residual_norm
    pairs = [(dev.get(at + "_weight"), dev.get(at + "_bias")) if c[at] else None for at in ("after", "before")]
    return residual_norm(dev["x"], dev.get("residual"), dev.get("gate"), c["scale"], *pairs, c["kind"], c["eps"], **more)


def placed(c, layout=None):
    """The leaves on the GPU; `layout` takes an image [B, ..., C] to [B, C, ...]."""
    layout = layout or (lambda t: t.movedim(-1, 1))
    dev = {}
    for k in LEAVES:
        if c[k] is not None:
            t = c[k].cuda()
            whole = k in ("x", "residual") or k == "gate" and c["gate_kind"] == "full"
            dev[k] = (layout(t) if whole else t).detach().requires_grad_(c["grad_stream"] is not None)
    return dev, layout


def run(c, layout=None):
    dev, layout = placed(c, layout)
    out = call(c, dev)
    named = dict(zip(("stream", "normed"), out)) if c["before"] else {"stream": out}
    if c["grad_stream"] is not None:
        grads = [layout(c[g].cuda()) for g in ("grad_stream", "grad_normed")[:len(named)]]
        named.update(zip(dev, torch.autograd.grad(list(named.values()), list(dev.values()), grads)))
    images = ("stream", "normed", "x", "residual") + (("gate",) if c["gate_kind"] == "full" else ())
    return {k: t.movedim(1, -1) if k in images else t for k, t in named.items()}


def expected(c):
    B, C = c["x"].size(0), c["x"].size(-1)

    def flat(t):
        return None if t is None else t.double().reshape(B, -1, C)

    def wide(t):
        return None if t is None else t.double()
    gate = flat(c["gate"]) if c["gate_kind"] == "full" else wide(c["gate"])
    pairs = [(wide(c[at + "_weight"]), wide(c[at + "_bias"])) if c[at] else None for at in ("after", "before")]
    return ref.residual_norm(flat(c["x"]), flat(c["residual"]), gate, c["scale"], *pairs, c["kind"], c["eps"], flat(c["grad_stream"]),
                             flat(c["grad_normed"]), c["dtype"], c["ptype"], c["gtype"])


# channels around vectors (4 or 8 elements), the lanes of a wave and of a workgroup, and beyond what registers hold; rows around what
# a workgroup takes
SIZES = [(1, 1, (1, 1)), (3, 3, (5,)), (2, 7, (3, 3)), (1, 8, (1,)), (2, 12, (31, 17)), (5, 16, ()), (3, 33, (9, 7)), (1, 52, (40, 41)), (4, 64, (16, 16)),
         (2, 100, (13, 3)), (7, 128, (11, 13)), (1, 130, (64,)), (2, 255, (9,)), (1, 256, (33, 3)), (2, 511, (5,)), (3, 512, (7,)), (1, 513, (70,)),
         (2, 1000, (3, 5)), (1, 1024, (257,)), (1, 1030, (19,)), (2, 2048, (17,)), (1, 4096, (1, 1)), (1, 4095, (30,)), (2, 5000, (9,)), (1, 8192, (40,)),
         (1, 8200, (3,)), (1, 16384, (5,)), (1, 16390, (4,)), (2, 20001, (2,)), (130, 24, (2, 2)), (2100, 8, (1,)), (1300, 20, (3,))]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("i", range(len(SIZES)))
def test_sizes(hip, i, dtype):
    """Every size with both norms, one gate (another for each type) and, in turn, kinds and types of the parameters."""
    t = TYPES.index(dtype)
    c = case(*SIZES[i], dtype, ("layer", "rms")[(i + t) % 2], GATES[(i + t) % 4], residual=i % 5 != 4, params=("float", "same")[(i // 2 + t) % 2],
             float_gate=i % 3 == 0 and GATES[(i + t) % 4] != "full")
    check(run(c), expected(c))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("C", [*range(1, 18), 519, 1023, 4099, 4101])
def test_last_rows_of_the_tensor(hip, C, dtype):
    """A row's last vector may not read beyond the tensor: every number of elements by which one would, in the last rows and in a tensor of less
    than a vector. A gate per element is read the same way."""
    for size in ((1, C, (1,)), (2, C, (2,)), (3, C, (1, 5))):
        c = case(*size, dtype, ("rms", "layer")[C % 2], "full" if C % 3 else "item", params=("same", "none")[C % 5 == 0])
        check(run(c), expected(c))


@pytest.mark.parametrize("C", [1, 2, 3, 5, 7, 9, 13, 130, 1021, 4103])
def test_last_rows_in_8_bits(hip, C):
    """The same reads where the normed rows leave in 8 bits: float32 rows are stored as they are quantized, so the codes are theirs; zeros behind a row, with a
    row of NaN among them too."""
    from box_convolution import quantize_blocks, residual_norm
    for rows in (1, 2, 5):
        torch.manual_seed(C * 8 + rows)
        x, r = (torch.randn(1, rows, C, device="cuda").movedim(-1, 1) for _ in range(2))
        w = torch.rand(C, device="cuda") + 0.5
        for k in range(2):
            stream, blocks = residual_norm(x, r, w, 0.5, (w, None), (w, w), "layer", quantize=True)
            same, normed = residual_norm(x, r, w, 0.5, (w, None), (w, w), "layer")
            want = quantize_blocks(normed.movedim(1, -1))
            assert torch.equal(stream.nan_to_num(7.0), same.nan_to_num(7.0))
            assert torch.equal(blocks.codes.view(torch.uint8), want.codes.view(torch.uint8)) and torch.equal(blocks.exponents, want.exponents)
            assert not blocks.codes[..., C:].float().any()
            x[0, 0, rows - 1] = float("nan")


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("after,before", [(True, True), (True, False), (False, True), (False, False)])
@pytest.mark.parametrize("gate", GATES)
def test_pieces(hip, after, before, gate, dtype):
    """Each norm, gate and residual with and without the others, on rows within a wave and of a whole workgroup."""
    for k, size in enumerate(((3, 40, (6, 7)), (2, 1500, (9,)))):
        for residual in (True, False):
            c = case(*size, dtype, ("rms", "layer")[k], gate, after, before, residual, ("none", "same")[residual])
            check(run(c), expected(c))


@pytest.mark.parametrize("size", [(2, 48, (30, 20)), (1, 1024, (33,)), (2, 3000, (7,)), (1, 17000, (3,))])
def test_mean_far_from_zero(hip, size):
    """The deviations are taken from the mean, not from sums of squares: a mean of 300 deviations costs its own digits only."""
    c = case(*size, torch.float32, "layer", "channel", shift=300.0)
    check(run(c), expected(c))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("C", [24, 700, 6000])
def test_rows_of_one_value(hip, C, dtype):
    """Nothing but eps under the root: a layer norm gives its bias; rows of zeros stay zeros in both kinds."""
    for kind in ("layer", "rms"):
        c = case(2, C, (5,), dtype, kind, params="same", residual=False, train=False, eps=1e-3)
        c["x"].fill_(0.0 if kind == "rms" else 2.0)
        out = run(c)
        bias = c["after_bias"] if kind == "layer" else torch.zeros(C, dtype=dtype)
        want = bias.double() * c["scale"]
        assert (out["stream"].double().cpu() - want).abs().max() <= torch.finfo(dtype).eps * 4
    c = case(1, C, (3,), dtype, "rms", before=False, residual=False)
    c["x"].zero_()
    check(run(c), expected(c))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("C", [20, 128, 1200, 17000])
def test_nan_and_infinity_stay_in_their_row(hip, C, dtype):
    c = case(2, C, (9,), dtype, "layer", "channel", train=True)
    for where, value in (("x", float("nan")), ("residual", float("inf")), ("x", float("-inf")), ("grad_normed", float("nan"))):
        d = {k: t.clone() if torch.is_tensor(t) else t for k, t in c.items()}
        d[where][1, 4, C // 2] = value
        out, plain = run(d), run(c)
        for k in ("stream", "normed", "x", "residual"):
            rows = torch.ones(2, 9, dtype=torch.bool)
            rows[1, 4] = False
            assert torch.equal(out[k][rows.cuda()], plain[k][rows.cuda()]), (where, value, k)
        bad = out["normed" if where != "grad_normed" else "residual"][1, 4]
        assert bad.isnan().all()
        if where == "grad_normed":
            assert torch.equal(out["normed"], plain["normed"])


def test_gradients_against_differences(hip):
    """Central differences of a weighted sum of both outputs along random directions of every input, in float32 with steps of 2^-7: the
    second-order error is a few times 2^-14 of the scale, the rounding of the sum divided by the step less."""
    from box_convolution import residual_norm
    torch.manual_seed(3)
    B, C, P = 2, 20, 6
    for kind in ("rms", "layer"):
        for gate_shape in ((C,), (B, C), (B, C, P)):
            leaves = [torch.randn(B, C, P), torch.randn(B, C, P), torch.rand(*gate_shape) + 0.5, torch.rand(C) + 0.5, torch.randn(C), torch.rand(C) + 0.5, torch.randn(C)]
            leaves = [t.cuda().requires_grad_(True) for t in leaves]
            g1, g2 = torch.randn(B, C, P).cuda(), torch.randn(B, C, P).cuda()

            def value(x, r, g, wa, ba, wb, bb):
                s, h = residual_norm(x, r, g, 0.6, (wa, ba), (wb, bb), kind, 1e-3)
                return (s.double() * g1).sum() + (h.double() * g2).sum()
            grads = torch.autograd.grad(value(*leaves), leaves)
            for i, (t, g) in enumerate(zip(leaves, grads)):
                d = torch.randn_like(t)
                step = 2.0 ** -7 / float(d.norm())
                with torch.no_grad():
                    up, down = (value(*[u + sign * step * d if j == i else u for j, u in enumerate(leaves)]) for sign in (1, -1))
                slope, want = float((up - down) / (2 * step)), float((g.double() * d).sum())
                assert abs(slope - want) <= 2e-3 * float(g.norm() * d.norm()), (kind, gate_shape, i)


def test_only_what_is_needed(hip):
    """Gradients for some of the inputs only, and of one output only, are those of all."""
    c = case(2, 40, (5, 6), torch.float32, "layer", "item")
    dev, layout = placed(c)
    names = list(dev)
    g1, g2 = layout(c["grad_stream"].cuda()), layout(c["grad_normed"].cuda())
    full = dict(zip(names, torch.autograd.grad(call(c, dev), list(dev.values()), (g1, g2))))
    for some in (["x"], ["gate"], ["before_weight"], ["residual", "after_bias"]):
        d = {k: t.detach().requires_grad_(k in some) for k, t in dev.items()}
        got = torch.autograd.grad(call(c, d), [d[k] for k in some], (g1, g2))
        assert all(torch.equal(a, full[k]) for k, a in zip(some, got)), some
    zero = torch.zeros_like(g1)
    for k, given in enumerate((g1, g2)):
        out = call(c, dev)
        some = [n for n in names if k == 1 or not n.startswith("before")]
        alone = torch.autograd.grad(out[k], [dev[n] for n in some], given)
        both = torch.autograd.grad(call(c, dev), [dev[n] for n in some], (given, zero) if k == 0 else (zero, given))
        assert all(torch.equal(a, b) for a, b in zip(alone, both)), k


def test_stream_is_the_input_where_nothing_is_done_to_it(hip):
    from box_convolution import residual_norm
    x = torch.randn(2, 24, 5, device="cuda").movedim(1, 2).contiguous().movedim(2, 1).requires_grad_(True)
    w = torch.randn(24, device="cuda", requires_grad=True)
    s, h = residual_norm(x, before=(w, None))
    assert s is x and residual_norm(x) is x
    r = x.detach().clone().requires_grad_(True)
    t, k = residual_norm(torch.zeros_like(x), r, before=(w, None))
    assert torch.equal(t, x) and torch.equal(h, k)
    g = torch.randn_like(x)
    assert torch.equal(torch.autograd.grad(h, x, g, retain_graph=True)[0], torch.autograd.grad(k, r, g, retain_graph=True)[0])
    a, b = torch.autograd.grad((s * 2).sum() + h.sum(), (x, w)), torch.autograd.grad((t * 2).sum() + k.sum(), (r, w))
    assert (a[0] - b[0]).abs().max() <= 4 * U32 * 16 and torch.equal(a[1], b[1])


@pytest.mark.parametrize("dtype", TYPES)
def test_layouts_and_addresses(hip, dtype):
    """Planes, slices and expanded tensors are copied; rows inside a larger buffer at any element are used as they lie."""
    for C in (40, 41, 1100):
        c = case(2, C, (5, 6), dtype, "layer", "full")
        plain = run(c)
        for layout in (lambda t: t.movedim(-1, 1).contiguous(), lambda t: torch.stack((t, t), -1)[..., 0].movedim(-1, 1)):
            other = run(c, layout)
            assert all(torch.equal(plain[k], other[k]) for k in plain)

        def shifted(t):
            big = torch.full((t.numel() + 2,), float("nan"), dtype=t.dtype, device=t.device)
            view = big[1:-1].view(t.shape)
            view.copy_(t)
            return view.movedim(-1, 1)
        other = run(c, shifted)
        assert all(torch.equal(plain[k], other[k]) for k in plain)
    # a broadcast gradient, and a broadcast gate
    c = case(2, 40, (5, 6), dtype, "rms", "channel")
    dev, _ = placed(c)
    s, h = call(c, dev)
    a = torch.autograd.grad(h.sum(), dev["x"], retain_graph=True)[0]
    assert torch.equal(a, torch.autograd.grad(h, dev["x"], torch.ones_like(h))[0])
    wide = {**dev, "gate": dev["gate"][None, :].expand(2, 40)}
    assert torch.equal(call(c, wide)[0], s)


def test_empty(hip):
    for size in ((0, 8, (3,)), (2, 8, (0,)), (2, 8, (3, 0))):
        for gate in GATES:
            c = case(*size, torch.float32, "layer", gate)
            out = run(c)
            assert out["stream"].numel() == 0 and not any(out[k].any() for k in out if k.startswith(("after", "before")) or k == "gate")


def test_another_stream_and_same_bits(hip):
    c = case(2, 48, (131, 77), torch.bfloat16, "layer", "item")
    first = run(c)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        second = run(c)
    side.synchronize()
    for k in first:
        assert torch.equal(first[k], second[k]), k


@pytest.mark.parametrize("size", [(2, 24, (12, 13)), (3, 1500, (40,)), (1, 17000, (5,))])
def test_graph_replays(hip, size):
    c = case(*size, torch.bfloat16, "layer", "item")
    dev = {k: t.detach() for k, t in placed(c)[0].items()}
    dev = {k: t.movedim(1, -1) if k in ("x", "residual") else t for k, t in dev.items()}
    params = [dev[k] for k in LEAVES[3:]]
    grads = [c[k].cuda() for k in ("grad_stream", "grad_normed")]
    norms = hip.NORM_AFTER | hip.NORM_BEFORE | hip.NORM_CENTRE

    def step():
        begin = (dev["x"], dev["residual"], dev["gate"], hip.GATE_ITEM, 0.5, norms, params, 1e-6)
        *out, statistics = hip.residual_norm_forward(*begin, True, None, True)
        return out + hip.residual_norm_backward(*begin, statistics, *grads, (True,) * 7)
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step()
    for k in range(3):
        dev["x"].copy_(dev["x"].roll(k + 1, -1))
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in captured]
        assert all(torch.equal(a, e) for a, e in zip(got, step()))


@pytest.fixture(params=["C++", "Python"])
def host_side(request, hip, monkeypatch):
    """Both host sides of the operators (the second one is what runs where the C++ extension was not built)."""
    if request.param == "Python":
        monkeypatch.setattr(hip, "_glue", False)
        assert hip.glue() is None
    elif hip.glue() is None:
        pytest.skip("the C++ extension was not built")
    return request.param


@pytest.mark.parametrize("dtype", TYPES)
def test_both_host_sides(host_side, dtype):
    for gate in GATES:
        for after, before in ((True, True), (True, False), (False, True)):
            c = case(2, 12, (9, 7), dtype, "layer" if gate else "rms", gate, after, before, gate != "full", "same", gate in ("channel", "item"))
            check(run(c), expected(c))
            c["grad_stream"] = None
            check(run(c), expected(c))


def test_refusals(host_side):
    from box_convolution import ResidualNorm, residual_norm
    x, one = torch.zeros(2, 8, 3, 3, device="cuda"), torch.ones(8, device="cuda")
    pair = (one, None)
    for bad, match in ((lambda: residual_norm(x.cpu(), before=pair), "AMD GPUs only"), (lambda: residual_norm(x.double(), before=pair), "float32, float16 or bfloat16"),
                       (lambda: residual_norm(x[:, 0, 0, 0], before=pair), ">=2 dimensions"), (lambda: residual_norm(x[:, :0], before=pair), "a channel"),
                       (lambda: residual_norm(x, x[:1], before=pair), "residual"), (lambda: residual_norm(x, x.half(), before=pair), "residual"),
                       (lambda: residual_norm(x, gate=one[:7]), "gate must have the shape"), (lambda: residual_norm(x, gate=x[:, :, 0]), "gate must have the shape"),
                       (lambda: residual_norm(x, gate=one.half()), "gate must be"), (lambda: residual_norm(x.half(), gate=x), "gate must be"),
                       (lambda: residual_norm(x, gate=one.cpu()), "gate must be"), (lambda: residual_norm(x, after=one), "pair"),
                       (lambda: residual_norm(x, before=(one,)), "pair"), (lambda: residual_norm(x, before=(one[:7], None)), "must hold 8 values"),
                       (lambda: residual_norm(x, before=(one.half(), None)), "float32"), (lambda: residual_norm(x.half(), None, None, 1.0, pair, (one.half(), None)), "all be float32"),
                       (lambda: residual_norm(x, before=(one.cpu(), None)), "must hold 8 values"), (lambda: residual_norm(x, before=pair, kind="batch"), "kind"),
                       (lambda: residual_norm(x, gate=one, quantize=True), "norm before"),
                       (lambda: residual_norm(x.clone().requires_grad_(True), before=pair, quantize=True), "inference"),
                       (lambda: ResidualNorm(8, kind="group"), "kind"), (lambda: ResidualNorm(8, layer_scale=0.1).cuda()(x, gate=one), "exclude")):
        with pytest.raises(RuntimeError, match=match):
            bad()


def test_not_twice(host_side):
    from box_convolution import residual_norm
    x, r = (torch.randn(2, 8, 3, 3, device="cuda", requires_grad=True) for _ in range(2))
    w = torch.ones(8, device="cuda", requires_grad=True)

    def value():
        s, h = residual_norm(x, r, w, 0.5, (w, None), (w, None))
        return s.sum() + h.square().sum()
    once = torch.autograd.grad(value(), [x, r, w])
    again = torch.autograd.grad(value(), [x, r, w], create_graph=True)
    assert all(torch.equal(a, b) for a, b in zip(once, again))
    for g in again:
        with pytest.raises(RuntimeError, match="not twice"):
            g.square().sum().backward(retain_graph=True)


def test_forward_mode_is_refused(host_side):
    import torch.autograd.forward_ad as forward_ad
    from box_convolution import residual_norm
    x, r = torch.randn(2, 8, 3, 3, device="cuda"), torch.randn(2, 8, 3, 3, device="cuda")
    g, w = torch.randn(2, 8, device="cuda"), torch.randn(8, device="cuda")
    with forward_ad.dual_level():
        for i in range(7):
            args = [forward_ad.make_dual(t, torch.ones_like(t)) if i == k else t for k, t in enumerate((x, r, g, w, w, w, w))]
            for recorded in (False, True):
                with torch.set_grad_enabled(recorded), pytest.raises(RuntimeError, match="forward-mode"):
                    residual_norm(*args[:3], 1.0, tuple(args[3:5]), tuple(args[5:]), "layer")
        leaf = x.clone().requires_grad_(True)
        s, h = residual_norm(leaf, r, g, 1.0, (w, w), (w, w), "layer")
        for y in (s, h):
            with pytest.raises(RuntimeError, match="forward-mode"):
                torch.autograd.grad(y, leaf, forward_ad.make_dual(torch.ones_like(y), torch.ones_like(y)), retain_graph=True)


@pytest.mark.parametrize("turned", [False, True])
def test_saved_tensors_of_another_layout(host_side, turned):
    def unpack(t):
        if not turned:
            return torch.empty(t.shape, dtype=t.dtype, device=t.device).copy_(t)
        return t.transpose(0, -1).contiguous().transpose(0, -1) if t.dim() > 1 else torch.stack((t, t), 1)[:, 0]
    for size in ((2, 12, (9, 7)), (3, 8, ())):
        for gate in (None, "item", "full"):
            c = case(*size, torch.float32, "layer", gate)
            plain = run(c)
            with torch.autograd.graph.saved_tensors_hooks(lambda t: t, unpack):
                hooked = run(c)
            assert all(torch.equal(plain[k], hooked[k]) for k in plain)


def test_module(hip):
    from box_convolution import ResidualNorm
    torch.manual_seed(0)
    module = ResidualNorm(24, kind="layer", scale=0.5, layer_scale=0.1).cuda()
    x, r = (torch.randn(2, 24, 9, 13, device="cuda") for _ in range(2))
    s, h = module(x, r)
    d = [t.double().movedim(1, -1) for t in (x, r)]
    want = d[1] + 0.05 * torch.nn.functional.layer_norm(d[0], (24,), eps=1e-6)
    assert (s.double().movedim(1, -1) - want).abs().max() <= 2.0 ** -18 * 8                 # (two dozen roundings of values up to 8)
    want = torch.nn.functional.layer_norm(want, (24,), eps=1e-6)
    assert (h.double().movedim(1, -1) - want).abs().max() <= 2.0 ** -18 * 8
    (s.sum() + h.square().sum()).backward()
    assert all(p.grad is not None for p in module.parameters()) and len(list(module.parameters())) == 5
    half = ResidualNorm(24, after=False).cuda()
    assert len(list(half.parameters())) == 1 and "rms" in repr(half)
    s, h = half(x.bfloat16(), r.bfloat16())
    assert s.dtype == h.dtype == torch.bfloat16


@pytest.mark.parametrize("gate", ["channel", "item"])
@pytest.mark.parametrize("size", [(40001, 16, ()), (3, 8, (200, 211)), (700, 24, (20,)), (2, 1024, (900,)), (600, 256, (3,))])
def test_sums_over_many_rows(hip, size, gate):
    """As many float32 additions in a row as the bound allows, however many rows: the same gradients everywhere, so that in one chain their
    roundings would add up."""
    c = case(*size, torch.float32, "layer", gate if size[2] else "channel")
    for k in ("grad_stream", "grad_normed"):
        c[k] = torch.full_like(c[k], 1.1)
    check(run(c), expected(c))


def test_more_than_2_31_elements(hip):
    """Rows beyond 2^31 elements are those of the same values in a smaller tensor, forward and backward."""
    from box_convolution import residual_norm
    C, small, repeats = 64, 1 << 15, 1040
    gen = torch.Generator(device="cuda").manual_seed(0)
    x, r, g = (torch.randn(small, C, generator=gen, device="cuda", dtype=torch.bfloat16) for _ in range(3))
    w = torch.rand(C, generator=gen, device="cuda") + 0.5

    def both(x, r, g):
        x, r = x.requires_grad_(True), r.requires_grad_(True)
        s, h = residual_norm(x, r, None, 0.5, (w, None), (w, None))
        return (s.detach(), h.detach(), *torch.autograd.grad(h, (x, r), g))
    want = both(x.clone(), r.clone(), g)
    got = both(*(t.repeat(repeats, 1) for t in (x, r, g)))
    assert got[0].numel() > 1 << 31
    for a, b in zip(got, want):
        for k in (0, repeats // 2, repeats - 1):
            assert torch.equal(a[k * small:(k + 1) * small], b)


@pytest.mark.parametrize("C", [520, 4097, 6000, 9001])
def test_kept_statistics_are_those_formed_again(hip, C):
    """The backward with the forward's statistics and without them: the same bits."""
    c = case(2, C, (5,), torch.bfloat16, "layer", "item")
    dev = {k: t.detach() for k, t in placed(c)[0].items()}
    dev = {k: t.movedim(1, -1) if k in ("x", "residual") else t for k, t in dev.items()}
    norms = hip.NORM_AFTER | hip.NORM_BEFORE | hip.NORM_CENTRE
    begin = (dev["x"], dev["residual"], dev["gate"], hip.GATE_ITEM, 0.5, norms, [dev[k] for k in LEAVES[3:]], 1e-6)
    statistics = hip.residual_norm_forward(*begin, True, None, True)[2]
    assert statistics.numel() == 2 * 5 * 4 and hip.residual_norm_forward(*begin, True)[2] is None
    grads = [c[k].cuda() for k in ("grad_stream", "grad_normed")]
    kept, again = (hip.residual_norm_backward(*begin, s, *grads, (True,) * 7) for s in (statistics, None))
    assert all(torch.equal(a, b) for a, b in zip(kept, again))


def test_random_sizes(hip):
    """Forty draws of everything at once."""
    rng = random.Random(5)
    for i in range(40):
        C, gate = int(2 ** rng.uniform(0, 12.5)), rng.choice(GATES)
        B, n = rng.randint(1, 5), rng.randint(1, max(1, min(400, 60000 // C)))
        c = case(B, C, (n,), rng.choice(TYPES), rng.choice(("rms", "layer")), gate, rng.random() < 0.7, rng.random() < 0.7, rng.random() < 0.7,
                 rng.choice(("none", "float", "same")), gate in ("channel", "item") and rng.random() < 0.5, seed=i)
        check(run(c), expected(c))


