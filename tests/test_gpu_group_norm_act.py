"""``group_norm_act`` and ``GroupNormAct`` against group norm in 64 bits (tests/operator_reference.py derives the
bounds), at numbers of channels, pixels and groups where lanes, vectors and workgroups end."""
import pytest
import torch

import operator_reference as ref

pytestmark = pytest.mark.gpu
TYPES = [torch.float32, torch.float16, torch.bfloat16]
ACTS = [None, "relu", "silu", "gelu"]
EPS = 1e-5


def case(B, C, G, spatial, dtype, name, residual, params, train=True, shift=0.0, seed=0):
    """Host tensors, channels last: x [B, *spatial, C]."""
    gen = torch.Generator().manual_seed(seed + B + 3 * C + 5 * G + sum(spatial))

    def image(scale=1.0, off=0.0):
        return (torch.randn((B, *spatial, C), generator=gen) * scale + off).to(dtype)
    kind = {"none": None, "float": torch.float32, "same": dtype}[params]
    x = (torch.randn((B, *spatial, C), generator=gen) + torch.randn(C, generator=gen) + shift).to(dtype)
    w = None if kind is None else (torch.randn(C, generator=gen) * 0.3 + 1).to(kind)
    b = None if kind is None else (torch.randn(C, generator=gen) * 0.3).to(kind)
    return {"x": x, "weight": w, "bias": b, "residual": image() if residual else None, "grad": image() if train else None,
            "groups": G, "name": name, "kind": kind, "dtype": dtype}


def run(c, layout=None):
    from box_convolution import group_norm_act
    layout = layout or (lambda t: t.movedim(-1, 1))
    train = c["grad"] is not None
    dev = {}
    for k in ("x", "weight", "bias", "residual"):
        if c[k] is not None:
            t = c[k].cuda()
            dev[k] = (layout(t) if k in ("x", "residual") else t).detach().requires_grad_(train)
    y = group_norm_act(dev["x"], c["groups"], dev.get("weight"), dev.get("bias"), dev.get("residual"), c["name"], EPS)
    out = {"y": y}
    if train:
        out.update(zip(dev, torch.autograd.grad(y, list(dev.values()), layout(c["grad"].cuda()))))
    return {k: t.movedim(1, -1) if t.dim() > 1 else t for k, t in out.items()}


def expected(c):
    B, C = c["x"].size(0), c["x"].size(-1)

    def flat(t):
        return None if t is None else t.double().reshape(B, -1, C)
    wide = [None if t is None else t.double() for t in (c["weight"], c["bias"])]
    return ref.group_norm(flat(c["x"]), c["groups"], *wide, flat(c["residual"]), c["name"], EPS, flat(c["grad"]), c["dtype"], c["kind"])


SIZES = [(1, 1, 1, (1, 1)), (3, 4, 2, ()), (2, 6, 3, (5, 7)), (1, 40, 8, (28, 28)), (32, 40, 8, (7, 9)), (3, 48, 6, (33, 17)), (2, 5, 5, (9,)),
         (2, 128, 32, (64, 64)), (1, 320, 32, (40, 41)), (2, 1031, 1, (3, 5)), (1, 1100, 275, (2, 3)), (1, 2048, 32, (3, 3)), (1, 7, 1, (300, 301)),
         (2, 64, 1, (100, 99)), (1, 256, 8, (96, 20)), (5, 333, 3, (11, 13)), (1, 24, 24, (200, 211)), (1, 8192, 64, (3, 7)), (2, 16, 4, (1, 1)),
         (1, 12, 2, (2, 3, 5)), (70, 32, 8, (65, 33)), (1, 8192, 8192, (5, 1)), (2, 4096, 4096, (7,))]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("i", range(len(SIZES)))
def test_sizes(hip, i, dtype):
    k = i + TYPES.index(dtype)
    c = case(*SIZES[i], dtype, ACTS[k % 4], residual=k % 2 == 1, params=("float", "same", "none")[k % 3])
    ref.check(run(c), expected(c))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("name", ACTS)
@pytest.mark.parametrize("residual,params", [(False, "float"), (True, "same"), (True, "float")])
def test_epilogues(hip, name, residual, params, dtype):
    """One workgroup per item, some channels of it, and several workgroups per item."""
    for size in ((2, 20, 4, (9, 10)), (2, 64, 2, (50, 60)), (2, 32, 8, (130, 131))):
        c = case(*size, dtype, name, residual, params, seed=2)
        ref.check(run(c), expected(c))


@pytest.mark.parametrize("size", [(2, 24, 4, (12, 13)), (1, 24, 4, (130, 140)), (1, 1031, 1, (3, 5))])
def test_mean_far_from_zero(hip, size):
    """A spread of 1 around 1000: the bound allows what rounding the mean costs, and nothing for sums of squares that cancel."""
    c = case(*size, torch.float32, "silu", False, "float", shift=1000.0)
    ref.check(run(c), expected(c))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("size", [(2, 24, 4, (12, 13)), (2, 24, 4, (130, 140)), (1, 1031, 1, (3, 5))])
def test_one_value_everywhere(hip, size, dtype):
    """No spread: the result is the bias (eps keeps the quotient finite)."""
    c = case(*size, dtype, None, False, "same", train=False)
    c["x"] = torch.full_like(c["x"], 2.5)
    y = run(c)["y"].cpu()
    assert torch.equal(y, c["bias"].expand_as(y))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("size", [(3, 24, 4, (12, 13)), (3, 24, 4, (130, 140)), (3, 1030, 2, (3, 5))])
def test_nan_and_infinity_stay_in_their_group(hip, size, dtype):
    for value in (float("nan"), float("inf")):
        c = case(*size, dtype, "relu", False, "float")
        G, C = size[2], size[1]
        c["x"].view(3, -1, C)[1, 7, C // G] = value                     # batch item 1, group 1
        out = run(c)
        bad = out["y"].reshape(3, -1, G, C // G).isnan().cpu()
        assert bad[1, :, 1].all() and bad.sum() == bad[1, :, 1].numel()
        bad = out["x"].reshape(3, -1, G, C // G).isnan().cpu()
        assert bad[1, :, 1].all() and bad.sum() == bad[1, :, 1].numel()


@pytest.mark.parametrize("dtype", TYPES)
def test_layouts(hip, dtype):
    """Other layouts are copied, results have channels-last memory; odd items inside a larger tensor start at any address."""
    c = case(2, 12, 3, (9, 7), dtype, "gelu", True, "float")
    plain = run(c)
    other = run(c, layout=lambda t: t.movedim(-1, 1).contiguous())
    from box_convolution import group_norm_act
    y = group_norm_act(c["x"].cuda().movedim(-1, 1), 3)
    assert y.is_contiguous(memory_format=torch.channels_last)
    for k in plain:
        assert torch.equal(plain[k], other[k]), k

    def inside(t):
        big = torch.full((t.numel() + 3,), float("nan"), dtype=t.dtype, device="cuda")
        view = big[1:1 + t.numel()].view(t.shape)
        view.copy_(t)
        return view.movedim(-1, 1)
    for size in ((3, 5, 1, (9, 7)), (3, 5, 1, (181, 191)), (3, 48, 6, (131, 91))):
        c = case(*size, dtype, "silu", True, "float")
        ref.check(run(c, layout=inside), expected(c))


def test_empty(hip):
    for shape in ((0, 8, 3, 3), (2, 8, 0, 3)):
        from box_convolution import group_norm_act
        x = torch.zeros(shape, device="cuda", requires_grad=True)
        w, b = (torch.ones(8, device="cuda", requires_grad=True) for _ in range(2))
        y = group_norm_act(x, 4, w, b, activation="silu")
        grads = torch.autograd.grad(y, (x, w, b), torch.zeros_like(y))
        assert y.shape == shape and grads[0].shape == shape and not grads[1].any() and not grads[2].any()


@pytest.mark.parametrize("name", [None, "silu", "gelu"])
def test_gradients_against_differences(hip, name):
    """As for the pointwise product (tests/test_gpu_linear_act.py)."""
    h = 2.0 ** -7
    for size in ((2, 12, 3, (6, 5)), (1, 12, 3, (160, 120))):
        c = case(*size, torch.float32, name, True, "float", seed=6)
        grads = run(c)
        gen = torch.Generator().manual_seed(2)
        g = c["grad"].double()
        for which in ("x", "weight", "bias", "residual"):
            v = torch.randn(c[which].shape, generator=gen, dtype=torch.float64)

            def loss(step, exact):
                moved = c[which].double() + step * v
                t = dict(c, grad=None, **{which: moved if exact else moved.float()})
                y = expected(t)["y"][0].reshape(g.shape) if exact else run(t)["y"].double().cpu()
                return (y * g).sum().item()
            quotient = (loss(h, False) - loss(-h, False)) / (2 * h)
            exact = [(loss(s, True) - loss(-s, True)) / (2 * s) for s in (h, 2 * h)]
            bound = (expected(dict(c, grad=None))["y"][1].reshape(g.shape) * g.abs()).sum().item()
            rounding = 2.0 ** -24 * (c[which].double().abs() * grads[which].double().cpu().abs()).sum().item()
            got = (grads[which].double().cpu() * v).sum().item()
            assert abs(got - quotient) <= 2 * (bound + rounding) / h + 2 * abs(exact[1] - exact[0]) + 1e-6 * abs(got), which


def test_only_what_is_needed(hip):
    from box_convolution import group_norm_act
    for size in ((2, 12, 3, (6, 5)), (1, 16, 4, (160, 120)), (1, 1031, 1, (3, 5))):
        c = case(*size, torch.float16, "silu", True, "same")
        full = run(c)
        dev = {k: c[k].cuda() for k in ("x", "weight", "bias", "residual")}
        for which in dev:
            t = {k: (v.movedim(-1, 1) if v.dim() > 1 else v).detach().requires_grad_(k == which) for k, v in dev.items()}
            y = group_norm_act(t["x"], c["groups"], t["weight"], t["bias"], t["residual"], "silu", EPS)
            got = torch.autograd.grad(y, t[which], c["grad"].cuda().movedim(-1, 1))[0]
            assert torch.equal(got.movedim(1, -1) if got.dim() > 1 else got, full[which]), which


def test_another_stream_and_same_bits(hip):
    c = case(2, 48, 6, (131, 77), torch.bfloat16, "gelu", True, "float")
    first = run(c)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        second = run(c)
    side.synchronize()
    for k in first:
        assert torch.equal(first[k], second[k]), k


def test_graph_replays(hip):
    for size in ((2, 24, 4, (12, 13)), (2, 24, 4, (130, 140))):
        c = case(*size, torch.bfloat16, "silu", True, "float")
        x, w, b, r, g = (c[k].cuda() for k in ("x", "weight", "bias", "residual", "grad"))

        def step():
            y, mean, rstd = hip.group_norm_forward(x, 4, w, b, r, "silu", EPS, True)
            return [y] + hip.group_norm_backward(x, 4, w, b, r, "silu", mean, rstd, g, (True,) * 4)
        side = torch.cuda.Stream()
        with torch.cuda.stream(side):
            step()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            captured = step()
        for k in range(3):
            x.copy_(x.roll(k + 1, 1))
            graph.replay()
            torch.cuda.synchronize()
            got = [t.clone() for t in captured]
            for a, e in zip(got, step()):
                assert torch.equal(a, e)


def test_output_in_place_of_an_input(hip):
    """The C entry may write its output over the input or the residual."""
    lib = hip.load()
    for size in ((2, 24, 4, (12, 13)), (2, 24, 4, (130, 140)), (1, 1031, 1, (3, 5))):
        c = case(*size, torch.float32, "relu", True, "float", train=False)
        B, C = c["x"].size(0), c["x"].size(-1)
        pixels = c["x"].numel() // (B * C)
        plain = run(c)["y"].reshape(-1)
        n = lib.boxconv_group_norm_workspace_bytes(B, pixels, C, c["groups"], 0, 0)
        ws = torch.empty(max(n, 16), dtype=torch.uint8, device="cuda")
        for over in ("x", "residual"):
            d = {k: c[k].cuda().contiguous() for k in ("x", "weight", "bias", "residual")}
            rc = lib.boxconv_group_norm_forward(d["x"].data_ptr(), d["weight"].data_ptr(), d["bias"].data_ptr(), 0, d["residual"].data_ptr(),
                                                d[over].data_ptr(), None, None, 0, B, pixels, C, c["groups"], EPS, 1, ws.data_ptr(), n,
                                                torch.cuda.current_stream().cuda_stream)
            assert rc == 0
            assert torch.equal(d[over].reshape(-1), plain)


def test_module_is_group_norm(hip):
    from box_convolution import GroupNormAct
    torch.manual_seed(1)
    module = GroupNormAct(4, 24, activation="relu").cuda()
    torch.nn.init.normal_(module.weight)
    torch.nn.init.normal_(module.bias)
    plain = torch.nn.GroupNorm(4, 24).double()
    plain.load_state_dict(module.state_dict())
    x, r = torch.randn(2, 24, 9, 13), torch.randn(2, 24, 9, 13)
    with torch.no_grad():
        e = torch.relu(plain(x.double()) + r.double())
    got = module(x.cuda(), r.cuda())
    assert (got.double().cpu() - e).abs().max() <= 2.0 ** -18 * 8       # (two dozen roundings of values up to 8)


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
    for name in ACTS:
        c = case(2, 12, 3, (9, 7), dtype, name, name != "relu", "float" if name else "none")
        ref.check(run(c), expected(c))
        other = run(c, layout=lambda t: t.movedim(-1, 1).contiguous())
        assert all(torch.equal(t, other[k]) for k, t in run(c).items())


def test_refusals(host_side):
    from box_convolution import GroupNormAct, group_norm_act
    x = torch.zeros(2, 8, 3, 3, device="cuda")
    one = torch.ones(8, device="cuda")
    for bad, match in ((lambda: group_norm_act(x, 3), "groups"), (lambda: group_norm_act(x, 0), "groups"),
                       (lambda: group_norm_act(x[:, :0], 1), "groups"), (lambda: group_norm_act(x, 4, one[:7]), "weight"),
                       (lambda: group_norm_act(x, 4, one.half()), "float32"), (lambda: group_norm_act(x.half(), 4, one, one.half()), "weight and bias"),
                       (lambda: group_norm_act(x, 4, one.cpu()), "weight"), (lambda: group_norm_act(x, 4, residual=x[:1]), "residual"),
                       (lambda: group_norm_act(x, 4, residual=x.half()), "residual"),
                       (lambda: group_norm_act(x, 4, activation="tanh"), "activation"), (lambda: group_norm_act(x.double(), 4), "float32, float16 or bfloat16"),
                       (lambda: group_norm_act(x.cpu(), 4), "AMD GPUs only"), (lambda: group_norm_act(x[:, 0, 0, 0], 1), ">=2 dimensions"),
                       (lambda: GroupNormAct(2, 8, activation=1), "activation")):
        with pytest.raises(RuntimeError, match=match):
            bad()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("size", [(2, 1031, 1, (41, 67)), (1, 2053, 2053, (7, 50)), (3, 3077, 17, (10, 11)), (1, 1, 1, (1, 1)), (2, 3, 1, (1, 2))])
def test_channels_that_no_lanes_repeat_over(hip, size, dtype):
    """Element by element, the pixels cut into chunks: one group, a group per channel, a last chunk that is shorter."""
    for name, residual, params in (("silu", True, "float"), (None, False, "none")):
        c = case(*size, dtype, name, residual, params)
        ref.check(run(c), expected(c))


def test_not_twice(host_side):
    """Gradients of gradients are refused, not taken for zero; asking for a graph alone changes no gradient."""
    from box_convolution import group_norm_act
    x, w = torch.randn(2, 8, 3, 3, device="cuda", requires_grad=True), torch.ones(8, device="cuda", requires_grad=True)
    once = torch.autograd.grad(group_norm_act(x, 4, w, activation="silu").sum(), [x, w])
    again = torch.autograd.grad(group_norm_act(x, 4, w, activation="silu").sum(), [x, w], create_graph=True)
    assert all(torch.equal(a, b) for a, b in zip(once, again))
    for g in again:
        with pytest.raises(RuntimeError, match="not twice"):
            g.square().sum().backward()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("size", [(2, 20, 4, (9, 10)), (2, 64, 2, (50, 60)), (2, 32, 8, (130, 131)), (1, 1031, 1, (3, 5))])
def test_relu_backward_sees_the_forwards_sign(hip, size, dtype):
    """The residual's gradient is grad_output exactly where the output is positive and 0 elsewhere: the backward forms the
    value in front of the activation again, to the same bits. (An output that is positive but rounds to 0 in float16
    has a gradient all the same.)"""
    c = case(*size, dtype, "relu", True, "float", seed=11)
    out = {k: t.reshape(-1).cpu() for k, t in run(c).items()}
    grad, live = c["grad"].reshape(-1), out["y"] > 0
    assert torch.equal(out["residual"][live], grad[live])
    rest = out["residual"][~live]
    assert int((rest != 0).sum()) == 0 or dtype == torch.float16 and int((rest != 0).sum()) < 10


def test_more_than_2_31_elements(hip):
    """An item of more than 2^31 elements: the result is the one of the same values in a smaller item (every row repeated:
    the statistics are the same up to their rounding), at its far end too."""
    from box_convolution import group_norm_act
    C, repeats, small = 32, 1040, 64 * 1024
    gen = torch.Generator(device="cuda").manual_seed(0)
    base = torch.randn(small, C, generator=gen, device="cuda")
    x = base.to(torch.bfloat16).repeat(repeats, 1)[None].movedim(-1, 1).requires_grad_(True)
    assert x.numel() > 1 << 31
    y = group_norm_act(x, 8, activation="silu")
    xs = base.to(torch.bfloat16)[None].movedim(-1, 1).requires_grad_(True)
    ys = group_norm_act(xs, 8, activation="silu")
    for k in (0, repeats // 2, repeats - 1):
        part = y[:, :, k * small:(k + 1) * small]
        assert (part.float() - ys.float()).abs().max() <= 2.0 ** -8 * ys.float().abs().max()          # one bfloat16 rounding either way
    g = torch.randn(small, C, generator=gen, device="cuda").to(torch.bfloat16)
    dxs = torch.autograd.grad(ys, xs, g[None].movedim(-1, 1))[0].float()
    dx = torch.autograd.grad(y, x, g.repeat(repeats, 1)[None].movedim(-1, 1))[0]
    for k in (0, repeats - 1):
        assert (dx[:, :, k * small:(k + 1) * small].float() - dxs).abs().max() <= 2.0 ** -8 * dxs.abs().max()


def _as_rows(t):
    """What saving to the CPU and back makes of a tensor: the same values in torch's default memory order."""
    return torch.empty(t.shape, dtype=t.dtype, device=t.device).copy_(t)


def _turned(t):
    return t.transpose(0, -1).contiguous().transpose(0, -1) if t.dim() > 1 else torch.stack((t, t), 1)[:, 0]


@pytest.mark.parametrize("unpack", [_as_rows, _turned])
def test_saved_tensors_of_another_layout(host_side, unpack):
    """Hooks on saved tensors may give the values back in any memory order."""
    for size in ((2, 12, 3, (9, 7)), (1, 24, 4, (130, 140)), (3, 8, 4, ())):
        for name in (None, "gelu"):
            c = case(*size, torch.float32, name, True, "float")
            plain = run(c)
            with torch.autograd.graph.saved_tensors_hooks(lambda t: t, unpack):
                hooked = run(c)
            for k in plain:
                assert torch.equal(plain[k], hooked[k]), (k, size, name)


def test_forward_mode_is_refused(host_side):
    """A tangent on any input, or on the gradient, is refused and not dropped, whether or not gradients are recorded."""
    import torch.autograd.forward_ad as forward_ad
    from box_convolution import group_norm_act
    x, r = torch.randn(2, 8, 3, 3, device="cuda"), torch.randn(2, 8, 3, 3, device="cuda")
    w, b = torch.randn(8, device="cuda"), torch.randn(8, device="cuda")
    with forward_ad.dual_level():
        for i in range(4):
            args = [forward_ad.make_dual(t, torch.ones_like(t)) if i == k else t for k, t in enumerate((x, w, b, r))]
            for recorded in (False, True):
                with torch.set_grad_enabled(recorded), pytest.raises(RuntimeError, match="forward-mode"):
                    group_norm_act(args[0], 4, *args[1:], activation="silu")
        leaf = x.clone().requires_grad_(True)
        y = group_norm_act(leaf, 4, w, b, r, "silu")
        with pytest.raises(RuntimeError, match="forward-mode"):
            torch.autograd.grad(y, leaf, forward_ad.make_dual(torch.ones_like(y), torch.ones_like(y)))
        assert torch.equal(group_norm_act(x, 4, w, b, r, "silu"), y)


@pytest.mark.parametrize("size", [(100001, 64, 8, ()), (30001, 8, 2, (2, 2)), (4097, 1031, 1, ()), (70003, 3, 1, ()), (257, 4, 2, (92, 91)), (4095, 16, 4, ())])
def test_parameter_gradients_over_many_items(hip, size):
    """The sums over the batch are joined as the others are: as many float32 additions in a row as the bound allows, whatever the batch.
    The same gradient everywhere, as a mean has it: in one chain of additions its roundings would add up."""
    c = case(*size, torch.float32, None, False, "float")
    c["grad"] = torch.full_like(c["grad"], 1.1)
    ref.check(run(c), expected(c))


@pytest.mark.parametrize("B,C,G", [(5000003, 4, 4), ((1 << 26) + 3, 8, 2)])
def test_more_workgroups_than_a_grid_takes(hip, B, C, G):
    """Items whose workgroups have 2^32 threads and more together (a workgroup per item and channel, and one per item): the first, the last
    and those around every 2^22nd are those of the same items alone, and the parameters' gradients the sums over parts."""
    from box_convolution import group_norm_act
    gen = torch.Generator(device="cuda").manual_seed(0)
    x, g = (torch.randn(B, C, generator=gen, device="cuda", dtype=torch.bfloat16) for _ in range(2))
    w, b = (torch.randn(C, generator=gen, device="cuda").requires_grad_(True) for _ in range(2))

    def both(part):
        xs = x[part].detach().requires_grad_(True)
        y = group_norm_act(xs, G, w, b, activation="silu")
        return (y.detach(), *torch.autograd.grad(y, (xs, w, b), g[part]))
    y, dx, dw, db = both(slice(0, B))
    for at in [0, B - 500] + list(range((1 << 22) - 250, B - 500, 1 << 22)):
        part = slice(at, at + 500)
        some = both(part)
        assert torch.equal(some[0], y[part]) and torch.equal(some[1], dx[part]), at
    step, sums = B // 4 + 1, [0.0, 0.0]
    for at in range(0, B, step):
        some = both(slice(at, at + step))
        sums = [s + t.double() for s, t in zip(sums, some[2:])]
    # (512 additions in a row, of B values of the size 1 to 4 that mostly cancel: both ways)
    for got, want in zip((dw, db), sums):
        assert (got.double() - want).abs().max() <= 2 * ref.DEPTH * ref.U32 * 4 * B


def test_nothing_to_sum_at_the_c_entry(hip):
    """Without rows the parameters' gradients are sums of nothing: 0, written by the call."""
    lib, stream = hip.load(), torch.cuda.current_stream().cuda_stream
    gw, gb = torch.full((8,), float("nan"), device="cuda"), torch.full((8,), float("nan"), device="cuda", dtype=torch.float32)
    for batch, pixels in ((0, 9), (2, 0)):
        gw.fill_(float("nan")), gb.fill_(float("nan"))
        assert lib.boxconv_group_norm_backward(None, None, None, 0, None, None, None, None, None, gw.data_ptr(), gb.data_ptr(), None, 1, batch, pixels, 8, 2,
                                               0, None, 0, stream) == 0
        assert not gw.any() and not gb.any()


def test_most_channels(hip):
    """More channels than the backward takes, in the forward: one item of 2^24 + 3 channels in one group."""
    from box_convolution import group_norm_act
    x = torch.randn(2, (1 << 24) + 3, generator=torch.Generator(device="cuda").manual_seed(0), device="cuda")
    y = group_norm_act(x, 1)
    d = x.double()
    d = (d - d.mean(1, keepdim=True)) / (d.var(1, unbiased=False, keepdim=True) + EPS).sqrt()
    assert (y - d).abs().max() <= ref.DEPTH * ref.U32 * x.abs().max()
    with pytest.raises(RuntimeError, match="too many"):
        group_norm_act(x.requires_grad_(True), 1).sum().backward()
