"""What lies between residual blocks and the 8-bit product without a GPU: argument errors that the C ABI reports before anything is
launched, sizes of workspaces, and the tests' own 64-bit formulas against torch's."""
import ctypes

import pytest
import torch

P = ctypes.c_void_p(256)


@pytest.fixture(scope="module")
def lib():
    from box_convolution import _native
    return _native.load()


def forward(lib, x=P, residual=None, gate=None, kind=0, gate_dtype=0, norms=3, param=0, stream=P, normed=P, exponents=None, statistics=None, dtype=0, batch=2, pixels=9, channels=8):
    return lib.boxconv_residual_norm_forward(x, residual, gate, kind, gate_dtype, 1.0, norms, P, P, P, P, param, 1e-6, stream, normed, exponents, statistics, dtype, batch,
                                             pixels, channels, None)


def backward(lib, gate=None, kind=0, norms=3, grads=(None,) * 7, statistics=None, stream=P, normed=P, x=P, batch=2, pixels=9, channels=8, ws=None, n=0):
    return lib.boxconv_residual_norm_backward(x, None, gate, kind, 0, 1.0, norms, P, P, P, P, 0, 1e-6, statistics, stream, normed, *grads, 0, batch, pixels, channels, ws, n, None)


def test_residual_norm_argument_errors(lib):
    odd = ctypes.c_void_p(264)
    for kw, code, text in (({"dtype": 8}, -1, b"dtype"), ({"dtype": 1, "param": 2}, -1, b"param_dtype"), ({"kind": 4, "gate": P}, -1, b"gate_kind"),
                           ({"kind": 1}, -1, b"do not agree"), ({"gate": P}, -1, b"do not agree"), ({"gate": P, "kind": 1, "gate_dtype": 2}, -1, b"gate_dtype"),
                           ({"gate": P, "kind": 3, "gate_dtype": 0, "dtype": 1, "param": 1}, -1, b"gate_dtype"), ({"norms": 8}, -1, b"norms"),
                           ({"channels": 0}, -1, b"sizes"), ({"batch": -1}, -1, b"sizes"), ({"pixels": -1}, -1, b"sizes"), ({"x": None}, -1, b"null"),
                           ({"norms": 1}, -1, b"BEFORE"), ({"normed": None, "exponents": P}, -1, b"without normed"), ({"normed": odd, "exponents": P}, -1, b"aligned"), ({"statistics": P}, -1, b"do without"), ({"statistics": odd, "channels": 1000}, -1, b"aligned"),
                           ({"batch": 1 << 31}, -3, b"too many"), ({"pixels": 1 << 46}, -3, b"too many"), ({"channels": (1 << 31) - 1}, -3, b"too many")):
        assert forward(lib, **kw) == code, kw
        assert text in lib.boxconv_last_error(), (kw, lib.boxconv_last_error())
    assert forward(lib, batch=0, x=None) == 0 and forward(lib, pixels=0, x=None) == 0 and forward(lib, stream=None, normed=None, norms=1) == 0
    assert backward(lib) == 0                                                        # nothing wanted
    for kw, code, text in (({"grads": (None, None, P, None, None, None, None)}, -1, b"grad_gate"), ({"norms": 2, "grads": (None, None, None, P, None, None, None)}, -1, b"norms"),
                           ({"norms": 1}, -1, b"norms"), ({"norms": 1, "normed": None, "grads": (None,) * 5 + (P, None)}, -1, b"norms"),
                           ({"x": None, "grads": (P,) + (None,) * 6}, -1, b"null"), ({"statistics": P, "grads": (P,) + (None,) * 6}, -1, b"do without"), ({"grads": (None,) * 3 + (P,) + (None,) * 3}, -2, b"workspace")):
        assert backward(lib, **kw) == code, kw
        assert text in lib.boxconv_last_error(), (kw, lib.boxconv_last_error())


def test_float8_argument_errors(lib):
    def quantize(x=P, ld=8, dtype=0, rows=4, columns=8, codes=P, exponents=P):
        return lib.boxconv_quantize_blocks(x, ld, dtype, rows, columns, codes, exponents, None)
    odd = ctypes.c_void_p(258)
    for kw, code, text in (({"dtype": 8}, -1, b"dtype"), ({"rows": -1}, -1, b"sizes"), ({"columns": -1}, -1, b"sizes"), ({"ld": -1}, -1, b"sizes"), ({"x": None}, -1, b"null"),
                           ({"codes": None}, -1, b"null"), ({"exponents": None}, -1, b"null"), ({"codes": odd}, -1, b"aligned"), ({"exponents": odd}, -1, b"aligned"),
                           ({"rows": 1 << 41}, -3, b"too large"), ({"columns": 1 << 31}, -3, b"too large")):
        assert quantize(**kw) == code, kw
        assert text in lib.boxconv_last_error(), lib.boxconv_last_error()
    assert quantize(rows=0, x=None) == 0 and quantize(columns=0, codes=None) == 0

    def product(x=P, ld=8, given=0, xe=None, w=P, we=P, ldr=0, out=P, dtype=0, rows=40, K=8, N=6, act=0, ws=None, n=0):
        return lib.boxconv_linear_float8_forward(x, ld, given, xe, w, we, None, None, ldr, out, dtype, rows, K, N, act, ws, n, None)
    for kw, code, text in (({"dtype": 8}, -1, b"dtype"), ({"given": 1}, -1, b"input_dtype"), ({"rows": -1}, -1, b"sizes"), ({"K": 0}, -1, b"sizes"), ({"ld": -1}, -1, b"sizes"),
                           ({"act": 4}, -1, b"activation"), ({"ldr": -1}, -1, b"ld_residual"), ({"x": None}, -1, b"null"), ({"w": None}, -1, b"null"), ({"we": None}, -1, b"null"),
                           ({"out": None}, -1, b"null"), ({"xe": P}, -1, b"exponents of values"), ({"given": 8}, -1, b"exponents"), ({"given": 8, "xe": odd}, -1, b"aligned"),
                           ({"w": odd}, -1, b"aligned"), ({"given": 8, "x": odd, "xe": P}, -1, b"aligned"), ({"K": (1 << 22) + 1}, -3, b"too large"),
                           ({"rows": 1 << 41}, -3, b"too large"), ({"rows": 4000}, -2, b"workspace")):
        assert product(**kw) == code, kw
        assert text in lib.boxconv_last_error(), (kw, lib.boxconv_last_error())
    assert product(rows=0, x=None) == 0 and product(N=0, w=None) == 0


def test_workspace_sizes(lib):
    assert lib.boxconv_residual_norm_statistics_bytes(4, 100, 512) == 0 and lib.boxconv_residual_norm_statistics_bytes(4, 100, 513) == 4 * 100 * 16
    assert lib.boxconv_residual_norm_statistics_bytes(4, 0, 1000) == 0 and lib.boxconv_residual_norm_statistics_bytes(4, 100, 0) == 0
    assert lib.boxconv_residual_norm_workspace_bytes(4, 100, 40, 1, 2) >= 5 * 40 * 4
    assert lib.boxconv_residual_norm_workspace_bytes(0, 100, 40, 0, 2) == 0 and lib.boxconv_residual_norm_workspace_bytes(4, 100, 0, 0, 2) == 0
    assert lib.boxconv_linear_float8_workspace_bytes(4000, 130, 64, 2, 2) >= 4000 * (256 + 4)      # the input's codes and exponents
    assert lib.boxconv_linear_float8_workspace_bytes(0, 130, 64, 2, 2) == 0


def test_no_cpu_path():
    from box_convolution import Float8Blocks, linear_act_float8, quantize_blocks, residual_norm
    x = torch.zeros(2, 128)
    blocks = Float8Blocks(torch.zeros(2, 128).to(torch.float8_e4m3fn), torch.full((2, 4), 127, dtype=torch.uint8), 100)
    assert blocks.shape == (2, 100) and blocks.dequantize().shape == (2, 100) and blocks.device.type == "cpu"
    for call in (lambda: residual_norm(x, before=(None, None)), lambda: quantize_blocks(x), lambda: linear_act_float8(x, blocks), lambda: linear_act_float8(blocks, blocks)):
        with pytest.raises(RuntimeError, match="AMD GPUs only"):
            call()


def test_norm_reference_against_torch():
    """The tests' formulas against torch's autograd of the definition, on the CPU."""
    import block_reference as ref
    torch.manual_seed(0)
    B, S, C = 2, 5, 12
    for kind in ("rms", "layer"):
        for gate_shape in ((C,), (B, C), (B, S, C)):
            x, r, g = torch.randn(B, S, C, dtype=torch.float64), torch.randn(B, S, C, dtype=torch.float64), torch.randn(gate_shape, dtype=torch.float64)
            params = [torch.randn(C, dtype=torch.float64) for _ in range(4)]
            leaves = [t.requires_grad_(True) for t in (x, r, g, *params)]

            def norm(v, w, b):
                if kind == "layer":
                    return torch.nn.functional.layer_norm(v, (C,), w, b, 1e-6)
                return v * torch.rsqrt(v.square().mean(-1, keepdim=True) + 1e-6) * w + b
            s = r + 0.7 * (g if len(gate_shape) != 2 else g[:, None]) * norm(x, *params[:2])
            h = norm(s, *params[2:])
            gs, gh = torch.randn(B, S, C, dtype=torch.float64), torch.randn(B, S, C, dtype=torch.float64)
            names = ("x", "residual", "gate", "after_weight", "after_bias", "before_weight", "before_bias")
            want = dict(zip(names, torch.autograd.grad([s, h], leaves, [gs, gh])), stream=s, normed=h)
            d = [t.detach() for t in leaves]
            got = ref.residual_norm(d[0], d[1], d[2], 0.7, tuple(d[3:5]), tuple(d[5:]), kind, 1e-6, gs, gh, *(torch.float32,) * 3)
            assert set(got) == set(want) and all(torch.allclose(got[k][0], want[k]) for k in want)


def test_quantize_reference_against_torchs_type():
    """Codes of the tests' own table against torch's conversion to the 8-bit type, on the CPU."""
    import block_reference as ref
    x = torch.randn(7, 300, generator=torch.Generator().manual_seed(0), dtype=torch.float64) * 3
    units, words = ref.quantize(x)
    power = ref.two_to(words[:, :3].to(torch.int64) - 127)
    full = torch.zeros(7, 384, dtype=torch.float64)
    full[:, :300] = x
    scaled = (full.view(7, 3, 128) / power[..., None]).reshape(7, -1)
    assert scaled.abs().max() <= 448
    # (values of float32, which torch converts rounding once)
    x = x.float().double()
    assert torch.equal(scaled.float().to(torch.float8_e4m3fn).double(), ref.quantize(x)[0])
    assert words.shape == (7, 4) and bool((words[:, 3] == 127).all())


def test_modules_hold_what_they_say():
    from box_convolution import ResidualNorm
    m = ResidualNorm(8, kind="layer", layer_scale=1e-4)
    assert sorted(n for n, _ in m.named_parameters()) == ["after_bias", "after_weight", "before_bias", "before_weight", "layer_scale"]
    assert sorted(n for n, _ in ResidualNorm(8, before=False).named_parameters()) == ["after_weight"] and "rms" in repr(ResidualNorm(8))


@pytest.mark.parametrize("call", ["residual_norm_backward", "linear_float8"])
def test_scratch_of_calls_that_overlap(monkeypatch, call):
    """While one call's kernels are being launched, another thread's must not get the same scratch memory. (The native library is replaced by one
    that starts the other call from within the first.)"""
    import contextlib
    import threading
    from box_convolution import _native
    x, w, g = torch.zeros(6, 8), torch.zeros(8, 128).to(torch.float8_e4m3fn), torch.zeros(6, 8)
    e, one = torch.zeros(8, 4, dtype=torch.uint8), torch.ones(8)
    calls = {"residual_norm_backward": lambda: _native.residual_norm_backward(x, None, None, 0, 1.0, 1, [one, None, None, None], 1e-6, None, g, None,
                                                                              (True, False, False, True, False, False, False)),
             "linear_float8": lambda: _native.linear_float8_forward(x, None, w, e, 8, None, None, None, torch.float32)}
    seen = []

    class Library:
        def __getattr__(self, name):
            return self.workspace_bytes if name.endswith("workspace_bytes") else self.entry

        def workspace_bytes(self, *args):
            return 256

        def entry(self, *args):
            seen.append(args[-3])
            if len(seen) == 1:
                other = threading.Thread(target=calls[call])
                other.start()
                other.join()
            return 0
    library = Library()
    monkeypatch.setattr(_native, "load", lambda: library)
    monkeypatch.setattr(_native, "_on_device", lambda device: contextlib.nullcontext())
    monkeypatch.setattr(_native, "_stream", lambda device: 0)
    monkeypatch.setattr(_native, "_workspace_bytes", {})
    calls[call]()
    assert len(seen) == 2 and None not in seen and seen[0] != seen[1]
