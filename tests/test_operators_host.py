"""The operators' entry points without a GPU: argument errors that the C ABI reports before anything is launched, sizes
of workspaces, modules that share their parameters with torch's."""
import ctypes

import pytest
import torch


@pytest.fixture(scope="module")
def lib():
    from box_convolution import _native
    return _native.load()


P = ctypes.c_void_p(256)


def norm(lib, x=P, out=P, dtype=0, param=0, batch=2, pixels=9, channels=8, groups=4, act=0, mean=None, rstd=None, ws=None, n=0):
    return lib.boxconv_group_norm_forward(x, P, P, param, None, out, mean, rstd, dtype, batch, pixels, channels, groups, 1e-5, act, ws, n, None)


def test_group_norm_argument_errors(lib):
    for kw, code, text in (({"dtype": 3}, -1, b"dtype"), ({"dtype": 1, "param": 2}, -1, b"param_dtype"), ({"groups": 3}, -1, b"sizes"),
                           ({"channels": 0}, -1, b"sizes"), ({"batch": -1}, -1, b"sizes"), ({"act": 4}, -1, b"activation"),
                           ({"x": None}, -1, b"null"), ({"out": None}, -1, b"null"), ({"mean": P}, -1, b"mean"),
                           ({"batch": 1 << 31}, -3, b"too many"), ({"pixels": 1 << 20, "channels": 64, "groups": 1}, -2, b"workspace")):
        assert norm(lib, **kw) == code, kw
        assert text in lib.boxconv_last_error(), lib.boxconv_last_error()
    assert norm(lib, batch=0, x=None, out=None) == 0 and norm(lib, pixels=0, x=None) == 0
    back = lib.boxconv_group_norm_backward
    assert back(P, P, P, 0, None, P, P, P, None, None, None, None, 0, 2, 9, 8, 4, 0, None, 0, None) == 0     # nothing wanted
    assert back(P, P, P, 0, None, P, None, P, P, None, None, None, 0, 2, 9, 8, 4, 0, None, 0, None) == -1
    assert back(P, P, P, 0, None, P, P, P, P, None, None, None, 0, 2, 9, 8, 4, 0, None, 0, None) == -2
    assert b"workspace" in lib.boxconv_last_error()


def test_linear_argument_errors(lib):
    def forward(x=P, ld=8, w=P, ldr=0, out=P, dtype=0, rows=4, K=8, N=6, act=0, ws=None, n=0):
        return lib.boxconv_linear_forward(x, ld, w, None, None, ldr, out, None, dtype, rows, K, N, act, ws, n, None)
    for kw, code, text in (({"dtype": 16}, -1, b"dtype"), ({"rows": -1}, -1, b"sizes"), ({"ld": -1}, -1, b"sizes"), ({"act": -1}, -1, b"activation"),
                           ({"ldr": -2}, -1, b"ld_residual"), ({"x": None}, -1, b"null"), ({"w": None}, -1, b"null"), ({"out": None}, -1, b"null"),
                           ({"rows": 1 << 41}, -3, b"too large"), ({"N": 1 << 31}, -3, b"too large"), ({"K": 1 << 20, "N": 64}, -2, b"workspace")):
        assert forward(**kw) == code, kw
        assert text in lib.boxconv_last_error(), lib.boxconv_last_error()
    assert forward(rows=0, x=None, w=None, out=None) == 0 and forward(N=0, w=None, out=None) == 0
    back = lib.boxconv_linear_backward
    assert back(P, 8, P, P, None, None, None, None, None, 0, 4, 8, 6, 0, None, 0, None) == 0                 # nothing wanted
    assert back(P, 8, P, P, None, P, None, None, None, 0, 4, 8, 6, 2, None, 0, None) == -1                   # silu without its slope
    assert b"kept" in lib.boxconv_last_error()
    assert back(P, 8, P, P, None, P, P, P, None, 0, 4, 8, 6, 0, None, 0, None) == -2


def test_workspace_sizes(lib):
    assert lib.boxconv_group_norm_workspace_bytes(4, 784, 40, 8, 2, 0) == 0          # one launch
    assert lib.boxconv_group_norm_workspace_bytes(4, 128 * 256, 128, 32, 2, 0) > 0
    assert lib.boxconv_group_norm_workspace_bytes(4, 784, 40, 8, 2, 1) >= 4 * 40 * 8  # two sums per item and channel
    assert lib.boxconv_group_norm_workspace_bytes(4, 784, 40, 7, 2, 1) == 0          # refused sizes
    assert lib.boxconv_linear_workspace_bytes(0, 8, 8, 0, 1) == 0
    for dtype in (0, 1, 2):
        assert lib.boxconv_linear_workspace_bytes(8192, 4096, 4096, dtype, 0) == 0   # enough tiles without a split


def test_no_cpu_path():
    from box_convolution import group_norm_act, linear_act
    with pytest.raises(RuntimeError, match="AMD GPUs only"):
        linear_act(torch.zeros(2, 3), torch.zeros(4, 3))
    with pytest.raises(RuntimeError, match="AMD GPUs only"):
        group_norm_act(torch.zeros(2, 4, 3, 3), 2)


def test_modules_share_parameters_with_torchs():
    from box_convolution import GroupNormAct, PointwiseConv2d
    a, b = PointwiseConv2d(5, 7, activation="silu"), torch.nn.Conv2d(5, 7, 1)
    b.load_state_dict(a.state_dict())
    a, b = GroupNormAct(2, 8, activation="relu"), torch.nn.GroupNorm(2, 8)
    b.load_state_dict(a.state_dict())
    assert "relu" in repr(a)


def test_reference_against_torch():
    """The 64-bit formulas of the tests against torch's own layers and autograd, on the CPU."""
    import operator_reference as ref
    torch.manual_seed(0)
    acts = {None: lambda z: z, "relu": torch.relu, "silu": torch.nn.functional.silu, "gelu": torch.nn.functional.gelu}
    for name, f in acts.items():
        x, w, b, r, g = (torch.randn(s, dtype=torch.float64) for s in ((6, 5), (4, 5), (4,), (6, 4), (6, 4)))
        leaves = [t.requires_grad_(True) for t in (x, w, b, r)]
        y = f(torch.nn.functional.linear(x, w, b) + r)
        e = dict(zip(("x", "weight", "bias", "residual"), torch.autograd.grad(y, leaves, g)), y=y)
        got = ref.linear(*[t.detach() for t in leaves], name, g, torch.float32)
        assert all(torch.allclose(got[k][0], e[k]) for k in e) and set(got) == set(e)
        x, r, g = (torch.randn(2, 7, 6, dtype=torch.float64) for _ in range(3))
        w, b = torch.randn(6, dtype=torch.float64), torch.randn(6, dtype=torch.float64)
        leaves = [t.requires_grad_(True) for t in (x, w, b, r)]
        y = f(torch.nn.functional.group_norm(x.movedim(-1, 1), 3, w, b, 1e-5).movedim(1, -1) + r)
        e = dict(zip(("x", "weight", "bias", "residual"), torch.autograd.grad(y, leaves, g)), y=y)
        got = ref.group_norm(*[x.detach(), 3] + [t.detach() for t in leaves[1:]], name, 1e-5, g, torch.float32, torch.float32)
        assert all(torch.allclose(got[k][0], e[k]) for k in e) and set(got) == set(e)


@pytest.mark.parametrize("call", ["norm", "norm_backward", "linear", "linear_backward"])
def test_scratch_of_calls_that_overlap(monkeypatch, call):
    """Two threads may launch on one stream in turn: while one call's kernels are being launched, another's must not get the same scratch
    memory. (The native library is replaced by one that starts the other call from within the first.)"""
    import contextlib
    import threading
    from box_convolution import _native
    x, w, g = torch.zeros(6, 8), torch.zeros(8, 8), torch.zeros(6, 8)
    stat = torch.zeros(6, 2)
    calls = {"norm": lambda: _native.group_norm_forward(x, 2, None, None, None, None, 1e-5, False),
             "norm_backward": lambda: _native.group_norm_backward(x, 2, None, None, None, None, stat, stat, g, (True, False, False, False)),
             "linear": lambda: _native.linear_forward(x, w, None, None, None, False),
             "linear_backward": lambda: _native.linear_backward(x, w, None, None, g, (True, True, False, False))}
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
    monkeypatch.setattr(_native, "_workspaces", {})
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)
    calls[call]()
    assert len(seen) == 2 and None not in seen and seen[0] != seen[1]


def test_sizes_that_no_launch_takes(lib):
    """A grid has fewer than 2^32 threads: one item's or one row of tiles' workgroups have to fit, and are refused where they do not."""
    most = (1 << 24) - 1
    assert norm(lib, batch=1, pixels=1, channels=most + 1, groups=most + 1) == -3 and b"too many" in lib.boxconv_last_error()
    assert norm(lib, batch=1, pixels=1, channels=most + 1, groups=1) == -2           # (a workspace is all that is missing)
    for channels, code in ((most, -2), (most + 1, -3)):
        assert lib.boxconv_group_norm_backward(P, P, P, 0, None, P, P, P, P, None, None, None, 0, 1, 1, channels, 1, 0, None, 0, None) == code
    back = lib.boxconv_linear_backward
    for K, code in ((64 * most, -2), (64 * most + 1, -3)):
        assert back(P, K, P, P, None, P, None, None, None, 1, 100, K, 1, 0, None, 0, None) == code, K
    assert b"too large" in lib.boxconv_last_error()
