"""What ``Float8Blocks`` and the calls that take it refuse, without a GPU: kernels address codes and exponents by the number of columns, so nothing that was
checked together may come apart."""
import pytest
import torch

from box_convolution import Float8Blocks, _native, linear_act_float8


def blocks(rows=6, columns=200):
    width, words = _native.block_sizes(columns)
    return Float8Blocks(torch.zeros(rows, width).to(torch.float8_e4m3fn), torch.full((rows, words), 127, dtype=torch.uint8), columns)


def other_memory(t, shape):
    t.set_(torch.zeros(shape, dtype=t.dtype))


SPOILED = {"fewer rows of codes": lambda b: b.codes.resize_(3, 256), "fewer codes": lambda b: b.codes.resize_(6, 128), "no exponents": lambda b: b.exponents.resize_(0),
           "fewer rows of exponents": lambda b: b.exponents.resize_(5, 4), "other exponents": lambda b: other_memory(b.exponents, (6, 2)),
           "rows apart": lambda b: (b.codes.set_(b.codes.untyped_storage(), 0, (3, 256), (512, 1)), b.exponents.resize_(3, 4)),
           "one more dimension": lambda b: other_memory(b.exponents, (1, 6, 4))}


def test_nothing_can_be_assigned():
    b = blocks()
    for name, value in (("codes", b.codes.clone()), ("exponents", b.exponents.clone()), ("columns", 100), ("other", 1)):
        with pytest.raises(AttributeError):
            setattr(b, name, value)
    assert b.columns == 200 and b.shape == (6, 200)
    b.codes.view(torch.uint8).fill_(56)                                     # (values may change: code 56 is 1)
    assert bool((b.dequantize() == 1).all())


@pytest.mark.parametrize("how", SPOILED)
def test_calls_look_again(how, monkeypatch):
    """Both host sides, on CPU tensors: they refuse before they come to a kernel."""
    monkeypatch.setattr(_native, "_require_device", lambda tensor, what: None)
    glue = _native.glue()
    for side in (False, glue) if glue is not None else (False,):
        monkeypatch.setattr(_native, "_glue", side)
        monkeypatch.setattr(_native, "_stream", lambda device: 0)
        spoiled = blocks()
        SPOILED[how](spoiled)
        for x, w in ((spoiled, blocks()), (blocks(), spoiled), (torch.zeros(4, 200, dtype=torch.bfloat16), spoiled)):
            if side and torch.is_tensor(x):
                continue                                                    # (values on the CPU are refused first there)
            with pytest.raises(RuntimeError, match="Float8Blocks"):
                linear_act_float8(x, w)


def test_values_of_every_exponent():
    """In 64 bits every code times every power is a number; in float32 those from 2^128 on are infinite."""
    import block_reference as ref
    units = torch.cat([ref.CODE_VALUES, -ref.CODE_VALUES[1:]])
    b = Float8Blocks(torch.zeros(254, 256).to(torch.float8_e4m3fn), torch.full((254, 4), 127, dtype=torch.uint8), units.numel())
    b.codes[:, :units.numel()] = units.to(torch.float8_e4m3fn)
    b.exponents[:, :2] = torch.arange(1, 255, dtype=torch.uint8)[:, None]
    want = units * ref.two_to(torch.arange(1, 255) - 127)[:, None]
    assert torch.equal(b.dequantize(torch.float64), want) and torch.equal(b.dequantize(), want.float())
