"""Which gates ``residual_norm`` takes for which inputs, without a GPU (its Python host side; tests/test_gpu_residual_norm_items.py has both)."""
import pytest
import torch

from box_convolution import _native
from box_convolution.operators import _gate_kind


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
def test_gates_of_every_shape_and_type(dtype):
    for shape in ((3, 8), (3, 8, 5), (3, 8, 2, 4)):
        x = torch.zeros(shape, dtype=dtype)
        assert _gate_kind(None, x) == _native.GATE_NONE
        for gate_type in (dtype, torch.float32):
            assert _gate_kind(torch.zeros(8, dtype=gate_type), x) == _native.GATE_CHANNEL
            # an input without further dimensions: a gate per item is one per element too
            want = _native.GATE_FULL if x.dim() == 2 and gate_type == dtype else _native.GATE_ITEM
            assert _gate_kind(torch.zeros(3, 8, dtype=gate_type), x) == want
        assert _gate_kind(torch.zeros_like(x), x) == _native.GATE_FULL
        for gate in (torch.zeros(9, dtype=dtype), torch.zeros(8, dtype=torch.float64), torch.zeros(3, 8, dtype=torch.float64), torch.zeros(2, 8, dtype=dtype)):
            with pytest.raises(RuntimeError, match="gate must"):
                _gate_kind(gate, x)
        if dtype != torch.float32 and x.dim() > 2:
            with pytest.raises(RuntimeError, match="float32"):
                _gate_kind(torch.zeros(shape), x)
