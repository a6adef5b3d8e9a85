"""Layouts of rows that the row operators take, on the CPU: what a tensor's leading dimensions are as rows of one pitch."""
import pytest
import torch

from flyhigh_engine_b200 import kernels as K


@pytest.mark.parametrize("shape", [(0, 16), (0, 5, 16), (5, 0, 16), (2, 0, 3, 16), (2, 3, 0, 16), (1, 0, 16), (0, 1, 1, 13), (3, 0, 13)], ids=str)
def test_no_rows_in_any_dimension(shape):
    """An empty dimension makes no rows wherever it is, whatever strides the others are left with."""
    t = torch.zeros(shape, dtype=torch.float16)
    assert K._rows("t", t, shape[-1], t.dtype, t.device)[2] == 0
    if len(shape) > 2:
        t = torch.zeros(*shape[:-1], shape[-1] + 5, dtype=torch.float16)[..., :shape[-1]].transpose(0, 1)
        assert K._rows("t", t, shape[-1], t.dtype, t.device)[2] == 0
    out = K._rows_like(t)
    assert out.shape == t.shape and K._rows("out", out, shape[-1], t.dtype, t.device)[2] == 0
