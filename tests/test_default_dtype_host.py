"""The float32 outputs of the row operators, which the kernels write 4 bytes an
element, are float32 whatever torch's default type is."""
import pytest
import torch


@pytest.mark.parametrize('default', [torch.float64, torch.bfloat16, torch.float16])
def test_outputs_are_float32(default):
    from d1 import _rows
    cpu, was = torch.device('cpu'), torch.get_default_dtype()
    _rows._F32.pop(cpu, None)
    torch.set_default_dtype(default)
    try:
        for shape in ((), (3,), (3, 2), ((4, 5),)):
            assert _rows.empty_f32(cpu, *shape).dtype is torch.float32
    finally:
        torch.set_default_dtype(was)
        _rows._F32.pop(cpu, None)
