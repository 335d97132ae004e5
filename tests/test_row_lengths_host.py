"""Rows that the C entries' int cannot count, and rows of nothing, are refused by name."""
import pytest
import torch


def test_lengths():
    from d1._rows import matrix
    assert matrix(torch.empty(3, 2 ** 31 - 1, device='meta'), 'x')[1:] == (3, 2 ** 31 - 1, 2 ** 31 - 1)
    for shape in ((1, 2 ** 31), (1, 2 ** 32 + 8), (2, 1, 2 ** 33), (2 ** 31 + 1,)):
        with pytest.raises(ValueError, match='longer'):
            matrix(torch.empty(shape, device='meta'), 'x')
    for shape in ((4, 0), (2, 3, 0), (0,), (0, 5, 0)):
        with pytest.raises(ValueError, match='empty'):
            matrix(torch.empty(shape), 'x')
    assert matrix(torch.empty(0, 5, 7), 'x')[1:3] == (0, 7)
