"""Temperatures without a finite fp32 reciprocal, and infinite ones, are refused by the C
entries and by the Python calls (before any CUDA call)."""
import math

import pytest
import torch

BAD, P = 9002, 1 << 20
REFUSED = (0.0, -1.0, 1e-46, 1e-39, 1.1e-38, math.inf, math.nan, -math.inf)


def test_c_entries():
    from d1 import _lib
    lib = _lib.library()
    for t in REFUSED:
        assert lib.d1_token_logprob(P, 40, 1, 2, 40, P, None, 0, t, 0, P, P, P, None, None, None) == BAD, t
        assert lib.d1_token_logprob_backward(P, 40, 1, 2, 40, P, None, 0, t, P, P, P, P, 2 * P, 40, None) == BAD, t
    for t in (1.2e-38, 1.0, 3e38):  # no rows: nothing is launched
        assert lib.d1_token_logprob(P, 40, 1, 0, 40, P, None, 0, t, 0, P, P, P, None, None, None) == 0, t


def test_python_calls(monkeypatch):
    from d1 import token_logprob as M
    monkeypatch.setattr(M, 'type_of', lambda t, name: 0)  # the temperature's check comes after the device's
    x, tokens = torch.zeros(4, 40), torch.zeros(4, dtype=torch.int64)
    for t in REFUSED + (4e38,):
        with pytest.raises(ValueError, match='temperature'):
            M.token_logprob(x, tokens, temperature=t)
        with pytest.raises(ValueError, match='temperature'):
            M.token_logprob_backward(x, tokens, None, None, None, temperature=t)
