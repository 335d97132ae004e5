"""The tensors that an AdamW step writes share no memory with one another or with
the gradients (the checks alone, on host tensors)."""
import pytest
import torch


def test_written_tensors_are_apart():
    from d1.adamw import _spans
    flat, half = torch.zeros(100), torch.zeros(100, dtype=torch.bfloat16)
    spans = _spans([('b', flat[50:]), ('a', flat[:50]), ('none', flat[:0]), ('copy', half)])
    assert sorted(spans[2]) == ['a', 'b', 'copy'] and list(spans[0]) == sorted(spans[0])
    assert _spans([('none', flat[:0])]) == ((), (), ())
    for bad in ([('a', flat), ('b', flat)], [('a', flat[:51]), ('b', flat[50:])], [('a', flat), ('b', flat[30:31])],
                [('a', flat), ('copy', flat.view(torch.bfloat16)[199:])]):
        with pytest.raises(ValueError):
            _spans(bad)


def test_gradients_are_outside():
    from d1.adamw import _outside, _spans
    flat = torch.zeros(100)
    spans = _spans([('a', flat[10:20]), ('b', flat[30:40]), ('c', flat[40:41])])
    for i in range(100):
        for n in (0, 1, 5, 12):
            part = flat[i:i + n]
            cells = set(range(i, min(100, i + n)))
            if cells & (set(range(10, 20)) | set(range(30, 41))):
                with pytest.raises(ValueError):
                    _outside(part, 'g', spans)
            else:
                _outside(part, 'g', spans)
    _outside(flat, 'g', _spans([]))
