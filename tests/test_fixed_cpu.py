"""CPU: an object whose calls pass pointers that were taken once keeps the tensors they are of."""

import pytest
import torch


def test_a_weight_keeps_its_tensors():
    from fp8 import CODES, Fp8Weight
    w = Fp8Weight.__new__(Fp8Weight)
    w._keep(None, torch.zeros(3, 64).to(CODES), torch.ones(1, 1))
    q, scale = w.q, w.scale
    for name, other in (("q", q.clone()), ("scale", scale.clone()), ("rows", 2), ("cols", 48)):
        with pytest.raises(AttributeError, match=name):
            setattr(w, name, other)
    assert w.q is q and w.scale is scale and (w.rows, w.cols) == (3, 64)
    w.scale.fill_(2)
    assert (w.values() == 0).all() and w.values().shape == (3, 64)
