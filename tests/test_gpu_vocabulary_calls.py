"""Calls of the operators for vocabularies that tensors of other kinds make: negated views, inputs on the host."""
import numpy as np
import pytest
import torch

from lbtree import _lib, ops
from test_gpu_vocabulary import inputs

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("native", [True, False])
def test_negated_views(native, monkeypatch):
    """The imaginary part of a conjugate is a view whose memory holds the negated values: of one element it is contiguous, too."""
    if not native:
        monkeypatch.setattr(ops, "_NATIVE", None)
    one = torch.complex(torch.zeros(1, device="cuda"), torch.full((1,), 3.0, device="cuda")).conj().imag
    assert one.is_neg() and one.is_contiguous() and float(one) == -3.0
    table = one.view(1, 1)
    token = torch.zeros(1, dtype=torch.int64, device="cuda")
    assert float(ops.embed_rows(table, token)) == -3.0
    assert float(ops.embed_rows_gradient(table, token, 1)) == -3.0
    x, w, y = inputs(12, 24, 60, "f32", seed=3)
    bias, weight = torch.randn(60, device="cuda"), torch.rand(12, device="cuda")
    want = ops.linear_log_loss_gradient(x, w, y, weight, bias)
    neg = torch._neg_view
    got = ops.linear_log_loss_gradient(neg(-x), neg(-w), y, neg(-weight), neg(-bias))
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    for moved in ((neg(-x), w, y, weight, bias), (x, neg(-w), y, weight, bias), (x, w, y, neg(-weight), bias), (x, w, y, weight, neg(-bias)),
                  (x, w, neg(-y), weight, bias)):
        assert all(torch.equal(a, b) for a, b in zip(ops.linear_log_loss_gradient(*moved), want))
    assert torch.equal(ops.linear_log_loss(x, w, neg(-y), neg(-bias)), ops.linear_log_loss(x, w, y, bias))
    tokens = neg(-y)
    assert torch.equal(ops.embed_rows(w, tokens), ops.embed_rows(w, y))
    assert torch.equal(ops.embed_rows_gradient(x, tokens, 60), ops.embed_rows_gradient(x, y, 60))
    # what is written in place is refused
    with pytest.raises(_lib.LbtError):
        ops.embed_rows_gradient(x, y, 60, add_to=neg(torch.zeros((60, 24), device="cuda")))
