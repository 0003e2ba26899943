"""Calls of the operators for vocabularies with tensors and values of other kinds: negated views, probabilities far apart."""
import pytest
import torch

from lbtree import _lib, ops
from test_gpu_vocabulary import TYPES, check, inputs

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


@pytest.mark.parametrize("n,f,k", [(1, 8, 20), (5, 40, 3000), (40, 16, 9000), (300, 64, 700), (1100, 30, 5000)])
def test_small_probabilities_keep_their_bits(n, f, k):
    """bfloat16 without a bias holds exponentials in 16 bits before G: 11 significant bits of them, down to 2^-62 of the largest beside
    them. Scores of which one leads by up to 40 (2^-58): each entry of grad_weight, of one row that counts, is p x within half a step of 11
    bits (2^-11), of G (2^-8) and of the result (2^-8), and what the score is off by (`rel` below, as in test_gpu_vocabulary.reference)."""
    gen = torch.Generator(device="cuda").manual_seed(n)
    x = torch.rand((n, f), generator=gen, device="cuda").add_(0.5).to(torch.bfloat16)
    w = (torch.randn((k, f), generator=gen, device="cuda") * 0.1).to(torch.bfloat16)
    y = torch.full((n,), -1, dtype=torch.int64, device="cuda")
    at = n // 2
    y[at] = 3
    # the first feature lifts the label's score, and lowers the others' by up to 38
    w[:, 0] = -torch.linspace(0, 24, k, device="cuda")[torch.randperm(k, generator=gen, device="cuda")].to(torch.bfloat16)
    w[3, 0] = 2.0
    x[at, 0] = 1.5
    loss, gx, gw = ops.linear_log_loss_gradient(x, w, y)
    X, W = x[at].double(), w.double()
    s = W @ X
    p = torch.exp(s - torch.logsumexp(s, 0))
    assert 2.0 ** -62 < float(p.min()) < 2.0 ** -45
    rest = torch.arange(k, device="cuda") != 3
    want = p[rest, None] * X[None, :]
    rel = float(2 * ((f + 8) * 2.0 ** -24 + 2.0 ** -22) * (W.abs() @ X.abs()).max() + 1e-4)
    bound = (2.0 ** -11 + 2 * 2.0 ** -8 + rel) * (1 + 2.0 ** -6)
    assert ((gw[rest].double() - want).abs() <= bound * want).all()


@pytest.mark.parametrize("native", [True, False])
@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("n,f,k", [(2000, 72, 60000), (1200, 520, 90001), (700, 2100, 20000)])
def test_where_memory_is_short(n, f, k, dtype, native, monkeypatch):
    """No room for the workspace that is asked for first: the least is, in pieces of the classes, and gives the same up to rounding."""
    if not native:
        monkeypatch.setattr(ops, "_NATIVE", None)
    size = _lib.lib.lbt_linear_log_loss_workspace_bytes
    kinds = [size(n, f, k, ops._DT_NARROW[TYPES[dtype]], kind) for kind in (1, 2, 5, 6)]
    assert kinds[2] < kinds[0] and kinds[3] < kinds[1]
    asked = []

    def scratch(nbytes, device):
        asked.append(nbytes)
        if nbytes > max(kinds[2:]):
            raise torch.OutOfMemoryError("no room")
        return torch.empty(nbytes, dtype=torch.uint8, device=device)

    monkeypatch.setattr(ops, "_scratch", scratch)
    x, w, y = inputs(n, f, k, dtype, seed=n)
    y[::7] = -1
    x[::7] = float("nan")
    gen = torch.Generator(device="cuda").manual_seed(k)
    bias = torch.randn(k, generator=gen, device="cuda")
    weight = torch.rand(n, generator=gen, device="cuda") + 0.1
    check(x, w, y, dtype)
    assert kinds[0] in asked and kinds[2] in asked
    check(x, w, y, dtype, bias=bias, weight=weight)
    assert kinds[1] in asked and kinds[3] in asked

    def none(nbytes, device):
        raise torch.OutOfMemoryError("no room")

    monkeypatch.setattr(ops, "_scratch", none)
    with pytest.raises(torch.OutOfMemoryError):
        ops.linear_log_loss_gradient(x, w, y)
    with pytest.raises(torch.OutOfMemoryError):
        ops.linear_log_loss(x, w, y)
