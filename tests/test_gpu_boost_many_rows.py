"""Steps of a round with more entries than a launch may have threads (2^32): each is several launches."""
import pytest
import torch

from lbtree import ops

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _large_arrays_go_back():
    yield
    torch.cuda.empty_cache()


def test_gather_rows():
    f = 64
    n = (1 << 32) // f + 1001
    X = torch.arange(50 * f, device="cuda", dtype=torch.float32).view(50, f)
    rows = torch.arange(n, device="cuda") % 53  # three of them outside
    got = ops.gather_rows(X, rows)
    want = torch.cat([X, torch.zeros((3, f), device="cuda")])
    for i in range(0, n, 1 << 22):
        assert torch.equal(got[i:i + (1 << 22)], want[rows[i:i + (1 << 22)]])


def test_leaf_values_and_probabilities():
    k = 8
    n = (1 << 32) // k + 1003
    leaf = torch.arange(7 * k, device="cuda", dtype=torch.float64).view(7, k) / 16
    row_leaf = (torch.arange(n, device="cuda") % 7).to(torch.int32)
    pred = torch.ones((n, k), dtype=torch.float64, device="cuda")
    ops.add_leaf_values(pred, leaf, row_leaf)
    step = 1 << 24
    for i in range(0, n, step):
        assert torch.equal(pred[i:i + step], leaf[row_leaf[i:i + step].long()] + 1)
    init = torch.zeros(k, dtype=torch.float64, device="cuda")
    few = ops.class_probabilities(pred[:7].contiguous(), init)
    got = ops.class_probabilities(pred, init)
    for i in range(0, n, step):
        assert torch.equal(got[i:i + step], few[row_leaf[i:i + step].long()])


@pytest.mark.parametrize("objective", ["squared_error", "log_loss"])
def test_gradients(objective):
    k, few = 4, 40
    n = (1 << 32) // k + 40
    pred = torch.linspace(-2, 2, few * k, dtype=torch.float64, device="cuda").view(few, k)
    y = (torch.arange(few, device="cuda") % k).double()
    if objective == "squared_error":
        y = torch.linspace(1, -3, few * k, dtype=torch.float64, device="cuda").view(few, k)
    w = torch.linspace(0.5, 1.5, few, dtype=torch.float64, device="cuda")
    want = ops.weighted_gradient(objective, y, pred, w, 0.3)
    times = -(-n // few)
    wide = [a.repeat((times,) + (1,) * (a.dim() - 1)) for a in (y, pred, w)]
    g, h = ops.weighted_gradient(objective, *wide, 0.3)
    del wide
    for got, one in zip((g, h), want):
        view = got.view(times, few, k)
        for i in range(0, times, 1 << 20):
            part = view[i:i + (1 << 20)]
            assert torch.equal(part, one.expand(part.shape))
    draw = torch.ones(few * times, dtype=torch.float64, device="cuda")
    draw[::few] = 0.0
    ops.keep_rows(draw, 0.5, g, h)  # the first row of each forty is kept
    for got, one in zip((g, h), want):
        view = got.view(times, few, k)
        for i in range(0, times, 1 << 20):
            part = view[i:i + (1 << 20)]
            assert torch.equal(part[:, 0], one[0].expand(part.shape[0], k)) and not part[:, 1:].any()
