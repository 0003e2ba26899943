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


def test_predictions():
    n, few = (1 << 30) + 1003, 59  # four threads a row, or more
    values = torch.linspace(-1, 1, few, device="cuda").view(few, 1)
    gen = torch.Generator(device="cuda").manual_seed(1)
    g = torch.randn((few, 1), generator=gen, device="cuda", dtype=torch.float64)
    trees = [ops.build_tree(values, g * (i + 1), torch.ones_like(g), max_depth=3, split_samples=16, seed=i) for i in range(9)]
    trees = [(t.leaf_value, t.feature, t.split_value) for t in trees]
    X = values.repeat((-(-n // few), 1))[:n].contiguous()
    packed = ops.PackedEnsemble(trees, 1, 1)
    want = packed.predict(values)
    assert want.unique().numel() > 5
    init = torch.full((1,), 0.75, dtype=torch.float64, device="cuda")
    for got, one in ((packed.predict(X), want), (ops.predict(X, trees, 1), want), (ops.predict(X, trees, 1, init=init), ops.predict(values, trees, 1, init=init))):
        assert got.shape == (n, 1)
        whole = n // few * few
        view = got[:whole].view(-1, few)
        for i in range(0, view.shape[0], 1 << 21):
            assert torch.equal(view[i:i + (1 << 21)], one.view(1, few).expand(min(1 << 21, view.shape[0] - i), few))
        assert torch.equal(got[whole:], one[:n - whole])


def test_predictions_of_no_tree():
    k = 8
    n = (1 << 32) // k + 1007
    X = torch.zeros((n, 1), device="cuda")
    fill = torch.full((n * k,), 3.0, dtype=torch.float64, device="cuda")  # what the output's memory held
    del fill
    init = torch.arange(k, dtype=torch.float64, device="cuda")
    got = ops.predict(X, [], k, init=init)
    for i in range(0, n, 1 << 25):
        assert torch.equal(got[i:i + (1 << 25)], init.expand(min(1 << 25, n - i), k))
