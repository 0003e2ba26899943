"""Linear log loss over many classes and embedding rows, with their gradients, against the definition in 64 bits.

The bounds follow the arithmetic. With u = 2^-24 (half a step of float) and t the type's own half step:
  a score is a sum of f products that are exact in float (of float inputs: up to 2^-22, what the three planes leave out), so
  it is off by at most d = ((f + 8) u + 2^-22) sum_i |x_i w_i| + u |bias|;
  a probability is off by a factor within 2 d + e, where e = 1e-4 bounds the sums of at most some hundred exponentials in a row
  (200 u) and the exponential itself, which is that of x log2(e) rounded (|x| <= 200 here: 200 * 2^-23), and the loss by
  2 d + e + 8 u |lse|;
  an entry of G is rounded once (t; float: three planes, 2^-23), and a gradient adds up to m of them, m u of the sum of sizes, and
  is rounded to its type."""
import numpy as np
import pytest
import torch

from lbtree import _lib, ops

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
STEP = {"f32": 2.0 ** -24, "bf16": 2.0 ** -8, "f16": 2.0 ** -11}   # half a step, relative
ENTRY = {"f32": 2.0 ** -23, "bf16": 2.0 ** -8, "f16": 2.0 ** -11}  # one entry of G
LEAST = {"f32": 0.0, "bf16": 0.0, "f16": 2.0 ** -24}               # the smallest step of half precision


def inputs(n, f, k, dtype, seed=0, lean=4.0):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    w = torch.randn((k, f), generator=gen, device="cuda") * (1.5 / f ** 0.5)
    y = torch.randint(0, k, (n,), generator=gen, device="cuda")
    x = torch.randn((n, f), generator=gen, device="cuda") + lean * (torch.rand((n, 1), generator=gen, device="cuda") < 0.5) * w[y]
    return x.to(TYPES[dtype]), w.to(TYPES[dtype]), y


def reference(x, w, y, bias=None, weight=None):
    """(loss, gx, gw, gb) in 64 bits, and the bounds of what each may be off by as functions of the type."""
    k = w.shape[0]
    counts = (y >= 0) & (y < k)
    rows = counts.nonzero()[:, 0]
    X, W, lab = x[rows].double(), w.double(), y[rows].long()
    s = X @ W.t()
    size = X.abs() @ W.abs().t()
    if bias is not None:
        s = s + bias.double()
        size_b = size + torch.where(torch.isfinite(bias), bias.abs(), 0.0).double()
    else:
        size_b = size
    here = torch.arange(rows.numel(), device=x.device)
    lse = torch.logsumexp(s, dim=1)
    loss = torch.zeros(x.shape[0], dtype=torch.float64, device=x.device)
    loss[rows] = lse - s[here, lab]
    p = torch.exp(s - lse[:, None])
    g = p.clone()
    g[here, lab] -= 1.0
    wt = torch.ones(rows.numel(), dtype=torch.float64, device=x.device) if weight is None else weight.double()[rows]
    g = g * wt[:, None]
    gx = torch.zeros(x.shape, dtype=torch.float64, device=x.device)
    gx[rows] = g @ W
    gw, gb = g.t() @ X, g.sum(dim=0)
    f, n = x.shape[1], rows.numel()
    d = ((f + 8) * U + 2.0 ** -22) * size_b.max(dim=1).values if n else torch.zeros(0, device=x.device, dtype=torch.float64)
    rel = 2 * d + 1e-4  # of a probability

    def bounds(t):
        off = g.abs() * ENTRY[t] + (p * rel[:, None] + g.abs() * 4 * U) * wt.abs()[:, None]
        bl = torch.zeros_like(loss)
        bl[rows] = rel + 8 * U * (lse.abs() + 1.0)
        bx = torch.zeros_like(gx)
        bx[rows] = off @ W.abs() + (k + 64) * U * (g.abs() @ W.abs())
        bw = off.t() @ X.abs() + (n + 64) * U * (g.abs().t() @ X.abs())
        ob = (p * rel[:, None] + g.abs() * 4 * U) * wt.abs()[:, None]
        bb = ob.sum(dim=0) + (n + 64) * U * g.abs().sum(dim=0)
        bx = bx * (1 + STEP[t]) + gx.abs() * STEP[t] + LEAST[t]
        bw = bw * (1 + STEP[t]) + gw.abs() * STEP[t] + LEAST[t]
        return bl, bx, bw, bb + gb.abs() * U

    return (loss, gx, gw, gb), bounds


def assert_within(got, want, bound, what):
    got = got.double()
    assert got.shape == want.shape, what
    assert torch.isfinite(got).all(), what
    over = (got - want).abs() - bound
    assert float(over.max() if over.numel() else 0.0) <= 0, (what, float(over.max()), float((got - want).abs().max()))


def check(x, w, y, dtype, bias=None, weight=None):
    want, bounds = reference(x, w, y, bias, weight)
    limits = bounds(dtype)
    got = ops.linear_log_loss(x, w, y, bias=bias)
    assert got.dtype == torch.float32
    assert_within(got, want[0], limits[0], "loss alone")
    out = ops.linear_log_loss_gradient(x, w, y, sample_weight=weight, bias=bias)
    assert len(out) == (3 if bias is None else 4)
    assert out[1].dtype == x.dtype and out[2].dtype == w.dtype
    for i, name in enumerate(("loss", "grad_X", "grad_weight", "grad_bias")[:len(out)]):
        assert_within(out[i], want[i], limits[i], name)
    return out


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("n,f,k", [(1, 1, 1), (1, 64, 1000), (2, 3, 2), (5, 7, 9), (16, 129, 255), (17, 8, 257), (64, 256, 1000),
                                   (130, 72, 300), (257, 200, 1031), (33, 1000, 517), (511, 65, 64), (48, 90, 70001), (63, 2049, 3000), (250, 136, 9000)])
def test_loss_and_gradients(n, f, k, dtype):
    check(*inputs(n, f, k, dtype, seed=n + f + k), dtype)


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
def test_tiles_of_256(dtype):
    """Sizes at which every product takes the large tiles, none of them a multiple of one."""
    check(*inputs(3900, {"bf16": 4104, "f16": 4099, "f32": 4100}[dtype], 5100, dtype, seed=3), dtype)


@pytest.mark.parametrize("dtype,n,f,k,biased", [("f16", 4100, 40, 170000, True), ("f16", 4100, 24, 165000, False),
                                                ("f32", 4100, 24, 100000, False), ("bf16", 40, 2050, 131001, True),
                                                ("bf16", 300, 1030, 261000, False)])
def test_several_pieces_of_the_classes(dtype, n, f, k, biased):
    """G of a piece takes 4 GiB, with float exponentials beside it but for bfloat16; weights that are laid out first 512 MiB."""
    entry = {"bf16": 2, "f16": 6, "f32": 10}[dtype]
    assert entry * ((n + 255) // 256 * 256) * k > 4 << 30 or 2 * ((f + 63) // 64 * 64) * k > 512 << 20
    bias = torch.randn(k, generator=torch.Generator(device="cuda").manual_seed(1), device="cuda") if biased else None
    check(*inputs(n, f, k, dtype, seed=5), dtype, bias=bias)


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("n,f,k", [(1, 1024, 5000), (16, 40, 33), (17, 1000, 700), (32, 2053, 70001), (33, 7, 90000), (64, 130, 66000),
                                   (65, 130, 66000), (3, 4096, 10), (200, 520, 3000), (256, 70, 70000), (257, 33, 3000)])
def test_loss_of_few_rows(n, f, k, dtype):
    x, w, y = inputs(n, f, k, dtype, seed=n * f)
    rs = np.random.RandomState(k)
    for bias in (None, torch.from_numpy(np.where(rs.rand(k) < 0.1, -np.inf, rs.normal(0, 2, k))).float().cuda()):
        if bias is not None:
            bias[y] = 0.25
        want, bounds = reference(x, w, y, bias)
        assert_within(ops.linear_log_loss(x, w, y, bias=bias), want[0], bounds(dtype)[0], "loss")


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("n", [300, 40])
def test_rows_that_do_not_count(n, dtype):
    f, k = 72, 700
    x, w, y = inputs(n, f, k, dtype, seed=11)
    y[::3] = -1
    y[1], y[4], y[7], y[10] = k, 2 ** 31, -2 ** 40, 2 ** 62
    out = (y < 0) | (y >= k)
    x[out] = float("nan")
    x[torch.nonzero(out)[5]] = float("inf")
    loss, gx, gw = check(x, w, y, dtype)
    assert (loss[out] == 0).all() and (gx[out] == 0).all()
    # not one counts
    y[:] = -100
    loss, gx, gw = ops.linear_log_loss_gradient(x, w, y)
    assert not loss.any() and not gx.any() and not gw.any()
    assert not ops.linear_log_loss(x, w, y).any()
    # no row at all
    loss, gx, gw, gb = ops.linear_log_loss_gradient(x[:0], w, y[:0], bias=torch.ones(k, device="cuda"))
    assert loss.shape == (0,) and gx.shape == (0, f) and not gw.any() and not gb.any() and gw.shape == w.shape
    assert ops.linear_log_loss(x[:0], w, y[:0]).shape == (0,)


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("n,k", [(100, 500), (9, 3000), (3900, 5100)])
def test_weights_and_bias(n, k, dtype):
    x, w, y = inputs(n, 64, k, dtype, seed=13)
    rs = np.random.RandomState(n)
    weight = torch.from_numpy(rs.choice([0.0, 1e-3, 0.5, 1.0, -2.0, 3.0, 100.0], n)).float().cuda()
    bias = torch.from_numpy(rs.normal(0, 3, k)).float().cuda()
    bias[rs.randint(0, k, k // 5)] = -float("inf")  # masked classes
    bias[y] = torch.where(torch.isfinite(bias[y]), bias[y], 0.0)
    check(x, w, y, dtype, bias=bias, weight=weight)
    # weights of float64 and of another shape are taken as they are everywhere in this package
    a = ops.linear_log_loss_gradient(x, w, y.to(torch.int32), sample_weight=weight.double()[:, None], bias=bias[:, None])
    b = ops.linear_log_loss_gradient(x, w, y, sample_weight=weight, bias=bias)
    assert all(torch.equal(p, q) for p, q in zip(a, b))


def test_half_precision_keeps_small_probabilities_and_weights():
    """Weights far apart in size: the rows of small ones keep their bits (their exponent stands apart)."""
    n, f, k = 64, 64, 2000
    x, w, y = inputs(n, f, k, "f16", seed=17)
    weight = 2.0 ** torch.arange(-12, 4, device="cuda").float().repeat(4) * 1.3
    check(x, w, y, "f16", weight=weight)


def test_masked_labels_and_no_class():
    x, w, y = inputs(20, 32, 50, "f32", seed=19)
    bias = torch.zeros(50, device="cuda")
    bias[y[0]] = -float("inf")
    loss, gx, gw, gb = ops.linear_log_loss_gradient(x, w, y, bias=bias)
    hit = y == y[0]
    assert torch.isinf(loss[hit]).all() and torch.isfinite(loss[~hit]).all()
    assert torch.isfinite(gx).all() and torch.isfinite(gw).all() and torch.isfinite(gb).all()
    # no class is left: p is 0 and the gradient that of the labels alone
    bias[:] = -float("inf")
    loss, gx, gw, gb = ops.linear_log_loss_gradient(x, w, y, bias=bias)
    assert torch.isinf(loss).all() and (loss > 0).all()
    assert torch.allclose(gx, -w[y], rtol=1e-6, atol=0)
    assert torch.equal(gb, -torch.bincount(y, minlength=50).float())
    # the lowest number as a mask is one more score
    bias[:] = torch.finfo(torch.float32).min
    assert torch.isfinite(ops.linear_log_loss(x[:1], w, y[:1], bias=bias)).all()


def test_nan_and_infinity_in_rows_that_count_stay_in_their_rows():
    x, w, y = inputs(40, 32, 300, "bf16", seed=23)
    x[7, 3] = float("nan")
    loss, gx, gw = ops.linear_log_loss_gradient(x, w, y)
    rest = torch.arange(40, device="cuda") != 7
    assert torch.isnan(loss[7]) and torch.isnan(gx[7]).all()
    clean = ops.linear_log_loss_gradient(x[rest].contiguous(), w, y[rest])
    assert torch.equal(loss[rest], clean[0]) and torch.equal(gx[rest], clean[1])


@pytest.mark.parametrize("n,f,k", [(70, 1, 200), (300, 31, 129), (300, 33, 64), (100, 4001, 500), (1100, 95, 1000), (1030, 64, 3000),
                                   (2000, 129, 20000), (600, 36, 24001), (20, 1003, 9001), (130, 2050, 3001), (700, 65, 130000),
                                   (257, 4001, 1003)])
def test_float_tiles(n, f, k):
    """Sizes beyond few rows: rows of the weights that end inside a stage and inside 16 bytes, tiles that lie past the last class."""
    x, w, y = inputs(n, f, k, "f32", seed=n + k)
    rs = np.random.RandomState(f)
    y[torch.from_numpy(rs.rand(n) < 0.2).cuda()] = -100
    bias = torch.from_numpy(rs.normal(0, 1, k)).float().cuda()
    check(x, w, y, "f32")
    check(x, w, y, "f32", bias=bias, weight=torch.from_numpy(rs.rand(n) + 0.1).float().cuda())
    # the weights as a part of a larger array: what lies behind them is not looked at
    wide = torch.full((k * f + 64,), float("nan"), device="cuda")
    wide[:k * f] = w.reshape(-1)
    assert torch.equal(ops.linear_log_loss(x, wide[:k * f].view(k, f), y, bias=bias), ops.linear_log_loss(x, w, y, bias=bias))


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("n,f,k", [(1024, 520, 300), (1025, 520, 300), (1024, 7, 4000), (600, 1033, 77)])
def test_rows_counted_and_laid_out_together_or_apart(n, f, k, dtype):
    x, w, y = inputs(n, f, k, dtype, seed=n + f)
    rs = np.random.RandomState(n)
    out = torch.from_numpy(rs.rand(n) < 0.4).cuda()
    y[out] = k
    x[out] = float("nan")
    got = check(x, w, y, dtype)
    assert not got[0][out].any() and not got[1][out].any()
    check(x, w, y, dtype, weight=torch.from_numpy(rs.rand(n) + 0.1).float().cuda())
    assert torch.equal(ops.linear_log_loss(x, w, torch.full_like(y, -1)), torch.zeros(n, device="cuda"))


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_large_scores(dtype):
    """Scores of some hundreds: tops are taken off before the exponentials."""
    x, w, y = inputs(50, 16, 400, dtype, seed=29)
    loss = ops.linear_log_loss((x * 64), w, y).double()
    s = (x * 64).double() @ w.double().t()
    want = torch.logsumexp(s, 1) - s[torch.arange(50, device="cuda"), y]
    size = ((x * 64).double().abs() @ w.double().abs().t()).max(1).values
    assert ((loss - want).abs() <= 2 * (24 * U + 2.0 ** -22) * size + 1e-4 + 8 * U * s.abs().max()).all()


def test_gradient_against_differences():
    """The loss itself, in float, at points a step apart: along the gradient, half turned away from it."""
    x, w, y = inputs(12, 24, 60, "f32", seed=31)
    bias = torch.randn(60, device="cuda")
    weight = torch.rand(12, device="cuda") + 0.5
    _, gx, gw, gb = ops.linear_log_loss_gradient(x, w, y, sample_weight=weight, bias=bias)
    gen = torch.Generator(device="cuda").manual_seed(1)
    h = 2.0 ** -7
    for a, g in ((0, gx), (1, gw), (2, gb)):
        at = [x, w, bias]
        turn = torch.randn(g.shape, generator=gen, device="cuda")
        step = g / g.norm() + turn / turn.norm()
        step /= step.norm()
        value = []
        for sign in (1.0, -1.0):
            moved = list(at)
            moved[a] = at[a] + sign * h * step
            loss = ops.linear_log_loss(moved[0], moved[1], y, bias=moved[2])
            value.append(float((loss.double() * weight.double()).sum()))
        slope = (value[0] - value[1]) / (2 * h)
        # The third derivative of log-sum-exp along a step that changes scores by c at most is below 2 c^3, and a difference
        # over 2 h leaves out a sixth of it times h^2. A loss is off by 2 d + e <= 2 * (32 u * 60) + 1e-4 (f = 24, sum |x w| < 60).
        change = 1.0 if a == 2 else float((w if a == 0 else x).double().norm(dim=1).max())
        limit = float(weight.sum()) * (h * h / 3 * change ** 3 + (2 * 32 * U * 60 + 1e-4) / h)
        assert abs(slope - float((g.double() * step.double()).sum())) <= limit


def test_calls_repeat_bit_for_bit_and_leave_their_inputs():
    x, w, y = inputs(700, 136, 3000, "bf16", seed=37)
    keep = [t.clone() for t in (x, w, y)]
    a = ops.linear_log_loss_gradient(x, w, y, bias=torch.zeros(3000, device="cuda"))
    ops.linear_log_loss_gradient(x.float(), w.float(), y)  # leaves other values in the scratch
    b = ops.linear_log_loss_gradient(x, w, y, bias=torch.zeros(3000, device="cuda"))
    assert all(torch.equal(p, q) for p, q in zip(a, b))
    assert all(torch.equal(p, q) for p, q in zip(keep, (x, w, y)))
    # The call without gradients may join the shares of a row in another order: of 3000 classes at most 94, of 32 each. Each order is
    # off by at most 94 u of the total and the exponentials by 2^-22, so the two differ by 2 (94 u + 2^-22) before the logarithm,
    # whose value and the sum with the top are rounded to u of sizes below 32.
    assert (ops.linear_log_loss(x, w, y) - a[0]).abs().max() <= 2 * (94 * U + 2.0 ** -22) + 4 * 32 * U


def test_strided_and_unaligned_inputs():
    x, w, y = inputs(60, 64, 200, "bf16", seed=41)
    want = ops.linear_log_loss_gradient(x, w, y)
    wide = torch.empty((60, 100), dtype=x.dtype, device="cuda")
    wide[:, 3:67] = x
    flat = torch.empty(200 * 64 + 1, dtype=w.dtype, device="cuda")
    flat[1:] = w.reshape(-1)
    got = ops.linear_log_loss_gradient(wide[:, 3:67], flat[1:].view(200, 64), torch.stack([y, y], 1)[:, 0])
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    got = ops.linear_log_loss_gradient(x.t().contiguous().t(), w.t().contiguous().t(), y)
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_another_stream_and_captured_graphs():
    x, w, y = inputs(200, 64, 900, "bf16", seed=43)
    want = ops.linear_log_loss_gradient(x, w, y)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = ops.linear_log_loss_gradient(x, w, y)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    tokens = torch.randint(0, 900, (3000,), device="cuda")
    g = torch.randn((3000, 64), device="cuda").to(torch.bfloat16)
    graphs = []
    for _ in range(2):  # two graphs: each has its scratch
        with torch.cuda.stream(side):
            ops.linear_log_loss_gradient(x, w, y)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = ops.linear_log_loss_gradient(x, w, y)
            table = ops.embed_rows_gradient(g, tokens, 900)
            rows = ops.embed_rows(w, tokens, 2.0)
        graphs.append((graph, out, table, rows))
    for turn in range(3):
        x.copy_(inputs(200, 64, 900, "bf16", seed=50 + turn)[0])
        tokens.copy_(torch.randint(0, 900, (3000,), device="cuda"))
        torch.cuda.synchronize()
        streams = [torch.cuda.Stream(), torch.cuda.Stream()]
        for (graph, *_), s in zip(graphs, streams):
            with torch.cuda.stream(s):
                graph.replay()
        torch.cuda.synchronize()
        want = ops.linear_log_loss_gradient(x, w, y)
        table, rows = ops.embed_rows_gradient(g, tokens, 900), ops.embed_rows(w, tokens, 2.0)
        for _, out, t, r in graphs:
            assert all(torch.equal(a, b) for a, b in zip(out, want))
            assert torch.equal(t, table) and torch.equal(r, rows)


def test_refusals():
    x, w, y = inputs(10, 16, 30, "bf16")
    for bad in (lambda: ops.linear_log_loss(x, w.float(), y), lambda: ops.linear_log_loss(x.double(), w.double(), y),
                lambda: ops.linear_log_loss(x, w[:, :8], y), lambda: ops.linear_log_loss(x[0], w, y),
                lambda: ops.linear_log_loss(x, w, y[:5]), lambda: ops.linear_log_loss(x, w, y.float()),
                lambda: ops.linear_log_loss(x, w, y, bias=torch.zeros(29, device="cuda")),
                lambda: ops.linear_log_loss(x, w[:0], y), lambda: ops.linear_log_loss(x[:, :0], w[:, :0], y),
                lambda: ops.linear_log_loss_gradient(x, w, y, sample_weight=torch.ones(9)),
                lambda: ops.embed_rows(w, y.float()), lambda: ops.embed_rows(w.double(), y), lambda: ops.embed_rows(w[0], y),
                lambda: ops.embed_rows_gradient(x, y[:5], 30), lambda: ops.embed_rows_gradient(x, y, 0),
                lambda: ops.embed_rows_gradient(x, y, -3), lambda: ops.embed_rows_gradient(x, y, 30, add_to=w.float()),
                lambda: ops.embed_rows_gradient(x, y, 30, add_to=w.t().contiguous().t()),
                lambda: ops.embed_rows_gradient(x, y, 31, add_to=w)):
        with pytest.raises(_lib.LbtError):
            bad()


# ---- rows of a table ---------------------------------------------------------------------------------


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("f", [1, 2, 3, 8, 130, 256, 1000])
def test_embed_rows(f, dtype):
    gen = torch.Generator(device="cuda").manual_seed(f)
    table = torch.randn((77, f), generator=gen, device="cuda").to(TYPES[dtype])
    table[5, 0], table[6, 0] = float("nan"), float("inf")
    for shape in ((), (0,), (1,), (3, 5), (1000,)):
        tokens = torch.randint(-3, 82, shape, generator=gen, device="cuda")
        for scale in (1.0, 11.3):
            got = ops.embed_rows(table, tokens, scale)
            inside = (tokens >= 0) & (tokens < 77)
            want = table[torch.where(inside, tokens, 0)].float() * torch.tensor(scale, dtype=torch.float32, device="cuda")
            want = torch.where(inside[..., None], want, 0.0).to(table.dtype)
            assert got.shape == tuple(shape) + (f,)
            assert torch.equal(torch.nan_to_num(got.float()), torch.nan_to_num(want.float()))
            assert torch.equal(got.isnan(), want.isnan())
            assert torch.equal(ops.embed_rows(table, tokens.to(torch.int32), scale).nan_to_num(), got.nan_to_num())


def embed_reference(grad, tokens, rows, scale, dtype, old=None):
    f = grad.shape[-1]
    t, g = tokens.reshape(-1).cpu(), grad.reshape(-1, f).double().cpu()
    inside = (t >= 0) & (t < rows)
    scale = float(np.float32(scale))
    out = torch.zeros((rows, f), dtype=torch.float64).index_add_(0, t[inside], g[inside]) * scale
    size = torch.zeros((rows, f), dtype=torch.float64).index_add_(0, t[inside], g[inside].abs()) * abs(scale)
    times = torch.bincount(t[inside], minlength=rows).double()[:, None]
    bound = (times + 3) * U * size
    if old is not None:
        out, bound = out + old.double().cpu(), bound + U * (out.abs() + old.double().cpu().abs())
    return out, bound * (1 + STEP[dtype]) + out.abs() * STEP[dtype] + LEAST[dtype], times[:, 0] > 0


def skewed(t, rows, kind, gen):
    if kind == "one":
        return torch.full((t,), rows // 2, device="cuda")
    if kind == "each":
        return torch.arange(t, device="cuda") % rows
    u = torch.rand(t, generator=gen, device="cuda", dtype=torch.float64)
    if kind == "skewed":
        return ((rows + 1.0) ** u - 1).long().clamp(0, rows - 1)
    tokens = (u * (rows + 4)).long() - 2  # some outside
    return tokens


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("t,f,rows,kind", [
    (1, 1, 1, "one"), (1, 8, 70000, "uniform"), (7, 3, 5, "uniform"), (63, 64, 10, "skewed"), (64, 2, 64, "each"),
    (65, 130, 3, "one"), (129, 1000, 40, "skewed"), (1000, 200, 5003, "skewed"), (1000, 33, 17, "uniform"),
    (8192, 24, 1000, "skewed"), (8193, 24, 1000, "skewed"), (8200, 5, 1, "one"), (20000, 72, 65535, "uniform"),
    (20001, 10, 65536, "skewed"), (33000, 512, 900, "one"), (50000, 1, 1500000, "uniform"), (9001, 4, 1023, "each"),
])
def test_embed_rows_gradient(t, f, rows, kind, dtype):
    gen = torch.Generator(device="cuda").manual_seed(t + f)
    tokens = skewed(t, rows, kind, gen)
    grad = torch.randn((t, f), generator=gen, device="cuda").to(TYPES[dtype])
    got = ops.embed_rows_gradient(grad, tokens, rows, scale=1.7)
    want, bound, named = embed_reference(grad, tokens, rows, 1.7, dtype)
    assert got.dtype == grad.dtype and got.shape == (rows, f)
    assert_within(got.cpu(), want, bound, "grad_table")
    assert not got.cpu()[~named].any()
    assert torch.equal(ops.embed_rows_gradient(grad, tokens.to(torch.int32), rows, scale=1.7), got)  # the same bits again
    # added to what is there; rows without a token keep their bits, NaN too
    old = torch.randn((rows, f), generator=gen, device="cuda").to(TYPES[dtype])
    want, bound, named = embed_reference(grad, tokens, rows, 1.7, dtype, old)
    old[~named.cuda()] = float("nan")
    to = old.clone()
    assert ops.embed_rows_gradient(grad, tokens, rows, scale=1.7, add_to=to) is to
    assert_within(to.cpu()[named], want[named], bound[named], "added")
    assert to.cpu()[~named].isnan().all()


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("lengths,f", [
    ((33, 32, 1, 0, 64, 700, 31, 1100), 130),  # at once: rows that one wave, and rows that four waves add up
    ((2048,), 40),
    ((3, 505, 512, 0, 520, 529, 1, 1040, 513), 24),  # 63, 64 and more chunks of 8
    ((5, 4096 * 8, 1, 20000, 4000, 3), 7),  # over 4096 of them
    ((1, 40000, 0, 25000, 7), 1030),
])
def test_embed_rows_gradient_of_rows_that_many_places_name(lengths, f, dtype):
    gen = torch.Generator(device="cuda").manual_seed(len(lengths) + f)
    tokens = torch.repeat_interleave(torch.arange(len(lengths)), torch.tensor(lengths)).cuda()
    tokens = tokens[torch.randperm(tokens.numel(), generator=gen, device="cuda")]
    grad = torch.randn((tokens.numel(), f), generator=gen, device="cuda").to(TYPES[dtype])
    got = ops.embed_rows_gradient(grad, tokens, len(lengths), scale=0.3)
    want, bound, named = embed_reference(grad, tokens, len(lengths), 0.3, dtype)
    assert_within(got.cpu(), want, bound, "grad_table")
    assert not got.cpu()[~named].any()
    assert torch.equal(ops.embed_rows_gradient(grad, tokens, len(lengths), scale=0.3), got)
    # one place more, that names no row and has no number: nothing changes but the order of the sums
    grad = torch.cat([torch.full((1, f), float("nan"), dtype=grad.dtype, device="cuda"), grad])
    tokens = torch.cat([torch.tensor([-100], device="cuda"), tokens])
    assert_within(ops.embed_rows_gradient(grad, tokens, len(lengths), scale=0.3).cpu(), want, bound, "grad_table")


def test_embed_gradient_shapes_and_places_that_name_no_row():
    grad = torch.randn((4, 6, 16), device="cuda")
    tokens = torch.randint(0, 9, (4, 6), device="cuda")
    flat = ops.embed_rows_gradient(grad.reshape(24, 16), tokens.reshape(24), 9)
    assert torch.equal(ops.embed_rows_gradient(grad, tokens, 9), flat)
    assert torch.equal(ops.embed_rows_gradient(grad.transpose(0, 1), tokens.t(), 9),
                       ops.embed_rows_gradient(grad.transpose(0, 1).contiguous(), tokens.t().contiguous(), 9))
    tokens[1] = -1
    tokens[2, 3] = 2 ** 40
    grad[1] = float("nan")
    grad[2, 3] = float("inf")
    assert torch.isfinite(ops.embed_rows_gradient(grad, tokens, 9)).all()
    assert not ops.embed_rows_gradient(grad, torch.full_like(tokens, -7), 9).any()
    assert not ops.embed_rows_gradient(grad[:0], tokens[:0], 9).any()
    to = torch.randn((9, 16), device="cuda")
    keep = to.clone()
    assert torch.equal(ops.embed_rows_gradient(grad[:0], tokens[:0], 9, add_to=to), keep)


def test_embed_gradient_against_differences():
    """The lookup is linear: its change along any table is the product with the gradient, but for rounding."""
    gen = torch.Generator(device="cuda").manual_seed(3)
    tokens = torch.randint(-1, 40, (500,), generator=gen, device="cuda")
    grad = torch.randn((500, 24), generator=gen, device="cuda")
    g = ops.embed_rows_gradient(grad, tokens, 40, scale=3.0).double()
    table, step = (torch.randn((40, 24), generator=gen, device="cuda") for _ in range(2))
    value = [float((ops.embed_rows(table + s * step, tokens, 3.0).double() * grad.double()).sum()) for s in (0.5, -0.5)]
    # 12000 products, each of a value below 3 * 6 rounded three times, times a gradient below 5
    assert abs(value[0] - value[1] - float((g * step.double()).sum())) <= 12000 * 18 * 5 * 4 * U


@pytest.mark.parametrize("n", [20, 200])
def test_losses_from_native_code_and_from_python_are_the_same(monkeypatch, n):
    x, w, y = inputs(n, 40, 600, "bf16", seed=47)
    w.requires_grad_()
    bias, weight = torch.randn(600, device="cuda"), torch.rand(n, device="cuda")

    def calls():
        return ((ops.linear_log_loss(x, w, y), ops.linear_log_loss(x, w, y, bias)) + ops.linear_log_loss_gradient(x, w, y)
                + ops.linear_log_loss_gradient(x, w, y, weight, bias) + ops.linear_log_loss_gradient(x, w, y, bias=bias))

    got = calls()
    assert not any(t.requires_grad for t in got)
    monkeypatch.setattr(ops, "_NATIVE", None)
    want = calls()
    assert len(got) == len(want) and all(torch.equal(a, b) and a.dtype == b.dtype and a.shape == b.shape for a, b in zip(got, want))


def test_lookups_from_native_code_and_from_python_are_the_same(monkeypatch):
    gen = torch.Generator(device="cuda").manual_seed(4)
    table = torch.randn((50, 24), generator=gen, device="cuda").to(torch.bfloat16).requires_grad_()
    tokens = torch.randint(-2, 52, (7, 300), generator=gen, device="cuda")
    grad = torch.randn((7, 300, 24), generator=gen, device="cuda").to(torch.bfloat16)
    assert ops._NATIVE is not None
    got = ops.embed_rows(table, tokens, 3.0), ops.embed_rows_gradient(grad, tokens, 50, 3.0)
    assert not got[0].requires_grad
    monkeypatch.setattr(ops, "_NATIVE", None)
    want = ops.embed_rows(table, tokens, 3.0), ops.embed_rows_gradient(grad, tokens, 50, 3.0)
    assert all(torch.equal(a, b) and a.shape == b.shape and a.dtype == b.dtype for a, b in zip(got, want))


def test_an_exception_of_the_library_is_left_to_python():
    import ctypes as C

    thrower = C.cast(C.CDLL("libstdc++.so.6")._ZSt17__throw_bad_allocv, C.c_void_p).value
    table, tokens = torch.zeros((4, 8), device="cuda"), torch.zeros(3, dtype=torch.int64, device="cuda")
    device = torch.cuda.current_device()
    for _ in range(3):
        assert _lib._host.embed_rows(table, tokens, thrower, 0, device, 1.0) is None
        assert _lib._host.embed_rows_gradient(table[:3], tokens, ops._scratch, thrower, ops._EMBED_BYTES, 0, device, 4, 1.0) is None
        for call, more in ((_lib._host.linear_log_loss, ()), (_lib._host.linear_log_loss_gradient, (None,))):
            assert call(table[:3], table, tokens, None, ops._scratch, thrower, ops._LOG_LOSS_BYTES, 0, device, *more) is None
    assert C.pythonapi.PyGILState_Check() == 1


def test_threads_on_streams_of_their_own():
    """Four threads at once, each with its stream and so with its scratch."""
    import threading

    cases = [inputs(150 + 40 * i, 64 + 8 * i, 700 + 300 * i, "bf16", seed=60 + i) for i in range(4)]
    tokens = [torch.randint(0, 500, (9000 + i,), device="cuda") for i in range(4)]
    grads = [torch.randn((9000 + i, 16), device="cuda") for i in range(4)]
    want = [ops.linear_log_loss_gradient(*c) + (ops.embed_rows_gradient(g, t, 500),) for c, t, g in zip(cases, tokens, grads)]
    torch.cuda.synchronize()
    got = [None] * 4

    def work(i):
        stream = torch.cuda.Stream()
        with torch.cuda.stream(stream):
            for _ in range(5):
                got[i] = ops.linear_log_loss_gradient(*cases[i]) + (ops.embed_rows_gradient(grads[i], tokens[i], 500),)
        stream.synchronize()

    threads = [threading.Thread(target=work, args=(i,)) for i in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    for a, b in zip(got, want):
        assert all(torch.equal(p, q) for p, q in zip(a, b))


@pytest.mark.parametrize("n,f,k", [(20, 1003, 9001), (300, 70, 900), (1500, 64, 2000)])
def test_float_captured_and_replayed(n, f, k):
    x, w, y = inputs(n, f, k, "f32", seed=n)
    bias = torch.randn(k, device="cuda")
    ops.linear_log_loss_gradient(x, w, y, bias=bias)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = ops.linear_log_loss_gradient(x, w, y, bias=bias) + (ops.linear_log_loss(x, w, y, bias=bias),)
    for turn in range(4):
        y.copy_((y + 7 * turn) % (k + 3))  # some that are no class
        w.mul_(0.9)
        graph.replay()
        want = ops.linear_log_loss_gradient(x, w, y, bias=bias) + (ops.linear_log_loss(x, w, y, bias=bias),)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_offsets_beyond_32_bits():
    """Weights and a table of 4.9 GB whose last rows differ from 0: 600000 rows of 4096 bfloat16."""
    rows, f = 600000, 4096
    w = torch.zeros((rows, f), dtype=torch.bfloat16, device="cuda")
    gen = torch.Generator(device="cuda").manual_seed(3)
    w[-300:] = torch.randn((300, f), generator=gen, device="cuda").to(w.dtype) * 0.02
    tokens = torch.tensor([rows - 1, 0, rows - 300, rows - 7, rows], device="cuda")
    got = ops.embed_rows(w, tokens, 0.5)
    assert torch.equal(got[:4], (w[tokens[:4]].float() * 0.5).to(w.dtype)) and not got[4].any()
    for n in (1, 70):
        x = torch.randn((n, f), generator=gen, device="cuda").to(w.dtype)
        y = torch.randint(rows - 300, rows, (n,), generator=gen, device="cuda")
        y[0] = 5
        s = x.double() @ w[-300:].double().t()
        label = torch.where(y >= rows - 300, s[torch.arange(n, device="cuda"), (y - (rows - 300)).clamp(min=0)], 0.0)
        want = torch.log(torch.exp(s).sum(1) + (rows - 300)) - label
        size = (x.double().abs() @ w[-300:].double().abs().t()).max(1).values
        loss = ops.linear_log_loss(x, w, y)
        # as in `reference`: 2 d + e, and the logarithm
        assert ((loss - want).abs() <= 2 * ((f + 8) * U + 2.0 ** -22) * size + 1e-4 + 8 * U * 20).all()
    g = torch.ones((3, f), dtype=torch.bfloat16, device="cuda")
    to = ops.embed_rows_gradient(g, torch.tensor([rows - 1, 3, rows - 1], device="cuda"), rows)
    assert torch.equal(to[-1], torch.full((f,), 2.0, dtype=to.dtype, device="cuda")) and (to[3] == 1).all()
    assert not to[-100:-1].any() and not to[:3].any() and not to[4:100].any() and not to[299990:300010].any()


# ---- together ------------------------------------------------------------------------------------------


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_leaves_as_tokens_through_one_table_and_back(dtype):
    """A tree's leaves are looked up in a table, the rows are scored against the same table, and both gradients meet in it."""
    rs = np.random.RandomState(0)
    X = rs.random_sample((2000, 8)).astype(np.float32)
    g = (rs.random_sample((2000, 1)) - X[:, :1]).astype(np.float64)
    tree = ops.build_tree(X, g, np.ones_like(g), max_depth=5, split_samples=32, seed=1, row_leaf=True)
    tokens = tree.row_leaf
    rows = tree.leaf_value.shape[0]
    table = (torch.randn((rows, 48), generator=torch.Generator(device="cuda").manual_seed(2), device="cuda") * 0.3).to(TYPES[dtype])
    y = torch.roll(tokens.long(), 1)
    y[:100] = -1
    weight = torch.full((2000,), 1.0 / 1900, device="cuda")
    hidden = ops.embed_rows(table, tokens, 2.0)
    loss, grad_hidden, grad_table = ops.linear_log_loss_gradient(hidden, table, y, sample_weight=weight)
    want, bounds = reference(hidden, table, y, weight=weight)
    limits = bounds(dtype)
    for got, w, b in zip((loss, grad_hidden, grad_table), want, limits):
        assert_within(got, w, b, "head")
    head = grad_table.clone()
    total = ops.embed_rows_gradient(grad_hidden, tokens, rows, scale=2.0, add_to=grad_table)
    want, bound, _ = embed_reference(grad_hidden, tokens.long(), rows, 2.0, dtype, head)
    assert_within(total.cpu(), want, bound, "both")
    # the tied table's gradient in 64 bits, end to end: what the types round on the way (hidden and grad_hidden are outputs
    # of their own) moves it by a few steps of the type
    t = table.double().requires_grad_()
    h = 2.0 * t[tokens.long()]
    s = h @ t.t()
    keep = (y >= 0).nonzero()[:, 0]
    nll = torch.logsumexp(s[keep], 1) - s[keep, y[keep]]
    (nll * weight.double()[keep]).sum().backward()
    off = (total.double() - t.grad).norm() / t.grad.norm()
    assert off <= (8 * STEP[dtype] if dtype == "bf16" else 1e-5)
