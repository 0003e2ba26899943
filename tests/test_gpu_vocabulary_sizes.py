"""The operators for vocabularies at sizes where a call is cut up: rows in parts, long sorts.

The bounds are those of test_gpu_vocabulary.py. Where a sum goes over hundreds of thousands of rows its worst case is a few hundredths of
the sum of sizes; the values here have one sign for half of the classes, so that a part left out, or added twice, is far more than that."""
import pytest
import torch

from lbtree import _lib, ops
from test_gpu_vocabulary import ENTRY, LEAST, STEP, TYPES, U, assert_within

pytestmark = pytest.mark.gpu


def reference_by_rows(x, w, y, bias, weight, t, step):
    """test_gpu_vocabulary.reference for many rows, `step` at a time: outputs in 64 bits and what they may be off by."""
    n, f = x.shape
    k = w.shape[0]
    W = w.double()
    kinds = dict(dtype=torch.float64, device=x.device)
    loss, gx, gw, gb = torch.zeros(n, **kinds), torch.zeros(n, f, **kinds), torch.zeros(k, f, **kinds), torch.zeros(k, **kinds)
    bl, bx, bw, bb = (torch.zeros_like(a) for a in (loss, gx, gw, gb))
    sw, sb = torch.zeros_like(gw), torch.zeros_like(gb)  # sums of sizes
    counted = 0
    for i in range(0, n, step):
        rows = ((y[i:i + step] >= 0) & (y[i:i + step] < k)).nonzero()[:, 0] + i
        X, lab, here = x[rows].double(), y[rows], torch.arange(rows.numel(), device=x.device)
        s, size = X @ W.t(), X.abs() @ W.abs().t()
        if bias is not None:
            s, size = s + bias.double(), size + bias.double().abs()
        d = ((f + 8) * U + 2.0 ** -22) * (size.max(dim=1).values if rows.numel() else size.sum(dim=1))
        rel = 2 * d + 1e-4
        lse = torch.logsumexp(s, dim=1)
        loss[rows], bl[rows] = lse - s[here, lab], rel + 8 * U * (lse.abs() + 1.0)
        p = torch.exp(s - lse[:, None])
        g = p.clone()
        g[here, lab] -= 1.0
        wt = torch.ones(rows.numel(), **kinds) if weight is None else weight.double()[rows]
        g = g * wt[:, None]
        off = g.abs() * 4 * U + p * rel[:, None] * wt.abs()[:, None]
        # an entry of G is rounded once; where bfloat16 has no bias the exponential is held in 11 bits before, half a step of which is 2^-11
        entry = off + g.abs() * (ENTRY[t] + (2.0 ** -11 if t == "bf16" and bias is None else 0.0))
        gx[rows] = g @ W
        bx[rows] = (entry @ W.abs() + (k + 64) * U * (g.abs() @ W.abs())) * (1 + STEP[t]) + gx[rows].abs() * STEP[t] + LEAST[t]
        gw += g.t() @ X
        gb += g.sum(dim=0)
        bw += entry.t() @ X.abs()
        bb += off.sum(dim=0)
        sw += g.abs().t() @ X.abs()
        sb += g.abs().sum(dim=0)
        counted += rows.numel()
    bw = (bw + (counted + 64) * U * sw) * (1 + STEP[t]) + gw.abs() * STEP[t] + LEAST[t]
    return (loss, gx, gw, gb), (bl, bx, bw, bb + (counted + 64) * U * sb + gb.abs() * U)


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("n,f,k,masked", [(300000, 20, 40, "some"), (131073, 100, 9, "none"), (280000, 7, 300, "first")])
def test_rows_in_parts(n, f, k, masked, dtype):
    """At most 131072 rows are one part."""
    gen = torch.Generator(device="cuda").manual_seed(n)
    x = (torch.rand((n, f), generator=gen, device="cuda") * 0.5).to(TYPES[dtype])
    w = (torch.randn((k, f), generator=gen, device="cuda") * 0.3).to(TYPES[dtype])
    y = torch.randint(0, k // 2, (n,), generator=gen, device="cuda")  # the other classes' entries of G are all positive
    if masked == "some":
        y[torch.rand(n, generator=gen, device="cuda") < 0.2] = k
    if masked == "first":  # not one row of the first part, and of the last one, counts
        y[:140001] = -1
        y[279000:] = -1
    x[(y < 0) | (y >= k)] = float("nan")
    # (weights far apart from part to part: half precision has a power of two for each)
    weight = (torch.rand(n, generator=gen, device="cuda") + 0.5) * torch.where(torch.arange(n, device="cuda") < n // 2, 2e-3, 1e-2)
    bias = torch.randn(k, generator=gen, device="cuda")
    for b, wt in ((None, None), (bias, weight), (None, weight)):
        if wt is None and dtype == "f16":
            wt = torch.full((n,), 2.0 ** -6, device="cuda")  # (the sums of 300000 rows pass the largest number)
        want, bound = reference_by_rows(x, w, y, b, wt, dtype, 50000)
        got = ops.linear_log_loss_gradient(x, w, y, sample_weight=wt, bias=b)
        for i, name in enumerate(("loss", "grad_X", "grad_weight", "grad_bias")[:len(got)]):
            assert_within(got[i], want[i], bound[i], name)
        again = ops.linear_log_loss_gradient(x, w, y, sample_weight=wt, bias=b)
        assert all(torch.equal(p, q) for p, q in zip(got, again))
        assert_within(ops.linear_log_loss(x, w, y, bias=b), want[0], bound[0], "loss alone")


def test_rows_in_parts_and_classes_in_pieces():
    """Two parts of 65792 rows: 4 GiB of G and its exponentials are 6400 classes of float."""
    n, f, k = 131100, 8, 6600
    assert 10 * 65792 * k > 4 << 30
    gen = torch.Generator(device="cuda").manual_seed(5)
    x = torch.rand((n, f), generator=gen, device="cuda") * 0.5
    w = torch.randn((k, f), generator=gen, device="cuda") * 0.3
    y = torch.randint(0, k // 2, (n,), generator=gen, device="cuda")
    want, bound = reference_by_rows(x, w, y, None, None, "f32", 20000)
    for i, got in enumerate(ops.linear_log_loss_gradient(x, w, y)):
        assert_within(got, want[i], bound[i], ("loss", "grad_X", "grad_weight")[i])
    assert_within(ops.linear_log_loss(x, w, y), want[0], bound[0], "loss alone")


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
def test_rows_in_parts_captured_and_replayed(dtype):
    n, f, k = 140000, 10, 9
    gen = torch.Generator(device="cuda").manual_seed(13)
    x = torch.rand((n, f), generator=gen, device="cuda").to(TYPES[dtype])
    w = torch.randn((k, f), generator=gen, device="cuda").to(TYPES[dtype])
    y = torch.randint(-1, k, (n,), generator=gen, device="cuda")
    weight, bias = torch.rand(n, generator=gen, device="cuda") * 1e-3, torch.randn(k, generator=gen, device="cuda")
    ops.linear_log_loss_gradient(x, w, y, sample_weight=weight, bias=bias)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = ops.linear_log_loss_gradient(x, w, y, sample_weight=weight, bias=bias) + (ops.linear_log_loss(x, w, y),)
    for _ in range(3):
        y.copy_(torch.roll(y, 70001))
        weight.mul_(3.0)
        graph.replay()
        want = ops.linear_log_loss_gradient(x, w, y, sample_weight=weight, bias=bias) + (ops.linear_log_loss(x, w, y),)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
def test_rows_in_parts_where_memory_is_short(dtype, monkeypatch):
    """Two parts of the rows, and the least workspace: several pieces of the classes in each."""
    n, f, k = 140000, 20, 3000
    size = _lib.lib.lbt_linear_log_loss_workspace_bytes
    full, least = (size(n, f, k, ops._DT_NARROW[TYPES[dtype]], kind) for kind in (2, 2 + _lib.LBT_LEAST_WORKSPACE))
    assert least < full / 2

    def scratch(nbytes, device):
        if nbytes > least:
            raise torch.OutOfMemoryError("no room")
        return torch.empty(nbytes, dtype=torch.uint8, device=device)

    monkeypatch.setattr(ops, "_scratch", scratch)
    gen = torch.Generator(device="cuda").manual_seed(11)
    x = (torch.rand((n, f), generator=gen, device="cuda") * 0.5).to(TYPES[dtype])
    w = (torch.randn((k, f), generator=gen, device="cuda") * 0.3).to(TYPES[dtype])
    y = torch.randint(0, k // 2, (n,), generator=gen, device="cuda")
    y[::5] = -1
    x[::5] = float("nan")
    weight = (torch.rand(n, generator=gen, device="cuda") + 0.5) * torch.where(torch.arange(n, device="cuda") < n // 2, 2e-3, 1e-2)
    bias = torch.randn(k, generator=gen, device="cuda")
    want, bound = reference_by_rows(x, w, y, bias, weight, dtype, 20000)
    for i, got in enumerate(ops.linear_log_loss_gradient(x, w, y, sample_weight=weight, bias=bias)):
        assert_within(got, want[i], bound[i], ("loss", "grad_X", "grad_weight", "grad_bias")[i])


@pytest.mark.parametrize("dtype,n,f", [("f32", 9000, 66000), ("f16", 8300, 132000), ("bf16", 8300, 131073)])
def test_parts_of_long_rows(dtype, n, f):
    """At most 2^30 values of planes are one part."""
    gen = torch.Generator(device="cuda").manual_seed(7)
    k = 20
    x = torch.rand((n, f), generator=gen, device="cuda").mul_(0.5).to(TYPES[dtype])
    w = (torch.randn((k, f), generator=gen, device="cuda") * 0.005).to(TYPES[dtype])
    y = torch.randint(0, k // 2, (n,), generator=gen, device="cuda")
    weight = torch.full((n,), 2.0 ** -4, device="cuda")
    want, bound = reference_by_rows(x, w, y, None, weight, dtype, 1500)
    for i, got in enumerate(ops.linear_log_loss_gradient(x, w, y, sample_weight=weight)):
        assert_within(got, want[i], bound[i], ("loss", "grad_X", "grad_weight")[i])


# ---- rows of a table ---------------------------------------------------------------------------------


@pytest.mark.parametrize("kind", ["uniform", "one", "few"])
@pytest.mark.parametrize("rows", [1, 700, 60000, 1500000])  # one, one, two and three digits of the sort
@pytest.mark.parametrize("t", [131073, 135201, 524288, 524289, 700003])
def test_long_sorts(t, rows, kind):
    """Beyond 131072 places a thread of the sort has four entries, beyond 524288 the blocks' offsets have a launch of their own. Whole
    numbers below 8 are summed exactly: any place that is lost, doubled or misplaced is seen."""
    gen = torch.Generator(device="cuda").manual_seed(t + rows)
    if kind == "uniform":
        tokens = torch.randint(-1, rows + 1, (t,), generator=gen, device="cuda")  # some name no row
    elif kind == "one":
        tokens = torch.full((t,), rows - 1, device="cuda")
    else:
        tokens = torch.randint(0, 5, (t,), generator=gen, device="cuda") * (rows // 5)
    grad = torch.randint(-8, 9, (t, 4), generator=gen, device="cuda").float()
    inside = (tokens >= 0) & (tokens < rows)
    # (on the host: atomic sums of equal tokens would wait for one another)
    want = torch.zeros((rows, 4), dtype=torch.float64).index_add_(0, tokens[inside].cpu(), grad[inside].double().cpu()).cuda()
    assert 8 * t < 1 << 24
    got = ops.embed_rows_gradient(grad, tokens, rows)
    assert torch.equal(got.double(), want)
    assert torch.equal(ops.embed_rows_gradient(grad, tokens.to(torch.int32), rows), got)
    old = torch.randint(-8, 9, (rows, 4), generator=gen, device="cuda").float()
    assert torch.equal(ops.embed_rows_gradient(grad, tokens, rows, add_to=old.clone()).double(), want + old.double())
    # numbers that round: the same bits from call to call
    grad = torch.randn((t, 4), generator=gen, device="cuda").to(torch.bfloat16)
    assert torch.equal(ops.embed_rows_gradient(grad, tokens, rows, scale=1.3), ops.embed_rows_gradient(grad, tokens, rows, scale=1.3))


# ---- more than 2^32 threads --------------------------------------------------------------------------
# (a launch has fewer: these are several)


@pytest.mark.parametrize("f,t", [(67, (1 << 26) + 1001), (9, (1 << 28) + 5)])  # 64 and 16 threads a row
def test_lookups_of_many_tokens(f, t):
    gen = torch.Generator(device="cuda").manual_seed(f)
    table = torch.randn((77, f), generator=gen, device="cuda").to(torch.bfloat16)
    tokens = torch.randint(-1, 78, (t,), generator=gen, device="cuda", dtype=torch.int32)
    got = ops.embed_rows(table, tokens, 2.0)
    clean = torch.cat([table * 2, torch.zeros((1, f), dtype=table.dtype, device="cuda")])  # (twice a number is exact)
    for i in range(0, t, 1 << 24):
        part = tokens[i:i + (1 << 24)].long()
        assert torch.equal(got[i:i + (1 << 24)], clean[torch.where(part < 0, 77, part)])


@pytest.mark.parametrize("t", [5, 3000])  # without sorting, and sorted with rows cleared apart
def test_tables_of_many_rows(t):
    rows = (1 << 30) - 64
    gen = torch.Generator(device="cuda").manual_seed(t)
    tokens = torch.randint(0, rows, (t,), generator=gen, device="cuda")
    tokens[0], tokens[1], tokens[2] = rows - 1, 0, rows
    grad = torch.randint(1, 9, (t, 1), generator=gen, device="cuda").to(torch.bfloat16)
    got = ops.embed_rows_gradient(grad, tokens, rows)
    named, where = torch.unique(tokens[tokens < rows], return_inverse=True)
    want = torch.zeros(named.numel(), dtype=torch.float64).index_add_(0, where.cpu(), grad[tokens < rows, 0].double().cpu())
    assert torch.equal(got[named, 0].double().cpu(), want)
    assert sum(int(torch.count_nonzero(got[i:i + (1 << 28)])) for i in range(0, rows, 1 << 28)) == named.numel()
    to = torch.ones((rows, 1), dtype=torch.bfloat16, device="cuda")
    ops.embed_rows_gradient(grad, tokens, rows, add_to=to)
    assert torch.equal(to[named, 0].double().cpu(), want + 1)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_bias_of_many_classes(dtype):
    n, f, k = 6, 8, (1 << 26) + 1000
    gen = torch.Generator(device="cuda").manual_seed(1)
    x = torch.rand((n, f), generator=gen, device="cuda").to(TYPES[dtype])
    w = (torch.randn((k, f), generator=gen, device="cuda") * 0.3).to(TYPES[dtype])
    y = torch.randint(0, k, (n,), generator=gen, device="cuda")
    bias = torch.randn(k, generator=gen, device="cuda")
    y[0], y[1] = k - 1, 0
    loss, _, _, gb = ops.linear_log_loss_gradient(x, w, y, bias=bias)
    alone = ops.linear_log_loss(x, w, y, bias=bias)
    want, off, sizes = (torch.zeros(k, dtype=torch.float64, device="cuda") for _ in range(3))
    for r in range(n):  # as reference_by_rows, loss and grad_bias alone
        s, size = bias.double(), bias.double().abs()
        for i in range(f):
            s, size = s + x[r, i].double() * w[:, i].double(), size + x[r, i].double().abs() * w[:, i].double().abs()
        rel = float(2 * ((f + 8) * U + 2.0 ** -22) * size.max() + 1e-4)
        lse = torch.logsumexp(s, dim=0)
        assert abs(float(lse - s[y[r]] - loss[r])) <= rel + 8 * U * (abs(float(lse)) + 1.0)
        assert abs(float(lse - s[y[r]] - alone[r])) <= rel + 8 * U * (abs(float(lse)) + 1.0)
        p = torch.exp(s - lse)
        off += p * rel
        p[y[r]] -= 1.0
        want += p
        sizes += p.abs()
    assert_within(gb, want, off + (n + 68) * U * sizes + want.abs() * U, "grad_bias")
