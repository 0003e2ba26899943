"""Performance cases of the operators for vocabularies: the softmax loss of linear scores over many classes with its gradient,
and the lookup of embedding rows with its gradient.

`listed()` names the cases, `draw(rng)` gives further ones of the same ranges, `prepare(case, seed)` makes what a program has in
hand before the call, `run(state)` is one pass, `work(case)` states the bytes and operations such a pass cannot do without,
`exact(case, seed)` gives the result from the definition in 64 bits.

With `own` false a pass is written with elementary torch operations in 32 bits, with `own` true it is the call of lbtree.ops.

Operations:
  loss            loss[r] = log sum_c exp(s[r, c]) - s[r, y[r]] with s = X weight^T + bias; 0 where y[r] is no class
  gradient        that loss, and the gradients of sum_r w[r] loss[r] with respect to X, weight and bias
  embed           out[t] = scale * table[tokens[t]]; zeros where tokens[t] is no row of the table
  embed_gradient  out[v] = scale * the sum of grad[t] over all t with tokens[t] = v
"""
import math
import os
import sys

import torch

own = False

_TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
_BYTES = {"bf16": 2, "f16": 2, "f32": 4}
# the most that a drawn case computes or writes: what the largest listed ones do
_MOST_PRODUCTS = 8192 * 4096 * 131072
_MOST_TABLE = 131072 * 2048


def _loss_case(name, op, dtype, rows, features, classes, masked=0.0, bias=False, weighted=False):
    case = {"op": op, "dtype": dtype, "rows": rows, "features": features, "classes": classes, "masked": masked, "bias": bias,
            "weighted": weighted}
    if name:
        case["name"] = name
    return case


def _embed_case(name, op, dtype, tokens, features, table):
    case = {"op": op, "dtype": dtype, "tokens": tokens, "features": features, "table": table}
    if name:
        case["name"] = name
    return case


def listed():
    return [
        # the score of one answer among a vocabulary: a single row, the time is that of reading the weights
        _loss_case("loss_1x1024x32768_bf16", "loss", "bf16", 1, 1024, 32768),
        # a small batch against a vocabulary of an odd size, single precision, class priors as the bias
        _loss_case("loss_33x1000x10007_f32", "loss", "f32", 33, 1000, 10007, bias=True),
        # evaluation over a batch of sequences, a tenth of the rows padded
        _loss_case("loss_8192x2048x65536_bf16", "loss", "bf16", 8192, 2048, 65536, masked=0.1),
        # a training step of a small head: a thousand classes, few rows
        _loss_case("gradient_64x256x1000_f32", "gradient", "f32", 64, 256, 1000),
        # an ordinary training step
        _loss_case("gradient_4096x2048x32768_bf16", "gradient", "bf16", 4096, 2048, 32768, masked=0.1),
        # odd sizes, weighted rows, a third of them left out, class priors: half precision, its loss scaled
        _loss_case("gradient_1531x1000x30011_f16", "gradient", "f16", 1531, 1000, 30011, masked=0.33, bias=True, weighted=True),
        # training in single precision
        _loss_case("gradient_2048x1024x16384_f32", "gradient", "f32", 2048, 1024, 16384),
        # the largest step
        _loss_case("gradient_8192x4096x131072_bf16", "gradient", "bf16", 8192, 4096, 131072),
        # the tokens of one step of a batch of sixteen
        _embed_case("embed_16x2048x32768_bf16", "embed", "bf16", 16, 2048, 32768),
        # a batch of training sequences
        _embed_case("embed_65536x2048x131072_bf16", "embed", "bf16", 65536, 2048, 131072),
        # categories of a table's column, odd sizes, single precision
        _embed_case("embed_gradient_1000x200x5003_f32", "embed_gradient", "f32", 1000, 200, 5003),
        # a batch of training sequences: few tokens take most of the places
        _embed_case("embed_gradient_65536x2048x65536_bf16", "embed_gradient", "bf16", 65536, 2048, 65536),
    ]


def _log_uniform(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["loss", "gradient", "gradient", "embed", "embed_gradient"])
    dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
    features = _log_uniform(rng, 64, 4096)
    if rng.random() < 0.5:
        features = max(64, features // 64 * 64)
    if op in ("loss", "gradient"):
        classes = _log_uniform(rng, 1000, 131072)
        most = _MOST_PRODUCTS // (features * classes)
        rows = _log_uniform(rng, 1 if op == "loss" else 16, max(16, min(8192, most)))
        masked = rng.choice([0.0, 0.1, 0.4])
        return _loss_case("", op, dtype, rows, features, classes, masked=masked if rows > 16 else 0.0,
                          bias=rng.random() < 0.4, weighted=op == "gradient" and rng.random() < 0.4)
    table = _log_uniform(rng, 1000, min(262144, _MOST_TABLE // features))
    tokens = _log_uniform(rng, 1, min(131072, 65536 * 2048 // features))
    return _embed_case("", op, dtype, tokens, features, table)


# ---- inputs ---------------------------------------------------------------------------------------------


def _skewed(gen, n, size):
    """n numbers below `size`, some far more frequent than others, as words and categories are, in no order of frequency."""
    u = torch.rand(n, generator=gen, device="cuda", dtype=torch.float64)
    rank = (torch.exp(u * math.log(size + 1.0)) - 1.0).to(torch.int64).clamp_(0, size - 1)
    step = int(size * 0.618) | 1
    while math.gcd(step, size) != 1:
        step += 2
    return (rank * step + 12345) % size


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dtype, f = _TYPES[case["dtype"]], case["features"]
    state = {"op": case["op"]}
    if case["op"] in ("loss", "gradient"):
        n, k = case["rows"], case["classes"]
        weight = torch.randn((k, f), generator=gen, device="cuda") * (1.5 / math.sqrt(f))
        y = _skewed(gen, n, k)
        # half of the rows lean towards their class, as those of a model that has learnt something
        lean = 4.0 * (torch.rand((n, 1), generator=gen, device="cuda") < 0.5)
        x = torch.randn((n, f), generator=gen, device="cuda") + lean * weight[y]
        left_out = torch.randperm(n, generator=gen, device="cuda")[:int(case["masked"] * n)]
        y[left_out] = -1
        state.update(x=x.to(dtype), weight=weight.to(dtype), y=y, bias=None, row_weight=None)
        if case["bias"]:
            state["bias"] = torch.randn(k, generator=gen, device="cuda") - math.log(k)
        if case["op"] == "gradient":
            # the mean over the rows that count; half precision takes the sum, which is the mean times a loss scale
            each = 1.0 if dtype == torch.float16 else 1.0 / (n - left_out.numel())
            if case["weighted"]:
                state["row_weight"] = (0.25 + 1.5 * torch.rand(n, generator=gen, device="cuda")) * each
            elif each != 1.0:
                state["row_weight"] = torch.full((n,), each, device="cuda")
        return state
    t, rows = case["tokens"], case["table"]
    tokens = _skewed(gen, t, rows)
    tokens[torch.rand(t, generator=gen, device="cuda") < 0.02] = -1  # padding
    state.update(tokens=tokens, scale=math.sqrt(f), rows=rows)
    if case["op"] == "embed":
        state["table"] = (torch.randn((rows, f), generator=gen, device="cuda") * 0.02).to(dtype)
    else:
        state["grad"] = torch.randn((t, f), generator=gen, device="cuda").to(dtype)
    return state


# ---- one pass -------------------------------------------------------------------------------------------


def run(state):
    op = state["op"]
    if own:
        ops = _ops()
        if op == "loss":
            return ops.linear_log_loss(state["x"], state["weight"], state["y"], bias=state["bias"])
        if op == "gradient":
            return ops.linear_log_loss_gradient(state["x"], state["weight"], state["y"], sample_weight=state["row_weight"],
                                                bias=state["bias"])
        if op == "embed":
            return ops.embed_rows(state["table"], state["tokens"], scale=state["scale"])
        return ops.embed_rows_gradient(state["grad"], state["tokens"], state["rows"], scale=state["scale"])
    if op in ("loss", "gradient"):
        return _plain_loss(state["x"], state["weight"], state["y"], state["bias"], state["row_weight"], op == "gradient")
    tokens = state["tokens"]
    counts = (tokens >= 0) & (tokens < state["rows"])
    at = torch.where(counts, tokens, 0)
    if op == "embed":
        table = state["table"]
        out = table[at].to(torch.float32) * state["scale"]
        return torch.where(counts[:, None], out, 0.0).to(table.dtype)
    grad = state["grad"]
    out = torch.zeros((state["rows"], grad.shape[1]), device=grad.device)
    out.index_add_(0, at, torch.where(counts[:, None], grad.to(torch.float32), 0.0))
    return (out * state["scale"]).to(grad.dtype)


def _plain_loss(x, weight, y, bias, row_weight, gradient):
    x32, weight32 = x.to(torch.float32), weight.to(torch.float32)
    scores = x32 @ weight32.t()
    if bias is not None:
        scores = scores + bias
    counts = (y >= 0) & (y < weight.shape[0])
    at = torch.where(counts, y, 0)[:, None]
    top = scores.max(dim=1, keepdim=True).values
    exps = torch.exp(scores - top)
    total = exps.sum(dim=1, keepdim=True)
    loss = torch.where(counts, (torch.log(total) + top - scores.gather(1, at))[:, 0], 0.0)
    if not gradient:
        return loss
    g = exps / total
    g = torch.where(torch.arange(weight.shape[0], device=x.device) == at, g - 1.0, g)
    if row_weight is not None:
        g = g * row_weight[:, None]
    g = torch.where(counts[:, None], g, 0.0)
    out = (loss, (g @ weight32).to(x.dtype), (g.t() @ x32).to(weight.dtype))
    return out if bias is None else out + (g.sum(dim=0),)


def _ops():
    package = os.path.join(os.getcwd(), "legate-boost_amd")
    if package not in sys.path:
        sys.path.insert(0, package)
    from lbtree import ops

    return ops


# ---- what a pass cannot do without ------------------------------------------------------------------------


def work(case):
    size, f = _BYTES[case["dtype"]], case["features"]
    if case["op"] in ("loss", "gradient"):
        n, k = case["rows"], case["classes"]
        counted = n - int(case["masked"] * n)
        read = (counted + k) * f * size + n * 8 + (k * 4 if case["bias"] else 0)
        if case["op"] == "loss":
            return {"bytes": read + n * 4, "flops": 2 * counted * k * f}
        read += n * 4 if case["weighted"] else 0
        written = (n + k) * f * size + n * 4 + (k * 4 if case["bias"] else 0)
        return {"bytes": read + written, "flops": 6 * counted * k * f}
    t, rows = case["tokens"], case["table"]
    if case["op"] == "embed":
        # how many rows of the table the tokens name, in the mean over their distribution
        rank = torch.arange(1, rows + 1, dtype=torch.float64)
        share = (torch.log(rank + 1.0) - torch.log(rank)) / math.log(rows + 1.0)
        named = float((1.0 - torch.exp(t * torch.log1p(-share))).sum())
        return {"bytes": int((named + t) * f * size) + t * 8, "flops": t * f}
    return {"bytes": (t + rows) * f * size + t * 8, "flops": t * f}


# ---- the definition in 64 bits ------------------------------------------------------------------------------


def exact(case, seed):
    state = prepare(case, seed)
    if case["op"] in ("loss", "gradient"):
        x, w, y = state["x"].double(), state["weight"].double(), state["y"].tolist()
        bias = None if state["bias"] is None else state["bias"].double()
        n, k = x.shape[0], w.shape[0]
        loss = torch.zeros(n, dtype=torch.float64, device="cuda")
        gradient = case["op"] == "gradient"
        if gradient:
            gx, gw, gb = torch.zeros_like(x), torch.zeros_like(w), torch.zeros(k, dtype=torch.float64, device="cuda")
        kept = [r for r in range(n) if 0 <= y[r] < k]
        step = max(1, (1 << 28) // k)
        for i in range(0, len(kept), step):
            rows = torch.tensor(kept[i:i + step], device="cuda")
            label = torch.tensor([y[r] for r in kept[i:i + step]], device="cuda")
            s = torch.mm(x[rows], w.t())
            if bias is not None:
                s += bias
            logp = torch.log_softmax(s, dim=1)
            here = torch.arange(rows.numel(), device="cuda")
            loss[rows] = -logp[here, label]
            if gradient:
                p = logp.exp_()
                p[here, label] -= 1.0
                if state["row_weight"] is not None:
                    p *= state["row_weight"].double()[rows][:, None]
                gx[rows] = torch.mm(p, w)
                gw += torch.mm(p.t(), x[rows])
                gb += p.sum(dim=0)
        if not gradient:
            return loss
        return (loss, gx, gw) if bias is None else (loss, gx, gw, gb)
    tokens = state["tokens"]
    named = tokens.ge(0).nonzero()[:, 0]
    if case["op"] == "embed":
        out = torch.zeros((tokens.numel(), case["features"]), dtype=torch.float64, device="cuda")
        out[named] = state["table"][tokens[named]].double() * state["scale"]
        return out
    # the sums of runs of equal tokens as products with the matrix of the tokens' places
    places = torch.sparse_coo_tensor(torch.stack([tokens[named], torch.arange(named.numel(), device="cuda")]),
                                     torch.ones(named.numel(), dtype=torch.float64, device="cuda"),
                                     (state["rows"], named.numel()))
    return torch.sparse.mm(places, state["grad"][named].double()) * state["scale"]
