"""Performance cases of the operators that a graph network needs between its sparse products: the classifier head with
its softmax cross entropy over the labelled nodes (``engine.linear_cross_entropy``, with and without gradients) and group
norm with an activation over the node features of one graph or a batch of graphs (``engine.group_norm``,
``engine.group_norm_backward``).

Inputs are drawn on the GPU from the seed alone.  ``run`` computes the plain form (elementary torch operations in 32 bits)
or, with ``own``, calls the library.
"""
import math

import torch

DEVICE = "cuda"
own = False
DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


# ---- cases -------------------------------------------------------------------------------------
def _xent(rows, dim, classes, dtype="f32", labelled=1.0, layout="dim", grads=True, **name):
    """``layout``: the axis of the weight that is contiguous: "class" as in ``hidden @ W2`` of a GCN, "dim" as in a table
    with one embedding per entity."""
    return dict(**name, path="xent", rows=rows, dim=dim, classes=classes, dtype=dtype, labelled=labelled, layout=layout, grads=grads)


def _norm(path, graphs, rows, channels, groups, dtype="f32", activation="none", ragged=False, **name):
    """``rows``: of a graph (the mean over the batch where the graphs are ``ragged``)."""
    return dict(**name, path=path, graphs=graphs, rows=rows, channels=channels, groups=groups, dtype=dtype, activation=activation, ragged=ragged)


def listed():
    return [
        # a citation graph, semi-supervised: a few labelled nodes, 16 hidden features, 7 classes; launches and host time count
        _xent(2708, 16, 7, labelled=0.05, layout="class", name="xent-citation"),
        # the head of the 130 000-node training step (128 features, 47 classes), a tenth of the nodes labelled
        _xent(130000, 128, 47, labelled=0.1, layout="class", name="xent-train-130k"),
        # the head of the 512-wide network with 512 classes, every node labelled
        _xent(1 << 18, 512, 512, layout="class", name="xent-gcn-512"),
        # entity prediction in a knowledge graph: a batch of queries against every entity, odd sizes
        _xent(1000, 200, 40943, name="xent-entities"),
        # the same against a large graph's entities in 16 bits: the largest head
        _xent(16384, 512, 131072, dtype="bf16", name="xent-entities-large"),
        # evaluation: only the loss of each row, odd number of classes
        _xent(8192, 256, 50001, dtype="bf16", grads=False, name="xent-eval"),
        # evaluation of a handful of queries
        _xent(16, 256, 100003, dtype="f16", grads=False, name="xent-eval-few"),
        # the citation graph's hidden layer
        _norm("norm", 1, 2708, 64, 8, activation="relu", name="norm-citation"),
        # a batch of molecule-sized graphs, backward
        _norm("norm-backward", 256, 39, 128, 16, dtype="bf16", activation="silu", ragged=True, name="norm-molecules-backward"),
        # hidden layer of a full graph
        _norm("norm", 1, 1 << 18, 512, 32, activation="relu", name="norm-graph-512"),
        # a batch of mid-sized graphs, ten channels a group
        _norm("norm", 32, 4096, 320, 32, dtype="f16", activation="silu", ragged=True, name="norm-batch-320"),
        # hidden layer of a full graph in 16 bits, backward
        _norm("norm-backward", 1, 300007, 256, 16, dtype="bf16", activation="silu", name="norm-graph-256-backward"),
    ]


def _log(rng, lo, hi):
    return math.exp(rng.uniform(math.log(lo), math.log(hi)))


def draw(rng):
    dtype = rng.choice(["f32", "f32", "bf16", "bf16", "f16"])
    path = rng.choice(["xent", "xent", "norm", "norm-backward"])
    if path == "xent":
        grads = rng.random() < 0.6
        dim, classes = int(_log(rng, 16, 1024)), int(_log(rng, 4, 131072))
        rows = _log(rng, 8, 1 << 18)
        rows = int(max(8, min(rows, (1 << 31) / classes, 1.0e12 / (dim * classes), (1 << 27) / dim)))
        labelled = 1.0 if rng.random() < 0.5 else round(rng.uniform(0.05, 1.0), 3)
        return _xent(rows, dim, classes, dtype, labelled, rng.choice(["dim", "class"]), grads)
    groups = rng.choice([1, 4, 8, 16, 32])
    channels = groups * max(1, int(_log(rng, 16, 512) / groups))
    graphs = rng.choice([1, 1, int(_log(rng, 2, 512))])
    # at least 64 values to a group: the gradient of a group of two values is all cancellation
    rows = int(max(64 * groups // channels, 2, min(_log(rng, 2, 1 << 18), (1 << 27) / (channels * graphs))))
    activation = rng.choice(["none", "silu", "relu"] if path == "norm" else ["none", "silu"])
    return _norm(path, graphs, rows, channels, groups, dtype, activation, graphs > 1 and rng.random() < 0.7)


# ---- inputs ------------------------------------------------------------------------------------
def _normal(gen, *shape):
    return torch.randn(*shape, generator=gen, device=DEVICE)


def _prepare_xent(case, gen):
    """Hidden features of unit variance; a weight whose logits have a standard deviation of about two; labels drawn evenly;
    the labelled nodes at random places, every other label -1.  16-bit floats train with a scaled loss."""
    R, D, V, dtype = case["rows"], case["dim"], case["classes"], DTYPES[case["dtype"]]
    hidden = _normal(gen, R, D).to(dtype)
    weight = (_normal(gen, V, D).mul_(2.0 / math.sqrt(D))).to(dtype)
    weight = weight.t() if case["layout"] == "dim" else weight.t().contiguous()
    labels = torch.randint(0, V, (R,), generator=gen, device=DEVICE)
    if case["labelled"] < 1.0:
        off = torch.randperm(R, generator=gen, device=DEVICE)[_labelled(case):]
        labels[off] = -1
    return dict(hidden=hidden, weight=weight, labels=labels, scale=4096.0 if case["dtype"] == "f16" else 1.0)


def _prepare_norm(case, gen):
    """Features with a mean per channel; the graphs' sizes of a ragged batch between a quarter and about twice the mean."""
    B, L, Ch, dtype = case["graphs"], case["rows"], case["channels"], DTYPES[case["dtype"]]
    sizes = torch.full((B,), L, device=DEVICE)
    if case["ragged"]:
        share = 0.25 + 1.5 * torch.rand(B, generator=gen, device=DEVICE)
        sizes = 1 + (share / share.sum() * (B * (L - 1))).to(torch.int64).clamp_(max=B * (L - 1))
        sizes[-1] = torch.clamp(B * L - sizes[:-1].sum(), min=1)
    offsets = torch.zeros(B + 1, dtype=torch.int32, device=DEVICE)
    offsets[1:] = torch.cumsum(sizes, 0)
    R = B * L
    x = (_normal(gen, R, Ch) * (0.5 + torch.rand(Ch, generator=gen, device=DEVICE)) + _normal(gen, Ch)).to(dtype)
    state = dict(x=x, offsets=offsets if B > 1 else None, weight=1.0 + 0.2 * _normal(gen, Ch), bias=0.2 * _normal(gen, Ch))
    if case["path"] == "norm-backward":
        state["grad"] = _normal(gen, R, Ch).to(dtype)
        # what the forward pass left behind
        n = torch.clamp(sizes, min=1).double()[:, None] * (Ch // case["groups"])
        sums = _per_graph(x.double(), state["offsets"], B).reshape(B, case["groups"], -1).sum(2)
        mean = sums / n
        centred = x.double() - _per_row(mean, state["offsets"], R).repeat_interleave(Ch // case["groups"], 1)
        var = _per_graph(centred.square(), state["offsets"], B).reshape(B, case["groups"], -1).sum(2) / n
        state["mean"], state["rstd"] = mean.float(), torch.rsqrt(var + 1e-5).float()
    return state


def prepare(case, seed):
    gen = torch.Generator(device=DEVICE).manual_seed(seed)
    state = _prepare_xent(case, gen) if case["path"] == "xent" else _prepare_norm(case, gen)
    return dict(state, case=case)


# ---- the plain form ------------------------------------------------------------------------------
def _per_graph(x, offsets, graphs):
    """Sums of the rows of each graph: [rows, channels] -> [graphs, channels]."""
    if offsets is None:
        return x.sum(0, keepdim=True)
    graph = torch.repeat_interleave(torch.arange(graphs, device=x.device), offsets.diff().long(), output_size=x.shape[0])
    return x.new_zeros(graphs, x.shape[1]).index_add_(0, graph, x)


def _per_row(v, offsets, rows):
    """Each graph's values for its rows: [graphs, n] -> [rows, n]."""
    return v.expand(rows, -1) if offsets is None else torch.repeat_interleave(v, offsets.diff().long(), 0, output_size=rows)


def _plain_xent(state):
    case, V = state["case"], state["case"]["classes"]
    labels = state["labels"]
    rows = torch.nonzero((labels >= 0) & (labels < V)).squeeze(1)
    h, w, y = state["hidden"][rows].float(), state["weight"].float(), labels[rows]
    logits = h @ w
    top = logits.amax(1, keepdim=True)
    p = torch.exp(logits - top)
    total = p.sum(1, keepdim=True)
    loss = (torch.log(total) + top - logits.gather(1, y[:, None])).squeeze(1)
    if not case["grads"]:
        out = torch.zeros(labels.shape, device=p.device)
        out[rows] = loss
        return {"loss": out}
    del logits
    p /= total
    at = torch.arange(len(y), device=p.device)
    p[at, y] -= 1.0
    p *= state["scale"] / len(y)
    dhidden = torch.zeros(state["hidden"].shape, device=p.device)
    dhidden[rows] = p @ w.t()
    return {"loss": loss.mean(), "dhidden": dhidden.to(state["hidden"].dtype), "dweight": (h.t() @ p).to(state["weight"].dtype)}


def _plain_norm(state):
    case, offsets, B, G = state["case"], state["offsets"], state["case"]["graphs"], state["case"]["groups"]
    x = state["x"].float()
    R, Ch = x.shape
    n = (offsets.diff().float()[:, None] if offsets is not None else float(R)) * (Ch // G)
    mean = _per_graph(x, offsets, B).reshape(B, G, -1).sum(2) / n
    centred = x - _per_row(mean.repeat_interleave(Ch // G, 1), offsets, R)
    var = _per_graph(centred.square(), offsets, B).reshape(B, G, -1).sum(2) / n
    rstd = torch.rsqrt(var + 1e-5)
    u = centred * _per_row(rstd.repeat_interleave(Ch // G, 1), offsets, R) * state["weight"] + state["bias"]
    if case["activation"] == "relu":
        u = torch.clamp(u, min=0.0)
    elif case["activation"] == "silu":
        u = u * torch.sigmoid(u)
    return {"y": u.to(state["x"].dtype), "mean": mean, "rstd": rstd}


def _plain_norm_backward(state):
    case, offsets, B, G = state["case"], state["offsets"], state["case"]["graphs"], state["case"]["groups"]
    x = state["x"].float()
    R, Ch = x.shape
    n = (offsets.diff().float()[:, None] if offsets is not None else float(R)) * (Ch // G)
    rstd = _per_row(state["rstd"].repeat_interleave(Ch // G, 1), offsets, R)
    xhat = (x - _per_row(state["mean"].repeat_interleave(Ch // G, 1), offsets, R)) * rstd
    du = state["grad"].float()
    if case["activation"] == "silu":
        u = xhat * state["weight"] + state["bias"]
        s = torch.sigmoid(u)
        du = du * (s * (1.0 + u * (1.0 - s)))
    s1, s2 = _per_graph(du, offsets, B), _per_graph(du * xhat, offsets, B)
    m1 = (s1 * state["weight"]).reshape(B, G, -1).sum(2) / n
    m2 = (s2 * state["weight"]).reshape(B, G, -1).sum(2) / n
    dx = rstd * (du * state["weight"] - _per_row(m1.repeat_interleave(Ch // G, 1), offsets, R)
                 - xhat * _per_row(m2.repeat_interleave(Ch // G, 1), offsets, R))
    return {"dx": dx.to(state["x"].dtype), "dweight": s2.sum(0), "dbias": s1.sum(0)}


def _own(state):
    from mask_b200 import engine
    case = state["case"]
    if case["path"] == "xent":
        operands = state["hidden"], state["weight"], state["labels"]
        if not case["grads"]:
            return {"loss": engine.linear_cross_entropy(*operands, reduction="none")}
        return dict(zip(("loss", "dhidden", "dweight"), engine.linear_cross_entropy(*operands, grads=True, grad_scale=state["scale"])))
    more = dict(weight=state["weight"], bias=state["bias"], offsets=state["offsets"], activation=case["activation"])
    if case["path"] == "norm":
        return dict(zip(("y", "mean", "rstd"), engine.group_norm(state["x"], case["groups"], eps=1e-5, **more)))
    return dict(zip(("dx", "dweight", "dbias"),
                    engine.group_norm_backward(state["grad"], state["x"], state["mean"], state["rstd"], case["groups"], **more)))


def run(state):
    if own:
        return _own(state)
    return {"xent": _plain_xent, "norm": _plain_norm, "norm-backward": _plain_norm_backward}[state["case"]["path"]](state)


# ---- what a pass cannot do without ---------------------------------------------------------------
def _labelled(case):
    return max(1, round(case["rows"] * case["labelled"]))


def work(case):
    """Head: the labelled rows, the weight and the labels read once, the gradients (or the loss of every row) written once; the
    logits' product, with gradients the two products behind it.  Norm: the features read once (backward: with the
    gradient), the result written once."""
    size = 4 if case["dtype"] == "f32" else 2
    if case["path"] == "xent":
        R, D, V, n = case["rows"], case["dim"], case["classes"], _labelled(case)
        read = size * D * (n + V) + 8 * R
        return {"bytes": float(read + (size * D * (R + V) if case["grads"] else 4 * R)), "flops": (6.0 if case["grads"] else 2.0) * n * D * V}
    elements = float(case["graphs"] * case["rows"] * case["channels"])
    return {"bytes": (2.0 if case["path"] == "norm" else 3.0) * size * elements, "flops": (8.0 if case["path"] == "norm" else 16.0) * elements}


# ---- the definition in 64 bits ---------------------------------------------------------------------
def _exact_xent(state):
    """Pieces of rows whose logits take a gigabyte; ``torch.nn`` functions instead of the formulas above."""
    case, D, V = state["case"], state["case"]["dim"], state["case"]["classes"]
    labels, w = state["labels"], state["weight"].double()
    rows = torch.arange(len(labels), device=DEVICE)[labels >= 0]
    loss, dw, dh = torch.zeros(len(labels), dtype=torch.float64, device=DEVICE), torch.zeros(D, V, dtype=torch.float64, device=DEVICE), torch.zeros(len(labels), D, dtype=torch.float64, device=DEVICE)
    for part in rows.split(max(1, (1 << 27) // V)):
        h = state["hidden"][part].double()
        logp = torch.log_softmax(h @ w, 1)
        hot = torch.zeros_like(logp).scatter_(1, labels[part, None], 1.0)
        loss[part] = -(logp * hot).sum(1)
        if case["grads"]:
            g = (logp.exp() - hot) * (state["scale"] / len(rows))
            dh[part], dw = g @ w.t(), dw + h.t() @ g
    return {"loss": loss.sum() / len(rows), "dhidden": dh, "dweight": dw} if case["grads"] else {"loss": loss}


def _exact_norm(state):
    """One graph at a time, through autograd for the gradients."""
    case, G = state["case"], state["case"]["groups"]
    bounds = state["offsets"].tolist() if state["offsets"] is not None else [0, len(state["x"])]
    backward = case["path"] == "norm-backward"
    w = state["weight"].double().requires_grad_(backward)
    b = state["bias"].double().requires_grad_(backward)
    y, means, rstds = [], [], []
    for lo, hi in zip(bounds, bounds[1:]):
        x = state["x"][lo:hi].double().requires_grad_(backward)
        per = x.reshape(hi - lo, G, -1)
        mean, var = per.mean((0, 2)), per.var((0, 2), unbiased=False)
        rstd = (var + 1e-5).rsqrt()
        u = ((per - mean[:, None]) * rstd[:, None]).reshape(hi - lo, -1) * w + b
        out = {"none": lambda v: v, "relu": torch.relu, "silu": torch.nn.functional.silu}[case["activation"]](u)
        if backward:
            out.backward(state["grad"][lo:hi].double())
            y.append(x.grad)
        else:
            y.append(out)
            means.append(mean)
            rstds.append(rstd)
    if backward:
        return {"dx": torch.cat(y), "dweight": w.grad, "dbias": b.grad}
    return {"y": torch.cat(y), "mean": torch.stack(means), "rstd": torch.stack(rstds)}


def exact(case, seed):
    state = prepare(case, seed)
    return _exact_xent(state) if case["path"] == "xent" else _exact_norm(state)
