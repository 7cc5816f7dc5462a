"""Training a two-layer GCN (``gcn.GCN2``) and the sharded evaluation loss: the chain of gradients on the CPU against
autograd with plain stand-ins for the device's pieces, and the whole step on the GPU against the same network in 64 bits."""
import numpy as np
import pytest
import torch

from mask_b200 import generators as G
from mask_b200.gcn import GCN2, FusedGCN2

NAMES = ("W1", "weight", "bias", "W2", "X")


def _dense(csr, device="cpu"):
    a = np.zeros((csr.M, csr.K))
    for i in range(csr.M):
        a[i, csr.colind[csr.rowptr[i]:csr.rowptr[i + 1]]] = csr.values[csr.rowptr[i]:csr.rowptr[i + 1]]
    return torch.from_numpy(a).to(device)


def _act(u, name):
    return {"none": lambda v: v, "relu": torch.relu, "silu": torch.nn.functional.silu}[name](u)


def _reference(A, X, W1, weight, bias, W2, labels, groups, activation, offsets, eps=1e-5, gate=None):
    """Loss and gradients in 64 bits through autograd.  ``gate``: where ReLU lets through, if another's rounding decides."""
    leaves = [t.double().clone().requires_grad_(True) for t in (W1, weight, bias, W2, X)]
    w1, w, b, w2, x = leaves
    z = A @ (x @ w1)
    bounds = offsets if offsets is not None else [0, len(X)]
    u = torch.cat([torch.nn.functional.group_norm(z[lo:hi].t()[None], groups, w, b, eps)[0].t() for lo, hi in zip(bounds, bounds[1:]) if hi > lo])
    h = _act(u, activation) if gate is None else u * gate
    logits = (A @ h) @ w2
    keep = (labels >= 0) & (labels < W2.shape[1])
    loss = torch.nn.functional.cross_entropy(logits[keep], labels[keep])
    return loss.detach(), torch.autograd.grad(loss, leaves)


class PlainOps:
    """What GCN2 asks of the device, from the formulas, in the operands' type."""

    def pack(self, csr):
        return _dense(csr)

    def spmm(self, packed, dense):
        return packed @ dense

    def _per_row(self, v, x, groups, offsets):
        sizes = offsets.diff().long() if offsets is not None else torch.tensor([len(x)])
        return v.repeat_interleave(x.shape[1] // groups, 1).repeat_interleave(sizes, 0)

    def group_norm(self, x, groups, weight, bias, offsets, eps, activation):
        bounds = offsets.tolist() if offsets is not None else [0, len(x)]
        parts = [x[lo:hi].reshape(hi - lo, groups, -1) for lo, hi in zip(bounds, bounds[1:])]
        mean = torch.stack([p.mean((0, 2)) for p in parts])
        rstd = torch.stack([(p.var((0, 2), unbiased=False) + eps).rsqrt() for p in parts])
        xhat = (x - self._per_row(mean, x, groups, offsets)) * self._per_row(rstd, x, groups, offsets)
        return _act(xhat * weight + bias, activation), mean, rstd

    def group_norm_backward(self, grad, x, mean, rstd, groups, weight, bias, offsets, activation):
        r = self._per_row(rstd, x, groups, offsets)
        xhat = (x - self._per_row(mean, x, groups, offsets)) * r
        u = xhat * weight + bias
        s = torch.sigmoid(u)
        du = grad * {"none": torch.ones_like(u), "relu": (u > 0).to(u.dtype), "silu": s * (1 + u * (1 - s))}[activation]
        bounds = offsets.tolist() if offsets is not None else [0, len(x)]
        dx = torch.empty_like(x)
        for lo, hi in zip(bounds, bounds[1:]):
            g, h = (t[lo:hi].reshape(hi - lo, groups, -1) for t in (du * weight, xhat))
            d = g - g.mean((0, 2))[:, None] - h * (g * h).mean((0, 2))[:, None]
            dx[lo:hi] = r[lo:hi] * d.reshape(hi - lo, -1)
        return dx, (du * xhat).sum(0), du.sum(0)

    def linear_cross_entropy(self, rows, weight, labels, reduction="mean", grads=False):
        keep = (labels >= 0) & (labels < weight.shape[1])
        logits = rows[keep] @ weight
        loss = torch.nn.functional.cross_entropy(logits, labels[keep], reduction=reduction)
        if not grads:
            return loss
        p = torch.softmax(logits, 1)
        p[torch.arange(len(p)), labels[keep]] -= 1
        p /= len(p)
        dh = torch.zeros_like(rows)
        dh[keep] = p @ weight.t()
        return loss, dh, rows[keep].t() @ p


def _problem(nodes, features, hidden, classes, seed, device="cpu", dtype=torch.float64):
    g = torch.Generator().manual_seed(seed)
    m = G.rmat_gcn_normalised(scale=int(np.log2(nodes)), samples_per_node=4, seed=seed)
    # not symmetric: the gradients need the transposed matrix
    m = G.CSR(m.M, m.K, m.rowptr, m.colind, (m.values * (1 + 0.5 * np.random.RandomState(seed).rand(len(m.values)))).astype(np.float32))
    labels = torch.randint(0, classes, (m.M,), generator=g)
    labels[torch.rand(m.M, generator=g) < 0.5] = -1
    tensors = [torch.randn(m.M, features, generator=g), torch.randn(features, hidden, generator=g) / features ** 0.5,
               1 + 0.2 * torch.randn(hidden, generator=g), 0.2 * torch.randn(hidden, generator=g), torch.randn(hidden, classes, generator=g) / hidden ** 0.5]
    return m, [t.to(dtype).to(device) for t in tensors], labels.to(device)


@pytest.mark.parametrize("activation,offsets", [("relu", None), ("silu", [0, 100, 101, 256]), ("none", [0, 256])])
def test_gradients_follow_the_chain(activation, offsets):
    m, (X, W1, weight, bias, W2), labels = _problem(256, 12, 16, 7, 3)
    net = GCN2(m, "cpu", 4, activation, offsets, ops=PlainOps())
    loss, grads = net.loss_and_gradients(X, W1, weight, bias, W2, labels, input_gradient=True)
    want, expected = _reference(_dense(m), X, W1, weight, bias, W2, labels, 4, activation, offsets)
    assert abs(float(loss - want)) < 1e-12 * abs(float(want))
    assert abs(float(net.loss(X, W1, weight, bias, W2, labels) - want)) < 1e-12 * abs(float(want))
    for name, e in zip(NAMES, expected):
        assert torch.allclose(getattr(grads, name), e, rtol=1e-9, atol=1e-12), name
    assert net.loss_and_gradients(X, W1, weight, bias, W2, labels)[1].X is None


def test_a_rectangular_matrix_is_refused():
    with pytest.raises(RuntimeError, match="square"):
        GCN2(G.CSR(2, 3, np.array([0, 0, 0], np.int32), np.zeros(0, np.int32), np.zeros(0, np.float32)), "cpu", 1, ops=PlainOps())


@pytest.mark.parametrize("offsets", [[0, 100], [5, 256], [0, 300, 256], [0], [0, 100, 50, 256]])
def test_offsets_that_leave_nodes_out_are_refused(offsets):
    m = G.rmat_gcn_normalised(scale=8, samples_per_node=4, seed=3)
    with pytest.raises(RuntimeError, match="offsets"):
        GCN2(m, "cpu", 4, offsets=offsets, ops=PlainOps())


class _Local:
    def __init__(self, t):
        self.local = t


class OneRankOps(PlainOps):
    def shared_h1(self, rows, cols):
        return [_Local(torch.zeros(rows, cols, dtype=torch.float64)) for _ in range(2)]

    def spmm_to_all(self, packed, dense, buf, r0, r1):
        buf.local[r0:r1] = torch.relu(packed @ dense)

    def close(self):
        pass


def test_evaluation_loss_of_the_sharded_forward():
    m, (X, W1, _, _, W2), labels = _problem(256, 12, 16, 7, 4)
    net = FusedGCN2(m, 0, 1, "cpu", np.arange(17) * 1.0, hidden=16, ops=OneRankOps())
    out = net.forward(X, W1, W2)
    want = torch.nn.functional.cross_entropy(out[labels >= 0], labels[labels >= 0])
    assert abs(float(net.loss(X, W1, W2, labels)) - float(want)) < 1e-6
    assert float(net.loss(X, W1, W2, torch.full_like(labels, -1))) == 0.0


@pytest.mark.gpu
@pytest.mark.parametrize("classes", [7, 47, 600])
@pytest.mark.parametrize("activation,offsets", [("silu", None), ("silu", [0, 300, 301, 700, 700, 1024]), ("relu", None)])
def test_training_step(activation, offsets, classes):
    """Errors of compensated products, the head and the norm are some 2^-20 of a few hundred terms each; they pass through three
    more products.  What is compared is each gradient's error against its size."""
    from mask_b200 import engine
    m, tensors, labels = _problem(1024, 50, 64, classes, 5, "cuda", torch.float32)
    net = GCN2(m, "cuda", 8, activation, offsets, tf32x3=True)
    loss, grads = net.loss_and_gradients(*tensors, labels, input_gradient=True)
    X, W1, weight, bias, W2 = tensors
    gate = None
    if activation == "relu":      # the gate is the sign of a rounded value: the kernel's own output says which
        Z = engine.spmm_any_width(net.A, X @ W1, tf32x3=True)
        gate = (engine.group_norm(Z, 8, weight, bias, net.offsets, activation="relu")[0] > 0).double()
    want, expected = _reference(_dense(m, "cuda"), *tensors, labels, 8, activation, offsets, gate=gate)
    assert abs(float(loss) - float(want)) < 2e-5 * abs(float(want))
    for name, e in zip(NAMES, expected):
        off = (getattr(grads, name).double() - e).norm() / e.norm()
        assert float(off) < 2e-4, (name, float(off))


@pytest.mark.gpu
def test_training_step_in_a_graph():
    """The step captured, replayed after its parameters were updated in place, while eager steps run between the replays."""
    m, tensors, labels = _problem(512, 48, 32, 300, 6, "cuda", torch.float32)
    net = GCN2(m, "cuda", 4, "silu")
    for _ in range(2):
        net.loss_and_gradients(*tensors, labels)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    side = torch.cuda.Stream()
    with torch.cuda.graph(graph, stream=side):
        loss, grads = net.loss_and_gradients(*tensors, labels)
    for step in range(3):
        want, expected = net.loss_and_gradients(*[t.clone() for t in tensors], labels)
        graph.replay()
        assert torch.equal(loss, want)
        for name in NAMES[:4]:
            assert torch.equal(getattr(grads, name), getattr(expected, name)), (step, name)
        for t, name in zip(tensors[1:], ("W1", "weight", "bias", "W2")):
            t -= 0.1 * getattr(expected, name)


@pytest.mark.gpu
def test_evaluation_loss_on_the_device():
    from mask_b200.gcn import cost_prefix_on_device
    m, (X, W1, _, _, W2), labels = _problem(1024, 64, 64, 100, 7, "cuda", torch.float32)
    net = FusedGCN2(m, 0, 1, torch.device("cuda"), cost_prefix_on_device(m, "cuda"), hidden=64)
    out = net.forward(X, W1, W2).double()
    want = torch.nn.functional.cross_entropy(out[labels >= 0], labels[labels >= 0])
    # both take the same sparse products; the dense one is torch's in float32
    assert abs(float(net.loss(X, W1, W2, labels)) - float(want)) < 1e-4 * float(want)
    net.close()


def _loss_rank(rank, world, port, shared, q):
    import os

    import torch.distributed as dist
    from tests.test_sharding import _CpuFusedOps
    os.environ["MASTER_ADDR"], os.environ["MASTER_PORT"] = "127.0.0.1", str(port)
    dist.init_process_group("gloo", rank=rank, world_size=world)
    try:
        import oracle
        from mask_b200.sharding import spmm_cost_prefix
        m, (X, W1, _, _, W2), labels = _problem(512, 24, 16, 9, 8, dtype=torch.float32)
        prefix = spmm_cost_prefix(oracle.pack_srbcrs(m.M, m.rowptr, m.colind, m.values)["val_soff"])
        ops = _CpuFusedOps(rank, shared, 0.0)
        ops.linear_cross_entropy = PlainOps().linear_cross_entropy
        net = FusedGCN2(m, rank, world, torch.device("cpu"), prefix, hidden=16, ops=ops)
        q.put((rank, [float(net.loss(X * s, W1, W2, labels[net.r0:net.r1])) for s in (1.0, -2.0)]))
        net.close()
    finally:
        dist.destroy_process_group()


def test_evaluation_loss_over_two_ranks():
    """Every rank gets the mean over all ranks' labelled rows."""
    import torch.multiprocessing as mp
    from tests.test_sharding import _free_port
    m, (X, W1, _, _, W2), labels = _problem(512, 24, 16, 9, 8, dtype=torch.float32)
    A = _dense(m).float()
    shared = [[torch.full((m.M, 16), float("nan")).share_memory_() for _ in range(2)] for _ in range(2)]
    ctx = mp.get_context("spawn")
    q, port = ctx.Queue(), _free_port()
    procs = [ctx.Process(target=_loss_rank, args=(r, 2, port, shared, q)) for r in range(2)]
    for p in procs:
        p.start()
    got = dict(q.get(timeout=180) for _ in procs)
    for p in procs:
        p.join(timeout=60)
        assert p.exitcode == 0
    for i, s in enumerate((1.0, -2.0)):
        out = (A @ torch.relu(A @ (X * s @ W1))) @ W2
        want = float(torch.nn.functional.cross_entropy(out[labels >= 0], labels[labels >= 0]))
        assert got[0][i] == got[1][i] and abs(got[0][i] - want) < 1e-5 * want
