"""Layer norm, 8-bit checkpoints and the many-class loss as a training step uses them: through autograd, and through
``DistSAGE(checkpoint_bits=8, chunked_loss=True)``."""
import pytest
import torch
import torch.nn.functional as F

from super_gnn_b200 import fused_layer, graphsage, supergnn_ops as ops, synthetic
from super_gnn_b200.data_manager import build_distributed_graph
from super_gnn_b200.layers import functional as L

pytestmark = pytest.mark.gpu
DEV = "cuda"


def graph_of(n, e, width, seed=5):
    dev = torch.device(DEV)
    s, t = synthetic.rmat_edges(n, e, 0.57, 0.19, 0.19, 0.05, seed=seed, device=dev)
    s, t = synthetic.symmetrize_dedup(s, t, n)
    return build_distributed_graph(torch.stack([s, t]), torch.zeros((2, 0), dtype=torch.int64, device=dev), [0, n],
                                   width, 32, device=dev)


def near(a, b, tol):
    """Both sides in fp32 with sums in another order: within ``tol`` of the largest value."""
    return float((a - b).abs().max()) <= tol * float(b.abs().max()) + 1e-30


def test_functional_forms_are_the_formulas():
    gen = torch.Generator(device=DEV).manual_seed(2)
    x = torch.randn(3, 50, 36, generator=gen, device=DEV, requires_grad=True)
    w = torch.rand(36, generator=gen, device=DEV).add_(0.5).requires_grad_()
    b = torch.randn(36, generator=gen, device=DEV, requires_grad=True)
    g = torch.randn(3, 50, 36, generator=gen, device=DEV)
    want = torch.autograd.grad(F.layer_norm(x.double(), (36,), w.double(), b.double()), (x, w, b), g.double())
    got = torch.autograd.grad(L.layer_norm(x, w, b), (x, w, b), g)
    for a, c in zip(got, want):
        assert near(a, c, 2e-6)  # sums of 36 and of 150 terms
    # from the checkpoint: the same with the restored x in the place of x, mean and deviation those of x
    flat = x.detach().reshape(-1, 36)
    kept = ops.checkpoint_unpack_rows(*ops.checkpoint_pack_rows(flat)).double()
    mean = flat.double().mean(1, keepdim=True)
    rstd = (flat.double().var(1, unbiased=False, keepdim=True) + 1e-5).rsqrt()
    xh, gy = (kept - mean) * rstd, g.reshape(-1, 36).double()
    a8 = gy * w.double()
    want8 = rstd * (a8 - a8.mean(1, keepdim=True) - xh * (a8 * xh).mean(1, keepdim=True))
    y8 = L.layer_norm(x, w, b, checkpoint_bits=8)
    assert torch.equal(y8, L.layer_norm(x, w, b))
    got8 = torch.autograd.grad(y8, (x, w, b), g)
    assert near(got8[0].reshape(-1, 36), want8, 2e-6) and near(got8[1], (gy * xh).sum(0), 2e-6) and near(got8[2], gy.sum(0), 2e-6)
    # a linear map: the gradient of the weight is the restored input's
    lw = torch.randn(20, 36, generator=gen, device=DEV, requires_grad=True)
    gl = torch.randn(150, 20, generator=gen, device=DEV)
    xf = flat.clone().requires_grad_()
    y = L.linear(xf, lw, checkpoint_bits=8)
    assert torch.equal(y, F.linear(xf, lw))
    gx, gw = torch.autograd.grad(y, (xf, lw), gl)
    assert torch.equal(gx, gl @ lw)
    assert near(gw, gl.double().t() @ kept, 2 ** -19)  # 10 x 3 additions towards zero, 2^-24 each, and g sc
    assert L.linear(xf, lw, checkpoint_bits=8).grad_fn is not None
    for bits in (4, 16, None):
        with pytest.raises(ValueError):
            L.linear(xf, lw, checkpoint_bits=bits)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_many_class_loss_through_autograd(dtype):
    gen = torch.Generator(device=DEV).manual_seed(2)
    x = torch.randn(90, 24, generator=gen, device=DEV).to(dtype).requires_grad_()
    w = (torch.randn(700, 24, generator=gen, device=DEV) * 0.3).to(dtype).requires_grad_()
    b = torch.randn(700, generator=gen, device=DEV).to(dtype).requires_grad_()
    labels = torch.randint(0, 700, (90,), generator=gen, device=DEV)
    mask = torch.rand(90, generator=gen, device=DEV) < 0.6
    loss = L.linear_nll_loss(x, w, b, labels, mask, 0.1)
    grads = torch.autograd.grad(3.0 * loss, (x, w, b))
    logp = torch.log_softmax(F.linear(x.double(), w.double(), b.double()), 1)
    want = -(logp.gather(1, labels[:, None])[:, 0] * mask).sum() * 0.1
    expect = torch.autograd.grad(3.0 * want, (x, w, b))
    assert abs(float(loss) - float(want)) <= 1e-5 * float(want)
    # bf16: G and the result are rounded to 8 bits of significand; fp32: sums of 700 terms
    tol = 3 * 2 ** -8 if dtype == torch.bfloat16 else 1e-5
    for a, c in zip(grads, expect):
        assert a.dtype == dtype and near(a.float(), c.float(), tol)
    with torch.no_grad():
        assert torch.equal(L.linear_nll_loss(x, w, b, labels, mask, 0.1), loss)
    frozen = L.linear_nll_loss(x.detach(), w.detach().requires_grad_(), None, labels, mask, 0.1)
    frozen.backward()


def step(model, graph, x, labels, mask, masks):
    model.dropout_masks = masks
    model.train()
    for p in model.parameters():
        p.grad = None
    core = model
    if core.can_fuse_loss(x, graph):
        loss = model(graph, x, labels, None, loss_mask=mask, loss_inv_count=0.01, loss_unit_grad=True)
    else:
        out = model(graph, x)
        loss = F.nll_loss(out[mask], labels[mask], reduction="sum") * 0.01
    loss.backward()
    return loss.detach(), {k: p.grad.clone() for k, p in model.named_parameters()}


def models(fin, hid, ncls, **kw):
    torch.manual_seed(0)
    base, _ = graphsage.create_model_and_optimizer(
        dict(in_channels=fin, hidden_channels=hid, out_channels=ncls, num_layers=3, dropout=0.5), device=torch.device(DEV))
    other, _ = graphsage.create_model_and_optimizer(
        dict(in_channels=fin, hidden_channels=hid, out_channels=ncls, num_layers=3, dropout=0.5, **kw),
        device=torch.device(DEV))
    other.load_state_dict(base.state_dict())
    return base, other


@pytest.mark.parametrize("fin,hid,ncls,fold", [(100, 64, 7, True), (100, 64, 7, False), (30, 64, 9, True), (33, 50, 5, True)])
def test_model_with_8_bit_checkpoints(fin, hid, ncls, fold):
    """The loss does not change; the gradients are those of activations that are off by half a step of 255."""
    n = 4000
    graph = graph_of(n, 40_000, max(fin, hid))
    graph.set_fold_mean(fold)
    base, small = models(fin, hid, ncls, checkpoint_bits=8)
    x = torch.randn(n, fin, device=DEV)
    labels = torch.randint(0, ncls, (n,), device=DEV)
    mask = torch.rand(n, device=DEV) < 0.3
    masks = [(torch.rand(n, hid, device=DEV) >= 0.5).float() * 2 for _ in range(2)]
    loss, grads = step(base, graph, x, labels, mask, masks)
    loss8, grads8 = step(small, graph, x, labels, mask, masks)
    # the same forward twice: the SpMM finishes rows that a chunk cuts with atomic adds, in an order that varies, so sums of up
    # to a few hundred neighbours differ by a few hundred 2^-24 of their terms, here and in what follows from them
    assert abs(float(loss) - float(loss8)) <= 1e-5 * abs(float(loss))
    for k in grads:
        a, c = grads8[k].double(), grads[k].double()
        # every activation is off by at most 1/510 of its row's range (about six deviations): 0.7 % of a deviation, of random
        # sign; a unit whose normalised value is that near zero changes sides at the relu, one in a hundred
        assert float((a - c).norm()) <= 0.15 * float(c.norm()), k
        assert float((a * c).sum()) >= 0.98 * float(a.norm() * c.norm()), k
    # the last layer's weight gradients are G^T of the restored input: nothing but that quantisation lies between them
    for k in ("convs.2.lin_neigh.weight", "convs.2.lin_self.weight"):
        assert float((grads8[k] - grads[k]).norm()) <= 0.01 * float(grads[k].norm()), k
    assert near(grads8["convs.2.bias"], grads["convs.2.bias"], 8e-5)


def test_checkpoints_take_a_quarter_of_the_memory():
    n, fin, hid, ncls = 200_000, 128, 256, 16
    graph = graph_of(n, 400_000, hid)
    graph.set_fold_mean(True)
    x = torch.randn(n, fin, device=DEV)
    labels = torch.randint(0, ncls, (n,), device=DEV)
    mask = torch.ones(n, dtype=torch.bool, device=DEV)
    held = {}
    for bits, model in zip((32, 8), models(fin, hid, ncls, checkpoint_bits=8)):
        model.train()
        model(graph, x, labels, None, loss_mask=mask, loss_inv_count=0.01, loss_unit_grad=True).backward()
        torch.cuda.synchronize()
        before = torch.cuda.memory_allocated()
        loss = model(graph, x, labels, None, loss_mask=mask, loss_inv_count=0.01, loss_unit_grad=True)
        torch.cuda.synchronize()
        held[bits] = torch.cuda.memory_allocated() - before
        loss.backward()
    # kept in fp32 / in 8 bits: h of two layers, agg of the first, [agg | x] of the second, x of the third
    elements = n * (2 * hid + fin + 2 * hid + hid)
    assert held[32] >= 4 * elements
    assert held[8] <= elements + n * (8 * 6 + 4 * 4 * 4) + n * 4 * 2 * ncls + (8 << 20)


@pytest.mark.parametrize("fin,hid,ncls,fold,fused", [(64, 64, 300, True, True), (30, 50, 1000, False, True), (32, 48, 261, True, False),
                                                     (20, 30, 9, True, True)])
def test_model_with_the_chunked_loss(fin, hid, ncls, fold, fused):
    n = 3000
    graph = graph_of(n, 30_000, max(fin, hid))
    graph.set_fold_mean(fold)
    base, chunked = models(fin, hid, ncls, chunked_loss=True)
    base.fused = chunked.fused = fused
    x = torch.randn(n, fin, device=DEV)
    labels = torch.randint(0, ncls, (n,), device=DEV)
    mask = torch.rand(n, device=DEV) < 0.3
    masks = [(torch.rand(n, hid, device=DEV) >= 0.5).float() * 2 for _ in range(2)]
    loss, grads = step(base, graph, x, labels, mask, masks)
    loss2, grads2 = step(chunked, graph, x, labels, mask, masks)
    assert abs(float(loss) - float(loss2)) <= 1e-5 * abs(float(loss))
    for k in grads:  # two fp32 computations of the same sums
        assert near(grads2[k], grads[k], 8e-5), k
    with torch.no_grad():
        chunked.eval()
        base.eval()
        value = chunked(graph, x, labels, None, loss_mask=mask, loss_inv_count=0.01)
        want = F.nll_loss(base(graph, x)[mask], labels[mask], reduction="sum") * 0.01
    assert abs(float(value) - float(want)) <= 1e-5 * abs(float(want))


def test_all_of_them_in_a_training_step():
    """Training steps with 8-bit checkpoints and the chunked loss run, and the gradient is the slope of the loss."""
    n, fin, hid, ncls = 5000, 64, 128, 500
    graph = graph_of(n, 50_000, hid)
    torch.manual_seed(1)
    model, opt = graphsage.create_model_and_optimizer(
        dict(in_channels=fin, hidden_channels=hid, out_channels=ncls, num_layers=3, dropout=0.0, checkpoint_bits=8,
             chunked_loss=True), device=torch.device(DEV))
    data = dict(graph=graph, nodes_features=torch.randn(n, fin, device=DEV),
                nodes_labels=torch.randint(0, ncls, (n,), device=DEV),
                nodes_train_masks=torch.rand(n, device=DEV) < 0.5)
    count = float(data["nodes_train_masks"].sum())
    first = graphsage.train_step(model, data, opt, count)
    for _ in range(3):
        loss = graphsage.train_step(model, data, opt, count)
        assert torch.isfinite(loss)
    # the loss through the gradient: a small step against it lowers the loss by step |grad|^2
    model.zero_grad()
    args = (graph, data["nodes_features"], data["nodes_labels"], None)
    kw = dict(loss_mask=data["nodes_train_masks"], loss_inv_count=1.0 / count)
    model.eval()
    before = model(*args, **kw)
    before.backward()
    square = sum(float(p.grad.double().square().sum()) for p in model.parameters())
    rate = 1e-3 * float(before) / square
    with torch.no_grad():
        for p in model.parameters():
            p -= rate * p.grad
        after = model(*args, **kw)
    drop = float(before) - float(after)
    assert 0.5 * rate * square <= drop <= 2.0 * rate * square and first.dim() == 0


def test_second_backward_pass_of_the_chunked_loss():
    n, fin, hid, ncls = 600, 20, 32, 300
    graph = graph_of(n, 6000, hid)
    _, model = models(fin, hid, ncls, chunked_loss=True)
    model.dropout = 0.0
    x = torch.randn(n, fin, device=DEV)
    labels = torch.randint(0, ncls, (n,), device=DEV)
    for unit in (True, False):
        model.zero_grad()
        conv = model.convs[-1]
        h = torch.randn(n, hid, device=DEV, requires_grad=True)
        loss = graphsage.FusedSAGELossManyClasses.apply(h, conv.lin_neigh.weight, conv.lin_self.weight, conv.bias, graph, 2, 32,
                                                        False, True, labels, None, 0.01, unit)
        first = torch.autograd.grad(loss, (h, conv.lin_self.weight), retain_graph=True)
        again = torch.autograd.grad(loss, (h, conv.lin_self.weight))
        for a, c in zip(first, again):
            assert torch.equal(a, c)


def kinds_of(call):
    """Entry points that a call launched."""
    ops.LAUNCH_LOG = []
    try:
        call()
        return {entry[0] for entry in ops.LAUNCH_LOG}
    finally:
        ops.LAUNCH_LOG = None


@pytest.mark.parametrize("fused,hid", [(True, 64), (True, 50), (False, 64)])
def test_an_evaluation_packs_nothing_and_computes_no_gradients(fused, hid):
    n, fin, ncls = 2000, 30, 300
    graph = graph_of(n, 20_000, hid)
    _, model = models(fin, hid, ncls, checkpoint_bits=8, chunked_loss=True)
    _, plain = models(fin, hid, ncls)
    model.fused = plain.fused = fused
    x, labels = torch.randn(n, fin, device=DEV), torch.randint(0, ncls, (n,), device=DEV)
    mask = torch.rand(n, device=DEV) < 0.3
    args, kw = (graph, x, labels, None), dict(loss_mask=mask, loss_inv_count=0.01)
    model.eval(), plain.eval()
    got = {}

    def evaluate():
        with torch.no_grad():
            got["loss"], got["out"] = model(*args, **kw), model(graph, x)

    assert kinds_of(evaluate).isdisjoint({"checkpoint_pack", "linear_nll_grad"})
    assert {"checkpoint_pack", "linear_nll_grad"} <= kinds_of(lambda: model(*args, **kw))
    with torch.no_grad():
        out = plain(graph, x)
    # the same forward through other kernels: sums of up to a few hundred neighbours in another order, 2^-24 each, in three layers
    assert float((got["out"] - out).abs().max()) <= 1e-4 * float(out.abs().max())
    want = F.nll_loss(out[mask], labels[mask], reduction="sum") * 0.01
    assert abs(float(got["loss"]) - float(want)) <= 1e-5 * float(want)


def test_functional_forms_without_a_backward_pass(monkeypatch):
    gen = torch.Generator(device=DEV).manual_seed(2)
    x = torch.randn(70, 36, generator=gen, device=DEV)
    w, lw = torch.nn.Parameter(torch.rand(36, device=DEV)), torch.nn.Parameter(torch.rand(300, 36, device=DEV))
    labels = torch.randint(0, 300, (70,), device=DEV)
    packed = []
    forward = ops.layer_norm_forward
    monkeypatch.setattr(ops, "layer_norm_forward",
                        lambda *a, **k: (packed.append(k.get("checkpoint", False)), forward(*a, **k))[1])

    def calls(weight, last):
        return (L.layer_norm(x, weight, checkpoint_bits=8), L.linear(x, last, checkpoint_bits=8),
                L.linear_nll_loss(x, last, None, labels, None, 0.1))

    want = calls(w, lw)
    assert packed == [True] and all(y.requires_grad for y in want)

    def quiet():
        with torch.no_grad():
            return calls(w, lw)

    for run in (quiet, lambda: calls(w.detach(), lw.detach())):
        packed.clear()
        got = []
        assert kinds_of(lambda: got.extend(run())) == {"layer_norm_fwd", "linear_nll"} and packed == [False]
        for a, b in zip(got, want):
            assert torch.equal(a, b) and not a.requires_grad
    # memory: neither gradients nor codes beside the result
    big = torch.randn(20_000, 36, device=DEV)
    torch.cuda.synchronize()
    with torch.no_grad():
        before = torch.cuda.memory_allocated()
        y = L.layer_norm(big, w, checkpoint_bits=8)
        assert torch.cuda.memory_allocated() - before <= y.numel() * 4 + 1024


def test_the_loss_alone_takes_the_exchange_of_the_mode(monkeypatch):
    """A model in training mode quantises the rows it exchanges, whether or not gradients are on."""
    n, fin, hid, ncls = 500, 20, 32, 300
    graph = graph_of(n, 5000, hid)
    _, model = models(fin, hid, ncls, chunked_loss=True)
    x, labels = torch.randn(n, fin, device=DEV), torch.randint(0, ncls, (n,), device=DEV)
    mask = torch.ones(n, dtype=torch.bool, device=DEV)
    seen = []
    inner = fused_layer.aggregate_forward

    def forward(ctx, graph, x, layer, num_bits, is_pre_delay, is_training, **kw):
        seen.append((layer, is_training))
        return inner(ctx, graph, x, layer, num_bits, is_pre_delay, is_training, **kw)

    monkeypatch.setattr(fused_layer, "aggregate_forward", forward)
    for training in (True, False):
        model.train(training)
        for grad in (True, False):
            seen.clear()
            with torch.set_grad_enabled(grad):
                model(graph, x, labels, None, loss_mask=mask, loss_inv_count=0.01)
            assert seen == [(0, training), (1, training), (2, training)], (training, grad, seen)


@pytest.mark.parametrize("unit", [True, False])
def test_gradients_of_several_backward_passes_add_up(unit):
    """What the loss keeps for its backward pass is not handed out as somebody's gradient to add to."""
    n, hid, ncls = 600, 32, 300
    graph = graph_of(n, 6000, hid)
    _, model = models(20, hid, ncls, chunked_loss=True)
    labels = torch.randint(0, ncls, (n,), device=DEV)
    conv = model.convs[-1]
    h = torch.randn(n, hid, device=DEV, requires_grad=True)
    loss = graphsage.FusedSAGELossManyClasses.apply(h, conv.lin_neigh.weight, conv.lin_self.weight, conv.bias, graph, 2, 32,
                                                    False, True, labels, None, 0.01, unit)
    leaves = (h, conv.lin_neigh.weight, conv.lin_self.weight, conv.bias)
    first = [g.clone() for g in torch.autograd.grad(loss, leaves, retain_graph=True)]
    for turn in range(1, 5):
        loss.backward(retain_graph=True)
        for leaf, g in zip(leaves, first):
            # sums of equal fp32 numbers: up to three roundings; h: an SpMM whose atomic adds come in any order
            assert near(leaf.grad, turn * g, 1e-5)


def test_features_are_not_packed_where_layers_are_not_fused():
    """The first layer's own input stays with the caller; everything between the layers is kept in 8 bits."""
    n, fin, hid, ncls = 1500, 30, 50, 6
    graph = graph_of(n, 9000, hid)
    base, small = models(fin, hid, ncls, checkpoint_bits=8)
    base.fused = small.fused = False
    base.dropout = small.dropout = 0.0
    x = torch.randn(n, fin, device=DEV)
    ops.LAUNCH_LOG = []
    try:
        out = small(graph, x)
        packs = [entry[1]["F"] for entry in ops.LAUNCH_LOG if entry[0] == "checkpoint_pack"]
    finally:
        ops.LAUNCH_LOG = None
    assert packs == [fin, hid, hid, hid, hid]  # aggregated features; (aggregated | own) of the two layers behind
    out.square().sum().backward()
    base(graph, x).square().sum().backward()
    for (k, a), b in zip(small.named_parameters(), base.parameters()):
        assert float((a.grad - b.grad).norm()) <= 0.15 * float(b.grad.norm()), k  # as in test_model_with_8_bit_checkpoints


def test_layers_wider_than_the_kernels_take():
    """Beyond 65536 columns a weight gradient is taken in parts; a layer norm beyond 16384 keeps its input; the loss in pieces is
    not offered beyond 8192 channels into the last layer.  None of them fails, at the first backward pass least of all."""
    n = 40
    graph = graph_of(n, 300, 16400)
    for fin, hid, ncls in ((70_000, 8, 3), (10, 16_400, 3), (10, 8, 70_001)):
        base, small = models(fin, hid, ncls, checkpoint_bits=8, chunked_loss=True)
        base.dropout = small.dropout = 0.0
        assert small.can_fuse_loss(torch.empty(n, fin, device=DEV), graph) == (hid <= 8192)
        x = torch.randn(n, fin, device=DEV)
        labels, mask = torch.randint(0, ncls, (n,), device=DEV), torch.ones(n, dtype=torch.bool, device=DEV)
        loss, grads = step(base, graph, x, labels, mask, None)
        loss8, grads8 = step(small, graph, x, labels, mask, None)
        assert abs(float(loss) - float(loss8)) <= 1e-4 * abs(float(loss))
        # With 40 nodes a few of the hundreds of units change sides at a relu (one in a hundred does), and each of them is a visible
        # part of the gradients before it, bias sums above all: no bound there but that they are numbers.  Between the loss
        # and the last layer's weights lies nothing but the quantisation of its input, as in test_model_with_8_bit_checkpoints.
        assert all(torch.isfinite(g).all() for g in grads8.values())
        for k in ("convs.2.lin_neigh.weight", "convs.2.lin_self.weight"):
            assert float((grads8[k] - grads[k]).norm()) <= 0.01 * float(grads[k].norm()), (fin, hid, ncls, k)


def test_weight_gradients_in_parts_are_those_in_one(monkeypatch):
    x, g = torch.randn(900, 500, device=DEV), torch.randn(900, 300, device=DEV)
    kept = ops.checkpoint_pack_rows(x)
    whole = ops.checkpoint_weight_grad(g, *kept)
    out = torch.randn(300, 507, device=DEV)[:, 3:503]
    want = whole + 0.5 * out
    monkeypatch.setattr(ops, "_MOST_COLUMNS", 64)
    # other row ranges: sums of 900 rows in another order
    assert near(ops.checkpoint_weight_grad(g, *kept), whole, 2 ** -19)
    assert ops.checkpoint_weight_grad(g, *kept, out=out, beta=0.5) is out and near(out, want, 2 ** -19)
