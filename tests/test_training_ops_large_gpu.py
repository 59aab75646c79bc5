"""Layer norm, checkpoints and the many-class loss on operands of more than 2^31 elements: the ends of the big operands
against the same rows alone."""
import pytest
import torch

from super_gnn_b200 import supergnn_ops as ops

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _need_memory(gb):
    free, _ = torch.cuda.mem_get_info()
    if free < gb * (1 << 30):
        pytest.skip(f"needs {gb} GB of free device memory")


@pytest.mark.parametrize("H", [520, 521])  # aligned rows, and rows through the ring
def test_layer_norm_and_checkpoint_rows_beyond_2_31_elements(H):
    _need_memory(40)
    n = (1 << 22) + 5
    x = torch.empty(n, H, dtype=torch.bfloat16, device=DEV)
    x.normal_()
    ends = torch.cat([torch.arange(9), torch.arange(n - 13, n)]).to(DEV)
    part = x[ends].contiguous()
    gamma, beta = torch.rand(H, device=DEV), torch.rand(H, device=DEV)
    y, stats, codes, params = ops.layer_norm_forward(x, gamma, beta, checkpoint=True)
    want = ops.layer_norm_forward(part, gamma, beta, checkpoint=True)
    plain = ops.layer_norm_forward(x, gamma, beta)[0]
    # the row sums of the variants are taken in another order: one step of bf16 where a value lies next to a border
    assert float((plain[ends].float() - want[0].float()).abs().max()) <= 2 ** -7 * float(want[0].float().abs().max())
    del plain
    for a, b in zip((y[ends], codes[ends], params[ends]), (want[0], want[2], want[3])):
        assert torch.equal(a, b)
    del y
    back = ops.checkpoint_unpack_rows(codes, params, torch.bfloat16)
    assert torch.equal(back[ends], ops.checkpoint_unpack_rows(want[2], want[3], torch.bfloat16))
    del back
    # gradients: nothing but the ends has one
    gy = torch.zeros_like(x)
    gy[ends] = torch.randn(len(ends), H, device=DEV).to(torch.bfloat16)
    gx, gg, gb = ops.layer_norm_backward(gy, x, stats, gamma)
    sx, sg, sb = ops.layer_norm_backward(gy[ends].contiguous(), part, stats[ends].contiguous(), gamma)
    assert float((gx[ends].float() - sx.float()).abs().max()) <= 2 ** -7 * float(sx.float().abs().max())
    # 22 terms a column, fp32
    assert float((gg - sg).abs().max()) <= 1e-5 * float(sg.abs().max()) and float((gb - sb).abs().max()) <= 1e-5 * float(sb.abs().max())
    del gx
    g = torch.zeros(n, 4, device=DEV)
    g[ends] = torch.randn(len(ends), 4, device=DEV)
    got, alone = ops.checkpoint_weight_grad(g, codes, params), ops.checkpoint_weight_grad(g[ends].contiguous(), want[2], want[3])
    # the same 22 terms, g sc in two bf16 terms each
    assert float((got - alone).abs().max()) <= 2 ** -16 * float(alone.abs().max())


def test_many_class_loss_with_weights_beyond_2_31_elements():
    _need_memory(60)
    n, K, C = 8, 520, (1 << 22) + 77
    w = torch.empty(C, K, dtype=torch.bfloat16, device=DEV)
    w.normal_(std=0.05)
    x = torch.randn(n, K, device=DEV).to(torch.bfloat16)
    labels = torch.tensor([0, 1, C - 1, C - 2, C // 2, 5, C - 77, -1], device=DEV)
    loss, lse = ops.linear_nll_loss(x, w, None, labels, None, 1.0)
    z = torch.cat([x.double() @ w[i:i + (1 << 20)].double().t() for i in range(0, C, 1 << 20)], 1)
    want = torch.logsumexp(z, 1)
    # K-term fp32 sums in a tensor core, and a sum of 4 M exponentials in a tree of pieces
    assert float((lse[:7].double() - want[:7]).abs().max()) <= 1e-4 and lse[7] == 0
    expect = (want[:7] - z[torch.arange(7), labels[:7]]).sum()
    assert abs(float(loss) - float(expect)) <= 1e-5 * abs(float(expect))
    _, gx, gw, _ = ops.linear_nll_loss_grad(x, w, None, labels, None, 1.0)
    at = torch.tensor([0, C - 1, C - 2, C // 2, C - 3], device=DEV)
    p = (z[:7, at] - want[:7, None]).exp() - (at[None, :] == labels[:7, None]).double()
    rows = p.t() @ x[:7].double()
    # G and the result in bf16
    assert float((gw[at].double() - rows).abs().max()) <= 2 ** -6 * float(rows.abs().max())
    assert not gx[7].any()


def test_weight_gradient_of_rows_beyond_2_31_elements_keeps_all_terms():
    """22 rows at both ends have a gradient: against the formula in 64 bits, at the accuracy of three terms of g sc."""
    _need_memory(20)
    n, F, M = (1 << 22) + 5, 520, 12
    x = torch.empty(n, F, dtype=torch.bfloat16, device=DEV)
    x.normal_()
    ends = torch.cat([torch.arange(9), torch.arange(n - 13, n)]).to(DEV)
    codes, params = ops.checkpoint_pack_rows(x)
    del x
    g = torch.zeros(n, M, device=DEV)
    g[ends] = torch.randn(len(ends), M, device=DEV)
    got = ops.checkpoint_weight_grad(g, codes, params)
    zp, sc, c = params[ends, :1].double(), params[ends, 1:].double(), codes[ends].double()
    ge = g[ends].double()
    want = ge.t() @ (zp + sc * c)
    typical = (ge.square().t() @ (sc * c + zp.abs()).square()).sqrt()
    # 2^-23 of each value for g sc in three terms (two would leave 2^-18), 2^-24 on average at each of the three additions for
    # sixteen rows, of which there are at most four at the ends; the rows between add zeros, which is exact; joining two row
    # ranges and adding the zero points' share a few roundings more
    assert (got.double() - want).norm() <= (2 ** -23 + (3 * 4 + 6) * 2 ** -24) * typical.norm()


def test_many_class_loss_of_a_whole_partition():
    """A few rows of very many are in the loss, as a model has it that hands over all of its nodes: what the same rows give alone."""
    _need_memory(20)
    n, K, C = 400_000, 256, 1000
    gen = torch.Generator(device=DEV).manual_seed(7)
    x = torch.randn(n, K, generator=gen, device=DEV)
    w = torch.randn(C, K, generator=gen, device=DEV) * (2 / K ** 0.5)
    b = torch.randn(C, generator=gen, device=DEV)
    labels = torch.randint(0, C, (n,), generator=gen, device=DEV)
    mask = torch.rand(n, generator=gen, device=DEV) < 0.08
    rows = mask.nonzero()[:, 0]
    inv = 1.0 / len(rows)
    loss, gx, gw, gb = ops.linear_nll_loss_grad(x, w, b, labels, mask, inv)
    want = ops.linear_nll_loss_grad(x[rows], w, b, labels[rows], None, inv)
    # the same products in other chunks of rows: each side is within 2^-20 of the formula
    for a, c in ((loss, want[0]), (gx[rows], want[1]), (gw, want[2]), (gb, want[3])):
        assert float((a - c).norm()) <= 2 * 2.0 ** -20 * float(c.norm())
    gx[rows] = 0
    assert not gx.any()
    value, lse = ops.linear_nll_loss(x, w, b, labels, mask, inv)
    assert torch.equal(value, loss) and not lse[~mask].any()
