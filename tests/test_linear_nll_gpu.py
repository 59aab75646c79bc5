"""The many-class loss of a linear classifier and its gradients against the formulas in 64 bits."""
import pytest
import torch

from super_gnn_b200 import supergnn_ops as ops

pytestmark = pytest.mark.gpu
DEV = "cuda"
STEP = 2.0 ** -23


def make(n, K, C, dtype, seed, bdtype=None, scale=2.0, on=0.7):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    x = torch.randn(n, K, generator=gen, device=DEV).to(dtype)
    w = (torch.randn(C, K, generator=gen, device=DEV) * (scale / K ** 0.5)).to(dtype)
    b = (torch.randn(C, generator=gen, device=DEV) * 0.5).to(bdtype or dtype)
    labels = torch.randint(0, C, (n,), generator=gen, device=DEV)
    mask = torch.rand(n, generator=gen, device=DEV) < on
    return x, w, b, labels, mask


class Ref:
    """The formulas in 64 bits, and bounds.

    A logit is a sum of K products of which each is off by at most a step 2^-23 of itself (fp32 operands are carried in
    22 bits or more; bf16 products are exact), every addition by 2^-23 of the magnitudes:
        e_z = (K + 16) 2^-23 (sum |x w| + |b|).
    lse moves by at most max_c e_z, and the sum of C exponentials in a tree of pieces adds (300 + C / 256) 2^-23.  p is
    then off by p (2 e_z + ...), G is rounded to the operand type (bf16: 2^-8 of it, fp32: 2^-20), and the two products are
    sums of C (gx) and m (gw) terms."""

    def __init__(self, x, w, b, labels, mask, inv):
        n, K = x.shape
        C = w.size(0)
        on = (labels >= 0) & (labels < C)
        if mask is not None:
            on &= mask.bool()
        self.rows = on.nonzero()[:, 0]
        dtype = x.dtype
        xr, w = x[self.rows].double(), w.double()
        b = torch.zeros(C, dtype=torch.float64, device=DEV) if b is None else b.double()
        lab = labels[self.rows]
        z = xr @ w.t() + b
        at = torch.arange(len(lab), device=DEV)
        finite_b = torch.where(torch.isfinite(b), b, torch.zeros_like(b))
        e_z = (K + 16) * STEP * (xr.abs() @ w.abs().t() + finite_b.abs())
        lse = torch.logsumexp(z, 1)
        e_lse = e_z.amax(1) + (300 + C / 256) * STEP + 2 * STEP * lse.abs()
        self.lse, self.e_lse = torch.zeros(n, dtype=torch.float64, device=DEV), torch.zeros(n, dtype=torch.float64, device=DEV)
        self.lse[self.rows], self.e_lse[self.rows] = lse, e_lse
        terms = lse - z[at, lab]
        self.loss = terms.sum() * inv
        self.e_loss = abs(inv) * ((e_lse + e_z[at, lab]).sum() + (len(lab) + 8) * STEP * terms.abs().sum())
        p = (z - lse[:, None]).exp()
        g = p.clone()
        g[at, lab] -= 1
        e_g = p * (e_z + e_lse[:, None] + 8 * STEP) * 1.01 + g.abs() * (2 ** -8 if dtype == torch.bfloat16 else 2 ** -20)
        e_g += 2.0 ** -38  # the smallest steps of a stored probability
        m = max(1, len(lab))
        self.gx, self.e_gx = torch.zeros(n, K, dtype=torch.float64, device=DEV), torch.zeros(n, K, dtype=torch.float64, device=DEV)
        self.gx[self.rows] = inv * (g @ w)
        self.e_gx[self.rows] = abs(inv) * (e_g @ w.abs() + (C + 16) * STEP * (g.abs() @ w.abs()))
        self.gw, self.e_gw = inv * (g.t() @ xr), abs(inv) * (e_g.t() @ xr.abs() + (m + 16) * STEP * (g.abs().t() @ xr.abs()))
        self.gb, self.e_gb = inv * g.sum(0), abs(inv) * (e_g.sum(0) + (m + 16) * STEP * g.abs().sum(0))


def close(got, want, err):
    off, bound = (got.double() - want).abs(), err + want.abs() * (torch.finfo(got.dtype).eps / 2) + 1e-37
    assert torch.isfinite(got).all()
    bad = off > bound
    assert not bad.any(), (off[bad][:4], bound[bad][:4], int(bad.sum()), tuple(got.shape))


def check(x, w, b, labels, mask, inv):
    ref = Ref(x, w, b, labels, mask, inv)
    loss, lse = ops.linear_nll_loss(x, w, b, labels, mask, inv)
    close(loss, ref.loss.reshape(1), ref.e_loss)
    close(lse, ref.lse, ref.e_lse)
    off = torch.ones(len(labels), dtype=torch.bool, device=DEV)
    off[ref.rows] = False
    assert (lse[off] == 0).all()
    loss2, gx, gw, gb = ops.linear_nll_loss_grad(x, w, b, labels, mask, inv)
    assert torch.equal(loss, loss2)
    assert gx.dtype == x.dtype and gw.dtype == w.dtype and (b is None) == (gb is None)
    close(gx, ref.gx, ref.e_gx)
    close(gw, ref.gw, ref.e_gw)
    assert (gx[off] == 0).all()
    if b is not None:
        assert gb.dtype == b.dtype
        close(gb, ref.gb, ref.e_gb)
    return loss, gx, gw, gb


@pytest.mark.parametrize("n,K,C", [(1, 1, 1), (1, 1, 2), (1, 8, 300), (2, 3, 5), (5, 64, 256), (127, 100, 257), (128, 64, 512),
                                   (129, 65, 511), (64, 256, 4099), (300, 130, 1000), (700, 602, 333), (2100, 20, 1025),
                                   (31, 1030, 700), (1000, 512, 3001)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_loss_and_gradients(n, K, C, dtype):
    check(*make(n, K, C, dtype, n + K + C), 1.0 / n)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_long_row_lists_and_several_pieces(dtype):
    """More rows than a listing block looks at, and more classes than a piece holds."""
    check(*make(5000, 16, 20_000, dtype, 3), 0.01)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_masks_and_labels(dtype):
    x, w, b, labels, mask = make(400, 40, 300, dtype, 9)
    labels[::7] = -1
    labels[3::11] = 300
    check(x, w, b, labels, mask, 0.5)
    check(x, w, b, labels, None, 0.5)
    check(x, w, None, labels, mask.to(torch.uint8), -2.0)
    check(x, w, b.float(), labels, mask, 0.5)
    block = torch.zeros_like(mask)
    block[130:140] = True  # only rows of the second tile
    check(x, w, b, labels, block, 0.5)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_nothing_in_the_loss(dtype):
    x, w, b, labels, mask = make(50, 40, 300, dtype, 9)
    for lab, m in ((labels, torch.zeros_like(mask)), (torch.full_like(labels, -1), None)):
        loss, gx, gw, gb = ops.linear_nll_loss_grad(x, w, b, lab, m, 1.0)
        assert loss.item() == 0 and not gx.any() and not gw.any() and not gb.any()
        assert not ops.linear_nll_loss(x, w, b, lab, m, 1.0)[1].any()
    loss, gx, gw, gb = ops.linear_nll_loss_grad(x[:0], w, b, labels[:0], None, 1.0)
    assert loss.item() == 0 and gx.shape == (0, 40) and not gw.any() and not gb.any()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_rows_outside_the_loss_may_hold_anything(dtype):
    x, w, b, labels, mask = make(300, 40, 500, dtype, 4)
    clean = ops.linear_nll_loss_grad(x, w, b, labels, mask, 0.1)
    x = x.clone()
    x[~mask] = float("nan")
    x[(~mask).nonzero()[0]] = float("inf")
    labels = torch.where(mask, labels, torch.full_like(labels, 1 << 40))
    for a, c in zip(ops.linear_nll_loss_grad(x, w, b, labels, mask, 0.1), clean):
        assert torch.equal(a, c)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_classes_that_a_bias_rules_out(dtype):
    x, w, b, labels, mask = make(200, 40, 700, dtype, 4, bdtype=torch.float32)
    b[256:512] = float("-inf")
    b[5] = torch.finfo(torch.float32).min
    labels = labels % 250 + 6  # none of them a label
    loss, gx, gw, gb = check(x, w, b, labels, mask, 0.1)
    assert not gw[256:512].any() and not gb[256:512].any() and not gb[5].any()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_large_logits_and_rows_of_very_different_size(dtype):
    x, w, b, labels, mask = make(200, 64, 400, dtype, 4, scale=40.0)
    x = (x.float() * torch.exp2(torch.randint(-6, 3, (200, 1), device=DEV).float())).to(dtype)
    check(x, w, b, labels, mask, 0.1)


def test_features_of_very_different_size():
    """Columns 2^30 apart: the gradient of each column keeps its own accuracy."""
    x, w, b, labels, mask = make(200, 64, 400, torch.float32, 4)
    s = torch.exp2(torch.linspace(-30, 0, 64, device=DEV).round())
    check(x * s, w / s.clamp(min=2.0 ** -10), b, labels, mask, 0.1)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("pad,offset", [(8, 0), (1, 0), (0, 1), (5, 3)])
def test_strides_and_alignment(dtype, pad, offset):
    x, w, b, labels, mask = make(150, 48, 600, dtype, 4)
    want = ops.linear_nll_loss_grad(x, w, b, labels, mask, 0.1)

    def inside(t):
        wide = torch.full((t.size(0), t.size(1) + pad + offset), float("nan"), dtype=dtype, device=DEV)
        wide[:, offset:offset + t.size(1)] = t
        return wide[:, offset:offset + t.size(1)]

    for xx, ww in ((inside(x), w), (x, inside(w)), (x.t().contiguous().t(), w.t().contiguous().t())):
        for a, c in zip(ops.linear_nll_loss_grad(xx, ww, b, labels, mask, 0.1), want):
            assert torch.equal(a, c)


def test_broadcast_input():
    _, w, b, labels, _ = make(20, 48, 300, torch.float32, 4)
    row = torch.randn(1, 48, device=DEV)
    check(row.expand(20, 48), w, b, labels, None, 0.1)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_repeatable(dtype):
    args = make(1500, 130, 3000, dtype, 4)
    first = ops.linear_nll_loss_grad(*args, 0.01)
    for _ in range(3):
        for a, c in zip(ops.linear_nll_loss_grad(*args, 0.01), first):
            assert torch.equal(a, c)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_captured_and_on_another_stream(dtype):
    """A captured call sees the inputs of the replay, next to calls of another size on another stream."""
    x, w, b, labels, mask = make(260, 72, 900, dtype, 4)
    other = make(90, 40, 400, dtype, 5)
    want_other = ops.linear_nll_loss_grad(*other, 0.1)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        ops.linear_nll_loss_grad(x, w, b, labels, mask, 0.1)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = ops.linear_nll_loss_grad(x, w, b, labels, mask, 0.1)
    for seed in (6, 7):
        new = make(260, 72, 900, dtype, seed)
        for t, v in zip((x, w, b, labels, mask), new):
            t.copy_(v)
        torch.cuda.synchronize()
        with torch.cuda.stream(side):
            others = [ops.linear_nll_loss_grad(*other, 0.1) for _ in range(3)]
        graph.replay()
        torch.cuda.synchronize()
        want = ops.linear_nll_loss_grad(*new, 0.1)
        for a, c in zip(got, want):
            assert torch.equal(a, c)
        for o in others:
            for a, c in zip(o, want_other):
                assert torch.equal(a, c)


def test_gradient_against_differences():
    x, w, b, labels, mask = make(12, 10, 40, torch.float32, 4)
    _, *grads = ops.linear_nll_loss_grad(x, w, b, labels, mask, 0.25)
    gen = torch.Generator(device=DEV).manual_seed(1)
    base = [x.double(), w.double(), b.double()]

    def value(xx, ww, bb):
        logp = torch.log_softmax(xx @ ww.t() + bb, 1)
        return float(-(logp.gather(1, labels[:, None])[:, 0] * mask).sum() * 0.25)

    for at, grad in enumerate(grads):
        v = torch.randn(base[at].shape, generator=gen, device=DEV, dtype=torch.float64)
        up, down = list(base), list(base)
        up[at], down[at] = base[at] + 1e-5 * v, base[at] - 1e-5 * v
        want = (value(*up) - value(*down)) / 2e-5
        # truncation 1e-10 of the third derivative, fp32 gradients
        assert abs(float((grad.double() * v).sum()) - want) <= 1e-5 * float((grad.double() * v).abs().sum())


@pytest.mark.parametrize("call", [
    lambda x, w, b, l, m: ops.linear_nll_loss(x.half(), w.half(), None, l, m, 1.0),
    lambda x, w, b, l, m: ops.linear_nll_loss(x, w.bfloat16(), b, l, m, 1.0),
    lambda x, w, b, l, m: ops.linear_nll_loss(x, w[:, :-1], b, l, m, 1.0),
    lambda x, w, b, l, m: ops.linear_nll_loss(x, w, b[:-1], l, m, 1.0),
    lambda x, w, b, l, m: ops.linear_nll_loss(x, w, b.double(), l, m, 1.0),
    lambda x, w, b, l, m: ops.linear_nll_loss(x, w, b, l.int(), m, 1.0),
    lambda x, w, b, l, m: ops.linear_nll_loss(x, w, b, l[:-1], m, 1.0),
    lambda x, w, b, l, m: ops.linear_nll_loss(x, w, b, l, m[:-1], 1.0),
    lambda x, w, b, l, m: ops.linear_nll_loss(x, w, b, l, m.float(), 1.0),
    lambda x, w, b, l, m: ops.linear_nll_loss(x, w, b, l, m, float("nan")),
    lambda x, w, b, l, m: ops.linear_nll_loss(x.cpu(), w, b, l, m, 1.0),
    lambda x, w, b, l, m: ops.linear_nll_loss(x, w[:0], None, l, m, 1.0),
    lambda x, w, b, l, m: ops.linear_nll_loss_grad(torch.empty(8, 16385, device=DEV), torch.empty(9, 16385, device=DEV), None,
                                                   l, m, 1.0),
])
def test_refusals(call):
    with pytest.raises(RuntimeError):
        call(*make(8, 16, 300, torch.float32, 1))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_results_of_two_blocks(dtype):
    """More than 1024 rows: the gradients (and fp32 logits) come from pairs of blocks, with ragged tiles on every side."""
    check(*make(1100, 200, 900, dtype, 3), 0.01)
    check(*make(1025, 40, 257, dtype, 4, on=1.0), 0.01)
    check(*make(2000, 264, 515, dtype, 5, on=0.1), 0.01)  # far fewer rows in the loss than the tiles allow for
    x, w, b, labels, mask = make(1500, 40, 300, dtype, 9)
    loss, gx, gw, gb = ops.linear_nll_loss_grad(x, w, b, labels, torch.zeros_like(mask), 1.0)
    assert loss.item() == 0 and not gx.any() and not gw.any() and not gb.any()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_several_chunks_of_rows(dtype):
    check(*make(20_000, 24, 600, dtype, 3), 0.01)
    check(*make(17_000, 9, 12_000, dtype, 4, on=0.8), 0.01)
    x, w, b, labels, mask = make(17_000, 24, 600, dtype, 5)
    mask[5000:] = False  # the later chunks have no rows in the loss
    check(x, w, b, labels, mask, 0.01)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_captured_call_of_two_blocks(dtype):
    x, w, b, labels, mask = make(1300, 72, 900, dtype, 4)
    ops.linear_nll_loss_grad(x, w, b, labels, mask, 0.1)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = ops.linear_nll_loss_grad(x, w, b, labels, mask, 0.1)
    new = make(1300, 72, 900, dtype, 6)
    for t, v in zip((x, w, b, labels, mask), new):
        t.copy_(v)
    for _ in range(2):
        graph.replay()
    torch.cuda.synchronize()
    for a, c in zip(got, ops.linear_nll_loss_grad(*new, 0.1)):
        assert torch.equal(a, c)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("K", [64, 200])
def test_rows_that_are_certain_of_their_label(dtype, K):
    """The largest logit is the label's and all others are far below: lse and that logit come from the same sums, so that their
    difference is off by the rounding of lse alone (and is never negative), not by the error of a dot product."""
    gen = torch.Generator(device=DEV).manual_seed(K)
    n, C = 150, 700
    w = torch.randn(C, K, generator=gen, device=DEV).to(dtype)
    labels = torch.randint(0, C, (n,), generator=gen, device=DEV)
    # the label's logit 90, the others' deviation 90 / sqrt(K) <= 12
    x = (w[labels].double() * (90 / w[labels].double().square().sum(1, keepdim=True))).to(dtype)
    z = x.double() @ w.double().t()
    lse = torch.logsumexp(z, 1)
    terms = lse - z[torch.arange(n, device=DEV), labels]
    assert float(terms.max()) < 1e-3 and float(terms.min()) >= 0
    # a step of lse in its units of log2, each way, and what moves the terms: the other classes' share p = terms, off by
    # p (2 e_z), e_z = (K + 16) 2^-23 sum |x w|
    e_z = (K + 16) * STEP * (x.double().abs() @ w.double().abs().t()).amax(1)
    bound = 2 * STEP * lse + 2.1 * terms * e_z
    assert float((e_z * terms).max()) < float(bound.min())
    loss, got_lse = ops.linear_nll_loss(x, w, None, labels, None, 1.0)
    assert float(loss) >= 0 and abs(float(loss) - float(terms.sum())) <= float(bound.sum())
    for r in range(0, n, 7):
        mask = torch.zeros(n, dtype=torch.bool, device=DEV)
        mask[r] = True
        one, gx, gw, gb = ops.linear_nll_loss_grad(x, w, torch.zeros(C, device=DEV), labels, mask, 1.0)
        assert float(one) >= 0 and abs(float(one) - float(terms[r])) <= float(bound[r])
        # p - 1 of the label: of the size of what the others have, or a step of lse
        assert float(gb[labels[r]]) <= 0 and abs(float(gb[labels[r]]) + float(-torch.expm1(-terms[r]))) <= float(bound[r])


@pytest.mark.parametrize("n,K", [(150, 24), (1200, 40)])
def test_weight_gradients_of_very_rare_classes(n, K):
    """Classes of probability 2^-30 to 2^-50 that no row has as its label: their gradients keep their own accuracy.  G is carried in
    22 bits down to 2^-28 and is 2^-51 off below, an operand's value likewise beside the largest of its column."""
    x, w, b, labels, mask = make(n, K, 300, torch.float32, n)
    labels = labels % 200
    b[200:225] -= 14.0
    b[225:250] -= 21.0
    b[250:] -= 27.0
    ref = Ref(x, w, b, labels, mask, 1.0)
    _, _, gw, gb = ops.linear_nll_loss_grad(x, w, b, labels, mask, 1.0)
    # the bound of a class's gradients from its own probabilities: p (e_z + e_lse) as in Ref, 2^-21 of G for its two planes and as
    # much for x's, sums of m terms
    xr = x[ref.rows].double()
    z = xr @ w.double().t() + b.double()
    p = (z - torch.logsumexp(z, 1, keepdim=True)).exp()[:, 200:]
    e_z = (K + 16) * STEP * (xr.abs() @ w.double().abs().t() + b.double().abs())
    e_p = p * (e_z[:, 200:] + ref.e_lse[ref.rows][:, None] + 8 * STEP) * 1.01
    m = len(ref.rows)
    e_w = (e_p + p * 2.0 ** -20 + 2.0 ** -50).t() @ xr.abs() + (m + 16) * STEP * (p.t() @ xr.abs())
    e_b = e_p.sum(0) + (m + 16) * STEP * p.sum(0)
    close(gw[200:], p.t() @ xr, e_w)
    close(gb[200:], p.sum(0), e_b)
    # How sharp that bound is (a statement about the reference alone): lse is about log 300 + 2 = 7.7, so classes 21 below are of
    # probability e^-28.7 = 2^-41, of which the absolute 2^-50 is 2^-9; the logits' share, 2 e_z, is below 2^-11
    assert float(p[:, 25:50].max()) < 2.0 ** -25 and float((e_w / (p.t() @ xr.abs()))[25:50].max()) < 2.0 ** -8


@pytest.mark.parametrize("n,K,C", [(5000, 512, 16), (700, 512, 46), (2500, 400, 300), (3000, 1100, 100)])
def test_fp32_gradients_over_many_features(n, K, C):
    """As exact as fp32 sums: a logit takes at most 32 additions that round towards zero before its sums move on, half a step of
    2^-23 each on average, of partial sums that grow like a random walk (two thirds of the whole): 32 x 2^-24 x 2/3 = 2^-20.6 of
    it at most, and a gradient is off by about what its logits are."""
    x, w, b, labels, mask = make(n, K, C, torch.float32, n + K + C)
    ref = Ref(x, w, b, labels, mask, 1.0 / n)
    _, *grads = ops.linear_nll_loss_grad(x, w, b, labels, mask, 1.0 / n)
    for got, want in zip(grads, (ref.gx, ref.gw, ref.gb)):
        assert float((got.double() - want).norm()) <= 2.0 ** -20 * float(want.norm())
    assert float((ops.linear_nll_loss(x, w, b, labels, mask, 1.0 / n)[0].double() - ref.loss).abs()) <= 2.0 ** -20 * float(ref.loss)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_the_most_features(dtype):
    check(*make(33, 16384, 40, dtype, 3), 0.1)
    check(*make(1100, 1500, 300, dtype, 4), 0.1)  # pairs of blocks, three windows


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_two_large_calls_at_once(dtype):
    """Calls whose kernels want all of an SM's tensor memory, on two streams."""
    a, b = make(1500, 300, 2000, dtype, 4), make(1300, 520, 1500, dtype, 5)
    want_a, want_b = ops.linear_nll_loss_grad(*a, 0.1), ops.linear_nll_loss_grad(*b, 0.1)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    got_a, got_b = [], []
    for _ in range(4):
        got_a.append(ops.linear_nll_loss_grad(*a, 0.1))
        with torch.cuda.stream(side):
            got_b.append(ops.linear_nll_loss_grad(*b, 0.1))
    torch.cuda.synchronize()
    for got, want in ((got_a, want_a), (got_b, want_b)):
        for one in got:
            for u, v in zip(one, want):
                assert torch.equal(u, v)
