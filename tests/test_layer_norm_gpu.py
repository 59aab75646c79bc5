"""Layer norm of any width against its formulas in 64 bits, with and without the 8-bit checkpoint of its input."""
import pytest
import torch

from super_gnn_b200 import supergnn_ops as ops

pytestmark = pytest.mark.gpu
DEV = "cuda"
U = 2.0 ** -24  # half a step of fp32, relative


def half_step(t, dtype):
    """A rounding to ``dtype`` is off by at most this (with the smallest fp16 / bf16 steps near zero)."""
    return t.abs() * (torch.finfo(dtype).eps / 2) + torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps


def depth(H):
    """Additions behind one fp32 row sum: at most H / 32 a lane of a warp (H / 256 a thread of a block), the shuffle
    tree, the eight warps of a block; or eight a lane and at most four shuffles where narrow rows share a warp."""
    return H / 32 + 5 + 8


class Ref:
    """The formulas in 64 bits on the inputs as given, and bounds of what 32-bit sums may be off by.

    mean: depth * U * mean|x|.  The variance is taken around the computed mean, which enters squared, so its relative
    error is (depth + 4) U, rstd's half of that plus 3 U.  xh = (x - mean) rstd then is off by at most
    e_xh = U (rstd depth mean|x| + |xh| (depth / 2 + 8))."""

    def __init__(self, x, gamma, beta, eps, kept=None):
        x = x.double()
        H = x.size(1)
        self.d = depth(H)
        self.mean = x.mean(1, keepdim=True)
        self.rstd = 1.0 / ((x - self.mean).square().mean(1, keepdim=True) + eps).sqrt()
        self.g = torch.ones(H, dtype=torch.float64, device=DEV) if gamma is None else gamma.double()
        b = torch.zeros(H, dtype=torch.float64, device=DEV) if beta is None else beta.double()
        k = x if kept is None else kept.double()
        self.xh = (x - self.mean) * self.rstd
        e_mean = self.d * U * x.abs().mean(1, keepdim=True)
        self.e_xh = self.rstd * e_mean + U * self.xh.abs() * (self.d / 2 + 8)
        self.y = self.xh * self.g + b
        self.e_y = self.g.abs() * self.e_xh + 2 * U * self.y.abs() + U * (self.xh * self.g).abs()
        self.kh = (k - self.mean) * self.rstd  # from the checkpoint: also the rounding of a restored value and of its centre
        self.e_kh = self.rstd * (e_mean + 3 * U * (k.abs() + self.mean.abs())) + U * self.kh.abs() * (self.d / 2 + 8)

    def backward(self, gy):
        gy = gy.double()
        n, d = gy.size(0), self.d
        a = gy * self.g
        m1, m2 = a.mean(1, keepdim=True), (a * self.kh).mean(1, keepdim=True)
        gx = self.rstd * (a - m1 - self.kh * m2)
        e1 = (d + 6) * U * a.abs().mean(1, keepdim=True)
        e2 = (d + 6) * U * (a * self.kh).abs().mean(1, keepdim=True) + (a.abs() * self.e_kh).mean(1, keepdim=True)
        e_gx = self.rstd * (e1 + self.kh.abs() * e2 + self.e_kh * m2.abs()
                            + 6 * U * (a.abs() + m1.abs() + (self.kh * m2).abs())) + gx.abs() * (d / 2 + 8) * U
        # column sums: the rows of a warp (at least one grid of 148 blocks of 8 warps), its block, the partial rows
        rows = n / (148 * 8) + 1 + 8 + 1184 / 32 + 32
        gg, e_gg = (gy * self.kh).sum(0), (rows + 2) * U * (gy * self.kh).abs().sum(0) + (gy.abs() * self.e_kh).sum(0)
        gb, e_gb = gy.sum(0), (rows + 2) * U * gy.abs().sum(0)
        return (gx, e_gx), (gg, e_gg), (gb, e_gb)


def close(got, want, err):
    off = (got.double() - want).abs()
    bound = err * (1 + 2 ** -6) + half_step(want, got.dtype)  # second-order terms: products of two of the errors above
    assert torch.isfinite(got).all()
    bad = off > bound
    assert not bad.any(), (off[bad][:4], bound[bad][:4], int(bad.sum()))


def make(n, H, dtype, pdtype, seed, pad=0, offset=0):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    buf = torch.randn(n, H + pad + offset, generator=gen, device=DEV) * 1.5
    buf = (buf + torch.randn(n, 1, generator=gen, device=DEV)).to(dtype)
    x = buf[:, offset:offset + H]
    gy = torch.randn(n, H, generator=gen, device=DEV).to(dtype)
    gamma = (1 + 0.3 * torch.randn(H, generator=gen, device=DEV)).to(pdtype)
    beta = (0.3 * torch.randn(H, generator=gen, device=DEV)).to(pdtype)
    return x, gy, gamma, beta


SIZES = [(1, 1), (3, 1), (1, 256), (7, 3), (33, 31), (64, 32), (50, 100), (257, 130), (41, 256), (19, 602), (9, 1000),
         (5, 1024), (6, 1025), (3, 1030), (2, 2052), (2, 5003), (1, 16384), (3000, 96)]


@pytest.mark.parametrize("n,H", SIZES)
@pytest.mark.parametrize("dtype,pdtype", [(torch.float32, torch.float32), (torch.bfloat16, torch.float32),
                                          (torch.bfloat16, torch.bfloat16), (torch.float16, torch.float16)])
@pytest.mark.parametrize("checkpoint", [False, True])
def test_forward_and_backward(n, H, dtype, pdtype, checkpoint):
    x, gy, gamma, beta = make(n, H, dtype, pdtype, seed=n * 7 + H)
    eps = 1e-5
    if checkpoint:
        y, stats, codes, params = ops.layer_norm_forward(x, gamma, beta, eps, checkpoint=True)
        want_codes, want_params = ops.checkpoint_pack_rows(x)
        assert torch.equal(codes, want_codes) and torch.equal(params, want_params)
        kept = params[:, :1].double() + params[:, 1:].double() * codes.double()
        ref = Ref(x, gamma, beta, eps, kept)
        got = ops.layer_norm_backward_checkpoint(gy, codes, params, stats, gamma)
    else:
        y, stats = ops.layer_norm_forward(x, gamma, beta, eps)
        ref = Ref(x, gamma, beta, eps)
        got = ops.layer_norm_backward(gy, x, stats, gamma)
    assert y.dtype == dtype and got[0].dtype == dtype and got[1].dtype == pdtype and got[2].dtype == pdtype
    close(y, ref.y, ref.e_y)
    for g, (want, err) in zip(got, ref.backward(gy)):
        close(g, want, err)


@pytest.mark.parametrize("n,H", [(150_001, 2), (150_007, 20), (90_002, 61), (60_003, 64), (60_005, 128)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("checkpoint", [False, True])
def test_narrow_rows_that_share_a_warp(n, H, dtype, checkpoint):
    """More rows than the resident warps take at once, and a last group that is not whole."""
    test_forward_and_backward(n, H, dtype, torch.float32, checkpoint)


@pytest.mark.parametrize("n,H", [(1501, 544), (1502, 840), (2003, 1026), (1501, 1301), (1999, 2048)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
@pytest.mark.parametrize("checkpoint", [False, True])
def test_long_rows_several_a_block(n, H, dtype, checkpoint):
    test_forward_and_backward(n, H, dtype, torch.float32, checkpoint)


@pytest.mark.parametrize("pad,offset", [(4, 0), (1, 0), (0, 1), (3, 2), (12, 4)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_strided_and_misaligned_rows(pad, offset, dtype):
    n, H = 37, 96
    x, gy, gamma, beta = make(n, H, dtype, torch.float32, 5, pad, offset)
    wide = torch.full((n, H + 9), 7.0, dtype=dtype, device=DEV)
    out = wide[:, 3:3 + H]
    y, stats = ops.layer_norm_forward(x, gamma, beta, out=out)
    assert y is out and (wide[:, :3] == 7).all() and (wide[:, 3 + H:] == 7).all()
    ref = Ref(x, gamma, beta, 1e-5)
    close(y, ref.y, ref.e_y)
    for g, (want, err) in zip(ops.layer_norm_backward(gy, x, stats, gamma), ref.backward(gy)):
        close(g, want, err)


def test_without_affine_with_expanded_and_transposed_gradients():
    x, gy, _, _ = make(24, 50, torch.float32, torch.float32, 3)
    y, stats = ops.layer_norm_forward(x)
    ref = Ref(x, None, None, 1e-5)
    close(y, ref.y, ref.e_y)
    ones = torch.ones((), device=DEV).expand(24, 50)  # the gradient of a plain sum: strides (0, 0)
    for g, (want, err) in zip(ops.layer_norm_backward(ones, x, stats), ref.backward(ones)):
        close(g, want, err)
    turned = gy.t().contiguous().t()
    for a, b in zip(ops.layer_norm_backward(turned, x, stats), ops.layer_norm_backward(gy, x, stats)):
        assert torch.equal(a, b)


def test_in_place_gradient_and_repeatability():
    x, gy, gamma, beta = make(700, 300, torch.float32, torch.float32, 8)
    _, stats = ops.layer_norm_forward(x, gamma, beta)
    first = ops.layer_norm_backward(gy, x, stats, gamma)
    own = gy.clone()
    again = ops.layer_norm_backward(own, x, stats, gamma, in_place=True)
    assert again[0] is own
    for a, b in zip(first, again):
        assert torch.equal(a, b)


def test_no_rows():
    x = torch.empty(0, 40, device=DEV)
    y, stats, codes, params = ops.layer_norm_forward(x, checkpoint=True)
    assert y.shape == (0, 40) and codes.shape == (0, 40)
    gx, gg, gb = ops.layer_norm_backward(x, x, stats)
    assert gx.shape == (0, 40) and not gg.any() and not gb.any()


def test_constant_rows_and_rows_with_nan():
    x = torch.full((4, 64), 3.0, device=DEV)
    x[1] = torch.arange(64.0, device=DEV)
    x[2, 5] = float("nan")
    x[3, 7] = float("inf")
    y, stats, codes, params = ops.layer_norm_forward(x, checkpoint=True)
    assert (y[0] == 0).all() and torch.isfinite(y[1]).all() and torch.isnan(y[2]).all() and torch.isnan(y[3]).any()
    gx, _, _ = ops.layer_norm_backward_checkpoint(torch.ones_like(x), codes, params, stats)
    assert torch.isfinite(gx[:2]).all() and torch.isnan(gx[2:]).all()


def test_gradient_against_differences():
    """gx along a random direction against a central difference of the loss sum(y * gy) in 64 bits."""
    x, gy, gamma, beta = make(6, 40, torch.float32, torch.float32, 11)
    _, stats = ops.layer_norm_forward(x, gamma, beta)
    gx, gg, gb = ops.layer_norm_backward(gy, x, stats, gamma)
    gen = torch.Generator(device=DEV).manual_seed(1)

    def value(xx, g, b):
        return float((Ref(xx, g, b, 1e-5).y * gy.double()).sum())

    for grad, at in ((gx, 0), (gg, 1), (gb, 2)):
        base = [x.double(), gamma.double(), beta.double()]
        v = torch.randn(base[at].shape, generator=gen, device=DEV, dtype=torch.float64)
        h = 1e-5
        up, down = list(base), list(base)
        up[at], down[at] = base[at] + h * v, base[at] - h * v
        want = (value(*up) - value(*down)) / (2 * h)
        # truncation h^2 |f'''| ~ 1e-10 times the sum of the terms, the fp32 gradient 1e-6 of them
        assert abs(float((grad.double() * v).sum()) - want) <= 1e-5 * float((grad.double() * v).abs().sum())


@pytest.mark.parametrize("call", [
    lambda x, g: ops.layer_norm_forward(x.double()),
    lambda x, g: ops.layer_norm_forward(x, g.half()),
    lambda x, g: ops.layer_norm_forward(x, g[:-1]),
    lambda x, g: ops.layer_norm_forward(x, g, g.bfloat16()),
    lambda x, g: ops.layer_norm_forward(x.cpu()),
    lambda x, g: ops.layer_norm_forward(x[0]),
    lambda x, g: ops.layer_norm_forward(x, eps=-1.0),
    lambda x, g: ops.layer_norm_forward(x, out=torch.empty(8, 4, device=DEV).t()),
    lambda x, g: ops.layer_norm_forward(torch.empty(2, 0, device=DEV)),
    lambda x, g: ops.layer_norm_forward(torch.empty(1, 16385, device=DEV)),
    lambda x, g: ops.layer_norm_backward(x, x[:2], torch.empty(4, 2, device=DEV)),
    lambda x, g: ops.layer_norm_backward(x, x, torch.empty(3, 2, device=DEV)),
    lambda x, g: ops.layer_norm_backward(x.t().contiguous().t(), x, torch.empty(4, 2, device=DEV), in_place=True),
    lambda x, g: ops.layer_norm_backward_checkpoint(x, torch.empty(4, 8, device=DEV), torch.empty(4, 2, device=DEV),
                                                    torch.empty(4, 2, device=DEV)),
])
def test_refusals(call):
    with pytest.raises(RuntimeError):
        call(torch.randn(4, 8, device=DEV), torch.ones(8, device=DEV))


@pytest.mark.parametrize("n,H,dtype", [(8, 601, torch.float32), (9, 601, torch.bfloat16), (4000, 257, torch.float32),
                                       (5003, 602, torch.bfloat16), (3001, 1021, torch.float16), (700, 300, torch.float16),
                                       (6007, 512, torch.bfloat16), (2500, 640, torch.float32), (10_000, 66, torch.bfloat16)])
def test_packed_rows_through_the_ring(n, H, dtype):
    """More batches of eight rows than the ring has buffers, a short last batch, and gx over gy."""
    x, gy, gamma, beta = make(n, H, dtype, torch.float32, seed=n + H)
    x = x.contiguous()
    y, stats = ops.layer_norm_forward(x, gamma, beta)
    ref = Ref(x, gamma, beta, 1e-5)
    close(y, ref.y, ref.e_y)
    got = ops.layer_norm_backward(gy, x, stats, gamma)
    for g, (want, err) in zip(got, ref.backward(gy)):
        close(g, want, err)
    own = gy.clone()
    for a, b in zip(ops.layer_norm_backward(own, x, stats, gamma, in_place=True), got):
        assert torch.equal(a, b)
    back = x.clone()  # y over x
    assert torch.equal(ops.layer_norm_forward(back, gamma, beta, out=back)[0], y)


@pytest.mark.parametrize("n,H,dtype,backward", [
    (20_003, 602, torch.float32, True), (10_003, 600, torch.float32, True), (40_005, 831, torch.float32, True),
    (10_003, 1301, torch.float32, False), (10_007, 2047, torch.float32, False), (10_005, 2038, torch.float16, False)])
def test_short_last_batch_in_a_ring_of_two_buffers(n, H, dtype, backward):
    """Rows so long that the ring has two buffers, at least three batches a block, and a last batch that is not whole: its
    rows are written over a buffer that a result has just left from.  (The rows before it are the ones that would suffer.)"""
    x, gy, gamma, beta = make(n, H, dtype, torch.float32, seed=n + H)
    x = x.contiguous()
    y, stats = ops.layer_norm_forward(x, gamma, beta)
    ref = Ref(x, gamma, beta, 1e-5)
    close(y, ref.y, ref.e_y)
    if not backward:
        for _ in range(4):
            assert torch.equal(ops.layer_norm_forward(x, gamma, beta)[0], y)
        return
    got = ops.layer_norm_backward(gy, x, stats, gamma)
    for g, (want, err) in zip(got, ref.backward(gy)):
        close(g, want, err)
    for _ in range(4):
        for a, b in zip(ops.layer_norm_backward(gy, x, stats, gamma), got):
            assert torch.equal(a, b)


def test_captured_and_on_another_stream():
    x, gy, gamma, beta = make(900, 300, torch.bfloat16, torch.float32, seed=3)
    x = x.contiguous()
    ops.layer_norm_backward(gy, x, ops.layer_norm_forward(x, gamma, beta)[1], gamma)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y, stats, codes, params = ops.layer_norm_forward(x, gamma, beta, checkpoint=True)
        grads = ops.layer_norm_backward_checkpoint(gy, codes, params, stats, gamma)
    x2, gy2, gamma2, beta2 = make(900, 300, torch.bfloat16, torch.float32, seed=4)
    for t, v in zip((x, gy, gamma, beta), (x2, gy2, gamma2, beta2)):
        t.copy_(v)
    graph.replay()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        want = ops.layer_norm_forward(x, gamma, beta, checkpoint=True)
        want_grads = ops.layer_norm_backward_checkpoint(gy, want[2], want[3], want[1], gamma)
    torch.cuda.synchronize()
    for a, b in zip((y, stats, codes, params) + grads, want + want_grads):
        assert torch.equal(a, b)


@pytest.mark.parametrize("n,H", [(700, 2049), (500, 5003), (333, 9000), (301, 16384)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("checkpoint", [False, True])
def test_rows_read_again_several_a_block(n, H, dtype, checkpoint):
    """Rows beyond what a block holds in registers, up to the limit, more of them than blocks."""
    test_forward_and_backward(n, H, dtype, torch.float32, checkpoint)


@pytest.mark.parametrize("n,H,dtype", [(8 * 296 * 3 + 5, 300, torch.bfloat16), (8 * 592 * 2 + 1, 201, torch.float32),
                                       (10_001, 129, torch.float16), (2377, 1024, torch.bfloat16)])
def test_short_last_batch_in_longer_rings(n, H, dtype):
    """Three and four buffers, where the short batch comes first, second or later in its block."""
    x, gy, gamma, beta = make(n, H, dtype, torch.float32, seed=n + H)
    for rows in (n, n - 1, 8, 9, 15):
        a, g = x[:rows].contiguous(), gy[:rows].contiguous()
        y, stats = ops.layer_norm_forward(a, gamma, beta)
        ref = Ref(a, gamma, beta, 1e-5)
        close(y, ref.y, ref.e_y)
        for got, (want, err) in zip(ops.layer_norm_backward(g, a, stats, gamma), ref.backward(g)):
            close(got, want, err)
