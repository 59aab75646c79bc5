"""8-bit activation checkpoints: codes bit for bit, restored values, and the weight gradient taken from the codes."""
import numpy as np
import pytest
import torch

from super_gnn_b200 import supergnn_ops as ops

pytestmark = pytest.mark.gpu
DEV = "cuda"
U = 2.0 ** -24


def expected(x):
    """Codes and parameters by IEEE fp32 arithmetic on the host."""
    x = x.float().cpu().numpy()
    low, high = x.min(1), x.max(1)
    scale = ((high - low) / np.float32(255)).astype(np.float32)
    scale[scale < np.finfo(np.float32).tiny] = 1
    codes = np.rint((x - low[:, None]) / scale[:, None])
    return torch.from_numpy(codes.astype(np.uint8)), torch.from_numpy(np.stack([low, scale], 1))


def rows(n, F, dtype, seed, spread=1.0):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    x = torch.randn(n, F, generator=gen, device=DEV)
    return (x * torch.exp(spread * torch.randn(n, 1, generator=gen, device=DEV))).to(dtype)


@pytest.mark.parametrize("n,F", [(1, 1), (5, 2), (9, 7), (33, 64), (70, 100), (13, 255), (40, 512), (11, 602), (3, 1024),
                                 (4, 1026), (3, 3001), (2, 9000), (5000, 33)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_pack_is_bit_exact_and_unpack_is_one_rounding(n, F, dtype):
    x = rows(n, F, dtype, n + F)
    codes, params = ops.checkpoint_pack_rows(x)
    want_codes, want_params = expected(x)
    assert torch.equal(params.cpu(), want_params)
    assert torch.equal(codes.cpu(), want_codes)
    kept = want_params[:, :1].double() + want_params[:, 1:].double() * want_codes.double()
    for out in (torch.float32, torch.bfloat16, torch.float16):
        got = ops.checkpoint_unpack_rows(codes, params, out)
        assert got.dtype == out and got.shape == x.shape
        fits = kept.abs() < torch.finfo(out).max
        # fused multiply-add, rounded to fp32 and then to the type
        bound = kept.abs() * (U + torch.finfo(out).eps / 2 * (1 + 2 * U)) + torch.finfo(out).smallest_normal * torch.finfo(out).eps
        assert ((got.cpu().double() - kept).abs()[fits] <= bound[fits]).all()
    # half a step of the code, and the roundings of the range and of the quotient
    step = want_params[:, 1:].double()
    assert ((kept - x.cpu().double()).abs() <= step * (0.5 + 2 ** -14) + 4 * U * x.cpu().double().abs()).all()


@pytest.mark.parametrize("n,F", [(150_001, 3), (150_006, 32), (90_007, 63), (60_001, 100)])
def test_narrow_rows_that_share_a_warp(n, F):
    x = rows(n, F, torch.float32, n)
    codes, params = ops.checkpoint_pack_rows(x)
    want_codes, want_params = expected(x)
    assert torch.equal(params.cpu(), want_params) and torch.equal(codes.cpu(), want_codes)
    kept = want_params[:, :1].double() + want_params[:, 1:].double() * want_codes.double()
    off = (ops.checkpoint_unpack_rows(codes, params).cpu().double() - kept).abs()
    assert (off <= kept.abs() * 2 * U + torch.finfo(torch.float32).smallest_normal * 2 * U).all()  # one fused multiply-add


def test_values_next_to_a_border_between_two_codes():
    """Quotients on and next to k + 1/2: the codes are those of the IEEE quotient, to nearest even."""
    base = torch.arange(0, 255, device=DEV, dtype=torch.float32) + 0.5
    row = torch.cat([torch.tensor([0.0, 255.0], device=DEV), base, torch.nextafter(base, torch.tensor(300.0, device=DEV)),
                     torch.nextafter(base, torch.tensor(-1.0, device=DEV))])
    x = torch.stack([row * s for s in (1.0, 3.0, 0.1, 1e-20, 1e20, 2.0 ** -126)])
    codes, params = ops.checkpoint_pack_rows(x)
    want_codes, want_params = expected(x)
    assert torch.equal(params.cpu(), want_params) and torch.equal(codes.cpu(), want_codes)


def test_rows_without_range_and_rows_that_cannot_be_kept():
    big = torch.finfo(torch.float32).max
    x = torch.zeros(8, 40, device=DEV)
    x[0] = 2.5
    x[1, 3] = float("nan")
    x[2, 4] = float("inf")
    x[3, 5] = float("-inf")
    x[4, 0], x[4, 1] = big, -big       # range above fp32
    x[5, 0], x[5, 1] = -big, 1.0       # a masked place of the type's lowest value
    x[6] = torch.arange(40, device=DEV) * 1e-45  # range below the smallest normal step
    x[7] = -1e-30
    codes, params = ops.checkpoint_pack_rows(x)
    got = ops.checkpoint_unpack_rows(codes, params)
    assert (got[0] == 2.5).all() and (got[7] == -1e-30).all() and (got[6] == 0).all()
    assert torch.isnan(got[1:5]).all()
    assert torch.isfinite(got[5]).all() and got[5, 0] == -big
    assert ((got[5, 1:].double() - x[5, 1:].double()).abs() <= big / 255 * 0.51).all()


def test_strided_input_and_codes():
    x = rows(50, 64, torch.float32, 4)
    wide = torch.zeros(50, 77, device=DEV)
    wide[:, 5:69] = x
    a, b = ops.checkpoint_pack_rows(x), ops.checkpoint_pack_rows(wide[:, 5:69])
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    store = torch.zeros(50, 70, dtype=torch.uint8, device=DEV)
    store[:, 3:67] = a[0]
    assert torch.equal(ops.checkpoint_unpack_rows(store[:, 3:67], a[1]), ops.checkpoint_unpack_rows(*a))
    g = rows(50, 9, torch.float32, 6)
    assert torch.equal(ops.checkpoint_weight_grad(g, store[:, 3:67], a[1]), ops.checkpoint_weight_grad(g, *a))


def grad_bounds(g, codes, params):
    """The product in 64 bits, the worst case of its error and the size its errors have when they are independent.

    g sc is rounded once (2^-24) and carried in three terms of eight bits (2^-27 more), the codes are exact, and every addition
    of a sum of 3 n terms (of the scaled codes; n of the zero points) is off by at most 2^-23 of the sum of the magnitudes."""
    g, c = g.double(), codes.double()
    zp, sc = params[:, :1].double(), params[:, 1:].double()
    n = g.size(0)
    kept = zp + sc * c
    want = g.t() @ kept
    mags = g.abs().t() @ (sc * c + zp.abs())
    worst = mags * (2 ** -23 + (3 * n + 40) * 2 ** -23)
    typical = (g.square().t() @ (sc * c + zp.abs()).square()).sqrt()
    return want, worst, typical


GRAD_SIZES = [(1, 1, 1), (2, 3, 5), (63, 47, 100), (64, 128, 256), (65, 129, 257), (100, 16, 16), (1000, 256, 512),
              (1531, 260, 130), (2500, 1, 600), (4096, 64, 1), (12345, 41, 602)]


@pytest.mark.parametrize("n,M,F", GRAD_SIZES)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_weight_grad(n, M, F, dtype):
    x = torch.relu(rows(n, F, torch.float32, n + M)) + 0.25
    g = rows(n, M, dtype, n + F, spread=0.3)
    codes, params = ops.checkpoint_pack_rows(x)
    want, worst, typical = grad_bounds(g, codes, params)
    got = ops.checkpoint_weight_grad(g, codes, params)
    assert got.dtype == torch.float32 and got.shape == (M, F)
    off = (got.double() - want).abs()
    assert (off <= worst).all(), float((off / worst).max())
    # 2^-23 of each value for g sc, and 2^-24 on average of a partial sum (of the typical size) at each of the three additions
    # for sixteen rows, all towards zero, of 256 rows at most; those sums then add up with errors of random sign
    assert off.norm() <= (2 ** -23 + (3 * min(n, 256) / 16 + 4 * (n / 256) ** 0.5 + 2) * 2 ** -24) * typical.norm()
    # adding onto an existing gradient: one more rounding
    base = torch.randn(M, F + 3, device=DEV)[:, 1:1 + F]
    out = torch.empty(M, F + 3, device=DEV)[:, 1:1 + F].copy_(base)
    assert ops.checkpoint_weight_grad(g, codes, params, out=out, beta=1.0) is out
    assert ((out.double() - (got.double() + base.double())).abs() <= 2 * U * (got.double().abs() + base.double().abs())).all()
    assert torch.equal(ops.checkpoint_weight_grad(g, codes, params), got)  # the order of the sums is fixed


def test_weight_grad_of_strided_gradients_and_no_rows():
    x, g = rows(300, 96, torch.float32, 1), rows(300, 40, torch.float32, 2)
    codes, params = ops.checkpoint_pack_rows(x)
    want = ops.checkpoint_weight_grad(g, codes, params)
    wide = torch.zeros(300, 53, device=DEV)
    wide[:, 7:47] = g
    assert torch.equal(ops.checkpoint_weight_grad(wide[:, 7:47], codes, params), want)
    assert torch.equal(ops.checkpoint_weight_grad(g.t().contiguous().t(), codes, params), want)
    one = torch.ones((), device=DEV).expand(300, 40)
    assert torch.equal(ops.checkpoint_weight_grad(one, codes, params), ops.checkpoint_weight_grad(one.contiguous(), codes, params))
    none = ops.checkpoint_pack_rows(x[:0])
    assert not ops.checkpoint_weight_grad(g[:0], *none).any()
    out = torch.ones(40, 96, device=DEV)
    ops.checkpoint_weight_grad(g[:0], *none, out=out, beta=0.5)
    assert (out == 0.5).all()


def test_weight_grad_shows_a_lost_row():
    x, g = rows(130, 40, torch.float32, 1), rows(130, 20, torch.float32, 2)
    x[77, 3] = float("nan")
    assert torch.isnan(ops.checkpoint_weight_grad(g, *ops.checkpoint_pack_rows(x))).all()


@pytest.mark.parametrize("call", [
    lambda x, c, p: ops.checkpoint_pack_rows(x.double()),
    lambda x, c, p: ops.checkpoint_pack_rows(x.cpu()),
    lambda x, c, p: ops.checkpoint_pack_rows(x[0]),
    lambda x, c, p: ops.checkpoint_pack_rows(x[:, :0]),
    lambda x, c, p: ops.checkpoint_unpack_rows(c.int(), p),
    lambda x, c, p: ops.checkpoint_unpack_rows(c, p[:-1]),
    lambda x, c, p: ops.checkpoint_unpack_rows(c, p, torch.float64),
    lambda x, c, p: ops.checkpoint_unpack_rows(c, p.cpu()),
    lambda x, c, p: ops.checkpoint_weight_grad(x[:-1], c, p),
    lambda x, c, p: ops.checkpoint_weight_grad(x, c, p, beta=1.0),
    lambda x, c, p: ops.checkpoint_weight_grad(x, c, p, out=torch.empty(3, 8, device=DEV)),
    lambda x, c, p: ops.checkpoint_weight_grad(x.double(), c, p),
])
def test_refusals(call):
    x = torch.randn(6, 8, device=DEV)
    with pytest.raises(RuntimeError):
        call(x, *ops.checkpoint_pack_rows(x))


def test_weight_grad_over_many_rounds_and_row_ranges():
    """Rows enough for several moves of the sums into registers in every row range, for both ways operands come in."""
    n, M, F = 300_007, 40, 96
    x = torch.relu(rows(n, F, torch.float32, 1))
    x[::3] = 0  # rows without a range: the zero point alone
    g = rows(n, M, torch.float32, 2, spread=0.3)
    codes, params = ops.checkpoint_pack_rows(x)
    want, worst, typical = grad_bounds(g, codes, params)
    wide = torch.zeros(n, M + 1, device=DEV)
    wide[:, 1:] = g  # rows that are not aligned
    for operand in (g, wide[:, 1:]):
        off = (ops.checkpoint_weight_grad(operand, codes, params).double() - want).abs()
        assert (off <= worst).all()
        # sums of 256 rows in tensor memory: 48 additions of 2^-24 on average, all towards zero, and 2^-23 for g sc and the rest
        assert off.norm() <= (2 ** -23 + 48 * 2 ** -24 + 4 * (n / 256) ** 0.5 * 2 ** -24) * typical.norm()


def test_captured_weight_grad():
    x, g = rows(700, 96, torch.float32, 1), rows(700, 40, torch.float32, 2)
    codes, params = ops.checkpoint_pack_rows(x)
    ops.checkpoint_weight_grad(g, codes, params)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        codes, params = ops.checkpoint_pack_rows(x)
        got = ops.checkpoint_weight_grad(g, codes, params)
        back = ops.checkpoint_unpack_rows(codes, params)
    x.copy_(rows(700, 96, torch.float32, 5))
    g.copy_(rows(700, 40, torch.float32, 6))
    graph.replay()
    torch.cuda.synchronize()
    want = ops.checkpoint_pack_rows(x)
    assert torch.equal(got, ops.checkpoint_weight_grad(g, *want)) and torch.equal(back, ops.checkpoint_unpack_rows(*want))


@pytest.mark.parametrize("n,M,F,dtype", [(1000, 127, 96, torch.float32), (1003, 255, 300, torch.bfloat16), (999, 255, 64, torch.float16),
                                         (700, 129, 40, torch.float32), (90, 5000, 33, torch.float32), (70, 9, 5001, torch.bfloat16),
                                         (33, 65536, 1, torch.float16), (31, 1, 65536, torch.float32)])
def test_weight_grad_of_packed_odd_rows_and_many_columns(n, M, F, dtype):
    """Rows of g that come as one run of bytes, the widest of them and one more, and results of many tiles."""
    test_weight_grad(n, M, F, dtype)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_weight_grad_of_a_gradient_that_is_not_finite(dtype):
    """Its row of the result says so; the others do not change."""
    x, g = rows(300, 40, torch.float32, 1), rows(300, 20, dtype, 2)
    kept = ops.checkpoint_pack_rows(x)
    want = ops.checkpoint_weight_grad(g, *kept)
    g[77, 3], g[299, 11] = float("inf"), float("nan")
    got = ops.checkpoint_weight_grad(g, *kept)
    assert torch.isnan(got[[3, 11]]).all()
    got[[3, 11]] = want[[3, 11]]
    assert torch.equal(got, want)


@pytest.mark.parametrize("M,F", [(70_001, 3), (5, 70_001), (65_537, 1)])
def test_weight_grad_of_more_columns_than_one_call_takes(M, F):
    test_weight_grad(25, M, F, torch.bfloat16)
