"""The 8-bit product where the scales' product leaves float32's normal range while the value does not.

Four roundings of half a step (e = 2^-24) of terms no larger than |sum sa sw| + |bias| lie between the output and the formula: the sum's conversion, the
product of the scales' mantissas, its product with the sum, the bias; and one of half the least subnormal (2^-150) where the value ends up there."""
import pytest
import torch

pytestmark = pytest.mark.gpu
E = 2.0 ** -24
# strips (one launch with quantised tokens and none), 64 x 64 tiles, K split over workgroups, 128 and 256 tiles
SIZES = [(3, 70, 500), (20, 70, 500), (40, 64, 500), (200, 200, 300), (64, 66, 16400), (2500, 1301, 140), (3600, 3500, 130)]


@pytest.fixture(scope="module")
def K():
    from controllable_agent_amd import kernels
    return kernels


def _rows(gen, rows, k):
    return torch.randint(-127, 128, (rows, (k + 15) // 16 * 16), generator=gen, dtype=torch.int8).cuda()[:, :k]


def _check(y, a, sa, w, sw, bias):
    sums = (a.float() @ w.float().t()).cpu().double() if a.shape[1] <= 1024 else a.cpu().double() @ w.cpu().double().t()      # (exact: below 2^24)
    main = sums * sa.cpu().double()[:, None] * sw.cpu().double()
    want = main if bias is None else main + bias.cpu().double()
    bound = 4 * E * (main.abs() + (0 if bias is None else bias.cpu().double().abs())) + 2.0 ** -149
    # float32 ends at 2^128 - 2^104; rounding to nearest makes an infinity of 2^128 - 2^103 and all beyond: what lies farther from there than the bound has
    # to be on its side, what lies nearer may be on either
    end = 2.0 ** 128 - 2.0 ** 103
    y = y.cpu().double()
    big, near = want.abs() - bound >= end, (want.abs() - end).abs() < bound
    assert (torch.isinf(y[big]) & (torch.sign(y[big]) == torch.sign(want[big]))).all()
    bad = ((y - want).abs() > bound) & ~big & ~(near & torch.isinf(y))
    assert not torch.isnan(y).any() and not bad.any(), (int(bad.sum()), bad.nonzero()[:4].tolist())


@pytest.mark.parametrize("M,N,Kd", SIZES)
@pytest.mark.parametrize("sa,sw", [(1e-30, 1.3e-13), (1.3e-13, 1e-30), (1.7e-22, 1.1e-22), (3e-42, 1.5), (1e-40, 1e20), (1e30, 1e10), (2e36, 2e36), (1.0, 1e-45)])
def test_products_of_scales_out_of_range(K, M, N, Kd, sa, sw):
    gen = torch.Generator().manual_seed(M + N)
    a, w = _rows(gen, M, Kd), _rows(gen, N, Kd)
    ta, tw = torch.full((M,), sa).cuda(), torch.full((N,), sw).cuda()
    # rows and channels with ordinary scales lie between them, and some of nothing
    ta[::3], tw[::4] = 0.03, 0.7
    a[::5] = 0
    w[1::7] = 0
    _check(K.gemm_i8(a, ta, w, tw), a, ta, w, tw, None)
    bias = torch.randn(N, generator=gen).cuda()
    y = K.gemm_i8(a, ta, w, tw, bias=bias)
    _check(y, a, ta, w, tw, bias)
    assert torch.equal(y[::5], bias.expand(len(y[::5]), N)) and torch.equal(y[:, 1::7], bias[1::7].expand(M, -1))         # a sum of nothing is the bias
    assert torch.equal(K.gemm_i8(a, ta, w, tw, bias=bias, relu=True), y.clamp_min(0))


@pytest.mark.parametrize("M", [1, 3, 7, 16, 40, 300])
def test_tokens_and_channels_of_extreme_size(K, M):
    gen = torch.Generator().manual_seed(M)
    x, w = torch.randn(M, 200, generator=gen), torch.randn(70, 200, generator=gen)
    for sx, sw in ((1e-22, 1e-20), (1e30, 1e12), (1e-37, 1e10), (1e35, 1e-36)):
        xs, ws = (x * sx).cuda(), (w * sw).cuda()
        xs[M // 2] = 0.0
        codes, scale = K.quantize_rows(ws)
        q, t = K.quantize_rows(xs)
        y = K.linear_i8(xs, codes, scale)
        _check(y, q, t, codes, scale, None)
        assert (y[M // 2] == 0).all()


def test_scales_that_are_no_numbers(K):
    gen = torch.Generator().manual_seed(1)
    for M in (5, 200):
        a, w = _rows(gen, M, 100), _rows(gen, 70, 100)
        sa, sw = torch.ones(M).cuda(), torch.ones(70).cuda()
        sa[1], sw[2], sw[3] = float("nan"), float("inf"), 0.0
        a[2] = 0
        y = K.gemm_i8(a, sa, w, sw).cpu()
        want = ((a.cpu().double() @ w.cpu().double().t()) * sa.cpu().double()[:, None] * sw.cpu().double()).float()
        assert torch.equal(torch.isnan(y), torch.isnan(want)) and torch.equal(y[~torch.isnan(y)], want[~torch.isnan(want)])
