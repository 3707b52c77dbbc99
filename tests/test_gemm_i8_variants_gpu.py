"""Every kernel that the 8-bit product launches, on both sides of each border of the choice between them: ragged edges, the end of K, bias, ReLU, each
output type, outputs with their own row stride and what lies around them.

The sum is exact; its conversion, two products with the scales and the addition of the bias are four roundings of half a step (e = 2^-24) of terms no
larger than |sum sa sw| + |bias|, then half a step of the output's type (bf16 2^-8, fp16 2^-11 of the value, 2^-25 below its normal range).  That every
kernel is among these sizes is checked on the CPU (test_launch_paths_cpu.py)."""
import pytest
import torch

pytestmark = pytest.mark.gpu
E = 2.0 ** -24
HALF = {torch.float32: 0.0, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
SIZES = [
    # strips of 16 channels: 16, 32 and 64 tokens
    (1, 33, 100), (16, 500, 1999), (17, 100, 130), (32, 526, 1051), (33, 70, 128), (64, 4096, 500),
    # strips of 32 channels from 8192 channels on: 32 and 64 tokens; below, and with more than 32 MB of weights, others take over
    (17, 8192, 128), (20, 8200, 130), (31, 8195, 77), (32, 8192, 4096), (32, 8191, 64), (33, 8200, 1000), (63, 8197, 333), (64, 8192, 300), (64, 8193, 4097),
    # 64 x 64 tiles: four steps deep, two steps deep; K split over workgroups (few channels with a long K among them)
    (65, 65, 64), (200, 300, 16), (1400, 1400, 96), (1500, 1500, 200), (1472, 1480, 1999), (300, 200, 4100), (65, 64, 4096), (16, 300, 17000), (3, 5, 20000),
    # 128 x 128 tiles from 192 of them on
    (1500, 2000, 300), (2500, 1301, 333), (1408, 2305, 128), (2049, 1537, 1030),
    # 256 x 256 tiles from 192 of them on
    (3000, 4000, 40), (3600, 3500, 130), (3329, 3841, 128), (2500, 5001, 1999), (2800, 4300, 257), (4097, 3841, 256),
]


@pytest.fixture(scope="module")
def K():
    from controllable_agent_amd import kernels
    return kernels


def _codes(gen, rows, k, extra=0):
    """random codes (-128 among them) on padded rows; what lies behind K is not zero"""
    return torch.randint(-128, 128, (rows, (k + 15) // 16 * 16 + extra), generator=gen, device="cuda", dtype=torch.int8)[:, :k]


def _sums(a, w):
    """exact: 1000 products of 2^14 stay below 2^24"""
    return sum((a[:, k:k + 1000].float() @ w[:, k:k + 1000].float().t()).double() for k in range(0, a.shape[1], 1000))


def _bad(y, sums, sa, sw, bias, relu):
    main = sums * sa.double()[:, None] * sw.double()
    want = main if bias is None else main + bias.double()
    err = 4 * E * (main.abs() + (0 if bias is None else bias.double().abs()))
    if relu:
        want = want.clamp_min(0)
    bound = err + HALF[y.dtype] * (want.abs() + err) + (2.0 ** -25 if y.dtype == torch.float16 else 0.0)
    return int(((y.double() - want).abs() > bound).sum()) + int(torch.isnan(y).sum())


@pytest.mark.parametrize("M,N,Kd", SIZES)
def test_every_kernel(K, M, N, Kd):
    gen = torch.Generator(device="cuda").manual_seed(M * 7 + N * 3 + Kd)
    a, w = _codes(gen, M, Kd, 16 * (Kd % 2)), _codes(gen, N, Kd, 16 * (Kd % 3))
    sums = _sums(a, w)
    rand = lambda n: torch.rand(n, generator=gen, device="cuda")  # noqa: E731
    # products of the order of 1 (fp16 has to hold them), whatever K is
    sa, sw = (rand(M) + 0.1) * 0.01, (rand(N) + 0.1) * 0.01 / Kd ** 0.5
    bias = torch.randn(N, generator=gen, device="cuda")
    assert _bad(K.gemm_i8(a, sa, w, sw), sums, sa, sw, None, False) == 0
    for dtype, b, relu, extra, start in ((torch.bfloat16, bias, True, 3, 1), (torch.float16, None, False, 8, 0), (torch.float32, bias, False, 1, 3)):
        buf = torch.full((M + 2, N + start + extra), 7.0, device="cuda", dtype=dtype)
        out = buf[1:M + 1, start:start + N]
        assert K.gemm_i8(a, sa, w, sw, bias=b, relu=relu, out=out) is out
        assert _bad(out, sums, sa, sw, b, relu) == 0
        out.fill_(7.0)
        assert bool((buf == 7.0).all())                                   # nothing else was written


@pytest.mark.parametrize("M,N,Kd", [(16, 8200, 1024), (40, 8200, 300), (64, 526, 1051), (1400, 1300, 200), (2500, 1301, 333), (3600, 3500, 130), (300, 200, 4100)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_quantised_on_the_way(K, M, N, Kd, dtype):
    gen = torch.Generator(device="cuda").manual_seed(M + N)
    x = torch.randn(M, Kd + 5, generator=gen, device="cuda").to(dtype)[:, 3:3 + Kd]
    w, sw = K.quantize_rows(torch.randn(N, Kd, generator=gen, device="cuda"))
    bias = torch.randn(N, generator=gen, device="cuda")
    q, s = K.quantize_rows(x)
    assert torch.equal(K.linear_i8(x, w, sw, bias=bias, relu=True), K.gemm_i8(q, s, w, sw, bias=bias, relu=True, out_dtype=dtype))


def test_more_rows_than_one_launch_takes(K):
    """2^26 + 5 rows of three values: a wave for each would be 2^32 threads and more"""
    rows = (1 << 26) + 5
    gen = torch.Generator(device="cuda").manual_seed(3)
    x = torch.randn(rows, 3, generator=gen, device="cuda")
    q, s = K.quantize_rows(x)
    assert torch.equal(s, x.abs().amax(1) * torch.tensor(1 / 127, device="cuda"))
    full = q.as_strided((rows, 128), (128, 1))
    for r in [0, rows - 1000] + [k * (1 << 23) - 500 for k in range(1, 9)]:
        some, t = K.quantize_rows(x[r:r + 1000])
        assert torch.equal(full[r:r + 1000], some.as_strided((len(some), 128), (128, 1))) and torch.equal(s[r:r + 1000], t), r
    assert bool((full[:, :3].abs().amax(1) == 127).all())


@pytest.mark.parametrize("M", [1, 16, 40])
def test_more_channels_than_a_launch_of_strips_takes(K, M):
    N = (1 << 26) + 1
    gen = torch.Generator(device="cuda").manual_seed(M)
    w = _codes(gen, N, 16)
    sw = torch.rand(N, generator=gen, device="cuda")
    x = torch.randn(M, 16, generator=gen, device="cuda")
    q, s = K.quantize_rows(x)
    y = K.linear_i8(x, w, sw)
    assert torch.equal(K.gemm_i8(q, s, w, sw), y)
    for n in (0, 1 << 25, N - 5000):
        assert _bad(y[:, n:n + 5000], _sums(q, w[n:n + 5000]), s, sw[n:n + 5000], None, False) == 0


@pytest.mark.parametrize("M,N,Kd", [(1, 64, 100), (16, 64, 1000), (40, 64, 1024), (300, 200, 500), (2500, 1301, 333)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_an_answer_beside_its_input(K, M, N, Kd, dtype):
    """input and output are columns of one buffer, as a layer that hands on both wants them"""
    gen = torch.Generator(device="cuda").manual_seed(M)
    w, sw = K.quantize_rows(torch.randn(N, Kd, generator=gen, device="cuda"))
    for before in (0, N):
        buf = torch.randn(M, Kd + N, generator=gen, device="cuda").to(dtype)
        x, out = buf[:, before:before + Kd], (buf[:, Kd:] if before == 0 else buf[:, :N])
        was = x.clone()
        want = K.linear_i8(x, w, sw)
        assert K.linear_i8(x, w, sw, out=out) is out and torch.equal(out, want) and torch.equal(x, was)
