"""Products in 8-bit integers against 64-bit arithmetic.

The codes are whole numbers and have to be equal.  The sum is exact; the output takes the sum's conversion to float32, two products with the
scales and the addition of the bias: four roundings of half a step (e = 2^-24) of terms no larger than |sum sa sw| + |bias|, then half a step of the
output's type (bf16 2^-9 relative to the value's power of two, that is 2^-8 of the value at most; fp16 2^-11, or 2^-25 below its normal range).
"""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
E = 2.0 ** -24
HALF = {torch.float32: 0.0, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}


@pytest.fixture(scope="module")
def K():
    from controllable_agent_amd import kernels
    return kernels


def _codes(gen, rows, k, junk=True, extra=0):
    """random codes on padded rows; what lies behind K is not zero"""
    ld = (k + 15) // 16 * 16 + extra
    buf = torch.randint(-127, 128, (rows, ld), generator=gen, dtype=torch.int8)
    if not junk:
        buf[:, k:] = 0
    return buf.cuda()[:, :k]


def _check(y, a, sa, w, sw, bias, relu, dtype):
    acc = a.cpu().double() @ w.cpu().double().t()
    main = acc * sa.cpu().double()[:, None] * sw.cpu().double()
    want = main if bias is None else main + bias.cpu().double()
    err = 4 * E * (main.abs() + (0 if bias is None else bias.cpu().double().abs()))
    if relu:
        want = want.clamp_min(0)
    assert y.dtype == dtype and y.shape == want.shape
    bound = err + HALF[dtype] * (want.abs() + err) + (2.0 ** -25 if dtype == torch.float16 else 0.0)
    bad = (y.cpu().double() - want).abs() > bound
    assert not bad.any(), (int(bad.sum()), bad.nonzero()[:4].tolist())


# the tiles' borders (16, 32, 64, 128, 256) and their neighbours; one token; layers of the agents' networks; uneven K
SIZES = [(1, 1, 1), (1, 6, 24), (1, 1024, 1024), (2, 50, 1024), (2, 8200, 1500), (1, 20000, 70), (3, 17, 130), (4, 4100, 1025), (4, 300, 17000), (4, 1000, 77), (5, 64, 128), (15, 16, 127), (16, 33, 129), (17, 526, 526), (31, 100, 256),
         (33, 65, 97), (63, 63, 4096), (64, 64, 384), (65, 70, 1000), (64, 6, 8191), (127, 129, 255), (128, 128, 512), (200, 300, 1051), (256, 256, 128), (257, 255, 640),
         (300, 1024, 74), (777, 526, 1051), (1000, 2048, 1024), (1024, 2048, 30), (2500, 1300, 333)]


@pytest.mark.parametrize("M,N,Kd", SIZES)
def test_sizes(K, M, N, Kd):
    gen = torch.Generator().manual_seed(M * 7 + N * 3 + Kd)
    a, w = _codes(gen, M, Kd), _codes(gen, N, Kd, extra=16 * (Kd % 3))
    sa, sw = (torch.rand(M, generator=gen) + 0.1).cuda(), (torch.rand(N, generator=gen) + 0.1).cuda()
    _check(K.gemm_i8(a, sa, w, sw), a, sa, w, sw, None, False, torch.float32)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("relu", [False, True])
@pytest.mark.parametrize("with_bias", [False, True])
@pytest.mark.parametrize("M,N,Kd", [(1, 70, 200), (3, 130, 640), (20, 51, 200), (150, 131, 300), (1030, 1500, 260)])
def test_epilogue(K, M, N, Kd, with_bias, relu, dtype):
    gen = torch.Generator().manual_seed(1)
    a, w = _codes(gen, M, Kd), _codes(gen, N, Kd)
    sa, sw = (torch.rand(M, generator=gen) * 1e-2).cuda(), (torch.rand(N, generator=gen) * 1e-2).cuda()
    bias = torch.randn(N, generator=gen).cuda() if with_bias else None
    _check(K.gemm_i8(a, sa, w, sw, bias=bias, relu=relu, out_dtype=dtype), a, sa, w, sw, bias, relu, dtype)


def test_scales_of_opposite_sizes(K):
    """the product of the scales is in range where neither scale times the sum would be"""
    gen = torch.Generator().manual_seed(9)
    for M in (3, 40, 300):
        a, w = _codes(gen, M, 500), _codes(gen, 70, 500)
        sa, sw = torch.full((M,), 1e36, device="cuda"), torch.full((70,), 1e-32, device="cuda")
        _check(K.gemm_i8(a, sa, w, sw), a, sa, w, sw, None, False, torch.float32)
        _check(K.gemm_i8(a, sw[:1].expand(M).contiguous(), w, sa[:1].expand(70).contiguous()), a, sw[:1].expand(M), w, sa[:1].expand(70), None, False,
               torch.float32)


@pytest.mark.parametrize("M,N,Kd", [(1, 40, 131071), (40, 24, 131071), (1, 2100, 131071), (300, 200, 16384)])
@pytest.mark.parametrize("code", [127, -128])
def test_largest_sums(K, M, N, Kd, code):
    """all codes of the largest magnitude: the sums reach 128^2 K = 2^31 - 16384 at the largest K"""
    full = lambda r: torch.full((r, (Kd + 15) // 16 * 16), code, dtype=torch.int8, device="cuda")[:, :Kd]  # noqa: E731
    a, w = full(M), full(N)
    w[1::2] = 127
    one = lambda n: torch.ones(n, device="cuda")  # noqa: E731
    y = K.gemm_i8(a, one(M), w, one(N)).double()
    even, odd = float(code * code * Kd), float(code * 127 * Kd)
    assert ((y[:, 0::2] - even).abs() <= E * abs(even)).all() and ((y[:, 1::2] - odd).abs() <= E * abs(odd)).all()


@pytest.mark.parametrize("M,N,Kd", [(1, 37, 100), (7, 37, 100), (100, 37, 100), (700, 600, 100)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_given_output_rows_and_what_lies_around_them(K, M, N, Kd, dtype):
    gen = torch.Generator().manual_seed(2)
    a, w = _codes(gen, M, Kd), _codes(gen, N, Kd)
    sa, sw = torch.rand(M, generator=gen).cuda(), torch.rand(N, generator=gen).cuda()
    for ld, start in ((N, 0), (N + 3, 0), (N + 8, 1), (N + 11, 4)):
        buf = torch.full((M + 2, ld + start), 7.0, device="cuda", dtype=dtype)
        out = buf[1:M + 1, start:start + N]
        got = K.gemm_i8(a, sa, w, sw, out=out)
        assert got is out
        _check(out, a, sa, w, sw, None, False, dtype)
        keep = torch.ones_like(buf, dtype=torch.bool)
        keep[1:M + 1, start:start + N] = False
        assert (buf[keep] == 7.0).all()


# --------------------------------------------------------------------------------------------------------------------------- quantiser
def _want_codes(x):
    """scale: the product with the float32 nearest to 1/127, in float32; quotient rounded to float32, nearest whole number, ties to even"""
    x = x.cpu().float()
    top = x.abs().amax(1)
    s = (top.double() * float(torch.tensor(1 / 127, dtype=torch.float32))).float()
    q = (x.double() / s.double().clamp_min(1e-300)[:, None]).float().round().clamp(-127, 127)
    return torch.where(s[:, None] > 0, q, torch.zeros_like(q)).to(torch.int8), s


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("rows,k", [(1, 1), (3, 7), (5, 64), (4, 255), (33, 256), (9, 1051), (2, 4096), (7, 8195), (2, 40000), (1500, 300)])
def test_quantize_rows(K, rows, k, dtype):
    gen = torch.Generator().manual_seed(rows + k)
    x = (torch.randn(rows, k, generator=gen) * torch.exp(2 * torch.randn(rows, 1, generator=gen))).to(dtype).cuda()
    want, s = _want_codes(x)
    for view in (x, torch.cat([x, x], 1)[:, :k], torch.cat([x[:, :1], x], 1)[:, 1:]):       # other strides, rows off their alignment
        q, scale = K.quantize_rows(view)
        assert torch.equal(scale.cpu(), s) and torch.equal(q.cpu(), want)
        full = q.as_strided((rows, q.stride(0)), (q.stride(0), 1)) if rows > 1 else q
        assert q.stride(0) % 128 == 0 and (full[:, k:] == 0).all()


def test_quantize_ties_and_extremes(K):
    """halves go to the even neighbour; the row's largest values become 127; tiny and huge rows; zeros"""
    x = torch.zeros(9, 300)
    x[0, :255] = torch.arange(-127, 128) + 0.0
    x[0, 255:] = torch.arange(45) + 0.5                       # scale 1: quotients are the values
    x[1, :2] = torch.tensor([3.4e38, -3.4e38])
    x[2, :3] = torch.tensor([1e-38, -1e-38, 5e-39])
    x[3, :2] = torch.tensor([1e-45, -1e-45])                    # scale underflows to 0
    x[4] = torch.linspace(-1, 1, 300)
    x[5, 7] = -2.5
    x[6] = torch.randn(300, generator=torch.Generator().manual_seed(0)) * 1e30
    x[7] = 0.1
    q, s = K.quantize_rows(x.cuda())
    want, ws = _want_codes(x)
    assert torch.equal(s.cpu(), ws) and torch.equal(q.cpu(), want)
    assert (q[3] == 0).all() and (q[8] == 0).all() and s[8] == 0 and q[1, 0] == 127 and q[1, 1] == -127 and q[5, 7] == -127


@pytest.mark.parametrize("rows", [1, 16, 400])
def test_codes_beside_the_halves(K, rows):
    """quotients within a few steps of a half, on scales from 2^-118 to 2^110: the code is the rounded quotient's, in the quantiser and in the product
    (127 times the identity hands the codes back: six roundings of half a step lie between them and code * scale, 4e-7; a wrong code is off by 1/127)"""
    gen = torch.Generator().manual_seed(rows)
    scale = torch.exp2(torch.rand(rows, 1, generator=gen) * 228 - 118)
    half = (torch.randint(-127, 127, (rows, 255), generator=gen) + 0.5) * scale
    steps = torch.randint(-4, 5, half.shape, generator=gen, dtype=torch.int32)
    x = torch.cat([127 * scale, (half.view(torch.int32) + steps).view(torch.float32)], 1)
    q, s = K.quantize_rows(x.cuda())
    want, ws = _want_codes(x)
    assert torch.equal(s.cpu(), ws) and torch.equal(q.cpu(), want)
    eye, one = K.quantize_rows(torch.eye(256, device="cuda") * 127)
    y = K.linear_i8(x.cuda(), eye, one / 127)
    assert torch.allclose(y.cpu().double() / ws.double()[:, None], want.double(), rtol=1e-5, atol=0)


@pytest.mark.parametrize("M", [1, 2, 3, 7, 16, 20, 200])
@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
def test_rows_that_hold_no_numbers(K, M, bad):
    """they come back as NaN, whatever the others hold; rows of zeros give the bias"""
    gen = torch.Generator().manual_seed(3)
    x, w = torch.randn(M, 300, generator=gen), torch.randn(70, 300, generator=gen)
    good = x.clone()
    x[M // 2, 17] = bad
    wq, ws = K.quantize_rows(w.cuda())
    bias = torch.randn(70, generator=gen).cuda()
    for relu in (False, True):
        y, ref = K.linear_i8(x.cuda(), wq, ws, bias=bias, relu=relu), K.linear_i8(good.cuda(), wq, ws, bias=bias, relu=relu)
        assert torch.isnan(y[M // 2]).all()
        rest = torch.arange(M) != M // 2
        assert torch.equal(y.cpu()[rest], ref.cpu()[rest])
    q, s = K.quantize_rows(x.cuda())
    assert torch.isnan(s[M // 2]) and (q[M // 2] == 0).all()
    y = K.linear_i8(torch.zeros(M, 300, device="cuda"), wq, ws, bias=bias)
    assert torch.equal(y, bias.expand(M, 70))


# ------------------------------------------------------------------------------------------------------------------------------ linear
@pytest.mark.parametrize("M", [1, 2, 3, 4, 5, 8, 9, 13, 16, 17, 48, 64, 65, 300])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("N,Kd", [(6, 30), (526, 1051), (1024, 1024), (64, 8200), (40, 33000), (20, 2048), (33, 4097)])
def test_linear_equals_quantize_then_product(K, M, N, Kd, dtype):
    gen = torch.Generator().manual_seed(M + N)
    x = torch.randn(M, Kd, generator=gen).to(dtype).cuda()
    w = torch.randn(N, Kd, generator=gen).cuda()
    bias = torch.randn(N, generator=gen).cuda()
    wq, ws = K.quantize_rows(w)
    want, s = _want_codes(x)
    y = K.linear_i8(x, wq, ws, bias=bias)
    _check(y, want, s, wq, ws, bias, False, dtype)
    # a column slice of a wider matrix, its rows off their alignment, and a given output type
    wide = torch.cat([x[:, :3], x, x[:, :2]], 1)[:, 3:3 + Kd]
    _check(K.linear_i8(wide, wq, ws, relu=True, out_dtype=torch.float32), want, s, wq, ws, None, True, torch.float32)


def test_linear_is_near_the_float_product(K):
    """A walker-sized layer.  Each code is off by at most half a step of its row: |x - s q| <= s/2, |w - t r| <= t/2, so that an output is off by at
    most sum_k (s/2 |w| + t/2 |x| + s t / 4)."""
    gen = torch.Generator().manual_seed(4)
    x, w = torch.randn(300, 1024, generator=gen), torch.randn(512, 1024, generator=gen) / 32
    wq, ws = K.quantize_rows(w.cuda())
    y = K.linear_i8(x.cuda(), wq, ws).cpu().double()
    s, t = x.abs().amax(1).double() / 127, ws.cpu().double()
    xd, wd = x.double(), w.double()
    bound = s[:, None] / 2 * wd.abs().sum(1) + t / 2 * xd.abs().sum(1, keepdim=True) + 1024 * s[:, None] * t / 4
    assert ((y - xd @ wd.t()).abs() <= bound * (1 + 1e-5)).all()


def test_empty_sides(K):
    q = torch.zeros(0, 32, dtype=torch.int8, device="cuda")
    w, s = torch.zeros(5, 32, dtype=torch.int8, device="cuda"), torch.ones(5, device="cuda")
    none = torch.zeros(0, device="cuda")
    assert K.gemm_i8(q, none, w, s).shape == (0, 5) and K.gemm_i8(w, s, q, none).shape == (5, 0)
    assert K.linear_i8(torch.zeros(0, 32, device="cuda"), w, s).shape == (0, 5)
    codes, scale = K.quantize_rows(torch.zeros(0, 7, device="cuda"))
    assert codes.shape == (0, 7) and scale.shape == (0,)


def test_refusals_on_the_device(K):
    x = torch.zeros(4, 20, device="cuda")
    w, s = K.quantize_rows(torch.zeros(6, 20, device="cuda"))
    v, t = K.quantize_rows(torch.zeros(6, 21, device="cuda"))
    for call in (lambda: K.linear_i8(x, v, t), lambda: K.gemm_i8(w, s, v, t), lambda: K.linear_i8(x, w, s, bias=torch.zeros(5, device="cuda")),
                 lambda: K.linear_i8(x, w, s, bias=torch.zeros(6)), lambda: K.linear_i8(x, w, s, out=torch.zeros(4, 5, device="cuda")),
                 lambda: K.linear_i8(x, w, s, out_dtype=torch.float64), lambda: K.linear_i8(x, w, s, out=torch.zeros(6, 4, device="cuda").t()),
                 lambda: K.linear_i8(x.cpu(), w, s), lambda: K.linear_i8(x, w[:, :20], s, out=x[:, :6]), lambda: K.linear_i8(x, w, s, out=torch.zeros(1, 6, device="cuda").expand(4, 6))):
        with pytest.raises(ValueError):
            call()
    with pytest.raises(RuntimeError, match="FBHIP_I8_MAX_K"):
        z = torch.zeros(1, 131072, dtype=torch.int8, device="cuda")
        K.gemm_i8(z, torch.ones(1, device="cuda"), z, torch.ones(1, device="cuda"))


# ------------------------------------------------------------------------------------------------------------------------------ its use
@pytest.mark.parametrize("M,N,Kd", [(1, 300, 512), (6, 300, 4096), (64, 200, 4096), (300, 300, 512)])
def test_captured_on_another_stream_and_replayed(K, M, N, Kd):
    gen = torch.Generator().manual_seed(5)
    xs = [torch.randn(M, Kd, generator=gen).cuda() for _ in range(4)]
    wq, ws = K.quantize_rows(torch.randn(N, Kd, generator=gen).cuda())
    eager = [K.linear_i8(x, wq, ws) for x in xs]
    x = xs[0].clone()
    torch.cuda.synchronize()
    graph, other = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = K.linear_i8(x, wq, ws)
        q, s = K.quantize_rows(y)
    with torch.cuda.graph(other):
        z = K.linear_i8(x, wq, ws, relu=True)
    for k, src in enumerate(xs + xs):
        x.copy_(src)
        graph.replay()
        other.replay()
        assert torch.equal(y, eager[k % 4]) and torch.equal(z, eager[k % 4].clamp_min(0))
        assert torch.equal(K.quantize_rows(eager[k % 4])[0], q)
        torch.cuda.synchronize()


def test_two_streams_at_once(K):
    gen = torch.Generator().manual_seed(6)
    wq, ws = K.quantize_rows(torch.randn(512, 2048, generator=gen).cuda())
    xs = [torch.randn(40, 2048, generator=gen).cuda() for _ in range(2)]
    want = [K.linear_i8(x, wq, ws) for x in xs]
    streams = [torch.cuda.Stream() for _ in xs]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(8):
        for i, st in enumerate(streams):
            with torch.cuda.stream(st):
                got[i].append(K.linear_i8(xs[i], wq, ws))
    torch.cuda.synchronize()
    assert all(torch.equal(y, want[i]) for i in range(2) for y in got[i])


def test_rows_far_apart(K):
    """row offsets beyond 2^32 bytes on both operands and on the output"""
    ld = 1 << 23
    a = torch.zeros(600, ld, dtype=torch.int8, device="cuda")[:, :200]
    gen = torch.Generator().manual_seed(7)
    a.copy_(torch.randint(-127, 128, (600, 200), generator=gen, dtype=torch.int8))
    s = torch.rand(600, generator=gen).cuda()
    out = torch.zeros(600, ld, dtype=torch.float32, device="cuda")[:, :600]
    K.gemm_i8(a, s, a, s, out=out)
    _check(out, a, s, a, s, None, False, torch.float32)
    few = torch.zeros(3, 1 << 23, dtype=torch.int8, device="cuda")[:, :200]
    few.copy_(a[:3])
    _check(K.gemm_i8(few, s[:3], a, s), few, s[:3], a, s, None, False, torch.float32)


def test_train_then_serve(K):
    """The operators together: a two-layer network trained with 8-bit moments, its weights quantised by channel, its answers from 8-bit products.  The
    bound is the quantisation's own, layer by layer (half a step of each operand), with the first layer's error carried through |w|."""
    from controllable_agent_amd import AdamW
    gen = torch.Generator().manual_seed(8)
    x, t = torch.randn(256, 30, generator=gen).cuda(), torch.randn(256, 6, generator=gen).cuda()
    p = [(torch.randn(s, generator=gen) * 0.2).cuda().requires_grad_(True) for s in ((64, 30), (64,), (6, 64), (6,))]
    opt = AdamW(p, lr=1e-2, state_bits=8, weight_decay=[0.01, 0.0, 0.01, 0.0])
    for _ in range(20):
        loss = (torch.relu(x @ p[0].t() + p[1]) @ p[2].t() + p[3] - t).square().mean()
        norm = opt.step(torch.autograd.grad(loss, p), max_norm=1.0)
    assert opt.step_count == 20 and math.isfinite(float(norm)) and all(torch.isfinite(q).all() for q in p)
    w1, b1, w2, b2 = (q.detach() for q in p)
    (q1, s1), (q2, s2) = K.quantize_rows(w1), K.quantize_rows(w2)
    h = K.linear_i8(x, q1, s1, bias=b1, relu=True)
    y = K.linear_i8(h, q2, s2, bias=b2)

    def bound(a, w, s, carried):
        sa = a.abs().amax(1, keepdim=True) / 127 + carried.amax(1, keepdim=True) / 127
        return carried @ w.abs().t() + sa / 2 * w.abs().sum(1) + s / 2 * (a.abs() + carried).sum(1, keepdim=True) + a.shape[1] * sa * s / 4
    xd, w1, b1, w2, b2, s1, s2 = (v.double() for v in (x, w1, b1, w2, b2, s1, s2))
    hd = torch.relu(xd @ w1.t() + b1)
    e1 = bound(xd, w1, s1, torch.zeros_like(xd))
    assert ((h.double() - hd).abs() <= e1 * 1.00001).all()
    e2 = bound(hd, w2, s2, e1)
    assert ((y.double() - (hd @ w2.t() + b2)).abs() <= e2 * 1.00001).all()
