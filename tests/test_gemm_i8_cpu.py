"""Products in 8-bit integers: what the entry points refuse before anything is launched."""
import pytest
import torch

from controllable_agent_amd import _lib, kernels as K


def _codes(rows, k, ld=None):
    return torch.zeros(rows, ld or (k + 15) // 16 * 16, dtype=torch.int8)[:, :k]


def test_code_matrices_that_are_refused():
    s = torch.ones(4)
    good = _codes(4, 20)
    assert K._code_rows(good, s, "A") == (4, 20, 32)
    assert K._code_rows(_codes(1, 5), torch.ones(1), "A")[:2] == (1, 5)
    buf = torch.zeros(4 * 32 + 16, dtype=torch.int8)
    off = (-buf.data_ptr()) % 16
    aligned = buf[off:off + 128].view(4, 32)
    bad = [good.float(), good[0], torch.zeros(4, 20, dtype=torch.int8), torch.zeros(20, 32, dtype=torch.int8).t()[:4], aligned[:, 1:21],
           torch.zeros(16 * 3 + 5, dtype=torch.int8).as_strided((4, 5), (16, 1))]           # the last row's 16 bytes are not there
    for q in bad:
        with pytest.raises(ValueError):
            K._code_rows(q, s, "A")
    for scale in (torch.ones(3), torch.ones(4, dtype=torch.float64), torch.ones(8)[::2], torch.ones(4, 1)):
        with pytest.raises(ValueError):
            K._code_rows(good, scale, "A")


def test_float_matrices_that_are_refused():
    assert K._float_rows(torch.zeros(3, 7), "x") == (3, 7, 7, 0) and K._float_rows(torch.zeros(1, 7)[:, :5], "x") == (1, 5, 5, 0)
    for x in (torch.zeros(3), torch.zeros(3, 7).t(), torch.zeros(3, 7, dtype=torch.float64), torch.zeros(1, 7).expand(3, 7), torch.zeros(3, 8)[:, ::2]):
        with pytest.raises(ValueError):
            K._float_rows(x, "x")


def test_outputs_that_are_refused():
    buf = torch.zeros(200)
    x, bias = buf[:60].view(3, 20), buf[100:105]
    cpu = x.device
    assert K._i8_output(buf[60:75].view(3, 5), None, 3, 5, cpu, bias, (x,))[1] == 5
    for out in (buf[59:74].view(3, 5), buf[96:111].view(3, 5), torch.zeros(5, 3), torch.zeros(3, 10)[:, ::2], torch.zeros(1, 5).expand(3, 5)):
        with pytest.raises(ValueError):
            K._i8_output(out, None, 3, 5, cpu, bias, (x,))
    for b in (torch.zeros(4), torch.zeros(5, dtype=torch.float64), torch.zeros(10)[::2]):
        with pytest.raises(ValueError):
            K._i8_output(None, torch.float32, 3, 5, cpu, b, (x,))
    with pytest.raises(ValueError):
        K._i8_output(None, torch.int8, 3, 5, cpu, None, (x,))


def test_host_tensors_are_refused():
    x = torch.zeros(4, 20)
    q, s = _codes(4, 20), torch.ones(4)
    with pytest.raises((ValueError, RuntimeError)):
        K.quantize_rows(x)
    with pytest.raises((ValueError, RuntimeError)):
        K.gemm_i8(q, s, q, s)
    with pytest.raises((ValueError, RuntimeError)):
        K.linear_i8(x, q, s)


def test_c_entries_refuse_bad_calls():
    lib = _lib.load()
    ok = dict(a=16, lda=20000, sa=16, w=16, ldw=20000, sw=16, bias=None, relu=0, y=16, ldy=4, yt=0, M=400, N=4, K=20000, ws=16)

    def gemm(**kw):
        d = dict(ok, **kw)
        return lib.fbhip_gemm_i8(d["a"], d["lda"], d["sa"], d["w"], d["ldw"], d["sw"], d["bias"], d["relu"], d["y"], d["ldy"], d["yt"], d["M"], d["N"],
                                 d["K"], d["ws"], None)
    for kw in (dict(a=None), dict(sa=None), dict(w=None), dict(sw=None), dict(y=None), dict(M=0), dict(N=0), dict(K=0), dict(K=131072, lda=131072, ldw=131072),
               dict(a=8), dict(w=8), dict(lda=20004), dict(ldw=20004), dict(lda=19984), dict(ldw=19984), dict(ldy=3), dict(ws=None), dict(ws=8), dict(yt=3), dict(yt=-1),
               dict(ldw=1 << 24), dict(lda=1 << 24), dict(M=2 ** 31 - 1, N=2 ** 31 - 1, ldy=2 ** 31)):
        assert gemm(**kw) == -1 and lib.fbhip_last_error(None), kw
    def lin(x=16, ldx=20000, xt=0, ws=16, **kw):
        d = dict(ok, **kw)
        return lib.fbhip_linear_i8(x, ldx, xt, d["w"], d["ldw"], d["sw"], None, 0, d["y"], d["ldy"], d["yt"], d["M"], d["N"], d["K"], ws, None)
    assert all(r == -1 for r in (lin(x=None), lin(ldx=19999), lin(xt=3), lin(ws=None), lin(ws=8), lin(w=None), lin(K=0)))

    def quant(x=16, ldx=20, xt=0, q=16, ldq=32, s=16, rows=4, k=20, kp=32):
        return lib.fbhip_quantize_rows(x, ldx, xt, q, ldq, s, rows, k, kp, None)
    assert all(r == -1 for r in (quant(x=None), quant(q=None), quant(s=None), quant(rows=0), quant(k=0), quant(kp=19), quant(ldq=31), quant(ldx=19),
                                 quant(xt=5)))
    assert lib.fbhip_linear_i8_workspace(40, 4, 20) >= 40 * 128 + 160 and lib.fbhip_linear_i8_workspace(0, 4, 20) == 0
    # few tokens whose values fit one launch: it needs none
    for tokens, most in ((1, 16384), (2, 8192), (3, 4096), (4, 4096), (5, 2048), (8, 2048), (9, 1024), (16, 1024)):
        assert lib.fbhip_linear_i8_workspace(tokens, 4, most) == 0 and lib.fbhip_linear_i8_workspace(tokens, 4, most + 1) > 0
    assert lib.fbhip_linear_i8_workspace(17, 4, 16) > 0
