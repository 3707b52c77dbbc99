"""Torch-tensor front-ends of the individually callable gfx950 kernels in libfbhip.so.

Each function takes CUDA(=HIP) float32 tensors, passes raw device pointers + leading dimensions over the
C ABI (include/fbhip.h) and launches on torch's current stream.  No arithmetic happens in Python.
"""
from __future__ import annotations

import typing as tp

import torch

from . import _lib
from ._lib import check, ptr, stream_ptr


def _ld(t: torch.Tensor) -> int:
    assert t.dtype == torch.float32 and t.is_cuda, "float32 device tensor expected"
    if t.dim() == 1:
        return t.shape[0]
    assert t.dim() == 2 and t.stride(1) == 1, "row-major 2-D tensor expected"
    return t.stride(0)


def gemm(A: torch.Tensor, B: torch.Tensor, *, a_kcontig: bool = True, b_kcontig: bool = True,
         bias: tp.Optional[torch.Tensor] = None, aux: tp.Optional[torch.Tensor] = None, epi: int = _lib.EPI_NONE,
         want_colsum: bool = False, out: tp.Optional[torch.Tensor] = None, cfg: tp.Optional[int] = None):
    """C[M,N] = epi(sum_k A(m,k) B(n,k)).  a_kcontig: A is [M,K] (else [K,M]); b_kcontig: B is [N,K] (else [K,N])."""
    _lib.require_device()
    M, K = (A.shape if a_kcontig else A.shape[::-1])
    N, K2 = (B.shape if b_kcontig else B.shape[::-1])
    assert K == K2, (A.shape, B.shape)
    Cm = out if out is not None else torch.empty((M, N), device=A.device, dtype=torch.float32)
    colsum = torch.zeros(M, device=A.device) if want_colsum else None
    lib = _lib.load()
    if cfg is not None:
        check(lib.fbhip_gemm_cfg(ptr(A), _ld(A), int(a_kcontig), ptr(B), _ld(B), int(b_kcontig), ptr(Cm), _ld(Cm),
                                 M, N, K, cfg, stream_ptr()))
        return Cm
    check(lib.fbhip_gemm(ptr(A), _ld(A), int(a_kcontig), ptr(B), _ld(B), int(b_kcontig), ptr(Cm), _ld(Cm), M, N, K,
                         ptr(bias), ptr(aux), 0 if aux is None else _ld(aux), epi, ptr(colsum), stream_ptr()))
    return (Cm, colsum) if want_colsum else Cm


def head(x: torch.Tensor, w: torch.Tensor, bias: torch.Tensor, *, normalize: bool = False, scale: float = 1.0, replicas: int = 1):
    """c = x @ w.T + bias for an embedding head (N <= 64) and, with ``normalize``, scale * c / |c|_row and the row norms
    (csrc/fused.hip).  bias must be readable up to pad4(N)."""
    _lib.require_device()
    rows, K = x.shape
    N = w.shape[0]
    ld = (N + 3) // 4 * 4
    c = torch.full((rows, ld), float("nan"), device=x.device)
    out2 = torch.full((rows, ld), float("nan"), device=x.device) if normalize else None
    norms = torch.empty(rows, device=x.device) if normalize else None
    check(_lib.load().fbhip_head(ptr(x), _ld(x), ptr(w), _ld(w), ptr(bias), ptr(c), ld, ptr(out2), ld, ptr(norms), scale, rows, N, K,
                                 replicas, stream_ptr()))
    return (c, out2, norms) if normalize else c


def ln_tanh_fwd(x: torch.Tensor, gamma: torch.Tensor, beta: torch.Tensor):
    """y = tanh(LayerNorm(x)), stats[rows,2] = (mean, rstd)   (fb_modules.py:49-50)."""
    _lib.require_device()
    rows, n = x.shape
    y = torch.empty((rows, n), device=x.device)
    stats = torch.empty((rows, 2), device=x.device)
    check(_lib.load().fbhip_ln_tanh_fwd(ptr(x), _ld(x), ptr(gamma), ptr(beta), ptr(y), _ld(y), ptr(stats), rows, n,
                                        stream_ptr()))
    return y, stats


def ln_tanh_bwd(dy, y, x, stats, gamma, want_param_grads: bool = True):
    _lib.require_device()
    rows, n = x.shape
    dx = torch.empty((rows, n), device=x.device)
    dg = torch.empty(n, device=x.device) if want_param_grads else None
    db = torch.empty(n, device=x.device) if want_param_grads else None
    part = torch.empty(((rows + 7) // 8) * 2 * n, device=x.device) if want_param_grads else None
    check(_lib.load().fbhip_ln_tanh_bwd(ptr(dy), _ld(dy), ptr(y), _ld(y), ptr(x), _ld(x), ptr(stats), ptr(gamma), ptr(dx),
                                        _ld(dx), ptr(dg), ptr(db), ptr(part), rows, n, stream_ptr()))
    return dx, dg, db


def l2norm_fwd(y: torch.Tensor):
    """sqrt(d) * F.normalize(y, dim=1) and the row norms."""
    _lib.require_device()
    rows, d = y.shape
    out = torch.empty((rows, d), device=y.device)
    norms = torch.empty(rows, device=y.device)
    check(_lib.load().fbhip_l2norm_fwd(ptr(y), _ld(y), ptr(out), _ld(out), ptr(norms), rows, d, stream_ptr()))
    return out, norms


def l2norm_bwd(dB, y, norms):
    _lib.require_device()
    rows, d = y.shape
    dy = torch.empty((rows, d), device=y.device)
    check(_lib.load().fbhip_l2norm_bwd(ptr(dB), _ld(dB), ptr(y), _ld(y), ptr(norms), ptr(dy), _ld(dy), rows, d,
                                       stream_ptr()))
    return dy


def pairwise_fb(F1, F2, Bm, tF1, tF2, tB, discount, ortho_coef: float):
    """FB + orthonormality loss and dF1, dF2, dB (fb_ddpg.py:313-348).  Returns (dF1, dF2, dB, metrics dict)."""
    _lib.require_device()
    Bn, d = F1.shape
    ld = _ld(F1)
    for t in (F2, Bm, tF1, tF2, tB):
        assert t.shape == F1.shape and _ld(t) == ld
    lib = _lib.load()
    # outputs share the inputs' leading dimension (one ``ld`` in the C ABI)
    dF1, dF2, dB = (torch.empty((Bn, ld), device=F1.device)[:, :d] for _ in range(3))
    metrics = torch.zeros(_lib.NUM_METRICS, device=F1.device)
    scratch = torch.empty(lib.fbhip_pairwise_scratch_floats(Bn, d), device=F1.device)
    disc = discount.reshape(-1).contiguous()
    check(lib.fbhip_pairwise_fb(ptr(F1), ptr(F2), ptr(Bm), ptr(tF1), ptr(tF2), ptr(tB), ptr(disc), Bn, d, ld,
                                float(ortho_coef), ptr(dF1), ptr(dF2), ptr(dB), ptr(metrics), ptr(scratch), stream_ptr()))
    m = metrics.cpu()
    names = ("fb_loss", "fb_offdiag", "fb_diag", "orth_loss", "orth_loss_diag", "orth_loss_offdiag", "target_M", "M1")
    return dF1, dF2, dB, {k: float(m[_lib.METRIC_INDEX[k]]) for k in names}


def pairwise_fb_block(F1, F2, Bm, tF1, tF2, tB, discount, ortho_coef: float, row_offset: int, rows: int):
    """Rows [row_offset, row_offset + rows) of ``pairwise_fb`` on the same panels: (dF1, dF2, dB) of those rows and this block's
    share of the scalars (fbhip_pairwise_fb_block; the global-batch data-parallel schedule)."""
    _lib.require_device()
    Bn, d = F1.shape
    ld = _ld(F1)
    for t in (F2, Bm, tF1, tF2, tB):
        assert t.shape == F1.shape and _ld(t) == ld
    lib = _lib.load()
    dF1, dF2, dB = (torch.empty((rows, ld), device=F1.device)[:, :d] for _ in range(3))
    metrics = torch.zeros(_lib.NUM_METRICS, device=F1.device)
    scratch = torch.empty(lib.fbhip_pairwise_scratch_floats(rows, d), device=F1.device)
    disc = discount.reshape(-1).contiguous()
    check(lib.fbhip_pairwise_fb_block(ptr(F1), ptr(F2), ptr(Bm), ptr(tF1), ptr(tF2), ptr(tB), ptr(disc), Bn, d, ld,
                                      float(ortho_coef), int(row_offset), int(rows), ptr(dF1), ptr(dF2), ptr(dB), ptr(metrics),
                                      ptr(scratch), stream_ptr()))
    m = metrics.cpu()
    names = ("fb_loss", "fb_offdiag", "fb_diag", "orth_loss", "orth_loss_diag", "orth_loss_offdiag", "target_M", "M1")
    return dF1, dF2, dB, {k: float(m[_lib.METRIC_INDEX[k]]) for k in names}


def adam_ema(params, grads, m, v, target, lr: float, t: int, grad_scale: float = 1.0, tau: float = 0.0) -> None:
    """In-place fused Adam (+ EMA into ``target`` when given) over flat tensors (numel % 4 == 0)."""
    _lib.require_device()
    check(_lib.load().fbhip_adam_ema(ptr(params), ptr(grads), ptr(m), ptr(v), ptr(target), params.numel(), float(lr),
                                     int(t), float(grad_scale), float(tau), stream_ptr()))


def inverse(A: torch.Tensor, scale: float = 1.0) -> torch.Tensor:
    """inverse(scale * A) of a [d, d] fp32 matrix (row stride >= d), 1 <= d <= 128."""
    _lib.require_device()
    d = A.shape[0]
    out = torch.empty((d, d), device=A.device)
    check(_lib.load().fbhip_inverse(ptr(A), A.stride(0), d, float(scale), ptr(out), d, stream_ptr()))
    return out


def actor_loss(F1, F2, z, mu, action, stddev: float):
    _lib.require_device()
    rows, d = F1.shape
    a = mu.shape[1]
    dF1, dF2 = (torch.empty((rows, _ld(F1)), device=F1.device)[:, :d] for _ in range(2))
    metrics = torch.zeros(_lib.NUM_METRICS, device=F1.device)
    scratch = torch.empty(3 * ((rows + 3) // 4), device=F1.device)
    check(_lib.load().fbhip_actor_loss(ptr(F1), ptr(F2), _ld(F1), ptr(z), _ld(z), ptr(mu), _ld(mu), ptr(action),
                                       _ld(action), float(stddev), ptr(dF1), ptr(dF2), ptr(metrics), ptr(scratch),
                                       rows, d, a, stream_ptr()))
    m = metrics.cpu()
    return dF1, dF2, {k: float(m[_lib.METRIC_INDEX[k]]) for k in ("actor_loss", "q", "actor_logprob", "q1_success")}


def policy_head(P, W4, b4, noise, stddev: float, clip: float, base=None, W1a=None, gamma=None, beta=None, keep_pre: bool = False):
    """(premu, mu, action[, t1, pre, stats]) of the policy head launch (csrc/rowops.hip row kernel or csrc/headtiles.hip MFMA tiles)."""
    _lib.require_device()
    rows, H = P.shape
    a = W4.shape[0]
    La = (a + 3) // 4 * 4
    premu, mu, action = (torch.zeros((rows, La), device=P.device) for _ in range(3))
    t1 = stats = pre = None
    if base is not None:
        pre = base.clone()
        t1 = torch.empty((rows, H), device=P.device)
        stats = torch.empty(2 * rows, device=P.device) if keep_pre else None
    check(_lib.load().fbhip_policy_head(ptr(P), _ld(P), ptr(W4), _ld(W4), ptr(b4), ptr(noise), float(stddev), float(clip), ptr(premu),
                                        ptr(mu), ptr(action), La, ptr(pre), 0 if pre is None else _ld(pre), ptr(W1a),
                                        0 if W1a is None else _ld(W1a), ptr(gamma), ptr(beta), ptr(t1), 0 if t1 is None else _ld(t1),
                                        ptr(stats), rows, H, a, stream_ptr()))
    return premu[:, :a], mu[:, :a], action[:, :a], t1, pre, stats


def actor_head_bwd(dt1, lnY, lnX, lnStats, lnGamma, W1a, mu, W4, P):
    """(d premu [rows, a], d p [rows, H]) of the actor's backward seam behind the LayerNorm + tanh backward."""
    _lib.require_device()
    rows, H = dt1.shape
    a = W4.shape[0]
    La = (a + 3) // 4 * 4
    dpremu = torch.zeros((rows, La), device=dt1.device)
    dp = torch.empty((rows, H), device=dt1.device)
    assert _ld(dt1) == _ld(lnY) == _ld(lnX) == _ld(P) == _ld(dp)
    check(_lib.load().fbhip_actor_head_bwd(ptr(dt1), _ld(dt1), ptr(lnY), ptr(lnX), ptr(lnStats), ptr(lnGamma), ptr(W1a), _ld(W1a), ptr(mu),
                                           _ld(mu), ptr(W4), _ld(W4), ptr(P), ptr(dpremu), La, ptr(dp), rows, H, a, stream_ptr()))
    return dpremu[:, :a], dp


# ------------------------------------------------------------------------------------------------------ products in 8-bit integers
_TYPE_CODE = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
_MOST = 2 ** 31 - 1024          # rows and columns that the entry points and the kernels' steps along a row count in 32 bits
_checked_devices: tp.Set[int] = set()


def _stream_on(t: torch.Tensor) -> int:
    """The current stream of ``t``'s device, which has to be the current device; the device itself is looked at once."""
    index = t.device.index
    if index is None or index != torch.cuda.current_device():
        raise ValueError(f"tensors on the current device expected, got {t.device}")
    if index not in _checked_devices:
        _lib.require_device()
        _checked_devices.add(index)
    return torch._C._cuda_getCurrentRawStream(index)          # (current_stream(index).cuda_stream without the stream object)


def _float_rows(x: torch.Tensor, name: str) -> tp.Tuple[int, int, int, int]:
    """(rows, K, row stride, type) of a 2-D float matrix whose rows are contiguous"""
    if x.dim() != 2 or x.dtype not in _TYPE_CODE or (x.shape[1] > 1 and x.stride(1) != 1):
        raise ValueError(f"{name}: a float32, bfloat16 or float16 matrix with contiguous rows expected, got {x.dtype} {tuple(x.shape)} strides {x.stride()}")
    rows, K = x.shape
    if rows > _MOST or K > _MOST:
        raise ValueError(f"{name}: at most {_MOST} rows and columns, got {tuple(x.shape)}")
    ld = x.stride(0) if rows > 1 else max(K, 1)
    if ld < K:
        raise ValueError(f"{name}: rows overlap (stride {ld} for {K} columns)")
    return rows, K, ld, _TYPE_CODE[x.dtype]


def _code_rows(q: torch.Tensor, scale: torch.Tensor, name: str) -> tp.Tuple[int, int, int]:
    """(rows, K, row stride) of an int8 matrix on 16-byte rows, and its scales' check"""
    if q.dim() != 2 or q.dtype != torch.int8 or (q.shape[1] > 1 and q.stride(1) != 1):
        raise ValueError(f"{name}: an int8 matrix with contiguous rows expected, got {q.dtype} {tuple(q.shape)} strides {q.stride()}")
    rows, K = q.shape
    if rows > _MOST or K > _MOST:
        raise ValueError(f"{name}: at most {_MOST} rows and columns, got {tuple(q.shape)}")
    K16 = (K + 15) // 16 * 16
    ld = q.stride(0) if rows > 1 else K16
    if q.numel() and (ld % 16 or ld < K or q.data_ptr() % 16 or
                      q.untyped_storage().nbytes() - q.storage_offset() < (rows - 1) * ld + K16):
        raise ValueError(f"{name}: rows on 16-byte boundaries that can be read to a multiple of 16 expected (quantize_rows makes them), got strides {q.stride()}")
    if scale.dtype != torch.float32 or scale.shape != (rows,) or (rows > 1 and scale.stride(0) != 1) or scale.device != q.device:
        raise ValueError(f"{name}: a contiguous float32 scale for each of the {rows} rows expected, got {scale.dtype} {tuple(scale.shape)}")
    return rows, K, ld


def _bytes_of(t: torch.Tensor) -> tp.Tuple[int, int, int, int]:
    """first and last byte (exclusive) of a matrix or vector with contiguous rows, the bytes of a row and from one row to the next (0: one row)"""
    rows, cols = (t.shape if t.dim() == 2 else (1, t.shape[0])) if t.numel() else (1, 0)
    step = t.stride(0) if rows > 1 else 0
    size = t.element_size()
    return t.data_ptr(), t.data_ptr() + ((rows - 1) * step + cols) * size, cols * size, step * size


def _share_memory(t: torch.Tensor, u: torch.Tensor) -> bool:
    first, last, row, step = _bytes_of(t)
    first2, last2, row2, step2 = _bytes_of(u)
    if first2 >= last or first >= last2:
        return False
    if step and step2 and step != step2:          # (rows that lie differently are not followed)
        return True
    step = step or step2
    away = (first2 - first) % step if step else 0
    return away < row or away + row2 > step       # columns of their own, in rows that lie alike


def _i8_output(out, out_dtype, M, N, device, bias, inputs):
    """(output, its row stride) after the checks of the bias and of a given output"""
    if bias is not None and (bias.dtype != torch.float32 or bias.shape != (N,) or (N > 1 and bias.stride(0) != 1) or bias.device != device):
        raise ValueError(f"bias: {N} contiguous float32 on {device} expected, got {bias.dtype} {tuple(bias.shape)} on {bias.device}")
    if out is None:
        if out_dtype not in _TYPE_CODE:
            raise ValueError(f"out_dtype: float32, bfloat16 or float16 expected, got {out_dtype}")
        return torch.empty((M, N), dtype=out_dtype, device=device), N
    rows, cols, ld, _ = _float_rows(out, "out")
    if (rows, cols) != (M, N) or out.device != device:
        raise ValueError(f"out: [{M}, {N}] on {device} expected, got {tuple(out.shape)} on {out.device}")
    for t in inputs + (() if bias is None else (bias,)):
        if _share_memory(out, t):
            raise ValueError("out: shares memory with an input")
    return out, ld


def quantize_rows(x: torch.Tensor) -> tp.Tuple[torch.Tensor, torch.Tensor]:
    """(codes, scale): scale[r] = max|x[r]| / 127 (as a product with the float32 nearest to 1/127), codes = nearest whole numbers to x / scale (int8,
    ties to even).

    The tokens of an activation matrix and the channels of a weight matrix [out, in] alike.  x: float32, bfloat16 or float16 [rows, K] with contiguous
    rows.  ``codes`` is a view of rows padded with zeros to a multiple of 128, which ``gemm_i8`` and ``linear_i8`` read as it is.  A row that holds a NaN or an
    infinity gets the scale NaN, so that its products are NaN; a row of zeros gets the scale 0.
    """
    rows, K, ld, code = _float_rows(x, "x")
    stream = _stream_on(x)
    Kp = (K + 127) // 128 * 128
    q = torch.empty((rows, Kp), dtype=torch.int8, device=x.device)
    scale = torch.empty(rows, dtype=torch.float32, device=x.device)
    if rows and K:
        check(_lib.load().fbhip_quantize_rows(x.data_ptr(), ld, code, q.data_ptr(), Kp, scale.data_ptr(), rows, K, Kp, stream))
    elif rows:
        scale.zero_()
    return q[:, :K], scale


def gemm_i8(A: torch.Tensor, a_scale: torch.Tensor, B: torch.Tensor, b_scale: torch.Tensor, *, bias: tp.Optional[torch.Tensor] = None,
            relu: bool = False, out_dtype: torch.dtype = torch.float32, out: tp.Optional[torch.Tensor] = None) -> torch.Tensor:
    """C[m, n] = act((sum_k A[m, k] B[n, k]) * a_scale[m] * b_scale[n] + bias[n]) on int8 codes A [M, K] (tokens) and B [N, K] (channels).

    The sums are exact (K <= 131071; M, N <= 2^30).  ``out`` may lie in columns of its own beside an input, but not share memory with one.  Rows lie on 16-byte boundaries and can be read to a multiple of 16, as ``quantize_rows`` makes them.
    """
    M, K, lda = _code_rows(A, a_scale, "A")
    N, K2, ldb = _code_rows(B, b_scale, "B")
    if K != K2 or A.device != B.device:
        raise ValueError(f"A {tuple(A.shape)} on {A.device} and B {tuple(B.shape)} on {B.device} do not go together")
    stream = _stream_on(A)
    C, ldc = _i8_output(out, out_dtype, M, N, A.device, bias, (A, a_scale, B, b_scale))
    if M == 0 or N == 0:
        return C
    lib = _lib.load()
    need = lib.fbhip_gemm_i8_workspace(M, N, K)
    ws = torch.empty(need, dtype=torch.uint8, device=A.device) if need else None
    check(lib.fbhip_gemm_i8(A.data_ptr(), lda, a_scale.data_ptr(), B.data_ptr(), ldb, b_scale.data_ptr(), ptr(bias), int(relu), C.data_ptr(), ldc,
                            _TYPE_CODE[C.dtype], M, N, K, ptr(ws), stream))
    return C


class _Codes(torch.autograd.Function):
    """``linear_i8`` of an ``x`` that requires a gradient: a backward pass that asks for it hears that there is none"""

    @staticmethod
    def forward(ctx, x, W, w_scale, bias, relu, out_dtype):  # noqa: D102
        return linear_i8(x, W, w_scale, bias=bias, relu=relu, out_dtype=out_dtype)          # (gradients are off in here)

    @staticmethod
    def backward(ctx, g):  # noqa: D102
        raise RuntimeError("linear_i8: no gradient flows through 8-bit codes (it is for answers): call it on x.detach() or under torch.no_grad()")


def linear_i8(x: torch.Tensor, W: torch.Tensor, w_scale: torch.Tensor, *, bias: tp.Optional[torch.Tensor] = None, relu: bool = False,
              out_dtype: tp.Optional[torch.dtype] = None, out: tp.Optional[torch.Tensor] = None) -> torch.Tensor:
    """act(x W^T + bias) with x quantised row by row on the way: ``gemm_i8(*quantize_rows(x), W, w_scale, ...)`` in one call.

    x: float32, bfloat16 or float16 [M, K] with contiguous rows; W, w_scale: ``quantize_rows`` of the [N, K] weights; the output has x's type
    unless ``out_dtype`` or ``out`` says otherwise.  For answers, not for training: no gradient flows through the codes.  Where ``x`` requires one, a
    backward pass through the result raises, and ``out`` is refused.
    """
    M, K, ldx, code = _float_rows(x, "x")
    N, K2, ldw = _code_rows(W, w_scale, "W")
    if K != K2 or x.device != W.device:
        raise ValueError(f"x {tuple(x.shape)} on {x.device} and W {tuple(W.shape)} on {W.device} do not go together")
    stream = _stream_on(x)
    if x.requires_grad and torch.is_grad_enabled():
        if out is not None:
            raise ValueError("linear_i8: out does not go with an x that requires a gradient: call it on x.detach() or under torch.no_grad()")
        return _Codes.apply(x, W, w_scale, bias, relu, out_dtype)
    y, ldy = _i8_output(out, x.dtype if out_dtype is None else out_dtype, M, N, x.device, bias, (x, W, w_scale))
    if M == 0 or N == 0:
        return y
    lib = _lib.load()
    need = lib.fbhip_linear_i8_workspace(M, N, K)
    ws = torch.empty(need, dtype=torch.uint8, device=x.device) if need else None
    check(lib.fbhip_linear_i8(x.data_ptr(), ldx, code, W.data_ptr(), ldw, w_scale.data_ptr(), ptr(bias), int(relu), y.data_ptr(), ldy,
                              _TYPE_CODE[y.dtype], M, N, K, ptr(ws), stream))
    return y
