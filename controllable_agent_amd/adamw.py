"""AdamW over a list of tensors in one launch (384 tensors each), moments in 32 or in 8 bits (csrc/adamw.hip).

``kernels.adam_ema`` moves one flat fp32 buffer with Adam's fixed settings, as the agents' own networks need it; this is the optimiser for
everything else a user trains beside them: any number of tensors of any sizes, fp32 or bf16, with decoupled weight decay, clipping by the
global gradient norm, and moments that take 2 bytes a parameter instead of 8.
"""
from __future__ import annotations

import array
import ctypes as C
import math
import operator
import typing as tp

import torch

from . import _lib
from ._lib import check

BLOCK = 256            # elements that share a scale of an 8-bit moment
CHUNK = 2048           # FBHIP_ADAMW_CHUNK
GRAD_DENSE = 4         # FBHIP_GRAD_DENSE
CONTROL_BYTES = 2304   # FBHIP_ADAMW_CONTROL_BYTES
_DTYPE = operator.attrgetter("dtype")
_FLOAT_MAX = torch.finfo(torch.float32).max
_TYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}


class _Tensor(C.Structure):
    _fields_ = [("p", C.c_void_p), ("numel", C.c_int64), ("at", C.c_int64), ("cols", C.c_int32), ("ld", C.c_int32),
                ("weight_decay", C.c_double), ("lr_scale", C.c_double), ("dtype", C.c_int32), ("reserved", C.c_int32)]


class _Opt(C.Structure):
    _fields_ = [("struct_size", C.c_uint32), ("n_tensors", C.c_int32), ("tensors", C.c_void_p), ("chunks", C.c_void_p),
                ("host_first_chunk", C.c_void_p), ("bits", C.c_int32), ("seed", C.c_uint32), ("m", C.c_void_p), ("v", C.c_void_p),
                ("m_scale", C.c_void_p), ("r_scale", C.c_void_p), ("control", C.c_void_p), ("partials", C.c_void_p),
                ("beta1", C.c_double), ("beta2", C.c_double), ("eps", C.c_float)]


def _dense(t: torch.Tensor) -> bool:
    """whether the elements fill one run of memory, in whatever order of the dimensions"""
    if t.is_contiguous():
        return True
    want = 1
    for stride, size in sorted((st, sz) for st, sz in zip(t.stride(), t.shape) if sz != 1):
        if stride != want:
            return False
        want *= size
    return True


def _per_tensor(name: str, value, n: int) -> tp.List[float]:
    values = [float(value)] * n if isinstance(value, (int, float)) else [float(x) for x in value]
    if len(values) != n or not all(math.isfinite(x) for x in values):
        raise ValueError(f"{name}: one finite number, or one for each of the {n} tensors")
    return values


class AdamW:
    """``opt = AdamW(params); opt.step(grads)``: p <- (1 - lr wd) p - lr m^ / (sqrt(v^) + eps), all tensors in one launch (384 of them a launch, and
    one more each to clip).  Every value is the formulas' chain of correctly rounded single-precision operations.

    ``params``: float32 or bfloat16 device tensors, changed in place; dense in any order of dimensions, or row-strided matrices (the
    agents' ``NetView`` entries).  bfloat16 parameters are rounded up or down at random, so that small updates count on average.
    ``weight_decay`` and ``lr_scale`` (a factor on ``lr``): a number, or one for each tensor.  ``state_bits=8`` holds the moments m and
    r = sqrt(v) as e4m3 codes with a power-of-two scale for each 256 elements of a tensor, rounded at random (``seed``).

    State: ``m``, ``v`` (float32) or ``m8``, ``m_scale``, ``r8``, ``r_scale``, flat over all tensors, each tensor padded to a multiple of 256
    elements; ``step_count``, kept on the device, so that a captured and replayed ``step`` counts too (it reads the gradient tensors that it was captured
    with; the numbers given to it, ``lr``, ``grad_scale``, ``max_norm``, and the seed stay what they were).  The same instance must not step on two streams at once; a step belongs
    to the stream that is current when it is called.  A parameter whose storage is exchanged afterwards (``p.data = ...``) is not followed.
    """

    def __init__(self, params: tp.Iterable[torch.Tensor], lr: tp.Union[float, torch.Tensor] = 1e-3, betas: tp.Tuple[float, float] = (0.9, 0.999),
                 eps: float = 1e-8, weight_decay: tp.Union[float, tp.Sequence[float]] = 0.01,
                 lr_scale: tp.Union[float, tp.Sequence[float]] = 1.0, state_bits: int = 32, seed: int = 0) -> None:
        self.params = [p.detach() for p in params]
        n = len(self.params)
        if n == 0:
            raise ValueError("AdamW: no parameters")
        if state_bits not in (8, 32):
            raise ValueError(f"AdamW: state_bits is 8 or 32, got {state_bits}")
        if not (0.0 <= betas[0] < 1.0 and 0.0 <= betas[1] < 1.0 and (eps == 0.0 or 1e-30 <= eps < math.inf)):
            raise ValueError(f"AdamW: 0 <= beta < 1 and eps 0 or at least 1e-30, got betas={betas}, eps={eps}")
        if not isinstance(lr, torch.Tensor) and not math.isfinite(lr):
            raise ValueError(f"AdamW: a finite lr expected, got {lr}")
        wd, scale = _per_tensor("weight_decay", weight_decay, n), _per_tensor("lr_scale", lr_scale, n)
        if min(wd) < 0:
            raise ValueError("AdamW: weight_decay >= 0 expected")
        self._layouts: tp.List[tp.Tuple[int, int]] = []          # (cols, ld); cols 0: dense
        spans = []
        for k, p in enumerate(self.params):
            if p.dtype not in (torch.float32, torch.bfloat16):
                raise TypeError(f"AdamW: parameter {k} is {p.dtype}: float32 or bfloat16 expected")
            if p.device != self.params[0].device:
                raise ValueError(f"AdamW: parameter {k} is on {p.device}, parameter 0 on {self.params[0].device}")
            if _dense(p):
                self._layouts.append((0, 0))
                extent = p.numel()
            elif p.dim() == 2 and p.stride(1) == 1 and p.shape[1] <= p.stride(0) < 2 ** 31:
                self._layouts.append((p.shape[1], p.stride(0)))
                extent = (p.shape[0] - 1) * p.stride(0) + p.shape[1]
            else:
                raise ValueError(f"AdamW: parameter {k} with shape {tuple(p.shape)} and strides {p.stride()} is neither dense nor a row-strided matrix")
            if p.numel():
                spans.append((p.data_ptr(), p.data_ptr() + extent * p.element_size(), k))
        spans.sort()
        open_spans: tp.List[tp.Tuple[int, int, int]] = []
        for start, end, j in spans:
            open_spans = [o for o in open_spans if o[1] > start]
            for other, _, i in open_spans:
                # column slices of one matrix may interleave; anything else that overlaps would be moved twice
                if other == start or not self._interleaved(i, j):
                    raise ValueError(f"AdamW: parameters {i} and {j} share memory")
            open_spans.append((start, end, j))
        self.device = self.params[0].device
        if self.device.type != "cuda":
            raise RuntimeError("AdamW: device tensors expected: controllable_agent_amd has no CPU fallback")
        with torch.cuda.device(self.device):
            _lib.require_device()
        self.lr, self.betas, self.eps, self.state_bits, self.seed = lr, (float(betas[0]), float(betas[1])), float(eps), state_bits, int(seed) & 0xFFFFFFFF
        table, first, at = (_Tensor * n)(), [0], 0
        self.offsets: tp.List[int] = []                          # first element of each tensor in the moments
        for k, p in enumerate(self.params):
            cols, ld = self._layouts[k]
            table[k] = _Tensor(p.data_ptr() or None, p.numel(), at, cols, ld, wd[k], scale[k], _TYPES[p.dtype], 0)
            self.offsets.append(at)
            at += -(-p.numel() // BLOCK) * BLOCK
            first.append(first[-1] + -(-p.numel() // CHUNK))
        if first[-1] >= 2 ** 31:
            raise ValueError("AdamW: too many elements for one instance")
        self._first = (C.c_int32 * (n + 1))(*first)
        first_t = torch.tensor(first, dtype=torch.int64)
        which = torch.repeat_interleave(torch.arange(n), first_t[1:] - first_t[:-1])
        chunks = torch.stack([which, torch.arange(first[-1]) - first_t[which]], dim=1).to(torch.int32)
        self._table = torch.frombuffer(bytearray(table), dtype=torch.uint8).to(self.device)
        self._chunks = torch.cat([chunks, torch.zeros(1, 2, dtype=torch.int32)]).to(self.device)      # (never an empty allocation)
        size = max(at, BLOCK)
        zeros = lambda m, t: torch.zeros(m, dtype=t, device=self.device)  # noqa: E731
        if state_bits == 32:
            self.m, self.v = zeros(size, torch.float32), zeros(size, torch.float32)
        else:
            self.m8, self.r8 = zeros(size, torch.uint8).view(torch.float8_e4m3fn), zeros(size, torch.uint8).view(torch.float8_e4m3fn)
            self.m_scale, self.r_scale = zeros(size // BLOCK, torch.float32), zeros(size // BLOCK, torch.float32)
        self._control = zeros(CONTROL_BYTES // 8, torch.int64)
        self._norm = self._control.view(torch.float32)[6]        # byte 24
        self._partials = zeros(_lib.load().fbhip_adamw_partials(n), torch.float64)
        m, v = (self.m, self.v) if state_bits == 32 else (self.m8, self.r8)
        self._opt = _Opt(C.sizeof(_Opt), n, self._table.data_ptr(), self._chunks.data_ptr(), C.addressof(self._first), state_bits, self.seed,
                         m.data_ptr(), v.data_ptr(), None if state_bits == 32 else self.m_scale.data_ptr(),
                         None if state_bits == 32 else self.r_scale.data_ptr(), self._control.data_ptr(), self._partials.data_ptr(),
                         *self.betas, self.eps)
        self._opt_ref = C.byref(self._opt)
        self._versioned = [p for p in self.params if not p.is_inference()]       # (tensors made in inference mode have no version)
        self._seen: tp.Any = None                  # strides, shapes, types and devices that passed the checks, and what they gave
        self._types = b""
        self._set_step(0)

    def _interleaved(self, i: int, j: int) -> bool:
        (ci, li), (cj, lj) = self._layouts[i], self._layouts[j]
        p, q = self.params[i], self.params[j]
        ld = li or lj                              # (what is dense is one row among the other's)
        if not ld or (li and lj and li != lj) or p.dtype != q.dtype:
            return False
        away = (q.data_ptr() - p.data_ptr()) // p.element_size() % ld
        return away >= (ci or p.numel()) and away + (cj or q.numel()) <= ld

    def _set_step(self, step: int) -> None:
        with torch.cuda.device(self.device):
            check(_lib.load().fbhip_adamw_set_step(C.byref(self._opt), int(step), torch.cuda.current_stream().cuda_stream))

    def _grad_types(self, grads: tp.List[torch.Tensor]) -> bytes:
        """the type of each gradient for the kernel, after the checks that its place beside the parameters needs"""
        if len(grads) != len(self.params):
            raise ValueError(f"AdamW.step: {len(grads)} gradients for {len(self.params)} parameters")
        try:
            # (shapes and strides together: the same strides and size may belong to a part of a larger matrix, or to rows that overlap; what is
            # contiguous has no strides to compare)
            strides = None if all(map(torch.Tensor.is_contiguous, grads)) else list(map(torch.Tensor.stride, grads))
            seen = (strides, list(map(torch.Tensor.size, grads)), list(map(_DTYPE, grads)), list(map(torch.Tensor.get_device, grads)))
        except (AttributeError, TypeError):
            raise ValueError("AdamW.step: a gradient is no tensor: leave its parameter out, or pass zeros (which decay its moments)") from None
        if seen == self._seen:                     # as in the last step
            return self._types
        types = bytearray()
        for k, (g, p) in enumerate(zip(grads, self.params)):
            if g.dtype not in _TYPES:
                raise TypeError(f"AdamW.step: gradients are float32, bfloat16 or float16, got {g.dtype}")
            if g.shape != p.shape or g.device != self.device:
                raise ValueError(f"AdamW.step: gradient {k} is {tuple(g.shape)} on {g.device}, its parameter {tuple(p.shape)} on {self.device}")
            cols = self._layouts[k][0]
            flag = 0
            if g.stride() != p.stride() and not (not cols and p.is_contiguous() and g.is_contiguous()):
                if not (cols and g.is_contiguous()):
                    raise ValueError(f"AdamW.step: gradient {k} has strides {g.stride()}, its parameter {p.stride()}: the same, or a "
                                     "contiguous gradient of a row-strided matrix, expected")
                flag = GRAD_DENSE
            types.append(_TYPES[g.dtype] | flag)
        self._seen, self._types = seen, bytes(types)
        return self._types

    def step(self, grads: tp.Sequence[torch.Tensor], *, lr: tp.Union[float, torch.Tensor, None] = None, grad_scale: float = 1.0,
             max_norm: tp.Optional[float] = None) -> tp.Optional[torch.Tensor]:
        """One step with the gradients ``grads`` (one for each parameter, its shape and strides; float32, bfloat16 or float16), times ``grad_scale``.

        ``lr`` (here or in the constructor): a number, or one float32 on the device, which a captured step reads anew at each replay.
        ``max_norm`` scales the gradients so that the norm over all of them is at most that (``inf``: the norm alone), and returns the norm
        before the scaling, a 0-d device tensor that the next step overwrites.  If it is not finite, the step leaves parameters, moments and
        step count as they were.  Without ``max_norm`` nothing is checked: what is no number stays with its own element.
        """
        grads = list(grads)
        types = self._grad_types(grads)
        lr = self.lr if lr is None else lr
        lr_ptr, lr_value = None, 0.0
        if isinstance(lr, torch.Tensor):
            if lr.dtype != torch.float32 or lr.numel() != 1 or lr.device != self.device:
                raise ValueError("AdamW.step: lr is a number, or one float32 on the parameters' device")
            lr_ptr = lr.data_ptr()
        else:
            lr_value = float(lr)
        if not (abs(lr_value) <= _FLOAT_MAX and abs(grad_scale) <= _FLOAT_MAX):
            raise ValueError(f"AdamW.step: finite lr and grad_scale (in float32) expected, got {lr} and {grad_scale}")
        if max_norm is not None and not max_norm > 0:
            raise ValueError(f"AdamW.step: max_norm > 0 expected, got {max_norm}")
        pointers = array.array("Q", map(torch.Tensor.data_ptr, grads))
        args = (self._opt_ref, pointers.buffer_info()[0], types, lr_ptr, lr_value, float(grad_scale), int(max_norm is not None),
                0.0 if max_norm is None else float(max_norm))
        if torch.cuda.current_device() == self.device.index:
            check(_lib.load().fbhip_adamw_step(*args, torch._C._cuda_getCurrentRawStream(self.device.index)))
        else:
            with torch.cuda.device(self.device):
                check(_lib.load().fbhip_adamw_step(*args, torch.cuda.current_stream().cuda_stream))
        torch.autograd.graph.increment_version(self._versioned)
        return None if max_norm is None else self._norm

    @property
    def step_count(self) -> int:
        """steps done (reads the device)"""
        return int(self._control[0].item())

    def moments(self, k: int) -> tp.Tuple[torch.Tensor, torch.Tensor]:
        """(m, v) of parameter ``k`` in float32, flat, in the order of its storage (rows one after another for a row-strided matrix)"""
        a, n = self.offsets[k], self.params[k].numel()
        if self.state_bits == 32:
            return self.m[a:a + n], self.v[a:a + n]
        b = -(-n // BLOCK) * BLOCK
        value = lambda c, s: (c[a:a + b].float().view(-1, BLOCK) * s[a // BLOCK:(a + b) // BLOCK, None]).view(-1)[:n]  # noqa: E731
        return value(self.m8, self.m_scale), value(self.r8, self.r_scale).square()

    def _state(self) -> tp.Dict[str, torch.Tensor]:
        names = ("m", "v") if self.state_bits == 32 else ("m8", "m_scale", "r8", "r_scale")
        return {n: getattr(self, n) for n in names}

    def state_dict(self) -> tp.Dict[str, tp.Any]:
        """copies of the moments, the step count and the seed"""
        return dict({n: t.clone() for n, t in self._state().items()}, step=self.step_count, seed=self.seed)

    def load_state_dict(self, state: tp.Mapping[str, tp.Any]) -> None:
        mine = self._state()
        missing = sorted((set(mine) | {"step", "seed"}) - set(state))
        if missing:
            raise ValueError(f"AdamW.load_state_dict: {missing} missing (a state of {self.state_bits} bits expected)")
        for n, t in mine.items():          # (everything is looked at before anything is changed)
            if not isinstance(state[n], torch.Tensor) or state[n].shape != t.shape or state[n].dtype != t.dtype:
                got = f"{state[n].dtype} {tuple(state[n].shape)}" if isinstance(state[n], torch.Tensor) else type(state[n]).__name__
                raise ValueError(f"AdamW.load_state_dict: {n} is {got}, {t.dtype} {tuple(t.shape)} expected")
        try:
            step, seed = int(state["step"]), int(state["seed"])
            whole = step == state["step"] and seed == state["seed"] and 0 <= step < 2 ** 63
        except (TypeError, ValueError, OverflowError):
            whole = False
        if not whole:
            raise ValueError(f"AdamW.load_state_dict: a step count and a seed expected, got {state['step']!r} and {state['seed']!r}")
        for n, t in mine.items():
            t.copy_(state[n])
        self.seed = self._opt.seed = seed & 0xFFFFFFFF
        self._set_step(step)
