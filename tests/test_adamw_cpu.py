"""AdamW over many tensors: what the constructor refuses before it touches the device, and the C entry's own checks."""
import ctypes as C

import pytest
import torch

from controllable_agent_amd import _lib
from controllable_agent_amd.adamw import AdamW, _Opt, _Tensor, _dense


def _p(*shape, dtype=torch.float32):
    return torch.zeros(*shape, dtype=dtype)


@pytest.mark.parametrize("kw,error", [
    (dict(params=[]), ValueError),
    (dict(params=[_p(3)], state_bits=16), ValueError),
    (dict(params=[_p(3)], betas=(1.0, 0.9)), ValueError),
    (dict(params=[_p(3)], betas=(0.9, -0.1)), ValueError),
    (dict(params=[_p(3)], eps=-1.0), ValueError),
    (dict(params=[_p(3)], eps=1e-40), ValueError),
    (dict(params=[_p(3)], lr=float("inf")), ValueError),
    (dict(params=[_p(3)], weight_decay=-0.1), ValueError),
    (dict(params=[_p(3)], weight_decay=[0.1, 0.2]), ValueError),
    (dict(params=[_p(3)], weight_decay=float("nan")), ValueError),
    (dict(params=[_p(3), _p(2)], lr_scale=[1.0]), ValueError),
    (dict(params=[_p(3, dtype=torch.float16)]), TypeError),
    (dict(params=[_p(3, dtype=torch.int32)]), TypeError),
    (dict(params=[_p(1).expand(4)]), ValueError),
    (dict(params=[_p(8)[::2]]), ValueError),
    (dict(params=[_p(4, 6, 8)[:, :, :3]]), ValueError),
    (dict(params=[_p(3)]), RuntimeError),                    # no CPU path
], ids=str)
def test_constructor_refusals(kw, error):
    with pytest.raises(error):
        AdamW(**kw)


def test_parameters_that_share_memory_are_refused():
    flat = _p(100)
    for params in ([flat, flat], [flat[:60], flat[50:]], [flat.view(10, 10)[:, :6], flat.view(10, 10)[:, 5:]], [flat.view(10, 10)[:, :6], flat],
                   [flat.view(10, 10)[:, :5], flat.view(10, 10)[1:, 6:8], flat.view(10, 10)[2:, 3:4]]):
        with pytest.raises(ValueError, match="share memory"):
            AdamW(params)
    # column slices of one matrix do not overlap: refused for the missing device only
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        AdamW([flat.view(10, 10)[:, :6], flat.view(10, 10)[:, 6:]])
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        AdamW([flat[:50], flat[50:]])


def test_dense_in_any_order_of_dimensions():
    t = _p(4, 5, 6)
    assert _dense(t) and _dense(t.permute(2, 0, 1)) and _dense(_p(3, 1, 4).transpose(0, 2)) and _dense(_p(()))
    assert not _dense(t[:, :4]) and not _dense(t[..., ::2]) and not _dense(_p(3, 1).expand(3, 4))


def test_c_entry_refuses_bad_calls():
    lib = _lib.load()
    assert C.sizeof(_Tensor) == 56 and lib.fbhip_adamw_partials(0) == 0 and lib.fbhip_adamw_partials(385) == 2 * lib.fbhip_adamw_partials(384)
    first = (C.c_int32 * 2)(0, 1)
    grads, types = (C.c_void_p * 1)(16), (C.c_uint8 * 1)(0)

    def opt(**kw):
        o = _Opt(C.sizeof(_Opt), 1, 16, 16, C.addressof(first), 32, 0, 16, 16, None, None, 16, 16, 0.9, 0.999, 1e-8)
        for k, v in kw.items():
            setattr(o, k, v)
        return o

    def step(o, g=grads, t=types, clip=0, max_norm=0.0):
        return lib.fbhip_adamw_step(C.byref(o) if o is not None else None, g, t, None, 1e-3, 1.0, clip, max_norm, None)
    for bad in (None, opt(struct_size=8), opt(n_tensors=0), opt(tensors=None), opt(control=None), opt(bits=16), opt(bits=8), opt(m=None),
                opt(beta1=1.0), opt(beta2=float("nan")), opt(eps=-1.0)):
        assert step(bad) == -1 and lib.fbhip_last_error(None)
    assert step(opt(), g=None) == -1 and step(opt(), t=None) == -1
    assert step(opt(), g=(C.c_void_p * 1)(None)) == -1 and step(opt(), t=(C.c_uint8 * 1)(3)) == -1
    assert step(opt(), clip=1) == -1 and step(opt(), clip=1, max_norm=float("nan")) == -1 and step(opt(partials=None), clip=1, max_norm=1.0) == -1
    assert lib.fbhip_adamw_set_step(C.byref(opt()), -1, None) == -1
