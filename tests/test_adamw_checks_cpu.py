"""AdamW's checks of a step's gradients, on host tensors: what a first step refuses, a later one refuses too."""
import pytest
import torch

from controllable_agent_amd.adamw import AdamW, GRAD_DENSE


def _checker(params, layouts=None):
    """an instance with what the checks look at (a whole one needs a device)"""
    opt = object.__new__(AdamW)
    opt.params = params
    opt.device = params[0].device
    opt._layouts = layouts or [(0, 0)] * len(params)
    opt._seen, opt._types = None, b""
    return opt


CASES = [
    # (parameter, gradient with the same strides, number of elements and type that is not its like)
    (torch.zeros(4, 6), torch.zeros(8, 6)[:, :3]),                             # every second run of three
    (torch.zeros(4, 6), torch.zeros(23).as_strided((3, 8), (6, 1))),           # rows that overlap, in a storage shorter than the parameter
    (torch.zeros(3, 4), torch.zeros(6, 4)[:, :2]),
    (torch.zeros(1, 4), torch.zeros(2, 4)[:, :2]),
    (torch.zeros(2, 3, 4), torch.zeros(4, 3, 4)[:, :, :2]),
    (torch.zeros(6, 4).t(), torch.zeros(31).as_strided((3, 8), (1, 4))),
]


@pytest.mark.parametrize("k", range(len(CASES)))
def test_gradients_of_another_shape_are_refused_at_every_step(k):
    p, bad = CASES[k]
    good = torch.empty_strided(p.shape, p.stride())
    for first in ([bad], [good, bad], [good, good, bad, good, bad]):
        opt = _checker([p])
        for g in first:
            if g is bad:
                with pytest.raises(ValueError):
                    opt._grad_types([g])
            else:
                assert opt._grad_types([g]) == b"\0"


def test_the_other_refusals_after_a_good_step():
    p, q = torch.zeros(8, 6), torch.zeros(5)
    g, h = torch.zeros(8, 6), torch.zeros(5)
    opt = _checker([p, q])
    bad = [([g], ValueError), ([g, None], ValueError), ([g, h.double()], TypeError), ([g.t(), h], ValueError),
           ([torch.zeros(6, 8).t(), h], ValueError), ([torch.zeros(8, 1).expand(8, 6), h], ValueError), ([g, torch.zeros(5, 1)], ValueError),
           ([g, torch.zeros(10)[::2]], ValueError), ([h, g], ValueError)]
    for grads, error in bad:
        assert opt._grad_types([g, h]) == b"\0\0"
        with pytest.raises(error):
            opt._grad_types(grads)
    assert opt._grad_types([g.bfloat16(), h.half()]) == bytes([1, 2]) and opt._grad_types([g, h]) == b"\0\0"


def test_matrices_with_rows_apart():
    p = torch.zeros(8, 12)[:, :6]
    opt = _checker([p], [(6, 12)])
    assert opt._grad_types([torch.zeros(8, 12)[:, :6]]) == b"\0" and opt._grad_types([torch.zeros(8, 6)]) == bytes([GRAD_DENSE])
    for bad in (torch.zeros(16, 12)[:, :3], torch.zeros(8, 10)[:, :6], torch.zeros(12, 12)[:, :4], torch.zeros(6, 8), torch.zeros(6, 8).t()):
        with pytest.raises(ValueError):
            opt._grad_types([bad])
        assert opt._grad_types([torch.zeros(8, 12)[:, :6]]) == b"\0"


@pytest.mark.parametrize("change", [dict(step=-1), dict(step=2.5), dict(step=None), dict(step=2 ** 63), dict(seed="x"), dict(m=[1.0]), dict(v=torch.zeros(256).double()),
                                    dict(v=torch.zeros(512))], ids=str)
def test_a_state_that_is_refused_leaves_everything_as_it_was(change):
    opt = object.__new__(AdamW)
    opt.state_bits, opt.seed = 32, 7
    opt.m, opt.v = torch.zeros(256), torch.zeros(256)
    steps = []
    opt._set_step = steps.append
    opt._opt = type("Opt", (), {"seed": 7})()
    with pytest.raises(ValueError):
        opt.load_state_dict({**dict(m=torch.ones(256), v=torch.ones(256), step=3, seed=9), **change})
    assert not steps and not opt.m.any() and not opt.v.any() and opt.seed == opt._opt.seed == 7
    for step in (3, 3.0, torch.tensor(3), torch.tensor(3.0)):
        opt.load_state_dict(dict(m=torch.ones(256), v=torch.ones(256), step=step, seed=9))
    assert steps == [3] * 4 and opt.m.all() and opt.v.all() and opt.seed == opt._opt.seed == 9


def test_a_row_beside_the_columns_of_the_others():
    """one row of a matrix is dense; it shares no memory with other columns of the same matrix"""
    buf = torch.zeros(10, 10)
    for params in ([buf[1:2, :5], buf[:, 5:]], [buf[:, :5], buf[3, 5:]], [buf[:, 3:5], buf[3, 5:], buf[4, :3], buf[5:6, 5:9]]):
        with pytest.raises(RuntimeError, match="no CPU fallback"):
            AdamW(params)
    for params in ([buf[1:2, :6], buf[:, 5:]], [buf[:, :5], buf[3, 4:]], [buf[:, :5], buf.view(-1)[35:46]], [buf[1], buf[:, 5:]], [buf[0, :3], buf[0, 2:5]]):
        with pytest.raises(ValueError, match="share memory"):
            AdamW(params)


@pytest.mark.parametrize("kw", [dict(grad_scale=1e39), dict(grad_scale=-1e39), dict(lr=1e39), dict(lr=float("nan")), dict(grad_scale=float("inf")), dict(max_norm=0.0)], ids=str)
def test_numbers_that_float32_does_not_hold(kw):
    opt = _checker([torch.zeros(4)])
    opt.lr = 1e-3
    with pytest.raises(ValueError):
        opt.step([torch.zeros(4)], **kw)
