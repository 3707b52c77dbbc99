"""8-bit products: an output may lie between the rows of an input, in columns of its own; it is refused only where it shares memory."""
import pytest
import torch

from controllable_agent_amd import kernels as K

BUF = torch.zeros(12, 40)
CPU = BUF.device


def _takes(out, x, bias=None):
    return K._i8_output(out, None, out.shape[0], out.shape[1], CPU, bias, (x,))[0] is out


@pytest.mark.parametrize("out,x", [
    (BUF[:, 20:], BUF[:, :20]), (BUF[:, :20], BUF[:, 20:]), (BUF[:, 30:35], BUF[:, :30]), (BUF[:, 5:9], BUF[3:, 9:40]), (BUF[2:7, 5:9], BUF[:, 9:30]),
    (BUF[4:5, 5:9], BUF[:, 9:30]), (BUF[:, 5:9], BUF[4:5, 9:30]), (BUF[3:, :10], BUF[:, 10:11]),
    (BUF.view(torch.bfloat16)[:, 41:60], BUF[:, :20]), (BUF[:6], BUF[6:]), (BUF[6:], BUF[:6]),
])
def test_columns_of_its_own(out, x):
    assert _takes(out, x)
    if x.shape[0] == 1:
        assert _takes(out, x[0])


@pytest.mark.parametrize("out,x", [
    (BUF[:, 19:], BUF[:, :20]), (BUF[:, :21], BUF[:, 20:]), (BUF[:, 30:35], BUF[:, :31]), (BUF[:, 5:9], BUF), (BUF, BUF[3:4, 5:9]), (BUF, BUF),
    (BUF.view(torch.bfloat16)[:, 39:60], BUF[:, :20]),
    (BUF.view(24, 20)[:, :10], BUF[:, 10:20]),                                    # another row stride: columns meet in other rows
    (BUF[:, 30:40], BUF.view(-1)[41:].as_strided((11, 31), (40, 1))),             # rows that run over the end of the output's
    (BUF[4:5, 5:9], BUF[:, 8:30]), (BUF[:, 5:9], BUF[4:5, 8:30]),
])
def test_shared_memory(out, x):
    with pytest.raises(ValueError, match="shares memory"):
        _takes(out, x)
    if x.shape[0] == 1:
        with pytest.raises(ValueError, match="shares memory"):
            _takes(out, x[0])


def test_a_bias_between_the_rows():
    out, x = BUF[:, :5], torch.zeros(12, 3)
    assert _takes(out, x, BUF[3, 10:15]) and _takes(out, x, BUF[3, 35:40])
    for bias in (BUF[3, 2:7], BUF.view(-1)[38:43], BUF[11, 0:5]):
        with pytest.raises(ValueError, match="shares memory"):
            _takes(out, x, bias)
