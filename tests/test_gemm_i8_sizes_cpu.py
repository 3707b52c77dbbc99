"""8-bit products: sizes that a 32-bit number does not hold are refused, not wrapped (tensors without storage stand for them)."""
import pytest
import torch

from controllable_agent_amd import _lib, kernels as K


@pytest.mark.parametrize("shape", [(2 ** 32 + 5, 4), (2 ** 31, 1), (3, 2 ** 32 + 5), (1, 2 ** 31), (1, 2 ** 31 - 1)])
def test_matrices_of_more_rows_or_columns_than_the_entry_points_count(shape):
    x = torch.empty(shape, dtype=torch.float16, device="meta")
    with pytest.raises(ValueError, match="rows and columns"):
        K._float_rows(x, "x")
    q = torch.empty((shape[0], -(-shape[1] // 16) * 16), dtype=torch.int8, device="meta")[:, :shape[1]]
    with pytest.raises(ValueError, match="rows and columns"):
        K._code_rows(q, torch.empty(shape[0], device="meta"), "A")
    with pytest.raises(ValueError, match="rows and columns"):
        K._i8_output(x, None, shape[0], shape[1], x.device, None, ())


def test_the_largest_that_they_count():
    x = torch.empty((1, 2 ** 31 - 1024), dtype=torch.float16, device="meta")
    assert K._float_rows(x, "x")[:2] == tuple(x.shape)
    assert K._float_rows(x.view(-1, 1), "x")[:2] == (2 ** 31 - 1024, 1)


def test_the_c_entry_refuses_rows_that_its_kernels_could_not_walk():
    lib = _lib.load()
    for k in (2 ** 31 - 1, 2 ** 31 - 200, 2 ** 31 - 1023):
        assert lib.fbhip_quantize_rows(16, k, 2, 16, k, 16, 1, k, k, None) == -1 and b"K" in lib.fbhip_last_error(None)
