"""The 8-bit product has no gradient: a backward pass through it says so."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("M", [1, 40, 300])
def test_a_backward_pass_through_the_codes_raises(M):
    from controllable_agent_amd import kernels as K
    gen = torch.Generator().manual_seed(M)
    x, w = torch.randn(M, 100, generator=gen).cuda(), torch.randn(30, 100, generator=gen).cuda()
    codes, scale = K.quantize_rows(w.requires_grad_(True))
    bias = torch.randn(30, generator=gen).cuda().requires_grad_(True)
    want = K.linear_i8(x, codes, scale, bias=bias, relu=True)
    assert not want.requires_grad                                        # (weights and bias of a network in service may be its parameters)
    y = K.linear_i8(x.requires_grad_(True), codes, scale, bias=bias, relu=True)
    assert torch.equal(y, want) and y.requires_grad
    with pytest.raises(RuntimeError, match="no gradient flows"):
        (y.sum() + x.square().sum()).backward()
    hidden = torch.relu(x * 2)
    with pytest.raises(RuntimeError, match="no gradient flows"):
        torch.autograd.grad(K.linear_i8(hidden, codes, scale, out_dtype=torch.bfloat16).float().sum(), x)
    with pytest.raises(ValueError, match="requires a gradient"):
        K.linear_i8(x, codes, scale, out=torch.empty(M, 30, device="cuda"))
    for again in (K.linear_i8(x.detach(), codes, scale, bias=bias, relu=True),):
        assert torch.equal(again, want) and not again.requires_grad
    with torch.no_grad():
        z = K.linear_i8(x, codes, scale, bias=bias, relu=True, out=torch.empty(M, 30, device="cuda"))
    assert torch.equal(z, want) and not z.requires_grad


def test_its_result_may_be_changed_in_place():
    from controllable_agent_amd import kernels as K
    gen = torch.Generator().manual_seed(0)
    x = torch.randn(20, 100, generator=gen).cuda()
    codes, scale = K.quantize_rows(torch.randn(30, 100, generator=gen).cuda())
    want = K.linear_i8(x, codes, scale).add_(1).mul_(2)
    got = K.linear_i8(x.clone().requires_grad_(True), codes, scale).add_(1).mul_(2)
    assert torch.equal(got, want)
    with pytest.raises(RuntimeError, match="no gradient flows"):
        got.sum().backward()
    assert torch.equal(K.linear_i8(x[:0].requires_grad_(True), codes, scale), torch.zeros(0, 30, device="cuda"))
