"""AdamW's arithmetic bit for bit, against the same operations in IEEE single precision on the host (numpy), and what a second step refuses.

Every value is one chain of correctly rounded float32 operations in the order of the formulas (the square root and the division among them), so that
parameters, moments, codes and scales have to be equal, not near.
"""
import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu
F = np.float32


@pytest.fixture(scope="module")
def AdamW():
    from controllable_agent_amd import AdamW
    return AdamW


def _finish(h):
    h = (h ^ (h >> np.uint32(16))) * np.uint32(0x85EBCA6B)
    h = (h ^ (h >> np.uint32(13))) * np.uint32(0xC2B2AE35)
    return h ^ (h >> np.uint32(16))


def _words(n, seed, step):
    with np.errstate(over="ignore"):
        key = _finish(np.array([seed ^ (step * 0x27D4EB2F & 0xFFFFFFFF)], dtype=np.uint32))
        return _finish(np.arange(n, dtype=np.uint32) * np.uint32(0x9E3779B1) + key)


def _encode(x, bits16, positive):
    """e4m3 codes and power-of-two scales, rounded up or down by 16 random bits"""
    mag = np.abs(x).reshape(-1, 256)
    field = np.maximum(((mag.max(1).view(np.uint32).astype(np.int64) + 0x1FFFFF) >> 23) - 8, 1)
    inv = ((254 - field) << 23).astype(np.uint32).view(F)
    y = (mag * inv[:, None]).reshape(-1)
    small = y < F(2.0 ** -6)
    z = np.where(small, y + F(2.0 ** -6), y)
    code = ((z.view(np.uint32).astype(np.int64) + (bits16.astype(np.int64) << 4)) >> 20) - np.where(small, 968, 960)
    if positive:
        code = np.where((code == 0) & (x > 0), 1, code)
    return (code | np.where(np.signbit(x), 128, 0)).astype(np.uint8), (field << 23).astype(np.uint32).view(F)


def _decode(codes, scale):
    return (torch.from_numpy(codes).view(torch.float8_e4m3fn).float().numpy().reshape(-1, 256) * scale[:, None]).reshape(-1)


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("max_norm", [None, 0.5, 1e6])
def test_every_bit_of_a_step(AdamW, bits, max_norm):
    n, lr, b1, b2, eps, wd, seed = 256 * 273, 1e-3, 0.9, 0.999, 1e-8, 0.01, 99
    gen = torch.Generator().manual_seed(bits)
    p = (torch.randn(n, generator=gen) * 0.1).cuda()
    opt = AdamW([p], lr=lr, betas=(b1, b2), eps=eps, weight_decay=wd, state_bits=bits, seed=seed)
    P, M, V = p.cpu().numpy().copy(), np.zeros(n, F), np.zeros(n, F)
    for t in range(1, 5):
        g = torch.randn(n, generator=gen) * torch.exp(torch.randn(n, generator=gen)) * 1e-2
        norm = opt.step([g.cuda()], max_norm=max_norm)
        G = g.numpy()
        if max_norm is not None:
            assert abs(float(norm) - float(np.sqrt((G.astype(np.float64) ** 2).sum()))) <= 2.0 ** -23 * float(norm)
            scale = F(norm.item())                                  # (the sum's order is the kernel's own: its norm is taken from there)
            G = G * (F(max_norm) / scale if scale > F(max_norm) else F(1))
        M = M + F(1 - b1) * (G - M)
        V = V * F(b2) + (F(1 - b2) * G) * G
        R = np.sqrt(V)
        P = P * F(1 - lr * wd) - F(lr / (1 - b1 ** t)) * (M / (R * F(1 / math.sqrt(1 - b2 ** t)) + F(eps)))
        assert np.array_equal(p.cpu().numpy(), P), t
        if bits == 32:
            assert np.array_equal(opt.m.cpu().numpy(), M) and np.array_equal(opt.v.cpu().numpy(), V), t
            continue
        word = _words(n, seed, t)
        m8, ms = _encode(M, word >> np.uint32(16), False)
        r8, rs = _encode(R, word & np.uint32(0xFFFF), True)
        for got, want in ((opt.m8, m8), (opt.r8, r8)):
            assert np.array_equal(got.view(torch.uint8).cpu().numpy(), want), t
        assert np.array_equal(opt.m_scale.cpu().numpy(), ms) and np.array_equal(opt.r_scale.cpu().numpy(), rs), t
        M, V = _decode(m8, ms), _decode(r8, rs) ** 2


def test_smallest_and_largest_second_moments(AdamW):
    """roots of subnormal and of huge numbers, and none: v = (1 - b2) g^2 with b2 = 0 is g^2"""
    g = torch.tensor([0.0, 1e-23, 3e-23, 1e-22, 1.1e-19, 1e-10, 1.0, 1e10, 1.8e19, 1e-45])
    p = torch.zeros(len(g), device="cuda")
    opt = AdamW([p], lr=1.0, betas=(0.0, 0.0), eps=1e-30, weight_decay=0.0)
    opt.step([g.cuda()])
    G = g.numpy()
    V = F(1) * G * G
    P = F(0) - F(1) * (G / (np.sqrt(V) + F(1e-30)))
    assert np.array_equal(p.cpu().numpy(), P) and np.array_equal(opt.v.cpu().numpy()[:len(g)], V)


def test_a_second_step_refuses_what_a_first_one_does(AdamW):
    """a gradient of the same strides, size, type and device that is not the parameter's like: part of a wider matrix"""
    p = torch.zeros(4, 6, device="cuda")
    opt = AdamW([p], lr=1e-2)
    opt.step([torch.ones(4, 6, device="cuda")])
    before = p.clone()
    for bad in (torch.ones(8, 6, device="cuda")[:, :3], torch.ones(24, device="cuda").as_strided((3, 8), (6, 1)), torch.ones(24, device="cuda"),
                torch.ones(4, 6), torch.ones(4, 6, device="cuda").double()):
        with pytest.raises((ValueError, TypeError)):
            opt.step([bad])
    assert opt.step_count == 1 and torch.equal(p, before)
    opt.step([torch.ones(4, 6, device="cuda", dtype=torch.float16)])
    assert opt.step_count == 2


@pytest.mark.parametrize("bits", [32, 8])
def test_the_agents_own_networks(AdamW, bits):
    """the rows of a NetView's matrices are padded in one flat buffer: a step moves what belongs to the network, bit for bit, and leaves the padding zero and
    the other networks as they were; gradients with the parameters' strides, or dense"""
    from oracle import fb_oracle as fo
    from tests import helpers as H
    cfg = fo.OracleConfig(obs_dim=5, action_dim=3, goal_dim=5, z_dim=10, hidden_dim=36, feature_dim=16, backward_hidden_dim=22, batch_size=32)
    rng = np.random.default_rng(4)
    agent = H.make_hip_agent(cfg, {n: fo.synthetic_params(rng, fo.NET_SHAPES[n](cfg)) for n in ("actor", "forward_net", "backward_net")})
    params = list(agent.forward_net.parameters()) + list(agent.backward_net.parameters())
    assert any(not p.is_contiguous() for p in params) and all(p.is_cuda for p in params)
    others = {n: {k: v.clone() for k, v in getattr(agent, n).state_dict().items()} for n in ("actor", "forward_target_net", "backward_target_net")}
    lr, b1, b2, eps, wd = 1e-3, 0.9, 0.999, 1e-8, 0.01
    opt = AdamW(params, lr=lr, betas=(b1, b2), eps=eps, weight_decay=wd, state_bits=bits)
    P = [p.cpu().numpy().copy() for p in params]
    gen = torch.Generator().manual_seed(bits)
    G = [(torch.randn(p.shape, generator=gen) * 1e-2) for p in params]
    grads = [g.cuda() if k % 2 else torch.empty_strided(p.shape, p.stride(), device="cuda").copy_(g) for k, (g, p) in enumerate(zip(G, params))]
    opt.step(grads)
    for k, (p, want, g) in enumerate(zip(params, P, (g.numpy() for g in G))):
        M = F(0) + F(1 - b1) * (g - F(0))
        V = F(0) * F(b2) + (F(1 - b2) * g) * g
        want = want * F(1 - lr * wd) - F(lr / (1 - b1)) * (M / (np.sqrt(V) * F(1 / math.sqrt(1 - b2)) + F(eps)))
        assert np.array_equal(p.cpu().numpy(), want), k
        if bits == 32:
            m, v = (x.cpu().numpy().reshape(p.shape) for x in opt.moments(k))
            assert np.array_equal(m, M) and np.array_equal(v, V), k
    assert agent.forward_net.pad_abs_max() == 0 and agent.backward_net.pad_abs_max() == 0 and agent.actor.pad_abs_max() == 0
    for n, was in others.items():
        assert all(torch.equal(v, was[k]) for k, v in getattr(agent, n).state_dict().items()), n
