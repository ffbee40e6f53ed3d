"""A router bias that requires a gradient: the few-token layer refuses it, and MoELayer runs the
assembled layer for it, which gives the gradient."""
import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

import moe_ops_b200 as M
from moe_ops_b200.moe_layer import MoELayer


def test_few_tokens_refuses():
    with FakeTensorMode():
        z = lambda *s: torch.empty(*s, device="cuda")  # noqa: E731
        args = (z(2, 8), z(4, 8), z(4, 6, 8), z(4, 6, 8), z(4, 8, 6), 2)
        bias = z(4).requires_grad_(True)
        with pytest.raises(RuntimeError, match="backward"):
            M.moe_few_tokens(*args, router_bias=bias)
        with torch.no_grad():
            assert M.moe_few_tokens(*args, router_bias=bias).shape == (2, 8)


def test_layer_does_not_take_the_forward_only_path():
    m = MoELayer(8, 4, 2, 6)
    m.few_tokens = 4
    m.requires_grad_(False)
    x = torch.zeros(3, 8)
    assert m._use_few_tokens(x)
    m.router_bias = torch.zeros(4)
    assert m._use_few_tokens(x)
    m.router_bias = torch.zeros(4, requires_grad=True)
    assert not m._use_few_tokens(x)
    with torch.no_grad():
        assert m._use_few_tokens(x)


@pytest.mark.gpu
def test_gradient_through_the_layer(cuda_dev):
    """Frozen weights, a bias that is learned: few_tokens changes nothing."""
    g = torch.Generator(device=cuda_dev).manual_seed(1)
    m = MoELayer(64, 4, 2, 48, device=cuda_dev, dtype=torch.float32)
    m.init_normal(0.2, g).requires_grad_(False)
    x = torch.randn(3, 64, device=cuda_dev, generator=g)
    got = []
    for few in (0, 4):
        m.few_tokens = few
        m.router_bias = torch.full((4,), 0.1, device=cuda_dev, requires_grad=True)
        (m(x) ** 2).sum().backward()
        got.append(m.router_bias.grad)
    assert (got[0] != 0).any() and torch.equal(got[0], got[1])
