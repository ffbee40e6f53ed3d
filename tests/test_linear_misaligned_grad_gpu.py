"""An output gradient that starts off a 16-byte boundary gives the gradients of an aligned one, bit for
bit: it is copied for the tensor cores."""
import math

import pytest
import torch

import moe_ops_b200 as M

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("act", ["none", "silu"])
@pytest.mark.parametrize("E", [0, 3])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_gradients(cuda_dev, dtype, E, act):
    m, k, n = 300, 512, 256
    g = torch.Generator(device=cuda_dev).manual_seed(E)
    rnd = lambda *s: torch.randn(*s, device=cuda_dev, generator=g)  # noqa: E731
    lead = (E,) if E else ()
    x, w, b = rnd(m, k).to(dtype), rnd(*lead, n, k).div(math.sqrt(k)).to(dtype), rnd(*lead, n).to(dtype)
    off = torch.tensor([0, 120, 120, 290], device=cuda_dev, dtype=torch.int32)
    dy = rnd(m, n).to(dtype)
    odd = torch.empty(m * n + 1, device=cuda_dev, dtype=dtype)[1:].view(m, n)
    odd.copy_(dy)
    assert odd.data_ptr() % 16 != 0 and odd.is_contiguous()
    got = []
    for d in (dy, odd):
        leaf = [t.clone().requires_grad_(True) for t in (x, w, b)]
        y = (M.grouped_linear(leaf[0], leaf[1], off, bias=leaf[2], activation=act) if E else
             M.linear(leaf[0], leaf[1], bias=leaf[2], activation=act))
        got.append(torch.autograd.grad(y, leaf, d))
    for a, c in zip(*got):
        assert torch.equal(a, c)
