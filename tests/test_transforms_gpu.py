"""The few-token layer and linear / grouped_linear under torch's tracers and forward-mode
differentiation: the same results as the eager call, or an error."""
import math

import pytest
import torch
import torch.autograd.forward_ad as fw
from torch._subclasses.fake_tensor import FakeTensorMode
from torch.fx.experimental.proxy_tensor import make_fx

import moe_ops_b200 as M
from moe_ops_b200.moe_layer import MoELayer

pytestmark = pytest.mark.gpu

BF = torch.bfloat16


def calls(dev):
    """name -> (function of one tensor, two inputs)."""
    g = torch.Generator(device=dev).manual_seed(3)
    rnd = lambda *s: torch.randn(*s, device=dev, generator=g).to(BF)  # noqa: E731
    w, b, r = rnd(40, 64), rnd(40), rnd(12, 40)
    B, off = rnd(3, 40, 64), torch.tensor([0, 5, 5, 11], device=dev, dtype=torch.int32)
    wo = rnd(33, 64)  # no 16-byte multiple
    wr, wg, wu, wd = rnd(8, 64), rnd(8, 48, 64), rnd(8, 48, 64), rnd(8, 64, 48)
    p, i = torch.rand(12, 2, device=dev, generator=g), torch.randint(0, 8, (12, 2), device=dev, generator=g)
    m = MoELayer(64, 8, 2, 48, device=dev, dtype=BF, shared_hidden=32)
    m.init_normal(0.1, g).requires_grad_(False)
    m.few_tokens = 16
    fs = {
        "linear": lambda x: M.linear(x, w, bias=b, activation="gelu", residual=r),
        "linear_odd": lambda x: M.linear(x, wo, activation="silu"),
        "grouped_linear": lambda x: M.grouped_linear(x, B, off, activation="relu", residual=r),
        "moe_few_tokens": lambda x: M.moe_few_tokens(x, wr, wg, wu, wd, 2),
        "moe_few_experts": lambda x: M.moe_few_experts(x, p, i, wg, wu, wd),
        "layer": lambda x: m(x),
    }
    return fs, (rnd(12, 64), rnd(12, 64))


NAMES = ["linear", "linear_odd", "grouped_linear", "moe_few_tokens", "moe_few_experts", "layer"]


@pytest.mark.parametrize("how", ["jit", "make_fx", "compile"])
@pytest.mark.parametrize("name", NAMES)
def test_recorded_calls_compute_again(cuda_dev, name, how):
    fs, (x0, x1) = calls(cuda_dev)
    f = fs[name]
    if how == "jit":
        t = torch.jit.trace(f, (x0,), check_trace=False)
    elif how == "make_fx":
        t = make_fx(f)(x0)
    else:
        t = torch.compile(f, backend="aot_eager")
        t(x0)
    want = f(x1)
    torch.empty_like(want).fill_(math.nan)  # what an unwritten result would show
    assert torch.equal(t(x1), want)


@pytest.mark.parametrize("act", ["none", "silu"])
def test_a_recorded_training_step_computes_again(cuda_dev, act):
    g = torch.Generator(device=cuda_dev).manual_seed(4)
    args = [[torch.randn(*s, device=cuda_dev, generator=g).to(BF)
             for s in ((20, 64), (24, 64), (24,), (20, 24), (20, 24))] for _ in range(2)]

    def step(x, w, b, r, dy):
        leaf = [t.detach().requires_grad_(True) for t in (x, w, b, r)]
        y = M.linear(leaf[0], leaf[1], bias=leaf[2], activation=act, residual=leaf[3])
        return [y.detach(), *torch.autograd.grad(y, leaf, dy)]

    t = make_fx(step)(*args[0])
    assert all(torch.equal(a, c) for a, c in zip(t(*args[1]), step(*args[1])))

    def loss(x, w, b, r, dy):
        return (M.linear(x, w, bias=b, activation=act, residual=r).float() * dy.float()).sum()

    both = []
    for f in (loss, torch.compile(loss, backend="aot_eager")):
        leaf = [t.clone().requires_grad_(True) for t in args[1][:4]]
        f(*leaf, args[1][4]).backward()
        both.append([t.grad for t in leaf])
    assert all(torch.equal(a, c) for a, c in zip(*both))


def test_gradients_of_fake_tensors(cuda_dev):
    with FakeTensorMode():
        x, w, b, dy = (torch.empty(*s, device=cuda_dev, dtype=BF) for s in ((40, 64), (24, 64), (24,), (40, 24)))
        leaf = [t.requires_grad_(True) for t in (x, w, b)]
        y = M.linear(leaf[0], leaf[1], bias=leaf[2], activation="silu")
        for got, t in zip(torch.autograd.grad(y, leaf, dy), leaf):
            assert got.shape == t.shape and got.dtype == t.dtype and got.device == t.device


@pytest.mark.parametrize("name", NAMES)
def test_forward_mode_raises(cuda_dev, name):
    fs, (x0, x1) = calls(cuda_dev)
    want = fs[name](x0)
    with fw.dual_level():
        with pytest.raises((RuntimeError, NotImplementedError)):
            fs[name](fw.make_dual(x0, x1))
        assert torch.equal(fs[name](x0), want)  # no tangent: as outside


def test_forward_mode_raises_for_every_operand(cuda_dev):
    g = torch.Generator(device=cuda_dev).manual_seed(5)
    rnd = lambda *s: torch.randn(*s, device=cuda_dev, generator=g)  # noqa: E731
    lin = [rnd(12, 64), rnd(40, 64), rnd(40), rnd(12, 40)]
    few = [rnd(6, 64), rnd(8, 64), rnd(8, 48, 64), rnd(8, 48, 64), rnd(8, 64, 48), rnd(8)]
    ex = [rnd(6, 64), rnd(6, 2), rnd(8, 48, 64), rnd(8, 48, 64), rnd(8, 64, 48)]
    idx = torch.randint(0, 8, (6, 2), device=cuda_dev, generator=g)
    fs = [(lin, lambda a: M.linear(a[0], a[1], bias=a[2], residual=a[3])),
          (few, lambda a: M.moe_few_tokens(*a[:5], 2, router_bias=a[5])),
          (ex, lambda a: M.moe_few_experts(a[0], a[1], idx, *a[2:]))]
    for args, f in fs:
        for j in range(len(args)):
            with fw.dual_level(), pytest.raises((RuntimeError, NotImplementedError)):
                f([fw.make_dual(t, torch.ones_like(t)) if i == j else t for i, t in enumerate(args)])


@pytest.mark.parametrize("name", NAMES)
def test_functorch_is_right_or_raises(cuda_dev, name):
    fs, (x0, x1) = calls(cuda_dev)
    f = fs[name]
    both = torch.stack([x0, x1])
    try:
        got = torch.vmap(f)(both)
    except (RuntimeError, NotImplementedError):
        pass
    else:
        assert torch.equal(got, torch.stack([f(x0), f(x1)]))
    with pytest.raises((RuntimeError, NotImplementedError)):
        torch.func.jvp(f, (x0,), (x1,))


def test_registered_ops(cuda_dev):
    g = torch.Generator(device=cuda_dev).manual_seed(6)
    rnd = lambda *s: torch.randn(*s, device=cuda_dev, generator=g).to(BF)  # noqa: E731
    ops, checks = torch.ops.moeb200, ("test_schema", "test_faketensor")
    x, w, b, r, dy = rnd(12, 64), rnd(40, 64), rnd(40), rnd(12, 40), rnd(12, 40)
    z = rnd(12, 40)
    for want_z in (False, True):
        torch.library.opcheck(ops.linear_fwd, (x, w, b, r, None, 4, True, want_z), test_utils=checks)
    for want in ((True, True, True), (True, False, False), (False, True, True)):
        torch.library.opcheck(ops.linear_bwd, (dy, x, w, z, None, 4, True, *want), test_utils=checks)
    B, off = rnd(3, 64, 40), torch.tensor([0, 5, 5, 11], device=cuda_dev, dtype=torch.int32)
    torch.library.opcheck(ops.linear_fwd, (x, B, None, None, off, 0, False, False), test_utils=checks)
    torch.library.opcheck(ops.linear_bwd, (dy, x, B, None, off, 0, False, True, True, True), test_utils=checks)
    wr, wg, wd = rnd(8, 64), rnd(8, 48, 64), rnd(8, 64, 48)
    torch.library.opcheck(ops.few_tokens, (x, wr, wg, wg, wd, 2, None), test_utils=checks)
    p, i = torch.rand(12, 2, device=cuda_dev), torch.zeros(12, 2, device=cuda_dev, dtype=torch.int32)
    torch.library.opcheck(ops.few_experts, (x, p, i, wg, wg, wd), test_utils=checks)


def test_a_tangent_of_the_output_gradient_raises(cuda_dev):
    g = torch.Generator(device=cuda_dev).manual_seed(7)
    x, w, dy = (torch.randn(*s, device=cuda_dev, generator=g) for s in ((9, 24), (16, 24), (9, 16)))
    x.requires_grad_(True)
    y = M.linear(x, w, activation="silu")
    with fw.dual_level(), pytest.raises((RuntimeError, NotImplementedError)):
        torch.autograd.grad(y, x, fw.make_dual(dy, torch.ones_like(dy)))
    y = M.linear(x, w, activation="silu")
    with fw.dual_level():
        got = torch.autograd.grad(y, x, dy)[0]
    y = M.linear(x, w, activation="silu")
    assert torch.equal(got, torch.autograd.grad(y, x, dy)[0])
