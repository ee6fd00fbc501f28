"""Activations kept in eight bits (``ecoint8.checkpoint``) against the oracle in 64 bits.

The eight bits themselves are defined by fp32 roundings, so they are compared for equality;
everything after them by a bound: half a step of the output's type, plus the fp32 error of
the formula (counted at each test).
"""

import math

import pytest
import torch

from oracle import ckpt8 as orc

pytestmark = pytest.mark.gpu

TYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
U = 2.0 ** -24


def _half(dtype):
    return torch.finfo(dtype).eps / 2


def _floor(dtype):
    """Half a step among the type's subnormal numbers."""
    return torch.finfo(dtype).tiny * torch.finfo(dtype).eps / 2


def _x(rows, cols, dtype, seed, scale=1.0):
    gen = torch.Generator().manual_seed(seed)
    x = torch.randn(rows, cols, generator=gen) * torch.exp(torch.randn(cols, generator=gen)) * scale
    return x.to(dtype).cuda(), gen


SHAPES = [(1, 1), (3, 2), (1, 127), (5, 128), (4, 129), (7, 784), (2, 1000), (33, 1337), (300, 9), (2, 4097),
          (1, 20011), (65, 2048)]


@pytest.mark.parametrize("name", TYPES)
@pytest.mark.parametrize("rows,cols", SHAPES)
def test_eight_bits_are_the_definitions(name, rows, cols):
    from ecoint8.checkpoint import checkpoint_i8, restore_i8

    x, _ = _x(rows, cols, TYPES[name], rows + cols)
    c = checkpoint_i8(x)
    want = orc.stands_for(x)
    got = restore_i8(c)
    assert got.shape == x.shape and got.dtype == x.dtype
    # q * scale is one fp32 product, rounded again to the type
    assert torch.equal(restore_i8(c, torch.float32).double(), want.float().double())
    assert torch.equal(got, want.float().to(x.dtype))
    # and what it is for: half a step of a block's scale, plus the fp32 roundings
    amax = torch.cat([p.abs().amax(1, keepdim=True).expand(-1, p.shape[1]) for p in x.double().split(128, 1)], 1)
    assert ((want - x.double()).abs() <= amax / 127 * (0.5 + 2.0 ** -15)).all()
    assert c.memory_bytes() == rows * (-(-cols // 16) * 16 + 4 * -(-cols // 128))


@pytest.mark.parametrize("name", TYPES)
def test_strides_alignment_and_shapes(name):
    from ecoint8.checkpoint import checkpoint_i8, restore_i8

    big, _ = _x(40, 700, TYPES[name], 3)
    for x in (big[:, 1:], big[:, 3:260], big[::3, 5:], big.t(), big[:, ::2], big.view(4, 10, 700)[:, 2:5, 7:],
              big[0], big[5, 3:9], big[1:2].expand(7, -1), big[:, :128], big[:0], big.view(5, 8, 700)[:, :0]):
        got = restore_i8(checkpoint_i8(x))
        assert got.shape == x.shape
        flat = x.reshape(-1, x.shape[-1])
        assert torch.equal(got.reshape(flat.shape), orc.stands_for(flat).float().to(x.dtype))


# More rows than are in work at a time, by the number of blocks that stand side by side in a CTA.
@pytest.mark.parametrize("name", TYPES)
@pytest.mark.parametrize("rows,cols", [(150001, 120), (90001, 256), (50003, 384), (20001, 1001), (10007, 2048)])
def test_eight_bits_of_many_rows(name, rows, cols):
    from ecoint8.checkpoint import checkpoint_i8, restore_i8

    x, _ = _x(rows, cols, TYPES[name], cols)
    assert torch.equal(restore_i8(checkpoint_i8(x), torch.float32).double(), orc.stands_for(x).float().double())
    assert torch.equal(restore_i8(checkpoint_i8(x)), orc.stands_for(x).float().to(x.dtype))


def test_zeros_tiny_huge_and_not_finite_blocks():
    from ecoint8.checkpoint import checkpoint_i8, restore_i8

    x = torch.zeros(8, 300)
    x[1, 5] = 2.0 ** -120           # below the smallest block maximum
    x[2, 7], x[2, 9] = 2.0 ** -118, -(2.0 ** -119)
    x[3, 128:256] = torch.linspace(-3.3e38, 3.4e38, 128)
    x[4, 130] = math.inf
    x[4, 3] = 2.0
    x[5, 299] = math.nan
    x[6, 0], x[6, 1] = -math.inf, math.nan
    got = restore_i8(checkpoint_i8(x.cuda())).cpu()
    want = orc.stands_for(x).float()
    assert torch.equal(torch.isnan(got), torch.isnan(want))
    assert torch.equal(torch.nan_to_num(got, nan=0.0), torch.nan_to_num(want, nan=0.0))
    assert (got[:2] == 0).all() and torch.isnan(got[4, 128:256]).all() and got[4, 3] == 2.0
    assert torch.isnan(got[5, 256:]).all() and torch.isnan(got[6, :128]).all() and (got[6, 128:] == 0).all()


# --------------------------------------------------------------------- rms norm

WIDTHS = [1, 2, 7, 128, 200, 256, 257, 784, 1000, 1024, 1025, 3001, 4096, 4097, 8192, 8200, 16384, 16385, 20001]


@pytest.mark.parametrize("name", TYPES)
@pytest.mark.parametrize("cols", WIDTHS)
def test_rms_norm(name, cols):
    _rms_case(TYPES[name], 5 if cols > 1000 else 23, cols, TYPES[name], cols)


@pytest.mark.parametrize("name,wname,rows,cols", [("bf16", "fp32", 700, 520), ("fp16", "fp32", 3, 8192),
                                                  ("fp32", None, 9, 333), ("bf16", None, 1, 18000),
                                                  ("fp32", "fp32", 1500, 96), ("bf16", "bf16", 5000, 40),
                                                  ("bf16", "fp32", 400, 17000)])
def test_rms_norm_weights_and_many_rows(name, wname, rows, cols):
    _rms_case(TYPES[name], rows, cols, TYPES[wname] if wname else None, rows)


# Every number of threads per row, with more rows than fit the stages of all CTAs at a time.
@pytest.mark.parametrize("name,rows,cols", [("bf16", 12001, 256), ("fp32", 12001, 256), ("fp16", 10001, 512),
                                            ("fp32", 10001, 388), ("bf16", 9001, 1000), ("fp32", 9001, 1024),
                                            ("bf16", 6001, 2048), ("fp32", 6001, 1500), ("fp16", 4001, 4096),
                                            ("fp32", 3001, 4096), ("bf16", 2001, 8192), ("fp32", 2001, 8000),
                                            ("bf16", 1101, 16384), ("fp32", 1101, 16384), ("fp16", 3001, 4095)])
def test_rms_norm_of_every_width_many_times_over(name, rows, cols):
    _rms_case(TYPES[name], rows, cols, TYPES[name], rows + cols)


def _rms_case(dtype, rows, cols, wtype, seed):
    from ecoint8.checkpoint import rms_norm_i8

    x, gen = _x(rows, cols, dtype, seed)
    w = None if wtype is None else (torch.rand(cols, generator=gen) + 0.5).to(wtype).cuda().requires_grad_()
    dy = torch.randn(rows, cols, generator=gen).to(dtype).cuda()
    leaf = x.detach().requires_grad_()
    y = rms_norm_i8(leaf, w, eps=1e-5)
    grads = torch.autograd.grad(y, (leaf,) if w is None else (leaf, w), dy)
    wy, wdx, wdw = orc.rms_norm(x, None if w is None else w.detach(), dy, 1e-5)
    # The sum of squares: at most 32 fp32 additions per thread in a row that its threads hold
    # (cols / 512 in wider ones) and 9 joins, every term positive; the root halves its error, and
    # rsqrt, the products and the division add 2^-22.
    adds = max(32, cols // 512) + 16
    e = adds * U
    assert y.dtype == dtype and y.shape == x.shape
    assert ((y.double() - wy).abs() <= wy.abs() * (_half(dtype) + e) + _floor(dtype)).all()
    # dx = rstd (w dy - u m): each factor has e; the mean's sum has the same additions, over terms of either sign
    rstd = 1 / torch.sqrt(x.double().square().mean(1, keepdim=True) + 1e-5)
    u = orc.stands_for(x) * rstd
    wd = (1.0 if w is None else w.detach().double()) * dy.double()
    mean_abs = (wd * u).abs().mean(1, keepdim=True)
    tol = wdx.abs() * _half(dtype) + rstd * (wd.abs() * e + u.abs() * mean_abs * 3 * e) + 2.0 ** -126 + _floor(dtype)
    assert grads[0].dtype == dtype and ((grads[0].double() - wdx).abs() <= tol).all()
    if w is not None:
        # a partial sum adds its rows in fp32 (each row group at most rows / 148 + 1 of them), joined in fp64
        size = (dy.double() * u).abs().sum(0)
        tol = wdw.abs() * _half(wtype) + size * (rows / 148 + 2 + 16) * U + size * e + torch.finfo(wtype).tiny
        assert grads[1].dtype == wtype and ((grads[1].double() - wdw).abs() <= tol).all()


def test_rms_norm_shapes_strides_and_one_gradient_at_a_time():
    from ecoint8.checkpoint import Int8RMSNorm, rms_norm_i8

    x, gen = _x(24, 260, torch.float32, 5)
    w = torch.rand(258, generator=gen).cuda().requires_grad_()
    part = x[:, 1:259]
    leaf = part.detach().view(24, 258).requires_grad_()
    dy = torch.randn(24, 520, generator=gen).cuda()[:, ::2][:, :258]
    y = rms_norm_i8(leaf, w)
    dx, dw = torch.autograd.grad(y, (leaf, w), dy)
    cube = part.reshape(2, 3, 4, 258).requires_grad_()
    y3 = rms_norm_i8(cube, w)
    dx3, dw3 = torch.autograd.grad(y3, (cube, w), dy.reshape(2, 3, 4, 258))
    assert torch.equal(y3.reshape(24, 258), y) and torch.equal(dx3.reshape(24, 258), dx) and torch.equal(dw, dw3)
    frozen = w.detach()
    (dx1,) = torch.autograd.grad(rms_norm_i8(leaf, frozen), leaf, dy)
    (dw1,) = torch.autograd.grad(rms_norm_i8(part.detach(), w), w, dy)
    assert torch.equal(dx1, dx) and torch.equal(dw1, dw)
    # an expanded gradient (of a sum) is read with its zero strides
    (ds,) = torch.autograd.grad(rms_norm_i8(leaf, w).sum(), leaf)
    (dt,) = torch.autograd.grad(rms_norm_i8(leaf, w), leaf, torch.ones(24, 258).cuda())
    assert torch.equal(ds, dt)
    with torch.no_grad():
        assert torch.equal(rms_norm_i8(leaf, w), y)
    m = Int8RMSNorm(258).cuda()
    assert torch.equal(m(part), rms_norm_i8(part, None, 1e-6))
    e = torch.zeros(0, 258).cuda().requires_grad_()
    de, dw0 = torch.autograd.grad(rms_norm_i8(e, w), (e, w), torch.zeros(0, 258).cuda())
    assert de.shape == (0, 258) and (dw0 == 0).all()


def test_rms_norm_of_zero_rows_and_differences():
    """A row of zeros: y = 0, dx = dy w / sqrt(eps).  And dx along a direction against central
    differences of the fp64 formula at the values that the eight bits stand for."""
    from ecoint8.checkpoint import rms_norm_i8

    z = torch.zeros(2, 300).cuda().requires_grad_()
    w = torch.rand(300).cuda()
    y = rms_norm_i8(z, w, eps=1e-4)
    (dz,) = torch.autograd.grad(y, z, torch.ones_like(y))
    assert (y == 0).all() and ((dz.double() - w.double() / 1e-2).abs() <= w.double() * 100 * 2.0 ** -20).all()
    gen = torch.Generator().manual_seed(2)
    x = orc.stands_for(torch.randn(3, 256, generator=gen)).float().cuda()  # its own eight bits
    x = torch.where(torch.isfinite(x), x, 0.0)
    if not torch.equal(orc.stands_for(x).float(), x):
        x = orc.stands_for(x).float()
    leaf = x.clone().requires_grad_()
    dy = torch.randn(3, 256, generator=gen).cuda()
    w = torch.rand(256, generator=gen).cuda()
    (dx,) = torch.autograd.grad(rms_norm_i8(leaf, w), leaf, dy)

    def f(v):
        return (v * torch.rsqrt(v.square().mean(1, keepdim=True) + 1e-6) * w.double() * dy.double()).sum()

    h = 2.0 ** -10
    for _ in range(3):
        d = torch.randn(3, 256, generator=gen).cuda().double()
        d /= d.norm()
        diff = (f(x.double() + h * d) - f(x.double() - h * d)) / (2 * h)
        # the norm's third derivative along a unit direction is below |dy w|_2 here: h^2 / 6 of it;
        # dx itself has fp32's 2^-18 of its size
        size = (dy.double() * w.double()).norm()
        assert abs(diff - (dx.double() * d).sum()) <= size * (h * h + 2.0 ** -18)


# --------------------------------------------------------------------- gated activation


@pytest.mark.parametrize("act", ["silu", "gelu"])
@pytest.mark.parametrize("name", TYPES)
@pytest.mark.parametrize("rows,cols,packed", [(1, 1, True), (3, 5, True), (4, 128, True), (9, 1337, True),
                                              (2, 2000, False), (40, 129, False), (300, 3, False), (5, 8192, True),
                                              (60001, 128, True), (30001, 200, False), (9001, 1001, True),
                                              (5003, 2048, False)])
def test_gated_activation(act, name, rows, cols, packed):
    from ecoint8.checkpoint import gated_act_i8

    dtype = TYPES[name]
    x, gen = _x(rows, 2 * cols, dtype, rows * cols)
    dy = torch.randn(rows, cols, generator=gen).to(dtype).cuda()
    gate, up = x[:, :cols], x[:, cols:]
    if packed:
        leaf = x.detach().requires_grad_()
        y = gated_act_i8(leaf, act=act)
        (dx,) = torch.autograd.grad(y, leaf, dy)
        assert dx.shape == x.shape
        dg, du = dx[:, :cols], dx[:, cols:]
    else:
        a, b = gate.detach().requires_grad_(), up.detach().requires_grad_()
        y = gated_act_i8(a, b, act=act)
        dg, du = torch.autograd.grad(y, (a, b), dy)
    wy, wg, wu = orc.gated(gate, up, dy, act)
    # fp32: the exponential's argument is rounded (|g| 2^-24 relative to the result, and the
    # result only matters while |g| < 104), erf and exp are good to 2^-21, a few products.
    g, u = gate.double(), up.double()
    kg, ku = orc.stands_for(gate), orc.stands_for(up)

    def err(v):
        return (v.abs().clamp(max=104) * 2 + 32) * U

    # gelu's distribution is a rational approximation with the absolute error 7.5e-8, evaluated in
    # fp32 from terms below 1 (2^-24 more): together below 2^-22
    low = (lambda v: v.abs() * 2.0 ** -22) if act == "gelu" else (lambda v: v.abs() * 2.0 ** -126)
    tol = wy.abs() * (_half(dtype) + err(g)) + low(g) * u.abs() + 2.0 ** -126
    if dtype == torch.float16:
        tol = tol + 2.0 ** -25
    assert y.dtype == dtype and ((y.double() - wy).abs() <= tol).all()
    d = dy.double().abs()
    extra = 2.0 ** -25 if dtype == torch.float16 else 2.0 ** -126
    tol = wu.abs() * (_half(dtype) + err(kg)) + low(kg) * d + extra
    assert ((du.double() - wu).abs() <= tol).all()
    # act' sums terms of either sign, each below 1 + |g|
    slope_err = (1 + kg.abs()) * err(kg) + (2.0 ** -22 if act == "gelu" else 0)
    tol = wg.abs() * _half(dtype) + d * ku.abs() * slope_err + extra
    assert dg.dtype == dtype and ((dg.double() - wg).abs() <= tol).all()


def test_gated_views_shapes_and_one_gradient_at_a_time():
    from ecoint8.checkpoint import Int8GatedAct, gated_act_i8

    x, gen = _x(12, 2 * 77, torch.bfloat16, 9)
    leaf = x.view(3, 4, 154).detach().requires_grad_()
    dy = torch.randn(3, 4, 77, generator=gen).to(torch.bfloat16).cuda()
    y = Int8GatedAct()(leaf)
    (dx,) = torch.autograd.grad(y, leaf, dy)
    a, b = leaf.detach()[..., :77].requires_grad_(), leaf.detach()[..., 77:].requires_grad_()
    y2 = gated_act_i8(a, b)
    da, db = torch.autograd.grad(y2, (a, b), dy)
    assert torch.equal(y, y2) and torch.equal(dx, torch.cat([da, db], -1))
    (da1,) = torch.autograd.grad(gated_act_i8(a, b.detach()), a, dy)
    assert torch.equal(da1, da)
    e = torch.zeros(0, 10).cuda().requires_grad_()
    assert torch.autograd.grad(gated_act_i8(e).sum(), e)[0].shape == (0, 10)


def test_inputs_that_are_not_finite_stay_visible():
    from ecoint8.checkpoint import gated_act_i8, rms_norm_i8

    x = torch.ones(2, 256).cuda()
    x[0, 3] = float("inf")
    leaf = x.requires_grad_()
    (dx,) = torch.autograd.grad(gated_act_i8(leaf).sum(), leaf)
    assert torch.isnan(dx[0, :128]).all() and torch.isfinite(dx[1]).all()
    (dx,) = torch.autograd.grad(rms_norm_i8(leaf).sum(), leaf)
    assert torch.isnan(dx[0]).any() and torch.isfinite(dx[1]).all()


def test_graph_streams_and_same_bits():
    from ecoint8.checkpoint import checkpoint_i8, gated_act_i8, restore_i8, rms_norm_i8

    x, gen = _x(70, 1026, torch.bfloat16, 4)
    w = torch.rand(1026, generator=gen).to(torch.bfloat16).cuda()
    dy = torch.randn(70, 1026, generator=gen).to(torch.bfloat16).cuda()

    def step():
        a, v = x.detach().requires_grad_(), w.detach().requires_grad_()
        y = rms_norm_i8(a, v)
        z = gated_act_i8(y)
        dx, dw = torch.autograd.grad((y, z), (a, v), (dy, dy[:, :513].contiguous()))
        return [y.detach(), z.detach(), dx, dw, restore_i8(checkpoint_i8(x))]

    want = step()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = step()
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    x.copy_(torch.randn(x.shape, generator=gen).to(x.dtype))
    graph.replay()
    want = step()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(out, want))


def test_backward_twice_and_of_two_calls_in_either_order():
    """Each call keeps its own bytes: a backward may run twice, or after another call's."""
    from ecoint8.checkpoint import gated_act_i8, rms_norm_i8

    x, gen = _x(40, 516, torch.float32, 8)
    x2, _ = _x(40, 516, torch.float32, 9)
    w = torch.rand(516, generator=gen).cuda().requires_grad_()
    a, b = x.requires_grad_(), x2.requires_grad_()
    dy = torch.randn(40, 516, generator=gen).cuda()
    ya, yb = rms_norm_i8(a, w), rms_norm_i8(b, w)
    gb, ga = torch.autograd.grad(yb, (b, w), dy, retain_graph=True), torch.autograd.grad(ya, (a, w), dy,
                                                                                        retain_graph=True)
    again = torch.autograd.grad(ya, (a, w), dy)
    assert all(torch.equal(u, v) for u, v in zip(ga, again))
    both = torch.autograd.grad(rms_norm_i8(a, w), (a, w), dy), torch.autograd.grad(rms_norm_i8(b, w), (b, w), dy)
    assert all(torch.equal(u, v) for u, v in zip(ga + gb, both[0] + both[1]))
    za, zb = gated_act_i8(a), gated_act_i8(b)
    (hb,), (ha,) = torch.autograd.grad(zb.sum(), b), torch.autograd.grad(za.sum(), a)
    assert torch.equal(ha, torch.autograd.grad(gated_act_i8(a).sum(), a)[0])
    assert torch.equal(hb, torch.autograd.grad(gated_act_i8(b).sum(), b)[0])


def test_offsets_beyond_32_bits():
    from ecoint8.checkpoint import checkpoint_i8, gated_act_i8, restore_i8, rms_norm_i8

    rows, cols = 131080, 16384
    x = torch.zeros(rows, cols, dtype=torch.bfloat16, device="cuda")
    x[-2:] = torch.randn(2, cols).to(torch.bfloat16).cuda()
    last = x[-2:].clone()
    c = checkpoint_i8(x)
    assert torch.equal(restore_i8(c)[-2:], restore_i8(checkpoint_i8(last)))
    del c
    assert torch.equal(rms_norm_i8(x)[-2:], rms_norm_i8(last))
    assert torch.equal(gated_act_i8(x)[-2:], gated_act_i8(last))
    torch.cuda.empty_cache()


def test_refusals():
    from ecoint8.checkpoint import checkpoint_i8, gated_act_i8, restore_i8, rms_norm_i8

    x = torch.ones(4, 8).cuda()
    for bad in (lambda: checkpoint_i8(x.int()), lambda: checkpoint_i8(x.double()), lambda: checkpoint_i8(x[0, 0]),
                lambda: checkpoint_i8(x[:, :0]), lambda: restore_i8(checkpoint_i8(x), torch.int8),
                lambda: rms_norm_i8(x, torch.ones(7).cuda()), lambda: rms_norm_i8(x, torch.ones(8).half().cuda()),
                lambda: gated_act_i8(x[:, :7]), lambda: gated_act_i8(x, x[:, :4]), lambda: gated_act_i8(x, x.half())):
        with pytest.raises(AssertionError):
            bad()
    for bad in (lambda: rms_norm_i8(x, eps=-1.0), lambda: gated_act_i8(x, act="relu")):
        with pytest.raises(ValueError):
            bad()
    for bad in (lambda: checkpoint_i8(x.cpu()), lambda: rms_norm_i8(x.cpu()), lambda: gated_act_i8(x.cpu())):
        with pytest.raises(RuntimeError, match="CUDA"):
            bad()


# --------------------------------------------------------------------- as they are used


def test_saved_activations_in_eight_bits():
    """y = a * b saves a and b: inside the context their gradients read what eight bits stand for."""
    from ecoint8.checkpoint import saved_i8

    gen = torch.Generator().manual_seed(0)
    w = torch.nn.Parameter(torch.randn(300, 300, generator=gen).cuda())
    x = torch.randn(260, 300, generator=gen).cuda().requires_grad_()
    dy = torch.randn(260, 300, generator=gen).cuda()
    with saved_i8(min_numel=1000):
        a, b = x * 2, x + 1
        (a * b + torch.nn.functional.linear(b, w)).backward(dy)
    k = orc.stands_for((x.detach() * 2)), orc.stands_for(x.detach() + 1)
    want = dy.double() * (k[1] * 2 + k[0]) + dy.double() @ w.detach().double()  # the weight is kept whole
    size = dy.double().abs() * (k[1].abs() * 2 + k[0].abs()) + dy.double().abs() @ w.detach().double().abs()
    assert ((x.grad.double() - want).abs() <= size * 310 * U).all()
    dw = dy.double().t() @ k[1]  # the product's input in eight bits
    assert ((w.grad.double() - dw).abs() <= (dy.double().abs().t() @ k[1].abs()) * 280 * U).all()


def test_losses_and_layers_under_saved_i8_keep_their_own_state():
    """The context packs what autograd saves of the logits; statistics and scales stay whole."""
    from ecoint8.checkpoint import rms_norm_i8, saved_i8
    from ecoint8.losses import token_logprobs

    gen = torch.Generator().manual_seed(1)
    x = torch.randn(600, 256, generator=gen).cuda()
    dy = torch.randn(600, 256, generator=gen).cuda()
    leaf = x.clone().requires_grad_()
    (want,) = torch.autograd.grad(rms_norm_i8(leaf), leaf, dy)
    with saved_i8(min_numel=1):
        y = rms_norm_i8(leaf)
    assert torch.equal(torch.autograd.grad(y, leaf, dy)[0], want)
    tokens = torch.randint(0, 256, (600,), generator=gen).cuda()
    with saved_i8(min_numel=1):
        lp = token_logprobs(leaf * 1.0, tokens)
    (g,) = torch.autograd.grad(lp.sum(), leaf)
    p = torch.softmax(x.double(), -1)
    want = torch.nn.functional.one_hot(tokens, 256) - p
    # a logit is off by half a step of its block: its probability by that much relatively, and a little more
    step = x.abs().double().view(600, 2, 128).amax(2).repeat_interleave(128, 1) / 254
    assert ((g.double() - want).abs() <= p * step * 1.1 + 2.0 ** -20).all()


def test_sparse_tensors_pass_through_saved_i8():
    from ecoint8.checkpoint import saved_i8

    a = torch.eye(40).cuda().to_sparse()
    x = torch.ones(40, 30).cuda().requires_grad_()
    with saved_i8(min_numel=1):
        y = torch.sparse.mm(a, x)
    (g,) = torch.autograd.grad(y.sum(), x)
    assert torch.equal(g, torch.ones_like(g))


def test_feed_forward_block_trains():
    """Norm, Int8Linear, gated activation, Int8Linear head and the policy loss: the embedding's
    gradient against the same products with the norm and activation written out on what the
    eight bits stand for."""
    from ecoint8 import EcoSGDM, Int8GatedAct, Int8Linear, Int8RMSNorm
    from ecoint8.losses import policy_loss

    torch.manual_seed(0)
    rows, width, hidden, vocab = 96, 64, 136, 211
    emb = torch.randn(rows, width).cuda().requires_grad_()
    norm, up, act, head = Int8RMSNorm(width).cuda(), Int8Linear(width, 2 * hidden).cuda(), Int8GatedAct(), \
        Int8Linear(hidden, vocab).cuda()
    tokens = torch.randint(0, vocab, (rows,)).cuda()
    old, adv = torch.full((rows,), -math.log(vocab)).cuda(), torch.randn(rows).cuda()

    class Written(torch.autograd.Function):  # the norm and the activation by the oracle
        @staticmethod
        def forward(ctx, x, w, kind):
            ctx.save_for_backward(x, w)
            ctx.kind = kind
            if kind == "norm":
                return norm(x).detach()
            return act(x).detach()

        @staticmethod
        def backward(ctx, dy):
            x, w = ctx.saved_tensors
            if ctx.kind == "norm":
                _, dx, dw = orc.rms_norm(x, w, dy, 1e-6)
                return dx.float(), dw.float(), None
            _, dg, du = orc.gated(x[:, :hidden], x[:, hidden:], dy, "silu")
            return torch.cat([dg, du], 1).float(), None, None

    def loss_of(x, written):
        n = Written.apply(x, norm.weight, "norm") if written else norm(x)
        h = up(n)
        h = Written.apply(h, None, "act") if written else act(h)
        return policy_loss(head(h), tokens, old, adv).loss

    a = loss_of(emb, False)
    ga, gwa = torch.autograd.grad(a, (emb, norm.weight))
    grads = [l._grad_w.clone() for l in (up, head)]
    b = loss_of(emb, True)
    gb, gwb = torch.autograd.grad(b, (emb, norm.weight))
    assert torch.equal(a, b)
    # the head's weight gradient depends on nothing that differs
    assert torch.equal(grads[1], head._grad_w)
    # Int8Linear quantizes its output gradient to int8: values that differ by fp32 rounding may
    # take another of its steps (amax / 127) here and there, never two
    for u, v in ((ga, gb), (gwa, gwb), (grads[0], up._grad_w)):
        assert torch.isfinite(u).all() and u.any()
        assert (u - v).norm() <= 0.02 * v.norm()
    before = [l.w_i8.clone() for l in (up, head)]
    EcoSGDM([up, head], lr=1.0).step()
    assert all(not torch.equal(w, l.w_i8) for w, l in zip(before, (up, head)))
