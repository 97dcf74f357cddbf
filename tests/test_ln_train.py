"""LayerNorm forward with saved statistics and its backward pass (star_layer_norm_train / star_layer_norm_bwd, ln_train.h) against the
formulas in 64 bits.  Bounds: one rounding of half a step to the 16-bit type per output, and fp32 sums (a lane adds at most 64 values of a row
and joins a tree of 8; a column's sum is a chain of at most `rows` adds)."""
import os
import sys

import pytest
import torch

sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "oracle"))
import train_ops_oracle as O  # noqa: E402
from util import BACKENDS, DTYPES, make_ctx  # noqa: E402

from star_amd import lib as L  # noqa: E402

U = O.U32


@pytest.fixture(params=BACKENDS)
def backend(request):
    return request.param


def ctx_of(backend, dtype, request):
    return make_ctx(backend, dtype, request.getfixturevalue("emu_lib") if backend == "emu" else None)


def rows_of(rows, C, dtype, seed, ld=None):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(rows, C, generator=g) * torch.exp2(2 * torch.randn(rows, 1, generator=g)) + 3 * torch.randn(rows, 1, generator=g)
    x = x.to(dtype)
    if ld is not None:
        buf = torch.full((rows, ld), float("nan")).to(dtype)
        buf[:, :C] = x
        x = buf[:, :C]
    return x


def forward_bounds(x, gamma, eps, y, stats, dtype):
    """of y, mean and rstd"""
    x = x.double()
    rstd = stats[:, 1:]
    e_mean = 80 * U * x.abs().mean(1, keepdim=True)
    e_xh = rstd * (e_mean + 2 * U * (x.abs() + stats[:, :1].abs()))
    xh = (x - stats[:, :1]) * rstd
    # variance: its terms off by twice their relative error, the mean's own error enters squared
    e_rstd = 0.5 * (2 * (e_xh * xh.abs()).mean(1, keepdim=True) + (e_xh ** 2).mean(1, keepdim=True) + 90 * U)
    g = gamma.double().abs() if gamma is not None else 1.0
    e_y = O.half_step(dtype) * y.abs() + (1 + O.half_step(dtype)) * (g * (e_xh + xh.abs() * (e_rstd + 4 * U)) + 4 * U * y.abs()) + (2.0 ** -25 if dtype == torch.float16 else 0)
    return e_y, e_mean, e_rstd * rstd


def check_forward(ctx, x, gamma, beta, eps=1e-5, out=None):
    dev = ctx.torch_device
    y, st = ctx.layer_norm_train(x if x.device == dev else x.to(dev), *(None if t is None else t.to(dev) for t in (gamma, beta)), eps=eps, out=out)
    xc = x.cpu()
    ry, rs = O.layer_norm_forward(xc, gamma, beta, eps)
    ey, em, er = forward_bounds(xc, gamma, eps, ry, rs, x.dtype)
    if beta is not None:
        ey = ey + 2 * U * beta.double().abs()
    y, st = y.cpu().double(), st.cpu().double()
    assert (y - ry).abs().le(ey).all(), float(((y - ry).abs() - ey).max())
    assert (st[:, :1] - rs[:, :1]).abs().le(em + 1e-30).all() and (st[:, 1:] - rs[:, 1:]).abs().le(er).all()


def check_backward(ctx, x, gamma, seed, eps=1e-5, dy=None):
    dev, dtype = ctx.torch_device, x.dtype
    rows, C = x.shape
    if dy is None:
        dy = (0.1 * torch.randn(rows, C, generator=torch.Generator().manual_seed(seed))).to(dtype)
    gd = None if gamma is None else gamma.to(dev)
    xd, dyd = (t if t.device == dev else t.to(dev) for t in (x, dy))
    _, st = ctx.layer_norm_train(xd, gd, None, eps=eps)
    dx, dg, db = ctx.layer_norm_backward(dyd, xd, st, gd)
    xc, dyc = x.cpu(), dy.cpu()
    rx, rg, rb = O.layer_norm_backward(dyc, xc, gamma, eps)
    _, rs = O.layer_norm_forward(xc, None, None, eps)
    _, em, er = forward_bounds(xc, gamma, eps, torch.zeros(rows, C, dtype=torch.float64), rs, dtype)
    mean, rstd = rs[:, :1], rs[:, 1:]
    xh = (xc.double() - mean) * rstd
    e_xh = rstd * (em + 2 * U * (xc.double().abs() + mean.abs())) + xh.abs() * (er / rstd + 2 * U)
    a = dyc.double().abs() * (gamma.double().abs() if gamma is not None else 1.0)
    m1, m2 = a.mean(1, keepdim=True), (a * xh.abs()).mean(1, keepdim=True)
    e = rstd * (90 * U * (m1 + xh.abs() * m2) + 8 * U * a + e_xh * m2 + xh.abs() * (a * e_xh).mean(1, keepdim=True)) + er * (a + m1 + xh.abs() * m2)
    u = O.half_step(dtype)
    assert (dx.cpu().double() - rx).abs().le(u * rx.abs() + (1 + u) * e + (2.0 ** -25 if dtype == torch.float16 else 0)).all()
    d = dyc.double().abs()
    assert (dg.cpu().double() - rg).abs().le((d * e_xh).sum(0) + (rows + 16) * U * (d * xh.abs()).sum(0) + 1e-30).all()
    assert (db.cpu().double() - rb).abs().le((rows + 16) * U * d.sum(0) + 1e-30).all()


SIZES = [(1, 1), (3, 7), (5, 8), (65, 40), (33, 64), (7, 333), (130, 320), (9, 640), (2, 1024), (3, 2560), (2, 2561), (2, 5120), (1, 6145), (2, 16384), (3, 16383)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,C", SIZES)
def test_forward_and_backward(backend, dtype, rows, C, request):
    ctx = ctx_of(backend, dtype, request)
    x = rows_of(rows, C, dtype, rows * 7919 + C)
    g = torch.Generator().manual_seed(C)
    gamma, beta = 1 + 0.3 * torch.randn(C, generator=g), 0.2 * torch.randn(C, generator=g)
    check_forward(ctx, x, gamma, beta)
    check_forward(ctx, x, None, None)
    check_backward(ctx, x, gamma, 5)
    check_backward(ctx, x, None, 6)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,C", [(10000, 320), (4097, 640), (70001, 24), (1500, 1279), (300, 9000)])
def test_many_rows(dtype, rows, C):
    ctx = L.Context(0, dtype)
    x = rows_of(rows, C, dtype, rows + C)
    gamma = 1 + 0.3 * torch.randn(C, generator=torch.Generator().manual_seed(1))
    check_forward(ctx, x, gamma, gamma - 1)
    check_backward(ctx, x, gamma, 2)


@pytest.mark.parametrize("C,ld", [(320, 328), (320, 321), (50, 64), (2600, 2608)])
def test_row_strides_and_offsets(backend, C, ld, request):
    """rows inside a wider buffer; a stride or a start that is no multiple of 16 bytes takes the element-wise path"""
    ctx = ctx_of(backend, torch.float16, request)
    dev = ctx.torch_device
    x = rows_of(11, C, torch.float16, C + ld, ld).to(dev)
    wide = torch.full((11, ld), 7.0, dtype=torch.float16, device=dev)
    gamma = torch.linspace(0.5, 1.5, C)
    check_forward(ctx, x, gamma, None, out=wide[:, :C])
    assert bool((wide[:, C:] == 7.0).all())
    shifted = torch.zeros(11 * ld + 1, dtype=torch.float16, device=dev)[1:].reshape(11, ld)[:, :C]
    shifted.copy_(x)
    check_forward(ctx, shifted, gamma, gamma)
    check_backward(ctx, shifted, gamma, 3)


def test_in_place(backend, request):
    ctx = ctx_of(backend, torch.bfloat16, request)
    dev = ctx.torch_device
    x = rows_of(37, 640, torch.bfloat16, 2).to(dev)
    dy = rows_of(37, 640, torch.bfloat16, 3).to(dev)
    gamma = torch.linspace(0.5, 1.5, 640).to(dev)
    y, st = ctx.layer_norm_train(x, gamma)
    dx, dg, db = ctx.layer_norm_backward(dy, x, st, gamma)
    for target in ("x", "dy"):
        xc, dyc = x.clone(), dy.clone()
        got, g2, b2 = ctx.layer_norm_backward(dyc, xc, st, gamma, dx=xc if target == "x" else dyc)
        assert torch.equal(got, dx) and torch.equal(g2, dg) and torch.equal(b2, db)
    xc = x.clone()
    assert torch.equal(ctx.layer_norm_train(xc, gamma, out=xc)[0], y)


def test_no_rows_and_constant_rows(backend, request):
    ctx = ctx_of(backend, torch.float16, request)
    dev = ctx.torch_device
    x = torch.empty(0, 64, dtype=torch.float16, device=dev)
    y, st = ctx.layer_norm_train(x)
    dx, dg, db = ctx.layer_norm_backward(x, x, st)
    assert y.shape == (0, 64) and st.shape == (0, 2) and not dg.any() and not db.any()
    c = torch.full((4, 64), 3.0, dtype=torch.float16, device=dev)
    y, st = ctx.layer_norm_train(c, eps=1e-5)
    assert not y.any() and torch.allclose(st[:, 1].cpu(), torch.tensor(1e-5 ** -0.5), rtol=1e-6)
    dx, dg, db = ctx.layer_norm_backward(c, c, st, need_weights=False)
    assert dg is None and db is None and torch.isfinite(dx).all()


def test_a_bad_row_stays_by_itself(backend, request):
    ctx = ctx_of(backend, torch.float16, request)
    dev = ctx.torch_device
    x = rows_of(9, 40, torch.float16, 4).to(dev)
    ref = ctx.layer_norm_train(x)[0]
    x[4, 3] = float("nan")
    y = ctx.layer_norm_train(x)[0]
    keep = [0, 1, 2, 3, 5, 6, 7, 8]
    assert torch.isnan(y[4]).all() and torch.equal(y[keep], ref[keep])


def test_gradient_against_differences(backend, request):
    """the kernel's gradients along random directions against central differences of the formula in 64 bits"""
    ctx = ctx_of(backend, torch.float16, request)
    dev = ctx.torch_device
    g = torch.Generator().manual_seed(0)
    x, dy = torch.randn(6, 48, generator=g).half(), torch.randn(6, 48, generator=g).half()
    gamma, beta = 1 + 0.3 * torch.randn(48, generator=g), torch.randn(48, generator=g)
    _, st = ctx.layer_norm_train(x.to(dev), gamma.to(dev), beta.to(dev))
    dx, dg, db = (t.cpu().double() for t in ctx.layer_norm_backward(dy.to(dev), x.to(dev), st, gamma.to(dev)))

    def loss(x_, g_, b_):
        return float((O.layer_norm_forward(x_, g_, b_, 1e-5)[0] * dy.double()).sum())

    h = 1e-5
    for seed in range(3):
        r = torch.Generator().manual_seed(100 + seed)
        vx, vg, vb = torch.randn(6, 48, generator=r).double(), torch.randn(48, generator=r).double(), torch.randn(48, generator=r).double()
        X, G, B = x.double(), gamma.double(), beta.double()
        for num, ana, bound in (
                ((loss(X + h * vx, G, B) - loss(X - h * vx, G, B)) / (2 * h), float((dx * vx).sum()), float((dx.abs() * vx.abs()).sum()) * 2.0 ** -10),
                ((loss(X, G + h * vg, B) - loss(X, G - h * vg, B)) / (2 * h), float((dg * vg).sum()), 1e-4),
                ((loss(X, G, B + h * vb) - loss(X, G, B - h * vb)) / (2 * h), float((db * vb).sum()), 1e-4)):
            assert abs(num - ana) <= bound + 1e-6, (num, ana, bound)


def test_same_bits_again(backend, request):
    ctx = ctx_of(backend, torch.bfloat16, request)
    dev = ctx.torch_device
    x = rows_of(300, 72, torch.bfloat16, 1).to(dev)
    st = ctx.layer_norm_train(x)[1]
    a, b = ctx.layer_norm_backward(x, x, st), ctx.layer_norm_backward(x, x, st)
    assert all(torch.equal(s, t) for s, t in zip(a, b))


def test_refusals(backend, request):
    ctx = ctx_of(backend, torch.float16, request)
    dev = ctx.torch_device
    x = torch.zeros(4, 64, dtype=torch.float16, device=dev)
    st = ctx.layer_norm_train(x)[1]
    gamma = torch.ones(64, device=dev)
    bad = [
        lambda: ctx.layer_norm_train(x.bfloat16()),
        lambda: ctx.layer_norm_train(x.float()),
        lambda: ctx.layer_norm_train(x[None]),
        lambda: ctx.layer_norm_train(x[0, 0]),
        lambda: ctx.layer_norm_train([1.0]),
        lambda: ctx.layer_norm_train(x.t()),
        lambda: ctx.layer_norm_train(x, gamma.half()),
        lambda: ctx.layer_norm_train(x, gamma[:32]),
        lambda: ctx.layer_norm_train(x, None, gamma.repeat(2)[::2]),
        lambda: ctx.layer_norm_train(x, out=torch.zeros(4, 65, dtype=torch.float16, device=dev)),
        lambda: ctx.layer_norm_train(x[:, :0]),
        lambda: ctx.layer_norm_train(torch.zeros(1, 16385, dtype=torch.float16, device=dev)),
        lambda: ctx.layer_norm_train(x[:1].expand(4, 64)),
        lambda: ctx.layer_norm_backward(x[:3], x, st),
        lambda: ctx.layer_norm_backward(x, x, st[:3]),
        lambda: ctx.layer_norm_backward(x, x, st.half()),
        lambda: ctx.layer_norm_backward(x, x, st, gamma, dx=x[:3]),
    ]
    for i, call in enumerate(bad):
        with pytest.raises(L.StarError):
            call()
            pytest.fail(f"call {i} was not refused")
    rc = ctx.lib.layer_norm_bwd(ctx.h, x.data_ptr(), 64, x.data_ptr(), 64, st.data_ptr(), None, x.data_ptr(), 64, gamma.data_ptr(), None, 4, 64, None, 0)
    assert rc and b"workspace" in ctx.lib.last_error(ctx.h)
    assert ctx.lib.layer_norm_train(ctx.h, None, 64, x.data_ptr(), 64, None, None, None, 4, 64, 1e-5)
    assert ctx.lib.layer_norm_train(None, x.data_ptr(), 64, x.data_ptr(), 64, None, None, None, 4, 64, 1e-5)
    assert ctx.lib.layer_norm_train(ctx.h, x.data_ptr(), 64, x.data_ptr(), 64, None, None, None, -1, 64, 1e-5)


@pytest.mark.parametrize("rows,C", [(1, 8), (3, 50), (5, 320), (3, 1024)])
def test_in_place_where_the_gradient_leaves_the_range(backend, rows, C, request):
    """dx overflows to infinity and is written over x or dy: the weight's gradients, finite numbers, are those of the call with an output of its own"""
    ctx = ctx_of(backend, torch.float16, request)
    dev = ctx.torch_device
    x = torch.randn(rows, C, generator=torch.Generator().manual_seed(1)).half().to(dev)
    dy = (6e4 * torch.sign(torch.randn(rows, C, generator=torch.Generator().manual_seed(2)))).half().to(dev)
    gamma = torch.full((C,), 1e4, device=dev)
    _, st = ctx.layer_norm_train(x, gamma)
    dx, dg, db = ctx.layer_norm_backward(dy, x, st, gamma)
    assert torch.isinf(dx).any(1).all() and torch.isfinite(dg).all() and torch.isfinite(db).all()
    for target in ("x", "dy"):
        xc, dyc = x.clone(), dy.clone()
        got, g2, b2 = ctx.layer_norm_backward(dyc, xc, st, gamma, dx=xc if target == "x" else dyc)
        assert torch.equal(got, dx) and torch.equal(g2, dg) and torch.equal(b2, db), target


def test_in_place_with_another_row_stride_is_refused(backend, request):
    """rows of y would lie over rows of x that are still to be read"""
    ctx = ctx_of(backend, torch.float16, request)
    dev = ctx.torch_device
    buf = torch.randn(16, 64, generator=torch.Generator().manual_seed(1)).half().to(dev)
    keep = buf.clone()
    wide, flat = buf.reshape(8, 128)[:, :64], buf[:8]
    st = ctx.layer_norm_train(wide)[1]
    other = torch.zeros(8, 64, dtype=torch.float16, device=dev)
    for x, y in ((wide, flat), (flat, wide)):
        for call in (lambda: ctx.layer_norm_train(x, out=y), lambda: ctx.layer_norm_backward(other, x, st, dx=y), lambda: ctx.layer_norm_backward(x, other, st, dx=y)):
            with pytest.raises(L.StarError, match="row stride"):
                call()
    assert torch.equal(buf, keep)
    one = ctx.layer_norm_train(wide[:1])[0]                                  # (of one row the stride says nothing)
    assert torch.equal(ctx.layer_norm_train(wide[:1], out=flat[:1])[0], one)
