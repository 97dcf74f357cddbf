"""Position-dependent attention (star_pos_attn_fwd / _bwd) at the ends of its inputs' range: large and small V and dO, large scores and biases,
against the formulas in 64 bits; bounds as in test_pos_attention.py, f16's absolute half steps by rows and key blocks (`tight`)."""
import os
import sys

import pytest
import torch

sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "oracle"))
import train_ops_oracle as O  # noqa: E402
from util import BACKENDS, DTYPES, make_ctx  # noqa: E402


@pytest.fixture(params=BACKENDS)
def backend(request):
    return request.param


def ctx_of(backend, dtype, request):
    return make_ctx(backend, dtype, request.getfixturevalue("emu_lib") if backend == "emu" else None)


def randn(seed, *shape):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed))


def within(got, ref, tol, what):
    got = got.detach().cpu().double()
    assert got.shape == ref.shape and torch.isfinite(got).all(), what
    over = (got - ref).abs() - tol
    assert float(over.max()) <= 0, f"{what}: off by {float(over.max()):.3g} more than its bound, largest value {float(ref.abs().max()):.3g}"


def check_backward(ctx, q, k, v, do, H, KH, *, window=(-1, -1), sinks=0, scale=0.125, bias=None):
    dev = ctx.torch_device
    kw = dict(scale=scale, window=window, sinks=sinks)
    if bias is not None:
        kw["bias"] = (bias[0].to(dev), torch.tensor(bias[1], dtype=torch.int32, device=dev))
    ref = O.pos_attention(q, k, v, H, KH, scale, *window, sinks, bias=bias, dout=do, tight=True)
    a = [t.to(dev) for t in (q, k, v)]
    _, lse = ctx.pos_attention(*a, H, KH, return_lse=True, **kw)
    got = dict(zip(("dq", "dk", "dv", "dtable"), ctx.pos_attention_backward(do.to(dev), *a, lse, H, KH, **kw)))
    for n, t in got.items():
        if t is not None:
            within(t, ref[n], ref["tol_" + n], n)


def bias_of(with_bias, H, seed):
    return (randn(seed, 16, H), O.bucket_scheme(16, 30, True)) if with_bias else None


# ------------------------------------------------------------------------------------------------------ sizes of V and dO
# N, window: a row sees two keys, a row sees a few dozen, and more keys than the span up to which the remainders of P and dS are kept
SPANS = [(40, (1, 0)), (150, (20, 20)), (600, (-1, -1))]
LARGE_V = [("aligned", 200.0, 1e-2), ("aligned", 500.0, 1e-4), ("aligned", 1000.0, 1e-5), ("channel", 8000.0, 1e-2), ("channel", 20000.0, 1e-4)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("with_bias", [False, True])
@pytest.mark.parametrize("N,window", SPANS)
@pytest.mark.parametrize("form,size,grad", LARGE_V)
def test_large_values_with_small_gradients(backend, dtype, N, window, with_bias, form, size, grad, request):
    """V rows of one sign and a common size, or one channel far above the others, with gradients that keep the results finite: dP = dO V^T passes
    f16's range relative to dO by far.  q and k are small beside `scale`, so that dq and dk are numbers of a normal size"""
    q, k = (2.0 ** -4 * randn(n, 1, N, 64) for n in (1, 2))
    do = grad * (1 + 0.3 * randn(3, 1, N, 64))
    if form == "aligned":
        v = size * torch.sign(randn(4, 1, N, 1)).expand(1, N, 64) * (1 + 0.01 * randn(5, 1, N, 64))
    else:
        v = randn(4, 1, N, 64)
        v[:, :, 5] = (size * v[:, :, 5]).clamp(-60000, 60000)
    check_backward(ctx_of(backend, dtype, request), *(t.to(dtype) for t in (q, k, v, do)), 1, 1, window=window, scale=32.0, bias=bias_of(with_bias, 1, 6))


@pytest.mark.parametrize("with_bias", [False, True])
@pytest.mark.parametrize("N,window", SPANS)
@pytest.mark.parametrize("size,grad", [(1.0, 2.0 ** -12), (1.0, 2.0 ** -18), (1e-3, 2.0 ** -10)])
def test_small_gradients_keep_their_digits(backend, N, window, with_bias, size, grad, request):
    """dS below f16's normal range, dq and dk inside it: scale k and scale q are large"""
    q, k = (2.0 ** -10 * randn(n, 1, N, 64) for n in (1, 2))
    v, do = size * randn(4, 1, N, 64), grad * randn(3, 1, N, 64)
    check_backward(ctx_of(backend, torch.float16, request), *(t.half() for t in (q, k, v, do)), 1, 1, window=window, scale=2.0 ** 17, bias=bias_of(with_bias, 1, 7))


@pytest.mark.parametrize("H,KH", [(1, 1), (4, 2)])
@pytest.mark.parametrize("turned", [False, True])
def test_rows_of_different_sizes(backend, H, KH, turned, request):
    """rows whose dO differ by 2^12, far apart along the sequence: each row's dq, and dk of the keys that only small rows see, keep their digits"""
    N = 500
    q, k = 2.0 ** -10 * randn(1, 1, N, H * 64), 2.0 ** -10 * randn(2, 1, N, KH * 64)
    v, do = randn(4, 1, N, KH * 64), 2.0 ** -4 * randn(3, 1, N, H * 64)
    do[:, 250:] *= 2.0 ** -12
    if turned:
        do = do.flip(1)
    check_backward(ctx_of(backend, torch.float16, request), *(t.half() for t in (q, k, v, do)), H, KH, window=(20, 20), scale=2.0 ** 17)


# ----------------------------------------------------------------------------------------------------- large scores and biases
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("Nq", [1, 130])
@pytest.mark.parametrize("score,bias", [(1e6, None), (-1e6, None), (1e9, None), (-1e9, None), (3e5, -2e6), (3e4, 5e5)])
def test_equal_scores_weigh_the_same(backend, dtype, Nq, score, bias, request):
    """every score is the same large number, whatever it rounds to: the output is the mean of V.  P is 1 for each key, its sum exact: rounded are the
    output and, twice at most, its terms' products with 1 (fp32 sums of 700 terms beside that)"""
    ctx = ctx_of(backend, dtype, request)
    dev = ctx.torch_device
    N = 700
    q, k = torch.ones(1, Nq, 64).to(dtype), torch.full((1, N, 64), 0.75).to(dtype)
    v = randn(3, 1, N, 64).to(dtype)
    kw = {}
    if bias is not None:
        kw["bias"] = (torch.full((16, 1), bias, device=dev), ctx.rel_buckets(16, 30))
    out, lse = ctx.pos_attention(q.to(dev), k.to(dev), v.to(dev), 1, scale=score / 48.0, return_lse=True, **kw)
    ref = v.double().mean(1, keepdim=True).expand(1, Nq, 64)
    u = O.half_step(dtype)
    within(out, ref, u * ref.abs() + 710 * O.U32 * v.double().abs().mean(1, keepdim=True) + (2.0 ** -25 if dtype == torch.float16 else 0), "out")
    # the score: 64 products, the scale, the base and back, and log 700 added to it
    total = score + (bias or 0.0)
    within(lse, torch.full((1, 1, Nq), total + 6.551080335).double(), torch.full((1, 1, Nq), 80 * O.U32 * (abs(score) + abs(bias or 0.0))).double(), "lse")


SHIFTS = [1500.0, -5000.0, 1e6, -7e6, 1e9, -1e9, 1e30, -1e30]


def shifted_backward(ctx, q, k, v, do, H, KH, shift, base, **kw):
    """gradients with a bias of `base` plus `shift` in every bucket"""
    dev = ctx.torch_device
    kw["bias"] = ((base[0] + shift).to(dev), torch.tensor(base[1], dtype=torch.int32, device=dev))
    a = [t.to(dev) for t in (q, k, v)]
    out, lse = ctx.pos_attention(*a, H, KH, return_lse=True, **kw)
    return (out, *ctx.pos_attention_backward(do.to(dev), *a, lse, H, KH, **kw))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shift", SHIFTS)
def test_one_visible_key_under_a_large_bias(backend, dtype, shift, request):
    """P is 1 whatever the score: out is V, dV is dO (rounded once; P within 2^-20 of 1), the other gradients are zero"""
    ctx = ctx_of(backend, dtype, request)
    q, k, v, do = (randn(n, 1, 200, 128).to(dtype) for n in range(4))
    out, dq, dk, dv, dt = shifted_backward(ctx, q, k, v, do, 2, 2, shift, (torch.zeros(16, 2), O.bucket_scheme(16, 30, True)), window=(0, 0))
    assert torch.equal(out.cpu(), v) and not dq.any() and not dk.any() and not dt.any()
    within(dv, do.double(), (O.half_step(dtype) + 2.0 ** -20) * do.double().abs() + 2.0 ** -25, "dv")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("window", [(-1, -1), (70, 0)])
@pytest.mark.parametrize("shift", SHIFTS)
def test_many_keys_under_a_large_bias(backend, dtype, window, shift, request):
    """q is zero, so that a score is the bias alone and a shift of all biases changes nothing: out and gradients are those without it"""
    ctx = ctx_of(backend, dtype, request)
    N, H, KH = 300, 2, 1
    q, k, v, do = torch.zeros(1, N, H * 64), randn(1, 1, N, 64), randn(2, 1, N, 64), randn(3, 1, N, H * 64)
    q, k, v, do = (t.to(dtype) for t in (q, k, v, do))
    base = (torch.zeros(16, H), O.bucket_scheme(16, 30, True))
    ref = O.pos_attention(q, k, v, H, KH, 0.125, *window, bias=base, dout=do, tight=True)
    got = shifted_backward(ctx, q, k, v, do, H, KH, shift, base, window=window)
    for n, t in zip(("out", "dq", "dk", "dv", "dtable"), got):
        within(t, ref[n], ref["tol_" + n], n)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shift", [1500.0, -5000.0])
def test_scores_beside_a_large_bias(backend, dtype, shift, request):
    """below and above the size from which scores are rounded one by one (the bounds count the rounding of a score of this size)"""
    N = 300
    q, k, v, do = (randn(n, 1, N, 64).to(dtype) for n in range(4))
    table, buckets = bias_of(True, 1, 9)
    for window in ((-1, -1), (40, 3)):
        check_backward(ctx_of(backend, dtype, request), q, k, v, do, 1, 1, window=window, bias=(table + shift, buckets))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("size", [1e5, 1e9])
def test_one_key_outweighs_the_others(backend, dtype, size, request):
    """scores of a large size, far apart: P is 1 at the largest and 0 elsewhere.  dV sums the dO of the rows that chose a key, dQ and dK are zero"""
    ctx = ctx_of(backend, dtype, request)
    dev = ctx.torch_device
    N = 150
    q, k, v, do = (randn(10 + n, 1, N, 64).to(dtype) for n in range(4))
    s = size / 8 * (q[0].double() @ k[0].double().T)
    top = s.topk(2, 1).values
    best = torch.nn.functional.one_hot(s.argmax(1), N).double()
    # rows whose first two scores are as near as roundings of 64 products are left out of what is compared: they see one key only
    near = (top[:, 0] - top[:, 1] <= 200 * O.U32 * size / 8 * (q[0].double().abs() @ k[0].double().abs().T).amax(1) + 50)
    assert int(near.sum()) <= 2
    do[:, near] = 0
    a = [t.to(dev) for t in (q, k, v)]
    out, lse = ctx.pos_attention(*a, 1, scale=size / 8, return_lse=True)
    dq, dk, dv, _ = ctx.pos_attention_backward(do.to(dev), *a, lse, 1, scale=size / 8)
    assert torch.equal(out.cpu()[0, ~near], v[0, s.argmax(1)[~near]])
    assert not dq.any() and not dk.any()
    g = do[0].double()
    within(dv[0], best.T @ g, O.half_step(dtype) * (best.T @ g).abs() + (N * O.U32 + 2.0 ** -20) * (best.T @ g.abs()) + 2.0 ** -25, "dv")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("score", [1e6, -1e9])
def test_gradient_of_equal_large_scores(backend, dtype, score, request):
    """q and k the same everywhere: each key weighs 1 / N, dV is the mean of dO; dS sums to zero along a row, its parts are (dP - mean dP) / N"""
    ctx = ctx_of(backend, dtype, request)
    dev = ctx.torch_device
    N = 200
    q, k = torch.ones(1, N, 64).to(dtype), torch.full((1, N, 64), 0.75).to(dtype)
    v, do = randn(1, 1, N, 64).to(dtype), randn(2, 1, N, 64).to(dtype)
    a = [t.to(dev) for t in (q, k, v)]
    bias = (torch.zeros(16, 1, device=dev), ctx.rel_buckets(16, 30))
    _, lse = ctx.pos_attention(*a, 1, scale=score / 48, bias=bias, return_lse=True)
    _, _, dv, dt = ctx.pos_attention_backward(do.to(dev), *a, lse, 1, scale=score / 48, bias=bias)
    zero = torch.zeros(1, N, 64).to(dtype)
    ref = O.pos_attention(zero, k, v, 1, 1, 0.125, bias=(torch.zeros(16, 1), O.bucket_scheme(16, 30, True)), dout=do, tight=True)
    within(dv, ref["dv"], ref["tol_dv"], "dv")
    within(dt, ref["dtable"], ref["tol_dtable"], "dtable")


MOST = torch.finfo(torch.float32).max


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("Nq", [1, 200])
@pytest.mark.parametrize("shift", [-MOST, MOST, -2.5e38])
def test_every_bias_at_the_end_of_the_range(backend, dtype, Nq, shift, request):
    """all keys weigh the same, their scores lost beside the bias; with q = 0 the gradients are those without a bias"""
    ctx = ctx_of(backend, dtype, request)
    q, k, v, do = torch.zeros(1, Nq, 64), randn(1, 1, 200, 64), randn(2, 1, 200, 64), randn(3, 1, Nq, 64)
    q, k, v, do = (t.to(dtype) for t in (q, k, v, do))
    base = (torch.zeros(16, 1), O.bucket_scheme(16, 30, True))
    ref = O.pos_attention(q, k, v, 1, 1, 0.125, bias=base, dout=do, tight=True)
    got = shifted_backward(ctx, q, k, v, do, 1, 1, shift, base)
    for n, t in zip(("out", "dq", "dk", "dv", "dtable"), got):
        within(t, ref[n], ref["tol_" + n], n)
    dev = ctx.torch_device
    bias = (torch.full((16, 1), shift, device=dev), torch.tensor(base[1], dtype=torch.int32, device=dev))
    out, lse = ctx.pos_attention(randn(4, 1, Nq, 64).to(dtype).to(dev), k.to(dev), v.to(dev), 1, bias=bias, return_lse=True)
    within(out, ref["out"], ref["tol_out"], "out")
    if abs(shift) == MOST:
        assert bool((lse == shift).all())


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("which", ["lowest", "highest", "both"])
def test_some_biases_at_the_end_of_the_range(backend, dtype, which, request):
    """buckets at the lowest value hide their keys from rows that see others, as -inf does; buckets at the highest hide all others"""
    ctx = ctx_of(backend, dtype, request)
    dev = ctx.torch_device
    N = 150
    q, k, v, do = (randn(20 + n, 1, N, 64).to(dtype) for n in range(4))
    q = q * (which == "lowest")                               # (a highest bias loses the scores beside it)
    table, buckets = bias_of(True, 1, 9)
    hidden = table.clone()
    if which != "highest":
        table[3], hidden[3] = -MOST, -float("inf")
    if which != "lowest":
        table[0], hidden = MOST, torch.full_like(hidden, -float("inf"))
        hidden[0] = 0.0
    want = O.pos_attention(q, k, v, 1, 1, 0.125, bias=(hidden, buckets), dout=do, tight=True)
    assert torch.isfinite(want["lse"]).all()
    kw = dict(bias=(table.to(dev), torch.tensor(buckets, dtype=torch.int32, device=dev)))
    a = [t.to(dev) for t in (q, k, v)]
    out, lse = ctx.pos_attention(*a, 1, return_lse=True, **kw)
    got = ctx.pos_attention_backward(do.to(dev), *a, lse, 1, **kw)
    for n, t in zip(("out", "dq", "dk", "dv", "dtable"), (out, *got)):
        within(t, want[n], want["tol_" + n], n)
    if which != "lowest":
        assert bool((lse == MOST).all())


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("with_bias", [False, True])
@pytest.mark.parametrize("H,KH", [(1, 1), (4, 2)])
def test_large_scores_in_some_rows_only(backend, dtype, H, KH, with_bias, request):
    """waves with large scores beside waves without, in one workgroup, and rows of both kinds in one tile of the dK / dV pass (the bounds of the other
    rows' gradients stay narrow)"""
    N = 330
    q = randn(1, 1, N, H * 64)
    for a, b in ((32, 40), (100, 101), (160, 192), (300, 330)):
        q[:, a:b] *= 4000
    k, v, do = randn(2, 1, N, KH * 64), randn(3, 1, N, KH * 64), 0.1 * randn(4, 1, N, H * 64)
    q, k, v, do = (t.to(dtype) for t in (q, k, v, do))
    for window, sinks in (((-1, -1), 0), ((60, 0), 5)):
        check_backward(ctx_of(backend, dtype, request), q, k, v, do, H, KH, window=window, sinks=sinks, bias=bias_of(with_bias, H, 9))
