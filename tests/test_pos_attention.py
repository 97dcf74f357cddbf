"""Position-dependent attention (star_pos_attn_fwd / _bwd, pattn.h, pattn_bwd.h): window, first tokens, lengths, caches, grouped heads and the
learned bias by buckets, forward, backward and one token at a time, against the formulas in 64 bits with the elementwise bounds that
oracle/train_ops_oracle.py derives (one half step for each rounding to 16 bits, fp32 sums)."""
import ctypes
import os
import sys

import pytest
import torch

sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "oracle"))
import train_ops_oracle as O  # noqa: E402
from util import BACKENDS, DTYPES, make_ctx  # noqa: E402

from star_amd import lib as L  # noqa: E402


@pytest.fixture(params=BACKENDS)
def backend(request):
    return request.param


def ctx_of(backend, dtype, request):
    return make_ctx(backend, dtype, request.getfixturevalue("emu_lib") if backend == "emu" else None)


def inputs(dtype, B, Nq, Nk, H, KH, seed, shared=False, buckets=0, distance=0, both=True, peaked=1.0):
    g = torch.Generator().manual_seed(seed)
    S = 1 if shared else B
    q = (peaked * torch.randn(B, Nq, H * 64, generator=g)).to(dtype)
    k, v = (torch.randn(S, Nk, KH * 64, generator=g).to(dtype) for _ in range(2))
    do = (0.2 * torch.randn(B, Nq, H * 64, generator=g)).to(dtype)
    bias = (torch.randn(buckets, H, generator=g), O.bucket_scheme(buckets, distance, both)) if buckets else None
    return q, k, v, do, bias


def within(got, ref, tol, what):
    got = got.detach().cpu().double()
    assert got.shape == ref.shape, (what, got.shape, ref.shape)
    fin = torch.isfinite(ref)
    assert torch.equal(torch.isfinite(got), fin), f"{what}: other values are finite"
    assert torch.equal(got[~fin], ref[~fin]), what
    over = ((got - ref).abs() - tol)[fin]
    assert not over.numel() or float(over.max()) <= 0, f"{what}: off by {float(over.max()):.3g} more than its bound, worst ratio {float(((got - ref).abs() / tol)[fin].max()):.3g}"


def run_case(ctx, q, k, v, do, H, KH, *, scale=0.125, window=None, sinks=0, causal=False, q_start=None, kv_len=None, bias=None, backward=True):
    dev = ctx.torch_device
    kw = dict(scale=scale, window=window, sinks=sinks, causal=causal)
    for n, t in (("q_start", q_start), ("kv_len", kv_len)):
        kw[n] = torch.tensor(t, dtype=torch.int32, device=dev) if t is not None else None
    if bias is not None:
        kw["bias"] = (bias[0].to(dev), torch.tensor(bias[1], dtype=torch.int32, device=dev))
    left, right = (-1, -1) if window is None else window
    if causal:
        right = 0
    ref = O.pos_attention(q, k, v, H, KH, scale, left, right, sinks, q_start, kv_len, bias, do if backward else None)
    qd, kd, vd = (t.to(dev) for t in (q, k, v))
    out, lse = ctx.pos_attention(qd, kd, vd, H, KH, return_lse=True, **kw)
    within(lse, ref["lse"], ref["tol_lse"], "lse")
    within(out, ref["out"], ref["tol_out"], "out")
    assert torch.equal(ctx.pos_attention(qd, kd, vd, H, KH, **kw), out)
    if backward:
        got = ctx.pos_attention_backward(do.to(dev), qd, kd, vd, lse, H, KH, **kw)
        for n, t in zip(("dv", "dk", "dq", "dtable"), (got[2], got[1], got[0], got[3])):
            if n != "dtable" or bias is not None:
                within(t, ref[n], ref["tol_" + n], n)
        if bias is None:
            assert got[3] is None
    return out, lse


# B, Nq, Nk, H, KH, arguments
WINDOWS = [
    (1, 1, 1, 1, 1, {}),
    (2, 77, 77, 2, 2, {"causal": True}),
    (1, 65, 65, 1, 1, {"window": (0, 0)}),
    (1, 130, 130, 2, 1, {"window": (5, 0), "sinks": 3}),
    (1, 200, 200, 1, 1, {"window": (40, 40), "sinks": 70}),
    (2, 150, 150, 2, 1, {"window": (16, 0), "sinks": 1, "kv_len": [150, 33]}),
    (2, 40, 300, 3, 1, {"window": (100, 0), "sinks": 4, "q_start": [200, 3], "kv_len": [240, 43]}),
    (1, 33, 20, 2, 2, {"causal": True}),
    (2, 64, 128, 2, 2, {"window": (-1, -1), "kv_len": [0, 128]}),
    (1, 20, 90, 4, 2, {"window": (10, 0), "q_start": [500]}),
    (1, 20, 90, 4, 2, {"window": (10, 3), "q_start": [-15]}),
    (3, 5, 70, 5, 1, {"window": (1000, 1000), "sinks": 10}),
    (1, 300, 300, 1, 1, {}),
]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("case", range(len(WINDOWS)))
def test_window_and_first_tokens(backend, dtype, case, request):
    B, Nq, Nk, H, KH, kw = WINDOWS[case]
    q, k, v, do, _ = inputs(dtype, B, Nq, Nk, H, KH, case, peaked=2.0 if case % 2 else 1.0)
    run_case(ctx_of(backend, dtype, request), q, k, v, do, H, KH, **kw)


BIASED = [
    (1, 1, 1, 1, 1, 8, 8, True, {}),
    (2, 77, 77, 2, 2, 32, 128, True, {"kv_len": [77, 20], "q_start": [0, 0]}),
    (1, 200, 200, 2, 1, 32, 40, True, {"scale": 1.0}),
    (1, 150, 150, 1, 1, 16, 20, False, {"causal": True}),
    (2, 100, 260, 2, 1, 32, 128, False, {"causal": True, "q_start": [100, 7], "kv_len": [200, 107]}),
    (1, 130, 130, 1, 1, 2, 1, True, {}),
    (1, 70, 300, 2, 2, 32, 16, True, {"window": (60, 10), "sinks": 5}),
]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("case", range(len(BIASED)))
def test_relative_position_bias(backend, dtype, case, request):
    B, Nq, Nk, H, KH, nb, dist, both, kw = BIASED[case]
    q, k, v, do, bias = inputs(dtype, B, Nq, Nk, H, KH, 50 + case, buckets=nb, distance=dist, both=both, peaked=0.5 if "scale" in kw else 1.0)
    run_case(ctx_of(backend, dtype, request), q, k, v, do, H, KH, bias=bias, **kw)


def test_bias_of_one_bucket_range_zero(backend, request):
    """a table of one entry for all positions changes nothing, and its gradient is zero up to the sums' roundings"""
    ctx = ctx_of(backend, torch.float16, request)
    q, k, v, do, _ = inputs(torch.float16, 1, 90, 90, 1, 1, 9)
    run_case(ctx, q, k, v, do, 1, 1, bias=(torch.tensor([[0.7]]), [0]))


@pytest.mark.parametrize("Nq,Nk,start", [(140, 1300, 1100), (200, 200, 0), (1, 2500, 2400)])
def test_the_largest_bias(backend, Nq, Nk, start, request):
    """the longest reach and the most buckets; a kernel's table then takes the greater part of the shared memory"""
    g = torch.Generator().manual_seed(Nk)
    q, k, v, do, _ = inputs(torch.float16, 1, Nq, Nk, 1, 1, 31)
    bias = (torch.randn(4096, 1, generator=g), torch.randint(0, 4096, (2049,), generator=g).tolist())
    run_case(ctx_of(backend, torch.float16, request), q, k, v, do, 1, 1, q_start=[start], bias=bias)


STEPS = [
    (3, 1, 700, 4, 1, {"kv_len": [700, 65, 1], "causal": True}),
    (2, 1, 1500, 2, 2, {"kv_len": [1500, 900], "window": (300, 0), "sinks": 4}),
    (1, 3, 1100, 8, 2, {"kv_len": [1000], "window": (600, 0), "sinks": 64}),
    (2, 1, 64, 40, 1, {"kv_len": [64, 0], "causal": True}),
    (1, 7, 600, 4, 1, {"kv_len": [600], "causal": True}),
    (1, 8, 600, 4, 1, {"kv_len": [577], "causal": True}),
]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("with_bias", [False, True])
@pytest.mark.parametrize("case", range(len(STEPS)))
def test_a_few_tokens_against_a_cache(backend, dtype, case, with_bias, request):
    """the split form: keys dealt to several workgroups and joined; what lies behind kv_len is not a number and must not be read"""
    B, Nq, Nk, H, KH, kw = STEPS[case]
    kw = dict(kw)
    q, k, v, do, bias = inputs(dtype, B, Nq, Nk, H, KH, 80 + case, buckets=32 if with_bias else 0, distance=128, both=False)
    for b, n in enumerate(kw["kv_len"]):
        k[b, n:] = float("nan")
        v[b, n:] = float("inf")
    kw["q_start"] = [n - Nq for n in kw["kv_len"]]
    run_case(ctx_of(backend, dtype, request), q, k, v, do, H, KH, bias=bias, **kw)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("B,Nq,Nk,H,KH,buckets,kw", [
    (2, 1111, 1111, 8, 2, 0, {"window": (300, 0), "sinks": 77, "kv_len": [1111, 640]}),
    (1, 700, 2500, 6, 2, 0, {"window": (900, 0), "sinks": 226, "q_start": [1800]}),
    (40, 513, 513, 16, 16, 32, {}),
    (1, 2049, 2049, 3, 3, 32, {"causal": True}),
    (1, 3000, 3000, 2, 2, 0, {"window": (1350, 1350), "sinks": 226}),
], ids=["ragged", "chunk", "many", "causal", "video"])
def test_larger(dtype, B, Nq, Nk, H, KH, buckets, kw):
    if B * H > 100 and dtype == torch.bfloat16:
        B = 34
    q, k, v, do, bias = inputs(dtype, B, Nq, Nk, H, KH, 7, buckets=buckets, distance=128)
    run_case(L.Context(0, dtype), q, k, v, do, H, KH, bias=bias, **kw)


@pytest.mark.gpu
def test_cache_past_32_bits():
    """a cache of more than 2^32 bytes: the last keys are the ones that count"""
    ctx = L.Context(0, torch.float16)
    Nk = (1 << 32) // (2 * 1024) + 300
    k = torch.zeros(1, Nk, 1024, dtype=torch.float16, device="cuda")[:, :, 960:]
    v = torch.zeros(1, Nk, 1024, dtype=torch.float16, device="cuda")[:, :, :64]
    g = torch.Generator().manual_seed(3)
    tail = 500
    k[:, -tail:] = torch.randn(1, tail, 64, generator=g).half().cuda()
    v[:, -tail:] = torch.randn(1, tail, 64, generator=g).half().cuda()
    for Nq in (1, 40):
        q = torch.randn(1, Nq, 64, generator=g).half()
        do = torch.randn(1, Nq, 64, generator=g).half()
        ref = O.pos_attention(q, k[:, -tail:].cpu(), v[:, -tail:].cpu(), 1, 1, 0.125, 200, 0, 0, None, None, None, do)
        out, lse = ctx.pos_attention(q.cuda(), k, v, 1, window=(200, 0), return_lse=True)
        within(out, ref["out"], ref["tol_out"], "out")
        dq, dk, dv, _ = ctx.pos_attention_backward(do.cuda(), q.cuda(), k, v, lse, 1, window=(200, 0))
        within(dq, ref["dq"], ref["tol_dq"], "dq")
        within(dk[:, -tail:], ref["dk"], ref["tol_dk"], "dk")
        assert not dk[:, :-tail].any() and not dv[:, :-tail].any()


@pytest.mark.parametrize("with_bias", [False, True])
def test_keys_shared_by_the_batch(backend, with_bias, request):
    """one K and V for all sequences: their gradients are sums over the batch and over the heads of a group"""
    ctx = ctx_of(backend, torch.bfloat16, request)
    q, k, v, do, bias = inputs(torch.bfloat16, 3, 50, 90, 4, 2, 21, shared=True, buckets=8 if with_bias else 0, distance=30)
    run_case(ctx, q, k, v, do, 4, 2, bias=bias, window=(30, 20), kv_len=[90, 50, 7], q_start=[40, 0, 0])


def test_one_visible_key_has_no_gradient(backend, request):
    """softmax over one key is 1 whatever the score: dQ and dK are exactly zero, dV is dO"""
    for dtype in (torch.float16, torch.bfloat16):
        ctx = ctx_of(backend, dtype, request)
        dev = ctx.torch_device
        q, k, v, do, bias = inputs(dtype, 1, 100, 100, 2, 2, 4, buckets=8, distance=30, peaked=3.0)
        for b in (None, (bias[0].to(dev), torch.tensor(bias[1], dtype=torch.int32, device=dev))):
            a = [t.to(dev) for t in (q, k, v)]
            out, lse = ctx.pos_attention(*a, 2, window=(0, 0), bias=b, return_lse=True)
            assert torch.equal(out.cpu(), v)
            dq, dk, dv, dt = ctx.pos_attention_backward(do.to(dev), *a, lse, 2, window=(0, 0), bias=b)
            assert not dq.any() and not dk.any() and (dt is None or not dt.any())
            assert (dv.cpu().double() - do.double()).abs().le(O.half_step(dtype) * do.double().abs() + 1e-9).all()


def test_rows_that_see_nothing(backend, request):
    """zeros and -inf, and no gradient; other rows as if those were not there"""
    ctx = ctx_of(backend, torch.float16, request)
    q, k, v, do, _ = inputs(torch.float16, 2, 70, 70, 1, 1, 5)
    out, lse = run_case(ctx, q, k, v, do, 1, 1, window=(3, 0), kv_len=[0, 20])
    assert not out[0].any() and torch.isinf(lse[0]).all() and torch.isinf(lse[1, 0, 23:]).all() and torch.isfinite(lse[1, 0, :23]).all()
    assert not out[1, 23:].any()


def test_bias_of_lowest_and_infinite_values(backend, request):
    """a bucket at -inf hides its keys; the type's lowest value stays a number: a row that sees only such keys averages them"""
    ctx = ctx_of(backend, torch.float16, request)
    dev = ctx.torch_device
    q, k, v, do, _ = inputs(torch.float16, 1, 40, 40, 1, 1, 6)
    bk = torch.tensor([1, 1, 0, 2, 2], dtype=torch.int32, device=dev)       # before, at, after the query
    table = torch.tensor([[0.0], [0.5], [-float("inf")]], device=dev)
    out = ctx.pos_attention(q.to(dev), k.to(dev), v.to(dev), 1, bias=(table, bk))
    ref = ctx.pos_attention(q.to(dev), k.to(dev), v.to(dev), 1, causal=True, bias=(table, bk))
    assert torch.isfinite(out).all() and (out - ref).abs().max() <= 2e-3
    low = torch.full((3, 1), torch.finfo(torch.float32).min, device=dev)
    out = ctx.pos_attention(q.to(dev), k.to(dev), v.to(dev), 1, bias=(low, bk))
    assert (out.cpu().double() - v.double().mean(1, keepdim=True)).abs().max() <= 2.0 ** -9
    none = torch.full((3, 1), -float("inf"), device=dev)
    out, lse = ctx.pos_attention(q.to(dev), k.to(dev), v.to(dev), 1, bias=(none, bk), return_lse=True)
    assert not out.any() and torch.isinf(lse).all()
    dq, dk, dv, dt = ctx.pos_attention_backward(do.to(dev), q.to(dev), k.to(dev), v.to(dev), lse, 1, bias=(none, bk))
    assert not dq.any() and not dk.any() and not dv.any() and not dt.any()


def test_large_scores_move_the_maximum(backend, request):
    """scores that grow along the keys, by far more than the lazy maximum allows, and a maximum that comes early"""
    for dtype in (torch.float16, torch.bfloat16):
        ctx = ctx_of(backend, dtype, request)
        q, k, v, do, _ = inputs(dtype, 1, 70, 400, 1, 1, 8)
        ramp = torch.linspace(-8, 8, 400)[None, :, None]
        for r in (ramp, -ramp):
            k2 = (k.float() * 0.1 + r * torch.sign(q[:, :1].float())).to(dtype)
            run_case(ctx, q, k2, v, do, 1, 1)


def test_small_and_large_gradients(backend, request):
    """f16: rows whose dO differ by a factor of 2^14 keep their digits (dS is scaled before it is rounded)"""
    ctx = ctx_of(backend, torch.float16, request)
    q, k, v, do, _ = inputs(torch.float16, 1, 150, 150, 1, 1, 12)
    do[:, :64] *= 2.0 ** -9
    do[:, 100:] *= 32
    run_case(ctx, q, k, v, do, 1, 1, window=(20, 20))


def test_fused_projection_views_and_given_outputs(backend, request):
    """q, k, v as slices of one buffer, heads-first storage, and outputs inside wider buffers whose other columns stay as they were"""
    ctx = ctx_of(backend, torch.float16, request)
    dev = ctx.torch_device
    q, k, v, do, _ = inputs(torch.float16, 2, 70, 70, 4, 2, 31)
    fused = torch.cat([q, k, v], 2).to(dev)
    qf, kf, vf = fused[:, :, :256], fused[:, :, 256:384], fused[:, :, 384:]
    ref, rl = ctx.pos_attention(q.to(dev), k.to(dev), v.to(dev), 4, 2, causal=True, return_lse=True)
    wide = torch.full((2, 70, 512), 5.0, dtype=torch.float16, device=dev)
    out, lse = ctx.pos_attention(qf, kf, vf, 4, 2, causal=True, return_lse=True, out=wide[:, :, 128:384])
    assert torch.equal(out, ref) and torch.equal(lse, rl) and bool((wide[:, :, :128] == 5).all()) and bool((wide[:, :, 384:] == 5).all())
    qs = q.to(dev).transpose(0, 1).contiguous().transpose(0, 1)              # token-major storage: the batch stride is the small one
    assert torch.equal(ctx.pos_attention(qs, kf, vf, 4, 2, causal=True), ref)
    g = ctx.pos_attention_backward(do.to(dev), q.to(dev), k.to(dev), v.to(dev), rl, 4, 2, causal=True)
    gf = torch.full_like(fused, 9.0)
    h = ctx.pos_attention_backward(do.to(dev), qf, kf, vf, rl, 4, 2, causal=True, dq=gf[:, :, :256], dk=gf[:, :, 256:384], dv=gf[:, :, 384:])
    assert torch.equal(torch.cat(g[:3], 2), gf) and h[0].data_ptr() == gf.data_ptr()


def test_same_bits_again(backend, request):
    ctx = ctx_of(backend, torch.float16, request)
    dev = ctx.torch_device
    q, k, v, do, bias = inputs(torch.float16, 1, 180, 180, 2, 1, 2, buckets=32, distance=50)
    b = (bias[0].to(dev), torch.tensor(bias[1], dtype=torch.int32, device=dev))
    a = [t.to(dev) for t in (q, k, v)]
    out, lse = ctx.pos_attention(*a, 2, 1, bias=b, return_lse=True)
    one = ctx.pos_attention_backward(do.to(dev), *a, lse, 2, 1, bias=b)
    two = ctx.pos_attention_backward(do.to(dev), *a, lse, 2, 1, bias=b)
    assert all(torch.equal(s, t) for s, t in zip(one, two))


def test_gradient_against_differences(backend, request):
    ctx = ctx_of(backend, torch.float16, request)
    dev = ctx.torch_device
    q, k, v, do, bias = inputs(torch.float16, 1, 24, 24, 2, 1, 77, buckets=8, distance=10)
    b = (bias[0].to(dev), torch.tensor(bias[1], dtype=torch.int32, device=dev))
    a = [t.to(dev) for t in (q, k, v)]
    kw = dict(window=(9, 4), sinks=2)
    _, lse = ctx.pos_attention(*a, 2, 1, bias=b, return_lse=True, **kw)
    grads = [t.cpu().double() for t in ctx.pos_attention_backward(do.to(dev), *a, lse, 2, 1, bias=b, **kw)]
    args = [q.double(), k.double(), v.double(), bias[0].double()]

    def loss(qx, kx, vx, tx):
        return float((O.pos_attention(qx, kx, vx, 2, 1, 0.125, 9, 4, 2, bias=(tx, bias[1]))["out"] * do.double()).sum())

    h = 1e-5
    for i in range(4):
        d = torch.randn(args[i].shape, generator=torch.Generator().manual_seed(i)).double()
        up, down = list(args), list(args)
        up[i], down[i] = args[i] + h * d, args[i] - h * d
        num = (loss(*up) - loss(*down)) / (2 * h)
        # every 16-bit gradient is off by at most two roundings of values of its own size
        bound = 4 * 2.0 ** -11 * float((grads[i].abs() * d.abs()).sum()) + 1e-5
        assert abs(num - float((grads[i] * d).sum())) <= bound, (i, num, float((grads[i] * d).sum()), bound)


@pytest.mark.parametrize("nb,dist,both", [(32, 128, True), (32, 128, False), (8, 64, True), (64, 500, False), (2, 1, True), (1, 5, False), (16, 1024, True), (20, 100, True)])
def test_bucket_scheme(nb, dist, both, emu_lib):
    """borders in whole numbers: those of powers of two among them, where a logarithm is off by its last bit"""
    ctx = L.Context(0, torch.float16, emu_lib)
    got = ctx.rel_buckets(nb, dist, bidirectional=both).tolist()
    assert got == O.bucket_scheme(nb, dist, both)
    assert len(got) == 2 * dist + 1 and min(got) >= 0 and max(got) < nb
    if (nb, dist, both) == (32, 128, True):      # 8 exact, then ratios of 2^(1/2): 16, 32, 64 are borders
        far = got[dist + 1:]
        assert [far[d - 1] - 16 for d in (7, 8, 15, 16, 31, 32, 63, 64, 127, 128)] == [7, 8, 9, 10, 11, 12, 13, 14, 15, 15]


def test_bucket_scheme_refusals(emu_lib):
    ctx = L.Context(0, torch.float16, emu_lib)
    for nb, dist, both in ((0, 10, False), (3, 10, True), (32, 0, True), (32, 8, True), (32, 16, False), (257, 1000, False), (32, 1025, True), (32, -4, True)):
        with pytest.raises(L.StarError):
            ctx.rel_buckets(nb, dist, bidirectional=both)


def test_buckets_outside_the_table_are_clamped(backend, request):
    ctx = ctx_of(backend, torch.float16, request)
    dev = ctx.torch_device
    q, k, v, do, _ = inputs(torch.float16, 1, 70, 70, 1, 1, 3)
    a = [t.to(dev) for t in (q, k, v)]
    t = torch.randn(4, 1, generator=torch.Generator().manual_seed(1)).to(dev)
    wild = torch.tensor([-(2 ** 31), -1, 0, 9, 2 ** 31 - 1], dtype=torch.int32, device=dev)
    tame = torch.tensor([0, 0, 0, 3, 3], dtype=torch.int32, device=dev)
    (o1, l1), (o2, l2) = (ctx.pos_attention(*a, 1, bias=(t, b), return_lse=True) for b in (wild, tame))
    assert torch.equal(o1, o2)
    for s, r in zip(*(ctx.pos_attention_backward(do.to(dev), *a, l1, 1, bias=(t, b)) for b in (wild, tame))):
        assert torch.equal(s, r)


def test_lengths_and_positions_out_of_range_are_clamped(backend, request):
    ctx = ctx_of(backend, torch.float16, request)
    dev = ctx.torch_device
    q, k, v, do, _ = inputs(torch.float16, 2, 33, 70, 1, 1, 3)
    a = [t.to(dev) for t in (q, k, v)]
    i32 = lambda *x: torch.tensor(x, dtype=torch.int32, device=dev)  # noqa: E731
    o1 = ctx.pos_attention(*a, 1, window=(5, 5), kv_len=i32(2 ** 31 - 1, -7), q_start=i32(30, 30))
    o2 = ctx.pos_attention(*a, 1, window=(5, 5), kv_len=i32(70, 0), q_start=i32(30, 30))
    assert torch.equal(o1, o2)
    for s in (2 ** 31 - 1, -(2 ** 31)):
        out, lse = ctx.pos_attention(*a, 1, window=(5, 5), q_start=i32(s, s), return_lse=True)
        assert not out.any() and torch.isinf(lse).all()
        grads = ctx.pos_attention_backward(do.to(dev), *a, lse, 1, window=(5, 5), q_start=i32(s, s))
        assert not any(g.any() for g in grads[:3])


def test_empty_dimensions(backend, request):
    ctx = ctx_of(backend, torch.float16, request)
    dev = ctx.torch_device
    z = lambda *s: torch.zeros(*s, dtype=torch.float16, device=dev)  # noqa: E731
    bias = (torch.ones(2, 2, device=dev), torch.tensor([0, 1, 1], dtype=torch.int32, device=dev))
    out, lse = ctx.pos_attention(z(2, 0, 128), z(2, 5, 128), z(2, 5, 128), 2, return_lse=True)
    assert out.shape == (2, 0, 128) and lse.shape == (2, 2, 0)
    g = ctx.pos_attention_backward(z(2, 0, 128), z(2, 0, 128), z(2, 5, 128), z(2, 5, 128), lse, 2, bias=bias)
    assert not g[1].any() and not g[2].any() and not g[3].any()
    out, lse = ctx.pos_attention(z(2, 3, 128) + 1, z(2, 0, 128), z(2, 0, 128), 2, return_lse=True)
    assert not out.any() and torch.isinf(lse).all()
    g = ctx.pos_attention_backward(z(2, 3, 128) + 1, z(2, 3, 128), z(2, 0, 128), z(2, 0, 128), lse, 2, bias=bias)
    assert not g[0].any() and not g[3].any()
    out = ctx.pos_attention(z(0, 3, 128), z(0, 4, 128), z(0, 4, 128), 2)
    assert out.shape == (0, 3, 128)


def test_refusals(backend, request):
    ctx = ctx_of(backend, torch.float16, request)
    dev = ctx.torch_device
    z = lambda *s, dt=torch.float16: torch.zeros(*s, dtype=dt, device=dev)  # noqa: E731
    i32 = torch.int32
    q, k, v = z(2, 8, 256), z(2, 9, 128), z(2, 9, 128)
    ok = ctx.pos_attention(q, k, v, 4, 2, return_lse=True)
    lse = ok[1]
    bad = [
        lambda: ctx.pos_attention(q.bfloat16(), k, v, 4, 2),
        lambda: ctx.pos_attention(q, k.float(), v, 4, 2),
        lambda: ctx.pos_attention(q, k, v, 4, 3),
        lambda: ctx.pos_attention(q, k, v, 4, 0),
        lambda: ctx.pos_attention(q, k, v, 0, 0),
        lambda: ctx.pos_attention(q, k, v, 4),
        lambda: ctx.pos_attention(q[0], k, v, 4, 2),
        lambda: ctx.pos_attention(q, k, v[:, :8], 4, 2),
        lambda: ctx.pos_attention(q, z(3, 9, 128), z(3, 9, 128), 4, 2),
        lambda: ctx.pos_attention(q, k[:1], v, 4, 2),
        lambda: ctx.pos_attention(q.transpose(1, 2).contiguous().transpose(1, 2), k, v, 4, 2),
        lambda: ctx.pos_attention(z(2, 8, 260)[:, :, 4:], k, v, 4, 2),
        lambda: ctx.pos_attention(z(2, 8, 257)[:, :, :256], k, v, 4, 2),
        lambda: ctx.pos_attention(q, k, v, 4, 2, kv_len=z(2, dt=torch.int64)),
        lambda: ctx.pos_attention(q, k, v, 4, 2, kv_len=z(3, dt=i32)),
        lambda: ctx.pos_attention(q, k, v, 4, 2, q_start=z(1, dt=i32)),
        lambda: ctx.pos_attention(q, k, v, 4, 2, sinks=-1),
        lambda: ctx.pos_attention(q, k, v, 4, 2, scale=float("nan")),
        lambda: ctx.pos_attention(q, k, v, 4, 2, scale=float("inf")),
        lambda: ctx.pos_attention(q, k, v, 4, 2, bias=(z(8, 2, dt=torch.float32), z(3, dt=i32))),
        lambda: ctx.pos_attention(q, k, v, 4, 2, bias=(z(8, 4), z(3, dt=i32))),
        lambda: ctx.pos_attention(q, k, v, 4, 2, bias=(z(0, 4, dt=torch.float32), z(3, dt=i32))),
        lambda: ctx.pos_attention(q, k, v, 4, 2, bias=(z(4097, 4, dt=torch.float32), z(3, dt=i32))),
        lambda: ctx.pos_attention(q, k, v, 4, 2, bias=(z(8, 4, dt=torch.float32), z(4, dt=i32))),
        lambda: ctx.pos_attention(q, k, v, 4, 2, bias=(z(8, 4, dt=torch.float32), z(2051, dt=i32))),
        lambda: ctx.pos_attention(q, k, v, 4, 2, out=z(2, 8, 128)),
        lambda: ctx.pos_attention(q, k, v, 4, 2, out=z(1, 8, 256).expand(2, 8, 256)),
        lambda: ctx.pos_attention_backward(q[:, :7], q, k, v, lse, 4, 2),
        lambda: ctx.pos_attention_backward(q, q, k, v, lse[:, :2], 4, 2),
        lambda: ctx.pos_attention_backward(q, q, k, v, lse.half(), 4, 2),
        lambda: ctx.pos_attention_backward(q, q, k, v, lse, 4, 2, dk=z(1, 9, 128)),
        lambda: ctx.pos_attention_backward(q, q, k, v, lse, 4, 2, dk=z(1, 9, 128).expand(2, 9, 128)),
        lambda: ctx.pos_attention_backward(q, q, k[:1].expand(2, 9, 128), v[:1].expand(2, 9, 128), lse, 4, 2),
    ]
    for i, call in enumerate(bad):
        with pytest.raises(L.StarError):
            call()
            pytest.fail(f"call {i} was not refused")
    assert torch.equal(ctx.pos_attention(q, k, v, 4, 2), ok[0])


def test_outputs_on_top_of_inputs_are_refused(backend, request):
    ctx = ctx_of(backend, torch.float16, request)
    q, k, v = (torch.randn(2, 9, 128).half().to(ctx.torch_device) for _ in range(3))
    out, lse = ctx.pos_attention(q, k, v, 2, return_lse=True)
    ref = ctx.pos_attention_backward(out, q, k, v, lse, 2)
    for t in (q, k, v):
        with pytest.raises(L.StarError, match="must not be"):
            ctx.pos_attention(q, k, v, 2, out=t)
    for kw in ({"dq": q}, {"dq": out}, {"dk": k}, {"dv": q}, {"dk": ref[2], "dv": ref[2]}, {"dq": ref[1], "dk": ref[1]}):
        with pytest.raises(L.StarError, match="must not be"):
            ctx.pos_attention_backward(out, q, k, v, lse, 2, **kw)
    again = ctx.pos_attention_backward(out, q, k, v, lse, 2)
    assert all(torch.equal(a, b) for a, b in zip(ref[:3], again[:3]))


def test_refusals_of_the_c_entry_points(backend, request):
    ctx = ctx_of(backend, torch.float16, request)
    dev = ctx.torch_device
    q = torch.zeros(1, 4, 64, dtype=torch.float16, device=dev)
    k = torch.zeros(1, 900, 64, dtype=torch.float16, device=dev)
    lib, err = ctx.lib, lambda: ctx.lib.last_error(ctx.h).decode()

    def desc():
        d = ctx._pos_desc(q, k, k, 1, 1, None, None, 0, False, None, None, None)
        out = torch.zeros(1, 4, 64, dtype=torch.float16, device=dev)
        d.O, d.ldo, d.bso = out.data_ptr(), 64, 0
        d._keep = out
        return d

    d = desc()
    need = lib.pos_attn_workspace(ctx.h, ctypes.byref(d), 0)
    assert need > 0 and lib.pos_attn_fwd(ctx.h, ctypes.byref(d)) and "workspace" in err()
    ws = torch.empty(need, dtype=torch.uint8, device=dev)
    d.workspace, d.workspace_bytes = ws.data_ptr(), need - 1
    assert lib.pos_attn_fwd(ctx.h, ctypes.byref(d)) and "workspace" in err()
    d.workspace_bytes = need
    assert lib.pos_attn_fwd(ctx.h, ctypes.byref(d)) == 0
    for field, value in (("Q", None), ("K", None), ("O", None), ("Q", q.data_ptr() + 2), ("ldq", 60), ("ldk", 1 << 24), ("ldk", -64), ("bsk", 4), ("heads", 0),
                         ("kv_heads", 2), ("Nq", -1), ("Nk", (1 << 28) + 1), ("batch", -1), ("sinks", -3), ("bias_table", q.data_ptr()), ("bias_buckets", q.data_ptr())):
        d = desc()
        d.workspace, d.workspace_bytes = ws.data_ptr(), need
        setattr(d, field, value)
        assert lib.pos_attn_fwd(ctx.h, ctypes.byref(d)), (field, value)
        assert "pos_attn_fwd" in err()
    assert lib.pos_attn_fwd(ctx.h, None) and lib.pos_attn_fwd(None, ctypes.byref(desc()))
    d, g = desc(), L.PosAttnGrads()
    assert lib.pos_attn_bwd(ctx.h, ctypes.byref(d), ctypes.byref(g)) and lib.pos_attn_bwd(ctx.h, ctypes.byref(d), None)


@pytest.mark.parametrize("dtype", DTYPES)
def test_streaming_equals_the_whole_sequence(backend, dtype, request):
    """a layer as it is used: norm, attention over the window and the first tokens; the sequence at once, in chunks, and a token at a time
    against a cache give the same outputs up to their roundings"""
    ctx = ctx_of(backend, dtype, request)
    dev = ctx.torch_device
    N, H, KH, C = 150, 2, 1, 128
    g = torch.Generator().manual_seed(5)
    x = torch.randn(N, C, generator=g).to(dtype).to(dev)
    w = (torch.randn(256, C, generator=g) / 11).to(dtype).to(dev)
    gamma = (1 + 0.2 * torch.randn(C, generator=g)).to(dev)
    table, bk = torch.randn(16, H, generator=g).to(dev), ctx.rel_buckets(16, 40, bidirectional=False)
    kw = dict(window=(50, 0), sinks=6, bias=(table, bk))

    def qkv(rows):
        y = ctx.layer_norm_train(rows, gamma)[0]
        f = ctx.gemm(y, w)
        return f[:, :128], f[:, 128:192], f[:, 192:]

    q, k, v = qkv(x)
    whole = ctx.pos_attention(q[None], k[None], v[None], H, KH, **kw)[0]
    ref = O.pos_attention(q[None].cpu(), k[None].cpu(), v[None].cpu(), H, KH, 0.125, 50, 0, 6, bias=(table.cpu(), bk.tolist()))
    within(whole[None], ref["out"], ref["tol_out"], "whole")
    cache_k = torch.full((1, 200, 64), float("nan"), dtype=dtype, device=dev)
    cache_v = torch.full((1, 200, 64), float("nan"), dtype=dtype, device=dev)
    done = 0
    for n in (40, 1, 1, 60, 1, 46, 1):
        qc, kc, vc = qkv(x[done:done + n])
        cache_k[0, done:done + n], cache_v[0, done:done + n] = kc, vc
        pos = torch.tensor([done], dtype=torch.int32, device=dev)
        length = torch.tensor([done + n], dtype=torch.int32, device=dev)
        got = ctx.pos_attention(qc[None], cache_k, cache_v, H, KH, q_start=pos, kv_len=length, **kw)
        within(got, ref["out"][:, done:done + n], ref["tol_out"][:, done:done + n], f"tokens from {done}")
        done += n
    assert done == N


@pytest.mark.parametrize("dtype", DTYPES)
def test_a_training_step_of_a_block(backend, dtype, request):
    """norm -> projection -> attention with bias, and back: the gradients of the table and of the norm's weights against autograd in 64
    bits through the whole block.  The kernels round the chain's tensors to 16 bits (y, qkv, dO, dq, dk, dv, dy: seven roundings of a half
    step each, root of their squares below 3 half steps of the gradient's norm; 8 is allowed)."""
    ctx = ctx_of(backend, dtype, request)
    dev = ctx.torch_device
    B, N, H, C = 2, 45, 2, 128
    g = torch.Generator().manual_seed(11)
    x = torch.randn(B * N, C, generator=g).to(dtype)
    w = (torch.randn(3 * 128, C, generator=g) / 11).to(dtype)
    gamma, beta, table = 1 + 0.2 * torch.randn(C, generator=g), 0.1 * torch.randn(C, generator=g), torch.randn(16, H, generator=g)
    do = (0.1 * torch.randn(B, N, 128, generator=g)).to(dtype)
    lens = [45, 30]
    bk = O.bucket_scheme(16, 20, True)

    with torch.enable_grad():
        leaves = [t.double().requires_grad_() for t in (x, gamma, beta, table)]
        X, Ga, Be, Ta = leaves
        xh = (X - X.mean(1, keepdim=True)) / torch.sqrt(X.var(1, keepdim=True, correction=0) + 1e-5)
        f = ((xh * Ga + Be) @ w.double().T).reshape(B, N, 3, H, 64)
        loss = 0
        for b in range(B):
            ok, rel = O.visible(N, N, start=0, n=lens[b])
            for h in range(H):
                s = f[b, :, 0, h] @ f[b, :, 1, h].T * 0.125 + Ta[:, h][torch.tensor(bk)[rel.clamp(-20, 20) + 20]]
                p = torch.softmax(s.masked_fill(~ok, -1e30), 1)
                loss = loss + ((p @ f[b, :, 2, h]) * do[b, :, h * 64:(h + 1) * 64].double()).sum()
        loss.backward()

    xd, wd, gd = x.to(dev), w.to(dev), gamma.to(dev)
    y, stats = ctx.layer_norm_train(xd, gd, beta.to(dev))
    qkv = ctx.gemm(y, wd).reshape(B, N, 384)
    kw = dict(kv_len=torch.tensor(lens, dtype=torch.int32, device=dev), bias=(table.to(dev), ctx.rel_buckets(16, 20)))
    q, k, v = qkv[:, :, :128], qkv[:, :, 128:256], qkv[:, :, 256:]
    _, lse = ctx.pos_attention(q, k, v, H, return_lse=True, **kw)
    dqkv = torch.empty_like(qkv)
    *_, dtable = ctx.pos_attention_backward(do.to(dev), q, k, v, lse, H, dq=dqkv[:, :, :128], dk=dqkv[:, :, 128:256], dv=dqkv[:, :, 256:], **kw)
    dy = ctx.gemm(dqkv.reshape(B * N, 384), wd.t().contiguous())
    dx, dgamma, dbeta = ctx.layer_norm_backward(dy, xd, stats, gd)
    for got, leaf, what in ((dx, X, "x"), (dgamma, Ga, "gamma"), (dbeta, Be, "beta"), (dtable, Ta, "table")):
        off = (got.cpu().double() - leaf.grad).norm() / leaf.grad.norm()
        assert off <= 8 * O.half_step(dtype), (what, float(off))


# ------------------------------------------------------------------------------------------------------ streams and graphs
@pytest.mark.gpu
def test_another_stream_and_two_at_once():
    """calls follow torch's current stream; two streams at once do not share scratch memory"""
    ctx = L.Context(0, torch.float16)
    q, k, v, do, _ = inputs(torch.float16, 4, 1, 5000, 8, 2, 1)
    a = [t.cuda() for t in (q, k, v)]
    b = [t.cuda() for t in inputs(torch.float16, 4, 1, 5000, 8, 2, 2)[:3]]
    ra, rb = ctx.pos_attention(*a, 8, 2), ctx.pos_attention(*b, 8, 2)
    torch.cuda.synchronize()
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    outs = []
    for _ in range(20):
        with torch.cuda.stream(s1):
            outs.append((ctx.pos_attention(*a, 8, 2), ra))
        with torch.cuda.stream(s2):
            outs.append((ctx.pos_attention(*b, 8, 2), rb))
    torch.cuda.synchronize()
    assert all(torch.equal(o, r) for o, r in outs)


def test_the_own_stream_stays(backend, request):
    """a call on another stream leaves the context's own one as it was for the calls that do not follow torch's; refused calls too"""
    ctx = ctx_of(backend, torch.float16, request)
    own, seen = ctypes.c_void_p(), ctypes.c_void_p()
    assert ctx.lib.borrow_stream(None, None, None)

    def own_stream():
        assert ctx.lib.borrow_stream(ctx.h, None, ctypes.byref(seen)) == 0 and ctx.lib.borrow_stream(ctx.h, seen, None) == 0
        return seen.value

    before = own_stream()
    x = torch.randn(70, 64).half().to(ctx.torch_device)
    ref = ctx.layer_norm_train(x)
    if backend == "emu":
        assert ctx.lib.borrow_stream(ctx.h, 4096, ctypes.byref(own)) == 0 and own.value == before and own_stream() == 4096
        assert ctx.lib.borrow_stream(ctx.h, own, None) == 0
        return
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        y = ctx.layer_norm_train(x)
        assert own_stream() == before
        with pytest.raises(L.StarError):
            ctx.pos_attention(x[None], x[None], x[None], 1, out=x[None])
    assert own_stream() == before
    s.synchronize()
    assert torch.equal(y[0], ref[0]) and torch.equal(y[1], ref[1])


@pytest.mark.gpu
def test_captured_graphs_replayed_together():
    """a training step and two decoding steps captured into graphs, replayed several times, on two streams, with eager work between"""
    ctx = L.Context(0, torch.bfloat16)
    dev = "cuda"
    g = torch.Generator().manual_seed(3)
    q, k, v, do, bias = inputs(torch.bfloat16, 2, 300, 300, 4, 2, 5, buckets=32, distance=128)
    q, k, v, do = (t.to(dev) for t in (q, k, v, do))
    table, bk = bias[0].to(dev), torch.tensor(bias[1], dtype=torch.int32, device=dev)
    x, gamma = torch.randn(600, 256, generator=g).bfloat16().to(dev), torch.ones(256, device=dev)
    lens = torch.tensor([300, 120], dtype=torch.int32, device=dev)

    def step():
        y, st = ctx.layer_norm_train(x, gamma)
        out, lse = ctx.pos_attention(q, k, v, 4, 2, kv_len=lens, bias=(table, bk), return_lse=True)
        grads = ctx.pos_attention_backward(do, q, k, v, lse, 4, 2, kv_len=lens, bias=(table, bk))
        return [y, out, *grads, *ctx.layer_norm_backward(y, x, st, gamma)]

    caches = [[t.to(dev) for t in inputs(torch.bfloat16, 2, 1, 4000, 4, 1, 60 + i)[:3]] for i in range(2)]
    works = [step] + [lambda c=c: [ctx.pos_attention(*c, 4, 1, window=(3000, 0), sinks=4)] for c in caches]
    graphs, outs = [], []
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for w in works:
            w()
    torch.cuda.current_stream().wait_stream(side)
    for w in works:
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            outs.append(w())
        graphs.append(gr)
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    for turn in range(4):
        x.normal_()
        q.normal_()
        for c in caches:
            c[0].normal_()
        torch.cuda.synchronize()
        for t in outs:
            for o in t:
                o.zero_()
        torch.cuda.synchronize()
        with torch.cuda.stream(s1):
            graphs[0].replay()
            graphs[1].replay()
        with torch.cuda.stream(s2):
            graphs[2].replay()
        torch.cuda.synchronize()
        eager = [w() for w in works]
        torch.cuda.synchronize()
        for a, b in zip(outs, eager):
            assert all(torch.equal(s, t) for s, t in zip(a, b)), turn


@pytest.mark.gpu
def test_capture_by_a_context_whose_arena_is_in_use():
    """a context that has run a layer with scratch memory of its own on the default stream is captured from another"""
    ctx = L.Context(0, torch.float16)
    big = torch.randn(1000, 320, device="cuda").half()
    ctx.group_norm(big, torch.ones(320, device="cuda"), torch.zeros(320, device="cuda"), 1000)      # (takes blocks of the arena)
    assert ctx.lib.pool_bytes(ctx.h) > 0
    x = torch.randn(64, 320, device="cuda").half()
    ref = ctx.layer_norm_train(x)[0]
    gr = torch.cuda.CUDAGraph()
    with torch.cuda.graph(gr):
        y, _ = ctx.layer_norm_train(x)
    y.zero_()
    for _ in range(3):
        gr.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, ref)
        y.zero_()
    assert torch.equal(ctx.layer_norm_train(x)[0], ref)
