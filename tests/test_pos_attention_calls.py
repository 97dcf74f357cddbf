"""Calls of the position-dependent attention (star_pos_attn_fwd / _bwd) that its documentation allows and that lie at an edge: empty batches over shared
keys, caches past 32 bits, launches past what a grid holds."""
import ctypes
import os
import sys

import pytest
import torch

sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "oracle"))
import train_ops_oracle as O  # noqa: E402
from util import BACKENDS, make_ctx  # noqa: E402

from star_amd import lib as L  # noqa: E402


@pytest.fixture(params=BACKENDS)
def backend(request):
    return request.param


def ctx_of(backend, dtype, request):
    return make_ctx(backend, dtype, request.getfixturevalue("emu_lib") if backend == "emu" else None)


def test_no_sequence_over_shared_keys(backend, request):
    """the gradients of keys that no sequence uses are zeros, also in given tensors"""
    ctx = ctx_of(backend, torch.float16, request)
    dev = ctx.torch_device
    q, kv = torch.zeros(0, 3, 128, dtype=torch.float16, device=dev), torch.ones(1, 4, 128, dtype=torch.float16, device=dev)
    bias = (torch.ones(2, 2, device=dev), torch.tensor([0, 1, 1], dtype=torch.int32, device=dev))
    out, lse = ctx.pos_attention(q, kv, kv, 2, return_lse=True)
    given = torch.full((2, 1, 4, 128), 7.0, dtype=torch.float16, device=dev)
    dq, dk, dv, dt = ctx.pos_attention_backward(out, q, kv, kv, lse, 2, bias=bias, dk=given[0], dv=given[1])
    assert dq.shape == (0, 3, 128) and dk.shape == dv.shape == kv.shape
    assert not given.any() and not dt.any()


def test_launches_past_what_a_grid_holds_are_refused(backend, request):
    """2^24 workgroups of 256 threads, or 2^26 of 64, are more threads than a launch counts: refused on the host, before anything runs"""
    ctx = ctx_of(backend, torch.float16, request)
    dev = ctx.torch_device
    t = torch.zeros(2, 64, dtype=torch.float16, device=dev)
    f = torch.zeros(64, dtype=torch.float32, device=dev)

    def call(batch, Nq, backward):
        d = L.PosAttnDesc()
        d.Q = d.K = d.V = t.data_ptr()
        d.O, d.lse = t[1:].data_ptr(), f.data_ptr()
        d.ldq = d.ldk = d.ldv = d.ldo = 64
        d.bsq, d.bsk, d.bsv, d.bso = 64 * Nq, 0, 0, 64 * Nq
        d.Nq, d.Nk, d.heads, d.kv_heads, d.batch, d.scale, d.left, d.right = Nq, 1, 1, 1, batch, 1.0, -1, -1
        need = ctx.lib.pos_attn_workspace(ctx.h, ctypes.byref(d), backward)
        d.workspace, d.workspace_bytes = f.data_ptr(), need      # (as if there were so much: nothing is launched)
        if not backward:
            return ctx.lib.pos_attn_fwd(ctx.h, ctypes.byref(d))
        g = L.PosAttnGrads()
        o = torch.zeros(3, 64, dtype=torch.float16, device=dev)
        g.dO, g.dQ, g.dK, g.dV = t[1:].data_ptr(), *(x.data_ptr() for x in o)
        g.lddo = g.lddq = g.lddk = g.lddv = 64
        g.bsdo, g.bsdq, g.bsdk, g.bsdv = 64 * Nq, 64 * Nq, 0, 0
        return ctx.lib.pos_attn_bwd(ctx.h, ctypes.byref(d), ctypes.byref(g))

    for batch, Nq, backward in ((1 << 26, 1, 0), (1 << 24, 33, 0), (1 << 24, 1, 1)):
        assert call(batch, Nq, backward) and b"too many workgroups" in ctx.lib.last_error(ctx.h), (batch, Nq, backward)
    x = t.data_ptr()
    for rows, C in ((1 << 24, 2561), (1 << 26, 2560), (1 << 26, 1304), (1 << 26, 512)):
        assert ctx.lib.layer_norm_train(ctx.h, x, C, x, C, None, None, None, rows, C, 1e-5) and b"too many rows" in ctx.lib.last_error(ctx.h), (rows, C)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_all_gradients_of_a_cache_past_32_bits(dtype):
    """the last keys of a cache of more than 2^32 bytes are the ones that count: dv of them too, with a bias and without"""
    ctx = L.Context(0, dtype)
    Nk, tail, Nq = (1 << 32) // (2 * 1024) + 300, 500, 70
    k = torch.zeros(1, Nk, 1024, dtype=dtype, device="cuda")[:, :, 960:]
    v = torch.zeros(1, Nk, 1024, dtype=dtype, device="cuda")[:, :, :64]
    g = torch.Generator().manual_seed(3)
    k[:, -tail:], v[:, -tail:] = (torch.randn(1, tail, 64, generator=g).to(dtype).cuda() for _ in range(2))
    q, do = (torch.randn(1, Nq, 64, generator=g).to(dtype) for _ in range(2))
    for bias in (None, (torch.randn(16, 1, generator=g), O.bucket_scheme(16, 30, True))):
        ref = O.pos_attention(q, k[:, -tail:].cpu(), v[:, -tail:].cpu(), 1, 1, 0.125, 200, 0, 0, bias=bias, dout=do, tight=True)
        kw = {"window": (200, 0)}
        if bias is not None:
            kw["bias"] = (bias[0].cuda(), torch.tensor(bias[1], dtype=torch.int32, device="cuda"))
        out, lse = ctx.pos_attention(q.cuda(), k, v, 1, return_lse=True, **kw)
        dq, dk, dv, dt = ctx.pos_attention_backward(do.cuda(), q.cuda(), k, v, lse, 1, **kw)
        for n, t in (("out", out), ("dq", dq), ("dk", dk[:, -tail:]), ("dv", dv[:, -tail:]), ("dtable", dt)):
            if t is not None:
                assert (t.cpu().double() - ref[n]).abs().le(ref["tol_" + n]).all(), n
        assert not dk[:, :-tail].any() and not dv[:, :-tail].any()
