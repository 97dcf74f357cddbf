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
