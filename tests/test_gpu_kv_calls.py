"""Calls of the cache and attention that their documentation allows or rules out, at its edges, on a B200."""

import ctypes

import numpy as np
import pytest

import kv_reference as R
import tritify_b200 as tb
from test_gpu_kv import Setup, _torch
from tritify_b200 import _native

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("n", [2 ** 30 + 1, 2 ** 31 - 1])
def test_more_sequences_than_a_batch_holds(ctx, n):
    """Refused before anything is read: the search for a row's sequence counts in 32 bits."""
    torch = _torch()
    s = Setup(ctx, [(1, 5)], 1, 1, 16, 16)
    b = _native.KtmoeKvBatch.from_buffer_copy(s.batch._c)
    b.n_seqs = n
    x, f = torch.zeros(1, 16, dtype=torch.int32, device="cuda"), torch.zeros(1, 16, device="cuda")
    sc, os_ = torch.zeros(1, 2, dtype=torch.int64, device="cuda"), torch.zeros(1, 1, 2, dtype=torch.int64, device="cuda")
    L, a = tb.lib(), [ctx.handle, s.cache._c, b]
    p, ps = x.data_ptr(), sc.data_ptr()
    assert L.ktmoe_kv_append_dev(*a, p, 16, p, 16, ps, None, 1, None, None) == _native.ERR_ARG
    assert L.ktmoe_kv_read_dev(*a, f.data_ptr(), 16, f.data_ptr(), 16, None) == _native.ERR_ARG
    assert L.ktmoe_attention_dev(*a, p, 16, ps, 1, None, 1, 1.0, 0, 0, p, 16, os_.data_ptr(), None) == _native.ERR_ARG
    ctx.sync()
