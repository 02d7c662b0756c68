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


@pytest.mark.parametrize("hk,launches", [(2, 1), (150, 2)])  # the few-row kernel, the tile kernel
@pytest.mark.parametrize("pad", [0, 4, 3])
@pytest.mark.parametrize("dim", [64, 256])
def test_outputs_over_the_queries(ctx, hk, launches, pad, dim):
    """o is q, contiguous, strided and unaligned: what separate buffers give, and nothing beside the rows is
    touched."""
    torch = _torch()
    s = Setup(ctx, [(40, 150), (33, 70), (1, 9)], 2 * hk, hk, dim, 16, rows_before=1, rows_behind=2)
    n = 2 * hk * dim
    table = torch.from_numpy(tb.rope_table(1e4, dim, 150)).cuda()
    whole = torch.from_numpy(s.codes(n + pad)).cuda()
    q, scale = whole[:, pad // 2:pad // 2 + n], torch.from_numpy(s.scales()).cuda()
    before_beside = torch.cat([whole[:, :pad // 2], whole[:, pad // 2 + n:]], 1)
    outs = []
    for o in (q.clone(), q):
        os_ = torch.full((s.rows, hk, 2), 77, dtype=torch.int64, device="cuda")
        before = ctx.launch_count()
        s.cache.attention(s.batch, q, scale, o, os_, 2 * hk, rope=tb.Rope(table), window=60, sinks=2)
        assert ctx.launch_count() - before == launches
        outs.append((o, os_))
    ctx.sync()
    torch.cuda.synchronize()
    assert torch.equal(outs[0][0], outs[1][0]) and torch.equal(outs[0][1], outs[1][1])
    beside = torch.cat([whole[:, :pad // 2], whole[:, pad // 2 + n:]], 1)
    assert torch.equal(beside, before_beside)


def test_outputs_over_the_queries_at_another_stride(ctx):
    """The same memory at another row stride would be written before it is read: refused."""
    torch = _torch()
    s = Setup(ctx, [(2, 9)], 2, 1, 16, 16)
    memory = torch.zeros(80, dtype=torch.int32, device="cuda")
    q, o = memory.as_strided((2, 32), (32, 1)), memory.as_strided((2, 32), (40, 1))
    scale, os_ = torch.from_numpy(s.scales()).cuda(), torch.zeros(2, 1, 2, dtype=torch.int64, device="cuda")
    for a, b in ((q, o), (o, q)):
        with pytest.raises(tb.KtmoeError) as e:
            s.cache.attention(s.batch, a, scale, b, os_, 2)
        assert e.value.status == _native.ERR_ARG
    ctx.sync()
