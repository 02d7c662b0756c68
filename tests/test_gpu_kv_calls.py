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


@pytest.mark.parametrize("dim", [144, 160, 208, 240])
def test_heads_between_128_and_256(ctx, dim):
    """Rows of one whole 128-byte block and a part, rotated, windowed, written, read and attended."""
    torch = _torch()
    s = Setup(ctx, [(70, 70), (1, 300), (35, 200)], 4, 2, dim, 32, seed=dim, rows_behind=1)
    table = tb.rope_table(1e4, dim - 16, 301)
    rope = tb.Rope(torch.from_numpy(table).cuda(), dim == 160)
    k, v, scale = s.codes(2 * dim), s.codes(2 * dim), s.scales()
    R.append(k.reshape(s.rows, 2, dim), v.reshape(s.rows, 2, dim), scale, s.begin, s.kv_len, s.write, table, dim == 160)
    s.cache.append(s.batch, torch.from_numpy(k).cuda(), torch.from_numpy(v).cuda(), torch.from_numpy(scale).cuda(), rope)
    ko, vo = torch.zeros(s.rows, 2 * dim, device="cuda"), torch.zeros(s.rows, 2 * dim, device="cuda")
    s.cache.read(s.batch, ko, vo)
    ctx.sync()
    torch.cuda.synchronize()
    for n, t in (("k", s.cache.k), ("v", s.cache.v), ("ks", s.cache.k_scale), ("vs", s.cache.v_scale)):
        assert (t.double().cpu().numpy() == s.pool[n].astype(np.float64)).all(), n
    page, place = s.place(0, 69)
    for n, o in (("k", ko), ("v", vo)):
        assert (o[69].reshape(2, dim).cpu().numpy() == s.pool[n][page, :, place] * s.pool[n + "s"][page, :, place][:, None]).all()
    s.check(s.codes(4 * dim), scale, table, dim == 160)
    s.check(s.codes(4 * dim), scale, table, dim == 160, window=50, sinks=3)


@pytest.mark.parametrize("window,sinks", [(0, 0), (40, 2)])
@pytest.mark.parametrize("heads,hk", [(4, 2), (8, 1)])
def test_a_chunk_among_decoding_sequences(ctx, heads, hk, window, sinks):
    """One long chunk in a batch of single tokens, sequences that add nothing between them, and a page table far wider
    than any sequence."""
    lens = [(1, 1 + 37 * i % 200) for i in range(9)] + [(280, 333), (0, 50)] + [(1, 300 - 13 * i) for i in range(14)]
    s = Setup(ctx, lens, heads, hk, 64, 16, seed=heads, rows_before=2, rows_behind=3)
    wide = _torch().full((len(lens), 3000), 2 ** 31 - 1, dtype=_torch().int32, device="cuda")  # no page of the pool
    wide[:, :s.max_pages] = s.batch.page_table
    s.batch = tb.KvBatch(s.batch.q_begin, s.batch.kv_len, wide, s.rows)
    q, scale = s.codes(heads * 64), s.scales()
    torch = _torch()
    for copies, launches in ((1, None), (-(-148 // hk), 2)):
        cache = tb.KvCache(ctx, s.cache.n_pages, 16, copies * hk, 64, pools=[
            t.repeat(1, copies, *[1] * (t.dim() - 2)) for t in (s.cache.k, s.cache.v, s.cache.k_scale, s.cache.v_scale)])
        o = torch.full((s.rows, copies * heads * 64), 77, dtype=torch.int32, device="cuda")
        os_ = torch.full((s.rows, copies * hk, 2), 77, dtype=torch.int64, device="cuda")
        before = ctx.launch_count()
        cache.attention(s.batch, torch.from_numpy(q).cuda().repeat(1, copies), torch.from_numpy(scale).cuda(), o, os_,
                        copies * heads, window=window, sinks=sinks)
        assert launches is None or heads < 8 or ctx.launch_count() - before == launches  # the tile kernel
        ctx.sync()
        torch.cuda.synchronize()
        want = np.full((s.rows, heads, 64), 77, np.int64)
        want_s = np.full((s.rows, hk, 2), 77, np.int64)
        R.attention(q.reshape(s.rows, heads, 64), scale, s.begin, s.kv_len, s.keys, want, want_s, 64 ** -0.5, window, sinks)
        want_s[..., 1] &= 0xFFFFFFFF
        for got, w in ((o, want.reshape(s.rows, -1)), (os_, want_s)):
            got = got.reshape(s.rows, copies, -1).cpu().numpy()
            assert (got == w.reshape(s.rows, 1, -1)).all()


def test_a_busy_stream_is_waited_for_where_it_is_given(ctx):
    """A wrong batch on a stream that is busy: the sync that is given the stream raises it."""
    torch = _torch()
    s = Setup(ctx, [(1, 100)], 4, 2, 64, 16)
    q, scale = torch.from_numpy(s.codes(256)).cuda(), torch.from_numpy(s.scales()).cuda()
    out, os_ = torch.zeros_like(q), torch.zeros(1, 2, 2, dtype=torch.int64, device="cuda")
    s.cache.attention(s.batch, q, scale, out, os_, 4)
    ctx.sync()
    s.batch.page_table[0, 2] = s.cache.n_pages
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        torch.cuda._sleep(200_000_000)  # about a tenth of a second
        s.cache.attention(s.batch, q, scale, out, os_, 4)
    with pytest.raises(tb.KtmoeError) as e:
        ctx.sync(side.cuda_stream)
    assert e.value.status == _native.ERR_ARG
    ctx.sync()


def test_the_cache_in_order_with_a_half(ctx):
    """A half's forward on the context's stream and, unsynchronised behind it, the rows that it wrote read back on that
    stream (stream=0): what they are once everything has come to rest."""
    torch = _torch()
    d, n = 2048, 64
    lin = lambda seed, out, k: tb.QuantLinear.from_weights("w", tb.synth_normal(seed, 0.05, out * k), out, k)
    half = tb.AttentionHalf(ctx, d, 4, 2, 64)
    half.set_qkv(lin(1, 256, d), lin(2, 128, d), lin(3, 128, d))
    half.set_out(lin(4, d, 256))
    norm = tb.QuantLinear.from_weights("n", tb.synth_normal(5, 1.0, d), 1, d)
    half.set_norm(norm.w_codes, norm.w_scale, tb.scale_from_f64(1e-6))
    i32 = lambda *a: torch.tensor(a, dtype=torch.int32, device="cuda")
    batch = tb.KvBatch(i32(0, n), i32(n), i32(2, 0, 1, 3).reshape(1, 4), n)
    cache = tb.KvCache(ctx, 4, 16, 2, 64)
    x = torch.from_numpy(tb.IntTensor.from_reals(tb.synth_normal(6, 1.0, n * d)).data.copy()).cuda()
    xs = torch.tensor([1, 28], dtype=torch.int64, device="cuda")
    y, ys = torch.zeros_like(x), torch.zeros_like(xs)
    got = [torch.zeros(n, 128, device="cuda") for _ in range(4)]
    torch.cuda.synchronize()
    half.forward_dev(cache, batch, x.data_ptr(), xs.data_ptr(), y.data_ptr(), ys.data_ptr())
    cache.read(batch, got[0], got[1], stream=0)
    ctx.sync()
    torch.cuda.synchronize()
    cache.read(batch, got[2], got[3])
    torch.cuda.synchronize()
    assert torch.equal(got[0], got[2]) and torch.equal(got[1], got[3])
    assert int((got[0] != 0).sum()) > n * 64
