"""Setting an attention half's weights on a B200: what is refused, and that a forward in flight keeps what it began with."""

import numpy as np
import pytest

import tritify_b200 as tb
from tritify_b200 import _native

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("bad", [tb.WLEVELS + 1, -tb.WLEVELS - 1, 2 ** 31 - 1, -2 ** 31])
def test_norm_codes_beyond_their_range(ctx, bad):
    """As a layer's norm: codes outside +-WLEVELS are refused; those at its ends are taken."""
    a = tb.AttentionHalf(ctx, 64, 2, 1, 16)
    codes = np.ones(64, np.int32)
    codes[:2] = tb.WLEVELS, -tb.WLEVELS
    a.set_norm(codes, tb.Scale(1, 0), tb.Scale(0, 0))
    codes[63] = bad
    with pytest.raises(tb.KtmoeError) as e:
        a.set_norm(codes, tb.Scale(1, 0), tb.Scale(0, 0))
    assert e.value.status == _native.ERR_RANGE


def _linear(seed, out, k):
    return tb.QuantLinear.from_weights("w", tb.synth_normal(seed, 1.0, out * k), out, k)


def _half(ctx, seed):
    a = tb.AttentionHalf(ctx, 64, 2, 1, 32)
    set_all(a, seed)
    return a


def set_all(a, seed, only=None):
    if only in (None, "qkv"):
        a.set_qkv(_linear(seed, 64, 64), _linear(seed + 1, 32, 64), _linear(seed + 2, 32, 64))
    if only in (None, "out"):
        a.set_out(_linear(seed + 3, 64, 64))
    if only in (None, "norm"):
        norm = tb.QuantLinear.from_weights("n", tb.synth_normal(seed + 4, 1.0, 64), 1, 64)
        a.set_norm(norm.w_codes, norm.w_scale, tb.scale_from_f64(1e-6))
    if only in (None, "rope"):
        a.set_rope(1e4 + 5e3 * seed, 32, 64)


@pytest.mark.parametrize("what", ["norm", "rope", "qkv", "out"])
def test_a_forward_in_flight_keeps_its_weights(ctx, what):
    """A forward that waits on the caller's stream while a setter is called: it gives what it gave before the call, and
    the next one what the new weights give."""
    import torch

    i32 = lambda *a: torch.tensor(a, dtype=torch.int32, device="cuda")
    batch = tb.KvBatch(i32(0, 9), i32(9), i32(0).reshape(1, 1), 9)
    x = torch.from_numpy(tb.IntTensor.from_reals(tb.synth_normal(9, 1.0, 9 * 64)).data.reshape(9, 64).copy()).cuda()
    xs = torch.tensor([1, 28], dtype=torch.int64, device="cuda")
    side = torch.cuda.Stream()

    def forward(a, y, ys, wait):
        with torch.cuda.stream(side):
            if wait:
                torch.cuda._sleep(200_000_000)  # about a tenth of a second
            a.forward_dev(cache, batch, x.data_ptr(), xs.data_ptr(), y.data_ptr(), ys.data_ptr(), side.cuda_stream)

    def results(n):
        return [(torch.zeros_like(x), torch.zeros(2, dtype=torch.int64, device="cuda")) for _ in range(n)]

    cache = tb.KvCache(ctx, 1, 16, 1, 32)
    fresh = _half(ctx, 100)
    set_all(fresh, 200, what)
    a = _half(ctx, 100)
    (first, delayed, after, want) = results(4)
    torch.cuda.synchronize()
    forward(a, *first, wait=False)
    torch.cuda.synchronize()
    forward(a, *delayed, wait=True)
    set_all(a, 200, what)
    forward(a, *after, wait=False)
    forward(fresh, *want, wait=False)
    ctx.sync(side.cuda_stream)
    assert torch.equal(first[0], delayed[0]) and torch.equal(first[1], delayed[1])
    assert torch.equal(after[0], want[0]) and torch.equal(after[1], want[1])
    assert not torch.equal(first[0], after[0])


def test_rotation_tables_that_grow_shrink_and_fail(ctx):
    """Each set_rope gives what a half with that table alone gives; one that is refused leaves the last one."""
    import torch

    i32 = lambda *a: torch.tensor(a, dtype=torch.int32, device="cuda")
    batch = tb.KvBatch(i32(0, 9), i32(9), i32(0).reshape(1, 1), 9)
    x = torch.from_numpy(tb.IntTensor.from_reals(tb.synth_normal(9, 1.0, 9 * 64)).data.reshape(9, 64).copy()).cuda()
    xs = torch.tensor([1, 28], dtype=torch.int64, device="cuda")
    cache = tb.KvCache(ctx, 1, 16, 1, 32)

    def result(a):
        y, ys = torch.zeros_like(x), torch.zeros(2, dtype=torch.int64, device="cuda")
        torch.cuda.synchronize()
        a.forward_dev(cache, batch, x.data_ptr(), xs.data_ptr(), y.data_ptr(), ys.data_ptr())
        ctx.sync()
        return y.cpu(), ys.cpu()

    a, seen = _half(ctx, 300), []
    for theta, rot, positions in ((1e4, 32, 64), (2e4, 32, 5000), (3e4, 16, 20), (3e4, 8, 100000)):
        a.set_rope(theta, rot, positions)
        with pytest.raises(tb.KtmoeError):
            a.set_rope(-1.0, 32, 64)
        fresh = tb.AttentionHalf(ctx, 64, 2, 1, 32)
        for what in ("qkv", "out", "norm"):
            set_all(fresh, 300, what)
        fresh.set_rope(theta, rot, positions)
        got, want = result(a), result(fresh)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
        assert all(not torch.equal(got[0], s) for s in seen)
        seen.append(got[0])


@pytest.mark.parametrize("rows", [1, 9])
def test_a_half_over_its_own_input(ctx, rows):
    """y is x, with its scale: what separate buffers give."""
    import torch

    i32 = lambda *a: torch.tensor(a, dtype=torch.int32, device="cuda")
    batch = tb.KvBatch(i32(0, rows), i32(rows), i32(0).reshape(1, 1), rows)
    x = torch.from_numpy(tb.IntTensor.from_reals(tb.synth_normal(9, 1.0, rows * 64)).data.reshape(rows, 64).copy()).cuda()
    xs = torch.tensor([1, 28], dtype=torch.int64, device="cuda")
    cache, a = tb.KvCache(ctx, 1, 16, 1, 32), _half(ctx, 400)
    y, ys = torch.zeros_like(x), torch.zeros_like(xs)
    torch.cuda.synchronize()
    a.forward_dev(cache, batch, x.data_ptr(), xs.data_ptr(), y.data_ptr(), ys.data_ptr())
    a.forward_dev(cache, batch, x.data_ptr(), xs.data_ptr(), x.data_ptr(), xs.data_ptr())
    ctx.sync()
    assert torch.equal(x, y) and torch.equal(xs, ys)


@pytest.mark.parametrize("rows", [2 ** 30 + 1, 2 ** 40, 2 ** 62, 2 ** 63 - 1, -1])
def test_more_rows_than_a_batch_holds(ctx, rows):
    """Refused before the scratch is sized for them, where 2^62 rows by four heads would count as none; the half serves on."""
    import torch

    a = tb.AttentionHalf(ctx, 64, 4, 4, 16)
    a.set_qkv(*(_linear(i, 64, 64) for i in range(3)))
    a.set_out(_linear(4, 64, 64))
    a.set_norm(np.ones(64, np.int32), tb.Scale(1, 0), tb.Scale(0, 0))
    i32 = lambda *a: torch.tensor(a, dtype=torch.int32, device="cuda")
    batch = tb.KvBatch(i32(0, 2), i32(2), i32(0).reshape(1, 1), 2)
    cache = tb.KvCache(ctx, 1, 16, 4, 16)
    x = torch.ones(2, 64, dtype=torch.int32, device="cuda")
    xs = torch.tensor([1, 0], dtype=torch.int64, device="cuda")
    wrong = _native.KtmoeKvBatch.from_buffer_copy(batch._c)
    wrong.rows = rows
    torch.cuda.synchronize()
    status = tb.lib().ktmoe_attn_forward_dev(a._h, cache._c, wrong, x.data_ptr(), xs.data_ptr(), x.data_ptr(), xs.data_ptr(), None)
    assert status == _native.ERR_ARG
    a.forward_dev(cache, batch, x.data_ptr(), xs.data_ptr(), x.data_ptr(), xs.data_ptr())
    ctx.sync()
