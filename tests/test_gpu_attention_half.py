"""The attention half of a decoder block, y = add(x, o(attention(q, k, v))) with q, k, v the linears of rms_norm(x), and
a stack of whole blocks, on the B200 against the oracle's RmsNorm, quantiser, linear and add with the plain 64-bit
restatement of the cache and the attention (tests/kv_reference.py) between them: integers, tolerance 0."""

import dataclasses
import os
import sys

import numpy as np
import pytest

import kv_reference as R
import tritify_b200 as tb
from tritify_b200 import _native

pytestmark = pytest.mark.gpu
HERE = os.path.dirname(os.path.abspath(__file__))
sys.path.insert(0, HERE)

import cases  # noqa: E402
import test_gpu_block as tgb  # noqa: E402

EPS = 1e-6
L28 = 1 << 28


def requant_rows(oracle, v, den):
    return np.array([oracle.requant_dyn(int(x), L28, int(den)) for x in np.asarray(v).ravel()], np.int32).reshape(np.shape(v))


def linear_row(oracle, x, xs, codes, ws):
    """QuantLinear::forward_int of one row: (int32 codes, scale)."""
    xmax = int(np.abs(x.astype(np.int64)).max())
    if xmax == 0:
        return np.zeros(codes.shape[0], np.int32), (0, 0)
    q = oracle.quant_to(x, xmax)
    acc = oracle.linear(q, codes.ravel(), 1, codes.shape[0], codes.shape[1])
    sq = oracle.mul(oracle.from_ratio(xmax, tb.WLEVELS), xs)
    ymax = int(np.abs(acc).max())
    c = oracle.mul(sq, ws)
    if ymax == 0 or c[0] == 0:
        return np.zeros(codes.shape[0], np.int32), (0, 0)
    return requant_rows(oracle, acc, ymax), oracle.mul(oracle.from_ratio(ymax, L28), c)


def merge(oracle, rows, scales):
    """Rows at their own scales into one tensor at one scale (the last largest; one row stays as it is)."""
    if len(rows) == 1:
        return rows, scales[0]
    common = (0, 0)
    for s in scales:
        if oracle.ge(s, common):
            common = s
    if common[0] == 0:
        return np.zeros_like(rows), (0, 0)
    inv = oracle.recip(common)
    f = [oracle.mul(s, inv) for s in scales]
    v = np.array([[oracle.apply(f[i], int(x)) for x in r] for i, r in enumerate(rows)], np.int64)
    gmax = int(np.abs(v).max())
    if gmax == 0:
        return np.zeros_like(rows), (0, 0)
    return requant_rows(oracle, v, gmax), oracle.mul(oracle.from_ratio(gmax, L28), common)


class Half:
    """One attention half with its weights, its cache on the device and a host copy of what the cache holds."""

    def __init__(self, ctx, d, heads, hk, dim, page, n_pages, seed, rope=None, window=0, sinks=0):
        def lin(name, out, k, s):
            return tb.QuantLinear.from_weights(name, tb.synth_normal(seed + s, 0.05, out * k), out, k)

        self.d, self.heads, self.hk, self.dim, self.page = d, heads, hk, dim, page
        self.q, self.k, self.v = lin("q", heads * dim, d, 1), lin("k", hk * dim, d, 2), lin("v", hk * dim, d, 3)
        self.out = lin("o", d, heads * dim, 4)
        self.norm_w = tb.synth_normal(seed + 5, 1.0, d)
        nq = tb.QuantLinear.from_weights("norm", self.norm_w, 1, d)
        self.dev = tb.AttentionHalf(ctx, d, heads, hk, dim)
        self.dev.set_qkv(self.q, self.k, self.v)
        self.dev.set_out(self.out)
        self.dev.set_norm(nq.w_codes, nq.w_scale, tb.scale_from_f64(EPS))
        self.rope, self.window, self.sinks = rope, window, sinks
        self.table = None
        if rope:
            self.dev.set_rope(*rope)
            self.table = tb.rope_table(rope[0], rope[1], rope[2])
        self.dev.set_mask(window, sinks)
        self.cache = tb.KvCache(ctx, n_pages, page, hk, dim)
        self.held = {}  # (sequence, position, head) -> k, sigma, v, sigma

    def expect(self, oracle, x, xs, begin, kv_len):
        rows = x.shape[0]
        xn, xns, _, _, _ = oracle.rmsnorm(self.norm_w, EPS, x, xs)
        xn = xn.reshape(rows, self.d)
        parts = [[linear_row(oracle, xn[t], xns, w.w_codes, (w.w_scale.mant, w.w_scale.shift)) for t in range(rows)]
                 for w in (self.q, self.k, self.v)]
        codes = [np.stack([r[0] for r in p]) for p in parts]
        scales = [np.array([r[1] for r in p], np.int64) for p in parts]

        def write(which, b, pos, h, c, sigma):
            self.held.setdefault((b, pos, h), {})[which] = (c, sigma)

        inter = bool(self.rope and len(self.rope) > 3 and self.rope[3])
        R.append(codes[1].reshape(rows, self.hk, self.dim), codes[2].reshape(rows, self.hk, self.dim), scales[1], begin,
                 kv_len, write, self.table, inter, scales[2])

        def keys(b, h):
            got = [self.held[(b, p, h)] for p in range(kv_len[b])]
            return (np.stack([g["k"][0] for g in got]), np.array([g["k"][1] for g in got]),
                    np.stack([g["v"][0] for g in got]), np.array([g["v"][1] for g in got]))

        o = np.zeros((rows, self.heads, self.dim), np.int64)
        os_ = np.zeros((rows, self.hk, 2), np.int64)
        R.attention(codes[0].reshape(rows, self.heads, self.dim), scales[0], begin, kv_len, keys, o, os_,
                    self.dim ** -0.5, self.window, self.sinks, self.table, inter)
        groups, gs = merge(oracle, o.reshape(rows * self.hk, -1).astype(np.int32), [tuple(map(int, s)) for s in os_.reshape(-1, 2)])
        outs = [linear_row(oracle, r, gs, self.out.w_codes, (self.out.w_scale.mant, self.out.w_scale.shift))
                for r in groups.reshape(rows, -1)]
        m, ms = merge(oracle, np.stack([r[0] for r in outs]), [r[1] for r in outs])
        y, ys = oracle.add(x.reshape(-1), xs, m.reshape(-1), ms)
        return y.reshape(rows, self.d), ys


def batch_of(lens, table, rows_behind=0):
    """lens: (new, total) of each sequence; table: [n][max_pages]."""
    import torch

    i32 = lambda a: torch.tensor(a, dtype=torch.int32, device="cuda")
    begin = [0]
    for new, _ in lens:
        begin.append(begin[-1] + new)
    kv = [t for _, t in lens]
    return begin, kv, tb.KvBatch(i32(begin), i32(kv), i32(table), begin[-1] + rows_behind)


def run_half(ctx, half, x, xs, batch):
    import torch

    xd = torch.from_numpy(np.ascontiguousarray(x)).cuda()
    s = torch.tensor([xs[0], xs[1] & 0xFFFFFFFF], dtype=torch.int64, device="cuda")
    yd, ys = torch.empty_like(xd), torch.zeros(2, dtype=torch.int64, device="cuda")
    torch.cuda.synchronize()
    half.dev.forward_dev(half.cache, batch, xd.data_ptr(), s.data_ptr(), yd.data_ptr(), ys.data_ptr())
    ctx.sync()
    a, b = ys.cpu().tolist()
    b &= 0xFFFFFFFF
    return yd.cpu().numpy(), (a, b - (1 << 32) if b >= 1 << 31 else b)


def x_of(rows, d, seed):
    t = tb.IntTensor.from_reals(tb.synth_normal(seed, 1.0, rows * d))
    return t.data.reshape(rows, d), (t.scale.mant, t.scale.shift)


@pytest.mark.parametrize("shape", [(64, 4, 2, 16, 16, (1e4, 16, 64)), (96, 6, 1, 32, 32, (1e4, 16, 64, True)),
                                   (40, 2, 2, 48, 16, None)])
@pytest.mark.parametrize("window,sinks", [(0, 0), (5, 2)])
def test_half_equals_the_restatement(ctx, oracle, shape, window, sinks):
    """Prompts, then steps of one token and a chunk, of two sequences; a row behind the batch gets no attention."""
    d, heads, hk, dim, page, rope = shape
    half = Half(ctx, d, heads, hk, dim, page, 12, 900 + d, rope, window, sinks)
    table = [[3, 0, 7], [5, 9, 1]]
    kv = [0, 0]
    for step, new in enumerate([(9, 4), (1, 1), (1, 0), (3, 6)]):
        kv = [a + b for a, b in zip(kv, new)]
        begin, lens, batch = batch_of(list(zip(new, kv)), table, rows_behind=step % 2)
        x, xs = x_of(batch.rows, d, 50 + step)
        want, ws = half.expect(oracle, x, xs, begin, lens)
        got, gs = run_half(ctx, half, x, xs, batch)
        assert gs == ws
        assert (got == want).all()


def test_one_row_alone(ctx, oracle):
    half = Half(ctx, 32, 1, 1, 16, 16, 3, 77)
    begin, lens, batch = batch_of([(1, 1)], [[2]])
    x, xs = x_of(1, 32, 3)
    want, ws = half.expect(oracle, x, xs, begin, lens)
    got, gs = run_half(ctx, half, x, xs, batch)
    assert gs == ws and (got == want).all()


@pytest.mark.parametrize("name", ["tiny_sigmoid_shared", "small_shared_softmax"])
def test_stack_of_whole_blocks(ctx, oracle, name):
    """Two blocks, attention half then FFN half, over two calls: a prompt and a chunk behind it."""
    base = cases.CASES[name]
    d, T = base.d, base.T
    layer_cases = [dataclasses.replace(base, name=f"{base.name}_block{i}", wseed=base.wseed + 100 * i) for i in range(2)]
    held = [cases.build_layer(c, ctx) for c in layer_cases]
    for m, c in zip(held, layer_cases):
        tgb.set_norm(m.device_layer(), c)
    pages = 2 * (-(-2 * T // 16)) + 2
    halves = [Half(ctx, d, 4, 2, 16, 16, pages, 300 + i, (1e4, 16, 4 * T)) for i in range(2)]
    stack = tb.MoeStack([m.device_layer() for m in held], [h.dev for h in halves], [h.cache for h in halves])
    table = [list(range(pages - 1, 0, -1))]
    total = 0
    for step in range(2):
        total += T
        begin, lens, batch = batch_of([(T, total)], table)
        x = tb.IntTensor.from_reals(tb.synth_normal(60 + step, 1.0, T * d).reshape(T, d))
        xi, xs = x.data.reshape(T, d), (x.scale.mant, x.scale.shift)
        for c, h in zip(layer_cases, halves):
            xi, xs = h.expect(oracle, xi, xs, begin, lens)
            o = cases.build_oracle(c, oracle)
            xn, xns, _, _, _ = oracle.rmsnorm(tgb.norm_weight(c), tgb.EPS, xi, xs)
            moe, ms = o.forward(xn.reshape(T, d), xns)
            y, xs = oracle.add(xi.reshape(-1), xs, moe.reshape(-1), ms)
            xi = y.reshape(T, d)
        got = stack.forward(x, batch)
        assert (got.scale.mant, got.scale.shift) == xs
        assert (got.data.reshape(T, d) == xi).all()
    with pytest.raises(ValueError):
        stack.forward(x)
    with pytest.raises(ValueError):
        tb.MoeStack(stack.layers, stack.attention, [halves[0].cache] * 2)
    with pytest.raises(ValueError):
        tb.MoeStack(stack.layers, stack.attention)


def test_refusals(ctx):
    with pytest.raises(tb.KtmoeError):
        tb.AttentionHalf(ctx, 64, 3, 2, 16)
    with pytest.raises(tb.KtmoeError):
        tb.AttentionHalf(ctx, 64, 2, 2, 24)
    a = tb.AttentionHalf(ctx, 64, 2, 1, 16)
    cache = tb.KvCache(ctx, 2, 16, 1, 16)
    _, _, batch = batch_of([(1, 1)], [[0]])
    with pytest.raises(tb.KtmoeError) as e:  # no weights yet
        a.forward_dev(cache, batch, 16, 16, 16, 16)
    assert e.value.status == _native.ERR_STATE
    lin = lambda o, k: tb.QuantLinear.from_weights("w", tb.synth_normal(1, 1.0, o * k), o, k)
    with pytest.raises(ValueError):
        a.set_qkv(lin(32, 64), lin(32, 64), lin(16, 64))
    a.set_qkv(lin(32, 64), lin(16, 64), lin(16, 64))
    a.set_out(lin(64, 32))
    with pytest.raises(ValueError):
        a.set_norm(np.ones(63, np.int32), tb.Scale(1, 0), tb.Scale(0, 0))
    a.set_norm(np.ones(64, np.int32), tb.Scale(1, 0), tb.Scale(0, 0))
    for kw in (dict(theta=1e4, rot_dim=18, positions=4), dict(theta=1e4, rot_dim=3, positions=4),
               dict(theta=-1.0, rot_dim=16, positions=4), dict(theta=1e4, rot_dim=16, positions=-1)):
        with pytest.raises(tb.KtmoeError):
            a.set_rope(**kw)
    with pytest.raises(tb.KtmoeError):
        a.set_mask(window=-1)
    with pytest.raises(tb.KtmoeError):
        a.set_mask(softmax_scale=float("nan"))
    with pytest.raises(ValueError):
        a.set_mask(window=1 << 32)
    with pytest.raises(tb.KtmoeError) as e:  # another head size
        a.forward_dev(tb.KvCache(ctx, 2, 16, 1, 32), batch, 16, 16, 16, 16)
    assert e.value.status == _native.ERR_ARG
    bad = np.full((32, 64), tb.WLEVELS + 1, np.int32)
    with pytest.raises(tb.KtmoeError) as e:
        a.set_qkv(tb.QuantLinear("q", bad, tb.Scale(1, 0), 32, 64), lin(16, 64), lin(16, 64))
    assert e.value.status == _native.ERR_RANGE


def test_a_context_closed_first(ctx):
    """The half ends with its context; what is called on it afterwards is refused."""
    own = tb.Context(0)
    a, b = tb.AttentionHalf(own, 64, 2, 1, 16), tb.AttentionHalf(own, 64, 2, 1, 16)
    del b
    own.close()
    with pytest.raises(tb.KtmoeError):
        a.set_mask(window=3)
    del a
    own.close()
    ctx.sync()


def test_captured_forwards(ctx, oracle):
    """A step captured into a graph, the scratch outgrown by a longer batch and the rotation changed after that, and the
    graph replayed: what the capture gave. A capture that would grow the scratch is refused and the stream's capture
    goes on."""
    import torch

    half = Half(ctx, 64, 4, 2, 16, 16, 12, 700, (1e4, 16, 64))
    _, _, prompt = batch_of([(9, 9)], [[1, 2, 3, 4]])
    run_half(ctx, half, *x_of(9, 64, 1), prompt)
    _, _, one = batch_of([(1, 10)], [[1, 2, 3, 4]])
    x, xs = x_of(1, 64, 2)
    want = run_half(ctx, half, x, xs, one)  # writes position 9, as each replay does
    xd = torch.from_numpy(np.ascontiguousarray(x)).cuda()
    s = torch.tensor([xs[0], xs[1] & 0xFFFFFFFF], dtype=torch.int64, device="cuda")
    yd, ys = torch.empty_like(xd), torch.zeros(2, dtype=torch.int64, device="cuda")
    _, _, long = batch_of([(40, 50)], [[1, 2, 3, 4]])
    xl = torch.zeros(40, 64, dtype=torch.int32, device="cuda")
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        at = torch.cuda.current_stream().cuda_stream
        half.dev.forward_dev(half.cache, one, xd.data_ptr(), s.data_ptr(), yd.data_ptr(), ys.data_ptr(), at)
        with pytest.raises(tb.KtmoeError) as e:
            half.dev.forward_dev(half.cache, long, xl.data_ptr(), s.data_ptr(), xl.data_ptr(), ys.data_ptr(), at)
        assert e.value.status == _native.ERR_STATE
    _, _, other = batch_of([(40, 40)], [[6, 7, 8, 9]])
    run_half(ctx, half, *x_of(40, 64, 3), other)
    half.dev.set_rope(5e3, 16, 4096)
    for _ in range(2):
        yd.zero_()
        graph.replay()
        torch.cuda.synchronize()
        ctx.sync()
        assert (yd.cpu().numpy() == want[0]).all()
        a, b = ys.cpu().tolist()
        assert (a, (b & 0xFFFFFFFF) - (1 << 32) if b & 1 << 31 else b & 0xFFFFFFFF) == want[1]
