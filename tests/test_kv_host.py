"""The KV cache's host side, on any machine: the rotation table, the refusals of the Python classes, and what the
integer definitions amount to (how near they come to softmax attention in real numbers)."""

import math

import numpy as np
import pytest

import kv_reference as R
import tritify_b200 as tb
from tritify_b200 import _native


def test_rope_table():
    t = tb.rope_table(1e4, 8, 50)
    for p in (0, 1, 7, 49):
        for i in range(4):
            a = p * 1e4 ** (-i / 4)
            assert abs(t[p, i, 0] - math.cos(a) * 2 ** 30) <= 0.5 + 2 ** 30 * 1e-14
            assert abs(t[p, i, 1] - math.sin(a) * 2 ** 30) <= 0.5 + 2 ** 30 * 1e-14
    L = tb.lib()
    buf = np.zeros(64, np.int32).ctypes.data_as(_native._i32p)
    for args in ((0.0, 8, 4), (-1.0, 8, 4), (math.nan, 8, 4), (math.inf, 8, 4), (1e4, 7, 4), (1e4, 0, 4), (1e4, 8, 0)):
        assert L.ktmoe_rope_table(*args, buf) == _native.ERR_ARG
    assert L.ktmoe_rope_table(1e4, 8, 4, None) == _native.ERR_ARG
    with pytest.raises(ValueError):
        tb.rope_table(1e4, 3, 4)


def test_quantised_rows_are_within_half_a_step():
    """|value - y s| <= sigma / 2 and a little for the two roundings of a code (2^-52 of at most 127 steps), and sigma
    wastes less than 2^-7 of the range."""
    rng = np.random.default_rng(0)
    for _ in range(200):
        y = rng.integers(-2 ** 28, 2 ** 28, 64) * int(rng.integers(1, 2 ** 20))
        s = math.ldexp(rng.random() + 0.5, int(rng.integers(-60, 10)))
        codes, sigma = R.quantise_row(y, s)
        assert np.abs(codes * sigma - y * s).max() <= sigma * (0.5 + 127 * 2.0 ** -51)
        top = np.abs(y).max() * s
        assert top / 127 <= sigma * (1 + 2.0 ** -51) and sigma < top / 127 * (1 + 2.0 ** -7) * (1 + 2.0 ** -51)


def test_weights_are_near_the_exponential():
    """w_j / 32512 against 2^-(distance): the cubic is within 1.03e-4, the distance's rounding to 2^-10 octaves within
    2^-11 ln 2 = 3.4e-4, the three roundings of 24 bits within 2e-7: 4.4e-4 together; beyond 32 octaves the weight
    rounds to nothing."""
    d = np.concatenate([np.linspace(0, 20, 4001), np.linspace(30, 200, 50)])
    w = R.weights(np.zeros(d.size), np.ones(d.size), 1.0)
    assert (w == 32512).all()
    x = rn = R.rn24(-d)
    w = R.weights(x, np.ones(d.size), 1.0)
    rel = w / 32512 / np.exp2(-(rn.max() - rn)) - 1
    assert np.abs(rel[d <= 31]).max() < 4.4e-4
    assert (np.rint(w[d > 17]) == 0).all()


@pytest.mark.parametrize("dim", [16, 64, 128])
def test_attention_is_near_softmax_attention(dim):
    """The integer attention against softmax attention in float64 of the values that the codes stand for. A weight is
    off by 4.4e-4 of itself (above), by half a unit of 32512 when rounded for L and by half a unit again, of the
    2^E-scaled weight, for O; q's codes add an error of the logits that is left out by quantising q first. With n keys of
    |v| <= vmax: |o - exact| <= vmax (2 * 4.4e-4 + n (0.5 + 1) / (L)) and the code's own half step."""
    rng = np.random.default_rng(dim)
    n, heads = 150, 4
    k8, v8 = rng.integers(-127, 128, (n, dim)), rng.integers(-127, 128, (n, dim))
    k8[:, :4] //= 8
    sk, sv = rng.integers(128, 256, n) / 2.0 ** 14, rng.integers(128, 256, n) / 2.0 ** 12
    q8 = rng.integers(-127, 128, (1, heads, dim))
    q8[..., 0] = 127  # so that q's codes are q itself
    out, out_s = np.zeros((1, heads, dim), np.int64), np.zeros((1, 1, 2), np.int64)
    scale = np.array([2 ** 31, 31 + 9])
    R.attention(q8, scale, [0, 1], [n], lambda b, h: (k8, sk, v8, sv), out, out_s, dim ** -0.5)
    real = out * R.value(out_s[0, 0])
    logits = np.einsum("hd,jd->hj", q8[0] * 2.0 ** -9, k8 * sk[:, None]) * dim ** -0.5
    p = np.exp(logits - logits.max(-1, keepdims=True))
    total = 32512 * p.sum(-1)
    want = p @ (v8 * sv[:, None]) / p.sum(-1, keepdims=True)
    vmax = np.abs(v8 * sv[:, None]).max()
    e_max = 2.0 ** (21 - out_s[0, 0, 1])
    bound = vmax * 2 * 4.4e-4 + (0.5 * n * vmax + 0.5 * n * 127 * e_max) / total + 2.0 ** -20 * e_max
    assert (np.abs(real[0] - want) <= bound[:, None]).all()


class _Ctx:
    device, handle = 0, None


def _cpu(*shape, dtype="int32"):
    import torch

    return torch.zeros(*shape, dtype=getattr(torch, dtype))


def _cache(**kw):
    import torch

    a = dict(n_pages=3, page_tokens=16, n_kv_heads=2, head_dim=32)
    a.update(kw)
    shape = (a["n_pages"], a["n_kv_heads"], a["page_tokens"])
    pools = kw.pop("pools", None) or (_cpu(*shape, a["head_dim"], dtype="int8"), _cpu(*shape, a["head_dim"], dtype="int8"),
                                      _cpu(*shape, dtype="bfloat16"), _cpu(*shape, dtype="bfloat16"))
    a["pools"] = pools
    return tb.KvCache(_Ctx(), **a)


def test_the_classes_refuse_what_does_not_fit():
    ok = _cache()
    for kw in (dict(page_tokens=8), dict(page_tokens=40), dict(page_tokens=256), dict(head_dim=8), dict(head_dim=40),
               dict(head_dim=272), dict(n_kv_heads=0), dict(n_kv_heads=1025), dict(n_pages=0)):
        with pytest.raises(ValueError):
            _cache(**kw)
    for i, bad in ((0, _cpu(3, 2, 16, 48, dtype="int8")), (1, _cpu(3, 2, 16, 32, dtype="int32")),
                   (2, _cpu(3, 2, 16, dtype="float16")), (3, _cpu(3, 2, 15, dtype="bfloat16")),
                   (0, _cpu(3, 2, 32, 16, dtype="int8").transpose(2, 3))):
        pools = [ok.k, ok.v, ok.k_scale, ok.v_scale]
        pools[i] = bad
        with pytest.raises(ValueError):
            tb.KvCache(_Ctx(), 3, 16, 2, 32, pools=tuple(pools))
    b = tb.KvBatch(_cpu(3), _cpu(2), _cpu(2, 4), 7)
    for args in ((_cpu(2), _cpu(2), _cpu(2, 4), 7), (_cpu(3), _cpu(2), _cpu(3, 4), 7), (_cpu(3), _cpu(2), _cpu(8), 7),
                 (_cpu(3, dtype="int64"), _cpu(2), _cpu(2, 4), 7), (_cpu(3), _cpu(2), _cpu(2, 4), -1),
                 (_cpu(3), _cpu(2), _cpu(4, 2).t(), 7), ([0, 1, 2], _cpu(2), _cpu(2, 4), 7)):
        with pytest.raises(ValueError):
            tb.KvBatch(*args)
    for args in ((_cpu(4, 3),), (_cpu(4, 3, 3),), (_cpu(4, 0, 2),), (_cpu(4, 3, 2, dtype="float32"),)):
        with pytest.raises(ValueError):
            tb.Rope(*args)
    kv, s = _cpu(7, 64), _cpu(7, 2, dtype="int64")
    q, o, os_ = _cpu(7, 128), _cpu(7, 128), _cpu(7, 2, 2, dtype="int64")
    for k, v, sc in ((_cpu(6, 64), kv, s), (_cpu(7, 63), kv, s), (kv, _cpu(7, 64, dtype="int64"), s),
                     (kv, _cpu(64, 7).t(), s), (kv, kv, _cpu(6, 2, dtype="int64")), (kv, kv, _cpu(7, 2)),
                     (kv, kv, _cpu(7, 3, dtype="int64")), (_cpu(1, 64).expand(7, 64), kv, s)):
        with pytest.raises(ValueError):
            ok.append(b, k, v, sc)
    with pytest.raises(ValueError):
        ok.read(b, kv, kv)  # float32 outputs
    for kw in (dict(n_heads=3), dict(n_heads=0), dict(n_heads=2), dict(window=-1), dict(sinks=-2), dict(window=1 << 32), dict(sinks=1 << 31),
               dict(out_scale=_cpu(6, 2, 2, dtype="int64")), dict(out_scale=_cpu(7, 4, dtype="int64")),
               dict(out=_cpu(7, 127)), dict(q=_cpu(3, 128))):
        a = dict(q=q, scale=s, out=o, out_scale=os_, n_heads=4)
        a.update(kw)
        with pytest.raises(ValueError):
            ok.attention(b, **a)
    # everything fits but the device
    with pytest.raises(ValueError, match="device"):
        ok.append(b, kv, kv, s)
    with pytest.raises(ValueError, match="device"):
        ok.attention(b, q, s, o, os_, 4)


def test_a_half_refuses_other_devices():
    """Host tensors, or another device's, in a half's batch or cache: refused before anything is launched."""
    half = object.__new__(tb.AttentionHalf)
    half.ctx, half._h = _Ctx(), None
    batch, cache = tb.KvBatch(_cpu(3), _cpu(2), _cpu(2, 4), 7), _cache()
    cache.ctx = half.ctx
    with pytest.raises(ValueError, match="device"):
        half.forward_dev(cache, batch, 16, 16, 16, 16)
    batch.device_index = 0
    with pytest.raises(ValueError, match="device"):
        half.forward_dev(cache, batch, 16, 16, 16, 16)
    batch.device_index, cache.device_index = 1, 0
    with pytest.raises(ValueError, match="device"):
        half.forward_dev(cache, batch, 16, 16, 16, 16)
    with pytest.raises(ValueError, match="context"):
        half.forward_dev(_cache(), batch, 16, 16, 16, 16)


def test_what_long_rows_lose():
    """A weight is rounded to a unit of 1/32512 of the row's largest: over n keys the total is off by n / 2 units at most
    (and 4.4e-4 of itself, above). With scores a few octaves apart that is little at any length; but keys 16 octaves below
    the largest (32512 2^-16 < 1/2) weigh nothing however many they are, up to n 2^-16 of the largest's weight."""
    n = 65536
    rng = np.random.default_rng(2)
    for spread in (0.0, 1.0, 3.0):
        x = R.rn24(spread * rng.standard_normal(n))
        w = np.rint(R.weights(x, np.ones(n), 1.0)).sum()
        exact = 32512 * np.exp2(x - x.max()).sum()
        assert abs(w - exact) <= 4.4e-4 * exact + n / 2
    assert n / 2 < 1e-2 * 32512 * np.exp2(R.rn24(rng.standard_normal(n)) - 4.5).sum()  # one octave's spread: below 1 %
    x = np.full(n, -16.05)
    x[7] = 0.0
    w = np.rint(R.weights(R.rn24(x), np.ones(n), 1.0))
    assert w[7] == 32512 and w.sum() == 32512
    assert 0.9 < np.exp2(x).sum() - 1 <= n * 2.0 ** -16
