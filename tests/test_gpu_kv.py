"""The paged KV cache and the attention over it on a B200: every integer against the plain 64-bit restatement
(tests/kv_reference.py), at the sizes, masks, strides and values where a kernel can go wrong. All arithmetic is exact by
definition, so the tolerance is zero."""

import ctypes
import math

import numpy as np
import pytest

import kv_reference as R
import tritify_b200 as tb
from tritify_b200 import _native

pytestmark = pytest.mark.gpu


def _torch():
    import torch

    return torch


class Setup:
    """A batch of sequences over a cache whose pages are dealt out at random, with a host copy of the pools."""

    def __init__(self, ctx, lens, heads, kv_heads, dim, page, seed=0, spare=2, rows_before=0, rows_behind=0, fill=True,
                 fill_scale=1.0):
        torch = _torch()
        self.ctx, self.lens, self.heads, self.hk, self.dim, self.page = ctx, lens, heads, kv_heads, dim, page
        self.rng = np.random.default_rng(seed)
        need = [max(0, -(-kv // page)) for _, kv in lens]
        self.max_pages = max(need + [1])
        n_pages = sum(need) + spare
        perm = self.rng.permutation(n_pages).astype(np.int32)
        self.table = np.zeros((len(lens), self.max_pages), np.int32)
        at = 0
        for b, k in enumerate(need):
            self.table[b, :k] = perm[at:at + k]
            at += k
        self.begin = [rows_before]
        for new, _ in lens:
            self.begin.append(self.begin[-1] + new)
        self.rows = self.begin[-1] + rows_behind
        self.kv_len = [kv for _, kv in lens]
        self.cache = tb.KvCache(ctx, n_pages, page, kv_heads, dim)
        shape = (n_pages, kv_heads, page)
        self.pool = {}
        for n in "kv":
            self.pool[n] = self.rng.integers(-127, 128, (*shape, dim)).astype(np.int8) if fill else np.zeros((*shape, dim), np.int8)
            sg = np.exp2(self.rng.integers(-9, -5, shape)) * self.rng.integers(128, 256, shape) / 128 * fill_scale
            self.pool[n + "s"] = sg.astype(np.float64)
        self.push()
        i32 = lambda a: torch.tensor(np.asarray(a, np.int32), device="cuda")
        self.batch = tb.KvBatch(i32(self.begin), i32(self.kv_len), i32(self.table).reshape(len(lens), -1), self.rows)

    def push(self):
        torch = _torch()
        for n, t in (("k", self.cache.k), ("v", self.cache.v)):
            t.copy_(torch.from_numpy(self.pool[n]))
        for n, t in (("ks", self.cache.k_scale), ("vs", self.cache.v_scale)):
            t.copy_(torch.from_numpy(self.pool[n]).to(torch.bfloat16))

    def place(self, b, pos):
        return self.table[b, pos // self.page], pos % self.page

    def keys(self, b, h):
        n = max(0, self.kv_len[b])
        pages, place = self.table[b, np.arange(n) // self.page], np.arange(n) % self.page
        return tuple(self.pool[x][pages, h, place] for x in ("k", "ks", "v", "vs"))

    def write(self, which, b, pos, h, codes, sigma):
        page, place = self.place(b, pos)
        self.pool[which][page, h, place] = codes
        self.pool[which + "s"][page, h, place] = sigma

    def codes(self, width, big=2 ** 28):
        return self.rng.integers(-big, big + 1, (self.rows, width)).astype(np.int32)

    def scales(self, lo=28, hi=36):
        mant = self.rng.integers(2 ** 31, 2 ** 32, self.rows)
        return np.stack([mant, self.rng.integers(lo, hi, self.rows) + 31], -1).astype(np.int64)

    def attend(self, q, scale, table=None, interleaved=False, window=0, sinks=0, softmax_scale=None, stream=None):
        """(codes, scales) from the GPU and from the restatement, both on outputs that held 77 before. Enough rows a
        sequence go to the tile kernel once the blocks fill the GPU: those run a second time with as many copies of
        all heads (its launches are two, the few-row kernel's one)."""
        torch = _torch()
        rope = None if table is None else tb.Rope(torch.from_numpy(table).cuda(), interleaved)
        sd = torch.from_numpy(scale).cuda()
        qd = torch.from_numpy(q).cuda() if isinstance(q, np.ndarray) else q

        def run(cache, qd, copies):
            out = torch.full((self.rows, copies * self.heads * self.dim), 77, dtype=torch.int32, device="cuda")
            os_ = torch.full((self.rows, copies * self.hk, 2), 77, dtype=torch.int64, device="cuda")
            before = self.ctx.launch_count()
            cache.attention(self.batch, qd, sd, out, os_, copies * self.heads, rope=rope, softmax_scale=softmax_scale,
                            window=window, sinks=sinks, stream=stream)
            launches = self.ctx.launch_count() - before
            self.ctx.sync()
            torch.cuda.synchronize()
            return out.reshape(self.rows, copies, -1), os_.reshape(self.rows, copies, -1), launches

        out, os_, _ = run(self.cache, qd, 1)
        if (self.begin[-1] - self.begin[0]) * (self.heads // self.hk) > 32 * len(self.lens):
            copies = -(-148 // self.hk)
            cache = tb.KvCache(self.ctx, self.cache.n_pages, self.page, copies * self.hk, self.dim, pools=[
                t.repeat(1, copies, *[1] * (t.dim() - 2)) for t in (self.cache.k, self.cache.v, self.cache.k_scale, self.cache.v_scale)])
            skew = 0 if qd.is_contiguous() else 1  # unaligned rows stay unaligned
            wide = torch.zeros(self.rows, copies * qd.shape[1] + skew, dtype=torch.int32, device="cuda")[:, skew:]
            wide.copy_(qd.repeat(1, copies))
            torch.cuda.synchronize()
            o, s, launches = run(cache, wide, copies)
            assert launches == 2
            assert (o == out).all() and (s == os_).all(), "the two kernels differ"
        want = np.full((self.rows, self.heads, self.dim), 77, np.int64)
        want_s = np.full((self.rows, self.hk, 2), 77, np.int64)
        R.attention(q.reshape(self.rows, self.heads, self.dim) if isinstance(q, np.ndarray) else
                    q.cpu().numpy().reshape(self.rows, self.heads, self.dim), scale, self.begin, self.kv_len, self.keys,
                    want, want_s, self.dim ** -0.5 if softmax_scale is None else softmax_scale, window, sinks, table,
                    interleaved)
        want_s[..., 1] &= 0xFFFFFFFF
        return out.cpu().numpy().reshape(want.shape), os_.cpu().numpy().reshape(want_s.shape), want, want_s

    def check(self, *a, **k):
        got, got_s, want, want_s = self.attend(*a, **k)
        bad = np.argwhere(got != want)
        assert bad.size == 0, f"{len(bad)} of {want.size} codes differ, first at {bad[0]}: {got[tuple(bad[0])]} != {want[tuple(bad[0])]}"
        assert (got_s == want_s).all()


# ── writing and reading back ──

CACHE = [  # lens (new, total), KV heads, dim, page, rotation (rot_dim, interleaved) or None
    ([(1, 1)], 1, 16, 16, None),
    ([(1, 100), (1, 1), (1, 64)], 8, 128, 64, (128, False)),
    ([(33, 40), (0, 7), (5, 5), (17, 300)], 3, 80, 16, (40, True)),
    ([(70, 70)], 2, 256, 32, (256, True)),
    ([(9, 500), (130, 130)], 5, 96, 128, (2, False)),
    ([(3, 2), (4, 0), (2, 90)], 2, 64, 16, (64, False)),  # positions below zero: no place
]


@pytest.mark.parametrize("case", CACHE, ids=[str(i) for i in range(len(CACHE))])
def test_append_and_read(ctx, case):
    torch = _torch()
    lens, hk, dim, page, rot = case
    s = Setup(ctx, lens, hk, hk, dim, page, seed=dim, rows_before=2, rows_behind=3)
    k, v, scale = s.codes(hk * dim), s.codes(hk * dim), s.scales()
    k[s.begin[0], :dim] = 0  # a row of zeros
    k[-4, dim - 16:dim] = -2 ** 31
    v[s.begin[0], :3] = [2 ** 31 - 1, -2 ** 31, 1]
    scale[-4] = (0, 5)
    table = None if rot is None else tb.rope_table(1e4, rot[0], max(kv for _, kv in lens) + 1)
    rope = None if rot is None else tb.Rope(torch.from_numpy(table).cuda(), rot[1])
    v_scale = s.scales(20, 50) if dim % 32 == 0 else None
    R.append(k.reshape(s.rows, hk, dim), v.reshape(s.rows, hk, dim), scale, s.begin, s.kv_len, s.write, table,
             rot is not None and rot[1], v_scale)
    s.cache.append(s.batch, torch.from_numpy(k).cuda(), torch.from_numpy(v).cuda(), torch.from_numpy(scale).cuda(), rope,
                   v_scale=None if v_scale is None else torch.from_numpy(v_scale).cuda())
    ko, vo = (torch.full((s.rows, hk * dim), -5.0, device="cuda") for _ in range(2))
    s.cache.read(s.batch, ko, vo)
    ctx.sync()
    torch.cuda.synchronize()
    # the whole pools: what was written, and everything else left as it was
    for n, t in (("k", s.cache.k), ("v", s.cache.v), ("ks", s.cache.k_scale), ("vs", s.cache.v_scale)):
        assert (t.double().cpu().numpy() == s.pool[n].astype(np.float64)).all(), n
    for n, o in (("k", ko), ("v", vo)):
        want = np.full((s.rows, hk, dim), -5.0)
        for t, b, pos in R.rows_of(s.begin, s.kv_len):
            if pos >= 0:
                page_, place = s.place(b, pos)
                want[t] = s.pool[n][page_, :, place].astype(np.float64) * s.pool[n + "s"][page_, :, place][:, None]
        assert (o.double().cpu().numpy() == want.reshape(s.rows, -1)).all(), n


def test_append_takes_strided_and_unaligned_rows_and_one_scale(ctx):
    torch = _torch()
    hk, dim = 2, 48
    s = Setup(ctx, [(6, 9), (1, 40)], hk, hk, dim, 16)
    both = np.random.default_rng(3).integers(-2 ** 28, 2 ** 28, (s.rows, 2 * hk * dim + 5)).astype(np.int32)
    d = torch.from_numpy(both).cuda()
    scale = np.array([3 * 2 ** 30, 60], np.int64)
    k, v = both[:, 1:1 + hk * dim], both[:, 3 + hk * dim:3 + 2 * hk * dim]
    R.append(k.reshape(s.rows, hk, dim), v.reshape(s.rows, hk, dim), scale, s.begin, s.kv_len, s.write)
    s.cache.append(s.batch, d[:, 1:1 + hk * dim], d[:, 3 + hk * dim:3 + 2 * hk * dim], torch.from_numpy(scale).cuda())
    wide = [torch.zeros(s.rows, hk * dim + 3, device="cuda") for _ in range(2)]
    s.cache.read(s.batch, wide[0][:, 1:-2], wide[1][:, 2:-1])
    ctx.sync()
    torch.cuda.synchronize()
    for n, t in (("k", s.cache.k), ("v", s.cache.v), ("ks", s.cache.k_scale), ("vs", s.cache.v_scale)):
        assert (t.double().cpu().numpy() == s.pool[n].astype(np.float64)).all(), n
    assert (wide[0][:, 0] == 0).all() and (wide[0][:, -2:] == 0).all()
    page_, place = s.place(0, 3)
    assert (wide[0][0, 1:-2].cpu().numpy() == (s.pool["k"][page_, :, place] * s.pool["ks"][page_, :, place][:, None]).ravel()).all()


@pytest.mark.parametrize("shift", [-300, -64, 0, 27, 90, 200, 900, 2 ** 31 - 1, -2 ** 31])
def test_append_at_extreme_scales(ctx, shift):
    """Scales far outside sigma's range: sigma stops at 2^-64 and 2^63 and the codes at 0 and 127."""
    torch = _torch()
    s = Setup(ctx, [(4, 4)], 1, 1, 16, 16)
    k, v = s.codes(16), s.codes(16)
    words = np.array([[2 ** 31 + 7, shift & 0xFFFFFFFF]] * s.rows, np.int64)
    host = words.copy()
    host[:, 1] = max(-900, min(2000, shift))  # beyond these the double is infinite or zero either way
    with np.errstate(over="ignore", invalid="ignore"):
        R.append(k.reshape(4, 1, 16), v.reshape(4, 1, 16), host, s.begin, s.kv_len, s.write)
    s.cache.append(s.batch, torch.from_numpy(k).cuda(), torch.from_numpy(v).cuda(), torch.from_numpy(words).cuda())
    ctx.sync()
    torch.cuda.synchronize()
    for n, t in (("k", s.cache.k), ("v", s.cache.v), ("ks", s.cache.k_scale), ("vs", s.cache.v_scale)):
        assert (t.double().cpu().numpy() == s.pool[n].astype(np.float64)).all(), n


# ── attention ──

ATTEND = [  # lens, query heads, KV heads, dim, page, rotation, window, sinks
    ([(1, 1)], 1, 1, 16, 16, None, 0, 0),
    ([(1, 1), (1, 2), (1, 15), (1, 16), (1, 17)], 2, 1, 64, 16, None, 0, 0),
    ([(1, 127), (1, 128), (1, 129), (1, 255), (1, 257)], 8, 2, 128, 64, (128, False), 0, 0),
    ([(1, 700), (1, 63)], 12, 1, 128, 32, (64, True), 0, 0),
    ([(1, 333)], 7, 1, 80, 16, None, 0, 0),
    ([(1, 200)], 40, 1, 96, 128, None, 0, 0),  # more query heads than one block takes
    ([(1, 90)], 65, 1, 32, 64, None, 0, 0),
    ([(2, 130), (3, 3), (0, 50), (5, 400)], 4, 2, 64, 64, (32, False), 0, 0),
    ([(16, 300)], 8, 8, 128, 64, None, 0, 0),
    ([(17, 17), (31, 145)], 6, 2, 112, 16, (112, True), 0, 0),
    ([(127, 127)], 3, 1, 128, 64, None, 0, 0),
    ([(129, 260)], 2, 2, 128, 128, None, 0, 0),
    ([(64, 64), (65, 190)], 5, 1, 256, 32, (256, False), 0, 0),
    ([(130, 130)], 2, 1, 48, 16, None, 0, 0),
    ([(4, 2), (3, 0), (1, 0), (2, 30)], 4, 2, 64, 16, None, 0, 0),  # rows that see nothing
    # windows: of one key, inside a page, a whole number of pages, wider than the sequence; sinks of all kinds
    ([(1, 300), (1, 5)], 4, 1, 128, 64, None, 1, 0),
    ([(1, 300), (1, 90)], 4, 1, 128, 64, None, 77, 3),
    ([(1, 500)], 4, 2, 64, 16, None, 64, 200),
    ([(40, 300), (9, 9)], 4, 2, 64, 32, (64, False), 33, 5),
    ([(150, 400)], 2, 1, 128, 64, None, 100, 1),
    ([(150, 400)], 2, 1, 128, 64, None, 100, 130),
    ([(150, 150)], 4, 1, 32, 16, None, 5, 0),
    ([(20, 600)], 2, 1, 128, 128, None, 1000, 4),
    ([(300, 700)], 1, 1, 128, 64, None, 128, 0),
]


@pytest.mark.parametrize("case", ATTEND, ids=[str(i) for i in range(len(ATTEND))])
def test_attention(ctx, case):
    lens, heads, hk, dim, page, rot, window, sinks = case
    s = Setup(ctx, lens, heads, hk, dim, page, seed=heads * dim, rows_before=1, rows_behind=2)
    table = None if rot is None else tb.rope_table(1e4, rot[0], max(kv for _, kv in lens) + 1)
    s.check(s.codes(heads * dim), s.scales(), table, rot is not None and rot[1], window, sinks)


@pytest.mark.parametrize("new", [1, 3, 40])
@pytest.mark.parametrize("kind", ["zero_q", "zero_v", "zero_k", "equal", "far", "tiny", "one_scale", "extreme", "softmax"])
def test_attention_of_unusual_values(ctx, kind, new):
    s = Setup(ctx, [(new, 200), (new, 64)], 4, 2, 64, 32, seed=new)
    q, scale, soft = s.codes(s.heads * s.dim), s.scales(), None
    if kind == "zero_q":
        q[:] = 0
    elif kind == "zero_v":
        s.pool["v"][:] = 0
    elif kind == "zero_k":
        s.pool["k"][:] = 0
    elif kind == "equal":  # one key many times over
        s.pool["k"][:] = s.pool["k"][0, 0, 0]
        s.pool["ks"][:] = 2.0 ** -7
    elif kind == "far":  # distances beyond any weight, and products beyond binary32
        s.pool["ks"] *= 2.0 ** 60
        scale[:, 1] -= 90
    elif kind == "tiny":
        s.pool["ks"] *= 2.0 ** -55
        s.pool["vs"] *= 2.0 ** -55
        scale[:, 1] += 90
    elif kind == "one_scale":
        scale = scale[0]
    elif kind == "extreme":
        q[:, ::3] = -2 ** 31
        q[:, 1::3] = 2 ** 31 - 1
        scale[:, 0] = 0  # the first row's scale is zero
        scale[1:, 0] = 2 ** 32 - 1
        s.pool["k"][:] = np.where(s.pool["k"] >= 0, 127, -127)
        s.pool["v"][:] = 127
        s.pool["vs"] *= np.exp2(s.rng.integers(-30, 30, s.pool["vs"].shape))
    elif kind == "softmax":
        soft = 3.7
    s.push()
    s.check(q, scale, softmax_scale=soft)


def test_attention_largest_sums(ctx):
    """All codes at their ends, the widest head: dot products of 127 * 127 * 256 and every weight 32512."""
    s = Setup(ctx, [(1, 300), (40, 300)], 4, 1, 256, 64)
    s.pool["k"][:], s.pool["v"][:], s.pool["ks"][:], s.pool["vs"][:] = 127, -127, 1.0, 255 / 128
    s.push()
    q = np.full((s.rows, 4 * 256), 2 ** 28, np.int32)
    s.check(q, s.scales())


def test_attention_beyond_131072_keys(ctx):
    """More keys than 32-bit sums of 8-bit products hold."""
    n = 140001
    s = Setup(ctx, [(1, n)], 2, 1, 16, 128)
    s.pool["k"][:], s.pool["v"][:], s.pool["ks"][:], s.pool["vs"][:] = 1, 127, 1.0, 255 / 256
    s.push()
    s.check(s.codes(2 * 16), s.scales())
    s2 = Setup(ctx, [(40, n)], 1, 1, 16, 128)
    s2.pool["k"][:], s2.pool["v"][:], s2.pool["ks"][:], s2.pool["vs"][:] = 1, -127, 1.0, 255 / 256
    s2.push()
    s2.check(s2.codes(16), s2.scales())


def test_attention_of_millions_of_keys(ctx):
    """So many keys that each block of a decode cluster takes its 32-bit sums out on the way."""
    n = 2300000
    s = Setup(ctx, [(1, n)], 1, 1, 16, 128)
    s.pool["k"][:], s.pool["v"][:], s.pool["ks"][:], s.pool["vs"][:] = 1, 127, 1.0, 255 / 256
    s.push()
    s.check(s.codes(16), s.scales())


@pytest.mark.parametrize("hk", [2, 150])
def test_attention_takes_strided_and_unaligned_queries(ctx, hk):
    torch = _torch()
    s = Setup(ctx, [(5, 90), (30, 200)], 2 * hk, hk, 48, 16)
    n = 2 * hk * 48
    wide = torch.from_numpy(s.rng.integers(-2 ** 28, 2 ** 28, (s.rows, n + 3)).astype(np.int32)).cuda()
    if hk == 2:
        s.check(wide[:, 1:-2], s.scales())
    scale = torch.from_numpy(s.scales()).cuda()
    outs = []
    for pad in (0, 7):  # the output's rows may be strided too
        o = torch.zeros(s.rows, n + pad, dtype=torch.int32, device="cuda")
        os_ = torch.zeros(s.rows, hk, 2, dtype=torch.int64, device="cuda")
        s.cache.attention(s.batch, wide[:, 1:-2], scale, o[:, pad // 2:pad // 2 + n], os_, 2 * hk)
        outs.append((o[:, pad // 2:pad // 2 + n].cpu(), os_.cpu()))
        assert (o[:, :pad // 2] == 0).all() and (o[:, pad // 2 + n:] == 0).all()
    ctx.sync()
    assert torch.equal(outs[0][0], outs[1][0]) and torch.equal(outs[0][1], outs[1][1])


@pytest.mark.parametrize("window,sinks", [(0, 0), (50, 3)])
@pytest.mark.parametrize("hk", [2, 60])  # 60: the long chunks go to the tile kernel
def test_chunks_equal_the_whole_prompt(ctx, hk, window, sinks):
    """A prompt written and attended in chunks of any size, down to single tokens, gives the bits of one call."""
    torch = _torch()
    n, heads, dim, page = 200, 3 * hk, 64, 16
    rng = np.random.default_rng(8)
    kv = torch.from_numpy(rng.integers(-2 ** 28, 2 ** 28, (n, 2 * hk * dim)).astype(np.int32)).cuda()
    q = torch.from_numpy(rng.integers(-2 ** 28, 2 ** 28, (n, heads * dim)).astype(np.int32)).cuda()
    scale = torch.from_numpy(np.stack([rng.integers(2 ** 31, 2 ** 32, n), rng.integers(59, 63, n)], -1)).cuda()
    rope = tb.Rope(torch.from_numpy(tb.rope_table(1e4, dim, n)).cuda())
    pages = torch.arange(-(-n // page), dtype=torch.int32, device="cuda")[None]
    results = []
    for sizes in ([n], [1] * 5 + [100] + [30] * 3 + [5], [64, 64, 64, 8], [199, 1]):
        cache = tb.KvCache(ctx, pages.shape[1], page, hk, dim)
        o = torch.zeros(n, heads * dim, dtype=torch.int32, device="cuda")
        os_ = torch.zeros(n, hk, 2, dtype=torch.int64, device="cuda")
        at = 0
        for c in sizes:
            b = tb.KvBatch(torch.tensor([0, c], dtype=torch.int32, device="cuda"),
                           torch.tensor([at + c], dtype=torch.int32, device="cuda"), pages, c)
            x = kv[at:at + c]
            cache.append(b, x[:, :hk * dim], x[:, hk * dim:], scale[at:at + c], rope)
            cache.attention(b, q[at:at + c], scale[at:at + c], o[at:at + c], os_[at:at + c], heads, rope=rope,
                            window=window, sinks=sinks)
            at += c
        assert at == n
        ctx.sync()
        torch.cuda.synchronize()
        results.append((o.cpu(), os_.cpu(), cache.k.cpu(), cache.v.cpu()))
    for r in results[1:]:
        assert all(torch.equal(a, b) for a, b in zip(results[0], r))


def test_offsets_beyond_32_bits(ctx):
    """Pools of more than 2^31 bytes, the sequence in the last pages."""
    torch = _torch()
    hk, dim, page = 8, 128, 128
    n_pages = (1 << 31) // (hk * page * dim) + 20
    cache = tb.KvCache(ctx, n_pages, page, hk, dim)
    small = tb.KvCache(ctx, 3, page, hk, dim)
    rng = np.random.default_rng(1)
    outs = []
    for c, first in ((cache, n_pages - 3), (small, 0)):
        rng = np.random.default_rng(1)
        for new, kv in ((300, 300), (1, 301)):
            b = tb.KvBatch(torch.tensor([0, new], dtype=torch.int32, device="cuda"),
                           torch.tensor([kv], dtype=torch.int32, device="cuda"),
                           torch.tensor([[first + 2, first, first + 1]], dtype=torch.int32, device="cuda"), new)
            x = torch.from_numpy(rng.integers(-2 ** 28, 2 ** 28, (new, 4 * hk * dim)).astype(np.int32)).cuda()
            s = torch.tensor([2 ** 31, 60], device="cuda")
            o = torch.zeros(new, 2 * hk * dim, dtype=torch.int32, device="cuda")
            os_ = torch.zeros(new, hk, 2, dtype=torch.int64, device="cuda")
            c.append(b, x[:, :hk * dim], x[:, hk * dim:2 * hk * dim], s)
            c.attention(b, x[:, 2 * hk * dim:], s, o, os_, 2 * hk)
            ko, vo = torch.zeros(new, hk * dim, device="cuda"), torch.zeros(new, hk * dim, device="cuda")
            c.read(b, ko, vo)
            outs.append((o.cpu(), os_.cpu(), ko.cpu(), vo.cpu()))
    ctx.sync()
    for a, b in zip(outs[:2], outs[2:]):
        assert all(torch.equal(x, y) for x, y in zip(a, b))
        assert int((a[0] != 0).sum()) > 0


# ── streams, graphs, errors ──


def test_two_streams_and_a_replayed_graph(ctx):
    """Calls on two streams at once, and a captured write-attend-read replayed on changed lengths and inputs: nothing is
    kept between calls."""
    torch = _torch()
    s = Setup(ctx, [(1, 150), (1, 70)], 4, 2, 64, 16, spare=30)
    s2 = Setup(ctx, [(30, 150), (20, 70)], 4, 2, 64, 16, spare=3, seed=5)
    q2, sc2 = s2.codes(4 * 64), s2.scales()
    kv = torch.from_numpy(s.codes(2 * 128)).cuda()
    q = torch.from_numpy(s.codes(4 * 64)).cuda()
    scale = torch.from_numpy(s.scales()).cuda()
    o, os_ = torch.zeros(2, 256, dtype=torch.int32, device="cuda"), torch.zeros(2, 2, 2, dtype=torch.int64, device="cuda")
    ko, vo = torch.zeros(2, 128, device="cuda"), torch.zeros(2, 128, device="cuda")

    def step():
        s.cache.append(s.batch, kv[:, :128], kv[:, 128:], scale)
        s.cache.attention(s.batch, q, scale, o, os_, 4, window=60, sinks=2)
        s.cache.read(s.batch, ko, vo)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    side.synchronize()

    def written():
        R.append(kv[:, :128].cpu().numpy().reshape(2, 2, 64), kv[:, 128:].cpu().numpy().reshape(2, 2, 64),
                 scale.cpu().numpy(), s.begin, s.kv_len, s.write)

    written()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for i in range(3):
        kv.copy_(torch.from_numpy(s.codes(2 * 128)))
        q.copy_(torch.from_numpy(s.codes(4 * 64)))
        s.kv_len = [151 + i - 20 * i, 71 + i]
        s.batch.kv_len.copy_(torch.tensor(s.kv_len, dtype=torch.int32))
        torch.cuda.synchronize()
        graph.replay()
        with torch.cuda.stream(side):  # beside the replay
            s2.check(q2, sc2)
        torch.cuda.synchronize()
        written()
        want, want_s = np.zeros((2, 4, 64), np.int64), np.zeros((2, 2, 2), np.int64)
        R.attention(q.cpu().numpy().reshape(2, 4, 64), scale.cpu().numpy(), s.begin, s.kv_len, s.keys, want, want_s,
                    64 ** -0.5, 60, 2)
        assert (o.cpu().numpy().reshape(want.shape) == want).all()
        for n, t in (("k", s.cache.k), ("vs", s.cache.v_scale)):
            assert (t.double().cpu().numpy() == s.pool[n].astype(np.float64)).all()
    ctx.sync()


@pytest.mark.parametrize("what", ["page", "negative_page", "long", "longest", "negative", "descending", "rows", "position"])
@pytest.mark.parametrize("new,hk", [(1, 2), (40, 2), (40, 150)])
def test_wrong_batches_are_reported_and_harmless(ctx, what, new, hk):
    """What only the device can see: the calls touch nothing outside their buffers, sync reports it, and the context
    serves on."""
    torch = _torch()
    s = Setup(ctx, [(new, 100), (new, 90)], 2 * hk, hk, 64, 16, rows_behind=1)
    n = hk * 64
    rope = None
    if what == "page":
        s.batch.page_table[1, 2] = s.cache.n_pages
    elif what == "negative_page":
        s.batch.page_table[0, 0] = -1
    elif what == "long":
        s.batch.kv_len[1] = s.max_pages * 16 + 1
    elif what == "longest":
        s.batch.kv_len[1] = 2 ** 31 - 1  # rounded up to pages it would pass 32 bits
    elif what == "negative":
        s.batch.kv_len[0] = -3
    elif what == "descending":
        s.batch.q_begin[1] = 2 * new + 1
    elif what == "rows":
        s.batch.q_begin[2] = 2 * new + 5
    elif what == "position":
        rope = tb.Rope(torch.from_numpy(tb.rope_table(1e4, 64, 80)).cuda())
    q = torch.from_numpy(s.codes(2 * n)).cuda()
    kv = torch.from_numpy(s.codes(2 * n)).cuda()
    scale = torch.from_numpy(s.scales()).cuda()
    guard = torch.full((s.rows + 2, 2 * n), 77, dtype=torch.int32, device="cuda")
    os_ = torch.zeros(s.rows, hk, 2, dtype=torch.int64, device="cuda")
    ko = torch.full((s.rows + 2, n), 7.0, device="cuda")

    def reported(call):
        call()
        torch.cuda.synchronize()
        with pytest.raises(tb.KtmoeError) as e:
            ctx.sync()
        assert e.value.status == _native.ERR_ARG
        ctx.sync()  # reported once

    reported(lambda: s.cache.attention(s.batch, q, scale, guard[1:-1], os_, 2 * hk, rope=rope))
    if what in ("page", "negative_page"):
        # a page that no new row lies in is no business of the write
        s.batch.page_table[:] = s.cache.n_pages if what == "page" else -7
    reported(lambda: s.cache.append(s.batch, kv[:, :n], kv[:, n:], scale, rope))
    if what != "position":
        reported(lambda: s.cache.read(s.batch, ko[1:-1], ko[1:-1].clone()))
    assert (guard[0] == 77).all() and (guard[-1] == 77).all()
    assert (ko[0] == 7).all() and (ko[-1] == 7).all()
    Setup(ctx, [(new, 100)], 4, 2, 64, 16).check(s.codes(256)[:new], s.scales()[:new])


def test_a_wrong_batch_leaves_other_work_alone(ctx):
    """Between a wrong batch and the sync that reports it, linears run and report for themselves."""
    torch = _torch()
    s = Setup(ctx, [(1, 100)], 4, 2, 64, 16)
    s.batch.page_table[0, 2] = s.cache.n_pages
    q = torch.from_numpy(s.codes(256)).cuda()
    scale = torch.from_numpy(s.scales()).cuda()
    out, os_ = torch.zeros_like(q), torch.zeros(1, 2, 2, dtype=torch.int64, device="cuda")
    torch.cuda.synchronize()
    s.cache.attention(s.batch, q, scale, out, os_, 4)
    torch.cuda.synchronize()
    rng = np.random.default_rng(5)
    x, w = rng.integers(-1000, 1000, (96, 256), dtype=np.int32), rng.integers(-1000, 1000, (128, 256), dtype=np.int32)
    y = ctx.linear(x, w, 96, 128, 256)
    assert (np.asarray(y).reshape(96, 128) == x.astype(np.int64) @ w.astype(np.int64).T).all()
    with pytest.raises(tb.KtmoeError) as e:
        ctx.sync()
    assert e.value.status == _native.ERR_ARG
    ctx.sync()


def test_nothing_to_do(ctx):
    torch = _torch()
    s = Setup(ctx, [(0, 5), (0, 0)], 2, 1, 16, 16, rows_behind=2)
    s.check(s.codes(32), s.scales())  # sequences without new tokens: nothing is touched
    none = tb.KvBatch(*(torch.zeros(n, dtype=torch.int32, device="cuda") for n in (1, 0)),
                      torch.zeros(0, 1, dtype=torch.int32, device="cuda"), 0)
    e = torch.zeros(0, 16, dtype=torch.int32, device="cuda")
    one = torch.tensor([1, 0], device="cuda")
    s.cache.append(none, e, e, one)
    s.cache.read(none, e.float(), e.float())
    s.cache.attention(none, e, one, e, torch.zeros(0, 1, 2, dtype=torch.int64, device="cuda"), 1)
    ctx.sync()


def test_refusals_of_the_c_entry_points(ctx):
    torch = _torch()
    L = tb.lib()
    s = Setup(ctx, [(1, 5)], 2, 1, 16, 16)
    q, o = torch.zeros(1, 32, dtype=torch.int32, device="cuda"), torch.full((1, 32), 7, dtype=torch.int32, device="cuda")
    sc, os_ = torch.zeros(1, 2, dtype=torch.int64, device="cuda"), torch.zeros(1, 1, 2, dtype=torch.int64, device="cuda")

    def cache(**kw):
        c = _native.KtmoeKvCache.from_buffer_copy(s.cache._c)
        for k, v in kw.items():
            setattr(c, k, v)
        return c

    def batch(**kw):
        b = _native.KtmoeKvBatch.from_buffer_copy(s.batch._c)
        for k, v in kw.items():
            setattr(b, k, v)
        return b

    table = torch.zeros(4, 8, 2, dtype=torch.int32, device="cuda")

    def attend(c=None, b=None, q_=None, ld=32, scale=None, stride=1, rope=None, heads=2, soft=1.0, window=0, sinks=0,
               out=None, ld_o=32, out_scale=None):
        return L.ktmoe_attention_dev(ctx.handle, c or cache(), b or batch(), q.data_ptr() if q_ is None else q_, ld,
                                     sc.data_ptr() if scale is None else scale, stride, rope, heads, soft, window, sinks,
                                     o.data_ptr() if out is None else out, ld_o,
                                     os_.data_ptr() if out_scale is None else out_scale, None)

    ARG, UNS = _native.ERR_ARG, _native.ERR_UNSUPPORTED
    rope = lambda **kw: _native.KtmoeRope(*{**dict(table=table.data_ptr(), positions=4, rot_dim=16, interleaved=0), **kw}.values())
    for kw, want in [
        (dict(c=cache(k=0)), ARG), (dict(c=cache(v_scale=0)), ARG), (dict(c=cache(k=s.cache.k.data_ptr() + 8)), ARG),
        (dict(c=cache(v=s.cache.v.data_ptr() + 8)), ARG), (dict(c=cache(k_scale=s.cache.k_scale.data_ptr() + 8)), ARG),
        (dict(c=cache(v_scale=s.cache.v_scale.data_ptr() + 8)), ARG),
        (dict(c=cache(head_dim=24)), UNS), (dict(c=cache(head_dim=272)), UNS), (dict(c=cache(head_dim=0)), UNS),
        (dict(c=cache(page_tokens=8)), UNS), (dict(c=cache(page_tokens=48)), UNS), (dict(c=cache(page_tokens=256)), UNS),
        (dict(c=cache(n_pages=0)), ARG), (dict(c=cache(n_kv_heads=0)), ARG), (dict(c=cache(n_kv_heads=1025)), ARG),
        (dict(b=batch(n_seqs=-1)), ARG), (dict(b=batch(rows=-1)), ARG), (dict(b=batch(max_pages=-1)), ARG),
        (dict(b=batch(max_pages=1 << 30)), ARG), (dict(b=batch(rows=1 << 40)), ARG), (dict(b=batch(q_begin=0)), ARG),
        (dict(b=batch(kv_len=0)), ARG), (dict(b=batch(page_table=0)), ARG),
        (dict(q_=0), ARG), (dict(q_=q.data_ptr() + 2), ARG), (dict(ld=31), ARG), (dict(scale=0), ARG),
        (dict(scale=sc.data_ptr() + 8), ARG), (dict(stride=2), ARG), (dict(stride=-1), ARG), (dict(heads=0), ARG),
        (dict(soft=0.0), ARG), (dict(soft=-1.0), ARG), (dict(soft=math.nan), ARG), (dict(soft=math.inf), ARG),
        (dict(window=-1), ARG), (dict(sinks=-1), ARG), (dict(out=0), ARG), (dict(ld_o=31), ARG), (dict(out_scale=0), ARG),
        (dict(out_scale=os_.data_ptr() + 8), ARG),
        (dict(rope=rope(table=0)), ARG), (dict(rope=rope(table=table.data_ptr() + 4)), ARG),
        (dict(rope=rope(positions=0)), ARG), (dict(rope=rope(rot_dim=3)), ARG), (dict(rope=rope(rot_dim=18)), ARG),
        (dict(rope=rope(rot_dim=0)), ARG),
    ]:
        assert attend(**kw) == want, kw
    c3 = cache(n_kv_heads=3)
    assert attend(c=c3) == ARG  # two query heads over three KV heads
    a = [ctx.handle, cache(), batch()]
    assert L.ktmoe_kv_append_dev(*a, q.data_ptr(), 15, q.data_ptr(), 16, sc.data_ptr(), None, 1, None, None) == ARG
    assert L.ktmoe_kv_append_dev(*a, q.data_ptr(), 16, q.data_ptr(), 15, sc.data_ptr(), None, 1, None, None) == ARG
    assert L.ktmoe_kv_append_dev(*a, None, 16, q.data_ptr(), 16, sc.data_ptr(), None, 1, None, None) == ARG
    assert L.ktmoe_kv_append_dev(*a, q.data_ptr(), 16, q.data_ptr(), 16, None, None, 1, None, None) == ARG
    assert L.ktmoe_kv_append_dev(*a, q.data_ptr(), 16, q.data_ptr(), 16, sc.data_ptr(), sc.data_ptr() + 8, 1, None, None) == ARG
    assert L.ktmoe_kv_append_dev(*a, q.data_ptr(), 16, q.data_ptr(), 16, sc.data_ptr(), None, 1, rope(rot_dim=5), None) == ARG
    assert L.ktmoe_kv_read_dev(*a, o.data_ptr(), 16, None, 16, None) == ARG
    assert L.ktmoe_kv_read_dev(*a, o.data_ptr(), 12, o.data_ptr(), 16, None) == ARG
    torch.cuda.synchronize()
    ctx.sync()
    assert (o == 7).all()
