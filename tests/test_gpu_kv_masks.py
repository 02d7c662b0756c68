"""Attention over the paged cache where a key that a row does not see could show in it all the same: value scales far
above those that it sees, on a B200, against the plain 64-bit restatement (tests/kv_reference.py). All arithmetic is exact
by definition, so the tolerance is zero. Setup.check runs each batch through the few-row kernel and, with copies of all
heads, through the tile kernel."""

import numpy as np
import pytest

import kv_reference as R
import tritify_b200 as tb
from test_gpu_kv import Setup, _torch

pytestmark = pytest.mark.gpu


def positions_of(s, b):
    """Pool pages and places of a sequence's positions."""
    j = np.arange(s.kv_len[b])
    return s.table[b, j // s.page], j % s.page


def set_value_scales(s, b, sigma):
    """sigma [kv_len]: of every KV head."""
    page, place = positions_of(s, b)
    s.pool["vs"][page, :, place] = sigma[:, None]


SHAPES = [  # new, total, query heads, KV heads, dim, page
    (64, 64, 4, 1, 64, 16),
    (150, 150, 3, 1, 128, 64),
    (70, 200, 4, 2, 48, 32),
    (64, 64, 4, 1, 256, 16),
]


@pytest.mark.parametrize("step", [17, 20, 40, 126])
@pytest.mark.parametrize("shape", SHAPES, ids=[str(i) for i in range(len(SHAPES))])
def test_later_tokens_of_larger_scales(ctx, shape, step):
    """Value scales that rise by 2^step every few tokens, and fall back: what a row does not see yet weighs nothing."""
    new, kv, heads, hk, dim, page = shape
    s = Setup(ctx, [(new, kv)], heads, hk, dim, page, seed=step)
    j = np.arange(kv)
    set_value_scales(s, 0, np.exp2((step * (j // 5)) % 127 - 64.0) * (1 + (j % 3) / 4))
    s.push()
    s.check(s.codes(heads * dim), s.scales())


@pytest.mark.parametrize("first", [0, 30])
def test_a_first_value_of_zeros(ctx, first):
    """The first value row is zeros (at 2^-64, as the cache writes it) and stands alone for row 0: zeros, at its scale."""
    s = Setup(ctx, [(64, 64 + first)], 4, 1, 64, 16, seed=first)
    page, place = positions_of(s, 0)
    s.pool["v"][page[:first + 1], :, place[:first + 1]] = 0
    s.pool["vs"][page[:first + 1], :, place[:first + 1]] = 2.0 ** -64
    s.push()
    got, got_s, want, want_s = s.attend(s.codes(4 * 64), s.scales())
    assert (want[0] == 0).all() and (want[1] != 0).any()
    assert (got == want).all() and (got_s == want_s).all()


@pytest.mark.parametrize("window,sinks", [(10, 0), (10, 3), (100, 1)])
@pytest.mark.parametrize("step", [20, 40, 110])
@pytest.mark.parametrize("since", [236, 240])  # 236: the first new token sees its own
def test_larger_scales_outside_the_window(ctx, since, window, sinks, step):
    s = Setup(ctx, [(64, 300)], 4, 1, 64, 32, seed=window + step)
    sigma = np.full(300, 2.0 ** -50)
    sigma[sinks:236 - window + 1] = 2.0 ** (step - 50)  # what no new token sees, but tiles hold with what they see
    sigma[since:260:7] = 2.0 ** (step - 50)  # what some of them see
    set_value_scales(s, 0, sigma)
    s.push()
    s.check(s.codes(4 * 64), s.scales(), window=window, sinks=sinks)


@pytest.mark.parametrize("hk", [2, 60])  # 60: the whole prompt goes to the tile kernel
def test_a_prompt_equals_its_tokens(ctx, hk):
    """A written prompt whose values grow from zeros over 2^80, at once and token by token."""
    torch = _torch()
    n, heads, dim, page = 140, 3 * hk, 64, 16
    rng = np.random.default_rng(4)
    kv = torch.from_numpy(rng.integers(-2 ** 28, 2 ** 28, (n, 2 * hk * dim)).astype(np.int32)).cuda()
    kv[0, hk * dim:] = 0
    q = torch.from_numpy(rng.integers(-2 ** 28, 2 ** 28, (n, heads * dim)).astype(np.int32)).cuda()
    scale = torch.from_numpy(np.stack([rng.integers(2 ** 31, 2 ** 32, n), rng.integers(59, 63, n)], -1)).cuda()
    v_scale = torch.from_numpy(np.stack([rng.integers(2 ** 31, 2 ** 32, n), 110 - 80 * np.arange(n) // n], -1)).cuda()
    pages = torch.arange(-(-n // page), dtype=torch.int32, device="cuda")[None]
    results = []
    for sizes in ([n], [1] * n):
        cache = tb.KvCache(ctx, pages.shape[1], page, hk, dim)
        o = torch.zeros(n, heads * dim, dtype=torch.int32, device="cuda")
        os_ = torch.zeros(n, hk, 2, dtype=torch.int64, device="cuda")
        at = 0
        for c in sizes:
            b = tb.KvBatch(torch.tensor([0, c], dtype=torch.int32, device="cuda"),
                           torch.tensor([at + c], dtype=torch.int32, device="cuda"), pages, c)
            x = kv[at:at + c]
            cache.append(b, x[:, :hk * dim], x[:, hk * dim:], scale[at:at + c], v_scale=v_scale[at:at + c])
            before = ctx.launch_count()
            cache.attention(b, q[at:at + c], scale[at:at + c], o[at:at + c], os_[at:at + c], heads)
            assert ctx.launch_count() - before == (2 if c == n and hk == 60 else 1)
            at += c
        ctx.sync()
        torch.cuda.synchronize()
        results.append((o.cpu(), os_.cpu()))
    assert int((results[1][0][0] != 0).sum()) == 0
    assert all(torch.equal(a, b) for a, b in zip(*results))


GARBAGE = [np.nan, np.inf, -np.inf, 2.0 ** 127, -1.0]


@pytest.mark.parametrize("garbage", GARBAGE, ids=[str(g) for g in GARBAGE])
@pytest.mark.parametrize("lens,heads,hk,dim,window,sinks", [
    ([(1, 1), (1, 5), (1, 126), (1, 131)], 4, 1, 64, 0, 0),
    ([(1, 198), (1, 67)], 4, 2, 128, 20, 2),
    ([(64, 65)], 4, 1, 64, 0, 0),
    ([(90, 201), (64, 64)], 4, 1, 128, 0, 0),
    ([(64, 398)], 4, 1, 256, 100, 5),
])
def test_places_that_were_never_written(ctx, lens, heads, hk, dim, window, sinks, garbage):
    """Pools of memory that nothing cleared: whatever lies behind a sequence's last token, and outside every window of
    the call, shows nowhere."""
    s = Setup(ctx, lens, heads, hk, dim, 16, seed=dim)
    seen = np.zeros(s.pool["vs"].shape, bool)
    for b, (new, kv) in enumerate(lens):
        j = np.arange(kv)
        if window:
            j = j[(j > kv - new - window) | (j < sinks)]
        seen[s.table[b, j // 16], :, j % 16] = True
    for n in "kv":
        s.pool[n][~seen] = -1
        s.pool[n + "s"][~seen] = garbage
    s.push()
    s.check(s.codes(heads * dim), s.scales(), window=window, sinks=sinks)


@pytest.mark.parametrize("window", [2 ** 31 - 1, 2 ** 31 - 5, 2 ** 30])
@pytest.mark.parametrize("sinks", [0, 3, 2 ** 31 - 1])
def test_the_widest_windows(ctx, window, sinks):
    """Rows at negative positions, which see nothing, in one group with rows that see keys, and a window near 2^31: it
    hides nothing."""
    s = Setup(ctx, [(19, 8), (41, 40)], 4, 1, 64, 16, rows_behind=1)
    q, scale = s.codes(4 * 64), s.scales()
    s.check(q, scale, window=window, sinks=sinks)
    wide, narrow = s.attend(q, scale, window=window, sinks=sinks), s.attend(q, scale)
    assert (wide[0] == narrow[0]).all() and (wide[1] == narrow[1]).all()


def test_pools_are_cleared_before_anything_is_written(ctx):
    """A cache made while torch's stream is busy and written at once on the context's stream: the clearing of its pools
    does not come after the writing."""
    torch = _torch()
    i32 = lambda *a: torch.tensor(a, dtype=torch.int32, device="cuda")
    batch = tb.KvBatch(i32(0, 9), i32(9), i32(0).reshape(1, 1), 9)
    kv = torch.full((9, 64), 2 ** 20, dtype=torch.int32, device="cuda")
    scale = torch.tensor([1, 20], dtype=torch.int64, device="cuda")
    tb.KvCache(ctx, 1, 16, 2, 32).append(batch, kv, kv, scale, stream=0)  # loads the kernel, which waits for the device
    torch.cuda.synchronize()
    torch.cuda._sleep(200_000_000)  # about a tenth of a second
    cache = tb.KvCache(ctx, 1, 16, 2, 32)
    cache.append(batch, kv, kv, scale, stream=0)  # the context's stream
    ctx.sync()
    torch.cuda.synchronize()
    codes, sigma = R.quantise_row(np.full(32, 2 ** 20), 2.0 ** -20)
    assert codes[0] == 126  # 1 / 127 is 1.0079 2^-7, sigma 1.015625 2^-7, and 128 / 1.015625 is 126.03
    assert (cache.k[0, :, :9] == 126).all() and (cache.v[0, :, :9] == 126).all()
    assert (cache.k_scale[0, :, :9] == sigma).all() and (cache.v_scale[0, :, 9:] == 0).all()
