"""The KV-cache operators measured here: writing new keys and values into a paged cache of 8-bit codes, reading them
back, and the attention of new tokens over such a cache, all in exact integers.

A case is one call (or one write followed by its read-back) with everything a serving program holds in hand: int32
activation codes with a scale per row, the batch's lengths and page table, the pools and the rotation table. ``run``
computes it in elementary torch operations, or through the framework (``own``). The outputs that are whole numbers are
defined exactly (each rounding is stated below), so both sides give the same integers; cache contents are returned as
the values their codes stand for.

Definitions. A scale is {mant, shift}, mant * 2^-shift. RN24 and RN64 round to 24 and 53 significant bits, ties to
even (binary32 and binary64); rne rounds to an integer, ties to even.

* rotation: with table codes c, s (cosine and sine times 2^30) a pair (a, b) becomes (a c - b s, b c + a s) and every
  other element x becomes 2^30 x, exactly, at 2^-30 times the row's scale.
* a cached row (one token, one KV head): t = RN64(RN64(max|y| * scale) / 127) held within [2^-64, 2^63], sigma = t
  rounded up to 8 significant bits, codes rne(RN64(y * RN64(scale / sigma))) within +-127.
* a query row: codes rne(RN64(y * RN64(127 / max|y|))), theta = RN24(min(2^60, RN64(RN64(RN64(max|y| * scale) / 127)
  * RN64(softmax_scale * log2 e)))).
* its visible keys: position j <= its own, and within the window or among the sinks. x_j = RN24((q . k_j) sigma_k),
  d_j = RN24(max x - x_j), z_j = min(32 * 2^10, rne(2^10 d_j theta)), n_j = rne(z_j / 2^10), r_j = n_j - z_j / 2^10,
  w_j = 2^-n_j * e(r_j), e a cubic with 32512 at 0 whose three steps are each rounded by RN24.
* the output: L = sum of rne(w_j), 2^E = the least power of two no smaller than any visible sigma_v,
  O = sum of rne(w_j sigma_v 2^-E) v_j, codes rne(RN64(O * RN64(2^21 / L))) at the scale {1, 21 - E}. A row that sees
  nothing is zeros at the scale {0, 0}.
"""

from __future__ import annotations

import math
import random

import torch

own = False

LOG2E = 1.4426950408889634
AMP = 32512.0  # 127 * 256: the largest weight, two balanced 8-bit digits
C1, C2, C3 = 127 * 45435 / 256, 127 * 15874 / 256, 127 * 3605 / 256  # the cubic's coefficients times 32512, exact


# ── cases ──


def _case(name, kind, seqs, new, kv, ragged, heads, kv_heads, dim, page, rope="half", rot=0, window=0, sinks=0, pad=0):
    return {**({"name": name} if name else {}), "kind": kind, "seqs": seqs, "new": new, "kv": kv, "ragged": ragged, "heads": heads,
            "kv_heads": kv_heads, "dim": dim, "page": page, "rope": rope, "rot": rot or dim, "window": window,
            "sinks": sinks, "pad": pad}


def listed():
    return [
        # one decode step's keys and values of a batch of 64 sequences
        _case("write_decode", "write", 64, 1, 4096, True, 32, 8, 128, 64),
        # the keys and values of a 16384-token prefill
        _case("write_prefill", "write", 1, 16384, 16384, False, 32, 8, 128, 64, rope="pairs", rot=64),
        # a ragged batch, no rotation, few odd heads, small pages, padding behind the batch
        _case("write_ragged", "write", 7, 301, 777, True, 15, 3, 80, 16, rope="none", pad=5),
        # a sequence's whole cache read back (to move it to another host)
        _case("read_sequence", "read", 1, 32768, 32768, False, 32, 8, 128, 64),
        # short sequences read back together
        _case("read_ragged", "read", 9, 211, 211, True, 14, 2, 64, 32),
        # the smallest call: one sequence decoding at a short length
        _case("decode_one", "attend", 1, 1, 1000, False, 32, 8, 128, 64),
        # a decode batch of 64 sequences of mixed lengths
        _case("decode_batch", "attend", 64, 1, 4096, True, 32, 8, 128, 64),
        # decode at long lengths with twelve query heads to a KV head, half of each head rotated
        _case("decode_long", "attend", 4, 1, 65536, True, 96, 8, 128, 64, rope="pairs", rot=64),
        # a whole prompt
        _case("prefill", "attend", 1, 4096, 4096, False, 32, 8, 128, 64),
        # prompts continued in chunks over what the cache already holds
        _case("chunk", "attend", 4, 512, 8192, True, 16, 16, 128, 128),
        # a long prompt with a sliding window and the first tokens kept
        _case("window_prefill", "attend", 1, 8192, 8192, False, 32, 8, 128, 64, window=1024, sinks=4),
        # small ragged chunks, seven heads to a KV head, a window that ends inside pages, padding
        _case("ragged_window", "attend", 11, 9, 1500, True, 14, 2, 64, 16, window=333, sinks=3, pad=3),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng: random.Random):
    kind = rng.choice(["write", "read", "attend", "attend", "attend"])
    dim = rng.choice([64, 128, 128, 80, 96, 256])
    kv_heads = rng.choice([1, 2, 4, 8, 8, 5])
    group = rng.choice([1, 2, 4, 4, 7, 8, 12, 16])
    page = rng.choice([16, 32, 64, 128])
    rope = rng.choice(["half", "pairs", "none"])
    rot = rng.choice([dim, dim // 2])
    seqs = _log(rng, 1, 64)
    if kind != "attend":
        new = _log(rng, 1, max(1, 16384 * 8 * 128 // (seqs * kv_heads * dim)))
        kv = new + (0 if kind == "read" else _log(rng, 1, 4096))
        return _case("", kind, seqs, new, kv, rng.random() < 0.7, kv_heads * group, kv_heads, dim, page, rope, rot,
                     pad=rng.choice([0, 0, 3]))
    new = rng.choice([1, 1, _log(rng, 2, 16), _log(rng, 2, 2048)])
    top = 4096 * 4096 * 32 * 128 // 4  # query-key pairs times heads times dim
    kv_top = max(new, min(65536, top // (seqs * new * kv_heads * group * dim), 2 ** 28 // (seqs * kv_heads * dim)))
    kv = _log(rng, min(new, kv_top), kv_top)
    new = min(new, kv)
    windowed = rng.random() < 0.4
    return _case("", kind, seqs, new, kv, rng.random() < 0.7, kv_heads * group, kv_heads, dim, page, rope, rot,
                 window=_log(rng, 1, max(2, kv)) if windowed else 0, sinks=rng.choice([0, 1, 4, 70]) if windowed else 0,
                 pad=rng.choice([0, 0, 3]))


def _lens(c):
    """New tokens and total length of each sequence; a ragged batch spreads both below the case's own sizes."""
    out = []
    for i in range(c["seqs"]):
        new, kv = c["new"], c["kv"]
        if c["ragged"]:
            a, b = (i * 2654435761 >> 5) % 61, (i * 40503 >> 2) % 53
            new = max(1, new - new * a // 122)
            kv = max(new, kv - kv * b // 80) if c["kind"] != "read" else new
        out.append((new, kv))
    return out


def _rows(c):
    return sum(n for n, _ in _lens(c)) + c["pad"]


def _visible(c, pos):
    """How many keys a row at position ``pos`` sees."""
    if not c["window"] or pos < c["window"]:
        return pos + 1
    return c["window"] + min(c["sinks"], pos + 1 - c["window"])


def work(c):
    lens, h, hk, d = _lens(c), c["heads"], c["kv_heads"], c["dim"]
    n = sum(a for a, _ in lens)
    codes = 2 * hk * (d + 2)  # one token's cached keys and values: codes and 16-bit scales
    rope = (8 if c["rope"] != "none" else 0) * (c["rot"] // 2)
    if c["kind"] == "write":  # int32 in, codes out; then codes in, float32 out
        return {"bytes": n * (2 * hk * d * 4 + 16 + rope + 2 * codes + 2 * hk * d * 4), "flops": n * 2 * hk * d * 8}
    if c["kind"] == "read":
        return {"bytes": n * (codes + 2 * hk * d * 4), "flops": n * 2 * hk * d}
    pairs, keys = 0, 0
    for new, kv in lens:
        pairs += sum(_visible(c, p) for p in range(kv - new, kv))
        keys += kv if not c["window"] else min(kv, new + c["window"] - 1 + c["sinks"])
    return {"bytes": keys * codes + n * (h * d * 8 + 16 + rope + 16 * hk), "flops": pairs * h * d * 4}


# ── inputs ──


def _two(e):
    """2^e in float64 for whole numbers e, exactly."""
    return ((e.to(torch.int64) + 1023) << 52).view(torch.float64)


def _scale_rows(v):
    """{mant, shift} of positive float64 values, as the two 64-bit words of a scale."""
    m, e = torch.frexp(v)
    mant = torch.round(m * 2.0 ** 32).to(torch.int64)
    shift = (32 - e.to(torch.int64)) & 0xFFFFFFFF
    return torch.stack([mant, shift], -1)


def _activation(gen, rows, width, dim, dev):
    """What a linear leaves: int32 codes filling 28 bits at each row's own scale; a few channels of a head are large."""
    x = torch.randn(rows, width, generator=gen, device=dev)
    gain = torch.ones(dim, device=dev)
    gain[::37] = 4.0
    x = x * gain.repeat(width // dim)
    top = x.abs().amax(1, keepdim=True).clamp_min(1e-6).double()
    return torch.round(x.double() / top * 2 ** 28).to(torch.int32), _scale_rows(top[:, 0] / 2 ** 28)


def _table(c, positions, dev):
    if c["rope"] == "none":
        return None
    half = c["rot"] // 2
    f = 10000.0 ** (-torch.arange(half, device=dev, dtype=torch.float64) / half)
    a = torch.arange(positions, device=dev, dtype=torch.float64)[:, None] * f
    return torch.round(torch.stack([a.cos(), a.sin()], -1) * 2 ** 30).to(torch.int32)


def prepare(c, seed):
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev)
    gen.manual_seed(int(seed))
    lens, hk, d, ps = _lens(c), c["kv_heads"], c["dim"], c["page"]
    need = [-(-kv // ps) for _, kv in lens]
    n_pages = sum(need) + 3
    perm = torch.randperm(n_pages, generator=gen, device=dev).to(torch.int32)
    table = torch.zeros(len(lens), max(need), dtype=torch.int32, device=dev)
    at = 0
    for b, k in enumerate(need):
        table[b, :k] = perm[at:at + k]
        at += k
    begin = [0]
    for new, _ in lens:
        begin.append(begin[-1] + new)
    rows = _rows(c)
    st = {"case": c, "lens": lens, "rows": rows, "n_pages": n_pages,
          "begin": torch.tensor(begin, dtype=torch.int32, device=dev),
          "kv_len": torch.tensor([kv for _, kv in lens], dtype=torch.int32, device=dev), "table": table,
          "rope": _table(c, max(kv for _, kv in lens), dev)}
    shape = (n_pages, hk, ps)
    st["k"] = torch.zeros(*shape, d, dtype=torch.int8, device=dev)
    st["v"] = torch.zeros(*shape, d, dtype=torch.int8, device=dev)
    st["ks"] = torch.zeros(shape, dtype=torch.bfloat16, device=dev)
    st["vs"] = torch.zeros(shape, dtype=torch.bfloat16, device=dev)
    if c["kind"] == "write":
        x, st["scale"] = _activation(gen, rows, 2 * hk * d, d, dev)
        st["kv_in"] = x  # keys and values side by side, as one linear leaves them
    else:  # a cache that already holds the sequences: codes of normal values at their rows' scales
        gain = torch.ones(d, device=dev)
        gain[::37] = 4.0
        step = max(1, 2 ** 26 // (hk * ps * d))
        for name, sc in (("k", "ks"), ("v", "vs")):
            for p in range(0, n_pages, step):
                y = torch.randn(min(step, n_pages - p), hk, ps, d, generator=gen, device=dev) * gain
                sg = _sigma(y.abs().amax(-1).double() / 127)
                st[name][p:p + step] = torch.round(y.double() / sg[..., None]).clamp(-127, 127).to(torch.int8)
                st[sc][p:p + step] = sg.to(torch.bfloat16)
    if c["kind"] == "attend":
        st["q"], st["scale"] = _activation(gen, rows, c["heads"] * d, d, dev)
        st["o"] = torch.zeros(rows, c["heads"] * d, dtype=torch.int32, device=dev)
        st["os"] = torch.zeros(rows, hk, 2, dtype=torch.int64, device=dev)
    else:
        st["ko"] = torch.zeros(rows, hk * d, dtype=torch.float32, device=dev)
        st["vo"] = torch.zeros(rows, hk * d, dtype=torch.float32, device=dev)
    if own:
        import tritify_b200 as tb

        st["cache"] = tb.KvCache(tb.default_context(), n_pages, ps, hk, d, pools=(st["k"], st["v"], st["ks"], st["vs"]))
        st["batch"] = tb.KvBatch(st["begin"], st["kv_len"], st["table"], rows)
        st["rot"] = None if st["rope"] is None else tb.Rope(st["rope"], interleaved=c["rope"] == "pairs")
    return st


# ── the operators, plainly ──


def _sigma(t):
    """t held within [2^-64, 2^63] and rounded up to 8 significant bits."""
    m, e = torch.frexp(t.clamp(2.0 ** -64, 2.0 ** 63))
    return torch.ceil(m * 256) * _two(e - 8)


def _value(scale):
    shift = scale[:, 1] & 0xFFFFFFFF
    shift = torch.where(shift >= 2 ** 31, shift - 2 ** 32, shift)
    return scale[:, 0].double() * _two(-shift)


def _rotate(x, value, pos, st):
    """x [n, heads, dim] int32 at positions pos: the rotated int64 codes and the rows' scale in float64."""
    c, tab = st["case"], st["rope"]
    y = x.to(torch.int64)
    if tab is None:
        return y, value
    half = c["rot"] // 2
    cs = tab[pos.clamp_min(0)].to(torch.int64)[:, None]
    co, si = cs[..., 0], cs[..., 1]
    out = y * 2 ** 30
    ia = torch.arange(half, device=x.device)
    ib = ia + half
    if c["rope"] == "pairs":
        ia, ib = 2 * ia, 2 * ia + 1
    a, b = y[..., ia], y[..., ib]
    out[..., ia] = a * co - b * si
    out[..., ib] = b * co + a * si
    return out, value * 2.0 ** -30


def _new_positions(st, b):
    new, kv = st["lens"][b]
    pos = torch.arange(kv - new, kv, device=st["table"].device)
    row0 = int(sum(n for n, _ in st["lens"][:b]))
    return pos, torch.arange(row0, row0 + new, device=pos.device)


def _places(st):
    """Of every new row of the batch: its position, pool page and place in the page."""
    begin, n = st["begin"].long(), st["rows"] - st["case"]["pad"]
    new = begin.diff()
    seq = torch.repeat_interleave(torch.arange(new.numel(), device=new.device), new, output_size=n)
    pos = torch.arange(n, device=new.device) - begin[seq + 1] + st["kv_len"][seq]
    ps = st["case"]["page"]
    return pos, st["table"][seq, pos // ps].long(), pos % ps


def _plain_write(st):
    c = st["case"]
    hk, d = c["kv_heads"], c["dim"]
    pos, page, place = _places(st)
    n = pos.numel()
    value = _value(st["scale"][:n])
    x = st["kv_in"][:n].view(n, 2, hk, d)
    for part, name, sc in ((0, "k", "ks"), (1, "v", "vs")):
        y, s = _rotate(x[:, 0], value, pos, st) if part == 0 else (x[:, 1].to(torch.int64), value)
        s = s[:, None]
        sg = _sigma(y.abs().amax(-1).double() * s / 127)
        st[name][page, :, place] = torch.round(y.double() * (s / sg)[..., None]).clamp(-127, 127).to(torch.int8)
        st[sc][page, :, place] = sg.to(torch.bfloat16)


def _plain_read(st):
    pos, page, place = _places(st)
    for name, sc, out in (("k", "ks", "ko"), ("v", "vs", "vo")):
        vals = st[name][page, :, place].float() * st[sc][page, :, place].float()[..., None]
        st[out][: pos.numel()] = vals.flatten(1)


def _weights(x, theta, seen):
    """The weights w_j (exact in float64) of rows x [.., keys] whose hidden keys are not ``seen``."""
    x = torch.where(seen, x, -math.inf)
    dist = x.amax(-1, keepdim=True) - x
    z = torch.round(dist.double() * theta * 1024)
    z = torch.where(seen, z.clamp_max(32768), 32768)
    n = torch.round(z / 1024)
    r = n - z / 1024
    e = (C3 * r + C2).float().double()
    e = (e * r + C1).float().double()
    e = (e * r + AMP).float().double()
    return torch.where(seen, e * _two(-n), 0)


def _plain_attend(st):
    c = st["case"]
    h, hk, d, ps = c["heads"], c["kv_heads"], c["dim"], c["page"]
    g = h // hk
    value = _value(st["scale"])
    soft = d ** -0.5 * LOG2E
    for b in range(c["seqs"]):
        new, kv = st["lens"][b]
        pos, row = _new_positions(st, b)
        y, s = _rotate(st["q"][row].view(new, h, d), value[row], pos, st)
        top = y.abs().amax(-1).double()
        q8 = torch.round(y.double() * (127 / top.clamp_min(1))[..., None])
        q8 = q8.view(new, hk, g, d).float()
        theta = (top * s[:, None] / 127 * soft).clamp_max(2.0 ** 60).float().double().view(new, hk, g)
        pages = st["table"][b, : -(-kv // ps)].long()
        key = torch.arange(kv, device=pos.device)
        step = max(1, 2 ** 26 // (g * kv))
        for i in range(hk):
            k8, v8 = (st[n][pages, i].reshape(-1, d)[:kv] for n in ("k", "v"))
            ks, vs = (st[n][pages, i].reshape(-1)[:kv] for n in ("ks", "vs"))
            for t in range(0, new, step):
                p = pos[t:t + step, None]
                seen = key <= p
                if c["window"]:
                    seen &= (key > p - c["window"]) | (key < c["sinks"])
                seen = seen[:, None]
                dots = q8[t:t + step, i].reshape(-1, d) @ k8.float().T
                x = (dots * ks.float()).view(-1, g, kv)
                w = _weights(x, theta[t:t + step, i, :, None], seen)
                m, e = torch.frexp(torch.where(seen, vs.double(), 0).amax(-1, keepdim=True))
                e = e - (m == 0.5).to(e.dtype)
                total = torch.round(w).sum(-1, keepdim=True)
                w = torch.round(w * (vs.double() * _two(-e)))
                o = torch.round((w.view(-1, kv) @ v8.double()).view(-1, g, d) * (2.0 ** 21 / total))
                rows = row[t:t + step]
                st["o"].view(-1, hk, g, d)[rows, i] = o.to(torch.int32)
                st["os"][rows, i, 0] = 1
                st["os"][rows, i, 1] = (21 - e[:, 0, 0]).to(torch.int64) & 0xFFFFFFFF


def run(st):
    c = st["case"]
    hk, d = c["kv_heads"], c["dim"]
    if not own:
        if c["kind"] == "attend":
            _plain_attend(st)
            return {"codes": st["o"], "scale": st["os"]}
        if c["kind"] == "write":
            _plain_write(st)
        _plain_read(st)
        return {"k": st["ko"], "v": st["vo"]}
    cache, batch = st["cache"], st["batch"]
    if c["kind"] == "attend":
        cache.attention(batch, st["q"], st["scale"], st["o"], st["os"], n_heads=c["heads"], rope=st["rot"],
                        window=c["window"], sinks=c["sinks"])
        return {"codes": st["o"], "scale": st["os"]}
    if c["kind"] == "write":
        x = st["kv_in"]
        cache.append(batch, x[:, : hk * d], x[:, hk * d:], st["scale"], rope=st["rot"])
    cache.read(batch, st["ko"], st["vo"])
    return {"k": st["ko"], "v": st["vo"]}


# ── the same from the definitions, in 64 bits ──


def _rn24(v):
    """v (float64) rounded to 24 significant bits, ties to even."""
    m, e = torch.frexp(v)
    return torch.round(m * 2.0 ** 24) * _two(e - 24)


def _exact_rotation(x, pos, c, tab):
    """[n, heads, dim] -> the rotated codes, element by element from its own partner."""
    n, h, d = x.shape
    x = x.long()
    if tab is None:
        return x
    half = c["rot"] // 2
    cols = []
    for i in range(d):
        if i >= c["rot"]:
            cols.append(x[:, :, i] << 30)
            continue
        j, first = (i // 2, i % 2 == 0) if c["rope"] == "pairs" else (i % half, i < half)
        mate = (i ^ 1) if c["rope"] == "pairs" else (i + half if first else i - half)
        co, si = tab[pos, j, 0].long()[:, None], tab[pos, j, 1].long()[:, None]
        cols.append(x[:, :, i] * co + x[:, :, mate] * (-si if first else si))
    return torch.stack(cols, -1)


def exact(c, seed):
    st = prepare(c, seed)
    dev, lens, hk, d, ps = st["table"].device, st["lens"], c["kv_heads"], c["dim"], c["page"]
    seq = torch.repeat_interleave(torch.arange(len(lens), device=dev), torch.tensor([n for n, _ in lens], device=dev))
    n = seq.numel()
    pos = torch.cat([torch.arange(kv - new, kv, device=dev) for new, kv in lens])
    page, place = st["table"][seq, pos // ps].long(), pos % ps
    if c["kind"] != "attend":
        out = {}
        for name, off in (("k", 0), ("v", hk * d)):
            res = torch.zeros(st["rows"], hk, d, dtype=torch.float64, device=dev)
            if c["kind"] == "read":
                res[:n] = st[name][page, :, place].double() * st[name + "s"][page, :, place].double()[..., None]
            else:
                x = st["kv_in"][:n, off:off + hk * d].view(n, hk, d)
                y = _exact_rotation(x, pos, c, st["rope"] if name == "k" else None)
                shift = st["scale"][:n, 1] << 32 >> 32
                if name == "k" and st["rope"] is not None:
                    shift = shift + 30
                s = (st["scale"][:n, 0].double() / _two(shift))[:, None]
                t = torch.maximum(y.amax(-1), -y.amin(-1)).double() * s / 127
                exp = torch.floor(torch.log2(t)) - 7
                # log2 may land on the wrong side of a power of two
                exp = torch.where(t >= _two(exp + 8), exp + 1, torch.where(t < _two(exp + 7), exp - 1, exp))
                sg = torch.ceil(t / _two(exp)) * _two(exp)
                res[:n] = torch.round(y.double() * (s / sg)[..., None]) * sg[..., None]
            out[name] = res.flatten(1)
        return out
    h = c["heads"]
    g = h // hk
    shift = st["scale"][:n, 1] << 32 >> 32
    if st["rope"] is not None:
        shift = shift + 30
    s = st["scale"][:n, 0].double() / _two(shift)
    y = _exact_rotation(st["q"][:n].view(n, h, d), pos, c, st["rope"])
    top = torch.maximum(y.amax(-1), -y.amin(-1)).double()
    q8 = torch.round(y.double() * (127 / top)[..., None])
    theta = _rn24((top * s[:, None] / 127) * (d ** -0.5 * LOG2E))
    del y
    codes = torch.zeros(st["rows"], h, d, dtype=torch.float64, device=dev)
    scales = torch.zeros(st["rows"], hk, 2, dtype=torch.int64, device=dev)
    for b, (new, kv) in enumerate(lens):
        mine = torch.nonzero(seq == b)[:, 0]
        j = torch.arange(kv, device=dev)
        where = st["table"][b, j // ps].long()
        step = max(1, 2 ** 25 // kv)
        for head in range(h):
            k = st["k"][where, head // g, j % ps].double()
            v = st["v"][where, head // g, j % ps].double()
            sk, sv = st["ks"][where, head // g, j % ps].double(), st["vs"][where, head // g, j % ps]
            bits = sv.view(torch.int16).long()
            up = (bits >> 7) - 127 + ((bits & 127) != 0).long()  # the least e with 2^e >= the scale
            sv = sv.double()
            for t in range(0, new, step):
                r = mine[t:t + step]
                p = pos[r][:, None]
                hidden = j > p
                if c["window"]:
                    hidden |= (j <= p - c["window"]) & (j >= c["sinks"])
                x = _rn24(q8[r, head] @ k.T * sk).masked_fill(hidden, -1e300)
                z = _rn24((x.amax(1, keepdim=True) - x).clamp_max(1e30)) * theta[r, head][:, None]
                z = torch.round(z * 1024).clamp_max(32768).long()
                nn = (z + 511 + ((z >> 10) & 1)) >> 10  # ties to the even side
                rr = (nn * 1024 - z).double() / 1024
                e = _rn24(_rn24(_rn24(rr * C3 + C2) * rr + C1) * rr + AMP)
                w = (e / (torch.ones_like(nn) << nn).double()).masked_fill(hidden, 0)
                ex = up.expand_as(hidden).masked_fill(hidden, -1000).amax(1, keepdim=True)
                total = torch.round(w).long().sum(1, keepdim=True)
                num = torch.round(w * sv / _two(ex)) @ v
                codes[r, head] = torch.round(num * (2097152 / total.double()))
                scales[r, head // g] = torch.stack([torch.ones_like(ex[:, 0]), 21 - ex[:, 0]], -1) & torch.tensor([-1, 0xFFFFFFFF], device=dev)
    return {"codes": codes.flatten(1), "scale": scales}
