"""The 8-bit paged KV cache and the attention over it, against plain 64-bit forms of their definition.

Tolerances.  Codes and scales are compared for equality: rows are bf16, scales powers of two, so x / s is exact and the only rounding is the one
to e4m3.  The fused step's slabs and rotation tables are numbers of few bits, so that its sums and products are exact in 32 bits too.
Attention, per output element: probabilities rounded to bf16 move the weighted sum by at most half a bf16 step of sum p |v|, the output's own
rounding is half a step of |o|.  Scores are sums of D products in 32 bits, then scaled and made powers of two: off by at most
(D + 8) 2^-24 of scale * sum |q k|, which moves a probability and the sum that divides it by that much, relative; sums over m tokens add m
2^-24 each.  ``attend`` returns sum p |v| and that relative error, taken at the row's largest sum |q k|.
"""
import itertools
import math

import pytest
import torch

from k8s_llm_monitor_amd import ops
from k8s_llm_monitor_amd.ops import kv8

HALF_STEP = torch.finfo(torch.bfloat16).eps / 2
NAN_CODE = 0x7F


# ---------------------------------------------------------------- the definition, in 64 bits

def code_value(y):
    """The e4m3 number nearest to y, halves to even, as a float64 (|y| <= 448)."""
    e = torch.floor(torch.log2(y.abs().clamp_min(2.0 ** -30))).clamp_min(-6)
    step = torch.exp2(e - 3)
    return torch.round(y / step) * step


def least_scale(amax):
    return max(2.0 ** -100, 2.0 ** math.ceil(math.log2(amax / 448.0))) if amax > 0 else 2.0 ** -100


class Book:
    """A cache as numbers: [pages, Hkv, 16, D] values of codes, [pages, Hkv] scales, for keys and for values."""

    def __init__(self, cache):
        self.n, self.hkv = cache.scales.shape[:2]
        self.D = cache.v.shape[2]
        k = cache.k.cpu().view(torch.uint8).view(kv8.E4M3).double()
        v = cache.v.cpu().view(torch.uint8).view(kv8.E4M3).double()
        self.codes = [k.permute(0, 1, 3, 2, 4).reshape(self.n, self.hkv, 16, self.D), v.transpose(2, 3).clone()]
        self.scales = [cache.scales[..., j].cpu().double().clone() for j in (0, 1)]

    def write(self, slots, k, v):
        """k, v [T, Hkv, D] float64, one row after the other, page by page."""
        slots = slots.tolist()
        t = 0
        while t < len(slots):
            if not 0 <= slots[t] < self.n * 16:
                t += 1
                continue
            n = 1
            while t + n < len(slots) and slots[t + n] == slots[t] + n and slots[t + n] % 16:
                n += 1
            page, off = divmod(slots[t], 16)
            for j, x in enumerate((k[t:t + n], v[t:t + n])):
                for h in range(self.hkv):
                    fine = x[:, h][x[:, h].isfinite()]
                    s = least_scale(float(fine.abs().max()) if fine.numel() else 0.0)
                    old = float(self.scales[j][page, h])
                    if off:
                        s = max(s, old)
                        if s != old:
                            self.codes[j][page, h, :off] = code_value(self.codes[j][page, h, :off] * (old / s))
                    y = x[:, h]
                    self.codes[j][page, h, off:off + n] = torch.where(y.isfinite(), code_value(torch.where(y.isfinite(), y, 0.0) / s), math.nan)
                    self.scales[j][page, h] = s
            t += n

    def tokens(self, pages, n):
        p = [min(max(int(x), 0), self.n - 1) for x in pages[: (n + 15) // 16]]
        return [(c[p] * s[p][..., None, None]).transpose(1, 2).reshape(-1, self.hkv, self.D)[:n] for c, s in zip(self.codes, self.scales)]

    def check(self, cache):
        now = Book(cache)
        for j in (0, 1):
            assert torch.equal(now.scales[j], self.scales[j]), f"scales {j}"
            a, b = now.codes[j], self.codes[j]
            assert torch.equal(a.isnan(), b.isnan()) and torch.equal(a.nan_to_num(), b.nan_to_num()), f"codes {j}"


def attend(q, k, v, scale, first):
    """q [n, Hq, D] at positions first.., k / v [m, Hkv, D]: (output, what it may be off by), each [n, Hq * D]."""
    n, hq, d = q.shape
    out, off = torch.empty_like(q), torch.empty_like(q)
    for h in range(hq):
        kh, vh = k[:, h // (hq // k.shape[1])], v[:, h // (hq // k.shape[1])]
        for i in range(n):
            m = first + i + 1
            p = torch.softmax(kh[:m] @ q[i, h] * scale, 0)
            rel = 2 * (d + 8) * 2.0 ** -24 * scale * float((kh[:m].abs() @ q[i, h].abs()).max()) + 2 * m * 2.0 ** -24 + 2.0 ** -20
            out[i, h] = p @ vh[:m]
            off[i, h] = (HALF_STEP + rel) * (p @ vh[:m].abs()) * (1 + HALF_STEP) + HALF_STEP * out[i, h].abs()
    return out.reshape(n, -1), off.reshape(n, -1)


def check_attention(got, want, off):
    got = got.cpu().double()
    assert torch.equal(got.isnan(), want.isnan())
    ok = ~want.isnan()
    err = ((got - want).abs() / (off + 2.0 ** -120))[ok]
    assert bool((err <= 1).all()), f"off by {float(err.max()):.3f} of the bound"


# ---------------------------------------------------------------- inputs

DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]


def rand(gen, *shape, spread=0.0):
    x = torch.randn(*shape, generator=gen)
    return x * torch.exp(spread * torch.randn(*shape[:-1], 1, generator=gen)) if spread else x


def garbage(cache, gen):
    """Pages as earlier users may have left them: any code, NaN among them, any scale."""
    cache.k.view(torch.uint8).copy_(torch.randint(0, 256, cache.k.shape, generator=gen, dtype=torch.uint8))
    cache.v.view(torch.uint8).copy_(torch.randint(0, 256, cache.v.shape, generator=gen, dtype=torch.uint8))
    cache.scales.copy_(torch.exp2(torch.randint(-20, 20, cache.scales.shape, generator=gen).float()))


def filled(gen, dev, lens, hkv, d, spare=2, spread=1.0):
    """(cache, table [S, W], Book): sequences of these lengths, written through the operator, pages shuffled, the rest garbage."""
    need = [(n + 15) // 16 for n in lens]
    cache = ops.kv8_cache(sum(need) + spare, hkv, d, device=dev)
    garbage(cache, gen)
    order = torch.randperm(sum(need) + spare, generator=gen)
    table = torch.full((len(lens), max(1, max(need))), -7, dtype=torch.int32)
    at = 0
    for i, k in enumerate(need):
        table[i, :k] = order[at:at + k].int()
        at += k
    book = Book(cache)
    T = sum(lens)
    rows = rand(gen, T, 2 * hkv, d, spread=spread).bfloat16()
    slots = torch.cat([table[i, :need[i]].repeat_interleave(16)[:n] * 16 + torch.arange(n, dtype=torch.int32) % 16 for i, n in enumerate(lens)])
    if T:
        qkv = torch.cat([torch.zeros(T, hkv, d, dtype=torch.bfloat16), rows], 1).reshape(T, -1).to(dev)
        ops.rope_and_cache_kv8(qkv, no_positions(T, dev), table_of(d, dev), cache, slots.to(dev), hkv, hkv, d, apply_rope=False)
        book.write(slots, rows[:, :hkv].double(), rows[:, hkv:].double())
    return cache, table, book


def no_positions(T, dev):
    return torch.zeros(T, dtype=torch.int32, device=dev)


def table_of(d, dev, n=4096):
    """A rotation table of numbers of seven bits: products with bf16 numbers, and their sums, are exact in 32 bits."""
    a = torch.arange(n, dtype=torch.float64)[:, None] * 10000.0 ** (-torch.arange(d // 2, dtype=torch.float64) * 2 / d)
    return (torch.round(torch.cat([a.cos(), a.sin()], 1) * 64) / 64).float().to(dev)


# ---------------------------------------------------------------- the write

@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("hkv", [1, 3, 8])
def test_write_whole_ragged_and_appended(dev, d, hkv):
    gen = torch.Generator().manual_seed(d + hkv)
    lens = [1, 15, 16, 17, 33, 80]
    cache, table, book = filled(gen, dev, lens, hkv, d)
    book.check(cache)
    # chunks that go on inside a page, larger and smaller than what is there; rows without a slot between them
    for size, more in ((1.0, [1, 1, 16, 14, 1, 5]), (300.0, [3, 16, 1, 1, 20, 31]), (0.001, [1] * 6)):
        rows, slots, at = [], [], sum((n + 15) // 16 for n in lens)
        pages = [table[i, : (n + 15) // 16].tolist() for i, n in enumerate(lens)]
        n_pages = sum((n + m + 15) // 16 for n, m in zip(lens, more)) + 1
        bigger = ops.kv8_cache(n_pages, hkv, d, device=dev)
        garbage(bigger, gen)
        new_table, used = [], 0
        order = torch.randperm(n_pages, generator=gen).tolist()
        for i, (n, m) in enumerate(zip(lens, more)):
            want = (n + m + 15) // 16
            mine = order[used:used + want]
            used += want
            for a, b in zip(pages[i], mine):
                for x, y in zip(bigger, cache):
                    (x.view(torch.uint8) if x.dtype == kv8.E4M3 else x)[b] = (y.view(torch.uint8) if y.dtype == kv8.E4M3 else y)[a]
            new_table.append(mine)
            slots += [mine[(n + j) // 16] * 16 + (n + j) % 16 for j in range(m)] + [-1]
        T = len(slots)
        x = (rand(gen, T, 3 * hkv, d, spread=1.0) * size).bfloat16()
        book = Book(bigger)
        sl = torch.tensor(slots, dtype=torch.int32)
        ops.rope_and_cache_kv8(x.reshape(T, -1).to(dev), no_positions(T, dev), table_of(d, dev), bigger, sl.to(dev), hkv, hkv, d, apply_rope=False)
        book.write(sl, x[:, hkv:2 * hkv].double(), x[:, 2 * hkv:].double())
        book.check(bigger)


@pytest.mark.parametrize("dev", DEVICES)
def test_write_every_magnitude(dev):
    """amax at, just below and just above 448 times a power of two; zero rows; the smallest and largest numbers; ties of the rounding."""
    hkv, d = 1, 64
    edge = [448.0, 446.0, 450.0, 1.0, 0.0, 2.0 ** -126, 3.0e38, 2.0 ** -133, 1.75, 1.7578125, 17.0 / 16, 19.0 / 16]
    T = 16 * len(edge)
    x = torch.zeros(T, 3, d)
    for i, e in enumerate(edge):
        x[16 * i:16 * i + 16] = e * torch.linspace(-1, 1, 16 * 3 * d).view(16, 3, d).bfloat16().float()
        x[16 * i + 7, 1:, 5] = e
    x = x.bfloat16()
    cache = ops.kv8_cache(len(edge), hkv, d, device=dev)
    book = Book(cache)
    slots = torch.arange(T, dtype=torch.int32)
    ops.rope_and_cache_kv8(x.reshape(T, -1).to(dev), no_positions(T, dev), table_of(d, dev), cache, slots.to(dev), 1, hkv, d, apply_rope=False)
    book.write(slots, x[:, 1:2].double(), x[:, 2:].double())
    book.check(cache)


@pytest.mark.parametrize("dev", DEVICES)
def test_write_numbers_that_are_not_finite(dev):
    hkv, d = 2, 128
    gen = torch.Generator().manual_seed(9)
    x = rand(gen, 20, 3 * hkv, d).bfloat16()
    x[3, hkv, 7], x[4, hkv + 1, 0], x[5, 2 * hkv, 127], x[18, 3 * hkv - 1, 64] = math.nan, math.inf, -math.inf, math.nan
    x[9, hkv] = math.inf  # a token without one finite number
    cache = ops.kv8_cache(3, hkv, d, device=dev)
    book = Book(cache)
    slots = torch.arange(16, 36, dtype=torch.int32)
    ops.rope_and_cache_kv8(x.reshape(20, -1).to(dev), no_positions(20, dev), table_of(d, dev), cache, slots.to(dev), hkv, hkv, d, apply_rope=False)
    book.write(slots, x[:, hkv:2 * hkv].double(), x[:, 2 * hkv:].double())
    book.check(cache)
    assert int(Book(cache).codes[0].isnan().sum()) == 2 + d


@pytest.mark.parametrize("dev", DEVICES)
def test_write_leaves_everything_else(dev):
    """Slots outside the cache are skipped; other pages, and tokens behind a run in its own page, keep every bit."""
    hkv, d = 2, 64
    gen = torch.Generator().manual_seed(10)
    cache = ops.kv8_cache(5, hkv, d, device=dev)
    garbage(cache, gen)
    before = [t.clone().view(torch.uint8).cpu() for t in (cache.k, cache.v)]
    x = rand(gen, 6, 3 * hkv, d).bfloat16()
    slots = torch.tensor([-1, 80, 1 << 30, 33, 34, -5], dtype=torch.int32)
    ops.rope_and_cache_kv8(x.reshape(6, -1).to(dev), no_positions(6, dev), table_of(d, dev), cache, slots.to(dev), hkv, hkv, d, apply_rope=False)
    k, v = (t.view(torch.uint8).cpu() for t in (cache.k, cache.v))
    others = [0, 1, 3, 4]
    assert torch.equal(k[others], before[0][others]) and torch.equal(v[others], before[1][others])
    assert torch.equal(k[2, :, :, 3:], before[0][2, :, :, 3:]) and torch.equal(v[2, :, :, 3:], before[1][2, :, :, 3:])


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("T", [5, 700])
def test_write_many_rows_rotated_and_from_slabs(dev, T):
    """The rows in the cache are the rows that the call leaves in qkv: summed from slabs, rotated."""
    hq, hkv, d = 4, 2, 128
    gen = torch.Generator().manual_seed(T)
    n = (hq + 2 * hkv) * d
    slabs = torch.randn(3, T, n, generator=gen).to(dev)
    qkv = torch.empty(T, n, dtype=torch.bfloat16, device=dev)
    cache = ops.kv8_cache(T // 16 + 2, hkv, d, device=dev)
    book = Book(cache)
    slots = torch.arange(5, 5 + T, dtype=torch.int32)
    pos = torch.arange(T, dtype=torch.int32, device=dev)
    cs = table_of(d, dev)
    ops.rope_and_cache_kv8(qkv, pos, cs, cache, slots.to(dev), hq, hkv, d, partial=slabs, nslabs=3)
    want = slabs.cpu().double().sum(0).view(T, -1, d)
    c, s = cs.cpu().double()[pos.cpu().long()].view(T, 1, 2, d // 2).unbind(2)
    a, b = want[:, : hq + hkv].split(d // 2, -1)
    want[:, : hq + hkv] = torch.cat([a * c - b * s, b * c + a * s], -1)
    x = qkv.cpu().double().view(T, -1, d)
    # the slab sum's rounding, then the rotated value's: half a step of each, on numbers of size sqrt(a^2 + b^2) <= 2^4
    assert float((x - want).abs().max()) <= 2 * HALF_STEP * 16 * math.sqrt(2)
    book.write(slots, x[:, hq:hq + hkv], x[:, hq + hkv:])
    book.check(cache)


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("T", [513, 2049, 4097, 5003])
def test_write_of_large_steps(dev, d, T):
    """Row counts on both sides of where a wave takes 2, 8 and 16 of them: sequences of 1 to 60 rows that begin anywhere in a page, so that
    runs lie across every border of 8 and 16 rows, rows without a slot between some of them, the last sequence cut by the end."""
    hkv = 2
    gen = torch.Generator().manual_seed(T + d)
    at = lambda n: int(torch.randint(0, n, (1,), generator=gen))  # noqa: E731
    slots, page = [], 0
    while len(slots) < T:
        n, first = 1 + at(60), at(16)
        slots += range(page * 16 + first, page * 16 + first + n)
        page += (first + n + 15) // 16
        slots += [-1] * (at(4) if at(3) == 0 else 0)
    order = torch.randperm(page, generator=gen)
    slots = torch.tensor([-1 if s < 0 else int(order[s // 16]) * 16 + s % 16 for s in slots[:T]], dtype=torch.int32)
    cache = ops.kv8_cache(page, hkv, d, device=dev)
    garbage(cache, gen)
    book = Book(cache)
    x = rand(gen, T, 3 * hkv, d, spread=1.0).bfloat16()
    wide = torch.zeros(T, 3 * hkv * d + 8, dtype=torch.bfloat16)
    wide[:, : 3 * hkv * d] = x.view(T, -1)
    ops.rope_and_cache_kv8(wide.to(dev), None, None, cache, slots.to(dev), hkv, hkv, d, apply_rope=False)
    book.write(slots, x[:, hkv:2 * hkv].double(), x[:, 2 * hkv:].double())
    book.check(cache)


def test_write_refuses_rows_out_of_order_on_the_cpu():
    cache = ops.kv8_cache(4, 1, 64)
    qkv = torch.zeros(3, 192, dtype=torch.bfloat16)
    for slots in ([1, 0, 2], [0, 2, 1], [0, 16, 1], [3, 3, 4], [0, 2, 3]):
        with pytest.raises(ValueError, match="follow one another"):
            ops.rope_and_cache_kv8(qkv, no_positions(3, "cpu"), table_of(64, "cpu"), cache, torch.tensor(slots, dtype=torch.int32), 1, 1, 64,
                                   apply_rope=False)


@pytest.mark.parametrize("dev", DEVICES)
def test_write_of_positions_outside_the_table(dev):
    """Positions are held to the rotation table's ends, in the write and in the fused step."""
    hq, hkv, d, n = 2, 1, 128, 20
    gen = torch.Generator().manual_seed(13)
    raw = (torch.randn(4, hq + 2 * hkv, d, generator=gen)).bfloat16()
    slots, cs = torch.tensor([0, 1, 16, 32], dtype=torch.int32, device=dev), table_of(d, dev, n)
    out = []
    for pos in ([-5, 19, 1 << 30, -(1 << 31)], [0, 19, 19, 0]):
        cache, qkv = ops.kv8_cache(4, hkv, d, device=dev), raw.clone().view(4, -1).to(dev)
        ops.rope_and_cache_kv8(qkv, torch.tensor(pos, dtype=torch.int32, device=dev), cs, cache, slots, hq, hkv, d)
        step = ops.kv8_cache(4, hkv, d, device=dev)
        o = ops.paged_decode_fused_kv8(raw.float().view(1, 4, -1).to(dev), 1, torch.tensor(pos, dtype=torch.int32, device=dev), cs,
                                       torch.tensor([0, 16, 32, 48], dtype=torch.int32, device=dev), step,
                                       torch.arange(4, dtype=torch.int32, device=dev)[:, None], torch.ones(4, dtype=torch.int32, device=dev), hq, hkv, d, 0.1)
        out.append([qkv, cache.k.view(torch.uint8), cache.v.view(torch.uint8), o, step.k.view(torch.uint8)])
    assert all(torch.equal(a, b) for a, b in zip(*out))


@pytest.mark.parametrize("dev", DEVICES)
def test_a_refused_write_changes_nothing(dev):
    """Arguments are looked at before the rows are summed and rotated."""
    hq, hkv, d = 2, 1, 128
    rows = torch.randn(3, (hq + 2 * hkv) * d, generator=torch.Generator().manual_seed(14)).bfloat16().to(dev)
    pos, cs = torch.tensor([5, 6, 7], dtype=torch.int32, device=dev), table_of(d, dev)
    i32 = lambda *v: torch.tensor(v, dtype=torch.int32, device=dev)  # noqa: E731
    bad = [dict(slots=i32(0, 1))] + ([dict(slots=i32(1, 0, 2))] if dev == "cpu" else
                                     [dict(cache=ops.kv8_cache(2, 3, d, device=dev)), dict(pos=pos[:2]), dict(cs=cs[:, :64]), dict(slots=i32(0, 1, 2).long())])
    for k in bad:
        for partial in (None, torch.ones(2, *rows.shape, device=dev)):
            k = {**dict(slots=i32(0, 1, 2), cache=ops.kv8_cache(2, hkv, d, device=dev), pos=pos, cs=cs), **k}
            qkv = rows.clone()
            with pytest.raises((RuntimeError, ValueError)):
                ops.rope_and_cache_kv8(qkv, k["pos"], k["cs"], k["cache"], k["slots"], hq, hkv, d, partial=partial, nslabs=2)
            assert torch.equal(qkv, rows)


# ---------------------------------------------------------------- single tokens

SHAPES = [(1, 1, 128), (8, 8, 64), (32, 8, 128), (7, 1, 128), (28, 4, 128), (16, 1, 64), (10, 2, 64)]


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("hq,hkv,d", SHAPES)
def test_decode(dev, hq, hkv, d):
    gen = torch.Generator().manual_seed(hq * 131 + d)
    lens = [1, 0, 16, 63, 64, 65, 255, 256, 257, 700]
    cache, table, book = filled(gen, dev, lens, hkv, d)
    q = rand(gen, len(lens), hq, d).bfloat16()
    wide = torch.zeros(len(lens), hq * d + 64, dtype=torch.bfloat16)
    wide[:, : hq * d] = q.view(len(lens), -1)
    sl = torch.tensor(lens, dtype=torch.int32)
    scale = 1 / math.sqrt(d)
    want = [attend(q[i:i + 1].double(), *book.tokens(table[i], n), scale, n - 1) if n else (torch.zeros(1, hq * d, dtype=torch.double),) * 2
            for i, n in enumerate(lens)]
    want, size = (torch.cat(x) for x in zip(*want))
    ws = ops.decode_workspace(len(lens), hq, d, device=dev)
    for splits, w in ((None, None), (1, None), (3, None), (3, ws), (2, ws), (64, ws)):
        got = ops.paged_decode_kv8(wide.to(dev), cache, table.to(dev), sl.to(dev), hq, hkv, d, scale, workspace=w, splits=splits)
        check_attention(got, want, size)
    if dev == "cuda":  # the row stride, the packed form, and counters left at zero
        assert int(ws[2].abs().sum()) == 0
        out = torch.full((len(lens), hq * d + 8), 7.0, dtype=torch.bfloat16, device=dev)
        ops.paged_decode_kv8(wide.to(dev), cache, table.to(dev), sl.to(dev), hq, hkv, d, scale, out=out[:, : hq * d])
        check_attention(out[:, : hq * d], want, size)
        assert bool((out[:, hq * d:] == 7).all())
    if hq * d % 32 == 0:
        p = ops.packed_empty(len(lens), hq * d, torch.bfloat16, dev)
        p.zero_()
        ops.paged_decode_kv8(wide.to(dev), cache, table.to(dev), sl.to(dev), hq, hkv, d, scale, out=p)
        check_attention(ops.unpack_skinny(p.cpu())[: len(lens)], want, size)


@pytest.mark.parametrize("dev", DEVICES)
def test_decode_of_bad_pages_and_lengths(dev):
    """Page numbers outside the cache are held to its ends; a length behind the block table ends with it."""
    hq = hkv = 2
    d = 64
    gen = torch.Generator().manual_seed(3)
    cache, table, book = filled(gen, dev, [64, 64], hkv, d, spare=0)
    table = torch.tensor([[-3, 1 << 30, 2, -(1 << 31)], [7, 3, 99, 1]], dtype=torch.int32)
    q = rand(gen, 2, hq, d).bfloat16()
    lens = torch.tensor([61, 1000], dtype=torch.int32)
    got = ops.paged_decode_kv8(q.view(2, -1).to(dev), cache, table.to(dev), lens.to(dev), hq, hkv, d, 0.125)
    want = [attend(q[i:i + 1].double(), *book.tokens(table[i], n), 0.125, n - 1) for i, n in ((0, 61), (1, 64))]
    check_attention(got, *(torch.cat(x) for x in zip(*want)))


@pytest.mark.gpu
def test_decode_replays_in_a_graph_and_beside_another_stream():
    gen = torch.Generator().manual_seed(4)
    hq, hkv, d, lens = 8, 2, 128, [5, 600, 333]
    cache, table, book = filled(gen, "cuda", lens, hkv, d)
    q = torch.zeros(3, hq * d, dtype=torch.bfloat16, device="cuda")
    sl, table_d = torch.tensor(lens, dtype=torch.int32, device="cuda"), table.cuda()
    out = torch.empty(3, hq * d, dtype=torch.bfloat16, device="cuda")
    ws = ops.decode_workspace(3, hq, d, device="cuda")
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        ops.paged_decode_kv8(q, cache, table_d, sl, hq, hkv, d, 0.1, workspace=ws, out=out, splits=3)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        ops.paged_decode_kv8(q, cache, table_d, sl, hq, hkv, d, 0.1, workspace=ws, out=out, splits=3)
    for k in range(4):
        x = rand(gen, 3, hq, d).bfloat16()
        q.copy_(x.view(3, -1))
        g.replay()
        torch.cuda.synchronize()
        eager = ops.paged_decode_kv8(q, cache, table_d, sl, hq, hkv, d, 0.1, splits=3)
        want = [attend(x[i:i + 1].double(), *book.tokens(table[i], n), 0.1, n - 1) for i, n in enumerate(lens)]
        check_attention(out, *(torch.cat(w) for w in zip(*want)))
        check_attention(eager, *(torch.cat(w) for w in zip(*want)))


# ---------------------------------------------------------------- the fused step

@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("hq,hkv", [(1, 1), (4, 2), (32, 8), (7, 1), (16, 1), (28, 4)])
@pytest.mark.parametrize("size", [1.0, 64.0, 2.0 ** -12])
def test_fused_step(dev, hq, hkv, size):
    """New tokens at every kind of place: a page's first, middle and last, chunk borders, a context of nothing; scales that grow and do not;
    rows without a slot and rows of length 0.  The cache's codes and scales are exact."""
    d, nslabs = 128, 3
    gen = torch.Generator().manual_seed(int(hq * 10 + size))
    before = [0, 1, 15, 16, 17, 47, 255, 256, 600, 40, 0]
    B = len(before)
    lens = [n + 1 for n in before]
    cache, table, book = filled(gen, dev, before, hkv, d, spare=B)
    free = [p for p in range(book.n) if p not in set(table.flatten().tolist())]
    table = torch.cat([table, torch.full((B, 1), -7, dtype=torch.int32)], 1)
    for i, n in enumerate(before):
        if n % 16 == 0:
            table[i, n // 16] = free.pop()
    slots = torch.tensor([int(table[i, n // 16]) * 16 + n % 16 for i, n in enumerate(before)], dtype=torch.int32)
    slots[9] = -1  # attended but not written
    lens[10] = 0   # a graph bucket's slack
    slots[10] = -1
    cols = (hq + 2 * hkv) * d
    slabs = torch.round(torch.randn(nslabs, B, cols, generator=gen) * 32) / 32 * size
    pos = torch.tensor(before, dtype=torch.int32)
    cs = table_of(d, dev)
    x = slabs.double().sum(0).bfloat16().double().view(B, -1, d)
    c, s = cs.cpu().double()[pos.long()].view(B, 1, 2, d // 2).unbind(2)
    a, b = x[:, : hq + hkv].split(d // 2, -1)
    rot = torch.cat([a * c - b * s, b * c + a * s], -1).bfloat16().double()
    q, k, v = rot[:, :hq], rot[:, hq:], x[:, hq + hkv:]
    book.write(slots, k, v)
    scale = 1 / math.sqrt(d) / size ** 2 if size > 1 else 1 / math.sqrt(d)
    want = []
    for i, n in enumerate(lens):
        if n == 0:
            want.append((torch.zeros(1, hq * d, dtype=torch.double),) * 2)
            continue
        kk, vv = book.tokens(table[i], n)
        if slots[i] < 0:
            for t, y in ((kk, k[i]), (vv, v[i])):
                for h in range(hkv):
                    sc = least_scale(float(y[h].abs().max()))
                    t[n - 1, h] = code_value(y[h] / sc) * sc
        want.append(attend(q[i:i + 1], kk, vv, scale, n - 1))
    want, weight = (torch.cat(w) for w in zip(*want))
    sl, tb = torch.tensor(lens, dtype=torch.int32, device=dev), table.to(dev)
    ws = ops.decode_workspace(B, hq, d, device=dev)
    for splits, w in ((1, None), (3, ws), (3, None), (64, ws), (None, ws)):  # writing the same token again changes nothing
        got = ops.paged_decode_fused_kv8(slabs.to(dev), nslabs, pos.to(dev), cs, slots.to(dev), cache, tb, sl, hq, hkv, d, scale, workspace=w,
                                         splits=splits)
        check_attention(got, want, weight)
        book.check(cache)
    if dev == "cuda":
        assert int(ws[2].abs().sum()) == 0


@pytest.mark.parametrize("dev", DEVICES)
def test_fused_step_goes_on_as_the_chunked_write_does(dev):
    """Forty tokens one step at a time leave the codes and scales that the definition says, page after page."""
    hq, hkv, d = 4, 2, 128
    gen = torch.Generator().manual_seed(12)
    cache = ops.kv8_cache(4, hkv, d, device=dev)
    garbage(cache, gen)
    book = Book(cache)
    table = torch.tensor([[2, 0, 3]], dtype=torch.int32)
    cs = torch.cat([torch.ones(64, d // 2), torch.zeros(64, d // 2)], 1).to(dev)  # no rotation
    for t in range(40):
        slabs = torch.round(torch.randn(1, 1, (hq + 2 * hkv) * d, generator=gen) * 16 * 2.0 ** (t % 7)) / 16
        x = slabs[0].bfloat16().double().view(1, -1, d)
        slot = torch.tensor([int(table[0, t // 16]) * 16 + t % 16], dtype=torch.int32)
        pos = torch.tensor([t], dtype=torch.int32)
        scale = 2.0 ** -14  # (keys grow up to 2^7)
        got = ops.paged_decode_fused_kv8(slabs.to(dev), 1, pos.to(dev), cs, slot.to(dev), cache, table.to(dev), (pos + 1).to(dev), hq, hkv, d, scale)
        book.write(slot, x[:, hq:hq + hkv], x[:, hq + hkv:])
        book.check(cache)
        check_attention(got, *attend(x[:, :hq], *book.tokens(table[0], t + 1), scale, t))


# ---------------------------------------------------------------- prompt chunks

@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("hq,hkv,d", SHAPES)
def test_prefill(dev, hq, hkv, d):
    gen = torch.Generator().manual_seed(hq * 7 + d)
    ctx, new = [0, 0, 5, 64, 130, 17, 0], [1, 70, 3, 64, 150, 1, 0]
    cache, table, book = filled(gen, dev, [a + b for a, b in zip(ctx, new)], hkv, d)
    T = sum(new)
    q = rand(gen, T + 2, hq, d).bfloat16()  # two rows behind the last sequence
    wide = torch.zeros(T + 2, (hq + 2 * hkv) * d, dtype=torch.bfloat16)
    wide[:, : hq * d] = q.view(T + 2, -1)
    cu = torch.tensor([0, *itertools.accumulate(new)], dtype=torch.int32)
    scale = 1 / math.sqrt(d)
    want = [attend(q[int(cu[i]):int(cu[i + 1])].double(), *book.tokens(table[i], a + b), scale, a) for i, (a, b) in enumerate(zip(ctx, new)) if b]
    want, size = (torch.cat(w) for w in zip(*want))
    out = torch.full((T + 2, hq * d + 8), 7.0, dtype=torch.bfloat16, device=dev)[:, : hq * d]
    got = ops.flash_prefill_kv8(wide.to(dev), cu.to(dev), torch.tensor(ctx, dtype=torch.int32, device=dev), cache, table.to(dev), hq, hkv, d, scale,
                                out=out)
    check_attention(got[:T], want, size)
    assert bool((out[T:] == 7).all())


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("width,ctx,new", [(1, 0, 40), (3, 0, 49), (2, 9, 300), (5, 70, 30), (20, 300, 40)])
def test_prefill_of_chunks_longer_than_their_table(dev, d, width, ctx, new):
    """The table ends the sequence: a context that does not fit is cut, rows behind the end see all that the table holds, and nothing twice."""
    hq, hkv = 4, 2
    gen = torch.Generator().manual_seed(width + new)
    n = 16 * width
    cache, table, book = filled(gen, dev, [n], hkv, d)
    q = rand(gen, new, hq, d).bfloat16()
    i32 = lambda *v: torch.tensor(v, dtype=torch.int32, device=dev)  # noqa: E731
    got = ops.flash_prefill_kv8(q.view(new, -1).to(dev), i32(0, new), i32(ctx), cache, table.to(dev), hq, hkv, d, 0.1)
    fit = min(new, n)
    k, v = book.tokens(table[0], n)
    first = max(0, min(ctx, n - fit))
    want = [attend(q[:fit].double(), k, v, 0.1, first)] + [attend(q[i:i + 1].double(), k, v, 0.1, n - 1) for i in range(fit, new)]
    check_attention(got, *(torch.cat(w) for w in zip(*want)))


@pytest.mark.parametrize("dev", DEVICES)
def test_prefill_few_rows_behind_a_long_context(dev):
    """One split of keys each: 3 and 40 rows behind contexts of 2000 and 9 tokens."""
    hq, hkv, d = 8, 2, 128
    gen = torch.Generator().manual_seed(21)
    ctx, new = [2000, 9, 777], [3, 40, 1]
    cache, table, book = filled(gen, dev, [a + b for a, b in zip(ctx, new)], hkv, d)
    q = rand(gen, sum(new), hq, d).bfloat16()
    cu = torch.tensor([0, *itertools.accumulate(new)], dtype=torch.int32)
    got = ops.flash_prefill_kv8(q.view(sum(new), -1).to(dev), cu.to(dev), torch.tensor(ctx, dtype=torch.int32, device=dev), cache, table.to(dev), hq,
                                hkv, d, 0.1)
    want = [attend(q[int(cu[i]):int(cu[i + 1])].double(), *book.tokens(table[i], a + b), 0.1, a) for i, (a, b) in enumerate(zip(ctx, new))]
    check_attention(got, *(torch.cat(w) for w in zip(*want)))


@pytest.mark.gpu
@pytest.mark.parametrize("ctx,new", [(0, 200), (50, 100), (1500, 20)])
def test_prefill_nan_counts_for_rows_that_see_it(ctx, new):
    """NaN keys and values: rows before their token are what they are without it, rows from it on are NaN (values: in that dim)."""
    hq, hkv, d = 4, 1, 128
    gen = torch.Generator().manual_seed(ctx + new)
    n = ctx + new
    cache, table, book = filled(gen, "cuda", [n], hkv, d)
    bad_v, bad_k = ctx + new // 3, ctx + new - 5
    page, off = int(table[0, bad_v // 16]), bad_v % 16
    cache.v.view(torch.uint8)[page, 0, 77, off] = NAN_CODE
    cache.v.view(torch.uint8)[page, 0, 3, off] = 0xFF
    page, off = int(table[0, bad_k // 16]), bad_k % 16
    cache.k.view(torch.uint8)[page, 0, 2, off, 9] = NAN_CODE
    book2 = Book(cache)
    q = rand(gen, new, hq, d).bfloat16()
    cu = torch.tensor([0, new], dtype=torch.int32)
    got = ops.flash_prefill_kv8(q.view(new, -1).cuda(), cu.cuda(), torch.tensor([ctx], dtype=torch.int32).cuda(), cache, table.cuda(), hq, hkv, d, 0.1)
    want, size = attend(q.double(), *book2.tokens(table[0], n), 0.1, ctx)
    _, size = attend(q.double(), *book.tokens(table[0], n), 0.1, ctx)
    assert bool(want.isnan().any()) and not bool(want[: new // 3].isnan().any())
    check_attention(got, want, size)


@pytest.mark.parametrize("dev", DEVICES)
def test_prefill_leaves_rows_that_no_block_names(dev):
    """Of the rows ahead of the first sequence, of a sequence without a block and of one whose blocks are named in part, nothing is written."""
    hq, hkv, d = 4, 2, 128
    gen = torch.Generator().manual_seed(22)
    new = [140, 20, 300]
    cache, table, book = filled(gen, dev, new, hkv, d)
    ahead = 3
    q = rand(gen, ahead + sum(new), hq, d).bfloat16()
    cu = torch.tensor([ahead + n for n in (0, *itertools.accumulate(new))], dtype=torch.int32)
    i32 = lambda *v: torch.tensor(v, dtype=torch.int32, device=dev)  # noqa: E731
    out = torch.full((len(q), hq * d), 7.0, dtype=torch.bfloat16, device=dev)
    blocks = (i32(0, 2, 0, -1, 3), i32(0, 128, 128, 0, 0))  # (sequences that there are not: nothing)
    ops.flash_prefill_kv8(q.view(len(q), -1).to(dev), cu.to(dev), i32(0, 0, 0), cache, table.to(dev), hq, hkv, d, 0.1, qblocks=blocks, out=out)
    named = torch.zeros(len(q), dtype=torch.bool)
    for i, first, n in ((0, 0, 140), (2, 128, 128)):
        rows = slice(int(cu[i]) + first, int(cu[i]) + first + n)
        named[rows] = True
        want = attend(q[rows].double(), *(t[: first + n] for t in book.tokens(table[i], new[i])), 0.1, first)
        check_attention(out[rows], *want)
    assert bool((out[~named.to(dev)] == 7).all())


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("hq,hkv,d", [(8, 8, 64), (16, 1, 64), (16, 1, 128), (7, 1, 128), (32, 8, 128)])
def test_prefill_with_split_keys_of_every_form(dev, hq, hkv, d):
    """Both head sizes, one and several groups of 256 (row, head) pairs a q-block, a split that ends behind the rows' last key."""
    gen = torch.Generator().manual_seed(hq + d)
    ctx, new = [1800, 3, 1021], [44, 40, 17]
    cache, table, book = filled(gen, dev, [a + b for a, b in zip(ctx, new)], hkv, d)
    q = rand(gen, sum(new), hq, d).bfloat16()
    cu = torch.tensor([0, *itertools.accumulate(new)], dtype=torch.int32)
    got = ops.flash_prefill_kv8(q.view(sum(new), -1).to(dev), cu.to(dev), torch.tensor(ctx, dtype=torch.int32, device=dev), cache, table.to(dev), hq,
                                hkv, d, 0.1)
    want = [attend(q[int(cu[i]):int(cu[i + 1])].double(), *book.tokens(table[i], a + b), 0.1, a) for i, (a, b) in enumerate(zip(ctx, new))]
    check_attention(got, *(torch.cat(w) for w in zip(*want)))


@pytest.mark.gpu
@pytest.mark.parametrize("ctx,new", [(0, 200), (50, 100), (1500, 20)])
def test_prefill_nan_counts_for_rows_that_see_it_at_head_size_64(ctx, new):
    hq, hkv, d = 4, 2, 64
    gen = torch.Generator().manual_seed(ctx + new + 1)
    n = ctx + new
    cache, table, book = filled(gen, "cuda", [n], hkv, d)
    bad_v, bad_k = ctx + new // 3, ctx + new - 5
    page, off = int(table[0, bad_v // 16]), bad_v % 16
    cache.v.view(torch.uint8)[page, 0, 61, off] = NAN_CODE
    cache.v.view(torch.uint8)[page, 1, 3, off] = 0xFF
    page, off = int(table[0, bad_k // 16]), bad_k % 16
    cache.k.view(torch.uint8)[page, 1, 2, off, 9] = NAN_CODE
    book2 = Book(cache)
    q = rand(gen, new, hq, d).bfloat16()
    cu = torch.tensor([0, new], dtype=torch.int32)
    got = ops.flash_prefill_kv8(q.view(new, -1).cuda(), cu.cuda(), torch.tensor([ctx], dtype=torch.int32).cuda(), cache, table.cuda(), hq, hkv, d, 0.1)
    want, _ = attend(q.double(), *book2.tokens(table[0], n), 0.1, ctx)
    _, size = attend(q.double(), *book.tokens(table[0], n), 0.1, ctx)
    assert bool(want.isnan().any()) and not bool(want[: new // 3].isnan().any())
    check_attention(got, want, size)


@pytest.mark.gpu
def test_prefill_does_not_depend_on_where_a_prompt_is_cut():
    hq, hkv, d = 8, 2, 128
    gen = torch.Generator().manual_seed(31)
    n = 300
    cache, table, book = filled(gen, "cuda", [n], hkv, d)
    q = rand(gen, n, hq, d).bfloat16()
    want, size = attend(q.double(), *book.tokens(table[0], n), 0.1, 0)
    for cuts in ([0, 300], [0, 1, 300], [0, 77, 200, 300]):
        for a, b in zip(cuts, cuts[1:]):
            got = ops.flash_prefill_kv8(q[a:b].reshape(b - a, -1).cuda(), torch.tensor([0, b - a], dtype=torch.int32).cuda(),
                                        torch.tensor([a], dtype=torch.int32).cuda(), cache, table.cuda(), hq, hkv, d, 0.1)
            check_attention(got, want[a:b], size[a:b])


# ---------------------------------------------------------------- together, and refusals

@pytest.mark.parametrize("dev", DEVICES)
def test_prompt_chunks_then_steps(dev):
    """As a server goes on: a prompt in two chunks, then five steps, the other sequence's prompt between them."""
    hq, hkv, d, scale = 4, 2, 128, 2.0 ** -6
    gen = torch.Generator().manual_seed(41)
    cache = ops.kv8_cache(12, hkv, d, device=dev)
    garbage(cache, gen)
    book = Book(cache)
    table = torch.tensor([[3, 7, 1, 9], [0, 11, 5, 2]], dtype=torch.int32)
    cs = torch.cat([torch.ones(64, d // 2), torch.zeros(64, d // 2)], 1).to(dev)
    slots = lambda i, a, b: torch.tensor([int(table[i, t // 16]) * 16 + t % 16 for t in range(a, b)], dtype=torch.int32)  # noqa: E731
    at = [0, 0]
    for kind, who, n in (("chunk", 0, 21), ("chunk", 0, 9), ("step", 0, 1), ("chunk", 1, 35), ("step", -1, 1), ("step", -1, 1), ("step", 1, 1)):
        seqs = [0, 1] if who < 0 else [who]
        sl = torch.cat([slots(i, at[i], at[i] + n) for i in seqs])
        pos = torch.cat([torch.arange(at[i], at[i] + n, dtype=torch.int32) for i in seqs])
        raw = torch.round(torch.randn(len(sl), hq + 2 * hkv, d, generator=gen) * 16) / 16
        x = raw.double()
        book.write(sl, x[:, hq:hq + hkv], x[:, hq + hkv:])
        want = [attend(x[j * n:(j + 1) * n, :hq], *book.tokens(table[i], at[i] + n), scale, at[i]) for j, i in enumerate(seqs)]
        if kind == "chunk":
            qkv = raw.view(n, -1).bfloat16().to(dev)
            ops.rope_and_cache_kv8(qkv, pos.to(dev), cs, cache, sl.to(dev), hq, hkv, d)
            got = ops.flash_prefill_kv8(qkv, torch.tensor([0, n], dtype=torch.int32, device=dev), torch.tensor([at[who]], dtype=torch.int32, device=dev),
                                        cache, table[who:who + 1].to(dev), hq, hkv, d, scale)
        else:
            got = ops.paged_decode_fused_kv8(raw.view(1, len(seqs), -1).to(dev), 1, pos.to(dev), cs, sl.to(dev), cache, table[seqs].to(dev),
                                             (pos + 1).to(dev), hq, hkv, d, scale)
        book.check(cache)
        check_attention(got, *(torch.cat(w) for w in zip(*want)))
        for i in seqs:
            at[i] += n


def test_cache_sizes():
    c = ops.kv8_cache(5, 3, 64, layers=2)
    assert c.k.shape == (2, 5, 3, 4, 16, 16) and c.v.shape == (2, 5, 3, 64, 16) and c.scales.shape == (2, 5, 3, 2)
    assert sum(t.numel() * t.element_size() for t in c) == 2 * 5 * ops.kv8_block_bytes(3, 64)
    assert c.layer(1).k.shape == (5, 3, 4, 16, 16)
    with pytest.raises(ValueError, match="head size"):
        ops.kv8_cache(5, 3, 96)


@pytest.mark.parametrize("dev", DEVICES)
def test_calls_of_nothing(dev):
    hq, hkv, d = 4, 2, 128
    cache = ops.kv8_cache(2, hkv, d, device=dev)
    i32 = lambda *s: torch.zeros(*s, dtype=torch.int32, device=dev)  # noqa: E731
    cols = (hq + 2 * hkv) * d
    none = torch.zeros(0, cols, dtype=torch.bfloat16, device=dev)
    ops.rope_and_cache_kv8(none, i32(0), table_of(d, dev), cache, i32(0), hq, hkv, d)
    assert ops.paged_decode_kv8(none, cache, i32(0, 1), i32(0), hq, hkv, d, 0.1).shape == (0, hq * d)
    assert ops.paged_decode_fused_kv8(torch.zeros(1, 0, cols, device=dev), 1, i32(0), table_of(d, dev), i32(0), cache, i32(0, 1), i32(0), hq, hkv, d,
                                      0.1).shape == (0, hq * d)
    assert ops.flash_prefill_kv8(none, i32(1), i32(0), cache, i32(0, 1), hq, hkv, d, 0.1).shape == (0, hq * d)
    x = torch.ones(3, cols, dtype=torch.bfloat16, device=dev)
    ops.rope_and_cache_kv8(x, i32(3), table_of(d, dev), cache, i32(3) - 1, hq, hkv, d, apply_rope=False)
    assert all(int(t.view(torch.uint8).sum()) == 0 for t in (cache.k, cache.v)) and float(cache.scales.sum()) == 0


@pytest.mark.gpu
def test_offsets_past_32_bits():
    """A cache of 4.4 GB of key codes: pages in its last part, whose byte offsets need 33 bits."""
    hq, hkv, d, dev = 4, 2, 128, "cuda"
    n = 1_100_000
    gen = torch.Generator().manual_seed(51)
    cache = ops.kv8_cache(n, hkv, d, device=dev)
    L = 40
    pages = [n - 1, 5, n - 77]
    table = torch.tensor([pages], dtype=torch.int32)
    slots = torch.tensor([pages[t // 16] * 16 + t % 16 for t in range(L)], dtype=torch.int32)
    x = torch.round(torch.randn(L, hq + 2 * hkv, d, generator=gen) * 16) / 16
    small = ops.kv8_cache(3, hkv, d)
    book = Book(small)
    near = torch.arange(L, dtype=torch.int32)
    book.write(near, x[:, hq:hq + hkv].double(), x[:, hq + hkv:].double())
    rows = x.bfloat16().view(L, -1).to(dev)
    ops.rope_and_cache_kv8(rows[:-1], no_positions(L - 1, dev), table_of(d, dev), cache, slots[:-1].to(dev), hq, hkv, d, apply_rope=False)
    cs = torch.cat([torch.ones(64, d // 2), torch.zeros(64, d // 2)], 1).to(dev)
    pos = torch.tensor([L - 1], dtype=torch.int32, device=dev)
    args = (hq, hkv, d, 2.0 ** -4)
    got = ops.paged_decode_fused_kv8(x[-1:].reshape(1, 1, -1).to(dev), 1, pos, cs, slots[-1:].to(dev), cache, table.to(dev), pos + 1, *args)
    at = torch.tensor(pages, device=dev)
    book.check(ops.KV8(*(t.view(torch.uint8)[at].view(kv8.E4M3) if t.dtype == kv8.E4M3 else t[at] for t in cache)))
    k, v = book.tokens([0, 1, 2], L)
    check_attention(got, *attend(x[-1:, :hq].double(), k, v, args[3], L - 1))
    check_attention(ops.paged_decode_kv8(rows[-1:], cache, table.to(dev), pos + 1, *args), *attend(x[-1:, :hq].double(), k, v, args[3], L - 1))
    got = ops.flash_prefill_kv8(rows, torch.tensor([0, L], dtype=torch.int32, device=dev), torch.zeros(1, dtype=torch.int32, device=dev), cache,
                                table.to(dev), *args)
    check_attention(got, *attend(x[:, :hq].double(), k, v, args[3], 0))


@pytest.mark.gpu
def test_prefill_in_a_graph_with_its_splits():
    """A captured chunk whose keys are split: the partials lie in the graph's own memory, every replay answers for the tokens of its time."""
    hq, hkv, d = 8, 2, 128
    gen = torch.Generator().manual_seed(61)
    ctx, new = 1200, 30
    cache, table, book = filled(gen, "cuda", [ctx + new], hkv, d)
    q = torch.zeros(new, hq * d, dtype=torch.bfloat16, device="cuda")
    cu, cs, tb = torch.tensor([0, new], dtype=torch.int32).cuda(), torch.tensor([ctx], dtype=torch.int32).cuda(), table.cuda()
    qb = (torch.zeros(1, dtype=torch.int32).cuda(), torch.zeros(1, dtype=torch.int32).cuda())
    run = lambda: ops.flash_prefill_kv8(q, cu, cs, cache, tb, hq, hkv, d, 0.1, qblocks=qb)  # noqa: E731
    run()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = run()
    for _ in range(3):
        x = rand(gen, new, hq, d).bfloat16()
        q.copy_(x.view(new, -1))
        g.replay()
        torch.cuda.synchronize()
        other = run()
        want = attend(x.double(), *book.tokens(table[0], ctx + new), 0.1, ctx)
        check_attention(out, *want)
        check_attention(other, *want)


@pytest.mark.gpu
def test_refusals():
    """Arguments that the kernels do not take are errors on the host."""
    dev, hq, hkv, d = "cuda", 4, 2, 128
    cache = ops.kv8_cache(4, hkv, d, device=dev)
    q = torch.zeros(2, hq * d, dtype=torch.bfloat16, device=dev)
    qkv = torch.zeros(2, (hq + 2 * hkv) * d, dtype=torch.bfloat16, device=dev)
    i32 = lambda *v: torch.tensor(v, dtype=torch.int32, device=dev)  # noqa: E731
    table, lens, cs = torch.zeros(2, 2, dtype=torch.int32, device=dev), i32(3, 4), table_of(d, dev)
    dec = lambda **k: ops.paged_decode_kv8(**{**dict(q=q, cache=cache, block_tables=table, seq_lens=lens, Hq=hq, Hkv=hkv, D=d, scale=0.1), **k})  # noqa: E731
    pre = lambda **k: ops.flash_prefill_kv8(**{**dict(qkv=qkv, cu_seqlens=i32(0, 1, 2), ctx_start=i32(0, 0), cache=cache, block_tables=table, Hq=hq,  # noqa: E731
                                                      Hkv=hkv, D=d, scale=0.1), **k})
    wr = lambda **k: ops.rope_and_cache_kv8(**{**dict(qkv=qkv, positions=i32(0, 0), cos_sin=cs, cache=cache, slot_mapping=i32(0, 1), Hq=hq, Hkv=hkv,  # noqa: E731
                                                      D=d, apply_rope=False), **k})
    slabs = torch.zeros(1, 2, (hq + 2 * hkv) * d, device=dev)
    fus = lambda **k: ops.paged_decode_fused_kv8(**{**dict(slabs=slabs, nslabs=1, positions=i32(2, 3), cos_sin=cs, slot_mapping=i32(2, 3), cache=cache,  # noqa: E731
                                                           block_tables=table, seq_lens=lens, Hq=hq, Hkv=hkv, D=d, scale=0.1), **k})
    for f in (dec, pre, wr, fus):
        f()
    wrong = ops.KV8(cache.k.view(torch.uint8), cache.v, cache.scales)
    cases = [(dec, dict(q=q.float())), (dec, dict(q=q[:, :-8])), (dec, dict(q=q[:1])), (dec, dict(cache=wrong)), (dec, dict(Hq=5)), (dec, dict(D=96)),
             (dec, dict(scale=0.0)), (dec, dict(scale=-1.0)), (dec, dict(scale=math.nan)), (dec, dict(seq_lens=lens.long())),
             (dec, dict(block_tables=table[:1])), (dec, dict(splits=65)), (dec, dict(cache=ops.kv8_cache(4, 3, d, device=dev))),
             (dec, dict(q=torch.zeros(2 * hq * d + 1, dtype=torch.bfloat16, device=dev)[1:].view(2, -1))),
             (dec, dict(out=torch.empty(1, hq * d, dtype=torch.bfloat16, device=dev))),
             (dec, dict(workspace=ops.decode_workspace(1, hq, d, device=dev), splits=64)),
             (dec, dict(cache=ops.KV8(cache.k, cache.v, cache.scales[:2]))), (dec, dict(Hq=64)),
             (pre, dict(ctx_start=i32(0))), (pre, dict(block_tables=table[:1])), (pre, dict(scale=math.inf)), (pre, dict(out=q[:1])),
             (wr, dict(slot_mapping=i32(0))), (wr, dict(qkv=qkv[:, : hq * d])), (wr, dict(slot_mapping=i32(0, 1).long())),
             (wr, dict(partial=torch.zeros(2 * 8 * 128, device=dev), nslabs=2)),
             (wr, dict(cache=ops.KV8(cache.k.cpu(), cache.v, cache.scales))),
             (fus, dict(nslabs=2)), (fus, dict(nslabs=0)), (fus, dict(positions=i32(2))), (fus, dict(cos_sin=cs[:, :64])),
             (fus, dict(slabs=slabs.bfloat16())), (fus, dict(slot_mapping=i32(1)))]
    for f, k in cases:
        with pytest.raises((RuntimeError, ValueError)):
            f(**k)
    torch.cuda.synchronize()


@pytest.mark.gpu
def test_prefill_of_few_named_rows_takes_little_memory():
    """One q-block of many rows: right for its rows, the others left as they are, and no partials for rows that nothing names."""
    hq, hkv, d, dev = 8, 2, 128, "cuda"
    gen = torch.Generator().manual_seed(71)
    ctx, new, T = 2000, 40, 4096
    cache, table, book = filled(gen, dev, [ctx + new], hkv, d)
    x = rand(gen, new, hq, d).bfloat16()
    q = torch.zeros(T, hq * d, dtype=torch.bfloat16, device=dev)
    q[:new] = x.view(new, -1)
    out = torch.full((T, hq * d), 7.0, dtype=torch.bfloat16, device=dev)
    i32 = lambda *v: torch.tensor(v, dtype=torch.int32, device=dev)  # noqa: E731
    args = (i32(0, new), i32(ctx), cache, table.to(dev), hq, hkv, d, 0.1)
    qb = (i32(0), i32(0))
    torch.cuda.synchronize()
    torch.cuda.reset_peak_memory_stats()
    before = torch.cuda.memory_allocated()
    ops.flash_prefill_kv8(q, *args, qblocks=qb, out=out)
    torch.cuda.synchronize()
    assert torch.cuda.max_memory_allocated() == before
    check_attention(out[:new], *attend(x.double(), *book.tokens(table[0], ctx + new), 0.1, ctx))
    assert bool((out[new:] == 7).all())


@pytest.mark.gpu
def test_refused_sizes_and_overlapping_rows():
    """Products of sizes past 32 (or 64) bits, and outputs whose rows share memory, are errors on the host."""
    dev, hq, hkv, d = "cuda", 2, 2, 128
    i32 = lambda *v: torch.tensor(v, dtype=torch.int32, device=dev)  # noqa: E731
    cache, cs = ops.kv8_cache(4, hkv, d, device=dev), table_of(d, dev)
    wide = ops.kv8_cache(1, 4096, 64, device=dev)
    rows = torch.zeros(1, 3 * 4096 * 64, dtype=torch.bfloat16, device=dev).expand(1 << 19, -1)
    with pytest.raises(RuntimeError, match="2.31"):
        ops.rope_and_cache_kv8(rows, None, None, wide, torch.full((1 << 19,), -1, dtype=torch.int32, device=dev), 4096, 4096, 64, apply_rope=False)
    slabs, table, lens = torch.zeros(1, 2, 3 * hq * d, device=dev), torch.zeros(2, 2, dtype=torch.int32, device=dev), i32(3, 4)
    with pytest.raises(RuntimeError, match="nslabs"):
        ops.paged_decode_fused_kv8(slabs, 1 << 60, i32(2, 3), cs, i32(2, 3), cache, table, lens, hq, hkv, d, 0.1)
    q = torch.zeros(2, hq * d, dtype=torch.bfloat16, device=dev)
    with pytest.raises(RuntimeError, match="out must be"):
        ops.flash_prefill_kv8(q, i32(0, 1, 2), i32(0, 0), cache, table, hq, hkv, d, 0.1, out=q[:1].expand(2, -1))
    c = ops.logit_controls(1, 64, 2, device=dev)
    with pytest.raises(RuntimeError, match="overlap"):
        ops.control_logits(torch.zeros(2, 64, device=dev), c, i32(0, 0), torch.zeros(1, 16, dtype=torch.int32, device=dev), table, lens,
                           out=torch.zeros(1, 64, device=dev).expand(2, -1))
    torch.cuda.synchronize()
