"""The operators of a decode step whose cache is held in 8 bits and whose answer is constrained, as cases that can be timed and compared.

Five operators of :mod:`k8s_llm_monitor_amd.ops`, each beside the one whose form it extends:

* ``write``: ``rope_and_cache_kv8`` - keys and values of new tokens into 16-token pages of e4m3 codes with a scale for each page and kv head;
* ``step``: ``paged_decode_fused_kv8`` - one token a sequence behind the qkv projection: the sum of its split-K slabs, rotation, cache write, attention;
* ``decode``: ``paged_decode_kv8`` - one token a sequence over cached ones;
* ``prefill``: ``flash_prefill_kv8`` - prompt chunks over the 8-bit pages that hold them and what came before;
* ``logits``: ``control_logits`` - penalties for repeated tokens, biases and allowed-token masks, the history read from pages of token ids.

The cache: keys ``[pages, Hkv, 4, 16, D / 4]`` (four runs of dims, then the page's tokens), values ``[pages, Hkv, D, 16]``, both e4m3, and
``scales [pages, Hkv, 2]`` fp32 (keys', values'): a code stands for its value times the scale, a power of two: the least one that brings the largest
finite magnitude written to the page and head to 448 or less, and not less than the page's scale before where it holds earlier tokens, whose codes
are rounded anew where the scale has grown.  Non-finite numbers become NaN codes and set no scale.

The keys of a case: ``op``; ``hq``, ``hkv``, ``d``: heads and head size; ``batch`` sequences with about ``context`` cached tokens each, ``ragged``:
by what part of its length the shortest is shorter than the longest; ``tokens``: new rows a sequence (write, prefill).  Of ``logits``: ``batch``
rows of ``vocab`` logits in ``dtype``, ``context`` tokens of history, ``bias`` biased tokens a row, ``masked``: whether rows have masks, ``plain``:
every how manieth row has no controls (0: none).
"""
from __future__ import annotations

import math

import torch

own = False

PAGE = 16
E4M3 = torch.float8_e4m3fn
LEAST = 2.0 ** -100  # of scales
SLABS = 4  # split-K slabs of the qkv projection at decode
THETA = 500000.0


def _case(name, op, **kw):
    c = dict(op=op, **kw)
    return dict(c, name=name) if name else c


def _attn(name, op, hq, hkv, d, batch, context, ragged=0.0, tokens=1):
    return _case(name, op, hq=hq, hkv=hkv, d=d, batch=batch, context=context, ragged=ragged, tokens=tokens)


def _logits(name, batch, vocab, context, dtype="bfloat16", bias=0, masked=False, plain=0):
    return _case(name, "logits", batch=batch, vocab=vocab, context=context, dtype=dtype, bias=bias, masked=masked, plain=plain)


def listed() -> list:
    return [
        # the cache write of a full prefill step: ten whole ~1.6 k token prompts of a Llama-3-8B, rotated by the qkv projection
        _attn("write-10x1636", "write", 32, 8, 128, 10, 0, 0.05, 1636),
        # a few follow-up questions: short ragged chunks that start inside a page
        _attn("write-3x37", "write", 32, 8, 128, 3, 1001, 0.3, 37),
        # one operator asking: the next token of one answer
        _attn("step-1x1700", "step", 32, 8, 128, 1, 1700),
        # the headline wave's decode step: 64 diagnostic queries at once
        _attn("step-64x1900", "step", 32, 8, 128, 64, 1900, 0.2),
        # long contexts, which 8-bit pages are for: eight sequences of 32 k tokens on a 64-head model
        _attn("step-8x32768", "step", 64, 8, 128, 8, 32768, 0.1),
        # GPT-2-small's heads (no groups, 64 dims): running sequences of a mixed step
        _attn("decode-24x900", "decode", 12, 12, 64, 24, 900, 0.9),
        # the running sequences of a large mixed step, seven heads a group
        _attn("decode-128x4097", "decode", 28, 4, 128, 128, 4097, 0.5),
        # a question behind a cached conversation: 45 new rows over 4 k tokens
        _attn("prefill-1x45", "prefill", 32, 8, 128, 1, 4096, 0.0, 45),
        # prompts that share a cached 512-token prefix
        _attn("prefill-10x1124", "prefill", 32, 8, 128, 10, 512, 0.1, 1124),
        # a long prompt's last chunk
        _attn("prefill-1x4096", "prefill", 32, 8, 128, 1, 12288, 0.0, 4096),
        # the headline wave's logits, penalised, biased and held to a grammar
        _logits("logits-64x128256", 64, 128256, 1900, bias=32, masked=True),
        # one row of GPT-2's vocabulary (odd), fp32
        _logits("logits-1x50257", 1, 50257, 700, dtype="float32", bias=5),
    ]


HEADS = ((32, 8, 128), (64, 8, 128), (8, 1, 128), (28, 4, 128), (40, 8, 128), (12, 12, 64), (12, 4, 128), (32, 2, 64), (4, 4, 64))


def _log(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng) -> dict:
    op = rng.choice(("write", "step", "step", "decode", "prefill", "logits", "logits"))
    if op == "logits":
        vocab = rng.choice((128256, 32000, 50257, _log(rng, 500, 128256)))
        return _logits(None, _log(rng, 1, 64), vocab, _log(rng, 1, 8192), dtype=rng.choice(("bfloat16", "float32")),
                       bias=rng.choice((0, rng.randint(1, 300))), masked=rng.random() < 0.5, plain=rng.choice((0, 2, 5)))
    hq, hkv, d = rng.choice([h for h in HEADS if op != "step" or h[2] == 128 and h[0] // h[1] <= 8])
    ragged = round(rng.uniform(0.0, 0.9), 2)
    if op in ("step", "decode"):
        batch = _log(rng, 1, 160)
        return _attn(None, op, hq, hkv, d, batch, _log(rng, 1, max(2, min(32768, 250000 // batch))), ragged)
    batch = _log(rng, 1, 12)
    if op == "write":
        return _attn(None, op, hq, hkv, d, batch, _log(rng, 1, 4096) - 1, ragged, _log(rng, 1, 16384 // batch))
    tokens = _log(rng, 1, 8192 // batch)
    room = (1 << 25) // (batch * tokens)  # (row, key) pairs a head, at most half the largest case's
    return _attn(None, op, hq if hq <= 32 else 32, hkv, d, batch, min(_log(rng, 1, 16384) - 1, max(0, room - tokens)), ragged, tokens)


def _lengths(n, longest, ragged):
    """n lengths from the longest down to (1 - ragged) of it, in a mixed order."""
    step = next(k for k in (7, 5, 3, 2, 1) if math.gcd(k, n) == 1)
    return [max(0, round(longest * (1.0 - ragged * ((i * step) % n) / max(1, n - 1)))) for i in range(n)]


def _spans(c):
    """(cached tokens, new rows) of each sequence."""
    ctx = _lengths(c["batch"], c["context"], c["ragged"])
    if c["op"] in ("step", "decode"):
        return [max(0, x - 1) for x in ctx], [1] * c["batch"]
    return ctx, [max(1, x) for x in _lengths(c["batch"], c["tokens"], c["ragged"])]


def _mask_words(vocab):
    return (vocab + 31) // 32


def work(c) -> dict:
    if c["op"] == "logits":
        size = 2 if c["dtype"] == "bfloat16" else 4
        words = _mask_words(c["vocab"]) if c["masked"] else 0
        return dict(bytes=c["batch"] * (2 * size * c["vocab"] + 4 * words + 4 * c["context"] + 8 * c["bias"]), flops=c["batch"] * 4 * c["vocab"])
    ctx, new = _spans(c)
    hq, hkv, d = c["hq"], c["hkv"], c["d"]
    rows = sum(new)
    if c["op"] == "write":
        pages = sum((a + n + PAGE - 1) // PAGE - a // PAGE for a, n in zip(ctx, new))
        return dict(bytes=rows * hkv * d * 2 * 3 + pages * hkv * 8, flops=4 * rows * hkv * d)
    total = sum(ctx) + rows
    held = total * hkv * d * 2 + (total + PAGE - 1) // PAGE * hkv * 8
    if c["op"] == "prefill":
        pairs = sum(n * a + n * (n + 1) // 2 for a, n in zip(ctx, new))
        return dict(bytes=held + 2 * rows * hq * d * 2, flops=4 * hq * d * pairs)
    read = rows * (hq + 2 * hkv) * d * 4 * SLABS if c["op"] == "step" else rows * hq * d * 2
    return dict(bytes=held + read + rows * hq * d * 2, flops=4 * hq * d * total)


# ---------------------------------------------------------------- inputs

def _pages(gen, need, spare, dev):
    """Page numbers of sequences that need so many each, out of a shuffled cache: [S, most], and how many pages it has."""
    n = sum(need) + spare
    order = torch.randperm(n, generator=gen, device=dev, dtype=torch.int64).to(torch.int32)
    table = torch.zeros(len(need), max(need), dtype=torch.int32, device=dev)
    at = 0
    for i, k in enumerate(need):
        table[i, :k] = order[at:at + k]
        at += k
    return table, n


def _cache(gen, n, hkv, d, dev):
    """A cache whose pages all hold tokens of earlier work: channels and tokens of different size, as projections give them."""
    k = torch.empty(n, hkv, 4, PAGE, d // 4, dtype=torch.uint8, device=dev)
    v = torch.empty(n, hkv, d, PAGE, dtype=torch.uint8, device=dev)
    scales = torch.empty(n, hkv, 2, dtype=torch.float32, device=dev)
    chan = torch.exp(0.7 * torch.randn(hkv, 4, 1, d // 4, generator=gen, device=dev))
    for a in range(0, n, 4096):
        b = min(n, a + 4096)
        x = torch.randn(b - a, hkv, 4, PAGE, d // 4, generator=gen, device=dev) * chan
        y = 0.5 * torch.randn(b - a, hkv, d, PAGE, generator=gen, device=dev)
        for codes, z, j in ((k, x, 0), (v, y, 1)):
            s = _scale(z.abs().amax((2, 3, 4) if j == 0 else (2, 3)))
            scales[a:b, :, j] = s
            codes[a:b] = (z / s.view(b - a, hkv, *([1] * (z.dim() - 2)))).to(E4M3).view(torch.uint8)
    return k.view(E4M3), v.view(E4M3), scales


def _i32(v, dev):
    return torch.tensor(v, dtype=torch.int32, device=dev)


def _cos_sin(n, d, dev):
    inv = THETA ** (-torch.arange(d // 2, dtype=torch.float64, device=dev) * 2 / d)
    a = torch.arange(n, dtype=torch.float64, device=dev)[:, None] * inv
    return torch.cat([a.cos(), a.sin()], 1).float()


def prepare(c, seed):
    dev = torch.device("cuda")
    gen = torch.Generator(dev).manual_seed(seed)
    if c["op"] == "logits":
        return _prepare_logits(c, gen, dev)
    ctx, new = _spans(c)
    hq, hkv, d, op = c["hq"], c["hkv"], c["d"], c["op"]
    rows, cols = sum(new), (hq + 2 * hkv) * d
    table, n = _pages(gen, [(a + k + PAGE - 1) // PAGE for a, k in zip(ctx, new)], 3, dev)
    k, v, scales = _cache(gen, n, hkv, d, dev)
    s = dict(op=op, hq=hq, hkv=hkv, d=d, scale=1.0 / math.sqrt(d), k=k, v=v, scales=scales, table=table)
    cu = [0]
    for m in new:
        cu.append(cu[-1] + m)
    seq = torch.repeat_interleave(torch.arange(len(new), device=dev), _i32(new, dev).long())
    pos = torch.arange(rows, device=dev) - _i32(cu, dev).long()[seq] + _i32(ctx, dev).long()[seq]
    s["positions"] = pos.to(torch.int32)
    s["slots"] = table[seq, pos // PAGE] * PAGE + (pos % PAGE).to(torch.int32)
    s["cos_sin"] = _cos_sin(max(a + m for a, m in zip(ctx, new)), d, dev)
    chan = torch.exp(0.5 * torch.randn(cols, generator=gen, device=dev))
    if op == "step":
        s["slabs"] = torch.randn(SLABS, rows, cols, generator=gen, device=dev) * chan * 0.5
    else:
        s["qkv"] = (torch.randn(rows, cols, generator=gen, device=dev) * chan).to(torch.bfloat16)
    if op in ("step", "decode"):
        s["lens"] = _i32([a + 1 for a in ctx], dev)
        # the buffers of split partials that a serving program keeps (the last one: counters, zero between calls)
        s["workspace"] = (torch.empty(rows, hq, 64, d, device=dev), torch.empty(rows, hq, 64, 2, device=dev),
                          torch.zeros(rows * hq, dtype=torch.int32, device=dev))
    if op == "prefill":
        s["cu"], s["ctx"], s["most"] = _i32(cu, dev), _i32(ctx, dev), max(new)
        # 128-row q-blocks, the longest sequence first and its heaviest block first
        q = sorted((-(a + m), i, -r) for i, (a, m) in enumerate(zip(ctx, new)) for r in range(0, m, 128))
        s["qblocks"] = (_i32([t[1] for t in q], dev), _i32([-t[2] for t in q], dev))
    return s


def _prepare_logits(c, gen, dev):
    b, vocab, bias = c["batch"], c["vocab"], c["bias"]
    lens = _lengths(b, c["context"], 0.3)
    table, n = _pages(gen, [max(1, (x + PAGE - 1) // PAGE) for x in lens], 1, dev)
    # token ids of different frequency, as text has them
    ids = (vocab * torch.rand(n, PAGE, generator=gen, device=dev) ** 6).to(torch.int32).clamp_(max=vocab - 1)
    rand = torch.rand(b, 3, generator=gen, device=dev)
    params = torch.stack([1 + 0.3 * rand[:, 0], rand[:, 1], 0.5 * rand[:, 2]], 1).contiguous()
    info = torch.stack([(0.7 * _i32(lens, dev)).to(torch.int32), torch.full((b,), int(c["masked"]), dtype=torch.int32, device=dev)], 1).contiguous()
    width = max(1, bias)
    bias_ids = torch.full((b, width), -1, dtype=torch.int32, device=dev)
    if bias:  # distinct ids a row
        step = max(1, vocab // width)
        at = torch.arange(width, device=dev) * step + torch.randint(0, step, (b, width), generator=gen, device=dev)
        bias_ids[:] = at.clamp(max=vocab - 1).to(torch.int32)
        if width > vocab:
            bias_ids[:, vocab:] = -1
    bias_vals = 5 * torch.randn(b, width, generator=gen, device=dev)
    words = _mask_words(vocab)
    masks = torch.full((b, words), -1, dtype=torch.int32, device=dev)
    if c["masked"]:  # every other row may go on with a few tokens only, the others with about half of all
        bits = torch.randint(-(1 << 31), 1 << 31, (b, words), generator=gen, device=dev, dtype=torch.int64)
        few = torch.rand(b, words, generator=gen, device=dev) < 0.01
        masks = torch.where((torch.arange(b, device=dev) % 2 == 0)[:, None] & ~few, torch.zeros_like(bits), bits).to(torch.int32)
    rows = torch.arange(b - 1, -1, -1, device=dev, dtype=torch.int32)
    if c["plain"]:
        rows[:: c["plain"]] = -1
    return dict(op="logits", logits=(4 * torch.randn(b, vocab, generator=gen, device=dev)).to(getattr(torch, c["dtype"])), rows=rows, tokens=ids,
                table=table, lens=_i32(lens, dev), params=params, info=info, bias_ids=bias_ids, bias_vals=bias_vals, masks=masks)


# ---------------------------------------------------------------- the operators

def run(s):
    return (_run_own if own else _run_plain)[s["op"]](s)


def _own_cache(ops, s):
    return ops.KV8(s["k"], s["v"], s["scales"])


def _own_write(s):
    from k8s_llm_monitor_amd import ops
    ops.rope_and_cache_kv8(s["qkv"], s["positions"], s["cos_sin"], _own_cache(ops, s), s["slots"], s["hq"], s["hkv"], s["d"], apply_rope=False)
    return dict(k=s["k"], v=s["v"], scales=s["scales"])


def _own_step(s):
    from k8s_llm_monitor_amd import ops
    o = ops.paged_decode_fused_kv8(s["slabs"], SLABS, s["positions"], s["cos_sin"], s["slots"], _own_cache(ops, s), s["table"], s["lens"],
                                   s["hq"], s["hkv"], s["d"], s["scale"], workspace=s["workspace"])
    return dict(o=o, k=s["k"], v=s["v"], scales=s["scales"])


def _own_decode(s):
    from k8s_llm_monitor_amd import ops
    return ops.paged_decode_kv8(s["qkv"], _own_cache(ops, s), s["table"], s["lens"], s["hq"], s["hkv"], s["d"], s["scale"], workspace=s["workspace"])


def _own_prefill(s):
    from k8s_llm_monitor_amd import ops
    return ops.flash_prefill_kv8(s["qkv"], s["cu"], s["ctx"], _own_cache(ops, s), s["table"], s["hq"], s["hkv"], s["d"], s["scale"], qblocks=s["qblocks"])


def _own_logits(s):
    from k8s_llm_monitor_amd import ops
    controls = ops.LogitControls(s["params"], s["info"], s["bias_ids"], s["bias_vals"], s["masks"])
    return ops.control_logits(s["logits"], controls, s["rows"], s["tokens"], s["table"], s["lens"])


_run_own = dict(write=_own_write, step=_own_step, decode=_own_decode, prefill=_own_prefill, logits=_own_logits)


def _scale(amax):
    """The least power of two s with amax / s <= 448 = 0.875 * 2^9."""
    m, e = torch.frexp(amax)
    return torch.where(amax > 0, torch.ldexp(torch.ones_like(amax), e - torch.where(m > 0.875, 8, 9)), torch.zeros_like(amax)).clamp_min(LEAST)


def _write(s, k_new, v_new):
    """k_new, v_new [T, Hkv, D] into the pages of s["slots"]."""
    hkv, d = s["hkv"], s["d"]
    pages, row = torch.unique((s["slots"] // PAGE).long(), return_inverse=True)
    off = (s["slots"] % PAGE).long()
    first = torch.full((pages.numel(),), PAGE, dtype=torch.int64, device=off.device).scatter_reduce_(0, row, off, "amin")
    at = torch.arange(PAGE, device=off.device)
    earlier = at[None] < first[:, None]  # [pages, 16]
    for j, (codes, x) in enumerate(((s["k"], k_new.float()), (s["v"], v_new.float()))):
        size = torch.where(x.isfinite(), x.abs(), torch.zeros_like(x)).amax(-1)  # [T, Hkv]
        amax = torch.zeros(pages.numel(), hkv, device=x.device).scatter_reduce_(0, row[:, None].expand(-1, hkv), size, "amax")
        old = s["scales"][pages, :, j]
        new = torch.maximum(_scale(amax), torch.where(first[:, None] > 0, old, torch.zeros_like(old)))
        s["scales"][pages, :, j] = new
        held = codes.view(torch.uint8)[pages]
        shrink = (old / new).view(-1, hkv, 1, 1)
        val = held.view(E4M3).float()
        got = (x / new[row][..., None]).to(E4M3).view(torch.uint8)
        if j == 0:
            again = (val * shrink[..., None]).to(E4M3).view(torch.uint8)
            held = torch.where(earlier[:, None, None, :, None], again, held)
            held[row, :, :, off, :] = got.view(-1, hkv, 4, d // 4)
        else:
            again = (val * shrink).to(E4M3).view(torch.uint8)
            held = torch.where(earlier[:, None, None, :], again, held)
            held[row, :, :, off] = got
        codes.view(torch.uint8)[pages] = held


def _read(s):
    """Keys and values of every sequence's pages as fp32 [S, Hkv, pages * 16, D]."""
    t = s["table"].long()
    S, w = t.shape
    hkv, d = s["hkv"], s["d"]
    sc = s["scales"][t]  # [S, W, Hkv, 2]
    k = s["k"].view(torch.uint8)[t].view(E4M3).float() * sc[..., 0, None, None, None]
    k = k.permute(0, 2, 1, 4, 3, 5).reshape(S, hkv, w * PAGE, d)
    v = s["v"].view(torch.uint8)[t].view(E4M3).float() * sc[..., 1, None, None]
    return k, v.permute(0, 2, 1, 4, 3).reshape(S, hkv, w * PAGE, d)


def _softmax(x):
    p = torch.exp(x - x.amax(-1, keepdim=True))
    return p / p.sum(-1, keepdim=True)


def _attend_one(s, q):
    """q [B, Hq, D] over the cached tokens; bf16 [B, Hq * D]."""
    k, v = _read(s)
    b, hq = q.shape[0], s["hq"]
    q = q.float().view(b, s["hkv"], hq // s["hkv"], -1)
    x = (q @ k.transpose(2, 3)) * s["scale"]
    x = x.masked_fill(torch.arange(k.shape[2], device=x.device) >= s["lens"][:, None, None, None], float("-inf"))
    return (_softmax(x) @ v).reshape(b, -1).to(torch.bfloat16)


def _plain_write(s):
    hq, hkv, d = s["hq"], s["hkv"], s["d"]
    x = s["qkv"].view(-1, hq + 2 * hkv, d)
    _write(s, x[:, hq:hq + hkv], x[:, hq + hkv:])
    return dict(k=s["k"], v=s["v"], scales=s["scales"])


def _plain_step(s):
    hq, hkv, d = s["hq"], s["hkv"], s["d"]
    x = s["slabs"].sum(0).to(torch.bfloat16).float().view(-1, hq + 2 * hkv, d)
    cs = s["cos_sin"][s["positions"].long()][:, None]
    c, sn = cs[..., : d // 2], cs[..., d // 2:]
    a, b = x[:, : hq + hkv, : d // 2], x[:, : hq + hkv, d // 2:]
    qk = torch.cat([a * c - b * sn, b * c + a * sn], -1).to(torch.bfloat16)
    _write(s, qk[:, hq:], x[:, hq + hkv:])
    return dict(o=_attend_one(s, qk[:, :hq]), k=s["k"], v=s["v"], scales=s["scales"])


def _plain_decode(s):
    return _attend_one(s, s["qkv"][:, : s["hq"] * s["d"]].view(-1, s["hq"], s["d"]))


def _plain_prefill(s):
    hq, hkv, d = s["hq"], s["hkv"], s["d"]
    k, v = _read(s)
    S, rows = s["ctx"].numel(), s["qkv"].shape[0]
    seq = torch.repeat_interleave(torch.arange(S, device=k.device), (s["cu"][1:] - s["cu"][:-1]).long(), output_size=rows)
    at = torch.arange(rows, device=k.device) - s["cu"].long()[seq]
    most = s["most"]
    q = torch.zeros(S, most, hq, d, device=k.device)
    q[seq, at] = s["qkv"][:, : hq * d].view(rows, hq, d).float()
    q = q.view(S, most, hkv, hq // hkv, d).permute(0, 2, 3, 1, 4).reshape(S, hkv, -1, d)
    x = (q @ k.transpose(2, 3)).view(S, hkv, hq // hkv, most, -1).mul_(s["scale"])
    last = s["ctx"][:, None] + torch.arange(most, device=k.device)  # the last key that a row sees
    x.masked_fill_((torch.arange(k.shape[2], device=k.device) > last[..., None])[:, None, None], float("-inf"))
    x.sub_(x.amax(-1, keepdim=True)).exp_()
    norm = x.sum(-1, keepdim=True)
    o = (x.view(S, hkv, -1, x.shape[-1]) @ v).view(S, hkv, hq // hkv, most, d) / norm
    return o.permute(0, 3, 1, 2, 4).reshape(S, most, hq * d)[seq, at].to(torch.bfloat16)


def _plain_logits(s):
    b, vocab = s["logits"].shape
    table = s["table"].long()
    ids = s["tokens"][table].view(b, -1).long()
    at = torch.arange(ids.shape[1], device=ids.device)[None]
    slot = s["rows"].long().clamp(min=0)
    active = (s["rows"] >= 0)[:, None]
    held = (at < s["lens"][:, None]) & active
    out = held & (at >= s["info"][slot, 0][:, None])
    zero = torch.zeros(b, vocab, device=ids.device)
    seen = zero.scatter_add(1, ids, held.float()) > 0
    count = zero.scatter_add(1, ids, out.float())
    p = s["params"][slot]
    x = s["logits"].float()
    y = torch.where(seen, torch.where(x > 0, x / p[:, :1], x * p[:, :1]), x)
    y = y - p[:, 2:] * count - p[:, 1:2] * (count > 0)
    bi = s["bias_ids"][slot].long()
    y = y.scatter_add(1, bi.clamp(min=0), torch.where(bi >= 0, s["bias_vals"][slot], 0.0))
    v = torch.arange(vocab, device=ids.device)
    allowed = ((s["masks"][slot][:, v // 32] >> (v % 32)) & 1 > 0) | (s["info"][slot, 1] == 0)[:, None]
    y = y.masked_fill(~allowed, float("-inf"))
    return torch.where(active, y, x).to(s["logits"].dtype)


_run_plain = dict(write=_plain_write, step=_plain_step, decode=_plain_decode, prefill=_plain_prefill, logits=_plain_logits)


# ---------------------------------------------------------------- the definition, in 64 bits

def _nearest_code(y):
    """The e4m3 number next to y, halves to even (|y| <= 448)."""
    e = torch.floor(torch.log2(y.abs().clamp_min(2.0 ** -20))).clamp_min(-6)
    step = torch.exp2(e - 3)
    return torch.round(y / step) * step


def _exact_page(tokens, held, old, first):
    """One page: tokens [n, Hkv, D] from offset `first` on, held [Hkv, 16, D] codes' values, old [Hkv] scales -> (values of codes, scales)."""
    amax = tokens.abs().amax((0, 2))
    need = torch.exp2(torch.ceil(torch.log2(amax / 448))).clamp_min(LEAST)
    new = torch.maximum(need, old) if first else need
    held = held.clone()
    if first:
        held[:, :first] = _nearest_code(held[:, :first] * (old / new)[:, None, None])
    held[:, first:first + tokens.shape[0]] = _nearest_code(tokens / new[None, :, None]).transpose(0, 1)
    return held, new


def _exact_write(s, k_new, v_new):
    """(values of K codes, of V codes, scales) in 64 bits after the write, in the cache's layouts."""
    hkv, d = s["hkv"], s["d"]
    k, v, scales = s["k"].double(), s["v"].double(), s["scales"].double()
    slots = s["slots"].tolist()
    i = 0
    while i < len(slots):
        n = 1
        while i + n < len(slots) and slots[i + n] == slots[i] + n and slots[i + n] % PAGE:
            n += 1
        page, first = slots[i] // PAGE, slots[i] % PAGE
        held = k[page].permute(0, 2, 1, 3).reshape(hkv, PAGE, d)
        held, scales[page, :, 0] = _exact_page(k_new[i:i + n], held, scales[page, :, 0].clone(), first)
        k[page] = held.view(hkv, PAGE, 4, d // 4).permute(0, 2, 1, 3)
        held, scales[page, :, 1] = _exact_page(v_new[i:i + n], v[page].transpose(1, 2), scales[page, :, 1].clone(), first)
        v[page] = held.transpose(1, 2)
        i += n
    return k, v, scales


def _exact_rows(q, first, pages, k, v, scales, scale):
    """Causal attention of one sequence's rows q [n, Hq, D], the first at position `first`, over its pages."""
    hkv, d = k.shape[1], q.shape[2]
    n, g = q.shape[0], q.shape[1] // hkv
    end = first + n
    pages = pages[: (end + PAGE - 1) // PAGE].long()
    out = torch.empty_like(q)
    for h in range(hkv):
        kh = (k[pages, h].double() * scales[pages, h, 0].double()[:, None, None, None]).permute(0, 2, 1, 3).reshape(-1, d)[:end]
        vh = (v[pages, h].double() * scales[pages, h, 1].double()[:, None, None]).transpose(1, 2).reshape(-1, d)[:end]
        for j in range(h * g, h * g + g):
            x = q[:, j] @ kh.t() * scale
            x = x.masked_fill(torch.arange(end, device=x.device) > first + torch.arange(n, device=x.device)[:, None], float("-inf"))
            out[:, j] = torch.softmax(x, -1) @ vh
    return out


def exact(c, seed):
    s = prepare(c, seed)
    if c["op"] == "logits":
        return _exact_logits(s)
    hq, hkv, d = s["hq"], s["hkv"], s["d"]
    ctx, new = _spans(c)
    if c["op"] == "step":
        x = s["slabs"].double().sum(0).to(torch.bfloat16).double().view(-1, hq + 2 * hkv, d)
        cs = s["cos_sin"].double()[s["positions"].long()]
        z = torch.complex(x[..., : d // 2].contiguous(), x[..., d // 2:].contiguous())[:, : hq + hkv]
        z = z * torch.complex(cs[:, : d // 2].contiguous(), cs[:, d // 2:].contiguous())[:, None]
        qk = torch.cat([z.real, z.imag], -1).to(torch.bfloat16).double()
        q, kn, vn = qk[:, :hq], qk[:, hq:], x[:, hq + hkv:]
    else:
        x = s["qkv"].double().view(-1, hq + 2 * hkv, d)
        q, kn, vn = x[:, :hq], x[:, hq:hq + hkv], x[:, hq + hkv:]
    k, v, scales = s["k"].view(torch.uint8), s["v"].view(torch.uint8), s["scales"]
    got = {}
    if c["op"] in ("write", "step"):
        k, v, scales = _exact_write(s, kn, vn)
        got = dict(k=k, v=v, scales=scales)
    if c["op"] == "write":
        return got
    if k.dtype == torch.uint8:
        codes = torch.arange(256, dtype=torch.int32, device=k.device).to(torch.uint8).view(E4M3).double()
        k, v = codes[k.int()], codes[v.int()]
    at, parts = 0, []
    for i, (a, n) in enumerate(zip(ctx, new)):
        parts.append(_exact_rows(q[at:at + n], a, s["table"][i], k, v, scales, s["scale"]))
        at += n
    o = torch.cat(parts).reshape(-1, hq * d)
    return dict(got, o=o) if got else o


def _exact_logits(s):
    y = s["logits"].double()
    for b, slot in enumerate(s["rows"].tolist()):
        if slot < 0:
            continue
        ids = s["tokens"][s["table"][b].long()].reshape(-1)[: int(s["lens"][b])].long()
        prompt, masked = s["info"][slot].tolist()
        rep, pres, freq = s["params"][slot].double().unbind()
        t = ids.unique()
        y[b, t] = torch.where(y[b, t] > 0, y[b, t] / rep, y[b, t] * rep)
        t, n = ids[prompt:].unique(return_counts=True)
        y[b, t] -= freq * n + pres
        keep = s["bias_ids"][slot] >= 0
        y[b, s["bias_ids"][slot][keep].long()] += s["bias_vals"][slot][keep].double()
        if masked:
            bits = (s["masks"][slot][:, None] >> torch.arange(32, device=y.device)) & 1
            y[b, bits.reshape(-1)[: y.shape[1]] == 0] = float("-inf")
    return y
