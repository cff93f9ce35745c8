"""A paged KV cache held in 8 bits, and the attention that reads it.

Pages are the bf16 cache's: 16 tokens of one sequence, named by block tables.  Keys ``[pages, Hkv, 4, 16, D / 4]`` (four runs of dims, then the
page's tokens) and values ``[pages, Hkv, D, 16]`` are e4m3 codes; ``scales [pages, Hkv, 2]`` (keys', values') fp32 belong to a page and kv
head.  A code stands for its value times the scale: the least power of two, 2^-100 or more, that brings the largest finite magnitude written to
448 or less, and not less than before where the page holds earlier tokens of its sequence - whose codes are then rounded anew, which changes
nothing but codes that become subnormal.  Numbers that are not finite become NaN codes and set no scale.

The operators stand beside ``rope_and_cache``, ``paged_decode``, ``paged_decode_fused`` and ``flash_prefill``, with the cache as one argument.
Head sizes 64 and 128 (the fused form: 128), any 1 to 16 query heads a kv head.  GPU: bf16 rows, the kernels of ``csrc/kv8_*.hip``; CPU: any
floating rows, the forms below.  What a page holds behind a sequence's end does not matter, NaN included; page numbers outside the cache are
held to its ends, block tables end a sequence (rows of a chunk that is longer than its table see all that it holds), slots outside the cache are not written.
"""
from __future__ import annotations

from typing import NamedTuple, Optional

import torch

from . import MAX_SPLITS, _gpu, native, pack_activation, prefill_qblocks
from . import reference as ref

PAGE = 16
E4M3 = torch.float8_e4m3fn
LARGEST = 448.0
LEAST_SCALE = 2.0 ** -100


class KV8(NamedTuple):
    """The pages of one layer."""

    k: torch.Tensor  # [pages, Hkv, 4, 16, D / 4] e4m3
    v: torch.Tensor  # [pages, Hkv, D, 16] e4m3
    scales: torch.Tensor  # [pages, Hkv, 2] fp32

    def layer(self, i: int) -> "KV8":
        """One layer of a cache whose tensors have layers in front."""
        return KV8(self.k[i], self.v[i], self.scales[i])


def kv8_cache(num_blocks: int, Hkv: int, D: int, device=None, layers: Optional[int] = None) -> KV8:
    """An empty cache; with ``layers`` its tensors have that many layers in front (:meth:`KV8.layer`)."""
    if D not in (64, 128):
        raise ValueError(f"kv8_cache: head size 64 or 128, is {D}")
    n = (num_blocks, Hkv) if layers is None else (layers, num_blocks, Hkv)
    return KV8(torch.zeros(*n, 4, PAGE, D // 4, dtype=torch.uint8, device=device).view(E4M3),
               torch.zeros(*n, D, PAGE, dtype=torch.uint8, device=device).view(E4M3),
               torch.zeros(*n, 2, dtype=torch.float32, device=device))


def kv8_block_bytes(Hkv: int, D: int) -> int:
    """Bytes of one page of one layer: keys, values and their scales."""
    return Hkv * (2 * D * PAGE + 8)


def rope_and_cache_kv8(qkv: torch.Tensor, positions: torch.Tensor, cos_sin: torch.Tensor, cache: KV8, slot_mapping: torch.Tensor, Hq: int,
                       Hkv: int, D: int, apply_rope: bool = True, partial: Optional[torch.Tensor] = None, nslabs: int = 0) -> None:
    """In place: rotate q and k inside the fused QKV rows (``apply_rope``; ``positions`` are held to the ends of ``cos_sin``); write k, v into the pages of ``slot_mapping`` [T] (page * 16 + token;
    < 0: not written).  Rows of one page follow one another, in the order of their slots, and go on where the page ends: what it holds at lower
    offsets are earlier tokens of the sequence, and its scale stays theirs or grows.  ``partial``: the rows are first the sum of ``nslabs`` fp32
    split-K slabs [nslabs, T, (Hq + 2 Hkv) * D]."""
    T = qkv.shape[0]
    if partial is not None:
        if qkv.shape[1] != (Hq + 2 * Hkv) * D or not qkv.is_contiguous() or not 1 <= nslabs or partial.numel() < nslabs * qkv.numel():
            raise ValueError("rope_and_cache_kv8: partial must hold nslabs x [T, (Hq + 2 Hkv) * D], qkv be contiguous rows of that many columns")
    if _gpu(qkv):
        native().kv8_write(qkv, positions if apply_rope else None, cos_sin if apply_rope else None, slot_mapping, cache.k, cache.v, cache.scales,
                           Hq, Hkv, D, apply_rope, partial, nslabs)
        return
    runs = _runs(cache, slot_mapping, T)  # (refuses before anything has changed)
    if partial is not None:
        qkv.copy_(partial.reshape(-1)[: nslabs * qkv.numel()].view(nslabs, *qkv.shape).sum(0))
    if apply_rope:
        _rotate(qkv, positions, cos_sin, Hq, Hkv, D)
    x = qkv[:, : (Hq + 2 * Hkv) * D].reshape(T, Hq + 2 * Hkv, D)
    _write(cache, runs, x[:, Hq:Hq + Hkv], x[:, Hq + Hkv:])


def paged_decode_kv8(q: torch.Tensor, cache: KV8, block_tables: torch.Tensor, seq_lens: torch.Tensor, Hq: int, Hkv: int, D: int, scale: float,
                     workspace: Optional[tuple] = None, out: Optional[torch.Tensor] = None, splits: Optional[int] = None) -> torch.Tensor:
    """``paged_decode`` over the 8-bit pages: one query row a sequence (``q`` [B, >= Hq * D]) over its ``seq_lens`` cached tokens; rows of length 0
    are zeros.  ``workspace``: ``decode_workspace``'s, of one stream."""
    if not _gpu(q):
        return _out(_decode_cpu(q, cache, block_tables, seq_lens, Hq, Hkv, D, scale), out)
    B = seq_lens.shape[0]
    S = splits or kv8_splits(B, Hkv)
    if out is None:
        out = torch.empty(B, Hq * D, dtype=q.dtype, device=q.device)
    if workspace is None:
        workspace = _workspace(B, Hq, D, S, q.device)
    native().kv8_decode(out, q, cache.k, cache.v, cache.scales, block_tables, seq_lens, workspace[0], workspace[1],
                        workspace[2] if len(workspace) > 2 else None, Hq, Hkv, D, scale, S)
    return out


def paged_decode_fused_kv8(slabs: torch.Tensor, nslabs: int, positions: torch.Tensor, cos_sin: torch.Tensor, slot_mapping: Optional[torch.Tensor],
                           cache: KV8, block_tables: torch.Tensor, seq_lens: torch.Tensor, Hq: int, Hkv: int, D: int, scale: float,
                           workspace: Optional[tuple] = None, out: Optional[torch.Tensor] = None, splits: Optional[int] = None) -> torch.Tensor:
    """``paged_decode_fused`` over the 8-bit pages (D = 128): q / k / v of the new tokens are the sum of ``nslabs`` fp32 slabs [nslabs, B, (Hq + 2
    Hkv) * D], rounded to bf16, q and k rotated at ``positions`` (held to the ends of ``cos_sin``); k, v go into the page of ``slot_mapping`` (which is the sequence's last one)
    as ``rope_and_cache_kv8`` writes them, and attention is over what the pages then stand for, the new token's codes among them."""
    B = seq_lens.shape[0]
    if not _gpu(slabs):
        n = (Hq + 2 * Hkv) * D
        dtype = out.dtype if out is not None else torch.bfloat16
        qkv = slabs.reshape(-1)[: nslabs * B * n].view(nslabs, B, n).sum(0).to(dtype)
        if slot_mapping is None:
            slot_mapping = torch.full((B,), -1, dtype=torch.int32)
        runs = _runs(cache, slot_mapping, B)
        _rotate(qkv, positions, cos_sin, Hq, Hkv, D)
        x = qkv.view(B, Hq + 2 * Hkv, D)
        kn, vn = x[:, Hq:Hq + Hkv], x[:, Hq + Hkv:]
        _write(cache, runs, kn, vn)
        fresh = [i for i in range(B) if int(slot_mapping[i]) < 0 and int(seq_lens[i]) > 0]
        new = {i: (_as_written(kn[i]), _as_written(vn[i])) for i in fresh}  # not written, attended as if alone in its page
        return _out(_decode_cpu(qkv, cache, block_tables, seq_lens, Hq, Hkv, D, scale, new), out)
    S = splits or kv8_splits(B, Hkv)
    if out is None:
        out = torch.empty(B, Hq * D, dtype=torch.bfloat16, device=slabs.device)
    if workspace is None:
        workspace = _workspace(B, Hq, D, S, slabs.device)
    native().kv8_decode_fused(out, slabs, nslabs, positions, cos_sin, slot_mapping, cache.k, cache.v, cache.scales, block_tables, seq_lens,
                              workspace[0], workspace[1], workspace[2] if len(workspace) > 2 else None, Hq, Hkv, D, scale, S)
    return out


def flash_prefill_kv8(qkv: torch.Tensor, cu_seqlens: torch.Tensor, ctx_start: torch.Tensor, cache: KV8, block_tables: torch.Tensor, Hq: int,
                      Hkv: int, D: int, scale: float, qblocks: Optional[tuple] = None, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Causal attention of prompt chunks: sequence i's rows ``cu_seqlens[i]..`` of ``qkv`` are its tokens at positions ``ctx_start[i]..``, every key
    and value - theirs too - is read from the 8-bit pages (``rope_and_cache_kv8`` has written them).  ``qblocks``: ``prefill_qblocks``'s two
    lists on the device (computed here, with a synchronisation, if not given); rows that none names are left as they are in ``out``."""
    if not _gpu(qkv):
        r = _prefill_cpu(qkv, cu_seqlens, ctx_start, cache, block_tables, Hq, Hkv, D, scale)
        if out is None:
            return r
        cu = cu_seqlens.tolist()
        named = qblocks if qblocks is not None else prefill_qblocks(cu)
        for i, at in zip(*(x.tolist() if torch.is_tensor(x) else x for x in named)):
            if 0 <= i < len(cu) - 1 and at >= 0:
                rows = slice(cu[i] + at, min(cu[i] + at + 128, cu[i + 1]))
                out[rows] = r[rows]
        return out
    if qblocks is None:
        if ctx_start.numel() < cu_seqlens.numel() - 1:
            raise ValueError("flash_prefill_kv8: cu_seqlens [S + 1], ctx_start [S]")
        qs, st = prefill_qblocks(cu_seqlens.tolist(), ctx_starts=ctx_start.tolist())
        qblocks = (torch.tensor(qs, dtype=torch.int32, device=qkv.device), torch.tensor(st, dtype=torch.int32, device=qkv.device))
    if out is None:
        out = torch.empty(qkv.shape[0], Hq * D, dtype=qkv.dtype, device=qkv.device)
    native().kv8_prefill(out, qkv, cu_seqlens, ctx_start, qblocks[0], qblocks[1], cache.k, cache.v, cache.scales, block_tables, Hq, Hkv, D, scale)
    return out


def kv8_splits(B: int, Hkv: int) -> int:
    """Splits of the context per (sequence, kv head): one workgroup a CU, up to the workspace's.  Measured (us): 8 x 32 k tokens, 8 kv heads: 4
    splits 93, 2 146, 8 98; 16 x 2 k: 2 20, 1 25, 4 22; 64 x 1.9 k: 1 51, 2 62; 1 x 100 k, one kv head: 64 30, 32 43."""
    return max(1, min(MAX_SPLITS, round(256 / max(1, B * Hkv))))


def _workspace(B: int, Hq: int, D: int, S: int, device) -> tuple:
    if S == 1:
        e = torch.empty(0, dtype=torch.float32, device=device)
        return e, e
    # (without decode_workspace's counters, which somebody has to clear once: a second launch joins the splits)
    return (torch.empty(B, Hq, S, D, dtype=torch.float32, device=device), torch.empty(B, Hq, S, 2, dtype=torch.float32, device=device))


# ---------------------------------------------------------------- CPU forms

def _out(r: torch.Tensor, out: Optional[torch.Tensor]) -> torch.Tensor:
    if out is None:
        return r
    if out.dim() == 4:  # fragment-packed (gemm_skinny's A operand)
        return out.copy_(pack_activation(r))
    out[: r.shape[0]] = r
    return out


def scale_of(amax: torch.Tensor) -> torch.Tensor:
    """The scale of a page whose largest magnitude is ``amax``."""
    m, e = torch.frexp(amax.float())  # amax = m 2^e, 448 = 0.875 * 2^9
    s = torch.ldexp(torch.ones_like(m), e - torch.where(m > LARGEST / 512, 8, 9))
    return torch.where(amax > 0, s, torch.zeros_like(s)).clamp_min(LEAST_SCALE)


def codes_of(x: torch.Tensor, s: torch.Tensor) -> torch.Tensor:
    """e4m3 codes of ``x`` over ``s`` (NaN where x is not finite)."""
    x = x.float()
    return torch.where(x.isfinite(), x / s, torch.full_like(x, float("nan"))).to(E4M3)


def _finite_max(x: torch.Tensor) -> torch.Tensor:
    x = x.float()
    return torch.where(x.isfinite(), x.abs(), torch.zeros_like(x)).amax(-1)


def _as_written(x: torch.Tensor) -> torch.Tensor:
    """What one token alone in its page stands for: [Hkv, D]."""
    s = scale_of(_finite_max(x))[:, None]
    return codes_of(x, s).float() * s


def _rotate(qkv: torch.Tensor, positions: torch.Tensor, cos_sin: torch.Tensor, Hq: int, Hkv: int, D: int) -> None:
    ref.rope_and_cache(qkv, positions[: qkv.shape[0]].clamp(0, cos_sin.shape[0] - 1), cos_sin, None, None, None, Hq, Hkv, D, True)


def _runs(cache: KV8, slots: torch.Tensor, T: int) -> tuple:
    """Of ``T`` rows: those that are written, their pages, each one's page among them and place in it, the first place of every page."""
    n = cache.scales.shape[0]
    if slots.numel() < T:
        raise ValueError("rope_and_cache_kv8: a slot for each row")
    sm = slots[:T].long()
    rows = ((sm >= 0) & (sm < n * PAGE)).nonzero()[:, 0]
    sm = sm[rows]
    pages, row = torch.unique(sm // PAGE, return_inverse=True)
    off = sm % PAGE
    first = torch.full_like(pages, PAGE).scatter_reduce(0, row, off, "amin")
    start = torch.full_like(pages, 1 << 62).scatter_reduce(0, row, rows, "amin")
    if not torch.equal(off - first[row], rows - start[row]):
        raise ValueError("rope_and_cache_kv8: rows of one page must follow one another in the order of their slots")
    return rows, pages, row, off, first


def _write(cache: KV8, runs: tuple, k_new: torch.Tensor, v_new: torch.Tensor) -> None:
    hkv = cache.scales.shape[1]
    rows, pages, row, off, first = runs
    earlier = torch.arange(PAGE) < first[:, None]  # [pages, 16]
    for j, (codes, x) in enumerate(((cache.k, k_new[rows].float()), (cache.v, v_new[rows].float()))):
        amax = torch.zeros(pages.numel(), hkv).scatter_reduce(0, row[:, None].expand(-1, hkv), _finite_max(x), "amax")
        old = torch.where(first[:, None] > 0, cache.scales[pages, :, j], torch.zeros(()))
        new = torch.maximum(scale_of(amax), old)
        raw = codes.view(torch.uint8)
        held = raw[pages]
        ratio = (old / new)[:, :, None, None]
        at = earlier[:, None, None, :, None] if j == 0 else earlier[:, None, None, :]
        again = (held.view(E4M3).float() * (ratio[..., None] if j == 0 else ratio)).to(E4M3).view(torch.uint8)
        held = torch.where(at & (ratio[..., None] if j == 0 else ratio).ne(1), again, held)
        got = codes_of(x, new[row][..., None]).view(torch.uint8)
        if j == 0:
            held[row, :, :, off, :] = got.view(-1, hkv, 4, got.shape[-1] // 4)
        else:
            held[row, :, :, off] = got
        raw[pages] = held
        cache.scales[pages, :, j] = new


def gather_kv8(cache: KV8, block_table: torch.Tensor, seq_len: int) -> tuple:
    """What one sequence's pages stand for: keys and values [seq_len, Hkv, D] fp32."""
    n, hkv = cache.scales.shape[:2]
    p = block_table[: (seq_len + PAGE - 1) // PAGE].long().clamp(0, n - 1)
    sc = cache.scales[p]
    k = cache.k.view(torch.uint8)[p].view(E4M3).float() * sc[..., 0, None, None, None]
    v = cache.v.view(torch.uint8)[p].view(E4M3).float() * sc[..., 1, None, None]
    D = v.shape[2]
    return (k.permute(0, 3, 1, 2, 4).reshape(-1, hkv, D)[:seq_len], v.permute(0, 3, 1, 2).reshape(-1, hkv, D)[:seq_len])


def _decode_cpu(q, cache, block_tables, seq_lens, Hq, Hkv, D, scale, new=None):
    B = seq_lens.shape[0]
    out = torch.zeros(B, Hq * D, dtype=q.dtype)
    for b in range(B):
        L = min(int(seq_lens[b]), block_tables.shape[1] * PAGE)
        if L <= 0:
            continue
        k, v = gather_kv8(cache, block_tables[b], L)
        if new and b in new:
            k[L - 1], v[L - 1] = new[b]
        out[b] = ref.attention(q[b, : Hq * D].view(1, Hq, D), k, v, scale, causal=False).reshape(-1).to(q.dtype)
    return out


def _prefill_cpu(qkv, cu_seqlens, ctx_start, cache, block_tables, Hq, Hkv, D, scale):
    out = torch.zeros(qkv.shape[0], Hq * D, dtype=qkv.dtype)
    cu, cs = cu_seqlens.tolist(), ctx_start.tolist()
    for i in range(len(cu) - 1):
        a, b = cu[i], cu[i + 1]
        if b > a:
            n = min(b - a, block_tables.shape[1] * PAGE)
            c = max(0, min(cs[i], block_tables.shape[1] * PAGE - n))
            k, v = gather_kv8(cache, block_tables[i], c + n)
            for r0, r1, causal in ((a, a + n, True), (a + n, b, False)):
                q = qkv[r0:r1, : Hq * D].reshape(r1 - r0, Hq, D)
                out[r0:r1] = ref.attention(q, k, v, scale, causal=causal).reshape(r1 - r0, Hq * D).to(qkv.dtype)
    return out
