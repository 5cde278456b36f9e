"""Operators of the 8-bit paged KV cache: step tables, quantised append, attention.

The cache is e4m3 ``[num_blocks, Hkv, block_size, 128]`` for K and for V (block size 16, 32 or
64) with fp32 scales ``[num_blocks, Hkv]``, one per block of tokens and KV head; a stored value
is ``code * scale``.  :func:`rope_kv_fp8` writes powers of two as scales; the attention takes any
positive normal ones, V's within a factor of 2**100 in a sequence and head, and 0 for blocks of
zeros.  One step uses the three together::

    t = ops.step_tables(ctx_lens, q_lens, rows, seq_tables, new_blocks, T, block_size, ...)
    q = ops.rope_kv_fp8(qkv, t.positions, t.slots, cos_sin, k, v, k_scale, v_scale, hq, hkv)
    n, most = ops.work_items(host_q_lens, group)      # entries in use, rows of the longest
    ops.paged_attention_fp8(q, k, v, k_scale, v_scale, t.block_tables, t.seq_lens, t.cu_q, out,
                            group, decode, tile_seq=t.tile_seq[:n], tile_row0=t.tile_row0[:n],
                            item_rows=most)
"""
from __future__ import annotations

import math
from typing import NamedTuple, Optional, Sequence, Tuple

import torch

from . import _launches, _need_c, scratch

FP8_KV_DTYPE = torch.float8_e4m3fn
FP8_MAX = 448.0                            # largest e4m3 value
FP8_SCALE_MIN_EXP, FP8_SCALE_MAX_EXP = -40, 119
MAX_REQUESTS = 4096                        # requests of a step, sequences of a decode call


_err_words: dict = {}       # device index -> error word of its scratch


def _err(t: torch.Tensor) -> torch.Tensor:
    """The error word of ``t``'s device (the scratch's; looked up once per device)."""
    i = t.get_device()
    w = _err_words.get(i)
    if w is None:
        w = _err_words[i] = scratch(t.device).err
    return w


def work_items(q_lens: Sequence[int], group: int, rows_per_tile: int = 256) -> Tuple[int, int]:
    """Of the work list that :func:`step_tables` builds for requests with ``q_lens`` new tokens (those
    from ``num_decode`` on): how many entries are in use, all in front, and the query rows of the
    longest."""
    rows = [int(n) * group for n in q_lens]
    return (sum(-(-r // rows_per_tile) for r in rows),
            min(max(rows, default=0), rows_per_tile))


class StepTables(NamedTuple):
    """Device-side integers of one step (all int32); see :func:`step_tables`."""

    block_tables: torch.Tensor    # [B, W], 0 past a request's last block
    seq_lens: torch.Tensor        # [B] cached tokens after the step
    cu_q: torch.Tensor            # [B + 1] first token row of each request
    positions: torch.Tensor       # [T]
    slots: torch.Tensor           # [T] block * block_size + offset, -1 for rows past the last token
    last_rows: torch.Tensor       # [B] row of the request's last new token, -1 if it has none
    tile_seq: torch.Tensor        # attention work list: request (-1: unused entry) ...
    tile_row0: torch.Tensor       # ... and first packed query row
    num_new: torch.Tensor         # [1] entries of new_blocks taken


def step_tables(ctx_lens: torch.Tensor, q_lens: torch.Tensor, rows: Optional[torch.Tensor],
                seq_tables: torch.Tensor, new_blocks: torch.Tensor, num_tokens: int,
                block_size: int, group: int = 1, rows_per_tile: int = 256,
                num_decode: int = 0) -> StepTables:
    """Block tables, slot map, positions and attention work list of a step, in one launch.

    Request b has ``ctx_lens[b]`` cached tokens, gets ``q_lens[b]`` new ones (0 allowed) and owns
    row ``rows[b]`` (``None``: row b) of the resident ``seq_tables`` [S, W].  The blocks it
    lacks come from ``new_blocks`` in request order and are entered into ``seq_tables`` in place.
    ``num_tokens`` is the number of token rows; rows past the last request's tokens get slot -1.
    The work list has one entry per ``rows_per_tile`` packed query rows (``group`` per token) of
    the requests from ``num_decode`` on.  Lengths below zero or beyond the table's width, rows
    outside ``seq_tables``, too few ``new_blocks`` or too few token rows are reported through
    the error word (:func:`check_errors`); what they concern gets slot -1."""
    b, w = ctx_lens.numel(), seq_tables.shape[1]
    if not 1 <= b <= MAX_REQUESTS:
        raise ValueError(f"step_tables: {b} requests (1 to {MAX_REQUESTS})")
    if num_tokens < 0 or group < 1 or rows_per_tile < 1:
        raise ValueError("step_tables: num_tokens, group, rows_per_tile")
    if block_size < 1 or block_size > 1024 or block_size & (block_size - 1):
        raise ValueError(f"step_tables: block size {block_size} is not a power of two up to 1024")
    if ctx_lens.is_cuda:
        out = StepTables(*_need_c().step_tables(
            ctx_lens, q_lens, rows, seq_tables, new_blocks, num_tokens, block_size, group,
            rows_per_tile, num_decode, _err(ctx_lens)))
        _launches[0] += 1
        return out
    tiles = num_tokens * group // rows_per_tile + b
    out = StepTables(*(torch.zeros(n, dtype=torch.int32) for n in (
        (b, w), b, b + 1, num_tokens, num_tokens, b, tiles, tiles, 1)))
    # CPU restatement
    out.slots.fill_(-1)
    out.tile_seq.fill_(-1)
    tok = used = tile = 0
    for i, (c, n) in enumerate(zip(ctx_lens.tolist(), q_lens.tolist())):
        row = i if rows is None else int(rows[i])
        if c < 0 or n < 0 or not 0 <= row < seq_tables.shape[0] or c + n > w * block_size:
            raise ValueError(f"step_tables: request {i}: lengths ({c}, {n}), row {row}")
        have, need = -(-c // block_size), -(-(c + n) // block_size)
        if used + need - have > new_blocks.numel() or tok + n > num_tokens:
            raise ValueError(f"step_tables: request {i}: too few new blocks or token rows")
        seq_tables[row, have:need] = new_blocks[used:used + need - have]
        out.block_tables[i, :need] = seq_tables[row, :need]
        pos = torch.arange(c, c + n)
        out.positions[tok:tok + n] = pos
        out.slots[tok:tok + n] = (seq_tables[row, pos // block_size] * block_size
                                  + pos % block_size)
        for r in range(0, n * group if i >= num_decode else 0, rows_per_tile):
            out.tile_seq[tile], out.tile_row0[tile] = i, r
            tile += 1
        tok, used = tok + n, used + need - have
        out.seq_lens[i], out.cu_q[i + 1] = c + n, tok
        out.last_rows[i] = tok - 1 if n else -1
    out.num_new[0] = used
    return out


def _pow2_scale(amax: torch.Tensor) -> torch.Tensor:
    """Smallest power of two s with amax / s <= 448 (within the scales' range)."""
    m, e = torch.frexp(amax.clamp(max=3.4e38))
    k = e - 9 + (m > 0.875).int()          # 448 = 0.875 * 2**9
    k = torch.where(amax > 0, k, torch.full_like(k, FP8_SCALE_MIN_EXP))
    return torch.ldexp(torch.ones_like(amax), k.clamp(FP8_SCALE_MIN_EXP, FP8_SCALE_MAX_EXP))


def rope_kv_fp8(qkv: torch.Tensor, positions: torch.Tensor, slots: torch.Tensor,
                cos_sin: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor,
                k_scale: torch.Tensor, v_scale: torch.Tensor, hq: int, hkv: int,
                q_norm: Optional[torch.Tensor] = None, k_norm: Optional[torch.Tensor] = None,
                norm_dim: int = 0, eps: float = 1e-6,
                out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Rotate q and k of ``qkv`` [T, (hq + 2 hkv) 128] (optional per-head RMSNorm first) and
    append k, v to the 8-bit cache at ``slots`` (-1: not stored).  Returns the rotated q
    [T, hq, 128]; ``qkv`` is left as it is.

    A block's scale is the smallest power of two that brings the largest magnitude of its tokens
    to 448 or below.  A block that this call enters at offset 0 is new: its scale comes from this
    call's tokens.  Otherwise the scale only grows, and the tokens stored before the call's first
    offset are rescaled.  Tokens are appended in order: what lies behind the call's last offset
    does not count as stored, and the rows that go to one block lie within ``block_size``
    consecutive rows, offsets rising.  Infinities are stored as the largest magnitude, NaN as
    NaN."""
    if qkv.is_cuda:
        _launches[0] += 1
        return _need_c().rope_kv_fp8(qkv, positions, slots, cos_sin, k_cache, v_cache, k_scale,
                                     v_scale, out, hq, hkv, q_norm, k_norm, norm_dim, eps,
                                     _err(qkv))
    # CPU restatement
    t, d = qkv.shape[0], k_cache.shape[-1]
    if out is None:
        out = torch.empty(t, hq, d, dtype=qkv.dtype)
    r, bs = cos_sin.shape[1], k_cache.shape[2]
    half = r // 2
    x = qkv[:, :(hq + 2 * hkv) * d].reshape(t, hq + 2 * hkv, d).float()
    cs = cos_sin[positions[:t].long()][:, None]
    c, s = cs[..., :half], cs[..., half:]
    parts = []
    for lo, hi, nw in ((0, hq, q_norm), (hq, hq + hkv, k_norm)):
        y = x[:, lo:hi]
        if nw is not None:
            y = y * torch.rsqrt(y.pow(2).sum(-1, keepdim=True) / (norm_dim or r) + eps) \
                * nw.float()
        y1, y2 = y[..., :half], y[..., half:r]
        parts.append(torch.cat([y1 * c - y2 * s, y1 * s + y2 * c, y[..., r:]], -1))
    out.copy_(parts[0].to(out.dtype))
    groups: dict = {}
    for i, sl in enumerate(slots[:t].tolist()):
        if sl >= 0:
            groups.setdefault(sl // bs, []).append((sl % bs, i))
    for y, cache, scale in ((parts[1], k_cache, k_scale), (x[:, hq + hkv:], v_cache, v_scale)):
        codes = cache.view(torch.uint8)
        for blk, toks in groups.items():
            y_b = y[[i for _, i in toks]]                               # [n, hkv, d]
            new = _pow2_scale(torch.nan_to_num(y_b.abs(), nan=0.0).amax((0, 2)))
            first = toks[0][0]
            if first > 0:
                old = scale[blk].clone()
                new = torch.maximum(new, old)
                kept = cache[blk, :, :first].float() * (old / new)[:, None, None]
                codes[blk, :, :first] = kept.to(FP8_KV_DTYPE).view(torch.uint8)
            q8 = (y_b / new[:, None]).clamp(-FP8_MAX, FP8_MAX).to(FP8_KV_DTYPE)
            codes[blk][:, [o for o, _ in toks]] = q8.view(torch.uint8).transpose(0, 1)
            scale[blk] = new
    return out


def paged_attention_fp8(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor,
                        k_scale: torch.Tensor, v_scale: torch.Tensor,
                        block_tables: torch.Tensor, seq_lens: torch.Tensor,
                        cu_q: Optional[torch.Tensor], out: torch.Tensor, group: int,
                        decode: bool, tile_seq: Optional[torch.Tensor] = None,
                        tile_row0: Optional[torch.Tensor] = None, causal: bool = True,
                        scale: Optional[float] = None, item_rows: int = 0) -> torch.Tensor:
    """Attention over the 8-bit cache; q, out [T, Hq, 128] bf16 (rows may be strided).

    ``decode``: token i belongs to sequence i and sees its ``seq_lens[i]`` keys.  Otherwise
    ``cu_q`` delimits each sequence's query tokens, the last of its keys, and the work list
    (``tile_seq``, ``tile_row0``: one entry per 256 packed rows, -1 entries skipped) says which
    sequences are computed; with ``causal`` a token sees the keys up to its own.  Rows without a
    visible key give 0; NaN among a sequence's values reaches its rows that share a tile of keys with
    it, seen or not.  ``scale`` defaults to 1 / sqrt(128) (pass 1 / sqrt(true head_dim) for
    zero-padded heads).

    ``item_rows``: query rows (tokens times ``group``) of the work list's longest item, which decides
    the kernel; results do not depend on it but for rounding.  0: the mean of q's rows over the list's
    entries stands in for it, so a list with many -1 entries, or a q with many rows that are not the
    list's, should come with the number (:func:`work_items`)."""
    d = q.shape[-1]
    if scale is None:
        scale = 1.0 / math.sqrt(d)
    if item_rows < 0:
        raise ValueError(f"paged_attention_fp8: item_rows {item_rows}")
    if q.is_cuda:
        _launches[0] += _need_c().paged_attention_fp8(
            q, k_cache, v_cache, k_scale, v_scale, out, block_tables, seq_lens, cu_q, tile_seq,
            tile_row0, group, scale, decode, causal, item_rows, _err(q))
        return out
    # CPU restatement
    from ..models.reference import attention_ref
    bs = k_cache.shape[2]
    seqs = range(seq_lens.shape[0]) if decode else \
        sorted({i for i in tile_seq.tolist() if i >= 0})
    for i in seqs:
        n = int(seq_lens[i])
        q0, q1 = (i, i + 1) if decode else (int(cu_q[i]), int(cu_q[i + 1]))
        out[q0:q1] = 0
        if q1 == q0 or n == 0:
            continue
        ids = block_tables[i, :-(-n // bs)].long()
        k, v = ((c.view(torch.uint8)[ids].view(FP8_KV_DTYPE).float() * s[ids][..., None, None])
                .permute(0, 2, 1, 3).reshape(-1, c.shape[1], d)[:n]
                for c, s in ((k_cache, k_scale), (v_cache, v_scale)))
        skip = max(0, q1 - q0 - n) if causal else 0      # tokens before the first key
        qpos = torch.arange(n - (q1 - q0) + skip, n)
        o = attention_ref(q[q0 + skip:q1], k, v, qpos, torch.arange(n), causal=causal,
                          scale=scale)
        out[q0 + skip:q1] = o.to(out.dtype)
    return out
