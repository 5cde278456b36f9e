"""Measured cases of the 8-bit paged KV cache: the step's tables, the append and the attention.

* ``tables``  : ``ops.step_tables``, the block tables, slot map, positions and attention work
  list of one step, built on the device from the requests' lengths;
* ``append``  : ``ops.rope_kv_fp8``, RoPE (optional per-head RMSNorm) of q and k and the
  quantised append of k and v to the paged cache, one power-of-two scale per block and KV head;
* ``decode``  : ``ops.paged_attention_fp8`` with one query token per sequence;
* ``prefill`` : ``ops.paged_attention_fp8`` for chunked prefill and speculative verification.

The cache is e4m3 [blocks, KV heads, block size, 128]; a stored value times its block's scale
is the value it stands for.  Heads are 128 wide, as everywhere on the device.
"""
import math
import random

import torch

own = False

D = 128                 # device head width
FP8_MAX = 448.0         # largest e4m3 value
MIN_EXP, MAX_EXP = -40, 119     # scales are 2**MIN_EXP .. 2**MAX_EXP
ROWS_PER_TILE = 256     # packed query rows per entry of the attention work list
E4M3 = torch.float8_e4m3fn


# --------------------------------------------------------------------------------------
# cases
# --------------------------------------------------------------------------------------
def listed():
    return [
        # a full decode batch: one token per request, a block in sixteen is new; two rows of
        # the batch are padding
        {"name": "tables-decode-256", "op": "tables", "batch": 256, "ctx": 2304, "chunk": 1,
         "block": 16, "group": 4, "empty": 2},
        # a prefill step of 512-token chunks behind long contexts
        {"name": "tables-chunks-40x512", "op": "tables", "batch": 40, "ctx": 30000,
         "chunk": 512, "block": 16, "group": 8, "empty": 0},
        # single-stream decode: latency
        {"name": "append-1", "op": "append", "batch": 1, "chunk": 1, "hq": 32, "hkv": 8,
         "rot": 128, "norm": False, "block": 16},
        # a full decode batch
        {"name": "append-256", "op": "append", "batch": 256, "chunk": 1, "hq": 32, "hkv": 8,
         "rot": 128, "norm": False, "block": 16},
        # ragged prefill chunks with per-head norms
        {"name": "append-16x512-norm", "op": "append", "batch": 16, "chunk": 512, "hq": 32,
         "hkv": 8, "rot": 128, "norm": True, "block": 16},
        # one short conversation: latency of a split context
        {"name": "decode-1x2047", "op": "decode", "batch": 1, "ctx": 2047, "chunk": 1,
         "ragged": False, "hq": 32, "hkv": 8, "block": 16},
        # the serving batch: ragged contexts up to prompt 2048 + 256 generated
        {"name": "decode-256x2304", "op": "decode", "batch": 256, "ctx": 2304, "chunk": 1,
         "ragged": True, "hq": 32, "hkv": 8, "block": 16},
        # multi-head attention (a KV head per query head), odd batch
        {"name": "decode-mha-37x3001", "op": "decode", "batch": 37, "ctx": 3001, "chunk": 1,
         "ragged": True, "hq": 32, "hkv": 32, "block": 16},
        # few long documents, group of eight, larger blocks
        {"name": "decode-7x100k", "op": "decode", "batch": 7, "ctx": 100003, "chunk": 1,
         "ragged": True, "hq": 64, "hkv": 8, "block": 64},
        # speculative verification: five tokens of every sequence
        {"name": "verify-32x5", "op": "prefill", "batch": 32, "ctx": 1280, "chunk": 5,
         "ragged": True, "hq": 32, "hkv": 8, "block": 16},
        # two 512-token chunks behind 4k of context
        {"name": "prefill-2x512-4k", "op": "prefill", "batch": 2, "ctx": 4096, "chunk": 512,
         "ragged": False, "hq": 32, "hkv": 8, "block": 16},
        # a long document's chunk
        {"name": "prefill-1x2048-18k", "op": "prefill", "batch": 1, "ctx": 18432, "chunk": 2048,
         "ragged": False, "hq": 32, "hkv": 8, "block": 32},
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    """One more case: sizes spread over the logarithm of their range, each kind's cost bounded
    by the largest listed case of the kind."""
    op = rng.choice(["tables", "append", "decode", "decode", "prefill"])
    block = rng.choice([16, 16, 32, 64])
    if op == "tables":
        chunk = rng.choice([1, 1, _log(rng, 2, 512)])
        batch = _log(rng, 1, 512 if chunk == 1 else max(1, 20000 // chunk))
        batch = min(batch, 512)
        cap = max(16, min(30000, 40 * 25000 * block // 16 // batch))
        return {"op": op, "batch": batch, "ctx": _log(rng, 16, cap),
                "chunk": chunk, "block": block, "group": rng.choice([1, 3, 4, 7, 8, 16]),
                "empty": rng.randrange(0, 1 + batch // 8)}
    hkv = rng.choice([1, 2, 3, 4, 8, 8, 16, 32])
    hq = min(64, hkv * rng.choice([1, 2, 3, 4, 4, 5, 7, 8, 16])) // hkv * hkv
    if op == "append":
        chunk = rng.choice([1, 1, _log(rng, 2, 700)])
        cap = 6600 * 48 // (hq + 2 * hkv) // chunk
        return {"op": op, "batch": _log(rng, 1, max(1, min(512, cap))), "chunk": chunk, "hq": hq,
                "hkv": hkv, "rot": rng.choice([128, 128, 96, 64]), "norm": rng.random() < 0.4,
                "block": block}
    if op == "decode":
        batch = _log(rng, 1, 400)
        cap = 7 * 100003 * 8 // 3 // (batch * hkv)
        return {"op": op, "batch": batch, "ctx": _log(rng, 1, max(1, min(100003, cap))),
                "chunk": 1, "ragged": rng.random() < 0.8, "hq": hq, "hkv": hkv, "block": block}
    chunk = _log(rng, 1, 2048)
    batch = _log(rng, 1, max(1, min(64, 4096 // chunk)))
    cap = 32 * 2048 * 18432 // 2 // (hq * batch * chunk)
    ctx = max(chunk, _log(rng, 16, max(16, min(20000, cap))))
    return {"op": op, "batch": batch, "ctx": ctx, "chunk": chunk, "ragged": rng.random() < 0.8,
            "hq": hq, "hkv": hkv, "block": block}


def _spread(rng, lo, hi, n):
    """n integers spread evenly over [lo, hi] with some jitter, shuffled: ragged lengths whose sum
    hardly depends on the seed."""
    v = [lo + int((hi - lo) * (i + rng.random()) / n) for i in range(n)]
    rng.shuffle(v)
    return v


def _lengths(case, seed):
    """Host integers of a case (what a scheduler knows): (context before the step, new tokens)
    per request.  Decode and prefill count the step's own tokens in the context they read.  The
    pairs belong to the case, their order to the seed, so every seed has the same shapes."""
    rng = random.Random(case["batch"] * 1009 + case["chunk"] * 31 + case.get("ctx", 0))
    b, op, chunk = case["batch"], case["op"], case["chunk"]
    if op == "tables":
        q = [1] * b if chunk == 1 else \
            [rng.choice([chunk, rng.randint(1, chunk)]) for _ in range(b)]
        ctx = [rng.randint(0, case["ctx"]) for _ in range(b)]
        for i in range(b - case["empty"], b):
            q[i] = ctx[i] = 0
    elif op == "append":
        q = [chunk - rng.randrange(1 + chunk // 5) for _ in range(b)]
        ctx = [rng.randint(0, 3 * case["block"]) + rng.choice([0, 0, 1024]) for _ in range(b)]
    elif not case["ragged"]:
        ctx, q = [case["ctx"]] * b, [chunk] * b
    elif op == "decode":
        ctx, q = _spread(rng, max(1, case["ctx"] // 18), case["ctx"], b), [1] * b
        if b > 8:
            ctx[rng.randrange(b)] = 0       # a padded row: no key to attend to
    else:
        q = _spread(rng, max(1, chunk // 2), chunk, b)
        ctx = [max(n, c) for n, c in zip(q, _spread(rng, 1, case["ctx"], b))]
    order = list(range(b))
    random.Random(seed * 7919 + 13).shuffle(order)
    return [ctx[i] for i in order], [q[i] for i in order]


# --------------------------------------------------------------------------------------
# inputs
# --------------------------------------------------------------------------------------
def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _i32(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def _pow2_scale(amax):
    """Smallest power of two s with amax / s <= 448, in [2**MIN_EXP, 2**MAX_EXP]."""
    m, e = torch.frexp(amax)
    k = torch.where(m <= 0.875, e - 9, e - 8)
    k = torch.where(amax > 0, k, torch.full_like(k, MIN_EXP)).clamp(MIN_EXP, MAX_EXP)
    return torch.ldexp(torch.ones_like(amax), k)


def _cache(shape, gen, heavy, chunk=2048):
    """A filled cache and its scales.  ``heavy``: a few channels eight times the others (keys),
    else magnitudes that differ from block to block (values)."""
    n, h, bs, _ = shape
    data = torch.empty(shape, dtype=E4M3, device="cuda")
    scale = torch.empty(n, h, device="cuda")
    ch = torch.ones(D, device="cuda")
    ch[torch.randperm(D, generator=gen, device="cuda")[:2]] = 8.0
    for i in range(0, n, chunk):
        j = min(n, i + chunk)
        x = torch.randn(j - i, h, bs, D, generator=gen, device="cuda")
        x = x * ch if heavy else \
            x * torch.exp(torch.randn(j - i, h, 1, 1, generator=gen, device="cuda"))
        s = _pow2_scale(x.abs().amax((2, 3)))
        data[i:j] = (x / s[:, :, None, None]).to(E4M3)
        scale[i:j] = s
    return data, scale


def _paged(case, seed, lens):
    """Caches, scales and block tables for sequences of the given lengths: blocks in random
    order; what lies past a sequence's end, and blocks that nobody owns, hold NaN."""
    g, bs, hkv = _gen(seed), case["block"], case["hkv"]
    counts = [-(-n // bs) for n in lens]
    used, width = sum(counts), max(1, max(counts))
    nb = used + 3
    order = torch.randperm(nb, generator=g, device="cuda").to(torch.int32)
    c = _i32(counts)
    col = torch.arange(width, device="cuda", dtype=torch.int32)
    first = torch.cumsum(c, 0) - c
    idx = first[:, None] + col
    tables = torch.where(col < c[:, None], order[idx.clamp(max=nb - 1).long()], 0).int()
    k, ks = _cache((nb, hkv, bs, D), g, True)
    v, vs = _cache((nb, hkv, bs, D), g, False)
    dead = torch.ones(nb, bs, dtype=torch.bool, device="cuda")
    pos = torch.arange(width * bs, device="cuda").view(width, bs)
    live = pos < _i32(lens)[:, None, None]
    ok = col < c[:, None]
    dead[tables[ok].long()] = ~live[ok]
    for t in (k, v):
        t.view(torch.uint8).masked_fill_(dead[:, None, :, None], 0x7F)
    for t in (ks, vs):
        t.masked_fill_(dead.all(1)[:, None], float("nan"))
    return k, v, ks, vs, tables


def prepare(case, seed):
    ctx, q = _lengths(case, seed)
    g = _gen(seed + 1)
    s = {"case": dict(case)}
    if case["op"] == "tables":
        b, bs = case["batch"], case["block"]
        width = (case["ctx"] + case["chunk"]) // bs + 1
        rows = 2 * b + 3                      # requests resident on the device
        pool = rows * width + b * (case["chunk"] // bs + 2)
        ids = torch.randperm(pool, generator=g, device="cuda").to(torch.int32)
        s["seq_tables"] = ids[:rows * width].view(rows, width).clone()
        s["new_blocks"] = ids[rows * width:].clone()
        s["rows"] = torch.randperm(rows, generator=g, device="cuda")[:b].to(torch.int32)
        s["ctx"], s["q"], s["tokens"] = _i32(ctx), _i32(q), sum(q)
        return s
    hq, hkv, bs = case["hq"], case["hkv"], case["block"]
    if case["op"] == "append":
        t = sum(q)
        heads = hq + 2 * hkv
        x = torch.randn(t, heads, D, generator=g, device="cuda")
        x *= torch.exp(0.7 * torch.randn(t, heads, 1, generator=g, device="cuda"))
        x[..., case["rot"]:] = 0              # zero-padded lanes of narrower heads
        s["qkv"] = x.bfloat16().view(t, heads * D)
        # only the blocks that the step writes to, and a few that it does not
        first = [c // bs for c in ctx]
        counts = [(c + n - 1) // bs - f + 1 for c, n, f in zip(ctx, q, first)]
        nb = sum(counts) + 5
        order = torch.randperm(nb, generator=g, device="cuda")
        s["k"], s["ks"] = _cache((nb, hkv, bs, D), g, True)
        s["v"], s["vs"] = _cache((nb, hkv, bs, D), g, False)
        qt, ct, n_blk = _i32(q), _i32(ctx), _i32(counts)
        seq = torch.repeat_interleave(torch.arange(len(q), device="cuda"), qt.long())
        pos = torch.arange(t, device="cuda") - (torch.cumsum(qt, 0) - qt)[seq] + ct[seq]
        blk = order[(torch.cumsum(n_blk, 0) - n_blk)[seq] + pos // bs - ct[seq] // bs]
        s["pos"], s["slots"] = pos.int(), (blk * bs + pos % bs).int()
        if t > 8:
            s["slots"][t // 2] = -1           # a padded row: nothing is stored
        half = case["rot"] // 2
        inv = 5e5 ** (-torch.arange(half, device="cuda", dtype=torch.float64) / half)
        ang = torch.arange(4096, device="cuda", dtype=torch.float64)[:, None] * inv
        s["cs"] = torch.cat([ang.cos(), ang.sin()], 1).float()
        s["qn"] = s["kn"] = None
        if case["norm"]:
            s["qn"], s["kn"] = ((1 + 0.2 * torch.randn(D, generator=g, device="cuda")).bfloat16()
                                for _ in range(2))
        return s
    s["k"], s["v"], s["ks"], s["vs"], s["tables"] = _paged(case, seed + 2, ctx)
    t = sum(q)
    # q is the head of a fused projection's row, as the model has it
    s["q"] = torch.randn(t, (hq + 2 * hkv) * D, generator=g,
                         device="cuda").bfloat16()[:, :hq * D].view(t, hq, D)
    s["lens"] = _i32(ctx)
    s["cu_q"] = _i32([0] + torch.tensor(q).cumsum(0).tolist())
    s["max_q"] = max(q)
    s["tile_seq"] = s["tile_row0"] = None
    if case["op"] == "prefill":
        tiles = [(i, r) for i, n in enumerate(q)
                 for r in range(0, n * (hq // hkv), ROWS_PER_TILE)]
        s["tile_seq"], s["tile_row0"] = _i32([a for a, _ in tiles]), _i32([r for _, r in tiles])
    return s


# --------------------------------------------------------------------------------------
# plain forms
# --------------------------------------------------------------------------------------
def _plain_tables(s):
    c = s["case"]
    bs, group, t = c["block"], c["group"], s["tokens"]
    ctx, q, rows = s["ctx"], s["q"], s["rows"].long()
    b, total = ctx.numel(), ctx + q
    have, need = (ctx + bs - 1) // bs, (total + bs - 1) // bs
    new = need - have
    end = torch.cumsum(new, 0)
    tab = s["seq_tables"][rows]
    col = torch.arange(tab.shape[1], device="cuda")
    idx = (end - new)[:, None] + col - have[:, None]
    is_new = (col >= have[:, None]) & (col < need[:, None])
    tab = torch.where(is_new, s["new_blocks"][idx.clamp(0, s["new_blocks"].numel() - 1)], tab)
    s["seq_tables"][rows] = tab
    tab = torch.where(col < need[:, None], tab, 0)
    cu = torch.cat([torch.zeros_like(q[:1]), torch.cumsum(q, 0).int()])
    i = torch.arange(t, device="cuda", dtype=torch.int32)
    seq = torch.searchsorted(cu[1:].contiguous(), i, right=True)
    pos = ctx[seq] + i - cu[seq]
    slots = tab[seq, (pos // bs).long()] * bs + pos % bs
    n = (q * group + ROWS_PER_TILE - 1) // ROWS_PER_TILE
    tend = torch.cumsum(n, 0)
    j = torch.arange(t * group // ROWS_PER_TILE + b, device="cuda")
    ts = torch.searchsorted(tend, j, right=True)
    real = ts < b
    ts = ts.clamp(max=b - 1)
    row0 = (j - (tend - n)[ts]) * ROWS_PER_TILE
    return {"seq_tables": s["seq_tables"], "block_tables": tab, "seq_lens": total, "cu_q": cu,
            "positions": pos, "slots": slots,
            "last_rows": torch.where(q > 0, cu[1:] - 1, -1),
            "tile_seq": torch.where(real, ts, -1).int(),
            "tile_row0": torch.where(real, row0, 0).int(), "num_new": end[-1:].int()}


def _plain_append(s):
    c = s["case"]
    hq, hkv, rot, bs = c["hq"], c["hkv"], c["rot"], c["block"]
    x = s["qkv"].view(-1, hq + 2 * hkv, D).float()
    t, half, nb = x.shape[0], rot // 2, s["k"].shape[0]
    q, k, v = x[:, :hq], x[:, hq:hq + hkv], x[:, hq + hkv:]
    if c["norm"]:
        q = q * torch.rsqrt((q * q).sum(-1, keepdim=True) / rot + 1e-6) * s["qn"].float()
        k = k * torch.rsqrt((k * k).sum(-1, keepdim=True) / rot + 1e-6) * s["kn"].float()
    cs = s["cs"][s["pos"].long()][:, None]
    co, si = cs[..., :half], cs[..., half:]
    turn = lambda y: torch.cat([y[..., :half] * co - y[..., half:rot] * si,  # noqa: E731
                                y[..., :half] * si + y[..., half:rot] * co, y[..., rot:]], -1)
    q, k = turn(q).bfloat16(), turn(k)
    # rows without a slot go to a block past the end, which is dropped
    sl = s["slots"].long()
    blk = torch.where(sl >= 0, sl // bs, nb)
    off = torch.where(sl >= 0, sl % bs, 0)
    first = torch.full((nb + 1,), bs, device="cuda", dtype=torch.int64)
    first = first.scatter_reduce(0, blk, off, "amin")[:nb, None]
    old = torch.arange(bs, device="cuda") < first              # tokens that were there before
    out = {"q": q}
    for name, y, data, scale in (("k", k, s["k"], s["ks"]), ("v", v, s["v"], s["vs"])):
        top = y.abs().amax(-1).clamp(max=3.4e38)
        need = torch.zeros(nb + 1, hkv, device="cuda")
        need = need.scatter_reduce(0, blk[:, None].expand(t, hkv), top, "amax")[:nb]
        need = _pow2_scale(need)
        now = torch.where(first == 0, need, torch.maximum(scale, need))
        now = torch.where(first < bs, now, scale)
        kept = data.float() * torch.where((first > 0) & (first < bs), scale / now,
                                          1.0)[:, :, None, None]
        kept = torch.where(old[:, None, :, None], kept, data.float()).to(E4M3)
        full = torch.cat([kept.view(torch.uint8),
                          torch.zeros_like(kept[:1]).view(torch.uint8)])
        s_tok = torch.cat([now, torch.ones_like(now[:1])])[blk]
        full[blk, :, off] = (y / s_tok[..., None]).clamp(-FP8_MAX,
                                                         FP8_MAX).to(E4M3).view(torch.uint8)
        data.copy_(full[:nb].view(E4M3))
        scale.copy_(now)
        out[name], out[name + "_scale"] = data, scale
    return out


def _values(data, scale, tables):
    """[B, KV heads, keys, 128] in 32 bits of the blocks in ``tables`` [B, W]."""
    b, w = tables.shape
    x = data.view(torch.uint8)[tables.long()].view(E4M3).float()
    x = x * scale[tables.long()][..., None, None]
    return x.permute(0, 2, 1, 3, 4).reshape(b, x.shape[2], w * x.shape[3], D)


def _plain_attention(s):
    c = s["case"]
    hq, hkv = c["hq"], c["hkv"]
    group = hq // hkv
    lens, cu, mq = s["lens"], s["cu_q"], s["max_q"]
    b, t = lens.numel(), s["q"].shape[0]
    n = cu[1:] - cu[:-1]
    j = torch.arange(mq, device="cuda")
    rows = (cu[:-1, None] + torch.minimum(j, n[:, None] - 1)).long()       # [B, mq]
    q = s["q"][rows].float().view(b, mq, hkv, group, D).permute(0, 2, 3, 1, 4)
    q = q.reshape(b, hkv, group * mq, D)
    k = _values(s["k"], s["ks"], s["tables"])
    key = torch.arange(k.shape[2], device="cuda")
    # a query token at index j of n new ones sees the keys up to its own
    seen = key <= (lens - n)[:, None, None] + j[:, None]                    # [B, mq, L]
    seen &= key < lens[:, None, None]
    seen = seen[:, None, None].expand(b, 1, group, mq, key.numel()).reshape(
        b, 1, group * mq, key.numel())
    p = torch.matmul(q, k.transpose(2, 3))
    del k
    p = p.mul_(D ** -0.5).masked_fill_(~seen, -math.inf)
    top = p.amax(-1, keepdim=True)
    top = torch.where(top == -math.inf, 0.0, top)
    p = p.sub_(top).exp_()
    del seen
    total = p.sum(-1, keepdim=True)
    v = _values(s["v"], s["vs"], s["tables"])
    v = torch.where((key < lens[:, None])[:, None, :, None], v, 0.0)
    o = torch.matmul(p, v) / torch.where(total == 0, 1.0, total)
    o = o.view(b, hkv, group, mq, D).permute(0, 3, 1, 2, 4).reshape(b, mq, hq, D)
    i = torch.arange(t, device="cuda", dtype=torch.int32)
    seq = torch.searchsorted(cu[1:].contiguous(), i, right=True)
    return {"out": o[seq, (i - cu[seq]).long()].bfloat16()}


# --------------------------------------------------------------------------------------
# one pass
# --------------------------------------------------------------------------------------
def run(s):
    c = s["case"]
    op = c["op"]
    if not own:
        return {"tables": _plain_tables, "append": _plain_append}.get(op, _plain_attention)(s)
    from lightbulb_b200 import ops
    if op == "tables":
        r = ops.step_tables(s["ctx"], s["q"], s["rows"], s["seq_tables"], s["new_blocks"],
                            s["tokens"], c["block"], group=c["group"],
                            rows_per_tile=ROWS_PER_TILE)
        return {"seq_tables": s["seq_tables"], "block_tables": r.block_tables,
                "seq_lens": r.seq_lens, "cu_q": r.cu_q, "positions": r.positions,
                "slots": r.slots, "last_rows": r.last_rows, "tile_seq": r.tile_seq,
                "tile_row0": r.tile_row0, "num_new": r.num_new}
    if op == "append":
        q = ops.rope_kv_fp8(s["qkv"], s["pos"], s["slots"], s["cs"], s["k"], s["v"], s["ks"],
                            s["vs"], c["hq"], c["hkv"], q_norm=s["qn"], k_norm=s["kn"],
                            norm_dim=c["rot"])
        return {"q": q, "k": s["k"], "k_scale": s["ks"], "v": s["v"], "v_scale": s["vs"]}
    q = s["q"]
    out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
    ops.paged_attention_fp8(q, s["k"], s["v"], s["ks"], s["vs"], s["tables"], s["lens"],
                            s["cu_q"], out, c["hq"] // c["hkv"], decode=op == "decode",
                            tile_seq=s["tile_seq"], tile_row0=s["tile_row0"])
    return {"out": out}


# --------------------------------------------------------------------------------------
# 64 bits
# --------------------------------------------------------------------------------------
def exact(case, seed):
    if case["op"] == "tables":
        return None
    s = prepare(case, seed)
    hq, hkv, bs = case["hq"], case["hkv"], case["block"]
    if case["op"] == "append":
        rot = case["rot"]
        x = s["qkv"].view(-1, hq + 2 * hkv, D).double()
        ang = s["cs"].double()[s["pos"].long()]
        pair = torch.complex(ang[:, :rot // 2], ang[:, rot // 2:])[:, None]

        def turned(y, w):
            if w is not None:
                y = y / ((y ** 2).sum(-1, keepdim=True) / rot + 1e-6).sqrt() * w.double()
            z = torch.complex(y[..., :rot // 2], y[..., rot // 2:rot].contiguous()) * pair
            return torch.cat([z.real, z.imag, y[..., rot:]], -1)

        out = {"q": turned(x[:, :hq], s["qn"])}
        slots = s["slots"].tolist()
        runs = {}
        for i, sl in enumerate(slots):
            if sl >= 0:
                runs.setdefault(sl // bs, []).append((sl % bs, i))
        for name, y, data, scale in (("k", turned(x[:, hq:hq + hkv], s["kn"]), s["k"], s["ks"]),
                                     ("v", x[:, hq + hkv:], s["v"], s["vs"])):
            val, sc = data.double(), scale.double()
            for blk, toks in runs.items():
                rows = y[[i for _, i in toks]]                               # [n, hkv, D]
                top = rows.abs().amax((0, 2)).clamp(min=2.0 ** -60)
                e = torch.ceil(torch.log2(top / FP8_MAX) - 1e-9).clamp(MIN_EXP, MAX_EXP)
                new = torch.ldexp(torch.ones_like(top), e)
                first = toks[0][0]
                if first:
                    new = torch.maximum(new, sc[blk])
                    val[blk, :, :first] *= (sc[blk] / new)[:, None, None]
                sc[blk] = new
                val[blk][:, [o for o, _ in toks]] = (rows / new[:, None]).transpose(0, 1)
            out[name], out[name + "_scale"] = val, sc
        return out
    lens, cu = s["lens"].tolist(), s["cu_q"].tolist()
    if hq * max(1, s["max_q"]) * max(lens) * case["batch"] > 3e9:
        return None
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    for i, n in enumerate(lens):
        if n == 0:
            continue
        ids = s["tables"][i, :-(-n // bs)].long()
        for h in range(hkv):
            kv = [(d[ids, h].double() * sc[ids, h].double()[:, None, None]).view(-1, D)[:n]
                  for d, sc in ((s["k"], s["ks"]), (s["v"], s["vs"]))]
            heads = slice(h * (hq // hkv), (h + 1) * (hq // hkv))
            q = s["q"][cu[i]:cu[i + 1], heads].double()
            z = torch.einsum("tgd,kd->gtk", q, kv[0]) / math.sqrt(D)
            m = q.shape[0]
            hide = torch.ones(m, n, dtype=torch.bool, device="cuda").triu(n - m + 1)
            w = torch.softmax(z.masked_fill(hide, -math.inf), -1)
            out[cu[i]:cu[i + 1], heads] = torch.einsum("gtk,kd->tgd", w, kv[1])
    return {"out": out}


# --------------------------------------------------------------------------------------
# what a pass cannot do without
# --------------------------------------------------------------------------------------
def work(case):
    ctx, q = _lengths(case, 0)
    t, b, bs = sum(q), case["batch"], case["block"]
    if case["op"] == "tables":
        width = (case["ctx"] + case["chunk"]) // bs + 1
        have = sum(-(-c // bs) for c in ctx)
        need = sum(-(-(c + n) // bs) for c, n in zip(ctx, q))
        tiles = t * case["group"] // ROWS_PER_TILE + b
        return {"bytes": 4 * (3 * b + have + 2 * (need - have) + b * width + 2 * t + 3 * b + 2
                              + 2 * tiles), "flops": 0}
    hq, hkv = case["hq"], case["hkv"]
    if case["op"] == "append":
        blocks = sum((c + n - 1) // bs - c // bs + 1 for c, n in zip(ctx, q))
        return {"bytes": t * D * (2 * (hq + 2 * hkv) + 2 * hq + 2 * hkv)
                + t * (8 + 4 * case["rot"]) + blocks * hkv * 16,
                "flops": t * D * (4 * (hq + hkv) + 4 * hkv)}
    blocks = sum(-(-c // bs) for c in ctx)
    pairs = sum(n * c - n * (n - 1) // 2 for c, n in zip(ctx, q) if c)
    return {"bytes": 2 * sum(ctx) * hkv * D + blocks * (8 * hkv + 4) + 4 * t * hq * D + 8 * b,
            "flops": 4 * D * hq * pairs}
