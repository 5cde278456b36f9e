"""The 8-bit paged KV cache's operators against plain 64-bit forms: step tables, append,
attention.  Every test runs on the CPU restatements and (``-m gpu``) on the kernels."""
import math

import pytest
import torch

from lightbulb_b200 import ops

D = 128
E4M3 = torch.float8_e4m3fn
DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]
on_devices = pytest.mark.parametrize("dev", DEVICES)


def _sync(dev):
    if dev == "cuda":
        torch.cuda.synchronize()
        ops.check_errors()


def _i32(v, dev="cpu"):
    return torch.tensor(v, dtype=torch.int32, device=dev)


# --------------------------------------------------------------------------------------
# step tables
# --------------------------------------------------------------------------------------
def _tables_ref(ctx, q, rows, seq_tables, new, t, bs, group, rpt, nd):
    """Python integers, straight from the definition."""
    w = len(seq_tables[0])
    tab, pos, slot, cu, last, tiles, used = [], [], [], [0], [], [], 0
    for b, (c, n) in enumerate(zip(ctx, q)):
        row = seq_tables[rows[b]]
        for j in range(-(-c // bs), -(-(c + n) // bs)):
            row[j] = new[used]
            used += 1
        need = -(-(c + n) // bs)
        tab.append(row[:need] + [0] * (w - need))
        for p in range(c, c + n):
            pos.append(p)
            slot.append(row[p // bs] * bs + p % bs)
        cu.append(cu[-1] + n)
        last.append(cu[-1] - 1 if n else -1)
        if b >= nd:
            tiles += [(b, r) for r in range(0, n * group, rpt)]
    pos += [0] * (t - len(pos))
    slot += [-1] * (t - len(slot))
    cap = t * group // rpt + len(ctx)
    tiles += [(-1, 0)] * (cap - len(tiles))
    return dict(block_tables=tab, seq_lens=[c + n for c, n in zip(ctx, q)], cu_q=cu,
                positions=pos, slots=slot, last_rows=last, tile_seq=[a for a, _ in tiles],
                tile_row0=[r for _, r in tiles], num_new=[used])


TABLE_CASES = [
    # ctx, q, block size, group, rows per tile, decode requests, padded rows
    ([0], [1], 16, 4, 256, 0, 0),
    ([0, 0], [0, 0], 16, 4, 256, 0, 0),
    ([15, 16, 17, 31, 32, 0], [1, 1, 1, 1, 1, 0], 16, 4, 256, 6, 2),
    ([5, 0, 16, 100], [40, 0, 16, 1], 16, 3, 64, 1, 7),
    ([63, 64, 1], [1, 65, 200], 64, 7, 256, 0, 0),
    ([7, 0, 3], [9, 130, 0], 32, 16, 256, 0, 1),
]


@on_devices
@pytest.mark.parametrize("case", range(len(TABLE_CASES)))
@pytest.mark.parametrize("use_rows", [False, True])
def test_step_tables(dev, case, use_rows):
    ctx, q, bs, group, rpt, nd, pad = TABLE_CASES[case]
    b, w = len(ctx), max(c + n for c, n in zip(ctx, q)) // bs + 3
    s = b + 4
    gen = torch.Generator().manual_seed(case)
    ids = torch.randperm(s * w + 64, generator=gen).tolist()
    tab = [ids[i * w:(i + 1) * w] for i in range(s)]
    new = ids[s * w:]
    rows = torch.randperm(s, generator=gen)[:b].tolist() if use_rows else list(range(b))
    t = sum(q) + pad
    seq = _i32(tab, dev)
    got = ops.step_tables(_i32(ctx, dev), _i32(q, dev), _i32(rows, dev) if use_rows else None,
                          seq, _i32(new, dev), t, bs, group=group, rows_per_tile=rpt,
                          num_decode=nd)
    _sync(dev)
    ref = _tables_ref(ctx, q, rows, tab, new, t, bs, group, rpt, nd)
    for name, want in ref.items():
        assert getattr(got, name).tolist() == want, name
    assert seq.tolist() == tab            # the resident tables got the new blocks, nothing else


@on_devices
@pytest.mark.parametrize("b,chunk", [(300, 1), (1000, 1), (37, 500), (257, 3)])
def test_step_tables_many(dev, b, chunk):
    gen = torch.Generator().manual_seed(b)
    ctx = torch.randint(0, 500, (b,), generator=gen).tolist()
    q = torch.randint(0, chunk + 1, (b,), generator=gen).tolist()
    w = 1000 // 16 + 2
    ids = torch.randperm(2 * b * w, generator=gen)
    tab, new = ids[:b * w].view(b, w).tolist(), ids[b * w:].tolist()
    seq = _i32(tab, dev)
    got = ops.step_tables(_i32(ctx, dev), _i32(q, dev), None, seq, _i32(new, dev), sum(q), 16,
                          group=4)
    _sync(dev)
    for name, want in _tables_ref(ctx, q, range(b), tab, new, sum(q), 16, 4, 256, 0).items():
        assert getattr(got, name).tolist() == want, name


def _tables_call(dev, ctx, q, rows=None, new=(7, 8, 9), t=4, w=4, s=3, **kw):
    seq = torch.arange(s * w, dtype=torch.int32, device=dev).view(s, w)
    return ops.step_tables(_i32(ctx, dev), _i32(q, dev),
                           None if rows is None else _i32(rows, dev), seq, _i32(list(new), dev),
                           t, 16, **kw)


@on_devices
def test_step_tables_refuses(dev):
    for kw in (dict(group=0), dict(rows_per_tile=0)):
        with pytest.raises(ValueError):
            _tables_call(dev, [1], [1], **kw)
    with pytest.raises(ValueError):
        _tables_call(dev, [], [])
    seq = torch.zeros(2, 4, dtype=torch.int32, device=dev)
    with pytest.raises(ValueError):
        ops.step_tables(_i32([1], dev), _i32([1], dev), None, seq, _i32([1], dev), 1, 12)


# negative length, beyond the table's width, row outside the table, too few blocks, too few rows
BAD_TABLES = [dict(ctx=[-1], q=[1]), dict(ctx=[3], q=[-2]), dict(ctx=[60], q=[5]),
              dict(ctx=[1], q=[1], rows=[3]), dict(ctx=[0], q=[40], new=(5,), t=40),
              dict(ctx=[0, 1], q=[3, 2])]


@pytest.mark.parametrize("bad", range(len(BAD_TABLES)))
def test_step_tables_bad_lengths_cpu(bad):
    with pytest.raises(ValueError):
        _tables_call("cpu", **BAD_TABLES[bad])


@pytest.mark.gpu
@pytest.mark.parametrize("bad", range(len(BAD_TABLES)))
def test_step_tables_bad_lengths_are_reported(bad):
    got = _tables_call("cuda", **BAD_TABLES[bad])
    torch.cuda.synchronize()
    with pytest.raises(ops.KernelError):
        ops.check_errors()
    assert int(got.slots.max()) < 16 * 12
    ops.check_errors()                    # reported once


# --------------------------------------------------------------------------------------
# append
# --------------------------------------------------------------------------------------
def _scale_ref(amax):
    """Smallest power of two s with amax <= 448 s, in [2^-40, 2^119] (Python floats)."""
    if amax == 0:
        return 2.0 ** -40
    k = math.frexp(amax / 448.0)
    e = k[1] - 1 if k[0] == 0.5 else k[1]
    return 2.0 ** min(119, max(-40, e))


def _append_ref(qkv, pos, slots, cs, kc, vc, ks, vs, hq, hkv, qn, kn, nd, eps):
    """64-bit append.  Returns rotated q, then per cache (values, scales, error bound)."""
    t, bs, rot = qkv.shape[0], kc.shape[2], cs.shape[1]
    x = qkv.double().view(t, -1, D)
    half = rot // 2
    c, s = cs.double()[pos.long()][:, None].split(half, -1)

    def turn(y, w):
        if w is not None:
            y = y / torch.sqrt((y * y).sum(-1, keepdim=True) / nd + eps) * w.double()
        a, b = y[..., :half], y[..., half:rot]
        return torch.cat([a * c - b * s, b * c + a * s, y[..., rot:]], -1)

    q = turn(x[:, :hq], qn)
    res = []
    for y, code, sc in ((turn(x[:, hq:hq + hkv], kn), kc, ks), (x[:, hq + hkv:], vc, vs)):
        val = code.double() * sc.double()[..., None, None]
        sc = sc.double().clone()
        tol = torch.zeros_like(val)
        byblk = {}
        for i, sl in enumerate(slots.tolist()):
            if sl >= 0:
                byblk.setdefault(sl // bs, []).append((sl % bs, i))
        for blk, toks in byblk.items():
            for h in range(hkv):
                rows = y[[i for _, i in toks], h]
                new = _scale_ref(float(rows.abs().max()))
                if toks[0][0] > 0:
                    old = float(sc[blk, h])
                    new = max(new, old)
                    if new > old:      # older codes lose what falls below the new smallest step
                        tol[blk, h, :toks[0][0]] = 2.0 ** -10 * new
                sc[blk, h] = new
                # behind the first new token nothing counts as stored: codes stay as they are
                val[blk, h, toks[0][0]:] = code[blk, h, toks[0][0]:].double() * new
                for o, i in toks:
                    val[blk, h, o] = y[i, h]
                    # half a step of e4m3 (3 stored mantissa bits; 2^-9 steps below 2^-6),
                    # plus the fp32 arithmetic before it
                    tol[blk, h, o] = torch.maximum(y[i, h].abs() * 2.0 ** -4,
                                                   torch.tensor(2.0 ** -10 * new)) \
                        + y[i, h].abs().max() * 2.0 ** -18
        res.append((val, sc, tol))
    return q, res


def _random_cache(gen, nb, hkv, bs):
    codes = (torch.randn(nb, hkv, bs, D, generator=gen) * 60).clamp(-448, 448).to(E4M3)
    scale = 2.0 ** torch.randint(-12, -4, (nb, hkv), generator=gen).float()
    return codes, scale


def _check_append(dev, seqs, hq, hkv, bs, rot, norm, seed=0, holes=(), pad_cols=0, spread=1.0,
                  qkv_edit=None, mags=None):
    """``seqs``: (first position, tokens) per sequence; every block that is touched is its own."""
    gen = torch.Generator().manual_seed(seed)
    t = sum(n for _, n in seqs)
    nblk = sum((c + n - 1) // bs - c // bs + 1 for c, n in seqs if n) + 2
    order = torch.randperm(nblk, generator=gen).tolist()
    pos, slots, used = [], [], 0
    for c, n in seqs:
        for p in range(c, c + n):
            slots.append(order[used + p // bs - c // bs] * bs + p % bs)
            pos.append(p)
        used += ((c + n - 1) // bs - c // bs + 1) if n else 0
    for h in holes:
        slots[h] = -1
    heads = hq + 2 * hkv
    x = torch.randn(t, heads, D, generator=gen) * torch.exp(
        spread * torch.randn(t, heads, 1, generator=gen))
    if mags is not None:
        x = x * torch.tensor(mags).view(t, 1, 1)
    x[..., rot:] = 0
    if qkv_edit is not None:
        qkv_edit(x)
    qkv = torch.zeros(t, heads * D + pad_cols).bfloat16()
    qkv[:, :heads * D] = x.bfloat16().view(t, -1)
    kc, ks = _random_cache(gen, nblk, hkv, bs)
    vc, vs = _random_cache(gen, nblk, hkv, bs)
    cs = ops.rope_table(4096, rot, 1e4, "cpu")
    qn = kn = None
    if norm:
        qn, kn = ((1 + 0.3 * torch.randn(D, generator=gen)).bfloat16() for _ in range(2))
    pos_t, slot_t = _i32(pos), _i32(slots)
    mv = lambda z: None if z is None else z.clone().to(dev)       # noqa: E731
    got = [mv(z) for z in (kc, vc, ks, vs)]
    q_in = mv(qkv)
    q = ops.rope_kv_fp8(q_in, mv(pos_t), mv(slot_t), mv(cs), *got, hq, hkv, q_norm=mv(qn),
                        k_norm=mv(kn), norm_dim=rot, eps=1e-6)
    _sync(dev)
    assert torch.equal(q_in.cpu(), qkv)
    qr, res = _append_ref(qkv[:, :heads * D], pos_t, slot_t, cs, kc, vc, ks, vs, hq, hkv, qn, kn,
                          rot, 1e-6)
    # bf16 has 8 significant bits: half a step is at most 2^-8 of the value; fp32 arithmetic
    # before it adds a few 2^-24 of the head's largest element
    big = qr.abs().amax(-1, keepdim=True)
    assert bool(((q.cpu().double() - qr).abs() <= 2.0 ** -8 * qr.abs() + 2.0 ** -18 * big).all())
    for (val, sc, tol), code, scale in zip(res, got[0:2], got[2:4]):
        assert torch.equal(scale.cpu().double(), sc)
        have = code.cpu().double() * sc[..., None, None]
        # what the call did not touch is untouched, what it wrote is within half a step
        assert bool(((have - val).abs() <= tol).all())
    return q, got


@on_devices
@pytest.mark.parametrize("bs", [16, 32, 64])
@pytest.mark.parametrize("rot,norm", [(128, False), (128, True), (96, False), (64, True),
                                      (16, False)])
def test_append_chunks(dev, bs, rot, norm):
    # one token, a block's last and first, runs over several blocks, odd ends
    _check_append(dev, [(0, 1), (bs - 1, 1), (bs, 1), (5, 3 * bs + 7), (0, 2 * bs), (bs - 3, 4)],
                  4, 2, bs, rot, norm, seed=bs + rot)


@on_devices
@pytest.mark.parametrize("hq,hkv", [(1, 1), (3, 1), (32, 8), (5, 5), (64, 4)])
def test_append_heads_and_row_stride(dev, hq, hkv):
    _check_append(dev, [(3, 20), (17, 1)], hq, hkv, 16, 128, False, seed=hq, pad_cols=8)


@on_devices
@pytest.mark.parametrize("holes", [(0,), (4,), (3, 4, 5, 6), tuple(range(10, 20)), (29,)])
def test_append_rows_without_slot(dev, holes):
    _check_append(dev, [(2, 30)], 2, 2, 16, 128, False, seed=9, holes=holes)


@on_devices
@pytest.mark.parametrize("bs", [16, 64])
def test_append_growing_and_shrinking_magnitudes(dev, bs):
    # magnitudes over 2^-30 .. 2^30: scales that grow a lot rescale what was there
    mags = [2.0 ** ((7 * i) % 61 - 30) for i in range(40)]
    _check_append(dev, [(bs - 1, 1), (9, 1), (11, 3), (1, 35)], 2, 2, bs, 128, False, seed=4,
                  mags=mags)


@on_devices
def test_append_zeros_then_values(dev):
    def edit(x):
        x[:5] = 0
    _check_append(dev, [(0, 4), (3, 2), (0, 1)], 2, 1, 16, 128, False, seed=5, qkv_edit=edit)


@on_devices
def test_append_one_token_at_a_time_matches_the_values(dev):
    """Tokens appended one per call: every stored value stays within half a step of its own
    scale plus one step of rounding per growth below the normal numbers."""
    gen = torch.Generator().manual_seed(3)
    hkv, bs, n = 2, 16, 16
    x = torch.randn(n, 3 * hkv, D, generator=gen) * (1.5 ** torch.arange(n).view(n, 1, 1))
    qkv = x.bfloat16().view(n, -1).to(dev)
    kc = torch.zeros(1, hkv, bs, D, dtype=E4M3, device=dev)
    vc, ks, vs = kc.clone(), torch.ones(1, hkv, device=dev), torch.ones(1, hkv, device=dev)
    cs = ops.rope_table(64, 128, 1e4, dev)
    for i in range(n):
        ops.rope_kv_fp8(qkv[i:i + 1], _i32([i], dev), _i32([i], dev), cs, kc, vc, ks, vs, hkv, hkv)
    _sync(dev)
    v = qkv.view(n, 3 * hkv, D)[:, 2 * hkv:].double().cpu().transpose(0, 1)
    got = vc[0].cpu().double() * vs[0].cpu().double()[:, None, None]
    tol = torch.maximum(v.abs() * 2.0 ** -4, 2.0 ** -9 * vs[0].cpu().double()[:, None, None])
    assert bool(((got - v).abs() <= tol).all())
    amax = v.abs().amax((1, 2))
    assert vs[0].tolist() == [_scale_ref(float(a)) for a in amax]


@on_devices
def test_append_infinities_and_nan(dev):
    hkv, bs = 1, 16
    qkv = torch.randn(3, 3 * D, generator=torch.Generator().manual_seed(1)).bfloat16()
    qkv[0, 2 * D + 3] = math.inf
    qkv[0, 2 * D + 4] = -math.inf
    qkv[1, 2 * D + 5] = math.nan
    kc = torch.zeros(2, hkv, bs, D, dtype=E4M3, device=dev)
    vc, ks, vs = kc.clone(), torch.ones(2, hkv, device=dev), torch.ones(2, hkv, device=dev)
    ops.rope_kv_fp8(qkv.to(dev), _i32([0, 1, 2], dev), _i32([0, bs, bs + 1], dev),
                    ops.rope_table(8, 128, 1e4, dev), kc, vc, ks, vs, 1, 1)
    _sync(dev)
    v, s = vc.cpu().float(), vs.cpu()
    assert v[0, 0, 0, 3] == 448 and v[0, 0, 0, 4] == -448 and s[0, 0] == 2.0 ** 119
    assert torch.isnan(v[1, 0, 0, 5]) and int(torch.isnan(v).sum()) == 1
    # the NaN does not count for the scale
    top = float(qkv[1:, 2 * D:].float().abs().nan_to_num(0).max())
    assert float(s[1, 0]) == _scale_ref(top)


@pytest.mark.gpu
def test_append_reports_bad_indexes():
    def call(pos, slot):
        kc = torch.zeros(2, 1, 16, D, dtype=E4M3, device="cuda")
        vc, ks = kc.clone(), torch.ones(2, 1, device="cuda")
        ops.rope_kv_fp8(torch.ones(1, 3 * D, device="cuda").bfloat16(), _i32([pos], "cuda"),
                        _i32([slot], "cuda"), ops.rope_table(8, 128, 1e4, "cuda"), kc, vc, ks,
                        ks.clone(), 1, 1)
        torch.cuda.synchronize()
        with pytest.raises(ops.KernelError):
            ops.check_errors()
        return kc
    assert not call(0, 2 * 16).float().any()      # a slot past the pool stores nothing
    call(8, 0)
    call(-1, 0)


@pytest.mark.gpu
def test_append_empty_and_other_stream():
    kc = torch.zeros(2, 1, 16, D, dtype=E4M3, device="cuda")
    vc, ks, vs = kc.clone(), torch.ones(2, 1, device="cuda"), torch.ones(2, 1, device="cuda")
    cs = ops.rope_table(8, 128, 1e4, "cuda")
    e = torch.empty(0, dtype=torch.int32, device="cuda")
    q = ops.rope_kv_fp8(torch.empty(0, 3 * D, device="cuda").bfloat16(), e, e, cs, kc, vc, ks, vs,
                        1, 1)
    assert q.shape == (0, 1, D)
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        torch.cuda._sleep(2_000_000)
        x = torch.ones(1, 3 * D, device="cuda").bfloat16()
        q = ops.rope_kv_fp8(x, _i32([0], "cuda"), _i32([3], "cuda"), cs, kc, vc, ks, vs, 1, 1)
    st.synchronize()
    assert bool((q == 1).all()) and bool((vc[0, 0, 3].float() * vs[0, 0] == 1).all())


@pytest.mark.gpu
def test_append_past_2_31_bytes():
    hkv, bs = 8, 16
    nb = 2 ** 31 // (hkv * bs * D) + 64
    kc = torch.zeros(nb, hkv, bs, D, dtype=E4M3, device="cuda")
    vc, ks = torch.zeros_like(kc), torch.ones(nb, hkv, device="cuda")
    vs = ks.clone()
    qkv = torch.randn(5, 3 * hkv * D, device="cuda").bfloat16()
    slots = torch.arange(5, dtype=torch.int32, device="cuda") + (nb - 1) * bs
    ops.rope_kv_fp8(qkv, _i32([0, 1, 2, 3, 4], "cuda"), slots, ops.rope_table(8, 128, 1e4, "cuda"),
                    kc, vc, ks, vs, hkv, hkv)
    out = torch.empty(1, hkv, D, dtype=torch.bfloat16, device="cuda")
    ops.paged_attention_fp8(qkv.view(5, -1, D)[4:, :hkv], kc, vc, ks, vs, _i32([[nb - 1]], "cuda"),
                            _i32([5], "cuda"), None, out, 1, True)
    _sync("cuda")
    v = qkv.view(5, 3 * hkv, D)[:, 2 * hkv:].float()
    got = vc[nb - 1, :, :5].float().transpose(0, 1) * vs[nb - 1][None, :, None]
    tol = v.abs() * 2.0 ** -4 + 2.0 ** -10 * vs[nb - 1][None, :, None]
    assert bool(((got - v).abs() <= tol).all())
    ref, bound = _attention_ref(qkv.view(5, -1, D)[4:, :hkv].cpu(), kc[nb - 1:].cpu(),
                                vc[nb - 1:].cpu(), ks[nb - 1:].cpu(), vs[nb - 1:].cpu(), [[0]],
                                [5], [1], 1, True, None)
    assert bool(((out.cpu().double() - ref).abs() <= bound).all())


# --------------------------------------------------------------------------------------
# attention
# --------------------------------------------------------------------------------------
def _attention_ref(q, kc, vc, ks, vs, tables, lens, n_q, group, causal, scale):
    """64-bit attention and what the kernel's roundings may change: bf16 output (2^-8 of the
    value); weights of 11 bits (2^-11 of sum p |v|); scores summed in fp32 (128 products whose
    magnitudes add up to less than about 2^7: less than 2^-10 of sum p |v|)."""
    scale = D ** -0.5 if scale is None else scale
    bs = kc.shape[2]
    out = torch.zeros(q.shape, dtype=torch.float64)
    tol = torch.zeros_like(out)
    t0 = 0
    for i, (n, m) in enumerate(zip(lens, n_q)):
        ids = torch.tensor(tables[i][:-(-n // bs)], dtype=torch.long)
        for h in range(q.shape[1] if n else 0):
            kv = h // group
            k, v = ((c[ids, kv].double() * s[ids, kv].double()[:, None, None]).reshape(-1, D)[:n]
                    for c, s in ((kc, ks), (vc, vs)))
            s = q[t0:t0 + m, h].double() @ k.T * scale
            if causal:
                s = s.masked_fill(torch.arange(n) > torch.arange(n - m, n)[:, None], -math.inf)
            seen = (s > -math.inf).any(-1)
            p = torch.softmax(s[seen], -1)
            rows = t0 + seen.nonzero()[:, 0]
            out[rows, h] = p @ v
            tol[rows, h] = 2.0 ** -8 * (p @ v).abs() + 2.0 ** -9 * (p @ v.abs()) + 1e-30
        t0 += m
    return out, tol


def _paged_inputs(lens, hkv, bs, seed, any_scale=False, width=None):
    """Caches whose blocks are scattered; what lies past a sequence's end is NaN."""
    gen = torch.Generator().manual_seed(seed)
    counts = [-(-n // bs) for n in lens]
    nb = sum(counts) + 3
    order = torch.randperm(nb, generator=gen).tolist()
    width = width or max(1, max(counts)) + 1
    tables, o = [], 0
    for c in counts:
        tables.append(order[o:o + c] + [order[-1]] * (width - c))
        o += c
    kc, vc = ((torch.randn(nb, hkv, bs, D, generator=gen) * 100).clamp(-448, 448).to(E4M3)
              for _ in range(2))
    ks = 2.0 ** torch.randint(-8, -5, (nb, hkv), generator=gen).float()
    vs = 2.0 ** torch.randint(-10, 3, (nb, hkv), generator=gen).float()
    if any_scale:
        ks = torch.rand(nb, hkv, generator=gen) * 0.02 + 1e-3
        vs = torch.rand(nb, hkv, generator=gen) * 7 + 1e-4
    live = torch.zeros(nb, bs, dtype=torch.bool)
    for i, n in enumerate(lens):
        for j, blk in enumerate(tables[i][:counts[i]]):
            live[blk, :n - j * bs] = True
    for c in (kc, vc):
        c.view(torch.uint8).masked_fill_(~live[:, None, :, None], 0x7F)
    for s in (ks, vs):
        s.masked_fill_(~live.any(1)[:, None], math.nan)
    return kc, vc, ks, vs, tables


def _check_attention(dev, lens, n_q, hq, hkv, bs, decode, seed=0, causal=True, scale=None,
                     any_scale=False, q_mag=1.0, inputs=None, pad_tiles=0):
    kc, vc, ks, vs, tables = inputs or _paged_inputs(lens, hkv, bs, seed, any_scale)
    gen = torch.Generator().manual_seed(seed + 1)
    t = sum(n_q)
    row = torch.randn(t, (hq + 2 * hkv) * D, generator=gen) * q_mag
    q = row.bfloat16()[:, :hq * D].view(t, hq, D)                # strided rows
    group = hq // hkv
    cu = [0]
    for m in n_q:
        cu.append(cu[-1] + m)
    tiles = [(i, r) for i, m in enumerate(n_q) for r in range(0, m * group, 256)]
    tiles += [(-1, 0)] * pad_tiles
    mv = lambda z: z.to(dev)                                      # noqa: E731
    obuf = torch.full((t, hq * D + 64), 7.0, dtype=torch.bfloat16, device=dev)
    out = obuf[:, :hq * D].view(t, hq, D)
    args = [mv(z) for z in (kc, vc, ks, vs)]
    qd = row.bfloat16().to(dev)[:, :hq * D].view(t, hq, D)
    for again in range(2):
        ops.paged_attention_fp8(qd, *args, _i32(tables, dev), _i32(lens, dev), _i32(cu, dev), out,
                                group, decode, tile_seq=_i32([a for a, _ in tiles], dev),
                                tile_row0=_i32([r for _, r in tiles], dev), causal=causal,
                                scale=scale)
        _sync(dev)
        if again:
            assert torch.equal(first, out.cpu())                  # the same bits every time
        first = out.cpu().clone()
    assert bool((obuf[:, hq * D:] == 7).all())
    ref, tol = _attention_ref(q, kc, vc, ks, vs, tables, lens, n_q, group, causal and not decode,
                              scale)
    err = (first.double() - ref).abs()
    assert bool((err <= tol).all()), float((err - tol).max())
    return first


@on_devices
@pytest.mark.parametrize("bs", [16, 32, 64])
@pytest.mark.parametrize("lens", [[1], [0, 1, 2], [15, 16, 17], [31, 32, 33, 63, 64, 65],
                                  [127, 0, 128, 129, 300, 5], [1000, 3, 0]])
def test_decode_lengths(dev, bs, lens):
    _check_attention(dev, lens, [1] * len(lens), 8, 2, bs, True, seed=bs + len(lens))


@on_devices
@pytest.mark.parametrize("hq,hkv", [(1, 1), (2, 2), (3, 1), (10, 2), (7, 1), (8, 1), (9, 1),
                                    (16, 1), (32, 2), (17, 1), (40, 1), (24, 8)])
def test_decode_groups(dev, hq, hkv):
    _check_attention(dev, [70, 1, 500, 0, 33], [1] * 5, hq, hkv, 16, True, seed=hq * 10 + hkv)


@on_devices
@pytest.mark.parametrize("any_scale", [False, True])
@pytest.mark.parametrize("scale", [None, 0.02, 1.0])
def test_decode_scales(dev, any_scale, scale):
    _check_attention(dev, [900, 17, 350], [1] * 3, 8, 2, 16, True, seed=5, any_scale=any_scale,
                     scale=scale, q_mag=0.3 if scale == 1.0 else 1.0)


@pytest.mark.gpu
@pytest.mark.parametrize("lens,hq,hkv,bs", [([20001], 8, 2, 16), ([9000, 1, 30000, 77], 4, 1, 64),
                                            ([2047] * 40, 8, 8, 16),
                                            (list(range(0, 1200, 3)), 2, 1, 32)])
def test_decode_long_and_many(lens, hq, hkv, bs):
    _check_attention("cuda", lens, [1] * len(lens), hq, hkv, bs, True, seed=len(lens))


@on_devices
@pytest.mark.parametrize("bs", [16, 32, 64])
@pytest.mark.parametrize("lens,n_q", [([1], [1]), ([40], [40]), ([300, 70], [5, 70]),
                                      ([129, 0, 128], [1, 0, 128]), ([513], [200]),
                                      ([64, 65, 500], [64, 65, 67])])
def test_prefill_lengths(dev, bs, lens, n_q):
    _check_attention(dev, lens, n_q, 8, 2, bs, False, seed=sum(lens) + bs, pad_tiles=3)


@on_devices
@pytest.mark.parametrize("hq,hkv", [(1, 1), (3, 1), (10, 2), (7, 1), (16, 1), (20, 1), (4, 4)])
def test_prefill_groups(dev, hq, hkv):
    _check_attention(dev, [200, 90], [60, 33], hq, hkv, 16, False, seed=hq)


@on_devices
def test_prefill_rows_that_see_nothing(dev):
    # more query tokens than keys: the first ones see no key and give 0
    out = _check_attention(dev, [3, 0, 20], [10, 4, 5], 4, 1, 16, False, seed=2)
    assert not out[:7].any() and not out[10:14].any()


@on_devices
@pytest.mark.parametrize("any_scale", [False, True])
def test_prefill_not_causal_and_scales(dev, any_scale):
    _check_attention(dev, [300, 40], [70, 90], 4, 2, 32, False, seed=8, causal=False,
                     any_scale=any_scale, scale=0.05)


@pytest.mark.gpu
@pytest.mark.parametrize("lens,n_q,hq,hkv,bs", [([5000], [300], 4, 1, 16),
                                                ([2100, 130, 700], [515, 129, 600], 8, 2, 64)])
def test_prefill_long(lens, n_q, hq, hkv, bs):
    _check_attention("cuda", lens, n_q, hq, hkv, bs, False, seed=len(lens))


@on_devices
@pytest.mark.parametrize("decode", [True, False])
def test_attention_extreme_magnitudes(dev, decode):
    """One key far ahead of all others, blocks of zeros, values over twelve orders."""
    lens = [400, 90]
    kc, vc, ks, vs, tables = _paged_inputs(lens, 2, 16, 3)
    ids = tables[0][:25]
    vs[ids[3]], vs[ids[7]], vs[ids[20]] = 2.0 ** -40, 2.0 ** 10, 2.0 ** -20
    vc.view(torch.uint8)[ids[5]] = 0
    ks[ids[9]] *= 8
    _check_attention(dev, lens, [1, 1] if decode else [30, 9], 8, 2, 16, decode, seed=3,
                     inputs=(kc, vc, ks, vs, tables), q_mag=0.5)


@pytest.mark.gpu
@pytest.mark.parametrize("decode", [True, False])
def test_attention_reports_bad_blocks(decode):
    kc, vc, ks, vs, tables = _paged_inputs([100], 1, 16, 1)
    for bad in (kc.shape[0], -1):
        tables[0][2] = bad
        q = torch.randn(1, 2, D, device="cuda").bfloat16()
        out = torch.empty_like(q)
        kc2, vc2 = (torch.nan_to_num(c.float()).to(E4M3).cuda() for c in (kc, vc))
        ks2, vs2 = (torch.nan_to_num(s, nan=1.0).cuda() for s in (ks, vs))
        ops.paged_attention_fp8(q, kc2, vc2, ks2, vs2, _i32(tables, "cuda"), _i32([100], "cuda"),
                                _i32([0, 1], "cuda"), out, 2, decode, tile_seq=_i32([0], "cuda"),
                                tile_row0=_i32([0], "cuda"))
        torch.cuda.synchronize()
        with pytest.raises(ops.KernelError):
            ops.check_errors()
        assert bool(torch.isfinite(out.float()).all())


@pytest.mark.gpu
@pytest.mark.parametrize("cu", [[0, 300], [-1, 3], [2, 1]])
@pytest.mark.parametrize("pad_tiles", [0, 20])        # both kernels: 9 or 189 rows per item
def test_prefill_reports_offsets_outside_q(cu, pad_tiles):
    kc, vc, ks, vs, tables = _paged_inputs([100], 1, 16, 1)
    q = torch.randn(3, 63, D, device="cuda").bfloat16()
    out = torch.full_like(q, 3.0)
    tiles = [0] + [-1] * pad_tiles
    ops.paged_attention_fp8(q, *(z.cuda() for z in (kc, vc, ks, vs)), _i32(tables, "cuda"),
                            _i32([100], "cuda"), _i32(cu, "cuda"), out, 63, False,
                            tile_seq=_i32(tiles, "cuda"), tile_row0=_i32([0] * len(tiles), "cuda"))
    torch.cuda.synchronize()
    with pytest.raises(ops.KernelError):
        ops.check_errors()
    assert bool((out == 3).all())


@pytest.mark.gpu
@pytest.mark.parametrize("decode", [True, False])
def test_attention_other_stream_and_graph(decode):
    kc, vc, ks, vs, tables = _paged_inputs([3000, 40], 2, 16, 1)
    args = [z.cuda() for z in (kc, vc, ks, vs)]
    tab, lens, cu = _i32(tables, "cuda"), _i32([3000, 40], "cuda"), _i32([0, 1, 2], "cuda")
    ts, tr = _i32([0, 1], "cuda"), _i32([0, 0], "cuda")
    q = torch.randn(2, 8, D, device="cuda").bfloat16()
    want, out = torch.empty_like(q), torch.zeros_like(q)

    def call(o):
        ops.paged_attention_fp8(q, *args, tab, lens, cu, o, 4, decode, tile_seq=ts, tile_row0=tr)
    call(want)
    torch.cuda.synchronize()
    st = torch.cuda.Stream()
    with torch.cuda.stream(st):
        torch.cuda._sleep(2_000_000)
        call(out)
    st.synchronize()
    assert torch.equal(out, want)
    g = torch.cuda.CUDAGraph()
    out.zero_()
    with torch.cuda.graph(g):
        call(out)
    for _ in range(3):
        out.zero_()
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want)
    ops.check_errors()


@pytest.mark.gpu
@pytest.mark.parametrize("lens,n_q,bs", [([320], [200], 16), ([513, 40], [200, 40], 32),
                                         ([1025, 1, 640], [1, 1, 1], 64), ([900] * 30, [3] * 30, 16)])
def test_attention_same_bits_cold_and_warm(lens, n_q, bs):
    """The pipelines' timing changes with what is in L2; the results do not."""
    hq, hkv = 8, 2
    kc, vc, ks, vs, tables = _paged_inputs(lens, hkv, bs, 7)
    args = [z.cuda() for z in (kc, vc, ks, vs)]
    t, decode = sum(n_q), max(n_q) == 1
    q = torch.randn(t, hq, D, generator=torch.Generator().manual_seed(1)).bfloat16().cuda()
    cu = [0]
    for m in n_q:
        cu.append(cu[-1] + m)
    tiles = [(i, r) for i, m in enumerate(n_q) for r in range(0, m * 4, 256)]
    idx = [_i32(v, "cuda") for v in (tables, lens, cu)]
    ts, tr = _i32([a for a, _ in tiles], "cuda"), _i32([r for _, r in tiles], "cuda")
    flush = torch.empty(48 << 20, dtype=torch.int32, device="cuda")
    first = None
    for i in range(40):
        if i % 2:
            flush.fill_(i)
        out = torch.zeros_like(q)
        torch.cuda.synchronize()
        ops.paged_attention_fp8(q, *args, *idx, out, 4, decode, tile_seq=ts, tile_row0=tr)
        torch.cuda.synchronize()
        if first is None:
            first = out.clone()
            ref, tol = _attention_ref(q.cpu(), kc, vc, ks, vs, tables, lens, n_q, 4, not decode,
                                      None)
            assert bool(((out.cpu().double() - ref).abs() <= tol).all())
        assert torch.equal(out, first), i
    ops.check_errors()


# --------------------------------------------------------------------------------------
# refusals
# --------------------------------------------------------------------------------------
def _good():
    kc = torch.zeros(4, 2, 16, D, dtype=E4M3, device="cuda")
    s = torch.ones(4, 2, device="cuda")
    return dict(q=torch.zeros(1, 4, D, device="cuda").bfloat16(), k_cache=kc, v_cache=kc.clone(),
                k_scale=s, v_scale=s.clone(), block_tables=_i32([[0]], "cuda"),
                seq_lens=_i32([1], "cuda"), cu_q=_i32([0, 1], "cuda"),
                out=torch.zeros(1, 4, D, device="cuda").bfloat16(), group=2, decode=True)


REFUSED = [lambda a: a.update(k_cache=a["k_cache"].bfloat16()),
           lambda a: a.update(k_cache=a["k_cache"][:, :, :8].contiguous(),
                              v_cache=a["v_cache"][:, :, :8].contiguous()),
           lambda a: a.update(k_cache=a["k_cache"].transpose(1, 2)),
           lambda a: a.update(v_cache=a["v_cache"][:3]),
           lambda a: a.update(k_scale=a["k_scale"].half()),
           lambda a: a.update(v_scale=a["v_scale"][:, :1]),
           lambda a: a.update(q=a["q"].float()),
           lambda a: a.update(q=a["q"][..., :64], out=a["out"][..., :64]),
           lambda a: a.update(group=4),
           lambda a: a.update(out=a["out"][:, :2]),
           lambda a: a.update(block_tables=a["block_tables"].long()),
           lambda a: a.update(seq_lens=a["seq_lens"].long()),
           lambda a: a.update(decode=False)]


@pytest.mark.gpu
@pytest.mark.parametrize("i", range(len(REFUSED)))
def test_attention_refuses(i):
    a = _good()
    ops.paged_attention_fp8(**a)
    REFUSED[i](a)
    with pytest.raises(RuntimeError):
        ops.paged_attention_fp8(**a)


@pytest.mark.gpu
def test_append_refuses():
    def call(**kw):
        kc = torch.zeros(4, 2, 16, D, dtype=E4M3, device="cuda")
        s = torch.ones(4, 2, device="cuda")
        a = dict(qkv=torch.zeros(1, 8 * D, device="cuda").bfloat16(), positions=_i32([0], "cuda"),
                 slots=_i32([0], "cuda"), cos_sin=ops.rope_table(8, 128, 1e4, "cuda"), k_cache=kc,
                 v_cache=kc.clone(), k_scale=s, v_scale=s.clone(), hq=4, hkv=2)
        a.update(kw)
        ops.rope_kv_fp8(**a)
    call()
    for kw in (dict(qkv=torch.zeros(1, 8 * D, device="cuda")),
               dict(qkv=torch.zeros(1, 7 * D, device="cuda").bfloat16()),
               dict(positions=torch.zeros(1, dtype=torch.int64, device="cuda")),
               dict(slots=torch.zeros(1, device="cuda")), dict(hkv=1),
               dict(cos_sin=ops.rope_table(8, 24, 1e4, "cuda")),
               dict(q_norm=torch.ones(64, device="cuda").bfloat16()),
               dict(k_scale=torch.ones(4, 2, device="cuda").double())):
        with pytest.raises(RuntimeError):
            call(**kw)
