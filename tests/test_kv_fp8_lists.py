"""Work lists of the attention over the 8-bit cache: which kernel they reach, and their edges on each of
them."""
import pytest
import torch

from lightbulb_b200 import ops
from test_kv_fp8 import D, _attention_ref, _i32, _paged_inputs, on_devices


@on_devices
@pytest.mark.parametrize("m", [5, 70])          # the kernel of few rows, the tcgen05 one
@pytest.mark.parametrize("row0", [2 ** 31 - 1, 2 ** 31 - 100, 2 ** 31 - 257, 1 << 30, 512])
def test_items_past_the_rows_write_nothing(dev, m, row0):
    lens, group = [300], 4
    kc, vc, ks, vs, tables = _paged_inputs(lens, 2, 16, 1)
    q = torch.randn(m, 8, D, generator=torch.Generator().manual_seed(1)).bfloat16()
    rows = list(range(0, m * group, 256))
    buf = torch.full((m + 64, 8, D), 3.0, dtype=torch.bfloat16, device=dev)
    out = buf[32:32 + m]
    n0 = ops.launch_counter_value()
    ops.paged_attention_fp8(q.to(dev), *(z.to(dev) for z in (kc, vc, ks, vs)), _i32(tables, dev),
                            _i32(lens, dev), _i32([0, m], dev), out, group, False,
                            tile_seq=_i32([0] * (len(rows) + 1), dev),
                            tile_row0=_i32(rows + [row0], dev))
    if dev == "cuda":
        torch.cuda.synchronize()
        ops.check_errors()
        assert ops.launch_counter_value() - n0 == (1 if m == 70 else 2)
    ref, tol = _attention_ref(q, kc, vc, ks, vs, tables, lens, [m], group, True, None)
    assert bool(((out.cpu().double() - ref).abs() <= tol).all())
    assert bool((buf[:32] == 3).all()) and bool((buf[32 + m:] == 3).all())


MIXED = [  # decodes, new tokens of each other request, group, kernels of the list's call
    (63, [70], 4, 1), (40, [130, 3], 1, 1), (255, [600], 4, 1), (30, [5, 4], 4, 2), (0, [40], 8, 1)]


@on_devices
@pytest.mark.parametrize("nd,chunks,group,kernels", MIXED)
def test_prompt_chunks_beside_decodes(dev, nd, chunks, group, kernels):
    """A step as the engine runs it: decodes first, their tokens in the same q, the list of
    step_tables.  The chunks' rows decide the kernel, however many decodes the step has."""
    gen = torch.Generator().manual_seed(nd + group)
    n_q = [1] * nd + chunks
    lens = [int(torch.randint(1, 90, (1,), generator=gen)) for _ in range(nd)] + \
        [n + 37 for n in chunks]
    kc, vc, ks, vs, tables = _paged_inputs(lens, 2, 16, nd)
    args = [z.to(dev) for z in (kc, vc, ks, vs)]
    t, hq, b = sum(n_q), 2 * group, len(n_q)
    st = ops.step_tables(_i32([n - m for n, m in zip(lens, n_q)], dev), _i32(n_q, dev), None,
                         _i32(tables, dev), _i32([0] * (t + b), dev), t, 16, group=group,
                         num_decode=nd)
    tab = _i32(tables, dev)             # the blocks that hold the tokens already
    q = torch.randn(t, hq, D, generator=gen).bfloat16()
    out = torch.full((t, hq, D), 7.0, dtype=torch.bfloat16, device=dev)
    qd = q.to(dev)
    if nd:
        ops.paged_attention_fp8(qd, *args, tab[:nd], st.seq_lens[:nd], None, out, group, True)
    n, most = ops.work_items(chunks, group)
    assert most == min(256, max(chunks) * group)
    assert (st.tile_seq >= 0).tolist() == [True] * n + [False] * (st.tile_seq.numel() - n)
    bits = []
    for k in (n, st.tile_seq.numel()):  # entries in use alone, and with the spare ones
        n0 = ops.launch_counter_value()
        ops.paged_attention_fp8(qd, *args, tab, st.seq_lens, st.cu_q, out, group, False,
                                tile_seq=st.tile_seq[:k], tile_row0=st.tile_row0[:k],
                                item_rows=most)
        if dev == "cuda":
            assert ops.launch_counter_value() - n0 == kernels
            torch.cuda.synchronize()
            ops.check_errors()
        bits.append(out.cpu().clone())
    assert torch.equal(*bits)
    ref, tol = _attention_ref(q, kc, vc, ks, vs, tables, lens, n_q, group, True, None)
    assert bool(((bits[0].double() - ref).abs() <= tol).all())


def test_engine_passes_the_items_in_use(monkeypatch):
    """Every list that reaches the attention has only real entries and says how long the longest
    is, also with more decodes than chunks."""
    from test_kv_fp8_engine import GREEDY, _engine
    _, _, _, eng = _engine("cpu", overlap=False)
    calls, inner = [], ops.paged_attention_fp8

    def watch(q, *a, **k):
        if not k["decode"]:
            seq, row0, cu = k["tile_seq"].tolist(), k["tile_row0"].tolist(), a[6].tolist()
            rows = [(cu[s + 1] - cu[s]) * eng.model.group for s in seq]
            assert min(seq) >= 0 and all(r < n for r, n in zip(row0, rows))
            assert k["item_rows"] == min(256, max(rows))
            calls.append((q.shape[0], sum(set(rows))))
        return inner(q, *a, **k)
    monkeypatch.setattr(ops, "paged_attention_fp8", watch)
    prompts = [[i + 1, 2, 3] for i in range(7)] + [list(range(200))]
    eng.generate(prompt_token_ids=prompts, params=GREEDY)
    assert any(t * eng.model.group > r for t, r in calls)      # steps with decodes and chunks
    with pytest.raises(ValueError):
        inner(torch.zeros(1, 1, D), *[None] * 8, 1, False, item_rows=-1)


# n_q whose longest item reaches each kernel (group 4): one, two, three column tiles of the kernel
# of few rows, and the tcgen05 one
REACH = {"8": [2, 1], "16": [4, 3], "24": [6, 5], "32": [8, 7], "tc": [70, 33]}


def _call(dev, inputs, lens, n_q, hq, hkv, q, out, cu=None):
    """The call of a list; checks which kernel it is."""
    kc, vc, ks, vs, tables = inputs
    group = hq // hkv
    rows = [m * group for m in n_q]
    tiles = [(i, r) for i, m in enumerate(rows) for r in range(0, m, 256)]
    offs = [0]
    for m in n_q:
        offs.append(offs[-1] + m)
    args = [z.to(dev) for z in (q, kc, vc, ks, vs)] + [
        _i32(tables, dev), _i32(lens, dev), _i32(cu or offs, dev), out, group, False]
    kw = dict(tile_seq=_i32([a for a, _ in tiles], dev), tile_row0=_i32([r for _, r in tiles], dev),
              item_rows=min(256, max(rows)))

    def call():
        n0 = ops.launch_counter_value()
        ops.paged_attention_fp8(*args, **kw)
        if dev == "cuda":
            assert ops.launch_counter_value() - n0 == (1 if max(rows) > 32 else 2)
    return call


@on_devices
@pytest.mark.parametrize("reach", REACH)
@pytest.mark.parametrize("bs", [16, 32, 64])
@pytest.mark.parametrize("lens", [[1, 2], [0, 40], [31, 33], [129, 700], [5, 0], [257, 128]])
def test_lengths_on_every_kernel(dev, reach, bs, lens):
    """Lengths down to none, shorter than the queries (rows that see no key, items without a tile),
    and ends inside tiles and blocks; two calls give the same bits."""
    n_q, hq, hkv = REACH[reach], 8, 2
    inputs = _paged_inputs(lens, hkv, bs, sum(lens) + bs)
    q = torch.randn(sum(n_q), hq, D, generator=torch.Generator().manual_seed(bs)).bfloat16()
    out = torch.full(q.shape, 7.0, dtype=torch.bfloat16, device=dev)
    call = _call(dev, inputs, lens, n_q, hq, hkv, q, out)
    bits = []
    for _ in range(2):
        call()
        if dev == "cuda":
            torch.cuda.synchronize()
            ops.check_errors()
        bits.append(out.cpu().clone())
    assert torch.equal(*bits)
    ref, tol = _attention_ref(q, *inputs, lens, n_q, hq // hkv, True, None)
    assert bool(((bits[0].double() - ref).abs() <= tol).all())
    t0 = 0
    for n, m in zip(lens, n_q):         # the first tokens, where there are more than keys
        assert not bits[0][t0:t0 + max(0, m - n)].any()
        t0 += m


@pytest.mark.gpu
@pytest.mark.parametrize("reach", REACH)
@pytest.mark.parametrize("bad", [-1, "past"])
def test_bad_blocks_on_every_kernel(reach, bad):
    n_q, lens = REACH[reach], [100, 300]
    kc, vc, ks, vs, tables = _paged_inputs(lens, 2, 16, 1)
    tables[1][2] = kc.shape[0] if bad == "past" else bad
    # block 0 stands in for the bad one: give it finite values
    kc, vc = (torch.nan_to_num(c.float()).to(c.dtype) for c in (kc, vc))
    ks, vs = (torch.nan_to_num(s, nan=1.0) for s in (ks, vs))
    q = torch.randn(sum(n_q), 8, D).bfloat16()
    out = torch.full(q.shape, 7.0, dtype=torch.bfloat16, device="cuda")
    _call("cuda", (kc, vc, ks, vs, tables), lens, n_q, 8, 2, q, out)()
    torch.cuda.synchronize()
    with pytest.raises(ops.KernelError):
        ops.check_errors()
    assert bool(torch.isfinite(out.float()).all())


@pytest.mark.gpu
@pytest.mark.parametrize("reach", REACH)
@pytest.mark.parametrize("cu", [[0, 300, 301], [-1, 3, 4], [2, 1, 0]])
def test_bad_offsets_on_every_kernel(reach, cu):
    n_q, lens = REACH[reach], [100, 300]
    q = torch.randn(sum(n_q), 8, D).bfloat16()
    buf = torch.full((q.shape[0] + 64, 8, D), 3.0, dtype=torch.bfloat16, device="cuda")
    _call("cuda", _paged_inputs(lens, 2, 16, 1), lens, n_q, 8, 2, q, buf[32:-32], cu=cu)()
    torch.cuda.synchronize()
    with pytest.raises(ops.KernelError):
        ops.check_errors()
    assert bool((buf[:32] == 3).all()) and bool((buf[-32:] == 3).all())


@pytest.mark.gpu
@pytest.mark.parametrize("reach", REACH)
def test_stream_and_graph_on_every_kernel(reach):
    n_q, lens = REACH[reach], [3000, 40]
    q = torch.randn(sum(n_q), 8, D).bfloat16()
    out = torch.zeros(q.shape, dtype=torch.bfloat16, device="cuda")
    call = _call("cuda", _paged_inputs(lens, 2, 16, 1), lens, n_q, 8, 2, q, out)
    call()
    torch.cuda.synchronize()
    want = out.clone()
    out.zero_()
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        torch.cuda._sleep(2_000_000)
        call()
    st.synchronize()
    assert torch.equal(out, want)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        call()
    for _ in range(3):
        out.zero_()
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want)
    ops.check_errors()


@on_devices
@pytest.mark.parametrize("reach", REACH)
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("hq,hkv", [(4, 1), (12, 3), (32, 8)])
def test_heads_masks_and_strides_on_every_kernel(dev, reach, causal, hq, hkv):
    """Strided q and out rows, any positive scales, more than one KV head."""
    n_q, lens = REACH[reach], [150, 77]
    inputs = _paged_inputs(lens, hkv, 32, hq, any_scale=True)
    t = sum(n_q)
    row = torch.randn(t, (hq + 2 * hkv) * D, generator=torch.Generator().manual_seed(hq)).bfloat16()
    q = row[:, :hq * D].view(t, hq, D)
    buf = torch.full((t, hq * D + 64), 7.0, dtype=torch.bfloat16, device=dev)
    group = hq // hkv
    offs = [0, n_q[0], t]
    tiles = [(i, r) for i, m in enumerate(n_q) for r in range(0, m * group, 256)]
    most = max(n_q) * group
    n0 = ops.launch_counter_value()
    ops.paged_attention_fp8(row.to(dev)[:, :hq * D].view(t, hq, D), *(z.to(dev) for z in inputs[:4]),
                            _i32(inputs[4], dev), _i32(lens, dev), _i32(offs, dev),
                            buf[:, :hq * D].view(t, hq, D), group, False,
                            tile_seq=_i32([a for a, _ in tiles], dev),
                            tile_row0=_i32([r for _, r in tiles], dev), causal=causal,
                            item_rows=min(most, 256))
    if dev == "cuda":
        assert ops.launch_counter_value() - n0 == (1 if most > 32 else 2)
        torch.cuda.synchronize()
        ops.check_errors()
    assert bool((buf[:, hq * D:] == 7).all())
    ref, tol = _attention_ref(q, *inputs, lens, n_q, group, causal, None)
    got = buf[:, :hq * D].view(t, hq, D).cpu().double()
    assert bool(((got - ref).abs() <= tol).all())
