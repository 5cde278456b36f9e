"""The engine with the 8-bit KV cache (``kv_dtype="fp8"``): step tables, append and attention
together, against the block manager's slots and the fp32 oracle."""
import numpy as np
import pytest
import torch

from lightbulb_b200 import ops
from lightbulb_b200.config import CacheConfig, EngineConfig, SchedulerConfig, get_preset
from lightbulb_b200.engine.llm_engine import LLMEngine
from lightbulb_b200.engine.sampling import SamplingParams
from lightbulb_b200.kv.device_tables import ResidentTables
from lightbulb_b200.models.llama import KVCache, kv_dtype_of
from lightbulb_b200.models.reference import ReferenceLlama
from lightbulb_b200.models.weights import pack_model, random_weights

DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]
on_devices = pytest.mark.parametrize("dev", DEVICES)
GREEDY = SamplingParams(temperature=0.0, max_tokens=12, ignore_eos=True)
PROMPTS = [list(range(5, 75)), [100, 200, 300], [7] * 50, [1], list(range(9, 42))]


def _engine(dev, kv_dtype="fp8", num_blocks=64, block_size=16, graphs=False, overlap=True,
            preset="tiny-test", **cache):
    cfg = get_preset(preset)
    w = random_weights(cfg, seed=1, std=0.05)
    w = {k: v.to(torch.bfloat16).float() for k, v in w.items()}
    packed = pack_model(cfg, w, dtype=torch.bfloat16, device=dev)
    ecfg = EngineConfig(model=cfg, cache=CacheConfig(num_blocks=num_blocks, block_size=block_size,
                                                     kv_dtype=kv_dtype, **cache),
                        scheduler=SchedulerConfig(max_num_seqs=8, max_num_batched_tokens=64,
                                                  chunk_size=32, max_model_len=256),
                        use_cuda_graphs=graphs, overlap_decode=overlap)
    return cfg, w, packed, LLMEngine(ecfg, packed)


def _check(dev):
    if dev == "cuda":
        torch.cuda.synchronize()
        ops.check_errors()


def _watch_slots(eng):
    """Every forward's device-built slots, positions and tables against the scheduler's."""
    seen = []
    execute, forward = eng.runner.execute, eng.model.forward

    def ex(so, *a, **k):
        seen.append(so.decode + so.prefill)
        return execute(so, *a, **k)

    def fw(b, kv):
        chunks = seen[-1]
        want = [s for c in chunks for s in c.slots]
        assert b.slots.tolist()[:len(want)] == want
        assert b.positions.tolist()[:len(want)] == [
            p for c in chunks for p in range(c.start, c.start + c.num_tokens)]
        for i, c in enumerate(chunks):
            t = eng.blocks.block_table(c.seq.seq_id)
            n = -(-(c.start + c.num_tokens) // eng.kv.block_size)
            assert b.block_tables[i, :n].tolist() == t[:n]
        return forward(b, kv)

    eng.runner.execute, eng.model.forward = ex, fw
    return seen


@on_devices
@pytest.mark.parametrize("preset", ["tiny-test", "qwen3-tiny-test"])
@pytest.mark.parametrize("block_size", [16, 32])
def test_generates_like_the_oracle(dev, preset, block_size):
    cfg, w, _, eng = _engine(dev, block_size=block_size, preset=preset)
    seen = _watch_slots(eng)
    seqs = eng.generate(prompt_token_ids=PROMPTS, params=GREEDY)
    _check(dev)
    assert len(seen) > 12
    ref = ReferenceLlama(cfg, w)
    for p, s in zip(PROMPTS, seqs):
        ref.reset()
        lg = ref.forward(torch.tensor(p + s.output_token_ids[:-1]))[len(p) - 1:]
        for i, t in enumerate(s.output_token_ids):
            # a stored element is off by up to 2^-4 of its value: an emitted token is the oracle's
            # best, or within 2^-3 of the logits' spread of it
            assert float(lg[i].max() - lg[i][t]) <= 0.125 * float(lg[i].std()) * 4
    assert eng.blocks.check_invariants()


@on_devices
def test_preemption_prefix_reuse_and_rows(dev):
    """Few blocks: sequences are preempted and recomputed, blocks change owners, prefixes are
    shared; the device's tables follow."""
    _, _, _, eng = _engine(dev, num_blocks=14, overlap=False)
    _watch_slots(eng)
    prompts = [list(range(40)), list(range(32)) + [500, 501], list(range(40)) + [3] * 9, [8] * 60,
               [9] * 20]
    sp = SamplingParams(temperature=0.0, max_tokens=50, ignore_eos=True)
    outs = []
    for _ in range(2):
        outs.append([s.output_token_ids for s in eng.generate(prompt_token_ids=prompts, params=sp)])
    _check(dev)
    assert eng.scheduler.num_preemptions > 0
    assert all(len(o) == 50 for r in outs for o in r)


@on_devices
def test_speculative_verify_runs_on_the_fp8_cache(dev):
    cfg, _, packed, eng = _engine(dev)
    plain = [s.output_token_ids for s in eng.generate(prompt_token_ids=PROMPTS[:3],
                                                      params=GREEDY)]
    _, _, _, eng2 = _engine(dev)
    spec = eng2.attach_draft(packed, cfg, k=3)
    out = [s.output_token_ids for s in eng2.generate(prompt_token_ids=PROMPTS[:3], params=GREEDY)]
    _check(dev)
    assert spec.stats.rounds > 0 and [len(o) for o in out] == [len(o) for o in plain]


@pytest.mark.gpu
@pytest.mark.parametrize("overlap", [False, True])
def test_graphs_and_overlap_give_the_same_tokens(overlap):
    a, b = (_engine("cuda", graphs=g, overlap=o)[3] for g, o in ((False, False), (True, overlap)))
    ra, rb = ([s.output_token_ids for s in e.generate(prompt_token_ids=PROMPTS, params=GREEDY)]
              for e in (a, b))
    _check("cuda")
    assert ra == rb
    # a steady decode uploads no table rows: only admissions do
    assert b.runner.tables.uploads <= 2 * len(PROMPTS)


@on_devices
def test_copy_blocks_copies_scales(dev):
    kv = KVCache(2, 6, 2, 16, 128, dtype=kv_dtype_of("fp8"), device=dev)
    raw = torch.randint(0, 120, kv.storage.shape, dtype=torch.uint8)
    kv.storage.view(torch.uint8).copy_(raw)
    kv.scales.copy_(torch.rand(kv.scales.shape) + 1)
    before = kv.scales.clone()
    kv.copy_blocks([1, 4, 0, 5])
    st = kv.storage.view(torch.uint8).cpu()
    for src, dst in ((1, 4), (0, 5)):
        assert torch.equal(st[:, :, dst], raw[:, :, src])
        assert torch.equal(kv.scales[:, :, dst], before[:, :, src])
    assert torch.equal(st[:, :, :4], raw[:, :, :4])


def test_half_the_bytes():
    bf, f8 = (KVCache.bytes_per_block(4, 8, 16, 128, kv_dtype_of(n).itemsize)
              for n in ("bf16", "fp8"))
    assert bf == 4 * 2 * 8 * 16 * 128 * 2 and f8 == bf // 2 + 4 * 2 * 8 * 4


@on_devices
def test_resident_tables_follow_a_changing_host(dev):
    rng = np.random.default_rng(0)
    bs, width, n_rows = 16, 8, 5
    t = ResidentTables(n_rows, width, dev)
    host, lens = {}, {}
    for step in range(60):
        ids = list(rng.choice(9, size=rng.integers(1, n_rows + 1), replace=False))
        ctx, q = [], []
        for sid in ids:
            if sid not in host or rng.random() < 0.1:      # new, or preempted and re-admitted
                host[sid], lens[sid] = rng.permutation(1000)[:width].astype(np.int32), 0
            elif rng.random() < 0.1:                       # copy-on-write of an old block
                host[sid][rng.integers(0, width)] += 1000
            n = int(rng.integers(0, min(20, width * bs - lens[sid]) + 1))
            ctx.append(lens[sid])
            q.append(n)
            lens[sid] += n
            if lens[sid] > width * bs - 20:
                host.pop(sid)
        tab = np.stack([host.get(s, np.arange(width, dtype=np.int32)) for s in ids])
        ctx, q = np.array(ctx, np.int32), np.array(q, np.int32)
        rows, new = t.place(ids, tab, ctx, q, bs)
        dv = lambda v: torch.from_numpy(np.ascontiguousarray(v, dtype=np.int32)).to(dev)  # noqa: E731
        r = ops.step_tables(dv(ctx), dv(q), dv(rows), t.tables, dv(new), int(q.sum()), bs)
        _check(dev)
        for i in range(len(ids)):
            need = -(-int(ctx[i] + q[i]) // bs)
            assert r.block_tables[i, :need].tolist() == tab[i, :need].tolist()
    assert t.tables.cpu().numpy().tolist() == t.mirror.tolist()
    with pytest.raises(ValueError):
        t.place(list(range(n_rows + 1)), np.zeros((n_rows + 1, width), np.int32),
                np.zeros(n_rows + 1, np.int32), np.zeros(n_rows + 1, np.int32), bs)


def test_refusals(tmp_path):
    with pytest.raises(ValueError):
        _engine("cpu", kv_dtype="int3")
    with pytest.raises(ValueError):
        _engine("cpu", block_size=8)
    with pytest.raises(ValueError):
        _engine("cpu", h2o_budget=32)
    _, _, _, eng = _engine("cpu")
    for call in (lambda: eng.enable_kv_compression("streaming", 64),
                 eng.enable_segmented_cache):
        with pytest.raises(ValueError):
            call()
    from lightbulb_b200.extras.state import save_engine_state
    with pytest.raises(ValueError):
        save_engine_state(eng, str(tmp_path / "s.bin"))
    assert save_engine_state(eng, str(tmp_path / "s.bin"), include_kv=False)["requests"] == 0
