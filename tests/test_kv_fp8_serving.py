"""What the engine generates from the 8-bit cache, token by token against the fp32 oracle."""
import pytest
import torch

from lightbulb_b200 import ops
from lightbulb_b200.config import CacheConfig, EngineConfig, SchedulerConfig
from lightbulb_b200.engine.llm_engine import LLMEngine
from lightbulb_b200.engine.sampling import SamplingParams
from lightbulb_b200.models.reference import ReferenceLlama
from test_kv_fp8_engine import GREEDY, PROMPTS, _check, _engine, _watch_slots, on_devices


def _check_tokens(cfg, w, prompts, outs):
    """Every emitted token's oracle logit lies within half a standard deviation of its row's best.
    (The cache's elements are off by up to 2^-4 of their value; a token picked at random lies about
    four deviations below the best of a vocabulary of this size.)"""
    ref = ReferenceLlama(cfg, w)
    for p, out in zip(prompts, outs):
        ref.reset()
        lg = ref.forward(torch.tensor(p + out[:-1]))[len(p) - 1:]
        for row, t in zip(lg, out):
            assert float(row.max() - row[t]) <= 0.5 * float(row.std())


@on_devices
def test_the_draft_has_the_engines_cache(dev):
    """The draft's pool is 8-bit too: as many blocks, half the bytes of a bf16 one.  With the
    target's own weights nearly every proposal is accepted, and what is emitted is right."""
    cfg, w, packed, eng = _engine(dev)
    spec = eng.attach_draft(packed, cfg, k=3)
    kv = spec.draft.kv
    assert kv.storage.dtype == eng.kv.storage.dtype and kv.num_blocks == eng.kv.num_blocks
    assert kv.storage.numel() * kv.storage.element_size() == eng.kv.storage.numel()
    _watch_slots(eng)
    outs = [s.output_token_ids for s in eng.generate(prompt_token_ids=PROMPTS, params=GREEDY)]
    _check(dev)
    assert spec.stats.rounds > 0 and spec.stats.acceptance_rate() > 0.7
    _check_tokens(cfg, w, PROMPTS, outs)


@pytest.mark.parametrize("name", ["bf16", "bfloat16", "auto"])
def test_names_of_the_bf16_cache(name):
    """The field was not read once: configurations that spell bf16 otherwise still run."""
    _, _, _, eng = _engine("cpu", kv_dtype=name, block_size=8)
    assert eng.kv.storage.dtype == torch.bfloat16 and not eng.kv.fp8


@on_devices
@pytest.mark.parametrize("graphs", [False, True])
def test_more_sequences_than_at_the_start(dev, graphs):
    """The batch-size adjuster raises the scheduler's limit while the engine runs: steps with more
    sequences than the resident tables have rows, and smaller ones (captured graphs) after them."""
    if graphs and dev == "cpu":
        pytest.skip("CUDA graphs")
    cfg, w, _, eng = _engine(dev, num_blocks=200, graphs=graphs)
    first = [s.output_token_ids for s in eng.generate(prompt_token_ids=PROMPTS, params=GREEDY)]
    rows = eng.runner.tables.tables.shape[0]
    n = rows + 5
    eng.scheduler.cfg.max_num_seqs = n
    prompts = [[i + 3, i, 2 * i] for i in range(n)]
    outs = [s.output_token_ids for s in eng.generate(prompt_token_ids=prompts, params=GREEDY)]
    again = [s.output_token_ids for s in eng.generate(prompt_token_ids=PROMPTS, params=GREEDY)]
    _check(dev)
    assert eng.runner.tables.tables.shape[0] >= n
    assert eng.runner.tables.tables.cpu().tolist() == eng.runner.tables.mirror.tolist()
    _check_tokens(cfg, w, PROMPTS + prompts + PROMPTS, first + outs + again)


def test_too_many_sequences_are_refused_when_the_engine_is_built():
    """Not by the step that first has them."""
    cfg, _, packed, _ = _engine("cpu")

    def build(kv_dtype, n):
        return LLMEngine(EngineConfig(model=cfg, cache=CacheConfig(num_blocks=16, kv_dtype=kv_dtype),
                                      scheduler=SchedulerConfig(max_num_seqs=n, max_model_len=64,
                                                                max_num_batched_tokens=64)), packed)
    build("bf16", ops.MAX_REQUESTS + 1)
    build("fp8", ops.MAX_REQUESTS)
    with pytest.raises(ValueError, match="max_num_seqs"):
        build("fp8", ops.MAX_REQUESTS + 1)


@on_devices
def test_preempted_and_prefix_sharing_requests(dev):
    """Few blocks: sequences are preempted and computed again, blocks change owners, prefixes are
    shared; twice over, so the second pass starts from a used cache.  Tokens, not lengths."""
    cfg, w, _, eng = _engine(dev, num_blocks=14, overlap=False)
    _watch_slots(eng)
    prompts = [list(range(40)), list(range(32)) + [500, 501], list(range(40)) + [3] * 9, [8] * 60,
               [9] * 20]
    sp = SamplingParams(temperature=0.0, max_tokens=30, ignore_eos=True)
    for _ in range(2):
        outs = [s.output_token_ids for s in eng.generate(prompt_token_ids=prompts, params=sp)]
        _check(dev)
        assert all(len(o) == 30 for o in outs)
        _check_tokens(cfg, w, prompts, outs)
    assert eng.scheduler.num_preemptions > 0


@on_devices
def test_prompts_arriving_while_others_decode(dev):
    """Steps that hold decodes and prompt chunks of both attention kernels' sizes."""
    cfg, w, _, eng = _engine(dev, overlap=False)
    seen = _watch_slots(eng)
    prompts = [list(range(i + 2, i + 2 + n)) for i, n in enumerate((3, 90, 5, 130, 1, 64, 40))]
    seqs = []
    for i, p in enumerate(prompts):
        seqs.append(eng.add_request(f"r{i}", prompt_token_ids=p, params=GREEDY))
        eng.step()
        eng.step()
    while eng.has_unfinished():
        eng.step()
    _check(dev)
    kinds = [sorted({c.num_tokens > 1 for c in chunks}) for chunks in seen]
    assert [False, True] in kinds
    _check_tokens(cfg, w, prompts, [s.output_token_ids for s in seqs])


@on_devices
@pytest.mark.parametrize("start", [3, 15, 16])
def test_append_after_a_rollback(dev, start):
    """Draft tokens of much larger magnitude are appended, rejected, and others take their slots: the
    tokens before them stay within a step of the grown scale, the new ones within half a step."""
    d, bs, n, k = 128, 16, 20, 5
    gen = torch.Generator().manual_seed(start)
    x = torch.randn(n, 3 * d, generator=gen).bfloat16()
    big = (torch.randn(k, 3 * d, generator=gen) * 300).bfloat16()
    kc = torch.zeros(2, 1, bs, d, dtype=ops.FP8_KV_DTYPE, device=dev)
    vc, ks, vs = kc.clone(), torch.ones(2, 1, device=dev), torch.ones(2, 1, device=dev)
    cs = ops.rope_table(64, d, 1e4, dev)

    def append(rows, first):
        pos = torch.arange(first, first + len(rows), dtype=torch.int32, device=dev)
        ops.rope_kv_fp8(rows.to(dev), pos, pos, cs, kc, vc, ks, vs, 1, 1)
    append(x[:start], 0)
    append(big, start)                # rejected
    append(x[start:], start)
    _check(dev)
    s = vs.cpu().double()[:, :, None, None]
    got = (vc.cpu().double() * s).view(2 * bs, d)[:n]
    want = x[:, 2 * d:].double()
    step = (s * torch.ones(2, 1, bs, 1, dtype=torch.float64)).view(2 * bs, 1)[:n] * 2.0 ** -9
    # half a step when stored (2^-4 of the value, 2^-10 of the scale), and half a step below the
    # normal numbers when the scale grew
    assert bool(((got - want).abs() <= torch.maximum(want.abs() * 2.0 ** -4, step / 2) + step / 2).all())
    # a block that the rejected tokens had begun starts anew: its scale is that of what it holds
    amax = float(want[bs:].abs().max())
    assert float(vs[1, 0]) * 448 >= amax > float(vs[1, 0]) * 224
