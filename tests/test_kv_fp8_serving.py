"""What the engine generates from the 8-bit cache, token by token against the fp32 oracle."""
import pytest
import torch

from lightbulb_b200 import ops
from lightbulb_b200.config import CacheConfig, EngineConfig, SchedulerConfig
from lightbulb_b200.engine.llm_engine import LLMEngine
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
