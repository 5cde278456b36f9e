"""The 8-bit cache's operators refuse tensors that lie elsewhere than the call's device."""
import pytest
import torch

from lightbulb_b200 import ops
from test_kv_fp8 import D, E4M3, _i32

pytestmark = pytest.mark.gpu


def _cache():
    kc = torch.zeros(4, 2, 16, D, dtype=E4M3, device="cuda")
    s = torch.ones(4, 2, device="cuda")
    return dict(k_cache=kc, v_cache=kc.clone(), k_scale=s, v_scale=s.clone())


def _attention(list_form):
    a = dict(q=torch.zeros(1, 4, D, device="cuda").bfloat16(), **_cache(),
             block_tables=_i32([[0]], "cuda"), seq_lens=_i32([1], "cuda"),
             cu_q=_i32([0, 1], "cuda"), out=torch.zeros(1, 4, D, device="cuda").bfloat16(), group=2,
             decode=not list_form)
    if list_form:
        a.update(tile_seq=_i32([0], "cuda"), tile_row0=_i32([0], "cuda"))
    return ops.paged_attention_fp8, a, ("q",) if list_form else ("q", "cu_q")


def _append():
    norm = torch.ones(D, device="cuda").bfloat16()
    return ops.rope_kv_fp8, dict(
        qkv=torch.zeros(1, 8 * D, device="cuda").bfloat16(), positions=_i32([0], "cuda"),
        slots=_i32([0], "cuda"), cos_sin=ops.rope_table(8, 128, 1e4, "cuda"), **_cache(), hq=4,
        hkv=2, q_norm=norm, k_norm=norm.clone(),
        out=torch.zeros(1, 4, D, device="cuda").bfloat16()), ("qkv",)


def _tables():
    return ops.step_tables, dict(
        ctx_lens=_i32([1], "cuda"), q_lens=_i32([1], "cuda"), rows=_i32([0], "cuda"),
        seq_tables=_i32([[0, 0]], "cuda"), new_blocks=_i32([1], "cuda"), num_tokens=1,
        block_size=16), ("ctx_lens",)


@pytest.mark.parametrize("make", [lambda: _attention(False), lambda: _attention(True), _append,
                                  _tables], ids=["decode", "list", "append", "tables"])
def test_tensors_on_the_host_are_refused(make):
    call, args, skip = make()       # skip: chooses the CPU form, or is not read
    call(**args)
    for name, t in args.items():
        if torch.is_tensor(t) and name not in skip:
            with pytest.raises(RuntimeError):
                call(**{**args, name: t.cpu()})
    torch.cuda.synchronize()
    ops.check_errors()
