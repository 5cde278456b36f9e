"""Work lists of the attention over the 8-bit cache: entries outside a sequence's rows."""
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
