"""Attention over the 8-bit cache at the ends of its scales' range, on both kernels, against
64-bit forms."""
import math

import pytest
import torch

from lightbulb_b200 import ops
from test_kv_fp8 import D, E4M3, _attention_ref, _i32, _paged_inputs, _sync, on_devices

# decode; 5 tokens of group 4 (20 rows an item: the kernel of few rows); 70 tokens (tcgen05)
FORMS = {"decode": (1, True), "few": (5, False), "chunk": (70, False)}
on_forms = pytest.mark.parametrize("form", FORMS)


def _run(dev, form, inputs, lens, q, scale=None):
    """One call; returns the output and the 64-bit values with their bound (bf16's rounding and
    the weights' 11 bits; nothing absolute)."""
    m, decode = FORMS[form]
    kc, vc, ks, vs, tables = inputs
    group = q.shape[1] // kc.shape[1]
    n_q = [m] * len(lens)
    cu = [m * i for i in range(len(lens) + 1)]
    tiles = [(i, r) for i in range(len(lens)) for r in range(0, m * group, 256)]
    out = torch.full(q.shape, 7.0, dtype=torch.bfloat16, device=dev)
    n0 = ops.launch_counter_value()
    ops.paged_attention_fp8(q.to(dev), *(z.to(dev) for z in (kc, vc, ks, vs)), _i32(tables, dev),
                            _i32(lens, dev), _i32(cu, dev), out, group, decode,
                            tile_seq=_i32([a for a, _ in tiles], dev),
                            tile_row0=_i32([r for _, r in tiles], dev), scale=scale)
    _sync(dev)
    if dev == "cuda":
        assert ops.launch_counter_value() - n0 == (1 if form == "chunk" else 2)
    ref, tol = _attention_ref(q, kc, vc, ks, vs, tables, lens, n_q, group, not decode, scale)
    return out.cpu().double(), ref, (tol - 1e-30).clamp(min=0)


def _ranged_inputs(form, bits, blocks, v_exp, seed):
    """One sequence of 300 keys.  Keys of ``blocks`` score ``bits`` (in powers of two of the
    weight) more than the others', whatever the query head; their V scale is 2**v_exp times the
    others'."""
    m, _ = FORMS[form]
    lens = [300]
    kc, vc, ks, vs, tables = _paged_inputs(lens, 2, 16, seed)
    ids = [tables[0][b] for b in blocks]
    ks[:] = torch.where(torch.isnan(ks), ks, 2.0 ** -8)
    vs[:] = torch.where(torch.isnan(vs), vs, 2.0 ** -6)
    live = kc.view(torch.uint8) != 0x7F
    # channel 0 carries the difference: q has 16 there; elsewhere the keys of `blocks` are zero
    kc.view(torch.uint8)[..., 0] = torch.where(live[..., 0], 0, 0x7F).to(torch.uint8)
    for i in ids:
        kc[i] = torch.zeros(kc.shape[1:]).to(E4M3)
        code = torch.tensor(bits * math.log(2) * math.sqrt(D) / 16).to(E4M3)
        kc.view(torch.uint8)[i, :, :, 0] = code.view(torch.uint8)
        ks[i] = 1.0
        vs[i] = 2.0 ** (v_exp - 6)
    q = torch.randn(m, 8, D, generator=torch.Generator().manual_seed(seed)) * 0.5
    q[..., 0] = 16
    return (kc, vc, ks, vs, tables), lens, q.bfloat16()


@on_devices
@on_forms
@pytest.mark.parametrize("blocks", [(4, 11), (0,), (18,)])
@pytest.mark.parametrize("bits,v_exp", [(40, -20), (60, -40), (110, -90),    # attended, small V
                                        (-30, 30), (-45, 45), (-90, 90)])    # faint, large V
def test_v_scales_far_apart(dev, form, blocks, bits, v_exp):
    """Blocks whose V scale lies up to 2^90 from the others' count by their weight times their
    scale, not by the scale alone."""
    inputs, lens, q = _ranged_inputs(form, bits, blocks, v_exp, seed=7)
    out, ref, tol = _run(dev, form, inputs, lens, q)
    assert bool(((out - ref).abs() <= tol).all())


@on_devices
@on_forms
@pytest.mark.parametrize("exp", [-112, -60, 60, 110])
def test_v_scales_small_and_large(dev, form, exp):
    """All V scales near one end of the range; a block of zeros in front."""
    lens = [300, 40, 129]
    kc, vc, ks, vs, tables = _paged_inputs(lens, 2, 16, 11)
    vs *= 2.0 ** exp
    vc.view(torch.uint8)[tables[0][0]] = 0
    m, _ = FORMS[form]
    lens = [max(n, m) for n in lens] if form == "few" else lens
    q = torch.randn(m * 3, 8, D, generator=torch.Generator().manual_seed(2)).bfloat16()
    out, ref, tol = _run(dev, form, (kc, vc, ks, vs, tables), lens, q)
    assert bool(((out - ref).abs() <= tol).all())


@on_devices
@on_forms
@pytest.mark.parametrize("q_exp,k_exp,scale", [(-100, -40, None), (-20, -40, 1e-30), (0, 0, 0.0),
                                               (0, 0, -0.1), (-100, -40, -1.0)])
def test_scores_that_vanish_or_change_sign(dev, form, q_exp, k_exp, scale):
    """A score factor (softmax scale, key scale, size of q) that underflows, is zero or negative:
    masked keys stay masked."""
    lens = [300, 75]
    kc, vc, ks, vs, tables = _paged_inputs(lens, 2, 16, 5)
    ks *= 2.0 ** k_exp
    m, _ = FORMS[form]
    q = torch.randn(m * 2, 8, D, generator=torch.Generator().manual_seed(3)) * 2.0 ** q_exp
    out, ref, tol = _run(dev, form, (kc, vc, ks, vs, tables), lens, q.bfloat16(), scale)
    assert bool(((out - ref).abs() <= tol).all())


@on_devices
@on_forms
@pytest.mark.parametrize("blocks", [(0,), (0, 1), (5, 6, 7), (18,), tuple(range(19))])
def test_scales_of_zero_stand_for_blocks_of_zeros(dev, form, blocks):
    """A block of zeros may have scales of 0: its values add nothing, its keys count."""
    lens = [300, 129]
    kc, vc, ks, vs, tables = _paged_inputs(lens, 2, 16, 13)
    for b in blocks:
        for c, s in ((kc, ks), (vc, vs)):
            c.view(torch.uint8)[tables[0][b]] = 0
            s[tables[0][b]] = 0
    m, _ = FORMS[form]
    q = torch.randn(m * 2, 8, D, generator=torch.Generator().manual_seed(4)).bfloat16()
    out, ref, tol = _run(dev, form, (kc, vc, ks, vs, tables), lens, q)
    assert bool(((out - ref).abs() <= tol).all())


@pytest.mark.gpu
@on_forms
@pytest.mark.parametrize("block", [0, 600, 1249])
@pytest.mark.parametrize("bits", [0, 115])
def test_long_sequences_at_both_ends_of_the_spread(form, block, bits):
    """20,000 keys of equal weight, their V scales 2^-100 of one block's whose keys score ``bits`` less:
    the sum of the weights over the scales stays in range at both ends."""
    lens = [20000]
    kc, vc, ks, vs, tables = _paged_inputs(lens, 1, 16, 17)
    kc.view(torch.uint8).masked_fill_(kc.view(torch.uint8) != 0x7F, 0)
    vs[:] = torch.where(torch.isnan(vs), vs, 2.0 ** -90)
    i = tables[0][block]
    vs[i], ks[i] = 2.0 ** 10, 1.0
    kc[i, :, :, 0] = torch.tensor(-bits * math.log(2) * math.sqrt(D) / 16).to(E4M3)
    m, decode = FORMS[form]
    q = torch.randn(m, 4, D, generator=torch.Generator().manual_seed(5))
    q[..., 0] = 16
    out, ref, tol = _run("cuda", form, (kc, vc, ks, vs, tables), lens, q.bfloat16())
    assert bool(((out - ref).abs() <= tol).all())
