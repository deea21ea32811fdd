"""GPU tests of tree attention over the 8-bit key/value cache, beside those of
test_gpu_kvq8.py: what the slots that no row sees may hold.
"""

import math

import pytest
import torch

from test_gpu_kvq8 import BF, DEV, F32, attention_ref, check, new_layer, rand, visible_ref

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ops():
    from ssd import ops as O

    return O


@pytest.fixture(scope="module")
def ws(ops):
    return ops.Workspace(torch.device(DEV), max_rows=512, vocab=128)


# ------------------------------------------------------------ unseen slots
@pytest.mark.parametrize("byte", [0, 247, 254, 255])
@pytest.mark.parametrize("T", [1, 6, 40, 300])
@pytest.mark.parametrize("dtype,hd", [(BF, 64), (BF, 128), (BF, 80), (F32, 64)])
def test_unseen_slots_may_hold_any_byte(ops, ws, dtype, hd, T, byte):
    """Any code and any scale byte, those beyond the largest written among them, in
    slots that no row sees: before and behind the ranges, and between the mask's
    bits, in blocks of which some slots are seen."""
    H, Hkv, slots, base = 8, 2, 1500, 1203
    q = rand(T, H * hd, dtype=dtype, seed=10)
    i32 = dict(dtype=torch.int32, device=DEV)
    plen = torch.arange(T, **i32) % 7 + 1100
    start = torch.full((T,), 70, **i32)
    mask = torch.zeros(T, 2, dtype=torch.int64, device=DEV)
    mask[:, 0], mask[:, 1] = 0x8001_0000_0011, 5
    see = visible_ref(T, slots, plen, start, base, mask)
    unseen = ~see.any(0)
    assert unseen[:70].all() and unseen[1204:1207].all() and not unseen[1203]
    outs = []
    for dirty in (False, True):
        layer = new_layer(ops, Hkv, slots, hd, seed=11)
        if dirty:
            codes = torch.randint(0, 256, (Hkv, slots, hd), generator=torch.Generator(DEV).manual_seed(12), device=DEV)
            for c, s in ((layer.k, layer.k_scale), (layer.v, layer.v_scale)):
                c.view(torch.uint8)[:, unseen] = codes.to(torch.uint8)[:, unseen]
                s[:, unseen] = byte
        out = torch.full((T, H * hd), math.nan, dtype=dtype, device=DEV)
        ops.tree_attention_q8(q, layer, H, Hkv, hd, plen, out, ws, prefix_start=start,
                              spec_base=torch.tensor([base], **i32), spec_mask=mask)
        outs.append(out)
        if not dirty:
            check(out, attention_ref(q, layer, H, see), layer, see, dtype)
    ws.check_status()
    assert torch.equal(outs[0], outs[1])
