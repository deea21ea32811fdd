"""GPU tests of tree attention over the 8-bit key/value cache, beside those of
test_gpu_kvq8.py: what the slots that no row sees may hold, and how exactly
weights are held that lie far below a row's largest.

Tolerance of the latter (bf16, tensor cores). A weight is off by 2^-10 of itself
at most plus 2^-12 for its fp16 form, and by 2^-27 of the largest where it is
smaller than 2^-18 of that; with n keys the mean of the values is then off by
(1.25 2^-10 + n 2^-27) max |v|, the bf16 result by 2^-9 of max |v| more. For
n = 32768 that is 0.0034, below the 2^-8 = 0.0039 that is asked for. Query elements
down to 2^-13 of their row's largest are exact.
"""

import math

import pytest
import torch

import kvq8_cases
from test_gpu_kvq8 import BF, DEV, F32, attention_ref, check, new_layer, quantise_ref, rand, visible_ref

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


# ------------------------------------------------------------ small weights
def sink_and_tail(ops, slots, hd, tail_v, sink_v):
    """One KV head: slot 77 with key (s, 0, ..), every other slot with key (0, 1, 0, ..)."""
    k = torch.zeros(1, slots, hd, device=DEV)
    k[:, :, 1], k[:, 77] = 1.0, 0.0
    k[:, 77, 0] = 1.0
    v = torch.full_like(k, tail_v)
    v[:, 77] = sink_v
    (kc, ks), (vc, vs) = quantise_ref(k), quantise_ref(v)
    return ops.KVLayerQ8(kc, vc, ks, vs)


def sweep_rows(T, H, hd, deepest, shallowest, seed):
    """Query rows whose tail keys lie 2^-deepest .. 2^-shallowest below the sink, evenly
    spaced in the exponent; off the whole exponents in both keys' scores."""
    q = torch.zeros(T * H, hd, device=DEV)
    depth = torch.linspace(deepest, shallowest, T * H, device=DEV, dtype=torch.float64)
    at = torch.linspace(0.13, 0.97, T * H, device=DEV, dtype=torch.float64)[
        torch.randperm(T * H, generator=torch.Generator(DEV).manual_seed(seed), device=DEV)]
    q[:, 0] = ((at + depth) * math.log(2) * math.sqrt(hd)).float()
    q[:, 1] = (at * math.log(2) * math.sqrt(hd)).float()
    return q.to(BF).view(T, H * hd)


@pytest.mark.parametrize("slots,deepest,shallowest", [(2048, 14, 8), (2049, 11, 10), (4096, 13, 11), (32768, 18, 12),
                                                      (32700, 16, 15), (32768, 23, 18)])
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("T,H", [(1, 4), (7, 4), (16, 4), (9, 8), (29, 4), (300, 4)])
def test_a_flat_tail_beside_a_sink_keeps_its_share(ops, ws, T, H, hd, slots, deepest, shallowest):
    """A strong key beside thousands of equal ones that hold from a few hundredths
    to nearly all of the weight together. Values of +1 and -1: the result shows the
    tail's share; values of one everywhere give one exactly."""
    q = sweep_rows(T, H, hd, deepest, shallowest, T)
    plen = torch.full((T,), slots, dtype=torch.int32, device=DEV)
    see = visible_ref(T, slots, plen)
    for tail_v, sink_v in ((1.0, -1.0), (-1.0, 0.25), (1.0, 1.0)):
        layer = sink_and_tail(ops, slots, hd, tail_v, sink_v)
        out = torch.empty_like(q)
        ops.tree_attention_q8(q, layer, H, 1, hd, plen, out, ws)
        ws.check_status()
        if tail_v == sink_v:
            assert (out == 1).all(), (out.double() - 1).abs().max().item()
            continue
        err = (out.double() - attention_ref(q, layer, H, see)).abs().max().item()
        assert err <= 2.0**-8, err


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("depth", [9, 11, 13])
def test_small_query_elements_are_exact(ops, ws, hd, depth):
    """Scores of about 20 from query elements 2^-depth of the row's largest, which
    meets zeros in the keys: of two keys one adds up many such elements with all of
    their 8 bits in use, the other a single one that is a power of two."""
    T, S, root = 64, 20.0, math.sqrt(hd)
    c = 2.0**-depth * (1 + (2 * torch.arange(T, device=DEV) + 1) / 128)  # the last of 8 bits is set
    q = c[:, None].repeat(1, hd)
    q[:, 0], q[:, 1] = 1.0, 2.0**-depth
    k, v = torch.zeros(1, 2, hd, device=DEV), torch.ones(1, 2, hd, device=DEV)
    k[0, 0, 2:] = S * root / ((hd - 2) * 1.4 * 2.0**-depth)
    k[0, 1, 1] = S * root * 2.0**depth
    v[0, 1] = -1
    (kc, ks), (vc, vs) = quantise_ref(k), quantise_ref(v)
    layer = ops.KVLayerQ8(kc, vc, ks, vs)
    q = q.to(BF)
    assert torch.equal(q[:, 2].float(), c)
    plen = torch.full((T,), 2, dtype=torch.int32, device=DEV)
    out = torch.empty_like(q)
    ops.tree_attention_q8(q, layer, 1, 1, hd, plen, out, ws)
    ws.check_status()
    ref = attention_ref(q, layer, 1, visible_ref(T, 2, plen))
    assert (ref.abs().amin() < 0.9)  # the keys compete in some rows
    err = (out.double() - ref).abs().max().item()
    assert err <= 2.0**-8, err


# -------------------------------------------------------------- visibility
@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("args", kvq8_cases.CASES, ids=lambda a: "-".join(map(str, a)))
def test_every_slot_counts(ops, ws, dtype, args):
    """Inputs in which one slot too many or too few shows (test_cpu_kvq8_visibility.py),
    against the 64-bit result, channel by channel."""
    c = kvq8_cases.case(*args, DEV)
    H, Hkv, hd, T = c["H"], c["Hkv"], c["hd"], c["T"]
    layer = ops.KVLayerQ8(c["k"], c["v"], c["ks"], c["vs"])
    q = c["q"].to(dtype)
    out = torch.full((T, H * hd), math.nan, dtype=dtype, device=DEV)
    ops.tree_attention_q8(q, layer, H, Hkv, hd, c["len"], out, ws, prefix_start=c["start"], spec_mask=c["mask"],
                          spec_base=None if c["base"] is None else torch.tensor([c["base"]], dtype=torch.int32, device=DEV),
                          kv_bound=c["bound"])
    ws.check_status()
    ref = kvq8_cases.attention(c, q, kvq8_cases.visible(c))
    err = ((out.double().view(T, H, hd) - ref).abs() / ref.abs().clamp(min=2.0**-40)).amax().item()
    assert err <= kvq8_cases.TOL, err
