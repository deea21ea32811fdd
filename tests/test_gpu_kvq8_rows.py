"""GPU tests of rows that reach the 8-bit key/value cache straight from a projection's
fp32 sums: the rotated query is rounded to bf16 once, keys and values only to their codes."""

import pytest
import torch

from test_gpu_kvq8 import BF, DEV, F32, WRITES, new_layer, quantise_ref, rand, rotate_ref, tables

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ops():
    from ssd import ops as O

    return O


@pytest.fixture(scope="module")
def ws(ops):
    return ops.Workspace(torch.device(DEV), max_rows=512, vocab=128)


@pytest.mark.parametrize("shift", [0, 1])  # rows in aligned vectors or not
@pytest.mark.parametrize("T,H,Hkv,hd,rot,inter", WRITES + [(600, 40, 40, 64, 24, False), (3, 8, 2, 128, 64, False),
                                                           (400, 3, 20, 128, 128, True)])
def test_fp32_rows_into_a_bf16_query(ops, ws, T, H, Hkv, hd, rot, inter, shift):
    wide = rand(T, (H + 2 * Hkv) * hd + 8, seed=1)[:, shift:]
    q, k, v = wide[:, :H * hd], wide[:, H * hd:(H + Hkv) * hd], wide[:, (H + Hkv) * hd:(H + 2 * Hkv) * hd]
    layer = new_layer(ops, Hkv, T, hd)
    cos, sin = tables(rot, 700) if rot else (None, None)
    i32 = dict(dtype=torch.int32, device=DEV)
    pos, where = torch.randint(0, 700, (T,), **i32), torch.randperm(T, device=DEV).to(torch.int32)
    out = torch.zeros(T, H * hd + 16, dtype=BF, device=DEV)
    ops.rope_kv_write_q8(q, k, v, H, Hkv, hd, cos, sin, pos, where, layer, out[:, 8 + shift:8 + shift + H * hd], ws,
                         interleaved=inter)
    ws.check_status()
    turn = (lambda x, n: rotate_ref(x.reshape(T, n, hd), cos, sin, pos, rot, inter)) if rot else \
        (lambda x, n: x.reshape(T, n, hd))
    want = torch.zeros_like(out)
    want[:, 8 + shift:8 + shift + H * hd] = turn(q, H).reshape(T, -1).to(BF)
    assert torch.equal(out, want)
    for x, codes, scale in ((turn(k, Hkv), layer.k, layer.k_scale), (v.reshape(T, Hkv, hd), layer.v, layer.v_scale)):
        c, s = quantise_ref(x)
        assert torch.equal(codes.view(torch.uint8)[:, where.long()], c.view(torch.uint8).transpose(0, 1))
        assert torch.equal(scale[:, where.long()], s.transpose(0, 1))


def test_wrong_pairs_of_types_are_refused(ops, ws):
    layer = new_layer(ops, 2, 4, 32)
    i32 = dict(dtype=torch.int32, device=DEV)
    cos, sin = tables(32, 8)
    pos = torch.arange(3, **i32)
    q, k = rand(3, 4 * 32), rand(3, 2 * 32)
    for q1, k1, out in ((q, k, q.half()), (q.to(BF), k.to(BF), q.clone()), (q, k.to(BF), q.to(BF)), (q.to(BF), k, q.to(BF))):
        with pytest.raises(ValueError):
            ops.rope_kv_write_q8(q1, k1, k1, 4, 2, 32, cos, sin, pos, pos, layer, out, ws)


@pytest.mark.parametrize("rows", [1, 7, 33, 200])
def test_a_forwards_queries_are_rounded_once(rows):
    """One layer of the 1B shape over either cache: the same sums, rotated and rounded
    once, so that the queries are equal but for what contracted products move (2^-24
    of a sum, across a border of bf16's 2^-8 in one of 10^4 elements or so). Rounded
    before the rotation too, one in four differed."""
    from ssd import synthetic as S
    from ssd.engine.speculative import TargetRunner

    base = S.build_base_model("llama32_1b", 1, torch.bfloat16, DEV, gen_device="cuda", num_hidden_layers=1, vocab_size=512)
    ids = torch.randint(0, 512, (1, rows), generator=torch.Generator().manual_seed(3)).to(DEV)
    got = []
    for kv in (None, "e4m3"):
        t = TargetRunner(base, kv_dtype=kv)
        t(ids, past_key_values=t.new_cache(256))
        got.append(t._scratch.q[:rows].clone())
    differ = (got[0] != got[1]).float().mean().item()
    assert differ < 0.005 and bool(got[0].abs().sum() > 0), differ
    off = (got[0].float() - got[1].float()).abs()  # a step of bf16 at most
    assert bool((off <= got[0].float().abs() * 2.0**-7 + 2.0**-20).all())
