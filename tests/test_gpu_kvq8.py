"""GPU tests of the 8-bit key/value cache: quantised writes (with the rotary
embedding), reading back, tree attention over it and compaction, against
plain 64-bit restatements.

Tolerances. The codes of a row follow from one rounding of exact products and
sums, done in the stated order, so they are compared for equality (the
rotation is restated in fp32 with the same single roundings). A value read back as
bf16 or fp32 is exact. Attention: outputs are weighted means of the values, so
errors are bounded against max |v|:
 * fp32 (CUDA cores): scores of up to 128 products and exp in fp32. A score
   |s| <= 40 is off by at most (hd + 2) 2^-24 sum |q k| scale, under 2^-24 * 130 *
   40; the weights move by twice that, the sums over n keys add n 2^-24 in the
   worst case: 1e-3 would be the bound, random signs give under 2e-6: 2e-5.
 * bf16 (tensor cores): P is held to 8 significant bits (relative 2^-8 per
   weight, so at most 2^-8 max |v| on the mean), plus half a step of the bf16
   output, 2^-9 of its binade's top: 2^-8 |out|; together 2 * 2^-8 max |v|.
"""

import math

import pytest
import torch

pytestmark = pytest.mark.gpu

DEV = "cuda"
BF, F32 = torch.bfloat16, torch.float32


@pytest.fixture(scope="module")
def ops():
    from ssd import ops as O

    return O


@pytest.fixture(scope="module")
def ws(ops):
    return ops.Workspace(torch.device(DEV), max_rows=512, vocab=128)


def rand(*shape, dtype=F32, scale=1.0, seed=0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    return (torch.randn(*shape, generator=g, device=DEV) * scale).to(dtype)


def two_to(e):
    """2^e exactly, for whole e (fp64)."""
    return ((e.to(torch.int64) + 1023) << 52).view(torch.float64)


def quantise_ref(x):
    """fp32 rows [..., hd] -> (codes e4m3, scale bytes), by the row format's definition."""
    mag = torch.where(torch.isfinite(x), x, torch.zeros_like(x)).abs().double().amax(-1)
    e = torch.full(mag.shape, -40, dtype=torch.int64, device=x.device)
    for cand in range(-40, 119):  # the smallest exponent that holds amax
        e = torch.where(mag > 448.0 * 2.0**cand, cand + 1, e)
    y = (x.double() / two_to(e).unsqueeze(-1)).clamp(-448, 448).float()  # exact: a power of two
    return y.to(torch.float8_e4m3fn), (e + 127).to(torch.uint8)


def value(codes, scale):
    return codes.double() * two_to(scale.to(torch.int64) - 127).unsqueeze(-1)


def new_layer(ops, n_kv, slots, hd, seed=None, pad=0):
    """A layer of garbage-free zeros, or of quantised normal rows; pad: extra slots between heads (a strided view)."""
    k = torch.zeros(n_kv, slots + pad, hd, device=DEV).to(torch.float8_e4m3fn)
    v, ks = k.clone(), torch.zeros(n_kv, slots + pad, dtype=torch.uint8, device=DEV)
    vs = ks.clone()
    if seed is not None:
        size = torch.exp2(rand(n_kv, slots + pad, 1, seed=seed + 2) * 2)
        (k, ks), (v, vs) = (quantise_ref(rand(n_kv, slots + pad, hd, seed=seed + i) * size) for i in (0, 1))
    return ops.KVLayerQ8(k[:, :slots], v[:, :slots], ks[:, :slots], vs[:, :slots])


def rotate_ref(x, cos, sin, pos, rot, interleaved):
    """Rotary embedding, products and sums rounded one by one in fp32 (x [T, n, hd] fp32)."""
    c, s = cos[pos.long()][:, None, :], sin[pos.long()][:, None, :]
    out = x.clone()
    first = torch.arange(rot // 2, device=DEV) * (2 if interleaved else 1)
    second = first + (1 if interleaved else rot // 2)
    a, b = x[..., first], x[..., second]
    out[..., first] = a * c - b * s
    out[..., second] = b * c + a * s
    return out


def tables(rot, max_pos):
    inv = 500000.0 ** (-torch.arange(0, rot, 2, dtype=torch.float64, device=DEV) / max(rot, 1))
    f = torch.arange(max_pos, dtype=torch.float64, device=DEV)[:, None] * inv
    return f.cos().float(), f.sin().float()


# (T, H, Hkv, hd, rot, interleaved): one token, odd counts, part of a head, halves that are no multiple of 8, no rotation
WRITES = [(1, 32, 8, 64, 64, False), (33, 32, 8, 128, 64, True), (7, 4, 2, 16, 12, False), (5, 3, 3, 48, 36, False),
          (130, 16, 1, 64, 48, True), (3, 8, 8, 80, 80, False), (2, 4, 4, 32, 0, False), (257, 64, 8, 128, 128, False),
          (4, 8, 2, 112, 112, True), (9, 8, 2, 96, 2, False)]


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("T,H,Hkv,hd,rot,inter", WRITES)
def test_write_rotates_quantises_and_reads_back(ops, ws, dtype, T, H, Hkv, hd, rot, inter):
    slots = T + 5
    layer = new_layer(ops, Hkv, slots, hd, seed=3, pad=3)
    before = [t.clone() for t in (layer.k.view(torch.uint8), layer.v.view(torch.uint8), layer.k_scale, layer.v_scale)]
    q, k, v = (rand(T, n * hd, dtype=dtype, seed=s) for n, s in ((H, 10), (Hkv, 11), (Hkv, 12)))
    k[0] *= 1e4
    v[-1] *= 1e-3
    cos, sin = tables(rot, 3000)
    pos = torch.randint(0, 3000, (T,), device=DEV, dtype=torch.int32)
    where = torch.randperm(slots, device=DEV)[:T].to(torch.int32)
    q_out = torch.empty_like(q)
    ops.rope_kv_write_q8(q, k, v, H, Hkv, hd, cos if rot else None, sin if rot else None, pos, where, layer, q_out, ws,
                         interleaved=inter)
    ws.check_status()
    turn = (lambda x, n: rotate_ref(x.float().view(T, n, hd), cos, sin, pos, rot, inter)) if rot else \
        (lambda x, n: x.float().view(T, n, hd))
    assert torch.equal(q_out, turn(q, H).reshape(T, -1).to(dtype))
    at = where.long()
    for x, codes, scale in ((turn(k, Hkv), layer.k, layer.k_scale), (v.float().view(T, Hkv, hd), layer.v, layer.v_scale)):
        c, s = quantise_ref(x)
        assert torch.equal(codes.view(torch.uint8)[:, at], c.view(torch.uint8).transpose(0, 1))
        assert torch.equal(scale[:, at], s.transpose(0, 1))
    left = torch.ones(slots, dtype=torch.bool, device=DEV)
    left[at] = False
    for old, new in zip(before, (layer.k.view(torch.uint8), layer.v.view(torch.uint8), layer.k_scale, layer.v_scale)):
        assert torch.equal(old[:, left], new[:, left])  # every other slot is as it was
    for out_dt in (BF, F32):
        ko, vo = (torch.empty(T, Hkv * hd, dtype=out_dt, device=DEV) for _ in range(2))
        ops.kv_read_q8(layer, where, ko, vo, ws)
        ws.check_status()
        assert torch.equal(ko.double().view(T, Hkv, hd), value(layer.k[:, at], layer.k_scale[:, at]).transpose(0, 1))
        assert torch.equal(vo.double().view(T, Hkv, hd), value(layer.v[:, at], layer.v_scale[:, at]).transpose(0, 1))


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("T,H,Hkv,hd,rot,inter", [(3, 8, 2, 128, 64, False), (600, 40, 40, 64, 24, False),
                                                  (2, 70, 33, 64, 64, False), (400, 3, 20, 128, 128, True),
                                                  (1, 1, 1, 16, 16, False), (150, 0, 37, 48, 32, False)])
def test_write_partial_rotation_and_many_heads(ops, ws, dtype, T, H, Hkv, hd, rot, inter):
    """Rotated parts that end inside a row, in vectors; more heads than a pass of
    rows, over one block a token and over several; no query rows (H = 0)."""
    layer = new_layer(ops, Hkv, T, hd)
    q, k, v = (rand(T, max(n, 1) * hd, dtype=dtype, seed=s) for n, s in ((H, 20), (Hkv, 21), (Hkv, 22)))
    cos, sin = tables(rot, 500)
    pos = torch.randint(0, 500, (T,), device=DEV, dtype=torch.int32)
    where = torch.randperm(T, device=DEV).to(torch.int32)
    q_out = torch.empty_like(q) if H else None
    ops.rope_kv_write_q8(q if H else None, k, v, H, Hkv, hd, cos, sin, pos, where, layer, q_out, ws, interleaved=inter)
    ws.check_status()
    if H:
        want = rotate_ref(q.float().view(T, H, hd), cos, sin, pos, rot, inter)
        assert torch.equal(q_out, want.reshape(T, -1).to(dtype))
    at = where.long()
    for x, codes, scale in ((rotate_ref(k.float().view(T, Hkv, hd), cos, sin, pos, rot, inter), layer.k, layer.k_scale),
                            (v.float().view(T, Hkv, hd), layer.v, layer.v_scale)):
        c, s = quantise_ref(x)
        assert torch.equal(codes.view(torch.uint8)[:, at], c.view(torch.uint8).transpose(0, 1))
        assert torch.equal(scale[:, at], s.transpose(0, 1))


def test_write_borders_of_the_scale(ops, ws):
    """Zero rows, subnormals, the largest values, amax at and next to 448 * 2^e, Inf and NaN."""
    hd = 64
    big = torch.finfo(F32).max
    tops = [0.0, 1e-45, 1e-38, 2.0**-32, 448.0, 448.0 * (1 + 2**-23), 447.9, 256.0, 1.0, 1.75, 1.75 * (1 + 2**-23), big,
            2.0**127, 3.0e-9]
    v = torch.zeros(len(tops) + 3, hd, device=DEV)
    for i, t in enumerate(tops):
        v[i] = torch.linspace(-1, 1, hd, device=DEV) * t
        v[i, 5] = t
    v[-3, 1], v[-3, 2], v[-3, 3] = math.inf, -math.inf, 2.5
    v[-2, 7], v[-2, 8] = math.nan, -3.25
    v[-1] = math.inf
    n = v.shape[0]
    layer = new_layer(ops, 1, n, hd)
    ops.rope_kv_write_q8(None, v, v, 1, 1, hd, None, None, None, torch.arange(n, device=DEV, dtype=torch.int32), layer,
                         None, ws)
    c, s = quantise_ref(v)
    assert torch.equal(layer.v_scale[0], s)
    got, want = layer.v[0].float(), c.float()
    assert torch.equal(torch.isnan(got), torch.isnan(want)) and torch.isnan(got).sum() == 1
    assert torch.equal(got.nan_to_num(0), want.nan_to_num(0))
    out = torch.empty(n, hd, dtype=BF, device=DEV)
    ops.kv_read_q8(layer, None, None, out, ws, first=0, n=n)
    ws.check_status()
    assert torch.isfinite(out).sum() == out.numel() - 1  # Inf is held as the row's largest value
    exact = v[: len(tops)].double()
    err = (out[: len(tops)].double() - exact).abs()
    # half a step of e4m3: 2^-4 of the value, or half a subnormal step 2^-10 of 2^e
    # (a value above 448 * 2^119, beyond the largest scale, saturates)
    assert (err <= exact.abs() * 2.0**-4 + two_to(s[: len(tops)].to(torch.int64) - 127)[:, None] * 2.0**-10)[
        exact.abs() <= 448 * 2.0**119].all()


def test_write_in_place_and_strided(ops, ws):
    """q_out = q, q / k / v as slices of one projection buffer, rows that are not 16-byte aligned."""
    T, H, Hkv, hd = 11, 8, 2, 64
    cos, sin = tables(hd, 100)
    pos = torch.arange(T, device=DEV, dtype=torch.int32)
    for dtype in (BF, F32):
        for lead in (0, 1):  # lead 1: every row starts off alignment
            width = (H + 2 * Hkv) * hd
            buf = rand(T, width + 1, dtype=dtype, seed=5)
            x = buf[:, lead:lead + width]
            q, k, v = x[:, :H * hd], x[:, H * hd:(H + Hkv) * hd], x[:, (H + Hkv) * hd:]
            want = rotate_ref(q.float().reshape(T, H, hd), cos, sin, pos, hd, False).reshape(T, -1).to(dtype)
            ck, sk = quantise_ref(rotate_ref(k.float().reshape(T, Hkv, hd), cos, sin, pos, hd, False))
            keep_k = k.clone()
            layer = new_layer(ops, Hkv, T, hd)
            ops.rope_kv_write_q8(q, k, v, H, Hkv, hd, cos, sin, pos, pos, layer, q, ws)
            ws.check_status()
            assert torch.equal(q, want) and torch.equal(k, keep_k)
            assert torch.equal(layer.k.view(torch.uint8), ck.view(torch.uint8).transpose(0, 1))
            out = torch.full((T, Hkv * hd + 3), 7.0, dtype=dtype, device=DEV)
            ops.kv_read_q8(layer, None, out[:, 1:1 + Hkv * hd], None, ws, n=T)
            assert torch.equal(out[:, 1:1 + Hkv * hd].double().reshape(T, Hkv, hd), value(ck, sk))
            assert (out[:, 0] == 7).all() and (out[:, -2:] == 7).all()


def test_bad_slots_and_positions_are_reported(ops, ws):
    T, hd = 4, 32
    layer = new_layer(ops, 1, 8, hd, seed=1)
    before = layer.k.view(torch.uint8).clone()
    x = rand(T, hd, seed=2)
    cos, sin = tables(hd, 10)
    i32 = dict(device=DEV, dtype=torch.int32)
    good, bad = torch.tensor([0, 1, 2, 3], **i32), torch.tensor([-1, 8, 2**30, -2**31], **i32)
    ops.rope_kv_write_q8(None, x, x, 1, 1, hd, cos, sin, good, bad, layer, None, ws)
    with pytest.raises(RuntimeError, match="out of range"):
        ws.check_status()
    assert torch.equal(layer.k.view(torch.uint8), before)
    ops.rope_kv_write_q8(None, x, x, 1, 1, hd, cos, sin, torch.tensor([0, 1, 10, -3], **i32), good, layer, None, ws)
    with pytest.raises(RuntimeError, match="out of range"):
        ws.check_status()
    out = torch.full((4, hd), 5.0, device=DEV)
    ops.kv_read_q8(layer, bad, out, None, ws)
    with pytest.raises(RuntimeError, match="out of range"):
        ws.check_status()
    assert (out == 0).all()
    ws.check_status()


# --------------------------------------------------------------- attention
def visible_ref(T, slots, plen, pstart=None, base=None, mask=None, bound=None):
    """bool [T, slots] from the arguments, slot by slot."""
    j = torch.arange(slots, device=DEV)
    see = j[None] < plen.long()[:, None]
    if pstart is not None:
        see &= j[None] >= pstart.long()[:, None]
    if mask is not None:
        for w in range(mask.shape[1]):
            for b in range(64):
                s = int(base) + 64 * w + b
                if 0 <= s < slots:
                    see[:, s] |= ((mask[:, w] >> b) & 1) == 1
    if bound:
        see &= j[None] < bound
    return see


def attention_ref(q, layer, H, see):
    """fp64 softmax attention over the cache's values; rows that see nothing give zeros."""
    T, hd, G = q.shape[0], layer.head_dim, H // layer.n_kv
    out = torch.zeros(T, H, hd, dtype=torch.float64, device=DEV)
    q = q.double().view(T, H, hd)
    some = see.any(0)
    for h in range(H):
        k = value(layer.k[h // G][some], layer.k_scale[h // G][some])
        v = value(layer.v[h // G][some], layer.v_scale[h // G][some])
        s = (q[:, h] @ k.T / math.sqrt(hd)).masked_fill(~see[:, some], -math.inf)
        out[:, h] = torch.softmax(s, -1).nan_to_num(0) @ v
    return out.reshape(T, H * hd)


def random_tree_mask(rows, words, seed):
    import random

    r = random.Random(seed)
    bits = [0]
    for i in range(rows - 1):
        bits.append(bits[r.randrange(len(bits))] | (1 << i))
    out = [[(b >> (64 * w)) & (2**64 - 1) for w in range(words)] for b in bits]
    return torch.tensor([[x - 2**64 if x >= 2**63 else x for x in row] for row in out], dtype=torch.int64, device=DEV)


def check(out, ref, layer, see, dtype):
    some = see.any(0)
    vmax = value(layer.v[:, some], layer.v_scale[:, some]).abs().max().item() if bool(some.any()) else 0.0
    tol = (2 * 2.0**-8 if dtype == BF else 2e-5) * vmax
    err = (out.double() - ref).abs().max().item()
    assert err <= tol, (err, tol)
    # on average far inside that bound: half a step of bf16 (2^-9) and of P, or fp32 sums
    rms = ref.pow(2).mean().sqrt().item()
    assert (out.double() - ref).pow(2).mean().sqrt().item() <= (2.0**-8 if dtype == BF else 1e-5) * max(rms, 2.0**-4 * vmax)


HEADS = [(32, 8, 128), (32, 8, 64), (8, 8, 128), (16, 1, 64), (4, 2, 16), (40, 1, 48), (64, 8, 128)]


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("H,Hkv,hd", HEADS)
@pytest.mark.parametrize("T,ctx", [(1, 1), (1, 700), (9, 63), (33, 1100), (25, 0), (65, 257), (130, 129)])
def test_attention_tree(ops, ws, dtype, H, Hkv, hd, T, ctx):
    """Root + tree rows over a prefix and the tree's own slots; lengths that end inside a block."""
    slots = ctx + T + 3
    layer = new_layer(ops, Hkv, slots, hd, seed=20, pad=1)
    q = rand(T, H * hd, dtype=dtype, scale=1.5, seed=23)
    words = (T - 1 + 63) // 64
    mask = random_tree_mask(T, words, T) if words else None
    base = torch.tensor([ctx], dtype=torch.int32, device=DEV)
    plen = torch.full((T,), ctx, dtype=torch.int32, device=DEV)
    out = torch.full((T, H * hd), math.nan, dtype=dtype, device=DEV)
    ops.tree_attention_q8(q, layer, H, Hkv, hd, plen, out, ws, spec_base=base if words else None, spec_mask=mask)
    ws.check_status()
    see = visible_ref(T, slots, plen, None, ctx, mask)
    check(out, attention_ref(q, layer, H, see), layer, see, dtype)
    if ctx == 0:
        assert (out[0] == 0).all()  # the root sees nothing


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("H,Hkv,hd", HEADS[:4])
@pytest.mark.parametrize("T,past", [(5, 0), (300, 0), (64, 500)])
def test_attention_causal(ops, ws, dtype, H, Hkv, hd, T, past):
    slots = past + T
    layer = new_layer(ops, Hkv, slots, hd, seed=30)
    q = rand(T, H * hd, dtype=dtype, scale=1.5, seed=33)
    plen = torch.arange(past + 1, past + T + 1, dtype=torch.int32, device=DEV)
    out = torch.empty_like(q)
    ops.tree_attention_q8(q, layer, H, Hkv, hd, plen, out, ws)
    ws.check_status()
    see = visible_ref(T, slots, plen)
    check(out, attention_ref(q, layer, H, see), layer, see, dtype)


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("H,Hkv,hd", HEADS[:4])
def test_attention_ranges_empty_rows_and_bounds(ops, ws, dtype, H, Hkv, hd):
    """Per-row slot ranges far apart, rows that see nothing, lengths beyond the
    cache, negative starts, a bound that cuts the range, mask bits before slot 0."""
    slots = 2000
    layer = new_layer(ops, Hkv, slots, hd, seed=40)
    i32 = dict(dtype=torch.int32, device=DEV)
    start = torch.tensor([0, 300, 1990, 700, 5, -7, 1999, 64, 128], **i32)
    plen = torch.tensor([0, 900, 1991, 700, 3, 1, 5000, 128, 129], **i32)
    T = start.numel()
    q = rand(T, H * hd, dtype=dtype, seed=41)
    for bound in (0, 1000):
        for base, bits in ((None, None), (1997, [1, 0, 2, 4, 0, 8, 0, 0, 3]), (-2, [1, 4, 2, 8, 0, 0, 0, 0, 16])):
            mask = None if bits is None else torch.tensor(bits, dtype=torch.int64, device=DEV)[:, None]
            out = torch.empty_like(q)
            ops.tree_attention_q8(q, layer, H, Hkv, hd, plen, out, ws, prefix_start=start, kv_bound=bound,
                                  spec_base=None if base is None else torch.tensor([base], **i32), spec_mask=mask)
            ws.check_status()
            see = visible_ref(T, slots, plen, start, base, mask, bound)
            check(out, attention_ref(q, layer, H, see), layer, see, dtype)
            assert (out[~see.any(1)] == 0).all()


@pytest.mark.parametrize("dtype", [BF, F32])
def test_attention_masked_garbage(ops, ws, dtype):
    """NaN codes and the largest scales in slots that no row sees change nothing."""
    H, Hkv, hd, T, slots = 8, 2, 64, 6, 700
    q = rand(T, H * hd, dtype=dtype, seed=50)
    plen = torch.tensor([300, 301, 302, 303, 304, 305], dtype=torch.int32, device=DEV)
    start = torch.full_like(plen, 70)
    outs = []
    for dirty in (False, True):
        layer = new_layer(ops, Hkv, slots, hd, seed=51)
        if dirty:
            for c, s in ((layer.k, layer.k_scale), (layer.v, layer.v_scale)):
                for lo, hi in ((0, 70), (305, slots)):
                    c.view(torch.uint8)[:, lo:hi] = 0x7f
                    s[:, lo:hi] = 246
        out = torch.empty_like(q)
        ops.tree_attention_q8(q, layer, H, Hkv, hd, plen, out, ws, prefix_start=start)
        outs.append(out)
    ws.check_status()
    assert torch.equal(outs[0], outs[1])


@pytest.mark.parametrize("dtype", [BF, F32])
def test_attention_extreme_values(ops, ws, dtype):
    """Rows of very different scales: a sink with a tiny value row, scores that
    rise along the slots (the running maximum keeps moving), large scores."""
    H, Hkv, hd, T, slots = 8, 2, 128, 3, 1500
    k, v = rand(Hkv, slots, hd, seed=60), rand(Hkv, slots, hd, seed=61)
    q = rand(T, H * hd, dtype=dtype, seed=62)
    k *= torch.linspace(0.1, 6, slots, device=DEV)[None, :, None]
    v[:, 0] *= 1e-9
    v[:, 700:] *= 40
    v[:, 3] = 0
    (kc, ks), (vc, vs) = quantise_ref(k), quantise_ref(v)
    layer = ops.KVLayerQ8(kc, vc, ks, vs)
    plen = torch.tensor([1500, 4, 1], dtype=torch.int32, device=DEV)
    out = torch.empty_like(q)
    ops.tree_attention_q8(q, layer, H, Hkv, hd, plen, out, ws)
    ws.check_status()
    see = visible_ref(T, slots, plen)
    ref = attention_ref(q, layer, H, see)
    for t in range(T):  # each row against its own largest value
        check(out[t:t + 1], ref[t:t + 1], layer, see[t:t + 1], dtype)


@pytest.mark.parametrize("T", [1, 9, 33, 300])
@pytest.mark.parametrize("hd", [64, 128])
def test_attention_weights_add_up_to_one(ops, ws, hd, T):
    """Values of one everywhere give exactly one: with scores close together every
    weight is held to 8 bits, and the sum that divides is that of the held ones
    (fp32 sums of 1000 terms are off by less than 2^-14, half a bf16 step below one
    is 2^-9)."""
    H, Hkv, slots = 16, 4, 1000
    k = rand(Hkv, slots, hd, seed=95, scale=0.25)
    v = torch.ones_like(k)
    (kc, ks), (vc, vs) = quantise_ref(k), quantise_ref(v)
    layer = ops.KVLayerQ8(kc, vc, ks, vs)
    q = rand(T, H * hd, dtype=BF, seed=96)
    plen = torch.randint(1, slots + 1, (T,), device=DEV, dtype=torch.int32)
    out = torch.zeros_like(q)
    ops.tree_attention_q8(q, layer, H, Hkv, hd, plen, out, ws)
    ws.check_status()
    assert (out == 1).all()


@pytest.mark.parametrize("slots,strong", [(4096, 10.0), (32768, 12.0)])
@pytest.mark.parametrize("hd", [64, 128])
def test_attention_sink_beside_a_flat_tail(ops, ws, hd, slots, strong):
    """One key with 5/6 of the weight, the rest spread evenly over thousands of
    keys 2^-14 .. 2^-17 below it: the even part must not get lost. As many rows
    as keep the keys of a head in one slice."""
    H, T = 8, 1300
    k = torch.zeros(H, slots, hd, device=DEV)
    k[:, :, 1] = torch.linspace(0.25, 0.4375, H, device=DEV)[:, None]  # away from whole exponents
    k[:, 77, 0] = strong
    v = torch.ones_like(k)
    v[:, 77] = -1
    (kc, ks), (vc, vs) = quantise_ref(k), quantise_ref(v)
    layer = ops.KVLayerQ8(kc, vc, ks, vs)
    q = torch.zeros(T, H, hd, device=DEV)
    q[:, :, :2] = math.sqrt(hd)
    q = q.to(BF).view(T, H * hd)
    plen = torch.full((T,), slots, dtype=torch.int32, device=DEV)
    out = torch.empty_like(q)
    ops.tree_attention_q8(q, layer, H, H, hd, plen, out, ws)
    ws.check_status()
    see = visible_ref(1, slots, plen[:1])
    ref = attention_ref(q[:1], layer, H, see)
    # all the rows are alike; the even keys hold (1 + ref) / 2 and are off by 2^-3 at most
    # (the nearest of 3 significant bits, all to the same side), the strong one by 2^-8, the result by 2^-9
    tol = (1 + ref.max().item()) / 2 * 2.0**-3 + 2.0**-8 + 2.0**-9
    err = (out.double() - ref).abs().max().item()
    assert err <= tol, (err, tol)


@pytest.mark.parametrize("dtype", [BF, F32])
def test_attention_long_and_wide(ops, ws, dtype):
    """A cache beyond 2^31 code bytes per head set: the last slots of the last head."""
    H, Hkv, hd, slots = 16, 8, 128, 2_200_000
    k = torch.zeros(Hkv, slots, hd, dtype=torch.uint8, device=DEV).view(torch.float8_e4m3fn)
    v = torch.zeros(Hkv, slots, hd, dtype=torch.uint8, device=DEV).view(torch.float8_e4m3fn)
    ks, vs = (torch.full((Hkv, slots), 127, dtype=torch.uint8, device=DEV) for _ in range(2))
    n = 333
    src = new_layer(ops, Hkv, n, hd, seed=70)
    k[:, -n:], v[:, -n:], ks[:, -n:], vs[:, -n:] = src.k, src.v, src.k_scale, src.v_scale
    layer = ops.KVLayerQ8(k, v, ks, vs)
    q = rand(2, H * hd, dtype=dtype, seed=71)
    i32 = dict(dtype=torch.int32, device=DEV)
    plen, start = torch.tensor([slots, slots - 1], **i32), torch.tensor([slots - n, slots - 5], **i32)
    out = torch.empty_like(q)
    ops.tree_attention_q8(q, layer, H, Hkv, hd, plen, out, ws, prefix_start=start)
    ws.check_status()
    see = visible_ref(2, n, plen - (slots - n), start - (slots - n))
    check(out, attention_ref(q, src, H, see), src, see, dtype)
    ko = torch.empty(n, Hkv * hd, dtype=BF, device=DEV)
    ops.kv_read_q8(layer, None, ko, None, ws, first=slots - n, n=n)
    assert torch.equal(ko.double().view(n, Hkv, hd), value(src.k, src.k_scale).transpose(0, 1))


def test_attention_q_strides_streams_and_graphs(ops):
    """q / out as strided slices; a side stream; one graph replayed on changed inputs; two workspaces at once."""
    H, Hkv, hd, T, slots = 8, 2, 64, 5, 900
    layer = new_layer(ops, Hkv, slots, hd, seed=80)
    plen = torch.tensor([900, 10, 500, 1, 64], dtype=torch.int32, device=DEV)
    see = visible_ref(T, slots, plen)
    wide = rand(T, H * hd + 40, dtype=BF, seed=81)
    q = wide[:, 8:8 + H * hd]
    res = torch.zeros(T, H * hd + 24, dtype=BF, device=DEV)
    out = res[:, 16:16 + H * hd]
    wss = [ops.Workspace(torch.device(DEV), max_rows=64, vocab=1) for _ in range(2)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    out2 = torch.empty_like(q).contiguous()
    with torch.cuda.stream(side):
        ops.tree_attention_q8(q, layer, H, Hkv, hd, plen, out, wss[0])
    ops.tree_attention_q8(q, layer, H, Hkv, hd, plen, out2, wss[1])
    torch.cuda.synchronize()
    check(out, attention_ref(q.contiguous(), layer, H, see), layer, see, BF)
    assert torch.equal(out, out2)
    assert (res[:, :16] == 0).all() and (res[:, 16 + H * hd:] == 0).all()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        ops.tree_attention_q8(q, layer, H, Hkv, hd, plen, out, wss[0])
    for seed in (82, 83):
        wide.copy_(rand(T, H * hd + 40, dtype=BF, seed=seed))
        plen.copy_(torch.tensor([5, 900, 3, 700, 0], dtype=torch.int32, device=DEV) if seed == 82 else plen.flip(0))
        g.replay()
        torch.cuda.synchronize()
        see = visible_ref(T, slots, plen)
        check(out, attention_ref(q.contiguous(), layer, H, see), layer, see, BF)
    for w in wss:
        w.check_status()


@pytest.mark.parametrize("dtype", [BF, F32])
def test_attention_two_graphs_share_a_workspace(ops, dtype):
    """One token (joined by the last slice) and many, captured over one workspace
    and replayed in turn; rows that start off alignment; the slices' counters end
    at zero."""
    H, Hkv, hd, slots = 32, 8, 128, 3000
    layer = new_layer(ops, Hkv, slots, hd, seed=90)
    ws = ops.Workspace(torch.device(DEV), max_rows=64, vocab=1)
    calls, graphs = [], []
    for T in (1, 33):
        wide = rand(T, H * hd + 3, dtype=dtype, seed=91)
        q, out = wide[:, 1:1 + H * hd], torch.zeros(T, H * hd + 1, dtype=dtype, device=DEV)[:, 1:]
        plen = torch.randint(1, slots + 1, (T,), device=DEV, dtype=torch.int32)
        calls.append((T, wide, q, plen, out))
    side = torch.cuda.Stream()
    for T, wide, q, plen, out in calls:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=side):
            ops.tree_attention_q8(q, layer, H, Hkv, hd, plen, out, ws)
        graphs.append(g)
    for turn in range(3):
        for (T, wide, q, plen, out), g in zip(calls, graphs):
            wide.copy_(rand(*wide.shape, dtype=dtype, seed=92 + turn))
            plen.copy_(torch.randint(0, slots + 1, (T,), device=DEV, dtype=torch.int32))
            g.replay()
        torch.cuda.synchronize()
        for T, wide, q, plen, out in calls:
            see = visible_ref(T, slots, plen)
            check(out, attention_ref(q.contiguous(), layer, H, see), layer, see, dtype)
    ws.check_status()


def test_attention_is_deterministic(ops, ws):
    H, Hkv, hd, T, slots = 32, 8, 128, 33, 4000
    layer = new_layer(ops, Hkv, slots, hd, seed=90)
    q = rand(T, H * hd, dtype=BF, seed=91)
    plen = torch.full((T,), 3990, dtype=torch.int32, device=DEV)
    outs = []
    for _ in range(5):
        out = torch.empty_like(q)
        ops.tree_attention_q8(q, layer, H, Hkv, hd, plen, out, ws)
        outs.append(out)
    assert all(torch.equal(o, outs[0]) for o in outs[1:])


# -------------------------------------------------------------- compaction
@pytest.mark.parametrize("hd,keep,start", [(128, [40, 43, 41, 50], 40), (64, [7], 3), (16, [9, 8, 5, 6, 7], 5), (48, [], 2)])
def test_compact_moves_codes_and_scales(ops, ws, hd, keep, start):
    Ln, Hkv, slots = 3, 2, 64
    x = torch.randint(0, 256, (Ln, 2, Hkv, slots, hd), dtype=torch.uint8, device=DEV)
    sc = torch.randint(0, 256, (Ln, 2, Hkv, slots), dtype=torch.uint8, device=DEV)
    codes = x.clone().view(torch.float8_e4m3fn)
    scales = sc.clone()
    i32 = dict(dtype=torch.int32, device=DEV)
    at = torch.tensor(keep + [0], **i32)
    ops.kv_compact_q8(codes, scales, torch.tensor([start], **i32), at, torch.tensor([len(keep)], **i32),
                      max(1, len(keep)), ws)
    ws.check_status()
    want, wants = x.clone(), sc.clone()
    if keep:
        want[:, :, :, start:start + len(keep)] = x[:, :, :, keep]
        wants[:, :, :, start:start + len(keep)] = sc[:, :, :, keep]
    assert torch.equal(codes.view(torch.uint8), want) and torch.equal(scales, wants)
    ops.kv_compact_q8(codes, scales, torch.tensor([start], **i32), torch.tensor([slots], **i32),
                      torch.tensor([1], **i32), 1, ws)
    with pytest.raises(RuntimeError, match="out of range"):
        ws.check_status()
    assert torch.equal(codes.view(torch.uint8), want)


def test_write_read_attend_compact_together(ops, ws):
    """One layer's round: prompt rows, a drafted tree, attention, the accepted
    path moved, the next root attending it: equal to a cache that was written
    with the path alone."""
    H, Hkv, hd, P, n = 8, 2, 64, 50, 6
    cos, sin = tables(hd, 200)
    i32 = dict(dtype=torch.int32, device=DEV)

    def cache():
        return (torch.zeros(1, 2, Hkv, 80, hd, device=DEV).to(torch.float8_e4m3fn),
                torch.zeros(1, 2, Hkv, 80, dtype=torch.uint8, device=DEV))

    def layer(c, s):
        return ops.KVLayerQ8(c[0, 0], c[0, 1], s[0, 0], s[0, 1])

    def put(lay, pos, slots, seed):
        T = len(pos)
        q, k, v = (rand(T, m * hd, dtype=BF, seed=seed + j) for j, m in enumerate((H, Hkv, Hkv)))
        ops.rope_kv_write_q8(q, k, v, H, Hkv, hd, cos, sin, torch.tensor(pos, **i32), torch.tensor(slots, **i32), lay, q, ws)
        return q

    a, b = cache(), cache()
    for c in (a, b):
        put(layer(*c), list(range(P)), list(range(P)), 100)
    put(layer(*a), [P + d for d in (0, 1, 1, 2, 2, 3)], list(range(P, P + n)), 200)  # the tree
    keep = [P, P + 2, P + 4, P + 5]
    T, (q, k, v) = n, tuple(rand(n, m * hd, dtype=BF, seed=200 + j) for j, m in enumerate((H, Hkv, Hkv)))
    rows = torch.tensor([i - P for i in keep], device=DEV)
    kk, vv, qq = k[rows].contiguous(), v[rows].contiguous(), q[rows].contiguous()
    ops.rope_kv_write_q8(qq, kk, vv, H, Hkv, hd, cos, sin, torch.tensor([P, P + 1, P + 2, P + 3], **i32),
                         torch.arange(P, P + 4, **i32), layer(*b), qq, ws)
    ops.kv_compact_q8(a[0], a[1], torch.tensor([P], **i32), torch.tensor(keep, **i32), torch.tensor([4], **i32), 4, ws)
    ql = put(layer(*a), [P + 4], [P + 4], 300)
    qr = put(layer(*b), [P + 4], [P + 4], 300)
    assert torch.equal(ql, qr)
    outs = []
    for c, q1 in ((a, ql), (b, qr)):
        out = torch.empty_like(q1)
        ops.tree_attention_q8(q1, layer(*c), H, Hkv, hd, torch.tensor([P + 5], **i32), out, ws)
        outs.append(out)
        ko = torch.empty(P + 5, Hkv * hd, dtype=BF, device=DEV)
        ops.kv_read_q8(layer(*c), None, ko, None, ws, n=P + 5)
        outs.append(ko)
    ws.check_status()
    assert torch.equal(outs[0], outs[2]) and torch.equal(outs[1], outs[3])


# --------------------------------------------------------------- refusals
def test_wrappers_refuse_wrong_tensors(ops, ws):
    H, Hkv, hd, T = 4, 2, 32, 3
    layer = new_layer(ops, Hkv, 8, hd, seed=1)
    i32 = dict(dtype=torch.int32, device=DEV)
    q, k = rand(T, H * hd, dtype=BF), rand(T, Hkv * hd, dtype=BF)
    cos, sin = tables(hd, 10)
    pos = torch.arange(T, **i32)
    good = dict(q=q, k=k, v=k.clone(), n_heads=H, n_kv=Hkv, head_dim=hd, cos=cos, sin=sin, positions=pos, slots=pos,
                layer=layer, q_out=q.clone(), ws=ws)
    ops.rope_kv_write_q8(**good)
    for bad in (dict(k=k.float()), dict(k=k.cpu()), dict(k=k[:, :-1]), dict(k=k.t().contiguous().t()), dict(n_kv=1),
                dict(head_dim=64), dict(cos=cos.double()), dict(cos=cos[:, :8]), dict(rot_dim=16), dict(cos=None, rot_dim=32),
                dict(positions=pos.long()), dict(positions=None), dict(slots=pos[:2]), dict(q_out=None), dict(sin=sin[:5]),
                dict(q_out=q.float()), dict(slots=torch.arange(2 * T, **i32)[::2])):
        with pytest.raises(ValueError):
            ops.rope_kv_write_q8(**{**good, **bad})
    out = torch.empty_like(k)
    for args, kw in (((layer, pos, None, None), {}), ((layer, pos, out.half(), None), {}), ((layer, pos, out, out.float()), {}),
                     ((layer, pos.long(), out, None), {}), ((layer, None, out, None), dict(first=6)),
                     ((layer, pos, out[:2], None), {}), ((layer, pos, out[:, :4], None), {})):
        with pytest.raises(ValueError):
            ops.kv_read_q8(*args, ws, **kw)
    att = dict(q=q, layer=layer, n_heads=H, n_kv=Hkv, head_dim=hd, prefix_len=pos, out=q.clone(), ws=ws)
    ops.tree_attention_q8(**att)
    mask = torch.zeros(T, 1, dtype=torch.int64, device=DEV)
    for bad in (dict(q=q.float()), dict(out=q.float()), dict(q=q.half(), out=q.half()), dict(n_heads=8), dict(n_kv=4),
                dict(prefix_len=pos[:1]), dict(prefix_len=pos.long()), dict(spec_mask=mask), dict(out=q[:2].clone()),
                dict(spec_mask=mask[:1], spec_base=pos), dict(spec_mask=mask.int(), spec_base=pos),
                dict(spec_mask=torch.zeros(T, 5, dtype=torch.int64, device=DEV), spec_base=pos),
                dict(prefix_start=pos.cpu())):
        with pytest.raises(ValueError):
            ops.tree_attention_q8(**{**att, **bad})
    ws.check_status()
