"""Measured cases of the 8-bit key/value cache: rotating and quantising rows as they
are written, reading rows back, and tree attention over the quantised cache.

A cache row (one token, one KV head) is `head_dim` e4m3 codes and one scale byte: the
exponent e + 127 of a power of two, the smallest e with amax <= 448 * 2^e (amax over the
finite elements, e limited to -40 .. 119). Element i stands for code[i] * 2^e.

`run` computes each operator in plain torch operations, or through the framework's entry
points where `own` is true. Both use the same state.
"""

import math
import os
import random
import sys

import torch

own = False

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
PACKAGE = os.path.join(ROOT, "subnetwork-speculative-decoding_b200")

E_MIN, E_MAX = -40, 119
DTYPES = {"bf16": torch.bfloat16, "fp32": torch.float32}


# ------------------------------------------------------------------- cases
def _heads(model: str) -> dict:
    """Head layouts of the repository's configurations (ssd/synthetic.py) and its tests."""
    return {
        "1b": dict(heads=32, kv_heads=8, head_dim=64),
        "8b": dict(heads=32, kv_heads=8, head_dim=128),
        "70b": dict(heads=64, kv_heads=8, head_dim=128),
        "mha": dict(heads=8, kv_heads=8, head_dim=128),
        "mqa": dict(heads=16, kv_heads=1, head_dim=64),
        "tiny": dict(heads=4, kv_heads=2, head_dim=16),
    }[model]


def listed():
    return [
        # one token of a draft or target step of the 1B shape: latency only
        dict(name="write_decode_1b", op="write", rows=1, cap=896, rot=64, interleaved=False, dtype="bf16", **_heads("1b")),
        # root + tree of a verify forward; half of each head rotated, pairs interleaved
        dict(name="write_verify_8b_partial", op="write", rows=33, cap=2432, rot=64, interleaved=True, dtype="bf16",
             **_heads("8b")),
        # the prompt of the 70B configuration
        dict(name="write_prefill_70b", op="write", rows=4096, cap=4352, rot=128, interleaved=False, dtype="bf16",
             **_heads("70b")),
        # the rows of one accepted tree, moved out of the cache
        dict(name="read_tree_8b", op="read", rows=33, cap=2432, dtype="bf16", **_heads("8b")),
        # a whole long context read back, as when a sequence leaves the 8-bit cache
        dict(name="read_context_8b", op="read", rows=32768, cap=32896, dtype="bf16", **_heads("8b")),
        # target-only decoding step after a 2k prompt
        dict(name="attn_decode_8b_2k", op="attn", kind="causal", rows=1, ctx=2048, cap=2432, dtype="bf16", **_heads("8b")),
        # the verify forward of the 8B configuration: root + 32 nodes
        dict(name="attn_verify_8b_2k", op="attn", kind="tree", rows=33, ctx=2176, cap=2432, dtype="bf16", **_heads("8b")),
        # verify forwards at the longest context of the attention sweep, 8- and 64-node trees
        dict(name="attn_verify_8b_32k_9", op="attn", kind="tree", rows=9, ctx=32768, cap=32896, dtype="bf16", **_heads("8b")),
        dict(name="attn_verify_8b_32k_65", op="attn", kind="tree", rows=65, ctx=32768, cap=32896, dtype="bf16",
             **_heads("8b")),
        # prefill of a 2k prompt
        dict(name="attn_prefill_8b_2k", op="attn", kind="causal", rows=2048, ctx=0, cap=2432, dtype="bf16", **_heads("8b")),
        # batched decoding: 8 sequences of different lengths, each in its own slot range
        dict(name="attn_batch8_1b", op="attn", kind="batch", rows=8, ctx=3500, cap=8 * 4096, dtype="bf16", **_heads("1b")),
        # the fp32 tier's draft level after a 128-token prompt
        dict(name="attn_fp32_1b", op="attn", kind="tree", rows=5, ctx=160, cap=256, dtype="fp32", **_heads("1b")),
    ]


def _log(rng: random.Random, lo: int, hi: int) -> int:
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["write", "write", "read", "attn", "attn", "attn", "attn"])
    heads = _heads(rng.choice(["1b", "8b", "8b", "70b", "mha", "mqa", "tiny"]))
    hd = heads["head_dim"]
    if op == "write":
        rows = _log(rng, 1, 3900)
        return dict(op=op, rows=rows, cap=rows + rng.randint(1, 700), rot=rng.choice([hd, hd, hd // 2, hd // 4 * 3]),
                    interleaved=rng.random() < 0.5, dtype=rng.choice(["bf16", "bf16", "fp32"]), **heads)
    if op == "read":
        rows = _log(rng, 1, 16000)
        return dict(op=op, rows=rows, cap=rows + rng.randint(1, 700), dtype=rng.choice(["bf16", "bf16", "fp32"]), **heads)
    kind = rng.choice(["tree", "tree", "tree", "causal", "batch"])
    dtype = "fp32" if hd == 16 or rng.random() < 0.15 else "bf16"
    if kind == "tree":
        rows = _log(rng, 2, 65 if dtype == "fp32" else 200)
        ctx = _log(rng, 1, 900 if dtype == "fp32" else 16000 * 65 // max(65, rows))
        return dict(op=op, kind=kind, rows=rows, ctx=ctx, cap=ctx + rows + rng.randint(0, 300), dtype=dtype, **heads)
    if kind == "causal":
        rows = _log(rng, 1, 60 if dtype == "fp32" else 700)
        ctx = rng.choice([0, _log(rng, 1, 1000)])
        return dict(op=op, kind=kind, rows=rows, ctx=ctx, cap=ctx + rows + rng.randint(0, 300), dtype=dtype, **heads)
    rows = rng.randint(2, 24)
    ctx = _log(rng, 20, 60 if dtype == "fp32" else 1500)
    return dict(op=op, kind=kind, rows=rows, ctx=ctx, cap=rows * (ctx + rng.randint(1, 200)), dtype=dtype, **heads)


# ------------------------------------------------------------------ inputs
def _codes(shape, g, dev):
    """Rows as a cache holds them: normal values with a few strong channels, one scale a row."""
    x = torch.randn(*shape, generator=g, device=dev)
    strong = 1.0 + 3.0 * (torch.rand(shape[0], 1, shape[2], generator=g, device=dev) < 0.05)
    size = torch.exp2(torch.randn(shape[0], shape[1], 1, generator=g, device=dev))
    return _quantise(x * strong * size)


def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(seed)
    pick = random.Random(seed)
    H, Hkv, hd, rows, cap = case["heads"], case["kv_heads"], case["head_dim"], case["rows"], case["cap"]
    dt = DTYPES[case["dtype"]]
    s = dict(case=dict(case))
    i32 = dict(dtype=torch.int32, device=dev)
    if case["op"] == "write":
        s["kc"], s["ks"] = torch.zeros(Hkv, cap, hd, device=dev).to(torch.float8_e4m3fn), torch.zeros(Hkv, cap, dtype=torch.uint8, device=dev)
        s["vc"], s["vs"] = s["kc"].clone(), s["ks"].clone()
        for name, n in (("q", H), ("k", Hkv), ("v", Hkv)):
            s[name] = torch.randn(rows, n * hd, generator=g, device=dev).to(dt)
        far = 131072  # positions of a long context, with the frequencies scaled down by 8 beyond their first turns
        inv = 500000.0 ** (-torch.arange(0, case["rot"], 2, dtype=torch.float64, device=dev) / case["rot"])
        turns = 8192 * inv / (2 * math.pi)
        inv = torch.where(turns > 4, inv, torch.where(turns < 1, inv / 8, inv / 8 + (inv - inv / 8) * (turns - 1) / 3))
        table = torch.arange(far, dtype=torch.float64, device=dev)[:, None] * inv
        s["cos"], s["sin"] = table.cos().float(), table.sin().float()
        base = pick.randrange(far - rows)
        s["positions"] = torch.arange(base, base + rows, **i32)
        s["slots"] = torch.randperm(cap, generator=g, device=dev)[:rows].to(torch.int32)
        s["q_out"] = torch.empty(rows, H * hd, dtype=dt, device=dev)
        s["k_out"] = torch.empty(rows, Hkv * hd, dtype=torch.bfloat16, device=dev)
        s["v_out"] = torch.empty_like(s["k_out"])
        return s
    s["kc"], s["ks"] = _codes((Hkv, cap, hd), g, dev)
    s["vc"], s["vs"] = _codes((Hkv, cap, hd), g, dev)
    if case["op"] == "read":
        s["slots"] = torch.randperm(cap, generator=g, device=dev)[:rows].to(torch.int32)
        s["k_out"] = torch.empty(rows, Hkv * hd, dtype=dt, device=dev)
        s["v_out"] = torch.empty_like(s["k_out"])
        return s
    s["q"] = (1.5 * torch.randn(rows, H * hd, generator=g, device=dev)).to(dt)
    s["out"] = torch.empty(rows, H * hd, dtype=dt, device=dev)
    s["start"] = s["base"] = s["mask"] = None
    ctx = case["ctx"]
    if case["kind"] == "causal":
        s["len"] = torch.arange(ctx + 1, ctx + rows + 1, **i32)
    elif case["kind"] == "batch":
        region = cap // rows
        lens = [pick.randint(max(1, ctx // 4), min(ctx, region)) for _ in range(rows)]
        s["start"] = torch.tensor([b * region for b in range(rows)], **i32)
        s["len"] = s["start"] + torch.tensor(lens, **i32)
    else:
        # a random tree of rows - 1 nodes, at most 6 deep: each node sees itself and its ancestors
        words, bits, depth = (rows - 1 + 63) // 64, [0], [0]
        for i in range(rows - 1):
            above = pick.choice([r for r in range(i + 1) if depth[r] < 6])
            bits.append(bits[above] | (1 << i))
            depth.append(depth[above] + 1)
        signed = [[(b >> (64 * w)) & (2**64 - 1) for w in range(words)] for b in bits]
        s["mask"] = torch.tensor([[x - 2**64 if x >= 2**63 else x for x in r] for r in signed], dtype=torch.int64, device=dev)
        s["base"] = torch.tensor([ctx], **i32)
        s["len"] = torch.full((rows,), ctx, **i32)
    return s


# ------------------------------------------------------------- plain forms
def _quantise(x):
    """fp32 rows [..., hd] -> (e4m3 codes, scale bytes [...])."""
    amax = torch.where(torch.isfinite(x), x, 0).abs().amax(-1)
    mant, exp = torch.frexp(amax)  # amax = mant * 2^exp, mant in [0.5, 1)
    e = torch.where(mant > 0.875, exp - 8, exp - 9)  # 448 = 0.875 * 2^9
    e = torch.where(amax == 0, E_MIN, e.clamp(E_MIN, E_MAX))
    y = (x * _power(-e).unsqueeze(-1)).clamp(-448, 448)
    return y.to(torch.float8_e4m3fn), (e + 127).to(torch.uint8)


def _power(e):
    """2^e in fp32 for whole e in -126 .. 127: the exponent's bits."""
    return ((e.to(torch.int32) + 127) << 23).view(torch.float32)


def _value(codes, scale):
    return codes.float() * _power(scale.to(torch.int32) - 127).unsqueeze(-1)


def _rotate(x, cos, sin, rot, interleaved):
    """Rotary positions on the first `rot` elements of each head; x [T, n, hd], cos / sin [T, rot / 2]."""
    c, s = cos.unsqueeze(1), sin.unsqueeze(1)
    head, rest = x[..., :rot], x[..., rot:]
    a, b = (head[..., 0::2], head[..., 1::2]) if interleaved else (head[..., : rot // 2], head[..., rot // 2:])
    ra, rb = a * c - b * s, b * c + a * s
    turned = torch.stack([ra, rb], -1).flatten(-2) if interleaved else torch.cat([ra, rb], -1)
    return torch.cat([turned, rest], -1)


def _put(x, at, codes, scales):
    """Quantise rows x [T, n, hd] into the slots `at` of one cache."""
    c, e = _quantise(x)
    codes.view(torch.uint8)[:, at] = c.view(torch.uint8).transpose(0, 1)
    scales[:, at] = e.transpose(0, 1)


def _read(s, slots, dtype):
    at = slots.long()
    return [_value(c[:, at], e[:, at]).transpose(0, 1).reshape(len(at), -1).to(dtype) for c, e in ((s["kc"], s["ks"]), (s["vc"], s["vs"]))]


def _visible(s, cap, dev):
    """bool [rows, cap]: the slots that each row attends."""
    slot = torch.arange(cap, device=dev)
    see = slot < s["len"].long()[:, None]
    if s["start"] is not None:
        see &= slot >= s["start"].long()[:, None]
    if s["mask"] is not None:
        bit = slot - s["base"].long()
        inside = (bit >= 0) & (bit < 64 * s["mask"].shape[1])
        bit = bit.clamp(0, 64 * s["mask"].shape[1] - 1)
        see |= inside & (((s["mask"][:, bit // 64] >> (bit % 64)) & 1) == 1)
    return see


def _plain(s):
    case = s["case"]
    H, Hkv, hd, rows, cap = case["heads"], case["kv_heads"], case["head_dim"], case["rows"], case["cap"]
    if case["op"] == "write":
        pos, at = s["positions"].long(), s["slots"].long()
        turn = (s["cos"][pos], s["sin"][pos], case["rot"], case["interleaved"])
        q = _rotate(s["q"].float().view(rows, H, hd), *turn).reshape(rows, H * hd).to(s["q"].dtype)
        _put(_rotate(s["k"].float().view(rows, Hkv, hd), *turn), at, s["kc"], s["ks"])
        _put(s["v"].float().view(rows, Hkv, hd), at, s["vc"], s["vs"])
        return [q, *_read(s, s["slots"], torch.bfloat16)]
    if case["op"] == "read":
        return _read(s, s["slots"], s["k_out"].dtype)
    G = H // Hkv
    q = s["q"].float().view(rows, Hkv, G, hd).permute(1, 2, 0, 3).reshape(Hkv, G * rows, hd)
    k, v = _value(s["kc"], s["ks"]), _value(s["vc"], s["vs"])
    score = (q @ k.transpose(1, 2)).view(Hkv, G, rows, cap) / math.sqrt(hd)
    see = _visible(s, cap, q.device)
    score = torch.where(see, score, -math.inf)
    top = score.amax(-1, keepdim=True)
    p = torch.exp(score - torch.where(top == -math.inf, 0, top))
    total = p.sum(-1, keepdim=True)
    out = (p.view(Hkv, G * rows, cap) @ v).view(Hkv, G, rows, hd) / torch.where(total == 0, 1, total)
    return out.permute(2, 0, 1, 3).reshape(rows, H * hd).to(s["q"].dtype)


# ------------------------------------------------------ the framework's calls
_workspace = None


def _framework():
    """(ssd.ops, the program's workspace, kept between calls as an engine keeps it)."""
    global _workspace
    if PACKAGE not in sys.path:
        sys.path.insert(0, PACKAGE)
    from ssd import ops

    if _workspace is None:
        _workspace = ops.Workspace(torch.device("cuda"), max_rows=2048, vocab=1, max_head_rows=1)
    return ops, _workspace


def _own(s):
    case = s["case"]
    ops, ws = _framework()
    H, Hkv, hd = case["heads"], case["kv_heads"], case["head_dim"]
    layer = ops.KVLayerQ8(s["kc"], s["vc"], s["ks"], s["vs"])
    if case["op"] == "write":
        ops.rope_kv_write_q8(s["q"], s["k"], s["v"], H, Hkv, hd, s["cos"], s["sin"], s["positions"], s["slots"], layer,
                             s["q_out"], ws, rot_dim=case["rot"], interleaved=case["interleaved"])
        ops.kv_read_q8(layer, s["slots"], s["k_out"], s["v_out"], ws)
        return [s["q_out"], s["k_out"], s["v_out"]]
    if case["op"] == "read":
        ops.kv_read_q8(layer, s["slots"], s["k_out"], s["v_out"], ws)
        return [s["k_out"], s["v_out"]]
    ops.tree_attention_q8(s["q"], layer, H, Hkv, hd, s["len"], s["out"], ws, spec_base=s["base"], spec_mask=s["mask"],
                          prefix_start=s["start"], kv_bound=case["cap"])
    return s["out"]


def run(state):
    if own:
        return _own(state)
    return _plain(state)


# -------------------------------------------------------------------- work
def _pairs(case):
    """(keys that some row attends, visible (row, key) pairs), from the case alone."""
    rows, ctx = case["rows"], case["ctx"]
    if case["kind"] == "causal":
        return ctx + rows, rows * ctx + rows * (rows + 1) // 2
    if case["kind"] == "batch":
        mean = (max(1, ctx // 4) + min(ctx, case["cap"] // rows)) // 2
        return rows * mean, rows * mean
    return ctx + rows - 1, rows * ctx + 3 * (rows - 1)


def work(case):
    H, Hkv, hd, rows = case["heads"], case["kv_heads"], case["head_dim"], case["rows"]
    size = DTYPES[case["dtype"]].itemsize
    row = 2 * Hkv * (hd + 1)  # codes and scale bytes of one token's keys and values
    if case["op"] == "write":
        moved = rows * (2 * H * hd * size + 2 * Hkv * hd * size + row + case["rot"] * 4 + 8)
        return {"bytes": moved + rows * 2 * Hkv * hd * 2, "flops": rows * (H + Hkv) * case["rot"] * 3 + rows * 2 * Hkv * hd * 3}
    if case["op"] == "read":
        return {"bytes": rows * (row + 2 * Hkv * hd * size + 4), "flops": rows * 2 * Hkv * hd}
    keys, pairs = _pairs(case)
    return {"bytes": keys * row + 2 * rows * H * hd * size, "flops": 4 * pairs * H * hd}


# ------------------------------------------------------ the definition in 64 bits
def _two(e):
    """2^e in 64 bits for whole e, without a rounding of pow()."""
    return ((e.to(torch.int64) + 1023) << 52).view(torch.float64)


def _exact_rows(x):
    """The value that each element of the rows x (64 bits) is held as."""
    mag = torch.where(torch.isfinite(x), x, torch.zeros_like(x)).abs()
    need = mag.max(-1, keepdim=True).values / 448.0
    e = torch.ceil(torch.log2(need.clamp(min=2.0**-60))).clamp(E_MIN, E_MAX)
    e = torch.where(need > _two(e), e + 1, torch.where(need <= _two(e - 1), e - 1, e)).clamp(E_MIN, E_MAX)
    unit = _two(e)
    y = (x / unit).clamp(-448.0, 448.0)
    step = _two(torch.floor(torch.log2(y.abs().clamp(min=2.0**-6))) - 3)  # 3 bits behind the point, subnormals below 2^-6
    return torch.round(y / step) * step * unit


def exact(case, seed):
    s = prepare(case, seed)
    H, Hkv, hd, rows, cap = case["heads"], case["kv_heads"], case["head_dim"], case["rows"], case["cap"]
    if case["op"] == "write":
        rot, half = case["rot"], case["rot"] // 2
        pos = s["positions"].long()
        c, si = s["cos"].double()[pos], s["sin"].double()[pos]

        def turned(x, n):
            z = x.double().view(rows, n, hd).clone()
            first = torch.arange(half, device=z.device) * 2 if case["interleaved"] else torch.arange(half, device=z.device)
            second = first + (1 if case["interleaved"] else half)
            z0, z1 = z[:, :, first].clone(), z[:, :, second].clone()
            z[:, :, first] = z0 * c[:, None] - z1 * si[:, None]
            z[:, :, second] = z0 * si[:, None] + z1 * c[:, None]
            return z

        k = _exact_rows(turned(s["k"], Hkv))
        v = _exact_rows(s["v"].double().view(rows, Hkv, hd))
        return [turned(s["q"], H).reshape(rows, -1), k.reshape(rows, -1), v.reshape(rows, -1)]

    def held(codes, scale):
        return codes.double() * _two(scale.double() - 127.0)[..., None]

    if case["op"] == "read":
        at = s["slots"].long()
        return [held(c[:, at], e[:, at]).permute(1, 0, 2).reshape(rows, -1) for c, e in ((s["kc"], s["ks"]), (s["vc"], s["vs"]))]
    q = s["q"].double().view(rows, H, hd)
    out = torch.zeros(rows, H, hd, dtype=torch.float64, device=q.device)
    see = torch.zeros(rows, cap, dtype=torch.bool, device=q.device)
    lens = s["len"].tolist()
    starts = s["start"].tolist() if s["start"] is not None else [0] * rows
    for t in range(rows):
        see[t, starts[t]:lens[t]] = True
    if s["mask"] is not None:
        base, words = int(s["base"]), s["mask"].tolist()
        for t in range(rows):
            for w, bits in enumerate(words[t]):
                for b in range(64):
                    if (bits >> b) & 1 and base + 64 * w + b < cap:
                        see[t, base + 64 * w + b] = True
    for h in range(H):
        kv = h // (H // Hkv)
        k, v = held(s["kc"][kv], s["ks"][kv]), held(s["vc"][kv], s["vs"][kv])
        p = torch.softmax((q[:, h] @ k.T / math.sqrt(hd)).masked_fill(~see, -math.inf), -1)
        out[:, h] = torch.nan_to_num(p) @ v
    return out.reshape(rows, H * hd)
