"""Inputs of tree attention over the 8-bit key/value cache in which every key counts,
their 64-bit result and the bound that separates right from nearly right.

Scores lie close together, so that no key hides behind a strong one, and the value
row of a slot is 1 in a single channel (another for each slot and head): an output
channel is the summed weight of the few slots that share it, all of one sign. One
slot too many or too few moves a channel by 1/40 of it or more; the kernels' errors
are relative to it:
 * bf16: 1.25 2^-10 for the weights and 2^-8, half a step, for the result's
   rounding: 0.0051, below 1.5 * 2^-8;
 * fp32: scores of up to 128 products (2^-17 relative for |s| <= 3) and sums of n
   <= 2^15 weights (n 2^-24 at most): below 2^-8.5, and on average far below.
"""

import math
import random

import torch

TOL = 1.5 * 2.0**-8
PER_CHANNEL = 40  # slots that share a channel, at most


def _tree(rows, seed):
    """Ancestor bits of rows - 1 nodes below a root, rows x words of 64."""
    r = random.Random(seed)
    bits = [0]
    for i in range(rows - 1):
        bits.append(bits[r.randrange(len(bits))] | (1 << i))
    words = (rows - 2) // 64 + 1
    out = [[(b >> (64 * w)) & (2**64 - 1) for w in range(words)] for b in bits]
    return [[x - 2**64 if x >= 2**63 else x for x in row] for row in out]


def case(kind, H, Hkv, hd, T, ctx, dev, seed=1):
    """Arguments of one call: dict with q (fp32), codes and scale bytes, lengths, mask."""
    g = torch.Generator().manual_seed(seed * 1000 + T * 10 + ctx)
    i32 = dict(dtype=torch.int32)
    c = dict(H=H, Hkv=Hkv, hd=hd, T=T, start=None, base=None, mask=None, bound=0)
    if kind == "tree":
        slots = ctx + T + 3
        c["len"] = torch.full((T,), ctx, **i32)
        if T > 1:
            c["base"], c["mask"] = ctx, torch.tensor(_tree(T, T + ctx), dtype=torch.int64)
    elif kind == "causal":
        slots = ctx + T
        c["len"] = torch.arange(ctx + 1, ctx + T + 1, **i32)
    else:  # ranges of many sequences, a bound, mask bits beside and inside the ranges
        slots, c["bound"], c["base"] = ctx, ctx - 5, ctx // 2
        edges = [int(x) for x in torch.randint(0, ctx, (2 * T,), generator=g)]
        edges[:6] = [0, 128, 127, 257, ctx - 1, ctx + 9]
        c["start"] = torch.tensor([min(edges[2 * t:2 * t + 2]) for t in range(T)], **i32)
        c["len"] = torch.tensor([max(edges[2 * t:2 * t + 2]) for t in range(T)], **i32)
        c["len"][3 % T] = c["start"][3 % T]  # a row without a range
        c["mask"] = torch.randint(0, 1 << 40, (T, 2), generator=g) & 0x1111_0101_1001
    c["slots"] = slots
    c["q"] = torch.randn(T, H * hd, generator=g)
    k = 0.3 * torch.randn(Hkv, slots, hd, generator=g)
    # slots that carry a value: all, or those next to multiples of 64 and to the rows' edges, thinned out
    j = torch.arange(slots)
    carries = torch.ones(slots, dtype=torch.bool)
    if slots > PER_CHANNEL * hd:
        near = torch.zeros(slots + 8, dtype=torch.bool)
        edges = c["len"].long() if c["start"] is None else torch.cat([c["len"].long(), c["start"].long()])
        for e in edges.clamp(0, slots).tolist():
            near[max(e - 2, 0):e + 2] = True
        if c["base"] is not None:
            near[c["base"]:c["base"] + 64 * c["mask"].shape[1]] = True
        near = near[:slots]
        step = 64 * max(1, 4 * slots // 64 // (PER_CHANNEL * hd - int(near.sum())) + 1)
        carries = near | ((j + 2) % step < 4)
    rank = carries.cumsum(0) - 1
    v = torch.zeros(Hkv, slots, hd)
    for h in range(Hkv):
        v[h, j[carries], (7 * rank[carries] + 13 * h) % hd] = 1.0
    c["carries"] = carries
    c["k"], c["ks"] = _rows(k)
    c["v"], c["vs"] = _rows(v)
    for name, x in c.items():
        if isinstance(x, torch.Tensor):
            c[name] = x.to(dev)
    return c


def _rows(x):
    """fp32 rows -> (e4m3 codes, scale bytes): a power of two that keeps amax <= 448."""
    amax = x.abs().amax(-1)
    e = torch.ceil(torch.log2(amax.clamp(min=2.0**-30) / 448)).clamp(-40, 119)
    return (x * torch.exp2(-e)[..., None]).to(torch.float8_e4m3fn), (e + 127).to(torch.uint8)


def values(codes, scales):
    return codes.double() * torch.exp2(scales.double() - 127)[..., None]


def visible(c):
    """bool [T, slots], from the arguments slot by slot."""
    j = torch.arange(c["slots"], device=c["q"].device)
    see = j[None] < c["len"].long()[:, None]
    if c["start"] is not None:
        see &= j[None] >= c["start"].long()[:, None]
    if c["mask"] is not None:
        bit = j - c["base"]
        n = 64 * c["mask"].shape[1]
        at = bit.clamp(0, n - 1)
        see |= (bit >= 0) & (bit < n) & (((c["mask"][:, at // 64] >> (at % 64)) & 1) == 1)
    if c["bound"]:
        see &= j[None] < c["bound"]
    return see


def attention(c, q, see, rows=None, heads=None):
    """64-bit result [rows, heads, hd]; rows that see nothing give zeros."""
    H, Hkv, hd = c["H"], c["Hkv"], c["hd"]
    rows = range(c["T"]) if rows is None else rows
    heads = range(H) if heads is None else heads
    rows = torch.tensor(list(rows), device=q.device)
    q = q.double().view(-1, H, hd)[rows]
    out = torch.zeros(len(rows), len(heads), hd, dtype=torch.float64, device=q.device)
    for n, h in enumerate(heads):
        k, v = values(c["k"][h * Hkv // H], c["ks"][h * Hkv // H]), values(c["v"][h * Hkv // H], c["vs"][h * Hkv // H])
        s = (q[:, h] @ k.T / math.sqrt(hd)).masked_fill(~see[rows], -math.inf)
        out[:, n] = torch.softmax(s, -1).nan_to_num(0) @ v
    return out


def wrong(out, ref):
    """Whether an output is off by more than twice the bound anywhere, so that no
    error within the bound hides it."""
    return bool(((out - ref).abs() > 2 * TOL * ref.abs()).any())


CASES = [("tree", 32, 8, 128, 1, 700), ("tree", 32, 8, 128, 9, 63), ("tree", 32, 8, 128, 33, 1100),
         ("tree", 32, 8, 128, 65, 2000), ("tree", 32, 8, 64, 25, 0), ("tree", 32, 8, 64, 40, 129),
         ("tree", 16, 1, 64, 9, 1500), ("tree", 8, 8, 128, 130, 257), ("tree", 8, 2, 128, 5, 20000),
         ("tree", 40, 1, 48, 12, 300), ("tree", 4, 4, 128, 1, 31000), ("tree", 20, 1, 64, 7, 900),
         ("causal", 32, 8, 128, 300, 0), ("causal", 8, 2, 64, 64, 500), ("causal", 8, 8, 128, 5, 0),
         ("ranges", 32, 8, 64, 9, 2000), ("ranges", 8, 8, 128, 24, 4000), ("ranges", 16, 2, 128, 40, 2500),
         ("ranges", 16, 1, 64, 7, 1000)]
