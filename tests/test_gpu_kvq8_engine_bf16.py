"""GPU tests of batched and sampled decoding over the 8-bit key/value cache in bf16:
the tensor-core attention with a slot range per sequence."""

import pytest
import torch

from ssd import ops
from ssd import synthetic as S
from ssd import _lib as L
from ssd.config import BridgeConfig, DraftingConfig
from ssd.engine.batch import BatchDecoder
from ssd.engine.speculative import SpeculativeGenerator, TargetRunner, autoregressive_generate
from ssd.models import SubnetworkDraftModel
from ssd.models import runner as R

pytestmark = pytest.mark.gpu

DEV = "cuda"
TREE = dict(depth=3, branch=[3, 2, 2], max_nodes=12)


@pytest.fixture(scope="module", params=["llama32_1b", "llama3_8b"])  # heads of 64 and of 128
def model(request):
    base = S.build_base_model(request.param, 2, torch.bfloat16, DEV, gen_device="cuda", num_hidden_layers=2, vocab_size=2048)
    draft = SubnetworkDraftModel(base, [0], BridgeConfig(hidden_dim=1024))
    S.init_bridges_(draft.bridges, 1, 0.02, 1e-4)
    draft.bridges.to(DEV, torch.bfloat16)
    return base, draft


def tokens(n, seed):
    return torch.randint(0, 2048, (n,), generator=torch.Generator().manual_seed(seed)).tolist()


def logits_of(dec, r0):
    """The head's fp32 logits of the decoder's last forward, rows r0 .. r0 + B."""
    xn, rn = R.head_input(dec.w, dec.scratch, r0, r0 + dec.B)
    out = torch.zeros(dec.B, dec.w.V, dtype=torch.float32, device=DEV)
    ops.linear(xn, [dec.w.lm_head], dec.ws, epilogue=L.EPI_STORE_F32, out=out, T=dec.B, in_norm=rn)
    dec.ws.check_status()
    return out


def run(target, prompts, more):
    """Logits after the prompts, and after each of the given tokens, all sequences together."""
    region = 64 * (-(-(max(map(len, prompts)) + len(more)) // 64))
    dec = BatchDecoder(target, len(prompts), region, sum(map(len, prompts)))
    n = len(prompts)
    ids = [t for p in prompts for t in p[:-1]] + [p[-1] for p in prompts]
    seqs = [b for b, p in enumerate(prompts) for _ in p[:-1]] + list(range(n))
    pos = [i for p in prompts for i in range(len(p) - 1)] + [len(p) - 1 for p in prompts]
    dec._forward(ids, seqs, pos)
    out = [logits_of(dec, len(ids) - n)]
    for step, row in enumerate(more):
        dec._forward([row[b] for b in range(n)], list(range(n)), [len(p) + step for p in prompts])
        out.append(logits_of(dec, 0))
    return out


def test_sequences_together_give_the_logits_of_each_alone(model):
    """Prompts of one token to several key blocks, then given tokens. Rows meet other
    rows in their tiles, so sums run in another order and bf16 roundings fall
    differently (2^-8 of an activation, through two layers): 2^-5 of the logits' norm
    bounds that, while a slot of another sequence moves them by their whole size."""
    base, _ = model
    target = TargetRunner(base, kv_dtype="e4m3")
    prompts = [tokens(n, n) for n in (3, 170, 1, 129, 400, 64)]
    more = [tokens(len(prompts), 900 + s) for s in range(3)]
    together = run(target, prompts, more)
    for b, p in enumerate(prompts):
        alone = run(target, [p], [[row[b]] for row in more])
        for x, y in zip(together, alone):
            assert bool(torch.isfinite(x).all())
            assert ((x[b] - y[0]).norm() <= 2.0**-5 * y[0].norm()), (b, ((x[b] - y[0]).norm() / y[0].norm()).item())


def test_batched_logits_near_the_plain_caches(model):
    """Against the bf16 cache: the codes' rounding (2^-4 of a key or value at most, random
    in sign) is left."""
    base, _ = model
    prompts = [tokens(n, n) for n in (5, 200, 90)]
    got = [run(TargetRunner(base, kv_dtype=kv), prompts, [tokens(3, 77)]) for kv in (None, "e4m3")]
    for x, y in zip(*got):
        assert bool((torch.nn.functional.cosine_similarity(x, y, dim=1) > 0.99).all())


def test_sampled_rounds_repeat_with_their_seed(model):
    base, draft = model
    cfg = DraftingConfig(**TREE, temperature=0.8, top_p=0.9)
    ids = torch.tensor([tokens(150, 8)], device=DEV)
    runs = [SpeculativeGenerator(base, draft, cfg, TargetRunner(base, kv_dtype="e4m3")).generate(
        ids, 20, set(), seed=s, use_graph=g) for s, g in ((3, True), (3, True), (3, False), (4, True))]
    assert runs[0].tokens == runs[1].tokens == runs[2].tokens and len(runs[0].tokens) == 20
    assert runs[0].tokens != runs[3].tokens and all(0 <= t < 2048 for r in runs for t in r.tokens)
    ar = [autoregressive_generate(TargetRunner(base, kv_dtype="e4m3"), ids, 10, set(), 0.8, 0.9, seed=7).tokens
          for _ in range(2)]
    assert ar[0] == ar[1]
