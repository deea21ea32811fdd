"""GPU tests of decoding over the 8-bit key/value cache (kv_dtype "e4m3"): the
engines, the forward API, batched decoding and the command line."""

import pytest
import torch

from ssd import synthetic as S
from ssd.config import BridgeConfig, DraftingConfig
from ssd.engine.kv_cache import KVCache
from ssd.engine.round import GreedyRound, TargetStep, TreePlan, cache_capacity
from ssd.engine.speculative import SpeculativeGenerator, TargetRunner, autoregressive_generate
from ssd.models import SubnetworkDraftModel

pytestmark = pytest.mark.gpu

DEV = "cuda"
TREE = dict(depth=3, branch=[3, 2, 2], max_nodes=12)


@pytest.fixture(scope="module")
def tiny():
    base = S.build_base_model("tiny", 0, torch.float32, "cpu").to(DEV)
    draft = SubnetworkDraftModel(base, [0, 3, 5], BridgeConfig(init_std=0.02))
    S.init_bridges_(draft.bridges, 0, in_std=0.125, out_std=0.02)
    draft.bridges.to(DEV)
    return base, draft


@pytest.fixture(scope="module")
def small_1b():
    """Two layers of the 1B shape in bf16: the tensor-core kernels."""
    base = S.build_base_model("llama32_1b", 1, torch.bfloat16, DEV, gen_device="cuda", num_hidden_layers=2,
                              vocab_size=4096)
    draft = SubnetworkDraftModel(base, [0], BridgeConfig(hidden_dim=1024))
    S.init_bridges_(draft.bridges, 1, 0.02, 1e-4)
    draft.bridges.to(DEV, torch.bfloat16)
    return base, draft


def prompt(n, vocab, seed=5):
    return torch.randint(0, vocab, (1, n), generator=torch.Generator().manual_seed(seed))


def test_cache_protocol_and_values():
    """update / k / v return the quantised values; crop, keep_positions and overflow as the plain cache."""
    c = KVCache(2, 40, "e4m3")
    k, v = (torch.randn(1, 2, 9, 32, generator=torch.Generator(DEV).manual_seed(s), device=DEV) for s in (1, 2))
    kk, vv = c.update(1, k, v)
    assert kk.shape == (1, 2, 9, 32) and kk.dtype == torch.float32
    for got, want in ((kk, k), (vv, v)):  # half a step of e4m3, or half a subnormal step of the row's scale
        unit = want.abs().amax(-1, keepdim=True) / 448 * 2
        assert ((got - want).abs() <= want.abs() * 2.0**-4 + unit * 2.0**-10).all()
    c.advance(9)
    assert torch.equal(c.k[1][:, :, :9], kk) and torch.equal(c.v[1][:, :, :9], vv) and (c.k[0] == 0).all()
    c.keep_positions(3, [8, 4, 6])
    assert c.seq_len == 6
    assert torch.equal(c.k[1][:, :, 3:6], kk[:, :, [8, 4, 6]]) and torch.equal(c.v[1][:, :, :3], vv[:, :, :3])
    with pytest.raises(RuntimeError, match="overflow"):
        c.update(0, k.new_zeros(1, 2, 35, 32), v.new_zeros(1, 2, 35, 32))
    with pytest.raises(ValueError):
        c.allocate(2, 64, torch.float32, DEV)
    with pytest.raises(ValueError):
        KVCache(1, 8, "e4m3").allocate(2, 24, torch.float32, DEV)


def test_forward_matches_the_plain_cache_closely(tiny):
    """Prompt, then a tree block, through forward(): hidden states near those over
    the fp32 cache, cached rows the quantised values of the plain cache's."""
    base, _ = tiny
    ids = prompt(40, 128)
    mask = torch.tril(torch.ones(6, 6, dtype=torch.bool))
    mask[4, 3] = mask[5, 4] = False
    outs, caches = [], []
    for kv in (None, "e4m3"):
        t = TargetRunner(base, kv_dtype=kv)
        c = t.new_cache(64)
        t(ids[:, :34].to(DEV), past_key_values=c)
        outs.append(t(ids[:, 34:].to(DEV), position_ids=torch.tensor([[34, 35, 35, 36, 36, 37]]), past_key_values=c,
                      tree_attention_mask=mask))
        caches.append(c)
    a, b = (o.hidden_states.float().flatten() for o in outs)
    assert torch.nn.functional.cosine_similarity(a, b, dim=0) > 0.99
    # layer 0 sees the same inputs: its rows differ by their rounding to e4m3 alone (2^-4 of the value, or half a
    # subnormal step, 2^-10 of a scale of at most amax / 224) and the projections' sum order (1e-5)
    for plain, q8 in ((caches[0].k[0], caches[1].k[0]), (caches[0].v[0], caches[1].v[0])):
        top = plain.abs().amax(-1, keepdim=True)
        assert ((q8 - plain).abs() <= plain.abs() * (2.0**-4 + 1e-5) + top * (2.0**-10 / 224 + 1e-5)).all()


@pytest.mark.parametrize("model", ["tiny", "small_1b"])
def test_speculative_equals_target_only(model, request):
    """Greedy speculative decoding over the 8-bit cache gives the target's own
    greedy tokens over the 8-bit cache (graphs and eager), up to a near-tie."""
    base, draft = request.getfixturevalue(model)
    n = 24
    ids = prompt(50, base.config.vocab_size).to(DEV)
    target = TargetRunner(base, kv_dtype="e4m3")
    gen = SpeculativeGenerator(base, draft, DraftingConfig(**TREE), target)
    sd = gen.generate(ids, n, set())
    assert gen.engine().cache.quantized
    eager = SpeculativeGenerator(base, draft, DraftingConfig(**TREE), target).generate(ids, n, set(), use_graph=False)
    assert sd.tokens == eager.tokens and sum(sd.accepted_per_round) >= n - 1
    eng = TargetStep(target, target.new_cache(cache_capacity(50, n, TreePlan(DraftingConfig(**TREE)))), n)
    eng.prefill(ids)
    ar, gaps = eng.tokens(), []
    while len(ar) < n:
        eng.run(1, use_graph=False)
        gaps.append(float(eng.gap[0]))
        ar = eng.tokens()
    eng.ws.check_status()
    for i, (x, y) in enumerate(zip(sd.tokens, ar)):
        if x != y:  # only where the two best logits nearly tie (the forwards sum in another order)
            assert i > 0 and gaps[i - 1] < (1e-2 if model == "small_1b" else 1e-4)
            break
    assert len(autoregressive_generate(target, ids, n, set()).tokens) == n


def test_sampled_rounds_are_deterministic(tiny):
    base, draft = tiny
    cfg = DraftingConfig(**TREE, temperature=0.8, top_p=0.9)
    ids = prompt(20, 128).to(DEV)
    runs = [SpeculativeGenerator(base, draft, cfg, TargetRunner(base, kv_dtype="e4m3")).generate(ids, 16, set(), seed=s)
            for s in (3, 3, 4)]
    assert runs[0].tokens == runs[1].tokens and len(runs[0].tokens) == 16
    assert all(0 <= t < 128 for r in runs for t in r.tokens)
    ar = [autoregressive_generate(TargetRunner(base, kv_dtype="e4m3"), ids, 10, set(), 0.8, 0.9, seed=7).tokens
          for _ in range(2)]
    assert ar[0] == ar[1]


def test_garbage_behind_the_prompt_changes_nothing(small_1b):
    """Codes and scales past the prompt filled with garbage (finite or NaN codes)
    leave the decode as it was: every slot is written before it is read."""
    base, draft = small_1b
    cfg = DraftingConfig(**TREE)
    ids = prompt(70, base.config.vocab_size).to(DEV)
    target = TargetRunner(base, kv_dtype="e4m3")
    got = []
    for fill in (None, 0x35, 0x7f):
        eng = GreedyRound(target, draft, cfg, target.new_cache(cache_capacity(70, 16, TreePlan(cfg))), 16)
        eng.prefill(ids)
        if fill is not None:
            eng.cache.buf.view(torch.uint8)[:, :, :, 70:] = fill
            eng.cache.scales[:, :, :, 70:] = 200
        for _ in range(5):
            eng.run_round()
        eng.ws.check_status()
        got.append(eng.tokens())
    assert got[0] == got[1] == got[2]


def test_batched_decoding_equals_single(tiny):
    from ssd.data.generate_selfdistill import generate_batch

    base, _ = tiny
    target = TargetRunner(base, kv_dtype="e4m3")
    prompts = [prompt(n, 128, seed=n)[0].tolist() for n in (3, 17, 1, 40)]
    together = generate_batch(target, prompts, 12, set(), 0.0, 1.0, 0)
    for p, toks in zip(prompts, together):
        assert toks == generate_batch(target, [p], 12, set(), 0.0, 1.0, 0)[0]
    sampled = [generate_batch(target, prompts, 8, set(), 0.9, 0.9, 0) for _ in range(2)]
    assert sampled[0] == sampled[1]


def test_a_change_of_kv_dtype_makes_a_new_engine(tiny):
    base, draft = tiny
    target = TargetRunner(base)
    gen = SpeculativeGenerator(base, draft, DraftingConfig(**TREE), target)
    ids = prompt(12, 128).to(DEV)
    plain = gen.generate(ids, 8, set()).tokens
    target.kv_dtype = "e4m3"
    gen.generate(ids, 8, set())
    assert gen.engine().cache.quantized
    target.kv_dtype = None
    assert gen.generate(ids, 8, set()).tokens == plain and not gen.engine().cache.quantized


def test_capture_outlives_the_graphs_of_dropped_engines(tiny):
    """A captured graph in a reference cycle, collected while another engine
    captures its own, does not disturb it."""
    import gc

    base, _ = tiny
    ids = prompt(9, 128).to(DEV)
    want = None
    for litter in (False, True):
        target = TargetRunner(base, kv_dtype="e4m3")
        step = TargetStep(target, target.new_cache(64), 16)
        step.prefill(ids)
        if litter:
            old, stream = [torch.cuda.CUDAGraph()], torch.cuda.Stream()
            x = torch.zeros(8, device=DEV)
            with torch.cuda.graph(old[0], stream=stream):
                x += 1
            real = step.step

            def littered():
                cycle = [old.pop()]
                cycle.append(cycle)
                del cycle
                assert len([[] for _ in range(1000)]) == 1000  # enough to set a collection off
                real()

            step.step = littered
        before = gc.get_threshold()
        gc.set_threshold(10, 1, 1)
        try:
            step.run(6)
        finally:
            gc.set_threshold(*before)
        torch.cuda.synchronize()
        want = want or step.tokens()
        assert step.tokens() == want


def test_command_line_runs_over_the_8_bit_cache(capsys):
    from ssd.cli import run

    run.main(["--synthetic", "tiny", "--prompt", "hello there", "--max-new-tokens", "8", "--kv-dtype", "e4m3"])
    out = capsys.readouterr().out
    assert "key/value cache: e4m3" in out and "greedy output identical to AR: True" in out
