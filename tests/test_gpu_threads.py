"""GPU test of calls from a host thread that has made no other CUDA call before: the
tensor-core entry points encode tensor maps, which needs a current context."""

import math
import threading

import pytest
import torch

pytestmark = pytest.mark.gpu

DEV = "cuda"
BF = torch.bfloat16


def attend_q8(ops, ws, seed):
    g = torch.Generator(DEV).manual_seed(seed)
    codes = torch.randint(0, 127, (2, 2, 300, 64), generator=g, device=DEV).to(torch.uint8).view(torch.float8_e4m3fn)
    scales = torch.full((2, 2, 300), 120, dtype=torch.uint8, device=DEV)
    layer = ops.KVLayerQ8(codes[0], codes[1], scales[0], scales[1])
    q, out = torch.randn(3, 8 * 64, generator=g, device=DEV).to(BF), torch.zeros(3, 8 * 64, dtype=BF, device=DEV)
    plen = torch.full((3,), 300, dtype=torch.int32, device=DEV)
    return out, lambda: ops.tree_attention_q8(q, layer, 8, 2, 64, plen, out, ws)


def attend(ops, ws, seed):
    g = torch.Generator(DEV).manual_seed(seed)
    k, v = (torch.randn(2, 300, 64, generator=g, device=DEV).to(BF) for _ in range(2))
    q, out = torch.randn(20, 8 * 64, generator=g, device=DEV).to(BF), torch.zeros(20, 8 * 64, dtype=BF, device=DEV)
    plen = torch.full((20,), 300, dtype=torch.int32, device=DEV)
    return out, lambda: ops.tree_attention(q, k, v, 8, 2, 64, plen, out, ws)


def linear(ops, ws, seed):
    g = torch.Generator(DEV).manual_seed(seed)
    x, w = torch.randn(5, 256, generator=g, device=DEV).to(BF), torch.randn(384, 256, generator=g, device=DEV).to(BF)
    out = torch.zeros(5, 384, dtype=BF, device=DEV)
    return out, lambda: ops.linear(x, [w], ws, out=out)


@pytest.mark.parametrize("make", [attend_q8, attend, linear])
def test_a_threads_first_cuda_call(make):
    """After the main thread's calls have set up the process, a new thread's first
    call gives the main thread's result."""
    from ssd import ops

    ws = ops.Workspace(torch.device(DEV), max_rows=64, vocab=64)
    for seed in (1, 2):  # the second: other tensors than any call before
        out, call = make(ops, ws, seed)
        if seed == 1:
            call()
            torch.cuda.synchronize()
            continue
        errors = []

        def work():
            try:
                call()
            except Exception as e:
                errors.append(e)

        t = threading.Thread(target=work)
        t.start()
        t.join()
        assert not errors, errors
        torch.cuda.synchronize()
        got = out.clone()
        out.fill_(math.nan)
        call()
        ws.check_status()
        assert torch.equal(got, out) and bool(got.abs().sum() > 0)
