"""GPU tests of compaction in an 8-bit key/value cache whose layers, keys / values
and heads lie in other orders, or are parts of a wider buffer."""

import pytest
import torch

pytestmark = pytest.mark.gpu

DEV = "cuda"


@pytest.mark.parametrize("Ln,Hkv", [(3, 2), (1, 2), (3, 1), (1, 1)])
@pytest.mark.parametrize("order", [(0, 1, 2), (2, 1, 0), (2, 0, 1), (1, 0, 2)])
@pytest.mark.parametrize("wide", [False, True])
def test_compact_over_any_layout(Ln, Hkv, order, wide):
    from ssd import ops

    slots, hd, start, keep = 48, 32, 11, [12, 14, 19]
    dims = (Ln, 2, Hkv)
    back = [order.index(i) for i in range(3)]
    rows = slots + (5 if wide else 0)
    x = torch.randint(0, 256, (*(dims[i] for i in order), rows, hd), dtype=torch.uint8, device=DEV)
    sc = torch.randint(0, 256, x.shape[:-1], dtype=torch.uint8, device=DEV)
    want, wants = x.clone(), sc.clone()
    want[..., start:start + 3, :], wants[..., start:start + 3] = x[..., keep, :], sc[..., keep]
    codes = x.view(torch.float8_e4m3fn).permute(*back, 3, 4)[:, :, :, :slots]
    scales = sc.permute(*back, 3)[..., :slots]
    i32 = dict(dtype=torch.int32, device=DEV)
    ws = ops.Workspace(torch.device(DEV), max_rows=16, vocab=16)
    ops.kv_compact_q8(codes, scales, torch.tensor([start], **i32), torch.tensor(keep, **i32), torch.tensor([3], **i32), 3, ws)
    ws.check_status()
    assert torch.equal(x, want) and torch.equal(sc, wants)
