"""CPU tests of the 8-bit key/value cache's entry points: every refusal happens
on the host, before a pointer is read or anything is launched."""

import ctypes as C

import pytest
import torch

from ssd import _lib as L
from ssd import ops

P = 1 << 20  # a 16-byte aligned address that is never read


def cache(**kw):
    f = dict(k=P, v=P, k_scale=P, v_scale=P, head_stride=64 * 64, scale_head_stride=64, max_slots=64, n_kv_heads=2,
             head_dim=64)
    f.update(kw)
    return C.byref(L.SsdKvQ8(*[f[n] for n, _ in L.SsdKvQ8._fields_]))


BAD_CACHES = [(dict(k=None), ValueError), (dict(v_scale=None), ValueError), (dict(head_dim=0), ValueError),
              (dict(head_dim=72), L.SSDError), (dict(head_dim=144), L.SSDError), (dict(n_kv_heads=0), ValueError),
              (dict(max_slots=0), ValueError), (dict(max_slots=2**31 - 1), L.SSDError),
              (dict(head_stride=64 * 64 - 16), ValueError), (dict(scale_head_stride=63), ValueError),
              (dict(head_stride=64 * 64 + 8), ValueError), (dict(v=P + 4), ValueError)]


def write(c=None, **kw):
    a = dict(q=P, ldq=512, k=P, ldk=128, v=P, ldv=128, T=4, H=8, cos=P, sin=P, max_pos=10, rot=64, inter=0, pos=P,
             slots=P, cache=c if c is not None else cache(), q_out=P, ldqo=512, dtype=L.SSD_BF16, status=None, stream=None)
    a.update(kw)
    L.call("ssd_rope_kv_write_q8", *a.values())


def read(c=None, **kw):
    a = dict(cache=c if c is not None else cache(), slots=None, first=0, n=4, k_out=P, ldk=128, v_out=P, ldv=128,
             dtype=L.SSD_BF16, status=None, stream=None)
    a.update(kw)
    L.call("ssd_kv_read_q8", *a.values())


def attend(c=None, **kw):
    a = dict(q=P, ldq=512, T=4, H=8, cache=c if c is not None else cache(), plen=P, pstart=None, base=None, mask=None,
             words=0, bound=0, out=P, ldo=512, dtype=L.SSD_BF16, ws=None, ws_bytes=0, status=None, stream=None)
    a.update(kw)
    L.call("ssd_tree_attention_q8", *a.values())


def compact(**kw):
    a = dict(codes=P, scales=P, layers=2, ls=2 * 2 * 4096, kvs=2 * 4096, hs=4096, sls=256, skvs=128, shs=64, n_kv=2, hd=64,
             slots=64, start=P, keep=P, n_keep=P, max_keep=4, status=None, stream=None)
    a.update(kw)
    L.call("ssd_kv_compact_q8", *a.values())


@pytest.mark.parametrize("fields,exc", BAD_CACHES)
@pytest.mark.parametrize("call", [write, read, attend])
def test_bad_caches_are_refused(call, fields, exc):
    with pytest.raises(exc):
        call(cache(**fields))


BAD = [(write, dict(T=0), ValueError), (write, dict(k=None), ValueError), (write, dict(slots=None), ValueError),
       (write, dict(q_out=None), ValueError), (write, dict(H=0), ValueError), (write, dict(rot=-2), ValueError),
       (write, dict(rot=65), ValueError), (write, dict(rot=66), ValueError), (write, dict(cos=None), ValueError),
       (write, dict(pos=None), ValueError), (write, dict(max_pos=0), ValueError), (write, dict(dtype=7), L.SSDError),
       (write, dict(H=1 << 24, ldq=1 << 40, ldqo=1 << 40), L.SSDError), (write, dict(ldq=511), ValueError), (write, dict(ldk=127), ValueError), (write, dict(ldqo=0), ValueError),
       (read, dict(n=0), ValueError), (read, dict(k_out=None, v_out=None), ValueError), (read, dict(first=61), ValueError),
       (read, dict(first=-1), ValueError), (read, dict(ldk=64), ValueError), (read, dict(dtype=-1), L.SSDError),
       (attend, dict(T=0), ValueError), (attend, dict(H=7), ValueError), (attend, dict(H=0), ValueError),
       (attend, dict(plen=None), ValueError), (attend, dict(out=None), ValueError), (attend, dict(mask=P), ValueError),
       (attend, dict(mask=P, base=P, words=5), ValueError), (attend, dict(mask=P, base=P, words=0), ValueError),
       (attend, dict(dtype=2), L.SSDError), (attend, dict(ldo=511), ValueError), (attend, dict(ldq=8), ValueError),
       (compact, dict(max_keep=33), L.SSDError), (compact, dict(max_keep=0), L.SSDError), (compact, dict(keep=None), ValueError),
       (compact, dict(hd=24), L.SSDError), (compact, dict(layers=0), ValueError), (compact, dict(hs=4100), ValueError),
       (compact, dict(codes=P + 8), ValueError)]


@pytest.mark.parametrize("call,fields,exc", BAD)
def test_bad_arguments_are_refused(call, fields, exc):
    with pytest.raises(exc):
        call(**fields)


def test_layer_wrapper_refuses_what_is_no_cache():
    f8, u8 = torch.float8_e4m3fn, torch.uint8
    k, s = torch.zeros(2, 8, 16).to(f8), torch.zeros(2, 8, dtype=u8)
    for args in ((k.view(u8), k, s, s), (k, k, s.float(), s), (k, k[:, :4], s, s), (k, k, s[:1], s),
                 (k.transpose(0, 1), k.transpose(0, 1), s, s), (k, k, s, s)):  # the last: not on a CUDA device
        with pytest.raises(ValueError):
            ops.KVLayerQ8(*args)


def test_kv_dtype_is_checked_where_it_is_given():
    from ssd.cli import run
    from ssd.config import SSDConfig
    from ssd.engine.kv_cache import KVCache

    raw = {"draft_layers": [0, 2], "model": {"kv_dtype": "e4m3"}}
    assert SSDConfig.from_dict(raw).model.kv_dtype == "e4m3"
    assert SSDConfig.from_dict({"draft_layers": [0, 2]}).model.kv_dtype is None
    with pytest.raises(ValueError):
        SSDConfig.from_dict({"draft_layers": [0, 2], "model": {"kv_dtype": "int8"}})
    with pytest.raises(ValueError):
        KVCache(1, 4, "fp8")
    with pytest.raises(ValueError, match="CUDA"):  # no CPU form: its rows are written by the kernels
        KVCache(1, 4, "e4m3").allocate(1, 16, torch.float32, "cpu")
    assert run.parser().parse_args(["--synthetic", "c2", "--prompt", "a", "--kv-dtype", "e4m3"]).kv_dtype == "e4m3"
    with pytest.raises(SystemExit):
        run.parser().parse_args(["--synthetic", "c2", "--prompt", "a", "--kv-dtype", "int4"])
