"""CPU tests of further refusals of the 8-bit key/value cache's entry points: calls
that would have read or written out of place. Nothing is read or launched."""

import pytest
import torch

from ssd import _lib as L
from ssd import ops
from test_cpu_kvq8 import attend, cache, compact, read, write


# ------------------------------------------------------------- compaction
@pytest.mark.parametrize("entries,max_keep", [(1, 2), (0, 1), (3, 4), (31, 32)])
def test_compact_refuses_a_keep_list_shorter_than_max_keep(entries, max_keep):
    """How many entries count is on the device, so the list has to hold max_keep of them."""
    codes = torch.zeros(1, 2, 1, 64, 16).to(torch.float8_e4m3fn)
    scales = torch.zeros(1, 2, 1, 64, dtype=torch.uint8)
    one = torch.zeros(1, dtype=torch.int32)
    with pytest.raises(ValueError, match="keep_slots has"):
        ops.kv_compact_q8(codes, scales, one, torch.zeros(entries, dtype=torch.int32), one, max_keep)


def test_compact_takes_keep_lists_of_max_keep_entries_and_more():
    """As KVCache.keep_positions passes them (as many) and a round (one more)."""
    codes = torch.zeros(1, 2, 1, 64, 16).to(torch.float8_e4m3fn)
    scales = torch.zeros(1, 2, 1, 64, dtype=torch.uint8)
    one = torch.zeros(1, dtype=torch.int32)
    for entries, max_keep in ((4, 4), (6, 5)):
        with pytest.raises(ValueError, match="CUDA"):  # past that check: these tensors are on the CPU
            ops.kv_compact_q8(codes, scales, one, torch.zeros(entries, dtype=torch.int32), one, max_keep)


@pytest.mark.parametrize("fields", [
    dict(hs=4080), dict(hs=0), dict(hs=-4096), dict(kvs=4096), dict(kvs=8176), dict(kvs=0), dict(ls=8192), dict(ls=16368),
    dict(shs=63), dict(shs=0), dict(skvs=64), dict(skvs=127), dict(sls=255), dict(sls=-256),
    dict(hs=16384, kvs=4096, ls=8176)])
def test_compact_refuses_layers_heads_or_keys_and_values_that_overlap(fields):
    with pytest.raises(ValueError, match="overlap"):
        compact(**fields)


# ----------------------------------------------------------- longest cache
LONGEST = 2**31 - 2**21


@pytest.mark.parametrize("call", [write, read, attend])
@pytest.mark.parametrize("slots", [LONGEST + 1, 2**31 - 2**20, 2**31 - 1024 - 1])
def test_caches_whose_rounded_slots_pass_32_bits_are_refused(call, slots):
    with pytest.raises(L.SSDError, match="too many slots"):
        call(cache(max_slots=slots, head_stride=slots * 64, scale_head_stride=slots))


def test_compaction_of_such_a_cache_is_refused():
    n = LONGEST + 1
    with pytest.raises(ValueError, match="cache shape"):
        compact(slots=n, hs=64 * n, kvs=2 * 64 * n, ls=4 * 64 * n, shs=n, skvs=2 * n, sls=4 * n)


def test_the_longest_cache_fits_32_bits_rounded_up():
    """The attention kernel's units, restated: as many key blocks of 128 slots as
    leave at most 4096 units; its last block's end is a 32-bit number."""
    for slots, fits in ((LONGEST, True), (2**31 - 1024 - 1, False)):
        blocks, shift = (slots + 127) // 128, 0
        while (blocks >> shift) >= 4096:
            shift += 1
        units = (blocks + (1 << shift) - 1) >> shift
        assert ((units << shift) * 128 <= 2**31 - 1) == fits


# ---------------------------------------------------------------- reading
@pytest.mark.parametrize("first,n", [(2**63 - 1, 4), (2**63 - 4, 64), (1, 2**63 - 1), (65, 1), (64, 1), (0, 65)])
def test_a_read_range_that_wraps_around_is_refused(first, n):
    with pytest.raises(ValueError, match="outside the cache"):
        read(first=first, n=n)


# ----------------------------------------------------------------- writing
@pytest.mark.parametrize("fields,exc", [(dict(dtype=16 | 2), L.SSDError), (dict(dtype=32 | 1), L.SSDError),
                                        (dict(dtype=-1), L.SSDError), (dict(dtype=16 | 1), ValueError)])
def test_write_refuses_unknown_types_and_fp32_rows_turned_in_place_into_bf16(fields, exc):
    with pytest.raises(exc):
        write(**fields)  # (q and q_out are one address here)
