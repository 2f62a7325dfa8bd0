"""CPU checks of the cache in 8 bits and of sampling: struct layouts, refusals that need no device, and the decode's plan,
which is host code."""
import ctypes

import numpy as np
import pytest

UNIT = np.dtype([("lane", "<u4"), ("head", "<u4"), ("first", "<u4"), ("count", "<u4"), ("tokens", "<u4"), ("slot", "<u4"),
                 ("reserved", "<u4", (2,))])
MERGE = np.dtype([("lane", "<u4"), ("tokens", "<u4"), ("first_slot", "<u4"), ("parts", "<u4")])
DIRECT = 0xFFFFFFFF


def test_struct_layouts(kimkv):
    d = kimkv.device
    assert d.SAMPLE_RULE.itemsize == 16
    assert ctypes.sizeof(d.QuantPlan) == 48
    assert ctypes.sizeof(d.QuantStorageInfo) == 64


@pytest.mark.parametrize("heads,dim,group", [(4, 64, 8), (8, 128, 4), (1, 64, 1), (3, 96, 5), (2, 12, 40)])
@pytest.mark.parametrize("compute_units", [256, 0, 2])
def test_plan_covers_every_token_once(kimkv, heads, dim, group, compute_units):
    """Every (lane, head, token) is in exactly one unit, parts begin at multiples of 64 tokens and sit in slots of their own
    that the lane's merge record names."""
    d = kimkv.device
    rng = np.random.default_rng(heads + dim)
    cases = [[], [0], [1], [0, 5, 0], [64, 63, 65], [1000] * 70, [40000, 3, 40000], [300000]]
    cases += [list(rng.integers(0, 9000, int(rng.integers(1, 200)))) for _ in range(4)]
    for counts in cases:
        entries, plan = d.quant_decode_plan(heads, dim, heads * group, compute_units, counts)
        assert plan.entry_bytes == len(entries) == plan.unit_count * 32 + plan.merge_lanes * 16
        assert (plan.kv_heads, plan.head_dim, plan.query_heads, plan.lane_count) == (heads, dim, heads * group, len(counts))
        units, merges = entries[:plan.unit_count * 32].view(UNIT), entries[plan.unit_count * 32:].view(MERGE)
        assert plan.workspace_bytes == plan.slot_count * group * (dim + 2) * 4
        seen, parts = {}, {}
        for u in units:
            lane, head = int(u["lane"]), int(u["head"])
            assert u["tokens"] == counts[lane] and u["count"] > 0 and u["first"] % 64 == 0
            seen.setdefault((lane, head), []).append((int(u["first"]), int(u["count"])))
            if u["slot"] != DIRECT:
                parts.setdefault(lane, {}).setdefault(head, []).append((int(u["first"]), int(u["slot"])))
        assert set(seen) == {(i, h) for i, t in enumerate(counts) if t for h in range(heads)}
        for (lane, _), runs in seen.items():
            at = 0
            for first, count in sorted(runs):
                assert first == at
                at += count
            assert at == counts[lane]
        assert sorted(parts) == sorted(int(m["lane"]) for m in merges)
        slots = []
        for m in merges:
            assert m["tokens"] == counts[m["lane"]]
            for h, found in parts[int(m["lane"])].items():
                assert len(found) == m["parts"] > 1
                assert sorted(s for _, s in found) == list(range(m["first_slot"] + h * m["parts"], m["first_slot"] + (h + 1) * m["parts"]))
                slots += [s for _, s in found]
        assert sorted(slots) == list(range(plan.slot_count))


def test_plan_refusals(kimkv):
    d = kimkv.device
    plan = d.QuantPlan()

    def refused(heads, dim, query_heads, counts, lanes=None, capacity=0, entries=None):
        c = np.array(counts, dtype=np.uint32)
        status = d.lib().kimkv_quant_decode_plan(heads, dim, query_heads, 256, c.ctypes.data_as(ctypes.c_void_p) if len(c) else None,
                                                 len(c) if lanes is None else lanes, entries, capacity, ctypes.byref(plan))
        return status == d.INVALID_ARGUMENT

    assert refused(0, 64, 8, [5]) and refused(4, 0, 8, [5]) and refused(4, 64, 0, [5]) and refused(4, 64, 6, [5])
    assert refused(4, 257, 8, [5]) and refused(1 << 16, 64, 1 << 16, [5]) and refused(4, 64, 8, [1 << 31])
    assert refused(1, 256, 1 << 23, [5])                       # a query row of 2^31 elements
    assert refused(4, 64, 8, [], lanes=3)                      # no counts
    assert refused(4, 64, 8, [5], capacity=64)                 # a capacity of nothing
    assert refused(65535, 1, 65535, [100] * 300)               # more units than a launch takes
    assert refused(4, 64, 8, [5]) and plan.entry_bytes == 4 * 32   # the size that is needed comes back
    assert d.lib().kimkv_quant_decode_plan(4, 64, 8, 256, None, 0, None, 0, None) == d.INVALID_ARGUMENT
    assert not refused(4, 64, 8, [])


def test_storage_refusals(kimkv):
    d = kimkv.device
    out = ctypes.c_void_p(1)

    def refused(layers=1, heads=4, dim=64, micro=4, extent=4, form=d.QUANT_INT8, micro_tokens=8, extent_tokens=64):
        status = d.lib().kimkv_quant_storage_create(ctypes.byref(out), d.Layout(layers, heads, dim), form, micro, extent, micro_tokens, extent_tokens)
        return status == d.INVALID_ARGUMENT and not out.value

    assert refused(layers=0) and refused(heads=0) and refused(dim=0) and refused(dim=257) and refused(layers=0x8000) and refused(heads=1 << 16)
    assert refused(form=0) and refused(form=3)
    assert refused(micro_tokens=0) and refused(micro_tokens=7) and refused(micro_tokens=12) and refused(extent_tokens=72) and refused(extent_tokens=0)
    assert refused(layers=0x7FFF, heads=65535, dim=256, micro=0xFFFFFFFF, extent=0xFFFFFFFF, micro_tokens=64)
    assert d.lib().kimkv_quant_storage_create(None, d.Layout(1, 1, 64), 1, 1, 1, 8, 64) == d.INVALID_ARGUMENT
    info = d.QuantStorageInfo()
    assert d.lib().kimkv_quant_storage_query(None, ctypes.byref(info)) == d.INVALID_ARGUMENT
    assert d.lib().kimkv_quant_storage_faults(None, None, None) == d.INVALID_ARGUMENT
    assert d.lib().kimkv_quant_storage_destroy(None) == d.OK


def test_launch_refusals_without_a_storage(kimkv):
    d = kimkv.device
    plan = d.QuantPlan()
    assert d.lib().kimkv_quant_append_batch(None, 16, 1, 1, None) == d.INVALID_ARGUMENT
    assert d.lib().kimkv_quant_gather(None, 16, 1, 0, 1, 0, 1, 16, None) == d.INVALID_ARGUMENT
    assert d.lib().kimkv_quant_promote_batch(None, 16, 1, None) == d.INVALID_ARGUMENT
    assert d.lib().kimkv_quant_decode_batch(None, 16, 16, ctypes.byref(plan), 16, None) == d.INVALID_ARGUMENT


def test_sample_refusals(kimkv):
    d = kimkv.device
    call = d.lib().kimkv_model_sample
    assert call(None, 1, 100, 16, 16, 16, None, None, None) == d.INVALID_ARGUMENT
    assert call(16, 1, 0, 16, 16, 16, None, None, None) == d.INVALID_ARGUMENT
    assert call(16, 1, (1 << 20) + 1, 16, 16, 16, None, None, None) == d.INVALID_ARGUMENT
    assert call(16, 1, 100, None, 16, 16, None, None, None) == d.INVALID_ARGUMENT
    assert call(16, 1, 100, 16, None, 16, None, None, None) == d.INVALID_ARGUMENT
    assert call(16, 1, 100, 16, 16, None, 16, None, None) == d.INVALID_ARGUMENT
    assert call(16, 0, 100, 16, 16, 16, None, None, None) == d.OK
