"""CPU checks of the token step's operators (rotated append, shared-prefix decode, adjusted logits): struct layouts,
refusals that need no device, and the shared decode's plan, which is host code."""
import ctypes

import numpy as np
import pytest

UNIT = np.dtype([("table_lane", "<u4"), ("lane", "<u4"), ("col0", "<u4"), ("cols", "<u4"), ("begin", "<u4"), ("end", "<u4"),
                 ("slot", "<u4"), ("head", "<u2"), ("heads", "u1"), ("kind", "u1")])
SINGLE = 0x80
LANE = np.dtype([("table_lane", "<u4"), ("tokens", "<u4"), ("prefix_slot", "<u4"), ("prefix_stride", "<u4"),
                 ("prefix_count", "<u4"), ("tail_slot", "<u4"), ("tail_count", "<u4"), ("merged", "<u4")])


def split_entries(entries, plan):
    units = entries[:plan.unit_count * UNIT.itemsize].view(UNIT)
    return units[units["cols"] != 0], entries[plan.unit_count * UNIT.itemsize:].view(LANE)


def test_struct_layouts(kimkv):
    d = kimkv.device
    assert d.APPEND_ROPE_JOB.itemsize == 28
    assert d.LOGITS_RULE.itemsize == 56
    assert ctypes.sizeof(d.Rope) == 16
    assert ctypes.sizeof(d.SharedGroup) == 12
    assert ctypes.sizeof(d.SharedPlan) == 56


@pytest.mark.parametrize("heads,dim,group", [(4, 64, 8), (8, 128, 4), (1, 64, 1), (3, 96, 5), (2, 12, 40), (16, 64, 1)])
def test_plan_covers_every_key_once(kimkv, heads, dim, group):
    """Every (lane, query head, token) is in exactly one unit; parts sit in slots of their own that the lane's record lists;
    a prefix is read through the group's first lane in blocks of 64 that every lane holds."""
    d = kimkv.device
    rng = np.random.default_rng(heads * dim + group)
    cases = [([1], []), ([0], []), ([0, 5, 0], [(0, 3, 5)]), ([64] * 3, [(0, 3, 64)]), ([500, 700], [(0, 2, 450)]),
             ([65, 63], [(0, 2, 64)]), ([3000] * 9 + [40], [(0, 9, 2999)]), ([9000, 100, 9000, 9000], [(2, 2, 8000)]),
             ([40000] * 3, [(0, 3, 40000)]), ([1000] * 70, [(0, 70, 900)]), ([2000] * 6, [(0, 2, 1000), (3, 3, 1999)])]
    for _ in range(6):
        n = int(rng.integers(2, 40))
        cut = int(rng.integers(1, n))
        prefixes = rng.integers(1, 5000, 2)
        counts = [int(prefixes[int(i >= cut)] + rng.integers(0, 900)) for i in range(n)]
        cases.append((counts, [(0, cut, int(prefixes[0])), (cut, n - cut, int(prefixes[1]))]))
    for compute_units, (counts, groups) in [(n, c) for n in (256, 3) for c in cases]:
        entries, plan = d.shared_decode_plan(heads, dim, heads * group, compute_units, counts, groups)
        assert plan.entry_bytes == len(entries) == plan.unit_count * 32 + len(counts) * 32
        units, lanes = split_entries(entries, plan)
        assert (plan.kv_heads, plan.head_dim, plan.query_heads, plan.lane_count) == (heads, dim, heads * group, len(counts))
        seen = [np.zeros((heads, group, t), dtype=np.int8) for t in counts]
        slots = {}
        of_lane = {i: first for first, n, _ in groups for i in range(first, first + n)}
        assert plan.unit_count % 8 == 0
        for u in units.tolist():
            table_lane, lane0, col0, cols, begin, end, slot, head, of_heads, kind = u
            assert begin < end and begin % 64 == 0 and of_heads > 0 and head + of_heads <= heads
            blocks = kind & 0x7F
            assert blocks in (1, 2, 4) and cols <= 16 * blocks and (of_heads == 1 or blocks == 1)
            for c in range(col0, col0 + cols):
                lane = lane0 + c // group
                seen[lane][head:head + of_heads, c % group, begin:end] += 1
                if lane != table_lane:
                    assert of_lane[lane] == table_lane and end <= groups[[g[0] for g in groups].index(of_lane[lane])][2]
                if not kind & SINGLE:
                    for h in range(head, head + of_heads):
                        q = h * group + c % group
                        assert (slot + c // group, q) not in slots
                        slots[slot + c // group, q] = lane
        for lane, marks in enumerate(seen):
            assert np.all(marks == 1), (counts, groups, lane)
        assert plan.merge_lanes == int(lanes["merged"].sum())
        for lane, rec in enumerate(lanes):
            assert rec["tokens"] == counts[lane]
            mine = [int(rec["prefix_slot"]) + k * int(rec["prefix_stride"]) for k in range(int(rec["prefix_count"]))]
            mine += [int(rec["tail_slot"]) + k for k in range(int(rec["tail_count"]))] if rec["merged"] else []
            want = sorted(s for (s, h), at in slots.items() if at == lane and h == 0)
            for q in range(heads * group):   # each part is whole
                assert all(slots.get((s, q)) == lane for s in want)
            assert sorted(map(int, mine)) == want and all(s < plan.slot_count for s in want)
            assert bool(rec["merged"]) == (len(want) > 0)
        o = (plan.slot_count * heads * group * dim * 4 + 15) // 16 * 16
        assert plan.workspace_bytes == o + plan.slot_count * heads * group * 8


@pytest.mark.parametrize("empty", [[0], [5], [39], [0, 1, 2, 20, 38, 39], list(range(9, 33))])
def test_plan_shares_beside_empty_lanes(kimkv, empty):
    """Lanes of no tokens in a group (requests that ended, padding) do not end the others' sharing."""
    lanes, prefix = 40, 8192
    counts = [0 if i in empty else prefix + 1 + i for i in range(lanes)]
    live = [i for i in range(lanes) if counts[i]]
    entries, plan = kimkv.device.shared_decode_plan(4, 64, 32, 8, counts, [(0, lanes, prefix)])
    units, records = split_entries(entries, plan)
    shared = units[units["cols"] > 8]
    assert len(shared) and np.all(shared["table_lane"] == live[0])
    for u in shared:   # none computes columns of empty lanes alone
        assert any(counts[int(u["lane"]) + c // 8] for c in range(int(u["col0"]), int(u["col0"] + u["cols"])))
    for head in range(4):   # every live lane's columns on every block of the prefix, once; of nobody past the last live lane
        seen = np.zeros((lanes, 8, prefix // 64), dtype=np.int8)
        for u in shared[shared["head"] == head]:
            for c in range(int(u["col0"]), int(u["col0"] + u["cols"])):
                seen[int(u["lane"]) + c // 8, c % 8, int(u["begin"]) // 64:int(u["end"]) // 64] += 1
        assert np.all(seen[live] == 1) and np.all(seen[:live[0]] == 0) and np.all(seen[live[-1] + 1:] == 0)
    used = set()
    for i, rec in enumerate(records):
        assert rec["tokens"] == counts[i] and bool(rec["merged"]) == (i in live) and (i in live or rec["prefix_count"] == rec["tail_count"] == 0)
        mine = [int(rec["prefix_slot"]) + k * int(rec["prefix_stride"]) for k in range(int(rec["prefix_count"]))]
        mine += [int(rec["tail_slot"]) + k for k in range(int(rec["tail_count"]))]
        assert not used.intersection(mine) and all(m < plan.slot_count for m in mine)
        used.update(mine)


@pytest.mark.parametrize("heads,dim,group,lanes,prefix,own", [
    (1, 64, 8, 512, 8192, 100), (1, 128, 8, 256, 8192, 100), (2, 128, 16, 256, 8192, 100), (2, 64, 8, 600, 4096, 1),
    (4, 64, 8, 512, 16384, 100), (4, 128, 4, 500, 2048, 30), (3, 96, 5, 300, 8192, 700), (1, 64, 64, 512, 4096, 100)])
@pytest.mark.parametrize("compute_units", [256, 64])
def test_plan_spreads_wide_groups(kimkv, heads, dim, group, lanes, prefix, own, compute_units):
    """More columns of one head and key range than an XCD has compute units go to several XCDs: none has more of them
    than run there at once, or much more than its share."""
    entries, plan = kimkv.device.shared_decode_plan(heads, dim, heads * group, compute_units, [prefix + own] * lanes, [(0, lanes, prefix)])
    units = entries[:plan.unit_count * UNIT.itemsize].view(UNIT).reshape(8, -1)   # a row an XCD
    shared = (units["end"] <= prefix) & (units["cols"] != 0)
    columns = {(int(u["head"]), int(u["begin"])) for u in units[shared]}
    assert shared.sum() > len(columns) * compute_units // 8   # wide indeed
    on_xcd = shared.sum(1)
    at_once = compute_units // 8 * (8 // plan.waves)
    assert on_xcd.max() <= max(at_once, 1.25 * on_xcd.mean()), on_xcd
    work = np.where(shared, (units["end"] - units["begin"]).astype(np.int64), 0).sum(1)
    assert work.max() <= max(1.25 * work.mean(), at_once * (units["end"] - units["begin"])[shared].max()), work


def test_plan_refusals(kimkv):
    d = kimkv.device
    lib = d.lib()
    counts = np.array([100, 200, 300], dtype=np.uint32)
    ptr = counts.ctypes.data_as(ctypes.c_void_p)
    plan = d.SharedPlan()

    def status(heads=4, dim=64, qh=32, lanes=3, groups=(), count_ptr=ptr, capacity=0, entries=None):
        shared = (d.SharedGroup * len(groups))(*[d.SharedGroup(*g) for g in groups])
        return lib.kimkv_shared_decode_plan(heads, dim, qh, 256, count_ptr, lanes, shared, len(groups), entries, capacity,
                                            ctypes.byref(plan))

    for bad in (dict(heads=0), dict(qh=0), dict(qh=30), dict(dim=0), dict(dim=257), dict(heads=1 << 16, qh=1 << 16), dict(count_ptr=None),
                dict(groups=[(0, 4, 64)]), dict(groups=[(3, 1, 64)]), dict(groups=[(0, 2, 64), (1, 2, 64)]),
                dict(groups=[(0xFFFFFFFF, 2, 64)]), dict(groups=[(1, 0xFFFFFFFF, 64)])):
        assert status(**bad) == d.INVALID_ARGUMENT, bad
        assert plan.entry_bytes == 0, bad
    assert lib.kimkv_shared_decode_plan(4, 64, 32, 256, ptr, 3, None, 1, None, 0, ctypes.byref(plan)) == d.INVALID_ARGUMENT
    assert lib.kimkv_shared_decode_plan(4, 64, 32, 256, ptr, 3, None, 0, None, 0, None) == d.INVALID_ARGUMENT
    for tokens in (1 << 31, 0xFFFFFFFF):
        counts[1] = tokens
        assert status() == d.INVALID_ARGUMENT and plan.entry_bytes == 0
    counts[1] = 200
    # Too small: the size comes back, and nothing is written past it.
    assert status() == d.INVALID_ARGUMENT and plan.entry_bytes > 0
    need = plan.entry_bytes
    buf = np.full(need + 64, 0xAB, dtype=np.uint8)
    assert status(capacity=need - 1, entries=buf.ctypes.data_as(ctypes.c_void_p)) == d.INVALID_ARGUMENT
    assert np.all(buf == 0xAB) and plan.entry_bytes == need
    assert status(capacity=need, entries=buf.ctypes.data_as(ctypes.c_void_p)) == d.OK and np.all(buf[need:] == 0xAB)
    # No lanes: nothing to do, no error.
    entries, empty = d.shared_decode_plan(4, 64, 32, 256, [], [])
    assert len(entries) == 0 and empty.unit_count == 0 and empty.workspace_bytes == 0
    # A group of lanes that do not all hold its prefix shares what they do hold.
    entries, p = d.shared_decode_plan(4, 64, 32, 256, [9000] * 100 + [4000] + [9000] * 100, [(0, 201, 8192)])
    units, _ = split_entries(entries, p)
    assert max(u["end"] for u in units if u["cols"] > 8) == 4000 // 64 * 64


@pytest.mark.parametrize("heads,dim,query_heads,lanes", [(1, 64, 1 << 28, 1), (65535, 8, 65535, 4200), (1, 64, 0xFFFFFFFF, 1), (1, 64, 8, 1 << 24)])
def test_plan_refuses_what_no_launch_takes(kimkv, heads, dim, query_heads, lanes):
    """A plan of more units than a launch has workgroups for is refused before it is made, and so is one of more lanes."""
    d = kimkv.device
    counts = np.zeros(lanes, dtype=np.uint32)
    counts[:4200] = 64
    plan = d.SharedPlan()
    assert d.lib().kimkv_shared_decode_plan(heads, dim, query_heads, 256, counts.ctypes.data_as(ctypes.c_void_p), lanes, None, 0, None, 0,
                                            ctypes.byref(plan)) == d.INVALID_ARGUMENT
    assert plan.entry_bytes == 0 and plan.unit_count == 0


def test_plan_refuses_rows_past_32_bit_offsets(kimkv):
    """A lane's query row is indexed in 32 bits: one of 2^31 elements or more is refused, one just below is planned."""
    d = kimkv.device
    counts = np.array([64], dtype=np.uint32)
    for query_heads, dim, want in ((1 << 25, 64, d.INVALID_ARGUMENT), (1 << 24, 128, d.INVALID_ARGUMENT), (1 << 23, 256, d.INVALID_ARGUMENT),
                                   ((1 << 23) - 16, 255, d.OK)):
        plan = d.SharedPlan()
        entries = np.empty(1 << 26, dtype=np.uint8)
        assert d.lib().kimkv_shared_decode_plan(1, dim, query_heads, 256, counts.ctypes.data_as(ctypes.c_void_p), 1, None, 0,
                                                entries.ctypes.data_as(ctypes.c_void_p), len(entries), ctypes.byref(plan)) == want, (query_heads, dim)


def test_entry_points_refuse_null(kimkv):
    d = kimkv.device
    lib = d.lib()
    rope = d.Rope(10000.0, 64, 0)
    assert lib.kimkv_append_rope_batch(None, None, 0, 0, 0, None, 0, 0, 32, rope, None, 0, None) == d.INVALID_ARGUMENT
    assert lib.kimkv_shared_decode_batch(None, None, None, d.SharedPlan(), None, None) == d.INVALID_ARGUMENT
    one = ctypes.c_void_p(16)
    for args in ((None, 1, 8, None, one, one), (one, 1, 0, None, one, one), (one, 1, 8, None, None, None),
                 (one, 1, 1 << 31, None, one, one)):
        assert lib.kimkv_model_logits_adjust(*args, None, None) == d.INVALID_ARGUMENT
    # Several slices of the vocabulary and no workspace, or one off its alignment.
    assert lib.kimkv_logits_workspace_bytes(3, 1 << 20) > 0
    assert lib.kimkv_model_logits_adjust(one, 3, 1 << 20, None, None, one, None, None) == d.INVALID_ARGUMENT
    assert lib.kimkv_model_logits_adjust(one, 3, 1 << 20, None, None, one, ctypes.c_void_p(20), None) == d.INVALID_ARGUMENT
    # No rows: nothing to do.
    assert lib.kimkv_model_logits_adjust(one, 0, 1 << 20, None, None, one, None, None) == d.OK


def test_logits_workspace_never_falls(kimkv):
    """Scratch for a batch is enough for any smaller one, of rows as of vocabulary."""
    size = kimkv.device.logits_workspace_bytes
    vocabularies = [1, 5, 4093, 4094, 8189, 8190, 16000, 16381, 16382, 32000, 50257, 128000, 1 << 20]
    for vocabulary in vocabularies:
        of_rows = [size(rows, vocabulary) for rows in range(300)]
        assert of_rows == sorted(of_rows), vocabulary
        assert of_rows[0] == 0 and size(1 << 20, vocabulary) >= of_rows[-1]
    for rows in (1, 16, 17, 64, 65, 128, 129, 256):
        of_vocabulary = [size(rows, v) for v in vocabularies]
        assert of_vocabulary == sorted(of_vocabulary), rows
