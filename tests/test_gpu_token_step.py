"""The token step's operators on the GPU against plain forms in 64 bits: rotated append (kimkv_append_rope_batch),
shared-prefix decode (kimkv_shared_decode_batch), adjusted logits (kimkv_model_logits_adjust), and the three of them
together."""
import ctypes
import math

import numpy as np
import pytest

from tests import helpers
from tests.test_token_step import UNIT, LANE

pytestmark = pytest.mark.gpu

FP16 = 2.0 ** -11   # half a step of fp16, relative
TINY = 2.0 ** -25   # half a step of its subnormals


def _fp16(rng, *shape, scale=1.0):
    return (scale * rng.standard_normal(shape)).astype(np.float16)


def _bits(a):
    return np.ascontiguousarray(a).view(np.uint16)


# ---- rotated append ----------------------------------------------------------


def _rotate(x, positions, theta, rotary, adjacent):
    """(rotated x, |a| + |b| of each element's plane), in 64 bits; x is [rows][heads][dim]."""
    x = x.astype(np.float64)
    out, size = x.copy(), np.zeros_like(x)
    i = np.arange(rotary // 2)
    first, second = (2 * i, 2 * i + 1) if adjacent else (i, i + rotary // 2)
    # Exact turns: the position times the frequency in extended precision.
    angle = positions.astype(np.longdouble)[:, None] * np.longdouble(theta) ** (-2 * i.astype(np.longdouble) / max(rotary, 1))[None]
    angle = (angle % (2 * np.longdouble(np.pi) + np.longdouble(2.4492935982947064e-16)))[:, None, :]
    cos, sin = np.cos(angle).astype(np.float64), np.sin(angle).astype(np.float64)
    a, b = x[..., first], x[..., second]
    out[..., first], out[..., second] = a * cos - b * sin, b * cos + a * sin
    size[..., first] = size[..., second] = np.abs(a) + np.abs(b)
    return out, size


def _near(got, want, size, positions):
    """Rounding to fp16, and 32-bit cosines, sines, products and sums (each within 2^-22 of the plane's size); a position's
    angle in 64 bits is off by up to three of its 2^-53, with the reference's reduction as much again."""
    p = positions.astype(np.float64)[:, None, None]
    bound = FP16 * np.abs(want) + TINY + size * (2.0 ** -21 + 6 * p * 2.0 ** -53)
    err = np.abs(got.astype(np.float64) - want)
    assert np.all(err <= bound), (float((err - bound).max()), np.unravel_index(np.argmax(err - bound), err.shape))


class _Append:
    """A storage with every page filled, jobs on it, and what the pages should hold afterwards ([kind] -> [slot][2][cap][H][D])."""

    def __init__(self, dev, heads, dim, layers=2, micro=24, extent=6, micro_tokens=8, extent_tokens=64, seed=1):
        self.dev, self.heads, self.dim, self.layers = dev, heads, dim, layers
        self.caps = (micro_tokens, extent_tokens)
        self.storage = dev.Storage(layers, heads, dim, micro, extent, micro_tokens, extent_tokens)
        rng = np.random.default_rng(seed)
        self.pages = []
        for kind, n in ((0, micro), (1, extent)):
            cap = self.caps[kind]
            table = np.array([(s, 1, s * cap, cap, cap, kind) for s in range(n)], dtype=helpers.DESC)
            kv = _fp16(rng, layers, 2, n * cap, heads, dim)
            buf = dev.upload(_bits(kv))
            jobs = np.zeros(n, dtype=dev.APPEND_JOB)
            row = heads * dim
            for s in range(n):
                jobs[s] = (buf.ptr + 2 * s * cap * row, buf.ptr + 2 * (n + s) * cap * row, 2 * n * cap * row, row, 0, layers, cap, s, 0, 0, 0,
                           kind, 0)
            self.storage.append_batch(jobs)
            self.pages.append((table, kv.copy()))

    def held(self):
        out = []
        for table, kv in self.pages:
            got = self.storage.gather(table, kv.shape[2]).view(np.float16)
            out.append(got.reshape(kv.shape))
        return out


def _run_append(t, jobs, rows, group, rope, layer, stream=None, q="rows", stride_pad=0, offset=0, max_tokens=None, seed=5):
    """Launches and checks the queries, every page token of every layer, and the bytes around the query rows."""
    dev, heads, dim = t.dev, t.heads, t.dim
    qh = heads * group
    width = (qh + 2 * heads) * dim + stride_pad
    rng = np.random.default_rng(seed)
    qkv = _fp16(rng, rows, width)
    buf = dev.upload(np.concatenate([np.zeros(offset, np.uint16), _bits(qkv).reshape(-1)]))
    q_stride = width if q == "in place" else qh * dim + stride_pad
    q_buf = buf if q == "in place" else dev.upload(np.full(offset + rows * q_stride, 0x1234, np.uint16))
    table = np.zeros(len(jobs), dtype=dev.APPEND_ROPE_JOB)
    for i, j in enumerate(jobs):
        for name, value in j.items():
            if name != "bad":
                table[i][name] = value
    on_gpu = dev.upload(table)
    most = int(table["token_count"].max()) if max_tokens is None else max_tokens
    t.storage.append_rope_launch(on_gpu.ptr, len(jobs), most, layer, buf.ptr + 2 * offset, width, rows, qh, rope,
                                 0 if q is None else q_buf.ptr + 2 * offset, q_stride, stream)
    dev.sync(stream)
    x = qkv[:, :(qh + 2 * heads) * dim].reshape(rows, qh + 2 * heads, dim)
    good = [j for j in jobs if not j.get("bad")]
    named = {}   # row -> (position, kind, slot, token)
    for j in good:
        for i in range(j["token_count"]):
            named[j["first_row"] + i] = (j["position"] + i, j["dst_kind"], j["dst_slot"], j["dst_token"] + i)
    for j in good:
        n, cap = j.get("cow_tokens", 0), t.caps
        if n:
            _, src = t.pages[j["cow_kind"]]
            _, dst = t.pages[j["dst_kind"]]
            a, b = j["dst_slot"] * cap[j["dst_kind"]], j["cow_slot"] * cap[j["cow_kind"]]
            dst[layer, :, a:a + n] = src[layer, :, b:b + n]
    at = np.array(sorted(named), dtype=np.int64)
    positions = np.array([named[r][0] for r in at], dtype=np.uint64)
    want, size = _rotate(x[at, :qh + heads], positions, rope.theta, rope.rotary_dim, rope.adjacent_pairs)
    kept = np.broadcast_to(np.arange(dim) >= rope.rotary_dim, want.shape)
    if q is not None:
        got = dev.download(q_buf.ptr + 2 * offset, (rows, q_stride), np.uint16)
        rows_got = got[at, :qh * dim].reshape(len(at), qh, dim).view(np.float16)
        _near(rows_got, want[:, :qh], size[:, :qh], positions)
        assert np.array_equal(rows_got[kept[:, :qh]], x[at, :qh][kept[:, :qh]])
        before = _bits(qkv).reshape(rows, width) if q == "in place" else np.full((rows, q_stride), 0x1234, np.uint16)
        assert np.array_equal(got[at, qh * dim:], before[at, qh * dim:])
        others = np.setdiff1d(np.arange(rows), at)
        assert np.array_equal(got[others], before[others])
    held = t.held()
    for k, (row, (_, kind, slot, token)) in enumerate(sorted(named.items())):
        p = slot * t.caps[kind] + token
        key = held[kind][layer, 0, p]
        _near(key[None], want[k:k + 1, qh:], size[k:k + 1, qh:], positions[k:k + 1])
        t.pages[kind][1][layer, 0, p] = key
        t.pages[kind][1][layer, 1, p] = x[row, qh + heads:]
    for kind in (0, 1):
        assert np.array_equal(_bits(held[kind]), _bits(t.pages[kind][1])), kind


def _job(row, n, position, kind, slot, token, cow=None, **more):
    job = {"first_row": row, "token_count": n, "position": position, "dst_kind": kind, "dst_slot": slot, "dst_token": token, **more}
    if cow:
        job.update(cow_kind=cow[0], cow_slot=cow[1], cow_tokens=cow[2])
    return job


FAR = (1 << 32) - 1
# Single tokens at every place of a micro page, copied tails, runs across groups of 8, whole pages, far positions, rows out of order.
JOBS = [_job(3, 1, 0, 0, 0, 0), _job(0, 1, 7, 0, 1, 7, (0, 2, 7)), _job(1, 1, 131071, 0, 3, 3, (0, 4, 2)), _job(2, 1, FAR, 0, 5, 5),
        _job(4, 8, 40, 0, 6, 0), _job(12, 5, 1000003, 0, 7, 3, (0, 8, 3)), _job(17, 64, 64, 1, 0, 0), _job(81, 17, 3, 1, 1, 6),
        _job(98, 30, FAR - 29, 1, 2, 34, (1, 3, 34)), _job(128, 0, 9, 0, 9, 4, (0, 10, 4)), _job(129, 3, 70000, 0, 11, 1)]


@pytest.mark.parametrize("heads,dim,group", [(4, 64, 8), (8, 128, 4), (1, 8, 1), (3, 96, 5), (2, 12, 2), (1, 256, 3)])
@pytest.mark.parametrize("adjacent", [0, 1])
@pytest.mark.parametrize("rotary", ["all", "half", "none", "two"])
def test_append_rope(dev, heads, dim, group, adjacent, rotary):
    rotary = {"all": dim, "half": dim // 2, "none": 0, "two": 2}[rotary]
    print(f"append_rope H={heads} D={dim} G={group} adjacent={adjacent} R={rotary}", flush=True)
    t = _Append(dev, heads, dim)
    _run_append(t, JOBS, 135, group, dev.Rope(10000.0, rotary, adjacent), layer=1)
    assert t.storage.faults() == (0, 0)


@pytest.mark.parametrize("form", ["no queries", "in place", "strides", "odd strides", "odd address", "stream"])
def test_append_rope_forms(dev, form):
    print(f"append_rope {form}", flush=True)
    t = _Append(dev, 4, 64)
    more = {"no queries": dict(q=None), "in place": dict(q="in place"), "strides": dict(stride_pad=24), "odd strides": dict(stride_pad=5),
            "odd address": dict(offset=3), "stream": dict(stream=dev.Stream() if form == "stream" else None)}[form]
    for rotary in (64, 32):
        _run_append(t, JOBS, 135, 8, dev.Rope(500000.0, rotary, rotary == 32), layer=0, **more)
    assert t.storage.faults() == (0, 0)


@pytest.mark.parametrize("tokens", [(6, 20), (12, 96), (1, 3)])
def test_append_rope_other_pages(dev, tokens):
    """Pages that are no multiple of 8 tokens, and ones of several 32-token blocks of V."""
    micro, extent = tokens
    print(f"append_rope pages of {tokens}", flush=True)
    t = _Append(dev, 2, 64, micro_tokens=micro, extent_tokens=extent)
    jobs = [_job(0, micro, 5, 0, 0, 0), _job(micro, 1, 99, 0, 1, micro - 1, (0, 2, micro - 1) if micro > 1 else None),
            _job(micro + 1, extent, 1000, 1, 0, 0), _job(micro + 1 + extent, extent - 2, 77, 1, 1, 2, (1, 2, 1))]
    _run_append(t, jobs, micro + 2 * extent, 4, dev.Rope(10000.0, 64, 0), layer=1)
    assert t.storage.faults() == (0, 0)


@pytest.mark.parametrize("heads,dim,group", [(4, 64, 8), (8, 128, 4), (2, 12, 2)])
def test_append_rope_fork_from_one_page(dev, heads, dim, group):
    """Requests leave one shared partial page, each with a copy of its own, while its last holder writes on behind what they
    copy; a micro page and an extent page, of which one goes on by a whole group of 8."""
    print(f"append_rope fork H={heads} D={dim}", flush=True)
    t = _Append(dev, heads, dim)
    jobs = [_job(i, 1, 5, 0, 1 + i, 5, (0, 0, 5)) for i in range(12)] + [_job(12, 1, 5, 0, 0, 5)]
    jobs += [_job(13, 1, 3, 0, 14, 3, (0, 0, 3)), _job(14, 2, 4, 0, 15, 4, (0, 0, 4))]
    jobs += [_job(16 + i, 1, 40, 1, 1 + i, 40, (1, 0, 40)) for i in range(3)] + [_job(19, 12, 40, 1, 0, 40), _job(31, 3, 37, 1, 4, 37, (1, 0, 37))]
    _run_append(t, jobs, 34, group, dev.Rope(10000.0, dim, 0), layer=1)
    assert t.storage.faults() == (0, 0)


def test_append_rope_equals_split_and_append_at_near_positions(dev):
    """What the rotation and the append do in two calls, to the angles' last bits."""
    heads, dim, group, rows = 4, 64, 8, 40
    t = _Append(dev, heads, dim, layers=1)
    rng = np.random.default_rng(8)
    qkv = _fp16(rng, rows, (group + 2) * heads * dim)
    pos = np.arange(rows, dtype=np.uint32)
    src, pbuf = dev.upload(_bits(qkv)), dev.upload(pos)
    q, k, v = (dev.DeviceBuffer(rows * n * dim * 2) for n in (group * heads, heads, heads))
    lib = dev.lib()
    lib.kimkv_model_rope_split.argtypes = [ctypes.c_void_p] * 2 + [ctypes.c_uint32] * 4 + [ctypes.c_float] + [ctypes.c_void_p] * 4
    dev.check(lib.kimkv_model_rope_split(src.ptr, pbuf.ptr, rows, group * heads, heads, dim, 10000.0, q.ptr, k.ptr, v.ptr, None), "rope")
    two = dev.download(k.ptr, (rows, heads, dim), np.uint16).view(np.float16).astype(np.float64)
    _run_append(t, [_job(0, rows, 0, 1, 0, 0)], rows, group, dev.Rope(10000.0, dim, 0), layer=0, seed=8)
    got = t.held()[1][0, 0, :rows].astype(np.float64)
    assert np.all(np.abs(got - two) <= 2 * FP16 * np.abs(two) + 1e-3)


@pytest.mark.parametrize("heads,dim,rotary", [(258, 128, 128), (1, 33024, 512)])
@pytest.mark.parametrize("adjacent", [0, 1])
def test_append_rope_past_32_bit_offsets(dev, heads, dim, rotary, adjacent):
    """Pages of 65528 tokens whose last heads' blocks, or last dims' V rows, begin more than 2^32 elements into the page: a
    prompt's rows, then a copied tail and the token after it."""
    print(f"append_rope huge H={heads} D={dim}", flush=True)
    storage = dev.Storage(1, heads, dim, 1, 2, 8, 65528)
    rng = np.random.default_rng(heads)
    qkv = _fp16(rng, 9, 3 * heads, dim)
    width = 3 * heads * dim
    src, q = dev.upload(_bits(qkv)), dev.upload(np.full((9, heads * dim), 0x1234, np.uint16))
    rope = dev.Rope(500000.0, rotary, adjacent)
    for job in [(0, 8, 70000, 0, 0, 0, 0, 1, 0, 0), (8, 1, 3, 1, 0, 5, 5, 1, 1, 0)]:
        table = dev.upload(np.array([job], dtype=dev.APPEND_ROPE_JOB))
        storage.append_rope_launch(table.ptr, 1, job[1], 0, src.ptr, width, 9, heads, rope, q.ptr, heads * dim)
        dev.sync()
    positions = np.array([*range(70000, 70008), 3], dtype=np.uint64)
    want, size = _rotate(qkv[:, :2 * heads], positions, 500000.0, rotary, adjacent)
    desc = lambda slot, n: np.array([(slot, 1, 0, n, 65528, 1)], dtype=helpers.DESC)  # noqa: E731
    held = storage.gather(desc(0, 8), 8).view(np.float16).reshape(2, 8, heads, dim)
    _near(held[0], want[:8, heads:], size[:8, heads:], positions[:8])
    assert np.array_equal(_bits(held[1]), _bits(qkv[:8, 2 * heads:]))
    fork = storage.gather(desc(1, 6), 6).view(np.float16).reshape(2, 6, heads, dim)
    assert np.array_equal(_bits(fork[:, :5]), _bits(held[:, :5]))
    _near(fork[0, 5:], want[8:, heads:], size[8:, heads:], positions[8:])
    assert np.array_equal(_bits(fork[1, 5]), _bits(qkv[8, 2 * heads:]))
    got = dev.download(q.ptr, (9, heads, dim), np.uint16).view(np.float16)
    _near(got, want[:, :heads], size[:, :heads], positions)
    assert storage.faults() == (0, 0)


def test_append_rope_rows_and_pages_far_away(dev):
    """Rows, queries and pages more than 2^32 elements from the start of their buffers, then attention to those pages."""
    heads, dim, group, stride, pages = 8, 128, 4, (1 << 30) + 8, 40000
    qh = heads * group
    storage = dev.Storage(1, heads, dim, 8, pages)   # 131072 elements a page
    rng = np.random.default_rng(31)
    # Row 5 is a token, rows 0..4 are not named.  The pages' other tokens come from plain rows, unrotated.
    far, q = dev.DeviceBuffer(6 * stride * 2), dev.DeviceBuffer(6 * stride * 2)
    row = _fp16(rng, qh + 2 * heads, dim)
    dev.copy_to_device(far.ptr + 2 * 5 * stride, _bits(row))
    lanes, prefix, slots = 2, 128, [[pages - 1, pages - 5, pages - 2], [pages - 1, pages - 5, pages - 3]]
    known = {slot: _fp16(rng, 64, qh + 2 * heads, dim) for slot in sorted({s for t in slots for s in t})}
    jobs = np.zeros(1, dtype=dev.APPEND_ROPE_JOB)
    for slot, x in known.items():
        src = dev.upload(_bits(x))
        jobs[0] = (0, 64, 0, slot, 0, 0, 0, 1, 0, 0)
        table = dev.upload(jobs)
        storage.append_rope_launch(table.ptr, 1, 64, 0, src.ptr, (qh + 2 * heads) * dim, 64, qh, dev.Rope(10000.0, 0, 0), 0, 0)
        dev.sync()
    rope, tokens = dev.Rope(10000.0, dim, 0), prefix + 40
    jobs[0] = (5, 1, tokens - 1, slots[1][2], 0, (tokens - 1) % 64, 0, 1, 0, 0)
    table = dev.upload(jobs)
    storage.append_rope_launch(table.ptr, 1, 1, 0, far.ptr, stride, 6, qh, rope, q.ptr, stride)
    dev.sync()
    want, size = _rotate(row[None, :qh + heads], np.array([tokens - 1], np.uint64), 10000.0, dim, 0)
    query = dev.download(q.ptr + 2 * 5 * stride, (qh, dim), np.uint16).view(np.float16)
    _near(query[None], want[:, :qh], size[:, :qh], np.array([tokens - 1], np.uint64))
    tables = [np.array([(s, 1, 64 * i, min(64, tokens - 64 * i), 64, 1) for i, s in enumerate(t)], dtype=dev.BLOCK_DESC) for t in slots]
    held = [storage.gather(t, tokens).view(np.float16).reshape(2, tokens, heads, dim) for t in tables]
    _near(held[1][0, -1:], want[:, qh:], size[:, qh:], np.array([tokens - 1], np.uint64))
    assert np.array_equal(_bits(held[1][1, -1]), _bits(row[qh + heads:]))
    for i in range(lanes):   # everything but the far token is as it was written
        for part in range(2):
            plain = np.concatenate([known[s][:, qh + part * heads:qh + (part + 1) * heads] for s in slots[i]])[:tokens - i]
            assert np.array_equal(_bits(held[i][part, :tokens - i]), _bits(plain))
    out = dev.upload(np.full((lanes, qh, dim), 0x1234, np.uint16))
    on_gpu = [dev.upload(t) for t in tables]
    items = np.zeros(lanes, dtype=dev.DECODE_ITEM)
    for i in range(lanes):
        items[i] = (on_gpu[i].ptr, len(tables[i]), tokens, 0, q.ptr + 2 * 5 * stride, 0, out.ptr + 2 * i * qh * dim, 1.0 / math.sqrt(dim))
    entries, plan = dev.shared_decode_plan(heads, dim, qh, 1, [tokens] * lanes, [(0, lanes, prefix)])
    buf, entries_buf, work = dev.upload(items), dev.upload(entries), dev.DeviceBuffer(max(16, plan.workspace_bytes))
    storage.shared_decode_launch(buf.ptr, entries_buf.ptr, plan, work.ptr)
    dev.sync()
    got = dev.download(out.ptr, (lanes, qh, dim), np.uint16).view(np.float16)
    for i in range(lanes):
        want, bound = reference(query, held[i][0], held[i][1], 1.0 / math.sqrt(dim))
        assert np.all(np.abs(got[i].astype(np.float64) - want) <= bound)
    assert storage.faults() == (0, 0)


def test_append_rope_faults(dev):
    """Jobs that name what is not there are reported and change nothing; the good one beside them runs."""
    t = _Append(dev, 4, 64)
    rope = dev.Rope(10000.0, 64, 0)
    bad = [_job(0, 1, 0, 0, 24, 0), _job(0, 1, 0, 1, 6, 0), _job(0, 1, 0, 2, 0, 0), _job(0, 1, 0, 0, 0, 8), _job(0, 2, 0, 0, 0, 7),
           _job(0, 9, 0, 0, 0, 0), _job(10, 1, 0, 0, 0, 0), _job(9, 2, 0, 0, 0, 0), _job(FAR, 2, 0, 0, 0, 0), _job(0, 2, FAR, 0, 0, 0),
           _job(0, 1, 0, 0, 0, 3, (0, 24, 2)), _job(0, 1, 0, 0, 0, 3, (0, 1, 4)), _job(0, 1, 0, 1, 0, 20, (0, 1, 9)), _job(0, 1, 0, 0, 0, 3, (7, 1, 1)),
           _job(0, 0xFFFFFFFF, 0, 1, 0, 1), _job(0, 9, 0, 1, 0, 0)]
    for j in bad:
        j["bad"] = True
        print("append_rope fault", j, flush=True)
        _run_append(t, [j, _job(3, 2, 50, 0, 20, 1)], 10, 8, rope, layer=1, max_tokens=8)
        assert t.storage.faults() == (dev.INVALID_ARGUMENT, dev.FAULT_APPEND_JOB)
    assert t.storage.faults() == (0, 0)


def test_append_rope_refusals(dev):
    t = _Append(dev, 4, 64)
    lib, buf = dev.lib(), dev.DeviceBuffer(1 << 20)
    width = 40 * 64

    def status(storage=t.storage.h, jobs=buf.ptr, count=1, layer=1, qkv=buf.ptr, stride=width, rows=4, qh=32, rope=(10000.0, 64, 0), q=buf.ptr,
               q_stride=32 * 64):
        return lib.kimkv_append_rope_batch(storage, jobs, count, 1, layer, qkv, stride, rows, qh, dev.Rope(*rope) if rope else None, q, q_stride,
                                           None)

    for bad in (dict(jobs=None), dict(qkv=None), dict(layer=2), dict(stride=width - 1), dict(rope=None), dict(rope=(0.0, 64, 0)),
                dict(rope=(float("nan"), 64, 0)), dict(rope=(float("inf"), 64, 0)), dict(rope=(10000.0, 63, 0)), dict(rope=(10000.0, 66, 0)),
                dict(q_stride=32 * 64 - 1), dict(qh=0), dict(stride=1 << 62), dict(q_stride=1 << 62), dict(count=1 << 31), dict(qh=0xFFFFFFFF)):
        assert status(**bad) == dev.INVALID_ARGUMENT, bad
    assert status(count=0) == dev.OK and status(count=0, jobs=None, qkv=None) == dev.OK


# ---- shared decode -----------------------------------------------------------


class _Batch:
    """Lanes on a storage; keys and values of each as a plain form reads them."""

    def __init__(self, dev, heads, dim, group, counts, groups, layers=1, layer=0, seed=3, micro_tokens=8, extent_tokens=64, pages="hetero",
                 q_scale=2.0, spread=None):
        self.dev, self.heads, self.dim, self.group, self.counts, self.groups, self.layer = dev, heads, dim, group, counts, groups, layer
        rng = np.random.default_rng(seed)
        total = sum(counts) + sum(p for _, _, p in groups)
        unit = min(micro_tokens, extent_tokens)
        short = micro_tokens if pages != "ragged" else max(1, micro_tokens - 2)
        slots = total // short + 4 * len(counts) + 16, total // unit + len(counts) + 8
        self.storage = dev.Storage(layers, heads, dim, *slots, micro_tokens, extent_tokens)
        alloc = helpers.SlotAllocator(*slots, seed=seed)
        self.k, self.v, self.tables, keep = [], [], [], []
        shared = {}
        for first, n, prefix in groups:
            for i in range(first, first + n):
                shared[i] = (first, prefix)
        caps = (micro_tokens, extent_tokens)
        for i, t in enumerate(counts):
            first, prefix = shared.get(i, (i, 0))
            k, v = _fp16(rng, t, heads, dim), _fp16(rng, t, heads, dim)
            if spread is not None:
                spread(rng, i, k, v)
            table, begin = [], 0
            if first != i:
                same = min(prefix, t)
                k[:same], v[:same] = self.k[first][:same], self.v[first][:same]
                for e in self.tables[first]:   # pages wholly inside the prefix
                    if e[2] + e[3] <= same and e[3] == e[4] and e[2] == begin:
                        table.append(e)
                        begin += e[3]
            while begin < t:
                kind = 1 if pages == "extents" or (pages == "hetero" and begin % extent_tokens == 0 and t - begin >= extent_tokens) else 0
                n = min(caps[kind], t - begin)
                if pages == "ragged" and begin % 3 == 0:
                    n = min(n, max(1, caps[kind] - 1 - begin % 2))
                table.append((alloc.take(kind), 1, begin, n, caps[kind], kind))
                begin += n
            self.k.append(k)
            self.v.append(v)
            self.tables.append(table)
            self._write(table, k, v)
        self.query = _fp16(rng, len(counts), heads * group, dim, scale=q_scale)
        self.scale = np.full(len(counts), 1.0 / math.sqrt(dim), dtype=np.float32)

    def _write(self, table, k, v):
        dev, row = self.dev, self.heads * self.dim
        kb, vb = dev.upload(_bits(k)), dev.upload(_bits(v))
        jobs = np.zeros(len(table), dtype=dev.APPEND_JOB)
        for j, e in enumerate(table):
            jobs[j] = (kb.ptr + 2 * e[2] * row, vb.ptr + 2 * e[2] * row, 0, row, self.layer, 1, e[3], e[0], 0, 0, 0, e[5], 0)
        self.storage.append_batch(jobs)

    def place(self, q_off=0, change=None):
        """Items on the GPU; `change(items)` may spoil them."""
        dev, n, qd = self.dev, len(self.counts), self.heads * self.group * self.dim
        self.q_buf = dev.upload(np.concatenate([np.zeros(q_off, np.uint16), _bits(self.query).reshape(-1)]))
        self.out = dev.upload(np.full(n * qd + 64, 0x1234, np.uint16))
        self.tab = [dev.upload(np.array(t, dtype=dev.BLOCK_DESC)) if t else None for t in self.tables]
        items = np.zeros(n, dtype=dev.DECODE_ITEM)
        for i, t in enumerate(self.counts):
            items[i] = (self.tab[i].ptr if t else 0, len(self.tables[i]), t, self.layer, self.q_buf.ptr + 2 * (q_off + i * qd), 0,
                        self.out.ptr + 2 * i * qd, self.scale[i])
        if change is not None:
            change(items)
        self.items = dev.upload(items)

    def plan(self, units=4):
        """A plan for a device of `units` compute units: on a small one every shared prefix pays, however short."""
        self.entries, self.p = self.dev.shared_decode_plan(self.heads, self.dim, self.heads * self.group, units, self.counts, self.groups)
        self.entries_buf = self.dev.upload(self.entries)
        # Bytes around the workspace are looked at afterwards.
        self.work = self.dev.upload(np.full(self.p.workspace_bytes + 4096, 0x5A, np.uint8))

    def launch(self, stream=None):
        self.storage.shared_decode_launch(self.items.ptr, self.entries_buf.ptr, self.p, self.work.ptr + 2048, stream)
        self.dev.sync(stream)

    def outputs(self):
        n, qd = len(self.counts), self.heads * self.group * self.dim
        got = self.dev.download(self.out.ptr, (n * qd + 64,), np.uint16)
        assert np.all(got[n * qd:] == 0x1234)
        edge = self.dev.download(self.work.ptr, (self.p.workspace_bytes + 4096,), np.uint8)
        assert np.all(edge[:2048] == 0x5A) and np.all(edge[2048 + self.p.workspace_bytes:] == 0x5A)
        return got[:n * qd].reshape(n, self.heads * self.group, self.dim)

    def check(self, got, lanes=None):
        for i in range(len(self.counts)) if lanes is None else lanes:
            if self.counts[i] == 0:
                assert np.all(got[i] == 0x1234), i
                continue
            want, bound = reference(self.query[i], self.k[i], self.v[i], float(self.scale[i]))
            err = np.abs(got[i].view(np.float16).astype(np.float64) - want)
            assert np.all(err <= bound), (i, self.counts[i], float((err / bound).max()))


def reference(query, k, v, scale):
    """One lane's attention in 64 bits and how far fp16 outputs may be from it.  A score is a 32-bit sum of D exact
    products times a 32-bit scale: within (D + 4) 2^-24 of the sum of their sizes; twice that, natural, is a weight's and its
    share of the denominator's relative error.  Exponentials are within 2^-21, weights are handed on within 2^-20, and the
    sums over n keys, in blocks of at least 8 and merged at most 64 times, within (n / 8 + 72) 2^-24.  Together with the
    denominator's twice, relative to the weighted sizes of V; and the output is rounded to fp16."""
    qh, dim = query.shape
    heads = k.shape[1]
    q = query.astype(np.float64).reshape(heads, qh // heads, dim)
    want, bound = np.empty((heads, qh // heads, dim)), np.empty((heads, qh // heads, dim))
    for h in range(heads):
        kk, vv = k[:, h].astype(np.float64), v[:, h].astype(np.float64)
        s = (q[h] @ kk.T) * scale
        size = (np.abs(q[h]) @ np.abs(kk).T) * abs(scale)
        p = np.exp(s - s.max(-1, keepdims=True))
        p /= p.sum(-1, keepdims=True)
        want[h] = p @ vv
        rel = 2 * (dim + 4) * 2.0 ** -24 * size + 2.0 ** -21 + 2.0 ** -20 + (len(kk) / 8 + 72) * 2.0 ** -24
        bound[h] = FP16 * np.abs(want[h]) + TINY + (p * rel) @ np.abs(vv) + (p * rel).sum(-1, keepdims=True) * (p @ np.abs(vv))
    return want.reshape(qh, dim), bound.reshape(qh, dim)


BATCHES = {
    "one token": ([1], []),
    "alone": ([1, 63, 64, 65, 700, 1500], []),
    "pair": ([500, 513], [(0, 2, 497)]),
    "prefix is all": ([128, 128, 200], [(0, 3, 128)]),
    "short lane in a group": ([900, 70, 901], [(0, 3, 890)]),
    "empty lanes": ([0, 300, 0, 310, 0], [(1, 1, 300), (3, 1, 300)]),
    "empty lane in a group": ([300, 0, 310], [(0, 3, 256)]),
    "many": ([1030 + 7 * i for i in range(33)], [(0, 33, 1030)]),
    "more": ([400 + i % 50 for i in range(70)], [(0, 70, 390)]),
    "two groups and alone": ([700, 701, 800, 2100, 2070, 2300, 90, 2111], [(0, 3, 690), (3, 3, 2065)]),
    "long prefix is all": ([2048, 2048, 2500, 40, 0], [(0, 3, 2048), (3, 2, 40)]),
    "shorter lane in a long group": ([5000, 3001, 5003], [(0, 3, 4990)]),
    "long": ([5200, 5000, 4990, 9000], [(0, 3, 4985)]),
}


def _kinds(b):
    """How the plan's units are computed: (blocks of columns and flags, whether they hold several lanes' columns)."""
    units = b.entries[:b.p.unit_count * UNIT.itemsize].view(UNIT)
    return {(int(u["kind"]) & 0x7F, bool(u["cols"] > b.group)) for u in units if u["cols"]}


@pytest.mark.parametrize("name", list(BATCHES))
@pytest.mark.parametrize("heads,dim,group", [(4, 64, 8), (8, 128, 4), (2, 64, 16)])
@pytest.mark.parametrize("units", [4, 256])
def test_shared_decode(dev, name, heads, dim, group, units):
    print(f"shared {name} H={heads} D={dim} G={group} units={units}", flush=True)
    b = _Batch(dev, heads, dim, group, *BATCHES[name])
    b.place()
    b.plan(units)
    b.launch()
    first = b.outputs()
    b.check(first)
    b.launch()
    assert np.array_equal(first, b.outputs()), "the same plan gives the same bits"
    assert b.storage.faults() == (0, 0)


@pytest.mark.parametrize("heads,dim,lanes,kind", [(2, 64, 2, 1), (2, 64, 4, 2), (2, 64, 8, 4), (1, 64, 25, 4), (1, 64, 70, 4), (2, 96, 2, 1),
                                                  (2, 96, 9, 2), (2, 128, 2, 1), (2, 128, 5, 2), (1, 128, 17, 2), (1, 128, 40, 2)])
@pytest.mark.parametrize("prefix", [64, 130, 2000, 9000])
def test_shared_decode_every_kind(dev, heads, dim, lanes, kind, prefix):
    """Groups of few and of many columns, which are computed differently, on prefixes of one block of 64 to several pieces."""
    print(f"shared kind {kind} H={heads} D={dim} lanes={lanes} prefix={prefix}", flush=True)
    b = _Batch(dev, heads, dim, 8, [prefix + 1 + 3 * i for i in range(lanes)], [(0, lanes, prefix)])
    b.place()
    b.plan(1)
    assert (kind, True) in _kinds(b) or prefix < 2000   # short ones may not pay
    b.launch()
    b.check(b.outputs())
    assert b.storage.faults() == (0, 0)


@pytest.mark.parametrize("heads,dim,group", [(4, 64, 8), (2, 128, 4), (2, 80, 3)])
@pytest.mark.parametrize("empty", [[0], [6], [11], [0, 1, 4, 5, 10, 11], [2, 3, 4, 5]])
def test_shared_decode_empty_lanes_in_a_group(dev, heads, dim, group, empty):
    """Ended requests and padding in a group: the others share its prefix, and nothing is written or reported for these,
    whatever their items hold."""
    print(f"shared empty {empty} H={heads} D={dim}", flush=True)
    prefix = 2000

    def spoil(items):
        items["layer"][empty] = 7
        items["token_count"][empty[-1]] = 5

    first = min(set(range(12)) - set(empty))
    b = _Batch(dev, heads, dim, group, [0 if i in empty else prefix + 3 * i for i in range(12)], [(first, 12 - first, prefix)])
    b.groups = [(0, 12, prefix)]
    b.place(change=spoil)
    b.plan(1)
    assert any(wide for _, wide in _kinds(b))
    b.launch()
    b.check(b.outputs())
    assert b.storage.faults() == (0, 0)


@pytest.mark.parametrize("heads,dim", [(1, 64), (2, 128), (3, 96)])
@pytest.mark.parametrize("units", [24, 256])
def test_shared_decode_wide_group(dev, heads, dim, units):
    """Columns of one head and key range that are more than an XCD computes at once, on several of them."""
    print(f"shared wide H={heads} D={dim} units={units}", flush=True)
    b = _Batch(dev, heads, dim, 8, [640 + i % 40 for i in range(270)], [(0, 270, 640)])
    b.place()
    b.plan(units)
    assert units == 256 or any(wide for _, wide in _kinds(b))   # a large device may read so little lane by lane
    b.launch()
    b.check(b.outputs())
    assert b.storage.faults() == (0, 0)


@pytest.mark.parametrize("heads,dim,lanes,kind", [(2, 64, 2, 1), (2, 64, 4, 2), (4, 64, 8, 4), (3, 96, 4, 2), (2, 128, 5, 2), (1, 128, 2, 1)])
@pytest.mark.parametrize("own", [40, 4500])
def test_shared_decode_workgroups(dev, heads, dim, lanes, kind, own):
    """Workgroups of many waves where prefixes are most of the work, of few where the lanes' own tokens are; units of
    several segments in both."""
    print(f"shared workgroups H={heads} D={dim} lanes={lanes} own={own}", flush=True)
    b = _Batch(dev, heads, dim, 8, [4200 + own + 30 * i for i in range(lanes)], [(0, lanes, 4200)])
    b.place()
    b.plan(1)
    assert (kind, True) in _kinds(b)
    assert b.p.waves == (8 if own == 40 else 4)
    b.launch()
    b.check(b.outputs())
    assert b.storage.faults() == (0, 0)


@pytest.mark.parametrize("heads,dim,group", [(1, 64, 8), (2, 128, 3), (1, 30, 2), (1, 96, 16)])
@pytest.mark.parametrize("units,split", [(12, 1), (40, 2), (64, 4), (2000, 4)])
def test_shared_decode_many_parts(dev, heads, dim, group, units, split):
    """Lanes cut into many parts, beside short ones, on a plan for a device with more compute units than this one."""
    print(f"shared parts H={heads} D={dim} units={units}", flush=True)
    b = _Batch(dev, heads, dim, group, [13000, 12500, 12460, 70, 5], [(0, 3, 12400)])
    b.place()
    b.plan(units)
    assert b.p.merge_split >= split or dim == 30
    b.launch()
    b.check(b.outputs())
    assert b.storage.faults() == (0, 0)


@pytest.mark.parametrize("heads,dim,group", [(1, 64, 1), (3, 64, 5), (2, 96, 3), (1, 128, 40), (5, 64, 2), (2, 32, 4), (1, 8, 2), (2, 200, 1),
                                             (1, 256, 7), (2, 12, 3), (1, 64, 33)])
@pytest.mark.parametrize("more", [0, 2000])
def test_shared_decode_other_shapes(dev, heads, dim, group, more):
    print(f"shared H={heads} D={dim} G={group} more={more}", flush=True)
    b = _Batch(dev, heads, dim, group, [330 + more, 400 + more, 345 + more, 12], [(0, 3, 321 + more)], layers=2, layer=1)
    b.place()
    b.plan(1 if more else 4)
    b.launch()
    b.check(b.outputs())
    assert b.storage.faults() == (0, 0)


@pytest.mark.parametrize("pages,micro,extent", [("ragged", 8, 64), ("micro", 6, 48), ("micro", 8, 64), ("hetero", 16, 128), ("extents", 8, 96),
                                                ("micro", 1, 8)])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("lanes", [3, 50])
def test_shared_decode_other_pages(dev, pages, micro, extent, dim, lanes):
    """Tables off the 8-token grid, pages that end inside a tile, pages of other sizes."""
    print(f"shared pages {pages} {micro} {extent} D={dim} lanes={lanes}", flush=True)
    b = _Batch(dev, 2, dim, 4, [600 + 7 * i for i in range(lanes)] + [77], [(0, lanes, 590)], pages=pages, micro_tokens=micro, extent_tokens=extent)
    b.place()
    b.plan()
    b.launch()
    b.check(b.outputs())
    assert b.storage.faults() == (0, 0)


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("lanes", [3, 40])
def test_shared_decode_hole(dev, lanes, dim):
    """A table with a page missing: its keys are not there for any lane, in the prefix as in a lane's own tokens."""
    b = _Batch(dev, 2, dim, 4, [700 + i for i in range(lanes)], [(0, lanes, 690)])
    for i in range(lanes):
        keep = [e for e in b.tables[i] if not e[2] <= 200 < e[2] + e[3]]
        gone = [e for e in b.tables[i] if e[2] <= 200 < e[2] + e[3]]
        if i % 2:
            gone.append(keep.pop())
        there = np.ones(b.counts[i], dtype=bool)
        for e in gone:
            there[e[2]:e[2] + e[3]] = False
        b.tables[i] = keep
        b.k[i], b.v[i] = b.k[i][there], b.v[i][there]
    b.place()
    b.plan()
    b.launch()
    b.check(b.outputs())


@pytest.mark.parametrize("dim", [64, 128])
def test_shared_decode_scales_and_addresses(dev, dim):
    """Lanes of one group with scales of their own (one negative, one zero), and queries off the vectors' alignment."""
    for off in (0, 1):
        b = _Batch(dev, 2, dim, 8, [1500 + i for i in range(20)], [(0, 20, 1490)])
        b.scale = np.array([0.01 * (i + 1) for i in range(20)], dtype=np.float32)
        b.scale[3], b.scale[7] = -0.1, 0.0
        b.place(q_off=off)
        b.plan()
        assert ({64: 4, 128: 2}[dim], True) in _kinds(b)
        b.launch()
        b.check(b.outputs())


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("lanes", [2, 24])
def test_shared_decode_large_scores(dev, dim, lanes):
    """Scores of hundreds that rise along the prefix, so that the running maximum moves all the way, and ones so far
    below it that they weigh nothing."""
    def spread(rng, i, k, v):
        k *= np.linspace(0.1, 6.0, len(k)).astype(np.float16)[:, None, None]

    b = _Batch(dev, 2, dim, 8, [1000 + i for i in range(lanes)], [(0, lanes, 960)], q_scale=6.0, spread=spread)
    b.place()
    b.plan()
    b.launch()
    b.check(b.outputs())


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("lanes", [2, 24])
@pytest.mark.parametrize("where", ["prefix", "own"])
def test_shared_decode_nonfinite_values(dev, dim, lanes, where):
    """Infinite V of a key that every lane sees is infinite in the output; at a key of weight 0 it is left out."""
    t = 100 if where == "prefix" else 520

    def spread(rng, i, k, v):
        v[t, 0, 3] = np.inf
        v[t + 1, 1, 5] = -np.inf
        k[t + 1] = 0   # raised below to a score of far under the others

    b = _Batch(dev, 2, dim, 4, [600 + i for i in range(lanes)], [(0, lanes, 512)], spread=spread, q_scale=1.0)
    # A key whose score is lowest by far for every query: minus 60000 along dim 0, queries all positive there.
    b.query[:, :, 0] = 4.0
    for i in range(lanes):
        b.k[i][t + 1] = 0
        b.k[i][t + 1, :, 0] = -60000.0
        b._write(b.tables[i], b.k[i], b.v[i])
    b.place()
    b.plan()
    b.launch()
    got = b.outputs().view(np.float16)
    assert np.all(np.isposinf(got[:, :4, 3]))
    assert np.all(np.isfinite(got[:, 4:]))
    clean = [x.copy() for x in b.v]
    for x in clean:
        x[t, 0, 3] = 0
        x[t + 1, 1, 5] = 0
    b.v = clean
    for i in range(lanes):
        want, bound = reference(b.query[i], b.k[i], b.v[i], float(b.scale[i]))
        ok = np.abs(got[i].astype(np.float64) - want) <= bound
        ok[:4, 3] = True
        assert np.all(ok), i


def test_shared_decode_all_scores_minus_infinity(dev):
    """Keys of minus infinity: no weight anywhere gives 0, some weight that of the rest."""
    for dim in (64, 128):
        def spread(rng, i, k, v):
            k[:, 0, 0] = -np.inf
            k[:320, 1, 0] = -np.inf

        b = _Batch(dev, 2, dim, 4, [400, 390, 380], [(0, 3, 320)], spread=spread)
        b.query[:, :, 0] = np.abs(b.query[:, :, 0]) + np.float16(0.5)
        b.place()
        b.plan()
        b.launch()
        got = b.outputs().view(np.float16)
        assert np.all(got[:, :4] == 0)
        for i in range(3):
            want, bound = reference(b.query[i, 4:], b.k[i][320:, 1:], b.v[i][320:, 1:], float(b.scale[i]))
            assert np.all(np.abs(got[i, 4:].astype(np.float64) - want) <= bound)


@pytest.mark.parametrize("dim", [64, 128, 80])
@pytest.mark.parametrize("lanes,prefix,units", [(3, 960, 4), (24, 960, 4), (2, 13000, 2000)])
@pytest.mark.parametrize("where", ["query", "one key", "first keys", "prefix", "own key"])
def test_shared_decode_nan_scores(dev, dim, lanes, prefix, units, where):
    """A score that is NaN makes its row NaN wherever its key lies, also where a step, a unit or a whole part has no other
    score; rows without one are as they should be."""
    print(f"shared NaN {where} D={dim} lanes={lanes} prefix={prefix}", flush=True)
    keys = {"query": (0, 0), "one key": (70, 71), "first keys": (0, 64), "prefix": (0, prefix), "own key": (prefix, prefix + 1)}[where]

    def spread(rng, i, k, v):
        k[keys[0]:keys[1], 1, 3] = np.nan

    b = _Batch(dev, 2, dim, 4, [prefix + 1 + i for i in range(lanes)], [(0, lanes, prefix)], spread=spread, q_scale=1.0)
    bad = np.zeros((lanes, 8), dtype=bool)
    if where == "query":
        b.query[1, 2, 5] = np.nan
        bad[1, 2] = True
    else:
        bad[:, 4:] = True
    b.place()
    b.plan(units)
    b.launch()
    got = b.outputs().view(np.float16)
    assert np.all(np.isnan(got[bad]))
    for i in range(lanes):
        query, k = np.nan_to_num(b.query[i]), np.nan_to_num(b.k[i])
        want, bound = reference(query, k, b.v[i], float(b.scale[i]))
        ok = np.abs(got[i].astype(np.float64) - want) <= bound
        assert np.all(ok[~bad[i]]), i


@pytest.mark.parametrize("dim", [64, 128, 80])
@pytest.mark.parametrize("low,prefix,units", [(64, 960, 4), (960, 960, 4), (500, 30000, 2000), (30000, 30000, 2000)])
def test_shared_decode_infinite_value_overtaken(dev, dim, low, prefix, units):
    """An infinite V of a key that outweighs all keys before it and weighs nothing beside those behind it is left out, as
    where it weighs nothing from the start."""
    print(f"shared overtaken D={dim} low={low} prefix={prefix}", flush=True)

    def spread(rng, i, k, v):
        k[:low, :, 0] = -60000.0
        v[3, 0, 5], v[40, 1, 7] = np.inf, -np.inf

    b = _Batch(dev, 2, dim, 4, [prefix + 50, prefix + 9], [(0, 2, prefix)], spread=spread, q_scale=1.0)
    b.query[:, :, 0] = 4.0
    b.place()
    b.plan(units)
    b.launch()
    for v in b.v:
        v[3, 0, 5] = v[40, 1, 7] = 0
    b.check(b.outputs())


def test_shared_decode_two_at_once(dev):
    """Two launches of one plan on two streams, each with a workspace and outputs of its own, and one on the first's
    stream again."""
    streams = [dev.Stream(), dev.Stream()]
    batches = [_Batch(dev, 4, 64, 8, [6000 + i for i in range(12)], [(0, 12, 5990)], seed=3 + i) for i in range(2)]
    for b in batches:
        b.place()
        b.plan(256)
        assert b.p.merge_lanes == 12
    for k in (0, 1, 0, 1):
        b = batches[k]
        b.storage.shared_decode_launch(b.items.ptr, b.entries_buf.ptr, b.p, b.work.ptr + 2048, streams[k])
    for stream, b in zip(streams, batches):
        stream.synchronize()
        b.check(b.outputs())
        stream.destroy()


def test_shared_decode_without_groups(dev):
    """The same batch with its groups and without them."""
    b = _Batch(dev, 4, 64, 8, *BATCHES["two groups and alone"])
    b.place()
    b.plan(1)
    b.launch()
    with_groups = b.outputs()
    b.check(with_groups)
    b.groups = []
    b.plan()
    b.launch()
    b.check(b.outputs())


def test_shared_decode_faults(dev):
    """A lane that is not as planned is reported and left alone, with its group where it is the group's first; the others
    come out as they should."""
    counts, groups = [2700, 2710, 2720, 2730, 300, 5], [(0, 2, 2690), (2, 2, 2690)]

    def spoil(lane, field, value):
        def change(items):
            items[lane][field] = value
        return change

    fields = [("query", 0), ("output", 0), ("descriptors", 0), ("descriptor_count", 0), ("token_count", 600), ("token_count", 0), ("layer", 7)]
    for lane, field, value in [(lane, *f) for lane in (0, 1, 4) for f in fields] + [(1, "layer", 1)]:
        print(f"shared fault lane {lane} {field}={value}", flush=True)
        b = _Batch(dev, 2, 64, 4, counts, groups, layers=2)
        b.place(change=spoil(lane, field, value))
        b.plan()
        assert (1, True) in _kinds(b)
        b.launch()
        got = b.outputs()
        gone = [lane] if lane else [0, 1]
        assert b.storage.faults() == (dev.INVALID_ARGUMENT, dev.FAULT_DECODE_ITEM)
        b.check(got, [i for i in range(6) if i not in gone])
        assert np.all(got[gone] == 0x1234)


def test_shared_decode_bad_entries(dev):
    """Entries that name what is not there are reported, not run: every index is checked against the launch's buffers."""
    counts, groups = [2700, 2710, 2720], [(0, 3, 2690)]
    for field, value in (("table_lane", 3), ("lane", 3), ("col0", 4), ("cols", 13), ("lane", 0xFFFFFFFF), ("col0", 0xFFFFFFFF), ("cols", 0xFFFFFFFF),
                         ("end", 1 << 20), ("begin", 1 << 20), ("slot", 1 << 20), ("slot", 0xFFFFFFFF), ("head", 2), ("heads", 3), ("heads", 0)):
        print(f"shared entry {field}={value}", flush=True)
        b = _Batch(dev, 2, 64, 4, counts, groups)
        b.place()
        b.plan(1)
        entries = b.entries.copy()
        units = entries[:b.p.unit_count * UNIT.itemsize].view(UNIT)
        at = [i for i in range(len(units)) if units[i]["cols"] > 4][0]   # 12 columns: three lanes
        units[at][field] = value
        b.entries_buf = dev.upload(entries)
        b.launch()
        b.outputs()
        assert b.storage.faults() == (dev.INVALID_ARGUMENT, dev.FAULT_DECODE_ITEM)
    for field, value in (("prefix_slot", 1 << 20), ("tail_slot", 0xFFFFFFFF), ("prefix_count", 1 << 20), ("tail_count", 1 << 20),
                         ("table_lane", 9)):
        print(f"shared record {field}={value}", flush=True)
        b = _Batch(dev, 2, 64, 4, counts, groups)
        b.place()
        b.plan(1)
        entries = b.entries.copy()
        entries[b.p.unit_count * UNIT.itemsize:].view(LANE)[1][field] = value
        b.entries_buf = dev.upload(entries)
        b.launch()
        got = b.outputs()
        assert np.all(got[1] == 0x1234)
        b.check(got, [0, 2])
        b.storage.faults()


def test_shared_decode_refusals(dev):
    b = _Batch(dev, 2, 64, 4, [2700, 2710, 2720], [(0, 3, 2690)])
    b.place()
    b.plan(1)
    lib = dev.lib()

    def status(storage=b.storage.h, items=b.items.ptr, entries=b.entries_buf.ptr, work=b.work.ptr + 2048, **fields):
        plan = dev.SharedPlan.from_buffer_copy(b.p)
        for name, value in fields.items():
            setattr(plan, name, value)
        return lib.kimkv_shared_decode_batch(storage, items, entries, plan, work, None)

    for bad in (dict(items=None), dict(entries=None), dict(work=None), dict(entries=b.entries_buf.ptr + 4), dict(work=b.work.ptr + 2052),
                dict(kv_heads=4), dict(head_dim=128), dict(query_heads=16), dict(query_heads=7), dict(query_heads=0), dict(lane_count=2),
                dict(lane_count=0), dict(unit_count=b.p.unit_count + 1), dict(slot_count=b.p.slot_count + 1), dict(entry_bytes=0),
                dict(workspace_bytes=0), dict(merge_split=0), dict(merge_split=3), dict(merge_split=16), dict(waves=0), dict(waves=6)):
        assert status(**bad) == dev.INVALID_ARGUMENT, bad
    assert lib.kimkv_shared_decode_batch(b.storage.h, None, None, None, None, None) == dev.INVALID_ARGUMENT
    other = dev.Storage(1, 4, 64, 8, 2)
    assert status(storage=other.h) == dev.INVALID_ARGUMENT
    assert np.all(b.outputs() == 0x1234)


# ---- logits ------------------------------------------------------------------


def _adjust_reference(row, rule):
    """(adjusted row in 64 bits, how far 32-bit values may be from it, allowed).  Each of the operations rounds its
    result by at most 2^-24 of it."""
    x = row.astype(np.float64)
    bound = np.zeros_like(x)
    half = 2.0 ** -24
    history = rule["history"][rule["history"] < len(x)]
    count = np.bincount(history.astype(np.int64), minlength=len(x)).astype(np.float64)
    r, f, p = (float(np.float32(rule[k])) for k in ("repetition", "frequency", "presence"))
    seen = count > 0
    with np.errstate(invalid="ignore", over="ignore"):
        turned = np.where(x > 0, x / r, x * r)
        less = f * count + p
        y = np.where(seen, turned - less, x)
        bound = np.where(seen, half * 2 * (np.abs(turned) + 2 * np.abs(less) + np.abs(f * count) + np.abs(y)), 0.0)
        for token, value in rule["biases"]:
            if token < len(x):
                y[token] += float(np.float32(value))
                # Each sum rounds by 2^-24 of it.
                bound[token] += half * 2 * (abs(float(np.float32(value))) * len(rule["biases"]) + abs(y[token]))
    top = float(np.finfo(np.float32).max)
    y[np.abs(y) > top] *= np.inf
    allowed = np.ones(len(x), dtype=bool) if rule["allowed"] is None else rule["allowed"]
    return np.where(allowed, y, -np.inf), bound + 1e-300, allowed


def _rule(rng, vocab, history=0, biases=0, masked=False, repetition=1.0, presence=0.0, frequency=0.0, repeats=True):
    tokens = rng.integers(0, vocab, history).astype(np.uint32)
    if repeats and history > 4:
        tokens[: history // 2] = rng.integers(0, max(1, vocab // 50), history // 2)
    ids = rng.integers(0, vocab, biases) if repeats else rng.permutation(vocab)[:biases]
    return {"history": tokens, "biases": [(int(t), float(v)) for t, v in zip(ids, rng.standard_normal(biases) * 4)],
            "allowed": rng.random(vocab) < 0.4 if masked else None, "repetition": repetition, "presence": presence, "frequency": frequency}


class _Logits:
    def __init__(self, dev, rows, rules, in_place=False, store=True, pick=True, offset=0, stream=None, spoil=None):
        self.dev, n, vocab = dev, *rows.shape
        buf = dev.upload(np.concatenate([np.zeros(offset, np.float32), rows.reshape(-1)]))
        out = buf if in_place else dev.upload(np.full(rows.size + offset + 16, 7.0, np.float32))
        tokens = dev.upload(np.full(n + 4, 0xABCD, np.uint32))
        table, keep = None, []
        if rules is not None:
            array = np.zeros(n, dtype=dev.LOGITS_RULE)
            for i, r in enumerate(rules):
                words = np.zeros((vocab + 31) // 32, np.uint32)
                if r["allowed"] is not None:
                    np.bitwise_or.at(words, np.nonzero(r["allowed"])[0] // 32, np.uint32(1) << (np.nonzero(r["allowed"])[0] % 32).astype(np.uint32))
                    # Bits past the vocabulary mean nothing.
                    if vocab % 32:
                        words[-1] |= np.uint32((0xFFFFFFFF << (vocab % 32)) & 0xFFFFFFFF)
                h, bt, bv, m = (dev.upload(a) for a in (r["history"], np.array([b[0] for b in r["biases"]], np.uint32),
                                                        np.array([b[1] for b in r["biases"]], np.float32), words))
                keep += [h, bt, bv, m]
                array[i] = (h.ptr, bt.ptr, bv.ptr, m.ptr if r["allowed"] is not None else 0, len(r["history"]), len(r["biases"]), r["repetition"],
                            r["presence"], r["frequency"])
            if spoil is not None:
                spoil(array)
            table = dev.upload(array)
        need = dev.logits_workspace_bytes(n, vocab)
        work = dev.upload(np.full(need + 64, 0x5A, np.uint8))
        dev.logits_adjust(buf.ptr + 4 * offset, n, vocab, table.ptr if table else 0, out.ptr + 4 * offset if store else 0, tokens.ptr if pick else 0,
                          work.ptr, stream)
        dev.sync(stream)
        assert np.all(dev.download(work.ptr, (need + 64,), np.uint8)[need:] == 0x5A)
        self.out = dev.download(out.ptr + 4 * offset, rows.shape, np.float32) if store else None
        if store and not in_place:
            assert np.all(dev.download(out.ptr, (rows.size + offset + 16,), np.float32)[offset + rows.size:] == 7.0)
        got = dev.download(tokens.ptr, (n + 4,), np.uint32)
        assert np.all(got[n if pick else 0:] == 0xABCD)
        self.tokens = got[:n]


def _check_logits(rows, rules, got):
    for i, row in enumerate(rows):
        rule = rules[i] if rules is not None else _rule(np.random.default_rng(0), len(row))
        want, bound, allowed = _adjust_reference(row, rule)
        if got.out is not None:
            x = got.out[i].astype(np.float64)
            finite = np.isfinite(want)
            assert np.array_equal(x[~finite], want[~finite], equal_nan=True), i
            assert np.all(np.abs(x[finite] - want[finite]) <= bound[finite]), i
            candidates = np.where(allowed & ~np.isnan(x), x, -np.inf)
            some = allowed & ~np.isnan(x)
            first = int(np.nonzero(some & (candidates == candidates.max()))[0][0]) if some.any() else 0xFFFFFFFF
            assert got.tokens[i] == first, i
        else:
            some = allowed & ~np.isnan(want)
            if not some.any():
                assert got.tokens[i] == 0xFFFFFFFF
            else:
                t = int(got.tokens[i])
                assert some[t] and want[t] >= want[some].max() - bound[t] - bound[some].max(), i


@pytest.mark.parametrize("vocab", [1, 2, 31, 33, 1000, 8191, 8192, 8193, 32000, 50257, 100003])
@pytest.mark.parametrize("form", ["both", "in place", "token only", "row only", "offset"])
def test_logits(dev, vocab, form):
    print(f"logits V={vocab} {form}", flush=True)
    rng = np.random.default_rng(vocab)
    n = 9
    rows = (3 * rng.standard_normal((n, vocab))).astype(np.float32)
    rules = [_rule(rng, vocab), _rule(rng, vocab, 1, repetition=1.3), _rule(rng, vocab, 500, repetition=1.2, presence=0.4, frequency=0.3),
             _rule(rng, vocab, 0, 3), _rule(rng, vocab, 0, 700), _rule(rng, vocab, 0, 0, True), _rule(rng, vocab, 3000, 300, True, 0.7, -0.2, 0.1),
             _rule(rng, vocab, 255, 256, True, repeats=False), _rule(rng, vocab, 70, 1, repetition=2.0)]
    more = {"both": {}, "in place": dict(in_place=True), "token only": dict(store=False), "row only": dict(pick=False), "offset": dict(offset=1)}[form]
    got = _Logits(dev, rows, rules, **more)
    if form == "row only":
        got.tokens = _Logits(dev, got.out, None, store=False).tokens
        # Masked-out logits are allowed ones for the second call: the same token wherever one was allowed.
        for i, r in enumerate(rules):
            if r["allowed"] is not None and not r["allowed"].any():
                got.tokens[i] = 0xFFFFFFFF
    _check_logits(rows, rules, got)


def test_logits_no_rules_is_argmax(dev):
    rng = np.random.default_rng(4)
    for vocab in (7, 9000):
        rows = rng.integers(-3, 3, (5, vocab)).astype(np.float32)   # ties everywhere
        got = _Logits(dev, rows, None)
        assert np.array_equal(got.out, rows)
        assert np.array_equal(got.tokens, rows.argmax(1))


def test_logits_empty_and_infinite_rows(dev):
    """Nothing allowed, NaN, infinities and minus infinities, the lowest number, ties across slices."""
    vocab = 20000
    rng = np.random.default_rng(6)
    low = np.finfo(np.float32).min
    rows = rng.standard_normal((9, vocab)).astype(np.float32)
    rules = [_rule(rng, vocab, 40, 5, True, 1.3, 0.1, 0.2) for _ in range(9)]
    rules[0]["allowed"][:] = False
    rows[1] = np.nan
    rows[2] = -np.inf
    rows[3, ::3] = np.nan
    rows[4, 12345] = np.inf
    rules[4]["allowed"][12345] = True
    rows[5] = low
    rows[6, 500] = rows[6, 19000] = 100.0
    rules[6]["allowed"][[500, 19000]] = True
    rules[6]["history"], rules[6]["biases"] = np.zeros(0, np.uint32), []
    rules[7]["allowed"][:] = False
    rules[7]["allowed"][vocab - 1] = True
    rows[7, vocab - 1] = -np.inf
    rows[8, 0] = -0.0
    got = _Logits(dev, rows, rules)
    _check_logits(rows, rules, got)
    assert got.tokens[0] == got.tokens[1] == 0xFFFFFFFF and got.tokens[6] == 500 and got.tokens[7] == vocab - 1 and got.tokens[4] == 12345


def test_logits_repeated_biases_add_up_in_order(dev):
    """Biases of one token whose order matters in 32 bits: 2^24 times, then ones, then minus 2^24."""
    vocab = 9000
    rows = np.zeros((2, vocab), dtype=np.float32)
    rng = np.random.default_rng(2)
    rules = [_rule(rng, vocab), _rule(rng, vocab)]
    rules[0]["biases"] = [(8200, 2.0 ** 24)] + [(8200, 1.0)] * 400 + [(8200, -(2.0 ** 24))] + [(17, 1.0)] * 300
    rules[1]["biases"] = [(8200, 1.0)] * 400 + [(8200, 2.0 ** 24), (8200, -(2.0 ** 24))] + [(5 + 1024 * (i % 8), 1.0) for i in range(700)]
    got = _Logits(dev, rows, rules)
    for i in range(2):
        want = np.zeros(vocab, dtype=np.float32)
        for token, value in rules[i]["biases"]:
            want[token] = np.float32(want[token] + np.float32(value))
        assert np.array_equal(got.out[i], want)


def test_logits_long_lists_and_wide_rows(dev):
    """Histories and bias lists longer than a block holds at once, rows in slices of every size."""
    for n, vocab, history, biases in ((3, 4093, 4096, 1024), (3, 4094, 4097, 1025), (2, 9001, 13000, 2500), (70, 130001, 5000, 1100)):
        print(f"logits lists {n} {vocab} {history} {biases}", flush=True)
        rng = np.random.default_rng(vocab)
        rows = (3 * rng.standard_normal((n, vocab), dtype=np.float32)).astype(np.float32)
        rules = [_rule(rng, vocab, history - i, biases - i if i < 3 else i, i % 2 == 1, 1.0 + 0.01 * i, 0.1, 0.05) for i in range(n)]
        _check_logits(rows, rules, _Logits(dev, rows, rules))


def test_logits_listed_tokens_past_the_vocabulary(dev):
    vocab = 100
    rng = np.random.default_rng(1)
    rows = rng.standard_normal((1, vocab)).astype(np.float32)
    rule = _rule(rng, vocab, 50, 4, repetition=1.5, presence=0.5)
    rule["history"][:5] = [100, 101, 0xFFFFFFFF, 0x80000000, 8192]
    rule["biases"] += [(100, 50.0), (0xFFFFFFFF, 50.0), (8192, 9.0)]
    got = _Logits(dev, rows, [rule])
    _check_logits(rows, [rule], got)


def test_logits_invalid_rules(dev):
    """A rule that cannot be applied leaves its row alone and picks no token; the other rows are made."""
    vocab = 9000
    rng = np.random.default_rng(3)
    rows = rng.standard_normal((9, vocab)).astype(np.float32)
    rules = [_rule(rng, vocab, 20, 3, repetition=1.1) for _ in range(9)]

    def spoil(array):
        array[0]["history"] = 0
        array[1]["bias_tokens"] = 0
        array[2]["bias_values"] = 0
        array[3]["repetition_penalty"] = 0.0
        array[4]["repetition_penalty"] = -1.0
        array[5]["repetition_penalty"] = np.nan
        array[6]["repetition_penalty"] = np.inf
        array[7]["history_count"] = 0x80000000

    got = _Logits(dev, rows, rules, spoil=spoil)
    assert np.all(got.tokens[:8] == 0xFFFFFFFF) and np.all(got.out[:8] == 7.0)
    got.out, got.tokens = got.out[8:], got.tokens[8:]
    _check_logits(rows[8:], rules[8:], got)


@pytest.mark.parametrize("vocab,most,rows", [(16000, 256, (128, 3)), (32000, 65, (64, 1)), (128000, 17, (16, 5))])
def test_logits_scratch_of_a_larger_batch(dev, vocab, most, rows):
    """Scratch made once for the largest batch serves the smaller ones that come after it; the bytes behind it stay."""
    rng = np.random.default_rng(most)
    need = dev.logits_workspace_bytes(most, vocab)
    for n in (most, *rows):
        print(f"logits scratch V={vocab} for {most}: {n} rows", flush=True)
        assert dev.logits_workspace_bytes(n, vocab) <= need   # else the call would write past it
        x = rng.standard_normal((n, vocab)).astype(np.float32)
        logits, tokens, work = dev.upload(x), dev.upload(np.zeros(n, np.uint32)), dev.upload(np.full(need + 65536, 0x5A, np.uint8))
        dev.logits_adjust(logits.ptr, n, vocab, 0, 0, tokens.ptr, work.ptr)
        dev.sync()
        assert np.array_equal(dev.download(tokens.ptr, (n,), np.uint32), x.argmax(1))
        assert np.all(dev.download(work.ptr, (need + 65536,), np.uint8)[need:] == 0x5A)


def test_logits_rows_far_away(dev):
    """Rows of more than 2^30 tokens, the last of them more than 2^32 logits from the first, in place."""
    rows, vocab = 4, (1 << 30) + 400_000_001
    buf = dev.DeviceBuffer(4 * rows * vocab)
    dev.fill_rows(buf.ptr, 2 * rows * vocab, 3, 0, 256)   # pairs of fp16 numbers below 4 are fp32 numbers below 512
    at = lambda r, t: buf.ptr + 4 * (r * vocab + t)   # noqa: E731
    for r in range(rows):
        for t, x in ((vocab - 2, 5000.0), (7 + r, 6000.0), (vocab // 2, 5050.0)):
            dev.copy_to_device(at(r, t), np.array([x], np.float32))
    tokens, work = dev.DeviceBuffer(4 * rows), dev.DeviceBuffer(dev.logits_workspace_bytes(rows, vocab))
    history = dev.upload(np.array([8, 8, vocab // 2, 0xFFFFFFFF], np.uint32))
    bias_tokens, bias_values = dev.upload(np.array([9, vocab - 1, 10], np.uint32)), dev.upload(np.array([-2000.0, 10000.0, -3000.0], np.float32))
    table = np.zeros(rows, dtype=dev.LOGITS_RULE)
    table["repetition_penalty"] = 1.0
    table[1] = (history.ptr, 0, 0, 0, 4, 0, 4.0, 0.0, 0.0)   # tokens 8 and vocab / 2 fall to a quarter
    table[2] = (0, bias_tokens.ptr, bias_values.ptr, 0, 0, 3, 1.0, 0.0, 0.0)
    table[3] = (0, bias_tokens.ptr, bias_values.ptr, 0, 0, 3, 1.0, 0.0, 0.0)
    rules = dev.upload(table)
    dev.logits_adjust(buf.ptr, rows, vocab, rules.ptr, buf.ptr, tokens.ptr, work.ptr)
    dev.sync()
    picked = dev.download(tokens.ptr, (rows,), np.uint32)
    read = lambda r, t: float(dev.download(at(r, t), (1,), np.float32)[0])   # noqa: E731
    assert list(picked) == [7, vocab - 2, vocab - 1, vocab - 1]
    assert (read(0, 7), read(1, 8), read(1, vocab // 2), read(1, vocab - 2)) == (6000.0, 1500.0, 1262.5, 5000.0)
    assert (read(2, 9), read(3, 10), read(3, vocab // 2)) == (4000.0, 3000.0, 5050.0) and 9488.0 < read(3, vocab - 1) < 10512.0


def test_logits_many_rows(dev):
    """More rows than a grid's y takes."""
    rng = np.random.default_rng(9)
    rows = rng.standard_normal((70000, 5)).astype(np.float32)
    got = _Logits(dev, rows, None)
    assert np.array_equal(got.tokens, rows.argmax(1)) and np.array_equal(got.out, rows)


# ---- together ----------------------------------------------------------------


def test_token_step_of_forked_requests(dev):
    """Four requests forked from one prompt: their rotated tokens appended (each to a copy of the partial page they
    share), attended to with the prompt read once, projected to logits, and picked under rules of their own, on a stream."""
    heads, dim, group, lanes, vocab, prompt = 4, 64, 8, 4, 1000, 707
    rng = np.random.default_rng(12)
    qd, rope, stream = heads * group * dim, dev.Rope(10000.0, dim, 0), dev.Stream()
    hidden = qd
    b = _Batch(dev, heads, dim, group, [prompt] * lanes, [])
    # Every lane's table: the first lane's full pages, then a page of its own that receives the shared tail and the new token.
    shared = [e for e in b.tables[0] if e[3] == e[4]]
    tail = b.tables[0][len(shared)]
    assert tail[3] == prompt % 8
    qkv = _fp16(rng, lanes, (heads * group + 2 * heads) * dim)
    jobs = np.zeros(lanes, dtype=dev.APPEND_ROPE_JOB)
    # Lanes 1.. go on in their own old tail pages, lane 0 in one that no table names.
    free = next(s for s in range(64) if s not in {e[0] for t in b.tables for e in t if e[5] == 0})
    slots = [free] + [b.tables[i][len(shared)][0] for i in range(1, lanes)]
    for i in range(lanes):
        jobs[i] = (i, 1, prompt, slots[i], tail[0], tail[3], tail[3], 0, 0, 0)
    b.tables = [shared + [(slots[i], 1, tail[2], tail[3] + 1, 8, 0)] for i in range(lanes)]
    src, job_buf, q_buf = dev.upload(_bits(qkv)), dev.upload(jobs), dev.DeviceBuffer(lanes * qd * 2)
    b.storage.append_rope_launch(job_buf.ptr, lanes, 1, 0, src.ptr, qkv.shape[1], lanes, heads * group, rope, q_buf.ptr, qd, stream)
    b.counts, b.groups = [prompt + 1] * lanes, [(0, lanes, prompt)]
    b.place()
    items = np.zeros(lanes, dtype=dev.DECODE_ITEM)
    for i in range(lanes):
        items[i] = (b.tab[i].ptr, len(b.tables[i]), prompt + 1, 0, q_buf.ptr + 2 * i * qd, 0, b.out.ptr + 2 * i * qd, 1.0 / math.sqrt(dim))
    b.items = dev.upload(items)
    b.plan()
    weight = _fp16(rng, vocab, hidden, scale=0.1)
    w_buf, logits = dev.upload(_bits(weight)), dev.DeviceBuffer(lanes * vocab * 4)
    rules = [_rule(rng, vocab, 30, 5, i % 2 == 1, 1.2, 0.3, 0.1) for i in range(lanes)]
    b.storage.shared_decode_launch(b.items.ptr, b.entries_buf.ptr, b.p, b.work.ptr + 2048, stream)
    dev.linear(b.out.ptr, lanes, hidden, w_buf.ptr, vocab, logits.ptr, True, 0.0, stream)
    stream.synchronize()
    got_logits = dev.download(logits.ptr, (lanes, vocab), np.float32)
    picked = _Logits(dev, got_logits, rules, stream=stream)
    _check_logits(got_logits, rules, picked)
    # The same in 64 bits from the start: rotated keys and queries rounded to fp16 as the cache holds them.
    x = qkv.reshape(lanes, -1, dim)
    turned, _ = _rotate(x[:, :heads * group + heads], np.full(lanes, prompt, np.uint64), 10000.0, dim, 0)
    held = b.storage.gather(np.array(b.tables[2], dtype=dev.BLOCK_DESC), prompt + 1).view(np.float16).reshape(2, prompt + 1, heads, dim)
    assert np.array_equal(_bits(held[0, :prompt]), _bits(b.k[0])) and np.array_equal(_bits(held[1, prompt]), _bits(x[2, -heads:]))
    query = dev.download(q_buf.ptr, (lanes, heads * group, dim), np.uint16).view(np.float16)
    out = b.outputs().view(np.float16)
    for i in range(lanes):
        assert np.all(np.abs(query[i].astype(np.float64) - turned[i, :heads * group]) <= FP16 * np.abs(turned[i, :heads * group]) + 2.0 ** -18)
        mine = b.storage.gather(np.array(b.tables[i], dtype=dev.BLOCK_DESC), prompt + 1).view(np.float16).reshape(2, prompt + 1, heads, dim)
        want, bound = reference(query[i], mine[0], mine[1], 1.0 / math.sqrt(dim))
        assert np.all(np.abs(out[i].astype(np.float64) - want) <= bound)
    assert b.storage.faults() == (0, 0)
    stream.destroy()


def _hip():
    """The HIP runtime that the library runs on."""
    with open("/proc/self/maps") as f:
        paths = {line.split()[-1] for line in f if "libamdhip64" in line}
    assert len(paths) == 1, paths
    return ctypes.CDLL(paths.pop())


def test_token_step_captured_in_a_graph(dev):
    """The three operators captured on a stream and replayed on new inputs, with eager work between the replays, give what
    eager calls give."""
    hip = _hip()
    heads, dim, group, vocab = 4, 64, 8, 20000
    b = _Batch(dev, heads, dim, group, [900, 901, 950, 1200, 60], [(0, 4, 890)])
    b.place()
    b.plan()
    qd, lanes, width, rope, stream = heads * group * dim, 5, (group + 2) * heads * dim, dev.Rope(10000.0, dim, 0), dev.Stream()
    jobs = np.zeros(lanes, dtype=dev.APPEND_ROPE_JOB)
    for i, t in enumerate(b.tables):   # each lane's last token written anew
        e = t[-1]
        jobs[i] = (i, 1, b.counts[i] - 1, e[0], 0, e[3] - 1, 0, e[5], 0, 0)
    job_buf, qkv, q = dev.upload(jobs), dev.DeviceBuffer(lanes * width * 2), dev.DeviceBuffer(lanes * qd * 2)
    logits, out, tokens = dev.DeviceBuffer(lanes * vocab * 4), dev.DeviceBuffer(lanes * vocab * 4), dev.DeviceBuffer(lanes * 4)
    work = dev.DeviceBuffer(dev.logits_workspace_bytes(lanes, vocab))
    table, keep = np.zeros(lanes, dtype=dev.LOGITS_RULE), []
    for i in range(lanes):
        r = _rule(np.random.default_rng(i), vocab, 50, 4)
        lists = [dev.upload(x) for x in (r["history"], np.array([t for t, _ in r["biases"]], np.uint32), np.array([v for _, v in r["biases"]], np.float32))]
        table[i] = (*[x.ptr for x in lists], 0, 50, 4, 1.2, 0.2, 0.1)
        keep += lists
    rules = dev.upload(table)
    items = np.zeros(lanes, dtype=dev.DECODE_ITEM)
    for i in range(lanes):
        items[i] = (b.tab[i].ptr, len(b.tables[i]), b.counts[i], 0, q.ptr + 2 * i * qd, 0, b.out.ptr + 2 * i * qd, 1.0 / math.sqrt(dim))
    item_buf = dev.upload(items)

    def step():
        b.storage.append_rope_launch(job_buf.ptr, lanes, 1, 0, qkv.ptr, width, lanes, heads * group, rope, q.ptr, qd, stream)
        b.storage.shared_decode_launch(item_buf.ptr, b.entries_buf.ptr, b.p, b.work.ptr + 2048, stream)
        dev.logits_adjust(logits.ptr, lanes, vocab, rules.ptr, out.ptr, tokens.ptr, work.ptr, stream)

    def results():
        stream.synchronize()
        return [dev.download(q.ptr, (lanes, qd), np.uint16), b.outputs(), dev.download(out.ptr, (lanes, vocab), np.uint32),
                dev.download(tokens.ptr, (lanes,), np.uint32)]

    graph, runs, handle = ctypes.c_void_p(), ctypes.c_void_p(), ctypes.c_void_p(stream.handle)
    assert hip.hipStreamBeginCapture(handle, 0) == 0
    step()
    assert hip.hipStreamEndCapture(handle, ctypes.byref(graph)) == 0
    assert hip.hipGraphInstantiate(ctypes.byref(runs), graph, None, None, 0) == 0
    rng = np.random.default_rng(4)
    for _ in range(4):
        dev.copy_to_device(qkv.ptr, _bits(_fp16(rng, lanes, width)))
        dev.copy_to_device(logits.ptr, rng.standard_normal((lanes, vocab)).astype(np.float32))
        assert hip.hipGraphLaunch(runs, handle) == 0
        replayed = results()
        for buf, n in ((q, 2 * qd), (out, 4 * vocab), (tokens, 4)):
            dev.copy_to_device(buf.ptr, np.zeros(lanes * n, np.uint8))
        step()
        for x, y in zip(replayed, results()):
            assert np.array_equal(x, y)
        assert np.all(replayed[3] < vocab)
    assert b.storage.faults() == (0, 0)
    hip.hipGraphExecDestroy(runs)
    hip.hipGraphDestroy(graph)
    stream.destroy()
