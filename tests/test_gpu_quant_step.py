"""A cache in 8 bits on the GPU against plain forms in 64 bits: quantised append (kimkv_quant_append_batch), read-back
(kimkv_quant_gather), promotion (kimkv_quant_promote_batch), decode (kimkv_quant_decode_batch), sampling
(kimkv_model_sample), and a token step of them together."""
import ctypes
import math

import numpy as np
import pytest

from tests import helpers
from tests.test_gpu_token_step import _hip

pytestmark = pytest.mark.gpu

INT8, E4M3 = 1, 2
FORMS = {"int8": INT8, "e4m3": E4M3}
LARGEST = {INT8: 127.0, E4M3: 448.0}
FP16 = 2.0 ** -11   # half a step of fp16, relative
TINY = 2.0 ** -25   # half a step of its subnormals


def _fp16(rng, *shape, scale=1.0):
    return (scale * rng.standard_normal(shape)).astype(np.float16)


def _bits(a):
    return np.ascontiguousarray(a).view(np.uint16)


def held(x, form):
    """What the cache holds of rows of fp16 [..., D], in 64 bits (every value is exact in them): NaN throughout for a row
    that is not finite."""
    with np.errstate(all="ignore"):
        x = x.astype(np.float64)
        a = np.abs(x).max(-1, keepdims=True)
        q = a / LARGEST[form]
        mantissa, exponent = np.frexp(q)
        s = np.ldexp(np.ceil(mantissa * 256), exponent - 8)
        y = x / np.where(s == 0, 1.0, s)
        if form == INT8:
            c = np.rint(y)
        else:
            step = np.ldexp(1.0, np.maximum(np.frexp(np.abs(y))[1] - 1, -6) - 3)
            c = np.rint(y / step) * step
        return np.where(np.isfinite(a), c * s, np.nan)


def read(values):
    """Rows as they are read back: rounded once, kept to the largest fp16."""
    return np.clip(values, -65504, 65504).astype(np.float16)


def _same(got, want):
    """Equal numbers, NaN where NaN is due (of any sign; -0 is 0)."""
    got, want = np.asarray(got), np.asarray(want)
    bad = ~((got == want) | (np.isnan(got) & np.isnan(want)))
    assert not bad.any(), (int(bad.sum()), np.argwhere(bad)[:4].tolist(), got[bad][:4], want[bad][:4])


class _Cache:
    """A storage with every page filled, and the 64-bit values its pages should hold ([kind] -> [layer][2][slot * cap][H][D])."""

    def __init__(self, dev, form, heads, dim, layers=2, micro=24, extent=6, micro_tokens=8, extent_tokens=64, seed=1):
        self.dev, self.form, self.heads, self.dim, self.layers = dev, form, heads, dim, layers
        self.caps = (micro_tokens, extent_tokens)
        self.storage = dev.QuantStorage(layers, heads, dim, micro, extent, form, micro_tokens, extent_tokens)
        rng = np.random.default_rng(seed)
        self.pages, self.tables = [], []
        for kind, n in ((0, micro), (1, extent)):
            cap = self.caps[kind]
            self.tables.append(np.array([(s, 1, s * cap, cap, cap, kind) for s in range(n)], dtype=helpers.DESC))
            kv = _fp16(rng, layers, 2, n * cap, heads, dim)
            buf = dev.upload(_bits(kv))
            jobs = self.jobs_of(buf.ptr, n * cap, [(s * cap, cap, kind, s, 0) for s in range(n)])
            self.storage.append_batch(jobs)
            self.pages.append(held(kv, form))

    def jobs_of(self, ptr, total, runs, cows=None, layer_begin=0, layer_count=None, token_stride=None):
        """Jobs of (row, tokens, kind, slot, page token) from [layer][2][total][H][D] at ptr."""
        row = token_stride or self.heads * self.dim
        jobs = np.zeros(len(runs), dtype=self.dev.APPEND_JOB)
        for i, (first, n, kind, slot, token) in enumerate(runs):
            cow = (cows or {}).get(i, (0, 0, 0))   # kind, slot, tokens
            jobs[i] = (ptr + 2 * first * row, ptr + 2 * (total + first) * row, 2 * total * row, row, layer_begin,
                       self.layers if layer_count is None else layer_count, n, slot, cow[1], token, cow[2], kind, cow[0])
        return jobs

    def expect(self, kv, runs, cows=None, layer_begin=0):
        """Takes the jobs' work over into what the pages should hold; kv: [layers of the jobs][2][total][H][D] fp16."""
        values = held(kv, self.form)
        layers = slice(layer_begin, layer_begin + len(kv))
        for i, (first, n, kind, slot, token) in enumerate(runs):
            at = slot * self.caps[kind]
            if i in (cows or {}):
                k, s, m = cows[i]
                self.pages[kind][layers, :, at:at + m] = self.pages[k][layers, :, s * self.caps[k]:s * self.caps[k] + m]
        for first, n, kind, slot, token in runs:
            at = slot * self.caps[kind] + token
            self.pages[kind][layers, :, at:at + n] = values[:, :, first:first + n]

    def check(self):
        for kind in (0, 1):
            want = self.pages[kind]
            got = self.storage.gather(self.tables[kind], want.shape[2]).view(np.float16).reshape(want.shape)
            _same(got, read(want))


SHAPES = [(4, 64), (8, 128), (3, 96), (1, 256), (2, 12), (5, 33), (1, 1), (2, 8)]
# Single tokens at every place of a micro page, copied tails, runs within and across groups of 8, whole pages.
RUNS = [(3, 1, 0, 0, 0), (0, 1, 0, 1, 7), (1, 1, 0, 3, 3), (2, 1, 0, 5, 5), (4, 8, 0, 6, 0), (12, 5, 0, 7, 3), (17, 64, 1, 0, 0), (81, 17, 1, 1, 6),
        (98, 30, 1, 2, 34), (128, 0, 0, 9, 4), (129, 3, 0, 11, 1), (132, 7, 0, 12, 0), (139, 8, 1, 4, 3), (147, 9, 1, 5, 55)]
COWS = {1: (0, 2, 7), 2: (0, 4, 2), 5: (0, 8, 3), 8: (1, 3, 34), 9: (0, 10, 4), 13: (1, 3, 55), 12: (0, 13, 3)}
ROWS = 156


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("heads,dim", SHAPES)
def test_append(dev, form, heads, dim):
    print(f"quant_append {form} H={heads} D={dim}", flush=True)
    c = _Cache(dev, FORMS[form], heads, dim)
    c.check()
    kv = _fp16(np.random.default_rng(5), 2, 2, ROWS, heads, dim)
    buf = dev.upload(_bits(kv))
    c.storage.append_batch(c.jobs_of(buf.ptr, ROWS, RUNS, COWS))
    c.expect(kv, RUNS, COWS)
    c.check()
    assert c.storage.faults() == (0, 0)


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("how", ["one layer", "odd address", "strides", "odd strides", "stream", "layers of unlike jobs"])
def test_append_forms(dev, form, how):
    print(f"quant_append {form} {how}", flush=True)
    heads, dim = 4, 64
    c = _Cache(dev, FORMS[form], heads, dim, layers=3)
    rng = np.random.default_rng(6)
    stream = dev.Stream() if how == "stream" else None
    offset, pad = (3 if how == "odd address" else 0), {"strides": 24, "odd strides": 5}.get(how, 0)
    layers, begin = (1, 2) if how == "one layer" else (3, 0)
    row = heads * dim + pad
    source = _fp16(rng, layers, 2, ROWS, row)
    buf = dev.upload(np.concatenate([np.zeros(offset, np.uint16), _bits(source).reshape(-1)]))
    jobs = c.jobs_of(buf.ptr + 2 * offset, ROWS, RUNS, COWS, begin, layers, row)
    kv = source[..., :heads * dim].reshape(layers, 2, ROWS, heads, dim)
    if how == "layers of unlike jobs":
        jobs["layer_count"][::2] = 1
        before = [p.copy() for p in c.pages]
        c.expect(kv, RUNS, COWS)
        after = c.pages
        c.pages = before
        for i, (first, n, kind, slot, token) in enumerate(RUNS):
            at = slice(slot * c.caps[kind], (slot + 1) * c.caps[kind])
            layer = slice(0, 1) if i % 2 == 0 else slice(0, 3)
            c.pages[kind][layer, :, at] = after[kind][layer, :, at]
    else:
        c.expect(kv, RUNS, COWS, begin)
    c.storage.append_batch(jobs, stream)
    c.check()
    assert c.storage.faults() == (0, 0)


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("tokens", [(16, 32), (24, 48), (64, 8), (8, 8)])
def test_append_other_pages(dev, form, tokens):
    print(f"quant_append {form} pages of {tokens}", flush=True)
    micro, extent = tokens
    c = _Cache(dev, FORMS[form], 2, 64, micro_tokens=micro, extent_tokens=extent)
    runs = [(0, micro, 0, 0, 0), (micro, 1, 0, 1, micro - 1), (micro + 1, extent, 1, 0, 0), (micro + 1 + extent, extent - 3, 1, 1, 2)]
    cows = {1: (1, 2, min(micro - 1, extent)), 3: (0, 2, 2)}
    total = micro + 2 * extent
    kv = _fp16(np.random.default_rng(7), 2, 2, total, 2, 64)
    buf = dev.upload(_bits(kv))
    c.storage.append_batch(c.jobs_of(buf.ptr, total, runs, cows))
    c.expect(kv, runs, cows)
    c.check()
    assert c.storage.faults() == (0, 0)


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("heads,dim", [(4, 64), (2, 12)])
def test_append_fork_from_one_page(dev, form, heads, dim):
    """Requests leave one shared partial page, each with a copy of its own, while its last holder writes on behind what they
    copy."""
    print(f"quant_append fork {form} H={heads} D={dim}", flush=True)
    c = _Cache(dev, FORMS[form], heads, dim)
    runs = [(i, 1, 0, 1 + i, 5) for i in range(12)] + [(12, 1, 0, 0, 5), (13, 1, 0, 14, 3)]
    runs += [(14 + i, 1, 1, 1 + i, 43) for i in range(3)] + [(17, 12, 1, 0, 43)]
    cows = {**{i: (0, 0, 5) for i in range(12)}, 13: (0, 0, 3), **{14 + i: (1, 0, 43) for i in range(3)}}
    kv = _fp16(np.random.default_rng(8), 2, 2, 29, heads, dim)
    buf = dev.upload(_bits(kv))
    c.storage.append_batch(c.jobs_of(buf.ptr, 29, runs, cows))
    c.expect(kv, runs, cows)
    c.check()


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("heads,dim", [(4, 64), (1, 128), (2, 12)])
def test_append_every_row_kind(dev, form, heads, dim):
    """Rows of zeros, of the largest and the smallest numbers, of ties, of infinities and NaN; other rows keep their values."""
    print(f"quant_append rows {form} H={heads} D={dim}", flush=True)
    c = _Cache(dev, FORMS[form], heads, dim, layers=1)
    rng = np.random.default_rng(9)
    kv = _fp16(rng, 1, 2, 128, heads, dim)
    kv[0, :, 0] = 0
    kv[0, :, 1] = -0.0
    kv[0, :, 2] = 65504
    kv[0, :, 3] = -65504
    kv[0, :, 4] = 2.0 ** -24
    kv[0, :, 5] = kv[0, :, 5] * np.float16(2.0 ** -20)
    kv[0, :, 6] = kv[0, :, 6] * np.float16(8000)
    kv[0, :, 7, :, 0] = np.inf
    kv[0, :, 8, :, -1] = -np.inf
    kv[0, :, 9, :, dim // 2] = np.nan
    kv[0, :, 10] = np.nan
    kv[0, 0, 11, 0, 0] = np.inf          # one head's K alone
    kv[0, 1, 12, heads - 1, 0] = np.nan  # one head's V alone
    # Ties: halves of a whole number beside 127, midpoints of e4m3's steps beside 448, for several scales.
    for i in range(64):
        power = np.float16(2.0 ** (i % 8 - 4))
        if form == "int8":
            row = (rng.integers(-126, 126, (2, heads, dim)) + 0.5)
            row[..., 0] = 127
        else:
            e = rng.integers(-6, 8, (2, heads, dim))
            row = np.ldexp((rng.integers(8, 16, (2, heads, dim)) * 2 + 1) / 16.0, e) * np.where(rng.random((2, heads, dim)) < 0.5, 1, -1)
            row[..., 0] = 448
        kv[0, :, 64 + i] = row * power
    runs = [(0, 64, 1, 0, 0), (64, 64, 1, 1, 0)] + [(i, 1, 0, i, i % 8) for i in range(16)]
    buf = dev.upload(_bits(kv))
    c.storage.append_batch(c.jobs_of(buf.ptr, 128, runs))
    c.expect(kv, runs)
    c.check()
    nan = np.isnan(c.pages[1][0, 0, 7])
    assert nan.all() and not np.isnan(c.pages[1][0, 0, 12]).any()


def test_append_faults(dev):
    """Bad jobs are skipped and reported; the others are done."""
    c = _Cache(dev, INT8, 2, 64, layers=2)
    kv = _fp16(np.random.default_rng(10), 2, 2, 64, 2, 64)
    buf = dev.upload(_bits(kv))
    good = [(0, 1, 0, 0, 0)]
    bad = {"slot": dict(dst_slot=24), "extent slot": dict(dst_kind=1, dst_slot=6), "kind": dict(dst_kind=2), "past the page": dict(dst_token=8),
           "long": dict(token_count=9), "far token": dict(dst_token=65535), "layer": dict(layer_begin=2), "far layer": dict(layer_begin=0xFFFFFFFF),
           "no key": dict(src_key=0), "no value": dict(src_value=0), "copy slot": dict(cow_tokens=1, cow_slot=99, dst_token=3),
           "copy kind": dict(cow_tokens=1, cow_kind=7, dst_token=3), "copy past its page": dict(cow_tokens=9, dst_kind=1, dst_slot=1, dst_token=20),
           "copy above": dict(cow_tokens=4, dst_token=3), "tokens": dict(token_count=0xFFFFFFFF, dst_token=2)}
    for name, change in bad.items():
        print(f"quant_append fault {name}", flush=True)
        jobs = c.jobs_of(buf.ptr, 64, good + [(1, 1, 0, 2, 1)])
        for field, value in change.items():
            jobs[1][field] = value
        c.storage.append_batch(jobs)
        assert c.storage.faults() == (dev.INVALID_ARGUMENT, dev.FAULT_APPEND_JOB), name
        assert c.storage.faults() == (0, 0)
    c.expect(kv, good)
    c.check()


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("heads,dim", [(4, 64), (8, 128), (3, 96), (5, 33), (2, 8)])
def test_gather(dev, form, heads, dim):
    """Ranges that begin and end inside pages, tables whose pages hold part of their tokens and begin anywhere, one layer and
    several, outputs at an odd address; tokens that the table leaves out stay."""
    print(f"quant_gather {form} H={heads} D={dim}", flush=True)
    c = _Cache(dev, FORMS[form], heads, dim, layers=3)
    entries, begin = [], 0
    for kind, slot, n in [(0, 3, 8), (1, 2, 64), (0, 5, 3), (1, 0, 37), (0, 9, 1), (1, 5, 64), (0, 1, 6)]:
        entries.append((slot, 1, begin, n, c.caps[kind], kind))
        begin += n
    table = np.array(entries, dtype=helpers.DESC)
    whole = np.concatenate([c.pages[e[5]][:, :, e[0] * c.caps[e[5]]:e[0] * c.caps[e[5]] + e[3]] for e in entries], 2)
    _same(c.storage.gather(table, begin).view(np.float16).reshape(whole.shape), read(whole))
    d = dev.upload(table)
    for first, n, layer, layers, odd in [(0, 1, 0, 3, 0), (70, 5, 1, 1, 0), (5, 100, 2, 1, 0), (72, 1, 0, 2, 0), (begin - 1, 1, 0, 1, 0), (11, 150, 1, 2, 1), (3, 90, 0, 1, 3)]:
        out = dev.upload(np.full(layers * 2 * n * heads * dim + 8, 0x1234, np.uint16))
        c.storage.gather_launch(d.ptr, len(table), first, n, layer, layers, out.ptr + 2 * odd)
        got = dev.download(out.ptr, (layers * 2 * n * heads * dim + 8,), np.uint16)
        want = whole[layer:layer + layers, :, first:first + n]
        _same(got[odd:odd + want.size].view(np.float16).reshape(want.shape), read(want))
        assert np.all(got[:odd] == 0x1234) and np.all(got[odd + want.size:] == 0x1234)
    # A table that leaves tokens out in front, within and behind.
    hole = table[[1, 3]]
    out = dev.upload(np.full(3 * 2 * begin * heads * dim, 0x1234, np.uint16))
    h = dev.upload(hole)
    c.storage.gather_launch(h.ptr, 2, 0, begin, 0, 3, out.ptr)
    got = dev.download(out.ptr, (3, 2, begin, heads, dim), np.uint16)
    covered = np.zeros(begin, bool)
    for e in hole:
        covered[e["logical_token_begin"]:e["logical_token_begin"] + e["valid_tokens"]] = True
    _same(got[:, :, covered].view(np.float16), read(whole[:, :, covered]))
    assert np.all(got[:, :, ~covered] == 0x1234)
    assert c.storage.faults() == (0, 0)
    for change in (dict(slot=99), dict(kind=2), dict(page_token_capacity=32), dict(valid_tokens=65)):
        bad = table.copy()
        for name, value in change.items():
            bad[1][name] = value
        c.storage.gather(bad[:2], 72)
        assert c.storage.faults() == (dev.INVALID_ARGUMENT, dev.FAULT_GATHER_ENTRY)


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("heads,dim", [(4, 64), (8, 128), (3, 96), (5, 33), (1, 1)])
def test_promote(dev, form, heads, dim):
    print(f"quant_promote {form} H={heads} D={dim}", flush=True)
    c = _Cache(dev, FORMS[form], heads, dim, layers=3)
    jobs = np.zeros(3, dtype=dev.PROMOTION_JOB)
    order = np.random.default_rng(3).permutation(24)
    for i, extent in enumerate((4, 0, 5)):
        jobs[i] = (order[8 * i:8 * i + 8], extent)
        rows = np.concatenate([np.arange(8) + 8 * s for s in order[8 * i:8 * i + 8]])
        c.pages[1][:, :, 64 * extent:64 * extent + 64] = c.pages[0][:, :, rows]
    c.storage.promote_batch(jobs)
    c.check()
    assert c.storage.faults() == (0, 0)
    bad = jobs.copy()
    bad["micro_slots"][0, 3] = 24
    bad["extent_slot"][2] = 6
    c.storage.promote_batch(bad)
    assert c.storage.faults() == (dev.INVALID_ARGUMENT, dev.FAULT_PROMOTION_JOB)
    c.check()


def test_page_refusals(dev):
    s = dev.QuantStorage(2, 2, 64, 4, 4, INT8)
    other = dev.QuantStorage(2, 2, 64, 4, 4, INT8, 16, 64)
    lib, buf = dev.lib(), dev.DeviceBuffer(4096)
    bad = dev.INVALID_ARGUMENT
    assert lib.kimkv_quant_append_batch(s.handle, None, 1, 1, None) == bad
    assert lib.kimkv_quant_append_batch(s.handle, buf.ptr, 1, 3, None) == bad
    assert lib.kimkv_quant_append_batch(s.handle, None, 0, 1, None) == dev.OK
    assert lib.kimkv_quant_append_batch(s.handle, buf.ptr, 1, 0, None) == dev.OK
    assert lib.kimkv_quant_gather(s.handle, None, 1, 0, 1, 0, 1, buf.ptr, None) == bad
    assert lib.kimkv_quant_gather(s.handle, buf.ptr, 0, 0, 1, 0, 1, buf.ptr, None) == bad
    assert lib.kimkv_quant_gather(s.handle, buf.ptr, 1, 0, 1, 0, 1, None, None) == bad
    assert lib.kimkv_quant_gather(s.handle, buf.ptr, 1, 0, 1, 1, 2, buf.ptr, None) == bad
    assert lib.kimkv_quant_gather(s.handle, buf.ptr, 1, 0, 1, 3, 0, buf.ptr, None) == bad
    assert lib.kimkv_quant_gather(s.handle, buf.ptr, 1, 0xFFFFFFFF, 1, 0, 1, buf.ptr, None) == bad
    assert lib.kimkv_quant_gather(s.handle, buf.ptr, 1, 5, 0, 0, 1, None, None) == dev.OK
    assert lib.kimkv_quant_promote_batch(s.handle, None, 1, None) == bad
    assert lib.kimkv_quant_promote_batch(other.handle, buf.ptr, 1, None) == bad
    assert lib.kimkv_quant_promote_batch(s.handle, None, 0, None) == dev.OK
    info = s.info()
    assert (info.format, info.micro_page_tokens, info.extent_page_tokens) == (INT8, 8, 64)
    assert info.extent_page_bytes == 2 * 2 * 64 * (2 * 64 + 4) and info.reserved_bytes == 4 * (info.extent_page_bytes + info.micro_page_bytes)


# ---- decode ------------------------------------------------------------------


class _Lanes:
    """Lanes of a cache: tables, the 64-bit values they read, items and outputs."""

    def __init__(self, dev, form, heads, dim, group, tables, micro, extent, layers=2, layer=1, caps=(8, 64), seed=2, scale=None, keys=None, values=None,
                 query=None, offset=0):
        self.dev, self.group, self.heads, self.dim = dev, group, heads, dim
        rng = np.random.default_rng(seed)
        self.storage = dev.QuantStorage(layers, heads, dim, micro, extent, form, *caps)
        self.scale = 1.0 / math.sqrt(dim) if scale is None else scale
        self.tables = [np.array(t, dtype=helpers.DESC) if len(t) else np.zeros(0, dtype=helpers.DESC) for t in tables]
        self.counts = [int(t["valid_tokens"].sum()) for t in self.tables]
        kv = _fp16(rng, 2, sum(self.counts), heads, dim)
        if keys is not None:
            kv[0] = keys(kv[0])
        if values is not None:
            kv[1] = values(kv[1])
        self.kv, self.buf = held(kv, form), dev.upload(_bits(kv))
        row, jobs, at = heads * dim, [], 0
        for t in self.tables:
            for e in t:
                n = int(e["valid_tokens"])
                jobs.append((self.buf.ptr + 2 * at * row, self.buf.ptr + 2 * (sum(self.counts) + at) * row, 0, row, layer, 1, n, e["slot"], 0, 0, 0, e["kind"], 0))
                at += n
        if jobs:
            self.storage.append_batch(np.array(jobs, dtype=dev.APPEND_JOB))
        n = len(tables)
        self.q = (2 * rng.standard_normal((n, heads * group, dim))).astype(np.float16)
        if query is not None:
            self.q = query(self.q)
        self.qbuf = dev.upload(np.concatenate([np.zeros(offset, np.uint16), _bits(self.q).reshape(-1)]))
        self.out = dev.upload(np.full(offset + self.q.size, 0x1234, np.uint16))
        self.offset = offset
        self.descs = [dev.upload(t) if len(t) else dev.DeviceBuffer(20) for t in self.tables]
        self.items = np.zeros(n, dtype=dev.DECODE_ITEM)
        for i, t in enumerate(self.tables):
            at = 2 * (offset + i * heads * group * dim)
            self.items[i] = (self.descs[i].ptr, len(t), self.counts[i], layer, self.qbuf.ptr + at, 0, self.out.ptr + at, self.scale)

    def run(self, stream=None, compute_units=None):
        dev = self.dev
        entries, plan = dev.quant_decode_plan(self.heads, self.dim, self.heads * self.group, compute_units or self.storage.info().compute_units, self.counts)
        e, items = dev.upload(entries) if len(entries) else dev.DeviceBuffer(16), dev.upload(self.items)
        # The scratch's contents are ignored: NaN.
        work = dev.upload(np.full(plan.workspace_bytes // 4 + 64, 0x7FC00000, np.uint32))
        self.storage.decode_launch(items.ptr, e.ptr, plan, work.ptr, stream)
        dev.sync(stream)
        tail = dev.download(work.ptr + plan.workspace_bytes, (64,), np.uint32)
        assert np.all(tail == 0x7FC00000)
        return dev.download(self.out.ptr + 2 * self.offset, self.q.shape, np.uint16)

    def want(self, seen=None):
        """(outputs, bounds) in 64 bits; seen: for each lane a mask of the tokens that take part.
        A score's dot product is of exact products summed in 32 bits, D terms: off by at most D 2^-24 of the terms' sizes, its
        scaling by 3 roundings; a weight by that much of itself, by the exponential's 2^-22 of its argument and 2^-20 of two fp16
        parts; sums of n terms by n 2^-24 at most."""
        out, bound, at = [], [], 0
        for i, n in enumerate(self.counts):
            k, v = self.kv[:, at:at + n]
            at += n
            if seen is not None:
                k, v = k[seen[i]], v[seen[i]]
            o = np.zeros((self.heads * self.group, self.dim))
            b = np.zeros_like(o)
            for j in range(self.heads * self.group):
                q, h = self.q[i, j].astype(np.float64), j // self.group
                if len(k) == 0:
                    continue
                s = k[:, h] @ q * self.scale
                off = (np.abs(k[:, h]) @ np.abs(q) * abs(self.scale) * (self.dim + 3) * 2.0 ** -24).max()
                p = np.exp(s - s.max())
                p /= p.sum()
                size = p @ np.abs(v[:, h])
                o[j] = p @ v[:, h]
                b[j] = FP16 * np.abs(o[j]) + TINY + size * (2 * off + (np.abs(s).max() + 1) * 2.0 ** -21 + 2.0 ** -19 + len(k) * 2.0 ** -24)
            out.append(o)
            bound.append(b)
        return np.array(out), np.array(bound)

    def check(self, seen=None, **more):
        got = self.run(**more).view(np.float16)
        want, bound = self.want(seen)
        for i, n in enumerate(self.counts):
            if n == 0:
                assert np.all(got[i].view(np.uint16) == 0x1234)
                continue
            err = np.abs(got[i].astype(np.float64) - want[i]) - bound[i]
            assert np.all(err <= 0), (i, n, float(err.max()), np.unravel_index(np.argmax(err), err.shape))


def _table(tokens, free, lead=0, caps=(8, 64), small=False):
    """Some small pages in front, large ones while they are full, small ones."""
    entries, at = [], 0
    while at < tokens:
        kind = 1 if not small and at >= lead * caps[0] and at + caps[1] <= tokens else 0
        n = min(caps[kind], tokens - at)
        entries.append((free[kind].pop(0), 1, at, n, caps[kind], kind))
        at += n
    return entries


def _pool(micro, extent, seed=4):
    return [list(helpers.splitmix_permutation(seed, micro)), list(helpers.splitmix_permutation(seed + 1, extent))]


LENGTHS = [1, 0, 7, 8, 9, 63, 64, 65, 127, 200, 256, 257, 300, 1000, 1029, 4160, 2500]


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("heads,dim,group", [(4, 64, 8), (8, 128, 4), (2, 96, 3), (1, 64, 16), (3, 64, 1), (2, 128, 16), (1, 96, 16), (2, 64, 17), (1, 128, 40),
                                             (2, 80, 4), (1, 256, 2), (3, 33, 5), (1, 1, 1)])
def test_decode(dev, form, heads, dim, group):
    """Lengths about every border, small pages in front that shift the large ones, one lane of small pages alone."""
    print(f"quant_decode {form} H={heads} D={dim} G={group}", flush=True)
    free = _pool(400, 160)
    tables = [_table(n, free, lead=i % 5 if i % 2 else 0, small=n == 1029) for i, n in enumerate(LENGTHS)]
    _Lanes(dev, FORMS[form], heads, dim, group, tables, 400, 160).check()


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("dim", [64, 96, 128, 40])
@pytest.mark.parametrize("units", [1, 2, 8, 256])
def test_decode_parts(dev, form, dim, units):
    """Lanes in one part and in many, merged."""
    print(f"quant_decode parts {form} D={dim} units={units}", flush=True)
    free = _pool(64, 400)
    tables = [_table(n, free, lead=lead) for n, lead in ((9000, 0), (5, 0), (8100, 3), (1100, 0))]
    lanes = _Lanes(dev, FORMS[form], 2, dim, 4, tables, 64, 400)
    lanes.check(compute_units=units)
    assert lanes.storage.faults() == (0, 0)


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("caps", [(16, 32), (24, 48), (64, 8), (8, 64)])
@pytest.mark.parametrize("dim", [64, 128])
def test_decode_other_pages(dev, form, caps, dim):
    print(f"quant_decode {form} pages of {caps} D={dim}", flush=True)
    free = _pool(200, 200)
    tables = [_table(n, free, lead=i, caps=caps) for i, n in enumerate((500, 129, 33, 700))]
    _Lanes(dev, FORMS[form], 2, dim, 4, tables, 200, 200, caps=caps).check()


@pytest.mark.parametrize("dim", [64, 128])
def test_decode_loose_tables(dev, dim):
    """Pages that hold part of their tokens in the middle of a table, so that groups of 8 tokens are not whole."""
    print(f"quant_decode loose D={dim}", flush=True)
    caps, tables = (8, 64), []
    pages = [[(0, 3), (1, 64), (0, 8), (1, 50), (0, 1)], [(1, 64)] * 5, [(1, 63), (1, 64), (0, 2)], [(1, 16), (1, 40), (0, 8), (1, 64), (0, 4)]]
    free = _pool(60, 60)
    for lane in pages:
        at, entries = 0, []
        for kind, n in lane:
            entries.append((free[kind].pop(0), 1, at, n, caps[kind], kind))
            at += n
        tables.append(entries)
    _Lanes(dev, INT8, 2, dim, 4, tables, 60, 60).check()


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("dim", [64, 128, 40])
def test_decode_tables_with_holes(dev, form, dim):
    """Tokens that a table leaves out, and pages that the storage does not hold, take no part; the latter are reported."""
    print(f"quant_decode holes {form} D={dim}", flush=True)
    free = _pool(60, 60)
    tables = [_table(n, free) for n in (700, 130, 64, 40)]
    lanes = _Lanes(dev, FORMS[form], 2, dim, 4, tables, 60, 60)
    seen = [np.ones(n, bool) for n in lanes.counts]
    short = lanes.tables[0][[0, 1, 2, 4, 5, 6, 7, 8, 9, 10]]   # the fourth page is left out
    seen[0][192:256] = False
    lanes.descs[0] = dev.upload(short)
    lanes.items[0]["descriptors"], lanes.items[0]["descriptor_count"] = lanes.descs[0].ptr, len(short)
    seen[0][int(short[-1]["logical_token_begin"] + short[-1]["valid_tokens"]):] = False
    lanes.check(seen)
    assert lanes.storage.faults() == (0, 0)
    bad = lanes.tables[1].copy()
    bad[1]["slot"] = 60
    seen[1][64:128] = False
    lanes.descs[1] = dev.upload(bad)
    lanes.items[1]["descriptors"] = lanes.descs[1].ptr
    none = lanes.tables[2].copy()
    none["kind"] = 2
    seen[2][:] = False
    lanes.descs[2] = dev.upload(none)
    lanes.items[2]["descriptors"] = lanes.descs[2].ptr
    lanes.check(seen)
    assert lanes.storage.faults() == (dev.INVALID_ARGUMENT, dev.FAULT_DECODE_ITEM)


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("dim", [64, 96, 128, 40])
@pytest.mark.parametrize("kind", ["scales far apart", "rising scales", "sharp", "flat", "negative scale", "zeros", "odd address", "stream"])
def test_decode_values(dev, form, dim, kind):
    print(f"quant_decode {form} D={dim} {kind}", flush=True)
    free = _pool(60, 100)
    tables = [_table(n, free, lead=n % 3) for n in (600, 1500, 70)]
    far = lambda x: (x * np.exp2(np.random.default_rng(1).integers(-14, 10, (len(x), 1, 1)))).astype(np.float16)  # noqa: E731
    rise = lambda x: (x * np.exp2(np.linspace(-14, 12, len(x)))[:, None, None]).astype(np.float16)  # noqa: E731
    more = {"scales far apart": dict(values=far), "rising scales": dict(values=rise), "sharp": dict(query=lambda q: (q * 6).astype(np.float16)),
            "flat": dict(scale=0.0), "negative scale": dict(scale=-0.1), "zeros": dict(keys=np.zeros_like, values=lambda v: v * (np.arange(len(v)) % 3 > 0)[:, None, None].astype(np.float16)),
            "odd address": dict(offset=3), "stream": {}}[kind]
    lanes = _Lanes(dev, FORMS[form], 2, dim, 4, tables, 60, 100, **more)
    lanes.check(stream=dev.Stream() if kind == "stream" else None)


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("dim", [64, 96, 128, 40])
@pytest.mark.parametrize("at", [0, 5, 70, 511, 600, 2047, 2060])
def test_decode_nan_rows(dev, form, dim, at):
    """A K row that is not finite makes its head NaN; a V row that is not makes it NaN where it has a weight, and is left out
    where it has none, also when later keys overtake it."""
    print(f"quant_decode nan rows {form} D={dim} token {at}", flush=True)
    heads, group, n = 2, 4, 2061

    def keys(x):
        x[at, 0] = np.inf
        return x

    free = _pool(60, 100)
    lanes = _Lanes(dev, FORMS[form], heads, dim, group, [_table(n, free)], 60, 100, keys=keys)
    for units in (1, 256):
        got = lanes.run(compute_units=units).view(np.float16)[0]
        assert np.isnan(got[:group]).all() and np.isfinite(got[group:]).all()

    def values(x):
        x[at, 1, 0] = np.nan
        return x

    lanes = _Lanes(dev, FORMS[form], heads, dim, group, [_table(n, free)], 60, 100, values=values)
    for units in (1, 256):
        got = lanes.run(compute_units=units).view(np.float16)[0]
        assert np.isfinite(got[:group]).all() and np.isnan(got[group:]).all()

    # Weights of 0: the token's key is far below the others' for every query.
    def low(x):
        x[:] = np.abs(x) + np.float16(1)
        x[at] = -200
        return x

    lanes = _Lanes(dev, FORMS[form], heads, dim, group, [_table(n, free)], 60, 100, keys=low, values=values, query=lambda q: np.abs(q) + np.float16(1), scale=1.0)
    seen = [np.arange(n) != at]
    for units in (1, 256):
        lanes.check(seen, compute_units=units)


def test_decode_all_scores_minus_infinity(dev):
    """Finite rows whose every score overflows to -inf: nothing weighs, the output is 0."""
    free = _pool(60, 100)
    for dim in (64, 128, 40):
        lanes = _Lanes(dev, E4M3, 1, dim, 2, [_table(100, free)], 60, 100, keys=lambda k: np.full_like(k, -60000), query=lambda q: np.full_like(q, 60000), scale=3e38)
        got = lanes.run().view(np.float16)
        assert np.all(got == 0)


def test_decode_two_at_once(dev):
    """Two streams on one storage, each with its scratch."""
    free = _pool(60, 200)
    a = _Lanes(dev, INT8, 4, 64, 8, [_table(n, free) for n in (3000, 2000)], 60, 200)
    want, bound = a.want()
    streams = [dev.Stream(), dev.Stream()]
    entries, plan = dev.quant_decode_plan(4, 64, 32, 4, a.counts)
    e, items = dev.upload(entries), dev.upload(a.items)
    second = a.items.copy()
    out = dev.upload(np.zeros(a.q.size, np.uint16))
    second["output"] = out.ptr + np.arange(2) * 2 * 32 * 64
    items2 = dev.upload(second)
    work = [dev.DeviceBuffer(plan.workspace_bytes) for _ in streams]
    assert plan.merge_lanes == 2
    for _ in range(5):
        for s, i, w in zip(streams, (items, items2), work):
            a.storage.decode_launch(i.ptr, e.ptr, plan, w.ptr, s)
    for s in streams:
        s.synchronize()
    first = dev.download(a.out.ptr, a.q.shape, np.uint16)
    assert np.array_equal(first, dev.download(out.ptr, a.q.shape, np.uint16))
    assert np.all(np.abs(first.view(np.float16).astype(np.float64) - want) <= bound)


def test_decode_faults(dev):
    """Lanes that are not as planned are skipped and reported; the others are done; lanes of no tokens may hold anything."""
    free = _pool(60, 200)
    for units in (2, 256):
        lanes = _Lanes(dev, INT8, 2, 64, 4, [_table(n, free) for n in (900, 200, 300)] + [[]], 60, 200)
        lanes.items[3] = (1, 7, 0, 99, 1, 0, 1, 1.0)
        lanes.check(compute_units=units)
        assert lanes.storage.faults() == (0, 0)
        for change in (dict(token_count=901), dict(descriptors=0), dict(descriptor_count=0), dict(layer=2), dict(query=0), dict(output=0)):
            keep = lanes.items.copy()
            for name, value in change.items():
                lanes.items[0][name] = value
            dev.copy_to_device(lanes.out.ptr, np.full(lanes.q.size, 0x4321, np.uint16))
            got = lanes.run(compute_units=units)
            assert lanes.storage.faults() == (dev.INVALID_ARGUMENT, dev.FAULT_DECODE_ITEM), change
            assert np.all(got[0] == 0x4321)
            want, bound = lanes.want()
            assert np.all(np.abs(got[1:3].view(np.float16).astype(np.float64) - want[1:3]) <= bound[1:3])
            lanes.items = keep


def test_decode_refusals(dev):
    s = dev.QuantStorage(2, 2, 64, 4, 4, INT8)
    entries, plan = s.decode_plan([100, 9000], 8)
    assert plan.merge_lanes == 1
    buf, bad = dev.DeviceBuffer(1 << 20), dev.INVALID_ARGUMENT
    call = lambda p, items=buf.ptr, e=buf.ptr, w=buf.ptr: dev.lib().kimkv_quant_decode_batch(s.handle, items, e, p, w, None)  # noqa: E731

    def changed(**fields):
        p = dev.QuantPlan.from_buffer_copy(plan)
        for name, value in fields.items():
            setattr(p, name, value)
        return p

    assert call(plan, items=None) == bad and call(plan, e=None) == bad and call(plan, w=None) == bad
    assert call(plan, e=buf.ptr + 8) == bad and call(plan, w=buf.ptr + 8) == bad
    assert dev.lib().kimkv_quant_decode_batch(s.handle, buf.ptr, buf.ptr, None, buf.ptr, None) == bad
    for fields in (dict(kv_heads=4), dict(head_dim=128), dict(query_heads=0), dict(query_heads=7), dict(unit_count=plan.unit_count + 1), dict(entry_bytes=0),
                   dict(workspace_bytes=0), dict(slot_count=0), dict(merge_lanes=0)):
        assert call(changed(**fields)) == bad, fields
    assert call(s.decode_plan([0, 0], 8)[1], items=None, e=None, w=None) == dev.OK


# ---- sampling ----------------------------------------------------------------


def _draw(x, u, temperature, top_k, top_p, min_p):
    """(token, probability) by the definition; numpy's extended precision."""
    x = np.where(np.isnan(x), -np.inf, x).astype(np.longdouble)
    if np.isposinf(x).any():
        x = np.where(np.isposinf(x), np.longdouble(0), -np.inf)
    if np.isneginf(x).all():
        return 0xFFFFFFFF, 0.0
    order = np.argsort(-x, kind="stable")
    if temperature == 0:
        return int(order[0]), 1.0
    w = np.exp((x - x[order[0]]) / np.longdouble(np.float32(temperature)))
    order = order[:top_k or None]
    if top_p < 1:
        sums = np.cumsum(w[order])
        order = order[:int(np.searchsorted(sums, np.longdouble(np.float32(top_p)) * sums[-1])) + 1]
    order = np.sort(order[w[order] >= np.longdouble(np.float32(min_p))])
    sums = np.cumsum(w[order])
    at = min(int(np.searchsorted(sums, np.longdouble(np.float32(u)) * sums[-1], side="right")), len(order) - 1)
    return int(order[at]), float(w[order[at]] / sums[-1])


def _sample(dev, logits, rules, uniforms, offset=0, probabilities=True, stream=None):
    rows, vocab = logits.shape
    buf = dev.upload(np.concatenate([np.zeros(offset, np.float32), logits.astype(np.float32).reshape(-1)]))
    table = np.zeros(rows, dtype=dev.SAMPLE_RULE)
    for name, column in zip(("temperature", "top_k", "top_p", "min_p"), zip(*rules)):
        table[name] = column
    r, u = dev.upload(table), dev.upload(np.asarray(uniforms, np.float32))
    tokens, chance = dev.upload(np.zeros(rows, np.uint32)), dev.upload(np.full(rows, 7, np.float32))
    work = dev.DeviceBuffer(max(1, dev.sample_workspace_bytes(rows, vocab)))
    dev.sample(buf.ptr + 4 * offset, rows, vocab, r.ptr, u.ptr, tokens.ptr, chance.ptr if probabilities else 0, work.ptr, stream)
    dev.sync(stream)
    return dev.download(tokens.ptr, (rows,), np.uint32), dev.download(chance.ptr, (rows,), np.float32)


def _check_sample(dev, logits, rules, uniforms, **more):
    tokens, chance = _sample(dev, logits, rules, uniforms, **more)
    for r in range(len(logits)):
        token, p = _draw(logits[r].astype(np.float32), uniforms[r], *rules[r])
        assert tokens[r] == token, (r, rules[r], int(tokens[r]), token)
        # One rounding to 32 bits, weights to 2^-47 of the highest, sums of them.
        assert more.get("probabilities") is False or abs(chance[r] - p) <= 2.0 ** -24 * p + logits.shape[1] * 2.0 ** -46, (r, chance[r], p)


SETTINGS = [(1.0, 0, 1.0, 0.0), (0.7, 50, 1.0, 0.0), (1.0, 0, 0.9, 0.0), (0.8, 40, 0.95, 0.0), (1.3, 0, 1.0, 0.05), (1.0, 300, 0.5, 0.01), (0.0, 0, 1.0, 0.0), (0.0, 5, 0.3, 0.5),
            (1.0, 1, 1.0, 0.0), (5.0, 3000, 0.99, 0.0), (0.05, 20, 0.9, 0.0), (1.0, 2, 0.001, 0.0), (1.0, 0, 1.0, 1.0), (100.0, 0, 0.7, 0.2), (1e-30, 0, 0.9, 0.0), (1e30, 70, 0.5, 0.0)]


@pytest.mark.parametrize("vocab", [1, 2, 3, 63, 64, 100, 1000, 4096, 4099, 20000, 32000, 50255, 128000, 300007])
@pytest.mark.parametrize("kind", ["normal", "peaks", "masked", "few values"])
def test_sample(dev, vocab, kind):
    print(f"sample V={vocab} {kind}", flush=True)
    rng = np.random.default_rng(vocab + len(kind))
    rows = len(SETTINGS)
    logits = (2 * rng.standard_normal((rows, vocab))).astype(np.float32)
    if kind == "peaks":
        logits[:, rng.integers(0, vocab, 5)] += 12
    if kind == "masked":
        logits[rng.random((rows, vocab)) < 0.7] = -np.inf
        logits[:, vocab // 2] = 1
    if kind == "few values":
        logits = np.rint(logits)
    _check_sample(dev, logits, SETTINGS, rng.random(rows).astype(np.float32), offset=vocab % 4)


@pytest.mark.parametrize("vocab", [5, 3000, 40000])
def test_sample_equal_logits(dev, vocab):
    """All alike: the cuts fall among equals, of which the lowest are kept; -0 equals 0."""
    print(f"sample equal V={vocab}", flush=True)
    logits = np.zeros((len(SETTINGS), vocab), np.float32)
    logits[:, ::2] = -0.0
    logits[-3:] = 1e30
    _check_sample(dev, logits, SETTINGS, np.linspace(0, 0.999, len(SETTINGS)).astype(np.float32))


def test_sample_narrow_and_wide_logits(dev):
    """Bins that hold more tokens than are sorted at once, again and again: thousands of neighbouring numbers beside far ones."""
    vocab = 60000
    rng = np.random.default_rng(3)
    rules, rows = [], []
    for spread in (1e-6, 1e-3, 1e30):
        x = 1 + spread * rng.random(vocab)
        x[::7] = np.float32(1) + np.float32(2.0 ** -23) * rng.integers(0, 900, len(x[::7]))
        x[5] = -3e38 if spread < 1 else 1
        for rule in ((1.0, 30000, 1.0, 0.0), (1.0, 0, 0.4, 0.0), (2.0, 20000, 0.7, 0.0), (1.0, 59999, 1.0, 0.0), (1e36, 10, 0.5, 0.0)):
            rows.append(x.astype(np.float32))
            rules.append(rule)
    _check_sample(dev, np.array(rows), rules, rng.random(len(rows)).astype(np.float32))


def test_sample_odd_rows(dev):
    """Rows of -inf and NaN, of +inf, of one token; random numbers at the ends; invalid rules and random numbers."""
    vocab = 3001
    rng = np.random.default_rng(4)
    base = rng.standard_normal(vocab).astype(np.float32)
    rows, rules, uniforms = [], [], []

    def add(x, rule=(1.0, 0, 1.0, 0.0), u=0.5):
        rows.append(x)
        rules.append(rule)
        uniforms.append(u)

    add(np.full(vocab, -np.inf))
    add(np.full(vocab, np.nan))
    one = np.full(vocab, -np.inf)
    one[2999] = -80
    for rule in SETTINGS:
        add(one, rule, 0.999)
    some = base.copy()
    some[[5, 2000, 3000]] = np.inf
    some[7] = np.nan
    for rule in SETTINGS:
        add(some, rule, 0.6)
    nan = base.copy()
    nan[::3] = np.nan
    for rule in SETTINGS:
        add(nan, rule, 0.3)
    for rule in SETTINGS:
        add(base, rule, 0.0)
        add(base, rule, 1 - 2.0 ** -24)
        add(base, rule, 1e-42)
    huge = base.copy()
    huge[[0, 1, 2]] = 3.4e38, -3.4e38, 3.4e38
    for rule in SETTINGS:
        add(huge, rule, 0.5)
    _check_sample(dev, np.array(rows), rules, uniforms)
    invalid = [(-1.0, 0, 1.0, 0.0), (np.inf, 0, 1.0, 0.0), (np.nan, 0, 1.0, 0.0), (1.0, 0, 0.0, 0.0), (1.0, 0, 1.1, 0.0), (1.0, 0, np.nan, 0.0), (1.0, 0, -0.5, 0.0),
               (1.0, 0, 1.0, -0.1), (1.0, 0, 1.0, 1.5), (1.0, 0, 1.0, np.nan)]
    tokens, chance = _sample(dev, np.tile(base, (len(invalid) + 3, 1)), invalid + [(1.0, 0, 1.0, 0.0)] * 3, [0.5] * len(invalid) + [1.0, -0.25, np.nan])
    assert np.all(tokens == dev.NO_TOKEN) and np.all(chance == 0)


def test_sample_without_probabilities_on_a_stream(dev):
    rng = np.random.default_rng(5)
    logits = rng.standard_normal((3, 5000)).astype(np.float32)
    _check_sample(dev, logits, SETTINGS[1:4], rng.random(3).astype(np.float32), probabilities=False, stream=dev.Stream())


def test_sample_many_rows_and_every_uniform(dev):
    """One row's distribution over evenly spread random numbers: each token as often as its weight says, in their order."""
    rng = np.random.default_rng(6)
    vocab, rows = 200, 4000
    x = rng.standard_normal(vocab).astype(np.float32)
    uniforms = ((np.arange(rows) + 0.5) / rows).astype(np.float32)
    tokens, _ = _sample(dev, np.tile(x, (rows, 1)), [(1.0, 50, 0.9, 0.0)] * rows, uniforms)
    want = [_draw(x, u, 1.0, 50, 0.9, 0.0)[0] for u in uniforms]
    assert np.array_equal(tokens, want) and np.all(np.diff(tokens.astype(int)) >= 0) and len(set(tokens.tolist())) > 10


# ---- a token step --------------------------------------------------------------


def test_token_step(dev):
    """Append, decode, logits and sampling as a server runs them, eager and captured in a graph with eager work between the
    replays; the step's new tokens count."""
    hip = _hip()
    heads, dim, group, vocab = 4, 64, 8, 20000
    counts = [900, 901, 1200, 60, 5000]
    free = _pool(64, 200)
    lanes = _Lanes(dev, INT8, heads, dim, group, [_table(n, free) for n in counts], 64, 200)
    n, row, stream = len(counts), heads * dim, dev.Stream()
    new = dev.DeviceBuffer(2 * 2 * n * row)
    jobs = np.zeros(n, dtype=dev.APPEND_JOB)
    for i, t in enumerate(lanes.tables):   # each lane's last token written anew
        e = t[-1]
        jobs[i] = (new.ptr + 2 * i * row, new.ptr + 2 * (n + i) * row, 0, row, 1, 1, 1, e["slot"], 0, e["valid_tokens"] - 1, 0, e["kind"], 0)
    job_buf, items = dev.upload(jobs), dev.upload(lanes.items)
    entries, plan = lanes.storage.decode_plan(counts, heads * group)
    e, work = dev.upload(entries), dev.DeviceBuffer(plan.workspace_bytes + 16)
    logits, adjusted, tokens, chance = (dev.DeviceBuffer(4 * k) for k in (n * vocab, n * vocab, n, n))
    scratch = dev.DeviceBuffer(dev.logits_workspace_bytes(n, vocab) + 16)
    table = np.zeros(n, dtype=dev.LOGITS_RULE)
    table["repetition_penalty"] = 1.0
    rules, sampling, uniforms = dev.upload(table), np.zeros(n, dtype=dev.SAMPLE_RULE), dev.DeviceBuffer(4 * n)
    sampling[:] = [(0.8, 0.9, 0.01, 50)] * n
    sampling_buf = dev.upload(sampling)
    draw_work = dev.DeviceBuffer(dev.sample_workspace_bytes(n, vocab) + 16)

    def step():
        lanes.storage.append_launch(job_buf.ptr, n, 1, stream)
        lanes.storage.decode_launch(items.ptr, e.ptr, plan, work.ptr, stream)
        dev.logits_adjust(logits.ptr, n, vocab, rules.ptr, adjusted.ptr, 0, scratch.ptr, stream)
        dev.sample(adjusted.ptr, n, vocab, sampling_buf.ptr, uniforms.ptr, tokens.ptr, chance.ptr, draw_work.ptr, stream)

    def results():
        stream.synchronize()
        return [dev.download(lanes.out.ptr, lanes.q.shape, np.uint16), dev.download(tokens.ptr, (n,), np.uint32), dev.download(chance.ptr, (n,), np.float32)]

    graph, runs, handle = ctypes.c_void_p(), ctypes.c_void_p(), ctypes.c_void_p(stream.handle)
    assert hip.hipStreamBeginCapture(handle, 0) == 0
    step()
    assert hip.hipStreamEndCapture(handle, ctypes.byref(graph)) == 0
    assert hip.hipGraphInstantiate(ctypes.byref(runs), graph, None, None, 0) == 0
    rng = np.random.default_rng(4)
    ends = np.cumsum(counts) - 1
    for _ in range(4):
        kv = _fp16(rng, 2, n, heads, dim)
        x, u = (2 * rng.standard_normal((n, vocab))).astype(np.float32), rng.random(n).astype(np.float32)
        for buf, a in ((new, _bits(kv)), (logits, x), (uniforms, u)):
            dev.copy_to_device(buf.ptr, a)
        assert hip.hipGraphLaunch(runs, handle) == 0
        replayed = results()
        for buf, size in ((lanes.out, 2 * lanes.q.size), (tokens, 4 * n), (chance, 4 * n)):
            dev.copy_to_device(buf.ptr, np.zeros(size, np.uint8))
        step()
        for a, b in zip(replayed, results()):
            assert np.array_equal(a, b)
        lanes.kv[:, ends] = held(kv, INT8)
        want, bound = lanes.want()
        assert np.all(np.abs(replayed[0].view(np.float16).astype(np.float64) - want) <= bound)
        assert [_draw(x[i], u[i], 0.8, 50, 0.9, 0.01)[0] for i in range(n)] == replayed[1].tolist()
    assert lanes.storage.faults() == (0, 0)
    hip.hipGraphExecDestroy(runs)
    hip.hipGraphDestroy(graph)
    stream.destroy()


def test_promoted_and_read_back_for_a_prefill(dev):
    """Small pages promoted, one layer read back into pages of fp16, and the prompt's next chunk attended there: what the
    quantised decode of the chunk's last token gives, to both roundings."""
    heads, dim, group, prompt = 2, 64, 4, 128
    form, rng = INT8, np.random.default_rng(11)
    c = _Cache(dev, form, heads, dim, layers=1, micro=24, extent=6)
    jobs = np.zeros(2, dtype=dev.PROMOTION_JOB)
    for i in range(2):
        jobs[i] = (np.arange(8 * i, 8 * i + 8), 4 - i)
    c.storage.promote_batch(jobs)
    table = np.array([(4, 1, 0, 64, 64, 1), (3, 1, 64, 64, 64, 1)], dtype=helpers.DESC)
    rows = c.storage.gather(table, prompt)
    plain = dev.Storage(1, heads, dim, 1, 2)
    buf, row = dev.upload(rows), heads * dim
    plain.append_batch(np.array([(buf.ptr + 2 * 64 * i * row, buf.ptr + 2 * (prompt + 64 * i) * row, 0, row, 0, 1, 64, i, 0, 0, 0, 1, 0) for i in range(2)],
                                dtype=dev.APPEND_JOB))
    fp16 = np.array([(0, 1, 0, 64, 64, 1), (1, 1, 64, 64, 64, 1)], dtype=helpers.DESC)
    q = _fp16(rng, heads * group, dim, scale=2.0)
    qbuf, outs = dev.upload(_bits(q)), [dev.DeviceBuffer(2 * q.size) for _ in range(2)]
    tables = [dev.upload(fp16), dev.upload(table)]
    item = np.zeros(1, dtype=dev.PREFILL_ITEM)
    item[0] = (tables[0].ptr, 2, prompt, 1, 0, qbuf.ptr, outs[0].ptr, 1.0 / math.sqrt(dim))
    _, prefix, blocks = plain.prefill_plan([1], heads * group)
    i, p = dev.upload(item), dev.upload(prefix)
    plain.prefill_launch(i.ptr, p.ptr, 1, blocks, heads * group)
    decode = np.zeros(1, dtype=dev.DECODE_ITEM)
    decode[0] = (tables[1].ptr, 2, prompt, 0, qbuf.ptr, 0, outs[1].ptr, 1.0 / math.sqrt(dim))
    entries, plan = c.storage.decode_plan([prompt], heads * group)
    d, e = dev.upload(decode), dev.upload(entries)
    c.storage.decode_launch(d.ptr, e.ptr, plan, 0)
    dev.sync()
    a, b = (dev.download(o.ptr, q.shape, np.uint16).view(np.float16).astype(np.float64) for o in outs)
    # Values rounded to fp16 on the way: each is off by FP16 of itself, a score by that of its terms.
    values = c.pages[0][0, :, :prompt]
    for j in range(heads * group):
        k, v = values[0, :, j // group], values[1, :, j // group]
        s = k @ q[j].astype(np.float64) / math.sqrt(dim)
        p = np.exp(s - s.max())
        p /= p.sum()
        size = p @ np.abs(v)
        off = (np.abs(k) @ np.abs(q[j].astype(np.float64))).max() / math.sqrt(dim) * (FP16 + 70 * 2.0 ** -24)
        assert np.all(np.abs(a[j] - b[j]) <= 2 * (FP16 * np.abs(p @ v) + TINY) + size * (FP16 + 2 * off + 2.0 ** -12))


# ---- launches and sizes at which kernels take other ways ------------------------


@pytest.mark.parametrize("form,heads,dim", [("int8", 3, 64), ("e4m3", 5, 33), ("int8", 3, 96), ("e4m3", 20, 12), ("int8", 5, 40), ("e4m3", 3, 128)])
def test_pages_of_many_layers(dev, form, heads, dim):
    """Launches that fill the chip, whose workgroups take several heads, the last ones fewer; appended, read back whole and
    in part."""
    print(f"quant pages of many layers {form} H={heads} D={dim}", flush=True)
    c = _Cache(dev, FORMS[form], heads, dim, layers=128, micro=14, extent=8)
    kv = _fp16(np.random.default_rng(5), 128, 2, ROWS, heads, dim)
    buf = dev.upload(_bits(kv))
    c.storage.append_batch(c.jobs_of(buf.ptr, ROWS, RUNS, COWS))
    c.expect(kv, RUNS, COWS)
    c.check()
    part = c.storage.gather(c.tables[1], 300, first_token=37).view(np.float16).reshape(128, 2, 300, heads, dim)
    _same(part, read(c.pages[1][:, :, 37:337]))
    assert c.storage.faults() == (0, 0)


@pytest.mark.parametrize("form,heads,dim", [("int8", 3, 64), ("e4m3", 3, 33), ("int8", 5, 12)])
def test_promote_many_layers(dev, form, heads, dim):
    print(f"quant_promote many layers {form} H={heads} D={dim}", flush=True)
    c = _Cache(dev, FORMS[form], heads, dim, layers=512, micro=16, extent=2)
    jobs = np.zeros(2, dtype=dev.PROMOTION_JOB)
    order = np.random.default_rng(3).permutation(16)
    for i in range(2):
        jobs[i] = (order[8 * i:8 * i + 8], 1 - i)
        rows = np.concatenate([np.arange(8) + 8 * s for s in order[8 * i:8 * i + 8]])
        c.pages[1][:, :, 64 * (1 - i):64 * (2 - i)] = c.pages[0][:, :, rows]
    c.storage.promote_batch(jobs)
    c.check()
    assert c.storage.faults() == (0, 0)


@pytest.mark.parametrize("form,dim", [("int8", 128), ("e4m3", 128)])
def test_pages_past_32_bits(dev, form, dim):
    """Pages that lie more than 2^32 bytes into the storage, small ones behind as many."""
    print(f"quant pages past 32 bits {form} D={dim}", flush=True)
    heads, group, micro, extent = 8, 2, 270000, 35000   # 4.5 and 4.6 GB
    free = [[micro - 1, micro - 7], [extent - 1, 3, extent - 5]]
    lanes = _Lanes(dev, FORMS[form], heads, dim, group, [_table(205, free)], micro, extent, layers=1, layer=0)
    lanes.check()
    rows = lanes.storage.gather(lanes.tables[0], 205).view(np.float16).reshape(2, 205, heads, dim)
    _same(rows, read(lanes.kv))
    assert lanes.storage.faults() == (0, 0)


LONG_LISTS = [(1.0, 600, 1.0, 0.0), (0.7, 1000, 0.95, 0.0), (1.0, 1024, 0.5, 0.001), (3.0, 1024, 1.0, 0.0), (1.0, 1025, 0.9, 0.0), (0.3, 1000, 1.0, 0.0), (1.0, 0, 1.0, 0.001),
              (1.0, 0, 1.0, 0.2), (1.5, 0, 1.0, 1e-6), (1.0, 0, 0.3, 0.0), (1.0, 0, 0.999, 0.01)]


@pytest.mark.parametrize("vocab", [1500, 4096, 32000, 50255, 270001])
@pytest.mark.parametrize("kind", ["normal", "falling", "rising", "one run", "blocks", "below zero", "not there"])
def test_sample_long_lists(dev, vocab, kind):
    """Lists of about as many tokens as are sorted at once; rows whose highest tokens lie beside each other, and in one
    place of every 256, so that many share a part of the row."""
    print(f"sample long lists V={vocab} {kind}", flush=True)
    rng = np.random.default_rng(vocab + len(kind))
    x = (2 * rng.standard_normal((len(LONG_LISTS), vocab))).astype(np.float32)
    if kind in ("falling", "rising"):
        x = np.sort(x, 1)[:, ::-1 if kind == "falling" else 1]
    if kind == "one run":
        x[:, vocab // 3:vocab // 3 + 1100] += 9
    if kind == "blocks":
        x[:, 77::256] += 9
    if kind == "below zero":
        x -= 300
    if kind == "not there":
        x[rng.random(x.shape) < 0.4] = np.nan
        x[rng.random(x.shape) < 0.4] = -np.inf
    _check_sample(dev, x, LONG_LISTS, rng.random(len(x)).astype(np.float32), offset=3)


def test_sample_rows_past_32_bits(dev):
    """The last of rows that together hold more than 2^32 logits; the others hold whatever the memory does."""
    print("sample rows past 32 bits", flush=True)
    vocab, rows = 1 << 17, (1 << 15) + 2
    x = (2 * np.random.default_rng(8).standard_normal((2, vocab))).astype(np.float32)
    buf = dev.DeviceBuffer(4 * rows * vocab)
    dev.copy_to_device(buf.ptr + 4 * (rows - 2) * vocab, x)
    table = np.zeros(rows, dtype=dev.SAMPLE_RULE)
    table[:] = (1.0, 1.0, 0.0, 1)
    table[-2:] = [(0.9, 0.95, 0.0, 50), (1.0, 0.9, 0.0, 0)]
    u = np.full(rows, 0.625, np.float32)
    r, d = dev.upload(table), dev.upload(u)
    tokens = dev.upload(np.zeros(rows, np.uint32))
    dev.sample(buf.ptr, rows, vocab, r.ptr, d.ptr, tokens.ptr)
    dev.sync()
    got = dev.download(tokens.ptr, (rows,), np.uint32)[-2:]
    assert got.tolist() == [_draw(x[0], u[0], 0.9, 50, 0.95, 0.0)[0], _draw(x[1], u[0], 1.0, 0, 0.9, 0.0)[0]]


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("dim,group", [(64, 2), (96, 3), (128, 2), (64, 16)])
def test_decode_many_lanes(dev, form, dim, group):
    """More units than compute units, of lanes in one part and in several; pages of all kinds, a lane of none."""
    print(f"quant_decode many lanes {form} D={dim} G={group}", flush=True)
    rng = np.random.default_rng(12)
    counts = [int(n) for n in np.exp(rng.uniform(0, math.log(1500), 110))] + [0, 2900, 4100]
    free = _pool(1400, 500)
    tables = [_table(n, free, lead=i % 4 if i % 3 == 0 else 0, small=i % 17 == 5 and n < 300) for i, n in enumerate(counts)]
    lanes = _Lanes(dev, FORMS[form], 3, dim, group, tables, 1400, 500)
    _, plan = lanes.storage.decode_plan(lanes.counts, 3 * group)
    assert plan.unit_count > lanes.storage.info().compute_units and plan.merge_lanes > 0
    lanes.check()
    # Query rows at an odd address.
    lanes = _Lanes(dev, FORMS[form], 3, dim, group, tables, 1400, 500, offset=3, seed=5)
    lanes.check()
    assert lanes.storage.faults() == (0, 0)


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("dim", [8, 64])
def test_append_every_scale(dev, form, dim):
    """Rows whose largest value is each finite number above 0, in long runs and, the last ones, as single tokens."""
    print(f"quant_append every scale {form} D={dim}", flush=True)
    c = _Cache(dev, FORMS[form], 1, dim, layers=1, micro=1, extent=496)
    rng = np.random.default_rng(2)
    largest = np.arange(31744, dtype=np.uint16).view(np.float16)
    kv = (largest[None, None, :, None, None].astype(np.float64) * rng.uniform(-1, 1, (1, 2, 31744, 1, dim))).astype(np.float16)
    kv[0, 0, :, 0, dim - 1] = largest
    kv[0, 1, :, 0, 3] = -largest
    runs = [(64 * i, 64, 1, i, 0) for i in range(490)] + [(31360 + i, 1, 1, 490 + i // 64, i % 64) for i in range(384)]
    buf = dev.upload(_bits(kv))
    c.storage.append_batch(c.jobs_of(buf.ptr, 31744, runs))
    c.expect(kv, runs)
    c.check()
    assert c.storage.faults() == (0, 0)


MANY_OF_TOP_K = [(1.0, 3000, 0.9, 0.0), (1.0, 3000, 0.9, 0.01), (0.01, 2000, 0.9, 0.0), (0.05, 3000, 0.5, 0.1), (2.0, 20000, 0.99, 1e-5), (1.0, 1100, 0.999999, 0.0),
                 (30.0, 4000, 0.5, 0.0), (1.0, 31999, 0.7, 0.0), (0.7, 1500, 0.01, 0.0)]


@pytest.mark.parametrize("vocab", [3001, 32000, 140001])
@pytest.mark.parametrize("kind", ["normal", "falling", "peaks", "few values", "not there"])
def test_sample_top_p_of_many(dev, vocab, kind):
    """Top-p of more tokens than are listed at once; of fewer that weigh anything than top_k; of many equal ones."""
    print(f"sample top-p of many V={vocab} {kind}", flush=True)
    rng = np.random.default_rng(vocab + len(kind))
    x = (2 * rng.standard_normal((len(MANY_OF_TOP_K), vocab))).astype(np.float32)
    if kind == "falling":
        x = np.sort(x, 1)[:, ::-1]
    if kind == "peaks":
        x[:, rng.integers(0, vocab, 9)] += 12
    if kind == "few values":
        x = np.rint(2 * x) / 2
    if kind == "not there":
        x[rng.random(x.shape) < 0.5] = -np.inf
        x[rng.random(x.shape) < 0.1] = np.nan
    for u in (0.0, 0.3, 1 - 2.0 ** -24):
        _check_sample(dev, x, MANY_OF_TOP_K, np.full(len(x), u, np.float32), offset=1)


@pytest.mark.parametrize("vocab", [3001, 6000, 40000])
def test_sample_min_p_of_far_logits(dev, vocab):
    """Temperatures at which T log min_p is past the largest number of 32 bits, of logits as far apart, so that min-p still
    leaves tokens out; alone, beside top-p, beside a long top_k and both."""
    print(f"sample min-p of far logits V={vocab}", flush=True)
    rng = np.random.default_rng(vocab)
    rows, rules = [], []
    for temperature in (2e37, 1e38, 3e38):
        for min_p in (0.5, 0.2, 0.02, 1e-4):
            for top_k, top_p in ((0, 1.0), (0, 0.9), (2500, 1.0), (2500, 0.9)):
                x = rng.uniform(-3.3e38, 3.3e38, vocab)
                if top_k == 0 and top_p == 1.0:   # a half that min-p leaves out, in front
                    x = np.where(np.arange(vocab) < vocab // 2, -3e38, 3e38)
                rows.append(x.astype(np.float32))
                rules.append((temperature, top_k, top_p, min_p))
    uniforms = rng.random(len(rows)).astype(np.float32)
    uniforms[::3] = 0
    _check_sample(dev, np.array(rows), rules, uniforms)


def test_sample_min_p_beside_the_last_bits_of_weights(dev):
    """Tokens just above and just below a min_p of a few units of 2^-46, drawn by a random number of 0 and by others: the
    first that is kept, wherever the weights' last bit puts it.  Ordinary rows go before, whose answers are not these rows'."""
    print("sample min-p beside the last bits", flush=True)
    vocab = 20000
    rng = np.random.default_rng(21)
    ordinary = (2 * rng.standard_normal(vocab)).astype(np.float32)
    border = np.full(vocab, -60, np.float32)
    border[:4096] = np.log(0.97e-13)
    border[4096:8192] = np.log(1.03e-13)
    border[15000] = 0
    rows = np.array([ordinary] * 600 + [border] * 600)
    rules = [(1.0, 0, 1.0, 0.0)] * 600 + [(1.0, 0, 1.0, 1e-13), (2.0, 0, 1.0, 1e-13), (1.0, 9000, 1.0, 1e-13)] * 200
    rows[601::3] *= 2
    uniforms = rng.random(1200).astype(np.float32)
    uniforms[600:900] = 0
    uniforms[900:] = 0.25 + 0.5 * uniforms[900:]
    tokens, chance = _sample(dev, rows, rules, uniforms)
    assert set(tokens[600:900].tolist()) == {4096} and set(tokens[900:].tolist()) == {15000}
    # A token's weight is off by half a unit at most.
    assert np.all(np.abs(chance[600:900] - 1.03e-13) <= 2.0 ** -47 + 2.0 ** -24 * 1.03e-13) and np.all(chance[900:] > 0.999)


@pytest.mark.parametrize("vocab", [1500, 5000])
def test_sample_logits_below_the_normal_numbers(dev, vocab):
    """The highest logit an odd multiple of 2^-149, of which half is no number, above and below 0."""
    print(f"sample below the normal numbers V={vocab}", flush=True)
    rng = np.random.default_rng(vocab)
    rules = [(1.0, 0, 0.5, 0.0), (1.0, 0, 0.9, 0.5), (1.0, 1200, 1.0, 0.0), (1.0, 1200, 0.3, 0.0), (1.0, 7, 1.0, 0.0), (2.0 ** -149, 0, 0.9, 0.0), (2.0 ** -149, 1300, 0.5, 0.0),
             (2.0 ** -149, 0, 1.0, 0.1), (2.0 ** -147, 0, 0.7, 0.01), (0.0, 0, 1.0, 0.0), (1e-44, 0, 1.0, 0.0)]
    for highest, low in ((3, -2), (1, -40), (-1, -6), (5, 4)):
        x = rng.integers(low, highest, (len(rules), vocab)) * 2.0 ** -149
        x[:, vocab - 7] = highest * 2.0 ** -149
        for u in (0.0, 0.4, 1 - 2.0 ** -24):
            _check_sample(dev, x, rules, np.full(len(rules), u, np.float32))


@pytest.mark.parametrize("form,heads,dim", [("int8", 2, 64), ("e4m3", 2, 12)])
def test_append_jobs_of_too_many_layers(dev, form, heads, dim):
    """A job that begins within the storage's layers and ends past them, or is of more layers than the launch, is skipped in
    every layer, its copy too; a job of no layers is none."""
    c = _Cache(dev, FORMS[form], heads, dim, layers=3)
    kv = _fp16(np.random.default_rng(14), 3, 2, 64, heads, dim)
    buf = dev.upload(_bits(kv))
    good = [(0, 1, 0, 0, 0), (1, 20, 1, 0, 3)]
    for name, change, most in (("one past", dict(layer_begin=1, layer_count=3), 3), ("many past", dict(layer_begin=2, layer_count=2), 3),
                               ("all but wrapped", dict(layer_begin=1, layer_count=0xFFFFFFFF), 3), ("more than the launch", dict(layer_count=3), 2)):
        print(f"quant_append layers {name}", flush=True)
        for bad in ((21, 1, 0, 2, 4), (22, 12, 1, 2, 9)):
            jobs = c.jobs_of(buf.ptr, 64, good + [bad], {2: (0, 5, 4)}, layer_count=most)
            for field, value in change.items():
                jobs[2][field] = value
            held_jobs = dev.upload(jobs)
            c.storage.append_launch(held_jobs.ptr, len(jobs), most)
            dev.sync()
            assert c.storage.faults() == (dev.INVALID_ARGUMENT, dev.FAULT_APPEND_JOB), name
        c.expect(kv[:most], good)
        c.check()
    jobs = c.jobs_of(buf.ptr, 64, good + [(21, 1, 0, 2, 4)])
    jobs[2]["layer_begin"], jobs[2]["layer_count"] = 0xFFFFFFFF, 0
    c.storage.append_batch(jobs)
    c.expect(kv, good)
    c.check()
    assert c.storage.faults() == (0, 0)


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("dim", [64, 96, 128, 40])
@pytest.mark.parametrize("size", [2.0 ** -12, 2.0 ** -17])
@pytest.mark.parametrize("kind", ["one row", "rows in all places", "overtaken"])
def test_decode_far_values_without_weight(dev, form, dim, size, kind):
    """Rows of V of up to 65504 that weigh nothing cost the others, far smaller, no bits: their keys lie far below, or later
    keys overtake them."""
    print(f"quant_decode far values {form} D={dim} {size} {kind}", flush=True)
    free = _pool(60, 100)
    tables = [_table(n, free, lead=n % 3) for n in (600, 1500, 70)]
    total = 600 + 1500 + 70
    far = np.zeros(total, bool)
    far[{"one row": [3, 603, 2103], "rows in all places": range(5, total, 13), "overtaken": [*range(20), *range(600, 640), *range(2100, 2110)]}[kind]] = True

    def keys(k):
        if kind == "overtaken":
            return np.where(far[:, None, None], 0, 3 + 0.1 * k.astype(np.float32)).astype(np.float16)
        return np.where(far[:, None, None], np.float16(-3), k)

    def values(v):
        return np.where(far[:, None, None], np.clip(30000 * v.astype(np.float32), -65504, 65504), size * v.astype(np.float32)).astype(np.float16)

    _Lanes(dev, FORMS[form], 2, dim, 4, tables, 60, 100, keys=keys, values=values, query=np.abs).check()


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("dim", [64, 96, 128, 40])
def test_decode_largest_values(dev, form, dim):
    """Rows of V about the largest numbers of fp16, which their codes and scales can be past: finite outputs, as what is read
    back; in one part and merged."""
    print(f"quant_decode largest {form} D={dim}", flush=True)
    free = _pool(60, 100)
    tables = [_table(n, free, lead=n % 3) for n in (1, 600, 2500, 70)]

    def values(v):
        big = np.where(np.random.default_rng(3).random(v.shape) < 0.9, 65504, 65000) * np.where(np.arange(dim) % 2, 1, -1)
        return big.astype(np.float16)

    lanes = _Lanes(dev, FORMS[form], 2, dim, 4, tables, 60, 100, values=values)
    want, bound = lanes.want()
    assert np.abs(want).max() > 65504
    for units in (256, 2):
        got = lanes.run(compute_units=units).view(np.float16).astype(np.float64)
        assert np.isfinite(got).all() and np.all(np.abs(got - np.clip(want, -65504, 65504)) <= bound)
