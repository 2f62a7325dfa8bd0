"""A token step on a cache of 8 bits, and the token it ends with, as cases that can be timed and checked.

  write    rows of K and V quantised into the pages of a cache (partial tails copied first where a request leaves a
           shared page), and the pages read back
  promote  eight small pages copied into one large page, and the large pages read back
  read     one request's pages back as rows of fp16
  decode   one layer's attention of one new token a lane over the pages
  sample   the next token of each row of logits from a given random number: temperature, top-k, top-p, min-p

A row of a cache is the D values of one token's K or V of one head: codes of 8 bits (whole numbers or e4m3) and one
scale.  `own` chooses who computes: False, elementary torch operations on tensors; True, the library's entry points on
its page storage.  Lengths, page tables and rules follow from the case alone (`mix`), contents from the seed.
"""
import math
import random

import numpy as np
import torch

own = False

MICRO, EXTENT = 8, 64
LARGEST = {"int8": 127.0, "e4m3": 448.0}


def listed():
    return [
        # A serving batch's token step; one lane in four leaves a page it shares.
        {"name": "write_step", "op": "write", "format": "int8", "layers": 1, "lanes": 128, "chunks": 0, "new": 0, "context": 8000, "kvh": 4, "dim": 64, "mix": 1},
        # Four long prompts of several layers, wide heads: bound by HBM.
        {"name": "write_prompts", "op": "write", "format": "e4m3", "layers": 6, "lanes": 0, "chunks": 4, "new": 4096, "context": 30000, "kvh": 8, "dim": 128, "mix": 2},
        # Two extents filled in a step: the smallest copy.
        {"name": "promote_few", "op": "promote", "format": "int8", "layers": 22, "jobs": 2, "kvh": 4, "dim": 64, "mix": 3},
        # A long prompt's pages promoted at once.
        {"name": "promote_many", "op": "promote", "format": "e4m3", "layers": 22, "jobs": 512, "kvh": 4, "dim": 64, "mix": 4},
        # One layer of a prompt's first part, read back for its next chunk's prefill.
        {"name": "read_layer", "op": "read", "format": "e4m3", "layers": 1, "tokens": 1943, "lead": 3, "kvh": 8, "dim": 128, "mix": 5},
        # A long request read back whole.
        {"name": "read_long", "op": "read", "format": "int8", "layers": 22, "tokens": 16384, "lead": 0, "kvh": 4, "dim": 64, "mix": 6},
        # A few chats: where latency is all there is.
        {"name": "decode_few", "op": "decode", "format": "int8", "lanes": 4, "least": 700, "most": 1300, "kvh": 4, "group": 8, "dim": 64, "mix": 7},
        # Ragged chats, wide heads, small pages in front of some.
        {"name": "decode_ragged", "op": "decode", "format": "e4m3", "lanes": 64, "least": 1, "most": 6000, "kvh": 8, "group": 4, "dim": 128, "mix": 8},
        # Long contexts under a large batch: bound by HBM.
        {"name": "decode_long", "op": "decode", "format": "int8", "lanes": 128, "least": 32768, "most": 32768, "kvh": 4, "group": 8, "dim": 64, "mix": 9},
        # A few chats' next tokens.
        {"name": "sample_few", "op": "sample", "rows": 4, "vocab": 32000, "top_k": 50, "top_p": 0.95, "min_p": 0.0, "spread": False, "mix": 10},
        # A serving batch of many settings, rows off the vectors' alignment.
        {"name": "sample_mixed", "op": "sample", "rows": 72, "vocab": 50255, "top_k": 400, "top_p": 0.8, "min_p": 0.05, "spread": True, "mix": 11},
        # A large vocabulary under a large batch of many settings.
        {"name": "sample_wide", "op": "sample", "rows": 256, "vocab": 128000, "top_k": 1000, "top_p": 0.9, "min_p": 0.02, "spread": True, "mix": 12},
    ]


def _log_uniform(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["write", "promote", "read", "decode", "decode", "sample", "sample"])
    mix = rng.randrange(1 << 20)
    form = rng.choice(["int8", "e4m3"])
    kvh, group, dim = rng.choice([(4, 8, 64), (4, 8, 64), (8, 4, 64), (2, 16, 64), (8, 4, 128), (4, 4, 128), (3, 5, 64), (1, 8, 128), (2, 3, 96)])
    head = {"op": op, "format": form, "kvh": kvh, "dim": dim, "mix": mix}
    width = kvh * dim
    if op == "write":
        layers = rng.choice([1, 1, 2, 6])
        return {**head, "layers": layers, "lanes": _log_uniform(rng, 1, 256), "chunks": rng.randint(0, 4), "new": _log_uniform(rng, 3, 4000), "context": _log_uniform(rng, 100, 30000)}
    if op == "promote":
        layers = rng.choice([1, 4, 22])
        return {**head, "layers": layers, "jobs": _log_uniform(rng, 1, min(512, 512 * 22 * 256 // (layers * width)))}
    if op == "read":
        layers = rng.choice([1, 1, 4, 22])
        return {**head, "layers": layers, "tokens": _log_uniform(rng, 1, min(32768, 16384 * 22 * 256 // (layers * width))), "lead": rng.randint(0, 7)}
    if op == "decode":
        lanes = _log_uniform(rng, 1, 128)
        most = _log_uniform(rng, 60, min(65536, 128 * 32768 * 256 // (lanes * width)))
        return {**head, "group": group, "lanes": lanes, "least": max(1, most // rng.choice([1, 4, 100])), "most": most}
    vocab = _log_uniform(rng, 1000, 128000)
    return {"op": op, "rows": _log_uniform(rng, 1, min(256, 32_000_000 // vocab)), "vocab": vocab, "top_k": rng.choice([0, 1, 40, 400, 3000]),
            "top_p": rng.choice([1.0, 0.95, 0.8, 0.3]), "min_p": rng.choice([0.0, 0.02, 0.2]), "spread": rng.random() < 0.5, "mix": mix}


# ---- shared pieces -----------------------------------------------------------


def _package():
    from _loader import load_package

    return load_package().device


def _normal(seed, tag, *shape):
    g = torch.Generator(device="cuda")
    g.manual_seed((int(seed) * 1_000_003 + tag * 7919 + 17) & 0x7FFFFFFFFFFFFFFF)
    return torch.randn(shape, generator=g, device="cuda", dtype=torch.float16)


def _on_gpu(array):
    """A numpy (structured) array as bytes on the GPU."""
    return torch.from_numpy(np.ascontiguousarray(array).view(np.uint8).reshape(-1).copy()).cuda()


def _ints(values):
    return torch.from_numpy(np.asarray(values, dtype=np.int64)).cuda()


def _quantised(rows, form):
    """(codes, scales) of rows of fp16, [..., D]: the scale is the least number of 8 significant bits that keeps the row's
    largest value within the codes."""
    x = rows.float()
    # A tensor's division: a number's is a product with its reciprocal, which is off where the quotient is exact.
    largest = x.abs().amax(-1)
    mantissa, exponent = torch.frexp(largest / torch.full_like(largest, LARGEST[form]))
    scale = torch.ldexp(torch.ceil(mantissa * 256), exponent - 8)
    x = x / torch.where(scale == 0, 1.0, scale)[..., None]
    return (x.round().to(torch.int8) if form == "int8" else x.to(torch.float8_e4m3fn).view(torch.uint8)), scale


def _values(codes, scale, form):
    """What codes and scales stand for, in 32 bits."""
    return (codes if form == "int8" else codes.view(torch.float8_e4m3fn)).float() * scale[..., None]


def _as_halves(values):
    return values.clamp(-65504, 65504).half()


def _exactly(rows, form):
    """The 64-bit values that a cache of 8 bits holds for rows of fp16."""
    x = rows.double()
    largest = x.abs().amax(-1, keepdim=True)
    least = largest / torch.full_like(largest, LARGEST[form])
    unit = torch.exp2(torch.floor(torch.log2(least)) - 7)
    scale = torch.where(largest == 0, 1.0, torch.ceil(least / unit) * unit)
    x /= scale
    if form == "int8":
        return torch.round(x) * scale
    step = torch.exp2(torch.floor(torch.log2(x.abs().clamp_min(2.0 ** -6))) - 3)
    return torch.round(x / step) * step * scale


def _write_rows(device, storage, rows, pages):
    """Puts rows ([layers][2][tokens][heads][dim]) into pages given as (kind, slot, tokens), one after the other."""
    layers, _, total, kvh, dim = rows.shape
    width = kvh * dim
    jobs = np.zeros(len(pages), dtype=device.APPEND_JOB)
    kind, slot, n = (np.array(v, dtype=np.int64) for v in zip(*pages))
    first = np.concatenate([[0], np.cumsum(n)[:-1]])
    jobs["src_key"], jobs["src_value"] = rows.data_ptr() + 2 * first * width, rows.data_ptr() + 2 * (total + first) * width
    jobs["src_layer_stride"], jobs["src_token_stride"] = 2 * total * width, width
    jobs["layer_count"], jobs["token_count"], jobs["dst_slot"], jobs["dst_kind"] = layers, n, slot, kind
    held = _on_gpu(jobs)
    storage.append_launch(held.data_ptr(), len(jobs), layers)
    torch.cuda.synchronize()


def _storage(device, case, micro, extent):
    return device.QuantStorage(case.get("layers", 1), case["kvh"], case["dim"], micro, extent, {"int8": device.QUANT_INT8, "e4m3": device.QUANT_E4M3}[case["format"]])


def _table(device, pages):
    """A block table of pages (kind, slot, tokens), one after the other."""
    flat = np.zeros(len(pages), dtype=device.BLOCK_DESC)
    kind, slot, n = (np.array(v, dtype=np.int64) for v in zip(*pages))
    flat["slot"], flat["generation"], flat["valid_tokens"], flat["kind"] = slot, 1, n, kind
    flat["logical_token_begin"] = np.concatenate([[0], np.cumsum(n)[:-1]])
    flat["page_token_capacity"] = np.where(kind == 1, EXTENT, MICRO)
    return flat


def _scattered(case, counts):
    """Pages in a scattered order, as a server's free lists hand them out."""
    return [np.random.RandomState(case["mix"] % (1 << 31)).permutation(max(1, n)) for n in counts]


def _rows_of(pages, micro):
    """Each page token's place among the rows of all pages, every micro page's first."""
    return np.concatenate([np.arange(n) + (micro * MICRO + slot * EXTENT if kind else slot * MICRO) for kind, slot, n in pages])


def _elements(case, tokens):
    return tokens * case.get("layers", 1) * 2 * case["kvh"] * case["dim"]


def _code_bytes(case, tokens):
    return _elements(case, tokens) * (1 + 2 / case["dim"])


# ---- write -------------------------------------------------------------------


def _write_plan(case):
    """(jobs, rows, micro pages, extent pages): a job is (first row, tokens, kind, slot, token in the page, slot copied from, tokens
    copied)."""
    rng = random.Random(case["mix"] * 1031)
    free, jobs, rows = [0, 0], [], 0

    def take(kind):
        free[kind] += 1
        return free[kind] - 1

    for _ in range(case["lanes"]):
        at = rng.randint(0, case["context"])
        copied = at % MICRO if rng.random() < 0.25 else 0
        source = take(0) if copied else 0
        jobs.append((rows, 1, 0, take(0), at % MICRO, source, copied))
        rows += 1
    for _ in range(case["chunks"]):
        at, new = rng.randint(0, case["context"]), rng.randint(max(1, case["new"] * 3 // 4), case["new"])
        end = at + new
        while at < end:
            kind = 1 if at // EXTENT * EXTENT + EXTENT <= end else 0
            cap = (MICRO, EXTENT)[kind]
            n = min(end, at // cap * cap + cap) - at
            jobs.append((rows, n, kind, take(kind), at % cap, 0, 0))
            at, rows = at + n, rows + n
    order = _scattered(case, free)
    jobs = [j[:3] + (int(order[j[2]][j[3]]), j[4], int(order[0][j[5]]) if j[6] else 0, j[6]) for j in jobs]
    return jobs, rows, max(1, free[0]), max(1, free[1])


def _all_pages(micro, extent):
    return [(0, s, MICRO) for s in range(micro)] + [(1, s, EXTENT) for s in range(extent)]


def _prepare_write(case, seed):
    jobs, rows, micro, extent = _write_plan(case)
    layers, kvh, dim = case["layers"], case["kvh"], case["dim"]
    new = _normal(seed, 1, layers, 2, rows, kvh, dim)
    before = _normal(seed, 2, layers, 2, micro * MICRO + extent * EXTENT, kvh, dim)
    pages = [(j[2], j[3], j[4] + j[1]) for j in jobs]
    if own:
        device = _package()
        storage = _storage(device, case, micro, extent)
        _write_rows(device, storage, before, _all_pages(micro, extent))
        table = np.zeros(len(jobs), dtype=device.APPEND_JOB)
        first, n, kind, slot, token, source, copied = (np.array(v, dtype=np.int64) for v in zip(*jobs))
        width = kvh * dim
        table["src_key"], table["src_value"] = new.data_ptr() + 2 * first * width, new.data_ptr() + 2 * (rows + first) * width
        table["src_layer_stride"], table["src_token_stride"], table["layer_count"], table["token_count"] = 2 * rows * width, width, layers, n
        table["dst_kind"], table["dst_slot"], table["dst_token"], table["cow_slot"], table["cow_tokens"] = kind, slot, token, source, copied
        tokens = sum(p[2] for p in pages)
        out = torch.empty(layers, 2, tokens, kvh, dim, dtype=torch.float16, device="cuda")
        return {"storage": storage, "jobs": _on_gpu(table), "count": (len(jobs), layers), "table": _on_gpu(_table(device, pages)), "pages": len(pages), "tokens": tokens,
                "layers": layers, "out": out, "new": new}
    codes, scale = _quantised(before, case["format"])
    copies = np.concatenate([np.zeros((0, 2), np.int64)] + [np.stack((j[3] * MICRO + np.arange(j[6]), j[5] * MICRO + np.arange(j[6])), 1) for j in jobs])
    written = [(j[2], j[3], j[4], j[1]) for j in jobs]
    at = np.concatenate([np.arange(t, t + n) + (micro * MICRO + slot * EXTENT if kind else slot * MICRO) for kind, slot, t, n in written])
    return {"case": case, "new": new, "codes": codes, "scale": scale, "copies": _ints(copies), "at": _ints(at), "read": _ints(_rows_of(pages, micro))}


def _run_write(s):
    if own:
        s["storage"].append_launch(s["jobs"].data_ptr(), *s["count"])
        s["storage"].gather_launch(s["table"].data_ptr(), s["pages"], 0, s["tokens"], 0, s["layers"], s["out"].data_ptr())
        return s["out"]
    form, codes, scale = s["case"]["format"], s["codes"], s["scale"]
    to, source = s["copies"].unbind(1)
    codes[:, :, to], scale[:, :, to] = codes[:, :, source], scale[:, :, source]
    codes[:, :, s["at"]], scale[:, :, s["at"]] = _quantised(s["new"], form)
    return _as_halves(_values(codes[:, :, s["read"]], scale[:, :, s["read"]], form))


def _exact_write(case, seed):
    jobs, rows, micro, extent = _write_plan(case)
    layers, kvh, dim = case["layers"], case["kvh"], case["dim"]
    new = _exactly(_normal(seed, 1, layers, 2, rows, kvh, dim), case["format"])
    before = _exactly(_normal(seed, 2, layers, 2, micro * MICRO + extent * EXTENT, kvh, dim), case["format"])
    parts = []
    for first, n, kind, slot, token, source, copied in jobs:
        base = micro * MICRO + slot * EXTENT if kind else slot * MICRO
        held = before[:, :, base:base + token]
        if copied:
            held = torch.cat((before[:, :, source * MICRO:source * MICRO + copied], held[:, :, copied:]), 2)
        parts += [held, new[:, :, first:first + n]]
    return torch.cat(parts, 2)


def _work_write(case):
    jobs, rows, _, _ = _write_plan(case)
    read, copied = sum(j[4] + j[1] for j in jobs), sum(j[6] for j in jobs)
    return {"bytes": 2 * _elements(case, rows) + _code_bytes(case, rows + 2 * copied + read) + 2 * _elements(case, read), "flops": 4 * _elements(case, rows) + _elements(case, read)}


# ---- promote -----------------------------------------------------------------


def _promote_plan(case):
    """Each extent's micro pages, and the extents."""
    order = _scattered(case, (8 * case["jobs"], case["jobs"]))
    return order[0].reshape(-1, 8), order[1]


def _prepare_promote(case, seed):
    micro, extent = _promote_plan(case)
    jobs = len(extent)
    layers, kvh, dim = case["layers"], case["kvh"], case["dim"]
    rows = _normal(seed, 1, layers, 2, jobs * EXTENT, kvh, dim)
    if own:
        device = _package()
        storage = _storage(device, case, 8 * jobs, jobs)
        _write_rows(device, storage, rows, [(0, s, MICRO) for s in range(8 * jobs)])
        table = np.zeros(jobs, dtype=device.PROMOTION_JOB)
        table["micro_slots"], table["extent_slot"] = micro, extent
        return {"storage": storage, "jobs": _on_gpu(table), "count": jobs, "table": _on_gpu(_table(device, [(1, int(s), EXTENT) for s in extent])), "layers": layers,
                "out": torch.empty_like(rows)}
    codes, scale = _quantised(rows, case["format"])
    large = torch.zeros_like(codes), torch.zeros_like(scale)
    token = np.arange(EXTENT)
    return {"case": case, "codes": codes, "scale": scale, "large": large, "source": _ints((micro[:, token // MICRO] * MICRO + token % MICRO).reshape(-1)),
            "at": _ints((extent[:, None] * EXTENT + token).reshape(-1))}


def _run_promote(s):
    if own:
        s["storage"].promote_launch(s["jobs"].data_ptr(), s["count"])
        s["storage"].gather_launch(s["table"].data_ptr(), s["count"], 0, s["count"] * EXTENT, 0, s["layers"], s["out"].data_ptr())
        return s["out"]
    codes, scale = s["large"]
    codes[:, :, s["at"]], scale[:, :, s["at"]] = s["codes"][:, :, s["source"]], s["scale"][:, :, s["source"]]
    return _as_halves(_values(codes[:, :, s["at"]], scale[:, :, s["at"]], s["case"]["format"]))


def _exact_promote(case, seed):
    micro, extent = _promote_plan(case)
    rows = _exactly(_normal(seed, 1, case["layers"], 2, len(extent) * EXTENT, case["kvh"], case["dim"]), case["format"])
    pages = rows.view(case["layers"], 2, -1, MICRO, case["kvh"], case["dim"])
    return pages[:, :, _ints(micro.reshape(-1))].reshape(rows.shape)


def _work_promote(case):
    tokens = case["jobs"] * EXTENT
    return {"bytes": 3 * _code_bytes(case, tokens) + 2 * _elements(case, tokens), "flops": _elements(case, tokens)}


# ---- read --------------------------------------------------------------------


def _pages_of(rng, tokens, lead):
    """A request's pages as (kind, tokens): some small ones in front, large ones while they are full, small ones."""
    pages, at = [], 0
    while at < tokens:
        kind = 1 if at >= lead * MICRO and at + EXTENT <= tokens else 0
        pages.append((kind, min((MICRO, EXTENT)[kind], tokens - at)))
        at += pages[-1][1]
    return pages


def _read_pages(case):
    pages, free = [], [0, 0]
    for kind, n in _pages_of(None, case["tokens"], case["lead"]):
        pages.append((kind, free[kind], n))
        free[kind] += 1
    order = _scattered(case, free)
    return [(kind, int(order[kind][slot]), n) for kind, slot, n in pages], max(1, free[0]), max(1, free[1])


def _prepare_read(case, seed):
    layers, kvh, dim, tokens = case["layers"], case["kvh"], case["dim"], case["tokens"]
    pages, micro, extent = _read_pages(case)
    rows = _normal(seed, 1, layers, 2, tokens, kvh, dim)
    if own:
        device = _package()
        storage = _storage(device, case, micro, extent)
        _write_rows(device, storage, rows, pages)
        return {"storage": storage, "table": _on_gpu(_table(device, pages)), "pages": len(pages), "tokens": tokens, "layers": layers, "out": torch.empty_like(rows)}
    # The pages' rows in the order of the pages.
    at = _ints(_rows_of(pages, micro))
    codes, scale = _quantised(rows, case["format"])
    held = (torch.zeros(layers, 2, micro * MICRO + extent * EXTENT, kvh, dim, dtype=codes.dtype, device="cuda"),
            torch.zeros(layers, 2, micro * MICRO + extent * EXTENT, kvh, device="cuda"))
    held[0][:, :, at], held[1][:, :, at] = codes, scale
    return {"case": case, "held": held, "at": at}


def _run_read(s):
    if own:
        s["storage"].gather_launch(s["table"].data_ptr(), s["pages"], 0, s["tokens"], 0, s["layers"], s["out"].data_ptr())
        return s["out"]
    codes, scale = s["held"]
    return _as_halves(_values(codes[:, :, s["at"]], scale[:, :, s["at"]], s["case"]["format"]))


def _exact_read(case, seed):
    return _exactly(_normal(seed, 1, case["layers"], 2, case["tokens"], case["kvh"], case["dim"]), case["format"])


def _work_read(case):
    return {"bytes": _code_bytes(case, case["tokens"]) + 2 * _elements(case, case["tokens"]), "flops": _elements(case, case["tokens"])}


# ---- decode ------------------------------------------------------------------


def _decode_plan(case):
    """(each lane's tokens, each lane's pages as (kind, slot, tokens), micro pages, extent pages)."""
    rng = random.Random(case["mix"] * 1033)
    counts = [_log_uniform(rng, case["least"], case["most"]) for _ in range(case["lanes"])]
    free, lanes = [0, 0], []
    for n in counts:
        pages = []
        # Three requests in ten have small pages in front.
        for kind, m in _pages_of(rng, n, rng.randint(1, 7) if rng.random() < 0.3 else 0):
            pages.append((kind, free[kind], m))
            free[kind] += 1
        lanes.append(pages)
    order = _scattered(case, free)
    return counts, [[(kind, int(order[kind][slot]), m) for kind, slot, m in pages] for pages in lanes], max(1, free[0]), max(1, free[1])


def _decode_inputs(case, seed, total):
    """Keys and values of all lanes' tokens, lane after lane; queries of twice unit variance, so that some keys weigh far more."""
    kvh, dim = case["kvh"], case["dim"]
    return _normal(seed, 1, 1, 2, total, kvh, dim), 2 * _normal(seed, 3, case["lanes"], kvh * case["group"], dim)


def _prepare_decode(case, seed):
    counts, lanes, micro, extent = _decode_plan(case)
    rows, query = _decode_inputs(case, seed, sum(counts))
    dim, qh = case["dim"], case["kvh"] * case["group"]
    if own:
        device = _package()
        storage = _storage(device, case, micro, extent)
        _write_rows(device, storage, rows, [p for pages in lanes for p in pages])
        tables = [_table(device, pages) for pages in lanes]
        # Entries are of 20 bytes; numpy's concatenation would pack them.
        flat = np.zeros(sum(len(t) for t in tables), dtype=device.BLOCK_DESC)
        for t, end in zip(tables, np.cumsum([len(t) for t in tables])):
            flat[end - len(t):end] = t
        flat = _on_gpu(flat)
        out = torch.zeros_like(query)
        items = np.zeros(len(counts), dtype=device.DECODE_ITEM)
        lengths = np.array([len(t) for t in tables], dtype=np.int64)
        items["descriptors"], items["descriptor_count"] = flat.data_ptr() + 20 * (np.cumsum(lengths) - lengths), lengths
        items["token_count"], items["attention_scale"] = counts, 1.0 / math.sqrt(dim)
        lane = np.arange(len(counts)) * 2 * qh * dim
        items["query"], items["output"] = query.data_ptr() + lane, out.data_ptr() + lane
        entries, plan = storage.decode_plan(counts, qh)
        work = torch.zeros(max(1, plan.workspace_bytes // 4), dtype=torch.float32, device="cuda")
        return {"storage": storage, "items": _on_gpu(items), "entries": _on_gpu(entries), "plan": plan, "work": work, "out": out, "held": (flat, query)}
    codes, scale = _quantised(rows[0], case["format"])
    most = max(counts)
    first = np.cumsum(counts) - counts
    index = np.minimum(first[:, None] + np.arange(most)[None], sum(counts) - 1)
    return {"case": case, "codes": codes, "scale": scale, "query": query, "index": _ints(index), "counts": _ints(counts)}


def _run_decode(s):
    if own:
        s["storage"].decode_launch(s["items"].data_ptr(), s["entries"].data_ptr(), s["plan"], s["work"].data_ptr())
        return s["out"]
    case, index = s["case"], s["index"]
    lanes, most = index.shape
    kvh, dim = case["kvh"], case["dim"]
    keys, values = (_values(s["codes"][i], s["scale"][i], case["format"])[index] for i in (0, 1))
    q = s["query"].float().view(lanes, kvh, case["group"], dim)
    scores = q @ keys.permute(0, 2, 3, 1) / math.sqrt(dim)
    scores.masked_fill_((torch.arange(most, device="cuda") >= s["counts"][:, None])[:, None, None, :], -math.inf)
    weights = (scores - scores.amax(-1, keepdim=True)).exp()
    out = weights @ values.transpose(1, 2) / weights.sum(-1, keepdim=True)
    return out.half().view(lanes, -1, dim)


def _exact_decode(case, seed):
    counts, _, _, _ = _decode_plan(case)
    rows, query = _decode_inputs(case, seed, sum(counts))
    kvh, group, dim = case["kvh"], case["group"], case["dim"]
    out = torch.empty(query.shape, dtype=torch.float64, device="cuda")
    at = 0
    for i, n in enumerate(counts):
        k, v = _exactly(rows[0, :, at:at + n], case["format"])
        at += n
        for h in range(kvh):
            p = torch.softmax(query[i, h * group:(h + 1) * group].double() @ k[:, h].t().contiguous() * dim ** -0.5, 1)
            out[i, h * group:(h + 1) * group] = p @ v[:, h].contiguous()
    return out


def _work_decode(case):
    counts = _decode_plan(case)[0]
    qh = case["kvh"] * case["group"]
    return {"bytes": _code_bytes(case, sum(counts)) + 4 * len(counts) * qh * case["dim"], "flops": 4 * qh * case["dim"] * sum(counts)}


# ---- sample ------------------------------------------------------------------


def _sample_plan(case):
    """Each row's (temperature, top-k, top-p, min-p, peaks, part of the tokens that are masked): the case's, or where the settings
    are spread each of them or none."""
    rng = random.Random(case["mix"] * 1039)
    rows = []
    for _ in range(case["rows"]):
        some = lambda v, off: v if not case["spread"] or rng.random() < 0.5 else off  # noqa: E731
        rows.append((rng.choice([0.0, 0.7, 1.0, 1.0, 1.3]) if case["spread"] else 0.8, some(case["top_k"], 0), some(case["top_p"], 1.0), some(case["min_p"], 0.0),
                     rng.choice([0, 5, 60]) if case["spread"] else 30, rng.choice([0.0, 0.0, 0.6]) if case["spread"] else 0.0))
    return rows


def _sample_inputs(case, seed):
    """Logits and random numbers: most tokens as noise, a few stand out; some rows masked as a grammar leaves them."""
    rows, vocab, plan = case["rows"], case["vocab"], _sample_plan(case)
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed) * 65537 + 11)
    logits = 2 * torch.randn(rows, vocab, generator=g, device="cuda")
    peaks = torch.randint(0, vocab, (rows, 60), generator=g, device="cuda")
    high = 14 * torch.rand(rows, 60, generator=g, device="cuda") * (torch.arange(60, device="cuda") < _ints([p[4] for p in plan])[:, None])
    logits.scatter_add_(1, peaks, high)
    masked = torch.tensor([p[5] for p in plan], device="cuda")[:, None]
    logits.masked_fill_(torch.rand(rows, vocab, generator=g, device="cuda") < masked, -math.inf)
    return logits, torch.rand(rows, generator=g, device="cuda"), plan


def _prepare_sample(case, seed):
    logits, uniform, plan = _sample_inputs(case, seed)
    rows, vocab = logits.shape
    tokens, chance = torch.zeros(rows, dtype=torch.int32, device="cuda"), torch.zeros(rows, device="cuda")
    if own:
        device = _package()
        rules = np.zeros(rows, dtype=device.SAMPLE_RULE)
        for name, k in (("temperature", 0), ("top_k", 1), ("top_p", 2), ("min_p", 3)):
            rules[name] = [p[k] for p in plan]
        work = torch.zeros(device.sample_workspace_bytes(rows, vocab) // 4 + 1, dtype=torch.int32, device="cuda")
        return {"device": device, "logits": logits, "rules": _on_gpu(rules), "uniform": uniform, "tokens": tokens, "chance": chance, "work": work}
    settings = [torch.tensor([p[k] for p in plan], dtype=torch.float32, device="cuda").double()[:, None] for k in range(4)]
    return {"logits": logits, "uniform": uniform, "settings": settings, "tokens": tokens, "chance": chance}


def _run_sample(s):
    logits = s["logits"]
    rows, vocab = logits.shape
    if own:
        s["device"].sample(logits.data_ptr(), rows, vocab, s["rules"].data_ptr(), s["uniform"].data_ptr(), s["tokens"].data_ptr(), s["chance"].data_ptr(), s["work"].data_ptr())
        return s["tokens"], s["chance"]
    temperature, top_k, top_p, min_p = s["settings"]
    # In 64 bits: sums of a vocabulary's weights, next to the border that a random number is.
    x, order = logits.double().sort(dim=1, descending=True, stable=True)
    weight = ((x - x[:, :1]) / torch.where(temperature == 0, 1.0, temperature)).exp()
    rank = torch.arange(vocab, device="cuda")
    weight = torch.where(rank < torch.where(temperature == 0, 1, torch.where(top_k == 0, vocab, top_k)), weight, 0.0)
    sums = weight.cumsum(1)
    keep = ((sums - weight < top_p * sums[:, -1:]) | (top_p >= 1)) & (weight >= min_p)
    weight = torch.zeros_like(weight).scatter_(1, order, torch.where(keep, weight, 0.0))
    sums = weight.cumsum(1)
    total = sums[:, -1:]
    last = torch.where(weight > 0, rank, -1).amax(1)
    token = torch.minimum((sums <= s["uniform"].double()[:, None] * total).sum(1), last)
    s["tokens"].copy_(token)
    s["chance"].copy_((weight.gather(1, token[:, None]) / total)[:, 0])
    return s["tokens"], s["chance"]


def _exact_sample(case, seed):
    logits, uniform, plan = _sample_inputs(case, seed)
    chances = []
    for row, u, (temperature, top_k, top_p, min_p, _, _) in zip(logits, uniform.tolist(), plan):
        if temperature == 0:
            chances.append(1.0)
            continue
        temperature, top_p, min_p = (float(np.float32(v)) for v in (temperature, top_p, min_p))
        x = row.double().cpu().numpy()
        kept = np.argsort(-x, kind="stable")[:top_k or None]
        p = np.exp((x[kept] - x[kept[0]]) / temperature)
        if top_p < 1:
            m = int(np.searchsorted(np.cumsum(p), top_p * np.cumsum(p)[-1])) + 1
            kept, p = kept[:m], p[:m]
        kept, p = kept[p >= min_p], p[p >= min_p]
        by_index = np.argsort(kept)
        p = p[by_index] / p.sum()
        chances.append(float(p[min(int(np.searchsorted(np.cumsum(p), u, side="right")), len(p) - 1)]))
    return None, torch.tensor(chances, dtype=torch.float64)


def _work_sample(case):
    return {"bytes": case["rows"] * (4 * case["vocab"] + 28), "flops": case["rows"] * case["vocab"]}


# ---- what is called ----------------------------------------------------------


def prepare(case, seed):
    return {"op": case["op"], **{"write": _prepare_write, "promote": _prepare_promote, "read": _prepare_read, "decode": _prepare_decode, "sample": _prepare_sample}[case["op"]](case, seed)}


def run(state):
    return {"write": _run_write, "promote": _run_promote, "read": _run_read, "decode": _run_decode, "sample": _run_sample}[state["op"]](state)


def exact(case, seed):
    return {"write": _exact_write, "promote": _exact_promote, "read": _exact_read, "decode": _exact_decode, "sample": _exact_sample}[case["op"]](case, seed)


def work(case):
    return {"write": _work_write, "promote": _work_promote, "read": _work_read, "decode": _work_decode, "sample": _work_sample}[case["op"]](case)
