"""Three operators of a token step of requests that share a prompt, as cases that can be timed and checked.

  append    rows of a fused q | k | v projection: q and k rotated by their positions, q stored as rows, k and v
            written into the pages of the cache, partial tails copied first where a request leaves a shared page
  shared    one layer's decode attention of lanes in groups that share their first tokens' pages
  logits    repetition, presence and frequency penalties, biases and an allowed-token mask on rows of logits,
            and the greedy token of each row

`own` chooses who computes: False, elementary torch operations on tensors; True, the library's entry points on
its page storage.  Lengths and page tables follow from the case alone (`mix`), contents from the seed.
"""
import math
import random

import numpy as np
import torch

own = False

MICRO, EXTENT = 8, 64


def listed():
    return [
        # A few chats' token step: the smallest append, where latency is all there is.
        {"name": "append_few", "op": "append", "lanes": 4, "chunks": 0, "new": 0, "context": 1000, "kvh": 4, "group": 8, "dim": 64,
         "rotary": 64, "adjacent": False, "theta": 10000.0, "mix": 1},
        # A serving batch's token step; one lane in four leaves a page it shares.
        {"name": "append_batch", "op": "append", "lanes": 128, "chunks": 0, "new": 0, "context": 8000, "kvh": 4, "group": 8, "dim": 64,
         "rotary": 64, "adjacent": False, "theta": 10000.0, "mix": 2},
        # One scheduler iteration: prompt chunks of up to 512 tokens beside decode lanes.
        {"name": "append_mixed", "op": "append", "lanes": 28, "chunks": 4, "new": 512, "context": 2000, "kvh": 4, "group": 8, "dim": 64,
         "rotary": 64, "adjacent": False, "theta": 10000.0, "mix": 3},
        # Long prompts at far positions, wide heads of which half the dims rotate, in adjacent pairs: bound by HBM.
        {"name": "append_prompts", "op": "append", "lanes": 0, "chunks": 4, "new": 4096, "context": 100000, "kvh": 8, "group": 4, "dim": 128,
         "rotary": 64, "adjacent": True, "theta": 500000.0, "mix": 4},
        # Four continuations of one short prompt: the smallest launch.
        {"name": "shared_few", "op": "shared", "groups": 1, "lanes": 4, "alone": 0, "prefix": 500, "least": 1, "most": 60, "kvh": 4, "group": 8,
         "dim": 64, "mix": 5},
        # Eight prompts of 2048 tokens with four requests each, ragged continuations, some requests on their own.
        {"name": "shared_groups", "op": "shared", "groups": 8, "lanes": 4, "alone": 4, "prefix": 2048, "least": 100, "most": 6000, "kvh": 4, "group": 8,
         "dim": 64, "mix": 6},
        # One system prompt under a batch of chats, wide heads.
        {"name": "shared_wide", "op": "shared", "groups": 1, "lanes": 64, "alone": 0, "prefix": 4100, "least": 20, "most": 1500, "kvh": 8, "group": 4,
         "dim": 128, "mix": 7},
        # Many answers on one long document: the largest.
        {"name": "shared_long", "op": "shared", "groups": 1, "lanes": 128, "alone": 0, "prefix": 32768, "least": 1, "most": 800, "kvh": 4, "group": 8,
         "dim": 64, "mix": 8},
        # A few chats' next tokens: penalties only, only the token asked for.
        {"name": "logits_few", "op": "logits", "rows": 4, "vocab": 32000, "history": 300, "biases": 0, "masked": 0.0, "store": False, "mix": 9},
        # A serving batch: penalties, biases, and grammars on half the rows.
        {"name": "logits_batch", "op": "logits", "rows": 72, "vocab": 32000, "history": 2000, "biases": 64, "masked": 0.5, "store": False, "mix": 10},
        # The adjusted logits as well (a sampler's input), rows off the vectors' alignment.
        {"name": "logits_odd", "op": "logits", "rows": 17, "vocab": 50255, "history": 1000, "biases": 300, "masked": 0.3, "store": True, "mix": 11},
        # A large vocabulary under a large batch: bound by HBM.
        {"name": "logits_wide", "op": "logits", "rows": 256, "vocab": 128000, "history": 4000, "biases": 100, "masked": 0.25, "store": True, "mix": 12},
    ]


def _log_uniform(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["append", "shared", "shared", "logits"])
    mix = rng.randrange(1 << 20)
    kvh, group, dim = rng.choice([(4, 8, 64), (4, 8, 64), (8, 4, 64), (2, 16, 64), (8, 4, 128), (4, 4, 128), (3, 5, 64), (2, 3, 96)])
    if op == "append":
        chunks = rng.randint(0, 4)
        return {"op": op, "lanes": _log_uniform(rng, 1, 256), "chunks": chunks, "new": _log_uniform(rng, 3, 4000), "context": _log_uniform(rng, 100, 100000),
                "kvh": kvh, "group": group, "dim": dim, "rotary": rng.choice([dim, dim, dim // 2]), "adjacent": rng.random() < 0.3,
                "theta": rng.choice([10000.0, 500000.0]), "mix": mix}
    if op == "shared":
        groups, prefix = _log_uniform(rng, 1, 16), _log_uniform(rng, 30, 32768)
        # Of bytes and of arithmetic no more than the largest listed case takes time for.
        prefix = min(prefix, 64_000_000 // (groups * kvh * dim))
        lanes = _log_uniform(rng, 1, max(1, min(128 // groups, 4_200_000 * 2048 // (prefix * groups * kvh * group * dim))))
        return {"op": op, "groups": groups, "lanes": lanes, "alone": rng.randint(0, 6), "prefix": prefix, "least": rng.choice([1, 1, 50]),
                "most": _log_uniform(rng, 60, max(61, min(6000, 100_000 // (groups * lanes)))), "kvh": kvh, "group": group, "dim": dim, "mix": mix}
    vocab = _log_uniform(rng, 1000, 128000)
    return {"op": op, "rows": _log_uniform(rng, 1, min(256, 32_000_000 // vocab)), "vocab": vocab, "history": _log_uniform(rng, 1, 8000),
            "biases": rng.choice([0, 1, 40, 300]), "masked": rng.choice([0.0, 0.3, 1.0]), "store": rng.random() < 0.5, "mix": mix}


# ---- shared pieces -----------------------------------------------------------


def _package():
    from _loader import load_package

    return load_package().device


def _normal(seed, tag, *shape, dtype=torch.float16):
    g = torch.Generator(device="cuda")
    g.manual_seed((int(seed) * 1_000_003 + tag * 7919 + 17) & 0x7FFFFFFFFFFFFFFF)
    return torch.randn(shape, generator=g, device="cuda", dtype=dtype)


def _on_gpu(array):
    """A numpy (structured) array as bytes on the GPU."""
    return torch.from_numpy(np.ascontiguousarray(array).view(np.uint8).reshape(-1).copy()).cuda()


def _ints(values):
    return torch.tensor(values, dtype=torch.int64, device="cuda")


class _Memory:
    """A storage's pool as a torch tensor sees it, which keeps the storage."""

    def __init__(self, storage, elements):
        self.storage, address = storage, storage.page(0, 0)
        self.__cuda_array_interface__ = {"shape": (elements,), "typestr": "<f2", "data": (address, False), "version": 3}


# ---- append ------------------------------------------------------------------
# A page's block of one layer holds, for each head, K of its `cap` tokens in blocks of 32 dims, then V transposed in
# blocks of 32 tokens (of cap tokens in a smaller page); a pool is every micro page's block, then every extent page's.


def _append_plan(case):
    """(jobs, tokens copied, micro pages, extent pages): a job is (first row, tokens, position, kind, slot, token in the page, slot
    copied from, tokens copied)."""
    rng = random.Random(case["mix"] * 1031)
    free = [0, 0]
    jobs, rows = [], 0

    def take(kind):
        free[kind] += 1
        return free[kind] - 1

    for _ in range(case["lanes"]):
        at = rng.randint(0, case["context"])
        copied = at % MICRO if rng.random() < 0.25 else 0
        source = take(0) if copied else 0
        jobs.append((rows, 1, at, 0, take(0), at % MICRO, source, copied))
        rows += 1
    for _ in range(case["chunks"]):
        at, new = rng.randint(0, case["context"]), rng.randint(max(1, case["new"] * 3 // 4), case["new"])
        end = at + new
        while at < end:
            kind = 1 if at // EXTENT * EXTENT + EXTENT <= end else 0
            cap = (MICRO, EXTENT)[kind]
            n = min(end, at // cap * cap + cap) - at
            jobs.append((rows, n, at, kind, take(kind), at % cap, 0, 0))
            at, rows = at + n, rows + n
    if not jobs:
        jobs, rows = [(0, 1, case["context"], 0, take(0), case["context"] % MICRO, 0, 0)], 1
    # Pages in a scattered order, as a server's free lists hand them out.
    order = [np.random.RandomState(case["mix"] % (1 << 31)).permutation(max(1, n)) for n in free]
    jobs = [j[:4] + (int(order[j[3]][j[4]]), j[5], int(order[0][j[6]]) if j[7] else 0, j[7]) for j in jobs]
    return jobs, rows, max(1, free[0]), max(1, free[1])


def _prepare_append(case, seed):
    jobs, rows, micro, extent = _append_plan(case)
    kvh, dim, qh = case["kvh"], case["dim"], case["kvh"] * case["group"]
    qkv = _normal(seed, 1, rows, (qh + 2 * kvh) * dim)
    q = torch.zeros(rows, qh * dim, dtype=torch.float16, device="cuda")
    elements = 2 * kvh * dim * (micro * MICRO + extent * EXTENT)
    if own:
        device = _package()
        storage = device.Storage(1, kvh, dim, micro, extent)
        pool = torch.as_tensor(_Memory(storage, elements), device="cuda")
        pool.copy_(_normal(seed, 2, elements))
        table = np.zeros(len(jobs), dtype=device.APPEND_ROPE_JOB)
        for name, k in (("first_row", 0), ("token_count", 1), ("position", 2), ("dst_kind", 3), ("dst_slot", 4), ("dst_token", 5), ("cow_slot", 6),
                        ("cow_tokens", 7)):
            table[name] = [j[k] for j in jobs]
        return {"storage": storage, "jobs": _on_gpu(table), "count": (len(jobs), max(j[1] for j in jobs)), "qkv": qkv, "rows": rows, "qh": qh,
                "rope": device.Rope(case["theta"], case["rotary"], case["adjacent"]), "q": q, "pool": pool}
    kind, slot, token, position, copies = [], [], [], [], []
    for _, n, at, k, s, t, source, copied in jobs:
        kind += [k] * n
        slot += [s] * n
        token += range(t, t + n)
        position += range(at, at + n)
        copies += [(source, s, c) for c in range(copied)]
    return {"case": case, "pool": _normal(seed, 2, elements), "qkv": qkv, "q": q, "where": [_ints(v) for v in (kind, slot, token)], "position": _ints(position),
            "copies": _ints(copies).reshape(-1, 3), "micro": micro}


def _offsets(case, micro, kind, slot, token):
    """Elements of (row, head, dim) in the pool, of K and of V."""
    kvh, dim = case["kvh"], case["dim"]
    cap = torch.where(kind == 1, EXTENT, MICRO)[:, None, None]
    base = 2 * kvh * dim * (torch.where(kind == 1, micro * MICRO + slot * EXTENT, slot * MICRO))[:, None, None]
    head = torch.arange(kvh, device="cuda")[None, :, None]
    d = torch.arange(dim, device="cuda")[None, None, :]
    token = token[:, None, None]
    base = base + head * 2 * cap * dim
    width = torch.where(kind == 1, 32, MICRO)[:, None, None]
    return base + d // 32 * cap * 32 + token * 32 + d % 32, base + cap * dim + token // width * dim * width + d * width + token % width


def _run_append(s):
    if own:
        s["storage"].append_rope_launch(s["jobs"].data_ptr(), *s["count"], 0, s["qkv"].data_ptr(), s["qkv"].shape[1], s["rows"], s["qh"], s["rope"],
                                        s["q"].data_ptr(), s["q"].shape[1])
        return s["q"], s["pool"]
    case, pool = s["case"], s["pool"]
    kvh, dim, rotary, qh = case["kvh"], case["dim"], case["rotary"], case["kvh"] * case["group"]
    if len(s["copies"]):
        source, slot, token = s["copies"].unbind(1)
        zero = torch.zeros_like(source)
        for a, b in zip(_offsets(case, s["micro"], zero, slot, token), _offsets(case, s["micro"], zero, source, token)):
            pool[a] = pool[b]
    x = s["qkv"].float().view(len(s["qkv"]), qh + 2 * kvh, dim)
    # Angles of far positions in 64 bits.
    frequency = case["theta"] ** (-torch.arange(0, rotary, 2, device="cuda", dtype=torch.float64) / rotary)
    angle = s["position"].double()[:, None, None] * frequency
    cos, sin = angle.cos().float(), angle.sin().float()
    turned = x[:, :qh + kvh, :rotary]
    if case["adjacent"]:
        a, b = turned[..., 0::2], turned[..., 1::2]
        turned = torch.stack((a * cos - b * sin, b * cos + a * sin), -1).flatten(2)
    else:
        a, b = turned[..., :rotary // 2], turned[..., rotary // 2:]
        turned = torch.cat((a * cos - b * sin, b * cos + a * sin), -1)
    turned = torch.cat((turned, x[:, :qh + kvh, rotary:]), -1).half()
    s["q"].copy_(turned[:, :qh].flatten(1))
    at_k, at_v = _offsets(case, s["micro"], *s["where"])
    pool[at_k] = turned[:, qh:]
    pool[at_v] = x[:, qh + kvh:].half()
    return s["q"], pool


def _exact_append(case, seed):
    jobs, rows, micro, extent = _append_plan(case)
    kvh, dim, rotary, qh = case["kvh"], case["dim"], case["rotary"], case["kvh"] * case["group"]
    qkv = _normal(seed, 1, rows, (qh + 2 * kvh) * dim).double().view(rows, qh + 2 * kvh, dim)
    pool = _normal(seed, 2, 2 * kvh * dim * (micro * MICRO + extent * EXTENT)).double()
    half = torch.arange(rotary // 2, device="cuda", dtype=torch.float64)
    positions = torch.cat([torch.arange(j[2], j[2] + j[1], device="cuda", dtype=torch.float64) for j in jobs])
    turn = torch.polar(torch.ones(rows, rotary // 2, device="cuda", dtype=torch.float64),
                       positions[:, None] * torch.exp(half * (-2.0 / rotary * math.log(case["theta"])))[None])
    first = 2 * torch.arange(rotary // 2, device="cuda") if case["adjacent"] else torch.arange(rotary // 2, device="cuda")
    second = first + (1 if case["adjacent"] else rotary // 2)
    z = torch.complex(qkv[:, :qh + kvh, first].contiguous(), qkv[:, :qh + kvh, second].contiguous()) * turn[:, None, :]
    qkv[:, :qh + kvh, first], qkv[:, :qh + kvh, second] = z.real, z.imag
    # K and V of a page's token as strided views of its block.
    size = 2 * kvh * dim
    views = []
    for pages, cap in ((pool[:size * micro * MICRO], MICRO), (pool[size * micro * MICRO:], EXTENT)):
        block = pages.view(-1, kvh, 2, cap * dim)
        width = 32 if cap % 32 == 0 else cap
        views.append((block[:, :, 0].view(-1, kvh, dim // 32, cap, 32), block[:, :, 1].view(-1, kvh, cap // width, dim, width), width))
    micro_k, micro_v, _ = views[0]
    for _, _, _, _, slot, _, source, copied in jobs:
        if copied:
            micro_k[slot, :, :, :copied] = micro_k[source, :, :, :copied]
            micro_v[slot, :, 0, :, :copied] = micro_v[source, :, 0, :, :copied]
    row = 0
    for kind in (0, 1):
        k, v, width = views[kind]
        mine = [(j[0] + i, j[4], j[5] + i) for j in jobs if j[3] == kind for i in range(j[1])]
        if mine:
            row, slot, token = _ints(mine).unbind(1)
            k[slot, :, :, token] = qkv[row, qh:qh + kvh].view(-1, kvh, dim // 32, 32)
            v[slot, :, token // width, :, token % width] = qkv[row, qh + kvh:]
    return qkv[:, :qh].reshape(rows, qh * dim), pool


def _work_append(case):
    jobs, rows, _, _ = _append_plan(case)
    kvh, dim, qh = case["kvh"], case["dim"], case["kvh"] * case["group"]
    copied = sum(j[7] for j in jobs)
    return {"bytes": rows * 4 * (qh + 2 * kvh) * dim + copied * 8 * kvh * dim, "flops": rows * (qh + kvh) * case["rotary"] * 3}


# ---- shared ------------------------------------------------------------------


def _shared_plan(case):
    """(groups as (first lane, lanes, prefix tokens), each lane's tokens after its prefix)."""
    rng = random.Random(case["mix"] * 1033)
    groups = [(g * case["lanes"], case["lanes"], case["prefix"] + rng.randint(0, 7)) for g in range(case["groups"])]
    count = case["groups"] * case["lanes"] + case["alone"]
    return groups, [_log_uniform(rng, case["least"], case["most"]) for _ in range(count)]


def _shared_tokens(case, seed):
    """Every physical token's K and V, ([tokens][kvh][dim]): the groups' prefixes, then each lane's own; the queries."""
    groups, tails = _shared_plan(case)
    total, kvh, dim = sum(p for _, _, p in groups) + sum(tails), case["kvh"], case["dim"]
    # Queries of twice unit variance, so that some keys weigh far more than others.
    return (_normal(seed, 1, total, kvh, dim), _normal(seed, 2, total, kvh, dim),
            (2 * _normal(seed, 3, len(tails), kvh * case["group"], dim).float()).half())


def _shared_spans(case):
    """For each lane the ranges of physical tokens that it attends to: its group's prefix, its own."""
    groups, tails = _shared_plan(case)
    own_at, at, shared = sum(p for _, _, p in groups), 0, {}
    for first, lanes, prefix in groups:
        shared.update({lane: (at, at + prefix) for lane in range(first, first + lanes)})
        at += prefix
    spans = []
    for lane, tail in enumerate(tails):
        spans.append((shared.get(lane, (0, 0)), (own_at, own_at + tail)))
        own_at += tail
    return spans


def _shared_pages(case):
    """(micro pages, extent pages, entries of each lane's table, pages as (kind, slot, tokens, how many of them the prefix's, and where the
    prefix's and the lane's own would begin)).  Full pages inside a prefix are shared; where a prefix ends inside a page, each lane
    holds a copy of it and goes on there."""
    groups, tails = _shared_plan(case)
    free, tables, contents, page_of = [0, 0], [], {}, {}
    spans = _shared_spans(case)
    for (p0, p1), (o0, o1) in spans:
        prefix, total, at, entries = p1 - p0, p1 - p0 + o1 - o0, 0, []
        while at < total:
            kind = 1 if at + EXTENT <= total and at % EXTENT == 0 and (at + EXTENT <= prefix or at >= prefix // MICRO * MICRO) else 0
            n = min((MICRO, EXTENT)[kind], total - at)
            key = (p0, at, kind) if at + n <= prefix and n == (MICRO, EXTENT)[kind] else None
            if key is None or key not in page_of:
                slot = free[kind]
                free[kind] += 1
                contents[kind, slot] = (n, max(0, min(n, prefix - at)), p0 + at, o0 + at - prefix)
                if key is not None:
                    page_of[key] = slot
            else:
                slot = page_of[key]
            entries.append((slot, 1, at, n, (MICRO, EXTENT)[kind], kind))
            at += n
        tables.append(entries)
    order = [np.random.RandomState(case["mix"] % (1 << 31)).permutation(max(1, n)) for n in free]
    tables = [[(int(order[e[5]][e[0]]),) + e[1:] for e in t] for t in tables]
    pages = [(kind, int(order[kind][slot]), *c) for (kind, slot), c in contents.items()]
    return max(1, free[0]), max(1, free[1]), tables, pages


def _prepare_shared(case, seed):
    keys, values, query = _shared_tokens(case, seed)
    spans = _shared_spans(case)
    kvh, dim, qh = case["kvh"], case["dim"], case["kvh"] * case["group"]
    counts = [p1 - p0 + o1 - o0 for (p0, p1), (o0, o1) in spans]
    if own:
        device = _package()
        micro, extent, tables, pages = _shared_pages(case)
        storage = device.Storage(1, kvh, dim, micro, extent)
        # A page's tokens come from the prefix, the lane's own or, at the fork, both.
        jobs = np.zeros(2 * len(pages), dtype=device.APPEND_JOB)
        n = 0
        row = 2 * kvh * dim
        for kind, slot, tokens, from_prefix, p, o in pages:
            for first, count, source in ((0, from_prefix, p), (from_prefix, tokens - from_prefix, o + from_prefix)):
                if count:
                    jobs[n] = (keys.data_ptr() + source * row, values.data_ptr() + source * row, 0, kvh * dim, 0, 1, count, slot, 0, first, 0, kind, 0)
                    n += 1
        held = _on_gpu(jobs[:n])
        if device.lib().kimkv_append_batch(storage.h, held.data_ptr(), n, 1, None):
            raise RuntimeError("append")
        out = torch.zeros_like(query)
        items = np.zeros(len(counts), dtype=device.DECODE_ITEM)
        # The lanes' tables one after the other.
        flat = np.array([e for t in tables for e in t], dtype=device.BLOCK_DESC)
        on_gpu, at = _on_gpu(flat), 0
        for i, t in enumerate(tables):
            items[i] = (on_gpu.data_ptr() + at * 20, len(t), counts[i], 0, query[i].data_ptr(), 0, out[i].data_ptr(), 1.0 / math.sqrt(dim))
            at += len(t)
        entries, plan = storage.shared_decode_plan(counts, _shared_plan(case)[0], qh)
        work = torch.zeros(max(1, plan.workspace_bytes // 4), dtype=torch.float32, device="cuda")
        return {"storage": storage, "items": _on_gpu(items), "entries": _on_gpu(entries), "plan": plan, "work": work, "out": out, "held": (on_gpu, query, held, keys, values)}
    index = np.zeros((len(counts), max(counts)), dtype=np.int64)
    for i, ((p0, p1), (o0, o1)) in enumerate(spans):
        index[i, :p1 - p0] = np.arange(p0, p1)
        index[i, p1 - p0:counts[i]] = np.arange(o0, o1)
    return {"case": case, "keys": keys, "values": values, "query": query, "index": torch.from_numpy(index).cuda(), "counts": _ints(counts)}


def _run_shared(s):
    if own:
        s["storage"].shared_decode_launch(s["items"].data_ptr(), s["entries"].data_ptr(), s["plan"], s["work"].data_ptr())
        return s["out"]
    case, index = s["case"], s["index"]
    lanes, most = index.shape
    kvh, dim = case["kvh"], case["dim"]
    q = s["query"].float().view(lanes, kvh, case["group"], dim)
    scores = q @ s["keys"].float()[index].permute(0, 2, 3, 1) / math.sqrt(dim)
    scores.masked_fill_((torch.arange(most, device="cuda") >= s["counts"][:, None])[:, None, None, :], -math.inf)
    weights = (scores - scores.amax(-1, keepdim=True)).exp()
    out = weights @ s["values"].float()[index].transpose(1, 2) / weights.sum(-1, keepdim=True)
    return out.half().view(lanes, -1, dim)


def _exact_shared(case, seed):
    keys, values, query = _shared_tokens(case, seed)
    kvh, group, dim = case["kvh"], case["group"], case["dim"]
    out = torch.empty(len(query), kvh * group, dim, dtype=torch.float64, device="cuda")
    for i, ((p0, p1), (o0, o1)) in enumerate(_shared_spans(case)):
        k = torch.cat((keys[p0:p1], keys[o0:o1])).double()
        v = torch.cat((values[p0:p1], values[o0:o1])).double()
        for h in range(kvh):
            p = torch.softmax(query[i, h * group:(h + 1) * group].double() @ k[:, h].t().contiguous() * dim ** -0.5, 1)
            out[i, h * group:(h + 1) * group] = p @ v[:, h].contiguous()
    return out


def _work_shared(case):
    groups, tails = _shared_plan(case)
    kvh, dim, qh = case["kvh"], case["dim"], case["kvh"] * case["group"]
    pairs = sum(lanes * prefix for _, lanes, prefix in groups) + sum(tails)
    return {"bytes": (sum(p for _, _, p in groups) + sum(tails)) * 4 * kvh * dim + len(tails) * 4 * qh * dim, "flops": 4 * qh * dim * pairs}


# ---- logits ------------------------------------------------------------------


def _logits_plan(case):
    """Each row's (history length, biases, masked, repetition, presence, frequency)."""
    rng = random.Random(case["mix"] * 1039)
    return [(rng.randint(0, case["history"]), rng.randint(0, min(case["biases"], case["vocab"] // 2)), rng.random() < case["masked"],
             rng.choice([1.0, 1.1, 1.3]), rng.choice([0.0, 0.5]), rng.choice([0.0, 0.2])) for _ in range(case["rows"])]


def _logits_inputs(case, seed):
    """Logits, histories, (bias tokens, bias values) and allowed tokens, on the GPU; lists by row."""
    rows, vocab = case["rows"], case["vocab"]
    plan = _logits_plan(case)
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed) * 65537 + 5)
    logits = 3 * torch.randn(rows, vocab, generator=g, device="cuda")
    # Text repeats itself: a few of the vocabulary's tokens make most of a history.
    pick = lambda n: (vocab * torch.rand(n, generator=g, device="cuda") ** 3).long().clamp_(max=vocab - 1)  # noqa: E731
    histories = list(pick(sum(p[0] for p in plan)).split([p[0] for p in plan]))
    # Distinct tokens in a scattered order, another start for each row.
    total = sum(p[1] for p in plan)
    order = torch.randperm(vocab, generator=g, device="cuda")
    start = torch.randint(0, vocab, (rows,), generator=g, device="cuda")
    values = (4 * torch.randn(total, generator=g, device="cuda")).split([p[1] for p in plan])
    biases = [(order[(start[r] + torch.arange(p[1], device="cuda")) % vocab], values[r]) for r, p in enumerate(plan)]
    words = (vocab + 31) // 32
    bits = torch.randint(-(1 << 31), 1 << 31, (rows, words), generator=g, device="cuda") & torch.randint(-(1 << 31), 1 << 31, (rows, words), generator=g, device="cuda")
    bits[~torch.tensor([p[2] for p in plan], device="cuda")] = -1
    return logits, plan, histories, biases, bits.int()


def _prepare_logits(case, seed):
    logits, plan, histories, biases, bits = _logits_inputs(case, seed)
    rows, vocab = logits.shape
    out = torch.empty_like(logits) if case["store"] else None
    if own:
        device = _package()
        history = torch.cat(histories).int()
        tokens, values = torch.cat([b[0] for b in biases]).int(), torch.cat([b[1] for b in biases])
        rules = np.zeros(rows, dtype=device.LOGITS_RULE)
        at_h = at_b = 0
        for r, (n, b, masked, repetition, presence, frequency) in enumerate(plan):
            rules[r] = (history.data_ptr() + 4 * at_h if n else 0, tokens.data_ptr() + 4 * at_b if b else 0, values.data_ptr() + 4 * at_b if b else 0,
                        bits[r].data_ptr() if masked else 0, n, b, repetition, presence, frequency)
            at_h, at_b = at_h + n, at_b + b
        picked = torch.zeros(rows, dtype=torch.int32, device="cuda")
        work = torch.zeros(device.logits_workspace_bytes(rows, vocab) // 4 + 1, dtype=torch.int32, device="cuda")
        return {"device": device, "logits": logits, "rules": _on_gpu(rules), "out": out, "picked": picked, "work": work, "held": (history, tokens, values, bits)}
    padded = torch.full((rows, max(1, max(p[0] for p in plan))), vocab, dtype=torch.int64, device="cuda")
    at, by = (torch.full((rows, max(1, max(p[1] for p in plan))), v, dtype=t, device="cuda") for v, t in ((vocab, torch.int64), (0.0, torch.float32)))
    for r in range(rows):
        padded[r, :plan[r][0]] = histories[r]
        at[r, :plan[r][1]], by[r, :plan[r][1]] = biases[r]
    factors = [torch.tensor([p[k] for p in plan], device="cuda")[:, None] for k in (3, 4, 5)]
    return {"logits": logits, "histories": padded, "biases": (at, by), "bits": bits, "factors": factors, "out": out, "picked": torch.zeros(rows, dtype=torch.int32, device="cuda")}


def _run_logits(s):
    logits, out, picked = s["logits"], s["out"], s["picked"]
    rows, vocab = logits.shape
    if own:
        s["device"].logits_adjust(logits.data_ptr(), rows, vocab, s["rules"].data_ptr(), out.data_ptr() if out is not None else 0, picked.data_ptr(), s["work"].data_ptr())
        return (picked,) if out is None else (picked, out)
    repetition, presence, frequency = s["factors"]
    # Padding counts for a token past the vocabulary.
    seen = torch.zeros(rows, vocab + 1, device="cuda").scatter_add_(1, s["histories"], torch.ones_like(s["histories"], dtype=torch.float32))[:, :vocab]
    bias = torch.zeros(rows, vocab + 1, device="cuda").scatter_add_(1, *s["biases"])[:, :vocab]
    x = torch.where(logits > 0, logits / repetition, logits * repetition)
    x = torch.where(seen > 0, x - (frequency * seen + presence), logits) + bias
    allowed = (s["bits"][:, :, None] >> torch.arange(32, device="cuda", dtype=torch.int32)) & 1
    x = torch.where(allowed.flatten(1)[:, :vocab] != 0, x, -math.inf)
    index = torch.arange(vocab, device="cuda")
    picked.copy_(torch.where(x == x.amax(1, keepdim=True), index, vocab).amin(1))
    if out is None:
        return (picked,)
    out.copy_(x)
    return picked, out


def _exact_logits(case, seed):
    logits, plan, histories, biases, bits = _logits_inputs(case, seed)
    if not case["store"]:
        return None
    x = logits.double()
    for r, (_, _, masked, repetition, presence, frequency) in enumerate(plan):
        # The factors as the 32-bit numbers that the rows hold.
        repetition, presence, frequency = (float(np.float32(v)) for v in (repetition, presence, frequency))
        token, count = torch.unique(histories[r], return_counts=True)
        v = x[r, token]
        x[r, token] = torch.where(v > 0, v / repetition, v * repetition) - frequency * count - presence
        x[r, biases[r][0]] += biases[r][1].double()
        if masked:
            bit = np.unpackbits(bits[r].cpu().numpy().view(np.uint8), bitorder="little")[:case["vocab"]]
            x[r, torch.from_numpy(bit == 0).cuda()] = -math.inf
    return None, x


def _work_logits(case):
    plan = _logits_plan(case)
    rows, vocab = case["rows"], case["vocab"]
    lists = sum(4 * p[0] + 8 * p[1] + (vocab // 8 if p[2] else 0) for p in plan)
    return {"bytes": rows * vocab * (8 if case["store"] else 4) + lists, "flops": rows * vocab}


# ---- what is called ----------------------------------------------------------


def prepare(case, seed):
    return {"op": case["op"], **{"append": _prepare_append, "shared": _prepare_shared, "logits": _prepare_logits}[case["op"]](case, seed)}


def run(state):
    return {"append": _run_append, "shared": _run_shared, "logits": _run_logits}[state["op"]](state)


def exact(case, seed):
    return {"append": _exact_append, "shared": _exact_shared, "logits": _exact_logits}[case["op"]](case, seed)


def work(case):
    return {"append": _work_append, "shared": _work_shared, "logits": _work_logits}[case["op"]](case)
