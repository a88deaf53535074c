"""What the page-pool operators are measured on: attention of a chunk of new tokens over the paged
cache, page copies, and row compaction.

The pool is ``[pages, 2 (k, v), layers, 128 rows, kv heads, 128]`` with its last page the null page, as
the decoder's cache has it. A case is a dict of plain values; ``op`` names the operator:

* ``chunk``: ``B`` requests with up to ``new`` new tokens behind up to ``cached`` rows. Every token
  attends its request's rows up to itself, all of them (``window`` 0) or the last ``window`` and the
  first ``prefix`` (the reference sliding window of this decoder); the new k and v rows are stored.
* ``copy``: ``count`` pages copied, whole (``tail`` 0) or their first rows (a fork's last page).
* ``compact``: of each request's ``rows`` rows, the first ``prefix`` and the last ``window`` kept in place
  (``share`` 0), or a random share of them moved into other pages (percent).
"""

import math

import torch

own = False

PAGE, DIM = 128, 128
TYPES = {"fp32": torch.float32, "bf16": torch.bfloat16}


def _chunk(name, **v):
    return {"name": name, "op": "chunk", "dtype": "fp32", "heads": 10, "kv_heads": 10, "layers": 2, "ragged": False,
            "window": 0, "prefix": 0, "pad": 0, **v}


def listed():
    return [
        # one request's next token at the decoder's longest context (512 prompt rows and a 128-row ring)
        _chunk("decode_b1_640", B=1, new=1, cached=639, layers=12),
        # the next token of the decoder's largest batch, contexts of all lengths
        _chunk("decode_b8_ragged", B=8, new=1, cached=639, layers=12, ragged=True),
        # drafted tokens checked against long contexts
        _chunk("verify_b8_8k", B=8, new=5, cached=8000, ragged=True),
        # one chunk of a long prompt that is fed in pieces
        _chunk("chunk_512_over_7700", B=1, new=512, cached=7700),
        # the prompt batch of the decoder's prefill benchmark: 8 sequences of 512 tokens
        _chunk("prompts_8x512", B=8, new=512, cached=0, layers=12),
        # a long prompt in one call: the largest case
        _chunk("prompt_8192", B=1, new=8192, cached=0),
        # shared KV heads in bf16, ragged chunks over a long cache, rows of padding behind the last request
        _chunk("gqa_bf16_2048", B=2, new=2048, cached=6000, dtype="bf16", heads=32, kv_heads=8, ragged=True, pad=100),
        # the sliding window with the prompt always visible, bf16 cache
        _chunk("window_bf16_700", B=4, new=700, cached=1500, dtype="bf16", ragged=True, window=128, prefix=512),
        # a batch forked: each request's last, partly filled page copied
        {"name": "fork_tails", "op": "copy", "dtype": "fp32", "heads": 10, "layers": 12, "count": 8, "tail": 77},
        # many whole pages moved (a pool defragmented, a batch of prefixes copied)
        {"name": "move_64_pages", "op": "copy", "dtype": "fp32", "heads": 10, "layers": 12, "count": 64, "tail": 0},
        # one long generation cut back to its prompt and its last 128 rows
        {"name": "compact_window", "op": "compact", "dtype": "fp32", "heads": 10, "layers": 12, "B": 1, "rows": 1500,
         "prefix": 512, "window": 128, "share": 0},
        # a batch's evicted rows dropped: the rows that stay go to fresh pages
        {"name": "compact_scattered", "op": "compact", "dtype": "bf16", "heads": 8, "layers": 4, "B": 8, "rows": 4000,
         "prefix": 0, "window": 0, "share": 60},
    ]


def _log(rng, low, high):
    return max(low, min(high, round(math.exp(rng.uniform(math.log(low), math.log(high + 0.5))))))


def draw(rng):
    kind = rng.random()
    dtype = rng.choice(["fp32", "fp32", "bf16"])
    if kind < 0.2:
        return {"op": "copy", "dtype": dtype, "heads": rng.choice([1, 2, 8, 10]), "layers": rng.randint(1, 12),
                "count": _log(rng, 1, 64), "tail": rng.choice([0, rng.randint(1, 128)])}
    if kind < 0.4:
        c = {"op": "compact", "dtype": dtype, "heads": rng.choice([1, 4, 8, 10]), "layers": rng.randint(1, 4),
             "B": rng.randint(1, 8), "rows": _log(rng, 64, 4000), "prefix": 0, "window": 0, "share": rng.randint(5, 95)}
        if rng.random() < 0.5 and c["rows"] > 600:
            c |= {"share": 0, "window": rng.randint(16, 128), "prefix": rng.randint(1, c["rows"] - 300)}
        return c
    while True:
        heads, kv_heads = rng.choice([(10, 10), (10, 10), (4, 4), (16, 2), (32, 8), (12, 3), (7, 1), (5, 5)])
        c = {"op": "chunk", "dtype": dtype, "heads": heads, "kv_heads": kv_heads, "layers": rng.randint(1, 3),
             "B": _log(rng, 1, 24), "new": _log(rng, 1, 8192), "cached": rng.choice([0, _log(rng, 1, 32000), _log(rng, 1, 32000)]),
             "ragged": rng.random() < 0.7, "window": 0, "prefix": 0, "pad": rng.choice([0, 0, 3, 64])}
        if rng.random() < 0.25:
            c |= {"window": _log(rng, 1, 1024), "prefix": rng.choice([0, rng.randint(1, 700)])}
        rows = c["new"] + c["cached"]
        elements = c["B"] * (rows + PAGE) * 2 * c["layers"] * kv_heads * DIM
        # no dearer than the largest listed case, in pairs of a query and a row, nor in cache
        if c["B"] * c["new"] * rows * heads <= 8192 * 8192 * 10 and elements <= 400e6:
            return c


def _spread(top, b, ragged, lowest):
    """Request b's length: `top`, or between an eighth of it and it."""
    return top if not ragged or b == 0 else max(lowest, min(top, top - top * (b * 5 % 8) // 8 - b))


def _lengths(case):
    """The requests' new tokens and cached rows."""
    n = [_spread(case["new"], b, case["ragged"], 1) for b in range(case["B"])]
    s = [_spread(case["cached"], b, case["ragged"], 0) for b in range(case["B"])]
    return n, s


def _keep_lists(case, g):
    """The rows that compaction keeps, ascending, per request."""
    lists = []
    for b in range(case["B"]):
        rows = max(1, case["rows"] - 37 * b) if case["share"] else case["rows"]
        if case["share"]:
            count = max(1, rows * case["share"] // 100)
            lists.append(torch.randperm(rows, generator=g)[:count].sort().values)
        else:
            lists.append(torch.cat([torch.arange(case["prefix"]), torch.arange(rows - case["window"], rows)]))
    return lists


def prepare(case, seed):
    dev = torch.device("cuda", torch.cuda.current_device())
    dt = TYPES[case["dtype"]]
    g = torch.Generator().manual_seed(seed)
    gd = torch.Generator(device=dev).manual_seed(seed)
    i32 = lambda v: torch.tensor(v, dtype=torch.int32).to(dev)  # noqa: E731

    def pool_of(pages, kv_heads):
        return torch.randn((pages, 2, case["layers"], PAGE, kv_heads, DIM), generator=gd, device=dev, dtype=dt)

    if case["op"] == "copy":
        count = case["count"]
        perm = torch.randperm(2 * count, generator=g).to(torch.int32)
        rows = None
        if case["tail"]:
            rows = i32([max(1, (case["tail"] + 29 * i) % PAGE) for i in range(count)])
        return {"case": case, "pool": pool_of(2 * count + 1, case["heads"]), "src": perm[:count].to(dev),
                "dst": perm[count:].to(dev), "rows": rows}
    if case["op"] == "compact":
        B = case["B"]
        lists = _keep_lists(case, g)
        most = max(len(k) for k in lists)
        keep = torch.zeros((B, most), dtype=torch.int32)
        for b, k in enumerate(lists):
            keep[b, : len(k)] = k.to(torch.int32)
        cols, to = -(-case["rows"] // PAGE), -(-most // PAGE)
        pages = B * (cols + (to if case["share"] else 0))
        perm = torch.randperm(pages, generator=g).to(torch.int32)
        src = perm[: B * cols].reshape(B, cols).to(dev)
        dst = perm[B * cols:].reshape(B, to).to(dev) if case["share"] else src
        return {"case": case, "pool": pool_of(pages + 1, case["heads"]), "src": src, "dst": dst, "keep": keep.to(dev),
                "keep_len": i32([len(k) for k in lists]), "total": sum(len(k) for k in lists)}
    n, s = _lengths(case)
    B, hq, hk = case["B"], case["heads"], case["kv_heads"]
    used = [-(-(n[b] + s[b]) // PAGE) for b in range(B)]
    pages = sum(used)
    perm = torch.randperm(pages, generator=g).to(torch.int32)
    lut = torch.full((B, max(used)), pages, dtype=torch.int32)  # unused entries: the null page
    at = 0
    for b in range(B):
        lut[b, : used[b]] = perm[at: at + used[b]]
        at += used[b]
    offsets = [sum(n[:b]) for b in range(B + 1)]
    T = offsets[B] + case["pad"]
    # q, k and v as slices of one fused projection's rows where the heads are shared, else buffers of their own
    if hq != hk:
        qkv = torch.randn((T, hq + 2 * hk, DIM), generator=gd, device=dev, dtype=dt)
        q, k, v = qkv[:, :hq], qkv[:, hq: hq + hk], qkv[:, hq + hk:]
    else:
        q, k, v = (torch.randn((T, hq, DIM), generator=gd, device=dev, dtype=dt) for _ in range(3))
    q.mul_(1.5)  # scores of a few units, so that some rows take most of a softmax
    return {"case": case, "pool": pool_of(pages + 1, hk), "q": q, "k": k, "v": v, "lut": lut.to(dev), "offsets": i32(offsets),
            "start": i32(s), "prefix": i32([case["prefix"]] * B) if case["prefix"] else None,
            "out": torch.zeros((T, hq, DIM), device=dev, dtype=dt), "tokens": offsets[B], "longest": max(n),
            "layer": case["layers"] - 1, "scale": 1.0 / math.sqrt(DIM)}


def _token_places(st):
    """(request, logical row) of each new token."""
    off = st["offsets"].long()
    n = off[1:] - off[:-1]
    req = torch.repeat_interleave(torch.arange(len(n), device=off.device), n, output_size=st["tokens"])
    i = torch.arange(st["tokens"], device=off.device) - off[req]
    return req, i, st["start"].long()[req] + i


def _plain_chunk(st):
    case, pool, layer = st["case"], st["pool"], st["layer"]
    hq, hk = case["heads"], case["kv_heads"]
    lut = st["lut"].long()
    B, cols = lut.shape
    req, i, row = _token_places(st)
    page, slot = lut[req, row // PAGE], row % PAGE
    pool[page, 0, layer, slot] = st["k"][: st["tokens"]]
    pool[page, 1, layer, slot] = st["v"][: st["tokens"]]
    keys = pool[lut, 0, layer].reshape(B, cols * PAGE, hk, DIM).permute(0, 2, 1, 3).float()
    values = pool[lut, 1, layer].reshape(B, cols * PAGE, hk, DIM).permute(0, 2, 1, 3).float()
    # each request's tokens in a row of their own, padded to the longest
    q = torch.zeros((B, st["longest"], hq, DIM), device=pool.device)
    q[req, i] = st["q"][: st["tokens"]].float()
    q = q.reshape(B, st["longest"], hk, hq // hk, DIM).permute(0, 2, 3, 1, 4)
    s = torch.matmul(q.reshape(B, hk, -1, DIM), keys.transpose(2, 3)).reshape(B, hk, hq // hk, st["longest"], cols * PAGE)
    s *= st["scale"]
    p = (st["start"].long()[:, None] + torch.arange(st["longest"], device=pool.device))[:, :, None]
    r = torch.arange(cols * PAGE, device=pool.device)[None, None, :]
    seen = r <= p
    if case["window"]:
        first = st["prefix"].long()[:, None, None] if st["prefix"] is not None else torch.zeros((1, 1, 1), device=pool.device)
        seen &= (r > p - case["window"]) | (r < first)
    s.masked_fill_(~seen[:, None, None], -math.inf)
    s -= s.max(-1, keepdim=True).values
    s.exp_()
    total = s.sum(-1, keepdim=True)
    o = torch.matmul(s.reshape(B, hk, -1, cols * PAGE), values).reshape(B, hk, hq // hk, st["longest"], DIM) / total
    o = o.permute(0, 3, 1, 2, 4).reshape(B, st["longest"], hq, DIM)
    out = torch.zeros_like(st["out"])
    out[: st["tokens"]] = o[req, i].to(out.dtype)
    return {"out": out, "pool": pool}


def _plain_copy(st):
    pool, src, dst = st["pool"], st["src"].long(), st["dst"].long()
    if st["rows"] is None:
        pool[dst] = pool[src]
    else:
        first = torch.arange(PAGE, device=pool.device)[None] < st["rows"][:, None]
        pool[dst] = torch.where(first[:, None, None, :, None, None], pool[src], pool[dst])
    return {"pool": pool}


def _plain_compact(st):
    pool, keep = st["pool"], st["keep"].long()
    n = st["keep_len"].long()
    req = torch.repeat_interleave(torch.arange(len(n), device=pool.device), n, output_size=st["total"])
    i = torch.arange(st["total"], device=pool.device) - (torch.cumsum(n, 0) - n)[req]
    old = keep[req, i]
    rows = pool[st["src"].long()[req, old // PAGE], :, :, old % PAGE]
    pool[st["dst"].long()[req, i // PAGE], :, :, i % PAGE] = rows
    return {"pool": pool}


def run(state):
    st = state
    if own:
        import importlib

        ops = importlib.import_module("unlimited-ocr-max_b200.ops")
        if st["case"]["op"] == "copy":
            ops.copy_pages(st["pool"], st["src"], st["dst"], rows=st["rows"])
            return {"pool": st["pool"]}
        if st["case"]["op"] == "compact":
            ops.compact_rows(st["pool"], st["src"], st["dst"], st["keep"], st["keep_len"])
            return {"pool": st["pool"]}
        out = ops.paged_chunk_attention(st["q"], st["k"], st["v"], st["pool"], st["layer"], st["lut"], st["offsets"],
                                        st["start"], st["scale"], window=st["case"]["window"], prefix=st["prefix"],
                                        out=st["out"])
        return {"out": out, "pool": st["pool"]}
    return {"chunk": _plain_chunk, "copy": _plain_copy, "compact": _plain_compact}[st["case"]["op"]](st)


def _pairs(case):
    """(visible pairs of a token and a row, cached rows that some token sees), over all requests."""
    pairs = seen = 0
    w, first = case["window"], case["prefix"]
    for n, s in zip(*_lengths(case)):
        if not w:
            pairs += n * s + n * (n + 1) // 2
            seen += s
        else:
            for p in range(s, s + n):
                low = max(0, p - w + 1)
                pairs += p + 1 - low + min(low, first)
            low = max(0, s - w + 1)
            seen += s - low + min(low, first)
    return pairs, seen


def work(case):
    size = TYPES[case["dtype"]].itemsize
    if case["op"] == "copy":
        row = 2 * case["layers"] * case["heads"] * DIM * size
        rows = [max(1, (case["tail"] + 29 * i) % PAGE) if case["tail"] else PAGE for i in range(case["count"])]
        return {"bytes": 2 * sum(rows) * row, "flops": 0}
    if case["op"] == "compact":
        row = 2 * case["layers"] * case["heads"] * DIM * size
        if not case["share"]:  # the prefix stays where it is
            moved = case["B"] * case["window"]
        else:
            moved = sum(max(1, max(1, case["rows"] - 37 * b) * case["share"] // 100) for b in range(case["B"]))
        return {"bytes": 2 * moved * row, "flops": 0}
    n, _ = _lengths(case)
    pairs, seen = _pairs(case)
    tokens = sum(n)
    q, kv = case["heads"] * DIM * size, 2 * case["kv_heads"] * DIM * size
    # q read, out written; the new rows read and stored; the cached rows read
    return {"bytes": tokens * (2 * q + 2 * kv) + seen * kv, "flops": 4 * DIM * case["heads"] * pairs}


def exact(case, seed):
    st = prepare(case, seed)
    pool = st["pool"]
    if case["op"] == "copy":
        was = pool.clone()
        limit = st["rows"].tolist() if st["rows"] is not None else [PAGE] * case["count"]
        for a, b, r in zip(st["src"].tolist(), st["dst"].tolist(), limit):
            pool[b, :, :, :r] = was[a, :, :, :r]
        return {"pool": pool}
    if case["op"] == "compact":
        was = pool.clone()
        src, dst = st["src"].tolist(), st["dst"].tolist()
        for b, count in enumerate(st["keep_len"].tolist()):
            old = st["keep"][b, :count].long()
            flat = torch.cat([was[p].transpose(0, 2) for p in src[b]])  # [rows, layers, 2, heads, dim]
            rows = flat[old]
            for c in range(-(-count // PAGE)):
                part = rows[c * PAGE: (c + 1) * PAGE]
                pool[dst[b][c], :, :, : len(part)] = part.transpose(0, 2)
        return {"pool": pool}
    n, s = _lengths(case)
    hq, hk, layer = case["heads"], case["kv_heads"], st["layer"]
    out = torch.zeros(st["out"].shape, dtype=torch.float64, device=pool.device)
    at = 0
    for b in range(case["B"]):
        pages = st["lut"][b].tolist()[: -(-(n[b] + s[b]) // PAGE)]
        for i in range(0, n[b] + s[b], PAGE):  # store this request's new rows that lie on page i / 128
            low, high = max(i, s[b]), min(i + PAGE, s[b] + n[b])
            if low < high:
                for kind, t in ((0, st["k"]), (1, st["v"])):
                    pool[pages[i // PAGE], kind, layer, low - i: high - i] = t[at + low - s[b]: at + high - s[b]]
        k = torch.cat([pool[p, 0, layer] for p in pages]).double()[: n[b] + s[b]]
        v = torch.cat([pool[p, 1, layer] for p in pages]).double()[: n[b] + s[b]]
        pos = torch.arange(s[b], s[b] + n[b], device=pool.device).unsqueeze(1)
        row = torch.arange(s[b] + n[b], device=pool.device).unsqueeze(0)
        hidden = row > pos
        if case["window"]:
            hidden |= (pos - row >= case["window"]) & (row >= case["prefix"])
        for h in range(hq):
            score = st["q"][at: at + n[b], h].double() @ k[:, h // (hq // hk)].T * st["scale"]
            weight = torch.exp(score - torch.logsumexp(score.masked_fill_(hidden, -math.inf), 1, keepdim=True))
            out[at: at + n[b], h] = weight @ v[:, h // (hq // hk)]
        at += n[b]
    return {"out": out, "pool": pool}
