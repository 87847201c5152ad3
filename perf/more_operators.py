"""Performance cases of a transformer layer's attention while it serves: rotary positions (HipRotary), the paged cache of
keys and values with its 8-bit form, written and read back, and the attention of new tokens over it (HipKvCache).

A case's "op":
  rotary  y = x with each head's first `rotary` channels turned by position * frequency, the frequencies scaled for
          long contexts where factor > 1.
  cache   k (turned) and v of the batch's new tokens into their pages, and the same tokens read back.
  attend  y = softmax(scale q k^T) v of the new tokens over their sequences' pages, causal, within `window` if any.
  step    the three as a layer calls them: q and k turned, k and v written, attended, and the new tokens read back.

A batch is sequences of `context` tokens (the new ones are its last), shorter by `skew` from the first to the last; each
has `new` new tokens, with "mixed" only the first and the others one.
"""
import math

import torch

own = False

DTYPES = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}


def listed():
    return [
        # one token of a small model: the smallest call, where latency counts
        {"name": "rotary one token f16", "op": "rotary", "storage": "f16", "rows": 1, "heads": 12, "dim": 64, "rotary": 64,
         "interleaved": False, "base": 1e4, "factor": 1.0, "far": 500, "pad": 0},
        # the query and key heads of a long prompt side by side in one buffer, frequencies scaled for a long context
        {"name": "rotary prompt bf16", "op": "rotary", "storage": "bf16", "rows": 8192, "heads": 40, "dim": 128,
         "rotary": 128, "interleaved": False, "base": 5e5, "factor": 8.0, "far": 0, "pad": 1024},
        # one new token for each of 48 sequences, cached in 8 bits
        {"name": "cache tokens i8 f16", "op": "cache", "storage": "f16", "format": "i8", "sequences": 48, "context": 1000,
         "new": 1, "skew": 0.7, "mixed": False, "kv": 8, "dim": 128, "page": 16, "rotary": 128, "interleaved": False,
         "base": 1e4, "factor": 1.0, "pad": 0},
        # four whole prompts, cached in 8 bits
        {"name": "cache prompts i8 bf16", "op": "cache", "storage": "bf16", "format": "i8", "sequences": 4,
         "context": 4096, "new": 4096, "skew": 0.0, "mixed": False, "kv": 8, "dim": 128, "page": 64, "rotary": 128,
         "interleaved": False, "base": 5e5, "factor": 8.0, "pad": 0},
        # full precision, odd sizes, neighbouring channels as pairs, a part of the head turned
        {"name": "cache ragged f32", "op": "cache", "storage": "f32", "format": "f32", "sequences": 7, "context": 911,
         "new": 301, "skew": 0.5, "mixed": False, "kv": 3, "dim": 40, "page": 8, "rotary": 20, "interleaved": True,
         "base": 1e4, "factor": 1.0, "pad": 5},
        # one token after a line of text: the smallest attention
        {"name": "attend short f16", "op": "attend", "storage": "f16", "format": "f16", "sequences": 1, "context": 77,
         "new": 1, "skew": 0.0, "mixed": False, "kv": 12, "group": 1, "dim": 64, "page": 16, "window": 0, "pad": 0},
        # full precision: a few ragged continuations
        {"name": "attend odd f32", "op": "attend", "storage": "f32", "format": "f32", "sequences": 3, "context": 333,
         "new": 45, "skew": 0.4, "mixed": False, "kv": 3, "group": 2, "dim": 72, "page": 8, "window": 0, "pad": 3},
        # continuations of several sequences within a sliding window
        {"name": "attend window f16", "op": "attend", "storage": "f16", "format": "f16", "sequences": 6, "context": 2500,
         "new": 131, "skew": 0.6, "mixed": False, "kv": 2, "group": 5, "dim": 80, "page": 16, "window": 512, "pad": 24},
        # one token of one very long sequence
        {"name": "attend long bf16", "op": "attend", "storage": "bf16", "format": "bf16", "sequences": 1,
         "context": 131072, "new": 1, "skew": 0.0, "mixed": False, "kv": 8, "group": 4, "dim": 128, "page": 64,
         "window": 0, "pad": 0},
        # a full batch of single tokens over an 8-bit cache: bound by reading it
        {"name": "attend tokens i8 bf16", "op": "attend", "storage": "bf16", "format": "i8", "sequences": 64,
         "context": 8192, "new": 1, "skew": 0.5, "mixed": False, "kv": 8, "group": 4, "dim": 128, "page": 16, "window": 0,
         "pad": 0},
        # two whole prompts: bound by the matrix cores, the largest case
        {"name": "attend prompts bf16", "op": "attend", "storage": "bf16", "format": "bf16", "sequences": 2,
         "context": 8192, "new": 8192, "skew": 0.0, "mixed": False, "kv": 8, "group": 4, "dim": 128, "page": 64,
         "window": 0, "pad": 0},
        # a server's step: a piece of one prompt beside the single tokens of 31 other sequences, cached in 8 bits
        {"name": "step mixed i8 bf16", "op": "step", "storage": "bf16", "format": "i8", "sequences": 32, "context": 4096,
         "new": 512, "skew": 0.8, "mixed": True, "kv": 8, "group": 4, "dim": 128, "page": 16, "window": 0, "rotary": 128,
         "interleaved": False, "base": 5e5, "factor": 8.0, "pad": 0},
    ]


# ---------------------------------------------------------------------------------------------
# drawn cases
# ---------------------------------------------------------------------------------------------
def _log(rng, lo, hi):
    """An integer of [lo, hi], spread evenly over its logarithm."""
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def _turns(rng, dim):
    rotary = rng.choice([dim, dim, dim // 2, max(2, dim // 4 // 2 * 2)])
    return {"rotary": rotary, "interleaved": rng.random() < 0.4, "base": rng.choice([1e4, 5e5]),
            "factor": rng.choice([1.0, 1.0, 4.0, 8.0])}


def draw(rng):
    op = rng.choice(["rotary", "cache", "cache", "attend", "attend", "attend", "attend", "step"])
    storage = rng.choice(["f16", "f16", "f16", "bf16", "bf16", "bf16", "f32"])
    dim = rng.choice([64, 64, 128, 128, 128, 256, 8 * rng.randint(4, 32)])
    case = {"op": op, "storage": storage, "dim": dim, "pad": rng.choice([0, 0, 0, rng.randint(1, 64)])}
    if op == "rotary":
        case.update(rows=_log(rng, 1, 8192), heads=_log(rng, 1, 64), far=rng.choice([0, 1000, 100000]), **_turns(rng, dim))
        while case["rows"] * case["heads"] * dim > 4e7:
            case["rows"] = max(1, case["rows"] // 2)
        return case
    kv, group = _log(rng, 1, 16), rng.choice([1, 1, 2, 4, 4, 5, 7, 8, 16])
    case.update(format=rng.choice([storage, storage, "i8"]), sequences=_log(rng, 1, 128), skew=rng.choice([0.0, 0.5, 0.9]),
                kv=kv, page=rng.choice([8, 16, 16, 32, 64, 128]), mixed=op == "step" and rng.random() < 0.7)
    if op != "cache":
        case.update(group=group, window=rng.choice([0, 0, 0, _log(rng, 16, 4096)]))
    if op != "attend":
        case.update(**_turns(rng, dim))
    shape = rng.choice(["tokens", "piece", "prompt"])
    case["context"] = _log(rng, 1, 65536 if shape == "tokens" else 8192)
    case["new"] = {"tokens": 1, "piece": min(case["context"], _log(rng, 2, 600)), "prompt": case["context"]}[shape]
    most = {"bytes": 8e8, "flops": 1.0e11 if storage == "f32" else 7e11}
    while any(work(case)[k] > most[k] for k in most) or _held(case) > 2e8:
        if case["sequences"] > 1:
            case["sequences"] //= 2
        else:
            case["context"] = max(1, case["context"] // 2)
            case["new"] = min(case["new"], case["context"])
    return case


# ---------------------------------------------------------------------------------------------
# state
# ---------------------------------------------------------------------------------------------
def _lengths(case):
    """(tokens, new tokens) of each sequence."""
    n, out = case["sequences"], []
    for s in range(n):
        length = max(1, round(case["context"] * (1 - case["skew"] * s / n)))
        out.append((length, min(length, 1 if case["mixed"] and s else case["new"])))
    return out


def _rows(case):
    return sum(new for _, new in _lengths(case))


def _held(case):
    """Values of K and V that the batch's pages hold."""
    return 2 * sum(length for length, _ in _lengths(case)) * case["kv"] * case["dim"]


def _seen(case):
    """(tokens that some new token attends to, pairs of a new token and one it attends to)."""
    tokens = pairs = 0
    for length, new in _lengths(case):
        window = case["window"] or length
        tokens += min(length, new - 1 + window)
        for first in range(length - new + 1, length + 1, 4096):  # (positions first .. last see min(position, window))
            last = min(first + 4095, length)
            if last <= window:
                pairs += (first + last) * (last - first + 1) // 2
            elif first >= window:
                pairs += window * (last - first + 1)
            else:
                pairs += (first + window) * (window - first + 1) // 2 + window * (last - window)
    return tokens, pairs


def _matrix(g, rows, cols, pad, dtype, by=1.0):
    """[rows, cols] inside rows of cols + pad values."""
    t = torch.randn((rows, cols + pad), generator=g, device="cuda", dtype=torch.float32)
    return (by * t).to(dtype)[:, :cols]


def _inputs(case, seed):
    """What both forms and the definition work on."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    dtype, dim, pad = DTYPES[case["storage"]], case["dim"], case["pad"]
    s = {"case": case, "dtype": dtype}
    if case["op"] == "rotary":
        s["x"] = _matrix(g, case["rows"], case["heads"] * dim, pad, dtype)
        s["positions"] = torch.arange(case["rows"], device="cuda", dtype=torch.int32) + case["far"] + seed % 3
        return s
    kv, page = case["kv"], case["page"]
    lengths = _lengths(case)
    rows, total = sum(n for _, n in lengths), sum(n for n, _ in lengths)
    host = torch.Generator().manual_seed(seed)
    counts = [-(-length // page) for length, _ in lengths]
    pages = sum(counts) + 3
    order, at = torch.randperm(pages, generator=host), 0
    tables = torch.full((len(lengths), max(counts) + 1), -1, dtype=torch.int32)
    for i, n in enumerate(counts):
        tables[i, :n] = order[at:at + n]
        at += n
    s.update(pages=pages, rows=rows, tables=tables.cuda(),
             lengths=torch.tensor([n for n, _ in lengths], dtype=torch.int32).cuda(),
             starts=torch.tensor([0] + [n for _, n in lengths]).cumsum(0).to(torch.int32).cuda())
    if case["op"] != "cache":  # the sequences' earlier tokens (an attention's new ones too)
        s["old_k"] = _matrix(g, total, kv * dim, 0, dtype)
        s["old_v"] = _matrix(g, total, kv * dim, 0, dtype)
    if case["op"] == "attend":
        s["q"] = _matrix(g, rows, kv * case["group"] * dim, pad, dtype, 1.5)
        return s
    # one row of a projection: query, key and value heads side by side
    q = kv * case["group"] * dim if case["op"] == "step" else 0
    fused = _matrix(g, rows, q + 2 * kv * dim, pad, dtype, 1.5)
    s["k"], s["v"] = fused[:, q:q + kv * dim], fused[:, q + kv * dim:]
    if q:
        s["q"] = fused[:, :q]
    return s


def prepare(case, seed):
    s = _inputs(case, seed)
    if own:
        _handles(s)
    elif case["op"] != "rotary":
        _plain_pool(s)
    if case["op"] != "rotary":
        s["old_k"] = s["old_v"] = None
    if "rotary" in case:
        s["frequencies"] = torch.tensor(_frequencies(case), device="cuda", dtype=torch.float64)
    return s


def _scaling(case):
    """Frequencies that turn less than once within the first 4096 positions are divided by the factor, those that turn
    more than four times kept, and those in between blended."""
    return {"factor": case["factor"], "original": 4096 if case["factor"] > 1 else 0, "low": 1.0, "high": 4.0}


def _frequencies(case):
    out, half, by = [], case["rotary"] // 2, _scaling(case)
    for j in range(half):
        f = case["base"] ** (-j / half)
        keep = (by["original"] * f / (2 * math.pi) - by["low"]) / (by["high"] - by["low"])
        keep = min(1.0, max(0.0, keep)) if by["original"] else 1.0
        out.append(f * (keep + (1 - keep) / by["factor"]))
    return out


def _handles(s):
    """What a program keeps of the framework: the rotation, the cache with its pages, the buffers."""
    from simdonnx_amd.backend import HipBackend, HipKvBatch, HipKvCache, HipRotary
    case, hip, dtype, dim = s["case"], HipBackend.default(), s["dtype"], s["case"]["dim"]
    if "rotary" in case:
        s["rotary"] = HipRotary(hip, dim, rotary_dim=case["rotary"], interleaved=case["interleaved"], base=case["base"],
                                **_scaling(case))
    if case["op"] == "rotary":
        s["y"] = torch.zeros((case["rows"], case["heads"] * dim + case["pad"]), device="cuda", dtype=dtype)[:, :case["heads"] * dim]
        return
    kv, rows = case["kv"], s["rows"]
    s["cache"] = cache = HipKvCache(hip, kv, dim, page=case["page"], format=case["format"])
    s["pool"] = torch.zeros(s["pages"] * cache.page_bytes, device="cuda", dtype=torch.uint8)
    batch = dict(pool=s["pool"].data_ptr(), pages=s["pages"], tables=s["tables"].data_ptr(), table_pages=s["tables"].shape[1],
                 lengths=s["lengths"].data_ptr(), sequences=case["sequences"])
    s["batch"] = HipKvBatch(starts=s["starts"].data_ptr(), rows=rows, **batch)
    if "old_k" in s:
        whole = torch.cat([s["lengths"].new_zeros(1), s["lengths"].cumsum(0)]).to(torch.int32)
        cache.write(HipKvBatch(starts=whole.data_ptr(), rows=s["old_k"].shape[0], **batch), s["old_k"].data_ptr(),
                    s["old_v"].data_ptr(), case["storage"], stream=torch.cuda.current_stream().cuda_stream)
        torch.cuda.synchronize()
    if "k" in s:
        s["k_back"] = torch.zeros((rows, kv * dim), device="cuda", dtype=dtype)
        s["v_back"] = torch.zeros((rows, kv * dim), device="cuda", dtype=dtype)
    if "q" in s:
        heads = kv * case["group"]
        s["turned"] = torch.zeros((rows, heads * dim), device="cuda", dtype=dtype)
        s["y"] = torch.zeros((rows, heads * dim + case["pad"]), device="cuda", dtype=dtype)[:, :heads * dim]
        size = cache.workspace(rows, case["sequences"], heads)
        s["work"] = torch.empty(max(1, size), device="cuda", dtype=torch.uint8)


def _plain_pool(s):
    """Pages as plain tensors: [page, token, kv head, channel], in 8 bits with a scale for each token and head."""
    case = s["case"]
    shape = (s["pages"], case["page"], case["kv"], case["dim"])
    for name in ("k", "v"):
        if case["format"] == "i8":
            s["pool_" + name] = torch.zeros(shape, device="cuda", dtype=torch.int8)
            s["scale_" + name] = torch.zeros(shape[:3], device="cuda", dtype=torch.float32)
        else:
            s["pool_" + name] = torch.zeros(shape, device="cuda", dtype=s["dtype"])
    if "old_k" in s:
        at = 0
        for i, (length, _) in enumerate(_lengths(case)):
            token = torch.arange(length, device="cuda")
            for name in ("k", "v"):
                x = s["old_" + name][at:at + length].view(length, case["kv"], case["dim"])
                _plain_store(s, name, s["tables"][i, token // case["page"]].long(), token % case["page"], x)
            at += length


# ---------------------------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------------------------
def run(state):
    if own:
        return _run_own(state)
    case = state["case"]
    if case["op"] == "rotary":
        return {"y": _plain_turned(state, state["x"], state["positions"], case["heads"]).to(state["dtype"]).flatten(1)}
    out = {}
    q = state.get("q")
    if "k" in state:
        page, token, position = _plain_slots(state)
        _plain_store(state, "k", page, token, _plain_turned(state, state["k"], position, case["kv"]))
        _plain_store(state, "v", page, token, state["v"].reshape(len(position), case["kv"], case["dim"]))
        for name in ("k", "v"):
            out[name] = _plain_load(state, name, page, token).to(state["dtype"]).flatten(1)
        if q is not None:
            q = _plain_turned(state, q, position, case["kv"] * case["group"]).to(state["dtype"]).flatten(1)
    if q is not None:
        out["y"] = _plain_attend(state, q)
    return out


def _run_own(state):
    case, stream, st = state["case"], torch.cuda.current_stream().cuda_stream, state["case"]["storage"]
    if case["op"] == "rotary":
        x, y = state["x"], state["y"]
        state["rotary"].run(x.data_ptr(), state["positions"].data_ptr(), case["rows"], case["heads"], y.data_ptr(), st,
                            x.stride(0), y.stride(0), stream=stream)
        return {"y": y}
    cache, batch, out, q = state["cache"], state["batch"], {}, state.get("q")
    heads = case["kv"] * case.get("group", 0)
    if "k" in state:
        k, v, turn = state["k"], state["v"], {}
        if q is not None:
            turn = dict(q=q.data_ptr(), ldq=q.stride(0), q_heads=heads, y=state["turned"].data_ptr())
            q = state["turned"]
        cache.write(batch, k.data_ptr(), v.data_ptr(), st, k.stride(0), v.stride(0), rotary=state["rotary"], stream=stream, **turn)
        out["k"], out["v"] = state["k_back"], state["v_back"]
    if q is not None:
        y, work = state["y"], state["work"]
        cache.attend(batch, q.data_ptr(), heads, y.data_ptr(), st, q.stride(0), y.stride(0), window=case["window"],
                     workspace=work.data_ptr(), workspace_bytes=work.numel(), stream=stream)
        out["y"] = y
    if "k" in out:
        cache.read(batch, out["k"].data_ptr(), out["v"].data_ptr(), st, stream=stream)
    return out


# ---- plain forms ----
def _plain_turned(s, x, positions, heads):
    """Angles in 64 bits, as far positions need, and the turned values too: their 8-bit form has borders."""
    case = s["case"]
    x = x.reshape(x.shape[0], heads, case["dim"])
    angle = positions.double()[:, None] * s["frequencies"]
    cos, sin = torch.cos(angle)[:, None, :], torch.sin(angle)[:, None, :]
    n, y = case["rotary"], x.double()
    at = (slice(0, n, 2), slice(1, n, 2)) if case["interleaved"] else (slice(0, n // 2), slice(n // 2, n))
    a, b = y[..., at[0]], y[..., at[1]]
    y = y.clone()
    y[..., at[0]], y[..., at[1]] = a * cos - b * sin, b * cos + a * sin
    return y.float()


def _plain_slots(s):
    """(page, token of the page, position) of each new token."""
    starts, lengths = s["starts"].long(), s["lengths"].long()
    row = torch.arange(s["rows"], device="cuda")
    sequence = (row[:, None] >= starts[None, 1:]).sum(1)
    position = lengths[sequence] - starts[sequence + 1] + row
    page = s["case"]["page"]
    return s["tables"][sequence, position // page].long(), position % page, position


def _plain_store(s, name, page, token, x):
    pool = s["pool_" + name]
    if pool.dtype != torch.int8:
        pool[page, token] = x.to(pool.dtype)
        return
    for i in range(0, x.shape[0], 65536):  # (in 64 bits next to a half)
        part = x[i:i + 65536].double()
        top = part.abs().amax(2, keepdim=True)
        pool[page[i:i + 65536], token[i:i + 65536]] = torch.round(part * 127 / torch.where(top > 0, top, torch.ones_like(top))).to(torch.int8)
        s["scale_" + name][page[i:i + 65536], token[i:i + 65536]] = top.float()[..., 0] / 127


def _plain_load(s, name, page, token):
    x = s["pool_" + name][page, token].float()
    return x * s["scale_" + name][page, token][..., None] if s["case"]["format"] == "i8" else x


def _plain_attend(s, q):
    case = s["case"]
    kv, group, dim, page = case["kv"], case["group"], case["dim"], case["page"]
    out = torch.empty((s["rows"], kv * group * dim), device="cuda", dtype=s["dtype"])
    start = 0
    for i, (length, new) in enumerate(_lengths(case)):
        token = torch.arange(length, device="cuda")
        at = s["tables"][i, token // page].long()
        k, v = (_plain_load(s, name, at, token % page) for name in ("k", "v"))
        mine = q[start:start + new].float().view(new, kv, group, dim)
        for first in range(0, new, 1024):
            part = mine[first:first + 1024]
            n = part.shape[0]
            position = length - new + first + torch.arange(n, device="cuda")
            hidden = token[None, :] > position[:, None]
            if case["window"]:
                hidden |= token[None, :] <= position[:, None] - case["window"]
            a = part.permute(1, 2, 0, 3).reshape(kv, group * n, dim)
            scores = torch.matmul(a, k.permute(1, 2, 0)).view(kv, group, n, length) / math.sqrt(dim)
            scores.masked_fill_(hidden, -math.inf)
            p = torch.exp(scores - scores.amax(3, keepdim=True))
            y = torch.matmul(p.view(kv, group * n, length), v.transpose(0, 1)).view(kv, group, n, dim) / p.sum(3, keepdim=True)
            out[start + first:start + first + n] = y.permute(2, 0, 1, 3).reshape(n, -1).to(s["dtype"])
        start += new
    return out


# ---------------------------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------------------------
def work(case):
    es = 4 if case["storage"] == "f32" else 2
    if case["op"] == "rotary":
        values = case["rows"] * case["heads"]
        return {"bytes": 2 * es * values * case["dim"] + 4 * case["rows"], "flops": 3 * values * case["rotary"]}
    kv, dim, rows = case["kv"], case["dim"], _rows(case)
    token = 2 * kv * (dim + 4 if case["format"] == "i8" else dim * es)  # K and V of a token as held
    total = flops = 0
    if case["op"] != "attend":  # k and v in, into the pages, and as read back
        total += 2 * 2 * rows * kv * dim * es + 2 * rows * token
        flops += 3 * rows * kv * (case["rotary"] + 2 * dim)
    if case["op"] != "cache":
        tokens, pairs = _seen(case)
        total += tokens * token + 2 * rows * kv * case["group"] * dim * es
        flops += 4 * pairs * kv * case["group"] * dim
    return {"bytes": total, "flops": flops}


# ---------------------------------------------------------------------------------------------
# the definition in 64 bits
# ---------------------------------------------------------------------------------------------
def exact(case, seed):
    s = _inputs(case, seed)
    dim, dtype = case["dim"], s["dtype"]

    def turned(x, positions, heads):
        """Pairs as complex numbers, times e^(i angle)."""
        x = x.double().unflatten(1, (heads, dim))
        n = case["rotary"]
        pairs = x[..., :n].unflatten(2, (n // 2, 2)) if case["interleaved"] else x[..., :n].unflatten(2, (2, n // 2)).transpose(2, 3)
        f = torch.tensor(_frequencies(case), dtype=torch.float64, device="cuda")
        angle = torch.outer(positions.double(), f)[:, None]
        z = torch.view_as_real(torch.view_as_complex(pairs.contiguous()) * torch.polar(torch.ones_like(angle), angle))
        z = z.flatten(2) if case["interleaved"] else z.transpose(2, 3).flatten(2)
        return torch.cat([z, x[..., n:]], 2)

    def held(x):
        """What the cache holds of values [tokens, heads, dim]."""
        if case["format"] != "i8":
            return x
        x = x.float().double()
        top = torch.linalg.vector_norm(x, ord=math.inf, dim=2, keepdim=True)
        q = torch.round(torch.nan_to_num(x * 127 / top))
        return q * (top.float() / 127).double()

    if case["op"] == "rotary":
        return {"y": turned(s["x"], s["positions"], case["heads"]).flatten(1)}
    kv, lengths = case["kv"], _lengths(case)
    ends, out = s["starts"].tolist(), {}
    position = torch.cat([torch.arange(length - new, length, device="cuda") for length, new in lengths])
    q = s.get("q")
    if "k" in s:
        k, v = held(turned(s["k"], position, kv)), held(s["v"].double().unflatten(1, (kv, dim)))
        out["k"], out["v"] = k.flatten(1), v.flatten(1)
        if q is not None:
            q = turned(q, position, kv * case["group"]).flatten(1).to(dtype)
    if q is None:
        return out
    if work(case)["flops"] > 1.5e12:
        return None
    group, at, ys = case["group"], 0, []
    for i, (length, new) in enumerate(lengths):
        ctx = []
        for name in ("k", "v"):
            t = held(s["old_" + name][at:at + length].double().unflatten(1, (kv, dim)))
            if name in s:
                mine = (k if name == "k" else v)[ends[i]:ends[i + 1]]
                t[length - new:] = mine if case["format"] == "i8" else mine.to(dtype).double()
            ctx.append(t)
        at += length
        mine = q[ends[i]:ends[i + 1]].double().unflatten(1, (kv, group, dim))
        y = torch.empty_like(mine)
        for h in range(kv):
            for first in range(0, new, 512):
                part = mine[first:first + 512, h]
                where = torch.arange(length - new + first, length - new + first + part.shape[0], device="cuda")[:, None]
                token = torch.arange(length, device="cuda")[None]
                sees = (token <= where) & (token > where - (case["window"] or length))
                w = torch.mm(part.flatten(0, 1), ctx[0][:, h].T).div_(math.sqrt(dim)).unflatten(0, part.shape[:2])
                w = torch.softmax(torch.where(sees[:, None], w, -math.inf), 2)
                y[first:first + 512, h] = torch.mm(w.flatten(0, 1), ctx[1][:, h]).unflatten(0, part.shape[:2])
        ys.append(y.flatten(1))
    out["y"] = torch.cat(ys)
    return out
