"""Performance cases of the 8-bit transformer operators: the product in 8-bit integers with a scale for each token
and each output channel (HipQuantLinear), and the norms around a transformer block with its gate and residual scale
(HipBlockNorm), which hand the next product its 8-bit rows.

A case's "op":
  linear  y = act((q . wq) * row scale * channel scale + bias (+ residual)) over floating rows x, which are brought
          to 8 bits on the way: q = round(127 x / max|x| of the row), row scale = max|x| / 127.
  norm    h = res_scale * residual + act(gate) * scale * post_norm(x), y = pre_norm(h).
  block   the norm's y as 8-bit rows and their scales, and the product that reads them: h and that product's y.

The inputs are activations as a transformer holds them: normal, with a few channels an order of magnitude larger.
"""
import math

import torch

own = False

DTYPES = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}


def listed():
    return [
        # one token through a square projection: the smallest call, where latency counts
        {"name": "linear one token f16", "op": "linear", "storage": "f16", "rows": 1, "k": 768, "n": 768, "act": "none",
         "bias": True, "residual": True, "pad": 0},
        # a few tokens through a wide layer: bound by streaming the weights
        {"name": "linear 7 tokens bf16", "op": "linear", "storage": "bf16", "rows": 7, "k": 4096, "n": 4096,
         "act": "swish", "bias": False, "residual": False, "pad": 0},
        # the text recognizer's MLP over a full batch of lines: 32 x 80 tokens of 192 channels
        {"name": "linear lines gelu f16", "op": "linear", "storage": "f16", "rows": 2560, "k": 192, "n": 768,
         "act": "gelu", "bias": True, "residual": False, "pad": 0},
        # a short ragged batch (6 x 131 tokens), an output width that fills no tile, rows inside a wider buffer
        {"name": "linear ragged bf16", "op": "linear", "storage": "bf16", "rows": 786, "k": 768, "n": 760, "act": "none",
         "bias": True, "residual": True, "pad": 24},
        # full precision outside the product, an odd inner size
        {"name": "linear odd f32", "op": "linear", "storage": "f32", "rows": 333, "k": 577, "n": 301, "act": "relu",
         "bias": True, "residual": False, "pad": 3},
        # a full batch of token sequences, 16 x 512, through the query / key / value projection
        {"name": "linear sequences f16", "op": "linear", "storage": "f16", "rows": 8192, "k": 768, "n": 2304,
         "act": "none", "bias": True, "residual": False, "pad": 0},
        # a long prompt through a wide layer: bound by the matrix cores, the largest case
        {"name": "linear large bf16", "op": "linear", "storage": "bf16", "rows": 4096, "k": 4096, "n": 8192,
         "act": "none", "bias": False, "residual": False, "pad": 0},
        # one token: the smallest norm
        {"name": "norm one token f16", "op": "norm", "storage": "f16", "rows": 1, "channels": 768, "post": "rms",
         "pre": "rms", "gate": "none", "gate_act": "none", "pad": 0},
        # the recognizer's residual Add and LayerNorm over a full batch of lines
        {"name": "norm lines f16", "op": "norm", "storage": "f16", "rows": 2560, "channels": 192, "post": "none",
         "pre": "layer", "gate": "none", "gate_act": "none", "pad": 0},
        # full precision, odd sizes, a gate of its own for every token
        {"name": "norm odd f32", "op": "norm", "storage": "f32", "rows": 1001, "channels": 1111, "post": "layer",
         "pre": "layer", "gate": "row", "gate_act": "sigmoid", "pad": 5},
        # wide rows past every cache, one gate for each of 16 sequences
        {"name": "norm large bf16", "op": "norm", "storage": "bf16", "rows": 16384, "channels": 4096, "post": "rms",
         "pre": "rms", "gate": "sequence", "gate_act": "none", "pad": 0},
        # the end of an attention block and the MLP's first product over 16 x 512 tokens
        {"name": "block sequences bf16", "op": "block", "storage": "bf16", "rows": 8192, "channels": 768, "post": "rms",
         "pre": "rms", "gate": "sequence", "gate_act": "none", "pad": 0, "n": 2048, "act": "gelu", "bias": True},
    ]


# ---------------------------------------------------------------------------------------------
# drawn cases
# ---------------------------------------------------------------------------------------------
def _log(rng, lo, hi):
    """An integer of [lo, hi], spread evenly over its logarithm."""
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def _width(rng, lo, hi):
    """A channel count: mostly multiples of 8 as networks have them, sometimes any number."""
    c = _log(rng, lo, hi)
    return c if rng.random() < 0.25 else max(8, c // 8 * 8)


def draw(rng):
    op = rng.choice(["linear", "linear", "linear", "norm", "norm", "block"])
    storage = rng.choice(["f16", "f16", "bf16", "bf16", "f32"])
    pad = rng.choice([0, 0, 0, rng.randint(1, 64)])
    if op == "linear":
        rows, k, n = _log(rng, 1, 8192), _width(rng, 32, 8192), _width(rng, 16, 8192)
        while 2.0 * rows * k * n > 2.7e11:
            rows = max(1, rows * 2 // 3)
        return {"op": op, "storage": storage, "rows": rows, "k": k, "n": n,
                "act": rng.choice(["none", "none", "gelu", "relu", "swish"]), "bias": rng.random() < 0.6,
                "residual": rng.random() < 0.4, "pad": pad}
    rows, channels = _log(rng, 1, 16384), _width(rng, 32, 8192)
    limit = 6.0e7 if op == "norm" else 1.6e7
    while rows * channels * (2 if storage == "f32" else 1) > limit:
        rows = max(1, rows * 2 // 3)
    case = {"op": op, "storage": storage, "rows": rows, "channels": channels,
            "post": rng.choice(["none", "rms", "layer"]), "pre": rng.choice(["rms", "layer"]),
            "gate": rng.choice(["none", "one", "row", "sequence"]), "gate_act": rng.choice(["none", "sigmoid", "swish"]),
            "pad": pad}
    if op == "block":
        # no full precision: 8-bit rows of computed values turn where one lies next to a half, which 32-bit outputs show
        case["storage"] = "f16" if storage == "f32" else storage
        n = _width(rng, 16, 4096)
        while 2.0 * rows * channels * n > 1.0e11:
            n = max(16, n // 2)
        case.update(n=n, act=rng.choice(["none", "gelu", "relu"]), bias=rng.random() < 0.6)
    return case


# ---------------------------------------------------------------------------------------------
# state
# ---------------------------------------------------------------------------------------------
def _sequences(case):
    """How many gate rows a case has, each shared by rows / that many consecutive rows."""
    if case["gate"] == "none":
        return 0
    if case["gate"] == "sequence":
        return next(s for s in (16, 8, 4, 3, 2, 1) if case["rows"] % s == 0)
    return case["rows"] if case["gate"] == "row" else 1


def _tensor(g, rows, cols, pad, dtype, spread=True):
    """[rows, cols] inside rows of cols + pad values: N(0, 1), every 61st channel 12 times as large."""
    t = torch.randn((rows, cols + pad), generator=g, device="cuda", dtype=torch.float32)
    if spread:
        t[:, ::61] *= 12.0
    return t.to(dtype)[:, :cols]


def _vector(g, n, around, by):
    return around + by * torch.randn((n,), generator=g, device="cuda", dtype=torch.float32)


def _weights(g, state, k, n, bias):
    """8-bit weights [k, n] with a scale for each column, and the float copy that the plain form multiplies."""
    w = torch.randn((k, n), generator=g, device="cuda", dtype=torch.float32) / math.sqrt(k)
    top = w.abs().amax(0)
    state["wf"] = torch.round(w / (top / 127)).clamp_(-127, 127)
    state["ws"] = top / 127
    state["bias"] = _vector(g, n, 0.0, 0.1) if bias else None


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    rows, pad, dtype = case["rows"], case["pad"], DTYPES[case["storage"]]
    state = {"case": case, "seed": seed}
    if case["op"] == "linear":
        state["x"] = _tensor(g, rows, case["k"], pad, dtype)
        state["residual"] = _tensor(g, rows, case["n"], pad, dtype, False) if case["residual"] else None
        _weights(g, state, case["k"], case["n"], case["bias"])
    else:
        c = case["channels"]
        state["x"] = _tensor(g, rows, c, pad, dtype)
        state["residual"] = _tensor(g, rows, c, pad, dtype)
        state["gate"] = None if case["gate"] == "none" else _tensor(g, _sequences(case), c, pad, dtype, False)
        for norm in ("post", "pre"):
            state[norm + "_gamma"] = None if case[norm] == "none" else _vector(g, c, 1.0, 0.1)
            state[norm + "_beta"] = _vector(g, c, 0.0, 0.1) if case[norm] == "layer" else None
        state["scale"] = _vector(g, c, 0.5, 0.1)
        state["res_scale"] = 1.0 if seed % 2 else 0.75
        if case["op"] == "block":
            _weights(g, state, c, case["n"], case["bias"])
    if own:
        _handles(state)
    return state


def _host(t):
    return None if t is None else t.cpu().numpy()


def _handles(state):
    """What a program keeps of the framework: the layers with their parameters, and the buffers they write."""
    from simdonnx_amd.backend import HipBackend, HipBlockNorm, HipQuantLinear
    case, hip = state["case"], HipBackend.default()
    rows, pad, dtype = case["rows"], case["pad"], DTYPES[case["storage"]]
    if "wf" in state:
        k, n = state["wf"].shape
        lin = HipQuantLinear(hip, state["wf"].to(torch.int8).cpu().numpy(), _host(state["bias"]), k, n,
                             scales=_host(state["ws"]))
        state["linear"] = lin
        state["y"] = torch.zeros((rows, n + pad), device="cuda", dtype=dtype)[:, :n]
    if case["op"] == "linear":
        state["work"] = torch.empty(max(1, lin.workspace(rows)), device="cuda", dtype=torch.uint8)
        return
    c = case["channels"]
    state["norm"] = HipBlockNorm(hip, c, post=case["post"], pre=case["pre"], post_gamma=_host(state["post_gamma"]),
                                 post_beta=_host(state["post_beta"]), pre_gamma=_host(state["pre_gamma"]),
                                 pre_beta=_host(state["pre_beta"]), scale=_host(state["scale"]),
                                 res_scale=state["res_scale"], gate_act=case["gate_act"], post_eps=1e-5, pre_eps=1e-6)
    state["h"] = torch.zeros((rows, c + pad), device="cuda", dtype=dtype)[:, :c]
    if case["op"] == "norm":
        state["y"] = torch.zeros((rows, c + pad), device="cuda", dtype=dtype)[:, :c]
    else:
        state["q"] = torch.zeros((rows, lin.pitch), device="cuda", dtype=torch.int8)
        state["qs"] = torch.zeros((rows,), device="cuda", dtype=torch.float32)


# ---------------------------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------------------------
def run(state):
    case = state["case"]
    if own:
        return _run_own(state)
    if case["op"] == "linear":
        return {"y": _plain_linear(state, *_plain_rows(state["x"]))}
    h, y = _plain_norm(state)
    dtype = state["x"].dtype
    if case["op"] == "norm":
        return {"h": h.to(dtype), "y": y.to(dtype)}
    return {"h": h.to(dtype), "y": _plain_linear(state, *_plain_rows(y))}


def _run_own(state):
    case, stream = state["case"], torch.cuda.current_stream().cuda_stream
    st, x, y, res = case["storage"], state["x"], state.get("y"), state["residual"]
    if case["op"] == "linear":
        state["linear"].run(x.data_ptr(), case["rows"], y.data_ptr(), st, x.stride(0), y.stride(0), act=case["act"],
                            residual=None if res is None else res.data_ptr(), ldr=0 if res is None else res.stride(0),
                            workspace=state["work"].data_ptr(), workspace_bytes=state["work"].numel(), stream=stream)
        return {"y": y}
    h, gate = state["h"], state["gate"]
    given = dict(x=x.data_ptr(), ldx=x.stride(0), gate=None if gate is None else gate.data_ptr(),
                 ldg=0 if gate is None else gate.stride(0), gate_rows=0 if gate is None else gate.shape[0],
                 h=h.data_ptr(), ldh=h.stride(0), stream=stream)
    if case["op"] == "norm":
        state["norm"].run(res.data_ptr(), case["rows"], st, res.stride(0), y=y.data_ptr(), ldy=y.stride(0), **given)
        return {"h": h, "y": y}
    q, qs = state["q"], state["qs"]
    state["norm"].run_quantized(res.data_ptr(), case["rows"], q.data_ptr(), qs.data_ptr(), st, res.stride(0),
                                ldq=q.stride(0), **given)
    state["linear"].run_quantized(q.data_ptr(), qs.data_ptr(), case["rows"], y.data_ptr(), st, q.stride(0), y.stride(0),
                                  act=case["act"], stream=stream)
    return {"h": h, "y": y}


# ---- plain forms ----
def _plain_rows(x):
    """(q, row scales): the rows as whole numbers of [-127, 127]. 16-bit values times 127 are exact in 32 bits and
    their quotients lie far enough from the halves; full precision needs 64 bits next to a half."""
    x = x.double() if x.dtype == torch.float32 else x.float()
    top = x.abs().amax(1, keepdim=True)
    q = torch.round(x * 127 / torch.where(top > 0, top, torch.ones_like(top)))
    return q.float(), top.float() / 127


def _plain_linear(state, q, scale):
    """The sums of whole numbers stay below 2^24 at these sizes and values, so 32 bits hold them exactly."""
    v = (q @ state["wf"]) * state["ws"] * scale
    if state["bias"] is not None:
        v = v + state["bias"]
    if state["case"]["op"] == "linear" and state["residual"] is not None:
        v = v + state["residual"].float()
    return _plain_act(v, state["case"]["act"]).to(state["x"].dtype)


def _plain_act(v, act):
    if act == "gelu":
        return 0.5 * v * (1 + torch.erf(v * math.sqrt(0.5)))
    if act == "relu":
        return torch.where(v < 0, torch.zeros_like(v), v)
    if act == "sigmoid":
        return 1 / (1 + torch.exp(-v))
    return v / (1 + torch.exp(-v)) if act == "swish" else v


def _plain_norm_of(v, kind, gamma, beta, eps):
    if kind == "none":
        return v
    if kind == "layer":
        v = v - v.mean(1, keepdim=True)
    v = v / torch.sqrt((v * v).mean(1, keepdim=True) + eps) * gamma
    return v if beta is None else v + beta


def _plain_norm(state):
    case = state["case"]
    a = _plain_norm_of(state["x"].float(), case["post"], state["post_gamma"], state["post_beta"], 1e-5) * state["scale"]
    if state["gate"] is not None:
        gate = _plain_act(state["gate"].float(), case["gate_act"])
        a = (a.view(gate.shape[0], -1, a.shape[1]) * gate[:, None, :]).view(a.shape)
    h = state["res_scale"] * state["residual"].float() + a
    return h, _plain_norm_of(h, case["pre"], state["pre_gamma"], state["pre_beta"], 1e-6)


# ---------------------------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------------------------
def work(case):
    rows, es = case["rows"], 4 if case["storage"] == "f32" else 2
    if case["op"] == "linear":
        k, n = case["k"], case["n"]
        values = rows * k + rows * n * (2 if case["residual"] else 1)
        return {"bytes": es * values + k * n + 4 * n * (2 if case["bias"] else 1), "flops": 2 * rows * k * n}
    c = case["channels"]
    vectors = 1 + (case["post"] != "none") + (case["post"] == "layer") + 1 + (case["pre"] == "layer")
    total = es * c * (4 * rows + _sequences(case)) + 4 * c * vectors
    flops = rows * c * (4 + (case["post"] != "none") * 4 + 4 + (case["gate"] != "none"))
    if case["op"] == "block":  # x, residual and h, and the product's weights and outputs in the place of y
        n = case["n"]
        total += es * (rows * n - rows * c) + c * n + 4 * n * (2 if case["bias"] else 1)
        flops += 2 * rows * c * n
    return {"bytes": total, "flops": flops}


# ---------------------------------------------------------------------------------------------
# the definition in 64 bits
# ---------------------------------------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    d = {name: t.double() for name, t in s.items() if isinstance(t, torch.Tensor)}
    acts = {"none": lambda v: v, "relu": lambda v: v.clamp_min(0), "sigmoid": torch.sigmoid,
            "swish": lambda v: v * torch.sigmoid(v), "gelu": lambda v: v * torch.special.ndtr(v)}

    def norm(v, which, eps):
        kind = case[which]
        if kind == "none":
            return v
        if kind == "rms":
            return d[which + "_gamma"] * v * torch.rsqrt(v.pow(2).sum(1, keepdim=True) / v.shape[1] + eps)
        var, mean = torch.var_mean(v, dim=1, correction=0, keepdim=True)
        return torch.addcmul(d[which + "_beta"], (v - mean) / (var + eps).sqrt(), d[which + "_gamma"])

    def product(v, residual):
        """Over pieces of the rows: the largest case would hold gigabytes in 64 bits."""
        out = []
        for i in range(0, v.shape[0], 1024):
            part = v[i:i + 1024]
            top = torch.linalg.vector_norm(part, ord=math.inf, dim=1, keepdim=True)
            y = torch.mm(torch.round(torch.nan_to_num(part * 127 / top)), d["wf"]).mul_(top / 127).mul_(d["ws"])
            if "bias" in d:
                y += d["bias"]
            if residual is not None:
                y += residual[i:i + 1024]
            out.append(acts[case["act"]](y))
        return torch.cat(out)

    if case["op"] == "linear":
        return {"y": product(d["x"], d.get("residual"))}
    branch = norm(d["x"], "post", 1e-5) * d["scale"]
    if "gate" in d:
        branch = branch * acts[case["gate_act"]](d["gate"]).repeat_interleave(case["rows"] // d["gate"].shape[0], 0)
    h = torch.add(branch, d["residual"], alpha=s["res_scale"])
    y = norm(h, "pre", 1e-6)
    return {"h": h, "y": y if case["op"] == "norm" else product(y, None)}
