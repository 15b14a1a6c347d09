"""Workloads of the serving operators: root-mean-square norm with the residual's addition, products with
4-bit weights, and sampling - the steps a served model ends with.

``run`` computes an operator in its plain form (elementary torch operations), or, where ``own`` is true,
through the library's entry points.  ``exact`` computes the same from the definition in 64 bits.
"""
import torch

own = False

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
CODES = {"f32": 0, "f16": 1, "bf16": 2, "i8": 3}     # DN_F32, DN_F16, DN_BF16, DN_I8
ACTIVATIONS = {"linear": 3, "relu": 1, "leaky": 7}   # DN_LINEAR, DN_RELU, DN_LEAKY
EPS = 1e-5


def listed():
    return [
        # one token's hidden state: nothing but latency
        {"name": "norm_token", "op": "norm", "rows": 1, "n": 4096, "type": "f32", "add": True, "q8": False, "group": 0},
        # a small batch at an odd width, 8 bits with one scale a row
        {"name": "norm_ragged_q8", "op": "norm", "rows": 37, "n": 5003, "type": "f16", "add": True, "q8": True, "group": 0},
        # a prompt in front of a quantised product: 8 bits with a scale for each 128 values
        {"name": "norm_prompt_q8", "op": "norm", "rows": 4096, "n": 8192, "type": "bf16", "add": True, "q8": True, "group": 128},
        # a long prompt in the library's own type
        {"name": "norm_prompt", "op": "norm", "rows": 16384, "n": 4096, "type": "f32", "add": True, "q8": False, "group": 0},
        # one token through a square layer
        {"name": "q4_token", "op": "q4", "batch": 1, "inputs": 4096, "outputs": 4096, "group": 128, "type": "f32", "out": "f32", "act": "linear", "bias": False},
        # the connected layer of the 7x7 detection network, one image
        {"name": "q4_connected", "op": "q4", "batch": 1, "inputs": 12544, "outputs": 1715, "group": 32, "type": "f32", "out": "f32", "act": "leaky", "bias": True},
        # a few tokens, ragged in every dimension
        {"name": "q4_ragged", "op": "q4", "batch": 3, "inputs": 5003, "outputs": 1470, "group": 64, "type": "f16", "out": "f16", "act": "relu", "bias": True},
        # a batch of tokens whose activations come in 8 bits from the norm
        {"name": "q4_batch_q8", "op": "q4", "batch": 16, "inputs": 8192, "outputs": 8192, "group": 128, "type": "i8", "out": "bf16", "act": "linear", "bias": False},
        # the output projection of a batch
        {"name": "q4_head", "op": "q4", "batch": 64, "inputs": 4096, "outputs": 131072, "group": 128, "type": "bf16", "out": "f32", "act": "linear", "bias": False},
        # one user's next token
        {"name": "sample_token", "op": "sample", "rows": 1, "n": 32768, "type": "f32", "mode": "kp", "masked": 0.0},
        # a few users, an odd vocabulary, nucleus sampling, some tokens forbidden
        {"name": "sample_ragged", "op": "sample", "rows": 7, "n": 50021, "type": "bf16", "mode": "p", "masked": 0.1},
        # a batch of users, each with settings of their own
        {"name": "sample_batch", "op": "sample", "rows": 64, "n": 131072, "type": "f32", "mode": "mixed", "masked": 0.01},
    ]


def _spread(rng, lo, hi):
    """A whole number between lo and hi, spread evenly over its logarithm."""
    return max(lo, min(hi, int(round(lo * (hi / lo) ** rng.random()))))


def _width(rng, lo, hi):
    """A width: half of them multiples of 128, the others whatever comes."""
    v = _spread(rng, lo, hi)
    return max(128, v // 128 * 128) if rng.random() < 0.5 else v


def draw(rng):
    op = rng.choice(["norm", "q4", "sample"])
    if op == "norm":
        n = _width(rng, 64, 16384)
        rows = _spread(rng, 1, max(1, min(16384, (1 << 25) // n)))
        q8 = rng.random() < 0.5
        return {"op": op, "rows": rows, "n": n, "type": rng.choice(["f32", "f16", "bf16"]), "add": rng.random() < 0.75,
                "q8": q8, "group": rng.choice([0, 32, 64, 128]) if q8 else 0}
    if op == "q4":
        inputs, outputs, batch = _width(rng, 128, 25088), _width(rng, 64, 65536), _spread(rng, 1, 64)
        outputs = max(64, min(outputs, (1 << 28) // inputs))
        return {"op": op, "batch": batch, "inputs": inputs, "outputs": outputs, "group": rng.choice([32, 64, 128]),
                "type": rng.choice(["f32", "f16", "bf16", "i8"]), "out": rng.choice(["f32", "f16", "bf16"]),
                "act": rng.choice(["linear", "relu", "leaky"]), "bias": rng.random() < 0.5}
    n = _width(rng, 1000, 262144)
    rows = _spread(rng, 1, max(1, min(256, (1 << 23) // n)))
    return {"op": op, "rows": rows, "n": n, "type": rng.choice(["f32", "f16", "bf16"]),
            "mode": rng.choice(["k", "p", "kp", "min", "all", "mixed"]), "masked": rng.choice([0.0, 0.01, 0.5])}


# ---- inputs -----------------------------------------------------------------------------------
def _groups(n, group):
    return 1 if group == 0 else -(-n // group)


def _prepare_norm(c, g):
    t, dev, shape = TYPES[c["type"]], "cuda", (c["rows"], c["n"])
    # a hidden state: a few columns are far larger than the rest
    columns = 1 + 20 * (torch.rand(c["n"], generator=g, device=dev) < 0.002).float()
    s = {"x": (torch.randn(shape, generator=g, device=dev) * 0.5).to(t),
         "add": (torch.randn(shape, generator=g, device=dev) * columns).to(t) if c["add"] else None,
         "scales": 1 + 0.1 * torch.randn(c["n"], generator=g, device=dev)}
    s["sum"] = torch.empty(shape, dtype=t, device=dev) if c["add"] else None
    if c["q8"]:
        s["q"] = torch.empty(shape, dtype=torch.int8, device=dev)
        s["q_scales"] = torch.empty(c["rows"], _groups(c["n"], c["group"]), device=dev)
    else:
        s["out"] = torch.empty(shape, dtype=t, device=dev)
    return s


def _prepare_q4(c, g):
    dev, n, k = "cuda", c["outputs"], c["inputs"]
    groups = _groups(k, c["group"])
    # codes of normally distributed weights, two to a byte, the lower half first; a scale and a zero for each group
    even = (torch.randn(n, (k + 1) // 2, generator=g, device=dev) * 2.6 + 7.5).round_().clamp_(0, 15).to(torch.uint8)
    odd = (torch.randn(n, (k + 1) // 2, generator=g, device=dev) * 2.6 + 7.5).round_().clamp_(0, 15).to(torch.uint8)
    s = {"codes": even | (odd << 4),
         "w_scales": (0.5 + torch.rand(n, groups, generator=g, device=dev)) * (0.4 / k ** 0.5),
         "zeros": torch.randint(6, 10, (n, groups), generator=g, device=dev, dtype=torch.uint8),
         "bias": 0.1 * torch.randn(n, generator=g, device=dev) if c["bias"] else None,
         "x_scales": None}
    if c["type"] == "i8":
        # 8-bit activations with a scale for each group, as the norm writes them
        s["x"] = (torch.randn(c["batch"], k, generator=g, device=dev) * 40).round_().clamp_(-127, 127).to(torch.int8)
        s["x_scales"] = (0.5 + torch.rand(c["batch"], groups, generator=g, device=dev)) / 40
    else:
        columns = 1 + 10 * (torch.rand(k, generator=g, device=dev) < 0.002).float()
        s["x"] = (torch.randn(c["batch"], k, generator=g, device=dev) * columns).to(TYPES[c["type"]])
    s["out"] = torch.empty(c["batch"], n, dtype=TYPES[c["out"]], device=dev)
    return s


def _prepare_sample(c, g):
    dev, rows, n = "cuda", c["rows"], c["n"]
    # most of the vocabulary is unlikely, a few tokens stand out; some are forbidden
    logits = torch.randn(rows, n, generator=g, device=dev) * 2.5
    # (24 places in each row, no place twice: which of two values a scatter leaves there is not determined)
    top = (torch.randint(0, n, (rows, 1), generator=g, device=dev) + torch.arange(24, device=dev) * (n // 24)) % n
    logits.scatter_(1, top, 6 + 8 * torch.rand(rows, 24, generator=g, device=dev))
    logits[torch.rand(rows, n, generator=g, device=dev) < c["masked"]] = float("-inf")
    u = torch.rand(rows, 6, generator=g, device=dev)
    mode = c["mode"]
    s = {"logits": logits.to(TYPES[c["type"]]), "uniform": u[:, 0].contiguous(), "temperature": 0.5 + u[:, 1],
         "top_k": (8 + 56 * u[:, 2]).int() if mode in ("k", "kp", "mixed") else None,
         "top_p": 0.7 + 0.29 * u[:, 3] if mode in ("p", "kp", "mixed") else None,
         "min_p": 0.02 + 0.1 * u[:, 4] if mode in ("min", "mixed") else None}
    if mode == "mixed":  # each user turns some of the settings off
        s["top_k"][u[:, 5] < 0.4] = 0
        s["top_p"][u[:, 5] > 0.7] = 1.0
        s["min_p"][(u[:, 5] > 0.2) & (u[:, 5] < 0.8)] = 0.0
    s["tokens"] = torch.empty(rows, dtype=torch.int32, device=dev)
    s["probs"] = torch.empty(rows, device=dev)
    return s


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed))
    s = {"norm": _prepare_norm, "q4": _prepare_q4, "sample": _prepare_sample}[case["op"]](case, g)
    s["case"] = dict(case)
    if own:
        _own_prepare(s, case)
    return s


# ---- plain forms ------------------------------------------------------------------------------
def _activate(y, act):
    if act == "relu":
        return y.clamp_min(0)
    return torch.where(y > 0, y, 0.1 * y) if act == "leaky" else y


def _plain_norm(s, c):
    x = s["x"]
    if c["add"]:
        x = (x.float() + s["add"].float()).to(x.dtype)
    if not c["q8"]:
        v = x.float()
        y = (v * (v.square().mean(1, keepdim=True) + EPS).rsqrt() * s["scales"]).to(x.dtype)
        return {"sum": x, "out": y} if c["add"] else {"out": y}
    # the 8-bit values are next to a border between two steps now and then: 64 bits
    v = x.double()
    y = v / (v.square().mean(1, keepdim=True) + EPS).sqrt() * s["scales"].double()
    group = c["group"] or c["n"]
    y = torch.nn.functional.pad(y, (0, -c["n"] % group)).view(c["rows"], -1, group)
    scale = (y.abs().amax(2, keepdim=True) / 127).float()
    q = (y / scale.double()).nan_to_num(0.0).round().clamp(-127, 127).float() * scale
    out = {"values": q.reshape(c["rows"], -1)[:, :c["n"]], "scales": scale[:, :, 0]}
    return {"sum": x, **out} if c["add"] else out


def _plain_q4(s, c):
    k, group = c["inputs"], c["group"]
    codes = torch.stack((s["codes"] & 15, s["codes"] >> 4), 2).flatten(1)[:, :k].float()
    w = (codes - s["zeros"].float().repeat_interleave(group, 1)[:, :k]) * s["w_scales"].repeat_interleave(group, 1)[:, :k]
    x = s["x"].float()
    if c["type"] == "i8":
        x = x * s["x_scales"].repeat_interleave(group, 1)[:, :k]
    y = x @ w.t()
    if c["bias"]:
        y = y + s["bias"]
    return {"out": _activate(y, c["act"]).to(TYPES[c["out"]])}


def _plain_sample(s, c):
    logits, n = s["logits"].double(), c["n"]
    order = torch.sort(logits, dim=1, descending=True, stable=True)
    place = torch.arange(n, device=logits.device)
    w = torch.exp((order.values - order.values[:, :1]) / s["temperature"].double()[:, None])
    keep = torch.isfinite(order.values)
    if s["top_k"] is not None:
        k = s["top_k"].long()[:, None]
        keep = keep & ((place < k) | (k <= 0))
    if s["top_p"] is not None:
        p = s["top_p"].double()[:, None]
        mass = (w * keep).cumsum(1)
        keep = keep & ((mass - w * keep < p * mass[:, -1:]) | (p >= 1) | (place == 0))
    if s["min_p"] is not None:
        keep = keep & (w >= s["min_p"].double()[:, None])
    mass = torch.zeros_like(w).scatter_(1, order.indices, w * keep)
    running = mass.cumsum(1)
    total = running[:, -1:]
    token = ((running >= s["uniform"].double()[:, None] * total) & (mass > 0)).int().argmax(1)
    return {"tokens": token.int(), "probs": (mass.gather(1, token[:, None]) / total)[:, 0].float()}


# ---- the library's entry points -----------------------------------------------------------------
def _own_prepare(s, c):
    from darknet_amd import lib
    L = s["lib"] = lib.load()
    L.hip_set_stream(torch.cuda.current_stream().cuda_stream)
    p = {k: (v.data_ptr() if isinstance(v, torch.Tensor) else None) for k, v in s.items()}
    if c["op"] == "norm":
        s["args"] = (p["x"], p["add"], p["scales"], p["sum"], p.get("out"), p.get("q"), p.get("q_scales"),
                     CODES[c["type"]], c["rows"], c["n"], c["group"], EPS)
        return
    if c["op"] == "q4":
        # the weights are laid out once, as a program does when it loads them
        s["packed"] = torch.empty(L.q4_packed_bytes(c["inputs"], c["outputs"], c["group"]), dtype=torch.uint8, device="cuda")
        L.q4_pack_codes_gpu(p["codes"], p["w_scales"], p["zeros"], s["packed"].data_ptr(), c["inputs"], c["outputs"], c["group"])
        size = L.connected_q4_workspace_bytes(CODES[c["type"]], c["batch"], c["inputs"], c["outputs"], c["group"])
        s["workspace"] = torch.empty(max(size, 1), dtype=torch.uint8, device="cuda")
        s["args"] = (p["x"], CODES[c["type"]], p["x_scales"], c["group"], s["packed"].data_ptr(), p["bias"], p["out"],
                     CODES[c["out"]], c["batch"], c["inputs"], c["outputs"], c["group"], ACTIVATIONS[c["act"]],
                     s["workspace"].data_ptr())
        return
    size = L.sample_workspace_bytes(c["rows"], c["n"])
    s["workspace"] = torch.empty(max(size, 1), dtype=torch.uint8, device="cuda")
    s["args"] = (p["logits"], CODES[c["type"]], c["rows"], c["n"], c["n"], p["temperature"], p["top_k"], p["top_p"],
                 p["min_p"], p["uniform"], p["tokens"], p["probs"], s["workspace"].data_ptr())


def _own_run(s, c):
    L = s["lib"]
    if c["op"] == "norm":
        L.forward_rmsnorm_gpu(*s["args"])
        out = {"sum": s["sum"]} if c["add"] else {}
        if not c["q8"]:
            return {**out, "out": s["out"]}
        rows, n, group = c["rows"], c["n"], c["group"] or c["n"]
        if n % group == 0:
            values = (s["q"].view(rows, -1, group) * s["q_scales"][:, :, None]).view(rows, n)
        else:
            values = s["q"] * s["q_scales"].repeat_interleave(group, 1)[:, :n]
        return {**out, "values": values, "scales": s["q_scales"]}
    if c["op"] == "q4":
        L.forward_connected_q4_gpu(*s["args"])
        return {"out": s["out"]}
    L.sample_rows_gpu(*s["args"])
    return {"tokens": s["tokens"], "probs": s["probs"]}


def run(state):
    c = state["case"]
    if own:
        return _own_run(state, c)
    return {"norm": _plain_norm, "q4": _plain_q4, "sample": _plain_sample}[c["op"]](state, c)


# ---- least work -----------------------------------------------------------------------------------
def work(case):
    c, size = case, {"f32": 4, "f16": 2, "bf16": 2, "i8": 1}
    if c["op"] == "norm":
        e, t = c["rows"] * c["n"], size[c["type"]]
        read = e * t * (2 if c["add"] else 1) + 4 * c["n"]
        # 8 bits are returned as the values they stand for: 4 bytes an element
        write = e * t * (1 if c["add"] else 0) + (4 * e + 4 * c["rows"] * _groups(c["n"], c["group"]) if c["q8"] else e * t)
        return {"bytes": read + write, "flops": 5 * e}
    if c["op"] == "q4":
        groups = _groups(c["inputs"], c["group"])
        weights = c["outputs"] * ((c["inputs"] + 1) // 2 + 5 * groups)
        x = c["batch"] * (c["inputs"] * size[c["type"]] + (4 * groups if c["type"] == "i8" else 0))
        return {"bytes": weights + x + c["batch"] * c["outputs"] * size[c["out"]] + (4 * c["outputs"] if c["bias"] else 0),
                "flops": 2 * c["batch"] * c["inputs"] * c["outputs"]}
    e = c["rows"] * c["n"]
    return {"bytes": e * size[c["type"]] + 28 * c["rows"], "flops": 3 * e}


# ---- the definitions in 64 bits -------------------------------------------------------------------
def _exact_norm(s, c):
    x = s["x"]
    # the sum is an output of the input's type: what follows is the norm of what was stored
    stored = torch.add(x.float(), s["add"].float()).to(x.dtype) if c["add"] else x
    h = stored.to(torch.float64)
    rms = torch.sqrt(torch.linalg.vecdot(h, h) / c["n"] + EPS)
    y = s["scales"].to(torch.float64) * (h / rms[:, None])
    out = {"sum": stored.to(torch.float64)} if c["add"] else {}
    if not c["q8"]:
        return {**out, "out": y}
    group = c["group"] or c["n"]
    index = torch.arange(c["n"], device=y.device) // group
    top = torch.zeros(c["rows"], _groups(c["n"], c["group"]), dtype=torch.float64, device=y.device)
    top.scatter_reduce_(1, index.expand(c["rows"], -1), y.abs(), "amax")
    step = (top / 127).to(torch.float32).to(torch.float64)  # the step is held in 32 bits
    wide = step[:, index]
    steps = torch.where(wide > 0, torch.round(y / wide.clamp_min(1e-300)), torch.zeros_like(y))
    return {**out, "values": steps.clamp(-127, 127) * wide, "scales": top / 127}


def _exact_q4(s, c):
    k, group, x = c["inputs"], c["group"], s["x"].to(torch.float64)
    index = torch.arange(k, device="cuda")
    if c["type"] == "i8":
        x = x * s["x_scales"].to(torch.float64)[:, index // group]
    parts = []
    for lo in range(0, c["outputs"], 8192):
        rows = slice(lo, lo + 8192)
        code = (s["codes"][rows][:, index // 2] >> (4 * (index % 2)).to(torch.uint8)) & 15
        w = code.to(torch.float64)
        w -= s["zeros"][rows].to(torch.float64)[:, index // group]
        w *= s["w_scales"][rows].to(torch.float64)[:, index // group]
        parts.append(torch.mm(w, x.t().contiguous()).t())
    y = torch.cat(parts, 1)
    if c["bias"]:
        y = y + s["bias"].to(torch.float64)
    if c["act"] == "relu":
        y = torch.relu(y)
    elif c["act"] == "leaky":
        y = torch.maximum(y, 0.1 * y)
    return {"out": y}


def _exact_sample(s, c):
    import numpy as np
    host = {k: v.cpu().double().numpy() for k, v in s.items() if isinstance(v, torch.Tensor) and k not in ("tokens", "probs")}
    tokens, probs = [], []
    for r in range(c["rows"]):
        row = host["logits"][r]
        order = np.lexsort((np.arange(c["n"]), -row))
        order = order[row[order] > -np.inf]
        w = np.exp((row[order] - row[order[0]]) / host["temperature"][r])
        if s["top_k"] is not None and host["top_k"][r] > 0:
            w = w[:int(host["top_k"][r])]
        if s["top_p"] is not None and host["top_p"][r] < 1:
            w = w[:int(np.searchsorted(np.cumsum(w), host["top_p"][r] * w.sum())) + 1]
        if s["min_p"] is not None:
            w = w[w >= host["min_p"][r]]
        kept = np.argsort(order[:len(w)])
        running = np.cumsum(w[kept])
        at = kept[min(int(np.searchsorted(running, host["uniform"][r] * running[-1])), len(w) - 1)]
        tokens.append(int(order[at]))
        probs.append(float(w[at] / running[-1]))
    return {"tokens": np.array(tokens, np.int32), "probs": np.array(probs)}


def exact(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed))
    s = {"norm": _prepare_norm, "q4": _prepare_q4, "sample": _prepare_sample}[case["op"]](case, g)
    return {"norm": _exact_norm, "q4": _exact_q4, "sample": _exact_sample}[case["op"]](s, case)
