"""The transformer-block operators of mggan.hip.blocks as measured cases: attention over the rows of scenes, the linear layer with
its epilogue and the gated feed-forward layer, each in its plain form (elementary torch operations in 32 bits), as the framework's
call, and in 64 bits from the definition."""
import math
import os
import random
import sys

import torch

own = False

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16}


def listed():
    return [
        # the scenes of one training batch: 64 scenes of 20 pedestrians, heads of the encoder's width, scores that fall with distance
        {"name": "attention_scenes_64x20_train", "op": "attention", "type": "f32", "train": True, "scenes": 64, "rows": 1280, "keys": 1280,
         "ragged": False, "heads": 4, "kv_heads": 4, "width": 32, "causal": False, "prefix": False, "cap": 0.0, "axes": 2},
        # the large batch: 8,192 pedestrians in scenes of uneven size, capped scores, both gradients
        {"name": "attention_scenes_8192_train", "op": "attention", "type": "f32", "train": True, "scenes": 256, "rows": 8192, "keys": 8192,
         "ragged": True, "heads": 4, "kv_heads": 2, "width": 32, "causal": False, "prefix": False, "cap": 20.0, "axes": 2},
        # packed sequences of uneven length with a prefix that every row sees, shared key heads, capped scores
        {"name": "attention_prefix_train", "op": "attention", "type": "bf16", "train": True, "scenes": 11, "rows": 8192, "keys": 8192,
         "ragged": True, "heads": 16, "kv_heads": 4, "width": 64, "causal": True, "prefix": True, "cap": 30.0, "axes": 0},
        # one long sequence read front to back, wide heads, scores that fall with the distance of the positions
        {"name": "attention_long_train", "op": "attention", "type": "bf16", "train": True, "scenes": 1, "rows": 16384, "keys": 16384,
         "ragged": False, "heads": 8, "kv_heads": 8, "width": 128, "causal": True, "prefix": False, "cap": 0.0, "axes": 1},
        # one new row of one sequence: the smallest call
        {"name": "attention_one_token", "op": "attention", "type": "bf16", "train": False, "scenes": 1, "rows": 1, "keys": 1000,
         "ragged": True, "heads": 8, "kv_heads": 2, "width": 64, "causal": True, "prefix": False, "cap": 30.0, "axes": 0},
        # one new row for each of 32 sequences with long caches
        {"name": "attention_tokens_long", "op": "attention", "type": "bf16", "train": False, "scenes": 32, "rows": 32, "keys": 32 * 16384,
         "ragged": True, "heads": 32, "kv_heads": 8, "width": 128, "causal": True, "prefix": False, "cap": 0.0, "axes": 0},
        # the output projection while serving a few rows
        {"name": "linear_tokens", "op": "linear", "type": "bf16", "train": False, "rows": 8, "inputs": 4096, "outputs": 4096,
         "act": "none", "bias": True, "residual": True},
        # classifier rows (pedestrians times samples) at the classifier's width
        {"name": "linear_rows_f32_train", "op": "linear", "type": "f32", "train": True, "rows": 25600, "inputs": 192, "outputs": 192,
         "act": "leaky", "bias": True, "residual": True},
        # a training step's projection with an activation and the residual stream
        {"name": "linear_train", "op": "linear", "type": "bf16", "train": True, "rows": 8192, "inputs": 4096, "outputs": 4096,
         "act": "gelu", "bias": True, "residual": True},
        # the feed-forward layer while serving a few rows
        {"name": "gated_tokens", "op": "gated", "type": "bf16", "train": False, "rows": 3, "inputs": 4096, "outputs": 12288,
         "act": "silu", "bias": False, "residual": False},
        # the feed-forward layer over the pedestrians of the large batch
        {"name": "gated_rows_f32_train", "op": "gated", "type": "f32", "train": True, "rows": 8192, "inputs": 128, "outputs": 512,
         "act": "gelu", "bias": True, "residual": False},
        # a training step's feed-forward layer
        {"name": "gated_train", "op": "gated", "type": "bf16", "train": True, "rows": 8192, "inputs": 4096, "outputs": 8192,
         "act": "silu", "bias": False, "residual": False},
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    kind = rng.choice(["scenes", "sequences", "sequences", "tokens", "linear", "linear", "linear_tokens", "gated", "gated", "gated_tokens"])
    if kind == "scenes":
        scenes = _log(rng, 4, 256)
        rows = scenes + _log(rng, scenes, scenes * 31)
        kv = rng.choice([1, 2, 4])
        return {"op": "attention", "type": "f32", "train": True, "scenes": scenes, "rows": rows, "keys": rows, "ragged": True,
                "heads": kv * rng.choice([1, 2]), "kv_heads": kv, "width": rng.choice([16, 32, 64]), "causal": False, "prefix": False,
                "cap": rng.choice([0.0, rng.uniform(5.0, 40.0)]), "axes": rng.choice([0, 2, 2])}
    if kind == "sequences":
        rows = _log(rng, 200, 12000)
        kv = rng.choice([1, 2, 4])
        causal = rng.random() < 0.75
        return {"op": "attention", "type": rng.choice(["bf16", "bf16", "f32"]), "train": rng.random() < 0.7, "scenes": rng.randint(1, 12),
                "rows": rows, "keys": rows, "ragged": True, "heads": kv * rng.choice([1, 2]), "kv_heads": kv,
                "width": rng.choice([32, 64, 80, 128]), "causal": causal, "prefix": causal and rng.random() < 0.5,
                "cap": rng.choice([0.0, rng.uniform(10.0, 50.0)]), "axes": rng.choice([0, 0, 1, 2])}
    if kind == "tokens":
        scenes, kv = _log(rng, 1, 32), rng.choice([1, 2, 8])
        return {"op": "attention", "type": rng.choice(["bf16", "bf16", "f32"]), "train": False, "scenes": scenes, "rows": scenes,
                "keys": scenes * _log(rng, 100, 16000), "ragged": True, "heads": kv * rng.choice([1, 3, 4]), "kv_heads": kv,
                "width": rng.choice([32, 64, 128]), "causal": True, "prefix": False, "cap": rng.choice([0.0, rng.uniform(10.0, 50.0)]),
                "axes": rng.choice([0, 0, 1])}
    op = kind.split("_")[0]
    case = {"op": op, "type": "bf16", "train": False, "act": rng.choice(["silu", "gelu"] if op == "gated" else ["none", "leaky", "silu", "gelu"]),
            "bias": rng.random() < 0.6, "residual": op == "linear" and rng.random() < 0.6}
    if kind.endswith("tokens"):
        return {**case, "rows": _log(rng, 1, 16), "inputs": 8 * _log(rng, 16, 512) + rng.choice([0, 0, 0, 5]), "outputs": _log(rng, 256, 12000)}
    case["train"] = rng.random() < 0.8
    if rng.random() < 0.4:
        return {**case, "type": "f32", "rows": _log(rng, 100, 25600), "inputs": _log(rng, 24, 600), "outputs": _log(rng, 24, 600)}
    return {**case, "rows": _log(rng, 100, 8192), "inputs": 8 * _log(rng, 32, 512) + rng.choice([0, 0, 0, 3]), "outputs": _log(rng, 256, 8000)}


# ---- inputs ----------------------------------------------------------------------------------------------------------------

def _lengths(case):
    """(query rows, keys, prefix) of each scene: given by the case, so that every seed has the same work."""
    r = random.Random(case["rows"] * 1009 + case["scenes"])
    S, rows, keys = case["scenes"], case["rows"], case["keys"]
    if rows == S and keys > rows:  # one new row per sequence: a cache of equal room each, filled unevenly
        room = keys // S
        k = [r.randint((room + 1) // 2, room) if case["ragged"] else room for _ in range(S)]
        return [1] * S, k, [0] * S
    if case["ragged"]:
        cuts = sorted(r.randint(0, rows) for _ in range(S - 1))
        q = [b - a for a, b in zip([0] + cuts, cuts + [rows])]
    else:
        q = [rows // S] * S
    return q, q, [r.randint(0, max(1, n // 3)) if case["prefix"] else 0 for n in q]


def _starts(case, lengths):
    if case["keys"] > case["rows"]:
        room = case["keys"] // case["scenes"]
        return [s * room for s in range(case["scenes"])]
    return [sum(lengths[:s]) for s in range(len(lengths))]


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dtype, train = DTYPES[case["type"]], case["train"]

    def normal(*shape, std=1.0, leaf=True):
        t = torch.randn(*shape, generator=gen, device="cuda").mul_(std).to(dtype)
        return t.requires_grad_(train and leaf)

    state = {"case": dict(case)}
    if case["op"] == "attention":
        q, k, prefix = _lengths(case)
        table = lambda start, n: torch.tensor([[a, a + b] for a, b in zip(start, n)], dtype=torch.int32, device="cuda")
        H, Hkv, D = case["heads"], case["kv_heads"], case["width"]
        state |= {"q": normal(case["rows"], H, D), "k": normal(case["keys"], Hkv, D), "v": normal(case["keys"], Hkv, D),
                  "scenes": table([sum(q[:s]) for s in range(len(q))], q), "kv_scenes": table(_starts(case, k), k),
                  "prefix": torch.tensor(prefix, dtype=torch.int32, device="cuda") if case["prefix"] else None,
                  "longest": (max(q), max(k)), "xy": None, "kv_xy": None, "slopes": None}
        if case["axes"] == 2:  # metres, as the trajectories are
            state["xy"] = torch.rand(case["rows"], 2, generator=gen, device="cuda").mul_(15.0)
            state["kv_xy"] = state["xy"] if case["keys"] == case["rows"] else torch.rand(case["keys"], 2, generator=gen, device="cuda").mul_(15.0)
        elif case["axes"] == 1:  # the row's place in its sequence
            at = torch.cat([torch.arange(n, device="cuda") for n in q]).float()
            if case["keys"] > case["rows"]:
                room = case["keys"] // case["scenes"]
                state["kv_xy"] = (torch.arange(case["keys"], device="cuda") % room).float()[:, None]
                at = torch.tensor([n - 1 for n in k], device="cuda").float()
            state["xy"] = at[:, None]
            state["kv_xy"] = state["kv_xy"] if case["keys"] > case["rows"] else state["xy"]
        if case["axes"]:
            low = 1.0 if case["axes"] == 2 else 0.25
            wander = torch.rand(H, generator=gen, device="cuda").mul_(0.2).add_(0.9)
            state["slopes"] = (low * wander * 2.0 ** (-6.0 * torch.arange(H, device="cuda") / H)).requires_grad_(train)
        if train:
            state["grad"] = normal(case["rows"], H, D, leaf=False)
        return state
    M, K, N = case["rows"], case["inputs"], case["outputs"]
    state |= {"x": normal(M, K), "weight": normal(N, K, std=K ** -0.5), "bias": normal(N, std=0.1) if case["bias"] else None}
    if case["op"] == "gated":
        state |= {"up": normal(N, K, std=K ** -0.5), "up_bias": normal(N, std=0.1) if case["bias"] else None}
    else:
        state["residual"] = normal(M, N) if case["residual"] else None
    if train:
        state["grad"] = normal(M, N, leaf=False)
    return state


# ---- the framework's calls -------------------------------------------------------------------------------------------------

def _blocks():
    root = os.path.join(os.getcwd(), "mg-gan_amd")
    if root not in sys.path:
        sys.path.insert(0, root)
    from mggan.hip import blocks

    return blocks


def _leaves(state):
    names = {"attention": ("q", "k", "v", "slopes"), "linear": ("x", "weight", "bias", "residual"),
             "gated": ("x", "weight", "up", "bias", "up_bias")}[state["case"]["op"]]
    return {n: state[n] for n in names if state[n] is not None}


def _call(state):
    case, blocks = state["case"], _blocks()
    if case["op"] == "attention":
        return blocks.attention(state["q"], state["k"], state["v"], state["scenes"], state["kv_scenes"], causal=case["causal"],
                                prefix=state["prefix"], cap=case["cap"], xy=state["xy"], kv_xy=state["kv_xy"], slopes=state["slopes"])
    act = {"none": blocks.ACT_NONE, "leaky": blocks.ACT_LEAKY, "silu": blocks.ACT_SILU, "gelu": blocks.ACT_GELU}[case["act"]]
    if case["op"] == "gated":
        return blocks.gated_linear(state["x"], state["weight"], state["up"], state["bias"], state["up_bias"], act=act)
    return blocks.linear_residual(state["x"], state["weight"], state["bias"], state["residual"], act=act, slope=0.2)


def run(state):
    if own:
        if not state["case"]["train"]:
            with torch.no_grad():
                return {"out": _call(state)}
        leaves = _leaves(state)
        out = _call(state)
        grads = torch.autograd.grad(out, list(leaves.values()), state["grad"])
        return {"out": out.detach(), **{"d" + n: g for n, g in zip(leaves, grads)}}
    with torch.no_grad():
        return _plain_attention(state) if state["case"]["op"] == "attention" else _plain_layer(state)


# ---- the plain forms -------------------------------------------------------------------------------------------------------

def _plain_attention(state):
    """Scenes padded to the longest, whole score matrices: out = softmax(cap tanh(scale q k / cap) - slope |xy - kv_xy|) v."""
    case = state["case"]
    H, Hkv, D, S = case["heads"], case["kv_heads"], case["width"], case["scenes"]
    G, (Lq, Lk), dev = H // Hkv, state["longest"], state["q"].device
    N, M, dtype = case["rows"], case["keys"], state["q"].dtype
    sq, sk = state["scenes"].long(), state["kv_scenes"].long()
    nq, nk = sq[:, 1] - sq[:, 0], sk[:, 1] - sk[:, 0]
    i, j = torch.arange(Lq, device=dev), torch.arange(Lk, device=dev)
    at_q = torch.where(i < nq[:, None], sq[:, :1] + i, N)  # (S, Lq); row N: a place for what is padding
    at_k = torch.where(j < nk[:, None], sk[:, :1] + j, M)
    rows = lambda t, at, n: t[at.clamp(max=n - 1)].float()
    q = rows(state["q"], at_q, N).view(S, Lq, Hkv, G, D).permute(0, 2, 3, 1, 4).reshape(S, Hkv, G * Lq, D)
    k = rows(state["k"], at_k, M).permute(0, 2, 1, 3).contiguous()
    v = rows(state["v"], at_k, M).permute(0, 2, 1, 3).contiguous()
    scale = D ** -0.5
    score = torch.matmul(q, k.transpose(2, 3)).mul_(scale)
    if case["cap"]:
        bent = torch.tanh(score / case["cap"])
        score = bent * case["cap"]
    score = score.view(S, Hkv, G, Lq, Lk)
    if case["axes"]:
        apart = rows(state["xy"], at_q, N)[:, :, None] - rows(state["kv_xy"], at_k, M)[:, None]
        dist = apart.square().sum(-1).sqrt()[:, None, None]
        score = score - state["slopes"].view(1, Hkv, G, 1, 1) * dist
    seen = (j < nk[:, None])[:, None, :] & (i < nq[:, None])[:, :, None]
    if case["causal"]:
        before = j[None, None, :] <= (i + (nk - nq)[:, None])[:, :, None]
        if state["prefix"] is not None:
            before = before | (j < state["prefix"][:, None])[:, None, :]
        seen = seen & before
    score = score.masked_fill(~seen[:, None, None], -math.inf)
    top = score.amax(-1, keepdim=True).clamp(min=-1e30)
    p = torch.exp(score - top)
    p = (p / p.sum(-1, keepdim=True).clamp(min=1e-30)).view(S, Hkv, G * Lq, Lk)
    o = torch.matmul(p, v)

    def query_rows(t):
        out = torch.zeros(N + 1, H, D, dtype=dtype, device=dev)
        out[at_q] = t.view(S, Hkv, G, Lq, D).permute(0, 3, 1, 2, 4).reshape(S, Lq, H, D).to(dtype)
        return out[:N]

    def key_rows(t):
        out = torch.zeros(M + 1, Hkv, D, dtype=dtype, device=dev)
        out[at_k] = t.permute(0, 2, 1, 3).to(dtype)
        return out[:M]

    if not case["train"]:
        return {"out": query_rows(o)}
    do = (rows(state["grad"], at_q, N) * (i < nq[:, None])[:, :, None, None]).view(S, Lq, Hkv, G, D).permute(0, 2, 3, 1, 4).reshape(S, Hkv, G * Lq, D)
    dv = torch.matmul(p.transpose(2, 3), do)
    ds = torch.matmul(do, v.transpose(2, 3))
    ds = p * (ds - (do * o).sum(-1, keepdim=True))
    grads = {"out": query_rows(o), "dv": key_rows(dv)}
    if case["axes"]:
        grads["dslopes"] = -(ds.view(S, Hkv, G, Lq, Lk) * dist).sum((0, 3, 4)).view(H)
    if case["cap"]:
        ds = ds * (1.0 - bent.square())
    ds = ds * scale
    return {**grads, "dq": query_rows(torch.matmul(ds, k)), "dk": key_rows(torch.matmul(ds.transpose(2, 3), q))}


def _act(z, act):
    """The activation and its derivative."""
    if act == "none":
        return z, torch.ones_like(z)
    if act == "leaky":
        return torch.where(z > 0, z, 0.2 * z), torch.where(z > 0, 1.0, 0.2)
    if act == "silu":
        s = 1.0 / (1.0 + torch.exp(-z))
        return z * s, s * (1.0 + z * (1.0 - s))
    half = 0.5 * (1.0 + torch.erf(z * math.sqrt(0.5)))
    return z * half, half + z * torch.exp(-0.5 * z * z) / math.sqrt(2.0 * math.pi)


def _plain_layer(state):
    case, dtype = state["case"], state["x"].dtype
    f = lambda n: state[n].float() if state.get(n) is not None else None
    x, w, b = f("x"), f("weight"), f("bias")
    z = torch.matmul(x, w.t())
    z = z if b is None else z + b
    if case["act"] == "none" and case["op"] == "linear":
        a, slope = z, None
    else:
        a, slope = _act(z, case["act"])
    if case["op"] == "gated":
        u_w, u_b = f("up"), f("up_bias")
        u = torch.matmul(x, u_w.t())
        u = u if u_b is None else u + u_b
        out = a * u
    else:
        out = a if state["residual"] is None else a + f("residual")
    outs = {"out": out}
    if case["train"]:
        dy = state["grad"].float()
        da = dy * u if case["op"] == "gated" else dy
        dz = da if slope is None else da * slope
        dx, outs["dweight"] = torch.matmul(dz, w), torch.matmul(dz.t(), x)
        if b is not None:
            outs["dbias"] = dz.sum(0)
        if case["op"] == "gated":
            du = dy * a
            dx, outs["dup"] = dx + torch.matmul(du, u_w), torch.matmul(du.t(), x)
            if u_b is not None:
                outs["dup_bias"] = du.sum(0)
        elif state["residual"] is not None:
            outs["dresidual"] = dy
        outs["dx"] = dx
    return {n: t.to(dtype) for n, t in outs.items()}


# ---- what a pass cannot do without -----------------------------------------------------------------------------------------

def work(case):
    size = 2 if case["type"] == "bf16" else 4
    if case["op"] == "attention":
        q, k, prefix = _lengths(case)
        pairs = 0
        for n, m, p in zip(q, k, prefix):
            if not case["causal"]:
                pairs += n * m
            else:  # row i sees max(min(p, m), i + 1 + m - n) keys
                first = m - n + 1
                over = max(0, min(n, min(p, m) - first + 1))
                pairs += over * min(p, m) + sum(range(first + over, first + n))
        H, Hkv, D = case["heads"], case["kv_heads"], case["width"]
        rows, keys = sum(q) * H * D, sum(k) * Hkv * D
        place = 4 * case["axes"] * (sum(q) + (sum(k) if case["keys"] > case["rows"] else 0))
        if not case["train"]:
            return {"bytes": size * (2 * rows + 2 * keys) + place, "flops": 4 * pairs * H * D}
        return {"bytes": size * (4 * rows + 4 * keys) + place, "flops": 12 * pairs * H * D}
    M, K, N = case["rows"], case["inputs"], case["outputs"]
    two = 2 if case["op"] == "gated" else 1
    weights, bias, res = two * N * K, two * N * case["bias"], M * N * case["residual"]
    if not case["train"]:
        return {"bytes": size * (M * K + weights + bias + res + M * N), "flops": 2 * two * M * N * K}
    return {"bytes": size * (2 * M * K + 2 * weights + 2 * bias + res + 2 * M * N), "flops": 6 * two * M * N * K}


# ---- in 64 bits ------------------------------------------------------------------------------------------------------------

def exact(case, seed):
    state = prepare(case, seed)
    return _exact_attention(case, state) if case["op"] == "attention" else _exact_layer(case, state)


def _exact_attention(case, state):
    """Scene by scene and key head by key head, gradients by differentiating the definition."""
    nq, nk, prefix = _lengths(case)
    G, D = case["heads"] // case["kv_heads"], case["width"]
    out = torch.zeros(case["rows"], case["heads"], D, dtype=torch.float64, device="cuda")
    grads = {n: torch.zeros_like(state[n], dtype=torch.float64) for n in ("q", "k", "v", "slopes") if case["train"] and state[n] is not None}
    for s, (n, m) in enumerate(zip(nq, nk)):
        if n == 0 or m == 0:
            continue
        a, b = sum(nq[:s]), _starts(case, nk)[s]
        row, col = torch.arange(n, device="cuda")[:, None], torch.arange(m, device="cuda")[None, :]
        hidden = (col > row + (m - n)) & (col >= prefix[s]) if case["causal"] else torch.zeros(n, m, dtype=torch.bool, device="cuda")
        dist = None
        if case["axes"]:
            place, kv_place = state["xy"][a:a + n].double(), state["kv_xy"][b:b + m].double()
            dist = (place[:, None] - kv_place[None]).norm(dim=-1)
        for h in range(case["heads"]):
            part = {"q": state["q"][a:a + n, h], "k": state["k"][b:b + m, h // G], "v": state["v"][b:b + m, h // G]}
            if case["axes"]:
                part["slopes"] = state["slopes"][h]
            part = {x: t.detach().double().requires_grad_(case["train"]) for x, t in part.items()}
            logit = part["q"] @ part["k"].t() / math.sqrt(D)
            if case["cap"]:
                logit = case["cap"] * torch.tanh(logit / case["cap"])
            if case["axes"]:
                logit = logit - part["slopes"] * dist
            o = torch.softmax(logit.masked_fill(hidden, -math.inf), -1) @ part["v"]
            out[a:a + n, h] = o.detach()
            if case["train"]:
                g = dict(zip(part, torch.autograd.grad(o, list(part.values()), state["grad"][a:a + n, h].double())))
                grads["q"][a:a + n, h] += g["q"]
                grads["k"][b:b + m, h // G] += g["k"]
                grads["v"][b:b + m, h // G] += g["v"]
                if case["axes"]:
                    grads["slopes"][h] += g["slopes"]
    return {"out": out, **{"d" + n: g for n, g in grads.items()}}


def _exact_layer(case, state):
    leaves = {n: t.detach().double().requires_grad_(case["train"]) for n, t in _leaves(state).items()}
    F = torch.nn.functional
    act = {"none": lambda z: z, "leaky": lambda z: F.leaky_relu(z, 0.2), "silu": F.silu, "gelu": F.gelu}[case["act"]]
    out = act(F.linear(leaves["x"], leaves["weight"], leaves.get("bias")))
    if case["op"] == "gated":
        out = out * F.linear(leaves["x"], leaves["up"], leaves.get("up_bias"))
    elif "residual" in leaves:
        out = out + leaves["residual"]
    grads = torch.autograd.grad(out, list(leaves.values()), state["grad"].double()) if case["train"] else []
    return {"out": out.detach(), **{"d" + n: g for n, g in zip(leaves, grads)}}
