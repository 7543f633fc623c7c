"""What is measured of the 8-bit grouped product, its row quantiser and the norms around an expert block.

``run`` computes an operator in plain torch operations (``own`` false) or with the calls a user makes of
``gmm_b200`` (``own`` true); ``exact`` gives the same results from the definitions in 64 bits.  The plain
grouped product pads every expert to the case's ``cap`` rows and multiplies them as one batch in fp32.
"""

import math

import torch

own = False

DEV = "cuda"
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
SIZE = {"bf16": 2, "fp16": 2, "fp32": 4}


# ------------------------------------------------------------------ the cases
def _int8(name, experts, empty, rows, cap, dim, dim_out, out, swiglu, sizes):
    return {"name": name, "op": "int8", "experts": experts, "empty": empty, "rows": rows, "cap": cap, "dim": dim,
            "dim_out": dim_out, "out": out, "swiglu": swiglu, "sizes": sizes}


def _quant(name, rows, dim, k, dtype):
    return {"name": name, "op": "quant", "rows": rows, "dim": dim, "k": k, "dtype": dtype}


def _norm(name, op, rows, dim, dtype, params, gate, act, following):
    return {"name": name, "op": op, "rows": rows, "dim": dim, "dtype": dtype, "params": params, "gate": gate,
            "act": act, "next": following}


def listed():
    return [
        # one token routed to 8 of 128 experts, gate/up projection: the smallest call of a decode step
        _int8("int8_one_token", 128, 120, 8, 1, 2048, 1536, "bf16", True, "device"),
        # a decode batch of 128 tokens, 8 experts each, down projection (1..16 rows an expert)
        _int8("int8_decode", 128, 0, 1024, 16, 768, 2048, "bf16", False, "device"),
        # fine-grained experts with uneven loads and some without a row, odd row count; the scaled sums left in fp32
        _int8("int8_fine", 64, 5, 4099, 160, 7168, 4096, "fp32", False, "host"),
        # gate/up projection with SwiGLU of a ragged prefill chunk on 8 experts
        _int8("int8_gate_up", 8, 0, 8195, 1536, 4096, 28672, "fp16", True, "host"),
        # the up projection of a large prefill on 8 experts
        _int8("int8_prefill", 8, 0, 16384, 2304, 4096, 14336, "bf16", False, "host"),
        # activations of a prefill quantised straight into expert order, top 2
        _quant("quant_prefill", 16384, 4096, 2, "bf16"),
        # a decode batch of tokens quantised for their 8 experts; width that is no multiple of 16
        _quant("quant_decode", 128, 2056, 8, "fp16"),
        # a decode step's tokens through post-norm, channel gate, residual and the next pre-norm
        _norm("norm_decode", "norm", 128, 7168, "bf16", "bf16", "channel", "none", True),
        # the same for a large prefill
        _norm("norm_prefill", "norm", 16384, 4096, "bf16", "fp32", "channel", "tanh", True),
        # a gate of its own for each element, odd row count, last block (no next norm)
        _norm("norm_full_gate", "norm", 8191, 6144, "fp16", "fp16", "full", "sigmoid", False),
        # forward and backward of a training step
        _norm("norm_train", "train", 16384, 4096, "bf16", "fp32", "channel", "tanh", True),
        # forward and backward in fp32 with one gate a token, odd sizes
        _norm("norm_train_fp32", "train", 1027, 2050, "fp32", "fp32", "token", "sigmoid", True),
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(["int8", "int8", "quant", "norm", "train"])
    if op == "int8":
        swiglu = rng.random() < 0.4
        while True:
            experts, dim, dim_out = _log(rng, 1, 256), 16 * _log(rng, 4, 448), (16 if swiglu else 8) * _log(rng, 8, 1024)
            empty = rng.randrange(0, experts) if rng.random() < 0.4 else 0
            live = experts - empty
            rows = max(live, _log(rng, 1, 16384))
            cap = rows if live == 1 else max(1, -(-rows * rng.choice([5, 6, 8]) // (4 * live)))
            # the weights and the padded plain product stay below the largest listed case's
            if experts * dim * dim_out <= 9e8 and 2.0 * experts * cap * dim * dim_out <= 2e12 and cap * experts * dim <= 4e8:
                break
        case = _int8(None, experts, empty, rows, cap, dim, dim_out, rng.choice(["bf16", "fp16"] if swiglu else ["bf16", "fp16", "fp32"]),
                     swiglu, rng.choice(["host", "device"]))
    elif op == "quant":
        while True:
            rows, dim, k = _log(rng, 1, 16384), _log(rng, 16, 8192), rng.randint(1, 8)
            if rows * dim * k <= 1.3e8:
                break
        case = _quant(None, rows, dim, k, rng.choice(["bf16", "fp16", "fp32"]))
    else:
        while True:
            rows, dim = _log(rng, 1, 16384), _log(rng, 16, 8192)
            dtype = rng.choice(["bf16", "fp16", "fp32"])
            if rows * dim * SIZE[dtype] <= 1.3e8:
                break
        case = _norm(None, op, rows, dim, dtype, rng.choice(["fp32", dtype]), rng.choice(["none", "channel", "token", "full"]),
                     rng.choice(["none", "tanh", "sigmoid"]), rng.random() < 0.7)
    del case["name"]
    return case


# ------------------------------------------------------------------ inputs
def _sizes(case, seed):
    """Rows of each expert: the live ones get one each, the rest by uneven weights, none above ``cap``."""
    g = torch.Generator().manual_seed(seed)
    live = torch.randperm(case["experts"], generator=g)[: case["experts"] - case["empty"]]
    n, cap = live.numel(), case["cap"]
    weights = 0.5 + torch.rand(n, generator=g, dtype=torch.float64)
    rest = case["rows"] - n
    more = torch.floor(rest * weights / weights.sum()).long().clamp_(max=cap - 1)
    room = (cap - 1) - more
    left = rest - int(more.sum())
    # what is left goes to the experts with room, in a random order
    order = torch.randperm(n, generator=g)
    ahead = room[order].cumsum(0) - room[order]
    more[order] += (left - ahead).clamp(min=0).minimum(room[order])
    sizes = torch.zeros(case["experts"], dtype=torch.int64)
    sizes[live] = more + 1
    return sizes


def _codes(shape, gen):
    """8-bit codes as rows quantised by their largest value have them: near normal, a quarter of the range wide."""
    return torch.randn(shape, generator=gen, device=DEV, dtype=torch.float16).mul_(34.0).round_().clamp_(-127, 127).to(torch.int8)


def prepare(case, seed):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    s = {"case": case}
    if case["op"] == "int8":
        T, E, K, N = case["rows"], case["experts"], case["dim"], case["dim_out"]
        s["sizes"] = _sizes(case, seed)
        if case["sizes"] == "device":
            s["sizes"] = s["sizes"].to(device=DEV, dtype=torch.int32)
        s["a"] = _codes((T, K), gen)
        s["b"] = _codes((E, N, K), gen)
        s["sa"] = torch.rand(T, generator=gen, device=DEV) * 0.02 + 0.01
        s["sb"] = (torch.rand(E, N, generator=gen, device=DEV) * 0.02 + 0.02) / math.sqrt(K)
    elif case["op"] == "quant":
        T, D, k = case["rows"], case["dim"], case["k"]
        x = torch.randn(T, D, generator=gen, device=DEV)
        x *= torch.rand(T, 1, generator=gen, device=DEV) * 4 + 0.1
        s["x"] = x.to(TYPES[case["dtype"]])
        s["place"] = torch.randperm(T * k, generator=gen, device=DEV).view(T, k).to(torch.int32)
    else:
        T, D, t = case["rows"], case["dim"], TYPES[case["dtype"]]
        pt = TYPES[case["params"]]
        s["y"] = (torch.randn(T, D, generator=gen, device=DEV) * 0.5).to(t)
        s["x"] = (torch.randn(T, D, generator=gen, device=DEV) * 2).to(t)
        s["w"] = (torch.rand(D, generator=gen, device=DEV) + 0.5).to(pt)
        s["v"] = (torch.rand(D, generator=gen, device=DEV) + 0.5).to(pt) if case["next"] else None
        shape = {"none": None, "channel": (D,), "token": (T, 1), "full": (T, D)}[case["gate"]]
        s["g"] = None if shape is None else torch.randn(shape, generator=gen, device=DEV).to(pt if case["gate"] == "channel" else t)
        if case["op"] == "train":
            s["dx"] = torch.randn(T, D, generator=gen, device=DEV).to(t)
            s["dh"] = torch.randn(T, D, generator=gen, device=DEV).to(t) if case["next"] else None
            for k in ("y", "x", "w", "v", "g"):
                s[k] = None if s[k] is None else s[k].requires_grad_()
    return s


SCALE, EPS = 0.7, 1e-5


# ------------------------------------------------------------------ one pass
def run(s):
    case = s["case"]
    if own:
        return _run_own(case, s)
    return {"int8": _plain_int8, "quant": _plain_quant, "norm": _plain_norm, "train": _plain_train}[case["op"]](case, s)


def _run_own(case, s):
    if case["op"] == "int8":
        from gmm_b200.int8 import gmm_int8, gmm_int8_dev
        call = gmm_int8_dev if case["sizes"] == "device" else gmm_int8
        return call(s["a"], s["sa"], s["b"], s["sb"], s["sizes"], out_dtype=TYPES[case["out"]], swiglu=case["swiglu"])
    if case["op"] == "quant":
        from gmm_b200.int8 import quantize_rows
        return quantize_rows(s["x"], s["place"])
    from gmm_b200.norms import post_norm
    out = post_norm(s["y"], s["x"], s["w"], gate=s["g"], gate_act=case["act"], residual_scale=SCALE, next_weight=s["v"], eps=EPS)
    if case["op"] == "norm":
        return out
    leaves = [s[k] for k in ("y", "x", "w", "v", "g") if s[k] is not None]
    outs, grads = (out, (s["dx"], s["dh"])) if case["next"] else ((out,), (s["dx"],))
    return [o.detach() for o in outs], list(torch.autograd.grad(outs, leaves, grads))


def _plain_int8(case, s):
    T, cap = case["rows"], case["cap"]
    sizes = s["sizes"].to(DEV, torch.int64)
    first = sizes.cumsum(0) - sizes
    place = torch.arange(cap, device=DEV)
    rows = (first[:, None] + place).clamp_(max=T - 1)
    padded = s["a"][rows].float()
    sums = torch.matmul(padded, s["b"].float().transpose(1, 2))
    sums *= s["sa"][rows][..., None]
    sums *= s["sb"][:, None, :]
    if case["swiglu"]:
        gate, up = sums.chunk(2, dim=-1)
        sums = gate * torch.sigmoid(gate) * up
    live = place < sizes[:, None]
    return sums.to(TYPES[case["out"]])[live]


def _plain_quant(case, s):
    T, D, k = case["rows"], case["dim"], case["k"]
    x = s["x"].float()
    top = x.abs().amax(dim=-1)
    scale = top / torch.full_like(top, 127.0)  # a tensor divisor: a true division, not a product with 1 / 127
    codes = torch.round(x / torch.where(scale > 0, scale, 1.0)[:, None]).clamp_(-127, 127).to(torch.int8)
    q = torch.zeros(T * k, -(-D // 16) * 16, dtype=torch.int8, device=DEV)
    place = s["place"].long()
    q[:, :D][place.reshape(-1)] = codes.repeat_interleave(k, dim=0)
    out_scale = torch.empty(T * k, device=DEV)
    out_scale[place.reshape(-1)] = scale.repeat_interleave(k)
    return q, out_scale


def _act(g, act):
    return torch.tanh(g) if act == "tanh" else torch.sigmoid(g) if act == "sigmoid" else g


def _plain_forward(case, y, x, w, v, g):
    n = y * torch.rsqrt(y.square().mean(-1, keepdim=True) + EPS) * w
    new = x + SCALE * (n if g is None else _act(g, case["act"]) * n)
    if v is None:
        return (new,)
    return new, new * torch.rsqrt(new.square().mean(-1, keepdim=True) + EPS) * v


def _plain_norm(case, s):
    t = TYPES[case["dtype"]]
    out = [o.to(t) for o in _plain_forward(case, *(None if s[k] is None else s[k].float() for k in ("y", "x", "w", "v", "g")))]
    return tuple(out) if case["next"] else out[0]


def _plain_train(case, s):
    t = TYPES[case["dtype"]]
    names = ("y", "x", "w", "v", "g")
    f = [None if s[k] is None else s[k].detach().float().requires_grad_() for k in names]
    outs = _plain_forward(case, *f)
    given = [s["dx"].float()] + ([s["dh"].float()] if case["next"] else [])
    grads = torch.autograd.grad(outs, [p for p in f if p is not None], given)
    types = [s[k].dtype for k in names if s[k] is not None]
    return [o.detach().to(t) for o in outs], [d.to(dt) for d, dt in zip(grads, types)]


# ------------------------------------------------------------------ what a pass cannot do without
def work(case):
    if case["op"] == "int8":
        T, E, K, N = case["rows"], case["experts"] - case["empty"], case["dim"], case["dim_out"]
        out = N // 2 if case["swiglu"] else N
        return {"bytes": T * K + E * N * K + 4 * (T + E * N) + T * out * SIZE[case["out"]], "flops": 2.0 * T * K * N}
    T, D = case["rows"], case["dim"]
    if case["op"] == "quant":
        k = case["k"]
        return {"bytes": T * D * SIZE[case["dtype"]] + T * k * (-(-D // 16) * 16 + 8), "flops": 4.0 * T * D}
    gate = {"none": 0, "channel": D * SIZE[case["params"]], "token": T * SIZE[case["dtype"]], "full": T * D * SIZE[case["dtype"]]}[case["gate"]]
    params = D * SIZE[case["params"]] * (2 if case["next"] else 1)
    one = T * D * SIZE[case["dtype"]]
    bytes_, flops = one * (4 if case["next"] else 3) + gate + params, 12.0 * T * D
    if case["op"] == "train":  # the backward pass: y, x and the outputs' gradients in, two gradients and the parameters' out
        bytes_ += one * (6 if case["next"] else 5) + 2 * (gate + params)
        flops += 30.0 * T * D
    return {"bytes": bytes_, "flops": flops}


# ------------------------------------------------------------------ the definitions in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    return {"int8": _exact_int8, "quant": _exact_quant, "norm": _exact_norm, "train": _exact_norm}[case["op"]](case, s)


def _exact_int8(case, s):
    at, parts = 0, []
    for e, m in enumerate(s["sizes"].tolist()):
        if m == 0:
            continue
        d = s["a"][at: at + m].double() @ s["b"][e].double().t()
        d = torch.einsum("ij,i,j->ij", d, s["sa"][at: at + m].double(), s["sb"][e].double())
        if case["swiglu"]:
            half = case["dim_out"] // 2
            d = d[:, :half] / (1 + torch.exp(-d[:, :half])) * d[:, half:]
        parts.append(d)
        at += m
    return torch.cat(parts)


def _exact_quant(case, s):
    scale = torch.empty(case["rows"] * case["k"], dtype=torch.float64, device=DEV)
    top = s["x"].double().abs().max(dim=1).values / 127
    for j in range(case["k"]):
        scale[s["place"][:, j].long()] = top
    return None, scale  # the codes are whole numbers


def _exact_norm(case, s):
    """Outputs, and the gradients from their formulas."""
    y, x, w, v, g = (None if s[k] is None else s[k].detach().double() for k in ("y", "x", "w", "v", "g"))
    ry = (y.pow(2).sum(1, keepdim=True) / case["dim"] + EPS) ** -0.5
    if g is None:
        a, da = torch.ones((), dtype=torch.float64, device=DEV), None
    elif case["act"] == "tanh":
        a = g.tanh()
        da = 1 - a * a
    elif case["act"] == "sigmoid":
        a = 1 / (1 + torch.exp(-g))
        da = a * (1 - a)
    else:
        a, da = g, torch.ones_like(g)
    unit = y * ry
    new = x + SCALE * a * w * unit
    rx = (new.pow(2).sum(1, keepdim=True) / case["dim"] + EPS) ** -0.5
    outs = [new] + ([new * rx * v] if v is not None else [])
    if case["op"] == "norm":
        return tuple(outs) if v is not None else outs[0]
    dnew = s["dx"].double()
    dv = None
    if v is not None:
        dh, xu = s["dh"].double(), new * rx
        u = dh * v
        dnew = dnew + rx * (u - xu * (u * xu).mean(1, keepdim=True))
        dv = (dh * xu).sum(0)
    dn = SCALE * a * dnew
    t = dn * w
    dy = ry * (t - unit * (t * unit).mean(1, keepdim=True))
    grads = [dy, dnew, (dn * unit).sum(0)] + ([dv] if dv is not None else [])
    if g is not None:
        dg = SCALE * w * unit * dnew * da
        grads.append({"channel": lambda: dg.sum(0), "token": lambda: dg.sum(1, keepdim=True), "full": lambda: dg}[case["gate"]]())
    return outs, grads
