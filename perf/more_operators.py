"""Serving in fewer bytes and fewer launches, as measurable calls: 8-bit products with a scale
for each block of 128, and a whole mixture-of-experts layer for a few tokens.

A case is one call of one of these kinds:

* ``quant``    values to e4m3 with an f32 scale for each 128 columns of a row (activations) or
               for each square of 128 x 128 (weights)
* ``product``  y = a b^T of two such matrices: a with scales by rows, b by squares
* ``ffn``      a dense SwiGLU feed-forward on 8-bit weights and activations
* ``few``      an MoE layer, router to weighted sum, for up to 64 rows; on request with its
               experts' weights in 8 bits, or under a routing that the caller has

A block's scale is the largest magnitude in it / 448 (at least 2^-126), as the nearest f32; a value
is divided by its block's scale and rounded to the nearest e4m3.  Activations are N(0, 1) with rows
of different sizes and a few large columns, weights N(0, 1/sqrt(fan-in)), biases N(0, 0.1).
"""
import math
import os
import sys

import torch

own = False

PATH = "blocks.0.moe"
FFN_PATH = "blocks.0.mlp"
LINEARS = ("gate.weight", "gate.bias", "up.weight", "up.bias", "down.weight", "down.bias")
BLOCK = 128
MOST = 448.0         # e4m3's largest value
LEAST = 2.0 ** -126  # the smallest scale
ROUTE_EPS = 1e-9     # of the renormalised weights
FEW_ROWS = 64


def _package():
    root = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))),
                        "hy-nomas-rs_amd")
    if root not in sys.path:
        sys.path.insert(0, root)
    import nomas_moe
    return nomas_moe


# ---- cases -------------------------------------------------------------------

def _quant(name, dtype, rows, cols, square):
    return {"name": name, "kind": "quant", "dtype": dtype, "rows": rows, "cols": cols,
            "square": square}


def _product(name, dtype, rows, k, n, bias=False):
    return {"name": name, "kind": "product", "dtype": dtype, "rows": rows, "k": k, "n": n,
            "bias": bias}


def _ffn(name, dtype, rows, dim, hidden):
    return {"name": name, "kind": "ffn", "dtype": dtype, "rows": rows, "dim": dim,
            "hidden": hidden}


def _few(name, dtype, rows, dim, hidden, experts, top_k, dense=0.0, fp8=False, given=False):
    return {"name": name, "kind": "few", "dtype": dtype, "rows": rows, "dim": dim,
            "hidden": hidden, "experts": experts, "top_k": top_k, "dense": dense, "fp8": fp8,
            "given": given}


def listed():
    return [
        # the activations of one branch of a turn (4,680 video and 64 text rows)
        _quant("quant_segment", "bf16", 4744, 2048, False),
        # a weight as a checkpoint of full precision holds it
        _quant("quant_weights", "f32", 8192, 2048, True),
        # one new row through one linear layer: the weight is streamed once
        _product("product_token", "bf16", 1, 2048, 8192),
        # a few rows, sums kept in f32
        _product("product_few", "f32", 40, 4096, 1536),
        # widths that no tile divides, with a bias
        _product("product_ragged", "f16", 1111, 1008, 2667, bias=True),
        # three guidance branches stacked
        _product("product_branches", "bf16", 14232, 2048, 8192),
        # a handful of rows through a dense feed-forward
        _ffn("ffn_few", "bf16", 16, 1536, 4096),
        # one branch of a turn
        _ffn("ffn_segment", "bf16", 4744, 2048, 8192),
        # the tiny preset's layer on two rows, with the shared dense branch: launches alone
        _few("few_tiny_f32", "f32", 2, 64, 128, 4, 2, dense=0.5),
        # one new token of a causal session through many fine experts
        _few("few_token", "bf16", 1, 2048, 768, 64, 8),
        # a batch of sessions, one row each: every expert is read
        _few("few_batch", "f16", 48, 1024, 2048, 16, 2),
        # a few rows under the caller's routing, on 8-bit weights
        _few("few_fp8", "bf16", 5, 1024, 2048, 16, 2, fp8=True, given=True),
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["quant", "product", "product", "ffn", "few", "few"])
    if kind == "quant":
        dtype = rng.choice(["bf16", "f16", "f32"])
        cols = 16 * _log_int(rng, 1, 512)
        rows = _log_int(rng, 1, min(32768, 8192 * 2048 // cols))
        case = _quant("", dtype, rows, cols, rng.random() < 0.4)
    elif kind == "product":
        k, n = 16 * _log_int(rng, 2, 256), _log_int(rng, 8, 8192)
        most = min(16384, 14232 * 2048 * 8192 // (k * n), 14232 * 8192 // n)
        case = _product("", rng.choice(["bf16", "bf16", "f16", "f32"]), _log_int(rng, 1, most), k,
                        n, rng.random() < 0.4)
    elif kind == "ffn":
        dim, hidden = 8 * _log_int(rng, 8, 256), _log_int(rng, 64, 8192)
        most = min(8192, 4744 * 2048 * 8192 // (dim * hidden))
        case = _ffn("", rng.choice(["bf16", "bf16", "f16"]), _log_int(rng, 1, most), dim, hidden)
    else:
        experts = rng.choice([4, 8, 16, 32, 64])
        dim, hidden = 8 * _log_int(rng, 8, 256), _log_int(rng, 64, 2048)
        while experts * dim * hidden > 16 * 1024 * 2048:
            experts //= 2
        experts = max(experts, 2)
        dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
        if dtype == "f32" and experts * dim * hidden > 8 * 1024 * 2048:
            hidden = (hidden + 1) // 2
        case = _few("", dtype, _log_int(rng, 1, FEW_ROWS), dim, hidden, experts,
                    min(experts, rng.choice([1, 2, 2, 4, 8])), rng.choice([0.0, 0.0, 0.5]),
                    dtype != "f32" and rng.random() < 0.4, rng.random() < 0.4)
    return {k: v for k, v in case.items() if k != "name"}


# ---- inputs ------------------------------------------------------------------

def _dtype(case):
    return {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}[case["dtype"]]


def _generator(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _randn(g, *shape, std=1.0, mean=0.0, to=torch.float32):
    return torch.randn(*shape, generator=g, device="cuda").mul_(std).add_(mean).to(to)


def _activations(g, rows, cols, to):
    x = _randn(g, rows, cols) * torch.exp(_randn(g, rows, 1, std=0.3))
    large = torch.rand(cols, generator=g, device="cuda") < 0.01
    return torch.where(large, 8.0 * x, x).to(to)


def _expand(scale, rows, cols, square):
    """A scale for each element."""
    s = scale.repeat_interleave(BLOCK, 1)[:, :cols]
    return s.repeat_interleave(BLOCK, 0)[:rows] if square else s


def _plain_quantize(x, square):
    """(values as e4m3, scales) of a matrix."""
    rows, cols = x.shape
    x = x.float()
    kb = -(-cols // BLOCK)
    size = torch.zeros(rows, kb * BLOCK, device=x.device)
    size[:, :cols] = x.abs()
    size = size.view(rows, kb, BLOCK).amax(-1)
    if square:
        rb = -(-rows // BLOCK)
        tall = torch.zeros(rb * BLOCK, kb, device=x.device)
        tall[:rows] = size
        size = tall.view(rb, BLOCK, kb).amax(1)
    scale = (size.double() / MOST).clamp(min=LEAST).float()
    # nearest in 64 bits: of values of 16 bits many quotients are next to the middle of two e4m3
    v = x.double() / _expand(scale, rows, cols, square).double()
    m = torch.frexp(v)[0]  # (v / m is a power of two)
    v = torch.where(v.abs() < 2.0 ** -6, torch.round(512.0 * v) / 512.0,
                    torch.round(16.0 * m) / 16.0 * (v / m))
    return v.float().to(torch.float8_e4m3fn), scale


def _plain_dequantize(q, scale, square):
    return q.float() * _expand(scale, *q.shape, square)


def _linears(g, case, lead):
    D, H, dt = case["dim"], case["hidden"], _dtype(case)
    return {name: _randn(g, *lead, *shape, std=std, to=dt)
            for name, shape, std in (("gate.weight", (H, D), D ** -0.5), ("gate.bias", (H,), 0.1),
                                     ("up.weight", (H, D), D ** -0.5), ("up.bias", (H,), 0.1),
                                     ("down.weight", (D, H), H ** -0.5), ("down.bias", (D,), 0.1))}


def _inputs(case, seed):
    g, kind, dt = _generator(seed), case["kind"], _dtype(case)
    if kind == "quant":
        if case["square"]:
            return {"x": _randn(g, case["rows"], case["cols"], std=case["cols"] ** -0.5, to=dt)}
        return {"x": _activations(g, case["rows"], case["cols"], dt)}
    if kind == "product":
        s = {}
        s["a"], s["a_scale"] = _plain_quantize(
            _activations(g, case["rows"], case["k"], torch.float32), False)
        s["b"], s["b_scale"] = _plain_quantize(
            _randn(g, case["n"], case["k"], std=case["k"] ** -0.5), True)
        s["bias"] = _randn(g, case["n"], std=0.1) if case["bias"] else None
        return s
    if kind == "ffn":
        s = _linears(g, case, ())
        s["x"] = _activations(g, case["rows"], case["dim"], dt)
        return s
    E, D, k, T = case["experts"], case["dim"], case["top_k"], case["rows"]
    s = _linears(g, case, (E + (1 if case["dense"] else 0),))  # the shared dense branch last
    s["x"] = _randn(g, T, D, to=dt)
    s["router"] = _randn(g, E, D, std=D ** -0.5, to=dt)
    s["idx"] = s["w"] = None
    if case["given"]:
        s["idx"] = _randn(g, T, E).argsort(-1)[:, :k].sort(-1).values.to(torch.int32)
        s["w"] = torch.softmax(_randn(g, T, k), -1)
    return s


def _layer(case, s):
    """The layer that a program keeps."""
    nm = _package()
    dt, D, H = nm.DataType.of(case["dtype"]), case["dim"], case["hidden"]
    host = {n: s[n].float().cpu().numpy() for n in LINEARS}
    if case["kind"] == "ffn":
        layer = nm.FeedForward.from_source(
            nm.Weights.tensors_({f"{FFN_PATH}.{n}": host[n] for n in LINEARS}, dt), FFN_PATH, D, H)
        layer.quantize()
        return layer
    E = case["experts"]
    named = {f"{PATH}.experts.{e}.{n}": host[n][e] for n in LINEARS for e in range(E)}
    if case["dense"]:
        named.update({f"{PATH}.dense.{n}": host[n][E] for n in LINEARS})
    named[f"{PATH}.router.weight"] = s["router"].float().cpu().numpy()
    layer = nm.MoeLayer.from_source(nm.Weights.tensors_(named, dt), PATH, D, H,
                                    nm.MoeConfig(E, case["top_k"], case["dense"]))
    if case["fp8"]:
        layer.quantize()
    return layer


def _in_8_bits(case, s):
    """The 8-bit weights that a program keeps, as e4m3 and scales."""
    kept = {}
    for n in ("gate.weight", "up.weight", "down.weight"):
        w = s[n] if case["kind"] == "few" else s[n][None]
        pairs = [_plain_quantize(w[e], True) for e in range(w.shape[0])]
        kept[n] = torch.stack([q for q, _ in pairs])
        kept[n + "_scale"] = torch.stack([c for _, c in pairs])
    return kept


def prepare(case, seed):
    state = _inputs(case, seed)
    if case["kind"] in ("ffn", "few"):
        if own:
            state["layer"] = _layer(case, state)
        elif case["kind"] == "ffn" or case["fp8"]:
            state.update(_in_8_bits(case, state))
    state["case"] = case
    return state


# ---- the plain forms -----------------------------------------------------------

def _silu(g):
    return g / (1.0 + torch.exp(-g))


def _plain_ffn(case, s):
    def product(x, name):
        w, ws = s[name + ".weight"][0], s[name + ".weight_scale"][0]
        q, qs = _plain_quantize(x, False)
        return _plain_dequantize(q, qs, False) @ _plain_dequantize(w, ws, True).T + \
            s[name + ".bias"].float()

    h = _silu(product(s["x"], "gate")) * product(s["x"], "up")
    return product(h, "down").to(_dtype(case))


def _plain_gates(case, s):
    """Each row's weight of each expert (0 where not chosen); the choice in 64 bits."""
    E, k, T = case["experts"], case["top_k"], case["rows"]
    gates = torch.zeros(T, E, dtype=torch.float64, device="cuda")
    if case["given"]:
        return gates.scatter_add_(1, s["idx"].long(), s["w"].double()).float()
    logits = s["x"].double() @ s["router"].double().T
    e = torch.exp(logits - logits.amax(-1, keepdim=True))
    p = e / e.sum(-1, keepdim=True)
    order = logits.sort(dim=-1, descending=True, stable=True).indices[:, :k]
    chosen = p.gather(1, order)
    return gates.scatter_(1, order, chosen / (chosen.sum(-1, keepdim=True) + ROUTE_EPS)).float()


def _plain_few(case, s):
    """Every expert on every row, weighed by its gate."""
    def weight(name):
        w = s[name + ".weight"]
        if not case["fp8"]:
            return w.float()
        scale = s[name + ".weight_scale"].repeat_interleave(BLOCK, 1)[:, :w.shape[1]]
        return w.float() * scale.repeat_interleave(BLOCK, 2)[:, :, :w.shape[2]]

    def linear(x, name):  # x: columns are rows of the call
        return torch.matmul(weight(name), x) + s[name + ".bias"].float()[:, :, None]

    gates = _plain_gates(case, s)
    if case["dense"]:
        gates = torch.cat([gates, torch.full_like(gates[:, :1], case["dense"])], 1)
    x = s["x"].float().T.contiguous()
    h = _silu(linear(x, "gate")) * linear(x, "up")
    y = linear(h, "down")  # (E, D, T)
    return (y * gates.T[:, None, :]).sum(0).T.to(_dtype(case))


# ---- one pass ------------------------------------------------------------------

def _run_own(state):
    nm, c = _package(), state["case"]
    kind = c["kind"]
    if kind == "quant":
        q, scale = nm.quantize_fp8(state["x"], square=c["square"])
        return {"q": q, "scale": scale}
    if kind == "product":
        return {"y": nm.matmul_fp8(state["a"], state["a_scale"], state["b"], state["b_scale"],
                                   state["bias"], dtype=_dtype(c))}
    if kind == "ffn":
        return {"y": state["layer"].forward_fp8(state["x"])}
    return {"y": state["layer"].forward_few(state["x"], state["idx"], state["w"], fp8=c["fp8"])}


def run(state):
    if own:
        return _run_own(state)
    c = state["case"]
    if c["kind"] == "quant":
        q, scale = _plain_quantize(state["x"], c["square"])
        return {"q": q, "scale": scale}
    if c["kind"] == "product":
        y = _plain_dequantize(state["a"], state["a_scale"], False) @ \
            _plain_dequantize(state["b"], state["b_scale"], True).T
        return {"y": (y if state["bias"] is None else y + state["bias"]).to(_dtype(c))}
    return {"y": (_plain_ffn if c["kind"] == "ffn" else _plain_few)(c, state)}


def work(case):
    kind, b = case["kind"], _dtype(case).itemsize
    if kind == "quant":
        T, K = case["rows"], case["cols"]
        scales = -(-K // BLOCK) * (-(-T // BLOCK) if case["square"] else T)
        return {"bytes": T * K * (b + 1) + 4 * scales, "flops": 3 * T * K}
    if kind == "product":
        M, K, N = case["rows"], case["k"], case["n"]
        kb = -(-K // BLOCK)
        return {"bytes": (M + N) * K + 4 * kb * (M + -(-N // BLOCK)) + M * N * b +
                (4 * N if case["bias"] else 0), "flops": 2 * M * N * K}
    T, D, H = case["rows"], case["dim"], case["hidden"]
    if kind == "ffn":
        return {"bytes": 3 * D * H + 2 * T * D * b + 4 * (2 * H + D), "flops": 6 * T * D * H}
    E, k = case["experts"], case["top_k"]
    dense = 1 if case["dense"] else 0
    live = min(E, T * k) + dense
    per = D * H * (1 if case["fp8"] else b)
    router = 0 if case["given"] else E * D * b
    return {"bytes": live * (3 * per + (2 * H + D) * b) + router + 2 * T * D * b +
            (8 * T * k if case["given"] else 0),
            "flops": 6 * T * (k + dense) * D * H + (0 if case["given"] else 2 * T * E * D)}


# ---- in 64 bits ------------------------------------------------------------------

def _nearest_e4m3(v):
    """The nearest of the type's values, counted through; in the middle of two the even one."""
    codes = torch.arange(127, dtype=torch.uint8, device=v.device)
    values = codes.view(torch.float8_e4m3fn).double()
    middles = (values[:-1] + values[1:]) / 2
    size = v.abs()
    below = torch.searchsorted(middles, size)  # middles that are smaller
    at = torch.searchsorted(middles, size, right=True)
    return torch.copysign(values[torch.where(at % 2 == 0, at, below)], v)


def _exact_blocks(x, square):
    """(values of the e4m3, scale of each element, scales) from the definition."""
    x = x.double()
    rows, cols = x.shape
    tall = BLOCK if square else 1
    padded = torch.nn.functional.pad(x.abs(), (0, -cols % BLOCK, 0, -rows % tall))
    top = torch.nn.functional.max_pool2d(padded[None, None], (tall, BLOCK))[0, 0]
    scale = torch.clamp(top / MOST, min=LEAST).float().double()
    each = torch.kron(scale, torch.ones(tall, BLOCK, dtype=torch.float64, device=x.device))
    each = each[:rows, :cols]
    return _nearest_e4m3(x / each), each, scale


def _exact_8_bit(x, square):
    q, each, _ = _exact_blocks(x, square)
    return q * each


def _exact_few(case, t):
    def weight(n, e):
        w = t[n][e].double()
        return _exact_8_bit(w, True) if case["fp8"] else w

    x, T, E = t["x"].double(), case["rows"], case["experts"]
    if case["given"]:
        idx, w = t["idx"].long(), t["w"].double()
    else:
        logits = torch.nn.functional.linear(x, t["router"].double())
        top = logits.topk(case["top_k"], dim=-1)
        p = torch.softmax(logits, -1).gather(1, top.indices)
        idx, w = top.indices, p / (p.sum(-1, keepdim=True) + ROUTE_EPS)
    y = torch.zeros_like(x)
    for e in range(E + (1 if case["dense"] else 0)):
        share = ((idx == e) * w).sum(-1, keepdim=True) if e < E else \
            torch.full((T, 1), case["dense"], dtype=torch.float64, device=x.device)
        f = torch.nn.functional
        a = f.linear(x, weight("gate.weight", e), t["gate.bias"][e].double())
        b = f.linear(x, weight("up.weight", e), t["up.bias"][e].double())
        y += share * f.linear(a * torch.sigmoid(a) * b, weight("down.weight", e),
                              t["down.bias"][e].double())
    return {"y": y}


def exact(case, seed):
    t, kind = _inputs(case, seed), case["kind"]
    if kind == "quant":
        q, _, scale = _exact_blocks(t["x"], case["square"])
        return {"q": q, "scale": scale}
    if kind == "product":
        def values(name, square):
            q, c = t[name].double(), t[name + "_scale"].double()
            each = torch.kron(c, torch.ones(BLOCK if square else 1, BLOCK, dtype=torch.float64,
                                            device=q.device))
            return q * each[:q.shape[0], :q.shape[1]]
        y = torch.nn.functional.linear(values("a", False), values("b", True))
        return {"y": y if t["bias"] is None else y + t["bias"].double()}
    if kind == "ffn":
        def linear(x, n):
            return torch.nn.functional.linear(_exact_8_bit(x, False),
                                              _exact_8_bit(t[n + ".weight"], True),
                                              t[n + ".bias"].double())
        a = linear(t["x"], "gate")
        return {"y": linear(a * torch.sigmoid(a) * linear(t["x"], "up"), "down")}
    return _exact_few(case, t)
