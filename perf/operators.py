"""The router and the seams of a DiT block's MoE half, as measurable calls.

A case is one call of one of these kinds:

* ``route``       scores, balance bias, groups, top-k and weights from a router's logits
* ``route_grad``  the gradient of the weights with respect to the logits
* ``experts``     an MoE layer's experts under a routing that the caller has
* ``seam``        what stands between two branches of a block: the norm after the
                  one, its gate, the (scaled) residual, and the modulated norm
                  before the next
* ``seam_grad``   the gradients of that seam

Logits are N(0, 1) with a spread of the experts' means, as a trained router has
them; the balance bias is small beside the scores.  ``padded`` is the share of
rows that are padding: every expert of theirs is masked (a logit of -inf).
Activations and their gradients are N(0, 1) with rows of different sizes,
modulation N(0, 0.3), norm gains near 1.
"""
import math
import os
import sys

import torch

own = False

PATH = "blocks.0.moe"
EPS = 1e-6        # of the norms
ROUTE_EPS = 1e-9  # of the renormalised weights
LINEARS = ("gate.weight", "gate.bias", "up.weight", "up.bias", "down.weight", "down.bias")


def _package():
    root = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))),
                        "hy-nomas-rs_amd")
    if root not in sys.path:
        sys.path.insert(0, root)
    import nomas_moe
    return nomas_moe


# ---- cases -------------------------------------------------------------------

def _route(name, kind, dtype, rows, experts, top_k, scoring, bias=True, groups=1, top_groups=1,
           group_top=2, renormalize=True, scale=1.0, padded=0.0):
    return {"name": name, "kind": kind, "dtype": dtype, "rows": rows, "experts": experts,
            "top_k": top_k, "scoring": scoring, "bias": bias, "groups": groups,
            "top_groups": top_groups, "group_top": group_top, "renormalize": renormalize,
            "scale": scale, "padded": padded}


def _experts(name, dtype, rows, dim, hidden, experts, top_k, padded=0.0):
    return {"name": name, "kind": "experts", "dtype": dtype, "rows": rows, "dim": dim,
            "hidden": hidden, "experts": experts, "top_k": top_k, "padded": padded}


def _seam(name, kind, dtype, batch, seq, dim, post=True, alpha=1.0):
    return {"name": name, "kind": kind, "dtype": dtype, "batch": batch, "seq": seq, "dim": dim,
            "post": post, "alpha": alpha}


def listed():
    return [
        # one new token of a causal session: a launch and a latency
        _route("route_token", "route", "f32", 1, 64, 8, "sigmoid", groups=8, top_groups=4,
               scale=2.5),
        # one branch of a turn (4,680 video and 64 text rows) through a softmax router
        # that leaves its logits in bf16, no balance bias
        _route("route_segment", "route", "bf16", 4744, 64, 8, "softmax", bias=False),
        # a training batch: many fine experts in groups, a balance bias, padded rows
        _route("route_batch", "route", "f32", 32768, 256, 8, "sigmoid", groups=8, top_groups=4,
               scale=2.5, padded=0.05),
        # the gradients of the same two
        _route("route_grad_segment", "route_grad", "bf16", 4744, 64, 8, "softmax", bias=False),
        _route("route_grad_batch", "route_grad", "f32", 32768, 256, 8, "sigmoid", groups=8,
               top_groups=4, scale=2.5, padded=0.05),
        # a handful of rows through a layer: its weights are streamed once
        _experts("experts_few", "bf16", 5, 1024, 2048, 16, 2),
        # one branch of a turn, some rows of it padding
        _experts("experts_segment", "bf16", 4744, 1024, 2048, 8, 2, padded=0.05),
        # a single token between two branches
        _seam("seam_token", "seam", "bf16", 1, 1, 2048),
        # three guidance branches stacked, modulation per branch
        _seam("seam_branches", "seam", "bf16", 3, 4744, 1536, alpha=0.5),
        # modulation per latent frame (each has its own noise level), no norm after the branch
        _seam("seam_frames", "seam", "f16", 12, 1560, 2560, post=False),
        # training on the three branches
        _seam("seam_grad_branches", "seam_grad", "bf16", 3, 4744, 1536, alpha=0.5),
        # f32 training at a width that no tile divides, ragged rows
        _seam("seam_grad_f32", "seam_grad", "f32", 2, 2999, 1000),
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["route", "route", "route", "route_grad", "route_grad", "experts", "seam",
                       "seam", "seam", "seam_grad", "seam_grad", "seam_grad"])
    dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
    padded = rng.choice([0.0, 0.0, 0.02, 0.2])
    if kind in ("route", "route_grad"):
        groups = rng.choice([1, 1, 1, 2, 4, 6, 8])
        experts = groups * _log_int(rng, 4, 512 // groups)
        top_groups = rng.randint(1, groups)
        top_k = min(rng.choice([1, 2, 4, 6, 8, 8, 16]), experts // groups * top_groups)
        case = _route("", kind, dtype, _log_int(rng, 1, 32768 * 256 // max(experts, 256)), experts,
                      top_k, rng.choice(["softmax", "sigmoid"]), rng.random() < 0.6, groups,
                      top_groups, rng.choice([1, 2]), rng.random() < 0.8,
                      rng.choice([1.0, 1.0, 2.5]), padded)
    elif kind == "experts":
        experts = rng.choice([4, 8, 16, 32])
        dim, hidden = 8 * _log_int(rng, 8, 128), _log_int(rng, 64, 2048)
        while experts * dim * hidden > 8 * 1024 * 2048:
            experts //= 2
        top_k = min(experts, rng.choice([1, 2, 2, 4]))
        # widths that no tile divides run on padded ones, f32 on six products
        slow = (4 if dtype == "f32" else 1) * (2 if dim % 256 or hidden % 128 else 1)
        most = 4744 * 2 * 1024 * 2048 // (slow * top_k * dim * hidden)
        case = _experts("", dtype, _log_int(rng, 1, max(1, min(8192, most))), dim, hidden, experts,
                        top_k, padded)
    else:
        dim = 8 * _log_int(rng, 8, 512)
        batch = _log_int(rng, 1, 16)
        passes = (4 if kind == "seam" else 6) * (4 if dtype == "f32" else 2)
        most = 8 * 12 * 1560 * 2560 // (passes * dim * batch)
        case = _seam("", kind, dtype, batch, _log_int(rng, 1, max(1, min(8192, most))), dim,
                     rng.random() < 0.6, rng.choice([1.0, 1.0, 0.5]))
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


def _padding(g, case):
    return torch.rand(case["rows"], generator=g, device="cuda") < case["padded"]


def _route_inputs(case, seed):
    g = _generator(seed)
    T, E = case["rows"], case["experts"]
    logits = _randn(g, T, E) + _randn(g, E, std=0.5)
    logits[_padding(g, case)] = -math.inf
    s = {"logits": logits.to(_dtype(case)), "bias": None}
    if case["bias"]:
        s["bias"] = _randn(g, E, std=0.05 if case["scoring"] == "sigmoid" else 0.2 / E)
    if case["kind"] == "route_grad":
        # the routing that the forward pass left, and the gradient of its weights
        s["idx"] = _plain_route(case, s["logits"], s["bias"])["idx"]
        s["dw"] = _randn(g, T, case["top_k"])
    return s


def _expert_inputs(case, seed):
    g = _generator(seed)
    dt = _dtype(case)
    T, D, H, E, k = (case[n] for n in ("rows", "dim", "hidden", "experts", "top_k"))
    s = {"x": _randn(g, T, D, to=dt)}
    order = _randn(g, T, E).argsort(-1)[:, :k].sort(-1).values
    w = torch.softmax(_randn(g, T, k), -1)
    pad = _padding(g, case)[:, None]
    s["idx"] = torch.where(pad, -1, order).to(torch.int32)
    s["w"] = torch.where(pad, 0.0, w)
    for name, shape, std in (("gate.weight", (H, D), D ** -0.5), ("gate.bias", (H,), 0.1),
                             ("up.weight", (H, D), D ** -0.5), ("up.bias", (H,), 0.1),
                             ("down.weight", (D, H), H ** -0.5), ("down.bias", (D,), 0.1)):
        s[name] = _randn(g, E, *shape, std=std, to=dt)
    return s


def _seam_inputs(case, seed):
    g = _generator(seed)
    dt = _dtype(case)
    B, S, D = case["batch"], case["seq"], case["dim"]

    def rows():
        return (_randn(g, B, S, D) * torch.exp(_randn(g, B, S, 1, std=0.3))).to(dt)

    names = ("x", "y") if case["kind"] == "seam" else ("out", "y", "dout", "dh")
    s = {n: rows() for n in names}
    for n in ("gate", "shift", "scale"):
        s[n] = _randn(g, B, D, std=0.3)
    s["norm_w"] = _randn(g, D, std=0.1, mean=1.0)
    s["post_w"] = _randn(g, D, std=0.1, mean=1.0) if case["post"] else None
    return s


def _inputs(case, seed):
    kind = case["kind"]
    return (_route_inputs if kind in ("route", "route_grad") else
            _expert_inputs if kind == "experts" else _seam_inputs)(case, seed)


def prepare(case, seed):
    state = _inputs(case, seed)
    state["case"] = case
    if own and case["kind"] == "experts":  # the layer that a program keeps
        nm = _package()
        dt = nm.DataType.of(case["dtype"])
        host = {n: state[n].float().cpu().numpy() for n in LINEARS}
        E, D, H = case["experts"], case["dim"], case["hidden"]
        named = {f"{PATH}.experts.{e}.{n}": host[n][e] for n in LINEARS for e in range(E)}
        # the layer's own router is not used
        named[f"{PATH}.router.weight"] = torch.zeros(E, D).numpy()
        state["layer"] = nm.MoeLayer.from_source(nm.Weights.tensors_(named, dt), PATH, D, H,
                                                 nm.MoeConfig(E, case["top_k"]))
    return state


# ---- the plain forms -----------------------------------------------------------

def _scores(logits, scoring):
    """Scores in 64 bits (equal or not next to the border of the choice); 0 where masked."""
    l = logits.double()
    masked = l == -math.inf
    if scoring == "sigmoid":
        s = 1.0 / (1.0 + torch.exp(-l))
    else:
        e = torch.exp(l - l.amax(-1, keepdim=True))
        s = e / e.sum(-1, keepdim=True)
    return torch.where(masked, 0.0, s), masked


def _plain_route(case, logits, bias):
    T, E = logits.shape
    k, G = case["top_k"], case["groups"]
    s, masked = _scores(logits, case["scoring"])
    key = s if bias is None else s + bias.double()
    if bias is None and G == 1:
        key = logits.double()  # the same order
    key = torch.where(masked, -math.inf, key)
    if G > 1:
        best = key.view(T, G, E // G).sort(-1, descending=True).values[..., :case["group_top"]]
        score = torch.where(best == -math.inf, 0.0, best).sum(-1)
        score = torch.where(best[..., 0] == -math.inf, -math.inf, score)
        order = score.sort(dim=-1, descending=True, stable=True).indices[:, :case["top_groups"]]
        keep = torch.zeros(T, G, dtype=torch.bool, device=key.device).scatter_(1, order, True)
        key = torch.where(keep.repeat_interleave(E // G, 1), key, -math.inf)
    top = key.sort(dim=-1, descending=True, stable=True)
    idx = torch.where(top.values[:, :k] == -math.inf, E, top.indices[:, :k]).sort(-1).values
    none = idx == E
    sel = torch.where(none, 0.0, s.gather(1, idx.clamp(max=E - 1)))
    w = sel / (sel.sum(-1, keepdim=True) + ROUTE_EPS) if case["renormalize"] else sel
    counts = torch.zeros(E + 1, dtype=torch.int32, device=key.device).index_add_(
        0, idx.reshape(-1), torch.ones(T * k, dtype=torch.int32, device=key.device))[:E]
    return {"idx": torch.where(none, -1, idx).to(torch.int32),
            "w": (w * case["scale"]).float(), "counts": counts}


def _plain_route_grad(case, logits, idx, dw):
    E = logits.shape[1]
    s, _ = _scores(logits, case["scoring"])
    at = torch.where(idx < 0, E, idx).long()
    padded = torch.cat([s, torch.zeros_like(s[:, :1])], 1)
    sel, d = padded.gather(1, at), dw.double()
    if case["renormalize"]:
        total = sel.sum(-1, keepdim=True) + ROUTE_EPS
        d = (d - (d * sel).sum(-1, keepdim=True) / total) / total
    ds = torch.zeros_like(padded).scatter_(1, at, d * case["scale"])[:, :E]
    if case["scoring"] == "sigmoid":
        dl = ds * s * (1.0 - s)
    else:
        dl = s * (ds - (s * ds).sum(-1, keepdim=True))
    return torch.where(logits == -math.inf, 0.0, dl).to(logits.dtype)


def _plain_experts(state, E, wide):
    x, idx, w = state["x"].to(wide), state["idx"], state["w"].to(wide)
    y = torch.zeros_like(x)
    for e in range(E):
        at, slot = torch.nonzero(idx == e, as_tuple=True)
        r = x[at]
        g = r @ state["gate.weight"][e].to(wide).T + state["gate.bias"][e].to(wide)
        u = r @ state["up.weight"][e].to(wide).T + state["up.bias"][e].to(wide)
        o = (g / (1.0 + torch.exp(-g)) * u) @ state["down.weight"][e].to(wide).T + \
            state["down.bias"][e].to(wide)
        y.index_add_(0, at, o * w[at, slot, None])
    return y


def _rms(v):
    return v * torch.rsqrt(v.square().mean(-1, keepdim=True) + EPS)


def _plain_seam(case, s):
    dt = _dtype(case)
    y = s["y"].float()
    n = _rms(y) * s["post_w"] if case["post"] else y
    out = case["alpha"] * s["x"].float() + s["gate"][:, None] * n
    h = _rms(out) * s["norm_w"] * (1.0 + s["scale"][:, None]) + s["shift"][:, None]
    return {"out": out.to(dt), "h": h.to(dt)}


def _plain_seam_grad(case, s):
    dt = _dtype(case)
    out, y, dout, dh = (s[n].float() for n in ("out", "y", "dout", "dh"))
    r = torch.rsqrt(out.square().mean(-1, keepdim=True) + EPS)
    unit = out * r
    g = dh * (1.0 + s["scale"][:, None]) * s["norm_w"]
    d = dout + r * (g - unit * (g * unit).mean(-1, keepdim=True))
    q = (dh * unit).sum(1)
    got = {"dx": (case["alpha"] * d).to(dt), "dshift": dh.sum(1), "dscale": q * s["norm_w"],
           "dnorm_w": (q * (1.0 + s["scale"])).sum(0)}
    dn = d * s["gate"][:, None]
    if case["post"]:
        ry = torch.rsqrt(y.square().mean(-1, keepdim=True) + EPS)
        yn = y * ry
        gy = dn * s["post_w"]
        got["dy"] = (ry * (gy - yn * (gy * yn).mean(-1, keepdim=True))).to(dt)
        p = (d * yn).sum(1)
        got["dgate"] = p * s["post_w"]
        got["dpost_w"] = (p * s["gate"]).sum(0)
    else:
        got["dy"] = dn.to(dt)
        got["dgate"] = (d * y).sum(1)
    return got


# ---- one pass ------------------------------------------------------------------

def _run_own(state):
    nm, c = _package(), state["case"]
    kind = c["kind"]
    if kind == "route":
        idx, w, counts = nm.route(
            state["logits"], c["top_k"], scoring=c["scoring"], bias=state["bias"],
            groups=c["groups"], top_groups=c["top_groups"], group_top=c["group_top"],
            renormalize=c["renormalize"], scale=c["scale"], eps=ROUTE_EPS)
        return {"idx": idx, "w": w, "counts": counts}
    if kind == "route_grad":
        return {"dlogits": nm.route_backward(
            state["logits"], state["idx"], state["dw"], scoring=c["scoring"],
            renormalize=c["renormalize"], scale=c["scale"], eps=ROUTE_EPS)}
    if kind == "experts":
        return {"y": state["layer"].forward_routed(state["x"], state["idx"], state["w"])}
    if kind == "seam":
        out, h = nm.block_seam(state["x"], state["y"], state["gate"], state["shift"],
                               state["scale"], post_norm=c["post"], post_w=state["post_w"],
                               norm_w=state["norm_w"], residual_scale=c["alpha"], eps=EPS)
        return {"out": out, "h": h}
    return nm.block_seam_backward(
        state["dout"], state["dh"], state["out"], state["y"], state["gate"], state["scale"],
        post_norm=c["post"], post_w=state["post_w"], norm_w=state["norm_w"],
        residual_scale=c["alpha"], eps=EPS)


def run(state):
    if own:
        return _run_own(state)
    c = state["case"]
    kind = c["kind"]
    if kind == "route":
        return _plain_route(c, state["logits"], state["bias"])
    if kind == "route_grad":
        return {"dlogits": _plain_route_grad(c, state["logits"], state["idx"], state["dw"])}
    if kind == "experts":
        return {"y": _plain_experts(state, c["experts"], torch.float32).to(state["x"].dtype)}
    return _plain_seam(c, state) if kind == "seam" else _plain_seam_grad(c, state)


def work(case):
    kind, b = case["kind"], _dtype(case).itemsize
    if kind in ("route", "route_grad"):
        T, E, k = case["rows"], case["experts"], case["top_k"]
        if kind == "route":
            # the logits and the bias; indices, weights and counts
            return {"bytes": T * E * b + 8 * T * k + 4 * E * (2 if case["bias"] else 1),
                    "flops": 10 * T * E}
        # the logits (sigmoid: the chosen ones), indices and weights' gradients; dlogits
        read = T * E if case["scoring"] == "softmax" else T * k
        return {"bytes": read * b + 8 * T * k + T * E * b, "flops": 10 * T * E}
    if kind == "experts":
        T, D, H, E, k = (case[n] for n in ("rows", "dim", "hidden", "experts", "top_k"))
        live = min(E, T * k)
        return {"bytes": b * (2 * T * D + live * (3 * D * H + 2 * H + D)) + 8 * T * k,
                "flops": 6 * T * k * D * H}
    B, S, D = case["batch"], case["seq"], case["dim"]
    gains = 4 * D * (2 if case["post"] else 1)
    if kind == "seam":
        return {"bytes": 4 * B * S * D * b + 3 * 4 * B * D + gains, "flops": 16 * B * S * D}
    return {"bytes": 6 * B * S * D * b + 5 * 4 * B * D + 2 * gains, "flops": 40 * B * S * D}


# ---- in 64 bits ------------------------------------------------------------------

def _exact_route(case, t):
    """Row by row on the host: the definition, spelled out (the first rows of a large case)."""
    import numpy as np
    l = t["logits"].double().cpu().numpy()
    bias = None if t["bias"] is None else t["bias"].double().cpu().numpy()
    T, E = l.shape
    G, k = case["groups"], case["top_k"]
    w = np.zeros((T, k))
    for r in range(T):
        live = np.nonzero(l[r] > -np.inf)[0]
        if not live.size:
            continue
        s = np.zeros(E)
        if case["scoring"] == "sigmoid":
            s[live] = 0.5 * (1.0 + np.tanh(0.5 * l[r, live]))
        else:
            s[live] = np.exp(l[r, live] - np.logaddexp.reduce(l[r, live]))
        rank = l[r] if bias is None and G == 1 else s if bias is None else s + bias
        pool = live
        if G > 1:
            worth = []
            for g in range(G):
                c = np.sort(rank[live[live // (E // G) == g]])[::-1][:case["group_top"]]
                worth.append((-c.sum() if c.size else np.inf, g))
            kept = [g for _, g in sorted(worth)[:case["top_groups"]]]
            pool = live[np.isin(live // (E // G), kept)]
        sel = np.sort(pool[np.lexsort((pool, -rank[pool]))][:k])
        v = s[sel]
        w[r, :sel.size] = case["scale"] * (v / (v.sum() + ROUTE_EPS) if case["renormalize"] else v)
    return {"idx": None, "w": torch.from_numpy(w), "counts": None}


def _exact_route_grad(case, t):
    """The gradient that torch's own differentiation gives of the weights in 64 bits."""
    live = t["logits"] > -math.inf
    l = torch.where(live, t["logits"].double(), -1e4).requires_grad_(True)
    s = torch.sigmoid(l) if case["scoring"] == "sigmoid" else torch.softmax(l, -1)
    s = torch.where(live, s, torch.zeros_like(s))
    some = t["idx"] >= 0
    v = torch.where(some, s.gather(1, t["idx"].clamp(min=0).long()), torch.zeros((), device="cuda",
                                                                             dtype=s.dtype))
    w = v / (v.sum(-1, keepdim=True) + ROUTE_EPS) if case["renormalize"] else v
    (case["scale"] * w * t["dw"].double()).sum().backward()
    return {"dlogits": torch.where(live, l.grad, torch.zeros_like(l.grad))}


def _exact_experts(case, t):
    gates = torch.zeros(case["rows"], case["experts"] + 1, dtype=torch.float64, device="cuda")
    at = torch.where(t["idx"] < 0, case["experts"], t["idx"]).long()
    gates.scatter_add_(1, at, t["w"].double())
    x, y = t["x"].double(), 0.0
    for e in range(case["experts"]):  # every expert on every row, weighed by its gate
        a = torch.nn.functional.linear(x, t["gate.weight"][e].double(), t["gate.bias"][e].double())
        b = torch.nn.functional.linear(x, t["up.weight"][e].double(), t["up.bias"][e].double())
        o = torch.nn.functional.linear(a * torch.sigmoid(a) * b, t["down.weight"][e].double(),
                                       t["down.bias"][e].double())
        y = y + gates[:, e, None] * o
    return {"y": y}


def _exact_branch(case, y, post_w):
    if not case["post"]:
        return y
    return y / (y.square().mean(-1, keepdim=True) + EPS).sqrt() * post_w


def _exact_modulated(out, norm_w, shift, scale):
    unit = out / (out.square().mean(-1, keepdim=True) + EPS).sqrt()
    return unit * norm_w * (1.0 + scale[:, None]) + shift[:, None]


def _exact_seam(case, t):
    d = {k: None if v is None else v.double() for k, v in t.items()}
    out = case["alpha"] * d["x"] + d["gate"][:, None] * _exact_branch(case, d["y"], d["post_w"])
    return {"out": out, "h": _exact_modulated(out, d["norm_w"], d["shift"], d["scale"])}


def _exact_seam_grad(case, t):
    """torch's own differentiation: of h with respect to out, then of out with respect to the rest."""
    d = {k: None if v is None else v.double() for k, v in t.items()}
    leaf = {k: d[k].requires_grad_(True) for k in ("out", "y", "gate", "shift", "scale", "norm_w")}
    if case["post"]:
        leaf["post_w"] = d["post_w"].requires_grad_(True)
    h = _exact_modulated(leaf["out"], leaf["norm_w"], leaf["shift"], leaf["scale"])
    (h * d["dh"]).sum().backward()
    total = d["dout"] + leaf["out"].grad
    branch = leaf["gate"][:, None] * _exact_branch(case, leaf["y"], leaf.get("post_w"))
    (branch * total).sum().backward()
    got = {"d" + k: leaf[k].grad for k in leaf if k != "out"}
    got["dx"] = case["alpha"] * total
    return got


def exact(case, seed):
    t = _inputs(case, seed)
    kind = case["kind"]
    return {"route": _exact_route, "route_grad": _exact_route_grad, "experts": _exact_experts,
            "seam": _exact_seam, "seam_grad": _exact_seam_grad}[kind](case, t)
