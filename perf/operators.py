"""The mixture-of-experts operators as cases to time: the router that picks each token's experts (`route`), and the
products of the rows with the block-quantised weights of the experts they were sent to - gate and up with SwiGLU on the
way in (`up`, matmul_experts), down with the weighted sum over a token's experts on the way out (`down`,
matmul_experts_sum) - plus the three in a row, as a layer runs them (`layer`).

Where `own` is false `run` computes the definitions with elementary torch operations in fp32 (the router in fp64: which
of two experts is chosen hangs on their last bits); where it is true it makes the calls of cyb_amd.Backend.

A stack of E experts is one quantised tensor of E * n rows, expert e = rows [e * n, (e + 1) * n); `gate` and `up` are
two such stacks, fused strip by strip for the library.  ids[t, j] is the j-th expert of token t, -1 for none (the rows of
a padded batch): such a row of `up` is left as it was (zeros here), in `down` it adds nothing.
"""
import math

import numpy as np
import torch

own = False

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZE = {"f32": 4, "f16": 2, "bf16": 2}


def _route(**kw):
    return dict({"kind": "route", "T": 1, "E": 128, "k": 8, "logits": "f32", "score": "softmax", "bias": False, "groups": 1,
                 "top_groups": 1, "group_best": 1, "renorm": True, "scale": 1.0}, **kw)


def _experts(kind, **kw):
    return dict({"kind": kind, "bits": 4, "T": 1, "E": 128, "k": 8, "hidden": 2048, "width": 768, "x": "f16", "y": "f16",
                 "pad": 0}, **kw)


def listed():
    return [
        # one token of one conversation on a model of many narrow experts: each of the three steps by itself, where
        # latency counts
        _route(name="route_token"),
        _experts("up", name="up_token"),
        _experts("down", name="down_token", y="f32"),
        # the three in a row for a few conversations at once, the router's products given
        _experts("layer", name="layer_tokens_4", T=4),
        # an odd number of experts in groups, sigmoid scores and a balancing bias, half-precision scores: a batch being decoded
        _route(name="route_batch_48", T=48, E=160, k=6, logits="bf16", score="sigmoid", bias=True, groups=8, top_groups=3),
        # a long prompt's routing: sigmoid scores, a balancing bias, the best four of eight groups by their two best experts
        _route(name="route_prompt_8192", T=8192, E=256, score="sigmoid", bias=True, groups=8, top_groups=4, group_best=2, scale=2.5),
        # few wide experts, a batch of conversations: a few rows for every expert
        _experts("up", name="up_batch_16", T=16, E=8, k=2, hidden=4096, width=14336, x="bf16", y="bf16"),
        _experts("down", name="down_batch_32", T=32, E=8, k=2, hidden=4096, width=14336),
        # Q8 experts of odd sizes, drafted tokens, the last rows of the batch padding
        _experts("up", name="up_draft_37_q8", bits=8, T=37, E=60, k=4, hidden=2592, width=1040, y="f32", pad=5),
        # a prompt being read: a couple of hundred rows for every narrow expert
        _experts("up", name="up_prompt_2048", T=2048, x="bf16", y="bf16"),
        _experts("down", name="down_prompt_2048", T=2048, x="bf16", y="bf16"),
        # the largest: a prompt chunk on the wide experts
        _experts("up", name="up_prompt_1024_wide", T=1024, E=8, k=2, hidden=4096, width=14336, x="bf16", y="bf16"),
    ]


def _log(rng, lo, hi, step=1):
    """A multiple of `step` between lo and hi, even over the logarithm."""
    v = lo * (hi / lo) ** rng.random()
    return int(max(-(-lo // step), min(hi // step, round(v / step))) * step)


def _divisors(n, most):
    return [d for d in range(1, most + 1) if n % d == 0]


def draw(rng):
    kind = rng.choice(["route", "up", "up", "down", "down", "layer"])
    E = rng.choice([8, 16, 60, 64, 128, 160, 256, rng.randint(4, 256)])
    k = min(E, rng.choice([1, 2, 4, 6, 8, 8]))
    T = rng.choice([1, rng.randint(2, 16), _log(rng, 17, 4096), _log(rng, 17, 4096)])
    if kind == "route":
        groups = rng.choice([1, rng.choice(_divisors(E, 16))])
        per = E // groups
        top = rng.randint(-(-k // per), groups)
        return _route(T=rng.choice([T, _log(rng, 1, 8192)]), E=E, k=k, logits=rng.choice(["f32", "f32", "f16", "bf16"]),
                      score=rng.choice(["softmax", "sigmoid"]), bias=rng.random() < 0.5, groups=groups, top_groups=top,
                      group_best=rng.choice([1, 2]), renorm=rng.random() < 0.7, scale=rng.choice([1.0, 1.0, 2.5]))
    bits = rng.choice([4, 4, 8])
    # no more weights, and no more multiplications, than the largest listed case has
    stacks = {"up": 2, "down": 1, "layer": 3}[kind]
    most = 9.3e8 * 4 / bits / (stacks * E)
    hidden = _log(rng, 512, min(4096, most / 256), 32)
    width = _log(rng, 256, min(14336, max(256, most / hidden)), 32)
    T = max(1, min(T, int(2.4e11 / (k * hidden * width * stacks))))
    x = rng.choice(["f16", "bf16", "f32"]) if T <= 64 else rng.choice(["f16", "bf16", "bf16"])
    return _experts(kind, bits=bits, T=T, E=E, k=k, hidden=hidden, width=width, x=x,
                    y=x if kind == "layer" else rng.choice([x, x, "f32"]), pad=rng.choice([0, 0, rng.randint(0, T - 1)]))


# ---- inputs -------------------------------------------------------------------------------------------------

def _gen(seed, what):
    g = torch.Generator(device="cuda")
    g.manual_seed((seed * 1000003 + what) & 0x7FFFFFFF)
    return g


def _randn(shape, gen, std=1.0):
    return torch.empty(shape, dtype=torch.float32, device="cuda").normal_(0.0, std, generator=gen)


def _logits(case, seed):
    """Router outputs: every token has its own taste, some experts are liked more than others."""
    g = _gen(seed, 1)
    z = _randn((case["T"], case["E"]), g, 1.5) + _randn((1, case["E"]), g, 0.3)
    return z.to(TYPES[case.get("logits", "f32")])


def _planes(case, n, K, gen):
    """A stack of E experts of n rows as it comes from an import: (q, scales) in the PLANAR layout, weights of N(0, 0.02)
    seen through their quantisation (the largest of a group of 32 at the end of the range)."""
    E, bits = case["E"], case["bits"]
    q = torch.empty((E, n, K * bits // 8), dtype=torch.uint8, device="cuda")
    for e in range(E):
        w = _randn((n, K), gen, 3.2 if bits == 4 else 56.0)
        if bits == 4:
            w = w.round_().clamp_(-8, 7).to(torch.int8)
            q[e] = (w[:, 0::2] & 15 | (w[:, 1::2] << 4)).view(torch.uint8)
        else:
            q[e] = w.round_().clamp_(-127, 127).to(torch.int8).view(torch.uint8)
    s = (_randn((E, n, K // 32), gen, 0.1) + 1.0).clamp_(0.5, 1.5) * (0.0063 if bits == 4 else 0.00036)
    return q, s.to(torch.float16)


def _ids(case, seed):
    """Distinct experts per token, the tokens of the padding with none."""
    top = _logits(case, seed).argsort(dim=1, descending=True)[:, :case["k"]].to(torch.int32)
    if case["pad"]:
        top[case["T"] - case["pad"]:] = -1
    return top.contiguous()


def _inputs(case, seed):
    if case["kind"] == "route":
        return {"logits": _logits(case, seed), "bias": _randn((case["E"],), _gen(seed, 2), 0.05) if case["bias"] else None}
    T, k, hidden, width, kind = case["T"], case["k"], case["hidden"], case["width"], case["kind"]
    s = {}
    if kind != "down":
        g = _gen(seed, 3)
        s["gate"], s["up"] = _planes(case, width, hidden, g), _planes(case, width, hidden, g)
        s["x"] = _randn((T, hidden), _gen(seed, 4)).to(TYPES[case["x"]])
    else:
        # what SwiGLU leaves: mostly small, a few large
        g = _gen(seed, 5)
        a = _randn((T * k, width), g)
        s["x"] = (a * torch.sigmoid(a) * _randn((T * k, width), g)).to(TYPES[case["x"]])
    if kind != "up":
        s["down"] = _planes(case, hidden, width, _gen(seed, 6))
        s["residual"] = _randn((T, hidden), _gen(seed, 7)).to(TYPES[case["y"]])
    if kind == "layer":
        s["logits"] = _logits(case, seed)
        if case["pad"]:                     # a padded batch: the router sees the real tokens alone
            s["logits"] = s["logits"][:T - case["pad"]].contiguous()
    else:
        s["ids"] = _ids(case, seed)
        if kind == "down":
            w = torch.rand((T, k), generator=_gen(seed, 8), device="cuda") + 0.05
            s["weights"] = w / w.sum(dim=1, keepdim=True)
    return s


_backend = None


def _library():
    """One context for the life of the process, as a runtime keeps it."""
    global _backend
    if _backend is None:
        from cyb_amd import Backend
        torch.cuda.init()
        _backend = Backend(0)
    return _backend


def _weight(case, planes, n, K):
    q, s = planes
    w = _library().weight_from_device(case["bits"], case["E"] * n, K, q, s)
    torch.cuda.synchronize()
    return w


def prepare(case, seed):
    """The inputs, the buffers that a program keeps for results and - the library's - the weight handles."""
    st = {"case": case, "in": _inputs(case, seed)}
    T, kind = case["T"], case["kind"]
    st["real"] = T
    if kind == "layer":
        st["real"] = T - case["pad"]
    if kind in ("route", "layer"):
        st["ids"] = torch.full((T, case["k"]), -1, dtype=torch.int32, device="cuda")
        st["weights"] = torch.zeros((T, case["k"]), dtype=torch.float32, device="cuda")
        st["chosen"] = st["ids"][:st["real"]], st["weights"][:st["real"]]
    if kind in ("up", "layer"):
        st["h"] = torch.zeros((T * case["k"], case["width"]), dtype=TYPES[case["x"] if kind == "layer" else case["y"]], device="cuda")
    if kind in ("down", "layer"):
        st["y"] = torch.zeros((T, case["hidden"]), dtype=TYPES[case["y"]], device="cuda")
    if own:
        be = _library()
        if kind in ("up", "layer"):
            g = _weight(case, st["in"]["gate"], case["width"], case["hidden"])
            u = _weight(case, st["in"]["up"], case["width"], case["hidden"])
            st["gate_up"] = be.fuse_pairs(g, u)
            g.free()
            u.free()
        if kind in ("down", "layer"):
            st["down"] = _weight(case, st["in"]["down"], case["hidden"], case["width"])
    torch.cuda.synchronize()
    return st


# ---- the library's calls ------------------------------------------------------------------------------------

def _own(st):
    case, a = st["case"], st["in"]
    be, kind, E = _library(), case["kind"], case["E"]
    if kind == "route":
        be.route(a["logits"], st["ids"], st["weights"], score=case["score"], bias=a["bias"], groups=case["groups"],
                 top_groups=case["top_groups"], group_best=case["group_best"], renormalise=case["renorm"], scale=case["scale"])
        return st["ids"], st["weights"]
    if kind == "up":
        be.matmul_experts(st["gate_up"], E, a["x"], a["ids"], st["h"], "swiglu")
        return st["h"]
    if kind == "down":
        be.matmul_experts_sum(st["down"], E, a["x"], a["ids"], a["weights"], st["y"], a["residual"])
        return st["y"]
    be.route(a["logits"], *st["chosen"])
    be.matmul_experts(st["gate_up"], E, a["x"], st["ids"], st["h"], "swiglu")
    be.matmul_experts_sum(st["down"], E, st["h"], st["ids"], st["weights"], st["y"], a["residual"])
    return st["y"], st["ids"], st["weights"]


# ---- the plain form -----------------------------------------------------------------------------------------

def _plain_weight(planes, bits, e):
    q, s = planes[0][e], planes[1][e]
    if bits == 4:
        v = torch.stack((q & 15, q >> 4), dim=2).reshape(q.shape[0], -1).to(torch.float32)
        v = torch.where(v >= 8, v - 16, v)
    else:
        v = q.view(torch.int8).to(torch.float32)
    n, K = v.shape
    return (v.reshape(n, K // 32, 32) * s.to(torch.float32).reshape(n, K // 32, 1)).reshape(n, K)


def _plain_route(logits, case):
    k, E = case["k"], case["E"]
    z = logits.to(torch.float64)
    if case.get("score", "softmax") == "softmax":
        s = torch.exp(z - z.max(dim=1, keepdim=True).values)
        s = s / s.sum(dim=1, keepdim=True)
    else:
        s = 1.0 / (1.0 + torch.exp(-z))
    bias, groups = case.get("bias_values"), case.get("groups", 1)
    choice = z if bias is None else s + bias.to(torch.float64)      # (without a bias scores are in the order of their logits)
    if groups > 1:
        c = (s if bias is None else choice).reshape(-1, groups, E // groups)
        best = c.sort(dim=2, descending=True, stable=True).values[:, :, :case["group_best"]].sum(dim=2)
        keep = best.sort(dim=1, descending=True, stable=True).indices[:, :case["top_groups"]]
        kept = torch.zeros_like(best, dtype=torch.bool).scatter_(1, keep, True)
        choice = torch.where(kept.repeat_interleave(E // groups, dim=1), choice, -math.inf)
    ids = choice.sort(dim=1, descending=True, stable=True).indices[:, :k]
    w = s.gather(1, ids)
    if case.get("renorm", True):
        w = w / w.sum(dim=1, keepdim=True)
    return ids.to(torch.int32), (w * case.get("scale", 1.0)).to(torch.float32)


def _plain_up(case, a, ids, out):
    flat = ids.reshape(-1)
    x = a["x"].to(torch.float32)
    for e in torch.unique(flat).tolist():
        if e < 0:
            continue
        pairs = torch.nonzero(flat == e).reshape(-1)
        rows = x[pairs // case["k"]]
        g = rows @ _plain_weight(a["gate"], case["bits"], e).T
        u = rows @ _plain_weight(a["up"], case["bits"], e).T
        out[pairs] = (g / (1.0 + torch.exp(-g)) * u).to(out.dtype)
    return out


def _plain_down(case, a, x, ids, weights, out):
    flat = ids.reshape(-1)
    z = torch.zeros((flat.numel(), case["hidden"]), dtype=torch.float32, device="cuda")
    for e in torch.unique(flat).tolist():
        if e < 0:
            continue
        pairs = torch.nonzero(flat == e).reshape(-1)
        z[pairs] = x[pairs].to(torch.float32) @ _plain_weight(a["down"], case["bits"], e).T
    z = (z * weights.reshape(-1, 1)).reshape(case["T"], case["k"], -1).sum(dim=1)
    out.copy_((a["residual"].to(torch.float32) + z).to(out.dtype))
    return out


def _plain(st):
    case, a, kind = st["case"], st["in"], st["case"]["kind"]
    if kind == "route":
        return _plain_route(a["logits"], dict(case, bias_values=a["bias"]))
    if kind == "up":
        return _plain_up(case, a, a["ids"], st["h"])
    if kind == "down":
        return _plain_down(case, a, a["x"], a["ids"], a["weights"], st["y"])
    ids, w = _plain_route(a["logits"], case)
    st["ids"][:st["real"]], st["weights"][:st["real"]] = ids, w
    h = _plain_up(case, a, st["ids"], st["h"])
    return _plain_down(case, a, h, st["ids"], st["weights"], st["y"]), st["ids"], st["weights"]


def run(state):
    return _own(state) if own else _plain(state)


# ---- work ---------------------------------------------------------------------------------------------------

def work(case):
    T, E, k = case["T"], case["E"], case["k"]
    route = {"bytes": T * E * SIZE[case.get("logits", "f32")] + T * k * 8 + (E * 4 if case.get("bias") else 0), "flops": T * E * 8}
    if case["kind"] == "route":
        return route
    real, hidden, width = T - case["pad"], case["hidden"], case["width"]
    pairs = real * k
    met = E * (1.0 - (1.0 - k / E) ** real)                       # experts that some token is sent to
    one = hidden * width * case["bits"] // 8 + hidden * width // 32 * 2
    up = {"bytes": met * 2 * one + real * hidden * SIZE[case["x"]] + pairs * width * SIZE[case["x" if case["kind"] == "layer" else "y"]] + pairs * 4,
          "flops": pairs * hidden * width * 4}
    down = {"bytes": met * one + pairs * width * SIZE[case["x"]] + (real + T) * hidden * SIZE[case["y"]] + pairs * 8,
            "flops": pairs * hidden * width * 2 + pairs * hidden * 2}
    if case["kind"] == "layer":       # (the rows between the two products need not leave the chip, nor the ids)
        both = up["bytes"] + down["bytes"] - 2 * pairs * width * SIZE[case["x"]] - pairs * 12
        return {"bytes": int(both + route["bytes"]), "flops": up["flops"] + down["flops"] + route["flops"]}
    w = up if case["kind"] == "up" else down
    return {"bytes": int(w["bytes"]), "flops": int(w["flops"])}


# ---- the definition in 64 bits ------------------------------------------------------------------------------

def _exact_route(logits, case, bias):
    z = logits.double().cpu().numpy()
    k, E, T = case["k"], case["E"], logits.shape[0]
    if case.get("score", "softmax") == "softmax":
        s = np.exp(z - z.max(axis=1)[:, None])
        s /= s.sum(axis=1)[:, None]
    else:
        s = 1.0 / (1.0 + np.exp(-z))
    c = s + bias.double().cpu().numpy() if bias is not None else s
    rank = c if bias is not None else z
    groups = case.get("groups", 1)
    allowed = np.ones((T, E), dtype=bool)
    if groups > 1:
        per = np.sort(c.reshape(T, groups, E // groups), axis=2)[:, :, ::-1][:, :, :case["group_best"]].sum(axis=2)
        best = np.argsort(-per, axis=1, kind="stable")[:, :case["top_groups"]]
        group_of = np.arange(E) // (E // groups)
        allowed = (best[:, :, None] == group_of).any(axis=1)
    ids = np.argsort(np.where(allowed, -rank, np.inf), axis=1, kind="stable")[:, :k]
    w = np.take_along_axis(s, ids, axis=1)
    if case.get("renorm", True):
        w = w / w.sum(axis=1)[:, None]
    return torch.from_numpy(ids.astype(np.int32)), torch.from_numpy(w * case.get("scale", 1.0))


def _exact_weight(planes, bits, e):
    """float64 weights of expert e, from the bytes: a table of what a byte's halves (or the byte) stand for."""
    q, s = planes[0][e].long(), planes[1][e].double()
    if bits == 4:
        half = [v if v < 8 else v - 16 for v in range(16)]
        table = torch.tensor([[half[b % 16], half[b // 16]] for b in range(256)], dtype=torch.float64, device=q.device)
        v = table[q].flatten(1)
    else:
        table = torch.tensor([b if b < 128 else b - 256 for b in range(256)], dtype=torch.float64, device=q.device)
        v = table[q]
    return v * s.repeat_interleave(32, dim=1)


def _exact_products(rows, of, planes, bits, ids, n):
    """rows[of[p]] times the weight of pair p's expert, zeros where it has none."""
    out = torch.zeros((ids.numel(), n), dtype=torch.float64, device="cuda")
    flat = ids.flatten()
    for e in range(planes[0].shape[0]):
        mine = (flat == e).nonzero().flatten()
        if mine.numel():
            out.index_copy_(0, mine, rows.index_select(0, of[mine]).double() @ _exact_weight(planes, bits, e).t().contiguous())
    return out


def exact(case, seed):
    a = _inputs(case, seed)
    if case["kind"] == "route":
        return _exact_route(a["logits"], case, a["bias"])
    T, k, bits = case["T"], case["k"], case["bits"]
    pair = torch.arange(T * k, device="cuda")
    if case["kind"] == "layer":
        real = T - case["pad"]
        ids = torch.full((T, k), -1, dtype=torch.int64, device="cuda")
        weights = torch.zeros((T, k), dtype=torch.float64, device="cuda")
        chosen, w = _exact_route(a["logits"], case, None)
        ids[:real], weights[:real] = chosen.long().cuda(), w.cuda()
    else:
        ids, weights = a["ids"], a.get("weights")
    x = a["x"]
    if case["kind"] != "down":
        g = _exact_products(x, pair // k, a["gate"], bits, ids, case["width"])
        u = _exact_products(x, pair // k, a["up"], bits, ids, case["width"])
        x = g * torch.sigmoid(g) * u
        if case["kind"] == "up":
            return x
    z = _exact_products(x, pair, a["down"], bits, ids, case["hidden"])
    y = a["residual"].double()
    for j in range(k):
        y = y + weights[:, j:j + 1].double() * z[j::k]
    return (y, ids.to(torch.int32), weights) if case["kind"] == "layer" else y
