"""The operators of a mixture-of-experts layer for a batch of tokens, as cases that can be timed and checked.

In such a layer every token goes through k of n experts, each a gated FFN with Q4_0 weights of its own:

* ``norm``     the residual's addition and the next norm, its result in f32 and as Q8_0 blocks;
* ``logits``   the router's product in f32;
* ``route``    scores, the k experts of every token, their weights, and the tokens sorted by expert;
* ``gate_up``  the experts' first two products over Q8_0 activations and the gated activation;
* ``down``     their last product, summed over a token's experts by its weights.

With ``own`` false ``run`` computes them with elementary torch operations, with ``own`` true through the framework.
Inputs are synthetic, made on the GPU from the seed.
"""

import importlib.util
import math
import sys
from pathlib import Path

import torch

own = False

DEV = "cuda"
EPS = 1e-6
SCORING = {"softmax": 0, "sigmoid": 1}
ACTIVATION = {"geglu": 0, "swiglu": 1}

_kept = {}


def _device():
    """One context for the program, its scratch reserved once."""
    if "dev" not in _kept:
        pkg = Path(__file__).resolve().parents[1] / "qt_llama.cpp_amd"
        name = "qt_llama_cpp_amd"  # the package's folder is no identifier, so it is loaded by path
        if name not in sys.modules:
            spec = importlib.util.spec_from_file_location(name, pkg / "__init__.py",
                                                          submodule_search_locations=[str(pkg)])
            mod = importlib.util.module_from_spec(spec)
            sys.modules[name] = mod
            spec.loader.exec_module(mod)
        _kept["dev"] = sys.modules[name].HipDevice.new(0)
        _kept["dev"].reserve_workspace(512 << 20)
    return _kept["dev"]


# ---- cases -------------------------------------------------------------------

# the expert layer of the reference's own model: width 2816, 128 experts of 704, eight a token
LAYER = dict(experts=128, k=8)


def listed():
    return [
        # one decoding sequence: the sandwich norm's addition, then the next norm; the smallest call
        dict(name="norm_decode_1", kind="norm", batch=1, dim=2816, post=True, pack=True),
        # a long prompt's rows at the benchmark model's width
        dict(name="norm_prompt_1900", kind="norm", batch=1900, dim=2304, post=False, pack=True),
        # router of a few decoding requests
        dict(name="logits_decode_5", kind="logits", batch=5, experts=128, cols=2816),
        # router of several prompts' chunks
        dict(name="logits_prompt_1999", kind="logits", batch=1999, experts=128, cols=2816),
        # choice of eight experts for one token
        dict(name="route_decode_1", kind="route", batch=1, scoring="softmax", bias=False, groups=1, top_groups=1,
             group_best=1, renormalise=True, scale=1.0, masked=False, **LAYER),
        # many experts in groups, chosen with a bias that balances their load; some experts switched off
        dict(name="route_groups_4001", kind="route", batch=4001, experts=256, k=8, scoring="sigmoid", bias=True, groups=8,
             top_groups=4, group_best=2, renormalise=True, scale=2.5, masked=True),
        # one decoding sequence through its eight experts: latency
        dict(name="gate_up_decode_1", kind="gate_up", batch=1, rows=704, cols=2816, act="geglu", **LAYER),
        # a server's decoding requests: most experts have a token or two, every weight is read
        dict(name="gate_up_decode_40", kind="gate_up", batch=40, rows=704, cols=2816, act="geglu", **LAYER),
        # prompts' chunks: about a hundred tokens an expert
        dict(name="gate_up_prompt_1501", kind="gate_up", batch=1501, rows=704, cols=2816, act="geglu", **LAYER),
        # the same three of the second product
        dict(name="down_decode_1", kind="down", batch=1, rows=2816, cols=704, **LAYER),
        dict(name="down_decode_40", kind="down", batch=40, rows=2816, cols=704, **LAYER),
        dict(name="down_prompt_1501", kind="down", batch=1501, rows=2816, cols=704, **LAYER),
    ]


def _log(rng, lo, hi):
    """A whole number of lo..hi, evenly over its logarithm."""
    return max(lo, min(hi, int(math.exp(rng.uniform(math.log(lo), math.log(hi + 1))))))


def draw(rng):
    kind = rng.choice(["norm", "logits", "route", "gate_up", "gate_up", "down", "down"])
    if kind == "norm":
        dim = 32 * _log(rng, 2, 256)
        return dict(kind=kind, batch=_log(rng, 1, min(2048, 4300000 // dim)), dim=dim, post=rng.random() < 0.5,
                    pack=rng.random() < 0.7)
    if kind == "logits":
        cols = 32 * _log(rng, 2, 128)
        return dict(kind=kind, batch=_log(rng, 1, min(2048, 5600000 // cols)), experts=_log(rng, 4, 128), cols=cols)
    if kind == "route":
        groups = rng.choice([1, 1, 1, 2, 4, 8])
        experts = groups * _log(rng, max(2, 4 // groups), 256 // groups)
        top_groups = rng.randint(1, groups)
        k = min(rng.choice([1, 2, 4, 6, 8, 8]), experts // groups * top_groups)
        return dict(kind=kind, batch=_log(rng, 1, 4001), experts=experts, k=k, scoring=rng.choice(list(SCORING)),
                    bias=rng.random() < 0.5, groups=groups, top_groups=top_groups, group_best=rng.choice([1, 2]),
                    renormalise=rng.random() < 0.7, scale=rng.choice([1.0, 2.5]), masked=rng.random() < 0.3)
    cols, rows = 32 * _log(rng, 2, 128), _log(rng, 30, 4096)
    experts = _log(rng, 4, max(4, min(128, 254000000 // (rows * cols))))
    k = min(experts, rng.choice([1, 2, 4, 6, 8, 8]))
    batch = _log(rng, 1, max(1, min(1501, 23700000000 // (k * rows * cols))))
    case = dict(kind=kind, batch=batch, experts=experts, k=k, rows=rows, cols=cols)
    return dict(case, act=rng.choice(list(ACTIVATION))) if kind == "gate_up" else case


# ---- inputs ------------------------------------------------------------------

def _normal(g, *shape, scale=1.0):
    return torch.randn(*shape, generator=g, device=DEV) * scale


def _matrices(g, n, rows, cols):
    """n Q4_0 matrices in the framework's layout (all quants, then all f16 scales), values of about cols^-1/2."""
    blocks = n * rows * (cols // 32)
    quants = torch.randint(0, 256, (blocks * 16,), generator=g, device=DEV, dtype=torch.uint8)
    scales = (torch.rand(blocks, generator=g, device=DEV) + 0.5) * (0.2 / math.sqrt(cols))
    return torch.cat([quants, scales.half().view(torch.uint8)])


def _plan(ids, experts):
    """The assignments (token * k + slot) sorted by expert, where each expert's begin, and the longest list."""
    flat = ids.reshape(-1).long()
    key = torch.where(flat < 0, experts, flat)
    order = torch.sort(key, stable=True).indices
    count = torch.bincount(key, minlength=experts + 1)[:experts]
    starts = torch.cat([torch.zeros(1, device=DEV, dtype=torch.long), torch.cumsum(count, 0)])
    order = torch.where(torch.arange(order.numel(), device=DEV) < starts[-1], order, -1)
    return starts.to(torch.int32), order.to(torch.int32), int(count.max())


def prepare(case, seed):
    c = dict(case)
    g = torch.Generator(device=DEV).manual_seed(seed)
    kind, n = c["kind"], c["batch"]
    s = {"c": c}
    if kind == "norm":
        d = c["dim"]
        s.update(t=_normal(g, n, d, scale=3.0), h=_normal(g, n, d, scale=8.0), w_post=1.0 + _normal(g, d, scale=0.2),
                 w_next=1.0 + _normal(g, d, scale=0.2), h_out=torch.zeros(n, d, device=DEV),
                 xn=torch.zeros(n, d, device=DEV))
        s["t"][:, ::97] *= 20.0  # residual streams have a few large channels
        s["pack"] = torch.zeros(n * d // 32 * 40, device=DEV, dtype=torch.uint8) if c["pack"] else None
    elif kind == "logits":
        s.update(x=_normal(g, n, c["cols"]), w=_normal(g, c["experts"], c["cols"], scale=c["cols"] ** -0.5),
                 logits=torch.zeros(n, c["experts"], device=DEV))
    elif kind == "route":
        e, a = c["experts"], n * c["k"]
        s["logits"] = _normal(g, n, e, scale=1.5) + _normal(g, e, scale=0.7)
        if c["masked"]:
            off = torch.rand(e, generator=g, device=DEV) < 0.1
            off[0] = False
            s["logits"][:, off] = -math.inf
        s["bias"] = _normal(g, e, scale=0.1) if c["bias"] else None
        s.update(ids=torch.zeros(n, c["k"], device=DEV, dtype=torch.int32), weights=torch.zeros(n, c["k"], device=DEV),
                 starts=torch.zeros(e + 1, device=DEV, dtype=torch.int32),
                 order=torch.zeros(a, device=DEV, dtype=torch.int32))
    else:
        e, k, rows, cols = c["experts"], c["k"], c["rows"], c["cols"]
        liking = _normal(g, n, e) + _normal(g, e, scale=0.5)  # some experts are asked for more than others
        best = torch.topk(liking, k, dim=1)
        s["ids"] = best.indices.to(torch.int32)
        s["weights"] = torch.softmax(best.values, -1)
        s["starts"], s["order"], s["most"] = _plan(s["ids"], e)
        if kind == "gate_up":
            s.update(w_gate=_matrices(g, e, rows, cols), w_up=_matrices(g, e, rows, cols), x=_normal(g, n, cols),
                     out=torch.zeros(n * k, rows, device=DEV))
        else:
            s.update(w_down=_matrices(g, e, rows, cols), act=_normal(g, n * k, cols) * _normal(g, n * k, cols),
                     out=torch.zeros(n, rows, device=DEV))
    torch.cuda.synchronize()
    return s


# ---- one pass ----------------------------------------------------------------

def run(s):
    kind = s["c"]["kind"]
    if own:
        return {"norm": _own_norm, "logits": _own_logits, "route": _own_route, "gate_up": _own_gate_up,
                "down": _own_down}[kind](s)
    return {"norm": _plain_norm, "logits": _plain_logits, "route": _plain_route, "gate_up": _plain_gate_up,
            "down": _plain_down}[kind](s)


def _ptr(x):
    return None if x is None else x.data_ptr()


def _own_norm(s):
    c = s["c"]
    _device().residual_rms_norm_batch(_ptr(s["t"]), _ptr(s["w_post"]) if c["post"] else None, _ptr(s["h"]),
                                      _ptr(s["h_out"]), _ptr(s["w_next"]), _ptr(s["xn"]), c["dim"], c["batch"], EPS,
                                      pack=_ptr(s["pack"]), norm_t=c["post"])
    return _norm_out(s)


def _own_logits(s):
    c = s["c"]
    _device().moe_logits(_ptr(s["x"]), _ptr(s["w"]), _ptr(s["logits"]), c["experts"], c["cols"], c["batch"])
    return {"logits": s["logits"]}


def _own_route(s):
    c = s["c"]
    _device().moe_route(_ptr(s["logits"]), _ptr(s["bias"]), _ptr(s["ids"]), _ptr(s["weights"]), _ptr(s["starts"]),
                        _ptr(s["order"]), c["experts"], c["batch"], c["k"], SCORING[c["scoring"]], c["groups"],
                        c["top_groups"], c["group_best"], c["renormalise"], c["scale"])
    return {k: s[k] for k in ("ids", "weights", "starts", "order")}


def _own_gate_up(s):
    c = s["c"]
    _device().moe_gate_up_q4_0(_ptr(s["w_gate"]), _ptr(s["w_up"]), _ptr(s["x"]), _ptr(s["ids"]), _ptr(s["starts"]),
                               _ptr(s["order"]), _ptr(s["out"]), c["experts"], c["rows"], c["cols"], c["batch"], c["k"],
                               ACTIVATION[c["act"]])
    return {"act": s["out"]}


def _own_down(s):
    c = s["c"]
    _device().moe_down_q4_0(_ptr(s["w_down"]), _ptr(s["act"]), _ptr(s["ids"]), _ptr(s["weights"]), _ptr(s["starts"]),
                            _ptr(s["order"]), _ptr(s["out"]), c["experts"], c["rows"], c["cols"], c["batch"], c["k"])
    return {"y": s["out"]}


def _norm_out(s):
    """The stream, the normed rows, and the parts of their Q8_0 pack: whole quants and block sums (which follow from xn
    without any freedom), and the blocks' scales."""
    out = {"h": s["h_out"], "xn": s["xn"]}
    if s["pack"] is not None:
        blocks = s["pack"].numel() // 40
        out["q"] = s["pack"][:blocks * 32].view(torch.int8)
        out["d"] = s["pack"][blocks * 32:blocks * 36].view(torch.float32)
        out["sums"] = s["pack"][blocks * 36:].view(torch.int32)
    return out


def _rms(v):
    """1 / sqrt(mean + eps) of rows, the sum in 64 bits, every later step rounded to 32."""
    mean = (v.double().square().sum(-1, keepdim=True) / v.shape[-1]).float()
    root = (mean + EPS).double().sqrt().float()
    return (1.0 / root.double()).float()


def _q8(x):
    """Rows as Q8_0 blocks of 32: quants, scales (amax/127 kept as a truncated half) in 32 bits."""
    b = x.reshape(-1, 32)
    scale = (b.abs().amax(1, keepdim=True).double() / 127.0).float()
    half = scale.half()
    half = torch.where(half.float() > scale, (half.view(torch.int16) - 1).view(torch.float16), half).float()
    half = torch.where(scale < 2.0 ** -14, 0.0, half)
    inverse = torch.where(scale > 0, (1.0 / scale.double()).float(), 0.0)
    v = (b * inverse).double()
    return (torch.sign(v) * torch.floor(v.abs() + 0.5)).clamp(-128, 127).float(), half


def _plain_norm(s):
    c = s["c"]
    t = s["t"]
    if c["post"]:
        t = t * _rms(t) * s["w_post"]
    torch.add(s["h"], t, out=s["h_out"])
    torch.mul(s["h_out"] * _rms(s["h_out"]), s["w_next"], out=s["xn"])
    out = _norm_out(s)
    if c["pack"]:
        q, d = _q8(s["xn"])
        out["q"].copy_(q.view(-1))
        out["d"].copy_(d.view(-1))
        out["sums"].copy_(q.sum(1))
    return out


def _plain_logits(s):
    torch.matmul(s["x"], s["w"].t().contiguous(), out=s["logits"])
    return {"logits": s["logits"]}


def _plain_route(s):
    """In 64 bits, so that the choice does not hang on how an exponential was rounded."""
    c, x = s["c"], s["logits"].double()
    n, e, k = c["batch"], c["experts"], c["k"]
    on = x > -math.inf  # neither switched off nor no number
    if c["scoring"] == "softmax":
        top = torch.where(on, x, -math.inf).amax(1, keepdim=True)
        p = torch.where(on, torch.where(x == top, 1.0, torch.exp(x - top)), 0.0)
        score = p / p.sum(1, keepdim=True)
    else:
        score = torch.where(on, 1.0 / (1.0 + torch.exp(-x)), 0.0)
    # experts are ordered by their logits, or by scores where something is added to them
    value = score + s["bias"].double() if c["bias"] else score if c["group_best"] == 2 and c["groups"] > 1 else x
    value = torch.where(on & ~value.isnan(), value, -math.inf)
    if c["groups"] > 1:
        inside = value.view(n, c["groups"], -1)
        best = torch.sort(inside, descending=True, stable=True).values[..., :c["group_best"]]
        rank = torch.where((best > -math.inf) | (torch.arange(best.shape[-1], device=DEV) == 0), best, 0.0).sum(-1)
        kept = torch.sort(rank, descending=True, stable=True).indices[:, :c["top_groups"]]
        allowed = torch.zeros(n, c["groups"], device=DEV, dtype=torch.bool).scatter_(1, kept, True)
        value = torch.where(allowed.unsqueeze(2), inside, -math.inf).view(n, e)
    ranked = torch.sort(value, descending=True, stable=True)
    ids, there = ranked.indices[:, :k], ranked.values[:, :k] > -math.inf
    w = torch.where(there, score.gather(1, ids), 0.0)
    if c["renormalise"]:
        total = w.sum(1, keepdim=True)
        w = torch.where(total > 0, w / total, 0.0)
    s["ids"].copy_(torch.where(there, ids, -1))
    s["weights"].copy_(w * c["scale"])
    flat = torch.where(there, ids, e).view(-1)
    order = torch.sort(flat, stable=True).indices
    ends = torch.cumsum((flat.unsqueeze(0) == torch.arange(e, device=DEV).unsqueeze(1)).sum(1), 0)
    s["starts"][0] = 0
    s["starts"][1:] = ends
    s["order"].copy_(torch.where(torch.arange(n * k, device=DEV) < ends[-1], order, -1))
    return {k: s[k] for k in ("ids", "weights", "starts", "order")}


def _weights(raw, n, rows, cols, pick=None):
    """Q4_0 matrices (those of `pick`, in its order, or all) as 32-bit values [n][rows][cols]."""
    quants = raw[:n * rows * cols // 2].view(n, rows, cols // 32, 16)
    scales = raw[n * rows * cols // 2:].view(torch.float16).view(n, rows, cols // 32, 1)
    if pick is not None:
        quants, scales = quants[pick], scales[pick]
    w = torch.cat([quants & 15, quants >> 4], -1).float() - 8.0
    return (w * scales.float()).view(-1, rows, cols)


def _products(s, x, matrices):
    """Each assignment's row of x (already gathered) times its expert's matrices."""
    c = s["c"]
    e, rows, cols, total = c["experts"], c["rows"], c["cols"], c["batch"] * c["k"]
    ids = s["ids"].view(-1).long()
    if total < e:  # few: their experts' matrices one by one
        return [torch.matmul(_weights(m, e, rows, cols, ids), x.unsqueeze(2)).squeeze(2) for m in matrices]
    # many: every expert's rows, padded to the longest list
    starts, order = s["starts"].long(), s["order"].long()
    at = starts[:-1, None] + torch.arange(s["most"], device=DEV)
    real = at < starts[1:, None]
    rows_of = order[torch.where(real, at, 0)]
    xe = torch.where(real.unsqueeze(2), x[rows_of], 0.0).transpose(1, 2).contiguous()
    found = []
    for m in matrices:
        y = torch.matmul(_weights(m, e, rows, cols), xe).transpose(1, 2)
        out = torch.zeros(total, rows, device=DEV)
        out[rows_of[real]] = y[real]
        found.append(out)
    return found


def _plain_gate_up(s):
    c = s["c"]
    q, d = _q8(s["x"])
    x = (q * d).view(s["x"].shape).repeat_interleave(c["k"], 0)
    g, u = _products(s, x, [s["w_gate"], s["w_up"]])
    if c["act"] == "geglu":
        f = 0.5 * g * (1.0 + torch.tanh(0.7978845608 * (g + 0.044715 * g * g * g)))
    else:
        f = g / (1.0 + torch.exp(-g))
    torch.mul(f, u, out=s["out"])
    return {"act": s["out"]}


def _plain_down(s):
    c = s["c"]
    q, d = _q8(s["act"])
    y, = _products(s, (q * d).view(s["act"].shape), [s["w_down"]])
    torch.sum(y.view(c["batch"], c["k"], -1) * s["weights"].unsqueeze(2), 1, out=s["out"])
    return {"y": s["out"]}


# ---- bytes and operations ----------------------------------------------------

def _asked(c):
    """Experts that have a token, of so many assignments: what is expected when all are equally liked."""
    return c["experts"] * (1.0 - (1.0 - c["k"] / c["experts"]) ** c["batch"])


def work(case):
    c = case
    n = c["batch"]
    if c["kind"] == "norm":
        d = c["dim"]
        return {"bytes": n * d * (16.0 + (1.25 if c["pack"] else 0.0)) + (8.0 if c["post"] else 4.0) * d,
                "flops": n * d * (8.0 if c["post"] else 5.0)}
    if c["kind"] == "logits":
        return {"bytes": 4.0 * (n * c["cols"] + c["experts"] * c["cols"] + n * c["experts"]),
                "flops": 2.0 * n * c["cols"] * c["experts"]}
    if c["kind"] == "route":
        return {"bytes": 4.0 * (n * c["experts"] + 3 * n * c["k"] + 2 * c["experts"] + 1),
                "flops": 6.0 * n * c["experts"]}
    a, matrices = n * c["k"], 2 if c["kind"] == "gate_up" else 1
    weights = matrices * _asked(c) * c["rows"] * c["cols"] * 18 / 32
    ends = n * c["cols"] + a * c["rows"] if c["kind"] == "gate_up" else a * c["cols"] + n * c["rows"] + a
    return {"bytes": weights + 4.0 * ends + 8.0 * a, "flops": 2.0 * matrices * a * c["rows"] * c["cols"]}


# ---- the same in 64 bits -----------------------------------------------------

def _q64(x):
    """The values that a row's Q8_0 blocks stand for, in 64 bits; the quantiser's own steps are in 32."""
    out = torch.empty_like(x, dtype=torch.float64)
    for b in range(x.shape[-1] // 32):
        v = x[:, 32 * b:32 * b + 32]
        top = v.abs().max(1, keepdim=True).values
        scale = top / torch.full_like(top, 127.0)
        d = (scale.view(torch.int32) & ~0x1FFF).view(torch.float32).double()  # the mantissa's upper ten bits
        d = torch.where(scale < 2.0 ** -14, torch.zeros_like(d), d)
        r = (v * torch.where(scale > 0, torch.ones_like(scale) / scale, torch.zeros_like(scale))).double()
        r = torch.where(r < 0, -torch.floor(0.5 - r), torch.floor(r + 0.5))
        out[:, 32 * b:32 * b + 32] = d * r.clamp(-128, 127)
    return out


def _matrix64(raw, n, rows, cols, i):
    """Matrix i of n."""
    nb = cols // 32
    b = raw[i * rows * nb * 16:(i + 1) * rows * nb * 16].reshape(rows, nb, 16).to(torch.int64)
    d = raw[n * rows * nb * 16:].view(torch.float16)[i * rows * nb:(i + 1) * rows * nb].double().reshape(rows, nb, 1)
    q = torch.empty(rows, nb, 32, device=DEV, dtype=torch.float64)
    q[..., :16] = b % 16 - 8
    q[..., 16:] = b // 16 - 8
    return (q * d).reshape(rows, cols)


def _exact_route(s):
    c, x = s["c"], s["logits"].double()
    off = x == -math.inf
    score = torch.softmax(x, 1) if c["scoring"] == "softmax" else torch.sigmoid(x)
    v = score + s["bias"] if c["bias"] else score  # logits of the cases lie where scores keep their order
    v = v.masked_fill(off, -math.inf)
    if c["groups"] > 1:
        size = c["experts"] // c["groups"]
        most = torch.topk(v.view(-1, c["groups"], size), min(c["group_best"], size), dim=2).values
        rank = most[..., 0] + (most[..., 1:].clamp(min=-1e300) * (most[..., 1:] > -math.inf)).sum(-1)
        worst = torch.topk(rank, c["top_groups"], dim=1).values[:, -1:]
        v = v.masked_fill((rank < worst).repeat_interleave(size, 1), -math.inf)
    ranked = torch.topk(v, c["k"], dim=1)
    w = score.gather(1, ranked.indices) * (ranked.values > -math.inf)
    if c["renormalise"]:
        w = w / w.sum(1, keepdim=True)
    return {"ids": None, "weights": w * c["scale"], "starts": None, "order": None}


def exact(case, seed):
    s = prepare(case, seed)
    c, kind, n = s["c"], s["c"]["kind"], s["c"]["batch"]
    if kind == "norm":
        t = s["t"].double()
        if c["post"]:
            t = t / torch.linalg.vector_norm(t, dim=1, keepdim=True).square().div(c["dim"]).add(EPS).sqrt() * s["w_post"]
        h = s["h"] + t
        xn = h / torch.linalg.vector_norm(h, dim=1, keepdim=True).square().div(c["dim"]).add(EPS).sqrt() * s["w_next"]
        return {"h": h, "xn": xn, **({"q": None, "d": None, "sums": None} if c["pack"] else {})}
    if kind == "logits":
        return {"logits": s["x"].double() @ s["w"].double().t().contiguous()}
    if kind == "route":
        return _exact_route(s)
    e, k, rows, cols = c["experts"], c["k"], c["rows"], c["cols"]
    ids = s["ids"].view(-1)
    if kind == "gate_up":
        x = _q64(s["x"])
        out = torch.zeros(n * k, rows, device=DEV, dtype=torch.float64)
        for i in torch.unique(ids).tolist():
            mine = (ids == i).nonzero().view(-1)
            rows_in = x[mine // k]
            g = rows_in @ _matrix64(s["w_gate"], e, rows, cols, i).t().contiguous()
            u = rows_in @ _matrix64(s["w_up"], e, rows, cols, i).t().contiguous()
            if c["act"] == "geglu":
                f = 0.5 * g * (1.0 + torch.tanh(math.sqrt(2.0 / math.pi) * (g + 0.044715 * g ** 3)))
            else:
                f = g * torch.sigmoid(g)
            out[mine] = f * u
        return {"act": out}
    x, w = _q64(s["act"]), s["weights"].double().view(-1)
    out = torch.zeros(n, rows, device=DEV, dtype=torch.float64)
    for i in torch.unique(ids).tolist():
        mine = (ids == i).nonzero().view(-1)
        out.index_add_(0, mine // k, (x[mine] @ _matrix64(s["w_down"], e, rows, cols, i).t().contiguous()) * w[mine, None])
    return {"y": out}
