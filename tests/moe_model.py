"""A mixture-of-experts layer in 64 bits with numpy: what the expert ops are held to."""

from __future__ import annotations

import numpy as np

U = 2.0 ** -24  # half a step of f32, relative
SOFTMAX, SIGMOID = 0, 1
GEGLU, SWIGLU = 0, 1


def q4_0_values(raw, rows, cols):
    """GGUF Q4_0 bytes as f64 [rows][cols]."""
    b = np.frombuffer(np.ascontiguousarray(raw).tobytes(), np.uint8).reshape(rows, cols // 32, 18)
    d = b[..., :2].copy().view(np.float16).astype(np.float64)
    q = np.concatenate([b[..., 2:] & 15, b[..., 2:] >> 4], -1).astype(np.float64) - 8.0
    return (d * q).reshape(rows, cols)


def q8_0_parts(orc, x):
    """Q8_0 of f32 values: (quants int8 [n/32][32], scales f16 [n/32])."""
    b = np.asarray(orc.quantize_q8_0(np.ascontiguousarray(x, np.float32).reshape(-1)), np.uint8).reshape(-1, 34)
    return b[:, 2:].view(np.int8), b[:, :2].copy().view(np.float16)[:, 0]


def q8_0_values(orc, x):
    q, d = q8_0_parts(orc, x)
    return (q.astype(np.float64) * d.astype(np.float64)[:, None]).reshape(x.shape)


def pack_parts(pack, n):
    """An activation pack's planes: quants [n/32][32], scales f32, sums i32."""
    nb = n // 32
    pack = np.asarray(pack, np.uint8)
    return (pack[:nb * 32].view(np.int8).reshape(nb, 32), pack[nb * 32:nb * 36].view(np.float32),
            pack[nb * 36:nb * 40].view(np.int32))


def rms_scale(v, eps):
    """f32 1 / sqrt(mean + eps) of f32 rows: the sum in 64 bits, every later step rounded."""
    mean = ((v.astype(np.float64) ** 2).sum(-1, keepdims=True) / v.shape[-1]).astype(np.float32)
    return np.float32(1.0) / np.sqrt(mean + np.float32(eps))


def residual_norm(t, w_post, h, w_next, eps, norm_t):
    t = t.astype(np.float32)
    if norm_t:
        t = t * rms_scale(t, eps)
        t = t if w_post is None else t * w_post
    h = h + t
    xn = h * rms_scale(h, eps)
    return h, xn if w_next is None else xn * w_next


def scores(x, scoring):
    """f64 scores of f32 logits [batch][experts]; 0 where switched off."""
    x = x.astype(np.float64)
    on = x > -np.inf
    with np.errstate(invalid="ignore", over="ignore", divide="ignore"):
        if scoring == SIGMOID:
            return np.where(on, 1.0 / (1.0 + np.exp(-x)), 0.0), on
        top = np.where(on, x, -np.inf).max(1, keepdims=True)
        p = np.where(on, np.where(x == top, 1.0, np.exp(x - top)), 0.0)
        return p / np.where(p.sum(1, keepdims=True) > 0, p.sum(1, keepdims=True), 1.0), on


def route(logits, bias, k, scoring, n_groups=1, top_groups=1, group_best=1, renormalise=True, scale=1.0):
    n, e = logits.shape
    score, on = scores(logits, scoring)
    if bias is not None:
        value = score + bias.astype(np.float64)
    else:
        value = score if group_best == 2 and n_groups > 1 else logits.astype(np.float64)
    with np.errstate(invalid="ignore"):
        value = np.where(on & (value > -np.inf), value, -np.inf)
    ids, w = np.full((n, k), -1, np.int32), np.zeros((n, k))
    for t in range(n):
        v = value[t].copy()
        if n_groups > 1:
            g = np.sort(v.reshape(n_groups, -1), 1)[:, ::-1]
            rank = g[:, 0].copy()
            if group_best == 2 and g.shape[1] > 1:
                rank = np.where(g[:, 1] > -np.inf, g[:, 0] + g[:, 1], rank)
            kept = np.argsort(-rank, kind="stable")[:top_groups]
            allowed = np.isin(np.arange(e) // (e // n_groups), kept)
            v[~allowed] = -np.inf
        best = [i for i in np.argsort(-v, kind="stable")[:k] if v[i] > -np.inf]
        ids[t, :len(best)] = best
        w[t, :len(best)] = score[t, best]
    if renormalise:
        total = w.sum(1, keepdims=True)
        w = np.where(total > 0, w / np.where(total > 0, total, 1.0), 0.0)
    return ids, w * scale


def plan(ids, n_experts):
    flat = ids.reshape(-1)
    order = [i for e in range(n_experts) for i in np.flatnonzero(flat == e)]
    starts = np.concatenate([[0], np.cumsum([(flat == e).sum() for e in range(n_experts)])]).astype(np.int32)
    return starts, np.array(order + [-1] * (flat.size - len(order)), np.int32)


def dot_error(nb):
    """The most that a sum of nb blocks of 32 products may be off in f32, in units of the sum of the products'
    magnitudes: a block's 32 products in at most two parts each, added in any order (63 roundings), its scales and the
    step into the running sum (4), and the nb running sums."""
    return (63 + 4 + nb) * U


def gated(g, u, activation):
    if activation == GEGLU:
        return 0.5 * g * (1.0 + np.tanh(np.sqrt(2.0 / np.pi) * (g + 0.044715 * g ** 3))) * u
    with np.errstate(over="ignore"):
        return g / (1.0 + np.exp(-g)) * u


def gate_up(wg, wu, xq, ids, k, activation):
    """(act, bound) [batch * k][rows] from f64 weights [experts][rows][cols] and f64 Q8_0 values; NaN without an
    expert.  The bound: f' is at most 1.13 in size, |f(g)| at most |g|, and the sigmoid in f (e^z off by (|z| + 2) steps,
    one addition, one reciprocal) is off by at most 8 U; then one product."""
    flat, nb = ids.reshape(-1), xq.shape[1] // 32
    act, bound = (np.full((flat.size, wg.shape[1]), np.nan) for _ in range(2))
    for a, e in enumerate(flat):
        if e < 0:
            continue
        x = xq[a // k]
        g, u = wg[e] @ x, wu[e] @ x
        eg, eu = (dot_error(nb) * (np.abs(w[e]) @ np.abs(x)) for w in (wg, wu))
        act[a] = gated(g, u, activation)
        ef = 1.13 * eg + 8 * U * np.abs(g)
        bound[a] = ef * (np.abs(u) + eu) + np.abs(g) * eu + 2 * U * np.abs(act[a]) + 1e-30
    return act, bound


def down(wd, aq, ids, weights, k):
    """(y, bound) [batch][rows] from f64 Q8_0 values [batch * k][cols]."""
    n, nb = ids.shape[0], aq.shape[1] // 32
    y, bound = np.zeros((n, wd.shape[1])), np.zeros((n, wd.shape[1]))
    for t in range(n):
        for s in range(k):
            e, w = ids[t, s], float(weights[t, s])
            if e < 0:
                continue
            y[t] += w * (wd[e] @ aq[t * k + s])
            bound[t] += abs(w) * (dot_error(nb) + (k + 2) * U) * (np.abs(wd[e]) @ np.abs(aq[t * k + s]))
    return y, bound + 1e-30
