"""The operators of a batch of requests over paged KV caches, as cases that can be timed and checked.

A program that serves several requests at once keeps K and V in pages that any request can hold, and often starts
every request with the same long text (a system prompt), whose K and V are in the cache once.  A step of such a
program is

* ``tables``     the step's bookkeeping from the requests' lengths: pages taken and returned, each new token's place
                 in the cache and its position;
* ``append``     RoPE of the new tokens' q and k, and their K and V stored at those places;
* ``attention``  the new tokens' attention over the shared prefix and their own request's positions.

With ``own`` false ``run`` computes them with elementary torch operations, with ``own`` true through the framework.
Inputs are synthetic, made on the GPU from the seed; lengths follow from the case alone.
"""

import importlib.util
import math
import sys
from pathlib import Path

import torch

own = False

FORMATS = {"f16": 0, "q8_0": 1, "q4_0": 2}
BLOCK_BYTES = {"q8_0": 34, "q4_0": 18}
BYTES_PER_VALUE = {"f16": 2.0, "q8_0": 34 / 32, "q4_0": 18 / 32}
ROPE_BASE = 10000.0
DEV = "cuda"

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
        _kept["dev"].reserve_workspace(256 << 20)
    return _kept["dev"]


# ---- cases -------------------------------------------------------------------
#
# seqs requests; each holds len_lo..len_hi own tokens before the step and adds new_lo..new_hi; finished: every so many
# requests one has ended (and every seventh is idle); pad: rows of the step's buffers past the last used one.

SHAPE_2B = dict(heads=8, kv_heads=4, head_dim=256)  # the repository's benchmark model


def listed():
    f16 = dict(k_format="f16", v_format="f16")
    return [
        # the bookkeeping of one decoded token for a handful of requests: the smallest call there is
        dict(name="tables_decode_6", kind="tables", seqs=6, page=16, len_lo=20, len_hi=900, new_lo=1, new_hi=1,
             prefix=1024, finished=0, pad=2),
        # a full server's step: most requests decode, some bring a prompt's chunk, some end
        dict(name="tables_mixed_700", kind="tables", seqs=700, page=16, len_lo=1, len_hi=6000, new_lo=1, new_hi=200,
             prefix=2048, finished=23, pad=513),
        # K and V of one decoded token for a small batch
        dict(name="append_decode_24", kind="append", seqs=24, page=16, len_lo=10, len_hi=600, new_lo=1, new_hi=1,
             prefix=1000, pad=8, **SHAPE_2B, **f16),
        # the chunks of several prompts in one call
        dict(name="append_chunks_1900", kind="append", seqs=19, page=32, len_lo=1, len_hi=1500, new_lo=37, new_hi=163,
             prefix=777, pad=100, **SHAPE_2B, **f16),
        # one request alone behind a short prefix: latency
        dict(name="attn_decode_1", kind="attention", seqs=1, page=16, len_lo=70, len_hi=70, new_lo=1, new_hi=1,
             prefix=500, window=0, pad=0, **SHAPE_2B, **f16),
        # a small server decoding behind a system prompt, a global layer
        dict(name="attn_decode_32", kind="attention", seqs=32, page=16, len_lo=30, len_hi=1200, new_lo=1, new_hi=1,
             prefix=4001, window=0, pad=0, **SHAPE_2B, **f16),
        # the same program's windowed layers: each request's window begins somewhere in the prefix
        dict(name="attn_decode_48_window", kind="attention", seqs=48, page=16, len_lo=30, len_hi=5000, new_lo=1,
             new_hi=1, prefix=6000, window=4096, pad=3, **SHAPE_2B, **f16),
        # a full server behind long shared documents
        dict(name="attn_decode_256_long", kind="attention", seqs=256, page=32, len_lo=16, len_hi=1000, new_lo=1,
             new_hi=1, prefix=32768, window=0, pad=0, **SHAPE_2B, **f16),
        # requests with nothing in common and very uneven lengths, wide groups
        dict(name="attn_decode_20_apart", kind="attention", seqs=20, page=64, len_lo=100, len_hi=30000, new_lo=1,
             new_hi=1, prefix=0, window=0, pad=0, heads=32, kv_heads=8, head_dim=128, **f16),
        # quantised caches, wide groups
        dict(name="attn_decode_40_q8_q4", kind="attention", seqs=40, page=32, len_lo=50, len_hi=2500, new_lo=1,
             new_hi=1, prefix=8100, window=0, pad=0, heads=16, kv_heads=2, head_dim=128, k_format="q8_0",
             v_format="q4_0"),
        # a few drafted tokens a request, small heads, pages that no tile divides
        dict(name="attn_draft_17", kind="attention", seqs=17, page=24, len_lo=1, len_hi=3000, new_lo=2, new_hi=5,
             prefix=1111, window=0, pad=5, heads=12, kv_heads=4, head_dim=64, **f16),
        # prompts' chunks behind a shared prefix: many rows, causal among themselves
        dict(name="attn_chunks_2000", kind="attention", seqs=11, page=16, len_lo=1, len_hi=1800, new_lo=60, new_hi=400,
             prefix=3000, window=0, pad=17, **SHAPE_2B, **f16),
    ]


def _log(rng, lo, hi):
    """A whole number of lo..hi, evenly over its logarithm."""
    return max(lo, min(hi, int(math.exp(rng.uniform(math.log(lo), math.log(hi + 1))))))


def draw(rng):
    kind = rng.choice(["tables", "append", "attention", "attention", "attention"])
    page = rng.choice([8, 16, 16, 24, 32, 64, 100, 128])
    if kind == "tables":
        hi = _log(rng, 1, 6000)
        return dict(kind=kind, seqs=_log(rng, 1, 700), page=page, len_lo=rng.randint(1, hi), len_hi=hi,
                    new_lo=1, new_hi=rng.choice([1, 1, _log(rng, 1, 200)]), prefix=rng.choice([0, _log(rng, 1, 32768)]),
                    finished=rng.choice([0, 5, 31]), pad=rng.randint(0, 600))
    group, kv, hd = rng.choice([1, 2, 2, 3, 4, 8, 16]), rng.choice([1, 2, 4, 8]), rng.choice([32, 64, 96, 128, 256, 256, 512])
    group = min(group, 4096 // hd)
    kv = min(kv, max(1, 1024 // hd), max(1, 4096 // (group * hd)))
    shape = dict(heads=group * kv, kv_heads=kv, head_dim=hd)
    if kind == "append":
        seqs = _log(rng, 1, 200)
        new = rng.choice([1, _log(rng, 1, max(1, 1900 // seqs))])
        return dict(kind=kind, seqs=seqs, page=page, len_lo=1, len_hi=_log(rng, 1, 1500), new_lo=1, new_hi=new,
                    prefix=_log(rng, 1, 4000), pad=rng.randint(0, 50), k_format="f16", v_format="f16", **shape)
    fmts = rng.choice([("f16", "f16"), ("f16", "f16"), ("f16", "f16"), ("q8_0", "q8_0"), ("q8_0", "q4_0"), ("q4_0", "q4_0")])
    rest = dict(page=page, window=rng.choice([0, 0, 0, 512, 4096]), pad=rng.randint(0, 20), k_format=fmts[0],
                v_format=fmts[1], **shape)
    form = rng.choice(["shared", "shared", "apart", "chunks"])
    if form == "shared":
        seqs = _log(rng, 1, 200)
        hi = _log(rng, 1, min(1500, 60000 // seqs))
        return dict(kind=kind, seqs=seqs, len_lo=rng.randint(1, hi), len_hi=hi, new_lo=1,
                    new_hi=rng.choice([1, 1, 4]), prefix=_log(rng, 16, 16000), **rest)
    if form == "apart":
        return dict(kind=kind, seqs=_log(rng, 1, 20), len_lo=_log(rng, 1, 200), len_hi=_log(rng, 200, 20000), new_lo=1,
                    new_hi=rng.choice([1, 3]), prefix=0, **rest)
    seqs = _log(rng, 1, 12)
    return dict(kind=kind, seqs=seqs, len_lo=1, len_hi=_log(rng, 1, 1800), new_lo=_log(rng, 8, 60),
                new_hi=max(60, _log(rng, 8, 1500 // seqs)), prefix=rng.choice([0, _log(rng, 1, 3000)]), **rest)


def _spread(lo, hi, n, turn):
    """n whole numbers of lo..hi (lo > 0), evenly over their logarithm, in an order without a pattern."""
    if lo >= hi:
        return [lo] * n
    return [min(hi, int(lo * ((hi + 1) / lo) ** ((turn + (r + 1) * 0.6180339887498949) % 1.0))) for r in range(n)]


def _layout(c):
    """What the requests look like: tokens held, tokens added, pages held, the first row of each."""
    lens = _spread(c["len_lo"], c["len_hi"], c["seqs"], 0.0)
    new = _spread(c["new_lo"], c["new_hi"], c["seqs"], 0.37)
    if c["kind"] == "tables":
        if c["new_hi"] > c["new_lo"]:  # a mixed step: decoding requests between the chunks
            new = [n if r % 5 == 0 else 1 for r, n in enumerate(new)]
        if c["finished"]:
            new = [-1 if r % c["finished"] == c["finished"] - 1 else 0 if r % 7 == 3 else n for r, n in enumerate(new)]
    starts = [0]
    for n in new:
        starts.append(starts[-1] + max(0, n))
    return lens, new, starts


def _pages(n, page):
    return -(-n // page)


# ---- inputs ------------------------------------------------------------------

def _ints(v):
    return torch.tensor(v, device=DEV, dtype=torch.int32)


def _table(lens, page, stride, perm):
    """Page tables of requests that hold `lens` tokens, their pages taken from `perm` in turn; -1 past them."""
    t = torch.full((len(lens), stride), -1, dtype=torch.int32)
    at, perm = 0, perm.cpu()
    for r, n in enumerate(lens):
        k = _pages(n, page)
        t[r, :k] = perm[at:at + k]
        at += k
    return t.to(DEV), at


def _cache(fmt, g, slots, kv_heads, head_dim):
    """K or V rows of about unit size in a cache's format."""
    if fmt == "f16":
        return torch.randn(slots, kv_heads, head_dim, generator=g, device=DEV, dtype=torch.float16)
    n = slots * kv_heads * head_dim // 32
    d = torch.rand(n, 1, generator=g, device=DEV) + 0.5
    if fmt == "q8_0":
        q = torch.randint(0, 256, (n, 32), generator=g, device=DEV, dtype=torch.uint8)
        return torch.cat([(d * (1.7 / 127)).half().view(torch.uint8), q], 1)
    q = torch.randint(0, 256, (n, 16), generator=g, device=DEV, dtype=torch.uint8)
    return torch.cat([(d * 0.22).half().view(torch.uint8), q], 1)


def prepare(case, seed):
    c = dict(case)
    g = torch.Generator(device=DEV).manual_seed(seed)
    lens, new, starts = _layout(c)
    n, page, rows = c["seqs"], c["page"], starts[-1]
    s = {"c": c, "rows": rows, "max_rows": max(1, rows + c["pad"]), "new": new, "before": lens, "added": _ints(new)}
    after = [0 if k < 0 else m + k for m, k in zip(lens, new)]
    held = lens if c["kind"] == "tables" else after
    s["stride"] = max(_pages(m + max(0, k), page) for m, k in zip(lens, new)) + 1
    prefix_pages = 0 if c["kind"] == "tables" else _pages(c["prefix"], page)
    used = sum(_pages(m, page) for m in held)
    s["n_pages"] = prefix_pages + used + (n + sum(_pages(max(0, k), page) for k in new) if c["kind"] == "tables" else 3)
    perm = torch.randperm(s["n_pages"], generator=g, device=DEV).to(torch.int32)
    s["prefix_table"] = perm[:prefix_pages].contiguous() if prefix_pages else _ints([0])
    s["table"], taken = _table(held, page, s["stride"], perm[prefix_pages:])
    s["row_start"] = _ints(starts)
    if c["kind"] == "tables":
        free = perm[taken:]
        s["free"] = torch.cat([free, torch.full((s["n_pages"] - free.numel(),), -1, device=DEV, dtype=torch.int32)])
        s["n_free"] = _ints([free.numel()])
        s.update(lens=_ints(lens), want=s["added"], lens_out=_ints([0] * n), n_free_out=_ints([0]),
                 row_start=_ints([0] * (n + 1)), slots=_ints([0] * s["max_rows"]), pos=_ints([0] * s["max_rows"]),
                 status=_ints([0] * n))
        torch.cuda.synchronize()
        return s
    h, kv, hd = c["heads"], c["kv_heads"], c["head_dim"]
    s["lens"] = _ints(after)
    s["k"], s["v"] = (_cache(c[f], g, s["n_pages"] * page, kv, hd) for f in ("k_format", "v_format"))
    at = torch.arange(rows, device=DEV)
    req = torch.repeat_interleave(torch.arange(n, device=DEV), s["added"].long())
    s["req"], s["i"] = req, at - s["row_start"].long()[req]  # the request of a row, and its place among the new ones
    own_pos = _ints(lens).long()[req] + s["i"]
    if c["kind"] == "append":
        slots = s["table"].long()[req, own_pos // page] * page + own_pos % page
        tail = torch.full((c["pad"],), -1, device=DEV, dtype=torch.int32)
        s["slots"] = torch.cat([slots.to(torch.int32), tail])
        s["pos"] = torch.cat([(own_pos + c["prefix"]).to(torch.int32), torch.zeros_like(tail)])
        s["qkv"] = torch.randn(s["max_rows"], (h + 2 * kv) * hd, generator=g, device=DEV)
        s["q"] = torch.zeros(s["max_rows"], h * hd, device=DEV)
        s["n_table"] = c["prefix"] + max(after)
        f = ROPE_BASE ** (-2.0 * torch.arange(hd // 2, device=DEV, dtype=torch.float64) / hd)
        a = torch.arange(s["n_table"], device=DEV, dtype=torch.float64)[:, None] * f
        s["angles"] = torch.stack([a.cos(), a.sin()], -1).float().contiguous()
    else:
        s["q"] = torch.randn(s["max_rows"], h * hd, generator=g, device=DEV)
        s["out"] = torch.zeros(s["max_rows"], h * hd, device=DEV)
    torch.cuda.synchronize()
    return s


# ---- one pass ----------------------------------------------------------------

def run(s):
    kind = s["c"]["kind"]
    if own:
        return {"tables": _own_tables, "append": _own_append, "attention": _own_attention}[kind](s)
    return {"tables": _plain_tables, "append": _plain_append, "attention": _plain_attention}[kind](s)


def _own_tables(s):
    c, dev = s["c"], _device()
    dev.block_tables(s["lens"].data_ptr(), s["want"].data_ptr(), c["seqs"], s["table"].data_ptr(), s["stride"],
                     c["page"], s["free"].data_ptr(), s["n_free"].data_ptr(), s["n_pages"], s["lens_out"].data_ptr(),
                     s["n_free_out"].data_ptr(), s["row_start"].data_ptr(), s["slots"].data_ptr(), s["pos"].data_ptr(),
                     s["max_rows"], s["status"].data_ptr(), c["prefix"])
    return _tables_out(s)


def _own_append(s):
    c, dev = s["c"], _device()
    dev.qkv_postprocess_paged(s["qkv"].data_ptr(), s["q"].data_ptr(), s["k"].data_ptr(), s["v"].data_ptr(),
                              s["slots"].data_ptr(), s["pos"].data_ptr(), s["max_rows"], s["n_pages"], c["page"],
                              c["heads"], c["kv_heads"], c["head_dim"], ROPE_BASE, FORMATS[c["k_format"]],
                              FORMATS[c["v_format"]], table=s["angles"].data_ptr(), n_table=s["n_table"])
    return {"q": s["q"], "k": s["k"], "v": s["v"]}


def _own_attention(s):
    c, dev = s["c"], _device()
    dev.attention_paged(s["q"].data_ptr(), s["k"].data_ptr(), s["v"].data_ptr(), s["out"].data_ptr(), s["n_pages"],
                        c["page"], s["prefix_table"].data_ptr(), c["prefix"], s["table"].data_ptr(), s["stride"],
                        s["lens"].data_ptr(), s["row_start"].data_ptr(), c["seqs"], s["max_rows"], c["heads"],
                        c["kv_heads"], c["head_dim"], 1.0 / math.sqrt(c["head_dim"]), c["window"] or None,
                        FORMATS[c["k_format"]], FORMATS[c["v_format"]])
    return {"out": s["out"]}


def _tables_out(s):
    return {k: s[k] for k in ("lens_out", "n_free_out", "row_start", "slots", "pos", "status", "table", "free")}


def _plain_tables(s):
    c = s["c"]
    page, lens, want, table, free = c["page"], s["lens"].long(), s["want"].long(), s["table"], s["free"]
    cols = torch.arange(s["stride"], device=DEV)
    held = (lens + page - 1) // page
    # pages of finished requests go onto the free list, in the requests' order
    back = torch.where(want == -1, held, 0)
    ends = torch.cumsum(back, 0)
    total = s["n_free"].long() + ends[-1]
    f = torch.arange(s["n_pages"], device=DEV) - s["n_free"].long()
    r = torch.searchsorted(ends, f, right=True).clamp(max=c["seqs"] - 1)
    given = (f >= 0) & (f < ends[-1])
    free.copy_(torch.where(given, table[r, torch.where(given, f - ends[r] + back[r], 0)], free))
    # served: valid, its table row long enough, its rows and new pages still there
    bad = (want < -1) | (lens < 0) | (lens > s["stride"] * page)
    ok = (want >= 0) & ~bad
    full = ok & ((lens + want + page - 1) // page > s["stride"])
    add = torch.where(ok & ~full, want, 0)
    need = (lens + add + page - 1) // page - held
    need = torch.where(ok & ~full, need, 0)
    no_rows = (add > 0) & (torch.cumsum(add, 0) > s["max_rows"])
    no_pages = ~no_rows & (need > 0) & (torch.cumsum(need, 0) > total)
    status = torch.where(full, 2, torch.where(no_rows, 3, torch.where(no_pages, 1, 0)))
    status = torch.where(bad, 4, status)
    served = status == 0
    before = torch.cumsum(need, 0) - need
    add, need = torch.where(served, add, 0), torch.where(served, need, 0)
    # new pages from the top of the free list
    k = cols - held[:, None]
    take = (k >= 0) & (k < need[:, None])
    table.copy_(torch.where(take, free[torch.where(take, total - 1 - before[:, None] - k, 0)], table))
    s["lens_out"].copy_(torch.where(served & (want == -1), 0, lens + add))
    s["n_free_out"].copy_(total - need.sum())
    ends = torch.cumsum(add, 0)
    s["row_start"][0] = 0
    s["row_start"][1:] = ends
    s["status"].copy_(status)
    row = torch.arange(s["max_rows"], device=DEV)
    r = torch.searchsorted(ends, row, right=True)
    used = r < c["seqs"]
    r = torch.where(used, r, 0)
    p = lens[r] + row - (ends[r] - add[r])
    page_of = table.long()[r, torch.where(used, p // page, 0)]
    s["slots"].copy_(torch.where(used, page_of * page + p % page, -1))
    s["pos"].copy_(torch.where(used, p + c["prefix"], 0))
    return _tables_out(s)


def _plain_append(s):
    c, n = s["c"], s["rows"]
    h, kv, hd = c["heads"], c["kv_heads"], c["head_dim"]
    x = s["qkv"][:n].view(n, h + 2 * kv, hd)
    cs = s["angles"][s["pos"][:n].long()][:, None]
    cos, sin = cs[..., 0], cs[..., 1]
    lo, hi = x[:, :h + kv, :hd // 2], x[:, :h + kv, hd // 2:]
    turned = torch.cat([lo * cos - hi * sin, lo * sin + hi * cos], -1)
    at = s["slots"][:n].long()
    s["q"][:n] = turned[:, :h].reshape(n, h * hd)
    s["k"][at] = turned[:, h:].half()
    s["v"][at] = x[:, h + kv:].half()
    return {"q": s["q"], "k": s["k"], "v": s["v"]}


def _values(raw, fmt, slots, kv, hd):
    """The rows at `slots`, as the 32-bit values they stand for."""
    shape = (*slots.shape, kv, hd)
    if fmt == "f16":
        return raw.view(-1, kv, hd)[slots].float()
    b = raw.view(-1, kv * hd // 32, BLOCK_BYTES[fmt])[slots]
    d = b[..., :2].contiguous().view(torch.float16).float()
    if fmt == "q8_0":
        return (d * b[..., 2:].contiguous().view(torch.int8).float()).view(shape)
    return (d * (torch.cat([b[..., 2:] & 15, b[..., 2:] >> 4], -1).float() - 8)).view(shape)


def _rounded_q(q):
    """q as Q8_0 blocks of 32, which is what quantised K rows are multiplied with: the scale amax/127 kept as a
    truncated half, the quants rounded half away from zero by the untruncated one."""
    x = q.reshape(-1, 32)
    scale = x.abs().amax(1, keepdim=True) / 127.0
    half = scale.half()
    half = torch.where(half.float() > scale, (half.view(torch.int16) - 1).view(torch.float16), half)
    half = torch.where(half.float() < 2.0 ** -14, 0.0, half.float())
    t = (x * torch.where(scale > 0, 1.0 / scale, 0.0)).double()
    return (half * (torch.sign(t) * torch.floor(t.abs() + 0.5)).clamp(-128, 127).float()).view(q.shape)


def _plain_attention(s):
    c, n, rows = s["c"], s["c"]["seqs"], s["rows"]
    h, kv, hd, page = c["heads"], c["kv_heads"], c["head_dim"], c["page"]
    grp, prefix, most, new = h // kv, c["prefix"], max(m + k for m, k in zip(s["before"], s["new"])), max(s["new"])
    q = s["q"][:rows].view(rows, h, hd) / math.sqrt(hd) if c["k_format"] == "f16" else \
        _rounded_q(s["q"][:rows].view(rows, h, hd)) / math.sqrt(hd)
    # the shared prefix, once for all rows
    t = torch.arange(prefix, device=DEV)
    slots = s["prefix_table"].long()[t // page] * page + t % page
    kp, vp = (_values(s[x], c[x + "_format"], slots, kv, hd).transpose(0, 1).contiguous() for x in ("k", "v"))
    qp = q.view(rows, kv, grp, hd).transpose(0, 1).reshape(kv, rows * grp, hd)
    sp = torch.matmul(qp, kp.transpose(1, 2).contiguous()).view(kv, rows, grp, prefix)
    # every request's own positions, padded to the longest
    u = torch.arange(most, device=DEV)
    slots = s["table"].long()[:, u // page] * page + u % page
    slots = torch.where(u < s["lens"][:, None], slots, 0)
    ko, vo = (_values(s[x], c[x + "_format"], slots, kv, hd).transpose(1, 2).contiguous() for x in ("k", "v"))
    qo = torch.zeros(n, new, h, hd, device=DEV)
    qo[s["req"], s["i"]] = q
    qo = qo.view(n, new, kv, grp, hd).permute(0, 2, 1, 3, 4).reshape(n, kv, new * grp, hd)
    so = torch.matmul(qo, ko.transpose(2, 3).contiguous()).view(n, kv, new, grp, most)
    so = so.permute(0, 2, 1, 3, 4)[s["req"], s["i"]].transpose(0, 1)  # [kv, rows, grp, most]
    # what a row sees: up to itself, and no further back than the window
    at = (s["lens"] - s["added"]).long()[s["req"]] + s["i"] + prefix
    first = at - c["window"] + 1 if c["window"] else torch.zeros_like(at)
    see_p = (t >= first[:, None]) & (t <= at[:, None])
    see_o = (u + prefix >= first[:, None]) & (u + prefix <= at[:, None])
    sc = torch.cat([sp.masked_fill(~see_p[None, :, None], -math.inf),
                    so.masked_fill(~see_o[None, :, None], -math.inf)], -1)
    p = torch.exp(sc - sc.amax(-1, keepdim=True))
    total = p.sum(-1, keepdim=True)
    out = torch.matmul(p[..., :prefix].reshape(kv, rows * grp, prefix), vp).view(kv, rows, grp, hd)
    po = torch.zeros(n, new, kv, grp, most, device=DEV)
    po[s["req"], s["i"]] = p[..., prefix:].transpose(0, 1)
    po = po.permute(0, 2, 1, 3, 4).reshape(n, kv, new * grp, most)
    oo = torch.matmul(po, vo).view(n, kv, new, grp, hd).permute(0, 2, 1, 3, 4)[s["req"], s["i"]].transpose(0, 1)
    s["out"][:rows] = ((out + oo) / total).transpose(0, 1).reshape(rows, h * hd)
    return {"out": s["out"]}


# ---- bytes and operations ----------------------------------------------------

def work(case):
    c = case
    lens, new, starts = _layout(c)
    rows, page = starts[-1], c["page"]
    if c["kind"] == "tables":
        pages = sum(_pages(m + max(0, k), page) - _pages(m, page) for m, k in zip(lens, new))
        back = sum(_pages(m, page) for m, k in zip(lens, new) if k < 0)
        # lengths in and out, tokens wanted, status, first rows; a place and a position a row; a page id in and out
        return {"bytes": 4.0 * (5 * c["seqs"] + 2 * (rows + c["pad"]) + 2 * (pages + back) + min(rows, c["seqs"])),
                "flops": 4.0 * (rows + c["seqs"])}
    h, kv, hd = c["heads"], c["kv_heads"], c["head_dim"]
    per = kv * hd * (BYTES_PER_VALUE[c["k_format"]] + BYTES_PER_VALUE[c["v_format"]])
    if c["kind"] == "append":
        distinct = len({m + i for m, k in zip(lens, new) for i in range(k)})
        return {"bytes": rows * (4.0 * (2 * h + 2 * kv) * hd + per + 8) + 4.0 * distinct * hd,
                "flops": 3.0 * rows * (h + kv) * hd}
    w, prefix = c["window"] or 1 << 40, c["prefix"]
    seen, own_rows, low = 0, 0, prefix
    for m, k in zip(lens, new):
        firsts = [max(0, prefix + m + i + 1 - w) for i in range(k)]
        seen += sum(prefix + m + i + 1 - f for i, f in enumerate(firsts))
        own_rows += m + k - max(0, firsts[0] - prefix)
        low = min(low, firsts[0])
    return {"bytes": (prefix - min(low, prefix) + own_rows) * per + 8.0 * rows * h * hd,
            "flops": 4.0 * hd * h * seen}


# ---- the same in 64 bits -----------------------------------------------------

def _row64(raw, fmt, slots, kv, hd):
    if fmt == "f16":
        return raw.reshape(-1, kv, hd).index_select(0, slots).double()
    size = BLOCK_BYTES[fmt]
    b = raw.reshape(-1, kv * hd // 32, size).index_select(0, slots)
    d = b[:, :, 0:2].contiguous().view(torch.float16).double()
    if fmt == "q8_0":
        q = b[:, :, 2:].to(torch.int64)
        q = q - 256 * (q > 127)
    else:
        q = torch.empty(*b.shape[:2], 32, device=b.device, dtype=torch.int64)
        q[:, :, :16] = b[:, :, 2:].to(torch.int64) % 16 - 8
        q[:, :, 16:] = b[:, :, 2:].to(torch.int64) // 16 - 8
    return (d * q).reshape(slots.numel(), kv, hd)


def _q64(q, fmt):
    """Query rows in 64 bits; behind a quantised K as the Q8_0 values that are multiplied with it."""
    if fmt == "f16":
        return q.double()
    out = torch.empty_like(q, dtype=torch.float64)
    for b in range(q.shape[-1] // 32):
        x = q[..., 32 * b:32 * b + 32]
        top = x.abs().max(-1, keepdim=True).values
        scale = top / 127.0  # in 32 bits: the quantiser's own division
        bits = scale.view(torch.int32)
        d = (bits & ~0x1FFF).view(torch.float32).double()  # the mantissa's upper ten bits
        d = torch.where(scale < 2.0 ** -14, torch.zeros_like(d), d)
        v = (x * torch.where(scale > 0, torch.ones_like(scale) / scale, torch.zeros_like(scale))).double()
        r = torch.where(v < 0, -torch.floor(-v + 0.5), torch.floor(v + 0.5)).clamp(-128, 127)
        out[..., 32 * b:32 * b + 32] = d * r
    return out


def exact(case, seed):
    if case["kind"] == "tables":
        return None
    s = prepare(case, seed)
    c, n, page = s["c"], s["rows"], s["c"]["page"]
    h, kv, hd = c["heads"], c["kv_heads"], c["head_dim"]
    if c["kind"] == "append":
        x = s["qkv"].double().view(s["max_rows"], h + 2 * kv, hd)
        q, k, v = (torch.zeros(s["max_rows"], h, hd, device=DEV, dtype=torch.float64), s["k"].double(), s["v"].double())
        cs = s["angles"].double()[s["pos"].long()]
        z = torch.complex(x[:n, :h + kv, :hd // 2], x[:n, :h + kv, hd // 2:]) * torch.complex(cs[:n, None, :, 0], cs[:n, None, :, 1])
        for part, lo, hi in ((q, 0, h), (k, h, h + kv)):
            both = torch.cat([z[:, lo:hi].real, z[:, lo:hi].imag], -1)
            if part is q:
                q[:n] = both
            else:
                k[s["slots"][:n].long()] = both
        v[s["slots"][:n].long()] = x[:n, h + kv:]
        return {"q": q.view(s["max_rows"], h * hd), "k": k, "v": v}
    out = torch.zeros(s["max_rows"], h, hd, device=DEV, dtype=torch.float64)
    q = _q64(s["q"].view(s["max_rows"], h, hd), c["k_format"])
    t = torch.arange(c["prefix"], device=DEV)
    shared = s["prefix_table"].long()[t // page] * page + t % page
    kp, vp = _row64(s["k"], c["k_format"], shared, kv, hd), _row64(s["v"], c["v_format"], shared, kv, hd)
    row = 0
    for r, (held, add) in enumerate(zip(s["before"], s["new"])):
        u = torch.arange(held + add, device=DEV)
        mine = s["table"][r].long()[u // page] * page + u % page
        k = torch.cat([kp, _row64(s["k"], c["k_format"], mine, kv, hd)])
        v = torch.cat([vp, _row64(s["v"], c["v_format"], mine, kv, hd)])
        where = torch.arange(k.shape[0], device=DEV)
        at = (c["prefix"] + held + torch.arange(add, device=DEV))[:, None]
        hidden = where > at
        if c["window"]:
            hidden |= where <= at - c["window"]
        for head in range(h):
            sc = q[row:row + add, head] @ k[:, head * kv // h].T.contiguous() / hd ** 0.5
            p = torch.softmax(sc.masked_fill(hidden, -math.inf), -1)
            out[row:row + add, head] = p @ v[:, head * kv // h].contiguous()
        row += add
    return {"out": out.view(s["max_rows"], h * hd)}
