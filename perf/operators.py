"""The 8-bit block-scaled K/V cache as cases that can be timed and compared: its writer and reader, the verify attention
over it, the attention weight each key has drawn, and the eviction those weights decide.

  append  K/V rows of new positions coded into the pages, then read back as fp32 rows
  attend  verify attention of one layer over the pages (1 to 64 tokens, hundreds to 128k keys), with its log-sum-exp
  mass    the attention weights of a round's committed rows added to every key's account
  evict   the keys of most weight kept (with the first and the last ones), compacted into other pages and read back

Pages hold 32 positions: codes [page][KV head][32][D] of one byte (int8 or e4m3), one fp32 scale for each page and head;
a value is code * scale. Sizes are those of the 16-layer configuration (32/8/64 heads) and of the reference geometry
(16/4/128), and others around them.

With `own` false the operators are computed in their plain form on the same pages; with `own` true by the framework.
"""
import importlib.util
import math
import os
import sys
import zlib

import torch

PAGE = 32
DEV = "cuda"
own = False


def _host():
    """The binding (its folder's name is not a Python identifier)."""
    name = "dspark_amd_host"
    if name not in sys.modules:
        path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "lfm3-1.7b-mi50_amd", "dspark.py")
        spec = importlib.util.spec_from_file_location(name, path)
        mod = importlib.util.module_from_spec(spec)
        sys.modules[name] = mod
        spec.loader.exec_module(mod)
    return sys.modules[name]


# ------------------------------------------------------------------------------------------------ the cases
def listed():
    return [
        # one verified block's K/V appended in mid-page at 32k: a call of every layer and round
        {"name": "append_block", "kind": "append", "code": "e4m3", "kv_heads": 8, "head_dim": 64, "pos0": 32749, "n": 16},
        # a chunk of a prompt behind a cached prefix, not page-aligned
        {"name": "append_chunk", "kind": "append", "code": "int8", "kv_heads": 8, "head_dim": 64, "pos0": 1003, "n": 8192},
        # a whole long prompt, wide heads
        {"name": "append_prompt", "kind": "append", "code": "e4m3", "kv_heads": 4, "head_dim": 128, "pos0": 0, "n": 32768},
        # a draft block early in a conversation, wide heads, ragged length
        {"name": "attend_short", "kind": "attend", "code": "e4m3", "q_heads": 16, "kv_heads": 4, "head_dim": 128,
         "ctx": 1001, "tokens": 8, "start": 0, "window": 0, "causal": True, "gate": True},
        # plain decoding: a single token at 32k
        {"name": "attend_token", "kind": "attend", "code": "int8", "q_heads": 32, "kv_heads": 8, "head_dim": 64,
         "ctx": 32768, "tokens": 1, "start": 0, "window": 0, "causal": True, "gate": False},
        # a 16-token block at 32k keys
        {"name": "attend_32k", "kind": "attend", "code": "e4m3", "q_heads": 32, "kv_heads": 8, "head_dim": 64,
         "ctx": 32768, "tokens": 16, "start": 0, "window": 0, "causal": True, "gate": True},
        # the reference geometry's verify width at the longest context
        {"name": "attend_128k", "kind": "attend", "code": "int8", "q_heads": 16, "kv_heads": 4, "head_dim": 128,
         "ctx": 131063, "tokens": 9, "start": 0, "window": 0, "causal": True, "gate": True},
        # the widest block of the configurations at the longest context
        {"name": "attend_128k_wide", "kind": "attend", "code": "e4m3", "q_heads": 32, "kv_heads": 8, "head_dim": 64,
         "ctx": 131072, "tokens": 33, "start": 0, "window": 0, "causal": True, "gate": False},
        # the account after a round early in a conversation
        {"name": "mass_short", "kind": "mass", "code": "int8", "q_heads": 16, "kv_heads": 4, "head_dim": 128, "ctx": 4099,
         "tokens": 8, "rows": 5, "start": 0, "window": 0, "causal": True},
        # the same for a fully accepted 16-token block at the longest context
        {"name": "mass_128k", "kind": "mass", "code": "e4m3", "q_heads": 32, "kv_heads": 8, "head_dim": 64, "ctx": 131072,
         "tokens": 16, "rows": 16, "start": 0, "window": 0, "causal": True},
        # a cache held at 8192 positions: what a few hundred new ones pushed out
        {"name": "evict_step", "kind": "evict", "code": "int8", "kv_heads": 8, "head_dim": 64, "length": 8709, "keep": 8192,
         "sinks": 4, "recent": 256},
        # a long prompt's cache cut to an eighth
        {"name": "evict_prompt", "kind": "evict", "code": "e4m3", "kv_heads": 4, "head_dim": 128, "length": 131072,
         "keep": 16384, "sinks": 4, "recent": 1024},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["append", "attend", "attend", "mass", "evict"])
    q_heads, kv_heads, dim = rng.choice([(32, 8, 64), (16, 4, 128), (16, 4, 128), (16, 2, 64), (8, 8, 128)])
    case = {"kind": kind, "code": rng.choice(["int8", "e4m3"]), "kv_heads": kv_heads, "head_dim": dim}
    if kind == "append":
        return {**case, "pos0": rng.randint(0, 40000), "n": _log(rng, 1, 16384)}
    if kind == "evict":
        length = _log(rng, 300, 131072)
        keep = min(16384, max(1, int(length * rng.uniform(0.05, 0.98))))
        sinks = rng.randint(0, min(16, keep))
        return {**case, "length": length, "keep": keep, "sinks": sinks, "recent": int((keep - sinks) * rng.uniform(0, 0.5))}
    tokens = rng.choice([1, 4, 8, 9, 16, 33, rng.randint(1, 64)])
    ctx = _log(rng, 40, 131072 if tokens <= 16 else 32768)
    case.update(q_heads=q_heads, ctx=ctx, tokens=tokens, start=rng.choice([0, 0, rng.randint(0, ctx)]),
                window=rng.choice([0, 0, 256, _log(rng, 64, 4096)]))
    if kind == "mass":
        return {**case, "rows": rng.randint(1, tokens), "causal": True}
    return {**case, "causal": rng.random() < 0.8, "gate": rng.random() < 0.5}


# ------------------------------------------------------------------------------------------------ inputs
def _gen(seed, name):
    g = torch.Generator(device=DEV)
    g.manual_seed((int(seed) << 32) ^ zlib.crc32(name.encode()))
    return g


def _randn(seed, name, shape, std=1.0, dtype=torch.float16):
    return torch.randn(shape, generator=_gen(seed, name), device=DEV).mul_(std).to(dtype)


def _rand(seed, name, shape, lo, hi):
    return torch.rand(shape, generator=_gen(seed, name), device=DEV).mul_(hi - lo).add_(lo)


def _pages(n):
    return (n + PAGE - 1) // PAGE


def _scale_of(code, amax):
    """The scale of a block whose largest magnitude is amax: int8, amax / 127 rounded up to 16 significant bits (so that
    code * scale is exact in fp32); e4m3, the least power of two that takes amax to at most 448."""
    if code == "int8":
        s = (amax.double() / 127).float()
        return ((s.view(torch.int32) + 255) & ~255).view(torch.float32)
    m, e = torch.frexp(amax.double() / 448)
    return torch.where(amax > 0, torch.exp2((e - (m == 0.5).to(e.dtype)).double()), torch.zeros_like(m)).float()


def _code_of(code, x, scale):
    """x / scale (scale broadcast, 0 where a block is all zeros) rounded once to a code."""
    y = torch.where(scale > 0, x.double() / scale.double(), torch.zeros((), dtype=torch.float64, device=x.device))
    return y.round().clamp(-127, 127).to(torch.int8) if code == "int8" else y.float().to(torch.float8_e4m3fn)


def _pool(seed, name, code, n_pages, kv_heads, dim):
    """Codes and scales of a cache that holds unit-normal values, blocks of other sizes among them."""
    amax = _rand(seed, name + ".amax", (n_pages, kv_heads), 0.0, 1.0).mul_(1.5).exp2_().mul_(2.5).half()
    scale = _scale_of(code, amax)
    top = 127 if code == "int8" else 448
    y = torch.randn((n_pages, kv_heads, PAGE, dim), generator=_gen(seed, name), device=DEV).mul_(top / 4).clamp_(-top, top)
    return (y.round_().to(torch.int8) if code == "int8" else y.to(torch.float8_e4m3fn)), scale


def _table(seed, name, n_pages):
    """A block table as a long-running cache has it: the logical pages anywhere in the pool."""
    return torch.randperm(n_pages, generator=_gen(seed, name), device=DEV).to(torch.int32)


def prepare(case, seed):
    s = dict(case)
    code, H, D = case["code"], case["kv_heads"], case["head_dim"]
    if case["kind"] == "append":
        end = case["pos0"] + case["n"]
    elif case["kind"] == "evict":
        end = case["length"]
    else:
        end = case["ctx"] + case["tokens"]
    n = _pages(end)
    k, ks = _pool(seed, "k", code, n, H, D)
    v, vs = _pool(seed, "v", code, n, H, D)
    s["cache"] = {"k": k, "v": v, "k_scale": ks, "v_scale": vs, "block_table": _table(seed, "table", n)}
    if case["kind"] == "append":  # K and V lie side by side in a row, as a projection writes them
        row = _randn(seed, "rows", (case["n"], 2 * H, D))
        row.mul_(_rand(seed, "size", (case["n"], 1, 1), 0.5, 2.0))
        s["rows"] = row[:, :H], row[:, H:]
    elif case["kind"] == "evict":
        m = _pages(case["keep"])
        kind = torch.int8 if code == "int8" else torch.float8_e4m3fn
        s["dst"] = {"k": torch.zeros((m, H, PAGE, D), dtype=torch.uint8, device=DEV).view(kind),
                    "v": torch.zeros((m, H, PAGE, D), dtype=torch.uint8, device=DEV).view(kind),
                    "k_scale": torch.zeros((m, H), device=DEV), "v_scale": torch.zeros((m, H), device=DEV),
                    "block_table": _table(seed, "dst", m)}
        # accounts of keys: most have drawn little, some a lot, and the oldest ones (fp32 steps apart) often the same
        s["mass"] = _randn(seed, "mass", (H, end), 2.0, torch.float32).exp_().half().float()
    else:
        QH, M = case["q_heads"], case["tokens"]
        s["q"] = _randn(seed, "q", (M, QH, D))
        if case["kind"] == "attend":
            s["gate"] = _randn(seed, "gate", (M, QH), dtype=torch.float32) if case["gate"] else None
        else:
            s["mass"] = _randn(seed, "mass", (H, end), 1.0, torch.float32).exp_()
            s["lse"] = _lse64(s).float()
            s["rows"] = torch.tensor([case["rows"]], dtype=torch.int32, device=DEV)
            s["account"] = torch.zeros((H, end), device=DEV)
    if own:  # the handles and buffers that a serving loop keeps
        h = _host()
        s["host"], s["workspace"] = h, h.Workspace(DEV)
        s["cache_h"] = h.B8Cache(**s["cache"])
        if "dst" in s:
            s["dst_h"] = h.B8Cache(**s["dst"])
    return s


# ------------------------------------------------------------------------------------------------ the plain forms
def _logical(cache, pool, pages):
    """The codes [KV head][32 pages][D] and their scales [KV head][32 pages][1] of logical pages `pages` (a slice)."""
    at = cache["block_table"][pages].long()
    codes, scale = cache[pool].view(torch.uint8)[at].view(cache[pool].dtype), cache[pool + "_scale"][at]
    P, H, _, D = codes.shape
    return codes.transpose(0, 1).reshape(H, P * PAGE, D), scale.t().repeat_interleave(PAGE, 1).unsqueeze(-1)


def _values(cache, pool, pages):
    codes, scale = _logical(cache, pool, pages)
    return codes.float() * scale


def _seen(s, T):
    """Which keys each token sees, [tokens][keys]: context keys by start and window, the block's by causal."""
    a, M = s["ctx"], s["tokens"]
    p, t = torch.arange(T, device=DEV), torch.arange(M, device=DEV)[:, None]
    ctx = (p < a) & (p >= s["start"])
    if s["window"]:
        ctx = ctx & (p > a + t - s["window"])
    return ctx | ((p >= a) & (p < a + M) & ((p - a <= t) | (not s["causal"])))


def _scores(s, dtype):
    """q k / sqrt(D) of every query row and key, [KV head][tokens][group][keys], masked."""
    H, D, M = s["kv_heads"], s["head_dim"], s["tokens"]
    k = _values(s["cache"], "k", slice(None)).to(dtype)
    q = s["q"].to(dtype).view(M, H, -1, D).transpose(0, 1).reshape(H, -1, D)
    x = torch.matmul(q, k.transpose(1, 2)).div_(math.sqrt(D)).view(H, M, -1, k.shape[1])
    return x.masked_fill_(~_seen(s, k.shape[1])[:, None, :], -math.inf)


def _lse64(s):
    x = _scores(s, torch.float64)
    m = x.amax(-1, keepdim=True)
    return (x.sub_(m).exp_().sum(-1).log() + m[..., 0]).permute(1, 0, 2).reshape(s["tokens"], -1)


def _attend(s):
    H, D, M = s["kv_heads"], s["head_dim"], s["tokens"]
    x = _scores(s, torch.float32)
    m = x.amax(-1, keepdim=True)
    p = x.sub_(m).exp_()
    l = p.sum(-1, keepdim=True)
    o = torch.matmul(p.view(H, -1, p.shape[-1]), _values(s["cache"], "v", slice(None))).view(H, M, -1, D) / l
    o = o.permute(1, 0, 2, 3).reshape(M, -1, D)
    if s["gate"] is not None:
        o = o * (1 / (1 + torch.exp(-s["gate"])))[..., None]
    return {"out": o.half(), "lse": (l.log() + m)[..., 0].permute(1, 0, 2).reshape(M, -1)}


def _mass(s):
    H, M, a, rows = s["kv_heads"], s["tokens"], s["ctx"], s["rows"]
    p = _scores(s, torch.float32).sub_(s["lse"].view(M, H, -1).permute(1, 0, 2)[..., None]).exp_()[..., :a + M]
    p = p * (torch.arange(M, device=DEV) < rows)[:, None, None]
    at = torch.arange(a + M, device=DEV)
    new = torch.where(at < a, s["mass"], torch.zeros_like(s["mass"])) + p.sum((1, 2))
    return {"mass": torch.where(at < a + rows, new, torch.zeros_like(new))}


def _append(s):
    c, code, pos0, n, H, D = s["cache"], s["code"], s["pos0"], s["n"], s["kv_heads"], s["head_dim"]
    first, s0, last = pos0 // PAGE, pos0 % PAGE, (pos0 + n - 1) // PAGE
    at, P = c["block_table"][first:last + 1].long(), last + 1 - first
    old = (torch.arange(P * PAGE, device=DEV) < s0).view(P, 1, PAGE, 1)  # rows of the first page that stay
    out = {}
    for name, rows in zip("kv", s["rows"]):
        x = torch.zeros((P * PAGE, H, D), device=DEV)
        x[s0:s0 + n] = rows.float()
        x = x.view(P, PAGE, H, D).transpose(1, 2)
        was, grown = c[name + "_scale"][at], _scale_of(code, x.abs().amax((2, 3)))
        if s0:
            grown[0] = torch.maximum(grown[0], was[0])
        held = c[name].view(torch.uint8)[at].view(c[name].dtype).float() * was[:, :, None, None]
        y = _code_of(code, torch.where(old, held, x), grown[:, :, None, None])
        c[name].view(torch.uint8)[at] = y.view(torch.uint8)
        c[name + "_scale"][at] = grown
        out[name] = _values(c, name, slice(first, last + 1)).transpose(0, 1)[:s0 + n]
        out[name + "_scale"] = c[name + "_scale"]
    return out


def _evict(s):
    c, dst, code, T, keep = s["cache"], s["dst"], s["code"], s["length"], s["keep"]
    H, D, sinks, recent = s["kv_heads"], s["head_dim"], s["sinks"], s["recent"]
    top = torch.sort(s["mass"][:, sinks:T - recent], dim=1, descending=True, stable=True)[1][:, :keep - sinks - recent] + sinks
    edge = torch.cat([torch.arange(sinks, device=DEV), torch.arange(T - recent, T, device=DEV)])
    kept = torch.cat([edge.expand(H, -1), top], 1).sort(1)[0]
    m = _pages(keep)
    out = {"kept": kept.int(), "mass": s["mass"].gather(1, kept)}
    for name in "kv":
        codes, scale = _logical(c, name, slice(None))
        codes = codes.view(torch.uint8).gather(1, kept[..., None].expand(-1, -1, D)).view(codes.dtype)
        scale = scale.gather(1, kept[..., None])
        x = torch.zeros((2, H, m * PAGE, D), device=DEV)
        x[0, :, :keep], x[1, :, :keep] = codes.float() * scale, scale
        x = x.view(2, H, m, PAGE, D)
        block = x[1].amax((2, 3))
        y = _code_of(code, x[0], block[..., None, None])
        at = dst["block_table"].long()
        dst[name].view(torch.uint8)[at] = y.view(torch.uint8).transpose(0, 1)
        dst[name + "_scale"][at] = block.t()
        out[name] = _values(dst, name, slice(None)).transpose(0, 1)[:keep]
        out[name + "_scale"] = dst[name + "_scale"]
    return out


# ------------------------------------------------------------------------------------------------ the framework's calls
def _own(s):
    h, c = s["host"], s["cache_h"]
    if s["kind"] == "append":
        h.kv_write_b8(*s["rows"], c, s["pos0"])
        first = s["pos0"] // PAGE * PAGE
        k, v = h.kv_read_b8(c, first, s["pos0"] + s["n"] - first)
        return {"k": k, "k_scale": s["cache"]["k_scale"], "v": v, "v_scale": s["cache"]["v_scale"]}
    if s["kind"] == "attend":
        lse = torch.empty(s["q"].shape[:2], device=DEV)
        out, _ = h.verify_attention_b8(s["q"], c, s["ctx"], start=s["start"], window=s["window"], causal=s["causal"],
                                       gate=s["gate"], lse=lse, workspace=s["workspace"])
        return {"out": out, "lse": lse}
    if s["kind"] == "mass":
        h.attention_mass_b8(s["q"], c, s["ctx"], s["lse"], s["account"], mass_in=s["mass"], rows=s["rows"], start=s["start"],
                            window=s["window"], causal=s["causal"])
        return {"mass": s["account"]}
    kept, mass = h.kv_evict_b8(c, s["dst_h"], s["length"], s["keep"], s["mass"], sinks=s["sinks"], recent=s["recent"],
                               workspace=s["workspace"])
    k, v = h.kv_read_b8(s["dst_h"], 0, s["keep"])
    d = s["dst"]
    return {"kept": kept, "mass": mass, "k": k, "k_scale": d["k_scale"], "v": v, "v_scale": d["v_scale"]}


def run(state):
    if own:
        return _own(state)
    return {"append": _append, "attend": _attend, "mass": _mass, "evict": _evict}[state["kind"]](state)


# ------------------------------------------------------------------------------------------------ work and exact values
def work(case):
    H, D = case["kv_heads"], case["head_dim"]
    if case["kind"] == "append":  # rows in, codes stored, values out; the page's earlier rows with them
        s0 = case["pos0"] % PAGE
        n, m = case["n"], s0 + case["n"]
        return {"bytes": 2 * H * (D * (2 * n + s0 + m + 4 * m) + 4 * _pages(m)), "flops": 4 * H * D * m}
    if case["kind"] == "evict":  # the accounts, then the kept rows: read, stored, and out as values
        T, keep = case["length"], case["keep"]
        return {"bytes": H * (4 * T + 8 * keep + 2 * D * keep * (1 + 1 + 4) + 8 * (_pages(T) + _pages(keep))),
                "flops": 2 * H * D * keep}
    QH, M, a = case["q_heads"], case["tokens"], case["ctx"]
    rows = case.get("rows", M)
    lo = max(case["start"], a - case["window"] + 1 if case["window"] else 0, 0)
    T = max(0, a - lo) + rows
    if case["kind"] == "attend":
        return {"bytes": H * (2 * T * D + 8 * _pages(T)) + QH * M * (4 * D + 4 + 4 * case["gate"]), "flops": 4 * QH * M * D * T}
    return {"bytes": H * (T * D + 4 * _pages(T) + 8 * a) + QH * rows * (2 * D + 4), "flops": 2 * QH * rows * D * T}


def _e4m3_table():
    """The 256 values of e4m3: sign, 4 exponent bits (bias 7, 0 the subnormals), 3 mantissa bits; all ones is no number."""
    b = torch.arange(256, device=DEV)
    e, m = (b >> 3) & 15, (b & 7).double()
    v = torch.where(e > 0, (8 + m) * torch.exp2((e - 10).double()), m * 2.0 ** -9)
    v = torch.where((b & 127) == 127, torch.full_like(v, math.nan), v)
    return torch.where(b > 127, -v, v)


def _decoded(cache, pool, code, n):
    """Positions 0 .. n - 1 in 64 bits, [n][KV head][D], and their blocks' scales [n][KV head]."""
    raw = cache[pool].view(torch.uint8).long()
    val = torch.where(raw > 127, raw - 256, raw).double() if code == "int8" else _e4m3_table()[raw]
    p = torch.arange(n, device=DEV)
    page, slot = cache["block_table"].long()[p // PAGE], p % PAGE
    scale = cache[pool + "_scale"].double()[page]
    return val[page, :, slot] * scale[..., None], scale


def _coded64(code, x, scale):
    """What the nearest code of x stands for (ties to the even one), in 64 bits; scale broadcasts."""
    y = x / torch.where(scale > 0, scale, torch.ones_like(scale))
    if code == "int8":
        step = torch.ones_like(y)
    else:
        step = torch.exp2(torch.floor(torch.log2(y.abs().clamp_min(2.0 ** -20))).clamp_min(-6) - 3)
    return torch.round(y / step) * step * scale


def _scale64(code, amax):
    if code == "int8":
        b = torch.frexp((amax / 127).float())[1].double()  # amax / 127 in [2^(b-1), 2^b): steps of 2^(b-16)
        return torch.where(amax > 0, torch.ceil((amax / 127).float().double() * torch.exp2(16 - b)) * torch.exp2(b - 16), 0 * amax)
    e = torch.ceil(torch.log2(amax.clamp_min(2.0 ** -40) / 448))
    e = e - ((448 * torch.exp2(e - 1)) >= amax).double()  # where the logarithm was rounded up past a whole number
    e = e + ((448 * torch.exp2(e)) < amax).double()
    return torch.where(amax > 0, torch.exp2(e), 0 * amax)


def exact(case, seed):
    s = prepare(case, seed)
    c, code, H, D = s["cache"], case["code"], case["kv_heads"], case["head_dim"]
    if case["kind"] == "append":
        pos0, n, s0 = case["pos0"], case["n"], case["pos0"] % PAGE
        lo, m, out = pos0 - s0, s0 + n, {}
        for name, rows in zip("kv", s["rows"]):
            x = torch.cat([_decoded(c, name, code, pos0)[0][lo:], rows.double()])
            block = torch.arange(m, device=DEV) // PAGE
            amax = torch.zeros((int(block[-1]) + 1, H), dtype=torch.float64, device=DEV)
            amax.index_reduce_(0, block[s0:], x[s0:].abs().amax(-1), "amax")
            scale = _scale64(code, amax)
            if s0:
                scale[0] = torch.maximum(scale[0], c[name + "_scale"].double()[c["block_table"][lo // PAGE].long()])
            whole = c[name + "_scale"].double().clone()
            whole[c["block_table"][lo // PAGE:lo // PAGE + len(scale)].long()] = scale
            out[name], out[name + "_scale"] = _coded64(code, x, scale[block][..., None]), whole
        return out
    if case["kind"] == "evict":
        T, keep, sinks, recent = case["length"], case["keep"], case["sinks"], case["recent"]
        rank = s["mass"].double().clone()
        rank[:, :sinks] = math.inf
        rank[:, T - recent:] = math.inf
        order = torch.argsort(-rank, dim=1, stable=True)[:, :keep]  # the largest first, the lowest of equal ones first
        kept = torch.sort(order, 1)[0]
        out = {"kept": kept.int(), "mass": s["mass"].double().gather(1, kept)}
        block = torch.arange(keep, device=DEV) // PAGE
        for name in "kv":
            x, scale = _decoded(c, name, code, T)
            head = torch.arange(H, device=DEV)[:, None]
            x, scale = x[kept, head].transpose(0, 1), scale[kept, head].t()
            top = torch.zeros((_pages(keep), H), dtype=torch.float64, device=DEV).index_reduce_(0, block, scale, "amax")
            whole = torch.empty_like(top)
            whole[s["dst"]["block_table"].long()] = top
            out[name], out[name + "_scale"] = _coded64(code, x, top[block][..., None]), whole
        return out
    M, a, QH, n = case["tokens"], case["ctx"], case["q_heads"], case["ctx"] + case["tokens"]
    rows = case.get("rows", M)
    k, p = _decoded(c, "k", code, n)[0], torch.arange(n, device=DEV)
    v = _decoded(c, "v", code, n)[0] if case["kind"] == "attend" else None
    out, lse = torch.zeros((M, QH, D), dtype=torch.float64, device=DEV), torch.zeros((M, QH), dtype=torch.float64, device=DEV)
    mass = torch.zeros((H, n), dtype=torch.float64, device=DEV)
    for t in range(rows):
        low = max(case["start"], a + t - case["window"] + 1 if case["window"] else 0)
        see = ((p < a) & (p >= low)) | ((p >= a) & (p <= (a + t if case["causal"] else n)))
        for h in range(H):
            g = slice(h * (QH // H), (h + 1) * (QH // H))
            x = (s["q"][t, g].double() @ k[see, h].t()) / math.sqrt(D)
            if v is None:
                mass[h, see] += torch.exp(x - s["lse"][t, g].double()[:, None]).sum(0)
            else:
                lse[t, g] = torch.logsumexp(x, 1)
                out[t, g] = torch.exp(x - lse[t, g][:, None]) @ v[see, h]
    if v is None:
        mass = torch.where(p < a, s["mass"].double(), 0 * mass) + mass
        return {"mass": torch.where(p < a + rows, mass, 0 * mass)}
    if case["gate"]:
        out = out * torch.sigmoid(s["gate"].double())[..., None]
    return {"out": out, "lse": lse}
