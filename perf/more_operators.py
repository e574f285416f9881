"""What a server does to draw several answers to one prompt, as cases that can be timed and compared:

  rope    rotary positions of a batch's q and k rows, at any positions; with `append` the rotated K rows and V go into the
          fp16 pages of the batch's sequences
  shared  verify attention of sequences that share a long prefix, each with its own pages behind it, with its log-sum-exp
  sample  a token for every row of logits from given random numbers: temperature, top-k, top-p, min-p

Pages are the fp16 pages of dspark_kv_write (32 positions; K in matrix-core operand order, V transposed). Sizes are those of
the 16-layer configuration (32/8/64 heads, vocabulary 65536) and of the reference geometry (16/4/128, 128000), and others
around them.

With `own` false the operators are computed in their plain form; with `own` true by the framework.
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
        # one new token of each of eight sequences, deep in a long context, into the pages: a call of every layer and step
        {"name": "rope_token", "kind": "rope", "type": "f16", "n": 8, "q_heads": 32, "kv_heads": 8, "head_dim": 64, "rot": 64,
         "interleaved": False, "inverse": False, "scaling": "none", "far": 32768, "append": True},
        # a prompt chunk whose rows go into the pages, the reference geometry's half of the head, long-context scaling
        {"name": "rope_prompt", "kind": "rope", "type": "f16", "n": 8192, "q_heads": 16, "kv_heads": 4, "head_dim": 128, "rot": 64,
         "interleaved": False, "inverse": False, "scaling": "ramp", "far": 131072, "append": True},
        # a ragged batch of a model with interleaved pairs, bfloat16
        {"name": "rope_ragged", "kind": "rope", "type": "bf16", "n": 1537, "q_heads": 32, "kv_heads": 8, "head_dim": 64, "rot": 64,
         "interleaved": True, "inverse": False, "scaling": "linear", "far": 524288, "append": False},
        # the way back of a training step: the gradients of q and k turned back, in 32 bits
        {"name": "rope_back", "kind": "rope", "type": "f32", "n": 4099, "q_heads": 16, "kv_heads": 4, "head_dim": 128, "rot": 128,
         "interleaved": False, "inverse": True, "scaling": "none", "far": 8192, "append": False},
        # four answers to a short prompt, their first tokens
        {"name": "shared_short", "kind": "shared", "q_heads": 16, "kv_heads": 4, "head_dim": 128, "seqs": 4, "tokens": 1,
         "prefix": 1001, "own": 37, "window": 0, "causal": True, "gate": False},
        # plain decoding of 32 requests behind a long common document
        {"name": "shared_decode", "kind": "shared", "q_heads": 32, "kv_heads": 8, "head_dim": 64, "seqs": 32, "tokens": 1,
         "prefix": 32768, "own": 300, "window": 0, "causal": True, "gate": False},
        # drafted blocks of 16 requests, ragged, the reference geometry with its output gate
        {"name": "shared_verify", "kind": "shared", "q_heads": 16, "kv_heads": 4, "head_dim": 128, "seqs": 16, "tokens": 9,
         "prefix": 8190, "own": 1200, "window": 0, "causal": True, "gate": True},
        # the widest batch over the longest prefix
        {"name": "shared_wide", "kind": "shared", "q_heads": 32, "kv_heads": 8, "head_dim": 64, "seqs": 64, "tokens": 4,
         "prefix": 131072, "own": 700, "window": 0, "causal": True, "gate": False},
        # one request's next token
        {"name": "sample_token", "kind": "sample", "type": "f32", "n": 1, "vocab": 65536},
        # a verified block's rows, the reference's vocabulary
        {"name": "sample_block", "kind": "sample", "type": "f32", "n": 9, "vocab": 128000},
        # one token of each of 64 requests, every one with its own settings
        {"name": "sample_batch", "kind": "sample", "type": "f16", "n": 64, "vocab": 65536},
        # drafted blocks of many requests
        {"name": "sample_wide", "kind": "sample", "type": "f16", "n": 256, "vocab": 128000},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["rope", "shared", "shared", "sample"])
    if kind == "sample":
        return {"kind": kind, "type": rng.choice(["f32", "f16", "bf16"]), "n": _log(rng, 1, 200), "vocab": _log(rng, 1000, 131072)}
    q_heads, kv_heads, dim = rng.choice([(32, 8, 64), (16, 4, 128), (16, 2, 64), (8, 8, 128)])
    case = {"kind": kind, "q_heads": q_heads, "kv_heads": kv_heads, "head_dim": dim}
    if kind == "rope":
        append = rng.random() < 0.5
        return {**case, "type": "f16" if append else rng.choice(["f16", "bf16", "f32"]), "n": _log(rng, 1, 8000),
                "rot": rng.choice([dim, dim // 2, dim - 16]), "interleaved": rng.random() < 0.5,
                "inverse": not append and rng.random() < 0.4, "scaling": rng.choice(["none", "linear", "base", "ramp"]),
                "far": _log(rng, 8000, 600000), "append": append}
    seqs, tokens = _log(rng, 1, 64), rng.choice([1, 1, 4, 9, rng.randint(1, 16)])
    rows = seqs * tokens * (q_heads // kv_heads)
    prefix = _log(rng, 40, 131072 if rows <= 600 else 16384)
    return {**case, "seqs": seqs, "tokens": tokens, "prefix": prefix, "own": tokens + _log(rng, 1, 1500),
            "window": rng.choice([0, 0, 0, _log(rng, 64, 4096)]), "causal": rng.random() < 0.8, "gate": rng.random() < 0.5}


# ------------------------------------------------------------------------------------------------ inputs
TYPES = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}


def _gen(seed, name):
    g = torch.Generator(device=DEV)
    g.manual_seed((int(seed) << 32) ^ zlib.crc32(name.encode()))
    return g


def _randn(seed, name, shape, std=1.0, dtype=torch.float16):
    return torch.randn(shape, generator=_gen(seed, name), device=DEV).mul_(std).to(dtype)


def _rand(seed, name, shape, lo, hi):
    return torch.rand(shape, generator=_gen(seed, name), device=DEV).mul_(hi - lo).add_(lo)


def _randint(seed, name, shape, lo, hi):
    return torch.randint(lo, hi, shape, generator=_gen(seed, name), device=DEV)


def _pages(n):
    return (n + PAGE - 1) // PAGE


def _scaling(case):
    """The scaling of the frequencies: (kind, factor, trained length)."""
    return {"none": (None, 1.0, 0), "linear": ("linear", 4.0, 0), "base": ("base", 8.0, 0), "ramp": ("ramp", 16.0, 8192)}[case["scaling"]]


def _lengths(case):
    """Tokens of each sequence in this call and keys in its own pages (this call's among them): ragged, the first the fullest."""
    m = [case["tokens"] - (5 * r) % case["tokens"] for r in range(case["seqs"])]
    return m, [max(x, case["own"] - (7919 * r) % max(1, case["own"] * 3 // 4)) for r, x in enumerate(m)]


def _prepare_rope(s):
    case, seed = s, s["seed"]
    n, H, KH, D = case["n"], case["q_heads"], case["kv_heads"], case["head_dim"]
    # q, k and v lie side by side in a row, as a projection writes them
    row = _randn(seed, "rows", (n, H + 2 * KH, D), dtype=TYPES[case["type"]])
    s["q"], s["k"], s["v"] = row[:, :H], row[:, H:H + KH], row[:, H + KH:]
    at = _randint(seed, "first", (1,), 0, case["far"] - n + 1) + torch.arange(n, device=DEV) if n > 64 \
        else _randint(seed, "at", (n,), case["far"] // 2, case["far"])
    s["positions"] = at.int()
    kind, factor, trained = _scaling(case)
    base, rot = 1e6 if case["far"] > 100000 else 1e4, case["rot"]
    f = torch.tensor([base ** (-2 * i / rot) for i in range(rot // 2)], dtype=torch.float64, device=DEV)
    s["scale"] = 1.0
    if kind == "linear":
        f = f / factor
    elif kind == "base":  # the base raised so that the slowest pair turns 1 / factor as fast
        f = torch.tensor([(base * factor ** (rot / (rot - 2))) ** (-2 * i / rot) for i in range(rot // 2)], dtype=torch.float64, device=DEV)
    elif kind == "ramp":  # pairs of under one turn in the trained length slowed down, of over 32 left, a ramp between
        keep = ((trained * f / (2 * math.pi) - 1.0) / 31.0).clamp(0, 1)
        f, s["scale"] = f * keep + f / factor * (1 - keep), 0.1 * math.log(factor) + 1
    s["freqs"] = f
    if case["append"]:
        # each row's slot: the sequences' last pages anywhere in the pool (a few rows), or a run of pages (a prompt)
        P = n if n <= 64 else _pages(n) + 1
        table = torch.randperm(P, generator=_gen(seed, "table"), device=DEV)
        local = torch.arange(n, device=DEV) * PAGE + _randint(seed, "slot", (n,), 0, PAGE) if n <= 64 else torch.arange(n, device=DEV) + 7
        s["slots"] = table[local // PAGE] * PAGE + local % PAGE
        s["k_pages"] = _randn(seed, "k_pages", (P, KH, PAGE, D))
        s["v_pages"] = _randn(seed, "v_pages", (P, KH, D, PAGE))


def _prepare_shared(s):
    case, seed = s, s["seed"]
    H, KH, D, R = case["q_heads"], case["kv_heads"], case["head_dim"], case["seqs"]
    m, own_len = _lengths(case)
    T, cols = sum(m), _pages(max(own_len))
    P = _pages(case["prefix"]) + R * cols
    s["q"] = _randn(seed, "q", (T, H, D), 1.5)
    s["k_pages"] = _randn(seed, "k", (P, KH, PAGE, D))
    s["v_pages"] = _randn(seed, "v", (P, KH, D, PAGE))
    table = torch.randperm(P, generator=_gen(seed, "table"), device=DEV).int()  # logical pages anywhere in the pool
    s["prefix_table"] = table[:_pages(case["prefix"])].contiguous()
    s["own_table"] = table[_pages(case["prefix"]):].view(R, cols).contiguous()
    s["q_start"] = torch.tensor([sum(m[:r]) for r in range(R + 1)], dtype=torch.int32, device=DEV)
    s["own_len"] = torch.tensor(own_len, dtype=torch.int32, device=DEV)
    s["gates"] = _randn(seed, "gate", (T, H), dtype=torch.float32) if case["gate"] else None


def _prepare_sample(s):
    n, V, seed = s["n"], s["vocab"], s["seed"]
    # most tokens far below a few likely ones, and rows more or less certain
    z = torch.randn((n, V), generator=_gen(seed, "z"), device=DEV).mul_(_rand(seed, "std", (n, 1), 1.5, 3.0))
    likely = _randint(seed, "likely", (n, 40), 0, V)
    z.scatter_add_(1, likely, _rand(seed, "boost", (n, 40), 2.0, 12.0))
    row = torch.arange(n, device=DEV)
    # a grammar's mask on some rows
    masked = (torch.rand((n, V), generator=_gen(seed, "mask"), device=DEV) < 0.3) & (row % 4 == 3)[:, None]
    s["logits"] = z.masked_fill_(masked, -math.inf).to(TYPES[s["type"]])
    s["u"] = torch.rand((n,), generator=_gen(seed, "u"), device=DEV)
    # settings as requests bring them: greedy ones, plain ones, and each kind of cut
    t = _rand(seed, "t", (n,), 0.5, 1.3)
    s["temperature"] = torch.where(row % 8 == 6, torch.zeros_like(t), t)
    k = _randint(seed, "k", (n,), 1, 200).int()
    s["top_k"] = torch.where(row % 3 == 1, k, torch.zeros_like(k))
    p = _rand(seed, "p", (n,), 0.7, 0.99)
    s["top_p"] = torch.where(row % 5 != 4, p, torch.ones_like(p))
    low = _rand(seed, "low", (n,), 0.01, 0.2)
    s["min_p"] = torch.where(row % 4 == 2, low, torch.zeros_like(low))


def prepare(case, seed):
    s = {**case, "seed": seed}
    {"rope": _prepare_rope, "shared": _prepare_shared, "sample": _prepare_sample}[case["kind"]](s)
    if own:  # the handles and buffers that a serving loop keeps
        s["host"] = _host()
        s["workspace"] = s["host"].Workspace(DEV)
        if case["kind"] == "rope":  # the frequencies as the framework gives them
            kind, factor, trained = _scaling(case)
            f, s["scale"] = s["host"].rope_freqs(case["rot"], 1e6 if case["far"] > 100000 else 1e4, kind, factor, trained)
            s["freqs"] = torch.from_numpy(f).to(DEV)
    return s


# ------------------------------------------------------------------------------------------------ the plain forms
def _k_index(D):
    """Where K[slot][d] of a (page, head) block lies among its 32 D halves."""
    slot, d = torch.arange(PAGE, device=DEV)[:, None], torch.arange(D, device=DEV)[None, :]
    block, row = (slot >> 2) & 1, 4 * (slot >> 3) + (slot & 3)
    return ((block * (D // 32) + d // 32) * 64 + row + 16 * ((d % 32) // 8)) * 8 + d % 8


def _turned(x, s):
    """x [n][heads][D] with the first `rot` values of each head turned, in 32 bits, angles in 64."""
    rot, P = s["rot"], s["rot"] // 2
    a = s["positions"].double()[:, None] * s["freqs"]
    cos, sin = (a.cos() * s["scale"]).float()[:, None], (a.sin() * s["scale"]).float()[:, None]
    if s["inverse"]:
        sin = -sin
    y = x.float().clone()
    if s["interleaved"]:
        i, j = y[..., 0:rot:2].clone(), y[..., 1:rot:2].clone()
        y[..., 0:rot:2], y[..., 1:rot:2] = i * cos - j * sin, j * cos + i * sin
    else:
        i, j = y[..., :P].clone(), y[..., P:rot].clone()
        y[..., :P], y[..., P:rot] = i * cos - j * sin, j * cos + i * sin
    return y.to(x.dtype)


def _rope(s):
    q, k = _turned(s["q"], s), _turned(s["k"], s)
    if not s["append"]:
        return {"q": q, "k": k}
    D, page, slot = s["head_dim"], s["slots"] // PAGE, s["slots"] % PAGE
    kp, vp = s["k_pages"], s["v_pages"]
    head = torch.arange(s["kv_heads"], device=DEV)[None, :, None]
    kp.view(kp.shape[0], kp.shape[1], PAGE * D)[page[:, None, None], head, _k_index(D)[slot][:, None, :]] = k
    vp[page[:, None, None], head, torch.arange(D, device=DEV), slot[:, None, None]] = s["v"]
    return {"q": q, "k_pages": kp, "v_pages": vp}


def _rows_of(s, pages):
    """K and V of pages (a tensor of indexes) in 32 bits, [KV head][positions][D]."""
    KH, D = s["kv_heads"], s["head_dim"]
    k = s["k_pages"][pages].view(-1, KH, PAGE * D)[:, :, _k_index(D)].float()
    v = s["v_pages"][pages].float().transpose(2, 3)
    return [x.transpose(0, 1).reshape(KH, -1, D) for x in (k, v)]


def _shared(s):
    H, KH, D, R, prefix = s["q_heads"], s["kv_heads"], s["head_dim"], s["seqs"], s["prefix"]
    G, T = H // KH, s["q"].shape[0]
    start, lens = s["q_start"].long(), s["own_len"].long()
    seq = torch.searchsorted(start[1:], torch.arange(T, device=DEV), right=True)
    pos = lens[seq] - (start[seq + 1] - torch.arange(T, device=DEV))  # of each token among its own keys
    q = s["q"].float().view(T, KH, G, D).permute(1, 0, 2, 3)  # [KV head][token][group][D]
    k, v = _rows_of(s, s["prefix_table"].long())
    x = torch.matmul(q.reshape(KH, T * G, D), k.transpose(1, 2)).div_(math.sqrt(D)).view(KH, T, G, -1)
    p = torch.arange(x.shape[-1], device=DEV)
    see = (p < prefix).expand(T, -1)
    if s["window"]:
        see = see & (p > (prefix + pos - s["window"])[:, None])
    x.masked_fill_(~see[:, None], -math.inf)
    # every sequence's own keys, tokens side by side in rows of the widest sequence
    M, cols = s["tokens"], s["own_table"].shape[1]
    ko, vo = [t.view(KH, R, cols * PAGE, D) for t in _rows_of(s, s["own_table"].long().reshape(-1))]
    i = torch.arange(T, device=DEV) - start[seq]
    qs = torch.zeros((KH, R, M, G, D), device=DEV)
    qs[:, seq, i] = q
    xo = torch.matmul(qs.view(KH, R, M * G, D), ko.transpose(2, 3)).div_(math.sqrt(D)).view(KH, R, M, G, -1)[:, seq, i]
    j = torch.arange(cols * PAGE, device=DEV)
    see = j < lens[seq][:, None]
    if s["causal"]:
        see = see & (j <= pos[:, None])
    if s["window"]:
        # (as in the framework's other attention, the window bounds the keys before the call's tokens)
        see = see & ((j > (pos - s["window"])[:, None]) | (j >= (lens - (start[1:] - start[:-1]))[seq][:, None]))
    xo.masked_fill_(~see[:, None], -math.inf)
    m = torch.maximum(x.amax(-1, keepdim=True), xo.amax(-1, keepdim=True))
    x.sub_(m).exp_()
    xo = xo.sub(m).exp()
    total = x.sum(-1, keepdim=True) + xo.sum(-1, keepdim=True)
    o = torch.matmul(x.view(KH, T * G, -1), v).view(KH, T, G, D)
    ps = torch.zeros((KH, R, M, G, cols * PAGE), device=DEV)
    ps[:, seq, i] = xo
    o = (o + torch.matmul(ps.view(KH, R, M * G, -1), vo).view(KH, R, M, G, D)[:, seq, i]) / total
    o = o.permute(1, 0, 2, 3).reshape(T, H, D)
    if s["gates"] is not None:
        o = o * (1 / (1 + torch.exp(-s["gates"])))[..., None]
    return {"out": o.half(), "lse": (total.log() + m)[..., 0].permute(1, 0, 2).reshape(T, H)}


def _sample(s):
    # in 64 bits: a draw next to a border, a nucleus that ends at one
    z, V = s["logits"].double(), s["vocab"]
    top = z.amax(1, keepdim=True)
    t = s["temperature"].double()[:, None]
    greedy = t <= 0
    w = ((z - top) / torch.where(greedy, torch.ones_like(t), t)).exp_()
    zs, order = torch.sort(z, dim=1, descending=True, stable=True)
    ws = w.gather(1, order)
    rank = torch.arange(V, device=DEV)
    k = s["top_k"].long()[:, None]
    keep = (rank < torch.where(greedy, torch.ones_like(k), torch.where(k > 0, k, V + 0 * k))) & (zs > -math.inf)
    ws = ws * keep
    p = s["top_p"].double()[:, None]
    before = ws.cumsum(1) - ws
    keep = keep & ((p >= 1) | (before < p * ws.sum(1, keepdim=True)) | (rank == 0))
    keep = keep & ((zs - top) / torch.where(greedy, torch.ones_like(t), t) >= s["min_p"].double().log()[:, None])
    kept = torch.zeros_like(keep).scatter_(1, order, keep)
    w = torch.where(kept, w, torch.zeros_like(w))
    sums = w.cumsum(1)
    token = torch.searchsorted(sums, s["u"].double()[:, None] * sums[:, -1:], right=True).clamp_(max=V - 1)
    lp = (w.gather(1, token) / sums[:, -1:]).log()
    return {"token": token[:, 0].int(), "kept": kept.sum(1).int(), "logprob": lp[:, 0].float()}


# ------------------------------------------------------------------------------------------------ the framework's calls
def _own(s):
    h = s["host"]
    if s["kind"] == "rope":
        how = {"interleaved": s["interleaved"], "scale": s["scale"]}
        if s["append"]:
            q = h.rope_append(s["q"], s["k"], s["v"], s["positions"], s["freqs"], s["k_pages"], s["v_pages"], s["slots"], **how)
            return {"q": q, "k_pages": s["k_pages"], "v_pages": s["v_pages"]}
        q, k = h.rope(s["q"], s["k"], s["positions"], s["freqs"], inverse=s["inverse"], **how)
        return {"q": q, "k": k}
    if s["kind"] == "shared":
        lse = torch.empty(s["q"].shape[:2], device=DEV)
        out, _ = h.verify_attention_shared(s["q"], s["k_pages"], s["v_pages"], s["prefix"], s["q_start"], s["own_len"], s["own_table"],
                                           max_tokens=s["tokens"], prefix_table=s["prefix_table"], window=s["window"],
                                           causal=s["causal"], gate=s["gates"], lse=lse, workspace=s["workspace"])
        return {"out": out, "lse": lse}
    got = h.verify_sample(s["logits"], s["u"], temperature=s["temperature"], top_k=s["top_k"], top_p=s["top_p"], min_p=s["min_p"],
                          kept=True, logprob=True, workspace=s["workspace"])
    return {"token": got.tokens, "kept": got.kept, "logprob": got.logprob}


def run(state):
    if own:
        return _own(state)
    return {"rope": _rope, "shared": _shared, "sample": _sample}[state["kind"]](state)


# ------------------------------------------------------------------------------------------------ work and exact values
def work(case):
    if case["kind"] == "sample":
        n, V = case["n"], case["vocab"]
        return {"bytes": n * (V * (4 if case["type"] == "f32" else 2) + 32), "flops": 4 * n * V}
    H, KH, D = case["q_heads"], case["kv_heads"], case["head_dim"]
    if case["kind"] == "rope":
        n, size = case["n"], 4 if case["type"] == "f32" else 2
        rows = 2 * (H + KH) + (2 * KH if case["append"] else 0)
        return {"bytes": n * (rows * D * size + (12 if case["append"] else 4)), "flops": 3 * n * (H + KH) * case["rot"]}
    m, lens = _lengths(case)
    T, w, prefix = sum(m), case["window"], case["prefix"]
    seen = lambda x, n: min(prefix + n, w + x - 1) if w else prefix + n  # noqa: E731 (keys that a sequence's tokens see)
    shared = min(prefix, max(max(0, seen(x, n) - n) for x, n in zip(m, lens)))
    keys = shared + sum(min(n, seen(x, n)) for x, n in zip(m, lens))
    return {"bytes": 4 * D * KH * keys + T * H * (4 * D + 4 + (4 if case["gate"] else 0)),
            "flops": 4 * D * H * sum(x * seen(x, n) for x, n in zip(m, lens))}


def _exact_rope(s):
    rot, out = s["rot"], {}
    # the frequencies anew: exp(-(2 i / rot) ln base), scaled as the case says
    i = torch.arange(0, rot, 2, device=DEV, dtype=torch.float64) / rot
    base, (kind, factor, trained) = math.log(1e6 if s["far"] > 100000 else 1e4), _scaling(s)
    size = 1.0
    if kind == "base":
        base += math.log(factor) * rot / (rot - 2)
    f = torch.exp(-i * base)
    if kind == "linear":
        f = f / factor
    elif kind == "ramp":
        turns = trained * f / (2 * math.pi)
        share = torch.where(turns <= 1, 0 * f, torch.where(turns >= 32, 0 * f + 1, (turns - 1) / 31))
        f, size = f * (share + (1 - share) / factor), 1 + math.log(factor) / 10
    e = torch.polar(torch.full_like(f, size).expand(s["n"], -1), s["positions"].double()[:, None] * f * (-1 if s["inverse"] else 1))[:, None]
    for name in "qk":
        x = s[name].double()
        head, rest = x[..., :rot], x[..., rot:]
        pair = head.unflatten(-1, (rot // 2, 2)) if s["interleaved"] else head.unflatten(-1, (2, rot // 2)).transpose(-1, -2)
        y = torch.view_as_real(torch.view_as_complex(pair.contiguous()) * e)
        y = y.flatten(-2) if s["interleaved"] else y.transpose(-1, -2).flatten(-2)
        out[name] = torch.cat([y, rest], -1)
    if not s["append"]:
        return out
    kp, vp, D, KH = s["k_pages"].double(), s["v_pages"].double(), s["head_dim"], s["kv_heads"]
    flat_k, flat_v = kp.view(-1), vp.view(-1)
    block = (s["slots"] // PAGE)[:, None] * KH + torch.arange(KH, device=DEV)  # (page, head) of each row and head
    slot, d = (s["slots"] % PAGE)[:, None, None], torch.arange(D, device=DEV)
    # the operand order: key block, k-step, quarter of the step, row, value
    at = slot // 4 % 2 * (16 * D) + d // 32 * 512 + d % 32 // 8 * 128 + (slot // 8 * 4 + slot % 4) * 8 + d % 8
    flat_k[block[..., None] * (PAGE * D) + at] = out["k"]
    flat_v[block[..., None] * (PAGE * D) + d * PAGE + slot] = s["v"].double()
    return {"q": out["q"], "k_pages": kp, "v_pages": vp}


def _exact_shared(s):
    H, KH, D, prefix, w = s["q_heads"], s["kv_heads"], s["head_dim"], s["prefix"], s["window"]
    G, (m, lens) = H // KH, _lengths(s)
    slot, d = torch.arange(PAGE, device=DEV)[:, None], torch.arange(D, device=DEV)
    at = slot // 4 % 2 * (16 * D) + d // 32 * 512 + d % 32 // 8 * 128 + (slot // 8 * 4 + slot % 4) * 8 + d % 8

    def rows(table, n, h):
        pages = table.long()[:_pages(n)]
        k = s["k_pages"][pages, h].reshape(len(pages), -1)[:, at.reshape(-1)].reshape(-1, D)
        return k[:n].double(), s["v_pages"][pages, h].transpose(1, 2).reshape(-1, D)[:n].double()

    out = torch.zeros((sum(m), H, D), dtype=torch.float64, device=DEV)
    lse = torch.zeros((sum(m), H), dtype=torch.float64, device=DEV)
    for h in range(KH):
        pk, pv = rows(s["prefix_table"], prefix, h)
        g, t0 = slice(h * G, (h + 1) * G), 0
        for r, (x, n) in enumerate(zip(m, lens)):
            k, v = rows(s["own_table"][r], n, h)
            k, v = torch.cat([pk, k]), torch.cat([pv, v])
            a = prefix + n - x  # the first token's position
            p, t = torch.arange(prefix + n, device=DEV), torch.arange(a, a + x, device=DEV)[:, None]
            see = (p <= t) if s["causal"] else (p >= 0).expand(x, -1)
            if w:
                see = see & ((p >= a) | (p > t - w))
            sc = (s["q"][t0:t0 + x, g].double() @ k.t()) / math.sqrt(D)
            sc = torch.where(see[:, None], sc, torch.full_like(sc, -math.inf))
            lse[t0:t0 + x, g] = torch.logsumexp(sc, -1)
            out[t0:t0 + x, g] = torch.softmax(sc, -1) @ v
            t0 += x
    if s["gates"] is not None:
        out = out * torch.sigmoid(s["gates"].double())[..., None]
    return {"out": out, "lse": lse}


def _exact_sample(s):
    """Row by row: the kept set by sorted values, the draw by the cumulative distribution of what is left."""
    token, kept, logprob = [], [], []
    rows = zip(s["logits"].double(), s["u"].tolist(), s["temperature"].tolist(), s["top_k"].tolist(), s["top_p"].tolist(), s["min_p"].tolist())
    for z, u, t, k, p, low in rows:
        if t <= 0:
            token.append(torch.argmax(z))
            kept.append(torch.ones_like(token[-1]))
            logprob.append(torch.zeros((), dtype=torch.float64, device=DEV))
            continue
        live = torch.nonzero(z > -math.inf)[:, 0]
        x = torch.log_softmax(z[live] / t, 0)
        order = torch.argsort(-x, stable=True)
        x, ids = x[order], live[order]
        if k > 0:
            x, ids = x[:k], ids[:k]
            x = x - torch.logsumexp(x, 0)
        stay = torch.ones_like(ids, dtype=torch.bool)
        if p < 1:  # those with less than p in front of them
            stay[1:] = torch.cumsum(x.exp(), 0)[:-1] < p
        if low > 0:
            stay &= x - x[0] >= math.log(low)
        x, ids = x[stay], ids[stay]
        ids, by = torch.sort(ids)
        x = x[by] - torch.logsumexp(x, 0)
        at = (torch.cumsum(x.exp(), 0) > u).int().argmax()
        token.append(ids[at])
        kept.append(torch.full_like(ids[0], len(ids)))
        logprob.append(x[at])
    return {"token": torch.stack(token).int(), "kept": torch.stack(kept).int(), "logprob": torch.stack(logprob)}


def exact(case, seed):
    s = prepare(case, seed)
    return {"rope": _exact_rope, "shared": _exact_shared, "sample": _exact_sample}[case["kind"]](s)
