"""The operators for a batch of sequences on the GPU against their restatement in float64 (oracle/batch.py): rotary positions with K/V
by slot, attention behind a shared prefix, sampling -- and all of them in turn, as a server's step has them."""
import math

import numpy as np
import pytest
import torch

from conftest import load_host
from oracle import batch

pytestmark = pytest.mark.gpu
TYPES = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}
HALF = {"f16": 2.0 ** -11, "bf16": 2.0 ** -8, "f32": 2.0 ** -24}  # half a step, relative
TINY = {"f16": 2.0 ** -25, "bf16": 2.0 ** -134, "f32": 2.0 ** -150}  # half a step among the subnormals


def dev(x):
    return torch.from_numpy(np.ascontiguousarray(x)).to("cuda")


def f64(t):
    return t.double().cpu().numpy()


# ------------------------------------------------------------------------------------------------ rotary positions
def rope_close(got, x, want, kind, scale, rot):
    """The type's rounding once; before it two fp32 products and a sum of the pair's values with sines and cosines each half a step off
    (and a fused product instead of a rounded one only brings it nearer): under 4 x 2^-24 scale (|x_i| + |x_j|), and that pair sum
    is at most 2 max |x| of the head."""
    top = np.abs(x).max(-1, keepdims=True)
    err = np.abs(f64(got) - want)
    turned = np.arange(x.shape[-1]) < rot
    bound = np.where(turned, np.abs(want) * HALF[kind] * 1.001 + TINY[kind] + 8 * 2.0 ** -24 * abs(scale) * top, 0)
    assert np.all(err <= bound), float(np.max(err - bound))


@pytest.mark.parametrize("kind", sorted(TYPES))
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("n,QH,KVH,D,rot", [(1, 32, 8, 64, 64), (1, 1, 0, 2, 2), (5, 16, 4, 128, 64), (37, 3, 1, 64, 48), (4, 2, 2, 10, 6),
                                             (130, 5, 5, 72, 8), (9, 0, 4, 256, 250), (3, 1, 1, 1024, 1024), (1500, 4, 2, 64, 32)])
def test_rope(kind, interleaved, n, QH, KVH, D, rot):
    h, rng = load_host(), np.random.default_rng(n * 1000 + D + rot)
    f, s = h.rope_freqs(rot, 1e6, "ramp", 8.0, 4096)
    pos = rng.integers(-(1 << 20), 1 << 20, n).astype(np.int32)
    pos[:2] = [0, (1 << 31) - 1][:min(n, 2)]
    q, k = [None if not heads else dev(rng.standard_normal((n, heads, D))).to(TYPES[kind]) for heads in (QH, KVH)]
    for inverse in (False, True):
        got = h.rope(q, k, dev(pos), dev(f), interleaved=interleaved, inverse=inverse, scale=s)
        for x, y in zip((q, k), got):
            assert (x is None) == (y is None)
            if x is not None:
                rope_close(y, f64(x), batch.rope(f64(x), pos, f, interleaved, inverse, s), kind, s, rot)


@pytest.mark.parametrize("kind", ["f16", "f32"])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("off,stride", [(0, 0), (8, 8), (1, 3)])
def test_rope_rows_in_wider_ones(kind, interleaved, off, stride):
    """q, k and what lies behind them in one row, turned in place and into another such tensor; the rest of both is left as it was."""
    h, rng = load_host(), np.random.default_rng(7)
    n, QH, KVH, D, rot = 33, 4, 2, 64, 32
    width = off + (QH + 2 * KVH) * D + stride
    base = dev(rng.standard_normal((n, width))).to(TYPES[kind])
    f, pos = batch.rope_freqs(rot, 1e4)[0], rng.integers(0, 9000, n).astype(np.int32)

    def parts(t):
        return t.as_strided((n, QH, D), (width, D, 1), off), t.as_strided((n, KVH, D), (width, D, 1), off + QH * D)

    q, k = parts(base)
    want = [batch.rope(f64(x), pos, f, interleaved) for x in (q, k)]
    first = [f64(x) for x in (q, k)]
    other = torch.full((n, width), 5.0, dtype=TYPES[kind], device="cuda")
    oq, ok = parts(other)
    h.rope(q, k, dev(pos), dev(f), interleaved=interleaved, q_out=oq, k_out=ok)
    rest = other.clone()
    for t in parts(rest):
        t.fill_(5.0)
    assert torch.equal(rest, torch.full_like(rest, 5.0))
    before = base.clone()
    h.rope(q, k, dev(pos), dev(f), interleaved=interleaved, q_out=q, k_out=k)
    for x, y, w in zip(first, (q, k), want):
        rope_close(y, x, w, kind, 1.0, rot)
    assert torch.equal(q, oq) and torch.equal(k, ok)
    for t, u in zip(parts(before), parts(base)):
        t.copy_(u)
    assert torch.equal(before, base)


@pytest.mark.parametrize("QH,KVH", [(128, 8), (100, 7), (1024, 1024)])
def test_rope_more_units_of_a_token_than_a_division_holds(QH, KVH):
    """Heads of 1022 values, turned value by value: 109247 units of a token and more."""
    h, rng, n, D = load_host(), np.random.default_rng(QH), 3, 1022
    q, k = (dev(rng.standard_normal((n, heads, D)).astype(np.float16)) for heads in (QH, KVH))
    f, pos = batch.rope_freqs(2, 1e4)[0], np.array([5, 70000, 3], np.int32)
    spare = torch.full((n + 2, QH, D), 7.0, dtype=torch.float16, device="cuda")
    oq, ok = h.rope(q, k, dev(pos), dev(f), q_out=spare[1:1 + n])
    for y, x in ((oq, q), (ok, k)):
        rope_close(y, f64(x), batch.rope(f64(x), pos, f), "f16", 1.0, 2)
    assert bool((spare[0] == 7).all()) and bool((spare[-1] == 7).all())


def test_rope_not_finite_and_nothing():
    h = load_host()
    f = dev(batch.rope_freqs(8, 1e4)[0])
    x = torch.ones((3, 2, 16), dtype=torch.float16, device="cuda")
    x[1, 0, 2] = math.nan
    x[1, 1, 15] = math.inf
    y, _ = h.rope(x, None, torch.arange(3, dtype=torch.int32, device="cuda"), f)
    bad = ~torch.isfinite(y)
    want = torch.zeros_like(bad)
    want[1, 0, 2] = want[1, 0, 6] = want[1, 1, 15] = True  # the pair of the NaN, and the infinity passed on
    assert torch.equal(bad, want)
    q, k = h.rope(x[:0], x[:0, :1], torch.zeros(0, dtype=torch.int32, device="cuda"), f)
    assert q.shape == (0, 2, 16) and k.shape == (0, 1, 16)


def test_rope_strides_of_what_is_not_there():
    """q alone, k alone and the pages: the strides of the rest may hold anything."""
    h, n, D, any_ = load_host(), 3, 64, 1 << 40
    x, pos, f = torch.randn((n, 2, D), device="cuda").half(), torch.arange(n, dtype=torch.int32, device="cuda"), dev(batch.rope_freqs(D, 1e4)[0])
    want, _ = h.rope(x, None, pos, f)
    common = dict(positions=pos.data_ptr(), freq=f.data_ptr(), scale=1.0, n=n, D=D, rot=D)
    stream = torch.cuda.current_stream().cuda_stream
    for t, other in (("q", "k"), ("k", "q")):
        y = torch.zeros_like(x)
        heads = {"QH" if t == "q" else "KVH": 2}
        a = h.RopeArgs(**{t: x.data_ptr(), t + "_out": y.data_ptr(), t + "_stride": 128, t + "_out_stride": 128, other + "_stride": any_,
                          other + "_out_stride": any_}, v_stride=any_, **heads, **common)
        assert h.lib().dspark_rope(a, stream) == 0
        assert torch.equal(y, want)
    kp, vp = h.kv_pages_alloc(1, 2, D)
    slots = torch.arange(n, device="cuda")
    a = h.RopeArgs(k=x.data_ptr(), k_stride=128, k_out_stride=any_, q_stride=any_, q_out_stride=any_, v=x.data_ptr(), v_stride=128, KVH=2,
                   k_pages=kp.data_ptr(), v_pages=vp.data_ptr(), slots=slots.data_ptr(), kv_pages=1, **common)
    assert h.lib().dspark_rope(a, stream) == 0
    k1, v1 = h.kv_from_pages(kp, vp, range(n))
    np.testing.assert_array_equal(k1, want.cpu().numpy())
    np.testing.assert_array_equal(v1, x.cpu().numpy())


@pytest.mark.parametrize("interleaved", [False, True])
def test_rope_gradient(interleaved):
    """The inverse is the backward pass: <rope(x), g> = <x, inverse(g)>, by the formula's autograd and by differences (rope is linear, so a
    difference is exact but for fp32's rounding)."""
    h, rng = load_host(), np.random.default_rng(3)
    n, H, D, rot, s = 6, 2, 24, 16, 1.25
    pos, f = dev(rng.integers(0, 100000, n).astype(np.int32)), batch.rope_freqs(rot, 1e4)[0]
    x, g = [dev(rng.standard_normal((n, H, D)).astype(np.float32)) for _ in range(2)]
    dx, _ = h.rope(g, None, pos, dev(f), interleaved=interleaved, inverse=True, scale=s)
    xt = x.double().cpu().requires_grad_()
    a = pos.cpu().double()[:, None] * torch.from_numpy(f)
    i, j = (slice(0, rot, 2), slice(1, rot, 2)) if interleaved else (slice(0, rot // 2), slice(rot // 2, rot))
    c, sn = a.cos()[:, None], a.sin()[:, None]
    y = torch.cat([xt[..., i] * c - xt[..., j] * sn, xt[..., j] * c + xt[..., i] * sn], -1) * s
    gi = torch.cat([g.double().cpu()[..., i], g.double().cpu()[..., j]], -1)
    ((y * gi).sum() + (xt[..., rot:] * g.double().cpu()[..., rot:]).sum()).backward()
    np.testing.assert_allclose(f64(dx), xt.grad.numpy(), atol=8 * 2.0 ** -24 * s * 5)
    y0, _ = h.rope(x, None, pos, dev(f), interleaved=interleaved, scale=s)
    for t, hd, d in ((0, 0, 0), (2, 1, 9), (5, 0, 15), (3, 1, 20)):
        xp = x.clone()
        xp[t, hd, d] += 1.0
        yp, _ = h.rope(xp, None, pos, dev(f), interleaved=interleaved, scale=s)
        diff = float(((yp.double() - y0.double()) * g.double()).sum())
        # two values of up to 1.25 x 7 each rounded to 2^-24 of it, twice, times |g| < 5
        assert abs(diff - float(dx[t, hd, d])) < 4 * 2.0 ** -23 * 9 * 5


@pytest.mark.parametrize("D,KVH", [(64, 8), (128, 4), (64, 1)])
@pytest.mark.parametrize("rot,interleaved,n,off", [(64, False, 1, 0), (32, True, 40, 0), (16, False, 77, 8), (10, False, 5, 0), (64, True, 70, 1),
                                                   (64, False, 4500, 0)])
def test_rope_append(D, KVH, rot, interleaved, n, off):
    """Pages against dspark_kv_write of the turned rows; slots anywhere, some outside the pools; every other slot as it was."""
    h, rng = load_host(), np.random.default_rng(D + n)
    QH, P = 2 * KVH, n // 32 + 9
    width = off + (QH + 2 * KVH) * D
    width += -width % 8 if off % 8 == 0 else 0
    base = dev(rng.standard_normal((n, width)).astype(np.float16))
    q, k, v = (base.as_strided((n, heads, D), (width, D, 1), off + at * D) for heads, at in ((QH, 0), (KVH, QH), (KVH, QH + KVH)))
    f, pos = batch.rope_freqs(rot, 1e4)[0], rng.integers(0, 70000, n).astype(np.int32)
    slots = rng.permutation(32 * P)[:n].astype(np.int64)
    if n > 4:
        slots[1], slots[3], slots[4] = -1, 32 * P, -(1 << 40)
    kp, vp = (dev(rng.standard_normal((P, KVH, 32 * D)).astype(np.float16)) for _ in range(2))
    kp, vp = kp.view(P, KVH, 32, D), vp.view(P, KVH, D, 32)
    k0, v0 = h.kv_from_pages(kp, vp, range(32 * P))
    want_q, want_k = h.rope(q, k, dev(pos), dev(f), interleaved=interleaved, scale=1.5)
    got = h.rope_append(q, k, v, dev(pos), dev(f), kp, vp, dev(slots), interleaved=interleaved, scale=1.5)
    assert torch.equal(got, want_q)
    there = (slots >= 0) & (slots < 32 * P)
    k0[slots[there]], v0[slots[there]] = want_k.cpu().numpy()[there], v.cpu().numpy()[there]
    k1, v1 = h.kv_from_pages(kp, vp, range(32 * P))
    np.testing.assert_array_equal(k1, k0)
    np.testing.assert_array_equal(v1, v0)


def test_rope_append_past_4_gib():
    h, KVH, D, n = load_host(), 8, 128, 6
    P = (9 << 29) // (KVH * 32 * D * 2)  # 4.5 GiB each
    kp = torch.zeros((P, KVH, 32, D), dtype=torch.float16, device="cuda")
    vp = torch.zeros((P, KVH, D, 32), dtype=torch.float16, device="cuda")
    q, k, v = (torch.randn((n, heads, D), device="cuda").half() for heads in (8, KVH, KVH))
    f, pos = dev(batch.rope_freqs(128, 1e4)[0]), torch.arange(n, dtype=torch.int32, device="cuda")
    slots = torch.tensor([32 * P - 1, 32 * P - 32, 0, 32 * (P - 1) + 5, 32 * P, 32 * (P // 2)], device="cuda")
    h.rope_append(q, k, v, pos, f, kp, vp, slots)
    _, want = h.rope(q, k, pos, f)
    k1, v1 = h.kv_from_pages(kp[-1:].contiguous(), vp[-1:].contiguous(), [31, 0, 5])
    for i, t in enumerate((0, 1, 3)):
        np.testing.assert_array_equal(k1[i], want[t].cpu().numpy())
        np.testing.assert_array_equal(v1[i], v[t].cpu().numpy())
    assert int((kp[:P - 1].view(torch.int16).count_nonzero(dim=(1, 2, 3)) > 0).sum()) == 2


# ------------------------------------------------------------------------------------------------ attention behind a shared prefix
class Batch:
    """Sequences with random rows in permuted pages; every slot that holds no key is filled with NaN."""

    def __init__(self, seed, QH, KVH, D, prefix, m, lens, absent=0.0, spare=0, before=0, behind=0, size=1.0):
        h, rng = load_host(), np.random.default_rng(seed)
        self.h, self.QH, self.KVH, self.D, self.prefix, self.R = h, QH, KVH, D, prefix, len(m)
        need = [(prefix + 31) // 32] + [(n + 31) // 32 for n in lens]
        self.cols = max(need[1:] + [0]) + spare
        P = max(1, sum(need)) + 3
        self.k = [rng.standard_normal((n, KVH, D)).astype(np.float16) for n in [prefix] + list(lens)]
        self.v = [(rng.standard_normal((n, KVH, D)) * size + 0.25).astype(np.float16) for n in [prefix] + list(lens)]
        self.kp, self.vp = h.kv_pages_alloc(P, KVH, D)
        self.kp.fill_(math.nan)
        self.vp.fill_(math.nan)
        order, tables = rng.permutation(P).astype(np.int32), []
        for n in need:
            tables.append(order[:n])
            order = order[n:]
        for t, k, v in zip(tables, self.k, self.v):
            if len(k):
                h.kv_write(dev(k).view(len(k), -1), dev(v).view(len(v), -1), self.kp, self.vp, 0, dev(t))
        self.there = []
        for i, (t, k) in enumerate(zip(tables, self.k)):
            gone = rng.random(len(t)) < absent
            t[gone] = rng.choice([-1, P, 1 << 30], gone.sum())
            self.there.append(~np.repeat(gone, 32)[:len(k)])
        self.prefix_table = dev(tables[0])
        own = np.full((self.R, max(self.cols, 1)), 1 << 20, np.int32)
        for r, t in enumerate(tables[1:]):
            own[r, :len(t)] = t
        self.own_table = dev(own)
        self.q_start_np = np.concatenate([[0], np.cumsum(m)]).astype(np.int32) + before
        self.T = int(self.q_start_np[-1]) + behind
        self.q_start, self.own_len = dev(self.q_start_np), dev(np.asarray(lens, np.int32))
        self.q_np = (rng.standard_normal((self.T, QH, D)) * 1.5).astype(np.float16)
        self.q = dev(self.q_np)
        self.max_tokens = max(list(m) + [1])

    def oracle(self, window=0, causal=True, gate=None, max_tokens=None):
        own = list(zip(self.k[1:], self.v[1:], self.there[1:]))
        return batch.shared_attention(self.q_np, self.k[0], self.v[0], self.there[0], self.q_start_np, own, max_tokens or self.max_tokens,
                                      window, causal, gate)

    def run(self, window=0, causal=True, gate=None, max_tokens=None, out=None, **kw):
        lse = torch.full((self.T, self.QH), 7.0, device="cuda")
        f32 = torch.full((self.T, self.QH, self.D), 7.0, device="cuda")
        out = torch.full((self.T, self.QH, self.D), 7.0, dtype=torch.float16, device="cuda")
        self.h.verify_attention_shared(self.q, self.kp, self.vp, self.prefix, self.q_start, self.own_len, self.own_table,
                                       max_tokens or self.max_tokens, prefix_table=kw.pop("prefix_table", self.prefix_table), window=window,
                                       causal=causal, out=out, out_f32=f32, lse=lse, gate=None if gate is None else dev(gate), **kw)
        return out, f32, lse

    def check(self, window=0, causal=True, gate=None, max_tokens=None, **kw):
        out, f32, lse = self.run(window, causal, gate, max_tokens, **kw)
        want, wlse, size = self.oracle(window, causal, gate, max_tokens)
        self.close(out, f32, lse, want, wlse, size)
        return out, f32, lse

    def close(self, out, f32, lse, want, wlse, size):
        """P is rounded to fp16: each weight is off by 2^-11 of itself in the products (were it in the sum too), so an output moves by at most
        2 x 2^-11 max |v|; a P below 2^-14 by 2^-25, of sums of at least 1, over all n keys: n 2^-25 (1 + max |v|), the one among
        the subnormals. Scores: D products of fp16 values, exact, summed in fp32: D roundings of 2^-24 of at most sum |q_i k_i|, which
        is under 2 D here (1.5 x 2 / pi D on average), over sqrt(D); the exponent's own rounding 2^-22. The gate's and the sums' own roundings are under 2^-20."""
        rows = ~np.isnan(wlse)
        for t, left in ((out, 7.0), (f32, 7.0), (lse, 7.0)):
            assert np.all(f64(t)[~rows] == left)
        n = self.prefix + max([len(k) for k in self.k[1:]] + [0])
        score = 2 * self.D ** 1.5 * 2.0 ** -24 + 2.0 ** -22
        got, l = f64(f32)[rows], f64(lse)[rows]
        want, wlse, size = want[rows], wlse[rows], size[rows]
        empty = np.isneginf(wlse)
        assert np.all(np.isneginf(l) == empty) and np.all(got[empty] == 0)
        bound = (2.0 ** -10 + 2 * score + 2.0 ** -20) * size + n * 2.0 ** -25 * (1 + size)
        assert np.all(np.abs(got - want) <= bound[..., None]), float(np.max(np.abs(got - want) - bound[..., None]))
        lb = 2.0 ** -11 + score + n * 2.0 ** -25 + 2.0 ** -22 * np.abs(np.where(empty, 0, wlse))
        assert np.all(np.abs(l[~empty] - wlse[~empty]) <= lb[~empty])
        assert np.array_equal(out[torch.from_numpy(rows).cuda().any(1)].cpu().numpy().astype(np.float32),
                              f32[torch.from_numpy(rows).cuda().any(1)].half().float().cpu().numpy())


GEOMETRY = [(32, 8, 64), (16, 4, 128), (8, 8, 128), (5, 1, 64), (12, 4, 64), (2, 1, 128)]


@pytest.mark.parametrize("QH,KVH,D", GEOMETRY)
@pytest.mark.parametrize("prefix,m,lens", [(1, [1], [1]), (0, [1, 2], [1, 40]), (33, [1, 1, 1], [1, 32, 33]), (500, [4, 1, 3], [4, 65, 200]),
                                            (64, [9], [9]), (1001, [1] * 20, list(range(1, 41, 2)))])
def test_shared(QH, KVH, D, prefix, m, lens):
    b = Batch(prefix + D, QH, KVH, D, prefix, m, lens)
    b.check(gate=np.random.default_rng(0).standard_normal((b.T, QH)).astype(np.float32))
    b.check(causal=False)


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("window", [1, 2, 31, 32, 33, 100, 400, 5000])
@pytest.mark.parametrize("causal", [True, False])
def test_shared_windows(D, window, causal):
    """Windows that end in the block, in the own keys, on the prefix's border, within the prefix and before everything."""
    b = Batch(window, 8, 2, D, 300, [3, 1, 5, 2], [3, 40, 130, 97])
    b.check(window=window, causal=causal)


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("prefix,m,lens", [(10, [20], [0]), (300, [20, 3, 9], [0, 3, 200]), (90, [1] * 30, [0] * 30), (1, [300], [2])])
def test_shared_windows_past_every_position(D, prefix, m, lens):
    """A window of at least all positions is none, bit for bit, up to the largest one and for sequences with fewer own keys than tokens: those
    in front of the first own key see the whole prefix."""
    b = Batch(prefix, 4, 2, D, prefix, m, lens)
    for causal in (True, False):
        want = b.run(causal=causal)
        if not causal:
            b.close(*want, *b.oracle(causal=False))
        for window in (prefix + 300, 5000, 1 << 30, 3 << 29, (1 << 31) - 5, (1 << 31) - 1):
            assert all(torch.equal(x, y) for x, y in zip(b.run(window=window, causal=causal), want)), window


@pytest.mark.parametrize("QH,KVH,D", [(32, 8, 64), (16, 4, 128)])
@pytest.mark.parametrize("seqs,tokens", [(1, 4), (8, 1), (12, 2), (5, 7), (17, 4), (33, 4), (65, 3)])
def test_shared_row_blocks(QH, KVH, D, seqs, tokens):
    """4 to 780 rows of a KV head: each shape of a prefix workgroup, whole and part blocks."""
    rng = np.random.default_rng(seqs)
    m = rng.integers(1, tokens + 1, seqs)
    m[0] = tokens
    b = Batch(seqs, QH, KVH, D, 203, m, m + rng.integers(0, 70, seqs))
    b.check()
    b.check(window=90)


@pytest.mark.parametrize("splits", [1, 2, 3, 7, 32, 1000])
@pytest.mark.parametrize("D,seqs", [(64, 3), (128, 3), (64, 40), (128, 40)])
def test_shared_splits(D, seqs, splits):
    b = Batch(splits, 8, 2, D, 999, [2] * seqs, list(range(2, 2 + seqs)))
    b.check(splits=splits)


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("seqs", [2, 40])
@pytest.mark.parametrize("share", [0.3, 1.0])
def test_shared_absent_pages(D, seqs, share):
    """Pages that no row sees, some or all of them: rows left with nothing give zeros and -inf."""
    b = Batch(seqs, 8, 2, D, 350, [3] * seqs, [3 + 41 * (r % 4) for r in range(seqs)], absent=share)
    b.check()
    b.check(window=60, causal=False)


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("seqs", [4, 50])
def test_shared_rows_and_tokens_left_out(D, seqs):
    """Rows before the first sequence, behind the last one and past max_tokens are left as they were; empty sequences between."""
    m = [(0, 3, 1, 6)[r % 4] for r in range(seqs)]
    b = Batch(seqs, 4, 2, D, 70, m, [x + 20 * (r % 3) for r, x in enumerate(m)], before=5, behind=7, spare=4)
    b.check()
    b.check(max_tokens=4)
    b.check(max_tokens=4, window=50)
    b.check(max_tokens=b.T)


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("what", [math.nan, math.inf, -math.inf])
def test_shared_not_finite_where_masked(D, what):
    """K and V rows of a block's last token (and of keys the window leaves out) that are not finite touch no row that does not see them;
    a row that sees one is not finite where V is not."""
    b = Batch(5, 4, 2, D, 64, [4, 2], [40, 2])
    at, d = 39, 7  # the first sequence's last token
    page, slot = int(b.own_table[0, at // 32]), at % 32
    b.vp[page, :, d, slot] = what
    b.v[1][at, :, d] = 0  # (for the restatement; the row that sees it is looked at below)
    out, f32, lse = b.run()
    want, wlse, size = b.oracle()
    assert not torch.isfinite(f32[3, :, d]).any()
    f32[3, :, d] = torch.from_numpy(want[3, :, d]).float().cuda()
    b.close(f32.half(), f32, lse, want, wlse, size)
    # a key of NaN that only the last token sees, and old ones behind the window
    b = Batch(6, 4, 2, D, 64, [4], [40])
    flat = b.kp.view(b.kp.shape[0], 2, 32 * D)
    idx = torch.from_numpy(b.h.k_page_index(D)).cuda()
    flat[int(b.own_table[0, 1]), :, idx[39 % 32]] = math.nan
    out, f32, lse = b.run(window=30)
    want, wlse, size = b.oracle(window=30)
    assert torch.isnan(f32[3]).all() and torch.isnan(lse[3]).all()
    f32[3], lse[3] = torch.from_numpy(want[3]).float().cuda(), torch.from_numpy(wlse[3]).float().cuda()
    b.close(f32.half(), f32, lse, want, wlse, size)


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("seqs", [3, 40])
def test_shared_growing_and_falling_scores(D, seqs):
    """Keys whose scores rise and fall by far more than the reference's slack, page after page."""
    b = Batch(11, 4, 2, D, 700, [2] * seqs, [40] * seqs)
    size = (0.05 + 6 * np.abs(np.sin(np.arange(700) / 90)))[:, None, None]
    b.k[0] = (b.k[0] * size).astype(np.float16)
    b.h.kv_write(dev(b.k[0]).view(700, -1), dev(b.v[0]).view(700, -1), b.kp, b.vp, 0, b.prefix_table)
    out, f32, lse = b.run()
    want, wlse, top = b.oracle()
    # scores are six times as large, and so is what fp32 sums of them lose: 6 x the bound of test_shared for the scores' part
    score = 6 * 2 * D ** 1.5 * 2.0 ** -24 + 2.0 ** -19
    assert np.all(np.abs(f64(f32) - want) <= ((2.0 ** -10 + 2 * score) * top + 740 * 2.0 ** -25 * (1 + top))[..., None])
    assert np.all(np.abs(f64(lse) - wlse) <= 2.0 ** -11 + score + 740 * 2.0 ** -25 + 2.0 ** -22 * np.abs(wlse))


@pytest.mark.parametrize("D,seqs", [(64, 1), (128, 1), (64, 20), (128, 20), (64, 70)])
def test_shared_lse(D, seqs):
    """lse is of the weights before they are rounded: scores and exponents as in Batch.close, n / 4 additions a lane and a logarithm."""
    b = Batch(seqs + D, 8, 2, D, 999, [2] * seqs, list(range(2, 2 + seqs)))
    _, _, lse = b.run()
    _, want, _ = b.oracle()
    n = 999 + 2 + seqs
    score = 2 * D ** 1.5 * 2.0 ** -24 + 2.0 ** -22
    assert np.all(np.abs(f64(lse) - want) <= score + (n / 4 + 64) * 2.0 ** -24 + 2.0 ** -22 * np.abs(want))


@pytest.mark.parametrize("seqs", [1, 20])
@pytest.mark.parametrize("D,b", [(64, 12.0), (128, 17.0)])
def test_shared_long_tail(D, b, seqs):
    """One key 18 above all others, with V of 0 where they have 1000: their share is n e^-18. P of a tail key is off by 2^-25 of a largest of 2^7
    at least, n 2^-32 of the whole; the rest as in Batch.close, of the output itself (the tail's weights are all alike)."""
    x = Batch(D, 2, 1, D, 20000, [1] * seqs, [1] * seqs)
    x.q_np[:] = 0
    x.q_np[:, :, 0] = 12
    for k, v in zip(x.k, x.v):
        k[:], v[:] = 0, 1000
    x.k[0][777, :, 0], x.v[0][777] = b, 0
    h, first = x.h, x.prefix_table.cpu().numpy()
    for t, k, v in zip([first] + list(x.own_table.cpu().numpy()), x.k, x.v):
        h.kv_write(dev(k).view(len(k), -1), dev(v).view(len(v), -1), x.kp, x.vp, 0, dev(t[:(len(k) + 31) // 32].copy()))
    x.q = dev(x.q_np)
    _, f32, lse = x.run()
    want, wlse, _ = x.oracle()
    score = 2 * D ** 1.5 * 2.0 ** -24 * 12 * b / 2 + 2.0 ** -22
    assert want.min() > 0.25
    assert np.all(np.abs(f64(f32) - want) <= 20001 * 2.0 ** -32 * 1000 + (2.0 ** -10 + score) * want)
    assert np.all(np.abs(f64(lse) - wlse) <= 20001 * 2.0 ** -32 + score + 2.0 ** -22 * np.abs(wlse))


def test_shared_is_verify_attention_of_each():
    """One sequence behind a prefix is the paged verify attention of the whole: both within their bounds, so within their sum."""
    h = load_host()
    b = Batch(21, 16, 4, 128, 96, [5], [37])
    _, f32, _ = b.run()
    k, v = (np.concatenate(x) for x in (b.k, b.v))
    kp, vp = h.kv_to_pages(dev(k).view(-1, 4, 128), dev(v).view(-1, 4, 128))
    ref = torch.empty((5, 16, 128), device="cuda")
    h.verify_attention(b.q, kp, vp, 128, out_f32=ref)
    assert float((f32 - ref).abs().max()) <= 2 * 2e-3


def test_shared_many_splits_of_many_rows():
    """64 sequences that may have 16384 tokens each, one of which has any: 2^24 rows asked for with more splits than a wave's two rounds. With
    one split the same within both bounds (P's roundings and scores', Batch.close; values are at most 4 here)."""
    h, T, QH, D, prefix = load_host(), 1 << 14, 16, 64, 67 * 32
    rng = np.random.default_rng(3)
    kp, vp = h.kv_pages_alloc(67, 1, D)
    k, v = ((rng.standard_normal((prefix, D))).clip(-4, 4).astype(np.float16) for _ in range(2))
    h.kv_write(dev(k), dev(v), kp, vp, 0, torch.arange(67, dtype=torch.int32, device="cuda"))
    q = dev(rng.standard_normal((64, QH, D)).astype(np.float16)).repeat(T // 64, 1, 1)
    start = torch.zeros(65, dtype=torch.int32, device="cuda")
    start[33:] = T
    none = torch.zeros(64, dtype=torch.int32, device="cuda")
    ws = h.Workspace("cuda")
    got = [h.verify_attention_shared(q, kp, vp, prefix, start, none, torch.zeros((64, 1), dtype=torch.int32, device="cuda"), T,
                                     causal=False, out_f32=torch.empty((T, QH, D), device="cuda"), splits=s, workspace=ws)[1] for s in (67, 1)]
    assert float((got[0] - got[1]).abs().max()) <= 2 * (2.0 ** -10 + 2 * (2 * D ** 1.5 * 2.0 ** -24 + 2.0 ** -22) + 2.0 ** -20) * 4 + 2 * prefix * 2.0 ** -25 * 5
    assert torch.equal(got[0][:64], got[0][-64:])


def test_shared_identity_table_and_strides():
    """No prefix table; q inside wider rows; own tables inside wider ones."""
    h = load_host()
    b = Batch(31, 8, 2, 64, 100, [2, 1], [34, 3])
    P = b.kp.shape[0]
    perm = torch.cat([b.prefix_table.long(), torch.tensor(sorted(set(range(P)) - set(b.prefix_table.tolist())), device="cuda")])
    where = torch.empty_like(perm)
    where[perm] = torch.arange(P, device="cuda")
    b.kp, b.vp = b.kp[perm].contiguous(), b.vp[perm].contiguous()
    wide = torch.full((2, 9), 1 << 20, dtype=torch.int32, device="cuda")
    old = b.own_table.long()
    wide[:, 3:3 + old.shape[1]] = torch.where(old < P, where[old.clamp(max=P - 1)], old).int()
    b.own_table = wide[:, 3:3 + old.shape[1]]
    b.prefix_table = None
    row = torch.zeros((b.T, 8 * 64 + 24), dtype=torch.float16, device="cuda")
    row[:, 16:16 + 512] = b.q.view(b.T, -1)
    b.q = row.as_strided((b.T, 8, 64), (8 * 64 + 24, 64, 1), 16)
    b.check()


@pytest.mark.parametrize("D,QH,KVH,prefix,m,lens", [(64, 32, 8, 9000, [1] * 8, [100] * 8), (128, 16, 4, 5003, [4] * 3, [900, 4, 2000]),
                                                    (64, 16, 2, 3000, [2] * 40, [50] * 40)])
def test_shared_long(D, QH, KVH, prefix, m, lens):
    """(Some thousand keys: what a P among the subnormals and fp32 sums lose stays within the bounds, which count keys.)"""
    Batch(77, QH, KVH, D, prefix, m, lens).check()


def test_shared_pools_past_4_gib():
    h, QH, KVH, D = load_host(), 8, 8, 128
    P = (9 << 29) // (KVH * 32 * D * 2)
    b = Batch(41, QH, KVH, D, 64, [2], [34])
    kp = torch.empty((P, KVH, 32, D), dtype=torch.float16, device="cuda")
    vp = torch.empty((P, KVH, D, 32), dtype=torch.float16, device="cuda")
    n = b.kp.shape[0]
    kp[-n:], vp[-n:] = b.kp, b.vp
    b.kp, b.vp = kp, vp
    b.prefix_table, b.own_table = b.prefix_table + (P - n), b.own_table + (P - n)
    b.check()


def test_shared_streams_and_graph():
    """A side stream; two calls at once with workspaces of their own; a captured call replayed after its lengths, table and rows changed,
    with eager work between; the same bits every time."""
    b = Batch(51, 16, 4, 128, 300, [3, 1, 2], [50, 7, 30], spare=1)
    c = Batch(52, 32, 8, 64, 150, [1] * 9, [40] * 9)
    eager = [b.run(), c.run()]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    spaces = [b.h.Workspace(), b.h.Workspace()]
    torch.cuda.synchronize()
    outs = []
    for _ in range(3):
        for x, s, w in zip((b, c), streams, spaces):
            with torch.cuda.stream(s):
                outs.append(x.run(workspace=w, stream=s))
    torch.cuda.synchronize()
    for i, o in enumerate(outs):
        assert all(torch.equal(x, y) for x, y in zip(o, eager[i % 2]))
    w = b.h.Workspace()
    static = [torch.full((b.T, 16, 128), 7.0, dtype=torch.float16, device="cuda"), torch.full((b.T, 16), 7.0, device="cuda")]

    def call():
        b.h.verify_attention_shared(b.q, b.kp, b.vp, b.prefix, b.q_start, b.own_len, b.own_table, b.max_tokens,
                                    prefix_table=b.prefix_table, out=static[0], lse=static[1], workspace=w)

    call()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        call()
    for i, lens in enumerate(([50, 7, 30], [3, 1, 2], [44, 6, 29], [50, 7, 30])):
        b.own_len.copy_(torch.tensor(lens, dtype=torch.int32))
        b.q.copy_(torch.randn_like(b.q))
        b.run()  # eager work of its own
        g.replay()
        torch.cuda.synchronize()
        want = b.run()
        assert torch.equal(static[0], want[0]) and torch.equal(static[1], want[2]), i


# ------------------------------------------------------------------------------------------------ sampling
def rows_of(kind, z):
    return dev(np.asarray(z, np.float32)).to(TYPES[kind])


def sample_check(logits, u, t=1.0, k=0, p=1.0, low=0.0, **kw):
    """Token and number kept exactly; the log-probability to the rounding of a weight (2^-45 of the largest one, of a token's share
    of the whole, e^lp x whole >= e^lp) and of the result."""
    h = load_host()
    n = logits.shape[0]
    per = [np.broadcast_to(np.asarray(x, ty), (n,)) for x, ty in ((u, np.float32), (t, np.float32), (k, np.int32), (p, np.float32), (low, np.float32))]
    args = [dev(per[i]) if np.ndim(x) or i == 0 else x for i, x in enumerate((u, t, k, p, low))]
    got = h.verify_sample(logits, args[0], temperature=args[1], top_k=args[2], top_p=args[3], min_p=args[4], keys=True, kept=True, logprob=True, **kw)
    z = logits.double().cpu().numpy()
    want = [batch.sample_row(z[r], *(float(x[r]) if i != 2 else int(x[r]) for i, x in enumerate(per))) for r in range(n)]
    token, kept, lp = got.tokens.cpu().numpy(), got.kept.cpu().numpy(), got.logprob.double().cpu().numpy()
    np.testing.assert_array_equal(kept, [w[1] for w in want])
    np.testing.assert_array_equal(token, [w[0] for w in want])
    np.testing.assert_array_equal(h.keys_to_tokens(got.keys).cpu().numpy()[token >= 0], token[token >= 0])
    assert np.all(got.keys.cpu().numpy()[token < 0] == 0)
    wl = np.array([w[2] for w in want])
    live = np.isfinite(wl)
    assert np.all(np.abs(lp[live] - wl[live]) <= 2.0 ** -23 * (np.abs(wl[live]) + 1) + 2.0 ** -43 * np.exp(-wl[live]))
    assert np.all(np.isneginf(lp[token < 0]))
    return got


U = [0.0, 1e-7, 0.03, 0.25, 0.5, 0.77, 0.9, 0.999, float(np.nextafter(np.float32(1), np.float32(0)))]


@pytest.mark.parametrize("kind", sorted(TYPES))
@pytest.mark.parametrize("V", [1, 2, 7, 64, 1000, 2048, 2049, 5003, 40000])
def test_sample(kind, V):
    rng = np.random.default_rng(V)
    n = len(U)
    logits = rows_of(kind, rng.standard_normal((n, V)) * 2.5)
    for how in (dict(), dict(t=0.7), dict(k=1), dict(k=min(V, 40)), dict(p=0.9), dict(low=0.05), dict(t=1.3, k=30, p=0.8, low=0.02), dict(p=0.0),
                dict(k=V), dict(k=V + 5), dict(low=1.0), dict(p=1e-9), dict(k=max(1, V - 1)), dict(t=0.05, p=0.99), dict(t=30.0, p=0.99),
                dict(k=200, p=0.95)):
        sample_check(logits, U, **how)


@pytest.mark.parametrize("kind", sorted(TYPES))
def test_sample_settings_by_row(kind):
    rng = np.random.default_rng(5)
    n, V = 300, 3001
    z = rng.standard_normal((n, V)) * rng.uniform(0.5, 4, (n, 1))
    z[rng.random((n, V)) < 0.2] = -np.inf
    sample_check(rows_of(kind, z), rng.random(n), t=rng.choice([0.0, 0.3, 1.0, 2.0], n), k=rng.choice([0, -3, 1, 5, 100, 4000], n),
                 p=rng.choice([0.0, 0.5, 0.9, 1.0, 2.0], n), low=rng.choice([0.0, -1.0, 0.01, 0.3, 1.0, 5.0], n))


@pytest.mark.parametrize("kind", sorted(TYPES))
@pytest.mark.parametrize("values", [1, 2, 5])
@pytest.mark.parametrize("V", [10, 3000, 30011])
def test_sample_ties(kind, values, V):
    """Rows of few different values: cuts within equal ones go by the index, whatever the number of them (over a list's length too)."""
    rng = np.random.default_rng(V + values)
    n = len(U)
    logits = rows_of(kind, rng.integers(0, values, (n, V)) * 0.5)
    for how in (dict(), dict(k=3), dict(k=V // 2), dict(p=0.5), dict(k=V // 2 + 1, p=0.7), dict(low=0.7), dict(p=0.999, low=0.7), dict(k=V - 1),
                dict(k=2500, p=0.99)):
        sample_check(logits, U, **how)


@pytest.mark.parametrize("kind", sorted(TYPES))
def test_sample_wide_nuclei(kind):
    """Cuts behind more tokens than a list holds: top-k alone, top-p alone, both, with min-p."""
    rng = np.random.default_rng(9)
    n, V = len(U), 50021
    logits = rows_of(kind, rng.standard_normal((n, V)) * 0.8)
    for how in (dict(k=9000), dict(p=0.95), dict(k=20000, p=0.9), dict(p=0.97, low=0.02), dict(k=30000, low=0.05), dict(k=2049), dict(k=2048),
                dict(p=0.2), dict(t=5.0, p=0.999)):
        sample_check(logits, U, **how)


@pytest.mark.parametrize("kind,V,values", [("bf16", 128001, "coarse"), ("f16", 60000, "coarse"), ("f32", 200003, "normal"), ("f32", 262144, "narrow"),
                                           ("f32", 30011, "close"), ("f32", 30011, "ends")])
def test_sample_crowded_bins(kind, V, values):
    """Cuts within a bin of more tokens than a list: equal logits by thousands (far from zero, coarse types), many different ones, pairs of
    values closer than the bin's parts, and whole rows of one value with a few above and below."""
    rng = np.random.default_rng(V)
    n = len(U)
    if values == "coarse":
        z = 40 + 2 * rng.standard_normal((n, V))
    elif values == "normal":
        z = 1.2 * rng.standard_normal((n, V)) + 7.0 * (rng.random((n, V)) < 1e-4)
    elif values == "narrow":
        z = -3 + 0.01 * rng.random((n, V)) + 3.0 * (rng.random((n, V)) < 1e-5)
    elif values == "close":
        z = -0.5 + 1e-6 * rng.integers(0, 2, (n, V)) + 0.5 * (np.arange(V) == 777)
    else:
        z = np.where(np.arange(V) % 997 == 5, 2.0, np.where(np.arange(V) % 991 == 7, -2.0, 0.0)) * np.ones((n, 1))
    logits = rows_of(kind, z)
    for how in (dict(p=0.3), dict(p=0.6), dict(p=0.9), dict(p=0.97, t=1.3), dict(p=0.99, low=0.3), dict(p=0.5, low=0.9), dict(k=50), dict(k=5000),
                dict(k=V // 2), dict(k=V // 2, low=0.2), dict(k=V - 9)):
        sample_check(logits, U, **how)


@pytest.mark.parametrize("kind", sorted(TYPES))
@pytest.mark.parametrize("ties", [257, 700, 2000, 3500])
def test_sample_ties_that_no_division_of_a_bin_parts(kind, ties):
    """A list of more than 256 tokens of which one 256th of the bin holds more than 256 as well, a few in the part before it: the cut by
    digits. Many rows, so that the waves of many workgroups come there at all kinds of times."""
    rng = np.random.default_rng(ties)
    n, V = 96, 9001
    z = np.full((n, V), -30.0)
    for r in range(n):
        at = rng.permutation(V)
        z[r, at[0]], z[r, at[1:11]], z[r, at[11:11 + ties]] = 0.0, -2.0, -2.0 if kind == "bf16" else -2.0 - 2.0 ** -7
    logits, u = rows_of(kind, z), rng.random(n)
    for how in (dict(p=0.5), dict(p=0.9, low=0.01), dict(p=rng.uniform(0.3, 0.95, n)), dict(k=20 + ties // 2), dict(k=rng.integers(12, 10 + ties, n)),
                dict(k=ties, p=0.6)):
        sample_check(logits, u, **how)


@pytest.mark.parametrize("kind", sorted(TYPES))
def test_sample_special_values(kind):
    inf, nan = math.inf, math.nan
    big = float(torch.finfo(TYPES[kind]).max)
    rows = [[-inf] * 6, [nan] * 6, [nan, -inf, 2, 1, nan, 2], [inf, 1, inf, -inf, nan, 0], [inf, -big, 3, 3, 3, 3], [-big] * 6, [big] * 6,
            [big, -big, 0, -big, big, -inf], [-0.0, 0.0, -0.0, 0.0, -1, -0.0], [0, 1e-7, 0, -1e-7, 0, 0], [-inf, -inf, -inf, -inf, -inf, -5]]
    for u in (0.0, 0.4, 0.99):
        for how in (dict(), dict(k=2), dict(p=0.6), dict(low=0.5), dict(t=0.0), dict(t=1e-30), dict(t=inf), dict(t=nan), dict(t=-1.0), dict(k=4, p=0.5),
                    dict(p=nan), dict(low=nan)):
            sample_check(rows_of(kind, rows), [u] * len(rows), **how)
    sample_check(rows_of(kind, rows), [nan, -1.0, 1.0, 2.0, inf, -inf, 0.5, 0.5, 0.5, 0.5, 0.5])


@pytest.mark.parametrize("kind", sorted(TYPES))
@pytest.mark.parametrize("V", [(1 << 20) - 1, 1 << 20])
def test_sample_the_largest_rows(kind, V):
    """2^20 tokens of the largest weight each, by every way through the launches: their sum has to fit. Flat rows, an infinite temperature
    and rows of infinities; one token above all others; ordinary values."""
    rng = np.random.default_rng(V)
    u = [0.0, 0.03, 0.5, 0.9999, U[-1]]
    flat = rows_of(kind, np.zeros((len(u), V)))
    for how in (dict(), dict(p=0.9), dict(p=1e-6), dict(low=0.5), dict(k=V - 1), dict(k=700000, p=0.5), dict(k=300), dict(t=math.inf, p=0.999)):
        sample_check(flat, u, **how)
    sample_check(rows_of(kind, np.full((len(u), V), math.inf)), u)
    sample_check(rows_of(kind, np.full((len(u), V), math.inf)), u, p=0.9)
    logits = rows_of(kind, rng.standard_normal((len(u), V)))
    for how in (dict(), dict(p=0.9), dict(t=math.inf), dict(k=40, p=0.9)):
        sample_check(logits, u, **how)


@pytest.mark.parametrize("n", [1, 3, 700, 5000])
def test_sample_rows(n):
    """One row to thousands, rows inside wider ones and off 16-byte boundaries."""
    rng = np.random.default_rng(n)
    V = 20011 if n < 100 else 501
    for off, stride in ((0, V), (1, V + 3), (8, V - V % 8 + 16)):
        flat = torch.full((off + n * stride + 8,), 9.0, dtype=torch.float16, device="cuda")
        view = flat.as_strided((n, V), (stride, 1), off)
        view.copy_(dev((rng.standard_normal((n, V)) * 2).astype(np.float16)))
        sample_check(view, rng.random(n), t=0.8, k=rng.integers(0, 50, n), p=0.9)


def test_sample_is_the_distribution():
    """u over a grid of 65535: each token is drawn as often as its probability says, to one step of the grid on either side."""
    n, V = 65535, 33
    z = np.random.default_rng(2).standard_normal(V) * 1.5
    logits = rows_of("f32", z).expand(n, V).contiguous()
    u = dev(((np.arange(n) + 0.5) / n).astype(np.float32))
    got = load_host().verify_sample(logits, u).tokens
    p = np.exp(z.astype(np.float32).astype(np.float64))
    count = np.bincount(got.cpu().numpy(), minlength=V)
    assert np.all(np.abs(count - n * p / p.sum()) <= 1.01)
    assert np.all(np.diff(got.cpu().numpy()) >= 0)


def test_sample_streams_graph_and_repeats():
    h, rng = load_host(), np.random.default_rng(4)
    n, V = 20, 30000
    logits, u = rows_of("f16", rng.standard_normal((n, V)) * 2), dev(rng.random(n).astype(np.float32))
    k = dev(rng.integers(0, 3, n).astype(np.int32) * 1200)
    how = dict(temperature=0.9, top_k=k, top_p=0.97, kept=True, logprob=True)
    want = h.verify_sample(logits, u, **how)
    same = lambda a, b: all(torch.equal(getattr(a, x), getattr(b, x)) for x in ("tokens", "kept", "logprob"))  # noqa: E731
    streams, spaces, got = [torch.cuda.Stream() for _ in range(2)], [h.Workspace() for _ in range(2)], []
    torch.cuda.synchronize()
    for _ in range(4):
        for s, w in zip(streams, spaces):
            got.append(h.verify_sample(logits, u, workspace=w, stream=s, **how))
    torch.cuda.synchronize()
    assert all(same(g, want) for g in got)
    w = h.Workspace()
    out = dict(tokens=torch.zeros(n, dtype=torch.int32, device="cuda"), kept=torch.zeros(n, dtype=torch.int32, device="cuda"),
               logprob=torch.zeros(n, device="cuda"))
    call = lambda: h.verify_sample(logits, u, temperature=0.9, top_k=k, top_p=0.97, workspace=w, **out)  # noqa: E731
    call()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        call()
    for i in range(4):
        u.copy_(torch.rand_like(u))
        logits.copy_(torch.randn_like(logits) * (i + 1))
        want = h.verify_sample(logits, u, **how)
        g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(out[x], getattr(want, x)) for x in out), i


def test_sample_keys_feed_accept_commit():
    """A round of drafts against draws: the longest prefix of drafts equal to their row's draw, then the draw that differs."""
    h, rng = load_host(), np.random.default_rng(6)
    M, V = 6, 4096
    logits, u = rows_of("f32", rng.standard_normal((M, V)) * 3), dev(rng.random(M).astype(np.float32))
    drawn = h.verify_sample(logits, u, temperature=0.8, top_k=50, keys=True)
    t = drawn.tokens.tolist()
    for agree in (0, 2, 5):
        drafts = t[:agree] + [(t[i] + 1) % V for i in range(agree, M - 1)]
        st = h.state_tensor(a=100, anchor=7, tokens=[7] + drafts, rounds_left=32, budget=512, eos=-1, stop_at=128, run=1, skip_rounds=1)
        out, seen = torch.zeros(64, dtype=torch.int32, device="cuda"), torch.zeros(V // 32, dtype=torch.int32, device="cuda")
        h.accept_commit(st, drawn.keys, M, out, seen)
        got = h.state_from_tensor(st)
        assert got.accepted == agree and got.a == 100 + agree + 1
        assert out[:agree + 1].tolist() == t[:agree + 1]


@pytest.mark.parametrize("empty,agree", [(0, 5), (2, 5), (5, 5), (3, 1), (2, 2)])
@pytest.mark.parametrize("pad", [False, True])
def test_sample_rows_with_nothing_to_draw_end_a_commit(orc, empty, agree, pad):
    """A masked row first, in the middle, last, behind the first miss (5 drafts, of which `agree` are their rows' draws; pad: the draft that
    answers the masked row is -1): State, tokens and bitmap are the oracle's, and the words around the bitmap stay as they are."""
    h, rng = load_host(), np.random.default_rng(empty)
    M, V = 6, 4096
    z = rng.standard_normal((M, V)) * 3
    z[empty] = -np.inf
    drawn = h.verify_sample(rows_of("f32", z), dev(rng.random(M).astype(np.float32)), temperature=0.8, top_k=50, keys=True)
    t = drawn.tokens.tolist()
    assert t[empty] == -1 and int(drawn.keys[empty]) == 0
    tokens = [7] + [max(t[i], 0) if i < agree else (t[i] + 1) % V for i in range(M - 1)]
    if pad and empty < M - 1:
        tokens[empty + 1] = -1
    base = dict(a=100, anchor=7, tokens=tokens, rounds_left=32, budget=512, eos=-1, stop_at=128, run=1, skip_rounds=1, count=3)
    st, out = h.state_tensor(**base), torch.full((64,), -7, dtype=torch.int32, device="cuda")
    words = torch.full((16 + V // 32 + 16,), 1 << 20, dtype=torch.int32, device="cuda")
    h.accept_commit(st, drawn.keys, M, out, words[16:16 + V // 32])
    got = h.state_from_tensor(st)
    want, wout, wseen = orc.new_state(**base), np.full(64, -7, np.int32), np.full(V // 32, 1 << 20, np.uint32)
    acc = orc.accept_commit(want, t, M, wout, wseen)
    assert acc == min(empty, agree) and got.run == (1 if agree < empty else 0)
    for f in h.STATE_FIELDS:
        assert getattr(got, f) == getattr(want, f), f
    assert [got.tokens[i] for i in range(64)] == [want.tokens[i] for i in range(64)]
    np.testing.assert_array_equal(out.cpu().numpy(), wout)
    words = words.cpu().numpy()
    np.testing.assert_array_equal(words[16:-16].view(np.uint32), wseen)
    assert np.all(words[:16] == 1 << 20) and np.all(words[-16:] == 1 << 20)


# ------------------------------------------------------------------------------------------------ together
@pytest.mark.parametrize("QH,KVH,D", [(32, 8, 64), (16, 4, 128)])
def test_a_server_step(QH, KVH, D):
    """Several answers to one prompt, steps of one token each and one of drafted blocks: q and k turned and appended by slot, attention
    behind the prompt, a head, a draw -- eager, then the same steps from one captured graph, the same bits."""
    h, rng = load_host(), np.random.default_rng(8)
    R, prefix, V, steps, P = 5, 70, 1000, 4, 3 + 5 * 2
    f, scale = h.rope_freqs(D // 2, 1e4, "ramp", 4.0, 64)
    fd = dev(f)
    pk, pv = (rng.standard_normal((prefix, KVH, D)).astype(np.float16) for _ in range(2))
    head = dev((rng.standard_normal((QH * D, V)) / 12).astype(np.float32))
    table = rng.permutation(P).astype(np.int32)
    own = dev(table[3:].reshape(R, 2))
    ppos = np.arange(prefix)
    proj = [dev((rng.standard_normal((R * 3, (QH + 2 * KVH) * D))).astype(np.float16)) for _ in range(steps)]
    us = [dev(rng.random(R * 3).astype(np.float32)) for _ in range(steps)]
    ms = [[1] * R, [1] * R, [3, 1, 2, 1, 3], [1] * R]

    def fresh():
        kp, vp = h.kv_pages_alloc(P, KVH, D)
        h.rope_append(torch.zeros((prefix, 1, D), dtype=torch.float16, device="cuda"), dev(pk), dev(pv), dev(ppos.astype(np.int32)), fd, kp, vp,
                      dev(table[:3].astype(np.int64)[ppos // 32] * 32 + ppos % 32), scale=scale)
        return kp, vp

    kp, vp = fresh()
    static = dict(row=torch.zeros_like(proj[0]), u=torch.zeros_like(us[0]), pos=torch.zeros(R * 3, dtype=torch.int32, device="cuda"),
                  slots=torch.zeros(R * 3, dtype=torch.int64, device="cuda"), start=torch.zeros(R + 1, dtype=torch.int32, device="cuda"),
                  len=torch.zeros(R, dtype=torch.int32, device="cuda"))
    w1, w2 = h.Workspace(), h.Workspace()
    prefix_table = dev(table[:3])

    def step():
        n, st = R * 3, static
        heads = st["row"].view(n, QH + 2 * KVH, D)
        q = h.rope_append(heads[:, :QH], heads[:, QH:QH + KVH], heads[:, QH + KVH:], st["pos"], fd, kp, vp, st["slots"], scale=scale)
        o = torch.zeros((n, QH, D), device="cuda")
        h.verify_attention_shared(q, kp, vp, prefix, st["start"], st["len"], own, 3, prefix_table=prefix_table, out_f32=o, workspace=w1)
        logits = o.view(n, -1) @ head
        return q, o, logits, h.verify_sample(logits, st["u"], temperature=0.9, top_k=40, top_p=0.95, keys=True, workspace=w2)

    def load(i, lens):
        """Tokens of each sequence side by side; rows behind the last one are nobody's (slot -1)."""
        m = ms[i]
        start = np.concatenate([[0], np.cumsum(m)])
        seq, at = np.repeat(np.arange(R), m), np.concatenate([np.arange(x) for x in m])
        local = np.asarray(lens)[seq] + at
        pad = R * 3 - len(seq)
        slots = own.cpu().numpy()[seq, local // 32].astype(np.int64) * 32 + local % 32
        static["row"].copy_(proj[i])
        static["u"].copy_(us[i])
        static["pos"].copy_(dev(np.concatenate([prefix + local, np.zeros(pad)]).astype(np.int32)))
        static["slots"].copy_(dev(np.concatenate([slots, np.full(pad, -1)])))
        static["start"].copy_(dev(start.astype(np.int32)))
        lens = [x + y for x, y in zip(lens, m)]
        static["len"].copy_(dev(np.asarray(lens, np.int32)))
        return lens, start

    lens0 = [0, 3, 31, 32, 40]  # (own rows before the first step hold zeros: keys like any other)
    lens, eager = lens0, []
    hist = [(np.zeros((n, KVH, D), np.float16), np.zeros((n, KVH, D), np.float16)) for n in lens0]
    pk_turned = batch.rope(pk, ppos, f, scale=scale).astype(np.float16)
    for i in range(steps):
        lens, start = load(i, lens)
        q, o, logits, s = step()
        eager.append([x.clone() for x in (q, o, logits, s.tokens, s.keys)])
        n, rows = start[-1], proj[i].cpu().numpy().reshape(R * 3, QH + 2 * KVH, D)
        pos = static["pos"].cpu().numpy()
        for r in range(R):
            at = slice(start[r], start[r + 1])
            k = batch.rope(rows[at, QH:QH + KVH], pos[at], f, scale=scale).astype(np.float16)
            hist[r] = np.concatenate([hist[r][0], k]), np.concatenate([hist[r][1], rows[at, QH + KVH:]])
        want, _, size = batch.shared_attention(q.cpu().numpy(), pk_turned, pv, np.ones(prefix), start, [(k, v, np.ones(len(k))) for k, v in hist], 3)
        # test_shared's bound with scores twice as large (scale 1.14 of q and k); a K value that rounds to the other neighbour after fp32's
        # products moves a score by 2^-11 |q_d k_d| / sqrt(D) < 2^-11 x 1.2, and is one in some hundred
        bound = (2.0 ** -10 + 2 * (4 * 2 * D ** 1.5 * 2.0 ** -24 + 2.0 ** -10)) * size[:n] + 2.0 ** -16
        assert np.all(np.abs(f64(o)[:n] - want[:n]) <= bound[..., None])
        assert bool((o[n:] == 0).all())
        z = logits.double().cpu().numpy()
        for t in range(R * 3):
            assert int(s.tokens[t]) == batch.sample_row(z[t], float(us[i][t]), np.float32(0.9), 40, float(np.float32(0.95)))[0]
    # the same steps from a graph, with the buffers' contents changed between replays
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        q, o, logits, s = step()
    a, b = fresh()
    kp.copy_(a)
    vp.copy_(b)
    lens = lens0
    for i in range(steps):
        lens, start = load(i, lens)
        g.replay()
        torch.cuda.synchronize()
        for name, x, y in zip(("q", "o", "logits", "tokens", "keys"), (q, o, logits, s.tokens, s.keys), eager[i]):
            assert torch.equal(x, y), (i, name)


def test_the_binding_refuses():
    h = load_host()
    E = h.DsparkError
    x = torch.zeros((4, 2, 64), dtype=torch.float16, device="cuda")
    pos, f = torch.zeros(4, dtype=torch.int32, device="cuda"), dev(batch.rope_freqs(64, 1e4)[0])
    kp, vp = h.kv_pages_alloc(2, 2, 64)
    slots = torch.zeros(4, dtype=torch.int64, device="cuda")
    for bad in ((x.double(), None, pos, f), (x, x[:3], pos, f), (x, x.float(), pos, f), (None, None, pos, f), (x, None, pos[:3], f),
                (x, None, pos.long(), f), (x, None, pos, f.float()), (x.transpose(0, 1), None, pos, f), (x, None, pos.cpu(), f),
                (x, None, pos, f.repeat(2)), (x[..., :33], None, pos, f[:4]), (x.cpu(), None, pos.cpu(), f.cpu())):
        with pytest.raises(E):
            h.rope(*bad)
    with pytest.raises(E):
        h.rope(x, None, pos, f, q_out=x[:3])
    for bad in ((x, x, x[:3], pos, f, kp, vp, slots), (x, x, x, pos, f, kp, vp, slots.int()), (x, x, x, pos, f, kp.float(), vp, slots),
                (x, x, x, pos, f, vp, kp, slots[:2]), (x, None, x, pos, f, kp, vp, slots), (x.float(), x.float(), x, pos, f, kp, vp, slots)):
        with pytest.raises(E):
            h.rope_append(*bad)
    start, lens = torch.tensor([0, 2, 4], dtype=torch.int32, device="cuda"), torch.full((2,), 2, dtype=torch.int32, device="cuda")
    table = torch.zeros((2, 1), dtype=torch.int32, device="cuda")
    ok = dict(q=x, k_pages=kp, v_pages=vp, prefix=1, q_start=start, own_len=lens, own_table=table, max_tokens=2)
    h.verify_attention_shared(**ok)
    for bad in (dict(q=x.float()), dict(q=x[..., :32]), dict(k_pages=kp.float()), dict(v_pages=kp), dict(prefix=-1), dict(prefix=65),
                dict(q_start=start[:2]), dict(q_start=start.long()), dict(own_len=lens.long()), dict(own_table=table[:1]), dict(own_table=table.long()),
                dict(own_table=table.cpu()), dict(max_tokens=0), dict(max_tokens=-1), dict(window=-1), dict(window=1 << 32),
                dict(prefix_table=torch.zeros(0, dtype=torch.int32, device="cuda")), dict(gate=torch.zeros(4, 2)),
                dict(gate=torch.zeros((4, 1), device="cuda")), dict(lse=torch.zeros((4, 2), device="cuda").t().contiguous()),
                dict(out=x), dict(out=torch.zeros((3, 2, 64), dtype=torch.float16, device="cuda"))):
        with pytest.raises(E):
            h.verify_attention_shared(**{**ok, **bad})
    z, u = torch.zeros((4, 10), device="cuda"), torch.zeros(4, device="cuda")
    for bad, how in (((z.double(), u), {}), ((z, u[:3]), {}), ((z, u.double()), {}), ((z.t(), u), {}), ((z[0], u), {}), ((z, u.cpu()), {}),
                     ((z, u), dict(top_k=u)), ((z, u), dict(temperature=u[:2])), ((z, u), dict(tokens=False)), ((z, u), dict(tokens=u)),
                     ((z, u), dict(top_k=1 << 31)), ((z, u), dict(kept=torch.zeros(3, dtype=torch.int32, device="cuda"))),
                     ((z.expand(4, 10)[:1].expand(4, 10), u), {}), ((z, z[:, 0].contiguous()), dict(logprob=z.view(-1)[:4]))):
        with pytest.raises(E):
            h.verify_sample(*bad, **how)
