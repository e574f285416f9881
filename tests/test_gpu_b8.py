"""The 8-bit block-scaled K/V cache on the GPU against its restatement in float64 (oracle/b8.py): the writer, reader and
eviction exactly, the attention and the accounts of attention weight within bounds derived below."""
import numpy as np
import pytest
import torch

from conftest import load_host
from oracle import b8

pytestmark = pytest.mark.gpu
KINDS = ["int8", "e4m3"]
TYPES = {"int8": torch.int8, "e4m3": torch.float8_e4m3fn}


def dev(x):
    return torch.from_numpy(np.ascontiguousarray(x)).to("cuda")


def gpu_cache(c):
    """A device cache with the oracle cache's contents."""
    h = load_host()
    codes = [dev(c.raw[x]).view(TYPES[c.code]) for x in "kv"]
    table = None if c.table is None else dev(np.asarray(c.table, np.int32))
    return h.B8Cache(*codes, *(dev(c.scale[x]) for x in "kv"), table)


def assert_same(g, c, where=""):
    """Scales and the values of every code equal (the two zeros of e4m3 are one value)."""
    for x in "kv":
        raw = getattr(g, x).view(torch.uint8).cpu().numpy()
        np.testing.assert_array_equal(getattr(g, x + "_scale").cpu().numpy(), c.scale[x], err_msg=where + x + "_scale")
        np.testing.assert_array_equal(b8.values(c.code, raw), b8.values(c.code, c.raw[x]), err_msg=where + x)


def rows(rng, n, KVH, D, size=1.0):
    return (rng.standard_normal((n, KVH, D)) * size).astype(np.float16)


def filled(code, T, KVH, D, seed, table=None, pages=None, size=1.0):
    """An oracle cache holding T positions whose blocks differ in size."""
    rng = np.random.default_rng(seed)
    n = (T + 31) // 32
    c = b8.Cache(code, pages or n, KVH, D, table)
    sz = np.repeat(2.0 ** rng.uniform(-2, 1, (n, KVH, 1)), 32, 0)[:T] * size
    c.write((rng.standard_normal((T, KVH, D)) * sz).astype(np.float16),
            (rng.standard_normal((T, KVH, D)) * sz[::-1] + 0.25).astype(np.float16), 0)
    return c


# ------------------------------------------------------------------------------------------------ append and read
@pytest.mark.parametrize("code", KINDS)
@pytest.mark.parametrize("KVH,D", [(8, 64), (4, 128), (1, 64), (3, 128)])
@pytest.mark.parametrize("spans", [[(0, 1)], [(0, 32)], [(0, 33), (33, 31)], [(0, 200), (131, 9), (140, 16), (150, 1)],
                                   [(0, 70), (64, 3), (95, 2), (96, 32)]])
def test_appends_and_reads(code, KVH, D, spans):
    """Appends in turn (some starting before the last one's end, sizes growing and shrinking) through a permuted table."""
    h = load_host()
    rng = np.random.default_rng(len(spans) * 1000 + D + KVH)
    table = rng.permutation(9).astype(np.int32)
    c = b8.Cache(code, 9, KVH, D, table)
    for x in "kv":  # what an earlier sequence left
        c.raw[x][:] = 5
        c.scale[x][:] = 0.5
    g = gpu_cache(c)
    for i, (pos0, n) in enumerate(spans):
        k, v = rows(rng, n, KVH, D, 2.0 ** (3 * (i % 2) - 1)), rows(rng, n, KVH, D, 2.0 ** -i)
        wide = torch.zeros((n, 2 * KVH * D + 8), dtype=torch.float16, device="cuda")  # K and V inside wider rows
        wide[:, :KVH * D], wide[:, KVH * D:2 * KVH * D] = dev(k).view(n, -1), dev(v).view(n, -1)
        h.kv_write_b8(wide[:, :KVH * D], wide[:, KVH * D:2 * KVH * D], g, pos0)
        c.write(k, v, pos0)
        assert_same(g, c, f"after append {i}: ")
        h.kv_write_b8(wide[:, :KVH * D], wide[:, KVH * D:2 * KVH * D], g, pos0)  # the same rows again change nothing
        assert_same(g, c, f"after append {i} again: ")
    end = spans[-1][0] + spans[-1][1]
    for pos0, n in ((0, end), (max(0, end - 1), 1), (min(5, end - 1), end - min(5, end - 1))):
        k, v = h.kv_read_b8(g, pos0, n)
        want = c.read(pos0, n)
        np.testing.assert_array_equal(k.cpu().numpy().astype(np.float64), want[0])
        np.testing.assert_array_equal(v.cpu().numpy().astype(np.float64), want[1])


@pytest.mark.parametrize("code", KINDS)
def test_append_special_values(code):
    """Zeros, subnormals, the largest halves, NaN and infinities, and rows on the borders between two codes."""
    h = load_host()
    KVH, D = 2, 64
    x = np.zeros((160, KVH, D), np.float16)
    x[0:32] = 0
    x[32:64] = np.linspace(-6e-8, 6e-8, D).astype(np.float16)
    x[64:96, 0] = np.linspace(-65504, 65504, D).astype(np.float16)
    x[64:96, 1] = np.float16(-0.0)
    x[96:128] = np.arange(-32, 32, dtype=np.float32).astype(np.float16) / 2 + np.float16(0.5)  # borders: scale 2^-3 below
    x[96, :, 0] = np.float16(127 / 8)
    x[128:160] = np.random.default_rng(3).standard_normal((32, KVH, D)).astype(np.float16)
    x[130, 0, 3:6] = [np.nan, np.inf, -np.inf]
    x[131, 1] = np.nan
    y = x[::-1].copy()
    c = b8.Cache(code, 5, KVH, D)
    g = gpu_cache(c)
    h.kv_write_b8(dev(x), dev(y), g, 0)
    c.write(x, y, 0)
    assert_same(g, c)
    # a block of nothing but NaN and infinities has scale 0
    bad = np.full((1, KVH, D), np.inf, np.float16)
    bad[0, 1] = np.nan
    h.kv_write_b8(dev(bad), dev(-bad), g, 32)
    c.write(bad, -bad, 32)
    assert_same(g, c)


@pytest.mark.parametrize("code", KINDS)
def test_append_borders_between_codes(code):
    """Values exactly between two codes and one half-precision step to either side, at a scale that is no power of two."""
    h = load_host()
    for amax in (1.0, 0.3, 63.5, 1016.0, 40000.0):
        a = np.float16(amax)
        s = float(b8.scale_of(code, np.float64(a)))
        mid = (np.arange(-127, 127) + 0.5) * s if code == "int8" else (b8._E4M3_POS[:-1] + b8._E4M3_POS[1:]) / 2 * s
        near = mid.astype(np.float16)
        near = np.concatenate([near, np.nextafter(near, np.float16(np.inf)), np.nextafter(near, np.float16(-np.inf)), -near])
        near = near[np.abs(near) <= a]
        x = np.zeros(32 * 128, np.float16)
        x[:len(near)], x[-1] = near[:len(x) - 1], a
        x = x.reshape(32, 1, 128)
        c = b8.Cache(code, 1, 1, 128)
        g = gpu_cache(c)
        h.kv_write_b8(dev(x), dev(-x), g, 0)
        c.write(x, -x, 0)
        assert_same(g, c, f"amax {amax}: ")


@pytest.mark.parametrize("code", KINDS)
def test_absent_pages_are_neither_written_nor_read(code):
    h = load_host()
    rng = np.random.default_rng(5)
    c = b8.Cache(code, 4, 2, 64, np.array([2, -1, 4, 0, 1 << 30, 3], np.int32))
    g = gpu_cache(c)
    k, v = rows(rng, 190, 2, 64), rows(rng, 190, 2, 64)
    h.kv_write_b8(dev(k), dev(v), g, 1)
    c.write(k, v, 1)
    assert_same(g, c)
    out = [torch.full((190, 2, 64), 7.0, device="cuda") for _ in "kv"]
    h.kv_read_b8(g, 1, 190, *out)
    want = c.read(1, 190)
    np.testing.assert_array_equal(out[0].cpu().numpy(), want[0].astype(np.float32))
    np.testing.assert_array_equal(out[1].cpu().numpy(), want[1].astype(np.float32))


def test_read_into_wider_rows_leaves_the_rest():
    h = load_host()
    c = filled("int8", 77, 3, 64, 1)
    g = gpu_cache(c)
    out = [torch.full((40, 3 * 64 + 4), 7.0, device="cuda") for _ in "kv"]
    h.kv_read_b8(g, 30, 39, *out)
    for o, want in zip(out, c.read(30, 39)):
        np.testing.assert_array_equal(o[:39, :192].cpu().numpy(), want.reshape(39, -1).astype(np.float32))
        assert bool((o[39:] == 7).all()) and bool((o[:, 192:] == 7).all())


@pytest.mark.parametrize("n", [1, 39])
def test_reads_and_appends_of_rows_side_by_side(n):
    h = load_host()
    c = filled("e4m3", 77, 3, 64, 2)
    wide = torch.full((n, 2, 3, 64), 7.0, device="cuda")
    h.kv_read_b8(gpu_cache(c), 30, n, wide[:, 0], wide[:, 1])
    for x, want in zip(wide.unbind(1), c.read(30, n)):
        np.testing.assert_array_equal(x.cpu().numpy(), want.astype(np.float32))
    half = wide.half()
    g = h.b8_cache_alloc(2, 3, 64, torch.float8_e4m3fn)
    h.kv_write_b8(half[:, 0], half[:, 1], g, 5)
    w = b8.Cache("e4m3", 2, 3, 64)
    w.write(*half.cpu().numpy().transpose(1, 0, 2, 3), 5)
    for x, want in zip(h.kv_read_b8(g, 5, n), w.read(5, n)):
        np.testing.assert_array_equal(x.cpu().numpy(), want.astype(np.float32))


# ------------------------------------------------------------------------------------------------ attention
# Of a result o = sum p v with A = sum p |v| (p the softmax): V's scale vs goes into the exponent and p vs, times a power of two
# that takes the row's largest to at least 2^8, is rounded to fp16 once: by 2^-11 of itself where that is a normal half, and
# by 2^-25 below 2^-14, which is 2^-33 of the row's largest. Codes c are up to T = 127 or 448, so the latter errors of N keys
# are under 2^-33 N max(p vs) T, and max(p vs T) <= B = sum p vs T. Scores of up to 64 (log2 units) are sums of exact products
# in fp32, off by about 2^-24 64 = 2^-18, log2 vs (up to 32) by 2^-19, and their exponential relatively by as much; sums in
# fp32 add a few 2^-24 more. 2^-16 A covers these. The fp16 output is rounded once more.
def bound(o, mag, half, N, B):
    return ((2.0 ** -11 + 2.0 ** -16) * mag + 2.0 ** -33 * N * B + (2.0 ** -11 * np.abs(o) + 2.0 ** -25 if half else 0) + 1e-9)


def tops(c, n):
    """What the largest code of each position's V block stands for, [n][KVH][1]."""
    pg = np.array([c.page(i // 32) for i in range(n)])
    return (np.where(pg[:, None] >= 0, c.scale["v"][pg], 0) * (127 if c.code == "int8" else 448))[..., None]


KEPT = []  # one workspace (and its arrival counters) for every shape


def run_attention(c, q, a, gate=None, splits=0, kept=False, **mask):
    h = load_host()
    if kept and not KEPT:
        KEPT.append(h.Workspace("cuda"))
    g = gpu_cache(c)
    M, QH, D = q.shape
    o16, o32 = torch.empty((M, QH, D), dtype=torch.float16, device="cuda"), torch.empty((M, QH, D), device="cuda")
    lse = torch.empty((M, QH), device="cuda")
    h.verify_attention_b8(dev(q), g, a, out=o16, out_f32=o32, lse=lse, gate=None if gate is None else dev(gate), splits=splits,
                          workspace=KEPT[0] if kept else None, **mask)
    if kept:
        assert not KEPT[0].words.any()
    return o16.cpu().numpy().astype(np.float64), o32.cpu().numpy().astype(np.float64), lse.cpu().numpy().astype(np.float64)


def check_attention(c, q, a, gate=None, splits=0, start=0, window=0, causal=True):
    M = len(q)
    k, v, here = c.read(0, a + M)
    see = b8.visible(M, a, start, window, causal, here)
    o, lse, mag = b8.attention(q, k, v, see, gate)
    B = b8.attention(q, k, np.broadcast_to(tops(c, a + M), v.shape), see, gate)[2]
    dead = np.isneginf(lse)
    for kept in (False, True):
        o16, o32, l = run_attention(c, q, a, gate, splits, kept, start=start, window=window, causal=causal)
        assert np.all(np.abs(o32 - o) <= bound(o, mag, False, a + M, B)), np.max(np.abs(o32 - o) - bound(o, mag, False, a + M, B))
        assert np.all(np.abs(o16 - o) <= bound(o, mag, True, a + M, B))
        assert np.array_equal(np.isneginf(l), dead) and not o32[dead].any() and not o16[dead].any()
        # a score is off by 2^-18 at most, the logarithm of the sum by a few 2^-24 of its size
        assert np.all(np.abs(l[~dead] - lse[~dead]) <= 2.0 ** -17 + 2.0 ** -21 * np.abs(lse[~dead]))
        if kept:  # whoever adds the splits, the bits are the same
            assert np.array_equal(o32, first[0]) and np.array_equal(l, first[1])
        first = o32, l
    return lse


@pytest.mark.parametrize("code", KINDS)
@pytest.mark.parametrize("QH,KVH,D", [(32, 8, 64), (16, 4, 128), (2, 2, 64), (20, 1, 128)])
@pytest.mark.parametrize("M", [1, 5, 16])
@pytest.mark.parametrize("a", [0, 1, 31, 32, 300])
def test_attention(code, QH, KVH, D, M, a):
    rng = np.random.default_rng(a * 100 + M)
    n = (a + M + 31) // 32
    c = filled(code, a + M, KVH, D, M, table=rng.permutation(n + 2)[:n].astype(np.int32), pages=n + 2)
    q = rng.standard_normal((M, QH, D)).astype(np.float16)
    check_attention(c, q, a, gate=rng.standard_normal((M, QH)).astype(np.float32))


@pytest.mark.parametrize("code", KINDS)
@pytest.mark.parametrize("start,window,causal", [(0, 0, False), (100, 0, True), (0, 17, True), (0, 32, False), (250, 100, True),
                                                 (400, 0, True), (0, 1, True), (290, 5000, False)])
@pytest.mark.parametrize("M,D", [(7, 64), (33, 128)])
def test_attention_masks(code, start, window, causal, M, D):
    rng = np.random.default_rng(start + window + M)
    a = 333
    c = filled(code, a + M, 2, D, 9)
    check_attention(c, rng.standard_normal((M, 6, D)).astype(np.float16), a, start=start, window=window, causal=causal)


@pytest.mark.parametrize("code", KINDS)
@pytest.mark.parametrize("QH,KVH,D,M,a", [(16, 4, 128, 8, 1001), (16, 4, 128, 9, 2000), (16, 4, 128, 12, 2900), (8, 4, 128, 2, 8000),
                                          (32, 8, 64, 16, 2100), (32, 8, 64, 16, 4100), (10, 2, 64, 5, 1500), (2, 1, 64, 1, 9000),
                                          (32, 8, 64, 3, 1020), (16, 4, 128, 3, 760)])
def test_attention_few_pages(code, QH, KVH, D, M, a):
    """One split of up to two pages a wave, and splits of a page a wave that the last of them adds: few and many of them."""
    rng = np.random.default_rng(a)
    c = filled(code, a + M, KVH, D, M, table=rng.permutation((a + M + 31) // 32).astype(np.int32))
    check_attention(c, rng.standard_normal((M, QH, D)).astype(np.float16), a, gate=rng.standard_normal((M, QH)).astype(np.float32))


@pytest.mark.parametrize("splits", [0, 1, 2, 3, 7, 64, 4096])
@pytest.mark.parametrize("M,QH,KVH,D", [(1, 8, 2, 64), (16, 16, 2, 64), (9, 16, 2, 128), (64, 32, 2, 64), (64, 32, 2, 128),
                                        (64, 16, 1, 64), (64, 16, 1, 128), (3, 40, 2, 64), (3, 70, 2, 128)])
def test_attention_splits_and_rows(splits, M, QH, KVH, D):
    """Any number of splits; up to 1024 rows a KV head (16 query heads, 64 tokens)."""
    rng = np.random.default_rng(splits)
    a = 1500
    c = filled("e4m3", a + M, KVH, D, 4)
    check_attention(c, rng.standard_normal((M, QH, D)).astype(np.float16), a, splits=splits)


@pytest.mark.parametrize("code", KINDS)
def test_attention_sizes_far_apart(code):
    """Blocks of V up to 2^30 apart and scores up to +-40: no block's weight is lost from the sum beside larger ones."""
    rng = np.random.default_rng(8)
    M, KVH, D, a = 3, 2, 64, 700
    c = filled(code, a + M, KVH, D, 2)
    c.scale["v"] *= np.exp2(rng.integers(-20, 10, c.scale["v"].shape)).astype(np.float32)
    q = (rng.standard_normal((M, 8, D)) * 6).astype(np.float16)
    check_attention(c, q, a)


@pytest.mark.parametrize("code", KINDS)
def test_attention_blocks_of_zeros(code):
    """Blocks of V (or K) that are all zeros, the first and the last of a cache, single and all: they weigh in the sum."""
    rng = np.random.default_rng(8)
    M, KVH, D, a = 3, 2, 64, 400
    for x in "vk":
        for gone in ([0], [3, 4], list(range(12)), list(range(13))):
            c = filled(code, a + M, KVH, D, 2)
            c.scale[x][gone] = 0
            c.raw[x][gone] = 0
            check_attention(c, rng.standard_normal((M, 8, D)).astype(np.float16), a)


@pytest.mark.parametrize("code", KINDS)
def test_attention_growing_and_falling_scores(code):
    """Scores that climb from page to page (every page moves the running reference) and that fall (none does)."""
    M, KVH, D, a = 2, 1, 64, 32 * 24
    c = filled(code, a + M, KVH, D, 2)
    q = np.full((M, 2, D), 0.5, np.float16)
    one = b8.codes_of(code, np.ones(1), np.ones(1))[0]
    c.raw["k"][:] = one
    for sign in (1, -1):
        c.scale["k"][:] = (np.arange(len(c.scale["k"]))[::sign, None] * 4).astype(np.float32)  # up to 92 * 64 / 2 / 8
        check_attention(c, q, a)


@pytest.mark.parametrize("code", KINDS)
def test_attention_absent_pages(code):
    """Pages that are not there, up to all of them: what is left is attended to, a row that sees nothing gives zeros."""
    rng = np.random.default_rng(1)
    M, KVH, D, a = 5, 2, 64, 300
    q = rng.standard_normal((M, 4, D)).astype(np.float16)
    for gone in ([0], [1, 2, 3], [9], list(range(9)), list(range(10))):
        table = np.arange(10).astype(np.int32)
        c = filled(code, a + M, KVH, D, 3, table=table)
        c.table = table.copy()
        c.table[gone] = [-1, 10, 1 << 30, -(1 << 31)][len(gone) % 4]
        lse = check_attention(c, q, a)
        assert np.isneginf(lse).all() == (len(gone) == 10)


def test_attention_ignores_what_is_masked():
    """Keys behind the block, and the block's own later keys, may hold anything a writer stores: outputs do not change."""
    rng = np.random.default_rng(2)
    M, KVH, D, a = 4, 2, 64, 61
    q = rng.standard_normal((M, 4, D)).astype(np.float16)
    got = []
    for fill in (3, 0x7b):  # the block's last key (position 64, page 2), the slots behind it and the page behind that
        c = b8.Cache("int8", 4, KVH, D)
        c.write(rows(np.random.default_rng(7), a + M, KVH, D), rows(np.random.default_rng(6), a + M, KVH, D), 0)
        for x in "kv":
            c.raw[x][2:] = fill
        got.append(run_attention(c, q, a)[1])
    assert np.array_equal(got[0][:3], got[1][:3]) and not np.array_equal(got[0][3], got[1][3])


def test_attention_query_rows_apart():
    """A NaN query head spoils its own row alone; q inside wider rows; a single token's stride is not read."""
    h = load_host()
    rng = np.random.default_rng(2)
    c = filled("e4m3", 210, 2, 64, 1)
    g = gpu_cache(c)
    q = rng.standard_normal((9, 8, 64)).astype(np.float16)
    wide = torch.zeros((9, 8 * 64 + 40), dtype=torch.float16, device="cuda")
    wide[:, :512] = dev(q).view(9, -1)
    qs = wide[:, :512].unflatten(1, (8, 64))
    want, _ = h.verify_attention_b8(dev(q), g, 200)
    got, _ = h.verify_attention_b8(qs, g, 200)
    assert torch.equal(want, got)
    wide[4, 64:128] = float("nan")
    bad, _ = h.verify_attention_b8(qs, g, 200)
    keep = torch.ones((9, 8), dtype=torch.bool, device="cuda")
    keep[4, 1] = False
    assert torch.equal(bad[keep], want[keep]) and bool(bad[4, 1].isnan().all())
    one, _ = h.verify_attention_b8(qs[2:3], g, 202)
    assert one.shape == (1, 8, 64)


@pytest.mark.parametrize("code,QH,KVH,D,M,a", [("e4m3", 32, 8, 64, 16, 32768), ("int8", 16, 4, 128, 9, 20011)])
def test_attention_long(code, QH, KVH, D, M, a):
    """Long caches against the same attention in float64 on the GPU."""
    h = load_host()
    rng = np.random.default_rng(4)
    n = (a + M + 31) // 32
    c = b8.Cache(code, n, KVH, D, rng.permutation(n).astype(np.int32))
    g = gpu_cache(c)
    kv = torch.randn((2, a + M, KVH, D), device="cuda").half()
    h.kv_write_b8(kv[0], kv[1], g, 0)
    k, v = (x.double().transpose(0, 1) for x in h.kv_read_b8(g, 0, a + M))
    q = torch.randn((M, QH, D), device="cuda").half()
    out, o32, lse = None, torch.empty((M, QH, D), device="cuda"), torch.empty((M, QH), device="cuda")
    h.verify_attention_b8(q, g, a, out_f32=o32, lse=lse)
    x = q.double().view(M, KVH, -1, D).transpose(0, 1).reshape(KVH, -1, D) @ k.transpose(1, 2).contiguous() / D ** 0.5
    x = x.view(KVH, M, -1, a + M)
    p, t = torch.arange(a + M, device="cuda"), torch.arange(M, device="cuda")[:, None]
    x = x.masked_fill((p - a > t)[:, None], -float("inf"))
    want = (torch.softmax(x, -1).view(KVH, -1, a + M) @ v).view(KVH, M, -1, D).transpose(0, 1).reshape(M, QH, D)
    mag = (torch.softmax(x, -1).view(KVH, -1, a + M) @ v.abs()).view(KVH, M, -1, D).transpose(0, 1).reshape(M, QH, D)
    assert bool(((o32 - want).abs() <= (2.0 ** -11 + 2.0 ** -16) * mag).all())
    wl = torch.logsumexp(x, -1).transpose(0, 1).reshape(M, QH)
    assert float((lse - wl).abs().max()) <= 2.0 ** -17 + 2.0 ** -21 * 16


def test_pool_past_4_gib():
    """Pages behind byte 2^32 of a pool: written, read, attended to and evicted from."""
    h = load_host()
    KVH, D, pages = 8, 64, (1 << 32) // (8 * 32 * 64) + 40
    far = np.array([pages - 1, 7, pages - 2, 0, pages - 5], np.int32)
    big = h.b8_cache_alloc(pages, KVH, D, dtype=torch.int8, block_table=dev(far))
    near = b8.Cache("int8", 5, KVH, D)
    g = gpu_cache(near)
    rng = np.random.default_rng(3)
    k, v, q = rows(rng, 150, KVH, D), rows(rng, 150, KVH, D), rng.standard_normal((4, 32, D)).astype(np.float16)
    got = []
    for c in (big, g):
        h.kv_write_b8(dev(k), dev(v), c, 0)
        lse = torch.empty((4, 32), device="cuda")
        o, _ = h.verify_attention_b8(dev(q), c, 146, lse=lse)
        m = h.attention_mass_b8(dev(q), c, 146, lse, torch.zeros((KVH, 160), device="cuda"))
        d = h.b8_cache_alloc(3, KVH, D)
        kept, km = h.kv_evict_b8(c, d, 150, 70, m, sinks=2, recent=4)
        got.append([o, lse, m, kept, km, d.k, d.v, d.k_scale, d.v_scale, *h.kv_read_b8(c, 0, 150)])
    for x, y in zip(*got):
        assert torch.equal(x, y)


# ------------------------------------------------------------------------------------------------ accounts
# Every weight exp(score - lse) is relatively off by the error of its exponent: a score of up to 64 (log2 units) and lse
# rounded and scaled in fp32, 2^-24 64 each, three roundings: 2^-16. Sums of non-negative numbers keep that.
def check_mass(c, q, a, rows_, start=0, window=0, causal=True, with_in=True, alias=False):
    h = load_host()
    g = gpu_cache(c)
    M = len(q)
    k, v, here = c.read(0, a + M)
    see = b8.visible(M, a, start, window, causal, here)
    lse = b8.attention(q, k, v, see)[1].astype(np.float32)
    rng = np.random.default_rng(a)
    m_in = rng.exponential(1.0, (c.KVH, a + M + 5)).astype(np.float32) if with_in else None
    out = dev(m_in) if alias else torch.full((c.KVH, a + M + 5), -3.0, device="cuda")
    word = torch.tensor([rows_], dtype=torch.int32, device="cuda")
    before = out.clone()
    h.attention_mass_b8(dev(q), g, a, dev(lse), out, mass_in=out if alias else None if m_in is None else dev(m_in), rows=word,
                        start=start, window=window, causal=causal)
    n = min(max(rows_, 0), M)
    want = b8.mass(q, k, see, lse, n, a, m_in)
    got = out[:, :a + n].cpu().numpy().astype(np.float64)
    assert np.all(np.abs(got - want) <= 2.0 ** -16 * want + 1e-9), np.max(np.abs(got - want) / (want + 1e-9))
    assert torch.equal(out[:, a + n:], before[:, a + n:])


@pytest.mark.parametrize("code", KINDS)
@pytest.mark.parametrize("QH,KVH,D,M,a", [(32, 8, 64, 16, 300), (16, 4, 128, 9, 1001), (2, 2, 64, 1, 0), (2, 2, 64, 1, 32),
                                          (20, 1, 128, 5, 95), (32, 2, 64, 64, 200)])
def test_mass(code, QH, KVH, D, M, a):
    rng = np.random.default_rng(M)
    c = filled(code, a + M, KVH, D, a, table=rng.permutation((a + M + 31) // 32).astype(np.int32))
    q = rng.standard_normal((M, QH, D)).astype(np.float16)
    check_mass(c, q, a, M)
    check_mass(c, q, a, (M + 1) // 2, with_in=False)
    check_mass(c, q, a, 0, alias=True)
    check_mass(c, q, a, M + 7, alias=True)
    check_mass(c, q, a, -1)


@pytest.mark.parametrize("start,window,causal", [(0, 0, False), (100, 0, True), (0, 17, True), (400, 0, True), (0, 1, True)])
def test_mass_masks(start, window, causal):
    rng = np.random.default_rng(start + window)
    c = filled("int8", 333 + 7, 2, 64, 9)
    check_mass(c, rng.standard_normal((7, 6, 64)).astype(np.float16), 333, 5, start=start, window=window, causal=causal)


def test_mass_absent_pages():
    """Absent pages draw nothing and keep their accounts; rows that saw nothing (lse -inf) add nothing."""
    rng = np.random.default_rng(0)
    for gone in ([2], list(range(11))):
        table = np.arange(11).astype(np.int32)
        c = filled("e4m3", 340, 2, 64, 9, table=table)
        c.table = table.copy()
        c.table[gone] = -1
        check_mass(c, rng.standard_normal((7, 6, 64)).astype(np.float16), 333, 5)


# ------------------------------------------------------------------------------------------------ eviction
def check_evict(c, length, keep, m, sinks, recent, dst_table=None):
    h = load_host()
    g = gpu_cache(c)
    n = (keep + 31) // 32
    d = b8.Cache(c.code, n if dst_table is None else len(dst_table), c.KVH, c.D, dst_table)
    for x in "kv":
        d.raw[x][:] = 9
    gd = gpu_cache(d)
    kept, mass = h.kv_evict_b8(g, gd, length, keep, dev(m), sinks=sinks, recent=recent)
    wk, wm = b8.evict(c, d, length, keep, m, sinks, recent)
    np.testing.assert_array_equal(kept.cpu().numpy(), wk)
    np.testing.assert_array_equal(mass.cpu().numpy(), wm)
    assert_same(gd, d)


@pytest.mark.parametrize("code", KINDS)
@pytest.mark.parametrize("KVH,D", [(8, 64), (3, 128)])
@pytest.mark.parametrize("length,keep,sinks,recent", [(1, 1, 0, 0), (40, 39, 0, 0), (333, 100, 4, 30), (333, 333, 0, 0),
                                                      (333, 333, 100, 233), (1030, 64, 0, 64), (1030, 65, 64, 1),
                                                      (2100, 1025, 7, 0), (5000, 31, 1, 1)])
def test_evict(code, KVH, D, length, keep, sinks, recent):
    rng = np.random.default_rng(length + keep)
    n = (length + 31) // 32
    c = filled(code, length, KVH, D, keep, table=rng.permutation(n).astype(np.int32))
    m = np.exp(2 * rng.standard_normal((KVH, length + 3))).astype(np.float16).astype(np.float32)
    check_evict(c, length, keep, m, sinks, recent, rng.permutation((keep + 31) // 32 + 1).astype(np.int32))


@pytest.mark.parametrize("name", ["equal", "few", "special", "negative", "subnormal", "bits"])
def test_evict_order(name):
    """Ties, infinities, NaN, both zeros, subnormal and negative accounts, and neighbours one bit apart."""
    rng = np.random.default_rng(12)
    KVH, T = 2, 1500
    m = np.ones((KVH, T), np.float32)
    if name == "few":
        m = rng.integers(0, 3, (KVH, T)).astype(np.float32)
    elif name == "special":
        m = rng.choice(np.array([np.nan, np.inf, -np.inf, 0.0, -0.0, 1.0], np.float32), (KVH, T))
        m.view(np.uint32)[:, 5] = 0xFFC00001  # a NaN with its sign bit set
    elif name == "negative":
        m = -rng.exponential(1.0, (KVH, T)).astype(np.float32)
    elif name == "subnormal":
        m = (rng.integers(0, 1 << 22, (KVH, T)).astype(np.uint32)).view(np.float32)
    elif name == "bits":
        m = (np.uint32(0x3F800000) + rng.integers(0, 700, (KVH, T)).astype(np.uint32)).view(np.float32)
    c = filled("int8", T, KVH, 64, 3)
    for keep, sinks, recent in ((700, 3, 40), (1400, 0, 0), (44, 4, 39)):
        check_evict(c, T, keep, m, sinks, recent)


def test_evict_absent_pages():
    """Rows of absent pages are kept as zeros; a destination page that is absent is not written."""
    rng = np.random.default_rng(12)
    table = np.arange(7).astype(np.int32)
    c = filled("e4m3", 200, 2, 64, 3, table=table)
    c.table = table.copy()
    c.table[[1, 4]] = [-1, 99]
    m = rng.exponential(1.0, (2, 200)).astype(np.float32)
    check_evict(c, 200, 130, m, 2, 5, np.array([3, -1, 0, 7, 1], np.int32))


@pytest.mark.parametrize("length,keep", [(16384, 5000), (40000, 39000), (131072, 16384), (300001, 1000)])
def test_evict_long(length, keep):
    """Long accounts, kept positions against a stable sort."""
    h = load_host()
    KVH, D = 2, 64
    g = h.b8_cache_alloc((length + 31) // 32, KVH, D, dtype=torch.float8_e4m3fn)
    d = h.b8_cache_alloc((keep + 31) // 32, KVH, D, dtype=torch.float8_e4m3fn)
    m = torch.randn((KVH, length), device="cuda").mul_(2).exp_().half().float()
    kept, mass = h.kv_evict_b8(g, d, length, keep, m, sinks=4, recent=100)
    for i in range(KVH):
        np.testing.assert_array_equal(kept[i].cpu().numpy(), b8.kept(m[i].cpu().numpy(), length, keep, 4, 100))
    assert torch.equal(mass, m.gather(1, kept.long()))


# ------------------------------------------------------------------------------------------------ together
@pytest.mark.parametrize("code,QH,KVH,D", [("int8", 32, 8, 64), ("e4m3", 16, 4, 128)])
def test_rounds_with_a_bounded_cache(code, QH, KVH, D):
    """Speculative rounds over one layer: append a block, attend, accept some drafts (accept_commit on the device State),
    account for the committed rows alone, and evict whenever the cache passes its limit."""
    h = load_host()
    rng = np.random.default_rng(21)
    M, limit, keep, V = 6, 130, 96, 4096
    pools = [b8.Cache(code, 6, KVH, D, rng.permutation(6).astype(np.int32)) for _ in range(2)]
    dev_pools = [gpu_cache(c) for c in pools]
    acc = [torch.zeros((KVH, 192), device="cuda") for _ in range(2)]
    cur, a = 0, 90
    k, v = rows(rng, a, KVH, D), rows(rng, a, KVH, D)
    pools[0].write(k, v, 0)
    h.kv_write_b8(dev(k), dev(v), dev_pools[0], 0)
    want_acc = np.zeros((KVH, 192))
    ws, seen = h.Workspace("cuda"), torch.zeros(V // 32, dtype=torch.int32, device="cuda")
    evictions = 0
    for r in range(14):
        c, g = pools[cur], dev_pools[cur]
        k, v, q = rows(rng, M, KVH, D), rows(rng, M, KVH, D), rng.standard_normal((M, QH, D)).astype(np.float16)
        c.write(k, v, a)
        h.kv_write_b8(dev(k), dev(v), g, a)
        o32, lse = torch.empty((M, QH, D), device="cuda"), torch.empty((M, QH), device="cuda")
        h.verify_attention_b8(dev(q), g, a, out_f32=o32, lse=lse, workspace=ws)
        kk, vv, here = c.read(0, a + M)
        see = b8.visible(M, a, 0, 0, True, here)
        o, wl, mag = b8.attention(q, kk, vv, see)
        B = b8.attention(q, kk, np.broadcast_to(tops(c, a + M), vv.shape), see)[2]
        assert np.all(np.abs(o32.cpu().numpy() - o) <= bound(o, mag, False, a + M, B))
        # drafts accepted up to a chosen one
        good = int(rng.integers(0, M))
        tokens = rng.integers(0, V, M)
        logits = np.zeros((M, V), np.float32)
        for t in range(M):
            logits[t, (tokens[t + 1] if t < good else (tokens[(t + 1) % M] + 1) % V)] = 5
        st = h.state_tensor(a=a, anchor=int(tokens[0]), tokens=tokens.tolist(), rounds_left=9, budget=500, eos=-1,
                            stop_at=10000, run=1, skip_rounds=1)
        best = h.verify_argmax(dev(logits), seen, st)
        h.accept_commit(st, best, M, torch.zeros(64, dtype=torch.int32, device="cuda"), seen)
        ctx_new = h.STATE_FIELDS.index("ctx_new")
        h.attention_mass_b8(dev(q), g, a, lse, acc[cur], mass_in=acc[cur], rows=st[ctx_new:ctx_new + 1])
        n = good + 1
        want_acc[:, :a + n] = b8.mass(q, kk, see, lse.cpu().numpy(), n, a, want_acc)
        a += n
        got = acc[cur][:, :a].cpu().numpy()
        assert np.all(np.abs(got - want_acc[:, :a]) <= 2.0 ** -15 * want_acc[:, :a] + 1e-9), r
        if a > limit:
            m = acc[cur].cpu().numpy()
            kept, _ = h.kv_evict_b8(g, dev_pools[1 - cur], a, keep, acc[cur], sinks=4, recent=32, mass_out=acc[1 - cur])
            wk, wm = b8.evict(c, pools[1 - cur], a, keep, m, 4, 32)
            np.testing.assert_array_equal(kept.cpu().numpy(), wk)
            cur, a = 1 - cur, keep
            np.testing.assert_array_equal(acc[cur][:, :keep].cpu().numpy(), wm)
            want_acc[:] = 0
            want_acc[:, :keep] = wm
            evictions += 1
    assert evictions >= 1
    n = (a + 31) // 32
    k, v = h.kv_read_b8(dev_pools[cur], 0, a)
    want = pools[cur].read(0, a)
    np.testing.assert_array_equal(k.cpu().numpy(), want[0].astype(np.float32))
    np.testing.assert_array_equal(v.cpu().numpy(), want[1].astype(np.float32))


def test_side_stream_and_repeats():
    """Calls on a stream that is not current (their buffers allocated there), and the same bits every time."""
    h = load_host()
    rng = np.random.default_rng(2)
    c = filled("int8", 2010, 4, 64, 1)
    g = gpu_cache(c)
    q = dev(rng.standard_normal((10, 16, 64)).astype(np.float16))
    lse = torch.empty((10, 16), device="cuda")
    want, _ = h.verify_attention_b8(q, g, 2000, lse=lse)
    want_mass = h.attention_mass_b8(q, g, 2000, lse, torch.zeros((4, 2010), device="cuda"))
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    for _ in range(5):
        got, _ = h.verify_attention_b8(q, g, 2000, stream=side)
        fill = torch.full((1 << 20,), 3.0, device="cuda")  # the current stream keeps allocating meanwhile
        mass = torch.zeros((4, 2010), device="cuda")
        side.wait_stream(torch.cuda.current_stream())
        h.attention_mass_b8(q, g, 2000, lse, mass, stream=side)
        side.synchronize()
        assert torch.equal(got, want) and torch.equal(mass, want_mass) and bool((fill == 3).all())


def test_two_streams_at_once():
    """Calls that overlap, each with its own workspace, caches, accounts and destination."""
    h = load_host()
    rng = np.random.default_rng(9)
    jobs = []
    for i, (QH, KVH, D, M, a) in enumerate([(32, 8, 64, 4, 20000), (16, 4, 128, 9, 17000)]):
        n = (a + M + 31) // 32
        g = h.b8_cache_alloc(n, KVH, D, dtype=TYPES[KINDS[i]])
        kv = torch.randn((2, a + M, KVH, D), device="cuda").half()
        q = torch.randn((M, QH, D), device="cuda").half()

        def run(stream, ws, g=g, kv=kv, q=q, KVH=KVH, D=D, M=M, a=a, kind=KINDS[i]):
            with torch.cuda.stream(stream):
                lse, acc = torch.empty(q.shape[:2], device="cuda"), torch.zeros((KVH, a + M), device="cuda")
                dst = h.b8_cache_alloc(40, KVH, D, dtype=TYPES[kind])
                h.kv_write_b8(kv[0, a:], kv[1, a:], g, a)
                o, _ = h.verify_attention_b8(q, g, a, lse=lse, workspace=ws)
                h.attention_mass_b8(q, g, a, lse, acc, mass_in=acc)
                kept, m = h.kv_evict_b8(g, dst, a + M, 1270, acc, sinks=4, recent=64, workspace=ws)
                return [o, lse, acc, kept, m, dst.k.view(torch.uint8), dst.v.view(torch.uint8), dst.k_scale, dst.v_scale]
        h.kv_write_b8(kv[0], kv[1], g, 0)
        jobs.append(run)
    torch.cuda.synchronize()
    alone = [run(torch.cuda.current_stream(), h.Workspace("cuda")) for run in jobs]
    torch.cuda.synchronize()
    streams, spaces = [torch.cuda.Stream() for _ in jobs], [h.Workspace("cuda") for _ in jobs]
    for _ in range(4):
        both = [[run(s, w) for _ in range(3)][-1] for run, s, w in zip(jobs, streams, spaces)]
        torch.cuda.synchronize()
        for x, y in zip(alone, both):
            for u, v in zip(x, y):
                assert torch.equal(u, v)


def test_graph_replays():
    """The whole chain captured once and replayed with other inputs between eager calls; every replay against eager calls."""
    h = load_host()
    rng = np.random.default_rng(5)
    KVH, D, M, a = 2, 64, 4, 500
    base = filled("e4m3", a, KVH, D, 1)
    g, eager = gpu_cache(base), gpu_cache(base)
    kv = torch.zeros((2, M, KVH, D), dtype=torch.float16, device="cuda")
    q = torch.zeros((M, 8, D), dtype=torch.float16, device="cuda")
    dst, dst_e = h.b8_cache_alloc(8, KVH, D, dtype=torch.float8_e4m3fn), h.b8_cache_alloc(8, KVH, D, dtype=torch.float8_e4m3fn)
    acc, word = torch.zeros((KVH, 512), device="cuda"), torch.tensor([3], dtype=torch.int32, device="cuda")
    out, lse = torch.empty((M, 8, D), dtype=torch.float16, device="cuda"), torch.empty((M, 8), device="cuda")
    kept, mout = torch.empty((KVH, 250), dtype=torch.int32, device="cuda"), torch.empty((KVH, 250), device="cuda")
    ws, ws_e = h.Workspace("cuda"), h.Workspace("cuda")

    def chain(c, d, o, l, m, ws, kept, mout):
        h.kv_write_b8(kv[0], kv[1], c, a)
        h.verify_attention_b8(q, c, a, out=o, lse=l, workspace=ws)
        h.attention_mass_b8(q, c, a, l, m, mass_in=m, rows=word)
        h.kv_evict_b8(c, d, a + 3, 250, m, sinks=2, recent=20, kept=kept, mass_out=mout, workspace=ws)

    chain(g, dst, out, lse, acc, ws, kept, mout)  # sizes the workspace
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        chain(g, dst, out, lse, acc, ws, kept, mout)
    acc.zero_()
    acc_e, out_e, lse_e = torch.zeros_like(acc), torch.empty_like(out), torch.empty_like(lse)
    kept_e, mout_e = torch.empty_like(kept), torch.empty_like(mout)
    for x in ("k", "v", "k_scale", "v_scale"):
        getattr(g, x).view(torch.uint8).copy_(getattr(eager, x).view(torch.uint8))
    for r in range(4):
        kv.copy_(torch.randn(kv.shape, device="cuda"))
        q.copy_(torch.randn(q.shape, device="cuda"))
        graph.replay()
        torch.cuda.synchronize()
        chain(eager, dst_e, out_e, lse_e, acc_e, ws_e, kept_e, mout_e)
        torch.cuda.synchronize()
        for x, y in ((out, out_e), (lse, lse_e), (acc, acc_e), (kept, kept_e), (mout, mout_e), (dst.k_scale, dst_e.k_scale),
                     (dst.v.view(torch.uint8), dst_e.v.view(torch.uint8)), (dst.k.view(torch.uint8), dst_e.k.view(torch.uint8)),
                     (g.k.view(torch.uint8), eager.k.view(torch.uint8))):
            assert torch.equal(x, y), r


def test_workspace_grows_after_a_capture():
    """A graph's workspace stays its own when an eager call makes the Workspace grow past it."""
    h = load_host()
    rng = np.random.default_rng(12)
    c = filled("int8", 9000 + 4, 2, 64, 3)
    g = gpu_cache(c)
    q = dev(rng.standard_normal((4, 8, 64)).astype(np.float16))
    ws = h.Workspace("cuda")
    out, _ = h.verify_attention_b8(q, g, 9000, workspace=ws)
    want, small = out.clone(), ws.buf.numel()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        h.verify_attention_b8(q, g, 9000, out=out, workspace=ws)
    h.verify_attention_b8(q.repeat(8, 1, 1), g, 8900, workspace=ws)
    assert ws.buf.numel() > small
    fill = [torch.full((small,), 7, dtype=torch.uint8, device="cuda") for _ in range(8)]  # would take a freed buffer
    for _ in range(3):
        out.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want) and all(bool((f == 7).all()) for f in fill)


@pytest.mark.parametrize("code", KINDS)
def test_pages_shared_by_readers(code):
    """Logical pages that share a physical one (a prefix read twice) are read like any other."""
    rng = np.random.default_rng(31)
    c = filled(code, 5 * 32, 2, 64, 6)
    c.table = np.array([0, 1, 0, 2, 2, 3, 0, 4], np.int32)
    M, a = 5, 8 * 32 - 5
    q = rng.standard_normal((M, 8, 64)).astype(np.float16)
    check_attention(c, q, a)
    check_mass(c, q, a, 3)
    check_evict(c, 8 * 32, 150, rng.exponential(1.0, (2, 8 * 32)).astype(np.float32), 3, 20)


def test_as_many_heads_as_there_may_be():
    rng = np.random.default_rng(8)
    KVH, D, M, a = 1024, 64, 2, 40
    c = filled("e4m3", a + M, KVH, D, 7)
    q = rng.standard_normal((M, KVH, D)).astype(np.float16)
    check_attention(c, q, a)
    check_mass(c, q, a, 1)
    check_evict(c, a + M, 35, rng.exponential(1.0, (KVH, a + M)).astype(np.float32), 2, 3)


@pytest.mark.parametrize("D", [64, 128])
def test_last_positions(D):
    """Positions up to the last one allowed give what the same rows give at the start of a cache."""
    h = load_host()
    END, M, n, KVH = (1 << 31) - 64, 9, 300, 2
    first = (END - n) // 32 * 32  # position of the rows' first page
    table = torch.full((END // 32,), -1, dtype=torch.int32, device="cuda")
    pages = (END - first) // 32
    table[first // 32:] = torch.arange(pages, dtype=torch.int32, device="cuda").flip(0)
    far, near = (h.b8_cache_alloc(pages, KVH, D, torch.int8, block_table=t) for t in (table, None))
    n = END - first
    kv = torch.randn((2, n, KVH, D), device="cuda").half()
    q = torch.randn((M, 8, D), device="cuda").half()
    got = []
    for c, at in ((far, first), (near, 0)):
        h.kv_write_b8(kv[0, :-M], kv[1, :-M], c, at)
        h.kv_write_b8(kv[0, -M:], kv[1, -M:], c, at + n - M)
        lse = torch.empty((M, 8), device="cuda")
        o, _ = h.verify_attention_b8(q, c, at + n - M, start=at + 3, window=250, lse=lse)
        got.append([o, lse, *h.kv_read_b8(c, at, n)])
    for x, y in zip(*got):
        assert torch.equal(x, y)
    with pytest.raises(h.DsparkError):
        h.kv_write_b8(kv[0], kv[1], far, first + 1)


def test_one_row_and_one_head_of_any_stride():
    """The stride of a dimension of one says nothing: single rows, tokens and heads cut from tensors of odd widths."""
    h = load_host()
    g, w = h.b8_cache_alloc(2, 1, 64), h.b8_cache_alloc(2, 1, 64)
    wide = torch.randn((3, 1, 64 * 3 + 1), device="cuda").half()
    k, v, q = wide[:1, :, :64], wide[:1, :, 64:128], wide[:1, :, 128:192]
    h.kv_write_b8(k, v, g, 0)
    h.kv_write_b8(k.contiguous(), v.contiguous(), w, 0)
    rows = torch.zeros((2, 64 * 2 + 3), device="cuda")
    h.kv_read_b8(g, 0, 1, rows[:1, :64], rows[:1, 64:128])
    for x, y in zip(h.kv_read_b8(w, 0, 1), (rows[0, :64], rows[0, 64:128])):
        assert torch.equal(x.view(-1), y)
    assert bool((rows[1:] == 0).all()) and bool((rows[:, 128:] == 0).all())
    lse = torch.empty((1, 1), device="cuda")
    o, _ = h.verify_attention_b8(q, g, 0, lse=lse)
    assert torch.equal(o, h.verify_attention_b8(q.contiguous(), w, 0)[0])
    acc, start = torch.full((1, 9), -1.0, device="cuda"), torch.ones((1, 5), device="cuda")
    h.attention_mass_b8(q, g, 0, lse, acc, mass_in=start)
    assert abs(float(acc[0, 0]) - 1) < 2.0 ** -15 and bool((acc[0, 1:] == -1).all())
    kept, m = h.kv_evict_b8(g, w, 1, 1, acc)
    assert kept.tolist() == [[0]] and torch.equal(m, acc[:, :1])


@pytest.mark.parametrize("code", KINDS)
@pytest.mark.parametrize("QH,KVH,D,M,a,window", [(8, 2, 64, 9, 300, 0), (16, 4, 128, 8, 300, 0), (16, 1, 64, 16, 200, 0), (8, 2, 64, 5, 600, 200)])
def test_mass_rows_that_draw_nothing(code, QH, KVH, D, M, a, window):
    """Rejected rows and rows of lse -inf draw nothing, whatever their q and lse hold: the accounts are those of zeros there."""
    h = load_host()
    rng = np.random.default_rng(M)
    g = gpu_cache(filled(code, a + M, KVH, D, 7))
    q = rng.standard_normal((M, QH, D)).astype(np.float16)
    lse = torch.empty((M, QH), device="cuda")
    h.verify_attention_b8(dev(q), g, a, window=window, lse=lse)
    n = M - 3
    word = torch.tensor([n], dtype=torch.int32, device="cuda")
    lse[0, 1] = -float("inf")  # a committed row that is to draw nothing

    def accounts(bad_q, bad_lse):
        x, l = q.copy(), lse.clone()
        x[n:], x[0, 1], l[n:] = bad_q, bad_q, bad_lse
        out = torch.full((KVH, a + M), 2.0, device="cuda")
        return h.attention_mass_b8(dev(x), g, a, l, out, mass_in=out, rows=word, window=window)
    want = accounts(0, 0)
    assert bool((want[:, :a + n] > 0).all())
    for bad in (np.nan, np.inf, -np.inf, 65504):
        for l in (0.0, float("nan"), float("inf"), -float("inf")):
            assert torch.equal(accounts(bad, l), want), (bad, l)


@pytest.mark.parametrize("code", KINDS)
@pytest.mark.parametrize("scale", [np.inf, np.nan, 1e-20, 1e30])
def test_absent_pages_have_no_scale(code, scale):
    """No entry points to physical page 0, and whatever it holds changes nothing of what is computed beside absent pages."""
    rng = np.random.default_rng(3)
    M, KVH, D, a = 5, 2, 64, 300
    q = rng.standard_normal((M, 4, D)).astype(np.float16)
    for gone in ([0], [1, 2, 3], [9], list(range(1, 9))):
        c = filled(code, a + M, KVH, D, 3, table=np.arange(1, 11).astype(np.int32), pages=11)
        c.table[gone] = -1
        for x in "kv":
            c.scale[x][0] = scale
        c.scale["v"][c.table[9]], c.raw["v"][c.table[9]] = 0, 0  # (a block of zeros beside them)
        check_attention(c, q, a)
        check_mass(c, q, a, 3)


def test_zeros_before_small_values():
    """Pages of nothing but zeros in V, then small values: the running reference after the former does not lift the latter's
    probabilities out of the half's range. 124 pages a wave, all of whose first 64 are zeros."""
    M, QH, D, waves, pages = 8, 4, 128, 8, 124
    a = waves * pages * 32 - M
    c = b8.Cache("int8", waves * pages, 1, D)
    zero = np.arange(waves * pages) % pages < 64
    c.scale["k"][:], c.scale["v"][:] = 1, np.where(zero, 0, 1.4140625 * 2.0 ** -26)[:, None]
    c.raw["v"][~zero] = 127
    check_attention(c, np.zeros((M, QH, D), np.float16), a, splits=1)


def test_reads_into_one_given_tensor():
    """K or V alone given: it is filled, and the other one created."""
    h = load_host()
    c = filled("int8", 77, 3, 64, 1)
    g, want = gpu_cache(c), c.read(30, 40)
    for i, x in enumerate("kv"):
        for given in (torch.full((40, 3, 64), 7.0, device="cuda"), torch.full((41, 200), 7.0, device="cuda")):
            got = h.kv_read_b8(g, 30, 40, **{x: given})
            assert got[i] is given
            for y, w in zip(got, want):
                y = y[:40, :192] if y.dim() == 2 else y
                np.testing.assert_array_equal(y.reshape(40, 3, 64).cpu().numpy(), w.astype(np.float32))
            assert given.dim() == 3 or (bool((given[40:] == 7).all()) and bool((given[:, 192:] == 7).all()))


def test_accounts_in_the_gaps_of_others():
    """Rows of accounts that lie in turn in one buffer share no byte and are taken; rows that meet are refused."""
    h = load_host()
    rng = np.random.default_rng(3)
    KVH, D, M, a, keep = 3, 64, 4, 300, 70
    n = a + M
    g = gpu_cache(filled("int8", n, KVH, D, 7))
    q, lse = dev(rng.standard_normal((M, 6, D)).astype(np.float16)), torch.empty((M, 6), device="cuda")
    h.verify_attention_b8(q, g, a, lse=lse)
    both = torch.rand((KVH, 2, n + keep), device="cuda")
    start = both[:, 0].clone()
    want = h.attention_mass_b8(q, g, a, lse, torch.zeros_like(start), mass_in=start)
    got = h.attention_mass_b8(q, g, a, lse, both[:, 1], mass_in=both[:, 0])
    assert torch.equal(got[:, :n], want[:, :n]) and torch.equal(both[:, 0], start)
    d = [h.b8_cache_alloc(3, KVH, D) for _ in "ab"]
    kept, m = h.kv_evict_b8(g, d[0], n, keep, want, sinks=2, recent=4)
    kept2, m2 = h.kv_evict_b8(g, d[1], n, keep, both[:, 1, :n], sinks=2, recent=4, mass_out=both[:, 1, n:])
    assert torch.equal(kept, kept2) and torch.equal(m, m2) and torch.equal(d[0].k, d[1].k)
    for mass_in, mass_out in ((both[:, 0], both[:, 0, 4:]), (both[:, 0, keep:], both[:, 0]), (both.view(KVH, -1)[:, n - 1:], both[:, 0])):
        with pytest.raises(h.DsparkError):
            h.attention_mass_b8(q, g, a, lse, mass_out, mass_in=mass_in)
    with pytest.raises(h.DsparkError):
        h.kv_evict_b8(g, d[1], n, keep, both[:, 1, :n], mass_out=both[:, 1, n - 1:n - 1 + keep])


@pytest.mark.parametrize("words", [False, True])
def test_workspace_grows_on_another_stream(words):
    """A buffer that work on the current stream still uses is not handed to its own stream when the workspace outgrows it."""
    h = load_host()
    side, ws = torch.cuda.Stream(), h.Workspace("cuda")
    old = ws.arrivals(1 << 18) if words else ws.get(1 << 20)
    at, size = old.data_ptr(), old.numel()
    x = torch.randn((8192, 8192), device="cuda")
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(4):  # work of some milliseconds that the buffer's last use stands behind
            x = (x @ x).clamp_(-1, 1)
        old.fill_(3)
        del old
        ws.arrivals(2 * size) if words else ws.get(2 * size)
    taken = [torch.empty(size, dtype=torch.int32 if words else torch.uint8, device="cuda") for _ in range(4)]
    busy = not side.query()
    assert busy and all(t.data_ptr() != at for t in taken)
    torch.cuda.synchronize()


@pytest.mark.parametrize("code", KINDS)
@pytest.mark.parametrize("D,M,waves", [(64, 4, 16), (64, 8, 12), (64, 12, 12), (64, 16, 8), (128, 3, 12), (128, 8, 8), (128, 16, 8)])
@pytest.mark.parametrize("extra", [0.4, 40])
def test_attention_many_pages_a_wave(code, D, M, waves, extra):
    """A split of 64 pages a wave, of one more for some of them, and of over 100, with blocks of zeros and absent pages
    anywhere."""
    rng = np.random.default_rng(int(extra) + M)
    pages = int(waves * (64 + extra))
    a, QH = pages * 32 - M - 3, 4
    c = b8.Cache(code, pages, 1, D, rng.permutation(pages).astype(np.int32))
    top = 127 if code == "int8" else 126  # (the largest code as a byte)
    for x in "kv":
        raw = rng.integers(0, top + 1, c.raw[x].shape).astype(np.uint8)
        if code == "int8":
            raw = (raw.astype(np.int8) * rng.choice([-1, 1], raw.shape).astype(np.int8)).view(np.uint8)
        else:
            raw |= rng.choice([0, 128], raw.shape).astype(np.uint8)
        c.raw[x][:] = raw
        c.scale[x][:] = b8.scale_of(code, rng.uniform(0.5, 4, c.scale[x].shape))
        none = rng.random(pages) < 0.15
        c.scale[x][none], c.raw[x][none] = 0, 0
    c.table[rng.random(pages) < 0.1] = -1
    check_attention(c, rng.standard_normal((M, QH, D)).astype(np.float16), a, splits=1)


@pytest.mark.parametrize("code", KINDS)
def test_mass_many_pages_a_wave(code):
    """So many heads that a wave has over 64 pages, against the accounts in float64 on the GPU."""
    h = load_host()
    KVH, D, M, pages = 1024, 64, 2, 270
    a = pages * 32 - 37
    kind = torch.randint(0, 127, (pages, KVH, 32, D), dtype=torch.uint8, device="cuda")
    v = torch.zeros((pages, KVH, 32, D), dtype=torch.uint8, device="cuda")
    scale = torch.rand((pages, KVH), device="cuda").mul_(2).sub_(8).exp2_() / (127 if code == "int8" else 448)
    scale = (scale.view(torch.int32) & ~0xffff).view(torch.float32)  # (8 significant bits: values are exact in fp32)
    table = torch.randperm(pages, device="cuda").int()
    table[[5, 63, 64, 200]] = -1
    c = h.B8Cache(kind.view(TYPES[code]), v.view(TYPES[code]), scale, scale.clone(), table)
    q = torch.randn((M, KVH, D), device="cuda").half()
    lse = torch.empty((M, KVH), device="cuda")
    h.verify_attention_b8(q, c, a, lse=lse)
    start = torch.rand((KVH, a + M), device="cuda")
    got = h.attention_mass_b8(q, c, a, lse, torch.zeros_like(start), mass_in=start)
    p, want = torch.arange(a + M, device="cuda"), torch.where(torch.arange(a + M, device="cuda") < a, start.double(), 0)
    here = (table >= 0)[p // 32]
    k = h.kv_read_b8(c, 0, a + M)[0]
    for t in range(M):
        see = here & (p <= a + t)
        for h0 in range(0, KVH, 128):
            x = (k[:, h0:h0 + 128].double() * q[t, h0:h0 + 128].double()).sum(-1).t() / D ** 0.5
            want[h0:h0 + 128] += torch.where(see, (x - lse[t, h0:h0 + 128, None].double()).exp(), 0)
    assert bool(((got - want).abs() <= 2.0 ** -16 * want + 1e-9).all())


def accounts_of(name, rng, shape):
    m = np.ones(shape, np.float32)
    if name == "few":
        m = rng.integers(0, 3, shape).astype(np.float32)
    elif name == "special":
        m = rng.choice(np.array([np.nan, np.inf, -np.inf, 0.0, -0.0, 1.0], np.float32), shape)
        m.view(np.uint32)[:, 5] = 0xFFC00001  # a NaN with its sign bit set
    elif name == "negative":
        m = -rng.exponential(1.0, shape).astype(np.float32)
    elif name == "subnormal":
        m = rng.integers(0, 1 << 22, shape).astype(np.uint32).view(np.float32)
    elif name == "bits":
        m = (np.uint32(0x3F800000) + rng.integers(0, 700, shape).astype(np.uint32)).view(np.float32)
    return m


def coded(code, T, KVH, D, rng):
    """A cache of random codes and scales."""
    n = (T + 31) // 32
    c = b8.Cache(code, n, KVH, D, rng.permutation(n).astype(np.int32))
    for x in "kv":
        c.raw[x][:] = rng.integers(-127, 128, c.raw[x].shape).astype(np.int8).view(np.uint8)
        if code == "e4m3":
            c.raw[x][c.raw[x] & 127 == 127] = 0
        c.scale[x][:] = b8.scale_of(code, rng.integers(1, 5, c.scale[x].shape).astype(np.float64))
    return c


@pytest.mark.parametrize("name,T", [(x, 40000) for x in ("equal", "few", "special", "negative", "subnormal", "bits")]
                         + [("few", 270011), ("special", 270011)])
def test_evict_order_by_parts(name, T):
    """The accounts of test_evict_order over several workgroups a head, of one tile and of two; the rows moved with them."""
    rng = np.random.default_rng(T)
    c = coded("int8" if T == 40000 else "e4m3", T, 2, 64, rng)
    m = accounts_of(name, rng, (2, T + 1))
    for keep, sinks, recent in ((T // 2, 3, 40), (T - 100, 0, 0), (1044, 4, 39)):
        check_evict(c, T, keep, m, sinks, recent)


@pytest.mark.parametrize("T,sinks,recent", [(40000, 4, 1020), (40000, 0, 33), (17000, 64, 0), (16400, 1, 2), (16384, 5, 7)])
def test_evict_all_but_the_ends(T, sinks, recent):
    """Nothing of the middle is kept, from few positions and from many."""
    rng = np.random.default_rng(recent)
    c = coded("int8", T, 3, 64, rng)
    check_evict(c, T, sinks + recent, accounts_of("few", rng, (3, T)), sinks, recent)


@pytest.mark.parametrize("QH,KVH,M", [(8, 8, 16), (8, 2, 5), (1, 1, 7), (4, 4, 1)])
def test_mass_takes_lse_of_any_strides(QH, KVH, M):
    """Heads before tokens in memory, and cut from wider rows; on the current stream and on another."""
    h = load_host()
    rng = np.random.default_rng(M)
    a, side = 300, torch.cuda.Stream()
    g = gpu_cache(filled("e4m3", a + M, KVH, 64, 7))
    q, lse = dev(rng.standard_normal((M, QH, 64)).astype(np.float16)), torch.empty((M, QH), device="cuda")
    h.verify_attention_b8(q, g, a, lse=lse)
    want = h.attention_mass_b8(q, g, a, lse, torch.zeros((KVH, a + M), device="cuda"))
    wide = torch.zeros((M, 2 * QH + 1), device="cuda")
    wide[:, 1::2] = lse
    for x in (lse.t().contiguous().t(), wide[:, 1::2]):
        assert x.shape == lse.shape and torch.equal(h.attention_mass_b8(q, g, a, x, torch.zeros_like(want)), want)
        got = torch.zeros_like(want)
        torch.cuda.synchronize()
        h.attention_mass_b8(q, g, a, x, got, stream=side)
        side.synchronize()
        assert torch.equal(got, want)
