"""CPU checks of the 8-bit block-scaled cache: what its entry points refuse before any launch (placeholder pointers are never
dereferenced), what the binding refuses, and the restatement's own properties."""
import ctypes

import numpy as np
import pytest

from conftest import load_host
from oracle import b8

EINVAL, ENOSPACE = 1001, 1002


def cache(**kw):
    h = load_host()
    c = h.B8CacheArgs(1 << 20, 2 << 20, 3 << 20, 4 << 20, None, 100, 8, 64, 0)
    for k, v in kw.items():
        setattr(c, k, v)
    return c


def attn(**kw):
    h = load_host()
    a = h.B8AttnArgs(q=16, q_stride=2048, out=1 << 30, workspace=16, workspace_bytes=1 << 40, M=16, QH=32, a=1000, causal=1)
    for k, v in kw.items():
        setattr(a, k, v)
    return a


BAD_CACHE = [dict(k=None), dict(v=None), dict(k_scale=None), dict(v_scale=None), dict(k=(1 << 20) + 8), dict(v=(2 << 20) + 4),
             dict(k_scale=(3 << 20) + 2), dict(block_table=6), dict(kv_pages=0), dict(kv_pages=1 << 31), dict(KVH=0),
             dict(KVH=1025), dict(D=96), dict(D=0), dict(code=2), dict(code=-1)]


@pytest.mark.parametrize("bad", BAD_CACHE)
def test_every_call_checks_the_cache(bad):
    L = load_host().lib()
    c, ok, a = ctypes.byref(cache(**bad)), ctypes.byref(cache()), ctypes.byref(attn())
    assert L.dspark_kv_write_b8(c, 16, 16, 512, 0, 1, None) == EINVAL
    assert L.dspark_kv_read_b8(c, 0, 1, 16, 16, 512, None) == EINVAL
    assert L.dspark_verify_attention_b8(c, a, None) == EINVAL
    assert L.dspark_verify_attention_b8_workspace(c, a) == 0
    assert L.dspark_attention_mass_b8(c, a, 16, None, None, 16, 4096, None) == EINVAL
    for src, dst in ((c, ok), (ok, c)):
        assert L.dspark_kv_evict_b8(src, dst, 64, 32, 0, 0, 16, 64, 1 << 30, 1 << 31, 64, None, 0, None) == EINVAL


def test_writer_and_reader_refuse():
    L = load_host().lib()
    c = ctypes.byref(cache())
    wide = ctypes.byref(cache(block_table=64))
    for args in ((None, 16, 512, 0, 1), (16, None, 512, 0, 1), (8, 16, 512, 0, 1), (16, 8, 512, 0, 1), (16, 16, 504, 0, 1),
                 (16, 16, 516, 0, 1), (16, 16, 512, -1, 1), (16, 16, 512, 0, -1), (16, 16, 512, 3199, 2)):
        assert L.dspark_kv_write_b8(c, *args, None) == EINVAL, args
    for k, v, row, pos0, n in ((None, 16, 512, 0, 1), (16, None, 512, 0, 1), (8, 16, 512, 0, 1), (16, 16, 508, 0, 1),
                               (16, 16, 514, 0, 1), (16, 16, 512, -1, 1), (16, 16, 512, 0, -1), (16, 16, 512, 3199, 2)):
        assert L.dspark_kv_read_b8(c, pos0, n, k, v, row, None) == EINVAL
    # positions past 2^31 - 64, with a table too
    assert L.dspark_kv_write_b8(wide, 16, 16, 512, (1 << 31) - 64, 1, None) == EINVAL
    assert L.dspark_kv_read_b8(wide, (1 << 31) - 64, 1, 16, 16, 512, None) == EINVAL
    # nothing to do: nothing is launched
    assert L.dspark_kv_write_b8(c, None, None, 0, 5, 0, None) == 0
    assert L.dspark_kv_read_b8(c, 5, 0, None, None, 0, None) == 0


BAD_ROWS = [dict(M=0), dict(M=65), dict(QH=4), dict(QH=12), dict(QH=0), dict(a=-1), dict(start=-1), dict(window=-1),
            dict(splits=-1), dict(a=3190), dict(a=(1 << 31) - 70), dict(QH=8 * 17, M=64)]


@pytest.mark.parametrize("bad", BAD_ROWS)
def test_attention_checks_its_shape(bad):
    L = load_host().lib()
    c, a = ctypes.byref(cache()), ctypes.byref(attn(q_stride=1 << 20, **bad))
    assert L.dspark_verify_attention_b8_workspace(c, a) == 0
    assert L.dspark_verify_attention_b8(c, a, None) == EINVAL
    assert L.dspark_attention_mass_b8(c, a, 16, None, None, 16, 1 << 40, None) == EINVAL


def test_attention_checks_its_pointers_and_workspace():
    L = load_host().lib()
    c = ctypes.byref(cache())
    for bad in (dict(q=None), dict(q=8), dict(q_stride=2040), dict(q_stride=2052), dict(out=None), dict(out=8),
                dict(out_f32=8)):
        assert L.dspark_verify_attention_b8(c, ctypes.byref(attn(**bad)), None) == EINVAL, bad
    q = 1 << 22  # outputs over the last and the first byte of q
    for bad in (dict(q=q, out=q + (15 * 2048 + 32 * 64) * 2 - 16), dict(q=q, out=q - 16 * 32 * 64 * 2 + 16),
                dict(q=q, out_f32=q), dict(q=q, out=None, out_f32=q - 16), dict(arrivals=2)):
        assert L.dspark_verify_attention_b8(c, ctypes.byref(attn(**bad)), None) == EINVAL, bad
    need = L.dspark_verify_attention_b8_workspace(c, ctypes.byref(attn()))
    assert need > 0
    for bad in (dict(workspace=None), dict(workspace=8), dict(workspace_bytes=need - 1)):
        assert L.dspark_verify_attention_b8(c, ctypes.byref(attn(**bad)), None) == ENOSPACE, bad
    a, M = 1000, 16
    ok = ctypes.byref(attn())
    for lse, rows, mi, mo, stride in ((None, None, None, 16, 4096), (2, None, None, 16, 4096), (16, 2, None, 16, 4096),
                                      (16, None, 2, 16, 4096), (16, None, None, None, 4096), (16, None, None, 16, a + M - 1),
                                      (16, None, 1 << 20, (1 << 20) + 4, 4096), (16, None, (1 << 20) + 4 * 4096, 1 << 20, 4096)):
        assert L.dspark_attention_mass_b8(c, ok, lse, rows, mi, mo, stride, None) == EINVAL


def test_eviction_refuses():
    L = load_host().lib()
    src, dst = cache(), cache(k=16 << 20, v=32 << 20, k_scale=48 << 20, v_scale=49 << 20)
    mass, kept, out = 64 << 20, 65 << 20, 66 << 20

    def call(s=src, d=dst, length=640, keep=320, sinks=4, recent=32, m=mass, ms=640, k=kept, mo=out, mos=320):
        return L.dspark_kv_evict_b8(ctypes.byref(s), ctypes.byref(d), length, keep, sinks, recent, m, ms, k, mo, mos, None, 0,
                                    None)
    assert call(keep=0, sinks=0, recent=0) == 0
    for bad in (dict(length=-1), dict(keep=-1), dict(keep=641), dict(sinks=-1), dict(recent=-1), dict(sinks=300, recent=21),
                dict(sinks=(1 << 31) - 1, recent=(1 << 31) - 1), dict(length=3201), dict(m=None), dict(k=None), dict(mo=None),
                dict(ms=639), dict(mos=319)):
        assert call(**bad) == EINVAL, bad
    for d in (cache(k=16 << 20, v=32 << 20, k_scale=48 << 20, v_scale=49 << 20, **x)
              for x in (dict(KVH=4), dict(D=128), dict(code=1))):
        assert call(d=d) == EINVAL
    # nothing that is written may be read: the same pools, K beside V, accounts inside the destination, kept over mass
    assert call(d=src) == EINVAL
    assert call(d=cache(k=2 << 20, v=32 << 20, k_scale=48 << 20, v_scale=49 << 20)) == EINVAL
    assert call(m=(16 << 20) + 100 * 8 * 32 * 64 - 4) == EINVAL
    assert call(k=mass + 4) == EINVAL and call(mo=mass) == EINVAL
    assert call(mo=kept) == EINVAL and call(k=16 << 20) == EINVAL
    assert call(d=cache(k=16 << 20, v=(16 << 20) + 64, k_scale=48 << 20, v_scale=49 << 20)) == EINVAL
    assert call(d=cache(k=16 << 20, v=32 << 20, k_scale=48 << 20, v_scale=49 << 20, block_table=kept)) == EINVAL
    # a selection by parts has a workspace
    big = dict(s=cache(block_table=1 << 10), length=100000, ms=100000)
    need = L.dspark_kv_evict_b8_workspace(8, 100000)
    assert need > 0 and L.dspark_kv_evict_b8_workspace(8, 8000) == 0 and L.dspark_kv_evict_b8_workspace(0, 100000) == 0
    assert call(**big) == ENOSPACE
    assert call(length=(1 << 30) + 1, ms=1 << 40, s=cache(block_table=1 << 10)) == EINVAL


def test_the_binding_refuses_on_the_host():
    import torch
    h = load_host()
    k = torch.zeros((4, 2, 32, 64), dtype=torch.int8)
    s = torch.zeros((4, 2))
    c = h.B8Cache(k, k.clone(), s, s.clone(), torch.arange(3, dtype=torch.int32))
    for bad in ((k[:, :, :16], k[:, :, :16], s, s), (k, k.float(), s, s), (k.half(), k.half(), s, s), (k, k, s[:2], s),
                (k, k, s.double(), s), (k, k, s, s, torch.arange(4)), (k.transpose(0, 1), k.transpose(0, 1), s.t(), s.t()),
                (k, k[:3], s, s)):
        with pytest.raises(h.DsparkError):
            h.B8Cache(*bad)
    row = torch.zeros((40, 2, 64), dtype=torch.float16)
    q = torch.zeros((4, 8, 64), dtype=torch.float16)
    acc = torch.zeros((2, 96))
    for call in (lambda: h.kv_write_b8(row, row, c, 60),                       # past the table's 3 pages
                 lambda: h.kv_write_b8(row.float(), row.float(), c, 0), lambda: h.kv_write_b8(row, row[:8], c, 0),
                 lambda: h.kv_write_b8(row[:, :1], row[:, :1], c, 0), lambda: h.kv_write_b8(row[..., ::2], row[..., ::2], c, 0),
                 lambda: h.kv_read_b8(c, 90, 7), lambda: h.verify_attention_b8(q, c, 93),
                 lambda: h.verify_attention_b8(q[..., :32], c, 0), lambda: h.verify_attention_b8(q.float(), c, 0),
                 lambda: h.attention_mass_b8(q, c, 93, acc, acc), lambda: h.attention_mass_b8(q, c, 0, acc, acc),
                 lambda: h.attention_mass_b8(q, c, 30, torch.zeros((4, 8)), acc[:, :33]),
                 lambda: h.kv_evict_b8(c, c, 97, 3, acc), lambda: h.kv_evict_b8(c, c, 96, 3, acc[:, :95])):
        with pytest.raises(h.DsparkError):
            call()


@pytest.mark.parametrize("code", ["int8", "e4m3"])
def test_scales_and_codes_of_the_restatement(code):
    """A scale takes its block to the code range and no further than need be; codes are the nearest values; code * scale is
    exact in fp32."""
    every = np.arange(0x7c00, dtype=np.uint16).view(np.float16).astype(np.float64)  # every non-negative finite half
    s = b8.scale_of(code, every).astype(np.float64)
    top = 127 if code == "int8" else 448
    assert s[0] == 0 and np.all(every <= s * top * (1 + 2.0 ** -23))
    assert np.all(every[1:] > s[1:] * top * (1 - 2.0 ** -15 if code == "int8" else 0.5))
    vals = np.unique(b8.values(code, np.arange(256, dtype=np.uint8)))
    vals = vals[np.isfinite(vals)]
    prod = vals[None] * s[::97, None]
    assert np.array_equal(prod.astype(np.float32).astype(np.float64), prod)
    x = np.random.default_rng(0).uniform(-1, 1, 4000) * top * 0.37
    got = b8.values(code, b8.codes_of(code, x, np.float64(0.37))) * 0.37
    inside = vals if code == "e4m3" else vals[vals >= -127]
    best = np.abs(x[:, None] - inside[None] * 0.37).min(1)
    assert np.allclose(np.abs(got - x), best, rtol=0, atol=1e-12)
    assert np.array_equal(b8.codes_of("int8", np.array([0.5, 1.5, -0.5, 2.5, np.nan, np.inf]), 1.0).view(np.int8), [0, 2, 0, 2, 0, 127])


def test_calls_refuse_memory_that_meets():
    """Every output against every input and the other outputs, by a word at either end."""
    L = load_host().lib()
    MB = 1 << 20
    pools = dict(k=16 * MB, v=32 * MB, k_scale=48 * MB, v_scale=49 * MB, block_table=50 * MB)
    codes, scales, table = 100 * 8 * 32 * 64, 100 * 8 * 4, 32 * 4
    c = ctypes.byref(cache(**pools))
    held = [(16 * MB, codes), (32 * MB, codes), (48 * MB, scales), (49 * MB, scales)]

    def over(spans, n):  # outputs of n bytes that reach a span's last and its first byte, on 16-byte boundaries
        return [x for at, size in spans for x in ((at + size - 1) // 16 * 16, (at - n) // 16 * 16 + 16)]

    # append: rows of 512 halves 600 apart, 10 of them; the table inside a pool
    n = (9 * 600 + 512) * 2
    for at in over(held, n):
        assert L.dspark_kv_write_b8(c, at, 60 * MB, 600, 990, 10, None) == EINVAL
        assert L.dspark_kv_write_b8(c, 60 * MB, at, 600, 990, 10, None) == EINVAL
    for at in (16 * MB + codes - 4, 16 * MB - table + 4):
        bad = ctypes.byref(cache(**{**pools, "block_table": at}))
        assert L.dspark_kv_write_b8(bad, 60 * MB, 61 * MB, 600, 990, 10, None) == EINVAL
    for bad in (dict(v=16 * MB + 64), dict(v=16 * MB), dict(v_scale=48 * MB), dict(k_scale=32 * MB + 64)):
        assert L.dspark_kv_write_b8(ctypes.byref(cache(**{**pools, **bad})), 60 * MB, 61 * MB, 600, 990, 10, None) == EINVAL
    # read back: rows of 512 words 1024 apart; k and v in each other's rows
    n = (9 * 1024 + 512) * 4
    for at in over(held + [(50 * MB, table)], n):
        assert L.dspark_kv_read_b8(c, 990, 10, at, 60 * MB, 1024, None) == EINVAL
        assert L.dspark_kv_read_b8(c, 990, 10, 60 * MB, at, 1024, None) == EINVAL
    for d in (0, 16, 2048 - 16, 4096 * 9, 4096 * 9 + 2032, 4096 - 2032, 4096 * 8 + 2064):
        assert L.dspark_kv_read_b8(c, 990, 10, 60 * MB, 60 * MB + d, 1024, None) == EINVAL
        assert L.dspark_kv_read_b8(c, 990, 10, 60 * MB + d, 60 * MB, 1024, None) == EINVAL
    # attention
    base = dict(q=60 * MB, out=61 * MB, out_f32=62 * MB, lse=63 * MB, gate=64 * MB, workspace=128 * MB, arrivals=65 * MB)
    out, heads, words = 16 * 2048, 16 * 32 * 4, 8 * 64 * 4
    need = L.dspark_verify_attention_b8_workspace(c, ctypes.byref(attn(**base)))
    reads = held + [(50 * MB, table), (60 * MB, 2 * out), (64 * MB, heads)]
    sizes = dict(out=2 * out, out_f32=4 * out, lse=heads, workspace=need, arrivals=words)
    for name, size in sizes.items():
        others = [(base[x], s) for x, s in sizes.items() if x != name]
        for at in over(reads + others, size):
            assert L.dspark_verify_attention_b8(c, ctypes.byref(attn(**{**base, name: at})), None) == EINVAL, (name, at)
    # accounts
    ok = ctypes.byref(attn(**base))
    bytes_ = (7 * 1100 + 1016) * 4
    for at in over([held[0], held[2], (50 * MB, table), (60 * MB, 2 * out), (63 * MB, heads), (70 * MB, 4), (80 * MB, bytes_)], bytes_):
        assert L.dspark_attention_mass_b8(c, ok, 63 * MB, 70 * MB, 80 * MB, at, 1100, None) == EINVAL, at


def test_attention_checks_the_alignment_of_lse_and_gate():
    L = load_host().lib()
    MB = 1 << 20
    c = ctypes.byref(cache(k=16 * MB, v=32 * MB, k_scale=48 * MB, v_scale=49 * MB))
    for bad in (dict(lse=63 * MB + 2), dict(lse=63 * MB + 1), dict(gate=64 * MB + 2), dict(gate=64 * MB + 3)):
        a = attn(**{**dict(q=60 * MB, out=61 * MB, lse=63 * MB, gate=64 * MB, workspace=128 * MB), **bad})
        assert L.dspark_verify_attention_b8(c, ctypes.byref(a), None) == EINVAL, bad


@pytest.mark.parametrize("far", [1 << 31, 1 << 32, (1 << 32) + 3, -1, -(1 << 32)])
def test_the_binding_refuses_positions_past_32_bits(far):
    """ctypes would hand over their low 32 bits, a position or count somewhere else."""
    import torch
    h = load_host()
    c, d = (h.b8_cache_alloc(4, 2, 64, device="cpu") for _ in "cd")
    row, q = torch.zeros((4, 2, 64), dtype=torch.float16), torch.zeros((4, 8, 64), dtype=torch.float16)
    lse, acc = torch.zeros((4, 8)), torch.zeros((2, 128))
    for call in (lambda: h.kv_write_b8(row, row, c, far), lambda: h.kv_read_b8(c, far, 4), lambda: h.kv_read_b8(c, 0, far),
                 lambda: h.verify_attention_b8(q, c, far), lambda: h.verify_attention_b8(q, c, 9, start=far),
                 lambda: h.verify_attention_b8(q, c, 9, window=far), lambda: h.verify_attention_b8(q, c, 9, splits=far),
                 lambda: h.attention_mass_b8(q, c, far, lse, acc), lambda: h.attention_mass_b8(q, c, 9, lse, acc, start=far),
                 lambda: h.attention_mass_b8(q, c, 9, lse, acc, window=far), lambda: h.kv_evict_b8(c, d, far, 5, acc),
                 lambda: h.kv_evict_b8(c, d, 90, far, acc), lambda: h.kv_evict_b8(c, d, 90, 5, acc, sinks=far),
                 lambda: h.kv_evict_b8(c, d, 90, 5, acc, recent=far)):
        with pytest.raises(h.DsparkError, match="counts and positions"):
            call()


def test_each_refusal_stands_alone():
    """Arguments that are refused for one reason, beside ones that nothing is wrong with (no memory meets other memory there)."""
    import torch
    L = load_host().lib()
    MB = 1 << 20
    c = ctypes.byref(cache(k=16 * MB, v=32 * MB, k_scale=48 * MB, v_scale=49 * MB))
    base = dict(q=60 * MB, out=61 * MB, out_f32=62 * MB, lse=63 * MB, gate=64 * MB, workspace=128 * MB, arrivals=65 * MB)

    def attend(**bad):
        return L.dspark_verify_attention_b8(c, ctypes.byref(attn(**{**base, **bad})), None)

    def mass(lse=63 * MB, rows=70 * MB, mi=80 * MB, mo=90 * MB, stride=1100):
        return L.dspark_attention_mass_b8(c, ctypes.byref(attn(**base)), lse, rows, mi, mo, stride, None)

    def write(k=60 * MB, v=61 * MB, row=600, pos0=990, n=10):
        return L.dspark_kv_write_b8(c, k, v, row, pos0, n, None)

    def read(k=60 * MB, v=61 * MB, row=600, pos0=990, n=10):
        return L.dspark_kv_read_b8(c, pos0, n, k, v, row, None)
    need = L.dspark_verify_attention_b8_workspace(c, ctypes.byref(attn(**base)))
    for bad in (dict(q=None), dict(q=60 * MB + 8), dict(q_stride=2040), dict(q_stride=2052), dict(out=None, out_f32=None),
                dict(out=61 * MB + 8), dict(out_f32=62 * MB + 8), dict(arrivals=65 * MB + 2), dict(M=0), dict(M=65), dict(QH=12),
                dict(a=-1), dict(a=3190), dict(start=-1), dict(window=-1), dict(splits=-1)):
        assert attend(**bad) == EINVAL, bad
    for bad in (dict(workspace=None), dict(workspace=128 * MB + 8), dict(workspace_bytes=need - 1)):
        assert attend(**bad) == ENOSPACE, bad
    for bad in (dict(lse=None), dict(lse=63 * MB + 2), dict(rows=70 * MB + 2), dict(mi=80 * MB + 2), dict(mo=None), dict(mo=90 * MB + 2),
                dict(stride=1015)):
        assert mass(**bad) == EINVAL, bad
    for bad in (dict(k=None), dict(v=None), dict(k=60 * MB + 8), dict(v=61 * MB + 8), dict(row=504), dict(pos0=-1), dict(n=-1),
                dict(pos0=3191)):
        assert write(**bad) == EINVAL and read(**bad) == EINVAL, bad
    assert write(row=516) == EINVAL and read(row=514) == EINVAL
    if not torch.cuda.is_available():  # (the launch itself fails here)
        assert not {0, EINVAL, ENOSPACE} & {attend(), mass(), mass(rows=None), mass(mi=None), mass(mi=90 * MB), write(), read()}


def test_no_launch_past_what_a_grid_holds():
    """A wave of 64 threads for each page, K or V, and head: under 2^32 threads. Sparse tables reach it with little memory."""
    L = load_host().lib()
    MB, GB = 1 << 20, 1 << 30
    for KVH, page in ((1, 1 << 25), (2, 1 << 24), (8, 1 << 22), (1024, 1 << 15), (1, (1 << 25) - 1)):
        n = 32 * page
        src = cache(k=16 * MB, v=32 * MB, k_scale=48 * MB, v_scale=49 * MB, block_table=GB, KVH=KVH, kv_pages=1)
        dst = cache(k=17 * MB, v=33 * MB, k_scale=50 * MB, v_scale=51 * MB, block_table=2 * GB, KVH=KVH, kv_pages=1)
        far = 1 << 50
        assert L.dspark_kv_evict_b8(ctypes.byref(src), ctypes.byref(dst), n, n, 0, 0, far, n, 2 * far, 3 * far, n, 4 * far, far, None) == EINVAL
        assert L.dspark_kv_write_b8(ctypes.byref(src), far, 2 * far, 64 * KVH, 0, n, None) == EINVAL
        assert L.dspark_kv_read_b8(ctypes.byref(src), 0, n, far, 2 * far, 64 * KVH, None) == EINVAL
