"""CPU checks of the operators for a batch of sequences: what their entry points refuse before any launch (placeholder pointers are
never dereferenced), what the binding refuses, the frequencies, and the restatement's own properties."""
import ctypes
import math

import numpy as np
import pytest

from conftest import load_host
from oracle import batch

EINVAL, ENOSPACE = 1001, 1002
M = 1 << 20


def rope_args(**kw):
    h = load_host()
    a = h.RopeArgs(q=1 * M, q_out=2 * M, k=3 * M, k_out=4 * M, q_stride=2048, q_out_stride=2048, k_stride=512, k_out_stride=512,
                   positions=5 * M, freq=6 * M, scale=1.0, n=16, QH=32, KVH=8, D=64, rot=64)
    for k, v in kw.items():
        setattr(a, k, v)
    return ctypes.byref(a)


def append_args(**kw):
    return rope_args(**{**dict(k_out=None, v=7 * M, v_stride=512, k_pages=64 * M, v_pages=128 * M, slots=8 * M, kv_pages=100), **kw})


def shared_args(**kw):
    h = load_host()
    a = h.SharedAttnArgs(q=1 * M, q_stride=2048, k_pages=1 << 32, v_pages=1 << 33, kv_pages=1000, prefix_table=2 * M, q_start=3 * M,
                         own_len=4 * M, own_table=5 * M, own_stride=10, out=6 * M, workspace=1 << 40, workspace_bytes=1 << 36,
                         prefix=1000, tokens=16, seqs=4, max_tokens=4, own_pages=10, QH=32, KVH=8, D=64, causal=1)
    for k, v in kw.items():
        setattr(a, k, v)
    return ctypes.byref(a)


def sample_args(**kw):
    h = load_host()
    a = h.SampleArgs(logits=64 * M, row_stride=1000, u=1 * M, tokens=2 * M, workspace=1 << 40, workspace_bytes=1 << 36, temperature_all=1,
                     top_p_all=1, n=8, V=1000, type=2)
    for k, v in kw.items():
        setattr(a, k, v)
    return ctypes.byref(a)


@pytest.mark.parametrize("bad", [dict(n=-1), dict(n=1 << 30), dict(QH=-1), dict(KVH=-1), dict(QH=1025), dict(KVH=1025), dict(QH=0, KVH=0),
                                 dict(D=63), dict(D=0), dict(D=1026), dict(rot=0), dict(rot=63), dict(rot=66), dict(type=3), dict(type=-1),
                                 dict(q=None), dict(q_out=None), dict(k=None), dict(k_out=None), dict(positions=None),
                                 dict(positions=5 * M + 2), dict(freq=None), dict(freq=6 * M + 4), dict(q=M + 1), dict(type=2, q=M + 2),
                                 dict(q_stride=2047), dict(q_out_stride=2047), dict(k_stride=511), dict(k_out_stride=511),
                                 dict(q_stride=1 << 30), dict(k_out_stride=1 << 30),
                                 dict(q_out=M + 2), dict(q_out=M, q_out_stride=2056), dict(q_out=3 * M), dict(k_out=2 * M),
                                 dict(k_out=5 * M), dict(q_out=6 * M), dict(q_out=3 * M - 2 * 2048 * 16 + 2)])
def test_rope_refuses(bad):
    assert load_host().lib().dspark_rope(rope_args(**bad), None) == EINVAL


@pytest.mark.parametrize("bad", [dict(k_out=4 * M), dict(type=1), dict(type=2), dict(inverse=1), dict(D=32, rot=32), dict(KVH=0, k=None),
                                 dict(v=None), dict(v=7 * M + 1), dict(v_stride=511), dict(v_stride=1 << 30), dict(slots=None),
                                 dict(slots=8 * M + 4), dict(k_pages=None), dict(v_pages=None), dict(k_pages=64 * M + 8),
                                 dict(v_pages=128 * M + 8), dict(kv_pages=0), dict(kv_pages=1 << 31), dict(v_pages=64 * M + 16),
                                 dict(q=64 * M), dict(v=128 * M + 2048), dict(slots=64 * M), dict(q_out=128 * M)])
def test_rope_append_refuses(bad):
    assert load_host().lib().dspark_rope(append_args(**bad), None) == EINVAL


def test_rope_refuses_launches_past_what_a_grid_holds():
    """Buffers far apart, so that nothing else is wrong with them."""
    L, far = load_host().lib(), {k: i << 44 for i, k in enumerate(("q", "q_out", "k", "k_out", "positions", "freq"), 1)}
    assert L.dspark_rope(rope_args(n=1 << 23, **far), None) == EINVAL
    far.update(k_out=None, v=7 << 44, slots=8 << 44, k_pages=9 << 44, v_pages=10 << 44)
    assert L.dspark_rope(append_args(n=1 << 20, KVH=128, k_stride=1 << 14, v_stride=1 << 14, kv_pages=1 << 20, **far), None) == EINVAL


def test_rope_of_nothing():
    L = load_host().lib()
    assert L.dspark_rope(None, None) == EINVAL
    assert L.dspark_rope(rope_args(n=0, q=None, positions=None), None) == 0
    assert L.dspark_rope(append_args(n=0), None) == 0


@pytest.mark.parametrize("rot", [2, 4, 64, 128, 6])
@pytest.mark.parametrize("scaling", [None, "linear", "base", "ramp"])
def test_rope_freqs(rot, scaling):
    for base, factor, trained, low, high in ((1e4, 1.0, 8192.0, 1.0, 32.0), (1e6, 16.0, 4096.0, 1.0, 32.0), (5e5, 3.5, 100.0, 0.0, 4.0)):
        got, scale = load_host().rope_freqs(rot, base, scaling, factor, trained, low, high)
        want, s = batch.rope_freqs(rot, base, scaling, factor, trained, low, high)
        np.testing.assert_allclose(got, want, rtol=1e-13)  # (pow to some units of 2^-53, the ramp's difference of turns)
        assert abs(scale - s) < 1e-14
        if scaling == "base" and rot > 2:  # the slowest pair turns 1 / factor as fast, the first as before
            np.testing.assert_allclose([got[0], got[-1]], [1.0, base ** (-(rot - 2) / rot) / factor], rtol=1e-13)


def test_rope_freqs_refuses():
    h = load_host()
    L, out = h.lib(), (ctypes.c_double * 64)()
    ok = (64, 1e4, 3, 2.0, 100.0, 1.0, 32.0)
    assert L.dspark_rope_freqs(*ok, out, None) == 0
    for i, bad in ((0, 0), (0, 63), (1, 0.0), (1, -1.0), (1, math.nan), (1, math.inf), (2, 4), (2, -1), (3, 0.5), (3, math.nan), (3, math.inf),
                   (4, 0.0), (4, math.nan), (5, -1.0), (6, 1.0), (6, math.nan)):
        assert L.dspark_rope_freqs(*ok[:i], bad, *ok[i + 1:], out, None) == EINVAL, (i, bad)
    assert L.dspark_rope_freqs(*ok, None, None) == EINVAL
    for bad in (("other", {}), ("ramp", {})):
        with pytest.raises(h.DsparkError):
            h.rope_freqs(64, 1e4, bad[0])


@pytest.mark.parametrize("bad", [dict(D=96), dict(KVH=0), dict(KVH=1025, QH=1025), dict(QH=4), dict(QH=33), dict(QH=4104, KVH=8),
                                 dict(prefix=-1), dict(prefix=1 << 30), dict(tokens=-1), dict(seqs=-1), dict(seqs=(1 << 20) + 1),
                                 dict(max_tokens=0), dict(max_tokens=17), dict(tokens=(1 << 18) + 1, max_tokens=4), dict(own_pages=-1),
                                 dict(own_pages=(1 << 24) + 1, own_stride=1 << 25), dict(own_pages=11), dict(own_stride=1 << 30),
                                 dict(kv_pages=0), dict(kv_pages=1 << 31), dict(prefix_table=None, prefix=32001),
                                 dict(window=-1), dict(splits=-1), dict(q_stride=2040), dict(q_stride=1 << 30),
                                 dict(seqs=1 << 20, tokens=1 << 18, max_tokens=1 << 18)])
def test_shared_refuses_shapes(bad):
    L = load_host().lib()
    assert L.dspark_verify_attention_shared(shared_args(**bad), None) == EINVAL
    assert L.dspark_verify_attention_shared_workspace(shared_args(**bad)) == 0


@pytest.mark.parametrize("bad", [dict(q=None), dict(q=M + 8), dict(q_stride=2052), dict(k_pages=None), dict(v_pages=None),
                                 dict(k_pages=(1 << 32) + 8), dict(v_pages=(1 << 33) + 8), dict(q_start=None), dict(q_start=3 * M + 2),
                                 dict(own_len=None), dict(own_table=None), dict(own_table=5 * M + 1), dict(prefix_table=2 * M + 2),
                                 dict(out=None), dict(out=6 * M + 8), dict(out_f32=7 * M + 8), dict(lse=7 * M + 2), dict(gate=7 * M + 1),
                                 dict(out=M), dict(out=1 << 32), dict(out=2 * M), dict(out=3 * M), dict(out=4 * M), dict(out=5 * M),
                                 dict(lse=6 * M), dict(gate=6 * M), dict(out_f32=6 * M), dict(workspace=1 << 33), dict(workspace=6 * M)])
def test_shared_refuses_pointers(bad):
    assert load_host().lib().dspark_verify_attention_shared(shared_args(**bad), None) == EINVAL


def test_shared_workspace_and_nothing():
    L = load_host().lib()
    need = L.dspark_verify_attention_shared_workspace(shared_args())
    assert need >= 16 * 32 * (64 + 2) * 4
    for bad in (dict(workspace=None), dict(workspace=(1 << 40) + 8), dict(workspace_bytes=need - 1)):
        assert L.dspark_verify_attention_shared(shared_args(**bad), None) == ENOSPACE
    assert L.dspark_verify_attention_shared(None, None) == EINVAL
    for none in (dict(tokens=0, max_tokens=0), dict(seqs=0)):
        assert L.dspark_verify_attention_shared(shared_args(**none), None) == 0
        assert L.dspark_verify_attention_shared_workspace(shared_args(**none)) == 256


@pytest.mark.parametrize("bad", [dict(n=-1), dict(n=65536), dict(V=0), dict(V=(1 << 20) + 1, row_stride=1 << 21), dict(type=3), dict(type=-1),
                                 dict(logits=None), dict(logits=64 * M + 2), dict(row_stride=999), dict(row_stride=1 << 30), dict(u=None),
                                 dict(u=M + 2), dict(tokens=None), dict(tokens=2 * M + 2), dict(keys=3 * M + 4), dict(kept=3 * M + 1),
                                 dict(logprob=3 * M + 2), dict(temperature=3 * M + 2), dict(top_k=3 * M + 2), dict(top_p=3 * M + 2),
                                 dict(min_p=3 * M + 2), dict(tokens=64 * M + 400), dict(kept=2 * M + 4), dict(keys=2 * M), dict(tokens=M),
                                 dict(logprob=3 * M, top_p=3 * M), dict(workspace=64 * M), dict(workspace=2 * M)])
def test_sample_refuses(bad):
    assert load_host().lib().dspark_verify_sample(sample_args(**bad), None) == EINVAL


def test_sample_workspace_and_nothing():
    L = load_host().lib()
    need = L.dspark_verify_sample_workspace(8, 1000)
    assert need > 0 and L.dspark_verify_sample_workspace(0, 1) > 0
    for bad in ((-1, 10), (65536, 10), (1, 0), (1, (1 << 20) + 1)):
        assert L.dspark_verify_sample_workspace(*bad) == 0
    for bad in (dict(workspace=None), dict(workspace=(1 << 40) + 8), dict(workspace_bytes=need - 1)):
        assert L.dspark_verify_sample(sample_args(**bad), None) == ENOSPACE
    assert L.dspark_verify_sample(None, None) == EINVAL
    assert L.dspark_verify_sample(sample_args(n=0, logits=None), None) == 0


def test_rows_of_one_stride_that_meet():
    """A shared byte is found whichever rows it lies in. (Rows in the gaps of others: the GPU tests.)"""
    L = load_host().lib()
    row = dict(n=7, QH=2, KVH=2, D=4, rot=4, q_stride=100, q_out_stride=100, k_stride=100, k_out_stride=100, q=M)
    base = dict(q_out=2 * M, k=8 * M, k_out=16 * M)
    for first, second in (("q_out", "k"), ("k_out", "q_out")):
        for off in range(-900, 900):  # in elements of two bytes; rows are 8 of every 100, seven of them
            if any(abs(off + 100 * d) < 8 for d in range(-6, 7)):
                at = {**base, first: 32 * M, second: 32 * M + 2 * off}
                assert L.dspark_rope(rope_args(**row, **at), None) == EINVAL, (first, off)


# ---------------------------------------------------------------- the restatement
def test_oracle_rope():
    rng = np.random.default_rng(0)
    x, pos = rng.standard_normal((5, 3, 10)), np.array([0, 1, -7, 100000, 3])
    f, _ = batch.rope_freqs(6, 1e4)
    for il in (False, True):
        y = batch.rope(x, pos, f, il)
        np.testing.assert_allclose(batch.rope(y, pos, f, il, inverse=True), x, atol=1e-12)
        np.testing.assert_array_equal(y[..., 6:], x[..., 6:])
        i, j = (0, 1) if il else (0, 3)  # the first pair: a complex number turned by p radians
        z = (x[..., i] + 1j * x[..., j]) * np.exp(1j * pos)[:, None]
        np.testing.assert_allclose(y[..., i] + 1j * y[..., j], z, atol=1e-9)


def test_oracle_shared_attention():
    """Against one softmax over a sequence's whole row of keys, and its masks by hand."""
    rng = np.random.default_rng(1)
    pk, pv = rng.standard_normal((2, 5, 2, 4))
    own = [(*rng.standard_normal((2, n, 2, 4)), np.ones(n)) for n in (3, 1)]
    q, start = rng.standard_normal((4, 4, 4)), [0, 3, 4]
    out, lse, _ = batch.shared_attention(q, pk, pv, np.ones(5), start, own, 3)
    for t, r, n in ((0, 0, 1), (1, 0, 2), (2, 0, 3), (3, 1, 1)):
        for h in range(4):
            k, v = np.concatenate([pk, own[r][0][:n]])[:, h // 2], np.concatenate([pv, own[r][1][:n]])[:, h // 2]
            e = np.exp(k @ q[t, h] / 2)
            np.testing.assert_allclose(out[t, h], e @ v / e.sum(), rtol=1e-12)
            np.testing.assert_allclose(lse[t, h], np.log(e.sum()), rtol=1e-12)


def test_oracle_sample():
    z = [1.0, 3.0, 3.0, -np.inf, np.nan, 2.0]
    assert batch.sample_row(z, 0.9, 0.0) == (1, 1, 0.0)
    assert batch.sample_row(z, 0.0, 1.0, k=1)[:2] == (1, 1)
    assert batch.sample_row(z, 0.99, 1.0, k=2)[:2] == (2, 2)
    assert batch.sample_row(z, 0.999, 1.0)[:2] == (5, 4)
    assert batch.sample_row(z, 0.0, 1.0)[:2] == (0, 4)
    assert batch.sample_row(z, 0.5, 1.0, p=0.0)[:2] == (1, 1)
    assert batch.sample_row(z, 0.999, 1.0, low=math.exp(-1.5))[:2] == (5, 3)
    assert batch.sample_row([-np.inf, np.nan], 0.5, 1.0) == (-1, 0, -math.inf)
    assert batch.sample_row([0.0, np.inf, 5.0, np.inf], 0.6, 1.0)[:2] == (3, 4)
    e = np.exp([1.0, 3.0, 3.0, 2.0])
    assert abs(batch.sample_row(z, 0.999, 1.0)[2] - math.log(e[3] / e.sum())) < 1e-12
