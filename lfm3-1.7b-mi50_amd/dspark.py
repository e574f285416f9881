"""Host-side binding of libdspark_amd.so (the C ABI in include/dspark.h).

ctypes over the C ABI; torch is used only for device memory and the current HIP stream. There is no fallback:
if the library is missing the import fails, and every call raises on a nonzero status.

Mirrors the reference's host path for the DSpark step (internal/model/dspark.go: State words 52-77, draftLaunch
537-621) at the level the C ABI exposes: per-round attention, argmax, acceptance and commit.
"""
import ctypes
import os

HERE = os.path.dirname(os.path.abspath(__file__))
LIB_PATH = os.path.join(HERE, "libdspark_amd.so")

MT_MAX = 64
PAGE = 32

STATE_FIELDS = ["a", "anchor", "count", "rounds_left", "limit", "budget", "eos", "M", "ctx_new", "ctx_pos", "ctx_lo",
                "run", "force_m", "rounds_done", "accepted", "verified", "miss", "skip", "skip_after", "skip_rounds",
                "stop_at", "ckpt_slot"]

ENOSPACE = 1002
ERRORS = {1001: "DSPARK_EINVAL", ENOSPACE: "DSPARK_ENOSPACE", 1003: "DSPARK_EUNSUPPORTED"}


class DsparkError(RuntimeError):
    pass


class State(ctypes.Structure):
    """struct dspark_state (include/dspark.h) = struct State of dspark.hip:134-158 with tokens[64]."""
    _fields_ = [(n, ctypes.c_int32) for n in STATE_FIELDS] + [("tokens", ctypes.c_int32 * MT_MAX)]


class AttnArgs(ctypes.Structure):
    _fields_ = [("q", ctypes.c_void_p), ("k_pages", ctypes.c_void_p), ("v_pages", ctypes.c_void_p),
                ("block_table", ctypes.c_void_p), ("kv_pages", ctypes.c_int64), ("out", ctypes.c_void_p), ("out_f32", ctypes.c_void_p),
                ("gate", ctypes.c_void_p), ("workspace", ctypes.c_void_p), ("workspace_bytes", ctypes.c_size_t),
                ("M", ctypes.c_int32), ("QH", ctypes.c_int32), ("KVH", ctypes.c_int32), ("D", ctypes.c_int32),
                ("a", ctypes.c_int32), ("start", ctypes.c_int32), ("window", ctypes.c_int32),
                ("causal", ctypes.c_int32), ("splits", ctypes.c_int32)]


class B8CacheArgs(ctypes.Structure):
    _fields_ = [("k", ctypes.c_void_p), ("v", ctypes.c_void_p), ("k_scale", ctypes.c_void_p), ("v_scale", ctypes.c_void_p),
                ("block_table", ctypes.c_void_p), ("kv_pages", ctypes.c_int64), ("KVH", ctypes.c_int32),
                ("D", ctypes.c_int32), ("code", ctypes.c_int32)]


class B8AttnArgs(ctypes.Structure):
    _fields_ = [("q", ctypes.c_void_p), ("q_stride", ctypes.c_int64), ("out", ctypes.c_void_p), ("out_f32", ctypes.c_void_p),
                ("lse", ctypes.c_void_p), ("gate", ctypes.c_void_p), ("workspace", ctypes.c_void_p),
                ("workspace_bytes", ctypes.c_size_t), ("arrivals", ctypes.c_void_p), ("M", ctypes.c_int32),
                ("QH", ctypes.c_int32), ("a", ctypes.c_int32), ("start", ctypes.c_int32), ("window", ctypes.c_int32), ("causal", ctypes.c_int32),
                ("splits", ctypes.c_int32)]


_lib = None

_SIGS = {
    "dspark_abi_version": (ctypes.c_int, []),
    "dspark_page_tokens": (ctypes.c_int, []),
    "dspark_max_tokens": (ctypes.c_int, []),
    "dspark_state_bytes": (ctypes.c_int, []),
    "dspark_verify_attention_workspace": (ctypes.c_size_t, [ctypes.POINTER(AttnArgs)]),
    "dspark_verify_attention": (ctypes.c_int, [ctypes.POINTER(AttnArgs), ctypes.c_void_p]),
    "dspark_verify_attention_splits": (ctypes.c_int, [ctypes.POINTER(AttnArgs), ctypes.c_void_p]),
    "dspark_verify_attention_combine": (ctypes.c_int, [ctypes.POINTER(AttnArgs), ctypes.c_void_p]),
    "dspark_verify_attention_noalloc": (ctypes.c_int, [ctypes.POINTER(AttnArgs), ctypes.c_void_p]),
    "dspark_kv_write": (ctypes.c_int, [ctypes.c_void_p, ctypes.c_void_p, ctypes.c_int64, ctypes.c_void_p,
                                       ctypes.c_void_p, ctypes.c_void_p, ctypes.c_int64, ctypes.c_int32, ctypes.c_int32,
                                       ctypes.c_int32, ctypes.c_int32, ctypes.c_void_p]),
    "dspark_kv_write_rec": (ctypes.c_int, [ctypes.c_void_p, ctypes.c_void_p, ctypes.c_int64, ctypes.c_void_p,
                                           ctypes.c_void_p, ctypes.c_int64, ctypes.c_int32, ctypes.c_int32,
                                           ctypes.c_int32, ctypes.c_void_p]),
    "dspark_verify_attention_rec_workspace": (ctypes.c_size_t, [ctypes.POINTER(AttnArgs)]),
    "dspark_verify_attention_rec": (ctypes.c_int, [ctypes.POINTER(AttnArgs), ctypes.c_void_p]),
    "dspark_verify_attention_rec_splits": (ctypes.c_int, [ctypes.POINTER(AttnArgs), ctypes.c_void_p]),
    "dspark_verify_attention_rec_combine": (ctypes.c_int, [ctypes.POINTER(AttnArgs), ctypes.c_void_p]),
    "dspark_kv_write_b8": (ctypes.c_int, [ctypes.POINTER(B8CacheArgs), ctypes.c_void_p, ctypes.c_void_p, ctypes.c_int64,
                                          ctypes.c_int32, ctypes.c_int32, ctypes.c_void_p]),
    "dspark_kv_read_b8": (ctypes.c_int, [ctypes.POINTER(B8CacheArgs), ctypes.c_int32, ctypes.c_int32, ctypes.c_void_p,
                                         ctypes.c_void_p, ctypes.c_int64, ctypes.c_void_p]),
    "dspark_verify_attention_b8_workspace": (ctypes.c_size_t, [ctypes.POINTER(B8CacheArgs), ctypes.POINTER(B8AttnArgs)]),
    "dspark_verify_attention_b8": (ctypes.c_int, [ctypes.POINTER(B8CacheArgs), ctypes.POINTER(B8AttnArgs),
                                                  ctypes.c_void_p]),
    "dspark_attention_mass_b8": (ctypes.c_int, [ctypes.POINTER(B8CacheArgs), ctypes.POINTER(B8AttnArgs), ctypes.c_void_p,
                                                ctypes.c_void_p, ctypes.c_void_p, ctypes.c_void_p, ctypes.c_int64,
                                                ctypes.c_void_p]),
    "dspark_kv_evict_b8": (ctypes.c_int, [ctypes.POINTER(B8CacheArgs), ctypes.POINTER(B8CacheArgs), ctypes.c_int32,
                                          ctypes.c_int32, ctypes.c_int32, ctypes.c_int32, ctypes.c_void_p, ctypes.c_int64,
                                          ctypes.c_void_p, ctypes.c_void_p, ctypes.c_int64, ctypes.c_void_p,
                                          ctypes.c_size_t, ctypes.c_void_p]),
    "dspark_kv_evict_b8_workspace": (ctypes.c_size_t, [ctypes.c_int32, ctypes.c_int32]),
    "dspark_rope_table": (ctypes.c_int, [ctypes.c_float, ctypes.c_int32, ctypes.c_int32, ctypes.c_int32,
                                         ctypes.c_void_p]),
    "dspark_verify_argmax_workspace": (ctypes.c_size_t, [ctypes.c_int32, ctypes.c_int32]),
    "dspark_verify_argmax": (ctypes.c_int, [ctypes.c_void_p, ctypes.c_int32, ctypes.c_int32, ctypes.c_int32,
                                            ctypes.c_void_p, ctypes.c_void_p, ctypes.c_float, ctypes.c_float,
                                            ctypes.c_void_p, ctypes.c_void_p, ctypes.c_size_t, ctypes.c_void_p]),
    "dspark_accept_commit": (ctypes.c_int, [ctypes.c_void_p, ctypes.c_void_p, ctypes.c_int32, ctypes.c_int32,
                                            ctypes.c_void_p, ctypes.c_int32, ctypes.c_void_p, ctypes.c_void_p]),
    "dspark_gemm_i8_workspace": (ctypes.c_size_t, [ctypes.c_int32, ctypes.c_int32, ctypes.c_int32]),
    "dspark_gemm_i8": (ctypes.c_int, [ctypes.c_void_p, ctypes.c_int32, ctypes.c_int32, ctypes.c_void_p,
                                      ctypes.c_void_p, ctypes.c_int32, ctypes.c_int32, ctypes.c_void_p,
                                      ctypes.c_void_p, ctypes.c_void_p, ctypes.c_size_t, ctypes.c_void_p]),
    "dspark_gemm_i8_g128": (ctypes.c_int, [ctypes.c_void_p, ctypes.c_int32, ctypes.c_int32, ctypes.c_void_p,
                                           ctypes.c_void_p, ctypes.c_int32, ctypes.c_int32, ctypes.c_void_p,
                                           ctypes.c_void_p, ctypes.c_void_p]),
    "dspark_gemm_i8_g128_x8": (ctypes.c_int, [ctypes.c_void_p, ctypes.c_void_p, ctypes.c_int32, ctypes.c_int32,
                                              ctypes.c_void_p, ctypes.c_void_p, ctypes.c_int32, ctypes.c_int32,
                                              ctypes.c_void_p, ctypes.c_void_p, ctypes.c_void_p]),
    "dspark_g128_scales": (ctypes.c_int, [ctypes.c_void_p, ctypes.c_int32, ctypes.c_int32, ctypes.c_void_p]),
    "dspark_head_argmax_workspace": (ctypes.c_size_t, [ctypes.c_int32, ctypes.c_int32]),
    "dspark_head_argmax_f16": (ctypes.c_int, [ctypes.c_void_p, ctypes.c_int32, ctypes.c_int32, ctypes.c_void_p,
                                              ctypes.c_int32, ctypes.c_void_p, ctypes.c_void_p, ctypes.c_void_p,
                                              ctypes.c_size_t, ctypes.c_void_p]),
}


ABI_VERSION = 5  # dspark_abi_version() of the library these signatures describe


def lib():
    """Load libdspark_amd.so; raises if it has not been built (no fallback path exists)."""
    global _lib
    if _lib is None:
        if not os.path.exists(LIB_PATH):
            raise DsparkError(f"{LIB_PATH} is missing: run __graft_entry__.build() (make -C {HERE})")
        L = ctypes.CDLL(LIB_PATH)
        for name, (res, args) in _SIGS.items():
            fn = getattr(L, name)
            fn.restype = res
            fn.argtypes = args
        if L.dspark_abi_version() != ABI_VERSION:
            raise DsparkError(f"{LIB_PATH} has ABI {L.dspark_abi_version()}, this module binds {ABI_VERSION}: "
                              "rebuild it")
        _lib = L
    return _lib


def check(rc, what):
    if rc != 0:
        raise DsparkError(f"{what} failed: {ERRORS.get(rc, 'hipError %d' % rc)}")


# ---------------------------------------------------------------- torch plumbing
def _torch():
    import torch
    return torch


def ptr(t):
    return None if t is None else ctypes.c_void_p(t.data_ptr())


def stream_handle(stream=None):
    torch = _torch()
    s = stream if stream is not None else torch.cuda.current_stream()
    return ctypes.c_void_p(s.cuda_stream)


class Workspace:
    """A growable device byte buffer reused across calls (caller-owned memory, as the reference's engine owns
    every buffer, internal/model/dspark.go:202-223)."""

    def __init__(self, device="cuda"):
        self.device = device
        self.buf = None
        self.words = None
        self.captured = []  # buffers that captured graphs write to: kept when the workspace grows past them

    def get(self, nbytes):
        torch = _torch()
        nbytes = max(int(nbytes), 256)
        if self.buf is None or self.buf.numel() < nbytes:
            self.let_go(self.buf)
            # zero-filled: the split-K GEMM keeps its arrival counters here (left at zero by every call)
            self.buf = torch.zeros(nbytes, dtype=torch.uint8, device=self.device)
        if self.buf.is_cuda and torch.cuda.is_current_stream_capturing():
            self.hold()
        return self.buf

    @staticmethod
    def let_go(t):
        """Work on the current stream may still use the buffer that is about to be replaced, which can belong to another one:
        its memory is not handed out before that work is done."""
        if t is not None and t.is_cuda:
            t.record_stream(_torch().cuda.current_stream(t.device))

    def hold(self):
        """The buffer stays allocated as long as the workspace: a graph that is being captured will write to it."""
        if not any(self.buf is b for b in self.captured):
            self.captured.append(self.buf)

    def arrivals(self, n):
        """n words apart from the buffer, zeroed once: arrival counters, which their user leaves at zero."""
        torch = _torch()
        if self.words is None or self.words.numel() < n:
            self.let_go(self.words)
            self.words = torch.zeros(n, dtype=torch.int32, device=self.device)
        return self.words


# ---------------------------------------------------------------- KV pages
def kv_pages_alloc(n_pages, KVH, D, device="cuda"):
    torch = _torch()
    k = torch.zeros((n_pages, KVH, PAGE, D), dtype=torch.float16, device=device)
    v = torch.zeros((n_pages, KVH, D, PAGE), dtype=torch.float16, device=device)
    return k, v


def kv_write(k, v, k_pages, v_pages, pos0, block_table=None, stream=None):
    """k, v: fp16 [n][KVH][D] (or [n][row] with row >= KVH*D) device tensors."""
    n = k.shape[0]
    KVH, D = k_pages.shape[1], k_pages.shape[3]
    row = k.stride(0)
    assert v.stride(0) == row and k.dtype == v.dtype == _torch().float16
    rc = lib().dspark_kv_write(ptr(k), ptr(v), row, ptr(k_pages), ptr(v_pages), ptr(block_table), k_pages.shape[0], KVH,
                               D, pos0, n, stream_handle(stream))
    check(rc, "dspark_kv_write")


def k_page_index(D):
    """For a (page, head) K block of 32*D halves: flat index of K[key][d], as a [32][D] int64 array (the operand
    order documented in include/dspark.h)."""
    import numpy as np
    key = np.arange(PAGE)[:, None]
    d = np.arange(D)[None, :]
    b = (key >> 2) & 1
    nrow = 4 * (key >> 3) + (key & 3)
    s, g, j = d // 32, (d % 32) // 8, d % 8
    return (((b * (D // 32) + s) * 64 + nrow + 16 * g) * 8 + j).astype(np.int64)


def kv_from_pages(k_pages, v_pages, positions, block_table=None):
    """Read K/V rows of the given positions back from the pages (host copy; for checks and debugging)."""
    import numpy as np
    kp = k_pages.detach().cpu().numpy()
    vp = v_pages.detach().cpu().numpy()
    n_pages, KVH = kp.shape[0], kp.shape[1]
    D = kp.size // (n_pages * KVH * PAGE)
    kflat = kp.reshape(n_pages, KVH, PAGE * D)
    vflat = vp.reshape(n_pages, KVH, D, PAGE)
    idx = k_page_index(D)
    bt = None if block_table is None else block_table.detach().cpu().numpy()
    ks, vs = [], []
    for pos in positions:
        lp, sl = divmod(int(pos), PAGE)
        pg = lp if bt is None else int(bt[lp])
        ks.append(kflat[pg][:, idx[sl]])
        vs.append(vflat[pg][:, :, sl])
    return np.stack(ks), np.stack(vs)


def kv_to_pages(k, v, n_pages=None, block_table=None):
    """Logical fp16 [T][KVH][D] K and V -> freshly allocated page pools (identity table unless given)."""
    T, KVH, D = k.shape
    if n_pages is None:
        n_pages = (T + PAGE - 1) // PAGE
    kp, vp = kv_pages_alloc(n_pages, KVH, D, device=k.device)
    kv_write(k.contiguous(), v.contiguous(), kp, vp, 0, block_table)
    return kp, vp


# ---------------------------------------------------------------- verify attention
def attn_args(q, k_pages, v_pages, a, start=0, window=0, causal=True, out=None, out_f32=None, gate=None,
              block_table=None, splits=0):
    M, QH, D = q.shape
    KVH = k_pages.shape[1]
    args = AttnArgs()
    args.q, args.k_pages, args.v_pages = q.data_ptr(), k_pages.data_ptr(), v_pages.data_ptr()
    args.block_table = block_table.data_ptr() if block_table is not None else None
    args.kv_pages = k_pages.shape[0]
    args.out = out.data_ptr() if out is not None else None
    args.out_f32 = out_f32.data_ptr() if out_f32 is not None else None
    args.gate = gate.data_ptr() if gate is not None else None
    args.M, args.QH, args.KVH, args.D = M, QH, KVH, D
    args.a, args.start, args.window, args.causal, args.splits = a, start, window, int(causal), splits
    return args


def verify_attention(q, k_pages, v_pages, a, start=0, window=0, causal=True, out=None, out_f32=None, gate=None,
                     block_table=None, splits=0, workspace=None, stream=None):
    """q fp16 [M][QH][D]; pages hold positions 0..a+M-1. Returns (out fp16, out_f32) tensors as given/created."""
    torch = _torch()
    M, QH, D = q.shape
    if out is None and out_f32 is None:
        out = torch.empty((M, QH, D), dtype=torch.float16, device=q.device)
    args = attn_args(q, k_pages, v_pages, a, start, window, causal, out, out_f32, gate, block_table, splits)
    need = lib().dspark_verify_attention_workspace(ctypes.byref(args))
    if need == 0:
        raise DsparkError("dspark_verify_attention_workspace rejected the arguments")
    ws = (workspace or Workspace(q.device)).get(need)
    args.workspace, args.workspace_bytes = ws.data_ptr(), ws.numel()
    check(lib().dspark_verify_attention(ctypes.byref(args), stream_handle(stream)), "dspark_verify_attention")
    return out, out_f32


# ---------------------------------------------------------------- int8 K/V records
REC_BYTES = 264


def rec_pages_alloc(n_pages, KVH, device="cuda"):
    """A record pool: [n_pages][32 slots][KVH][264 bytes] (internal/model/engine.go:30-32)."""
    return _torch().zeros((n_pages, PAGE, KVH, REC_BYTES), dtype=_torch().uint8, device=device)


def kv_write_rec(k, v, pages, pos0, block_table=None, stream=None):
    """k, v: fp32 [n][KVH][128] (or [n][row], row >= KVH*128) device tensors -> quantize_pair records."""
    torch = _torch()
    n = k.shape[0]
    KVH = pages.shape[2]
    row = k.stride(0)
    assert v.stride(0) == row and k.dtype == v.dtype == torch.float32 and pages.dtype == torch.uint8
    rc = lib().dspark_kv_write_rec(ptr(k), ptr(v), row, ptr(pages), ptr(block_table), pages.shape[0], KVH, pos0, n,
                                   stream_handle(stream))
    check(rc, "dspark_kv_write_rec")


def rec_attn_args(q, pages, a, start=0, window=0, causal=True, out=None, out_f32=None, gate=None, block_table=None,
                  splits=0):
    M, QH, D = q.shape
    args = AttnArgs()
    args.q, args.k_pages, args.v_pages = q.data_ptr(), pages.data_ptr(), None
    args.block_table = block_table.data_ptr() if block_table is not None else None
    args.kv_pages = pages.shape[0]
    args.out = out.data_ptr() if out is not None else None
    args.out_f32 = out_f32.data_ptr() if out_f32 is not None else None
    args.gate = gate.data_ptr() if gate is not None else None
    args.M, args.QH, args.KVH, args.D = M, QH, pages.shape[2], D
    args.a, args.start, args.window, args.causal, args.splits = a, start, window, int(causal), splits
    return args


def verify_attention_rec(q, pages, a, start=0, window=0, causal=True, out=None, out_f32=None, gate=None,
                         block_table=None, splits=0, workspace=None, stream=None):
    """q fp16 [M][QH][128]; pages: a record pool holding positions 0..a+M-1."""
    torch = _torch()
    M, QH, D = q.shape
    if out is None and out_f32 is None:
        out = torch.empty((M, QH, D), dtype=torch.float16, device=q.device)
    args = rec_attn_args(q, pages, a, start, window, causal, out, out_f32, gate, block_table, splits)
    need = lib().dspark_verify_attention_rec_workspace(ctypes.byref(args))
    if need == 0:
        raise DsparkError("dspark_verify_attention_rec_workspace rejected the arguments")
    ws = (workspace or Workspace(q.device)).get(need)
    args.workspace, args.workspace_bytes = ws.data_ptr(), ws.numel()
    check(lib().dspark_verify_attention_rec(ctypes.byref(args), stream_handle(stream)), "dspark_verify_attention_rec")
    return out, out_f32


# ---------------------------------------------------------------- 8-bit block-scaled K/V cache
B8_INT8, B8_E4M3 = 0, 1
B8_ARRIVALS = 64


class B8Cache:
    """A cache of "b8" pages (include/dspark.h): codes k, v [n_pages][KVH][32][D] as torch.int8 or torch.float8_e4m3fn,
    scales fp32 [n_pages][KVH], and an int32 block table (None = identity). Holds the tensors and their descriptor."""

    def __init__(self, k, v, k_scale, v_scale, block_table=None):
        torch = _torch()
        codes = {torch.int8: B8_INT8, torch.float8_e4m3fn: B8_E4M3}
        if k.dim() != 4 or k.shape != v.shape or k.dtype != v.dtype or k.dtype not in codes or k.shape[2] != PAGE:
            raise DsparkError("B8Cache: k and v are [n_pages][KVH][32][D] of int8 or float8_e4m3fn")
        for t in (k_scale, v_scale):
            if t.shape != k.shape[:2] or t.dtype != torch.float32:
                raise DsparkError("B8Cache: scales are fp32 [n_pages][KVH]")
        if block_table is not None and (block_table.dtype != torch.int32 or block_table.dim() != 1):
            raise DsparkError("B8Cache: the block table is int32 [pages]")
        every = [t for t in (k, v, k_scale, v_scale, block_table) if t is not None]
        if any(t.device != k.device or not t.is_contiguous() for t in every):
            raise DsparkError("B8Cache: contiguous tensors of one device")
        self.k, self.v, self.k_scale, self.v_scale, self.block_table = k, v, k_scale, v_scale, block_table
        self.KVH, self.D, self.device, self.index = k.shape[1], k.shape[3], k.device, k.get_device()
        self.positions = None if block_table is None else block_table.shape[0] * PAGE  # that the table has entries for
        self.args = B8CacheArgs(k.data_ptr(), v.data_ptr(), k_scale.data_ptr(), v_scale.data_ptr(),
                                None if block_table is None else block_table.data_ptr(), k.shape[0], self.KVH, self.D,
                                codes[k.dtype])
        self.ref = ctypes.byref(self.args)

    def check(self, end, *tensors):
        """`end` positions have table entries, and the tensors are the cache's device's."""
        if self.positions is not None and end > self.positions:
            raise DsparkError(f"{end} positions need {(end + PAGE - 1) // PAGE} entries in the block table")
        for t in tensors:
            if t is not None and t.get_device() != self.index:
                raise DsparkError("tensors and cache are on different devices")


def b8_cache_alloc(n_pages, KVH, D, dtype=None, device="cuda", block_table=None):
    """An empty cache; dtype torch.int8 (the default) or torch.float8_e4m3fn."""
    torch = _torch()
    codes = [torch.zeros((n_pages, KVH, PAGE, D), dtype=torch.uint8, device=device).view(dtype or torch.int8) for _ in "kv"]
    scales = [torch.zeros((n_pages, KVH), dtype=torch.float32, device=device) for _ in "kv"]
    return B8Cache(*codes, *scales, block_table)


def _b8_words(every, what):
    """`every`, the bitwise or of a call's counts and positions, says whether one is negative or past the 31 bits of the C ABI's
    (ctypes would cut it to its low 32 in silence)."""
    if every >> 31:
        raise DsparkError(f"{what}: counts and positions are from 0 to 2^31 - 1")


def _b8_on(cache, stream, call, *args):
    """call(handle of the stream, cache, *args) with the cache's device current and `stream` (default: that device's current
    one) the stream that allocations belong to."""
    torch = _torch()
    if stream is None and cache.index >= 0 and torch.cuda.current_device() == cache.index:
        return call(torch._C._cuda_getCurrentRawStream(cache.index), cache, *args)
    if cache.index < 0:
        raise DsparkError("the cache is not on a GPU")
    stream = stream if stream is not None else torch.cuda.current_stream(cache.device)
    if stream.device_index != cache.index:
        raise DsparkError("the stream belongs to another device than the cache")
    with torch.cuda.stream(stream):
        return call(stream.cuda_stream, cache, *args)


def _b8_row(t, cache, what):
    """Elements between the rows of a [n][KVH][D] (or [n][row]) tensor whose rows are contiguous."""
    shape, stride, H, D = t.shape, t.stride(), cache.KVH, cache.D
    if len(shape) == 3 and shape[1] == H and shape[2] == D and stride[2] == 1 and (H == 1 or stride[1] == D) \
            or len(shape) == 2 and shape[1] >= H * D and stride[1] == 1:
        return stride[0] if shape[0] > 1 else H * D
    raise DsparkError(f"{what}: rows of {H} heads x {D}")


def _kv_write_b8(s, cache, k, v, row, pos0, n):
    check(lib().dspark_kv_write_b8(cache.ref, k.data_ptr(), v.data_ptr(), row, pos0, n, s), "dspark_kv_write_b8")


def kv_write_b8(k, v, cache, pos0, stream=None):
    """Append k, v fp16 [n][KVH][D] (or [n][row >= KVH*D]; rows may lie inside wider ones) as positions pos0 .. pos0+n-1."""
    f16 = _torch().float16
    row, n = _b8_row(k, cache, "kv_write_b8"), k.shape[0]
    _b8_words(pos0 | n, "kv_write_b8")
    if v.shape != k.shape or _b8_row(v, cache, "kv_write_b8") != row or k.dtype != f16 or v.dtype != f16:
        raise DsparkError("kv_write_b8: k and v are fp16, of one shape and row stride")
    cache.check(pos0 + n, k, v)
    _b8_on(cache, stream, _kv_write_b8, k, v, row, pos0, n)


def _kv_read_b8(s, cache, pos0, n, k, v):
    torch = _torch()
    if k is None and v is None:
        k, v = torch.empty((2, n, cache.KVH, cache.D), dtype=torch.float32, device=cache.device).unbind()
    elif k is None or v is None:  # the other one laid out alike
        given = k if v is None else v
        made = torch.empty_strided(given.shape, given.stride(), dtype=torch.float32, device=cache.device)
        k, v = (given, made) if v is None else (made, given)
    row = _b8_row(k, cache, "kv_read_b8")
    if k.dtype != torch.float32 or v.dtype != torch.float32 or k.shape[0] < n or v.shape != k.shape \
            or _b8_row(v, cache, "kv_read_b8") != row:
        raise DsparkError("kv_read_b8: k and v are fp32 rows of one shape and stride")
    check(lib().dspark_kv_read_b8(cache.ref, pos0, n, k.data_ptr(), v.data_ptr(), row, s), "dspark_kv_read_b8")
    return k, v


def kv_read_b8(cache, pos0, n, k=None, v=None, stream=None):
    """The values of positions pos0 .. pos0+n-1 as fp32 [n][KVH][D] tensors, given (as rows) or created; one of them alone
    given, the other is created of its shape and strides."""
    _b8_words(pos0 | n, "kv_read_b8")
    cache.check(pos0 + n, k, v)
    return _b8_on(cache, stream, _kv_read_b8, pos0, n, k, v)


def _b8_attn_args(q, cache, a, start, window, causal, splits=0):
    shape, stride = q.shape, q.stride()
    if len(shape) != 3 or shape[2] != cache.D or q.dtype != _torch().float16 or stride[2] != 1 \
            or (shape[1] > 1 and stride[1] != cache.D):
        raise DsparkError("q is fp16 [M][QH][D] of contiguous rows, D the cache's")
    M, QH, D = shape
    _b8_words(a | start | window | splits, "b8 attention")
    cache.check(a + M, q)
    return B8AttnArgs(q.data_ptr(), stride[0] if M > 1 else QH * D, None, None, None, None, None, 0, None,
                      M, QH, a, start, window, 1 if causal else 0, splits)


def _b8_full(t, shape, dtype, cache, what):
    """The data pointer of an optional tensor that has to be contiguous and of this shape and type."""
    if t is None:
        return None
    if t.shape != shape or t.dtype != dtype or not t.is_contiguous() or t.get_device() != cache.index:
        raise DsparkError(f"{what} is a contiguous {dtype} tensor of shape {tuple(shape)} on the cache's device")
    return t.data_ptr()


def _b8_workspace(cache, workspace, need):
    ws = (workspace or Workspace(cache.device)).get(need)
    if ws.get_device() != cache.index:
        raise DsparkError("workspace and cache are on different devices")
    return ws


def _verify_attention_b8(s, cache, q, args, out, out_f32, workspace):
    torch = _torch()
    if out is None and out_f32 is None:
        out = q.new_empty(q.shape)
    args.out = _b8_full(out, q.shape, torch.float16, cache, "out")
    args.out_f32 = _b8_full(out_f32, q.shape, torch.float32, cache, "out_f32")
    # The counters save a launch, which costs the host more than the last split's work the GPU; a graph's launch costs little,
    # and zeroing counters for one call a launch itself.
    if workspace is not None:
        if not torch.cuda.is_current_stream_capturing():
            args.arrivals = workspace.arrivals(cache.KVH * B8_ARRIVALS).data_ptr()
        elif workspace.buf is not None:
            workspace.hold()
    ref, ws = ctypes.byref(args), workspace and workspace.buf
    while True:  # with the workspace as it is first, then with one that is large enough
        if ws is not None:
            if ws.get_device() != cache.index:
                raise DsparkError("workspace and cache are on different devices")
            args.workspace, args.workspace_bytes = ws.data_ptr(), ws.numel()
        rc = lib().dspark_verify_attention_b8(cache.ref, ref, s)
        if rc != ENOSPACE:
            check(rc, "dspark_verify_attention_b8")
            return out, out_f32
        need = lib().dspark_verify_attention_b8_workspace(cache.ref, ref)
        if need <= args.workspace_bytes:
            check(rc, "dspark_verify_attention_b8")
        ws = _b8_workspace(cache, workspace, need)


def verify_attention_b8(q, cache, a, start=0, window=0, causal=True, out=None, out_f32=None, lse=None, gate=None, splits=0,
                        workspace=None, stream=None):
    """verify_attention over a B8Cache that holds positions 0..a+M-1. q fp16 [M][QH][D]; lse (optional) fp32 [M][QH] receives
    the log-sum-exp of the scores. A workspace that is kept saves a launch for few rows: it holds the counters by which the
    last key split to finish adds them all. Returns (out fp16, out_f32) tensors as given/created."""
    args = _b8_attn_args(q, cache, a, start, window, causal, splits)
    f32 = _torch().float32
    args.lse = _b8_full(lse, q.shape[:2], f32, cache, "lse")
    args.gate = _b8_full(gate, q.shape[:2], f32, cache, "gate")
    return _b8_on(cache, stream, _verify_attention_b8, q, args, out, out_f32, workspace)


def _b8_accounts(t, n, cache, what):
    """Elements between the heads of an fp32 [KVH][>= n] tensor."""
    shape, stride = t.shape, t.stride()
    if len(shape) != 2 or shape[0] != cache.KVH or shape[1] < n or t.dtype != _torch().float32 \
            or (shape[1] > 1 and stride[1] != 1) or t.get_device() != cache.index:
        raise DsparkError(f"{what} is fp32 [KVH][>= {n}] on the cache's device")
    return stride[0] if shape[0] > 1 else n


def _attention_mass_b8(s, cache, args, lse, rows, mass_in, mass_out, stride):
    lse = lse.contiguous()
    check(lib().dspark_attention_mass_b8(cache.ref, ctypes.byref(args), lse.data_ptr(), None if rows is None else rows.data_ptr(),
                                         None if mass_in is None else mass_in.data_ptr(), mass_out.data_ptr(), stride, s),
          "dspark_attention_mass_b8")
    return mass_out


def attention_mass_b8(q, cache, a, lse, mass_out, mass_in=None, rows=None, start=0, window=0, causal=True, stream=None):
    """Add the attention weights of tokens t < rows (an int32 device word, None = all of q's) to the accounts of the keys they
    see: mass_out fp32 [KVH][>= a+M] from mass_in (None = zeros, or mass_out itself) and verify_attention_b8's lse (copied
    if its strides are others)."""
    torch = _torch()
    args = _b8_attn_args(q, cache, a, start, window, causal)
    if lse is None or lse.shape != q.shape[:2] or lse.dtype != torch.float32 or lse.get_device() != cache.index:
        raise DsparkError(f"lse is fp32 of shape {tuple(q.shape[:2])} on the cache's device")
    stride = _b8_accounts(mass_out, a + args.M, cache, "mass_out")
    if mass_in is not None and _b8_accounts(mass_in, a + args.M, cache, "mass_in") != stride:
        raise DsparkError("attention_mass_b8: mass_in and mass_out have one stride")
    if rows is not None and (rows.dtype != torch.int32 or rows.numel() < 1 or rows.get_device() != cache.index):
        raise DsparkError("attention_mass_b8: rows is an int32 word on the cache's device")
    return _b8_on(cache, stream, _attention_mass_b8, args, lse, rows, mass_in, mass_out, stride)


def _kv_evict_b8(s, cache, dst, length, keep, mass, stride, sinks, recent, kept, mass_out, workspace):
    torch = _torch()
    if kept is None:
        kept = torch.empty((cache.KVH, keep), dtype=torch.int32, device=cache.device)
    if mass_out is None:
        mass_out = torch.empty((cache.KVH, keep), dtype=torch.float32, device=cache.device)
    kept_ptr = _b8_full(kept, (cache.KVH, keep), torch.int32, cache, "kept")
    out_stride = _b8_accounts(mass_out, keep, cache, "mass_out")
    need = lib().dspark_kv_evict_b8_workspace(cache.KVH, length)
    ws = _b8_workspace(cache, workspace, need) if need else None
    check(lib().dspark_kv_evict_b8(cache.ref, dst.ref, length, keep, sinks, recent, mass.data_ptr(), stride, kept_ptr,
                                   mass_out.data_ptr(), out_stride, None if ws is None else ws.data_ptr(),
                                   0 if ws is None else ws.numel(), s), "dspark_kv_evict_b8")
    return kept, mass_out


def kv_evict_b8(cache, dst, length, keep, mass, sinks=0, recent=0, kept=None, mass_out=None, workspace=None, stream=None):
    """Keep `keep` of the cache's `length` positions per KV head -- the first `sinks`, the last `recent`, and the rest by mass
    (fp32 [KVH][>= length]) -- as positions 0..keep-1 of `dst`, another B8Cache of the same heads and codes. Returns
    (kept int32 [KVH][keep] ascending, their mass), as given/created."""
    _b8_words(length | keep | sinks | recent, "kv_evict_b8")
    cache.check(length, dst.k)
    dst.check(keep)
    stride = _b8_accounts(mass, length, cache, "mass")
    return _b8_on(cache, stream, _kv_evict_b8, dst, length, keep, mass, stride, sinks, recent, kept, mass_out, workspace)


# ---------------------------------------------------------------- argmax / accept
def state_tensor(device="cuda", **fields):
    """A device dspark_state initialised from keyword fields (tokens=list)."""
    torch = _torch()
    st = State()
    for k, v in fields.items():
        if k == "tokens":
            for i, t in enumerate(v):
                st.tokens[i] = int(t)
        else:
            setattr(st, k, int(v))
    raw = bytes(st)
    host = torch.frombuffer(bytearray(raw), dtype=torch.int32).clone()
    return host.to(device)


def state_from_tensor(t):
    st = State()
    ctypes.memmove(ctypes.byref(st), bytes(t.cpu().numpy().tobytes()), ctypes.sizeof(State))
    return st


def verify_argmax(logits, seen, st, rep=1.0, inv_rep=None, best=None, workspace=None, stream=None):
    torch = _torch()
    M, V = logits.shape
    f16 = logits.dtype == torch.float16
    if inv_rep is None:
        inv_rep = float(torch.tensor(1.0, dtype=torch.float32) / torch.tensor(rep, dtype=torch.float32))
    if best is None:
        best = torch.empty(M, dtype=torch.int64, device=logits.device)
    need = lib().dspark_verify_argmax_workspace(M, V)
    ws = (workspace or Workspace(logits.device)).get(need)
    rc = lib().dspark_verify_argmax(ptr(logits), int(f16), M, V, ptr(seen), ptr(st), rep, inv_rep, ptr(best), ptr(ws),
                                    ws.numel(), stream_handle(stream))
    check(rc, "dspark_verify_argmax")
    return best


def accept_commit(st, best, M, out_tokens, seen, skip_now=0, stream=None):
    rc = lib().dspark_accept_commit(ptr(st), ptr(best), M, skip_now, ptr(out_tokens), out_tokens.numel(), ptr(seen),
                                    stream_handle(stream))
    check(rc, "dspark_accept_commit")


def keys_to_tokens(keys):
    """u64 keys held in an int64 tensor -> token ids."""
    torch = _torch()
    low = keys & 0xFFFFFFFF
    return (0xFFFFFFFF - low).to(torch.int64)


# ---------------------------------------------------------------- GEMMs
def gemm_i8(x, w_biased, scale, epilogue=0, y_f32=None, y_f16=None, workspace=None, stream=None):
    torch = _torch()
    M, K = x.shape
    N = w_biased.shape[0]
    if epilogue == 0 and y_f32 is None and y_f16 is None:
        y_f32 = torch.empty((M, N), dtype=torch.float32, device=x.device)
    if epilogue != 0 and y_f16 is None:
        y_f16 = torch.empty((M, N // 2 if epilogue == 1 else N), dtype=torch.float16, device=x.device)
    need = lib().dspark_gemm_i8_workspace(M, N, K)
    ws = (workspace or Workspace(x.device)).get(need)
    rc = lib().dspark_gemm_i8(ptr(x), M, K, ptr(w_biased), ptr(scale), N, epilogue, ptr(y_f32), ptr(y_f16), ptr(ws),
                              ws.numel(), stream_handle(stream))
    check(rc, "dspark_gemm_i8")
    return y_f32 if epilogue == 0 and y_f32 is not None else y_f16


def gemm_i8_g128(x, w_biased, gscale, epilogue=0, y_f32=None, y_f16=None, stream=None):
    """x fp16 [M][K] (M <= 16); w uint8 [N][K] biased; gscale fp16 [K/128][N] (per-128-column group scales)."""
    torch = _torch()
    M, K = x.shape
    N = w_biased.shape[0]
    if epilogue == 0 and y_f32 is None and y_f16 is None:
        y_f32 = torch.empty((M, N), dtype=torch.float32, device=x.device)
    rc = lib().dspark_gemm_i8_g128(ptr(x), M, K, ptr(w_biased), ptr(gscale), N, epilogue, ptr(y_f32), ptr(y_f16),
                                   stream_handle(stream))
    check(rc, "dspark_gemm_i8_g128")
    return y_f32, y_f16


def gemm_i8_g128_x8(x, w_biased, gscale, xscale=None, epilogue=0, y_f32=None, y_f16=None, stream=None):
    """The LFM3_X8 form of gemm_i8_g128: x fp16 [M][K] quantized per 16 columns on load (xscale None), or x the int8
    codes as integer-valued fp16 with xscale fp32 [M][K/16]."""
    torch = _torch()
    M, K = x.shape
    N = w_biased.shape[0]
    if epilogue == 0 and y_f32 is None and y_f16 is None:
        y_f32 = torch.empty((M, N), dtype=torch.float32, device=x.device)
    rc = lib().dspark_gemm_i8_g128_x8(ptr(x), ptr(xscale), M, K, ptr(w_biased), ptr(gscale), N, epilogue, ptr(y_f32),
                                      ptr(y_f16), stream_handle(stream))
    check(rc, "dspark_gemm_i8_g128_x8")
    return y_f32, y_f16


def g128_scales(packed, N, K):
    """The packer's scale rows (uint16 [N][SRow]) -> group-major [K/128][N] (host numpy)."""
    import numpy as np
    packed = np.ascontiguousarray(packed, dtype=np.uint16)
    out = np.empty((K // 128, N), dtype=np.uint16)
    check(lib().dspark_g128_scales(packed.ctypes.data_as(ctypes.c_void_p), N, K, out.ctypes.data_as(ctypes.c_void_p)),
          "dspark_g128_scales")
    return out


def head_argmax(x, w, y_f32=None, best=None, workspace=None, stream=None):
    torch = _torch()
    M, K = x.shape
    N = w.shape[0]
    if best is None:
        best = torch.empty(M, dtype=torch.int64, device=x.device)
    need = lib().dspark_head_argmax_workspace(M, N)
    ws = (workspace or Workspace(x.device)).get(need)
    rc = lib().dspark_head_argmax_f16(ptr(x), M, K, ptr(w), N, ptr(y_f32), ptr(best), ptr(ws), ws.numel(),
                                      stream_handle(stream))
    check(rc, "dspark_head_argmax_f16")
    return best


# ---------------------------------------------------------------- the full step (engine)
MAX_LAYERS = 64
MAX_TAPS = 8


class ModelDesc(ctypes.Structure):
    _fields_ = [("hidden", ctypes.c_int32), ("ffn", ctypes.c_int32), ("vocab", ctypes.c_int32),
                ("n_layers", ctypes.c_int32), ("layer_kind", ctypes.c_int32 * MAX_LAYERS),
                ("q_heads", ctypes.c_int32), ("kv_heads", ctypes.c_int32), ("head_dim", ctypes.c_int32),
                ("conv_kernel", ctypes.c_int32), ("window", ctypes.c_int32), ("rope_base", ctypes.c_float),
                ("rope_pairs", ctypes.c_int32), ("draft_layers", ctypes.c_int32), ("draft_ffn", ctypes.c_int32),
                ("block", ctypes.c_int32), ("max_drafts", ctypes.c_int32), ("crop_rows", ctypes.c_int32),
                ("markov_rank", ctypes.c_int32), ("n_taps", ctypes.c_int32), ("tap_layer", ctypes.c_int32 * MAX_TAPS),
                ("draft_window", ctypes.c_int32), ("ring_positions", ctypes.c_int32), ("mask_token", ctypes.c_int32),
                ("conf_bias", ctypes.c_float), ("conf_thr", ctypes.c_float), ("eps", ctypes.c_float),
                ("rope_base_swa", ctypes.c_float), ("rope_pairs_swa", ctypes.c_int32), ("conv_slots", ctypes.c_int32),
                ("kv_format", ctypes.c_int32), ("weight_format", ctypes.c_int32), ("x_format", ctypes.c_int32)]


class LaunchArgs(ctypes.Structure):
    _fields_ = [("a", ctypes.c_int32), ("anchor", ctypes.c_int32), ("budget", ctypes.c_int32), ("eos", ctypes.c_int32),
                ("rep", ctypes.c_float), ("rounds", ctypes.c_int32), ("ctx_new", ctypes.c_int32),
                ("ctx_pos", ctypes.c_int32), ("ctx_lo", ctypes.c_int32), ("force_m", ctypes.c_int32),
                ("tokens", ctypes.c_int32 * MT_MAX), ("max_drafts", ctypes.c_int32), ("miss", ctypes.c_int32),
                ("skip", ctypes.c_int32), ("conv_slot", ctypes.c_int32), ("ckpt_slot", ctypes.c_int32)]


class LaunchResult(ctypes.Structure):
    _fields_ = [("count", ctypes.c_int32), ("rounds", ctypes.c_int32), ("accepted", ctypes.c_int32),
                ("verified", ctypes.c_int32), ("boundary", ctypes.c_int32), ("ckpt_written", ctypes.c_int32),
                ("state", State), ("rounds_enqueued", ctypes.c_int32)]


_SIGS.update({
    "dspark_engine_create": (ctypes.c_int, [ctypes.POINTER(ModelDesc), ctypes.c_int32, ctypes.POINTER(ctypes.c_void_p)]),
    "dspark_engine_destroy": (None, [ctypes.c_void_p]),
    "dspark_engine_init_random": (ctypes.c_int, [ctypes.c_void_p, ctypes.c_uint64, ctypes.c_void_p]),
    "dspark_engine_tensor": (ctypes.c_int, [ctypes.c_void_p, ctypes.c_char_p, ctypes.POINTER(ctypes.c_void_p),
                                            ctypes.POINTER(ctypes.c_size_t)]),
    "dspark_engine_tensor_count": (ctypes.c_int, [ctypes.c_void_p]),
    "dspark_engine_tensor_name": (ctypes.c_char_p, [ctypes.c_void_p, ctypes.c_int32]),
    "dspark_engine_debug_layers": (ctypes.c_int, [ctypes.c_void_p, ctypes.c_int32]),
    "dspark_engine_prepare": (ctypes.c_int, [ctypes.c_void_p, ctypes.c_void_p]),
    "dspark_engine_round": (ctypes.c_int, [ctypes.c_void_p, ctypes.c_int32, ctypes.c_int32, ctypes.c_void_p]),
    "dspark_engine_launch": (ctypes.c_int, [ctypes.c_void_p, ctypes.POINTER(LaunchArgs), ctypes.c_void_p, ctypes.c_int32,
                                            ctypes.POINTER(LaunchResult), ctypes.c_void_p]),
    "dspark_engine_init_seen": (ctypes.c_int, [ctypes.c_void_p, ctypes.c_void_p, ctypes.c_int32, ctypes.c_float,
                                               ctypes.c_void_p]),
    "dspark_engine_capture_tap": (ctypes.c_int, [ctypes.c_void_p, ctypes.c_int32, ctypes.c_void_p, ctypes.c_int64,
                                                 ctypes.c_int32, ctypes.c_int32, ctypes.c_int32, ctypes.c_void_p]),
    "dspark_engine_project_prompt": (ctypes.c_int, [ctypes.c_void_p, ctypes.c_int32, ctypes.c_int32, ctypes.c_void_p]),
    "dspark_engine_conv_copy": (ctypes.c_int, [ctypes.c_void_p, ctypes.c_int32, ctypes.c_int32, ctypes.c_void_p]),
    "dspark_engine_trace": (ctypes.c_int, [ctypes.c_void_p, ctypes.c_int32, ctypes.c_void_p]),
    "dspark_engine_trace_read": (ctypes.c_int, [ctypes.c_void_p, ctypes.c_void_p, ctypes.c_int32,
                                                ctypes.POINTER(ctypes.c_int32)]),
})

TRACE_PHASES = {0: "begin", 1: "context", 2: "drafter", 3: "crop_head", 4: "markov", 5: "lm_head", 6: "commit"}
TRACE_VERIFY_LAYER = 16


def trace_phase_name(phase):
    return TRACE_PHASES.get(phase, f"verify_L{phase - TRACE_VERIFY_LAYER}")


def rope_table(base, pairs, head_dim, positions):
    """The RoPE table the engine builds (uint16 fp16 bits [positions][head_dim]: cos | sin), host code of the library."""
    import numpy as np
    out = np.empty((positions, head_dim), np.uint16)
    check(lib().dspark_rope_table(base, pairs, head_dim, positions, out.ctypes.data_as(ctypes.c_void_p)),
          "dspark_rope_table")
    return out


def model_desc(**kw):
    d = ModelDesc()
    d.conv_slots = 1
    for k, v in kw.items():
        if k in ("layer_kind", "tap_layer"):
            arr = getattr(d, k)
            for i, x in enumerate(v):
                arr[i] = int(x)
        else:
            setattr(d, k, v)
    return d


def c4_desc(block=16, vocab=65536):
    """16-layer LFM-style target (10 gated short-conv k=3 + 6 GQA 32/8/64), hidden 2048, FFN 8192,
    vocab 65536, int8 weights; 4-layer drafter proposing 16-token blocks."""
    kinds = [0, 0, 1, 0, 0, 1, 0, 0, 1, 0, 1, 0, 1, 0, 1, 0]
    return model_desc(hidden=2048, ffn=8192, vocab=vocab, n_layers=16, layer_kind=kinds, q_heads=32, kv_heads=8,
                      head_dim=64, conv_kernel=3, window=0, rope_base=1e6, rope_pairs=32, draft_layers=4,
                      draft_ffn=8192, block=block, max_drafts=block - 1, crop_rows=16384, markov_rank=256, n_taps=5,
                      tap_layer=[1, 4, 8, 11, 15], draft_window=2048, ring_positions=4096, mask_token=vocab - 1,
                      conf_bias=3.0, conf_thr=-0.4, eps=1e-5)


def ref_desc(block=9, max_drafts=7, vocab=128000, kv_format=1, weight_format=1, x_format=0):
    """The reference model's geometry (internal/model/engine.go:23-40; internal/model/dspark.go:22-41;
    cmd/pack/main.go:193, 329): 24 target layers in the reference order (13 gated short-conv k=7, 6 full and 5
    sliding-window-256 GQA attention layers, 16/4/128), hidden 2048, gated FFN 7680, vocab 128000; 3 attention-only
    drafter layers (FFN 7680) over 9-token blocks, 16384-row cropped head, Markov rank 256, taps {2, 6, 12, 18, 23},
    drafter window 2048, ring 4096. max_drafts follows the reference policy (7, or 3 from position 57344,
    generate.go:136). RoPE per layer kind as the reference builds it (engine.go:333-338): full attention and the
    drafter at base 1e6 with 32 rotating pairs, sliding layers at base 1e4 with 64. K/V in the reference's int8
    records (264 bytes per position and KV head, quantize_pair; engine.go:30-32, ops.hip:212-251) unless
    kv_format=0 (fp16 pages); int8 weights with the reference's per-128-column fp16 scales (weights.Pack,
    quant.go:66-104) unless weight_format=0 (one scale per row). x_format=1: the GEMM inputs as int8 per 16 columns, the
    reference's default build (LFM3_X8, kernels/dspark.hip:24-26); needs weight_format=1."""
    kinds = [0, 0, 1, 0, 2, 0, 1, 0, 2, 0, 1, 0, 2, 0, 1, 0, 2, 0, 1, 0, 2, 0, 1, 0]
    return model_desc(hidden=2048, ffn=7680, vocab=vocab, n_layers=24, layer_kind=kinds, q_heads=16, kv_heads=4,
                      head_dim=128, conv_kernel=7, window=256, rope_base=1e6, rope_pairs=32, rope_base_swa=1e4,
                      rope_pairs_swa=64, draft_layers=3,
                      draft_ffn=7680, block=block, max_drafts=max_drafts, crop_rows=16384, markov_rank=256, n_taps=5,
                      tap_layer=[2, 6, 12, 18, 23], draft_window=2048, ring_positions=4096, mask_token=vocab - 1,
                      conf_bias=3.0, conf_thr=-0.4, eps=1e-5, kv_format=kv_format, weight_format=weight_format,
                      x_format=x_format)


class Engine:
    """One model + one request's device buffers (dspark_engine_* in include/dspark.h)."""

    def __init__(self, desc, max_context):
        self.desc = desc
        self.max_context = max_context
        h = ctypes.c_void_p()
        check(lib().dspark_engine_create(ctypes.byref(desc), max_context, ctypes.byref(h)), "dspark_engine_create")
        self.h = h

    def close(self):
        if self.h:
            lib().dspark_engine_destroy(self.h)
            self.h = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass

    def tensor(self, name):
        p = ctypes.c_void_p()
        n = ctypes.c_size_t()
        check(lib().dspark_engine_tensor(self.h, name.encode(), ctypes.byref(p), ctypes.byref(n)), f"tensor {name}")
        return p.value, n.value

    def names(self):
        n = lib().dspark_engine_tensor_count(self.h)
        return [lib().dspark_engine_tensor_name(self.h, i).decode() for i in range(n)]

    def init_random(self, seed, stream=None):
        check(lib().dspark_engine_init_random(self.h, seed, stream_handle(stream)), "dspark_engine_init_random")

    def prepare(self, stream=None):
        check(lib().dspark_engine_prepare(self.h, stream_handle(stream)), "dspark_engine_prepare")

    def round(self, force_m=0, plan_a=0, stream=None):
        check(lib().dspark_engine_round(self.h, force_m, plan_a, stream_handle(stream)), "dspark_engine_round")

    def launch(self, a, anchor, budget=512, eos=-1, rep=1.0, rounds=32, ctx_new=0, ctx_pos=0, ctx_lo=0, force_m=0,
               tokens=(), max_out=1024, max_drafts=0, miss=0, skip=0, conv_slot=-1, ckpt_slot=-1, stream=None):
        """draftLaunch (dspark_engine_launch): returns (emitted tokens, LaunchResult)."""
        args = LaunchArgs()
        args.a, args.anchor, args.budget, args.eos, args.rep, args.rounds = a, anchor, budget, eos, rep, rounds
        args.ctx_new, args.ctx_pos, args.ctx_lo, args.force_m = ctx_new, ctx_pos, ctx_lo, force_m
        args.max_drafts, args.miss, args.skip, args.conv_slot, args.ckpt_slot = max_drafts, miss, skip, conv_slot, ckpt_slot
        for i, t in enumerate(tokens):
            args.tokens[i] = int(t)
        out = (ctypes.c_int32 * max_out)()
        res = LaunchResult()
        check(lib().dspark_engine_launch(self.h, ctypes.byref(args), out, max_out, ctypes.byref(res),
                                         stream_handle(stream)), "dspark_engine_launch")
        return list(out[:res.count]), res

    def init_seen(self, tokens, rep=1.0, stream=None):
        """InitSeen (dspark_engine_init_seen): the penalty mask = exactly `tokens`."""
        arr = (ctypes.c_int32 * max(1, len(tokens)))(*[int(t) for t in tokens])
        check(lib().dspark_engine_init_seen(self.h, arr, len(tokens), rep, stream_handle(stream)),
              "dspark_engine_init_seen")

    def capture_tap(self, slot, h, context, tap_from, stream=None):
        """captureTap (dspark_engine_capture_tap): h = fp16 device tensor [tokens][>= hidden] of positions
        context .. context + tokens - 1."""
        check(lib().dspark_engine_capture_tap(self.h, slot, ptr(h), h.stride(0), context, h.shape[0], tap_from,
                                              stream_handle(stream)), "dspark_engine_capture_tap")

    def project_prompt(self, first, end, stream=None):
        check(lib().dspark_engine_project_prompt(self.h, first, end, stream_handle(stream)),
              "dspark_engine_project_prompt")

    def debug_layers(self, enable=True):
        """Layer-boundary dumps into the tensor "debug_layers" (dspark_engine_debug_layers)."""
        check(lib().dspark_engine_debug_layers(self.h, int(enable)), "dspark_engine_debug_layers")

    def trace(self, enable=True, stream=None):
        """Phase tracing on (a fresh trace) or off for the rounds enqueued after this call."""
        check(lib().dspark_engine_trace(self.h, int(enable), stream_handle(stream)), "dspark_engine_trace")

    def trace_read(self, cap=65536):
        """The marks since tracing was turned on: list of (round, phase, clock ns)."""
        import numpy as np
        out = np.zeros(2 * cap, np.uint64)
        n = ctypes.c_int32()
        check(lib().dspark_engine_trace_read(self.h, out.ctypes.data_as(ctypes.c_void_p), cap, ctypes.byref(n)),
              "dspark_engine_trace_read")
        k = min(n.value, cap)
        return [(int(out[2 * i]) >> 32, int(out[2 * i]) & 0xFFFFFFFF, int(out[2 * i + 1])) for i in range(k)]

    def conv_copy(self, src, dst, stream=None):
        check(lib().dspark_engine_conv_copy(self.h, src, dst, stream_handle(stream)), "dspark_engine_conv_copy")

    # host <-> device copies of named tensors (plumbing for tests, loaders and benchmarks)
    def upload(self, name, array):
        import numpy as np
        ptr_, nbytes = self.tensor(name)
        a = np.ascontiguousarray(array)
        assert a.nbytes <= nbytes, (name, a.nbytes, nbytes)
        _hip().hipMemcpy(ctypes.c_void_p(ptr_), a.ctypes.data_as(ctypes.c_void_p), ctypes.c_size_t(a.nbytes), 1)

    def download(self, name, dtype, shape=None):
        import numpy as np
        ptr_, nbytes = self.tensor(name)
        out = np.empty(nbytes // np.dtype(dtype).itemsize, dtype=dtype)
        _hip().hipMemcpy(out.ctypes.data_as(ctypes.c_void_p), ctypes.c_void_p(ptr_), ctypes.c_size_t(out.nbytes), 2)
        if shape is not None:
            out = out[:int(np.prod(shape))].reshape(shape)
        return out

    def state(self):
        import numpy as np
        raw = self.download("state", np.int32)
        st = State()
        ctypes.memmove(ctypes.byref(st), raw.tobytes(), ctypes.sizeof(State))
        return st

    def set_state(self, **fields):
        import numpy as np
        st = State()
        for k, v in fields.items():
            if k == "tokens":
                for i, t in enumerate(v):
                    st.tokens[i] = int(t)
            else:
                setattr(st, k, int(v))
        self.upload("state", np.frombuffer(bytes(st), dtype=np.int32))


_hip_lib = None


def _hip():
    global _hip_lib
    if _hip_lib is None:
        _hip_lib = ctypes.CDLL("libamdhip64.so")
        _hip_lib.hipMemcpy.restype = ctypes.c_int
        _hip_lib.hipMemcpy.argtypes = [ctypes.c_void_p, ctypes.c_void_p, ctypes.c_size_t, ctypes.c_int]
    return _hip_lib
