"""ctypes bindings of libltx_amd.so (include/ltx_block.h, include/ltx_loader.h).

Device memory and streams come from PyTorch (plumbing only); every compute
call goes through the C ABI into the gfx950 kernels. There is no fallback:
a missing library or a failed call raises.
"""
from __future__ import annotations

import ctypes as C
import pathlib
import weakref

import numpy as np

from . import blockfmt as bf

PKG_DIR = pathlib.Path(__file__).resolve().parent.parent
LIB_PATH = PKG_DIR / "libltx_amd.so"

MODE_F16, MODE_BF16, MODE_F32 = 0, 1, 2
ATTN_Q_SCALED = 0x100  # ltx_op_attention mode flag
ATTN_C = float(np.float32(1.4426950408889634 / 11.313708498984761))  # log2(e) / sqrt(128)
MODES = {"f16": MODE_F16, "bf16": MODE_BF16, "f32": MODE_F32}
STAGES = ["norm_msa", "q1", "k1", "v1", "glog1", "attn1", "x_sa", "attn_in", "attn2", "x_ca", "ff_in", "ff_h",
          "glog2", "q2", "k2", "v2", "velocity"]

W_COUNT, Q_COUNT = 28, 10

_lib = None


class LtxError(RuntimeError):
    pass


def lib() -> C.CDLL:
    global _lib
    if _lib is not None:
        return _lib
    if not LIB_PATH.exists():
        raise LtxError(f"{LIB_PATH} is not built; run `python ltx-zml_amd/build.py`")
    L = C.CDLL(str(LIB_PATH))
    vp, i32, i64, u64 = C.c_void_p, C.c_int, C.c_int64, C.c_uint64
    sig = {
        "ltx_init": (i32, [i32, C.POINTER(vp)]),
        "ltx_destroy": (None, [vp]),
        "ltx_last_error": (C.c_char_p, [vp]),
        "ltx_version": (C.c_char_p, []),
        "ltx_block_weights_from_blob": (i32, [vp, vp, u64, C.c_char_p, i64, C.POINTER(vp)]),
        "ltx_block_weights_from_host": (i32, [vp, C.POINTER(vp), C.POINTER(vp), C.POINTER(vp), i32, C.POINTER(vp)]),
        "ltx_block_weights_from_blob_async": (i32, [vp, vp, u64, C.c_char_p, i64, vp, vp, C.POINTER(vp)]),
        "ltx_block_weights_free": (None, [vp, vp]),
        "ltx_block_weights_bytes": (u64, [vp]),
        "ltx_block_forward": (i32, [vp, vp, vp, vp, i32, vp, vp, i32, vp, vp, vp, i32, vp, i32, vp]),
        "ltx_block_graph_create": (i32, [vp, vp, vp, vp, i32, vp, vp, i32, vp, vp, vp, i32, vp, i32, C.POINTER(vp)]),
        "ltx_block_graph_launch": (i32, [vp, vp]),
        "ltx_block_graph_destroy": (None, [vp]),
        "ltx_block_stage": (i32, [vp, i32, C.POINTER(vp), C.POINTER(u64)]),
        "ltx_range_count": (i32, [vp, vp, C.POINTER(u64), i32]),
        "ltx_op_linear_q8": (i32, [vp, vp, vp, vp, i32, vp, vp, i32, i32, i32, i32, i32, i32, vp]),
        "ltx_op_linear_q8_noalloc": (i32, [vp, vp, vp, vp, i32, vp, vp, i32, i32, i32, i32, i32, i32, vp]),
        "ltx_op_attention": (i32, [vp, vp, vp, vp, vp, vp, i32, i32, i32, vp]),
        "ltx_op_linear_q4": (i32, [vp, vp, vp, vp, i32, vp, vp, i32, i32, i32, i32, i32, i32, vp]),
        "ltx_op_mx4_quantise": (i32, [vp, vp, i64, vp, vp, i32, i32, i32, vp]),
        "ltx_op_mx4_values": (i32, [vp, vp, vp, vp, i64, i32, i32, i32, vp]),
        "ltx_op_linear_mx4": (i32, [vp, vp, vp, vp, vp, vp, vp, i32, i32, i32, i32, i32, i32, vp]),
        "ltx_rope_create": (i32, [vp, i32, i32, vp, vp, vp, C.POINTER(vp)]),
        "ltx_rope_create_grid": (i32, [vp, C.POINTER(vp)]),
        "ltx_rope_free": (None, [vp, vp]),
        "ltx_op_qk_rope": (i32, [vp, vp, vp, i32, vp, i64, vp, vp, i64, i32, vp, i64, vp, vp, i64, i32, C.c_float, i32,
                                 vp]),
        "ltx_kv_cache_create": (i32, [vp, i32, i32, i32, C.POINTER(vp)]),
        "ltx_kv_cache_free": (None, [vp, vp]),
        "ltx_kv_cache_bytes": (u64, [vp]),
        "ltx_kv_cache_faults": (i32, [vp, vp, vp, C.POINTER(u64), i32]),
        "ltx_op_kv_write": (i32, [vp, vp, vp, vp, i64, vp, i64, vp]),
        "ltx_op_kv_read": (i32, [vp, vp, vp, vp, i64, vp, i64, vp]),
        "ltx_op_kv_attention_workspace": (i32, [vp, vp, vp, i32, C.POINTER(u64)]),
        "ltx_op_kv_attention": (i32, [vp, vp, vp, vp, i64, i32, i32, vp, vp, i64, vp, u64, vp]),
        "ltx_op_kv_attention_window_workspace": (i32, [vp, vp, vp, i32, i32, i32, i32, C.POINTER(u64)]),
        "ltx_op_kv_attention_window": (i32, [vp, vp, vp, vp, i64, i32, i32, i32, i32, vp, vp, i64, vp, u64, vp]),
        "ltx_op_dequant": (i32, [vp, vp, vp, i32, i32, i32, vp, vp, i32, vp]),
        "ltx_rope_tables": (i32, [vp, i32, vp, vp, i32]),
        "ltx_profile_enable": (i32, [vp, i32]),
        "ltx_profile_read": (i32, [vp, C.c_char_p, C.POINTER(C.c_double), C.POINTER(i32)]),
        "ltx_profile_reset": (i32, [vp]),
        "ltx_blob_open": (i32, [C.c_char_p, C.POINTER(vp)]),
        "ltx_blob_close": (None, [vp]),
        "ltx_blob_check_layout": (i32, [vp]),
        "ltx_blob_verify": (i32, [vp]),
        "ltx_blob_data": (vp, [vp, C.POINTER(u64)]),
        "ltx_blob_manifest_text": (C.c_char_p, [vp]),
        "ltx_blob_block_index": (i64, [vp]),
        "ltx_blob_find": (i32, [vp, C.c_char_p, C.POINTER(u64), C.POINTER(u64), C.c_char_p, i32]),
        "ltx_ring_create": (i32, [C.POINTER(vp), i32, C.POINTER(i32), i32, i32, u64, i32, C.POINTER(vp)]),
        "ltx_ring_static_check": (i32, [vp]),
        "ltx_ring_start": (i32, [vp]),
        "ltx_ring_acquire": (i32, [vp, i32, C.POINTER(vp), C.POINTER(u64)]),
        "ltx_ring_release": (i32, [vp, i32]),
        "ltx_ring_abort": (None, [vp]),
        "ltx_ring_stats": (i32, [vp, C.POINTER(u64), C.POINTER(u64), C.POINTER(u64), C.POINTER(u64)]),
        "ltx_ring_set_reader_delay_us": (i32, [vp, C.c_uint32]),
        "ltx_ring_destroy": (None, [vp]),
        "ltx_loader_last_error": (C.c_char_p, []),
        "ltx_sha256_hex": (i32, [vp, u64, C.c_char_p]),
        "ltx_core_weights_from_host": (i32, [vp, C.POINTER(vp), C.POINTER(vp)]),
        "ltx_core_weights_free": (None, [vp, vp]),
        "ltx_core_conditioning": (i32, [vp, vp, vp, i32, vp, vp, vp, vp, vp]),
        "ltx_core_patchify": (i32, [vp, vp, vp, i32, vp, vp]),
        "ltx_core_tail": (i32, [vp, vp, vp, vp, vp, i32, vp, vp]),
        "ltx_sched_sigmas": (i32, [i32, vp, C.POINTER(i32)]),
        "ltx_sched_noise_init": (i32, [vp, vp, vp, vp, vp, i32, i32, C.c_float, vp, vp]),
        "ltx_sched_step": (i32, [vp, vp, vp, vp, vp, vp, vp, i32, i32, C.c_float, C.c_float, vp, vp]),
        "ltx_denoise": (i32, [vp, C.POINTER(vp), i32, vp, vp, vp, vp, vp, i32, vp, i32, vp, vp, i32, vp, i32, i32,
                              vp]),
    }
    for name, (res, args) in sig.items():
        f = getattr(L, name)
        f.restype = res
        f.argtypes = args
    _lib = L
    return L


def _ptr(t) -> int | None:
    """Device/host address of a torch tensor or numpy array (None -> NULL)."""
    if t is None:
        return None
    if isinstance(t, np.ndarray):
        return t.ctypes.data
    return t.data_ptr()


def rope_tables(grid: np.ndarray, graph_layout: bool = True) -> tuple[np.ndarray, np.ndarray]:
    """Host f64 3D-RoPE tables (ltx/block_conformance.zig:87-126)."""
    grid = np.ascontiguousarray(grid, dtype=np.float32)
    T = grid.shape[1]
    shape = (T, 32, 64) if graph_layout else (32, T, 64)
    cos, sin = np.empty(shape, np.float32), np.empty(shape, np.float32)
    if not lib().ltx_rope_tables(_ptr(grid), T, _ptr(cos), _ptr(sin), int(graph_layout)):
        raise LtxError(lib().ltx_last_error(None).decode())
    return cos, sin


def sha256_hex(data: bytes) -> str:
    out = C.create_string_buffer(65)
    lib().ltx_sha256_hex(data, len(data), out)
    return out.value.decode()


def sched_sigmas(stage: int = 1) -> np.ndarray:
    """The distilled sigma list of a stage (ltx/scheduler.zig:15-18)."""
    n = C.c_int()
    if not lib().ltx_sched_sigmas(stage, None, C.byref(n)):
        raise LtxError(lib().ltx_last_error(None).decode())
    out = np.empty(n.value, np.float32)
    lib().ltx_sched_sigmas(stage, out.ctypes.data, C.byref(n))
    return out


class CoreWeights:
    """Device copy of the parts around the blocks (ltx/core_parts.zig:86-104)."""

    def __init__(self, ctx: "Context", handle: int):
        self.ctx, self.handle = ctx, handle

    def free(self):
        if self.handle:
            lib().ltx_core_weights_free(self.ctx.handle, self.handle)
            self.handle = None

    def __del__(self):
        try:
            self.free()
        except Exception:
            pass


class Weights:
    def __init__(self, ctx: "Context", handle: int):
        self.ctx, self.handle = ctx, handle

    @property
    def nbytes(self) -> int:
        return lib().ltx_block_weights_bytes(self.handle)

    def free(self):
        if self.handle:
            lib().ltx_block_weights_free(self.ctx.handle, self.handle)
            self.handle = None

    def __del__(self):
        try:
            self.free()
        except Exception:
            pass


class BlockGraph:
    """One block forward captured with its buffers bound (ltx_block_graph_*);
    launch() replays it on a stream."""

    def __init__(self, ctx: "Context", handle: int, keep: tuple):
        self.ctx, self.handle = ctx, handle
        self._keep = keep  # the bound tensors stay alive with the graph

    def launch(self, stream=None):
        st = stream.cuda_stream if stream is not None else _current_stream(self.ctx.device)
        self.ctx._check(lib().ltx_block_graph_launch(self.handle, st), "ltx_block_graph_launch")

    def free(self):
        if self.handle:
            lib().ltx_block_graph_destroy(self.handle)
            self.handle = None
            self._keep = ()

    def __del__(self):
        try:
            self.free()
        except Exception:
            pass


class _KvBatchArgs(C.Structure):  # ltx_kv_batch
    _fields_ = [("nseq", C.c_int), ("rows", C.c_int), ("row_start", C.c_void_p), ("kv_len", C.c_void_p),
                ("pages", C.c_void_p), ("max_pages", C.c_int)]


class KvBatch:
    """The sequences of a call on a KvCache (ltx_kv_batch): int32 device tensors
    kv_len [nseq], pages [nseq, max_pages] and row_start [nseq + 1] (None: one row
    a sequence), and the rows that the call's tensors have."""

    def __init__(self, kv_len, pages, row_start=None, rows: int | None = None):
        import torch
        nseq = kv_len.shape[0]
        for t, shape in ((kv_len, (nseq,)), (pages, (nseq, pages.shape[-1])), (row_start, (nseq + 1,))):
            if t is not None and (t.dtype != torch.int32 or tuple(t.shape) != shape or not t.is_contiguous()):
                raise LtxError(f"KvBatch: an int32 contiguous tensor of shape {shape} is needed")
        if rows is None and row_start is not None:
            raise LtxError("KvBatch: row_start needs rows")
        self.rows = nseq if rows is None else rows
        self.device = kv_len.get_device()
        if any(t is not None and t.get_device() != self.device for t in (pages, row_start)):
            raise LtxError("KvBatch: the tensors are on different devices")
        self._keep = (kv_len, pages, row_start)
        self.args = _KvBatchArgs(nseq, self.rows, _ptr(row_start), _ptr(kv_len), _ptr(pages), pages.shape[1])
        self.ref = C.addressof(self.args)


class KvCache:
    """A key/value cache in 4 bits (ltx_kv_cache)."""

    def __init__(self, ctx: "Context", handle: int, kv_heads: int, pages: int, mode: int):
        self.ctx, self.handle = ctx, handle
        self.kv_heads, self.pages, self.mode = kv_heads, pages, mode

    @property
    def nbytes(self) -> int:
        return lib().ltx_kv_cache_bytes(self.handle)

    def faults(self, reset: bool = True, stream=None) -> int:
        """Page indices outside the pool met since the last reset (ltx_kv_cache_faults)."""
        st = stream.cuda_stream if stream is not None else _current_stream(self.ctx.device)
        n = C.c_uint64()
        self.ctx._check(lib().ltx_kv_cache_faults(self.ctx.handle, self.handle, st, C.byref(n), int(reset)),
                        "ltx_kv_cache_faults")
        return n.value

    def free(self):
        if self.handle:
            lib().ltx_kv_cache_free(self.ctx.handle, self.handle)
            self.handle = None

    def __del__(self):
        try:
            self.free()
        except Exception:
            pass


class Rope:
    """What the pairs of q and k turn by (ltx_rope)."""

    def __init__(self, ctx: "Context", handle: int, heads: int, axes: int):
        self.ctx, self.handle = ctx, handle
        self.heads, self.axes = heads, axes

    def free(self):
        if self.handle:
            lib().ltx_rope_free(self.ctx.handle, self.handle)
            self.handle = None

    def __del__(self):
        try:
            self.free()
        except Exception:
            pass


class Context:
    """One device context (ltx_init). Not thread-safe."""

    def __init__(self, device: int = 0):
        h = C.c_void_p()
        if not lib().ltx_init(device, C.byref(h)):
            raise LtxError("ltx_init: " + lib().ltx_last_error(None).decode())
        self.handle = h.value
        self.device = device
        self._graphs = weakref.WeakSet()
        self._caches = weakref.WeakSet()
        self._ropes = weakref.WeakSet()

    def _check(self, ok: int, what: str):
        if not ok:
            raise LtxError(f"{what}: " + lib().ltx_last_error(self.handle).decode())

    def close(self):
        if self.handle:
            for g in list(self._graphs):  # graphs hold the context's workspace
                g.free()
            for k in list(self._caches) + list(self._ropes):
                k.free()
            lib().ltx_destroy(self.handle)
            self.handle = None

    # ---- weights ----
    def upload(self, bt: bf.BlockTensors) -> Weights:
        base = (C.c_void_p * W_COUNT)()
        for i, f in enumerate(bf.FIELDS):
            base[i] = bt.base[f].ctypes.data
        q8 = (C.c_void_p * Q_COUNT)()
        q8s = (C.c_void_p * Q_COUNT)()
        for i, qn in enumerate(bf.Q8_FIELDS):
            if qn in bt.q8:
                q8[i] = bt.q8[qn].ctypes.data
                q8s[i] = bt.q8s[qn].ctypes.data
        h = C.c_void_p()
        self._check(lib().ltx_block_weights_from_host(self.handle, base, q8, q8s, int(bt.scale_f16), C.byref(h)),
                    "ltx_block_weights_from_host")
        return Weights(self, h.value)

    def upload_blob(self, blob: bytes | np.ndarray, manifest_json: str, block: int) -> Weights:
        buf = np.frombuffer(blob, dtype=np.uint8) if not isinstance(blob, np.ndarray) else blob
        h = C.c_void_p()
        self._check(lib().ltx_block_weights_from_blob(self.handle, buf.ctypes.data, buf.nbytes,
                                                      manifest_json.encode(), block, C.byref(h)),
                    "ltx_block_weights_from_blob")
        return Weights(self, h.value)

    def upload_blob_async(self, mem_ptr: int, nbytes: int, manifest_json: str, block: int, reuse: Weights | None = None,
                          stream=None) -> Weights:
        """Streaming upload from `mem_ptr` (pinned host memory, e.g. a ring
        slot) on `stream`; returns at once. Keep the memory unchanged until
        the stream passes this call."""
        st = stream.cuda_stream if stream is not None else _current_stream(self.device)
        h = C.c_void_p()
        self._check(lib().ltx_block_weights_from_blob_async(self.handle, mem_ptr, nbytes, manifest_json.encode(),
                                                            block, reuse.handle if reuse else None, st, C.byref(h)),
                    "ltx_block_weights_from_blob_async")
        return reuse if reuse is not None else Weights(self, h.value)

    # ---- forward ----
    def forward(self, w: Weights, x, tstab, tidx, ctx, pts2, cos, sin, y, mode: int = MODE_F16, stream=None):
        T, S, K = x.shape[0], ctx.shape[0], tstab.shape[0]
        st = stream.cuda_stream if stream is not None else _current_stream(self.device)
        self._check(lib().ltx_block_forward(self.handle, w.handle, _ptr(x), _ptr(tstab), K, _ptr(tidx), _ptr(ctx), S,
                                            _ptr(pts2), _ptr(cos), _ptr(sin), T, _ptr(y), mode, st),
                    "ltx_block_forward")
        return y

    def block_graph(self, w: Weights, x, tstab, tidx, ctx, pts2, cos, sin, y, mode: int = MODE_F16) -> BlockGraph:
        """The forward of ``forward`` with these tensors, captured once
        (ltx_block_graph_create); BlockGraph.launch() runs it."""
        T, S, K = x.shape[0], ctx.shape[0], tstab.shape[0]
        h = C.c_void_p()
        self._check(lib().ltx_block_graph_create(self.handle, w.handle, _ptr(x), _ptr(tstab), K, _ptr(tidx), _ptr(ctx),
                                                 S, _ptr(pts2), _ptr(cos), _ptr(sin), T, _ptr(y), mode, C.byref(h)),
                    "ltx_block_graph_create")
        g = BlockGraph(self, h.value, (w, x, tstab, tidx, ctx, pts2, cos, sin, y))
        self._graphs.add(g)
        return g

    def range_count(self, reset: bool = True, stream=None) -> int:
        """16-bit stores out of range since the last reset (ltx_range_count)."""
        st = stream.cuda_stream if stream is not None else _current_stream(self.device)
        n = C.c_uint64()
        self._check(lib().ltx_range_count(self.handle, st, C.byref(n), int(reset)), "ltx_range_count")
        return n.value

    def stage(self, name: str):
        import torch
        p, n = C.c_void_p(), C.c_uint64()
        self._check(lib().ltx_block_stage(self.handle, STAGES.index(name), C.byref(p), C.byref(n)), "ltx_block_stage")
        out = torch.empty(n.value, dtype=torch.uint8, device="cuda")
        torch.cuda.synchronize()
        _memcpy_dtod(out.data_ptr(), p.value, n.value)
        return out

    # ---- operators ----
    def linear_q8(self, a, q, s, bias, y, mode=MODE_F16, gelu=False, stream=None, noalloc=False):
        """noalloc: the entry point with its scratch in the library's static
        device array (ltx_op_linear_q8_noalloc)."""
        M, K = a.shape
        N = q.shape[0]
        import torch
        st = stream.cuda_stream if stream is not None else _current_stream(self.device)
        name = "ltx_op_linear_q8_noalloc" if noalloc else "ltx_op_linear_q8"
        self._check(getattr(lib(), name)(self.handle, _ptr(a), _ptr(q), _ptr(s), int(s.dtype == torch.float16),
                                         _ptr(bias), _ptr(y), int(y.dtype == torch.float32), M, N, K, int(gelu),
                                         mode, st), name)
        return y

    def attention(self, q, k, v, glog, out, lq, lkv, mode=MODE_F16, stream=None, q_scaled=False):
        """q_scaled: q already holds q * log2(e) / sqrt(128) (LTX_ATTN_Q_SCALED)."""
        st = stream.cuda_stream if stream is not None else _current_stream(self.device)
        m = mode | (ATTN_Q_SCALED if q_scaled else 0)
        self._check(lib().ltx_op_attention(self.handle, _ptr(q), _ptr(k), _ptr(v), _ptr(glog), _ptr(out), lq, lkv,
                                           m, st), "ltx_op_attention")
        return out

    def linear_q4(self, a, q, s, bias, y, mode=MODE_F16, gelu=False, stream=None):
        """a [M, K], q uint8 [N, K / 2] (two weights a byte), s [N, K / 128]."""
        import torch
        (M, K), N = a.shape, q.shape[0]
        if not (q.shape == (N, K // 2) and K % 128 == 0 and s.shape == (N, K // 128) and y.shape == (M, N)
                and (bias is None or bias.shape == (N,))):
            raise LtxError("linear_q4: the shapes do not fit")
        if not (a.get_device() == q.get_device() == s.get_device() == y.get_device() == self.device
                and (bias is None or bias.get_device() == self.device)):
            raise LtxError("linear_q4: tensors on the context's device are needed")
        if not (a.is_contiguous() and q.is_contiguous() and s.is_contiguous() and y.is_contiguous()
                and (bias is None or bias.is_contiguous())):
            raise LtxError("linear_q4: contiguous tensors are needed")
        x, f32, half = _torch_dtype(mode), torch.float32, torch.float16
        if not (a.dtype == x and q.dtype == torch.uint8 and (s.dtype == half or s.dtype == f32)
                and (y.dtype == x or y.dtype == f32) and (bias is None or bias.dtype == f32)):
            raise LtxError("linear_q4: the types do not fit the mode")
        st = stream.cuda_stream if stream is not None else _current_stream(self.device)
        self._check(lib().ltx_op_linear_q4(self.handle, _ptr(a), _ptr(q), _ptr(s), int(s.dtype == torch.float16),
                                           _ptr(bias), _ptr(y), int(y.dtype == torch.float32), M, N, K, int(gelu),
                                           mode, st), "ltx_op_linear_q4")
        return y

    # ---- microscaled 4-bit operands ----
    def mx4_quantise(self, x, q, s, mode=MODE_F16, stream=None):
        """x [rows, K] (rows may be strided) -> codes q uint8 [rows, K / 2] and scales s
        uint8 [K / 128, rows, 4], which it returns (ltx_op_mx4_quantise). Here and below
        torch's float4_e2m1fn_x2 and float8_e8m0fnu will do for codes and scales: the same
        bytes."""
        st = stream.cuda_stream if stream is not None else _current_stream(self.device)
        rows, K, ld = self._mx4_rows("mx4_quantise", x, q, s, mode)
        self._check(lib().ltx_op_mx4_quantise(self.handle, x.data_ptr(), ld, q.data_ptr(), s.data_ptr(), rows, K, mode, st),
                    "ltx_op_mx4_quantise")
        return q, s

    def mx4_values(self, q, s, y, mode=MODE_F16, stream=None):
        """What codes and scales stand for -> y [rows, K] (ltx_op_mx4_values)."""
        st = stream.cuda_stream if stream is not None else _current_stream(self.device)
        rows, K, ld = self._mx4_rows("mx4_values", y, q, s, mode)
        self._check(lib().ltx_op_mx4_values(self.handle, q.data_ptr(), s.data_ptr(), y.data_ptr(), ld, rows, K, mode, st),
                    "ltx_op_mx4_values")
        return y

    def linear_mx4(self, a, a_s, q, s, bias, y, mode=MODE_F16, gelu=False, stream=None):
        """a and a_s, q and s: M and N rows as mx4_quantise makes them, or a_s None and a at
        most 64 rows [M, K] of the mode's type (ltx_op_linear_mx4)."""
        (M, N), K, device = y.shape, 2 * q.shape[1], self.device
        x, f32, out = _torch_dtype(mode), _torch_dtype(MODE_F32), y.dtype
        _mx4_held("linear_mx4", q, s, N, K, device)
        if a_s is not None:
            _mx4_held("linear_mx4", a, a_s, M, K, device)
        elif not (a.shape == (M, K) and a.dtype == x and a.is_contiguous() and a.get_device() == device):
            raise LtxError(f"linear_mx4: a contiguous a {[M, K]} of the mode's type on the context's device is needed")
        if not (y.is_contiguous() and (out == x or out == f32) and y.get_device() == device):
            raise LtxError("linear_mx4: a contiguous y of the mode's type or f32 on the context's device is needed")
        if bias is not None and not (bias.shape == (N,) and bias.dtype == f32 and bias.is_contiguous()
                                     and bias.get_device() == device):
            raise LtxError(f"linear_mx4: bias must be f32 {[N]}, contiguous, on the context's device")
        st = stream.cuda_stream if stream is not None else _current_stream(device)
        self._check(lib().ltx_op_linear_mx4(self.handle, a.data_ptr(), _ptr(a_s), q.data_ptr(), s.data_ptr(), _ptr(bias),
                                            y.data_ptr(), int(out == f32), M, N, K, int(gelu), mode, st),
                    "ltx_op_linear_mx4")
        return y

    def _mx4_rows(self, name, x, q, s, mode):
        (rows, K), (ld, unit) = x.shape, x.stride()
        if x.dtype != _torch_dtype(mode) or unit != 1 or x.get_device() != self.device:
            raise LtxError(f"{name}: rows of the mode's type on the context's device are needed")
        _mx4_held(name, q, s, rows, K, self.device)
        return rows, K, ld if rows > 1 else K

    # ---- rotary positions on several axes ----
    def rope(self, freq, phase=None, axis=None, axes: int = 1) -> Rope:
        """freq, phase f64 and axis int32, host arrays [heads, 64] (ltx_rope_create)."""
        f = np.ascontiguousarray(freq, np.float64)
        if f.ndim != 2 or f.shape[1] != 64:
            raise LtxError("rope: freq must be [heads, 64]")
        p = None if phase is None else np.ascontiguousarray(phase, np.float64)
        a = np.zeros(f.shape, np.int32) if axis is None else np.asarray(axis)
        if a.shape != f.shape or (p is not None and p.shape != f.shape):
            raise LtxError("rope: phase and axis must have freq's shape")
        if not 1 <= axes <= 8 or not ((a >= 0) & (a < axes) & (a == np.floor(a))).all():
            raise LtxError("rope: axes must be 1 .. 8, axis whole numbers of 0 .. axes - 1")
        x = np.ascontiguousarray(a, np.int32)
        h = C.c_void_p()
        self._check(lib().ltx_rope_create(self.handle, f.shape[0], axes, _ptr(f), _ptr(p), _ptr(x), C.byref(h)),
                    "ltx_rope_create")
        r = Rope(self, h.value, f.shape[0], axes)
        self._ropes.add(r)
        return r

    def rope_grid(self) -> Rope:
        """The plan of this model's blocks (ltx_rope_create_grid)."""
        h = C.c_void_p()
        self._check(lib().ltx_rope_create_grid(self.handle, C.byref(h)), "ltx_rope_create_grid")
        r = Rope(self, h.value, 32, 3)
        self._ropes.add(r)
        return r

    def qk_rope(self, rope: Rope, pos, q, q_out, k=None, k_out=None, q_norm=None, k_norm=None, eps: float = 1e-6,
                mode=MODE_F16, stream=None):
        """q, q_out [rows, heads * 128] and k, k_out [rows, kv_heads * 128] (rows may be
        strided), pos f64 [rows, axes], norms f32 [heads * 128] or None (ltx_op_qk_rope)."""
        rows, dt, f32, device = q.shape[0], _torch_dtype(mode), _torch_dtype(MODE_F32), self.device
        if (k is None) != (k_out is None):
            raise LtxError("qk_rope: k and k_out belong together")

        def strides(x, y, w):  # of x and y, and the heads (a row's call costs a few us: each question once)
            shape, sx, sy = x.shape, x.stride(), y.stride()
            if not (len(shape) == 2 and shape == y.shape and shape[0] == rows and x.dtype == dt and y.dtype == dt
                    and sx[1] == 1 and sy[1] == 1):
                raise LtxError("qk_rope: rows of one shape and of the mode's type are needed")
            if shape[1] % 128:
                raise LtxError("qk_rope: rows of heads of 128 values are needed")
            if w is not None and not (w.shape == shape[1:] and w.dtype == f32 and w.is_contiguous()):
                raise LtxError("qk_rope: norm weights must be f32, one for each value of a row")
            if not (x.get_device() == device and y.get_device() == device and (w is None or w.get_device() == device)):
                raise LtxError("qk_rope: tensors on the context's device are needed")
            return *((sx[0], sy[0]) if rows > 1 else 2 * (shape[1],)), shape[1] // 128

        ql = strides(q, q_out, q_norm)
        kl = (0, 0, 0) if k is None else strides(k, k_out, k_norm)
        if not (pos.shape == (rows, rope.axes) and pos.is_floating_point() and pos.element_size() == 8 and pos.is_contiguous()
                and pos.get_device() == device):
            raise LtxError(f"qk_rope: contiguous f64 positions {[rows, rope.axes]} on the context's device are needed")
        st = stream.cuda_stream if stream is not None else _current_stream(device)
        self._check(lib().ltx_op_qk_rope(self.handle, rope.handle, pos.data_ptr(), rows, q.data_ptr(), ql[0], _ptr(q_norm),
                                         q_out.data_ptr(), ql[1], ql[2], _ptr(k), kl[0], _ptr(k_norm), _ptr(k_out), kl[1],
                                         kl[2], eps, mode, st), "ltx_op_qk_rope")

    # ---- the 4-bit key/value cache ----
    def kv_cache(self, kv_heads: int, pages: int, mode: int = MODE_F16) -> KvCache:
        h = C.c_void_p()
        self._check(lib().ltx_kv_cache_create(self.handle, mode, kv_heads, pages, C.byref(h)), "ltx_kv_cache_create")
        c = KvCache(self, h.value, kv_heads, pages, mode)
        self._caches.add(c)
        return c

    def kv_write(self, cache: KvCache, batch: KvBatch, k, v, stream=None):
        """k, v [rows, kv_heads * 128] (rows may be strided) -> the cache (ltx_op_kv_write)."""
        st = stream.cuda_stream if stream is not None else _current_stream(self.device)
        _rows("kv_write", batch, cache, cache.kv_heads, k, v)
        self._check(lib().ltx_op_kv_write(self.handle, cache.handle, batch.ref, _ptr(k), _ld(k), _ptr(v),
                                          _ld(v), st), "ltx_op_kv_write")

    def kv_read(self, cache: KvCache, batch: KvBatch, k, v, stream=None):
        """What the cache holds of the batch's rows -> k, v (ltx_op_kv_read)."""
        st = stream.cuda_stream if stream is not None else _current_stream(self.device)
        _rows("kv_read", batch, cache, cache.kv_heads, k, v)
        self._check(lib().ltx_op_kv_read(self.handle, cache.handle, batch.ref, _ptr(k), _ld(k), _ptr(v),
                                         _ld(v), st), "ltx_op_kv_read")

    def kv_attention_workspace(self, cache: KvCache, batch: KvBatch, heads: int) -> int:
        """Bytes of `work` for kv_attention with this batch's nseq, rows and max_pages."""
        n = C.c_uint64()
        self._check(lib().ltx_op_kv_attention_workspace(self.handle, cache.handle, batch.ref, heads, C.byref(n)),
                    "ltx_op_kv_attention_workspace")
        return n.value

    def kv_attention(self, cache: KvCache, batch: KvBatch, q, out, heads: int, causal: bool = True, glog=None,
                     work=None, stream=None):
        """q, out [rows, heads * 128] (rows may be strided); glog [rows, heads] f32
        or None; work: a uint8 tensor of kv_attention_workspace bytes, or None
        (ltx_op_kv_attention)."""
        st = stream.cuda_stream if stream is not None else _current_stream(self.device)
        self._kv_attention_checks("kv_attention", cache, batch, q, out, heads, glog, work)
        self._check(lib().ltx_op_kv_attention(self.handle, cache.handle, batch.ref, _ptr(q), _ld(q), heads,
                                              int(causal), _ptr(glog), _ptr(out), _ld(out), _ptr(work),
                                              0 if work is None else work.numel() * work.element_size(), st),
                    "ltx_op_kv_attention")
        return out

    def kv_attention_window_workspace(self, cache: KvCache, batch: KvBatch, heads: int, window: int, sinks: int = 0,
                                      causal: bool = True) -> int:
        """Bytes of `work` for kv_attention_window with this batch's nseq, rows and max_pages."""
        n = C.c_uint64()
        window, sinks = _keys(window), _keys(sinks)
        self._check(lib().ltx_op_kv_attention_window_workspace(self.handle, cache.handle, batch.ref, heads, int(causal),
                                                               window, sinks, C.byref(n)),
                    "ltx_op_kv_attention_window_workspace")
        return n.value

    def kv_attention_window(self, cache: KvCache, batch: KvBatch, q, out, heads: int, window: int, sinks: int = 0,
                            causal: bool = True, glog=None, work=None, stream=None):
        """kv_attention to the last `window` of the keys that a row would see and the first
        `sinks` (ltx_op_kv_attention_window)."""
        st = stream.cuda_stream if stream is not None else _current_stream(self.device)
        self._kv_attention_checks("kv_attention_window", cache, batch, q, out, heads, glog, work)
        window, sinks = _keys(window), _keys(sinks)
        self._check(lib().ltx_op_kv_attention_window(self.handle, cache.handle, batch.ref, _ptr(q), _ld(q), heads,
                                                     int(causal), window, sinks, _ptr(glog), _ptr(out), _ld(out),
                                                     _ptr(work), 0 if work is None else work.numel() * work.element_size(),
                                                     st), "ltx_op_kv_attention_window")
        return out

    def _kv_attention_checks(self, name, cache, batch, q, out, heads, glog, work):
        _rows(name, batch, cache, heads, q, out)
        if glog is not None and not (glog.shape == (batch.rows, heads) and glog.is_contiguous()
                                     and glog.dtype == _torch_dtype(MODE_F32)
                                     and glog.get_device() == self.device):
            raise LtxError(f"{name}: glog must be f32 [rows, heads] on the context's device")
        if work is not None and not (work.is_contiguous() and work.get_device() == self.device):
            raise LtxError(f"{name}: work must be contiguous, on the context's device")

    def dequant(self, q, s, out32, out16, mode=MODE_F16, stream=None):
        import torch
        N, K = q.shape
        st = stream.cuda_stream if stream is not None else _current_stream(self.device)
        self._check(lib().ltx_op_dequant(self.handle, _ptr(q), _ptr(s), int(s.dtype == torch.float16), N, K,
                                         _ptr(out32), _ptr(out16), mode, st), "ltx_op_dequant")

    # ---- parts around the blocks and the scheduler ----
    def upload_core(self, tensors: dict) -> CoreWeights:
        """tensors: field -> numpy array in CORE_SPECS order (bf16 bits as
        uint16, fsst f32), e.g. conditioning.make_core()."""
        from .conditioning import CORE_FIELDS
        arrs = [np.ascontiguousarray(tensors[f]) for f in CORE_FIELDS]
        ptrs = (C.c_void_p * len(arrs))(*[a.ctypes.data for a in arrs])
        h = C.c_void_p()
        self._check(lib().ltx_core_weights_from_host(self.handle, ptrs, C.byref(h)), "ltx_core_weights_from_host")
        return CoreWeights(self, h.value)

    def conditioning(self, cw: CoreWeights, t, sigma, tstab, emb, pts2, stream=None):
        """t [K] f32, sigma [1] f32 (device) -> tstab [K, 9, D], emb [K, D], pts2 [2, D]."""
        st = stream.cuda_stream if stream is not None else _current_stream(self.device)
        self._check(lib().ltx_core_conditioning(self.handle, cw.handle, _ptr(t), t.shape[0], _ptr(sigma), _ptr(tstab),
                                                _ptr(emb), _ptr(pts2), st), "ltx_core_conditioning")

    def patchify(self, cw: CoreWeights, latent, x, stream=None):
        st = stream.cuda_stream if stream is not None else _current_stream(self.device)
        self._check(lib().ltx_core_patchify(self.handle, cw.handle, _ptr(latent), latent.shape[0], _ptr(x), st),
                    "ltx_core_patchify")
        return x

    def tail(self, cw: CoreWeights, x, emb, tidx, vel, stream=None):
        st = stream.cuda_stream if stream is not None else _current_stream(self.device)
        self._check(lib().ltx_core_tail(self.handle, cw.handle, _ptr(x), _ptr(emb), _ptr(tidx), x.shape[0], _ptr(vel),
                                        st), "ltx_core_tail")
        return vel

    def noise_init(self, clean, noise, maskk, tidx, noise_scale: float, out, stream=None):
        T, Cc = clean.shape
        st = stream.cuda_stream if stream is not None else _current_stream(self.device)
        self._check(lib().ltx_sched_noise_init(self.handle, _ptr(clean), _ptr(noise), _ptr(maskk), _ptr(tidx), T, Cc,
                                               float(noise_scale), _ptr(out), st), "ltx_sched_noise_init")
        return out

    def sched_step(self, x, vel, tk, maskk, tidx, clean, sigma: float, sigma_next: float, out, stream=None):
        T, Cc = x.shape
        st = stream.cuda_stream if stream is not None else _current_stream(self.device)
        self._check(lib().ltx_sched_step(self.handle, _ptr(x), _ptr(vel), _ptr(tk), _ptr(maskk), _ptr(tidx),
                                         _ptr(clean), T, Cc, float(sigma), float(sigma_next), _ptr(out), st),
                    "ltx_sched_step")
        return out

    def denoise(self, blocks: list, cw: CoreWeights, latent, clean, maskk, tidx, ctx, cos, sin, sigmas,
                mode: int = MODE_F16, stream=None):
        """Runs len(sigmas) - 1 steps over the resident blocks; latent [T, 128]
        is updated in place."""
        sig = np.ascontiguousarray(sigmas, np.float32)
        hs = (C.c_void_p * len(blocks))(*[b.handle for b in blocks])
        st = stream.cuda_stream if stream is not None else _current_stream(self.device)
        self._check(lib().ltx_denoise(self.handle, hs, len(blocks), cw.handle, _ptr(latent), _ptr(clean), _ptr(maskk),
                                      _ptr(tidx), maskk.shape[0], _ptr(ctx), ctx.shape[0], _ptr(cos), _ptr(sin),
                                      latent.shape[0], sig.ctypes.data, len(sig) - 1, mode, st), "ltx_denoise")
        return latent

    # ---- profiling ----
    def profile(self, enable: bool):
        self._check(lib().ltx_profile_enable(self.handle, int(enable)), "ltx_profile_enable")

    def profile_reset(self):
        self._check(lib().ltx_profile_reset(self.handle), "ltx_profile_reset")

    def profile_read(self, substr: str = "") -> tuple[float, int]:
        ms, n = C.c_double(), C.c_int()
        self._check(lib().ltx_profile_read(self.handle, substr.encode(), C.byref(ms), C.byref(n)), "ltx_profile_read")
        return ms.value, n.value


_DTYPES: dict = {}


def _torch_dtype(mode: int):
    if not _DTYPES:
        import torch
        _DTYPES.update({MODE_F16: torch.float16, MODE_BF16: torch.bfloat16, MODE_F32: torch.float32})
    return _DTYPES.get(mode)


def _ld(t) -> int:
    """Elements from a row to the next: the length of one that is alone, whose stride says nothing."""
    return t.stride(0) if t.shape[0] > 1 else t.shape[1]


def _rows(name: str, batch: KvBatch, cache: KvCache, heads: int, *tensors):
    """Tensors [rows, heads * 128] of the cache's type, values of a row next to each other."""
    shape, dt, device = (batch.rows, heads * 128), _torch_dtype(cache.mode), cache.ctx.device
    if batch.device != device:
        raise LtxError(f"{name}: a batch on the context's device is needed")
    for t in tensors:
        if t.get_device() != device:
            raise LtxError(f"{name}: tensors on the context's device are needed")
        if t.shape != shape or t.dtype != dt or t.stride(1) != 1:
            raise LtxError(f"{name}: {list(shape)} tensors of the cache's type are needed")


def _keys(n: int) -> int:
    """A count of keys within 32 bits: no table holds more than 2^30, and less than 0 is refused."""
    return max(-1, min(n, 1 << 30))


def _mx4_bytes(t, own: str) -> bool:
    """Whether t is of plain bytes, or of torch's own type for the same bytes."""
    if t.element_size() != 1:
        return False
    if not t.is_floating_point():
        return True
    import torch
    return t.dtype == getattr(torch, own, None)


def _mx4_held(name: str, q, s, rows: int, K: int, device: int):
    """Codes [rows, K / 2] and scales [K / 128, rows, 4], uint8 or float4_e2m1fn_x2 and float8_e8m0fnu."""
    if K % 128:
        raise LtxError(f"{name}: K must be a multiple of 128")
    if not (q.shape == (rows, K // 2) and s.shape == (K // 128, rows, 4) and _mx4_bytes(q, "float4_e2m1fn_x2")
            and _mx4_bytes(s, "float8_e8m0fnu") and q.is_contiguous() and s.is_contiguous()):
        raise LtxError(f"{name}: contiguous tensors {[rows, K // 2]} and {[K // 128, rows, 4]} of uint8, or of torch's "
                       "float4_e2m1fn_x2 and float8_e8m0fnu, are needed")
    if not q.get_device() == s.get_device() == device:
        raise LtxError(f"{name}: tensors on the context's device are needed")


def _current_stream(device: int) -> int:
    """The handle of a device's current stream."""
    import torch
    try:  # without a Stream object: 0.2 us, against 3 us
        return torch._C._cuda_getCurrentRawStream(device)
    except AttributeError:  # not part of torch's public interface
        return torch.cuda.current_stream(device).cuda_stream


def _memcpy_dtod(dst: int, src: int, n: int):
    import torch
    # a uint8 view of the source allocation through torch's storage API is not
    # available for foreign pointers; use hipMemcpy from the HIP runtime.
    hip = C.CDLL("libamdhip64.so")
    hip.hipMemcpy.argtypes = [C.c_void_p, C.c_void_p, C.c_size_t, C.c_int]
    hip.hipMemcpy.restype = C.c_int
    rc = hip.hipMemcpy(dst, src, n, 3)  # hipMemcpyDeviceToDevice
    if rc != 0:
        raise LtxError(f"hipMemcpy failed ({rc})")
    torch.cuda.synchronize()
