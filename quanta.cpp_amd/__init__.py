"""Python binding of libquanta_hip.so (C-ABI in include/quanta_hip.h) for tests and benchmarks.

The directory name is not an importable identifier, so callers load this file by path under the module
name ``quanta_cpp_amd`` (see ``load_package``). Device memory and streams come from torch; every call
goes through the C-ABI into the gfx950 kernels. There is no CPU fallback: if the library is missing or
a call fails, a ``QHError`` is raised.
"""
from __future__ import annotations

import ctypes as C
import os
import subprocess

import numpy as np

HERE = os.path.dirname(os.path.abspath(__file__))
LIB_PATH = os.path.join(HERE, "libquanta_hip.so")
QK = 32
F32, F16, Q8_0, Q4_0 = 0, 1, 2, 3
Q8_0_PLANES = 16  # device-only nibble-plane layout of a Q8_0 head (qh_head_planes)
HEAD_MAX_TOPK = 256
NOALLOC_SCRATCH_BYTES = 4 << 20  # QH_NOALLOC_SCRATCH_BYTES
# status codes (quanta_hip.h)
OK, ERR_ARG, ERR_DTYPE, ERR_SHAPE, ERR_ALIGN, ERR_HIP, ERR_NOMEM, ERR_UNSUPPORTED = range(8)


class QHError(RuntimeError):
    pass


class qh_tensor(C.Structure):
    _fields_ = [("dtype", C.c_int32), ("rows", C.c_int32), ("cols", C.c_int32), ("data", C.c_void_p)]


class qh_head_query(C.Structure):
    _fields_ = [("top_k", C.c_int32), ("n_valid", C.c_int32), ("must", C.c_void_p), ("n_must", C.c_int32)]


class qh_head_stats(C.Structure):
    _fields_ = [("top1", C.c_int32), ("n_rows", C.c_int32), ("n_seeds", C.c_int32), ("n_cand", C.c_int32),
                ("n_must", C.c_int32), ("seed_tie", C.c_int32), ("tau", C.c_float), ("top1_logit", C.c_float)]


class qh_head_out(C.Structure):
    _fields_ = [("logits", C.c_void_p), ("coarse", C.c_void_p), ("upper", C.c_void_p), ("rows", C.c_void_p),
                ("stats", C.c_void_p)]


class qh_model_desc(C.Structure):
    _fields_ = [(n, C.c_int32) for n in ("vocab_size", "dim", "n_layers", "n_heads", "n_kv_heads", "head_dim",
                                         "ffn_dim", "ctx_len", "qkv_bias")] + [("rope_theta", C.c_float),
                                                                              ("norm_eps", C.c_float),
                                                                              ("flags", C.c_uint32),
                                                                              ("kv_f32", C.c_int32)]


class qh_decoder_state(C.Structure):
    _fields_ = [(n, C.c_void_p) for n in ("logits", "hidden", "xq", "xd", "stats", "top1_full", "pos", "n_out",
                                          "token", "kcache", "vcache", "status", "history", "history_len",
                                          "rng_state", "kcache_f32", "vcache_f32")]


class qh_sampler_params(C.Structure):
    """The reference's SamplerParams (sampler.h) without the seed."""
    _fields_ = [("temperature", C.c_float), ("top_k", C.c_int32), ("top_p", C.c_float), ("min_p", C.c_float),
                ("repeat_penalty", C.c_float), ("repeat_window", C.c_int32)]


def sampler_params(temperature=0.7, top_k=20, top_p=0.8, min_p=0.0, repeat_penalty=1.1, repeat_window=0):
    """qh_sampler_params with the reference's defaults (sampler.h: Qwen2.5-Instruct's generation config)."""
    return qh_sampler_params(temperature, top_k, top_p, min_p, repeat_penalty, repeat_window)


BEAM_MAX_BEAMS, BEAM_MAX_K = 256, 256  # QH_BEAM_MAX_*
KV8_BLOCK = 16  # QH_KV8_BLOCK: tokens that share a scale
KV8_NO_PAGES, KV8_BAD_LIST, KV8_SHARED = 1, 2, 4  # bits of KV8Cache.status


class qh_kv8_cache(C.Structure):
    _fields_ = [(n, C.c_void_p) for n in ("pages", "table", "lens", "refs", "status")] + [
        (n, C.c_int32) for n in ("n_layers", "n_pages", "page_tokens", "n_kv_heads", "head_dim", "n_seqs", "seq_pages")]


KV8_WHOLE, KV8_SHARES, KV8_TILES = 0, 1, 2  # qh_kv8_plan.kernel


class qh_kv8_plan(C.Structure):
    _fields_ = [(n, C.c_int32) for n in ("kernel", "rows", "waves", "splits", "launches")]


ROPE_PLAIN, ROPE_LINEAR, ROPE_BASE, ROPE_PARTS = range(4)  # qh_rope_desc.scaling


class qh_rope_desc(C.Structure):
    _fields_ = [("theta", C.c_double), ("rot_dim", C.c_int32), ("scaling", C.c_int32)] + [
        (n, C.c_double) for n in ("factor", "context", "low", "high")]


class qh_rope_rows(C.Structure):
    _fields_ = [("x", C.c_void_p), ("out", C.c_void_p), ("ld", C.c_int64), ("ldo", C.c_int64), ("n_heads", C.c_int32)]


STAGE_QKV, STAGE_ATTENTION, STAGE_O, STAGE_GATE_UP, STAGE_DOWN, STAGES_PER_LAYER = 0, 1, 2, 3, 4, 8
STAGE_FINAL_NORM, STAGE_HEAD, STAGE_PICK = 1 << 20, (1 << 20) + 1, (1 << 20) + 2

# Every symbol include/quanta_hip.h declares, in header order.
EXPORTS = ("qh_last_error", "qh_version", "qh_init", "qh_quant_bytes", "qh_tensor_bytes", "qh_validate_tensor",
           "qh_malloc", "qh_fault_alloc", "qh_free", "qh_memcpy_h2d", "qh_memcpy_d2h", "qh_memset", "qh_stream_sync",
           "qh_stream_create", "qh_stream_destroy",
           "qh_quantize_q8", "qh_matvec_q", "qh_matvec_ref", "qh_matmul_q", "qh_argmax_workspace_bytes", "qh_argmax",
           "qh_shortlist_workspace_bytes", "qh_shortlist_head", "qh_shortlist_head_noalloc",
           "qh_head_planes", "qh_shortlist_planes",
           "qh_sampler_state", "qh_sample", "qh_sample_workspace_bytes", "qh_sample_ws",
           "qh_kv8_page_bytes", "qh_kv8_reset", "qh_kv8_pages_workspace_bytes", "qh_kv8_resize", "qh_kv8_fork",
           "qh_kv8_reorder_workspace_bytes", "qh_kv8_reorder",
           "qh_kv8_compact", "qh_kv8_append", "qh_kv8_read", "qh_kv8_attention_workspace_bytes", "qh_kv8_attention",
           "qh_kv8_attention_plan",
           "qh_rmsnorm", "qh_rope_turns", "qh_rope", "qh_attention_workspace_bytes",
           "qh_attention", "qh_beam_workspace_bytes", "qh_beam_select",
           "qh_decoder_create",
           "qh_decoder_destroy",
           "qh_decoder_prefill", "qh_decoder_begin", "qh_decoder_step", "qh_decoder_views",
           "qh_decoder_set_prefill_stack", "qh_decoder_bind_kv8", "qh_decoder_step_timed",
           "qh_decoder_set_query",
           "qh_decoder_set_sampler")


def build() -> None:
    """Compile libquanta_hip.so for gfx950 (always recompiles what changed)."""
    subprocess.run(["make", "-s", "-C", HERE, "-j8", "lib"], check=True)


def _bind(lib):
    vp, i32, sz = C.c_void_p, C.c_int, C.c_size_t
    kv8 = C.POINTER(qh_kv8_cache)
    sig = {
        "qh_last_error": ([], C.c_char_p), "qh_version": ([], C.c_char_p), "qh_init": ([i32], i32),
        "qh_quant_bytes": ([i32, i32, i32], sz), "qh_tensor_bytes": ([i32, i32, i32], sz),
        "qh_validate_tensor": ([C.POINTER(qh_tensor)], i32), "qh_malloc": ([C.POINTER(vp), sz], i32),
        "qh_fault_alloc": ([i32], i32),
        "qh_free": ([vp], i32), "qh_memcpy_h2d": ([vp, vp, sz, vp], i32), "qh_memcpy_d2h": ([vp, vp, sz, vp], i32),
        "qh_memset": ([vp, i32, sz, vp], i32), "qh_stream_sync": ([vp], i32),
        "qh_stream_create": ([C.POINTER(vp)], i32), "qh_stream_destroy": ([vp], i32),
        "qh_quantize_q8": ([vp, i32, i32, vp, vp, vp], i32),
        "qh_matvec_q": ([vp, C.POINTER(qh_tensor), vp, vp, i32, i32, vp], i32),
        "qh_matvec_ref": ([vp, C.POINTER(qh_tensor), vp, i32, i32, vp], i32),
        "qh_matmul_q": ([vp, i32, C.POINTER(qh_tensor), vp, vp, i32, i32, i32, vp], i32),
        "qh_argmax_workspace_bytes": ([i32], sz),
        "qh_argmax": ([vp, i32, vp, vp, sz, vp], i32),
        "qh_shortlist_workspace_bytes": ([i32, i32, i32], sz),
        "qh_shortlist_head": ([C.POINTER(qh_tensor)] * 3 + [vp, vp, C.POINTER(qh_head_query), C.POINTER(qh_head_out),
                               vp, sz, vp], i32),
        "qh_shortlist_head_noalloc": ([C.POINTER(qh_tensor)] * 3 + [vp, vp, C.POINTER(qh_head_query),
                                       C.POINTER(qh_head_out), vp], i32),
        "qh_head_planes": ([C.POINTER(qh_tensor), vp, vp], i32),
        "qh_shortlist_planes": ([C.POINTER(qh_tensor), vp, vp, C.POINTER(qh_head_query), C.POINTER(qh_head_out), vp,
                                 sz, vp], i32),
        "qh_kv8_page_bytes": ([i32, i32, i32], sz),
        "qh_kv8_reset": ([kv8, vp], i32),
        "qh_kv8_pages_workspace_bytes": ([kv8], sz),
        "qh_kv8_resize": ([kv8, vp, vp, i32, vp, sz, vp], i32),
        "qh_kv8_fork": ([kv8, vp, vp, i32, i32, vp, sz, vp], i32),
        "qh_kv8_reorder_workspace_bytes": ([kv8], sz),
        "qh_kv8_reorder": ([kv8, vp, vp, i32, vp, sz, vp], i32),
        "qh_kv8_compact": ([kv8, vp, vp, sz, vp], i32),
        "qh_kv8_append": ([kv8, i32, vp, vp, i32, C.c_int64, C.c_int64, vp, vp, i32, i32, vp], i32),
        "qh_kv8_read": ([kv8, i32, vp, vp, i32, C.c_int64, C.c_int64, vp, vp, i32, i32, vp], i32),
        "qh_kv8_attention_workspace_bytes": ([kv8, i32, i32, i32], sz),
        "qh_kv8_attention": ([kv8, i32, vp, vp, i32, i32, C.c_int64, C.c_int64, vp, vp, i32, i32, i32, C.c_float, vp, sz,
                              vp], i32),
        "qh_kv8_attention_plan": ([kv8, i32, i32, i32, i32, C.POINTER(qh_kv8_plan)], i32),
        "qh_rmsnorm": ([vp, vp, vp, i32, C.c_int64, C.c_int64, i32, i32, C.c_double, vp, C.c_int64, vp, C.c_int64, vp, vp, vp],
                       i32),
        "qh_rope_turns": ([C.POINTER(qh_rope_desc), vp], i32),
        "qh_rope": ([vp, i32, i32, C.c_float, i32, C.POINTER(qh_rope_rows), C.POINTER(qh_rope_rows), i32, vp, i32, vp], i32),
        "qh_attention_workspace_bytes": ([i32] * 7, sz),
        "qh_attention": ([vp, vp, vp, vp, i32, i32, i32, i32] + [C.c_int64] * 4 + [vp, vp, i32, i32, i32, i32, C.c_float, vp, sz,
                          vp], i32),
        "qh_beam_workspace_bytes": ([i32, i32, i32, i32], sz),
        "qh_beam_select": ([vp, i32, C.c_int64, vp, i32, i32, i32, i32, vp, vp, vp, vp, sz, vp], i32),
        "qh_decoder_create": ([C.POINTER(qh_model_desc), C.POINTER(qh_tensor), i32, C.POINTER(vp)], i32),
        "qh_decoder_destroy": ([vp], i32),
        "qh_decoder_prefill": ([vp, vp, i32, i32, i32, vp], i32),
        "qh_decoder_begin": ([vp, i32, vp, i32, vp], i32),
        "qh_decoder_step": ([vp, i32, vp], i32),
        "qh_decoder_views": ([vp, C.POINTER(qh_decoder_state)], i32),
        "qh_decoder_set_prefill_stack": ([vp, i32], i32),
        "qh_decoder_bind_kv8": ([vp, kv8, i32], i32),
        "qh_decoder_step_timed": ([vp, i32, vp, vp, vp, i32, vp], i32),
        "qh_sampler_state": ([C.c_uint64], C.c_uint64),
        "qh_sample": ([vp, i32, vp, vp, vp, i32, C.POINTER(qh_sampler_params), vp, vp, vp], i32),
        "qh_sample_workspace_bytes": ([i32], C.c_size_t),
        "qh_sample_ws": ([vp, i32, vp, vp, vp, i32, C.POINTER(qh_sampler_params), vp, vp, vp, C.c_size_t, vp], i32),
        "qh_decoder_set_query": ([vp, C.POINTER(qh_sampler_params)], i32),
        "qh_decoder_set_sampler": ([vp, C.POINTER(qh_sampler_params), C.c_uint64], i32),
    }
    for name, (args, res) in sig.items():
        fn = getattr(lib, name)
        fn.argtypes, fn.restype = args, res
    return lib


_lib = None


def lib():
    """The loaded library; raises QHError when it has not been built."""
    global _lib
    if _lib is None:
        if not os.path.exists(LIB_PATH):
            raise QHError(f"{LIB_PATH} is missing: build it with `make -C {HERE}` (no CPU fallback exists)")
        _lib = _bind(C.CDLL(LIB_PATH))
    return _lib


def _check(rc: int) -> None:
    if rc != 0:
        raise QHError(f"status {rc}: {lib().qh_last_error().decode()}")


_torch_module = None


def _torch():
    global _torch_module
    if _torch_module is None:
        import torch
        _torch_module = torch
    return _torch_module


def _stream() -> int:
    """The current stream's handle, without building a Stream object for it (2 us of a 7 us call)."""
    torch = _torch()
    if torch.cuda.is_initialized():
        return torch._C._cuda_getCurrentRawStream(torch._C._cuda_getDevice())
    return torch.cuda.current_stream().cuda_stream


def _ptr(t) -> int:
    return t.data_ptr()


def init(device: int = 0) -> None:
    _check(lib().qh_init(device))


def tensor_bytes(dtype: int, rows: int, cols: int) -> int:
    return lib().qh_tensor_bytes(dtype, rows, cols)


class DeviceTensor:
    """A .qnt tensor resident in device memory (quants then scales, one allocation)."""

    def __init__(self, buf, dtype: int, rows: int, cols: int):
        self.buf, self.dtype, self.rows, self.cols = buf, dtype, rows, cols
        self.view = qh_tensor(dtype, rows, cols, buf.data_ptr())

    @staticmethod
    def upload(host: np.ndarray, dtype: int, rows: int, cols: int, device="cuda") -> "DeviceTensor":
        torch = _torch()
        host = np.ascontiguousarray(host).view(np.uint8).reshape(-1)
        buf = torch.from_numpy(host.copy()).to(device)
        return DeviceTensor(buf, dtype, rows, cols)

    def validate(self) -> None:
        _check(lib().qh_validate_tensor(C.byref(self.view)))


def quantize_q8(x, q=None, d=None):
    """x: f32 [n_tok][n] (or [n]) device tensor -> (q int8, d f32) device tensors."""
    torch = _torch()
    x2 = x if x.dim() == 2 else x.reshape(-1, x.shape[-1])
    n_tok, n = x2.shape
    if q is None:
        q = torch.empty((n_tok, n), dtype=torch.int8, device=x.device)
    if d is None:
        d = torch.empty((n_tok, n // QK), dtype=torch.float32, device=x.device)
    _check(lib().qh_quantize_q8(_ptr(x2), n_tok, n, _ptr(q), _ptr(d), _stream()))
    if q.shape == x.shape and d.dim() == x.dim() and d.shape[:-1] == x.shape[:-1] and d.shape[-1] == n // QK:
        return q, d
    shape = x.shape[:-1]
    return q.reshape(*shape, n), d.reshape(*shape, n // QK)


def matvec_q(W: DeviceTensor, xq, xd, out=None, r0: int = 0, r1: int | None = None):
    torch = _torch()
    if out is None:
        out = torch.zeros(W.rows, dtype=torch.float32, device=xq.device)
    r1 = W.rows if r1 is None else r1
    _check(lib().qh_matvec_q(_ptr(out), C.byref(W.view), _ptr(xq), _ptr(xd), r0, r1, _stream()))
    return out


def matvec_ref(W: DeviceTensor, x, out=None, r0: int = 0, r1: int | None = None):
    """W F32 / F16, x [cols] f32 (a device tensor) -> out [rows] with rows [r0, r1) written (matvec_ref)."""
    torch = _torch()
    if out is None:
        out = torch.zeros(W.rows, dtype=torch.float32, device=x.device)
    r1 = W.rows if r1 is None else r1
    _check(lib().qh_matvec_ref(_ptr(out), C.byref(W.view), _ptr(x), r0, r1, _stream()))
    return out


def matmul_q(W: DeviceTensor, xq, xd, out=None, r0: int = 0, r1: int | None = None, ldo: int | None = None):
    """xq [n][cols], xd [n][cols/32] -> out [n][ldo] with rows [r0, r1) written."""
    torch = _torch()
    n = xq.shape[0]
    ldo = W.rows if ldo is None else ldo
    if out is None:
        out = torch.zeros((n, ldo), dtype=torch.float32, device=xq.device)
    r1 = W.rows if r1 is None else r1
    _check(lib().qh_matmul_q(_ptr(out), ldo, C.byref(W.view), _ptr(xq), _ptr(xd), n, r0, r1, _stream()))
    return out


class Argmax:
    """Greedy token of a logits vector of up to `n` entries, with its own workspace."""

    def __init__(self, n: int, device="cuda"):
        torch = _torch()
        self.n = n
        self.ws = torch.empty(lib().qh_argmax_workspace_bytes(n), dtype=torch.uint8, device=device)
        self.index = torch.empty(1, dtype=torch.int32, device=device)

    def __call__(self, logits, n: int | None = None):
        n = logits.numel() if n is None else n
        if n > self.n:
            raise QHError(f"argmax over {n} entries, workspace sized for {self.n}")
        _check(lib().qh_argmax(_ptr(logits), n, _ptr(self.index), _ptr(self.ws), self.ws.numel(), _stream()))
        return self.index


def argmax(logits, n: int | None = None):
    return Argmax(logits.numel(), device=logits.device)(logits, n)


def sampler_state(seed: int) -> int:
    """The generator state a reference Sampler constructed with a nonzero seed starts from."""
    return int(lib().qh_sampler_state(seed))


def sample(logits, params: qh_sampler_params, state, history=None, n_valid: int | None = None, head=None,
           ws=None):
    """One Sampler::sample draw on the device: returns the chosen id as a device int32 tensor of one element.
    state: device uint64 tensor of one element (advanced in place); history: device int32 tensor or None;
    head: a ShortlistHead whose last call's row list and stats restrict the candidates; ws: a sample_workspace(n_valid)
    (qh_sample_ws), or None. Draws over full logits take a fraction of the time with one (151,936 ids, top-k 20: 20 us
    against 72), and more than 256 survivors of the top-k need one; calls that share one must not overlap."""
    torch = _torch()
    out = torch.empty(1, dtype=torch.int32, device=logits.device)
    nv = logits.numel() if n_valid is None else n_valid
    nh = 0 if history is None else int(history.numel())
    _check(lib().qh_sample_ws(_ptr(logits), nv, _ptr(head.rows) if head is not None else None,
                              _ptr(head.stats_dev) if head is not None else None, _ptr(history) if nh else None, nh,
                              C.byref(params), _ptr(state), _ptr(out), _ptr(ws) if ws is not None else None,
                              0 if ws is None else ws.numel(), _stream()))
    return out


def sample_workspace(n_valid: int, device="cuda"):
    """A device workspace for sample(..., ws=) over n_valid candidates."""
    torch = _torch()
    return torch.empty(int(lib().qh_sample_workspace_bytes(n_valid)), dtype=torch.uint8, device=device)


def head_planes(head8: DeviceTensor) -> DeviceTensor:
    """The nibble-plane layout of a Q8_0 head (qh_head_planes), a new device tensor of the same size."""
    torch = _torch()
    buf = torch.empty(tensor_bytes(Q8_0_PLANES, head8.rows, head8.cols), dtype=torch.uint8, device=head8.buf.device)
    _check(lib().qh_head_planes(C.byref(head8.view), _ptr(buf), _stream()))
    return DeviceTensor(buf, Q8_0_PLANES, head8.rows, head8.cols)


class ShortlistHead:
    """Device-resident Exact Shortlist Head: Q8_0 head, its Q4_0 copy and f16 block error bounds; or a nibble-plane
    head alone (head8 of dtype Q8_0_PLANES, head4 and err None: qh_shortlist_planes)."""

    def __init__(self, head8: DeviceTensor, head4: DeviceTensor | None, err: DeviceTensor | None, top_k: int = 1):
        torch = _torch()
        self.head8, self.head4, self.err = head8, head4, err
        self.V, self.D = head8.rows, head8.cols
        self.top_k = top_k
        nbytes = lib().qh_shortlist_workspace_bytes(self.V, self.D, top_k)
        if nbytes == 0:
            raise QHError(f"unsupported shortlist shape/top_k: {self.V} x {self.D}, k={top_k}")
        dev = head8.buf.device
        self.ws = torch.zeros(nbytes, dtype=torch.uint8, device=dev)
        self.logits = torch.empty(self.V, dtype=torch.float32, device=dev)
        self.coarse = torch.empty(self.V, dtype=torch.float32, device=dev)
        self.upper = torch.empty(self.V, dtype=torch.float32, device=dev)
        self.stats_dev = torch.zeros(8, dtype=torch.int32, device=dev)
        self._rows_cap = 0
        self.rows = None

    def __call__(self, xq, xd, n_valid: int = 0, must=None, top_k: int | None = None):
        """Enqueues one head call; results stay on the device (see `stats()`)."""
        torch = _torch()
        k = self.top_k if top_k is None else top_k
        if k != self.top_k:
            raise QHError("top_k differs from the one the workspace was sized for")
        n_must = 0 if must is None else int(must.numel())
        if self._rows_cap < self.V + n_must:
            self._rows_cap = self.V + n_must
            self.rows = torch.empty(self._rows_cap, dtype=torch.int32, device=self.logits.device)
        q = qh_head_query(k, n_valid, must.data_ptr() if n_must else None, n_must)
        o = qh_head_out(self.logits.data_ptr(), self.coarse.data_ptr(), self.upper.data_ptr(), self.rows.data_ptr(),
                        self.stats_dev.data_ptr())
        if self.head8.dtype == Q8_0_PLANES:
            _check(lib().qh_shortlist_planes(C.byref(self.head8.view), _ptr(xq), _ptr(xd), C.byref(q), C.byref(o),
                                             _ptr(self.ws), self.ws.numel(), _stream()))
            return
        _check(lib().qh_shortlist_head(C.byref(self.head8.view), C.byref(self.head4.view), C.byref(self.err.view),
                                       _ptr(xq), _ptr(xd), C.byref(q), C.byref(o), _ptr(self.ws),
                                       self.ws.numel(), _stream()))

    def stats(self) -> dict:
        raw = self.stats_dev.cpu().numpy()
        s = qh_head_stats.from_buffer_copy(raw.tobytes())
        return {f: getattr(s, f) for f, _ in qh_head_stats._fields_}


# ------------------------------------------------------------------------------------ 8-bit paged key / value cache

class KV8Cache:
    """A key / value cache in 8 bits for many sequences, in pages that they may share (qh_kv8_*). State on the device:
    ``table`` [n_seqs][seq_pages], ``lens`` [n_seqs], ``refs`` [n_pages], ``status`` [1] (KV8_* bits) and ``pages``
    [n_layers][n_pages][page_bytes]. Calls run on the current stream of the cache's device and read their lists there.

    A batch's rows are the last tokens of its sequences: ``start`` (int32 [n + 1], on the device) gives each entry's rows,
    None one row each; ``seqs`` (int32 [n]) their sequences, None sequence b for entry b. So a step is: ``resize`` to the
    new lengths, then for each layer ``append`` the new rows and ``attention`` of their queries."""

    def __init__(self, n_layers: int, n_pages: int, page_tokens: int, n_kv_heads: int, head_dim: int, n_seqs: int,
                 seq_pages: int, device="cuda"):
        torch = _torch()
        page_bytes = lib().qh_kv8_page_bytes(page_tokens, n_kv_heads, head_dim)
        if page_bytes == 0:
            raise QHError(f"unsupported cache shape: pages of {page_tokens} tokens, {n_kv_heads} KV heads of {head_dim}")
        if min(n_layers, n_pages, n_seqs, seq_pages) < 1:
            raise QHError(f"{n_layers} layers of {n_pages} pages, {n_seqs} sequences of {seq_pages} pages")
        self.n_layers, self.n_pages, self.page_tokens = n_layers, n_pages, page_tokens
        self.n_kv_heads, self.head_dim, self.n_seqs, self.seq_pages = n_kv_heads, head_dim, n_seqs, seq_pages
        self.pages = torch.empty((n_layers, n_pages, page_bytes), dtype=torch.uint8, device=device)
        self.device = self.pages.device
        self.table = torch.empty((n_seqs, seq_pages), dtype=torch.int32, device=device)
        self.lens = torch.empty(n_seqs, dtype=torch.int32, device=device)
        self.refs = torch.empty(n_pages, dtype=torch.int32, device=device)
        self.status = torch.empty(1, dtype=torch.int32, device=device)
        self.view = qh_kv8_cache(_ptr(self.pages), _ptr(self.table), _ptr(self.lens), _ptr(self.refs), _ptr(self.status),
                                 n_layers, n_pages, page_tokens, n_kv_heads, head_dim, n_seqs, seq_pages)
        self._ref = C.byref(self.view)
        # what every call looks up, kept here: the calls on a small batch take a few microseconds
        self._index = self.device.index
        self._int32, self._uint8, self._empty, self._empty_like = torch.int32, torch.uint8, torch.empty, torch.empty_like
        self._raw, self._float32 = torch._C, torch.float32
        self._append, self._read, self._attend = lib().qh_kv8_append, lib().qh_kv8_read, lib().qh_kv8_attention
        self._dtypes = {torch.float32: F32, torch.float16: F16}
        self._pages_bytes = lib().qh_kv8_pages_workspace_bytes(self._ref)
        # resize, fork and compact change the cache, so they are in order and can share a workspace
        self._pages_ws = torch.empty(self._pages_bytes, dtype=torch.uint8, device=device)
        self._pages_ptr = self._pages_ws.data_ptr()
        self._reorder_bytes = lib().qh_kv8_reorder_workspace_bytes(self._ref)
        self._reorder_ws = torch.empty(self._reorder_bytes, dtype=torch.uint8, device=device)
        self._attention_ws = {}  # bytes by (heads, entries, rows)
        self._scale = head_dim ** -0.5
        self.reset()

    def _here(self) -> int:
        """The current stream, on the cache's device."""
        raw = self._raw
        device = raw._cuda_getDevice()
        if device != self._index:
            raise QHError(f"the cache is on {self.device}, the current device is cuda:{device}")
        return raw._cuda_getCurrentRawStream(device)

    def _ints(self, t, n, what):
        if t.dtype is not self._int32 or t.device != self.device or not t.is_contiguous() or t.dim() != 1:
            raise QHError(f"{what} must be a contiguous int32 vector on {self.device}")
        if t.shape[0] != n:
            raise QHError(f"{what} has {t.shape[0]} entries, expected {n}")
        return t.data_ptr()

    def _batch(self, n_tok, start, seqs):
        """(start, seqs, n) of a batch as the C calls take them."""
        if start is not None:
            n = start.shape[0] - 1 if start.dim() == 1 else -1
            if n < 0:
                raise QHError("start has no entries")
            start = self._ints(start, n + 1, "start")
        else:
            n = n_tok
        if seqs is not None:
            return start, self._ints(seqs, n, "seqs"), n
        if n > self.n_seqs:
            raise QHError(f"{n} entries for {self.n_seqs} sequences")
        return start, None, n

    def _rows(self, t, heads, what):
        """(dtype, row stride) of rows [n_tok][heads][head_dim], or [n_tok][heads * head_dim], with contiguous heads."""
        dtype = self._dtypes.get(t.dtype)
        if dtype is None or t.device != self.device:
            raise QHError(f"{what} must be float32 or float16 on {self.device}")
        shape, stride, hd = t.shape, t.stride(), self.head_dim
        if len(shape) == 3 and shape[1] == heads and shape[2] == hd:
            ok = stride[2] == 1 and (heads == 1 or stride[1] == hd)
        elif len(shape) == 2 and shape[1] == heads * hd:
            ok = stride[1] == 1
        else:
            raise QHError(f"{what} is {tuple(shape)}, expected [rows][{heads}][{hd}]")
        if not ok:
            raise QHError(f"the heads of a row of {what} must be contiguous")
        return dtype, (stride[0] if shape[0] > 1 else heads * hd)

    def reset(self) -> None:
        """Every page free, every sequence empty, status 0."""
        _check(lib().qh_kv8_reset(self._ref, self._here()))

    def _pages_call(self, name, *args):
        _check(getattr(lib(), name)(self._ref, *args, self._pages_ptr, self._pages_bytes, self._here()))

    def resize(self, seqs, lens) -> None:
        """Sequence seqs[i] gets length lens[i] (int32 device vectors): pages past it are given back, missing ones taken."""
        n = seqs.numel()
        self._pages_call("qh_kv8_resize", self._ints(seqs, n, "seqs"), self._ints(lens, n, "lens"), n)

    def fork(self, src, dst, copy: bool = False) -> None:
        """Sequence dst[i] becomes a fork of src[i]: it shares its pages, or (copy) holds copies of them."""
        n = src.numel()
        self._pages_call("qh_kv8_fork", self._ints(src, n, "src"), self._ints(dst, n, "dst"), n, int(copy))

    def reorder(self, src, dst=None) -> None:
        """Sequence dst[i] (i itself without dst) takes what src[i] held before the call, all at once: src may name the same
        sequences, any number of times, and -1 leaves its dst empty. Pages are shared; `resize` then makes room."""
        n = src.numel()
        _check(lib().qh_kv8_reorder(self._ref, self._ints(src, n, "src"), None if dst is None else self._ints(dst, n, "dst"),
                                    n, self._reorder_ws.data_ptr() if self._reorder_bytes else None, self._reorder_bytes,
                                    self._here()))

    def compact(self):
        """Moves the pages in use to the front of the pool; returns how many there are (int32 device tensor [1])."""
        live = self._empty(1, dtype=self._int32, device=self.device)
        self._pages_call("qh_kv8_compact", _ptr(live))
        return live

    def append(self, layer: int, k, v, start=None, seqs=None) -> None:
        """Stores the rows k and v ([rows][n_kv_heads][head_dim], float32 or float16; views of a wider row are fine)."""
        dtype, ldk = self._rows(k, self.n_kv_heads, "k")
        dtype_v, ldv = self._rows(v, self.n_kv_heads, "v")
        rows = k.shape[0]
        if dtype != dtype_v or rows != v.shape[0]:
            raise QHError("k and v differ in dtype or rows")
        start, seqs, n = self._batch(rows, start, seqs)
        _check(self._append(self._ref, layer, k.data_ptr(), v.data_ptr(), dtype, ldk, ldv, start, seqs, n, rows,
                            self._here()))

    def read(self, layer: int, n_tok: int, start=None, seqs=None, dtype=None):
        """The stored values (k, v) of the batch's tokens, [n_tok][n_kv_heads][head_dim] of dtype (float32). Rows outside
        the entries are undefined."""
        heads, hd, dtype = self.n_kv_heads, self.head_dim, dtype or self._float32
        code = self._dtypes.get(dtype)
        if code is None:
            raise QHError("read gives float32 or float16")
        k = self._empty(n_tok, heads, hd, dtype=dtype, device=self.device)
        v = self._empty(n_tok, heads, hd, dtype=dtype, device=self.device)
        start, seqs, n = self._batch(n_tok, start, seqs)
        _check(self._read(self._ref, layer, k.data_ptr(), v.data_ptr(), code, heads * hd, heads * hd, start, seqs, n, n_tok,
                          self._here()))
        return k, v

    def attention(self, layer: int, q, start=None, seqs=None, causal: bool = True, scale: float | None = None, out=None):
        """Attention of the rows q ([rows][n_heads][head_dim]) over their sequences, each row up to its own position
        (causal) or over all of its sequence; scale: 1 / sqrt(head_dim). Rows outside the entries keep out's values (a new
        out's are undefined)."""
        rows = q.shape[0]
        heads = q.shape[1] if q.dim() == 3 else q.shape[-1] // self.head_dim
        dtype, ldq = self._rows(q, heads, "q")
        if out is None:
            out = self._empty_like(q) if q.is_contiguous() else self._empty(q.shape, dtype=q.dtype, device=self.device)
            ldo = heads * self.head_dim
        else:
            if out.shape != q.shape or out.dtype != q.dtype:
                raise QHError("out differs from q in shape or dtype")
            _, ldo = self._rows(out, heads, "out")
        start, seqs, n = self._batch(rows, start, seqs)
        need = self._attention_ws.get((heads, n, rows))
        if need is None:
            need = lib().qh_kv8_attention_workspace_bytes(self._ref, heads, n, rows)
            if len(self._attention_ws) > 4096:
                self._attention_ws.clear()
            self._attention_ws[heads, n, rows] = need
        # a tensor for each call: nothing of one call (or captured graph) is shared with the next
        ws = self._empty(need, dtype=self._uint8, device=self.device) if need else None
        _check(self._attend(self._ref, layer, q.data_ptr(), out.data_ptr(), dtype, heads, ldq, ldo, start, seqs, n, rows,
                            1 if causal else 0, self._scale if scale is None else scale, ws.data_ptr() if need else None,
                            need, self._here()))
        return out

    def attention_plan(self, heads: int, entries: int, rows: int, single: bool = False):
        """Which kernels `attention` takes for a batch of this shape (qh_kv8_plan; single: without start)."""
        plan = qh_kv8_plan()
        _check(lib().qh_kv8_attention_plan(self._ref, heads, entries, rows, int(single), C.byref(plan)))
        return plan


# ------------------------------------------------------------------------------- rows of a step of many sequences

# What these calls look up is kept short: on a few rows they take a few microseconds, most of them here.

def _here(t) -> int:
    """The current stream, on the device of a call's tensor t, which has to be the current one."""
    raw = _torch()._C
    device = raw._cuda_getDevice()
    if t.get_device() != device:
        raise QHError(f"the tensors are on {t.device}, the current device is cuda:{device}")
    return raw._cuda_getCurrentRawStream(device)


def _dtype_of(t, what) -> int:
    torch, dtype = _torch(), t.dtype
    if dtype is torch.float32:
        return F32
    if dtype is torch.float16:
        return F16
    raise QHError(f"{what} is {dtype}, expected float32 or float16")


def _like(t, shape, other, what):
    """Checks that a tensor has this shape and another's dtype and device."""
    if t.shape != shape or t.dtype is not other.dtype or t.get_device() != other.get_device():
        raise QHError(f"{what} is {tuple(t.shape)} {t.dtype} on {t.device}, expected {tuple(shape)} {other.dtype} on "
                      f"{other.device}")


def _row_stride(t, what) -> int:
    """Elements from row to row of a matrix with contiguous rows."""
    shape, stride = t.shape, t.stride()
    if len(shape) != 2 or (shape[1] > 1 and stride[1] != 1):
        raise QHError(f"{what} must be a matrix with contiguous rows")
    return stride[0] if shape[0] > 1 else shape[1]


def _rmsnorm(x, w, eps, residual, sum, out, q, d):
    torch = _torch()
    dtype, ldx, shape = _dtype_of(x, "x"), _row_stride(x, "x"), x.shape
    rows, n = shape
    stream = _here(x)
    if w.dtype is not torch.float32 or w.shape != (n,) or not w.is_contiguous() or w.get_device() != x.get_device():
        raise QHError(f"w must be a contiguous float32 vector of {n} on {x.device}")
    ldr = lds = ldy = n
    pr = ps = py = None
    if residual is not None:
        _like(residual, shape, x, "residual")
        ldr, pr = _row_stride(residual, "residual"), residual.data_ptr()
        if sum is None:
            sum = _new_like(x)
        else:
            _like(sum, shape, x, "sum")
            lds = _row_stride(sum, "sum")
        ps = sum.data_ptr()
    elif sum is not None:
        raise QHError("sum without residual")
    if q is None:
        if out is None:
            out = _new_like(x)
        else:
            _like(out, shape, x, "out")
            ldy = _row_stride(out, "out")
        py = out.data_ptr()
    rc = (_lib or lib()).qh_rmsnorm(x.data_ptr(), pr, w.data_ptr(), dtype, ldx, ldr, rows, n, eps, ps, lds, py, ldy,
                                    None if q is None else q.data_ptr(), None if d is None else d.data_ptr(), stream)
    if rc:
        _check(rc)
    return sum, out


def _new_like(t):
    """A new contiguous tensor of t's shape and dtype."""
    torch = _torch()
    return torch.empty_like(t, memory_format=torch.contiguous_format)


def rmsnorm(x, w, eps: float = 1e-6, residual=None, sum=None, out=None):
    """Root-mean-square norm of the rows x [rows][n] (float32 or float16; views of wider rows are fine) with weight w
    (float32 [n]) -> out. With residual: (sum, out), where sum = x + residual is what is normalized; sum may be x or
    residual itself (in place). See qh_rmsnorm."""
    sum, out = _rmsnorm(x, w, eps, residual, sum, out, None, None)
    return out if residual is None else (sum, out)


def rmsnorm_q8(x, w, eps: float = 1e-6, residual=None, sum=None):
    """The same into the 8-bit blocks that the quantized matmuls take: (q, d), as quantize_q8 makes them of the normalized
    rows in float32; with residual (sum, q, d). n is a multiple of 32."""
    torch, shape = _torch(), x.shape
    if len(shape) != 2 or shape[1] % QK:
        raise QHError(f"x is {tuple(shape)}, expected [rows][a multiple of {QK}]")
    q = torch.empty_like(x, dtype=torch.int8, memory_format=torch.contiguous_format)
    d = torch.empty((shape[0], shape[1] // QK), dtype=torch.float32, device=x.device)
    sum, _ = _rmsnorm(x, w, eps, residual, sum, None, q, d)
    return (q, d) if residual is None else (sum, q, d)


class Rope:
    """Rotary positions of heads of head_dim, the first rot_dim dims of each (all by default) in pairs (i, i + rot_dim / 2),
    or (2 i, 2 i + 1) when interleaved. scaling: None, "linear", "base" or "parts" (qh_rope_desc), with factor and, by
    parts, context, low and high (the ramp between them is linear in a pair's turns, not in its index); magnitude: what
    cosines and sines are multiplied by. turns: a table of one's own in place of those (float64 [rot_dim / 2]: turns of 2 pi per
    position)."""

    def __init__(self, head_dim: int, rot_dim: int | None = None, interleaved: bool = False, theta: float = 1e6,
                 scaling: str | None = None, factor: float = 1.0, context: float = 0.0, low: float = 1.0, high: float = 32.0,
                 magnitude: float = 1.0, turns=None, device="cuda"):
        torch = _torch()
        self.head_dim, self.rot_dim = head_dim, head_dim if rot_dim is None else rot_dim
        self.interleaved, self.magnitude = int(bool(interleaved)), float(magnitude)
        if turns is None:
            kinds = {None: ROPE_PLAIN, "linear": ROPE_LINEAR, "base": ROPE_BASE, "parts": ROPE_PARTS}
            if scaling not in kinds:
                raise QHError(f"scaling {scaling!r} is none of {list(kinds)}")
            desc = qh_rope_desc(theta, self.rot_dim, kinds[scaling], factor, context, low, high)
            host = np.empty(max(self.rot_dim // 2, 1), np.float64)
            _check(lib().qh_rope_turns(C.byref(desc), host.ctypes.data))
            turns = torch.from_numpy(host)
        if turns.dtype is not torch.float64 or turns.numel() != self.rot_dim // 2:
            raise QHError(f"turns must be {self.rot_dim // 2} float64 values")
        self.turns = turns.reshape(-1).to(device).contiguous()
        self._table, self._index = self.turns.data_ptr(), self.turns.get_device()

    def _rows(self, x, out, what):
        hd, shape = self.head_dim, x.shape
        if len(shape) != 3 or shape[2] != hd or x.get_device() != self._index:
            raise QHError(f"{what} is {tuple(shape)} on {x.device}, expected [rows][heads][{hd}] on {self.turns.device}")
        ld = _head_stride(x, what)
        if out is None:
            out = _new_like(x)
            return out, qh_rope_rows(x.data_ptr(), out.data_ptr(), ld, shape[1] * hd, shape[1])
        _like(out, shape, x, f"{what}_out")
        return out, qh_rope_rows(x.data_ptr(), out.data_ptr(), ld, _head_stride(out, f"{what}_out"), shape[1])

    def __call__(self, q, k=None, *, pos, q_out=None, k_out=None):
        """The rows q and k ([rows][heads][head_dim], float32 or float16; views of one wider row are fine) turned by the
        positions pos (int32 [rows], on the device) -> (q', k'), or q' without k. q_out / k_out may be q / k (in place)."""
        torch, rows = _torch(), q.shape[0]
        stream = _here(q)
        if (pos.dtype is not torch.int32 or pos.shape != (rows,) or pos.get_device() != q.get_device() or
                not pos.is_contiguous()):
            raise QHError(f"pos must be a contiguous int32 vector of {rows} on {q.device}")
        dtype, b = _dtype_of(q, "q"), None
        q_out, a = self._rows(q, q_out, "q")
        if k is not None:
            if k.shape[0] != rows or k.dtype is not q.dtype:
                raise QHError("q and k differ in rows or dtype")
            k_out, b = self._rows(k, k_out, "k")
        rc = (_lib or lib()).qh_rope(self._table, self.rot_dim, self.interleaved, self.magnitude, self.head_dim, a, b, dtype,
                                     pos.data_ptr(), rows, stream)
        if rc:
            _check(rc)
        return q_out if k is None else (q_out, k_out)


def _head_stride(t, what) -> int:
    """Elements from row to row of [rows][heads][head_dim] with the heads of a row contiguous."""
    shape, stride = t.shape, t.stride()
    if len(shape) == 3:
        rows, heads, hd = shape
        if (stride[2] == 1 or hd == 1) and (stride[1] == hd or heads == 1) or rows * heads * hd == 0:
            return stride[0] if rows > 1 else heads * hd
    raise QHError(f"{what} is {tuple(shape)} with strides {stride}, expected [rows][heads][head_dim] with the heads of a row "
                  "contiguous")


def attention(q, k, v, start=None, kstart=None, causal: bool = True, scale: float | None = None, out=None):
    """Attention of packed prompts over their own keys and values (qh_attention): q [rows][heads][head_dim], k and v
    [keys][KV heads][head_dim] (float32 or float16; views of wider rows are fine). start (int32 [n + 1], on the device): the
    rows of each of n sequences, None: one sequence of all; kstart: their keys, None: the same rows. causal: the rows are
    each sequence's last positions; scale: 1 / sqrt(head_dim). Rows outside the sequences keep out's values (a new out's are
    undefined)."""
    torch = _torch()
    stream, dtype, ldq = _here(q), _dtype_of(q, "q"), _head_stride(q, "q")
    ldk, ldv = _head_stride(k, "k"), _head_stride(v, "v")
    rows, heads, hd = q.shape
    keys, kv, _ = k.shape
    _like(k, (keys, kv, hd), q, "k")
    _like(v, (keys, kv, hd), q, "v")
    dev = q.device
    if out is None:
        out, ldo = _new_like(q), heads * hd
    else:
        _like(out, q.shape, q, "out")
        ldo = _head_stride(out, "out")
    if start is None:
        if kstart is not None:
            raise QHError("kstart without start")
        start = torch.arange(2, dtype=torch.int32, device=dev) * rows
        if keys != rows:
            kstart = torch.arange(2, dtype=torch.int32, device=dev) * keys
    n = start.shape[0] - 1 if start.dim() == 1 else -1
    for t, what in ((start, "start"), (kstart, "kstart")):
        if t is not None and (t.dtype is not torch.int32 or t.shape != (n + 1,) or n < 0 or t.get_device() != q.get_device() or
                              not t.is_contiguous()):
            raise QHError(f"{what} must be a contiguous int32 vector of sequences + 1 on {dev}")
    L = _lib or lib()
    need = L.qh_attention_workspace_bytes(dtype, heads, kv, hd, n, rows, keys)
    # a tensor for each call: nothing of one call (or captured graph) is shared with the next
    ws = torch.empty(need, dtype=torch.uint8, device=dev) if need else None
    rc = L.qh_attention(q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), dtype, heads, kv, hd, ldq, ldk, ldv, ldo,
                        start.data_ptr(), None if kstart is None else kstart.data_ptr(), n, rows, keys, int(causal),
                        hd ** -0.5 if scale is None else scale, None if ws is None else ws.data_ptr(), need, stream)
    if rc:
        _check(rc)
    return out


def beam_select(logits, scores, beams: int, k: int, n_valid: int | None = None):
    """The k best continuations of each prompt's beams: logits [prompts * beams][vocabulary] (float32 or float16; views of
    wider rows are fine), scores float32 [prompts * beams] or None (0), n_valid: ids from it on do not count. Returns
    (parent, token, score), each [prompts][k], best first: the row that is continued, the id (both int32) and
    score + log-softmax (float32); -1, -1 and -inf where there are fewer candidates. The three are views of one tensor that also
    holds the call's workspace (up to a few KB a row): clone what is kept for long. See qh_beam_select."""
    torch = _torch()
    stream, dtype, ld = _here(logits), _dtype_of(logits, "logits"), _row_stride(logits, "logits")
    rows, n = logits.shape
    n_valid = n if n_valid is None else n_valid
    if beams < 1 or rows % beams or not 1 <= n_valid <= n:
        raise QHError(f"{rows} rows of {beams} beams, {n_valid} of {n} ids")
    if not 1 <= k <= BEAM_MAX_K:
        raise QHError(f"k {k} outside [1, {BEAM_MAX_K}]")
    if scores is not None and (scores.dtype is not torch.float32 or scores.shape != (rows,) or
                               scores.get_device() != logits.get_device() or not scores.is_contiguous()):
        raise QHError(f"scores must be a contiguous float32 vector of {rows} on {logits.device}")
    prompts, dev, L = rows // beams, logits.device, _lib or lib()
    need = L.qh_beam_workspace_bytes(dtype, prompts, beams, n_valid)
    # the results and the workspace in one tensor, a new one for each call: nothing of one call (or captured graph) is shared
    # with the next
    each, shape, strides = (prompts * k + 3) // 4 * 4, (prompts, k), (k, 1)
    held = torch.empty(3 * each + (need + 3) // 4, dtype=torch.int32, device=dev)
    at = held.data_ptr()
    rc = L.qh_beam_select(logits.data_ptr(), dtype, ld, None if scores is None else scores.data_ptr(), prompts, beams, n_valid,
                          k, at, at + 4 * each, at + 8 * each, at + 12 * each, need, stream)
    if rc:
        _check(rc)
    return (held.as_strided(shape, strides), held.as_strided(shape, strides, each),
            held.view(torch.float32).as_strided(shape, strides, 2 * each))


# ------------------------------------------------------------------------------------------------ decoder

LAYER_ORDER = ("input_layernorm.weight", "self_attn.q_proj.weight", "self_attn.k_proj.weight", "self_attn.v_proj.weight",
               "self_attn.o_proj.weight", "self_attn.q_proj.bias", "self_attn.k_proj.bias", "self_attn.v_proj.bias",
               "post_attention_layernorm.weight", "mlp.gate_proj.weight", "mlp.up_proj.weight",
               "mlp.down_proj.weight")


def _d2h(ptr, nbytes, dtype):
    out = np.empty(nbytes // np.dtype(dtype).itemsize, dtype)
    _check(lib().qh_memcpy_d2h(out.ctypes.data, C.c_void_p(ptr), nbytes, _stream()))
    return out


class Decoder:
    """The GPU-resident decoder (qh_decoder_*) over a .qnt tensor set (quanta_cpp_amd.qnt records), uploaded once.
    hp.tied_embeddings false takes lm_head.weight as the LM head, hp.flags carries FLAG_HADAMARD_DOWN, and kv_f32
    keeps an f32 KV cache (Model::load's kv_f16 = false, model.cpp:10, 96-104)."""

    def __init__(self, hp, tensors: dict, ctx_len: int | None = None, device="cuda", kv_f32: bool = False,
                 head_planes: bool = False):
        """head_planes: the Q8_0 LM head (the embedding when tied) is stored as nibble planes (qh_head_planes) in place
        of its Q8_0 form, and the shortlist head screens with the high plane: no head_q4 / head_err are uploaded (the
        scope's nibble-plane variant, zero extra memory)."""
        torch = _torch()
        self.hp = hp
        self.kv_f32 = bool(kv_f32)
        names = ["model.embed_tokens.weight", "model.norm.weight"]
        for l in range(hp.n_layers):
            names += [f"model.layers.{l}.{n}" for n in LAYER_ORDER]
        names += ["quanta.head_q4", "quanta.head_err"]
        tied = getattr(hp, "tied_embeddings", True)
        if not tied:
            names.append("lm_head.weight")
        lm_name = "model.embed_tokens.weight" if tied else "lm_head.weight"
        skip = {"quanta.head_q4", "quanta.head_err"} if head_planes else set()
        if head_planes and tensors[lm_name].dtype != Q8_0:
            raise QHError("head_planes needs a Q8_0 LM head")
        offs, total = [], 0
        for n in names:
            offs.append(total)
            if n in tensors and n not in skip:
                total += (tensors[n].data.size + 255) // 256 * 256
        self.buf = torch.empty(max(total, 256), dtype=torch.uint8, device=device)
        host = np.zeros(max(total, 256), np.uint8)
        for n, o in zip(names, offs):
            if n in tensors and n not in skip and not (head_planes and n == lm_name):
                host[o:o + tensors[n].data.size] = np.asarray(tensors[n].data)
        self.buf.copy_(torch.from_numpy(host))
        del host
        arr = (qh_tensor * len(names))()
        base = self.buf.data_ptr()
        for i, (n, o) in enumerate(zip(names, offs)):
            t = None if n in skip else tensors.get(n)
            arr[i] = qh_tensor(0, 0, 0, None) if t is None else qh_tensor(t.dtype, t.rows, t.cols, base + o)
            if head_planes and n == lm_name:  # the Q8_0 copy goes through a scratch upload into its slot as planes
                q8 = torch.from_numpy(np.ascontiguousarray(t.data).view(np.uint8).reshape(-1)).to(device)
                src = qh_tensor(Q8_0, t.rows, t.cols, q8.data_ptr())
                _check(lib().qh_head_planes(C.byref(src), C.c_void_p(base + o), _stream()))
                torch.cuda.synchronize()
                del q8
                arr[i] = qh_tensor(Q8_0_PLANES, t.rows, t.cols, base + o)
        self._tensors = arr
        self.desc = qh_model_desc(hp.vocab_size, hp.dim, hp.n_layers, hp.n_heads, hp.n_kv_heads, hp.head_dim,
                                  hp.ffn_dim, ctx_len or hp.max_seq, int(hp.qkv_bias), hp.rope_theta, hp.norm_eps,
                                  int(getattr(hp, "flags", 0)), int(self.kv_f32))
        h = C.c_void_p()
        _check(lib().qh_decoder_create(C.byref(self.desc), arr, len(names), C.byref(h)))
        self.h = h
        st = qh_decoder_state()
        _check(lib().qh_decoder_views(self.h, C.byref(st)))
        self.views = st
        self.tokens = None
        self.out = None

    def close(self):
        if getattr(self, "h", None):
            lib().qh_decoder_destroy(self.h)
            self.h = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass

    def set_prefill_stack(self, stack: int):
        """Prompt tokens per launch of each layer's norms, matmuls and (f16 cache) attention (32 = the reference's chunk;
        up to 1024), with bit-identical results; the device views are re-read (the work buffers move)."""
        _check(lib().qh_decoder_set_prefill_stack(self.h, stack))
        st = qh_decoder_state()
        _check(lib().qh_decoder_views(self.h, C.byref(st)))
        self.views = st

    def bind_kv8(self, cache: KV8Cache | None, seq: int = 0):
        """Later prefill and step calls keep their keys and values in sequence `seq` of an 8-bit cache and attend to it
        (qh_decoder_bind_kv8); None: the decoder's own cache again."""
        if cache is not None and cache.device != self.buf.device:
            raise QHError(f"the cache is on {cache.device}, the decoder on {self.buf.device}")
        _check(lib().qh_decoder_bind_kv8(self.h, None if cache is None else cache._ref, seq))
        self._kv8 = cache

    def prefill(self, tokens, pos0: int = 0, top_k: int = 1):
        torch = _torch()
        self.tokens = torch.as_tensor(np.ascontiguousarray(tokens, np.int32)).to(self.buf.device)
        _check(lib().qh_decoder_prefill(self.h, _ptr(self.tokens), self.tokens.numel(), pos0, top_k, _stream()))

    def begin(self, out_cap: int, top_k: int = 1):
        """Starts a greedy generation into an output list of out_cap tokens. The list's buffer is kept across calls
        with the same capacity, so a decode step captured in a graph after one begin() stays valid after the next."""
        torch = _torch()
        if self.out is None or self.out.numel() != out_cap:
            self.out = torch.zeros(out_cap, dtype=torch.int32, device=self.buf.device)
        else:
            self.out.zero_()
        _check(lib().qh_decoder_begin(self.h, top_k, _ptr(self.out), out_cap, _stream()))

    def step(self, top_k: int = 1):
        _check(lib().qh_decoder_step(self.h, top_k, _stream()))

    def set_query(self, params: qh_sampler_params | None):
        """Head queries as Session::head_query builds them from these sampler parameters (None: plain queries)."""
        self._qp = params
        _check(lib().qh_decoder_set_query(self.h, C.byref(params) if params is not None else None))

    def set_sampler(self, params: qh_sampler_params | None, seed: int = 1):
        """Tokens from Sampler::sample with these parameters and seed (None: the head's greedy top-1)."""
        self._sp = params
        _check(lib().qh_decoder_set_sampler(self.h, C.byref(params) if params is not None else None, seed))

    def history(self):
        """The token history (prompt ids since position 0, then each chosen id)."""
        n = int(_d2h(self.views.history_len, 4, np.int32)[0])
        return _d2h(self.views.history, 4 * n, np.int32) if n else np.zeros(0, np.int32)

    # host copies of the device state (synchronous)
    def stats(self) -> dict:
        raw = _d2h(self.views.stats, C.sizeof(qh_head_stats), np.uint8)
        st = qh_head_stats.from_buffer_copy(raw.tobytes())
        return {f: getattr(st, f) for f, _ in qh_head_stats._fields_}

    def hidden(self):
        return _d2h(self.views.hidden, 4 * self.hp.dim, np.float32)

    def hq(self):
        return _d2h(self.views.xq, self.hp.dim, np.int8), _d2h(self.views.xd, 4 * (self.hp.dim // QK), np.float32)

    def logits(self):
        return _d2h(self.views.logits, 4 * self.hp.vocab_size, np.float32)

    def top1_full(self) -> int:
        return int(_d2h(self.views.top1_full, 4, np.int32)[0])

    def status(self) -> int:
        """0, or bit 0: a step ran past the context (nothing was written); bit 1: a prompt token was out of range; bit 2: a
        bound 8-bit cache had no place for a forward's tokens."""
        return int(_d2h(self.views.status, 4, np.int32)[0])

    def kv(self, layer: int, n_pos: int):
        """The KV cache of one layer, positions [0, n_pos): (k, v) [n_pos][n_kv_heads*head_dim], as uint16 f16 bits,
        or float32 with kv_f32."""
        kvd = self.hp.n_kv_heads * self.hp.head_dim
        ctx = self.desc.ctx_len
        if self.kv_f32:  # the reference's layout, [ctx][kv_dim] per layer
            off = 4 * layer * ctx * kvd
            return (_d2h(self.views.kcache_f32 + off, 4 * n_pos * kvd, np.float32).reshape(n_pos, kvd),
                    _d2h(self.views.vcache_f32 + off, 4 * n_pos * kvd, np.float32).reshape(n_pos, kvd))
        # K is stored in chunks of 8 dimensions, [n_kv_heads][head_dim / 8][ctx][8]
        rawk = _d2h(self.views.kcache + 2 * layer * ctx * kvd, 2 * ctx * kvd, np.uint16)
        k = np.ascontiguousarray(rawk.reshape(kvd // 8, ctx, 8)[:, :n_pos].transpose(1, 0, 2).reshape(n_pos, kvd))
        # V is stored in blocks of 8 positions, [pos / 8][kv_dim][8]
        nblk = (n_pos + 7) // 8
        raw = _d2h(self.views.vcache + 2 * layer * ((ctx + 7) // 8 * 8) * kvd, 2 * nblk * 8 * kvd, np.uint16)
        v = raw.reshape(nblk, kvd, 8).transpose(0, 2, 1).reshape(nblk * 8, kvd)[:n_pos]
        return k, np.ascontiguousarray(v)

    def position(self) -> int:
        return int(_d2h(self.views.pos, 4, np.int32)[0])

    def outputs(self, n: int):
        return self.out[:n].cpu().numpy()
