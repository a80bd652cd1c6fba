"""Python host binding of the gfx950 token sampler (libgs_sampler.so).

Mirrors the reference interface of gguf-rs-cli's src/sampler.rs:

    set_seed(s)                                          src/sampler.rs:5
    sample(logits, temperature, top_k, top_p,
           rep_penalty, recent) -> int                   src/sampler.rs:35-36

with the same argument meaning, the same process-global LCG stream
(one draw per call iff temperature > 0) and errors where the reference
panics (NaN logits, empty logits with T > 0).  It adds the `Sampler`
object (construction = params + seed) and a batched entry over B rows of
device-resident logits.

The library must be built (gguf-rs-cli_amd/build.py).  There is no CPU
fallback: if the HIP library is missing, importing this module fails.
"""
import ctypes
import os

_HERE = os.path.dirname(os.path.abspath(__file__))
LIB_PATH = os.path.join(_HERE, "libgs_sampler.so")

GS_OK = 0
GS_ERR_INVALID = -1
GS_ERR_EMPTY = -2
GS_ERR_NAN = -3
GS_ERR_HIP = -5
GS_ERR_NOMEM = -6
GS_ERR_UNSUPPORTED = -7
_ERRNAMES = {
    GS_ERR_INVALID: "invalid argument",
    GS_ERR_EMPTY: "empty logits (reference panics at pairs[0], src/sampler.rs:53)",
    GS_ERR_NAN: "NaN logit (reference panics in partial_cmp().unwrap(), src/sampler.rs:17,45)",
    GS_ERR_HIP: "HIP runtime error",
    GS_ERR_NOMEM: "device allocation failed",
    GS_ERR_UNSUPPORTED: "outside implemented limits",
}

# Symbols declared in include/gs_sampler.h.
EXPORTS = [
    "gs_sampler_create", "gs_sampler_destroy", "gs_sampler_set_params",
    "gs_sampler_set_seed", "gs_sampler_get_state", "gs_sampler_set_state",
    "gs_sampler_reserve", "gs_sample", "gs_sample_mut", "gs_logits_writeback", "gs_sample_detail", "gs_sample_batch", "gs_sample_batch_noalloc", "gs_window_push",
    "gs_synth_logits", "gs_limits", "gs_version",
    # include/gs_gemv.h
    "gs_qmatrix_upload", "gs_qmatrix_destroy", "gs_qmatrix_shape", "gs_gemv",
    # include/gs_decode.h
    "gs_sampler_get_params", "gs_sampler_fallback_rows", "gs_decode_init", "gs_decode_commit", "gs_decode_step",
    # include/gs_tokens.h
    "gs_vocab_create", "gs_vocab_destroy", "gs_vocab_find", "gs_token_decode", "gs_tokens_decode",
    "gs_chat_template_detect", "gs_stop_tokens",
    # include/gs_rope.h
    "gs_rope_create", "gs_rope_destroy", "gs_rope_apply",
    # include/gs_cache.h
    "gs_kv_workspace", "gs_kv_reset", "gs_kv_extend", "gs_kv_fork", "gs_kv_free", "gs_kv_drop", "gs_kv_append",
    "gs_kv_evict_workspace", "gs_kv_evict", "gs_kv_free_mass", "gs_kv_drop_mass",
    # include/gs_attn.h
    "gs_attn_workspace", "gs_attn", "gs_attn_lse", "gs_attn_shared", "gs_attn_shared_workspace", "gs_attn_weigh",
    "gs_attn_weigh_workspace",
]


class SamplerError(RuntimeError):
    def __init__(self, code, where=""):
        self.code = code
        super().__init__("%s: %s (%d)" % (where or "gs_sampler", _ERRNAMES.get(code, "error"), code))


class GsParams(ctypes.Structure):
    _fields_ = [("temperature", ctypes.c_float), ("top_k", ctypes.c_uint32),
                ("top_p", ctypes.c_float), ("rep_penalty", ctypes.c_float)]


class GsDetail(ctypes.Structure):
    """gs_detail (include/gs_sampler.h)."""
    _fields_ = [("ids", ctypes.c_void_p), ("p", ctypes.c_void_p), ("cap", ctypes.c_size_t),
                ("n_kept", ctypes.c_void_p), ("cut", ctypes.c_void_p), ("sums", ctypes.c_void_p),
                ("ties", ctypes.c_void_p)]


class DecodeCtx(ctypes.Structure):
    """gs_decode_ctx (include/gs_decode.h)."""
    _fields_ = [("B", ctypes.c_size_t), ("rows", ctypes.c_void_p), ("window", ctypes.c_void_p),
                ("ld_window", ctypes.c_size_t), ("W", ctypes.c_size_t), ("window_len", ctypes.c_void_p),
                ("stop", ctypes.c_void_p), ("n_stop", ctypes.c_size_t), ("max_new", ctypes.c_uint32),
                ("generated", ctypes.c_void_p), ("ld_generated", ctypes.c_size_t), ("next", ctypes.c_void_p),
                ("u", ctypes.c_void_p), ("tokens", ctypes.c_void_p), ("status", ctypes.c_void_p),
                ("n_active", ctypes.c_void_p)]


class RopeParams(ctypes.Structure):
    """gs_rope_params (include/gs_rope.h)."""
    _fields_ = [("d", ctypes.c_uint32), ("rot", ctypes.c_uint32), ("layout", ctypes.c_uint32),
                ("scaling", ctypes.c_uint32), ("base", ctypes.c_double), ("factor", ctypes.c_double),
                ("context", ctypes.c_uint32), ("beta_fast", ctypes.c_double), ("beta_slow", ctypes.c_double),
                ("gain", ctypes.c_double), ("divisors", ctypes.c_void_p)]


class GsKVCache(ctypes.Structure):
    """gs_kv_cache (include/gs_cache.h)."""
    _fields_ = [("k", ctypes.c_void_p), ("v", ctypes.c_void_p), ("type", ctypes.c_uint32),
                ("n_layers", ctypes.c_uint32), ("n_pages", ctypes.c_uint32), ("n_kv", ctypes.c_uint32),
                ("page_size", ctypes.c_uint32), ("d", ctypes.c_uint32), ("rows", ctypes.c_uint32),
                ("ld_table", ctypes.c_uint32), ("table", ctypes.c_void_p), ("len", ctypes.c_void_p),
                ("ref", ctypes.c_void_p), ("ws", ctypes.c_void_p)]


class GsKVBatch(ctypes.Structure):
    """gs_kv_batch (include/gs_cache.h)."""
    _fields_ = [("n", ctypes.c_uint32), ("n_tokens", ctypes.c_uint32), ("rows", ctypes.c_void_p),
                ("start", ctypes.c_void_p)]


class GsKVNew(ctypes.Structure):
    """gs_kv_new (include/gs_cache.h)."""
    _fields_ = [("type", ctypes.c_uint32), ("k", ctypes.c_void_p), ("v", ctypes.c_void_p), ("ld_k", ctypes.c_size_t),
                ("ld_v", ctypes.c_size_t), ("q", ctypes.c_void_p), ("ld_q", ctypes.c_size_t),
                ("q_out", ctypes.c_void_p), ("ld_q_out", ctypes.c_size_t), ("q_out_type", ctypes.c_uint32),
                ("n_heads", ctypes.c_uint32)]


class GsAttnArgs(ctypes.Structure):
    """gs_attn_args (include/gs_attn.h)."""
    _fields_ = [("type", ctypes.c_uint32), ("n_heads", ctypes.c_uint32), ("q", ctypes.c_void_p), ("ld_q", ctypes.c_size_t),
                ("out", ctypes.c_void_p), ("ld_out", ctypes.c_size_t), ("scale", ctypes.c_float),
                ("window", ctypes.c_uint32), ("max_q", ctypes.c_uint32), ("ws", ctypes.c_void_p),
                ("ws_bytes", ctypes.c_size_t)]


class GsWeighArgs(ctypes.Structure):
    """gs_weigh_args: include/gs_attn.h."""
    _fields_ = [("type", ctypes.c_uint32), ("n_heads", ctypes.c_uint32), ("q", ctypes.c_void_p), ("ld_q", ctypes.c_size_t),
                ("lse", ctypes.c_void_p), ("mass", ctypes.c_void_p), ("ld_mass", ctypes.c_size_t), ("keep", ctypes.c_float),
                ("scale", ctypes.c_float), ("window", ctypes.c_uint32), ("max_q", ctypes.c_uint32), ("ws", ctypes.c_void_p),
                ("ws_bytes", ctypes.c_size_t)]


class GsKVEvictArgs(ctypes.Structure):
    """gs_kv_evict_args: include/gs_cache.h."""
    _fields_ = [("rows", ctypes.c_void_p), ("n", ctypes.c_size_t), ("budget", ctypes.c_void_p), ("budget_all", ctypes.c_uint32),
                ("first", ctypes.c_uint32), ("recent", ctypes.c_uint32), ("mass", ctypes.c_void_p), ("ld_mass", ctypes.c_size_t),
                ("rope", ctypes.c_void_p), ("status", ctypes.c_void_p), ("ws", ctypes.c_void_p), ("ws_bytes", ctypes.c_size_t)]


_lib = None


def load_library(path=LIB_PATH):
    """Load libgs_sampler.so (raises OSError if it has not been built)."""
    global _lib
    if _lib is not None:
        return _lib
    if not os.path.exists(path):
        raise OSError("libgs_sampler.so not built: run gguf-rs-cli_amd/build.py (%s)" % path)
    lib = ctypes.CDLL(path)
    P, U64, SZ, I = ctypes.c_void_p, ctypes.c_uint64, ctypes.c_size_t, ctypes.c_int
    sig = {
        "gs_sampler_create": ([ctypes.POINTER(GsParams), U64, ctypes.POINTER(P)], I),
        "gs_sampler_destroy": ([P], I),
        "gs_sampler_set_params": ([P, ctypes.POINTER(GsParams)], I),
        "gs_sampler_set_seed": ([P, U64], I),
        "gs_sampler_get_state": ([P, ctypes.POINTER(U64)], I),
        "gs_sampler_set_state": ([P, U64], I),
        "gs_sampler_reserve": ([P, SZ, SZ], I),
        "gs_sample": ([P, P, SZ, P, SZ, ctypes.POINTER(ctypes.c_uint32)], I),
        "gs_sample_mut": ([P, P, SZ, P, SZ, ctypes.POINTER(ctypes.c_uint32)], I),
        "gs_logits_writeback": ([P, P, SZ, SZ, SZ, P, P, SZ, P, SZ, P], I),
        "gs_sample_detail": ([P, P, SZ, SZ, SZ, P, P, SZ, P, SZ, P, P, P, ctypes.POINTER(GsDetail), P], I),
        "gs_sample_batch": ([P, P, SZ, SZ, SZ, P, P, SZ, P, SZ, P, P, P, P], I),
        "gs_sample_batch_noalloc": ([P, P, SZ, SZ, SZ, P, P, SZ, P, SZ, P, P, P, P], I),
        "gs_window_push": ([P, SZ, SZ, SZ, SZ, P, P], I),
        "gs_synth_logits": ([P, SZ, SZ, SZ, U64, U64, ctypes.c_float, P], I),
        "gs_limits": ([ctypes.POINTER(ctypes.c_uint32), ctypes.POINTER(ctypes.c_uint32)], I),
        "gs_version": ([], ctypes.c_char_p),
        "gs_qmatrix_upload": ([ctypes.c_uint32, P, SZ, SZ, ctypes.POINTER(P)], I),
        "gs_qmatrix_destroy": ([P], I),
        "gs_qmatrix_shape": ([P, ctypes.POINTER(ctypes.c_uint32), ctypes.POINTER(SZ), ctypes.POINTER(SZ)], I),
        "gs_gemv": ([P, P, SZ, P, P], I),
        "gs_sampler_get_params": ([P, ctypes.POINTER(GsParams)], I),
        "gs_sampler_fallback_rows": ([P, P, ctypes.POINTER(ctypes.c_size_t)], I),
        "gs_decode_init": ([P, P, ctypes.POINTER(DecodeCtx), P, P, P], I),
        "gs_decode_commit": ([P, P, ctypes.POINTER(DecodeCtx), P], I),
        "gs_decode_step": ([P, P, P, P, SZ, SZ, P, ctypes.POINTER(DecodeCtx), P], I),
        "gs_vocab_create": ([P, P, SZ, P, SZ, ctypes.c_uint32, ctypes.POINTER(P)], I),
        "gs_vocab_destroy": ([P], I),
        "gs_vocab_find": ([P, ctypes.c_char_p, SZ, ctypes.POINTER(ctypes.c_uint32)], I),
        "gs_token_decode": ([P, ctypes.c_uint32, P, SZ, ctypes.POINTER(SZ)], I),
        "gs_tokens_decode": ([P, P, SZ, P, SZ, ctypes.POINTER(SZ)], I),
        "gs_chat_template_detect": ([P, ctypes.c_char_p, ctypes.POINTER(ctypes.c_uint32)], I),
        "gs_stop_tokens": ([P, ctypes.c_uint32, P, SZ, P, SZ, ctypes.POINTER(SZ)], I),
        "gs_rope_create": ([ctypes.POINTER(RopeParams), ctypes.POINTER(P)], I),
        "gs_rope_destroy": ([P], I),
        "gs_rope_apply": ([P, ctypes.c_uint32, P, SZ, P, SZ, SZ, ctypes.c_uint32, P, P], I),
        "gs_kv_workspace": ([ctypes.POINTER(GsKVCache)], SZ),
        "gs_kv_reset": ([ctypes.POINTER(GsKVCache), P], I),
        "gs_kv_extend": ([ctypes.POINTER(GsKVCache), P, SZ, P, ctypes.c_uint32, P, P], I),
        "gs_kv_fork": ([ctypes.POINTER(GsKVCache), P, P, SZ, P, P], I),
        "gs_kv_free": ([ctypes.POINTER(GsKVCache), P, SZ, P], I),
        "gs_kv_drop": ([ctypes.POINTER(GsKVCache), P, SZ, P, P, P, P, P], I),
        "gs_kv_free_mass": ([ctypes.POINTER(GsKVCache), P, SZ, P, SZ, P], I),
        "gs_kv_drop_mass": ([ctypes.POINTER(GsKVCache), P, SZ, P, P, P, P, SZ, P, P], I),
        "gs_kv_evict_workspace": ([ctypes.POINTER(GsKVCache), SZ, ctypes.c_uint32], SZ),
        "gs_kv_evict": ([ctypes.POINTER(GsKVCache), ctypes.POINTER(GsKVEvictArgs), P], I),
        "gs_kv_append": ([ctypes.POINTER(GsKVCache), ctypes.c_uint32, ctypes.POINTER(GsKVBatch), P,
                          ctypes.POINTER(GsKVNew), P], I),
        "gs_attn_workspace": ([ctypes.POINTER(GsKVCache), ctypes.c_uint32], SZ),
        "gs_attn": ([ctypes.POINTER(GsKVCache), ctypes.c_uint32, ctypes.POINTER(GsKVBatch), ctypes.POINTER(GsAttnArgs), P], I),
        "gs_attn_lse": ([ctypes.POINTER(GsKVCache), ctypes.c_uint32, ctypes.POINTER(GsKVBatch), ctypes.POINTER(GsAttnArgs), P, P], I),
        "gs_attn_shared": ([ctypes.POINTER(GsKVCache), ctypes.c_uint32, ctypes.POINTER(GsKVBatch), P, ctypes.c_uint32,
                            ctypes.POINTER(GsAttnArgs), P, P], I),
        "gs_attn_weigh_workspace": ([ctypes.POINTER(GsKVCache)], SZ),
        "gs_attn_weigh": ([ctypes.POINTER(GsKVCache), ctypes.c_uint32, ctypes.POINTER(GsKVBatch), ctypes.POINTER(GsWeighArgs), P], I),
        "gs_attn_shared_workspace": ([ctypes.POINTER(GsKVCache)] + 4 * [ctypes.c_uint32], SZ),
    }
    for name, (args, res) in sig.items():
        f = getattr(lib, name)
        f.argtypes = args
        f.restype = res
    _lib = lib
    return lib


def _check(rc, where):
    if rc != GS_OK:
        raise SamplerError(rc, where)


def _ptr(x):
    """Device/host address of a torch tensor, numpy array, int or None."""
    if x is None:
        return None
    if isinstance(x, int):
        return x
    if hasattr(x, "data_ptr"):
        return x.data_ptr()
    if hasattr(x, "ctypes"):
        return x.ctypes.data
    raise TypeError("unsupported buffer type %r" % type(x))


_TORCH = None


def _torch_fast_args(logits, recent):
    """(ptr, V, recent ptr, W) for a contiguous torch f32 row and a window
    that is a torch tensor of 4-byte ids, a contiguous numpy uint32 array or
    None / empty; None for anything else."""
    global _TORCH
    if _TORCH is None:
        import sys
        t = sys.modules.get("torch")
        if t is None:
            return None
        import numpy as np
        _TORCH = (t.Tensor, t.float32, (t.int32, t.uint32), np.ndarray, np.dtype(np.uint32))
    tensor, f32, ids, ndarray, u32 = _TORCH
    if type(logits) is not tensor or logits.dtype is not f32 or not logits.is_contiguous():
        return None
    if recent is None or (type(recent) is tuple and not recent):
        return logits.data_ptr(), logits.numel(), None, 0
    if type(recent) is ndarray:
        if recent.dtype != u32 or not recent.flags.c_contiguous:
            return None
        W = recent.size
        return logits.data_ptr(), logits.numel(), (recent.ctypes.data if W else None), W
    if type(recent) is not tensor or recent.dtype not in ids or not recent.is_contiguous():
        return None
    W = recent.numel()
    return logits.data_ptr(), logits.numel(), (recent.data_ptr() if W else None), W


def _stream_handle(stream):
    """The HIP stream of a call: `stream` (a torch.cuda.Stream or a handle),
    or by default torch's current stream when torch has initialised the GPU
    (so calls order with torch's work, inside torch.cuda.stream() blocks and
    under graph capture), else the NULL stream."""
    if stream is None:
        import sys as _sys
        torch = _sys.modules.get("torch")
        if torch is not None and torch.cuda.is_initialized():
            return torch.cuda.current_stream().cuda_stream
        return None
    if isinstance(stream, int):
        return stream
    return stream.cuda_stream  # torch.cuda.Stream


class Sampler:
    """Sampler construction of the drop-in: the four scalars of
    src/sampler.rs:35-36 plus the LCG seed of src/sampler.rs:3-5.
    Defaults are the reference CLI's (src/main.rs:24-31, 48-49)."""

    def __init__(self, temperature=0.7, top_k=40, top_p=0.9, rep_penalty=1.1, seed=42):
        self._lib = load_library()
        self._h = ctypes.c_void_p()
        self.params = GsParams(temperature, top_k, top_p, rep_penalty)
        self._out = ctypes.c_uint32()
        self._outref = ctypes.byref(self._out)
        _check(self._lib.gs_sampler_create(ctypes.byref(self.params), seed, ctypes.byref(self._h)),
               "gs_sampler_create")

    def close(self):
        if self._h:
            self._lib.gs_sampler_destroy(self._h)
            self._h = ctypes.c_void_p()

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass

    def set_params(self, temperature, top_k, top_p, rep_penalty):
        self.params = GsParams(temperature, top_k, top_p, rep_penalty)
        _check(self._lib.gs_sampler_set_params(self._h, ctypes.byref(self.params)), "set_params")

    def fallback_rows(self, stream=None):
        """Rows of the last full-vocabulary call finished by the fallback
        forms instead of the increment-histogram path (waits for the stream)."""
        n = ctypes.c_size_t()
        _check(self._lib.gs_sampler_fallback_rows(self._h, _stream_handle(stream), ctypes.byref(n)), "fallback_rows")
        return n.value

    def set_seed(self, seed):
        _check(self._lib.gs_sampler_set_seed(self._h, seed), "set_seed")

    @property
    def state(self):
        v = ctypes.c_uint64()
        _check(self._lib.gs_sampler_get_state(self._h, ctypes.byref(v)), "get_state")
        return v.value

    @state.setter
    def state(self, v):
        _check(self._lib.gs_sampler_set_state(self._h, v), "set_state")

    def reserve(self, B, V):
        _check(self._lib.gs_sampler_reserve(self._h, B, V), "reserve")

    def sample(self, logits, recent=()):
        """sample(logits, recent) -> token; logits: numpy f32 (host) or a
        torch f32 tensor (host or device).  Synchronous."""
        fast = _torch_fast_args(logits, recent)
        if fast is not None:
            if logits.is_cuda or (recent is not None and getattr(recent, "is_cuda", False)):
                # gs_sample runs on the sampler's own non-blocking stream:
                # wait for torch's current stream, which may still be writing
                # the logits (or the window)
                import torch
                torch.cuda.current_stream(logits.device if logits.is_cuda else None).synchronize()
            rc = self._lib.gs_sample(self._h, fast[0], fast[1], fast[2], fast[3], self._outref)
            if rc != GS_OK:
                raise SamplerError(rc, "gs_sample")
            return self._out.value
        import numpy as np
        keep = []
        if isinstance(logits, (list, tuple)):
            logits = np.asarray(logits, dtype=np.float32)
        if hasattr(logits, "dtype") and str(logits.dtype) not in ("float32", "torch.float32"):
            raise TypeError("logits must be float32")
        if hasattr(logits, "is_contiguous") and not logits.is_contiguous():
            raise TypeError("logits must be contiguous")
        if isinstance(logits, np.ndarray):
            logits = np.ascontiguousarray(logits)
            keep.append(logits)
        V = int(logits.numel() if hasattr(logits, "numel") else logits.size)
        if recent is None or (not hasattr(recent, "data_ptr") and not hasattr(recent, "ctypes")):
            recent = np.ascontiguousarray(np.asarray(list(recent or ()), dtype=np.uint32))
        elif isinstance(recent, np.ndarray):
            recent = np.ascontiguousarray(recent.astype(np.uint32, copy=False))   # ids are u32 (&[u32])
        keep.append(recent)
        if hasattr(recent, "element_size") and recent.element_size() != 4:
            raise TypeError("recent ids must be 4-byte integers")
        W = int(recent.numel() if hasattr(recent, "numel") else recent.size)
        out = ctypes.c_uint32()
        _check(self._lib.gs_sample(self._h, _ptr(logits), V, _ptr(recent) if W else None, W,
                                   ctypes.byref(out)), "gs_sample")
        return int(out.value)

    def sample_mut(self, logits, recent=()):
        """sample(&mut logits, ...) as the reference takes it: returns the
        token and leaves `logits` (a contiguous numpy f32 array, or a torch
        f32 tensor on the host or the device) penalized and divided by T
        (src/sampler.rs:37,41), in place."""
        import numpy as np
        if isinstance(logits, np.ndarray):
            if logits.dtype != np.float32 or not logits.flags.c_contiguous or not logits.flags.writeable:
                raise TypeError("logits must be a writeable contiguous float32 array")
        elif hasattr(logits, "data_ptr"):
            if str(logits.dtype) != "torch.float32" or not logits.is_contiguous():
                raise TypeError("logits must be a contiguous float32 tensor")
            if logits.is_cuda:
                import torch
                torch.cuda.current_stream(logits.device).synchronize()
        else:
            raise TypeError("logits must be a numpy array or a torch tensor (mutated in place)")
        V = int(logits.numel() if hasattr(logits, "numel") else logits.size)
        if recent is None or (not hasattr(recent, "data_ptr") and not hasattr(recent, "ctypes")):
            recent = np.ascontiguousarray(np.asarray(list(recent or ()), dtype=np.uint32))
        elif isinstance(recent, np.ndarray):
            recent = np.ascontiguousarray(recent.astype(np.uint32, copy=False))
        W = int(recent.numel() if hasattr(recent, "numel") else recent.size)
        out = ctypes.c_uint32()
        _check(self._lib.gs_sample_mut(self._h, _ptr(logits), V, _ptr(recent) if W else None, W,
                                       ctypes.byref(out)), "gs_sample_mut")
        return int(out.value)

    def logits_writeback(self, logits, params=None, recent=None, recent_len=None, stream=None,
                         V=None, ld=None, W=None, ld_recent=None):
        """Batched write-back of the reference's mutation (penalty, then / T)
        into device rows `logits` [B, ld]; stream-ordered, after
        sample_batch on the same rows."""
        B = int(logits.shape[0])
        V = int(logits.shape[1]) if V is None else V
        ld = (int(logits.stride(0)) if B > 1 else V) if ld is None else ld
        if recent is not None:
            W = int(recent.shape[1]) if W is None else W
            if ld_recent is None:
                ld_recent = int(recent.stride(0)) if recent.shape[0] > 1 else W
        else:
            W, ld_recent = 0, 0
        _check(self._lib.gs_logits_writeback(self._h, _ptr(logits), B, V, ld, _ptr(params), _ptr(recent),
                                             ld_recent, _ptr(recent_len), W, _stream_handle(stream)),
               "gs_logits_writeback")

    def sample_detail(self, logits, tokens, cap, params=None, recent=None, recent_len=None, u=None,
                      status=None, stream=None):
        """gs_sample_detail: the tokens of sample_batch plus, per row, the
        kept candidates (ids, post-softmax p; the first `cap`), n_kept, the
        nucleus cut, (S, s2) and the tie flag.  Returns a dict of device
        tensors; rows with T > 0 are sorted (slow)."""
        import torch
        B, V = int(logits.shape[0]), int(logits.shape[1])
        ld = int(logits.stride(0)) if B > 1 else V
        dev = logits.device
        out = {"ids": torch.zeros((B, cap), dtype=torch.int32, device=dev),
               "p": torch.zeros((B, cap), dtype=torch.float32, device=dev),
               "n_kept": torch.zeros(B, dtype=torch.int32, device=dev),
               "cut": torch.zeros(B, dtype=torch.int32, device=dev),
               "sums": torch.zeros((B, 2), dtype=torch.float32, device=dev),
               "ties": torch.zeros(B, dtype=torch.int32, device=dev)}
        det = GsDetail(_ptr(out["ids"]), _ptr(out["p"]), cap, _ptr(out["n_kept"]), _ptr(out["cut"]),
                       _ptr(out["sums"]), _ptr(out["ties"]))
        if recent is not None:
            W = int(recent.shape[1])
            ld_recent = int(recent.stride(0)) if recent.shape[0] > 1 else W
        else:
            W, ld_recent = 0, 0
        _check(self._lib.gs_sample_detail(self._h, _ptr(logits), B, V, ld, _ptr(params), _ptr(recent), ld_recent,
                                          _ptr(recent_len), W, _ptr(u), _ptr(tokens), _ptr(status),
                                          ctypes.byref(det), _stream_handle(stream)), "gs_sample_detail")
        return out

    def sample_batch(self, logits, tokens, params=None, recent=None, recent_len=None,
                     u=None, status=None, stream=None, V=None, ld=None, W=None, ld_recent=None,
                     noalloc=False):
        """Batched sampling over B device rows (torch tensors on cuda).
        logits [B, ld] f32; tokens [B] int32/uint32; params [B, 4]-shaped
        gs_params buffer (or None); recent [B, ld_recent] uint32 ids (or None);
        u [B] f32 draws (or None = this sampler's LCG stream).  Asynchronous.
        noalloc=True calls gs_sample_batch_noalloc (static scratch, no
        device allocation)."""
        B = int(logits.shape[0])
        V = int(logits.shape[1]) if V is None else V
        # a size-1 leading dimension may carry any stride (numpy gives 0)
        ld = (int(logits.stride(0)) if B > 1 else V) if ld is None else ld
        if recent is not None:
            W = int(recent.shape[1]) if W is None else W
            if ld_recent is None:
                ld_recent = int(recent.stride(0)) if recent.shape[0] > 1 else W
        else:
            W, ld_recent = 0, 0
        fn = self._lib.gs_sample_batch_noalloc if noalloc else self._lib.gs_sample_batch
        _check(fn(
            self._h, _ptr(logits), B, V, ld, _ptr(params), _ptr(recent), ld_recent,
            _ptr(recent_len), W, _ptr(u), _ptr(tokens), _ptr(status),
            _stream_handle(stream)), "gs_sample_batch_noalloc" if noalloc else "gs_sample_batch")


def window_push(window, tokens, pos, W=None, stream=None):
    lib = load_library()
    B = int(window.shape[0])
    W = int(window.shape[1]) if W is None else W
    ld = int(window.stride(0)) if B > 1 else int(window.shape[1])
    _check(lib.gs_window_push(_ptr(window), B, ld, W, pos, _ptr(tokens),
                              _stream_handle(stream)), "gs_window_push")


def synth_logits(out, seed, counter0, sigma, V=None, stream=None):
    lib = load_library()
    B = int(out.shape[0])
    V = int(out.shape[1]) if V is None else V
    ld = int(out.stride(0)) if B > 1 else int(out.shape[1])
    _check(lib.gs_synth_logits(_ptr(out), B, V, ld, seed, counter0, sigma,
                               _stream_handle(stream)), "gs_synth_logits")


def params_array(rows):
    """Pack [(T, top_k, top_p, rep), ...] as a numpy structured array whose
    bytes are B gs_params (16 bytes each)."""
    import numpy as np
    dt = np.dtype([("temperature", "<f4"), ("top_k", "<u4"), ("top_p", "<f4"), ("rep_penalty", "<f4")])
    return np.array([tuple(r) for r in rows], dtype=dt)


# ---- the reference's free-function API over a process-global sampler -----
_global = None
_global_seed = 12345  # src/sampler.rs:3


def _get_global():
    global _global
    if _global is None:
        _global = Sampler(0.7, 40, 0.9, 1.1, seed=_global_seed)
    return _global


def set_seed(s):
    """src/sampler.rs:5"""
    global _global_seed
    _global_seed = s
    if _global is not None:
        _global.set_seed(s)


def sample(logits, temperature, top_k, top_p, rep_penalty, recent):
    """src/sampler.rs:35-36 -- returns the token id.  Raises SamplerError
    where the reference panics."""
    g = _get_global()
    g.set_params(temperature, top_k, top_p, rep_penalty)
    return g.sample(logits, recent)


def sample_mut(logits, temperature, top_k, top_p, rep_penalty, recent):
    """sample() that also leaves `logits` mutated in place as the reference
    does (src/sampler.rs:37,41): penalized, then divided by T when T > 0."""
    g = _get_global()
    g.set_params(temperature, top_k, top_p, rep_penalty)
    return g.sample_mut(logits, recent)


# ---- quantized output projection (include/gs_gemv.h) --------------------------
QTYPE_Q4_0 = 2     # GgmlType::Q4_0 (src/gguf/types.rs:42)
QTYPE_Q4_1 = 3     # GgmlType::Q4_1
QTYPE_Q8_0 = 8     # GgmlType::Q8_0 (src/gguf/types.rs:43)
QTYPE_Q3_K = 11    # GgmlType::Q3K  (src/gguf/types.rs:44)
QTYPE_Q4_K = 12    # GgmlType::Q4K
QTYPE_Q5_K = 13    # GgmlType::Q5K
QTYPE_Q6_K = 14    # GgmlType::Q6K


class QMatrix:
    """A quantized matrix on the device: Gpu::upload (src/gpu/mod.rs:222-238)
    of a Q4_0 / Q4_1 / Q8_0 / Q3_K / Q4_K / Q5_K / Q6_K GGUF tensor.  `blocks` are the tensor's raw bytes (a
    numpy uint8 array or bytes), rows x cols weights, cols = dims[0].
    gemv(x, out) is Gpu::cmd_gemv (src/gpu/mod.rs:438-443): out = W x for
    device f32 vectors (torch tensors or device addresses), B = len(x) / cols
    vectors per call."""

    def __init__(self, qtype, blocks, rows, cols):
        import numpy as np
        self._lib = load_library()
        b = np.ascontiguousarray(np.frombuffer(blocks, dtype=np.uint8) if isinstance(blocks, (bytes, bytearray))
                                 else blocks, dtype=np.uint8)
        h = ctypes.c_void_p()
        _check(self._lib.gs_qmatrix_upload(qtype, b.ctypes.data, rows, cols, ctypes.byref(h)),
               "gs_qmatrix_upload")
        self._h = h
        self.qtype, self.rows, self.cols = qtype, rows, cols

    def gemv(self, x, out, B=1, stream=None):
        st = None
        if stream is not None:
            st = stream.cuda_stream if hasattr(stream, "cuda_stream") else stream
        _check(self._lib.gs_gemv(self._h, _ptr(x), B, _ptr(out), st), "gs_gemv")

    def close(self):
        if self._h:
            self._lib.gs_qmatrix_destroy(self._h)
            self._h = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass


# ---- device-resident decode loop (include/gs_decode.h) ------------------------
DONE_RUNNING, DONE_STOP, DONE_MAX, DONE_ERROR = 0, 1, 2, 3


def decode_row_dtype():
    """numpy dtype of gs_decode_row (24 bytes)."""
    import numpy as np
    return np.dtype([("rng", "<u8"), ("n_gen", "<u4"), ("wpos", "<u4"), ("done", "<u4"), ("last", "<u4")])


class Decoder:
    """Device buffers of B decoding rows and the step of generate_collect
    (src/main.rs:279-311) over them: sample, stop check, max-length check,
    window push, generated push.  Buffers are torch tensors on cuda; every
    method is stream-ordered and, apart from init() and the read-outs,
    asynchronous."""

    def __init__(self, B, W=64, max_new=256, stop=(), device="cuda"):
        import torch
        self._lib = load_library()
        self.B, self.W, self.max_new = B, W, max_new
        dev = torch.device(device)
        u32 = torch.int32
        self.rows = torch.zeros(B * 24, dtype=torch.uint8, device=dev)
        self.window = torch.zeros((B, max(W, 1)), dtype=u32, device=dev)
        self.window_len = torch.zeros(B, dtype=u32, device=dev)
        stop = [int(s) for s in stop]
        self.stop = torch.tensor(stop if stop else [0], dtype=torch.int64).to(u32).to(dev)
        self.generated = torch.zeros((B, max(max_new, 1)), dtype=u32, device=dev)
        self.next = torch.zeros(B, dtype=u32, device=dev)
        self.u = torch.zeros(B, dtype=torch.float32, device=dev)
        self.tokens = torch.zeros(B, dtype=u32, device=dev)
        self.status = torch.zeros(B, dtype=torch.int32, device=dev)
        self.n_active = torch.zeros(1, dtype=u32, device=dev)
        self.ctx = DecodeCtx(B, self.rows.data_ptr(), self.window.data_ptr() if W else None,
                             self.window.stride(0), W, self.window_len.data_ptr() if W else None,
                             self.stop.data_ptr() if stop else None, len(stop), max_new,
                             self.generated.data_ptr(), self.generated.stride(0), self.next.data_ptr(),
                             self.u.data_ptr(), self.tokens.data_ptr(), self.status.data_ptr(),
                             self.n_active.data_ptr())

    def init(self, sampler, seeds, init_recent=None, params=None, stream=None):
        """Reset every row: LCG state = seeds[b] (set_seed, src/sampler.rs:5)
        and the window holding init_recent[b] (the reference's `recent` at
        the start of a turn, oldest first; at most W ids); then the first
        step's draws with the rows' temperatures (params: device gs_params
        per row, or None = the sampler's)."""
        import numpy as np
        import torch
        sd = np.ascontiguousarray(np.asarray(seeds, dtype=np.uint64).reshape(self.B))
        ln = np.zeros(self.B, np.uint32)
        if init_recent is not None:
            for b, r in enumerate(init_recent):
                r = np.asarray(r, dtype=np.uint32)
                if r.size > self.W:
                    raise ValueError("init_recent row %d longer than W" % b)
                ln[b] = r.size
                if r.size:
                    self.window[b, :r.size] = torch.from_numpy(r.view(np.int32)).to(self.window.device)
        _check(self._lib.gs_decode_init(sampler._h, _ptr(params), ctypes.byref(self.ctx), sd.ctypes.data,
                                        ln.ctypes.data, _stream_handle(stream)), "gs_decode_init")

    def step(self, sampler, logits=None, lm_head=None, x=None, params=None, stream=None):
        """One step.  Either lm_head (a QMatrix) and x [B, cols] f32 with
        `logits` a [B, rows] f32 output buffer, or logits [B, ld] holding
        this step's logits."""
        V = lm_head.rows if lm_head is not None else int(logits.shape[1])
        ld = V if lm_head is not None else (int(logits.stride(0)) if self.B > 1 else V)
        _check(self._lib.gs_decode_step(sampler._h, lm_head._h if lm_head is not None else None,
                                        _ptr(x), _ptr(logits), V, ld, _ptr(params), ctypes.byref(self.ctx),
                                        _stream_handle(stream)), "gs_decode_step")

    def commit(self, sampler, params=None, stream=None):
        """gs_decode_commit: commit self.tokens (sampled by the caller) and
        draw the next step's u."""
        _check(self._lib.gs_decode_commit(sampler._h, _ptr(params), ctypes.byref(self.ctx),
                                          _stream_handle(stream)), "gs_decode_commit")

    def row_state(self):
        """The B gs_decode_row records, copied to the host (synchronises)."""
        import numpy as np
        return self.rows.cpu().numpy().view(decode_row_dtype()).copy()

    def generated_ids(self):
        """Per row, the generated ids (list of numpy uint32 arrays)."""
        st = self.row_state()
        g = self.generated.cpu().numpy().view("<u4")
        return [g[b, :min(int(st["n_gen"][b]), g.shape[1])].copy() for b in range(self.B)]


# ---- rotary positions and the paged cache (include/gs_rope.h, gs_cache.h) ------
TYPE_F32, TYPE_F16, TYPE_BF16 = 0, 1, 30        # numbered as GgmlType
ROPE_LAYOUTS = {"interleaved": 0, "half": 1}
ROPE_SCALINGS = {"none": 0, "linear": 1, "yarn": 2}
KV_NONE = 0xFFFFFFFF
_DT = None


def _dtypes():
    """torch's value types and what they are here, its 4-byte integers, the
    current stream's handle without an object on the way, the current device's
    number (None: there is one device), and whether its stream is captured."""
    global _DT
    if _DT is None:
        import torch
        _DT = ({torch.float32: TYPE_F32, torch.float16: TYPE_F16, torch.bfloat16: TYPE_BF16}, (torch.int32, torch.uint32),
               getattr(torch._C, "_cuda_getCurrentRawStream", None),
               torch.cuda.current_device if torch.cuda.device_count() > 1 else None,
               getattr(torch._C, "_cuda_isCurrentStreamCapturing", torch.cuda.is_current_stream_capturing))
    return _DT


def _type(x, what):
    try:
        return (_DT or _dtypes())[0][x.dtype]
    except KeyError:
        raise TypeError("%s must be float32, float16 or bfloat16" % what) from None


def _call(dev, f, what, *args):
    """f(*args) of the library, with the tensors' device dev the current one."""
    now = (_DT or _dtypes())[3]
    if now is None or now() == dev:
        _check(f(*args), what)
    else:
        import torch
        with torch.cuda.device(dev):
            _check(f(*args), what)


def _heads(x, what, dev, heads=None, d=None):
    """(tokens, heads, d, values from token to token) of a [T, heads, d]
    tensor on device dev whose heads are contiguous."""
    shape = x.shape
    if len(shape) != 3 or x.get_device() != dev or dev < 0:
        raise TypeError("%s must be a [tokens, heads, d] tensor on the device" % what)
    T, h, n = shape
    if (heads is not None and h != heads) or (d is not None and n != d):
        raise ValueError("%s has heads of another number or size" % what)
    if x.is_contiguous():
        return T, h, n, h * n
    st, sh, sn = x.stride()
    if (n > 1 and sn != 1) or (h > 1 and sh != n):
        raise TypeError("the heads of %s must be contiguous" % what)
    return T, h, n, (st if T > 1 else h * n)


def _words(x, what, dev, n=None):
    """The address of a contiguous tensor of 4-byte integers (n of them) on device dev, or None."""
    if x is None:
        return None
    try:
        wrong = x.get_device() != dev or x.dtype not in (_DT or _dtypes())[1] or not x.is_contiguous()
    except AttributeError:
        wrong = True
    if wrong or dev < 0:
        raise TypeError("%s must be a contiguous tensor of 4-byte integers on the device" % what)
    if n is not None and x.numel() != n:
        raise ValueError("%s must have %d values" % (what, n))
    return x.data_ptr()


def _stream_of(dev, stream):
    """The HIP stream of a call on device dev: `stream`, or the one that torch
    works on there now (_stream_handle, without a Stream object on the way)."""
    if stream is None:
        raw = (_DT or _dtypes())[2]
        if raw is not None:
            return raw(dev)
    return _stream_handle(stream)


def _may_capture(dev, st):
    """Whether a call on the stream st of device dev may be recorded into a
    graph now: it is unless st is torch's stream of the moment and records none."""
    _, _, raw, now, capturing = _DT or _dtypes()
    return (now is not None and now() != dev) or raw is None or st != raw(dev) or capturing()


def _empty_on(st, shape, dtype, like):
    """A new tensor on like's device for work on the HIP stream st.  Memory that
    torch's stream of the moment has freed may still be in use there: on
    another stream the tensor comes from that one's memory."""
    import torch
    if st == _stream_of(like.get_device(), None):
        return torch.empty(shape, dtype=dtype, device=like.device)
    now = torch.cuda.current_stream(like.device)
    on = torch.cuda.ExternalStream(st, like.device) if st else torch.cuda.default_stream(like.device)
    with torch.cuda.stream(on):
        x = torch.empty(shape, dtype=dtype, device=like.device)
    x.record_stream(now)
    return x


def _turn(rope):
    """The handle of a rotation, or None for none; a closed one is no rotation to go without."""
    if rope is None:
        return None
    if not rope._h:
        raise ValueError("the rotation is closed")
    return rope._h


class Rope:
    """The plan of a rotation (include/gs_rope.h): the first `rot` values of
    heads of d, in the "interleaved" or the "half" layout, with the scaling
    "none", "linear" or "yarn" (`factor`, and for YaRN the trained `context`)
    and the divisors of a rope_freqs tensor."""

    def __init__(self, d, rot=None, layout="half", base=10000.0, scaling="none", factor=1.0, context=0, beta_fast=0.0,
                 beta_slow=0.0, gain=0.0, divisors=None):
        import numpy as np
        self._lib = load_library()
        self._h = None
        rot = d if rot is None else rot
        div = None
        if divisors is not None:
            div = np.ascontiguousarray(np.asarray(divisors, dtype=np.float32))
            if div.size != rot // 2:
                raise ValueError("divisors must have rot / 2 values")
        p = RopeParams(d, rot, ROPE_LAYOUTS[layout], ROPE_SCALINGS[scaling], base, factor, context, beta_fast,
                       beta_slow, gain, None if div is None else div.ctypes.data)
        h = ctypes.c_void_p()
        _check(self._lib.gs_rope_create(ctypes.byref(p), ctypes.byref(h)), "gs_rope_create")
        self._h = h
        self.d, self.rot = d, rot

    def apply(self, x, pos, out=None, stream=None):
        """x [T, heads, d] turned to positions pos [T] (4-byte integers), to
        `out` (None: in place)."""
        out, dev = x if out is None else out, x.get_device()
        T, heads, d, ld = _heads(x, "x", dev, d=self.d)
        T2, _, _, ld_out = _heads(out, "out", dev, heads, d)
        if T2 != T or out.dtype != x.dtype:
            raise ValueError("out must be as x")
        _call(dev, self._lib.gs_rope_apply, "gs_rope_apply", _turn(self), _type(x, "x"), x.data_ptr(), ld, out.data_ptr(), ld_out,
              T, heads, _words(pos, "pos", dev, T), _stream_of(dev, stream))
        return out

    def close(self):
        if self._h:
            self._lib.gs_rope_destroy(self._h)
            self._h = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass


class KVCache:
    """The paged cache of keys and values (include/gs_cache.h) over tensors on
    the device: k, v [layers, pages, kv heads, page, d] in float16 or bfloat16,
    table [rows, pages of a row], len [rows] and ref [pages] of 4-byte
    integers (-1 in the table: no page).  KVCache.empty allocates them.  Row
    numbers and other arguments of the calls are device tensors of 4-byte
    integers; every call is stream-ordered and asynchronous."""

    def __init__(self, k, v, table, len, ref):
        import torch
        self._lib = load_library()
        if k.dim() != 5 or v.shape != k.shape or v.dtype != k.dtype or not k.is_contiguous() or not v.is_contiguous():
            raise ValueError("k and v must be contiguous [layers, pages, heads, page, d] tensors alike")
        if table.dim() != 2 or len.dim() != 1 or table.shape[0] != len.shape[0] or ref.numel() != k.shape[1]:
            raise ValueError("table must be [rows, pages of a row], len [rows], ref [pages]")
        self.dev = k.get_device()
        if self.dev < 0 or v.get_device() != self.dev:
            raise TypeError("k and v must be on one device")
        for x, what in ((table, "table"), (len, "len"), (ref, "ref")):
            _words(x, what, self.dev)
        self.k, self.v, self.table, self.len, self.ref = k, v, table, len, ref
        self.layers, self.pages, self.kv, self.page, self.d = k.shape
        self.rows, ld = table.shape
        self.type = _type(k, "k")
        self.c = GsKVCache(k.data_ptr(), v.data_ptr(), self.type, self.layers, self.pages, self.kv, self.page, self.d,
                           self.rows, ld, table.data_ptr(), len.data_ptr(), ref.data_ptr(), None)
        self._c = ctypes.byref(self.c)
        words = self._lib.gs_kv_workspace(self._c)
        if not words:
            raise SamplerError(GS_ERR_UNSUPPORTED, "gs_kv_workspace")
        self.ws = torch.empty(words, dtype=torch.int32, device=k.device)
        self.c.ws = self.ws.data_ptr()
        self._attn_ws = {}
        self._more_ws = {}
        self._weigh_bytes = self._lib.gs_attn_weigh_workspace(self._c)
        self._graph_ws = set()          # of these, whose last one a capture may have been given

    @classmethod
    def empty(cls, layers, pages, kv, d, rows, max_len, page=16, dtype=None, device="cuda"):
        """A new cache: every row empty, every page free."""
        import torch
        dtype = torch.float16 if dtype is None else dtype
        shape = (layers, pages, kv, page, d)
        i32 = dict(dtype=torch.int32, device=device)
        c = cls(torch.empty(shape, dtype=dtype, device=device), torch.empty(shape, dtype=dtype, device=device),
                torch.empty((rows, -(-max_len // page)), **i32), torch.empty(rows, **i32), torch.empty(pages, **i32))
        c.reset()
        return c

    def reset(self, stream=None):
        _call(self.dev, self._lib.gs_kv_reset, "gs_kv_reset", self._c, _stream_of(self.dev, stream))

    def extend(self, add, rows=None, status=None, stream=None):
        """Room for new tokens: `add` for each of `rows` (None: every row), a
        number or a tensor of one per row."""
        n, dev = self.rows if rows is None else rows.numel(), self.dev
        each = isinstance(add, int)
        if each and not 0 <= add <= 0xFFFFFFFF:
            raise ValueError("add must be a number of tokens")
        _call(dev, self._lib.gs_kv_extend, "gs_kv_extend", self._c, _words(rows, "rows", dev), n,
              None if each else _words(add, "add", dev, n), add if each else 0, _words(status, "status", dev, n),
              _stream_of(self.dev, stream))

    def fork(self, src, dst, status=None, stream=None):
        """Rows dst become copies of rows src, sharing their full pages (-1: empty)."""
        n, dev = dst.numel(), self.dev
        _call(dev, self._lib.gs_kv_fork, "gs_kv_fork", self._c, _words(src, "src", dev, n), _words(dst, "dst", dev), n,
              _words(status, "status", dev, n), _stream_of(self.dev, stream))

    def free(self, rows, stream=None, mass=None):
        """`rows` become empty; their weights in `mass` (as mass() makes it) 0."""
        at, ld = (None, 0) if mass is None else (mass.data_ptr(), self._mass(mass))
        _call(self.dev, self._lib.gs_kv_free_mass, "gs_kv_free", self._c, _words(rows, "rows", self.dev), rows.numel(), at, ld,
              _stream_of(self.dev, stream))

    def drop(self, start, end, rows, rope=None, status=None, stream=None, mass=None):
        """Tokens start .. end - 1 of each of `rows` leave it (gs_kv_drop); with
        `rope` the keys after them are turned back to their new positions, and
        their weights in `mass` (as mass() makes it) move with them."""
        turn = _turn(rope)
        n, dev = rows.numel(), self.dev
        at, ld = (None, 0) if mass is None else (mass.data_ptr(), self._mass(mass))
        _call(dev, self._lib.gs_kv_drop_mass, "gs_kv_drop", self._c, _words(rows, "rows", dev), n, _words(start, "start", dev, n),
              _words(end, "end", dev, n), turn, at, ld, _words(status, "status", dev, n), _stream_of(self.dev, stream))

    def mass(self):
        """A new tensor for the weights that weigh() adds up and evict() goes by:
        [rows, most tokens of a row] float32, zeros.  A weight belongs to a place
        of a row, so give the tensor to free() and drop() too, or tokens have the
        weights of those that were there before; after reset() the weights are
        the caller's to clear, after fork(), mass[dst] = mass[src] to do."""
        import torch
        return torch.zeros((self.rows, self.table.shape[1] * self.page), device=self.k.device)

    def _mass(self, mass):
        """Values from row to row of a tensor as mass() makes it."""
        if (_DT or _dtypes())[0].get(mass.dtype) != TYPE_F32 or mass.dim() != 2 or mass.get_device() != self.dev or mass.stride(1) != 1:
            raise TypeError("mass must be a [rows, tokens] tensor of float32 on the cache's device")
        if mass.shape[0] != self.rows or mass.shape[1] < self.table.shape[1] * self.page:
            raise ValueError("mass must have the cache's rows and room for the most tokens of each")
        if mass.stride(0) < mass.shape[1] and self.rows > 1:
            raise TypeError("the rows of mass must not overlap")
        return mass.stride(0) if self.rows > 1 else mass.shape[1]

    def evict(self, mass, budget, rows, first=0, recent=0, rope=None, status=None, stream=None):
        """Each of `rows` that holds more than `budget` tokens (a number, or a
        tensor of one per row) keeps its newest `recent`, its `first` ones and
        those of greatest weight between (gs_kv_evict); they move down, their
        weights in `mass` with them, and with `rope` keys are turned back as
        far as they move.
        The cache keeps a workspace of 4 bytes for each token that may stay for
        each stream that evict was called on, as attend does."""
        turn, dev = _turn(rope), self.dev
        n, ld = rows.numel(), self._mass(mass)
        each = isinstance(budget, int)
        for x, what in ((budget if each else 0, "budget"), (first, "first"), (recent, "recent")):
            if not 0 <= x <= 0xFFFFFFFF:
                raise ValueError("%s must be a number of tokens" % what)
        st = _stream_of(dev, stream)
        most = budget if each else 0
        ws = self._workspace("evict", st, self._lib.gs_kv_evict_workspace(self._c, n, most), mass)
        x = GsKVEvictArgs(_words(rows, "rows", dev), n, None if each else _words(budget, "budget", dev, n), most, first, recent,
                          mass.data_ptr(), ld, turn, _words(status, "status", dev, n), ws.data_ptr(), ws.numel())
        _call(dev, self._lib.gs_kv_evict, "gs_kv_evict", self._c, ctypes.byref(x), st)

    def _workspace(self, what, st, n, like):
        """A workspace of n bytes for the calls of one kind on the stream st,
        where they do not overlap: up to an eighth more, so that calls of about
        one size share it.  A larger one takes its place, unless a captured graph
        may hold it: then it stays and the new one is at least twice its size."""
        if not n:
            raise SamplerError(GS_ERR_INVALID, what)
        key = (what, st)
        held = self._more_ws.setdefault(key, [])
        if not held or held[-1].numel() < n:
            import torch
            step = 1 << max(n.bit_length() - 4, 0)
            size = -(-n // step) * step
            if key in self._graph_ws:
                size = max(size, 2 * held[-1].numel())
                self._graph_ws.remove(key)
            elif held:
                held.pop()
            held.append(_empty_on(st, size, torch.uint8, like))
        if key not in self._graph_ws and _may_capture(self.dev, st):
            self._graph_ws.add(key)
        return held[-1]

    def _batch(self, T, rows, q_start):
        if q_start is None:
            n = T
        else:
            n = q_start.numel() - 1
        return GsKVBatch(n, T, _words(rows, "rows", self.dev, n), _words(q_start, "q_start", self.dev))

    def append(self, layer, k, v, q=None, q_out=None, rope=None, rows=None, q_start=None, stream=None):
        """The newest tokens' keys and values [T, kv heads, d] (float32 or the
        cache's type) to their pages, keys turned to their positions by
        `rope`; q [T, heads, d] turned to q_out (None: in place).  One token
        for each of `rows` (None: row i), or those from q_start[i] to
        q_start[i + 1]."""
        turn, dev = _turn(rope), self.dev
        T, _, _, ld_k = _heads(k, "k", dev, self.kv, self.d)
        Tv, _, _, ld_v = _heads(v, "v", dev, self.kv, self.d)
        if Tv != T or v.dtype != k.dtype:
            raise ValueError("v must be as k")
        x = GsKVNew(_type(k, "k"), k.data_ptr(), v.data_ptr(), ld_k, ld_v, None, 0, None, 0, 0, 0)
        if q is not None:
            q_out = q if q_out is None else q_out
            Tq, heads, _, ld_q = _heads(q, "q", dev, d=self.d)
            To, _, _, ld_o = _heads(q_out, "q_out", dev, heads, self.d)
            if Tq != T or To != T or q.dtype != k.dtype:
                raise ValueError("q must have k's tokens and type, q_out q's heads")
            x.q, x.ld_q, x.q_out, x.ld_q_out = q.data_ptr(), ld_q, q_out.data_ptr(), ld_o
            x.q_out_type, x.n_heads = _type(q_out, "q_out"), heads
        b = self._batch(T, rows, q_start)
        _call(dev, self._lib.gs_kv_append, "gs_kv_append", self._c, layer, ctypes.byref(b), turn, ctypes.byref(x),
              _stream_of(self.dev, stream))

    def _lse(self, lse, T, heads):
        """The address of a contiguous [T, heads] float32 tensor, or None."""
        if lse is None:
            return None
        if (_DT or _dtypes())[0].get(lse.dtype) != TYPE_F32 or lse.get_device() != self.dev or not lse.is_contiguous():
            raise TypeError("lse must be a contiguous tensor of float32 on the cache's device")
        if lse.shape != (T, heads):
            raise ValueError("lse must be [tokens, heads]")
        return lse.data_ptr()

    def attend(self, layer, q, out=None, rows=None, q_start=None, scale=0.0, window=0, max_q=0, stream=None, lse=None):
        """Causal attention of the rows' newest tokens (as append takes them) over
        the rows' pages: q and out [T, heads, d] (float32 or the cache's type;
        out None: a new tensor).  window: how many positions back a token
        sees, itself included (0: all).  max_q: the most tokens of one
        sequence, if the caller knows it.  lse [T, heads] float32: gets the
        logarithm of each softmax's sum, which weigh() takes.
        The cache keeps a workspace of 43 to 85 MB for each stream that attend
        was called on.  A captured graph uses that of the stream it was captured
        on, wherever it is replayed: replays of such graphs, and calls on that
        stream, must not overlap."""
        import torch
        if not 0 <= window <= 0xFFFFFFFF:
            raise ValueError("window must be a number of positions")
        T, heads, _, ld_q = _heads(q, "q", self.dev, d=self.d)
        st = _stream_of(self.dev, stream)
        out = _empty_on(st, (T, heads, self.d), q.dtype, q) if out is None else out
        To, _, _, ld_o = _heads(out, "out", self.dev, heads, self.d)
        if To != T or out.dtype != q.dtype:
            raise ValueError("out must be as q")
        ws = self._attn_ws.get((st, heads))         # calls on one stream do not overlap
        if ws is None:
            n = self._lib.gs_attn_workspace(self._c, heads)
            if not n:
                raise SamplerError(GS_ERR_INVALID, "gs_attn_workspace")
            # (its size depends on the heads' values, not on their number)
            ws = next((w for (s, _), w in self._attn_ws.items() if s == st and w.numel() >= n), None)
            ws = self._attn_ws[st, heads] = _empty_on(st, n, torch.uint8, q) if ws is None else ws
        b = self._batch(T, rows, q_start)
        a = GsAttnArgs(_type(q, "q"), heads, q.data_ptr(), ld_q, out.data_ptr(), ld_o, scale, window, max_q, ws.data_ptr(),
                       ws.numel())
        _call(self.dev, self._lib.gs_attn_lse, "gs_attn", self._c, layer, ctypes.byref(b), ctypes.byref(a), self._lse(lse, T, heads), st)
        return out

    def attend_shared(self, layer, q, families, out=None, rows=None, q_start=None, scale=0.0, window=0, max_q=0, stream=None, lse=None):
        """attend() of sequences that come in families: sequences families[j] to
        families[j + 1] - 1 of the call, whose rows begin with the same pages,
        as fork() leaves them.  A family's common pages are read once, not once
        for each row; the result is attend()'s formula's whatever the rows
        hold, and never less precise (gs_attn_shared).
        It has three launches for attend()'s two, about 12 us more, so it pays
        where attend() would read a family's common pages often: single tokens
        of 16 bits from some 250 MB of keys and values a call on (rows x common
        tokens x bytes; 16 rows over 4000, 8 heads of 128), with f32 queries from
        2 GB on, in families of 16 rows or more.  For less, and for chunks of
        hundreds of tokens, attend() is faster.
        The cache keeps a workspace of 43 to 85 MB, and of 8 d + 44 bytes for each
        token and head (d as 64, 128 or 256), for each stream that attend_shared
        was called on, as attend does; a call of more tokens than those before
        makes a larger one, and the smaller one stays only if a captured graph
        may use it (it was given to a capture, or to a call on a stream that was
        not torch's current one)."""
        if not 0 <= window <= 0xFFFFFFFF:
            raise ValueError("window must be a number of positions")
        T, heads, _, ld_q = _heads(q, "q", self.dev, d=self.d)
        st = _stream_of(self.dev, stream)
        out = _empty_on(st, (T, heads, self.d), q.dtype, q) if out is None else out
        To, _, _, ld_o = _heads(out, "out", self.dev, heads, self.d)
        if To != T or out.dtype != q.dtype:
            raise ValueError("out must be as q")
        b = self._batch(T, rows, q_start)
        m = families.numel() - 1
        if m < 1:
            raise ValueError("families must have the begin of each and the end of the last")
        ws = self._workspace("attend_shared", st, self._lib.gs_attn_shared_workspace(self._c, heads, b.n, m, T), q)
        a = GsAttnArgs(_type(q, "q"), heads, q.data_ptr(), ld_q, out.data_ptr(), ld_o, scale, window, max_q, ws.data_ptr(),
                       ws.numel())
        _call(self.dev, self._lib.gs_attn_shared, "gs_attn_shared", self._c, layer, ctypes.byref(b),
              _words(families, "families", self.dev), m, ctypes.byref(a), self._lse(lse, T, heads), st)
        return out


    def weigh(self, layer, q, lse, mass, rows=None, q_start=None, scale=0.0, window=0, max_q=0, keep=1.0, stream=None):
        """The weight that each token of the rows gets from their newest ones in
        this layer, summed over those and the heads, is added to `keep` times
        `mass` (as mass() makes it; 0: begins anew).  q, rows, q_start, scale,
        window as attend() had them, lse [T, heads] as it left it.
        The cache keeps a workspace of 1 MB for each stream that weigh was
        called on, as attend does."""
        if not 0 <= window <= 0xFFFFFFFF:
            raise ValueError("window must be a number of positions")
        T, heads, _, ld_q = _heads(q, "q", self.dev, d=self.d)
        if lse is None:
            raise TypeError("lse must be given")
        ld = self._mass(mass)
        b = self._batch(T, rows, q_start)
        st = _stream_of(self.dev, stream)
        ws = self._workspace("weigh", st, self._weigh_bytes, mass)
        a = GsWeighArgs(_type(q, "q"), heads, q.data_ptr(), ld_q, self._lse(lse, T, heads), mass.data_ptr(), ld, keep, scale, window,
                        max_q, ws.data_ptr(), ws.numel())
        _call(self.dev, self._lib.gs_attn_weigh, "gs_attn_weigh", self._c, layer, ctypes.byref(b), ctypes.byref(a), st)
        return mass


# ---- token text and stop set (include/gs_tokens.h) -----------------------------
TOK_LLAMA, TOK_GPT2 = 0, 1
TMPL_CHATML, TMPL_LLAMA3, TMPL_LLAMA2, TMPL_GEMMA, TMPL_PHI3, TMPL_SIMPLE = range(6)


class Vocab:
    """The tokenizer's vocabulary for the text step after the sampler:
    decode(id) is Tokenizer::decode (src/tokenizer/bpe.rs:180-197),
    detect / stop_tokens are ChatTemplate's (src/tokenizer/chat.rs:9-72).
    `tokens` are str or bytes; `types` the GGUF token types; `model` is
    TOK_LLAMA or TOK_GPT2.  Host-only."""

    def __init__(self, tokens, types=(), model=TOK_LLAMA):
        import numpy as np
        self._lib = load_library()
        raw = [t.encode("utf-8") if isinstance(t, str) else bytes(t) for t in tokens]
        off = np.zeros(len(raw) + 1, np.uint64)
        off[1:] = np.cumsum([len(r) for r in raw], dtype=np.uint64)
        data = b"".join(raw)
        ty = np.ascontiguousarray(np.asarray(types, dtype=np.uint32))
        self._data = ctypes.create_string_buffer(data, max(len(data), 1))
        h = ctypes.c_void_p()
        _check(self._lib.gs_vocab_create(self._data, off.ctypes.data, len(raw),
                                         ty.ctypes.data if ty.size else None, ty.size, model,
                                         ctypes.byref(h)), "gs_vocab_create")
        self._h = h

    def find(self, s):
        b = s.encode("utf-8") if isinstance(s, str) else bytes(s)
        out = ctypes.c_uint32()
        _check(self._lib.gs_vocab_find(self._h, b, len(b), ctypes.byref(out)), "gs_vocab_find")
        return None if out.value == 0xFFFFFFFF else int(out.value)

    def decode_bytes(self, ids):
        """The UTF-8 bytes of decode(id) concatenated over ids (an int or a sequence)."""
        import numpy as np
        a = np.ascontiguousarray(np.atleast_1d(np.asarray(ids, dtype=np.uint32)))
        n = ctypes.c_size_t()
        _check(self._lib.gs_tokens_decode(self._h, a.ctypes.data, a.size, None, 0, ctypes.byref(n)),
               "gs_tokens_decode")
        buf = ctypes.create_string_buffer(max(n.value, 1))
        _check(self._lib.gs_tokens_decode(self._h, a.ctypes.data, a.size, buf, n.value, ctypes.byref(n)),
               "gs_tokens_decode")
        return buf.raw[:n.value]

    def decode(self, ids):
        return self.decode_bytes(ids).decode("utf-8")

    def detect(self, tmpl=None):
        out = ctypes.c_uint32()
        _check(self._lib.gs_chat_template_detect(self._h, None if tmpl is None else tmpl.encode("utf-8"),
                                                 ctypes.byref(out)), "gs_chat_template_detect")
        return int(out.value)

    def stop_tokens(self, kind, eos_ids):
        import numpy as np
        e = np.ascontiguousarray(np.asarray(eos_ids, dtype=np.uint32))
        n = ctypes.c_size_t()
        out = np.zeros(len(eos_ids) + 8, np.uint32)
        _check(self._lib.gs_stop_tokens(self._h, kind, e.ctypes.data if e.size else None, e.size,
                                        out.ctypes.data, out.size, ctypes.byref(n)), "gs_stop_tokens")
        return [int(x) for x in out[:n.value]]

    def close(self):
        if self._h:
            self._lib.gs_vocab_destroy(self._h)
            self._h = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass
