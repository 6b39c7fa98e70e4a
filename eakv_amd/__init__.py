"""eakv_amd — Python binding of libeakv.so (Q4_1 KV cache on MI355X).

The library is the C ABI declared in include/eakv.h (the reference eakv API,
reference include/eakv.h:14-83) and include/eakv_hip.h (device-pointer,
batched and fused extensions).  This module loads it with ctypes and offers

  * ``lib()``     the raw ctypes handle, with argtypes set for every symbol;
  * ``Cache``     an object wrapper whose methods mirror the C calls one to one
                  and take / return numpy arrays for the host-pointer calls;
  * ``EakvError`` raised for non-zero return codes and recorded errors.

There is no fallback: if libeakv.so is missing or cannot be loaded, every entry
point raises.
"""
from __future__ import annotations

import ctypes as C
import os

import numpy as np

EAKV_OK = 0
EAKV_ERR_IO = -1
EAKV_ERR_FORMAT = -2
EAKV_ERR_ALLOC = -3
EAKV_ERR_INVALID = -4
EAKV_ERR_DEVICE = -5

EAKV_F32 = 0
EAKV_BF16 = 1
EAKV_TREE_MAX = 64

_HERE = os.path.dirname(os.path.abspath(__file__))
LIB_PATH = os.path.join(_HERE, "libeakv.so")

_f32p = C.POINTER(C.c_float)
_u8p = C.POINTER(C.c_uint8)
_vp = C.c_void_p

# name -> (restype, argtypes); every symbol exported by libeakv.so
SIGNATURES = {
    # include/eakv.h
    "eakv_cache_create": (_vp, [C.c_int, C.c_int, C.c_int, C.c_int]),
    "eakv_cache_free": (None, [_vp]),
    "eakv_cache_load_raw": (C.c_int, [_vp, _vp, C.c_int]),
    "eakv_cache_append": (C.c_int, [_vp, _vp, C.c_int, C.c_int, C.c_int]),
    "eakv_cache_advance": (C.c_int, [_vp, C.c_int]),
    "eakv_cache_clear": (None, [_vp]),
    "eakv_checkpoint": (C.c_int, [_vp]),
    "eakv_restore": (C.c_int, [_vp, C.c_int]),
    "eakv_attention_scores": (None, [_vp, _vp, C.c_int, C.c_int, C.c_int, _vp]),
    "eakv_attention_output": (None, [_vp, _vp, C.c_int, C.c_int, C.c_int, _vp]),
    "eakv_cache_save": (C.c_int, [_vp, C.c_char_p]),
    "eakv_cache_load": (C.c_int, [C.c_char_p, C.POINTER(_vp)]),
    "eakv_cache_seq_len": (C.c_int, [_vp]),
    "eakv_cache_n_layers": (C.c_int, [_vp]),
    "eakv_cache_n_heads": (C.c_int, [_vp]),
    "eakv_cache_head_dim": (C.c_int, [_vp]),
    "eakv_cache_max_seq_len": (C.c_int, [_vp]),
    "eakv_cache_compression_ratio": (C.c_float, [_vp]),
    # include/eakv_hip.h
    "eakv_last_error": (C.c_int, []),
    "eakv_last_error_message": (C.c_char_p, []),
    "eakv_clear_error": (None, []),
    "eakv_cache_device": (C.c_int, [_vp]),
    "eakv_cache_stream": (_vp, [_vp]),
    "eakv_cache_sync": (C.c_int, [_vp]),
    "eakv_cache_read_planes": (C.c_int, [_vp, C.c_int, C.c_int, _vp, _vp, _vp]),
    "eakv_cache_load_raw_device": (C.c_int, [_vp, _vp, C.c_int, _vp]),
    "eakv_cache_append_device": (C.c_int, [_vp, _vp, C.c_int, C.c_int, C.c_int, _vp]),
    "eakv_append_batch_device": (C.c_int, [_vp, C.c_int, _vp, C.c_int, _vp]),
    "eakv_attention_scores_device": (C.c_int, [_vp, _vp, C.c_int, C.c_int, C.c_int, _vp, _vp]),
    "eakv_attention_output_device": (C.c_int, [_vp, _vp, C.c_int, C.c_int, C.c_int, _vp, _vp]),
    "eakv_attention_fused": (C.c_int, [_vp, _vp, C.c_int, C.c_int, C.c_int, _vp]),
    "eakv_attention_fused_batch_device": (
        C.c_int, [_vp, C.c_int, C.c_int, _vp, C.c_int, C.c_int, _vp, _vp]),
    "eakv_attention_fused_batch_device_noalloc": (
        C.c_int, [_vp, C.c_int, C.c_int, _vp, C.c_int, C.c_int, _vp, _vp]),
    "eakv_attention_window_batch_device": (
        C.c_int, [_vp, C.c_int, C.c_int, _vp, _vp, _vp, C.c_int, C.c_int, C.c_int, _vp, _vp, _vp,
                  C.c_size_t, _vp]),
    "eakv_attention_window_work_bytes": (
        C.c_size_t, [_vp, C.c_int, _vp, _vp, C.c_int, C.c_int, C.c_int]),
    "eakv_verify_drafts_device": (
        C.c_int, [C.c_int, C.c_int, C.c_int, _vp, _vp, _vp, C.c_int64, _vp, C.c_int64, _vp, _vp,
                  _vp, _vp, C.c_size_t, _vp]),
    "eakv_verify_drafts_work_bytes": (C.c_size_t, [C.c_int, C.c_int, C.c_int]),
    "eakv_cache_copy_batch_device": (
        C.c_int, [_vp, C.c_int, _vp, C.c_int, C.c_int, C.c_int, _vp]),
    "eakv_cache_gather_batch_device": (C.c_int, [_vp, _vp, C.c_int, _vp, _vp, _vp, _vp]),
    "eakv_cache_fork": (_vp, [_vp, C.c_int, C.c_int]),
    "eakv_cache_compact": (C.c_int, [_vp, C.c_int, _vp, C.c_int]),
    "eakv_cache_planes_device": (C.c_int, [_vp, C.c_int, C.c_int, _vp, _vp, _vp]),
    "eakv_attention_fused_plan": (C.c_int, [_vp, C.c_int, C.c_int, C.c_int, C.c_int, _vp]),
    "eakv_dequantize_range_device": (
        C.c_int, [_vp, C.c_int, C.c_int, C.c_int64, C.c_int64, _vp, _vp]),
    "eakv_dequantize_range": (C.c_int, [_vp, C.c_int, C.c_int, C.c_int64, C.c_int64, _vp]),
    "eakv_validate": (C.c_int, [_vp, _vp]),
    "eakv_ggml_quantize_row_device": (C.c_int, [_vp, _vp, C.c_int64, _vp]),
    "eakv_ggml_dequantize_row_device": (C.c_int, [_vp, _vp, C.c_int64, _vp]),
    "eakv_ggml_vec_dot_device": (C.c_int, [C.c_int, _vp, C.c_size_t, _vp, C.c_size_t, _vp,
                                           C.c_size_t, C.c_int, _vp]),
}

_LIB = None


class EakvError(RuntimeError):
    def __init__(self, code: int, msg: str):
        super().__init__(f"eakv error {code}: {msg}")
        self.code = code


def lib():
    """Load libeakv.so (once) and return the ctypes handle."""
    global _LIB
    if _LIB is None:
        if not os.path.exists(LIB_PATH):
            raise ImportError(
                f"{LIB_PATH} is not built; run __graft_entry__.build() "
                "(make -C eakv_amd)")
        h = C.CDLL(LIB_PATH)
        for name, (res, args) in SIGNATURES.items():
            fn = getattr(h, name)
            fn.restype = res
            fn.argtypes = args
        _LIB = h
    return _LIB


def last_error():
    L = lib()
    return L.eakv_last_error(), (L.eakv_last_error_message() or b"").decode()


def _check(rc: int):
    if rc != EAKV_OK:
        code, msg = last_error()
        raise EakvError(rc, msg)
    return rc


def _ptr(a: np.ndarray):
    return a.ctypes.data_as(_vp)


def _f32(a) -> np.ndarray:
    return np.ascontiguousarray(a, dtype=np.float32)


class Cache:
    """An eakv_cache_t* on the current HIP device.

    Methods mirror include/eakv.h (reference include/eakv.h:25-83); host
    buffers are numpy arrays.
    """

    def __init__(self, n_layers, n_kv_heads, head_dim, max_seq_len, _handle=None):
        L = lib()
        if _handle is None:
            _handle = L.eakv_cache_create(n_layers, n_kv_heads, head_dim, max_seq_len)
            if not _handle:
                code, msg = last_error()
                raise EakvError(code or EAKV_ERR_INVALID, msg or "cache_create failed")
        self.h = _handle

    # -- lifecycle
    def free(self):
        if self.h:
            lib().eakv_cache_free(self.h)
            self.h = None

    def __del__(self):
        try:
            self.free()
        except Exception:
            pass

    def __enter__(self):
        return self

    def __exit__(self, *a):
        self.free()

    # -- info
    @property
    def seq_len(self):
        return lib().eakv_cache_seq_len(self.h)

    @property
    def n_layers(self):
        return lib().eakv_cache_n_layers(self.h)

    @property
    def n_heads(self):
        return lib().eakv_cache_n_heads(self.h)

    @property
    def head_dim(self):
        return lib().eakv_cache_head_dim(self.h)

    @property
    def max_seq_len(self):
        return lib().eakv_cache_max_seq_len(self.h)

    @property
    def compression_ratio(self):
        return lib().eakv_cache_compression_ratio(self.h)

    @property
    def stream(self):
        return lib().eakv_cache_stream(self.h)

    # -- quantization
    def load_raw(self, data, seq_len):
        d = _f32(data)
        return _check(lib().eakv_cache_load_raw(self.h, _ptr(d), seq_len))

    def append(self, data, layer, kv_idx, n_tokens):
        d = _f32(data)
        return _check(lib().eakv_cache_append(self.h, _ptr(d), layer, kv_idx, n_tokens))

    def advance(self, n_tokens):
        return _check(lib().eakv_cache_advance(self.h, n_tokens))

    def clear(self):
        lib().eakv_cache_clear(self.h)

    def checkpoint(self):
        return lib().eakv_checkpoint(self.h)

    def restore(self, seq_len):
        return _check(lib().eakv_restore(self.h, seq_len))

    # -- attention (host pointers)
    def attention_scores(self, queries, layer, n_q, n_kv):
        q = _f32(queries)
        out = np.zeros((n_q, self.seq_len), np.float32)
        L = lib()
        L.eakv_clear_error()
        L.eakv_attention_scores(self.h, _ptr(q), layer, n_q, n_kv, _ptr(out))
        code, msg = last_error()
        if code:
            raise EakvError(code, msg)
        return out

    def attention_output(self, weights, layer, n_q, n_kv):
        w = _f32(weights)
        out = np.zeros((n_q, self.head_dim), np.float32)
        L = lib()
        L.eakv_clear_error()
        L.eakv_attention_output(self.h, _ptr(w), layer, n_q, n_kv, _ptr(out))
        code, msg = last_error()
        if code:
            raise EakvError(code, msg)
        return out

    def attention_fused(self, queries, layer, n_q, n_kv):
        q = _f32(queries)
        out = np.zeros((n_q, self.head_dim), np.float32)
        _check(lib().eakv_attention_fused(self.h, _ptr(q), layer, n_q, n_kv, _ptr(out)))
        return out

    # -- planes
    def read_planes(self, layer, kv_idx):
        ng = self.n_heads * self.max_seq_len * self.head_dim // 64
        w = np.zeros((ng, 32), np.uint8)
        s = np.zeros(ng, np.float32)
        b = np.zeros(ng, np.float32)
        _check(lib().eakv_cache_read_planes(self.h, layer, kv_idx, _ptr(w), _ptr(s), _ptr(b)))
        return w, s, b

    def dequantize_range(self, layer, kv_idx, group_start, group_count):
        """f32[group_count][64] of plane groups [group_start, +group_count)."""
        out = np.zeros((group_count, 64), np.float32)
        _check(lib().eakv_dequantize_range(self.h, layer, kv_idx, group_start, group_count,
                                           _ptr(out)))
        return out

    def validate(self):
        """int32[n_layers * 2]: the integrity code of every (layer, kv) block."""
        res = np.zeros(2 * self.n_layers, np.int32)
        _check(lib().eakv_validate(self.h, _ptr(res)))
        return res

    def planes_device(self, layer, kv_idx):
        """Device addresses of a block's packed codes, scales and biases."""
        p = [_vp() for _ in range(3)]
        _check(lib().eakv_cache_planes_device(self.h, layer, kv_idx, *map(C.byref, p)))
        return tuple(x.value for x in p)

    # -- tokens moved
    def fork(self, n_tokens=None, max_seq_len=None):
        """A new cache holding the first n_tokens (all) of this one."""
        L = lib()
        L.eakv_clear_error()
        h = L.eakv_cache_fork(self.h, self.seq_len if n_tokens is None else n_tokens,
                              self.max_seq_len if max_seq_len is None else max_seq_len)
        if not h:
            code, msg = last_error()
            raise EakvError(code or EAKV_ERR_INVALID, msg or "cache_fork failed")
        return type(self)(0, 0, 0, 0, _handle=h)

    def compact(self, keep, start=0):
        """Keep the tokens before start and, of the others, those at `keep`."""
        k = np.frombuffer(ints(keep), np.int32) if len(keep) else np.zeros(0, np.int32)
        return _check(lib().eakv_cache_compact(self.h, start, _ptr(k), k.size))

    def sync(self):
        return _check(lib().eakv_cache_sync(self.h))

    # -- files
    def save(self, path):
        return _check(lib().eakv_cache_save(self.h, os.fsencode(path)))

    @classmethod
    def load(cls, path):
        out = _vp()
        _check(lib().eakv_cache_load(os.fsencode(path), C.byref(out)))
        return cls(0, 0, 0, 0, _handle=out.value)


def handles(caches):
    """ctypes array of eakv_cache_t* for the batched entry points."""
    arr = (_vp * len(caches))()
    for i, c in enumerate(caches):
        arr[i] = c.h
    return arr


def ints(values):
    """ctypes int32 array for the batched entry points."""
    values = [int(v) for v in values]
    if any(not -2 ** 31 <= v < 2 ** 31 for v in values):
        raise ValueError("a value beyond 32 bits")
    return (C.c_int32 * len(values))(*values)


class WindowPlan:
    """One shape of eakv_attention_window_batch_device: the caches, the tokens of each
    window, where the windows begin (None: at each cache's seq_len when run) and the
    head split.  Buffers are device addresses."""

    def __init__(self, caches, n_tokens, n_q, n_kv, starts=None, dtype="f32"):
        self.caches = list(caches)
        # the library reads one entry of each list per cache
        for name, x in (("n_tokens", n_tokens), ("starts", starts)):
            if x is not None and len(x) != len(self.caches):
                raise ValueError(f"{name}: {len(x)} entries for {len(self.caches)} caches")
        self._h, self._n = handles(self.caches), ints(n_tokens)
        self._starts = None if starts is None else ints(starts)
        self._args = ({"f32": EAKV_F32, "bf16": EAKV_BF16}[dtype], n_q, n_kv)

    @property
    def work_bytes(self):
        """Bytes of scratch that a run with a workspace of its own needs."""
        L = lib()
        L.eakv_clear_error()
        n = L.eakv_attention_window_work_bytes(self._h, len(self.caches), self._starts, self._n,
                                               *self._args)
        code, msg = last_error()
        if code:
            raise EakvError(code, msg)
        return n

    def run(self, layer, d_q, d_out, d_tree=None, d_work=None, work_bytes=0, stream=None):
        return _check(lib().eakv_attention_window_batch_device(
            self._h, len(self.caches), layer, self._starts, self._n, d_q, *self._args, d_tree,
            d_out, d_work, work_bytes, stream))


FUSED_PLAN_KEYS = ("mfma", "chunks", "merge_levels", "tile_tokens", "waves_per_block",
                   "tiles_per_wave", "quads", "split")


def fused_plan(caches, n_q, n_kv, noalloc=False):
    """The launch eakv_attention_fused_batch_device (or, noalloc, its
    allocation-free form) makes for these caches at their current seq_len:
    a dict over FUSED_PLAN_KEYS (eakv_attention_fused_plan)."""
    plan = (C.c_int32 * 8)()
    _check(lib().eakv_attention_fused_plan(handles(caches), len(caches), n_q, n_kv,
                                           int(bool(noalloc)), plan))
    return dict(zip(FUSED_PLAN_KEYS, list(plan)))
