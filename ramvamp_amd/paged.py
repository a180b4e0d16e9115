"""Rotary positions and a paged KV cache on the GPU (include/ramvamp_paged.h).

No reference counterpart: the reference runs one sequence over one linear cache
and rotates whole heads in NeoX order. Here a batch of independent sequences
draws on one pool of pages, through tables the caller owns; ``Rope`` covers both
pairings, a rotated part of the head, and the scalings for long contexts.

Device tensors only, on the cache's GPU; calls are queued on torch's current
stream of that GPU. Rows (float32, 2-D) may be strided views (columns of a fused
qkv matrix), with the values of a row side by side. Positions, lengths, sequence
numbers and tables are int32 and are read when the call runs: one that names what
is not there is refused on the device, for its row alone, and
``PagedKvCache.device_status`` raises what was recorded.
"""
from __future__ import annotations

import ctypes
import threading
from ctypes import byref, c_double, c_uint64, c_void_p

import numpy as np

from . import _lib as L
from .attention import _check, _elem_code, _lib, _raw_stream

_LAYOUTS = {"half": L.RV_ROPE_HALF, "interleaved": L.RV_ROPE_INTERLEAVED}
_SCALINGS = {"none": L.RV_ROPE_UNSCALED, "linear": L.RV_ROPE_LINEAR, "ntk": L.RV_ROPE_NTK, "yarn": L.RV_ROPE_YARN}

_torch = _F32 = _I32 = _current_device = None


def _t():
    global _torch, _F32, _I32, _current_device
    if _torch is None:
        import torch

        _F32, _I32 = torch.float32, torch.int32
        _current_device = getattr(torch._C, "_cuda_getDevice", None) or torch.cuda.current_device
        _torch = torch
    return _torch


# The checks below are most of a small call's time on the host, so the ordinary
# arguments (contiguous, of the right type, on the call's device) pass on few
# attribute reads; what does not is looked at one property at a time.


def _rows(x, what, device):
    """(address, rows, width, stride) of a float32 matrix whose rows lie in one piece each."""
    torch = _torch or _t()
    if type(x) is torch.Tensor and x.dtype is _F32 and x.get_device() == device >= 0 and x.is_contiguous():
        shape = x.shape
        if len(shape) == 2:
            return x.data_ptr(), shape[0], shape[1], shape[1]
    if not isinstance(x, torch.Tensor) or x.dtype is not torch.float32 or not x.is_cuda:
        raise TypeError(f"{what} must be a float32 torch tensor on the GPU")
    if x.dim() != 2:
        raise ValueError(f"{what} must be 2-D: rows x width")
    rows, width = x.shape
    stride, one = x.stride()
    if one != 1 and width > 1:
        raise TypeError(f"{what}: the values of a row must lie side by side")
    if x.get_device() != device:
        raise ValueError(f"{what} is on another device than the call's")
    return x.data_ptr(), rows, width, width if rows <= 1 else stride


def _ints(x, n, what, device) -> int:
    torch = _torch or _t()
    if type(x) is torch.Tensor and x.dtype is _I32 and x.get_device() == device >= 0 and x.is_contiguous():
        shape = x.shape
        if len(shape) == 1 and shape[0] == n:
            return x.data_ptr()
    if not isinstance(x, torch.Tensor) or x.dtype is not torch.int32 or not x.is_cuda:
        raise TypeError(f"{what} must be an int32 torch tensor on the GPU")
    if x.dim() != 1 or x.shape[0] != n or (n > 1 and x.stride(0) != 1):
        raise ValueError(f"{what} must be contiguous, one entry per row")
    if x.get_device() != device:
        raise ValueError(f"{what} is on another device than the call's")
    return x.data_ptr()


def _weight(x, what, device):
    if x is None:
        return None, 0
    torch = _torch or _t()
    if not isinstance(x, torch.Tensor) or x.dtype is not torch.float32 or not x.is_cuda or not x.is_contiguous():
        raise TypeError(f"{what} must be a contiguous float32 torch tensor on the GPU")
    if x.get_device() != device:
        raise ValueError(f"{what} is on another device than the call's")
    return x.data_ptr(), x.numel()


def _table(x, device) -> L.RvPageTable:
    torch = _torch or _t()
    if type(x) is torch.Tensor and x.dtype is _I32 and x.get_device() == device >= 0 and x.is_contiguous():
        shape = x.shape
        if len(shape) == 2:
            return L.RvPageTable(x.data_ptr(), shape[0], shape[1], shape[1])
    if not isinstance(x, torch.Tensor) or x.dtype is not torch.int32 or not x.is_cuda or x.dim() != 2:
        raise TypeError("table must be a 2-D int32 torch tensor on the GPU: sequences x pages")
    n, pages = x.shape
    stride, one = x.stride()
    if one != 1 and pages > 1:
        raise TypeError("table: a sequence's page ids must lie side by side")
    if x.get_device() != device:
        raise ValueError("table is on another device than the call's")
    return L.RvPageTable(x.data_ptr(), n, pages, pages if n <= 1 else stride)


class Rope:
    """The rotary frequencies of a model (rv_rope_new), for any device.

    The first ``rotary_dim`` values of a head (all by default) turn in pairs:
    ``layout`` "half" pairs (i, i + rotary_dim / 2), "interleaved" (2 i, 2 i + 1).
    ``scaling`` for contexts ``factor`` times the trained one: "none", "linear",
    "ntk" (a larger base) or "yarn" (fast pairs as trained, slow ones
    interpolated, by the turns they make within ``trained_positions``)."""

    def __init__(self, head_dim: int, theta: float, rotary_dim: int | None = None, layout: str = "half",
                 scaling: str | None = "none", factor: float = 1.0, trained_positions: int = 0,
                 beta_fast: float = 32.0, beta_slow: float = 1.0):
        self._h = c_void_p()
        if layout not in _LAYOUTS:
            raise ValueError(f"layout must be one of {sorted(_LAYOUTS)}, got {layout!r}")
        if (scaling or "none") not in _SCALINGS:
            raise ValueError(f"scaling must be one of {sorted(_SCALINGS)}, got {scaling!r}")
        self.head_dim = head_dim
        self.rotary_dim = head_dim if rotary_dim is None else rotary_dim
        err = L.RvError()
        _check(_lib().rv_rope_new(head_dim, self.rotary_dim, _LAYOUTS[layout], theta, _SCALINGS[scaling or "none"],
                                  factor, trained_positions, beta_fast, beta_slow, byref(self._h), byref(err)), err)

    def __del__(self):
        h = getattr(self, "_h", None)
        if h is not None and h.value:
            try:
                _lib().rv_rope_free(h)
            except Exception:
                pass
            self._h = None

    def frequencies(self):
        """(radians per position of each pair, float64; what cosine and sine are multiplied by)."""
        f, gain, err = np.empty(self.rotary_dim // 2), c_double(), L.RvError()
        _check(_lib().rv_rope_frequencies(self._h, f.ctypes.data_as(ctypes.POINTER(c_double)), f.size, byref(gain),
                                          byref(err)), err)
        return f, gain.value


def rope_rows(x, positions, rope: Rope, out=None):
    """rv_rope_rows: the heads of row r of x rotated at positions[r], into out
    (a new tensor by default; x itself rotates in place). Returns out."""
    torch = _torch or _t()
    if out is None:
        out = torch.empty(x.shape, dtype=torch.float32, device=x.device)
    device = x.get_device() if isinstance(x, torch.Tensor) else -1
    xp, rows, width, xs = _rows(x, "x", device)
    op, out_rows, out_width, os = _rows(out, "out", device)
    if out_rows != rows or out_width != width:
        raise ValueError("out must have the shape of x")
    pos = _ints(positions, rows, "positions", device)
    if _current_device() != device:
        with torch.cuda.device(device):
            return rope_rows(x, positions, rope, out)
    err = L.RvError()
    rc = _lib().rv_rope_rows(rope._h, xp, xs, rows, width, pos, op, os, _raw_stream(device), 0, byref(err))
    if rc:
        _check(rc, err)
    return out


class PagedKvCache:
    """A pool of ``n_pages`` pages of ``page_rows`` rows in each of ``n_layers``
    layers (rv_paged_new). Row p of sequence s is row p % page_rows of page
    table[s][p // page_rows]; which pages are whose is the caller's to know."""

    def __init__(self, n_layers: int, n_kv_heads: int, head_dim: int, n_pages: int, page_rows: int = 64, elem="f16",
                 device: int = 0):
        self._h = c_void_p()
        err = L.RvError()
        _check(_lib().rv_paged_new(n_layers, n_kv_heads, head_dim, n_pages, page_rows, _elem_code(elem), device,
                                   byref(self._h), byref(err)), err)
        self.n_layers, self.n_kv_heads, self.head_dim = n_layers, n_kv_heads, head_dim
        self.n_pages, self.page_rows, self.kv_dim = n_pages, page_rows, n_kv_heads * head_dim
        self.elem = {L.RV_ELEM_F16: "f16", L.RV_ELEM_F32: "f32", L.RV_ELEM_Q8_0: "q8_0"}[_elem_code(elem)]
        self.device = device
        torch = _t()
        self._dtype = torch.float32 if self.elem == "f32" else torch.float16  # of rows read back
        self._torch_device = torch.device("cuda", device)
        self._stream = None
        # One call at a time binds the stream, queues its work and has the error's place.
        self._lock = threading.Lock()
        self._lib, self._err = _lib(), err
        self._err_ref = byref(err)

    def __del__(self):
        h = getattr(self, "_h", None)
        if h is not None and h.value:
            try:
                _lib().rv_paged_free(h)
            except Exception:
                pass
            self._h = None

    def close(self):
        self.__del__()

    @staticmethod
    def projected_bytes(n_layers, n_kv_heads, head_dim, n_pages, page_rows=64, elem="f16") -> int:
        out, err = c_uint64(), L.RvError()
        _check(_lib().rv_paged_projected_bytes(n_layers, n_kv_heads, head_dim, n_pages, page_rows, _elem_code(elem),
                                               byref(out), byref(err)), err)
        return int(out.value)

    def _call(self, fn, *args):
        with self._lock:
            s = _raw_stream(self.device)
            if s != self._stream:
                _check(self._lib.rv_paged_set_stream(self._h, s, self._err_ref), self._err)
                self._stream = s
            if fn(self._h, *args, self._err_ref):
                _check(self._err.code, self._err)

    def set_tuning(self, knob: int, value: int):
        """rv_paged_set_tuning: ``RV_TUNE_PAGED_JOIN``, 0 or 2."""
        with self._lock:
            if self._lib.rv_paged_set_tuning(self._h, knob, value, self._err_ref):
                _check(self._err.code, self._err)

    def synchronize(self):
        self._call(self._lib.rv_paged_synchronize)

    def device_status(self):
        """Waits for the stream; raises KvError (PageOutOfRange, SequenceOutOfRange or
        PositionOutOfTable) when the device refused a row since the last read."""
        self._call(self._lib.rv_paged_device_status)

    def append_rows(self, layer: int, k_rows, v_rows, table, positions, seqs=None, rope: Rope | None = None,
                    k_norm_w=None, eps: float = 0.0):
        """rv_paged_append_rows: row r of k_rows and v_rows becomes the row at
        positions[r] of sequence seqs[r] (of sequence r without seqs); k is RMS-normed
        per head by k_norm_w and rotated by rope where they are given. A negative
        position writes nothing."""
        kp, rows, width, ks = _rows(k_rows, "k_rows", self.device)
        vp, v_n, v_width, vs = _rows(v_rows, "v_rows", self.device)
        if width != self.kv_dim or v_n != rows or v_width != width:
            raise ValueError("k_rows and v_rows must both be rows x kv_dim")
        wp, wn = _weight(k_norm_w, "k_norm_w", self.device)
        self._call(self._lib.rv_paged_append_rows, layer, rope._h if rope else None, kp, ks, vp, vs, rows,
                   _ints(positions, rows, "positions", self.device),
                   None if seqs is None else _ints(seqs, rows, "seqs", self.device),
                   byref(_table(table, self.device)), wp, wn, eps, 0)

    def read_rows(self, layer: int, table, positions, seqs=None, k=None, v=None):
        """rv_paged_read_rows: (k, v) [rows][kv_dim], the rows at positions[r] of
        sequence seqs[r] as attention reads them: float32 of an f32 cache, else
        float16; zeros for a negative position or one refused. Into the tensors
        given, else into new ones."""
        rows = positions.shape[0] if isinstance(positions, _torch.Tensor) and positions.dim() == 1 else 0
        pos = _ints(positions, rows, "positions", self.device)
        if k is None and v is None:
            d = self.kv_dim
            k, v = _torch.empty_strided((2, rows, d), (rows * d, d, 1), dtype=self._dtype,
                                        device=self._torch_device).unbind(0)
            kp, vp = k.data_ptr(), v.data_ptr()
        else:
            kp, vp = self._row_buffer(k, "k", rows), self._row_buffer(v, "v", rows)
        self._call(self._lib.rv_paged_read_rows, layer, rows, pos,
                   None if seqs is None else _ints(seqs, rows, "seqs", self.device),
                   byref(_table(table, self.device)), kp, vp, 0)
        return k, v

    def _row_buffer(self, x, what, rows):
        if x is None:
            return None
        if not isinstance(x, _torch.Tensor) or x.dtype is not self._dtype or not x.is_cuda or not x.is_contiguous():
            raise TypeError(f"{what} must be a contiguous {self._dtype} torch tensor on the GPU")
        if x.numel() != rows * self.kv_dim:
            raise ValueError(f"{what} must be rows x kv_dim")
        if x.get_device() != self.device:
            raise ValueError(f"{what} is on another device than the call's")
        return x.data_ptr()


def paged_attention(q_rows, cache: PagedKvCache, layer: int, table, lens, scale: float, out):
    """rv_paged_attention: row i of q_rows (post-RoPE) attends rows 0 .. lens[i] of
    sequence i of the table; length 0 gives zeros."""
    qp, n, width, qs = _rows(q_rows, "q_rows", cache.device)
    op, out_n, out_width, os = _rows(out, "out", cache.device)
    if out_n != n or out_width != width:
        raise ValueError("out must have the shape of q_rows")
    cache._call(cache._lib.rv_paged_attention, layer, qp, qs, n, width, byref(_table(table, cache.device)),
                _ints(lens, n, "lens", cache.device), scale, op, os, 0)
    return out


def paged_decode_step(cache: PagedKvCache, layer: int, q_rows, k_rows, v_rows, q_norm_w, k_norm_w, eps: float,
                      rope: Rope | None, table, positions, scale: float, out):
    """rv_paged_decode_step: one token of each sequence through a layer's attention:
    q and k RMS-normed per head (a weight may be None) and rotated at positions[i], k
    and v appended there, then attention over positions[i] + 1 rows. A negative
    position gives zeros and writes nothing. out may be q_rows, or overlap any of the
    float inputs."""
    d = cache.device
    qp, n, width, qs = _rows(q_rows, "q_rows", d)
    kp, k_n, k_width, ks = _rows(k_rows, "k_rows", d)
    vp, v_n, v_width, vs = _rows(v_rows, "v_rows", d)
    op, out_n, out_width, os = _rows(out, "out", d)
    if out_n != n or out_width != width:
        raise ValueError("out must have the shape of q_rows")
    if k_n != n or v_n != n or k_width != cache.kv_dim or v_width != cache.kv_dim:
        raise ValueError("k_rows and v_rows must be rows x kv_dim with q_rows' rows")
    wqp, wqn = _weight(q_norm_w, "q_norm_w", d)
    wkp, wkn = _weight(k_norm_w, "k_norm_w", d)
    cache._call(cache._lib.rv_paged_decode_step, layer, rope._h if rope else None, qp, qs, kp, ks, vp, vs, n, width, wqp,
                wqn, wkp, wkn, eps, byref(_table(table, d)), _ints(positions, n, "positions", d), scale, op, os, 0)
    return out
