"""Operator-level entry points over the C ABI, on torch device tensors.

These are the calls the MoE blocks make; each validates shapes/dtypes on the
host, then launches on the current stream (or `stream`).
"""
from __future__ import annotations

import ctypes as C
import functools
import math
import threading
from collections import OrderedDict

import torch

from . import _lib
from .geometry import Geometry


def _p(t):
    return None if t is None else t.data_ptr()


def _req(t, dtype, name, numel=None, device=None):
    if t.dtype != dtype:
        raise TypeError(f"{name}: expected {dtype}, got {t.dtype}")
    if not t.is_cuda:
        raise TypeError(f"{name}: must be a device tensor")
    if not t.is_contiguous():
        raise ValueError(f"{name}: must be contiguous")
    if numel is not None and t.numel() != numel:
        raise ValueError(f"{name}: expected {numel} elements, got {t.numel()}")
    if device is not None and t.device != device:
        raise ValueError(f"{name}: on {t.device}, expected {device}")


def _side(stream, device):
    """`stream` as a torch stream where it is another than the current one (any
    object with a cuda_stream handle), else None."""
    if stream is None or stream.cuda_stream == torch.cuda.current_stream(device).cuda_stream:
        return None
    if isinstance(stream, torch.cuda.Stream):
        return stream
    return torch.cuda.ExternalStream(int(stream.cuda_stream), device=device)


def _empty(shape, dtype, device, side):
    """A tensor for kernels on stream `side` (None: the current one) to write:
    allocated in that stream's order, so that the work of the block's last owner is
    not still under way, and kept from reuse while the current stream reads it."""
    if side is None:
        return torch.empty(shape, dtype=dtype, device=device)
    cur = torch.cuda.current_stream(device)
    with torch.cuda.stream(side):
        t = torch.empty(shape, dtype=dtype, device=device)
    t.record_stream(cur)
    return t


class Workspace(threading.local):
    """Grow-only device scratch buffers, one per purpose, device and stream in every
    thread: a call's launches are not one unit, so calls that can run beside each
    other must not share one.  A buffer belongs to its stream's order (a replaced or
    evicted one is reused only behind the calls that hold it).  The KEEP used last
    stay; a call under graph capture takes a buffer of the graph's own instead, since
    a replay can run beside any stream's calls."""

    KEEP = 16

    def __init__(self):
        self._bufs = OrderedDict()

    def get(self, key, nbytes: int, device, handle: int = 0, zero: bool = False,
            side=None) -> torch.Tensor:
        """At least nbytes for calls on the stream of that handle: `side`, or the
        current one."""
        if side is not None:
            with torch.cuda.stream(side):
                return self.get(key, nbytes, device, handle, zero)
        k = (key, device, handle)
        b = self._bufs.get(k)
        own = device.type == "cuda" and _capturing()
        if b is None or own or b.numel() < nbytes:
            b = (torch.zeros if zero else torch.empty)(max(nbytes, 256), dtype=torch.uint8,
                                                       device=device)
            if own:
                return b
            self._bufs[k] = b
            if len(self._bufs) > self.KEEP:
                self._bufs.popitem(last=False)
        self._bufs.move_to_end(k)
        return b


_capturing = torch.cuda.is_current_stream_capturing
_WS = Workspace()


def ffn_decode(pool, slot_refs: torch.Tensor, scores: torch.Tensor,
               x: torch.Tensor, out: torch.Tensor | None = None,
               out_f32: torch.Tensor | None = None, stream=None,
               workspace: torch.Tensor | None = None):
    """Fused expert block for T tokens x k routed experts.

    x bf16 [T, D]; slot_refs int32 [T, k]; scores fp32 [T, k].  Returns bf16
    [T, D] (and fills out_f32 when given)."""
    return _ffn("moe_ffn_decode", "moe_ffn_decode_workspace", "ffn", pool, slot_refs,
                scores, x, out, out_f32, stream, workspace)


def ffn_decode_up(pool, slot_refs: torch.Tensor, x: torch.Tensor,
                  workspace: torch.Tensor | None = None, stream=None) -> torch.Tensor:
    """First half of ffn_decode: the gate/up projections and activation of
    every (token, expert) pair into the workspace, which is returned for
    ffn_decode_down (pass the same tensor; it is not shared with ffn_decode's
    cached workspace)."""
    geom: Geometry = pool.geom
    x = x.view(1, -1) if x.dim() == 1 else x
    T, D = x.shape
    if D != geom.d_model:
        raise ValueError(f"x has {D} features, geometry {geom.d_model}")
    k = slot_refs.numel() // T
    _req(x, torch.bfloat16, "x", device=pool.device)
    _req(slot_refs, torch.int32, "slot_refs", T * k, pool.device)
    g = geom.c_geom()
    L = _lib.lib()
    need = L.moe_ffn_decode_workspace(C.byref(g), T, k)
    if need == 0:
        raise ValueError(f"moe_ffn_decode_up: unsupported T={T}, k={k}")
    if workspace is None:
        workspace = _empty(need, torch.uint8, x.device, _side(stream, x.device))
    _lib.check(L.moe_ffn_decode_up(
        C.byref(pool.c_view()), C.byref(g), _p(slot_refs), _p(x), T, k,
        _p(workspace), workspace.numel(), _lib.stream_ptr(stream)))
    return workspace


def ffn_decode_down(pool, slot_refs: torch.Tensor, scores: torch.Tensor,
                    workspace: torch.Tensor, out: torch.Tensor | None = None,
                    out_f32: torch.Tensor | None = None, stream=None):
    """Second half of ffn_decode: the down projections of the activations
    ffn_decode_up left in `workspace`, weighted by scores and summed per
    token.  slot_refs int32 [T, k] and scores fp32 [T, k] as for ffn_decode."""
    geom: Geometry = pool.geom
    T, k = slot_refs.shape
    D = geom.d_model
    _req(slot_refs, torch.int32, "slot_refs", T * k, pool.device)
    _req(scores, torch.float32, "scores", T * k, pool.device)
    _req(workspace, torch.uint8, "workspace", device=pool.device)
    if out is None and out_f32 is None:
        dev = slot_refs.device
        out = _empty((T, D), torch.bfloat16, dev, _side(stream, dev))
    if out is not None:
        _req(out, torch.bfloat16, "out", T * D, pool.device)
    if out_f32 is not None:
        _req(out_f32, torch.float32, "out_f32", T * D, pool.device)
    g = geom.c_geom()
    _lib.check(_lib.lib().moe_ffn_decode_down(
        C.byref(pool.c_view()), C.byref(g), _p(slot_refs), _p(scores), T, k,
        _p(out), _p(out_f32), _p(workspace), workspace.numel(),
        _lib.stream_ptr(stream)))
    return out if out is not None else out_f32


def slot_lookup(table: torch.Tensor, ids: torch.Tensor,
                miss: torch.Tensor | None = None, stream=None) -> torch.Tensor:
    """slot_refs = table[ids] on device (engine_v3.py:550-552).  table int32
    [E]; ids int32 of any shape.  miss (int32 [1], optional) is incremented
    by the number of refs < 0; an id outside [0, E) gives ref 0 and raises
    the device error flag that check_device_error reports."""
    _req(table, torch.int32, "table")
    _req(ids, torch.int32, "ids", device=table.device)
    if miss is not None:
        _req(miss, torch.int32, "miss", 1, table.device)
    refs = _empty(ids.shape, ids.dtype, ids.device, _side(stream, ids.device))
    _lib.check(_lib.lib().moe_slot_lookup(
        _p(table), table.numel(), _p(ids), ids.numel(), _p(refs), _p(miss),
        _lib.stream_ptr(stream)))
    return refs


def ffn_grouped(pool, slot_refs: torch.Tensor, scores: torch.Tensor,
                x: torch.Tensor, out: torch.Tensor | None = None,
                out_f32: torch.Tensor | None = None, stream=None,
                workspace: torch.Tensor | None = None):
    """The expert block for many tokens (prefill): pairs grouped per slot,
    bf16 MFMA per group.  Same arguments and result as ffn_decode."""
    return _ffn("moe_ffn_grouped", "moe_ffn_grouped_workspace", "ffn_grouped", pool,
                slot_refs, scores, x, out, out_f32, stream, workspace)


# Above this many tokens per call the grouped MFMA path runs; at or below it,
# the decode kernels (which group the pairs by slot from 2 tokens on and give
# results bit-identical to one call per token).  Per step of the 48-layer
# Qwen3 stack on one MI355X (HIP graph of router + expert block per layer):
# 4 tokens 2.05 ms (decode kernels) vs 1.97 ms (MFMA block), 8 tokens 2.80
# vs 2.38 ms, 16 tokens 4.33 vs 2.79 ms.
GROUPED_MIN_TOKENS = 4


def ffn(pool, slot_refs, scores, x, out=None, out_f32=None, stream=None):
    """The expert block, choosing the decode or the grouped path by T (the
    decode/prefill split of engine_v3.py:555-600)."""
    T = 1 if x.dim() == 1 else x.shape[0]
    f = ffn_grouped if T > GROUPED_MIN_TOKENS else ffn_decode
    return f(pool, slot_refs, scores, x, out, out_f32, stream)


def _ffn(entry, ws_entry, ws_key, pool, slot_refs, scores, x, out, out_f32, stream,
         workspace):
    geom: Geometry = pool.geom
    if x.dim() == 1:
        x = x.view(1, -1)
    T, D = x.shape
    if D != geom.d_model:
        raise ValueError(f"x has {D} features, geometry {geom.d_model}")
    k = slot_refs.numel() // T
    _req(x, torch.bfloat16, "x", device=pool.device)
    _req(slot_refs, torch.int32, "slot_refs", T * k, pool.device)
    _req(scores, torch.float32, "scores", T * k, pool.device)
    side, handle = _side(stream, x.device), _lib.stream_ptr(stream)
    if out is None and out_f32 is None:
        out = _empty((T, D), torch.bfloat16, x.device, side)
    if out is not None:
        _req(out, torch.bfloat16, "out", T * D, pool.device)
    if out_f32 is not None:
        _req(out_f32, torch.float32, "out_f32", T * D, pool.device)
    g = geom.c_geom()
    L = _lib.lib()
    need = getattr(L, ws_entry)(C.byref(g), T, k)
    if need == 0:
        raise ValueError(f"{entry}: unsupported T={T}, k={k}")
    ws = workspace if workspace is not None else _WS.get(ws_key, need, x.device, handle,
                                                         side=side)
    _lib.check(getattr(L, entry)(
        C.byref(pool.c_view()), C.byref(g), _p(slot_refs), _p(scores), _p(x),
        T, k, _p(out), _p(out_f32), _p(ws), ws.numel(), handle))
    return out if out is not None else out_f32


class RouteBuffers:
    """Device outputs of one routing call for T tokens."""

    def __init__(self, T: int, k: int, k_pred: int, device):
        # one zeroed allocation, each output at a 16-byte boundary: an
        # allocation and a fill kernel per output were most of a one-token
        # routing call's time when the caller keeps no buffers
        kp = max(k_pred, 1)
        a, b = -(-T * k // 4) * 4, -(-T * kp // 4) * 4
        m = torch.zeros(3 * a + b + 1, dtype=torch.int32, device=device)
        self.ids = m[:T * k].view(T, k)
        self.scores = m[a:a + T * k].view(torch.float32).view(T, k)
        self.slot_refs = m[2 * a:2 * a + T * k].view(T, k)
        self.pred = m[3 * a:3 * a + T * kp].view(T, kp)
        self.miss = m[3 * a + b:]


def route(x: torch.Tensor, W: torch.Tensor, bias: torch.Tensor | None, mode: int,
          renorm: bool, k: int, W_next: torch.Tensor | None = None,
          bias_next: torch.Tensor | None = None, k_pred: int = 0,
          table: torch.Tensor | None = None, bufs: RouteBuffers | None = None,
          stream=None, workspace: torch.Tensor | None = None) -> RouteBuffers:
    """Router + top-k (+ lookahead + slot lookup) on device.

    x bf16 [T, D]; W bf16 [E, D]; bias bf16 [E] or None; table int32 [E]
    (slot refs of this layer) or None."""
    if x.dim() == 1:
        x = x.view(1, -1)
    T, D = x.shape
    E = W.shape[0]
    dev = x.device
    _req(x, torch.bfloat16, "x")
    _req(W, torch.bfloat16, "W", E * D, dev)
    if bias is not None:
        _req(bias, torch.bfloat16, "bias", E, dev)
    if W_next is not None:
        _req(W_next, torch.bfloat16, "W_next", E * D, dev)
        if bias_next is not None:
            _req(bias_next, torch.bfloat16, "bias_next", E, dev)
    if table is not None:
        _req(table, torch.int32, "table", E, dev)
    side, handle = _side(stream, dev), _lib.stream_ptr(stream)
    if bufs is None and side is None:
        bufs = RouteBuffers(T, k, k_pred, dev)
    elif bufs is None:   # (zeroed in the stream's order, as _empty)
        cur = torch.cuda.current_stream(dev)
        with torch.cuda.stream(side):
            bufs = RouteBuffers(T, k, k_pred, dev)
        bufs.miss.record_stream(cur)   # (one allocation)
    L = _lib.lib()
    need = L.moe_route_workspace(T, E)
    ws = workspace if workspace is not None else _WS.get("route", need, dev, handle, True, side)
    _lib.check(L.moe_route(
        _p(x), T, D, _p(W), _p(bias), E, mode, int(renorm), k,
        _p(bufs.ids), _p(bufs.scores),
        _p(W_next), _p(bias_next), k_pred if W_next is not None else 0,
        _p(bufs.pred) if W_next is not None else None,
        _p(table), _p(bufs.slot_refs) if table is not None else None,
        _p(bufs.miss), _p(ws), ws.numel(), handle))
    return bufs


def check_device_error(stream=None):
    _lib.check(_lib.lib().moe_check_device_error(_lib.stream_ptr(stream)))


# ---------------------------------------------------------------------------
# Operators around the expert block: norm, 8-bit product, rotary positions into
# the paged cache, attention over it.  Tensors of 16 bits are bf16 or fp16.
# ---------------------------------------------------------------------------
_DT16 = {torch.bfloat16: _lib.MOE_DTYPE_BF16, torch.float16: _lib.MOE_DTYPE_F16}


def _dt16(t, name) -> int:
    d = _DT16.get(t.dtype)
    if d is None:
        raise TypeError(f"{name}: expected bfloat16 or float16, got {t.dtype}")
    if not t.is_cuda:
        raise TypeError(f"{name}: must be a device tensor")
    return d


def _rows(t, name, dtype, shape, device):
    """t of this type, shape and device whose last dim is contiguous; its strides."""
    if t.dtype != dtype:
        raise TypeError(f"{name}: expected {dtype}, got {t.dtype}")
    if t.shape != shape:
        raise ValueError(f"{name}: expected shape {tuple(shape)}, got {tuple(t.shape)}")
    if t.device != device:
        raise ValueError(f"{name}: on {t.device}, expected {device}")
    st = t.stride()
    if st[-1] != 1 and shape[-1] > 1:
        raise ValueError(f"{name}: the last dim must be contiguous")
    return st


def _on_device(f):
    """Runs an operator with its first argument's device current, so that its stream
    and workspace are that device's."""
    @functools.wraps(f)
    def call(first, *args, **kw):
        if first.is_cuda and first.device.index != torch.cuda.current_device():
            with torch.cuda.device(first.device):
                return f(first, *args, **kw)
        return f(first, *args, **kw)
    return call


def _stream_of(stream, device):
    if stream is not None and getattr(stream, "device", device) != device:
        raise ValueError(f"stream: on {stream.device}, expected {device}")
    return _side(stream, device), _lib.stream_ptr(stream)


@_on_device
def add_rms_norm(x: torch.Tensor, weight: torch.Tensor, residual: torch.Tensor | None = None,
                 eps: float = 1e-6, fp8: bool = False, out: torch.Tensor | None = None,
                 scales: torch.Tensor | None = None, summed: torch.Tensor | None = None,
                 stream=None):
    """Root-mean-square norm behind the residual's addition.

    h = x + residual (rounded to x's type; x itself without a residual);
    y = h * rsqrt(mean(h^2) + eps) * weight.  x, residual [T, D] (or [D]), rows at any
    stride; weight [D].  Returns (y, h), y of x's type, what ops.route and ops.ffn
    read; or with fp8 (q, scales, h): q float8_e4m3fn [T, D] and scales fp32
    [T, ceil(D / 128)], scale = max(largest |y| of the block, 1e-30) / 448, what
    linear_fp8 reads.  out, scales and summed are written where given (out and summed
    may be x or residual themselves)."""
    dt = _dt16(x, "x")
    shape = x.shape
    if x.dim() == 1:
        x = x.view(1, -1)
        residual = residual.view(1, -1) if residual is not None else None
    if x.dim() != 2 or x.shape[1] == 0:
        raise ValueError(f"x: expected [T, D], got {tuple(shape)}")
    T, D = x.shape
    dev = x.device
    xs = _rows(x, "x", x.dtype, x.shape, dev)[0]
    rs = _rows(residual, "residual", x.dtype, x.shape, dev)[0] if residual is not None else D
    _req(weight, x.dtype, "weight", D, dev)
    if summed is not None and residual is None:
        raise ValueError("summed given without residual")
    if scales is not None and not fp8:
        raise ValueError("scales given without fp8")
    side, handle = _stream_of(stream, dev)
    ydt = torch.float8_e4m3fn if fp8 else x.dtype
    if out is None:
        out = _empty(shape, ydt, dev, side)
    else:
        _req(out, ydt, "out", T * D, dev)
    if fp8:
        nb = -(-D // 128)
        if scales is None:
            scales = _empty((T, nb) if len(shape) == 2 else (nb,), torch.float32, dev, side)
        else:
            _req(scales, torch.float32, "scales", T * nb, dev)
    if residual is None:
        h = x.view(shape)
    else:
        h = summed
        if h is None:
            h = _empty(shape, x.dtype, dev, side)
        else:
            _req(h, x.dtype, "summed", T * D, dev)
    _lib.check(_lib.lib().moe_add_rms_norm(
        x.data_ptr(), xs if T > 1 else D, _p(residual), rs if T > 1 else D, weight.data_ptr(), dt,
        T, D, eps, None if fp8 else out.data_ptr(), out.data_ptr() if fp8 else None, _p(scales),
        None if residual is None else h.data_ptr(), handle))
    return (out, scales, h) if fp8 else (out, h)


@_on_device
def linear_fp8(x: torch.Tensor, w: torch.Tensor, w_scales: torch.Tensor,
               x_scales: torch.Tensor | None = None, bias: torch.Tensor | None = None,
               dtype: torch.dtype | None = None, out: torch.Tensor | None = None,
               stream=None, workspace: torch.Tensor | None = None) -> torch.Tensor:
    """y = x w^T (+ bias) with x and w in e4m3 and a scale per block of 128.

    x float8_e4m3fn [T, K] with x_scales fp32 [T, ceil(K / 128)] (add_rms_norm's
    output), or 16 bits, quantised the same way on the way in; w float8_e4m3fn [N, K]
    with w_scales fp32 [ceil(N / 128), ceil(K / 128)]; bias [N] of the output's type:
    `dtype` (bf16 or fp16), else out's, else x's where it has 16 bits, else bf16.
    K is a multiple of 16.  Returns y [T, N] ([N] for x [K])."""
    shape = x.shape
    if x.dim() == 1:
        x = x.view(1, -1)
        x_scales = x_scales.view(1, -1) if x_scales is not None else None
    if x.dim() != 2 or w.dim() != 2:
        raise ValueError(f"expected x [T, K] and w [N, K], got {tuple(shape)}, {tuple(w.shape)}")
    T, K = x.shape
    N = w.shape[0]
    dev = x.device
    x8 = x.dtype == torch.float8_e4m3fn
    if x8:
        if not x.is_cuda:
            raise TypeError("x: must be a device tensor")
        if x_scales is None:
            raise ValueError("an 8-bit x needs x_scales")
        dt = _lib.MOE_DTYPE_E4M3
        nb = -(-K // 128)
        _req(x_scales, torch.float32, "x_scales", T * nb, dev)
    else:
        dt = _dt16(x, "x")
        if x_scales is not None:
            raise ValueError("x_scales given with a 16-bit x")
    if w.shape[1] != K:
        raise ValueError(f"x has {K} columns, w {w.shape[1]}")
    xs = _rows(x, "x", x.dtype, x.shape, dev)[0]
    _req(w, torch.float8_e4m3fn, "w", N * K, dev)
    _req(w_scales, torch.float32, "w_scales", -(-N // 128) * -(-K // 128), dev)
    if dtype is None:
        dtype = out.dtype if out is not None else torch.bfloat16 if x8 else x.dtype
    odt = _DT16.get(dtype)
    if odt is None:
        raise TypeError(f"dtype: expected bfloat16 or float16, got {dtype}")
    if bias is not None:
        _req(bias, dtype, "bias", N, dev)
    side, handle = _stream_of(stream, dev)
    if out is None:
        out = _empty((T, N) if len(shape) == 2 else (N,), dtype, dev, side)
    else:
        _req(out, dtype, "out", T * N, dev)
    L = _lib.lib()
    need = L.moe_linear_fp8_workspace(T, K, N, dt)
    ws = workspace
    if ws is None and need:
        ws = _WS.get("linear_fp8", need, dev, handle, side=side)
    _lib.check(L.moe_linear_fp8(
        x.data_ptr(), dt, xs if T > 1 else K, _p(x_scales), w.data_ptr(), w_scales.data_ptr(),
        _p(bias), T, K, N, odt, out.data_ptr(), _p(ws), ws.numel() if ws is not None else 0,
        handle))
    return out


def rope_freqs(rot: int, base: float = 10000.0, factor: float = 1.0, kind: str = "none",
               original: int = 4096, beta_fast: float = 32.0, beta_slow: float = 1.0,
               low: float = 1.0, high: float = 4.0, device="cuda"):
    """Frequencies of rope_cache's pairs in radians a position, fp64 [rot / 2], and the
    factor mscale that goes with them: freq[i] = base^(-2i / rot), for contexts longer
    than the `original` one of training by kind

    "linear"  every frequency divided by factor
    "yarn"    a pair that turns over beta_fast times within `original` keeps its
              frequency, one that turns under beta_slow times is divided by factor,
              with a linear ramp over the pair's index between (ends rounded outwards);
              mscale = 0.1 ln(factor) + 1
    "llama3"  the same by its wavelength: kept below original / high, divided above
              original / low, and between them weighted by
              (original / wavelength - low) / (high - low)"""
    if rot <= 0 or rot % 2:
        raise ValueError(f"rot={rot} must be positive and even")
    if not base > 1 or not factor >= 1 or original <= 0:
        raise ValueError(f"base={base}, factor={factor}, original={original}: base above 1, "
                         "factor from 1 on and a positive length are needed")
    i = torch.arange(rot // 2, dtype=torch.float64)
    f = base ** (-2.0 * i / rot)
    mscale = 1.0
    if kind == "linear":
        f = f / factor
    elif kind == "yarn":
        def pair(turns):   # the (real) index whose pair turns that often in `original`
            return rot * math.log(original / (turns * 2 * math.pi)) / (2 * math.log(base))
        lo = max(math.floor(pair(beta_fast)), 0)
        hi = min(math.ceil(pair(beta_slow)), rot - 1)
        ramp = ((i - lo) / max(hi - lo, 1e-3)).clamp(0, 1)
        f = f * (1 - ramp) + f / factor * ramp
        mscale = 0.1 * math.log(factor) + 1.0
    elif kind == "llama3":
        if not high > low:
            raise ValueError(f"high={high} must be above low={low}")
        keep = ((original * f / (2 * math.pi) - low) / (high - low)).clamp(0, 1)
        f = f * keep + f / factor * (1 - keep)
    elif kind != "none":
        raise ValueError(f"unknown kind {kind!r}")
    return f.to(device), mscale


def _kv_view(k_pages, v_pages, page_table, q_starts, seq_lens, dev):
    """The C view of a paged cache and its batch."""
    if k_pages.dim() != 4:
        raise ValueError("k_pages: expected [n_pages, kv_heads, page_size, head_dim], got "
                         f"{tuple(k_pages.shape)}")
    dt = _dt16(k_pages, "k_pages")
    n = k_pages.numel()
    _req(k_pages, k_pages.dtype, "k_pages", n, dev)
    _req(v_pages, k_pages.dtype, "v_pages", n, dev)
    if v_pages.shape != k_pages.shape:
        raise ValueError(f"v_pages: expected {tuple(k_pages.shape)}, got {tuple(v_pages.shape)}")
    S = seq_lens.numel()
    if page_table.dim() != 2 or page_table.shape[0] != S:
        raise ValueError(f"page_table: expected [{S}, pages], got {tuple(page_table.shape)}")
    _req(seq_lens, torch.int32, "seq_lens", device=dev)
    _req(page_table, torch.int32, "page_table", device=dev)
    _req(q_starts, torch.int32, "q_starts", S + 1, dev)
    P, H, page, D = k_pages.shape
    return _lib.KvView(k_pages.data_ptr(), v_pages.data_ptr(), page_table.data_ptr(),
                       q_starts.data_ptr(), seq_lens.data_ptr(), P, H, page, D, dt, S,
                       page_table.shape[1])


@_on_device
def rope_cache(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, k_pages: torch.Tensor,
               v_pages: torch.Tensor, page_table: torch.Tensor, q_starts: torch.Tensor,
               seq_lens: torch.Tensor, freqs: torch.Tensor, interleaved: bool = False,
               mscale: float = 1.0, q_weight: torch.Tensor | None = None,
               k_weight: torch.Tensor | None = None, eps: float = 1e-6,
               out: torch.Tensor | None = None, stream=None) -> torch.Tensor:
    """Rotary positions of T new tokens' queries and keys, keys and values put into the
    paged cache.  Returns the turned queries [T, H, D]; out may be q itself.

    q [T, H, D], k and v [T, HK, D] with a contiguous last dim, at any token and head
    strides (column ranges of one product's output).  k_pages, v_pages
    [n_pages, HK, page_size, D]; page_table int32 [S, pages], q_starts int32 [S + 1],
    seq_lens int32 [S], the new tokens included: sequence s's new tokens are rows
    q_starts[s] to q_starts[s + 1], at the positions that end its seq_lens[s], and
    position p is in page page_table[s, p // page_size].  freqs fp64 [R / 2] and
    mscale: as rope_freqs gives them; the first R dims of a head turn, pairs
    (i, i + R/2), or (2i, 2i + 1) interleaved.  q_weight, k_weight [D]: the heads'
    root-mean-square norm before it.

    The batch's arrays stay on the device: an entry out of range is not followed, and
    check_device_error reports it.  Rows behind the last sequence are left as they
    were."""
    dt = _dt16(q, "q")
    if q.dim() != 3:
        raise ValueError(f"q: expected [T, H, D], got {tuple(q.shape)}")
    T, H, D = q.shape
    dev = q.device
    kv = _kv_view(k_pages, v_pages, page_table, q_starts, seq_lens, dev)
    if kv.dtype != dt or kv.head_dim != D:
        raise ValueError(f"q of {q.dtype} and {D} dims, pages of {k_pages.dtype} and {kv.head_dim}")
    qs = _rows(q, "q", q.dtype, q.shape, dev)
    ks = _rows(k, "k", q.dtype, (T, kv.kv_heads, D), dev)
    vs = _rows(v, "v", q.dtype, (T, kv.kv_heads, D), dev)
    _req(freqs, torch.float64, "freqs", device=dev)
    for w, name in ((q_weight, "q_weight"), (k_weight, "k_weight")):
        if w is not None:
            _req(w, q.dtype, name, D, dev)
    side, handle = _stream_of(stream, dev)
    if out is None:
        out = _empty(q.shape, q.dtype, dev, side)
    else:
        _req(out, q.dtype, "out", T * H * D, dev)
    _lib.check(_lib.lib().moe_rope_cache(
        C.byref(kv), q.data_ptr(), qs[0], qs[1], k.data_ptr(), ks[0], ks[1], v.data_ptr(), vs[0],
        vs[1], T, H, freqs.data_ptr(), 2 * freqs.numel(), interleaved, mscale, _p(q_weight),
        _p(k_weight), eps, out.data_ptr(), handle))
    return out


@_on_device
def attn_paged(q: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor,
               page_table: torch.Tensor, q_starts: torch.Tensor, seq_lens: torch.Tensor,
               scale: float | None = None, window: int = 0, sinks: torch.Tensor | None = None,
               out: torch.Tensor | None = None, stream=None,
               workspace: torch.Tensor | None = None) -> torch.Tensor:
    """Causal attention of T new tokens over the paged cache that holds their keys and
    values already (rope_cache's arguments and batch).  Returns [T, H, D].

    q [T, H, D] with 16-byte aligned heads at any token and head strides; head h reads
    key head h // (H / HK); scale defaults to D^-0.5.  window > 0: a row sees the last
    `window` positions up to its own.  sinks fp32 [H]: exp(sinks[h]) joins the softmax's
    sum.  D is 64 or 128.  A row that sees no key is zero; keys that a row does not see
    have no influence, whatever their bits.  Rows behind the last sequence are left as
    they were (in a new output: undefined)."""
    dt = _dt16(q, "q")
    if q.dim() != 3:
        raise ValueError(f"q: expected [T, H, D], got {tuple(q.shape)}")
    T, H, D = q.shape
    dev = q.device
    kv = _kv_view(k_pages, v_pages, page_table, q_starts, seq_lens, dev)
    if kv.dtype != dt or kv.head_dim != D:
        raise ValueError(f"q of {q.dtype} and {D} dims, pages of {k_pages.dtype} and {kv.head_dim}")
    qs = _rows(q, "q", q.dtype, q.shape, dev)
    if sinks is not None:
        _req(sinks, torch.float32, "sinks", H, dev)
    side, handle = _stream_of(stream, dev)
    if out is None:
        out = _empty(q.shape, q.dtype, dev, side)
    else:
        _req(out, q.dtype, "out", T * H * D, dev)
    L = _lib.lib()
    need = L.moe_attn_paged_workspace(C.byref(kv), T, H, window)
    ws = workspace
    if ws is None and need:
        ws = _WS.get("attn_paged", need, dev, handle, side=side)
    _lib.check(L.moe_attn_paged(
        C.byref(kv), q.data_ptr(), qs[0] if T > 1 else 0, qs[1] if H > 1 else 0, T, H,
        D ** -0.5 if scale is None else scale, window, _p(sinks), out.data_ptr(), _p(ws),
        ws.numel() if ws is not None else 0, handle))
    return out
