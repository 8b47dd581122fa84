"""Operator-level entry points over the C ABI, on torch device tensors.

These are the calls the MoE blocks make; each validates shapes/dtypes on the
host, then launches on the current stream (or `stream`).
"""
from __future__ import annotations

import ctypes as C
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


# These calls take a few microseconds on the GPU for single tokens, so their checks are
# made in one expression where all is well, and named one by one where it is not.
def _dt16(t, name) -> int:
    d = _DT16.get(t.dtype)
    if d is None:
        raise TypeError(f"{name}: expected bfloat16 or float16, got {t.dtype}")
    if not t.is_cuda:
        raise TypeError(f"{name}: must be a device tensor")
    return d


def _flat(t, dtype, name, numel, dev: int):
    """_req with a device index."""
    if (t.dtype is not dtype or t.numel() != numel or t.get_device() != dev
            or not t.is_contiguous()):
        _req(t, dtype, name, numel, torch.device("cuda", dev))


def _rows(t, name, dtype, shape, dev: int):
    """t of this type, shape and device whose last dim is contiguous; its strides."""
    st = t.stride()
    if (t.dtype is dtype and t.shape == shape and t.get_device() == dev
            and (st[-1] == 1 or shape[-1] == 1)):
        return st
    if t.dtype != dtype:
        raise TypeError(f"{name}: expected {dtype}, got {t.dtype}")
    if t.shape != shape:
        raise ValueError(f"{name}: expected shape {tuple(shape)}, got {tuple(t.shape)}")
    if t.get_device() != dev:
        raise ValueError(f"{name}: on {t.device}, expected cuda:{dev}")
    raise ValueError(f"{name}: the last dim must be contiguous")


def _on(stream, dev: int):
    """(the stream where it is another than the current one, the handle) for a call on
    device index `dev`, which is the current one."""
    if stream is None:
        return None, torch._C._cuda_getCurrentRawStream(dev)
    device = torch.device("cuda", dev)
    if getattr(stream, "device", device) != device:
        raise ValueError(f"stream: on {stream.device}, expected {device}")
    return _side(stream, device), int(stream.cuda_stream)


def _new(like, shape, dtype, side):
    if side is not None:
        return _empty(shape, dtype, like.device, side)
    if dtype is like.dtype and shape == like.shape and like.is_contiguous():
        return torch.empty_like(like)   # (a third quicker)
    return torch.empty(shape, dtype=dtype, device=like.device)


def _elsewhere(f, dev: int, *args, **kw):
    """f with device index `dev` current, so that its stream and workspace are its."""
    with torch.cuda.device(dev):
        return f(*args, **kw)


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
    dev = x.get_device()
    if dev != torch._C._cuda_getDevice():
        return _elsewhere(add_rms_norm, dev, x, weight, residual, eps, fp8, out, scales, summed,
                          stream)
    shape = x.shape
    if len(shape) == 1:
        x = x.view(1, -1)
        residual = residual.view(1, -1) if residual is not None else None
    elif len(shape) != 2:
        raise ValueError(f"x: expected [T, D], got {tuple(shape)}")
    T, D = rows = x.shape
    dtype = x.dtype
    xs = _rows(x, "x", dtype, rows, dev)[0]
    _flat(weight, dtype, "weight", D, dev)
    rp = rs = hp = h = None
    side, handle = _on(stream, dev)
    if residual is not None:
        rs = _rows(residual, "residual", dtype, rows, dev)[0] if T > 1 else D
        rp = residual.data_ptr()
        if summed is None:
            h = _new(x, shape, dtype, side)
        else:
            h = summed
            _flat(h, dtype, "summed", T * D, dev)
        hp = h.data_ptr()
    elif summed is not None:
        raise ValueError("summed given without residual")
    else:
        h = x.view(shape)
    ydt = torch.float8_e4m3fn if fp8 else dtype
    if out is None:
        out = _new(x, shape, ydt, side)
    else:
        _flat(out, ydt, "out", T * D, dev)
    if not fp8:
        if scales is not None:
            raise ValueError("scales given without fp8")
        _lib.check(_lib.lib().moe_add_rms_norm(
            x.data_ptr(), xs if T > 1 else D, rp, rs or D, weight.data_ptr(), dt, T, D, eps,
            out.data_ptr(), None, None, hp, handle))
        return out, h
    nb = -(-D // 128)
    if scales is None:
        scales = _new(x, (T, nb) if len(shape) == 2 else (nb,), torch.float32, side)
    else:
        _flat(scales, torch.float32, "scales", T * nb, dev)
    _lib.check(_lib.lib().moe_add_rms_norm(
        x.data_ptr(), xs if T > 1 else D, rp, rs or D, weight.data_ptr(), dt, T, D, eps,
        None, out.data_ptr(), scales.data_ptr(), hp, handle))
    return out, scales, h


def linear_fp8(x: torch.Tensor, w: torch.Tensor, w_scales: torch.Tensor,
               x_scales: torch.Tensor | None = None, bias: torch.Tensor | None = None,
               dtype: torch.dtype | None = None, out: torch.Tensor | None = None,
               stream=None, workspace: torch.Tensor | None = None) -> torch.Tensor:
    """y = x w^T (+ bias) with x and w in e4m3 and a scale per block of 128.

    x float8_e4m3fn [T, K] with x_scales fp32 [T, ceil(K / 128)] (add_rms_norm's
    output), or 16 bits, quantised the same way on the way in; w float8_e4m3fn [N, K]
    with w_scales fp32 [ceil(N / 128), ceil(K / 128)]; bias [N] of the output's type:
    `dtype` (bf16 or fp16), else out's, else x's where it has 16 bits, else bf16.
    K is a multiple of 16.  workspace: uint8 on x's device, moe_linear_fp8_workspace
    bytes, by default one of the stream's own.  Returns y [T, N] ([N] for x [K])."""
    x8 = x.dtype is torch.float8_e4m3fn
    if not x8:
        dt = _dt16(x, "x")
        if x_scales is not None:
            raise ValueError("x_scales given with a 16-bit x")
    elif not x.is_cuda:
        raise TypeError("x: must be a device tensor")
    elif x_scales is None:
        raise ValueError("an 8-bit x needs x_scales")
    else:
        dt = _lib.MOE_DTYPE_E4M3
    dev = x.get_device()
    if dev != torch._C._cuda_getDevice():
        return _elsewhere(linear_fp8, dev, x, w, w_scales, x_scales, bias, dtype, out, stream,
                          workspace)
    shape = x.shape
    if len(shape) == 1:
        x = x.view(1, -1)
    if x.dim() != 2 or w.dim() != 2:
        raise ValueError(f"expected x [T, K] and w [N, K], got {tuple(shape)}, {tuple(w.shape)}")
    T, K = x.shape
    N = w.shape[0]
    nb = -(-K // 128)
    if w.shape[1] != K:
        raise ValueError(f"x has {K} columns, w {w.shape[1]}")
    xs = _rows(x, "x", x.dtype, x.shape, dev)[0]
    _flat(w, torch.float8_e4m3fn, "w", N * K, dev)
    _flat(w_scales, torch.float32, "w_scales", -(-N // 128) * nb, dev)
    if x8:
        _flat(x_scales, torch.float32, "x_scales", T * nb, dev)
    if dtype is None:
        dtype = out.dtype if out is not None else torch.bfloat16 if x8 else x.dtype
    odt = _DT16.get(dtype)
    if odt is None:
        raise TypeError(f"dtype: expected bfloat16 or float16, got {dtype}")
    if bias is not None:
        _flat(bias, dtype, "bias", N, dev)
    side, handle = _on(stream, dev)
    if out is None:
        out = _new(x, (T, N) if len(shape) == 2 else (N,), dtype, side)
    else:
        _flat(out, dtype, "out", T * N, dev)
    L = _lib.lib()
    ws = workspace
    if ws is not None:
        _flat(ws, torch.uint8, "workspace", ws.numel(), dev)
    elif not x8:
        need = L.moe_linear_fp8_workspace(T, K, N, dt)
        if need:
            ws = _WS.get("linear_fp8", need, x.device, handle, side=side)
    _lib.check(L.moe_linear_fp8(
        x.data_ptr(), dt, xs if T > 1 else K, _p(x_scales), w.data_ptr(), w_scales.data_ptr(),
        _p(bias), T, K, N, odt, out.data_ptr(), _p(ws), 0 if ws is None else ws.numel(), handle))
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


def _kv_view(dtype, dim, k_pages, v_pages, page_table, q_starts, seq_lens, dev: int):
    """The C view of a paged cache of this type and head size, and its batch."""
    shape = k_pages.shape
    if len(shape) != 4:
        raise ValueError("k_pages: expected [n_pages, kv_heads, page_size, head_dim], got "
                         f"{tuple(shape)}")
    if v_pages.shape != shape:
        raise ValueError(f"v_pages: expected {tuple(shape)}, got {tuple(v_pages.shape)}")
    dt = _DT16.get(dtype)
    P, H, page, D = shape
    n = P * H * page * D
    _flat(k_pages, dtype, "k_pages", n, dev)
    _flat(v_pages, dtype, "v_pages", n, dev)
    S = seq_lens.numel()
    _flat(seq_lens, torch.int32, "seq_lens", S, dev)
    _flat(q_starts, torch.int32, "q_starts", S + 1, dev)
    if page_table.dim() != 2 or page_table.shape[0] != S:
        raise ValueError(f"page_table: expected [{S}, pages], got {tuple(page_table.shape)}")
    width = page_table.shape[1]
    _flat(page_table, torch.int32, "page_table", S * width, dev)
    if D != dim:
        raise ValueError(f"q of {dim} dims, pages of {D}")
    return _lib.KvView(k_pages.data_ptr(), v_pages.data_ptr(), page_table.data_ptr(),
                       q_starts.data_ptr(), seq_lens.data_ptr(), P, H, page, D, dt, S, width)


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
    _dt16(q, "q")
    dev = q.get_device()
    if dev != torch._C._cuda_getDevice():
        return _elsewhere(rope_cache, dev, q, k, v, k_pages, v_pages, page_table, q_starts,
                          seq_lens, freqs, interleaved, mscale, q_weight, k_weight, eps, out,
                          stream)
    shape, dtype = q.shape, q.dtype
    if len(shape) != 3:
        raise ValueError(f"q: expected [T, H, D], got {tuple(shape)}")
    T, H, D = shape
    kv = _kv_view(dtype, D, k_pages, v_pages, page_table, q_starts, seq_lens, dev)
    qs = _rows(q, "q", dtype, shape, dev)
    new = (T, kv.kv_heads, D)
    ks = _rows(k, "k", dtype, new, dev)
    vs = _rows(v, "v", dtype, new, dev)
    half = freqs.numel()
    _flat(freqs, torch.float64, "freqs", half, dev)
    qw = kw = None
    if q_weight is not None:
        _flat(q_weight, dtype, "q_weight", D, dev)
        qw = q_weight.data_ptr()
    if k_weight is not None:
        _flat(k_weight, dtype, "k_weight", D, dev)
        kw = k_weight.data_ptr()
    side, handle = _on(stream, dev)
    if out is None:
        out = _new(q, shape, dtype, side)
    else:
        _flat(out, dtype, "out", T * H * D, dev)
    _lib.check(_lib.lib().moe_rope_cache(
        C.byref(kv), q.data_ptr(), qs[0], qs[1], k.data_ptr(), ks[0], ks[1], v.data_ptr(), vs[0],
        vs[1], T, H, freqs.data_ptr(), 2 * half, interleaved, mscale, qw, kw, eps, out.data_ptr(),
        handle))
    return out


def attn_paged(q: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor,
               page_table: torch.Tensor, q_starts: torch.Tensor, seq_lens: torch.Tensor,
               scale: float | None = None, window: int = 0, sinks: torch.Tensor | None = None,
               out: torch.Tensor | None = None, stream=None,
               workspace: torch.Tensor | None = None) -> torch.Tensor:
    """Causal attention of T new tokens over the paged cache that holds their keys and
    values already (rope_cache's arguments and batch).  Returns [T, H, D].

    q [T, H, D] with 16-byte aligned heads at any token and head strides; head h reads
    key head h // (H / HK); scale in [0, 1e30], D^-0.5 by default.  window > 0: a row sees the last
    `window` positions up to its own.  sinks fp32 [H]: exp(sinks[h]) joins the softmax's
    sum.  D is 64 or 128.  A row that sees no key is zero; keys that a row does not see
    have no influence, whatever their bits.  Rows behind the last sequence are left as
    they were (in a new output: undefined).  workspace: uint8 on q's device,
    moe_attn_paged_workspace bytes, by default one of the stream's own."""
    _dt16(q, "q")
    dev = q.get_device()
    if dev != torch._C._cuda_getDevice():
        return _elsewhere(attn_paged, dev, q, k_pages, v_pages, page_table, q_starts, seq_lens,
                          scale, window, sinks, out, stream, workspace)
    shape, dtype = q.shape, q.dtype
    if len(shape) != 3:
        raise ValueError(f"q: expected [T, H, D], got {tuple(shape)}")
    T, H, D = shape
    kv = _kv_view(dtype, D, k_pages, v_pages, page_table, q_starts, seq_lens, dev)
    qs = _rows(q, "q", dtype, shape, dev)
    if sinks is not None:
        _flat(sinks, torch.float32, "sinks", H, dev)
    side, handle = _on(stream, dev)
    if out is None:
        out = _new(q, shape, dtype, side)
    else:
        _flat(out, dtype, "out", T * H * D, dev)
    L, view = _lib.lib(), C.byref(kv)
    ws = workspace
    if ws is not None:
        _flat(ws, torch.uint8, "workspace", ws.numel(), dev)
    else:
        need = L.moe_attn_paged_workspace(view, T, H, window)
        if need:
            ws = _WS.get("attn_paged", need, q.device, handle, side=side)
    _lib.check(L.moe_attn_paged(
        view, q.data_ptr(), qs[0] if T > 1 else 0, qs[1] if H > 1 else 0, T, H,
        D ** -0.5 if scale is None else scale, window, _p(sinks), out.data_ptr(), _p(ws),
        0 if ws is None else ws.numel(), handle))
    return out
