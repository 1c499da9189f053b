"""torch-facing wrappers of the C ABI: allocate outputs, pass raw pointers and
the current CUDA stream, raise on a non-zero status.

Every function runs the sm_100a kernels; tensors on the CPU are copied to the
current CUDA device first and results are returned on the input's device, so
the functions can stand in for the reference emulators that take CPU tensors.
"""
from __future__ import annotations

import ctypes
import threading

import torch

from . import _lib
from ._lib import (DTYPE_BF16, DTYPE_F16, DTYPE_F32, FMT_FP3, FMT_NVFP4, FMT_SPFP2, FMT_SPFP2_V1,
                   FMT_TWOFOUR, LAYOUT_TILED, PATH_TCGEN05, EPILOGUE_SILU, call)

_DT = {torch.float32: DTYPE_F32, torch.bfloat16: DTYPE_BF16, torch.float16: DTYPE_F16}

FORMATS = {"spfp2": FMT_SPFP2, "spfp2_v1": FMT_SPFP2_V1, "fp3": FMT_FP3, "nvfp4": FMT_NVFP4,
           "twofour": FMT_TWOFOUR}


def _dt(t: torch.Tensor) -> int:
    try:
        return _DT[t.dtype]
    except KeyError:
        raise TypeError(f"unsupported dtype {t.dtype}; expected float32, bfloat16 or float16") from None


def _cuda(t: torch.Tensor) -> torch.Tensor:
    if not torch.cuda.is_available():
        raise RuntimeError("spark_b200 needs a CUDA device (no CPU fallback)")
    if not t.is_cuda:
        t = t.to(torch.device("cuda", torch.cuda.current_device()))
    return t.contiguous()


def _p(t):
    return ctypes.c_void_p(t.data_ptr()) if t is not None else None


def _stream(t: torch.Tensor):
    return ctypes.c_void_p(torch.cuda.current_stream(t.device).cuda_stream)


def _bytes(t: torch.Tensor) -> torch.Tensor:
    """uint8 view of a packed buffer (uint8 or float8_e4m3fn)."""
    t = _cuda(t)
    return t.view(torch.uint8) if t.dtype != torch.uint8 else t


def _home(out: torch.Tensor, like: torch.Tensor) -> torch.Tensor:
    return out if like.is_cuda else out.to(like.device)


# ------------------------------------------------------------------ SPFP2
def spfp2_pack(w: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """pack_blockwise_paired: (packed uint8[ceil(nb/2)*5], expv uint8[nb])."""
    x = _cuda(w.detach())
    n = x.numel()
    nb = n // 8
    packed = torch.empty(((nb + 1) // 2) * 5, dtype=torch.uint8, device=x.device)
    expv = torch.empty(nb, dtype=torch.uint8, device=x.device)
    call("spark_spfp2_pack", _p(x), _dt(x), n, _p(packed), _p(expv), _stream(x))
    return _home(packed, w), _home(expv, w)


def spfp2_pack_v1(w: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """pack_blockwise_search(window=2): (packed uint8[nb*3], expv uint8[nb])."""
    x = _cuda(w.detach())
    n = x.numel()
    nb = n // 8
    packed = torch.empty(nb * 3, dtype=torch.uint8, device=x.device)
    expv = torch.empty(nb, dtype=torch.uint8, device=x.device)
    call("spark_spfp2_pack_v1", _p(x), _dt(x), n, _p(packed), _p(expv), _stream(x))
    return _home(packed, w), _home(expv, w)


def spfp2_unpack(packed: torch.Tensor, n_elements: int, dtype=torch.float32) -> torch.Tensor:
    """unpack_blockwise_paired."""
    p = _bytes(packed)
    out = torch.empty(n_elements, dtype=dtype, device=p.device)
    if p.numel() < (n_elements + 15) // 16 * 5:
        raise ValueError(f"packed has {p.numel()} bytes, {n_elements} elements need {(n_elements + 15) // 16 * 5}")
    call("spark_spfp2_unpack", _p(p), n_elements, _p(out), _DT[dtype], _stream(p))
    return _home(out, packed)


def spfp2_unpack_v1(packed: torch.Tensor, dtype=torch.float32) -> torch.Tensor:
    """unpack_blockwise (3-byte blocks)."""
    p = _bytes(packed)
    nb = p.numel() // 3
    out = torch.empty(nb * 8, dtype=dtype, device=p.device)
    call("spark_spfp2_unpack_v1", _p(p), nb, _p(out), _DT[dtype], _stream(p))
    return _home(out, packed)


def spfp2_fake_quant(w: torch.Tensor, out_dtype=None) -> torch.Tensor:
    """channel_fake_quantize forward over the flattened tensor's 8-blocks."""
    x = _cuda(w.detach())
    out = torch.empty(x.shape, dtype=out_dtype or x.dtype, device=x.device)
    call("spark_spfp2_fake_quant", _p(x), _dt(x), x.numel(), _p(out), _dt(out), _stream(x))
    return _home(out, w)


# ------------------------------------------------------------------ FP3 / NVFP4
def _codes_shapes(oc: int, ic: int):
    nb = (ic + 15) // 16
    return oc * nb, oc * nb * 16


def fp3_pack(w: torch.Tensor, nibble: bool = False) -> tuple[torch.Tensor, torch.Tensor]:
    """fp3_pack_3bit (nibble=False) or fp3_pack (nibble=True): (codes, scales e4m3fn)."""
    x = _cuda(w.detach())
    oc, ic = x.shape
    nblk, n = _codes_shapes(oc, ic)
    codes = torch.empty((n + 1) // 2 if nibble else (n + 7) // 8 * 3, dtype=torch.uint8, device=x.device)
    scales = torch.empty(nblk, dtype=torch.uint8, device=x.device)
    call("spark_fp3_pack_nibble" if nibble else "spark_fp3_pack", _p(x), _dt(x), oc, ic, _p(codes), _p(scales),
         _stream(x))
    return _home(codes, w), _home(scales.view(torch.float8_e4m3fn), w)


def fp3_unpack(codes: torch.Tensor, scales: torch.Tensor, oc: int, ic: int, nibble: bool = False,
               dtype=torch.float32) -> torch.Tensor:
    c, s = _bytes(codes), _bytes(scales)
    out = torch.empty(oc, ic, dtype=dtype, device=c.device)
    call("spark_fp3_unpack_nibble" if nibble else "spark_fp3_unpack", _p(c), _p(s), oc, ic, _p(out), _DT[dtype],
         _stream(c))
    return _home(out, codes)


def fp3_fake_quant(w: torch.Tensor, out_dtype=None) -> torch.Tensor:
    x = _cuda(w.detach())
    oc, ic = x.shape
    out = torch.empty(oc, ic, dtype=out_dtype or torch.float32, device=x.device)
    call("spark_fp3_fake_quant", _p(x), _dt(x), oc, ic, _p(out), _dt(out), _stream(x))
    return _home(out, w)


def nvfp4_pack(w: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    x = _cuda(w.detach())
    oc, ic = x.shape
    nblk, n = _codes_shapes(oc, ic)
    codes = torch.empty((n + 1) // 2, dtype=torch.uint8, device=x.device)
    scales = torch.empty(nblk, dtype=torch.uint8, device=x.device)
    call("spark_nvfp4_pack", _p(x), _dt(x), oc, ic, _p(codes), _p(scales), _stream(x))
    return _home(codes, w), _home(scales.view(torch.float8_e4m3fn), w)


def nvfp4_unpack(codes: torch.Tensor, scales: torch.Tensor, oc: int, ic: int, dtype=torch.float32) -> torch.Tensor:
    c, s = _bytes(codes), _bytes(scales)
    out = torch.empty(oc, ic, dtype=dtype, device=c.device)
    call("spark_nvfp4_unpack", _p(c), _p(s), oc, ic, _p(out), _DT[dtype], _stream(c))
    return _home(out, codes)


def nvfp4_native_linear(codes: torch.Tensor, scales: torch.Tensor, x: torch.Tensor, oc: int, ic: int,
                        out_dtype=torch.bfloat16, xq=None) -> torch.Tensor:
    """Native NVFP4 x NVFP4 linear (spark_nvfp4_native_linear, a reported mode:
    the activations are quantised to NVFP4 by the weights' own quantiser, so
    the result differs from the parity path `linear("nvfp4", ...)` by the
    activations' FP4 rounding).  codes / scales: nvfp4_pack of the weight;
    x: [M, ic]; xq: an already packed (codes, scales) of x, to skip that step."""
    xc, xs = nvfp4_pack(x) if xq is None else xq
    M = x.shape[0]
    y = torch.empty(M, oc, dtype=out_dtype, device=x.device)
    ws = workspace(x.device, 1 << 20)
    call("spark_nvfp4_native_linear", _p(_bytes(codes)), _p(_bytes(scales)), _p(_bytes(xc)), _p(_bytes(xs)), M, oc,
         ic, _p(y), _dt(y), oc, _p(ws), _stream(x))
    return y


def twofour_sparse_linear(packed: torch.Tensor, x: torch.Tensor, oc: int, ic: int, bias=None,
                          out_dtype=torch.bfloat16) -> torch.Tensor:
    """2:4 linear on the sparse tensor cores (spark_twofour_sparse_linear):
    the kept values of every group of four with their positions as the MMA's
    sparsity metadata.  x: bf16 [M, ic]; packed: twofour_pack of [oc, ic]."""
    x2 = _cuda(x).contiguous()
    if x2.dtype != torch.bfloat16:
        raise TypeError("twofour_sparse_linear: bf16 activations")
    M = x2.shape[0]
    y = torch.empty(M, oc, dtype=out_dtype, device=x2.device)
    ws = workspace(x2.device, 1 << 20)
    b = _cuda(bias) if bias is not None else None
    call("spark_twofour_sparse_linear", _p(_bytes(packed)), _p(x2), M, oc, ic, _p(b), _dt(b) if b is not None else 0,
         _p(y), _dt(y), oc, _p(ws), _stream(x2))
    return y


def nvfp4_fake_quant(w: torch.Tensor, out_dtype=None) -> torch.Tensor:
    x = _cuda(w.detach())
    oc, ic = x.shape
    out = torch.empty(oc, ic, dtype=out_dtype or torch.float32, device=x.device)
    call("spark_nvfp4_fake_quant", _p(x), _dt(x), oc, ic, _p(out), _dt(out), _stream(x))
    return _home(out, w)


# ------------------------------------------------------------------ 2:4
def nvfp4_embedding(codes: torch.Tensor, scales: torch.Tensor, num_embeddings: int, dim: int,
                    ids: torch.Tensor, dtype=torch.float32) -> torch.Tensor:
    """Rows `ids` of a packed NVFP4 [num_embeddings, dim] table, decoded:
    F.embedding(ids, nvfp4_unpack(table)) without unpacking the table.  Out-of-
    range ids give zero rows and an error that check_device_errors() raises."""
    if not ids.is_cuda:
        raise RuntimeError("spark_b200.nvfp4_embedding: ids must be a CUDA tensor")
    flat = ids.reshape(-1).to(torch.int64).contiguous()
    out = torch.empty(flat.numel(), dim, dtype=dtype, device=ids.device)
    if out.numel() == 0:
        return out.reshape(*ids.shape, dim)
    ws = workspace(ids.device, 1 << 20)
    call("spark_nvfp4_embedding", _p(_bytes(codes)), _p(_bytes(scales)), num_embeddings, dim, _p(flat), flat.numel(),
         _p(out), _dt(out), _p(ws), _stream(ids))
    return out.reshape(*ids.shape, dim)


def twofour_pack(w: torch.Tensor) -> torch.Tensor:
    x = _cuda(w.detach())
    oc, ic = x.shape
    nblk, _ = _codes_shapes(oc, ic)
    packed = torch.empty((nblk + 1) // 2 * 7, dtype=torch.uint8, device=x.device)
    call("spark_twofour_pack", _p(x), _dt(x), oc, ic, _p(packed), _stream(x))
    return _home(packed, w)


def twofour_unpack(packed: torch.Tensor, n_elements: int, dtype=torch.float32) -> torch.Tensor:
    p = _bytes(packed)
    out = torch.empty(n_elements, dtype=dtype, device=p.device)
    call("spark_twofour_unpack", _p(p), n_elements, _p(out), _DT[dtype], _stream(p))
    return _home(out, packed)


def twofour_fake_quant(w: torch.Tensor, out_dtype=None) -> torch.Tensor:
    x = _cuda(w.detach())
    out = torch.empty(x.shape, dtype=out_dtype or x.dtype, device=x.device)
    call("spark_twofour_fake_quant", _p(x), _dt(x), x.numel(), _p(out), _dt(out), _stream(x))
    return _home(out, w)


# ------------------------------------------------------------------ INT8
def int8_fake_quant(w: torch.Tensor, out_dtype=None) -> torch.Tensor:
    """int8_fake_quant: per-row symmetric INT8 round trip (fp32 out by default)."""
    x = _cuda(w.detach())
    oc, ic = x.shape
    out = torch.empty(oc, ic, dtype=out_dtype or torch.float32, device=x.device)
    call("spark_int8_fake_quant", _p(x), _dt(x), oc, ic, _p(out), _dt(out), _stream(x))
    return _home(out, w)


def int8_pack(w: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """ptq_int8_pack: (q int8 [oc, ic], scale fp32 [oc])."""
    x = _cuda(w.detach())
    oc, ic = x.shape
    q = torch.empty(oc, ic, dtype=torch.int8, device=x.device)
    scale = torch.empty(oc, dtype=torch.float32, device=x.device)
    call("spark_int8_pack", _p(x), _dt(x), oc, ic, _p(q), _p(scale), _stream(x))
    return _home(q, w), _home(scale, w)


def int8_unpack(q: torch.Tensor, scale: torch.Tensor, dtype=torch.float32) -> torch.Tensor:
    """ptq_int8_unpack: q * scale[row]."""
    qq, s = _cuda(q), _cuda(scale.float())
    oc, ic = qq.shape
    out = torch.empty(oc, ic, dtype=dtype, device=qq.device)
    call("spark_int8_unpack", _p(qq), _p(s), oc, ic, _p(out), _DT[dtype], _stream(qq))
    return _home(out, q)


# ------------------------------------------------------------------ linear
_ws_lock = threading.Lock()
_ws: dict[tuple[int, int], torch.Tensor] = {}


def _zeroed(nbytes: int, device: torch.device) -> torch.Tensor:
    """Zeros to keep between calls.  Where the current stream is being captured the fill
    would be a node of that graph, which its replays alone run, and each of them, and the
    memory the graph's, shared with its other tensors: there they are allocated and
    filled on another stream at once."""
    with torch.cuda.device(device):
        if not torch.cuda.is_current_stream_capturing():
            return torch.zeros(nbytes, dtype=torch.uint8, device=device)
        mode = ctypes.c_int(2)      # relaxed: this thread may allocate and wait beside the capture
        call("spark_capture_mode", ctypes.byref(mode))
        try:
            while True:
                side = torch.cuda.Stream()      # (of a pool, in turn: the captured stream is one of them)
                with torch.cuda.stream(side):
                    if not torch.cuda.is_current_stream_capturing():
                        buf = torch.zeros(nbytes, dtype=torch.uint8, device=device)
                        side.synchronize()
                        return buf
        finally:
            call("spark_capture_mode", ctypes.byref(mode))


def workspace(device: torch.device, nbytes: int, stream=None) -> torch.Tensor:
    """Zero-initialised scratch for spark_linear, one per (device, stream)."""
    s = stream if stream is not None else torch.cuda.current_stream(device)
    key = (device.index if device.index is not None else torch.cuda.current_device(), s.cuda_stream)
    with _ws_lock:
        buf = _ws.get(key)
        if buf is None or buf.numel() < nbytes:
            with torch.cuda.stream(s):
                buf = _zeroed(max(nbytes, 1 << 20), device)
            _ws[key] = buf
    return buf


def workspace_size(fmt: int, M: int, oc: int, ic: int) -> int:
    return int(_lib.lib().spark_linear_workspace_size(fmt, M, oc, ic))


def tiled_bytes(fmt, oc: int, ic: int) -> int:
    f = FORMATS[fmt] if isinstance(fmt, str) else int(fmt)
    return int(_lib.lib().spark_tiled_bytes(f, oc, ic))


def tile_weights(fmt, wq: torch.Tensor, scales, oc: int, ic: int) -> torch.Tensor | None:
    """Fragment-major copy of a packed weight for the decode GEMV (None when the
    shape has no tiled layout).  Same bytes, permuted; scales embedded."""
    f = FORMATS[fmt] if isinstance(fmt, str) else int(fmt)
    n = tiled_bytes(f, oc, ic)
    if n == 0:
        return None
    w = _bytes(wq)
    s = _bytes(scales) if scales is not None else None
    out = torch.empty(n, dtype=torch.uint8, device=w.device)
    call("spark_tile_weights", f, _p(w), _p(s), oc, ic, _p(out), _stream(w))
    return out


def linear(fmt, wq: torch.Tensor, scales, x: torch.Tensor, oc: int, ic: int, bias=None, out_dtype=None,
           out: torch.Tensor | None = None, tiled: bool = False, tcgen05: bool = False,
           prefetch: torch.Tensor | None = None, silu: bool = False) -> torch.Tensor:
    """y[..., oc] = x[..., ic] . decode(W)^T (+ bias) with W packed in `fmt`
    (reference layout, or the tile_weights copy with tiled=True).  tcgen05=True
    runs the tensor-memory kernel (SPFP2 reference layout, bf16 x).  prefetch:
    a tensor (typically the next layer's weight) the decode GEMV pulls into L2
    while it runs.  silu: the weight holds gate/up rows in groups of 8 + 8
    (V3GateUpSiLU) and the result is SiLU(gate) * up, oc // 2 wide (decode
    GEMV paths)."""
    f = FORMATS[fmt] if isinstance(fmt, str) else int(fmt)
    if tcgen05:
        f |= PATH_TCGEN05
    if tiled:
        f |= LAYOUT_TILED
        scales = None
    if silu:
        f |= EPILOGUE_SILU
    if not x.is_cuda:
        raise RuntimeError("spark_b200.linear: x must be a CUDA tensor")
    lead = x.shape[:-1]
    if x.shape[-1] != ic:
        raise ValueError(f"x has {x.shape[-1]} features, the weight has {ic}")
    x2 = x.reshape(-1, ic)
    if x2.stride(-1) != 1:
        x2 = x2.contiguous()
    M = x2.shape[0]
    w = _bytes(wq)
    s = _bytes(scales) if scales is not None else None
    b = bias.contiguous() if bias is not None else None
    width = oc // 2 if silu else oc
    y = out if out is not None else torch.empty(M, width, dtype=out_dtype or x.dtype, device=x.device)
    nbytes = workspace_size(f & 0xff, M, oc, ic)
    ws = workspace(x.device, nbytes)
    if prefetch is None:
        call("spark_linear", f, _p(w), _p(s), _p(x2), _dt(x2), M, oc, ic, x2.stride(0), _p(b),
             _dt(b) if b is not None else DTYPE_F32, _p(y), _dt(y), y.stride(0), _p(ws), ws.numel(), _stream(x))
    else:
        call("spark_linear_prefetch", f, _p(w), _p(s), _p(x2), _dt(x2), M, oc, ic, x2.stride(0), _p(b),
             _dt(b) if b is not None else DTYPE_F32, _p(y), _dt(y), y.stride(0), _p(ws), ws.numel(),
             _p(prefetch), prefetch.numel() * prefetch.element_size(), _stream(x))
    return y.reshape(*lead, width)


class ChainOp:
    """One op of linear_chain: a dequant linear or SiLU(gate) * up.

    Linear: ChainOp("linear", fmt=, wq=, scales=, x=, y=, bias=, deps=[...]).
    SiLU:   ChainOp("silu_mul", x=gate, x2=up, y=out, deps=[gate op, up op]).
    deps: indices of earlier ops whose output this op reads."""

    def __init__(self, kind, x, y, fmt="spfp2", wq=None, scales=None, x2=None, bias=None, deps=()):
        self.kind, self.fmt, self.wq, self.scales, self.x, self.x2, self.y = kind, fmt, wq, scales, x, x2, y
        self.bias, self.deps = bias, list(deps)


_chain_ws: dict[tuple[int, int], torch.Tensor] = {}


def linear_chain(chain: list[ChainOp], stream=None) -> None:
    """Run the ops in one persistent launch (spark_linear_chain).  Outputs are
    the caller's preallocated y tensors; every activation is bf16 [M, n]."""
    if not chain:
        return
    x0 = chain[0].x
    M = x0.shape[0]
    arr = (_lib.SparkChainOp * len(chain))()
    keep = []
    for k, op in enumerate(chain):
        c = arr[k]
        deps = op.deps + [-1] * (2 - len(op.deps))
        c.dep[0], c.dep[1] = deps[0], deps[1]
        c.x, c.y = op.x.data_ptr(), op.y.data_ptr()
        if op.kind == "silu_mul":
            c.kind, c.x2, c.ic = _lib.CHAIN_SILU_MUL, op.x2.data_ptr(), op.x.shape[1]
            continue
        f = FORMATS[op.fmt] if isinstance(op.fmt, str) else int(op.fmt)
        w = _bytes(op.wq)
        s = _bytes(op.scales) if op.scales is not None else None
        keep += [w, s]
        oc = op.y.shape[1]
        c.kind, c.fmt, c.wq, c.scales = _lib.CHAIN_LINEAR, f, w.data_ptr(), (s.data_ptr() if s is not None else None)
        c.ic, c.ldx, c.oc, c.ldy, c.y_dtype = op.x.shape[1], op.x.stride(0), oc, op.y.stride(0), _dt(op.y)
        if op.bias is not None:
            c.bias, c.bias_dtype = op.bias.data_ptr(), _dt(op.bias)
    n = int(_lib.lib().spark_linear_chain_workspace_size(len(chain)))
    st = stream if stream is not None else torch.cuda.current_stream(x0.device)
    key = (x0.device.index, st.cuda_stream)
    ws = _chain_ws.get(key)
    if ws is None or ws.numel() < n:
        with torch.cuda.stream(st):
            ws = _zeroed(n, x0.device)
        _chain_ws[key] = ws
    call("spark_linear_chain", ctypes.cast(arr, ctypes.c_void_p), len(chain), M, _p(ws), ws.numel(),
         ctypes.c_void_p(st.cuda_stream))


class BatchOp:
    """One linear of linear_batch: y = x . decode(W)^T (+ bias) on tiled weights
    (tile_weights), bf16 x [M, ic]; silu: the weight holds gate/up rows in
    groups of 8 + 8 and y = SiLU(gate) * up, oc // 2 wide.  deps: indices of
    earlier ops of the batch whose output this op reads."""

    def __init__(self, fmt, wq_tiled: torch.Tensor, x: torch.Tensor, y: torch.Tensor, bias=None,
                 silu: bool = False, deps=()):
        self.fmt, self.wq, self.x, self.y, self.bias, self.silu, self.deps = fmt, wq_tiled, x, y, bias, silu, list(deps)


def _batch_array(batch: list[BatchOp]):
    arr = (_lib.SparkChainOp * len(batch))()
    for k, op in enumerate(batch):
        c = arr[k]
        if op.x.dtype != torch.bfloat16:
            raise TypeError("linear_batch: activations must be bfloat16")
        if op.x.dim() != 2 or op.x.stride(1) != 1 or op.y.dim() != 2 or op.y.stride(1) != 1:
            raise ValueError("linear_batch: x and y must be 2-D with unit column stride")
        deps = op.deps + [-1] * (2 - len(op.deps))
        if len(deps) > 2:
            raise ValueError("linear_batch: at most two deps per op")
        f = FORMATS[op.fmt] if isinstance(op.fmt, str) else int(op.fmt)
        c.kind, c.fmt = _lib.CHAIN_LINEAR, f | LAYOUT_TILED | (EPILOGUE_SILU if op.silu else 0)
        c.wq, c.scales = _bytes(op.wq).data_ptr(), None
        c.x, c.ic, c.ldx = op.x.data_ptr(), op.x.shape[1], op.x.stride(0)
        c.oc = op.y.shape[1] * (2 if op.silu else 1)
        c.y, c.y_dtype, c.ldy = op.y.data_ptr(), _dt(op.y), op.y.stride(0)
        if op.bias is not None:
            c.bias, c.bias_dtype = op.bias.data_ptr(), _dt(op.bias)
        c.dep[0], c.dep[1] = deps[0], deps[1]
    return arr


def linear_batch(batch: list[BatchOp], stream=None) -> None:
    """Run the linears in one persistent launch (spark_linear_batch).  Every op
    shares the token count M (rows of x); outputs are the ops' preallocated y."""
    if not batch:
        return
    x0 = batch[0].x
    M = x0.shape[0]
    arr = _batch_array(batch)
    st = stream if stream is not None else torch.cuda.current_stream(x0.device)
    n = int(_lib.lib().spark_linear_batch_workspace_size(ctypes.cast(arr, ctypes.c_void_p), len(batch), M))
    if n == 0:
        # an invalid batch: let the call itself report why
        n = 1 << 20
    ws = workspace(x0.device, n, stream=st)
    call("spark_linear_batch", ctypes.cast(arr, ctypes.c_void_p), len(batch), M, _p(ws), ws.numel(),
         ctypes.c_void_p(st.cuda_stream))


def linear_batch_allreduce(batch: list[BatchOp], op: int, world: int, rank: int, recv_ptrs, counter: torch.Tensor,
                           stream=None) -> None:
    """linear_batch whose op `op` is all-reduced over `world` ranks inside the
    same launch (spark_linear_batch_ar): every rank runs the same batch on its
    own shard (e.g. the K-sharded down projection of a tensor-parallel MLP)
    and gets the rank-order sum of the ranks' fp32 results (+ bias) in that
    op's y.  recv_ptrs: device addresses of every rank's receive buffer, as
    this process maps them; counter: this rank's call counter (one int32).
    tp.BatchAllReduce shares and owns both."""
    if not batch:
        raise ValueError("linear_batch_allreduce: empty batch")
    x0 = batch[0].x
    M = x0.shape[0]
    arr = _batch_array(batch)
    recv = (ctypes.c_void_p * world)(*recv_ptrs)
    ar = _lib.SparkBatchAllReduce(op, world, rank, ctypes.cast(recv, ctypes.c_void_p), counter.data_ptr())
    st = stream if stream is not None else torch.cuda.current_stream(x0.device)
    n = int(_lib.lib().spark_linear_batch_ar_workspace_size(ctypes.cast(arr, ctypes.c_void_p), len(batch), M,
                                                             ctypes.byref(ar)))
    ws = workspace(x0.device, n if n else 1 << 20, stream=st)
    call("spark_linear_batch_ar", ctypes.cast(arr, ctypes.c_void_p), len(batch), M, ctypes.byref(ar), _p(ws),
         ws.numel(), ctypes.c_void_p(st.cuda_stream))


def check_device_errors(device=None) -> None:
    """Raise if a kernel left an error in a workspace.  Synchronises the devices: a
    workspace is used on its stream, and by the graphs captured there on any."""
    all_ws = list(_ws.items()) + list(_chain_ws.items()) + list(_tree_ws.items()) + _tree_outgrown
    for dev in {dev for (dev, _), _ in all_ws if device is None or dev == device}:
        torch.cuda.synchronize(dev)
    for (dev, sh), buf in all_ws:
        if device is not None and dev != device:
            continue
        try:
            call("spark_workspace_check", _p(buf), ctypes.c_void_p(sh))
        except _lib.SparkError:
            if any(buf is other for _, other in [*_tree_ws.items(), *_tree_outgrown]):
                # an expired wait may leave its counters behind; cleared before the next launch on any stream
                stream = torch.cuda.ExternalStream(sh, device=buf.device)
                with torch.cuda.stream(stream):
                    buf[:_lib.TREE_ATTENTION_ZEROED].zero_()
                stream.synchronize()
            raise


def silu_mul(gate: torch.Tensor, up: torch.Tensor) -> torch.Tensor:
    """SiLU(gate) * up.  2-D views with unit column stride and a common row
    stride (the two halves of a row-merged gate|up output) are read in place."""
    if gate.shape != up.shape:
        raise ValueError("silu_mul: gate and up shapes differ")
    if (gate.dim() == 2 and gate.stride(1) == 1 and up.stride(1) == 1 and gate.stride(0) == up.stride(0)
            and gate.dtype == up.dtype):
        rows, cols = gate.shape
        out = torch.empty(rows, cols, dtype=gate.dtype, device=gate.device)
        call("spark_silu_mul_rows", _p(gate), _p(up), gate.stride(0), _p(out), cols, _dt(gate), rows, cols,
             _stream(gate))
        return out
    g, u = gate.contiguous(), up.contiguous()
    out = torch.empty_like(g)
    call("spark_silu_mul", _p(g), _p(u), _p(out), _dt(g), g.numel(), _stream(g))
    return out


# ------------------------------------------------------------------ tree decoding
MAX_TREE_NODES = 64    # of one sequence in tree_attention (SPARK_MAX_TREE_NODES)

_tree_ws: dict[tuple[int, int], torch.Tensor] = {}
_tree_outgrown: list[tuple[tuple[int, int], torch.Tensor]] = []
_native_module = None


def _native():
    """spark_b200._native: checks, outputs and the C call of the functions below."""
    global _native_module
    if _native_module is None:
        _lib.lib()
        try:
            from . import _native as module
        except ImportError as e:
            raise RuntimeError("spark_b200._native is missing or does not load: build it with "
                               "`python -c 'import __graft_entry__ as g; g.build()'`") from e
        _native_module = module
    return _native_module


def _check(name: str, rc: int) -> None:
    if rc != _lib.OK:
        raise _lib.SparkError(name, rc, _lib.last_error())


def _tree_workspace(device: torch.device, stream: int, nbytes: int = 256) -> torch.Tensor:
    """Scratch of the tree-decoding calls, one per (device, stream): an error word,
    counters that are zero between calls, then partial results.  A larger one takes its
    place when a call needs it; the old one stays, with the errors left in it, for the
    CUDA graphs and backward passes that have its address."""
    key = (device.index, stream)
    buf = _tree_ws.get(key)
    if buf is None or buf.numel() < nbytes:
        with _ws_lock:
            buf = _tree_ws.get(key)
            if buf is None or buf.numel() < nbytes:
                if buf is not None:
                    _tree_outgrown.append((key, buf))
                    nbytes = max(nbytes, 2 * buf.numel())     # (all the old ones together are no larger)
                buf = _zeroed(max(nbytes, 1 << 16), device)
                _tree_ws[key] = buf
    return buf


def _place(what: str, t: torch.Tensor, nbytes: int = 256):
    """(workspace, its address, the current stream's handle) on t's device."""
    index = t.get_device()
    if index < 0:
        raise RuntimeError(f"spark_b200.{what}: expected a CUDA tensor, got one on {t.device}")
    # (torch.cuda.current_stream builds an object for it, 2 us)
    stream = torch._C._cuda_getCurrentRawStream(index)
    ws = _tree_workspace(t.device, stream, nbytes)
    return ws, ws.data_ptr(), stream


def _stream_of(what: str, t: torch.Tensor) -> int:
    """The current stream's handle on t's device."""
    index = t.get_device()
    if index < 0:
        raise RuntimeError(f"spark_b200.{what}: expected a CUDA tensor, got one on {t.device}")
    return torch._C._cuda_getCurrentRawStream(index)


def rope(q: torch.Tensor, k: torch.Tensor | None, positions: torch.Tensor, table: torch.Tensor,
         interleaved: bool = False, inverse: bool = False, out=None):
    """Rotary positions of q [..., tokens, heads, head_dim] and k (the same with its
    own heads, or None) in one launch (spark_rope): (q', k').  positions: [...,
    tokens] int32 or int64; table: rotary.rope_table's fp32 [rows, rot_dim], whose
    width says how much of the head turns.  Pairs are (i, i + rot_dim / 2), or
    (2 i, 2 i + 1) when interleaved.  inverse turns back (the backward pass).  Up to
    one leading (batch) dimension; strided views are read in place.  out: (q', k')
    tensors to write to, q and k themselves among them.  A position outside the
    table gives a zero row and an error that check_device_errors() raises."""
    _, ws, stream = _place("rope", q)
    q_out, k_out = (None, None) if out is None else out
    q_out, k_out, rc = _native().rope(q, k, positions, table, interleaved, inverse, q_out, k_out, ws, stream)
    if rc:
        _check("spark_rope", rc)
    return q_out, k_out


def qk_norm_rope(q: torch.Tensor, k: torch.Tensor | None, q_weight: torch.Tensor | None, k_weight: torch.Tensor | None,
                 positions: torch.Tensor, table: torch.Tensor, eps: float = 1e-6, interleaved: bool = False, out=None):
    """RMS norms of q and k for each head and their rotary positions in one launch
    (spark_qk_norm_rope): (q', k'), q' = rope(q / sqrt(mean q^2 + eps) * q_weight).  q [...,
    tokens, heads, head_dim], k, positions, table, interleaved and out as in rope;
    head_dim even, up to 256.  The weights [head_dim] are float32, bfloat16 or float16,
    None for ones.  All in fp32, rounded once.  Not differentiable:
    rotary.apply_qk_norm_rope is the form that is."""
    _, ws, stream = _place("qk_norm_rope", q)
    q_out, k_out = (None, None) if out is None else out
    q_out, k_out, rc = _native().qk_norm_rope(q, k, q_weight, k_weight, positions, table, eps, interleaved, q_out, k_out,
                                              ws, stream)
    if rc:
        _check("spark_qk_norm_rope", rc)
    return q_out, k_out


def kv_append(k_new: torch.Tensor, v_new: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor,
              page_table: torch.Tensor, context_lens: torch.Tensor, index: torch.Tensor | None = None,
              counts: torch.Tensor | None = None) -> torch.Tensor:
    """Writes K/V rows of new tokens [batch, tokens, kv_heads, head_dim] into the paged
    cache [pages, page_size, kv_heads, head_dim] behind each sequence's context_lens
    tokens (spark_kv_append) and returns the new lengths (int32 [batch], a new tensor).
    index (int32 [batch, n]): which tokens, in order, e.g. tree_verify's path; counts
    (int32 [batch]): how many of them.  Without both, all tokens go in.  What does not
    fit a sequence's pages is left out and reported by check_device_errors()."""
    _, ws, stream = _place("kv_append", k_cache)
    new_lens, rc = _native().kv_append(k_new, v_new, k_cache, v_cache, page_table, context_lens, index, counts, ws, stream)
    if rc:
        _check("spark_kv_append", rc)
    return new_lens


def tree_attention(q: torch.Tensor, k_tree: torch.Tensor, v_tree: torch.Tensor, k_cache: torch.Tensor,
                   v_cache: torch.Tensor, page_table: torch.Tensor, context_lens: torch.Tensor,
                   parents: torch.Tensor, scale: float | None = None, out: torch.Tensor | None = None,
                   return_lse: bool = False):
    """Attention of up to 64 drafted tokens per sequence (a tree) over the paged cache
    and over the tree itself (spark_tree_attention).  q [batch, nodes, q_heads,
    head_dim], k_tree / v_tree [batch, nodes, kv_heads, head_dim] (not in the cache),
    the cache [pages, page_size, kv_heads, head_dim], page_table int32 [batch,
    max_pages], context_lens int32 [batch], parents int32 [batch, nodes] or [nodes]:
    -1 hangs a node on the context, j < i node i on node j, -2 marks it unused (a zero
    row).  Each node sees the context, itself and its ancestors.  scale defaults to
    head_dim ** -0.5, it must be positive.  page_size and head_dim (up to 256) must be
    multiples of 8, q_heads at most 128 times kv_heads.  Returns out [batch, nodes, q_heads, head_dim], with return_lse
    also the natural log of the softmax sums, fp32 [batch, nodes, q_heads]."""
    ws, ptr, stream = _place("tree_attention", q)
    args = (q, k_tree, v_tree, k_cache, v_cache, page_table, context_lens, parents, scale)
    out, lse, rc, need = _native().tree_attention(*args, out, return_lse, ptr, ws.numel(), stream)
    if rc == _lib.ERR_WORKSPACE and need > ws.numel():
        ws, ptr, stream = _place("tree_attention", q, need)
        out, lse, rc, need = _native().tree_attention(*args, out, return_lse, ptr, ws.numel(), stream)
    if rc:
        _check("spark_tree_attention", rc)
    return (out, lse) if return_lse else out


def tree_verify(logits: torch.Tensor, tokens: torch.Tensor, parents: torch.Tensor, uniforms: torch.Tensor,
                noise: torch.Tensor, draft_probs: torch.Tensor | None = None,
                temperature: torch.Tensor | float = 1.0):
    """Verification of a drafted tree by rejection sampling (spark_tree_verify).
    logits [batch, nodes, vocab]: the target's at every node; tokens int64 and parents
    int32 [batch, nodes] (parents also [nodes]); node 0 is the last token already
    accepted.  uniforms fp32 [batch, nodes] in [0, 1), noise fp32 [batch, vocab]
    exponential variates.  draft_probs [batch, nodes, vocab]: the distribution that
    each node's children were sampled from (independently); None for deterministic
    children.  temperature: a number or fp32 [batch]; 0 takes the argmax.  Returns
    path int32 [batch, nodes] (accepted nodes from node 0, then -1), accepted int32
    [batch] (how many) and next int64 [batch], the token after them (-1 where the
    logits give no distribution)."""
    _, ws, stream = _place("tree_verify", logits)
    if not isinstance(temperature, torch.Tensor):
        temperature = None if temperature == 1.0 else torch.full((logits.shape[0],), float(temperature), device=logits.device)
    path, accepted, last, rc = _native().tree_verify(logits, tokens, parents, uniforms, noise, draft_probs, temperature, ws,
                                                     stream)
    if rc:
        _check("spark_tree_verify", rc)
    return path, accepted, last


# ------------------------------------------------------------------ sampling
def sample(logits: torch.Tensor, noise: torch.Tensor, temperature: torch.Tensor | float = 1.0, top_k: torch.Tensor | int = 0,
           top_p: torch.Tensor | float = 1.0, min_p: torch.Tensor | float = 0.0, return_logprob: bool = False):
    """Tokens drawn from logits [batch, vocab] with the given random numbers (spark_sample):
    int64 [batch]; with return_logprob also the log of the probability that each was drawn
    with, fp32 [batch].  noise fp32 [batch, vocab]: exponential variates, as tree_verify's;
    equal ones give equal tokens.  Of the distribution at the temperature stay the top_k
    likeliest tokens (0: all), of those the fewest that have top_p of their mass, of those
    the ones at least min_p as likely as the likeliest.  Temperature 0 takes the argmax.
    Settings are numbers or tensors [batch], top_k int32, the others fp32.  A row without a
    distribution (a NaN, +inf, nothing above -inf) gives -1 and NaN.  Not differentiable, the
    logarithm neither."""
    stream = _stream_of("sample", logits)
    token, logprob, rc = _native().sample(logits, noise, temperature, top_k, top_p, min_p, return_logprob, stream)
    if rc:
        _check("spark_sample", rc)
    return (token, logprob) if return_logprob else token


def filter_logits(logits: torch.Tensor, temperature: torch.Tensor | float = 1.0, top_k: torch.Tensor | int = 0,
                  top_p: torch.Tensor | float = 1.0, min_p: torch.Tensor | float = 0.0, out: torch.Tensor | None = None) -> torch.Tensor:
    """logits [batch, (nodes,) vocab] with -inf in place of what sample's settings leave out:
    tree_verify of these at the same temperature samples from the cut distribution.  out: a
    tensor to write to, logits themselves for instance.  A row without a distribution is
    copied.  Not differentiable."""
    stream = _stream_of("filter_logits", logits)
    out, rc = _native().filter_logits(logits, temperature, top_k, top_p, min_p, out, stream)
    if rc:
        _check("spark_sample", rc)
    return out


# ------------------------------------------------------------------ adapters
def lora_add(y: torch.Tensor, x: torch.Tensor, a: torch.Tensor, b: torch.Tensor, adapter: torch.Tensor,
             scale: torch.Tensor | float = 1.0, out: torch.Tensor | None = None) -> torch.Tensor:
    """Low-rank adapters of many requests on top of a shared projection's y (spark_lora):
    y[t] + scale[i] * b[i] @ (a[i] @ x[t]), i = the token's adapter, a negative one for none.
    x [..., in_features], y [..., out_features], a pool of a [adapters, rank, in_features] and
    b [adapters, out_features, rank], bfloat16 or float16 alike, y also float32; smaller ranks
    padded with zeros, 256 at most.  adapter int32: one for each token, or for each run of as many
    tokens (of [batch, tokens, ...] one for each sequence).  scale: a number or fp32
    [adapters].  out: a tensor to write to, y itself for instance; otherwise a new one.
    An adapter outside the pool counts as none and is reported by
    check_device_errors().  Not differentiable."""
    _, ws, stream = _place("lora_add", y)
    out, rc = _native().lora_add(y, x, a, b, adapter, scale, out, ws, stream)
    if rc:
        _check("spark_lora", rc)
    return out
