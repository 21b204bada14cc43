"""Microscaled 4-bit floating point (MXFP4): quantisation and products on the tensor cores. No counterpart in the
reference, whose narrowest type is fp8; here it stands beside `GemmOnly` and the grouped ops for serving with weights of
4.25 bits a value.

Format: 32 consecutive values along K share a power of two (e8m0: the exponent + 127 in a byte, 255 = NaN), the values
are e2m1 (0, 0.5, 1, 1.5, 2, 3, 4, 6 and their negatives), two to a byte, the first in the low half.

    w = flux.mx_quantize(weight)                        # once, when the weights are loaded
    y = flux.mx_gemm(flux.mx_quantize(x), w)            # y[M, N] = x[M, K] . weight[N, K]^T
"""
from __future__ import annotations

import math
import threading
from typing import Dict, List, Optional

import torch
from torch.autograd import forward_ad as _forward_ad

from . import _lib
from .moe import _FLOATS, _check_index, _on_device, _refuse_tangent
from .ops import _check, _cur_device, _cur_stream, _ptr, _tuning
from .shm import _LAST, Comm, fluxb_dtype

BLOCK = 32
_COMMS: Dict[int, Comm] = {}
_USED: Dict[int, List[Comm]] = {}  # per device: the communicators whose status word its products were given
_LOCK = threading.Lock()


def _comm() -> Comm:
    """A communicator of the current device, for its status word and time-out: the default one, or, where there is none or it is
    another device's, one of one rank that this module keeps and that does not become the default."""
    dev = _cur_device()
    c = _LAST[0] if _LAST else None
    if c is None or c.device.index != dev:
        c = _COMMS.get(dev)
        if c is None:
            with _LOCK:
                c = _COMMS.get(dev)
                if c is None:
                    c = _COMMS[dev] = Comm(None)
    used = _USED.get(dev)
    if used is None or used[-1] is not c:
        with _LOCK:
            _USED[dev] = [u for u in _USED.get(dev, ()) if u is not c] + [c]  # (the last one that was used last)
    return c


def mx_check_status() -> None:
    """Raise if a bounded wait of a product on the current device has run out, whose output is then incomplete (call after a
    synchronize). It reads the status of every communicator that this device's products have used: the default ones, which
    `Comm.check_status` reads as well, and the one that they make where there is none."""
    for c in _USED.get(_cur_device(), ()):
        c.check_status()


def _check_size(name: str, rows: int, k: int) -> None:
    """The library takes sizes of 31 bits; larger ones would arrive there as others."""
    if k >= 1 << 31:
        raise RuntimeError(f"{name}: K {k} is too large")
    if rows >= 1 << 31:
        raise RuntimeError(f"{name}: {rows} rows are too many")


def _blocks_shape(lead, rows: int, k: int):
    return (*lead, (rows + 127) // 128, (k + 127) // 128, 512)


class MXTensor:
    """Matrices [..., N, K] as packed e2m1 values and scales. The constructor takes them as a checkpoint holds them, `data`
    uint8 [..., N, K / 2] and `scales` uint8 [..., N, K / 32], and lays the scales out once, in the blocks of 128 rows x 4
    scales that the tensor cores read (fluxb.h); `mx_quantize` makes them that way. `data`, `blocks` (the laid-out scales)
    and `scales` (row by row again, a copy) are tensors.

    What a product needs of it is kept as plain numbers, and `mx_quantize` puts values and scales into one allocation, of
    which `data` and `blocks` are views made when asked for: a call's tensor bookkeeping took as long as its launch."""

    __slots__ = ("lead", "rows", "k", "_dev", "_store", "_data", "_blocks", "_data_ptr", "_blocks_ptr")

    def __init__(self, data: torch.Tensor, scales: torch.Tensor):
        _check(_on_device(data) and _on_device(scales), "MXTensor: data and scales must be on the current CUDA device")
        _check(data.dtype == torch.uint8 and scales.dtype == torch.uint8, "MXTensor: data and scales must be uint8")
        _check(data.dim() >= 2 and data.shape[-1] >= BLOCK // 2 and data.shape[-1] % (BLOCK // 2) == 0,
               "MXTensor: data must be [..., N, K / 2] with K a multiple of 32")
        *lead, n, _ = data.shape
        k = data.shape[-1] * 2
        if tuple(scales.shape) != (*lead, n, k // BLOCK):
            raise RuntimeError(f"MXTensor: scales shape {tuple(scales.shape)} != {(*lead, n, k // BLOCK)}")
        _check_size("MXTensor", math.prod(lead) * n, k)
        data = data.contiguous()
        if data.data_ptr() % 16:
            data = data.clone()
        shape = _blocks_shape(lead, n, k)
        rows = torch.zeros((*lead, shape[-3] * 128, shape[-2] * 4), dtype=torch.uint8, device=data.device)
        rows[..., :n, :k // BLOCK] = scales
        # row = 128 block + 32 column + lane, scale = 4 group + s  ->  [block, group, lane, column, s]
        self._set(data, rows.view(-1, shape[-3], 4, 32, shape[-2], 4).permute(0, 1, 4, 3, 2, 5).contiguous().view(shape))

    def _set(self, data: torch.Tensor, blocks: torch.Tensor) -> None:
        *lead, self.rows, half = data.shape
        self.lead, self.k, self._dev = tuple(lead), half * 2, data.get_device()
        self._store, self._data, self._blocks = None, data, blocks
        self._data_ptr, self._blocks_ptr = data.data_ptr(), blocks.data_ptr()

    @classmethod
    def _of(cls, data: torch.Tensor, blocks: torch.Tensor) -> "MXTensor":
        t = cls.__new__(cls)
        t._set(data, blocks)
        return t

    def __getstate__(self):
        return self.data, self.blocks  # (addresses are this object's: copies and what is loaded from a file have their own)

    def __setstate__(self, state) -> None:
        self._set(*state)

    @property
    def data(self) -> torch.Tensor:
        if self._data is None:
            n = math.prod(self.lead) * self.rows * (self.k // 2)
            self._data = self._store[:n].view(*self.lead, self.rows, self.k // 2)
        return self._data

    @property
    def blocks(self) -> torch.Tensor:
        if self._blocks is None:
            self._blocks = self._store[self._blocks_ptr - self._data_ptr:].view(_blocks_shape(self.lead, self.rows, self.k))
        return self._blocks

    @property
    def scales(self) -> torch.Tensor:
        *lead, nb, groups, _ = self.blocks.shape
        rows = self.blocks.view(-1, nb, groups, 32, 4, 4).permute(0, 1, 4, 3, 2, 5).reshape(*lead, nb * 128, groups * 4)
        return rows[..., :self.rows, :self.k // BLOCK].contiguous()

    @property
    def shape(self) -> torch.Size:
        return torch.Size((*self.lead, self.rows, self.k))

    @property
    def device(self) -> torch.device:
        return torch.device("cuda", self._dev)

    def dequantize(self, dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
        return mx_dequantize(self, dtype)

    def __repr__(self) -> str:
        return f"MXTensor(shape={tuple(self.shape)}, device={self.device})"


def mx_quantize(x: torch.Tensor, splits: Optional[torch.Tensor] = None, scatter_index: Optional[torch.Tensor] = None) -> MXTensor:
    """Quantise x [..., N, K] (fp32, bf16 or fp16; K a multiple of 32): scale 2^(floor(log2 max|x|) - 2) for every 32
    values, values rounded to nearest, ties to even, at most 6 in magnitude. Values among which there is an infinity or a NaN
    become NaN, all 32.
    With `splits` and `scatter_index` (as `calc_scatter_index` makes them) the tokens x [ntokens, K] go into the order of
    their experts on the way, as in `moe_permute`: the result has ntokens * topk rows, and the rows past sum(splits) are
    zero. Has no gradient."""
    shape = x.shape
    if not (_on_device(x) and len(shape) >= 2 and x.dtype in _FLOATS and shape[-1] >= BLOCK and shape[-1] % BLOCK == 0):
        raise RuntimeError("mx_quantize: x must be a fp32, bf16 or fp16 [..., N, K] tensor on the current CUDA device, K a multiple of 32")
    if x.requires_grad and torch.is_grad_enabled():
        raise RuntimeError("mx_quantize has no gradient: detach x, or call it under torch.no_grad()")
    if _forward_ad._current_level >= 0:
        _refuse_tangent("mx_quantize", x)
    n, k = shape[-2:]
    lead, batch = (), 1
    if len(shape) > 2:
        lead = tuple(shape[:-2])
        batch = math.prod(lead)
    _check_size("mx_quantize", batch * n, k)
    if lead:
        x = x.contiguous()
        ldx = k  # (a contiguous tensor's stride along a dimension of one row may be any number)
    else:
        if x.stride(1) != 1:
            x = x.contiguous()
        ldx = x.stride(0) if n > 1 else k
    out_rows, topk, nexperts = n, 0, 0
    if scatter_index is not None:
        if splits is None or lead:
            raise RuntimeError("mx_quantize: into the order of experts go [ntokens, K] tokens, with splits and scatter_index")
        ntokens, topk = _check_index("mx_quantize", x.get_device(), splits, scatter_index)
        if ntokens != n:
            raise RuntimeError(f"mx_quantize: scatter_index has {ntokens} tokens, not {n}")
        out_rows, nexperts = n * topk, splits.shape[0]
    elif splits is not None:
        raise RuntimeError("mx_quantize: splits and scatter_index belong together")
    t = MXTensor.__new__(MXTensor)
    t.lead, t.rows, t.k, t._dev = lead, out_rows, k, x.get_device()
    at = (batch * out_rows * (k // 2) + 15) & ~15  # where the scales start
    t._store = x.new_empty(at + batch * ((out_rows + 127) // 128) * ((k + 127) // 128) * 512, dtype=torch.uint8)
    t._data = t._blocks = None
    t._data_ptr = t._store.data_ptr()
    t._blocks_ptr = t._data_ptr + at
    _lib.check(_lib.load().fluxb_mx_quantize(x.data_ptr(), fluxb_dtype(x.dtype), batch, n, k, ldx, t._data_ptr, t._blocks_ptr,
                                             _ptr(splits), nexperts, _ptr(scatter_index), topk, _cur_stream()))
    return t


def _like(q: MXTensor) -> torch.Tensor:
    return q._data if q._store is None else q._store


def mx_dequantize(q: MXTensor, dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """The values that `q` stands for, as fp32, bf16 or fp16 (exact in bf16 but beyond its range)."""
    if not (isinstance(q, MXTensor) and q._dev == _cur_device()):
        raise RuntimeError("mx_dequantize: q must be an MXTensor on the current CUDA device")
    if dtype not in _FLOATS:
        raise RuntimeError("mx_dequantize: the output must be fp32, bf16 or fp16")
    out = _like(q).new_empty((*q.lead, q.rows, q.k), dtype=dtype)
    _lib.check(_lib.load().fluxb_mx_dequantize(q._data_ptr, q._blocks_ptr, math.prod(q.lead), q.rows, q.k, fluxb_dtype(dtype), out.data_ptr(), _cur_stream()))
    return out


def _check_operands(name: str, x: MXTensor, w: MXTensor, wdim: int, output_dtype: torch.dtype) -> None:
    if not (isinstance(x, MXTensor) and isinstance(w, MXTensor) and not x.lead and len(w.lead) == wdim - 2):
        raise RuntimeError(f"{name}: operands must be MXTensors, [rows, K] and {'[N, K]' if wdim == 2 else '[nexperts, N, K]'}")
    if not x._dev == w._dev == _cur_device():
        raise RuntimeError(f"{name}: operands must be on the current CUDA device")
    if x.k != w.k:
        raise RuntimeError(f"{name}: weight K {w.k} != input K {x.k}")
    if x.rows >= 1 << 31 or w.rows >= 1 << 31:
        raise RuntimeError(f"{name}: {x.rows} x {w.rows} is too large")
    if output_dtype not in _FLOATS:
        raise RuntimeError(f"{name}: the output must be fp32, bf16 or fp16")


def _output(name: str, output: Optional[torch.Tensor], rows: int, n: int, dtype: torch.dtype, like: torch.Tensor) -> torch.Tensor:
    if output is None:
        return like.new_empty((rows, n), dtype=dtype)
    _check(_on_device(output) and tuple(output.shape) == (rows, n) and output.dtype == dtype and output.is_contiguous(),
           f"{name}: output has the wrong shape, dtype or layout")
    return output


def mx_gemm(x: MXTensor, w: MXTensor, bias: Optional[torch.Tensor] = None, output_dtype: torch.dtype = torch.bfloat16,
            output: Optional[torch.Tensor] = None, tuning=None) -> torch.Tensor:
    """y[M, N] = x[M, K] . w[N, K]^T (+ bias [N] of the output's type): exact products, summed in fp32, rounded once. M, N of
    any size."""
    _check_operands("mx_gemm", x, w, 2, output_dtype)
    m, n = x.rows, w.rows
    if bias is not None:
        _check(_on_device(bias) and bias.dtype == output_dtype and tuple(bias.shape) in ((n,), (1, n)) and bias.is_contiguous(),
               "mx_gemm: bias must be a contiguous [N] tensor of the output's type")
        if bias.requires_grad and torch.is_grad_enabled():
            raise RuntimeError("mx_gemm has no gradient: detach the bias, or call it under torch.no_grad()")
        if _forward_ad._current_level >= 0:
            _refuse_tangent("mx_gemm", bias)
    out = _output("mx_gemm", output, m, n, output_dtype, _like(x))
    if n == 0:
        return out
    comm = _comm()
    _lib.check(_lib.load().fluxb_mx_gemm(comm.handle, x._data_ptr, x._blocks_ptr, w._data_ptr, w._blocks_ptr, out.data_ptr(), m, n, x.k,
                                         fluxb_dtype(output_dtype), _ptr(bias), _tuning(tuning), _cur_stream()))
    return out


def mx_grouped_gemm(x: MXTensor, w: MXTensor, splits: torch.Tensor, output_dtype: torch.dtype = torch.bfloat16,
                    output: Optional[torch.Tensor] = None, tuning=None) -> torch.Tensor:
    """The experts' products: rows of x [rows, K] in the order of their experts, splits[e] of them for expert e (int32
    [nexperts], on the GPU: nothing is read back), times w [nexperts, N, K]. Rows past sum(splits) are not written: they
    stay as they were in a given `output`, and are undefined in a fresh one."""
    _check_operands("mx_grouped_gemm", x, w, 3, output_dtype)
    nexperts, n, rows = w.lead[0], w.rows, x.rows
    if not (splits.get_device() == x._dev and splits.dtype is torch.int32 and tuple(splits.shape) == (nexperts,) and splits.is_contiguous()):
        raise RuntimeError(f"mx_grouped_gemm: splits must be a contiguous int32 [{nexperts}] tensor on the current CUDA device")
    out = _output("mx_grouped_gemm", output, rows, n, output_dtype, _like(x))
    if n == 0 or nexperts == 0:
        return out
    lib = _lib.load()
    workspace = _like(x).new_empty(lib.fluxb_mx_grouped_workspace_bytes(rows, nexperts, x.k))
    comm = _comm()
    _lib.check(lib.fluxb_mx_grouped_gemm(comm.handle, x._data_ptr, x._blocks_ptr, rows, w._data_ptr, w._blocks_ptr, nexperts,
                                         splits.data_ptr(), out.data_ptr(), n, x.k, fluxb_dtype(output_dtype), workspace.data_ptr(), _tuning(tuning),
                                         _cur_stream()))
    return out
